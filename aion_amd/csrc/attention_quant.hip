// Attention over caches held in 8 or 4 bits (the layout: cache_quant.h). For query row r, visible keys t and 32-element blocks j of a head
//   S[r,t] = scale * sum_j sk[t,j] * (q[r,j] . ck[t,j]),   P = softmax(S),   O[r,j] = sum_t P[r,t] * sv[t,j] * cv[t,j]
// with codes c and scales s as they are stored. Sums, the running maximum and the scales are f32 throughout.
//
// quant_generic_kernel - any head size: one wavefront per query row, keys 64 at a time, in f32. Slow; it exists so that every shape the
//   step allows has a path.
#include "attention_common.h"
#include "cache_quant.h"

namespace attn {
namespace {
using cq::Cache;

struct QuantArgs {
    const void *q;
    float *out;
    Cache k, v;
    const int *positions, *kv_lengths;
    int B, L, T, Tp, Hq, Hkv, groups, d_k, d_v;
    int ring;      // rolling caches: T (logical key t lives in row t % T); 0: row t is key t
    int q_dtype;
    float scale, soft_cap;
    unsigned win_left, win_right, win_chunk;
};

// visible keys [lo, hi) of query `li` of sequence b
__device__ __forceinline__ void visible(const QuantArgs &a, int b, int li, int &lo, int &hi) {
    const int kv_end = clip_kv_end(a.ring, a.T, a.kv_lengths ? a.kv_lengths[b] : a.T);
    const int pos = a.positions ? a.positions[(size_t)b * a.L + li] : li;
    window_keys(a.win_left, a.win_right, a.win_chunk, max(pos, 0), kv_end, lo, hi);
    clip_to_ring(a.ring, kv_end, lo, hi);
}

template <int DT>
__device__ __forceinline__ float code_at(const unsigned char *row, int col) {
    if constexpr (DT == AIONHIP_Q8_0) return (float)((int)row[col] - 128);
    return (float)((int)(row[col >> 1] >> (4 * (col & 1)) & 15) - 8);
}

constexpr int GENERIC_HEAD = 1024;      // most elements of a head: a wavefront keeps its query and its output row in LDS
template <int DT>
__global__ __launch_bounds__(256) void quant_generic_kernel(QuantArgs a) {
    extern __shared__ float generic_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = (size_t)blockIdx.x * 4 + wave;
    if (row >= (size_t)a.B * a.L * a.Hq) return;
    float *qs = generic_lds + wave * (a.d_k + a.d_v), *acc = qs + a.d_k;
    const int hq = (int)(row % a.Hq), li = (int)(row / a.Hq % a.L), b = (int)(row / ((size_t)a.Hq * a.L));
    const size_t unit = (size_t)b * a.Hkv + hq / a.groups;
    const int rb_k = DT == AIONHIP_Q8_0 ? a.d_k : a.d_k / 2, rb_v = DT == AIONHIP_Q8_0 ? a.d_v : a.d_v / 2;
    const unsigned char *kc = a.k.codes + unit * a.Tp * rb_k, *vc = a.v.codes + unit * a.Tp * rb_v;
    const __half *ks = a.k.scales + unit * (a.d_k / 32) * a.Tp, *vs = a.v.scales + unit * (a.d_v / 32) * a.Tp;
    int lo, hi;
    visible(a, b, li, lo, hi);
    for (int j = lane; j < a.d_k; j += 64) qs[j] = load_scalar(a.q, a.q_dtype, row * a.d_k + j);
    for (int j = lane; j < a.d_v; j += 64) acc[j] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int t0 = lo; t0 < hi; t0 += 64) {
        const int t = t0 + lane;
        float s = -INFINITY;
        if (t < hi) {
            const size_t r = (size_t)phys_key(a.ring, t);
            s = 0.f;
            for (int j = 0; j < a.d_k / 32; ++j) {
                float dot = 0.f;
                for (int i = 0; i < 32; ++i) dot = fmaf(qs[j * 32 + i], code_at<DT>(kc + r * rb_k, j * 32 + i), dot);
                s = fmaf(dot, __half2float(ks[(size_t)j * a.Tp + r]), s);
            }
            s *= a.scale;
            if (a.soft_cap > 0.f) s = a.soft_cap * tanhf(s / a.soft_cap);
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float shrink = m > -INFINITY ? exp2f((m - m_new) * LOG2E) : 0.f;
        const float p = t < hi && s != -INFINITY ? exp2f((s - m_new) * LOG2E) : 0.f;
        l = l * shrink + wave_sum(p);
        m = m_new;
        for (int j0 = 0; j0 < a.d_v; j0 += 64) {
            const int j = min(j0 + lane, a.d_v - 1);                         // (every lane hands its probability on, also where there is no column for it)
            float o = acc[j] * shrink;
            for (int i = 0; i < min(64, hi - t0); ++i) {
                const size_t r = (size_t)phys_key(a.ring, t0 + i);
                o = fmaf(__shfl(p, i, 64), code_at<DT>(vc + r * rb_v, j) * __half2float(vs[(size_t)(j / 32) * a.Tp + r]), o);
            }
            if (j0 + lane < a.d_v) acc[j] = o;
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    for (int j = lane; j < a.d_v; j += 64) a.out[row * a.d_v + j] = acc[j] * inv;
}

template <int DT>
int launch_generic(aionhip_ctx *ctx, const QuantArgs &a) {
    const size_t rows = (size_t)a.B * a.L * a.Hq;
    if ((rows + 3) / 4 > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: dimension too large");
    ProfScope scope(ctx, "attn_quant_generic");
    launch_k(ctx, quant_generic_kernel<DT>, dim3((unsigned)((rows + 3) / 4)), dim3(256), (size_t)4 * (a.d_k + a.d_v) * sizeof(float), a);
    LAUNCH_CHECK(ctx, "attn_quant_generic");
    return AIONHIP_OK;
}

template <int DT>
int launch(aionhip_ctx *ctx, const QuantArgs &a) {
    return launch_generic<DT>(ctx, a);
}

}  // namespace

// The step over quantized caches; its operands have been checked as far as every cache type wants them checked (attention.hip).
int run_attention_quant(aionhip_ctx *ctx, const aionhip_attention *p) {
    if (p->d_k % 32 != 0 || p->d_v % 32 != 0) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention: head sizes over a quantized cache are multiples of 32");
    if (p->d_k > GENERIC_HEAD || p->d_v > GENERIC_HEAD) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: head sizes above %d over a quantized cache", GENERIC_HEAD);
    if ((p->k | p->v) & 15) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention: a quantized cache begins at a multiple of 16 bytes");
    if (p->t_kv && (!aionhip_cache_quant_bytes(p->kv_dtype, p->batch, p->t_kv, p->h_kv, p->d_k) || !aionhip_cache_quant_bytes(p->kv_dtype, p->batch, p->t_kv, p->h_kv, p->d_v)))
        return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: dimension too large");
    QuantArgs a{};
    a.q = (const void *)(uintptr_t)p->q;
    a.out = (float *)(uintptr_t)p->out;
    a.k = cq::view(p->k, p->kv_dtype, p->batch, p->t_kv, p->h_kv, p->d_k);
    a.v = cq::view(p->v, p->kv_dtype, p->batch, p->t_kv, p->h_kv, p->d_v);
    a.positions = (const int *)(uintptr_t)p->query_positions;
    a.kv_lengths = (const int *)(uintptr_t)p->kv_lengths;
    a.B = (int)p->batch; a.L = (int)p->l_q; a.T = (int)p->t_kv; a.Tp = (int)cq::padded(p->t_kv); a.Hq = (int)p->h_q; a.Hkv = (int)p->h_kv;
    a.groups = a.Hq / a.Hkv;
    a.d_k = (int)p->d_k; a.d_v = (int)p->d_v;
    a.ring = p->rolling ? a.T : 0;
    a.q_dtype = p->q_dtype;
    a.scale = p->scale; a.soft_cap = p->attn_logits_soft_cap;
    a.win_left = p->window_left; a.win_right = p->window_right; a.win_chunk = p->window_chunk;
    return p->kv_dtype == AIONHIP_Q8_0 ? launch<AIONHIP_Q8_0>(ctx, a) : launch<AIONHIP_Q4_0>(ctx, a);
}

}  // namespace attn
