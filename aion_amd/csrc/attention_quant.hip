// Attention over caches held in 8 or 4 bits (the layout: cache_quant.h). For query row r, visible keys t and 32-element blocks j of a head
//   S[r,t] = scale * sum_j sk[t,j] * (q[r,j] . ck[t,j]),   P = softmax(S),   O[r,j] = sum_t P[r,t] * sv[t,j] * cv[t,j]
// with codes c and scales s as they are stored. Sums, the running maximum and the scales are f32 throughout.
//
// quant_decode_kernel - up to 64 or 128 query rows of a key head, head sizes 64, 128, 256: bound by memory over long caches, by latency over short ones.
// quant_prompt_kernel - more rows: bound by instruction issue.
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
    const int keys = hi - lo;                                                // (counted from the first: a ring's keys may end where int does)
    for (int t0 = 0; t0 < keys; t0 += 64) {
        const int t = t0 + lane;
        float s = -INFINITY;
        if (t < keys) {
            const size_t r = (size_t)phys_key(a.ring, lo + t);
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
        const float p = t < keys && s != -INFINITY ? exp2f((s - m_new) * LOG2E) : 0.f;
        l = l * shrink + wave_sum(p);
        m = m_new;
        for (int j0 = 0; j0 < a.d_v; j0 += 64) {
            const int j = min(j0 + lane, a.d_v - 1);                         // (every lane hands its probability on, also where there is no column for it)
            float o = acc[j] * shrink;
            for (int i = 0; i < min(64, keys - t0); ++i) {
                const size_t r = (size_t)phys_key(a.ring, lo + t0 + i);
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

// ---------------------------------------------------------------------------------------------------------------------- few query rows
using h2 = __attribute__((ext_vector_type(2))) _Float16;

// In registers where the compiler would use a constant: one operand of an instruction may be a scalar, so that a mask and an exponent merge into one
// instruction only if one of them is a vector register; and a product by one or plus zero is replaced by more instructions than it was.
struct Constants {
    unsigned one = 0x64006400u;                      // two f16 1024
    float zero = 0.f, minus = -1.f;
    __device__ __forceinline__ Constants() { asm volatile("" : "+v"(one), "+v"(zero), "+v"(minus)); }
};
// Codes as the half-precision numbers they are, offset taken off: a code under the mantissa of 1024 is 1024 + code, and the rest is exact.
// 4 bits: eight codes of a word, in the order 0 4 1 5 2 6 3 7 (a mask takes every fourth nibble of them).
__device__ __forceinline__ u32x4 halves_q4(const Constants &k, unsigned w) {
    const unsigned m = 0x000F000Fu, v = w >> 8;
    const h2 low{(_Float16)-1032.f, (_Float16)-1032.f}, high{(_Float16)-72.f, (_Float16)-72.f}, by{(_Float16)0.0625f, (_Float16)0.0625f};
    const h2 a = __builtin_bit_cast(h2, (w & m) | k.one) + low, b = __builtin_bit_cast(h2, (w & (m << 4)) | k.one) * by + high;
    const h2 c = __builtin_bit_cast(h2, (v & m) | k.one) + low, d = __builtin_bit_cast(h2, (v & (m << 4)) | k.one) * by + high;
    return u32x4{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, c), __builtin_bit_cast(unsigned, d)};
}
// 8 bits: the eight codes of two words, in order
__device__ __forceinline__ u32x4 halves_q8(const Constants &k, unsigned w0, unsigned w1) {
    const h2 off{(_Float16)-1152.f, (_Float16)-1152.f};
    auto pair = [&](unsigned w, unsigned sel) {
        return __builtin_bit_cast(unsigned, __builtin_bit_cast(h2, __builtin_amdgcn_perm(k.one, w, sel)) + off);
    };
    return u32x4{pair(w0, 0x07010700u), pair(w0, 0x07030702u), pair(w1, 0x07010700u), pair(w1, 0x07030702u)};
}
// The same for keys under few query rows: the codes as they are stored, under the mantissa of zero, are f16 numbers of 2^-24 a step, which the matrix pipe
// multiplies exactly, subnormal or not. Fewer instructions to a pair; the offset is taken back as -offset * sum(q), with which a product begins. The pipe lines products
// up by their exponents and a subnormal number's leading zeros are lost below: a nibble stands sixteen times higher, 2^-20 a step (relative error 3e-7; 2.5e-6
// with every other one in the lowest four bits).
constexpr float raw_step(int dt) { return dt == AIONHIP_Q8_0 ? 1.f / 16777216.f : 1.f / 1048576.f; }
__device__ __forceinline__ u32x4 raw_q4(unsigned w) {
    const unsigned m = 0x00F000F0u;
    return u32x4{(w << 4) & m, w & m, (w >> 4) & m, (w >> 8) & m};
}
__device__ __forceinline__ u32x4 raw_q8(unsigned w0, unsigned w1) {
    return u32x4{__builtin_amdgcn_perm(0u, w0, 0x0C010C00u), __builtin_amdgcn_perm(0u, w0, 0x0C030C02u), __builtin_amdgcn_perm(0u, w1, 0x0C010C00u),
                 __builtin_amdgcn_perm(0u, w1, 0x0C030C02u)};
}
// element of a block that lies in slot j of a query operand, and key of eight in slot j of a P operand: the order the codes come out of their words
template <int DT>
__device__ __forceinline__ constexpr int element_slot(int j) { return DT == AIONHIP_Q8_0 ? j : (j >> 1) + (j & 1) * 4; }
template <int DT>
__device__ __forceinline__ constexpr int key_slot(int j) { return DT == AIONHIP_Q8_0 ? j : (j & 4) + (j >> 1 & 1) + (j & 1) * 2; }

__device__ __forceinline__ void swap32(unsigned &a, unsigned &b) {
    const auto x = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = x[0];
    b = x[1];
}
__device__ __forceinline__ void swap16(unsigned &a, unsigned &b) {
    const auto x = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = x[0];
    b = x[1];
}
// Half k (0: low) of a pair of scales times x, plus y: one mixed-precision multiply-add
__device__ __forceinline__ float fma_half(float x, unsigned pair, int k, float y) {
    const h2 h = __builtin_bit_cast(h2, pair);
    return fmaf(x, (float)(k ? h.y : h.x), y);
}
// In the body of a rare condition: or the compiler computes what it changes for every tile and selects, and has both forms in registers
__device__ __forceinline__ void stay_branch() { asm volatile(""); }
__device__ __forceinline__ unsigned pack_half(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b)); }

// A query row times a power of two that leaves its largest element in [2^8, 2^9): shrink = 2^(8 - e), grow = 2^(e - 8), both normal floats. A row without a finite
// maximum stays as it is.
struct Power2 {
    float shrink, grow;
    __device__ __forceinline__ explicit Power2(float amax) {
        const unsigned e = amax < INFINITY ? min(max(__float_as_uint(amax) >> 23, 10u), 252u) - 8u : 127u;
        shrink = __uint_as_float((254u - e) << 23);
        grow = __uint_as_float(e << 23);
    }
};
// eight elements of each block of a query row, from element `at` of the queries on (any alignment their type allows)
template <int KK>
__device__ __forceinline__ void load_query(const QuantArgs &a, size_t at, float (&x)[KK][8]) {
    if (a.q_dtype == AIONHIP_F32) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) __builtin_memcpy(x[kk], (const float *)a.q + at + kk * 32, 32);
        return;
    }
    unsigned short h[KK][8];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) __builtin_memcpy(h[kk], (const unsigned short *)a.q + at + kk * 32, 16);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[kk][j] = a.q_dtype == AIONHIP_F16 ? __half2float(__ushort_as_half(h[kk][j])) : bf16_bits_to_f32(h[kk][j]);
}
// Eight elements of a block times `by` as the sum of two f16 each, in the order of K's codes. Returns the sum of what the operands hold.
template <int DT>
__device__ __forceinline__ float split_query(const float (&q)[8], float by, u32x4 (&op)[2]) {
    float x[8], y[8], sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = q[element_slot<DT>(j)] * by;
        const float high = (float)(_Float16)x[j];
        y[j] = x[j] - high;
        sum += high + (float)(_Float16)y[j];
    }
    op[0] = u32x4{pack2<AIONHIP_F16>(x[0], x[1]), pack2<AIONHIP_F16>(x[2], x[3]), pack2<AIONHIP_F16>(x[4], x[5]), pack2<AIONHIP_F16>(x[6], x[7])};
    op[1] = u32x4{pack2<AIONHIP_F16>(y[0], y[1]), pack2<AIONHIP_F16>(y[2], y[3]), pack2<AIONHIP_F16>(y[4], y[5]), pack2<AIONHIP_F16>(y[6], y[7])};
    return sum;
}
// The largest of three (fmaxf multiplies what it cannot see the origin of by one first, to quiet a signalling NaN that none of these can be). Not for what the matrix
// pipe wrote: the wait for its results is the compiler's, and it does not look in here.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// cap * tanh(s * by) * log2(e), as 1 - 2 / (e^2x + 1): off by less than 2^-22 of the cap wherever s lies, without a branch
__device__ __forceinline__ float capped(float s, float by, float cap) {
    const float t = __builtin_amdgcn_exp2f(s * by * (2.f * LOG2E));
    return cap * LOG2E * fmaf(-2.f, __builtin_amdgcn_rcpf(t + 1.f), 1.f);
}

// N transposing reads (8 rows x 16 bytes within sixteen lanes: lane 2 r + q gives the address of half q of row r, lane i gets byte i of the rows), complete
// when the statement is. The builtin would wait for every load in flight, whose target LDS may be.
template <int N>
__device__ __forceinline__ void read_transposed(const unsigned (&at)[N], u32x2 (&r)[N]) {
    static_assert(N == 1 || N == 2 || N == 4 || N == 8, "reads to a statement");
    if constexpr (N == 1)
        asm volatile("ds_read_b64_tr_b8 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(r[0]) : "v"(at[0]) : "memory");
    else if constexpr (N == 2)
        asm volatile("ds_read_b64_tr_b8 %0, %2\n\tds_read_b64_tr_b8 %1, %3\n\ts_waitcnt lgkmcnt(0)" : "=&v"(r[0]), "=&v"(r[1]) : "v"(at[0]), "v"(at[1]) : "memory");
    else if constexpr (N == 4)
        asm volatile("ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\tds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]) : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]) : "memory");
    else
        asm volatile("ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\tds_read_b64_tr_b8 %2, %10\n\tds_read_b64_tr_b8 %3, %11\n\t"
                     "ds_read_b64_tr_b8 %4, %12\n\tds_read_b64_tr_b8 %5, %13\n\tds_read_b64_tr_b8 %6, %14\n\tds_read_b64_tr_b8 %7, %15\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7]) : "memory");
}
// sixteen bytes from each of four places, complete when the statement is
__device__ __forceinline__ void read_four(unsigned at, u32x4 (&r)[4]) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]) : "v"(at), "n"(1024), "n"(2 * 1024), "n"(3 * 1024) : "memory");
}

// Key segments: every workgroup of a row tile takes a share of its sequence's 64-key tiles and leaves sums over them; `parts` holds those, `tickets`
// (not null) lets the workgroup that ends last add them up, otherwise quant_merge_kernel does.
struct Split {
    float *parts;
    unsigned *tickets;
    int nseg, row_tiles;
};
constexpr int NW = 4;                       // wavefronts of a workgroup
constexpr int MAX_SEG = 256;                // most segments of a row tile

template <int D, int REP>
struct Part {                               // a row tile's sums: o [rows][D], then (reference, sum) of its 16 columns
    static constexpr int ROWS = 16 / REP, FLOATS = ROWS * D + 32;
};

// Sums of a row tile's segments -> output rows. A thread has four columns of a row and every `groups`-th run of eight segments, all of a run's loads in
// flight at once (reference, sum and columns: one memory round trip); the groups meet in LDS. The elements are [first, last) of rows x D / 4.
// `load(2 or 4, i)`: that many floats of the tile's parts from the i-th on.
constexpr int RUN = 8;
template <int D, int REP, class Load, class Store>
__device__ __forceinline__ void merge_parts(int nseg, int first, int last, int groups, f32x4 *meet_o, float2 *meet_s, Load &&load, Store &&store) {
    constexpr int ROWS = Part<D, REP>::ROWS, FLOATS = Part<D, REP>::FLOATS;
    const int per = NW * 64 / groups, group = (int)threadIdx.x / per, runs = (nseg + RUN - 1) / RUN;
    for (int e0 = first; e0 < last; e0 += per) {
        const int e = min(e0 + (int)threadIdx.x % per, last - 1), row = e / (D / 4), col = e % (D / 4) * 4, c = (col / 32) % REP * ROWS + row;
        const bool mine = group < groups && e0 + (int)threadIdx.x % per < last;
        float ref = REF_NONE, l = 0.f;
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int run = group; run < runs && mine; run += groups) {
            u32x2 st[RUN];
            u32x4 x[RUN];
#pragma unroll
            for (int u = 0; u < RUN; ++u) {
                const size_t part = (size_t)min(run * RUN + u, nseg - 1) * FLOATS;
                st[u] = load(std::integral_constant<int, 2>{}, part + ROWS * D + 2 * c);
                x[u] = load(std::integral_constant<int, 4>{}, part + row * D + col);
            }
            float top = ref;
#pragma unroll
            for (int u = 0; u < RUN; ++u) top = fmaxf(top, __uint_as_float(st[u].x));
            const float keep = __builtin_amdgcn_exp2f(ref - top);
            o *= keep;
            l *= keep;
            ref = top;
#pragma unroll
            for (int u = 0; u < RUN; ++u)
                if (run * RUN + u < nseg) {
                    const float f = __builtin_amdgcn_exp2f(__uint_as_float(st[u].x) - top);
                    l += __uint_as_float(st[u].y) * f;
                    o += __builtin_bit_cast(f32x4, x[u]) * f;
                }
        }
        if (groups > 1) {
            __syncthreads();                                                  // (what the threads met in before has been read)
            if (group < groups) {
                meet_o[threadIdx.x] = o;
                meet_s[threadIdx.x] = make_float2(ref, l);
            }
            __syncthreads();
            if (group == 0) {
                float top = ref;
                for (int k = 1; k < groups; ++k) top = fmaxf(top, meet_s[threadIdx.x + k * per].x);
                const float keep = __builtin_amdgcn_exp2f(ref - top);
                o *= keep;
                l *= keep;
                for (int k = 1; k < groups; ++k) {
                    const float2 st = meet_s[threadIdx.x + k * per];
                    const float f = __builtin_amdgcn_exp2f(st.x - top);
                    l += st.y * f;
                    o += meet_o[threadIdx.x + k * per] * f;
                }
            }
        }
        if (group == 0 && mine) store(row, col, o * (l != 0.f ? 1.f / l : 0.f));
    }
}

// Few query rows over many keys. A workgroup has one row tile and a segment of the keys, its wavefronts 64 keys at a time, each with a running maximum,
// sum and output of its own; they meet in LDS, the segments in memory.
//   S^T[keys x cols] = K . Q^T: the operands are the codes as f16, exact, and the query row times a power of two as the sum of two f16 (22 bits). A
//     product of the matrix pipe spans 32 elements, a block, so that the scale goes onto its result.
//   O^T[dv x cols] += V^T . P'^T with P'[t] = P[t] * sv[t, block]: the scale of a value differs from key to key and can only be in P. P' is a sum of two f16 as well.
// The matrix pipe has 16 columns; few rows leave most of them idle, and the vector pipe is what bounds the kernel beside memory (unpacking two codes costs
// more than multiplying them). So the 16 columns are REP groups of 16 / REP rows, and group u works for the blocks j = u mod REP only: its query is
// zero elsewhere, REP blocks add up in one chain of products and one scale per key suffices for all of them (the groups' scores are added at the end), and
// its P' carries the scales of its own blocks, so that P' is made once per REP blocks instead of once per block. What a column accumulates in other
// groups' value columns is not read.
// Keys of a tile of TK: sub-tile h, row m holds key TK / 4 * (m / 4) + 4 h + m % 4, which gives the lanes 16 g .. of a result neighbouring keys, whose
// scales are one load or two. V goes to LDS as it is and comes back transposed, eight keys of a byte at a time: of two value columns where a byte holds two.
// P' is kept where f16 is accurate: a column's reference is its maximum minus a power of two that keeps the largest P' seen (it decays as the maximum grows)
// between 2^9 and 2^15; the low part then ends 2^-34 below it. A value that is not finite has no part in it. The shift has an end, 2^MOST_BIAS: where the keys with
// the highest scores have values of zero (a block that f16 holds no scale of, a row of zeros), P' comes from keys far below them, and P itself, whose largest is
// 2^bias, is what leaves f32's range first. Beyond the end P' keeps an absolute 2^-24, which is 2^-104 of the normalizer; and P, its sum and what
// a merge takes one by the other stay finite with room (P' at most 2^96, a part that a merge loses below 2^-42 of the whole).
// Measured (32 query heads on 8 of 128): one token over 131072 keys in 8 bits 57 us, 5.0 TB/s (a copy reaches 5.1, a read 6.8); 32 tokens over 16384 keys
// each in 4 bits 85 us, 5.2 TB/s; one token over 531 keys of one head of 256 11.1 us, of which 4 are the launch and 3 the meeting of its segments.
// Tiles are 64 keys, 32 at head size 256; there, and where sixteen rows share the columns, the query's operands lie in LDS as well: the registers hold no more.
constexpr float MOST_BIAS = 80.f;
constexpr int decode_waves(int d, int rep) { return d > 128 || (d == 128 && rep < 4) ? 2 : d == 128 || rep == 1 ? 3 : 4; }      // to a SIMD
template <int DT, int D, int REP>
struct DecodeCfg {
    static constexpr int TK = D > 128 ? 32 : 64, RB = DT == AIONHIP_Q8_0 ? D : D / 2, ROWS = 16 / REP;
    static constexpr bool Q_LDS = D >= 128;
    static constexpr bool PV_TWICE = D / 32 / REP * (TK / 4) > 32;              // P' is made once for its maximum and again for its use
    static constexpr int Q_BYTES = Q_LDS ? D / 32 * (2048 + 64) + 256 : 0, V_BYTES = NW * TK * RB;
    static constexpr int MEET_BYTES = NW * (ROWS * (D + 4) + 32) * 4, MERGE_BYTES = NW * 64 * 24;
    static constexpr int MOST = MEET_BYTES > MERGE_BYTES ? MEET_BYTES : MERGE_BYTES;
    static constexpr int LDS_BYTES = Q_BYTES + V_BYTES > MOST ? Q_BYTES + V_BYTES : MOST;
};
template <int DT, int D, int REP>
__global__ __launch_bounds__(NW * 64, decode_waves(D, REP)) void quant_decode_kernel(QuantArgs a, Split sp) {
    using Cfg = DecodeCfg<DT, D, REP>;
    constexpr int ROWS = 16 / REP, KK = D / 32, MT = D / 16, SETS = KK / REP;
    constexpr int TK = Cfg::TK, H = TK / 16, KG = TK / 4;                                  // keys of a tile; its sub-tiles; keys of a lane
    constexpr int RB = Cfg::RB, CH = RB / 16, KD = RB / 16;                                // bytes of a row; its 16-byte chunks; words of a K operand
    constexpr int FLOATS = Part<D, REP>::FLOATS;
    static_assert(KK % REP == 0 && SETS >= 1, "whole groups of blocks");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int rt = sp.row_tiles == 1 ? 0 : (int)blockIdx.x / sp.nseg, seg = (int)blockIdx.x - rt * sp.nseg, hk = (int)blockIdx.y, b = (int)blockIdx.z;
    const int unit = b * a.Hkv + hk, rows_total = a.L * a.groups;
    const int rows = min(ROWS, rows_total - rt * ROWS);
    const int sub = n / ROWS;

    // ---- this lane's query row (columns past the last row repeat it) and its visible keys
    const int r = rt * ROWS + min(n % ROWS, rows - 1), li = a.L == 1 ? 0 : r / a.groups, hq = hk * a.groups + (r - li * a.groups);
    const size_t qbase = (((size_t)b * a.L + li) * a.Hq + hq) * D;
    constexpr int E0G = DT == AIONHIP_Q8_0 || D == 64;                  // where a lane's eight elements of a block begin, by how K is loaded
    const int e0 = E0G ? (g & 1) * 16 + (g >> 1) * 8 : g * 8;
    // (each wavefront has the blocks it makes operands of; all of them where they stay in its registers)
    constexpr int QB = Cfg::Q_LDS ? KK / NW : KK;
    const int first_block = Cfg::Q_LDS ? wave * QB : 0;
    float qx[QB][8];
    load_query<QB>(a, qbase + first_block * 32 + e0, qx);
    int lo, hi, uni_lo, uni_hi, full_lo, full_hi;
    visible(a, b, li, lo, hi);
    if (hi <= lo) lo = hi = 0;
    if (a.L == 1) {                                                          // one token: every row sees the same keys
        uni_lo = full_lo = __builtin_amdgcn_readfirstlane(lo);
        uni_hi = full_hi = __builtin_amdgcn_readfirstlane(hi);
    } else {
        uni_lo = rows16_min_i(hi > lo ? lo : INT_MAX), uni_hi = rows16_max_i(hi);
        full_lo = rows16_max_i(lo), full_hi = rows16_min_i(hi);
    }
    const int kv_end = clip_kv_end(a.ring, a.T, a.kv_lengths ? a.kv_lengths[b] : a.T);

    // ---- the tiles of the segment. A ring is walked by its rows: row p holds step base + p before the row the next step goes to, and a round less from there on.
    const int wrap = a.ring ? kv_end % a.ring : INT_MAX, base = a.ring ? kv_end - wrap : 0;
    int first_tile = 0, count = 0;
    const int all_tiles = (a.T + TK - 1) / TK;
    if (uni_hi > uni_lo) {
        const int p0 = phys_key(a.ring, uni_lo);
        first_tile = p0 / TK;
        const long span = (long)(p0 % TK) + (uni_hi - uni_lo);
        count = (int)min((long)all_tiles, (span + TK - 1) / TK + (a.ring && (long)p0 + (uni_hi - uni_lo) > a.ring ? 1 : 0));
    }
    const int per = sp.nseg == 1 ? count : (count + sp.nseg - 1) / sp.nseg;
    const int t_end = min((seg + 1) * per, count);
    int t = seg * per + wave;
    auto tile_of = [&](int i) { const int x = first_tile + i; return x >= all_tiles ? x - all_tiles : x; };

    const size_t unit_rows = (size_t)unit * a.Tp;
    const unsigned char *kc = a.k.codes + unit_rows * RB;
    [[maybe_unused]] const unsigned char *vc = a.v.codes + unit_rows * RB;
    const __half *ks = a.k.scales + unit_rows * KK + (size_t)sub * a.Tp + g * KG, *vs = a.v.scales + unit_rows * KK + (size_t)sub * a.Tp + g * KG;
    unsigned char *v_lds = lds + Cfg::Q_BYTES + wave * (TK * RB);

    unsigned kw[H][KD];
    u32x4 ksc[SETS][KG / 8], vsc[SETS][KG / 8];
    const unsigned k_lane = (unsigned)(((n >> 2) * KG + (n & 3)) * RB + g * (KD == 2 ? 8 : 16));
    // Up to eight rows are one row tile, which reads every code once: past the caches (32 sequences of 16384 keys in 4 bits 91 -> 85 us). The row tiles of more rows read
    // a key together (8 sequences of 96 rows over 4000 keys in 8 bits: 82 us, past the caches 104).
    constexpr bool ONCE = REP > 1;
    auto load_k = [&](int i) __attribute__((always_inline)) {
        const int row0 = tile_of(i) * TK;
        const unsigned char *p = kc + (size_t)row0 * RB + k_lane;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if constexpr (KD == 2) {
                const u32x2 x = ONCE ? __builtin_nontemporal_load((const u32x2 *)(p + h * 4 * RB)) : *(const u32x2 *)(p + h * 4 * RB);
                kw[h][0] = x.x;
                kw[h][1] = x.y;
            } else {
#pragma unroll
                for (int c = 0; c < KD / 4; ++c) {
                    const u32x4 *from = (const u32x4 *)(p + h * 4 * RB + c * 64), x = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
                    for (int j = 0; j < 4; ++j) kw[h][c * 4 + j] = x[j];
                }
            }
        }
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int j = 0; j < KG / 8; ++j) ksc[s][j] = *(const u32x4 *)(ks + (size_t)s * REP * a.Tp + row0 + j * 8);
    };
    // V: 1 KB of the tile per instruction, lane after lane; chunk c of row r lies in slot c ^ f(r), f(r) = r RB / 256 in the chunk's bits, which spreads a
    // transposing read's rows over the banks. The slot is the lane's, so it is the address that is permuted.
    [[maybe_unused]] constexpr int NVI = TK * RB / 1024;
    [[maybe_unused]] const unsigned v_lane = (unsigned)((lane / CH) * RB) + (unsigned)((((lane % CH) ^ (lane >> 4)) & (CH - 1)) << 4);
    auto load_v = [&](int i) __attribute__((always_inline)) {
        const int row0 = tile_of(i) * TK;
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int j = 0; j < KG / 8; ++j) vsc[s][j] = *(const u32x4 *)(vs + (size_t)s * REP * a.Tp + row0 + j * 8);
        asm volatile("" ::: "memory");                                        // requested ahead of the codes: they are waited for first
#if defined(__HIP_DEVICE_COMPILE__)   // the builtin exists in the device pass only
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(vc + (size_t)row0 * RB), 0, TK * RB, 0x00027000);
#pragma unroll
        for (int j = 0; j < NVI; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(v_lds + j * 1024), 16, (int)(v_lane ^ (unsigned)(((4 * j) & (CH - 1)) << 4)), j * 1024, 0, ONCE ? 2 : 0);
#endif
    };

    if (t < t_end) {
        load_k(t);
        load_v(t);
    }
    // ---- Q^T: eight elements of each block, in the order of K's codes, times a power of two and the sign of the scale, in two parts
    float amax = 0.f;
#pragma unroll
    for (int kk = 0; kk < QB; ++kk)
#pragma unroll
        for (int j = 0; j < 8; j += 2) amax = max3(amax, fabsf(qx[kk][j]), fabsf(qx[kk][j + 1]));
    amax = groups4_max(amax);
    constexpr int Q_OFFSETS = KK * 2048, Q_MAXIMA = Q_OFFSETS + KK * 64;      // in LDS: the operands, the blocks' offsets by columns, the wavefronts' maxima by columns
    const unsigned q_addr = (unsigned)(size_t)(lds_void *)lds + lane * 16, n_addr = (unsigned)(size_t)(lds_void *)lds + n * 4;
    if constexpr (Cfg::Q_LDS) {                                               // (no wait for the loads in flight)
        asm volatile("ds_write_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::"v"(n_addr + Q_MAXIMA + wave * 64), "v"(amax) : "memory");
        float m0, m1, m2, m3;
        asm volatile("ds_read_b32 %0, %4 offset:%5\n\tds_read_b32 %1, %4 offset:%6\n\tds_read_b32 %2, %4 offset:%7\n\tds_read_b32 %3, %4 offset:%8\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(m0), "=&v"(m1), "=&v"(m2), "=&v"(m3)
                     : "v"(n_addr), "n"(Q_MAXIMA), "n"(Q_MAXIMA + 64), "n"(Q_MAXIMA + 128), "n"(Q_MAXIMA + 192) : "memory");
        amax = max3(max3(m0, m1, m2), m3, m3);
    }
    const Power2 by(amax);
    const float sign = a.scale < 0.f ? -by.shrink : by.shrink;
    const float row_scale = fabsf(a.scale) * (1.f / raw_step(DT)) * by.grow;
    const float to_log2 = a.soft_cap > 0.f ? 1.f : fmaxf(row_scale * LOG2E, 1e-30f);          // (not zero: the score of a key that is not seen is minus infinity)
    const float inv_cap = a.soft_cap > 0.f ? 1.f / a.soft_cap : 0.f;
    const Constants cst;
    constexpr float OFFSET = (DT == AIONHIP_Q8_0 ? -128.f : -8.f) * raw_step(DT);
    u32x4 q_op[Cfg::Q_LDS ? 1 : KK][2];
    float offset[SETS] = {};
#pragma unroll
    for (int j = 0; j < QB; ++j) {
        const int kk = first_block + j;
        u32x4 op[2];
        const float sum = split_query<DT>(qx[j], kk % REP == sub ? sign : 0.f, op);
        if constexpr (Cfg::Q_LDS) {
            asm volatile("ds_write_b128 %0, %2\n\tds_write_b128 %0, %3 offset:1024\n\tds_write_b32 %1, %4" ::"v"(q_addr + kk * 2048),
                         "v"(n_addr + Q_OFFSETS + kk * 64), "v"(op[0]), "v"(op[1]), "v"(groups4_sum(sum) * OFFSET) : "memory");
        } else {
            q_op[j][0] = op[0];
            q_op[j][1] = op[1];
            offset[j / REP] += sum;
        }
    }
    if constexpr (Cfg::Q_LDS) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int st = 0; st < SETS; ++st)
            asm volatile("ds_read_b32 %0, %1 offset:%2\n\ts_waitcnt lgkmcnt(0)" : "=&v"(offset[st]) : "v"(n_addr + sub * 64), "n"(Q_OFFSETS + st * REP * 64) : "memory");
    } else {
#pragma unroll
        for (int st = 0; st < SETS; ++st) offset[st] = groups4_sum(offset[st]) * OFFSET;
    }

    f32x4 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = REF_NONE, l_run = 0.f, bias = 16.f, largest = 0.f;          // of this column; l_run: this lane's keys

    const unsigned v_row = (unsigned)(g * KG + (n >> 1));
    const unsigned v_addr = (unsigned)(size_t)(lds_void *)v_lds + v_row * RB + (((v_row * RB / 256) & (CH - 1)) << 4) + (n & 1) * 8;

    auto tile = [&](int i, auto more_c) __attribute__((always_inline)) {
        constexpr bool more = decltype(more_c)::value;
        const int row0 = tile_of(i) * TK;
        // -- scores
        float s[KG];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int c = 0; c < (KD + 3) / 4; ++c) {
                unsigned *w = &kw[h][c * 4];
                if constexpr (KD == 2) {
                    swap32(w[0], w[1]);
                } else {
                    swap32(w[0], w[2]);
                    swap32(w[1], w[3]);
                    if constexpr (DT == AIONHIP_Q4_0) {
                        swap16(w[0], w[1]);
                        swap16(w[2], w[3]);
                    }
                }
            }
        u32x4 q4[4];
#pragma unroll
        for (int st = 0; st < SETS; ++st) {
            f32x4 d[H];
#pragma unroll
            for (int h = 0; h < H; ++h) d[h] = f32x4{offset[st], offset[st], offset[st], offset[st]};
#pragma unroll
            for (int u = 0; u < REP; ++u) {
                const int kk = st * REP + u;
                if constexpr (Cfg::Q_LDS)
                    if (kk % 2 == 0) read_four(q_addr + kk * 2048, q4);
                const u32x4 high = Cfg::Q_LDS ? q4[kk % 2 * 2] : q_op[Cfg::Q_LDS ? 0 : kk][0], low = Cfg::Q_LDS ? q4[kk % 2 * 2 + 1] : q_op[Cfg::Q_LDS ? 0 : kk][1];
                u32x4 k8[H];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    k8[h] = DT == AIONHIP_Q8_0 ? raw_q8(kw[h][2 * kk % KD], kw[h][(2 * kk + 1) % KD]) : raw_q4(kw[h][kk % KD]);
                    d[h] = mfma16<AIONHIP_F16>(k8[h], high, d[h]);
                }
#pragma unroll
                for (int h = 0; h < H; ++h) d[h] = mfma16<AIONHIP_F16>(k8[h], low, d[h]);
            }
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = h * 4 + j;
                    s[key] = fma_half(d[h][j], ksc[st][key >> 3][(key & 7) >> 1], key & 1, st ? s[key] : cst.zero);
                }
        }
        if (more) {
            load_k(i + NW);
            asm volatile("" ::: "memory");
        }
        if constexpr (REP >= 2) {
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                if constexpr (REP == 4) s[j] += dpp_f<0x124>(s[j]);           // row_ror 4
                s[j] += dpp_f<0x128>(s[j]);                                   // row_ror 8
            }
        }
        if (a.soft_cap > 0.f) {
            stay_branch();
#pragma unroll
            for (int j = 0; j < KG; ++j) s[j] = capped(s[j], row_scale * inv_cap, a.soft_cap);
        }
        // -- which keys this row sees; whole tiles that every row sees need no mask
        bool whole = row0 + TK <= a.T;
        {
            const int first = row0 < wrap ? base + row0 : base - a.ring + row0;
            whole = whole && !(row0 < wrap && row0 + TK > wrap) && first >= full_lo && first <= full_hi - TK;
        }
        if (!whole) {
            stay_branch();                                                    // a key that is not seen: no score, and a scale of zero (what is there may be anything)
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                const int p = row0 + g * KG + j, key = p < wrap ? base + p : base - a.ring + p;
                const bool ok = p < a.T && key >= lo && key < hi;
                s[j] = ok ? s[j] : -INFINITY;
#pragma unroll
                for (int st = 0; st < SETS; ++st) {
                    const unsigned w = vsc[st][j >> 3][(j & 7) >> 1];
                    vsc[st][j >> 3][(j & 7) >> 1] = ok ? w : w & (j & 1 ? 0xFFFFu : 0xFFFF0000u);
                }
            }
        }
        float mx = max3(s[0], s[1], s[1]);
#pragma unroll
        for (int j = 2; j < KG; j += 2) mx = max3(mx, s[j], s[j + 1]);
        mx = groups4_max(mx);
        const float m_new = fmaxf(m_run, mx * to_log2);
        float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        const float ref = m_new - bias;
        float p[16], sum = 0.f;
#pragma unroll
        for (int j = 0; j < KG; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[j], to_log2, -ref));
        m_run = m_new;
        // -- the largest P' of the column, and the shift that keeps it in range
        auto times_scale = [&](int st, int j) __attribute__((always_inline)) { return fma_half(p[j], vsc[st][j >> 3][(j & 7) >> 1], j & 1, cst.zero); };
        float pv[Cfg::PV_TWICE ? 1 : SETS][KG], top = 0.f;
        // An infinite scale has no range to keep, the column's other blocks do: the largest is taken again without it. Where the products are not kept, after the
        // scale has become a NaN, which no maximum takes; by the same code at head size 256 (20 rows over 9000 keys 46 us, 49 with code of its own,
        // for want of registers).
        constexpr int PASSES = Cfg::PV_TWICE && SETS > 1 ? 2 : 1;
#pragma unroll D > 128 ? 1 : 2
        for (int pass = 0; pass < PASSES; ++pass) {
            float before = 0.f;
            top = 0.f;
#pragma unroll
            for (int st = 0; st < SETS; ++st)
#pragma unroll
                for (int j = 0; j < KG; ++j) {
                    const float x = times_scale(st, j);
                    if (j % 2) top = max3(top, before, x);
                    before = x;
                    if constexpr (!Cfg::PV_TWICE) pv[st][j] = x;
                }
            top = fmaxf(largest * alpha, groups4_max(top));
            if (pass + 1 == PASSES || !__any(top == INFINITY)) break;
#pragma unroll
            for (int st = 0; st < SETS; ++st)
#pragma unroll
                for (int j = 0; j < KG; j += 2) {
                    const unsigned w = vsc[st][j >> 3][(j & 7) >> 1];
                    vsc[st][j >> 3][(j & 7) >> 1] = w | ((w & 0x7FFFu) == 0x7C00u ? 0x200u : 0u) | ((w >> 16 & 0x7FFFu) == 0x7C00u ? 0x2000000u : 0u);
                }
        }
        if constexpr (!Cfg::PV_TWICE && SETS > 1) {
            if (__any(top == INFINITY)) {
                stay_branch();
                int most = 1 << 23;                                           // bits of the largest finite one plus 2^23: what is not finite is negative or less
#pragma unroll
                for (int st = 0; st < SETS; ++st)
#pragma unroll
                    for (int j = 0; j < KG; ++j) most = max(most, (int)(__float_as_uint(pv[st][j]) + (1u << 23)));
                top = fmaxf(largest * alpha, groups4_max(__int_as_float(most - (1 << 23))));
            }
        }
        if (__any(top > 32768.f || top < 512.f)) {
            const bool move = top > 0.f && top < INFINITY && (top > 32768.f || top < 512.f);
            const float by = move ? fminf((float)(139 - (int)(__float_as_uint(top) >> 23)), MOST_BIAS - bias) : 0.f;      // to 2^12 .. 2^13
            const float f = __builtin_amdgcn_exp2f(by);
            bias += by;
            top *= f;
            alpha *= f;
#pragma unroll
            for (int j = 0; j < KG; ++j) p[j] *= f;
            if constexpr (!Cfg::PV_TWICE) {
#pragma unroll
                for (int st = 0; st < SETS; ++st)
#pragma unroll
                    for (int j = 0; j < KG; ++j) pv[st][j] *= f;
            }
        }
        if constexpr (Cfg::PV_TWICE) {
#pragma unroll
            for (int j = 0; j < KG; ++j) asm volatile("" : "+v"(p[j]));        // (or the compiler would keep the first)
        }
        largest = top < INFINITY ? top : 0.f;
#pragma unroll
        for (int j = 0; j < KG; ++j) sum += p[j];
        l_run = l_run * alpha + sum;
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt] *= alpha;
        }
        // -- this tile's V is in LDS once only the younger K loads are outstanding (loads complete in order)
        constexpr int YOUNGER = (KD == 2 ? H : H * KD / 4) + SETS * (KG / 8);
        if (more) __builtin_amdgcn_s_waitcnt(vmcnt_imm(YOUNGER));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        constexpr int STEPS = KG / 8, CB = DT == AIONHIP_Q8_0 ? 2 : 1;         // eight keys of a lane to a product; chunks of a block
        static_for<0, SETS>([&](auto st_c) __attribute__((always_inline)) {
            constexpr int st = decltype(st_c)::value;
            u32x4 ph[STEPS], pl[STEPS];
#pragma unroll
            for (int step = 0; step < STEPS; ++step)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k0 = step * 8 + key_slot<DT>(2 * j), k1 = step * 8 + key_slot<DT>(2 * j + 1);
                    const float x = Cfg::PV_TWICE ? times_scale(st, k0) : pv[Cfg::PV_TWICE ? 0 : st][k0], y = Cfg::PV_TWICE ? times_scale(st, k1) : pv[Cfg::PV_TWICE ? 0 : st][k1];
                    const unsigned high = pack_half(x, y);
                    ph[step][j] = high;
                    pl[step][j] = pack_half(fma_half(cst.minus, high, 0, x), fma_half(cst.minus, high, 1, y));
                }
            constexpr int READS = REP * CB * STEPS, N = READS < 8 ? READS : 8;
            static_for<0, READS / N>([&](auto part_c) __attribute__((always_inline)) {
                constexpr int c0 = st * REP * CB + decltype(part_c)::value * N / STEPS;
                unsigned at[N];
                u32x2 v[N];
#pragma unroll
                for (int c = 0; c < N / STEPS; ++c)
#pragma unroll
                    for (int step = 0; step < STEPS; ++step)                  // (eight rows on, a row's f is its f with the upper bit the other way)
                        at[c * STEPS + step] = (v_addr ^ (unsigned)((c0 + c) << 4) ^ (unsigned)(step ? CH / 2 << 4 : 0)) + (unsigned)(step * 8 * RB);
                read_transposed<N>(at, v);
#pragma unroll
                for (int c = 0; c < N / STEPS; ++c)
#pragma unroll
                    for (int step = 0; step < STEPS; ++step) {
                        const u32x2 w = v[c * STEPS + step];
                        if constexpr (DT == AIONHIP_Q8_0) {
                            f32x4 &o = acc[c0 + c];
                            const u32x4 x = halves_q8(cst, w.x, w.y);
                            o = mfma16<AIONHIP_F16>(x, ph[step], o);
                            o = mfma16<AIONHIP_F16>(x, pl[step], o);
                        } else {                                              // the even columns of the block, and the odd ones
                            const u32x4 x = halves_q4(cst, w.x), y = halves_q4(cst, w.y);
                            f32x4 &o = acc[(c0 + c) * 2], &o2 = acc[(c0 + c) * 2 + 1];
                            const u32x4 even{x.x, x.z, y.x, y.z}, odd{x.y, x.w, y.y, y.w};
                            o = mfma16<AIONHIP_F16>(even, ph[step], o);
                            o = mfma16<AIONHIP_F16>(even, pl[step], o);
                            o2 = mfma16<AIONHIP_F16>(odd, ph[step], o2);
                            o2 = mfma16<AIONHIP_F16>(odd, pl[step], o2);
                        }
                    }
            });
        });
        if (more) {
            asm volatile("" ::: "memory");
            load_v(i + NW);
        }
    };
    if (t < t_end) {
        for (; t + NW < t_end; t += NW) tile(t, std::true_type{});
        tile(t, std::false_type{});
    }
    l_run = groups4_sum(l_run);

    // ---- the wavefronts meet
    __syncthreads();
    constexpr int RS = D + 4;                                                 // rows apart by 16 bytes more: fewer of a store's lanes on one bank
    constexpr int WS = ROWS * RS + 32;
    float *mg = (float *)lds;
    {
        float *w = mg + wave * WS;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
            if (kk % REP == sub) {
                const f32x4 x = acc[2 * kk], y = acc[2 * kk + 1];
                float *o = w + n % ROWS * RS + kk * 32;
                if constexpr (DT == AIONHIP_Q8_0) {
                    *(f32x4 *)(o + g * 4) = x;
                    *(f32x4 *)(o + 16 + g * 4) = y;
                } else {
                    *(f32x4 *)(o + g * 8) = f32x4{x.x, y.x, x.y, y.y};
                    *(f32x4 *)(o + g * 8 + 4) = f32x4{x.z, y.z, x.w, y.w};
                }
            }
        if (g == 0) {
            w[ROWS * RS + 2 * n] = m_run > REF_NONE ? m_run - bias : REF_NONE;
            w[ROWS * RS + 2 * n + 1] = l_run;
        }
    }
    __syncthreads();
    const size_t meeting = (size_t)unit * sp.row_tiles + rt;
    [[maybe_unused]] float *const parts = sp.parts + meeting * sp.nseg * FLOATS;
    [[maybe_unused]] constexpr int DEVICE_SCOPE = 16;                          // the sc1 bit of a buffer access: where the XCDs' caches agree
#if defined(__HIP_DEVICE_COMPILE__)
    [[maybe_unused]] const __amdgpu_buffer_rsrc_t parts_rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)parts, 0, (unsigned)(sp.nseg * FLOATS * 4), 0x00027000);
#endif
    auto store_out = [&](int row, int col, f32x4 v) {
        const int rr = rt * ROWS + row, l2 = a.L == 1 ? 0 : rr / a.groups, g2 = rr - l2 * a.groups;
        __builtin_memcpy(a.out + (((size_t)b * a.L + l2) * a.Hq + hk * a.groups + g2) * D + col, &v, 16);
    };
    auto meet = [&](int c, float (&f)[NW], float &ref, float &l) {
        float x[NW];
        ref = REF_NONE;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) ref = fmaxf(ref, x[w] = mg[w * WS + ROWS * RS + 2 * c]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            f[w] = __builtin_amdgcn_exp2f(x[w] - ref);
            l += mg[w * WS + ROWS * RS + 2 * c + 1] * f[w];
        }
    };
    for (int e = threadIdx.x; e < rows * (D / 4); e += NW * 64) {
        const int row = e / (D / 4), col = e % (D / 4) * 4, c = (col / 32) % REP * ROWS + row;
        float f[NW], ref, l;
        meet(c, f, ref, l);
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) o += *(const f32x4 *)(mg + w * WS + row * RS + col) * f[w];
        if (sp.nseg == 1) store_out(row, col, o * (l != 0.f ? 1.f / l : 0.f));
#if defined(__HIP_DEVICE_COMPILE__)
        else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), parts_rsrc, (seg * FLOATS + row * D + col) * 4, 0, DEVICE_SCOPE);
#endif
    }
    if (sp.nseg == 1) return;
    if (threadIdx.x < 16) {
        float f[NW], ref, l;
        meet((int)threadIdx.x, f, ref, l);
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(ref), __float_as_uint(l)}, parts_rsrc, (seg * FLOATS + ROWS * D + 2 * (int)threadIdx.x) * 4, 0, DEVICE_SCOPE);
#endif
    }
    if (!sp.tickets) return;
    // The workgroup that ends last adds the segments up: each waits until its stores have been acknowledged, then draws a ticket; nobody waits for anybody.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int *drawn = (int *)lds;
    if (threadIdx.x == 0) *drawn = (int)__hip_atomic_fetch_add(sp.tickets + meeting * MEET_TICKET_WORDS, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int mine = *drawn;
    __syncthreads();
    if (mine != sp.nseg - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(sp.tickets + meeting * MEET_TICKET_WORDS, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int elements = rows * (D / 4);
    merge_parts<D, REP>(
        sp.nseg, 0, elements, max(1, min(NW * 64 / elements, (sp.nseg + RUN - 1) / RUN)), (f32x4 *)lds, (float2 *)(lds + NW * 64 * 16),
        [&](auto count_c, size_t at) __attribute__((always_inline)) {
            if constexpr (decltype(count_c)::value == 2) {
                u32x2 x = {};
#if defined(__HIP_DEVICE_COMPILE__)
                x = __builtin_amdgcn_raw_buffer_load_b64(parts_rsrc, (int)at * 4, 0, DEVICE_SCOPE);
#endif
                return x;
            } else {
                u32x4 x = {};
#if defined(__HIP_DEVICE_COMPILE__)
                x = __builtin_amdgcn_raw_buffer_load_b128(parts_rsrc, (int)at * 4, 0, DEVICE_SCOPE);
#endif
                return x;
            }
        },
        store_out);
}

// The merge as a launch, for row tiles whose parts are too much for one workgroup or come from quant_prompt_kernel: (row tile and share of its elements, unit)
template <int D, int REP>
__global__ __launch_bounds__(NW * 64) void quant_merge_kernel(QuantArgs a, Split sp, int groups, int shares) {
    __shared__ f32x4 meet_o[NW * 64];
    __shared__ float2 meet_s[NW * 64];
    constexpr int ROWS = Part<D, REP>::ROWS, FLOATS = Part<D, REP>::FLOATS;
    const int rt = blockIdx.x / shares, share = blockIdx.x % shares, unit = blockIdx.y, b = unit / a.Hkv, hk = unit % a.Hkv, per = NW * 64 / groups;
    const int elements = min(ROWS, a.L * a.groups - rt * ROWS) * (D / 4);
    const float *parts = sp.parts + ((size_t)unit * sp.row_tiles + rt) * sp.nseg * FLOATS;
    merge_parts<D, REP>(
        sp.nseg, share * per, min((share + 1) * per, elements), groups, meet_o, meet_s,
        [&](auto count_c, size_t at) __attribute__((always_inline)) {
            if constexpr (decltype(count_c)::value == 2) return *(const u32x2 *)(parts + at);
            else return *(const u32x4 *)(parts + at);
        },
        [&](int row, int col, f32x4 v) {
            const int rr = rt * ROWS + row, l2 = rr / a.groups, g2 = rr - l2 * a.groups;
            __builtin_memcpy(a.out + (((size_t)b * a.L + l2) * a.Hq + hk * a.groups + g2) * D + col, &v, 16);
        });
}
template <int D, int REP>
void launch_merge(aionhip_ctx *ctx, const QuantArgs &a, const Split &sp) {
    const int groups = (sp.nseg + RUN - 1) / RUN, per = NW * 64 / groups, shares = (Part<D, REP>::ROWS * (D / 4) + per - 1) / per;
    ProfScope scope(ctx, "attn_quant_merge");
    launch_k(ctx, quant_merge_kernel<D, REP>, dim3((unsigned)(sp.row_tiles * shares), (unsigned)(a.B * a.Hkv)), dim3(NW * 64), 0, a, sp, groups, shares);
}

template <int DT, int D, int REP>
int launch_decode(aionhip_ctx *ctx, const QuantArgs &a) {
    using Cfg = DecodeCfg<DT, D, REP>;
    constexpr int ROWS = Cfg::ROWS, LDS = Cfg::LDS_BYTES;
    const int cus = ctx->cu_count > 0 ? ctx->cu_count : 256;
    Split sp{};
    const long rows = (long)a.L * a.groups, units = (long)a.B * a.Hkv;
    sp.row_tiles = (int)((rows + ROWS - 1) / ROWS);
    const long tiles = units * sp.row_tiles;
    long keys = a.T;
    if (a.win_chunk == 0 && a.win_right < (unsigned)a.T && a.win_left < (unsigned)a.T) keys = min(keys, (long)a.win_left + (long)a.win_right + a.L + Cfg::TK);
    const long key_tiles = (keys + Cfg::TK - 1) / Cfg::TK;
    // As many as two workgroups to a CU take, each wavefront with a tile at least. us a step with one / two / four to a CU: 32 sequences of 16384 keys, 8 x 128 in 4
    // bits, 167 / 139 / 144; 4 x 5 queries over 3001 keys of 32 x 128 20 / 19 / 28; 16 over 9692 of 2 x 256 in 8 bits 34 / 34 / 53; 131072 keys of 8 x 128 50 / 53 / 48.
    // Up to two tiles to a wavefront are not worth a meeting: one token over 256 keys of one head of 256 10.4 in two segments, 8.6 in one; 512 keys 10.3 in four, 12.1.
    sp.nseg = key_tiles <= 2 * NW ? 1 : (int)max(1L, min(min((long)MAX_SEG, 2 * cus / tiles), (key_tiles + NW - 1) / NW));
    if (sp.nseg > 1) {
        if (const int rc = ensure_scratch2(ctx, (size_t)tiles * sp.nseg * Part<D, REP>::FLOATS * sizeof(float))) return rc;
        sp.parts = (float *)ctx->scratch2;
        if (tiles <= cus && sp.nseg <= 64) {
            if (const int rc = ensure_tickets(ctx, (size_t)tiles * MEET_TICKET_WORDS * sizeof(unsigned))) return rc;
            sp.tickets = (unsigned *)ctx->tickets;
        }
    }
    if ((long)sp.row_tiles * sp.nseg > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: dimension too large");
    static std::atomic<uint64_t> attr{0};
    if (const int rc = allow_lds(ctx, attr, (const void *)quant_decode_kernel<DT, D, REP>, LDS)) return rc;
    {
        ProfScope scope(ctx, "attn_quant_decode");
        launch_k(ctx, quant_decode_kernel<DT, D, REP>, dim3((unsigned)(sp.row_tiles * sp.nseg), (unsigned)a.Hkv, (unsigned)a.B), dim3(NW * 64), LDS, a, sp);
    }
    if (sp.nseg > 1 && !sp.tickets) launch_merge<D, REP>(ctx, a, sp);
    LAUNCH_CHECK(ctx, "attn_quant_decode");
    return AIONHIP_OK;
}
template <int DT, int D>
int launch_decode_rows(aionhip_ctx *ctx, const QuantArgs &a) {
    const long rows = (long)a.L * a.groups;
    if constexpr (D >= 128)
        if (rows <= 4) return launch_decode<DT, D, 4>(ctx, a);
    if (rows <= 8) return launch_decode<DT, D, 2>(ctx, a);
    return launch_decode<DT, D, 1>(ctx, a);
}

// --------------------------------------------------------------------------------------------------------------------- many query rows
// A workgroup has ROWS query rows, 32 to a wavefront (16 at head size 256), and walks its keys a tile at a time. What bounds it is the arithmetic, so the
// conversions are made once for all of its rows: eight wavefronts turn a tile's codes into operands in LDS around their products of the tile before it
// (two stages, one barrier a tile; four convert first and four last, of which each SIMD has one: 377 us against 379 and 398 where all do so first or last). The
// tile after that is asked for between the softmax and P V, when the scores' registers are free.
//   K: the codes as f16, exact, [block][lane group][row of a sub-tile] of 16 bytes: an operand is one read, and its scale goes onto the product (a block long).
//     The query row is the sum of two f16, as in quant_decode_kernel.
//   V: here the scale can go onto the value, which many rows share: code * scale (19 bits) times a power of two as the sum of two f16, exact down to 2^-18 of the
//     largest that the workgroup's rows see in that block of columns, and good to 2^-40 of it (two bf16, which need no power, were off by 2^-17: 3e-6 of
//     an output where this is 3e-7). The largest is found first, from the scales alone, 1/32 to 1/16 of V. P is the sum of two f16 too, and of the four products
//     the smallest, 2^-22, is left out. Eight keys of a byte come by a transposing read; the exchange is a wavefront's own.
// Measured: 4096 tokens, 32 heads on 8 of 128, q8_0: 333 us, 413 TFLOP/s (of the products as formulas write them; the matrix cores make five for two); 2 x 500 tokens
// at 9000 keys, 8 heads on 2 of 256, q4_0: 191 us and 8.5 for the merge. (After 0.3 s of passes. The forms compared here had twenty passes each, with the clock
// still rising: 377 us as it is.) It is bound by issue: a wavefront's tile is 160 matrix instructions and 590 others (128 scales onto products, 180
// conversions, the softmax 280). Asking for a tile a whole round ahead cost the products their registers (428 us before), four wavefronts' operands read one product
// ahead and higher wave priority around the products gave the rest.
// A scale that is not finite would reach rows that do not see its key (0 * NaN), as would one that none of the rows sees and that the power of two takes past f16:
// such a value is taken as zero, and the rows that see one that is not finite get their NaN by hand.
template <int DT, int D>
struct PromptCfg {
    static constexpr int WAVES = 8, TK = D > 128 ? 32 : 64, CT = D > 128 ? 1 : 2, ROWS = WAVES * 16 * CT;
    static constexpr int RB = DT == AIONHIP_Q8_0 ? D : D / 2;
    static constexpr int K_BYTES = TK * D * 2, V_BYTES = TK * D * 2, S_BYTES = D / 32 * TK * 2;       // V_BYTES: of either part
    static constexpr int STAGE = K_BYTES + 2 * V_BYTES + S_BYTES;
    static constexpr int LDS_BYTES = 2 * STAGE + WAVES * 512 + 64;
};
typedef __attribute__((ext_vector_type(2))) int v2i;
typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
__device__ __forceinline__ unsigned max_u16x2(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

template <int DT, int D>
__global__ __launch_bounds__(512, 2) void quant_prompt_kernel(QuantArgs a, Split sp) {
    using Cfg = PromptCfg<DT, D>;
    constexpr int WAVES = Cfg::WAVES, TK = Cfg::TK, CT = Cfg::CT, RB = Cfg::RB, CH = RB / 16, KK = D / 32, MT = D / 16;
    constexpr int H = TK / 16, KG = TK / 4, STEPS = KG / 8;                  // sub-tiles; keys of a lane; products they make
    constexpr int K_ALL = TK * RB / 512, KI = (K_ALL + WAVES - 1) / WAVES;   // loads of a tile, 512 bytes each: of K, and of V
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    // longest first: the last rows of all units, then those before them
    const int units = a.B * a.Hkv, group_tiles = (sp.row_tiles * 16 + Cfg::ROWS - 1) / Cfg::ROWS;
    const int per_place = units * sp.nseg, place = group_tiles - 1 - (int)(blockIdx.x / per_place), rest = (int)(blockIdx.x % per_place);
    const int unit = rest / sp.nseg, seg = rest - unit * sp.nseg, b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const int rows_total = a.L * a.groups, row_first = place * Cfg::ROWS + wave * 16 * CT;

    // ---- query rows (past the last one: that one again)
    int lo[CT], hi[CT];
    int uni_lo = INT_MAX, uni_hi = 0, full_lo = 0, full_hi = INT_MAX;        // of the wavefront's rows
    size_t qbase[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int r = min(row_first + ct * 16 + n, rows_total - 1), li = r / a.groups;
        qbase[ct] = (((size_t)b * a.L + li) * a.Hq + hk * a.groups + (r - li * a.groups)) * D;
        visible(a, b, li, lo[ct], hi[ct]);
        if (hi[ct] <= lo[ct]) lo[ct] = hi[ct] = 0;
        uni_lo = min(uni_lo, rows16_min_i(hi[ct] > lo[ct] ? lo[ct] : INT_MAX));
        uni_hi = max(uni_hi, rows16_max_i(hi[ct]));
        full_lo = max(full_lo, rows16_max_i(lo[ct]));
        full_hi = min(full_hi, rows16_min_i(hi[ct]));
    }
    // ---- the workgroup's keys
    int *meet_lds = (int *)(lds + 2 * Cfg::STAGE + WAVES * 512);
    if (threadIdx.x == 0) {
        meet_lds[0] = INT_MAX;
        meet_lds[1] = 0;
        meet_lds[2] = meet_lds[3] = 0;                                       // one more than the last tile with a value whose scale is not finite, by stages
        for (int kk = 0; kk < KK; ++kk) meet_lds[4 + kk] = 0;                // the blocks' largest scales
    }
    __syncthreads();
    if (lane == 0) {
        atomicMin(&meet_lds[0], uni_lo);
        atomicMax(&meet_lds[1], uni_hi);
    }
    __syncthreads();
    const int wg_lo = __builtin_amdgcn_readfirstlane(meet_lds[0]), wg_hi = __builtin_amdgcn_readfirstlane(meet_lds[1]);
    const int kv_end = clip_kv_end(a.ring, a.T, a.kv_lengths ? a.kv_lengths[b] : a.T);
    const int wrap = a.ring ? kv_end % a.ring : INT_MAX, base = a.ring ? kv_end - wrap : 0;      // (rings by their rows: see quant_decode_kernel)
    int first_tile = 0, count = 0;
    const int all_tiles = (a.T + TK - 1) / TK;
    if (wg_hi > wg_lo) {
        const int p0 = phys_key(a.ring, wg_lo);
        first_tile = p0 / TK;
        const long span = (long)(p0 % TK) + (wg_hi - wg_lo);
        count = (int)min((long)all_tiles, (span + TK - 1) / TK + (a.ring && (long)p0 + (wg_hi - wg_lo) > a.ring ? 1 : 0));
    }
    const int per = (count + sp.nseg - 1) / sp.nseg, t0 = seg * per, t_end = min((seg + 1) * per, count);
    auto row0_of = [&](int i) { const int x = first_tile + i; return (x >= all_tiles ? x - all_tiles : x) * TK; };

    const size_t unit_rows = (size_t)unit * a.Tp;
    const unsigned char *kc = a.k.codes + unit_rows * RB, *vc = a.v.codes + unit_rows * RB;
    const __half *ks = a.k.scales + unit_rows * KK, *vs = a.v.scales + unit_rows * KK;

    const Constants cst;
    // ---- a tile on its way: 512 bytes to an instruction, K in order, V as eight keys x 16 bytes to sixteen lanes
    u32x2 kraw[KI], vraw[KI];
    u32x4 vscale[KI], kscale{};
    static_assert(32 % CH == 0, "a load's chunk is its lane's");
    auto seen = [&](int p) __attribute__((always_inline)) {                  // by a row of the workgroup
        const int key = p < wrap ? base + p : base - a.ring + p;
        return p < a.T && key >= wg_lo && key < wg_hi;
    };
    unsigned limit = 0;                                                      // of the scales of the lane's block of V, and what brings it below 2^8
    float grow = 1.f;
    const int octet0 = (wave * 4 + g) / CH, chunk = (wave * 4 + g) % CH;     // of V, the lane's; each further load 32 / CH octets on
    auto v_octet = [&](int j) { return j * (32 / CH) + octet0; };
    const int k_lane = wave * 512 + lane * 8, v_lane = (octet0 * 8 + (n >> 1)) * RB + chunk * 16 + (n & 1) * 8;
    const __half *vs_lane = vs + (size_t)(DT == AIONHIP_Q8_0 ? chunk / 2 : chunk) * a.Tp + octet0 * 8;
    const __half *ks_lane = ks + (size_t)(threadIdx.x / (TK / 8)) * a.Tp + (threadIdx.x % (TK / 8)) * 8;
    auto request = [&](int i) __attribute__((always_inline)) {
        const int row0 = row0_of(i);
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *)(kc + (size_t)row0 * RB), 0, TK * RB, 0x00027000);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *)(vc + (size_t)row0 * RB), 0, TK * RB, 0x00027000);
#pragma unroll
        for (int j = 0; j < KI; ++j)
            if (K_ALL % WAVES == 0 || j * WAVES + wave < K_ALL) {
                kraw[j] = __builtin_amdgcn_raw_buffer_load_b64(rk, k_lane, j * WAVES * 512, 0);
                vraw[j] = __builtin_amdgcn_raw_buffer_load_b64(rv, v_lane, j * WAVES * 512, 0);
                vscale[j] = *(const u32x4 *)(vs_lane + row0 + j * (256 / CH));
            }
        if (threadIdx.x < KK * TK / 8) kscale = *(const u32x4 *)(ks_lane + row0);
    };
    auto convert = [&](int i, int stage) __attribute__((always_inline)) {
        unsigned char *k_op = lds + stage * Cfg::STAGE, *v_op = k_op + Cfg::K_BYTES, *s_op = v_op + 2 * Cfg::V_BYTES, *swap = lds + 2 * Cfg::STAGE + wave * 512;
        if (threadIdx.x < KK * TK / 8) *(u32x4 *)(s_op + threadIdx.x * 16) = kscale;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < KI; ++j)
            if (K_ALL % WAVES == 0 || j * WAVES + wave < K_ALL) {
                const int off = (j * WAVES + wave) * 512 + lane * 8, key = off / RB, piece = off % RB / 8;
                const int pos = key % KG / 4 * 16 + key / KG * 4 + key % 4;
                if constexpr (DT == AIONHIP_Q8_0) {
                    *(u32x4 *)(k_op + (piece * TK + pos) * 16) = halves_q8(cst, kraw[j].x, kraw[j].y);
                } else {
                    *(u32x4 *)(k_op + (piece * 2 * TK + pos) * 16) = halves_q4(cst, kraw[j].x);
                    *(u32x4 *)(k_op + ((piece * 2 + 1) * TK + pos) * 16) = halves_q4(cst, kraw[j].y);
                }
                *(u32x2 *)(swap + lane * 8) = vraw[j];
                v2i w{};
#if defined(__HIP_DEVICE_COMPILE__)   // the builtin exists in the device pass only
                w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(lds_void *)(swap + lane * 8));
#endif
                u32x4 sc = vscale[j];
                const unsigned most = max_u16x2(max_u16x2(sc.x & 0x7FFF7FFFu, sc.y & 0x7FFF7FFFu), max_u16x2(sc.z & 0x7FFF7FFFu, sc.w & 0x7FFF7FFFu));
                if (__any(max(most >> 16, most & 0xFFFFu) > limit)) {                  // not finite, or of no key that the workgroup's rows see
                    stay_branch();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const unsigned half = sc[k >> 1] >> (16 * (k & 1)) & 0x7FFFu;
                        const int p = row0_of(i) + v_octet(j) * 8 + k;
                        odd |= half >= 0x7C00u && seen(p);
                        if (half > limit) sc[k >> 1] &= k & 1 ? 0xFFFFu : 0xFFFF0000u;
                    }
                }
                float by[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) by[k] = fma_half(grow, sc[k >> 1], k & 1, cst.zero);
                // x: pairs of codes of the keys ka, kb; stored at column `col` of the octet
                auto store = [&](const u32x4 &x, int col) __attribute__((always_inline)) {
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[key_slot<DT>(k)] = fma_half(by[key_slot<DT>(k)], x[k >> 1], k & 1, cst.zero);
                    u32x4 high, low;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        high[k] = pack_half(v[2 * k], v[2 * k + 1]);
                        low[k] = pack_half(fma_half(cst.minus, high[k], 0, v[2 * k]), fma_half(cst.minus, high[k], 1, v[2 * k + 1]));
                    }
                    unsigned char *o = v_op + (v_octet(j) * D + col) * 16;
                    *(u32x4 *)o = high;
                    *(u32x4 *)(o + Cfg::V_BYTES) = low;
                };
                if constexpr (DT == AIONHIP_Q8_0) {
                    store(halves_q8(cst, (unsigned)w.x, (unsigned)w.y), chunk * 16 + n);
                } else {
                    const u32x4 x = halves_q4(cst, (unsigned)w.x), y = halves_q4(cst, (unsigned)w.y);
                    store(u32x4{x.x, x.z, y.x, y.z}, chunk * 32 + n);
                    store(u32x4{x.y, x.w, y.y, y.w}, chunk * 32 + 16 + n);
                }
            }
        if (__any(odd) && lane == 0) meet_lds[2 + stage] = i + 1;
    };

    if (t0 < t_end) request(t0);
    // ---- the largest scale of each block of V that a row of the workgroup sees, in the tiles it is about to walk
    constexpr int LOADS = KK * TK / 8;                                       // of a tile's scales
    {
        const int slot = threadIdx.x % LOADS, kk = slot / (TK / 8), at = slot % (TK / 8) * 8;
        unsigned most = 0;
#pragma unroll 4
        for (int i = t0 + (int)threadIdx.x / LOADS; i < t_end; i += WAVES * 64 / LOADS) {
            const int row = row0_of(i) + at;
            const u32x4 sc = *(const u32x4 *)(vs + (size_t)kk * a.Tp + row);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const unsigned half = sc[k >> 1] >> (16 * (k & 1)) & 0x7FFFu;
                most = max(most, half < 0x7C00u && seen(row + k) ? half : 0u);
            }
        }
        atomicMax(&meet_lds[4 + kk], (int)most);
        __syncthreads();
        limit = (unsigned)meet_lds[4 + (DT == AIONHIP_Q8_0 ? chunk / 2 : chunk)];
        grow = __uint_as_float((149u - max(limit >> 10, 1u)) << 23);
    }
    // ---- Q^T, two parts of eight elements of each block
    const float inv_cap = a.soft_cap > 0.f ? 1.f / a.soft_cap : 0.f;
    u32x4 q_op[CT][KK][2];
    float row_scale[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        float x[KK][8], amax = 0.f;
        load_query<KK>(a, qbase[ct] + g * 8, x);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[kk][j]));
        const Power2 by(groups4_max(amax));
        row_scale[ct] = fabsf(a.scale) * by.grow;
        const float sign = a.scale < 0.f ? -by.shrink : by.shrink;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) (void)split_query<DT>(x[kk], sign, q_op[ct][kk]);
    }

    f32x4 acc[CT][MT];
    float m_ref[CT], l_run[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        m_ref[ct] = REF_NONE;
        l_run[ct] = 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[ct][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const bool early = wave < WAVES / 2;
    if (t0 < t_end) {
        convert(t0, 0);
        if (early && t0 + 1 < t_end) request(t0 + 1);
    }
    __syncthreads();
    for (int i = t0; i < t_end; ++i) {
        const int stage = (i - t0) & 1, row0 = row0_of(i);
        if (early && i + 1 < t_end) convert(i + 1, stage ^ 1);
        __builtin_amdgcn_sched_barrier(0);
        const unsigned char *k_op = lds + stage * Cfg::STAGE, *v_op = k_op + Cfg::K_BYTES, *s_op = v_op + 2 * Cfg::V_BYTES;
        // keys of the tile: `first` the first row's, one after the other but where a ring begins again
        const int first = row0 < wrap ? base + row0 : base - a.ring + row0;
        auto ask = [&]() __attribute__((always_inline)) {
            const int ahead = i + (early ? 2 : 1);
            if (ahead < t_end) request(ahead);
        };
        const bool plain = row0 + TK <= a.T && !(row0 < wrap && row0 + TK > wrap);
        if (!plain || (first < uni_hi && uni_lo - TK < first)) {
            float s[CT][KG];
            // Products of a sub-tile and a block at a time: the scales meet one's while the matrix cores work on the next's, whose operands have been on their way for
            // three. (Two sub-tiles share their scales' load.)
            constexpr int UNITS = H * KK;
            u32x4 k_at[4], sc_at[2];
            f32x4 d[2][CT];
            auto k_load = [&](int x) __attribute__((always_inline)) {
                k_at[x & 3] = *(const u32x4 *)(k_op + ((x / 2 % KK * 4 + g) * TK + (x / (2 * KK) * 2 + (x & 1)) * 16 + n) * 16);
            };
            auto s_load = [&](int x) __attribute__((always_inline)) {
                if ((x & 1) == 0) sc_at[x / 2 & 1] = *(const u32x4 *)(s_op + (x / 2 % KK * TK + g * KG + x / (2 * KK) * 8) * 2);
            };
            auto scaled = [&](int x) __attribute__((always_inline)) {
                const int kk = x / 2 % KK, at = x / (2 * KK) * 8 + (x & 1) * 4;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[ct][at + j] = fma_half(d[x & 1][ct][j], sc_at[x / 2 & 1][(x & 1) * 2 + (j >> 1)], j & 1, kk ? s[ct][at + j] : cst.zero);
            };
            __builtin_amdgcn_s_setprio(1);
            k_load(0);
            k_load(1);
            k_load(2);
            s_load(0);
#pragma unroll
            for (int x = 0; x <= UNITS; ++x) {
                if (x < UNITS) {
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) d[x & 1][ct] = mfma16<AIONHIP_F16>(k_at[x & 3], q_op[ct][x / 2 % KK][part], part ? d[x & 1][ct] : f32x4{0.f, 0.f, 0.f, 0.f});
                }
                if (x > 0) scaled(x - 1);
                if (x + 2 < UNITS) s_load(x + 2);
                if (x + 3 < UNITS) k_load(x + 3);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)                                   // (or the products of the second column group would wait, unscaled, behind the first's softmax)
#pragma unroll
                for (int j = 0; j < KG; ++j) asm volatile("" : "+v"(s[ct][j]));
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            const bool whole = plain && first >= full_lo && first <= full_hi - TK;
            u32x4 ph[CT][STEPS], pl[CT][STEPS];
            auto sees = [&](int ct, int p) __attribute__((always_inline)) {
                const int key = p < wrap ? base + p : base - a.ring + p;
                return p < a.T && key >= lo[ct] && key < hi[ct];
            };
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float to_log2 = fmaxf(row_scale[ct] * LOG2E, 1e-30f);
                if (a.soft_cap > 0.f) {
                    stay_branch();
                    to_log2 = 1.f;
#pragma unroll
                    for (int j = 0; j < KG; ++j) s[ct][j] = capped(s[ct][j], row_scale[ct] * inv_cap, a.soft_cap);
                }
                if (!whole) {
                    int p0 = row0 + g * KG;
                    asm volatile("" : "+v"(p0));                              // (made anew for each column group, not kept)
#pragma unroll
                    for (int j = 0; j < KG; ++j) s[ct][j] = sees(ct, p0 + j) ? s[ct][j] : -INFINITY;
                }
                float mx = max3(s[ct][0], s[ct][1], s[ct][1]);
#pragma unroll
                for (int j = 2; j < KG; j += 2) mx = max3(mx, s[ct][j], s[ct][j + 1]);
                mx = groups4_max(mx) * to_log2;
                // the reference is the maximum less 7, and follows it only where that has grown by another 8: exponentials of up to 2^15, whose two f16 end 2^-32 below
                // the largest
                if (__any(mx > m_ref[ct] + 15.f)) {
                    stay_branch();
                    const float m_new = mx > m_ref[ct] + 15.f ? mx - 7.f : m_ref[ct];
                    const float alpha = __builtin_amdgcn_exp2f(m_ref[ct] - m_new);
                    m_ref[ct] = m_new;
                    l_run[ct] *= alpha;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) acc[ct][mt] *= alpha;
                }
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < KG; ++j) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[ct][j], to_log2, -m_ref[ct]));
                    s[ct][j] = p;
                    sum += p;
                }
                l_run[ct] += sum;
#pragma unroll
                for (int step = 0; step < STEPS; ++step)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x = s[ct][step * 8 + 2 * k], y = s[ct][step * 8 + 2 * k + 1];
                        const unsigned high = pack_half(x, y);
                        ph[ct][step][k] = high;
                        pl[ct][step][k] = pack_half(fma_half(cst.minus, high, 0, x), fma_half(cst.minus, high, 1, y));
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            ask();
            u32x4 v_at[2][2];                                                 // the operands of a product and of the next
            auto v_load = [&](int x) __attribute__((always_inline)) {
                const unsigned char *o = v_op + ((g * STEPS + x % STEPS) * D + x / STEPS * 16 + n) * 16;
                v_at[x & 1][0] = *(const u32x4 *)o;
                v_at[x & 1][1] = *(const u32x4 *)(o + Cfg::V_BYTES);
            };
            __builtin_amdgcn_s_setprio(1);
            v_load(0);
#pragma unroll
            for (int x = 0; x < MT * STEPS; ++x) {
                const int mt = x / STEPS, step = x % STEPS;
                if (x + 1 < MT * STEPS) v_load(x + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) acc[ct][mt] = mfma16<AIONHIP_F16>(v_at[x & 1][0], ph[ct][step], acc[ct][mt]);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) acc[ct][mt] = mfma16<AIONHIP_F16>(v_at[x & 1][0], pl[ct][step], acc[ct][mt]);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) acc[ct][mt] = mfma16<AIONHIP_F16>(v_at[x & 1][1], ph[ct][step], acc[ct][mt]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            if (meet_lds[2 + stage] == i + 1) {
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        float gone = 0.f;
#pragma unroll 1
                        for (int j = 0; j < KG; ++j) {
                            const float v = __half2float(vs[(size_t)kk * a.Tp + row0 + g * KG + j]);
                            if (sees(ct, row0 + g * KG + j) && !(fabsf(v) < INFINITY)) gone = 1.f;
                        }
                        if (groups4_max(gone) > 0.f) acc[ct][2 * kk] = acc[ct][2 * kk + 1] = f32x4{NAN, NAN, NAN, NAN};
                    }
            }
        } else {
            ask();
        }
        if (!early && i + 1 < t_end) convert(i + 1, stage ^ 1);
        __syncthreads();
    }

#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const float l = groups4_sum(l_run[ct]);
        const int r = row_first + ct * 16 + n;
        if (r >= rows_total) continue;
        float *o;
        float inv = 1.f;
        if (sp.nseg == 1) {
            const int li = r / a.groups;
            o = a.out + (((size_t)b * a.L + li) * a.Hq + hk * a.groups + (r - li * a.groups)) * D;
            inv = l != 0.f ? 1.f / l : 0.f;
        } else {
            float *part = sp.parts + (((size_t)unit * sp.row_tiles + r / 16) * sp.nseg + seg) * Part<D, 1>::FLOATS;
            o = part + n * D;
            if (g == 0) {
                part[16 * D + 2 * n] = m_ref[ct];
                part[16 * D + 2 * n + 1] = l;
            }
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const float back = inv * __uint_as_float((105u + max((unsigned)meet_lds[4 + kk] >> 10, 1u)) << 23);
            const f32x4 x = acc[ct][2 * kk] * back, y = acc[ct][2 * kk + 1] * back;
            f32x4 first4, second4;
            int at, next;
            if constexpr (DT == AIONHIP_Q8_0) {
                first4 = x, second4 = y, at = kk * 32 + g * 4, next = 16;
            } else {
                first4 = f32x4{x.x, y.x, x.y, y.y}, second4 = f32x4{x.z, y.z, x.w, y.w}, at = kk * 32 + g * 8, next = 4;
            }
            __builtin_memcpy(o + at, &first4, 16);
            __builtin_memcpy(o + at + next, &second4, 16);
        }
    }
}

template <int DT, int D>
int launch_prompt(aionhip_ctx *ctx, const QuantArgs &a) {
    using Cfg = PromptCfg<DT, D>;
    const int cus = ctx->cu_count > 0 ? ctx->cu_count : 256;
    const long rows = (long)a.L * a.groups, units = (long)a.B * a.Hkv, wgs = units * ((rows + Cfg::ROWS - 1) / Cfg::ROWS);
    Split sp{};
    sp.row_tiles = (int)((rows + 15) / 16);
    long keys = a.T;
    if (a.win_chunk == 0 && a.win_right < (unsigned)a.T && a.win_left < (unsigned)a.T) keys = min(keys, (long)a.win_left + (long)a.win_right + a.L + Cfg::TK);
    const long key_tiles = (keys + Cfg::TK - 1) / Cfg::TK;
    // One workgroup per CU. Two where the rows see half the keys on average (a prompt on its own), so that short workgroups follow long ones - but for prompts whose
    // parts take longer to merge: with 256 tiles of rows 4096 keys at D = 64 go from 187 to 142 us, twice 1024 at D = 128 would go from 89 to 99.
    // Never more than the scratch memory that a recording finds there (aionhip_program_begin), so that a step has the same segments recorded or not. That keeps 2048
    // keys at D = 128 in one segment, 158 us, where two took 151.
    const size_t part_bytes = (size_t)units * sp.row_tiles * Part<D, 1>::FLOATS * sizeof(float);
    const long want = 2 * (long)a.L > keys && key_tiles >= 32 ? 2L * cus : cus, fit = (long)(prefill_added_scratch(cus) / part_bytes);
    sp.nseg = (int)max(1L, min(min(min(want / wgs, fit), 16L), key_tiles / 4));
    if (wgs * sp.nseg > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: dimension too large");
    if (sp.nseg > 1) {
        if (const int rc = ensure_scratch2(ctx, sp.nseg * part_bytes)) return rc;
        sp.parts = (float *)ctx->scratch2;
    }
    static std::atomic<uint64_t> attr{0};
    if (const int rc = allow_lds(ctx, attr, (const void *)quant_prompt_kernel<DT, D>, Cfg::LDS_BYTES)) return rc;
    {
        ProfScope scope(ctx, "attn_quant_prompt");
        launch_k(ctx, quant_prompt_kernel<DT, D>, dim3((unsigned)(wgs * sp.nseg)), dim3(Cfg::WAVES * 64), Cfg::LDS_BYTES, a, sp);
    }
    if (sp.nseg > 1) launch_merge<D, 1>(ctx, a, sp);
    LAUNCH_CHECK(ctx, "attn_quant_prompt");
    return AIONHIP_OK;
}

template <int DT, int D>
int launch_rows(aionhip_ctx *ctx, const QuantArgs &a) {
    // Few rows are cheaper tile by tile. us, rows a tile / many rows: 96 rows of 8 x 128 in 8 bits over 4000 keys 23 / 37, eight sequences of them 80 / 109, 192 rows
    // 29 / 41 and 142 / 111; 96 rows of 4 x 64 over 3000 keys, four sequences, 15 / 27; 64 rows of 256 in 4 bits over 5000 keys 38 / 41, 96 rows over 3000 38 / 35.
    if ((long)a.L * a.groups > (D > 128 ? 64 : 128)) return launch_prompt<DT, D>(ctx, a);
    return launch_decode_rows<DT, D>(ctx, a);
}

template <int DT>
int launch(aionhip_ctx *ctx, const QuantArgs &a) {
    if (a.d_k == a.d_v) {
        if (a.d_k == 64) return launch_rows<DT, 64>(ctx, a);
        if (a.d_k == 128) return launch_rows<DT, 128>(ctx, a);
        if (a.d_k == 256) return launch_rows<DT, 256>(ctx, a);
    }
    return launch_generic<DT>(ctx, a);
}

}  // namespace

// The step over quantized caches; its operands have been checked as far as every cache type wants them checked (attention.hip).
int run_attention_quant(aionhip_ctx *ctx, const aionhip_attention *p) {
    if (p->d_k % 32 != 0 || p->d_v % 32 != 0) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention: head sizes over a quantized cache are multiples of 32");
    if (p->d_k > GENERIC_HEAD || p->d_v > GENERIC_HEAD) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: head sizes above %d over a quantized cache", GENERIC_HEAD);
    if ((p->k | p->v) & 15) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention: a quantized cache begins at a multiple of 16 bytes");
    const size_t k_bytes = aionhip_cache_quant_bytes(p->kv_dtype, p->batch, p->t_kv, p->h_kv, p->d_k), v_bytes = aionhip_cache_quant_bytes(p->kv_dtype, p->batch, p->t_kv, p->h_kv, p->d_v);
    if (!k_bytes || !v_bytes) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention: dimension too large");
    const aionhip_handle out_end = p->out + p->batch * p->l_q * p->h_q * p->d_v * sizeof(float);
    if ((p->out < p->k + k_bytes && p->k < out_end) || (p->out < p->v + v_bytes && p->v < out_end))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention: the output lies in a quantized cache of the call");
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
