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

// ---------------------------------------------------------------------------------------------------------------------- few query rows
using h2 = __attribute__((ext_vector_type(2))) _Float16;

// Codes as the half-precision numbers they are, offset taken off: a code under the mantissa of 1024 is 1024 + code, and the rest is exact.
// 4 bits: eight codes of a word, in the order 0 4 1 5 2 6 3 7 (a mask takes every fourth nibble of them).
__device__ __forceinline__ u32x4 halves_q4(unsigned w) {
    const unsigned m = 0x000F000Fu, one = 0x64006400u, v = w >> 8;
    const h2 low{(_Float16)-1032.f, (_Float16)-1032.f}, high{(_Float16)-72.f, (_Float16)-72.f}, by{(_Float16)0.0625f, (_Float16)0.0625f};
    const h2 a = __builtin_bit_cast(h2, (w & m) | one) + low, b = __builtin_bit_cast(h2, (w & (m << 4)) | one) * by + high;
    const h2 c = __builtin_bit_cast(h2, (v & m) | one) + low, d = __builtin_bit_cast(h2, (v & (m << 4)) | one) * by + high;
    return u32x4{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, c), __builtin_bit_cast(unsigned, d)};
}
// 8 bits: the eight codes of two words, in order
__device__ __forceinline__ u32x4 halves_q8(unsigned w0, unsigned w1) {
    const h2 off{(_Float16)-1152.f, (_Float16)-1152.f};
    auto pair = [&](unsigned w, unsigned sel) {
        return __builtin_bit_cast(unsigned, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, sel)) + off);
    };
    return u32x4{pair(w0, 0x04010400u), pair(w0, 0x04030402u), pair(w1, 0x04010400u), pair(w1, 0x04030402u)};
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
__device__ __forceinline__ unsigned pack_half(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b)); }

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
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\tds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %4 offset:3072\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]) : "v"(at) : "memory");
}

// Key segments: every workgroup of a row tile takes a share of its sequence's 64-key tiles and leaves sums over them; `parts` holds those, `tickets`
// (not null) lets the workgroup that ends last add them up, otherwise quant_merge_kernel does.
struct Split {
    float *parts;
    unsigned *tickets;
    int nseg, row_tiles;
};
constexpr int NW = 4;                       // wavefronts of a workgroup
constexpr int MAX_SEG = 256;                // most segments of a row tile (the merge's table of factors)

template <int D, int REP>
struct Part {                               // a row tile's sums: o [rows][D], then (reference, sum) of its 16 columns
    static constexpr int ROWS = 16 / REP, FLOATS = ROWS * D + 32;
};

// Sums of all segments of a row tile -> output rows. The wavefronts derive the segments' factors, a lane to a segment, then every thread adds four
// columns of a row over the segments in their order. `at(i, n)`: n (2 or 4) floats of the tile's parts from the i-th on.
template <int D, int REP, class Load, class Store>
__device__ __forceinline__ void merge_parts(int nseg, int rows, int first, int step, float (*factor)[MAX_SEG], float *total, Load &&load, Store &&store) {
    constexpr int ROWS = Part<D, REP>::ROWS, FLOATS = Part<D, REP>::FLOATS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int c = wave; c < 16; c += NW) {
        float ref[MAX_SEG / 64], top = REF_NONE, sum = 0.f;
        float l[MAX_SEG / 64];
#pragma unroll
        for (int j = 0; j < MAX_SEG / 64; ++j) {
            const int s = lane + 64 * j;
            const u32x2 x = s < nseg ? load(std::integral_constant<int, 2>{}, (size_t)s * FLOATS + ROWS * D + 2 * c) : u32x2{__float_as_uint(REF_NONE), 0u};
            ref[j] = __uint_as_float(x.x);
            l[j] = __uint_as_float(x.y);
            top = fmaxf(top, ref[j]);
        }
        top = lanes_max(top);
#pragma unroll
        for (int j = 0; j < MAX_SEG / 64; ++j) {
            const float f = exp2f(ref[j] - top);
            if (lane + 64 * j < nseg) factor[c][lane + 64 * j] = f;
            sum += l[j] * f;
        }
        sum = lanes_sum(sum);
        if (lane == 0) total[c] = sum;
    }
    __syncthreads();
    for (int e = first; e < rows * (D / 4); e += step) {
        const int row = e / (D / 4), col = e % (D / 4) * 4, c = (col / 32) % REP * ROWS + row;
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < nseg; s0 += 8) {
            u32x4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = load(std::integral_constant<int, 4>{}, (size_t)min(s0 + u, nseg - 1) * FLOATS + row * D + col);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (s0 + u < nseg) o += __builtin_bit_cast(f32x4, x[u]) * factor[c][s0 + u];
        }
        const float l = total[c];
        store(row, col, o * (l != 0.f ? 1.f / l : 0.f));
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
// between 2^9 and 2^15; the low part then ends 2^-34 below it. No shift is made for a value that is not finite.
// Tiles are 64 keys, 32 at head size 256; there, and where sixteen rows share the columns, the query's operands lie in LDS as well: the registers hold no more.
template <int DT, int D, int REP>
struct DecodeCfg {
    static constexpr int TK = D > 128 ? 32 : 64, RB = DT == AIONHIP_Q8_0 ? D : D / 2, ROWS = 16 / REP;
    static constexpr bool Q_LDS = D > 128 || (D == 128 && REP == 1);
    static constexpr bool PV_TWICE = D / 32 / REP * (TK / 4) > 32;              // P' is made once for its maximum and again for its use
    static constexpr int Q_BYTES = Q_LDS ? D / 32 * 2 * 1024 : 0, V_BYTES = NW * TK * RB;
    static constexpr int MEET_BYTES = NW * (ROWS * (D + 4) + 32) * 4, TABLE_BYTES = (16 * MAX_SEG + 16) * 4;
    static constexpr int MOST = MEET_BYTES > TABLE_BYTES ? MEET_BYTES : TABLE_BYTES;
    static constexpr int LDS_BYTES = Q_BYTES + V_BYTES > MOST ? Q_BYTES + V_BYTES : MOST;
};
template <int DT, int D, int REP>
__global__ __launch_bounds__(NW * 64, 2) void quant_decode_kernel(QuantArgs a, Split sp) {
    using Cfg = DecodeCfg<DT, D, REP>;
    constexpr int ROWS = 16 / REP, KK = D / 32, MT = D / 16, SETS = KK / REP;
    constexpr int TK = Cfg::TK, H = TK / 16, KG = TK / 4;                                  // keys of a tile; its sub-tiles; keys of a lane
    constexpr int RB = Cfg::RB, CH = RB / 16, KD = RB / 16;                                // bytes of a row; its 16-byte chunks; words of a K operand
    constexpr int FLOATS = Part<D, REP>::FLOATS;
    static_assert(KK % REP == 0 && SETS >= 1, "whole groups of blocks");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int rt = (int)blockIdx.x / sp.nseg, seg = (int)blockIdx.x - rt * sp.nseg, hk = (int)blockIdx.y, b = (int)blockIdx.z;
    const int unit = b * a.Hkv + hk, rows_total = a.L * a.groups;
    const int rows = min(ROWS, rows_total - rt * ROWS);
    const int sub = n / ROWS;

    // ---- this lane's query row (columns past the last row repeat it) and its visible keys
    const int r = rt * ROWS + min(n % ROWS, rows - 1), li = r / a.groups, hq = hk * a.groups + (r - li * a.groups);
    const size_t qbase = (((size_t)b * a.L + li) * a.Hq + hq) * D;
    constexpr int E0G = DT == AIONHIP_Q8_0 || D == 64;                  // where a lane's eight elements of a block begin, by how K is loaded
    const int e0 = E0G ? (g & 1) * 16 + (g >> 1) * 8 : g * 8;
    int lo, hi;
    visible(a, b, li, lo, hi);
    if (hi <= lo) lo = hi = 0;
    const int kv_end = clip_kv_end(a.ring, a.T, a.kv_lengths ? a.kv_lengths[b] : a.T);
    const int uni_lo = rows16_min_i(hi > lo ? lo : INT_MAX), uni_hi = rows16_max_i(hi), full_lo = rows16_max_i(lo), full_hi = rows16_min_i(hi);

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
    const int per = (count + sp.nseg - 1) / sp.nseg;
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
    auto load_k = [&](int i) __attribute__((always_inline)) {
        const int row0 = tile_of(i) * TK;
        const unsigned char *p = kc + (size_t)row0 * RB + k_lane;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if constexpr (KD == 2) {
                const u32x2 x = *(const u32x2 *)(p + h * 4 * RB);
                kw[h][0] = x.x;
                kw[h][1] = x.y;
            } else {
#pragma unroll
                for (int c = 0; c < KD / 4; ++c) {
                    const u32x4 x = *(const u32x4 *)(p + h * 4 * RB + c * 64);
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
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(v_lds + j * 1024), 16, (int)(v_lane ^ (unsigned)(((4 * j) & (CH - 1)) << 4)), j * 1024, 0, 0);
#endif
    };

    // ---- Q^T: eight elements of each block, in the order of K's codes, times 2^-e and the sign of the scale, in two parts
    float qx[KK][8], amax = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        if (a.q_dtype == AIONHIP_F32) {
            __builtin_memcpy(qx[kk], (const float *)a.q + qbase + kk * 32 + e0, 32);
        } else {
            unsigned short x[8];
            __builtin_memcpy(x, (const unsigned short *)a.q + qbase + kk * 32 + e0, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) qx[kk][j] = a.q_dtype == AIONHIP_F16 ? __half2float(__ushort_as_half(x[j])) : bf16_bits_to_f32(x[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qx[kk][j]));
    }
    if (t < t_end) {
        load_k(t);
        load_v(t);
    }
    amax = groups4_max(amax);
    const int e_q = amax < INFINITY ? max((int)(__float_as_uint(amax) >> 23), 2) : 127;           // (1 <= the biased exponents of 2^-e and 2^e <= 254)
    const float shrink_q = __uint_as_float((unsigned)(254 - min(e_q, 253)) << 23), grow_q = __uint_as_float((unsigned)min(e_q, 253) << 23);
    const float sign = a.scale < 0.f ? -shrink_q : shrink_q;
    const float row_scale = fabsf(a.scale) * grow_q;
    const float to_log2 = a.soft_cap > 0.f ? 1.f : row_scale * LOG2E;
    u32x4 q_op[Cfg::Q_LDS ? 1 : KK][2];
    const unsigned q_addr = (unsigned)(size_t)(lds_void *)lds + lane * 16;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        float x[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = kk % REP == sub ? qx[kk][element_slot<DT>(j)] * sign : 0.f;
            y[j] = x[j] - (float)(_Float16)x[j];
        }
        const u32x4 high{pack2<AIONHIP_F16>(x[0], x[1]), pack2<AIONHIP_F16>(x[2], x[3]), pack2<AIONHIP_F16>(x[4], x[5]), pack2<AIONHIP_F16>(x[6], x[7])};
        const u32x4 low{pack2<AIONHIP_F16>(y[0], y[1]), pack2<AIONHIP_F16>(y[2], y[3]), pack2<AIONHIP_F16>(y[4], y[5]), pack2<AIONHIP_F16>(y[6], y[7])};
        if constexpr (Cfg::Q_LDS) {                                           // (every wavefront has the same rows: each stores its share of the blocks)
            if (kk % NW == wave) {
                asm volatile("ds_write_b128 %0, %1 offset:%3\n\tds_write_b128 %0, %2 offset:%4" ::"v"(q_addr), "v"(high), "v"(low), "n"(kk * 2048), "n"(kk * 2048 + 1024) : "memory");
            }
        } else {
            q_op[kk][0] = high;
            q_op[kk][1] = low;
        }
    }
    if constexpr (Cfg::Q_LDS) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // (no wait for the loads in flight)

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
            for (int h = 0; h < H; ++h) d[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < REP; ++u) {
                const int kk = st * REP + u;
                if constexpr (Cfg::Q_LDS)
                    if (kk % 2 == 0) read_four(q_addr + kk * 2048, q4);
                const u32x4 high = Cfg::Q_LDS ? q4[kk % 2 * 2] : q_op[Cfg::Q_LDS ? 0 : kk][0], low = Cfg::Q_LDS ? q4[kk % 2 * 2 + 1] : q_op[Cfg::Q_LDS ? 0 : kk][1];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const u32x4 k8 = DT == AIONHIP_Q8_0 ? halves_q8(kw[h][2 * kk % KD], kw[h][(2 * kk + 1) % KD]) : halves_q4(kw[h][kk % KD]);
                    d[h] = mfma16<AIONHIP_F16>(k8, high, d[h]);
                    d[h] = mfma16<AIONHIP_F16>(k8, low, d[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = h * 4 + j;
                    s[key] = fma_half(d[h][j], ksc[st][key >> 3][(key & 7) >> 1], key & 1, st ? s[key] : 0.f);
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
#pragma unroll
            for (int j = 0; j < KG; ++j) s[j] = a.soft_cap * tanhf(s[j] * row_scale / a.soft_cap) * LOG2E;
        }
        // -- which keys this row sees; whole tiles that every row sees need no mask
        bool whole = row0 + TK <= a.T;
        {
            const int first = row0 < wrap ? base + row0 : base + row0 - a.ring;
            whole = whole && !(row0 < wrap && row0 + TK > wrap) && first >= full_lo && first + TK <= full_hi;
        }
        unsigned seen = 0xFFFFu;
        if (!whole) {
            seen = 0u;
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                const int p = row0 + g * KG + j, key = p < wrap ? base + p : base + p - a.ring;
                const bool ok = p < a.T && key >= lo && key < hi;
                seen |= ok ? 1u << j : 0u;
                s[j] = ok ? s[j] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < KG; ++j) mx = fmaxf(mx, s[j]);
        mx = groups4_max(mx);
        const float m_new = fmaxf(m_run, mx * to_log2);
        float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        const float ref = m_new - bias;
        float p[16], sum = 0.f;
#pragma unroll
        for (int j = 0; j < KG; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[j], to_log2, -ref));
        if (!whole) {
#pragma unroll
            for (int j = 0; j < KG; ++j) p[j] = seen >> j & 1 ? p[j] : 0.f;
        }
        m_run = m_new;
        // -- the largest P' of the column, and the shift that keeps it in range
        if (!whole) {                                                         // (the scale of a key that is not seen may be anything)
#pragma unroll
            for (int st = 0; st < SETS; ++st)
#pragma unroll
                for (int j = 0; j < KG; ++j) {
                    const unsigned w = vsc[st][j >> 3][(j & 7) >> 1];
                    vsc[st][j >> 3][(j & 7) >> 1] = seen >> j & 1 ? w : w & (j & 1 ? 0xFFFFu : 0xFFFF0000u);
                }
        }
        auto times_scale = [&](int st, int j) __attribute__((always_inline)) { return fma_half(p[j], vsc[st][j >> 3][(j & 7) >> 1], j & 1, 0.f); };
        float pv[Cfg::PV_TWICE ? 1 : SETS][KG], top = 0.f;
#pragma unroll
        for (int st = 0; st < SETS; ++st)
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                const float x = times_scale(st, j);
                top = fmaxf(top, x);
                if constexpr (!Cfg::PV_TWICE) pv[st][j] = x;
            }
        top = fmaxf(largest * alpha, groups4_max(top));
        if (__any(top > 32768.f || top < 512.f)) {
            const bool move = top > 0.f && top < INFINITY && (top > 32768.f || top < 512.f);
            const float by = move ? (float)(139 - (int)(__float_as_uint(top) >> 23)) : 0.f;      // to 2^12 .. 2^13
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
                    pl[step][j] = pack_half(fma_half(-1.f, high, 0, x), fma_half(-1.f, high, 1, y));
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
                            const u32x4 x = halves_q8(w.x, w.y);
                            o = mfma16<AIONHIP_F16>(x, ph[step], o);
                            o = mfma16<AIONHIP_F16>(x, pl[step], o);
                        } else {                                              // the even columns of the block, and the odd ones
                            const u32x4 x = halves_q4(w.x), y = halves_q4(w.y);
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
        const int rr = rt * ROWS + row, l2 = rr / a.groups, g2 = rr - l2 * a.groups;
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
            f[w] = exp2f(x[w] - ref);
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
    merge_parts<D, REP>(
        sp.nseg, rows, (int)threadIdx.x, NW * 64, (float (*)[MAX_SEG])lds, (float *)lds + 16 * MAX_SEG,
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

// The merge as a launch, for row tiles whose parts are too much for one workgroup: (row tile, share of the rows' columns, unit)
constexpr int MERGE_SHARES = 16;
template <int D, int REP>
__global__ __launch_bounds__(NW * 64) void quant_merge_kernel(QuantArgs a, Split sp) {
    __shared__ float factor[16][MAX_SEG], total[16];
    constexpr int ROWS = Part<D, REP>::ROWS, FLOATS = Part<D, REP>::FLOATS;
    const int rt = blockIdx.x / MERGE_SHARES, share = blockIdx.x % MERGE_SHARES, unit = blockIdx.y, b = unit / a.Hkv, hk = unit % a.Hkv;
    const float *parts = sp.parts + ((size_t)unit * sp.row_tiles + rt) * sp.nseg * FLOATS;
    merge_parts<D, REP>(
        sp.nseg, min(ROWS, a.L * a.groups - rt * ROWS), share * NW * 64 + (int)threadIdx.x, MERGE_SHARES * NW * 64, factor, total,
        [&](auto count_c, size_t at) __attribute__((always_inline)) {
            if constexpr (decltype(count_c)::value == 2) return *(const u32x2 *)(parts + at);
            else return *(const u32x4 *)(parts + at);
        },
        [&](int row, int col, f32x4 v) {
            const int rr = rt * ROWS + row, l2 = rr / a.groups, g2 = rr - l2 * a.groups;
            __builtin_memcpy(a.out + (((size_t)b * a.L + l2) * a.Hq + hk * a.groups + g2) * D + col, &v, 16);
        });
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
    sp.nseg = (int)max(1L, min(min((long)MAX_SEG, 4 * cus / tiles), (key_tiles + NW - 1) / NW));
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
    if (sp.nseg > 1 && !sp.tickets) {
        ProfScope scope(ctx, "attn_quant_merge");
        launch_k(ctx, quant_merge_kernel<D, REP>, dim3((unsigned)(sp.row_tiles * MERGE_SHARES), (unsigned)units), dim3(NW * 64), 0, a, sp);
    }
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

template <int DT>
int launch(aionhip_ctx *ctx, const QuantArgs &a) {
    if (a.d_k == a.d_v) {
        if (a.d_k == 64) return launch_decode_rows<DT, 64>(ctx, a);
        if (a.d_k == 128) return launch_decode_rows<DT, 128>(ctx, a);
        if (a.d_k == 256) return launch_decode_rows<DT, 256>(ctx, a);
    }
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
