// Writing rows into caches held in 8 or 4 bits and reading them back (the layout: cache_quant.h). One pass over the data each; what a call
// of a few rows costs is its launch, what one of many rows costs is memory.
#include "cache_quant.h"

#include <cmath>
#include <cstring>
#include <initializer_list>
#include <type_traits>
#include <utility>

namespace {
using namespace cq;

template <typename T> T *dp(aionhip_handle h) { return reinterpret_cast<T *>((uintptr_t)h); }

// eight values of any alignment their type allows (global memory takes wide accesses at any address)
__device__ __forceinline__ void load8(const void *src, int dtype, size_t i, float (&x)[8]) {
    if (dtype == AIONHIP_F32) {
        __builtin_memcpy(x, (const float *)src + i, 32);
        return;
    }
    unsigned short h[8];
    __builtin_memcpy(h, (const unsigned short *)src + i, 16);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = dtype == AIONHIP_F16 ? __half2float(__ushort_as_half(h[j])) : __uint_as_float((unsigned)h[j] << 16);
}

// the row of a cache that step `t` of a sequence lives in, or -1: outside of a linear cache, or before the first step
__device__ __forceinline__ long row_of(long t, int t_cap, int rolling) {
    if (t < 0) return -1;
    if (rolling) return (long)((unsigned)t % (unsigned)t_cap);              // (an index and a count of rows, below 2^31 each)
    return t < (long)t_cap ? t : -1;
}

// four lanes store a block: `at` = its head's row, `col` = the lane's first element
template <int DT>
__device__ __forceinline__ void store_block8(unsigned char *codes, __half *scales, size_t unit, long row, int tp, int d, int col, const float (&x)[8]) {
    unsigned word[2];
    __half scale;
    quantize8<DT>(x, word, scale);
    if (row < 0) return;                                       // (behind the exchange between the lanes)
    if constexpr (DT == AIONHIP_Q8_0) {
        unsigned char *o = codes + (unit * tp + (size_t)row) * d + col;
        *(uint2 *)o = make_uint2(word[0], word[1]);
    } else {
        *(unsigned *)(codes + (unit * tp + (size_t)row) * (d / 2) + col / 2) = word[0];
    }
    if ((col & 31) == 0) scales[(unit * (d / 32) + col / 32) * tp + (size_t)row] = scale;
}

struct Pair {
    unsigned char *codes[2];
    __half *scales[2];
    const void *rows[2];
};

// How append_quant_kernel and cache_read_kernel share the rows out: a workgroup has ROWS_EACH * `rows` tokens of one head, so that what it touches of the cache is
// one run of codes and a run of each block's scales; a thread has the same few
// elements of ROWS_EACH of them, all asked for before the first is used.
constexpr int ROWS_EACH = 2;
struct Tiles {
    unsigned per, rows, wgs;     // threads to a row, rows side by side, workgroups of a head
};
struct Place {
    unsigned unit, first, piece;      // sequence and head; the thread's first token (past every length: none) and its elements
};
__device__ __forceinline__ Place place_of(const Tiles &t) {
    const unsigned unit = blockIdx.x / t.wgs, row = threadIdx.x / min(t.per, 256u);
    return Place{unit, row < t.rows ? (blockIdx.x - unit * t.wgs) * t.rows * ROWS_EACH + row : 0xFFFF0000u, threadIdx.x - row * t.per};
}

// SequenceAppend with the quantization in it: four threads hold a block. 8000 tokens of 8 heads of 128, k and v, f32 to
// q4_0: 15.7 us, 4.8 TB/s of 5.1 that a copy reaches (twenty passes from rest 16.7; one token to a thread 17.3, four 19.0).
template <int DT>
__global__ __launch_bounds__(256) void append_quant_kernel(Pair p, const int *write_index, int src_dtype, int s_len, int t_cap, int tp, int h, int d, int rolling, Tiles tiles) {
    const Place at = place_of(tiles);
    const unsigned b = at.unit / (unsigned)h, head = at.unit - b * (unsigned)h;
    const int which = blockIdx.y, index = write_index[b];
    for (unsigned piece = at.piece; piece < tiles.per; piece += 256) {
        float x[ROWS_EACH][8];
#pragma unroll
        for (int r = 0; r < ROWS_EACH; ++r) {
            const unsigned s = at.first + r * tiles.rows;
            if (s < (unsigned)s_len) load8(p.rows[which], src_dtype, (((size_t)b * s_len + s) * h + head) * d + piece * 8, x[r]);
        }
#pragma unroll
        for (int r = 0; r < ROWS_EACH; ++r) {
            const unsigned s = at.first + r * tiles.rows;
            if (s < (unsigned)s_len) store_block8<DT>(p.codes[which], p.scales[which], at.unit, row_of((long)index + s, t_cap, rolling), tp, d, (int)piece * 8, x[r]);
        }
    }
}

// RoPE1D on q and k, and the append of k and v, for the tokens of one step: a thread holds eight elements of one head of one token. What it rotates
// with lies half a head away, in another thread, and is read a second time rather than exchanged. The bits of aionhip_step_rope and aionhip_step_append_quant.
// 4096 tokens, 32 + 8 + 8 heads of 128, q4_0: 39.9 us, 4.3 TB/s, the second reading not counted; one token 3.9 us, the launch and two loads that wait for each other.
template <int DT>
__global__ __launch_bounds__(256) void rope_append_quant_kernel(float *q_out, const float *q, const float *k, const float *v, Cache kc, Cache vc, const int *positions,
                                                                const int *write_index, int s_len, int t_cap, int tp, int h_q, int h_kv, int d, int rope_pairs,
                                                                const float *freq, int rolling, unsigned total) {
    const unsigned gid = blockIdx.x * 256u + threadIdx.x;
    if (gid >= total) return;
    const unsigned per = (unsigned)d / 8, slots = h_q + 2 * h_kv;
    const int half = d / 2;
    const unsigned head_at = gid / per, tok32 = head_at / slots;
    const int col = (int)(gid - head_at * per) * 8;
    const int slot = (int)(head_at - tok32 * slots);
    const size_t tok = tok32;
    const bool is_q = slot < h_q, is_v = slot >= h_q + h_kv;
    const int head = is_q ? slot : is_v ? slot - h_q - h_kv : slot - h_q;
    const size_t row0 = is_q ? (tok * h_q + head) * d : (tok * h_kv + head) * d;
    const float *src = is_q ? q : is_v ? v : k;
    const unsigned b = tok32 / (unsigned)s_len;
    const int pos = positions[tok], at = write_index[b];
    float x[8];
    load8(src, AIONHIP_F32, row0 + col, x);
    const bool high = col >= half;
    const int first = high ? col - half : col;                               // of its eight pairs (half a head is a multiple of sixteen)
    if (!is_v && first < rope_pairs) {
        float other[8];
        load8(src, AIONHIP_F32, row0 + (high ? first : col + half), other);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (first + i >= rope_pairs) continue;
            float sn, cs, yl, yh;
            sincosf((float)pos * freq[first + i], &sn, &cs);
            rope_rotate(high ? other[i] : x[i], high ? x[i] : other[i], sn, cs, yl, yh);
            x[i] = high ? yh : yl;
        }
    }
    if (is_q) {
        __builtin_memcpy(q_out + row0 + col, x, 32);
        return;                                                              // (whole blocks: the four lanes of one leave together)
    }
    const long row = row_of((long)at + (long)(tok32 - b * (unsigned)s_len), t_cap, rolling);
    const Cache &c = is_v ? vc : kc;
    store_block8<DT>(c.codes, c.scales, (size_t)b * h_kv + head, row, tp, d, col, x);
}

struct ReadPair {
    const unsigned char *codes[2];
    const __half *scales[2];
    void *out[2];
};

// Rows first[b] .. first[b] + s_len - 1 as numbers; a row that the cache does not hold is zeros. The product of a code and a scale is exact in f32 and rounded once.
// A thread has sixteen bytes of the result, so that a wavefront's store is whole lines, which pass the caches by: they would push out what is read.
// 4 x 16000 tokens of 8 heads of 128, q4_0 to f16: 25.8 us, 6.5 TB/s (twenty passes from rest 28.3; 41.5 through the caches; there 45.7 with one token to a thread, and 58
// with the threads in the result's order, where a workgroup has two bytes of each scale line). 8000 tokens of k and v, q4_0 to f32: 14.8 us, 5.1 TB/s (32 bytes a thread:
// 16.7, and 28 past the caches, half lines at a time).
constexpr int read_each(int out) { return out == AIONHIP_F32 ? 4 : 8; }      // elements of a thread
template <int DT, int OUT>
__global__ __launch_bounds__(256) void cache_read_kernel(ReadPair p, const int *first, int s_len, int t_cap, int tp, int h, int d, int rolling, Tiles tiles) {
    constexpr int E = read_each(OUT), BYTES = DT == AIONHIP_Q8_0 ? E : E / 2;
    using Codes = std::conditional_t<BYTES == 8, unsigned long, std::conditional_t<BYTES == 4, unsigned, unsigned short>>;
    typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(2)));
    const Place at = place_of(tiles);
    const unsigned b = at.unit / (unsigned)h, head = at.unit - b * (unsigned)h;
    const int which = blockIdx.y, index = first[b];
    for (unsigned piece = at.piece; piece < tiles.per; piece += 256) {
        Codes w[ROWS_EACH];
        float scale[ROWS_EACH];
#pragma unroll
        for (int r = 0; r < ROWS_EACH; ++r) {
            const unsigned s = at.first + r * tiles.rows;
            const long row = s < (unsigned)s_len ? row_of((long)index + s, t_cap, rolling) : -1;
            w[r] = DT == AIONHIP_Q8_0 ? (Codes)0x8080808080808080ul : (Codes)0x88888888u;
            scale[r] = 0.f;
            if (row >= 0) {
                scale[r] = __half2float(p.scales[which][((size_t)at.unit * (d / 32) + piece / (32 / E)) * tp + (size_t)row]);
                w[r] = *(const Codes *)(p.codes[which] + ((size_t)at.unit * tp + (size_t)row) * (DT == AIONHIP_Q8_0 ? d : d / 2) + piece * BYTES);
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS_EACH; ++r) {
            const unsigned s = at.first + r * tiles.rows;
            if (s >= (unsigned)s_len) continue;
            const size_t o_at = (((size_t)b * s_len + s) * h + head) * d + piece * E;
            float x[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if constexpr (DT == AIONHIP_Q8_0) x[i] = (float)((int)(w[r] >> (8 * i) & 255u) - 128) * scale[r];
                else x[i] = (float)((int)(w[r] >> (4 * i) & 15u) - 8) * scale[r];
            }
            u32x4u o;
            if constexpr (OUT == AIONHIP_F32) {
                __builtin_memcpy(&o, x, 16);
                __builtin_nontemporal_store(o, (u32x4u *)((float *)p.out[which] + o_at));
            } else {
                unsigned short half[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (OUT == AIONHIP_F16) half[i] = __half_as_ushort(__float2half_rn(x[i]));
                    else half[i] = __builtin_bit_cast(unsigned short, (__bf16)x[i]);
                }
                __builtin_memcpy(&o, half, 16);
                __builtin_nontemporal_store(o, (u32x4u *)((unsigned short *)p.out[which] + o_at));
            }
        }
    }
}

int check_shape(aionhip_ctx *ctx, const char *who, int dtype, size_t b, size_t s, size_t t_cap, size_t h, size_t d) {
    if (!is_quant(dtype)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: caches are q8_0 or q4_0, not dtype %d", who, dtype);
    if (d % 32 != 0) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: head size %zu is not a multiple of 32", who, d);
    if (d > MAX_HEAD || h > MAX_HEADS || t_cap > MAX_ROWS || b > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: dimension too large", who);
    if (s > t_cap) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: %zu tokens exceed the cache capacity %zu", who, s, t_cap);
    if (b && h && d && t_cap && !aionhip_cache_quant_bytes(dtype, b, t_cap, h, d)) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: size overflow", who);
    return AIONHIP_OK;
}
// the workgroups of `b` sequences' `h` heads with `s` rows of `per` threads each
int tiles_of(aionhip_ctx *ctx, const char *who, size_t b, size_t s, size_t h, size_t per, Tiles *tiles, unsigned *grid) {
    const size_t rows = per < 256 ? 256 / per : 1, wgs = (s + rows * ROWS_EACH - 1) / (rows * ROWS_EACH);
    if (b > 0x7FFFFFFF / h || b * h > 0x7FFFFFFF / wgs) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: too many rows for one launch", who);
    *tiles = Tiles{(unsigned)per, (unsigned)rows, (unsigned)wgs};
    *grid = (unsigned)(b * h * wgs);
    return AIONHIP_OK;
}
bool overlap(aionhip_handle a, size_t a_bytes, aionhip_handle b, size_t b_bytes) { return a && b && a < b + b_bytes && b < a + a_bytes; }
// rows that are read or written while the caches are written or read lie outside of both
int check_rows(aionhip_ctx *ctx, const char *who, std::initializer_list<std::pair<aionhip_handle, size_t>> rows, aionhip_handle k_cache, aionhip_handle v_cache, size_t cache_bytes) {
    for (const auto &r : rows)
        if (overlap(r.first, r.second, k_cache, cache_bytes) || overlap(r.first, r.second, v_cache, cache_bytes))
            return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: rows lie in a cache of the call", who);
    return AIONHIP_OK;
}
int check_cache(aionhip_ctx *ctx, const char *who, aionhip_handle c) {
    return c & 15 ? set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a cache begins at a multiple of 16 bytes", who) : AIONHIP_OK;
}

}  // namespace

extern "C" {

size_t aionhip_cache_quant_bytes(int dtype, size_t b, size_t t_cap, size_t h, size_t d) {
    if (!is_quant(dtype) || !b || !t_cap || !h || !d || d % 32 != 0 || d > MAX_HEAD || h > MAX_HEADS || t_cap > MAX_ROWS) return 0;
    const size_t rows = h * padded(t_cap), row = row_bytes(dtype, d) + d / 32 * 2;          // < 2^48 * 2^17
    if (rows > ((size_t)1 << 46) || b > ((size_t)1 << 62) / (rows * row)) return 0;
    return b * rows * row;
}

int aionhip_step_append_quant(aionhip_ctx *ctx, int dtype, aionhip_handle k_cache, aionhip_handle k, aionhip_handle v_cache, aionhip_handle v, int src_dtype,
                              aionhip_handle write_index, size_t b, size_t s, size_t t_cap, size_t h, size_t d, int rolling) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (!k_cache || !k || !write_index || !v_cache != !v) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "append_quant: null operand");
    if (src_dtype != AIONHIP_F32 && src_dtype != AIONHIP_F16 && src_dtype != AIONHIP_BF16)
        return set_err(ctx, AIONHIP_UNSUPPORTED, "append_quant: rows are f32, f16 or bf16, not dtype %d", src_dtype);
    int rc = check_shape(ctx, "append_quant", dtype, b, s, t_cap, h, d);
    if (!rc) rc = check_cache(ctx, "append_quant", k_cache | v_cache);
    if (rc || !b || !s || !h || !d) return rc;
    const size_t bytes = aionhip_cache_quant_bytes(dtype, b, t_cap, h, d);
    if (overlap(k_cache, bytes, v_cache, bytes)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "append_quant: the caches of keys and values overlap");
    Tiles tiles;
    unsigned grid;
    if ((rc = tiles_of(ctx, "append_quant", b, s, h, d / 8, &tiles, &grid))) return rc;
    const size_t row_bytes = b * s * h * d * (src_dtype == AIONHIP_F32 ? 4 : 2);
    if ((rc = check_rows(ctx, "append_quant", {{k, row_bytes}, {v, row_bytes}}, k_cache, v_cache, bytes))) return rc;
    const Cache kc = view(k_cache, dtype, b, t_cap, h, d), vc = v_cache ? view(v_cache, dtype, b, t_cap, h, d) : kc;
    const Pair p{{kc.codes, vc.codes}, {kc.scales, vc.scales}, {dp<void>(k), dp<void>(v)}};
    ProfScope scope(ctx, "append_quant");
    launch_k(ctx, dtype == AIONHIP_Q8_0 ? append_quant_kernel<AIONHIP_Q8_0> : append_quant_kernel<AIONHIP_Q4_0>, dim3(grid, v ? 2 : 1), dim3(256), 0, p,
             dp<const int>(write_index), src_dtype, (int)s, (int)t_cap, (int)padded(t_cap), (int)h, (int)d, rolling ? 1 : 0, tiles);
    LAUNCH_CHECK(ctx, "append_quant");
    return AIONHIP_OK;
}

int aionhip_step_rope_append_quant(aionhip_ctx *ctx, int dtype, aionhip_handle q_out, aionhip_handle q, aionhip_handle k, aionhip_handle v, aionhip_handle k_cache,
                                   aionhip_handle v_cache, aionhip_handle positions, aionhip_handle write_index, size_t b, size_t s, size_t t_cap, size_t h_q, size_t h_kv,
                                   size_t d, float base_frequency, float scale_factor, float rope_proportion, int rolling) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (!q_out || !q || !k || !v || !k_cache || !v_cache || !positions || !write_index) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rope_append_quant: null operand");
    if (!(base_frequency > 0.f) || !(base_frequency < INFINITY) || !(scale_factor > 0.f) || !(scale_factor < INFINITY) || !(rope_proportion >= 0.f && rope_proportion <= 1.f))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rope_append_quant: base/scale must be positive and finite, proportion in [0,1]");
    int rc = check_shape(ctx, "rope_append_quant", dtype, b, s, t_cap, h_kv, d);
    if (!rc) rc = check_cache(ctx, "rope_append_quant", k_cache | v_cache);
    if (rc || !b || !s || !h_q || !h_kv || !d) return rc;
    if (h_q > MAX_HEADS) return set_err(ctx, AIONHIP_UNSUPPORTED, "rope_append_quant: dimension too large");
    const size_t bytes = aionhip_cache_quant_bytes(dtype, b, t_cap, h_kv, d);
    if (overlap(k_cache, bytes, v_cache, bytes)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rope_append_quant: the caches of keys and values overlap");
    const size_t half = d / 2, slots = (h_q + 2 * h_kv) * (d / 8);
    if (b > 0x7FFFFFFF / s || b * s > 0xFFFFFF00u / slots) return set_err(ctx, AIONHIP_UNSUPPORTED, "rope_append_quant: too many rows for one launch");
    const unsigned total = (unsigned)(b * s * slots), grid = (total + 255) / 256;
    const size_t q_bytes = b * s * h_q * d * sizeof(float), kv_bytes = b * s * h_kv * d * sizeof(float);
    if (overlap(q_out, q_bytes, q, q_bytes) || overlap(q_out, q_bytes, k, kv_bytes) || overlap(q_out, q_bytes, v, kv_bytes))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rope_append_quant: q, k and v are still read while q_out is written");
    if ((rc = check_rows(ctx, "rope_append_quant", {{q_out, q_bytes}, {q, q_bytes}, {k, kv_bytes}, {v, kv_bytes}}, k_cache, v_cache, bytes))) return rc;
    size_t rope_pairs = (size_t)floorf(rope_proportion * (float)half);
    if (rope_pairs > half) rope_pairs = half;
    const float freq_step = (float)pow((double)base_frequency, (double)(-2.0f / (float)d));
    const float *freq = nullptr;
    if ((rc = rope_table(ctx, (int)rope_pairs, freq_step, scale_factor, &freq))) return rc;
    ProfScope scope(ctx, "rope_append_quant");
    launch_k(ctx, dtype == AIONHIP_Q8_0 ? rope_append_quant_kernel<AIONHIP_Q8_0> : rope_append_quant_kernel<AIONHIP_Q4_0>, dim3(grid), dim3(256), 0, dp<float>(q_out),
             dp<const float>(q), dp<const float>(k), dp<const float>(v), view(k_cache, dtype, b, t_cap, h_kv, d), view(v_cache, dtype, b, t_cap, h_kv, d),
             dp<const int>(positions), dp<const int>(write_index), (int)s, (int)t_cap, (int)padded(t_cap), (int)h_q, (int)h_kv, (int)d, (int)rope_pairs, freq,
             rolling ? 1 : 0, total);
    LAUNCH_CHECK(ctx, "rope_append_quant");
    return AIONHIP_OK;
}

int aionhip_step_cache_read(aionhip_ctx *ctx, int dtype, int out_dtype, aionhip_handle k_out, aionhip_handle k_cache, aionhip_handle v_out, aionhip_handle v_cache,
                            aionhip_handle first, size_t b, size_t s, size_t t_cap, size_t h, size_t d, int rolling) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (!k_out || !k_cache || !first || !v_out != !v_cache) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "cache_read: null operand");
    if (out_dtype != AIONHIP_F32 && out_dtype != AIONHIP_F16 && out_dtype != AIONHIP_BF16)
        return set_err(ctx, AIONHIP_UNSUPPORTED, "cache_read: rows are f32, f16 or bf16, not dtype %d", out_dtype);
    int rc = check_shape(ctx, "cache_read", dtype, b, s, t_cap, h, d);
    if (!rc) rc = check_cache(ctx, "cache_read", k_cache | v_cache);
    if (rc || !b || !s || !h || !d) return rc;
    const size_t out_bytes = b * s * h * d * (out_dtype == AIONHIP_F32 ? 4 : 2);
    if (overlap(k_out, out_bytes, v_out, out_bytes)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "cache_read: the rows of keys and values overlap");
    Tiles tiles;
    unsigned grid;
    if ((rc = tiles_of(ctx, "cache_read", b, s, h, d / read_each(out_dtype), &tiles, &grid))) return rc;
    if ((rc = check_rows(ctx, "cache_read", {{k_out, out_bytes}, {v_out, out_bytes}}, k_cache, v_cache, aionhip_cache_quant_bytes(dtype, b, t_cap, h, d)))) return rc;
    const Cache kc = view(k_cache, dtype, b, t_cap, h, d), vc = v_cache ? view(v_cache, dtype, b, t_cap, h, d) : kc;
    const ReadPair p{{kc.codes, vc.codes}, {kc.scales, vc.scales}, {dp<void>(k_out), dp<void>(v_out)}};
    const auto kernel = dtype == AIONHIP_Q8_0 ? (out_dtype == AIONHIP_F32 ? cache_read_kernel<AIONHIP_Q8_0, AIONHIP_F32>
                                                 : out_dtype == AIONHIP_F16 ? cache_read_kernel<AIONHIP_Q8_0, AIONHIP_F16> : cache_read_kernel<AIONHIP_Q8_0, AIONHIP_BF16>)
                                              : (out_dtype == AIONHIP_F32 ? cache_read_kernel<AIONHIP_Q4_0, AIONHIP_F32>
                                                 : out_dtype == AIONHIP_F16 ? cache_read_kernel<AIONHIP_Q4_0, AIONHIP_F16> : cache_read_kernel<AIONHIP_Q4_0, AIONHIP_BF16>);
    ProfScope scope(ctx, "cache_read");
    launch_k(ctx, kernel, dim3(grid, v_out ? 2 : 1), dim3(256), 0, p, dp<const int>(first), (int)s, (int)t_cap, (int)padded(t_cap), (int)h, (int)d, rolling ? 1 : 0, tiles);
    LAUNCH_CHECK(ctx, "cache_read");
    return AIONHIP_OK;
}

}  // extern "C"
