// Rows turned by their positions, written to caches in pages and read back (the layout: cache_paged.h). One pass over the data each; what a call
// of a few rows costs is its launch, what one of many rows costs is memory.
#include "cache_paged.h"

#include <cmath>
#include <cstring>
#include <type_traits>

namespace {
using namespace paged;

template <typename T> T *dp(aionhip_handle h) { return reinterpret_cast<T *>((uintptr_t)h); }

template <int DT> struct Elem { using T = unsigned short; };
template <> struct Elem<AIONHIP_F32> { using T = float; };

template <int ALIGN> struct Wide;
template <> struct Wide<2> { typedef unsigned T __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Wide<4> { typedef unsigned T __attribute__((ext_vector_type(4), aligned(4))); };
template <size_t ALIGN> using u32x4u = typename Wide<(int)ALIGN>::T;

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::T x) {
    if constexpr (DT == AIONHIP_F32) return x;
    else if constexpr (DT == AIONHIP_F16) return __half2float(__ushort_as_half(x));
    else return __uint_as_float((unsigned)x << 16);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T from_f32(float x) {
    if constexpr (DT == AIONHIP_F32) return x;
    else if constexpr (DT == AIONHIP_F16) return __half_as_ushort(__float2half_rn(x));
    else return __builtin_bit_cast(unsigned short, (__bf16)x);
}
// N neighbouring elements, n of them there, of any alignment their type allows (global memory takes wide accesses at any address)
template <int DT, int N, bool ONCE = false>
__device__ __forceinline__ void load_n(const void *src, size_t i, int n, float (&x)[N]) {
    typename Elem<DT>::T h[N];
    const auto *p = (const typename Elem<DT>::T *)src + i;
    if (n == N) {
        if constexpr (ONCE && sizeof h >= 16) {
#pragma unroll
            for (size_t k = 0; k < sizeof h / 16; ++k) {
                const u32x4 w = __builtin_nontemporal_load((const u32x4u<sizeof h[0]> *)p + k);
                __builtin_memcpy((char *)h + 16 * k, &w, 16);
            }
        } else {
            __builtin_memcpy(h, p, sizeof h);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = j < n ? p[j] : typename Elem<DT>::T(0);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = to_f32<DT>(h[j]);
}
template <int DT, int N, bool ONCE = false>
__device__ __forceinline__ void store_n(void *dst, size_t i, int n, const float (&x)[N]) {
    typename Elem<DT>::T h[N];
#pragma unroll
    for (int j = 0; j < N; ++j) h[j] = from_f32<DT>(x[j]);
    auto *p = (typename Elem<DT>::T *)dst + i;
    if (n == N) {
        if constexpr (ONCE && sizeof h >= 16) {
#pragma unroll
            for (size_t k = 0; k < sizeof h / 16; ++k) {
                u32x4u<sizeof h[0]> w;
                __builtin_memcpy(&w, (const char *)h + 16 * k, 16);
                __builtin_nontemporal_store(w, (u32x4u<sizeof h[0]> *)p + k);
            }
        } else {
            __builtin_memcpy(p, h, sizeof h);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) p[j] = h[j];
    }
}

// Sine and cosine of an angle given as a fraction of a turn, 2^64 to the whole: the nearest quarter turn is taken off in integers, what is left, up to an eighth
// of a turn, is exact to 2^-32 and goes into the two power series (cut where the next term is below 2e-9). Every step is written out, here and in the rotation: left to itself
// the compiler fuses differently from kernel to kernel, and a row would have other bits alone than in front of an append.
__device__ __forceinline__ void sincos_turn(unsigned long turn, float &sn, float &cs) {
#pragma clang fp contract(off)
    const unsigned t = (unsigned)(turn >> 32), quarter = (t + 0x20000000u) >> 30;
    const float x = (float)(int)(t - (quarter << 30)) * 1.4629180792671596e-9f;            // 2 pi / 2^32
    const float z = x * x;
    const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    sn = quarter & 2 ? -a : a;
    cs = (quarter + 1) & 2 ? -b : b;
}

// A thread has E pairs, or 2 E elements that stay, of HEADS heads of one token: the angles, and the token's place in the pages, are found once for all of them. A head's
// elements are dealt out as `turning` pieces of pairs, then pieces of those that stay; the threads of a workgroup lie over pieces, then heads. One token, 32 + 8 + 8 heads of
// 128: 4.0 us, the launch and two loads. 8000 tokens of these, f32 to f16 pages: 60 us, 6.0 TB/s, with four heads to a thread (69 with one) and past the caches (71 through
// them: what is read and written here is more than they hold). 18000 rows of 32 heads of 128, f32, 96 elements turning: 110 us, 5.4 TB/s, with one head (120 with
// two or four), 138 through the caches.
struct Rotate {
    void *q_out;
    const void *q, *k, *v;
    const int *positions, *write_index;
    const unsigned long *turns;           // a pair's fraction of a turn a position
    float magnitude;
    int dims, interleaved, d, h_q, h_kv, s_len;
    int pieces, turning, heads_wg;        // of a head; of those that turn; heads side by side in a workgroup
    Table table;
    unsigned char *k_pages, *v_pages;
};
constexpr int pairs_each(int dt) { return dt == AIONHIP_F32 ? 4 : 8; }

template <int DT, int CT, int HEADS, bool ONCE>
__global__ __launch_bounds__(256) void rotary_kernel(Rotate a) {
    constexpr int E = pairs_each(DT);
    const int slot0 = (int)threadIdx.x / a.pieces, piece = (int)threadIdx.x - slot0 * a.pieces;
    if (slot0 >= a.heads_wg) return;
    const size_t tok = blockIdx.x;
    const int slots = a.h_q + 2 * a.h_kv, first = (int)blockIdx.y * a.heads_wg * HEADS + slot0;
    const int half = a.dims >> 1;
    const bool turns = piece < a.turning;
    // the thread's two runs of elements of a head: the two sides of its pairs, or a piece from either half of what lies side by side
    int lo, hi, n_lo, n_hi;
    if (turns && !a.interleaved) {
        lo = piece * E, hi = half + lo;
        n_lo = n_hi = min(E, half - lo);
    } else {
        const int begin = turns ? 0 : a.dims, end = turns ? a.dims : a.d, count = turns ? a.turning : a.pieces - a.turning, at = turns ? piece : piece - a.turning;
        lo = begin + at * E, hi = begin + (count + at) * E;
        n_lo = min(E, end - lo), n_hi = max(0, min(E, end - hi));
    }
    // what the heads need is asked for before the first of them is used
    float x[HEADS][2][E];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int slot = first + i * a.heads_wg;
        if (slot >= slots) break;
        const bool is_q = slot < a.h_q, is_v = slot >= a.h_q + a.h_kv;
        const void *src = is_q ? a.q : is_v ? a.v : a.k;
        const size_t at = is_q ? (tok * a.h_q + slot) * a.d : (tok * a.h_kv + (slot - a.h_q - (is_v ? a.h_kv : 0))) * a.d;
        load_n<DT, E, ONCE>(src, at + lo, n_lo, x[i][0]);
        load_n<DT, E, ONCE>(src, at + hi, n_hi, x[i][1]);
    }
    float sn[E], cs[E];
    if (turns) {
        const int pos = a.positions[tok];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int pair = !a.interleaved ? lo + j : j < E / 2 ? lo / 2 + j : hi / 2 + j - E / 2;
            sincos_turn(a.turns[min(pair, half - 1)] * (unsigned long)(long)pos, sn[j], cs[j]);
            sn[j] *= a.magnitude;
            cs[j] *= a.magnitude;
        }
    }
    int page = -1, row = 0;
    size_t seq = 0;
    if (a.write_index) {
        seq = (unsigned)tok / (unsigned)a.s_len;
        const long step = (long)a.write_index[seq] + (long)(tok - seq * (unsigned)a.s_len);
        page = step >= 0 && step < (long)MAX_ROWS ? page_of(a.table, seq, (int)step) : -1;
        row = (int)step & ((1 << a.table.shift) - 1);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int slot = first + i * a.heads_wg;
        if (slot >= slots) break;
        const bool is_q = slot < a.h_q, is_v = slot >= a.h_q + a.h_kv;
        float(&l)[E] = x[i][0], (&h)[E] = x[i][1];
        if (turns && !is_v) {
            if (a.interleaved) {
#pragma unroll
                for (int j = 0; j < E / 2; ++j) {
                    const float p = l[2 * j], r = l[2 * j + 1], u = h[2 * j], v = h[2 * j + 1];
                    rope_rotate(p, r, sn[j], cs[j], l[2 * j], l[2 * j + 1]);
                    rope_rotate(u, v, sn[E / 2 + j], cs[E / 2 + j], h[2 * j], h[2 * j + 1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const float p = l[j], r = h[j];
                    rope_rotate(p, r, sn[j], cs[j], l[j], h[j]);
                }
            }
        }
        if (is_q) {
            const size_t at = (tok * a.h_q + slot) * a.d;
            store_n<DT, E, ONCE>(a.q_out, at + lo, n_lo, l);
            store_n<DT, E, ONCE>(a.q_out, at + hi, n_hi, h);
        } else if (page >= 0) {
            const int head = slot - a.h_q - (is_v ? a.h_kv : 0);
            const size_t at = ((((size_t)page * a.h_kv + head) << a.table.shift) + row) * a.d;
            store_n<CT, E>(is_v ? a.v_pages : a.k_pages, at + lo, n_lo, l);
            store_n<CT, E>(is_v ? a.v_pages : a.k_pages, at + hi, n_hi, h);
        }
    }
}

// The same where a head does not come apart into whole pieces (62 of 64 elements turning in halves: runs at odd places, and short ones): a thread has eight neighbouring elements of a
// row whatever they are; the angles, and what they turn with in the other half, come through LDS, where element and pair e lie at [e % 8][e / 8], so that neighbouring threads meet
// neighbouring banks. Every element is the sum that rope_rotate writes for its side, with the same bits. us in pieces / so:
// 14 x 132 bf16 rows of 32 + 32 + 32 heads of 128, 106 elements turning in halves, 54 / 32; 37 x 30 f16 of 96 heads, 116 turning, 34 / 22; 2 x 1863 f16 of 24 heads of 64, 50 as neighbours,
// 17 / 11. Four heads to a thread, as above, are no faster here. Whole pieces are faster by themselves: 8000 tokens, 60, would take 72 this way.
template <int DT, int CT, bool ONCE>
__global__ __launch_bounds__(256) void rotary_rows_kernel(Rotate a) {
#pragma clang fp contract(off)
    __shared__ float rows[8][256], sines[8][MAX_HEAD / 16], cosines[8][MAX_HEAD / 16];
    const int chunks = a.d >> 3, slot0 = (int)threadIdx.x / chunks, at = ((int)threadIdx.x - slot0 * chunks) * 8;
    const size_t tok = blockIdx.x;
    const int slot = (int)blockIdx.y * a.heads_wg + slot0, half = a.dims >> 1;
    const bool mine = slot0 < a.heads_wg && slot < a.h_q + 2 * a.h_kv, is_q = slot < a.h_q, is_v = slot >= a.h_q + a.h_kv;
    const int head = is_q ? slot : slot - a.h_q - (is_v ? a.h_kv : 0);
    const size_t from = (tok * (is_q ? a.h_q : a.h_kv) + head) * a.d + at;
    float x[8] = {};
    if (mine) load_n<DT, 8, ONCE>(is_q ? a.q : is_v ? a.v : a.k, from, 8, x);
    const int pos = half > 0 ? a.positions[tok] : 0;               // (an append alone has none)
    for (int pair = (int)threadIdx.x; pair < half; pair += (int)blockDim.x) {
        float sn, cs;
        sincos_turn(a.turns[pair] * (unsigned long)(long)pos, sn, cs);
        sines[pair & 7][pair >> 3] = sn * a.magnitude;
        cosines[pair & 7][pair >> 3] = cs * a.magnitude;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) rows[j][threadIdx.x] = x[j];
    __syncthreads();
    if (!mine) return;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int e = at + j;
        const bool upper = a.interleaved ? j & 1 : e >= half;
        const int pair = max(0, min(a.interleaved ? e >> 1 : upper ? e - half : e, half - 1)), with = upper ? max(0, e - half) : min(e + half, a.d - 1);
        const float own = x[j], beside = x[j ^ 1], across = rows[with & 7][slot0 * chunks + (with >> 3)], sn = sines[pair & 7][pair >> 3], cs = cosines[pair & 7][pair >> 3];
        const float turned = own * cs + (a.interleaved ? beside : across) * (upper ? sn : -sn);
        y[j] = e < a.dims && !is_v ? turned : own;
    }
    if (is_q) {
        store_n<DT, 8, ONCE>(a.q_out, from, 8, y);
    } else if (a.write_index) {
        const size_t seq = (unsigned)tok / (unsigned)a.s_len;
        const long step = (long)a.write_index[seq] + (long)(tok - seq * (unsigned)a.s_len);
        const int page = step >= 0 && step < (long)MAX_ROWS ? page_of(a.table, seq, (int)step) : -1;
        if (page >= 0)
            store_n<CT, 8>(is_v ? a.v_pages : a.k_pages, ((((size_t)page * a.h_kv + head) << a.table.shift) + ((int)step & ((1 << a.table.shift) - 1))) * a.d + at, 8, y);
    }
}

struct ReadArgs {
    const unsigned char *pages[2];
    void *out[2];
    const int *first;
    Table table;
    int s_len, h, d;
};
// Rows back as numbers: a thread has eight elements of a row. Keys and values of 4 sequences, 8 heads of 128, f16: 4000 rows (125 MiB read and written) 20 us, 6.5 TB/s; 16000 104 us,
// 5.1 TB/s, memory's rate for copies (99 past the caches, which cost 50 instead of 37 at 8000 rows and is not done).
template <int CT, int OUT>
__global__ __launch_bounds__(256) void read_paged_kernel(ReadArgs a, size_t total) {
    const size_t gid = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (gid >= total) return;
    const unsigned per = (unsigned)a.d / 8;
    const size_t row = gid / per, tok = row / (unsigned)a.h, seq = (unsigned)tok / (unsigned)a.s_len;
    const int piece = (int)(gid - row * per), head = (int)(row - tok * (unsigned)a.h);
    const long step = (long)a.first[seq] + (long)(tok - seq * (unsigned)a.s_len);
    const int page = step >= 0 && step < (long)MAX_ROWS ? page_of(a.table, seq, (int)step) : -1;
    float x[8] = {};
    if (page >= 0) load_n<CT, 8>(a.pages[blockIdx.y], ((((size_t)page * a.h + head) << a.table.shift) + ((int)step & ((1 << a.table.shift) - 1))) * a.d + piece * 8, 8, x);
    store_n<OUT, 8>(a.out[blockIdx.y], row * a.d + piece * 8, 8, x);
}

bool row_type(int dt) { return dt == AIONHIP_F32 || dt == AIONHIP_F16 || dt == AIONHIP_BF16; }
size_t size_of(int dt) { return dt == AIONHIP_F32 ? 4 : 2; }

int check_rotary(aionhip_ctx *ctx, const char *who, const aionhip_rotary *r, size_t d) {
    if (!r) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: no rotary", who);
    auto positive = [](float x) { return x > 0.f && x < INFINITY; };
    if (r->dims % 2 != 0 || r->dims > d) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: %u turning elements of a head of %zu (an even number of them)", who, r->dims, d);
    if (r->scaling < AIONHIP_ROTARY_PLAIN || r->scaling > AIONHIP_ROTARY_RAMP) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: unknown scaling %d", who, r->scaling);
    if (!positive(r->base) || !(fabsf(r->magnitude) < INFINITY)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: base must be positive and finite, magnitude finite", who);
    if (r->scaling != AIONHIP_ROTARY_PLAIN && !positive(r->factor)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: factor must be positive and finite", who);
    if (r->scaling >= AIONHIP_ROTARY_BANDS && (!positive(r->original_length) || !positive(r->low) || !positive(r->high) || !(r->low < r->high)))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: original_length, low and high must be positive and finite, low below high", who);
    if (r->scaling == AIONHIP_ROTARY_RAMP && !(r->base > 1.f)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: a ramp needs a base above one", who);
    return AIONHIP_OK;
}

// each pair's fraction of a turn a position, 2^64 to the whole; one table per kind of turning, kept by the context as RoPE's are
int turn_table(aionhip_ctx *ctx, const aionhip_rotary *r, const unsigned long **out) {
    aionhip_rotary key{};
    key.dims = r->dims, key.scaling = r->scaling, key.base = r->base;
    if (r->scaling != AIONHIP_ROTARY_PLAIN) key.factor = r->factor;
    if (r->scaling >= AIONHIP_ROTARY_BANDS) key.original_length = r->original_length, key.low = r->low, key.high = r->high;
    for (const auto &t : ctx->turn_tables)
        if (std::memcmp(&t.key, &key, sizeof key) == 0) {
            *out = (const unsigned long *)t.turns;
            return AIONHIP_OK;
        }
    if (ctx->capturing)
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "a table of rotary turns cannot be built while a program is being recorded: run the steps once before recording");
    const long double two_pi = 6.283185307179586476925286766559L, base = r->base, dims = r->dims;
    std::vector<unsigned long> host(r->dims / 2);
    long double a = 0, b = 0;
    if (r->scaling == AIONHIP_ROTARY_RAMP) {
        auto at = [&](long double turns) { return dims * logl((long double)r->original_length / (turns * two_pi)) / (2 * logl(base)); };
        a = fmaxl(floorl(at(r->high)), 0);
        b = fminl(ceill(at(r->low)), dims - 1);
    }
    for (uint32_t i = 0; i < r->dims / 2; ++i) {
        long double f = powl(base, -2.0L * i / dims), kept = 1;
        if (r->scaling == AIONHIP_ROTARY_LINEAR) kept = 0;
        else if (r->scaling == AIONHIP_ROTARY_BANDS)
            kept = ((long double)r->original_length * f / two_pi - r->low) / ((long double)r->high - r->low);
        else if (r->scaling == AIONHIP_ROTARY_RAMP)
            kept = 1 - (i - a) / fmaxl(b - a, 0.001L);
        kept = fminl(fmaxl(kept, 0), 1);
        f *= kept + (1 - kept) / (r->scaling == AIONHIP_ROTARY_PLAIN ? 1.0L : (long double)r->factor);
        const long double turn = f / two_pi;
        host[i] = (unsigned long)ldexpl(turn - floorl(turn), 64);          // (a base below one may turn more than once a position: whole turns are none)
    }
    void *dev = nullptr;
    if (const int rc = dev_malloc(ctx, &dev, host.size() * sizeof(host[0]), "a table of rotary turns")) return rc;
    hipError_t e = hipMemcpyAsync(dev, host.data(), host.size() * sizeof(host[0]), hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        (void)hipFree(dev);
        return set_err(ctx, AIONHIP_EXECUTION_FAILED, "upload of a table of rotary turns: %s", hipGetErrorString(e));
    }
    ctx->turn_tables.push_back({key, dev});
    *out = (const unsigned long *)dev;
    return AIONHIP_OK;
}

// rows that take this many bytes, read and written, go past the caches (see the kernel)
constexpr size_t ONCE_BYTES = (size_t)128 << 20;

// the launch of `tokens` rows; `rotary` null or of no pairs: nothing turns
int launch_rotary(aionhip_ctx *ctx, const char *who, Rotate a, const aionhip_rotary *rotary, size_t tokens, int dtype, int cache_dtype) {
    if (rotary && rotary->dims) {
        a.dims = (int)rotary->dims;
        a.interleaved = rotary->interleaved ? 1 : 0;
        a.magnitude = rotary->magnitude;
    }
    const int each = pairs_each(dtype);
    a.turning = (a.dims / 2 + each - 1) / each;
    a.pieces = a.turning + (a.d - a.dims + 2 * each - 1) / (2 * each);
    const int slots = a.h_q + 2 * a.h_kv;
    const bool once = tokens * slots * a.d * (dtype == AIONHIP_F32 ? 8 : 4) >= ONCE_BYTES;
    // (f32 rows past the caches, 56 x 214 of 12 heads of 256, 196 elements turning: 61 us in pieces, 64 so)
    const bool whole = (a.interleaved ? a.dims % (2 * each) : a.dims / 2 % each) == 0 && (a.d - a.dims) % (2 * each) == 0;
    const bool by_rows = !whole && a.d % 8 == 0 && !(once && dtype == AIONHIP_F32);
    if (by_rows) a.pieces = a.d / 8;
    a.heads_wg = min(256 / a.pieces, slots);                             // (heads of up to 1024 have 129 pieces at most)
    // (measured at the kernel)
    const int heads = !by_rows && tokens >= 1024 && a.h_kv ? 4 : 1;
    const dim3 grid((unsigned)tokens, (unsigned)((slots + a.heads_wg * heads - 1) / (a.heads_wg * heads)));
    const unsigned threads = (unsigned)((a.heads_wg * a.pieces + 63) / 64 * 64);
    if (tokens > MAX_THREADS / threads) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: too many rows for one launch", who);
    if (a.dims) {
        if (const int rc = turn_table(ctx, rotary, &a.turns)) return rc;
    }
    ProfScope scope(ctx, who);
    auto go = [&](auto dt, auto ct) {
        constexpr int DT = decltype(dt)::value, CT = decltype(ct)::value;
        constexpr bool PAST = DT != AIONHIP_F32;
        if (by_rows) launch_k(ctx, once ? rotary_rows_kernel<DT, CT, PAST> : rotary_rows_kernel<DT, CT, false>, grid, dim3(threads), 0, a);
        else if (heads == 1) launch_k(ctx, once ? rotary_kernel<DT, CT, 1, true> : rotary_kernel<DT, CT, 1, false>, grid, dim3(threads), 0, a);
        else launch_k(ctx, once ? rotary_kernel<DT, CT, 4, true> : rotary_kernel<DT, CT, 4, false>, grid, dim3(threads), 0, a);
    };
    auto types = [&](auto dt) {
        if (cache_dtype == AIONHIP_F16) go(dt, std::integral_constant<int, AIONHIP_F16>{});
        else go(dt, std::integral_constant<int, AIONHIP_BF16>{});
    };
    if (dtype == AIONHIP_F32) types(std::integral_constant<int, AIONHIP_F32>{});
    else if (dtype == AIONHIP_F16) types(std::integral_constant<int, AIONHIP_F16>{});
    else types(std::integral_constant<int, AIONHIP_BF16>{});
    LAUNCH_CHECK(ctx, who);
    return AIONHIP_OK;
}

int append(aionhip_ctx *ctx, const char *who, const aionhip_paged_cache *c, const aionhip_rotary *rotary, aionhip_handle q_out, aionhip_handle q, aionhip_handle k, aionhip_handle v,
           int dtype, aionhip_handle positions, aionhip_handle write_index, size_t s, size_t h_q) {
    int rc = check_cache(ctx, who, c);
    if (rc) return rc;
    if (!k || !v || !write_index) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: null operand", who);
    if (!row_type(dtype)) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: rows are f32, f16 or bf16, not dtype %d", who, dtype);
    if (s > capacity(c)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: %zu rows exceed the capacity %zu", who, s, capacity(c));
    if (h_q > 65535) return set_err(ctx, AIONHIP_UNSUPPORTED, "%s: dimension too large", who);
    if (!c->batch || !s) return AIONHIP_OK;
    const size_t tokens = c->batch * s, q_bytes = tokens * h_q * c->d * size_of(dtype), kv_bytes = tokens * c->h_kv * c->d * size_of(dtype);
    if (in_cache(c, q, q_bytes) || in_cache(c, q_out, q_bytes) || in_cache(c, k, kv_bytes) || in_cache(c, v, kv_bytes) || in_cache(c, positions, tokens * 4) ||
        in_cache(c, write_index, c->batch * 4))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: rows or indices lie in the cache", who);
    if ((q_out != q && overlap(q_out, q_bytes, q, q_bytes)) || overlap(q_out, q_bytes, k, kv_bytes) || overlap(q_out, q_bytes, v, kv_bytes) ||
        overlap(q_out, q_bytes, positions, tokens * 4) || overlap(q_out, q_bytes, write_index, c->batch * 4))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "%s: q, k, v and the indices are still read while q_out is written", who);
    Rotate a{};
    a.q_out = dp<void>(q_out), a.q = dp<const void>(q), a.k = dp<const void>(k), a.v = dp<const void>(v);
    a.positions = dp<const int>(positions), a.write_index = dp<const int>(write_index);
    a.d = (int)c->d, a.h_q = (int)h_q, a.h_kv = (int)c->h_kv, a.s_len = (int)s;
    a.table = table_of(c);
    a.k_pages = dp<unsigned char>(c->k_pages), a.v_pages = dp<unsigned char>(c->v_pages);
    return launch_rotary(ctx, who, a, rotary, tokens, dtype, c->dtype);
}

}  // namespace

extern "C" {

int aionhip_step_rotary(aionhip_ctx *ctx, aionhip_handle out, aionhip_handle x, aionhip_handle positions, int dtype, size_t b, size_t t, size_t h, size_t d,
                        const aionhip_rotary *rotary) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (!out || !x || !positions) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rotary: null operand");
    if (!row_type(dtype)) return set_err(ctx, AIONHIP_UNSUPPORTED, "rotary: rows are f32, f16 or bf16, not dtype %d", dtype);
    if (const int rc = check_rotary(ctx, "rotary", rotary, d)) return rc;
    if (d > MAX_HEAD || h > 65535 || b > 0x7FFFFFFF || t > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "rotary: dimension too large");
    if (!b || !t || !h || !d) return AIONHIP_OK;
    if (b > 0x7FFFFFFF / t) return set_err(ctx, AIONHIP_UNSUPPORTED, "rotary: too many rows for one launch");
    const size_t bytes = b * t * h * d * size_of(dtype);
    if ((out != x && overlap(out, bytes, x, bytes)) || overlap(out, bytes, positions, b * t * 4))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rotary: x and the positions are still read while out is written");
    Rotate a{};
    a.q_out = dp<void>(out), a.q = dp<const void>(x), a.positions = dp<const int>(positions);
    a.d = (int)d, a.h_q = (int)h;
    return launch_rotary(ctx, "rotary", a, rotary, b * t, dtype, AIONHIP_F16);
}

int aionhip_step_append_paged(aionhip_ctx *ctx, const aionhip_paged_cache *cache, aionhip_handle k, aionhip_handle v, int src_dtype, aionhip_handle write_index, size_t s) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    return append(ctx, "append_paged", cache, nullptr, 0, 0, k, v, src_dtype, 0, write_index, s, 0);
}

int aionhip_step_rotary_append_paged(aionhip_ctx *ctx, const aionhip_paged_cache *cache, const aionhip_rotary *rotary, aionhip_handle q_out, aionhip_handle q,
                                     aionhip_handle k, aionhip_handle v, int dtype, aionhip_handle positions, aionhip_handle write_index, size_t s, size_t h_q) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (!q_out || !q || !positions) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "rotary_append_paged: null operand");
    if (const int rc = check_cache(ctx, "rotary_append_paged", cache)) return rc;
    if (const int rc = check_rotary(ctx, "rotary_append_paged", rotary, cache->d)) return rc;
    return append(ctx, "rotary_append_paged", cache, rotary, q_out, q, k, v, dtype, positions, write_index, s, h_q);
}

int aionhip_step_read_paged(aionhip_ctx *ctx, const aionhip_paged_cache *c, aionhip_handle k_out, aionhip_handle v_out, int out_dtype, aionhip_handle first, size_t s) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (const int rc = check_cache(ctx, "read_paged", c)) return rc;
    if (!k_out || !v_out || !first) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "read_paged: null operand");
    if (!row_type(out_dtype)) return set_err(ctx, AIONHIP_UNSUPPORTED, "read_paged: rows are f32, f16 or bf16, not dtype %d", out_dtype);
    if (s > capacity(c)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "read_paged: %zu rows exceed the capacity %zu", s, capacity(c));
    if (!c->batch || !s) return AIONHIP_OK;
    const size_t rows = c->batch * s * c->h_kv, bytes = rows * c->d * size_of(out_dtype), total = rows * (c->d / 8);
    if (overlap(k_out, bytes, v_out, bytes) || overlap(k_out, bytes, first, c->batch * 4) || overlap(v_out, bytes, first, c->batch * 4))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "read_paged: the rows of keys and values overlap each other or the indices");
    if (in_cache(c, k_out, bytes) || in_cache(c, v_out, bytes)) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "read_paged: rows lie in the cache");
    if (total > MAX_THREADS - 255) return set_err(ctx, AIONHIP_UNSUPPORTED, "read_paged: too many rows for one launch");
    const ReadArgs a{{dp<const unsigned char>(c->k_pages), dp<const unsigned char>(c->v_pages)}, {dp<void>(k_out), dp<void>(v_out)}, dp<const int>(first), table_of(c), (int)s, (int)c->h_kv,
                     (int)c->d};
    const bool f16 = c->dtype == AIONHIP_F16;
    const auto kernel = out_dtype == AIONHIP_F32   ? (f16 ? read_paged_kernel<AIONHIP_F16, AIONHIP_F32> : read_paged_kernel<AIONHIP_BF16, AIONHIP_F32>)
                        : out_dtype == AIONHIP_F16 ? (f16 ? read_paged_kernel<AIONHIP_F16, AIONHIP_F16> : read_paged_kernel<AIONHIP_BF16, AIONHIP_F16>)
                                                   : (f16 ? read_paged_kernel<AIONHIP_F16, AIONHIP_BF16> : read_paged_kernel<AIONHIP_BF16, AIONHIP_BF16>);
    ProfScope scope(ctx, "read_paged");
    launch_k(ctx, kernel, dim3((unsigned)((total + 255) / 256), 2), dim3(256), 0, a, total);
    LAUNCH_CHECK(ctx, "read_paged");
    return AIONHIP_OK;
}

}  // extern "C"
