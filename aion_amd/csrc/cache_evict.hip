// Eviction from caches in pages by accumulated attention weight: which rows stay, and the move of those (the layout: cache_paged.h). Two launches: a workgroup a
// sequence and head finds its rows (select_kernel), then their keys and values move (move_kernel).
#include "cache_paged.h"

#include <type_traits>

namespace {
using namespace paged;

template <typename T> T *dp(aionhip_handle h) { return reinterpret_cast<T *>((uintptr_t)h); }

// a weight's place in the order that the greatest is taken from, as a number: a NaN above all, -0 as 0
__device__ __forceinline__ unsigned rank_of(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const unsigned u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Select {
    const float *weights;
    const int *lengths;
    float *weights_out;
    int *kept, *counts;
    int h, cap, cap_out, limit, keep, first, recent;
    int in_place, tell;           // tell: what an uncut sequence keeps is asked for, or copied
};
constexpr int SELECT_THREADS = 1024, DIGIT = 256;

// sums of v over the threads before this one, and over all of them; red: 17 ints of LDS
__device__ __forceinline__ int scan_1024(int v, int *red, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o, 64);
        if (lane >= o) sum += up;
    }
    __syncthreads();
    if (lane == 63) red[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < SELECT_THREADS / 64; ++w) {
        const int x = red[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return before + sum - v;
}

// The m-th greatest rank of a head's middle rows by four rounds over its digits, greatest digit first, then one pass that numbers what stays.
__global__ __launch_bounds__(SELECT_THREADS) void select_kernel(Select a) {
    __shared__ int hist[DIGIT], red[SELECT_THREADS / 64], s_digit, s_above;
    const int b = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
    const size_t unit = (size_t)b * a.h + head;
    const int n = max(0, min(a.lengths[b], a.cap));
    const bool cut = n > a.limit;
    const int count = cut ? a.keep : n;
    if (head == 0 && tid == 0) a.counts[b] = cut || !a.in_place ? count : -1;
    const float *w = a.weights + unit * a.cap;
    float *out = a.weights_out + unit * a.cap_out;
    int *kept = a.kept + unit * a.limit;
    if (!cut) {
        if (a.tell)
            for (int i = tid; i < a.limit; i += SELECT_THREADS) kept[i] = i < n ? i : -1;
        if (out != w)                             // (in place an uncut sequence costs nothing but the look at its length)
            for (int i = tid; i < a.cap_out; i += SELECT_THREADS) out[i] = i < n ? w[i] : 0.f;
        return;
    }
    const int lo = a.first, hi = n - a.recent;
    int want = a.keep - a.first - a.recent;
    unsigned prefix = 0;
    bool none = want == 0;
    if (!none) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < DIGIT) hist[tid] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += SELECT_THREADS) {
                const unsigned r = rank_of(w[i]);
                if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[r >> shift & 255u], 1);
            }
            __syncthreads();
            if (tid < 64) {                       // one wavefront: four digits a lane, counted from the top
                int c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = hist[255 - (tid * 4 + j)], sum += c[j];
                int upto = sum;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int up = __shfl_up(upto, o, 64);
                    if (tid >= o) upto += up;
                }
                int above = upto - sum;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (above < want && above + c[j] >= want) s_digit = 255 - (tid * 4 + j), s_above = above;
                    above += c[j];
                }
            }
            __syncthreads();
            prefix |= (unsigned)s_digit << shift;
            want -= s_above;
            __syncthreads();
        }
    }
    // `want` of the rows whose rank is `prefix` stay, the oldest of them. Chunks in order: what is read of a chunk lies behind everything written so far, so that weights may move in place.
    int at = 0, equal = 0;
    for (int base = 0; base < n; base += SELECT_THREADS) {
        const int i = base + tid;
        const float x = i < n ? w[i] : 0.f;
        const bool middle = i >= lo && i < hi;
        const unsigned r = rank_of(x);
        const bool same = middle && !none && r == prefix;
        int total;
        const int eq = equal + scan_1024(same ? 1 : 0, red, total);
        equal += total;
        const bool stays = i < n && (!middle || (!none && (r > prefix || (same && eq < want))));
        const int to = at + scan_1024(stays ? 1 : 0, red, total);
        at += total;
        if (stays) {
            kept[to] = i;
            out[to] = x;
        }
    }
    __syncthreads();
    for (int i = a.keep + tid; i < a.limit; i += SELECT_THREADS) kept[i] = -1;
    for (int i = a.keep + tid; i < a.cap_out; i += SELECT_THREADS) out[i] = 0.f;
}

struct Move {
    unsigned char *pages[2];
    const int *kept, *counts;
    int *lengths_out;
    const int *lengths;
    Table from, to;
    int h, d, limit, cap;
    int lanes;                    // 16-byte columns of a row that a workgroup moves
    int slices, parts;            // workgroups over the columns, over the rows
};
// Rows in their order, so many at a time that every thread has EACH 16-byte pieces in flight. In place a workgroup moves all rows of its columns: a
// chunk is read before it is written, its rows come from at or behind where they go, and the next chunk's from behind that.
constexpr int MOVE_EACH = 4;
__global__ __launch_bounds__(256) void move_kernel(Move a) {
    const int b = blockIdx.z, head = blockIdx.y % a.h, which = blockIdx.y / a.h;
    const int slice = blockIdx.x % a.slices, part = blockIdx.x / a.slices;
    const int count = a.counts[b];
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.lengths_out[b] = count >= 0 ? count : max(0, min(a.lengths[b], a.cap));
    if (count <= 0) return;
    const int rows = 256 / a.lanes, row = threadIdx.x / a.lanes, col = slice * a.lanes + threadIdx.x % a.lanes;
    const bool live = row < rows && col < a.d / 8;
    const int chunk = rows * MOVE_EACH;
    const int chunks = (count + chunk - 1) / chunk, per = (chunks + a.parts - 1) / a.parts;
    const int *kept = a.kept + ((size_t)b * a.h + head) * a.limit;
    unsigned char *pages = a.pages[which];
    const int mask = (1 << a.from.shift) - 1;
    for (int c = part * per; c < min((part + 1) * per, chunks); ++c) {
        u32x4 x[MOVE_EACH];
        int target[MOVE_EACH];
#pragma unroll
        for (int j = 0; j < MOVE_EACH; ++j) {
            const int to = c * chunk + j * rows + row;
            target[j] = -1;
            if (live && to < count) {
                const int from = kept[to], source = page_of(a.from, b, from);
                if (source >= 0) {
                    target[j] = page_of(a.to, b, to);
                    x[j] = *(const u32x4 *)(pages + (((((size_t)source * a.h + head) << a.from.shift) + (from & mask)) * a.d + col * 8) * 2);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int j = 0; j < MOVE_EACH; ++j) {
            const int to = c * chunk + j * rows + row;
            if (target[j] >= 0) *(u32x4 *)(pages + (((((size_t)target[j] * a.h + head) << a.from.shift) + (to & mask)) * a.d + col * 8) * 2) = x[j];
        }
        __syncthreads();
    }
}

}  // namespace

extern "C" int aionhip_step_evict_paged(aionhip_ctx *ctx, const aionhip_paged_cache *c, const aionhip_eviction *e) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (const int rc = check_cache(ctx, "evict_paged", c)) return rc;
    if (!e || !e->weights || !e->kv_lengths || !e->weights_out || !e->lengths_out) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "evict_paged: null operand");
    const size_t cap = capacity(c);
    if (e->limit > MAX_ROWS || e->keep > e->limit || e->first > e->keep || e->recent > e->keep - e->first)
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "evict_paged: first %zu + recent %zu <= keep %zu <= limit %zu must hold", e->first, e->recent, e->keep, e->limit);
    if (!e->table_out && e->width_out) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "evict_paged: a width without a table");
    if (e->table_out && (e->table_out == c->page_table || e->width_out > MAX_ROWS / c->page_rows || e->width_out * c->page_rows < e->limit))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "evict_paged: table_out is the cache's own, or %zu entries of %zu rows do not hold %zu", e->width_out, c->page_rows, e->limit);
    if (!c->batch) return AIONHIP_OK;
    const size_t cap_out = e->table_out ? e->width_out * c->page_rows : cap, units = c->batch * c->h_kv;
    const size_t limit = min(e->limit, cap), kept_bytes = units * e->limit * 4;
    if (units > 0x7FFFFFFF || 2 * c->h_kv > 65535) return set_err(ctx, AIONHIP_UNSUPPORTED, "evict_paged: dimension too large");
    const size_t w_bytes = units * cap * 4, wo_bytes = units * cap_out * 4, l_bytes = c->batch * 4, t_bytes = c->batch * e->width_out * 4;
    const bool same_w = e->weights_out == e->weights, same_l = e->lengths_out == e->kv_lengths;
    if ((same_w && e->table_out) || (!same_w && overlap(e->weights_out, wo_bytes, e->weights, w_bytes)) || (!same_l && overlap(e->lengths_out, l_bytes, e->kv_lengths, l_bytes)) ||
        overlap(e->weights_out, wo_bytes, e->lengths_out, l_bytes) || overlap(e->weights_out, wo_bytes, e->kv_lengths, l_bytes) ||
        overlap(e->weights, w_bytes, e->lengths_out, l_bytes) || overlap(e->kept, kept_bytes, e->weights, w_bytes) || overlap(e->kept, kept_bytes, e->weights_out, wo_bytes) ||
        overlap(e->kept, kept_bytes, e->kv_lengths, l_bytes) || overlap(e->kept, kept_bytes, e->lengths_out, l_bytes) || in_cache(c, e->weights_out, wo_bytes) ||
        in_cache(c, e->lengths_out, l_bytes) || in_cache(c, e->kept, kept_bytes) || overlap(e->table_out, t_bytes, e->weights_out, wo_bytes) ||
        overlap(e->table_out, t_bytes, e->lengths_out, l_bytes) || overlap(e->table_out, t_bytes, e->kept, kept_bytes) || overlap(e->table_out, t_bytes, c->k_pages, pool_bytes(c)) ||
        overlap(e->table_out, t_bytes, c->v_pages, pool_bytes(c)) || in_cache(c, e->weights, w_bytes) || in_cache(c, e->kv_lengths, l_bytes))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "evict_paged: an operand that is written overlaps another");
    if (const int rc = ensure_scratch2(ctx, (c->batch * 4 + 255) / 256 * 256 + (e->kept ? 0 : kept_bytes))) return rc;
    int *counts = (int *)ctx->scratch2, *kept = e->kept ? dp<int>(e->kept) : counts + (c->batch + 63) / 64 * 64;
    const Select s{dp<const float>(e->weights), dp<const int>(e->kv_lengths), dp<float>(e->weights_out), kept, counts, (int)c->h_kv, (int)cap, (int)cap_out, (int)e->limit, (int)e->keep,
                   (int)e->first, (int)e->recent, e->table_out ? 0 : 1, e->table_out || e->kept ? 1 : 0};
    {
        ProfScope scope(ctx, "evict_select");
        launch_k(ctx, select_kernel, dim3((unsigned)c->h_kv, (unsigned)c->batch), dim3(SELECT_THREADS), 0, s);
        LAUNCH_CHECK(ctx, "evict_select");
    }
    Move m{{dp<unsigned char>(c->k_pages), dp<unsigned char>(c->v_pages)}, kept, counts, dp<int>(e->lengths_out), dp<const int>(e->kv_lengths), table_of(c), table_of(c), (int)c->h_kv, (int)c->d,
           (int)e->limit, (int)cap, 0, 0, 0};
    const int cols = (int)(c->d / 8);
    if (e->table_out) {
        m.to.pages = dp<const int>(e->table_out);
        m.to.width = (int)e->width_out;
        m.lanes = min(cols, 256);
        m.slices = 1;
        const int chunk = 256 / m.lanes * MOVE_EACH;
        m.parts = (int)max((size_t)1, min((limit + chunk - 1) / chunk, (size_t)65536));
    } else {
        m.lanes = min(cols, 4);
        m.slices = (cols + m.lanes - 1) / m.lanes;
        m.parts = 1;
    }
    ProfScope scope(ctx, "evict_move");
    launch_k(ctx, move_kernel, dim3((unsigned)(m.slices * m.parts), (unsigned)(2 * c->h_kv), (unsigned)c->batch), dim3(256), 0, m);
    LAUNCH_CHECK(ctx, "evict_move");
    return AIONHIP_OK;
}
