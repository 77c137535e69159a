// Eviction from caches in pages by accumulated attention weight: which rows stay, and the move of those (the layout: cache_paged.h). Two launches: a workgroup a
// sequence and head finds its rows (select_kernel), then their keys and values move (move_kernel).
#include "cache_paged.h"

#include <type_traits>

namespace {
using namespace paged;

template <typename T> T *dp(aionhip_handle h) { return reinterpret_cast<T *>((uintptr_t)h); }

// a weight's place in the order that the greatest is taken from, as a number: a NaN above all, -0 as 0
__device__ __forceinline__ unsigned rank_of(float w) {
    const unsigned u = __float_as_uint(w + 0.f);
    const unsigned r = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
    return w != w ? 0xFFFFFFFFu : r;
}

struct Select {
    const float *weights;
    const int *lengths;
    float *weights_out;
    int *kept, *counts;
    int h, cap, cap_out, limit, keep, first, recent;
    int in_place, tell;           // tell: what an uncut sequence keeps is asked for, or copied
};
constexpr int SELECT_EACH = 8;        // neighbouring rows of a thread in a chunk
constexpr int HELD = 4;               // chunks of weights that a workgroup keeps in registers; longer sequences read the others again in every round
constexpr int DIGITS = 2048;

// sum over the lanes up to this one: shifts within rows of sixteen, then the last of a row (of half a wavefront) added to the rows behind it
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);      // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);      // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);      // row_bcast 31 into rows 2 and 3
    return v;
}
// sums of v over the threads before this one, and over all of them; red: an int of LDS to each wavefront
template <int THREADS>
__device__ __forceinline__ int scan_all(int v, int *red, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = wave_scan(v);
    __syncthreads();
    if (lane == 63) red[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        const int x = red[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return before + sum - v;
}

// The m-th greatest rank of a head's middle rows by three rounds over its digits (11, 11 and 10 bits, greatest first), each of which counts the digits of what the rounds
// before left; then one pass that numbers what stays. A thread has eight neighbouring rows of a chunk, so that the places of what stays are one sum over the
// workgroup to a chunk; a digit's count has copies, as sums of probabilities share their exponents. What bounds it is one CU's instruction issue (long sequences: of 23 us for
// 32768 rows 6 are the first round, 9 the last pass) and the barriers (short ones: 7 us for 1280 rows). Tried and not kept: what stays gathered in LDS and written side by side
// (25.5), ranks instead of weights in registers (the same), 64 neighbouring rows to a wavefront, with masks and counts of bits in place of sums (30).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void select_kernel(Select a) {
    constexpr unsigned CHUNK = THREADS * SELECT_EACH;
    constexpr int COPIES = THREADS / 256, OWN = DIGITS / THREADS;
    __shared__ int hist[DIGITS * COPIES], red[THREADS / 64], s_digit, s_above;
    const int b = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
    const size_t unit = (size_t)b * a.h + head;
    // (steps are unsigned: a capacity goes up to 2^31 - 64, and the places after a chunk, or a thread's last row, past 2^31)
    const unsigned n = (unsigned)max(0, min(a.lengths[b], a.cap)), limit = (unsigned)a.limit, cap_out = (unsigned)a.cap_out;
    const bool cut = n > limit;
    const int count = cut ? a.keep : (int)n;
    if (head == 0 && tid == 0) a.counts[b] = cut || !a.in_place ? count : -1;
    const float *w = a.weights + unit * a.cap;
    float *out = a.weights_out + unit * a.cap_out;
    int *kept = a.kept + unit * a.limit;
    if (!cut) {
        if (a.tell)
            for (unsigned i = tid; i < limit; i += THREADS) kept[i] = i < n ? (int)i : -1;
        if (out != w)                             // (in place an uncut sequence costs nothing but the look at its length)
            for (unsigned i = tid; i < cap_out; i += THREADS) out[i] = i < n ? w[i] : 0.f;
        return;
    }
    const unsigned lo = (unsigned)a.first, hi = n - (unsigned)a.recent;
    auto load = [&](unsigned chunk, float (&x)[SELECT_EACH]) __attribute__((always_inline)) {
        const unsigned i = chunk * CHUNK + (unsigned)tid * SELECT_EACH;
        if (i + SELECT_EACH <= n) {
            __builtin_memcpy(x, w + i, sizeof x);
        } else {
#pragma unroll
            for (int j = 0; j < SELECT_EACH; ++j) x[j] = i + j < n ? w[i + j] : 0.f;
        }
    };
    float held[HELD][SELECT_EACH];
#pragma unroll
    for (unsigned c = 0; c < HELD; ++c)
        if (c * CHUNK < n) load(c, held[c]);
    int want = a.keep - a.first - a.recent;
    unsigned prefix = 0;
    const bool none = want == 0;
    if (!none) {
#pragma unroll 1
        for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift - 10) {
            const int bits = shift == 0 ? 10 : 11;
            for (int i = tid; i < DIGITS * COPIES; i += THREADS) hist[i] = 0;
            __syncthreads();
            auto add = [&](unsigned chunk, const float (&x)[SELECT_EACH]) __attribute__((always_inline)) {
                const unsigned i = chunk * CHUNK + (unsigned)tid * SELECT_EACH;
#pragma unroll
                for (int j = 0; j < SELECT_EACH; ++j) {
                    const unsigned r = rank_of(x[j]);
                    if (i + j >= lo && i + j < hi && (shift == 21 || r >> (shift + bits) == prefix >> (shift + bits)))
                        atomicAdd(&hist[(r >> shift & (DIGITS - 1u) >> (11 - bits)) * COPIES + (tid & (COPIES - 1))], 1);
                }
            };
#pragma unroll
            for (unsigned c = 0; c < HELD; ++c)
                if (c * CHUNK < n) add(c, held[c]);
            for (unsigned c = HELD; c * CHUNK < n; ++c) {
                float x[SELECT_EACH];
                load(c, x);
                add(c, x);
            }
            __syncthreads();
            int c[OWN], sum = 0, all;             // a thread's digits, counted from the top
#pragma unroll
            for (int j = 0; j < OWN; ++j) {
                c[j] = 0;
#pragma unroll
                for (int k = 0; k < COPIES; ++k) c[j] += hist[(DIGITS - 1 - OWN * tid - j) * COPIES + k];
                sum += c[j];
            }
            int above = scan_all<THREADS>(sum, red, all);
#pragma unroll
            for (int j = 0; j < OWN; ++j) {
                if (above < want && above + c[j] >= want) s_digit = DIGITS - 1 - OWN * tid - j, s_above = above;
                above += c[j];
            }
            __syncthreads();
            prefix |= (unsigned)s_digit << shift;
            want -= s_above;
        }
    }
    // `want` of the rows whose rank is `prefix` stay, the oldest of them. Chunks in order: what is read of a chunk lies behind everything written so far, and its ranks have been
    // taken when the workgroup meets, so that weights may move in place.
    int sure = 0, equal = 0;                      // rows before the chunk that stay whatever `want` is, and of that rank
    auto place = [&](unsigned chunk, const float (&x)[SELECT_EACH]) __attribute__((always_inline)) {
        const unsigned i = chunk * CHUNK + (unsigned)tid * SELECT_EACH;
        unsigned stays = 0, same = 0;
#pragma unroll
        for (int j = 0; j < SELECT_EACH; ++j) {
            const unsigned r = rank_of(x[j]);
            const bool middle = i + j >= lo && i + j < hi;
            stays |= (i + j < n && (!middle || (!none && r > prefix)) ? 1u : 0u) << j;
            same |= (middle && !none && r == prefix ? 1u : 0u) << j;
        }
        int total;
        const int before = scan_all<THREADS>(__popc(stays) | __popc(same) << 16, red, total);
        int s = sure + (before & 0xFFFF), e = equal + (int)((unsigned)before >> 16);
#pragma unroll
        for (int j = 0; j < SELECT_EACH; ++j) {
            const bool mine = stays >> j & 1u, alike = same >> j & 1u;
            if (mine || (alike && e < want)) {
                const int to = s + min(e, want);
                kept[to] = (int)(i + j);
                out[to] = x[j];
            }
            s += mine ? 1 : 0;
            e += alike ? 1 : 0;
        }
        sure += total & 0xFFFF;
        equal += (int)((unsigned)total >> 16);
    };
#pragma unroll
    for (unsigned c = 0; c < HELD; ++c)
        if (c * CHUNK < n) place(c, held[c]);
    for (unsigned c = HELD; c * CHUNK < n; ++c) {
        float x[SELECT_EACH];
        load(c, x);
        place(c, x);
    }
    __syncthreads();
    for (unsigned i = (unsigned)(a.keep + tid); i < limit; i += THREADS) kept[i] = -1;
    for (unsigned i = (unsigned)(a.keep + tid); i < cap_out; i += THREADS) out[i] = 0.f;
}

struct Move {
    unsigned char *pages[2], *held;
    const int *kept, *counts;
    int *lengths_out;
    const int *lengths;
    Table from, to;
    int h, d, limit, cap, keep;
    int first_unit;               // of the sequences' heads that this launch moves
    int lanes, parts;             // 16-byte columns of a row; workgroups over the rows
};
// The rows that stay, keys and values together, a 16-byte piece of each to a thread. TO_PAGES: to pages of their own. In place the rows go through memory outside the cache (HOLD,
// then BACK), as one that moves may lie where another goes to; those in front of the first that leaves do not move. 4 sequences of 32768 rows of 8 heads of 128 cut to 8192:
// 53.2 us to pages of their own, 5.0 TB/s of rows of 256 bytes picked from four times as many. In place 106 with the choice of the rows (24, then 42 and 40), and one of 4352 cut to
// 4096 27 (193 and 86 by workgroups that moved all rows of a few columns in order).
enum { TO_PAGES, HOLD, BACK };
template <int MODE>
__global__ __launch_bounds__(256) void move_kernel(Move a) {
    const int unit = a.first_unit + (int)blockIdx.y, b = unit / a.h, head = unit - b * a.h;
    const int count = a.counts[b];
    if (MODE != HOLD && blockIdx.x == 0 && head == 0 && threadIdx.x == 0) a.lengths_out[b] = count >= 0 ? count : max(0, min(a.lengths[b], a.cap));
    const int rows = 256 / a.lanes, row = threadIdx.x / a.lanes, col = threadIdx.x - row * a.lanes;
    if (row >= rows) return;
    const int *kept = a.kept + (size_t)unit * a.limit;
    const int mask = (1 << a.from.shift) - 1;
    const unsigned places = (unsigned)max(count, 0), stride = (unsigned)(a.parts * rows);         // (unsigned: a stride behind the last place may pass 2^31)
    for (unsigned place = blockIdx.x * (unsigned)rows + row; place < places; place += stride) {
        const int to = (int)place, from = kept[to];
        if (MODE != TO_PAGES && from == to) continue;
        const int source = page_of(a.from, b, from), target = MODE == HOLD ? 0 : page_of(a.to, b, to);
        if (source < 0 || target < 0) continue;
        const size_t source_at = (((((size_t)source * a.h + head) << a.from.shift) + (from & mask)) * a.d + col * 8) * 2;
        const size_t target_at = (((((size_t)target * a.h + head) << a.from.shift) + (to & mask)) * a.d + col * 8) * 2;
        const size_t held_at = (((size_t)blockIdx.y * 2 * a.keep + to) * a.d + col * 8) * 2, held_next = (size_t)a.keep * a.d * 2;
        u32x4 x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (MODE == BACK) x[i] = *(const u32x4 *)(a.held + held_at + i * held_next);
            else x[i] = __builtin_nontemporal_load((const u32x4 *)(a.pages[i] + source_at));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (MODE == HOLD) *(u32x4 *)(a.held + held_at + i * held_next) = x[i];
            else __builtin_nontemporal_store(x[i], (u32x4 *)(a.pages[i] + target_at));
        }
    }
}
constexpr size_t MOVE_WORKGROUPS = 32768, HELD_BYTES = (size_t)256 << 20;      // of one launch; of memory that rows go through at a time (a head's rows at least)

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
    // (a limit that no sequence passes may be any number: the list of what stays, and the memory between, are of the rows there can be)
    const size_t limit = min(e->limit, cap), keep = min(e->keep, limit), kept_bytes = units * e->limit * 4, listed = e->kept ? e->limit : limit;
    if (units > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "evict_paged: dimension too large");
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
    const size_t row_bytes = c->d * 4, counts_bytes = (c->batch * 4 + 255) / 256 * 256, list_bytes = e->kept ? 0 : (units * listed * 4 + 255) / 256 * 256;
    // in place: as many heads of sequences at once as the memory between takes
    const size_t group = e->table_out || !keep ? units : min(units, max((size_t)1, HELD_BYTES / (keep * row_bytes)));
    if (const int rc = ensure_scratch2(ctx, counts_bytes + list_bytes + (e->table_out ? 0 : group * keep * row_bytes))) return rc;
    int *counts = (int *)ctx->scratch2, *kept = e->kept ? dp<int>(e->kept) : (int *)((char *)ctx->scratch2 + counts_bytes);
    const Select s{dp<const float>(e->weights), dp<const int>(e->kv_lengths), dp<float>(e->weights_out), kept, counts, (int)c->h_kv, (int)cap, (int)cap_out, (int)listed, (int)keep,
                   (int)e->first, (int)e->recent, e->table_out ? 0 : 1, e->table_out || e->kept ? 1 : 0};
    {
        ProfScope scope(ctx, "evict_select");
        // (what a short sequence costs is the barriers between the rounds, and those the wavefronts that meet there)
        if (cap <= 8192) launch_k(ctx, select_kernel<256>, dim3((unsigned)c->h_kv, (unsigned)c->batch), dim3(256), 0, s);
        else launch_k(ctx, select_kernel<1024>, dim3((unsigned)c->h_kv, (unsigned)c->batch), dim3(1024), 0, s);
        LAUNCH_CHECK(ctx, "evict_select");
    }
    Move m{{dp<unsigned char>(c->k_pages), dp<unsigned char>(c->v_pages)}, (unsigned char *)ctx->scratch2 + counts_bytes + list_bytes, kept, counts, dp<int>(e->lengths_out),
           dp<const int>(e->kv_lengths), table_of(c), table_of(c), (int)c->h_kv, (int)c->d, (int)listed, (int)cap, (int)keep, 0, (int)(c->d / 8), 0};
    ProfScope scope(ctx, "evict_move");
    if (e->table_out) {
        m.to.pages = dp<const int>(e->table_out);
        m.to.width = (int)e->width_out;
    }
    const size_t rows = 256 / m.lanes, most = e->table_out ? limit : keep;
    for (size_t u = 0; u < units; u += 65535 < group ? 65535 : group) {
        const size_t n = min(units - u, min(group, (size_t)65535));
        m.first_unit = (int)u;
        m.parts = (int)max((size_t)1, min((most + rows - 1) / rows, MOVE_WORKGROUPS / n));      // (a limit far above the lengths would be workgroups that find nothing)
        const dim3 grid((unsigned)m.parts, (unsigned)n);
        if (e->table_out) {
            launch_k(ctx, move_kernel<TO_PAGES>, grid, dim3(256), 0, m);
        } else {
            launch_k(ctx, move_kernel<HOLD>, grid, dim3(256), 0, m);
            launch_k(ctx, move_kernel<BACK>, grid, dim3(256), 0, m);
        }
    }
    LAUNCH_CHECK(ctx, "evict_move");
    return AIONHIP_OK;
}
