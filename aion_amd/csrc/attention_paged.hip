// Attention over caches in pages (the layout: cache_paged.h): one to a few tokens a sequence, f32 accuracy, and with it what each key's probabilities add up to.
//
// paged_attn_kernel - head sizes 64, 128, 256. A workgroup has sixteen query rows of one KV head (position-major, query head fastest), one segment of their keys and, in small
//   calls, a share of the value columns; its wavefronts take tiles of 32 keys in turn:
//       S^T[keys x rows] = K[keys x d] . Q^T[d x rows]          O^T[d x rows] += V^T[d x keys] . P^T[keys x rows]
//   K goes from the pages to registers in the order the matrix instruction wants it, V through LDS, where it is read transposed. Sixteen keys lie in one page, so a
//   page number is a scalar to each half tile: a lane fetches one of the next 64, and they become addresses without a load in between.
//   Accuracy: q and P enter the products as sums of halves (two f16, three bf16; q that comes in the cache's type as it is), K and V are exact, sums are f32.
//   The workgroup that ends last adds the segments of its rows and, where the capacity is small, what the keys draw.
//   What bounds it, us: large calls HBM (one token over 131072 keys, 8 heads of 128 for 32, 90, 6.0 TB/s; 32 sequences of up to 16384 252, 6.3 TB/s, the last tenth of it
//   the unevenness of the sequences); small ones a chain of latencies (531 keys, one head of 256 for 8, 7.5: launch 4, length and page, keys and values, products, one
//   exchange between the segments). Five queries, 4 sequences over 3001 keys, 32 heads of 128: 35, 4.6 TB/s.
// paged_weights_kernel - what the keys draw elsewhere, from the scores that the first kernel left.
// paged_generic_kernel - other head sizes: a wavefront a key at a time, f32. It is there so that every shape has a path.
#include "attention_common.h"
#include "cache_paged.h"

#include <cstddef>
#include <type_traits>

namespace {
using namespace attn;
using paged::Table;

constexpr float MASKED = -INFINITY;
// Probabilities are held as 2^(s - ref + head_room), over f16 2^15 at most, which fits f16; a pair of f16 rounds to 2^-22 of itself or 2^-25, whichever is more. So the reference goes by the tile: it is
// raised when the tile's largest score passes it by more than SLACK, and over f16 values lowered when that lies more than DROP below it, by up to DEPTH below the largest score of all.
// What a key loses is then 2^-31 of the largest probability of its own tile of 32, and an answer 2^-26 of the largest value, however many keys there are. (A reference that only rises loses
// as much of the row's largest with every key: of a hundred thousand keys 22 nats below one whose value is zero nothing was left.) DEPTH keeps the sums, 2^31 keys of 65504 times
// 2^(15 + 64) at most, and the factors between segments in f32. A reference is a whole number, so that sums come from one to another without a rounding (a thousand of which, where tiles
// lie far apart in turn, were 2e-6). Three bf16 need no lowering, and no room above: below one
// the sums have room for values that bf16 has and f16 has not, up to 2^100 whatever their number (with the room that f16 takes, values were infinite from 2^112 on).
constexpr float SLACK = 5.f, DROP = 3.f, DEPTH = 64.f, LOW = -16.f;
__host__ __device__ constexpr float head_room(int kv) { return kv == AIONHIP_F16 ? 10.f : LOW; }
__host__ __device__ constexpr float two_to(float e) { return e < 0.f ? 1.f / two_to(-e) : (float)(1 << (int)e); }

struct PagedArgs {
    float *out, *partial, *scores;
    const float *weights_before;
    float *weights;
    float2 *stats;            // of each row: its reference (log2) and the reciprocal of its sum of 2^(s - reference)
    int streams;              // of keys: segments of heads of sequences
    int beside;               // workgroups that read the same keys lie side by side behind one L2
    int draws;                // the workgroup that ends last adds up the weights itself
    unsigned *tickets;
    Table table;
    int T, tpad, L, Hkv, groups, rows_total, row_tiles, nseg, shares;
    int d, q_dtype, kv_dtype;
    float scale, soft_cap;
    unsigned win_left, win_right, win_chunk;
    const void *q;
    const unsigned char *k, *v;
    const int *kv_lengths, *positions;
};

// the keys [lo, hi) of query li of sequence b
__device__ __forceinline__ void row_keys(const PagedArgs &a, int b, int li, int len_raw, int pos_raw, int &lo, int &hi) {
    const int len = a.kv_lengths ? max(0, min(len_raw, a.T)) : a.T;
    const int pos = a.positions ? max(pos_raw, 0) : len - a.L + li;
    lo = hi = 0;
    if (pos < 0) return;
    window_keys(a.win_left, a.win_right, a.win_chunk, pos, len, lo, hi);
    if (hi < lo) hi = lo;
}

// The arguments behind the leading ones, read where they are used: left to itself the compiler asks for all of them at the kernel's start and waits there for the lines that only its end
// needs. One token over 531 keys, one head of 256 for 8: 8.0 -> 7.5 us.
struct KernelArgs {
    const void *pointers[5];
    int numbers[4];
    PagedArgs tail;
};
static_assert(offsetof(KernelArgs, tail) == 56, "paged_attn_kernel's arguments");
__device__ __forceinline__ PagedArgs late_args() {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef const __attribute__((address_space(4))) char *Bytes;
    Bytes at = (Bytes)__builtin_amdgcn_kernarg_segment_ptr() + offsetof(KernelArgs, tail);
    asm volatile("" : "+s"(at));
    return *(const __attribute__((address_space(4))) PagedArgs *)at;
#else
    return PagedArgs{};
#endif
}

constexpr int MOST_SEGMENTS = 256;      // of a row tile
constexpr int wavefronts(int d) { return d == 256 ? 8 : 4; }     // of a workgroup
template <int D, int SHARES>
struct Cfg {
    static constexpr int NW = wavefronts(D), DV = D / SHARES;    // value columns of a workgroup
    static constexpr int ROW = D * 2, V_ROW = DV * 2, TILE = TILE_KEYS * V_ROW;
    static constexpr int SLOT = 16 * (DV + 4) + 32;              // a wavefront's results where they meet: [16][DV + 4], 16 references, 16 sums
    static constexpr int PART = 16 * DV + 32;                    // a segment's results in memory: [16][DV], [16] (reference, sum)
    static constexpr int MOST = MOST_SEGMENTS;
    static constexpr int MEET = NW * SLOT * 4, JOIN = (16 * MOST + 64) * 4 + NW * 64 * 16;          // LDS where wavefronts, where segments meet
    static constexpr int MAIN = NW * TILE > MEET ? (NW * TILE > JOIN ? NW * TILE : JOIN) : MEET > JOIN ? MEET : JOIN;
};
// 16 bytes of LDS by address, not waited for (as a builtin the compiler would wait for every load in flight into LDS first)
template <int OFF>
__device__ __forceinline__ u32x4 lds_read(unsigned addr) {
    u32x4 x;
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(x) : "v"(addr), "n"(OFF) : "memory");
    return x;
}

// One row's share of one wavefront, a key at a time: what its lanes have of the sums (columns dv0 + lane, dv0 + lane + 64, ..), its reference and its sum. See paged_attn_kernel.
template <int D, int DV>
__device__ __forceinline__ void walk_again(const PagedArgs &a, int b, int hk, int r, int rows_total, int L, int lo, int hi, int t_begin, int steps, int stride, int dv0, float (&o)[DV / 64],
                                                     float &top_out, float &sum_out) {
    const int lane = threadIdx.x & 63, li = r / a.groups, gi = r - li * a.groups;
    const size_t qbase = (((size_t)b * L + li) * (a.Hkv * a.groups) + hk * a.groups + gi) * D;
    float q[D / 64], ref = MASKED, l = 0.f;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        q[j] = load_scalar(a.q, a.q_dtype, qbase + lane + 64 * j);
    }
#pragma unroll
    for (int j = 0; j < DV / 64; ++j) o[j] = 0.f;
#pragma unroll 1
    for (int i = 0; i < steps; ++i)
#pragma unroll 1
        for (int k = 0; k < TILE_KEYS; ++k) {
            const int key = (t_begin + i * stride) * TILE_KEYS + k;
            if (key < lo || key >= hi) continue;
            const int page = paged::page_of(a.table, b, key);
            if (page < 0) continue;
            const size_t at = ((((size_t)page * a.Hkv + hk) << a.table.shift) + (key & ((1 << a.table.shift) - 1))) * D;
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < D / 64; ++j) dot += q[j] * load_scalar(a.k, a.kv_dtype, at + lane + 64 * j);
            dot = lanes_sum(dot);
            const float s = a.soft_cap > 0.f ? a.soft_cap * LOG2E * tanhf(dot * (a.scale / a.soft_cap)) : dot * (a.scale * LOG2E);
            if (a.scores && lane == 0 && dv0 == 0)
                __hip_atomic_store(a.scores + ((size_t)(b * a.Hkv + hk) * rows_total + r) * a.tpad + key, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const float top = fmaxf(ref, s), alpha = ref > MASKED ? __builtin_amdgcn_exp2f(ref - top) : 1.f, p = __builtin_amdgcn_exp2f(s - (top > MASKED ? top : 0.f) + head_room(a.kv_dtype));
            l = l * alpha + p;
#pragma unroll
            for (int j = 0; j < DV / 64; ++j) o[j] = o[j] * alpha + p * load_scalar(a.v, a.kv_dtype, at + dv0 + lane + 64 * j);
            ref = top;
        }
    top_out = ref;
    sum_out = l;
}

// QP: how many halves a query element is the sum of. MULTI: several queries a sequence, whose keys may differ (of one query all rows see the same). ONCE: keys and values
// go past the caches. SHARES: workgroups that divide the value columns. The leading arguments, 14 words, arrive in SGPRs with the wavefront. heads: KV heads, query heads of each << 16;
// form: segments, log2 of a page's rows << 12, query type << 16, rows of the queries in LDS << 24, whether the grid is of one dimension << 31.
template <int KV, int D, int QP, bool MULTI, bool ONCE, int SHARES>
__global__ __launch_bounds__(wavefronts(D) * 64, D == 256 ? 2 : 3) void paged_attn_kernel(const int *kv_lengths, const void *q, const int *table, const unsigned char *k, const unsigned char *v, int T, int queries,
                                                                     unsigned heads, unsigned form, PagedArgs tail) {
    using C = Cfg<D, SHARES>;
    constexpr int NW = C::NW, DV = C::DV, KK = D / 32, MT = DV / 16;
    constexpr int PP = KV == AIONHIP_F16 ? 2 : 3;                // parts of a probability
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    PagedArgs a = tail;
    const int L = MULTI ? queries : 1;
    a.kv_lengths = kv_lengths, a.q = q, a.table.pages = table, a.T = T, a.L = L;
    a.Hkv = (int)(heads & 0xFFFFu), a.groups = (int)(heads >> 16);
    a.nseg = (int)(form & 0xFFFu), a.table.shift = (int)(form >> 12 & 0xFu), a.q_dtype = (int)(form >> 16 & 0xFFu);
    a.table.width = T >> a.table.shift;
    a.k = k, a.v = v, a.kv_dtype = KV;
    const int q_rows = D == 256 ? (int)(form >> 24 & 0x1Fu) : 16;        // 8 or 16
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int rows_total = L * a.groups;
    int rt = 0, share = 0, seg, hk = blockIdx.y, b = blockIdx.z;
    if (form >> 31) {
        // Workgroups are dealt to the eight XCDs in turn, so of eight streams of keys (segments of heads of sequences) the first workgroups, a row tile's share, lie next to each other, then
        // their second ones, and so on: those of a stream run side by side behind one L2.
        const PagedArgs z = late_args();
        const unsigned kinds = (unsigned)(z.row_tiles * SHARES), streams = (unsigned)z.streams, first = blockIdx.x / (8 * kinds) * 8, beside = min(8u, streams - first);
        const unsigned within = blockIdx.x - first * kinds, kind = within / beside;
        unsigned stream = first + within - kind * beside;
        rt = (int)(kind / SHARES), share = (int)(kind % SHARES);
        seg = (int)(stream % (unsigned)a.nseg), stream /= (unsigned)a.nseg;
        hk = (int)(stream % (unsigned)a.Hkv), b = (int)(stream / (unsigned)a.Hkv);
    } else {
        const int place = blockIdx.x / SHARES;
        share = blockIdx.x % SHARES;
        rt = rows_total <= 16 ? 0 : place / a.nseg, seg = place - rt * a.nseg;
    }
    const int dv0 = share * DV;
    const int unit = b * a.Hkv + hk;
    const int len_raw = kv_lengths ? kv_lengths[b] : 0;

    // ---- the pages of this wavefront's first tiles are asked for beside the length: the segments take a sequence's tiles in turn, their first wavefronts first, so that
    // which are whose does not depend on how many there are (behind a window they begin later, and are asked for again)
    const int *pages = table + (size_t)b * a.table.width;
    const int stride = a.nseg * NW;
    int t_begin = wave * a.nseg + seg;
    // the pages of the half tiles of 32 steps, one to a lane; -1: none
    auto fetch_pages = [&](int step0) __attribute__((always_inline)) {
        const int e = (int)(((unsigned)(t_begin + (step0 + (lane >> 1)) * stride) * TILE_KEYS + (lane & 1) * 16u) >> a.table.shift);
        return e >= 0 && e < a.table.width ? pages[e] : -1;
    };
    int ids = fetch_pages(0);

    // ---- the queries: a thread asks for eight elements of one row (of two, at head size 256) before anything is waited for
    constexpr int QT = D / 8, QROWS = NW * 64 / QT, QSETS = QROWS >= 16 ? 1 : 16 / QROWS;
    const int q_row = (int)threadIdx.x / QT, q_col = (int)threadIdx.x % QT * 8;
    float qx[QSETS][8];
    u32x4 qh[QSETS];
#pragma unroll
    for (int i = 0; i < QSETS; ++i) {
        const int r = rt * 16 + q_row + i * QROWS;
        const bool there = q_row + i * QROWS < 16 && r < rows_total;
        const int l2 = L > 1 && there ? r / a.groups : 0, g2 = there ? r - l2 * a.groups : 0;
        const size_t at = (((size_t)b * L + l2) * (a.Hkv * a.groups) + hk * a.groups + g2) * D + q_col;
        if constexpr (QP == 1) {
            __builtin_memcpy(&qh[i], (const unsigned short *)q + at, 16);
            if (!there) qh[i] = u32x4{0u, 0u, 0u, 0u};
        } else {
            if (a.q_dtype == AIONHIP_F32) {
                __builtin_memcpy(qx[i], (const float *)q + at, 32);
            } else {
                unsigned short h[8];
                __builtin_memcpy(h, (const unsigned short *)q + at, 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) qx[i][j] = a.q_dtype == AIONHIP_F16 ? __half2float(__ushort_as_half(h[j])) : bf16_bits_to_f32(h[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) qx[i][j] = there ? qx[i][j] : 0.f;
        }
    }

    // ---- what this lane's row sees
    const int r = rt * 16 + n;
    const bool row_ok = r < rows_total;
    const int li = MULTI && row_ok ? r / a.groups : 0;
    int lo, hi;
    row_keys(a, b, li, len_raw, a.positions ? a.positions[(size_t)b * L + li] : 0, lo, hi);
    int uni_lo, uni_hi, all_lo, all_hi;                          // of any row's keys, of those that every row sees
    if constexpr (MULTI) {
        if (!row_ok) lo = hi = 0;
        const bool some = hi > lo;
        uni_lo = rows16_min_i(some ? lo : INT_MAX), uni_hi = rows16_max_i(some ? hi : 0);
        all_lo = rows16_max_i(row_ok ? (some ? lo : INT_MAX) : 0), all_hi = rows16_min_i(row_ok ? (some ? hi : 0) : INT_MAX);
    } else {
        lo = uni_lo = all_lo = __builtin_amdgcn_readfirstlane(lo);
        hi = uni_hi = all_hi = __builtin_amdgcn_readfirstlane(hi);
    }

    // ---- this wavefront's tiles
    int tb = 0, te = 0;
    if (uni_hi > uni_lo) tb = uni_lo / TILE_KEYS, te = (uni_hi + TILE_KEYS - 1) / TILE_KEYS;
    const int live = min(a.nseg, te - tb);                       // segments that have tiles
    if (seg >= max(live, 1)) return;
    if (tb > 0) {
        t_begin += tb;
        ids = fetch_pages(0);
    }
    const int steps = t_begin < te ? (te - t_begin + stride - 1) / stride : 0;

    unsigned char *vs = lds + wave * C::TILE;
    const size_t page_bytes = ((size_t)a.Hkv << a.table.shift) * C::ROW, head_bytes = ((size_t)hk << a.table.shift) * C::ROW;
    const unsigned char *kp = k + head_bytes, *vp = v + head_bytes;
    const int row_mask = (1 << a.table.shift) - 1;
    u32x4 kf[2][KK];
    auto load_k = [&](int t, int id0, int id1) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned char *at = kp + (size_t)(unsigned)max(h ? id1 : id0, 0) * page_bytes + (size_t)((t * TILE_KEYS + h * 16) & row_mask) * C::ROW;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const u32x4 *from = (const u32x4 *)(at + (unsigned)(n * C::ROW + g * 16) + kk * 64);
                kf[h][kk] = ONCE ? __builtin_nontemporal_load(from) : *from;
            }
        }
    };
    // V: 1 KiB an instruction, straight into LDS. 16-byte chunk c of key k lies at slot c ^ (2 * ((k >> 2) & 3)) ^ (8 * (k & 1)) of its row (the last term for rows
    // of 256 bytes and more), so that the sixteen keys of a transposing read fall on distinct banks.
    constexpr int NVI = C::TILE / 1024, KEYS_PER_VI = 1024 / C::V_ROW;
    const int v_key_in = (lane * 16) / C::V_ROW, v_slot = ((lane * 16) % C::V_ROW) / 16;
    constexpr int NON_TEMPORAL = 2;                              // the nt bit of a buffer access
    (void)v_slot; (void)vp; (void)NON_TEMPORAL;
    auto load_v = [&](int t, int id0, int id1) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned char *at = vp + (size_t)(unsigned)max(h ? id1 : id0, 0) * page_bytes + (size_t)((t * TILE_KEYS + h * 16) & row_mask) * C::ROW;
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, 16 * C::ROW, 0x00027000);
#pragma unroll
            for (int i = 0; i < NVI / 2; ++i) {
                const int key = i * KEYS_PER_VI + v_key_in;
                const int chunk = v_slot ^ (2 * ((key >> 2) & 3)) ^ (DV >= 128 ? 8 * (key & 1) : 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(vs + (h * (NVI / 2) + i) * 1024), 16, key * C::ROW + dv0 * 2 + chunk * 16, 0, 0, ONCE ? NON_TEMPORAL : 0);
            }
        }
#endif
    };
    // a lane's page number as a scalar, -1: none
    auto page_at = [&](int l) __attribute__((always_inline)) {
        const int id = __builtin_amdgcn_readlane(ids, l);
        return (unsigned)id < (unsigned)a.table.count ? id : -1;
    };
    int id0 = -1, id1 = -1;
    auto begin = [&]() __attribute__((always_inline)) {
        id0 = page_at(0), id1 = page_at(1);
        load_k(t_begin, id0, id1);
        load_v(t_begin, id0, id1);
    };
    if (steps > 0) begin();

    // ---- the queries as operands in LDS, under the first tile's way: [part][k-step][16-byte piece of 4][row]
    unsigned char *qs = lds + C::MAIN;
    float *q_scale = (float *)(qs + QP * q_rows * C::ROW);       // what brings a row's products back to q . k
    const int q_shift = q_rows == 16 ? 4 : 3;
#pragma unroll
    for (int i = 0; i < QSETS; ++i) {
        const int row = q_row + i * QROWS;
        const unsigned at = (unsigned)(((q_col / 8) << q_shift) + row) * 16;
        if constexpr (QP == 1) {
            if (row < q_rows) *(u32x4 *)(qs + at) = qh[i];
            if (row < q_rows && q_col == 0) q_scale[row] = 1.f;
        } else {
            float factor = 1.f, back = 1.f;
            if constexpr (KV == AIONHIP_F16) {
                // a row goes into f16's range by a power of two that takes its largest element to 2^10: what the second half rounds away then lies 2^-35 below that
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(qx[i][j]));
                top = fmaxf(top, dpp_f<DPP_QUAD_XOR1>(top));
                top = fmaxf(top, dpp_f<DPP_QUAD_XOR2>(top));
                top = fmaxf(top, dpp_f<DPP_ROW_HALF_MIRROR>(top));
                if constexpr (QT > 8) top = fmaxf(top, dpp_f<DPP_ROW_MIRROR>(top));
                if constexpr (QT > 16) {
                    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
                }
                const int e = (int)(__float_as_uint(top) >> 23);
                const int f = e == 255 ? 127 : max(1, min(264 - e, 253));
                factor = __uint_as_float((unsigned)f << 23);
                back = __uint_as_float((unsigned)(254 - f) << 23);
            }
            u32x4 part[QP];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float u = qx[i][j] * factor, w = qx[i][j + 1] * factor;
#pragma unroll
                for (int p = 0; p < QP; ++p) {
                    const unsigned both = pack2<KV>(u, w);
                    part[p][j / 2] = both;
                    // (an infinite element has no rest)
                    const float ru = u - from_half_bits<KV>((unsigned short)both), rw = w - from_half_bits<KV>((unsigned short)(both >> 16));
                    u = fabsf(ru) < INFINITY ? ru : 0.f;
                    w = fabsf(rw) < INFINITY ? rw : 0.f;
                }
            }
            if (row < q_rows) {
#pragma unroll
                for (int p = 0; p < QP; ++p) *(u32x4 *)(qs + p * q_rows * C::ROW + at) = part[p];
                if (q_col == 0) q_scale[row] = back;
            }
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");       // (no wait for the K and V loads in flight)
    const int q_mine = n & (q_rows - 1);                         // (of eight rows, the upper eight columns are the lower once more, and nobody's)
    const unsigned q_addr = (unsigned)(size_t)(lds_void *)qs + (unsigned)(((g << q_shift) + q_mine) * 16), q_part = (unsigned)(q_rows * C::ROW), q_step = 64u << q_shift;
    float to_log2;
    {
        u32x2 x;
        asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(x.x) : "v"((unsigned)(size_t)(lds_void *)q_scale + (unsigned)q_mine * 4) : "memory");
        const float back = __uint_as_float(x.x);
        to_log2 = a.soft_cap > 0.f ? back * (a.scale / a.soft_cap) : back * (a.scale * LOG2E);
    }
    const float cap_log2 = a.soft_cap * LOG2E;

    const int tr_r = (lane >> 2) & 3, tr_q = lane & 3;
    const unsigned v_rowaddr = (unsigned)(size_t)(lds_void *)vs + (unsigned)((4 * g + tr_r) * C::V_ROW + (tr_q & 1) * 8);
    const unsigned v_slot_l = (unsigned)(((tr_q >> 1) ^ (2 * g) ^ (DV >= 128 ? 8 * (tr_r & 1) : 0)) << 4);
    auto v_operand = [&](unsigned vr, unsigned vl, auto mt_c) __attribute__((always_inline)) {
        constexpr int mt = decltype(mt_c)::value;
        const unsigned addr = vr + (vl ^ (unsigned)(mt << 5));
        u32x2 a0, a1;
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3" : "=&v"(a0), "=&v"(a1) : "v"(addr), "n"(16 * C::V_ROW) : "memory");
        return u32x4{a0.x, a0.y, a1.x, a1.y};
    };

    f32x4 acc[MT];
    float ref = MASKED, peak = MASKED, l_run = 0.f;              // peak: the largest score; l_run: of this lane's keys
    constexpr int DEVICE_SCOPE = 16;                             // the sc1 bit of a buffer access: written through, read at the point where the XCDs' caches agree
    (void)DEVICE_SCOPE;
#if defined(__HIP_DEVICE_COMPILE__)
    const __amdgpu_buffer_rsrc_t scores_rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(a.scores + ((size_t)unit * rows_total + rt * 16) * a.tpad), 0,
                                                                                 a.scores ? (unsigned)min(16, rows_total - rt * 16) * (unsigned)a.tpad * 4u : 0u, 0x00027000);
#endif
    // MORE: another tile of this wavefront follows (two copies of the body, so that every path requests K and V in the same order and the count of loads in flight holds)
    auto tile = [&](int t, bool ok0, bool ok1, int next0, int next1, auto more_c) __attribute__((always_inline)) {
        constexpr bool more = decltype(more_c)::value;
        const int key0 = t * TILE_KEYS;
        f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        // (the operands' addresses are made anew for each tile: kept, they would take the registers of two wavefronts' worth of keys in flight)
        unsigned qa = q_addr, vr = v_rowaddr, vl = v_slot_l;
        asm volatile("" : "+v"(qa), "+v"(vr), "+v"(vl));
        constexpr int QA = KK * QP < 4 ? KK * QP : 4;            // operands requested ahead
        u32x4 qf[QA];
        auto q_operand = [&](auto ic) __attribute__((always_inline)) {
            constexpr int i = decltype(ic)::value;
            return lds_read<0>(qa + (unsigned)(i / QP) * q_step + (unsigned)(i % QP) * q_part);
        };
        static_for<0, QA>([&](auto ic) __attribute__((always_inline)) { qf[decltype(ic)::value] = q_operand(ic); });
        static_for<0, KK * QP>([&](auto ic) __attribute__((always_inline)) {
            constexpr int i = decltype(ic)::value, later = KK * QP - 1 - i < QA - 1 ? KK * QP - 1 - i : QA - 1;
            asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(qf[i % QA]) : "n"(later));
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = mfma16<KV>(kf[h][i / QP], qf[i % QA], s[h]);
            if constexpr (i + QA < KK * QP) qf[i % QA] = q_operand(std::integral_constant<int, i + QA>{});
        });
        const bool full = key0 >= all_lo && key0 + TILE_KEYS <= all_hi && ok0 && ok1;      // every row sees every key
        // lane: keys key0 + h * 16 + g * 4 + i of row n
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = s[j >> 2][j & 3] * to_log2;
        if (a.soft_cap > 0.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = cap_log2 * tanhf(p[j]);
        }
        if (!full) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = key0 + (j >> 2) * 16 + g * 4 + (j & 3);
                p[j] = key >= lo && key < hi && (j < 4 ? ok0 : ok1) ? p[j] : MASKED;
            }
        }
        const bool scored = a.scores && share == 0;              // (some lane of every wavefront has a row)
#if defined(__HIP_DEVICE_COMPILE__)
        if (scored && row_ok) {
            const int at = (int)((unsigned)(n * a.tpad + g * 4) * 4u);
            const u32x4 lower = __builtin_bit_cast(u32x4, f32x4{p[0], p[1], p[2], p[3]}), upper = __builtin_bit_cast(u32x4, f32x4{p[4], p[5], p[6], p[7]});
            if (a.draws) {
                __builtin_amdgcn_raw_buffer_store_b128(lower, scores_rsrc, at, key0 * 4, DEVICE_SCOPE);
                __builtin_amdgcn_raw_buffer_store_b128(upper, scores_rsrc, at + 64, key0 * 4, DEVICE_SCOPE);
            } else {                               // (written through they would cost a long call a tenth)
                __builtin_amdgcn_raw_buffer_store_b128(lower, scores_rsrc, at, key0 * 4, 0);
                __builtin_amdgcn_raw_buffer_store_b128(upper, scores_rsrc, at + 64, key0 * 4, 0);
            }
        }
#endif
        if (more) {
            load_k(t + stride, next0, next1);
            asm volatile("" ::: "memory");         // requested here, ahead of the counted wait for V below
        }
        float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        mx = groups4_max(mx);
        peak = fmaxf(peak, mx);
        const float ref_new = __builtin_ceilf(KV == AIONHIP_F16 ? fmaxf(mx, peak - DEPTH) : mx);
        const bool moves = ref_new > ref + SLACK || (KV == AIONHIP_F16 && mx > MASKED && ref_new < ref - DROP);
        if (__any(moves)) {
            if (moves) {
                const float alpha = ref > MASKED ? __builtin_amdgcn_ldexpf(1.f, (int)fmaxf(fminf(ref - ref_new, 200.f), -200.f)) : 0.f;
                l_run *= alpha;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt] *= alpha;
                ref = ref_new;
            }
        }
        const float base = (ref > MASKED ? ref : 0.f) - head_room(KV);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = __builtin_amdgcn_exp2f(p[j] - base);
            sum += p[j];
        }
        l_run += sum;
        u32x4 pf[PP];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            float u = p[j], w = p[j + 1];
#pragma unroll
            for (int part = 0; part < PP; ++part) {
                const unsigned both = pack2<KV>(u, w);
                pf[part][j / 2] = both;
                u -= from_half_bits<KV>((unsigned short)both);
                w -= from_half_bits<KV>((unsigned short)(both >> 16));
            }
        }
        // V has landed once only what is younger is outstanding, K and the two stores of scores (they complete in order); the tile is this wavefront's alone
        if (more && scored) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * KK + 2));
        else if (more) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * KK));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        asm volatile("" ::: "memory");
        if (!full) {
            // rows that no query sees count as zeros: they may hold anything, and zero times that need not be zero
#pragma unroll 1
            for (int i = 0; i < NVI; ++i) {
                const int key = key0 + i * KEYS_PER_VI + v_key_in;
                if (key < uni_lo || key >= uni_hi || !(i < NVI / 2 ? ok0 : ok1)) *(u32x4 *)(vs + i * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        constexpr int VA = MT < 4 ? MT : 4;                  // operands requested ahead
        u32x4 vop[VA];
        static_for<0, VA>([&](auto mc) __attribute__((always_inline)) { vop[decltype(mc)::value] = v_operand(vr, vl, mc); });
        static_for<0, MT>([&](auto mc) __attribute__((always_inline)) {
            constexpr int mt = decltype(mc)::value;
            constexpr int later = MT - 1 - mt < VA - 1 ? MT - 1 - mt : VA - 1;
            asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(vop[mt % VA]) : "n"(2 * later));
#pragma unroll
            for (int part = 0; part < PP; ++part) acc[mt] = mfma16<KV>(vop[mt % VA], pf[part], acc[mt]);
            if constexpr (mt + VA < MT) vop[mt % VA] = v_operand(vr, vl, std::integral_constant<int, mt + VA>{});
        });
        if (more) {
            asm volatile("" ::: "memory");         // the operand reads above are complete: each was waited for before its product
            load_v(t + stride, next0, next1);
        }
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (steps > 0) {
        int t = t_begin;
        for (int i = 1; i < steps; ++i, t += stride) {
            if ((i & 31) == 0) ids = fetch_pages(i);
            const int next0 = page_at(2 * (i & 31)), next1 = page_at(2 * (i & 31) + 1);
            tile(t, id0 >= 0, id1 >= 0, next0, next1, std::true_type{});
            id0 = next0, id1 = next1;
        }
        tile(t, id0 >= 0, id1 >= 0, 0, 0, std::false_type{});
        // What is infinite or no number may have spoilt a row that does not see it (zero times it is no number), or that does (so is a sum of halves times infinity): rows that end
        // as no number are walked again, a key at a time and in f32, which has what they see and nothing else.
        bool none = l_run != l_run;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j) none |= acc[mt][j] != acc[mt][j];
        const uint64_t spoilt = __ballot(none && row_ok);
        if (spoilt) {
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
                if (!(spoilt >> i & 0x0001000100010001ull)) continue;
                float o[DV / 64], top, sum;
                walk_again<D, DV>(a, b, hk, rt * 16 + i, rows_total, L, __builtin_amdgcn_readlane(lo, i), __builtin_amdgcn_readlane(hi, i), t_begin, steps, stride, dv0, o, top, sum);
#pragma unroll
                for (int j = 0; j < DV / 64; ++j) ((float *)vs)[lane + 64 * j] = o[j];
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (n == i) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) acc[mt] = *(const f32x4 *)((const float *)vs + mt * 16 + g * 4);
                    ref = top;
                    l_run = g == 0 ? sum : 0.f;
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
    }
    l_run = groups4_sum(l_run);

    const PagedArgs z = late_args();
    const int rows = min(16, rows_total - rt * 16);
    float2 *const s_stat = (float2 *)qs;                         // (the queries are dead)
    auto put = [&](int row, int col, f32x4 o, float top, float l) __attribute__((always_inline)) {
        const int rr = rt * 16 + row, l2 = L > 1 ? rr / a.groups : 0, g2 = rr - l2 * a.groups;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *(f32x4 *)(z.out + (((size_t)b * L + l2) * (a.Hkv * a.groups) + hk * a.groups + g2) * D + dv0 + col) = o * inv;
        if (a.scores && dv0 + col == 0) {
            const float2 st{top > MASKED ? top : 0.f, inv * two_to(head_room(KV))};
            if (z.draws) s_stat[row] = st;
            else z.stats[(size_t)unit * rows_total + rr] = st;
        }
    };
    // What the keys draw, in calls of few scores: a thread has four keys and adds the rows' probabilities in order, as paged_weights_kernel does.
    auto draw = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const bool in_place = z.weights == z.weights_before;
        for (int key = (int)threadIdx.x * 4; key < a.T; key += NW * 256) {
            const bool seen = key < uni_hi && key + 4 > uni_lo;
            if (in_place && !seen) continue;
            const size_t at = (size_t)unit * a.T + key;
            f32x4 w = f32x4{0.f, 0.f, 0.f, 0.f}, before = w;
            if (z.weights_before) __builtin_memcpy(&before, z.weights_before + at, 16);
            u32x4 x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = u32x4{0u, 0u, 0u, 0u};
#if defined(__HIP_DEVICE_COMPILE__)
                if (seen && i < rows) x[i] = __builtin_amdgcn_raw_buffer_load_b128(scores_rsrc, (i * a.tpad + key) * 4, 0, DEVICE_SCOPE);
#endif
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (i >= rows) break;
                const int from = MULTI ? __builtin_amdgcn_readlane(lo, i) : lo, end = MULTI ? __builtin_amdgcn_readlane(hi, i) : hi;
                const float2 st = s_stat[i];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (key + j >= from && key + j < end) w[j] += __builtin_amdgcn_exp2f(__uint_as_float(x[i][j]) - st.x) * st.y;
            }
            w += before;
            __builtin_memcpy(z.weights + at, &w, 16);
        }
    };
    const int meeting = (unit * z.row_tiles + rt) * SHARES + share;
    [[maybe_unused]] float *const slots = z.partial + (size_t)meeting * a.nseg * C::PART;
#if defined(__HIP_DEVICE_COMPILE__)
    const __amdgpu_buffer_rsrc_t slots_rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)slots, 0, (unsigned)(a.nseg * C::PART * 4), 0x00027000);
#endif
    auto publish = [&](int row, int col, f32x4 o, float top, float l) __attribute__((always_inline)) {
        if (live <= 1) {
            put(row, col, o, top, l);
            return;
        }
#if defined(__HIP_DEVICE_COMPILE__)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), slots_rsrc, (seg * C::PART + row * DV + col) * 4, 0, DEVICE_SCOPE);
        if (col == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(top), __float_as_uint(l)}, slots_rsrc, (seg * C::PART + 16 * DV + row * 2) * 4, 0, DEVICE_SCOPE);
#endif
    };
    if (te - tb <= a.nseg) {                                     // the first wavefront has all there is
        if (wave == 0 && row_ok) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) publish(n, mt * 16 + g * 4, acc[mt], ref, l_run);
        }
    } else {
        // ---- the wavefronts meet in LDS
        __syncthreads();
        float *mg = (float *)lds;
        if (row_ok) {
            float *w = mg + wave * C::SLOT;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) *(f32x4 *)(w + n * (DV + 4) + mt * 16 + g * 4) = acc[mt];
            if (g == 0) { w[16 * (DV + 4) + n] = ref; w[16 * (DV + 4) + 16 + n] = l_run; }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < rows * (DV / 4); e += NW * 64) {
            const int row = e / (DV / 4), col = (e % (DV / 4)) * 4;
            float rw[NW], lw[NW], top = MASKED, l = 0.f;
            f32x4 ow[NW], o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                rw[w] = mg[w * C::SLOT + 16 * (DV + 4) + row];
                lw[w] = mg[w * C::SLOT + 16 * (DV + 4) + 16 + row];
                ow[w] = *(const f32x4 *)(mg + w * C::SLOT + row * (DV + 4) + col);
                top = fmaxf(top, rw[w]);
            }
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                // (a wavefront without a reference has seen nothing, or what is not a number: its sums then say so)
                const float f = rw[w] > MASKED ? __builtin_amdgcn_exp2f(rw[w] - top) : 1.f;
                l += lw[w] * f;
                o += ow[w] * f;
            }
            publish(row, col, o, top, l);
        }
    }
    if (live > 1) {
        // ---- the workgroup that ends last adds the segments: each publishes its part, waits until the stores have been acknowledged and takes a ticket; whoever draws the
        // last one finds all of them. Nobody waits for anybody.
        __syncthreads();
        int *s_ticket = (int *)lds;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) *s_ticket = (int)__hip_atomic_fetch_add(z.tickets + meeting * MEET_TICKET_WORDS, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (*s_ticket != live - 1) return;
        if (threadIdx.x == 0) __hip_atomic_store(z.tickets + meeting * MEET_TICKET_WORDS, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        float *s_f = (float *)lds, *s_top = s_f + 16 * C::MOST, *s_l = s_top + 16;      // factors of the segments of each row
        f32x4 *s_o = (f32x4 *)(lds + (16 * C::MOST + 64) * 4);
        // A wavefront derives the segments' factors for every NW-th row, a lane to a segment; all are asked for at once.
        constexpr int EACH = 16 / NW;
        u32x2 st[EACH][C::MOST / 64];
#pragma unroll
        for (int i = 0; i < EACH; ++i)
#pragma unroll
            for (int j = 0; j < C::MOST / 64; ++j) {
                st[i][j] = u32x2{__float_as_uint(MASKED), 0u};
#if defined(__HIP_DEVICE_COMPILE__)
                if (wave + i * NW < rows && lane + 64 * j < live)
                    st[i][j] = __builtin_amdgcn_raw_buffer_load_b64(slots_rsrc, ((lane + 64 * j) * C::PART + 16 * DV + (wave + i * NW) * 2) * 4, 0, DEVICE_SCOPE);
#endif
            }
        // A thread has four columns of a row; where there are more threads than that, several share the segments. Eight parts at a time, the next eight asked for ahead.
        const int pieces = rows * (DV / 4), sets = max(1, NW * 64 / pieces), set = (int)threadIdx.x / pieces;
        const bool mine = set < sets;
        int e = (int)threadIdx.x - set * pieces, s0 = set;
        u32x4 x[2][8];
        auto ask = [&](u32x4 (&to)[8], int e, int s0) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                [[maybe_unused]] const int s = s0 + j * sets;        // (past the last segment: past the buffer's end, which reads as zeros)
                to[j] = u32x4{0u, 0u, 0u, 0u};
#if defined(__HIP_DEVICE_COMPILE__)
                to[j] = __builtin_amdgcn_raw_buffer_load_b128(slots_rsrc, s < live && e < pieces ? (s * C::PART + e / (DV / 4) * DV + e % (DV / 4) * 4) * 4 : 0x7FFFFFF0, 0, DEVICE_SCOPE);
#endif
            }
        };
        ask(x[0], e, s0);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int row = wave + i * NW;
            if (row >= rows) break;
            float top = MASKED, sum = 0.f;
#pragma unroll
            for (int j = 0; j < C::MOST / 64; ++j) top = fmaxf(top, __uint_as_float(st[i][j].x));
            top = lanes_max(top);
#pragma unroll
            for (int j = 0; j < C::MOST / 64; ++j) {
                const float sr = __uint_as_float(st[i][j].x), f = sr > MASKED ? __builtin_amdgcn_exp2f(sr - top) : 1.f;
                s_f[row * C::MOST + lane + 64 * j] = lane + 64 * j < live ? f : 0.f;
                sum += __uint_as_float(st[i][j].y) * f;
            }
            sum = lanes_sum(sum);
            if (lane == 0) s_top[row] = top, s_l[row] = sum;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
        // one round: eight parts added, and the piece written with its last ones; false: none are left
        auto round = [&](u32x4 (&now)[8], u32x4 (&next)[8]) __attribute__((always_inline)) {
            const bool last = s0 + 8 * sets - set >= live;           // (the same for all threads)
            const int e2 = last ? e + NW * 64 : e, s2 = last ? set : s0 + 8 * sets;
            const bool more = !last || (sets == 1 && e2 - (int)threadIdx.x < pieces);
            if (more) ask(next, e2, s2);
            const int row = min(e / (DV / 4), 15);
#pragma unroll
            for (int j = 0; j < 8; ++j) o += __builtin_bit_cast(f32x4, now[j]) * (s0 + j * sets < live ? s_f[row * C::MOST + s0 + j * sets] : 0.f);
            if (last) {
                if (sets > 1) {
                    s_o[threadIdx.x] = o;
                    __syncthreads();
                    if (set == 0)
                        for (int i = 1; i < sets; ++i) o += s_o[i * pieces + threadIdx.x];
                }
                if (mine && set == 0 && e < pieces) put(row, e % (DV / 4) * 4, o, s_top[row], s_l[row]);
                o = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            e = e2, s0 = s2;
            return more;
        };
        while (round(x[0], x[1]) && round(x[1], x[0])) {}
    }
    if (z.draws && share == 0) draw();
}

// What the keys draw: a thread has KEYS of them and adds the rows' probabilities in order, AHEAD rows asked for before the first is used. stats: a row's reference and the reciprocal of
// its sum. What it costs is the rows' loads one after another where there are few keys, so a thread has one and eight rows ahead (64 rows of 8 heads over 4000 keys 9 us; four keys, a
// row at a time, 33), and the bytes of the scores where there are many, so it has four and four ahead (32 sequences, 8 heads, over 8192 keys 10 us).
constexpr int WEIGH_ROWS = 64;
constexpr size_t WEIGH_MANY = (size_t)512 << 10;
template <int KEYS, int AHEAD>
__global__ __launch_bounds__(256) void paged_weights_kernel(PagedArgs a) {
    __shared__ float2 s_stat[WEIGH_ROWS];
    __shared__ int2 s_keys[WEIGH_ROWS];
    const int hk = blockIdx.y, b = blockIdx.z, unit = b * a.Hkv + hk, tid = threadIdx.x, key = ((int)blockIdx.x * 256 + tid) * KEYS;
    const size_t at = (size_t)unit * a.T + key;
    float w[KEYS] = {};
    const int len = a.kv_lengths ? a.kv_lengths[b] : 0;
    bool seen = a.weights != a.weights_before;   // (in place what nobody sees stays as it is: a capacity may be far past the lengths)
    if (!seen && a.kv_lengths && (int)blockIdx.x * 256 * KEYS >= len) return;
    for (int r0 = 0; r0 < a.rows_total; r0 += WEIGH_ROWS) {
        const int rows = min(WEIGH_ROWS, a.rows_total - r0);
        if (r0) __syncthreads();
        if (tid < rows) {
            const int r = r0 + tid, li = a.L > 1 ? r / a.groups : 0;
            int lo, hi;
            row_keys(a, b, li, len, a.positions ? a.positions[(size_t)b * a.L + li] : 0, lo, hi);
            s_keys[tid] = int2{lo, hi};
            s_stat[tid] = a.stats[(size_t)unit * a.rows_total + r];
        }
        __syncthreads();
        if (key < a.T) {
            const float *from = a.scores + ((size_t)unit * a.rows_total + r0) * a.tpad + key;
            for (int i0 = 0; i0 < rows; i0 += AHEAD) {
                float s[AHEAD][KEYS];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) __builtin_memcpy(s[i], from + (size_t)min(i0 + i, rows - 1) * a.tpad, sizeof s[i]);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int2 see = s_keys[min(i0 + i, rows - 1)];
                    const float2 st = s_stat[min(i0 + i, rows - 1)];
                    const int end = i0 + i < rows ? see.y : 0;
                    seen |= key < end && key + KEYS > see.x;
#pragma unroll
                    for (int j = 0; j < KEYS; ++j) w[j] += key + j >= see.x && key + j < end ? __builtin_amdgcn_exp2f(s[i][j] - st.x) * st.y : 0.f;
                }
            }
        }
    }
    if (key < a.T && seen) {                     // (a capacity is a multiple of sixteen)
        if (a.weights_before) {
            float before[KEYS];
            __builtin_memcpy(before, a.weights_before + at, sizeof w);
#pragma unroll
            for (int j = 0; j < KEYS; ++j) w[j] += before[j];
        }
        __builtin_memcpy(a.weights + at, w, sizeof w);
    }
}

// One workgroup a query row, any head size: its four wavefronts take keys in turn. One token of 8 heads of 96 over 1024 keys 290 us, a chain of loads and sums to each key.
__global__ __launch_bounds__(256) void paged_generic_kernel(PagedArgs a) {
    constexpr int EACH = (int)paged::MAX_HEAD / 64;
    __shared__ float s_o[4][paged::MAX_HEAD], s_top[4], s_l[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, unit = b * a.Hkv + hk, li = r / a.groups, gi = r - li * a.groups;
    int lo, hi;
    row_keys(a, b, li, a.kv_lengths ? a.kv_lengths[b] : 0, a.positions ? a.positions[(size_t)b * a.L + li] : 0, lo, hi);
    const size_t qbase = (((size_t)b * a.L + li) * (a.Hkv * a.groups) + hk * a.groups + gi) * a.d;
    float q[EACH], o[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        q[j] = lane + 64 * j < a.d ? load_scalar(a.q, a.q_dtype, qbase + lane + 64 * j) : 0.f;
        o[j] = 0.f;
    }
    float ref = MASKED, l = 0.f;
    for (int key = lo + wave; key < hi; key += 4) {
        const int page = paged::page_of(a.table, b, key);
        float s = MASKED;
        size_t at = 0;
        if (page >= 0) {
            at = ((((size_t)page * a.Hkv + hk) << a.table.shift) + (key & ((1 << a.table.shift) - 1))) * a.d;
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (lane + 64 * j < a.d) dot += q[j] * load_scalar(a.k, a.kv_dtype, at + lane + 64 * j);
            dot = lanes_sum(dot);
            s = a.soft_cap > 0.f ? a.soft_cap * LOG2E * tanhf(dot * (a.scale / a.soft_cap)) : dot * (a.scale * LOG2E);
        }
        if (a.scores && lane == 0) a.scores[((size_t)unit * a.rows_total + r) * a.tpad + key] = s;
        if (page < 0) continue;
        const float top = fmaxf(ref, s);
        const float alpha = ref > MASKED ? __builtin_amdgcn_exp2f(ref - top) : 1.f, p = __builtin_amdgcn_exp2f(s - (top > MASKED ? top : 0.f) + LOW);
        l = l * alpha + p;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if (lane + 64 * j < a.d) o[j] = o[j] * alpha + p * load_scalar(a.v, a.kv_dtype, at + lane + 64 * j);
        ref = top;
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j)
        if (lane + 64 * j < a.d) s_o[wave][lane + 64 * j] = o[j];
    if (lane == 0) s_top[wave] = ref, s_l[wave] = l;
    __syncthreads();
    const float top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    float f[4], sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = s_top[w] > MASKED ? __builtin_amdgcn_exp2f(s_top[w] - top) : 1.f;
        sum += s_l[w] * f[w];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int c = threadIdx.x; c < a.d; c += 256) a.out[qbase + c] = (s_o[0][c] * f[0] + s_o[1][c] * f[1] + s_o[2][c] * f[2] + s_o[3][c] * f[3]) * inv;
    if (a.stats && threadIdx.x == 0) a.stats[(size_t)unit * a.rows_total + r] = float2{top > MASKED ? top : 0.f, inv * two_to(LOW)};
}

template <int KV, int D, int QP, bool MULTI, bool ONCE, int SHARES = 1>
int launch(aionhip_ctx *ctx, const PagedArgs &a, int batch) {
    using C = Cfg<D, SHARES>;
    const auto kernel = paged_attn_kernel<KV, D, QP, MULTI, ONCE, SHARES>;
    const int q_rows = D == 256 && a.rows_total <= 8 ? 8 : 16;
    const size_t lds = C::MAIN + QP * q_rows * C::ROW + 64;
    static std::atomic<uint64_t> attr{0};
    if (const int rc = allow_lds(ctx, attr, (const void *)kernel, C::MAIN + QP * 16 * C::ROW + 64)) return rc;
    ProfScope scope(ctx, "paged_attn");
    // (one dimension where keys are read by several workgroups, if it takes them all)
    const size_t wgs = (size_t)a.row_tiles * a.nseg * SHARES * a.Hkv * batch;
    const bool flat = a.beside && wgs <= paged::MAX_THREADS / (C::NW * 64);
    const dim3 grid = flat ? dim3((unsigned)wgs) : dim3((unsigned)(a.row_tiles * a.nseg * SHARES), (unsigned)a.Hkv, (unsigned)batch);
    launch_k(ctx, kernel, grid, dim3(C::NW * 64), lds, a.kv_lengths, a.q, a.table.pages, a.k, a.v, a.T, a.L,
             (unsigned)a.Hkv | (unsigned)a.groups << 16, (unsigned)a.nseg | (unsigned)a.table.shift << 12 | (unsigned)a.q_dtype << 16 | (unsigned)q_rows << 24 | (flat ? 1u << 31 : 0u), a);
    LAUNCH_CHECK(ctx, "paged_attn");
    return AIONHIP_OK;
}
template <int KV, int D, int QP>
int launch_form(aionhip_ctx *ctx, const PagedArgs &a, int batch, bool once) {
    if constexpr (D > 64)
        if (a.shares > 1) return a.L > 1 ? launch<KV, D, QP, true, false, D / 64>(ctx, a, batch) : launch<KV, D, QP, false, false, D / 64>(ctx, a, batch);
    if (a.L > 1) return launch<KV, D, QP, true, false>(ctx, a, batch);
    return once ? launch<KV, D, QP, false, true>(ctx, a, batch) : launch<KV, D, QP, false, false>(ctx, a, batch);
}
template <int KV, int D>
int launch_parts(aionhip_ctx *ctx, const PagedArgs &a, int batch, bool once) {
    if (a.q_dtype == KV) return launch_form<KV, D, 1>(ctx, a, batch, once);
    return launch_form<KV, D, KV == AIONHIP_F16 ? 2 : 3>(ctx, a, batch, once);
}
template <int KV>
int launch_head(aionhip_ctx *ctx, const PagedArgs &a, int batch, bool once) {
    if (a.d == 64) return launch_parts<KV, 64>(ctx, a, batch, once);
    if (a.d == 128) return launch_parts<KV, 128>(ctx, a, batch, once);
    return launch_parts<KV, 256>(ctx, a, batch, once);
}

// How a row tile is split: key segments, and shares of the value columns (each share computes all of the scores; the reads of V, the second product, the meetings and the
// joining are divided). As many segments as give each CU two workgroups at once (one of head size 256, whose LDS does not hold two), or four (two) in turn where the sequences alone
// fill the CUs, since these are of uneven lengths: 32 sequences of up to 16384 keys, 8 heads of 128, 253 us in four segments, 263 in two, 277 in one. Fewer, and in shares of 64
// columns while those leave no CU with two workgroups, where that is less by what the parts of a call took one by one, us: a tile (a CU has only so many loads
// in flight, so that two workgroups on one take 1.4 to 1.6 times as long), whole rows of V on their way through the first one, the wavefronts' meeting, the segments' joining,
// of which the workgroup that joins reads NW * 8 KiB of parts to a memory round trip. Over 40 shapes the choice is within 8 % of the best of 30 on all but one (12).
// One token, one head of 256 for 8, whole / in four shares, us: 100 keys 7.8 / 6.4, 531 10.4 / 7.3, 2048 11.0 / 8.4, 8192 14.6 / 9.8, 131072 38 / 54; 8 heads of 128 for 32, whole / in two: 100 keys
// 6.2 / 5.5, 531 7.5 / 6.9, 2048 7.4 / 7.3, 8192 (whole in 32 segments, which two shares have no room for) 10.0 / 13.1.
struct Split { int segments, shares; };
Split split_of(long wgs, long tiles, int rows, int d, long cus) {
    const long at_once = d == 256 ? 1 : 2;
    const int nw = wavefronts(d);
    Split best{1, 1};
    float least = INFINITY;
    for (int shares = 1; shares == 1 || (shares == d / 64 && wgs * shares <= cus); shares = d / 64) {
        const long room = shares > 1 ? cus / (wgs * shares) : wgs >= cus ? (2 * at_once * cus + wgs - 1) / wgs : max(1L, at_once * cus / wgs);
        const float tile_us = d == 256 ? (shares > 1 ? 0.55f : 0.6f) : (shares > 1 ? 0.45f : 0.35f) * d / 128, whole_us = shares > 1 ? 0.f : d == 256 ? 1.5f : 0.5f, meet_us = (d == 256 ? 2.f : 0.6f) / shares, part_bytes = (float)rows * d * 4 / shares;
        for (long n = max(1L, min(min(room, tiles), (long)MOST_SEGMENTS));; n = (n + 1) / 2) {
            const long each = (tiles + n - 1) / n;
            const bool two = wgs * n * shares > cus;             // workgroups of a CU: they share what it has of loads in flight
            const float us = whole_us + tile_us * each * (!two ? 1.f : d == 64 ? 1.4f : 1.6f) + (two ? 0.5f : 0.f) + (each > 1 ? meet_us : 0.f) +
                             (n > 1 ? 1.f + 0.25f * nw + 0.7f * n * part_bytes / (nw * 8192) : 0.f);
            if (us < least) least = us, best = Split{(int)n, shares};
            if (n == 1) break;
        }
        if (shares == d / 64) break;
    }
    return best;
}

// keys and values of this many bytes go past the caches: what is read once a step would push out what is read again. One token over 131072 keys, 8 heads of 128 (512 MiB),
// 101 -> 91 us; 55 MB, which the memory-side cache holds from step to step, 14.2 us, and 16.9 past it.
constexpr size_t ONCE_BYTES = (size_t)192 << 20;

// Up to this capacity the workgroup that ends last adds up what the keys draw, in two rounds of its threads; past it a launch of its own does, which takes about five us more
// than no weights at whatever length. us a weighed token, within the launch / in one of their own / without weights: one head of 256 for 8, 500 keys 9.4 / 12.9 / 7.8, 2000 11.4 / 14.3 / 8.9,
// 4000 13.6 / 15.7 / 9.9, 8000 17.3 / 16.8 / 10.8; 8 heads of 128 for 32, 1000 keys 9.5 / 12.4 / 8.1, 2000 11.1 / 13.1 / 8.6, 4000 13.7 / 13.8 / 9.3, 8000 18.9 / 15.7 / 10.8.
constexpr int draws_keys(int d) { return wavefronts(d) * 64 * 4 * 2; }

}  // namespace

extern "C" int aionhip_step_attention_paged(aionhip_ctx *ctx, const aionhip_attention *p, const aionhip_paged_cache *c, aionhip_handle weights_before, aionhip_handle weights) {
    if (!ctx) return AIONHIP_INVALID_ARGUMENT;
    if (const int rc = paged::check_cache(ctx, "attention_paged", c)) return rc;
    if (!p || !p->out || !p->q) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention_paged: null operand");
    const size_t T = paged::capacity(c);
    if (p->k || p->v || p->rolling || p->batch != c->batch || p->t_kv != T || p->h_kv != c->h_kv || p->d_k != c->d || p->d_v != c->d || p->kv_dtype != c->dtype)
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention_paged: the step and the cache disagree (k and v 0, no ring; batch, capacity, heads, head size and dtype the cache's)");
    if (p->q_dtype != AIONHIP_F32 && p->q_dtype != AIONHIP_F16 && p->q_dtype != AIONHIP_BF16)
        return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: queries are f32, f16 or bf16, not dtype %d", p->q_dtype);
    if (p->h_q == 0 || p->h_q % p->h_kv != 0) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention_paged: h_q %zu is not a multiple of h_kv %zu", p->h_q, p->h_kv);
    if (weights_before && !weights) return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention_paged: weights to add to, and none to write");
    if (!p->batch || (!p->l_q && (!weights || weights == weights_before))) return AIONHIP_OK;
    const size_t groups = p->h_q / p->h_kv;
    if (p->h_q > 65535 || p->l_q > 0x7FFFFFFF / 16 / groups || p->batch * p->h_kv > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: dimension too large");
    const size_t rows = p->l_q * groups, units = p->batch * p->h_kv, q_bytes = units * rows * c->d * (p->q_dtype == AIONHIP_F32 ? 4 : 2), out_bytes = units * rows * c->d * 4;
    const size_t w_bytes = weights ? units * T * 4 : 0;
    if (paged::in_cache(c, p->out, out_bytes) || paged::in_cache(c, weights, w_bytes) || paged::overlap(p->out, out_bytes, p->q, q_bytes) ||
        paged::overlap(weights, w_bytes, p->out, out_bytes) || paged::overlap(weights, w_bytes, p->q, q_bytes) ||
        (weights_before != weights && paged::overlap(weights, w_bytes, weights_before, w_bytes)) || paged::overlap(p->out, out_bytes, weights_before, w_bytes) ||
        paged::overlap(p->out, out_bytes, p->kv_lengths, p->batch * 4) || paged::overlap(weights, w_bytes, p->kv_lengths, p->batch * 4) ||
        paged::overlap(p->out, out_bytes, p->query_positions, p->batch * p->l_q * 4) || paged::overlap(weights, w_bytes, p->query_positions, p->batch * p->l_q * 4))
        return set_err(ctx, AIONHIP_INVALID_ARGUMENT, "attention_paged: an operand that is written overlaps another");
    PagedArgs a{};
    a.out = (float *)(uintptr_t)p->out;
    a.q = (const void *)(uintptr_t)p->q;
    a.k = (const unsigned char *)(uintptr_t)c->k_pages;
    a.v = (const unsigned char *)(uintptr_t)c->v_pages;
    a.kv_lengths = (const int *)(uintptr_t)p->kv_lengths;
    a.positions = (const int *)(uintptr_t)p->query_positions;
    a.weights = (float *)(uintptr_t)weights;
    a.weights_before = (const float *)(uintptr_t)weights_before;
    a.table = paged::table_of(c);
    a.T = (int)T, a.L = (int)p->l_q, a.Hkv = (int)p->h_kv, a.groups = (int)groups, a.rows_total = (int)rows, a.row_tiles = (int)((rows + 15) / 16);
    a.tpad = (int)((T + TILE_KEYS - 1) / TILE_KEYS * TILE_KEYS);
    a.d = (int)c->d, a.q_dtype = p->q_dtype, a.kv_dtype = c->dtype;
    a.scale = p->scale, a.soft_cap = p->attn_logits_soft_cap;
    a.win_left = p->window_left, a.win_right = p->window_right, a.win_chunk = p->window_chunk;
    const bool none = p->l_q == 0;               // the weights stay what they were
    const bool fast = (c->d == 64 || c->d == 128 || c->d == 256) && (p->out & 15) == 0 && !none;
    a.nseg = a.shares = 1;
    bool once = false;
    if (fast) {
        // Behind a window there are no more keys than it shows to the call's consecutive queries.
        long keys = a.T;
        if (!a.positions && a.win_chunk == 0 && a.win_right < (unsigned)a.T && a.win_left < (unsigned)a.T) keys = min(keys, (long)a.win_left + (long)a.win_right + a.L + TILE_KEYS);
        const long cus = ctx->cu_count > 0 ? ctx->cu_count : 256, wgs = (long)units * a.row_tiles, tiles = (keys + TILE_KEYS - 1) / TILE_KEYS;
        const Split split = split_of(wgs, tiles, min(a.rows_total, 16), a.d, cus);
        a.nseg = split.segments, a.shares = split.shares;
        // Five queries of 32 sequences of up to 8192 keys, 32 heads on 8 of 128 (two row tiles), 237 -> 180 us (four queries, one tile, 156); 7 of 5 sequences of up to 62761, 310 -> 232. Shares
        // of few tiles do not wait for what places them: one token, one head of 256 for 8, 4096 keys 10.0 in plain order and 10.5 so, 32768 20.0 and 17.3.
        a.beside = a.row_tiles > 1 || (a.shares > 1 && tiles >= 8L * a.nseg);
        once = a.row_tiles == 1 && (size_t)units * keys * c->d * 4 >= ONCE_BYTES;
    }
    if ((fast ? (size_t)a.row_tiles * a.nseg * a.shares * (c->d == 256 ? wavefronts(256) : wavefronts(128)) * 64 : rows * 256) > paged::MAX_THREADS)
        return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: dimension too large");
    if (weights && rows && units > (((size_t)4 << 30) - 1) / (rows * a.tpad * 4))
        return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: the scores of %zu rows over %zu keys take 4 GiB or more; ask for weights with fewer queries", units * rows, T);
    a.streams = (int)(units * (size_t)a.nseg);
    a.draws = fast && weights && a.row_tiles == 1 && T <= (size_t)draws_keys(a.d) ? 1 : 0;
    const size_t meetings = a.nseg > 1 ? units * a.row_tiles * a.shares : 0, partial_bytes = meetings * a.nseg * (16 * c->d / a.shares + 32) * 4;
    const size_t stats_bytes = weights && !a.draws ? (units * rows * 8 + 255) / 256 * 256 : 0, scores_bytes = weights ? units * rows * a.tpad * 4 : 0;
    if (const int rc = ensure_scratch2(ctx, partial_bytes + stats_bytes + scores_bytes)) return rc;
    if (meetings) {
        if (const int rc = ensure_tickets(ctx, meetings * MEET_TICKET_WORDS * sizeof(unsigned))) return rc;
        a.tickets = (unsigned *)ctx->tickets;
        a.partial = (float *)ctx->scratch2;
    }
    if (weights) {
        a.stats = (float2 *)((char *)ctx->scratch2 + partial_bytes);
        a.scores = (float *)((char *)ctx->scratch2 + partial_bytes + stats_bytes);
    }
    if (fast) {
        if (const int rc = c->dtype == AIONHIP_F16 ? launch_head<AIONHIP_F16>(ctx, a, (int)p->batch, once) : launch_head<AIONHIP_BF16>(ctx, a, (int)p->batch, once)) return rc;
    } else if (!none) {
        ProfScope scope(ctx, "paged_generic");
        launch_k(ctx, paged_generic_kernel, dim3((unsigned)rows, (unsigned)p->h_kv, (unsigned)p->batch), dim3(256), 0, a);
        LAUNCH_CHECK(ctx, "paged_generic");
    }
    if (weights && !a.draws) {
        ProfScope scope(ctx, "paged_weights");
        // (measured at the kernel)
        const size_t keys = units * T >= WEIGH_MANY ? 4 : 1;
        launch_k(ctx, keys == 4 ? paged_weights_kernel<4, 4> : paged_weights_kernel<1, 8>, dim3((unsigned)((T + 256 * keys - 1) / (256 * keys)), (unsigned)p->h_kv, (unsigned)p->batch),
                 dim3(256), 0, a);
        LAUNCH_CHECK(ctx, none ? "paged_weights" : fast ? "paged_attn" : "paged_generic");
    }
    return AIONHIP_OK;
}
