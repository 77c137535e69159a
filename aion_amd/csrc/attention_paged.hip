// Attention over caches in pages (the layout: cache_paged.h): one to a few tokens a sequence, f32 accuracy, and with it what each key's probabilities add up to.
//
// paged_attn_kernel - head sizes 64, 128, 256. A workgroup has sixteen query rows of one KV head (position-major, query head fastest) and one segment of their keys; its
//   wavefronts take tiles of 32 keys in turn:
//       S^T[keys x rows] = K[keys x d] . Q^T[d x rows]          O^T[d x rows] += V^T[d x keys] . P^T[keys x rows]
//   K goes from the pages to registers in the order the matrix instruction wants it, V through LDS, where it is read transposed. Sixteen keys lie in one page, so a
//   page number is a scalar to each half tile: a lane fetches one of the next 64, and they become addresses without a load in between.
//   Accuracy: q and P enter the products as sums of halves (two f16, three bf16; q that comes in the cache's type as it is), K and V are exact, sums are f32.
// paged_merge_kernel - adds the segments of a row, and forms the keys' weights from the scores that the first kernel left.
// paged_generic_kernel - other head sizes: a wavefront a key at a time, f32. It is there so that every shape has a path.
#include "attention_common.h"
#include "cache_paged.h"

#include <type_traits>

namespace {
using namespace attn;
using paged::Table;

constexpr float MASKED = -INFINITY;
// Probabilities are held as 2^(s - ref + HEAD_ROOM), the reference being raised only when a score passes it by more than SLACK: 2^14 at most fits f16, and what f16
// pairs round away lies 2^-31 below the largest.
constexpr float HEAD_ROOM = 6.f, SLACK = 8.f;
// A number becomes a sum of halves that all have its sign and are not zero, each but the last taken from slightly less than what is left: an infinite key or value then
// has products of one sign, and no zero times infinity, as the number itself has.
template <int KV> constexpr float LESS = KV == AIONHIP_F16 ? 1.f - 0x1p-11f : 1.f - 0x1p-8f;

struct PagedArgs {
    float *out, *partial, *scores;
    const float *weights_before;
    float *weights;
    float2 *stats;            // [unit][padded rows][nseg] reference (log2) and sum
    Table table;
    int T, tpad, L, Hkv, groups, rows_total, row_tiles, nseg;
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

template <int D>
struct Cfg {
    static constexpr int NW = D == 256 ? 4 : 8;
    static constexpr int ROW = D * 2, TILE = TILE_KEYS * ROW;
    static constexpr int SLOT = 16 * (D + 4) + 32;               // a wavefront's results in the merge: [16][D + 4], 16 references, 16 sums
    static constexpr int MERGE = NW * SLOT * 4, LDS = NW * TILE > MERGE ? NW * TILE : MERGE;
};
// tiles of a segment: the tiles are dealt out evenly, no fewer than one to a wavefront
__device__ __forceinline__ int tiles_each(int tiles, int nseg, int nw) { return max(nw, (tiles + nseg - 1) / nseg); }

// Q parts: how many halves a query element is the sum of
template <int KV, int D, int QP, bool WEIGH>
__global__ __launch_bounds__(Cfg<D>::NW * 64) void paged_attn_kernel(PagedArgs a) {
    using C = Cfg<D>;
    constexpr int NW = C::NW, KK = D / 32, MT = D / 16;
    constexpr int PP = KV == AIONHIP_F16 ? 2 : 3;                // parts of a probability
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int rt = blockIdx.x / a.nseg, seg = blockIdx.x - rt * a.nseg, hk = blockIdx.y, b = blockIdx.z;
    const int unit = b * a.Hkv + hk;
    const int r = rt * 16 + n;
    const bool row_ok = r < a.rows_total;
    const int li = row_ok ? r / a.groups : 0, gi = row_ok ? r - li * a.groups : 0;
    int lo, hi;
    row_keys(a, b, li, a.kv_lengths ? a.kv_lengths[b] : 0, a.positions ? a.positions[(size_t)b * a.L + li] : 0, lo, hi);
    if (!row_ok) lo = hi = 0;
    const bool some = hi > lo;
    const int uni_lo = rows16_min_i(some ? lo : INT_MAX), uni_hi = rows16_max_i(some ? hi : 0);
    // keys that every row sees
    const int all_lo = rows16_max_i(row_ok ? (some ? lo : INT_MAX) : 0), all_hi = rows16_min_i(row_ok ? (some ? hi : 0) : INT_MAX);

    // ---- the queries
    const size_t qbase = (((size_t)b * a.L + li) * (a.Hkv * a.groups) + hk * a.groups + gi) * D;
    u32x4 qf[QP][KK];
    float to_score = 1.f;                                        // a product's sum times this is q . k
    if constexpr (QP == 1) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            __builtin_memcpy(&qf[0][kk], (const unsigned short *)a.q + qbase + kk * 32 + g * 8, 16);
            if (!row_ok) qf[0][kk] = u32x4{0u, 0u, 0u, 0u};
        }
    } else {
        float x[KK][8];
        float top = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const size_t at = qbase + kk * 32 + g * 8;
            if (a.q_dtype == AIONHIP_F32) {
                __builtin_memcpy(x[kk], (const float *)a.q + at, 32);
            } else {
                unsigned short h[8];
                __builtin_memcpy(h, (const unsigned short *)a.q + at, 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[kk][j] = a.q_dtype == AIONHIP_F16 ? __half2float(__ushort_as_half(h[j])) : bf16_bits_to_f32(h[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (!row_ok) x[kk][j] = 0.f;
                top = fmaxf(top, fabsf(x[kk][j]));
            }
        }
        float factor = 1.f;
        if constexpr (KV == AIONHIP_F16) {
            // a row goes into f16's range by a power of two that takes its largest element to 2^10: what the second half rounds away then lies 2^-35 below that
            top = groups4_max(top);
            const int e = (int)(__float_as_uint(top) >> 23);
            const int f = e == 255 ? 127 : max(1, min(264 - e, 253));
            factor = __uint_as_float((unsigned)f << 23);
            to_score = __uint_as_float((unsigned)(254 - f) << 23);
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float u = x[kk][j] * factor, w = x[kk][j + 1] * factor;
#pragma unroll
                for (int p = 0; p < QP; ++p) {
                    const unsigned both = p + 1 < QP ? pack2<KV>(u * LESS<KV>, w * LESS<KV>) : pack2<KV>(u, w);
                    qf[p][kk][j / 2] = both;
                    // (an infinite element has no rest)
                    const float ru = u - from_half_bits<KV>((unsigned short)both), rw = w - from_half_bits<KV>((unsigned short)(both >> 16));
                    u = fabsf(ru) < INFINITY ? ru : u;
                    w = fabsf(rw) < INFINITY ? rw : w;
                }
            }
    }
    const float to_log2 = a.soft_cap > 0.f ? to_score * (a.scale / a.soft_cap) : to_score * (a.scale * LOG2E), cap_log2 = a.soft_cap * LOG2E;

    // ---- this wavefront's tiles
    int t_begin = 0, t_end = 0;
    if (uni_hi > uni_lo) {
        const int tb = uni_lo / TILE_KEYS, te = (uni_hi + TILE_KEYS - 1) / TILE_KEYS, per = tiles_each(te - tb, a.nseg, NW);
        t_begin = tb + seg * per;
        t_end = min(t_begin + per, te);
    }
    if (t_begin >= t_end && (seg > 0 || a.nseg > 1)) return;     // (the merge counts the segments that have tiles)
    t_begin += wave;
    const int steps = t_begin < t_end ? (t_end - t_begin + NW - 1) / NW : 0;

    unsigned char *vs = lds + wave * C::TILE;
    const size_t page_bytes = ((size_t)a.Hkv << a.table.shift) * C::ROW, head_bytes = ((size_t)hk << a.table.shift) * C::ROW;
    const unsigned char *kp = a.k + head_bytes, *vp = a.v + head_bytes;
    const int row_mask = (1 << a.table.shift) - 1;
    const int *pages = a.table.pages + (size_t)b * a.table.width;
    // the pages of the half tiles of 32 steps, one to a lane; -1: none
    auto fetch_pages = [&](int step0) __attribute__((always_inline)) {
        const int tile = t_begin + (step0 + (lane >> 1)) * NW, e = (tile * TILE_KEYS + (lane & 1) * 16) >> a.table.shift;
        int id = -1;
        if (tile < t_end && e < a.table.width) id = pages[e];
        return (unsigned)id < (unsigned)a.table.count ? id : -1;
    };
    u32x4 kf[2][KK];
    auto load_k = [&](int t, int id0, int id1) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned char *at = kp + (size_t)(unsigned)max(h ? id1 : id0, 0) * page_bytes + (size_t)((t * TILE_KEYS + h * 16) & row_mask) * C::ROW;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) kf[h][kk] = *(const u32x4 *)(at + (unsigned)(n * C::ROW + g * 16) + kk * 64);
        }
    };
    // V: 1 KiB an instruction, straight into LDS. 16-byte chunk c of key k lies at slot c ^ (2 * ((k >> 2) & 3)) ^ (8 * (k & 1)) of its row (the last term for rows
    // of 256 bytes and more), so that the sixteen keys of a transposing read fall on distinct banks.
    constexpr int NVI = C::TILE / 1024, KEYS_PER_VI = 1024 / C::ROW;
    const int v_key_in = (lane * 16) / C::ROW, v_slot = ((lane * 16) % C::ROW) / 16;
    (void)v_key_in; (void)v_slot; (void)vp; (void)NVI; (void)KEYS_PER_VI;
    auto load_v = [&](int t, int id0, int id1) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned char *at = vp + (size_t)(unsigned)max(h ? id1 : id0, 0) * page_bytes + (size_t)((t * TILE_KEYS + h * 16) & row_mask) * C::ROW;
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, 16 * C::ROW, 0x00027000);
#pragma unroll
            for (int i = 0; i < NVI / 2; ++i) {
                const int key = i * KEYS_PER_VI + v_key_in;
                const int chunk = v_slot ^ (2 * ((key >> 2) & 3)) ^ (D >= 128 ? 8 * (key & 1) : 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(vs + (h * (NVI / 2) + i) * 1024), 16, key * C::ROW + chunk * 16, 0, 0, 0);
            }
        }
#endif
    };
    const int tr_r = (lane >> 2) & 3, tr_q = lane & 3;
    const unsigned v_rowaddr = (unsigned)(size_t)(lds_void *)vs + (unsigned)((4 * g + tr_r) * C::ROW + (tr_q & 1) * 8);
    const unsigned v_slot_l = (unsigned)(((tr_q >> 1) ^ (2 * g) ^ (D >= 128 ? 8 * (tr_r & 1) : 0)) << 4);
    auto v_operand = [&](auto mt_c) __attribute__((always_inline)) {
        constexpr int mt = decltype(mt_c)::value;
        const unsigned addr = v_rowaddr + (v_slot_l ^ (unsigned)(mt << 5));
        u32x2 a0, a1;
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3" : "=&v"(a0), "=&v"(a1) : "v"(addr), "n"(16 * C::ROW) : "memory");
        return u32x4{a0.x, a0.y, a1.x, a1.y};
    };

    f32x4 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = MASKED, l_run = 0.f;                             // l_run: of this lane's keys
    float *scores = WEIGH ? a.scores + ((size_t)unit * a.rows_total + r) * a.tpad : nullptr;

    // MORE: another tile of this wavefront follows (two copies of the body, so that every path requests K and V in the same order and the count of loads in flight holds)
    auto tile = [&](int t, bool ok0, bool ok1, int next0, int next1, auto more_c) __attribute__((always_inline)) {
        constexpr bool more = decltype(more_c)::value;
        const int key0 = t * TILE_KEYS;
        f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int p = 0; p < QP; ++p)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[h] = mfma16<KV>(kf[h][kk], qf[p][kk], s[h]);
        const bool full = key0 >= all_lo && key0 + TILE_KEYS <= all_hi && ok0 && ok1;      // every row sees every key
        // lane: keys key0 + h * 16 + g * 4 + i of row n
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = s[j >> 2][j & 3] * to_log2;
        if (a.soft_cap > 0.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = cap_log2 * tanhf(p[j]);
        }
        unsigned seen = 0xFF;
        if (!full) {
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = key0 + (j >> 2) * 16 + g * 4 + (j & 3);
                const bool see = key >= lo && key < hi && (j < 4 ? ok0 : ok1);
                p[j] = see ? p[j] : MASKED;
                seen |= see ? 1u << j : 0u;
            }
        }
        if constexpr (WEIGH) {
            if (row_ok) {
                *(f32x4 *)(scores + key0 + g * 4) = f32x4{p[0], p[1], p[2], p[3]};
                *(f32x4 *)(scores + key0 + 16 + g * 4) = f32x4{p[4], p[5], p[6], p[7]};
            }
        }
        if (more) {
            load_k(t + NW, next0, next1);
            asm volatile("" ::: "memory");         // requested here, ahead of the counted wait for V below
        }
        float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        mx = groups4_max(mx);
        if (__any(mx > ref + SLACK)) {
            const float ref_new = fmaxf(ref, mx), alpha = ref > MASKED ? __builtin_amdgcn_exp2f(ref - ref_new) : 0.f;
            if (ref_new > ref) {
                l_run *= alpha;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt] *= alpha;
                ref = ref_new;
            }
        }
        const float base = (ref > MASKED ? ref : 0.f) - HEAD_ROOM;
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
                const unsigned both = part + 1 < PP ? pack2<KV>(u * LESS<KV>, w * LESS<KV>) : pack2<KV>(u, w);
                pf[part][j / 2] = both;
                u -= from_half_bits<KV>((unsigned short)both);
                w -= from_half_bits<KV>((unsigned short)(both >> 16));
            }
        }
        // V has landed once only the younger K loads are outstanding (loads complete in order); the tile is this wavefront's alone
        if (more) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * KK));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        asm volatile("" ::: "memory");
        bool odd = false;
        if (!full) {
            // Rows that no query sees count as zeros (they may hold anything, and zero times that need not be zero). Where a row is seen by some and not finite, the
            // queries are taken one by one below.
#pragma unroll
            for (int i = 0; i < NVI; ++i) {
                const int key = key0 + i * KEYS_PER_VI + v_key_in;
                u32x4 *at = (u32x4 *)(vs + i * 1024 + lane * 16);
                if (key < uni_lo || key >= uni_hi || !(i < NVI / 2 ? ok0 : ok1)) {
                    *at = u32x4{0u, 0u, 0u, 0u};
                } else {
                    constexpr unsigned EXP = KV == AIONHIP_F16 ? 0x7C00u : 0x7F80u;
                    const u32x4 x = *at;
#pragma unroll
                    for (int j = 0; j < 4; ++j) odd |= (x[j] & EXP) == EXP || (x[j] >> 16 & EXP) == EXP;
                }
            }
            odd = __any(odd);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        if (!odd) {
            constexpr int VA = MT < 4 ? MT : 4;                  // operands requested ahead
            u32x4 vop[VA];
            static_for<0, VA>([&](auto mc) __attribute__((always_inline)) { vop[decltype(mc)::value] = v_operand(mc); });
            static_for<0, MT>([&](auto mc) __attribute__((always_inline)) {
                constexpr int mt = decltype(mc)::value;
                constexpr int later = MT - 1 - mt < VA - 1 ? MT - 1 - mt : VA - 1;
                asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(vop[mt % VA]) : "n"(2 * later));
#pragma unroll
                for (int part = 0; part < PP; ++part) acc[mt] = mfma16<KV>(vop[mt % VA], pf[part], acc[mt]);
                if constexpr (mt + VA < MT) vop[mt % VA] = v_operand(std::integral_constant<int, mt + VA>{});
            });
        } else {
            // a query at a time, with zeros for the keys that it does not see, into that query's sums alone
            for (int q = 0; q < 16; ++q) {
                const unsigned mine = (unsigned)__shfl((int)seen, (lane & 48) + q, 64);
                static_for<0, MT>([&](auto mc) __attribute__((always_inline)) {
                    constexpr int mt = decltype(mc)::value;
                    u32x4 v = v_operand(mc);
                    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v));
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] &= (mine >> (2 * j) & 1u ? 0xFFFFu : 0u) | (mine >> (2 * j + 1) & 1u ? 0xFFFF0000u : 0u);
                    f32x4 c = acc[mt];
#pragma unroll
                    for (int part = 0; part < PP; ++part) c = mfma16<KV>(v, pf[part], c);
                    if (n == q) acc[mt] = c;
                });
            }
        }
        if (more) {
            asm volatile("" ::: "memory");         // the operand reads above are complete: each was waited for before its product
            load_v(t + NW, next0, next1);
        }
    };
    if (steps > 0) {
        int ids = fetch_pages(0);
        int id0 = __builtin_amdgcn_readlane(ids, 0), id1 = __builtin_amdgcn_readlane(ids, 1);
        load_k(t_begin, id0, id1);
        load_v(t_begin, id0, id1);
        int t = t_begin;
        for (int i = 1; i < steps; ++i, t += NW) {
            if ((i & 31) == 0) ids = fetch_pages(i);
            const int next0 = __builtin_amdgcn_readlane(ids, 2 * (i & 31)), next1 = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + 1);
            tile(t, id0 >= 0, id1 >= 0, next0, next1, std::true_type{});
            id0 = next0, id1 = next1;
        }
        tile(t, id0 >= 0, id1 >= 0, 0, 0, std::false_type{});
    }
    l_run = groups4_sum(l_run);

    // ---- the wavefronts meet in LDS
    __syncthreads();
    float *mg = (float *)lds;
    {
        float *w = mg + wave * C::SLOT;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) *(f32x4 *)(w + n * (D + 4) + mt * 16 + g * 4) = acc[mt];
        if (g == 0) { w[16 * (D + 4) + n] = ref; w[16 * (D + 4) + 16 + n] = l_run; }
    }
    __syncthreads();
    const bool alone = !WEIGH && a.nseg == 1;
    for (int e = threadIdx.x; e < 16 * D / 4; e += NW * 64) {
        const int row = e / (D / 4), col = (e % (D / 4)) * 4, rr = rt * 16 + row;
        if (rr >= a.rows_total) break;
        float top = MASKED, l = 0.f;
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, mg[w * C::SLOT + 16 * (D + 4) + row]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float rw = mg[w * C::SLOT + 16 * (D + 4) + row];
            // (a wavefront without a reference has seen nothing, or what is not a number: its sums then say so)
            const float f = rw > MASKED ? __builtin_amdgcn_exp2f(rw - top) : 1.f;
            l += mg[w * C::SLOT + 16 * (D + 4) + 16 + row] * f;
            o += *(const f32x4 *)(mg + w * C::SLOT + row * (D + 4) + col) * f;
        }
        if (alone) {
            const int l2 = rr / a.groups, g2 = rr - l2 * a.groups;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            *(f32x4 *)(a.out + (((size_t)b * a.L + l2) * (a.Hkv * a.groups) + hk * a.groups + g2) * D + col) = o * inv;
        } else {
            *(f32x4 *)(a.partial + (((size_t)(unit * a.row_tiles + rt) * a.nseg + seg) * 16 + row) * D + col) = o;
            if (col == 0) a.stats[((size_t)unit * a.rows_total + rr) * a.nseg + seg] = float2{top, l};
        }
    }
}

// How many segments of a row's tile have tiles; every row of the tile agrees on it.
__device__ __forceinline__ int segments_of(const PagedArgs &a, int b, int rt, int nw) {
    int uni_lo = INT_MAX, uni_hi = 0;
    const int len = a.kv_lengths ? a.kv_lengths[b] : 0;
    for (int i = 0; i < 16; ++i) {
        const int r = rt * 16 + i;
        if (r >= a.rows_total) break;
        int lo, hi;
        const int li = r / a.groups;
        row_keys(a, b, li, len, a.positions ? a.positions[(size_t)b * a.L + li] : 0, lo, hi);
        if (hi > lo) uni_lo = min(uni_lo, lo), uni_hi = max(uni_hi, hi);
    }
    if (uni_hi <= uni_lo) return 0;
    const int tiles = (uni_hi + TILE_KEYS - 1) / TILE_KEYS - uni_lo / TILE_KEYS, per = tiles_each(tiles, a.nseg, nw);
    return (tiles + per - 1) / per;
}

// The first merge_rows workgroups of a unit add the segments of a row each, the others (where weights are asked for) have 1024 keys each.
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a, int nw, int merge_rows) {
    __shared__ float red[256];
    __shared__ __attribute__((aligned(16))) f32x4 s_o[256];
    const int hk = blockIdx.y, b = blockIdx.z, unit = b * a.Hkv + hk, tid = threadIdx.x;
    if ((int)blockIdx.x < merge_rows) {
        const int r = blockIdx.x, rt = r >> 4, nseg = segments_of(a, b, rt, nw);
        const float2 *st = a.stats + ((size_t)unit * a.rows_total + r) * a.nseg;
        const int per = a.d / 4, sets = 256 / per, set = tid / per, col = (tid - set * per) * 4;
        float top = MASKED;
        for (int s = 0; s < nseg; ++s) top = fmaxf(top, st[s].x);
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
        for (int s = set; s < nseg; s += sets) {
            const float f = st[s].x > MASKED ? __builtin_amdgcn_exp2f(st[s].x - top) : 1.f;
            l += st[s].y * f;
            o += *(const f32x4 *)(a.partial + (((size_t)(unit * a.row_tiles + rt) * a.nseg + s) * 16 + (r & 15)) * a.d + col) * f;
        }
        s_o[tid] = o;
        red[tid] = l;
        __syncthreads();
        if (set > 0) return;
        for (int i = 1; i < sets; ++i) o += s_o[i * per + tid], l += red[i * per + tid];
        const int l2 = r / a.groups, g2 = r - l2 * a.groups;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *(f32x4 *)(a.out + (((size_t)b * a.L + l2) * (a.Hkv * a.groups) + hk * a.groups + g2) * a.d + col) = o * inv;
        return;
    }
    const int key = ((int)blockIdx.x - merge_rows) * 1024 + tid * 4;
    __shared__ float s_top[16], s_inv[16];
    __shared__ int s_lo[16], s_hi[16];
    f32x4 w = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int rt = 0; rt < (a.rows_total + 15) / 16; ++rt) {
        const int nseg = segments_of(a, b, rt, nw);
        __syncthreads();
        if (tid < 16) {
            const int r = rt * 16 + tid;
            int lo = 0, hi = 0;
            float top = MASKED, l = 0.f;
            if (r < a.rows_total) {
                const int li = r / a.groups;
                row_keys(a, b, li, a.kv_lengths ? a.kv_lengths[b] : 0, a.positions ? a.positions[(size_t)b * a.L + li] : 0, lo, hi);
                const float2 *st = a.stats + ((size_t)unit * a.rows_total + r) * a.nseg;
                for (int s = 0; s < nseg; ++s) top = fmaxf(top, st[s].x);
                for (int s = 0; s < nseg; ++s) l += st[s].y * (st[s].x > MASKED ? __builtin_amdgcn_exp2f(st[s].x - top) : 1.f);
            }
            s_lo[tid] = lo, s_hi[tid] = hi;
            s_top[tid] = (top > MASKED ? top : 0.f) - HEAD_ROOM;
            s_inv[tid] = l == 0.f ? 0.f : 1.f / l;
        }
        __syncthreads();
        if (key < a.T)
            for (int i = 0; i < 16 && rt * 16 + i < a.rows_total; ++i) {
                if (key >= s_hi[i] || key + 4 <= s_lo[i]) continue;
                const f32x4 s = *(const f32x4 *)(a.scores + ((size_t)unit * a.rows_total + rt * 16 + i) * a.tpad + key);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (key + j >= s_lo[i] && key + j < s_hi[i]) w[j] += __builtin_amdgcn_exp2f(s[j] - s_top[i]) * s_inv[i];
            }
    }
    if (key < a.T) {                             // (a capacity is a multiple of sixteen)
        const size_t at = (size_t)unit * a.T + key;
        if (a.weights_before)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] += a.weights_before[at + j];
#pragma unroll
        for (int j = 0; j < 4; ++j) a.weights[at + j] = w[j];
    }
}

// One workgroup a query row, any head size: its four wavefronts take keys in turn.
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
        const float alpha = ref > MASKED ? __builtin_amdgcn_exp2f(ref - top) : 1.f, p = __builtin_amdgcn_exp2f(s - (top > MASKED ? top : 0.f));
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
    if (a.stats && threadIdx.x == 0) a.stats[(size_t)unit * a.rows_total + r] = float2{top, sum * __builtin_amdgcn_exp2f(HEAD_ROOM)};
}

template <int KV, int D, int QP>
int launch(aionhip_ctx *ctx, const PagedArgs &a, int batch) {
    ProfScope scope(ctx, "paged_attn");
    const dim3 grid((unsigned)(a.row_tiles * a.nseg), (unsigned)a.Hkv, (unsigned)batch), block(Cfg<D>::NW * 64);
    static std::atomic<uint64_t> attr[2];
    const void *fn = a.weights ? (const void *)paged_attn_kernel<KV, D, QP, true> : (const void *)paged_attn_kernel<KV, D, QP, false>;
    if (const int rc = allow_lds(ctx, attr[a.weights ? 1 : 0], fn, Cfg<D>::LDS)) return rc;
    if (a.weights) launch_k(ctx, paged_attn_kernel<KV, D, QP, true>, grid, block, Cfg<D>::LDS, a);
    else launch_k(ctx, paged_attn_kernel<KV, D, QP, false>, grid, block, Cfg<D>::LDS, a);
    LAUNCH_CHECK(ctx, "paged_attn");
    return AIONHIP_OK;
}
template <int KV, int D>
int launch_parts(aionhip_ctx *ctx, const PagedArgs &a, int batch) {
    if (a.q_dtype == KV) return launch<KV, D, 1>(ctx, a, batch);
    return launch<KV, D, KV == AIONHIP_F16 ? 2 : 3>(ctx, a, batch);
}
template <int KV>
int launch_head(aionhip_ctx *ctx, const PagedArgs &a, int batch) {
    if (a.d == 64) return launch_parts<KV, 64>(ctx, a, batch);
    if (a.d == 128) return launch_parts<KV, 128>(ctx, a, batch);
    return launch_parts<KV, 256>(ctx, a, batch);
}

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
    if (!p->batch || !p->l_q) return AIONHIP_OK;
    const size_t groups = p->h_q / p->h_kv;
    if (p->h_q > 65535 || p->l_q > 0x7FFFFFFF / 16 / groups || p->batch * p->h_kv > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: dimension too large");
    const size_t rows = p->l_q * groups, units = p->batch * p->h_kv, q_bytes = units * rows * c->d * (p->q_dtype == AIONHIP_F32 ? 4 : 2), out_bytes = units * rows * c->d * 4;
    const size_t w_bytes = weights ? units * T * 4 : 0;
    if (paged::in_cache(c, p->out, out_bytes) || paged::in_cache(c, weights, w_bytes) || paged::overlap(p->out, out_bytes, p->q, q_bytes) ||
        paged::overlap(weights, w_bytes, p->out, out_bytes) || paged::overlap(weights, w_bytes, p->q, q_bytes) ||
        (weights_before != weights && paged::overlap(weights, w_bytes, weights_before, w_bytes)) || paged::overlap(p->out, out_bytes, weights_before, w_bytes))
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
    const bool fast = (c->d == 64 || c->d == 128 || c->d == 256) && (p->out & 15) == 0;
    const int nw = c->d == 256 ? 4 : 8;
    a.nseg = 1;
    if (fast) {
        // Behind a window there are no more keys than it shows to the call's consecutive queries.
        long keys = a.T;
        if (!a.positions && a.win_chunk == 0 && a.win_right < (unsigned)a.T && a.win_left < (unsigned)a.T) keys = min(keys, (long)a.win_left + (long)a.win_right + a.L + TILE_KEYS);
        const long cus = ctx->cu_count > 0 ? ctx->cu_count : 256, wgs = (long)units * a.row_tiles;
        a.nseg = (int)max(1L, min(min((4 * cus + wgs - 1) / wgs, (keys + nw * TILE_KEYS - 1) / (nw * TILE_KEYS)), 256L));
    }
    if ((size_t)a.row_tiles * a.nseg > 0x7FFFFFFF) return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: dimension too large");
    const bool merge = fast && (a.nseg > 1 || weights);
    const size_t partial_bytes = merge ? units * a.row_tiles * a.nseg * 16 * c->d * 4 : 0, stats_bytes = merge || weights ? (units * rows * a.nseg * 8 + 255) / 256 * 256 : 0;
    if (weights && units > ((size_t)4 << 30) / (rows * a.tpad * 4))
        return set_err(ctx, AIONHIP_UNSUPPORTED, "attention_paged: the scores of %zu rows over %zu keys take more than 4 GiB; ask for weights with fewer queries", units * rows, T);
    const size_t scores_bytes = weights ? units * rows * a.tpad * 4 : 0;
    if (const int rc = ensure_scratch2(ctx, partial_bytes + stats_bytes + scores_bytes)) return rc;
    if (merge || weights) {
        a.stats = (float2 *)ctx->scratch2;
        a.partial = (float *)((char *)ctx->scratch2 + stats_bytes);
        a.scores = weights ? (float *)((char *)ctx->scratch2 + stats_bytes + partial_bytes) : nullptr;
    }
    if (fast) {
        if (const int rc = c->dtype == AIONHIP_F16 ? launch_head<AIONHIP_F16>(ctx, a, (int)p->batch) : launch_head<AIONHIP_BF16>(ctx, a, (int)p->batch)) return rc;
    } else {
        ProfScope scope(ctx, "paged_generic");
        launch_k(ctx, paged_generic_kernel, dim3((unsigned)rows, (unsigned)p->h_kv, (unsigned)p->batch), dim3(256), 0, a);
        LAUNCH_CHECK(ctx, "paged_generic");
    }
    if (merge || weights) {
        ProfScope scope(ctx, "paged_merge");
        const unsigned merge_rows = fast ? (unsigned)rows : 0, chunks = weights ? (unsigned)((T + 1023) / 1024) : 0;
        launch_k(ctx, paged_merge_kernel, dim3(merge_rows + chunks, (unsigned)p->h_kv, (unsigned)p->batch), dim3(256), 0, a, nw, (int)merge_rows);
        LAUNCH_CHECK(ctx, fast ? "paged_attn" : "paged_generic");
    }
    return AIONHIP_OK;
}
