// Key/value caches held in 8 or 4 bits: the layout, and the quantization of a block by the lanes that hold it (cache_quant.hip, attention_quant.hip).
//
// One buffer: codes [B][H][Tp][D * bits / 8], then scales [B][H][D / 32][Tp] f16, Tp = the capacity rounded up to 64 rows. A code is stored with its
// offset (q8_0: 128, q4_0: 8, the even element in the low half of the byte), an element is code * scale of its 32. Heads lie outside tokens and a
// block's scales run along the tokens, because a step reads one head's keys in order: 64 keys are then one contiguous run of codes, and the scales
// of sixteen neighbouring keys two 16-byte loads. The padding keeps a tile of 64 keys inside the buffer whatever the capacity.
#pragma once
#include "common.h"

namespace cq {

constexpr int TILE = 64;      // rows the capacity is rounded up to

inline size_t padded(size_t t_cap) { return (t_cap + TILE - 1) / TILE * TILE; }
inline size_t row_bytes(int dtype, size_t d) { return dtype == AIONHIP_Q8_0 ? d : d / 2; }
inline size_t codes_bytes(int dtype, size_t b, size_t t_cap, size_t h, size_t d) { return b * h * padded(t_cap) * row_bytes(dtype, d); }

// largest capacity, and the most heads and elements of a head, that the kernels' index arithmetic takes
constexpr size_t MAX_ROWS = 0x7FFFFFC0, MAX_HEADS = 65535, MAX_HEAD = 65504;

inline bool is_quant(int dtype) { return dtype == AIONHIP_Q8_0 || dtype == AIONHIP_Q4_0; }

struct Cache {
    unsigned char *codes;
    __half *scales;
};
inline Cache view(aionhip_handle cache, int dtype, size_t b, size_t t_cap, size_t h, size_t d) {
    unsigned char *p = (unsigned char *)(uintptr_t)cache;
    return Cache{p, (__half *)(p + codes_bytes(dtype, b, t_cap, h, d))};
}

// Eight elements of a block held by each of four neighbouring lanes. The arithmetic is the block quantizers' (quant.hip) but for one step: the scale is the
// maximum times the f32 nearest to 1 / 127 (1 / 7), a product in place of a quotient, which may differ in its last f32 bit and so, in one block of 15 000 (q4_0) or 3 million (q8_0), by the
// last bit of the f16. q8_0 codes go by the scale as it is stored, q4_0 codes by the scale before it is rounded, halves are rounded away from zero. A block that holds an infinity or a NaN gets
// a NaN as its scale, so that reading it back says so: a maximum alone would drop the NaN and store a number in its place.
template <int DT>
__device__ __forceinline__ void quantize8(const float (&x)[8], unsigned (&word)[2], __half &scale) {
    float amax = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        amax = fmaxf(amax, fabsf(x[i]));
        odd |= !(fabsf(x[i]) < INFINITY);
    }
    int odd_i = odd ? 1 : 0;
    amax = fmaxf(amax, dpp_f<DPP_QUAD_XOR1>(amax));
    amax = fmaxf(amax, dpp_f<DPP_QUAD_XOR2>(amax));
    odd_i |= dpp_i<DPP_QUAD_XOR1>(odd_i);
    odd_i |= dpp_i<DPP_QUAD_XOR2>(odd_i);
    constexpr float STEP = DT == AIONHIP_Q8_0 ? 1.f / 127.f : 1.f / 7.f;
    const float full = amax == 0.f ? 1.f : amax * STEP;
    scale = odd_i ? __ushort_as_half((unsigned short)0x7E00) : __float2half_rn(full);
    word[0] = word[1] = 0u;
    if constexpr (DT == AIONHIP_Q8_0) {
        const float eff = __half2float(scale);
        const float inv = (amax == 0.f || eff == 0.f) ? 0.f : 1.f / eff;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int q = (int)fminf(127.f, fmaxf(-128.f, roundf(x[i] * inv))) + 128;
            word[i >> 2] |= (unsigned)q << (8 * (i & 3));
        }
    } else {
        // the quotient by the reciprocal, within 2e-6: it rounds as the exact one does but beside a half, and there (3 elements in 100 000) and where the reciprocal
        // may leave f32's range the divisions are made
        float c[8];
        const float inv = __builtin_amdgcn_rcpf(full);
        bool near = !(full > 1e-36f && full < 1e36f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = x[i] * inv;
            c[i] = rintf(t);
            near |= fabsf(t - c[i]) > 0.49999f;
        }
        if (__any(near)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = roundf(x[i] / full);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) word[0] |= (unsigned)((int)fminf(7.f, fmaxf(-8.f, c[i])) + 8) << (4 * i);
    }
}

}  // namespace cq
