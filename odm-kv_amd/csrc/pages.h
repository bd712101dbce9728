// The paged 8-bit cache's layout and conversions, shared by its kernels (pages.hip, attend.hip).
#pragma once

#include "common.h"

#define BLOCK_TOKENS TILE                       // tokens of a block = of a page = of a tail
#define PAGE_BYTES (BLOCK_TOKENS * HD)          // codes of a page and head, keys or values
#define TAIL_ELEMS (BLOCK_TOKENS * HD)
#define MAX_ROWS 1024                           // rows of a cache: the bookkeeping runs in one workgroup, a thread a row

// status words
#define ST_FREE 0                               // pages that no row holds
#define ST_HINT 1                               // no page below this one is free
#define ST_REFUSED 2                            // set when a call was refused on the device
#define ST_LIVE 3                               // pages in use, as the last compaction counted them

__host__ __device__ static inline size_t page_at(const odmkv_pages_t& p, int layer, int page, int h) {
    return (((size_t)layer * p.pages + page) * p.Hkv + h) * PAGE_BYTES;
}
__host__ __device__ static inline size_t scale_at(const odmkv_pages_t& p, int layer, int page, int h) {
    return ((size_t)layer * p.pages + page) * p.Hkv + h;
}
__host__ __device__ static inline size_t tail_at(const odmkv_pages_t& p, int layer, int slot, int h) {
    return (((size_t)layer * p.rows + slot) * p.Hkv + h) * TAIL_ELEMS;
}

// what is not finite is stored as 0, two 16-bit values at a time
template <int DT>
__device__ static inline uint32_t finite_pair(uint32_t w) {
    constexpr uint32_t E = DT == ODMKV_F16 ? 0x7c00u : 0x7f80u;
    if ((w & E) == E) w &= 0xffff0000u;
    if ((w & (E << 16)) == (E << 16)) w &= 0x0000ffffu;
    return w;
}
template <int DT>
__device__ static inline uint4 finite8(uint4 v) {
    return make_uint4(finite_pair<DT>(v.x), finite_pair<DT>(v.y), finite_pair<DT>(v.z), finite_pair<DT>(v.w));
}
// the largest of |x| of a pair, as the bits of a 16-bit number (finite values order as their bits do)
__device__ static inline uint32_t abs_max_pair(uint32_t w) { return max(w & 0x7fffu, (w >> 16) & 0x7fffu); }

// The scale of a block whose largest |x| is a: the smallest number of 8 significant bits that is not below a / top.  x (11 bits at
// the most) over s (8 bits) is either exactly half-way between two codes or off it by 2^-13 of itself, so that any quotient good to
// 2^-22 rounds to the right code, if only exact quotients come out exact.
template <int KIND>
__device__ static inline float block_scale(float a) {
    if (!(a > 0.0f)) return 0.0f;
    const float q = __fdiv_rn(a, KIND == ODMKV_E4M3 ? 448.0f : 127.0f);
    return fmaxf(__uint_as_float((__float_as_uint(q) + 0xffffu) & 0xffff0000u), 0x1p-100f);
}
// four values to four codes; inv = 1 / s (0 where s is 0).  The correction makes exact quotients exact.
template <int KIND>
__device__ static inline uint32_t codes4(float x0, float x1, float x2, float x3, float s, float inv) {
    const auto over = [&](float x) {
        const float y = x * inv;
        return __fmaf_rn(__fmaf_rn(-y, s, x), inv, y);
    };
    if constexpr (KIND == ODMKV_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(over(x0), over(x1), 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(over(x2), over(x3), w, true);
    } else {
        const auto byte = [&](float x) { return (uint32_t)(int)rintf(over(x)) & 0xffu; };
        return byte(x0) | byte(x1) << 8 | byte(x2) << 16 | byte(x3) << 24;
    }
}
// four codes as numbers
template <int KIND>
__device__ static inline void values4(uint32_t w, float* x) {
    if constexpr (KIND == ODMKV_E4M3) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
    }
}
// to 16 bits, nearest even; a scale is up to 1/128 above a / top, so the largest codes of the largest values would pass the type's range: they
// stop at its end (NaN stays NaN)
template <int DT>
__device__ static inline uint16_t to_16(float x) {
    constexpr float M = DT == ODMKV_F16 ? 65504.0f : 3.3895313892515355e38f;
    return Elem<DT>::from_f32(x > M ? M : x < -M ? -M : x);
}
// 16 bytes that are read once, or written for somebody else: the caches need not keep them
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ static inline uint4 load_once(const void* at) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ static inline void store_once(void* at, const uint4& v) { __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(at)); }
