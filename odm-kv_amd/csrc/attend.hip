// Attention over the paged 8-bit cache: queries of the newest tokens, with any of a tanh cap, a bias by distance, a window, a prefix and
// document starts.
//
//   x_j = scaling * s_k (q . c_j), capped and biased;  out = sum_j softmax(x)_j s_v v_j over lo <= j < hi
#include <algorithm>
#include <type_traits>
#include "pages.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct AttendArgs {
    odmkv_pages_t p;
    const uint16_t* q;
    int64_t qb, qh, ql;
    uint16_t* out;
    float* lse;
    const int32_t* counts;
    const float* slopes;
    const int32_t* prefix;
    const int32_t* starts;
    int64_t sb, sl;
    int layer, L, Hq, G, window;
    float scaling, cap;
    int splits;          // workgroups of a kv-head (narrow), or that share a row and kv-head's blocks (wide)
    float* part_out;     // narrow [Hkv, splits, G L, 128], wide [rows, Hkv, splits, G L, 128]
    float* part_lse;     // the same without the 128, base 2
};

#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f

// what query l of a row of `len` tokens, `n` of whose newest have queries, stands at and sees
struct Sight { int pos, lo, hi; };
__device__ static inline Sight sight_of(const AttendArgs& a, int row, int len, int n, int l) {
    Sight s;
    s.pos = len - n + l;
    s.lo = max(0, a.starts ? a.starts[row * a.sb + l * a.sl] : 0);
    if (a.window > 0) s.lo = max(s.lo, s.pos - a.window + 1);
    s.hi = s.pos + 1;
    if (a.prefix) s.hi = max(s.hi, a.prefix[row]);
    s.hi = s.pos < 0 ? 0 : min(s.hi, len);
    return s;
}

// tanh: by its series where 1 - e loses digits, else by e = exp(-2 |t|)
__device__ static inline float tanh_of(float t) {
    const float a = fabsf(t), b = t * t;
    float f = __fmaf_rn(b, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    f = __fmaf_rn(b, f, -17.0f / 315.0f);
    f = __fmaf_rn(b, f, 2.0f / 15.0f);
    f = __fmaf_rn(b, f, -1.0f / 3.0f);
    const float e = __builtin_amdgcn_exp2f(-2.0f * LOG2E * a);
    const float far = __builtin_copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), t);
    return a < 0.3f ? __fmaf_rn(t * b, f, t) : far;
}

// a piece of codes; STREAM: read once, so that the caches need not keep it
template <bool STREAM>
__device__ static inline uint4 piece16(const uint8_t* at) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    if (!STREAM) return *reinterpret_cast<const uint4*>(at);
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// eight codes as fp16, all of them exactly.  int8: c + 128 is the low byte of the fp16 number 1024 + (c + 128)
template <int KIND>
__device__ static inline f16x8 codes_f16(uint32_t w0, uint32_t w1) {
    f16x2 h[4];
    if constexpr (KIND == ODMKV_E4M3) {
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
    } else {
        const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        w0 ^= 0x80808080u;
        w1 ^= 0x80808080u;
        h[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) + off;
        h[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) + off;
        h[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) + off;
        h[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) + off;
    }
    return f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// 16-bit numbers on the fp16 matrix cores: times a power of two that takes the largest of them (its bits: `top`) to 64 .. 128 (fp16 numbers: by 2^15 at the
// most, which loses nothing either).  Nothing that counts is lost: what falls out of fp16's range is 2^-30 of the largest and less.
struct Power { float up, down; };
template <int DT>
__device__ static inline Power power_for(uint32_t top) {
    const float t = Elem<DT>::to_f32((uint16_t)top);
    const int e = min(max((int)(__float_as_uint(t) >> 23) - 127, DT == ODMKV_F16 ? -9 : -100), 127);
    return {__uint_as_float((uint32_t)(127 + 6 - e) << 23), __uint_as_float((uint32_t)(127 - 6 + e) << 23)};
}
template <int DT>
__device__ static inline f16x8 scaled_f16(const uint4& v, float up) {
    if constexpr (DT == ODMKV_F16) return __builtin_bit_cast(f16x8, v) * (_Float16)up;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)                                 // (towards zero: exact but for the numbers that fall out of the range)
        h[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up));
    return __builtin_bit_cast(f16x8, make_uint4(h[0], h[1], h[2], h[3]));
}
__device__ static inline uint32_t abs_max8(const uint4& v) {
    return max(max(abs_max_pair(v.x), abs_max_pair(v.y)), max(abs_max_pair(v.z), abs_max_pair(v.w)));
}

// over the four lanes l, l ^ 16, l ^ 32, l ^ 48 of a query
template <typename F>
__device__ static inline float column_fold(float v, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ static inline float column_max(float v) { return column_fold(v, [](float x, float y) { return fmaxf(x, y); }); }
__device__ static inline float column_sum(float v) { return column_fold(v, [](float x, float y) { return x + y; }); }
__device__ static inline uint32_t larger_bits(uint32_t v, bool whole_wave) {
    const auto f = [](float x, float y) { return __uint_as_float(max(__float_as_uint(x), __float_as_uint(y))); };
    return __float_as_uint(whole_wave ? wave_fold(__uint_as_float(v), f) : column_fold(__uint_as_float(v), f));
}
__device__ static inline int wave_min_int(int v) {
    return __float_as_int(wave_fold(__int_as_float(v), [](float x, float y) { return __int_as_float(min(__float_as_int(x), __float_as_int(y))); }));
}

// ---- up to sixteen queries of a kv-head -----------------------------------------------------------
// A step of one token (G query heads share a kv-head's keys), or of a few.  The queries are the sixteen columns of the matrix instructions: keys times
// queries (rows: 16 tokens), then values times weights (rows: 16 dims, contraction: 32 tokens).  Which token a row of the first product is, is free:
// row 4 j + r of product tb is token 16 j + 4 tb + r, so that a lane ends with the weights of the sixteen tokens whose values of a dim it reads as
// one piece of 16 bytes; and lane (n, j) takes dims 32 j .. 32 j + 31 of its token, 32 bytes that lie together.  No weight changes lanes.
//
// Codes are exact in fp16, queries as they are (bf16: times a power of two each), products and sums fp32; a block's scale joins the scores and, for values,
// the weights: weights are rounded to fp16 (half a step, 2^-12 to 2^-11 of themselves) times 2^7 s / (largest s of the wavefront's blocks).
//
// A wavefront takes every fourth (or eighth) block of its workgroup's share, its pages and scales looked up 64 at a time, the next block's keys and values requested
// as soon as this one's are used.  Bound by memory (256 bytes a token and head); the arithmetic of a block is about a third of the time its bytes take.
#define NARROW 16
#define RISE 8.0f            // how far scores may pass the reference (base 2) before the sums are brought to a new one
#define NARROW_LDS(waves) ((waves) * NARROW * (HD + 4 + 2) * 4)

// The workgroups of a kv-head, `splits` of them, go to the rows by their lengths: one each, the others in proportion.  Given a workgroup (`at`): its row;
// given a row: its first workgroup; and how many it has.  A wavefront does this by itself, 64 rows at a time.
struct Share { int row, first, count; };
__device__ static inline int wave_scan(int v) {                 // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
template <bool BY_ROW>
__device__ static inline Share share_of(const AttendArgs& a, int at) {
    const odmkv_pages_t& p = a.p;
    const int lane = threadIdx.x & 63;
    if (p.rows == 1) return {0, 0, a.splits};
    if (a.splits == p.rows) return {at, at, 1};
    const auto blocks = [&](int row) {
        if (row >= p.rows) return 0;
        const int len = p.length[row];
        return (a.window > 0 ? min(len, min(a.window, 1 << 29) + a.L) : len) / BLOCK_TOKENS + 1;
    };
    long long total = 0;
    int mine = 0;
    for (int r0 = 0; r0 < p.rows; r0 += 64) {
        mine = blocks(r0 + lane);
        total += __builtin_amdgcn_readlane(wave_scan(mine), 63);
    }
    const int spare = a.splits - p.rows;
    int before = 0;
    for (int r0 = 0; r0 < p.rows; r0 += 64) {
        if (p.rows > 64) mine = blocks(r0 + lane);
        const int count = r0 + lane < p.rows ? 1 + (int)((long long)mine * spare / total) : 0;
        const int upto = before + wave_scan(count);
        if (BY_ROW) {
            if (at < r0 + 64) return {at, __builtin_amdgcn_readlane(upto - count, at - r0), __builtin_amdgcn_readlane(count, at - r0)};
        } else {
            const unsigned long long behind = __ballot(upto > at);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                return {r0 + l, __builtin_amdgcn_readlane(upto - count, l), __builtin_amdgcn_readlane(count, l)};
            }
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return {-1, 0, 0};
}

template <int DT, int KIND, bool PLAIN, int WAVES, bool STREAM>
__global__ __launch_bounds__(WAVES * 64, 2) void attend_narrow_kernel(AttendArgs a) {
    const odmkv_pages_t& p = a.p;
    extern __shared__ __align__(16) float narrow_lds[];
    float (*acc_of)[NARROW][HD + 4] = reinterpret_cast<float (*)[NARROW][HD + 4]>(narrow_lds);      // [WAVES]
    float (*ref_of)[NARROW] = reinterpret_cast<float (*)[NARROW]>(narrow_lds + WAVES * NARROW * (HD + 4));
    float (*sum_of)[NARROW] = ref_of + WAVES;
    // heads vary fastest: every head's longest row first, all heads alike
    const int h = blockIdx.x % p.Hkv, group = blockIdx.x / p.Hkv;
    const Share own = share_of<false>(a, group);
    const int row = __builtin_amdgcn_readfirstlane(own.row), splits = __builtin_amdgcn_readfirstlane(own.count);
    if (row < 0) return;
    const int split = group - __builtin_amdgcn_readfirstlane(own.first);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, j = lane >> 4;
    const int R = a.G * a.L, len = p.length[row], count = a.counts ? min(max(a.counts[row], 0), a.L) : a.L, slot = p.slot[row];
    const int l = n / a.G, hq = h * a.G + n - l * a.G;
    const bool valid = n < R && l < count;
    Sight s = {0, 0, 0};
    if (valid) s = sight_of(a, row, len, count, l);
    const bool sees = valid && s.lo < s.hi;
    const int first = wave_min_int(sees ? s.lo : 0x7fffffff) / BLOCK_TOKENS;
    const int last = (-wave_min_int(sees ? -s.hi : 0) + BLOCK_TOKENS - 1) / BLOCK_TOKENS;        // one past the last block that is seen
    // blocks from lo_max on and up to hi_min are seen by every query
    const int lo_max = valid && !sees ? 0x7fffffff : s.lo;
    const int open_from = -wave_min_int(valid ? -lo_max : 0), open_to = wave_min_int(valid ? s.hi : 0x7fffffff);
    const int blocks = max(last - first, 0), share = (blocks + splits - 1) / splits;
    const int b0 = first + split * share, mine = min(share, blocks - split * share);             // may be negative: nothing to do
    const int full = len / BLOCK_TOKENS, codes = min(mine, full - b0);                           // of the blocks those that lie in pages
    // 64 blocks of this wavefront at a time: their pages
    const auto pages_at = [&](int g0) {
        const int at = g0 + WAVES * lane;
        return at < codes ? p.table[(size_t)slot * p.blocks + b0 + at] : 0;
    };
    int page_of = pages_at(wave);                               // (asked for ahead of the queries: the codes wait for it)

    f16x8 q[4];
    float qdown = 1.0f;
    uint4 raw[4];
    {
        const uint16_t* src = a.q + row * a.qb + hq * a.qh + l * a.ql + 32 * j;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) raw[kk] = valid ? *reinterpret_cast<const uint4*>(src + 8 * kk) : make_uint4(0, 0, 0, 0);
    }
    const float slope = !PLAIN && a.slopes && valid ? a.slopes[hq] * LOG2E : 0.0f;
    const float inv_cap = !PLAIN && a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    float qs = 0.0f;
    const auto take_queries = [&]() {
        if constexpr (DT == ODMKV_BF16) {
            const uint32_t top = larger_bits(max(max(abs_max8(raw[0]), abs_max8(raw[1])), max(abs_max8(raw[2]), abs_max8(raw[3]))), false);
            const Power pw = power_for<DT>(top);
            qdown = pw.down;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) q[kk] = scaled_f16<DT>(raw[kk], pw.up);
        } else {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) q[kk] = __builtin_bit_cast(f16x8, raw[kk]);
        }
        qs = a.scaling * qdown * (PLAIN ? LOG2E : 1.0f);
    };

    float ref = -INFINITY, sum = 0.0f, vref = 0.0f;
    f32x4 acc[8];
#pragma unroll
    for (int m = 0; m < 8; ++m) acc[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // raw products of a block to weights: x [tb][r] is token 64 block + 16 j + 4 tb + r.  Back come the weights as operands, times f.
    const auto weigh = [&](const f32x4* dot, int block, float ks, float f, f16x8* w) {
        float x[16];
        const float c = ks * qs;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = dot[i >> 2][i & 3] * c;
        const int t0 = block * BLOCK_TOKENS + 16 * j;
        if constexpr (!PLAIN) {
            if (inv_cap > 0.0f) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = a.cap * tanh_of(x[i] * inv_cap);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __fmaf_rn(x[i], LOG2E, -slope * fabsf((float)(s.pos - t0 - i)));
        }
        if (block * BLOCK_TOKENS < open_from || block * BLOCK_TOKENS + BLOCK_TOKENS > open_to) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = t0 + i >= s.lo && t0 + i < s.hi ? x[i] : -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
        if (__any(top > ref + RISE)) {
            const float to = fmaxf(ref, column_max(top)), by = to > -INFINITY ? to : 0.0f, old = __builtin_amdgcn_exp2f(ref - by);
            ref = to;
            sum *= old;
#pragma unroll
            for (int m = 0; m < 8; ++m) acc[m] *= old;
        }
        const float by = ref > -INFINITY ? ref : 0.0f;
        float z0 = 0.0f, z1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            x[i] = __builtin_amdgcn_exp2f(x[i] - by);
            x[i + 1] = __builtin_amdgcn_exp2f(x[i + 1] - by);
            z0 += x[i];
            z1 += x[i + 1];
        }
        sum += z0 + z1;
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = (_Float16)(x[i] * f);
    };
    const auto values_up_to = [&](float v) {                    // the sums' values are in units of vref from here on
        if (v <= vref) return;
        const float old = vref / v;
#pragma unroll
        for (int m = 0; m < 8; ++m) acc[m] *= old;
        vref = v;
    };

    const size_t kat = (size_t)(16 * (n >> 2) + (n & 3)) * HD + 32 * j, vat = (size_t)n * BLOCK_TOKENS + 16 * j;
    bool first_group = true;
#pragma unroll 1
    for (int g0 = wave; g0 < codes; g0 += 64 * WAVES) {
        const int at = g0 + WAVES * lane, todo = min((codes - g0 + WAVES - 1) / WAVES, 64);
        if (!first_group) page_of = pages_at(g0);
        uint4 k[8], v[8];
        const auto request_keys = [&](int i) {
            const uint8_t* src = p.kcodes + page_at(p, a.layer, __builtin_amdgcn_readlane(page_of, i), h) + kat;
#pragma unroll
            for (int c = 0; c < 8; ++c) k[c] = piece16<STREAM>(src + (c >> 1) * 4 * HD + (c & 1) * 16);
        };
        const auto request_values = [&](int i) {
            const uint8_t* src = p.vcodes + page_at(p, a.layer, __builtin_amdgcn_readlane(page_of, i), h) + vat;
#pragma unroll
            for (int m = 0; m < 8; ++m) v[m] = piece16<STREAM>(src + m * 16 * BLOCK_TOKENS);
        };
        request_keys(0);
        const float ks_of = at < codes ? p.kscale[scale_at(p, a.layer, page_of, h)] : 0.0f;
        const float vs_of = at < codes ? p.vscale[scale_at(p, a.layer, page_of, h)] : 0.0f;
        request_values(0);
        if (first_group) take_queries();
        first_group = false;
        values_up_to(wave_max(vs_of));
        const float f_of = vref > 0.0f ? 128.0f * (vs_of / vref) : 0.0f;
#pragma unroll 1
        for (int i = 0; i < todo; ++i) {
            f32x4 dot[4];
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                dot[tb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint4& c = k[2 * tb + (kk >> 1)];
                    dot[tb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk & 1 ? codes_f16<KIND>(c.z, c.w) : codes_f16<KIND>(c.x, c.y), q[kk], dot[tb], 0, 0, 0);
                }
            }
            if (i + 1 < todo) request_keys(i + 1);
            f16x8 w[2];
            weigh(dot, b0 + g0 + WAVES * i, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_of), i)),
                  __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f_of), i)), w);
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16<KIND>(v[m].x, v[m].y), w[0], acc[m], 0, 0, 0);
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16<KIND>(v[m].z, v[m].w), w[1], acc[m], 0, 0, 0);
            }
            if (i + 1 < todo) request_values(i + 1);
        }
    }
    // the open block, by the wavefront whose turn it is
    if (mine > 0 && b0 + mine > full && (mine - 1) % WAVES == wave) {
        const uint16_t* kt = p.ktail + tail_at(p, a.layer, slot, h) + kat;
        const uint16_t* vt = p.vtail + tail_at(p, a.layer, slot, h) + vat;
        uint4 k[16], v[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) k[c] = *reinterpret_cast<const uint4*>(kt + (c >> 2) * 4 * HD + (c & 3) * 8);
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = *reinterpret_cast<const uint4*>(vt + (c >> 1) * 16 * BLOCK_TOKENS + (c & 1) * 8);
        if (first_group) take_queries();
        Power pk = {1.0f, 1.0f};
        if constexpr (DT == ODMKV_BF16) {                       // (fp16 keys are taken as they are)
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < 16; ++c) top = max(top, abs_max8(k[c]));
            pk = power_for<DT>(larger_bits(top, true));
        }
        f32x4 dot[4];
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
            dot[tb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                f16x8 x;
                if constexpr (DT == ODMKV_BF16) x = scaled_f16<DT>(k[4 * tb + kk], pk.up);
                else x = __builtin_bit_cast(f16x8, k[4 * tb + kk]);
                dot[tb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[kk], dot[tb], 0, 0, 0);
            }
        }
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c) top = max(top, abs_max8(v[c]));
        top = larger_bits(top, true);
        const Power pv = power_for<DT>(top);
        if (top > 0) values_up_to(pv.down);
        f16x8 w[2];
        weigh(dot, full, pk.down, top > 0 ? 128.0f * (pv.down / vref) : 0.0f, w);
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(scaled_f16<DT>(v[2 * m], pv.up), w[0], acc[m], 0, 0, 0);
            acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(scaled_f16<DT>(v[2 * m + 1], pv.up), w[1], acc[m], 0, 0, 0);
        }
    }

    sum = column_sum(sum);
    const float unit = vref * (1.0f / 128.0f);
#pragma unroll
    for (int m = 0; m < 8; ++m) *reinterpret_cast<f32x4*>(&acc_of[wave][n][16 * m + 4 * j]) = acc[m] * unit;
    if (j == 0) {
        ref_of[wave][n] = ref;
        sum_of[wave][n] = sum;
    }
    __syncthreads();
    // a thread takes eight dims of a query
    const int r = tid >> 4, d = (tid & 15) * 8, rl = r / a.G, rh = h * a.G + r - rl * a.G;
    if (r >= R || rl >= count) return;                          // (of eight wavefronts the last four have no query)
    float to = ref_of[0][r], total = 0.0f, o[8];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) to = fmaxf(to, ref_of[w][r]);
    const float by = to > -INFINITY ? to : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(ref_of[w][r] - by);
        // (a query that is not a number has a sum that is not, and a reference that may be anything)
        total += sum_of[w][r] == 0.0f ? 0.0f : sum_of[w][r] * f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __fmaf_rn(acc_of[w][r][d + e], f, o[e]);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = total == 0.0f ? 0.0f : o[e] * inv;
    const float lse2 = total == 0.0f ? -INFINITY : to + __builtin_amdgcn_logf(total);
    if (splits > 1) {
        const size_t unit_at = ((size_t)h * a.splits + group) * R + r;
        f32x4* dst = reinterpret_cast<f32x4*>(a.part_out + unit_at * HD + d);
        dst[0] = f32x4{o[0], o[1], o[2], o[3]};
        dst[1] = f32x4{o[4], o[5], o[6], o[7]};
        if (d == 0) a.part_lse[unit_at] = lse2;
        return;
    }
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = (uint32_t)to_16<DT>(o[2 * e]) | (uint32_t)to_16<DT>(o[2 * e + 1]) << 16;
    *reinterpret_cast<uint4*>(a.out + (((size_t)row * a.L + rl) * a.Hq + rh) * HD + d) = make_uint4(b[0], b[1], b[2], b[3]);
    if (a.lse && d == 0) a.lse[((size_t)row * a.Hq + rh) * a.L + rl] = lse2 * LN2;
}

// The shares of a row and kv-head's blocks, put together: a workgroup a query, its four wavefronts every fourth share, a lane two dims.
template <int DT, bool NARROW_PARTS>
__global__ __launch_bounds__(256) void attend_merge_kernel(AttendArgs a) {
    const odmkv_pages_t& p = a.p;
    const int R = a.G * a.L, r = blockIdx.x, h = blockIdx.y, row = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = r / a.G, hq = h * a.G + r - l * a.G;
    if (l >= (a.counts ? min(max(a.counts[row], 0), a.L) : a.L)) return;
    __shared__ float part[4][HD], top_of[4], sum_of[4];
    int splits = a.splits;
    size_t at = ((size_t)row * p.Hkv + h) * a.splits * R + r;
    if (NARROW_PARTS) {
        const Share own = share_of<true>(a, row);
        if (own.count == 1) return;                             // that workgroup has written the result
        splits = own.count;
        at = ((size_t)h * a.splits + own.first) * R + r;
    }
    float top = -INFINITY;
    for (int i = lane; i < splits; i += 64) top = fmaxf(top, a.part_lse[at + (size_t)i * R]);
    top = wave_max(top);
    const float by = top > -INFINITY ? top : 0.0f;
    float sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll 4
    for (int i = wave; i < splits; i += 4) {
        const float lse = a.part_lse[at + (size_t)i * R];
        const float2 v = *reinterpret_cast<const float2*>(a.part_out + (at + (size_t)i * R) * HD + 2 * lane);
        const float w = __builtin_amdgcn_exp2f(lse - by);
        sum += w;
        o0 = __fmaf_rn(w, v.x, o0);
        o1 = __fmaf_rn(w, v.y, o1);
    }
    part[wave][2 * lane] = o0;
    part[wave][2 * lane + 1] = o1;
    if (lane == 0) sum_of[wave] = sum;
    __syncthreads();
    if (tid >= 64) return;
    sum = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    o0 = ((part[0][2 * lane] + part[1][2 * lane]) + (part[2][2 * lane] + part[3][2 * lane])) * inv;
    o1 = ((part[0][2 * lane + 1] + part[1][2 * lane + 1]) + (part[2][2 * lane + 1] + part[3][2 * lane + 1])) * inv;
    *reinterpret_cast<uint32_t*>(a.out + (((size_t)row * a.L + l) * a.Hq + hq) * HD + 2 * lane) = (uint32_t)to_16<DT>(o0) | (uint32_t)to_16<DT>(o1) << 16;
    if (a.lse && lane == 0) a.lse[((size_t)row * a.Hq + hq) * a.L + l] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// ---- many queries of a kv-head --------------------------------------------------------------------
// A wavefront holds 32 queries (the columns of v_mfma_f32_32x32x16_f16), a workgroup 32 WAVES of them, token by token with the G heads of a
// token together, so that a workgroup's tokens lie together and blocks that none of them sees are passed over.  A block of 64 tokens is turned into fp16 once a workgroup
// and lies in LDS, the next block's codes are on their way in registers; rows of the first product are tokens as they lie, and row r of a half
// wavefront's sixteen (8 (r / 4) + 4 half + r % 4) decides the order in which values lie in LDS: what a lane holds of the weights is
// then its operand of the second product.  16-byte pieces of a row are moved by the row's number (xor), so that no two of eight rows meet in a bank.
#define WIDE_WAVES 8
#define WIDE_LDS (2 * (BLOCK_TOKENS * HD * 2 * 2))
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT, int KIND, bool PLAIN, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attend_wide_kernel(AttendArgs a) {
    const odmkv_pages_t& p = a.p;
    extern __shared__ __align__(16) uint8_t lds[];              // [2][keys 64 x 256 bytes, values 128 x 128 bytes]
    __shared__ int range[2][WAVES];
    __shared__ uint32_t tops[2][WAVES];
    constexpr int THREADS = WAVES * 64, BUFFER = BLOCK_TOKENS * HD * 4, VALUES = BLOCK_TOKENS * HD * 2;
    const int pairs = p.rows * p.Hkv, R = a.G * a.L, tiles = (R + 32 * WAVES - 1) / (32 * WAVES);
    // heads vary fastest (a die of the chip then keeps few heads' pages in its L2), the longest rows of blocks come first
    const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs, split = rest % a.splits, tile = tiles - 1 - rest / a.splits;
    const int row = pair / p.Hkv, h = pair % p.Hkv, tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int len = p.length[row], count = a.counts ? min(max(a.counts[row], 0), a.L) : a.L, slot = p.slot[row];
    const int r0 = tile * 32 * WAVES + 32 * wave, r = r0 + col, l = r / a.G, hq = h * a.G + r - l * a.G;
    const bool valid = r < R && l < count;
    Sight s = {0, 0, 0};
    if (valid) s = sight_of(a, row, len, count, l);
    const bool sees = valid && s.lo < s.hi;
    const int wave_lo = wave_min_int(sees ? s.lo : 0x7fffffff), wave_hi = -wave_min_int(sees ? -s.hi : 0);       // what some query of the wavefront sees
    const int open_from = -wave_min_int(valid ? -(sees ? s.lo : 0x7fffffff) : 0), open_to = wave_min_int(valid ? s.hi : 0x7fffffff);    // what all of them see
    if (lane == 0) {
        range[0][wave] = wave_lo;
        range[1][wave] = wave_hi;
    }
    __syncthreads();
    int lo = range[0][0], hi = range[1][0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        lo = min(lo, range[0][w]);
        hi = max(hi, range[1][w]);
    }
    const int first = lo / BLOCK_TOKENS, blocks = max((hi + BLOCK_TOKENS - 1) / BLOCK_TOKENS - first, 0), share = (blocks + a.splits - 1) / a.splits;
    const int b0 = __builtin_amdgcn_readfirstlane(first + split * share), mine = __builtin_amdgcn_readfirstlane(min(share, blocks - split * share));
    const int full = len / BLOCK_TOKENS;

    f16x8 q[8];                                                 // dims 16 st + 8 half + e
    float qdown = 1.0f;
    {
        uint4 raw[8];
        const uint16_t* src = a.q + row * a.qb + hq * a.qh + l * a.ql + 8 * half;
#pragma unroll
        for (int st = 0; st < 8; ++st) raw[st] = valid ? *reinterpret_cast<const uint4*>(src + 16 * st) : make_uint4(0, 0, 0, 0);
        if constexpr (DT == ODMKV_BF16) {
            uint32_t top = 0;
#pragma unroll
            for (int st = 0; st < 8; ++st) top = max(top, abs_max8(raw[st]));
            const auto o = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            const Power pw = power_for<DT>(max(o[0], o[1]));
            qdown = pw.down;
#pragma unroll
            for (int st = 0; st < 8; ++st) q[st] = scaled_f16<DT>(raw[st], pw.up);
        } else {
#pragma unroll
            for (int st = 0; st < 8; ++st) q[st] = __builtin_bit_cast(f16x8, raw[st]);
        }
    }
    const float slope = !PLAIN && a.slopes && valid ? a.slopes[hq] * LOG2E : 0.0f;
    const float inv_cap = !PLAIN && a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    const float qs = a.scaling * qdown * (PLAIN ? LOG2E : 1.0f);

    float ref = -INFINITY, sum = 0.0f, vref = 0.0f;
    f32x16 acc[4];                                              // dims 32 db + 8 (r / 4) + 4 half + r % 4 of query `col`
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.0f;

    const auto values_up_to = [&](float v) {                    // the sums' values are in units of vref from here on
        if (v <= vref) return;
        const float old = vref / v;
#pragma unroll
        for (int db = 0; db < 4; ++db) acc[db] *= old;
        vref = v;
    };

    // ---- a block on its way: pieces of 16 codes, a token's 16 dims or a dim's 16 tokens
    constexpr int PIECES = PAGE_BYTES / 16 / THREADS;
    uint4 kc[PIECES], vc[PIECES];
    int page_of = 0;
    const auto look_up = [&](int i) { return i + lane < mine && b0 + i + lane < full ? p.table[(size_t)slot * p.blocks + b0 + i + lane] : 0; };
    const auto request = [&](int i) {                           // block b0 + i, which lies in a page
        if ((i & 63) == 0) page_of = look_up(i);
        const size_t at = page_at(p, a.layer, __builtin_amdgcn_readlane(page_of, i & 63), h);
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            kc[c] = *reinterpret_cast<const uint4*>(p.kcodes + at + (size_t)(tid + c * THREADS) * 16);
            vc[c] = *reinterpret_cast<const uint4*>(p.vcodes + at + (size_t)(tid + c * THREADS) * 16);
        }
    };
    const auto key_piece = [&](uint8_t* buf, int token, int piece) { return reinterpret_cast<f16x8*>(buf + token * 256 + ((piece ^ (token & 15)) << 4)); };
    const auto value_piece = [&](uint8_t* buf, int dim, int piece) { return buf + VALUES + dim * 128 + ((piece ^ (dim & 7)) << 4); };
    const auto put = [&](uint8_t* buf) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            const int i = tid + c * THREADS;
            *key_piece(buf, i >> 3, 2 * (i & 7)) = codes_f16<KIND>(kc[c].x, kc[c].y);
            *key_piece(buf, i >> 3, 2 * (i & 7) + 1) = codes_f16<KIND>(kc[c].z, kc[c].w);
            *reinterpret_cast<f16x8*>(value_piece(buf, i >> 2, 2 * (i & 3))) = codes_f16<KIND>(vc[c].x, vc[c].z);
            *reinterpret_cast<f16x8*>(value_piece(buf, i >> 2, 2 * (i & 3) + 1)) = codes_f16<KIND>(vc[c].y, vc[c].w);
        }
    };
    float tail_k = 1.0f, tail_v = 0.0f;                         // what the open block's numbers in LDS are to be multiplied by
    const auto put_tail = [&](uint8_t* buf) {
        const uint4* kt = reinterpret_cast<const uint4*>(p.ktail + tail_at(p, a.layer, slot, h));
        const uint4* vt = reinterpret_cast<const uint4*>(p.vtail + tail_at(p, a.layer, slot, h));
        uint32_t top[2] = {0, 0};
#pragma unroll 1
        for (int i = tid; i < TAIL_ELEMS / 8; i += THREADS) {
            top[0] = max(top[0], abs_max8(kt[i]));
            top[1] = max(top[1], abs_max8(vt[i]));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t t = larger_bits(top[x], true);
            if (lane == 0) tops[x][wave] = t;
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top[x] = max(top[x], tops[x][w]);
        const Power pk = power_for<DT>(top[0]), pv = power_for<DT>(top[1]);
        tail_k = pk.down;
        tail_v = top[1] > 0 ? pv.down : 0.0f;
#pragma unroll 1
        for (int i = tid; i < TAIL_ELEMS / 8; i += THREADS) {
            const int dim = i >> 3, u = i & 7;
            *key_piece(buf, i >> 4, i & 15) = scaled_f16<DT>(kt[i], pk.up);
            const uint4 x = __builtin_bit_cast(uint4, scaled_f16<DT>(vt[i], pv.up));
            *reinterpret_cast<uint2*>(value_piece(buf, dim, u & ~1) + 8 * (u & 1)) = make_uint2(x.x, x.y);
            *reinterpret_cast<uint2*>(value_piece(buf, dim, u | 1) + 8 * (u & 1)) = make_uint2(x.z, x.w);
        }
    };

    const int codes = min(mine, full - b0);                     // of the blocks those that lie in pages
    if (codes > 0) request(0);
    float ks_of = 0.0f, f_of = 0.0f;
#pragma unroll 1
    for (int i = -1; i < mine; ++i) {
        uint8_t* buf = lds + (i & 1) * BUFFER;
        __syncthreads();                                        // this block lies there, and nobody reads the one before any more
        if (i + 1 < codes) put(lds + ((i + 1) & 1) * BUFFER);
        else if (i + 1 < mine) put_tail(lds + ((i + 1) & 1) * BUFFER);
        if (i + 2 < codes) request(i + 2);
        if (i < 0) continue;
        const int t0 = (b0 + i) * BLOCK_TOKENS;
        float ks, f;
        if (i < codes) {
            if ((i & 63) == 0) {                                // 64 blocks' scales at a time
                const bool in = i + lane < codes;
                const int page = look_up(i);
                const float vs = in ? p.vscale[scale_at(p, a.layer, page, h)] : 0.0f;
                ks_of = in ? p.kscale[scale_at(p, a.layer, page, h)] : 0.0f;
                values_up_to(wave_max(vs));
                f_of = vref > 0.0f ? 128.0f * (vs / vref) : 0.0f;
            }
            ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_of), i & 63));
            f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f_of), i & 63));
        } else {
            ks = tail_k;
            values_up_to(tail_v);
            f = tail_v > 0.0f ? 128.0f * (tail_v / vref) : 0.0f;
        }
        if (t0 >= wave_hi || t0 + BLOCK_TOKENS <= wave_lo) continue;      // (of the wavefront's own queries none sees the block)
        f32x16 dot[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) dot[tb][e] = 0.0f;
#pragma unroll
            for (int st = 0; st < 8; ++st)
                dot[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*key_piece(buf, 32 * tb + col, 2 * st + half), q[st], dot[tb], 0, 0, 0);
        }
        const float c = ks * qs;
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = dot[e >> 4][e & 15] * c;
        const int tl = t0 + 4 * half;                           // token of x[e]: tl + 8 (e / 4) + e % 4
        if constexpr (!PLAIN) {
            if (inv_cap > 0.0f) {
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = a.cap * tanh_of(x[e] * inv_cap);
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = __fmaf_rn(x[e], LOG2E, -slope * fabsf((float)(s.pos - tl - 8 * (e >> 2) - (e & 3))));
        }
        if (t0 < open_from || t0 + BLOCK_TOKENS > open_to) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                const int t = tl + 8 * (e >> 2) + (e & 3);
                x[e] = t >= s.lo && t < s.hi ? x[e] : -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, x[e]);
        if (__any(top > ref + RISE)) {
            const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            const float to = fmaxf(ref, fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1]))), by = to > -INFINITY ? to : 0.0f;
            const float old = __builtin_amdgcn_exp2f(ref - by);
            ref = to;
            sum *= old;
#pragma unroll
            for (int db = 0; db < 4; ++db) acc[db] *= old;
        }
        const float by = ref > -INFINITY ? ref : 0.0f;
        float z0 = 0.0f, z1 = 0.0f;
        f16x8 w[4];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            const float p0 = __builtin_amdgcn_exp2f(x[e] - by), p1 = __builtin_amdgcn_exp2f(x[e + 1] - by);
            z0 += p0;
            z1 += p1;
            w[e >> 3][e & 7] = (_Float16)(p0 * f);
            w[e >> 3][(e & 7) + 1] = (_Float16)(p1 * f);
        }
        sum += z0 + z1;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int st = 0; st < 4; ++st)
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8*>(value_piece(buf, 32 * db + col, 2 * st + half)), w[st], acc[db], 0, 0, 0);
    }

    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(o[0]) + __uint_as_float(o[1]);
    if (!valid) return;
    const bool none = sum == 0.0f;
    const float unit = none ? 0.0f : vref * (1.0f / 128.0f) / sum, lse2 = none ? -INFINITY : ref + __builtin_amdgcn_logf(sum);
    if (a.splits > 1) {
        const size_t unit_at = ((size_t)pair * a.splits + split) * R + r;
        float* dst = a.part_out + unit_at * HD + 4 * half;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = none ? 0.0f : acc[db][4 * g + e] * unit;
                *reinterpret_cast<f32x4*>(dst + 32 * db + 8 * g) = v;
            }
        if (half == 0) a.part_lse[unit_at] = lse2;
        return;
    }
    uint16_t* dst = a.out + (((size_t)row * a.L + l) * a.Hq + hq) * HD + 4 * half;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint32_t v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                v[e] = none ? 0u : (uint32_t)to_16<DT>(acc[db][4 * g + 2 * e] * unit) | (uint32_t)to_16<DT>(acc[db][4 * g + 2 * e + 1] * unit) << 16;
            *reinterpret_cast<uint2*>(dst + 32 * db + 8 * g) = make_uint2(v[0], v[1]);
        }
    if (a.lse && half == 0) a.lse[((size_t)row * a.Hq + hq) * a.L + l] = none ? -INFINITY : lse2 * LN2;
}

// How a call is cut: wavefronts of a workgroup (0: the narrow kernel) and workgroups that share a row's blocks, two a compute unit in all,
// each with a few blocks at least.
struct Cut { int waves, splits; bool wide, stream; size_t parts; };     // stream: pages pass by the caches; parts: partial results
static Cut cut_of(const odmkv_pages_t& p, int R, int max_length) {
    const int blocks = max_length / BLOCK_TOKENS + 1, units = compute_units();
    Cut c = {4, 1, R > NARROW, false, 0};
    if (c.wide) {
        c.waves = R > 128 ? WIDE_WAVES : 4;
        const long long groups = (long long)p.rows * p.Hkv * ((R + 32 * c.waves - 1) / (32 * c.waves));
        c.splits = (int)std::max(1LL, std::min((c.waves == WIDE_WAVES ? 1 : 2) * units / groups, (long long)blocks / 4));
        c.parts = c.splits > 1 ? (size_t)p.rows * p.Hkv * c.splits * R : 0;
    } else {
        // Pages that all layers together have too many of for the last-level cache (256 MB) to keep from one call to the next: nothing is gained by keeping any, and
        // reads that do not ask for it reach 5.9 TB/s instead of 5.0 (268 MB a call 59.7 -> 51.4 us; 67 MB a call over three caches in turn, which do fit, 18.7 -> 20.2).
        c.stream = (size_t)p.layers * p.pages * p.Hkv * 2 * PAGE_BYTES > ((size_t)128 << 20);
        // Eight wavefronts where they hold a row's blocks by themselves, so that nothing is merged (500 tokens: 10.8 -> 9.7 us), and for one row so long that
        // each has several (131071 tokens of 4 heads: 35.4 -> 33.2 us; half as many shares to merge); four otherwise: twice as many compute units for 2000 tokens
        // (13.1 -> 11.2 us), finer shares for rows of their own lengths (16 of up to 8192: 50.6 -> 40.4 us).
        c.waves = blocks <= 8 || (p.rows == 1 && (long long)blocks * p.Hkv >= 24LL * units) ? 8 : 4;
        const long long most = (long long)p.rows * std::max(1, blocks / c.waves);
        c.splits = (int)std::max((long long)p.rows, std::min((long long)(8 / c.waves) * units / p.Hkv, most));
        c.parts = c.splits > p.rows ? (size_t)p.Hkv * c.splits * R : 0;
    }
    return c;
}

extern "C" size_t odmkv_pages_attend_workspace_bytes(const odmkv_pages_t* p, int Hq, int L, int max_length) {
    if (!p || p->Hkv <= 0 || p->rows <= 0 || Hq <= 0 || L <= 0 || max_length < 0) return 0;
    return align_up(cut_of(*p, Hq / p->Hkv * L, max_length).parts * (HD + 1) * sizeof(float), 256);
}

template <int DT, int KIND>
static int launch_attend(const AttendArgs& a, const Cut& cut, hipStream_t st) {
    const bool plain = a.cap == 0.0f && !a.slopes;
    const int R = a.G * a.L;
    const long long groups = cut.wide ? (long long)a.p.rows * a.p.Hkv * a.splits * ((R + 32 * cut.waves - 1) / (32 * cut.waves)) : (long long)a.p.Hkv * a.splits;
    ODMKV_CHECK_ARG(groups < 0x7fffffffLL, "pages_attend: too many queries");
    const size_t lds = cut.wide ? WIDE_LDS : NARROW_LDS(cut.waves);
    const auto run = [&](auto kernel) -> int {
        if (lds > 65536) ODMKV_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(cut.waves * 64), lds, st, a);
        ODMKV_CHECK_LAUNCH("attend kernel");
        return 0;
    };
    const auto narrow = [&](auto plain_, auto waves_, auto stream_) { return run(attend_narrow_kernel<DT, KIND, plain_.value, waves_.value, stream_.value>); };
    const auto narrow_of = [&](auto waves_) {
        const std::true_type yes;
        const std::false_type no;
        return plain ? (cut.stream ? narrow(yes, waves_, yes) : narrow(yes, waves_, no)) : (cut.stream ? narrow(no, waves_, yes) : narrow(no, waves_, no));
    };
    int rc;
    if (!cut.wide) {
        rc = cut.waves == 4 ? narrow_of(std::integral_constant<int, 4>()) : narrow_of(std::integral_constant<int, 8>());
    } else if (cut.waves == 4) rc = plain ? run(attend_wide_kernel<DT, KIND, true, 4>) : run(attend_wide_kernel<DT, KIND, false, 4>);
    else rc = plain ? run(attend_wide_kernel<DT, KIND, true, WIDE_WAVES>) : run(attend_wide_kernel<DT, KIND, false, WIDE_WAVES>);
    if (rc || !cut.parts) return rc;
    const dim3 grid(R, a.p.Hkv, a.p.rows);
    if (cut.wide) hipLaunchKernelGGL((attend_merge_kernel<DT, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attend_merge_kernel<DT, true>), grid, dim3(256), 0, st, a);
    ODMKV_CHECK_LAUNCH("attend_merge_kernel");
    return 0;
}

extern "C" int odmkv_pages_attend(const odmkv_attend_t* d, void* stream) {
    ODMKV_CHECK_ARG(d && d->pages, "pages_attend: null pointer");
    const odmkv_pages_t& p = *d->pages;
    ODMKV_CHECK_ARG(p.kcodes && p.vcodes && p.kscale && p.vscale && p.ktail && p.vtail && p.table && p.length && p.slot, "pages_attend: null pointer");
    ODMKV_CHECK_ARG(p.layers > 0 && p.rows > 0 && p.rows <= MAX_ROWS && p.Hkv > 0 && p.Hkv <= 65535 && p.pages > 0 && p.blocks > 0, "pages_attend: bad shape");
    ODMKV_CHECK_ARG(p.dtype == ODMKV_F16 || p.dtype == ODMKV_BF16, "pages_attend: bad dtype %d", p.dtype);
    ODMKV_CHECK_ARG(p.kind == ODMKV_INT8 || p.kind == ODMKV_E4M3, "pages_attend: bad kind %d", p.kind);
    ODMKV_CHECK_ARG(d->layer >= 0 && d->layer < p.layers, "pages_attend: layer %d of %d", d->layer, p.layers);
    ODMKV_CHECK_ARG(d->Hq > 0 && d->Hq % p.Hkv == 0 && d->Hq / p.Hkv <= ODMKV_MAX_GROUP, "pages_attend: %d query heads over %d kv-heads", d->Hq, p.Hkv);
    ODMKV_CHECK_ARG(d->L >= 0 && d->L <= (1 << 26) && d->window >= 0 && d->max_length >= 0, "pages_attend: bad length");
    ODMKV_CHECK_ARG(d->cap >= 0.0f && d->cap < INFINITY, "pages_attend: bad cap");
    if (d->L == 0) return 0;
    ODMKV_CHECK_ARG(d->q && d->out, "pages_attend: null pointer");
    ODMKV_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->out) & 15) == 0 && ((d->q_stride_b | d->q_stride_h | d->q_stride_l) & 7) == 0,
                    "pages_attend: rows must be 16-byte aligned");
    AttendArgs a = {p, (const uint16_t*)d->q, d->q_stride_b, d->q_stride_h, d->q_stride_l, (uint16_t*)d->out, d->lse, d->counts, d->slopes,
                    d->prefix, d->starts, d->start_stride_b, d->start_stride_l, d->layer, d->L, d->Hq, d->Hq / p.Hkv, d->window, d->scaling, d->cap,
                    1, nullptr, nullptr};
    const size_t need = odmkv_pages_attend_workspace_bytes(&p, d->Hq, d->L, d->max_length);
    if (need > 0 && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < need)) {
        odmkv_set_error("pages_attend: workspace too small");
        return ODMKV_ENOSPACE;
    }
    const Cut cut = cut_of(p, a.G * a.L, d->max_length);
    a.splits = cut.splits;
    a.part_out = (float*)d->workspace;
    a.part_lse = a.part_out + cut.parts * HD;
    hipStream_t st = (hipStream_t)stream;
    if (p.dtype == ODMKV_F16) return p.kind == ODMKV_INT8 ? launch_attend<ODMKV_F16, ODMKV_INT8>(a, cut, st) : launch_attend<ODMKV_F16, ODMKV_E4M3>(a, cut, st);
    return p.kind == ODMKV_INT8 ? launch_attend<ODMKV_BF16, ODMKV_INT8>(a, cut, st) : launch_attend<ODMKV_BF16, ODMKV_E4M3>(a, cut, st);
}
