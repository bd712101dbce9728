// Attention over the paged 8-bit cache (attend.hip: its entry; attend_narrow.h, attend_wide.h: its kernels): queries of the newest tokens, with any of a tanh cap, a bias by distance, a window, a prefix and
// document starts.
//
//   x_j = scaling * s_k (q . c_j), capped and biased;  out = sum_j softmax(x)_j s_v v_j over lo <= j < hi
#pragma once

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
    // rows that have their first blocks in common (attend_shared.h)
    const int32_t* plan;
    int spare;           // workgroups of a kv-head beyond one for each 128 of a group's queries
    float* common_out;   // partial results of what is in common: a kv-head's `common_parts`, each of 128
    float* common_lse;
    long long common_parts;
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

// Scores in base 2 from raw products: cap tanh(c x / cap) log2(e) = C - 2 C / (1 + 2^(k x)).  The reciprocal is off by 2^-23 of at most 1, the score by
// 2^-22 C: 1.1e-5 for the largest cap that goes this way, of weights that fp16 rounds by 2.4e-4.  Larger caps take tanh by itself.
#define CAP_BY_EXP 64.0f
// A larger one counts as this: times log2(e) it would pass 32 bits, and its reciprocal would lose digits.  It changes scores of up to 2^88 by less than they are rounded.
#define LARGEST_CAP 0x1p100f
struct Cap { float by, twice, plain; };                         // C, 2 C, and what makes k of c
__device__ static inline float capped(float kx, const Cap& m) {
    return __fmaf_rn(-m.twice, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(kx)), m.by);
}

// What a query's sums are relative to: weights to 2^ref, values that are weighted to 2^(ref + unit - 8).  Both are made of tokens that the query sees: what else lies in the
// row, and what other queries of the wavefront see, changes nothing.
//
// The values' operand is fp16: weights go there times 2^8 s / 2^unit, s what a code of one stands for in their block.  unit follows the largest weight times s, as ref follows
// the largest weight: where it is set that one is 2^8 exactly, so that a token that outweighs the others is not rounded at all, and it may grow to 2^15 (e4m3, whose codes are
// larger: 2^6 and 2^13).  A weight below fp16's normal numbers is off by 2^-25, 2^-33 of that (2^-31) at the most, whatever the scales are.
struct Sums { float ref, sum, unit; };
#define NO_UNIT -10000.0f
#define RISE 8.0f            // how far scores may pass the reference (base 2) before the sums are brought to a new one
#define UNIT_RISE 7.0f       // how far weights times s may pass the unit

// log2 s as a whole number and the rest, the latter 8 more; and what the unit has to follow: log2 s, 2 more for e4m3, whose codes go up to 448 where int8's end at 127.
// Values that are all 0 take the smallest, whose weights have no say.
struct Log2 { float whole, rest8, lift; };
template <int KIND>
__device__ static inline Log2 log2_of(float s) {
    const uint32_t bits = __float_as_uint(s);
    const float whole = s > 0.0f ? (float)((int)(bits >> 23) - 127) : -300.0f;
    const float rest = s > 0.0f ? __builtin_amdgcn_logf(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u)) : 0.0f;
    return {whole, rest + 8.0f, whole + (rest + (KIND == ODMKV_E4M3 ? 2.0f : 0.0f))};
}
// What goes for a block, until the sums move: a score above `limit` moves them; scores go to weights in the unit by `shift`, whose sum is freed of 2^factor.
// (Where s is nothing beside the unit, 2^-64 is as good, and the sum does not lose them.  The upper end is met where no token has been seen yet alone.)
struct Terms { float limit, factor, shift; };
__device__ static inline Terms terms_of(const Sums& s, const Log2& u) {
    const float factor = __builtin_amdgcn_fmed3f((u.whole - s.unit) + u.rest8, -64.0f, 1000.0f);
    return {s.ref + fminf(RISE, (s.unit + UNIT_RISE) - u.lift), factor, factor - fmaxf(s.ref, -1e30f)};
}
// The query's largest score, and the largest score plus log2 s as a sum of two, where they pass what they may; what the values' sums are to be multiplied by.
// Each query by itself: brought to a new reference with any other of its wavefront, a query would have bits that hang on what the others see.  (That would save a
// move here and there: documents 83.5 us for 86.6, 2048 queries over a window 185 for 189.)
__device__ static inline float raise(Sums& s, float most, float valued, float lift) {
    const bool some = s.ref > -INFINITY, up = most > s.ref + RISE || (valued - s.ref) + lift > s.unit + UNIT_RISE;
    const float to = up ? fmaxf(s.ref, most) : s.ref, rise = some ? to - s.ref : 0.0f;
    const float at = s.unit - rise, want = (valued - to) + lift, next = up ? (some ? fmaxf(at, want) : want) : at;
    s = {to, s.sum * __builtin_amdgcn_exp2f(-rise), next};
    return __builtin_amdgcn_exp2f(at - next);
}
// 2^(unit - 8 - less) x, all that it may be
__device__ static inline float in_unit(const Sums& s, float x, int less = 0) {
    const float power = fmaxf(s.unit - 8.0f, -500.0f), whole = floorf(power);
    return __builtin_amdgcn_ldexpf(x * __builtin_amdgcn_exp2f(power - whole), (int)whole - less);
}
// Products to scores; never 0, so that a place that is not seen (-inf) stays that (a block whose keys are all 0 has products of 0 alone).
__device__ static inline float scale_of(float ks, float qs) { return ks * qs != 0.0f ? ks * qs : 0x1p-120f; }

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

// 16-bit numbers of a token (or a query) on the fp16 matrix cores: times a power of two that takes the largest of them (its bits: `top`) to 64 .. 128 (fp16 numbers:
// by 2^15 at the most, which loses nothing either).  Nothing that counts is lost: what falls out of fp16's range is 2^-30 of the token's largest and less.  Tokens
// of a tail have a power each, since there may be queries that see one of them and not the others.
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

// the first n of eight numbers, 0 for the rest: what a tail holds behind its row's end is of tokens that are gone
__device__ static inline uint4 first_of8(int n) {                // as a mask
    uint32_t m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = n > 2 * i + 1 ? 0xffffffffu : n > 2 * i ? 0xffffu : 0u;
    return make_uint4(m[0], m[1], m[2], m[3]);
}
__device__ static inline uint4 masked8(const uint4& v, const uint4& m) { return make_uint4(v.x & m.x, v.y & m.y, v.z & m.z, v.w & m.w); }

// Powers of two tokens (a pair) of 16-bit numbers each, as power_for's, from the bits of their largest |x|.  The units' logarithms come as the numbers' own exponent
// fields, BIAS too large.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ static inline uint32_t magnitudes(uint32_t w) { return w & 0x7fff7fffu; }
__device__ static inline uint32_t larger_pair(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int DT, int PAIRS>
struct TokenPowers {
    static constexpr bool F16 = DT == ODMKV_F16;
    static constexpr float BIAS = F16 ? 15 + 6 : 127 + 6;
    uint32_t up[F16 ? PAIRS : 2 * PAIRS];       // fp16: pairs of fp16 numbers; bf16: fp32 numbers
    float log2[2 * PAIRS];
    __device__ inline void take(int pair, uint32_t top) {
        constexpr uint16_t SHIFT = F16 ? 10 : 7, LEAST = F16 ? 15 - 9 : 127 - 100;
        const u16x2 e = __builtin_elementwise_max(__builtin_bit_cast(u16x2, top) >> u16x2{SHIFT, SHIFT}, u16x2{LEAST, LEAST});
        log2[2 * pair] = (float)e[0];
        log2[2 * pair + 1] = (float)e[1];
        if constexpr (F16) up[pair] = __builtin_bit_cast(uint32_t, (u16x2{36, 36} - e) << u16x2{10, 10});
        else {
            up[2 * pair] = (260u - e[0]) << 23;
            up[2 * pair + 1] = (260u - e[1]) << 23;
        }
    }
    // the tokens of four pairs
    __device__ inline f16x8 scaled(const uint4& v, int pair) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (F16) h[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w[i]) * __builtin_bit_cast(f16x2, up[pair + i]));
            else h[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(w[i] << 16) * __uint_as_float(up[2 * (pair + i)]),
                                                                                __uint_as_float(w[i] & 0xffff0000u) * __uint_as_float(up[2 * (pair + i) + 1])));
        }
        return __builtin_bit_cast(f16x8, make_uint4(h[0], h[1], h[2], h[3]));
    }
};

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
__device__ static inline uint32_t column_larger(uint32_t v) {        // of 16-bit numbers' bits
    return __float_as_uint(column_fold(__uint_as_float(v), [](float x, float y) { return __uint_as_float(max(__float_as_uint(x), __float_as_uint(y))); }));
}
// over the sixteen lanes of a row
__device__ static inline uint32_t row_fold_pair(uint32_t v) {
    const auto of = [](uint32_t x, auto step) { return larger_pair(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(step)::value, 0xf, 0xf, false)); };
    v = of(v, std::integral_constant<int, 0xB1>());
    v = of(v, std::integral_constant<int, 0x4E>());
    v = of(v, std::integral_constant<int, 0x141>());
    return of(v, std::integral_constant<int, 0x140>());
}
__device__ static inline float read_float(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }
__device__ static inline int wave_min_int(int v) {
    return __float_as_int(wave_fold(__int_as_float(v), [](float x, float y) { return __int_as_float(min(__float_as_int(x), __float_as_int(y))); }));
}

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
template <bool BY_ROW, bool SHARED = false>
__device__ static inline Share share_of(const AttendArgs& a, int at) {
    const odmkv_pages_t& p = a.p;
    const int lane = threadIdx.x & 63;
    if (p.rows == 1) return {0, 0, a.splits};
    if (a.splits == p.rows) return {at, at, 1};
    const auto blocks = [&](int row) {
        if (row >= p.rows) return 0;
        const int len = p.length[row] - (SHARED ? a.plan[1 + row] * BLOCK_TOKENS : 0);
        return (a.window > 0 ? min(len, min(a.window, 1 << 29) + a.L) : len) / BLOCK_TOKENS + 1;
    };
    long long total = 0;
    int mine = 0;
    for (int r0 = 0; r0 < p.rows; r0 += 64) {
        mine = blocks(r0 + lane);
        total += __builtin_amdgcn_readlane(wave_scan(mine), 63);
    }
    const int spare = a.splits - p.rows;
    const auto share = [&](int blocks) {                        // (SHARED: what is not in common is short as a rule, and a share of less than a block a wavefront is none)
        const int n = 1 + (int)((long long)blocks * spare / total);
        return SHARED ? min(n, max(blocks / 4, 1)) : n;
    };
    int before = 0;
    for (int r0 = 0; r0 < p.rows; r0 += 64) {
        if (p.rows > 64) mine = blocks(r0 + lane);
        const int count = r0 + lane < p.rows ? share(mine) : 0;
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

// The plan of common blocks (pages.hip): groups of rows that have their first blocks in common.
struct Plan {
    const int32_t* at;
    int rows;
    __device__ inline Plan(const AttendArgs& a) : at(a.plan), rows(a.p.rows) {}
    __device__ inline int groups() const { return at[0]; }
    __device__ inline int common(int row) const { return at[1 + row]; }                     // blocks; 0: the row is in no group
    __device__ inline int group(int row) const { return at[1 + rows + row]; }
    __device__ inline int member(int row) const { return at[1 + 2 * rows + row]; }          // its place in the group
    __device__ inline int order(int i) const { return at[1 + 3 * rows + i]; }               // rows, a group's behind one another
    __device__ inline int begin(int g) const { return at[1 + 4 * rows + 4 * g]; }
    __device__ inline int members(int g) const { return at[2 + 4 * rows + 4 * g]; }
    __device__ inline int blocks(int g) const { return at[3 + 4 * rows + 4 * g]; }
    __device__ inline int slot(int g) const { return at[4 + 4 * rows + 4 * g]; }            // where its first row's table lies
};

#define SHARED_COLS 128      // queries of a kv-head that a workgroup takes over what is in common
// The workgroups of a kv-head that take what is in common: one for each tile of a group, the `spare` others in proportion to the tiles' blocks, several blocks each at least:
// a share costs its partial results.  Given a workgroup: its tile and share; given a group: how its tiles are shared; and where the group's partial results begin.
struct CommonShare { int group, tile, split, splits, parts, begin, cols, blocks, slot; };
template <bool BY_GROUP = false>
__device__ static inline CommonShare common_share_of(const AttendArgs& a, int at) {
    const Plan plan(a);
    const int lane = threadIdx.x & 63, R = a.G * a.L, most = a.p.rows / 2 - 1;
    // (asked for beside the number of groups, not behind it)
    struct Group { int begin, cols, blocks, slot; };
    const auto group_of = [&](int g) {
        const int at = min(g, most), begin = plan.begin(at), members = plan.members(at), blocks = plan.blocks(at), slot = plan.slot(at);
        return g < plan.groups() ? Group{begin, members * R, blocks, slot} : Group{0, 0, 0, 0};
    };
    const auto tiles_of = [](const Group& g) { return (g.cols + SHARED_COLS - 1) / SHARED_COLS; };
    Group mine = group_of(lane);
    const int groups = plan.groups();
    long long total = __builtin_amdgcn_readlane(wave_scan(tiles_of(mine) * mine.blocks), 63);
    for (int g0 = 64; g0 < groups; g0 += 64) {
        const Group next = group_of(g0 + lane);
        total += __builtin_amdgcn_readlane(wave_scan(tiles_of(next) * next.blocks), 63);
    }
    int before = 0, parts = 0;
    for (int g0 = 0; g0 < groups; g0 += 64) {
        if (g0 > 0) mine = group_of(g0 + lane);
        const int tiles = tiles_of(mine);
        const int splits = min(1 + (int)((long long)mine.blocks * a.spare / max(total, 1LL)), max(mine.blocks / (mine.cols > 64 ? 8 : 4), 1));
        const int upto = before + wave_scan(tiles * splits), parts_upto = parts + wave_scan(splits * mine.cols);
        const unsigned long long here = BY_GROUP ? (at < g0 + 64 ? 1ULL << (at - g0) : 0) : __ballot(upto > at);
        if (here) {
            const int l = __builtin_ctzll(here), n = __builtin_amdgcn_readlane(splits, l), first = __builtin_amdgcn_readlane(upto - tiles * splits, l);
            return {g0 + l, (at - first) / n, (at - first) % n, n, __builtin_amdgcn_readlane(parts_upto - splits * mine.cols, l),
                    __builtin_amdgcn_readlane(mine.begin, l), __builtin_amdgcn_readlane(mine.cols, l), __builtin_amdgcn_readlane(mine.blocks, l), __builtin_amdgcn_readlane(mine.slot, l)};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        parts = __builtin_amdgcn_readlane(parts_upto, 63);
    }
    return {-1, 0, 0, 0, 0, 0, 0, 0, 0};
}

#define NARROW 16            // queries of a kv-head that the narrow kernel takes
#define WIDE_WAVES 8

// How a call is cut.
struct Cut {
    int waves, splits;       // wavefronts of a workgroup; workgroups of a kv-head (narrow), or that share a row and kv-head's blocks (wide)
    int groups;              // wide: 32s of queries of a workgroup; two for four wavefronts: two take the first half of every block, two the second
    bool wide, stream;       // stream: pages pass by the caches
    size_t parts;            // partial results
    bool shared;             // rows have blocks in common: workgroups of a kv-head for those, of which `spare` beyond a tile's one, and their partial results
    int workgroups, spare;
    long long common_parts;
};
int launch_attend_narrow_f16(const AttendArgs& a, const Cut& cut, hipStream_t st);
int launch_attend_narrow_bf16(const AttendArgs& a, const Cut& cut, hipStream_t st);
int launch_attend_shared_f16(const AttendArgs& a, int workgroups, hipStream_t st);
int launch_attend_shared_bf16(const AttendArgs& a, int workgroups, hipStream_t st);
int launch_attend_wide_f16(const AttendArgs& a, const Cut& cut, hipStream_t st);
int launch_attend_wide_bf16(const AttendArgs& a, const Cut& cut, hipStream_t st);

template <typename K>
static int launch_attend(K kernel, const AttendArgs& a, long long groups, int waves, size_t lds, hipStream_t st) {
    ODMKV_CHECK_ARG(groups * waves * 64 < 0x100000000LL, "pages_attend: too many queries");
    if (lds > 65536) ODMKV_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(waves * 64), lds, st, a);
    ODMKV_CHECK_LAUNCH("pages_attend");
    return 0;
}
template <int V> using Int = std::integral_constant<int, V>;
