// Attention over the paged 8-bit cache for up to sixteen queries of a kv-head.
//
// A step of one token (G query heads share a kv-head's keys), or of a few.  The queries are the sixteen columns of the matrix instructions: keys times
// queries (rows: 16 tokens), then values times weights (rows: 16 dims, contraction: 32 tokens).  Which token a row of the first product is, is free:
// row 4 j + r of product tb is token 16 j + 4 tb + r, so that a lane ends with the weights of the sixteen tokens whose values of a dim it reads as
// one piece of 16 bytes; and lane (n, j) takes dims 32 j .. 32 j + 31 of its token, 32 bytes that lie together.  No weight changes lanes.
//
// Codes are exact in fp16, queries as they are (bf16: times a power of two each), products and sums fp32; a block's scale joins the scores and, for values,
// the weights: weights are rounded to fp16 (half a step, 2^-12 to 2^-11 of themselves) in a unit of
// each query's own, which the tokens that it sees decide (attend.h: Sums).
//
// A wavefront takes every fourth (or eighth) block of its workgroup's share, its pages and scales looked up 64 at a time, the next block's keys and values requested
// as soon as this one's are used: no tile passes through LDS, which holds what the wavefronts join at the end alone.  Bound by memory (256 bytes a token and head) and
// by what a launch costs, the arithmetic of a block being about a third of the time its bytes take.  Four query heads to a kv-head, one token: 32768 tokens of 8 heads,
// 67 MB, 15.6 us (4.3 TB/s) and 4.0 of the merge behind it; 16 rows of up to 8192 tokens, 165 MB, 35.9 (4.6 TB/s) and 4.8; 131071 tokens of 8 heads, 268 MB, 50.8
// with its merge (5.3 TB/s; a plain read reaches 6.4); 500 tokens, one launch, 8.4, of which a call on empty rows takes 4.2.
#pragma once

#include "attend.h"

#define NARROW_LDS(waves) ((waves) * NARROW * (HD + 4 + 2) * 4)

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
    const bool by_exp = !PLAIN && a.cap > 0.0f && a.cap <= CAP_BY_EXP;
    const Cap cap = {a.cap * LOG2E, 2.0f * LOG2E * a.cap, 2.0f * LOG2E * inv_cap};
    float qs = 0.0f;
    const auto take_queries = [&]() {
        if constexpr (DT == ODMKV_BF16) {
            const uint32_t top = column_larger(max(max(abs_max8(raw[0]), abs_max8(raw[1])), max(abs_max8(raw[2]), abs_max8(raw[3]))));
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

    Sums sums = {-INFINITY, 0.0f, NO_UNIT};
    f32x4 acc[8];
#pragma unroll
    for (int m = 0; m < 8; ++m) acc[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // raw products of a block to weights: x [tb][r] is token 64 block + 16 j + 4 tb + r.  Back come the weights as operands, in the query's unit.
    const auto weigh = [&](const f32x4* dot, int block, float ks, const Log2& u, f16x8* w) {
        float x[16];
        const float c = scale_of(ks, qs);
        const int t0 = block * BLOCK_TOKENS + 16 * j;
        if constexpr (PLAIN) {                                  // (c is not negative: the largest product is the largest score)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = dot[i >> 2][i & 3];
        } else {
            if (by_exp) {
                const float k = c * cap.plain;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = capped(dot[i >> 2][i & 3] * k, cap);
            } else if (inv_cap > 0.0f) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = cap.by * tanh_of(dot[i >> 2][i & 3] * (c * inv_cap));
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = dot[i >> 2][i & 3] * (c * LOG2E);
            }
            if (a.slopes) {
                const float ahead = (float)(s.pos - t0);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = __fmaf_rn(-slope, fabsf(ahead - (float)i), x[i]);
            }
        }
        if (block * BLOCK_TOKENS < open_from || block * BLOCK_TOKENS + BLOCK_TOKENS > open_to) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = t0 + i >= s.lo && t0 + i < s.hi ? x[i] : -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
        if constexpr (PLAIN) top = top > -INFINITY ? top * c : top;
        Terms z = terms_of(sums, u);
        if (__any(top > z.limit)) {
            const float most = column_max(top), old = raise(sums, most, most, u.lift);
            z = terms_of(sums, u);
#pragma unroll
            for (int m = 0; m < 8; ++m) acc[m] *= old;
        }
        // the factor comes out of the exponential itself, the block's sum is freed of it
        float z0 = 0.0f, z1 = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            x[i] = __builtin_amdgcn_exp2f(PLAIN ? __fmaf_rn(x[i], c, z.shift) : x[i] + z.shift);
            x[i + 1] = __builtin_amdgcn_exp2f(PLAIN ? __fmaf_rn(x[i + 1], c, z.shift) : x[i + 1] + z.shift);
            z0 += x[i];
            z1 += x[i + 1];
        }
        sums.sum = __fmaf_rn(z0 + z1, __builtin_amdgcn_exp2f(-z.factor), sums.sum);
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = (_Float16)x[i];
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
        const Log2 u_of = log2_of<KIND>(vs_of);
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
            weigh(dot, b0 + g0 + WAVES * i, read_float(ks_of, i), Log2{read_float(u_of.whole, i), read_float(u_of.rest8, i), read_float(u_of.lift, i)}, w);
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
        const int held = len - full * BLOCK_TOKENS;
        const uint4 low = first_of8(held - 16 * j), high = first_of8(held - 16 * j - 8);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            if (16 * (n >> 2) + (n & 3) + 4 * (c >> 2) >= held) k[c] = make_uint4(0, 0, 0, 0);
            v[c] = masked8(v[c], c & 1 ? high : low);
        }
        // keys by their tokens' powers (fp16 ones as they are), and the powers to the lanes that have the tokens' products
        float up_k[4], down_k[4];
        if constexpr (DT == ODMKV_BF16) {
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                const Power pk = power_for<DT>(column_larger(max(max(abs_max8(k[4 * tb]), abs_max8(k[4 * tb + 1])), max(abs_max8(k[4 * tb + 2]), abs_max8(k[4 * tb + 3])))));
                up_k[tb] = pk.up;
                down_k[tb] = pk.down;
            }
        }
        f32x4 dot[4];
#pragma unroll
        for (int tb = 0; tb < 4; ++tb) {
            dot[tb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                f16x8 x;
                if constexpr (DT == ODMKV_BF16) x = scaled_f16<DT>(k[4 * tb + kk], up_k[tb]);
                else x = __builtin_bit_cast(f16x8, k[4 * tb + kk]);
                dot[tb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[kk], dot[tb], 0, 0, 0);
            }
        }
        // values: the largest of a token's 128 lie in the sixteen lanes of its quarter, which have its weights as well
        TokenPowers<DT, 8> pv;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            uint32_t top = 0;
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const uint4& p = v[2 * m + (x >> 2)];
                top = larger_pair(top, magnitudes((x & 3) == 0 ? p.x : (x & 3) == 1 ? p.y : (x & 3) == 2 ? p.z : p.w));
            }
            pv.take(x, row_fold_pair(top));
        }
        // scores, in base 2
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float down = DT == ODMKV_BF16 ? __shfl(down_k[i >> 2], 4 * j + (i & 3)) : 1.0f, c = scale_of(down, qs), raw = dot[i >> 2][i & 3];
            x[i] = PLAIN ? raw * c : by_exp ? capped(raw * (c * cap.plain), cap) : inv_cap > 0.0f ? cap.by * tanh_of(raw * (c * inv_cap)) : raw * (c * LOG2E);
            const int t = full * BLOCK_TOKENS + 16 * j + i;
            if (!PLAIN && a.slopes) x[i] = __fmaf_rn(-slope, fabsf((float)(s.pos - t)), x[i]);
            x[i] = t >= s.lo && t < s.hi ? x[i] : -INFINITY;
        }
        float top = x[0], top_v = x[0] + pv.log2[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            top = fmaxf(top, x[i]);
            top_v = fmaxf(top_v, x[i] + pv.log2[i]);
        }
        const float old = raise(sums, column_max(top), column_max(top_v), -pv.BIAS);
#pragma unroll
        for (int m = 0; m < 8; ++m) acc[m] *= old;
        const float by = sums.ref > -INFINITY ? sums.ref : 0.0f, shift = 8.0f - pv.BIAS - sums.unit - by;
        f16x8 w[2];
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            z += __builtin_amdgcn_exp2f(x[i] - by);
            w[i >> 3][i & 7] = (_Float16)__builtin_amdgcn_exp2f(x[i] + (pv.log2[i] + shift));
        }
        sums.sum += z;
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pv.scaled(v[2 * m], 0), w[0], acc[m], 0, 0, 0);
            acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pv.scaled(v[2 * m + 1], 4), w[1], acc[m], 0, 0, 0);
        }
    }

    // every wavefront's result, of the sum of its own weights
    sums.sum = column_sum(sums.sum);
    const float own_inv = sums.sum == 0.0f ? 0.0f : 1.0f / sums.sum;
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc_of[wave][n][16 * m + 4 * j + e] = in_unit(sums, acc[m][e] * own_inv);
    if (j == 0) {
        ref_of[wave][n] = sums.ref;
        sum_of[wave][n] = sums.sum;
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
        // (a query that is not a number has a sum that is not, and a reference that may be anything)
        const float f = sum_of[w][r] == 0.0f ? 0.0f : sum_of[w][r] * __builtin_amdgcn_exp2f(ref_of[w][r] - by);
        total += f;
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

template <int DT>
static int launch_narrow_of(const AttendArgs& a, const Cut& cut, hipStream_t st) {
    const bool plain = a.cap == 0.0f && !a.slopes && a.scaling > 0.0f;
    const auto run = [&](auto dt, auto kind, auto plain_, auto waves, auto stream) {
        return launch_attend(attend_narrow_kernel<dt.value, kind.value, plain_.value, waves.value, stream.value>, a, (long long)a.p.Hkv * a.splits, waves.value,
                             NARROW_LDS(waves.value), st);
    };
    const auto of_stream = [&](auto dt, auto kind, auto plain_, auto waves) {
        return cut.stream ? run(dt, kind, plain_, waves, std::true_type()) : run(dt, kind, plain_, waves, std::false_type());
    };
    const auto of_waves = [&](auto dt, auto kind, auto plain_) { return cut.waves == 4 ? of_stream(dt, kind, plain_, Int<4>()) : of_stream(dt, kind, plain_, Int<8>()); };
    const auto of_scores = [&](auto dt, auto kind) { return plain ? of_waves(dt, kind, std::true_type()) : of_waves(dt, kind, std::false_type()); };
    const Int<DT> dt;
    return a.p.kind == ODMKV_INT8 ? of_scores(dt, Int<ODMKV_INT8>()) : of_scores(dt, Int<ODMKV_E4M3>());
}
