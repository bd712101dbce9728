// Attention over the paged 8-bit cache of rows that have their first blocks in common (samples, beams: pages.hip, plan of common blocks): those are read once for all rows of a group.
//
// The first workgroups of a launch take what is in common: 128 queries of a kv-head, of all rows of a group together (row by row, token by token, the heads of a token side by
// side), over a share of the group's blocks.  A wavefront holds 32 queries, the columns of v_mfma_f32_32x32x16_f16, as in the kernel for many queries (attend_wide.h): a block is turned into
// fp16 once a workgroup; where a tile has 64 queries or fewer, two wavefronts share 32 of them and take a half of every block each.  The workgroups behind them take the rows' own
// blocks (attend_narrow.h).  Both leave partial results, which a second launch puts together.  Codes, weights and sums are treated as in the other two kernels.
//
// What is left is mostly fixed cost: 64 samples of 8192 tokens (8 heads, e4m3, 52 MB that have to be read) take 33.1 us here and 7.7 in the merge, where the ordinary way reads 1.1 GB.
// 16 beams of 32768 tokens, 28 heads over 4, 31.7 and 8.4: 3 for the launch, 3 for the plan and what it leads to, 3.5 for the first of a share's 8 blocks, 15 for the others (2.1 each: one wavefront a SIMD, whose
// reads, products and weights wait for one another), 7 for the partial results.  The rows' own blocks alone take 12 to 18 and stand beside that.  Shares of 16 blocks take 47, of 4 blocks the same 31.9; partial
// results in whole rows by way of LDS no less (8 samples 17.8 -> 19); eight wavefronts, a half of a block each, leave no place for the rows' own workgroups beside them (31.7 -> 39.9).
#pragma once

#include "attend_narrow.h"

#define SHARED_LDS (2 * (BLOCK_TOKENS * HD * 2 * 2))

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT, int KIND, bool PLAIN>
__device__ static inline void attend_common(const AttendArgs& a, unsigned workgroup, uint8_t* lds) {
    const odmkv_pages_t& p = a.p;
    constexpr int WAVES = 4, THREADS = WAVES * 64, BUFFER = BLOCK_TOKENS * HD * 4, VALUES = BLOCK_TOKENS * HD * 2;
    __shared__ int range[2][WAVES];
    const int h = workgroup % p.Hkv, R = a.G * a.L;
    const CommonShare own = common_share_of(a, workgroup / p.Hkv);
    if (own.group < 0) return;
    const Plan plan(a);
    const int begin = own.begin, cols = own.cols, in_common = own.blocks, split = own.split, splits = own.splits, col0 = own.tile * SHARED_COLS, slot = own.slot;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool halves = cols - col0 <= 64;                      // two wavefronts a 32 of queries
    const int group = halves ? wave & 1 : wave, part = halves ? wave >> 1 : 0;
    const int c0 = col0 + 32 * group + col, at = min(c0, cols - 1), member = at / R, r = at - member * R, l = r / a.G, hq = h * a.G + r - l * a.G;
    const bool in = c0 < cols;                                  // (where there is no query the last one stands, and is left out at the end)
    const int row = plan.order(begin + member), len = p.length[row], count = a.counts ? min(max(a.counts[row], 0), a.L) : a.L;
    const bool valid = in && l < count;
    // ---- a block on its way: pieces of 16 codes, a token's 16 dims or a dim's 16 tokens
    constexpr int PIECES = PAGE_BYTES / 16 / THREADS;
    uint4 kc[PIECES], vc[PIECES];
    int page_of = 0;
    int b0 = split * ((in_common + splits - 1) / splits), mine = min(in_common - b0, (in_common + splits - 1) / splits);
    const auto look_up = [&](int i) { return i + lane < mine ? p.table[(size_t)slot * p.blocks + b0 + i + lane] : 0; };
    const auto request = [&](int i) {                           // block b0 + i
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
    // (asked for as if all of what is in common were seen: what each query sees is known a few reads later)
    if (mine > 0) request(0);
    Sight s = {0, 0, 0};
    if (valid) s = sight_of(a, row, len, count, l);
    s.hi = min(s.hi, in_common * BLOCK_TOKENS);
    const bool sees = valid && s.lo < s.hi;
    const int wave_lo = wave_min_int(sees ? s.lo : 0x7fffffff), wave_hi = -wave_min_int(sees ? -s.hi : 0);       // what some query of the wavefront sees
    const int open_from = -wave_min_int(valid ? -(sees ? s.lo : 0x7fffffff) : 0), open_to = wave_min_int(valid ? s.hi : 0x7fffffff);    // what all of them see
    if (lane == 0) {
        range[0][wave] = wave_lo;
        range[1][wave] = wave_hi;
    }
    __syncthreads();
    const int lo = min(min(range[0][0], range[0][1]), min(range[0][2], range[0][3])), hi = max(max(range[1][0], range[1][1]), max(range[1][2], range[1][3]));
    const int first = lo / BLOCK_TOKENS, blocks = max((hi + BLOCK_TOKENS - 1) / BLOCK_TOKENS - first, 0), share = (blocks + splits - 1) / splits;
    if (first + split * share != b0 || min(share, blocks - split * share) != mine) {
        b0 = __builtin_amdgcn_readfirstlane(first + split * share);
        mine = __builtin_amdgcn_readfirstlane(min(share, blocks - split * share));
        if (mine > 0) request(0);
    }

    f16x8 q[8];                                                 // dims 16 st + 8 half + e
    float qdown = 1.0f;
    {
        uint4 raw[8];
        const uint16_t* src = a.q + row * a.qb + hq * a.qh + l * a.ql + 8 * half;
#pragma unroll
        for (int st = 0; st < 8; ++st) raw[st] = *reinterpret_cast<const uint4*>(src + 16 * st);
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
    const bool by_exp = !PLAIN && a.cap > 0.0f && a.cap <= CAP_BY_EXP;
    const Cap cap = {a.cap * LOG2E, 2.0f * LOG2E * a.cap, 2.0f * LOG2E * inv_cap};
    const float qs = a.scaling * qdown * (PLAIN ? LOG2E : 1.0f);

    Sums sums = {-INFINITY, 0.0f, NO_UNIT};
    f32x16 acc[4];                                              // dims 32 db + 8 (r / 4) + 4 half + r % 4 of query `col`
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.0f;

    float ks_of = 0.0f;
    Log2 u_of = {0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int i = -1; i < mine; ++i) {
        uint8_t* buf = lds + (i & 1) * BUFFER;
        __syncthreads();                                        // this block lies there, and nobody reads the one before any more
        if (i + 1 < mine) put(lds + ((i + 1) & 1) * BUFFER);
        if (i + 2 < mine) request(i + 2);
        if (i < 0) continue;
        const int t0 = (b0 + i) * BLOCK_TOKENS;
        if ((i & 63) == 0) {                                    // 64 blocks' scales at a time
            const bool there = i + lane < mine;
            const int page = look_up(i);
            ks_of = there ? p.kscale[scale_at(p, a.layer, page, h)] : 0.0f;
            u_of = log2_of<KIND>(there ? p.vscale[scale_at(p, a.layer, page, h)] : 0.0f);
        }
        const float ks = read_float(ks_of, i & 63);
        const Log2 u = {read_float(u_of.whole, i & 63), read_float(u_of.rest8, i & 63), read_float(u_of.lift, i & 63)};
        if (t0 >= wave_hi || t0 + BLOCK_TOKENS <= wave_lo) continue;      // (of the wavefront's own queries none sees the block)
        const float c = scale_of(ks, qs);
        const bool cut = t0 < open_from || t0 + BLOCK_TOKENS > open_to;
        Terms z = terms_of(sums, u);
#pragma unroll 1
        for (int place = part; place < (halves ? part + 1 : 2); ++place) {
            f32x16 x;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
            for (int st = 0; st < 8; ++st) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(*key_piece(buf, 32 * place + col, 2 * st + half), q[st], x, 0, 0, 0);
            const int tl = t0 + 32 * place + 4 * half;             // token of score e: tl + 8 (e / 4) + e % 4
            if constexpr (!PLAIN) {                                // (PLAIN: they stay products)
                if (by_exp) {
                    const float k = c * cap.plain;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = capped(x[e] * k, cap);
                } else if (inv_cap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = cap.by * tanh_of(x[e] * (c * inv_cap));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] *= c * LOG2E;
                }
                if (a.slopes) {
                    const float ahead = (float)(s.pos - tl);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = __fmaf_rn(-slope, fabsf(ahead - (float)(8 * (e >> 2) + (e & 3))), x[e]);
                }
            }
            if (cut) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int t = tl + 8 * (e >> 2) + (e & 3);
                    x[e] = t >= s.lo && t < s.hi ? x[e] : -INFINITY;
                }
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
            if (PLAIN) top = top > -INFINITY ? top * c : top;      // (c is not negative: the largest product is the largest score)
            if (__any(top > z.limit)) {
                const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                const float most = fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1])), old = raise(sums, most, most, u.lift);
                z = terms_of(sums, u);
#pragma unroll
                for (int db = 0; db < 4; ++db) acc[db] *= old;
            }
            // the factor comes out of the exponential itself, the sum is freed of it
            f16x8 w[2];
            float z0 = 0.0f, z1 = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(PLAIN ? __fmaf_rn(x[e], c, z.shift) : x[e] + z.shift);
                const float p1 = __builtin_amdgcn_exp2f(PLAIN ? __fmaf_rn(x[e + 1], c, z.shift) : x[e + 1] + z.shift);
                z0 += p0;
                z1 += p1;
                w[e >> 3][e & 7] = (_Float16)p0;
                w[e >> 3][(e & 7) + 1] = (_Float16)p1;
            }
            sums.sum = __fmaf_rn(z0 + z1, __builtin_amdgcn_exp2f(-z.factor), sums.sum);
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int db = 0; db < 4; ++db)
                    acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8*>(value_piece(buf, 32 * db + col, 2 * (2 * place + st) + half)), w[st], acc[db],
                                                                     0, 0, 0);
        }
    }
    if (halves) {                                               // the second half's sums join the first's, by way of LDS
        float* const other = reinterpret_cast<float*>(lds) + group * 67 * 64 + lane;
        __syncthreads();
        if (part) {
#pragma unroll
            for (int e = 0; e < 64; ++e) other[64 * e] = acc[e >> 4][e & 15];
            other[64 * 64] = sums.ref;
            other[65 * 64] = sums.sum;
            other[66 * 64] = sums.unit;
        }
        __syncthreads();
        if (part) return;
        const Sums theirs = {other[64 * 64], other[65 * 64], other[66 * 64]};
        const float to = fmaxf(sums.ref, theirs.ref), by = to > -INFINITY ? to : 0.0f;
        const auto unit_at = [&](const Sums& s) { return s.ref > -INFINITY ? s.unit + (s.ref - by) : 2.0f * NO_UNIT; };
        const float unit = fmaxf(unit_at(sums), unit_at(theirs));
        const float mine_by = __builtin_amdgcn_exp2f(unit_at(sums) - unit), other_by = __builtin_amdgcn_exp2f(unit_at(theirs) - unit);
        sums = {to, __fmaf_rn(theirs.sum, __builtin_amdgcn_exp2f(theirs.ref - by), sums.sum * __builtin_amdgcn_exp2f(sums.ref - by)), unit};
#pragma unroll
        for (int e = 0; e < 64; ++e) acc[e >> 4][e & 15] = __fmaf_rn(other[64 * e], other_by, acc[e >> 4][e & 15] * mine_by);
    }

    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(sums.sum), __float_as_uint(sums.sum), false, false);
    const float sum = __uint_as_float(o[0]) + __uint_as_float(o[1]);
    if (!valid) return;
    const bool none = sum == 0.0f;
    const float by = none ? 0.0f : 1.0f / sum;
    const size_t to = (size_t)h * a.common_parts + own.parts + (size_t)split * cols + c0;
    float* dst = a.common_out + to * HD + 4 * half;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = none ? 0.0f : in_unit(sums, acc[db][4 * g + e] * by);
            *reinterpret_cast<f32x4*>(dst + 32 * db + 8 * g) = v;
        }
    if (half == 0) a.common_lse[to] = none ? -INFINITY : sums.ref + __builtin_amdgcn_logf(sum);
}

template <int DT, int KIND, bool PLAIN>
__global__ __launch_bounds__(256, 2) void attend_shared_kernel(AttendArgs a, unsigned in_common) {
    extern __shared__ __align__(16) uint8_t shared_lds[];
    if (blockIdx.x < in_common) attend_common<DT, KIND, PLAIN>(a, blockIdx.x, shared_lds);
    else attend_rows<DT, KIND, PLAIN, 4, false, true>(a, blockIdx.x - in_common, reinterpret_cast<float*>(shared_lds));
}

template <int DT>
static int launch_shared_of(const AttendArgs& a, int workgroups, hipStream_t st) {
    const bool plain = a.cap == 0.0f && !a.slopes && a.scaling > 0.0f;
    const unsigned in_common = (unsigned)workgroups * a.p.Hkv;
    const auto run = [&](auto kind, auto plain_) {
        const auto kernel = attend_shared_kernel<DT, kind.value, plain_.value>;
        ODMKV_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, SHARED_LDS));
        hipLaunchKernelGGL(kernel, dim3(in_common + (unsigned)a.p.Hkv * a.splits), dim3(256), SHARED_LDS, st, a, in_common);
        ODMKV_CHECK_LAUNCH("attend_shared_kernel");
        return 0;
    };
    const auto of_kind = [&](auto kind) { return plain ? run(kind, std::true_type()) : run(kind, std::false_type()); };
    return a.p.kind == ODMKV_INT8 ? of_kind(Int<ODMKV_INT8>()) : of_kind(Int<ODMKV_E4M3>());
}
