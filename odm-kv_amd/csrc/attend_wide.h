// Attention over the paged 8-bit cache for many queries of a kv-head.
//
// A wavefront holds 32 queries (the columns of v_mfma_f32_32x32x16_f16), a workgroup 32 GROUPS of them, token by token with the G heads of a
// token together, so that a workgroup's tokens lie together and blocks that none of them sees are passed over.  GROUPS is WAVES, or, for 64 queries at the most, half of
// it: two wavefronts then share 32 queries, each with a half of every block, and join at the end (29 tokens of four heads take 116 queries, 20 tokens 80: those
// fill four wavefronts).  Eight wavefronts turn a block into fp16 for twice as many queries as four: 2048 tokens of 32 heads over 12000 took 391 us for 432, over a
// window of 4096 with a cap 182 for 202; four rows of 777 with a prefix, which leave compute units without work, 46.4 for 45.9.
//
// A block of 64 tokens is turned into fp16 once a workgroup
// and lies in LDS, the next block's codes are on their way in registers; rows of the first product are tokens as they lie, and row r of a half
// wavefront's sixteen (8 (r / 4) + 4 half + r % 4) decides the order in which values lie in LDS: what a lane holds of the weights is
// then its operand of the second product.  16-byte pieces of a row are moved by the row's number (xor), so that no two of eight rows meet in a bank.
// Codes and weights are treated as in the narrow kernel: codes exact in fp16, weights rounded to it once (at most 2^-11 of themselves) in a unit of each
// query's own, products and sums fp32.
//
// Bound by the vector instructions of the softmax (a scale, a maximum, an exponential, a sum and a conversion a score; a cap takes a second exponential and a reciprocal)
// beside the matrix cores: over a window with a cap they take 64 % of the SIMDs' cycles and the matrix cores are busy 29 %; without either 48 and 39 %, with a bias 60 and 31 %.
// 2048 tokens of 32 heads over 12000: 914 TFLOP/s (a bf16 product of 8192 reaches 1429), with a bias 778, with a cap besides 633; over a window of 4096 with a cap 746; 4096
// over themselves 861; 29 tokens over 32768 35.4 us and 7.4 of the merge.
// The halves of a block, each one's vector work beside the other's products, brought 905 -> 942 TFLOP/s; where scores have a bias, one half's vector work behind the other's
// is faster instead, both halves' scores under one look for a new reference (543 -> 473 us).
#pragma once

#include "attend.h"

#define WIDE_LDS (2 * (BLOCK_TOKENS * HD * 2 * 2))
// what becomes of a product besides its factor: nothing; a cap by the exponential; a bias by distance; any of it
enum { SCORES_PLAIN, SCORES_CAPPED, SCORES_BIASED, SCORES_ANY };
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT, int KIND, int MODE, int WAVES, int GROUPS>
__global__ __launch_bounds__(WAVES * 64, 2) void attend_wide_kernel(AttendArgs a) {
    const odmkv_pages_t& p = a.p;
    constexpr bool PLAIN = MODE == SCORES_PLAIN, HALVES = GROUPS < WAVES;
    constexpr bool SIDE = MODE == SCORES_PLAIN || MODE == SCORES_CAPPED;      // a half's vector work beside the other half's products
    extern __shared__ __align__(16) uint8_t lds[];              // [2][keys 64 x 256 bytes, values 128 x 128 bytes]
    __shared__ int range[2][WAVES];
    // of the tail's tokens: pairs of largest values by wavefront; what their keys' products are multiplied by, and log2 of their values' unit
    __shared__ uint32_t tops[WAVES][BLOCK_TOKENS / 2];
    __shared__ __align__(16) float tail_down[BLOCK_TOKENS], tail_log2[BLOCK_TOKENS];
    constexpr int THREADS = WAVES * 64, BUFFER = BLOCK_TOKENS * HD * 4, VALUES = BLOCK_TOKENS * HD * 2;
    const int pairs = p.rows * p.Hkv, R = a.G * a.L, tiles = (R + 32 * GROUPS - 1) / (32 * GROUPS);
    // heads vary fastest (a die of the chip then keeps few heads' pages in its L2), the longest rows of blocks come first
    const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs, split = rest % a.splits, tile = tiles - 1 - rest / a.splits;
    const int row = pair / p.Hkv, h = pair % p.Hkv, tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave % GROUPS;
    const int part = HALVES ? wave / GROUPS : 0;                // the half of every block that this wavefront takes
    const int len = p.length[row], count = a.counts ? min(max(a.counts[row], 0), a.L) : a.L, slot = p.slot[row];
    const int r = tile * 32 * GROUPS + 32 * group + col, l = r / a.G, hq = h * a.G + r - l * a.G;
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
    const bool by_exp = MODE == SCORES_CAPPED || (!PLAIN && a.cap > 0.0f && a.cap <= CAP_BY_EXP);
    const Cap cap = {a.cap * LOG2E, 2.0f * LOG2E * a.cap, 2.0f * LOG2E * inv_cap};
    const float qs = a.scaling * qdown * (PLAIN ? LOG2E : 1.0f);

    Sums sums = {-INFINITY, 0.0f, NO_UNIT};
    f32x16 acc[4];                                              // dims 32 db + 8 (r / 4) + 4 half + r % 4 of query `col`
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.0f;

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
    const auto put_tail = [&](uint8_t* buf) {
        const uint4* kt = reinterpret_cast<const uint4*>(p.ktail + tail_at(p, a.layer, slot, h));
        const uint4* vt = reinterpret_cast<const uint4*>(p.vtail + tail_at(p, a.layer, slot, h));
        const int held = len - full * BLOCK_TOKENS;
        const auto keys_of = [&](int i) { return i >> 4 < held ? kt[i] : make_uint4(0, 0, 0, 0); };
        const auto values_of = [&](int i) { return masked8(vt[i], first_of8(held - 8 * (i & 7))); };
        uint32_t top[4] = {0, 0, 0, 0};                         // tokens 8 (tid % 8) + 2 x and the next
#pragma unroll 1
        for (int i = tid; i < TAIL_ELEMS / 8; i += THREADS) {
            uint4 k = keys_of(i);
            if constexpr (DT == ODMKV_BF16) {                   // (fp16 keys are taken as they are; a token's lie in sixteen lanes)
                const Power pk = power_for<DT>(row_fold_pair(abs_max8(k)));
                if ((i & 15) == 0) tail_down[i >> 4] = pk.down;
                k = __builtin_bit_cast(uint4, scaled_f16<DT>(k, pk.up));
            }
            *key_piece(buf, i >> 4, i & 15) = __builtin_bit_cast(f16x8, k);
            const uint4 v = values_of(i);
            top[0] = larger_pair(top[0], magnitudes(v.x));
            top[1] = larger_pair(top[1], magnitudes(v.y));
            top[2] = larger_pair(top[2], magnitudes(v.z));
            top[3] = larger_pair(top[3], magnitudes(v.w));
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int d = 8; d < 64; d <<= 1) top[x] = larger_pair(top[x], __shfl_xor(top[x], d));
            if (lane < 8) tops[wave][4 * lane + x] = top[x];
        }
        __syncthreads();
        TokenPowers<DT, 4> pv;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top[x] = larger_pair(top[x], tops[w][4 * (tid & 7) + x]);
            pv.take(x, top[x]);
            if (tid < 8) {
                tail_log2[8 * tid + 2 * x] = pv.log2[2 * x] - pv.BIAS;
                tail_log2[8 * tid + 2 * x + 1] = pv.log2[2 * x + 1] - pv.BIAS;
            }
        }
#pragma unroll 1
        for (int i = tid; i < TAIL_ELEMS / 8; i += THREADS) {
            const int dim = i >> 3, u = i & 7;
            const uint4 x = __builtin_bit_cast(uint4, pv.scaled(values_of(i), 0));
            *reinterpret_cast<uint2*>(value_piece(buf, dim, u & ~1) + 8 * (u & 1)) = make_uint2(x.x, x.y);
            *reinterpret_cast<uint2*>(value_piece(buf, dim, u | 1) + 8 * (u & 1)) = make_uint2(x.z, x.w);
        }
    };

    // half a block's keys, a quarter's values
    const auto keys_times_queries = [&](uint8_t* buf, f32x16& x, int place) {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
        for (int st = 0; st < 8; ++st) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(*key_piece(buf, 32 * place + col, 2 * st + half), q[st], x, 0, 0, 0);
    };
    const auto values_times_weights = [&](uint8_t* buf, const f16x8& w, int place) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
            acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8*>(value_piece(buf, 32 * db + col, 2 * place + half)), w, acc[db], 0, 0, 0);
    };

    const int codes = min(mine, full - b0);                     // of the blocks those that lie in pages
    if (codes > 0) request(0);
    if (WAVES == 8 && wave < 4) __builtin_amdgcn_s_setprio(2);
    float ks_of = 0.0f;
    Log2 u_of = {0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int i = -1; i < codes; ++i) {
        uint8_t* buf = lds + (i & 1) * BUFFER;
        __syncthreads();                                        // this block lies there, and nobody reads the one before any more
        if (i + 1 < codes) put(lds + ((i + 1) & 1) * BUFFER);
        else if (i + 1 < mine) put_tail(lds + ((i + 1) & 1) * BUFFER);
        if (i + 2 < codes) request(i + 2);
        if (i < 0) continue;
        const int t0 = (b0 + i) * BLOCK_TOKENS;
        if ((i & 63) == 0) {                                    // 64 blocks' scales at a time
            const bool in = i + lane < codes;
            const int page = look_up(i);
            ks_of = in ? p.kscale[scale_at(p, a.layer, page, h)] : 0.0f;
            u_of = log2_of<KIND>(in ? p.vscale[scale_at(p, a.layer, page, h)] : 0.0f);
        }
        const float ks = read_float(ks_of, i & 63);
        const Log2 u = {read_float(u_of.whole, i & 63), read_float(u_of.rest8, i & 63), read_float(u_of.lift, i & 63)};
        if (t0 >= wave_hi || t0 + BLOCK_TOKENS <= wave_lo) continue;      // (of the wavefront's own queries none sees the block)
        const float c = scale_of(ks, qs);
        const bool cut = t0 < open_from || t0 + BLOCK_TOKENS > open_to;
        f32x16 dot[2];
        f16x8 w[4];
        Terms z = terms_of(sums, u);
        const auto multiply_keys = [&](int tb, int place) { keys_times_queries(buf, dot[tb], place); };
        const auto multiply_values = [&](int st, int place) { values_times_weights(buf, w[st], place); };
        // products of half a block to scores (PLAIN: they stay products); the largest score
        const auto to_scores = [&](int tb, int place) {
            f32x16& x = dot[tb];
            const int tl = t0 + 32 * place + 4 * half;             // token of score e: tl + 8 (e / 4) + e % 4
            if constexpr (!PLAIN) {
                if (by_exp) {
                    const float k = c * cap.plain;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = capped(x[e] * k, cap);
                } else if (MODE == SCORES_ANY && inv_cap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = cap.by * tanh_of(x[e] * (c * inv_cap));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] *= c * LOG2E;
                }
                if (MODE == SCORES_BIASED || (MODE == SCORES_ANY && a.slopes)) {
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
            return PLAIN && top > -INFINITY ? top * c : top;         // (c is not negative: the largest product is the largest score)
        };
        // the sums' references where a score is to move them: what the values' sums are to be multiplied by, before weights of the new ones are, and behind those of the old
        const auto move_sums = [&](float top, float& old) {
            if (!__any(top > z.limit)) return false;
            const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            const float most = fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1]));
            old = raise(sums, most, most, u.lift);
            z = terms_of(sums, u);
            return true;
        };
        const auto multiply_sums = [&](float old) {
#pragma unroll
            for (int db = 0; db < 4; ++db) acc[db] *= old;
        };
        // the factor comes out of the exponential itself, the block's sum is freed of it
        const auto weigh = [&](int tb) {
            float z0 = 0.0f, z1 = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(PLAIN ? __fmaf_rn(dot[tb][e], c, z.shift) : dot[tb][e] + z.shift);
                const float p1 = __builtin_amdgcn_exp2f(PLAIN ? __fmaf_rn(dot[tb][e + 1], c, z.shift) : dot[tb][e + 1] + z.shift);
                z0 += p0;
                z1 += p1;
                w[2 * tb + (e >> 3)][e & 7] = (_Float16)p0;
                w[2 * tb + (e >> 3)][(e & 7) + 1] = (_Float16)p1;
            }
            sums.sum = __fmaf_rn(z0 + z1, __builtin_amdgcn_exp2f(-z.factor), sums.sum);
        };
        // SIDE: the two halves' vector work stands beside the other half's matrix work: a matrix instruction takes 32 cycles, which some eight vector instructions fill.
        multiply_keys(0, part);
        const float top = to_scores(0, part);
        float old;
        if constexpr (HALVES) {
            if (move_sums(top, old)) multiply_sums(old);
            weigh(0);
            multiply_values(0, 2 * part);
            multiply_values(1, 2 * part + 1);
        } else if constexpr (!SIDE) {
            multiply_keys(1, 1);
            if (move_sums(fmaxf(top, to_scores(1, 1)), old)) multiply_sums(old);
            weigh(0);
            weigh(1);
#pragma unroll
            for (int st = 0; st < 4; ++st) multiply_values(st, st);
        } else {
            if (move_sums(top, old)) multiply_sums(old);
            multiply_keys(1, 1);
            weigh(0);
            const bool moved = move_sums(to_scores(1, 1), old);
            multiply_values(0, 0);
            multiply_values(1, 1);
            weigh(1);
            if (moved) multiply_sums(old);
            multiply_values(2, 2);
            multiply_values(3, 3);
        }
    }
    // the open block, last of its row: a power of two a token, a half of it behind the other
    if (mine > 0 && codes < mine) {
        uint8_t* buf = lds + (codes & 1) * BUFFER;
        __syncthreads();
        const int t0 = full * BLOCK_TOKENS;
        const bool none_seen = t0 >= wave_hi || t0 + BLOCK_TOKENS <= wave_lo;
#pragma unroll 1
        for (int place = part; !none_seen && place < (HALVES ? part + 1 : 2); ++place) {
            f32x16 x;
            keys_times_queries(buf, x, place);
            const int tl = 32 * place + 4 * half;
            float top = -INFINITY, top_v = -INFINITY, log2_v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int at = tl + 8 * (e >> 2) + (e & 3), t = t0 + at;
                const float c = scale_of(DT == ODMKV_BF16 ? tail_down[at] : 1.0f, qs);
                x[e] = PLAIN ? x[e] * c : by_exp ? capped(x[e] * (c * cap.plain), cap) : inv_cap > 0.0f ? cap.by * tanh_of(x[e] * (c * inv_cap)) : x[e] * (c * LOG2E);
                if (!PLAIN && a.slopes) x[e] = __fmaf_rn(-slope, fabsf((float)(s.pos - t)), x[e]);
                x[e] = t >= s.lo && t < s.hi ? x[e] : -INFINITY;
                log2_v[e] = tail_log2[at];
                top = fmaxf(top, x[e]);
                top_v = fmaxf(top_v, x[e] + log2_v[e]);
            }
            const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            const auto ov = __builtin_amdgcn_permlane32_swap(__float_as_uint(top_v), __float_as_uint(top_v), false, false);
            const float old = raise(sums, fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1])), fmaxf(__uint_as_float(ov[0]), __uint_as_float(ov[1])), 0.0f);
#pragma unroll
            for (int db = 0; db < 4; ++db) acc[db] *= old;
            const float by = sums.ref > -INFINITY ? sums.ref : 0.0f, shift = 8.0f - sums.unit - by;
            f16x8 w[2];
            float z = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                z += __builtin_amdgcn_exp2f(x[e] - by);
                w[e >> 3][e & 7] = (_Float16)__builtin_amdgcn_exp2f(x[e] + (log2_v[e] + shift));
            }
            sums.sum += z;
            values_times_weights(buf, w[0], 2 * place);
            values_times_weights(buf, w[1], 2 * place + 1);
        }
    }
    if constexpr (HALVES) {                                     // the second half's sums join the first's, by way of LDS
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
    float by = none ? 0.0f : 1.0f / sum;
    const float lse2 = none ? -INFINITY : sums.ref + __builtin_amdgcn_logf(sum);
    if (__any(sums.unit < -60.0f)) {                            // (a factor of its own, which the reciprocal need not take to where fp32 ends)
#pragma unroll
        for (int e = 0; e < 64; ++e) acc[e >> 4][e & 15] = in_unit(sums, acc[e >> 4][e & 15]);
    } else by *= __builtin_amdgcn_exp2f(sums.unit - 8.0f);
    const auto result = [&](int db, int e) { return none ? 0.0f : acc[db][e] * by; };
    if (a.splits > 1) {
        const size_t unit_at = ((size_t)pair * a.splits + split) * R + r;
        float* dst = a.part_out + unit_at * HD + 4 * half;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = result(db, 4 * g + e);
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
                v[e] = (uint32_t)to_16<DT>(result(db, 4 * g + 2 * e)) | (uint32_t)to_16<DT>(result(db, 4 * g + 2 * e + 1)) << 16;
            *reinterpret_cast<uint2*>(dst + 32 * db + 8 * g) = make_uint2(v[0], v[1]);
        }
    if (a.lse && half == 0) a.lse[((size_t)row * a.Hq + hq) * a.L + l] = none ? -INFINITY : lse2 * LN2;
}

template <int DT>
static int launch_wide_of(const AttendArgs& a, const Cut& cut, hipStream_t st) {
    const bool capped = a.cap > 0.0f;
    const int R = a.G * a.L, mode = a.slopes ? (capped ? SCORES_ANY : SCORES_BIASED)
                                  : capped ? (a.cap <= CAP_BY_EXP ? SCORES_CAPPED : SCORES_ANY) : a.scaling > 0.0f ? SCORES_PLAIN : SCORES_ANY;
    const long long groups = (long long)a.p.rows * a.p.Hkv * a.splits * ((R + 32 * cut.groups - 1) / (32 * cut.groups));
    const auto run = [&](auto dt, auto kind, auto mode_, auto waves, auto groups_) {
        return launch_attend(attend_wide_kernel<dt.value, kind.value, mode_.value, waves.value, groups_.value>, a, groups, waves.value, WIDE_LDS, st);
    };
    const auto of_waves = [&](auto dt, auto kind, auto mode_) {
        if (cut.groups == 2) return run(dt, kind, mode_, Int<4>(), Int<2>());
        return cut.waves == 4 ? run(dt, kind, mode_, Int<4>(), Int<4>()) : run(dt, kind, mode_, Int<WIDE_WAVES>(), Int<WIDE_WAVES>());
    };
    const auto of_mode = [&](auto dt, auto kind) {
        switch (mode) {
            case SCORES_PLAIN: return of_waves(dt, kind, Int<SCORES_PLAIN>());
            case SCORES_CAPPED: return of_waves(dt, kind, Int<SCORES_CAPPED>());
            case SCORES_BIASED: return of_waves(dt, kind, Int<SCORES_BIASED>());
            default: return of_waves(dt, kind, Int<SCORES_ANY>());
        }
    };
    const Int<DT> dt;
    return a.p.kind == ODMKV_INT8 ? of_mode(dt, Int<ODMKV_INT8>()) : of_mode(dt, Int<ODMKV_E4M3>());
}
