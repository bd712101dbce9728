// Attention of whole prompts over their own keys and values in 16 bits: grouped heads, sequences of their own lengths packed one behind the other, later chunks (fewer
// queries than keys), with a cap and a window.
//
//   x_j = scaling q . k_j, capped;  out = sum_j softmax(x)_j v_j over lo <= j < hi
//
// A wavefront holds 32 queries (the columns of the 32x32x16 matrix instructions), a workgroup WAVES times as many, token by token with the G heads of a token together, so that
// a workgroup's tokens lie together: a block of 64 keys and values serves all heads of the group, and few blocks lie across a query's end.  The rows of the first product are
// tokens; what a lane holds of the weights is its operand of the second product as it is, whose other operand, values dim by dim, comes out of LDS by transposing reads.
// Blocks go from memory into LDS without passing through registers, the next one on its way while this one is used: one barrier a block.
//
// Bound by the products and by the vector work that finds no place beside them: 16384 tokens, 32 heads over 8, in 2.02 ms, 1085 TFLOP/s (a library's product of 8192^3: 1219 to 1429;
// this kernel without any vector work: 1245), matrix cores busy 52 % of the cycles, vector instructions 43 %.  A product of 32 cycles takes 18 ns, a 16-byte read of LDS beside it 6
// more, its share of the vector work 5: so operands are read as rarely as 32 queries a wavefront allow (64 would not leave room for two wavefronts a SIMD), without bank conflicts,
// and the largest score of a block is not looked for.  With a cap 34 % and 57 %: 12001 tokens in a window of 4096 in 419 us.  Prompts of 1500 tokens on average, 28 heads over 4, 455 us
// (800 TFLOP/s): some twenty tiles of four wavefronts a compute unit, each with a first block to wait for and a last one that few queries see whole.  One prompt of 1024, 2048, 3000 or 4096 tokens,
// 32 heads over 8: 32, 62, 93 and 144 us (272, 556, 794 and 957 TFLOP/s): one round of tiles up to some 3000, as long as the last of them, which sees all keys.
//
// A query's bits hang on the 31 others of its wavefront: weights are made in one of two ways, and sums a second time, for all of them together.  Both ways are as far from the formula as they may be, and
// the same call gives the same bits.
#include <algorithm>
#include "attend.h"
#include "spans.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

#define PROMPT_COLS(waves) (32 * (waves))
#define PROMPT_TILE (BLOCK_TOKENS * HD * 2)                      // bytes of a block of keys, or of values
#define PROMPT_LDS(waves) (2 * PROMPT_TILE + max(2 * PROMPT_TILE, (waves) * 32 * HD * 2))

struct PromptArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    int64_t qb, qh, qt, kb, kh, kt, vb, vh, vt;
    uint16_t* out;               // [rows, L, Hq, 128], packed [L, Hq, 128]
    float* lse;                  // [rows, Hq, L], packed [Hq, L]
    const int32_t* offsets;      // packed: where the rows' queries begin, rows + 1 of them; L and T are all rows' together then
    const int32_t* key_offsets;
    const int32_t* starts;
    int rows, L, T, Hq, Hkv, G, causal, window;
    float scaling, cap;
    int splits;                  // workgroups that share a tile's blocks
    int larger;                  // 0: equal shares; or how many 1024ths of them the first of two has
    float* part_out;             // [splits, queries in all, Hq, 128]
    float* part_lse;             // the same without the 128, base 2
};

// a tile of queries: of row `row` (-1: of none, queries that no row has), n of them from q0 on, over m keys from k0 on
struct Tile { int row, nth, q0, n, k0, m; };

// Packed rows' tiles one behind the other, before and behind them those of the queries that no row has.  What offsets say is kept within what there is.
template <int COLS>
__device__ static inline Tile tile_of(const PromptArgs& a, int at) {
    if (!a.offsets) {
        const int tiles = (a.G * a.L + COLS - 1) / COLS, nth = tiles - 1 - at / a.rows;         // (the last tiles see most: they come first)
        return {nth < 0 ? -2 : at % a.rows, nth, 0, a.L, 0, a.T};
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = -1; s0 <= a.rows; s0 += 64) {
        const int s = s0 + lane;
        const Span here = s <= a.rows ? span_of(s < 0 ? 0 : a.offsets[s], s == a.rows ? a.L : a.offsets[s + 1], a.L) : Span{0, 0};
        const int count = (int)(((int64_t)a.G * here.n + COLS - 1) / COLS), upto = before + wave_scan(count);
        const unsigned long long behind = __ballot(upto > at);
        if (behind) {
            const int l = __builtin_ctzll(behind), row = s0 + l, nth = __builtin_amdgcn_readlane(upto, l) - 1 - at;
            const int q0 = __builtin_amdgcn_readlane(here.begin, l), n = __builtin_amdgcn_readlane(here.n, l);
            if (row < 0 || row >= a.rows) return {-1, nth, q0, n, 0, 0};
            const int32_t* const of = a.key_offsets ? a.key_offsets : a.offsets;
            const Span keys = span_of(of[row], of[row + 1], a.T);
            return {row, nth, q0, n, keys.begin, keys.n};
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return {-2, 0, 0, 0, 0, 0};
}

// operands of the matrix instructions
template <int DT>
__device__ static inline f32x16 multiply(const uint4& x, const uint4& y, const f32x16& to) {
    if constexpr (DT == ODMKV_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), to, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), to, 0, 0, 0);
}
template <int DT>
__device__ static inline uint32_t pair_16(float x, float y) {
    if constexpr (DT == ODMKV_F16) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)x, (_Float16)y});
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((__attribute__((ext_vector_type(2))) float){x, y}, __attribute__((ext_vector_type(2))) __bf16));
}

// Values' weights are rounded, those in the weights' sum are not: of fp16 values at the type's end a mean may come out 2^-11 past it, which would be infinite, and is stopped there
// (two packed instructions behind the conversion; in 32 bits in front of it they took 2 %, and what was rounded once was rounded twice).  An infinity, and what is not a number, stay that where they are
// said to be `odd`.  bf16 needs no stop: one weight is exactly one, and the others of values at the type's end are less than 2^-8 together, or their sum is past 32 bits and made once more.
template <int DT>
__device__ static inline uint32_t stopped_pair(uint32_t w, bool odd_low, bool odd_high) {
    if constexpr (DT != ODMKV_F16) return w;
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
    const u16x2 below = {(uint16_t)(odd_low ? 0xffff : 0xfbff), (uint16_t)(odd_high ? 0xffff : 0xfbff)};      // (of numbers below 0 as they lie there the larger ones are the lower ones)
    const i16x2 above = {(int16_t)(odd_low ? 0x7fff : 0x7bff), (int16_t)(odd_high ? 0x7fff : 0x7bff)};
    const u16x2 x = __builtin_elementwise_min(__builtin_bit_cast(u16x2, w), below);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(i16x2, x), above));
}

// Weights go to 16 bits relative to a reference, a score of the query's own: its weight is 2^LIFT, and where the sum of sixteen weights passes LIMIT the reference moves to the
// largest score.  fp16: so no weight passes the type's end, and one below its normal numbers is off by 2^-25, 2^-33 of the largest at the most; bf16 has the range of 32 bits.
template <int DT> struct Weights {
    static constexpr float LIFT = DT == ODMKV_F16 ? 8.0f : 0.0f, LIMIT = 32768.0f;
};

// (without conflicts: 1 % of the time of 16384 tokens)
__device__ static inline int value_turn(int t) { return (t & 3) << 1 | (t >> 2 & 1); }

template <int DT, int MODE, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void prompt_kernel(PromptArgs a) {
    constexpr bool PLAIN = MODE == 0, by_exp = MODE == 1;       // 1: a cap by the exponential; 2: a larger one, or a scaling that is not above 2^-100
    constexpr int COLS = PROMPT_COLS(WAVES), PIECES = PROMPT_TILE / 16 / (WAVES * 64);
    constexpr float LIFT = Weights<DT>::LIFT;
    extern __shared__ __align__(16) uint8_t smem[];             // [2][keys 64 x 256 bytes, values 64 x 256 bytes]
    __shared__ int range[2][WAVES];
    // heads vary fastest: a die of the chip then keeps few heads' keys and values in its L2
    // (of unequal shares the larger ones come first, all of them)
    const int h = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, tiles = gridDim.x / a.Hkv / a.splits, split = a.larger ? rest / tiles : rest % a.splits;
    const Tile tile = tile_of<COLS>(a, a.larger ? rest - split * tiles : rest / a.splits);
    if (tile.row < -1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    const int r = tile.nth * COLS + 32 * wave + col, l = r / a.G, hq = h * a.G + r - l * a.G;
    const bool valid = l < tile.n;
    const int row = max(tile.row, 0), pos = tile.m - tile.n + l;
    int lo = 0, hi = 0;
    if (valid && tile.row >= 0) {
        lo = a.starts ? max(a.starts[row], 0) : 0;
        if (a.window > 0) lo = max(lo, pos - a.window + 1);
        hi = a.causal ? max(pos + 1, 0) : tile.m;
    }
    const bool sees = lo < hi;
    const auto least = [](int x) { return __builtin_amdgcn_readfirstlane(wave_min_int(x)); };
    const int wave_lo = least(sees ? lo : 0x7fffffff), wave_hi = -least(sees ? -hi : 0);                        // what some query of the wavefront sees
    const int open_from = -least(valid ? -(sees ? lo : 0x7fffffff) : 0), open_to = least(valid ? hi : 0x7fffffff);      // what all of them see
    if (lane == 0) {
        range[0][wave] = wave_lo;
        range[1][wave] = wave_hi;
    }
    __syncthreads();
    int from = range[0][0], upto = range[1][0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        from = min(from, range[0][w]);
        upto = max(upto, range[1][w]);
    }
    const int first = from / BLOCK_TOKENS, blocks = max((upto + BLOCK_TOKENS - 1) / BLOCK_TOKENS - first, 0);
    const int share = a.larger ? (int)(((int64_t)blocks * a.larger + 1023) / 1024) : (blocks + a.splits - 1) / a.splits;
    const int b0 = __builtin_amdgcn_readfirstlane(first + split * share), mine = __builtin_amdgcn_readfirstlane(min(a.larger && split ? blocks : share, blocks - split * share));

    // 16-byte piece p of token t lies at p ^ (t % 16) of the token's place; of values 32-byte pieces at p ^ value_turn(t): what half a wavefront reads at a time, 32 bytes of
    // two pieces of four tokens, falls on distinct banks.
    // Tokens behind the row's end repeat its last one and are masked.
    const uint16_t* const K = a.k + (a.offsets ? tile.k0 * a.kt : row * a.kb) + h * a.kh;
    const uint16_t* const V = a.v + (a.offsets ? tile.k0 * a.vt : row * a.vb) + h * a.vh;
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)smem;
    uint32_t key_from[PIECES], value_from[PIECES];              // bytes from a block's first token
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        const int e = tid + WAVES * 64 * c, t = e >> 4, p = e & 15;
        key_from[c] = 2 * (t * (int)a.kt + 8 * (p ^ (t & 15)));
        value_from[c] = 2 * (t * (int)a.vt + 8 * (p ^ (value_turn(t) << 1)));
    }
    const auto request = [&](int i) {
        const int t0 = (b0 + i) * BLOCK_TOKENS, behind = tile.m - 1 - t0;
        const uint16_t* const keys = K + t0 * a.kt;
        const uint16_t* const values = V + t0 * a.vt;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            const uint32_t to = lds0 + (i & 1) * 2 * PROMPT_TILE + (WAVES * 64 * c + 64 * wave) * 16;
            uint32_t of_key = key_from[c], of_value = value_from[c];
            if (behind < BLOCK_TOKENS - 1) {
                const int over = max(((tid + WAVES * 64 * c) >> 4) - behind, 0);
                of_key -= 2 * over * (int)a.kt;
                of_value -= 2 * over * (int)a.vt;
            }
            request_to_lds(keys, of_key, to);
            request_to_lds(values, of_value, to + PROMPT_TILE);
        }
    };
    if (mine > 0) request(0);

    // The queries come the same way, four rows a request, behind the first block's place.
    const uint32_t queries_at = lds0 + 2 * PROMPT_TILE + wave * 32 * HD * 2;
    {
        const int at = min(l, tile.n - 1);
        const uint64_t src = (uint64_t)(a.q + (a.offsets ? (int64_t)(tile.q0 + at) * a.qt : row * a.qb + at * a.qt) + hq * a.qh);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int of = 4 * j + (lane >> 4);
            const uint64_t from = (uint64_t)(uint32_t)__shfl((int)(src >> 32), of) << 32 | (uint32_t)__shfl((int)src, of);
            request_to_lds((const uint16_t*)from + (((lane ^ of) & 15) << 3), queries_at + 1024 * j);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    uint4 q[8];                                                 // dims 16 st + 8 half + e; of the last query where there is none
#pragma unroll
    for (int st = 0; st < 8; ++st) {
        const u32x4 x = *(const __attribute__((address_space(3))) u32x4*)(size_t)(queries_at + col * 256 + (((2 * st + half) ^ (col & 15)) << 4));
        q[st] = make_uint4(x[0], x[1], x[2], x[3]);
    }
    const float inv_cap = !PLAIN && a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    const Cap cap = {a.cap * LOG2E, 2.0f * LOG2E * a.cap, 2.0f * LOG2E * inv_cap};
    const float c = PLAIN ? a.scaling * LOG2E : a.scaling;
    const auto score = [&](float x) {                           // of a product, base 2
        return PLAIN ? x * c : by_exp ? capped(x * (c * cap.plain), cap) : inv_cap > 0.0f ? cap.by * tanh_of(x * (c * inv_cap)) : x * (c * LOG2E);
    };

    float ref = -INFINITY, sum = 0.0f;
    f32x16 acc[4];                                              // dims 32 db + 8 (e / 4) + 4 half + e % 4 of query `col`
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[db][e] = 0.0f;

    // where a lane's operands lie in LDS, of the first buffer: of token `col` its pieces 2 st + half; of values four dims of a token, of which the lane gets four tokens of a dim
    uint32_t key_at[8], value_at[4];
    const int value_token = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int st = 0; st < 8; ++st) key_at[st] = lds0 + col * 256 + (((2 * st + half) ^ (col & 15)) << 4);
#pragma unroll
    for (int db = 0; db < 4; ++db) value_at[db] = lds0 + PROMPT_TILE + value_token * 256 + (((2 * db + (lane >> 4 & 1)) ^ value_turn(value_token)) << 5) + ((lane & 3) << 3);

    float shift = INFINITY;                                     // LIFT - ref; what a score is to have added on its way into the exponential
    // Half a block's products to weights, and their sum.  Vector work is what there is too much of beside the products, so that the largest score is not looked for: where the
    // sum says that a weight may have grown too large, or nothing has been seen yet (the sum is infinite then, or not a number), they are made once more.
    const auto weigh = [&](const f32x16& x, uint4* w) {
        float z0 = 0.0f, z1 = 0.0f;
        uint32_t word[8];
        const auto weight = [&](float y) {
            if constexpr (PLAIN) return __builtin_amdgcn_exp2f(__fmaf_rn(y, c, shift));
            else if constexpr (MODE == 1) return __builtin_amdgcn_exp2f(__fmaf_rn(-cap.twice, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * (c * cap.plain))), cap.by + shift));
            else return __builtin_amdgcn_exp2f(score(y) + shift);
        };
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float p0 = weight(x[e]), p1 = weight(x[e + 1]);
            z0 += p0;
            z1 += p1;
            word[e >> 1] = pair_16<DT>(p0, p1);
        }
        w[0] = make_uint4(word[0], word[1], word[2], word[3]);
        w[1] = make_uint4(word[4], word[5], word[6], word[7]);
        return z0 + z1;
    };
    // Once more: what is not seen is left out, the reference moves to the largest score where that is above it, each query's by itself, and the sums with it.
    const auto weigh_again = [&](const f32x16& x, uint4* w, int tl, bool cut) {
        float y[16], top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int t = tl + 8 * (e >> 2) + (e & 3);
            y[e] = !cut || (t >= lo && t < hi) ? score(x[e]) : -INFINITY;
            top = fmaxf(top, y[e]);
        }
        const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        const float most = fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1])), to = most > ref + 2.0f ? most : ref;
        const float old = ref > -INFINITY ? __builtin_amdgcn_exp2f(ref - to) : 1.0f;
        sum *= old;
#pragma unroll
        for (int db = 0; db < 4; ++db) acc[db] *= old;
        ref = to;
        shift = to > -INFINITY ? LIFT - to : INFINITY;
        float z = 0.0f;
        uint32_t word[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float p0 = __builtin_amdgcn_exp2f(y[e] + (to > -INFINITY ? shift : 0.0f)), p1 = __builtin_amdgcn_exp2f(y[e + 1] + (to > -INFINITY ? shift : 0.0f));
            z += p0 + p1;
            word[e >> 1] = pair_16<DT>(p0, p1);
        }
        w[0] = make_uint4(word[0], word[1], word[2], word[3]);
        w[1] = make_uint4(word[4], word[5], word[6], word[7]);
        return z;
    };
    const auto block = [&](auto buffer_, int t0) {
        constexpr uint32_t buffer = buffer_.value * 2 * PROMPT_TILE;
        const bool cut = t0 < open_from || t0 + BLOCK_TOKENS > open_to;
        f32x16 dot[2];
        uint4 w[4];
        const auto multiply_keys = [&](int tb) {
            typedef const __attribute__((address_space(3))) u32x4* place;
#pragma unroll
            for (int e = 0; e < 16; ++e) dot[tb][e] = 0.0f;
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                const u32x4 x = *(place)(size_t)(key_at[st] + (buffer + 32 * 256 * tb));
                dot[tb] = multiply<DT>(make_uint4(x[0], x[1], x[2], x[3]), q[st], dot[tb]);
            }
        };
        const auto multiply_values = [&](int st) {
            typedef __attribute__((address_space(3))) s16x4* place;
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                const uint32_t at = value_at[db] + (buffer + 16 * 256 * st);
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(size_t)at), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(size_t)(at + 8 * 256));
                const uint2 u = __builtin_bit_cast(uint2, x), v = __builtin_bit_cast(uint2, y);
                acc[db] = multiply<DT>(make_uint4(u.x, u.y, v.x, v.y), w[st], acc[db]);
            }
        };
        const int tl = t0 + 4 * half;                           // token of score e: tl + 8 (e / 4) + e % 4
        multiply_keys(0);
        // one half's vector work stands beside the other's products
        multiply_keys(1);
        float z = INFINITY;
        if (PLAIN || !cut) z = weigh(dot[0], w);                // (under a cap it is work that counts; without, products of the other half stand beside it)
        if (cut || __any(!(z <= Weights<DT>::LIMIT))) z = weigh_again(dot[0], w, tl, cut);
        sum += z;
        multiply_values(0);
        multiply_values(1);
        if (PLAIN || !cut) z = weigh(dot[1], w + 2);
        if (cut || __any(!(z <= Weights<DT>::LIMIT))) z = weigh_again(dot[1], w + 2, tl + 32, cut);
        sum += z;
        multiply_values(2);
        multiply_values(3);
    };
    const auto turn = [&](int i, auto buffer) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // this block has come, and nobody reads the one before any more
        if (i + 1 < mine) request(i + 1);
        const int t0 = (b0 + i) * BLOCK_TOKENS;
        if (t0 < wave_hi && t0 + BLOCK_TOKENS > wave_lo) block(buffer, t0);           // (of the wavefront's own queries some see the block)
    };
#pragma unroll 1
    for (int i = 0; i < mine; i += 2) {
        turn(i, Int<0>());
        if (i + 1 < mine) turn(i + 1, Int<1>());
    }

    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(o[0]) + __uint_as_float(o[1]);
    const bool none = sum == 0.0f;
    float by = none ? 0.0f : 1.0f / sum;
    const float lse2 = none ? -INFINITY : ref - LIFT + __builtin_amdgcn_logf(sum);
    // A value that is not finite has spoilt the queries that do not see its token as well (0 times it is not 0), and bf16 values at the type's end may have passed 32 bits: their
    // sums are made once more, token by token, of what is seen alone, and of halves of the values.
    bool spoilt = false;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) spoilt |= !(fabsf(acc[db][e]) < INFINITY);
    bool odd = spoilt || !(sum < INFINITY);                     // (or will not be a number)
    if (__any(spoilt && sum < INFINITY)) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[db][e] = 0.0f;
        const int t_from = max(wave_lo, b0 * BLOCK_TOKENS), t_upto = min(wave_hi, (b0 + mine) * BLOCK_TOKENS);
#pragma unroll 1
        for (int t = t_from; t < t_upto; ++t) {
            float x = 0.0f;
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                const uint4 u = *reinterpret_cast<const uint4*>(K + (int64_t)t * a.kt + 16 * st + 8 * half);
                const uint32_t kw[4] = {u.x, u.y, u.z, u.w}, qw[4] = {q[st].x, q[st].y, q[st].z, q[st].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x = __fmaf_rn(Elem<DT>::to_f32((uint16_t)(kw[e] & 0xffff)), Elem<DT>::to_f32((uint16_t)(qw[e] & 0xffff)), x);
                    x = __fmaf_rn(Elem<DT>::to_f32((uint16_t)(kw[e] >> 16)), Elem<DT>::to_f32((uint16_t)(qw[e] >> 16)), x);
                }
            }
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            x = __uint_as_float(both[0]) + __uint_as_float(both[1]);
            const bool seen = t >= lo && t < hi;
            const float p = seen ? __builtin_amdgcn_exp2f(score(x) - lse2) : 0.0f;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint2 u = *reinterpret_cast<const uint2*>(V + (int64_t)t * a.vt + 32 * db + 8 * g + 4 * half);
                    const uint32_t vw[2] = {u.x, u.y};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = 0.5f * Elem<DT>::to_f32((uint16_t)(vw[e >> 1] >> (16 * (e & 1))));
                        acc[db][4 * g + e] = seen ? __fmaf_rn(p, v, acc[db][4 * g + e]) : acc[db][4 * g + e];
                    }
                }
        }
        // (an infinite value that is seen stays one; what is finite ends where the type does)
        constexpr float HALF_MOST = DT == ODMKV_F16 ? 32752.0f : 1.6947656946257677e38f;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[db][e] = fabsf(acc[db][e]) < INFINITY ? __builtin_amdgcn_fmed3f(acc[db][e], -HALF_MOST, HALF_MOST) : acc[db][e];
        by = 2.0f;
        odd = true;
    }
    const auto result = [&](int db, int e) { return none ? 0.0f : acc[db][e] * by; };
    const int64_t nth = (a.offsets ? 0 : (int64_t)row * a.L) + tile.q0 + l;                         // of all queries
    // Through the wavefront's own part of LDS, which nobody reads any more, so that a store writes four whole rows; 8 bytes of a row each, as the lanes hold them, took 4 % longer
    // for packed prompts of up to 2999 tokens (454 us for 436, the queries' way among it), 25 % for queries over 64 keys.
    uint8_t* const rows_at = smem + wave * 32 * HD * 2;
    const uint32_t to = valid ? (uint32_t)(nth * a.Hq + hq) : 0xffffffffu;
    const auto rows_of = [&](auto write) {                      // 256 bytes of each row: write(row's place in the outputs, its 16 bytes)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int of = 4 * j + (lane >> 4);
            const uint4 x = *reinterpret_cast<const uint4*>(rows_at + of * 256 + (((lane ^ of) & 15) << 4));
            const uint32_t at = (uint32_t)__shfl((int)to, of);
            if (at != 0xffffffffu) write(at, x);
        }
        __builtin_amdgcn_wave_barrier();
    };
    __syncthreads();
    if (a.splits > 1) {
        const int64_t all = a.offsets ? a.L : (int64_t)a.rows * a.L, part = split * all * a.Hq;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
#pragma unroll
            for (int db = 0; db < 2; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = result(2 * side + db, 4 * g + e);
                    *reinterpret_cast<f32x4*>(rows_at + col * 256 + (((8 * db + 2 * g + half) ^ (col & 15)) << 4)) = x;
                }
            rows_of([&](uint32_t at, const uint4& x) { *reinterpret_cast<uint4*>(a.part_out + (part + at) * HD + 64 * side + 4 * (lane & 15)) = x; });
        }
        if (valid && half == 0) a.part_lse[part + to] = lse2;
        return;
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint32_t x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) x[e] = stopped_pair<DT>(pair_16<DT>(result(db, 4 * g + 2 * e), result(db, 4 * g + 2 * e + 1)), odd, odd);
            *reinterpret_cast<uint2*>(rows_at + col * 256 + (((4 * db + g) ^ (col & 15)) << 4) + 8 * half) = make_uint2(x[0], x[1]);
        }
    rows_of([&](uint32_t at, const uint4& x) { *reinterpret_cast<uint4*>(a.out + (int64_t)at * HD + 8 * (lane & 15)) = x; });
    if (valid && a.lse && half == 0) a.lse[((a.offsets ? 0 : (int64_t)row * a.Hq) + hq) * a.L + tile.q0 + l] = lse2 * LN2;
}

// The shares of a query's blocks, put together by their log-sum-exps: half a wavefront a query, a lane four dims.  Bound by memory: two shares of 2048 queries of 24 heads, 63 MB, in 13 us
// (4.8 TB/s).  bf16: the weights, of one at most each, meet the values smaller by a power of two that takes their sum to a half or below: values at the type's end are as good as at 32 bits' own.
template <int DT>
__global__ __launch_bounds__(256) void prompt_merge_kernel(PromptArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t all = a.offsets ? a.L : (int64_t)a.rows * a.L, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (at >= all * a.Hq) return;
    float top = -INFINITY, sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[s * all * a.Hq + at]);
    const float by = top > -INFINITY ? top : 0.0f;
    const int less = DT == ODMKV_F16 ? 0 : 33 - __builtin_clz(a.splits);
    const float down = __builtin_amdgcn_ldexpf(1.0f, -less);
#pragma unroll 2
    for (int s = 0; s < a.splits; ++s) {
        const float w = __builtin_amdgcn_exp2f(a.part_lse[s * all * a.Hq + at] - by);
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.part_out + (s * all * a.Hq + at) * HD + 4 * lane);
        sum += w;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __fmaf_rn(w * down, v[e], o[e]);
    }
    const float inv = sum == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(1.0f / sum, less);
    const auto odd = [&](int e) { return !(fabsf(o[e]) < INFINITY); };
    *reinterpret_cast<uint2*>(a.out + at * HD + 4 * lane) = make_uint2(stopped_pair<DT>(pair_16<DT>(o[0] * inv, o[1] * inv), odd(0), odd(1)),
                                                                       stopped_pair<DT>(pair_16<DT>(o[2] * inv, o[3] * inv), odd(2), odd(3)));
    if (a.lse && lane == 0) {
        const int64_t nth = at / a.Hq, row = a.offsets ? 0 : nth / a.L;
        a.lse[(row * a.Hq + at % a.Hq) * a.L + nth - row * a.L] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
    }
}

// How a call is cut: wavefronts of a workgroup, tiles of queries at the most, and workgroups that share a tile's blocks.
//
// Eight wavefronts share a block among twice as many queries; two workgroups of four, which do not wait for one another, leave more of the vector work beside the products, and what a
// workgroup does before its first block and behind its last one beside the other's.  A cap is vector work above all: 12001 tokens in a window of 4096 with a cap 480 us for 429, but 16384
// without 2049 for 2141.  Few keys: 300 packed prompts of 64 tokens 169 us for 129, 40 of 500 202 for 190, 16384 tokens in a window of 700 287 for 275; a prompt of 60 tokens 10.1 for 8.8;
// the same at 16 prompts of 1500 on average (484), and at 512 keys for every query.
//
// Shares: what they are to gain is compute units that would have no tile, or none in the last round; what they cost is their partial results.
struct PromptCut { int waves; long long tiles; int splits, larger; };
static PromptCut cut_of(bool packed, int rows, int G, int Hkv, int L, int T, bool causal, int window, bool capped) {
    PromptCut c;
    const int keys = packed ? T / rows : T, of_tile = causal && L == T ? keys / 2 : keys;          // what a tile sees, about
    c.waves = capped || (window > 0 ? std::min(of_tile, window) : of_tile) <= 768 ? 4 : 8;
    const long long cols = PROMPT_COLS(c.waves), slots = compute_units() * (8 / c.waves);
    c.tiles = packed ? ((long long)G * L + cols - 1) / cols + rows + 2 : (long long)rows * (((long long)G * L + cols - 1) / cols);
    const long long blocks = (window > 0 ? std::min((long long)keys, window + cols / G) : keys) / BLOCK_TOKENS + 1, groups = c.tiles * Hkv;
    // in units of a block's time, about a microsecond: a workgroup's fixed part is some four of them, the merge a launch and its reading
    const double partial = (double)(packed ? 1 : rows) * L * G * Hkv * (HD + 1) * 4 * 2 / 5e6;
    double least = 0.0;
    c.splits = 1;
    c.larger = 0;
    for (int s = 1; s <= 128 && (s == 1 || s * 4LL <= blocks) && (s == 1 || groups * s <= 4 * slots); ++s) {
        const double cost = (double)((groups * s + slots - 1) / slots) * ((double)blocks / s + 4.0) + (s > 1 ? 4.0 + s * partial : 0.0);
        if (s > 1 && cost >= least) continue;
        least = cost;
        c.splits = s;
    }
    // Two unequal shares, where tiles leave compute units without one: those take the smaller shares, `turns` one after the other, in the time that a larger one takes.
    // (2048 queries over 12800 keys, 24 heads over 8, 192 tiles: 386 us with whole tiles, 346 with shares of 76 and 24 %, of which 12 put them together.)
    if (groups < slots) {
        const double turns = (double)((groups + slots - groups - 1) / (slots - groups)), smaller = (blocks + 4.0 - 4.0 * turns) / (turns + 1.0), cost = blocks - smaller + 8.0 + 2 * partial;
        if (smaller >= 4.0 && cost < least) {
            c.splits = 2;
            c.larger = 1024 - (int)(1024.0 * smaller / blocks);
        }
    }
    return c;
}

extern "C" size_t odmkv_prompt_attend_workspace_bytes(int packed, int rows, int Hq, int Hkv, int L, int T, int causal, int window, float cap) {
    if (rows <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || L <= 0 || T < 0) return 0;
    const PromptCut c = cut_of(packed != 0, rows, Hq / Hkv, Hkv, L, T, causal != 0, window, cap > 0.0f);
    return c.splits > 1 ? align_up((size_t)c.splits * (packed ? 1 : rows) * L * Hq * (HD + 1) * sizeof(float), 256) : 0;
}

extern "C" int odmkv_prompt_attend(const odmkv_prompt_attend_t* d, void* stream) {
    ODMKV_CHECK_ARG(d != nullptr, "prompt_attend: null pointer");
    ODMKV_CHECK_ARG(d->dtype == ODMKV_F16 || d->dtype == ODMKV_BF16, "prompt_attend: bad dtype %d", d->dtype);
    ODMKV_CHECK_ARG(d->rows > 0 && d->L >= 0 && d->T >= 0 && d->L <= (1 << 26) && d->T <= (1 << 26) && d->rows <= (1 << 20), "prompt_attend: bad shape");
    ODMKV_CHECK_ARG(d->Hkv > 0 && d->Hq > 0 && d->Hq % d->Hkv == 0 && d->Hq <= 65535, "prompt_attend: %d query heads over %d kv-heads", d->Hq, d->Hkv);
    ODMKV_CHECK_ARG(d->window >= 0 && (d->window == 0 || d->causal), "prompt_attend: bad window");
    ODMKV_CHECK_ARG(d->cap == 0.0f || (d->cap >= 0x1p-100f && d->cap < INFINITY), "prompt_attend: bad cap");
    ODMKV_CHECK_ARG(!d->key_offsets || d->offsets, "prompt_attend: the keys' offsets without the queries'");
    if (d->L == 0) return 0;
    ODMKV_CHECK_ARG(d->q && d->out && ((d->k && d->v) || d->T == 0), "prompt_attend: null pointer");
    ODMKV_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->out) & 15) == 0 &&
                    ((d->q_stride_b | d->q_stride_h | d->q_stride_t | d->k_stride_b | d->k_stride_h | d->k_stride_t | d->v_stride_b | d->v_stride_h | d->v_stride_t) & 7) == 0,
                    "prompt_attend: rows must be 16-byte aligned");
    ODMKV_CHECK_ARG(d->k_stride_t >= 0 && d->k_stride_t < (1 << 24) && d->v_stride_t >= 0 && d->v_stride_t < (1 << 24), "prompt_attend: a token's stride must be below 2^24");
    const int G = d->Hq / d->Hkv;
    const PromptCut cut = cut_of(d->offsets != nullptr, d->rows, G, d->Hkv, d->L, d->T, d->causal != 0, d->window, d->cap > 0.0f);
    const long long all = d->offsets ? d->L : (long long)d->rows * d->L, groups = cut.tiles * d->Hkv * cut.splits;
    ODMKV_CHECK_ARG((long long)G * d->L < 0x7fff0000LL && groups * cut.waves * 64 < 0x100000000LL && all * d->Hq < 0x100000000LL, "prompt_attend: too many queries");
    const size_t need = odmkv_prompt_attend_workspace_bytes(d->offsets != nullptr, d->rows, d->Hq, d->Hkv, d->L, d->T, d->causal, d->window, d->cap);
    if (need > 0 && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < need)) {
        odmkv_set_error("prompt_attend: workspace too small");
        return ODMKV_ENOSPACE;
    }
    float* const parts = (float*)d->workspace;
    const PromptArgs a = {(const uint16_t*)d->q, (const uint16_t*)d->k, (const uint16_t*)d->v, d->q_stride_b, d->q_stride_h, d->q_stride_t, d->k_stride_b, d->k_stride_h,
                          d->k_stride_t, d->v_stride_b, d->v_stride_h, d->v_stride_t, (uint16_t*)d->out, d->lse, d->offsets, d->key_offsets, d->starts, d->rows, d->L, d->T,
                          d->Hq, d->Hkv, G, d->causal != 0, d->window, d->scaling, std::min(d->cap, LARGEST_CAP), cut.splits, cut.larger, parts, parts + (size_t)cut.splits * all * d->Hq * HD};
    const int mode = d->cap > 0.0f ? (d->cap <= CAP_BY_EXP ? 1 : 2) : d->scaling > 0x1p-100f ? 0 : 2;
    const hipStream_t st = (hipStream_t)stream;
    const auto run = [&](auto dt, auto mode_, auto waves) {
        const auto kernel = prompt_kernel<dt.value, mode_.value, waves.value>;
        ODMKV_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, PROMPT_LDS(waves.value)));
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(waves.value * 64), PROMPT_LDS(waves.value), st, a);
        ODMKV_CHECK_LAUNCH("prompt_kernel");
        if (cut.splits > 1) {
            hipLaunchKernelGGL(prompt_merge_kernel<dt.value>, dim3((unsigned)((all * d->Hq + 7) / 8)), dim3(256), 0, st, a);
            ODMKV_CHECK_LAUNCH("prompt_merge_kernel");
        }
        return 0;
    };
    const auto of_waves = [&](auto dt, auto mode_) { return cut.waves == 8 ? run(dt, mode_, Int<8>()) : run(dt, mode_, Int<4>()); };
    const auto of_mode = [&](auto dt) { return mode == 0 ? of_waves(dt, Int<0>()) : mode == 1 ? run(dt, Int<1>(), Int<4>()) : of_waves(dt, Int<2>()); };
    return d->dtype == ODMKV_F16 ? of_mode(Int<ODMKV_F16>()) : of_mode(Int<ODMKV_BF16>());
}
