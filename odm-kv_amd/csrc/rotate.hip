// Tokens into the paged 8-bit cache with their keys turned by their positions on the way, and the queries turned beside them: one launch.
//
//   a pair (a, b) of a token at position p:  (a c - b s, b c + a s),  c, s = cosine[p, i], sine[p, i],  the i-th of `turned` / 2 pairs
//
// The pairs are dims (i, i + turned / 2), or neighbours (2 i, 2 i + 1); dims from `turned` on stay as they are.  Two products and their sum, each rounded to 32 bits (the
// same bits as those three operations one by one), then once to 16 bits, as a model that turns its keys itself hands them over.  Keys are stored as pages_write stores them:
// what the cache holds hangs on the turned keys in 16 bits alone, not on how they arrive.
#include <algorithm>
#include <type_traits>
#include "pages_write.h"

struct RotateArgs {
    WriteArgs w;
    const uint16_t* q;
    int64_t qb, qh, qt;
    uint16_t* q_out;             // [rows, T, Hq, 128], packed [N, Hq, 128]
    uint16_t* k_out;             // the same of the kv-heads, or null
    const float* cosine;
    const float* sine;
    const int32_t* offsets;      // packed: where rows begin, rows + 1 of them
    const int32_t* positions;
    int64_t pb, pt;
    const int32_t* starts;
    int Hq, turned, interleaved, table, tokens;      // table: positions of cosine and sine; tokens: of the packed rows together, or T
    int heads, kv_groups, head_groups;               // query heads of a workgroup; workgroups of the keys and values; workgroups of the same queries
};

// A token's position in the table; one behind the table's ends counts as the last there, and is said to be so.
__device__ static inline int position_of(const RotateArgs& a, int row, int start, int64_t at) {
    if (!a.positions) {
        const int64_t p = start + at - (a.starts ? a.starts[row] : 0);                  // (padding stands at 0)
        if (p >= a.table) atomicOr(&a.w.p.status[ST_REFUSED], 1);
        return (int)(p < 0 ? 0 : p >= a.table ? a.table - 1 : p);
    }
    const int64_t first = a.offsets ? a.offsets[row] : 0;
    const int p = a.positions[row * a.pb + (first + at) * a.pt];
    if (p < 0 || p >= a.table) atomicOr(&a.w.p.status[ST_REFUSED], 1);
    return min(max(p, 0), a.table - 1);
}

// eight pairs' cosines and sines
struct Angles { float c[8], s[8]; };
__device__ static inline Angles angles_at(const RotateArgs& a, int position, int x) {
    Angles z;
    const int half = a.turned / 2;
    const float4* c = reinterpret_cast<const float4*>(a.cosine + (size_t)position * half + 8 * x);
    const float4* s = reinterpret_cast<const float4*>(a.sine + (size_t)position * half + 8 * x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 u = c[i], v = s[i];
        z.c[4 * i] = u.x; z.c[4 * i + 1] = u.y; z.c[4 * i + 2] = u.z; z.c[4 * i + 3] = u.w;
        z.s[4 * i] = v.x; z.s[4 * i + 1] = v.y; z.s[4 * i + 2] = v.z; z.s[4 * i + 3] = v.w;
    }
    return z;
}
// The two pieces of eight dims that the x-th of a token's eight threads takes: eight pairs of the dims that are turned, or two pieces of those that are not.
__device__ static inline int first_piece(int turned, int interleaved, int x) { return x < turned / 16 && !interleaved ? x : 2 * x; }
__device__ static inline int second_piece(int turned, int interleaved, int x) { return x < turned / 16 && !interleaved ? x + turned / 16 : 2 * x + 1; }

// KEY: what 32 bits do not hold counts as 0, and what 16 do not stops at the type's end, as everything that the cache holds; a query goes to 16 bits as it is
template <int DT, bool KEY>
__device__ static inline uint32_t turned_pair_16(float x, float y) {
    if constexpr (KEY) {
        x = fabsf(x) < INFINITY ? x : 0.0f;
        y = fabsf(y) < INFINITY ? y : 0.0f;
        return (uint32_t)to_16<DT>(x) | (uint32_t)to_16<DT>(y) << 16;
    } else return (uint32_t)Elem<DT>::from_f32(x) | (uint32_t)Elem<DT>::from_f32(y) << 16;
}
template <int DT, bool KEY>
__device__ static inline void turn(uint4& k0, uint4& k1, const Angles& z, bool interleaved) {
    const uint32_t w[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
    uint32_t out[8];
    const auto low = [](uint32_t v) { return Elem<DT>::to_f32((uint16_t)(v & 0xffff)); };
    const auto high = [](uint32_t v) { return Elem<DT>::to_f32((uint16_t)(v >> 16)); };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = low(w[i]), y = high(w[i]);
            out[i] = turned_pair_16<DT, KEY>(x * z.c[i] - y * z.s[i], y * z.c[i] + x * z.s[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = low(w[i]), x1 = high(w[i]), y0 = low(w[4 + i]), y1 = high(w[4 + i]);
            out[i] = turned_pair_16<DT, KEY>(x0 * z.c[2 * i] - y0 * z.s[2 * i], x1 * z.c[2 * i + 1] - y1 * z.s[2 * i + 1]);
            out[4 + i] = turned_pair_16<DT, KEY>(y0 * z.c[2 * i] + x0 * z.s[2 * i], y1 * z.c[2 * i + 1] + x1 * z.s[2 * i + 1]);
        }
    }
    k0 = make_uint4(out[0], out[1], out[2], out[3]);
    k1 = make_uint4(out[4], out[5], out[6], out[7]);
}

// new keys, turned (pages_write.h: store_block)
struct KeysTurned {
    static constexpr bool ADJACENT = false;
    const RotateArgs& a;
    int start;
    __device__ inline int first(int x) const { return first_piece(a.turned, a.interleaved, x); }
    __device__ inline int second(int x) const { return second_piece(a.turned, a.interleaved, x); }
    __device__ inline int64_t token0(int row, int64_t stride_b, int64_t stride_t) const { return a.offsets ? a.offsets[row] * stride_t : row * stride_b; }
    template <int DT>
    __device__ inline void take(uint4& k0, uint4& k1, int row, int h, int64_t at, int x) const {
        if (x < a.turned / 16) turn<DT, true>(k0, k1, angles_at(a, position_of(a, row, start, at), x), a.interleaved);
        else {
            k0 = finite8<DT>(k0);
            k1 = finite8<DT>(k1);
        }
        if (!a.k_out) return;
        uint16_t* const to = a.k_out + ((a.offsets ? a.offsets[row] + at : row * (int64_t)a.w.T + at) * a.w.p.Hkv + h) * HD;
        *reinterpret_cast<uint4*>(to + 8 * first(x)) = k0;
        *reinterpret_cast<uint4*>(to + 8 * second(x)) = k1;
    }
};

// a row's new tokens are where they are said to be
__device__ static inline bool row_fits(const RotateArgs& a, int row, int start, int len) {
    if (len < start || len - start > a.w.T) return false;
    return !a.offsets || (a.offsets[row] >= 0 && a.offsets[row + 1] <= a.tokens && a.offsets[row + 1] - (int64_t)a.offsets[row] == len - start);
}

// The first workgroups store a block of a row and kv-head each, the others turn the queries of 32 tokens: eight threads a token, which keep its eight pairs' angles for
// `heads` heads one behind the other.
//
// Bound by memory: 32768 tokens of 32 heads over 8, 738 MB of queries, keys, values and codes, in 153 us (4.8 TB/s; a large copy reaches 4.7 to 5.15).  Packed prompts of 10294 tokens, 28 heads over
// 4, in 35 us; a step of eight rows in 4.5, a launch and three round trips behind one another.  Up to four heads a workgroup (eight: 158 us for 153, packed 37 for 35), two ahead (one:
// 164).
//
// STREAM: queries pass by the caches, both ways.  Those of a prompt that the last-level cache (256 MB) would not keep until they are read again cost the codes their places there, and the
// loads themselves are faster: 32768 tokens of 32 heads (268 MB) 171 us for 158, and the cache's rows read back behind it 51 for 40.  Queries that come out of that cache (130 MB) take 38
// us, and 55 past it.
#define QUERIES_AHEAD 2
template <int DT, int KIND, bool STREAM>
__global__ __launch_bounds__(256) void pages_rotate_kernel(RotateArgs a) {
    const odmkv_pages_t& p = a.w.p;
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < a.kv_groups) {
        const int h = blockIdx.x % p.Hkv, rest = blockIdx.x / p.Hkv, row = rest % p.rows, nth = rest / p.rows;
        const int start = p.start[row], len = p.length[row];
        if (!row_fits(a, row, start, len)) {
            if (nth == 0 && h == 0 && tid == 0) atomicOr(&p.status[ST_REFUSED], 1);
            return;
        }
        if (len > start) store_block<DT, KIND>(a.w, nth, h, row, start, len, KeysTurned{a, start});
        return;
    }
    __shared__ int32_t begins[MAX_ROWS + 1];
    if (a.offsets) {
        for (int i = tid; i <= p.rows; i += 256) begins[i] = a.offsets[i];
        __syncthreads();
    }
    const int group = blockIdx.x - a.kv_groups, h0 = (group % a.head_groups) * a.heads, h1 = min(h0 + a.heads, a.Hq), x = tid & 7;
    const int64_t n = (int64_t)(group / a.head_groups) * 32 + (tid >> 3), all = a.offsets ? a.tokens : (int64_t)p.rows * a.w.T;
    if (n >= all) return;
    int row;
    int64_t at;                                                // of the row's new tokens
    if (a.offsets) {
        int lo = 0, hi = p.rows;                               // rows that begin at n or before, less one: the last of them, which is not empty if any is that has n
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (begins[mid + 1] > n) hi = mid; else lo = mid + 1;
        }
        row = lo;
        at = row < p.rows ? n - begins[row] : -1;
    } else {
        row = (int)(n / a.w.T);
        at = n - (int64_t)row * a.w.T;
    }
    bool valid = row < p.rows && at >= 0;
    int position = 0;
    if (valid) {
        const int start = p.start[row], len = p.length[row];
        valid = at < len - start && row_fits(a, row, start, len);
        if (valid && x < a.turned / 16) position = position_of(a, row, start, at);
    }
    const int d0 = 8 * first_piece(a.turned, a.interleaved, x), d1 = 8 * second_piece(a.turned, a.interleaved, x);
    const uint16_t* src = a.q + (a.offsets ? n * a.qt : row * a.qb + at * a.qt);
    uint16_t* dst = a.q_out + n * a.Hq * HD;
    if (!valid) {                                              // behind a row's tokens
        for (int h = h0; h < h1; ++h) {
            *reinterpret_cast<uint4*>(dst + h * HD + d0) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(dst + h * HD + d1) = make_uint4(0, 0, 0, 0);
        }
        if (a.k_out && h0 == 0) {
            for (int h = 0; h < p.Hkv; ++h) {
                uint16_t* const to = a.k_out + (n * p.Hkv + h) * HD;
                *reinterpret_cast<uint4*>(to + d0) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(to + d1) = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    Angles z = {};
    if (x < a.turned / 16) z = angles_at(a, position, x);
    for (int h = h0; h < h1; h += QUERIES_AHEAD) {
        uint4 q0[QUERIES_AHEAD], q1[QUERIES_AHEAD];
#pragma unroll
        for (int i = 0; i < QUERIES_AHEAD; ++i) {
            const uint16_t* const from = src + min(h + i, h1 - 1) * a.qh;
            q0[i] = STREAM ? load_once(from + d0) : *reinterpret_cast<const uint4*>(from + d0);
            q1[i] = STREAM ? load_once(from + d1) : *reinterpret_cast<const uint4*>(from + d1);
        }
#pragma unroll
        for (int i = 0; i < QUERIES_AHEAD; ++i) {
            if (h + i >= h1) break;
            if (x < a.turned / 16) turn<DT, false>(q0[i], q1[i], z, a.interleaved);
            uint16_t* const to = dst + (h + i) * HD;
            if (STREAM) {
                store_once(to + d0, q0[i]);
                store_once(to + d1, q1[i]);
            } else {
                *reinterpret_cast<uint4*>(to + d0) = q0[i];
                *reinterpret_cast<uint4*>(to + d1) = q1[i];
            }
        }
    }
}

extern "C" int odmkv_pages_write_rotated(const odmkv_rotate_t* d, void* stream) {
    ODMKV_CHECK_ARG(d && d->pages, "pages_write_rotated: null pointer");
    const odmkv_pages_t& p = *d->pages;
    if (int rc = check_layer("pages_write_rotated", &p, d->layer)) return rc;
    ODMKV_CHECK_ARG(d->T >= 0 && d->T <= (1 << 26) && d->tokens >= 0, "pages_write_rotated: bad token count");
    ODMKV_CHECK_ARG(d->Hq >= 0 && d->Hq <= 65535, "pages_write_rotated: %d query heads", d->Hq);
    ODMKV_CHECK_ARG(d->turned > 0 && d->turned <= HD && d->turned % 16 == 0, "pages_write_rotated: %d dims to turn: multiples of 16 up to %d are built", d->turned, HD);
    ODMKV_CHECK_ARG(!d->positions || !d->starts, "pages_write_rotated: positions and starts");
    if (d->T == 0 || (d->offsets && d->tokens == 0)) return 0;
    ODMKV_CHECK_ARG(d->k && d->v && d->cosine && d->sine && (d->Hq == 0 || (d->q && d->q_out)), "pages_write_rotated: null pointer");
    ODMKV_CHECK_ARG(d->table > 0, "pages_write_rotated: a table of %d positions", d->table);
    ODMKV_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->q_out | (uintptr_t)d->k_out | (uintptr_t)d->cosine | (uintptr_t)d->sine) & 15) == 0 &&
                    ((d->q_stride_b | d->q_stride_h | d->q_stride_t | d->k_stride_b | d->k_stride_h | d->k_stride_t | d->v_stride_b | d->v_stride_h | d->v_stride_t) & 7) == 0,
                    "pages_write_rotated: rows must be 16-byte aligned");
    RotateArgs a = {};
    a.w = {p, (const uint16_t*)d->k, (const uint16_t*)d->v, d->k_stride_b, d->k_stride_h, d->k_stride_t, d->v_stride_b, d->v_stride_h, d->v_stride_t, d->layer, d->T};
    a.q = (const uint16_t*)d->q;
    a.qb = d->q_stride_b;
    a.qh = d->q_stride_h;
    a.qt = d->q_stride_t;
    a.q_out = (uint16_t*)d->q_out;
    a.k_out = (uint16_t*)d->k_out;
    a.cosine = d->cosine;
    a.sine = d->sine;
    a.offsets = d->offsets;
    a.positions = d->positions;
    a.pb = d->position_stride_b;
    a.pt = d->position_stride_t;
    a.starts = d->starts;
    a.Hq = d->Hq;
    a.turned = d->turned;
    a.interleaved = d->interleaved != 0;
    a.table = d->table;
    a.tokens = d->offsets ? d->tokens : d->T;
    // a row's T tokens touch at most this many blocks
    const long long kv_groups = (long long)((d->T + BLOCK_TOKENS - 2) / BLOCK_TOKENS + 1) * p.Hkv * p.rows;
    const long long tiles = d->Hq == 0 && !d->k_out ? 0 : ((d->offsets ? (long long)d->tokens : (long long)p.rows * d->T) + 31) / 32;
    a.heads = 1;
    while (a.heads < 4 && tiles * ((d->Hq + 2 * a.heads - 1) / (2 * a.heads)) >= 4LL * compute_units()) a.heads *= 2;
    a.head_groups = std::max(1, (d->Hq + a.heads - 1) / a.heads);
    a.kv_groups = (int)kv_groups;
    const long long groups = kv_groups + tiles * a.head_groups;
    ODMKV_CHECK_ARG(groups * 256 < 0x100000000LL, "pages_write_rotated: too many tokens");
    const auto run = [&](auto dt, auto kind) {
        const bool past = (long long)(d->offsets ? 1 : p.rows) * a.tokens * d->Hq * HD * 2 > (192LL << 20);
        if (past) hipLaunchKernelGGL((pages_rotate_kernel<dt.value, kind.value, true>), dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((pages_rotate_kernel<dt.value, kind.value, false>), dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a);
    };
    const auto of_kind = [&](auto dt) {
        if (p.kind == ODMKV_INT8) run(dt, std::integral_constant<int, ODMKV_INT8>());
        else run(dt, std::integral_constant<int, ODMKV_E4M3>());
    };
    if (p.dtype == ODMKV_F16) of_kind(std::integral_constant<int, ODMKV_F16>());
    else of_kind(std::integral_constant<int, ODMKV_BF16>());
    ODMKV_CHECK_LAUNCH("pages_rotate_kernel");
    return 0;
}
