// Tokens into pages and tails: what the paged 8-bit cache's writing kernels (pages.hip: keys as they come; rotate.hip: turned by their positions) have in common.
#pragma once

#include "pages.h"

struct WriteArgs {
    odmkv_pages_t p;
    const uint16_t* K;
    const uint16_t* V;
    int64_t kb, kh, kt, vb, vh, vt;
    int layer, T;
};

// Where element (token, dim) of a value block lies in LDS: rows of 256 bytes, their 16-byte pieces moved by the token's quarter, so that the
// sixteen dims and four quarters that a wavefront reads at a time fall on distinct banks.
__device__ static inline int v_place(int token, int dim) { return token * HD + (((dim >> 3) ^ ((token >> 4) << 1)) << 3) + (dim & 7); }

// Keys as they come.  (What a writing kernel does with keys: which two pieces of 8 dims the x-th of a token's eight threads takes, where a row's tokens begin in K and V, and
// what becomes of two pieces of the row's `at`-th new token.)
struct KeysAsTheyCome {
    static constexpr bool ADJACENT = true;                     // a thread's pieces lie side by side, and may be taken apart
    __device__ inline int first(int x) const { return 2 * x; }
    __device__ inline int second(int x) const { return 2 * x + 1; }
    __device__ inline int64_t token0(int row, int64_t stride_b, int64_t) const { return row * stride_b; }
    template <int DT>
    __device__ inline void take(uint4& k0, uint4& k1, int, int, int64_t, int) const {
        k0 = finite8<DT>(k0);
        k1 = finite8<DT>(k1);
    }
};

// A workgroup stores one block of a row and kv-head: the largest of its values has to be known before the first code, and 64 tokens of 128 stay in registers (keys as
// they come, values once through LDS, which turns them), so that they are read once.  Bound by memory, 16 bits read and 8 written a value: 32768 tokens of 8 heads,
// 201 MB, in 40.4 us (5.0 TB/s; a large copy reaches 5.15).  The tokens pass by the caches, the codes, which the attention behind reads, do not.
template <int DT, int KIND, typename KEYS>
__device__ static inline void store_block(const WriteArgs& a, int nth, int h, int row, int start, int len, const KEYS& keys) {
    const odmkv_pages_t& p = a.p;
    const int tid = threadIdx.x;
    const int block = start / BLOCK_TOKENS + nth, open = len / BLOCK_TOKENS, slot = p.slot[row];
    const int begun = start / BLOCK_TOKENS < open ? start % BLOCK_TOKENS : 0;      // tokens of the first block, if it is completed, that the tail holds
    if (block > open) return;
    __shared__ __align__(16) uint16_t vs[BLOCK_TOKENS * HD];
    __shared__ uint32_t top[2][4];
    uint16_t* ktail = p.ktail + tail_at(p, a.layer, slot, h);
    uint16_t* vtail = p.vtail + tail_at(p, a.layer, slot, h);
    const uint16_t* K = a.K + keys.token0(row, a.kb, a.kt) + h * a.kh;
    const uint16_t* V = a.V + keys.token0(row, a.vb, a.vt) + h * a.vh;
    const int first = 8 * keys.first(tid & 7), second = 8 * keys.second(tid & 7);      // dims of a token that a thread takes
    if (block < open) {
        const int old = max(start - block * BLOCK_TOKENS, 0);  // tokens of the block that the tail holds
        const int page = p.table[(size_t)slot * p.blocks + block];
        uint4 k[2][2];                                         // sixteen dims of two tokens
        uint32_t ka = 0, va = 0;
        uint16_t was[2][16];
        if (old > 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) __builtin_memcpy(was[i], vtail + ((tid >> 2) + 64 * i) * BLOCK_TOKENS + (tid & 3) * 16, 32);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = (tid >> 3) + 32 * i, d = (tid & 7) * 16;
            if (t < old) {
                k[i][0] = *reinterpret_cast<const uint4*>(ktail + t * HD + first);
                k[i][1] = *reinterpret_cast<const uint4*>(ktail + t * HD + second);
            } else {
                const int64_t at = block * (int64_t)BLOCK_TOKENS + t - start;
                const uint16_t* vsrc = V + at * a.vt + d;
                k[i][0] = load_once(K + at * a.kt + first);
                k[i][1] = load_once(K + at * a.kt + second);
#pragma unroll
                for (int c = 0; c < 2; ++c) *reinterpret_cast<uint4*>(vs + v_place(t, d + 8 * c)) = finite8<DT>(load_once(vsrc + 8 * c));
                keys.template take<DT>(k[i][0], k[i][1], row, h, at, tid & 7);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
                ka = max(max(ka, max(abs_max_pair(k[i][c].x), abs_max_pair(k[i][c].y))), max(abs_max_pair(k[i][c].z), abs_max_pair(k[i][c].w)));
        }
        __syncthreads();
        // values: thread (dim, quarter of the tokens) of either half of the dims; what the tail holds of them lies dim by dim already
        uint16_t v[2][16];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                v[i][e] = vs[v_place((tid & 3) * 16 + e, (tid >> 2) + 64 * i)];
                if (old > 0) v[i][e] = (tid & 3) * 16 + e < old ? was[i][e] : v[i][e];
                va = max(va, (uint32_t)(v[i][e] & 0x7fffu));
            }
        }
        const int lane = tid & 63;
        const auto larger = [](float x, float y) { return __uint_as_float(max(__float_as_uint(x), __float_as_uint(y))); };
        ka = __float_as_uint(wave_fold(__uint_as_float(ka), larger));
        va = __float_as_uint(wave_fold(__uint_as_float(va), larger));
        if (lane == 0) {
            top[0][tid >> 6] = ka;
            top[1][tid >> 6] = va;
        }
        __syncthreads();
        ka = max(max(top[0][0], top[0][1]), max(top[0][2], top[0][3]));
        va = max(max(top[1][0], top[1][1]), max(top[1][2], top[1][3]));
        const float sk = block_scale<KIND>(Elem<DT>::to_f32((uint16_t)ka)), sv = block_scale<KIND>(Elem<DT>::to_f32((uint16_t)va));
        const float ik = sk > 0.0f ? __fdiv_rn(1.0f, sk) : 0.0f, iv = sv > 0.0f ? __fdiv_rn(1.0f, sv) : 0.0f;
        const size_t at = page_at(p, a.layer, page, h);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t x[4] = {k[i][c].x, k[i][c].y, k[i][c].z, k[i][c].w};
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    w[2 * c + q] = codes4<KIND>(Elem<DT>::to_f32((uint16_t)(x[2 * q] & 0xffff)), Elem<DT>::to_f32((uint16_t)(x[2 * q] >> 16)),
                                                Elem<DT>::to_f32((uint16_t)(x[2 * q + 1] & 0xffff)), Elem<DT>::to_f32((uint16_t)(x[2 * q + 1] >> 16)), sk, ik);
            }
            uint8_t* const kto = p.kcodes + at + ((tid >> 3) + 32 * i) * HD;
            if constexpr (KEYS::ADJACENT) *reinterpret_cast<uint4*>(kto + first) = make_uint4(w[0], w[1], w[2], w[3]);
            else {
                *reinterpret_cast<uint2*>(kto + first) = make_uint2(w[0], w[1]);
                *reinterpret_cast<uint2*>(kto + second) = make_uint2(w[2], w[3]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                w[q] = codes4<KIND>(Elem<DT>::to_f32(v[i][4 * q]), Elem<DT>::to_f32(v[i][4 * q + 1]), Elem<DT>::to_f32(v[i][4 * q + 2]),
                                    Elem<DT>::to_f32(v[i][4 * q + 3]), sv, iv);
            *reinterpret_cast<uint4*>(p.vcodes + at + ((tid >> 2) + 64 * i) * BLOCK_TOKENS + (tid & 3) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (tid == 0) {
            p.kscale[scale_at(p, a.layer, page, h)] = sk;
            p.vscale[scale_at(p, a.layer, page, h)] = sv;
        }
    }
    // The open block: by its own workgroup, or, where the row's first block is completed from the tail that the open one goes to, by that one, behind it.
    if (begun > 0 ? nth != 0 : block != open) return;
    __syncthreads();                                           // the old tail, and what lay in LDS, have been read
    // (tokens that complete the block that the tail had begun, with none behind them, go there as well: a token at a time, the tail takes every one)
    const int newest = start > open * BLOCK_TOKENS - BLOCK_TOKENS && len == open * BLOCK_TOKENS ? len - BLOCK_TOKENS : open * BLOCK_TOKENS;
    const int from = max(start, newest), n = len - from;
    const bool fresh = from == newest;                         // nothing of the block lies in the tail yet: its values go there by whole pieces
    if (n == 0) return;
    for (int i = tid; i < (fresh ? BLOCK_TOKENS : n) * 16; i += 256) {
        const int d = (i & 15) * 8, place = from - newest + (i >> 4);
        const int64_t at = from - start + (i >> 4);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (i >> 4 < n) v = finite8<DT>(*reinterpret_cast<const uint4*>(V + at * a.vt + d));
        if constexpr (KEYS::ADJACENT) {                        // (keys as they come: a piece by itself)
            if (i >> 4 < n) *reinterpret_cast<uint4*>(ktail + place * HD + d) = finite8<DT>(*reinterpret_cast<const uint4*>(K + at * a.kt + d));
        }
        if (fresh) *reinterpret_cast<uint4*>(vs + v_place(place, d)) = v;
        else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) vtail[(d + e) * BLOCK_TOKENS + place] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
    }
    if constexpr (!KEYS::ADJACENT) {
        for (int i = tid; i < n * 8; i += 256) {
            const int place = from - newest + (i >> 3);
            const int64_t at = from - start + (i >> 3);
            uint4 k0 = *reinterpret_cast<const uint4*>(K + at * a.kt + first), k1 = *reinterpret_cast<const uint4*>(K + at * a.kt + second);
            keys.template take<DT>(k0, k1, row, h, at, tid & 7);
            *reinterpret_cast<uint4*>(ktail + place * HD + first) = k0;
            *reinterpret_cast<uint4*>(ktail + place * HD + second) = k1;
        }
    }
    if (!fresh) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint16_t v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = vs[v_place((tid & 3) * 16 + e, (tid >> 2) + 64 * i)];
        __builtin_memcpy(vtail + ((tid >> 2) + 64 * i) * BLOCK_TOKENS + (tid & 3) * 16, v, 32);
    }
}
