// The paged 8-bit cache without its attention: bookkeeping on the device (lengths, tables, holders of a page), tokens into pages
// and tails, dense rows back, forks, rewinds and compaction.  Full pages are never written again, so that a fork shares them by a
// count and copies the 16-bit tail alone: nothing is copied on a later write.
#include <algorithm>
#include "pages_write.h"

#define BOOK_THREADS 1024

// one whole number a row: from the device, from the host by way of the launch's arguments, or the same for all
struct RowInts {
    const int32_t* device;
    int all, from_host;
    int32_t host[ODMKV_PAGES_HOST_ROWS];
};
__device__ static inline int row_int(const RowInts& a, int row) { return a.device ? a.device[row] : a.from_host ? a.host[row] : a.all; }
static int make_row_ints(const char* who, RowInts& a, int rows, const int32_t* device, const int32_t* host, int all) {
    ODMKV_CHECK_ARG(!device || !host, "%s: numbers from the device and from the host", who);
    ODMKV_CHECK_ARG(!host || rows <= ODMKV_PAGES_HOST_ROWS, "%s: %d rows' numbers from the host", who, rows);
    a.device = device;
    a.all = all;
    a.from_host = host != nullptr;
    for (int i = 0; i < ODMKV_PAGES_HOST_ROWS; ++i) a.host[i] = host && i < rows ? host[i] : 0;
    return 0;
}

// ---- bookkeeping ----------------------------------------------------------------------------------
// inclusive prefix sum over the workgroup's threads; total: of all.  part: one int a wavefront.
__device__ static inline int book_scan(int v, int* part, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();                                           // part of the scan before has been read
    if (lane == 63) part[wave] = v;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < BOOK_THREADS / 64; ++w) {
        const int x = part[w];
        if (w < wave) before += x;
        total += x;
    }
    return before + v;
}

// everything that decides what the other kernels look at is cleared; codes and scales of pages that no row holds are never read
__global__ __launch_bounds__(256) void pages_init_kernel(odmkv_pages_t p) {
    const size_t i0 = (size_t)blockIdx.x * 256 + threadIdx.x, step = (size_t)gridDim.x * 256;
    for (size_t i = i0; i < (size_t)p.pages; i += step) p.refs[i] = 0;
    for (size_t i = i0; i < (size_t)p.rows * p.blocks; i += step) p.table[i] = 0;
    const size_t pieces = (size_t)p.layers * p.rows * p.Hkv * (TAIL_ELEMS / 8);
    for (size_t i = i0; i < pieces; i += step) {
        reinterpret_cast<uint4*>(p.ktail)[i] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(p.vtail)[i] = make_uint4(0, 0, 0, 0);
    }
    for (size_t i = i0; i < (size_t)p.rows; i += step) {
        p.length[i] = p.start[i] = 0;
        p.slot[i] = (int)i;
    }
    if (i0 == 0) {
        p.status[ST_FREE] = p.pages;
        p.status[ST_HINT] = p.status[ST_REFUSED] = p.status[ST_LIVE] = 0;
    }
}

extern "C" int odmkv_pages_init(const odmkv_pages_t* p, void* stream) {
    if (int rc = check_pages("pages_init", p)) return rc;
    hipLaunchKernelGGL(pages_init_kernel, dim3(1024), dim3(256), 0, (hipStream_t)stream, *p);
    ODMKV_CHECK_LAUNCH("pages_init_kernel");
    return 0;
}

// One workgroup, a thread a row; the lowest free pages are found by going over the holders' counts from the hint on, and each goes to
// the row and block of its rank.  Bound by its launch and two or three dependent reads: 4 us for a row's 512 pages, 5 for a
// token of 16 rows, 10 for 16 rows that fill 4096 pages at once.
__global__ __launch_bounds__(BOOK_THREADS) void pages_extend_kernel(odmkv_pages_t p, RowInts counts, int max_count) {
    __shared__ int part[BOOK_THREADS / 64], upto[MAX_ROWS], first[MAX_ROWS], slots[MAX_ROWS];
    __shared__ int refused, last;
    const int tid = threadIdx.x;
    int len = 0, c = 0, need = 0;
    bool bad = false;
    if (tid == 0) refused = last = 0;
    if (tid < p.rows) {
        len = p.length[tid];
        c = row_int(counts, tid);
        bad = c < 0 || c > max_count;
        if (bad) c = 0;
        const long long held = (long long)p.blocks * BLOCK_TOKENS + BLOCK_TOKENS - 1;
        bad = bad || (long long)len + c > (p.max_tokens > 0 ? min((long long)p.max_tokens, held) : held);
        if (!bad) need = (len + c) / BLOCK_TOKENS - len / BLOCK_TOKENS;
        first[tid] = len / BLOCK_TOKENS;
        slots[tid] = p.slot[tid];
    }
    int total;
    const int sum = book_scan(need, part, total);
    if (tid < MAX_ROWS) upto[tid] = sum;
    if (bad) atomicOr(&refused, 1);
    const int free_pages = p.status[ST_FREE], hint = p.status[ST_HINT];
    __syncthreads();
    if (refused || total > free_pages) {
        if (tid < p.rows) p.start[tid] = len;
        if (tid == 0) p.status[ST_REFUSED] = 1;
        return;
    }
    int found = 0;
    for (int base = hint; found < total && base < p.pages; base += BOOK_THREADS) {
        const int page = base + tid;
        const bool is_free = page < p.pages && p.refs[page] == 0;
        int n;
        const int rank = found + book_scan(is_free ? 1 : 0, part, n) - 1;
        found += n;
        if (!is_free || rank >= total) continue;
        int lo = 0, hi = p.rows - 1;                           // the first row whose blocks reach past this rank
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto[mid] > rank) hi = mid; else lo = mid + 1;
        }
        p.table[(size_t)slots[lo] * p.blocks + first[lo] + rank - (lo ? upto[lo - 1] : 0)] = page;
        p.refs[page] = 1;
        if (rank == total - 1) last = page + 1;
    }
    __syncthreads();
    if (tid < p.rows) {
        p.start[tid] = len;
        p.length[tid] = len + c;
    }
    if (tid == 0 && total > 0) {
        p.status[ST_FREE] = free_pages - total;
        p.status[ST_HINT] = last;
    }
}

extern "C" int odmkv_pages_extend(const odmkv_pages_t* p, const int32_t* counts, const int32_t* counts_host, int count, int max_count, void* stream) {
    if (int rc = check_pages("pages_extend", p)) return rc;
    ODMKV_CHECK_ARG(max_count >= 0 && (counts || counts_host || (count >= 0 && count <= max_count)), "pages_extend: bad count");
    RowInts c;
    if (int rc = make_row_ints("pages_extend", c, p->rows, counts, counts_host, count)) return rc;
    hipLaunchKernelGGL(pages_extend_kernel, dim3(1), dim3(BOOK_THREADS), 0, (hipStream_t)stream, *p, c, max_count);
    ODMKV_CHECK_LAUNCH("pages_extend_kernel");
    return 0;
}

// ---- tokens into pages and tails ------------------------------------------------------------------
template <int DT, int KIND>
__global__ __launch_bounds__(256) void pages_write_kernel(WriteArgs a) {
    const int row = blockIdx.z, start = a.p.start[row], len = a.p.length[row];
    if (len <= start || len - start > a.T) return;
    store_block<DT, KIND>(a, blockIdx.x, blockIdx.y, row, start, len, KeysAsTheyCome());
}

extern "C" int odmkv_pages_write(const odmkv_pages_t* p, int layer, const void* K, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t,
                                 const void* V, int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, int T, void* stream) {
    if (int rc = check_layer("pages_write", p, layer)) return rc;
    ODMKV_CHECK_ARG(T >= 0, "pages_write: bad token count");
    if (T == 0) return 0;
    ODMKV_CHECK_ARG(K && V, "pages_write: null pointer");
    ODMKV_CHECK_ARG((((uintptr_t)K | (uintptr_t)V) & 15) == 0 && ((k_stride_b | k_stride_h | k_stride_t | v_stride_b | v_stride_h | v_stride_t) & 7) == 0,
                    "pages_write: rows must be 16-byte aligned");
    const WriteArgs a = {*p, (const uint16_t*)K, (const uint16_t*)V, k_stride_b, k_stride_h, k_stride_t, v_stride_b, v_stride_h, v_stride_t, layer, T};
    // tokens of T touch at most this many blocks
    const dim3 grid((unsigned)((T + BLOCK_TOKENS - 2) / BLOCK_TOKENS + 1), p->Hkv, p->rows);
    PAGES_DISPATCH(pages_write_kernel, p, grid, dim3(256), 0, (hipStream_t)stream, a);
    ODMKV_CHECK_LAUNCH("pages_write_kernel");
    return 0;
}

// ---- dense rows back ------------------------------------------------------------------------------
// A workgroup a block and kv-head: keys as they lie, values through LDS.  Bound by memory, as the way in: 201 MB in 40.7 us (4.9 TB/s); stores past the caches took longer
// (both ways and the bookkeeping 107 us for 100).
template <int DT, int KIND, int OUT>
__global__ __launch_bounds__(256) void pages_read_kernel(odmkv_pages_t p, int layer, typename Elem<OUT>::raw* K, typename Elem<OUT>::raw* V, int T) {
    const int row = blockIdx.z, h = blockIdx.y, block = blockIdx.x, tid = threadIdx.x;
    const int len = p.length[row], open = len / BLOCK_TOKENS, slot = p.slot[row];
    __shared__ float vs[BLOCK_TOKENS * (HD + 1)];
    float k[2][16];
    const bool full = block < open, tail = block == open && len > open * BLOCK_TOKENS;
    const int t0 = block * BLOCK_TOKENS, held = min(len - t0, BLOCK_TOKENS);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) k[i][e] = 0.0f;
    if (full || tail) {
        const int page = full ? p.table[(size_t)slot * p.blocks + block] : 0;
        const size_t at = page_at(p, layer, page, h), tat = tail_at(p, layer, slot, h);
        const float sk = full ? p.kscale[scale_at(p, layer, page, h)] : 0.0f, sv = full ? p.vscale[scale_at(p, layer, page, h)] : 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = (tid >> 3) + 32 * i, d = (tid & 7) * 16, vd = (tid >> 2) + 64 * i, vt = (tid & 3) * 16;
            float v[16];
            if (full) {
                const uint4 kc = *reinterpret_cast<const uint4*>(p.kcodes + at + t * HD + d);
                const uint4 vc = *reinterpret_cast<const uint4*>(p.vcodes + at + vd * BLOCK_TOKENS + vt);
                const uint32_t kw[4] = {kc.x, kc.y, kc.z, kc.w}, vw[4] = {vc.x, vc.y, vc.z, vc.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    values4<KIND>(kw[q], k[i] + 4 * q);
                    values4<KIND>(vw[q], v + 4 * q);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    k[i][e] *= sk;
                    v[e] *= sv;
                }
            } else {
                uint16_t kt[16], vt16[16];
                __builtin_memcpy(kt, p.ktail + tat + t * HD + d, 32);
                __builtin_memcpy(vt16, p.vtail + tat + vd * BLOCK_TOKENS + vt, 32);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    k[i][e] = t < held ? Elem<DT>::to_f32(kt[e]) : 0.0f;
                    v[e] = vt + e < held ? Elem<DT>::to_f32(vt16[e]) : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) vs[(vt + e) * (HD + 1) + vd] = v[e];
        }
        __syncthreads();
    }
    const auto narrow = [](float x) -> typename Elem<OUT>::raw {
        if constexpr (OUT == ODMKV_F32) return x;
        else return to_16<OUT>(x);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = (tid >> 3) + 32 * i, d = (tid & 7) * 16;
        if (t0 + t >= T) continue;
        const size_t to = (((size_t)row * p.Hkv + h) * T + t0 + t) * HD + d;
        typename Elem<OUT>::raw ko[16], vo[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            ko[e] = narrow(k[i][e]);
            vo[e] = full || tail ? narrow(vs[t * (HD + 1) + d + e]) : narrow(0.0f);
        }
        constexpr int W = 16 / (int)sizeof(ko[0]);
#pragma unroll
        for (int c = 0; c < 16 / W; ++c) {
            uint4 kv, vv;
            __builtin_memcpy(&kv, ko + c * W, 16);
            __builtin_memcpy(&vv, vo + c * W, 16);
            *reinterpret_cast<uint4*>(K + to + c * W) = kv;
            *reinterpret_cast<uint4*>(V + to + c * W) = vv;
        }
    }
}
template <int DT, int KIND>
static void launch_read(const odmkv_pages_t* p, int layer, void* K, void* V, int out_dtype, int T, dim3 grid, hipStream_t st) {
    if (out_dtype == ODMKV_F16) hipLaunchKernelGGL((pages_read_kernel<DT, KIND, ODMKV_F16>), grid, dim3(256), 0, st, *p, layer, (uint16_t*)K, (uint16_t*)V, T);
    else if (out_dtype == ODMKV_BF16) hipLaunchKernelGGL((pages_read_kernel<DT, KIND, ODMKV_BF16>), grid, dim3(256), 0, st, *p, layer, (uint16_t*)K, (uint16_t*)V, T);
    else hipLaunchKernelGGL((pages_read_kernel<DT, KIND, ODMKV_F32>), grid, dim3(256), 0, st, *p, layer, (float*)K, (float*)V, T);
}

extern "C" int odmkv_pages_read(const odmkv_pages_t* p, int layer, void* K, void* V, int out_dtype, int T, void* stream) {
    if (int rc = check_layer("pages_read", p, layer)) return rc;
    ODMKV_CHECK_ARG(T >= 0, "pages_read: bad token count");
    ODMKV_CHECK_ARG(out_dtype == ODMKV_F16 || out_dtype == ODMKV_BF16 || out_dtype == ODMKV_F32, "pages_read: bad dtype %d", out_dtype);
    if (T == 0) return 0;
    ODMKV_CHECK_ARG(K && V && (((uintptr_t)K | (uintptr_t)V) & 15) == 0, "pages_read: null or unaligned pointer");
    const dim3 grid((unsigned)((T + BLOCK_TOKENS - 1) / BLOCK_TOKENS), p->Hkv, p->rows);
    hipStream_t st = (hipStream_t)stream;
    if (p->dtype == ODMKV_F16 && p->kind == ODMKV_INT8) launch_read<ODMKV_F16, ODMKV_INT8>(p, layer, K, V, out_dtype, T, grid, st);
    else if (p->dtype == ODMKV_F16) launch_read<ODMKV_F16, ODMKV_E4M3>(p, layer, K, V, out_dtype, T, grid, st);
    else if (p->kind == ODMKV_INT8) launch_read<ODMKV_BF16, ODMKV_INT8>(p, layer, K, V, out_dtype, T, grid, st);
    else launch_read<ODMKV_BF16, ODMKV_E4M3>(p, layer, K, V, out_dtype, T, grid, st);
    ODMKV_CHECK_LAUNCH("pages_read_kernel");
    return 0;
}

// ---- forks ----------------------------------------------------------------------------------------
// What the copying kernel does for a row: the slot that is copied and its tokens, the slot that takes the copy and the full blocks it gives up.
struct Move { int from, to, length, dropped; };      // to < 0: nothing

// One workgroup, a thread a row: 4 us, a launch and its reads.  A parent's slot goes to the row itself if it stays, or else to its first child; every other row takes a
// slot that no row uses any more, both in ascending order.
__global__ __launch_bounds__(BOOK_THREADS) void pages_plan_kernel(odmkv_pages_t p, const int64_t* parents, RowInts known, Move* moves) {
    __shared__ int part[BOOK_THREADS / 64], slots[MAX_ROWS], lengths[MAX_ROWS], heir[MAX_ROWS], owner[MAX_ROWS], unused[MAX_ROWS];
    __shared__ int refused;
    const int tid = threadIdx.x, rows = p.rows;
    const bool mine = tid < rows;
    int64_t parent = 0;
    if (tid == 0) refused = 0;
    heir[tid] = rows;
    if (mine) {
        slots[tid] = p.slot[tid];
        lengths[tid] = p.length[tid];
        parent = parents ? parents[tid] : row_int(known, tid);
    }
    __syncthreads();
    if (mine) owner[slots[tid]] = tid;                         // which row a slot belongs to
    const bool bad = mine && (parent < 0 || parent >= rows);
    if (bad) atomicOr(&refused, 1);
    __syncthreads();
    if (refused) {
        if (mine) moves[tid] = {0, -1, 0, 0};
        if (tid == 0) p.status[ST_REFUSED] = 1;
        return;
    }
    if (mine) atomicMin(&heir[parent], parent == tid ? -1 : tid);
    __syncthreads();
    const bool takes_over = mine && (parent == tid || heir[parent] == tid);
    int n;
    // unused slots in ascending order: those of rows that are nobody's parent
    const bool idle = mine && heir[owner[tid]] == rows;        // (tid as a slot)
    const int at = book_scan(idle ? 1 : 0, part, n) - 1;
    if (idle) unused[at] = tid;
    const int rank = book_scan(mine && !takes_over ? 1 : 0, part, n) - 1;      // (its barriers come between the list and its readers)
    if (!mine) return;
    const int from = slots[parent], len = lengths[parent];
    if (takes_over) {
        p.slot[tid] = from;
        moves[tid] = {0, -1, 0, 0};
    } else {
        const int to = unused[rank];
        p.slot[tid] = to;
        moves[tid] = {from, to, len, lengths[owner[to]] / BLOCK_TOKENS};
    }
    p.length[tid] = p.start[tid] = len;
}

// the rows of another batch over the same pages: every row is copied
__global__ __launch_bounds__(BOOK_THREADS) void pages_plan_select_kernel(odmkv_pages_t p, odmkv_pages_t to, const int64_t* parents, Move* moves) {
    __shared__ int refused;
    const int tid = threadIdx.x;
    const bool mine = tid < to.rows;
    int64_t parent = 0;
    if (tid == 0) refused = 0;
    __syncthreads();
    if (mine) {
        parent = parents[tid];
        if (parent < 0 || parent >= p.rows) atomicOr(&refused, 1);
    }
    __syncthreads();
    if (refused) {
        if (mine) moves[tid] = {0, -1, 0, 0};
        if (tid == 0) p.status[ST_REFUSED] = 1;
        return;
    }
    if (!mine) return;
    const int len = p.length[parent];
    moves[tid] = {p.slot[parent], to.slot[tid], len, 0};
    to.length[tid] = to.start[tid] = len;
}

// Pages that lose a holder; those that lose their last are free.  A wavefront's are counted together before the pool's words are touched.
struct Freed { int count, lowest; };
__device__ static inline void drop_page(const odmkv_pages_t& p, int page, Freed& f) {
    if (atomicSub(&p.refs[page], 1) == 1) {
        f.count += 1;
        f.lowest = min(f.lowest, page);
    }
}
__device__ static inline void give_back(const odmkv_pages_t& p, const Freed& f) {      // by all lanes of a wavefront
    const auto add = [](float x, float y) { return __int_as_float(__float_as_int(x) + __float_as_int(y)); };
    const auto less = [](float x, float y) { return __int_as_float(min(__float_as_int(x), __float_as_int(y))); };
    const int count = __float_as_int(wave_fold(__int_as_float(f.count), add)), lowest = __float_as_int(wave_fold(__int_as_float(f.lowest), less));
    if (count > 0 && (threadIdx.x & 63) == 0) {
        atomicAdd(&p.status[ST_FREE], count);
        atomicMin(&p.status[ST_HINT], lowest);
    }
}

// blockIdx.y == 0: the table row, and who holds its pages (whole-number atomics: their order changes nothing); from 1 on: a layer and head's tail.
// A copied page has its source's row for a holder throughout: its count does not pass zero.  Bound by the latency of a table's and a tail's reads behind the plan's: 8 us
// for 8 of 16 rows, four layers of 8 heads (32 KB of tails read and written a row, layer and head: 17 MB).
__global__ __launch_bounds__(256) void pages_move_kernel(odmkv_pages_t p, odmkv_pages_t to, const Move* moves) {
    const Move m = moves[blockIdx.x];
    if (m.to < 0) return;
    const int tid = threadIdx.x;
    if (blockIdx.y == 0) {
        const int full = m.length / BLOCK_TOKENS;
        const int32_t* src = p.table + (size_t)m.from * p.blocks;
        int32_t* dst = to.table + (size_t)m.to * to.blocks;
        Freed freed = {0, 0x7fffffff};
        for (int j = tid; j < to.blocks; j += 256) {
            const int was = j < m.dropped ? dst[j] : -1, is = src[j];
            dst[j] = is;
            if (j < full) atomicAdd(&p.refs[is], 1);
            if (was >= 0) drop_page(p, was, freed);
        }
        give_back(p, freed);
        return;
    }
    const int lh = blockIdx.y - 1, layer = lh / p.Hkv, h = lh % p.Hkv;
    const size_t src = tail_at(p, layer, m.from, h), dst = tail_at(to, layer, m.to, h);
    for (int i = tid; i < TAIL_ELEMS / 8; i += 256) {
        reinterpret_cast<uint4*>(to.ktail + dst)[i] = reinterpret_cast<const uint4*>(p.ktail + src)[i];
        reinterpret_cast<uint4*>(to.vtail + dst)[i] = reinterpret_cast<const uint4*>(p.vtail + src)[i];
    }
}

extern "C" size_t odmkv_pages_reorder_workspace_bytes(int rows) { return rows > 0 ? align_up((size_t)rows * sizeof(Move), 256) : 0; }

static int launch_moves(const odmkv_pages_t* p, const odmkv_pages_t* to, const Move* moves, hipStream_t st) {
    ODMKV_CHECK_ARG((long long)p->layers * p->Hkv < 65535, "pages: more than 65534 layers and heads");
    hipLaunchKernelGGL(pages_move_kernel, dim3(to->rows, 1 + p->layers * p->Hkv), dim3(256), 0, st, *p, *to, moves);
    ODMKV_CHECK_LAUNCH("pages_move_kernel");
    return 0;
}

extern "C" int odmkv_pages_reorder(const odmkv_pages_t* p, const int64_t* parents, const int32_t* parents_host, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    if (int rc = check_pages("pages_reorder", p)) return rc;
    ODMKV_CHECK_ARG((parents != nullptr) != (parents_host != nullptr), "pages_reorder: parents from the device or from the host");
    RowInts known;
    if (int rc = make_row_ints("pages_reorder", known, p->rows, nullptr, parents_host, 0)) return rc;
    ODMKV_CHECK_ARG((long long)p->layers * p->Hkv < 65535, "pages_reorder: more than 65534 layers and heads");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < odmkv_pages_reorder_workspace_bytes(p->rows)) {
        odmkv_set_error("pages_reorder: workspace too small");
        return ODMKV_ENOSPACE;
    }
    hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(BOOK_THREADS), 0, (hipStream_t)stream, *p, parents, known, (Move*)workspace);
    ODMKV_CHECK_LAUNCH("pages_plan_kernel");
    return launch_moves(p, p, (const Move*)workspace, (hipStream_t)stream);
}

extern "C" int odmkv_pages_select(const odmkv_pages_t* p, const odmkv_pages_t* to, const int64_t* parents, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    if (int rc = check_pages("pages_select", p)) return rc;
    if (int rc = check_pages("pages_select", to)) return rc;
    ODMKV_CHECK_ARG(parents != nullptr, "pages_select: null pointer");
    ODMKV_CHECK_ARG(p->layers == to->layers && p->Hkv == to->Hkv && p->pages == to->pages && p->blocks == to->blocks && p->dtype == to->dtype &&
                    p->kind == to->kind && p->kcodes == to->kcodes && p->refs == to->refs && p->status == to->status,
                    "pages_select: the two batches must share their pages");
    ODMKV_CHECK_ARG(p->table != to->table && p->length != to->length && p->slot != to->slot && p->ktail != to->ktail && p->vtail != to->vtail,
                    "pages_select: the two batches must have rows of their own");
    ODMKV_CHECK_ARG((long long)p->layers * p->Hkv < 65535, "pages_select: more than 65534 layers and heads");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < odmkv_pages_reorder_workspace_bytes(to->rows)) {
        odmkv_set_error("pages_select: workspace too small");
        return ODMKV_ENOSPACE;
    }
    hipLaunchKernelGGL(pages_plan_select_kernel, dim3(1), dim3(BOOK_THREADS), 0, (hipStream_t)stream, *p, *to, parents, (Move*)workspace);
    ODMKV_CHECK_LAUNCH("pages_plan_select_kernel");
    return launch_moves(p, to, (const Move*)workspace, (hipStream_t)stream);
}

// ---- rewinds --------------------------------------------------------------------------------------
struct TruncateArgs {
    odmkv_pages_t p;
    RowInts lengths;
    uint32_t rows[MAX_ROWS / 32];
};
__device__ static inline int cut_length(const TruncateArgs& a, int row, int len) {
    if (!(a.rows[row >> 5] >> (row & 31) & 1u)) return len;
    return min(len, max(row_int(a.lengths, row), 0));
}

// blockIdx.y == 0: the pages given up; from 1 on: a layer and head of the block that becomes the tail
template <int DT, int KIND>
__global__ __launch_bounds__(256) void pages_truncate_kernel(TruncateArgs a) {
    const odmkv_pages_t& p = a.p;
    const int row = blockIdx.x, tid = threadIdx.x, len = p.length[row], cut = cut_length(a, row, len);
    const int keep = cut / BLOCK_TOKENS, full = len / BLOCK_TOKENS, slot = p.slot[row];
    if (gridDim.y == 1) {                                      // (the row is this workgroup's alone: no tail is made of any)
        __syncthreads();
        if (tid == 0) p.length[row] = p.start[row] = cut;
    }
    if (keep >= full) return;
    if (blockIdx.y == 0) {
        Freed freed = {0, 0x7fffffff};
        for (int j = keep + tid; j < full; j += 256) drop_page(p, p.table[(size_t)slot * p.blocks + j], freed);
        give_back(p, freed);
        return;
    }
    if (cut == keep * BLOCK_TOKENS) return;
    const int lh = blockIdx.y - 1, layer = lh / p.Hkv, h = lh % p.Hkv, page = p.table[(size_t)slot * p.blocks + keep];
    const size_t at = page_at(p, layer, page, h), to = tail_at(p, layer, slot, h);
    for (int i = tid; i < 2 * PAGE_BYTES / 16; i += 256) {
        const bool value = i >= PAGE_BYTES / 16;
        const size_t o = (size_t)(value ? i - PAGE_BYTES / 16 : i) * 16;
        const uint4 c = *reinterpret_cast<const uint4*>((value ? p.vcodes : p.kcodes) + at + o);
        const float s = (value ? p.vscale : p.kscale)[scale_at(p, layer, page, h)];
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        uint32_t out[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float x[4];
            values4<KIND>(w[q], x);
            out[2 * q] = (uint32_t)to_16<DT>(x[0] * s) | (uint32_t)to_16<DT>(x[1] * s) << 16;
            out[2 * q + 1] = (uint32_t)to_16<DT>(x[2] * s) | (uint32_t)to_16<DT>(x[3] * s) << 16;
        }
        uint4* dst = reinterpret_cast<uint4*>((value ? p.vtail : p.ktail) + to + o);
        dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
        dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
}

__global__ __launch_bounds__(BOOK_THREADS) void pages_cut_kernel(TruncateArgs a) {
    const int row = threadIdx.x;
    if (row >= a.p.rows) return;
    a.p.length[row] = a.p.start[row] = cut_length(a, row, a.p.length[row]);
}

extern "C" int odmkv_pages_truncate(const odmkv_pages_t* p, const int32_t* lengths, const int32_t* lengths_host, int length, const uint32_t* row_mask,
                                    void* stream) {
    if (int rc = check_pages("pages_truncate", p)) return rc;
    ODMKV_CHECK_ARG(lengths || lengths_host || length >= 0, "pages_truncate: bad length");
    ODMKV_CHECK_ARG((long long)p->layers * p->Hkv < 65535, "pages_truncate: more than 65534 layers and heads");
    TruncateArgs a;
    a.p = *p;
    if (int rc = make_row_ints("pages_truncate", a.lengths, p->rows, lengths, lengths_host, length)) return rc;
    for (int i = 0; i < MAX_ROWS / 32; ++i) a.rows[i] = row_mask ? row_mask[i] : 0xffffffffu;
    const int tails = lengths || lengths_host || length % BLOCK_TOKENS ? p->layers * p->Hkv : 0;
    PAGES_DISPATCH(pages_truncate_kernel, p, dim3(p->rows, 1 + tails), dim3(256), 0, (hipStream_t)stream, a);
    ODMKV_CHECK_LAUNCH("pages_truncate_kernel");
    if (tails == 0) return 0;
    hipLaunchKernelGGL(pages_cut_kernel, dim3(1), dim3(BOOK_THREADS), 0, (hipStream_t)stream, a);
    ODMKV_CHECK_LAUNCH("pages_cut_kernel");
    return 0;
}

// ---- what rows have in common ---------------------------------------------------------------------
// Rows whose first page is the same are a group; two rows have blocks in common up to the first whose pages differ (a page that two rows hold at the same block came there by
// a copy of everything before it), a group what each of its rows has in common with its first one.  One workgroup, a thread a row; the first different block is looked for
// in eight places at a time.  Bound by round trips to the tables, of which there are four: 8 rows in 4.9 us, 64 of 128 common blocks in 6.5; once a move of rows, not once a layer.
__global__ __launch_bounds__(BOOK_THREADS) void pages_plan_common_kernel(odmkv_pages_t p, int32_t* plan) {
    __shared__ int part[BOOK_THREADS / 64], page0[MAX_ROWS], full[MAX_ROWS], slots[MAX_ROWS], leaders[MAX_ROWS], least[MAX_ROWS], count[MAX_ROWS], begin[MAX_ROWS], number[MAX_ROWS];
    const int tid = threadIdx.x, rows = p.rows;
    const bool mine = tid < rows;
    if (mine) {
        slots[tid] = p.slot[tid];
        full[tid] = p.length[tid] / BLOCK_TOKENS;
        page0[tid] = full[tid] > 0 ? p.table[(size_t)slots[tid] * p.blocks] : -1 - tid;
        least[tid] = full[tid];
        count[tid] = 0;
    }
    __syncthreads();
    int leader = tid, rank = 0;
    if (mine) {
        for (int j = tid - 1; j >= 0; --j) {
            if (page0[j] != page0[tid]) continue;
            leader = j;
            rank += 1;
        }
        leaders[tid] = leader;
        int same = min(full[tid], full[leader]);
        if (leader != tid) {
            const int32_t* a = p.table + (size_t)slots[tid] * p.blocks;
            const int32_t* b = p.table + (size_t)slots[leader] * p.blocks;
            int lo = 1, hi = same;                             // as many blocks are the same, and no more than that
            while (lo < hi) {
                const int step = (hi - lo + 7) / 8;
                int equal = 0;
#pragma unroll
                for (int k = 1; k <= 8; ++k) {
                    const int at = min(lo + k * step, hi) - 1;
                    equal += a[at] == b[at] ? 1 : 0;
                }
                if (equal < 8) hi = min(lo + (equal + 1) * step, hi + 1) - 1;
                lo = min(lo + equal * step, hi);
            }
            same = lo;
        }
        atomicMin(&least[leader], same);
        atomicAdd(&count[leader], 1);
    }
    __syncthreads();
    const bool is_group = mine && leader == tid && count[tid] > 1;
    int n, total;
    const int g = book_scan(is_group ? 1 : 0, part, n) - 1, end = book_scan(is_group ? count[tid] : 0, part, total);
    if (is_group) {
        number[tid] = g;
        begin[tid] = end - count[tid];
        int32_t* const to = plan + 1 + 4 * rows + 4 * g;
        to[0] = begin[tid];
        to[1] = count[tid];
        to[2] = least[tid];
        to[3] = slots[tid];
    }
    if (tid == 0) plan[0] = n;
    __syncthreads();
    if (!mine) return;
    const bool grouped = count[leader] > 1;
    plan[1 + tid] = grouped ? least[leader] : 0;
    plan[1 + rows + tid] = grouped ? number[leader] : -1;
    plan[1 + 2 * rows + tid] = rank;
    if (grouped) plan[1 + 3 * rows + begin[leader] + rank] = tid;
}

extern "C" size_t odmkv_pages_plan_bytes(int rows) { return rows > 0 ? align_up(plan_words(rows) * sizeof(int32_t), 256) : 0; }

extern "C" int odmkv_pages_plan(const odmkv_pages_t* p, int32_t* plan, size_t plan_bytes, void* stream) {
    if (int rc = check_pages("pages_plan", p)) return rc;
    ODMKV_CHECK_ARG(plan != nullptr && ((uintptr_t)plan & 15) == 0, "pages_plan: null or unaligned pointer");
    if (plan_bytes < odmkv_pages_plan_bytes(p->rows)) {
        odmkv_set_error("pages_plan: plan too small");
        return ODMKV_ENOSPACE;
    }
    hipLaunchKernelGGL(pages_plan_common_kernel, dim3(1), dim3(BOOK_THREADS), 0, (hipStream_t)stream, *p, plan);
    ODMKV_CHECK_LAUNCH("pages_plan_common_kernel");
    return 0;
}

// ---- compaction -----------------------------------------------------------------------------------
// One workgroup: where every page goes (its rank among those in use, -1: free), and the new pool's counts.
__global__ __launch_bounds__(BOOK_THREADS) void pages_rank_kernel(odmkv_pages_t p, odmkv_pages_t to, int32_t* where) {
    __shared__ int part[BOOK_THREADS / 64];
    const int tid = threadIdx.x;
    int live = 0;
    for (int base = 0; base < p.pages; base += 4 * BOOK_THREADS) {
        int r[4], n = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int page = base + 4 * tid + i;
            r[i] = page < p.pages ? p.refs[page] : 0;
            n += r[i] > 0;
        }
        int at = live + book_scan(n, part, total) - n;
        live += total;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int page = base + 4 * tid + i;
            if (page >= p.pages) break;
            const bool kept = r[i] > 0 && at < to.pages;
            where[page] = kept ? at : -1;
            if (kept) to.refs[at] = r[i];
            at += r[i] > 0;
        }
    }
    for (int page = live + tid; page < to.pages; page += BOOK_THREADS) to.refs[page] = 0;
    if (tid < p.rows) {
        to.length[tid] = p.length[tid];
        to.start[tid] = p.start[tid];
        to.slot[tid] = p.slot[tid];
    }
    if (tid == 0) {
        p.status[ST_LIVE] = live;
        to.status[ST_FREE] = max(to.pages - live, 0);
        to.status[ST_HINT] = min(live, to.pages);
        to.status[ST_REFUSED] = live > to.pages;
        to.status[ST_LIVE] = live;
    }
}

// A workgroup a page and layer: all heads' codes and scales.  Bound by memory: 1.07 GB in 202 us (5.3 TB/s), past the caches, which would keep neither side.
__global__ __launch_bounds__(256) void pages_copy_kernel(odmkv_pages_t p, odmkv_pages_t to, const int32_t* where) {
    const int page = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x, dst = where[page];
    if (dst < 0) return;
    const size_t from = page_at(p, layer, page, 0), at = page_at(to, layer, dst, 0);
    const int pieces = p.Hkv * (PAGE_BYTES / 16);
#pragma unroll 4
    for (int i = tid; i < pieces; i += 256) {
        store_once(to.kcodes + at + (size_t)i * 16, load_once(p.kcodes + from + (size_t)i * 16));
        store_once(to.vcodes + at + (size_t)i * 16, load_once(p.vcodes + from + (size_t)i * 16));
    }
    for (int h = tid; h < p.Hkv; h += 256) {
        to.kscale[scale_at(to, layer, dst, h)] = p.kscale[scale_at(p, layer, page, h)];
        to.vscale[scale_at(to, layer, dst, h)] = p.vscale[scale_at(p, layer, page, h)];
    }
}

// blockIdx.y == 0: a row's table; from 1 on: a layer and head's tail
__global__ __launch_bounds__(256) void pages_rows_kernel(odmkv_pages_t p, odmkv_pages_t to, const int32_t* where) {
    const int row = blockIdx.x, tid = threadIdx.x, slot = p.slot[row];
    if (blockIdx.y == 0) {
        const int full = p.length[row] / BLOCK_TOKENS;
        for (int j = tid; j < to.blocks; j += 256) {
            const int is = j < full && j < p.blocks ? where[p.table[(size_t)slot * p.blocks + j]] : 0;
            to.table[(size_t)slot * to.blocks + j] = max(is, 0);
        }
        return;
    }
    const int lh = blockIdx.y - 1, layer = lh / p.Hkv, h = lh % p.Hkv;
    const size_t at = tail_at(p, layer, slot, h);
    for (int i = tid; i < TAIL_ELEMS / 8; i += 256) {
        reinterpret_cast<uint4*>(to.ktail + at)[i] = reinterpret_cast<const uint4*>(p.ktail + at)[i];
        reinterpret_cast<uint4*>(to.vtail + at)[i] = reinterpret_cast<const uint4*>(p.vtail + at)[i];
    }
}

extern "C" size_t odmkv_pages_compact_workspace_bytes(int pages) { return pages > 0 ? align_up((size_t)pages * sizeof(int32_t), 256) : 0; }

extern "C" int odmkv_pages_compact(const odmkv_pages_t* p, const odmkv_pages_t* to, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_pages("pages_compact", p)) return rc;
    if (int rc = check_pages("pages_compact", to)) return rc;
    ODMKV_CHECK_ARG(p->layers == to->layers && p->Hkv == to->Hkv && p->rows == to->rows && p->dtype == to->dtype && p->kind == to->kind,
                    "pages_compact: the two caches must have the same layers, heads, rows and types");
    ODMKV_CHECK_ARG(p->kcodes != to->kcodes && p->vcodes != to->vcodes && p->table != to->table && p->refs != to->refs && p->status != to->status &&
                    p->ktail != to->ktail && p->vtail != to->vtail, "pages_compact: the two caches must not share memory");
    ODMKV_CHECK_ARG((long long)p->layers * p->Hkv < 65535, "pages_compact: more than 65534 layers and heads");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < odmkv_pages_compact_workspace_bytes(p->pages)) {
        odmkv_set_error("pages_compact: workspace too small");
        return ODMKV_ENOSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    int32_t* where = (int32_t*)workspace;
    hipLaunchKernelGGL(pages_rank_kernel, dim3(1), dim3(BOOK_THREADS), 0, st, *p, *to, where);
    ODMKV_CHECK_LAUNCH("pages_rank_kernel");
    hipLaunchKernelGGL(pages_copy_kernel, dim3(p->pages, p->layers), dim3(256), 0, st, *p, *to, where);
    ODMKV_CHECK_LAUNCH("pages_copy_kernel");
    hipLaunchKernelGGL(pages_rows_kernel, dim3(p->rows, 1 + p->layers * p->Hkv), dim3(256), 0, st, *p, *to, where);
    ODMKV_CHECK_LAUNCH("pages_rows_kernel");
    return 0;
}
