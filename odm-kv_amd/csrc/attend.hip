// Attention over the paged 8-bit cache: queries of the newest tokens, with any of a tanh cap, a bias by distance, a window, a prefix and
// document starts.
//
//   x_j = scaling * s_k (q . c_j), capped and biased;  out = sum_j softmax(x)_j s_v v_j over lo <= j < hi
#include <algorithm>
#include "pages.h"

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
};

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

// the simplest form: a workgroup a query, a thread a token and then a thread a dim
template <int DT, int KIND>
__global__ __launch_bounds__(128) void attend_simple_kernel(AttendArgs a) {
    const odmkv_pages_t& p = a.p;
    const int row = blockIdx.z, hq = blockIdx.y, l = blockIdx.x, tid = threadIdx.x, h = hq / a.G;
    const int len = p.length[row], n = a.counts ? min(max(a.counts[row], 0), a.L) : a.L, slot = p.slot[row];
    if (l >= n) return;
    const Sight s = sight_of(a, row, len, n, l);
    __shared__ float q[HD], w[128], red[4];
    q[tid] = Elem<DT>::to_f32(a.q[row * a.qb + hq * a.qh + l * a.ql + tid]);
    __syncthreads();
    const float slope = a.slopes ? a.slopes[hq] : 0.0f;
    float m = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (int base = s.lo / 64 * 64; base < s.hi; base += 64) {
        const bool full = base / 64 < len / 64;
        const int page = full ? p.table[(size_t)slot * p.blocks + base / 64] : 0;
        const size_t at = page_at(p, a.layer, page, h), tat = tail_at(p, a.layer, slot, h);
        const float sk = full ? p.kscale[scale_at(p, a.layer, page, h)] : 1.0f, sv = full ? p.vscale[scale_at(p, a.layer, page, h)] : 1.0f;
        float x = -INFINITY;
        if (tid < 64 && base + tid >= s.lo && base + tid < s.hi) {
            float dot = 0.0f;
            for (int d = 0; d < HD; d += 4) {
                float k[4];
                if (full) values4<KIND>(*reinterpret_cast<const uint32_t*>(p.kcodes + at + tid * HD + d), k);
                else for (int e = 0; e < 4; ++e) k[e] = Elem<DT>::to_f32(p.ktail[tat + tid * HD + d + e]);
                for (int e = 0; e < 4; ++e) dot = __fmaf_rn(q[d + e], k[e], dot);
            }
            x = dot * sk * a.scaling;
            if (a.cap > 0.0f) x = a.cap * tanhf(x / a.cap);
            x -= slope * fabsf((float)(s.pos - base - tid));
        }
        if (tid < 64) {
            const float top = wave_max(x);
            if (tid == 0) red[0] = top;
        }
        __syncthreads();
        const float mn = fmaxf(m, red[0]), by = mn > -INFINITY ? mn : 0.0f, old = expf(m - by);
        const float e = x > -INFINITY || x != x ? expf(x - by) : 0.0f;
        if (tid < 64) {
            w[tid] = e;
            const float z = wave_sum(e);
            if (tid == 0) red[1] = z;
        }
        __syncthreads();
        sum = sum * old + red[1];
        acc *= old;
        m = mn;
        for (int t = 0; t < 64; t += 4) {
            float v[4];
            if (full) values4<KIND>(*reinterpret_cast<const uint32_t*>(p.vcodes + at + tid * 64 + t), v);
            else for (int e2 = 0; e2 < 4; ++e2) v[e2] = Elem<DT>::to_f32(p.vtail[tat + tid * 64 + t + e2]);
            for (int e2 = 0; e2 < 4; ++e2) acc = __fmaf_rn(w[t + e2] * sv, v[e2], acc);
        }
        __syncthreads();
    }
    const bool none = s.hi <= s.lo;
    a.out[(((size_t)row * a.L + l) * a.Hq + hq) * HD + tid] = to_16<DT>(none ? 0.0f : acc / sum);
    if (a.lse && tid == 0) a.lse[((size_t)row * a.Hq + hq) * a.L + l] = none ? -INFINITY : m + logf(sum);
}

extern "C" size_t odmkv_pages_attend_workspace_bytes(const odmkv_pages_t* p, int Hq, int L, int max_length) {
    (void)p; (void)Hq; (void)L; (void)max_length;
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
    ODMKV_CHECK_ARG(d->L >= 0 && d->window >= 0 && d->max_length >= 0, "pages_attend: bad length");
    ODMKV_CHECK_ARG(d->cap >= 0.0f && d->cap < INFINITY, "pages_attend: bad cap");
    if (d->L == 0) return 0;
    ODMKV_CHECK_ARG(d->q && d->out, "pages_attend: null pointer");
    ODMKV_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->out) & 15) == 0 && ((d->q_stride_b | d->q_stride_h | d->q_stride_l) & 7) == 0,
                    "pages_attend: rows must be 16-byte aligned");
    const AttendArgs a = {p, (const uint16_t*)d->q, d->q_stride_b, d->q_stride_h, d->q_stride_l, (uint16_t*)d->out, d->lse, d->counts, d->slopes,
                          d->prefix, d->starts, d->start_stride_b, d->start_stride_l, d->layer, d->L, d->Hq, d->Hq / p.Hkv, d->window, d->scaling, d->cap};
    const dim3 grid(d->L, d->Hq, p.rows);
    hipStream_t st = (hipStream_t)stream;
    if (p.dtype == ODMKV_F16 && p.kind == ODMKV_INT8) hipLaunchKernelGGL((attend_simple_kernel<ODMKV_F16, ODMKV_INT8>), grid, dim3(128), 0, st, a);
    else if (p.dtype == ODMKV_F16) hipLaunchKernelGGL((attend_simple_kernel<ODMKV_F16, ODMKV_E4M3>), grid, dim3(128), 0, st, a);
    else if (p.kind == ODMKV_INT8) hipLaunchKernelGGL((attend_simple_kernel<ODMKV_BF16, ODMKV_INT8>), grid, dim3(128), 0, st, a);
    else hipLaunchKernelGGL((attend_simple_kernel<ODMKV_BF16, ODMKV_E4M3>), grid, dim3(128), 0, st, a);
    ODMKV_CHECK_LAUNCH("attend_simple_kernel");
    return 0;
}
