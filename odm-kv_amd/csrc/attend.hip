// The entry of the attention over the paged 8-bit cache: its checks, how a call is cut into workgroups, the merge of partial results.
#include "attend.h"

// The shares of a row and kv-head's blocks, put together: out = sum_s w_s out_s / sum_s w_s, w_s = exp(lse_s - largest).  A workgroup a query, its four wavefronts every
// fourth share, eight shares of a wavefront on their way at a time, a lane two dims.  Bound by the latency of two dependent reads: 4.0 us behind a step over 32768 tokens
// (32 queries, 64 shares each), 7.2 for 928 queries of 64 shares (31 MB).
#define MERGE_AHEAD 8

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
    // (each wavefront by its own largest: the partial results need not wait for the largest of all)
    float top = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int i0 = wave; i0 < splits; i0 += 4 * MERGE_AHEAD) {
        float lse[MERGE_AHEAD];
        float2 v[MERGE_AHEAD];
#pragma unroll
        for (int k = 0; k < MERGE_AHEAD; ++k) {
            const size_t from = at + (size_t)min(i0 + 4 * k, splits - 1) * R;
            lse[k] = a.part_lse[from];
            v[k] = *reinterpret_cast<const float2*>(a.part_out + from * HD + 2 * lane);
        }
        float to = top;
#pragma unroll
        for (int k = 0; k < MERGE_AHEAD; ++k) {
            if (i0 + 4 * k >= splits) lse[k] = -INFINITY;
            to = fmaxf(to, lse[k]);
        }
        const float by = to > -INFINITY ? to : 0.0f, old = __builtin_amdgcn_exp2f(top - by);
        top = to;
        sum *= old;
        o0 *= old;
        o1 *= old;
#pragma unroll
        for (int k = 0; k < MERGE_AHEAD; ++k) {
            const float w = __builtin_amdgcn_exp2f(lse[k] - by);
            sum += w;
            o0 = __fmaf_rn(w, v[k].x, o0);
            o1 = __fmaf_rn(w, v[k].y, o1);
        }
    }
    part[wave][2 * lane] = o0;
    part[wave][2 * lane + 1] = o1;
    if (lane == 0) {
        sum_of[wave] = sum;
        top_of[wave] = top;
    }
    __syncthreads();
    if (tid >= 64) return;
    top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
    const float by = top > -INFINITY ? top : 0.0f;
    sum = o0 = o1 = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(top_of[w] - by);
        sum = __fmaf_rn(f, sum_of[w], sum);
        o0 = __fmaf_rn(f, part[w][2 * lane], o0);
        o1 = __fmaf_rn(f, part[w][2 * lane + 1], o1);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    o0 *= inv;
    o1 *= inv;
    *reinterpret_cast<uint32_t*>(a.out + (((size_t)row * a.L + l) * a.Hq + hq) * HD + 2 * lane) = (uint32_t)to_16<DT>(o0) | (uint32_t)to_16<DT>(o1) << 16;
    if (a.lse && lane == 0) a.lse[((size_t)row * a.Hq + hq) * a.L + l] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

static int launch_attend_merge(const AttendArgs& a, const Cut& cut, hipStream_t st) {
    const dim3 grid(a.G * a.L, a.p.Hkv, a.p.rows);
    if (a.p.dtype == ODMKV_F16) {
        if (cut.wide) hipLaunchKernelGGL((attend_merge_kernel<ODMKV_F16, false>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((attend_merge_kernel<ODMKV_F16, true>), grid, dim3(256), 0, st, a);
    } else {
        if (cut.wide) hipLaunchKernelGGL((attend_merge_kernel<ODMKV_BF16, false>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((attend_merge_kernel<ODMKV_BF16, true>), grid, dim3(256), 0, st, a);
    }
    ODMKV_CHECK_LAUNCH("attend_merge_kernel");
    return 0;
}

// Rows that leave compute units without work have their blocks shared out, a few at least to a workgroup: two workgroups of four wavefronts a compute unit, or
// one of eight.  (A share more than that costs its partial results: with two of eight, 2048 queries over 4096 tokens took 330 us for 273, four of 777 145 for 51.)
static Cut cut_of(const odmkv_pages_t& p, int R, int max_length) {
    const int blocks = max_length / BLOCK_TOKENS + 1, units = compute_units();
    Cut c = {4, 1, 4, R > NARROW, false, 0};
    if (c.wide) {
        c.waves = R > 128 ? WIDE_WAVES : 4;
        c.groups = R <= 64 ? 2 : c.waves;
        const long long groups = (long long)p.rows * p.Hkv * ((R + 32 * c.groups - 1) / (32 * c.groups));
        c.splits = (int)std::max(1LL, std::min((c.waves == WIDE_WAVES ? 1 : 2) * units / groups, (long long)blocks / 4));
        c.parts = c.splits > 1 ? (size_t)p.rows * p.Hkv * c.splits * R : 0;
    } else {
        // Pages that the last-level cache (256 MB) would not keep from one call to the next, with what else passes between: nothing is gained by keeping any, and reads
        // that do not ask for it are faster (268 MB a call 59.7 -> 51.4 us; three caches of 134 MB in turn 33.3 -> 30.3).  Where they would be kept, it costs: 134 MB
        // and nothing else 28.2 -> 28.7 us, three caches of 67 MB in turn 18.7 -> 20.2.
        c.stream = (size_t)p.layers * p.pages * p.Hkv * 2 * PAGE_BYTES > ((size_t)96 << 20);
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
    ODMKV_CHECK_ARG(d->cap == 0.0f || (d->cap >= 0x1p-100f && d->cap < INFINITY), "pages_attend: bad cap");
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
    const bool f16 = p.dtype == ODMKV_F16;
    const int rc = cut.wide ? (f16 ? launch_attend_wide_f16(a, cut, st) : launch_attend_wide_bf16(a, cut, st))
                            : (f16 ? launch_attend_narrow_f16(a, cut, st) : launch_attend_narrow_bf16(a, cut, st));
    if (rc) return rc;
    return cut.parts ? launch_attend_merge(a, cut, st) : 0;
}
