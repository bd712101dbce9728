// The entry of the attention over the paged 8-bit cache: its checks, how a call is cut into workgroups, the merge of partial results.
#include <cfloat>
#include "attend.h"
#include "parts.h"

// The shares of a row and kv-head's blocks, put together: out = sum_s w_s out_s / sum_s w_s, w_s = exp(lse_s - largest).  A workgroup a query, its four wavefronts every
// fourth share, eight shares of a wavefront on their way at a time, a lane two dims.  Bound by the latency of two dependent reads: 4.0 us behind a step over 32768 tokens
// (32 queries, 64 shares each), 7.2 for 928 queries of 64 shares (31 MB).
//
// bf16: values may lie at the type's end, and a result that stands for codes a little past 32 bits' own.  The latter are stopped there, and the weights, of one at most each, meet the values smaller
// by a power of two that takes their sum to a half or below, so that nothing is infinite on its way to a mean that is not.  (A power of two: every other result keeps its bits.)
#define MERGE_AHEAD 8
#define MERGE_MANY 1024

// SHARED: those of what the row has in common with others come first, its own behind them.
// APART: a query's wavefronts, four of them, or one where there are many queries: finding out where a query's partial results lie is what takes the time then.
template <int DT, bool NARROW_PARTS, bool SHARED, int APART>
__global__ __launch_bounds__(256) void attend_merge_kernel(AttendArgs a) {
    const odmkv_pages_t& p = a.p;
    const int R = a.G * a.L, h = blockIdx.y, row = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int of_workgroup = APART == 4 ? tid >> 6 : __builtin_amdgcn_readfirstlane(tid >> 6), wave = APART == 4 ? of_workgroup : 0;
    const int r = APART == 4 ? blockIdx.x : 4 * blockIdx.x + of_workgroup;
    if (APART == 1 && r >= R) return;
    const int l = r / a.G, hq = h * a.G + r - l * a.G;
    if (l >= (a.counts ? min(max(a.counts[row], 0), a.L) : a.L)) return;
    __shared__ float part[4][HD], top_of[4], sum_of[4];
    int splits = a.splits;
    size_t at = ((size_t)row * p.Hkv + h) * a.splits * R + r;
    int in_common = 0, cols = 0;
    size_t common_at = 0;
    if (SHARED) {                                               // (nothing here waits for anything else here)
        const Plan plan(a);
        const int common = plan.common(row), g = max(plan.group(row), 0), member = plan.member(row);
        const CommonShare share = common_share_of<true>(a, g);
        in_common = common > 0 ? share.splits : 0;
        cols = share.cols;
        common_at = (size_t)h * a.common_parts + share.parts + (size_t)member * R + r;
    }
    if (NARROW_PARTS) {
        const Share own = share_of<true, SHARED>(a, row);
        if (own.count == 1 && in_common == 0) return;           // that workgroup has written the result
        splits = own.count + in_common;
        at = ((size_t)h * a.splits + own.first) * R + r;
    }
    const int less = DT == ODMKV_F16 ? 0 : 33 - __builtin_clz(splits);
    const float down = __builtin_amdgcn_ldexpf(1.0f, -less);
    const auto held = [](float x) { return DT == ODMKV_F16 ? x : __builtin_amdgcn_fmed3f(x, -FLT_MAX, FLT_MAX); };      // (of a query that is not a number the weights are not)
    // (each wavefront by its own largest: the partial results need not wait for the largest of all)
    float top = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int i0 = wave; i0 < splits; i0 += APART * MERGE_AHEAD) {
        float lse[MERGE_AHEAD];
        float2 v[MERGE_AHEAD];
#pragma unroll
        for (int k = 0; k < MERGE_AHEAD; ++k) {
            const int i = min(i0 + APART * k, splits - 1);
            const bool common = SHARED && i < in_common;
            const size_t from = common ? common_at + (size_t)i * cols : at + (size_t)(i - in_common) * R;
            lse[k] = (common ? a.common_lse : a.part_lse)[from];
            v[k] = *reinterpret_cast<const float2*>((common ? a.common_out : a.part_out) + from * HD + 2 * lane);
        }
        float to = top;
#pragma unroll
        for (int k = 0; k < MERGE_AHEAD; ++k) {
            if (i0 + APART * k >= splits) lse[k] = -INFINITY;
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
            o0 = __fmaf_rn(w * down, held(v[k].x), o0);
            o1 = __fmaf_rn(w * down, held(v[k].y), o1);
        }
    }
    if constexpr (APART == 4) {
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
    }
    const float inv = sum == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(1.0f / sum, less);
    o0 *= inv;
    o1 *= inv;
    *reinterpret_cast<uint32_t*>(a.out + (((size_t)row * a.L + l) * a.Hq + hq) * HD + 2 * lane) = (uint32_t)to_16<DT>(o0) | (uint32_t)to_16<DT>(o1) << 16;
    if (a.lse && lane == 0) a.lse[((size_t)row * a.Hq + hq) * a.L + l] = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

static int launch_attend_merge(const AttendArgs& a, const Cut& cut, hipStream_t st) {
    const int R = a.G * a.L;
    const dim3 grid(R, a.p.Hkv, a.p.rows);
    // (a wavefront a query: 2048 queries of 18 parts each 9.2 -> 7.7 us, 48 rows of 64 queries of 8 parts 13.6 -> 6.6, but 448 of 65 parts 8.4 -> 13.1)
    const bool many = (long long)R * a.p.Hkv * a.p.rows > MERGE_MANY;
    const auto of_type = [&](auto dt) {
        if (cut.shared && many) hipLaunchKernelGGL((attend_merge_kernel<dt.value, true, true, 1>), dim3((R + 3) / 4, a.p.Hkv, a.p.rows), dim3(256), 0, st, a);
        else if (cut.shared) hipLaunchKernelGGL((attend_merge_kernel<dt.value, true, true, 4>), grid, dim3(256), 0, st, a);
        else if (cut.wide) hipLaunchKernelGGL((attend_merge_kernel<dt.value, false, false, 4>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((attend_merge_kernel<dt.value, true, false, 4>), grid, dim3(256), 0, st, a);
    };
    if (a.p.dtype == ODMKV_F16) of_type(Int<ODMKV_F16>());
    else of_type(Int<ODMKV_BF16>());
    ODMKV_CHECK_LAUNCH("attend_merge_kernel");
    return 0;
}

// Rows that leave compute units without work have their blocks shared out, a few at least to a workgroup: two workgroups of four wavefronts a compute unit, or
// one of eight.  (A share more than that costs its partial results: with two of eight, 2048 queries over 4096 tokens took 330 us for 273, four of 777 145 for 51.)
static Cut cut_of(const odmkv_pages_t& p, int R, int max_length) {
    const int blocks = max_length / BLOCK_TOKENS + 1, units = compute_units();
    Cut c = {4, 1, 4, R > NARROW, false, 0, false, 0, 0, 0};
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

// Rows with blocks in common: how many workgroups what is in common gets is known on the device alone, which has one for each of a group's tiles and shares out the others: as many as there are
// compute units (twice as many: 6 x 8 samples of 3001 tokens 31 -> 35.5 us, 64 of 8192 33.1 -> 34.5; half: 37 and 38), beside the rows' own.
static Cut cut_shared(const odmkv_pages_t& p, int R, int max_length) {
    Cut c = cut_of(p, R, max_length);
    if (R > NARROW || p.rows < 2) return c;
    const int blocks = max_length / BLOCK_TOKENS + 1, units = compute_units();
    c.shared = true;
    c.waves = 4;
    c.stream = false;
    c.splits = (int)std::max((long long)p.rows, std::min(2LL * units / p.Hkv, (long long)p.rows * std::max(1, blocks / 4)));
    c.parts = (size_t)p.Hkv * c.splits * R;
    c.spare = std::max(1, units / p.Hkv);
    c.workgroups = (int)(((long long)p.rows * R + SHARED_COLS - 1) / SHARED_COLS) + p.rows / 2 + c.spare;
    c.common_parts = (long long)p.rows * R + (long long)SHARED_COLS * c.spare;
    return c;
}

extern "C" size_t odmkv_pages_attend_shared_workspace_bytes(const odmkv_pages_t* p, int Hq, int L, int max_length) {
    if (!p || p->Hkv <= 0 || p->rows <= 0 || Hq <= 0 || L <= 0 || max_length < 0) return 0;
    const Cut c = cut_shared(*p, Hq / p->Hkv * L, max_length);
    return align_up(part_places(c.parts, (size_t)p->Hkv * c.common_parts).floats * sizeof(float), 256);
}

extern "C" size_t odmkv_pages_attend_workspace_bytes(const odmkv_pages_t* p, int Hq, int L, int max_length) {
    if (!p || p->Hkv <= 0 || p->rows <= 0 || Hq <= 0 || L <= 0 || max_length < 0) return 0;
    return align_up(part_places(cut_of(*p, Hq / p->Hkv * L, max_length).parts, 0).floats * sizeof(float), 256);
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
                    d->prefix, d->starts, d->start_stride_b, d->start_stride_l, d->layer, d->L, d->Hq, d->Hq / p.Hkv, d->window, d->scaling, std::min(d->cap, LARGEST_CAP),
                    1, nullptr, nullptr, d->plan, 0, nullptr, nullptr, 0};
    const size_t need = (d->plan ? odmkv_pages_attend_shared_workspace_bytes : odmkv_pages_attend_workspace_bytes)(&p, d->Hq, d->L, d->max_length);
    if (need > 0 && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < need)) {
        odmkv_set_error("pages_attend: workspace too small");
        return ODMKV_ENOSPACE;
    }
    const Cut cut = (d->plan ? cut_shared : cut_of)(p, a.G * a.L, d->max_length);
    a.splits = cut.splits;
    a.part_out = (float*)d->workspace;
    const PartPlaces at = part_places(cut.parts, (size_t)p.Hkv * cut.common_parts);
    a.part_lse = a.part_out + at.lse;
    hipStream_t st = (hipStream_t)stream;
    const bool f16 = p.dtype == ODMKV_F16;
    a.spare = cut.spare;
    a.common_out = a.part_out + at.common_out;
    a.common_parts = cut.common_parts;
    a.common_lse = a.part_out + at.common_lse;
    const int rc = cut.shared ? (f16 ? launch_attend_shared_f16(a, cut.workgroups, st) : launch_attend_shared_bf16(a, cut.workgroups, st))
                 : cut.wide ? (f16 ? launch_attend_wide_f16(a, cut, st) : launch_attend_wide_bf16(a, cut, st))
                            : (f16 ? launch_attend_narrow_f16(a, cut, st) : launch_attend_narrow_bf16(a, cut, st));
    if (rc) return rc;
    return cut.parts ? launch_attend_merge(a, cut, st) : 0;
}
