/*
 * plan.hip -- the pages, offsets, positions and slots of a step's requests
 * (nmoe_kv_plan).
 *
 * Everything follows from prefix sums over the requests: the pages that come
 * back, the pages and rows that are asked for (who is served), and those that
 * are given (who gets which).  It moves a few bytes a request and 12 a row, so
 * it is bound by its chain of dependent accesses.
 */
#include "nmoe_context.h"

#define NMOE_PLAN_THREADS 1024
#define NMOE_PLAN_SEQS 65536
#define NMOE_PLAN_ROWS 256 /* threads of a block of the rows' launch */
#define NMOE_PLAN_HERE 4096 /* rows up to which the first launch writes them too */

/* Sums stay at 2^30 once they are there, which is more than there can be of
 * anything: pages below 2^27, rows at most 2^22. */
__device__ __forceinline__ uint32_t nmoe_plan_add(uint32_t a, uint32_t b) { return min(a + b, 1u << 30); }

/* The sum of v over this thread and those before it; *total: over all. */
__device__ __forceinline__ uint32_t nmoe_plan_scan(uint32_t v, uint32_t *scratch, uint32_t *total) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t u = __shfl_up(v, d, 64);
        if (lane >= d) v = nmoe_plan_add(v, u);
    }
    __syncthreads(); /* scratch may still be read for the last sum */
    if (lane == 63) scratch[wave] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NMOE_PLAN_THREADS / 64; w++) {
        const uint32_t u = scratch[w];
        if (w < wave) before = nmoe_plan_add(before, u);
        all = nmoe_plan_add(all, u);
    }
    *total = all;
    return nmoe_plan_add(before, v);
}

/* The last of n places with first[place] <= i (first[0] <= i, ascending). */
__device__ __forceinline__ int nmoe_plan_find(const uint32_t *first, int n, uint32_t i) {
    int lo = 0;
    while (n > 1) {
        const int half = n / 2;
        if (first[lo + half] <= i) lo += half;
        n -= half;
    }
    return lo;
}

__device__ __forceinline__ void nmoe_plan_row(const nmoe_hip_kv_requests &r, int t, int b, int position) {
    if (r.positions != NULL) r.positions[t] = position;
    if (r.slots != NULL)
        r.slots[t] = b < 0 ? -1
                           : (int64_t)r.page_table[(int64_t)b * r.max_pages + (uint32_t)position / (uint32_t)r.page_size] *
                                     r.page_size + (uint32_t)position % (uint32_t)r.page_size;
}

/* One block: a request a thread, in rounds of 1024. */
__global__ void __launch_bounds__(NMOE_PLAN_THREADS) nmoe_kv_plan_kernel(nmoe_hip_kv_requests r, int nseq, int rows_here) {
    __shared__ uint32_t s_first[NMOE_PLAN_THREADS], s_scan[NMOE_PLAN_THREADS / 64];
    __shared__ int s_len[NMOE_PLAN_THREADS];
    const int tid = threadIdx.x;
    const int64_t cap = (int64_t)r.max_pages * r.page_size;
    auto pages_of = [&](int64_t tokens) { return (uint32_t)((tokens + r.page_size - 1) / r.page_size); };
    uint32_t total;

    /* pages that come back */
    uint32_t free = (uint32_t)min(max(*r.free_count, 0), r.num_pages);
    for (int b0 = 0; b0 < nseq; b0 += NMOE_PLAN_THREADS) {
        const int b = b0 + tid, len = b < nseq ? r.lens[b] : 0;
        const uint32_t back = b < nseq && r.new_tokens[b] < 0 && len >= 0 && len <= cap ? pages_of(len) : 0u;
        const uint32_t first = nmoe_plan_scan(back, s_scan, &total) - back;
        s_first[tid] = first;
        __syncthreads();
        for (uint32_t i = tid; i < total; i += NMOE_PLAN_THREADS) {
            const int x = nmoe_plan_find(s_first, NMOE_PLAN_THREADS, i);
            if (free + i < (uint32_t)r.num_pages) r.free_pages[free + i] = r.page_table[(int64_t)(b0 + x) * r.max_pages + (i - s_first[x])];
        }
        free = min(free + total, (uint32_t)r.num_pages);
    }
    __syncthreads();

    /* who is served, and with what */
    uint32_t asked_pages = 0, asked_rows = 0, pages = 0, rows = 0;
    if (tid == 0) r.cu[0] = 0;
    for (int b0 = 0; b0 < nseq; b0 += NMOE_PLAN_THREADS) {
        const int b = b0 + tid, len = b < nseq ? r.lens[b] : 0, want = b < nseq ? r.new_tokens[b] : 0;
        const bool bad = len < 0 || len > cap, fits = !bad && want >= 0 && len + (int64_t)want <= cap;
        uint32_t need = fits ? pages_of(len + (int64_t)want) - pages_of(len) : 0u, more = fits ? (uint32_t)want : 0u;
        const uint32_t p = nmoe_plan_add(asked_pages, nmoe_plan_scan(need, s_scan, &total));
        asked_pages = nmoe_plan_add(asked_pages, total);
        const uint32_t m = nmoe_plan_add(asked_rows, nmoe_plan_scan(min(more, 1u << 30), s_scan, &total));
        asked_rows = nmoe_plan_add(asked_rows, total);
        const bool ok = fits && (need == 0 || p <= free) && (more == 0 || m <= (uint32_t)r.max_rows);
        if (!ok) need = more = 0;
        uint32_t round_pages, round_rows;
        const uint32_t page = nmoe_plan_scan(need, s_scan, &round_pages) - need;
        const uint32_t row = nmoe_plan_scan(more, s_scan, &round_rows) - more;
        s_first[tid] = page;
        s_len[tid] = len;
        if (b < nseq) {
            r.cu[b + 1] = (int)(rows + row + more);
            r.lens_out[b] = bad ? len : want < 0 ? 0 : len + (int)more;
            r.status[b] = bad ? 2 : ok || want < 0 ? 0 : 1;
        }
        __syncthreads();
        for (uint32_t i = tid; i < round_pages; i += NMOE_PLAN_THREADS) {
            const int x = nmoe_plan_find(s_first, NMOE_PLAN_THREADS, i);
            r.page_table[(int64_t)(b0 + x) * r.max_pages + pages_of(s_len[x]) + (i - s_first[x])] =
                r.free_pages[free - 1 - (pages + i)];
        }
        if (rows_here) {
            __syncthreads();
            s_first[tid] = row;
            __syncthreads();
            for (uint32_t i = tid; i < round_rows; i += NMOE_PLAN_THREADS) {
                const int x = nmoe_plan_find(s_first, NMOE_PLAN_THREADS, i);
                nmoe_plan_row(r, (int)(rows + i), b0 + x, s_len[x] + (int)(i - s_first[x]));
            }
        }
        __syncthreads();
        pages += round_pages;
        rows += round_rows;
    }
    if (tid == 0) *r.free_count_out = (int)(free - pages);
    if (rows_here)
        for (int t = (int)rows + tid; t < r.max_rows; t += NMOE_PLAN_THREADS) nmoe_plan_row(r, t, -1, 0);
}

/* Many rows: a thread a row, behind the first launch. */
__global__ void __launch_bounds__(NMOE_PLAN_ROWS) nmoe_kv_plan_rows_kernel(nmoe_hip_kv_requests r, int nseq) {
    const int t = blockIdx.x * NMOE_PLAN_ROWS + threadIdx.x;
    if (t >= r.max_rows) return;
    if (t >= r.cu[nseq]) {
        nmoe_plan_row(r, t, -1, 0);
        return;
    }
    const int b = nmoe_plan_find((const uint32_t *)r.cu, nseq, (uint32_t)t);
    nmoe_plan_row(r, t, b, r.lens_out[b] - (r.cu[b + 1] - t));
}

extern "C" int nmoe_kv_plan(nmoe_hip_ctx *ctx, const nmoe_hip_kv_requests *req, int nseq, void *stream) {
    if (ctx == NULL) return NMOE_HIP_EINVAL;
    if (req == NULL) return nmoe_fail(ctx, NMOE_HIP_EINVAL, "plan: requests are required");
    const nmoe_hip_kv_requests r = *req;
    if (r.page_size < 16 || r.page_size % 16 != 0 || r.num_pages < 1 || (int64_t)r.page_size * r.num_pages > 0x7fffffff)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "plan: page_size %d (a multiple of 16) times num_pages %d outside 1..2^31-1",
                         r.page_size, r.num_pages);
    if (r.max_pages < 1 || r.max_pages > 1 << 27 || r.max_rows < 0 || r.max_rows > NMOE_MAX_ROWS || nseq < 0 ||
        nseq > NMOE_PLAN_SEQS)
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "plan: %d requests (0..65536) of %d pages (1..2^27), %d rows (0..2^22)", nseq,
                         r.max_pages, r.max_rows);
    const void *const need[] = {r.lens, r.new_tokens, r.free_count, r.free_pages, r.page_table, r.lens_out, r.free_count_out,
                                r.cu, r.status};
    for (const void *p : need)
        if (p == NULL || !nmoe_aligned(p, 4))
            return nmoe_fail(ctx, NMOE_HIP_EINVAL, "plan: every array but positions and slots is required, 4-byte aligned");
    if (!nmoe_aligned(r.positions, 4) || !nmoe_aligned(r.slots, 8))
        return nmoe_fail(ctx, NMOE_HIP_EINVAL, "plan: positions 4-byte and slots 8-byte aligned");
    nmoe_on_device here(ctx);
    hipStream_t s = nmoe_stream_of(ctx, stream);
    const bool rows = r.max_rows > 0 && (r.positions != NULL || r.slots != NULL);
    const bool rows_here = rows && r.max_rows <= NMOE_PLAN_HERE;
    hipLaunchKernelGGL(nmoe_kv_plan_kernel, dim3(1), dim3(NMOE_PLAN_THREADS), 0, s, r, nseq, rows_here);
    if (rows && !rows_here)
        hipLaunchKernelGGL(nmoe_kv_plan_rows_kernel, dim3((r.max_rows + NMOE_PLAN_ROWS - 1) / NMOE_PLAN_ROWS),
                           dim3(NMOE_PLAN_ROWS), 0, s, r, nseq);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
