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

#define NMOE_PLAN_THREADS 1024 /* most; 64, 256 and 512 for as many requests (8 requests: 4.3 us, by 1024 threads 7.0; 512: 5.9, 7.2) */
#define NMOE_PLAN_SEQS 65536
#define NMOE_PLAN_ROWS 256 /* threads of a block of the rows' launch */
#define NMOE_PLAN_OFFSETS 4096 /* offsets that it holds in LDS */
/* Rows up to which the first launch writes them too (200 requests and rows: 4.7 us, by two launches 7.1; 4000 rows of 512
 * requests: 8.8, 8.6; 6000: 9.4, 8.0). */
#define NMOE_PLAN_HERE 4096

/* Sums stay at 2^30 once they are there, which is more than there can be of
 * anything: pages below 2^27, rows at most 2^22. */
__device__ __forceinline__ uint32_t nmoe_plan_add(uint32_t a, uint32_t b) { return min(a + b, 1u << 30); }

/* N sums at once, of v[i] over this thread and those before it; total[i]: over all. */
template <int THREADS, int N>
__device__ __forceinline__ void nmoe_plan_scan(uint32_t (&v)[N], uint32_t (*scratch)[THREADS / 64], uint32_t (&total)[N]) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t u = __shfl_up(v[i], d, 64);
            if (lane >= d) v[i] = nmoe_plan_add(v[i], u);
        }
    __syncthreads(); /* scratch may still be read for the last sums */
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane == 63) scratch[i][wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) {
            const uint32_t u = scratch[i][w];
            if (w < wave) before = nmoe_plan_add(before, u);
            all = nmoe_plan_add(all, u);
        }
        total[i] = all;
        v[i] = nmoe_plan_add(before, v[i]);
    }
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

/* One block: a request a thread, in rounds where there are more.  Its time is
 * the chain of length, sums, stack and table: 4.0 us a call for one request, 5.9
 * for 512 of a token, of which a launch alone is about 3. */
template <int THREADS>
__global__ void __launch_bounds__(THREADS) nmoe_kv_plan_kernel(nmoe_hip_kv_requests r, int nseq, int rows_here) {
    __shared__ uint32_t s_first[THREADS], s_scan[3][THREADS / 64];
    __shared__ int s_len[THREADS];
    const int tid = threadIdx.x;
    const int64_t cap = min((int64_t)r.max_pages * r.page_size, (int64_t)0x7fffffff); /* lengths are 32 bits, whatever the row holds */
    auto pages_of = [&](int64_t tokens) { return (uint32_t)((tokens + r.page_size - 1) / r.page_size); };
    uint32_t free = (uint32_t)min(max(*r.free_count, 0), r.num_pages);
    /* pages that come back, `back` of a thread's request with `first` before them, go on the stack */
    auto push = [&](int b0, uint32_t first, uint32_t total) {
        if (total != 0) { /* of the whole block */
            s_first[tid] = first;
            __syncthreads();
            for (uint32_t i = tid; i < total; i += THREADS) {
                const int x = nmoe_plan_find(s_first, THREADS, i);
                if (free + i < (uint32_t)r.num_pages)
                    r.free_pages[free + i] = r.page_table[(int64_t)(b0 + x) * r.max_pages + (i - s_first[x])];
            }
            __syncthreads();
        }
        free = min(free + total, (uint32_t)r.num_pages);
    };
    struct request {
        int len;
        bool bad, ends, fits;
        uint32_t back, need, more;
    };
    auto request_of = [&](int b) {
        request q = {b < nseq ? r.lens[b] : 0, false, false, false, 0, 0, 0};
        const int want = b < nseq ? r.new_tokens[b] : 0;
        q.bad = q.len < 0 || q.len > cap;
        q.ends = !q.bad && want < 0;
        q.fits = !q.bad && want >= 0 && q.len + (int64_t)want <= cap;
        if (q.ends) q.back = pages_of(q.len);
        if (q.fits) {
            q.need = pages_of(q.len + (int64_t)want) - pages_of(q.len);
            q.more = min((uint32_t)want, 1u << 30);
        }
        return q;
    };
    if (nseq > THREADS) /* else together with what is asked for */
        for (int b0 = 0; b0 < nseq; b0 += THREADS) {
            const uint32_t back = request_of(b0 + tid).back;
            uint32_t v[1] = {back}, total[1];
            nmoe_plan_scan<THREADS, 1>(v, s_scan, total);
            push(b0, v[0] - back, total[0]);
        }

    /* who is served, and with what */
    uint32_t asked_pages = 0, asked_rows = 0, pages = 0, rows = 0;
    if (tid == 0) r.cu[0] = 0;
    for (int b0 = 0; b0 < nseq; b0 += THREADS) {
        const int b = b0 + tid;
        request q = request_of(b);
        uint32_t v[3] = {q.need, q.more, q.back}, total[3];
        nmoe_plan_scan<THREADS, 3>(v, s_scan, total);
        if (nseq <= THREADS) push(b0, v[2] - q.back, total[2]);
        const uint32_t p = nmoe_plan_add(asked_pages, v[0]), m = nmoe_plan_add(asked_rows, v[1]);
        asked_pages = nmoe_plan_add(asked_pages, total[0]);
        asked_rows = nmoe_plan_add(asked_rows, total[1]);
        const bool ok = q.fits && (q.need == 0 || p <= free) && (q.more == 0 || m <= (uint32_t)r.max_rows);
        /* all are served as a rule: then the sums of what they get are those of what they ask for */
        uint32_t page = v[0] - q.need, row = v[1] - q.more, round_pages = total[0], round_rows = total[1];
        if (asked_pages > free || asked_rows > (uint32_t)r.max_rows) {
            if (!ok) q.need = q.more = 0;
            uint32_t w[2] = {q.need, q.more}, got[2];
            nmoe_plan_scan<THREADS, 2>(w, s_scan, got);
            page = w[0] - q.need;
            row = w[1] - q.more;
            round_pages = got[0];
            round_rows = got[1];
        }
        if (b < nseq) {
            r.cu[b + 1] = (int)(rows + row + q.more);
            r.lens_out[b] = q.ends ? 0 : q.len + (int)q.more;
            r.status[b] = q.bad ? 2 : ok || q.ends ? 0 : 1;
        }
        s_first[tid] = page;
        s_len[tid] = q.len;
        __syncthreads();
        for (uint32_t i = tid; i < round_pages; i += THREADS) {
            const int x = nmoe_plan_find(s_first, THREADS, i);
            r.page_table[(int64_t)(b0 + x) * r.max_pages + pages_of(s_len[x]) + (i - s_first[x])] =
                r.free_pages[free - 1 - (pages + i)];
        }
        __syncthreads();
        if (rows_here) {
            s_first[tid] = row;
            __syncthreads();
            for (uint32_t i = tid; i < round_rows; i += THREADS) {
                const int x = nmoe_plan_find(s_first, THREADS, i);
                nmoe_plan_row(r, (int)(rows + i), b0 + x, s_len[x] + (int)(i - s_first[x]));
            }
            __syncthreads();
        }
        pages += round_pages;
        rows += round_rows;
    }
    if (tid == 0) *r.free_count_out = (int)(free - pages);
    if (rows_here)
        for (int t = (int)rows + tid; t < r.max_rows; t += THREADS) nmoe_plan_row(r, t, -1, 0);
}

/* Many rows: a thread a row, behind the first launch.  The offsets are looked
 * through in LDS, where they fit: each step of the search in memory took as
 * long as reading them all (512 requests: 4.5 us, now 3.5). */
__global__ void __launch_bounds__(NMOE_PLAN_ROWS) nmoe_kv_plan_rows_kernel(nmoe_hip_kv_requests r, int nseq) {
    __shared__ uint32_t s_first[NMOE_PLAN_OFFSETS];
    const int t = blockIdx.x * NMOE_PLAN_ROWS + threadIdx.x, rows = r.cu[nseq];
    const uint32_t *first = (const uint32_t *)r.cu;
    if (nseq <= NMOE_PLAN_OFFSETS) { /* the whole block */
        for (int b = threadIdx.x; b < nseq; b += NMOE_PLAN_ROWS) s_first[b] = first[b];
        __syncthreads();
    }
    if (t >= r.max_rows) return;
    if (t >= rows) {
        nmoe_plan_row(r, t, -1, 0);
        return;
    }
    const int b = nseq <= NMOE_PLAN_OFFSETS ? nmoe_plan_find(s_first, nseq, (uint32_t)t) : nmoe_plan_find(first, nseq, (uint32_t)t);
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
    /* as many threads as requests, or rows: fewer wavefronts wait for each other sooner */
    const int threads = nseq > (rows_here ? r.max_rows / 4 : 0) ? nseq : r.max_rows / 4;
    if (threads <= 64)
        hipLaunchKernelGGL((nmoe_kv_plan_kernel<64>), dim3(1), dim3(64), 0, s, r, nseq, rows_here);
    else if (threads <= 256)
        hipLaunchKernelGGL((nmoe_kv_plan_kernel<256>), dim3(1), dim3(256), 0, s, r, nseq, rows_here);
    else if (threads <= 512)
        hipLaunchKernelGGL((nmoe_kv_plan_kernel<512>), dim3(1), dim3(512), 0, s, r, nseq, rows_here);
    else
        hipLaunchKernelGGL((nmoe_kv_plan_kernel<NMOE_PLAN_THREADS>), dim3(1), dim3(NMOE_PLAN_THREADS), 0, s, r, nseq, rows_here);
    if (rows && !rows_here)
        hipLaunchKernelGGL(nmoe_kv_plan_rows_kernel, dim3((r.max_rows + NMOE_PLAN_ROWS - 1) / NMOE_PLAN_ROWS),
                           dim3(NMOE_PLAN_ROWS), 0, s, r, nseq);
    NMOE_HIP_TRY(ctx, hipGetLastError());
    return NMOE_HIP_OK;
}
