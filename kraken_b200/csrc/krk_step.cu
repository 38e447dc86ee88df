// krk_cuda_step_plan: pages, slots and positions of a step's new tokens from the requests' lengths.
//
// Tokens and new pages are prefix sums over the sequences. Sequence s, with b positions before and c new ones, takes the pages
// ceil(b / page) .. ceil((b + c) / page); its i-th one is the stack's (pages taken before + i)-th from the top. Every block of threads adds up all
// sequences for itself (two numbers each, out of level 2: no block waits for another one) and keeps those that reach into its 1024 tokens:
// each leaves a mark at its first token there, a maximum over the marks tells every token its sequence. A new page's number is written by
// the token of its first position; pages of old positions are read from the table, which nobody writes there.
//
// Bound: a launch's latency and two trips to memory (the sums, then the pages); 12 bytes a token. Measured: 8 requests 10 us a call, 512 requests and 131,072 places 9.8
// (6.2 on the device).
#include "krk_common.cuh"

namespace krk_cuda {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

struct StepParams {
    const int32_t *before, *fresh, *free_pages, *n_free;
    int32_t *table, *q_start, *kv_len, *last, *positions, *counts;
    int64_t *slots;
    int64_t max_tok;
    int free_cap, n_seq, width, page;
};

// Sums of a and b over the threads up to each one; both totals.
__device__ __forceinline__ void block_scan(int64_t &a, int64_t &total_a, int64_t (*warp_sum)) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, a, o);
        if (lane >= o) a += v;
    }
    if (lane == 31) warp_sum[warp] = a;
    __syncthreads();
    if (warp == 0) {
        int64_t w = warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xFFFFFFFFu, w, o);
            if (lane >= o) w += v;
        }
        warp_sum[lane] = w;
    }
    __syncthreads();
    if (warp > 0) a += warp_sum[warp - 1];
    total_a = warp_sum[kWarps - 1];
    __syncthreads();
}

struct Mark {
    int32_t seq, before, have;
    int64_t start, rank;   // its first token; pages taken before it
};

__global__ void __launch_bounds__(kThreads)
step_plan_kernel(const __grid_constant__ StepParams p) {
    __shared__ Mark marks[kThreads];
    __shared__ int mark_at[kThreads];
    __shared__ int64_t warp_sum[kWarps];
    __shared__ int warp_max[kWarps];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t first = (int64_t)blockIdx.x * kThreads, behind = first + kThreads;
    const bool writes = blockIdx.x == 0;
    mark_at[tid] = -1;
    int64_t tokens = 0, pages = 0, beyond = 0;   // of the sequences before this round's; pages wanted, and those outside the table
    __syncthreads();
    for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) {
        const int s = s0 + tid;
        const int before = s < p.n_seq ? max(p.before[s], 0) : 0, want = s < p.n_seq ? min(max(p.fresh[s], 0), INT32_MAX - before) : 0;
        int64_t upto = want, all;
        block_scan(upto, all, warp_sum);
        const int64_t start = min(tokens + upto - want, p.max_tok), end = min(tokens + upto, p.max_tok);
        const int64_t length = before + (end - start);
        const int64_t have = ((int64_t)before + p.page - 1) / p.page, need = (length + p.page - 1) / p.page;
        const int64_t takes = min(need, (int64_t)p.width) - min(have, (int64_t)p.width);
        int64_t rank = takes, all_pages;
        block_scan(rank, all_pages, warp_sum);
        rank += pages - takes;
        if (s < p.n_seq && start < end && start < behind && end > first) {
            const int at = (int)max(start - first, (int64_t)0);
            marks[at] = {s, before, (int)min(have, (int64_t)INT32_MAX), start, rank};
            mark_at[at] = at;
        }
        if (writes && s < p.n_seq) {
            p.q_start[s] = (int32_t)start;
            if (s == p.n_seq - 1) p.q_start[p.n_seq] = (int32_t)end;
            p.kv_len[s] = (int32_t)length;
            p.last[s] = end > start ? (int32_t)(end - 1) : -1;
        }
        int64_t out = (need - have) - takes;
        if (writes) {
            int64_t all_out;
            block_scan(out, all_out, warp_sum);
            beyond += all_out;
        }
        tokens += all;
        pages += all_pages;
    }
    __syncthreads();
    const int n_free = min(max(p.n_free[0], 0), p.free_cap);
    if (writes && tid == 0) {
        if (p.n_seq == 0) p.q_start[0] = 0;
        const int64_t taken = min(pages, (int64_t)n_free), there = min(tokens, p.max_tok);
        p.counts[0] = n_free - (int32_t)taken;
        p.counts[1] = (int32_t)min(pages - taken + beyond, (int64_t)INT32_MAX);
        p.counts[2] = (int32_t)there;
        p.counts[3] = (int32_t)min(tokens - there, (int64_t)INT32_MAX);
    }
    // the nearest mark at or before each token
    int at = mark_at[tid];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, at, o);
        if (lane >= o) at = max(at, v);
    }
    if (lane == 31) warp_max[warp] = at;
    __syncthreads();
    for (int w = 0; w < warp; w++) at = max(at, warp_max[w]);
    const int64_t t = first + tid;
    if (t >= p.max_tok) return;
    int32_t position = 0;
    int64_t slot = -1;
    if (t < tokens) {   // (a mark there is: the sequence of a token before the end reaches into this block)
        const Mark m = marks[at];
        position = m.before + (int32_t)(t - m.start);
        const int i = position / p.page, place = position - i * p.page;
        if (i < p.width) {
            int32_t *entry = p.table + (int64_t)m.seq * p.width + i;
            int32_t page;
            if (i < m.have) {
                page = *entry;
            } else {
                const int64_t k = m.rank + i - m.have;
                page = k < n_free ? p.free_pages[n_free - 1 - k] : -1;
                if (place == 0) *entry = page;
            }
            if (page >= 0) slot = (int64_t)page * p.page + place;
        }
    }
    p.positions[t] = position;
    p.slots[t] = slot;
}

} // namespace

int launch_step_plan(const krk_cuda_step &s, cudaStream_t st) {
    StepParams p;
    p.before = static_cast<const int32_t *>(s.kv_before), p.fresh = static_cast<const int32_t *>(s.n_new);
    p.free_pages = static_cast<const int32_t *>(s.free_pages), p.n_free = static_cast<const int32_t *>(s.n_free);
    p.table = static_cast<int32_t *>(s.page_table), p.q_start = static_cast<int32_t *>(s.q_start), p.kv_len = static_cast<int32_t *>(s.kv_len);
    p.last = static_cast<int32_t *>(s.last), p.positions = static_cast<int32_t *>(s.positions), p.counts = static_cast<int32_t *>(s.counts);
    p.slots = static_cast<int64_t *>(s.slots);
    p.max_tok = s.max_tok;
    p.free_cap = (int)s.free_cap, p.n_seq = s.n_seq, p.width = s.table_width, p.page = s.page_size;
    const int64_t blocks = (s.max_tok + kThreads - 1) / kThreads;
    return launched(launch_overlapped(step_plan_kernel, dim3((unsigned)(blocks < 1 ? 1 : blocks)), dim3(kThreads), st, p));
}

} // namespace krk_cuda
