// krk_cuda_verify_draft: drafted tokens against the target's probabilities, from given random numbers.
//
//   p = softmax(target row / T), q = softmax(drafter's row / T'):   token t of row r stays where  u_r q_r(t) < p_r(t)
//   the first row that refuses: the lowest i with  sum_{k <= i} w_k > u sum w,  w = max(p - q, 0);   all stayed: the same with w = p of the last row
// A drafter whose temperature is not above 0 took its greatest value: q is 1 there.
//
// Two kernels. The first reads every row once: maximum, where it is, and the sum of exponentials, by slices; bound by reading the rows. The second has a
// cluster of blocks for each sequence: all its blocks judge the drafted tokens from the slices' sums, then the row that stopped is gone through again for
// its weights' sums, and the one warp whose part the random number falls into finds the token.
//
// Where the number falls among a hundred thousand weights, most of them of 1e-6 and less, the sums' own rounding decides: with f32 exponentials (6e-8 each, a sum
// 2e-8 off) one draw in 250 came out as a neighbour. So the drawn row's weights, their sums and the sums before them have 64 bits (weights to 4e-14). The
// judgement compares two numbers once, for which sums of f32 exponentials do (their arguments' rounding: under 1e-6 of a sum), with the token's own in 64 bits.
//
// Measured, 128,256 tokens: one sequence of five rows 17.5 to 19 us (5 for the sums; the drawing waits for memory and for four meetings of its blocks), 64 sequences of up to
// eight rows with a drafter's 130 us: 58 for the sums (265 MB, 4.6 TB/s), 72 for the drawing, bound by arithmetic in 64 bits (each weight twice: sums, then weights;
// for p alone once). A block of 512 threads an SM, with exponentials of CUDA's own, took 182 there, and a scan of 32 weights after the other 51 for one sequence.
#include "krk_common.cuh"

#include <cooperative_groups.h>

namespace krk_cuda {

namespace {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kStatPer = 32, kSlice = kStatThreads * kStatPer;
constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kCluster = 8, kParts = kCluster * kDrawWarps;

struct Part {   // of a slice of a row
    float m;
    int32_t at;     // of the lowest of the greatest values, -1: none
    double sum;     // exp((x - m) / T)
};

struct VerifyParams {
    const float *p, *q;
    const int32_t *row_start, *draft;
    const float *accept_u, *sample_u, *temp, *draft_temp;
    int32_t *tokens, *n_accepted;
    float *logprob;
    Part *part;               // [1 or 2][n_rows][slices]
    int64_t p_stride, q_stride;
    int n_rows, n_vocab, n_seq, slices, vec;   // vec: rows begin on 16-byte boundaries
};

// The reciprocal of a temperature; greedy requests and drafters: 1.
__device__ __forceinline__ double per_temp(const float *t, int s) {
    const float v = t ? t[s] : 1.0f;
    return v > 0.0f ? 1.0 / (double)v : 1.0;
}

template <bool VEC>
__global__ void __launch_bounds__(kStatThreads)
verify_stats_kernel(const __grid_constant__ VerifyParams p) {
    __shared__ int s_seq;
    __shared__ float s_m[kStatThreads / 32];
    __shared__ int s_at[kStatThreads / 32];
    __shared__ double s_sum[kStatThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int item = blockIdx.x / p.slices, slice = blockIdx.x - item * p.slices, row = item % p.n_rows;
    const bool drafter = item >= p.n_rows;
    const int lo = slice * kSlice, n = min(kSlice, p.n_vocab - lo);
    const float *x = (drafter ? p.q + row * p.q_stride : p.p + row * p.p_stride) + lo;
    if (tid == 0) s_seq = -1;
    __syncthreads();
    auto find = [&] {
        for (int s = tid; s < p.n_seq; s += kStatThreads) {
            const int a = p.row_start[s], b = p.row_start[s + 1];
            if (row >= a && row < b && !(drafter && row == b - 1)) s_seq = s;   // (the drafter has nothing to say about a sequence's last row)
        }
        __syncthreads();
        return s_seq;
    };
    // (a drafter's row may be one of those; the target's are read while their sequence is looked for)
    int s = -1;
    if (drafter && (s = find()) < 0) return;
    float v[kStatPer];
    auto at = [&](int i) { return VEC ? (i >> 2) * 4 * kStatThreads + 4 * tid + (i & 3) : i * kStatThreads + tid; };
#pragma unroll
    for (int i = 0; i < kStatPer; i += 4) {
        if (VEC && at(i) + 3 < n) {
            *reinterpret_cast<float4 *>(v + i) = *reinterpret_cast<const float4 *>(x + at(i));
        } else {
#pragma unroll
            for (int c = i; c < i + 4; c++) v[c] = at(c) < n ? x[at(c)] : -INFINITY;
        }
    }
    if (!drafter && (s = find()) < 0) return;
    const float inv = (float)fmin(per_temp(drafter && p.draft_temp ? p.draft_temp : p.temp, s), 1e37) * 1.44269504f;
    float m = -INFINITY;
    int best = INT32_MAX;
#pragma unroll
    for (int i = 0; i < kStatPer; i++) {   // (a thread's places rise)
        if (v[i] > m) m = v[i], best = lo + at(i);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xFFFFFFFFu, m, o);
        const int ob = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        if (om > m || (om == m && ob < best)) m = om, best = ob;
    }
    if (lane == 0) s_m[warp] = m, s_at[warp] = best;
    __syncthreads();
    m = s_m[0], best = s_at[0];
#pragma unroll
    for (int w = 1; w < kStatThreads / 32; w++)
        if (s_m[w] > m || (s_m[w] == m && s_at[w] < best)) m = s_m[w], best = s_at[w];
    const float from = m == -INFINITY ? 0.0f : m;   // (nothing but -infinity: a sum of zeros; infinity: no number)
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kStatPer; i++) sum += exp2f((v[i] - from) * inv);
    double all = sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
    if (lane == 0) s_sum[warp] = all;
    __syncthreads();
    if (tid == 0) {
        all = 0.0;
        for (int w = 0; w < kStatThreads / 32; w++) all += s_sum[w];
        Part out;
        out.m = m;
        out.at = m == -INFINITY ? -1 : best;
        out.sum = all;
        p.part[(size_t)item * p.slices + slice] = out;
    }
}

// 2^(t / 64), t <= 0, to 4e-14 of itself: t's whole part by a table of 2^(j / 64) and the exponent, the rest, in +-1/2, by the series of e^(r ln 2 / 64) to the
// fourth power. Below 2^-1000: 0; a NaN stays one.
constexpr double kSteps = 92.332482616893657;   // 64 / ln 2
__device__ __forceinline__ double exp_step(double t, const double *table) {
    constexpr double c = 0.010830424696249145;   // ln 2 / 64
    const double whole = t + 6755399441055744.0;   // 1.5 * 2^52
    const double r = t - (whole - 6755399441055744.0);
    const int n = __double2loint(whole);
    const double e = fma(r, fma(r, fma(r, fma(r, c * c * c * c / 24.0, c * c * c / 6.0), c * c / 2.0), c), 1.0) * table[n & 63];
    const double y = __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
    return t >= -64000.0 ? y : t < -64000.0 ? 0.0 : t;
}
__device__ __forceinline__ double exp_of(double a, const double *table) { return exp_step(a * kSteps, table); }
// log z, z >= 1, from the f32 one by a step of Newton's.
__device__ __forceinline__ double log_of(double z, const double *table) {
    const double y = (double)logf((float)z);
    return y + (z * exp_of(-y, table) - 1.0);
}

// A row's slices together, by a warp: the maximum, its lowest place, the sum of exponentials.
struct Row {
    float m;
    int at;
    double sum;
};
__device__ __forceinline__ Row row_of(const VerifyParams &p, int item, double inv, const double *table) {
    const int lane = threadIdx.x & 31;
    const Part *part = p.part + (size_t)item * p.slices;
    Part first = {-INFINITY, -1, 0.0};
    if (lane < p.slices) first = part[lane];
    Row r = {first.m, first.at >= 0 ? first.at : INT32_MAX, 0.0};
    for (int i = lane + 32; i < p.slices; i += 32) {
        const Part o = part[i];
        if (o.at >= 0 && (o.m > r.m || r.at == INT32_MAX)) r.at = o.at;
        r.m = fmaxf(r.m, o.m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xFFFFFFFFu, r.m, o);
        const int oa = __shfl_xor_sync(0xFFFFFFFFu, r.at, o);
        if (om > r.m || (om == r.m && oa < r.at)) r.m = om, r.at = oa;
    }
    for (int i = lane; i < p.slices; i += 32) {
        const Part o = i == lane ? first : part[i];
        if (o.m != -INFINITY || o.sum != 0.0) r.sum += o.m == -INFINITY ? o.sum : o.sum * exp_of(((double)o.m - (double)r.m) * inv, table);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.sum += __shfl_xor_sync(0xFFFFFFFFu, r.sum, o);
    if (r.m == -INFINITY) r.at = -1;
    return r;
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kDrawThreads, 2)
verify_draw_kernel(const __grid_constant__ VerifyParams p) {
    __shared__ double table[64], sums[3][kParts];   // [sum of p's exponentials, of q's, of weights][warps of the cluster]: this block writes its own to all of them
    __shared__ int s_stop, s_token, s_certain;
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank(), s = blockIdx.x / kCluster;
    if (tid < 64) table[tid] = exp2((double)tid / 64.0);   // (published by the cluster's meeting)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int r0 = p.row_start[s], r1 = p.row_start[s + 1], rows = r0 >= 0 && r1 <= p.n_rows ? r1 - r0 : 0;
    if (rows <= 0) {
        if (rank == 0 && tid == 0) p.n_accepted[s] = 0;
        return;   // (all blocks of the cluster)
    }
    const float t = p.temp ? p.temp[s] : 1.0f;
    const bool greedy = !(t > 0.0f), sure = p.draft_temp && !(p.draft_temp[s] > 0.0f);   // sure: q is 1 at the lowest of the drafter's greatest values
    const double inv_p = fmin(per_temp(p.temp, s), 1e37), inv_q = fmin(per_temp(p.draft_temp ? p.draft_temp : p.temp, s), 1e37);
    if (tid == 0) s_stop = rows - 1, s_token = -1;
    cluster.sync();   // (all blocks are there to be written to)
    // ---- the drafted tokens, a row a warp.
    for (int j = warp; j < rows - 1; j += kDrawWarps) {
        if (j > __shfl_sync(0xFFFFFFFFu, *(volatile int *)&s_stop, 0)) break;   // (an earlier one has been refused)
        const int row = r0 + j, token = p.draft[row];
        const Row pr = row_of(p, row, inv_p, table);
        bool ok = token >= 0 && token < p.n_vocab;
        if (ok) {
            const double a = ((double)p.p[row * p.p_stride + token] - (double)pr.m) * inv_p;
            if (greedy) {
                ok = pr.at == token;
            } else {
                double qt = 1.0;
                if (p.q) {
                    const Row qr = row_of(p, p.n_rows + row, inv_q, table);
                    if (sure) qt = qr.at == token ? 1.0 : 0.0, ok = qr.at >= 0;
                    else qt = exp_of(((double)p.q[row * p.q_stride + token] - (double)qr.m) * inv_q, table) / qr.sum;
                }
                ok = ok && (double)p.accept_u[row] * qt < exp_of(a, table) / pr.sum;   // (no number: refused)
            }
            if (ok && rank == 0 && p.logprob && lane == 0) p.logprob[row] = (float)(a - log_of(pr.sum, table));
        }
        if (!ok && lane == 0) atomicMin(&s_stop, j);
    }
    __syncthreads();
    const int stop = s_stop, row = r0 + stop;
    const bool last = stop == rows - 1;
    // a token that has nothing left (by way of shared memory: beside the sums, in every warp's registers, it cost spills, 64 sequences 189 us for 184)
    if (warp == 0 && !last) {
        const int at = !p.q ? p.draft[row] : sure ? row_of(p, p.n_rows + row, inv_q, table).at : -1;
        if (lane == 0) s_certain = at;
    }
    if (tid == 0 && last) s_certain = -1;
    __syncthreads();
    const int certain = s_certain;
    const float *x = p.p + row * p.p_stride, *y = p.q + row * p.q_stride;
    const bool two = p.q && !last && !sure;
    int token = -1;
    // (every warp for itself: they all find the same)
    const Row pr = row_of(p, row, inv_p, table);
    if (greedy) {
        token = pr.at;
    } else {
        const Row qr = two ? row_of(p, p.n_rows + row, inv_q, table) : Row{0.0f, 0, 1.0};
        // ---- the sums of exponentials in 64 bits: each warp of the cluster has a part of the row, a lane eight values of 256 that follow each other
        const int per = ((p.n_vocab + kParts - 1) / kParts + 7) / 8 * 8, part = rank * kDrawWarps + warp;
        const int lo = min(p.n_vocab, part * per), hi = min(p.n_vocab, lo + per);
        const double m_p = pr.m, m_q = qr.m, k_p = inv_p * kSteps, k_q = inv_q * kSteps;
        auto e_p = [&](float v) { return exp_step(((double)v - m_p) * k_p, table); };   // (the difference first: by a small temperature a product would lose it)
        auto e_q = [&](float v) { return exp_step(((double)v - m_q) * k_q, table); };
        auto load = [&](const float *row, int i0, float (&v)[8]) {
            if (p.vec && i0 + 8 <= hi) {
                *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(row + i0);
                *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(row + i0 + 4);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = i0 + j < hi ? row[i0 + j] : -INFINITY;
            }
        };
        auto warp_sum = [&](double v) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
            return v;
        };
        auto tell = [&](int what, double v) {   // to every block of the cluster
            if (lane < kCluster) *cluster.map_shared_rank(&sums[what][part], lane) = v;
        };
        static_assert(kParts == 128, "four parts a lane");
        auto upto = [&](const double *v) {   // sums of the parts up to a lane's last one, in the same order everywhere
            double a = ((v[4 * lane] + v[4 * lane + 1]) + v[4 * lane + 2]) + v[4 * lane + 3];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double b = __shfl_up_sync(0xFFFFFFFFu, a, o);
                if (lane >= o) a += b;
            }
            return a;
        };
        auto total = [&](const double *v) { return __shfl_sync(0xFFFFFFFFu, upto(v), 31); };
        // (weights that are p need not be divided by its sum: it scales them all)
        double per_p = 1.0, per_q = 0.0;
        if (two) {
            double a = 0.0, b = 0.0;
            for (int i0 = lo + 8 * lane; i0 < hi; i0 += 256) {
                float xp[8], xq[8];
                load(x, i0, xp);
                load(y, i0, xq);
                double a2[2] = {0.0, 0.0}, b2[2] = {0.0, 0.0};
#pragma unroll
                for (int j = 0; j < 8; j++) a2[j & 1] += e_p(xp[j]), b2[j & 1] += e_q(xq[j]);
                a += a2[0] + a2[1], b += b2[0] + b2[1];
            }
            tell(0, warp_sum(a));
            tell(1, warp_sum(b));
            cluster.sync();
            per_p = 1.0 / total(sums[0]), per_q = 1.0 / total(sums[1]);
        }
        bool whole = !two && certain < 0;   // weights are p
        auto weights = [&](int i0, double (&w)[8]) {
            float xp[8], xq[8];
            load(x, i0, xp);
            if (two && !whole) load(y, i0, xq);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                w[j] = e_p(xp[j]) * per_p;
                if (two && !whole) w[j] = fmax(w[j] - e_q(xq[j]) * per_q, 0.0);
                if (i0 + j == certain && !whole) w[j] = 0.0;
            }
        };
        double all = 0.0;
        for (int round = 0; round < 2; round++) {
            double w = 0.0;
            for (int i0 = lo + 8 * lane; i0 < hi; i0 += 256) {
                double v[8];
                weights(i0, v);
                w += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            }
            tell(2, warp_sum(w));
            cluster.sync();
            all = total(sums[2]);
            if (all > 0.0 || whole) break;   // (the same answer in all blocks)
            whole = true;                    // nothing is left: p itself
            cluster.sync();                  // (the sums have been read)
        }
        // ---- the part that the number falls into, and in it the token
        const double goal = (double)p.sample_u[s] * all;
        int found = -1;
        double before = 0.0;
        if (all > 0.0) {   // (a number)
            const double mine = upto(sums[2]), ahead = __shfl_up_sync(0xFFFFFFFFu, mine, 1);
            const unsigned over = __ballot_sync(0xFFFFFFFFu, mine > goal), some = __ballot_sync(0xFFFFFFFFu, sums[2][4 * lane] + sums[2][4 * lane + 1] + sums[2][4 * lane + 2] + sums[2][4 * lane + 3] > 0.0);
            const int l = over ? __ffs(over) - 1 : 31 - __clz(some);   // (none over: a number of 1)
            before = l > 0 ? __shfl_sync(0xFFFFFFFFu, ahead, l) : 0.0;
            int kept = -1;
            double kept_before = 0.0;
            for (int i = 4 * l; i < 4 * l + 4 && found < 0; i++) {
                if (sums[2][i] > 0.0) kept = i, kept_before = before;
                if (before + sums[2][i] > goal) found = i;
                else before += sums[2][i];
            }
            if (found < 0) found = kept, before = kept_before;   // (the same sums in another order fell short by a rounding)
        }
        if (found == part) {
            int at = -1, last_at = -1;
            for (int i0 = lo; i0 < hi && at < 0; i0 += 256) {
                double v[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
                if (i0 + 8 * lane < hi) weights(i0 + 8 * lane, v);
                double upto = 0.0;
                int mine_last = -1;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    upto += v[j];
                    if (v[j] > 0.0) mine_last = i0 + 8 * lane + j;
                }
                const double own = upto;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                    if (lane >= o) upto += u;
                }
                // the first lane whose sums pass the number, and of its values the first one
                double here = before + (upto - own);
                int mine = -1;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    here += v[j];
                    if (mine < 0 && v[j] > 0.0 && here > goal) mine = i0 + 8 * lane + j;
                }
                const unsigned over = __ballot_sync(0xFFFFFFFFu, mine >= 0), some = __ballot_sync(0xFFFFFFFFu, mine_last >= 0);
                if (over) at = __shfl_sync(0xFFFFFFFFu, mine, __ffs(over) - 1);
                if (some) last_at = __shfl_sync(0xFFFFFFFFu, mine_last, 31 - __clz(some));
                before += __shfl_sync(0xFFFFFFFFu, upto, 31);
            }
            if (at < 0) at = last_at;   // (likewise)
            if (lane == 0) *cluster.map_shared_rank(&s_token, 0) = at;
        }
        cluster.sync();
        token = s_token;
    }
    if (rank != 0) return;
    for (int j = tid; j < rows; j += kDrawThreads) {
        p.tokens[r0 + j] = j < stop ? p.draft[r0 + j] : j == stop ? token : -1;
        if (p.logprob && j >= stop) p.logprob[r0 + j] = j == stop && token >= 0 ? (float)(((double)x[token] - (double)pr.m) * inv_p - log_of(pr.sum, table)) : 0.0f;
    }
    if (tid == 0) p.n_accepted[s] = stop;
}

// Sequences without a row, where there are none at all.
__global__ void no_rows_kernel(int32_t *n_accepted, int n_seq) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s < n_seq) n_accepted[s] = 0;
}

int slices_of(const krk_cuda_verify &v) { return (int)((v.n_vocab + kSlice - 1) / kSlice); }

} // namespace

size_t verify_draft_workspace_bytes(const krk_cuda_verify &v) { return (size_t)(v.draft_logits ? 2 : 1) * v.n_rows * slices_of(v) * sizeof(Part); }

int launch_verify_draft(int32_t *tokens, int32_t *n_accepted, float *logprob, const float *logits, const krk_cuda_verify &v, void *workspace, cudaStream_t st) {
    VerifyParams p;
    p.p = logits, p.q = static_cast<const float *>(v.draft_logits);
    p.row_start = static_cast<const int32_t *>(v.row_start), p.draft = static_cast<const int32_t *>(v.draft);
    p.accept_u = static_cast<const float *>(v.accept_u), p.sample_u = static_cast<const float *>(v.sample_u);
    p.temp = static_cast<const float *>(v.temp), p.draft_temp = static_cast<const float *>(v.draft_temp);
    p.tokens = tokens, p.n_accepted = n_accepted, p.logprob = logprob;
    p.part = static_cast<Part *>(workspace);
    p.p_stride = v.stride, p.q_stride = v.draft_stride;
    p.n_rows = (int)v.n_rows, p.n_vocab = (int)v.n_vocab, p.n_seq = v.n_seq, p.slices = slices_of(v);
    if (v.n_rows == 0)
        return launched(launch_overlapped(no_rows_kernel, dim3((unsigned)((v.n_seq + 255) / 256)), dim3(256), st, n_accepted, v.n_seq));
    const int64_t blocks = (int64_t)(p.q ? 2 : 1) * p.n_rows * p.slices;
    if (blocks > INT32_MAX || (int64_t)v.n_seq * kCluster > INT32_MAX) return KRK_CUDA_ESHAPE;
    const bool vec = ((reinterpret_cast<uintptr_t>(p.p) | reinterpret_cast<uintptr_t>(p.q)) & 15) == 0 && (v.n_rows == 1 || (v.stride % 4 == 0 && (!p.q || v.draft_stride % 4 == 0)));
    p.vec = vec;
    if (blocks > 0) {
        const int rc = launched(launch_overlapped(vec ? verify_stats_kernel<true> : verify_stats_kernel<false>, dim3((unsigned)blocks), dim3(kStatThreads), st, p));
        if (rc != KRK_CUDA_OK) return rc;
    }
    return launched(launch_overlapped(verify_draw_kernel, dim3((unsigned)(v.n_seq * kCluster)), dim3(kDrawThreads), st, p));
}

} // namespace krk_cuda
