// krk_cuda_logits_adjust: what a sampler does to the rows of logits before it ranks them, in one pass: sparse biases, penalties for
// tokens of the row's history, a grammar's mask.
//
//   v = x + bias[id];   c = times of id in the history;   c > 0:  v = v > 0 ? v / rep : v * rep,  v -= freq * c + pres;
//   the grammar does not allow id:  v = -inf
//
// Bound: reading and writing the rows once. The lists name few ids of a row, many of them more than once, so a block of threads counts those
// of its slice of the row in shared memory (whole numbers: the order of the atomics does not matter; of an id's biases the
// highest place in the list is kept, the same way) while its slice of the logits is on its way into registers.
#include "krk_common.cuh"

namespace krk_cuda {

namespace {

constexpr int kThreads = 256;

struct AdjustParams {
    const float *x;
    float *y;
    int64_t x_stride, y_stride, hist_stride, bias_stride, mask_stride, n;
    const int32_t *hist, *hist_len, *bias_ids, *bias_len, *mask_row;
    const float *bias, *rep, *freq, *pres;
    const uint32_t *mask;
    int hist_n, bias_n, n_masks, slice, slices;
};

// PER: values of a thread. VEC: rows begin on 16-byte boundaries, four values at a time.
template <int PER, bool VEC>
__global__ void __launch_bounds__(kThreads)
logits_adjust_kernel(const __grid_constant__ AdjustParams p) {
    constexpr int kSlice = PER * kThreads;
    __shared__ int count[kSlice];
    __shared__ int last[kSlice];   // place in the list of biases, plus one
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / p.slices;
    const int64_t lo = (int64_t)(blockIdx.x - row * p.slices) * kSlice;
    const int n = (int)min((int64_t)kSlice, p.n - lo);
    const float *x = p.x + row * p.x_stride + lo;
    float v[PER];
    auto at = [&](int i) { return VEC ? (i >> 2) * 4 * kThreads + 4 * tid + (i & 3) : i * kThreads + tid; };
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const int j = at(i);
            if (j + 3 < n) {
                const float4 f = *reinterpret_cast<const float4 *>(x + j);
                v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++) v[i + c] = j + c < n ? x[j + c] : 0.0f;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = at(i) < n ? x[at(i)] : 0.0f;
    }
    const int n_hist = !p.hist ? 0 : p.hist_len ? min(max(p.hist_len[row], 0), p.hist_n) : p.hist_n;
    const int n_bias = !p.bias ? 0 : p.bias_len ? min(max(p.bias_len[row], 0), p.bias_n) : p.bias_n;
    if (n_hist > 0) {
        for (int i = tid; i < kSlice; i += kThreads) count[i] = 0;
    }
    if (n_bias > 0) {
        for (int i = tid; i < kSlice; i += kThreads) last[i] = 0;
    }
    __syncthreads();
    // (an id outside the row is outside every slice)
    const int32_t *hist = p.hist + row * p.hist_stride;
    for (int i = tid; i < n_hist; i += kThreads) {
        const int64_t j = (int64_t)hist[i] - lo;
        if (j >= 0 && j < n) atomicAdd(&count[j], 1);
    }
    const int32_t *ids = p.bias_ids + row * p.bias_stride;
    for (int i = tid; i < n_bias; i += kThreads) {
        const int64_t j = (int64_t)ids[i] - lo;
        if (j >= 0 && j < n) atomicMax(&last[j], i + 1);
    }
    __syncthreads();
    const float rep = p.rep ? p.rep[row] : 1.0f, freq = p.freq ? p.freq[row] : 0.0f, pres = p.pres ? p.pres[row] : 0.0f;
    const bool repeats = rep > 0.0f && rep != 1.0f;
    const float *bias = p.bias + row * p.bias_stride;
    const int32_t m_row = !p.mask ? -1 : p.mask_row ? p.mask_row[row] : (int32_t)row;
    const uint32_t *mask = m_row >= 0 && m_row < p.n_masks ? p.mask + m_row * p.mask_stride : nullptr;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = at(i);
        if (j >= n) continue;
        if (n_bias > 0 && last[j]) v[i] += bias[last[j] - 1];
        if (n_hist > 0 && count[j]) {
            if (repeats) v[i] = v[i] > 0.0f ? __fdiv_rn(v[i], rep) : __fmul_rn(v[i], rep);
            v[i] = __fsub_rn(v[i], __fadd_rn(__fmul_rn(freq, (float)count[j]), pres));
        }
        if (mask && !((mask[(lo + j) >> 5] >> ((lo + j) & 31)) & 1u)) v[i] = -INFINITY;
    }
    float *y = p.y + row * p.y_stride + lo;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const int j = at(i);
            if (j + 3 < n) {
                *reinterpret_cast<float4 *>(y + j) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (j + c < n) y[j + c] = v[i + c];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (at(i) < n) y[at(i)] = v[i];
    }
}

} // namespace

int launch_logits_adjust(float *out, const float *logits, const krk_cuda_adjust &a, cudaStream_t st) {
    AdjustParams p;
    p.x = logits;
    p.y = out;
    p.x_stride = a.stride, p.y_stride = a.out_stride, p.hist_stride = a.hist_stride, p.bias_stride = a.bias_stride, p.mask_stride = a.mask_stride;
    p.n = a.n_vocab;
    p.hist = static_cast<const int32_t *>(a.hist), p.hist_len = static_cast<const int32_t *>(a.hist_len);
    p.bias_ids = static_cast<const int32_t *>(a.bias_ids), p.bias = static_cast<const float *>(a.bias), p.bias_len = static_cast<const int32_t *>(a.bias_len);
    p.rep = static_cast<const float *>(a.rep), p.freq = static_cast<const float *>(a.freq), p.pres = static_cast<const float *>(a.pres);
    p.mask = static_cast<const uint32_t *>(a.mask), p.mask_row = static_cast<const int32_t *>(a.mask_row);
    p.hist_n = (int)a.hist_n, p.bias_n = (int)a.bias_n, p.n_masks = a.mask ? a.n_masks : 0;
    const bool vec = ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                     (a.n_rows == 1 || (a.stride % 4 == 0 && a.out_stride % 4 == 0));
    const int per = 4;
    p.slice = per * kThreads;
    const int64_t slices = (a.n_vocab + p.slice - 1) / p.slice;
    if (slices * a.n_rows > INT32_MAX) return KRK_CUDA_ESHAPE;
    p.slices = (int)slices;
    auto kernel = vec ? logits_adjust_kernel<4, true> : logits_adjust_kernel<4, false>;
    return launched(launch_overlapped(kernel, dim3((unsigned)(slices * a.n_rows)), dim3(kThreads), st, p));
}

} // namespace krk_cuda
