// krk_cuda_logits_adjust: what a sampler does to the rows of logits before it ranks them, in one pass: sparse biases, penalties for
// tokens of the row's history, a grammar's mask.
//
//   v = x + bias[id];   c = times of id in the history;   c > 0:  v = v > 0 ? v / rep : v * rep,  v -= freq * c + pres;
//   the grammar does not allow id:  v = -inf
//
// Bound: reading and writing the rows once. The lists name few ids of a row, many of them more than once, so a block of threads counts those
// of its slice of the row in shared memory (whole numbers: the order of the atomics does not matter; of an id's biases the
// highest place in the list is kept, the same way) while its slice of the logits is on its way into registers. 64 rows of 128,256: 23 us
// with histories, biases and masks, 12 with none of them, a plain copy 10.6.
#include "krk_common.cuh"

namespace krk_cuda {

namespace {

struct AdjustParams {
    const float *x;
    float *y;
    int64_t x_stride, y_stride, hist_stride, bias_stride, mask_stride, n;
    const int32_t *hist, *hist_len, *bias_ids, *bias_len, *mask_row;
    const float *bias, *rep, *freq, *pres;
    const uint32_t *mask;
    int hist_n, bias_n, n_masks, slices;
};

// PER: values of a thread. VEC: rows begin on 16-byte boundaries, four values at a time. PACKED: lists of less than 2^16 ids, whose
// counts and places share a word.
template <int kThreads, int PER, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads)
logits_adjust_kernel(const __grid_constant__ AdjustParams p) {
    constexpr int kSlice = PER * kThreads, kEarly = 1;
    __shared__ __align__(16) int table[PACKED ? kSlice : 2 * kSlice];
    int *const count = table, *const last = table + (PACKED ? 0 : kSlice);   // last: place in the list of biases plus one, in the upper half of a word if packed
    constexpr int kPlace = PACKED ? 16 : 0, kTimes = PACKED ? 0xFFFF : -1;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / p.slices;
    const int lo = (int)(blockIdx.x - row * p.slices) * kSlice, n = min(kSlice, (int)p.n - lo);
    // values 4 i .. 4 i + 3 of a thread follow each other (VEC), or lie kThreads apart
    auto at = [&](int i) { return VEC ? (i >> 2) * 4 * kThreads + 4 * tid + (i & 3) : i * kThreads + tid; };
    // all that does not wait for anything: the values, the first ids (those behind the row's are dropped below), the mask's words
    const float *x = p.x + row * p.x_stride + lo;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
        if (VEC && at(i) + 3 < n) {
            *reinterpret_cast<float4 *>(v + i) = *reinterpret_cast<const float4 *>(x + at(i));
        } else {
#pragma unroll
            for (int c = i; c < i + 4; c++) v[c] = at(c) < n ? x[at(c)] : 0.0f;
        }
    }
    const int32_t *hist = p.hist + row * p.hist_stride;
    const int wide = (reinterpret_cast<uintptr_t>(hist) & 15) == 0 ? p.hist_n & ~3 : 0;
    int4 early[kEarly];
#pragma unroll
    for (int i = 0; i < kEarly; i++) early[i] = 4 * (tid + i * kThreads) < wide ? reinterpret_cast<const int4 *>(hist)[tid + i * kThreads] : make_int4(-1, -1, -1, -1);
    const int32_t *bias_ids = p.bias_ids + row * p.bias_stride;
    const int early_bias = p.bias && tid < p.bias_n ? bias_ids[tid] : -1;
    const int n_hist = !p.hist ? 0 : p.hist_len ? min(max(p.hist_len[row], 0), p.hist_n) : p.hist_n;
    const int n_bias = !p.bias ? 0 : p.bias_len ? min(max(p.bias_len[row], 0), p.bias_n) : p.bias_n;
    const int32_t m_row = !p.mask ? -1 : p.mask_row ? p.mask_row[row] : (int32_t)row;
    const uint32_t *mask = m_row >= 0 && m_row < p.n_masks ? p.mask + m_row * p.mask_stride : nullptr;
    uint32_t ok[VEC ? PER / 4 : PER];
#pragma unroll
    for (int i = 0; i < (VEC ? PER / 4 : PER); i++) {
        const int j = at(VEC ? 4 * i : i);
        ok[i] = mask && j < n ? mask[(lo + j) >> 5] >> ((lo + j) & 31) : 0xFFFFFFFFu;
    }
    if (n_hist > 0 || n_bias > 0)
        for (int i = 4 * tid; i < (PACKED ? kSlice : 2 * kSlice); i += 4 * kThreads) *reinterpret_cast<int4 *>(table + i) = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (n_bias > 0) {
        for (int i = tid; i < n_bias; i += kThreads) {
            const uint32_t j = (uint32_t)(i == tid ? early_bias : bias_ids[i]) - (uint32_t)lo;
            if (j < (uint32_t)n) atomicMax(reinterpret_cast<unsigned *>(&last[j]), (unsigned)(i + 1) << kPlace);
        }
        if (PACKED) __syncthreads();   // (the counts go on top)
    }
    // (an id outside the row is outside every slice: those below lo, and -1, wrap around)
    auto meet = [&](int32_t id) {
        const uint32_t j = (uint32_t)id - (uint32_t)lo;
        if (j < (uint32_t)n) atomicAdd(&count[j], 1);
    };
    auto meet4 = [&](int4 id, int i) {
        if (i < n_hist) meet(id.x);
        if (i + 1 < n_hist) meet(id.y);
        if (i + 2 < n_hist) meet(id.z);
        if (i + 3 < n_hist) meet(id.w);
    };
#pragma unroll
    for (int i = 0; i < kEarly; i++)
        if (4 * (tid + i * kThreads) < n_hist) meet4(early[i], 4 * (tid + i * kThreads));
    for (int i = 4 * (tid + kEarly * kThreads); i < wide && i < n_hist; i += 4 * kThreads) meet4(*reinterpret_cast<const int4 *>(hist + i), i);
    for (int i = wide + tid; i < n_hist; i += kThreads) meet(hist[i]);
    __syncthreads();
    const float rep = p.rep ? p.rep[row] : 1.0f, freq = p.freq ? p.freq[row] : 0.0f, pres = p.pres ? p.pres[row] : 0.0f;
    const bool repeats = rep > 0.0f && rep != 1.0f;
    const float *bias = p.bias + row * p.bias_stride;
    float *y = p.y + row * p.y_stride + lo;
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
        int word[4], place[4];
        const bool listed = n_hist > 0 || n_bias > 0;
        if constexpr (VEC) {
            *reinterpret_cast<int4 *>(word) = listed ? *reinterpret_cast<const int4 *>(count + at(i)) : make_int4(0, 0, 0, 0);
            if constexpr (!PACKED) *reinterpret_cast<int4 *>(place) = listed ? *reinterpret_cast<const int4 *>(last + at(i)) : make_int4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                word[c] = listed ? count[at(i + c)] : 0;
                if constexpr (!PACKED) place[c] = listed ? last[at(i + c)] : 0;
            }
        }
        int any = word[0] | word[1] | word[2] | word[3];
        if constexpr (!PACKED) any |= place[0] | place[1] | place[2] | place[3];
        if (any) {   // (few ids are in a list)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                float &z = v[i + c];
                const int of = PACKED ? (int)((unsigned)word[c] >> kPlace) : place[c], times = word[c] & kTimes;
                if (of) z += bias[of - 1];
                if (times) {
                    if (repeats) z = z > 0.0f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
                    z = __fsub_rn(z, __fadd_rn(__fmul_rn(freq, (float)times), pres));
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t w = VEC ? ok[i / 4] >> c : ok[VEC ? 0 : i + c];
            if (!(w & 1u)) v[i + c] = -INFINITY;
        }
        if (VEC && at(i) + 3 < n) {
            *reinterpret_cast<float4 *>(y + at(i)) = *reinterpret_cast<const float4 *>(v + i);
        } else {
#pragma unroll
            for (int c = i; c < i + 4; c++)
                if (at(c) < n) y[at(c)] = v[c];
        }
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
    p.hist_n = a.hist ? (int)a.hist_n : 0, p.bias_n = a.bias ? (int)a.bias_n : 0, p.n_masks = a.mask ? a.n_masks : 0;
    const bool vec = ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
                     (a.n_rows == 1 || (a.stride % 4 == 0 && a.out_stride % 4 == 0));
    // A block looks through the whole lists for its slice: 4096 values a block, but 1024 where the longer slices would leave SMs without one
    // (64 rows of 128,256 with up to 4096 ids each: 38.6 us with 1024, 23 with 4096, 26 with 8192).
    const bool packed = p.hist_n < 65536 && p.bias_n < 65535, wide = packed && (a.n_vocab + 4095) / 4096 * a.n_rows >= 2 * sm_count();
    const int threads = wide ? 512 : 256, slice = wide ? 4096 : 1024;
    const int64_t slices = (a.n_vocab + slice - 1) / slice;
    if (slices * a.n_rows > INT32_MAX) return KRK_CUDA_ESHAPE;
    p.slices = (int)slices;
    auto kernel = wide ? (vec ? logits_adjust_kernel<512, 8, true, true> : logits_adjust_kernel<512, 8, false, true>)
                  : packed ? (vec ? logits_adjust_kernel<256, 4, true, true> : logits_adjust_kernel<256, 4, false, true>)
                           : (vec ? logits_adjust_kernel<256, 4, true, false> : logits_adjust_kernel<256, 4, false, false>);
    return launched(launch_overlapped(kernel, dim3((unsigned)(slices * a.n_rows)), dim3(threads), st, p));
}

} // namespace krk_cuda
