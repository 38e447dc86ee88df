// krk_cuda_block_norm: what lies between two blocks' matmuls, in one pass over the rows.
//
//   h = residual + alpha * gate * P(x),  P(x) = x / sqrt(mean(x^2) + eps) * (offset + post_weight);   y = h / sqrt(mean(h^2) + eps) * (offset + weight)
//
// Bound: reading x and the residual and writing h and y once. A block of threads has a row in registers from its loads to the last store: the two sums of
// squares are a shuffle and a trip through shared memory each. Sums are f32, a thread's values first, then a tree. Weights and a shared gate come out of level 2.
// Measured: one row of 4096 5.7 us (a launch; two trips to memory); 2048 rows, f16 out, two norms and a gate 25.4 us, 4.6 TB/s of a copy's 6.5. There two groups of four
// values a thread are best of a block a row: one (1024 threads) 29.5, four 27.6, eight 37.2; blocks that stay, below, 21.1, 5.5 TB/s.
#include "krk_common.cuh"

#include <atomic>

namespace krk_cuda {

namespace {

struct NormParams {
    const float *x, *residual, *gate, *post_weight, *weight;
    float *h;
    void *y;
    int64_t x_stride, residual_stride, gate_stride, h_stride, y_stride;
    int n, post_norm, half;
    float alpha, eps, offset;
};

__device__ __forceinline__ float block_sum(float v, float *part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

__device__ __forceinline__ void copy16_ahead(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// VEC values at a time, PER times a thread; PER 0: rows wider than the registers of a block, walked again for each step (h and then x from memory).
template <int VEC, int PER>
__global__ void __launch_bounds__(PER == 0 ? 1024 : 512)
block_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float part[2][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t row = blockIdx.x;
    const float *x = p.x + row * p.x_stride, *res = p.residual ? p.residual + row * p.residual_stride : nullptr, *gate = p.gate ? p.gate + row * p.gate_stride : nullptr;
    float *h = p.h ? p.h + row * p.h_stride : nullptr;
    const int step = VEC * (int)blockDim.x, at0 = VEC * (int)threadIdx.x;
    auto load = [&](float (&v)[VEC], const float *from, int at) {
        if constexpr (VEC == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(from + at);
        else v[0] = from[at];
    };
    auto store_y = [&](const float (&v)[VEC], int at) {
        if (p.half) {
            __half *y = static_cast<__half *>(p.y) + row * p.y_stride + at;
            if constexpr (VEC == 4) {
                __half2 two[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
                *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<uint2 *>(two);
            } else {
                *y = __float2half_rn(v[0]);
            }
        } else {
            float *y = static_cast<float *>(p.y) + row * p.y_stride + at;
            if constexpr (VEC == 4) *reinterpret_cast<float4 *>(y) = *reinterpret_cast<const float4 *>(v);
            else *y = v[0];
        }
    };
    // h of a group of values, from x (times the norm's factor) and the rest
    auto mix = [&](float (&v)[VEC], const float (&r)[VEC], float f, int at) {
        if (p.post_norm) {
            float w[VEC];
            if (p.post_weight) load(w, p.post_weight, at);
#pragma unroll
            for (int c = 0; c < VEC; c++) v[c] = p.post_weight ? v[c] * f * (p.offset + w[c]) : v[c] * f;
        }
        if (gate) {
            float w[VEC];
            load(w, gate, at);
#pragma unroll
            for (int c = 0; c < VEC; c++) v[c] *= w[c];
        }
#pragma unroll
        for (int c = 0; c < VEC; c++) v[c] = res ? fmaf(p.alpha, v[c], r[c]) : p.alpha * v[c];
    };
    auto scale = [&](float (&v)[VEC], float f, int at) {
        float w[VEC];
        if (p.weight) load(w, p.weight, at);
#pragma unroll
        for (int c = 0; c < VEC; c++) v[c] = p.weight ? v[c] * f * (p.offset + w[c]) : v[c] * f;
    };
    auto factor = [&](float sum) { return 1.0f / sqrtf(sum / (float)p.n + p.eps); };
    float f = 1.0f, sum = 0.0f;
    if constexpr (PER > 0) {
        float v[PER][VEC], r[PER][VEC];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = at0 + i * step;
#pragma unroll
            for (int c = 0; c < VEC; c++) v[i][c] = r[i][c] = 0.0f;
            if (at < p.n) {
                load(v[i], x, at);
                if (res) load(r[i], res, at);
            }
        }
        if (p.post_norm) {
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
                for (int c = 0; c < VEC; c++) sum = fmaf(v[i][c], v[i][c], sum);
            f = factor(block_sum(sum, part[0]));
            sum = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = at0 + i * step;
            if (at >= p.n) continue;
            mix(v[i], r[i], f, at);
            if (h) {
                if constexpr (VEC == 4) *reinterpret_cast<float4 *>(h + at) = *reinterpret_cast<const float4 *>(v[i]);
                else h[at] = v[i][0];
            }
#pragma unroll
            for (int c = 0; c < VEC; c++) sum = fmaf(v[i][c], v[i][c], sum);
        }
        f = factor(block_sum(sum, part[1]));
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = at0 + i * step;
            if (at >= p.n) continue;
            scale(v[i], f, at);
            store_y(v[i], at);
        }
    } else {
        if (p.post_norm) {
            for (int at = at0; at < p.n; at += step) {
                float v[VEC];
                load(v, x, at);
#pragma unroll
                for (int c = 0; c < VEC; c++) sum = fmaf(v[c], v[c], sum);
            }
            f = factor(block_sum(sum, part[0]));
            sum = 0.0f;
        }
        // (h may lie in x's place: without it x is walked again; a thread meets its own values each time)
        for (int at = at0; at < p.n; at += step) {
            float v[VEC], r[VEC] = {};
            load(v, x, at);
            if (res) load(r, res, at);
            mix(v, r, f, at);
            if (h) {
                if constexpr (VEC == 4) *reinterpret_cast<float4 *>(h + at) = *reinterpret_cast<const float4 *>(v);
                else h[at] = v[0];
            }
#pragma unroll
            for (int c = 0; c < VEC; c++) sum = fmaf(v[c], v[c], sum);
        }
        const float g = factor(block_sum(sum, part[1]));
        for (int at = at0; at < p.n; at += step) {
            float v[VEC];
            if (h) {
                load(v, h, at);
            } else {
                float r[VEC] = {};
                load(v, x, at);
                if (res) load(r, res, at);
                mix(v, r, f, at);
            }
            scale(v, g, at);
            store_y(v, at);
        }
    }
}

// Many rows of 2564 values and more: blocks that stay, two a multiprocessor, each with every gridDim.x-th row. A thread's values of the next two rows are on their way while it works on one
// (asynchronous copies into places of its own in shared memory, which nobody else reads), weights and a shared gate stay in its registers.
// A thread has two groups of four values of a row.
constexpr int kRowsPer = 2, kRowsThreads = 512;
__global__ void __launch_bounds__(kRowsThreads, 2)
block_norm_rows_kernel(const __grid_constant__ NormParams p, int64_t rows) {
    constexpr int PER = kRowsPer;
    __shared__ float part[4][32];
    extern __shared__ float4 ahead[];   // [stage][x, residual][PER][thread]
    const int tid = threadIdx.x, threads = (int)blockDim.x, groups = p.n / 4;
    float4 post[PER], gate[PER], weight[PER];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool gated = p.gate != nullptr;
    auto value = [&](const float *from, int at, float otherwise, float more) {
        const float4 v = from ? reinterpret_cast<const float4 *>(from)[at] : make_float4(otherwise, otherwise, otherwise, otherwise);
        return make_float4(v.x + more, v.y + more, v.z + more, v.w + more);
    };
    auto ask = [&](int64_t row, int stage) {
        if (row < rows) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int at = tid + i * threads;
                if (at >= groups) continue;
                float4 *to = ahead + (stage * 2 * PER + i) * threads + tid;
                copy16_ahead(to, p.x + row * p.x_stride + 4 * at);
                if (p.residual) copy16_ahead(to + PER * threads, p.residual + row * p.residual_stride + 4 * at);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ask(blockIdx.x, 0);
    ask((int64_t)blockIdx.x + gridDim.x, 1);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int at = min(tid + i * threads, groups - 1);
        // (what a norm multiplies by without a weight is 1)
        post[i] = value(p.post_weight, at, 1.0f, p.post_weight ? p.offset : 0.0f);
        weight[i] = value(p.weight, at, 1.0f, p.weight ? p.offset : 0.0f);
        gate[i] = value(p.gate, at, 1.0f, 0.0f);
    }
    auto squares = [](float4 v, float sum) { return fmaf(v.w, v.w, fmaf(v.z, v.z, fmaf(v.y, v.y, fmaf(v.x, v.x, sum)))); };
    auto times = [](float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); };
    auto factor = [&](float sum) { return 1.0f / sqrtf(sum / (float)p.n + p.eps); };
    int stage = 0, turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 2) {
        ask(row + 2 * (int64_t)gridDim.x, stage == 0 ? 2 : stage - 1);
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        float4 v[PER];
        float sum = 0.0f, f = 1.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (tid + i * threads < groups) v[i] = ahead[(stage * 2 * PER + i) * threads + tid];
            sum = squares(v[i], sum);
        }
        if (p.post_norm) f = factor(block_sum(sum, part[turn]));
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = tid + i * threads;
            if (at >= groups) continue;
            if (p.post_norm) {
                v[i] = make_float4(v[i].x * f, v[i].y * f, v[i].z * f, v[i].w * f);
                if (p.post_weight) v[i] = times(v[i], post[i]);
            }
            if (gated) v[i] = times(v[i], gate[i]);
            if (p.residual) {
                const float4 r = ahead[(stage * 2 * PER + PER + i) * threads + tid];
                v[i] = make_float4(fmaf(p.alpha, v[i].x, r.x), fmaf(p.alpha, v[i].y, r.y), fmaf(p.alpha, v[i].z, r.z), fmaf(p.alpha, v[i].w, r.w));
            } else {
                v[i] = make_float4(p.alpha * v[i].x, p.alpha * v[i].y, p.alpha * v[i].z, p.alpha * v[i].w);
            }
            if (p.h) reinterpret_cast<float4 *>(p.h + row * p.h_stride)[at] = v[i];
            sum = squares(v[i], sum);
        }
        f = factor(block_sum(sum, part[turn + 1]));
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int at = tid + i * threads;
            if (at >= groups) continue;
            v[i] = make_float4(v[i].x * f, v[i].y * f, v[i].z * f, v[i].w * f);
            if (p.weight) v[i] = times(v[i], weight[i]);
            if (p.half) {
                __half2 two[2] = {__floats2half2_rn(v[i].x, v[i].y), __floats2half2_rn(v[i].z, v[i].w)};
                reinterpret_cast<uint2 *>(static_cast<__half *>(p.y) + row * p.y_stride)[at] = *reinterpret_cast<uint2 *>(two);
            } else {
                reinterpret_cast<float4 *>(static_cast<float *>(p.y) + row * p.y_stride)[at] = v[i];
            }
        }
        stage = stage == 2 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Once a device: the limit of shared memory.
int raise_shared() {
    static std::atomic<uint64_t> ready = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        e = cudaFuncSetAttribute(block_norm_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 2 * kRowsPer * kRowsThreads * 16);
        if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e == cudaSuccess) return KRK_CUDA_OK;
    note_cuda_error(e);
    return KRK_CUDA_ELAUNCH;
}

} // namespace

int launch_block_norm(void *y, float *h_out, const float *x, const krk_cuda_norm &m, cudaStream_t st) {
    NormParams p;
    p.x = x, p.residual = static_cast<const float *>(m.residual), p.gate = static_cast<const float *>(m.gate);
    p.post_weight = static_cast<const float *>(m.post_weight), p.weight = static_cast<const float *>(m.weight);
    p.h = h_out, p.y = y;
    p.x_stride = m.x_stride, p.residual_stride = m.residual_stride, p.gate_stride = m.gate_stride, p.h_stride = m.h_stride, p.y_stride = m.y_stride;
    p.n = (int)m.n, p.post_norm = m.post_norm != 0, p.half = m.y_dtype == KRK_CUDA_X_F16;
    p.alpha = m.alpha, p.eps = m.eps, p.offset = m.offset;
    // four values at a time where every row of everything begins on their boundary
    const uintptr_t bases = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(m.residual) | reinterpret_cast<uintptr_t>(m.gate) | reinterpret_cast<uintptr_t>(m.post_weight) |
                            reinterpret_cast<uintptr_t>(m.weight) | reinterpret_cast<uintptr_t>(h_out);
    bool vec = bases % 16 == 0 && reinterpret_cast<uintptr_t>(y) % (p.half ? 8 : 16) == 0 && m.n % 4 == 0;
    if (m.rows > 1) vec = vec && (m.x_stride | m.y_stride | (m.residual ? m.residual_stride : 0) | (m.gate ? m.gate_stride : 0) | (h_out ? m.h_stride : 0)) % 4 == 0;
    const int groups = (int)(vec ? m.n / 4 : m.n);
    const int per = groups <= 512 ? 1 : groups <= 1024 ? 2 : groups <= 2048 ? 4 : groups <= 4096 ? 8 : 0;
    const int threads = per == 0 ? 1024 : ((groups + per - 1) / per + 31) / 32 * 32;
    // Two norms, a gate, f16 out, us by blocks that stay and by a block a row: rows of 4096 values, 300 6.8 and 6.5, 600 9.9 and 10.7, 2048 21.1 and 23.3, 7000 71.1 and 66.4; 2048 rows of
    // 3584 values 19.2 and 21.6, of 2640 16.5 and 17.2, of 2560 19.2 and 16.8, of 2304 17.9 and 14.9. One group of values a thread: 2048 rows of 2048 14.3 and 15.1, of 2044 15.3 both,
    // of 1280 13.3 and 10.5, which does not pay for a form of its own.
    const int stay = 2 * sm_count();
    if (vec && per == kRowsPer && groups > 640 && m.gate_stride == 0 && m.rows >= 2 * (int64_t)stay && m.rows * m.n <= 1 << 24) {
        const size_t shared = (size_t)3 * 2 * kRowsPer * threads * 16;
        const int rc = raise_shared();
        if (rc != KRK_CUDA_OK) return rc;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)stay), cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = shared, cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr, cfg.numAttrs = 1;
        return launched(cudaLaunchKernelEx(&cfg, block_norm_rows_kernel, p, (int64_t)m.rows));
    }
    auto kernel = vec ? (per == 1 ? block_norm_kernel<4, 1> : per == 2 ? block_norm_kernel<4, 2> : per == 4 ? block_norm_kernel<4, 4> : per == 8 ? block_norm_kernel<4, 8> : block_norm_kernel<4, 0>)
                      : (per == 1 ? block_norm_kernel<1, 1> : per == 2 ? block_norm_kernel<1, 2> : per == 4 ? block_norm_kernel<1, 4> : per == 8 ? block_norm_kernel<1, 8> : block_norm_kernel<1, 0>);
    return launched(launch_overlapped(kernel, dim3((unsigned)m.rows), dim3(threads), st, p));
}

} // namespace krk_cuda
