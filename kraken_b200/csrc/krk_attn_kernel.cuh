// The kernel of krk_cuda_attention_tree, one instantiation per cache type, head size and number of row tiles.
//
// What bounds it: reading the cache, while a key head's rows are few (a decode step: one to four drafted tokens times the group); the
// issue slots and the tensor pipe beyond. Hence the split: a warp takes 16 positions at a time of its own (a piece of one page), copies
// them with 16-byte asynchronous copies into a ring of its own, and keeps the running maximum, sum and output of all rows of
// the block in registers; no warp waits for another one until the item's end, where the four of a CTA add up.
//
// The products are `mma.sync` m16n8k16 of f16 with f32 sums, with the cache as the operand of 16 rows and the queries as the one of
// eight columns: S^T = K Q^T, O^T = V^T P^T. (Queries as the 16 rows: a group of four heads filled a quarter of each product, 131,072
// positions in 8 bits took 97 us.) Activations are f32, so a query enters as two f16 terms under a power of two of its row (22 bits),
// and so do the weights of a step (times 2^14: terms far below the maximum keep their bits). Up to four rows the two terms are
// neighbouring columns of one product, else products in a row. Cache values enter exactly: f16 as they are; 8- and 4-bit quants as whole
// numbers, whose block scales multiply the f32 sums of a block's products (keys) and the weights before they are split (values; there
// under the power of two of the greatest scale that any row of the block has seen so far, which the sums are rescaled to like to a new maximum).
//
// Measured, 16 sequences of 8192 positions in pages of 64, 8 key heads of 128 values, four rows each (bytes of the cache a second): f16 90.7 us
// (5.9 TB/s), 8 bits 72.0 (4.0), 4 bits 70.0 (2.2). In 8 and 4 bits the latency of the dependent steps from quants to operands bounds it: 15 % fewer
// instructions changed nothing.
//
// Two terms of 11 bits where f32 has 24 are a choice: a third one is half as many products again. Against 64 bits the outputs are as near as
// those of f32 products, whose own sums round as much: one token over 131,072 positions in 8 bits 6.7e-7 relative (f32 1.6e-6), 48 ragged sequences 1.1e-6 (1.1e-6).
#pragma once

#include <atomic>
#include <type_traits>

#include "krk_attn_tree.cuh"

namespace krk_cuda {
namespace attn {

__host__ __device__ constexpr int row_bytes_of(int type, int d) { return type == KRK_CUDA_KV_F16 ? 2 * d : type == KRK_CUDA_KV_Q8 ? d : d / 2; }
__host__ __device__ constexpr int scale_bytes_of(int type, int d) { return type == KRK_CUDA_KV_F16 ? 0 : d / 16; }   // of a row

// R: rows of a block, 4 (both terms of a query in one product), 8 or 16.
// Shared memory of a CTA: the ring, the query block, row data. As many CTAs an SM as registers and a ring of three stages (of two, for the
// second CTA) leave room for.
__host__ __device__ constexpr int stage_bytes(int ct, int d) { return 2 * kChunk * (row_bytes_of(ct, d) + scale_bytes_of(ct, d)); }   // keys and values of a chunk, then their scales
__host__ __device__ constexpr int q_bytes(int d, int r) { return 4 * r * (d + 8); }
__host__ __device__ constexpr int fixed_bytes(int d, int r) { return q_bytes(d, r) + r * 32 + kWarps * r * 8 + kWarps * 6 * 8; }
__host__ __device__ constexpr int sums_bytes(int d, int r) { return kWarps * r * (d + 4) * 4; }   // the warps' outputs, in place of the ring
__host__ __device__ constexpr int room_of(int ctas, int d, int r) { return 226 * 1024 / ctas - 1024 - fixed_bytes(d, r); }
__host__ __device__ constexpr int ring_of(int ctas, int ct, int d, int r) {
    const int n = room_of(ctas, d, r) / (kWarps * stage_bytes(ct, d));
    return n > 6 ? 6 : n;
}
__host__ __device__ constexpr bool fits(int ctas, int ct, int d, int r) { return ring_of(ctas, ct, d, r) >= 3 && sums_bytes(d, r) <= room_of(ctas, d, r); }
__host__ __device__ constexpr int ctas_per_sm(int ct, int d, int r) {
    const int out_regs = d / 16 * 4 * (r <= 8 ? 1 : r / 8), most = r == 4 && d <= 128 ? 4 : out_regs <= 32 ? 3 : 2;
    return most >= 4 && fits(4, ct, d, r) ? 4 : most >= 3 && fits(3, ct, d, r) ? 3 : ring_of(2, ct, d, r) >= 2 && sums_bytes(d, r) <= room_of(2, d, r) ? 2 : 1;
}
template <int D, int CT, int R>
struct Shape {
    static constexpr bool kPair = R == 4;                          // both terms of a row in one tile of columns
    static constexpr int NT = R <= 8 ? 1 : R / 8;                  // tiles of columns
    static constexpr int NC = kPair ? 1 : 2;                       // rows of a tile that a lane has
    static constexpr int RB = row_bytes_of(CT, D);
    static constexpr int SB = scale_bytes_of(CT, D);
    static constexpr int kStage = stage_bytes(CT, D);
    static constexpr int kPitch = D + 8;                           // of a query row, in halves
    static constexpr int kQ = q_bytes(D, R);
    static constexpr int kRows = R * 32;                           // see Rows
    static constexpr bool kQInRegs = D / 16 * 4 * NT <= 64;        // registers of a lane for the queries' terms (kPair: half of them), as many as for outputs
    static constexpr int kSumPitch = D + 4;
    static constexpr int kCtas = ctas_per_sm(CT, D, R);
    static constexpr int kRing = ring_of(kCtas, CT, D, R);
    static constexpr int kRingBytes = kWarps * kRing * kStage;
    static constexpr int kFront = kRingBytes > sums_bytes(D, R) ? kRingBytes : sums_bytes(D, R);
    static constexpr int kBytes = kFront + fixed_bytes(D, R);
    static_assert(kRing >= 2, "ring");
    static_assert(kBytes <= 226 * 1024 / kCtas - 1024, "shared memory");
};

// 16-byte pieces of a row lie exclusive-ored, so that eight rows' pieces of a column, and four rows' pairs of pieces, meet
// different banks. RB % 32 == 16: they do as they are.
template <int RB>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (RB % 128 == 0) return ((row & 3) << 1) | ((row >> 2) & 1);
    else if constexpr (RB % 64 == 0) return (row & 2) | ((row >> 2) & 1);
    else if constexpr (RB % 32 == 0) return (row >> 2) & 1;
    else return 0;
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm2(uint32_t r[2], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm2t(uint32_t r[2], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a));
}
// An 8 x 8 tile of f16 in the layout of sums (row g, columns 2t and 2t + 1) as an operand's: transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma0(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {   // onto zeros
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The soft limit of a score, in the log2 domain (log2(e) goes to the tangent: times a limit beyond 2.3e38 it would be infinite).
static __device__ __noinline__ float capped(float x, float cap) { return cap * (1.44269504f * tanhf(x / cap)); }
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// Two f32 as the sum of two f16 each.
__device__ __forceinline__ void split(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = bits(h);
    lo = bits(__floats2half2_rn(a - f.x, b - f.y));
}
// Bytes i and j of w, which hold u, as the f16 u - off: 0x6400 | u is 1024 + u.
template <int I, int J>
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t off) {
    const uint32_t v = __byte_perm(w, 0x64646464u, I | 0x40 | J << 8 | 0x4000);
    return bits(__hsub2(half2_of(v), half2_of(off)));
}

// Where value d of a query row goes, so that the four values a lane reads of a key's packed bytes are those that the fragment's
// layout gives it: a 32-value block is two steps of 16, lane t has columns 2t, 2t + 1, 2t + 8, 2t + 9 of a step.
template <int CT>
__device__ __forceinline__ int column_of(int d) {
    if constexpr (CT == KRK_CUDA_KV_F16) return d;
    const int e = d & 31, c = e & 3;
    const int t = CT == KRK_CUDA_KV_Q8 ? e >> 3 : (e & 15) >> 2, step = CT == KRK_CUDA_KV_Q8 ? (e >> 2) & 1 : e >> 4;
    return (d & ~31) + 16 * step + 2 * t + (c & 1) + (c >= 2 ? 8 : 0);
}
// The value of output tile m that a lane has in its half h (rows g and g + 8 of the tile). Packed values: even ones in the upper
// rows, odd ones in the lower.
template <int CT>
__device__ __forceinline__ int value_of(int m, int g, int h) {
    if constexpr (CT == KRK_CUDA_KV_F16) return 16 * m + g + 8 * h;
    return 16 * m + 2 * g + h;
}
// NB f16 scales of a position.
template <int NB>
__device__ __forceinline__ void scales(float (&d)[NB], const uint8_t *from) {
    if constexpr (NB % 2 == 0) {
        uint32_t w[NB / 2];
        if constexpr (NB % 8 == 0) {
            *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(from);
        } else if constexpr (NB % 4 == 0) {
            *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(from);
        } else {
#pragma unroll
            for (int j = 0; j < NB / 2; j++) w[j] = reinterpret_cast<const uint32_t *>(from)[j];
        }
#pragma unroll
        for (int j = 0; j < NB / 2; j++) {
            const float2 f = __half22float2(half2_of(w[j]));
            d[2 * j] = f.x, d[2 * j + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NB; j++) d[j] = __half2float(reinterpret_cast<const __half *>(from)[j]);
    }
}

struct Rows {   // of a block of rows, in shared memory
    float scale;       // takes a row's sum of products to its score in the log2 domain (softcap: to the natural score)
    int first;         // first position before the drafted tokens that it sees
    uint64_t mask;     // drafted tokens that it sees
    int q_row, head;   // its place in q and out; -1: no row
    uint64_t any;      // of the first row: drafted tokens that some row of the block sees
};
static_assert(sizeof(Rows) == 32, "Shape::kRows");

template <int D, int CT, int R>
__global__ void __launch_bounds__(kThreads, Shape<D, CT, R>::kCtas)
attn_kernel(const __grid_constant__ Params p) {
    using S = Shape<D, CT, R>;
    constexpr int RB = S::RB, SB = S::SB, NB = D / 32, NT = S::NT, NC = S::NC, NM = D / 16;
    constexpr bool kQuant = CT != KRK_CUDA_KV_F16, kPair = S::kPair;
    constexpr uint32_t kOff = CT == KRK_CUDA_KV_Q8 ? 0x64806480u : 0x64086408u;   // 1024 + 128 (signed bytes with their top bit turned over), 1024 + 8
    extern __shared__ __align__(128) uint8_t smem[];
    float *sums = reinterpret_cast<float *>(smem);
    // rows of the query block: with kPair a row's second terms follow its first ones, else all second terms the first ones
    __half *q_mem = reinterpret_cast<__half *>(smem + S::kFront);
    Rows *rows = reinterpret_cast<Rows *>(smem + S::kFront + S::kQ);
    float2 *warp_ml = reinterpret_cast<float2 *>(smem + S::kFront + S::kQ + S::kRows);   // [warp][R]

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    Walk<R> walk;
    walk.start(p);
    if (!p.whole && tid == 0) p.shared[blockIdx.x].parts = 0;
    const uint32_t ring = smem_addr(smem) + warp * S::kRing * S::kStage;
    uint8_t *ring_mem = smem + warp * S::kRing * S::kStage;
    int64_t *stage_rows = reinterpret_cast<int64_t *>(warp_ml + kWarps * R) + warp * S::kRing;   // the pool's row that a stage begins with

    while (walk.next(p)) {
        const Seq &sq = walk.sq;
        const int s = walk.s, kvh = walk.kvh, block = walk.block, n_rows = walk.n_rows, n_tiles = (n_rows + 7) / 8, tile0 = walk.tile0, tile1 = tile0 + walk.tiles;
        const bool begins = walk.begins, ends = walk.ends;
        if (walk.parts > 0 && tid == 0) walk.note(p);

        // ---- the block's queries: a warp takes rows in turn; all its rows' loads go out before the pages are waited for
        constexpr int kPer = R / kWarps;
        float x[kPer][NB];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int r = warp + kWarps * j, rr = block * R + r, i = rr / p.group;
            const float *from = p.q + (int64_t)(sq.q0 + i) * p.q_stride + (kvh * p.group + rr - i * p.group) * D + lane;
#pragma unroll
            for (int c = 0; c < NB; c++) x[j][c] = r < n_rows ? from[32 * c] : 0.0f;
        }

        // ---- pages of this warp's chunks: lane l holds that of the l-th from the last refill on, as a row of the pool
        const int chunk0 = tile0 * kWarps + warp, n_chunks = tile1 - tile0;
        const int32_t *table = p.table + (size_t)s * p.table_width;
        auto find_row = [&](int i) -> int64_t {   // -1: behind the last position, or not a page
            const int pos = (chunk0 + i * kWarps) * kChunk;
            if (i >= n_chunks || pos >= sq.len) return -1;
            const int page = table[pos / p.page_size];
            return page < 0 || page >= p.n_pages ? -1 : ((int64_t)page * p.n_kv + kvh) * p.page_size + pos % p.page_size;
        };
        int64_t pool_rows = 0;
        int to_stage = 0;
        auto load = [&](int i) {   // the warp's i-th chunk (in turn) into the next place of the ring
            if ((i & 31) == 0) pool_rows = find_row(i + lane);
            const int64_t row0 = __shfl_sync(0xFFFFFFFFu, pool_rows, i & 31);
            const int stage = to_stage;
            to_stage = stage + 1 == S::kRing ? 0 : stage + 1;
            if (lane == 0) stage_rows[stage] = row0;
            if (row0 >= 0) {
                const int left = sq.len - (chunk0 + i * kWarps) * kChunk;   // rows behind the last position come in as zeros
                const uint32_t dst = ring + stage * S::kStage;
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const uint8_t *src = (kv ? p.v : p.k) + row0 * RB;
#pragma unroll
                    for (int j = 0; j < (kChunk * RB / 16 + 31) / 32; j++) {
                        const int c = lane + 32 * j, row = c / (RB / 16), col = c % (RB / 16);
                        if (kChunk * RB / 16 % 32 == 0 || c < kChunk * RB / 16)
                            copy16(dst + kv * kChunk * RB + row * RB + ((col ^ swizzle<RB>(row)) << 4), src + 16 * c, row < left);
                    }
                }
                if constexpr (kQuant) {   // (SB 16-byte pieces of scales; those of rows behind the last position are not looked at)
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        const uint8_t *src = reinterpret_cast<const uint8_t *>(kv ? p.v_scale : p.k_scale) + row0 * SB;
                        if (lane < SB) copy16(dst + 2 * kChunk * RB + kv * kChunk * SB + 16 * lane, src + 16 * lane, true);
                    }
                }
            }
            copies_commit();
        };
#pragma unroll
        for (int i = 0; i < S::kRing - 1; i++) load(i);

        // ---- the rows' data, and the queries in two f16 terms
        float most[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            most[j] = fabsf(x[j][0]);
#pragma unroll
            for (int c = 1; c < NB; c++) most[j] = fmaxf(most[j], fabsf(x[j][c]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int j = 0; j < kPer; j++) most[j] = fmaxf(most[j], __shfl_xor_sync(0xFFFFFFFFu, most[j], o));
        int exponent = 0;   // lane j: the j-th row's
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            // the largest value comes to lie in [2^10, 2^11): the second terms' last bits are far above the f16 underflow
            const int e = most[j] > 0.0f && most[j] <= 3.4028234e38f ? 10 - max((int)(__float_as_uint(most[j]) >> 23) - 127, -110) : 0;
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            if (lane == j) exponent = e;
#pragma unroll
            for (int c = 0; c < NB; c++) {
                const int r = warp + kWarps * j, col = column_of<CT>(32 * c + lane);
                const float v = x[j][c] * up;
                const __half h = __float2half_rn(v);
                q_mem[(kPair ? 2 * r : r) * S::kPitch + col] = h;
                q_mem[(kPair ? 2 * r + 1 : R + r) * S::kPitch + col] = __float2half_rn(v - __half2float(h));
            }
        }
        if (lane < kPer) {
            const int r = warp + kWarps * lane, rr = block * R + r, i = rr / p.group;
            const bool ok = r < n_rows;
            const uint64_t mask = !ok ? 0 : p.tree ? p.tree[sq.q0 + i] : (2ull << i) - 1ull;
            Rows row;
            row.scale = ldexpf(p.scale * (p.softcap > 0.0f ? 1.0f : 1.44269504f), -exponent);
            row.first = !ok ? INT32_MAX : p.window > 0 ? sq.before + __popcll(mask) - p.window : 0;
            row.mask = mask;
            row.q_row = ok ? sq.q0 + i : -1;
            row.head = kvh * p.group + rr - i * p.group;
            row.any = 0;
            rows[r] = row;
        }
        __syncthreads();
        if constexpr (kQuant) {   // (each warp for itself: they all write the same)
            const uint64_t mask = rows[lane % R].mask;
            const uint32_t lo = __reduce_or_sync(0xFFFFFFFFu, (uint32_t)mask), hi = __reduce_or_sync(0xFFFFFFFFu, (uint32_t)(mask >> 32));
            if (lane == 0) rows[0].any = (uint64_t)hi << 32 | lo;
            __syncwarp();
        }
        // every row sees [all_from, before), none what is before any_from
        const int all_from = p.window > 0 ? sq.before + KRK_CUDA_MAX_DRAFT - p.window : 0, any_from = p.window > 0 ? sq.before - p.window : 0;

        // Sums of a lane: tile of 16 values m, tile of columns n, [2 h + c]: value value_of(m, g, h) of row 8 n + 2 t + c; with kPair row t, c the
        // term of the weight. Scores and maxima: rows 8 n + 2 t + c (row t), positions g and g + 8.
        float o[NM][NT][4], m[NT][NC], l[NT][NC], row_scale[NT][NC];
        int e_run = -24;   // (values) the power of two above the scales met so far
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int i = 0; i < NM; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[i][n][c] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                m[n][c] = -INFINITY;
                l[n][c] = 0.0f;
                row_scale[n][c] = rows[kPair ? t : 8 * n + 2 * t + c].scale;
            }
        }
        auto row_of = [&](int n, int c) -> const Rows & { return rows[kPair ? t : 8 * n + 2 * t + c]; };
        // fragments of the query of step k, tile n: first terms in [0], [1], second terms in [2], [3]; with kPair both in [0], [1]
        const uint32_t q_at = smem_addr(q_mem) + (kPair ? (lane & 7) * S::kPitch + ((lane >> 3) & 1) * 8 : ((lane & 7) + (lane >> 4) * R) * S::kPitch + ((lane >> 3) & 1) * 8) * 2;
        constexpr int kQF = kPair ? 2 : 4;
        uint32_t qf[S::kQInRegs ? NT : 1][S::kQInRegs ? NM : 1][kQF];
        auto q_load = [&](int n, int k, uint32_t (&f)[kQF]) {
            if constexpr (kPair) ldsm2(f, q_at + 32 * k);
            else ldsm4(f, q_at + 8 * n * S::kPitch * 2 + 32 * k);
        };
        if constexpr (S::kQInRegs) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < NM; k++) q_load(n, k, qf[n][k]);
        }
        auto q_frag = [&](int n, int k, uint32_t (&f)[kQF]) {
            if constexpr (S::kQInRegs) {
#pragma unroll
                for (int c = 0; c < kQF; c++) f[c] = qf[n][k][c];
            } else {
                q_load(n, k, f);
            }
        };
        // a lane's row of a matrix load: of keys (positions in eights, then pieces), of values (transposed; f16: pieces in eights of
        // values, then positions; packed: positions, then pieces)
        const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_piece = lane >> 4;
        const int v_row = kQuant ? k_row : (lane & 7) + (lane >> 4) * 8, v_piece = kQuant ? lane >> 4 : (lane >> 3) & 1;
        auto sees = [&](const Rows &r, int pos) {
            return pos < sq.len && (pos < sq.before ? pos >= r.first : ((r.mask >> (pos - sq.before)) & 1) != 0);
        };

        // (compiled for each number of tiles of columns that has rows: branches around single products cost twice the time)
        auto chunks = [&](auto na) {
            constexpr int NA = decltype(na)::value;
            int stage = 0;
            for (int i = 0; i < n_chunks; i++, stage = stage + 1 == S::kRing ? 0 : stage + 1) {
                const int pos0 = (chunk0 + i * kWarps) * kChunk;
                copies_wait<S::kRing - 2>();
                __syncwarp();
                load(i + S::kRing - 1);
                const int64_t row0 = stage_rows[stage];
                if (row0 < 0) continue;
                const uint32_t k_at = ring + stage * S::kStage, v_at = k_at + kChunk * RB;
                const uint8_t *k_mem = ring_mem + stage * S::kStage;
                const bool masked = pos0 + kChunk > min(sq.before, sq.len) || pos0 < all_from;

                // ---- scores: [n][h][c], h: position g or g + 8
                float sc[NA][2][NC];
                if constexpr (!kQuant) {
                    float sum[NA][2][4];   // first and second terms; with kPair even and odd steps
    #pragma unroll
                    for (int k = 0; k < NM; k++) {
                        uint32_t a[4];
                        ldsm4(a, k_at + k_row * RB + (((2 * k + k_piece) ^ swizzle<RB>(k_row)) << 4));
    #pragma unroll
                        for (int n = 0; n < NA; n++) {
                            uint32_t f[kQF];
                            q_frag(n, k, f);
                            if constexpr (kPair) {
                                if (k < 2) mma0(sum[n][k & 1], a, f[0], f[1]);
                                else mma(sum[n][k & 1], a, f[0], f[1]);
                            } else if (k == 0) {
                                mma0(sum[n][0], a, f[0], f[1]);
                                mma0(sum[n][1], a, f[2], f[3]);
                            } else {
                                mma(sum[n][0], a, f[0], f[1]);
                                mma(sum[n][1], a, f[2], f[3]);
                            }
                        }
                    }
                    auto second = [](float x) { return fabsf(x) <= 3.4028234e38f ? x : 0.0f; };   // (an infinite key: the first term has the sign)
    #pragma unroll
                    for (int n = 0; n < NA; n++) {
    #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            if constexpr (kPair) {
                                sc[n][h][0] = (sum[n][0][2 * h] + sum[n][1][2 * h]) + second(sum[n][0][2 * h + 1] + sum[n][1][2 * h + 1]);
                            } else {
                                sc[n][h][0] = sum[n][0][2 * h] + second(sum[n][1][2 * h]);
                                sc[n][h][1] = sum[n][0][2 * h + 1] + second(sum[n][1][2 * h + 1]);
                            }
                        }
                    }
                } else {
                    float kd[2][NB];
    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        scales<NB>(kd[h], k_mem + 2 * kChunk * RB + (g + 8 * h) * SB);
    #pragma unroll
                        for (int b = 0; b < NB; b++) kd[h][b] = fmaf(kd[h][b], 0.0f, kd[h][b]);   // (infinite: values of either sign, whose products have no sum)
                    }
    #pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t a[2][4];   // [step]: positions g and g + 8, then again
    #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int row = g + 8 * h;
                            uint32_t w[2];
                            if constexpr (CT == KRK_CUDA_KV_Q8) {
                                const uint2 u = *reinterpret_cast<const uint2 *>(k_mem + row * RB + (((2 * b + (t >> 1)) ^ swizzle<RB>(row)) << 4) + 8 * (t & 1));
                                w[0] = u.x ^ 0x80808080u, w[1] = u.y ^ 0x80808080u;
                            } else {
                                const uint32_t u = *reinterpret_cast<const uint32_t *>(k_mem + row * RB + ((b ^ swizzle<RB>(row)) << 4) + 4 * t);
                                w[0] = u & 0x0F0F0F0Fu, w[1] = (u >> 4) & 0x0F0F0F0Fu;
                            }
    #pragma unroll
                            for (int step = 0; step < 2; step++) {
                                a[step][h] = halves<0, 1>(w[step], kOff);
                                a[step][2 + h] = halves<2, 3>(w[step], kOff);
                            }
                        }
    #pragma unroll
                        for (int n = 0; n < NA; n++) {
                            float sum[4];
    #pragma unroll
                            for (int step = 0; step < 2; step++) {
                                uint32_t f[kQF];
                                q_frag(n, 2 * b + step, f);
                                if (step == 0) mma0(sum, a[step], f[0], f[1]);
                                else mma(sum, a[step], f[0], f[1]);
                                if constexpr (!kPair) mma(sum, a[step], f[2], f[3]);
                            }
    #pragma unroll
                            for (int h = 0; h < 2; h++) {
                                if constexpr (kPair) sum[2 * h] += sum[2 * h + 1];
    #pragma unroll
                                for (int c = 0; c < NC; c++) sc[n][h][c] = b == 0 ? kd[h][b] * sum[2 * h + c] : fmaf(kd[h][b], sum[2 * h + c], sc[n][h][c]);
                            }
                        }
                    }
                }
                // ---- the scales of the values, and the power of two above them
                float vd[2][NB], e_corr = 1.0f;
                if constexpr (kQuant) {
                    float own[2] = {0.0f, 0.0f};   // the greatest of a position (a NaN is none)
    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        scales<NB>(vd[h], k_mem + 2 * kChunk * RB + kChunk * SB + (g + 8 * h) * SB);
    #pragma unroll
                        for (int b = 0; b < NB; b++) own[h] = fmaxf(own[h], fabsf(vd[h][b]));
                    }
                    // What no row of the block sees does not count, nor does an infinite one that not all of them see (the values of those that do are
                    // no numbers): f16 has sixteen bits below the two terms of a weight, and a scale far above the others takes them.
                    if (masked) {
                        const uint64_t any = rows[0].any;
    #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int pos = pos0 + g + 8 * h, bit = pos - sq.before;
                            const bool counts = bit < 0 ? pos >= any_from : ((any >> (bit & 63)) & 1) != 0;
                            own[h] = counts && pos < sq.len && own[h] <= 65504.0f ? own[h] : 0.0f;
                        }
                    }
                    float most = fmaxf(own[0], own[1]);
    #pragma unroll
                    for (int o2 = 4; o2 < 32; o2 <<= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o2));
                    const int e = min(16, (int)(__float_as_uint(most) >> 23) - 126);
                    if (e > e_run) {   // (the whole warp's)
                        e_corr = __uint_as_float((uint32_t)(127 + e_run - e) << 23);
                        e_run = e;
                    }
                }

                // ---- weights. (What is rarely done has loops of its own: in one with the rest, each value's code was jumped over, and fetching
                // the instructions behind it took half of the time.)
#pragma unroll
                for (int n = 0; n < NA; n++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int c = 0; c < NC; c++) sc[n][h][c] *= row_scale[n][c];
                if (p.softcap > 0.0f) {
#pragma unroll
                    for (int n = 0; n < NA; n++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int c = 0; c < NC; c++) sc[n][h][c] = capped(sc[n][h][c], p.softcap);
                }
                if (masked) {
#pragma unroll
                    for (int n = 0; n < NA; n++)
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            const Rows &r = row_of(n, c);
#pragma unroll
                            for (int h = 0; h < 2; h++)
                                if (!sees(r, pos0 + g + 8 * h)) sc[n][h][c] = -INFINITY;
                        }
                }
                float base[NA][NC];
                bool higher = e_corr != 1.0f;
#pragma unroll
                for (int n = 0; n < NA; n++)
#pragma unroll
                    for (int c = 0; c < NC; c++) base[n][c] = fmaxf(sc[n][0][c], sc[n][1][c]);
#pragma unroll
                for (int o2 = 4; o2 < 32; o2 <<= 1)
#pragma unroll
                    for (int n = 0; n < NA; n++)
#pragma unroll
                        for (int c = 0; c < NC; c++) base[n][c] = fmaxf(base[n][c], __shfl_xor_sync(0xFFFFFFFFu, base[n][c], o2));
#pragma unroll
                for (int n = 0; n < NA; n++)
#pragma unroll
                    for (int c = 0; c < NC; c++) higher |= base[n][c] > m[n][c];
                if (__any_sync(0xFFFFFFFFu, higher)) {
#pragma unroll
                    for (int n = 0; n < NA; n++) {
                        float corr[NC];
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            const float top = fmaxf(base[n][c], m[n][c]);
                            corr[c] = top == -INFINITY ? 1.0f : ex2(m[n][c] - top);
                            m[n][c] = top;
                            l[n][c] *= corr[c];
                            corr[c] *= e_corr;
                        }
#pragma unroll
                        for (int j = 0; j < NM; j++)
#pragma unroll
                            for (int c = 0; c < 4; c++) o[j][n][c] *= corr[kPair ? 0 : c & 1];
                    }
                }
#pragma unroll
                for (int n = 0; n < NA; n++)
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        const float from = m[n][c] == -INFINITY ? 0.0f : m[n][c];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            sc[n][h][c] = ex2(sc[n][h][c] - from);
                            l[n][c] += sc[n][h][c];
                        }
                    }
                // weights w[h][c] as an operand: [first terms of positions 0 - 7, of 8 - 15, second terms]; with kPair both in [0], [1]
                auto operand = [&](const float (&w)[2][NC], uint32_t (&f)[kQF]) {
    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if constexpr (kPair) {
                            const __half hi = __float2half_rn(w[h][0]);
                            f[h] = transposed(bits(__halves2half2(hi, __float2half_rn(w[h][0] - __half2float(hi)))));
                        } else {
                            uint32_t hi, lo;
                            split(w[h][0], w[h][1], hi, lo);
                            f[h] = transposed(hi);
                            f[2 + h] = transposed(lo);
                        }
                    }
                };

                // ---- values
                if constexpr (!kQuant) {
                    // Where some rows do not see a position, one that holds an infinity or a NaN must not reach them through a product
                    // with zero: such values are taken out of the tile and added to the rows that see them one by one.
                    uint32_t odd = 0u;
                    if (masked) {
                        uint8_t *v_mem = ring_mem + stage * S::kStage + kChunk * RB;
                        for (int c = lane; c < kChunk * RB / 2; c += 32) {
                            const int row = c / (RB / 2);
                            __half *x2 = reinterpret_cast<__half *>(v_mem) + c;
                            if ((__half_as_ushort(*x2) & 0x7C00) == 0x7C00) {
                                *x2 = __float2half_rn(0.0f);
                                odd |= 1u << row;
                            }
                        }
                        odd = __reduce_or_sync(0xFFFFFFFFu, odd);
                        __syncwarp();
                    }
                    uint32_t w[NA][kQF];
    #pragma unroll
                    for (int n = 0; n < NA; n++) {
                        float up[2][NC];
    #pragma unroll
                        for (int h = 0; h < 2; h++)
    #pragma unroll
                            for (int c = 0; c < NC; c++) up[h][c] = sc[n][h][c] * 16384.0f;
                        operand(up, w[n]);
                    }
    #pragma unroll
                    for (int j = 0; j < NM; j++) {
                        uint32_t a[4];
                        ldsm4t(a, v_at + v_row * RB + (((2 * j + v_piece) ^ swizzle<RB>(v_row)) << 4));
    #pragma unroll
                        for (int n = 0; n < NA; n++) {
                            mma(o[j][n], a, w[n][0], w[n][1]);
                            if constexpr (!kPair) mma(o[j][n], a, w[n][2], w[n][3]);
                        }
                    }
                    if (odd) {
                        const __half *v_pool = reinterpret_cast<const __half *>(p.v) + row0 * D;
                        for (int j = 0; j < kChunk; j++) {
                            if (!((odd >> j) & 1)) continue;
    #pragma unroll
                            for (int n = 0; n < NA; n++)
    #pragma unroll
                                for (int c = 0; c < NC; c++) {
                                    // the weight lies with the lane of position j % 8
                                    const float x2 = __shfl_sync(0xFFFFFFFFu, j < 8 ? sc[n][0][c] : sc[n][1][c], 4 * (j & 7) + t);
                                    if (!sees(row_of(n, c), pos0 + j)) continue;
    #pragma unroll
                                    for (int k = 0; k < NM; k++)
    #pragma unroll
                                        for (int h = 0; h < 2; h++) {
                                            const float v = __half2float(v_pool[(int64_t)j * D + value_of<CT>(k, g, h)]);
                                            if (!(fabsf(v) <= 65504.0f)) o[k][n][2 * h + c] += x2 * v;
                                        }
                                }
                            __syncwarp();
                        }
                    }
                } else {
                    const float up = __uint_as_float((uint32_t)(127 + 14 - e_run) << 23);
    #pragma unroll
                    for (int b = 0; b < NB; b++) {
                        uint32_t a[2][4];   // output tiles 2 b and 2 b + 1
                        if constexpr (CT == KRK_CUDA_KV_Q8) {
                            uint32_t r[4];   // positions 0 - 7, 8 - 15 of a piece, then of the next
                            ldsm4t(r, v_at + v_row * RB + (((2 * b + v_piece) ^ swizzle<RB>(v_row)) << 4));
    #pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const uint32_t x2 = r[j] ^ 0x80808080u;
                                a[j >> 1][2 * (j & 1)] = halves<0, 2>(x2, kOff);
                                a[j >> 1][2 * (j & 1) + 1] = halves<1, 3>(x2, kOff);
                            }
                        } else {
                            uint32_t r[2];
                            ldsm2t(r, v_at + v_row * RB + ((b ^ swizzle<RB>(v_row)) << 4));
    #pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const uint32_t x2 = r[j] & 0x0F0F0F0Fu, y2 = (r[j] >> 4) & 0x0F0F0F0Fu;
                                a[0][2 * j] = halves<0, 2>(x2, kOff), a[0][2 * j + 1] = halves<1, 3>(x2, kOff);
                                a[1][2 * j] = halves<0, 2>(y2, kOff), a[1][2 * j + 1] = halves<1, 3>(y2, kOff);
                            }
                        }
                        const float d2[2] = {vd[0][b] * up, vd[1][b] * up};
    #pragma unroll
                        for (int n = 0; n < NA; n++) {
                            float w[2][NC];
                            uint32_t f[kQF];
    #pragma unroll
                            for (int h = 0; h < 2; h++)
    #pragma unroll
                                for (int c = 0; c < NC; c++) {
                                    w[h][c] = sc[n][h][c] * d2[h];
                                    if (masked && sc[n][h][c] == 0.0f) w[h][c] = 0.0f;   // (a scale that is no number stays with the rows that see it)
                                }
                            operand(w, f);
    #pragma unroll
                            for (int j = 0; j < 2; j++) {
                                mma(o[2 * b + j][n], a[j], f[0], f[1]);
                                if constexpr (!kPair) mma(o[2 * b + j][n], a[j], f[2], f[3]);
                            }
                        }
                    }
                }
            }
        };
        if (NT == 1 || n_tiles == 1) chunks(std::integral_constant<int, 1>{});
        else chunks(std::integral_constant<int, NT>{});
        copies_wait<0>();

        // ---- the warps' sums together. The outputs lie where the ring was.
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < NC; c++) {
#pragma unroll
                for (int o2 = 4; o2 < 32; o2 <<= 1) l[n][c] += __shfl_xor_sync(0xFFFFFFFFu, l[n][c], o2);
                if (g == 0) warp_ml[warp * R + (kPair ? t : 8 * n + 2 * t + c)] = make_float2(m[n][c], l[n][c]);
            }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int r = kPair ? t : 8 * n + 2 * t + c;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; w++) top = fmaxf(top, warp_ml[w * R + r].x);
                // the weights' 2^14 goes, and the values' power of two comes back
                const float f = m[n][c] == -INFINITY ? 0.0f : ex2(m[n][c] - top) * (kQuant ? exp2f((float)(e_run - 14)) : 1.0f / 16384.0f);
                float *to = sums + (warp * R + r) * S::kSumPitch;
                if (r < n_rows) {
#pragma unroll
                    for (int j = 0; j < NM; j++) {
                        float v[2];
#pragma unroll
                        for (int h = 0; h < 2; h++) v[h] = (kPair ? o[j][n][2 * h] + o[j][n][2 * h + 1] : o[j][n][2 * h + c]) * f;
                        if constexpr (kQuant) {
                            *reinterpret_cast<float2 *>(to + value_of<CT>(j, g, 0)) = make_float2(v[0], v[1]);
                        } else {
                            to[value_of<CT>(j, g, 0)] = v[0];
                            to[value_of<CT>(j, g, 1)] = v[1];
                        }
                    }
                }
            }
        __syncthreads();
        const bool whole = begins && ends;
        for (int j = tid; j < n_rows * (D / 4); j += kThreads) {
            const int r = j / (D / 4), c = 4 * (j - r * (D / 4));
            float top = -INFINITY, all = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) top = fmaxf(top, warp_ml[w * R + r].x);
            float4 x2 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float2 ml = warp_ml[w * R + r];
                if (ml.x != -INFINITY) all += ml.y * ex2(ml.x - top);
                const float4 y2 = *reinterpret_cast<const float4 *>(sums + (w * R + r) * S::kSumPitch + c);
                x2.x += y2.x, x2.y += y2.y, x2.z += y2.z, x2.w += y2.w;
            }
            if (whole) {
                float keep;
                const float f = norm_of(p, rows[r].head, top, all, keep);
                float *to = p.out + (int64_t)rows[r].q_row * p.out_stride + rows[r].head * D + c;
                *reinterpret_cast<float4 *>(to) = make_float4(x2.x * f, x2.y * f, x2.z * f, x2.w * f);
            } else {
                float *to = part_row<D, R>(p, blockIdx.x, begins ? 1 : 0, r);
                *reinterpret_cast<float2 *>(to + c) = make_float2(x2.x, x2.y);
                *reinterpret_cast<float2 *>(to + c + 2) = make_float2(x2.z, x2.w);
                if (c == 0) *reinterpret_cast<float2 *>(to + D) = make_float2(top, all);
            }
        }
        __syncthreads();
    }
}

template <int D, int CT, int R>
int launch_one(const Params &p, cudaStream_t st) {
    using S = Shape<D, CT, R>;
    static std::atomic<uint64_t> ready{0};   // devices whose limit of shared memory is raised for this kernel
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        e = cudaFuncSetAttribute(attn_kernel<D, CT, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) {
        note_cuda_error(e);
        return KRK_CUDA_ELAUNCH;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&cfg, attn_kernel<D, CT, R>, p));
}

#define KRK_ATTN_FORMS(d, r, call)                                                    \
    switch (d) {                                                                      \
    case 64: return r == 4 ? call(64, 4) : r == 8 ? call(64, 8) : call(64, 16);       \
    case 96: return r == 4 ? call(96, 4) : r == 8 ? call(96, 8) : call(96, 16);       \
    case 128: return r == 4 ? call(128, 4) : r == 8 ? call(128, 8) : call(128, 16);   \
    case 192: return r == 4 ? call(192, 4) : r == 8 ? call(192, 8) : call(192, 16);   \
    default: return r == 4 ? call(256, 4) : r == 8 ? call(256, 8) : call(256, 16);    \
    }
template <int CT>
int launch_type(const Params &p, int d, int r, cudaStream_t st) {
#define KRK_ATTN_LAUNCH(D, R) launch_one<D, CT, R>(p, st)
    KRK_ATTN_FORMS(d, r, KRK_ATTN_LAUNCH)
#undef KRK_ATTN_LAUNCH
}
}   // namespace attn
}   // namespace krk_cuda
