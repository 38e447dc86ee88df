// The kernel of krk_cuda_attention_tree, one instantiation per cache type, head size and number of row tiles.
//
// What bounds it: reading the cache, while a key head's rows are few (a decode step: one to four drafted tokens times the group);
// the tensor pipe beyond. Hence the split: a warp takes 16 positions at a time of its own (a piece of one page), copies them with
// 16-byte asynchronous copies into a ring of its own, and keeps the running maximum, sum and output of all rows of the
// block in registers; no warp waits for another one until the item's end, where the four of a CTA add up. (A page is found once
// per step; the work of a launch is dealt in equal shares, see Params.)
//
// Arithmetic. The products are `mma.sync` m16n8k16 of f16 with f32 sums. Activations are f32, so a query enters as two f16 terms
// under a power of two of its row (22 bits), and so do the weights of a step (times 2^14: terms far below the maximum keep their
// bits). Cache values enter exactly: f16 as they are; 8- and 4-bit quants as whole numbers, whose block scales multiply the f32
// sums of a block's products (keys) and the weights before they are split (values; there under the power of two of the greatest scale
// met so far, which the sums are rescaled to like to a new maximum).
#pragma once

#include <atomic>

#include "krk_attn_tree.cuh"

namespace krk_cuda {
namespace attn {

__host__ __device__ constexpr int row_bytes_of(int type, int d) { return type == KRK_CUDA_KV_F16 ? 2 * d : type == KRK_CUDA_KV_Q8 ? d : d / 2; }
__host__ __device__ constexpr int scale_bytes_of(int type, int d) { return type == KRK_CUDA_KV_F16 ? 0 : d / 16; }   // of a row

// Shared memory of a CTA: the query block, row data, the ring. As many stages as two CTAs an SM leave room for, up to six; one CTA an SM
// where that would be fewer than two.
template <int D, int CT, int MT>
struct Shape {
    static constexpr int BM = 16 * MT;
    static constexpr int RB = row_bytes_of(CT, D);
    static constexpr int SB = scale_bytes_of(CT, D);
    static constexpr int kStage = 2 * kChunk * (RB + SB);          // keys and values of a chunk, then their scales
    static constexpr int kPitch = D + 8;                           // of a query row, in halves
    static constexpr int kQ = 2 * BM * kPitch * 2;
    static constexpr int kRows = BM * 32;                          // scale, mask, window, (m, l) of the warps: see Rows
    static constexpr int kFixed = kQ + kRows + kWarps * BM * 8 + kWarps * 6 * 8;
    static constexpr int kRing2 = (112 * 1024 - kFixed) / (kWarps * kStage);
    static constexpr int kRing1 = (224 * 1024 - kFixed) / (kWarps * kStage);
    static constexpr int kCtas = kRing2 >= 2 ? 2 : 1;
    static constexpr int kRing = kCtas == 2 ? (kRing2 < 6 ? kRing2 : 6) : (kRing1 < 6 ? kRing1 : 6);
    static constexpr int kRingBytes = kWarps * kRing * kStage;
    static constexpr int kSums = kWarps * BM * (D + 8) * 4;        // the warps' outputs, in place of the ring
    static constexpr int kBytes = kFixed + (kRingBytes > kSums ? kRingBytes : kSums);
    static constexpr int kNT = D / 8;                              // 8-column tiles of the output
    static constexpr bool kQInRegs = D * MT <= 128;                // query fragments stay in registers
    static_assert(kRing >= 2, "ring");
    static_assert(kBytes <= (kCtas == 2 ? 113 : 227) * 1024, "shared memory");
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
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm2t(uint32_t r[2], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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
constexpr uint32_t kOff8 = 0x64806480u;   // 1024 + 128: signed bytes with their top bit turned over
constexpr uint32_t kOff4 = 0x64086408u;   // 1024 + 8

// The i-th of the scales of a position and the next one, NB each.
template <int NB>
__device__ __forceinline__ float scale_of(const uint32_t (&w)[NB], int i) {
    const __half2 h = half2_of(w[i >> 1]);
    return (i & 1) ? __high2float(h) : __low2float(h);
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
// The value of column `col` (0, 1: 2t + col of the fragment) of output tile n for lane t.
template <int CT>
__device__ __forceinline__ int value_of(int n, int t, int col) {
    if constexpr (CT == KRK_CUDA_KV_F16) return 8 * n + 2 * t + col;
    return 16 * (n >> 1) + 4 * t + 2 * col + (n & 1);   // even values in one tile, odd ones in the next
}

struct Rows {   // of a block of rows, in shared memory
    float scale;       // takes a row's sum of products to its score in the log2 domain (softcap: to the natural score)
    int first;         // first position before the drafted tokens that it sees
    uint64_t mask;     // drafted tokens that it sees
    int q_row, head;   // its place in q and out; -1: no row
    int pad[2];
};
static_assert(sizeof(Rows) == 32, "Shape::kRows");

template <int D, int CT, int MT>
__global__ void __launch_bounds__(kThreads, Shape<D, CT, MT>::kCtas)
attn_kernel(const __grid_constant__ Params p) {
    using S = Shape<D, CT, MT>;
    constexpr int BM = S::BM, RB = S::RB, SB = S::SB, NB = D / 32, NT = S::kNT;
    constexpr bool kQuant = CT != KRK_CUDA_KV_F16;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring_base = smem;
    float *sums = reinterpret_cast<float *>(smem);
    constexpr int kFront = S::kRingBytes > S::kSums ? S::kRingBytes : S::kSums;
    __half *q_hi = reinterpret_cast<__half *>(smem + kFront);
    __half *q_lo = q_hi + BM * S::kPitch;
    Rows *rows = reinterpret_cast<Rows *>(smem + kFront + S::kQ);
    float2 *warp_ml = reinterpret_cast<float2 *>(smem + kFront + S::kQ + S::kRows);   // [warp][BM]

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const Place place = find_place<BM>(p, blockIdx.x);
    int64_t at = place.at;
    const int64_t end = first_unit(place.total, p.grid, blockIdx.x + 1);
    if (at >= end) return;
    int s = place.seq;
    int64_t in_seq = at - place.before;
    Seq sq = sequence<BM>(p, s);
    const uint32_t ring = smem_addr(ring_base) + warp * S::kRing * S::kStage;
    uint8_t *ring_mem = ring_base + warp * S::kRing * S::kStage;
    int64_t *stage_rows = reinterpret_cast<int64_t *>(warp_ml + kWarps * BM) + warp * S::kRing;   // the pool's row that a stage begins with

    while (at < end) {
        while (in_seq >= units_of(p, sq)) {   // (sequences without drafted tokens have no units)
            in_seq -= units_of(p, sq);
            sq = sequence<BM>(p, ++s);
        }
        const int per_item = item_units(p, sq);
        const int item = (int)(in_seq / per_item), from_unit = (int)(in_seq - (int64_t)item * per_item);
        const int units = (int)min((int64_t)(per_item - from_unit), end - at);
        // units to tiles: the first kSetup units of an item stand for what it costs beside its tiles
        const int from = p.whole ? 0 : max(from_unit - kSetup, 0), upto = p.whole ? sq.tiles : from_unit + units - kSetup;
        at += units;
        in_seq += units;
        if (upto <= from) continue;
        const bool begins = from == 0, ends = upto == sq.tiles;
        const int kvh = item / sq.blocks, block = item - kvh * sq.blocks;
        const int tile0 = sq.tile0 + from, tile1 = sq.tile0 + upto;
        const int n_rows = min(BM, sq.n_q * p.group - block * BM);
        const bool two = MT == 2 && n_rows > 16;

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
        auto load = [&](int i) {   // the warp's i-th chunk (in turn) into its place of the ring
            if ((i & 31) == 0) pool_rows = find_row(i + lane);
            const int64_t row0 = __shfl_sync(0xFFFFFFFFu, pool_rows, i & 31);
            const int stage = i % S::kRing;
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

        // ---- the block's rows: data, and queries in two f16 terms. A warp takes rows in turn; all its rows' loads go out first.
        constexpr int kPer = BM / kWarps;
        float x[kPer][NB];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const int r = warp + kWarps * j, rr = block * BM + r, i = rr / p.group;
            const float *from = p.q + (int64_t)(sq.q0 + i) * p.q_stride + (kvh * p.group + rr - i * p.group) * D + lane;
#pragma unroll
            for (int c = 0; c < NB; c++) x[j][c] = r < n_rows ? from[32 * c] : 0.0f;
        }
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
                const int at_c = (warp + kWarps * j) * S::kPitch + column_of<CT>(32 * c + lane);
                const float v = x[j][c] * up;
                const __half h = __float2half_rn(v);
                q_hi[at_c] = h;
                q_lo[at_c] = __float2half_rn(v - __half2float(h));
            }
        }
        if (lane < kPer) {
            const int r = warp + kWarps * lane, rr = block * BM + r, i = rr / p.group;
            const bool ok = r < n_rows;
            const uint64_t mask = !ok ? 0 : p.tree ? p.tree[sq.q0 + i] : (2ull << i) - 1ull;
            Rows row;
            row.scale = ldexpf(p.scale * (p.softcap > 0.0f ? 1.0f : 1.44269504f), -exponent);
            row.first = !ok ? INT32_MAX : p.window > 0 ? sq.before + __popcll(mask) - p.window : 0;
            row.mask = mask;
            row.q_row = ok ? sq.q0 + i : -1;
            row.head = kvh * p.group + rr - i * p.group;
            row.pad[0] = row.pad[1] = 0;
            rows[r] = row;
        }
        __syncthreads();
        // every row sees [all_from, before), none what is before any_from
        const int all_from = p.window > 0 ? sq.before + KRK_CUDA_MAX_DRAFT - p.window : 0, any_from = p.window > 0 ? sq.before - p.window : 0;

        float o[MT][NT][4], m[MT][2], l[MT][2];
        int e_run = -24;   // (values) the power of two above the scales met so far
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[mt][n][c] = 0.0f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.0f;
        }
        // fragments of the query: rows 16 mt + (0..15), columns 16 k + (0..15)
        const uint32_t q_at = (uint32_t)(((lane & 15) * S::kPitch + (lane >> 4) * 8) * 2);
        const uint32_t q_hi_at = smem_addr(q_hi) + q_at, q_lo_at = smem_addr(q_lo) + q_at;
        uint32_t qf[S::kQInRegs ? MT : 1][S::kQInRegs ? D / 16 : 1][2][4];
        if constexpr (S::kQInRegs) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    ldsm4(qf[mt][k][0], q_hi_at + (mt * 16 * S::kPitch + 16 * k) * 2);
                    ldsm4(qf[mt][k][1], q_lo_at + (mt * 16 * S::kPitch + 16 * k) * 2);
                }
        }
        auto q_frag = [&](int mt, int k, uint32_t hi[4], uint32_t lo[4]) {
            if constexpr (S::kQInRegs) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    hi[c] = qf[mt][k][0][c];
                    lo[c] = qf[mt][k][1][c];
                }
            } else {
                ldsm4(hi, q_hi_at + (mt * 16 * S::kPitch + 16 * k) * 2);
                ldsm4(lo, q_lo_at + (mt * 16 * S::kPitch + 16 * k) * 2);
            }
        };
        // a lane's row of a matrix load: of keys (16 positions x 16 columns), of values (16 positions x two pieces)
        const int k_row = (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
        const int v_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_piece = lane >> 4;

        float row_scale[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            row_scale[mt][0] = rows[16 * mt + g].scale;
            row_scale[mt][1] = rows[16 * mt + g + 8].scale;
        }
        auto sees = [&](const Rows &r, int pos) {
            return pos < sq.before ? pos >= r.first : pos < sq.len && ((r.mask >> (pos - sq.before)) & 1) != 0;
        };

        for (int i = 0; i < n_chunks; i++) {
            const int pos0 = (chunk0 + i * kWarps) * kChunk;
            copies_wait<S::kRing - 2>();
            __syncwarp();
            load(i + S::kRing - 1);
            const int stage = i % S::kRing;
            const int64_t row0 = stage_rows[stage];
            if (row0 < 0) continue;
            const uint32_t k_at = ring + stage * S::kStage, v_at = k_at + kChunk * RB;
            const uint8_t *k_mem = ring_mem + stage * S::kStage;
            const bool masked = pos0 + kChunk > sq.before || pos0 < all_from;

            // ---- scores
            float sc[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) sc[mt][n][c] = 0.0f;
            if constexpr (!kQuant) {
                float lo_sum[MT][2][4] = {};
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    uint32_t b[4], hi[4], lo[4];
                    ldsm4(b, k_at + k_row * RB + (((2 * k + k_piece) ^ swizzle<RB>(k_row)) << 4));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (mt == 1 && !two) continue;
                        q_frag(mt, k, hi, lo);
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            mma(sc[mt][n], hi, b[2 * n], b[2 * n + 1]);
                            mma(lo_sum[mt][n], lo, b[2 * n], b[2 * n + 1]);
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++)   // (an infinite key: the first term has the sign)
                            sc[mt][n][c] += fabsf(lo_sum[mt][n][c]) <= 3.4028234e38f ? lo_sum[mt][n][c] : 0.0f;
            } else {
                // scales of positions 8 n + 2 t and the next one, NB each
                uint32_t kd[2][NB];
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int j = 0; j < NB; j++) kd[n][j] = *reinterpret_cast<const uint32_t *>(k_mem + 2 * kChunk * RB + 4 * (NB * (4 * n + t) + j));
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t kb[2][2][2];   // [n][step][register]
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const int row = 8 * n + g;
                        if constexpr (CT == KRK_CUDA_KV_Q8) {
                            const uint2 w = *reinterpret_cast<const uint2 *>(k_mem + row * RB + (((2 * b + (t >> 1)) ^ swizzle<RB>(row)) << 4) + 8 * (t & 1));
                            const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
                            kb[n][0][0] = halves<0, 1>(x, kOff8), kb[n][0][1] = halves<2, 3>(x, kOff8);
                            kb[n][1][0] = halves<0, 1>(y, kOff8), kb[n][1][1] = halves<2, 3>(y, kOff8);
                        } else {
                            const uint32_t w = *reinterpret_cast<const uint32_t *>(k_mem + row * RB + ((b ^ swizzle<RB>(row)) << 4) + 4 * t);
                            const uint32_t x = w & 0x0F0F0F0Fu, y = (w >> 4) & 0x0F0F0F0Fu;
                            kb[n][0][0] = halves<0, 1>(x, kOff4), kb[n][0][1] = halves<2, 3>(x, kOff4);
                            kb[n][1][0] = halves<0, 1>(y, kOff4), kb[n][1][1] = halves<2, 3>(y, kOff4);
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (mt == 1 && !two) continue;
                        float sum[2][4] = {}, lo_sum[2][4] = {};
#pragma unroll
                        for (int step = 0; step < 2; step++) {
                            uint32_t hi[4], lo[4];
                            q_frag(mt, 2 * b + step, hi, lo);
#pragma unroll
                            for (int n = 0; n < 2; n++) {
                                mma(sum[n], hi, kb[n][step][0], kb[n][step][1]);
                                mma(lo_sum[n], lo, kb[n][step][0], kb[n][step][1]);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            // (an infinite scale: values of either sign, whose products have no sum; infinity times zero is NaN)
                            const float e0 = scale_of<NB>(kd[n], b), e1 = scale_of<NB>(kd[n], NB + b), d0 = fmaf(e0, 0.0f, e0), d1 = fmaf(e1, 0.0f, e1);
                            sc[mt][n][0] += d0 * (sum[n][0] + lo_sum[n][0]);
                            sc[mt][n][1] += d1 * (sum[n][1] + lo_sum[n][1]);
                            sc[mt][n][2] += d0 * (sum[n][2] + lo_sum[n][2]);
                            sc[mt][n][3] += d1 * (sum[n][3] + lo_sum[n][3]);
                        }
                    }
                }
            }
            // ---- the scales of the values, and the power of two above them
            uint32_t vd[2][NB];
            float e_corr = 1.0f;
            if constexpr (kQuant) {
                float most = 0.0f;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        vd[n][j] = *reinterpret_cast<const uint32_t *>(k_mem + 2 * kChunk * RB + kChunk * SB + 4 * (NB * (4 * n + t) + j));
                        const float2 f = __half22float2(half2_of(vd[n][j]));
                        const int in_x = pos0 + 8 * n + 2 * t + (2 * j) / NB, in_y = pos0 + 8 * n + 2 * t + (2 * j + 1) / NB;
                        if (in_x >= any_from && in_x < sq.len) most = fmaxf(most, fabsf(f.x));   // (a NaN is no maximum)
                        if (in_y >= any_from && in_y < sq.len) most = fmaxf(most, fabsf(f.y));
                    }
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
                const int e = min(16, (int)(__float_as_uint(most) >> 23) - 126);
                if (e > e_run) {   // (the whole warp's: every four lanes have all positions)
                    e_corr = __uint_as_float((uint32_t)(127 + e_run - e) << 23);
                    e_run = e;
                }
            }

            // ---- weights
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                if (mt == 1 && !two) continue;
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        float x = sc[mt][n][c] * row_scale[mt][c >> 1];
                        if (p.softcap > 0.0f) x = p.softcap * 1.44269504f * tanhf(x / p.softcap);
                        sc[mt][n][c] = x;
                    }
                if (masked) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const Rows &r = rows[16 * mt + g + 8 * h];
#pragma unroll
                        for (int n = 0; n < 2; n++)
#pragma unroll
                            for (int c = 0; c < 2; c++)
                                if (!sees(r, pos0 + 8 * n + 2 * t + c)) sc[mt][n][2 * h + c] = -INFINITY;
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) top[c >> 1] = fmaxf(top[c >> 1], sc[mt][n][c]);
                float base[2], corr[2];
                bool higher = e_corr != 1.0f;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2));
                    top[h] = fmaxf(top[h], m[mt][h]);
                    higher |= top[h] > m[mt][h];
                    base[h] = top[h] == -INFINITY ? 0.0f : top[h];
                    corr[h] = ex2(m[mt][h] - base[h]);
                    m[mt][h] = top[h];
                }
                if (__any_sync(0xFFFFFFFFu, higher)) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        l[mt][h] *= corr[h];
                        corr[h] *= e_corr;
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) o[mt][n][c] *= corr[c >> 1];
                }
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        sc[mt][n][c] = ex2(sc[mt][n][c] - base[c >> 1]);
                        l[mt][c >> 1] += sc[mt][n][c];
                    }
            }

            // ---- values
            if constexpr (!kQuant) {
                // Where some rows do not see a position, one that holds an infinity or a NaN must not reach them through a product
                // with zero: such values are taken out of the tile and added to the rows that see them one by one.
                uint32_t odd = 0u;
                if (masked) {
                    uint8_t *v_mem = ring_mem + stage * S::kStage + kChunk * RB;
                    for (int c = lane; c < kChunk * RB / 2; c += 32) {
                        const int row = c / (RB / 2);
                        __half *h = reinterpret_cast<__half *>(v_mem) + c;
                        if ((__half_as_ushort(*h) & 0x7C00) == 0x7C00) {
                            *h = __float2half_rn(0.0f);
                            odd |= 1u << row;
                        }
                    }
                    odd = __reduce_or_sync(0xFFFFFFFFu, odd);
                    __syncwarp();
                }
                uint32_t w_hi[MT][4], w_lo[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int r = 0; r < 4; r++)   // rows g, g + 8 of positions 2t.., then of positions 2t + 8..
                        split(sc[mt][r >> 1][2 * (r & 1)] * 16384.0f, sc[mt][r >> 1][2 * (r & 1) + 1] * 16384.0f, w_hi[mt][r], w_lo[mt][r]);
#pragma unroll
                for (int j = 0; j < NT / 2; j++) {
                    uint32_t b[4];
                    ldsm4t(b, v_at + v_row * RB + (((2 * j + v_piece) ^ swizzle<RB>(v_row)) << 4));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (mt == 1 && !two) continue;
                        mma(o[mt][2 * j], w_hi[mt], b[0], b[1]);
                        mma(o[mt][2 * j + 1], w_hi[mt], b[2], b[3]);
                        mma(o[mt][2 * j], w_lo[mt], b[0], b[1]);
                        mma(o[mt][2 * j + 1], w_lo[mt], b[2], b[3]);
                    }
                }
                if (odd) {
                    const __half *v_pool = reinterpret_cast<const __half *>(p.v) + row0 * D;
                    for (int j = 0; j < kChunk; j++) {
                        if (!((odd >> j) & 1)) continue;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                // the weight lies with lane 4 g + (j % 8) / 2
                                const float even = j < 8 ? sc[mt][0][2 * h] : sc[mt][1][2 * h], uneven = j < 8 ? sc[mt][0][2 * h + 1] : sc[mt][1][2 * h + 1];
                                const float w = __shfl_sync(0xFFFFFFFFu, (j & 1) ? uneven : even, 4 * g + ((j & 7) >> 1));
                                if (!sees(rows[16 * mt + g + 8 * h], pos0 + j)) continue;
#pragma unroll
                                for (int n = 0; n < NT; n++)
#pragma unroll
                                    for (int c = 0; c < 2; c++) {
                                        const float v = __half2float(v_pool[(int64_t)j * D + value_of<CT>(n, t, c)]);
                                        if (!(fabsf(v) <= 65504.0f)) o[mt][n][2 * h + c] += w * v;
                                    }
                            }
                        __syncwarp();
                    }
                }
            } else {
                const float up = __uint_as_float((uint32_t)(127 + 14 - e_run) << 23);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t w_hi[MT][4], w_lo[MT][4];
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float d0 = scale_of<NB>(vd[n], b) * up, d1 = scale_of<NB>(vd[n], NB + b) * up;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const float p0 = sc[mt][n][2 * h], p1 = sc[mt][n][2 * h + 1];
                                float w0 = p0 * d0, w1 = p1 * d1;
                                if (masked) {   // (a scale that is no number stays with the rows that see it)
                                    if (p0 == 0.0f) w0 = 0.0f;
                                    if (p1 == 0.0f) w1 = 0.0f;
                                }
                                split(w0, w1, w_hi[mt][2 * n + h], w_lo[mt][2 * n + h]);
                            }
                    }
                    uint32_t vb[4][2];   // output tiles 4 b .. 4 b + 3
                    if constexpr (CT == KRK_CUDA_KV_Q8) {
                        uint32_t r[4];
                        ldsm4t(r, v_at + v_row * RB + (((2 * b + v_piece) ^ swizzle<RB>(v_row)) << 4));
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint32_t x = r[j] ^ 0x80808080u;
                            vb[2 * (j >> 1)][j & 1] = halves<0, 2>(x, kOff8);
                            vb[2 * (j >> 1) + 1][j & 1] = halves<1, 3>(x, kOff8);
                        }
                    } else {
                        uint32_t r[2];
                        ldsm2t(r, v_at + v_row * RB + ((b ^ swizzle<RB>(v_row)) << 4));
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const uint32_t x = r[j] & 0x0F0F0F0Fu, y = (r[j] >> 4) & 0x0F0F0F0Fu;
                            vb[0][j] = halves<0, 2>(x, kOff4), vb[1][j] = halves<1, 3>(x, kOff4);
                            vb[2][j] = halves<0, 2>(y, kOff4), vb[3][j] = halves<1, 3>(y, kOff4);
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        if (mt == 1 && !two) continue;
#pragma unroll
                        for (int j = 0; j < 4; j++) mma(o[mt][4 * b + j], w_hi[mt], vb[j][0], vb[j][1]);
#pragma unroll
                        for (int j = 0; j < 4; j++) mma(o[mt][4 * b + j], w_lo[mt], vb[j][0], vb[j][1]);
                    }
                }
            }
        }
        copies_wait<0>();

        // ---- the warps' sums together. The outputs lie where the ring was.
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 1);
                l[mt][h] += __shfl_xor_sync(0xFFFFFFFFu, l[mt][h], 2);
                if (t == 0) warp_ml[warp * BM + 16 * mt + g + 8 * h] = make_float2(m[mt][h], l[mt][h]);
            }
        __syncthreads();
        constexpr int kSumPitch = D + 8;
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 16 * mt + g + 8 * h;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; w++) top = fmaxf(top, warp_ml[w * BM + r].x);
                // the weights' 2^14 goes, and the values' power of two comes back
                const float f = m[mt][h] == -INFINITY ? 0.0f : ex2(m[mt][h] - top) * (kQuant ? exp2f((float)(e_run - 14)) : 1.0f / 16384.0f);
                float *to = sums + (size_t)(warp * BM + r) * kSumPitch;
                if (r < n_rows)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 2; c++) to[value_of<CT>(n, t, c)] = o[mt][n][2 * h + c] * f;
            }
        __syncthreads();
        const bool whole = begins && ends;
        for (int j = tid; j < n_rows * (D / 4); j += kThreads) {
            const int r = j / (D / 4), c = 4 * (j - r * (D / 4));
            float top = -INFINITY, all = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) top = fmaxf(top, warp_ml[w * BM + r].x);
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float2 ml = warp_ml[w * BM + r];
                if (ml.x != -INFINITY) all += ml.y * ex2(ml.x - top);
                const float4 y = *reinterpret_cast<const float4 *>(sums + (size_t)(w * BM + r) * kSumPitch + c);
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            if (whole) {
                float keep;
                const float f = norm_of(p, rows[r].head, top, all, keep);
                float *to = p.out + (int64_t)rows[r].q_row * p.out_stride + rows[r].head * D + c;
                *reinterpret_cast<float4 *>(to) = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
            } else {
                float *to = part_row<D, BM>(p, blockIdx.x, begins ? 1 : 0, r);
                *reinterpret_cast<float2 *>(to + c) = make_float2(x.x, x.y);
                *reinterpret_cast<float2 *>(to + c + 2) = make_float2(x.z, x.w);
                if (c == 0) *reinterpret_cast<float2 *>(to + D) = make_float2(top, all);
            }
        }
        __syncthreads();
    }
}

template <int D, int CT, int MT>
int launch_one(const Params &p, cudaStream_t st) {
    using S = Shape<D, CT, MT>;
    static std::atomic<uint64_t> ready{0};   // devices whose limit of shared memory is raised for this kernel
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        e = cudaFuncSetAttribute(attn_kernel<D, CT, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
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
    return launched(cudaLaunchKernelEx(&cfg, attn_kernel<D, CT, MT>, p));
}

// Two row tiles up to heads of 128 values: their outputs take 128 registers of a lane.
template <int CT>
int launch_type(const Params &p, int d, int mt, cudaStream_t st) {
    switch (d) {
    case 64: return mt == 2 ? launch_one<64, CT, 2>(p, st) : launch_one<64, CT, 1>(p, st);
    case 96: return mt == 2 ? launch_one<96, CT, 2>(p, st) : launch_one<96, CT, 1>(p, st);
    case 128: return mt == 2 ? launch_one<128, CT, 2>(p, st) : launch_one<128, CT, 1>(p, st);
    case 192: return launch_one<192, CT, 1>(p, st);
    case 256: return launch_one<256, CT, 1>(p, st);
    default: return KRK_CUDA_ESHAPE;
    }
}
template <int CT>
constexpr int ctas_of(int d, int mt) {
    return d == 64 ? (mt == 2 ? Shape<64, CT, 2>::kCtas : Shape<64, CT, 1>::kCtas) : d == 96 ? (mt == 2 ? Shape<96, CT, 2>::kCtas : Shape<96, CT, 1>::kCtas)
           : d == 128 ? (mt == 2 ? Shape<128, CT, 2>::kCtas : Shape<128, CT, 1>::kCtas) : d == 192 ? Shape<192, CT, 1>::kCtas : Shape<256, CT, 1>::kCtas;
}

}   // namespace attn
}   // namespace krk_cuda
