// krk_cuda_attention_tree for many rows to a key head (a tree of drafted tokens times the group): the products on tcgen05.
//
// A block of up to 64 rows, a tile of 128 positions. S^T = K Q^T has the positions as the 128 lanes of tensor memory and the rows as
// columns, so that a thread of the softmax has a position and every one has work however few the rows are; O^T = V^T P^T has
// the values as lanes. Both operands come from shared memory in the 128-byte swizzle: keys as rows of values (K-major), values as
// the same rows read across (MN-major), weights as [position][row] (MN-major). As in krk_attn_kernel.cuh, queries and weights
// enter as two f16 terms each: the second terms are columns behind the first ones of one product, so that the 128-row operand is read once.
//
// What bounds it: with 64 rows a product has 128 columns, 64 clocks for 16 values of 128 positions, as the reading of its operands out of
// shared memory takes: 8 clocks a position in all, against 22 for its bytes out of HBM (f16, 128 values; mma.sync: 128 clocks); the softmax, whose
// phases wait for each other, is what it runs at. (Terms as products in a row, 64 columns each: shared memory was busy twice as long.) It
// has its maxima across threads: a reference m stands until a score is more than 4 (log2) above it (a weight is
// at most 2^4, times 2^11 it is below the f16 range), which a vote finds; only then are columns reduced and sums rescaled.
//
// Warps 0 - 15: softmax, four groups that have 16 columns each; 16 - 18: copies of keys and values into a ring of half tiles (16 bytes
// a lane, asynchronous); 19: issue of the products. (Two groups with 32 columns each: an item cost 17 us beside its tiles instead of 11, for
// its phases wait for each other.) Four sequences of up to 16,384 positions and 64 drafted
// tokens, 32 heads of 128 values on 8: 119 us (both forms side by side: form_of in krk_attn_tree.cu); 8.6e-7 off 64 bits, relative, where f32 products
// with blocked sums are 4.5e-7 off: a sum in tensor memory goes through all positions of its item. Waits are bounded as in krk_gemm_tc.cu: one that gives up raises the status word, and
// the CTA runs to its end without waiting again, lets the products that it issued finish (bounded too) and frees its tensor memory. What is
// in shared memory may be anything by then: the softmax's barriers, which have no bound, are met on the sequences' lengths alone, by all of
// its threads, and what is found in a tile decides on no address that is not checked.
#pragma once

#include "krk_attn_kernel.cuh"

namespace krk_cuda {
namespace attn {

constexpr int kSoftWarps = 16, kCopyWarps = 3, kWideThreads = 32 * (kSoftWarps + kCopyWarps + 1);
constexpr int kSoftThreads = 32 * kSoftWarps;
constexpr int kSlots = 4;                       // half tiles (keys, values in turn) in shared memory
constexpr uint32_t kTmemCols = 512, kTmemO = 256;   // scores at 0 and 128, outputs at 256
constexpr float kHeadroom = 4.0f;               // log2: scores stay below m + this
constexpr float kWeightUp = 2048.0f;            // 2^11: weights in two f16 terms
constexpr long long kWaitLimit = 4000000000ll;  // clocks

template <int D>
struct Wide {
    static constexpr int kCols = (D + 63) / 64;                 // column blocks of 64 values
    static constexpr int kHalf = kCols * kWideTile * 128;       // bytes of a half tile
    static constexpr int kQBlock = 2 * kWideRows * 128;         // of 64 values of the queries, both terms
    static constexpr int kQ = kSlots * kHalf;                   // offsets
    static constexpr int kP = kQ + kCols * kQBlock;
    static constexpr int kMeta = kP + 2 * kWideTile * 128;
    static constexpr int kBytes = kMeta + 8 * 1024;
    static_assert(kBytes + 1024 <= 227 * 1024, "shared memory");
};

// Which of a group's columns see a thread's position: bit j for column c0 + j. (Out of line: its registers are not the main path's.)
static __device__ __noinline__ uint32_t seen_of(const Rows *rows, int c0, int pos, int before, int len) {
    // the word that decides is at the same place of each row: its first position, or half of its mask
    const bool earlier = pos < before;
    const int bit = pos - before, at = earlier ? (int)offsetof(Rows, first) : (int)offsetof(Rows, mask) + 4 * ((bit >> 5) & 1);
    const uint8_t *from = reinterpret_cast<const uint8_t *>(rows + c0) + at;
    uint32_t seen = 0;
#pragma unroll 8
    for (int j = 0; j < 16; j++) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(from + j * sizeof(Rows));
        seen |= (earlier ? (uint32_t)(pos >= (int)w) : (w >> (bit & 31)) & 1u) << j;
    }
    return pos < len ? seen : 0u;
}

struct WideMeta {
    unsigned long long kv_full[kSlots], kv_empty[kSlots], s_full[2], s_empty[2], q_full, p_full, pv_done, drained;
    alignas(16) Rows rows[kWideRows];
    // of columns, read four at a time: a score's log2 is product * scale; base: less the reference m (the weights' 2^11 in it took three bits of the greatest ones)
    alignas(16) float scale[kWideRows];
    alignas(16) float one[kWideRows];
    alignas(16) float base[kWideRows];
    float corr[kWideRows], more[kWideRows];   // a new reference: factor of the sums, difference of the bases
    float m[kWideRows];
    float *to[kWideRows];         // where a row's outputs go
    float red[4][kWideRows];
    unsigned long long ok[kSlots];   // byte c: chunk c of the half tile (values) is there
    uint32_t odd[4];              // positions of the tile that have a value which is no number
    Walk<kWideRows> walk;         // the softmax's: in registers it made them spill
    int goes_on;
    uint32_t tmem;
    int gave_up;
};
static_assert(sizeof(WideMeta) <= 8 * 1024, "Wide::kMeta");

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Without waiting (a try waits for a while, which would keep back what others wait for).
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
static __device__ __noinline__ void bar_wait_long(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status) {
    const long long t0 = clock64();
    for (;;) {
        for (int i = 0; i < 32; i++) {
            if (bar_try(bar, parity)) return;
            __nanosleep(32);
        }
        if (*gave_up) return;
        if (clock64() - t0 > kWaitLimit) {
            *gave_up = 1;
            atomicExch(status, KRK_CUDA_ETIMEOUT);
            return;
        }
    }
}
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status) {
    if (bar_try(bar, parity)) return;
    if (*gave_up) return;
    bar_wait_long(bar, parity, gave_up, status);
}
// The products in flight of a CTA that has given up.
static __device__ __noinline__ void bar_wait_drained(uint32_t bar) {
    const long long t0 = clock64();
    while (!bar_try(bar, 0) && clock64() - t0 <= kWaitLimit) __nanosleep(32);
}
// The 128 threads of a group of softmax warps: meet, and learn whether any of them says so. All groups: meet.
__device__ __forceinline__ bool group_any(int group, bool mine) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 q, %1, 0;\n barrier.cta.red.or.pred p, %2, 128, q;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r) : "r"((uint32_t)mine), "r"(1 + group) : "memory");
    return r != 0;
}
__device__ __forceinline__ void group_sync(int group) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + group) : "memory"); }
__device__ __forceinline__ bool soft_any(bool mine) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 q, %1, 0;\n barrier.cta.red.or.pred p, 5, %2, q;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r) : "r"((uint32_t)mine), "n"(kSoftThreads) : "memory");
    return r != 0;
}
__device__ __forceinline__ void soft_sync() { asm volatile("barrier.cta.sync 5, %0;" ::"n"(kSoftThreads) : "memory"); }
// 16 values of each of 32 lanes: op of the lanes' values i goes to lanes i and i + 16 (31 exchanges; a value at a time 80).
template <class Op>
__device__ __forceinline__ float across(float (&v)[16], Op &&op) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = op(v[i], __shfl_xor_sync(0xFFFFFFFFu, v[i], 16));
#pragma unroll
    for (int s = 8; s > 0; s >>= 1)
#pragma unroll
        for (int i = 0; i < s; i++) {
            const bool up = lane & s;
            const float mine = up ? v[i + s] : v[i], other = up ? v[i] : v[i + s];
            v[i] = op(mine, __shfl_xor_sync(0xFFFFFFFFu, other, s));
        }
    return v[0];
}
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint32_t elected_lane() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
    return e;
}
// D[tmem] (+)= A B, both in shared memory. Executed by a converged warp with uniform operands, issued by the elected lane.
__device__ __forceinline__ void product(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t onto, uint32_t elected) {
    asm volatile("{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 q, %8, 0;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, {%7, %7, %7, %7}, p;\n}\n"
                 ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(onto), "r"(0u), "r"(elected) : "memory");
}
__device__ __forceinline__ void products_commit(uint32_t bar, uint32_t elected) {
    asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(elected) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
                   "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptors of 128-byte-swizzle tiles (rows of 128 bytes, eight rows an atom): address >> 4, leading offset >> 4 in bits 16 - 29, stride offset >> 4
// in bits 32 - 45, version 1, layout 2. K-major: stride = atoms of eight rows apart. MN-major: stride = groups of eight k apart, leading =
// groups of 64 m or n apart.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) { return ((addr & 0x3FFFFu) >> 4) | (lead >> 4) << 16; }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// D f32, A and B f16, M = 128; bit 15, 16: A, B MN-major
__device__ __forceinline__ uint32_t wide_idesc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (uint32_t)a_mn << 15 | (uint32_t)b_mn << 16 | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}

template <int D>
__global__ void __launch_bounds__(kWideThreads, 1)
attn_wide_kernel(const __grid_constant__ Params p) {
    using W = Wide<D>;
    constexpr int CT = KRK_CUDA_KV_F16, NB = D / 32, RB = 2 * D;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_addr(smem);
    WideMeta &meta = *reinterpret_cast<WideMeta *>(smem + W::kMeta);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int *gave_up = &meta.gave_up;
    auto bar = [&](unsigned long long &b) { return smem_addr(&b); };

    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < kSlots; i++) {
                bar_init(bar(meta.kv_full[i]), kCopyWarps);
                bar_init(bar(meta.kv_empty[i]), 1);
            }
            for (int i = 0; i < 2; i++) {
                bar_init(bar(meta.s_full[i]), 1);
                bar_init(bar(meta.s_empty[i]), kSoftWarps);
            }
            bar_init(bar(meta.q_full), kSoftWarps);
            bar_init(bar(meta.p_full), kSoftWarps);
            bar_init(bar(meta.pv_done), 1);
            bar_init(bar(meta.drained), 1);
            meta.gave_up = 0;
        }
        __syncwarp();
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        async_fence();
    }
    if (warp == kSoftWarps + kCopyWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&meta.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Walk<kWideRows> walk;
    walk.start(p);   // (its barriers publish those above)
    if (!p.whole && tid == 0) p.shared[blockIdx.x].parts = 0;
    if (tid == 0) meta.walk = walk;
    __syncthreads();
    tc_after();
    const uint32_t tmem = meta.tmem;

    if (warp < kSoftWarps) {
        // ===== softmax: thread = lane of tensor memory, 16 columns
        const int group = warp >> 2, lanes = warp & 3, place_in = 32 * lanes + lane;
        const uint32_t t_lane = tmem + ((uint32_t)(32 * lanes) << 16), c0 = 16 * group;   // its columns: c0 .. c0 + 15
        const uint32_t col = (uint32_t)c0;
        uint32_t n_tile = 0;      // tiles so far: phases of scores, weights and products
        int n_half = 0;           // half tiles before this item
        for (;;) {
            if (tid == 0) {
                Walk<kWideRows> w = meta.walk;
                meta.goes_on = w.next(p);
                if (meta.goes_on && w.parts > 0) w.note(p);
                meta.walk = w;
            }
            soft_sync();
            if (!meta.goes_on) break;
            const volatile Walk<kWideRows> &walk = meta.walk;
            const volatile Seq &sq = walk.sq;
            const int n_rows = walk.n_rows, tiles = walk.tiles, before = sq.before, n_cols = (n_rows + 15) / 16 * 16;
            const bool has = c0 < n_cols;
            // ---- queries in two f16 terms; a warp takes rows in turn, four at a time
#pragma unroll 1
            for (int r0 = warp; r0 < n_cols; r0 += 4 * kSoftWarps) {
                float x[4][NB], most[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int r = r0 + j * kSoftWarps, rr = walk.block * kWideRows + r, i = rr / p.group;
                    const float *from = p.q + (int64_t)(sq.q0 + i) * p.q_stride + (walk.kvh * p.group + rr - i * p.group) * D + lane;
#pragma unroll
                    for (int c = 0; c < NB; c++) x[j][c] = r < n_rows ? from[32 * c] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    most[j] = fabsf(x[j][0]);
#pragma unroll
                    for (int c = 1; c < NB; c++) most[j] = fmaxf(most[j], fabsf(x[j][c]));
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                    for (int j = 0; j < 4; j++) most[j] = fmaxf(most[j], __shfl_xor_sync(0xFFFFFFFFu, most[j], o));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int r = r0 + j * kSoftWarps;
                    if (r >= n_cols) continue;
                    const int e = most[j] > 0.0f && most[j] <= 3.4028234e38f ? 10 - max((int)(__float_as_uint(most[j]) >> 23) - 127, -110) : 0;
                    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                    for (int c = 0; c < NB; c++) {
                        const int d = 32 * c + lane;
                        const float v = x[j][c] * up;
                        const __half h = __float2half_rn(v);
                        // (second terms n_cols rows on, a multiple of eight: the same swizzle)
                        uint8_t *to = smem + W::kQ + (d >> 6) * W::kQBlock + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + 2 * (d & 7);
                        *reinterpret_cast<__half *>(to) = h;
                        *reinterpret_cast<__half *>(to + n_cols * 128) = __float2half_rn(v - __half2float(h));
                    }
                    if (lane == 0) meta.scale[r] = p.scale * (p.softcap > 0.0f ? 1.0f : 1.44269504f) * __uint_as_float((uint32_t)(127 - e) << 23);
                }
            }
            if (tid < n_cols) {
                const int r = tid, rr = walk.block * kWideRows + r, i = rr / p.group;
                const bool ok = r < n_rows;
                const uint64_t mask = !ok ? 0 : p.tree ? p.tree[sq.q0 + i] : (2ull << i) - 1ull;
                Rows row;
                row.scale = 0.0f;
                row.first = !ok ? INT32_MAX : p.window > 0 ? sq.before + __popcll(mask) - p.window : 0;
                row.mask = mask;
                row.q_row = ok ? sq.q0 + i : -1;
                row.head = walk.kvh * p.group + rr - i * p.group;
                row.any = 0;
                meta.rows[r] = row;
                meta.one[r] = 1.0f;
                meta.m[r] = -INFINITY;
                meta.base[r] = 0.0f;
                meta.to[r] = walk.begins && walk.ends ? p.out + (int64_t)row.q_row * p.out_stride + row.head * D : part_row<D, kWideRows>(p, blockIdx.x, walk.begins ? 1 : 0, r);
            }
            async_fence();
            soft_sync();
            if (lane == 0) bar_arrive(bar(meta.q_full));
            const int all_from = p.window > 0 ? before + KRK_CUDA_MAX_DRAFT - p.window : 0;
            // weights [position][column, second terms n_cols on], 64 columns a block
            auto weight_at = [&](int position, int c) { return smem + W::kP + (c >> 6) * (kWideTile * 128) + position * 128 + ((((c & 63) >> 3) ^ (position & 7)) << 4) + 2 * (c & 7); };
            float l[16];
#pragma unroll
            for (int j = 0; j < 16; j++) l[j] = 0.0f;
            bool pending = true;   // (a column has no reference yet)

            for (int i = 0; i < tiles; i++, n_tile++) {
                const int pos0 = (walk.tile0 + i) * kWideTile;
                // (of the halves only the values are waited for: they stay until this tile's weights are multiplied, the keys' place may
                // already be filled again)
                const int hv = n_half + 2 * i + 1;
                bar_wait(bar(meta.kv_full[hv % kSlots]), (hv / kSlots) & 1, gave_up, p.status);
                const unsigned long long there = *reinterpret_cast<volatile unsigned long long *>(&meta.ok[hv % kSlots]);
                // masked: not all rows see all positions, by the lengths; holes: pages that are not there (zeros, which no row sees)
                const bool masked = pos0 + kWideTile > min(before, sq.len) || pos0 < all_from, holes = there != 0x0101010101010101ull, mine = (there >> (8 * (place_in / kChunk))) & 1;
                bar_wait(bar(meta.s_full[n_tile & 1]), (n_tile >> 1) & 1, gave_up, p.status);
                tc_after();
                uint32_t v[16];
                if (has) {
                    uint32_t second[16];
                    tmem_load16(t_lane + 128 * (n_tile & 1) + col, v);
                    tmem_load16(t_lane + 128 * (n_tile & 1) + n_cols + col, second);
                    tmem_loaded();
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(second[j]));
                }
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(meta.s_empty[n_tile & 1]));

                // What is rarely done has code of its own, in loops where it can be: code that is jumped over, or met for the first time, is
                // fetched at the pace of thousands of clocks. It leaves log2 scores in place of the products.
                const float *scale = meta.scale;
                if (has && (masked || holes || p.softcap > 0.0f)) {
                    const uint32_t seen = !mine ? 0u : !masked ? 0xFFFFu : seen_of(meta.rows, c0, pos0 + place_in, before, sq.len);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        float x = __uint_as_float(v[j]) * meta.scale[c0 + j];
                        if (p.softcap > 0.0f) x = capped(x, p.softcap);
                        v[j] = (seen >> j) & 1 ? __float_as_uint(x) : __float_as_uint(-INFINITY);
                    }
                    scale = meta.one;
                }
                // x = score - m, the weight's log2, and whether one is too far above the reference
                float x[16], most = -INFINITY;
                if (has) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 s4 = *reinterpret_cast<const float4 *>(scale + c0 + j), b4 = *reinterpret_cast<const float4 *>(&meta.base[c0 + j]);
                        x[j] = fmaf(__uint_as_float(v[j]), s4.x, b4.x);
                        x[j + 1] = fmaf(__uint_as_float(v[j + 1]), s4.y, b4.y);
                        x[j + 2] = fmaf(__uint_as_float(v[j + 2]), s4.z, b4.z);
                        x[j + 3] = fmaf(__uint_as_float(v[j + 3]), s4.w, b4.w);
                        most = fmaxf(fmaxf(fmaxf(most, x[j]), fmaxf(x[j + 1], x[j + 2])), x[j + 3]);
                    }
                }
                if (has && group_any(group, pending || most > kHeadroom)) {
                    // ---- new references: the columns' maxima over the 128 lanes
                    const int c = c0 + (lane & 15);
                    {
                        float y[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) y[j] = x[j];
                        const float top = across(y, [](float a, float b) { return fmaxf(a, b); });
                        if (lane < 16) meta.red[lanes][c] = top;
                    }
                    group_sync(group);
                    bool none = false;
                    if (lanes == 0 && lane < 16) {
                        const float old = meta.m[c], from = meta.base[c];
                        const float top = fmaxf(fmaxf(meta.red[0][c], meta.red[1][c]), fmaxf(meta.red[2][c], meta.red[3][c]));
                        const float now = fmaxf(old, top - from);
                        meta.m[c] = now;
                        meta.base[c] = now == -INFINITY ? 0.0f : -now;
                        meta.more[c] = meta.base[c] - from;
                        meta.corr[c] = now == -INFINITY ? 1.0f : ex2(old - now);
                        none = now == -INFINITY;
                    }
                    pending = group_any(group, none);   // (a column that sees nothing yet takes its reference from what it sees first)
                    if (i > 0) bar_wait(bar(meta.pv_done), (n_tile - 1) & 1, gave_up, p.status);
                    tc_after();
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        l[j] *= meta.corr[c0 + j];
                        x[j] += meta.more[c0 + j];
                    }
                    if (i > 0) {
#pragma unroll 1
                        for (int k = 0; k < 2; k++) {
                            uint32_t o[16];
                            tmem_load16(t_lane + kTmemO + col + k * n_cols, o);
                            tmem_loaded();
#pragma unroll
                            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * meta.corr[c0 + j]);
                            tmem_store16(t_lane + kTmemO + col + k * n_cols, o);
                        }
                        tmem_stored();
                    }
                    tc_before();
                } else if (i > 0) {
                    bar_wait(bar(meta.pv_done), (n_tile - 1) & 1, gave_up, p.status);   // the weights' place is free
                }
                // ---- values that are no numbers, where not all rows see all positions (see krk_attn_kernel.cuh)
                bool any_odd = false;
                uint8_t *v_tile = smem + (hv % kSlots) * W::kHalf;
                if (masked) {
                    bool odd = false;
                    if (group == 0) {
                        for (int d = 0; d < D; d += 8) {
                            uint4 *at = reinterpret_cast<uint4 *>(v_tile + (d >> 6) * (kWideTile * 128) + place_in * 128 + ((((d & 63) >> 3) ^ (place_in & 7)) << 4));
                            uint4 w = *at;
                            uint32_t *ws = reinterpret_cast<uint32_t *>(&w);
                            bool bad = false;
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                if ((ws[c] & 0x7C00u) == 0x7C00u) ws[c] &= 0xFFFF0000u, bad = true;
                                if ((ws[c] & 0x7C000000u) == 0x7C000000u) ws[c] &= 0xFFFFu, bad = true;
                            }
                            if (bad) *at = w;
                            odd |= bad;
                        }
                        const uint32_t which = __ballot_sync(0xFFFFFFFFu, odd);
                        if (lane == 0) meta.odd[lanes] = which;
                    }
                    any_odd = soft_any(odd);
                }
                // ---- weights, in two terms, to [position][row]
                if (has) {
#pragma unroll
                    for (int j = 0; j < 16; j += 8) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int c = 0; c < 8; c += 2) {
                            const float w0 = kWeightUp * ex2(x[j + c]), w1 = kWeightUp * ex2(x[j + c + 1]);
                            l[j + c] += w0;
                            l[j + c + 1] += w1;
                            split(w0, w1, hi[c / 2], lo[c / 2]);
                        }
                        *reinterpret_cast<uint4 *>(weight_at(place_in, c0 + j)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(weight_at(place_in, n_cols + c0 + j)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                async_fence();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(meta.p_full));
                if (any_odd) {
                    // the products are waited for, and what was taken out is added to the rows that see it
                    bar_wait(bar(meta.pv_done), n_tile & 1, gave_up, p.status);
                    tc_after();
                    const int dim = place_in;
                    if (has) {
                        uint32_t o[16];
                        tmem_load16(t_lane + kTmemO + col, o);
                        tmem_loaded();
                        for (int j = 0; j < kWideTile; j++) {
                            if (!((meta.odd[j >> 5] >> (j & 31)) & 1)) continue;
                            if (pos0 + j >= sq.len) continue;   // (its values were there, unless a wait gave up: the page likewise)
                            const int page = p.table[(size_t)walk.s * p.table_width + (pos0 + j) / p.page_size];
                            if (page < 0 || page >= p.n_pages) continue;
                            const int64_t row = ((int64_t)page * p.n_kv + walk.kvh) * p.page_size + (pos0 + j) % p.page_size;
                            const float y = dim < D ? __half2float(reinterpret_cast<const __half *>(p.v)[row * D + dim]) : 0.0f;
                            if (fabsf(y) <= 65504.0f) continue;
                            const uint32_t seen = seen_of(meta.rows, c0, pos0 + j, before, sq.len);
#pragma unroll
                            for (int c = 0; c < 16; c++) {
                                if (!((seen >> c) & 1)) continue;
                                const float w = __half2float(*reinterpret_cast<const __half *>(weight_at(j, c0 + c))) + __half2float(*reinterpret_cast<const __half *>(weight_at(j, n_cols + c0 + c)));
                                o[c] = __float_as_uint(__uint_as_float(o[c]) + w * y);
                            }
                        }
                        __syncwarp();
                        tmem_store16(t_lane + kTmemO + col, o);
                        tmem_stored();
                    }
                    tc_before();
                    soft_sync();   // (the weights are read until here)
                }
            }
            n_half += 2 * tiles;

            // ---- the sums of weights, over the lanes; what a row's outputs are multiplied with
            if (has) {
                const int c = c0 + (lane & 15);
                const float sum = across(l, [](float a, float b) { return a + b; });
                if (lane < 16) meta.red[lanes][c] = sum;
                group_sync(group);
                constexpr float kDown = 1.0f / kWeightUp;
                if (lanes == 0 && lane < 16) {
                    const float all = kDown * ((meta.red[0][c] + meta.red[1][c]) + (meta.red[2][c] + meta.red[3][c]));
                    float keep;
                    if (walk.begins && walk.ends) meta.corr[c] = kDown * norm_of(p, meta.rows[c].head, meta.m[c], all, keep);
                    else {
                        meta.corr[c] = kDown;
                        if (c < n_rows) *reinterpret_cast<float2 *>(meta.to[c] + D) = make_float2(meta.m[c], all);
                    }
                }
                group_sync(group);
                bar_wait(bar(meta.pv_done), (n_tile - 1) & 1, gave_up, p.status);
                tc_after();
                uint32_t o[16], second[16];
                tmem_load16(t_lane + kTmemO + col, o);
                tmem_load16(t_lane + kTmemO + n_cols + col, second);
                tmem_loaded();
#pragma unroll
                for (int j = 0; j < 16; j++)
                    if (c0 + j < n_rows && place_in < D) meta.to[c0 + j][place_in] = (__uint_as_float(o[j]) + __uint_as_float(second[j])) * meta.corr[c0 + j];
            } else {
                bar_wait(bar(meta.pv_done), (n_tile - 1) & 1, gave_up, p.status);
            }
            tc_before();
            soft_sync();
        }
    } else if (warp < kSoftWarps + kCopyWarps) {
        // ===== copies: half tiles (keys, values in turn), the chunks of each dealt to the warps, the first one to another warp each time
        const int w = warp - kSoftWarps;
        constexpr int kPieces = RB / 16, kChunks = kWideTile / kChunk, kCopies = kChunk * kPieces / 32;
        // where a lane's copies of a chunk go: the pattern repeats every eight rows
        uint32_t to[kCopies / 2];
#pragma unroll
        for (int j = 0; j < kCopies / 2; j++) {
            const int c = lane + 32 * j, row = c / kPieces, piece = c % kPieces;
            to[j] = base + (piece >> 3) * (kWideTile * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
        }
        int h = 0, told = 0;   // half tiles asked for, and told of
        auto tell = [&](int n) {   // all but the n last ones have arrived
            if (n == 0) copies_wait<0>();
            else copies_wait<2>();
            async_fence();
            __syncwarp();
            for (; told < h - n; told++)
                if (lane == 0) bar_arrive(bar(meta.kv_full[told % kSlots]));
        };
        while (walk.next(p)) {
            const Seq &sq = walk.sq;
            const int32_t *table = p.table + (size_t)walk.s * p.table_width;
            int64_t pool_rows = 0;
#pragma unroll 1
            for (int i = 0; i < walk.tiles; i++) {
                if (i % (32 / kChunks) == 0) {   // lane: chunk lane % kChunks of tile i + lane / kChunks
                    const int tile = i + lane / kChunks, position = (walk.tile0 + tile) * kWideTile + lane % kChunks * kChunk;
                    pool_rows = -1;
                    if (tile < walk.tiles && position < sq.len) {
                        const int page = table[position / p.page_size];
                        if (page >= 0 && page < p.n_pages) pool_rows = ((int64_t)page * p.n_kv + walk.kvh) * p.page_size + position % p.page_size;
                    }
                }
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++) {
                    const int slot = h % kSlots;
                    const uint32_t empty = bar(meta.kv_empty[slot]), parity = ((h / kSlots) & 1) ^ 1;
                    if (!bar_test(empty, parity)) {
                        tell(0);   // (who frees the place may wait for these)
                        bar_wait(empty, parity, gave_up, p.status);
                    }
#pragma unroll 1
                    for (int chunk = (w + h) % kCopyWarps; chunk < kChunks; chunk += kCopyWarps) {
                        const int position = (walk.tile0 + i) * kWideTile + chunk * kChunk;
                        const int64_t row0 = __shfl_sync(0xFFFFFFFFu, pool_rows, kChunks * (i % (32 / kChunks)) + chunk);
                        const int left = row0 < 0 ? 0 : sq.len - position;   // rows that are not there come in as zeros
                        if (kv == 1 && lane == 0) reinterpret_cast<uint8_t *>(&meta.ok[slot])[chunk] = row0 >= 0;
                        const uint8_t *src = (kv ? p.v : p.k) + (row0 < 0 ? 0 : row0) * RB + 16 * lane;
                        const uint32_t at = slot * W::kHalf + chunk * (kChunk * 128);
                        if (left >= kChunk) {
#pragma unroll
                            for (int j = 0; j < kCopies; j++) copy16(to[j % (kCopies / 2)] + at + (j / (kCopies / 2)) * 1024, src + 512 * j, true);
                        } else {
#pragma unroll
                            for (int j = 0; j < kCopies; j++) copy16(to[j % (kCopies / 2)] + at + (j / (kCopies / 2)) * 1024, src + 512 * j, (lane + 32 * j) / kPieces < left);
                        }
                    }
                    copies_commit();
                    h++;
                    if (h - told > 2) tell(2);
                }
            }
        }
        tell(0);
    } else {
        // ===== products
        const uint32_t elected = elected_lane();
        uint32_t n_tile = 0, n_item = 0;
        int n_half = 0;
        while (walk.next(p)) {
            const int n = 2 * ((walk.n_rows + 15) / 16 * 16);   // both terms
            const uint32_t qk = wide_idesc(n, false, false), pv = wide_idesc(n, true, true);
            bar_wait(bar(meta.q_full), n_item & 1, gave_up, p.status);
            n_item++;
            auto scores = [&](int i) {
                const int hk = n_half + 2 * i, slot = hk % kSlots;
                const uint32_t nt = n_tile + i;
                bar_wait(bar(meta.kv_full[slot]), (hk / kSlots) & 1, gave_up, p.status);
                bar_wait(bar(meta.s_empty[nt & 1]), ((nt >> 1) & 1) ^ 1, gave_up, p.status);
                tc_after();
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const uint32_t a = desc_lo(base + slot * W::kHalf + (k >> 2) * (kWideTile * 128) + 32 * (k & 3), 16);
                    const uint32_t b = desc_lo(base + W::kQ + (k >> 2) * W::kQBlock + 32 * (k & 3), 16);
                    product(tmem + 128 * (nt & 1), a, kDescHi, b, kDescHi, qk, k > 0, elected);
                }
                products_commit(bar(meta.s_full[nt & 1]), elected);
                products_commit(bar(meta.kv_empty[slot]), elected);
            };
            scores(0);
            for (int i = 0; i < walk.tiles; i++) {
                if (i + 1 < walk.tiles) scores(i + 1);
                const int hv = n_half + 2 * i + 1, slot = hv % kSlots;
                bar_wait(bar(meta.kv_full[slot]), (hv / kSlots) & 1, gave_up, p.status);
                bar_wait(bar(meta.p_full), (n_tile + i) & 1, gave_up, p.status);
                tc_after();
#pragma unroll
                for (int k = 0; k < kWideTile / 16; k++) {
                    const uint32_t a = desc_lo(base + slot * W::kHalf + 2048 * k, kWideTile * 128);
                    const uint32_t b = desc_lo(base + W::kP + 2048 * k, kWideTile * 128);
                    product(tmem + kTmemO, a, kDescHi, b, kDescHi, pv, i > 0 || k > 0, elected);
                }
                products_commit(bar(meta.pv_done), elected);
                products_commit(bar(meta.kv_empty[slot]), elected);
            }
            n_tile += walk.tiles;
            n_half += 2 * walk.tiles;
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == kSoftWarps + kCopyWarps && *gave_up) {   // (nobody waits any more, so this is the last word on it)
        products_commit(bar(meta.drained), elected_lane());
        bar_wait_drained(bar(meta.drained));
    }
    if (warp == kSoftWarps + kCopyWarps) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <int D>
int launch_wide(const Params &p, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};   // devices whose limit of shared memory is raised for this kernel
    constexpr int kBytes = Wide<D>::kBytes + 1024;   // (begins on a 1024-byte boundary)
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        e = cudaFuncSetAttribute(attn_wide_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) {
        note_cuda_error(e);
        return KRK_CUDA_ELAUNCH;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid);
    cfg.blockDim = dim3(kWideThreads);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&cfg, attn_wide_kernel<D>, p));
}

}   // namespace attn
}   // namespace krk_cuda
