// krk_cuda_attention_chunk: the kernel on tcgen05, instantiated per cache type in krk_attn_chunk_f16.cu / _q8.cu / _q4.cu; the entry point is in
// krk_attn_chunk.cu.
//
//   out[r] = sum_p w_rp v_p / sum_p w_rp,   w_rp = exp(score_rp - max),   score = scale * q_r . k_p,   p up to r's own position
//
// A row is a (token, query head) pair; the `group` query heads of a key head are rows of one product. A block of threads has two tiles of 128 rows and goes
// through tiles of 128 positions: S = Q K^T with the rows as the lanes of tensor memory, so that a thread of the softmax has a row to itself; the weights go
// back to the place of the scores as the operand of O += P V. While one tile of rows is in its softmax the products of the other one run. Where shared memory has
// no room for that (heads of more than 128 values, two terms of keys and values) it is one tile of rows and tiles of 64 positions, with two places of scores in
// turn. Keys and values lie in shared memory in the 128-byte swizzle, keys as rows (K-major), values read across (MN-major).
//
// The reference that a softmax subtracts stands until a score passes it by 2^8: the sums in tensor memory are rescaled a few times a row, not each tile. The work
// is divided by what blocks of rows cost (ChunkWalk), partial sums of divided items are added up by a second kernel in the order of the blocks.
//
// f16 results: queries (f32 ones) and weights have one f16 term, quants times scales are rounded to f16, half of the exponentials are 7.5e-5 off, all of them below the rounding of the
// result or near it: against 64 bits 2.9e-4 over an f16 cache, 5.1e-4 to 6.4e-4 over 8 and 4 bits, where 2.1e-4 is the result's rounding alone. Second terms would be twice the products, as
// f32 results have them: those are 2e-6 off over 2048 positions (additions in tensor memory cut off; see add_run).
//
// Bound, f16 results of long chunks: 4096 tokens behind 8192, 32 heads of 128 over 8, 633 us on a cool card, 655 with pauses (1965 MHz), 720 to 745 back to back, where the power
// limit holds the clock at 1642 MHz (993 W): 920 to 1080 TFLOP/s; cuBLAS sustains 1372 on this card. The tensor pipe is busy 54 % of the cycles, the issue slots 47 %: products and the
// softmax of the other tile of rows wait for each other. Half of the exponentials are a polynomial's since the exponential unit would be as busy as the pipe (604 -> 548 us for 8192 tokens).
// f32 results take two terms of queries and weights, twice the products: 2048 tokens 121 to 124 us (2 x 280 TFLOP/s), 8192 tokens 980 to 1170. Over 8 and 4 bits what unpacks
// the quants is the limit, each block of rows for itself: 24 ragged sequences of up to 512 tokens behind up to 8000, 8 bits, 557 us; 4096 behind 8192 950 to 990; f32, three products, two
// chunks of up to 700 behind 5000, 405. A soft limit is a pass of its own over the scores: 2048 tokens 133 us for 74, f32 168 for 121. Few tokens: a launch, pages, one item's latency:
// 33 tokens 21 us.
#pragma once

#include <cuda.h>

#include "krk_attn_wide.cuh"

namespace krk_cuda {
namespace attn {

struct ChunkParams {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;         // elements from a token to the next
    const uint8_t *k, *v;
    const __half *k_scale, *v_scale;
    const int32_t *table, *q_start, *kv_len;
    const float *sinks;
    Shared *shared;                       // [grid]
    int *beyond;                          // [grid]: 1 where a value of keys or values lay beyond f16 (two terms of 8 and 4 bits)
    float *part;                          // [grid][2]: sums [R][D], maxima (log2) and weights [R][2], on 32-byte boundaries
    float *runs, *run_tops;               // f32: [grid][R][D] sums of the runs of tiles behind an item's last one, [grid][R] their references (log2)
    int64_t n_pages;
    int table_width, page_size, max_len, n_seq, n_heads, n_kv, group, max_q, window, whole, grid, q_half, out_half, out_wide;   // out_wide: rows of out begin on 32-byte boundaries
    uint32_t group_mul, group_shift;      // row / group = row * group_mul >> group_shift, rows below 2^30
    float scale, softcap, per_cap;        // per_cap: 1 / softcap, finite
    int *status;
    // f16 caches: the pool's rows as boxes of 64 values of box_rows positions, a part of one page; behind the last row zeros come in
    int box_rows, pool_rows;
    // queries: boxes of 128 bytes of 128 rows, where that many are whole tokens (q_boxes)
    int q_boxes;
    alignas(64) CUtensorMap k_map, v_map, q_map;
};
// n / d for n below 2^31: with 2^(s - 1) < d <= 2^s the factor ceil(2^(31 + s) / d) is less than one above the quotient, which n times it is at most 2^31 off.
inline void divide_by(int d, uint32_t &mul, uint32_t &shift) {
    int s = 0;
    while ((1ll << s) < d) s++;
    mul = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
    shift = 31 + s;
}
__host__ __device__ __forceinline__ int token_of(const ChunkParams &p, int row) { return (int)(((uint64_t)(uint32_t)row * p.group_mul) >> p.group_shift); }

// kt: terms of keys and values
__host__ __device__ constexpr int chunk_tiles_of(int d, int kt) { return d <= 128 && kt == 1 ? 2 : 1; }           // of rows, 128 each
__host__ __device__ constexpr int chunk_positions(int d, int kt) { return d <= 128 && kt == 1 ? 128 : 64; }       // of a tile
__host__ __device__ constexpr int chunk_rows(int d, int kt) { return 128 * chunk_tiles_of(d, kt); }
constexpr int kChunkSetup = 3;        // an item beside its tiles, in tiles
constexpr int kChunkWholeTiles = 8;   // contexts of up to so many tiles of positions are not divided
constexpr int kPolyOf8 = 4;           // f16: of eight exponentials, those by a polynomial
constexpr float kLetBe = 8.0f;        // log2: a reference stands until a score is more than this above it
constexpr float kUp = 128.0f, kUpLog2 = 7.0f;   // of weights: times 2^8 they stay below the f16 range

struct ChunkSeq {
    int q0, n_q, len, before, blocks;
};
// Blocks of R rows of a sequence, and what they cost: prefix(b) the units of its first b blocks, a closed formula (positions that a block's rows see, times the
// group, rather than its tiles), the same wherever it is worked out. An item's units a tile are bounded, see ChunkWalk::start.
__host__ __device__ __forceinline__ int64_t clamped_sum(int64_t x, int64_t step, int64_t cap, int64_t b) {   // of clamp(x + i step, 0, cap) over i < b
    const int64_t n0 = min(b, x >= 0 ? 0 : (-x + step - 1) / step), n1 = min(b, max(n0, cap <= x ? 0 : (cap - x + step - 1) / step)), n = n1 - n0;
    return n * x + step * ((n0 + n1 - 1) * n / 2) + (b - n1) * cap;
}
template <int R, int TP>
struct ChunkCost {
    int64_t ends, starts, cap, k0, last, head;   // group times: the end of block 0, its start, the positions there are
    bool window;
    __host__ __device__ __forceinline__ int64_t prefix(int64_t b) const { return b * k0 + 4 * (clamped_sum(ends, R, cap, b) - (window ? clamped_sum(starts, R, cap, b) : 0)); }
};
template <int R>
__host__ __device__ __forceinline__ ChunkSeq chunk_sequence(const ChunkParams &p, int s) {
    ChunkSeq q;
    q.q0 = p.q_start[s];
    q.n_q = min(max(p.q_start[s + 1] - q.q0, 0), p.max_q);
    const int len = min(max(p.kv_len[s], 0), 1 << 30);
    q.len = min(len, p.max_len);
    q.before = len - q.n_q;
    q.blocks = (q.n_q * p.group + R - 1) / R;   // (fewer than 2^30 rows)
    return q;
}
template <int R, int TP>
__host__ __device__ __forceinline__ ChunkCost<R, TP> chunk_cost(const ChunkParams &p, const ChunkSeq &q) {
    ChunkCost<R, TP> c;
    const int64_t g = p.group;
    c.ends = g * q.before + R;
    c.starts = g * ((int64_t)q.before - p.window + 1);
    c.cap = g * q.len;
    c.window = p.window > 0;
    c.k0 = 4 * g * TP * kChunkSetup;
    c.head = c.last = 0;
    if (q.blocks > 0) {
        const int64_t done = (int64_t)(q.blocks - 1) * R, left = q.n_q * g - done;
        const int64_t end = min(max(g * ((int64_t)q.before + q.n_q), (int64_t)0), c.cap), start = c.window ? min(max(c.starts + done, (int64_t)0), c.cap) : 0;
        c.last = c.k0 + (left > 128 ? 4 : 3) * max(end - start, (int64_t)0);
        c.head = c.prefix(q.blocks - 1) + c.last;
    }
    return c;
}
// The tiles of positions that some row of block b sees (one at least).
template <int R, int TP>
__host__ __device__ __forceinline__ void chunk_tiles(const ChunkParams &p, const ChunkSeq &q, int b, int &tile0, int &tiles) {
    const int rows = q.n_q * p.group, t0 = token_of(p, b * R), t1 = token_of(p, min(rows, (b + 1) * R) - 1);
    const int end = max(min(q.len, q.before + t1 + 1), 0), start = p.window > 0 ? max(0, q.before + t0 - p.window + 1) : 0;
    tile0 = min(start, max(end - 1, 0)) / TP;
    tiles = max(1, (end + TP - 1) / TP - tile0);
}

// A place in the work: a tile of a block of rows of a key head of a sequence.
struct ChunkPlace {
    int s, kvh, b, tile;
};
template <int R, int TP>
struct ChunkWalk {
    ChunkPlace at, end;    // at.tile: the first tile of the current item that is this CTA's
    ChunkSeq sq;
    int64_t total, base;   // units in all, and before the first item's sequence
    int64_t first_unit, behind_unit;
    double per_cta;
    int grid, cta;
    bool first, over;
    // of the current item; parts: see Shared
    int kvh, block, s, n_rows, tile0, tiles, parts;
    bool begins, ends;

    // (in f64, the same in every CTA and rising with b; quotients of 64 bits take a thread some 400 clocks)
    __host__ __device__ __forceinline__ int64_t unit_of(int b) const { return b >= grid ? total : min((int64_t)(per_cta * (double)b), total); }
    // The tile that a border lies at, `off` units into an item of `cost`: borders near an item's ends are at them. (f32: off by a tile at most, of millions.)
    __host__ __device__ __forceinline__ static int tile_at(int64_t off, int64_t cost, int tiles, int whole) {
        if (whole) return 2 * off < cost ? 0 : tiles;
        const int t = (int)((float)off / (float)cost * (float)tiles);
        return t < 2 ? 0 : t > tiles - 2 ? tiles : t;
    }
    // Where unit in_seq of sequence s lies. On the device by a warp, whose halves may ask for two units.
    __host__ __device__ __forceinline__ static ChunkPlace place(const ChunkParams &p, int s, int64_t in_seq) {
        ChunkPlace r;
        const ChunkSeq q = chunk_sequence<R>(p, s);
        const ChunkCost<R, TP> c = chunk_cost<R, TP>(p, q);
        r.s = s;
        r.kvh = min((int)((float)in_seq / (float)c.head), p.n_kv - 1);
        if (r.kvh * c.head > in_seq) r.kvh--;
        else if (r.kvh + 1 < p.n_kv && (r.kvh + 1) * c.head <= in_seq) r.kvh++;
        const int64_t in_head = in_seq - r.kvh * c.head;
        int lo = 0;   // the last block that begins at or before it
#ifdef __CUDA_ARCH__
        const int lane = threadIdx.x & 31;
        for (int n = q.blocks; __any_sync(0xFFFFFFFFu, n > 1);) {
            const int step = (n + 15) / 16, i = (lane & 15) * step;
            const int ahead = __popc(__ballot_sync(0xFFFFFFFFu, i < n && c.prefix(lo + i) <= in_head) >> (lane & 16) & 0xFFFFu) - 1;
            lo += ahead * step;
            n = min(step, n - ahead * step);
        }
#else
        for (int hi = q.blocks - 1; lo < hi;) {
            const int mid = (lo + hi + 1) / 2;
            if (c.prefix(mid) <= in_head) lo = mid;
            else hi = mid - 1;
        }
#endif
        r.b = lo;
        int t0, tiles;
        chunk_tiles<R, TP>(p, q, lo, t0, tiles);
        const int64_t from = c.prefix(lo);
        r.tile = tile_at(in_head - from, (lo == q.blocks - 1 ? c.last : c.prefix(lo + 1) - from), tiles, p.whole);
        return r;
    }
    // Undivided items, no more of them than blocks of threads: each has one, whatever it costs. (Units and places would take 9000 clocks, most of them for fetching code.)
    __device__ __forceinline__ bool start_with_one(const ChunkParams &p) {
        const int lane = threadIdx.x & 31, me = (int)blockIdx.x;
        ChunkPlace mine = {p.n_seq, 0, 0, 0};
        int64_t before = 0;
        for (int s0 = 0; s0 < p.n_seq; s0 += 32) {
            const int blocks = s0 + lane < p.n_seq ? chunk_sequence<R>(p, s0 + lane).blocks : 0;
            const int64_t items = (int64_t)blocks * p.n_kv;
            int64_t upto = items;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                if (lane >= o) upto += v;
            }
            const int64_t off = me - (before + upto - items);
            const uint32_t here = __ballot_sync(0xFFFFFFFFu, off >= 0 && off < items);
            if (here) {
                const int l = __ffs(here) - 1, n = __shfl_sync(0xFFFFFFFFu, blocks, l), item = (int)__shfl_sync(0xFFFFFFFFu, off, l);
                mine = {s0 + l, item / n, item % n, 0};
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
            if (before > (int64_t)gridDim.x) return false;
        }
        total = before, grid = (int)before, cta = me, first_unit = 0, behind_unit = 1, per_cta = 1.0;
        ChunkPlace behind = mine;
        behind.tile = INT_MAX;
        begin(p, mine, behind, 0);
        return true;
    }
    // By a warp.
    __device__ __forceinline__ void start(const ChunkParams &p) {
        const int lane = threadIdx.x & 31;
        if (p.whole && start_with_one(p)) return;
        auto units = [&](int s0) { return s0 + lane < p.n_seq ? p.n_kv * chunk_cost<R, TP>(p, chunk_sequence<R>(p, s0 + lane)).head : 0; };
        int64_t mine = 0;
        total = 0;
        for (int s0 = 0; s0 < p.n_seq; s0 += 32) {
            mine = units(s0);
            int64_t all = mine;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
            total += all;
        }
        share(p, (int)blockIdx.x);
        const int64_t u[2] = {first_unit, behind_unit};
        int found[2] = {p.n_seq, p.n_seq};
        int64_t before[2] = {total, total}, from = 0;
        for (int s0 = 0; s0 < p.n_seq && found[1] == p.n_seq; s0 += 32) {
            if (p.n_seq > 32) mine = units(s0);   // (up to 32 sequences the first ones stand)
            int64_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                if (lane >= o) upto += v;
            }
            const int64_t lo = from + upto - mine;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t here = __ballot_sync(0xFFFFFFFFu, u[i] >= lo && u[i] < lo + mine);
                if (here) found[i] = s0 + __ffs(here) - 1, before[i] = __shfl_sync(0xFFFFFFFFu, lo, __ffs(here) - 1);
            }
            from += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
        ChunkPlace mine_at = {p.n_seq, 0, 0, 0};
        if (found[0] < p.n_seq) {
            const int half = lane >> 4, s0 = half ? found[1] : found[0];
            const ChunkPlace r = place(p, min(s0, p.n_seq - 1), s0 < p.n_seq ? (half ? u[1] - before[1] : u[0] - before[0]) : 0);
            mine_at = {s0, r.kvh, r.b, r.tile};
        }
        auto from_lane = [&](int l) {
            return ChunkPlace{__shfl_sync(0xFFFFFFFFu, mine_at.s, l), __shfl_sync(0xFFFFFFFFu, mine_at.kvh, l), __shfl_sync(0xFFFFFFFFu, mine_at.b, l), __shfl_sync(0xFFFFFFFFu, mine_at.tile, l)};
        };
        begin(p, from_lane(0), from_lane(16), before[0]);
    }
    // Of CTA b, with the total of units: how many share them, and its own.
    __host__ __device__ __forceinline__ void share(const ChunkParams &p, int b) {
        // A share is longer than what an item costs beside its tiles: no two borders lie at one tile inside an item, which is not near its ends where it has
        // four tiles and more, of 4 group (TP kChunkSetup / tiles + TP + 2) units at most. Undivided items have a share each if there are CTAs.
        const int64_t least = p.whole ? 1 : (int64_t)4 * p.group * TP * (kChunkSetup + 1);
        cta = b;
        const int most = (int)fminf((float)p.grid, (float)total / (float)least);
        grid = max(most, 1);
        per_cta = (double)total * (double)(1.0f / (float)grid);   // (to f32: shares are so far from equal, and the last one ends at the total)
        first_unit = unit_of(b);
        behind_unit = unit_of(b + 1);
    }
    // From the places of its first unit and of the one behind its last (s n_seq: none), and the units before the first one's sequence.
    __host__ __device__ __forceinline__ void begin(const ChunkParams &p, const ChunkPlace &from, const ChunkPlace &upto, int64_t units_before) {
        at = from, end = upto, base = units_before;
        over = first_unit >= behind_unit || at.s >= p.n_seq;
        if (!over) sq = chunk_sequence<R>(p, at.s);
        first = true;
        kvh = block = s = n_rows = tile0 = tiles = parts = 0;
        begins = ends = false;
    }
    // Parts of the item that this CTA has the second one of, 0 if it has not.
    __host__ __device__ __forceinline__ int count_parts(const ChunkParams &p, int all) const {
        const ChunkCost<R, TP> c = chunk_cost<R, TP>(p, sq);
        const int64_t from = base + at.kvh * c.head + c.prefix(at.b), cost = at.b == sq.blocks - 1 ? c.last : c.prefix(at.b + 1) - c.prefix(at.b);
        const int me = cta;
        if (me == 0) return 0;
        const int64_t before = unit_of(me - 1) - from;
        if (before >= 0 && tile_at(before, cost, all, p.whole) > 0) return 0;
        // the borders behind it that lie in the item, one behind the other
        int n = 0;
        auto inside = [&](int e) {
            const int64_t off = unit_of(e) - from;
            return e < grid && off < cost && tile_at(off, cost, all, p.whole) < all;
        };
#ifdef __CUDA_ARCH__
        for (int e = me + 1;; e += 32) {
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, inside(e + (int)(threadIdx.x & 31)));
            n += __popc(some);
            if (some != 0xFFFFFFFFu) break;
        }
#else
        while (inside(me + 1 + n)) n++;
#endif
        return n + 2;
    }
    template <bool PARTS = false>
    __host__ __device__ __forceinline__ bool next(const ChunkParams &p) {
        while (!over) {
            int t0, all;
            chunk_tiles<R, TP>(p, sq, at.b, t0, all);
            const bool last = at.s == end.s && at.kvh == end.kvh && at.b == end.b;
            const int from = at.tile, upto = last ? min(end.tile, all) : all;
            const bool some = upto > from;
            if (some) {
                kvh = at.kvh, block = at.b, s = at.s;
                n_rows = min(R, sq.n_q * p.group - at.b * R);
                tile0 = t0 + from, tiles = upto - from;
                begins = from == 0, ends = upto == all;
                if constexpr (PARTS) parts = first && from > 0 ? count_parts(p, all) : 0;
            }
            const ChunkSeq was = sq;
            first = false;
            at.tile = 0;
            if (last) over = true;
            else if (++at.b >= sq.blocks) {
                at.b = 0;
                if (++at.kvh >= p.n_kv) {
                    at.kvh = 0;
                    do {
                        if (++at.s >= p.n_seq) {
                            over = true;
                            break;
                        }
                        sq = chunk_sequence<R>(p, at.s);
                    } while (sq.blocks == 0);
                    if (!over && at.s > end.s) over = true;
                }
            }
            if (some) {
                now = was;
                return true;
            }
        }
        return false;
    }
    ChunkSeq now;   // the current item's sequence
    __host__ __device__ __forceinline__ void note(const ChunkParams &p) const {   // by one thread
        Shared it;
        it.parts = parts;
        it.n_rows = n_rows;
        it.kvh = kvh;
        it.row0 = block * R;
        it.q0 = now.q0;
        it.pad[0] = it.pad[1] = it.pad[2] = 0;
        p.shared[blockIdx.x] = it;
    }
};

template <int D, int NT, int CT>
struct Chunk {
    static constexpr bool QUANT = CT != KRK_CUDA_KV_F16;
    static constexpr int KT = QUANT && NT == 2 ? 2 : 1;              // terms of keys and values: quants times their scales have 18 bits
    static constexpr int NQ = chunk_tiles_of(D, KT), TP = chunk_positions(D, KT), R = chunk_rows(D, KT);
    static constexpr int kMetaBytes = 1920;
    static constexpr int kPanels = (D + 63) / 64;                    // blocks of 64 values
    static constexpr int kTerm = kPanels * 128 * 128, kQTile = NT * kTerm;
    static constexpr int kQSets = NT == 1 && !QUANT ? 2 : 1, kQSet = NQ * kQTile;   // the queries of this item and, where there is room, of the next one
    static constexpr int kSlotTerm = kPanels * TP * 128, kSlot = KT * kSlotTerm;   // half a tile: keys or values
    static constexpr int kRawChunk = QUANT ? kChunk * (row_bytes_of(CT, D) + scale_bytes_of(CT, D)) : 0, kRaws = 3, kRaw = TP / kChunk * kRawChunk;   // 8 and 4 bits as they are: quants and scales of a half tile
    static constexpr int kRoom = 227 * 1024 - 1024 - kMetaBytes - kQSets * kQSet - kRaws * kRaw;
    static constexpr int kSlots = kRoom / kSlot > 6 ? 6 : kRoom / kSlot;
    static constexpr int kQ = kSlots * kSlot, kRawAt = kQ + kQSets * kQSet, kMeta = kRawAt + kRaws * kRaw, kBytes = kMeta + kMetaBytes + 1024;   // (begins on a 1024-byte boundary)
    // warps: softmax, copies, products, the one that finds items
    static constexpr int kSoft = 4 * NQ, kCopies = KT == 2 ? 8 : QUANT ? 4 : 2, kProduct = kSoft + kCopies, kFinder = kProduct + 1, kWarps = kSoft + (KT == 2 ? 12 : QUANT ? 8 : 4), kThreads = 32 * kWarps;
    // Registers of a thread, traded between groups of four warps (a spill goes to level 2: shared memory has what level 1 had). Launched with: 384 threads 168, 512 128.
    static constexpr bool kTrade = NQ == 2 || KT == 2;
    static constexpr int kSoftRegs = KT == 2 ? 184 : QUANT ? 168 : 200, kCopyRegs = KT == 2 ? 112 : QUANT ? 88 : 104, kOtherRegs = KT == 2 ? 104 : QUANT ? 88 : 104;
    static_assert(!kTrade || 32 * (kSoft * kSoftRegs + (QUANT ? kCopies * kCopyRegs + 4 * kOtherRegs : 4 * kCopyRegs)) <= (QUANT ? 512 * 128 : 384 * 168), "registers of a launch");
    static constexpr uint32_t kO = 256;                              // column of the sums; of the second tile's: 128 more
    static constexpr uint32_t kS = NQ == 2 ? 128 : 64;               // from a place of scores to the next
    static_assert(kSlots >= 3, "a half tile of values and one of keys at work, one on its way");
    static_assert(kBytes <= 227 * 1024, "shared memory");
    using Walk = ChunkWalk<R, TP>;
    // f32: tiles whose values are summed in tensor memory. Its sums are cut off, not rounded: a step of 16 positions loses up to a last place of what the sum has come to,
    // always towards zero, and behind 5000 positions three terms' steps had lost 1.6e-5. So the sums of a run go to memory, where runs are added in f32. Products with second
    // terms have sums of their own where there is room (8 bits, 8600 positions of values of one sign: 5.7e-6; in one sum, with runs of 1024, 7.3e-6). 4096 tokens behind 8192
    // take 5 to 10 % longer than without.
    static constexpr int kRun = 2048 / TP;
    static constexpr bool kApart = KT == 2;
};

struct ChunkItem {
    int goes_on, q0, len, before, s, kvh, block, n_rows, tile0, all, tiles[2], all_from, all_to, any_from;   // all: its tiles, tiles: that the rows of a tile see; every row sees [all_from, all_to), none what is before any_from
    int rows_from[2], rows_to[2];   // every row of a tile of rows sees [rows_from, rows_to)
    bool whole, begins;
};
constexpr int kChunkItems = 3;   // found ahead
struct ChunkMeta {
    unsigned long long kv_full[6], kv_empty[6], s_full[2], p_half[2], p_full[2], pv_done[2], q_full[2][2], q_empty[2], q_raw, item_full[kChunkItems], item_empty[kChunkItems], drained;
    uint32_t odd[2][8];       // of a tile of rows, an item in turn: values of a tile that not all rows see are no numbers
    uint8_t there[8];         // of a tile of positions, in turn: bit c: chunk c is a page's
    uint32_t tmem;
    int gave_up, beyond;
    ChunkItem item[kChunkItems], mine[2];   // mine: of a tile of rows, what its first thread has read
};
// A place of a ring and the parity of its turn.
template <int N>
struct Ring {
    int at = 0;
    uint32_t turn = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) at = 0, turn ^= 1;
    }
};

__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
                 "%26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
                   "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
                 "%27, %28, %29, %30, %31, %32};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
                   "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
                   "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ bool take_out(uint32_t &x) {   // of two f16, those that are no numbers
    bool bad = false;
    if ((x & 0x7C00u) == 0x7C00u) x &= 0xFFFF0000u, bad = true;
    if ((x & 0x7C000000u) == 0x7C000000u) x &= 0xFFFFu, bad = true;
    return bad;
}
// As bar_wait, without a call: a kernel whose warps trade registers has none. Tries that follow each other take the path to shared memory from the other
// warps' exchanges and loads; a warp with time sleeps between them.
template <int SLEEP>
__device__ __forceinline__ void bar_wait_here(uint32_t bar, uint32_t parity, volatile int *gave_up, int *status) {
    if (bar_try(bar, parity)) return;
    const long long t0 = clock64();
#pragma unroll 1
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 16; i++) {
            if (SLEEP > 0) __nanosleep(SLEEP);
            if (bar_try(bar, parity)) return;
        }
        if (*gave_up) return;
        if (clock64() - t0 > kWaitLimit) {
            *gave_up = 1;
            atomicExch(status, KRK_CUDA_ETIMEOUT);
            return;
        }
    }
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// The 128 threads of a tile of rows meet. (Warps whole: one whose first thread had been apart stayed in two parts, and took twice its time and 440 clocks an exchange.)
__device__ __forceinline__ void rows_sync(int tile) {
    __syncwarp();
    asm volatile("barrier.cta.sync.aligned %0, 128;" ::"r"(1 + tile) : "memory");
}
// 32 bytes of a thread: a sector (wide: on its boundary).
__device__ __forceinline__ void store32(void *to, const uint32_t *w, int wide) {
    if (wide)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    else {
        reinterpret_cast<uint4 *>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4 *>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
// N products over 16 values each, both operands from shared memory; the next 16 values are 32 bytes on. Executed as `product`.
template <int N>
__device__ __forceinline__ void products_k(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t onto, uint32_t elected) {
    static_assert(N == 2 || N == 4, "");
    if constexpr (N == 4)
        asm volatile("{\n .reg .pred p, q, t;\n .reg .b64 a0, b0, a1, b1, a2, b2, a3, b3;\n .reg .b32 x1, x2, x3, y1, y2, y3;\n"
                     " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n setp.eq.b32 t, 0, 0;\n"
                     " add.s32 x1, %1, 2;\n add.s32 x2, %1, 4;\n add.s32 x3, %1, 6;\n add.s32 y1, %2, 2;\n add.s32 y2, %2, 4;\n add.s32 y3, %2, 6;\n"
                     " mov.b64 a0, {%1, %7};\n mov.b64 a1, {x1, %7};\n mov.b64 a2, {x2, %7};\n mov.b64 a3, {x3, %7};\n"
                     " mov.b64 b0, {%2, %7};\n mov.b64 b1, {y1, %7};\n mov.b64 b2, {y2, %7};\n mov.b64 b3, {y3, %7};\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %3, {%5, %5, %5, %5}, p;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, {%5, %5, %5, %5}, t;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, {%5, %5, %5, %5}, t;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, {%5, %5, %5, %5}, t;\n}\n"
                     ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(onto), "r"(0u), "r"(elected), "r"(kDescHi) : "memory");
    else
        asm volatile("{\n .reg .pred p, q, t;\n .reg .b64 a0, b0, a1, b1;\n .reg .b32 x1, y1;\n"
                     " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n setp.eq.b32 t, 0, 0;\n add.s32 x1, %1, 2;\n add.s32 y1, %2, 2;\n"
                     " mov.b64 a0, {%1, %7};\n mov.b64 a1, {x1, %7};\n mov.b64 b0, {%2, %7};\n mov.b64 b1, {y1, %7};\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %3, {%5, %5, %5, %5}, p;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, {%5, %5, %5, %5}, t;\n}\n"
                     ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(onto), "r"(0u), "r"(elected), "r"(kDescHi) : "memory");
}
// The products over 32 positions with the weights in tensor memory (lane = row, a column two f16): 16 columns of first terms, NT 2: 16 of second ones behind
// them; the next 16 positions of the values are 2048 bytes on.
template <int NT>
__device__ __forceinline__ void products_p(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t onto, uint32_t elected) {
    if constexpr (NT == 1)
        asm volatile("{\n .reg .pred p, q, t;\n .reg .b64 b0, b1;\n .reg .b32 x1, y1;\n"
                     " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n setp.eq.b32 t, 0, 0;\n add.s32 x1, %1, 8;\n add.s32 y1, %2, 128;\n"
                     " mov.b64 b0, {%2, %7};\n mov.b64 b1, {y1, %7};\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b0, %3, {%5, %5, %5, %5}, p;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [x1], b1, %3, {%5, %5, %5, %5}, t;\n}\n"
                     ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(onto), "r"(0u), "r"(elected), "r"(kDescHi) : "memory");
    else
        asm volatile("{\n .reg .pred p, q, t;\n .reg .b64 b0, b1;\n .reg .b32 x1, x2, x3, y1;\n"
                     " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n setp.eq.b32 t, 0, 0;\n add.s32 x1, %1, 8;\n add.s32 x2, %1, 16;\n add.s32 x3, %1, 24;\n add.s32 y1, %2, 128;\n"
                     " mov.b64 b0, {%2, %7};\n mov.b64 b1, {y1, %7};\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b0, %3, {%5, %5, %5, %5}, p;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [x2], b0, %3, {%5, %5, %5, %5}, t;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [x1], b1, %3, {%5, %5, %5, %5}, t;\n"
                     " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [x3], b1, %3, {%5, %5, %5, %5}, t;\n}\n"
                     ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(onto), "r"(0u), "r"(elected), "r"(kDescHi) : "memory");
}
// As capped, without a call: the hyperbolic tangent from one exponential, 2^-22 of 1 off. Below 1/4, where that would be more and more of it (under a limit far above the scores
// all of it), from its series, whose next term is 2^-26 of it there. per_cap: a quotient's rounding and its own, 2^-22 at the largest limits, whose reciprocals have no leading bit.
__device__ __forceinline__ float capped_here(float x, float cap, float per_cap) {
    const float y = x * per_cap, z = y * y;
    float r;   // (to its last place or the one beside)
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(y * (2.0f * 1.44269504f))));
    float t = 1.0f - 2.0f * r;
    if (z < 0.0625f) t = fmaf(y * z, fmaf(z, fmaf(z, fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), y);
    return cap * (1.44269504f * t);
}
// Two f32 at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of two x to 7.5e-5 of itself (x up to 15; an f16 weight's rounding is 2.4e-4 at most): the whole part goes to the exponent, the rest, in +-1/2, to the polynomial
// of third degree whose greatest relative error is least. Below 2^-40 it is 2^-40, which f16 does not hold; a NaN stays one.
__device__ __forceinline__ uint64_t exp2_poly(uint64_t xx) {
    float a, b, ta, tb;
    unpair(xx, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-40.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-40.0f));
    const uint64_t x = pair(a, b), t = add2(x, pair(12582912.0f, 12582912.0f)), n = add2(t, pair(-12582912.0f, -12582912.0f));   // 1.5 * 2^23: to whole numbers
    const uint64_t r = fma2(n, pair(-1.0f, -1.0f), x);
    uint64_t y = fma2(pair(0.055171668f, 0.055171668f), r, pair(0.242611122f, 0.242611122f));
    y = fma2(y, r, pair(0.693260986f, 0.693260986f));
    y = fma2(y, r, pair(0.999928074f, 0.999928074f));
    unpair(y, a, b);
    unpair(t, ta, tb);
    return pair(__int_as_float(__float_as_int(a) + (__float_as_int(ta) << 23)), __int_as_float(__float_as_int(b) + (__float_as_int(tb) << 23)));
}
// A value of a cache as f16 products see it, by a slow path.
template <int CT, int D>
__device__ __forceinline__ float value_at(const uint8_t *pool, const __half *scale, int64_t row, int c) {
    if constexpr (CT == KRK_CUDA_KV_F16) return __half2float(reinterpret_cast<const __half *>(pool)[row * D + c]);
    const __half d = scale[row * (D / 32) + c / 32];
    int q;
    if constexpr (CT == KRK_CUDA_KV_Q8) q = (int8_t)pool[row * D + c];
    else {
        const int b = pool[row * (D / 2) + c / 32 * 16 + c % 16];
        q = ((c & 16) ? b >> 4 : b & 15) - 8;
    }
    return __half2float(__hmul(d, __int2half_rn(q)));
}

// Log2 scores under a soft limit in place of products.
template <int TP>
__device__ __forceinline__ void soft_limit(uint32_t t_s, float sc, float cap, float per_cap) {
#pragma unroll 1
    for (int c = 0; c < TP; c += 16) {
        uint32_t v[16];
        tmem_load16(t_s + c, v);
        tmem_loaded();
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = __float_as_uint(capped_here(__uint_as_float(v[j]) * sc, cap, per_cap));
        tmem_store16(t_s + c, v);
    }
    tmem_stored();
}
// A row's sums out of tensor memory, under the reference m, onto those that are kept under another one. Nobody else adds to them: additions in memory come in the
// order of the runs, and their thread does not wait for them. (Read, added to and written back they took a tenth of the time.)
template <int D, bool APART>
__device__ __forceinline__ void add_run(uint32_t t_o, float *kept, float *kept_top, float m, bool onto) {
    if (onto && __any_sync(0xFFFFFFFFu, *kept_top != m)) {
        const float top = *kept_top, f = top == -INFINITY ? 0.0f : ex2(top - m);
#pragma unroll 1
        for (int c = 0; c < D; c += 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(kept + c));   // (level 2, where the additions are)
            *reinterpret_cast<float4 *>(kept + c) = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
        }
        __syncwarp();
    }
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
        uint32_t o[16], rest[APART ? 16 : 1];
        tmem_load16(t_o + c, o);
        if constexpr (APART) tmem_load16(t_o + 128 + c, rest);
        tmem_loaded();
        if constexpr (APART)
#pragma unroll
            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(rest[j]));
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            if (onto)
                asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                             ::"l"(kept + c + j), "f"(__uint_as_float(o[j])), "f"(__uint_as_float(o[j + 1])), "f"(__uint_as_float(o[j + 2])), "f"(__uint_as_float(o[j + 3])) : "memory");
            else
                *reinterpret_cast<uint4 *>(kept + c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
    }
    *kept_top = m;
    __syncwarp();
}
// Values that are no numbers, in tiles that not all rows of an item see, were taken out of the products: here they are, for the rows that see them. A thread's
// row sees [pos0, end); tiles that every row sees were left as they are.
template <int CT, int D, int TP>
__device__ __forceinline__ void add_odd(const ChunkParams &p, const volatile ChunkItem &it, uint32_t t_o, int pos0, int end) {
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
        uint32_t o[16];
        tmem_load16(t_o + c, o);
        tmem_loaded();
        for (int pos = pos0; pos < end; pos++) {
            const int t0 = pos / TP * TP;
            if (t0 + TP <= it.all_to && t0 >= it.all_from) {
                pos = t0 + TP - 1;
                continue;
            }
            const int page = p.table[(size_t)it.s * p.table_width + pos / p.page_size];
            if (page < 0 || page >= p.n_pages) continue;
            const int64_t row = ((int64_t)page * p.n_kv + it.kvh) * p.page_size + pos % p.page_size;
            for (int j = 0; j < 16; j++) {
                const float y = value_at<CT, D>(p.v, p.v_scale, row, c + j);
                if (fabsf(y) <= 65504.0f) continue;
#pragma unroll
                for (int k = 0; k < 16; k++)
                    if (k == j) o[k] = __float_as_uint(__uint_as_float(o[k]) + y);
            }
        }
        __syncwarp();
        tmem_store16(t_o + c, o);
    }
    tmem_stored();
}

// HALF: f16 out, one term of each query and weight (NT), else f32 and two.
template <int D, int CT, bool HALF>
__global__ void __launch_bounds__((Chunk<D, HALF ? 1 : 2, CT>::kThreads), 1)
attn_chunk_kernel(const __grid_constant__ ChunkParams p) {
    constexpr int NT = HALF ? 1 : 2;
    using C = Chunk<D, NT, CT>;
    constexpr int KT = C::KT;
    using Walk = typename C::Walk;
    constexpr int NQ = C::NQ, TP = C::TP, R = C::R, RB = row_bytes_of(CT, D), kChunks = TP / kChunk;
    constexpr bool kQuant = CT != KRK_CUDA_KV_F16;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = smem_addr(smem);
    using Meta = ChunkMeta;
    static_assert(sizeof(Meta) <= C::kMetaBytes, "Chunk::kMeta");
    Meta &meta = *reinterpret_cast<Meta *>(smem + C::kMeta);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int *gave_up = &meta.gave_up;
    auto bar = [&](unsigned long long &b) { return smem_addr(&b); };
    auto wait = [&](unsigned long long &b, uint32_t parity) { bar_wait_here<0>(bar(b), parity, gave_up, p.status); };
    auto wait_idle = [&](unsigned long long &b, uint32_t parity) { bar_wait_here<100>(bar(b), parity, gave_up, p.status); };

    // f16 queries enter as they are, and are copied ahead
    const bool as_they_are = HALF && p.q_half && p.scale >= 0.0f;
    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < C::kSlots; i++) {
                bar_init(bar(meta.kv_full[i]), kQuant ? C::kCopies : 1);
                bar_init(bar(meta.kv_empty[i]), 1);
            }
            for (int i = 0; i < 2; i++) {
                bar_init(bar(meta.s_full[i]), 1);
                bar_init(bar(meta.p_half[i]), 4);
                bar_init(bar(meta.p_full[i]), 4);
                bar_init(bar(meta.pv_done[i]), 1);
                for (int j = 0; j < 2; j++) bar_init(bar(meta.q_full[i][j]), as_they_are ? (kQuant ? C::kCopies : 1) : 4);   // [set][tile of rows]
                bar_init(bar(meta.q_empty[i]), 1);
            }
            bar_init(bar(meta.q_raw), kQuant ? C::kCopies : 1);
            bar_init(bar(meta.drained), 1);
            for (int i = 0; i < kChunkItems; i++) {
                bar_init(bar(meta.item_full[i]), 1);
                bar_init(bar(meta.item_empty[i]), NQ + C::kCopies + 1);
            }
            meta.gave_up = 0, meta.beyond = 0;
        }
        if (lane < 16) meta.odd[lane >> 3][lane & 7] = 0;
        __syncwarp();
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        async_fence();
    }
    if (warp == C::kProduct) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&meta.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    tc_after();
    const uint32_t tmem = meta.tmem;

    if (warp < C::kSoft) {
        // ===== softmax: thread = row
        if constexpr (C::kTrade) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
        const int tq = warp >> 2, r_in = tid & 127, quarter = warp & 3;
        const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16), t_o = t_lane + C::kO + 128 * tq;
        uint32_t n_tile = 0, n_item = 0, n_all = 0;   // tiles of this tile of rows, items, tiles of all items
        Ring<kChunkItems> found;
        for (;; n_item++, found.next()) {
            if (r_in == 0) {   // (one thread decides for its barriers' 128)
                wait(meta.item_full[found.at], found.turn);
                ChunkItem it = meta.item[found.at];
                if (*gave_up) it.goes_on = 0;
                meta.mine[tq] = it;
                bar_arrive(bar(meta.item_empty[found.at]));
            }
            rows_sync(tq);
            // (read again where it is wanted, not kept beside a tile's scores: registers)
            const volatile ChunkItem &it = meta.mine[tq];
            if (!it.goes_on) break;
            const int tiles = it.tiles[tq];
            n_all += it.all;
            if (it.n_rows <= 128 * tq) {
                if (!HALF) wait(meta.q_raw, n_item & 1);   // (a parity tells one turn from the next)
                rows_sync(tq);
                continue;
            }
            float sc;             // takes a row's products to its log2 scores (with a soft limit: to the scores)
            int from, behind;     // what the row sees: [from, behind)
            const float row_scale = fabsf(p.scale) * (p.softcap > 0.0f ? 1.0f : 1.44269504f);
            {
                const int row0 = it.block * R + 128 * tq, token = token_of(p, row0 + min(r_in, min(128, it.n_rows - 128 * tq) - 1));   // row0: among the key head's
                behind = min((int)it.len, it.before + token + 1), from = p.window > 0 ? max(0, it.before + token - p.window + 1) : 0;
            }
            sc = row_scale;
            if (!as_they_are) {
                // ---- queries under a power of two of their row: the largest value in [2^10, 2^11)
                const int kvh = it.kvh, q0 = it.q0, row0 = it.block * R + 128 * tq, mine_rows = min(128, it.n_rows - 128 * tq);
                const uint32_t q_off = C::kQ + (C::kQSets == 2 ? n_item & 1 : 0) * C::kQSet + tq * C::kQTile;
                uint8_t *q_tile = smem + q_off;
                const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
                auto power_of = [](float most) { return most > 0.0f && most <= 3.4028234e38f ? 10 - max((int)(__float_as_uint(most) >> 23) - 127, -110) : 0; };
                auto put = [&](int r, int d, float4 x, int e) {   // four values of a row, under 2^e
                    const float up = sign * __uint_as_float((uint32_t)(127 + e) << 23);
                    uint32_t hi[2], lo[2];
                    split(x.x * up, x.y * up, hi[0], lo[0]);
                    split(x.z * up, x.w * up, hi[1], lo[1]);
                    uint8_t *to = q_tile + (d >> 6) * (128 * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + 2 * (d & 7);
                    *reinterpret_cast<uint2 *>(to) = make_uint2(hi[0], hi[1]);
                    if constexpr (NT == 2) *reinterpret_cast<uint2 *>(to + C::kTerm) = make_uint2(lo[0], lo[1]);
                };
                auto greatest = [](float4 x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); };
                constexpr int NL = (D + 127) / 128, kPer = D / 4;   // pieces of four values
                if constexpr (!HALF) wait(meta.q_raw, n_item & 1);   // (as they are, each row in the 128-byte places that its terms will have)
                constexpr int kRows = NL == 1 ? 8 : 4;   // at a time
#pragma unroll 1
                for (int j0 = 0; j0 < 32; j0 += kRows) {
                    float4 x[kRows][NL];
                    float most[kRows];
#pragma unroll
                    for (int j = 0; j < kRows; j++) {
                        const int r = 32 * quarter + j0 + j, i = token_of(p, row0 + r);
                        const int64_t at = (int64_t)(q0 + i) * p.q_stride + (int64_t)(kvh * p.group + row0 + r - i * p.group) * D;
#pragma unroll
                        for (int c = 0; c < NL; c++) {
                            const int piece = 32 * c + lane, place = piece >> 3;
                            x[j][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (D % 128 != 0 && piece >= kPer) continue;
                            if constexpr (!HALF) {
                                x[j][c] = *reinterpret_cast<const float4 *>(q_tile + place / C::kPanels * C::kTerm + place % C::kPanels * (128 * 128) + r * 128 + ((piece & 7) << 4));
                            } else if (r < mine_rows) {
                                if (p.q_half) {
                                    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const __half *>(p.q) + at + 4 * piece);
                                    const float2 a = __half22float2(half2_of(w.x)), b = __half22float2(half2_of(w.y));
                                    x[j][c] = make_float4(a.x, a.y, b.x, b.y);
                                } else {
                                    x[j][c] = *reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + at + 4 * piece);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kRows; j++) {
                        most[j] = greatest(x[j][0]);
#pragma unroll
                        for (int c = 1; c < NL; c++) most[j] = fmaxf(most[j], greatest(x[j][c]));
                    }
                    // (an exchange at a time of all rows: the warp-wide maximum as one instruction took 440 clocks a row)
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                        for (int j = 0; j < kRows; j++) most[j] = fmaxf(most[j], __shfl_xor_sync(0xFFFFFFFFu, most[j], o));
#pragma unroll
                    for (int j = 0; j < kRows; j++) {
                        const int r = 32 * quarter + j0 + j, e = power_of(most[j]);
#pragma unroll
                        for (int c = 0; c < NL; c++)
                            if (D % 128 == 0 || 32 * c + lane < kPer) put(r, 128 * c + 4 * lane, x[j][c], e);
                        // (never 0, which would make a NaN of a masked score's -infinity: products are below 2^35, those of the smallest normal factor as good as 0)
                        if (lane == j0 + j) sc = fmaxf(row_scale * __uint_as_float((uint32_t)(127 - e) << 23), 1.17549435e-38f);
                    }
                }
                async_fence();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(meta.q_full[C::kQSets == 2 ? n_item & 1 : 0][tq]));
            }
            float m = -INFINITY, l = 0.0f;
#pragma unroll 1
            for (int i = 0; i < tiles; i++, n_tile++) {
                const int sb = NQ == 2 ? tq : (int)(n_tile & 1);
                const uint32_t s_phase = NQ == 2 ? n_tile & 1 : (n_tile >> 1) & 1, t_s = t_lane + C::kS * sb;
                const int pos0 = (it.tile0 + i) * TP, all_to = it.all_to, all_from = it.all_from, rows_to = it.rows_to[tq], rows_from = it.rows_from[tq];
                const uint32_t tile_no = n_all - it.all + i;
                bool masked = (pos0 + TP > rows_to) | (pos0 < rows_from);
                const bool look = !kQuant && ((pos0 + TP > all_to) | (pos0 < all_from));
                wait(meta.s_full[sb], s_phase);
                tc_after();
                const uint32_t there = *reinterpret_cast<volatile uint8_t *>(&meta.there[tile_no & 7]);
                masked |= there != (1u << kChunks) - 1u;
                float f = sc;
                if (!HALF && i > 0 && i % C::kRun == 0) {   // a run's sums leave tensor memory (its last products are behind the one before them, whose end s_full has told)
                    wait(meta.pv_done[tq], (n_tile - 1) & 1);
                    tc_after();
                    const size_t at = (size_t)blockIdx.x * R + 128 * tq + r_in;
                    add_run<D, C::kApart>(t_o, p.runs + at * D, p.run_tops + at, m, i > C::kRun);
                }
                // What is rarely done has code of its own, and no more of it than has to be: code that is jumped over, or met for the first time, is fetched at
                // the pace of thousands of clocks.
                if (p.softcap > 0.0f) {   // log2 scores in place of the products
                    soft_limit<TP>(t_s, sc, p.softcap, p.per_cap);
                    f = 1.0f;
                }
                uint32_t v[TP];
#pragma unroll
                for (int c = 0; c < TP; c += 32) tmem_load32(t_s + c, v + c);
                tmem_loaded();
                if (masked) {
                    const int lo = from - pos0, hi = behind - pos0;
#pragma unroll
                    for (int c = 0; c < TP; c += 32) {
                        const uint32_t ok = (there >> (c / 16)) & 3u;
                        const int a = max(lo - c, 0), b = hi - c;
                        const uint32_t seen = (a >= 32 ? 0u : 0xFFFFFFFFu << a) & (b >= 32 ? 0xFFFFFFFFu : b <= 0 ? 0u : 0xFFFFFFFFu >> (32 - b)) & ((ok & 1u ? 0xFFFFu : 0u) | (ok & 2u ? 0xFFFF0000u : 0u));
#pragma unroll
                        for (int j = 0; j < 32; j++) v[c + j] = seen & (1u << j) ? v[c + j] : 0xFF800000u;
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < TP; j += 8)
#pragma unroll
                    for (int k = 0; k < 4; k++) tops[k] = fmaxf(tops[k], fmaxf(__uint_as_float(v[j + 2 * k]), __uint_as_float(v[j + 2 * k + 1])));
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * f;
                if (__any_sync(0xFFFFFFFFu, top > m + kLetBe || (m == -INFINITY && top != -INFINITY))) {
                    const float now = fmaxf(m, top), corr = now == -INFINITY ? 1.0f : ex2(m - now);
                    m = now;
                    l *= corr;
                    if (i > 0) {
                        wait(meta.pv_done[tq], (n_tile - 1) & 1);
                        tc_after();
#pragma unroll 1
                        for (int c = 0; c < (C::kApart ? D + 128 : D); c += 16) {   // (apart: the second terms' 128 columns on; what is between does not matter)
                            uint32_t o[16];
                            tmem_load16(t_o + c, o);
                            tmem_loaded();
#pragma unroll
                            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                            tmem_store16(t_o + c, o);
                        }
                        tmem_stored();
                    }
                }
                // ---- values that are no numbers, where not all rows of the item see all positions: out of the tile (add_odd brings them to those that see them). Told
                // of before they go, since both tiles of rows look.
                if (look) {
                    const uint32_t h = 2 * tile_no + 1, slot = h % C::kSlots;
                    wait(meta.kv_full[slot], h / C::kSlots & 1);
                    uint8_t *at = smem + slot * C::kSlot + (r_in % TP) * 128;
                    constexpr int kFrom = 128 / TP;   // threads of a position, which take blocks of 64 values in turn
                    uint32_t any = 0;
#pragma unroll 1
                    for (int c = r_in / TP; c < C::kPanels; c += kFrom)
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            if (64 * c + 8 * u >= D) continue;
                            const uint4 w = *reinterpret_cast<const uint4 *>(at + c * (TP * 128) + ((u ^ (r_in & 7)) << 4));
                            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int k = 0; k < 4; k++) any |= ((ws[k] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;   // (an exponent of ones carries into the sign's place)
                        }
                    if (any) {
                        atomicOr(&meta.odd[0][n_item & 7], 1u);
                        atomicOr(&meta.odd[1][n_item & 7], 1u);
                        __threadfence_block();
                        for (int c = r_in / TP; c < C::kPanels; c += kFrom)
                            for (int u = 0; u < 8; u++) {
                                uint4 *w = reinterpret_cast<uint4 *>(at + c * (TP * 128) + (u << 4));
                                uint4 x = *w;
                                const bool b0 = take_out(x.x), b1 = take_out(x.y), b2 = take_out(x.z), b3 = take_out(x.w);
                                if (b0 || b1 || b2 || b3) *w = x;
                            }
                    }
                    // (whoever took them out: a thread of the other tile of rows may have, and this one's products may be asked for before that thread's fence)
                    async_fence();
                    __syncwarp();
                }
                // (one tile of rows: the products of two tiles may be in flight, which a parity does not tell apart behind the last one)
                if (NQ == 1 && i > 0 && i == tiles - 1) wait(meta.pv_done[tq], (n_tile - 1) & 1);
                const float less = (m == -INFINITY ? 0.0f : -m) + (HALF ? kUpLog2 : 0.0f);
                uint64_t sum[2] = {0, 0};
                const uint64_t ff = pair(f, f), ll = pair(less, less);
#pragma unroll
                for (int c = 0; c < TP; c += 16) {   // (16 at a time: registers)
                    uint32_t w[NT * 8];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        uint64_t x = fma2(pair(__uint_as_float(v[c + j]), __uint_as_float(v[c + j + 1])), ff, ll);
                        float a, b;
                        // (the exponential unit takes a warp eight clocks a value, as long as the products of one tile of rows: some go another way)
                        if (HALF && j % 8 < kPolyOf8) {
                            x = exp2_poly(x);
                            unpair(x, a, b);
                        } else {
                            unpair(x, a, b);
                            a = ex2(a), b = ex2(b);
                            if (!HALF) a *= kUp, b *= kUp;   // (in the exponent it would take bits of the greatest ones)
                            x = pair(a, b);
                        }
                        if constexpr (HALF) w[j / 2] = bits(__floats2half2_rn(a, b));
                        else split(a, b, w[j / 2], w[8 + j / 2]);
                        sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], x);
                    }
                    // (of 32 scores first terms in 16 columns, then the second ones: the place of scores that were read before)
                    tmem_store8(t_s + (HALF ? c / 2 : (c & ~31) + (c & 16) / 2), w);
                    if constexpr (!HALF) tmem_store8(t_s + (c & ~31) + 16 + (c & 16) / 2, w + 8);
                    if (c + 16 == TP / 2) {   // the first half's products begin
                        tmem_stored();
                        tc_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(bar(meta.p_half[sb]));
                    }
                }
                {
                    float a, b;
                    unpair(add2(sum[0], sum[1]), a, b);
                    l += a + b;
                }
                tmem_stored();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(meta.p_full[sb]));
            }

            // ---- the row's factor, and its outputs, whole sectors at a time
            const int kvh = it.kvh, q0 = it.q0, row0 = it.block * R + 128 * tq, mine_rows = min(128, it.n_rows - 128 * tq), tile0 = it.tile0;
            const float all = l * (1.0f / kUp);
            float out_f = 1.0f / kUp;
            const bool whole = it.whole;
            float *part = p.part + ((size_t)blockIdx.x * 2 + it.begins) * R * (D + 2);
            if (whole) {
                float lw = all, keep = 1.0f;
                if (p.sinks) {
                    const int rr = row0 + min(r_in, mine_rows - 1);   // (again below: registers)
                    const float sink = p.sinks[kvh * p.group + rr - token_of(p, rr) * p.group] * 1.44269504f, t = fmaxf(m, sink);
                    keep = m == -INFINITY ? 0.0f : exp2f(m - t);
                    lw = lw * keep + (sink == -INFINITY ? 0.0f : sink == t ? 1.0f : exp2f(sink - t));
                }
                out_f *= lw == 0.0f ? 0.0f : keep / lw;
            } else if (r_in < mine_rows) {
                reinterpret_cast<float2 *>(part + R * D)[128 * tq + r_in] = make_float2(m, all);
            }
            wait(meta.pv_done[tq], (n_tile - 1) & 1);
            tc_after();
            if (*reinterpret_cast<volatile uint32_t *>(&meta.odd[tq][n_item & 7]) != 0) add_odd<CT, D, TP>(p, it, t_o, max(from, tile0 * TP), min(behind, (tile0 + tiles) * TP));
            const float *run = nullptr;   // the sums of the runs before
            float run_f = 0.0f;
            if (!HALF && tiles > C::kRun) {
                const size_t at = (size_t)blockIdx.x * R + 128 * tq + r_in;
                const float top = p.run_tops[at];
                run = p.runs + at * D, run_f = top == -INFINITY ? 0.0f : ex2(top - m);
            }
            const int rr = row0 + min(r_in, mine_rows - 1), token = token_of(p, rr);
            const int64_t to = (int64_t)(q0 + token) * p.out_stride + (int64_t)(kvh * p.group + rr - token * p.group) * D;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_load32(t_o + c, o);
                if constexpr (C::kApart) {
                    uint32_t rest[32];
                    tmem_load32(t_o + 128 + c, rest);
                    tmem_loaded();
#pragma unroll
                    for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(rest[j]));
                } else {
                    tmem_loaded();
                }
                if (r_in < mine_rows) {
                    if (!HALF || !whole) {
                        float *at = (whole ? static_cast<float *>(p.out) + to : part + (128 * tq + r_in) * D) + c;
                        const int wide = whole ? p.out_wide : 1;
                        if (!HALF && run) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                const float4 x = __ldcg(reinterpret_cast<const float4 *>(run + c + j));
                                o[j] = __float_as_uint(fmaf(x.x, run_f, __uint_as_float(o[j]))), o[j + 1] = __float_as_uint(fmaf(x.y, run_f, __uint_as_float(o[j + 1])));
                                o[j + 2] = __float_as_uint(fmaf(x.z, run_f, __uint_as_float(o[j + 2]))), o[j + 3] = __float_as_uint(fmaf(x.w, run_f, __uint_as_float(o[j + 3])));
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            uint32_t w[8];
#pragma unroll
                            for (int k = 0; k < 8; k++) w[k] = __float_as_uint(__uint_as_float(o[j + k]) * out_f);
                            store32(at + j, w, wide);
                        }
                    } else {
                        __half *at = static_cast<__half *>(p.out) + to + c;
#pragma unroll
                        for (int j = 0; j < 32; j += 16) {
                            uint32_t w[8];
#pragma unroll
                            for (int k = 0; k < 8; k++) w[k] = bits(__floats2half2_rn(__uint_as_float(o[j + 2 * k]) * out_f, __uint_as_float(o[j + 2 * k + 1]) * out_f));
                            store32(at + j, w, p.out_wide);
                        }
                    }
                }
                __syncwarp();
            }
            tc_before();
            rows_sync(tq);
            if (r_in == 0) meta.odd[tq][n_item & 7] = 0;
        }
    } else if (warp < C::kProduct) {
        // ===== keys and values into a ring of half tiles (keys, values in turn). f16: one warp, boxes of 64 values; the other one brings queries. 8 and 4 bits: a warp
        // has a quarter of the chunks of 16 positions
        if constexpr (C::kTrade) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kCopyRegs));
        // chunks of a warp, or warps of a chunk; tiles whose rows the lanes hold
        constexpr int kPart = kQuant && C::kCopies > kChunks ? C::kCopies / kChunks : 1, kMine = kQuant && kPart == 1 ? kChunks / C::kCopies : 1, kAhead = 32 / kChunks, kRows = kChunk / kPart;
        const int w = warp - C::kSoft, row_w = kRows * (w % kPart);   // its first row of a chunk
        int n_item = 0, n_tile = 0;
        Ring<kChunkItems> found;
        Ring<C::kSlots> to_slot;
        // (also where others have given up: a copy in flight has to land before the block ends)
        auto landed = [&](uint32_t full, uint32_t parity) {
            const long long t0 = clock64();
            while (!bar_try(full, parity) && clock64() - t0 <= kWaitLimit) __nanosleep(32);
        };
        auto tell_odd = [&](int item) {
            atomicOr(&meta.odd[0][item & 7], 1u);
            atomicOr(&meta.odd[1][item & 7], 1u);
        };
        int64_t pool_rows = 0;   // lane: of chunk lane % kChunks of tile i + lane / kChunks, -1: none
        constexpr int kPieces = RB / 16, kCopies = (kRows * kPieces + 31) / 32;
        for (;; n_item++, found.next()) {
            wait(meta.item_full[found.at], found.turn);
            // (read where it is wanted, where registers are few)
            std::conditional_t<KT == 2, const ChunkItem, const volatile ChunkItem &> it = meta.item[found.at];
            if (!it.goes_on || *gave_up) break;
            auto done = [&] {
                __syncwarp();
                if (lane == 0) bar_arrive(bar(meta.item_empty[found.at]));
            };
            if ((kQuant || w == 1) && (!HALF || as_they_are)) {
                // The item's queries, into the place of the last but one's (f32: of the last one's): f16 as the products take them; f32 for the softmax to divide into terms, each
                // row in the 128-byte places that its terms will have. Tiles of 128 rows as boxes, others 16 bytes a lane.
                const int set = C::kQSets == 2 ? n_item & 1 : 0;
                wait_idle(meta.q_empty[set], ((C::kQSets == 2 ? n_item >> 1 : n_item) & 1) ^ 1);
                constexpr int kBytes = HALF ? 2 : 4, kPer = D * kBytes / 16, kPlaces = (D * kBytes + 127) / 128, kWarps = kQuant ? C::kCopies : 1, kAll = 128 * kPer / (32 * kWarps);
                auto place_at = [](int place) { return HALF ? place * (128 * 128) : place / C::kPanels * C::kTerm + place % C::kPanels * (128 * 128); };
                const uint32_t to_set = base + C::kQ + set * C::kQSet, full = HALF ? bar(meta.q_full[set][0]) : bar(meta.q_raw);
                uint32_t boxed = 0;   // bytes that come in boxes
                for (int t = 0; t < NQ; t++)
                    if (p.q_boxes && it.n_rows >= 128 * (t + 1)) boxed += kPlaces * 128 * 128;
                const bool tells = !kQuant || w == 0;
                if (tells && lane == 0 && boxed > 0) asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(full), "r"(boxed) : "memory");
                __syncwarp();
#pragma unroll 1
                for (int t = 0; t < NQ; t++) {
                    const int rows = it.n_rows - 128 * t, first = it.block * R + 128 * t;
                    if (rows <= 0) break;
                    if (p.q_boxes && rows >= 128) {
                        if (tells && lane < kPlaces)
                            asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                         ::"r"(to_set + t * C::kQTile + place_at(lane)), "l"(&p.q_map), "r"(128 / kBytes * lane), "r"(it.kvh * p.group), "r"(it.q0 + token_of(p, first)), "r"(full) : "memory");
                        continue;
                    }
#pragma unroll 4
                    for (int j = 0; j < kAll; j++) {
                        const int c = lane + 32 * ((kQuant ? w : 0) + kWarps * j), r = c / kPer, piece = c % kPer, g = first + r, i = token_of(p, g);
                        const bool there = r < rows;
                        const uint8_t *src = static_cast<const uint8_t *>(p.q) + ((int64_t)(it.q0 + i) * p.q_stride + (int64_t)(it.kvh * p.group + g - i * p.group) * D) * kBytes + 16 * piece;
                        copy16(to_set + t * C::kQTile + place_at(piece >> 3) + r * 128 + (((piece & 7) ^ (HALF ? r & 7 : 0)) << 4), there ? static_cast<const void *>(src) : p.q, there);
                    }
                }
                copies_commit();
                if constexpr (!kQuant) {
                    copies_wait<0>();
                    async_fence();
                    __syncwarp();
                    if (lane == 0) bar_arrive(full);
                }
            }
            if (!kQuant && w == 1) {
                done();
                continue;
            }
            const int32_t *table = p.table + (size_t)it.s * p.table_width;
            auto looked_at = [&](int i) { return (it.tile0 + i) * TP + TP > it.all_to || (it.tile0 + i) * TP < it.all_from; };
            auto find_rows = [&](int i) -> int64_t {
                const int tile = i + lane / kChunks, position = (it.tile0 + tile) * TP + lane % kChunks * kChunk;
                if (tile >= it.all || position >= it.len) return -1;
                const int page = table[position / p.page_size];
                return page < 0 || page >= p.n_pages ? -1 : ((int64_t)page * p.n_kv + it.kvh) * p.page_size + position % p.page_size;
            };
            // of tile i: its rows, and which chunks there are, for the softmax
            auto begin_tile = [&](int i) {
                if (i % kAhead == 0) pool_rows = find_rows(i);
                const uint32_t there = __ballot_sync(0xFFFFFFFFu, pool_rows >= 0) >> (kChunks * (i % kAhead)) & ((1u << kChunks) - 1u);
                if (w == 0 && lane == 0) meta.there[n_tile & 7] = (uint8_t)there;
                n_tile++;
            };
            auto row_of = [&](int i, int m) { return __shfl_sync(0xFFFFFFFFu, pool_rows, kChunks * (i % kAhead) + w / kPart * kMine + m); };
            if constexpr (!kQuant) {
                // a half tile is TP / box_rows boxes for each 64 values, a lane each
                const int per = p.box_rows / kChunk, boxes = TP / p.box_rows, box = lane / C::kPanels, panel = lane % C::kPanels;
#pragma unroll 1
                for (int i = 0; i < it.all; i++) {
                    begin_tile(i);
                    const int64_t row = __shfl_sync(0xFFFFFFFFu, pool_rows, kChunks * (i % kAhead) + min(box * per, kChunks - 1));
                    const int y = row < 0 ? p.pool_rows : (int)row;
#pragma unroll 1
                    for (int kv = 0; kv < 2; kv++) {
                        wait_idle(meta.kv_empty[to_slot.at], to_slot.turn ^ 1);
                        const uint32_t full = bar(meta.kv_full[to_slot.at]);
                        if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "r"((uint32_t)C::kSlot) : "memory");
                        __syncwarp();
                        if (box < boxes)
                            asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                                         ::"r"(base + to_slot.at * C::kSlot + panel * (TP * 128) + box * p.box_rows * 128), "l"(kv ? &p.v_map : &p.k_map), "r"(64 * panel), "r"(y), "r"(full) : "memory");
                        to_slot.next();
                    }
                }
            } else {
                // 8 and 4 bits: quants and scales of a warp's chunks come asynchronously, two half tiles ahead, and are unpacked to f16. (Through registers the loads' own
                // took so many that others went to level 2.) What is not there has a scale of zero.
                constexpr int SB = scale_bytes_of(CT, D);
                const int half_tiles = 2 * it.all;
                uint8_t *raw_mem = smem + C::kRawAt + w * kMine * (C::kRawChunk / kPart);
                const uint32_t raw_at = base + C::kRawAt + w * kMine * (C::kRawChunk / kPart);
                uint32_t there = 0;   // kMine bits of a half tile, the last asked for lowest
                auto ask = [&](int t, int raw) {
                    const int i = t >> 1;
                    if ((t & 1) == 0) begin_tile(i);
#pragma unroll
                    for (int m = 0; m < kMine; m++) {
                        const int64_t chunk_row = row_of(i, m), row0 = chunk_row + row_w;
                        there = there << 1 | (uint32_t)(chunk_row >= 0);
                        if (chunk_row < 0) continue;
                        const uint8_t *from = (t & 1 ? p.v : p.k) + row0 * RB + 16 * lane;
                        const uint32_t to = raw_at + raw * C::kRaw + m * C::kRawChunk + 16 * lane;
#pragma unroll
                        for (int j = 0; j < kCopies; j++)
                            if (kRows * kPieces % 32 == 0 || lane + 32 * j < kRows * kPieces) copy16(to + 512 * j, from + 512 * j, true);
                        if (lane < SB / kPart) copy16(to + kRows * RB, reinterpret_cast<const uint8_t *>(t & 1 ? p.v_scale : p.k_scale) + row0 * SB + 16 * lane, true);
                    }
                };
                Ring<C::kRaws> raw;
                bool beyond = false;
                ask(0, 0);
                copies_commit();
                ask(1, 1);
                copies_commit();
#pragma unroll 1
                for (int t = 0; t < half_tiles; t++) {
                    const int i = t >> 1;
                    if (t + 2 < half_tiles) ask(t + 2, raw.at == 0 ? 2 : raw.at - 1);
                    else there <<= kMine;
                    copies_commit();
                    copies_wait<2>();
                    const bool look = (t & 1) && looked_at(i);
                    bool bad = false;
                    __syncwarp();
                    wait_idle(meta.kv_empty[to_slot.at], to_slot.turn ^ 1);
#pragma unroll 1
                    for (int m = 0; m < kMine; m++) {
                        const int chunk = w / kPart * kMine + m, left = there >> (3 * kMine - 1 - m) & 1 ? it.len - ((it.tile0 + i) * TP + chunk * kChunk + row_w) : 0;
                        const int unseen = KT == 2 ? it.any_from - ((it.tile0 + i) * TP + chunk * kChunk + row_w) : 0;
                        uint8_t *chunk_at = smem + to_slot.at * C::kSlot + chunk * (kChunk * 128) + row_w * 128;
                        const uint8_t *from = raw_mem + raw.at * C::kRaw + m * C::kRawChunk;
                        uint4 x[kCopies];
                        uint32_t d[kCopies];
#pragma unroll
                        for (int j = 0; j < kCopies; j++) {
                            const int c = lane + 32 * j, row = c / kPieces;
                            x[j] = make_uint4(0u, 0u, 0u, 0u), d[j] = 0;
                            if (kRows * kPieces % 32 != 0 && c >= kRows * kPieces) continue;
                            x[j] = *reinterpret_cast<const uint4 *>(from + 16 * c);
                            d[j] = *reinterpret_cast<const uint16_t *>(from + kRows * RB + row * SB + 2 * (c % kPieces / (CT == KRK_CUDA_KV_Q8 ? 2 : 1)));
                        }
#pragma unroll
                        for (int j = 0; j < kCopies; j++) {
                            const int c = lane + 32 * j, row = c / kPieces, pc = c % kPieces;
                            const uint32_t words[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
                            const uint32_t scale = row < left ? d[j] : 0u;
                            const __half2 s2 = half2_of(scale * 0x10001u);
                            // (two terms: a scale that may take a value beyond f16, of a position that some row sees)
                            if constexpr (KT == 2) beyond |= (scale & 0x7FFFu) > (CT == KRK_CUDA_KV_Q8 ? 0x5FFFu : 0x6FFFu) && (scale & 0x7C00u) != 0x7C00u && row >= unseen;
                            constexpr int kUnits = CT == KRK_CUDA_KV_Q8 ? 2 : 4;   // of eight values
                            uint32_t y[4 * kUnits], rest[KT == 2 ? 4 * kUnits : 1];
                            auto times = [&](int k, uint32_t quants) {   // (what rounds off a product is exact, and has few bits)
                                const __half2 x = __hmul2(half2_of(quants), s2);
                                y[k] = bits(x);
                                if constexpr (KT == 2) rest[k] = bits(__hfma2(half2_of(quants), s2, __hneg2(x)));
                            };
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                if constexpr (CT == KRK_CUDA_KV_Q8) {
                                    const uint32_t u = words[k] ^ 0x80808080u;
                                    times(2 * k, halves<0, 1>(u, 0x64806480u));
                                    times(2 * k + 1, halves<2, 3>(u, 0x64806480u));
                                } else {
                                    const uint32_t u = words[k] & 0x0F0F0F0Fu, u2 = (words[k] >> 4) & 0x0F0F0F0Fu;
                                    times(2 * k, halves<0, 1>(u, 0x64086408u));
                                    times(2 * k + 1, halves<2, 3>(u, 0x64086408u));
                                    times(8 + 2 * k, halves<0, 1>(u2, 0x64086408u));
                                    times(8 + 2 * k + 1, halves<2, 3>(u2, 0x64086408u));
                                }
                            }
                            if (look) {
#pragma unroll
                                for (int k = 0; k < 4 * kUnits; k++) {
                                    bad |= take_out(y[k]);
                                    if constexpr (KT == 2) take_out(rest[k]);
                                }
                            }
                            if (kRows * kPieces % 32 != 0 && c >= kRows * kPieces) continue;
#pragma unroll
                            for (int k = 0; k < kUnits; k++) {
                                const int unit = kUnits * pc + k;
                                uint8_t *to = chunk_at + (unit >> 3) * (TP * 128) + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
                                *reinterpret_cast<uint4 *>(to) = make_uint4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
                                if constexpr (KT == 2) *reinterpret_cast<uint4 *>(to + C::kSlotTerm) = make_uint4(rest[4 * k], rest[4 * k + 1], rest[4 * k + 2], rest[4 * k + 3]);
                            }
                        }
                    }
                    if (bad) tell_odd(n_item);
                    async_fence();
                    __syncwarp();
                    if (lane == 0) {
                        if (t == 0 && (!HALF || as_they_are)) bar_arrive(HALF ? bar(meta.q_full[0][0]) : bar(meta.q_raw));   // (their copies were asked for before the second half tile's)
                        bar_arrive(bar(meta.kv_full[to_slot.at]));
                    }
                    to_slot.next();
                    raw.next();
                }
                copies_wait<0>();
                if (KT == 2 && beyond) meta.beyond = 1;
            }
            done();
        }
        // (what others, having given up, have not waited for)
        if (*gave_up && !kQuant && w == 0)
            for (int i = 0; i < C::kSlots; i++) landed(bar(meta.kv_full[i]), i < to_slot.at ? to_slot.turn : to_slot.turn ^ 1);
        if (*gave_up && w == (kQuant ? 0 : 1) && n_item > 0 && (!HALF || as_they_are))
            landed(HALF ? bar(meta.q_full[C::kQSets == 2 ? (n_item - 1) & 1 : 0][0]) : bar(meta.q_raw), (C::kQSets == 2 ? (n_item - 1) >> 1 : n_item - 1) & 1);
    } else {
        if constexpr (C::kTrade) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
        if (warp == C::kProduct) {
            // ===== products, of the two tiles of rows in turn: while one is in its softmax the other one's run. (A warp each: both came to be in their softmax, and
            // both waited for products, at the same time.)
            const uint32_t elected = elected_lane();
            constexpr uint32_t qk = (1u << 4) | (uint32_t)(TP >> 3) << 17 | (128u >> 4) << 24, pv = (1u << 4) | 1u << 16 | (uint32_t)(D >> 3) << 17 | (128u >> 4) << 24;
            const uint32_t rows = desc_lo(base + C::kQ, 16), slots_k = desc_lo(base, 16), slots_v = desc_lo(base, TP * 128), t_o = tmem + C::kO;
            uint32_t n_tile[2] = {0, 0}, n_item = 0;   // n_tile: of a tile of rows
            Ring<kChunkItems> found;
            Ring<C::kSlots> keys, values;   // half tiles 2 i and 2 i + 1
            values.next();
            auto free = [&](Ring<C::kSlots> &r) {
                products_commit(bar(meta.kv_empty[r.at]), elected);
                r.next(), r.next();
            };
            auto place_of = [&](int q, uint32_t t) { return NQ == 2 ? (uint32_t)q : t & 1; };
            uint32_t set = 0, rows_set = rows, q_turns = 0;   // of the queries; q_turns: bit 2 set + q, of those that the softmax brings
            auto scores = [&](int q, uint32_t t) {   // of the t-th tile of all
                const uint32_t at = slots_k + keys.at * (C::kSlot >> 4), d = tmem + C::kS * place_of(q, t);
#pragma unroll
                for (int term = NT + KT - 2; term >= 0; term--)   // (those with second terms first: sums lose last places of what they are by then; both second terms' is left out, 2^-22)
#pragma unroll
                    for (int c = 0; c < D; c += 64) {
                        const uint32_t a = rows_set + q * (C::kQTile >> 4) + (term == 1 ? C::kTerm >> 4 : 0) + (c >> 6) * (128 * 128 >> 4),
                                       b = at + (term == 2 ? C::kSlotTerm >> 4 : 0) + (c >> 6) * (TP * 128 >> 4);
                        const uint32_t onto = term < NT + KT - 2 || c > 0;
                        if (D - c >= 64) products_k<4>(d, a, b, qk, onto, elected);
                        else products_k<2>(d, a, b, qk, onto, elected);
                    }
                products_commit(bar(meta.s_full[place_of(q, t)]), elected);
            };
            auto sums = [&](int q, uint32_t t, bool onto) {
                const uint32_t at = slots_v + values.at * (C::kSlot >> 4), from = tmem + C::kS * place_of(q, t), phase = (NQ == 2 ? t : t >> 1) & 1;
#pragma unroll
                for (int c = 0; c < TP; c += 32) {
                    if (c == 0) {
                        wait(meta.p_half[place_of(q, t)], phase);
                        tc_after();
                    } else if (c == TP / 2) {
                        wait(meta.p_full[place_of(q, t)], phase);
                        tc_after();
                    }
                    if constexpr (C::kApart) {
                        products_p<1>(t_o, from + c, at + c * 8, pv, onto || c > 0, elected);
                        products_p<1>(t_o + 128, from + c + 16, at + c * 8, pv, onto || c > 0, elected);
                        products_p<1>(t_o + 128, from + c, at + (C::kSlotTerm >> 4) + c * 8, pv, 1u, elected);
                    } else {
                        products_p<NT>(t_o + 128 * q, from + c * NT / 2, at + c * 8, pv, onto || c > 0, elected);
                    }
                }
                products_commit(bar(meta.pv_done[q]), elected);
            };
            auto onto = [&](int i) { return HALF ? i > 0 : i % C::kRun != 0; };
            auto keys_there = [&] { wait(meta.kv_full[keys.at], keys.turn); };
            auto values_there = [&] { wait(meta.kv_full[values.at], values.turn); };
            for (;; found.next()) {
                wait(meta.item_full[found.at], found.turn);
                const int goes_on = meta.item[found.at].goes_on, all = meta.item[found.at].all, n[2] = {meta.item[found.at].tiles[0], NQ == 2 ? meta.item[found.at].tiles[1] : 0};
                __syncwarp();
                if (lane == 0) bar_arrive(bar(meta.item_empty[found.at]));
                if (!goes_on || *gave_up) break;
                set = C::kQSets == 2 ? n_item & 1 : 0, rows_set = rows + set * (C::kQSet >> 4);
                keys_there();
#pragma unroll
                for (int q = 0; q < NQ; q++)
                    if (n[q] > 0) {
                        if (as_they_are) {
                            if (q == 0) wait(meta.q_full[set][0], (C::kQSets == 2 ? n_item >> 1 : n_item) & 1);
                        } else {
                            wait_idle(meta.q_full[set][q], q_turns >> (2 * set + q) & 1);
                            q_turns ^= 1u << (2 * set + q);
                        }
                        tc_after();
                        scores(q, n_tile[q]);
                    }
                free(keys);
                if (all == 1) products_commit(bar(meta.q_empty[set]), elected);
#pragma unroll 1
                for (int i = 0; i < all; i++) {
                    const bool more = i + 1 < all;
                    if constexpr (NQ == 1) {
                        if (more) {
                            keys_there();
                            tc_after();
                            scores(0, n_tile[0] + i + 1);
                            free(keys);
                            if (i + 2 == all) products_commit(bar(meta.q_empty[set]), elected);
                        }
                        values_there();
                        sums(0, n_tile[0] + i, onto(i));
                    } else {
                        values_there();
#pragma unroll
                        for (int q = 0; q < NQ; q++) {
                            if (i < n[q]) sums(q, n_tile[q] + i, onto(i));
                            if (q == 0 && more) keys_there();
                            if (i + 1 < n[q]) scores(q, n_tile[q] + i + 1);
                        }
                        if (more) free(keys);
                        if (i + 2 == all) products_commit(bar(meta.q_empty[set]), elected);
                    }
                    free(values);
                }
                n_item++;
#pragma unroll
                for (int q = 0; q < NQ; q++) n_tile[q] += n[q];
            }
        } else if (warp == C::kFinder) {
            // ===== items
            Walk walk;
            walk.start(p);
            if (!p.whole && lane == 0) p.shared[blockIdx.x].parts = 0;
            Ring<kChunkItems> found;
            for (;; found.next()) {
                const bool more = walk.template next<true>(p);
                wait_idle(meta.item_empty[found.at], found.turn ^ 1);
                if (*gave_up) break;
                if (lane == 0) {
                    ChunkItem &it = meta.item[found.at];
                    it.goes_on = more;
                    if (more) {
                        const ChunkSeq &q = walk.now;
                        const int first = walk.block * R, last = first + walk.n_rows - 1;
                        it.q0 = q.q0, it.len = q.len, it.before = q.before, it.s = walk.s, it.kvh = walk.kvh, it.block = walk.block, it.n_rows = walk.n_rows, it.tile0 = walk.tile0, it.all = walk.tiles;
                        it.whole = walk.begins && walk.ends, it.begins = walk.begins;
                        it.all_to = min(q.len, q.before + token_of(p, first) + 1), it.all_from = p.window > 0 ? q.before + token_of(p, last) - p.window + 1 : 0;
                        it.any_from = p.window > 0 ? q.before + token_of(p, first) - p.window + 1 : 0;
                        // tiles that rows of the first tile of rows see: they end earlier
                        const int end = min(q.len, q.before + token_of(p, min(last, first + 127)) + 1);
                        it.tiles[0] = min(walk.tiles, max((end + TP - 1) / TP - walk.tile0, 1));
                        it.tiles[1] = walk.n_rows > 128 ? walk.tiles : 0;
                        for (int t = 0; t < 2; t++) {
                            it.rows_to[t] = min(q.len, q.before + token_of(p, min(last, first + 128 * t)) + 1);
                            it.rows_from[t] = p.window > 0 ? q.before + token_of(p, min(last, first + 128 * t + 127)) - p.window + 1 : 0;
                        }
                        if (walk.parts > 0) walk.note(p);
                    }
                    bar_arrive(bar(meta.item_full[found.at]));
                }
                __syncwarp();
                if (!more) break;
            }
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (KT == 2 && tid == 0) p.beyond[blockIdx.x] = meta.beyond;
    if (warp == C::kProduct && *gave_up) {   // (nobody waits any more, so this is the last word on it)
        products_commit(bar(meta.drained), elected_lane());
        const long long t0 = clock64();
        while (!bar_try(bar(meta.drained), 0) && clock64() - t0 <= kWaitLimit) __nanosleep(32);
    }
    if (warp == C::kProduct) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <int D, int CT, bool HALF>
int launch_chunk_one(const ChunkParams &p, cudaStream_t st) {
    using C = Chunk<D, HALF ? 1 : 2, CT>;
    static std::atomic<uint64_t> ready{0};   // devices whose limit of shared memory is raised for this kernel
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !((ready.load(std::memory_order_acquire) >> dev) & 1)) {
        e = cudaFuncSetAttribute(attn_chunk_kernel<D, CT, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
        if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) {
        note_cuda_error(e);
        return KRK_CUDA_ELAUNCH;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&cfg, attn_chunk_kernel<D, CT, HALF>, p));
}
template <int CT, bool HALF>
int launch_chunk_type(const ChunkParams &p, int d, cudaStream_t st) {
    if constexpr (CT != KRK_CUDA_KV_F16 && !HALF)   // (two terms of queries, keys and values: no room for longer heads)
        return d == 64 ? launch_chunk_one<64, CT, HALF>(p, st) : d == 96 ? launch_chunk_one<96, CT, HALF>(p, st) : launch_chunk_one<128, CT, HALF>(p, st);
    else
    switch (d) {
    case 64: return launch_chunk_one<64, CT, HALF>(p, st);
    case 96: return launch_chunk_one<96, CT, HALF>(p, st);
    case 128: return launch_chunk_one<128, CT, HALF>(p, st);
    case 192: return launch_chunk_one<192, CT, HALF>(p, st);
    default: return launch_chunk_one<256, CT, HALF>(p, st);
    }
}

}   // namespace attn

int launch_attn_chunk_f16(const attn::ChunkParams &p, int head_dim, int half, cudaStream_t st);
int launch_attn_chunk_f16_half(const attn::ChunkParams &p, int head_dim, cudaStream_t st);
int launch_attn_chunk_q8(const attn::ChunkParams &p, int head_dim, int half, cudaStream_t st);
int launch_attn_chunk_q4(const attn::ChunkParams &p, int head_dim, int half, cudaStream_t st);

}   // namespace krk_cuda
