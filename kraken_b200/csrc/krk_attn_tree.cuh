// Attention of drafted tokens over a paged cache (krk_cuda_attention_tree): declarations shared by the kernel, which is
// instantiated per cache type in krk_attn_f16.cu / _q8.cu / _q4.cu, and the entry point in krk_attn_tree.cu.
//
//   out[r] = sum_p w_rp v_p / sum_p w_rp,   w_rp = exp(score_rp - max),   score = scale * q_r . k_p
//
// over the positions p that row r sees: all before its sequence's drafted tokens (inside the window), and of the drafted
// tokens those in its mask. A row is a (drafted token, query head) pair; the `group` query heads of a key head are rows of
// one product, so that a cached row is read once for all of them.
#pragma once

#include "krk_common.cuh"

namespace krk_cuda {
namespace attn {

constexpr int kWarps = 4;                 // of a CTA; each takes chunks of its own
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 16;                // positions of a step of a warp; pages hold whole chunks
constexpr int kTile = kChunk * kWarps;    // positions the warps of a CTA take together
constexpr int kWideRows = 64;             // the form on tcgen05 (krk_attn_wide.cuh): rows of a block, positions of a tile
constexpr int kWideTile = 128;
__host__ __device__ constexpr int tile_of(int r) { return r == kWideRows ? kWideTile : kTile; }
// Units of work: of a tile of a block of R rows of which `rows` are there, and of an item beside its tiles (its queries, the joining of sums, the
// fetching of code and data that nothing overlaps). About 0.6 us, measured with one item of one tile and one of 32 to a CTA, heads of 128 values in 8 bits
// (the form on tcgen05: in f16). For other head sizes and types the shares are only about as equal; no result depends on them.
__host__ __device__ constexpr int tile_units(int r, int rows) { return r == kWideRows ? (rows > 32 ? 4 : 3) : rows <= 8 ? 2 : 3; }
__host__ __device__ constexpr int setup_units(int r) { return r == kWideRows ? 26 : 14; }
constexpr int kWholeTiles = 8;            // up to so many tiles an item is not divided, see launch

// An item that several CTAs have parts of, noted by the second one of them: parts 0 elsewhere.
struct Shared {
    int parts, n_rows, kvh, row0;   // row0: of the item's first row among its key head's
    int q0, pad[3];
};
inline size_t shared_bytes(int grid) { return (size_t)grid * sizeof(Shared); }

struct Params {
    const float *q;
    float *out;
    int64_t q_stride, out_stride;         // floats from a token to the next
    const uint8_t *k, *v;
    const __half *k_scale, *v_scale;
    const int32_t *table;                 // [n_seq][table_width] pages
    const int32_t *q_start, *kv_len;
    const uint64_t *tree;
    const float *sinks;
    Shared *shared;                       // [grid]
    float *part;                          // [grid][2][R][D + 2]: see part_row
    int64_t n_pages;
    int table_width, page_size, max_len, n_seq, n_heads, n_kv, group, max_q, window, whole, grid;
    int pieces, piece_q;                  // a chunk of up to piece_q tokens is so many sequences of max_q; trees: 1 and 0
    float scale, softcap;
    int *status;                          // raised where a bounded wait gives up
    const int *only_if;                   // nothing is done where all only_ifs of them are 0; trees: null
    int only_ifs;
};
// Whether the launch has anything to do: the same for all threads of a block.
__device__ __forceinline__ bool called_for(const Params &p) {
    if (!p.only_if) return true;
    int any = 0;
    for (int i = threadIdx.x; i < p.only_ifs; i += blockDim.x) any |= p.only_if[i];
    return __syncthreads_or(any) != 0;
}

// The work, in the order of its units: sequences, their key heads, blocks of R rows (items), tiles of positions. The CTAs take equal
// shares of the units, whatever the lengths are, and a tile belongs to the CTA that has its first unit; where items are not
// divided (Params::whole) all of an item does. So at most a CTA's first and last items are shared with others; those leave partial
// sums, which a second kernel adds up in the order of the CTAs (the same bits every time; finding the items anew in that kernel took it 14 to 24 us).
// (With equal units for all tiles, and none for items, a CTA whose share was 40 items of one tile took four times as long as the others.)
struct Seq {
    int q0, n_q, len, before;   // first row of q, drafted tokens, positions that are looked at, positions before the drafted ones (may be negative, or beyond len)
    int blocks, tile0, tiles;   // blocks of rows; first tile that any row sees, tiles from there on (at least one where there are rows)
};
template <int R>
__device__ __forceinline__ Seq sequence(const Params &p, int s) {
    Seq q;
    int len;
    if (p.pieces == 1) {
        q.q0 = p.q_start[s];
        q.n_q = min(max(p.q_start[s + 1] - q.q0, 0), p.max_q);
        len = min(max(p.kv_len[s], 0), 1 << 30);
    } else {
        // sequence s is piece s % pieces of a chunk: what is behind it in the chunk is not there for it
        const int of = s / p.pieces, first = (s - of * p.pieces) * p.max_q, q0 = p.q_start[of], n_q = min(max(p.q_start[of + 1] - q0, 0), p.piece_q);
        q.q0 = q0 + first;
        q.n_q = min(max(n_q - first, 0), p.max_q);
        len = min(max(p.kv_len[of], 0), 1 << 30) - max(n_q - first - q.n_q, 0);
    }
    q.len = min(len, p.max_len);
    q.before = len - q.n_q;
    q.blocks = (q.n_q * p.group + R - 1) / R;
    const int first = p.window > 0 ? max(0, q.before - p.window) : 0;   // (the shallowest row is at `before`, or a position less where its mask is empty)
    q.tile0 = min(first, max(q.len - 1, 0)) / tile_of(R);
    q.tiles = max(1, (q.len + tile_of(R) - 1) / tile_of(R) - q.tile0);
    return q;
}
// Units of a full block of rows and of a sequence's last one, of a key head, of the sequence.
struct Cost {
    int full, last;
    int64_t head, all;
};
template <int R>
__device__ __forceinline__ Cost cost_of(const Params &p, const Seq &q) {
    Cost c;
    const int rows = q.n_q * p.group;
    c.full = setup_units(R) + q.tiles * tile_units(R, R);
    c.last = setup_units(R) + q.tiles * tile_units(R, rows - (q.blocks - 1) * R);
    c.head = q.blocks > 0 ? (int64_t)(q.blocks - 1) * c.full + c.last : 0;
    c.all = p.n_kv * c.head;
    return c;
}

// Units [first(b), first(b + 1)) are CTA b's.
__device__ __forceinline__ int64_t first_unit(int64_t total, int grid, int b) { return total * min(b, grid) / grid; }

// By a whole CTA of 128 threads or more: the number of all units, the CTAs that share them,
// and the sequence that CTA b's first one lies in (n_seq where it has none) with the units before that sequence.
struct Place {
    int64_t total, at, before;
    int grid, seq;
};
template <int R>
__device__ __forceinline__ Place find_place(const Params &p, int b) {
    __shared__ int64_t s_sum[kWarps];
    __shared__ int64_t s_before;
    __shared__ int s_found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Place r;
    r.total = 0;
    int64_t lo = 0, mine = 0;   // of this thread's sequence of the last 128
    auto scan = [&](int s0, int64_t base) {
        const int s = s0 + tid;
        mine = tid < kThreads && s < p.n_seq ? cost_of<R>(p, sequence<R>(p, s)).all : 0;
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31 && warp < kWarps) s_sum[warp] = upto;
        __syncthreads();
        int64_t all = 0;
        lo = base + upto - mine;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) lo += s_sum[w];
            all += s_sum[w];
        }
        __syncthreads();
        return all;
    };
    for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) r.total += scan(s0, r.total);
    r.grid = (int)max(min((int64_t)p.grid, r.total / tile_units(R, R)), (int64_t)1);   // (a share holds a tile's first unit, at least)
    r.at = first_unit(r.total, r.grid, b);
    if (tid == 0) {
        s_found = p.n_seq;
        s_before = r.total;
    }
    __syncthreads();
    int64_t base = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += kThreads) {
        if (p.n_seq > kThreads) base += scan(s0, base);   // (up to 128 sequences the first scan's values stand)
        if (r.at >= lo && r.at < lo + mine) {   // (none of a thread beyond the first 128)
            s_found = s0 + tid;
            s_before = lo;
        }
    }
    __syncthreads();
    r.seq = s_found;
    r.before = s_before;
    return r;
}

// The items of a CTA, in order.
template <int R>
struct Walk {
    int64_t at, end, in_seq, total;
    int grid, s;
    Seq sq;
    // of the current item; parts: see Shared, 0 where this CTA does not have its second part
    int kvh, block, n_rows, tile0, tiles, parts;
    bool begins, ends;
    __device__ __forceinline__ void start(const Params &p) {   // by the whole CTA
        const Place place = find_place<R>(p, blockIdx.x);
        at = place.at;
        total = place.total;
        grid = place.grid;
        end = first_unit(total, grid, blockIdx.x + 1);
        s = place.seq;
        in_seq = at - place.before;
        if (at < end) sq = sequence<R>(p, s);
    }
    __device__ __forceinline__ bool next(const Params &p) {
        while (at < end) {
            Cost cost = cost_of<R>(p, sq);
            while (in_seq >= cost.all) {   // (sequences without drafted tokens have no units)
                in_seq -= cost.all;
                sq = sequence<R>(p, ++s);
                cost = cost_of<R>(p, sq);
            }
            kvh = (int)(in_seq / cost.head);
            const int64_t in_head = in_seq - kvh * cost.head;
            block = (int)min(in_head / cost.full, (int64_t)(sq.blocks - 1));
            const int64_t from_unit = in_head - (int64_t)block * cost.full;
            n_rows = min(R, sq.n_q * p.group - block * R);
            const int per_item = block == sq.blocks - 1 ? cost.last : cost.full, w = tile_units(R, n_rows);
            const int64_t units = min(per_item - from_unit, end - at), item_at = at - from_unit;
            int from, upto;
            if (p.whole) {
                from = 0;
                upto = from_unit == 0 ? sq.tiles : 0;
            } else {
                from = ((int)max(from_unit - setup_units(R), (int64_t)0) + w - 1) / w;
                upto = ((int)max(from_unit + units - setup_units(R), (int64_t)0) + w - 1) / w;
            }
            at += units;
            in_seq += units;
            if (upto <= from) continue;
            begins = from == 0, ends = upto == sq.tiles;
            tile0 = sq.tile0 + from, tiles = upto - from;
            const int64_t first = item_at + setup_units(R);   // of the item's tiles
            parts = from > 0 && first_unit(total, grid, blockIdx.x - 1) <= first
                        ? (int)min((int64_t)grid, ((first + (int64_t)(sq.tiles - 1) * w + 1) * grid + total - 1) / total) - (int)blockIdx.x + 1 : 0;
            return true;
        }
        return false;
    }
    __device__ __forceinline__ void note(const Params &p) const {   // by one thread
        Shared it;
        it.parts = parts;
        it.n_rows = n_rows;
        it.kvh = kvh;
        it.row0 = block * R;
        it.q0 = sq.q0;
        it.pad[0] = it.pad[1] = it.pad[2] = 0;
        p.shared[blockIdx.x] = it;
    }
};

// Rows of partial sums of CTA b: place 0 its first item's, where that began before the CTA; place 1 its last item's, where that
// goes on behind it and place 0 is not it. A row: D sums, the maximum (log2 domain), the sum of weights.
template <int D, int R>
__device__ __forceinline__ float *part_row(const Params &p, int b, int place, int row) {
    return p.part + (((size_t)b * 2 + place) * R + row) * (D + 2);
}

// out = sums / weights, with the sink's weight among the latter. Nothing seen: zero.
__device__ __forceinline__ float norm_of(const Params &p, int head, float m, float l, float &keep) {
    keep = 1.0f;
    if (p.sinks) {
        const float sink = p.sinks[head] * 1.44269504f;
        const float top = fmaxf(m, sink);
        keep = m == -INFINITY ? 0.0f : exp2f(m - top);
        l = l * keep + (sink == -INFINITY ? 0.0f : sink == top ? 1.0f : exp2f(sink - top));
    }
    return l == 0.0f ? 0.0f : keep / l;
}

}   // namespace attn

int launch_attn_f16(const attn::Params &p, int head_dim, int rows, cudaStream_t st);
int launch_attn_q8(const attn::Params &p, int head_dim, int rows, cudaStream_t st);
int launch_attn_q4(const attn::Params &p, int head_dim, int rows, cudaStream_t st);
// The form on tcgen05: blocks of kWideRows rows, head sizes up to 128.
int launch_attn_wide_f16(const attn::Params &p, int head_dim, cudaStream_t st);
// CTAs that an SM holds at once
int attn_ctas_f16(int head_dim, int rows);
int attn_ctas_q8(int head_dim, int rows);
int attn_ctas_q4(int head_dim, int rows);

}   // namespace krk_cuda
