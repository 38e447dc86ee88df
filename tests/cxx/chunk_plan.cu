// How attention of chunks divides its work (ChunkWalk), on the host: every tile of every item belongs to one block of threads, parts of divided items are
// noted by the second one that has any, and copies, products and softmax agree on what is behind the rows.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "krk_attn_chunk.cuh"

using namespace krk_cuda;
using namespace krk_cuda::attn;

static int bad = 0, cases = 0, divided = 0;
static void check(bool ok, const char *what, int a = 0, int b = 0, int c = 0) {
    if (ok) return;
    if (bad++ < 20) std::printf("case %d: %s: %d %d %d\n", cases, what, a, b, c);
}

template <int R, int TP>
static void check_plan(const std::vector<int> &count, const std::vector<int> &len, int group, int n_kv, int window, int max_len, int max_q, int grid, int whole) {
    cases++;
    std::vector<int32_t> start(1, 0);
    for (int c : count) start.push_back(start.back() + c);
    ChunkParams p = {};
    p.q_start = start.data(), p.kv_len = len.data(), p.n_seq = (int)count.size(), p.group = group, p.n_kv = n_kv, p.window = window, p.max_len = max_len, p.max_q = max_q, p.grid = grid;
    p.whole = whole;
    divide_by(group, p.group_mul, p.group_shift);
    for (int64_t n : {0ll, 1ll, (long long)group - 1, (long long)group, 5ll * group - 1, 5ll * group, (1ll << 30), (1ll << 30) / group * group, (1ll << 30) / group * group - 1})
        check(token_of(p, (int)n) == n / group, "quotient", group, (int)n);
    std::vector<int64_t> before(1, 0);
    std::map<std::tuple<int, int, int>, std::vector<int>> owner;   // of an item's tiles
    for (int s = 0; s < p.n_seq; s++) {
        const ChunkSeq q = chunk_sequence<R>(p, s);
        const ChunkCost<R, TP> c = chunk_cost<R, TP>(p, q);
        check(q.blocks == 0 || c.head > 0, "no units", s);
        for (int b = 0; b + 1 < q.blocks; b++) check(c.prefix(b + 1) > c.prefix(b), "units fall", s, b);
        check(q.blocks == 0 || c.prefix(q.blocks - 1) + c.last == c.head, "units of a head", s);
        before.push_back(before.back() + n_kv * c.head);
        for (int h = 0; h < n_kv; h++)
            for (int b = 0; b < q.blocks; b++) {
                int t0, tiles;
                chunk_tiles<R, TP>(p, q, b, t0, tiles);
                check(tiles >= 1 && t0 >= 0 && (t0 + tiles) * TP < q.len + 2 * TP, "tiles", s, t0, tiles);
                // every position that one of the block's rows sees
                const int64_t rows = (int64_t)q.n_q * group;
                for (int64_t r : {(int64_t)b * R, std::min(rows, (int64_t)(b + 1) * R) - 1}) {
                    const int own = q.before + (int)(r / group), hi = std::min(own + 1, q.len), lo = window ? std::max(0, own - window + 1) : 0;
                    if (lo < hi) check(t0 * TP <= lo && hi <= (t0 + tiles) * TP, "what a row sees", s, b, (int)r);
                }
                owner[{s, h, b}] = std::vector<int>(tiles, -1);
            }
    }
    std::map<std::tuple<int, int, int>, int> notes;
    for (int cta = 0; cta < grid; cta++) {
        ChunkWalk<R, TP> w;
        w.total = before.back();
        w.share(p, cta);
        auto find = [&](int64_t u) {
            for (int s = 0; s < p.n_seq; s++)
                if (u >= before[s] && u < before[s + 1]) return s;
            return p.n_seq;
        };
        const int s0 = find(w.first_unit), s1 = find(w.behind_unit);
        const ChunkPlace none = {p.n_seq, 0, 0, 0};
        w.begin(p, s0 < p.n_seq ? w.place(p, s0, w.first_unit - before[s0]) : none, s1 < p.n_seq ? w.place(p, s1, w.behind_unit - before[s1]) : none, before[s0]);
        int items = 0;
        bool went_on = false;
        while (w.template next<true>(p)) {
            auto &o = owner[{w.s, w.kvh, w.block}];
            int t0, tiles;
            chunk_tiles<R, TP>(p, w.now, w.block, t0, tiles);
            check(w.tiles >= 1 && w.tile0 >= t0 && w.tile0 + w.tiles <= t0 + (int)o.size(), "part", cta, w.tile0, w.tiles);
            check(w.begins == (w.tile0 == t0) && w.ends == (w.tile0 + w.tiles == t0 + tiles), "ends of a part", cta);
            check(items == 0 || w.begins, "a later item that does not begin here", cta, items);
            check(!went_on, "an item behind one that goes on", cta);
            check(!(whole && !(w.begins && w.ends)), "divided", cta);
            went_on = !w.ends;
            for (int i = 0; i < w.tiles; i++) {
                check(o[w.tile0 - t0 + i] == -1, "a tile twice", cta, w.tile0 + i);
                o[w.tile0 - t0 + i] = cta;
            }
            check(w.parts == 0 || !w.begins, "parts of an item that begins here", cta);
            if (w.parts > 0) {
                check(notes.count({w.s, w.kvh, w.block}) == 0, "noted twice", cta);
                notes[{w.s, w.kvh, w.block}] = w.parts * 100000 + cta;
            }
            items++;
        }
    }
    for (auto &[item, o] : owner) {
        int parts = 1;
        for (size_t i = 0; i < o.size(); i++) {
            check(o[i] >= 0, "a tile that nobody has", std::get<0>(item), std::get<2>(item), (int)i);
            if (i > 0 && o[i] != o[i - 1]) {
                check(o[i] == o[i - 1] + 1, "parts of CTAs apart", o[i - 1], o[i]);
                parts++;
            }
        }
        divided += parts > 1;
        check(parts == 1 ? notes.count(item) == 0 : notes.count(item) == 1 && notes[item] == parts * 100000 + o[0] + 1, "note", parts, notes.count(item) ? notes[item] : -1, o[0]);
    }
}

template <int R, int TP>
static void all(std::mt19937 &rng) {
    auto number = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    auto log_number = [&](int hi) { return (int)std::exp(std::uniform_real_distribution<>(0.0, std::log(hi + 1.0))(rng)); };
    const int groups[] = {1, 2, 3, 4, 5, 7, 8, 16, 20, 64, 300};
    for (int i = 0; i < 4000; i++) {
        const int n = i % 10 == 0 ? number(129, 300) : log_number(20), most = i % 10 == 0 ? 4 : log_number(i % 3 ? 300 : 5000), context = number(0, 2) ? log_number(30000) : 0;
        std::vector<int> count, len;
        for (int s = 0; s < n; s++) {
            count.push_back(number(0, 3) ? number(0, most) : number(0, 1));
            len.push_back(number(0, 9) ? count.back() + (context ? number(0, context) : 0) : number(-5, most));   // now and then shorter than the rows
        }
        const int longest = std::max(1, *std::max_element(len.begin(), len.end()));
        const int max_len = number(0, 3) ? std::max(longest, log_number(60000)) : number(1, longest);
        const int window = number(0, 1) ? 0 : log_number(5000), grid = number(0, 3) ? 148 : number(1, 200);
        check_plan<R, TP>(count, len, groups[number(0, 10)], number(1, 8), window, max_len, number(0, 5) ? most : number(1, most), grid, number(0, 4) == 0);
    }
    check_plan<R, TP>({1}, {131072}, 4, 8, 0, 131072, 1, 148, 0);
    check_plan<R, TP>({1}, {1 << 30}, 1, 1, 0, 1 << 30, 1, 148, 0);
    check_plan<R, TP>({4096}, {12288}, 4, 8, 0, 12288, 4096, 148, 0);
    check_plan<R, TP>({100000}, {100000}, 8, 1, 1, 100000, 100000, 148, 0);
    check_plan<R, TP>({8192, 8192}, {300, 20000}, 8, 2, 0, 300, 8192, 148, 0);
}

int main() {
    std::mt19937 rng(5);
    all<256, 128>(rng);
    all<128, 64>(rng);
    std::printf("%d cases, %d divided items, %d wrong\n", cases, divided, bad);
    return bad != 0 || divided < 1000;
}
