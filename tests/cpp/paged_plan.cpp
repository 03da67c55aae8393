// The plan of the paged cache's attention of draft trees (csrc/paged_plan.h), over random batches on the host: each workgroup has an item
// of its own, every item a workgroup, and every row one that writes it; the
// workspace holds the sums of split row tiles. The sequences are a vector here, there a wavefront's lanes.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <numeric>
#include <random>
#include <vector>

#include "paged_plan.h"

using namespace gcq;

namespace {

struct Batch {
    int D, tile_rows, Hkv, G, window;
    int64_t slots;  // of a sequence
    std::vector<int> rows, past;
};
struct Seq {
    int s, tiles, row_tiles;
};
struct Item {
    int s, hk, row_tile, split, ns, first_unit;
};

struct Plan {
    std::vector<Item> items;
    int grid = 0, target = 0, chunk = 0;
    bool sorted = false;
};

Plan plan_of(const Batch & b) {
    Plan p;
    p.target = plan_target(b.D, b.tile_rows);
    std::vector<Seq> seqs;
    double u = 0.0, n = 0.0;
    int64_t n_rows = 0, max_rows = 0;
    for (size_t s = 0; s < b.rows.size(); s++) {
        const int64_t hi = std::min<int64_t>((int64_t) b.past[s] + b.rows[s], b.slots);
        const int64_t lo = b.window ? std::max<int64_t>(0, (int64_t) b.past[s] - b.window + 1) : 0;
        Seq q{(int) s, 0, (int) (((int64_t) b.rows[s] * b.G + b.tile_rows - 1) / b.tile_rows)};
        if (q.row_tiles && hi > lo) q.tiles = (int) ((hi + 31) / 32 - lo / 32);
        seqs.push_back(q);
        u += (double) q.row_tiles * q.tiles * b.Hkv, n += (double) q.row_tiles * b.Hkv;
        n_rows += b.rows[s], max_rows = std::max<int64_t>(max_rows, b.rows[s]);
    }
    // what is launched: no fewer than there can be items
    const int64_t tiles = b.Hkv * std::min<int64_t>(n_rows * b.G / b.tile_rows + std::min<int64_t>(b.rows.size(), n_rows),
                                                    b.rows.size() * ((max_rows * b.G + b.tile_rows - 1) / b.tile_rows));
    int64_t longest = b.slots / 32;
    if (b.window) longest = std::min<int64_t>(longest, (b.window + max_rows - 2) / 32 + 2);
    const int64_t most = longest <= 2 * kMinChunk ? 1 : (longest + kMinChunk - 1) / kMinChunk;
    p.grid = (int) std::min(tiles + p.target, tiles * most);

    const bool fill = b.rows.size() <= 64 && n < p.target && most > 1;
    const double cut = fill ? p.target : std::max(p.target - n, 0.5 * p.target);
    p.chunk = most == 1 ? 1 << 30 : plan_chunk(u, cut, kMinChunk);
    for (int turn = 0; fill && turn < 8; turn++) {
        int64_t items = 0;
        for (const Seq & q : seqs) items += (int64_t) q.row_tiles * splits(q.tiles, p.chunk);
        const double more = (double) b.Hkv * items / p.target;
        if (more <= 1.0) break;
        p.chunk = plan_longer(p.chunk, more);
    }
    if (fill && b.rows.size() > 1 && p.chunk > 32) {
        p.sorted = true;
        const auto length = [&](const Seq & q) {
            const int ns = splits(q.tiles, p.chunk);
            return q.row_tiles ? (q.tiles + ns - 1) / ns : -1;
        };
        std::stable_sort(seqs.begin(), seqs.end(), [&](const Seq & x, const Seq & y) { return length(x) > length(y); });
    }
    for (const Seq & q : seqs) {
        const int ns = splits(q.tiles, p.chunk);
        for (int hk = 0; hk < b.Hkv; hk++)
            for (int rt = q.row_tiles - 1; rt >= 0; rt--) {
                const int first = (int) p.items.size();
                for (int i = 0; i < ns; i++) p.items.push_back({q.s, hk, rt, i, ns, first});
            }
    }
    return p;
}

int turned_blocks = 0, over = 0, sorted = 0, failed = 0;

void report(const Batch & b, const char * what, int count, int grid) {
    if (failed++ >= 5) return;
    printf("%s: %d of a grid of %d; heads of %d, row tiles of %d, %d KV heads of %d heads, window %d:", what, count, grid, b.D, b.tile_rows, b.Hkv, b.G, b.window);
    for (size_t s = 0; s < std::min<size_t>(b.rows.size(), 8); s++) printf(" %d behind %d", b.rows[s], b.past[s]);
    printf("%s\n", b.rows.size() > 8 ? " .." : "");
}

void check(const Batch & b) {
    const Plan p = plan_of(b);
    const int n = (int) p.items.size();
    sorted += p.sorted, over += p.sorted && n > p.target;
    if (n > p.grid) report(b, "items past the grid", n - p.grid, p.grid);
    const int sums = (int) std::count_if(p.items.begin(), p.items.end(), [](const Item & it) { return it.ns > 1; });
    if (sums > std::min(p.grid, 2 * p.target)) report(b, "sums past the workspace", sums, p.grid);
    // (any grid that holds the items will do)
    std::vector<int> grids{p.grid, n};
    for (int more : {1, 77, 256, 300}) grids.push_back(n + more);
    for (int grid : grids) {
        std::vector<int> runs(n);
        for (int block = 0; block < grid; block++) {
            const int unit = unit_of(block, grid, p.sorted);
            turned_blocks += unit != block;
            if (unit < 0 || unit >= grid) report(b, "unit past the grid", unit, grid);
            else if (unit < n) runs[unit]++;
        }
        const int missing = (int) std::count_if(runs.begin(), runs.end(), [](int x) { return x != 1; });
        if (missing) report(b, "items not run once", missing, grid);
        // the splits of a row tile share its rows, row y to split y % ns's workgroup
        std::vector<std::vector<int>> rows(n);
        for (int block = 0; block < grid; block++) {
            const int unit = unit_of(block, grid, p.sorted);
            if (unit < 0 || unit >= n || !all_there(unit, p.items[unit].split, p.items[unit].ns, grid)) continue;
            const Item & it = p.items[unit];
            const int64_t all = (int64_t) b.rows[it.s] * b.G;
            auto & seen = rows[it.first_unit];
            seen.resize(std::min<int64_t>(b.tile_rows, all - (int64_t) it.row_tile * b.tile_rows));
            for (size_t y = it.split; y < seen.size(); y += it.ns) seen[y]++;
        }
        int lost = 0;
        for (const Item & it : p.items)
            if (it.split == 0) {
                const auto & seen = rows[it.first_unit];
                lost += seen.empty() || std::any_of(seen.begin(), seen.end(), [](int x) { return x != 1; });
            }
        if (lost) report(b, "row tiles not written once", lost, grid);
    }
}

}  // namespace

int main() {
    // several sequences of long splits, and batches of nearly as many row tiles as are resident
    check({128, 16, 8, 4, 0, 1 << 17, {4, 4}, {130000, 5000}});
    check({128, 16, 8, 4, 0, 1 << 17, {4, 4}, {70000, 70000}});
    check({256, 16, 8, 4, 0, 1 << 16, {4, 4}, {36000, 36000}});
    check({128, 32, 8, 4, 0, 1 << 17, {38, 20, 49, 35}, {76116, 41908, 31893, 63026}});
    check({128, 32, 4, 8, 0, 131072, {32, 32, 32, 32, 32}, {100000, 100000, 100000, 100000, 1000}});
    check({256, 32, 8, 4, 0, 32768, {32, 32, 32, 32, 32, 32, 32}, {30000, 200, 200, 200, 200, 200, 200}});
    std::mt19937_64 rng(1);
    const auto log_int = [&](int lo, int hi) {
        return (int) std::lround(std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi))(rng)));
    };
    const auto any = [&](std::initializer_list<int> x) { return x.begin()[rng() % x.size()]; };
    for (int i = 0; i < 20000; i++) {
        Batch b{any({64, 128, 256}), any({16, 32}), any({1, 2, 4, 8, 8}), any({1, 2, 4, 4, 7, 8}), any({0, 0, 0, 1024, 4096, 20000}), 0, {}, {}};
        const int n_seq = rng() % 3 ? log_int(1, 8) : log_int(1, 64), most = log_int(1, 64), least = log_int(1, most);
        const int last = log_int(200, 131072), first = log_int(1, last);
        for (int s = 0; s < n_seq; s++) b.rows.push_back(rng() % 16 ? log_int(least, most) : 0), b.past.push_back(log_int(first, last));
        int64_t keys = 0;
        for (int s = 0; s < n_seq; s++) keys = std::max<int64_t>(keys, b.past[s] + b.rows[s]);
        b.slots = (keys + 63) / 64 * 64 + 64 * (int64_t) (rng() % 4);
        check(b);
    }
    printf("sorted %d, of them not all resident %d, blocks turned %d, failed %d\n", sorted, over, turned_blocks, failed);
    return failed != 0;
}
