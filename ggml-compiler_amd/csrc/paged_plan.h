// paged_plan.h - the arithmetic by which paged_attn.hip's workgroups share out a batch, without the wavefronts that do it there (a sequence
// to a lane), so that it also compiles for the host: tests/cpp/paged_plan.cpp runs it over many batches.
#pragma once

namespace gcq {

constexpr int kMinChunk = 16;  // tiles of a split: four to a wavefront (32 sequences' step: 25.3 us, with 32 tiles 28.6)

// Wavefronts per SIMD that the registers (and, heads of 256, LDS) hold; and of a workgroup.
// (Eight wavefronts to a workgroup, heads of 128: 32 sequences' step 32.1 us for 25.3 with four, four prompts 134 for 86; heads of
// 256 with 32 rows, whose four wavefronts would fill half the LDS: 52.6 us with eight, 80.3 with four.)
constexpr int per_simd(int D, int RT) { return D * RT <= 128 ? 4 : D * RT == 256 && RT == 2 ? 3 : 2; }
constexpr int waves(int D, int rows) { return D == 256 && rows == 32 ? 8 : 4; }
// Workgroups resident at once, those that the splits aim at.
constexpr int plan_target(int D, int rows) { return 256 * 4 * per_simd(D, rows / 16) / waves(D, rows); }

constexpr int splits(int tiles, int chunk) { return tiles > chunk ? (tiles + chunk - 1) / chunk : 1; }

// Tiles to a split, so that u tiles come to about `cut` splits.
constexpr int plan_chunk(double u, double cut, int min_chunk) {
    const double chunk = u / cut + 1.0;
    return (int) (chunk < min_chunk ? (double) min_chunk : chunk < 1e9 ? chunk : 1e9);
}
// A longer one, where items come to `more` times as many as are resident.
constexpr int plan_longer(int chunk, double more) { return (int) (chunk * (more < 2.0 ? 0.5 + 0.5 * more : 1.5)) + 1; }

// The item of a workgroup, of a grid of at least as many as there are items: its own number, or (turned) every second 256 in the other
// order. The last of the grid's 256s stay as they are if they are not all there: each has an item of its own and none is left over, also
// where there are more items than are resident at once.
constexpr int unit_of(int block, int grid, bool turned) { return turned && (block & 256) && (block | 255) < grid ? block ^ 255 : block; }
// Whether all splits of the row tile whose split `split` of ns is item `unit` are there to be joined.
constexpr bool all_there(int unit, int split, int ns, int grid) { return unit - split + ns <= grid; }

}  // namespace gcq
