// How rows of logits are cut into tiles, how those fall to CTAs, and where a
// CTA's warps meet: plain arithmetic, for the log-probability kernels, their
// launches, and a replay of the schedule on the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define MTPB_HD __host__ __device__ __forceinline__
#else
#define MTPB_HD inline
#endif

namespace mtpb {

constexpr int kLpWarps = 8;  // that compute; one more copies and finds the floors
constexpr int kLpVecs = 4;   // 16-byte vectors a lane and tile
constexpr int kLpTile = kLpWarps * 32 * kLpVecs;  // vectors
// Ring of tiles: what three CTAs an SM leave beside the candidates.
template <bool TOP>
constexpr int kLpStages = TOP ? 3 : 4;

// How the tiles of `rows` rows of `tiles` tiles fall to CTAs of `run` tiles each.
struct LpPlan {
  int tiles, run, parts;  // parts: the most CTAs that share a row
  MTPB_HD long long first(long long row) const { return row * tiles / run; }  // CTA of a row's first tile
  MTPB_HD int count(long long row) const { return int(((row + 1) * tiles - 1) / run - first(row)) + 1; }
};

// A function of the sizes alone, so that every rank cuts its shard alike. Three
// CTAs for each of B200's 148 SMs, which is what the ring leaves room for.
MTPB_HD LpPlan lp_plan(long long rows, int V, int elem_bytes) {
  LpPlan b;
  const int cols = kLpTile * (16 / elem_bytes);
  b.tiles = (V + cols - 1) / cols;
  const long long total = rows * b.tiles, ctas = total < 3 * 148 ? total : 3 * 148;
  b.run = int((total + ctas - 1) / ctas);
  b.parts = (b.tiles - 2) / b.run + 2;  // a row that begins at a run's last tile; never more than its tiles
  if (b.parts > b.tiles) b.parts = b.tiles;
  if (b.parts < 1) b.parts = 1;
  return b;
}

// A row of V columns at `at`: `head` columns before its first 16-byte boundary, whole vectors, `tail` columns behind them.
struct LpCols {
  int head, nvec, tail;
};
MTPB_HD LpCols lp_cols(uintptr_t at, int V, int elem_bytes) {
  const int ve = 16 / elem_bytes, off = int((at & 15u) / elem_bytes);
  LpCols c;
  c.head = off ? ve - off : 0;
  if (c.head > V) c.head = V;
  c.nvec = (V - c.head) / ve;
  c.tail = V - c.head - c.nvec * ve;
  return c;
}

// Whole vectors of a row's tile; none or less where the shard has fewer columns
// than were planned for, and where a row's last columns are head and tail alone.
MTPB_HD int lp_tile_vecs(int nvec, int tile) {
  const int n = nvec - tile * kLpTile;
  return n < kLpTile ? n : kLpTile;
}

// Whether all warps of a CTA meet after tile i of a part whose last is `last`:
// after the tiles 0 and 3 (of many candidates 0, 1, 3, 7 ..) the k-th of all
// warps' candidates becomes the floor. A later value then enters with odds k /
// (values seen by the CTA), not k / (values of one warp's first tile). (2048
// bf16 rows of 151936, never / 0, 3 / 0, 1, 3, 7 ..: 1 alternative 172 / 174 /
// 183 us, 64 alternatives 546 / 444 / 326; 512 rows, 20: 90 / 74 / 76.)
MTPB_HD bool lp_refloor(int k, int i, int last) { return i < last && (k > 32 ? (i & (i + 1)) == 0 : i == 0 || i == 3); }

}  // namespace mtpb
