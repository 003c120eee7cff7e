// Log-probabilities of given tokens, the entropy and the top alternatives of
// every row of logits. For a row x[v] with m = max x, S = sum_v exp(x[v] - m):
//   log p(v) = x[v] - m - log S
//   H = - sum_v p(v) log p(v) = log S - sum_v exp(x[v] - m) (x[v] - m) / S
// and the k largest log p(v), equal ones by the lower v. A NaN logit counts as
// -inf (a banned token), as in the beam selection, and a token of probability
// 0 adds nothing to the entropy. With m = +inf the difference of two
// infinities is taken as 0, so the +inf tokens share the probability. A row
// without any token above -inf has no alternatives, entropy 0, and every
// token's log-probability is -inf.
//
// The rows' columns are cut into tiles of 16 KB, and all tiles of all rows, in
// order, into equal runs, one a CTA: so every CTA streams the same bytes, and a
// row may be reduced by several, each to its statistics and its k best logits
// (packed keys: value, then lower id). A second kernel joins them, of every
// shard of the vocabulary.
//
// Sums are fp32 per lane against a reference that follows the maximum only when
// it has to; parts of a row are joined in fp64.
//
// Without alternatives bound by HBM: 4096 bf16 rows of 151936 235 us, 5.3 TB/s;
// DRAM reads are the logits once. With alternatives each part of a row costs its
// start, floors and ranking, about 10 000 cycles beside 2400 a tile: 2048 rows of
// 151936 124 us without, 175 / 230 / 324 with 1 / 20 / 64; 512 rows with 20 76.
#pragma once

#include "logprobs_plan.cuh"
#include "topk.cuh"

namespace mtpb {

constexpr int kLpMaxK = kBeamMaxK;

// Of a part of a row: m = max x, s = sum exp(x - m), w = sum exp(x - m) (x - m),
// and the target's logit (NaN: the target lies elsewhere). s 0: no token; NaN: a
// wait for the part's logits ran out, and its row comes out as NaN.
struct LpStat {
  float m, s, w, xt;
};

static_assert(kLpWarps == kBeamWarps, "beam_floor takes the candidates of as many warps");
template <bool TOP>
constexpr size_t kLpRing = size_t(kLpStages<TOP>) * kLpTile * 16;
constexpr int kLpThreads = kLpWarps * 32;

struct LpRowsParams {
  const void* logits;
  int64_t ld;      // elements between rows
  int rows, V, k;  // columns of this shard, candidates a part
  int64_t vstart;  // id of column 0
  LpPlan plan;
  const long long* targets;  // [rows] or NULL
  LpStat* stat;    // [rows][parts]
  uint64_t* cand;  // [rows][parts][k], best first, 0-padded
};

// Set when a bounded wait of a log-probability kernel ran out (its results are then void).
__device__ uint32_t g_lp_status;

// A lane's sums over its values so far, and its reference.
struct LpLane {
  float m = -INFINITY, c = 0.f, s = 0.f, w = 0.f;
};

// Takes a tile's values in: vector u of this lane holds columns col + u * 32 * VE
// ... `first`: the warp's first tile (which sets a floor for its candidates).
template <typename T, bool TOP>
__device__ __forceinline__ void lp_step(LpLane& a0, BeamList& l, const uint4 (&v)[kLpVecs], int col, bool first, int k,
                                        int64_t vstart, uint32_t* floor_key) {
  constexpr int VE = VecTraits<T>::kElems, kLow = sizeof(T) == 2 ? 16 : 0;
  const int lane = threadIdx.x & 31;
  float m = a0.m, c = a0.c, s = a0.s, ws = a0.w;
          float q[kLpVecs];  // max of each vector, at least -2^126
          uint32_t y[kLpVecs][4];
#pragma unroll
          for (int u = 0; u < kLpVecs; ++u) {
            const uint32_t raw[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            if constexpr (sizeof(T) == 2) {
#pragma unroll
              for (int i = 0; i < 4; ++i) asm("max.bf16x2 %0, %1, %2;" : "=r"(y[u][i]) : "r"(raw[i]), "r"(0xFE80FE80u));
              uint32_t a, b;
              asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(y[u][0]), "r"(y[u][1]));
              asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(y[u][2]), "r"(y[u][3]));
              asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
              q[u] = fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) y[u][i] = __float_as_uint(fmaxf(__uint_as_float(raw[i]), -0x1p126f));
              q[u] = fmaxf(max3(__uint_as_float(y[u][0]), __uint_as_float(y[u][1]), __uint_as_float(y[u][2])),
                           __uint_as_float(y[u][3]));
            }
          }
          float top = fmaxf(max3(q[0], q[1], q[2]), q[3]);
          // (read early: an older floor is a floor too)
          const uint32_t common = TOP ? *static_cast<volatile uint32_t*>(floor_key) : 0u;
          // ---- sums
          if (!beam_far(fmaxf(m, top))) {
            if (top - m > 8.f) {
              if (beam_far(m)) {  // nothing yet, or values that count for nothing beside these
                s = ws = 0.f;
              } else {
                const float d = beam_ref(m) - beam_ref(top), a = exp2_approx(d);
                ws = fmaf(s, d, ws) * a;
                s *= a;
              }
              m = top;
              c = beam_ref(m);
            }
            float2 sum = make_float2(0.f, 0.f), mean = make_float2(0.f, 0.f);
#pragma unroll
            for (int u = 0; u < kLpVecs; ++u)
#pragma unroll
              for (int i = 0; i < 4; i += sizeof(T) == 2 ? 1 : 2) {
                float2 x;
                if constexpr (sizeof(T) == 2)
                  x = make_float2(__uint_as_float(y[u][i] << 16), __uint_as_float(y[u][i] & 0xFFFF0000u));
                else
                  x = make_float2(__uint_as_float(y[u][i]), __uint_as_float(y[u][i + 1]));
                const float2 d = fma2(x, make_float2(kBeamLog2e, kBeamLog2e), make_float2(-c, -c));
                const float2 e = make_float2(exp2_approx(d.x), exp2_approx(d.y));
                sum = add2(sum, e);
                mean = fma2(e, d, mean);
              }
            s += sum.x + sum.y;
            ws += mean.x + mean.y;
          } else {
            float raw_top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kLpVecs; ++u) {
              float g[VE];
              unpack(v[u], g);
#pragma unroll
              for (int e = 0; e < VE; ++e) raw_top = fmaxf(raw_top, g[e]);
            }
            if (raw_top > m) {
              m = raw_top;
              s = ws = 0.f;
            }
            if (m > -INFINITY)
#pragma unroll
              for (int u = 0; u < kLpVecs; ++u) {
                float g[VE];
                unpack(v[u], g);
#pragma unroll
                for (int e = 0; e < VE; ++e) s += g[e] == m ? 1.f : 0.f;
              }
          }
          // ---- candidates
          if constexpr (TOP) {
            if (first) {
              // the k-th of the warp's 32 * kLpVecs vector maxima: k values lie at or above it
              uint32_t kq[kLpVecs];
#pragma unroll
              for (int u = 0; u < kLpVecs; ++u) kq[u] = q[u] > -0x1p126f ? beam_logit_key(q[u]) : 0u;
              const uint32_t most = __reduce_max_sync(0xffffffffu, max(max(kq[0], kq[1]), max(kq[2], kq[3])));
              // 32 lanes reach the least of their maxima; for more than 32 the least of all bounds the k-th
              const uint32_t least = __reduce_min_sync(0xffffffffu, k <= 32 ? max(max(kq[0], kq[1]), max(kq[2], kq[3]))
                                                                              : min(min(kq[0], kq[1]), min(kq[2], kq[3])));
              const uint32_t cut = beam_search(k, least, most, kLow, [&](uint32_t x) {
                uint32_t n = 0;
#pragma unroll
                for (int u = 0; u < kLpVecs; ++u) n += kq[u] >= x ? 1u : 0u;
                return int(__reduce_add_sync(0xffffffffu, n));
              });
              if (lane == 0) atomicMax(floor_key, cut);
              l.least = max(l.least, cut);
            }
            l.least = max(l.least, common);
            const float ge = beam_key_val(l.least);
            // (q is -2^126 where a vector holds nothing above it: its values are then looked at one by one)
            if (__any_sync(0xffffffffu, top >= ge || !(ge > -0x1p126f))) {
              uint32_t mine = 0;  // this lane's values that enter
#pragma unroll
              for (int u = 0; u < kLpVecs; ++u) {
                if (!__any_sync(0xffffffffu, q[u] >= ge || !(ge > -0x1p126f))) continue;
                float g[VE];
                unpack(v[u], g);
#pragma unroll
                for (int e = 0; e < VE; ++e) mine |= g[e] >= ge ? 1u << (u * VE + e) : 0u;
              }
              while (true) {  // one value of each lane at a time
                const uint32_t b = __ballot_sync(0xffffffffu, mine != 0);
                if (!b) break;
                if (mine) {
                  const int i = __ffs(mine) - 1, u = i / VE, e = i - u * VE;
                  mine &= mine - 1;
                  const uint4 x = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
                  const int word = e * int(sizeof(T)) / 4;
                  const uint32_t bits = word == 0 ? x.x : word == 1 ? x.y : word == 2 ? x.z : x.w;
                  const float val = sizeof(T) == 4 ? __uint_as_float(bits) : __uint_as_float(e & 1 ? bits & 0xFFFF0000u : bits << 16);
                  const uint32_t id = uint32_t(vstart + col + u * 32 * VE + e);
                  l.buf[l.n + __popc(b & ((1u << lane) - 1u))] = beam_key(beam_logit_key(val), id);
                }
                l.n += __popc(b);
                __syncwarp();
                if (l.n > kBeamCap - 32) beam_cut<kLow>(l, k, floor_key);
              }
              // later columns have higher ids: they have to beat the k-th, not to equal it
              if (l.kth) l.least = max(l.least, l.kth + 1);
            }
          }
  a0 = LpLane{m, c, s, ws};
}

// Sums against mm as sums against the larger top (natural units).
__device__ __forceinline__ void lp_raise(float mm, float top, float& ss, float& ww) {
  if (mm == top) return;
  const float d = mm - top, a = exp2_approx(d * kBeamLog2e);
  ww = a > 0.f ? fmaf(d, ss, ww) * a : 0.f;
  ss *= a;
}

// The warp's statistics from its lanes'.
__device__ __forceinline__ LpStat lp_warp_stat(LpLane a) {
  float cm = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
  if (!beam_far(a.m)) {  // against m itself, in natural units
    const float d = fmaf(a.m, kBeamLog2e, -a.c), f = exp2_approx(-d);
    a.w = fmaf(-d, a.s, a.w) * f * 0.69314718055994530942f;
    a.s *= f;
  }
  lp_raise(a.m, cm, a.s, a.w);
  return LpStat{cm, warp_sum(a.s), warp_sum(a.w), 0.f};
}

// The vector of a row's first or last columns, those outside its whole vectors:
// columns col .. col + n - 1, n < VE, one a lane.
template <typename T>
__device__ __forceinline__ void lp_edge(const T* x, int n, int col, uint4 (&v)[kLpVecs]) {
  constexpr int VE = VecTraits<T>::kElems;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < kLpVecs; ++u) {
    float g[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) g[e] = u == 0 && e == 0 && lane < n ? to_f(x[col + lane]) : -INFINITY;
    v[u] = pack_vec(g);
  }
}

// Row r of the logits.
template <typename T>
struct LpRow : LpCols {
  const T* x;
  __device__ __forceinline__ LpRow(const LpRowsParams& p, int r) {
    x = static_cast<const T*>(p.logits) + int64_t(r) * p.ld;
    static_cast<LpCols&>(*this) = lp_cols(reinterpret_cast<uintptr_t>(x), p.V, int(sizeof(T)));
  }
};

// One pass over the logits, bound by their bytes for many rows. A lane keeps
// a reference m, s = sum 2^d and w = sum 2^d d with d = x L - c (c = m L
// rounded, beam_ref), in fp32; the reference follows the lane's maximum when
// that has passed it by 8 (natural units), so that d stays small and the
// entropy's logarithm and mean, which are taken from each other, lose little.
// Values are raised to at least -2^126 first, which takes NaN and -inf along:
// they then add 2^d d = 0 x finite. Where the reference is far (2^30 or more:
// neighbours then lie 64 apart, and the raised ones may hide below) the values
// equal to the maximum are counted from the bits as they are.
// Without candidates (TOP false) two thirds of the instructions are left.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads + 32, 3) lp_rows_kernel(const LpRowsParams p) {
  constexpr int VE = VecTraits<T>::kElems, kLow = sizeof(T) == 2 ? 16 : 0, NS = kLpStages<TOP>;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ uint64_t buf[TOP ? kLpWarps : 1][TOP ? kBeamCap : 1];
  __shared__ uint64_t all[TOP ? kLpWarps * kLpMaxK : 1];
  __shared__ uint64_t full[NS], empty[NS];
  __shared__ LpStat stat[kLpWarps];
  __shared__ uint32_t floors[2];  // by the part's parity: at least k of its values have this key or a higher one
  __shared__ int totals[2], count[kLpWarps], abort_sh;
  volatile int* abort = &abort_sh;
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t0 = (long long)blockIdx.x * p.plan.run;
  const long long t1 = min(t0 + p.plan.run, (long long)p.rows * p.plan.tiles);
  if (threadIdx.x == kLpThreads) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kLpWarps);
    }
    mbar_init_fence();
  }
  if (threadIdx.x == 0) {
    floors[0] = floors[1] = 0;
    totals[0] = totals[1] = 0;
    *abort = 0;
  }
  __syncthreads();
  auto row_at = [&](int r) { return LpRow<T>(p, r); };
  int row = int(t0 / p.plan.tiles), tile = int(t0 - (long long)row * p.plan.tiles);
  int sg = 0;
  uint32_t phase = 0;
  auto refloor = [&](int i, int last) { return TOP && lp_refloor(p.k, i, last); };
  if (warp == kLpWarps) {  // ---- copies, a ring ahead of the tiles that the others are at, and floors
    int row2 = row, tile2 = tile, issued = 0, s2 = 0;  // of the next copy
    uint32_t ph2 = 0;
    long long t2 = t0;
    LpRow<T> w2 = row_at(row2);
    bool ok = true;
    // One call a tile, whether it holds vectors or not: the slot that a call waits
    // for then held a tile at or before the one that the others are at. (A call
    // that passed over empty tiles would be ahead of them by a tile for each of
    // those, and both would wait, here and at the floor's barrier, for one another.)
    auto copy = [&]() {
      if (t2 >= t1) return;
      const int n = lp_tile_vecs(w2.nvec, tile2);
      const T* from = w2.x + w2.head + int64_t(tile2) * kLpTile * VE;
      ++t2;
      if (++tile2 == p.plan.tiles) {
        tile2 = 0;
        w2 = row_at(min(++row2, p.rows - 1));
      }
      if (n <= 0) return;
      ok = ok && (issued < NS || __all_sync(0xffffffffu, mbar_wait_lean(empty + s2, ph2 ^ 1u, abort)));
      if (!ok) {
        *abort = 1;
        return;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(full + s2, uint32_t(n) * 16);
        bulk_g2s(ring + s2 * kLpTile, from, uint32_t(n) * 16, full + s2);
      }
      __syncwarp();
      if (issued < NS) ++issued;
      if (++s2 == NS) {
        s2 = 0;
        ph2 ^= 1u;
      }
    };
    for (int i = 0; i < NS; ++i) copy();
    int odd = 0;
    for (long long t = t0; t < t1; ++row, tile = 0, odd ^= 1) {
      const int n = int(min((long long)p.plan.tiles - tile, t1 - t));
      t += n;
      for (int i = 0; i < n; ++i) {
        if (refloor(i, n - 1)) {
          named_sync(2, kLpThreads + 32);
          uint32_t key[kLpWarps];
#pragma unroll
          for (int u = 0; u < kLpWarps; ++u) key[u] = lane < count[u] ? uint32_t(buf[TOP ? u : 0][TOP ? lane : 0] >> 32) : 0;
          named_sync(2, kLpThreads + 32);  // the lists may change again
          beam_floor<kLow>(key, p.k, floors + odd);
        }
        copy();
      }
    }
    // copies in flight land before the memory goes away
    int never = 0;
    if (issued < NS)
      s2 = 0, ph2 = 0;
    else
      ph2 ^= 1u;
    for (int i = 0; i < issued; ++i) {
      mbar_wait_lean(full + s2, ph2, &never);
      if (++s2 == NS) {
        s2 = 0;
        ph2 ^= 1u;
      }
    }
  } else {
    bool ok = true;
    int odd = 0;  // parity of the part
    long long next_goal = threadIdx.x == 0 && p.targets ? p.targets[row] : 0;
    for (long long t = t0; t < t1; ++row, tile = 0, odd ^= 1) {
      uint32_t* floor_key = floors + odd;
      // ---- this CTA's part of a row
      const LpRow<T> w = row_at(row);
      const int end = int(min((long long)p.plan.tiles, tile + (t1 - t)));
      const int c0 = tile == 0 ? 0 : min(p.V, w.head + tile * kLpTile * VE);
      const int c1 = end == p.plan.tiles ? p.V : min(p.V, w.head + end * kLpTile * VE);
      t += end - tile;
      // (the target's logit is not looked at before the part's end, and the next row's target read ahead)
      float xt = 0.f;
      const long long goal = next_goal - p.vstart;
      const bool here = threadIdx.x == 0 && p.targets && goal >= c0 && goal < c1;
      if (here) xt = to_f(w.x[goal]);
      if (threadIdx.x == 0 && p.targets && t < t1) next_goal = p.targets[row + 1];
      BeamList l{TOP ? buf[warp] : nullptr, 0, 0x00800000u, 0u};  // least: the key of the lowest finite value
      LpLane sums;
      auto step = [&](const uint4 (&v)[kLpVecs], int col, bool first) {
        lp_step<T, TOP>(sums, l, v, col, first, p.k, p.vstart, floor_key);
      };
      constexpr uint32_t kNone = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;  // -inf
      auto edge = [&](int n, int col) {
        uint4 v[kLpVecs];
        lp_edge(w.x, n, col, v);
        step(v, col + lane, false);
      };
      if (warp == 0 && tile == 0 && w.head) edge(w.head, 0);
      bool first = true;
      for (int i = 0, last = end - 1 - tile; tile < end; ++tile, ++i) {
        const int n = lp_tile_vecs(w.nvec, tile), at = warp * 32 * kLpVecs + lane;
        auto join_floor = [&]() {
          if (!refloor(i, last)) return;
          beam_drop(l, *static_cast<volatile uint32_t*>(floor_key));
          if (lane == 0) count[warp] = l.n;
          named_sync(2, kLpThreads + 32);
          named_sync(2, kLpThreads + 32);
        };
        if (n <= 0) {
          join_floor();
          continue;
        }
        ok = ok && mbar_wait_lean(full + sg, phase, abort);
        if (!__all_sync(0xffffffffu, ok)) {
          *abort = 1;
          ok = false;
        }
        uint4 v[kLpVecs];
#pragma unroll
        for (int u = 0; u < kLpVecs; ++u)
          v[u] = ok && at + 32 * u < n ? ring[sg * kLpTile + at + 32 * u] : make_uint4(kNone, kNone, kNone, kNone);
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + sg);
        if (++sg == NS) {
          sg = 0;
          phase ^= 1u;
        }
        if (at - lane < n) step(v, w.head + (tile * kLpTile + at) * VE, first);
        first = false;
        join_floor();
      }
      if (warp == kLpWarps - 1 && end == p.plan.tiles && w.tail) edge(w.tail, p.V - w.tail);
      // ---- the part's statistics
      const LpStat mine = lp_warp_stat(sums);
      if (lane == 0) stat[warp] = mine;
      const size_t at = size_t(row) * p.plan.parts + size_t(blockIdx.x - p.plan.first(row));
      if constexpr (TOP) {
        // ---- its k best: the warps' candidates (at most 64 each) from the common floor on, ranked
        if (l.n > kLpMaxK) beam_cut<kLow>(l, p.k, floor_key);
        named_sync(1, kLpThreads);
        const uint32_t fk = *floor_key;
        for (int i = lane; i < l.n; i += 32) {
          const uint64_t o = l.buf[i];
          if (uint32_t(o >> 32) >= fk) all[atomicAdd(totals + odd, 1)] = o;
        }
        named_sync(1, kLpThreads);
        const int n = totals[odd];
        uint64_t* out = p.cand + at * p.k;
        for (int i = threadIdx.x; i < n; i += kLpThreads) {
          const uint64_t o = all[i];
          int rank = 0;
          for (int j = 0; j < n; ++j) rank += all[j] > o ? 1 : 0;
          if (rank < p.k) out[rank] = o;
        }
        for (int i = n + threadIdx.x; i < p.k; i += kLpThreads) out[i] = 0;
      } else {
        named_sync(1, kLpThreads);
      }
      if (warp == 0) {
        LpStat r = stat[lane & (kLpWarps - 1)];
        float top = r.m;
#pragma unroll
        for (int o = kLpWarps / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        lp_raise(r.m, top, r.s, r.w);
#pragma unroll
        for (int o = kLpWarps / 2; o > 0; o >>= 1) {
          r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
          r.w += __shfl_xor_sync(0xffffffffu, r.w, o);
        }
        if (lane == 0) {
          r.m = top;
          r.xt = !here ? __int_as_float(0x7fffffff) : xt == xt ? xt : -INFINITY;
          if (*abort) r.s = __int_as_float(0x7fffffff);
          p.stat[at] = r;
          floors[odd ^ 1] = 0;  // (the part before's, which nobody reads any more)
          totals[odd ^ 1] = 0;
        }
      }
      named_sync(1, kLpThreads);  // the next part's lists and statistics
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicOr(&g_lp_status, kStatusTimeout);
}

// Many rows of one tile or less: a warp a row, straight from global memory,
// without the barriers and the ring's start that a part of a CTA's run costs
// (8192 bf16 rows of 1000 columns with 5 alternatives: 25 us instead of 94).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kLpThreads, 3) lp_short_kernel(const LpRowsParams p) {
  constexpr int VE = VecTraits<T>::kElems, kLow = sizeof(T) == 2 ? 16 : 0;
  __shared__ uint64_t buf[TOP ? kLpWarps : 1][TOP ? kBeamCap : 1];
  __shared__ uint32_t floors[kLpWarps];
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int row = blockIdx.x * kLpWarps + warp; row < p.rows; row += gridDim.x * kLpWarps) {
    const LpRow<T> w(p, row);
    float xt = __int_as_float(0x7fffffff);
    if (lane == 0 && p.targets) {
      const long long c = p.targets[row] - p.vstart;
      if (c >= 0 && c < p.V) xt = to_f(w.x[c]);
      if (c >= 0 && c < p.V && xt != xt) xt = -INFINITY;
    }
    if (lane == 0) floors[warp] = 0;
    __syncwarp();
    BeamList l{TOP ? buf[warp] : nullptr, 0, 0x00800000u, 0u};
    LpLane sums;
    uint4 v[kLpVecs];
    const uint4* x = reinterpret_cast<const uint4*>(w.x + w.head);
    constexpr uint32_t kNone = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;  // -inf
    if (w.head) {
      lp_edge(w.x, w.head, 0, v);
      lp_step<T, TOP>(sums, l, v, lane, false, p.k, p.vstart, floors + warp);
    }
    for (int i = lane; i - lane < w.nvec; i += 32 * kLpVecs) {
#pragma unroll
      for (int u = 0; u < kLpVecs; ++u)
        v[u] = i + 32 * u < w.nvec ? ld_stream(x + i + 32 * u) : make_uint4(kNone, kNone, kNone, kNone);
      lp_step<T, TOP>(sums, l, v, w.head + i * VE, i == lane, p.k, p.vstart, floors + warp);
    }
    if (w.tail) {
      lp_edge(w.x, w.tail, p.V - w.tail, v);
      lp_step<T, TOP>(sums, l, v, p.V - w.tail + lane, false, p.k, p.vstart, floors + warp);
    }
    LpStat r = lp_warp_stat(sums);
    r.xt = xt;
    if (lane == 0) p.stat[row] = r;
    if constexpr (TOP) {
      if (l.n > kLpMaxK) beam_cut<kLow>(l, p.k, floors + warp);
      __syncwarp();
      uint64_t* out = p.cand + size_t(row) * p.k;
      for (int i = lane; i < l.n; i += 32) {
        const uint64_t o = l.buf[i];
        int place = 0;
        for (int j = 0; j < l.n; ++j) place += l.buf[j] > o ? 1 : 0;
        if (place < p.k) out[place] = o;
      }
      for (int i = l.n + lane; i < p.k; i += 32) out[i] = 0;
      __syncwarp();
    }
  }
}

struct LpJoinParams {
  const LpStat* stat;    // [shards][rows][parts]
  const uint64_t* cand;  // [shards][rows][parts][kc]
  size_t stat_shard, cand_shard;  // elements between the shards' blocks
  LpPlan plan;
  int shards, rows, k, kc;
  float *logprobs, *entropy;  // [rows]; logprobs NULL without targets
  float* top_logprobs;        // [rows][k]
  long long* top_ids;
};

constexpr int kLpJoinWarps = 4;
constexpr int kLpRanked = 512;  // candidates of a row that are ranked against each other

// A warp a row, in fp64.
__global__ void __launch_bounds__(32 * kLpJoinWarps) lp_join_kernel(const LpJoinParams p) {
  extern __shared__ uint64_t lp_cands[];  // [warps][kLpRanked]; then [warps][lists] bytes: entries of each list that were taken
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t row = size_t(blockIdx.x) * kLpJoinWarps + warp;
  if (row >= size_t(p.rows)) return;
  const int per = p.plan.count((long long)row), lists = p.shards * per;
  auto stat = [&](int i) { return p.stat + (i / per) * p.stat_shard + row * p.plan.parts + i % per; };
  auto cand = [&](int i) { return p.cand + (i / per) * p.cand_shard + (row * p.plan.parts + i % per) * p.kc; };
  float m = -INFINITY, xt = -INFINITY;
  bool found = false, lost = false;
  for (int i = lane; i < lists; i += 32) {
    const LpStat s = *stat(i);
    lost = lost || s.s != s.s;
    if (s.s > 0.f) m = fmaxf(m, s.m);
    if (s.xt == s.xt) {
      xt = s.xt;
      found = true;
    }
  }
  found = __any_sync(0xffffffffu, found);
  lost = __any_sync(0xffffffffu, lost);
  const float nan = __int_as_float(0x7fffffff);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    xt = fmaxf(xt, __shfl_xor_sync(0xffffffffu, xt, o));
  }
  double sum = 0.0, w = 0.0;
  for (int i = lane; i < lists; i += 32) {
    const LpStat s = *stat(i);
    if (!(s.s > 0.f)) continue;
    const double d = s.m == m ? 0.0 : double(s.m) - double(m), e = exp(d);
    sum += e * s.s;
    if (e > 0.0) w += e * (double(s.w) + d * s.s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
  }
  const double logs = sum > 0.0 ? log(sum) : 0.0;
  auto logp = [&](float x) {
    if (lost) return nan;
    if (x == -INFINITY) return -INFINITY;
    return float((x == m ? 0.0 : double(x) - double(m)) - logs);
  };
  if (lane == 0) {
    p.entropy[row] = lost ? nan : sum > 0.0 ? float(logs - w / sum) : 0.f;
    if (p.logprobs) p.logprobs[row] = found ? logp(xt) : nan;
  }
  if (!p.k) return;
  const int n = lists * p.kc;
  uint64_t* mine = lp_cands + warp * kLpRanked;
  auto load = [&](int i) -> uint64_t {
    return i < n ? __ldcg(reinterpret_cast<const unsigned long long*>(cand(i / p.kc)) + i % p.kc) : 0;
  };
  int left = n;  // candidates in `mine`; more than kLpRanked: they did not fit
  if (n <= 64) {
    for (int i = lane; i < n; i += 32) mine[i] = load(i);
  } else if (n <= kLpRanked) {  // those below the k-th go first
    constexpr int H = kLpRanked / 32;
    uint64_t held[H];
#pragma unroll
    for (int h = 0; h < H; ++h) held[h] = load(lane + 32 * h);
    uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const uint32_t v = uint32_t(held[h] >> 32);
      most = max(most, v);
      least = min(least, v);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    const uint32_t cut = beam_search(p.k, least, most, 0, [&](uint32_t v) {
      uint32_t c = 0;
#pragma unroll
      for (int h = 0; h < H; ++h) c += uint32_t(held[h] >> 32) >= v ? 1u : 0u;
      return int(__reduce_add_sync(0xffffffffu, c));
    });
    left = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const bool in = held[h] && uint32_t(held[h] >> 32) >= cut;
      const uint32_t b = __ballot_sync(0xffffffffu, in);
      if (in) mine[left + __popc(b & ((1u << lane) - 1u))] = held[h];
      left += __popc(b);
    }
  } else {  // many lists (few rows, or many shards): each has its c best, c * lists >= k, at or above the least of those
    const int c = (p.k + lists - 1) / lists;
    uint32_t least = 0xFFFFFFFFu;
    for (int i = lane; i < lists; i += 32) least = min(least, uint32_t(load(i * p.kc + min(c, p.kc) - 1) >> 32));
    least = __reduce_min_sync(0xffffffffu, least);
    left = 0;
    for (int i0 = 0; i0 < lists && left <= kLpRanked; i0 += 32) {
      for (int j = 0; j < p.kc && left <= kLpRanked; ++j) {
        const uint64_t o = i0 + lane < lists ? load((i0 + lane) * p.kc + j) : 0;
        const bool in = o && uint32_t(o >> 32) >= least;
        const uint32_t b = __ballot_sync(0xffffffffu, in);
        if (!b) break;
        const int at = left + __popc(b & ((1u << lane) - 1u));
        if (in && at < kLpRanked) mine[at] = o;
        left += __popc(b);
      }
    }
  }
  if (left <= kLpRanked) {
    __syncwarp();
    int live = 0;
    for (int i = lane; i < left; i += 32) {
      const uint64_t o = mine[i];
      if (!o) continue;
      ++live;
      int place = 0;  // how many are better
      for (int j = 0; j < left; ++j) place += mine[j] > o ? 1 : 0;
      if (place < p.k) {
        p.top_logprobs[row * p.k + place] = logp(beam_key_val(uint32_t(o >> 32)));
        p.top_ids[row * p.k + place] = (long long)(0xFFFFFFFFu - uint32_t(o));
      }
    }
    live = __reduce_add_sync(0xffffffffu, live);
    for (int j = live + lane; j < p.k; j += 32) {
      p.top_logprobs[row * p.k + j] = logp(-INFINITY);
      p.top_ids[row * p.k + j] = 0;
    }
    return;
  }
  // the lists are sorted: the best of their heads is the next
  uint8_t* head = reinterpret_cast<uint8_t*>(lp_cands + kLpJoinWarps * kLpRanked) + warp * (p.shards * p.plan.parts);
  for (int i = lane; i < lists; i += 32) head[i] = 0;
  for (int j = 0; j < p.k; ++j) {
    uint64_t b = 0;
    int at = -1;
    for (int i = lane; i < lists; i += 32) {
      const uint64_t o = head[i] < p.kc ? __ldcg(reinterpret_cast<const unsigned long long*>(cand(i)) + head[i]) : 0;
      if (o > b) {
        b = o;
        at = i;
      }
    }
    const uint64_t top = warp_max_u64(b);
    if (top && b == top) ++head[at];
    if (lane == 0) {
      p.top_logprobs[row * p.k + j] = logp(top ? beam_key_val(uint32_t(top >> 32)) : -INFINITY);
      p.top_ids[row * p.k + j] = top ? (long long)(0xFFFFFFFFu - uint32_t(top)) : 0;
    }
  }
}

}  // namespace mtpb
