// Beam search: selection over beams and vocabulary, and the KV cache rows
// that follow the chosen beams.
//
// Selection. For beam b of a prompt with logits x[v] and running score s:
//   total(b, v) = s + (x[v] - m) - log(sum_v exp(x[v] - m)),  m = max_v x[v]
// and the k best of (b, v) by (total descending, b * V + v ascending). A NaN
// logit counts as -inf (a banned token). With m = +inf the difference of two
// infinities is taken as 0, so the +inf tokens share the probability. A
// finished beam has one candidate: the end token at its own score. A beam
// whose score is -inf or NaN, or whose logits are all -inf, has none.
//
// Inside one row the order of totals is the order of the logits, so the
// vocabulary is cut into chunks: one CTA per (row, chunk) reduces its columns
// in one pass to the sum and the k best logits (packed keys: value, then lower
// id), and one CTA per prompt merges the chunks of all its beams.
#pragma once

#include "tma.cuh"

namespace mtpb {

constexpr int kBeamMaxK = 64;
constexpr int kBeamMaxW = 64;

// Sum of a chunk's exponentials, s = sum exp(x - m). m need not be the maximum:
// it keeps s in range. -inf: nothing summed.
struct BeamStat {
  float m, s;
};
// While a lane sums, it takes 2^(x L - c) with one fused multiply-add a value:
// L is log2(e) and c = m L, both rounded to fp32. The exponent is then off by
// m L - c for every x alike: up to 64 for |m| below 2^30, so that sums stay in
// range, and beam_own takes it out of the lane's sum. (Over a difference x - m,
// L's own rounding counts 1.3e-8 of it.) From 2^30 on fp32 neighbours are at
// least 64 apart (those below too): no other value's exponential counts beside
// m's, so s counts the values equal to m, infinities among them.
constexpr float kBeamLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float beam_ref(float m) { return __fmul_rn(m, kBeamLog2e); }
__device__ __forceinline__ bool beam_far(float m) { return !(fabsf(m) < 1073741824.f); }
// A lane's sum against m itself.
__device__ __forceinline__ float beam_own(float m, float s) {
  return beam_far(m) ? s : s * exp2_approx(-fmaf(m, kBeamLog2e, -beam_ref(m)));
}

// Order-preserving key of a finite or +inf logit and its id; 0: no candidate.
__device__ __forceinline__ uint32_t beam_val_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_key_val(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// Key of a logit that may be -inf or NaN (0), or -0 (as +0).
__device__ __forceinline__ uint32_t beam_logit_key(float v) { return v > -INFINITY ? beam_val_key(v + 0.f) : 0u; }
__device__ __forceinline__ uint64_t beam_key(uint32_t key, uint32_t id) { return (uint64_t(key) << 32) | (0xFFFFFFFFu - id); }

// What a sum against m counts in one against the larger top.
__device__ __forceinline__ float beam_weight(float m, float top) {
  return m == top ? 1.f : exp2_approx((m - top) * kBeamLog2e);  // (equal infinities: 1)
}
__device__ __forceinline__ uint64_t warp_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

struct BeamRowsParams {
  const void* logits;
  int64_t ld;      // elements between rows
  int V, k;        // vocabulary of this shard, candidates a chunk
  int64_t vstart;  // id of column 0
  int nchunk, chunk;  // chunks a row, columns a chunk
  const uint8_t* finished;  // [rows] or NULL: rows that need no scan
  BeamStat* stat;  // [rows][nchunk]
  uint64_t* cand;  // [rows][nchunk][k], best first, 0-padded
};

constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kBeamVecs = 4;   // 16-byte vectors a lane and tile
constexpr int kBeamCap = 160;  // candidates a warp holds between two cuts to the k best: 64, and room for 32 at a time

// One warp's candidates: every value of the warp's columns so far that may be
// among the chunk's k best, i.e. whose key is at least `least`.
struct BeamList {
  uint64_t* buf;  // [kBeamCap], shared memory
  int n;
  uint32_t least;
  uint32_t kth;  // after a cut: key of the k-th; else 0
};

// Largest t, in steps of 2^low, with count(t) >= k, for keys that lie in
// [least, most]: bit by bit below the bits that those two share, until the
// count is k.
template <typename Count>
__device__ __forceinline__ uint32_t beam_search(int k, uint32_t least, uint32_t most, int low, const Count& count) {
  const uint32_t diff = least ^ most;
  if (!diff) return most;
  const int high = 31 - __clz(diff);
  uint32_t t = high == 31 ? 0u : most & ~((2u << high) - 1u);
  for (int b = high; b >= low; --b) {
    const int n = count(t | (1u << b));
    if (n >= k) t |= 1u << b;
    if (n == k) break;
  }
  return t;
}

// Cuts the warp's buffer of more than k to its k best (in no order). The keys
// of bf16 values differ in their upper halves only (LOW 16): the k-th is then
// found to that step, which is exact (a positive one's lower half is 0, a
// negative one's all ones).
template <int LOW>
__device__ __forceinline__ void beam_cut(BeamList& l, int k, uint32_t* floor_key) {
  const int lane = threadIdx.x & 31;
  constexpr int E = kBeamCap / 32;
  uint32_t hi[E], lo[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint64_t o = lane + 32 * e < l.n ? l.buf[lane + 32 * e] : 0;
    hi[e] = uint32_t(o >> 32);
    lo[e] = uint32_t(o);
  }
  auto count = [&](auto&& in) {
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) n += in(e) ? 1u : 0u;
    return int(__reduce_add_sync(0xffffffffu, n));
  };
  uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (hi[e]) {
      most = max(most, hi[e]);
      least = min(least, hi[e]);
    }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  uint32_t t = beam_search(k, least, most, LOW, [&](uint32_t v) { return count([&](int e) { return hi[e] >= v; }); });
  if (LOW == 16 && !(t & 0x80000000u)) t |= 0xFFFFu;
  const int above = count([&](int e) { return hi[e] > t; });
  uint32_t u = 0;  // of those equal to t, the lowest ids (the largest low words)
  if (above + count([&](int e) { return hi[e] == t; }) > k && above < k)
    u = beam_search(k - above, 0u, 0xFFFFFFFFu, 0,
                    [&](uint32_t v) { return count([&](int e) { return hi[e] == t && lo[e] >= v; }); });
  least = 0xFFFFFFFFu;
  int n = 0;
  __syncwarp();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = hi[e] > t || (hi[e] == t && lo[e] >= u);
    const uint32_t b = __ballot_sync(0xffffffffu, in);
    if (in) {
      l.buf[n + __popc(b & ((1u << lane) - 1u))] = (uint64_t(hi[e]) << 32) | lo[e];
      least = min(least, hi[e]);
    }
    n += __popc(b);
  }
  __syncwarp();
  l.n = n;
  l.kth = __reduce_min_sync(0xffffffffu, least);
  l.least = max(l.least, l.kth);
  if (lane == 0) atomicMax(floor_key, l.kth);
}

// Takes the candidates below `least` out of the warp's buffer.
__device__ __forceinline__ void beam_drop(BeamList& l, uint32_t least) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int i0 = 0; i0 < l.n; i0 += 32) {
    const uint64_t o = i0 + lane < l.n ? l.buf[i0 + lane] : 0;
    const bool in = uint32_t(o >> 32) >= least && o;
    const uint32_t b = __ballot_sync(0xffffffffu, in);  // (reads of this step before its writes, which go no further)
    if (in) l.buf[n + __popc(b & ((1u << lane) - 1u))] = o;
    n += __popc(b);
    __syncwarp();
  }
  l.n = n;
}

// The k-th key among the warps' candidates (at most 32 of each, a lane's keys
// here), as the chunk's floor.
template <int LOW>
__device__ __forceinline__ void beam_floor(const uint32_t (&key)[kBeamWarps], int k, uint32_t* floor_key) {
  uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
  for (int w = 0; w < kBeamWarps; ++w) {
    most = max(most, key[w]);
    least = min(least, key[w] ? key[w] : 0xFFFFFFFFu);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  auto above = [&](uint32_t x) {
    uint32_t n = 0;
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) n += key[w] >= x ? 1u : 0u;
    return int(__reduce_add_sync(0xffffffffu, n));
  };
  if (least > most || above(least) < k) return;
  const uint32_t cut = beam_search(k, least, most, LOW, above);
  if ((threadIdx.x & 31) == 0) atomicMax(floor_key, cut);
}

// The chunk's 16-byte vectors come through a ring in shared memory, 16 KB
// rounds filled by bulk copies (warp 8, which also finds the floors), so that what is in flight does not
// depend on the registers of the warps that compute. One pass over the logits:
// bound by their bytes for many rows (512 fp32 rows of 151937: 53 us, 4.3 TB/s,
// with a tail of a seventh of the CTAs), by a chunk's start and end for few (64
// bf16 rows of 152064 in 4 chunks each: 18.8 us with the merge). Warp w < 8 takes vectors
// 128 w .. of each round; columns before the first and behind the last whole
// vector are warp 0's first and warp 7's last.
constexpr int kBeamRound = kBeamWarps * 32 * kBeamVecs;  // vectors
constexpr int kBeamStages = 4;
constexpr size_t kBeamRing = size_t(kBeamStages) * kBeamRound * 16;

// Set when a bounded wait of a selection ran out (its results are then void).
__device__ uint32_t g_beam_status;

// (CTAs an SM: three of fp32 took 66 us where two took 88, on 32 x 16 rows of
// 151937; two of bf16 20.8 where three, which spill, took 23.2, on 8 x 8 of 152064.)
template <typename T>
__global__ void __launch_bounds__(kBeamThreads + 32, sizeof(T) == 2 ? 2 : 3) beam_rows_kernel(const BeamRowsParams p) {
  constexpr int VE = VecTraits<T>::kElems, kLow = sizeof(T) == 2 ? 16 : 0;
  constexpr uint64_t kBudget = 2000000000ull;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ uint64_t buf[kBeamWarps][kBeamCap];
  uint64_t* all = reinterpret_cast<uint64_t*>(ring);  // at the end: [kBeamWarps * kBeamMaxK]
  __shared__ uint64_t full[kBeamStages], empty[kBeamStages];
  __shared__ float2 stat[kBeamWarps];
  __shared__ uint32_t floor_key;  // at least k of the chunk's values have this key or a higher one
  __shared__ int total, count[kBeamWarps], abort_sh;
  volatile int* abort = &abort_sh;
  pdl_launch();
  pdl_wait();
  const int row = blockIdx.y, ch = blockIdx.x;
  if (p.finished && p.finished[row]) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = ch * p.chunk, c1 = max(c0, min(p.V, c0 + p.chunk));
  const T* x = static_cast<const T*>(p.logits) + int64_t(row) * p.ld;
  const int off = int((reinterpret_cast<uintptr_t>(x + c0) & 15u) / sizeof(T));
  const int head = min(c1 - c0, off ? VE - off : 0);  // columns before the first vector
  const int nvec = (c1 - c0 - head) / VE, tail = c1 - c0 - head - nvec * VE;
  const int v0 = c0 + head;  // first column of vector 0
  const int rounds = (nvec + kBeamRound - 1) / kBeamRound;
  auto copy = [&](int r) {  // one thread
    const int s = r % kBeamStages, n = min(kBeamRound, nvec - r * kBeamRound);
    mbar_arrive_expect_tx(full + s, uint32_t(n) * 16);
    bulk_g2s(ring + s * kBeamRound, x + v0 + int64_t(r) * kBeamRound * VE, uint32_t(n) * 16, full + s);
  };
  if (threadIdx.x == kBeamThreads) {
    for (int s = 0; s < kBeamStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kBeamWarps);
    }
    mbar_init_fence();
    for (int r = 0; r < min(rounds, kBeamStages); ++r) copy(r);
  }
  if (threadIdx.x == 0) {
    floor_key = 0;
    total = 0;
    *abort = 0;
  }
  __syncthreads();
  BeamList l{buf[warp & 7], 0, 0x00800000u, 0u};  // least: the key of the lowest finite value
  float m = -INFINITY, c = 0.f, s = 0.f;  // reference and sum of this lane
  // after the rounds 1, 2, 4, 8 .. (all of them full) the k-th of all warps' candidates becomes the floor:
  // a later value enters with odds k / (values seen), not k / (values of one warp's first tile)
  auto refloor = [&](int r) { return r + 1 < rounds && (r & (r + 1)) == 0; };
  // a tile: vector u of this lane holds columns col + u * 32 * VE ..
  auto tile = [&](const uint4 (&v)[kBeamVecs], int col, bool first) {
    float q[kBeamVecs];  // max of each vector (a NaN is passed over)
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) {
      float f[VE];
      unpack(v[u], f);
      q[u] = fmaxf(f[0], f[1]);
#pragma unroll
      for (int e = 2; e < VE; e += 2) q[u] = max3(q[u], f[e], f[e + 1]);
    }
    const float top = fmaxf(max3(q[0], q[1], q[2]), q[3]);
    // ---- sum: the reference follows the maximum only when it has to
    if (top - m > 40.f) {  // (every larger value, from 2^29 on)
      s = beam_far(m) || beam_far(top) ? 0.f : s * exp2_approx(beam_ref(m) - beam_ref(top));
      m = top;
      c = beam_ref(m);
    }
    float part = 0.f;
    if (!beam_far(m)) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < kBeamVecs; ++u) {
        float f[VE];
        unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < VE; e += 2) {
          float2 d = fma2(make_float2(f[e], f[e + 1]), make_float2(kBeamLog2e, kBeamLog2e), make_float2(-c, -c));
          d.x = exp2_approx(d.x);
          d.y = exp2_approx(d.y);
          sum = add2(sum, d);
        }
      }
      part = sum.x + sum.y;
    }
    if (beam_far(m) || !(part < INFINITY)) {  // counted values, or a NaN among them
      part = 0.f;
#pragma unroll
      for (int u = 0; u < kBeamVecs; ++u) {
        float f[VE];
        unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if (beam_far(m))
            part += f[e] == m && m > -INFINITY ? 1.f : 0.f;
          else if (f[e] == f[e])
            part += exp2_approx(fmaf(f[e], kBeamLog2e, -c));
        }
      }
    }
    s += part;
    // ---- candidates
    if (first) {
      // the k-th of the warp's 32 * kBeamVecs vector maxima: k values lie at or above it
      uint32_t kq[kBeamVecs];
#pragma unroll
      for (int u = 0; u < kBeamVecs; ++u) kq[u] = beam_logit_key(q[u]);
      const uint32_t most = __reduce_max_sync(0xffffffffu, max(max(kq[0], kq[1]), max(kq[2], kq[3])));
      // 32 lanes reach the least of their maxima; for more than 32 the least of all bounds the k-th
      const uint32_t least = __reduce_min_sync(0xffffffffu, p.k <= 32 ? max(max(kq[0], kq[1]), max(kq[2], kq[3]))
                                                                      : min(min(kq[0], kq[1]), min(kq[2], kq[3])));
      const uint32_t cut = beam_search(p.k, least, most, kLow, [&](uint32_t x) {
        uint32_t n = 0;
#pragma unroll
        for (int u = 0; u < kBeamVecs; ++u) n += kq[u] >= x ? 1u : 0u;
        return int(__reduce_add_sync(0xffffffffu, n));
      });
      if (lane == 0) atomicMax(&floor_key, cut);
      l.least = max(l.least, cut);
    }
    l.least = max(l.least, *reinterpret_cast<volatile uint32_t*>(&floor_key));
    float ge = beam_key_val(l.least);
    if (__any_sync(0xffffffffu, top >= ge)) {
      uint32_t mine = 0;  // this lane's values that enter
#pragma unroll
      for (int u = 0; u < kBeamVecs; ++u) {
        if (!__any_sync(0xffffffffu, q[u] >= ge)) continue;
        float f[VE];
        unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < VE; ++e) mine |= f[e] >= ge ? 1u << (u * VE + e) : 0u;
      }
      // one value of each lane at a time
      while (true) {
        const uint32_t b = __ballot_sync(0xffffffffu, mine != 0);
        if (!b) break;
        if (mine) {
          const int i = __ffs(mine) - 1, u = i / VE, e = i - u * VE;
          mine &= mine - 1;
          const uint4 w = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
          const int word = e * int(sizeof(T)) / 4;
          const uint32_t bits = word == 0 ? w.x : word == 1 ? w.y : word == 2 ? w.z : w.w;
          const float val = sizeof(T) == 4 ? __uint_as_float(bits) : __uint_as_float(e & 1 ? bits & 0xFFFF0000u : bits << 16);
          const uint32_t id = uint32_t(p.vstart + col + u * 32 * VE + e);
          l.buf[l.n + __popc(b & ((1u << lane) - 1u))] = beam_key(beam_logit_key(val), id);
        }
        l.n += __popc(b);
        __syncwarp();
        if (l.n > kBeamCap - 32) beam_cut<kLow>(l, p.k, &floor_key);
      }
      // later columns have higher ids: they have to beat the k-th, not to equal it
      if (l.kth) l.least = max(l.least, l.kth + 1);
    }
  };
  auto edge = [&](int n, int col) {  // columns col .. col + n - 1, n < VE
    uint4 v[kBeamVecs];
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) {
      float f[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = u == 0 && e == 0 && lane < n ? to_f(x[col + lane]) : -INFINITY;
      v[u] = pack_vec(f);
    }
    tile(v, col + lane, false);
  };
  if (warp == kBeamWarps) {
    int copied = min(rounds, kBeamStages);
    for (int r = 0; r + 1 < rounds; ++r) {
      if (r + kBeamStages < rounds && !__any_sync(0xffffffffu, *abort)) {
        const bool ok =
            mbar_wait_soon(empty + r % kBeamStages, uint32_t((r / kBeamStages) & 1), kBudget, abort);
        if (__all_sync(0xffffffffu, ok)) {
          if (lane == 0) copy(r + kBeamStages);
          copied = r + kBeamStages + 1;
        } else {
          *abort = 1;
        }
        __syncwarp();
      }
      if (refloor(r)) {  // (with or without an abort: the other warps come there)
        named_sync(1, kBeamThreads + 32);
        uint32_t key[kBeamWarps];
#pragma unroll
        for (int w = 0; w < kBeamWarps; ++w) key[w] = lane < count[w] ? uint32_t(buf[w][lane] >> 32) : 0;
        named_sync(1, kBeamThreads + 32);  // the buffers may change again
        beam_floor<kLow>(key, p.k, &floor_key);
      }
    }
    if (*abort) {  // copies in flight land before the memory goes away
      int never = 0;
      for (int i = max(0, copied - kBeamStages); i < copied; ++i)
        mbar_wait(full + i % kBeamStages, uint32_t((i / kBeamStages) & 1), kBudget, &never);
    }
    __syncwarp();
  } else {
    if (warp == 0 && head) edge(head, c0);
    for (int r = 0; r < rounds; ++r) {
      const int sg = r % kBeamStages, at = r * kBeamRound + warp * 32 * kBeamVecs + lane;
      const bool ok = mbar_wait_soon(full + sg, uint32_t((r / kBeamStages) & 1), kBudget, abort);
      if (!__all_sync(0xffffffffu, ok)) {
        *abort = 1;
        for (int i = r; i < rounds; ++i)
          if (refloor(i)) {  // the others come there
            if (lane == 0) count[warp] = 0;
            named_sync(1, kBeamThreads + 32);
            named_sync(1, kBeamThreads + 32);
          }
        break;
      }
      uint4 v[kBeamVecs];
      constexpr uint32_t kNone = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;  // -inf
#pragma unroll
      for (int u = 0; u < kBeamVecs; ++u)
        v[u] = at + 32 * u < nvec ? ring[sg * kBeamRound + warp * 32 * kBeamVecs + lane + 32 * u]
                                  : make_uint4(kNone, kNone, kNone, kNone);
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + sg);
      if (at - lane >= nvec) break;  // nothing more for this warp (the last round)
      tile(v, v0 + at * VE, r == 0);
      if (refloor(r)) {
        beam_drop(l, *reinterpret_cast<volatile uint32_t*>(&floor_key));
        if (lane == 0) count[warp] = l.n;
        named_sync(1, kBeamThreads + 32);
        named_sync(1, kBeamThreads + 32);  // warp 8 has the keys; it finds the floor under the next round
      }
    }
    if (warp == kBeamWarps - 1 && tail) edge(tail, c1 - tail);
  }
  __syncthreads();
  if (*abort && threadIdx.x == 0) atomicOr(&g_beam_status, kStatusTimeout);
  if (warp < kBeamWarps) {
    // ---- the chunk's sum
    float cm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
    s = warp_sum(beam_own(m, s) * beam_weight(m, cm));
    if (lane == 0) stat[warp] = make_float2(cm, s);
    // ---- the chunk's k best: the warps' candidates (at most 64 each) from the common floor on, ranked
    if (l.n > kBeamMaxK) beam_cut<kLow>(l, p.k, &floor_key);
    named_sync(2, kBeamThreads);
    const uint32_t fk = floor_key;
    for (int i = lane; i < l.n; i += 32) {
      const uint64_t o = l.buf[i];
      if (uint32_t(o >> 32) >= fk) all[atomicAdd(&total, 1)] = o;
    }
    named_sync(2, kBeamThreads);
    const int n = total;
    uint64_t* out = p.cand + (size_t(row) * p.nchunk + ch) * p.k;
    for (int i = threadIdx.x; i < n; i += kBeamThreads) {
      const uint64_t o = all[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += all[j] > o ? 1 : 0;
      if (rank < p.k) out[rank] = o;
    }
    for (int i = n + threadIdx.x; i < p.k; i += kBeamThreads) out[i] = 0;
    if (threadIdx.x == 0) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kBeamWarps; ++w) top = fmaxf(top, stat[w].x);
#pragma unroll
      for (int w = 0; w < kBeamWarps; ++w) sum += stat[w].y * beam_weight(stat[w].x, top);
      p.stat[size_t(row) * p.nchunk + ch] = BeamStat{top, sum};
    }
  }
}

struct BeamPickParams {
  const BeamStat* stat;  // [parts][rows][nchunk]
  const uint64_t* cand;  // [parts][rows][nchunk][k]
  size_t stat_part, cand_part;  // elements between the shards' blocks
  int parts, rows, nchunk;
  const float* scores;  // [G][W]
  const uint8_t* finished;  // [G][W] or NULL
  int W, k, kc;  // beams, candidates to pick, candidates a chunk
  int64_t eos;   // < 0: none
  float* out_scores;
  long long *out_parents, *out_tokens;
  uint8_t* out_finished;  // or NULL
};

// A candidate of the merge: better() is the selection's order.
struct BeamCand {
  double total;
  uint32_t b, id;
};
__device__ __forceinline__ bool beam_better(const BeamCand& x, const BeamCand& y) {
  if (x.total != y.total) return x.total > y.total;
  if (x.b != y.b) return x.b < y.b;
  return x.id < y.id;
}

// One CTA a prompt, bound by the latency of its steps (load, sums, floor, rank:
// 10.8 us alone with cold caches for 8 beams of 4 chunks). Totals are formed in
// fp64, so that two beams' candidates are not put in order by a rounding.
constexpr int kPickCap = 512;  // candidates ranked against each other
constexpr int kPickHeld = 4;   // keys a thread keeps in registers
constexpr int kPickAll = 96;   // candidates ranked without a floor

__global__ void __launch_bounds__(kBeamThreads) beam_pick_kernel(const BeamPickParams p) {
  // of each beam: total = (x - top) + base
  __shared__ double base[kBeamMaxW];
  __shared__ float top[kBeamMaxW];
  __shared__ uint8_t fin[kBeamMaxW];
  __shared__ BeamCand list[kPickCap];
  __shared__ int total;
  __shared__ uint32_t most_sh, least_sh;
  pdl_launch();
  pdl_wait();
  const int g = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = p.nchunk * p.kc, n = p.parts * p.W * per;
  // candidate i is of beam b; its key (a finished beam's were not written, and are not used)
  auto where = [&](int i, int& q, int& b, int& o) {
    q = i / (p.W * per);
    const int r = i - q * p.W * per;
    b = r / per;
    o = r - b * per;
  };
  auto key_at = [&](int i) -> uint64_t {
    int q, b, o;
    where(i, q, b, o);
    return __ldcg(p.cand + q * p.cand_part + size_t(g * p.W + b) * per + o);
  };
  uint64_t held[kPickHeld];  // the keys of the first candidates of each thread, loaded under the sums
#pragma unroll
  for (int h = 0; h < kPickHeld; ++h) held[h] = tid + h * kBeamThreads < n ? key_at(tid + h * kBeamThreads) : 0;
  if (tid == 0) {
    total = 0;
    most_sh = 0;
    least_sh = 0xFFFFFFFFu;
  }
  for (int b = warp; b < p.W; b += kBeamWarps) {  // a warp a beam
    const int row = g * p.W + b;
    const double sc = p.scores[row];
    const bool f = p.finished && p.finished[row];
    double bs = sc;
    float m = -INFINITY;
    if (!f) {
      const int n = p.parts * p.nchunk;
      auto at = [&](int i) {
        const int q = i / p.nchunk;
        return p.stat[q * p.stat_part + size_t(row) * p.nchunk + (i - q * p.nchunk)];
      };
      const BeamStat mine = lane < n ? at(lane) : BeamStat{-INFINITY, 0.f};
      m = mine.m;
      for (int i = lane + 32; i < n; i += 32) m = fmaxf(m, at(i).m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      double s = 0.0;
      constexpr double kLog2ed = 1.44269504088896340736, kLn2d = 0.69314718055994530942;
      auto add = [&](const BeamStat& t) {
        s += double(t.s) * (t.m == m ? 1.0 : exp2((double(t.m) - double(m)) * kLog2ed));
      };
      add(mine);
      for (int i = lane + 32; i < n; i += 32) add(at(i));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      bs = sc - kLn2d * log2(s);
    }
    if (lane == 0) {
      base[b] = bs;
      top[b] = m;
      fin[b] = f;
    }
  }
  __syncthreads();
  // candidate i with its key; total -inf: none
  auto cand = [&](int i, uint64_t key) {
    BeamCand c{-INFINITY, 0u, 0u};
    int q, b, o;
    where(i, q, b, o);
    c.b = b;
    if (fin[b]) {
      if (q || o) return c;
      c.id = uint32_t(p.eos);
      c.total = base[b];
    } else {
      if (!key) return c;
      c.id = 0xFFFFFFFFu - uint32_t(key);
      const float x = beam_key_val(uint32_t(key >> 32));
      c.total = (x == top[b] ? 0.0 : double(x) - double(top[b])) + base[b];
    }
    if (!(c.total > -INFINITY)) c.total = -INFINITY;  // (or NaN)
    return c;
  };
  auto each = [&](auto&& f) {
#pragma unroll
    for (int h = 0; h < kPickHeld; ++h)
      if (tid + h * kBeamThreads < n) f(cand(tid + h * kBeamThreads, held[h]));
    for (int i = tid + kPickHeld * kBeamThreads; i < n; i += kBeamThreads) f(cand(i, key_at(i)));
  };
  // a floor that k candidates reach: the k-th of the threads' best totals,
  // rounded to fp32 (which keeps the order); few candidates are all ranked
  uint32_t cut = 0;
  if (n > kPickAll) {
    float best = -INFINITY;
    each([&](const BeamCand& c) { best = fmaxf(best, float(c.total)); });
    const uint32_t key = beam_logit_key(best);
    const uint32_t hi = __reduce_max_sync(0xffffffffu, key), lo = __reduce_min_sync(0xffffffffu, key);
    if (lane == 0) {
      atomicMax(&most_sh, hi);
      atomicMin(&least_sh, lo);
    }
    __syncthreads();
    cut = beam_search(p.k, least_sh, most_sh, 0, [&](uint32_t v) { return __syncthreads_count(key >= v); });
  }
  each([&](const BeamCand& c) {
    const uint32_t ck = beam_logit_key(float(c.total));
    if (ck && ck >= cut) {
      const int at = atomicAdd(&total, 1);
      if (at < kPickCap) list[at] = c;
    }
  });
  __syncthreads();
  auto put = [&](int j, bool none, const BeamCand& c) {
    const size_t o = size_t(g) * p.k + j;
    const long long tok = none ? (p.eos >= 0 ? p.eos : 0) : (long long)c.id;
    const int par = none ? 0 : int(c.b);
    p.out_scores[o] = none ? -INFINITY : float(c.total);
    p.out_parents[o] = par;
    p.out_tokens[o] = tok;
    if (p.out_finished) p.out_finished[o] = (p.eos >= 0 && tok == p.eos) || fin[par];
  };
  const int got = total;
  if (got <= kPickCap) {
    for (int i = tid; i < got; i += kBeamThreads) {
      const BeamCand c = list[i];
      int rank = 0;
      for (int j = 0; j < got; ++j) rank += beam_better(list[j], c) ? 1 : 0;
      if (rank < p.k) put(rank, false, c);
    }
    for (int j = got + tid; j < p.k; j += kBeamThreads) put(j, true, BeamCand{});
    return;
  }
  // more equal totals than the list holds: the k best one after another
  BeamCand last{INFINITY, 0, 0};
  for (int j = 0; j < p.k; ++j) {
    BeamCand win{-INFINITY, ~0u, ~0u};
    each([&](const BeamCand& c) {
      if (c.total > -INFINITY && (j == 0 || beam_better(last, c)) && beam_better(c, win)) win = c;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      BeamCand c;
      c.total = __shfl_xor_sync(0xffffffffu, win.total, o);
      c.b = __shfl_xor_sync(0xffffffffu, win.b, o);
      c.id = __shfl_xor_sync(0xffffffffu, win.id, o);
      if (beam_better(c, win)) win = c;
    }
    __syncthreads();
    if (lane == 0) list[warp] = win;
    __syncthreads();
    for (int i = 0; i < kBeamWarps; ++i)
      if (beam_better(list[i], win)) win = list[i];
    last = win;
    if (tid == 0) put(j, win.b == ~0u, win);
  }
}

// ---------------------------------------------------------------------------
// Cache reordering: in every layer's K and V, row g * W + w takes the first
// lens[src] positions of row src = g * W + parents[g][w]. In place: a thread
// owns one 16-byte column (head, position, part of the head's vector) of all
// W rows, reads every row that another one takes, then writes, so no row is
// overwritten before it is read. A row that keeps its place is not written.
// Bound by HBM: 961 MB in 159 us, 6.0 TB/s (28 layers of 64 rows, 250 positions).
// ---------------------------------------------------------------------------
constexpr int kReorderLayers = 64;  // layers a launch
constexpr int kReorderThreads = 256;  // 165 us on the 7B shape's 64 rows; 64, 128 and 512 take 174

struct ReorderParams {
  void* k[kReorderLayers];
  void* v[kReorderLayers];
  const long long* parents;  // [G][W]
  const int* lens;           // device [G * W], or NULL: len for all
  int len;
  int G, W, hkv, cap;
  int rv;  // vectors a position of a head
};

template <typename Vec, int MAXW>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const ReorderParams p) {
  __shared__ int par[MAXW], len[MAXW];
  __shared__ int most;
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x;
  const int g = blockIdx.y / p.hkv, h = blockIdx.y - g * p.hkv;
  if (tid == 0) most = 0;
  __syncthreads();
  if (tid < MAXW) {
    int src = tid, n = 0;
    if (tid < p.W) {
      const long long q = p.parents[size_t(g) * p.W + tid];
      if (q >= 0 && q < p.W) src = int(q);
      if (src != tid) {
        n = p.lens ? p.lens[size_t(g) * p.W + src] : p.len;
        n = max(0, min(n, p.cap));
      }
    }
    par[tid] = src;
    len[tid] = n;
    if (n) atomicMax(&most, n);
  }
  __syncthreads();
  const long long col = (long long)blockIdx.x * kReorderThreads + tid;
  if (col >= (long long)most * p.rv) return;
  const int pos = int(col / p.rv);
  const int l = blockIdx.z >> 1;
  Vec* base = static_cast<Vec*>((blockIdx.z & 1) ? p.v[l] : p.k[l]);
  const size_t row = size_t(p.hkv) * p.cap * p.rv;
  base += size_t(g) * p.W * row + size_t(h) * p.cap * p.rv + col;
  Vec val[MAXW];
#pragma unroll
  for (int w = 0; w < MAXW; ++w)
    if (pos < len[w]) val[w] = base[par[w] * row];
#pragma unroll
  for (int w = 0; w < MAXW; ++w)
    if (pos < len[w]) base[w * row] = val[w];
}

}  // namespace mtpb
