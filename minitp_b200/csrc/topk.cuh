// Selecting the k best of a row of logits: keys, a warp's candidate list, and
// the reference of a lane's sum of exponentials (beam selection,
// log-probabilities).
#pragma once

#include "tma.cuh"

namespace mtpb {

constexpr int kBeamMaxK = 64;
constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;

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

}  // namespace mtpb
