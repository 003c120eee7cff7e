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
// A row is cut into chunks; each is reduced to its statistics and its k best
// logits (packed keys: value, then lower id), and a second kernel joins the
// chunks, of every shard of the vocabulary.
#pragma once

#include "common.cuh"

namespace mtpb {

constexpr int kLpMaxK = 64;

// Of a chunk: m = max x, s = sum exp(x - m), w = sum exp(x - m) (x - m), and
// the target's logit (NaN: the target lies elsewhere). m -inf: no token.
struct LpStat {
  float m, s, w, xt;
};

struct LpRowsParams {
  const void* logits;
  int64_t ld;      // elements between rows
  int V, k;        // columns of this shard, candidates a chunk
  int64_t vstart;  // id of column 0
  int nchunk, chunk;
  const long long* targets;  // [rows] or NULL
  LpStat* stat;    // [rows][nchunk]
  uint64_t* cand;  // [rows][nchunk][k], best first, 0-padded
};

__device__ __forceinline__ uint64_t lp_key(float v, uint32_t id) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(v + 0.f);  // (-0 as +0)
  return (uint64_t(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ float lp_key_val(uint64_t o) {
  const uint32_t k = uint32_t(o >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ uint64_t lp_warp_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

constexpr int kLpThreads = 256;

// A CTA a row and chunk: the maximum, the sums, and k times the best below the last.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) lp_rows_kernel(const LpRowsParams p) {
  __shared__ float red[32];
  __shared__ uint64_t best[kLpThreads / 32];
  pdl_launch();
  pdl_wait();
  const size_t row = blockIdx.x / p.nchunk;
  const int ch = blockIdx.x % p.nchunk, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c0 = min(p.V, ch * p.chunk), c1 = min(p.V, c0 + p.chunk);
  const T* x = static_cast<const T*>(p.logits) + int64_t(row) * p.ld;
  auto at = [&](int c) {
    const float v = to_f(x[c]);
    return v == v ? v : -INFINITY;
  };
  float m = -INFINITY;
  for (int c = c0 + tid; c < c1; c += kLpThreads) m = fmaxf(m, at(c));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = red[0];
  for (int i = 1; i < kLpThreads / 32; ++i) m = fmaxf(m, red[i]);
  float s = 0.f, w = 0.f;
  if (m > -INFINITY)
    for (int c = c0 + tid; c < c1; c += kLpThreads) {
      const float v = at(c), d = v == m ? 0.f : v - m, e = expf(d);
      s += e;
      if (e > 0.f) w = fmaf(e, d, w);
    }
  s = block_sum(s, red);
  w = block_sum(w, red);
  if (tid == 0) {
    LpStat st{m, s, w, __int_as_float(0x7fffffff)};
    if (p.targets) {
      const long long c = p.targets[row] - p.vstart;
      if (c >= c0 && c < c1) st.xt = at(int(c));
    }
    p.stat[row * p.nchunk + ch] = st;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < p.k; ++i) {
    uint64_t b = 0;
    if (last)
      for (int c = c0 + tid; c < c1; c += kLpThreads) {
        const uint64_t o = lp_key(at(c), uint32_t(p.vstart + c));
        if (o < last && o > b) b = o;
      }
    b = lp_warp_max(b);
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    for (int j = 0; j < kLpThreads / 32; ++j) b = best[j] > b ? best[j] : b;
    last = b;
    if (tid == 0) p.cand[(row * p.nchunk + ch) * p.k + i] = b;
  }
}

struct LpJoinParams {
  const LpStat* stat;    // [parts][rows][nchunk]
  const uint64_t* cand;  // [parts][rows][nchunk][kc]
  size_t stat_part, cand_part;  // elements between the shards' blocks
  int parts, rows, nchunk, k, kc;
  const long long* targets;  // [rows] or NULL
  float *logprobs, *entropy;  // [rows]; logprobs NULL without targets
  float* top_logprobs;        // [rows][k]
  long long* top_ids;
};

constexpr int kLpJoinWarps = 4;
constexpr int kLpMaxLists = 64 * 32;  // shards x chunks

// A warp a row, in fp64. The lists of the chunks are sorted: the best of their
// heads is the next, k times.
__global__ void __launch_bounds__(32 * kLpJoinWarps) lp_join_kernel(const LpJoinParams p) {
  extern __shared__ uint8_t lp_heads[];  // [warps][lists]: entries of each list that were taken
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lists = p.parts * p.nchunk;
  const size_t row = size_t(blockIdx.x) * kLpJoinWarps + warp;
  if (row >= p.rows) return;
  auto stat = [&](int i) { return p.stat + (i / p.nchunk) * p.stat_part + row * p.nchunk + i % p.nchunk; };
  auto cand = [&](int i) { return p.cand + (i / p.nchunk) * p.cand_part + (row * p.nchunk + i % p.nchunk) * p.kc; };
  float m = -INFINITY, xt = -INFINITY;
  bool found = false;
  for (int i = lane; i < lists; i += 32) {
    const LpStat s = *stat(i);
    m = fmaxf(m, s.m);
    if (s.xt == s.xt) {
      xt = s.xt;
      found = true;
    }
  }
  found = __any_sync(0xffffffffu, found);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    xt = fmaxf(xt, __shfl_xor_sync(0xffffffffu, xt, o));
  }
  double sum = 0.0, w = 0.0;
  for (int i = lane; i < lists; i += 32) {
    const LpStat s = *stat(i);
    if (s.m == -INFINITY) continue;
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
    if (x == -INFINITY) return -INFINITY;
    return float((x == m ? 0.0 : double(x) - double(m)) - logs);
  };
  if (lane == 0) {
    p.entropy[row] = sum > 0.0 ? float(logs - w / sum) : 0.f;
    if (p.logprobs) p.logprobs[row] = found ? logp(xt) : __int_as_float(0x7fffffff);
  }
  if (!p.k) return;
  uint8_t* head = lp_heads + warp * lists;
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
    const uint64_t top = lp_warp_max(b);
    if (top && b == top) ++head[at];
    if (lane == 0) {
      p.top_logprobs[row * p.k + j] = top ? logp(lp_key_val(top)) : -INFINITY;
      p.top_ids[row * p.k + j] = top ? (long long)(0xFFFFFFFFu - uint32_t(top)) : 0;
    }
  }
}

}  // namespace mtpb
