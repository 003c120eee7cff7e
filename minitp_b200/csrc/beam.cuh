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
// vocabulary is cut into chunks: one CTA per (row, chunk) finds the chunk's
// max, sum and k best logits (packed keys: value, then lower id), and one CTA
// per prompt merges the chunks of all its beams.
#pragma once

#include "common.cuh"

namespace mtpb {

constexpr int kBeamMaxK = 64;
constexpr int kBeamMaxW = 64;

struct BeamStat {
  float m, s;  // max of the chunk's logits and sum of exp(x - m)
};

// Order-preserving key of a finite or +inf logit and its id; 0: no candidate.
__device__ __forceinline__ uint32_t beam_val_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_key_val(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ uint64_t beam_key(float v, uint32_t id) {
  if (v == -INFINITY) return 0;
  return (uint64_t(beam_val_key(v == 0.f ? 0.f : v)) << 32) | (0xFFFFFFFFu - id);
}

// max of key over the block; valid in every thread. `red`: one word per warp.
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  for (int i = 0; i < nw; ++i) v = red[i] > v ? red[i] : v;
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

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_rows_kernel(const BeamRowsParams p) {
  __shared__ uint64_t red[kBeamThreads / 32];
  __shared__ float redf[kBeamThreads / 32];
  pdl_launch();
  pdl_wait();
  const int row = blockIdx.y, ch = blockIdx.x;
  if (p.finished && p.finished[row]) return;
  const int c0 = ch * p.chunk, c1 = min(p.V, c0 + p.chunk);
  const T* x = static_cast<const T*>(p.logits) + int64_t(row) * p.ld;
  uint64_t* out = p.cand + (size_t(row) * p.nchunk + ch) * p.k;
  uint64_t last = ~0ull;
  float m = -INFINITY;
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    for (int c = c0 + threadIdx.x; c < c1; c += kBeamThreads) {
      const uint64_t key = beam_key(fmaxf(to_f(x[c]), -INFINITY), uint32_t(p.vstart + c));
      if (key < last && key > best) best = key;
    }
    best = block_max_u64(best, red);
    if (threadIdx.x == 0) out[j] = best;
    if (j == 0) m = best ? beam_key_val(uint32_t(best >> 32)) : -INFINITY;
    last = best;
    if (best == 0) {
      for (int i = j + 1 + threadIdx.x; i < p.k; i += kBeamThreads) out[i] = 0;
      break;
    }
  }
  float s = 0.f;
  for (int c = c0 + threadIdx.x; c < c1; c += kBeamThreads)
    s += expf(fminf(fmaxf(to_f(x[c]), -INFINITY) - m, 0.f));
  s = block_sum(s, redf);
  if (threadIdx.x == 0) p.stat[size_t(row) * p.nchunk + ch] = BeamStat{m, s};
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

__global__ void __launch_bounds__(kBeamThreads) beam_pick_kernel(const BeamPickParams p) {
  // per beam: score - (max + log sum), as total = (x - max) + base; base NaN: no candidate
  __shared__ double base[kBeamMaxW];
  __shared__ float top[kBeamMaxW];
  __shared__ double red_t[kBeamThreads / 32];
  __shared__ uint32_t red_b[kBeamThreads / 32], red_i[kBeamThreads / 32];
  pdl_launch();
  pdl_wait();
  const int g = blockIdx.x, tid = threadIdx.x;
  if (tid < p.W) {
    const int row = g * p.W + tid;
    const double sc = p.scores[row];
    if (p.finished && p.finished[row]) {
      top[tid] = 0.f;
      base[tid] = sc;
    } else {
      float m = -INFINITY;
      for (int q = 0; q < p.parts; ++q)
        for (int c = 0; c < p.nchunk; ++c) m = fmaxf(m, p.stat[q * p.stat_part + size_t(row) * p.nchunk + c].m);
      double s = 0.0;
      for (int q = 0; q < p.parts; ++q)
        for (int c = 0; c < p.nchunk; ++c) {
          const BeamStat t = p.stat[q * p.stat_part + size_t(row) * p.nchunk + c];
          if (t.m != -INFINITY) s += double(t.s) * exp(t.m == m ? 0.0 : double(t.m) - double(m));
        }
      top[tid] = m;
      base[tid] = sc - log(s);
    }
  }
  __syncthreads();
  const int n = p.parts * p.W * p.nchunk * p.kc;
  BeamCand last{INFINITY, 0, 0};
  bool first = true;
  for (int j = 0; j < p.k; ++j) {
    BeamCand best{-INFINITY, ~0u, ~0u};
    for (int i = tid; i < n; i += kBeamThreads) {
      const int per = p.nchunk * p.kc;
      const int q = i / (p.W * per), r = i - q * p.W * per, b = r / per, o = r - b * per;
      const int row = g * p.W + b;
      BeamCand c;
      c.b = b;
      if (p.finished && p.finished[row]) {
        if (q || o) continue;
        c.id = uint32_t(p.eos);
        c.total = base[b];
      } else {
        const uint64_t key = p.cand[q * p.cand_part + size_t(row) * per + o];
        if (!key) continue;
        c.id = 0xFFFFFFFFu - uint32_t(key);
        const float x = beam_key_val(uint32_t(key >> 32));
        c.total = (x == top[b] ? 0.0 : double(x) - double(top[b])) + base[b];
      }
      if (!(c.total > -INFINITY)) continue;
      if (!first && !beam_better(last, c)) continue;
      if (beam_better(c, best)) best = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      BeamCand c;
      c.total = __shfl_xor_sync(0xffffffffu, best.total, o);
      c.b = __shfl_xor_sync(0xffffffffu, best.b, o);
      c.id = __shfl_xor_sync(0xffffffffu, best.id, o);
      if (beam_better(c, best)) best = c;
    }
    __syncthreads();
    if ((tid & 31) == 0) {
      red_t[tid >> 5] = best.total;
      red_b[tid >> 5] = best.b;
      red_i[tid >> 5] = best.id;
    }
    __syncthreads();
    for (int i = 0; i < kBeamThreads / 32; ++i) {
      const BeamCand c{red_t[i], red_b[i], red_i[i]};
      if (beam_better(c, best)) best = c;
    }
    last = best;
    first = false;
    if (tid == 0) {
      const bool none = best.b == ~0u;
      const size_t o = size_t(g) * p.k + j;
      const long long tok = none ? (p.eos >= 0 ? p.eos : 0) : (long long)best.id;
      const int par = none ? 0 : int(best.b);
      p.out_scores[o] = none ? -INFINITY : float(best.total);
      p.out_parents[o] = par;
      p.out_tokens[o] = tok;
      if (p.out_finished)
        p.out_finished[o] = (p.eos >= 0 && tok == p.eos) || (p.finished && p.finished[size_t(g) * p.W + par]);
    }
  }
}

// ---------------------------------------------------------------------------
// Cache reordering: in every layer's K and V, row g * W + w takes the first
// lens[src] positions of row src = g * W + parents[g][w]. In place: a thread
// owns one 16-byte column (head, position, part of the head's vector) of all
// W rows, reads every row that another one takes, then writes, so no row is
// overwritten before it is read. A row that keeps its place is not written.
// ---------------------------------------------------------------------------
constexpr int kReorderLayers = 64;  // layers a launch
constexpr int kReorderThreads = 128;

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
