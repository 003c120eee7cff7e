// Causal attention over whole prompts of different lengths, packed one behind
// the other. Prompt s holds tokens [starts[s], starts[s + 1]) of the packed
// rows; token i of it, query head h, KV head h / G (G = hq / hkv):
//   o_i = sum_{j <= i} exp(s_ij - m_i) v_j / sum_{j <= i} exp(s_ij - m_i),
//   s_ij = q_i . k_j / sqrt(hd), both sums over tokens of prompt s alone.
// q and out may hold a piece of the packed tokens, [first, first + n), against
// K and V of all. A token of no prompt gets 0, and so does one whose scores
// are all -inf.
//
// The (token, head) rows of a prompt that share a KV head are put side by
// side, G rows a token, and cut into tiles: an item is a tile and its prompt's
// keys up to the tile's last token. So a short prompt fills a tile with the
// heads of its few tokens, and of the keys at the diagonal only those of
// (rows / G) tokens are masked in vain.
//
// NaN and infinities go where the formula takes them and nowhere else: a score
// that is NaN makes its row NaN, a NaN among V the dim of the rows that see
// it, and what a token does not see does not reach it.
#pragma once

#include "tcgen05.cuh"

namespace mtpb {

struct PaParams {
  const void *q, *k, *v;
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // elements from token to token, from head to head
  void* out;          // [n][hq][hd]
  const int* starts;  // device [S + 1]
  int S, first, n, total, hq, hkv;
  int tiles;  // row tiles a KV head that the grid covers: at least as many as there are
  float scale;
  uint32_t* status;  // error bits
};

// Set when a bounded wait of a prompt attention ran out (its results are then void).
__device__ uint32_t g_pa_status;

constexpr float kPaLog2e = 1.44269504088896340736f;

// One tile's rows. Row r is token lo + (row0 + r) / G, query head
// kvh * G + (row0 + r) % G, of a prompt from token `start` on.
struct PaItem {
  int start, lo;  // packed tokens
  int row0, rows;  // rows 0: no tile; the CTA is then number `spare` of `spares`
  int spare, spares;
  int gap0, gap1;  // tokens [first, gap0) and [gap1, first + n) are of no prompt
};

// Prompts whose tiles are put in order (a lane has its share in registers).
constexpr int kPaOrdered = 4 * 32;

// Tile number i, by one warp. Tiles come in descending order of their place in
// their prompt, which is how many keys they see, over all prompts, so that
// the longest do not start last; with more than kPaOrdered prompts prompt after
// prompt. The starts are made non-decreasing and cut to [0, total] first, so
// that no values of theirs lead out of the tensors or make two tiles of a row.
template <int ROWS>
__device__ __forceinline__ PaItem pa_item(const PaParams& p, int i) {
  const int lane = threadIdx.x & 31, G = p.hq / p.hkv, end = p.first + p.n;
  PaItem it;
  it.start = it.lo = it.row0 = it.rows = 0;
  auto cut = [&](int t) { return min(max(t, 0), p.total); };
  int at_least = cut(__ldg(p.starts));  // the largest start so far
  it.gap0 = min(max(at_least, p.first), end);
  struct Seq {
    int start, lo, rows, nt, off;  // off: place of the first tile
  };
  auto load = [&](int b) {  // prompt 32 b + lane
    const int s = 32 * b + lane;
    int hi = max(at_least, s < p.S ? cut(__ldg(p.starts + s + 1)) : 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, hi, o);
      if (lane >= o) hi = max(hi, u);
    }
    const int prev = __shfl_up_sync(0xffffffffu, hi, 1);
    Seq q;
    q.start = lane ? prev : at_least;
    q.lo = max(q.start, p.first);
    q.rows = max(0, min(hi, end) - q.lo) * G;
    q.nt = (q.rows + ROWS - 1) / ROWS;
    q.off = q.rows ? int((long long)(q.lo - q.start) * G / ROWS) : 0;
    at_least = __shfl_sync(0xffffffffu, hi, 31);
    return q;
  };
  auto take = [&](int from, const Seq& q, int tile) {  // tile of lane `from`'s prompt
    it.start = __shfl_sync(0xffffffffu, q.start, from);
    it.lo = __shfl_sync(0xffffffffu, q.lo, from);
    it.row0 = tile * ROWS;
    it.rows = min(ROWS, __shfl_sync(0xffffffffu, q.rows, from) - it.row0);
  };
  int all = 0;
  if (p.S <= kPaOrdered) {
    Seq q[kPaOrdered / 32];
    int most = 0;
#pragma unroll
    for (int b = 0; b < kPaOrdered / 32; ++b) {
      q[b] = Seq{0, 0, 0, 0, 0};
      if (32 * b < p.S) q[b] = load(b);
      if (q[b].nt) most = max(most, q[b].off + q[b].nt);
      all += q[b].nt;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    all = __reduce_add_sync(0xffffffffu, all);
    if (i < all) {
      auto above = [&](int c) {  // tiles at place c or behind it
        int n = 0;
#pragma unroll
        for (int b = 0; b < kPaOrdered / 32; ++b) n += max(0, q[b].off + q[b].nt - max(c, q[b].off));
        return __reduce_add_sync(0xffffffffu, n);
      };
      int lo = 0, hi = most;  // above(lo) > i >= above(hi)
      while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (above(mid) > i)
          lo = mid;
        else
          hi = mid;
      }
      int left = i - above(lo + 1);  // of the tiles at place lo
#pragma unroll
      for (int b = 0; b < kPaOrdered / 32; ++b) {
        const uint32_t m = __ballot_sync(0xffffffffu, q[b].off <= lo && lo < q[b].off + q[b].nt);
        const int c = __popc(m);
        if (left >= 0 && left < c) {
          const int from = __fns(m, 0, left + 1);
          take(from, q[b], lo - __shfl_sync(0xffffffffu, q[b].off, from));
        }
        left -= c;
      }
    }
  } else {
    for (int b = 0; 32 * b < p.S; ++b) {
      const Seq q = load(b);
      int upto = q.nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const int sum = __shfl_sync(0xffffffffu, upto, 31);
      if (i >= all && i < all + sum) {
        const int from = __popc(__ballot_sync(0xffffffffu, all + upto <= i));
        take(from, q, all + __shfl_sync(0xffffffffu, upto, from) - 1 - i);  // a prompt's last tile first
      }
      all += sum;
    }
  }
  it.gap1 = min(max(at_least, p.first), end);
  it.spare = i - all;
  it.spares = p.tiles - all;
  return it;
}

// What a CTA without a tile does: its share of the tokens of no prompt gets 0.
template <typename T>
__device__ __forceinline__ void pa_zero(const PaParams& p, const PaItem& it, int kvh, int hd, int threads) {
  constexpr int VE = VecTraits<T>::kElems;
  const int G = p.hq / p.hkv, vecs = G * hd / VE;  // of a token
  const int n0 = it.gap0 - p.first, n1 = p.first + p.n - it.gap1;
  for (int t = it.spare; t < n0 + n1; t += it.spares) {
    const int at = t < n0 ? t : it.gap1 - p.first + (t - n0);
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + ((size_t)at * p.hq + size_t(kvh) * G) * hd);
    for (int i = threadIdx.x; i < vecs; i += threads) o[i] = make_uint4(0, 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------
// Tiles on the CUDA cores: fp32, and bf16 with head dims 16 and 32 (the models
// served have 64 and 128; those are on the tensor cores). 256 threads as 16 x
// 16; RPT rows and 4 keys a thread of a tile of 16 RPT rows and 64 keys, in
// fp32; a row's 16 threads are half a warp, so its probabilities go through
// shared memory without a barrier of the CTA.
// ---------------------------------------------------------------------------
constexpr int kPaKeys = 64;
constexpr int kPaThreads = 256;

template <int HD, int RPT>
constexpr size_t pa_simt_smem() {
  return sizeof(float) * (size_t(16 * RPT) * (HD + 4) + size_t(kPaKeys) * (HD + 4) + size_t(kPaKeys) * (HD + 4) +
                          size_t(16 * RPT) * (kPaKeys + 4));
}

template <typename T, int HD, int RPT>
__global__ void __launch_bounds__(kPaThreads) pa_simt_kernel(const PaParams p) {
  constexpr int ROWS = 16 * RPT, LD = HD + 4, LP = kPaKeys + 4, VE = VecTraits<T>::kElems;
  constexpr int DP = HD / 16;  // dims a thread of the result: tx, tx + 16, ..
  extern __shared__ __align__(16) float pa_sm[];
  float* sq = pa_sm;
  float* sk = sq + ROWS * LD;
  float* sv = sk + kPaKeys * LD;
  float* sp = sv + kPaKeys * LD;
  __shared__ PaItem it_sh;
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, G = p.hq / p.hkv;
  const int kvh = blockIdx.x % p.hkv;
  if (tid < 32) {
    const PaItem it = pa_item<ROWS>(p, blockIdx.x / p.hkv);
    if (tid == 0) it_sh = it;
  }
  __syncthreads();
  const PaItem it = it_sh;
  if (it.rows <= 0) {
    pa_zero<T>(p, it, kvh, HD, kPaThreads);
    return;
  }
  const T* q = static_cast<const T*>(p.q);
  const T* k = static_cast<const T*>(p.k) + kvh * p.k_hs;
  const T* v = static_cast<const T*>(p.v) + kvh * p.v_hs;
  auto token = [&](int r) { return it.lo + (it.row0 + r) / G; };
  for (int i = tid; i < ROWS * (HD / VE); i += kPaThreads) {
    const int r = i / (HD / VE), c = (i - r * (HD / VE)) * VE;
    float f[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = 0.f;
    if (r < it.rows) {
      const int row = it.row0 + r;
      unpack(ld_vec(q + (it.lo + row / G - p.first) * p.q_ts + (kvh * G + row % G) * p.q_hs + c), f);
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) sq[r * LD + c + e] = f[e];
  }
  int lim[RPT];  // keys [0, lim) of the prompt are seen
#pragma unroll
  for (int a = 0; a < RPT; ++a) lim[a] = token(min(ty * RPT + a, it.rows - 1)) + 1 - it.start;
  const int keys = token(it.rows - 1) + 1 - it.start, low = token(0) + 1 - it.start;
  float o[RPT][DP], m[RPT], l[RPT];
#pragma unroll
  for (int a = 0; a < RPT; ++a) {
    m[a] = -INFINITY;
    l[a] = 0.f;
#pragma unroll
    for (int d = 0; d < DP; ++d) o[a][d] = 0.f;
  }
  const float sl2 = p.scale * kPaLog2e;
  for (int j = 0; j < keys; j += kPaKeys) {
    __syncthreads();
    for (int i = tid; i < kPaKeys * (HD / VE); i += kPaThreads) {
      const int r = i / (HD / VE), c = (i - r * (HD / VE)) * VE;
      float f[VE], g[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = g[e] = 0.f;
      if (j + r < keys) {
        unpack(ld_vec(k + (long long)(it.start + j + r) * p.k_ts + c), f);
        unpack(ld_vec(v + (long long)(it.start + j + r) * p.v_ts + c), g);
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        sk[r * LD + c + e] = f[e];
        sv[r * LD + c + e] = g[e];
      }
    }
    __syncthreads();
    float s[RPT][4];
#pragma unroll
    for (int a = 0; a < RPT; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) s[a][b] = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      float4 kk[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) kk[b] = *reinterpret_cast<const float4*>(sk + (tx + 16 * b) * LD + d);
#pragma unroll
      for (int a = 0; a < RPT; ++a) {
        const float4 qq = *reinterpret_cast<const float4*>(sq + (ty * RPT + a) * LD + d);
#pragma unroll
        for (int b = 0; b < 4; ++b)
          s[a][b] = fmaf(qq.w, kk[b].w, fmaf(qq.z, kk[b].z, fmaf(qq.y, kk[b].y, fmaf(qq.x, kk[b].x, s[a][b]))));
      }
    }
    const bool masked = j + kPaKeys > low;
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        s[a][b] *= sl2;
        if (masked && j + tx + 16 * b >= lim[a]) s[a][b] = -INFINITY;
        top = fmaxf(top, s[a][b]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(m[a], top);
      const float ref = top == -INFINITY ? 0.f : top, w = exp2f(m[a] - ref);
      m[a] = top;
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float e = exp2f(s[a][b] - ref);
        sum += e;
        sp[(ty * RPT + a) * LP + tx + 16 * b] = e;
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[a] = fmaf(l[a], w, sum);
#pragma unroll
      for (int d = 0; d < DP; ++d) o[a][d] *= w;
    }
    __syncwarp();
    const int nk = min(kPaKeys, keys - j);
    if (!masked) {
#pragma unroll 2
      for (int key = 0; key < kPaKeys; key += 4) {
        float4 pp[RPT];
#pragma unroll
        for (int a = 0; a < RPT; ++a) pp[a] = *reinterpret_cast<const float4*>(sp + (ty * RPT + a) * LP + key);
#pragma unroll
        for (int d = 0; d < DP; ++d) {
          const float v0 = sv[key * LD + tx + 16 * d], v1 = sv[(key + 1) * LD + tx + 16 * d];
          const float v2 = sv[(key + 2) * LD + tx + 16 * d], v3 = sv[(key + 3) * LD + tx + 16 * d];
#pragma unroll
          for (int a = 0; a < RPT; ++a)
            o[a][d] = fmaf(pp[a].w, v3, fmaf(pp[a].z, v2, fmaf(pp[a].y, v1, fmaf(pp[a].x, v0, o[a][d]))));
        }
      }
    } else {  // a key that a row does not see adds nothing to it, whatever its V
      for (int key = 0; key < nk; ++key)
#pragma unroll
        for (int a = 0; a < RPT; ++a) {
          const float pr = sp[(ty * RPT + a) * LP + key];
#pragma unroll
          for (int d = 0; d < DP; ++d) {
            const float x = fmaf(pr, sv[key * LD + tx + 16 * d], o[a][d]);
            o[a][d] = j + key < lim[a] ? x : o[a][d];
          }
        }
    }
    __syncwarp();
  }
#pragma unroll
  for (int a = 0; a < RPT; ++a) {
    const int r = ty * RPT + a, row = it.row0 + r;
    if (r < it.rows) {
      T* out = static_cast<T*>(p.out) + (size_t(it.lo + row / G - p.first) * p.hq + kvh * G + row % G) * HD;
#pragma unroll
      for (int d = 0; d < DP; ++d) out[tx + 16 * d] = from_f<T>(l[a] == 0.f ? 0.f : o[a][d] / l[a]);
    }
  }
}

}  // namespace mtpb
