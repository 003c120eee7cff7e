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

#include <type_traits>

#include "softmax.cuh"

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
  const float sl2 = p.scale * kLog2e;
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

// ---------------------------------------------------------------------------
// Tiles on the tensor cores (bf16, head dim 64 or 128), one item a CTA, key
// tiles of 128. Two streams share the ring of K and V tiles, each with an MMA
// warp, a softmax warpgroup (a row a thread) and its own tensor memory:
//   MT 2: stream x has rows 128 x .. of the item's 256 and their keys, so a
//         K/V byte brought in from L2 serves 256 rows;
//   MT 1: both have the item's 128 rows, stream x the key tiles t = x mod 2,
//         and the streams are joined at the end.
// One stream's softmax runs under the other's and under the MMAs:
//   warp 0 loads (TMA, 128 keys x 64 dims boxes, 128-byte swizzle), warps 1
//   and 2 issue S = Q K^T and O += P V of their stream, warps 4-7 and 8-11
//   turn S into P, with the registers that warps 0-3 hand over (56 and 224 of
//   168 a thread at launch).
// P is bf16 in tensor memory, the A operand of P V; for head dim 128, where S
// and O fill the 512 columns, it takes the place of its S, and the stream's
// next S waits for the P V that reads it. V is read as it lies (N-major B).
// The max that the exponentials are taken against is replaced, and O rescaled
// in tensor memory, only when a row's max has grown by more than 2^8: until
// then P is at most 2^8, which costs no precision, as the division by the sum
// takes the factor out.
// Keys that a row does not see are masked by selection. V rows behind the
// tile's last key are zeroed in shared memory, since 0 x NaN would not be 0;
// of those that not every row of the tile sees, the NaN and infinities are
// zeroed and added at the end to the rows that do see them.
// ---------------------------------------------------------------------------
constexpr int kPaTcKeys = 128;
constexpr int kPaTcThreads = 384;
constexpr int kPaCubic = 4;  // of 16 pairs of exponentials, on the fp32 pipe

template <int HD, int MT>
struct PaTcCfg {
  static constexpr int kSubs = HD / 64;
  static constexpr uint32_t kTile = kSubs * kTcSub;  // a K, V or Q tile
  // ring of K and V tiles: what 224 KB leave beside Q (at most six of each)
  static constexpr int kRing = HD == 128 ? 7 - MT : 12;
  static constexpr uint32_t kOffRing = MT * kTile;
  static constexpr size_t kSmem = size_t(kOffRing) + kRing * kTile + 1024;
  static constexpr bool kAlias = HD == 128;  // P in the place of S
  static constexpr uint32_t kS = 128;        // columns from stream to stream of S; of O: HD
  static constexpr uint32_t kO = 256, kP = kAlias ? 0 : 384, kPStep = kAlias ? 128 : 64;
  static constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);
  // B of P V: N (dims) contiguous
  static constexpr uint32_t kIdescO =
      (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(HD >> 3) << 17) | (uint32_t(128 >> 4) << 24);
};

template <int HD, int MT>
__global__ void __launch_bounds__(kPaTcThreads, 1)
    pa_tc_kernel(const PaParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using C = PaTcCfg<HD, MT>;
  constexpr int NB = C::kRing, ROWS = 128 * MT;
  constexpr uint64_t kBudget = 2000000000ull;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[NB], empty[NB], qfull, s_full[2], s_free[2], p_full[2][2], pv_done[2], drain[2], turn[2][4];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_sh, odd_sh;  // odd_sh: values of V were zeroed
  __shared__ float2 ml_sh[128];  // MT 1: stream 1's statistics
  __shared__ PaItem it_sh;
  volatile int* abort = &abort_sh;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  const int G = p.hq / p.hkv, kvh = blockIdx.x % p.hkv;
  pdl_launch();
  pdl_wait();
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp == 0) {
    const PaItem mine = pa_item<ROWS>(p, blockIdx.x / p.hkv);
    if (lane == 0) it_sh = mine;
  } else if (threadIdx.x == 32) {
    for (int s = 0; s < NB; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, MT);  // each stream that reads the tile
    }
    mbar_init(&qfull, 8);
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_full + x, 1);
      mbar_init(s_free + x, 4);
      for (int h = 0; h < 2; ++h) mbar_init(&p_full[x][h], 4);
      mbar_init(pv_done + x, 1);
      mbar_init(drain + x, 1);
      for (int q = 0; q < 4; ++q) mbar_init(&turn[x][q], 1);
    }
    *abort = 0;
    odd_sh = 0;
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  const PaItem it = it_sh;
  // keys of the prompt that row r of the tile sees
  auto seen = [&](int r) { return it.lo + (it.row0 + r) / G + 1 - it.start; };
  const int keys = it.rows > 0 ? seen(it.rows - 1) : 0;
  // tiles of stream x: first, step, and how many
  constexpr int kStep = MT == 2 ? 1 : 2;
  const int nt = (keys + kPaTcKeys - 1) / kPaTcKeys;
  auto tiles_of = [&](int x) {
    if (MT == 1) return (nt - x + 1) / 2;
    return it.rows > 128 * x ? (seen(min(it.rows, 128 * x + 128) - 1) + kPaTcKeys - 1) / kPaTcKeys : 0;
  };

  // the end of every role: nobody uses tensor or shared memory any more
  auto leave = [&]() {
    tc_fence_before();
    __syncwarp();
    named_sync(2, kPaTcThreads);
    if (warp == 3) {
      tc_fence_after();
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
      if (lane == 0 && *abort) atomicOr(p.status ? p.status : &g_pa_status, kStatusTimeout);
    }
  };

  if (it.rows <= 0) {
    pa_zero<bf16>(p, it, kvh, HD, kPaTcThreads);
    leave();
  } else if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      int issued = 0;  // ring entries whose copies were issued
      for (int i = 0; i < 2 * nt; ++i) {  // K and V of each tile in turn
        const int s = i % NB, j = it.start + (i >> 1) * kPaTcKeys;
        const bool ok = i < NB || mbar_wait_soon(empty + s, uint32_t((i / NB) & 1) ^ 1u, kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) {
          *abort = 1;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(full + s, C::kTile);
#pragma unroll
          for (int b = 0; b < C::kSubs; ++b)
            tma_load_3d(base + C::kOffRing + s * C::kTile + b * kTcSub, i & 1 ? &map_v : &map_k, b * 64, j, kvh, full + s);
        }
        issued = i + 1;
      }
      // copies in flight land before the memory goes away
      int never = 0;
      for (int i = max(0, issued - NB); i < issued; ++i) mbar_wait(full + i % NB, uint32_t((i / NB) & 1), kBudget, &never);
    } else if (warp < 3) {
      // ---- MMA issue of stream x
      const int x = warp - 1, first = MT == 2 ? 0 : x, mine = tiles_of(x);
      const uint64_t dq = tc_smem_desc(base + (MT == 2 ? x : 0) * C::kTile);
      const uint32_t ts = tmem + x * C::kS, to = tmem + C::kO + x * HD, tp = tmem + C::kP + x * C::kPStep;
      auto wait = [&](uint64_t* bar, int phase) {
        return __all_sync(0xffffffffu, mbar_wait_soon(bar, uint32_t(phase & 1), kBudget, abort));
      };
      auto qk = [&](int k) {
        const int i = 2 * (first + k * kStep), s = i % NB;
        // S is free: read by the softmax, and (aliased) its P read by P V
        if (!wait(full + s, i / NB) || (k > 0 && !wait(C::kAlias ? pv_done + x : s_free + x, k - 1))) return false;
        tc_fence_after();
        const uint64_t dk = tc_smem_desc(base + C::kOffRing + s * C::kTile);
        if (elect_one()) {
#pragma unroll
          for (int q = 0; q < HD / 16; ++q) {
            const uint32_t off = ((q >> 2) * kTcSub + (q & 3) * 32) >> 4;
            tc_mma(ts, dq + off, dk + off, C::kIdescS, q > 0 ? 1u : 0u);
          }
          tc_commit(s_full + x);
          tc_commit(empty + s);
        }
        __syncwarp();
        return true;
      };
      auto pv = [&](int k) {
        const int i = 2 * (first + k * kStep) + 1, s = i % NB;
        if (!wait(full + s, i / NB)) return false;
        const uint64_t dv = tc_smem_desc_mn(base + C::kOffRing + s * C::kTile, kTcSub);
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // the first half of the keys under the second half's exponentials
          if (!wait(&p_full[x][h], k)) return false;
          tc_fence_after();
          const uint32_t acc = h > 0 || k > 0 ? 1u : 0u;
          if (elect_one()) {
#pragma unroll
            for (int q = 4 * h; q < 4 * h + 4; ++q)
              tc_mma_ta(to, tp + q * 8, dv + ((q * 2048) >> 4), C::kIdescO, q > 4 * h ? 1u : acc);
            if (h == 1) {
              tc_commit(pv_done + x);
              tc_commit(empty + s);
            }
          }
          __syncwarp();
        }
        return true;
      };
      bool ok = mine == 0 || wait(&qfull, 0);
      if (C::kAlias) {
        for (int k = 0; ok && k < mine; ++k) ok = qk(k) && pv(k);
      } else {  // the next S under this one's softmax
        if (ok && mine > 0) ok = qk(0);
        for (int k = 0; ok && k < mine; ++k) {
          if (k + 1 < mine) ok = qk(k + 1);
          ok = ok && pv(k);
        }
      }
      if (MT == 2)  // the other stream's tiles, which this one does not read
        for (int i = 2 * mine; ok && i < 2 * nt; ++i) {
          ok = wait(full + i % NB, i / NB);
          if (ok && lane == 0) mbar_arrive(empty + i % NB);
        }
      if (!ok) *abort = 1;
      // behind every MMA of the warp (a commit follows those of its own thread:
      // the elected lane is the same each time)
      int never = 0;
      if (elect_one()) tc_commit(drain + x);
      __syncwarp();
      mbar_wait(drain + x, 0u, kBudget, &never);
    }
    leave();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ---- softmax of stream x
    const int stid = int(threadIdx.x) - 128, x = stid >> 7;
    const int quarter = warp & 3, r = quarter * 32 + lane;
    {  // Q: a warp's rows, whole rows side by side in the lanes, all loads in flight at once
      constexpr int RW = 16 * MT, CH = HD / 8, RI = 32 / CH, N = RW / RI;  // rows a warp, chunks a row, rows a load
      const int row0 = (warp - 4) * RW, at = row0 + (lane & (RW - 1));
      unsigned long long off = ~0ull;  // of row `at` in q
      if (at < it.rows) {
        const int row = it.row0 + at, t = row / G;
        off = (it.lo + t - p.first) * p.q_ts + (kvh * G + row - t * G) * p.q_hs;
      }
      uint4 v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned long long o = __shfl_sync(0xffffffffu, off, i * RI + lane / CH);
        v[i] = o != ~0ull ? ld_vec(static_cast<const bf16*>(p.q) + o + (lane % CH) * 8) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = row0 + i * RI + lane / CH, c = lane % CH;
        *reinterpret_cast<uint4*>(smem + (row >> 7) * C::kTile + (c >> 3) * kTcSub + (row & 127) * 128 +
                                  (((c & 7) ^ (row & 7)) << 4)) = v[i];
      }
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&qfull);
    const uint32_t trow = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t ts = trow + x * C::kS, to = trow + C::kO + x * HD, tp = trow + C::kP + x * C::kPStep;
    const int row = MT == 2 ? x * 128 + r : r;
    const bool write = row < it.rows;
    const int lim = write ? seen(row) : keys;  // keys [0, lim) are seen
    const int low = seen(0);  // keys [0, low) are seen by all
    const int mine = tiles_of(x), others = tiles_of(1 - x);
    const float sl2 = p.scale * kLog2e;
    float m = -INFINITY, l = 0.f;  // reference max (scaled, base 2), sum
    bool ok = true;
    int k = 0;
    for (; k < mine; ++k) {
      const int t = MT == 2 ? k : 2 * k + x, j = t * kPaTcKeys;
      ok = mbar_wait_soon(s_full + x, uint32_t(k & 1), kBudget, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      float sc[kPaTcKeys];
#pragma unroll
      for (int c = 0; c < kPaTcKeys; c += 32) tc_ld32(ts + c, reinterpret_cast<uint32_t*>(sc + c));
      tc_wait_ld();
      if (!C::kAlias) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free + x);
      }
      const bool masked = __any_sync(0xffffffffu, j + kPaTcKeys > lim);
      if (masked) {
#pragma unroll
        for (int c = 0; c < kPaTcKeys; ++c) sc[c] = j + c < lim ? sc[c] : -INFINITY;
      }
      float mx[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
      for (int c = 4; c < kPaTcKeys - 4; c += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3_nan(mx[i], sc[c + i], sc[c + 4 + i]);
      mx[0] = max3_nan(mx[0], sc[124], sc[125]);
      mx[1] = max3_nan(mx[1], sc[126], sc[127]);
      const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * sl2;
      const bool grow = !(top <= m + 8.f);  // (NaN stays: exp2_cubic would lose it)
      if (!C::kAlias && k > 0) {  // the stream's previous P V has read P (aliased: it came before this S)
        ok = mbar_wait_soon(pv_done + x, uint32_t((k - 1) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, grow)) {
        const float a = grow ? exp2_approx(m - top) : 1.f;
        if (grow) m = top;
        l *= a;
        if (k > 0) {
#pragma unroll
          for (int c = 0; c < HD; c += 16) {
            uint32_t o[16];
            tc_ld16(to + c, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
            tc_st16(to + c, o);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.f : m;
      if (j + kPaTcKeys > low) {  // V rows behind the keys, or not seen by all (MT 2: both streams write the same zeros)
        const int i = 2 * t + 1, s = i % NB;
        ok = mbar_wait_soon(full + s, uint32_t((i / NB) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_clean_row<HD>(smem + C::kOffRing + s * C::kTile, r, j + r >= keys, j + r >= low, &odd_sh);
        fence_async_smem();
      }
      // the exponentials of the two warps of a scheduler take turns: one stream's
      // run under the other's MMAs, and not both at half pace
      if (x == 1 ? k < others : k > 0 && k - 1 < others) {
        ok = mbar_wait_soon(&turn[x][quarter], uint32_t(x == 1 ? k & 1 : (k - 1) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      // kCubic of 16 pairs on the fp32 pipe, which the special-function unit
      // (8 cycles a warp and value) leaves idle; masked tiles need exact zeros
      auto exps = [&](auto cubic) {
        constexpr int kCubic = decltype(cubic)::value;
#pragma unroll
        for (int c = 0; c < kPaTcKeys; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float2 e = fma2(make_float2(sc[c + i], sc[c + i + 1]), make_float2(sl2, sl2), make_float2(-ref, -ref));
            if ((i >> 1) * kCubic % 16 < kCubic) {
              e = exp2_cubic(e);
            } else {
              e.x = exp2_approx(e.x);
              e.y = exp2_approx(e.y);
            }
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
            pk[i / 2] = pack_bf16(e.x, e.y);
          }
          if (c == 64) {  // the first half of the keys: its stores have landed meanwhile
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[x][0]);
          }
          tc_st16(tp + c / 2, pk);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&turn[1 - x][quarter]);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x][1]);
      };
      if (masked)
        exps(std::integral_constant<int, 0>{});
      else
        exps(std::integral_constant<int, kPaCubic>{});
      sum[0] = add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
    }
    if (ok && k > 0) ok = mbar_wait_soon(pv_done + x, uint32_t((k - 1) & 1), kBudget, abort);
    if (!ok) *abort = 1;
    tc_fence_after();
    float wb = 0.f, wa = 1.f;
    if (MT == 1) {
      if (x == 1) ml_sh[r] = make_float2(k > 0 ? m : -INFINITY, l);
      tc_fence_before();
      named_sync(1, 256);
      tc_fence_after();
      const float2 b = ml_sh[r];
      // (a NaN max or sum of either stream makes both weights, or the sum, NaN)
      const float top = max3_nan(m, b.x, b.x), ref = top == -INFINITY ? 0.f : top;
      wa = exp2_approx(m - ref);
      wb = exp2_approx(b.x - ref);
      l = l * wa + b.y * wb;
    }
    if ((MT == 2 || x == 0) && __any_sync(0xffffffffu, write)) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const bool odd = *static_cast<volatile int*>(&odd_sh) != 0, two = MT == 1 && nt > 1;
      const int tok = it.lo + (it.row0 + row) / G, head = kvh * G + (it.row0 + row) % G;
      bf16* out = static_cast<bf16*>(p.out) + (size_t(tok - p.first) * p.hq + head) * HD;
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        uint32_t o0[16], o1[16];
        tc_ld16(to + c, o0);
        if (two) tc_ld16(to + HD + c, o1);
        tc_wait_ld();
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          f[e] = __uint_as_float(o0[e]) * wa;
          if (two) f[e] = fmaf(__uint_as_float(o1[e]), wb, f[e]);
        }
        if (write) {
          if (odd) {  // what was taken out of V
            const bf16* v = static_cast<const bf16*>(p.v) + kvh * p.v_hs + it.start * p.v_ts + c;
            for (int key = low; key < lim; ++key)
              for (int e = 0; e < 16; ++e) {
                const float y = to_f(v[key * p.v_ts + e]);
                if (!(fabsf(y) < INFINITY))
#pragma unroll
                  for (int u = 0; u < 16; ++u) f[u] = u == e ? f[u] + y : f[u];
              }
          }
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            *reinterpret_cast<uint4*>(out + c + e) =
                l == 0.f ? make_uint4(0, 0, 0, 0)
                         : make_uint4(pack_bf16(f[e] * inv, f[e + 1] * inv), pack_bf16(f[e + 2] * inv, f[e + 3] * inv),
                                      pack_bf16(f[e + 4] * inv, f[e + 5] * inv), pack_bf16(f[e + 6] * inv, f[e + 7] * inv));
        }
      }
    }
    leave();
  }
}

}  // namespace mtpb
