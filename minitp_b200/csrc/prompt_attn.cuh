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
// it, and what a token does not see does not reach it. (Of an infinity of V under
// a probability that is 0, or that fp32 or bf16 take for 0, the sum is NaN or that
// infinity.)
#pragma once

#include <type_traits>

#include "prompt_tiles.cuh"
#include "softmax.cuh"

namespace mtpb {

// Set when a bounded wait of a prompt attention ran out (its results are then void).
__device__ uint32_t g_pa_status;

// A share of the tokens of no prompt gets 0: one warp, when all tiles have been found.
template <typename T>
__device__ __forceinline__ void pa_zero(const PaParams& p, const PaTiles& t, int hd, int share, int shares) {
  constexpr int VE = VecTraits<T>::kElems;
  const int vecs = p.hq * hd / VE;  // of a token
  const int n0 = t.gap0 - p.first, n1 = p.first + p.n - t.gap1;
  for (int i = share; i < n0 + n1; i += shares) {
    const int at = i < n0 ? i : t.gap1 - p.first + (i - n0);
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (size_t)at * p.hq * hd);
    for (int e = threadIdx.x & 31; e < vecs; e += 32) o[e] = make_uint4(0, 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------
// Tiles on the CUDA cores: fp32, and bf16 with head dims 16 and 32 (the models
// served have 64 and 128; those are on the tensor cores). 256 threads as 16 x
// 16; RPT rows and 4 keys a thread of a tile of 16 RPT rows and 64 keys, in
// fp32; a row's 16 threads are half a warp, so its probabilities go through
// shared memory without a barrier of the CTA. The next tile's K and V are on
// their way into registers under the arithmetic of this one. Two products an
// instruction, over even and odd dims (fp32 us without / with, 64-row tiles: 4
// prompts of <= 2048 tokens, 7 heads of 128: 410 / 332; 5 of <= 701, 8 heads of 32:
// 45 / 43). Two CTAs an SM up to 64 dims, at 128 registers (one / two: 8 of <= 1024,
// 14 heads of 64: 182 / 156; one of 1000: 78 / 103). What binds these thread tiles
// is shared memory reads beside the fused multiply-adds (a float4 of K serves RPT
// rows, one of V as well): 31 to 37 TFLOP/s of 72. Tiles of 4 rows x 8 keys a thread,
// which would read less for a product, have not been tried.
// ---------------------------------------------------------------------------
constexpr int kPaKeys = 64;
constexpr int kPaThreads = 256;

template <int HD, int RPT>
constexpr size_t pa_simt_smem() {
  return sizeof(float) * (size_t(16 * RPT) * (HD + 4) + 2 * size_t(kPaKeys) * (HD + 4) + size_t(16 * RPT) * (kPaKeys + 4));
}

template <typename T, int HD, int RPT>
__global__ void __launch_bounds__(kPaThreads, HD <= 64 ? 2 : 1) pa_simt_kernel(const PaParams p) {
  constexpr int ROWS = 16 * RPT, LD = HD + 4, LP = kPaKeys + 4, VE = VecTraits<T>::kElems;
  constexpr int DP = HD / 16;  // dims a thread of the result, in runs of DV: tx * DV + 16 * DV * g ..
  constexpr int DV = DP < 4 ? DP : 4, DG = DP / DV;
  constexpr int NV = (kPaKeys * HD / VE + kPaThreads - 1) / kPaThreads;  // vectors of K (and of V) a thread loads
  extern __shared__ __align__(16) float pa_sm[];
  float* sq = pa_sm;
  float* sk = sq + ROWS * LD;
  float* sv = sk + kPaKeys * LD;
  float* sp = sv + kPaKeys * LD;
  __shared__ PaItem it_sh;
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  if (tid < 32) {
    PaTiles tiles;
    PaItem it = tiles.only(p, blockIdx.x / p.planes);
    it.plane = blockIdx.x % p.planes;
    if (tid == 0) it_sh = it;
    pa_zero<T>(p, tiles, HD, blockIdx.x, gridDim.x);
  }
  __syncthreads();
  const PaItem it = it_sh;
  if (it.ntok == 0) return;
  const int rows = it.ntok * p.gs, kvh = it.plane / p.subs, head0 = it.plane * p.gs;
  const T* q = static_cast<const T*>(p.q);
  const T* k = static_cast<const T*>(p.k) + kvh * p.k_hs + it.start * p.k_ts;
  const T* v = static_cast<const T*>(p.v) + kvh * p.v_hs + it.start * p.v_ts;
  auto token = [&](int r) { return it.tok0 + pa_div_gs(p, r); };
  const int keys = it.tok0 + it.ntok - it.start, low = it.tok0 + 1 - it.start;
  uint4 hk[NV], hv[NV];  // the next tile
  auto fetch = [&](int j) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = tid + n * kPaThreads, r = i / (HD / VE), c = (i - r * (HD / VE)) * VE;
      hk[n] = hv[n] = make_uint4(0, 0, 0, 0);
      if (r < kPaKeys && j + r < keys) {
        hk[n] = ld_vec(k + (long long)(j + r) * p.k_ts + c);
        hv[n] = ld_vec(v + (long long)(j + r) * p.v_ts + c);
      }
    }
  };
  fetch(0);
  for (int i = tid; i < ROWS * (HD / VE); i += kPaThreads) {
    const int r = i / (HD / VE), c = (i - r * (HD / VE)) * VE;
    float f[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = 0.f;
    if (r < rows) unpack(ld_vec(q + (token(r) - p.first) * p.q_ts + (head0 + r - pa_div_gs(p, r) * p.gs) * p.q_hs + c), f);
#pragma unroll
    for (int e = 0; e < VE; ++e) sq[r * LD + c + e] = f[e];
  }
  int lim[RPT];  // keys [0, lim) of the prompt are seen
#pragma unroll
  for (int a = 0; a < RPT; ++a) lim[a] = token(min(ty * RPT + a, rows - 1)) + 1 - it.start;
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
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = tid + n * kPaThreads, r = i / (HD / VE), c = (i - r * (HD / VE)) * VE;
      if (r < kPaKeys) {
        float f[VE];
        unpack(hk[n], f);
#pragma unroll
        for (int e = 0; e < VE; e += 4) *reinterpret_cast<float4*>(sk + r * LD + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
        unpack(hv[n], f);
#pragma unroll
        for (int e = 0; e < VE; e += 4) *reinterpret_cast<float4*>(sv + r * LD + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      }
    }
    __syncthreads();
    if (j + kPaKeys < keys) fetch(j + kPaKeys);
    float2 s2[RPT][4];  // sums over even and odd dims: two products an instruction
#pragma unroll
    for (int a = 0; a < RPT; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) s2[a][b] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      float4 kk[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) kk[b] = *reinterpret_cast<const float4*>(sk + (tx + 16 * b) * LD + d);
#pragma unroll
      for (int a = 0; a < RPT; ++a) {
        const float4 qq = *reinterpret_cast<const float4*>(sq + (ty * RPT + a) * LD + d);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          s2[a][b] = fma2(make_float2(qq.x, qq.y), make_float2(kk[b].x, kk[b].y), s2[a][b]);
          s2[a][b] = fma2(make_float2(qq.z, qq.w), make_float2(kk[b].z, kk[b].w), s2[a][b]);
        }
      }
    }
    float s[RPT][4];
#pragma unroll
    for (int a = 0; a < RPT; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) s[a][b] = s2[a][b].x + s2[a][b].y;
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
      const float ref = top == -INFINITY ? 0.f : top, w = exp2_approx(m[a] - ref);
      m[a] = top;
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float e = exp2_approx(s[a][b] - ref);
        sum += e;
        sp[(ty * RPT + a) * LP + tx + 16 * b] = e;
      }
      l[a] = fmaf(l[a], w, sum);  // (of this thread's keys)
#pragma unroll
      for (int d = 0; d < DP; ++d) o[a][d] *= w;
    }
    __syncwarp();
    const int nk = min(kPaKeys, keys - j);
    auto v_at = [&](int key, float (&x)[DP]) {
#pragma unroll
      for (int g = 0; g < DG; ++g) {
        const float* at = sv + key * LD + tx * DV + g * 16 * DV;
        if constexpr (DV == 4) {
          const float4 y = *reinterpret_cast<const float4*>(at);
          x[4 * g] = y.x, x[4 * g + 1] = y.y, x[4 * g + 2] = y.z, x[4 * g + 3] = y.w;
        } else if constexpr (DV == 2) {
          const float2 y = *reinterpret_cast<const float2*>(at);
          x[2 * g] = y.x, x[2 * g + 1] = y.y;
        } else {
          x[g] = *at;
        }
      }
    };
    if (!masked) {
#pragma unroll 2
      for (int key = 0; key < kPaKeys; key += 4) {
        float4 pp[RPT];
#pragma unroll
        for (int a = 0; a < RPT; ++a) pp[a] = *reinterpret_cast<const float4*>(sp + (ty * RPT + a) * LP + key);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[DP];
          v_at(key + i, x);
#pragma unroll
          for (int a = 0; a < RPT; ++a) {
            const float pr = i == 0 ? pp[a].x : i == 1 ? pp[a].y : i == 2 ? pp[a].z : pp[a].w;
            if constexpr (DP == 1) {
              o[a][0] = fmaf(pr, x[0], o[a][0]);
            } else {
#pragma unroll
              for (int d = 0; d < DP; d += 2) {
                const float2 y = fma2(make_float2(pr, pr), make_float2(x[d], x[d + 1]), make_float2(o[a][d], o[a][d + 1]));
                o[a][d] = y.x;
                o[a][d + 1] = y.y;
              }
            }
          }
        }
      }
    } else {  // a key that a row does not see adds nothing to it, whatever its V
#pragma unroll 2
      for (int key = 0; key < nk; ++key) {
        float x[DP];
        v_at(key, x);
#pragma unroll
        for (int a = 0; a < RPT; ++a)
          if (j + key < lim[a]) {
            const float pr = sp[(ty * RPT + a) * LP + key];
#pragma unroll
            for (int d = 0; d < DP; ++d) o[a][d] = fmaf(pr, x[d], o[a][d]);
          }
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int a = 0; a < RPT; ++a) {
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) l[a] += __shfl_xor_sync(0xffffffffu, l[a], x);
    const int r = ty * RPT + a;
    if (r < rows) {
      T* out = static_cast<T*>(p.out) + (size_t(token(r) - p.first) * p.hq + head0 + r - pa_div_gs(p, r) * p.gs) * HD;
#pragma unroll
      for (int d = 0; d < DP; ++d)
        out[tx * DV + (d / DV) * 16 * DV + d % DV] = from_f<T>(l[a] == 0.f ? 0.f : o[a][d] / l[a]);
    }
  }
}

// ---------------------------------------------------------------------------
// Tiles on the tensor cores (bf16, head dim 64 or 128), key tiles of 128. Two
// streams share the ring of K and V tiles, each with an MMA warp, a softmax
// warpgroup (a row a thread) and its own tensor memory:
//   MT 2: stream x has rows 128 x .. of the item's 256 and their keys, so a
//         K/V byte brought in from L2 serves 256 rows;
//   MT 1: both have the item's 128 rows, stream x the key tiles t = x mod 2,
//         and the streams are joined at the end.
// One stream's softmax runs under the other's and under the MMAs:
//   warp 0 loads (TMA, 128-byte swizzle: boxes of 128 keys x 64 dims, and of a
//   tile's tokens x heads x 64 dims), warps 1 and 2 issue S = Q K^T and O += P V
//   of their stream, warps 4-7 and 8-11 turn S into P, with the registers that
//   warps 0-3 hand over.
// A CTA an SM takes items in turn, which warp 3 finds two ahead: the next
// item's Q, K and V are loaded, and its first S made, under the end of the last.
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
//
// Bound by the softmax: a key tile of both streams costs 3500 to 3900 cycles
// (head dim 128), of which the products take 2048 of the tensor cores, the 7/8
// of the exponentials that the special-function unit makes 1800 of that unit,
// and the softmax warps alone, with no products to wait for, 2700. Measured, GPU time of
// single calls (1965 MHz) and of a second of calls (1580 to 1800 MHz, under the power
// cap): one prompt of 32768 tokens, 28 heads of 128: 6.3 to 6.9 / 7.1 ms, 1.08 PFLOP/s of
// the latter; 12 of <= 4096, 28 heads of 128: 480 / 564 us, 0.88; of short prompts the turn from item to item (3000 to
// 4000 cycles: the last P V, the output) weighs as much as their one or two key
// tiles. Four softmax warpgroups (half a row a thread), S in two halves of 64
// keys, and rolled loops that read S twice were 10 to 40 % slower.
// ---------------------------------------------------------------------------
constexpr int kPaTcKeys = 128;
constexpr int kPaTcThreads = 384;
template <int HD>
constexpr int kPaCubic = HD == 128 ? 2 : 4;  // of 16 pairs of exponentials, on the fp32 pipe (1, 3, 6, 8: 15 to 25 % slower)

template <int HD, int MT>
struct PaTcCfg {
  static constexpr int kRows = 128 * MT;
  static constexpr int kSubs = HD / 64;
  static constexpr uint32_t kTile = kSubs * kTcSub;  // a K or V tile
  static constexpr uint32_t kQSub = kRows * 128;     // 64 dims of the Q rows
  // ring of K and V tiles: what 224 KB leave beside Q
  static constexpr int kRing = HD == 128 ? 5 : 12;
  static constexpr uint32_t kOffRing = kSubs * kQSub;
  static constexpr size_t kSmem = size_t(kOffRing) + kRing * kTile + 1024;
  // registers a thread of warps 0-3 and of the softmax (168 at launch): 128 x a + 256 x b = 384 x 168
  static constexpr int kRegs = HD == 128 ? 72 : 56, kRegsSoftmax = HD == 128 ? 216 : 224;
  static_assert(128 * kRegs + 256 * kRegsSoftmax <= 384 * 168, "registers handed over");
  static constexpr bool kAlias = HD == 128;  // P in the place of S
  static constexpr uint32_t kS = 128;        // columns from stream to stream of S; of O: HD
  static constexpr uint32_t kO = 256, kP = kAlias ? 0 : 384, kPStep = kAlias ? 128 : 64;
  static constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);
  // B of P V: N (dims) contiguous
  static constexpr uint32_t kIdescO =
      (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(HD >> 3) << 17) | (uint32_t(128 >> 4) << 24);
};

// A place in a ring of N barriers and its phase.
template <int N>
struct PaSlot {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1u;
    }
  }
};

__device__ __forceinline__ void st_v8(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <int HD, int MT>
__global__ void __launch_bounds__(kPaTcThreads, 1)
    pa_tc_kernel(const PaParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v) {
  using C = PaTcCfg<HD, MT>;
  constexpr int NB = C::kRing;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[NB], empty[NB], raw[NB], q_full, q_empty, item_full[2], item_empty[2];
  __shared__ uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2], o_free[2], drain[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_sh;
  __shared__ int odd_sh[2];  // by the item's parity: its number + 1 when values of V were zeroed
  __shared__ float2 ml_sh[MT == 1 ? 2 : 1][2][MT == 1 ? 128 : 1];  // MT 1: by the item's parity and stream, statistics
  __shared__ PaItem items[2];
  volatile int* abort = &abort_sh;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  pdl_launch();
  pdl_wait();
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (threadIdx.x == 0) {
    for (int s = 0; s < NB; ++s) {
      mbar_init(full + s, 1);
      mbar_init(raw + s, 1);
      mbar_init(empty + s, MT);  // each stream that reads the tile
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 2);
    for (int x = 0; x < 2; ++x) {
      mbar_init(item_full + x, 1);
      mbar_init(item_empty + x, 11);  // warps 0 to 2 and the softmax's
      mbar_init(s_full + x, 1);
      mbar_init(s_free + x, 4);
      for (int h = 0; h < 2; ++h) mbar_init(&p_full[x][h], 4);
      mbar_init(pv_done + x, 1);
      mbar_init(o_free + x, MT == 1 ? 8 : 4);
      mbar_init(drain + x, 1);
      odd_sh[x] = 0;
    }
    *abort = 0;
    mbar_init_fence();
  } else if (warp >= 4) {  // rows that no copy of Q writes (those behind tt * gs) stay zeros
    const int used = p.tt * p.gs, left = (C::kRows - used) * 8;
    for (int i = threadIdx.x - 128; i < left * C::kSubs; i += kPaTcThreads - 128)
      *reinterpret_cast<uint4*>(smem + (i / left) * C::kQSub + used * 128 + (i % left) * 16) = make_uint4(0, 0, 0, 0);
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_lean(bar, parity & 1u, abort); };
  // keys that the item's tile sees; key tiles of stream x (all of them in turn, or MT 1: every second)
  auto keys_of = [&](const PaItem& it) { return it.tok0 + it.ntok - it.start; };
  auto tiles_of = [&](const PaItem& it, int x) {
    const int nt = (keys_of(it) + kPaTcKeys - 1) / kPaTcKeys;
    if (MT == 1) return (nt - x + 1) / 2;
    if (x == 1) return it.ntok * p.gs > 128 ? nt : 0;
    const int last = min(it.ntok * p.gs, 128) - 1;  // of the stream's rows
    return (it.tok0 + pa_div_gs(p, last) + 1 - it.start + kPaTcKeys - 1) / kPaTcKeys;
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

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegs));
    if (warp == 3) {
      // ---- items: tiles blockIdx, and then every gridDim-th, the direction
      // reversed each time (the numbers go by falling cost). And the V tiles at
      // an item's end: rows behind its keys become zeros, and of those that not
      // every row of the item sees the NaN and infinities.
      PaTiles tiles;
      tiles.open(p);
      PaSlot<NB> at;  // of the item's first K tile
      uint32_t raws = 0;  // phases of `raw`, a bit each
      bool ok = true;
      PaItem it{0, 0, 0, 0};
#pragma unroll 1
      for (int n = -1; ok && (n < 0 || it.ntok > 0); ++n) {
        const long long i = (long long)(n + 1) * gridDim.x + (n & 1 ? blockIdx.x : gridDim.x - 1 - blockIdx.x);
        PaItem next = tiles.find(p, int(min(i / p.planes, 0x7FFFFFFFll)));
        next.plane = int(i % p.planes);
        const int keys = keys_of(it), low = it.tok0 + 1 - it.start, nt = n < 0 ? 0 : (keys + kPaTcKeys - 1) / kPaTcKeys;
#pragma unroll 1
        for (int t = 0; ok && t < nt; ++t) {
          at.next();
          if ((t + 1) * kPaTcKeys > low) {
            ok = __all_sync(0xffffffffu, wait(raw + at.i, raws >> at.i));
            raws ^= 1u << at.i;
#pragma unroll 1
            for (int r = max(low - t * kPaTcKeys, 0) + lane; ok && r < kPaTcKeys; r += 32)
              tc_clean_row<HD>(smem + C::kOffRing + at.i * C::kTile, r, t * kPaTcKeys + r >= keys, true, odd_sh + (n & 1), n + 1);
            fence_async_smem();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(full + at.i);
          }
          at.next();
        }
        if (n >= 1 && ok) ok = __all_sync(0xffffffffu, wait(item_empty + (~n & 1), ((n + 1) >> 1) - 1));
        if (ok && lane == 0) {
          items[~n & 1] = next;
          mbar_arrive(item_full + (~n & 1));
        }
        __syncwarp();
        it = next;
      }
      if (!ok) *abort = 1;
      pa_zero<bf16>(p, tiles, HD, blockIdx.x, gridDim.x);
    } else if (elect_one()) {
      // The item of number n, or none: one thread's.
      auto item = [&](int n, PaItem* it) {
        if (!wait(item_full + (n & 1), n >> 1)) {
          *abort = 1;
          return false;
        }
        *it = items[n & 1];
        mbar_arrive(item_empty + (n & 1));
        return it->ntok > 0;
      };
      PaItem it;
      bool ok = true;
      if (warp == 0) {
        PaSlot<NB> at;
        int issued = 0, queries = 0;
        uint32_t raws = 0, phases = 0;  // slots whose last copy completes on `raw`; the phases of those, a bit each
        for (int n = 0; ok && item(n, &it); ++n) {
          const int nt = (keys_of(it) + kPaTcKeys - 1) / kPaTcKeys, kvh = it.plane / p.subs;
          for (int i = 0; ok && i < 2 * nt; ++i) {  // K and V of each tile in turn
            ok = issued < NB || wait(empty + at.i, at.phase ^ 1u);
            if (!ok) break;
            // V tiles that not every row sees whole go by way of warp 3
            const bool unseen = (i & 1) && ((i >> 1) + 1) * kPaTcKeys > it.tok0 + 1 - it.start;
            uint64_t* bar = unseen ? raw + at.i : full + at.i;
            raws = unseen ? raws | (1u << at.i) : raws & ~(1u << at.i);
            if (unseen) phases ^= 1u << at.i;
            mbar_arrive_expect_tx(bar, C::kTile);
#pragma unroll
            for (int b = 0; b < C::kSubs; ++b)
              tma_load_3d(base + C::kOffRing + at.i * C::kTile + b * kTcSub, i & 1 ? &map_v : &map_k, b * 64,
                          it.start + (i >> 1) * kPaTcKeys, kvh, bar);
            at.next();
            if (issued < NB) ++issued;
            if (i == 0) {  // Q: when the item before has made its last S
              ok = n == 0 || wait(&q_empty, n - 1);
              if (!ok) break;
              ++queries;
              mbar_arrive_expect_tx(&q_full, uint32_t(p.tt * p.gs) * 128 * C::kSubs);
#pragma unroll
              for (int b = 0; b < C::kSubs; ++b)
                tma_load_3d(base + b * C::kQSub, &map_q, b * 64, it.plane * p.gs, it.tok0 - p.first, &q_full);
            }
          }
          if (!ok) *abort = 1;
        }
        // copies in flight land before the memory goes away: those of the last round of the ring, and Q
        int never = 0;
        if (issued < NB)
          at = PaSlot<NB>();
        else
          at.phase ^= 1u;
        for (int i = 0; i < issued; ++i) {
          if (raws >> at.i & 1u)
            mbar_wait_lean(raw + at.i, (phases >> at.i & 1u) ^ 1u, &never);
          else
            mbar_wait_lean(full + at.i, at.phase, &never);
          at.next();
        }
        if (queries > 0) mbar_wait_lean(&q_full, uint32_t(queries - 1) & 1u, &never);
      } else {
        // ---- MMA issue of stream x, by one thread
        const int x = warp - 1;
        const uint64_t dq = tc_smem_desc(base + (MT == 2 ? x : 0) * 128 * 128);
        const uint32_t ts = tmem + x * C::kS, to = tmem + C::kO + x * HD, tp = tmem + C::kP + x * C::kPStep;
        PaSlot<NB> ks, vs;  // of the next K and V tile of the item's
        vs.next();
        auto skip = [&](PaSlot<NB>& sl, int entries) {
          for (int e = 0; e < entries; ++e) sl.next();
        };
        auto landed = [&](const PaSlot<NB>& sl) { return wait(full + sl.i, sl.phase); };
        uint32_t kk = 0;  // tiles so far
        auto qk = [&]() {
          const uint64_t dk = tc_smem_desc(base + C::kOffRing + ks.i * C::kTile);
          tc_fence_after();
#pragma unroll
          for (int q = 0; q < HD / 16; ++q)
            tc_mma(ts, dq + (((q >> 2) * C::kQSub + (q & 3) * 32) >> 4), dk + (((q >> 2) * kTcSub + (q & 3) * 32) >> 4),
                   C::kIdescS, q > 0 ? 1u : 0u);
          tc_commit(s_full + x);
          tc_commit(empty + ks.i);
        };
        auto pv = [&](bool first, int h) {  // the first half of the keys under the second half's exponentials
          const uint64_t dv = tc_smem_desc_mn(base + C::kOffRing + vs.i * C::kTile, kTcSub);
          tc_fence_after();
#pragma unroll
          for (int q = 4 * h; q < 4 * h + 4; ++q)
            tc_mma_ta(to, tp + q * 8, dv + ((q * 2048) >> 4), C::kIdescO, q > 0 || !first ? 1u : 0u);
          if (h == 1) {
            tc_commit(pv_done + x);
            tc_commit(empty + vs.i);
          }
        };
        // entries of the ring from one tile of the stream to its next
        constexpr int kStep = MT == 2 ? 2 : 4;
        for (int n = 0; ok && item(n, &it); ++n) {
          const int nt = (keys_of(it) + kPaTcKeys - 1) / kPaTcKeys, mine = tiles_of(it, x);
          int left = 2 * nt;  // entries of the item that ks has not passed
          auto pass = [&](int entries) {
            skip(ks, entries);
            skip(vs, entries);
            left -= entries;
          };
          if (MT == 1 && x == 1) pass(2);
          ok = wait(&q_full, n);
          if (ok && mine == 0) mbar_arrive(&q_empty);
#pragma unroll 1
          for (int k = 0; ok && k <= mine; ++k) {  // S of tile k, P V of tile k - 1
            // S of tile k is free: read by the softmax, or (aliased) in the place of the P that the MMAs before
            // it read: one thread's MMAs run in order
            auto ready = [&]() {
              if (k > 0 && k < mine) skip(ks, kStep);
              return k == mine || (landed(ks) && (C::kAlias || kk == 0 || wait(s_free + x, kk - 1)));
            };
            auto scores = [&]() {
              if (!ok || k == mine) return;
              qk();
              if (k + 1 == mine) tc_commit(&q_empty);
            };
            if (!C::kAlias) {  // under the softmax of the tile before
              ok = ready();
              scores();
            }
            if (k > 0) {
              ok = ok && landed(vs) && (k > 1 || n == 0 || wait(o_free + x, n - 1)) && wait(&p_full[x][0], kk - 1);
              if (ok) pv(k == 1, 0);
            }
            if (C::kAlias) ok = ok && ready();
            if (k > 0) {
              ok = ok && wait(&p_full[x][1], kk - 1);
              if (ok) pv(k == 1, 1);
              if (k < mine) skip(vs, kStep);
            }
            if (C::kAlias) scores();
            if (k < mine) ++kk;
          }
          // on to the next item's entries, past those that this stream does not read
          if (mine > 0) left -= (mine - 1) * kStep;
          if (MT == 2) {
            if (mine > 0) {
              skip(ks, 2);
              skip(vs, 2);
              left -= 2;
            }
            for (; ok && left > 0; left -= 2) {  // the other stream's tiles
              ok = landed(ks) && landed(vs);
              if (ok) {
                mbar_arrive(empty + ks.i);
                mbar_arrive(empty + vs.i);
              }
              skip(ks, 2);
              skip(vs, 2);
            }
          } else {
            skip(ks, left);
            skip(vs, left);
          }
        }
        if (!ok) *abort = 1;
        int never = 0;
        tc_commit(drain + x);  // behind every MMA of the thread
        mbar_wait_lean(drain + x, 0u, &never);
      }
    }
    leave();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
    // ---- softmax of stream x
    const int x = (int(threadIdx.x) - 128) >> 7;
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t trow = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t ts = trow + x * C::kS, to = trow + C::kO + x * HD, tp = trow + C::kP + x * C::kPStep;
    const int row = MT == 2 ? x * 128 + r : r;
    const float sl2 = p.scale * kLog2e;
    uint32_t kk = 0;  // tiles so far
    bool ok = true;
    for (int n = 0;; ++n) {
      ok = ok && wait(item_full + (n & 1), n >> 1);
      if (!__all_sync(0xffffffffu, ok)) ok = false;
      if (!ok || items[n & 1].ntok == 0) {
        if (!ok) *abort = 1;
        // (MT 1: a warp whose wait ran out and one at the end, or with the item, meet at one barrier)
        if (MT == 1) named_sync_and(1, 256, false);
        break;
      }
      int lim, mine;  // keys [0, lim) are seen
      {
        const PaItem it = items[n & 1];
        mine = tiles_of(it, x);
        lim = it.tok0 + min(pa_div_gs(p, row), it.ntok - 1) + 1 - it.start;
      }
      const int wlo = __reduce_min_sync(0xffffffffu, lim), whi = __reduce_max_sync(0xffffffffu, lim);
      float m = -INFINITY, l = 0.f;  // reference max (scaled, base 2), sum
      for (int k = 0; k < mine; ++k, ++kk) {
        const int t = MT == 2 ? k : 2 * k + x, j = t * kPaTcKeys;
        ok = wait(s_full + x, kk);
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
        const bool masked = j + kPaTcKeys > wlo;
        if (masked) {
#pragma unroll
          for (int c = 0; c < kPaTcKeys; c += 32)
            if (j + c + 32 > wlo) {
#pragma unroll
              for (int i = 0; i < 32; ++i) sc[c + i] = c + i < lim - j ? sc[c + i] : -INFINITY;
            }
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
          ok = wait(pv_done + x, kk - 1);
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
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // kCubic of 16 pairs on the fp32 pipe, which the special-function unit
        // (8 cycles a warp and value) leaves idle; masked tiles need exact zeros,
        // and of 32 keys that no row of the warp sees none at all
        auto exps = [&](auto mask) {
          constexpr bool kMask = decltype(mask)::value;
          constexpr int kCubic = kMask ? 0 : kPaCubic<HD>;
#pragma unroll
          for (int c = 0; c < kPaTcKeys; c += 32) {
            uint32_t pk[16];
            const bool none = kMask && j + c >= whi;
            if (none) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = 0u;
            }
            if (!none) {
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
            }
            if (c == 64) {  // the first half of the keys: its stores have landed meanwhile
              tc_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[x][0]);
            }
            tc_st16(tp + c / 2, pk);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x][1]);
        };
        if (masked)
          exps(std::true_type{});
        else
          exps(std::false_type{});
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      if (ok && mine > 0) ok = wait(pv_done + x, kk - 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        *abort = 1;
      }
      tc_fence_after();
      // no score above -inf: the sum is what the cubic, which ends at 2^-125, made of those (the growth from -inf
      // to a first score takes it out, and so does MT 1's weight of a stream). A NaN sum stays: behind a NaN score
      // a tile that the row does not see sets m to -inf.
      if (m == -INFINITY && l == l) l = 0.f;
      float w0 = 1.f, w1 = 0.f;  // weights of this stream's O and the other's
      if (MT == 1) {
        ml_sh[n & 1][x][r] = make_float2(m, l);
        tc_fence_before();
        ok = named_sync_and(1, 256, ok);
        tc_fence_after();
        const float2 b = ml_sh[n & 1][1 - x][r];
        // (a NaN sum of either stream makes the whole sum NaN)
        const float top = fmaxf(m, b.x), ref = top == -INFINITY ? 0.f : top;
        w0 = exp2_approx(m - ref);
        w1 = exp2_approx(b.x - ref);
        l = l * w0 + b.y * w1;
      }
      if (!ok) break;
      {
        const PaItem it = items[n & 1];
        const bool write = row < it.ntok * p.gs, two = MT == 1 && keys_of(it) > kPaTcKeys;
        const int of = pa_div_gs(p, row), tok = it.tok0 + of;
        const bool odd = *static_cast<volatile int*>(odd_sh + (n & 1)) == n + 1;
        const bool none = __any_sync(0xffffffffu, l == 0.f);
        const float inv = 1.f / l;
        // MT 1: of the sum of both streams' each warpgroup writes half the dims
        constexpr int kCols = MT == 1 ? HD / 2 : HD;
        const int c0 = MT == 1 ? x * kCols : 0;
        const uint32_t oo = trow + C::kO + (1 - x) * HD + c0;
        bf16* out = static_cast<bf16*>(p.out) + (size_t(tok - p.first) * p.hq + it.plane * p.gs + row - of * p.gs) * HD + c0;
        // (MT 1, one key tile: stream 1 has no O)
        const bool own = MT == 2 || two || x == 0;
#pragma unroll 1
        for (int c = 0; c < kCols; c += 32) {
          float f[32];
          if (MT == 2 ? mine > 0 : true) {
            tc_ld32((own ? to + c0 : oo) + c, reinterpret_cast<uint32_t*>(f));
            tc_wait_ld();
            const float wi = (own ? w0 : w1) * inv;
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] *= wi;
            if (two) {
              uint32_t o1[32];
              tc_ld32(oo + c, o1);
              tc_wait_ld();
              const float wj = w1 * inv;
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = fmaf(__uint_as_float(o1[e]), wj, f[e]);
            }
          }
          if (c == kCols - 32) {  // O may be written again
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(o_free + x);
              if (MT == 1) mbar_arrive(o_free + 1 - x);
            }
          }
          if (write) {
            if (odd) {  // what was taken out of V
              const bf16* v = static_cast<const bf16*>(p.v) + (it.plane / p.subs) * p.v_hs + it.start * p.v_ts + c0 + c;
#pragma unroll 1
              for (int i = (it.tok0 + 1 - it.start) * 32; i < lim * 32; ++i) {  // (earlier keys are seen by all)
                const float y = to_f(v[(i >> 5) * p.v_ts + (i & 31)]);
                if (!(fabsf(y) < INFINITY))
#pragma unroll
                  for (int e = 0; e < 32; ++e) f[e] = e == (i & 31) ? f[e] + y : f[e];
              }
            }
            if (none) {
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = l == 0.f ? 0.f : f[e];
            }
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack_bf16(f[h + 2 * e], f[h + 2 * e + 1]);
              st_v8(out + c + h, w);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty + (n & 1));
    }
    leave();
  }
}

}  // namespace mtpb
