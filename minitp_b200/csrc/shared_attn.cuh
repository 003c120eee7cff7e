// Attention of rows that share a prefix. Rows come in groups of W; group g has
// one prefix cache and every row its own. Token t (of T) of row n = g * W + w
// attends to positions [0, prefix_lens[g]) of the prefix and to positions
// [0, cache_lens[n] - (T - 1 - t)) of its own cache:
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = q . k_j / sqrt(hd)
// over both. A token that sees no position gives 0.
//
// The work is cut into items of one key range: prefix items hold the (token,
// head) rows of the whole group that share a KV head, so a prefix position is
// read once per row tile and not once per row; own items hold those of one
// row. Every item writes its rows' unnormalised sums with their max and
// denominator (a slot per key range), and a second kernel joins the slots.
//
// NaN and infinities go where the formula takes them and nowhere else: a score
// that is NaN or +inf makes its row NaN (a sum that is NaN is handed on with a
// NaN max, which no join passes over), and a NaN among V makes its dim NaN,
// whatever the weight (but for a key range whose scores are all -inf, which
// counts as not seen); positions that a token does not see reach it neither
// through K (its scores are selected away) nor through V (0 times NaN would be
// NaN: such terms are left out or zeroed).
#pragma once

#include <type_traits>

#include "softmax.cuh"

namespace mtpb {

struct SaParams {
  const void* q;
  const void *kp, *vp;
  const int* plen;
  int plen_all;
  const void *kc, *vc;
  const int* clen;
  int clen_stride, clen_add;
  void* out;
  int G, W, T, hq, hkv, cap_p, cap;
  float scale;
  int sp, so;        // key ranges of the prefix and of an own cache
  int ptiles, otiles;  // row tiles of a (group, KV head) and of a (row, KV head)
  int pitems, items;   // prefix items, all items
  int item0;           // CUDA-core items: first of this launch
  // partial sums, in blocks of 32 rows (SaPart)
  int pblocks, oblocks;  // blocks of a prefix plane, of an own plane
  float* part_o;         // [block][hd / 4][32 rows][4]
  float2* part_ml;       // [block][32 rows]: max (base e, scaled), sum
  uint32_t* status;  // of a communicator, or NULL: g_sa_status
};

// Error bits of calls without a communicator's status word.
__device__ uint32_t g_sa_status;


__device__ __forceinline__ int sa_prefix_len(const SaParams& p, int g) {
  const int n = p.plen ? p.plen[g] : p.plen_all;
  return max(0, min(n, p.cap_p));
}
__device__ __forceinline__ int sa_cache_len(const SaParams& p, int n) {
  // 64 bits: the sum of a length from the device and the host's offset
  const long long c = (p.clen ? (long long)p.clen[size_t(n) * p.clen_stride] : 0) + p.clen_add;
  return int(c < 0 ? 0 : c > p.cap ? p.cap : c);
}

// What an item covers.
struct SaItem {
  const void *k, *v;  // first position of this KV head
  int row0, rows;     // (token, head) rows of the tile: first, count (of the item's own numbering)
  int j0, j1;         // keys [j0, j1)
  int n0, kvh, split;  // first batch row
  int plane;          // (group or row) x KV head: which [cap][hd] block of the cache
  bool own;
};

// Where a row's partial sums lie. A plane is a (group, KV head) or (row, KV
// head); its rows (token, head) are cut into blocks of 32 that lie dims-major,
// so that the 32 lanes of a warp, each with a row, move 512 bytes at once.
struct SaPart {
  size_t ml, o;  // elements of part_ml, part_o (dims 0..3; + 128 every 4 dims)
};
template <int HD>
__device__ __forceinline__ SaPart sa_part(const SaParams& p, bool own, int split, int plane, int r) {
  const size_t pp = size_t(p.G) * p.hkv, op = pp * p.W;
  const size_t b = (own ? p.sp * pp * p.pblocks + (split * op + plane) * p.oblocks
                        : (split * pp + plane) * p.pblocks) + (r >> 5);
  return SaPart{b * 32 + (r & 31), b * 32 * HD + (r & 31) * 4};
}

// Row r of an item: token r / per of the item's rows, query head r % per of its KV head.
struct SaRow {
  int n, t, head;
};

template <int HD, int ES>
__device__ __forceinline__ SaItem sa_item(const SaParams& p, int it, int tile, int align) {
  SaItem s;
  const int per = p.hq / p.hkv;
  s.own = it >= p.pitems;
  int split, len, total, splits;
  if (!s.own) {
    splits = p.sp;
    split = it % p.sp;
    int r = it / p.sp;
    const int t = r % p.ptiles;
    r /= p.ptiles;
    s.kvh = r % p.hkv;
    const int g = r / p.hkv;
    len = sa_prefix_len(p, g);
    s.n0 = g * p.W;
    total = p.W * p.T * per;
    s.row0 = t * tile;
    s.plane = g * p.hkv + s.kvh;
    const size_t off = size_t(s.plane) * p.cap_p * HD * ES;
    s.k = static_cast<const char*>(p.kp) + off;
    s.v = static_cast<const char*>(p.vp) + off;
    s.split = split;
  } else {
    splits = p.so;
    it -= p.pitems;
    split = it % p.so;
    int r = it / p.so;
    const int t = r % p.otiles;
    r /= p.otiles;
    s.kvh = r % p.hkv;
    s.n0 = r / p.hkv;
    len = sa_cache_len(p, s.n0);
    total = p.T * per;
    s.row0 = t * tile;
    s.plane = s.n0 * p.hkv + s.kvh;
    const size_t off = size_t(s.plane) * p.cap * HD * ES;
    s.k = static_cast<const char*>(p.kc) + off;
    s.v = static_cast<const char*>(p.vc) + off;
    s.split = split;
  }
  s.rows = min(tile, total - s.row0);
  if (s.own) {  // no key past the last token of the tile
    const int t_last = (s.row0 + s.rows - 1) / per;
    len = max(0, len - (p.T - 1 - t_last));
  }
  // ranges of whole key tiles
  int chunk = (len + splits - 1) / splits;
  chunk = (chunk + align - 1) / align * align;
  s.j0 = min(len, split * chunk);
  s.j1 = min(len, s.j0 + chunk);
  return s;
}

__device__ __forceinline__ SaRow sa_row(const SaParams& p, const SaItem& s, int r) {
  const int per = p.hq / p.hkv;
  const int tok = (s.row0 + r) / per;
  SaRow x;
  x.head = s.kvh * per + (s.row0 + r) - tok * per;
  x.n = s.n0 + tok / p.T;
  x.t = tok % p.T;
  return x;
}
// Keys that row x of an item sees: [0, limit).
__device__ __forceinline__ int sa_limit(const SaParams& p, const SaItem& s, const SaRow& x) {
  return s.own ? sa_cache_len(p, x.n) - (p.T - 1 - x.t) : s.j1;
}
// The max handed on with sum l.
__device__ __forceinline__ float sa_max_of(float m, float l) { return l == l ? m : l; }

// ---------------------------------------------------------------------------
// Items on the CUDA cores (fp32, and bf16 head dims below 64): tiles of
// 16 * RPT rows by 64 keys in shared memory, all fp32; thread (rg, sub) of
// 16 x 16 holds rows rg * RPT.. against keys sub + 16 k, then the same rows'
// dims sub * HD / 16... A row's max and sum are half-warp shuffles. Prefix and
// own items are two launches where their row counts call for other tiles. The
// next tile's loads (V after K in one place) are in flight under the arithmetic.
// Bound by shared memory reads: 64 fp32 rows of the 7B heads behind 16384
// positions take 617 us in all, 25 TFLOP/s, a third of the FMA pipes' rate.
// ---------------------------------------------------------------------------
constexpr int kSaThreads = 256;
constexpr int kSaKT = 64;
constexpr int kSaPad = 4;

template <int HD, int RPT>
__host__ __device__ constexpr size_t sa_simt_smem() {
  return (size_t(16 * RPT) * (HD + kSaPad) + size_t(kSaKT) * (HD + kSaPad) + size_t(16 * RPT) * (kSaKT + kSaPad)) *
         sizeof(float);
}

template <typename T, int HD, int RPT>
__global__ void __launch_bounds__(kSaThreads, RPT == 8 ? 1 : 2) sa_simt_kernel(const SaParams p) {
  constexpr int VE = VecTraits<T>::kElems;
  constexpr int R = 16 * RPT;
  constexpr int DPT = HD / 16;
  constexpr int QS = HD + kSaPad, PS = kSaKT + kSaPad;
  extern __shared__ __align__(16) float smf[];
  float* qs = smf;
  float* ks = qs + size_t(R) * QS;  // a tile of K, then of V
  float* vs = ks;
  float* ps = ks + size_t(kSaKT) * QS;
  pdl_wait();
  pdl_launch();  // after the wait: sa_token_kernel counts on it
  const int tid = threadIdx.x, rg = tid >> 4, sub = tid & 15;
  const SaItem s = sa_item<HD, int(sizeof(T))>(p, p.item0 + blockIdx.x, R, kSaKT);
  for (int i = tid; i < R * (HD / VE); i += kSaThreads) {
    const int r = i / (HD / VE), c = i - r * (HD / VE);
    float f[VE];
    if (r < s.rows) {
      const SaRow x = sa_row(p, s, r);
      unpack(ld_vec(static_cast<const T*>(p.q) + ((size_t(x.n) * p.T + x.t) * p.hq + x.head) * HD + c * VE), f);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) qs[size_t(r) * QS + c * VE + e] = f[e] * p.scale;
  }
  int lim[RPT], low = s.j1;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg * RPT + i;
    lim[i] = r < s.rows ? sa_limit(p, s, sa_row(p, s, r)) : s.j1;
    low = min(low, lim[i]);
  }
  float m[RPT], l[RPT], o[RPT][DPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DPT; ++d) o[i][d] = 0.f;
  }
  // a tile on its way from memory: loaded under the arithmetic on the one before
  constexpr int NV = kSaKT * (HD / VE) / kSaThreads > 0 ? kSaKT * (HD / VE) / kSaThreads : 1;
  uint4 next[NV];
  auto fetch = [&](const void* from, int j0) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = tid + u * kSaThreads, j = i / (HD / VE), c = i - j * (HD / VE);
      next[u] = j < kSaKT && j0 + j < s.j1 ? ld_vec(static_cast<const T*>(from) + size_t(j0 + j) * HD + c * VE)
                                           : make_uint4(0, 0, 0, 0);
    }
  };
  auto put = [&]() {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = tid + u * kSaThreads, j = i / (HD / VE), c = i - j * (HD / VE);
      if (j >= kSaKT) break;
      float f[VE];
      unpack(next[u], f);
#pragma unroll
      for (int e = 0; e < VE; e += 4)
        *reinterpret_cast<float4*>(ks + size_t(j) * QS + c * VE + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    }
  };
  if (s.j0 < s.j1) fetch(s.k, s.j0);
  for (int j0 = s.j0; j0 < s.j1; j0 += kSaKT) {
    __syncthreads();  // the last tile of V is used up (and q is there)
    put();
    __syncthreads();
    fetch(s.v, j0);
    float sc[RPT][4];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) sc[i][k] = 0.f;
    for (int d = 0; d < HD; d += 4) {
      float4 kv[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) kv[k] = *reinterpret_cast<const float4*>(ks + size_t(sub + 16 * k) * QS + d);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 qv = *reinterpret_cast<const float4*>(qs + size_t(rg * RPT + i) * QS + d);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          sc[i][k] = fmaf(qv.w, kv[k].w, fmaf(qv.z, kv[k].z, fmaf(qv.y, kv[k].y, fmaf(qv.x, kv[k].x, sc[i][k]))));
      }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float tm = m[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + sub + 16 * k;
        sc[i][k] = j < s.j1 && j < lim[i] ? sc[i][k] : -INFINITY;
        tm = fmaxf(tm, sc[i][k]);
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, off));
      const float ref = tm == -INFINITY ? 0.f : tm;  // a row that has seen nothing yet keeps exp(-inf) = 0
      const float alpha = expf(m[i] - ref);
      float ts = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = expf(sc[i][k] - ref);
        ps[size_t(rg * RPT + i) * PS + sub + 16 * k] = e;
        ts += e;
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) ts += __shfl_xor_sync(0xffffffffu, ts, off);
      l[i] = l[i] * alpha + ts;
      m[i] = tm;
#pragma unroll
      for (int d = 0; d < DPT; ++d) o[i][d] *= alpha;
    }
    __syncthreads();  // K is used up
    put();
    __syncthreads();
    if (j0 + kSaKT < s.j1) fetch(s.k, j0 + kSaKT);
    // (four keys at a time: behind the range both factors are 0)
    const int kn = min(kSaKT, s.j1 - j0);
    if (j0 + kn > low) {  // keys that not every row sees
#pragma unroll 1
      for (int j = 0; j < kn; ++j)
#pragma unroll
        for (int i = 0; i < RPT; ++i)
          if (j0 + j < lim[i]) {
            const float w = ps[size_t(rg * RPT + i) * PS + j];
#pragma unroll
            for (int d = 0; d < DPT; ++d) o[i][d] = fmaf(w, vs[size_t(j) * QS + sub * DPT + d], o[i][d]);
          }
      continue;
    }
    for (int j = 0; j < kn; j += 4) {
      float4 pr[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) pr[i] = *reinterpret_cast<const float4*>(ps + size_t(rg * RPT + i) * PS + j);
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        float vv[DPT];
        const float* vr = vs + size_t(j + jj) * QS + sub * DPT;
        if constexpr (DPT % 4 == 0) {
#pragma unroll
          for (int d = 0; d < DPT; d += 4) *reinterpret_cast<float4*>(vv + d) = *reinterpret_cast<const float4*>(vr + d);
        } else {
#pragma unroll
          for (int d = 0; d < DPT; ++d) vv[d] = vr[d];
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float w = jj == 0 ? pr[i].x : jj == 1 ? pr[i].y : jj == 2 ? pr[i].z : pr[i].w;
#pragma unroll
          for (int d = 0; d < DPT; ++d) o[i][d] = fmaf(w, vv[d], o[i][d]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg * RPT + i;
    if (r >= s.rows) continue;
    const SaPart at = sa_part<HD>(p, s.own, s.split, s.plane, s.row0 + r);
    if (sub == 0) p.part_ml[at.ml] = make_float2(sa_max_of(m[i], l[i]), l[i]);
    if (s.j0 < s.j1)
#pragma unroll
      for (int d = 0; d < DPT; ++d) {
        const int dim = sub * DPT + d;
        p.part_o[at.o + (dim >> 2) * 128 + (dim & 3)] = o[i][d];
      }
  }
}

// ---------------------------------------------------------------------------
// One token a row, bf16, head dim 64 or 128: a CTA takes up to 16 query heads
// of one (row, KV head) and streams the row's own cache (and, inline, the
// prefix) from global memory straight into mma.sync fragments, 16 keys a warp
// and step, the warps on every NW-th block of 16 keys. A K or V byte is used
// once, so the kernel is bound by the loads (a block's are in flight under the
// arithmetic of the one before), and the tensor instructions cost less than
// unpacking to fp32 would. S = Q K^T has 16 rows (heads, half of them unused
// below 9), O^T = V^T P^T has 8 or 16 columns (heads): the registers of P, a
// result of the first, are as they stand the B operand of the second.
//
// Fragments without shared memory: the dot product's order of dims and the
// output's order of dims are free, so both are chosen to make every load 16
// bytes. Thread (g = lane / 4, c = lane % 4) loads dims 32 j + 8 c .. + 7 of
// key g (K) or head g (Q): four register pairs that serve as the "k" and
// "k + 8" halves of two steps. For V it loads keys 2c, 2c+1, 2c+8, 2c+9 at
// dims 64 b + 8 g .. + 7; two keys' values of a dim, put together by a byte
// permute, are an operand of row g of an output tile.
//
// Probabilities are rounded to bf16 for the second product (the sums of the
// denominator are not): half a step of bf16 of each term, as the result's own
// rounding.
//
// 64 rows of the 7B heads with 500 own positions (66 MB) add 14 us to a call,
// 4.7 TB/s.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kSaTokenWarps = 4;  // 8 took 57.5 us where 4 took 55.8 (64 rows of the 7B heads behind 16384 positions)
constexpr int kSaMaxSplits = 64, kSaMaxOwn = 32;  // key ranges of a prefix, of an own cache

// WIDE: more than 8 heads a tile (rows 8..15 in use).
template <int HD, bool WIDE>
__host__ __device__ constexpr size_t sa_token_smem() {
  return size_t(kSaTokenWarps) * (WIDE ? 16 : 8) * (HD + 2) * sizeof(float);
}

template <int HD, bool WIDE>
__global__ void __launch_bounds__(32 * kSaTokenWarps, 2) sa_token_kernel(const SaParams p, const int inline_prefix) {  // inline_prefix: so == 1, no prefix items
  constexpr int NT = WIDE ? 2 : 1, R = 8 * NT;
  constexpr int JB = HD / 32, VB = HD / 64, NW = kSaTokenWarps;
  extern __shared__ __align__(16) float smf[];
  __shared__ float2 pml[kSaMaxSplits * R];  // max and sum of the prefix's key ranges
  float* so = smf;                  // [NW][R][HD]
  float* sml = so + NW * R * HD;    // [NW][R][2]
  // the kernel of the prefix items, if one runs before this, has waited for
  // the kernels before it: only its partial sums are not yet there
  pdl_launch();
  if (inline_prefix) pdl_wait();
  const int per = p.hq / p.hkv;
  const int tile = blockIdx.x % p.otiles, kvh = blockIdx.x / p.otiles;
  const int n = blockIdx.y, split = blockIdx.z;
  const int rows = min(16, per - tile * 16);
  const int head0 = kvh * per + tile * 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int gi = n / p.W;
  const size_t po = (size_t(gi) * p.hkv + kvh) * p.cap_p * HD, co = (size_t(n) * p.hkv + kvh) * p.cap * HD;
  const int plen = inline_prefix ? sa_prefix_len(p, gi) : 0;
  const int clen = sa_cache_len(p, n);
  const int chunk = ((clen + p.so - 1) / p.so + 15) / 16 * 16;
  const int own0 = min(clen, split * chunk), own1 = min(clen, own0 + chunk);
  uint4 q0[JB], q1[JB];
  {
    const bf16* qp = static_cast<const bf16*>(p.q) + (size_t(n) * p.hq + head0) * HD + c * 8;
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      q0[j] = g < rows ? ld_vec(qp + size_t(g) * HD + 32 * j) : make_uint4(0, 0, 0, 0);
      q1[j] = WIDE && g + 8 < rows ? ld_vec(qp + size_t(g + 8) * HD + 32 * j) : make_uint4(0, 0, 0, 0);
    }
  }
  const float sl2 = p.scale * kLog2e;
  float m[NT], l[NT];  // of heads g and g + 8: max (scaled, base 2), this thread's part of the sum
  float o[NT][VB * 4][4];  // dims x heads: [head half][64 v + 8 g + 2 w + row half][head 2c, 2c + 1]
#pragma unroll
  for (int h = 0; h < NT; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < VB * 4; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
  }
  const int nb0 = (plen + 15) / 16, nb = nb0 + (own1 - own0 + 15) / 16;
  struct Block {
    uint4 k[2][JB], v[4][VB];
  };
  auto load = [&](Block& f, int b) {
    if (b >= nb) return;
    const bool own = b >= nb0;
    const int key0 = own ? own0 + (b - nb0) * 16 : b * 16, end = own ? own1 : plen;
    const size_t at = (own ? co : po) + size_t(key0) * HD;
    const bf16* kp = static_cast<const bf16*>(own ? p.kc : p.kp) + at + c * 8;
    const bf16* vp = static_cast<const bf16*>(own ? p.vc : p.vp) + at + g * 8;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < JB; ++j)
        f.k[t][j] = key0 + 8 * t + g < end ? ld_stream(kp + size_t(8 * t + g) * HD + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 2 * c + (r & 1) + (r >> 1) * 8;
#pragma unroll
      for (int v = 0; v < VB; ++v)
        f.v[r][v] = key0 + k < end ? ld_stream(vp + size_t(k) * HD + 64 * v) : make_uint4(0, 0, 0, 0);
    }
  };
  auto step = [&](const Block& f, int b) {
    const bool own = b >= nb0;
    const int key0 = own ? own0 + (b - nb0) * 16 : b * 16, end = own ? own1 : plen;
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        mma_bf16(s[t], q0[j].x, q1[j].x, q0[j].y, q1[j].y, f.k[t][j].x, f.k[t][j].y);
        mma_bf16(s[t], q0[j].z, q1[j].z, q0[j].w, q1[j].w, f.k[t][j].z, f.k[t][j].w);
      }
    }
    float x[NT];
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      x[h] = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[t][2 * h + e] = key0 + 8 * t + 2 * c + e < end ? s[t][2 * h + e] * sl2 : -INFINITY;
          x[h] = fmaxf(x[h], s[t][2 * h + e]);
        }
      x[h] = fmaxf(x[h], __shfl_xor_sync(0xffffffffu, x[h], 1));
      x[h] = fmaxf(x[h], __shfl_xor_sync(0xffffffffu, x[h], 2));
    }
    // (a row of scores that are all -inf keeps its max: exp(-inf - 0) = 0)
    if (__any_sync(0xffffffffu, x[0] > m[0] || x[NT - 1] > m[NT - 1])) {
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        const float top = fmaxf(m[h], x[h]), a = exp2_approx(m[h] - (top == -INFINITY ? 0.f : top));
        m[h] = top;
        l[h] *= a;
        const float a0 = __shfl_sync(0xffffffffu, a, 8 * c), a1 = __shfl_sync(0xffffffffu, a, 8 * c + 4);
#pragma unroll
        for (int i = 0; i < VB * 4; ++i) {
          o[h][i][0] *= a0;
          o[h][i][1] *= a1;
          o[h][i][2] *= a0;
          o[h][i][3] *= a1;
        }
      }
    }
    uint32_t pb[NT][2];  // [head half][key half]
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      const float ref = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float e0 = exp2_approx(s[t][2 * h] - ref), e1 = exp2_approx(s[t][2 * h + 1] - ref);
        l[h] += e0 + e1;
        pb[h][t] = pack_bf16(e0, e1);
      }
    }
#pragma unroll
    for (int v = 0; v < VB; ++v) {
      const uint32_t* k0 = reinterpret_cast<const uint32_t*>(&f.v[0][v]);
      const uint32_t* k1 = reinterpret_cast<const uint32_t*>(&f.v[1][v]);
      const uint32_t* k8 = reinterpret_cast<const uint32_t*>(&f.v[2][v]);
      const uint32_t* k9 = reinterpret_cast<const uint32_t*>(&f.v[3][v]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // lower and upper halves of the two keys' words: dims 2w and 2w + 1
        const uint32_t a0 = __byte_perm(k0[w], k1[w], 0x5410u), a1 = __byte_perm(k0[w], k1[w], 0x7632u);
        const uint32_t a2 = __byte_perm(k8[w], k9[w], 0x5410u), a3 = __byte_perm(k8[w], k9[w], 0x7632u);
#pragma unroll
        for (int h = 0; h < NT; ++h) mma_bf16(o[h][v * 4 + w], a0, a1, a2, a3, pb[h][0], pb[h][1]);
      }
    }
  };
  // the next block's loads are in flight under this one's arithmetic
  Block f0, f1;
  load(f0, warp);
  for (int b = warp; b < nb; b += 2 * NW) {
    load(f1, b + NW);
    step(f0, b);
    if (b + NW >= nb) break;
    load(f0, b + 2 * NW);
    step(f1, b + NW);
  }
#pragma unroll
  for (int h = 0; h < NT; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (c == 0) *reinterpret_cast<float2*>(sml + (warp * R + g + 8 * h) * 2) = make_float2(sa_max_of(m[h] * kLn2, l[h]), l[h]);
#pragma unroll
    for (int v = 0; v < VB; ++v)
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(so + (warp * R + 8 * h + 2 * c + e) * HD + 64 * v + 8 * g + 2 * w) =
              make_float2(o[h][v * 4 + w][e], o[h][v * 4 + w][2 + e]);
  }
  if (!inline_prefix) pdl_wait();  // the prefix items' partial sums
  const bool last = p.so == 1;  // else partial sums for the join
  const int pslots = last && !inline_prefix ? p.sp : 0;
  const int pplane = gi * p.hkv + kvh, pr0 = (n - gi * p.W) * per + tile * 16;  // this tile's first row of the prefix plane
  for (int i = threadIdx.x; i < pslots * R; i += 32 * NW)
    if (i % R < rows) pml[i] = __ldcg(p.part_ml + sa_part<HD>(p, false, i / R, pplane, pr0 + i % R).ml);
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (HD / 4); i += 32 * NW) {
    const int q = i / rows, r = i - q * rows;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sml[(w * R + r) * 2]);
    for (int s = 0; s < pslots; ++s) mx = fmaxf(mx, pml[s * R + r].x);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
    auto add = [&](float m, float l, const float4& f) {
      const float w = m == -INFINITY ? 0.f : expf(m - ref);
      den = fmaf(w, l, den);
      if (m != -INFINITY) {  // an empty range leaves its sums unwritten; one of weight 0 may hold a NaN
        num[0] = fmaf(w, f.x, num[0]);
        num[1] = fmaf(w, f.y, num[1]);
        num[2] = fmaf(w, f.z, num[2]);
        num[3] = fmaf(w, f.w, num[3]);
      }
    };
#pragma unroll
    for (int w = 0; w < NW; ++w)
      add(sml[(w * R + r) * 2], sml[(w * R + r) * 2 + 1], *reinterpret_cast<const float4*>(so + (w * R + r) * HD + 4 * q));
    constexpr int U = 4;  // ranges whose sums are loaded together
    for (int s0 = 0; s0 < pslots; s0 += U) {
      float4 f[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s0 + u < pslots)
          f[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + sa_part<HD>(p, false, s0 + u, pplane, pr0 + r).o + q * 128));
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s0 + u < pslots) add(pml[(s0 + u) * R + r].x, pml[(s0 + u) * R + r].y, f[u]);
    }
    if (last) {
      const float inv = den > 0.f ? 1.f / den : 0.f;
      *reinterpret_cast<uint2*>(static_cast<bf16*>(p.out) + (size_t(n) * p.hq + head0 + r) * HD + 4 * q) =
          make_uint2(pack_bf16(num[0] * inv, num[1] * inv), pack_bf16(num[2] * inv, num[3] * inv));
    } else {
      const SaPart at = sa_part<HD>(p, true, split, n * p.hkv + kvh, tile * 16 + r);
      if (q == 0) p.part_ml[at.ml] = make_float2(sa_max_of(mx, den), den);
      *reinterpret_cast<float4*>(p.part_o + at.o + q * 128) = make_float4(num[0], num[1], num[2], num[3]);
    }
  }
}

// ---------------------------------------------------------------------------
// Items on the tensor cores (bf16, head dim 64 or 128), one item a CTA, key
// tiles of 128. Two streams share the K and V tiles' ring, each with an MMA
// warp, a softmax warpgroup (a row a thread) and its own tensor memory:
//   MT 2: stream x has rows 128 x .. of the item's 256 and all key tiles, so
//         a K/V byte brought in from L2 serves 256 rows;
//   MT 1: both have the item's 128 rows, stream x the key tiles t = x mod 2,
//         and the streams are joined at the end.
// One stream's softmax runs under the other's and under the MMAs:
//   warp 0 loads (TMA, 128 keys x 64 dims boxes, 128-byte swizzle), warps 1
//   and 2 issue S = Q K^T and O += P V of their stream, warps 4-7 and 8-11
//   turn S into P.
// P is bf16 in tensor memory, the A operand of P V; for head dim 128, where S
// and O fill the 512 columns, it takes the place of its S, and the stream's
// next S waits for the P V that reads it. V is read as it lies (N-major B).
// The max that the exponentials are taken against is replaced, and O rescaled
// in tensor memory, only when a row's max has grown by more than 2^8: until
// then P is at most 2^8, which costs no precision, as the division by the sum
// takes the factor out.
// Keys from the end of the range on are masked by selection; their V rows are
// zeroed in shared memory, since 0 x NaN would not be 0. In tiles of own items
// that not every token sees, the NaN and infinities among V are zeroed too; a
// negative sum tells the join, which adds them to the rows that do see them.
// (Added here they cost the softmax registers: 66 -> 76 us on 16 rows of 128
// tokens behind 4001.)
//
// A key tile is bound by the chain S -> softmax -> P V of a stream, of which two
// run against each other: about 3580 cycles a pair of key tiles for head dim 128
// and 3010 for 64, of which the special-function unit has 1430. An item's start
// (barriers, tensor memory, Q, the first tiles) and end (the partial sums) come
// on top, 8 us where a call's items have one tile instead of none. 64 rows of the
// 7B heads behind 16384 positions: 28 us, 0.54 PFLOP/s, of which the 8 tiles of a
// range are 15, on 128 of 148 SMs; 16 rows of 128 tokens of the 0.5B heads behind
// 4001 and 150: 57 us, 0.52 PFLOP/s, of which the 32 tiles are 51, on 112 SMs.
// ---------------------------------------------------------------------------
constexpr int kSaTcKeys = 128;
// Of 16 pairs of exponentials, on the fp32 pipe (0, 2, 4, 6: 46.6, 46.8, 46.5,
// 47.1 us on 64 rows of the 7B heads behind 16384 positions; 67.4, 68.8, 65.9,
// 71.2 us on 16 rows of 128 tokens behind 4001).
constexpr int kSaCubic = 4;
constexpr int kSaTcThreads = 384;
constexpr uint32_t kSaTcSub = kTcSub;

template <int HD, int MT>
struct SaTcCfg {
  static constexpr int kSubs = HD / 64;
  static constexpr uint32_t kTile = kSubs * kSaTcSub;  // a K, V or Q tile
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
__global__ void __launch_bounds__(kSaTcThreads, 1)
    sa_tc_kernel(const SaParams p, const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                 const __grid_constant__ CUtensorMap map_kc, const __grid_constant__ CUtensorMap map_vc) {
  using C = SaTcCfg<HD, MT>;
  constexpr int NB = C::kRing;
  constexpr uint64_t kBudget = 2000000000ull;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[NB], empty[NB], qfull, s_full[2], s_free[2], p_full[2][2], pv_done[2], drain[2], turn[2][4];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_sh, odd_sh;  // odd_sh: values of V were zeroed
  __shared__ float2 ml_sh[128];  // MT 1: stream 1's statistics
  volatile int* abort = &abort_sh;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  pdl_wait();
  pdl_launch();  // after the wait: sa_token_kernel counts on it
  const SaItem it = sa_item<HD, 2>(p, blockIdx.x, 128 * MT, kSaTcKeys);
  if (it.j0 >= it.j1) {
    for (int r = threadIdx.x; r < it.rows; r += kSaTcThreads)
      p.part_ml[sa_part<HD>(p, it.own, it.split, it.plane, it.row0 + r).ml] = make_float2(-INFINITY, 0.f);
    return;
  }
  const int nt = (it.j1 - it.j0 + kSaTcKeys - 1) / kSaTcKeys;
  // tiles of a stream: first, step
  constexpr int kStep = MT == 2 ? 1 : 2;
  if (threadIdx.x == 0) {
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
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  int issued = 0;  // warp 0: ring entries whose copies were issued

  if (warp == 0) {
    const CUtensorMap* mk = it.own ? &map_kc : &map_kp;
    const CUtensorMap* mv = it.own ? &map_vc : &map_vp;
    for (int i = 0; i < 2 * nt; ++i) {  // K and V of each tile in turn
      const int s = i % NB, j = it.j0 + (i >> 1) * kSaTcKeys;
      const bool ok = i < NB || mbar_wait_soon(empty + s, uint32_t((i / NB) & 1) ^ 1u, kBudget, abort);
      if (!__all_sync(0xffffffffu, ok)) {
        *abort = 1;
        break;
      }
      if (elect_one()) {
        mbar_arrive_expect_tx(full + s, C::kTile);
#pragma unroll
        for (int b = 0; b < C::kSubs; ++b)
          tma_load_3d(base + C::kOffRing + s * C::kTile + b * kSaTcSub, i & 1 ? mv : mk, b * 64, j, it.plane, full + s);
      }
      issued = i + 1;
    }
  } else if (warp == 1 || warp == 2) {
    // ---- MMA issue of stream x
    const int x = warp - 1, first = MT == 2 ? 0 : x;
    const uint64_t dq = tc_smem_desc(base + (MT == 2 ? x : 0) * C::kTile);
    const uint32_t ts = tmem + x * C::kS, to = tmem + C::kO + x * HD, tp = tmem + C::kP + x * C::kPStep;
    auto wait = [&](uint64_t* bar, int phase) {
      return __all_sync(0xffffffffu, mbar_wait_soon(bar, uint32_t(phase & 1), kBudget, abort));
    };
    auto qk = [&](int t, int k) {
      const int i = 2 * t, s = i % NB;
      // S is free: read by the softmax, and (aliased) its P read by P V
      if (!wait(full + s, i / NB) || (k > 0 && !wait(C::kAlias ? pv_done + x : s_free + x, k - 1))) return false;
      tc_fence_after();
      const uint64_t dk = tc_smem_desc(base + C::kOffRing + s * C::kTile);
      if (elect_one()) {
#pragma unroll
        for (int q = 0; q < HD / 16; ++q) {
          const uint32_t off = ((q >> 2) * kSaTcSub + (q & 3) * 32) >> 4;
          tc_mma(ts, dq + off, dk + off, C::kIdescS, q > 0 ? 1u : 0u);
        }
        tc_commit(s_full + x);
        tc_commit(empty + s);
      }
      __syncwarp();
      return true;
    };
    auto pv = [&](int t, int k) {
      const int i = 2 * t + 1, s = i % NB;
      if (!wait(full + s, i / NB)) return false;
      const uint64_t dv = tc_smem_desc_mn(base + C::kOffRing + s * C::kTile, kSaTcSub);
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
    bool ok = first >= nt || wait(&qfull, 0);
    if (C::kAlias) {
      for (int t = first, k = 0; ok && t < nt; t += kStep, ++k) ok = qk(t, k) && pv(t, k);
    } else {  // the next S under this one's softmax
      if (ok && first < nt) ok = qk(first, 0);
      for (int t = first, k = 0; ok && t < nt; t += kStep, ++k) {
        if (t + kStep < nt) ok = qk(t + kStep, k + 1);
        ok = ok && pv(t, k);
      }
    }
    if (!ok) *abort = 1;
  } else if (warp >= 4) {
    // ---- softmax of stream x
    const int stid = int(threadIdx.x) - 128, x = stid >> 7;
    const int quarter = warp & 3, r = quarter * 32 + lane;
    {  // Q: a warp's rows, whole rows side by side in the lanes, all loads in flight at once
      constexpr int RW = 16 * MT, CH = HD / 8, RI = 32 / CH, N = RW / RI;  // rows a warp, chunks a row, rows a load
      const int row0 = (warp - 4) * RW, at = row0 + (lane & (RW - 1));
      unsigned long long off = ~0ull;  // of row `at` in q
      if (at < it.rows) {
        const SaRow w = sa_row(p, it, at);
        off = ((size_t(w.n) * p.T + w.t) * p.hq + w.head) * HD;
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
        *reinterpret_cast<uint4*>(smem + (row >> 7) * C::kTile + (c >> 3) * kSaTcSub + (row & 127) * 128 +
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
    SaRow w = {};
    if (write) w = sa_row(p, it, row);
    const int lim = write ? min(it.j1, sa_limit(p, it, w)) : it.j1;  // keys [0, lim) are seen
    const float sl2 = p.scale * kLog2e;
    const int low = p.T > 1 ? min(it.j1, sa_limit(p, it, sa_row(p, it, 0))) : it.j1;  // keys [0, low) are seen by all
    float m = -INFINITY, l = 0.f;  // reference max (scaled, base 2), sum
    bool ok = true;
    int k = 0;
    for (int t = MT == 2 ? 0 : x; t < nt; t += kStep, ++k) {
      const int j = it.j0 + t * kSaTcKeys;
      ok = mbar_wait_soon(s_full + x, uint32_t(k & 1), kBudget, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      float sc[kSaTcKeys];
#pragma unroll
      for (int c = 0; c < kSaTcKeys; c += 32) tc_ld32(ts + c, reinterpret_cast<uint32_t*>(sc + c));
      tc_wait_ld();
      if (!C::kAlias) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free + x);
      }
      const bool masked = __any_sync(0xffffffffu, j + kSaTcKeys > lim);
      if (masked) {
#pragma unroll
        for (int c = 0; c < kSaTcKeys; ++c) sc[c] = j + c < lim ? sc[c] : -INFINITY;
      }
      float mx[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
      for (int c = 4; c < kSaTcKeys - 4; c += 8)
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
      if (j + kSaTcKeys > low) {  // V rows behind the range, or not seen by all (MT 2: both streams write the same zeros)
        const int i = 2 * t + 1, s = i % NB;
        ok = mbar_wait_soon(full + s, uint32_t((i / NB) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_clean_row<HD>(smem + C::kOffRing + s * C::kTile, r, j + r >= it.j1, j + r >= low, &odd_sh);
        fence_async_smem();
      }
      // the exponentials of the two warps of a scheduler take turns: one stream's
      // run under the other's MMAs, and not both at half pace (51.3 -> 49.1 us)
      if (x == 1 || k > 0) {
        ok = mbar_wait_soon(&turn[x][quarter], uint32_t(x == 1 ? k & 1 : (k - 1) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      // kCubic of 16 pairs on the fp32 pipe, which the special-function unit
      // (8 cycles a warp and value) leaves idle; masked tiles need exact zeros
      auto exps = [&](auto cubic) {
        constexpr int kCubic = decltype(cubic)::value;
#pragma unroll
        for (int c = 0; c < kSaTcKeys; c += 32) {
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
        exps(std::integral_constant<int, kSaCubic>{});
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
      const float top = fmaxf(m, b.x), ref = top == -INFINITY ? 0.f : top;
      wa = exp2_approx(m - ref);
      wb = exp2_approx(b.x - ref);
      l = l * wa + b.y * wb;
      m = top;
    }
    m = sa_max_of(m, l);  // (MT 2: tiles behind the NaN have set another max)
    if (MT == 2 || x == 0) {
      const SaPart at = sa_part<HD>(p, it.own, it.split, it.plane, it.row0 + row);
      if (odd_sh) l = -l;
      if (write) p.part_ml[at.ml] = make_float2(m * kLn2, l);
#pragma unroll
      for (int c = 0; c < HD; c += 16) {
        uint32_t o0[16], o1[16];
        tc_ld16(to + c, o0);
        if (MT == 1 && nt > 1) tc_ld16(to + HD + c, o1);
        tc_wait_ld();
        if (write) {
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f[i] = __uint_as_float(o0[e + i]) * wa;
              if (MT == 1 && nt > 1) f[i] = fmaf(__uint_as_float(o1[e + i]), wb, f[i]);
            }
            *reinterpret_cast<float4*>(p.part_o + at.o + (c + e) * 32) = make_float4(f[0], f[1], f[2], f[3]);
          }
        }
      }
    }
  }
  __syncwarp();
  // ---- teardown: copies and MMAs in flight land before the memory goes away
  if (warp == 0) {
    int never = 0;
    for (int i = max(0, issued - NB); i < issued; ++i) mbar_wait(full + i % NB, uint32_t((i / NB) & 1), kBudget, &never);
  }
  if (warp == 1 || warp == 2) {
    // behind every MMA of the warp (a commit follows those of its own thread:
    // the elected lane is the same each time)
    int never = 0;
    if (elect_one()) tc_commit(drain + warp - 1);
    __syncwarp();
    mbar_wait(drain + warp - 1, 0u, kBudget, &never);
  }
  tc_fence_before();
  __syncthreads();

  if (threadIdx.x == 0 && *abort) atomicOr(p.status ? p.status : &g_sa_status, kStatusTimeout);
  if (warp == 3) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Join of the key ranges: a CTA takes 32 rows of an own plane. The ranges'
// weights come first (a thread a row and range); then a thread sums 4 dims of
// a row over the ranges, four loads in flight; the result goes through shared
// memory so that whole rows are written. Latency and the partial sums' bytes:
// 10 us with the launch before it for 28672 rows of head dim 64.
// ---------------------------------------------------------------------------
constexpr int kSaJoinThreads = 256;

template <typename T, int HD>
__global__ void __launch_bounds__(kSaJoinThreads) sa_join_kernel(const SaParams p) {
  constexpr int VE = VecTraits<T>::kElems, U = 4;
  extern __shared__ float2 sa_ml[];  // a range and row: max, sum; then weight, -1 for an empty range
  float2* ml = sa_ml;
  __shared__ float res[32][HD + 1];
  __shared__ float inv[32];
  __shared__ int odd[32];  // keys [odd, ..) of the own cache may hold values of V that were left out; -1: none
  pdl_launch();
  pdl_wait();
  const int per = p.hq / p.hkv, tid = threadIdx.x;
  const int blk = blockIdx.x % p.oblocks, plane = blockIdx.x / p.oblocks;
  const int n = plane / p.hkv, kvh = plane - n * p.hkv, gi = n / p.W;
  const int total = p.T * per, rows = min(32, total - blk * 32), slots = p.sp + p.so;
  const int pr0 = (n - gi * p.W) * total + blk * 32, pplane = gi * p.hkv + kvh;
  auto part = [&](int s, int r) {
    return s < p.sp ? sa_part<HD>(p, false, s, pplane, pr0 + r) : sa_part<HD>(p, true, s - p.sp, plane, blk * 32 + r);
  };
  for (int i = tid; i < slots * 32; i += kSaJoinThreads)
    if ((i & 31) < rows) ml[i] = __ldcg(p.part_ml + part(i >> 5, i & 31).ml);
  __syncthreads();
  if (tid < rows) {
    float mx = -INFINITY, den = 0.f;
    bool left_out = false;
    for (int s = 0; s < slots; ++s) mx = fmaxf(mx, ml[s * 32 + tid].x);
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int s = 0; s < slots; ++s) {
      const float2 v = ml[s * 32 + tid];
      left_out |= v.y < 0.f;
      if (v.x == -INFINITY) {
        ml[s * 32 + tid].x = -1.f;
        continue;
      }
      const float w = expf(v.x - ref);
      den = fmaf(w, fabsf(v.y), den);
      ml[s * 32 + tid].x = w;
    }
    odd[tid] = left_out ? max(0, sa_cache_len(p, n) - (p.T - 1)) : -1;
    inv[tid] = den > 0.f ? 1.f / den : 0.f;
  }
  __syncthreads();
  for (int i = tid; i < rows * (HD / 4); i += kSaJoinThreads) {
    const int q = i / rows, r = i - q * rows;
    float num[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < slots; s0 += U) {
      float4 f[U];
      float w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        w[u] = s0 + u < slots ? ml[(s0 + u) * 32 + r].x : -1.f;
        if (!(w[u] < 0.f))  // an empty range leaves its sums unwritten
          f[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + part(s0 + u, r).o + q * 128));
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!(w[u] < 0.f)) {  // (a weight of 0 takes a NaN or an infinity among the sums along)
          num[0] = fmaf(w[u], f[u].x, num[0]);
          num[1] = fmaf(w[u], f[u].y, num[1]);
          num[2] = fmaf(w[u], f[u].z, num[2]);
          num[3] = fmaf(w[u], f[u].w, num[3]);
        }
    }
    if (odd[r] >= 0) {
      const T* v = static_cast<const T*>(p.vc) + size_t(plane) * p.cap * HD + 4 * q;
      const int end = sa_cache_len(p, n) - (p.T - 1 - (blk * 32 + r) / per);
      for (int key = odd[r]; key < end; ++key)
        for (int e = 0; e < 4; ++e) {
          const float x = to_f(v[size_t(key) * HD + e]);
          if (!(fabsf(x) < INFINITY)) num[e] += x;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) res[r][4 * q + e] = num[e] * inv[r];
  }
  __syncthreads();
  for (int i = tid; i < rows * (HD / VE); i += kSaJoinThreads) {
    const int r = i / (HD / VE), c = (i - r * (HD / VE)) * VE, row = blk * 32 + r;
    float f[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = res[r][c + e];
    const int t = row / per, head = kvh * per + row - t * per;
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + ((size_t(n) * p.T + t) * p.hq + head) * HD + c) = pack_vec(f);
  }
}

}  // namespace mtpb
