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
#pragma once

#include "common.cuh"

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
  float* part_o;     // [slot][row = (n * T + t) * hq + h][hd]
  float* part_ml;    // [slot][row][2]: max (base e, scaled), sum
};

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
  int n0, kvh, slot;  // first batch row
  bool own;
};

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
    const size_t off = (size_t(g) * p.hkv + s.kvh) * p.cap_p * HD * ES;
    s.k = static_cast<const char*>(p.kp) + off;
    s.v = static_cast<const char*>(p.vp) + off;
    s.slot = split;
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
    const size_t off = (size_t(s.n0) * p.hkv + s.kvh) * p.cap * HD * ES;
    s.k = static_cast<const char*>(p.kc) + off;
    s.v = static_cast<const char*>(p.vc) + off;
    s.slot = p.sp + split;
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

// ---------------------------------------------------------------------------
// Items on the CUDA cores (fp32, and bf16 head dims below 64): tiles of
// 16 * RPT rows by 64 keys in shared memory, all fp32; thread (rg, sub) of
// 16 x 16 holds rows rg * RPT.. against keys sub + 16 k, then the same rows'
// dims sub * HD / 16... A row's max and sum are half-warp shuffles.
// ---------------------------------------------------------------------------
constexpr int kSaThreads = 256;
constexpr int kSaKT = 64;
constexpr int kSaPad = 4;

template <int HD, int RPT>
__host__ __device__ constexpr size_t sa_simt_smem() {
  return (size_t(16 * RPT) * (HD + kSaPad) + 2 * size_t(kSaKT) * (HD + kSaPad) + size_t(16 * RPT) * (kSaKT + kSaPad)) *
         sizeof(float);
}

template <typename T, int HD, int RPT>
__global__ void __launch_bounds__(kSaThreads) sa_simt_kernel(const SaParams p) {
  constexpr int VE = VecTraits<T>::kElems;
  constexpr int R = 16 * RPT;
  constexpr int DPT = HD / 16;
  constexpr int QS = HD + kSaPad, PS = kSaKT + kSaPad;
  extern __shared__ __align__(16) float smf[];
  float* qs = smf;
  float* ks = qs + size_t(R) * QS;
  float* vs = ks + size_t(kSaKT) * QS;
  float* ps = vs + size_t(kSaKT) * QS;
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x, rg = tid >> 4, sub = tid & 15;
  const SaItem s = sa_item<HD, int(sizeof(T))>(p, blockIdx.x, R, kSaKT);
  const size_t nrow = size_t(p.G) * p.W * p.T * p.hq;
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
  int lim[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg * RPT + i;
    lim[i] = r < s.rows ? sa_limit(p, s, sa_row(p, s, r)) : 0;
  }
  float m[RPT], l[RPT], o[RPT][DPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DPT; ++d) o[i][d] = 0.f;
  }
  for (int j0 = s.j0; j0 < s.j1; j0 += kSaKT) {
    __syncthreads();
    for (int i = tid; i < kSaKT * (HD / VE); i += kSaThreads) {
      const int j = i / (HD / VE), c = i - j * (HD / VE);
      float kf[VE], vf[VE];
      if (j0 + j < s.j1) {
        unpack(ld_vec(static_cast<const T*>(s.k) + size_t(j0 + j) * HD + c * VE), kf);
        unpack(ld_vec(static_cast<const T*>(s.v) + size_t(j0 + j) * HD + c * VE), vf);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) kf[e] = vf[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        ks[size_t(j) * QS + c * VE + e] = kf[e];
        vs[size_t(j) * QS + c * VE + e] = vf[e];
      }
    }
    __syncthreads();
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
    __syncwarp();
    const int kn = min(kSaKT, s.j1 - j0);
    for (int j = 0; j < kn; ++j) {
      float vv[DPT];
#pragma unroll
      for (int d = 0; d < DPT; ++d) vv[d] = vs[size_t(j) * QS + sub * DPT + d];
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float pr = ps[size_t(rg * RPT + i) * PS + j];
#pragma unroll
        for (int d = 0; d < DPT; ++d) o[i][d] = fmaf(pr, vv[d], o[i][d]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg * RPT + i;
    if (r >= s.rows) continue;
    const SaRow x = sa_row(p, s, r);
    const size_t at = s.slot * nrow + (size_t(x.n) * p.T + x.t) * p.hq + x.head;
    if (sub == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m[i], l[i]);
    if (s.j0 < s.j1)
#pragma unroll
      for (int d = 0; d < DPT; ++d) p.part_o[at * HD + sub * DPT + d] = o[i][d];
  }
}

// ---------------------------------------------------------------------------
// Join of the slots: one thread per (row, 4 dims).
// ---------------------------------------------------------------------------
constexpr int kSaJoinThreads = 256;

template <typename T, int HD>
__global__ void __launch_bounds__(kSaJoinThreads) sa_join_kernel(const SaParams p) {
  pdl_launch();
  pdl_wait();
  const size_t nrow = size_t(p.G) * p.W * p.T * p.hq;
  const size_t i = size_t(blockIdx.x) * kSaJoinThreads + threadIdx.x;
  const size_t row = i / (HD / 4);
  const int d = int(i - row * (HD / 4)) * 4;
  if (row >= nrow) return;
  const int slots = p.sp + p.so;
  float mx = -INFINITY;
  for (int s = 0; s < slots; ++s) mx = fmaxf(mx, p.part_ml[(s * nrow + row) * 2]);
  float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
  for (int s = 0; s < slots; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * nrow + row) * 2);
    if (ml.x == -INFINITY) continue;
    const float w = expf(ml.x - mx);
    den = fmaf(w, ml.y, den);
    const float4 o = *reinterpret_cast<const float4*>(p.part_o + (s * nrow + row) * HD + d);
    num[0] = fmaf(w, o.x, num[0]);
    num[1] = fmaf(w, o.y, num[1]);
    num[2] = fmaf(w, o.z, num[2]);
    num[3] = fmaf(w, o.w, num[3]);
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  T* dst = static_cast<T*>(p.out) + row * HD + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) dst[e] = from_f<T>(num[e] * inv);
}

}  // namespace mtpb
