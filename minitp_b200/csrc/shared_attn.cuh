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

#include "tcgen05.cuh"

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
  int n0, kvh, slot;  // first batch row
  int plane;          // (group or row) x KV head: which [cap][hd] block of the cache
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
    s.plane = g * p.hkv + s.kvh;
    const size_t off = size_t(s.plane) * p.cap_p * HD * ES;
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
    s.plane = s.n0 * p.hkv + s.kvh;
    const size_t off = size_t(s.plane) * p.cap * HD * ES;
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
  pdl_wait();
  pdl_launch();  // after the wait: sa_token_kernel counts on it
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
// One token a row, bf16, head dim 64 or 128: a CTA takes up to 16 query heads
// of one (row, KV head) and streams the row's own cache (and, inline, the
// prefix) from global memory straight into mma.sync fragments: 16 rows (heads)
// x 16 keys a warp and step, the warps on every NW-th block of 16 keys. A
// K or V byte is used once, so the kernel is bound by the loads, and the
// 16-row tensor instructions cost less than unpacking to fp32 would.
//
// Fragments without shared memory: the dot product's order of dims and the
// output's order of dims are free, so both are chosen to make every load 16
// bytes. Thread (g = lane / 4, c = lane % 4) loads dims 32 j + 8 c .. + 7 of
// key g (K) or head g (Q): four register pairs that serve as the "k" and
// "k + 8" halves of two steps. For V it loads keys 2c, 2c+1, 2c+8, 2c+9 at
// dims 64 b + 8 g .. + 7; two keys' values of a dim, put together by a byte
// permute, are the operand of column g of output tile i = dim % 8.
//
// Probabilities are rounded to bf16 for the second product (the sums of the
// denominator are not): half a step of bf16 of each term, as the result's own
// rounding.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// NW warps; WIDE: more than 8 heads a tile (rows 8..15 in use).
template <int HD, int NW, bool WIDE>
__host__ __device__ constexpr size_t sa_token_smem() {
  return size_t(NW) * (WIDE ? 16 : 8) * (HD + 2) * sizeof(float);
}

template <int HD, int NW, bool WIDE>
__global__ void __launch_bounds__(32 * NW) sa_token_kernel(const SaParams p, const int inline_prefix) {  // inline_prefix: so == 1, no prefix items
  constexpr int R = WIDE ? 16 : 8;
  constexpr int JB = HD / 32, VB = HD / 64;
  extern __shared__ __align__(16) float smf[];
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
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // max (scaled, base 2) and this thread's part of the sum
  float o[VB * 8][4];
#pragma unroll
  for (int i = 0; i < VB * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const int nb0 = (plen + 15) / 16, nb = nb0 + (own1 - own0 + 15) / 16;
  for (int b = warp; b < nb; b += NW) {
    const bool own = b >= nb0;
    const int key0 = own ? own0 + (b - nb0) * 16 : b * 16, end = own ? own1 : plen;
    uint4 kf[2][JB], vf[4][VB];
    const size_t at = (own ? co : po) + size_t(key0) * HD;
    const bf16* kp = static_cast<const bf16*>(own ? p.kc : p.kp) + at + c * 8;
    const bf16* vp = static_cast<const bf16*>(own ? p.vc : p.vp) + at + g * 8;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < JB; ++j)
        kf[t][j] = key0 + 8 * t + g < end ? ld_stream(kp + size_t(8 * t + g) * HD + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 2 * c + (r & 1) + (r >> 1) * 8;
#pragma unroll
      for (int v = 0; v < VB; ++v)
        vf[r][v] = key0 + k < end ? ld_stream(vp + size_t(k) * HD + 64 * v) : make_uint4(0, 0, 0, 0);
    }
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        mma_bf16(s[t], q0[j].x, q1[j].x, q0[j].y, q1[j].y, kf[t][j].x, kf[t][j].y);
        mma_bf16(s[t], q0[j].z, q1[j].z, q0[j].w, q1[j].w, kf[t][j].z, kf[t][j].w);
      }
    }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool in = key0 + 8 * t + 2 * c + e < end;
        s[t][e] = in ? s[t][e] * sl2 : -INFINITY;
        x0 = fmaxf(x0, s[t][e]);
        if (WIDE) {
          s[t][2 + e] = in ? s[t][2 + e] * sl2 : -INFINITY;
          x1 = fmaxf(x1, s[t][2 + e]);
        }
      }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      if (WIDE) x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    // the block's first key is inside the range: the new maxima are not -inf
    // (but for a key whose score is: then the row keeps exp(-inf - 0) = 0)
    if (__any_sync(0xffffffffu, x0 > m0 || (WIDE && x1 > m1))) {
      const float n0 = fmaxf(m0, x0), a0 = exp2_approx(m0 - (n0 == -INFINITY ? 0.f : n0));
      const float n1 = fmaxf(m1, x1), a1 = WIDE ? exp2_approx(m1 - (n1 == -INFINITY ? 0.f : n1)) : 1.f;
      m0 = n0;
      l0 *= a0;
      m1 = n1;
      l1 *= a1;
#pragma unroll
      for (int i = 0; i < VB * 8; ++i) {
        o[i][0] *= a0;
        o[i][1] *= a0;
        if (WIDE) {
          o[i][2] *= a1;
          o[i][3] *= a1;
        }
      }
    }
    const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
    uint32_t pa[2][2];  // [key half][row half]
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float e0 = exp2_approx(s[t][0] - r0), e1 = exp2_approx(s[t][1] - r0);
      l0 += e0 + e1;
      pa[t][0] = pack_bf16(e0, e1);
      pa[t][1] = 0;
      if (WIDE) {
        const float e2 = exp2_approx(s[t][2] - r1), e3 = exp2_approx(s[t][3] - r1);
        l1 += e2 + e3;
        pa[t][1] = pack_bf16(e2, e3);
      }
    }
#pragma unroll
    for (int v = 0; v < VB; ++v) {
      const uint32_t* k0 = reinterpret_cast<const uint32_t*>(&vf[0][v]);
      const uint32_t* k1 = reinterpret_cast<const uint32_t*>(&vf[1][v]);
      const uint32_t* k8 = reinterpret_cast<const uint32_t*>(&vf[2][v]);
      const uint32_t* k9 = reinterpret_cast<const uint32_t*>(&vf[3][v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t sel = i & 1 ? 0x7632u : 0x5410u;  // upper or lower halves of two words
        mma_bf16(o[v * 8 + i], pa[0][0], pa[0][1], pa[1][0], pa[1][1], __byte_perm(k0[i / 2], k1[i / 2], sel),
                 __byte_perm(k8[i / 2], k9[i / 2], sel));
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    if (WIDE) l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }
  if (c == 0) {
    *reinterpret_cast<float2*>(sml + (warp * R + g) * 2) = make_float2(m0 * kLn2, l0);
    if (WIDE) *reinterpret_cast<float2*>(sml + (warp * R + g + 8) * 2) = make_float2(m1 * kLn2, l1);
  }
#pragma unroll
  for (int v = 0; v < VB; ++v)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = 64 * v + 8 * (2 * c + e) + i;
        so[(warp * R + g) * HD + d] = o[v * 8 + i][e];
        if (WIDE) so[(warp * R + g + 8) * HD + d] = o[v * 8 + i][2 + e];
      }
  __syncthreads();
  if (!inline_prefix) pdl_wait();  // the prefix items' partial sums
  const bool last = p.so == 1;  // else a slot for the join
  const size_t nrow = size_t(p.G) * p.W * p.hq;
  for (int i = threadIdx.x; i < rows * (HD / 4); i += 32 * NW) {
    const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
    const size_t row = size_t(n) * p.hq + head0 + r;
    float mx = -INFINITY;
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sml[(w * R + r) * 2]);
    if (last && !inline_prefix)
      for (int s = 0; s < p.sp; ++s) mx = fmaxf(mx, __ldcg(p.part_ml + (s * nrow + row) * 2));
    float num[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
    auto add = [&](float m, float l, const float4& f) {
      const float w = expf(m - mx);
      den = fmaf(w, l, den);
      num[0] = fmaf(w, f.x, num[0]);
      num[1] = fmaf(w, f.y, num[1]);
      num[2] = fmaf(w, f.z, num[2]);
      num[3] = fmaf(w, f.w, num[3]);
    };
    for (int w = 0; w < NW; ++w) {
      const float m = sml[(w * R + r) * 2];
      if (m != -INFINITY) add(m, sml[(w * R + r) * 2 + 1], *reinterpret_cast<const float4*>(so + (w * R + r) * HD + d));
    }
    if (last && !inline_prefix)
      for (int s = 0; s < p.sp; ++s) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (s * nrow + row) * 2));
        if (ml.x != -INFINITY) add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(p.part_o + (s * nrow + row) * HD + d)));
      }
    if (last) {
      const float inv = den > 0.f ? 1.f / den : 0.f;
      *reinterpret_cast<uint2*>(static_cast<bf16*>(p.out) + row * HD + d) =
          make_uint2(pack_bf16(num[0] * inv, num[1] * inv), pack_bf16(num[2] * inv, num[3] * inv));
    } else {
      const size_t at = size_t(p.sp + split) * nrow + row;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mx, den);
      *reinterpret_cast<float4*>(p.part_o + at * HD + d) = make_float4(num[0], num[1], num[2], num[3]);
    }
  }
}

// ---------------------------------------------------------------------------
// Items on the tensor cores (bf16, head dim 64 or 128): tiles of 128 (token,
// head) rows by 128 keys, one item a CTA.
//   warp 0      TMA: K and V tiles (128 keys x 64 dims boxes, 128-byte
//               swizzle) into their rings;
//   warp 1      MMA issue: S = Q K^T into one of two tensor-memory tiles,
//               O += P V into one of two accumulators;
//   warps 2-5   softmax of the even key tiles, a row a thread; warps 6-9 of
//               the odd ones. The two streams have their own max, sum and O
//               and are joined at the end, so one stream's softmax runs under
//               the other's and under the MMAs.
// P goes through shared memory as bf16 (K-major A operand); V is read as it
// lies (N-major B operand). The max that the exponentials are taken against is
// replaced, and O rescaled in tensor memory, only when a row's max has grown by
// more than 2^8: until then P is at most 2^8, which costs no precision, as a
// later division by the sum takes the factor out.
// Keys from the end of the range on are masked by selection; their V rows are
// zeroed in shared memory, since 0 x NaN would not be 0.
// ---------------------------------------------------------------------------
constexpr int kSaTcRows = 128, kSaTcKeys = 128;
constexpr int kSaTcThreads = 320;
constexpr uint32_t kSaTcSub = 128 * 64 * 2;  // a 128 x 64 bf16 subtile

template <int HD>
struct SaTcCfg {
  static constexpr int kSubs = HD / 64;
  static constexpr int kStages = HD == 128 ? 2 : 4;
  static constexpr uint32_t kTile = kSubs * kSaTcSub;  // a K, V or Q tile
  static constexpr uint32_t kP = 2 * kSaTcSub;
  static constexpr uint32_t kOffK = kTile, kOffV = kOffK + kStages * kTile, kOffP = kOffV + kStages * kTile;
  static constexpr size_t kSmem = size_t(kOffP) + 2 * kP + 1024;
  static constexpr uint32_t kTmemCols = 512, kTmemO = 256;  // S tiles at 0 and 128
  static constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 >> 3) << 17) | (uint32_t(128 >> 4) << 24);
  // B of P V: N (dims) contiguous
  static constexpr uint32_t kIdescO =
      (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(HD >> 3) << 17) | (uint32_t(128 >> 4) << 24);
};

template <int HD>
__global__ void __launch_bounds__(kSaTcThreads, 1)
    sa_tc_kernel(const SaParams p, const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                 const __grid_constant__ CUtensorMap map_kc, const __grid_constant__ CUtensorMap map_vc) {
  using C = SaTcCfg<HD>;
  constexpr int S = C::kStages;
  constexpr uint64_t kBudget = 2000000000ull;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t kfull[S], kempty[S], vfull[S], vempty[S], qfull, s_full[2], s_free[2], p_full[2], pv_done[2], drain;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_sh;
  volatile int* abort = &abort_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  pdl_wait();
  pdl_launch();  // after the wait: sa_token_kernel counts on it
  const SaItem it = sa_item<HD, 2>(p, blockIdx.x, kSaTcRows, kSaTcKeys);
  const size_t nrow = size_t(p.G) * p.W * p.T * p.hq;
  if (it.j0 >= it.j1) {
    for (int r = threadIdx.x; r < it.rows; r += kSaTcThreads) {
      const SaRow x = sa_row(p, it, r);
      const size_t at = it.slot * nrow + (size_t(x.n) * p.T + x.t) * p.hq + x.head;
      *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(-INFINITY, 0.f);
    }
    return;
  }
  const int nt = (it.j1 - it.j0 + kSaTcKeys - 1) / kSaTcKeys;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(kfull + s, 1);
      mbar_init(kempty + s, 1);
      mbar_init(vfull + s, 1);
      mbar_init(vempty + s, 1);
    }
    mbar_init(&qfull, 8);
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_full + x, 1);
      mbar_init(s_free + x, 4);
      mbar_init(p_full + x, 4);
      mbar_init(pv_done + x, 1);
    }
    mbar_init(&drain, 1);
    *abort = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  int issued = 0;  // warp 0: tiles whose copies were issued

  if (warp == 0) {
    if (lane == 0) {
      const CUtensorMap* mk = it.own ? &map_kc : &map_kp;
      const CUtensorMap* mv = it.own ? &map_vc : &map_vp;
      for (int t = 0; t < nt && !*abort; ++t) {
        const int s = t % S, j = it.j0 + t * kSaTcKeys;
        const uint32_t par = uint32_t((t / S) & 1) ^ 1u;
        if (t >= S && !(mbar_wait(kempty + s, par, kBudget, abort) && mbar_wait(vempty + s, par, kBudget, abort))) {
          *abort = 1;
          break;
        }
        mbar_arrive_expect_tx(kfull + s, C::kTile);
#pragma unroll
        for (int b = 0; b < C::kSubs; ++b)
          tma_load_3d(base + C::kOffK + s * C::kTile + b * kSaTcSub, mk, b * 64, j, it.plane, kfull + s);
        mbar_arrive_expect_tx(vfull + s, C::kTile);
#pragma unroll
        for (int b = 0; b < C::kSubs; ++b)
          tma_load_3d(base + C::kOffV + s * C::kTile + b * kSaTcSub, mv, b * 64, j, it.plane, vfull + s);
        issued = t + 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = mbar_wait(&qfull, 0u, kBudget, abort);
      auto pv = [&](int u) {
        const int y = u & 1, s = u % S;
        if (!mbar_wait(vfull + s, uint32_t((u / S) & 1), kBudget, abort) ||
            !mbar_wait(p_full + y, uint32_t((u >> 1) & 1), kBudget, abort))
          return false;
        tc_fence_after();
        const uint32_t pa = base + C::kOffP + y * C::kP, vb = base + C::kOffV + s * C::kTile;
#pragma unroll
        for (int k = 0; k < kSaTcKeys / 16; ++k)
          tc_mma(tmem + C::kTmemO + y * HD, tc_smem_desc(pa + (k >> 2) * kSaTcSub + (k & 3) * 32),
                 tc_smem_desc_mn(vb + k * 2048, kSaTcSub), C::kIdescO, (u > 1 || k > 0) ? 1u : 0u);
        tc_commit(vempty + s);
        tc_commit(pv_done + y);
        return true;
      };
      for (int t = 0; ok && t < nt; ++t) {
        const int x = t & 1, s = t % S;
        ok = mbar_wait(kfull + s, uint32_t((t / S) & 1), kBudget, abort) &&
             (t < 2 || mbar_wait(s_free + x, uint32_t(((t >> 1) - 1) & 1), kBudget, abort));
        if (!ok) break;
        tc_fence_after();
        const uint32_t kb = base + C::kOffK + s * C::kTile;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          tc_mma(tmem + x * 128, tc_smem_desc(base + (k >> 2) * kSaTcSub + (k & 3) * 32),
                 tc_smem_desc(kb + (k >> 2) * kSaTcSub + (k & 3) * 32), C::kIdescS, k > 0 ? 1u : 0u);
        tc_commit(kempty + s);
        tc_commit(s_full + x);
        if (t > 0) ok = pv(t - 1);
      }
      if (ok) ok = pv(nt - 1);
      if (!ok) *abort = 1;
    }
  } else {
    // ---- softmax warps
    const int stid = int(threadIdx.x) - 64, x = stid >> 7;
    const int quarter = warp & 3, r = quarter * 32 + lane;
    for (int i = stid; i < kSaTcRows * (HD / 8); i += 256) {
      const int row = i / (HD / 8), c = i - row * (HD / 8);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < it.rows) {
        const SaRow w = sa_row(p, it, row);
        v = ld_vec(static_cast<const bf16*>(p.q) + ((size_t(w.n) * p.T + w.t) * p.hq + w.head) * HD + c * 8);
      }
      *reinterpret_cast<uint4*>(smem + (c >> 3) * kSaTcSub + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v;
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&qfull);
    const uint32_t trow = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t ts = trow + x * 128, to = trow + C::kTmemO + x * HD;
    unsigned char* pbuf = smem + C::kOffP + x * C::kP + r * 128;
    int lim = it.j1;  // keys [0, lim) are seen
    if (r < it.rows) lim = min(lim, sa_limit(p, it, sa_row(p, it, r)));
    const float sl2 = p.scale * kLog2e;
    float m = -INFINITY, l = 0.f;  // reference max (scaled, base 2), sum
    bool ok = true;
    for (int u = x; u < nt; u += 2) {
      const int k = u >> 1, j = it.j0 + u * kSaTcKeys;
      ok = mbar_wait(s_full + x, uint32_t(k & 1), kBudget, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      float sc[kSaTcKeys];
#pragma unroll
      for (int c = 0; c < kSaTcKeys; c += 32) tc_ld32(ts + c, reinterpret_cast<uint32_t*>(sc + c));
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free + x);
      if (__any_sync(0xffffffffu, j + kSaTcKeys > lim)) {
#pragma unroll
        for (int c = 0; c < kSaTcKeys; ++c) sc[c] = j + c < lim ? sc[c] : -INFINITY;
      }
      float mx[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
      for (int c = 4; c < kSaTcKeys; ++c) mx[c & 3] = fmaxf(mx[c & 3], sc[c]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
      const bool grow = top > m + 8.f;
      if (k > 0) {  // the stream's previous P V has read P and written O
        ok = mbar_wait(pv_done + x, uint32_t((k - 1) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, grow)) {
        const float a = grow ? exp2_approx(m - top) : 1.f;
        if (grow) m = top;
        l *= a;
        if (k > 0) {
#pragma unroll
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tc_ld32(to + c, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
            tc_st16(to + c, o);
            tc_st16(to + c + 16, o + 16);
          }
          tc_wait_st();
        }
      }
      const float ref = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kSaTcKeys; c += 8) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = exp2_approx(fmaf(sc[c + i], sl2, -ref));
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i & 3] += e[i];
        *reinterpret_cast<uint4*>(pbuf + (c >> 6) * kSaTcSub + ((((c & 63) >> 3) ^ (r & 7)) << 4)) =
            make_uint4(pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7]));
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (j + kSaTcKeys > it.j1) {  // the last tile: V rows behind the range
        const int s = u % S;
        ok = mbar_wait(vfull + s, uint32_t((u / S) & 1), kBudget, abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (j + r >= it.j1) {
#pragma unroll
          for (int b = 0; b < C::kSubs; ++b)
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(smem + C::kOffV + s * C::kTile + b * kSaTcSub + r * 128 + c * 16) =
                  make_uint4(0, 0, 0, 0);
        }
      }
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + x);
    }
    const int mine = (nt + 1 - x) >> 1;  // tiles of this stream
    if (ok && mine > 0) ok = mbar_wait(pv_done + x, uint32_t((mine - 1) & 1), kBudget, abort);
    if (!ok) *abort = 1;
    // statistics of the streams, each in its own P buffer (read for the last time)
    float2* ml_sh = reinterpret_cast<float2*>(smem + C::kOffP);
    ml_sh[x * (C::kP / 8) + r] = make_float2(mine > 0 ? m : -INFINITY, l);
    tc_fence_before();
    named_sync(1, 256);  // both streams' O and statistics
    tc_fence_after();
    const float2 a = ml_sh[r], b = ml_sh[C::kP / 8 + r];
    const float top = fmaxf(a.x, b.x), ref = top == -INFINITY ? 0.f : top;
    const float wa = exp2_approx(a.x - ref), wb = exp2_approx(b.x - ref);
    const bool write = r < it.rows;
    size_t at = 0;
    if (write) {
      const SaRow w = sa_row(p, it, r);
      at = it.slot * nrow + (size_t(w.n) * p.T + w.t) * p.hq + w.head;
      if (x == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(top * kLn2, a.y * wa + b.y * wb);
    }
    // stream x joins dims [x * HD / 2, (x + 1) * HD / 2)
#pragma unroll
    for (int c = x * (HD / 2); c < (x + 1) * (HD / 2); c += 16) {
      uint32_t o0[16], o1[16];
      tc_ld16(trow + C::kTmemO + c, o0);
      if (nt > 1) tc_ld16(trow + C::kTmemO + HD + c, o1);
      tc_wait_ld();
      if (write) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          float f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[i] = __uint_as_float(o0[e + i]) * wa;
            if (nt > 1) f[i] = fmaf(__uint_as_float(o1[e + i]), wb, f[i]);
          }
          *reinterpret_cast<float4*>(p.part_o + at * HD + c + e) = make_float4(f[0], f[1], f[2], f[3]);
        }
      }
    }
  }
  __syncwarp();
  // ---- teardown: copies and MMAs in flight land before the memory goes away
  if (warp == 0 && lane == 0) {
    int never = 0;
    for (int t = max(0, issued - S); t < issued; ++t) {
      mbar_wait(kfull + t % S, uint32_t((t / S) & 1), kBudget, &never);
      mbar_wait(vfull + t % S, uint32_t((t / S) & 1), kBudget, &never);
    }
  }
  if (warp == 1 && lane == 0) {
    int never = 0;
    tc_commit(&drain);
    mbar_wait(&drain, 0u, kBudget, &never);
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicOr(p.status ? p.status : &g_sa_status, kStatusTimeout);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
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
