// Packed prompts and their tiles: the parameters of a prompt attention, and how a
// warp finds the tile of a number from the prompts' starts. No more than warp
// intrinsics, so that the tests can run it on the host.
#pragma once

#include <stdint.h>

namespace mtpb {

struct PaParams {
  const void *q, *k, *v;
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // elements from token to token, from head to head
  void* out;          // [n][hq][hd]
  const int* starts;  // device [S + 1]
  int S, first, n, total, hq, hkv;
  int gs, subs;  // heads of a row group, groups of a KV head: gs * subs = G
  int tt;        // tokens a tile: as many as its rows hold, gs rows each
  unsigned long long tt_mul;  // ceil(2^37 / tt): n / tt = n * tt_mul >> 37, exact for the n there can be (n * hq <= 2^28)
  uint32_t gs_mul;            // ceil(2^16 / gs), the same for rows of a tile
  int planes;    // hkv * subs
  float scale;
  uint32_t* status;  // error bits
};

__device__ __forceinline__ int pa_div_tt(const PaParams& p, int n) { return int((unsigned long long)n * p.tt_mul >> 37); }
__device__ __forceinline__ int pa_div_gs(const PaParams& p, int row) { return int(uint32_t(row) * p.gs_mul >> 16); }

// Row groups and tokens of tiles of `rows` rows, and the items that there can
// be at most: all heads of a KV head side by side, or as many of them as divide
// them and fit.
inline long long pa_items(PaParams* p, int rows) {
  const int G = p->hq / p->hkv;
  p->subs = 1;
  while (G % p->subs || G / p->subs > rows) ++p->subs;
  p->gs = G / p->subs;
  p->planes = p->hkv * p->subs;
  p->tt = rows / p->gs;
  p->tt_mul = ((1ull << 37) + p->tt - 1) / p->tt;
  p->gs_mul = (65536u + p->gs - 1) / p->gs;
  return ((long long)p->n / p->tt + p->S) * p->planes;
}

// A tile: row r is token tok0 + r / gs, head r % gs of the row group.
struct PaItem {
  int start;  // of the prompt (packed tokens)
  int tok0, ntok;  // ntok 0: no tile
  int plane;  // KV head and row group
};

// Prompts whose tiles are put in order (a lane has its share in registers).
constexpr int kPaOrdered = 2 * 32;

// The tiles of all prompts, by one warp, in the order of growing numbers. They
// are numbered in descending order of their place in their prompt, which is how
// many keys they see, over all prompts, so that the longest do not start last;
// with more than kPaOrdered prompts prompt after prompt (the last tile first; a
// long prompt that comes last then starts last).
// The starts are made non-decreasing and cut to [0, total] first, so that no
// values of theirs lead out of the tensors or make two tiles of a token.
struct PaTiles {
  struct Seq {
    int start, lo, n, nt, off;  // packed tokens from lo on, tiles, place of the first tile
  };
  int at_least;  // the largest start so far
  int gap0, gap1;  // tokens [first, gap0) and [gap1, first + n) are of no prompt (gap1: once all were read)
  int all;  // tiles: of all prompts, or (not ordered) of those before block b
  int b, most, ahead;  // ahead: ends of block b + 1, loaded
  Seq q[kPaOrdered / 32];

  static __device__ __forceinline__ int cut(const PaParams& p, int t) { return min(max(t, 0), p.total); }

  // the end of prompt 32 blk + lane (behind the last prompt: 0)
  static __device__ __forceinline__ int end_of(const PaParams& p, int blk) {
    const int s = 32 * blk + (threadIdx.x & 31);
    return s < p.S ? cut(p, __ldg(p.starts + s + 1)) : 0;
  }
  __device__ __forceinline__ Seq load(const PaParams& p, int its_end) {
    const int lane = threadIdx.x & 31, end = p.first + p.n;
    int hi = max(at_least, its_end);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, hi, o);
      if (lane >= o) hi = max(hi, u);
    }
    const int prev = __shfl_up_sync(0xffffffffu, hi, 1);
    Seq r;
    r.start = lane ? prev : at_least;
    r.lo = max(r.start, p.first);
    r.n = max(0, min(hi, end) - r.lo);
    r.nt = pa_div_tt(p, r.n + p.tt - 1);
    r.off = r.n ? pa_div_tt(p, r.lo - r.start) : 0;
    at_least = __shfl_sync(0xffffffffu, hi, 31);
    return r;
  }

  __device__ __forceinline__ void open(const PaParams& p) {
    int ends[kPaOrdered / 32];  // (all loads in flight at once)
#pragma unroll
    for (int i = 0; i < kPaOrdered / 32; ++i) ends[i] = end_of(p, i);
    at_least = cut(p, __ldg(p.starts));
    gap0 = min(max(at_least, p.first), p.first + p.n);
    all = b = most = 0;
    if (p.S > kPaOrdered) {
      gap1 = p.first + p.n;  // (not read yet)
      q[0] = load(p, ends[0]);
      ahead = ends[1];
      return;
    }
#pragma unroll
    for (int i = 0; i < kPaOrdered / 32; ++i) {
      q[i] = Seq{0, 0, 0, 0, 0};
      if (32 * i < p.S) q[i] = load(p, ends[i]);
      if (q[i].nt) most = max(most, q[i].off + q[i].nt);
      all += q[i].nt;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    all = __reduce_add_sync(0xffffffffu, all);
    gap1 = min(max(at_least, p.first), p.first + p.n);
  }

  __device__ __forceinline__ PaItem take(const PaParams& p, int from, const Seq& r, int tile) {
    PaItem it;
    it.start = __shfl_sync(0xffffffffu, r.start, from);
    it.tok0 = __shfl_sync(0xffffffffu, r.lo, from) + tile * p.tt;
    it.ntok = min(p.tt, __shfl_sync(0xffffffffu, r.n, from) - tile * p.tt);
    return it;
  }

  // Tile number i (no smaller than in the call before); ntok 0 when there is none. (Few instructions
  // count: what is fetched here pushes the softmax's out of the instruction cache.)
  __device__ __forceinline__ PaItem find(const PaParams& p, int i) {
    const int lane = threadIdx.x & 31;
    PaItem it{0, 0, 0, 0};
    if (p.S > kPaOrdered) {
      for (;; ++b) {
        int upto = q[0].nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += u;
        }
        const int sum = __shfl_sync(0xffffffffu, upto, 31);
        if (i < all + sum) {
          const int from = __popc(__ballot_sync(0xffffffffu, all + upto <= i));
          return take(p, from, q[0], all + __shfl_sync(0xffffffffu, upto, from) - 1 - i);
        }
        if (32 * (b + 1) >= p.S) break;
        all += sum;
        q[0] = load(p, ahead);
        ahead = end_of(p, b + 2);
      }
      gap1 = min(max(at_least, p.first), p.first + p.n);
      return it;
    }
    if (i >= all) return it;
    auto above = [&](int c) {  // tiles at place c or behind it
      int n = 0;
#pragma unroll
      for (int k = 0; k < kPaOrdered / 32; ++k) n += max(0, q[k].off + q[k].nt - max(c, q[k].off));
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
    for (int k = 0; k < kPaOrdered / 32; ++k) {
      const bool in = q[k].off <= lo && lo < q[k].off + q[k].nt;
      const uint32_t m = __ballot_sync(0xffffffffu, in);
      const int c = __popc(m);
      if (left >= 0 && left < c) {
        const int from = __ffs(__ballot_sync(0xffffffffu, in && __popc(m & ((1u << lane) - 1u)) == left)) - 1;
        it = take(p, from, q[k], lo - __shfl_sync(0xffffffffu, q[k].off, from));
      }
      left -= c;
    }
    return it;
  }

  // Tile number i by itself, for a grid of a CTA a tile; open() and find() are
  // not called. More prompts than are put in order are not walked through (S CTAs
  // would read S starts each): with c_s tokens of the queries before prompt s, its
  // numbers are c_s / tt + s up to c_(s+1) / tt + s. Those are at least as many as
  // it has tiles, the rest are no tiles, and all together as many as pa_items
  // plans. s comes from a search with 32 places a step. (fp32, 4 heads of 16, walked
  // through / searched: 1000 prompts of up to 20 tokens 82 / 38 us, 5000 of up to 12
  // 1103 / 146, 65536 of up to 5 150.8 / 1.8 ms; 200 17 / 17 us. Decreasing starts: places
  // outside the tensors are still cut off, but a token may have two tiles or none.)
  __device__ __forceinline__ PaItem only(const PaParams& p, int i) {
    if (p.S <= kPaOrdered) {
      open(p);
      return find(p, i);
    }
    const int lane = threadIdx.x & 31;
    auto start_of = [&](int s) { return cut(p, __ldg(p.starts + s)); };
    auto before = [&](int start) { return min(max(start - p.first, 0), p.n); };
    auto number = [&](int s) { return pa_div_tt(p, before(start_of(s))) + s; };
    gap0 = p.first + before(start_of(0));
    gap1 = p.first + before(start_of(p.S));
    int s = 0, hi = p.S;  // number(s) <= i < number(hi), or s = 0
    while (hi - s > 1) {
      const int step = (hi - s + 31) / 32, at = s + step * (lane + 1);
      s += step * __popc(__ballot_sync(0xffffffffu, at < hi && number(at) <= i));
      hi = min(hi, s + step);
    }
    const int start = start_of(s), c = before(start), n = before(start_of(s + 1)) - c;
    const int tiles = n > 0 ? pa_div_tt(p, n + p.tt - 1) : 0, tile = tiles - 1 - (i - pa_div_tt(p, c) - s);
    if (tile < 0 || tile >= tiles) return PaItem{0, 0, 0, 0};
    return PaItem{start, p.first + c + tile * p.tt, min(p.tt, n - tile * p.tt), 0};
  }
};

}  // namespace mtpb
