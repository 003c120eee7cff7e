// C ABI of beam search and of attention over a shared prefix (declared in
// include/minitp_b200.h): host checks, launch plans and workspaces.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "beam.cuh"
#include "host_util.cuh"
#include "shared_attn.cuh"

#include <cudaTypedefs.h>

#include <mutex>

using namespace mtpb;

namespace mtpb {

cudaError_t host_allow_smem(const void* kern, size_t smem) noexcept {
  struct Entry {
    const void* kern;
    int dev;
    size_t smem;
  };
  static Entry known[64];
  static int n = 0;
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  int i = 0;
  while (i < n && (known[i].kern != kern || known[i].dev != dev)) ++i;
  if (i < n && known[i].smem >= smem) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
  if (e == cudaSuccess && i < 64) {  // (a full table asks again each time)
    known[i] = Entry{kern, dev, smem};
    n = std::max(n, i + 1);
  }
  return e;
}

}  // namespace mtpb

namespace {

int bad(const char* msg) { return host_fail(MTPB_ERR_INVALID, msg); }
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
size_t es_of(int dtype) { return dtype == MTPB_BF16 ? 2 : 4; }
bool dtype_ok(int dtype) { return dtype == MTPB_BF16 || dtype == MTPB_F32; }

// ------------------------------------------------------------------ selection
// Chunks of a row: a function of the sizes alone, so that every rank cuts its
// shard alike.
struct BeamPlan {
  int nchunk, chunk;
};

BeamPlan beam_plan(long long rows, int V) {
  BeamPlan b;
  // at most two CTAs for each of B200's 148 SMs, and no more than chunks of 8192
  // columns call for (equal ones, so of 4097 columns at least): a chunk's own
  // start and end cost more than a fuller last wave gives (512 fp32 rows of
  // 151937: one chunk a row 62.6 us, two 73.9, four 93.2)
  const long long want = std::max<long long>(1, 2 * 148 / rows);
  b.nchunk = int(std::min<long long>(want, (V + 8191) / 8192));
  b.chunk = (V + b.nchunk - 1) / b.nchunk;
  b.chunk = (b.chunk + 7) / 8 * 8;
  b.nchunk = (V + b.chunk - 1) / b.chunk;
  return b;
}

size_t beam_cand_bytes(long long rows, const BeamPlan& b, int k) { return size_t(rows) * b.nchunk * k * 8; }
size_t beam_block(long long rows, const BeamPlan& b, int k) {
  return (beam_cand_bytes(rows, b, k) + size_t(rows) * b.nchunk * sizeof(BeamStat) + 15) / 16 * 16;
}

constexpr int kBeamMaxRows = 65535;  // a grid axis

int beam_check(long long rows, long long V, int k) {
  if (rows < 1 || rows > kBeamMaxRows) return bad("beam selection: need 1 .. 65535 rows");
  if (V < 1 || V >= 1ll << 30) return bad("beam selection: empty vocabulary, or one of 2^30 or more");
  if (k < 1 || k > kBeamMaxK) return bad("beam selection: k must be in [1, 64]");
  return MTPB_OK;
}

int beam_rows(const void* logits, long long ld, int rows, int V, long long vstart, int V_plan, int k,
              const uint8_t* finished, void* block, int dtype, cudaStream_t st) {
  const BeamPlan b = beam_plan(rows, V_plan);
  BeamRowsParams p;
  p.logits = logits;
  p.ld = ld;
  p.V = V;
  p.k = k;
  p.vstart = vstart;
  p.nchunk = b.nchunk;
  p.chunk = b.chunk;
  p.finished = finished;
  p.cand = static_cast<uint64_t*>(block);
  p.stat = reinterpret_cast<BeamStat*>(static_cast<char*>(block) + beam_cand_bytes(rows, b, k));
  const dim3 grid(b.nchunk, rows);
  const dim3 threads(kBeamThreads + 32);
  return dtype == MTPB_BF16 ? host_launch(beam_rows_kernel<bf16>, grid, threads, kBeamRing, st, p)
                            : host_launch(beam_rows_kernel<float>, grid, threads, kBeamRing, st, p);
}

int beam_pick(const void* blocks, int parts, int G, int W, int V_plan, int kc, const float* scores,
              const uint8_t* finished, long long eos, int k, float* out_scores, int64_t* out_parents,
              int64_t* out_tokens, uint8_t* out_finished, cudaStream_t st) {
  const int rows = G * W;
  const BeamPlan b = beam_plan(rows, V_plan);
  const size_t block = beam_block(rows, b, kc);
  BeamPickParams p;
  p.cand = static_cast<const uint64_t*>(blocks);
  p.stat = reinterpret_cast<const BeamStat*>(static_cast<const char*>(blocks) + beam_cand_bytes(rows, b, kc));
  p.cand_part = block / 8;
  p.stat_part = block / sizeof(BeamStat);
  p.parts = parts;
  p.rows = rows;
  p.nchunk = b.nchunk;
  p.scores = scores;
  p.finished = finished;
  p.W = W;
  p.k = k;
  p.kc = kc;
  p.eos = eos;
  p.out_scores = out_scores;
  p.out_parents = reinterpret_cast<long long*>(out_parents);
  p.out_tokens = reinterpret_cast<long long*>(out_tokens);
  p.out_finished = out_finished;
  return host_launch(beam_pick_kernel, dim3(G), dim3(kBeamThreads), 0, st, p);
}

int pick_check(int G, int W, const float* scores, const uint8_t* finished, long long eos, const float* out_scores,
               const int64_t* out_parents, const int64_t* out_tokens) {
  if (G < 1 || W < 1 || W > kBeamMaxW || (long long)G * W > kBeamMaxRows)
    return bad("beam selection: need 1 .. 64 beams and at most 65535 rows");
  if (!scores || !out_scores || !out_parents || !out_tokens) return bad("beam selection: null tensor");
  if (finished && eos < 0) return bad("beam selection: finished beams need an end token");
  if (eos > 0xFFFFFFFFll) return bad("beam selection: end token out of range");
  return MTPB_OK;
}

}  // namespace

extern "C" {

long long mtpb_beam_block_bytes(int rows, int V_plan, int k) {
  const int r = beam_check(rows, V_plan, k);
  if (r != MTPB_OK) return r;
  return (long long)beam_block(rows, beam_plan(rows, V_plan), k);
}

int mtpb_beam_candidates(const void* logits, int64_t ld, int rows, int V_local, int64_t vstart, int V_plan, int k,
                         const uint8_t* finished, void* block, int dtype, void* stream) {
  const int r = beam_check(rows, V_plan, k);
  if (r != MTPB_OK) return r;
  if ((!logits && V_local > 0) || !block) return bad("beam_candidates: null tensor");
  if (!dtype_ok(dtype)) return bad("unsupported dtype");
  if (V_local < 0 || V_local > V_plan || ld < V_local) return bad("beam_candidates: need 0 <= V_local <= V_plan, ld");
  if (vstart < 0 || vstart > 0xFFFFFFFFll - V_local) return bad("beam_candidates: vocabulary ids out of range");
  if (!al16(block)) return bad("beam_candidates: block must be 16-byte aligned");
  return beam_rows(logits, ld, rows, V_local, vstart, V_plan, k, finished, block, dtype,
                   static_cast<cudaStream_t>(stream));
}

int mtpb_beam_pick(const void* blocks, int parts, int G, int W, int V_plan, int k_block, const float* scores,
                   const uint8_t* finished, int64_t eos, int k, float* out_scores, int64_t* out_parents,
                   int64_t* out_tokens, uint8_t* out_finished, void* stream) {
  int r = pick_check(G, W, scores, finished, eos, out_scores, out_parents, out_tokens);
  if (r != MTPB_OK) return r;
  r = beam_check((long long)G * W, V_plan, k_block);
  if (r != MTPB_OK) return r;
  if (!blocks || !al16(blocks)) return bad("beam_pick: blocks must be 16-byte aligned");
  if (parts < 1 || parts > 64) return bad("beam_pick: need 1 .. 64 shards");
  if (k < 1 || k > k_block) return bad("beam_pick: k must be in [1, the blocks' k]");
  return beam_pick(blocks, parts, G, W, V_plan, k_block, scores, finished, eos, k, out_scores, out_parents,
                   out_tokens, out_finished, static_cast<cudaStream_t>(stream));
}

int mtpb_beam_select(const void* logits, int64_t ld, int G, int W, int V, const float* scores,
                     const uint8_t* finished, int64_t eos, int k, float* out_scores, int64_t* out_parents,
                     int64_t* out_tokens, uint8_t* out_finished, void* block, int dtype, void* stream) {
  int r = pick_check(G, W, scores, finished, eos, out_scores, out_parents, out_tokens);
  if (r != MTPB_OK) return r;
  r = mtpb_beam_candidates(logits, ld, G * W, V, 0, V, k, finished, block, dtype, stream);
  if (r != MTPB_OK) return r;
  return beam_pick(block, 1, G, W, V, k, scores, finished, eos, k, out_scores, out_parents, out_tokens, out_finished,
                   static_cast<cudaStream_t>(stream));
}

// Whether two of the caches (n of `bytes` each) share memory; < 0: no memory to tell.
static int caches_overlap(void* const* k, void* const* v, int n, size_t bytes) {
  auto* at = static_cast<uintptr_t*>(std::malloc(2 * size_t(n) * sizeof(uintptr_t)));
  if (!at) return -1;
  for (int l = 0; l < n; ++l) {
    at[2 * l] = reinterpret_cast<uintptr_t>(k[l]);
    at[2 * l + 1] = reinterpret_cast<uintptr_t>(v[l]);
  }
  std::sort(at, at + 2 * size_t(n));
  int found = 0;
  for (size_t i = 1; i < 2 * size_t(n); ++i) found |= at[i] - at[i - 1] < bytes;
  std::free(at);
  return found;
}

int mtpb_kv_reorder(void* const* k_caches, void* const* v_caches, int n_layers, const int64_t* parents,
                    const int* lens, int len, int G, int W, int hkv, int cap, int hd, int dtype, void* stream) {
  if (!k_caches || !v_caches || !parents) return bad("kv_reorder: null tensor");
  if (!dtype_ok(dtype)) return bad("unsupported dtype");
  if (n_layers < 1 || G < 1 || W < 1 || W > kBeamMaxW || hkv < 1 || cap < 1 || hd < 1)
    return bad("kv_reorder: sizes must be positive, with at most 64 rows a group");
  if ((long long)G * hkv > 65535) return bad("kv_reorder: groups x heads exceed 65535");
  if (!lens && (len < 0 || len > cap)) return bad("kv_reorder: length outside the cache");
  const size_t bytes = size_t(hd) * es_of(dtype);
  if (bytes % 16) return bad("kv_reorder: head_dim x element size must be a multiple of 16 bytes");
  for (int l = 0; l < n_layers; ++l)
    if (!k_caches[l] || !v_caches[l] || !al16(k_caches[l]) || !al16(v_caches[l]))
      return bad("kv_reorder: caches must be 16-byte aligned");
  const bool wide = W > 32;  // 8-byte columns keep 64 rows in registers
  const long long rv = bytes / (wide ? 8 : 16);
  const long long top = lens ? cap : len;
  if (W == 1 || top == 0) return MTPB_OK;
  const long long blocks = (top * rv + kReorderThreads - 1) / kReorderThreads;
  if (blocks > 0x7FFFFFFFll) return bad("kv_reorder: cache too long");
  // (one launch works on all of them at once)
  const int shared = caches_overlap(k_caches, v_caches, n_layers, size_t(G) * W * hkv * cap * bytes);
  if (shared) return bad(shared < 0 ? "kv_reorder: out of memory" : "kv_reorder: caches overlap");
  for (int l0 = 0; l0 < n_layers; l0 += kReorderLayers) {
    const int n = std::min(kReorderLayers, n_layers - l0);
    ReorderParams p;
    std::memset(&p, 0, sizeof(p));
    for (int l = 0; l < n; ++l) {
      p.k[l] = k_caches[l0 + l];
      p.v[l] = v_caches[l0 + l];
    }
    p.parents = reinterpret_cast<const long long*>(parents);
    p.lens = lens;
    p.len = len;
    p.G = G;
    p.W = W;
    p.hkv = hkv;
    p.cap = cap;
    p.rv = int(rv);
    const dim3 grid((unsigned)blocks, G * hkv, 2 * n), block(kReorderThreads);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int r = wide      ? host_launch(reorder_kernel<uint2, 64>, grid, block, 0, st, p)
                  : W <= 4  ? host_launch(reorder_kernel<uint4, 4>, grid, block, 0, st, p)
                  : W <= 8  ? host_launch(reorder_kernel<uint4, 8>, grid, block, 0, st, p)
                  : W <= 16 ? host_launch(reorder_kernel<uint4, 16>, grid, block, 0, st, p)
                            : host_launch(reorder_kernel<uint4, 32>, grid, block, 0, st, p);
    if (r != MTPB_OK) return r;
  }
  return MTPB_OK;
}

}  // extern "C"

// ------------------------------------------------------------------ attention over a shared prefix
namespace {

struct SaPlan {
  bool token;       // one token a row on sa_token_kernel
  bool inline_pre;  // it reads the prefix too: no other launch
  bool tc;          // the other items on sa_tc_kernel, else on the CUDA cores
  int mt;           // its row tiles a CTA
  int prpt, orpt;  // CUDA-core items: rows a tile / 16, of prefix and of own items
  int sp, so, ptiles, otiles;
  int pblocks, oblocks;
  long long pitems, items;
  size_t rows, ml_bytes, o_bytes;
};

// Key ranges for `base` tensor-core items of up to `top` keys: the number that
// makes waves x (key tiles a range + a start-up of four) smallest, with the
// partial sums' traffic (written and read again) beside it. The 0.7 us a tile are
// a fit to whole calls, below a tile's own pace (1.8 us for 256 rows of head dim
// 128, 1.5 of 64, half of that for 128 rows): with the pace in its place 4 x 4
// rows of 16 tokens behind 2048 take 38.2 us and not 31.9, 8 rows of 64 tokens
// behind 10000 41.8 and not 35.3, and eight other shapes the same.
int sa_tc_splits(long long base, int top, int limit, size_t rows, int hd, int sms) {
  const int tiles = std::max(1, (top + kSaTcKeys - 1) / kSaTcKeys);
  int best = 1;
  double least = 0;
  for (int s = 1; s <= std::min(tiles, limit); ++s) {
    const double waves = double((base * s + sms - 1) / sms);
    const double us = waves * (0.7 * ((tiles + s - 1) / s) + 2.8) + double(rows) * s * hd * 8 / 4e6;
    if (s == 1 || us < least) {
      best = s;
      least = us;
    }
  }
  return best;
}

int sa_plan(const SharedAttnArgs& a, SaPlan* out) {
  if (a.G < 1 || a.W < 1 || a.T < 1 || a.hq < 1 || a.hkv < 1 || a.cap_p < 1 || a.cap < 1)
    return bad("shared_attention: sizes must be positive");
  if (a.cap_p > 1 << 30 || a.cap > 1 << 30) return bad("shared_attention: caches of more than 2^30 positions");
  if (a.hq % a.hkv) return bad("shared_attention: hq must be a multiple of hkv");
  if (a.hd != 16 && a.hd != 32 && a.hd != 64 && a.hd != 128)
    return bad("shared_attention: head_dim must be 16, 32, 64 or 128");
  if (!dtype_ok(a.dtype)) return bad("unsupported dtype");
  const double rows = double(a.G) * a.W * a.T * a.hq;
  if (rows > double(1 << 28)) return bad("shared_attention: more than 2^28 (token, head) rows");
  SaPlan pl = {};
  pl.rows = size_t(rows);
  const int per = a.hq / a.hkv;
  const int top_p = a.prefix_lens ? a.cap_p : a.prefix_len, top_o = a.cache_lens ? a.cap : a.cache_len;
  const long long N = (long long)a.G * a.W;
  const int sms = host_sms();
  pl.tc = a.dtype == MTPB_BF16 && (a.hd == 64 || a.hd == 128);
  pl.token = pl.tc && a.T == 1 && N <= 65535;
  const long long prow = (long long)a.W * a.T * per, orow = (long long)a.T * per;
  // CUDA-core items: row tiles of 128, 64 or 16 by the rows there are (a larger
  // tile reads less shared memory a product, which bounds these items; fp32, 64
  // rows of the 7B heads behind 16384: 617 us, in tiles of 64 at most 703; but
  // 28 rows in one tile of 64 take 22 us where two of 16 take 12)
  auto rpt = [](long long rows_) { return rows_ > 96 ? 8 : rows_ > 32 ? 4 : 1; };
  pl.prpt = rpt(prow);
  pl.orpt = rpt(orow);
  // two row tiles a CTA from the second on (for most items)
  pl.mt = prow > 128 ? 2 : 1;
  const int ptile = pl.tc ? 128 * pl.mt : 16 * pl.prpt, otile = pl.token ? 16 : pl.tc ? 128 * pl.mt : 16 * pl.orpt;
  pl.ptiles = int((prow + ptile - 1) / ptile);
  pl.otiles = int((orow + otile - 1) / otile);
  const long long pbase = (long long)a.G * a.hkv * pl.ptiles, obase = N * a.hkv * pl.otiles;
  // key ranges until the items give every SM four, but none below two key tiles
  auto splits = [&](long long base, int top, int limit) {
    const long long most = std::max(1, (top + 2 * kSaKT - 1) / (2 * kSaKT)), want = 4ll * sms;
    return int(std::max<long long>(1, std::min<long long>(std::min<long long>(most, limit), (want + base - 1) / base)));
  };
  if (pl.token) {
    // long own caches of few rows in ranges of at least 512 keys (about 5 us of
    // one CTA's pace), which a third launch joins
    pl.so = 1;
    while (obase * pl.so * 2 <= 2 * sms && top_o / (pl.so * 2) >= 512 && pl.so < kSaMaxOwn) pl.so *= 2;
    // the prefix read by every row's CTA: one launch, but N / G reads of each
    // position, through L2, and one CTA's pace along it. 4 beams behind 128
    // positions: 3.4 us against 7 with the tensor-core items; 8 x 8 beams
    // behind 1024: 30 us against 21.
    const long long pre = (long long)top_p * a.hd * 4;
    pl.inline_pre = pl.so == 1 && pre <= (256 << 10) && obase * pre <= (32ll << 20);
  } else {
    pl.so = pl.tc ? sa_tc_splits(obase, top_o, kSaMaxOwn, pl.rows, a.hd, sms) : splits(obase, top_o, kSaMaxOwn);
  }
  pl.sp = pl.inline_pre ? 0
          : pl.tc       ? sa_tc_splits(pbase, top_p, kSaMaxSplits, pl.rows, a.hd, sms)
                        : splits(pbase, top_p, kSaMaxSplits);
  pl.pitems = pbase * pl.sp;
  pl.items = pl.pitems + (pl.token ? 0 : obase * pl.so);
  if (pl.items > 0x7FFFFFFFll) return bad("shared_attention: too many rows");
  pl.pblocks = int((prow + 31) / 32);
  pl.oblocks = int((orow + 31) / 32);
  const size_t blocks = size_t(pl.sp) * a.G * a.hkv * pl.pblocks +
                        size_t(pl.token && pl.so == 1 ? 0 : pl.so) * N * a.hkv * pl.oblocks;
  pl.ml_bytes = blocks * 32 * 8;
  pl.o_bytes = blocks * 32 * a.hd * 4;
  if (N * a.hkv * pl.oblocks > 0x7FFFFFFFll) return bad("shared_attention: too many rows");
  *out = pl;
  return MTPB_OK;
}

// The call with lengths that are known on the device only: planned by the capacities.
SharedAttnArgs by_capacity(SharedAttnArgs a) {
  static const int any = 0;
  a.prefix_lens = a.cache_lens = &any;
  return a;
}

// Map of caches [planes][cap][hd] bf16, boxes of 128 positions x 64 dims with
// the 128-byte swizzle; positions from cap on read as zeros.
int sa_map(CUtensorMap* map, const void* ptr, long long planes, int cap, int hd) {
  const auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(host_tensor_map_encoder());
  if (!enc) return host_fail(MTPB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  if (planes > 0x7FFFFFFFll) return bad("shared_attention: too many rows");
  const cuuint64_t dims[3] = {cuuint64_t(hd), cuuint64_t(cap), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(hd) * 2, cuuint64_t(cap) * hd * 2};
  const cuuint32_t box[3] = {64, kSaTcKeys, 1}, one[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MTPB_OK : host_fail(MTPB_ERR_CUDA, "cuTensorMapEncodeTiled failed");
}

template <int HD>
int sa_launch_tc(const SaPlan& pl, const SaParams& p, cudaStream_t st) {
  CUtensorMap m[4];
  const long long N = (long long)p.G * p.W;
  int r = sa_map(m, p.kp, (long long)p.G * p.hkv, p.cap_p, HD);
  if (r == MTPB_OK) r = sa_map(m + 1, p.vp, (long long)p.G * p.hkv, p.cap_p, HD);
  if (r == MTPB_OK) r = sa_map(m + 2, p.kc, N * p.hkv, p.cap, HD);
  if (r == MTPB_OK) r = sa_map(m + 3, p.vc, N * p.hkv, p.cap, HD);
  if (r != MTPB_OK) return r;
  const dim3 grid((unsigned)pl.items), block(kSaTcThreads);
  return pl.mt == 2 ? host_launch(sa_tc_kernel<HD, 2>, grid, block, SaTcCfg<HD, 2>::kSmem, st, p, m[0], m[1], m[2], m[3])
                    : host_launch(sa_tc_kernel<HD, 1>, grid, block, SaTcCfg<HD, 1>::kSmem, st, p, m[0], m[1], m[2], m[3]);
}

template <int HD>
int sa_launch_token(const SaPlan& pl, const SaParams& p, cudaStream_t st) {
  const dim3 grid(unsigned(p.hkv * pl.otiles), unsigned(p.G * p.W), unsigned(pl.so)), block(32 * kSaTokenWarps);
  const int inl = pl.inline_pre;
  return p.hq / p.hkv > 8 ? host_launch(sa_token_kernel<HD, true>, grid, block, sa_token_smem<HD, true>(), st, p, inl)
                          : host_launch(sa_token_kernel<HD, false>, grid, block, sa_token_smem<HD, false>(), st, p, inl);
}

template <typename T, int HD>
int sa_launch(const SaPlan& pl, const SaParams& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 2 && HD >= 64) {
    if (pl.items > 0) {
      const int r = sa_launch_tc<HD>(pl, p, st);
      if (r != MTPB_OK) return r;
    }
    if (pl.token) {
      const int r = sa_launch_token<HD>(pl, p, st);
      if (r != MTPB_OK || pl.so == 1) return r;
    }
  } else {
    auto items = [&](int rpt, long long first, long long n) {
      SaParams q = p;
      q.item0 = int(first);
      const dim3 grid((unsigned)n), block(kSaThreads);
      return rpt == 8   ? host_launch(sa_simt_kernel<T, HD, 8>, grid, block, sa_simt_smem<HD, 8>(), st, q)
             : rpt == 4 ? host_launch(sa_simt_kernel<T, HD, 4>, grid, block, sa_simt_smem<HD, 4>(), st, q)
                        : host_launch(sa_simt_kernel<T, HD, 1>, grid, block, sa_simt_smem<HD, 1>(), st, q);
    };
    const bool both = pl.prpt == pl.orpt;
    int r = items(pl.prpt, 0, both ? pl.items : pl.pitems);
    if (r == MTPB_OK && !both) r = items(pl.orpt, pl.pitems, pl.items - pl.pitems);
    if (r != MTPB_OK) return r;
  }
  return host_launch(sa_join_kernel<T, HD>, dim3(unsigned(p.G * p.W * p.hkv * pl.oblocks)), dim3(kSaJoinThreads),
                     size_t(p.sp + p.so) * 32 * sizeof(float2), st, p);
}

template <typename T>
int sa_launch_hd(const SaPlan& pl, const SaParams& p, int hd, cudaStream_t st) {
  switch (hd) {
    case 16: return sa_launch<T, 16>(pl, p, st);
    case 32: return sa_launch<T, 32>(pl, p, st);
    case 64: return sa_launch<T, 64>(pl, p, st);
    default: return sa_launch<T, 128>(pl, p, st);
  }
}

}  // namespace

namespace mtpb {

long long shared_attn_workspace(const SharedAttnArgs& a) {
  SaPlan pl;
  const int r = sa_plan(by_capacity(a), &pl);
  return r == MTPB_OK ? (long long)(pl.ml_bytes + pl.o_bytes) : r;
}

int shared_attn_run(const SharedAttnArgs& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  SaPlan pl;
  int r = sa_plan(a, &pl);
  // fewer keys than the capacity can call for more ranges, and more partial
  // sums, than the workspace was made for: then the capacities' plan
  if (r == MTPB_OK && pl.ml_bytes + pl.o_bytes > ws_bytes) r = sa_plan(by_capacity(a), &pl);
  if (r != MTPB_OK) return r;
  if (!a.q || !a.k_prefix || !a.v_prefix || !a.k_cache || !a.v_cache || !a.out ||
      (!ws && pl.ml_bytes + pl.o_bytes > 0))
    return bad("shared_attention: null tensor");
  if (!al16(a.q) || !al16(a.k_prefix) || !al16(a.v_prefix) || !al16(a.k_cache) || !al16(a.v_cache) || !al16(a.out) ||
      !al16(ws))
    return bad("shared_attention: tensors must be 16-byte aligned");
  if (!a.prefix_lens && (a.prefix_len < 0 || a.prefix_len > a.cap_p))
    return bad("shared_attention: prefix length outside the prefix cache");
  if (!a.cache_lens && (a.cache_len < 0 || a.cache_len > a.cap))
    return bad("shared_attention: length outside the cache");
  if (ws_bytes < pl.ml_bytes + pl.o_bytes) return bad("shared_attention: workspace too small");
  SaParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = a.q;
  p.kp = a.k_prefix;
  p.vp = a.v_prefix;
  p.plen = a.prefix_lens;
  p.plen_all = a.prefix_len;
  p.kc = a.k_cache;
  p.vc = a.v_cache;
  p.clen = a.cache_lens;
  p.clen_stride = a.cache_stride;
  p.clen_add = a.cache_len;
  p.out = a.out;
  p.G = a.G;
  p.W = a.W;
  p.T = a.T;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.cap_p = a.cap_p;
  p.cap = a.cap;
  p.scale = 1.0f / std::sqrt(float(a.hd));
  p.sp = pl.sp;
  p.so = pl.so;
  p.ptiles = pl.ptiles;
  p.otiles = pl.otiles;
  p.pitems = int(pl.pitems);
  p.items = int(pl.items);
  p.pblocks = pl.pblocks;
  p.oblocks = pl.oblocks;
  p.part_ml = static_cast<float2*>(ws);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + pl.ml_bytes);
  p.status = a.status;
  return a.dtype == MTPB_BF16 ? sa_launch_hd<bf16>(pl, p, a.hd, st) : sa_launch_hd<float>(pl, p, a.hd, st);
}

}  // namespace mtpb

extern "C" {

long long mtpb_shared_attention_workspace(int G, int W, int T, int hq, int hkv, int hd, int cap_p, int cap,
                                          int dtype) {
  SharedAttnArgs a = {};
  a.G = G;
  a.W = W;
  a.T = T;
  a.hq = hq;
  a.hkv = hkv;
  a.hd = hd;
  a.cap_p = cap_p;
  a.cap = cap;
  a.dtype = dtype;
  return shared_attn_workspace(a);
}

int mtpb_shared_attention(const void* q, const void* k_prefix, const void* v_prefix, const int* prefix_lens,
                          int prefix_len, const void* k_cache, const void* v_cache, const int* cache_lens,
                          int cache_len, void* out, int G, int W, int T, int hq, int hkv, int hd, int cap_p, int cap,
                          int dtype, void* ws, uint64_t ws_bytes, void* stream) {
  SharedAttnArgs a;
  a.q = q;
  a.k_prefix = k_prefix;
  a.v_prefix = v_prefix;
  a.prefix_lens = prefix_lens;
  a.prefix_len = prefix_len;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.cache_lens = cache_lens;
  a.cache_len = cache_lens ? 0 : cache_len;
  a.out = out;
  a.G = G;
  a.W = W;
  a.T = T;
  a.hq = hq;
  a.hkv = hkv;
  a.hd = hd;
  a.cap_p = cap_p;
  a.cap = cap;
  a.dtype = dtype;
  return shared_attn_run(a, ws, size_t(ws_bytes), static_cast<cudaStream_t>(stream));
}

}  // extern "C"

extern "C" int mtpb_beam_status(uint32_t* status_out) {
  if (!status_out) return bad("beam_status: null argument");
  uint32_t a = 0, b = 0;
  const uint32_t zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&a, g_sa_status, sizeof(a));
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&b, g_beam_status, sizeof(b));
  if (e == cudaSuccess && a) e = cudaMemcpyToSymbol(g_sa_status, &zero, sizeof(zero));
  if (e == cudaSuccess && b) e = cudaMemcpyToSymbol(g_beam_status, &zero, sizeof(zero));
  if (e != cudaSuccess) return host_fail_cuda(e, "beam_status");
  *status_out = a | b;
  return MTPB_OK;
}
