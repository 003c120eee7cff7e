// C ABI of packed prompt attention and token log-probabilities (declared in
// include/minitp_b200.h): host checks, launch plans and workspaces.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "host_util.cuh"
#include "logprobs.cuh"
#include "prompt_attn.cuh"

#include <cudaTypedefs.h>

using namespace mtpb;

namespace {

int bad(const char* msg) { return host_fail(MTPB_ERR_INVALID, msg); }
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool dtype_ok(int dtype) { return dtype == MTPB_BF16 || dtype == MTPB_F32; }

// ------------------------------------------------------------------ log-probabilities
constexpr long long kLpMaxRows = 1ll << 24;

LpPlan lp_plan_of(long long rows, int V, int dtype) { return lp_plan(rows, V, dtype == MTPB_BF16 ? 2 : 4); }

size_t lp_stat_bytes(long long rows, const LpPlan& b) { return size_t(rows) * b.parts * sizeof(LpStat); }
size_t lp_block(long long rows, const LpPlan& b, int k) {
  return (lp_stat_bytes(rows, b) + size_t(rows) * b.parts * k * 8 + 15) / 16 * 16;
}

int lp_check(long long rows, long long V, int k) {
  if (rows < 1 || rows > kLpMaxRows) return bad("token_logprobs: need 1 .. 2^24 rows");
  if (V < 1 || V >= 1ll << 30) return bad("token_logprobs: empty vocabulary, or one of 2^30 or more");
  if (rows * V > 1ll << 40) return bad("token_logprobs: more than 2^40 logits");
  if (k < 0 || k > kLpMaxK) return bad("token_logprobs: the alternatives must be in [0, 64]");
  return MTPB_OK;
}

template <typename T, bool TOP>
int lp_rows(const LpRowsParams& p, cudaStream_t st) {
  // a warp a row where every row is one tile and a CTA would have several of them
  if (p.plan.tiles == 1 && p.plan.run > 1) {
    const int grid = std::min((p.rows + kLpWarps - 1) / kLpWarps, 3 * host_sms());
    return host_launch(lp_short_kernel<T, TOP>, dim3(unsigned(grid)), dim3(kLpThreads), 0, st, p);
  }
  const auto kern = lp_rows_kernel<T, TOP>;
  // (with the static part it passes the 48 KB that a kernel gets unasked)
  const cudaError_t e = host_allow_smem(reinterpret_cast<const void*>(kern), kLpRing<TOP>);
  if (e != cudaSuccess) return host_fail_cuda(e, "cudaFuncSetAttribute");
  const long long total = (long long)p.rows * p.plan.tiles;
  return host_launch(kern, dim3(unsigned((total + p.plan.run - 1) / p.plan.run)), dim3(kLpThreads + 32), kLpRing<TOP>, st, p);
}

int lp_join(const void* blocks, int shards, int rows, const LpPlan& b, int kc, const int64_t* targets, int k,
            float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids, cudaStream_t st) {
  const size_t block = lp_block(rows, b, kc);
  LpJoinParams p;
  std::memset(&p, 0, sizeof(p));
  p.stat = static_cast<const LpStat*>(blocks);
  p.cand = reinterpret_cast<const uint64_t*>(static_cast<const char*>(blocks) + lp_stat_bytes(rows, b));
  p.stat_shard = block / sizeof(LpStat);
  p.cand_shard = block / 8;
  p.plan = b;
  p.shards = shards;
  p.rows = rows;
  p.k = k;
  p.kc = kc;
  p.logprobs = targets ? logprobs : nullptr;
  p.entropy = entropy;
  p.top_logprobs = top_logprobs;
  p.top_ids = reinterpret_cast<long long*>(top_ids);
  return host_launch(lp_join_kernel, dim3((rows + kLpJoinWarps - 1) / kLpJoinWarps), dim3(32 * kLpJoinWarps),
                     size_t(k ? kLpJoinWarps : 0) * (kLpRanked * 8 + size_t(shards) * b.parts), st, p);
}

int join_check(const int64_t* targets, int k, const float* logprobs, const float* entropy, const float* top_logprobs,
               const int64_t* top_ids) {
  if (!entropy || (targets && !logprobs) || (k > 0 && (!top_logprobs || !top_ids)))
    return bad("token_logprobs: null tensor");
  return MTPB_OK;
}

}  // namespace

extern "C" {

long long mtpb_logprobs_block_bytes(int rows, int V_plan, int k, int dtype) {
  const int r = lp_check(rows, V_plan, k);
  if (r != MTPB_OK) return r;
  if (!dtype_ok(dtype)) return bad("unsupported dtype");
  return (long long)lp_block(rows, lp_plan_of(rows, V_plan, dtype), k);
}

int mtpb_logprobs_block(const void* logits, int64_t ld, int rows, int V_local, int64_t vstart, int V_plan,
                        const int64_t* targets, int k, void* block, int dtype, void* stream) {
  const int r = lp_check(rows, V_plan, k);
  if (r != MTPB_OK) return r;
  if ((!logits && V_local > 0) || !block) return bad("token_logprobs: null tensor");
  if (!dtype_ok(dtype)) return bad("unsupported dtype");
  if (V_local < 0 || V_local > V_plan || ld < V_local)
    return bad("token_logprobs: need 0 <= V_local <= V_plan, ld");
  if (vstart < 0 || vstart > 0xFFFFFFFFll - V_local) return bad("token_logprobs: vocabulary ids out of range");
  if (!al16(block)) return bad("token_logprobs: block must be 16-byte aligned");
  LpRowsParams p;
  std::memset(&p, 0, sizeof(p));
  p.plan = lp_plan_of(rows, V_plan, dtype);
  p.logits = logits;
  p.ld = ld;
  p.rows = rows;
  p.V = V_local;
  p.k = k;
  p.vstart = vstart;
  p.targets = reinterpret_cast<const long long*>(targets);
  p.stat = static_cast<LpStat*>(block);
  p.cand = reinterpret_cast<uint64_t*>(static_cast<char*>(block) + lp_stat_bytes(rows, p.plan));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MTPB_BF16 ? (k ? lp_rows<bf16, true>(p, st) : lp_rows<bf16, false>(p, st))
                            : (k ? lp_rows<float, true>(p, st) : lp_rows<float, false>(p, st));
}

int mtpb_logprobs_join(const void* blocks, int shards, int rows, int V_plan, int k_block, const int64_t* targets, int k,
                       float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids, int dtype, void* stream) {
  int r = lp_check(rows, V_plan, k_block);
  if (r == MTPB_OK) r = join_check(targets, k, logprobs, entropy, top_logprobs, top_ids);
  if (r != MTPB_OK) return r;
  if (!dtype_ok(dtype)) return bad("unsupported dtype");
  if (!blocks || !al16(blocks)) return bad("token_logprobs: blocks must be 16-byte aligned");
  if (shards < 1 || shards > 64) return bad("token_logprobs: need 1 .. 64 shards");
  if (k < 0 || k > k_block) return bad("token_logprobs: more alternatives than the blocks hold");
  return lp_join(blocks, shards, rows, lp_plan_of(rows, V_plan, dtype), k_block, targets, k, logprobs, entropy, top_logprobs,
                 top_ids, static_cast<cudaStream_t>(stream));
}

int mtpb_token_logprobs(const void* logits, int64_t ld, int rows, int V, const int64_t* targets, int k, float* logprobs,
                        float* entropy, float* top_logprobs, int64_t* top_ids, void* block, int dtype, void* stream) {
  int r = lp_check(rows, V, k);
  if (r == MTPB_OK) r = join_check(targets, k, logprobs, entropy, top_logprobs, top_ids);
  if (r == MTPB_OK) r = mtpb_logprobs_block(logits, ld, rows, V, 0, V, targets, k, block, dtype, stream);
  if (r != MTPB_OK) return r;
  return lp_join(block, 1, rows, lp_plan_of(rows, V, dtype), k, targets, k, logprobs, entropy, top_logprobs, top_ids,
                 static_cast<cudaStream_t>(stream));
}

}  // extern "C"

// ------------------------------------------------------------------ attention over packed prompts
namespace {

// Map of [tokens][heads][hd] bf16 with the given strides, boxes of 64 dims x
// `bh` heads x `bt` tokens with the 128-byte swizzle. The coordinates are (dim,
// head, token) for queries and (dim, token, head) for keys and values, whose
// boxes hold one head. Tokens from the last on read as zeros.
int pa_map(CUtensorMap* map, const void* ptr, int tokens, int heads, long long ts, long long hs, int hd, bool query, int bt,
           int bh) {
  const auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(host_tensor_map_encoder());
  if (!enc) return host_fail(MTPB_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const int h = query ? 1 : 2, t = 3 - h;  // the axes of heads and of tokens
  cuuint64_t dims[3] = {cuuint64_t(hd)}, strides[2];
  cuuint32_t box[3] = {64}, one[3] = {1, 1, 1};
  dims[h] = cuuint64_t(heads);
  dims[t] = cuuint64_t(tokens);
  strides[h - 1] = cuuint64_t(hs) * 2;
  strides[t - 1] = cuuint64_t(ts) * 2;
  box[h] = cuuint32_t(bh);
  box[t] = cuuint32_t(bt);
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MTPB_OK : host_fail(MTPB_ERR_CUDA, "cuTensorMapEncodeTiled failed");
}

template <int HD, int MT>
int pa_launch_tc(PaParams p, cudaStream_t st) {
  const long long items = pa_items(&p, 128 * MT);
  CUtensorMap mq, mk, mv;
  int r = pa_map(&mq, p.q, p.n, p.hq, p.q_ts, p.q_hs, HD, true, p.tt, p.gs);
  if (r == MTPB_OK) r = pa_map(&mk, p.k, p.total, p.hkv, p.k_ts, p.k_hs, HD, false, kPaTcKeys, 1);
  if (r == MTPB_OK) r = pa_map(&mv, p.v, p.total, p.hkv, p.v_ts, p.v_hs, HD, false, kPaTcKeys, 1);
  if (r != MTPB_OK) return r;
  const unsigned grid = unsigned(std::max<long long>(1, std::min<long long>(items, host_sms())));
  return host_launch(pa_tc_kernel<HD, MT>, dim3(grid), dim3(kPaTcThreads), PaTcCfg<HD, MT>::kSmem, st, p, mq, mk, mv);
}

template <typename T, int HD, int RPT>
int pa_launch_simt(PaParams p, cudaStream_t st) {
  const long long items = std::max<long long>(1, pa_items(&p, 16 * RPT));
  if (items > 0x7FFFFFFFll) return bad("prompt_attention: too many rows");
  return host_launch(pa_simt_kernel<T, HD, RPT>, dim3(unsigned(items)), dim3(kPaThreads), pa_simt_smem<HD, RPT>(), st, p);
}

template <typename T, int HD>
int pa_launch(PaParams p, cudaStream_t st) {
  const long long rows = (long long)p.n * p.hq;
  if constexpr (sizeof(T) == 2 && HD >= 64) {
    // Two row tiles an item as soon as there is one of those for every SM (us of one / two: one prompt of 512
    // tokens, 14 heads of 64: 12 / 15; of 1024, 7 heads of 128: 17 / 25; of 2048, 28 heads of 128: 45 / 42; 64 of
    // <= 509, 14 heads of 64: 59 / 44)
    return rows > 256ll * 148 ? pa_launch_tc<HD, 2>(p, st) : pa_launch_tc<HD, 1>(p, st);
  } else {
    // Rows a tile: 64; 32 while those leave SMs idle (head dims 16 and 32, whose CTAs do less: one of two places an
    // SM); 16 while 16 do. fp32 us of 16 / 32 / 64: 3 prompts of <= 300 tokens, 4 heads of 16: 11 / 12 / 15; one of 300,
    // 14 of 64: 27 / 25 / 31; 10 of <= 200, 7 of 128: 54 / 37 / 43; 5 of <= 701, 8 of 32: 79 / 38 / 43; one of 2300:
    // - / 149 / 136; one of 1300, 14 of 64: 261 / 164 / 140; 4 of <= 2048, 7 of 128: 888 / 556 / 332. 128 rows spill
    // registers at 128 dims (one of 7000, 7 heads: 2384 with 64, 2559 with 128).
    if (rows <= 16ll * 148) return pa_launch_simt<T, HD, 1>(p, st);
    return rows <= (HD <= 32 ? 128ll : 64ll) * 148 ? pa_launch_simt<T, HD, 2>(p, st) : pa_launch_simt<T, HD, 4>(p, st);
  }
}

template <typename T>
int pa_launch_hd(const PaParams& p, int hd, cudaStream_t st) {
  switch (hd) {
    case 16: return pa_launch<T, 16>(p, st);
    case 32: return pa_launch<T, 32>(p, st);
    case 64: return pa_launch<T, 64>(p, st);
    default: return pa_launch<T, 128>(p, st);
  }
}

}  // namespace

namespace mtpb {

int prompt_attn_check(const PromptAttnArgs& a) {
  if (a.n < 0 || a.total < 0 || a.S < 0 || a.hq < 1 || a.hkv < 1) return bad("prompt_attention: negative size");
  if (a.hq % a.hkv) return bad("prompt_attention: hq must be a multiple of hkv");
  if (a.hd != 16 && a.hd != 32 && a.hd != 64 && a.hd != 128)
    return bad("prompt_attention: head_dim must be 16, 32, 64 or 128");
  if (!dtype_ok(a.dtype)) return bad("unsupported dtype");
  if (a.first < 0 || (long long)a.first + a.n > a.total)
    return bad("prompt_attention: the queries' tokens lie outside the packed tokens");
  if ((long long)a.total * a.hq > 1 << 28) return bad("prompt_attention: more than 2^28 (token, head) rows");
  if (a.hq > 1 << 16) return bad("prompt_attention: more than 2^16 heads");
  if (a.S > 1 << 20) return bad("prompt_attention: more than 2^20 prompts");
  return MTPB_OK;
}

int prompt_attn_run(const PromptAttnArgs& a, cudaStream_t st) {
  const int fits = prompt_attn_check(a);
  if (fits != MTPB_OK) return fits;
  if (a.n == 0) return MTPB_OK;
  if (!a.q || !a.k || !a.v || !a.out || !a.seq_starts) return bad("prompt_attention: null tensor");
  const int es = a.dtype == MTPB_BF16 ? 2 : 4, ve = 16 / es;
  if (!al16(a.q) || !al16(a.k) || !al16(a.v) || (reinterpret_cast<uintptr_t>(a.out) & 31u))
    return bad("prompt_attention: tensors must be 16-byte aligned, out 32-byte aligned");
  const long long strides[6] = {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head};
  for (long long s : strides)
    if (s < a.hd || s % ve || s >= 1ll << 38)
      return bad("prompt_attention: strides must be multiples of 16 bytes and no smaller than head_dim");
  PaParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_ts = a.q_token;
  p.q_hs = a.q_head;
  p.k_ts = a.k_token;
  p.k_hs = a.k_head;
  p.v_ts = a.v_token;
  p.v_hs = a.v_head;
  p.out = a.out;
  p.starts = a.seq_starts;
  p.S = a.S;
  p.first = a.first;
  p.n = a.n;
  p.total = a.total;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.scale = 1.0f / std::sqrt(float(a.hd));
  p.status = a.status;
  return a.dtype == MTPB_BF16 ? pa_launch_hd<bf16>(p, a.hd, st) : pa_launch_hd<float>(p, a.hd, st);
}

}  // namespace mtpb

extern "C" int mtpb_prompt_attention(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                                     int64_t k_head, const void* v, int64_t v_token, int64_t v_head, void* out,
                                     const int* seq_starts, int S, int first, int n, int total, int hq, int hkv, int hd,
                                     int dtype, void* stream) {
  PromptAttnArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_token = q_token;
  a.q_head = q_head;
  a.k_token = k_token;
  a.k_head = k_head;
  a.v_token = v_token;
  a.v_head = v_head;
  a.out = out;
  a.seq_starts = seq_starts;
  a.S = S;
  a.first = first;
  a.n = n;
  a.total = total;
  a.hq = hq;
  a.hkv = hkv;
  a.hd = hd;
  a.dtype = dtype;
  return prompt_attn_run(a, static_cast<cudaStream_t>(stream));
}

extern "C" int mtpb_scoring_status(uint32_t* status_out) {
  if (!status_out) return bad("scoring_status: null argument");
  uint32_t a = 0, b = 0;
  const uint32_t zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&a, g_pa_status, sizeof(a));
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&b, g_lp_status, sizeof(b));
  if (e == cudaSuccess && a) e = cudaMemcpyToSymbol(g_pa_status, &zero, sizeof(zero));
  if (e == cudaSuccess && b) e = cudaMemcpyToSymbol(g_lp_status, &zero, sizeof(zero));
  if (e != cudaSuccess) return host_fail_cuda(e, "scoring_status");
  *status_out = a | b;
  return MTPB_OK;
}
