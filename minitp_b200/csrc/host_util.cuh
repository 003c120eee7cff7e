// Host helpers shared by the translation units of the C ABI: the per-thread
// error text, launch settings, and the operators one unit offers another.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "minitp_b200.h"

namespace mtpb {

// Records `msg` as the calling thread's error text and returns `code`.
int host_fail(int code, const char* msg) noexcept;
int host_fail_cuda(cudaError_t e, const char* what) noexcept;
// Whether later launches use programmatic dependent launch (mtpb_set_pdl).
bool host_pdl() noexcept;

// cuTensorMapEncodeTiled (a PFN_cuTensorMapEncodeTiled_v12000), or NULL.
void* host_tensor_map_encoder() noexcept;

// Lets `kern` use `smem` bytes of shared memory on the current device (asked
// of the driver once for each kernel, device and larger size).
cudaError_t host_allow_smem(const void* kern, size_t smem) noexcept;

// Multiprocessors of the current device (a constant of the device, asked once).
inline int host_sms() {
  static int per_dev[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (!per_dev[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    per_dev[dev] = n > 0 ? n : 148;
  }
  return per_dev[dev];
}

template <typename Kern, typename... Args>
int host_launch(Kern kern, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const Args&... args) {
  if (smem > 48 * 1024) {
    const cudaError_t e = host_allow_smem(reinterpret_cast<const void*>(kern), smem);
    if (e != cudaSuccess) return host_fail_cuda(e, "cudaFuncSetAttribute");
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = host_pdl() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e == cudaSuccess ? MTPB_OK : host_fail_cuda(e, "kernel launch");
}

// Attention over a shared prefix and each row's own cache (mtpb_shared_attention).
struct SharedAttnArgs {
  const void* q;                        // [N*T][hq*hd]
  const void *k_prefix, *v_prefix;      // [G][hkv][cap_p][hd]
  const int* prefix_lens;               // device [G], or NULL: prefix_len for all
  int prefix_len;
  const void *k_cache, *v_cache;        // [N][hkv][cap][hd]
  const int* cache_lens;                // device [N], or NULL
  int cache_stride = 1;                 // 0: every row reads cache_lens[0]
  int cache_len;                        // added to the device value (alone without one)
  void* out;                            // [N*T][hq*hd]
  int G, W, T, hq, hkv, hd, cap_p, cap; // N = G * W
  int dtype;
  uint32_t* status = nullptr;           // word for error bits, or NULL: the library's own
};
// Workspace bytes of calls of these sizes, whatever their lengths (no device
// access; < 0: an MTPB_ERR_* code).
long long shared_attn_workspace(const SharedAttnArgs& a);
int shared_attn_run(const SharedAttnArgs& a, void* ws, size_t ws_bytes, cudaStream_t st);

}  // namespace mtpb
