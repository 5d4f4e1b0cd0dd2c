// Host services shared by the translation units of libmoonpoly_gemm.so; defined in mp_abi.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>

#include "../../include/moonpoly_abi.h"

namespace mp {

// Records the calling thread's error text (mp_last_error_string) and returns `code`.
int host_fail(int code, const char* fmt, ...);
void host_count_launches(int n);
bool host_use_pdl();             // MOONPOLY_DISABLE_PDL

// The current device: its SM count and the address of the status word that kernels report to (mp_device_status).
struct HostDevice { int index; int sms; int* status; };
int host_device(HostDevice* out);

// 2-D tensor map over `rows` lines of `inner` elements, `row_bytes` apart.  swizzle: 128, 64 or 0.
enum { kTmap16 = 0, kTmapByte = 1 };
int host_tmap(CUtensorMap* tm, int type, const void* ptr, long long inner, long long rows, long long row_bytes, int box_inner,
              int box_rows, int swizzle);
// The same matrix of 16-bit elements as [inner / 64][rows][64] (inner a multiple of 64): a box brings `box_blocks` blocks
// of 128 bytes, contiguous in memory, of every line; 128-byte swizzle.
int host_tmap_blocks(CUtensorMap* tm, const void* ptr, long long inner, long long rows, long long row_bytes, int box_rows, int box_blocks);

// dst[r][0 .. kp) = src[r][0 .. k) followed by zeros, 16-bit elements; kp a multiple of 8, dst 16-byte aligned.
int host_pad_rows16(const void* src, long long ld, void* dst, int rows, int k, int kp, cudaStream_t stream);

}  // namespace mp

#define MP_HOST_CUDA_TRY(expr)                                                                                        \
  do {                                                                                                                \
    cudaError_t e__ = (expr);                                                                                         \
    if (e__ != cudaSuccess)                                                                                           \
      return mp::host_fail(MP_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e__), __FILE__, __LINE__); \
  } while (0)

namespace mp {

// A launch that may begin while the previous kernel of the stream ends (programmatic dependent launch); its kernel waits
// (griddepcontrol.wait) before it touches memory.
template <typename... P, typename... A>
int host_launch(void (*kern)(P...), int grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = host_use_pdl() ? 1 : 0;
  MP_HOST_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, P(args)...));
  host_count_launches(1);
  return MP_OK;
}

}  // namespace mp
