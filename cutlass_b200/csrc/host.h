// Host helpers shared by the translation units of the library (defined in bsgemm.cu, not exported).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <cstring>

namespace bsg {

#define BSG_HIDDEN __attribute__((visibility("hidden")))

// Records the text that bsg_last_error_string returns on this thread, and returns `code`.
BSG_HIDDEN int32_t host_fail(int32_t code, const char* fmt, ...);
// Tensor map of K-major byte matrices (batches x rows x row_bytes), box = 128 bytes x box_rows, 128-byte swizzle.
BSG_HIDDEN int32_t host_operand_map(CUtensorMap* map, const void* base, uint64_t row_bytes, uint64_t rows, uint64_t batches,
                                    uint64_t pitch_bytes, uint64_t batch_stride_bytes, uint32_t box_rows);
// Tensor map of a row-major bf16, fp16 or fp32 output matrix, box = 32 rows x 128 bytes, 128-byte swizzle.
BSG_HIDDEN int32_t host_out_map(CUtensorMap* map, const void* base, int32_t out_kind, uint64_t cols, uint64_t rows, uint64_t pitch_elems);

inline bool host_aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Current device and its SM count; refuses devices that are not sm_100.
BSG_HIDDEN int32_t host_device(int32_t not_sm100, int32_t cuda_error, int* dev, int* sms);

// Launch with programmatic stream serialisation: the kernel's CTAs are set up while what runs before on the stream ends, and wait
// for its end and its writes (griddepcontrol.wait) before they touch global memory.
template <class... P>
cudaError_t host_launch(void (*kernel)(P...), unsigned grid, unsigned threads, size_t shared, cudaStream_t s, const P&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace bsg
