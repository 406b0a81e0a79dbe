// Host-side helpers shared by the launchers: error reporting and TMA
// tensor-map encoding.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "../../include/bsa.h"

namespace bsa {

// Records a thread-local error message and returns `st`.
bsa_status fail(bsa_status st, const std::string &msg);

// Maps the last CUDA runtime error (if any) to BSA_ERR_LAUNCH.
bsa_status check_launch(const char *what);

// Launches `kern` so that it may start before the kernel in front of it on the stream
// has finished (programmatic dependent launch): it must call pdl_wait() before it
// touches anything that kernel writes or reads.
template <typename K, typename... A>
inline void launch_after(K kern, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, args...);
}

// Raises a kernel's dynamic shared-memory limit once per device (`done`: one bit each,
// a static of the call site).
inline void allow_smem(const void *kern, int bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess)
    done.fetch_or(bit, std::memory_order_relaxed);
}

inline size_t elem_size(int dtype) { return dtype == BSA_F32 ? 4 : 2; }

// Whether the elements of an operand that a kernel writes, (B, H, L) rows of D, lie apart:
// each stride steps over what the shorter ones span (an expanded axis does not).
bool lies_apart(int64_t B, int64_t sb, int64_t H, int64_t sh, int64_t L, int64_t sl, int64_t D);

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Encodes a 4-D tiled tensor map over a (B, H, L, D) view of 16-bit elements
// with a box of 64 columns x `rows` rows and 128-byte swizzle.  The three
// outer axes are ordered by increasing stride before encoding; `perm[i]` gives
// the encoded position (1..3) of axis i (0 = L, 1 = H, 2 = B).
struct TensorMap4 {
  CUtensorMap map;
  int perm[3];
};
bsa_status make_tmap(TensorMap4 *out, const void *ptr, int dtype, int B, int H, int L, int D,
                     int64_t sb, int64_t sh, int64_t sl, int rows, const char *name);

// Encodes a 3-D tiled tensor map over a contiguous fp32 (G, rows, dim) array
// with a box of 32 columns (128 bytes) x `box_rows` rows x 1 and 128-byte
// swizzle; rows past `rows` read as zero.  dim must be a multiple of 4.
bsa_status make_tmap_f32_rows(CUtensorMap *out, const float *ptr, int G, int rows, int dim,
                              int box_rows, const char *name);

}  // namespace bsa
