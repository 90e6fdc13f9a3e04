// Helpers shared by the token-generation kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../common.hpp"

namespace pfb {

// n / d for any 32-bit n below 2^31 and any d in [1, 2^31): with
// s = ceil(log2 d) and m = ceil(2^(31+s) / d), the error m*d - 2^(31+s) is
// below d <= 2^s, so (n * m) >> (31 + s) is exact for n < 2^31; m is below
// 2^32.
struct FastDiv {
  unsigned d = 1, m = 1u << 31, s = 0;
  FastDiv() = default;
  explicit FastDiv(unsigned div) : d(div) {
    while (s < 31 && (1u << s) < d) ++s;
    m = (unsigned)(((1ull << (31 + s)) + d - 1) / d);
  }
  __host__ __device__ __forceinline__ unsigned div(unsigned n) const {
    return (unsigned)(((unsigned long long)n * m) >> (31 + s));
  }
};

// These kernels follow one another within microseconds, so each is launched
// as a programmatic dependent: its CTAs come up as the kernel before it in the
// stream ends, and begin() waits until everything before it is finished and
// visible.  Nothing is read or written before that, and every thread passes
// it, so a kernel is done only when all before it are.  In a stream of calls
// this takes 1 to 3 us off each (one of 8191 tokens appended: 41.0 -> 38.0,
// 48 sequences attended: 144.8 -> 142.8).  A kernel does not let the next one
// come up before it ends: CTAs that wait take room from those that work (128
// sequences attended: 448 us for 425; 2047 tokens rotated: 5.8 for 4.3).
__device__ __forceinline__ void begin() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename A>
inline void launch_following(void (*kernel)(A), dim3 grid, int threads, size_t smem, cudaStream_t stream, const A& args,
                             int cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  PFB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
}

inline void check_decode_dtype(int dtype) {
  PFB_CHECK_ARG(dtype == PFC_DTYPE_FLOAT32 || dtype == PFC_DTYPE_FLOAT16 || dtype == PFC_DTYPE_BFLOAT16,
                "dtype must be float32, float16 or bfloat16");
}

inline void check_paged_cache(const pfk_paged_cache& c) {
  check_decode_dtype(c.dtype);
  PFB_CHECK_ARG(c.num_pages >= 1 && c.page_size >= 1 && c.heads >= 1 && c.head_dim >= 1,
                "paged cache: sizes must be positive");
  PFB_CHECK_ARG(c.num_pages <= INT32_MAX && c.page_size <= INT32_MAX && c.num_pages * c.page_size <= INT32_MAX,
                "paged cache: 2^31 tokens or more");
  PFB_CHECK_ARG(c.heads <= 65536, "paged cache: more than 65536 heads");
  PFB_CHECK_ARG(c.page_stride >= 0 && c.token_stride >= 0 && c.head_stride >= 0, "paged cache: negative stride");
  PFB_CHECK_ARG(c.k && c.v, "paged cache: null pointer");
}

}  // namespace pfb
