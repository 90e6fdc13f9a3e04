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
