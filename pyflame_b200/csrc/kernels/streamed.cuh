// Products of matrix rows that stream from memory with a few vectors, on
// mma.sync: rows and vectors come by asynchronous copies into shared memory,
// where each lane finds its operand registers as it copied them (adapters.cu's
// second product of many rows loads its weights straight into registers).
//
// A chunk is 64 bytes of a row.  Lane (g, t) = (lane / 4, lane % 4) of a warp
// holds bytes 16t ... 16t + 15 of a chunk of rows g and g + 8 of 16 matrix
// rows, and of vector g of eight: the order of the summed axis is free as long
// as both operands agree, so those 16 bytes are the registers of two
// instructions (m16n8k16, or m16n8k8 in fp32).  Results: rows g (c[0], c[1])
// and g + 8 (c[2], c[3]) with vectors 2t and 2t + 1.
//
// fp32 operands are split into tf32 high and low parts, three products (the
// dropped low-low term is below 2^-22 of the product).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace pfb {
namespace {

__device__ __forceinline__ void mma16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                      unsigned b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                      unsigned b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_tf32(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                          unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x = hi + lo: hi is x rounded to tf32's 10 bits of mantissa by an integer
// addition, lo the rest exactly, 12 bits and a sign, of which the tensor cores
// take 11: what is lost is below 2^-22 of x and has either sign, as has the
// product of the low parts, which is left out.  (hi by its mask alone, an
// instruction less, has low parts of x's sign: their products' mean was 2^-22
// of the result.)  An infinity has a low part of NaN, so its products are NaN;
// numbers above 2^127 (2 - 2^-11) round to one.
__device__ __forceinline__ void split_tf32(unsigned x, unsigned& hi, unsigned& lo) {
  hi = (x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}

// Asynchronous copies of 16 bytes into shared memory; of size 0: zeros, and
// nothing is read.  A lane reads only what it copied itself, so that waiting
// for its own copies is enough.
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// c[n] += 16 rows x 8 vectors of one chunk, for NT blocks of vectors
template <typename T, int NT>
__device__ __forceinline__ void chunk_product(float (&c)[NT][4], const uint4& a0, const uint4& a1, const uint4 (&b)[NT]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int n = 0; n < NT; ++n) mma16(c[n], a0.x, a1.x, a0.y, a1.y, b[n].x, b[n].y, T());
#pragma unroll
    for (int n = 0; n < NT; ++n) mma16(c[n], a0.z, a1.z, a0.w, a1.w, b[n].z, b[n].w, T());
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      unsigned h0, h1, h2, h3, l0, l1, l2, l3;
      split_tf32(e ? a0.z : a0.x, h0, l0);
      split_tf32(e ? a1.z : a1.x, h1, l1);
      split_tf32(e ? a0.w : a0.y, h2, l2);
      split_tf32(e ? a1.w : a1.y, h3, l3);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        unsigned bh0, bh1, bl0, bl1;
        split_tf32(e ? b[n].z : b[n].x, bh0, bl0);
        split_tf32(e ? b[n].w : b[n].y, bh1, bl1);
        mma8_tf32(c[n], l0, l1, l2, l3, bh0, bh1);
        mma8_tf32(c[n], h0, h1, h2, h3, bl0, bl1);
        mma8_tf32(c[n], h0, h1, h2, h3, bh0, bh1);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// v as a 16-bit part and the rest of it, which leave 2^-17 of v in bfloat16, and
// in float16, up to 65504, 2^-22 of v or 2^-25, whichever is more; an infinity
// has no rest (its NaN would hide it)
template <typename T>
__device__ __forceinline__ void two_parts(float v, T& hi, T& lo) {
  hi = from_float<T>(v);
  const float back = to_float<T>(hi);
  lo = from_float<T>(fabsf(back) <= 3.402823466e38f ? v - back : 0.f);
}

}  // namespace
}  // namespace pfb
