// linear_w4.cu — products with 4-bit weights for single tokens and small
// batches.
//
//   y[m,n] = sum_g s[n,g] sum_{k in g} x[m,k] (q[n,k] - z[n,g])  (+ bias[n])
//
// The weights are read once, at half a byte each; with few rows of x that
// read bounds the product, so the arithmetic must cost little per weight.  It
// runs on mma.sync: q - z is an integer of at most 5 bits, exact in fp16 and
// bf16, and so are 16-bit values of x; the products accumulate in fp32 over a
// group and the group's sum is multiplied by its scale in fp32, so no weight
// is ever rounded.  fp32 x enters as three bf16 parts (8 bits each, 24 in
// all), which take three columns of the instruction instead of three
// instructions.  Two weights cost one logic operation and one subtraction:
// a nibble pair OR-ed into the mantissas of two 16-bit numbers is 2^7 + q
// (2^10 + q in fp16), from which 2^7 + z is subtracted exactly.
//
// A CTA of 8 warps takes 16 output rows; its warps take the blocks of 128
// columns in turn and add their sums through shared memory in a fixed order.
// In a block a lane holds 16 bytes of two weight rows: the words of the
// arranged layout give each lane 8 columns of each of the four 32-column
// groups, so that no instruction mixes two groups.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>

#include "../common.hpp"
#include "decode.cuh"
#include "kernels.hpp"

namespace pfb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBlock = 128;            // columns of a warp's step
constexpr int kStep = kBlock * kWarps; // of a CTA's step
constexpr int kPad = 32;               // values between rows of x in shared memory: rows start 64 bytes apart mod 128
constexpr int kRing = 4;               // blocks in flight per warp
constexpr size_t kStageMax = 96 * 1024;

struct Args {
  const void* x;
  long long x_st;
  void* y;
  long long y_st;
  const uint4* weight;
  const void* scales;
  const uint8_t* zeros;
  const void* bias;
  int rows, inner, outer;
  int blocks;    // of 128 columns
  int groups;    // of a row
  int group_blocks;  // blocks that share a scale, for groups of 128 and more
  int scale_dtype;
  int chunk;     // rows of x that a CTA takes
  int tile;      // columns of x in shared memory, a multiple of kStep
  int vector;    // rows of x are 16-byte aligned
};

template <typename T>
struct Num {  // 16-bit type of the products, its magic number for 4-bit integers, and the parts of x
  using N = __nv_bfloat16;
  using N2 = __nv_bfloat162;
  static constexpr unsigned kMagic = 0x43004300u;  // 128
  static constexpr float kBase = 128.f;
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  static __device__ __forceinline__ N of(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ N2 both(float v) { return __float2bfloat162_rn(v); }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Num<__half> {
  using N = __half;
  using N2 = __half2;
  static constexpr unsigned kMagic = 0x64006400u;  // 1024
  static constexpr float kBase = 1024.f;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ N of(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ N2 both(float v) { return __float2half2_rn(v); }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float load_float(const void* p, long long i, int dtype) {
  if (dtype == PFC_DTYPE_FLOAT32) return ((const float*)p)[i];
  if (dtype == PFC_DTYPE_FLOAT16) return __half2float(((const __half*)p)[i]);
  return __bfloat162float(((const __nv_bfloat16*)p)[i]);
}

__device__ __forceinline__ uint4 load_weight(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__device__ __forceinline__ unsigned word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// The columns [k0, k0 + tile) of the CTA's rows of x into shared memory, as
// 16-bit parts: part p of row r in row p*rows + r; zeros behind the last.
template <typename T>
__device__ __forceinline__ void stage(const Args& a, typename Num<T>::N* xs, int first, int rows, int k0) {
  using NT = Num<T>;
  const int pitch = a.tile + kPad;
  const int width = min(a.tile, a.blocks * kBlock - k0);
  for (int i = threadIdx.x * 8; i < rows * width; i += kThreads * 8) {  // width is a multiple of 128
    const int r = i / width, c = i - r * width, k = k0 + c;
    const T* src = (const T*)a.x + (long long)(first + r) * a.x_st + k;
    alignas(16) T v[8];
    if (a.vector && k + 8 <= a.inner) {
#pragma unroll
      for (int e = 0; e < (int)sizeof(T) / 2; ++e) reinterpret_cast<uint4*>(v)[e] = reinterpret_cast<const uint4*>(src)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < a.inner ? src[e] : T(0.f);
    }
    alignas(16) typename NT::N part[8];
    if constexpr (NT::kParts == 1) {
      *reinterpret_cast<uint4*>(xs + r * pitch + c) = *reinterpret_cast<uint4*>(v);
    } else {
      float rest[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
      for (int p = 0; p < NT::kParts; ++p) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          part[e] = NT::of(rest[e]);
          const float left = rest[e] - __bfloat162float(part[e]);
          rest[e] = isfinite(left) ? left : 0.f;  // an infinity or NaN is the first part
        }
        *reinterpret_cast<uint4*>(xs + (p * rows + r) * pitch + c) = *reinterpret_cast<uint4*>(part);
      }
    }
  }
}

// NT: 8-column blocks of x rows (times parts).  G: columns that share a scale
// within a block: 32, 64, or 128 for groups of 128 and more.
template <typename T, int NT, int G>
__global__ void __launch_bounds__(kThreads) linear_kernel(const Args a) {
  using M = Num<T>;
  using N = typename M::N;
  using N2 = typename M::N2;
  extern __shared__ __align__(16) char smem[];
  N* xs = reinterpret_cast<N*>(smem);
  float* red = reinterpret_cast<float*>(smem);  // after the last step: [warp][16][NT * 8 + 1]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int first = blockIdx.y * a.chunk, rows = min(a.chunk, a.rows - first);
  const int cols = rows * M::kParts, pitch = a.tile + kPad;
  const int n0 = blockIdx.x * 16;
  // weight rows g and g + 8; rows behind the last repeat it and are not stored
  const int na = min(n0 + g, a.outer - 1), nb = min(n0 + g + 8, a.outer - 1);
  const uint4* wa = a.weight + (long long)na * a.blocks * 4 + t;
  const uint4* wb = a.weight + (long long)nb * a.blocks * 4 + t;
  const long long sa = (long long)na * a.groups, sb = (long long)nb * a.groups;
  const int steps = (a.blocks + kWarps - 1) / kWarps;

  uint4 ring[kRing][2];
  auto fetch = [&](int step, uint4 (&w)[2]) {
    const int kb = step * kWarps + warp;
    w[0] = w[1] = make_uint4(0, 0, 0, 0);
    if (kb < a.blocks) {
      w[0] = load_weight(wa + (long long)kb * 4);
      w[1] = load_weight(wb + (long long)kb * 4);
    }
  };
#pragma unroll
  for (int i = 0; i < kRing; ++i) fetch(i, ring[i]);

  float acc[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[nt][r] = 0.f;

  const int per_tile = a.tile / kStep;
  for (int base = 0; base < steps; base += kRing) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      const int step = base + i;
      if (step < steps) {
        if (step % per_tile == 0) {
          __syncthreads();
          stage<T>(a, xs, first, rows, step * kStep);
          __syncthreads();
        }
        const int kb = step * kWarps + warp;
        if (kb < a.blocks) {
          const N* xk = xs + g * pitch + (kb * kBlock - step / per_tile * a.tile) + t * 8;
          float part[NT][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // 32 columns
            if (j * 32 % G == 0) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) part[nt][r] = 0.f;
            }
            const int group = G == 128 ? kb / a.group_blocks : (kb * kBlock + j * 32) / G;
            const bool real = group < a.groups;  // groups of padding have no scale; their x is zero
            const N2 za = M::both(M::kBase + (real && a.zeros ? (float)a.zeros[sa + group] : 8.f));
            const N2 zb = M::both(M::kBase + (real && a.zeros ? (float)a.zeros[sb + group] : 8.f));
            const unsigned ua = word(ring[i][0], j), ub = word(ring[i][1], j);
            unsigned qa[4], qb[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const unsigned pa = ((ua >> (4 * e)) & 0x000f000fu) | M::kMagic, pb = ((ub >> (4 * e)) & 0x000f000fu) | M::kMagic;
              const N2 da = __hsub2(*reinterpret_cast<const N2*>(&pa), za), db = __hsub2(*reinterpret_cast<const N2*>(&pb), zb);
              qa[e] = *reinterpret_cast<const unsigned*>(&da);
              qb[e] = *reinterpret_cast<const unsigned*>(&db);
            }
            const unsigned f1[4] = {qa[0], qb[0], qa[1], qb[1]}, f2[4] = {qa[2], qb[2], qa[3], qb[3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 b = make_uint4(0, 0, 0, 0);
              if (nt * 8 + g < cols) b = *reinterpret_cast<const uint4*>(xk + nt * 8 * pitch + j * 32);
              M::mma(part[nt], f1, b.x, b.y);
              M::mma(part[nt], f2, b.z, b.w);
            }
            if ((j + 1) * 32 % G == 0) {
              const float ca = real ? load_float(a.scales, sa + group, a.scale_dtype) : 0.f;
              const float cb = real ? load_float(a.scales, sb + group, a.scale_dtype) : 0.f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                acc[nt][0] = fmaf(ca, part[nt][0], acc[nt][0]);
                acc[nt][1] = fmaf(ca, part[nt][1], acc[nt][1]);
                acc[nt][2] = fmaf(cb, part[nt][2], acc[nt][2]);
                acc[nt][3] = fmaf(cb, part[nt][3], acc[nt][3]);
              }
            }
          }
        }
        fetch(step + kRing, ring[i]);
      }
    }
  }

  // add the warps' sums: accumulator (row g or g + 8, column 2t or 2t + 1)
  __syncthreads();
  constexpr int kPitch = NT * 8 + 1;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      red[(warp * 16 + g + 8 * (r >> 1)) * kPitch + nt * 8 + 2 * t + (r & 1)] = acc[nt][r];
  __syncthreads();
  for (int i = tid; i < 16 * rows; i += kThreads) {
    const int m = i >> 4, n = i & 15;
    if (n0 + n >= a.outer) continue;
    float v = 0.f;
#pragma unroll
    for (int p = M::kParts - 1; p >= 0; --p)
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += red[(w * 16 + n) * kPitch + p * rows + m];
    if (a.bias) v += (float)((const T*)a.bias)[n0 + n];
    ((T*)a.y)[(long long)(first + m) * a.y_st + n0 + n] = T(v);
  }
}

__global__ void arrange_kernel(const uint8_t* packed, long long pitch, int inner, int blocks, long long words, uint32_t* weight) {
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (long long)gridDim.x * blockDim.x) {
    const int w = (int)(i & 15), t = w >> 2, j = w & 3;
    const long long row = (i >> 4) / blocks;
    const int col = (int)((i >> 4) - row * blocks) * kBlock + j * 32 + t * 8;
    uint32_t u = 0;
    for (int e = 0; e < 8; ++e) {
      const int k = col + e;
      const unsigned q = k < inner ? (packed[row * pitch + (k >> 1)] >> (4 * (k & 1))) & 15u : 0u;
      // even columns in nibbles 0-3, odd ones in 4-7
      u |= q << (4 * ((e >> 1) + 4 * (e & 1)));
    }
    weight[i] = u;
  }
}

template <typename T, int NT, int G>
void launch_sized(const Args& a, cudaStream_t stream) {
  static std::once_flag once[64];
  const int dev = current_device();
  constexpr size_t kMost = kStageMax + 64 * 1024;
  std::call_once(once[dev], [] {
    PFB_CUDA(cudaFuncSetAttribute(linear_kernel<T, NT, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost));
  });
  const int rows = std::min(a.chunk, a.rows);
  const size_t smem = std::max<size_t>((size_t)rows * Num<T>::kParts * (a.tile + kPad) * 2, (size_t)kWarps * 16 * (NT * 8 + 1) * 4);
  PFB_CHECK_ARG(smem <= kMost, "linear w4: tile does not fit");
  const dim3 grid((unsigned)ceil_div(a.outer, 16), (unsigned)ceil_div(a.rows, a.chunk));
  linear_kernel<T, NT, G><<<grid, kThreads, smem, stream>>>(a);
  PFB_CUDA(cudaGetLastError());
}

template <typename T>
void launch_typed(Args& a, int64_t group, cudaStream_t stream) {
  constexpr int parts = Num<T>::kParts;
  const int64_t most = 64 / parts;  // rows of x whose parts fit eight column blocks
  const int64_t chunks = ceil_div(a.rows, most);
  a.chunk = (int)ceil_div(a.rows, chunks);
  const int cols = a.chunk * parts;
  // all of x, or as many steps of it as the stage holds
  const int64_t whole = round_up((int64_t)a.blocks * kBlock, kStep);
  const int64_t fits = std::max<int64_t>(kStep, (int64_t)(kStageMax / (2 * cols)) / kStep * kStep);
  a.tile = (int)std::min(whole, fits);
  auto grouped = [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    if (group == 32) launch_sized<T, NT, 32>(a, stream);
    else if (group == 64) launch_sized<T, NT, 64>(a, stream);
    else launch_sized<T, NT, 128>(a, stream);
  };
  if (cols <= 8) grouped(std::integral_constant<int, 1>());
  else if (cols <= 16) grouped(std::integral_constant<int, 2>());
  else if (cols <= 32) grouped(std::integral_constant<int, 4>());
  else grouped(std::integral_constant<int, 8>());
}

}  // namespace

void launch_w4_arrange(const uint8_t* packed, int64_t outer, int64_t inner, uint32_t* weight, cudaStream_t stream) {
  PFB_CHECK_ARG(outer >= 0 && inner >= 0 && outer <= (1 << 28) && inner <= (1 << 28), "w4 arrange: bad size");
  if (outer == 0 || inner == 0) return;
  PFB_CHECK_ARG(packed && weight, "w4 arrange: null pointer");
  const int64_t blocks = ceil_div(inner, kBlock), words = outer * blocks * 16;
  arrange_kernel<<<(unsigned)std::min<int64_t>(ceil_div(words, 256), 148 * 16), 256, 0, stream>>>(
      packed, (inner + 1) / 2, (int)inner, (int)blocks, words, weight);
  PFB_CUDA(cudaGetLastError());
}

void launch_linear_w4(const pfk_linear_w4_params& p, cudaStream_t stream) {
  check_decode_dtype(p.dtype);
  check_decode_dtype(p.scale_dtype);
  PFB_CHECK_ARG(p.rows >= 0 && p.rows <= (1 << 20), "linear w4: rows must be 0 to 2^20");
  PFB_CHECK_ARG(p.inner >= 1 && p.inner <= (1 << 28) && p.outer >= 1 && p.outer <= (1 << 28),
                "linear w4: inner and outer must be 1 to 2^28");
  PFB_CHECK_ARG(p.group == 32 || p.group == 64 || (p.group >= 128 && p.group % 128 == 0 && p.group <= INT32_MAX),
                "linear w4: group must be 32, 64 or a multiple of 128");
  if (p.rows == 0) return;
  PFB_CHECK_ARG(p.x && p.y && p.weight && p.scales, "linear w4: null pointer");
  PFB_CHECK_ARG((uintptr_t)p.weight % 16 == 0, "linear w4: weight must be 16-byte aligned");
  Args a = {};
  const int64_t es = p.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  a.x = p.x;
  a.x_st = p.rows > 1 ? p.x_st : 0;
  a.y = p.y;
  a.y_st = p.y_st;
  a.weight = (const uint4*)p.weight;
  a.scales = p.scales;
  a.scale_dtype = p.scale_dtype;
  a.zeros = p.zeros;
  a.bias = p.bias;
  a.rows = (int)p.rows;
  a.inner = (int)p.inner;
  a.outer = (int)p.outer;
  a.blocks = (int)ceil_div(p.inner, kBlock);
  a.groups = (int)ceil_div(p.inner, p.group);
  a.group_blocks = (int)std::max<int64_t>(1, p.group / kBlock);
  a.vector = (uintptr_t)p.x % 16 == 0 && a.x_st * es % 16 == 0;
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_typed<float>(a, p.group, stream);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_typed<__half>(a, p.group, stream);
  else launch_typed<__nv_bfloat16>(a, p.group, stream);
}

}  // namespace pfb
