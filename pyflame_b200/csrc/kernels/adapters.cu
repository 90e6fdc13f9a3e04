// adapters.cu — low-rank adapters of many requests beside a shared projection.
//
//   out[m] = base[m] + s_i B_i (A_i x[m]),   i = index[m]
//
// x is read, base read and out written once, and so are A and B of the
// adapters in use: 2 * rank operations for each value of x and out, so memory
// is the bound.  One kernel does both products, since what passes between
// them is a few numbers a row.
//
// A tile is 32 consecutive rows.  Its rows that share an adapter form a group
// (a prompt's tile is one group, a tile of 32 users' tokens 32): the rows are
// the vectors of A's products (streamed.cuh).  A cluster of CTAs takes a
// group, few rows several CTAs: each a part of x's axis in the first product,
// whose sums meet through distributed shared memory in the order of the
// ranks, and a part of the outputs in the second.  There the group's rows are
// the 16 rows of a matrix instruction, and what lies between the products
// enters as two 16-bit parts (fp32: split tf32), so that it rounds far less
// than the output.  A lane ends with 8 neighbouring outputs of a row.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "../common.hpp"
#include "decode.cuh"
#include "kernels.hpp"
#include "streamed.cuh"

namespace pfb {
namespace {

namespace cg = cooperative_groups;

constexpr int kTile = 32;  // rows; a warp's lanes look them over
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMostRank = 256;
constexpr int kMostRanks = 8;  // CTAs of a cluster

struct Args {
  int rows, inner, outer, rank, adapters;
  const void* x;
  long long x_st;
  const int* index;
  const void* base;
  long long base_st;
  void* out;
  long long out_st;
  const char* a;
  long long a_row;  // bytes
  const void* b;
  const float* scales;
  int* err;
  int x_wide, out_wide;  // rows may be accessed 16 bytes at a time
  int most_slots;        // 8, 16 or 32: of a group at most
  int per_tile;          // clusters that share a tile's groups
};

// 16 bytes of a row of x from byte `at` on, zeros behind the row's end
template <typename T>
__device__ __forceinline__ uint4 load_row(const T* row, int at, int inner, bool wide) {
  constexpr int VEC = 16 / sizeof(T);
  const int first = at / (int)sizeof(T);
  if (wide && first + VEC <= inner) return *reinterpret_cast<const uint4*>(row + first);
  alignas(16) T v[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = first + e < inner ? row[first + e] : from_float<T>(0.f);
  return *reinterpret_cast<const uint4*>(v);
}

// The first product over the CTA's pieces of x's axis, for RT blocks of 16
// ranks from r0 on: sums[rank][slots], NT * 8 slots.
template <typename T, int RT, int NT, int UNROLL>
__device__ __forceinline__ void shrink(const Args& a, int adapter, int r0, const T* const (&rows)[4], int q, int of, float4* red,
                                       float* sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const char* weights = a.a + ((long long)adapter * a.rank + r0 + g) * a.a_row;
  const int bytes = (int)a.a_row, pieces = (bytes + 63) / 64;
  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int c0 = q; c0 < pieces; c0 += of * UNROLL) {
    uint4 w[UNROLL][RT][2], v[UNROLL][NT];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int at = (c0 + u * of) * 64 + t * 16;
      const bool in = at < bytes;
#pragma unroll
      for (int n = 0; n < NT; ++n) v[u][n] = in && rows[n] ? load_row<T>(rows[n], at, a.inner, a.x_wide) : zero;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        w[u][r][0] = in ? *reinterpret_cast<const uint4*>(weights + (r * 16) * a.a_row + at) : zero;
        w[u][r][1] = in ? *reinterpret_cast<const uint4*>(weights + (r * 16 + 8) * a.a_row + at) : zero;
      }
    }
    // a step's sums are added in fp32, rounded to nearest: the tensor cores truncate
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float sum[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) chunk_product<T, NT>(sum, w[u][r][0], w[u][r][1], v[u]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] += sum[n][i];
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
      red[((warp * RT + r) * NT + n) * 32 + lane] = make_float4(acc[r][n][0], acc[r][n][1], acc[r][n][2], acc[r][n][3]);
  __syncthreads();
  for (int i = tid; i < RT * NT * 32; i += kThreads) {
    float4 s = red[i];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float4 v = red[w * RT * NT * 32 + i];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    const int l = i & 31, n = (i >> 5) % NT, r = (i >> 5) / NT;
    float* to = sums + (r0 + r * 16 + (l >> 2)) * (NT * 8) + n * 8 + 2 * (l & 3);
    to[0] = s.x;
    to[1] = s.y;
    to[8 * NT * 8] = s.z;
    to[8 * NT * 8 + 1] = s.w;
  }
  __syncthreads();
}

template <typename T, int NT>
__device__ __forceinline__ void shrink_all(const Args& a, int adapter, const T* const (&rows)[4], int q, int of, float4* red,
                                           float* sums) {
  int r0 = 0;
  if constexpr (NT == 1)
    for (; r0 + 64 <= a.rank; r0 += 64) shrink<T, 4, NT, 2>(a, adapter, r0, rows, q, of, red, sums);
  for (; r0 + 32 <= a.rank; r0 += 32) shrink<T, 2, NT, NT == 4 ? 2 : 4>(a, adapter, r0, rows, q, of, red, sums);
  for (; r0 < a.rank; r0 += 16) shrink<T, 1, NT, NT == 4 ? 2 : 4>(a, adapter, r0, rows, q, of, red, sums);
}

// The second product: h [slots][pitch] in shared memory (16-bit: the high
// parts, then the low ones), the group's rows of 16, MT blocks of them; the
// warp's blocks of 32 outputs u = q, q + of, ...
template <typename T, int MT>
__device__ __forceinline__ void expand(const Args& a, int adapter, const T* h, int pitch, int part, const int* slots, int count,
                                       int row0, int q, int of) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const T* weights = (const T*)a.b + (long long)adapter * a.outer * a.rank;
  const int blocks = (a.outer + 31) / 32;
  for (int u = q; u < blocks; u += of) {
    float acc[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
    // column c of block j is output 32u + 8 (c / 2) + 2j + c % 2
    const int n0 = 32 * u + 8 * (g >> 1) + (g & 1);
#pragma unroll 2
    for (int k = 0; k < a.rank; k += 16) {
      const int at = k + 4 * t;
      if constexpr (sizeof(T) == 2) {
        uint2 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = n0 + 2 * j < a.outer ? *reinterpret_cast<const uint2*>(weights + (long long)(n0 + 2 * j) * a.rank + at) : make_uint2(0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 1; p >= 0; --p) {
            const uint2 x0 = *reinterpret_cast<const uint2*>(h + p * part + (m * 16 + g) * pitch + at);
            const uint2 x1 = *reinterpret_cast<const uint2*>(h + p * part + (m * 16 + g + 8) * pitch + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma16(acc[m][j], x0.x, x1.x, x0.y, x1.y, w[j].x, w[j].y, T());
          }
      } else {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = n0 + 2 * j < a.outer ? *reinterpret_cast<const uint4*>(weights + (long long)(n0 + 2 * j) * a.rank + at)
                                      : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 x0 = *reinterpret_cast<const uint4*>(h + (m * 16 + g) * pitch + at);
          const uint4 x1 = *reinterpret_cast<const uint4*>(h + (m * 16 + g + 8) * pitch + at);
          float sum[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j][0] = sum[j][1] = sum[j][2] = sum[j][3] = 0.f;
          chunk_product<T, 4>(sum, x0, x1, w);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[m][j][r] += sum[j][r];
        }
      }
    }
    const int n = 32 * u + 8 * t;  // the lane's 8 outputs
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int slot = m * 16 + g + 8 * r;
        if (slot >= count || n >= a.outer) continue;
        const long long row = row0 + slots[slot];
        const T* from = a.base ? (const T*)a.base + row * a.base_st + n : nullptr;
        T* to = (T*)a.out + row * a.out_st + n;
        constexpr int WORDS = 8 * (int)sizeof(T) / 16;
        union {
          uint4 raw[WORDS];
          T v[8];
        } io;
        const bool wide = a.out_wide && n + 8 <= a.outer;
        if (wide) {
#pragma unroll
          for (int i = 0; i < WORDS; ++i) io.raw[i] = from ? reinterpret_cast<const uint4*>(from)[i] : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) io.v[e] = from && n + e < a.outer ? from[e] : from_float<T>(0.f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) io.v[2 * j + i] = from_float<T>(to_float<T>(io.v[2 * j + i]) + acc[m][j][2 * r + i]);
        if (wide) {
#pragma unroll
          for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint4*>(to)[i] = io.raw[i];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < a.outer) to[e] = io.v[e];
        }
      }
  }
}

template <typename T>
struct Layout {
  static constexpr int kParts = sizeof(T) == 2 ? 2 : 1;
  static __host__ __device__ int pitch(int rank) { return rank + (int)(16 / sizeof(T)); }  // of h: rows in other banks
  // the warps' sums, or h after them, then the sums that the cluster reads
  static __host__ __device__ int first_bytes(int rank, int slots) {
    const int blocks = (rank < 64 ? (rank < 32 ? 1 : 2) : (slots <= 8 ? 4 : 2)) * (slots / 8);
    const int red = kWarps * blocks * 32 * 16, h = kParts * (slots < 16 ? 16 : slots) * pitch(rank) * (int)sizeof(T);
    return red > h ? red : h;
  }
  static int bytes(int rank, int slots) { return first_bytes(rank, slots) + rank * slots * 4; }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) adapters_kernel(Args a) {
  using L = Layout<T>;
  extern __shared__ __align__(16) char smem[];
  __shared__ int slots[kTile];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  float4* red = reinterpret_cast<float4*>(smem);
  T* h = reinterpret_cast<T*>(smem);
  float* sums = reinterpret_cast<float*>(smem + L::first_bytes(a.rank, a.most_slots));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2;
  const int unit = (int)(blockIdx.x / ranks), row0 = unit / a.per_tile * kTile, first_group = unit % a.per_tile;
  begin();

  int mine = INT_MIN;  // the lane's row's adapter
  if (row0 + lane < a.rows) {
    mine = a.index[row0 + lane];
    if (mine >= a.adapters) {
      if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
      mine = -1;
    }
    mine = max(mine, -1);
  }
  const unsigned same = __match_any_sync(~0u, mine);
  // groups by their first rows
  const unsigned firsts = __ballot_sync(~0u, mine != INT_MIN && (int)(__ffs(same) - 1) == lane);
  const int groups = __popc(firsts);

  const int q = rank * kWarps + warp, of = ranks * kWarps;
  for (int i = first_group; i < groups; i += a.per_tile) {
    unsigned left = firsts;
    for (int k = 0; k < i; ++k) left &= left - 1;
    const int leader = __ffs(left) - 1;
    const unsigned members = __shfl_sync(~0u, same, leader);
    const int adapter = __shfl_sync(~0u, mine, leader), count = __popc(members);
    if (adapter < 0) {  // rows without one
      if (a.out == a.base && a.out_st == a.base_st) continue;
      for (unsigned m = members; m; m &= m - 1) {
        const long long row = row0 + __ffs(m) - 1;
        const T* from = a.base ? (const T*)a.base + row * a.base_st : nullptr;
        T* to = (T*)a.out + row * a.out_st;
        for (int n = rank * kThreads + tid; n < a.outer; n += ranks * kThreads) to[n] = from ? from[n] : from_float<T>(0.f);
      }
      continue;
    }
    if (warp == 0 && (members >> lane & 1)) slots[__popc(members & ((1u << lane) - 1))] = lane;
    __syncthreads();
    const T* rows[4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      rows[n] = n * 8 + g < count ? (const T*)a.x + (long long)(row0 + slots[n * 8 + g]) * a.x_st : nullptr;
    const int wide = count <= 8 ? 8 : count <= 16 ? 16 : 32;
    if (wide == 8) shrink_all<T, 1>(a, adapter, rows, q, of, red, sums);
    else if (wide == 16) shrink_all<T, 2>(a, adapter, rows, q, of, red, sums);
    else shrink_all<T, 4>(a, adapter, rows, q, of, red, sums);
    if (ranks > 1) cluster.sync();
    // h, the cluster's sums times the adapter's scale; blocks of 16 rows, of
    // which those behind the last slot are zeros
    const float scale = a.scales[adapter];
    const int pitch = L::pitch(a.rank), part = max(wide, 16) * pitch;
    for (int j = tid; j < max(wide, 16) * a.rank; j += kThreads) {
      const int s = j / a.rank, r = j - s * a.rank;
      float v = 0.f;
      if (s < wide) {
        const int at = r * wide + s;
        if (ranks > 1) {
#pragma unroll
          for (int c = 0; c < kMostRanks; ++c)
            if (c < ranks) v += cluster.map_shared_rank(sums, c)[at];
        } else {
          v = sums[at];
        }
        v *= scale;
      }
      if constexpr (sizeof(T) == 4) {
        h[s * pitch + r] = v;
      } else {
        T hi, lo;
        two_parts(v, hi, lo);
        h[s * pitch + r] = hi;
        h[part + s * pitch + r] = lo;
      }
    }
    // the others have read this CTA's sums before it writes the next ones or ends
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    if (wide <= 16) expand<T, 1>(a, adapter, h, pitch, part, slots, count, row0, q, of);
    else expand<T, 2>(a, adapter, h, pitch, part, slots, count, row0, q, of);
    __syncthreads();  // h's place is the warps' sums of the next group
  }
}

void check(const pfk_adapters_params& p) {
  check_decode_dtype(p.dtype);
  const int64_t es = p.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  PFB_CHECK_ARG(p.rows >= 0 && p.rows <= INT32_MAX - kTile, "adapters: bad number of rows");
  PFB_CHECK_ARG(p.inner >= 1 && p.inner <= (1 << 24) && p.outer >= 1 && p.outer <= (1 << 24), "adapters: inner and outer must be 1 to 2^24");
  PFB_CHECK_ARG(p.adapters >= 1 && p.adapters <= INT32_MAX, "adapters: their number must be 1 to 2^31 - 1");
  PFB_CHECK_ARG(p.rank >= 16 && p.rank % 16 == 0 && p.rank <= kMostRank, "adapters: rank must be a multiple of 16, at most 256");
  PFB_CHECK_ARG(p.x_st >= 0 && p.base_st >= 0 && p.out_st >= 0, "adapters: negative stride");
  PFB_CHECK_ARG(p.a_st >= p.inner && p.a_st * es % 16 == 0, "adapters: rows of a must be padded to multiples of 16 bytes");
}

template <typename T>
void launch_typed(Args& a, int64_t ctas, int ranks, cudaStream_t stream) {
  static std::once_flag once[64];
  std::call_once(once[current_device()], [] {
    PFB_CUDA(cudaFuncSetAttribute(adapters_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<T>::bytes(kMostRank, kTile)));
  });
  launch_following<Args>(adapters_kernel<T>, dim3((unsigned)ctas), kThreads, (size_t)Layout<T>::bytes(a.rank, a.most_slots), stream, a,
                         ranks);
}

}  // namespace

void launch_adapters(const pfk_adapters_params& p, cudaStream_t stream) {
  check(p);
  if (p.rows == 0) return;
  PFB_CHECK_ARG(p.x && p.index && p.out && p.a && p.b && p.scales, "adapters: null pointer");
  PFB_CHECK_ARG((uintptr_t)p.a % 16 == 0 && (uintptr_t)p.b % 16 == 0, "adapters: a and b must be 16-byte aligned");
  PFB_CHECK_ARG(p.out != p.base || p.rows == 1 || p.out_st == p.base_st, "adapters: out shares base's memory with another stride");
  const int64_t es = p.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  Args a = {};
  a.rows = (int)p.rows;
  a.inner = (int)p.inner;
  a.outer = (int)p.outer;
  a.rank = (int)p.rank;
  a.adapters = (int)p.adapters;
  a.x = p.x;
  a.index = p.index;
  a.base = p.base;
  a.out = p.out;
  if (p.rows > 1) {  // one row's stride says nothing
    a.x_st = p.x_st;
    a.base_st = p.base_st;
    a.out_st = p.out_st;
  }
  a.a = (const char*)p.a;
  a.a_row = p.a_st * es;
  a.b = p.b;
  a.scales = p.scales;
  a.err = p.err;
  a.x_wide = (uintptr_t)p.x % 16 == 0 && a.x_st * es % 16 == 0;
  a.out_wide = (uintptr_t)p.out % 16 == 0 && a.out_st * es % 16 == 0 && (uintptr_t)p.base % 16 == 0 && a.base_st * es % 16 == 0;
  a.most_slots = p.rows <= 8 ? 8 : p.rows <= 16 ? 16 : 32;
  // A tile has up to as many groups as rows or adapters; clusters for all of
  // them, which end at once where there are fewer, as long as these do not
  // become thousands of CTAs.
  const int64_t tiles = ceil_div(p.rows, kTile), groups = std::min<int64_t>({kTile, p.rows, p.adapters + 1});
  a.per_tile = (int)std::min(groups, std::max<int64_t>(1, 2048 / tiles));
  const int64_t units = tiles * a.per_tile;
  PFB_CHECK_ARG(units <= INT32_MAX / kMostRanks, "adapters: too many rows");
  // few groups: several CTAs each, as long as all warps have something of one of the products
  const int64_t work = std::max(ceil_div(a.a_row, 64), ceil_div(p.outer, 32));
  int ranks = 1;
  while (ranks < kMostRanks && units * ranks <= 512 && work > ranks * kWarps) ranks *= 2;
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_typed<float>(a, units * ranks, ranks, stream);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_typed<__half>(a, units * ranks, ranks, stream);
  else launch_typed<__nv_bfloat16>(a, units * ranks, ranks, stream);
}

}  // namespace pfb
