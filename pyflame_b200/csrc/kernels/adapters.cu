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
// ranks, and a part of the outputs in the second.  What lies between the
// products enters the second as two 16-bit parts (fp32: split tf32), so that
// it rounds far less than the output.
//
// Groups of up to 8 rows read A and B, which are most of their bytes, through
// a ring of asynchronous copies for each warp: B's copies are on their way
// before the first product's sums have met.  In larger groups x, base and out
// are most of the bytes: x comes through the ring, and in the second product
// the rows are the 16 rows of a matrix instruction, so that a lane ends with 8
// neighbouring outputs of a row.
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
  int most_slots;        // 8 or 32: of a group at most
  int per_tile;          // clusters that share a tile's groups
};

constexpr int kRing = 10752;  // bytes of a warp's ring: 7 stages of few rows, 3 of many

// 16 bytes of a row of x from byte `at` on, zeros behind the row's end
template <typename T>
__device__ __forceinline__ uint4 load_row(const T* row, int at, int inner) {
  constexpr int VEC = 16 / sizeof(T);
  const int first = at / (int)sizeof(T);
  alignas(16) T v[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = first + e < inner ? row[first + e] : from_float<T>(0.f);
  return *reinterpret_cast<const uint4*>(v);
}

__device__ __forceinline__ uint4 read_shared(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}

// Adds up what the warps left of `blocks` blocks of 16 ranks x 8 vectors, at
// red + warp * pitch (in float4), to sums[rank][slots].
__device__ __forceinline__ void add_warps(const float4* red, int pitch, int blocks, int nt, int r0, int slots, float* sums) {
  for (int i = threadIdx.x; i < blocks * 32; i += kThreads) {
    float4 s = red[i];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float4 v = red[w * pitch + i];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    const int l = i & 31, b = i >> 5, n = b % nt, r = b / nt;
    float* to = sums + (r0 + r * 16 + (l >> 2)) * slots + n * 8 + 2 * (l & 3);
    to[0] = s.x;
    to[1] = s.y;
    to[8 * slots] = s.z;
    to[8 * slots + 1] = s.w;
  }
}

// Shared memory: the warps' rings, then (a group of few rows) the warps' sums
// of up to two blocks of ranks and h, then the sums that the cluster reads.  A
// group of many rows has its warps' sums and h in the rings' place.
template <typename T>
struct Layout {
  static constexpr int kParts = sizeof(T) == 2 ? 2 : 1;
  // of a row of h: the ranks, rounded up to whole pieces of 64 bytes, and rows in other banks
  static __host__ __device__ int pitch(int rank) { return (rank * (int)sizeof(T) + 63) / 64 * (64 / (int)sizeof(T)) + 16 / (int)sizeof(T); }
  static constexpr int kRed = kWarps * 2 * 512;
  static __host__ __device__ int h_bytes(int rank, int slots) { return kParts * slots * pitch(rank) * (int)sizeof(T); }
  static __host__ __device__ int sums_at(int rank) { return kWarps * kRing + kRed + h_bytes(rank, 8); }
  static int bytes(int rank, int slots) { return sums_at(rank) + rank * slots * 4; }
};

// h [slots][pitch], the cluster's sums times the adapter's scale, in parts;
// zeros behind the ranks.
template <typename T>
__device__ __forceinline__ void make_h(const Args& a, cg::cluster_group& cluster, int ranks, float scale, float* sums, int slots, T* h, int part) {
  const int pitch = Layout<T>::pitch(a.rank), wide = pitch - 16 / (int)sizeof(T);
  for (int j = threadIdx.x; j < slots * wide; j += kThreads) {
    const int s = j / wide, r = j - s * wide;
    float v = 0.f;
    if (r < a.rank) {
      const int at = r * slots + s;
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
}

// A group of up to 8 rows.
template <typename T>
__device__ __forceinline__ void few_rows(const Args& a, cg::cluster_group& cluster, int ranks, int adapter, const int* slots, int count,
                                         int row0, int q, int of, char* smem) {
  using L = Layout<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  constexpr int kStage = 1536, kDepth = kRing / kStage;
  float4* red = reinterpret_cast<float4*>(smem + kWarps * kRing);
  T* h = reinterpret_cast<T*>(smem + kWarps * kRing + L::kRed);
  float* sums = reinterpret_cast<float*>(smem + L::sums_at(a.rank));
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * kRing) + lane * 16;

  const int a_bytes = (int)a.a_row, b_bytes = a.rank * (int)sizeof(T);
  const int a_pieces = (a_bytes + 63) / 64, b_pieces = (b_bytes + 63) / 64;
  const T* row = g < count ? (const T*)a.x + (long long)(row0 + slots[g]) * a.x_st : nullptr;
  const int x_size = row && a.x_wide ? 16 : 0;
  const char* a_first = a.a + ((long long)adapter * a.rank + g) * a.a_row;
  const char* b_first = (const char*)a.b + (long long)adapter * a.outer * b_bytes;
  const int blocks = (a.outer + 15) / 16;

  // What the copies stand at: pieces q, q + of, ... of A's blocks of 16 rows,
  // one block after the other, then all pieces of B's blocks q, q + of, ...
  int r_ahead = q < a_pieces ? 0 : a.rank, c_ahead = q, u_ahead = q, k_ahead = 0;
  auto copy = [&](uint32_t to) {
    if (r_ahead < a.rank) {
      const int at = c_ahead * 64 + t * 16;
      const int size = at < a_bytes ? 16 : 0;
      const char* from = a_first + r_ahead * a.a_row + at;
      copy_async(to, from, size);
      copy_async(to + 512, from + 8 * a.a_row, size);
      // rows of x end where their values do: a last piece that is not whole is read by elements
      copy_async(to + 1024, row ? (const char*)row + at : a.a, at + 16 <= a.inner * (int)sizeof(T) ? x_size : 0);
      c_ahead += of;
      if (c_ahead >= a_pieces) {
        c_ahead = q;
        r_ahead += 16;
      }
    } else if (u_ahead < blocks) {
      const int at = k_ahead * 64 + t * 16, n = u_ahead * 16 + g;
      const int size = at < b_bytes ? 16 : 0;
      const char* from = b_first + (long long)min(n, a.outer - 1) * b_bytes + at;
      copy_async(to, from, n < a.outer ? size : 0);
      copy_async(to + 512, n + 8 < a.outer ? from + 8 * b_bytes : from, n + 8 < a.outer ? size : 0);
      if (++k_ahead == b_pieces) {
        k_ahead = 0;
        u_ahead += of;
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kDepth; ++s) copy(ring + s * kStage);
  uint32_t at = ring;
  auto next = [&]() { at = at == ring + (kDepth - 1) * kStage ? ring : at + kStage; };

  for (int r0 = 0; r0 < a.rank; r0 += 32) {
    const int some = min(2, (a.rank - r0) / 16);
    for (int r = 0; r < some; ++r) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c = q; c < a_pieces; c += of) {
        copy_wait<kDepth - 1>();
        uint4 v[1] = {read_shared(at + 1024)};
        const int byte = c * 64 + t * 16;
        if (row && (!a.x_wide || byte + 16 > a.inner * (int)sizeof(T))) v[0] = load_row<T>(row, byte, a.inner);
        float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
        chunk_product<T, 1>(sum, read_shared(at), read_shared(at + 512), v);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += sum[0][i];
        copy(at);
        next();
      }
      red[(warp * 2 + r) * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    }
    __syncthreads();
    add_warps(red, 64, some, 1, r0, 8, sums);
    __syncthreads();
  }
  if (ranks > 1) cluster.sync();
  const int pitch = L::pitch(a.rank), part = 8 * pitch;
  make_h<T>(a, cluster, ranks, a.scales[adapter], sums, 8, h, part);
  // the others have read this CTA's sums before it writes the next ones or ends
  if (ranks > 1) cluster.sync();
  else __syncthreads();

  // outputs 16u + g and + 8 of the rows in slots 2t and 2t + 1
  const T* from[2] = {nullptr, nullptr};
  T* to[2] = {nullptr, nullptr};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (2 * t + i < count) {
      const long long m = row0 + slots[2 * t + i];
      from[i] = a.base ? (const T*)a.base + m * a.base_st : nullptr;
      to[i] = (T*)a.out + m * a.out_st;
    }
  float base[4], next_base[4];
  auto load_base = [&](int u, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = u * 16 + g + 8 * (i >> 1);
      v[i] = from[i & 1] && n < a.outer ? to_float<T>(from[i & 1][n]) : 0.f;
    }
  };
  if (q < blocks) load_base(q, next_base);
  const uint32_t h_at = (uint32_t)__cvta_generic_to_shared(h) + (g * pitch) * (int)sizeof(T) + t * 16;
  for (int u = q; u < blocks; u += of) {
#pragma unroll
    for (int i = 0; i < 4; ++i) base[i] = next_base[i];
    if (u + of < blocks) load_base(u + of, next_base);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < b_pieces; ++k) {
      copy_wait<kDepth - 1>();
      const uint4 w0 = read_shared(at), w1 = read_shared(at + 512);
      float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int p = L::kParts - 1; p >= 0; --p) {
        const uint4 v[1] = {read_shared(h_at + p * part * (int)sizeof(T) + k * 64)};
        chunk_product<T, 1>(sum, w0, w1, v);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += sum[0][i];
      copy(at);
      next();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = u * 16 + g + 8 * (i >> 1);
      if (to[i & 1] && n < a.outer) to[i & 1][n] = from_float<T>(base[i] + acc[i]);
    }
  }
  __syncthreads();  // h and the sums are written again for the next group
}

// The second product for up to 32 rows: h [slots][pitch] in shared memory
// (16-bit: the high parts, then the low ones), MT blocks of 16 of them; the
// warp's blocks of 32 outputs u = q, q + of, ...
template <typename T, int MT>
__device__ __forceinline__ void expand(const Args& a, int adapter, const T* h, int part, const int* slots, int count, int row0, int q, int of) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pitch = Layout<T>::pitch(a.rank);
  const T* weights = (const T*)a.b + (long long)adapter * a.outer * a.rank;
  const int blocks = (a.outer + 31) / 32;
  constexpr int WORDS = 8 * (int)sizeof(T) / 16;
  union Eight {
    uint4 raw[WORDS];
    T v[8];
    __device__ Eight() {}
  };
  long long rows[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) rows[m][r] = m * 16 + g + 8 * r < count ? row0 + slots[m * 16 + g + 8 * r] : -1;
  // base is loaded a block ahead
  auto load_base = [&](int u, Eight (&io)[MT][2]) {
    const int n = 32 * u + 8 * t;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool there = rows[m][r] >= 0 && a.base;
        const T* from = (const T*)a.base + (there ? rows[m][r] * a.base_st + n : 0);
        if (a.out_wide && n + 8 <= a.outer) {
#pragma unroll
          for (int i = 0; i < WORDS; ++i) io[m][r].raw[i] = there ? __ldcs(reinterpret_cast<const uint4*>(from) + i) : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) io[m][r].v[e] = there && n + e < a.outer ? from[e] : from_float<T>(0.f);
        }
      }
  };
  Eight io[MT][2], ahead[MT][2];
  if (q < blocks) load_base(q, ahead);
  for (int u = q; u < blocks; u += of) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < WORDS; ++i) io[m][r].raw[i] = ahead[m][r].raw[i];
    float acc[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
    // column c of block j is output 32u + 8 (c / 2) + 2j + c % 2
    const int n0 = 32 * u + 8 * (g >> 1) + (g & 1);
    bool first = true;
    for (int k = 0; k < a.rank; k += 16) {
      const int at = k + 4 * t;
      using Word = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
      Word w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = n0 + 2 * j < a.outer ? *reinterpret_cast<const Word*>(weights + (long long)(n0 + 2 * j) * a.rank + at) : Word();
      if (first && u + of < blocks) load_base(u + of, ahead);
      first = false;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int p = 1; p >= 0; --p) {
            const uint2 x0 = *reinterpret_cast<const uint2*>(h + p * part + (m * 16 + g) * pitch + at);
            const uint2 x1 = *reinterpret_cast<const uint2*>(h + p * part + (m * 16 + g + 8) * pitch + at);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma16(acc[m][j], x0.x, x1.x, x0.y, x1.y, w[j].x, w[j].y, T());
          }
        } else {
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
        if (rows[m][r] < 0 || n >= a.outer) continue;
        T* to = (T*)a.out + rows[m][r] * a.out_st + n;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            T& v = io[m][r].v[2 * j + i];
            v = from_float<T>(to_float<T>(v) + acc[m][j][2 * r + i]);
          }
        if (a.out_wide && n + 8 <= a.outer) {
#pragma unroll
          for (int i = 0; i < WORDS; ++i) __stcs(reinterpret_cast<uint4*>(to) + i, io[m][r].raw[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < a.outer) to[e] = io[m][r].v[e];
        }
      }
  }
}

// A group of 9 to 32 rows.
template <typename T>
__device__ __forceinline__ void many_rows(const Args& a, cg::cluster_group& cluster, int ranks, int adapter, const int* slots, int count,
                                          int row0, int q, int of, char* smem) {
  using L = Layout<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  constexpr int NT = 4, kStage = 1024 + NT * 512, kDepth = kRing / kStage;
  float* sums = reinterpret_cast<float*>(smem + L::sums_at(a.rank));
  T* h = reinterpret_cast<T*>(smem);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * kRing) + lane * 16;
  const int bytes = (int)a.a_row, pieces = (bytes + 63) / 64, x_bytes = a.inner * (int)sizeof(T);
  const T* rows[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) rows[n] = n * 8 + g < count ? (const T*)a.x + (long long)(row0 + slots[n * 8 + g]) * a.x_st : nullptr;

  for (int r0 = 0; r0 < a.rank; r0 += 16) {  // x is read again, from L2, for every 16 ranks
    const char* weights = a.a + ((long long)adapter * a.rank + r0 + g) * a.a_row;
    int c_ahead = q;
    auto copy = [&](uint32_t to) {
      if (c_ahead < pieces) {
        const int at = c_ahead * 64 + t * 16;
        const int size = at < bytes ? 16 : 0, x_size = a.x_wide && at + 16 <= x_bytes ? 16 : 0;
        copy_async(to, weights + at, size);
        copy_async(to + 512, weights + 8 * a.a_row + at, size);
#pragma unroll
        for (int n = 0; n < NT; ++n) copy_async(to + 1024 + n * 512, rows[n] ? (const char*)rows[n] + at : a.a, rows[n] ? x_size : 0);
        c_ahead += of;
      }
      copy_commit();
    };
#pragma unroll
    for (int s = 0; s < kDepth; ++s) copy(ring + s * kStage);
    uint32_t at = ring;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    for (int c = q; c < pieces; c += of) {
      copy_wait<kDepth - 1>();
      uint4 v[NT];
      const int byte = c * 64 + t * 16;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        v[n] = read_shared(at + 1024 + n * 512);
        if (rows[n] && (!a.x_wide || byte + 16 > x_bytes)) v[n] = load_row<T>(rows[n], byte, a.inner);
      }
      float sum[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
      chunk_product<T, NT>(sum, read_shared(at), read_shared(at + 512), v);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] += sum[n][i];
      copy(at);
      at = at == ring + (kDepth - 1) * kStage ? ring : at + kStage;
    }
    copy_wait<0>();
    float4* red = reinterpret_cast<float4*>(smem);  // in the warps' rings
#pragma unroll
    for (int n = 0; n < NT; ++n) red[warp * (kRing / 16) + n * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    __syncthreads();
    add_warps(red, kRing / 16, NT, NT, r0, 8 * NT, sums);
    __syncthreads();
  }
  if (ranks > 1) cluster.sync();
  const int part = 32 * L::pitch(a.rank);
  make_h<T>(a, cluster, ranks, a.scales[adapter], sums, 32, h, part);
  // the others have read this CTA's sums before it writes the next ones or ends
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  if constexpr (sizeof(T) == 2) {
    if (count <= 16) expand<T, 1>(a, adapter, h, part, slots, count, row0, q, of);
    else expand<T, 2>(a, adapter, h, part, slots, count, row0, q, of);
  } else {  // (two blocks of fp32 rows do not fit the registers)
    for (int s = 0; s < count; s += 16) expand<T, 1>(a, adapter, h + s * L::pitch(a.rank), part, slots + s, count - s, row0, q, of);
  }
  __syncthreads();  // h's place is the rings of the next group
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) adapters_kernel(Args a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ int slots[kTile];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
    if (count <= 8) few_rows<T>(a, cluster, ranks, adapter, slots, count, row0, q, of, smem);
    else many_rows<T>(a, cluster, ranks, adapter, slots, count, row0, q, of, smem);
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
  a.most_slots = p.rows <= 8 ? 8 : 32;
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
