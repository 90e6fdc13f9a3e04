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
// products enters the second as two 16-bit parts, of float16 calls with a power
// of two for each row (make_h) (fp32: split tf32), so that it rounds far less
// than the output.
//
// Groups of up to 8 rows read A and B, which are most of their bytes, through
// a ring of asynchronous copies for each warp: B's copies are on their way
// before the first product's sums have met.  In larger groups x, base and out
// are most of the bytes: x comes through the ring, and in the second product
// the rows are the 16 rows of a matrix instruction, so that a lane ends with 8
// neighbouring outputs of a row, to which base has come through the ring.
//
// Rows that do not begin on 16 bytes (odd sizes, slices) come through the same
// rings, as the aligned blocks around them, and are shifted in registers; the
// outputs of such large groups change places in shared memory, so that a warp
// stores 32 neighbours.  Read and written by elements, 1900 rows, 4175 to 6129,
// of five mixed adapters of rank 17, bf16, took 144 us, so 89; 3630 rows, 74 to
// 2305, of five prompts and 403 rows without an adapter, fp16, 109 and 37.
//
// Measured (device time, replayed from a graph; the bytes at 6.56 TB/s in
// brackets): one row, 4096 to 4096, rank 16, bf16: 6.1 us, latency alone; 61
// rows with 55 adapters of rank 64, 4096 to 16384, fp16, 149 MB: 39.2 us
// (22.7); 8191 rows of five prompts, rank 16, bf16, 203 MB: 45.1 us (30.9),
// where all CTAs read x and then update the outputs at about the same time.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <type_traits>

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
  long long a_row;  // bytes from a row to the next; of them a_bytes count, zeros behind inner up to 16 bytes
  int a_bytes;
  const void* b;
  const float* scales;
  int* err;
  int most_slots;        // 8 or 32: of a group at most
  int tiles, per_tile;   // per_tile: clusters that share a tile's groups
  int apart;             // CTAs of a cluster take a group each where a tile has more groups than clusters
};

constexpr int kFewBlocks = 4;  // of 16 ranks, whose sums few rows' warps leave at a time
constexpr int kRing = 10752;  // bytes of a warp's ring: 7 stages of few rows, 3 of many (5 and 2 of rows that do not begin on 16 bytes)

// Copies 16 bytes, of which those from `left` on are zeros.
__device__ __forceinline__ void copy_up_to(uint32_t to, const void* from, int left) { copy_async(to, from, min(max(left, 0), 16)); }

// Rows that do not begin on 16 bytes come as the aligned blocks around them:
// the 4 * N words from byte s (0 to 15, even) of N + 1 blocks on.
template <int N>
__device__ __forceinline__ void shift(unsigned (&w)[4 * N + 4], int s) {
#pragma unroll
  for (int i = 0; i < 4 * N + 2; ++i) w[i] = s & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 4 * N + 1; ++i) w[i] = s & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (s & 2) * 8);
}

__device__ __forceinline__ int behind_16(const void* p) { return (int)((uintptr_t)p & 15); }

__device__ __forceinline__ uint4 read_shared(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}

// A lane's 16 bytes of a row that begins s bytes behind 16: of a stage's block
// and, unless all rows begin on 16 bytes (WIDE), of the one 512 bytes on.
template <bool WIDE>
__device__ __forceinline__ uint4 read_row(uint32_t at, int s) {
  const uint4 a = read_shared(at);
  if constexpr (WIDE) return a;
  const uint4 b = read_shared(at + 512);
  unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  shift<1>(w, s);
  return make_uint4(w[0], w[1], w[2], w[3]);
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

// Shared memory: the warps' rings, then the warps' sums of up to four blocks
// of ranks and h (a group of many rows has its warps' sums in the rings and h
// here), then the sums that the cluster reads.
template <typename T>
struct Layout {
  static constexpr int kParts = sizeof(T) == 2 ? 2 : 1;
  // of a row of h: the ranks, rounded up to whole pieces of 64 bytes, and rows in other banks
  static __host__ __device__ int pitch(int rank) { return (rank * (int)sizeof(T) + 63) / 64 * (64 / (int)sizeof(T)) + 16 / (int)sizeof(T); }
  static constexpr int kRed = kWarps * kFewBlocks * 512;
  static __host__ __device__ int h_bytes(int rank, int slots) { return kParts * slots * pitch(rank) * (int)sizeof(T); }
  static __host__ __device__ int sums_at(int rank, int slots) {
    const int few = kRed + h_bytes(rank, 8), many = slots > 8 ? h_bytes(rank, slots) : 0;
    return kWarps * kRing + (few > many ? few : many);
  }
  static int bytes(int rank, int slots) { return sums_at(rank, slots) + rank * slots * 4; }
};

// What the cluster's CTAs have of a sum: a place of `sums` in each.
__device__ __forceinline__ float cluster_sum(cg::cluster_group& cluster, int ranks, float* sums, int at) {
  if (ranks == 1) return sums[at];
  float v = 0.f;
#pragma unroll
  for (int c = 0; c < kMostRanks; ++c)
    if (c < ranks) v += cluster.map_shared_rank(sums, c)[at];
  return v;
}

// h [slots][pitch], the cluster's sums times the adapter's scale, in parts;
// zeros behind the ranks.  fp16 parts reach from 2^-25 to 65504, not as far as
// the sums: a warp takes a slot, whose values are multiplied by the power of two
// that puts the largest between 2^14 and 2^15, so that the parts lose 2^-22 of a
// value, or 2^-39 of the largest where that is more, whatever their size; its
// inverse, in `undo`, goes on the second product's sums (61 rows of 55 adapters
// of rank 64: 39.0 us; without, 38.5).
template <typename T>
__device__ __forceinline__ void make_h(const Args& a, cg::cluster_group& cluster, int ranks, float scale, float* sums, int slots, int count, T* h, int part,
                                       float* undo) {
  const int pitch = Layout<T>::pitch(a.rank), wide = pitch - 16 / (int)sizeof(T);
  if constexpr (std::is_same<T, __half>::value) {
    const int lane = threadIdx.x & 31;
    for (int s = threadIdx.x >> 5; s < slots; s += kWarps) {
      float v[kMostRank / 32], top = 0.f;
#pragma unroll
      for (int i = 0; i < kMostRank / 32; ++i) {
        if (32 * i >= a.rank) break;  // the same in all lanes
        const int r = 32 * i + lane;
        v[i] = r < a.rank && s < count ? cluster_sum(cluster, ranks, sums, r * slots + s) * scale : 0.f;
        top = fmaxf(top, fabsf(v[i]));
      }
      top = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top)));  // in the order of the numbers: none is negative
      // its exponent, not so low that the factors leave fp32's range
      const int e = max((int)(__float_as_uint(top) >> 23) - 127, -112);
      const float times = __uint_as_float((unsigned)(127 + 14 - e) << 23);
      if (lane == 0) undo[s] = __uint_as_float((unsigned)(127 - 14 + e) << 23);
#pragma unroll
      for (int i = 0; i < kMostRank / 32; ++i) {
        if (32 * i >= a.rank) break;
        T hi, lo;
        two_parts(v[i] * times, hi, lo);
        h[s * pitch + 32 * i + lane] = hi;
        h[part + s * pitch + 32 * i + lane] = lo;
      }
    }
  } else {
    for (int j = threadIdx.x; j < slots * wide; j += kThreads) {
      const int s = j / wide, r = j - s * wide;
      const float v = r < a.rank && s < count ? cluster_sum(cluster, ranks, sums, r * slots + s) * scale : 0.f;
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
}

// The factor on the sums of a slot's second product (bfloat16 parts and tf32
// ones reach as far as fp32).
template <typename T>
__device__ __forceinline__ float undo_of(const float* undo, int slot) {
  if constexpr (std::is_same<T, __half>::value) return undo[slot];
  return 1.f;
}

// A group of up to 8 rows.
template <typename T, bool WIDE>
__device__ __forceinline__ void few_rows(const Args& a, cg::cluster_group& cluster, int adapter, const int* slots, int count,
                                         int row0, int q, int of, char* smem, float* undo) {
  using L = Layout<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  constexpr int kStage = WIDE ? 1536 : 2048, kDepth = kRing / kStage;
  float4* red = reinterpret_cast<float4*>(smem + kWarps * kRing);
  T* h = reinterpret_cast<T*>(smem + kWarps * kRing + L::kRed);
  float* sums = reinterpret_cast<float*>(smem + L::sums_at(a.rank, a.most_slots));
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * kRing) + lane * 16;

  const int a_bytes = a.a_bytes, b_bytes = a.rank * (int)sizeof(T);
  const int a_pieces = (a_bytes + 63) / 64, b_pieces = (b_bytes + 63) / 64;
  const T* row = g < count ? (const T*)a.x + (long long)(row0 + slots[g]) * a.x_st : nullptr;
  const int x_shift = WIDE ? 0 : behind_16(row), x_bytes = row ? x_shift + a.inner * (int)sizeof(T) : 0;  // from the 16 bytes that the row begins in
  const char* x_first = row ? (const char*)row - x_shift : a.a;
  const char* a_first = a.a + ((long long)adapter * a.rank + g) * a.a_row;
  const char* b_first = (const char*)a.b + (long long)adapter * a.outer * b_bytes;
  const int blocks = (a.outer + 15) / 16;

  // What the copies stand at: pieces q, q + of, ... of A's blocks of 16 rows,
  // one block after the other, then all pieces of B's blocks q, q + of, ...
  int r_left = q < a_pieces ? a.rank / 16 : 0, a_at = q * 64 + t * 16, u_ahead = q, b_at = t * 16;
  const char *from_a = a_first + a_at, *from_x = x_first + a_at;
  const char* from_b = b_first + ((long long)q * 16 + g) * b_bytes + b_at;
  const long long a_back = 16 * a.a_row + q * 64 + t * 16, b_skip = (long long)of * 16 * b_bytes;
  auto copy = [&](uint32_t to) {
    if (r_left) {
      const int size = a_at < a_bytes ? 16 : 0;
      copy_async(to, from_a, size);
      copy_async(to + 512, from_a + 8 * a.a_row, size);
      copy_up_to(to + 1024, from_x, x_bytes - a_at);
      if constexpr (!WIDE) copy_up_to(to + 1536, from_x + 16, x_shift ? x_bytes - a_at - 16 : 0);
      a_at += of * 64;
      from_a += of * 64;
      from_x += of * 64;
      if (a_at - t * 16 >= a_bytes) {
        from_a += a_back - a_at;
        a_at = q * 64 + t * 16;
        from_x = x_first + a_at;
        --r_left;
      }
    } else if (u_ahead < blocks) {
      const int n = u_ahead * 16 + g, size = b_at < b_bytes ? 16 : 0;
      copy_async(to, n < a.outer ? from_b : b_first, n < a.outer ? size : 0);
      copy_async(to + 512, n + 8 < a.outer ? from_b + 8 * b_bytes : b_first, n + 8 < a.outer ? size : 0);
      b_at += 64;
      from_b += 64;
      if (b_at - t * 16 >= b_bytes) {
        from_b += b_skip + t * 16 - b_at;
        b_at = t * 16;
        u_ahead += of;
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kDepth; ++s) copy(ring + s * kStage);
  uint32_t at = ring;
  auto next = [&]() { at = at == ring + (kDepth - 1) * kStage ? ring : at + kStage; };

  for (int r0 = 0; r0 < a.rank; r0 += 16 * kFewBlocks) {
    const int some = min(kFewBlocks, (a.rank - r0) / 16);
    for (int r = 0; r < some; ++r) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int byte = q * 64 + t * 16; byte - t * 16 < a_bytes; byte += of * 64) {
        copy_wait<kDepth - 1>();
        const uint4 v[1] = {read_row<WIDE>(at + 1024, x_shift)};
        float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
        chunk_product<T, 1>(sum, read_shared(at), read_shared(at + 512), v);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += sum[0][i];
        copy(at);
        next();
      }
      red[(warp * kFewBlocks + r) * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    }
    __syncthreads();
    add_warps(red, kFewBlocks * 32, some, 1, r0, 8, sums);
    __syncthreads();
  }
  const int ranks = of / kWarps;
  if (ranks > 1) cluster.sync();
  const int pitch = L::pitch(a.rank), part = 8 * pitch;
  make_h<T>(a, cluster, ranks, a.scales[adapter], sums, 8, count, h, part, undo);
  // the others have read this CTA's sums before it writes the next ones or ends
  if (ranks > 1) cluster.sync();
  else __syncthreads();

  // outputs 16u + g and + 8 of the rows in slots 2t and 2t + 1
  const T* from[2] = {nullptr, nullptr};
  T* to[2] = {nullptr, nullptr};
  float times[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    times[i] = undo_of<T>(undo, 2 * t + i);
    if (2 * t + i < count) {
      const long long m = row0 + slots[2 * t + i];
      from[i] = a.base ? (const T*)a.base + m * a.base_st : nullptr;
      to[i] = (T*)a.out + m * a.out_st;
    }
  }
  // base is loaded two blocks ahead (and converted when it is there)
  auto load_base = [&](int u, T (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = u * 16 + g + 8 * (i >> 1);
      v[i] = from[i & 1] && n < a.outer ? from[i & 1][n] : from_float<T>(0.f);
    }
  };
  T base[3][4];
  load_base(q, base[1]);
  load_base(q + of, base[2]);
  const uint32_t h_at = (uint32_t)__cvta_generic_to_shared(h) + (g * pitch) * (int)sizeof(T) + t * 16;
  for (int u = q; u < blocks; u += of) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      base[0][i] = base[1][i];
      base[1][i] = base[2][i];
    }
    load_base(u + 2 * of, base[2]);
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
      if (to[i & 1] && n < a.outer) to[i & 1][n] = from_float<T>(fmaf(acc[i], times[i & 1], to_float<T>(base[0][i])));
    }
  }
  __syncthreads();  // h and the sums are written again for the next group
}

// Two neighbouring values of a word of a row (fp32: of two words), plus x and y times f.
__device__ __forceinline__ void add_two(unsigned* w, int i, float x, float y, float f, __half) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(w + i));
  const __half2 r = __floats2half2_rn(fmaf(x, f, v.x), fmaf(y, f, v.y));
  w[i] = *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ void add_two(unsigned* w, int i, float x, float y, float, __nv_bfloat16) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float(w[i] << 16) + x, __uint_as_float(w[i] & 0xffff0000u) + y);
  w[i] = *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ void add_two(unsigned* w, int i, float x, float y, float, float) {
  w[2 * i] = __float_as_uint(__uint_as_float(w[2 * i]) + x);
  w[2 * i + 1] = __float_as_uint(__uint_as_float(w[2 * i + 1]) + y);
}

// The second product for up to 32 rows: h [slots][pitch] in shared memory
// (16-bit: the high parts, then the low ones), MT blocks of 16 of them; the
// warp's blocks of 32 outputs u = q, q + of, ...; ring: the lane's place in
// the warp's, which begins at stage.
template <typename T, int MT, bool WIDE>
__device__ __forceinline__ void expand(const Args& a, int adapter, const T* h, int part, const int* slots, const float* undo, int count, int row0, int q, int of, uint32_t ring, T* stage) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pitch = Layout<T>::pitch(a.rank);
  const T* weights = (const T*)a.b + (long long)adapter * a.outer * a.rank;
  const int blocks = (a.outer + 31) / 32, whole = a.outer / 32;
  constexpr int WORDS = 2 * (int)sizeof(T);  // of a lane's 8 outputs
  int rows[MT][2];
  float times[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      rows[m][r] = m * 16 + g + 8 * r < count ? row0 + slots[m * 16 + g + 8 * r] : -1;
      times[m][r] = undo_of<T>(undo, m * 16 + g + 8 * r);
    }
  // Base comes through the warp's ring, several blocks ahead, 16
  // ranks' weights while the 16 before them are used.
  constexpr int PARTS = WORDS / 4 + (WIDE ? 0 : 1);  // of 16 bytes, of a lane's outputs
  constexpr int kStage = MT * 2 * PARTS * 512, kDepth = kRing / kStage;
  static_assert(kDepth >= 2, "a block ahead at least");
  int u_ahead = q;
  auto copy = [&](uint32_t to) {
    if (u_ahead < blocks && a.base) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int n = 32 * u_ahead + 8 * t;
          const char* from = (const char*)((const T*)a.base + max(rows[m][r], 0) * a.base_st + n);
          const int s = WIDE ? 0 : behind_16(from);
          const int left = rows[m][r] < 0 || n >= a.outer ? 0 : s + (a.outer - n) * (int)sizeof(T);
#pragma unroll
          for (int i = 0; i < PARTS; ++i) copy_up_to(to + ((m * 2 + r) * PARTS + i) * 512, from - s + 16 * i, left - 16 * i);
        }
    }
    u_ahead += of;
    copy_commit();
  };
  auto take_base = [&](uint32_t at, unsigned (&io)[MT][2][WORDS]) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        unsigned w[WORDS + 4];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const uint4 v = a.base ? read_shared(at + ((m * 2 + r) * PARTS + i) * 512) : make_uint4(0, 0, 0, 0);
          w[4 * i] = v.x;
          w[4 * i + 1] = v.y;
          w[4 * i + 2] = v.z;
          w[4 * i + 3] = v.w;
        }
        if constexpr (!WIDE) shift<WORDS / 4>(w, behind_16((const T*)a.base + max(rows[m][r], 0) * a.base_st));
#pragma unroll
        for (int i = 0; i < WORDS; ++i) io[m][r][i] = w[i];
      }
  };
  using Word = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
  // column c of block j is output 32u + 8 (c / 2) + 2j + c % 2
  auto load_weights = [&](int u, int k, Word (&w)[4]) {
    const int n0 = 32 * u + 8 * (g >> 1) + (g & 1);
    const T* from = weights + (long long)n0 * a.rank + k + 4 * t;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = n0 + 2 * j < a.outer ? *reinterpret_cast<const Word*>(from + 2 * j * a.rank) : Word();
  };
  unsigned io[MT][2][WORDS];
  Word next[4];
#pragma unroll
  for (int s = 0; s < kDepth; ++s) copy(ring + s * kStage);
  uint32_t ring_at = ring;
  if (q < blocks) load_weights(q, 0, next);
  for (int u = q; u < blocks; u += of) {
    float acc[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
    for (int k = 0; k < a.rank; k += 16) {
      const int at = k + 4 * t;
      Word w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = next[j];
      const bool more = k + 16 < a.rank;
      const int u_next = more ? u : u + of;
      if (u_next < blocks) load_weights(u_next, more ? k + 16 : 0, next);
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
    copy_wait<kDepth - 1>();
    take_base(ring_at, io);
    if constexpr (WIDE) copy(ring_at);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (rows[m][r] < 0) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) add_two(io[m][r], j, acc[m][j][2 * r], acc[m][j][2 * r + 1], times[m][r], T());
        if constexpr (WIDE) {
          T* to = (T*)a.out + rows[m][r] * a.out_st + 32 * u + 8 * t;
          if (u < whole) {
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i)
              __stcs(reinterpret_cast<uint4*>(to) + i, make_uint4(io[m][r][4 * i], io[m][r][4 * i + 1], io[m][r][4 * i + 2], io[m][r][4 * i + 3]));
          } else {
            const T* v = reinterpret_cast<const T*>(io[m][r]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (32 * u + 8 * t + e < a.outer) to[e] = v[e];
          }
        }
      }
    if constexpr (!WIDE) {
      // out by rows, of which a warp stores 32 neighbouring outputs at a time:
      // they change places in the stage that base has left
      T* mine = stage + (ring_at - ring) / sizeof(T);
      __syncwarp();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < WORDS / 4; ++i)
            *reinterpret_cast<uint4*>(mine + (m * 16 + g + 8 * r) * 32 + 8 * t + 16 / sizeof(T) * i) =
                make_uint4(io[m][r][4 * i], io[m][r][4 * i + 1], io[m][r][4 * i + 2], io[m][r][4 * i + 3]);
      __syncwarp();
      const int n = 32 * u + lane;
      if (n < a.outer) {
        const int some = min(count, MT * 16);
#pragma unroll 4
        for (int k = 0; k < some; ++k) ((T*)a.out)[(row0 + slots[k]) * a.out_st + n] = mine[k * 32 + lane];
      }
      __syncwarp();
      copy(ring_at);
    }
    ring_at = ring_at == ring + (kDepth - 1) * kStage ? ring : ring_at + kStage;
  }
  copy_wait<0>();
}

// Ranks r0 to r0 + 16 * RT of A's products with up to 32 rows of x, which is
// read, from L2 but for the first time, for each of them: the warp's pieces of
// x's axis q, q + of, ..., then the sums of all warps.
template <typename T, bool WIDE, int RT>
__device__ __forceinline__ void reduce(const Args& a, int adapter, const int (&rows)[4], int r0, int q, int of, uint32_t ring, char* smem, float* sums) {
  constexpr int NT = 4, kX = WIDE ? 512 : 1024, kStage = RT * 1024 + NT * kX, kDepth = kRing / kStage;
  static_assert(kDepth >= 2, "a piece ahead at least");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int bytes = a.a_bytes, pieces = (bytes + 63) / 64, x_bytes = a.inner * (int)sizeof(T);
  const char* weights = a.a + ((long long)adapter * a.rank + r0 + g) * a.a_row;
  int c_ahead = q;
  auto copy = [&](uint32_t to) {
    if (c_ahead < pieces) {
      const int at = c_ahead * 64 + t * 16;
      const int size = at < bytes ? 16 : 0;
#pragma unroll
      for (int r = 0; r < 2 * RT; ++r) copy_async(to + r * 512, weights + r * 8 * a.a_row + at, size);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const char* from = (const char*)((const T*)a.x + max(rows[n], 0) * a.x_st);
        const int s = WIDE ? 0 : behind_16(from), left = rows[n] >= 0 ? s + x_bytes - at : 0;
        from += at - s;
        copy_up_to(to + RT * 1024 + n * kX, from, left);
        if constexpr (!WIDE) copy_up_to(to + RT * 1024 + 512 + n * kX, from + 16, s ? left - 16 : 0);
      }
      c_ahead += of;
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kDepth; ++s) copy(ring + s * kStage);
  uint32_t at = ring;
  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
  for (int c = q; c < pieces; c += of) {
    copy_wait<kDepth - 1>();
    uint4 v[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) v[n] = read_row<WIDE>(at + RT * 1024 + n * kX, behind_16((const T*)a.x + max(rows[n], 0) * a.x_st));
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float sum[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
      chunk_product<T, NT>(sum, read_shared(at + r * 1024), read_shared(at + r * 1024 + 512), v);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] += sum[n][i];
    }
    copy(at);
    at = at == ring + (kDepth - 1) * kStage ? ring : at + kStage;
  }
  copy_wait<0>();
  __syncwarp();
  float4* red = reinterpret_cast<float4*>(smem);  // in the warps' rings
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
      red[warp * (kRing / 16) + (r * NT + n) * 32 + lane] = make_float4(acc[r][n][0], acc[r][n][1], acc[r][n][2], acc[r][n][3]);
  __syncthreads();
  add_warps(red, kRing / 16, RT * NT, NT, r0, 8 * NT, sums);
  __syncthreads();
}

// A group of 9 to 32 rows.
template <typename T, bool WIDE, int RT>
__device__ __forceinline__ void many_rows(const Args& a, cg::cluster_group& cluster, int adapter, const int* slots, int count,
                                          int row0, int q, int of, char* smem, float* undo) {
  using L = Layout<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  constexpr int NT = 4;
  float* sums = reinterpret_cast<float*>(smem + L::sums_at(a.rank, a.most_slots));
  T* h = reinterpret_cast<T*>(smem + kWarps * kRing);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * kRing) + lane * 16;
  int rows[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) rows[n] = n * 8 + g < count ? row0 + slots[n * 8 + g] : -1;

  int r0 = 0;
  if constexpr (RT > 1)
    for (; r0 + 16 * RT <= a.rank; r0 += 16 * RT) reduce<T, WIDE, RT>(a, adapter, rows, r0, q, of, ring, smem, sums);
  for (; r0 < a.rank; r0 += 16) reduce<T, WIDE, 1>(a, adapter, rows, r0, q, of, ring, smem, sums);
  const int ranks = of / kWarps;
  if (ranks > 1) cluster.sync();
  const int part = 32 * L::pitch(a.rank);
  make_h<T>(a, cluster, ranks, a.scales[adapter], sums, 32, count, h, part, undo);
  // the others have read this CTA's sums before it writes the next ones or ends
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  T* stage = reinterpret_cast<T*>(smem + warp * kRing);
  if constexpr (sizeof(T) == 2) {
    if (count <= 16) expand<T, 1, WIDE>(a, adapter, h, part, slots, undo, count, row0, q, of, ring, stage);
    else expand<T, 2, WIDE>(a, adapter, h, part, slots, undo, count, row0, q, of, ring, stage);
  } else {  // (two blocks of fp32 rows do not fit the registers)
    for (int s = 0; s < count; s += 16) expand<T, 1, WIDE>(a, adapter, h + s * L::pitch(a.rank), part, slots + s, undo + s, count - s, row0, q, of, ring, stage);
  }
  __syncthreads();  // h and the sums are written again for the next group
}

// The rows in `slots` from base to out, or zeros: a warp takes 32 * 4 units of
// 16 bytes, or values, of a row, loads all of them and stores them (3630 rows of
// 72 to 2304, of which 403 have no adapter, fp16: 17.6 us; row by row, value by
// value 53).
template <typename T, typename U>
__device__ __forceinline__ void copy_rows(const Args& a, const int* slots, int count, int row0, int q, int of) {
  constexpr int EACH = sizeof(U) / sizeof(T), BATCH = 4;
  const int lane = threadIdx.x & 31, units = a.outer / EACH, spans = (units + 32 * BATCH - 1) / (32 * BATCH);
  for (long long i = q; i < (long long)count * spans; i += of) {
    const int k = (int)(i / spans), n0 = (int)(i - (long long)k * spans) * 32 * BATCH + lane;
    const long long row = row0 + slots[k];
    const U* from = a.base ? reinterpret_cast<const U*>((const T*)a.base + row * a.base_st) : nullptr;
    U* to = reinterpret_cast<U*>((T*)a.out + row * a.out_st);
    U v[BATCH];
#pragma unroll
    for (int e = 0; e < BATCH; ++e) v[e] = from && n0 + 32 * e < units ? from[n0 + 32 * e] : U();
#pragma unroll
    for (int e = 0; e < BATCH; ++e)
      if (n0 + 32 * e < units) to[n0 + 32 * e] = v[e];
  }
  if constexpr (EACH > 1)  // what is left of a row
    for (int k = q; k < count; k += of) {
      const long long row = row0 + slots[k];
      const int n = units * EACH + lane;
      if (n < a.outer) ((T*)a.out)[row * a.out_st + n] = a.base ? ((const T*)a.base)[row * a.base_st + n] : from_float<T>(0.f);
    }
}

// RT: blocks of 16 ranks that many rows' first product takes at a time, two
// where the rank has them (8191 rows of five prompts, 4096 to 4096, rank 64,
// bf16: 97.9 us with one, 88.4 with two; fp32: 259 and 236, though it spills).
// Rows that are shifted leave no room for two in the rings, and a kernel with
// the second block's registers took 1.4 us more of the 45 of rank 16.
template <typename T, bool WIDE, int RT>
__global__ void __launch_bounds__(kThreads, 2) adapters_kernel(Args a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ int slots[kTile];
  __shared__ float undo[kTile];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int unit = (int)(blockIdx.x / ranks), row0 = unit % a.tiles * kTile;
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
  const bool alone = a.apart && groups > a.per_tile;  // the same in all CTAs of the cluster
  const int first_group = alone ? unit / a.tiles * ranks + rank : unit / a.tiles, step = alone ? a.per_tile * ranks : a.per_tile;
  const int q = alone ? warp : rank * kWarps + warp, of = alone ? kWarps : ranks * kWarps;
  for (int i = first_group; i < groups; i += step) {
    unsigned left = firsts;
    for (int k = 0; k < i; ++k) left &= left - 1;
    const int leader = __ffs(left) - 1;
    const unsigned members = __shfl_sync(~0u, same, leader);
    const int adapter = __shfl_sync(~0u, mine, leader), count = __popc(members);
    if (adapter < 0 && a.out == a.base && a.out_st == a.base_st) continue;  // rows without one are there
    if (warp == 0 && (members >> lane & 1)) slots[__popc(members & ((1u << lane) - 1))] = lane;
    __syncthreads();
    if (adapter < 0) {
      copy_rows<T, typename std::conditional<WIDE, uint4, T>::type>(a, slots, count, row0, q, of);
      __syncthreads();  // the slots are written again
    } else if (count <= 8) {
      few_rows<T, WIDE>(a, cluster, adapter, slots, count, row0, q, of, smem, undo);
    } else {
      many_rows<T, WIDE, RT>(a, cluster, adapter, slots, count, row0, q, of, smem, undo);
    }
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

template <typename T, bool WIDE, int RT>
void launch_typed(Args& a, int64_t ctas, int ranks, cudaStream_t stream) {
  static std::once_flag once[64];
  std::call_once(once[current_device()], [] {
    PFB_CUDA(cudaFuncSetAttribute(adapters_kernel<T, WIDE, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<T>::bytes(kMostRank, kTile)));
  });
  launch_following<Args>(adapters_kernel<T, WIDE, RT>, dim3((unsigned)ctas), kThreads, (size_t)Layout<T>::bytes(a.rank, a.most_slots), stream, a,
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
  a.a_bytes = (int)round_up(p.inner * es, 16);
  a.b = p.b;
  a.scales = p.scales;
  a.err = p.err;
  auto wide = [&](const void* p, int64_t st) { return (uintptr_t)p % 16 == 0 && st * es % 16 == 0; };
  const bool all_wide = wide(a.x, a.x_st) && wide(a.out, a.out_st) && wide(a.base, a.base_st);
  a.most_slots = p.rows <= 8 ? 8 : 32;
  // A tile has up to as many groups as rows or adapters.  A cluster for all of
  // them, as long as these do not become thousands of CTAs: the first groups
  // of all tiles in front, so that those of prompts start at once, then the
  // others, which end at once where there are none (one cluster a tile took 82
  // us for the 60 of prompts of 8191 rows: two groups where prompts meet, one
  // after the other).
  const int64_t tiles = ceil_div(p.rows, kTile), groups = std::min<int64_t>({kTile, p.rows, p.adapters + 1});
  const int64_t sms = device_sm_count(current_device());
  a.tiles = (int)tiles;
  a.per_tile = (int)std::min(groups, std::max<int64_t>(1, 2048 / tiles));
  int64_t units = tiles * a.per_tile;
  PFB_CHECK_ARG(units <= INT32_MAX / kMostRanks, "adapters: too many rows");
  // few groups: several CTAs each, as many as the device holds at once, as long
  // as all warps have something of one of the products
  const int64_t work = std::max(ceil_div(a.a_bytes, 64), ceil_div(p.outer, 32));
  int ranks = 1;
  while (ranks < kMostRanks && units * ranks <= sms && work > ranks * kWarps) ranks *= 2;
  // Many groups at most, but tiles of one or two would leave the device idle:
  // the two CTAs of a cluster work on a group together or, where a tile has
  // more groups than clusters, on one each.  4096 to 4096, rank 16, bf16, us
  // with one CTA and with two: 3000 rows of five prompts 33.8 and 23.7, 1200
  // 21.8 and 15.0; 3000 mixed rows of 16 adapters 126.8 and 132.9 (four CTAs:
  // 1200 rows of prompts 17.2, of mixed adapters 61.7 for 48.4).
  if (ranks == 1 && tiles <= sms && work > kWarps) {
    ranks = 2;
    a.apart = 1;
    a.per_tile = (int)ceil_div(a.per_tile, 2);
    units = tiles * a.per_tile;
  }
  auto launch = [&](auto t) {
    if (!all_wide) launch_typed<decltype(t), false, 1>(a, units * ranks, ranks, stream);
    else if (p.rank < 32 || p.rows <= 8) launch_typed<decltype(t), true, 1>(a, units * ranks, ranks, stream);
    else launch_typed<decltype(t), true, 2>(a, units * ranks, ranks, stream);
  };
  if (p.dtype == PFC_DTYPE_FLOAT32) launch(float());
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch(__half());
  else launch(__nv_bfloat16());
}

}  // namespace pfb
