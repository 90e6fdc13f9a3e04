// linear_w4.cu — products with 4-bit weights for single tokens and small
// batches.
//
//   y[m,n] = sum_g s[n,g] sum_{k in g} x[m,k] (q[n,k] - z[n,g])  (+ bias[n])
//
// The weights are read once for up to 48 rows of x (16 in fp32; more rows
// read and unpack them again for each such chunk), at half a byte each; with
// few rows that read bounds the product, so the arithmetic must cost little
// per weight.  It runs on mma.sync: q - z is an integer of at most 5 bits,
// exact in fp16 and bf16, and so are 16-bit values of x; the products
// accumulate in fp32 over a group and the group's sum is multiplied by its
// scale in fp32, so no weight is ever rounded.  fp32 x enters as three bf16
// parts (8 bits each, 24 in all), which take three columns of the instruction
// instead of three instructions.  Two weights cost one logic operation and
// one subtraction: a nibble pair OR-ed into the mantissas of two 16-bit
// numbers of value 2^10 is 2^10 + q in fp16, from which 2^10 + z is
// subtracted exactly; in bf16 it is 2^-4 + 2^-11 q, and the result is
// multiplied by 2^11.
//
// A lane holds 16 bytes of each of two weight rows in a block of 128 columns:
// the arranged layout gives it 8 columns of each of the four 32-column groups,
// so that no instruction mixes two groups, and puts a warp's 1 KB together
// (with whole rows in turn every load was eight pieces of 64 bytes: one fp32
// row times 16384 x 4096 weights 22.3 us for 19.7 at that stage).
//
// Three shapes of CTA, 8 warps each:
//   few rows of x (8 columns of the instruction): the warps share the columns
//   of 16 weight rows, or in pairs those of 64; a CTA walks over row tiles and
//   keeps its part of x, which is staged once (again for each tile, through
//   two buffers, where it does not fit);
//   more, and weight rows that fill the device: 128 weight rows (32 a warp, so
//   that a fragment of x read from shared memory serves two instructions), in
//   pairs over the columns, x in chunks through two buffers;
//   more, and fewer weight rows: 32 weight rows, four warps over the columns.
// Weights, scales and zeros reach a warp through a ring of its own in shared
// memory, filled by asynchronous copies several steps ahead.  Where the rows
// alone do not fill the device, the CTAs of a cluster share the columns and
// add their sums through distributed shared memory, in the order of their
// ranks: results do not depend on timing and nothing needs a workspace.
//
// Measured (device time in a stream of calls; the bytes at 6.4 TB/s in
// brackets): one bf16 row, 4096 x 4096, groups of 128: 4.7 us (1.4), latency:
// no load is on its way before the kernel in front has ended; one fp32 row,
// 16384 x 4096, groups of 64: 14.2 us (5.8), of which its 7.4 M instructions
// would take 6.6 at full issue, but 256 tiles leave 40 SMs with one CTA and
// give 108 two, and the 13 warps of an SM that are there on average issue in
// 56% of the cycles; 33 fp16 rows, 4096 x 16384, groups of 32: 32.7 us (6.4),
// the tensor pipe 34% busy, the rest latency between the instructions of two
// warps a scheduler (16 narrower warps measured the same).
#include <cooperative_groups.h>
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

constexpr int kBlock = 128;  // columns of a warp's step
constexpr int kPad = 32;     // values between rows of x in shared memory: rows start 64 bytes apart mod 128
constexpr int kSmemMost = 220 * 1024;
constexpr int kSmemHalf = 112 * 1024;  // two CTAs an SM

struct Args {
  const void* x;
  long long x_st;
  void* y;
  long long y_st;
  const uint4* weight;
  const unsigned* meta;
  const void* bias;
  int rows, inner, outer;
  int blocks;        // of 128 columns
  int part_blocks;   // of a cluster's CTA
  int row_blocks;    // of 16 weight rows
  int groups;        // of a row, for groups of 128 and more
  int group_blocks;  // blocks that share a scale, for groups of 128 and more
  int chunk;         // rows of x that a CTA takes
  int tile;          // columns of x in a buffer
  int whole;         // the CTA's columns of x fit one buffer, staged once
  int vector;        // rows of x are 16-byte aligned
  int tiles;         // of weight rows
};

template <typename T>
struct Num {  // 16-bit type of the products, its magic number for 4-bit integers and their unit, and the parts of x
  using N = __nv_bfloat16;
  using N2 = __nv_bfloat162;
  // 2^-4, in whose mantissa a unit is 2^-11: q - z enters as its 2^-11th, and a
  // sum of 128 columns, at most 15 * 128 of the largest x, stays in fp32's
  // range whatever x is.  Nothing is lost at the other end: with x in steps of
  // bf16's smallest, 2^-133, the products are in steps of 2^-144, and fp32's
  // smallest is 2^-149.  (Results below 2^-115 come in steps of 2^-138.)
  static constexpr unsigned kMagic = 0x3d803d80u;
  static constexpr float kUnit = 2048.f;
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  static __device__ __forceinline__ N of(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // c = the product, with nothing added
  static __device__ __forceinline__ void mma_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
};
template <>
struct Num<__half> {
  using N = __half;
  using N2 = __half2;
  static constexpr unsigned kMagic = 0x64006400u;  // 1024; sums of fp16 products are far inside fp32's range
  static constexpr float kUnit = 1.f;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ N of(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // c = the product, with nothing added
  static __device__ __forceinline__ void mma_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
};

// A group's word: the scale's fp32 bits (of fp16 or bf16, so the lowest 13 are
// 0), with the zero in the lowest four.
__device__ __forceinline__ float scale_of(unsigned meta) { return __uint_as_float(meta & ~15u); }

// (u & 0x000f000f) | magic in one instruction: two nibbles as 16-bit numbers
// (written out, it became two: only one of the constants fits the instruction)
__device__ __forceinline__ unsigned with_magic(unsigned u, unsigned magic) {
  unsigned r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(u), "r"(0x000f000fu), "r"(magic));
  return r;
}

// c += s * p in pairs
__device__ __forceinline__ void fma2(float& c0, float& c1, float s, float p0, float p1) {
  asm("{\n\t.reg .b64 c, s, p;\n\tmov.b64 c, {%0, %1};\n\tmov.b64 s, {%2, %2};\n\tmov.b64 p, {%3, %4};\n\t"
      "fma.rn.f32x2 c, s, p, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(c0), "+f"(c1)
      : "f"(s), "f"(p0), "f"(p1));
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

__device__ __forceinline__ unsigned word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// Eight values in as many 16-bit parts as their type needs.
template <typename T>
__device__ __forceinline__ void store_parts(typename Num<T>::N* dst, int between, const T (&v)[8]) {
  using M = Num<T>;
  if constexpr (M::kParts == 1) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
  } else {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = v[e] + 0.f;  // a NaN has its highest bit set, and stays one when cut off
#pragma unroll
    for (int p = 0; p < M::kParts; ++p) {
      unsigned w[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if (p == 0) {  // cut off: fp32 has finite numbers that bf16 would round to an infinity
          w[e / 2] = __byte_perm(__float_as_uint(rest[e]), __float_as_uint(rest[e + 1]), 0x7632);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(rest[e], rest[e + 1]);
          w[e / 2] = *reinterpret_cast<const unsigned*>(&h);
        }
        const float x = rest[e] - __uint_as_float(w[e / 2] << 16), y = rest[e + 1] - __uint_as_float(w[e / 2] & 0xffff0000u);
        rest[e] = isfinite(x) ? x : 0.f;  // an infinity or NaN is the first part
        rest[e + 1] = isfinite(y) ? y : 0.f;
      }
      *reinterpret_cast<uint4*>(dst + p * between) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// `width` columns of the CTA's rows of x from column k0 on into a buffer, as
// 16-bit parts: part p of row r in row p*rows + r; zeros behind the last
// column.  16-bit rows that are aligned go by asynchronous copies, to be
// waited for; width is a multiple of 128.  A warp takes rows, or warps share
// one, 256 columns at a time, with several copies on their way (a division
// and a jump for each took 10.2 us to 15.1 with 40 rows of 8000 x 1000).
template <typename T, int W>
__device__ __noinline__ void stage(const T* x, long long x_st, int inner, int vector, typename Num<T>::N* xs, int pitch,
                                   int rows, int k0, int width) {
  using M = Num<T>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int log = rows >= 5 ? 0 : rows >= 3 ? 1 : rows == 2 ? 2 : 3, share = 1 << log;  // warps of a row
  static_assert(W == 8, "the table above is for 8 warps");
  const int first = warp >> log, stride = W >> log;
  const int sure = vector ? min(width, max(0, inner - k0)) & ~7 : 0;  // columns in whole aligned pieces
  for (int r = first; r < rows; r += stride) {
    const T* src = x + r * x_st + k0;
    typename M::N* dst = xs + r * pitch;
    int c = ((warp - first * share) * 32 + lane) * 8;
    if constexpr (M::kParts == 1) {
#pragma unroll 4
      for (; c < sure; c += share * 256) copy16(dst + c, src + c);
    } else {
#pragma unroll 2
      for (; c < sure; c += share * 256) {
        alignas(16) T v[8];
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; ++e) reinterpret_cast<uint4*>(v)[e] = reinterpret_cast<const uint4*>(src + c)[e];
        store_parts<T>(dst + c, rows * pitch, v);
      }
    }
    for (; c < width; c += share * 256) {
      alignas(16) T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k0 + c + e < inner ? src[c + e] : T(0.f);
      store_parts<T>(dst + c, rows * pitch, v);
    }
  }
}

// NT: 8-column blocks of x rows (times parts).  G: columns that share a scale
// within a block: 32, 64, or 128 for groups of 128 and more.  MT: 16-row
// blocks of a warp.  RW: warps along the weight rows; the others share the
// columns.
template <typename T, int NT, int G, int MT, int RW>
struct Shape {
  static constexpr bool kMany = NT > 1;             // rows of x: one tile a CTA, x in chunks
  static constexpr int kWarps = 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kAcross = kWarps / RW;       // warps along the columns
  static constexpr int kRows = 16 * MT * RW;        // weight rows of a tile
  static constexpr int kStep = kBlock * kAcross;    // columns of a CTA's step
  static constexpr int kDepth = kMany ? 4 : 6;     // slots of a warp's ring; all but one are on their way
  static constexpr int kWords = kBlock / G;         // meta words of a block's row
  static constexpr int kSlot = MT * (1024 + 64 * kWords);
  static constexpr int kRing = kDepth * kSlot;
  static constexpr int kPitch = NT * 8 + 4;
  static constexpr size_t ring_bytes = (size_t)kWarps * kRing;
  static constexpr size_t red_bytes = (size_t)kAcross * kRows * kPitch * 4;
};

template <typename T, int NT, int G, int MT, int RW>
__global__ void __launch_bounds__((Shape<T, NT, G, MT, RW>::kThreads), (Shape<T, NT, G, MT, RW>::kMany ? 1 : 2)) linear_kernel(Args a) {
  using M = Num<T>;
  using N = typename M::N;
  using N2 = typename M::N2;
  using S = Shape<T, NT, G, MT, RW>;
  constexpr int MW = S::kWords, D = S::kDepth;
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  char* ring = smem + warp * S::kRing;
  N* xs = reinterpret_cast<N*>(smem + S::ring_bytes + (S::kMany ? 0 : S::red_bytes));
  float* red = reinterpret_cast<float*>(smem + S::ring_bytes);  // [across][rows][kPitch]; of a single tile in x's place
  const int rw = warp % RW, kw = warp / RW;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long first = (long long)blockIdx.y * a.chunk;
  const int rows = (int)min((long long)a.chunk, a.rows - first);
  const int cols = rows * M::kParts, pitch = a.tile + kPad;
  const int b0 = rank * a.part_blocks, b1 = min(b0 + a.part_blocks, a.blocks);  // this CTA's blocks
  const int steps = (a.part_blocks + S::kAcross - 1) / S::kAcross;              // of a tile, the same in all warps
  const int stride = gridDim.x / ranks;
  const int per_buffer = a.tile / S::kStep;
  const size_t buffer = (size_t)cols * pitch;

  auto stage_from = [&](int step) {  // the buffer's columns from a step of the tile on
    const int k = (b0 + step * S::kAcross) * kBlock;
    const int width = min(a.tile, (b1 - b0) * kBlock - step * S::kStep);
    if (width > 0)
      stage<T, S::kWarps>((const T*)a.x + first * a.x_st, a.x_st, a.inner, a.vector, xs + (a.whole ? 0 : (step / per_buffer & 1) * buffer), pitch, rows, k, width);
  };
  begin();
  stage_from(0);
  commit();

  // of the next fetch: its tile, the step there, its block, its slot, and
  // where the weights and words of its rows are (the host checked that these
  // offsets fit 32 bits)
  int f_tile = (int)blockIdx.x / ranks, f_step = 0, f_block, f_slot = 0;
  unsigned f_w[MT], f_m[MT];
  auto aim = [&]() {
    f_block = b0 + kw;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      // blocks of 16 rows behind the last repeat it and are not stored
      const unsigned n = min(f_tile * S::kRows / 16 + rw * MT + mt, a.row_blocks - 1);
      f_w[mt] = (n * a.blocks + f_block) * 64 + lane;
      f_m[mt] = G == 128 ? n * a.groups * 16 : (n * a.blocks + f_block) * 16 * MW;
    }
  };
  aim();
  auto fetch = [&]() {
    char* to = ring + f_slot * S::kSlot;
    if (f_block < b1) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        copy16(to + mt * 1024 + lane * 16, a.weight + f_w[mt]);
        copy16(to + mt * 1024 + 512 + lane * 16, a.weight + f_w[mt] + 32);
        if (lane < 4 * MW)
          copy16(to + MT * 1024 + mt * 64 * MW + lane * 16,
                 a.meta + f_m[mt] + (G == 128 ? 16 * (a.group_blocks == 1 ? f_block : f_block / a.group_blocks) : 0) + lane * 4);
      }
    }
    commit();  // empty or not: the waits count groups
    f_slot = f_slot + 1 == D ? 0 : f_slot + 1;
    f_block += S::kAcross;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f_w[mt] += S::kAcross * 64;
      if (G != 128) f_m[mt] += S::kAcross * 16 * MW;
    }
    if (++f_step == steps) {
      f_step = 0;
      f_tile += stride;
      if (f_tile < a.tiles) aim();
      else f_block = b1, f_step = INT32_MIN;  // nothing more
    }
  };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) fetch();

  int at[NT];  // the lane's columns of x; those behind the last repeat it, and what they give is not read
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) at[nt] = min(nt * 8 + g, cols - 1) * pitch;
  int slot = 0;

  for (int tile = (int)blockIdx.x / ranks; tile < a.tiles; tile += stride) {
    const bool again = tile != (int)blockIdx.x / ranks;
    float acc[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[mt][nt][r] = 0.f;
    int in_buffer = a.whole && again ? 1 : 0;  // steps into the buffer; 0: wait for it
    const N* xk = xs + kw * kBlock + t * 8;
    for (int step = 0; step < steps; ++step) {
      if (in_buffer == 0) {
        // This buffer was staged per_buffer steps ago, before as many groups
        // of the ring: the wait for this step's slot covers it unless that is
        // fewer than stay pending.
        if ((again && step == 0) || per_buffer < D - 2) wait_copies<0>();
        else wait_copies<D - 2>();
        __syncthreads();  // this buffer is filled, and the other one's reads are over
        if (!a.whole) {
          if (step) xk += ((step / per_buffer & 1) ? (long long)buffer : -(long long)buffer) - per_buffer * S::kStep;
          if (step + per_buffer < steps) {
            stage_from(step + per_buffer);
            commit();
          }
        }
      }
      wait_copies<D - 2>();
      __syncwarp();  // the slot's words are there for all lanes, and the slot before it has been read
      fetch();
      if (b0 + step * S::kAcross + kw < b1) {
        const uint4* ws = reinterpret_cast<const uint4*>(ring + slot * S::kSlot) + lane;
        const unsigned* mp = reinterpret_cast<const unsigned*>(ring + slot * S::kSlot + MT * 1024) + g * MW;
        uint4 w[MT][2];
        unsigned meta[MT][2][MW];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[mt][h] = ws[mt * 64 + h * 32];
            const unsigned* m = mp + (mt * 16 + h * 8) * MW;
            if constexpr (MW == 4) {
              const uint4 u = *reinterpret_cast<const uint4*>(m);
              meta[mt][h][0] = u.x, meta[mt][h][MW / 4] = u.y, meta[mt][h][MW / 2] = u.z, meta[mt][h][MW - 1] = u.w;
            } else if constexpr (MW == 2) {
              const uint2 u = *reinterpret_cast<const uint2*>(m);
              meta[mt][h][0] = u.x, meta[mt][h][MW - 1] = u.y;
            } else {
              meta[mt][h][0] = *m;
            }
          }
        // With many columns of x the scales are applied every 32 weight columns,
        // whatever the group: sums of a whole group would not fit the registers.
        constexpr int GG = S::kMany ? 32 : G;
        float part[MT][NT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // 32 columns
          unsigned f1[MT][4], f2[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned zz = (meta[mt][h][j * 32 / G] & 15u) * 0x10001u + M::kMagic;
              const N2 z = *reinterpret_cast<const N2*>(&zz);
              const unsigned u = word(w[mt][h], j);
              unsigned q[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const unsigned p = with_magic(u >> (4 * e), M::kMagic);
                const N2 d = __hsub2(*reinterpret_cast<const N2*>(&p), z);
                q[e] = *reinterpret_cast<const unsigned*>(&d);
              }
              f1[mt][h] = q[0];
              f1[mt][h + 2] = q[1];
              f2[mt][h] = q[2];
              f2[mt][h + 2] = q[3];
            }
          // two instructions a column block and 16 rows; those of one sum are
          // kept apart (next to each other each waits for the one before it)
          uint4 b[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            b[nt] = *reinterpret_cast<const uint4*>(xk + at[nt] + j * 32);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              if (j * 32 % GG == 0) M::mma_first(part[mt][nt], f1[mt], b[nt].x, b[nt].y);
              else M::mma(part[mt][nt], f1[mt], b[nt].x, b[nt].y);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) M::mma(part[mt][nt], f2[mt], b[nt].z, b[nt].w);
          if ((j + 1) * 32 % GG == 0) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const float ca = scale_of(meta[mt][0][j * 32 / G]), cb = scale_of(meta[mt][1][j * 32 / G]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                fma2(acc[mt][nt][0], acc[mt][nt][1], ca, part[mt][nt][0], part[mt][nt][1]);
                fma2(acc[mt][nt][2], acc[mt][nt][3], cb, part[mt][nt][2], part[mt][nt][3]);
              }
            }
          }
        }
      }
      slot = slot + 1 == D ? 0 : slot + 1;
      xk += S::kStep;
      if (++in_buffer == per_buffer && !a.whole) in_buffer = 0;
    }

    // the tile is done: add the warps' sums, accumulator (row g or g + 8,
    // column 2t or 2t + 1), then the cluster's
    const int n0 = tile * S::kRows;
    __syncthreads();  // the previous tile's sums have been read, and all of x
    if (!S::kMany && !a.whole && tile + stride < a.tiles) {
      stage_from(0);
      commit();
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          red[(kw * S::kRows + (rw * MT + mt) * 16 + g + 8 * (r >> 1)) * S::kPitch + nt * 8 + 2 * t + (r & 1)] = acc[mt][nt][r];
    __syncthreads();
    int n_first = 0, n_count = S::kRows, sums = S::kAcross;
    if (ranks > 1) {  // each rank adds up a share of the tile's rows, 16 bytes at a time
      const int quads = (cols + 3) / 4;
      auto quad = [&](const float* of, int w, int n, int c) -> float4 {
        return *reinterpret_cast<const float4*>(of + (w * S::kRows + n) * S::kPitch + c);
      };
      auto add = [](float4& x, const float4& y) { x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w; };
      if constexpr (S::kAcross > 1) {
        for (int j = tid; j < S::kRows * quads; j += S::kThreads) {
          const int n = j % S::kRows, c = j / S::kRows * 4;
          float4 v = quad(red, 0, n, c);
#pragma unroll
          for (int w = 1; w < S::kAcross; ++w) add(v, quad(red, w, n, c));
          *reinterpret_cast<float4*>(red + n * S::kPitch + c) = v;  // read and written by this thread alone
        }
      }
      cluster.sync();
      n_count = S::kRows / ranks;
      n_first = rank * n_count;
      sums = 1;
      for (int j = tid; j < n_count * quads; j += S::kThreads) {
        const int n = n_first + j % n_count, c = j / n_count * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int r = 0; r < ranks; ++r) add(v, quad(cluster.map_shared_rank(red, r), 0, n, c));
        *reinterpret_cast<float4*>(red + n * S::kPitch + c) = v;  // only this rank reads this share
      }
      cluster.sync();
    }
    for (int j = tid; j < n_count * rows; j += S::kThreads) {
      const int m = j / n_count, n = n_first + j % n_count;
      if (n0 + n >= a.outer) continue;
      float v = 0.f;
#pragma unroll
      for (int p = M::kParts - 1; p >= 0; --p) {
        const float* of = red + n * S::kPitch + p * rows + m;
        for (int w = 0; w < sums; ++w) v += of[w * S::kRows * S::kPitch];
      }
      v *= M::kUnit;
      if (a.bias) v += (float)((const T*)a.bias)[n0 + n];
      ((T*)a.y)[(long long)(first + m) * a.y_st + n0 + n] = T(v);
    }
  }
}

struct ArrangeArgs {
  const uint8_t* packed;
  const unsigned short* scales;
  const uint8_t* zeros;
  uint32_t* weight;
  uint32_t* meta;
  long long words, metas;  // of the outputs
  int inner, outer, blocks, groups, group, bf16;
};

__global__ void arrange_kernel(const ArrangeArgs a) {
  const long long step = (long long)gridDim.x * blockDim.x, start = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long pitch = (a.inner + 1) / 2;
  for (long long i = start; i < a.words; i += step) {
    const int j = (int)(i & 3), t = (int)(i >> 2 & 3), r = (int)(i >> 4 & 15);  // r: half * 8 + g
    const long long rb = (i >> 8) / a.blocks, row = rb * 16 + r;
    const int col = (int)((i >> 8) - rb * a.blocks) * kBlock + j * 32 + t * 8;
    uint32_t u = 0;
    for (int e = 0; e < 8; ++e) {
      const int k = col + e;
      const unsigned q = row < a.outer && k < a.inner ? (a.packed[row * pitch + (k >> 1)] >> (4 * (k & 1))) & 15u : 0u;
      // even columns in nibbles 0-3, odd ones in 4-7
      u |= q << (4 * ((e >> 1) + 4 * (e & 1)));
    }
    a.weight[i] = u;
  }
  const int mw = a.group < kBlock ? kBlock / a.group : 1;             // words of a row in a step
  const int along = a.group < kBlock ? a.blocks : a.groups;           // steps
  for (long long i = start; i < a.metas; i += step) {
    const long long rb = i / mw / 16 / along, row = rb * 16 + i / mw % 16;
    const int m = (int)(i / mw / 16 - rb * along) * mw + (int)(i % mw);  // the group
    uint32_t u = 0;
    if (row < a.outer && m < a.groups) {
      const unsigned short b = a.scales[row * a.groups + m];
      const float f = a.bf16 ? __uint_as_float((unsigned)b << 16) : __half2float(__ushort_as_half(b));
      // a NaN stays one without its lowest bits
      u = (isnan(f) ? 0x7fc00000u : __float_as_uint(f)) | (a.zeros ? a.zeros[row * a.groups + m] & 15u : 8u);
    }
    a.meta[i] = u;
  }
}

// CTAs of a cluster: the columns are shared as long as that fills the device
// and leaves each CTA two steps.
int ranks_of(int64_t tiles, int64_t slots, int64_t blocks, int across) {
  int ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= slots && blocks >= ranks * 2 * 2 * across) ranks *= 2;
  return ranks;
}

template <typename T, int NT, int G, int MT, int RW>
void launch_sized(Args a, cudaStream_t stream) {
  using S = Shape<T, NT, G, MT, RW>;
  const auto kernel = linear_kernel<T, NT, G, MT, RW>;
  static std::once_flag once[64];
  const int dev = current_device(), sms = device_sm_count(dev);
  std::call_once(once[dev], [&] {
    PFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost));
  });
  a.tiles = (int)ceil_div(a.outer, S::kRows);
  const int64_t slots = (S::kMany ? 1 : 2) * (int64_t)sms;
  const int ranks = ranks_of(a.tiles, slots, a.blocks, S::kAcross);
  a.part_blocks = (int)ceil_div(a.blocks, ranks);
  const int cols = a.chunk * Num<T>::kParts;
  const int64_t mine = round_up((int64_t)a.part_blocks * kBlock, S::kStep);
  auto bytes = [&](int64_t width) { return (int64_t)cols * (width + kPad) * 2; };
  // a CTA's part of x in one buffer, where as many CTAs still fit an SM
  constexpr int64_t fixed = (int64_t)S::ring_bytes + (S::kMany ? 0 : (int64_t)S::red_bytes);
  constexpr int64_t room = (S::kMany ? (int64_t)kSmemMost : kSmemHalf) - fixed;
  a.whole = bytes(mine) <= room;
  int64_t width = mine;
  if (!a.whole) {
    width = S::kStep;
    while (width + S::kStep < mine && width < 2048 && 2 * bytes(width + S::kStep) <= room) width += S::kStep;
  }
  a.tile = (int)width;
  const int64_t x_bytes = (a.whole ? 1 : 2) * bytes(width);
  const int64_t smem = fixed + (S::kMany ? std::max<int64_t>(x_bytes, S::red_bytes) : x_bytes);
  PFB_CHECK_ARG(smem <= kSmemMost, "linear w4: tile does not fit");
  // a CTA walks over row tiles (few rows of x), keeping x
  const int64_t wave = std::max<int64_t>(1, slots / ranks);
  const int64_t across = S::kMany ? a.tiles : std::min<int64_t>(a.tiles, wave);
  launch_following<Args>(kernel, dim3((unsigned)(across * ranks), (unsigned)ceil_div(a.rows, a.chunk)), S::kThreads, (size_t)smem, stream, a, ranks);
}

template <typename T>
void launch_typed(Args& a, int64_t group, cudaStream_t stream) {
  constexpr int parts = Num<T>::kParts;
  const int64_t most = 48 / parts;  // rows of x whose parts fit six column blocks
  const int64_t chunks = ceil_div(a.rows, most);
  a.chunk = (int)ceil_div(a.rows, chunks);
  const int cols = a.chunk * parts;
  auto grouped = [&](auto nt, auto mt, auto rw) {
    constexpr int NT = decltype(nt)::value, MT = decltype(mt)::value, RW = decltype(rw)::value;
    if (group == 32) launch_sized<T, NT, 32, MT, RW>(a, stream);
    else if (group == 64) launch_sized<T, NT, 64, MT, RW>(a, stream);
    else launch_sized<T, NT, 128, MT, RW>(a, stream);
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  using I4 = std::integral_constant<int, 4>;
  using I5 = std::integral_constant<int, 5>;
  using I6 = std::integral_constant<int, 6>;
  const int64_t sms = device_sm_count(current_device());
  if (cols <= 8) {
    // With long rows of weights, enough of them for one wave of 64-row tiles,
    // the warps take rows of their own and join only in pairs, once a tile
    // (one fp32 row, 16384 x 4096: 14.1 us for 14.9; 12000 x 2000 in fp16: 7.4
    // for 6.8, 4096 x 4096 in bf16 5.8 for 4.7); so do they where all of x does
    // not fit beside the ring.
    const bool tall = (ceil_div(a.outer, 64) >= sms && a.blocks >= 32) || (int64_t)cols * a.blocks * kBlock * 2 > 40 * 1024;
    tall ? grouped(I1(), I1(), I4()) : grouped(I1(), I1(), I1());
    return;
  }
  // 128-row tiles, or 32-row ones where those would leave half of the device
  // idle (40 rows of x in fp16, 128- / 32-row tiles: 200 x 12000 weights 14.4
  // / 7.6 us, 1000 x 8000 11.9 / 8.8, 4000 x 1000 10.9 / 6.5, 4000 x 12000 26.7
  // / 37.1)
  const int64_t tiles = ceil_div(a.outer, 128);
  const bool low = tiles * ranks_of(tiles, sms, a.blocks, 2) * 2 < sms;
  auto many = [&](auto nt) { low ? grouped(nt, I1(), I2()) : grouped(nt, I2(), I4()); };
  if (cols <= 16) many(I2());
  else if (cols <= 24) many(I3());
  else if (cols <= 32) many(I4());
  else if (cols <= 40) many(I5());
  else many(I6());
}

void check_group(int64_t group) {
  PFB_CHECK_ARG(group == 32 || group == 64 || (group >= 128 && group % 128 == 0 && group <= INT32_MAX),
                "linear w4: group must be 32, 64 or a multiple of 128");
}

}  // namespace

void launch_w4_arrange(const pfk_w4_arrange_params& p, cudaStream_t stream) {
  PFB_CHECK_ARG(p.outer >= 0 && p.inner >= 0 && p.outer <= (1 << 28) && p.inner <= (1 << 28), "w4 arrange: bad size");
  check_group(p.group);
  PFB_CHECK_ARG(p.scale_dtype == PFC_DTYPE_FLOAT16 || p.scale_dtype == PFC_DTYPE_BFLOAT16,
                "w4 arrange: scale_dtype must be float16 or bfloat16");
  if (p.outer == 0 || p.inner == 0) return;
  PFB_CHECK_ARG(p.packed && p.scales && p.weight && p.meta, "w4 arrange: null pointer");
  ArrangeArgs a = {p.packed, p.scales, p.zeros, p.weight, p.meta, 0, 0, (int)p.inner, (int)p.outer};
  a.blocks = (int)ceil_div(p.inner, kBlock);
  a.groups = (int)ceil_div(p.inner, p.group);
  a.group = (int)p.group;
  a.bf16 = p.scale_dtype == PFC_DTYPE_BFLOAT16;
  const int64_t row_blocks = ceil_div(p.outer, 16);
  a.words = row_blocks * a.blocks * 256;
  a.metas = row_blocks * 16 * (p.group < kBlock ? a.blocks * (kBlock / p.group) : a.groups);
  arrange_kernel<<<(unsigned)std::min<int64_t>(ceil_div(a.words, 256), 148 * 16), 256, 0, stream>>>(a);
  PFB_CUDA(cudaGetLastError());
}

void launch_linear_w4(const pfk_linear_w4_params& p, cudaStream_t stream) {
  check_decode_dtype(p.dtype);
  // a grid has up to 65535 chunks of rows, of 16 in float32
  PFB_CHECK_ARG(p.rows >= 0 && p.rows <= 65535 * 16, "linear w4: rows must be 0 to 1048560");
  PFB_CHECK_ARG(p.inner >= 1 && p.inner <= (1 << 28) && p.outer >= 1 && p.outer <= (1 << 28),
                "linear w4: inner and outer must be 1 to 2^28");
  check_group(p.group);
  PFB_CHECK_ARG(round_up(p.outer, 16) * ceil_div(p.inner, kBlock) * 4 < (1ll << 32), "linear w4: weights of 64 GiB or more");
  if (p.rows == 0) return;
  PFB_CHECK_ARG(p.x && p.y && p.weight && p.meta, "linear w4: null pointer");
  PFB_CHECK_ARG((uintptr_t)p.weight % 16 == 0 && (uintptr_t)p.meta % 16 == 0,
                "linear w4: weight and meta must be 16-byte aligned");
  Args a = {};
  const int64_t es = p.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  a.x = p.x;
  a.x_st = p.rows > 1 ? p.x_st : 0;
  a.y = p.y;
  a.y_st = p.y_st;
  a.weight = (const uint4*)p.weight;
  a.meta = p.meta;
  a.bias = p.bias;
  a.rows = (int)p.rows;
  a.inner = (int)p.inner;
  a.outer = (int)p.outer;
  a.blocks = (int)ceil_div(p.inner, kBlock);
  a.row_blocks = (int)ceil_div(p.outer, 16);
  a.groups = (int)ceil_div(p.inner, p.group);
  a.group_blocks = (int)std::max<int64_t>(1, p.group / kBlock);
  a.vector = (uintptr_t)p.x % 16 == 0 && a.x_st * es % 16 == 0;
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_typed<float>(a, p.group, stream);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_typed<__half>(a, p.group, stream);
  else launch_typed<__nv_bfloat16>(a, p.group, stream);
}

}  // namespace pfb
