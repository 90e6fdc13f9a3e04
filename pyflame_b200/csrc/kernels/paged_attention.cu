// paged_attention.cu — attention of one new token per sequence over a paged
// key-value cache.
//
//   s_j = scale q.k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// Keys and values are read once for every unit of work: 2 * D values for
// 4 * D * G operations (G query heads of the unit), so memory bounds it as long
// as the products run on the tensor cores and the loads never pause.
//
// Work.  A unit is one sequence, one key-value head and some of its query
// heads: in 16-bit types up to 16, of heads above 128 values up to 8; in fp32
// up to 8, of heads above 128 up to 2 (what the registers hold).  Wider
// groups are several units, each of which reads all of the keys again: 40
// query heads on one key-value head three times in 16 bits.  A unit's keys
// are cut into tiles, a step of a CTA's 4 warps each.  The tiles of all units
// form one list, and each of a fixed number of CTAs (one wave) takes an equal
// run of it, whatever the sequences' lengths: lengths are device data, so the
// host could not balance them.  A CTA that has a whole unit writes its
// output; a unit that is shared leaves (m, sum, o) of each share in the
// workspace, and a second small kernel joins the shares in the order of the
// list, so that results do not depend on timing and nothing has to be zero
// beforehand.  Few units of short sequences have a cluster of CTAs each
// instead, which joins its shares through distributed shared memory.
//
// Step.  A warp takes 16 keys at a time (8 on the CUDA cores), straight from
// global memory into registers, without shared memory: lane (g, t) = (lane /
// 4, lane % 4) holds 16-byte pieces of the key rows g and g + 8 and of the
// value rows 2t, 2t + 1, 8 + 2t and 9 + 2t.  Those are the operand registers
// of mma.sync: S^T = K Q^T has the keys as its rows, and since the order of
// the summed axis is free as long as both operands agree, a fragment of K is
// 16 consecutive bytes; O^T = V^T P^T has the values' axis as its rows, whose
// pairs of keys come from byte permutes.  P is turned from the first
// product's accumulator layout into the second's operand layout by movmatrix.
// A group of 8 query heads fills the 8 columns of the instruction; tcgen05
// would need 128 rows of one operand in shared memory for the same, and the
// products are far from being the limit.  The next step's keys are loaded as
// soon as this step's scores are done, its values as soon as the products are.
//
// Types.  16-bit: Q, K, V enter exactly; P is split into a high and a low
// part, so its rounding (2^-18 in bf16, less in fp16) stays far below that of
// the output, 2^-8 and 2^-11.  fp16 P is scaled by 2^14 to keep small weights
// out of its subnormal range.  Exponentials are one ex2.approx.ftz in all
// types: its error, 2^-22 of a weight, is what rounding an fp32 score of size 4
// does to it, and a weight below 2^-126 of the largest may count as 0.
// fp32, up to 4 query heads a key-value head, and heads above 128: fp32 FMAs
// on the CUDA cores.  fp32, more: both operands are split into tf32 high and
// low parts, three products (the dropped low-low term is below 2^-22 of the
// product).  Scores, maxima, sums and outputs are held in fp32.  The tensor
// cores truncate what they add, so nothing runs on in their accumulators: a
// step's products of weights and values have one of their own, which is added
// to the running output in fp32, rounded to nearest (added to it by the
// instruction, 131072 keys of a 16-bit type lost up to 3e-5 of the values'
// size; the addition costs 1% of the time: one sequence of 131071 103 us for
// 102, 48 of 0 to 8192 151 for 149.5).
//
// Measured (device time, replayed from a graph; the bytes at 6.4 TB/s in
// brackets): 128 sequences of 2048 to 8192 keys, bf16, 32/8 heads of 128, 2.69
// GB: 407 to 440 us, by the machine (420); 48 of 0 to 8192, fp16: 137 to 140
// us (126); one of 131071, 64/8 heads: 97 us (84); 7 with a window of 1000,
// fp32, 20 heads of 80: 23 us (11.7), of which a warp spends most on 8 to 9
// dependent steps of 8 keys, over registers laid out for heads of 128 (three
// CTAs an SM), and the join's launch the rest; one of 333, fp32, 12 heads of
// 64: 5.4 us, latency alone: lengths, page numbers, keys and the join follow
// one another.
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

namespace pfb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMostRanks = 8;  // CTAs of a cluster
constexpr unsigned kNone = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Args {
  const char* k;
  const char* v;
  unsigned long long unit_bytes;  // page_units and token_units count these
  unsigned page_units, token_units;
  long long head_bytes;
  unsigned num_pages;
  FastDiv by_page;
  int* err;
  int batch, q_heads, kv_heads, group;
  int unit_heads, chunks;  // a key-value head has `chunks` units of up to unit_heads query heads
  int head_dim;
  const void* q;
  long long q_sb, q_sh;
  void* out;
  long long o_sb, o_sh;
  float* lse;
  const int* table;
  long long table_stride;
  const int* seq_lens;
  long long most;  // tokens that the table has room for
  int window;
  float scale;
  // workspace: a record of each CTA (the unit that began there and goes on in
  // later CTAs, if there is one), the shares' maxima and sums
  // [ctas][2][heads], and their outputs [ctas][2][heads][D]
  int4* records;  // row, unit, last CTA, whether there is one
  float2* stats;
  float* parts;
  int ctas;
  int heads;  // of a full unit: min(group, unit_heads)
};

__device__ const uint4 kZeros[64] = {};  // a row of the widest head

struct Span {
  int begin, end, tiles;  // seen keys, and the tiles that cover them
};

template <int TILE>
__device__ __forceinline__ Span span_of(const Args& a, int b) {
  long long n = a.seq_lens[b];
  if (n < 0 || n > a.most) {
    if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
    n = n < 0 ? 0 : a.most;
  }
  Span s;
  s.end = (int)n;
  s.begin = a.window > 0 && n > a.window ? (int)n - a.window : 0;
  s.tiles = n ? (s.end + TILE - 1) / TILE - s.begin / TILE : 0;
  return s;
}

template <typename T>
struct Traits;
template <>
struct Traits<__nv_bfloat16> {
  static constexpr int kVec = 8;  // values of a 16-byte access
  static constexpr float kShift = 0.f;
  static __device__ __forceinline__ unsigned pack(float x, float y) {
    __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<unsigned*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(unsigned u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                             unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // c = the product, with nothing added
  static __device__ __forceinline__ void mma_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                                   unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Traits<__half> {
  static constexpr int kVec = 8;
  static constexpr float kShift = 14.f;
  static __device__ __forceinline__ unsigned pack(float x, float y) {
    __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<unsigned*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(unsigned u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                             unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // c = the product, with nothing added
  static __device__ __forceinline__ void mma_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                                   unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Traits<float> {
  static constexpr int kVec = 4;
  static constexpr float kShift = 0.f;
  static __device__ __forceinline__ float from(float v) { return v; }
};

__device__ __forceinline__ void mma_tf32(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                         unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x = hi + lo, both tf32, hi the nearest: lo is at most 2^-11 of x and loses
// 2^-11 of itself.
__device__ __forceinline__ void split(float x, unsigned& hi, unsigned& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}

__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint4 load16(const char* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ unsigned word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

__device__ __forceinline__ unsigned long long divide(unsigned long long a, unsigned long long b) {
  return ((a | b) >> 32) ? a / b : (unsigned)a / (unsigned)b;
}

// DP: head_dim rounded up to the size that the registers are laid out for.
// CORES: fp32 on the CUDA cores, NT the query heads of a unit (1, 2 or 4);
// otherwise on the tensor cores, NT blocks of 8 query heads.
template <typename T, int DP, int NT, bool CORES>
struct Layout {
  static constexpr int kVec = Traits<T>::kVec;
  static constexpr int kQ = DP / (4 * kVec);  // 16-byte chunks of a K row that a lane holds
  static constexpr int kV = DP / (8 * kVec);  // of a V row
  static constexpr int kHeads = CORES ? NT : NT * 8;
  static constexpr int kPitch = DP + 4;
  // a step's keys in blocks of 8: 16 fp32 rows of 256 do not fit the registers
  static constexpr int kRows = CORES ? 1 : 2;
  static constexpr int kTile = 8 * kRows * kWarps;  // keys of a CTA's step
  static constexpr size_t q_bytes = CORES ? (size_t)NT * DP * 4 : (size_t)kQ * NT * 32 * 16 * (sizeof(T) == 4 ? 2 : 1);
  static constexpr size_t o_bytes = (size_t)kWarps * kHeads * kPitch * 4;
  static constexpr size_t m_bytes = (size_t)2 * kWarps * kHeads * 4;
  static constexpr size_t smem = q_bytes + o_bytes + m_bytes;
  // CTAs that share an SM: as many warps' loads in flight as the registers hold
  static constexpr int kResident = CORES ? (DP <= 64 ? 4 : DP <= 128 ? 3 : 2) : sizeof(T) == 2 ? (DP <= 64 ? (NT == 1 ? 4 : 3) : DP <= 128 && NT == 1 ? 3 : 2) : DP <= 64 ? 3 : 2;
};

// CLUSTER: a cluster of CTAs for each unit, each an equal part of its tiles;
// otherwise runs of the list of all tiles.
template <typename T, int DP, int NT, bool CORES, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, (Layout<T, DP, NT, CORES>::kResident)) attend_kernel(Args a) {
  using L = Layout<T, DP, NT, CORES>;
  using Tr = Traits<T>;
  constexpr int VEC = L::kVec, HEADS = L::kHeads;
  constexpr bool k32 = sizeof(T) == 4;
  extern __shared__ __align__(16) char smem[];
  uint4* qs = reinterpret_cast<uint4*>(smem);  // [split][nt][chunk][lane], or [head][DP] floats
  float* os = reinterpret_cast<float*>(smem + L::q_bytes);
  float* ms = reinterpret_cast<float*>(smem + L::q_bytes + L::o_bytes);  // [warp][head] maxima, then sums
  float* ls = ms + kWarps * HEADS;
  __shared__ long long scan[kWarps];
  __shared__ int found_row;
  __shared__ long long found_before;
  __shared__ Span found_span;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  begin();
  const int per_row = a.kv_heads * a.chunks;
  int row, unit, tile;  // unit: of the row
  Span sp;
  long long t0, t1, list_total = 0;
  int list_ctas = 0;
  namespace cg = cooperative_groups;
  __shared__ float2 part[HEADS];  // of a cluster's CTA: each head's maximum and sum
  if constexpr (CLUSTER) {
    const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const int u = blockIdx.x / ranks;
    row = u / per_row;
    unit = u - row * per_row;
    sp = span_of<L::kTile>(a, row);
    t0 = (long long)sp.tiles * rank / ranks;
    t1 = (long long)sp.tiles * (rank + 1) / ranks;
    tile = (int)t0;
    if (t0 == t1 && tid < HEADS) part[tid] = make_float2(-INFINITY, 0.f);
  } else {
    // the join may come up as soon as the last of these CTAs has started
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // the list of tiles: its length, and the row that holds this CTA's first
    Span mine = {0, 0, 0};
    auto scan_rows = [&](int b) -> long long {  // tiles of the rows before b in its block of rows; scan: warps' sums
      mine = b < a.batch ? span_of<L::kTile>(a, b) : Span{0, 0, 0};
      const long long own = (long long)mine.tiles * per_row;
      long long sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += up;
      }
      if (lane == 31) scan[warp] = sum;
      __syncthreads();
      long long start = sum - own;
      for (int w = 0; w < warp; ++w) start += scan[w];
      return start;
    };
    auto scanned = [&]() -> long long { return scan[0] + scan[1] + scan[2] + scan[3]; };
    static_assert(kWarps == 4, "scanned() adds four warps' sums");
    long long total = 0, start = 0;
    if (a.batch > kThreads) {
      for (int b = tid; b < a.batch; b += kThreads) total += (long long)span_of<L::kTile>(a, b).tiles * per_row;
#pragma unroll
      for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
      if (lane == 0) scan[warp] = total;
      __syncthreads();
      total = scanned();
    } else {
      start = scan_rows(tid);
      total = scanned();
    }
    // runs of total / ctas tiles, the longer ones spread evenly (neighbouring
    // CTAs share an SM: 505 us for 487 with the longer runs first)
    // at least four tiles each: more shares cost more than they save (one
    // sequence of 4096 keys and 8 units: 21.4 us with one, 16.0 two, 14.3 four)
    const int ctas = (int)min((long long)a.ctas, (total + 3) / 4);
    const long long c = min((int)blockIdx.x, ctas);
    t0 = ctas ? (long long)divide(total * c, ctas) : 0;
    t1 = c < ctas ? (long long)divide(total * (c + 1), ctas) : t0;
    if (t0 >= t1) {
      if (tid == 0) a.records[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    long long before = 0;
    for (int base = 0;; base += kThreads) {
      if (a.batch > kThreads) {
        __syncthreads();
        start = scan_rows(base + tid);
      }
      if (t0 >= before + start && t0 < before + start + (long long)mine.tiles * per_row) {
        found_row = base + tid;
        found_before = before + start;
        found_span = mine;
      }
      before += scanned();
      if (before > t0) break;  // total > t0: some block of rows gets there
    }
    __syncthreads();
    row = found_row;
    sp = found_span;
    unit = (int)divide(t0 - found_before, sp.tiles);
    tile = (int)((t0 - found_before) - (long long)unit * sp.tiles);
    list_total = total;
    list_ctas = ctas;
  }
  int4 record = make_int4(0, 0, 0, 0);

  const float scale2 = a.scale * kLog2e;

  // The loads run ahead of the products and over the borders of units: ahead
  // stands at the step after the next, whose place in the cache it looks up.
  struct {
    long long at;
    int row, unit, tile, begin, end, tiles;
  } ahead = {t0, row, unit, tile, sp.begin, sp.end, sp.tiles};
  struct Place {
    unsigned where;  // of one of the warp's keys (lane modulo their number), in units
    int head;
  };
  auto place = [&]() -> Place {
    Place p = {kNone, 0};
    if (ahead.at >= t1) return p;
    p.head = ahead.unit / a.chunks;
    const int key = (ahead.begin / L::kTile + ahead.tile) * L::kTile + warp * 8 * L::kRows + (lane & (8 * L::kRows - 1));
    if (key >= ahead.begin && key < ahead.end) {
      const unsigned i = a.by_page.div((unsigned)key);
      const unsigned page = (unsigned)a.table[(long long)ahead.row * a.table_stride + i];
      if (page < a.num_pages) p.where = page * a.page_units + ((unsigned)key - i * a.by_page.d) * a.token_units;
      else if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
    }
    ++ahead.at;
    if (++ahead.tile == ahead.tiles) {
      ahead.tile = 0;
      if (++ahead.unit == per_row) {
        ahead.unit = 0;
        if (ahead.at < t1) {
          Span n;
          do n = span_of<L::kTile>(a, ++ahead.row);
          while (n.tiles == 0);  // there is one: the list goes on
          ahead.begin = n.begin;
          ahead.end = n.end;
          ahead.tiles = n.tiles;
        }
      }
    }
    return p;
  };
  // Keys that are not there (masked, or of a bad page) are read from a row of
  // zeros: what lies in their place may be NaN, which a weight of 0 would not
  // hide.  Chunks behind head_dim stay the zeros they start as.
  uint4 kr[L::kRows][L::kQ], vr[2 * L::kRows][L::kV];
#pragma unroll
  for (int r = 0; r < L::kRows; ++r)
#pragma unroll
    for (int c = 0; c < L::kQ; ++c) kr[r][c] = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 2 * L::kRows; ++r)
#pragma unroll
    for (int c = 0; c < L::kV; ++c) vr[r][c] = make_uint4(0, 0, 0, 0);
  const char *kp[L::kRows], *vp[2 * L::kRows];  // the rows that are loaded next
  bool seen[L::kRows];                          // whether those keys are there
  auto aim = [&](const Place& p) {
    const char* k = a.k + p.head * a.head_bytes;
    const char* v = a.v + p.head * a.head_bytes;
    const char* none = reinterpret_cast<const char*>(kZeros);
#pragma unroll
    for (int r = 0; r < L::kRows; ++r) {
      const unsigned u = __shfl_sync(~0u, p.where, g + 8 * r);
      seen[r] = u != kNone;
      kp[r] = (u != kNone ? k + u * a.unit_bytes : none) + t * 16;
    }
#pragma unroll
    for (int r = 0; r < 2 * L::kRows; ++r) {
      const unsigned u = __shfl_sync(~0u, p.where, 2 * t + (r & 1) + 8 * (r >> 1));
      vp[r] = (u != kNone ? v + u * a.unit_bytes : none) + g * 16;
    }
  };
  auto load_k = [&](int c) {
#pragma unroll
    for (int r = 0; r < L::kRows; ++r)
      if ((c * 4 + t) * VEC < a.head_dim) kr[r][c] = load16(kp[r] + c * 64);
  };
  auto load_v = [&](int c) {
#pragma unroll
    for (int r = 0; r < 2 * L::kRows; ++r)
      if ((c * 8 + g) * VEC < a.head_dim) vr[r][c] = load16(vp[r] + c * 128);
  };
  // Q in the order of the second operand's registers
  auto stage_q = [&](int row, int first_q, int heads) {
    const T* qp = (const T*)a.q + (long long)row * a.q_sb + (long long)first_q * a.q_sh;
    if constexpr (CORES) {
      for (int i = tid; i < NT * DP; i += kThreads) {
        const int h = i / DP, d = i - h * DP;
        reinterpret_cast<float*>(qs)[i] = h < heads && d < a.head_dim ? qp[h * a.q_sh + d] : 0.f;
      }
    } else {
      for (int i = tid; i < NT * L::kQ * 32; i += kThreads) {
        const int l = i & 31, c = (i >> 5) % L::kQ, nt = (i >> 5) / L::kQ;
        const int h = nt * 8 + (l >> 2), d0 = (c * 4 + (l & 3)) * VEC;
        if constexpr (k32) {
          uint4 hi = {}, lo = {};
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = h < heads && d0 + e < a.head_dim ? qp[h * a.q_sh + d0 + e] : 0.f;
          split(x[0], hi.x, lo.x);
          split(x[1], hi.y, lo.y);
          split(x[2], hi.z, lo.z);
          split(x[3], hi.w, lo.w);
          qs[i] = hi;
          qs[NT * L::kQ * 32 + i] = lo;
        } else {
          alignas(16) T x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = h < heads && d0 + e < a.head_dim ? qp[h * a.q_sh + d0 + e] : Tr::from(0.f);
          qs[i] = *reinterpret_cast<uint4*>(x);
        }
      }
    }
  };
  // the first unit's before the chain of loads that leads to its first keys
  if (t0 < t1) {
    const int head = unit / a.chunks, first_q = head * a.group + (unit - head * a.chunks) * a.unit_heads;
    stage_q(row, first_q, min(a.unit_heads, (head + 1) * a.group - first_q));
  }
  aim(place());
#pragma unroll
  for (int c = 0; c < L::kQ; ++c) load_k(c);
#pragma unroll
  for (int c = 0; c < L::kV; ++c) load_v(c);
  Place next = place();

  for (long long at = t0; at < t1;) {
    while (sp.tiles == 0) sp = span_of<L::kTile>(a, ++row);
    const int count = (int)min((long long)(sp.tiles - tile), t1 - at);
    const int head = unit / a.chunks;
    const int first_q = head * a.group + (unit - head * a.chunks) * a.unit_heads;
    const int heads = min(a.unit_heads, (head + 1) * a.group - first_q);

    if (at != t0) {
      __syncthreads();  // the previous piece's reads of shared memory are over
      stage_q(row, first_q, heads);
    }
    __syncthreads();

    // Running maxima, sums and outputs.  On the tensor cores a lane has query
    // heads nt*8 + 2t and + 1, of o the value pairs 2j, 2j + 1 of its chunk;
    // on the CUDA cores every head, of o its own keys' part.
    constexpr int MH = CORES ? 1 : 2;
    float m[NT][MH], l[NT][MH], o[NT][L::kV][VEC / 2][CORES ? 2 : 4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MH; ++i) {
        m[nt][i] = -INFINITY;
        l[nt][i] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < L::kV; ++c)
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j)
#pragma unroll
          for (int r = 0; r < (CORES ? 2 : 4); ++r) o[nt][c][j][r] = 0.f;
    }
    for (int step = 0; step < count; ++step) {
      bool live[L::kRows];
#pragma unroll
      for (int r = 0; r < L::kRows; ++r) live[r] = seen[r];
      aim(next);
      if constexpr (CORES) {
        float s[NT][L::kRows];  // of keys g (and g + 8), the same in a quad's lanes
#pragma unroll
        for (int h = 0; h < NT; ++h) {
          float sum[L::kRows][4];
#pragma unroll
          for (int r = 0; r < L::kRows; ++r) sum[r][0] = sum[r][1] = sum[r][2] = sum[r][3] = 0.f;
#pragma unroll
          for (int c = 0; c < L::kQ; ++c) {
            const float4 q = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(qs) + h * DP + (c * 4 + t) * 4);
#pragma unroll
            for (int r = 0; r < L::kRows; ++r) {
              sum[r][0] = fmaf(q.x, __uint_as_float(kr[r][c].x), sum[r][0]);
              sum[r][1] = fmaf(q.y, __uint_as_float(kr[r][c].y), sum[r][1]);
              sum[r][2] = fmaf(q.z, __uint_as_float(kr[r][c].z), sum[r][2]);
              sum[r][3] = fmaf(q.w, __uint_as_float(kr[r][c].w), sum[r][3]);
            }
            if (h == NT - 1) load_k(c);
          }
#pragma unroll
          for (int r = 0; r < L::kRows; ++r) s[h][r] = (sum[r][0] + sum[r][1]) + (sum[r][2] + sum[r][3]);
        }
        float p[NT][2 * L::kRows];  // of the lane's value rows
#pragma unroll
        for (int h = 0; h < NT; ++h) {
          float top = -INFINITY;
#pragma unroll
          for (int r = 0; r < L::kRows; ++r) {
            s[h][r] += __shfl_xor_sync(~0u, s[h][r], 1);
            s[h][r] += __shfl_xor_sync(~0u, s[h][r], 2);
            s[h][r] = live[r] ? s[h][r] * scale2 : -INFINITY;
            top = fmaxf(top, s[h][r]);
          }
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          if (top > m[h][0]) {  // the same in all lanes
            const float f = exp2_fast(m[h][0] - top);
            m[h][0] = top;
            l[h][0] *= f;
#pragma unroll
            for (int c = 0; c < L::kV; ++c)
#pragma unroll
              for (int j = 0; j < VEC / 2; ++j) {
                o[h][c][j][0] *= f;
                o[h][c][j][1] *= f;
              }
          }
          const float base = m[h][0] == -INFINITY ? 0.f : m[h][0];
#pragma unroll
          for (int r = 0; r < L::kRows; ++r) {
            const float e = exp2_fast(s[h][r] - base);
            l[h][0] += e;
            p[h][2 * r] = __shfl_sync(~0u, e, 8 * t);
            p[h][2 * r + 1] = __shfl_sync(~0u, e, 8 * t + 4);
          }
        }
#pragma unroll
        for (int c = 0; c < L::kV; ++c) {
#pragma unroll
          for (int h = 0; h < NT; ++h)
#pragma unroll
            for (int r = 0; r < 2 * L::kRows; ++r)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[h][c][e >> 1][e & 1] = fmaf(p[h][r], __uint_as_float(word(vr[r][c], e)), o[h][c][e >> 1][e & 1]);
          load_v(c);
        }
      } else {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // one accumulator for a score's 4 to 16 instructions of 16-bit types,
          // which truncate less than 2^-19 of its terms in all (two accumulators
          // measured 505 us for 423 at 128 sequences of 5000 keys); in fp32 one
          // for each chunk's six, added up in fp32
#pragma unroll
          for (int r = 0; r < 4; ++r) s[nt][r] = 0.f;
#pragma unroll
          for (int c = 0; c < L::kQ; ++c) {
            const uint4 b = qs[(nt * L::kQ + c) * 32 + lane];
            if constexpr (k32) {
              const uint4 bl = qs[(NT * L::kQ + nt * L::kQ + c) * 32 + lane];
              float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                unsigned h0, h1, h2, h3, l0, l1, l2, l3;
                split(__uint_as_float(word(kr[0][c], 2 * e)), h0, l0);
                split(__uint_as_float(word(kr[1][c], 2 * e)), h1, l1);
                split(__uint_as_float(word(kr[0][c], 2 * e + 1)), h2, l2);
                split(__uint_as_float(word(kr[1][c], 2 * e + 1)), h3, l3);
                mma_tf32(part, l0, l1, l2, l3, word(b, 2 * e), word(b, 2 * e + 1));
                mma_tf32(part, h0, h1, h2, h3, word(bl, 2 * e), word(bl, 2 * e + 1));
                mma_tf32(part, h0, h1, h2, h3, word(b, 2 * e), word(b, 2 * e + 1));
              }
#pragma unroll
              for (int r = 0; r < 4; ++r) s[nt][r] += part[r];
            } else {
              Tr::mma(s[nt], kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, b.x, b.y);
              Tr::mma(s[nt], kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, b.z, b.w);
            }
            if (nt == NT - 1) load_k(c);
          }
        }

        unsigned pt[NT][4];  // P as the second operand: 16-bit hi, lo of keys 0-7 and 8-15; fp32 its four values
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = live[r >> 1] ? s[nt][r] * scale2 : -INFINITY;
          float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
          bool moved = false;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 4));
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 8));
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 16));
            moved |= top[i] > m[nt][i];
          }
          if (__any_sync(~0u, moved)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float to = fmaxf(m[nt][i], top[i]);
              const float f = to == -INFINITY ? 1.f : exp2_fast(m[nt][i] - to);
              m[nt][i] = to;
              l[nt][i] *= f;
#pragma unroll
              for (int c = 0; c < L::kV; ++c)
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                  o[nt][c][j][i] *= f;
                  o[nt][c][j][i + 2] *= f;
                }
            }
          }
          float p[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float base = m[nt][r & 1] == -INFINITY ? 0.f : m[nt][r & 1];
            p[r] = exp2_fast(x[r] - base + Tr::kShift);
            l[nt][r & 1] += p[r];
          }
          if constexpr (k32) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const unsigned u0 = __float_as_uint(p[2 * i]), u1 = __float_as_uint(p[2 * i + 1]);
              const unsigned lo = transpose8x8(__byte_perm(u0, u1, 0x5410));
              const unsigned hi = transpose8x8(__byte_perm(u0, u1, 0x7632));
              pt[nt][2 * i] = __byte_perm(lo, hi, 0x5410);      // key 8i + 2t of head g
              pt[nt][2 * i + 1] = __byte_perm(lo, hi, 0x7632);  // key 8i + 2t + 1
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const unsigned hi = Tr::pack(p[2 * i], p[2 * i + 1]);
              const float2 back = Tr::unpack(hi);
              pt[nt][2 * i] = transpose8x8(hi);
              pt[nt][2 * i + 1] = transpose8x8(Tr::pack(p[2 * i] - back.x, p[2 * i + 1] - back.y));
            }
          }
        }

#pragma unroll
        for (int c = 0; c < L::kV; ++c) {
          if constexpr (k32) {
            // with the instruction adding to the running output, 16 steps
            // lost 3e-6 of it
            float sum[NT][2][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[nt][j][r] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // keys 8i ... 8i + 7
              unsigned bh[NT][2], bl[NT][2];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                split(__uint_as_float(pt[nt][2 * i]), bh[nt][0], bl[nt][0]);
                split(__uint_as_float(pt[nt][2 * i + 1]), bh[nt][1], bl[nt][1]);
              }
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                unsigned h0, h1, h2, h3, l0, l1, l2, l3;
                split(__uint_as_float(word(vr[2 * i][c], 2 * j)), h0, l0);
                split(__uint_as_float(word(vr[2 * i][c], 2 * j + 1)), h1, l1);
                split(__uint_as_float(word(vr[2 * i + 1][c], 2 * j)), h2, l2);
                split(__uint_as_float(word(vr[2 * i + 1][c], 2 * j + 1)), h3, l3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma_tf32(sum[nt][j], l0, l1, l2, l3, bh[nt][0], bh[nt][1]);
                  mma_tf32(sum[nt][j], h0, h1, h2, h3, bl[nt][0], bl[nt][1]);
                  mma_tf32(sum[nt][j], h0, h1, h2, h3, bh[nt][0], bh[nt][1]);
                }
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[nt][c][j][r] += sum[nt][j][r];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const unsigned a0 = __byte_perm(word(vr[0][c], j), word(vr[1][c], j), 0x5410);
              const unsigned a1 = __byte_perm(word(vr[0][c], j), word(vr[1][c], j), 0x7632);
              const unsigned a2 = __byte_perm(word(vr[2][c], j), word(vr[3][c], j), 0x5410);
              const unsigned a3 = __byte_perm(word(vr[2][c], j), word(vr[3][c], j), 0x7632);
              float sum[NT][4];  // the step's
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) Tr::mma_first(sum[nt], a0, a1, a2, a3, pt[nt][1], pt[nt][3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) Tr::mma(sum[nt], a0, a1, a2, a3, pt[nt][0], pt[nt][2]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[nt][c][j][r] += sum[nt][r];
            }
          }
          load_v(c);
        }
      }
      next = place();
    }

    // join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MH; ++i) {
        const int h = warp * HEADS + (CORES ? nt : nt * 8 + 2 * t + i);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], off);
        if (CORES ? lane == 0 : g == 0) {
          ms[h] = m[nt][i];
          ls[h] = l[nt][i];
        }
#pragma unroll
        for (int c = 0; c < L::kV; ++c)
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            float2 pair;
            if constexpr (CORES) {  // the quad's lanes have different keys of the same values
              pair = make_float2(o[nt][c][j][0], o[nt][c][j][1]);
#pragma unroll
              for (int off = 1; off < 4; off <<= 1) {
                pair.x += __shfl_xor_sync(~0u, pair.x, off);
                pair.y += __shfl_xor_sync(~0u, pair.y, off);
              }
            } else {
              pair = make_float2(o[nt][c][j][i], o[nt][c][j][CORES ? 0 : i + 2]);
            }
            if (!CORES || t == j) *reinterpret_cast<float2*>(os + (size_t)h * L::kPitch + (c * 8 + g) * VEC + 2 * j) = pair;
          }
      }
    }
    __syncthreads();
    const bool whole = tile == 0 && count == sp.tiles;
    const int slot = tile == 0 ? 1 : 0;  // a unit that began here, or one that began in an earlier CTA
    const long long share = ((long long)blockIdx.x * 2 + slot) * a.heads;
    for (int i = tid; i < heads * a.head_dim; i += kThreads) {
      const int h = i / a.head_dim, d = i - h * a.head_dim;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ms[w * HEADS + h]);
      float v = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = ms[w * HEADS + h];
        const float f = mw == -INFINITY ? (top == -INFINITY ? 1.f : 0.f) : exp2_fast(mw - top);
        v += f * os[(size_t)(w * HEADS + h) * L::kPitch + d];
        sum += f * ls[w * HEADS + h];
      }
      if constexpr (CLUSTER) {
        os[(size_t)h * L::kPitch + d] = v;  // read and written by this thread alone
        if (d == 0) part[h] = make_float2(top, sum);
      } else if (whole) {
        ((T*)a.out)[(long long)row * a.o_sb + (long long)(first_q + h) * a.o_sh + d] = Tr::from(sum == 0.f ? 0.f : v / sum);
        if (d == 0 && a.lse)
          a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (top + log2f(sum) - Tr::kShift) * kLn2;
      } else {
        a.parts[(share + h) * a.head_dim + d] = v;
        if (d == 0) a.stats[share + h] = make_float2(top, sum);
      }
    }
    if (CLUSTER) break;
    if (tile == 0 && !whole) {  // the CTA that has the unit's last tile
      // tile x is in the last CTA c with floor(total c / ctas) <= x
      record = make_int4(row, unit, (int)divide((at + sp.tiles) * list_ctas + list_total - 1, list_total) - 1, 1);
    }
    at += count;
    tile = 0;
    if (++unit == per_row) {
      unit = 0;
      sp.tiles = 0;
      if (at < t1) sp = span_of<L::kTile>(a, ++row);
    }
  }
  if constexpr (CLUSTER) {  // each CTA joins a part of the outputs, in the order of the ranks
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int ranks = (int)cluster.num_blocks();
    const int head = unit / a.chunks, first_q = head * a.group + (unit - head * a.chunks) * a.unit_heads;
    const int heads = min(a.unit_heads, (head + 1) * a.group - first_q);
    for (int i = (int)cluster.block_rank() * kThreads + tid; i < heads * a.head_dim; i += kThreads * ranks) {
      const int h = i / a.head_dim, d = i - h * a.head_dim;
      float2 st[kMostRanks];
      float o[kMostRanks];
#pragma unroll
      for (int r = 0; r < kMostRanks; ++r) {
        st[r] = make_float2(-INFINITY, 0.f);
        o[r] = 0.f;
        if (r < ranks) {
          st[r] = cluster.map_shared_rank(part, r)[h];
          o[r] = cluster.map_shared_rank(os, r)[(size_t)h * L::kPitch + d];
        }
      }
      float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
      for (int r = 0; r < kMostRanks; ++r) top = fmaxf(top, st[r].x);
#pragma unroll
      for (int r = 0; r < kMostRanks; ++r) {
        if (st[r].x == -INFINITY && st[r].y == 0.f) continue;  // no keys: its outputs were never written
        const float f = st[r].x == top ? 1.f : exp2_fast(st[r].x - top);
        v += f * o[r];
        sum += f * st[r].y;
      }
      ((T*)a.out)[(long long)row * a.o_sb + (long long)(first_q + h) * a.o_sh + d] = Tr::from(sum == 0.f ? 0.f : v / sum);
      if (d == 0 && a.lse)
        a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (top + log2f(sum) - Tr::kShift) * kLn2;
    }
    cluster.sync();  // the others' reads of this CTA's part are over
  } else if (tid == 0) {
    a.records[blockIdx.x] = record;
  }
}

constexpr int kJoinThreads = 256;

// CTA (c, h): joins the shares of query head h of the unit that began in CTA
// c of the first kernel and went on, in the order of the list; and writes
// the outputs of sequence c if it is empty.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(Args a) {
  using Tr = Traits<T>;
  __shared__ float4 acc[kJoinThreads];
  __shared__ float2 stats[kJoinThreads / 16];
  const int tid = threadIdx.x, c0 = blockIdx.x;
  begin();
  if (c0 < a.batch && span_of<64>(a, c0).tiles == 0) {
    for (int qh = blockIdx.y; qh < a.q_heads; qh += gridDim.y) {
      for (int d = tid; d < a.head_dim; d += kJoinThreads)
        ((T*)a.out)[(long long)c0 * a.o_sb + (long long)qh * a.o_sh + d] = Tr::from(0.f);
      if (tid == 0 && a.lse) a.lse[(long long)c0 * a.q_heads + qh] = -INFINITY;
    }
  }
  if (c0 >= a.ctas) return;
  const int4 rec = a.records[c0];
  if (!rec.w) return;
  const int b = rec.x, head = rec.y / a.chunks, h = blockIdx.y;
  const int qh = head * a.group + (rec.y - head * a.chunks) * a.unit_heads + h;
  if (qh >= (head + 1) * a.group) return;
  const int shares = rec.z - c0 + 1;
  // the first share is slot 1 of its CTA, the others slot 0 of theirs
  auto share = [&](int i) -> long long { return ((long long)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * a.heads + h; };
  const int cols = a.head_dim / 4;                        // of 4 values
  const int across = cols <= 16 ? 16 : cols <= 32 ? 32 : 64;  // threads of a share
  const int groups = kJoinThreads / across, gi = tid / across, col = tid % across;

  // x, of maximum m, joined to (top, sum, v): one pass, each of its loads
  // independent of the others
  float top = -INFINITY, sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](float m, float l, float4 x) {
    const float to = fmaxf(top, m);
    const float f = top == to ? 1.f : exp2_fast(top - to), g = m == to ? 1.f : exp2_fast(m - to);
    v.x = v.x * f + x.x * g;
    v.y = v.y * f + x.y * g;
    v.z = v.z * f + x.z * g;
    v.w = v.w * f + x.w * g;
    sum = sum * f + l * g;
    top = to;
  };
  if (col < cols) {
#pragma unroll 4
    for (int i = gi; i < shares; i += groups) {
      const float2 st = a.stats[share(i)];
      join(st.x, st.y, *reinterpret_cast<const float4*>(a.parts + share(i) * a.head_dim + col * 4));
    }
  }
  acc[tid] = v;
  if (col == 0) stats[gi] = make_float2(top, sum);
  __syncthreads();
  if (gi == 0 && col < cols) {
    for (int w = 1; w < groups; ++w) join(stats[w].x, stats[w].y, acc[w * across + col]);
    T* out = (T*)a.out + (long long)b * a.o_sb + (long long)qh * a.o_sh + col * 4;
    const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = Tr::from(sum == 0.f ? 0.f : r[e] / sum);
    if (col == 0 && a.lse) a.lse[(long long)b * a.q_heads + qh] = sum == 0.f ? -INFINITY : (top + log2f(sum) - Tr::kShift) * kLn2;
  }
}

// CTAs of one wave of a kernel on the current device, asked once per device.
template <class K>
int wave() {
  static std::once_flag once[64];
  static int ctas[64];
  const int dev = current_device();
  std::call_once(once[dev], [dev] {
    PFB_CUDA(cudaFuncSetAttribute(K::run, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)K::L::smem));
    PFB_CUDA(cudaFuncSetAttribute(K::run_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)K::L::smem));
    int per = 0;
    PFB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, K::run, kThreads, K::L::smem));
    ctas[dev] = std::max(1, per) * device_sm_count(dev);
  });
  return ctas[dev];
}

template <class K>
void launch_sized(Args& a, int ranks, cudaStream_t stream) {
  if (ranks) {
    const int64_t ctas = (int64_t)a.batch * a.kv_heads * a.chunks * ranks;
    launch_following<Args>(K::run_cluster, dim3((unsigned)ctas), kThreads, K::L::smem, stream, a, ranks);
    return;
  }
  launch_following<Args>(K::run, dim3((unsigned)a.ctas), kThreads, K::L::smem, stream, a);
  launch_following<Args>(join_kernel<typename K::T>, dim3((unsigned)std::max(a.ctas, a.batch), (unsigned)a.heads), kJoinThreads, 0, stream, a);
}

template <typename T_, int DP, int NT, bool CORES>
struct Kernel {
  using T = T_;
  using L = Layout<T, DP, NT, CORES>;
  static constexpr auto run = attend_kernel<T, DP, NT, CORES, false>;
  static constexpr auto run_cluster = attend_kernel<T, DP, NT, CORES, true>;
};

// Query heads of a unit, as many as the registers hold: on the tensor cores
// two column blocks (16 heads) only with 16-bit types and head_dim up to 128;
// on the CUDA cores up to 4, of wide heads up to 2.
int unit_heads(const pfk_paged_attention_params& p) {
  const int64_t group = p.q_heads / p.cache.heads;
  const bool wide = p.cache.head_dim > 128;
  if (p.cache.dtype != PFC_DTYPE_FLOAT32) return group > 8 && !wide ? 16 : 8;
  if (group <= 1) return 1;
  if (group <= 2 || wide) return 2;
  return group <= 4 ? 4 : 8;
}

template <class F>
void dispatch32(int heads, int64_t head_dim, F&& f) {
  if (head_dim > 128) {
    heads == 1 ? f(Kernel<float, 256, 1, true>()) : f(Kernel<float, 256, 2, true>());
  } else if (head_dim > 64) {
    if (heads == 1) f(Kernel<float, 128, 1, true>());
    else if (heads == 2) f(Kernel<float, 128, 2, true>());
    else if (heads == 4) f(Kernel<float, 128, 4, true>());
    else f(Kernel<float, 128, 1, false>());
  } else {
    if (heads == 1) f(Kernel<float, 64, 1, true>());
    else if (heads == 2) f(Kernel<float, 64, 2, true>());
    else if (heads == 4) f(Kernel<float, 64, 4, true>());
    else f(Kernel<float, 64, 1, false>());
  }
}

template <typename T, class F>
void dispatch16(int heads, int64_t head_dim, F&& f) {
  if (head_dim > 128) f(Kernel<T, 256, 1, false>());
  else if (head_dim > 64) heads == 16 ? f(Kernel<T, 128, 2, false>()) : f(Kernel<T, 128, 1, false>());
  else heads == 16 ? f(Kernel<T, 64, 2, false>()) : f(Kernel<T, 64, 1, false>());
}

// Calls f(Kernel<...>()) for the call's type and sizes.
template <class F>
void dispatch(const pfk_paged_attention_params& p, F&& f) {
  const int heads = unit_heads(p);
  const int64_t d = p.cache.head_dim;
  if (p.cache.dtype == PFC_DTYPE_FLOAT16) dispatch16<__half>(heads, d, f);
  else if (p.cache.dtype == PFC_DTYPE_BFLOAT16) dispatch16<__nv_bfloat16>(heads, d, f);
  else dispatch32(heads, d, f);
}

void check(const pfk_paged_attention_params& p) {
  const pfk_paged_cache& c = p.cache;
  check_paged_cache(c);
  const int64_t es = c.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  PFB_CHECK_ARG(c.head_dim % 8 == 0 && c.head_dim <= 256, "paged attention: head_dim must be a multiple of 8, at most 256");
  PFB_CHECK_ARG((uintptr_t)c.k % 16 == 0 && (uintptr_t)c.v % 16 == 0 && c.page_stride * es % 16 == 0 &&
                    c.token_stride * es % 16 == 0 && c.head_stride * es % 16 == 0,
                "paged attention: the cache's pointers and strides must be multiples of 16 bytes");
  PFB_CHECK_ARG(p.batch >= 0 && p.q_heads >= c.heads && p.q_heads % c.heads == 0 && p.q_heads <= 65536,
                "paged attention: q_heads must be a multiple of the cache's heads, at most 65536");
  PFB_CHECK_ARG(p.batch <= INT32_MAX / p.q_heads, "paged attention: 2^31 or more query heads in a batch");
  PFB_CHECK_ARG(p.table_width >= 0 && p.table_width <= INT32_MAX && p.table_stride >= 0,
                "paged attention: bad block table size");
  PFB_CHECK_ARG(p.window >= 0, "paged attention: negative window");
  PFB_CHECK_ARG(std::isfinite(p.scale), "paged attention: scale is not finite");
}

constexpr int64_t kClusterTiles = 64;  // of 64 keys: the longest sequences that clusters take

struct Plan {
  int ctas, heads;
  int ranks;  // CTAs of a unit's cluster; 0: runs of the list of all tiles
  int64_t stats_at, parts_at, bytes;
};

Plan plan_of(const pfk_paged_attention_params& p) {
  Plan w;
  const int64_t group = p.q_heads / p.cache.heads;
  w.heads = (int)std::min<int64_t>(group, unit_heads(p));
  dispatch(p, [&](auto k) { w.ctas = wave<decltype(k)>(); });
  // Few units with tables for short sequences: a cluster takes each, with no
  // list, no workspace and no second launch (one sequence, 8 units, list /
  // cluster: 100 keys 9.4 / 7.3 us, 1000 keys 11.3 / 8.0, 4096 keys 14.3 /
  // 13.6, 16384 keys 28 / 47; 8 sequences of up to 1000 keys, 64 units: 15.4
  // / 20.4).
  int64_t seen = p.table_width * p.cache.page_size;
  if (p.window) seen = std::min<int64_t>(seen, std::min<int64_t>(p.window, INT32_MAX) + 64);
  const int64_t units = p.batch * p.cache.heads * ceil_div(group, unit_heads(p)), tiles = ceil_div(seen, 64);
  w.ranks = 0;
  w.stats_at = w.parts_at = w.bytes = 0;
  if (tiles <= kClusterTiles && units * kMostRanks <= device_sm_count(current_device())) {
    w.ranks = 1;
    while (w.ranks < kMostRanks && w.ranks < tiles) w.ranks *= 2;
    return w;
  }
  w.stats_at = (int64_t)w.ctas * 16;
  w.parts_at = round_up(w.stats_at + (int64_t)w.ctas * 2 * w.heads * 8, 16);
  w.bytes = w.parts_at + (int64_t)w.ctas * 2 * w.heads * p.cache.head_dim * 4;
  return w;
}

int64_t gcd(int64_t a, int64_t b) {
  while (b) {
    const int64_t r = a % b;
    a = b;
    b = r;
  }
  return a;
}

}  // namespace

size_t paged_attention_workspace(const pfk_paged_attention_params& p) {
  check(p);
  if (p.batch == 0) return 0;
  return (size_t)plan_of(p).bytes;
}

void launch_paged_attention(const pfk_paged_attention_params& p, cudaStream_t stream) {
  check(p);
  if (p.batch == 0) return;
  PFB_CHECK_ARG(p.q && p.out && p.seq_lens && (p.block_table || p.table_width == 0), "paged attention: null pointer");
  // a CTA reads its unit's queries before any of the unit's outputs are
  // written, so the output may take the queries' place, row for row
  PFB_CHECK_ARG(p.out != p.q || ((p.batch == 1 || p.q_sb == p.o_sb) && (p.q_heads == 1 || p.q_sh == p.o_sh)),
                "paged attention: out shares q's memory with other strides");
  const pfk_paged_cache& c = p.cache;
  const int64_t es = c.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  Args a = {};
  // places in the cache fit 32 bits in units of the strides' common divisor
  const int64_t page_bytes = c.num_pages > 1 ? c.page_stride * es : 0, token_bytes = c.page_size > 1 ? c.token_stride * es : 0;
  const int64_t unit = std::max<int64_t>(16, gcd(page_bytes, token_bytes));
  const int64_t span = (c.num_pages - 1) * (page_bytes / unit) + (c.page_size - 1) * (token_bytes / unit);
  PFB_CHECK_ARG(span < 0xffffffffll, "paged attention: the cache spans more than 2^32 - 1 of its strides' common divisor");
  const Plan w = plan_of(p);
  PFB_CHECK_ARG(w.bytes == 0 || (p.workspace && p.workspace_bytes >= (size_t)w.bytes && (uintptr_t)p.workspace % 16 == 0),
                "paged attention: workspace missing, too small or not 16-byte aligned");
  a.k = (const char*)c.k;
  a.v = (const char*)c.v;
  a.unit_bytes = (unsigned long long)unit;
  a.page_units = (unsigned)(page_bytes / unit);
  a.token_units = (unsigned)(token_bytes / unit);
  a.head_bytes = c.head_stride * es;
  a.num_pages = (unsigned)c.num_pages;
  a.by_page = FastDiv((unsigned)c.page_size);
  a.err = c.err;
  a.batch = (int)p.batch;
  a.q_heads = (int)p.q_heads;
  a.kv_heads = (int)c.heads;
  a.group = (int)(p.q_heads / c.heads);
  a.unit_heads = unit_heads(p);
  a.chunks = (int)ceil_div(a.group, a.unit_heads);
  a.head_dim = (int)c.head_dim;
  a.q = p.q;
  a.q_sb = p.q_sb;
  a.q_sh = p.q_sh;
  a.out = p.out;
  a.o_sb = p.o_sb;
  a.o_sh = p.o_sh;
  a.lse = p.lse;
  a.table = p.block_table;
  a.table_stride = p.table_stride;
  a.seq_lens = p.seq_lens;
  a.most = std::min<int64_t>(p.table_width * c.page_size, INT32_MAX - 64);
  a.window = (int)std::min<int64_t>(p.window, INT32_MAX);
  a.scale = p.scale;
  char* ws = (char*)p.workspace;
  a.records = (int4*)ws;
  a.stats = (float2*)(ws + w.stats_at);
  a.parts = (float*)(ws + w.parts_at);
  a.ctas = w.ctas;
  a.heads = w.heads;
  dispatch(p, [&](auto k) { launch_sized<decltype(k)>(a, w.ranks, stream); });
}

}  // namespace pfb
