// The kernels of cache4_attention.cu: attention of one new token per sequence over a paged
// key-value cache held in 4 bits.
//
//   s_j = scale q.k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//   k_j = low + step * code for each group of values, v_j likewise
//
// A key and its value are D + 8 * groups bytes for 4 * D * G operations (G
// query heads of a unit): memory bounds it only as long as the codes reach the
// tensor cores in few instructions.
//
// Codes as operands.  The bits of a code c in the lowest or second lowest
// nibble of a 16-bit half are the subnormal fp16 numbers c 2^-24 and c 2^-20,
// which the tensor cores multiply exactly.  So a word of 8 codes becomes four
// operand registers by one shift and four masks, with no conversion and
// nothing to subtract.  Scales and lows are applied to sums instead:
//   q.k = sum over groups of step (q.code) + low (sum of q),
//   sum_j p_j v_j = sum_j (p_j step_j) code_j + sum_j p_j low_j.
// q enters as fp16 numbers scaled by a power of two for each head, its largest
// in 2^14 ... 2^15 and a sixteenth of that beside the codes that count sixteen
// times: exact for fp16 and bf16 down to 2^-20 of the head's largest, and in
// two parts (2^-22) for fp32.  p step enters as a multiple of a power of two
// that follows the largest product of its head and group so far (the largest
// step may be that of a key without weight), in two parts, which lose 2^-22 of
// a product (2^-21 where 16-bit calls truncate the high one), or 2^-25 of that
// power, of which the largest is near 2^8: one alone, 2^-11, showed in bf16
// outputs, whose error rose from 1.66e-3 to 1.72e-3.  An instruction has eight
// columns: a unit of up to four heads has the two parts of a head side by side,
// so that a lane has the weights of one head and adds both parts' sums (128
// sequences, bf16: 165 us; two instructions took 200, and one part alone, with
// two heads a lane, 169); more heads take two instructions (one sequence of
// 131071, 8 heads a unit, bf16: 53 us; one part took 43).  For fp32 the codes
// are centred, c - 8 (four instructions a word more): with many keys the values
// average out, and the large part that codes from 0 on have in common lost 5e-5
// of what remains to the tensor cores' truncation.
//
// Work.  As for the cache in the model's type: a unit is one sequence, one
// key-value head and up to 8 of its query heads; its keys are cut into tiles,
// a step of a CTA's 4 warps each; the tiles of all units form one list, of
// which each CTA of one wave takes an equal run, and a second small kernel
// joins the shares of units that several CTAs have, in a fixed order.  Few
// units of short sequences have a cluster of CTAs each.
//
// Step.  A warp takes 32 keys (16 of heads above 128 values, of pages that are
// no multiple of 16 tokens, and in clusters): lane (g, t) = (lane / 4, lane %
// 4) holds a quarter of the codes of key rows g and g + 8 (and 16 on), and an
// eighth of those of value rows 2t, 2t + 1, 2t + 8 and 2t + 9, which the cache
// keeps in pairs as the operand wants them.  S^T = K Q^T and O^T = V^T P^T, P
// turned by movmatrix in between.  The maxima move only where a score is 2^7
// above them, and keys are masked only in steps that do not see all of theirs.
// Scores, maxima, sums and outputs are held in fp32, and what the tensor cores
// add up, a group's products or a step's, is added to them in fp32, rounded to
// nearest: the cores truncate.
//
// Measured (device time, replayed from a graph; the bytes at 6.56 TB/s in
// brackets): 128 sequences of 2048 to 8192 keys, bf16, 32/8 heads of 128,
// groups of 64, 757 MB: 165 us (115); 48 of 0 to 8192, fp16, groups of 32: 79
// us (38.5); one of 131071, 64/8 heads, bf16: 53 us (23); one of 333 with a
// window of 250, fp32, 20 heads of 80: 5.9 us.  The long ones are bound by their
// instructions, 590 for a warp's 32 keys (groups of 32 750, 8 heads 770), and by
// what few warps an SM, 12 or 16, hide of latencies: 52 to 58 % of the issue
// slots are used.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "../common.hpp"
#include "cache4.cuh"
#include "decode.cuh"
#include "kernels.hpp"
#include "streamed.cuh"

namespace pfb {
namespace cache4 {

constexpr int kHeads = 8;      // query heads of a unit
constexpr int kMostRanks = 8;  // CTAs of a cluster

struct Args {
  const char *k, *v, *k_scales, *v_scales;
  unsigned num_pages, head_pairs;  // head_pairs: pairs of a page's tokens
  FastDiv by_page;
  int* err;
  int batch, q_heads, kv_heads, group;
  int chunks;  // a key-value head has `chunks` units of up to 8 query heads
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
  int heads;  // of a full unit: min(group, 8)
};

// CTAs of one wave of a call's kernel, and its launch; defined for each type
// in a file of its own.
template <typename T>
int wave_of(int width, int64_t group, bool runs, bool beside);
template <typename T>
void launch_of(Args& a, int width, int64_t group, bool runs, bool beside, int ranks, cudaStream_t stream);

}  // namespace cache4
}  // namespace pfb

#ifdef PFB_CACHE4_KERNELS
namespace pfb {
namespace cache4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr unsigned kNone = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Weights are held as 2^-24 exp(s - m): sums over values of 2^126, sixteen
// times as large where codes count sixteen times, stay in fp32's range for 2^18
// keys at the least.  (Multiplied: in the exponential's argument, 24 would leave
// 2^-20 of it to rounding, fp32 outputs an error of 4.1e-7 for 2.3e-7.)
constexpr int kShift = -24;
constexpr float kWeight = 0x1p-24f;
constexpr float kSlack = 3.f;  // of 2: m moves when a score is this far above it (a weight is below 2^-21)
// Weights times steps enter as multiples of a power of two, their unit: below
// 2^8 of it when it is chosen, and below 2^15 as long as the steps' bits are
// below the unit's and kRoom (Layout).

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

__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  mma16(c, a0, a1, a2, a3, b0, b1, __half());
}

// c = the product, with nothing added
__device__ __forceinline__ void mma_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ unsigned pack_half(float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const unsigned*>(&v);
}

__device__ __forceinline__ unsigned long long divide(unsigned long long a, unsigned long long b) {
  return ((a | b) >> 32) ? a / b : (unsigned)a / (unsigned)b;
}

// The codes of two nibbles of each half of w, the lowest and the second, as
// operands: subnormal (c 2^-24 and c 2^-20), or CENTRED, c - 8 both.
template <bool CENTRED>
__device__ __forceinline__ void operands(unsigned w, unsigned& even, unsigned& odd) {
  if constexpr (CENTRED) {  // 1024 + c - 1032, and (1024 + 16 c) / 16 - 72
    const unsigned e = (w & 0x000f000fu) | 0x64006400u, o = (w & 0x00f000f0u) | 0x64006400u;
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&e), __float2half2_rn(1032.f));
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&o), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
    even = *reinterpret_cast<const unsigned*>(&x);
    odd = *reinterpret_cast<const unsigned*>(&y);
  } else {
    even = w & 0x000f000fu;
    odd = w & 0x00f000f0u;
  }
}

// What a group's codes, or codes - 8, are added to.
template <bool CENTRED>
__device__ __forceinline__ float low_of(unsigned scales) {
  const float low = __uint_as_float(scales << 16);
  return CENTRED ? fmaf(__uint_as_float(scales & 0xffff0000u), 8.f, low) : low;
}

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// WORDS 32-bit words from p, aligned to their number's largest power of two
// (up to 4)
template <int WORDS>
__device__ __forceinline__ void load_words(unsigned* to, const char* p) {
  if constexpr (WORDS >= 4) {
    const uint4 r = load_stream(p);
    to[0] = r.x;
    to[1] = r.y;
    to[2] = r.z;
    to[3] = r.w;
    if constexpr (WORDS > 4) load_words<WORDS - 4>(to + 4, p + 16);
  } else if constexpr (WORDS >= 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(to[0]), "=r"(to[1]) : "l"(p));
    static_assert(WORDS == 2, "a power of two");
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(to[0]) : "l"(p));
  }
}

// T: of queries and output; W: the head's values with padding; G: a group's;
// BESIDE: units of up to 4 heads, with both parts of a weight in one instruction.
template <typename T, int W, int G, bool RUNS, bool BESIDE>
struct Layout {
  static constexpr int kBlocks = W / 32;
  static constexpr int kPaired = kBlocks & ~1;
  static constexpr int kFold = G < W ? G / 32 : kBlocks;            // blocks of a group
  static constexpr int kGroups = (kBlocks + kFold - 1) / kFold;
  static constexpr int kScales = kGroups <= 1 ? 1 : kGroups <= 2 ? 2 : kGroups <= 4 ? 4 : 8;  // words of a record
  static constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
  static constexpr int kPParts = BESIDE ? 1 : 2;  // instructions for a weight's parts
  static constexpr int kOwn = BESIDE ? 1 : 2;     // heads of a lane
  static constexpr unsigned kRound = sizeof(T) == 4 ? 0x1000 : 0;  // BESIDE: high parts are rounded, or truncated
  static constexpr bool kCentred = sizeof(T) == 4;
  // what the codes' operands and q's scaling leave to multiply with
  static constexpr int kQShift = kCentred ? -14 : 10;  // of 2, with q's exponent
  static constexpr float kOdd = kCentred ? 1.f : 0x1p-4f;
  // Units are held times what the codes' operands leave, 2^24, so that sums do not leave fp32's range: the least one's
  // bits, how far a step's may be above a unit's, and those of a unit and of its inverse, without that factor, together.
  static constexpr int kLeft = kCentred ? 0 : 24;
  static constexpr unsigned kLeastUnit = (unsigned)(1 + kLeft) << 23, kRoom = (unsigned)(12 - kShift - kLeft) << 23;
  static constexpr unsigned kInverse = (unsigned)(2 * 127 + kLeft) << 23;
  static constexpr int kRows = RUNS && W <= 128 ? 2 : 1;  // blocks of 16 keys of a warp's step
  static constexpr int kTile = 16 * kRows * kWarps;
  static constexpr int kPitch = W + 4;
  static constexpr size_t q_bytes = (size_t)kQParts * kBlocks * 32 * 16;
  static constexpr size_t o_bytes = (size_t)kWarps * kHeads * kPitch * 4;
  static constexpr size_t smem = q_bytes + o_bytes;
  // CTAs that share an SM: more warps help (128 sequences of 5000 keys, bf16,
  // groups of 64: 165 us with four, 170 with three), but not where 128
  // registers a thread spill (fp16, groups of 32: 84 us for 80; one of 131071
  // keys, 8 heads a unit, bf16: 51.3 us for 50.3)
  static constexpr int kResident = W <= 64 ? 4 : W <= 128 ? (sizeof(T) == 2 && kGroups <= 2 && BESIDE ? 4 : 3) : 2;
};

// CLUSTER: a cluster of CTAs for each unit, each an equal part of its tiles;
// otherwise runs of the list of all tiles.  RUNS: pages are multiples of 16
// tokens, so that 16 keys of a step follow one another in memory: a lane's
// rows are at fixed distances, and only the first's place is looked up.
template <typename T, int W, int G, bool CLUSTER, bool RUNS, bool BESIDE>
__global__ void __launch_bounds__(kThreads, (Layout<T, W, G, RUNS, BESIDE>::kResident)) attend_kernel(Args a) {
  using L = Layout<T, W, G, RUNS, BESIDE>;
  constexpr int R = L::kRows, B = L::kBlocks, NG = L::kGroups, H = L::kOwn;
  extern __shared__ __align__(16) char smem[];
  uint4* qs = reinterpret_cast<uint4*>(smem);  // [part][block][lane]
  float* os = reinterpret_cast<float*>(smem + L::q_bytes);
  __shared__ float ms[kWarps * kHeads], ls[kWarps * kHeads];  // [warp][head] maxima, sums
  __shared__ float factors[kHeads], q_sums[NG][kHeads];
  __shared__ long long scan[kWarps];
  __shared__ int found_row;
  __shared__ long long found_before;
  __shared__ Span found_span;
  __shared__ float2 part[kHeads];  // of a cluster's CTA: each head's maximum and sum

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  begin();
  const int per_row = a.kv_heads * a.chunks;
  int row, unit, tile;  // unit: of the row
  Span sp;
  long long t0, t1, list_total = 0;
  int list_ctas = 0;
  if constexpr (CLUSTER) {
    const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const int u = blockIdx.x / ranks;
    row = u / per_row;
    unit = u - row * per_row;
    sp = span_of<L::kTile>(a, row);
    t0 = (long long)sp.tiles * rank / ranks;
    t1 = (long long)sp.tiles * (rank + 1) / ranks;
    tile = (int)t0;
    if (t0 == t1 && tid < kHeads) part[tid] = make_float2(-INFINITY, 0.f);
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
    // equal runs of at least two tiles: more shares cost more than they save
    const int ctas = (int)min((long long)a.ctas, (total + 1) / 2);
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

  // The loads run ahead of the products and over the borders of units: ahead
  // stands at the step after the next, whose place in the cache it looks up.
  struct {
    int left, row, unit, tile, begin, end, tiles;
  } ahead = {(int)min(t1 - t0, (long long)INT_MAX), row, unit, tile, sp.begin, sp.end, sp.tiles};
  struct Place {
    unsigned where;  // the lane's key's (lane modulo their number) offset among its head's records of the page
    unsigned page;   // times the pages' heads
    unsigned seen;   // a bit for each of the warp's keys
  };
  constexpr unsigned kAll = R == 2 ? 0xffffffffu : 0xffffu;
  auto place = [&]() -> Place {
    Place p = {0, 0, 0};
    if (ahead.left == 0) return p;
    const int head = ahead.unit / a.chunks;
    const int start = (ahead.begin / L::kTile + ahead.tile) * L::kTile + warp * 16 * R, key = start + (lane & (16 * R - 1));
    // RUNS: the first of 16 keys has a place if any of them is seen
    const int low = RUNS ? key & ~15 : key, high = RUNS ? key | 15 : key;
    bool seen = false;
    if (low < ahead.end && high >= ahead.begin) {
      const unsigned i = a.by_page.div((unsigned)key);
      const unsigned page = (unsigned)a.table[(long long)ahead.row * a.table_stride + i];
      if (page < a.num_pages) {
        p.where = (unsigned)key - i * a.by_page.d;
        p.page = page * (unsigned)a.kv_heads + (unsigned)head;
        seen = key >= ahead.begin && key < ahead.end;
      } else if (a.err) {
        *a.err = PFC_ERR_INVALID_ARGUMENT;
      }
    }
    p.seen = __ballot_sync(~0u, seen) & kAll;
    --ahead.left;
    if (++ahead.tile == ahead.tiles) {
      ahead.tile = 0;
      if (++ahead.unit == per_row) {
        ahead.unit = 0;
        if (ahead.left) {
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
  // Keys that are not there (masked, or of a bad page) are read from some
  // record (the page's, or the first): its codes are finite, whatever they
  // are, and its scales are put away where not all of a step's keys are seen.
  constexpr int VK = RUNS ? 2 : 4;  // loads of value rows: of two keys next to each other, or of one
  unsigned kc[R][2][B], vc[R][VK][B];  // codes; of values, 4 of an even token in the low half, of the odd one in the high half
  unsigned kw[R][2][L::kScales], vw[R][2][L::kScales];
  // the keys that are loaded next: their records, and the values' pairs of tokens (RUNS: of the first of 16)
  unsigned next_k[R][RUNS ? 1 : 2], next_v[R][RUNS ? 1 : 4], next_seen, seen, odd = 0;
  auto aim = [&](const Place& p) {
    next_seen = p.seen;
    const unsigned record = p.page * a.by_page.d + p.where, pair = p.page * a.head_pairs + (p.where >> 1);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if constexpr (RUNS) {
        next_k[r][0] = __shfl_sync(~0u, record, 16 * r);
        next_v[r][0] = __shfl_sync(~0u, pair, 16 * r);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) next_k[r][i] = __shfl_sync(~0u, record, 16 * r + 8 * i + g);
#pragma unroll
        for (int i = 0; i < 4; ++i) next_v[r][i] = __shfl_sync(~0u, pair, 16 * r + 8 * (i >> 1) + 2 * t + (i & 1));
      }
    }
  };
  // The lane's places in record 0 (RUNS: of its row among 16): the record's
  // offset is one multiplication and addition, the other rows' an immediate.
  const char* const lane_k = a.k + (RUNS ? g * (W / 2) : 0) + t * (4 * L::kPaired);
  const char* const lane_v = a.v + (RUNS ? t * W : 0) + g * (4 * L::kPaired);
  const char* const lane_ks = a.k_scales + (RUNS ? g * (4 * L::kScales) : 0);
  const char* const lane_vs = a.v_scales + (RUNS ? g * (4 * L::kScales) : 0);
  auto load_k = [&]() {
    seen = next_seen;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned long long u = next_k[r][RUNS ? 0 : i];
        const int more = RUNS ? 8 * i : 0;  // rows
        const char* at = lane_k + u * (W / 2) + more * (W / 2);
        load_words<L::kPaired>(kc[r][i], at);
        if constexpr (B & 1) load_words<1>(kc[r][i] + L::kPaired, at + 16 * L::kPaired - t * (4 * L::kPaired - 4));
        load_words<L::kScales>(kw[r][i], lane_ks + u * (4 * L::kScales) + more * (4 * L::kScales));
        load_words<L::kScales>(vw[r][i], lane_vs + u * (4 * L::kScales) + more * (4 * L::kScales));
      }
  };
  auto load_v = [&](unsigned parity) {
    odd = parity;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < VK; ++i) {
        const unsigned long long u = next_v[r][RUNS ? 0 : i];
        const char* at = lane_v + u * W + (RUNS ? 4 * i * W : 0);
        load_words<L::kPaired>(vc[r][i], at);
        if constexpr (B & 1) load_words<1>(vc[r][i] + L::kPaired, at + 32 * L::kPaired - g * (4 * L::kPaired - 4));
      }
  };
  // of the lane's four keys of a step's values: which are odd tokens of their pages
  auto parity_of = [&](const Place& p) -> unsigned {
    if (RUNS) return 0;
    const unsigned odds = __ballot_sync(~0u, p.where & 1);
    return (odds >> (2 * t) & 3u) | (odds >> (8 + 2 * t) & 3u) << 2;
  };
  // Q in the order of the second operand's registers: a warp takes two heads
  // (BESIDE: each twice)
  auto stage_q = [&](int row, int first_q, int heads) {
    const T* qp = (const T*)a.q + (long long)row * a.q_sb + (long long)first_q * a.q_sh;
    __half* to = reinterpret_cast<__half*>(qs);
#pragma unroll
    for (int i = 0; i < kHeads / kWarps; ++i) {
      const int h = warp * (kHeads / kWarps) + i, from = BESIDE ? h >> 1 : h;
      float x[B], top = 0.f;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const int d = 32 * j + lane;
        x[j] = from < heads && d < a.head_dim ? to_float<T>(qp[from * a.q_sh + d]) : 0.f;
        top = fmaxf(top, fabsf(x[j]));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      // its exponent, not so low that the factor leaves fp32's range
      const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
      const float times = __uint_as_float((unsigned)(127 + 14 - e) << 23);
      if (lane == 0) {  // times 2^(e + kQShift), in two steps: the power alone may leave fp32's range
        const int half = (e + L::kQShift) >> 1, rest = e + L::kQShift - half;
        factors[h] = a.scale * kLog2e * __uint_as_float((unsigned)(127 + half) << 23) * __uint_as_float((unsigned)(127 + rest) << 23);
      }
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        float s = x[j];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        sum += s;
        if (j % L::kFold == L::kFold - 1 || j == B - 1) {
          if (lane == 0) q_sums[j / L::kFold][h] = sum * (a.scale * kLog2e);
          sum = 0.f;
        }
        // value 32j + 8 (lane / 8) + b goes with nibble b, whose mask and shift make it one of four operand halves
        const int b = lane & 7, comp = (b & 1) * 2 + ((b >> 1) & 1);
        const float v = x[j] * times * (!L::kCentred && b & 1 ? 0.0625f : 1.f);
        const int at = ((j * 32 + h * 4 + (lane >> 3)) * 4 + comp) * 2 + (b >> 2);
        const __half hi = __float2half_rn(v);
        to[at] = hi;
        if constexpr (L::kQParts == 2) to[at + B * 32 * 8] = __float2half_rn(v - __half2float(hi));
      }
    }
  };
  // the first unit's before the chain of loads that leads to its first keys
  if (t0 < t1) {
    const int head = unit / a.chunks, first_q = head * a.group + (unit - head * a.chunks) * kHeads;
    stage_q(row, first_q, min(kHeads, (head + 1) * a.group - first_q));
  }
  Place next = place();
  aim(next);
  load_k();
  load_v(parity_of(next));
  next = place();

  for (long long at = t0; at < t1;) {
    while (sp.tiles == 0) sp = span_of<L::kTile>(a, ++row);
    const int count = (int)min((long long)(sp.tiles - tile), t1 - at);
    const int head = unit / a.chunks;
    const int first_q = head * a.group + (unit - head * a.chunks) * kHeads;
    const int heads = min(kHeads, (head + 1) * a.group - first_q);

    if (at != t0) {
      __syncthreads();  // the previous piece's reads of shared memory are over
      stage_q(row, first_q, heads);
    }
    __syncthreads();

    // A lane has query heads 2t and 2t + 1 (BESIDE: t); of o the values 32b + 4g + 2j, and behind the heads' the next
    // ones, sixteenfold
    float m[H], l[H], z[NG][H], o[B][2][2 * H], f[H], qsum[NG][H];
    unsigned unit_of[NG][H];  // what a head's weights times a group's steps are multiples of: a power of two, its bits
#pragma unroll
    for (int i = 0; i < H; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
      f[i] = factors[2 * t + i];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        z[n][i] = 0.f;
        unit_of[n][i] = L::kLeastUnit;
        qsum[n][i] = q_sums[n][2 * t + i];
      }
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2 * H; ++i) o[b][j][i] = 0.f;

    for (int step = 0; step < count; ++step) {
      float s[R][2 * H], lows[R][2 * H];  // of a key and the one 8 on, H heads each
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float sum[R][4];
#pragma unroll
        for (int j = n * L::kFold; j < (n + 1) * L::kFold && j < B; ++j) {
          const uint4 qv = qs[j * 32 + lane];
          uint4 ql;
          if constexpr (L::kQParts == 2) ql = qs[(B + j) * 32 + lane];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const unsigned c0 = kc[r][0][j], c1 = kc[r][1][j];
            unsigned a0, a1, a2, a3, b0, b1, b2, b3;
            operands<L::kCentred>(c0, a0, b0);
            operands<L::kCentred>(c1, a1, b1);
            operands<L::kCentred>(c0 >> 8, a2, b2);
            operands<L::kCentred>(c1 >> 8, a3, b3);
            const uint4 first = L::kQParts == 2 ? ql : qv;
            if (j == n * L::kFold) mma_first(sum[r], a0, a1, a2, a3, first.x, first.y);
            else mma(sum[r], a0, a1, a2, a3, first.x, first.y);
            mma(sum[r], b0, b1, b2, b3, first.z, first.w);
            if constexpr (L::kQParts == 2) {
              mma(sum[r], a0, a1, a2, a3, qv.x, qv.y);
              mma(sum[r], b0, b1, b2, b3, qv.z, qv.w);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 2 * H; ++i) {
            const unsigned w = kw[r][i / H][n];
            const float step = __uint_as_float(w & 0xffff0000u), low = low_of<L::kCentred>(w), x = sum[r][BESIDE ? 2 * i : i];
            s[r][i] = n ? fmaf(step, x, s[r][i]) : step * x;
            lows[r][i] = n ? fmaf(low, qsum[n][i % H], lows[r][i]) : low * qsum[n][i % H];
          }
      }
      // the values' scales are kept: the next keys' come with their keys
      unsigned vs[R][2][NG];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NG; ++n) vs[r][i][n] = vw[r][i][n];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2 * H; ++i) s[r][i] = fmaf(s[r][i], f[i % H], lows[r][i]);
      if (seen != kAll) {  // the same in all lanes
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (seen >> (16 * r + 8 * i + g) & 1) continue;
#pragma unroll
            for (int h = 0; h < H; ++h) s[r][H * i + h] = -INFINITY;
#pragma unroll
            for (int n = 0; n < NG; ++n) vs[r][i][n] = 0;
          }
      }
      aim(next);
      load_k();

      // The maxima move, and with them all sums, only where a score is far
      // above them; the units of weights times steps, then or where a step is
      // so large that a product might leave fp16's range: to 2^-8 of the largest
      // product, or up to 2^8 more where that spares the next steps as large.
      float top[H];
      bool rises = false, large = false;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        top[i] = s[0][i];
#pragma unroll
        for (int k = 1; k < 2 * R; ++k) top[i] = fmaxf(top[i], s[k >> 1][H * (k & 1) + i]);
        rises |= top[i] > m[i] + kSlack;
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        unsigned largest = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) largest = max(largest, max(vs[r][0][n], vs[r][1][n]));
        large |= largest >= min(unit_of[n][0], unit_of[n][H - 1]) + L::kRoom;
      }
      const bool moved = __any_sync(~0u, rises);
      if (moved || __any_sync(~0u, large)) {
        if (moved) {
#pragma unroll
          for (int i = 0; i < H; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 4));
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 8));
            top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 16));
            const float to = fmaxf(m[i], top[i]);
            const float down = to == -INFINITY ? 1.f : exp2_fast(m[i] - to);
            m[i] = to;
            l[i] *= down;
#pragma unroll
            for (int n = 0; n < NG; ++n) z[n][i] *= down;
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                o[b][j][i] *= down;
                o[b][j][i + H] *= down;
              }
          }
        }
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int i = 0; i < H; ++i) {
            // exponents: of the largest product (which is below 2^(product - 252)), and of the largest step
            int product = 0, step = 0;
#pragma unroll
            for (int k = 0; k < 2 * R; ++k) {
              const float weight = exp2_fast(s[k >> 1][H * (k & 1) + i] - (m[i] == -INFINITY ? 0.f : m[i])) * kWeight;
              const int u = __float_as_uint(weight) >> 23, v = vs[k >> 1][k & 1][n] >> 23;
              if (u && v) product = max(product, u + v);
              step = max(step, v);
            }
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              product = max(product, __shfl_xor_sync(~0u, product, off));
              step = max(step, __shfl_xor_sync(~0u, step, off));
            }
            const int enough = product - 133 + L::kLeft, unit = max(enough, min(step + kShift - 7 + L::kLeft, enough + 8));
            const unsigned to = (unsigned)min(max(unit, (int)(L::kLeastUnit >> 23)), 253) << 23;
            unit_of[n][i] = moved ? to : max(to, unit_of[n][i]);
          }
      }
      float base[H];
#pragma unroll
      for (int i = 0; i < H; ++i) base[i] = m[i] == -INFINITY ? 0.f : m[i];
      float p[R][2 * H];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2 * H; ++i) {
          p[r][i] = exp2_fast(s[r][i] - base[i % H]) * kWeight;
          l[i % H] += p[r][i];
        }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        unsigned pt[R][L::kPParts][2];  // weights times steps as the second operand, of keys 0-7 and 8-15
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned w = vs[r][i][n];
            const float st = __uint_as_float(w & 0xffff0000u), low = low_of<L::kCentred>(w);
#pragma unroll
            for (int h = 0; h < H; ++h) z[n][h] = fmaf(p[r][H * i + h], low, z[n][h]);
            const float x = p[r][H * i] * __uint_as_float(L::kInverse - unit_of[n][0]) * st;
            if constexpr (BESIDE) {  // both parts, next to each other
              const float hi = __uint_as_float((__float_as_uint(x) + L::kRound) & 0xffffe000u);  // 11 bits of x
              pt[r][0][i] = transpose8x8(pack_half(hi, x - hi));
            } else {
              const float y = p[r][H * i + 1] * __uint_as_float(L::kInverse - unit_of[n][H - 1]) * st;
              const unsigned hi = pack_half(x, y);
              const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              pt[r][0][i] = transpose8x8(hi);
              pt[r][1][i] = transpose8x8(pack_half(x - back.x, y - back.y));
            }
          }
#pragma unroll
        for (int b = n * L::kFold; b < (n + 1) * L::kFold && b < B; ++b) {
          float sum[2][4];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            unsigned x = vc[r][0][b], y = vc[r][1][b];  // of keys 2t and 2t + 1, and of 2t + 8 and 2t + 9
            if constexpr (!RUNS) {
              x = __byte_perm(vc[r][0][b], vc[r][1][b], (odd & 1 ? 0x32 : 0x10) | (odd & 2 ? 0x7600 : 0x5400));
              y = __byte_perm(vc[r][2][b], vc[r][3][b], (odd & 4 ? 0x32 : 0x10) | (odd & 8 ? 0x7600 : 0x5400));
            }
            unsigned e0, o0, e1, o1, e2, o2, e3, o3;
            operands<L::kCentred>(x, e0, o0);
            operands<L::kCentred>(y, e1, o1);
            operands<L::kCentred>(x >> 8, e2, o2);
            operands<L::kCentred>(y >> 8, e3, o3);
#pragma unroll
            for (int q = L::kPParts - 1; q >= 0; --q) {
              if (r == 0 && q == L::kPParts - 1) {
                mma_first(sum[0], e0, o0, e1, o1, pt[r][q][0], pt[r][q][1]);
                mma_first(sum[1], e2, o2, e3, o3, pt[r][q][0], pt[r][q][1]);
              } else {
                mma(sum[0], e0, o0, e1, o1, pt[r][q][0], pt[r][q][1]);
                mma(sum[1], e2, o2, e3, o3, pt[r][q][0], pt[r][q][1]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2 * H; ++i) o[b][j][i] = fmaf(__uint_as_float(unit_of[n][i % H]), BESIDE ? sum[j][2 * i] + sum[j][2 * i + 1] : sum[j][i], o[b][j][i]);
        }
      }
      load_v(parity_of(next));
      next = place();
    }

    // join the warps
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const int h = warp * kHeads + H * t + i;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[i] += __shfl_xor_sync(~0u, l[i], off);
#pragma unroll
        for (int n = 0; n < NG; ++n) z[n][i] += __shfl_xor_sync(~0u, z[n][i], off);
      }
      if (g == 0) {
        ms[h] = m[i];
        ls[h] = l[i];
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const float low = z[b / L::kFold][i];
        float4 v;
        v.x = o[b][0][i] + low;
        v.y = fmaf(o[b][0][i + H], L::kOdd, low);
        v.z = o[b][1][i] + low;
        v.w = fmaf(o[b][1][i + H], L::kOdd, low);
        *reinterpret_cast<float4*>(os + (size_t)h * L::kPitch + 32 * b + 4 * g) = v;
      }
    }
    __syncthreads();
    const bool whole = tile == 0 && count == sp.tiles;
    const int slot = tile == 0 ? 1 : 0;  // a unit that began here, or one that began in an earlier CTA
    const long long share = ((long long)blockIdx.x * 2 + slot) * a.heads;
    for (int i = tid; i < heads * a.head_dim; i += kThreads) {
      const int h = i / a.head_dim, d = i - h * a.head_dim;
      float most = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) most = fmaxf(most, ms[w * kHeads + h]);
      float v = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = ms[w * kHeads + h];
        const float by = mw == -INFINITY ? (most == -INFINITY ? 1.f : 0.f) : exp2_fast(mw - most);
        v += by * os[(size_t)(w * kHeads + h) * L::kPitch + d];
        sum += by * ls[w * kHeads + h];
      }
      if constexpr (CLUSTER) {
        os[(size_t)h * L::kPitch + d] = v;  // read and written by this thread alone
        if (d == 0) part[h] = make_float2(most, sum);
      } else if (whole) {
        ((T*)a.out)[(long long)row * a.o_sb + (long long)(first_q + h) * a.o_sh + d] = from_float<T>(sum == 0.f ? 0.f : v / sum);
        if (d == 0 && a.lse) a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (most + log2f(sum * (1.f / kWeight))) * kLn2;
      } else {
        a.parts[(share + h) * a.head_dim + d] = v;
        if (d == 0) a.stats[share + h] = make_float2(most, sum);
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
    const int head = unit / a.chunks, first_q = head * a.group + (unit - head * a.chunks) * kHeads;
    const int heads = min(kHeads, (head + 1) * a.group - first_q);
    for (int i = (int)cluster.block_rank() * kThreads + tid; i < heads * a.head_dim; i += kThreads * ranks) {
      const int h = i / a.head_dim, d = i - h * a.head_dim;
      float2 st[kMostRanks];
      float v[kMostRanks];
#pragma unroll
      for (int r = 0; r < kMostRanks; ++r) {
        st[r] = make_float2(-INFINITY, 0.f);
        v[r] = 0.f;
        if (r < ranks) {
          st[r] = cluster.map_shared_rank(part, r)[h];
          v[r] = cluster.map_shared_rank(os, r)[(size_t)h * L::kPitch + d];
        }
      }
      float most = -INFINITY, sum = 0.f, all = 0.f;
#pragma unroll
      for (int r = 0; r < kMostRanks; ++r) most = fmaxf(most, st[r].x);
#pragma unroll
      for (int r = 0; r < kMostRanks; ++r) {
        if (st[r].x == -INFINITY && st[r].y == 0.f) continue;  // no keys: its outputs were never written
        const float by = st[r].x == most ? 1.f : exp2_fast(st[r].x - most);
        all += by * v[r];
        sum += by * st[r].y;
      }
      ((T*)a.out)[(long long)row * a.o_sb + (long long)(first_q + h) * a.o_sh + d] = from_float<T>(sum == 0.f ? 0.f : all / sum);
      if (d == 0 && a.lse) a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (most + log2f(sum * (1.f / kWeight))) * kLn2;
    }
    cluster.sync();  // the others' reads of this CTA's part are over
  } else if (tid == 0) {
    a.records[blockIdx.x] = record;
  }
}

// A join's shares are split among groups of its threads.  Few units have many
// shares each: one CTA for a unit, of all the threads that it may have.  Many
// units have few shares each, and a CTA of 256 for each CTA of the first kernel,
// with no unit to look for (whole calls, bf16, heads of 128, us in the first form
// and in the second: 1 unit of 60000 keys 16.7 and 24.4, 8 33.8 and 35.1, 16 of
// up to 30000 22.9 and 23.6, 32 of up to 16384 23.9 and 24.1, 48 32.5 and 28.8,
// 128 44.6 and 34.4).
constexpr int kFewUnits = 32;

// CTA (c, h): joins the shares of query head h of a unit that went on beyond
// the CTA it began in, in a fixed order: with FIND the c-th such unit,
// else the one that began in CTA c of the first kernel; and writes the outputs
// of sequence c if it is empty.
template <typename T, int THREADS, bool FIND>
__global__ void __launch_bounds__(THREADS) join_kernel(Args a) {
  __shared__ float4 acc[THREADS];
  __shared__ float2 stats[THREADS / 16];
  const int tid = threadIdx.x;
  int c0 = blockIdx.x;
  begin();
  if (c0 < a.batch && span_of<64>(a, c0).tiles == 0) {
    for (int qh = blockIdx.y; qh < a.q_heads; qh += gridDim.y) {
      for (int d = tid; d < a.head_dim; d += THREADS)
        ((T*)a.out)[(long long)c0 * a.o_sb + (long long)qh * a.o_sh + d] = from_float<T>(0.f);
      if (tid == 0 && a.lse) a.lse[(long long)c0 * a.q_heads + qh] = -INFINITY;
    }
  }
  if constexpr (FIND) {
    __shared__ int in_warp[THREADS / 32], found;
    if (tid == 0) found = -1;
    int left = c0;  // such units before this CTA's that are still to come
    for (int base = 0; base < a.ctas; base += THREADS) {
      const bool on = base + tid < a.ctas && a.records[base + tid].w;
      const unsigned lanes = __ballot_sync(~0u, on);
      if (tid % 32 == 0) in_warp[tid / 32] = __popc(lanes);
      __syncthreads();
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < tid / 32) before += in_warp[w];
        all += in_warp[w];
      }
      if (on && before + __popc(lanes & ((1u << tid % 32) - 1)) == left) found = base + tid;
      left -= all;
      __syncthreads();
    }
    c0 = found;
    if (c0 < 0) return;
  }
  if (c0 >= a.ctas) return;
  const int4 rec = a.records[c0];
  if (!rec.w) return;
  const int b = rec.x, head = rec.y / a.chunks, h = blockIdx.y;
  const int qh = head * a.group + (rec.y - head * a.chunks) * kHeads + h;
  if (qh >= (head + 1) * a.group) return;
  const int shares = rec.z - c0 + 1;
  // the first share is slot 1 of its CTA, the others slot 0 of theirs
  auto share = [&](int i) -> long long { return ((long long)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * a.heads + h; };
  const int cols = a.head_dim / 4;                            // of 4 values
  const int across = cols <= 16 ? 16 : cols <= 32 ? 32 : 64;  // threads of a share
  const int groups = THREADS / across, gi = tid / across, col = tid % across;

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
  if constexpr (FIND) {  // many groups: by halves
    for (int half = groups / 2; half > 0; half /= 2) {
      if (gi >= half && gi < 2 * half) {
        acc[tid] = v;
        if (col == 0) stats[gi] = make_float2(top, sum);
      }
      __syncthreads();
      if (gi < half) join(stats[gi + half].x, stats[gi + half].y, acc[(gi + half) * across + col]);
    }
  } else {
    acc[tid] = v;
    if (col == 0) stats[gi] = make_float2(top, sum);
    __syncthreads();
    for (int w = 1; gi == 0 && w < groups; ++w) join(stats[w].x, stats[w].y, acc[w * across + col]);
  }
  if (gi == 0 && col < cols) {
    T* out = (T*)a.out + (long long)b * a.o_sb + (long long)qh * a.o_sh + col * 4;
    const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = from_float<T>(sum == 0.f ? 0.f : r[e] / sum);
    if (col == 0 && a.lse) a.lse[(long long)b * a.q_heads + qh] = sum == 0.f ? -INFINITY : (top + log2f(sum * (1.f / kWeight))) * kLn2;
  }
}

template <typename T_, int W, int G, bool RUNS, bool BESIDE>
struct Kernel {
  using T = T_;
  using L = Layout<T, W, G, RUNS, BESIDE>;
  using LC = Layout<T, W, G, false, false>;  // of the clusters' kernel
  static constexpr auto run = attend_kernel<T, W, G, false, RUNS, BESIDE>;
  static constexpr auto run_cluster = attend_kernel<T, W, G, true, false, false>;
};

// CTAs of one wave of a kernel on the current device, asked once per device.
template <class K>
int wave() {
  static std::once_flag once[64];
  static int ctas[64];
  const int dev = current_device();
  std::call_once(once[dev], [dev] {
    PFB_CUDA(cudaFuncSetAttribute(K::run, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)K::L::smem));
    PFB_CUDA(cudaFuncSetAttribute(K::run_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)K::LC::smem));
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
    launch_following<Args>(K::run_cluster, dim3((unsigned)ctas), kThreads, K::LC::smem, stream, a, ranks);
    return;
  }
  launch_following<Args>(K::run, dim3((unsigned)a.ctas), kThreads, K::L::smem, stream, a);
  const int64_t units = (int64_t)a.batch * a.kv_heads * a.chunks;
  if (units <= kFewUnits && units < a.ctas)
    launch_following<Args>(join_kernel<typename K::T, 1024, true>, dim3((unsigned)units, (unsigned)a.heads), 1024, 0, stream, a);
  else
    launch_following<Args>(join_kernel<typename K::T, 256, false>, dim3((unsigned)std::max(a.ctas, a.batch), (unsigned)a.heads), 256, 0, stream, a);
}

// Calls f(Kernel<...>()) for the call's sizes.  Groups as wide as the head are
// one group, whatever their size.
template <typename T, bool RUNS, bool BESIDE, class F>
void dispatch_sized(int width, int64_t group, F&& f) {
  if (width == 64) {
    group == 32 ? f(Kernel<T, 64, 32, RUNS, BESIDE>()) : f(Kernel<T, 64, 64, RUNS, BESIDE>());
  } else if (width == 96) {
    if (group == 32) f(Kernel<T, 96, 32, RUNS, BESIDE>());
    else group == 64 ? f(Kernel<T, 96, 64, RUNS, BESIDE>()) : f(Kernel<T, 96, 128, RUNS, BESIDE>());
  } else if (width == 128) {
    if (group == 32) f(Kernel<T, 128, 32, RUNS, BESIDE>());
    else group == 64 ? f(Kernel<T, 128, 64, RUNS, BESIDE>()) : f(Kernel<T, 128, 128, RUNS, BESIDE>());
  } else {
    if (group == 32) f(Kernel<T, 256, 32, RUNS, BESIDE>());
    else group == 64 ? f(Kernel<T, 256, 64, RUNS, BESIDE>()) : f(Kernel<T, 256, 128, RUNS, BESIDE>());
  }
}
template <typename T, class F>
void dispatch(int width, int64_t group, bool runs, bool beside, F&& f) {
  if (runs) beside ? dispatch_sized<T, true, true>(width, group, f) : dispatch_sized<T, true, false>(width, group, f);
  else beside ? dispatch_sized<T, false, true>(width, group, f) : dispatch_sized<T, false, false>(width, group, f);
}

}  // namespace

template <typename T>
int wave_of(int width, int64_t group, bool runs, bool beside) {
  int ctas = 0;
  dispatch<T>(width, group, runs, beside, [&](auto k) { ctas = wave<decltype(k)>(); });
  return ctas;
}

template <typename T>
void launch_of(Args& a, int width, int64_t group, bool runs, bool beside, int ranks, cudaStream_t stream) {
  dispatch<T>(width, group, runs, beside, [&](auto k) { launch_sized<decltype(k)>(a, ranks, stream); });
}

}  // namespace cache4
}  // namespace pfb
#endif  // PFB_CACHE4_KERNELS
