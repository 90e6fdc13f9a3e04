// cache4_attention.cu — attention of one new token per sequence over a paged
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
// two parts (2^-22) for fp32.  p step enters scaled by 2^14 over a power of
// two above the step's largest step (one reduction of the warp), in two parts
// for fp32 and fp16 and in one, 2^-12, for bf16 outputs, 2^-9.
//
// Work.  As for the cache in the model's type: a unit is one sequence, one
// key-value head and up to 8 of its query heads; its keys are cut into tiles,
// a step of a CTA's 4 warps each; the tiles of all units form one list, of
// which each CTA of one wave takes an equal run, and a second small kernel
// joins the shares of units that several CTAs have, in the order of the list.
// Few units of short sequences have a cluster of CTAs each.
//
// Step.  A warp takes 32 keys (16 of heads above 128 values): lane (g, t) =
// (lane / 4, lane % 4) holds a quarter of the codes of key rows g and g + 8
// (and 16 on) and an eighth of those of the value rows 2t, 2t + 1, 2t + 8, 2t
// + 9.  S^T = K Q^T and O^T = V^T P^T, P turned by movmatrix in between.
// Scores, maxima, sums and outputs are held in fp32, and what the tensor cores
// add up, a group's products or a step's, is added to them in fp32, rounded to
// nearest: the cores truncate.
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
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kHeads = 8;      // query heads of a unit
constexpr int kMostRanks = 8;  // CTAs of a cluster
constexpr unsigned kNone = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kShift = 14.f;  // weights are held as 2^14 exp(s - m)

struct Args {
  const char *k, *v, *k_scales, *v_scales;
  unsigned num_pages, page_records;  // page_records: heads * page_size
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

// T: of queries and output; W: the head's values with padding; G: a group's.
template <typename T, int W, int G>
struct Layout {
  static constexpr int kBlocks = W / 32;
  static constexpr int kPaired = kBlocks & ~1;
  static constexpr int kFold = G < W ? G / 32 : kBlocks;            // blocks of a group
  static constexpr int kGroups = (kBlocks + kFold - 1) / kFold;
  static constexpr int kScales = kGroups <= 1 ? 1 : kGroups <= 2 ? 2 : kGroups <= 4 ? 4 : 8;  // words of a record
  static constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
  static constexpr int kPParts = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
  static constexpr bool kCentred = sizeof(T) == 4;
  // what the codes' operands and q's scaling leave to multiply with
  static constexpr int kQShift = kCentred ? -14 : 10;  // of 2, with q's exponent
  static constexpr float kEven = kCentred ? 1.f : 0x1p24f, kOdd = kCentred ? 1.f : 0x1p20f;
  static constexpr int kRows = W <= 128 ? 2 : 1;  // blocks of 16 keys of a warp's step
  static constexpr int kTile = 16 * kRows * kWarps;
  static constexpr int kPitch = W + 4;
  static constexpr size_t q_bytes = (size_t)kQParts * kBlocks * 32 * 16;
  static constexpr size_t o_bytes = (size_t)kWarps * kHeads * kPitch * 4;
  static constexpr size_t smem = q_bytes + o_bytes;
  static constexpr int kResident = W <= 64 ? 4 : W <= 128 ? 3 : 2;  // CTAs that share an SM
};

// CLUSTER: a cluster of CTAs for each unit, each an equal part of its tiles;
// otherwise runs of the list of all tiles.
template <typename T, int W, int G, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, (Layout<T, W, G>::kResident)) attend_kernel(Args a) {
  using L = Layout<T, W, G>;
  constexpr int R = L::kRows, B = L::kBlocks, NG = L::kGroups;
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
    long long at;
    int row, unit, tile, begin, end, tiles;
  } ahead = {t0, row, unit, tile, sp.begin, sp.end, sp.tiles};
  auto place = [&]() -> unsigned {  // the record of the lane's key (lane modulo their number)
    unsigned where = kNone;
    if (ahead.at >= t1) return where;
    const int head = ahead.unit / a.chunks;
    const int key = (ahead.begin / L::kTile + ahead.tile) * L::kTile + warp * 16 * R + (lane & (16 * R - 1));
    if (key >= ahead.begin && key < ahead.end) {
      const unsigned i = a.by_page.div((unsigned)key);
      const unsigned page = (unsigned)a.table[(long long)ahead.row * a.table_stride + i];
      if (page < a.num_pages) where = page * a.page_records + (unsigned)head * a.by_page.d + ((unsigned)key - i * a.by_page.d);
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
    return where;
  };
  // Keys that are not there (masked, or of a bad page) have scales of 0 and
  // the codes of the first record: whatever those are, they are finite.
  unsigned kc[R][2][B], vc[R][4][(B + 1) / 2];  // codes; of values two blocks a word
  unsigned kw[R][2][L::kScales], vw[R][2][L::kScales];
  unsigned next_rec[R][2];  // records of the keys that are loaded next, kNone: not there
  const char* next_v[R][4];
  bool seen[R][2];
  auto aim = [&](unsigned p) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < 2; ++i) next_rec[r][i] = __shfl_sync(~0u, p, 16 * r + 8 * i + g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned u = __shfl_sync(~0u, p, 16 * r + 8 * (i >> 1) + 2 * t + (i & 1));
        next_v[r][i] = a.v + (unsigned long long)(u == kNone ? 0 : u) * (W / 2);
      }
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const unsigned u = next_rec[r][i];
        seen[r][i] = u != kNone;
        const char* at = a.k + (unsigned long long)(u == kNone ? 0 : u) * (W / 2);
        load_words<L::kPaired>(kc[r][i], at + t * (4 * L::kPaired));
        if constexpr (B & 1) load_words<1>(kc[r][i] + L::kPaired, at + 16 * L::kPaired + 4 * t);
#pragma unroll
        for (int s = 0; s < L::kScales; ++s) kw[r][i][s] = vw[r][i][s] = 0;
        if (u != kNone) {
          load_words<L::kScales>(kw[r][i], a.k_scales + (unsigned long long)u * (4 * L::kScales));
          load_words<L::kScales>(vw[r][i], a.v_scales + (unsigned long long)u * (4 * L::kScales));
        }
      }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        load_words<L::kPaired / 2>(vc[r][i], next_v[r][i] + g * (2 * L::kPaired));
        if constexpr (B & 1) {
          unsigned short h;
          asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(h) : "l"(next_v[r][i] + 16 * L::kPaired + 2 * g));
          vc[r][i][L::kPaired / 2] = h;
        }
      }
  };
  // Q in the order of the second operand's registers: a warp takes two heads
  auto stage_q = [&](int row, int first_q, int heads) {
    const T* qp = (const T*)a.q + (long long)row * a.q_sb + (long long)first_q * a.q_sh;
    __half* to = reinterpret_cast<__half*>(qs);
#pragma unroll
    for (int i = 0; i < kHeads / kWarps; ++i) {
      const int h = warp * (kHeads / kWarps) + i;
      float x[B], top = 0.f;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const int d = 32 * j + lane;
        x[j] = h < heads && d < a.head_dim ? to_float<T>(qp[h * a.q_sh + d]) : 0.f;
        top = fmaxf(top, fabsf(x[j]));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
      // its exponent, not so low that the factor leaves fp32's range
      const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
      const float times = __uint_as_float((unsigned)(127 + 14 - e) << 23);
      if (lane == 0) factors[h] = a.scale * kLog2e * exp2f((float)(e + L::kQShift));
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
  aim(place());
  load_k();
  load_v();
  unsigned next = place();

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

    // A lane has query heads 2t and 2t + 1; of o the values 32b + 4g + 2j (o[..][0..1]) and the next, sixteenfold
    float m[2], l[2], z[NG][2], o[B][2][4], f[2], qsum[NG][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
      f[i] = factors[2 * t + i];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        z[n][i] = 0.f;
        qsum[n][i] = q_sums[n][2 * t + i];
      }
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) o[b][j][0] = o[b][j][1] = o[b][j][2] = o[b][j][3] = 0.f;

    for (int step = 0; step < count; ++step) {
      bool live[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) live[r][i] = seen[r][i];
      float s[R][4], lows[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[r][i] = lows[r][i] = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float sum[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) sum[r][0] = sum[r][1] = sum[r][2] = sum[r][3] = 0.f;
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
            if constexpr (L::kQParts == 2) {
              mma(sum[r], a0, a1, a2, a3, ql.x, ql.y);
              mma(sum[r], b0, b1, b2, b3, ql.z, ql.w);
            }
            mma(sum[r], a0, a1, a2, a3, qv.x, qv.y);
            mma(sum[r], b0, b1, b2, b3, qv.z, qv.w);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned w = kw[r][i >> 1][n];
            s[r][i] = fmaf(__uint_as_float(w & 0xffff0000u), sum[r][i], s[r][i]);
            lows[r][i] = fmaf(low_of<L::kCentred>(w), qsum[n][i & 1], lows[r][i]);
          }
      }
      // the values' scales are kept: the next keys' come with their keys'
      unsigned vs[R][2][NG];
      unsigned largest = 0;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            vs[r][i][n] = vw[r][i][n];
            largest = max(largest, vw[r][i][n]);
          }
      aim(next);
      load_k();

      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[r][i] = live[r][i >> 1] ? fmaf(s[r][i], f[i & 1], lows[r][i]) : -INFINITY;
          top[i & 1] = fmaxf(top[i & 1], s[r][i]);
        }
      bool moved = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 4));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 8));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 16));
        moved |= top[i] > m[i];
      }
      if (__any_sync(~0u, moved)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
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
              o[b][j][i + 2] *= down;
            }
        }
      }
      // a power of two above the step's largest step, and its inverse; a NaN's exponent counts as the largest that a step has
      const unsigned e = min(__reduce_max_sync(~0u, largest) >> 23, 252u);
      const float above = __uint_as_float((e + 1) << 23), below = __uint_as_float((253u - e) << 23);
      unsigned pt[R][NG][L::kPParts][2];  // weights times steps as the second operand, of keys 0-7 and 8-15
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float base = m[i & 1] == -INFINITY ? 0.f : m[i & 1];
          p[i] = exp2_fast(s[r][i] - base + kShift);
          l[i & 1] += p[i];
        }
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const unsigned w = vs[r][i][n];
            const float st = __uint_as_float(w & 0xffff0000u) * below, low = low_of<L::kCentred>(w);
            z[n][0] = fmaf(p[2 * i], low, z[n][0]);
            z[n][1] = fmaf(p[2 * i + 1], low, z[n][1]);
            const float x = p[2 * i] * st, y = p[2 * i + 1] * st;
            const unsigned hi = pack_half(x, y);
            pt[r][n][0][i] = transpose8x8(hi);
            if constexpr (L::kPParts == 2) {
              const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              pt[r][n][1][i] = transpose8x8(pack_half(x - back.x, y - back.y));
            }
          }
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        constexpr int F = L::kFold;
        float sum[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) sum[j][0] = sum[j][1] = sum[j][2] = sum[j][3] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const unsigned sel = b & 1 ? 0x7632 : 0x5410;
          const unsigned x = __byte_perm(vc[r][0][b >> 1], vc[r][1][b >> 1], sel), y = __byte_perm(vc[r][2][b >> 1], vc[r][3][b >> 1], sel);
          unsigned e0, o0, e1, o1, e2, o2, e3, o3;
          operands<L::kCentred>(x, e0, o0);
          operands<L::kCentred>(y, e1, o1);
          operands<L::kCentred>(x >> 8, e2, o2);
          operands<L::kCentred>(y >> 8, e3, o3);
#pragma unroll
          for (int q = L::kPParts - 1; q >= 0; --q) {
            mma(sum[0], e0, o0, e1, o1, pt[r][b / F][q][0], pt[r][b / F][q][1]);
            mma(sum[1], e2, o2, e3, o3, pt[r][b / F][q][0], pt[r][b / F][q][1]);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[b][j][i] = fmaf(above, sum[j][i], o[b][j][i]);
      }
      load_v();
      next = place();
    }

    // join the warps
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int h = warp * kHeads + 2 * t + i;
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
        v.x = fmaf(o[b][0][i], L::kEven, low);
        v.y = fmaf(o[b][0][i + 2], L::kOdd, low);
        v.z = fmaf(o[b][1][i], L::kEven, low);
        v.w = fmaf(o[b][1][i + 2], L::kOdd, low);
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
        if (d == 0 && a.lse) a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (most + log2f(sum) - kShift) * kLn2;
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
      if (d == 0 && a.lse) a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (most + log2f(sum) - kShift) * kLn2;
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
  __shared__ float4 acc[kJoinThreads];
  __shared__ float2 stats[kJoinThreads / 16];
  const int tid = threadIdx.x, c0 = blockIdx.x;
  begin();
  if (c0 < a.batch && span_of<64>(a, c0).tiles == 0) {
    for (int qh = blockIdx.y; qh < a.q_heads; qh += gridDim.y) {
      for (int d = tid; d < a.head_dim; d += kJoinThreads)
        ((T*)a.out)[(long long)c0 * a.o_sb + (long long)qh * a.o_sh + d] = from_float<T>(0.f);
      if (tid == 0 && a.lse) a.lse[(long long)c0 * a.q_heads + qh] = -INFINITY;
    }
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
    for (int e = 0; e < 4; ++e) out[e] = from_float<T>(sum == 0.f ? 0.f : r[e] / sum);
    if (col == 0 && a.lse) a.lse[(long long)b * a.q_heads + qh] = sum == 0.f ? -INFINITY : (top + log2f(sum) - kShift) * kLn2;
  }
}

template <typename T_, int W, int G>
struct Kernel {
  using T = T_;
  using L = Layout<T, W, G>;
  static constexpr auto run = attend_kernel<T, W, G, false>;
  static constexpr auto run_cluster = attend_kernel<T, W, G, true>;
};

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

// Groups as wide as the head are one group, whatever their size.
template <typename T, class F>
void dispatch_typed(int width, int64_t group, F&& f) {
  if (width == 64) {
    group == 32 ? f(Kernel<T, 64, 32>()) : f(Kernel<T, 64, 64>());
  } else if (width == 96) {
    if (group == 32) f(Kernel<T, 96, 32>());
    else group == 64 ? f(Kernel<T, 96, 64>()) : f(Kernel<T, 96, 128>());
  } else if (width == 128) {
    if (group == 32) f(Kernel<T, 128, 32>());
    else group == 64 ? f(Kernel<T, 128, 64>()) : f(Kernel<T, 128, 128>());
  } else {
    if (group == 32) f(Kernel<T, 256, 32>());
    else group == 64 ? f(Kernel<T, 256, 64>()) : f(Kernel<T, 256, 128>());
  }
}

// Calls f(Kernel<...>()) for the call's type and sizes.
template <class F>
void dispatch(const pfk_cache4_attention_params& p, F&& f) {
  const int width = cache4_width(p.cache.head_dim);
  if (p.dtype == PFC_DTYPE_FLOAT16) dispatch_typed<__half>(width, p.cache.group, f);
  else if (p.dtype == PFC_DTYPE_BFLOAT16) dispatch_typed<__nv_bfloat16>(width, p.cache.group, f);
  else dispatch_typed<float>(width, p.cache.group, f);
}

void check(const pfk_cache4_attention_params& p) {
  const pfk_cache4& c = p.cache;
  check_cache4(c);
  check_decode_dtype(p.dtype);
  PFB_CHECK_ARG(p.batch >= 0 && p.q_heads >= c.heads && p.q_heads % c.heads == 0 && p.q_heads <= 65536,
                "4-bit attention: q_heads must be a multiple of the cache's heads, at most 65536");
  PFB_CHECK_ARG(p.batch <= INT32_MAX / p.q_heads / kMostRanks, "4-bit attention: too many query heads in a batch");
  PFB_CHECK_ARG(p.table_width >= 0 && p.table_width <= INT32_MAX && p.table_stride >= 0, "4-bit attention: bad block table size");
  PFB_CHECK_ARG(p.q_sb >= 0 && p.q_sh >= 0 && p.o_sb >= 0 && p.o_sh >= 0, "4-bit attention: negative stride");
  PFB_CHECK_ARG(p.window >= 0, "4-bit attention: negative window");
  PFB_CHECK_ARG(std::isfinite(p.scale), "4-bit attention: scale is not finite");
}

constexpr int64_t kClusterTiles = 64;  // of 128 keys: the longest sequences that clusters take

struct Plan {
  int ctas, heads;
  int ranks;  // CTAs of a unit's cluster; 0: runs of the list of all tiles
  int64_t stats_at, parts_at, bytes;
};

Plan plan_of(const pfk_cache4_attention_params& p) {
  Plan w;
  const int64_t group = p.q_heads / p.cache.heads;
  w.heads = (int)std::min<int64_t>(group, kHeads);
  dispatch(p, [&](auto k) { w.ctas = wave<decltype(k)>(); });
  int64_t seen = std::min<int64_t>(p.table_width * p.cache.page_size, INT32_MAX);
  if (p.window) seen = std::min<int64_t>(seen, std::min<int64_t>(p.window, INT32_MAX) + 128);
  const int64_t units = p.batch * p.cache.heads * ceil_div(group, kHeads), tiles = ceil_div(seen, 128);
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

}  // namespace

size_t cache4_attention_workspace(const pfk_cache4_attention_params& p) {
  check(p);
  if (p.batch == 0) return 0;
  return (size_t)plan_of(p).bytes;
}

void launch_cache4_attention(const pfk_cache4_attention_params& p, cudaStream_t stream) {
  check(p);
  if (p.batch == 0) return;
  PFB_CHECK_ARG(p.q && p.out && p.seq_lens && (p.block_table || p.table_width == 0), "4-bit attention: null pointer");
  // a CTA reads its unit's queries before any of the unit's outputs are
  // written, so the output may take the queries' place, row for row
  PFB_CHECK_ARG(p.out != p.q || ((p.batch == 1 || p.q_sb == p.o_sb) && (p.q_heads == 1 || p.q_sh == p.o_sh)),
                "4-bit attention: out shares q's memory with other strides");
  const pfk_cache4& c = p.cache;
  const Plan w = plan_of(p);
  PFB_CHECK_ARG(w.bytes == 0 || (p.workspace && p.workspace_bytes >= (size_t)w.bytes && (uintptr_t)p.workspace % 16 == 0),
                "4-bit attention: workspace missing, too small or not 16-byte aligned");
  Args a = {};
  a.k = (const char*)c.k;
  a.v = (const char*)c.v;
  a.k_scales = (const char*)c.k_scales;
  a.v_scales = (const char*)c.v_scales;
  a.num_pages = (unsigned)c.num_pages;
  a.page_records = (unsigned)(c.heads * c.page_size);
  a.by_page = FastDiv((unsigned)c.page_size);
  a.err = c.err;
  a.batch = (int)p.batch;
  a.q_heads = (int)p.q_heads;
  a.kv_heads = (int)c.heads;
  a.group = (int)(p.q_heads / c.heads);
  a.chunks = (int)ceil_div(a.group, kHeads);
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
  a.most = std::min<int64_t>(p.table_width * c.page_size, INT32_MAX - 128);
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
