// experts.cu — a mixture-of-experts layer for a few tokens.
//
//   logits = R x, the `top` largest of them, w = their softmax
//   y = sum_j w_j D_j (act(G_j x) * (U_j x))
//
// The weights of the chosen experts are the work: 3 * width * inner values
// each, read once for all the tokens that chose the expert, and with a few
// tokens memory is the bound.  Kernels, each launched as a programmatic
// dependent of the one before:
//
// 1. route: a cluster of 8 CTAs for up to 8 tokens, or for 4 of more: each CTA an eighth of the
//    experts' logits, in 64 bits, since which expert a token takes is a
//    decision that no rounding should make (mma.sync in 64 bits takes 500
//    cycles an instruction on this device); the first CTA gathers them through
//    distributed shared memory and picks.  It copies x, aligned and padded,
//    for the next kernel, and lists the (token, choice) pairs by expert.  With
//    more than 8 tokens a kernel of one CTA lists them.
// 2. up: a CTA of 4 warps takes 8 gate rows and their 8 up rows of an expert,
//    which share the 16 rows of a matrix instruction, so that a lane ends with
//    a gate and its up value.  The warps share the summed axis, 64 bytes of a
//    row at a time (256 consecutive bytes a CTA).  What leaves is w act(g) u
//    in two 16-bit parts (one fp32 value): a single one would round as
//    coarsely as the output does.  fp16 parts reach from 2^-25 to 65504: 8
//    values (a unit's of a pair) have a power of two of their own (Scaled).
// 3. down: a cluster for 16 rows of the output.  All (expert, 64 bytes) pieces
//    of those rows form one list, of which each warp of the cluster takes an
//    equal run; at an expert's end it adds what it has to its own table of
//    tokens in shared memory.  The tables are added in the order of warps and
//    ranks: no atomics, the same bits each time.
//
// The rows come through a ring of asynchronous copies in shared memory for
// each warp, whose lanes read what they copied, as operand registers
// (streamed.cuh): the copies run ahead over the borders of rows and experts.
//
// Measured (device time, replayed from a graph; the bytes at 6.56 TB/s in
// brackets): 64 tokens, 8 of 128 experts, 2048 x 768, fp16, 1.19 GB: 231 us
// (181), of which route and list 22, up 132 and down 84; one token, 6 of 64
// experts, 2048 x 1408, bf16, 104 MB: 32.6 us (15.9), route 8.7, up 15.6 and
// down 10.5, of which 8 stay when its weights are in L2: what begins and ends
// a kernel; five tokens, 2 of 8 experts, 768 x 2048, fp32: 40 us (17.6).
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
#include "act.cuh"
#include "decode.cuh"
#include "kernels.hpp"
#include "streamed.cuh"

namespace pfb {
namespace {

namespace cg = cooperative_groups;

constexpr int kBlockTokens = 128;  // tokens of one pass over the weights
constexpr int kMostExperts = 1024;
constexpr int kMostTop = 32;
constexpr int kMostRanks = 8;  // CTAs of a cluster
constexpr int kRouteRanks = kMostRanks;
constexpr int kRouteThreads = 256;
constexpr int kRouteBlock = 2048;  // values of x that it holds of a token at a time
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct Args {
  int tokens, width, inner, experts, top;
  int renormalize, act;
  const void* x;
  long long x_st;
  const float* router;
  long long router_st;
  const char* gate_up;
  long long up_row, up_expert;  // bytes
  const char* down;
  long long down_row, down_expert;
  void* y;
  long long y_st;
  int* chosen;     // [tokens][top]
  float* weights;  // [tokens][top]
  // workspace
  char* xs;  // x, [tokens][x_row bytes], zeros behind width
  long long x_row;
  char* h;  // [parts][tokens * top][h_row bytes], zeros behind inner
  long long h_row, h_part;
  // fp16: exponents of the powers of two on 8 values of h each, [tokens * top][e_row]
  signed char* e;
  long long e_row;
  // parts of experts' pairs: how many, then of each: expert, first of its pairs, their number (at most 8 NT),
  // whether a power of two of theirs is not 2^0
  int4* parts;
  int* pairs;  // [tokens * top] by expert
  int most_parts;
};

// fp16 intermediate values are held times 2^10, and 8 of them over a power of two
// of their own, 2^e: 2^0 where the largest is then from 2^-8 to 65504, or that
// with e a multiple of 8 which puts it between 2^7 and 2^15, so that a value
// loses 2^-22, or 2^-17 of the largest of the 8.  Zeros have the least exponent.
// Products add four of them up (64 bytes of a row): with powers that differ,
// which multiples of 8 seldom do, the values are multiplied by what they are
// below the largest.  The down products look at the powers of a part only where
// one is not 2^0, as seldom happens to values from 2^-18 to 2^6 (64 tokens, 8 of
// 128 experts, 2048 x 768: 231 us; with a few values of 10^4 in all parts 253, with
// all values near 10^-9 272).
template <typename T>
struct Scaled {
  static constexpr bool kIs = std::is_same<T, __half>::value;
  static constexpr float kTimes = kIs ? 1024.f : 1.f;
};
constexpr int kZeros = -128;
__device__ __forceinline__ int exponent_for(float largest) {
  if (largest == 0.f) return kZeros;
  return largest >= 0x1p-8f && largest <= 65504.f ? 0 : max(((int)(__float_as_uint(largest) >> 23) - 127 - 7) & ~7, -120);
}

// Lets the next kernel come up while this one works: the kernels in front of
// another leave room for its CTAs, or their own are all there already.  The
// next one's wait in begin() is the same.
__device__ __forceinline__ void let_next_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------
// route
// ---------------------------------------------------------------------------

// Lists the pairs by expert, those of an expert in their order, in parts of at
// most `most`: a CTA of kRouteThreads; shared: list_ints() ints.  (An order that
// depended on timing would put a pair in one part or another, whose rows'
// pieces are shared out among warps in another way.)  A warp counts a run of
// the pairs, 32 at a time.
constexpr int kListWarps = kRouteThreads / 32;
constexpr size_t list_ints(int64_t experts, int64_t pairs) { return (size_t)(kListWarps * experts + 2 * pairs); }

__device__ void list_pairs(const Args& a, const int* chosen, int* shared, int most) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pairs = a.tokens * a.top;
  int *counts = shared, *place = shared + kListWarps * a.experts, *expert = place + pairs;  // counts: [warp][expert]
  const int run = (pairs + 32 * kListWarps - 1) / (32 * kListWarps) * 32;
  for (int i = tid; i < kListWarps * a.experts; i += kRouteThreads) counts[i] = 0;
  for (int p = tid; p < pairs; p += kRouteThreads) expert[p] = chosen[p];
  __syncthreads();
  int* mine = counts + warp * a.experts;
  for (int base = warp * run; base < min(pairs, (warp + 1) * run); base += 32) {
    const int p = base + lane, e = p < pairs ? expert[p] : -1;
    const unsigned same = __match_any_sync(~0u, e), before = same & ((1u << lane) - 1);
    if (e >= 0) place[p] = mine[e] + __popc(before);
    __syncwarp();
    if (e >= 0 && !before) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = tid; e < a.experts; e += kRouteThreads) {  // how many an expert has in the runs up to and with each warp's
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kListWarps; ++w) sum += counts[w * a.experts + e], counts[w * a.experts + e] = sum;
  }
  __syncthreads();
  int* all = counts + (kListWarps - 1) * a.experts;
  if (warp == 0) {
    int start = 0, parts = 0;
    for (int base = 0; base < a.experts; base += 32) {
      const int e = base + lane, n = e < a.experts ? all[e] : 0, own = (n + most - 1) / most;
      int sum = n, before = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int s = __shfl_up_sync(~0u, sum, o), b = __shfl_up_sync(~0u, before, o);
        if (lane >= o) {
          sum += s;
          before += b;
        }
      }
      const int first = start + sum - n;
      for (int k = 0; k < own; ++k) a.parts[1 + parts + before - own + k] = make_int4(e, first + k * most, min(most, n - k * most), 0);
      if (e < a.experts) all[e] = first;
      start += __shfl_sync(~0u, sum, 31);
      parts += __shfl_sync(~0u, before, 31);
    }
    if (lane == 0) a.parts[0] = make_int4(parts, 0, 0, 0);
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kRouteThreads) {
    const int e = expert[p], w = p / run;
    a.pairs[all[e] + (w ? counts[(w - 1) * a.experts + e] : 0) + place[p]] = p;
  }
}

// Parts of the logits of EP experts and TB tokens, over `len` values (a
// multiple of 4) of the router's rows and of x in shared memory: a warp, whose
// lanes share the summed axis; sum[e][n] is whole in every lane.
template <int TB, int EP>
__device__ __forceinline__ void logits_of(double (&sum)[EP][TB], const float* const (&rows)[EP], const float* xs, int len) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < EP; ++e)
#pragma unroll
    for (int n = 0; n < TB; ++n) sum[e][n] = 0.;
  constexpr int UNROLL = TB == 1 ? 16 : 4;  // loads on their way
  for (int d0 = 4 * lane; d0 < len; d0 += 128 * UNROLL) {
    float4 r[UNROLL][EP];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int e = 0; e < EP; ++e)
        r[u][e] = d0 + 128 * u < len ? __ldg(reinterpret_cast<const float4*>(rows[e] + d0 + 128 * u)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (d0 + 128 * u >= len) break;
      double w[EP][4];
#pragma unroll
      for (int e = 0; e < EP; ++e) {
        w[e][0] = r[u][e].x;
        w[e][1] = r[u][e].y;
        w[e][2] = r[u][e].z;
        w[e][3] = r[u][e].w;
      }
#pragma unroll
      for (int n = 0; n < TB; ++n) {
        const float4 v = *reinterpret_cast<const float4*>(xs + n * kRouteBlock + d0 + 128 * u);
        const double y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < EP; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[e][n] = fma(w[e][i], y[i], sum[e][n]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < EP; ++e)
#pragma unroll
    for (int n = 0; n < TB; ++n)
#pragma unroll
      for (int o = 16; o; o >>= 1) sum[e][n] += __shfl_xor_sync(~0u, sum[e][n], o);
}

// Numbers in the order of their values; NaN as the lowest.
__device__ __forceinline__ unsigned long long ordered(double v) {
  if (!(v >= -1.7976931348623157e308)) v = -INFINITY;
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(unsigned long long o) {
  return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}

// TB tokens a cluster
template <typename T, int TB>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(Args a) {
  extern __shared__ __align__(16) double shared[];
  __shared__ int choice[TB * kMostTop];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = (int)(blockIdx.x / kRouteRanks) * TB, mine = min(TB, a.tokens - first);
  const int share = (a.experts + kRouteRanks - 1) / kRouteRanks, e0 = rank * share, e1 = min(a.experts, e0 + share);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(shared);  // rank 0: [tokens][experts]
  double* logits = shared + TB * a.experts;                                  // [tokens][share]
  float* xs = reinterpret_cast<float*>(logits + TB * share + (TB * (a.experts + share) & 1));  // [tokens][kRouteBlock]
  if (gridDim.x == kRouteRanks) let_next_come();  // the others' SMs are free
  // rank 0 has started, and its memory can be written
  cluster.sync();
  begin();

  const T* x = (const T*)a.x + first * a.x_st;
  const int padded = (int)(a.x_row / (int)sizeof(T));
  constexpr int kWarpsHere = kRouteThreads / 32;
  auto row = [&](int e, int base) { return a.router + (long long)min(e, a.experts - 1) * a.router_st + base; };
  for (int base = 0; base < padded; base += kRouteBlock) {
    if (base) __syncthreads();
    // x in fp32 for this kernel, and as it is, a part by each rank, for the next
#pragma unroll
    for (int n = 0; n < TB; ++n) {
      T v[kRouteBlock / kRouteThreads];
#pragma unroll
      for (int i = 0; i < kRouteBlock / kRouteThreads; ++i) {
        const int d = base + i * kRouteThreads + tid;
        v[i] = n < mine && d < a.width ? x[n * a.x_st + d] : from_float<T>(0.f);
      }
#pragma unroll
      for (int i = 0; i < kRouteBlock / kRouteThreads; ++i) {
        const int d = base + i * kRouteThreads + tid;
        xs[n * kRouteBlock + d - base] = to_float<T>(v[i]);
        if (i % kRouteRanks == rank && n < mine && d < padded) reinterpret_cast<T*>(a.xs + (first + n) * a.x_row)[d] = v[i];
      }
    }
    __syncthreads();
    const int len = (int)min((long long)kRouteBlock, a.router_st - base);
    auto put = [&](int e, int n, double s) {
      double* to = logits + n * share + e - e0;
      *to = base ? *to + s : s;
    };
    if (TB > 1 && share > kWarpsHere) {  // x is read and converted once for two experts
      for (int e = e0 + 2 * warp; e < e1; e += 2 * kWarpsHere) {
        double sum[2][TB];
        const float* rows[2] = {row(e, base), row(e + 1, base)};
        logits_of<TB, 2>(sum, rows, xs, len);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int n = 0; n < TB; ++n)
            if (lane == 0 && e + k < e1) put(e + k, n, sum[k][n]);
      }
    } else {
      for (int e = e0 + warp; e < e1; e += kWarpsHere) {
        double sum[1][TB];
        const float* rows[1] = {row(e, base)};
        logits_of<TB, 1>(sum, rows, xs, len);
#pragma unroll
        for (int n = 0; n < TB; ++n)
          if (lane == 0) put(e, n, sum[0][n]);
      }
    }
  }
  __syncthreads();
  unsigned long long* to = cluster.map_shared_rank(keys, 0);
  for (int i = tid; i < mine * (e1 - e0); i += kRouteThreads) {
    const int n = i / (e1 - e0), e = i - n * (e1 - e0);
    to[n * a.experts + e0 + e] = ordered(logits[n * share + e]);
  }
  cluster.sync();
  if (rank != 0) return;

  if (warp < mine) {  // a warp picks for a token
    const unsigned long long* l = keys + warp * a.experts;
    unsigned taken = 0;  // of the lane's experts lane + 32 i
    unsigned long long best = 0;
    int at = INT_MAX;  // the lane's best that is not taken
    auto look = [&]() {
      best = 0;
      at = INT_MAX;
      for (int e = lane, i = 0; e < a.experts; e += 32, ++i)
        if (!(taken >> i & 1) && (at == INT_MAX || l[e] > best)) {
          best = l[e];
          at = e;
        }
    };
    look();
    double top = 0.;
    float total = 0.f, own_part = 0.f;
    int kept = 0;
    for (int j = 0; j < a.top; ++j) {
      const unsigned high = __reduce_max_sync(~0u, (unsigned)(best >> 32));
      const unsigned low = __reduce_max_sync(~0u, (unsigned)(best >> 32) == high ? (unsigned)best : 0u);
      const unsigned long long won = (unsigned long long)high << 32 | low;
      const int e = (int)__reduce_min_sync(~0u, best == won ? (unsigned)at : (unsigned)INT_MAX);
      const double v = value_of(won);
      if (j == 0) top = v;
      const float w = expf((float)(v - top));
      total += w;
      if (lane == j) {
        own_part = w;
        kept = e;
      }
      if (at == e) {
        taken |= 1u << (e >> 5);
        look();
      }
    }
    if (!a.renormalize) {
      total = 0.f;
      for (int e = lane; e < a.experts; e += 32) total += expf((float)(value_of(l[e]) - top));
#pragma unroll
      for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    }
    if (lane < a.top) {
      a.chosen[(long long)(first + warp) * a.top + lane] = kept;
      a.weights[(long long)(first + warp) * a.top + lane] = own_part / total;
      choice[warp * a.top + lane] = kept;
    }
  }
  if (a.tokens <= TB) {
    __syncthreads();
    list_pairs(a, choice, reinterpret_cast<int*>(shared), 8);
  }
}

__global__ void __launch_bounds__(kRouteThreads) list_kernel(Args a) {
  extern __shared__ double shared[];
  let_next_come();
  begin();
  list_pairs(a, a.chosen, reinterpret_cast<int*>(shared), 16);
}

// ---------------------------------------------------------------------------
// up and down
// ---------------------------------------------------------------------------

template <typename T>
struct Parts {
  static constexpr int kH = sizeof(T) == 2 ? 2 : 1;  // of an intermediate value
};

// A warp's ring: stages of a piece of 16 rows and of the vectors, NB blocks of 8.
template <int NB, int DEPTH>
struct Ring {
  static constexpr int kStage = (2 + NB) * 512, kBytes = kStage * DEPTH;
  uint32_t base;  // of the lane
  __device__ __forceinline__ Ring(char* warp_memory) : base((uint32_t)__cvta_generic_to_shared(warp_memory) + (threadIdx.x & 31) * 16) {}
  static __device__ __forceinline__ uint4 read(uint32_t at) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
    return r;
  }
};

// Eight fp16 numbers times two, the same.
__device__ __forceinline__ uint4& times_half(uint4& v, unsigned by) {
  const __half2 f = *reinterpret_cast<const __half2*>(&by);
  unsigned* w = &v.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(w + i), f);
    w[i] = *reinterpret_cast<const unsigned*>(&x);
  }
  return v;
}

// What the vectors of a piece add up to with its rows, added to acc in fp32,
// rounded to nearest: the tensor cores truncate what they add.
// SCALED: exponents: of the four powers of two of each of the lane's vectors.
template <typename T, int NT, int PARTS, bool SCALED, class R>
__device__ __forceinline__ void take_piece(float (&acc)[NT][4], uint32_t at, bool second, const int (&exponents)[NT]) {
  const uint4 a0 = R::read(at), a1 = R::read(at + 512);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n && !second) continue;  // the same in all lanes
    float sum[1][4] = {{0.f, 0.f, 0.f, 0.f}};
    float times[2] = {1.f, 1.f};  // of the vectors 2t and 2t + 1
    uint4 b[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) b[p] = R::read(at + 1024 + (p * NT + n) * 512);
    if constexpr (SCALED) {
      const int e = exponents[n];
      if (__any_sync(~0u, e != 0)) {
        const int t = threadIdx.x & 3, own = (signed char)(e >> (8 * t));
        const int most = max(max((int)(signed char)e, (int)(signed char)(e >> 8)), max((int)(signed char)(e >> 16), e >> 24));
        const int down = own - most;
        if (__any_sync(~0u, down != 0 && own != kZeros)) {
          // 2^down as a product of two fp16 numbers; below 2^-38, 0
          const int rest = min(max(down, -40) + 14, 0);
          const unsigned first = (unsigned)(15 + max(down, -14)) << 10;
          const unsigned second = rest >= -14 ? (unsigned)(15 + rest) << 10 : rest >= -24 ? 1u << (24 + rest) : 0u;
#pragma unroll
          for (int p = 0; p < PARTS; ++p) times_half(times_half(b[p], first << 16 | first), second << 16 | second);
        }
        const float mine = __uint_as_float((unsigned)(127 + max(most, -126)) << 23);
        times[0] = __shfl_sync(~0u, mine, 8 * t);
        times[1] = __shfl_sync(~0u, mine, 8 * t + 4);
      }
    }
#pragma unroll
    for (int p = PARTS - 1; p >= 0; --p) {
      const uint4 one[1] = {b[p]};
      chunk_product<T, 1>(sum, a0, a1, one);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[n][r] = SCALED ? fmaf(sum[0][r], times[r & 1], acc[n][r]) : acc[n][r] + sum[0][r];
  }
}

template <typename T, int NT>
struct Up {
  static constexpr int kDepth = NT == 1 ? 8 : 6;
  using R = Ring<NT, kDepth>;
  static constexpr int kResident = 4;  // CTAs an SM
  static size_t smem(int parts, int pairs) { return (size_t)kWarps * R::kBytes + (size_t)parts * 16 + (size_t)((pairs + 3) / 4) * 16; }
};

// Units are 8 rows of a part of an expert's pairs; CTAs take them in turn, part
// by part.  An expert of more than 16 pairs has several, each of which reads all
// its rows again.  (The parts' units of the same rows next to each other, so that
// they come from L2: 128 tokens, 2 of 8 experts, 4096 x 14336, fp16: 876 us so,
// 835 then; the down products by stretches of 16 pieces 734 and 857, and smaller
// layers 2 to 5 % slower.)
template <typename T, int NT>
__global__ void __launch_bounds__(kThreads, (Up<T, NT>::kResident)) up_kernel(Args a) {
  using U = Up<T, NT>;
  extern __shared__ __align__(16) char smem[];
  __shared__ float4 red[2][kWarps][NT][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  int4* parts = reinterpret_cast<int4*>(smem + kWarps * U::R::kBytes);
  int* pairs = reinterpret_cast<int*>(parts + a.most_parts);
  typename U::R ring(smem + warp * U::R::kBytes);
  begin();
  for (int i = tid; i < a.most_parts; i += kThreads) parts[i] = a.parts[1 + i];  // those behind the last are not looked at
  for (int i = tid; i < a.tokens * a.top; i += kThreads) pairs[i] = a.pairs[i];
  const int blocks = (a.inner + 7) / 8, units = a.parts[0].x * blocks;
  const int bytes = (int)min(a.x_row, a.up_row), pieces = (bytes + 63) / 64;
  __syncthreads();
  if ((int)blockIdx.x >= units) return;

  // What the copies stand at.  Rows and vectors that are not there are read
  // nowhere: their size is 0, their place some other's.
  struct {
    int unit, at;
    const char *gate, *up, *vec[NT];
    int rows, vecs[NT];  // sizes
    bool second;
  } ahead = {};
  auto aim = [&]() {  // at the unit's rows
    const int i = ahead.unit / blocks, f = (ahead.unit - i * blocks) * 8 + g;
    const int4 p = parts[i];
    ahead.at = warp * 64 + t * 16;
    ahead.rows = f < a.inner ? 16 : 0;
    ahead.gate = a.gate_up + p.x * a.up_expert + min(f, a.inner - 1) * a.up_row + ahead.at;
    ahead.up = ahead.gate + a.inner * a.up_row;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int slot = n * 8 + g;
      ahead.vecs[n] = slot < p.z ? 16 : 0;
      ahead.vec[n] = a.xs + (long long)(pairs[p.y + min(slot, p.z - 1)] / a.top) * a.x_row + ahead.at;
    }
    ahead.second = p.z > 8;
  };
  auto copy = [&](uint32_t to) {
    if (ahead.unit < units) {
      const bool in = ahead.at < bytes;
      copy_async(to, ahead.gate, in ? ahead.rows : 0);
      copy_async(to + 512, ahead.up, in ? ahead.rows : 0);
      copy_async(to + 1024, ahead.vec[0], in ? ahead.vecs[0] : 0);
      if (NT > 1 && ahead.second) {
#pragma unroll
        for (int n = 1; n < NT; ++n) copy_async(to + 1024 + n * 512, ahead.vec[n], in ? ahead.vecs[n] : 0);
      }
      constexpr int kStep = kWarps * 64;
      ahead.at += kStep;
      ahead.gate += kStep;
      ahead.up += kStep;
#pragma unroll
      for (int n = 0; n < NT; ++n) ahead.vec[n] += kStep;
      if (ahead.at - t * 16 >= bytes) {
        ahead.unit += gridDim.x;
        if (ahead.unit < units) aim();
      }
    }
    copy_commit();
  };
  ahead.unit = warp < pieces ? (int)blockIdx.x : units;  // a warp without pieces has nothing to copy
  if (ahead.unit < units) aim();
  uint32_t at = ring.base;
#pragma unroll
  for (int s = 0; s < U::kDepth; ++s) copy(at + s * U::R::kStage);

  int turn = 0;
  int told = -1;
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x, turn ^= 1) {
    const int i = unit / blocks, f = (unit - i * blocks) * 8 + g;
    const int4 p = parts[i];
    // The warp finishes vectors 2t + k of block n, a value of the unit's each lane: all of them for 16 vectors, two for 8.
    const int n = warp >> 1, k = warp & 1;
    int pair = -1;
    float weight = 0.f;
    if (warp < 2 * NT) {
      const int slot = n * 8 + 2 * t + k;
      if (slot < p.z) {
        pair = pairs[p.y + slot];
        weight = a.weights[pair] * Scaled<T>::kTimes;
      }
    }
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    for (int c = warp; c < pieces; c += kWarps) {
      copy_wait<U::kDepth - 1>();
      take_piece<T, NT, 1, false, typename U::R>(acc, at, p.z > 8, {});
      copy(at);
      at = at == ring.base + (U::kDepth - 1) * U::R::kStage ? ring.base : at + U::R::kStage;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) red[turn][warp][n][lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    __syncthreads();
    static_assert(2 * NT <= kWarps, "a warp finishes half of a block of vectors");
    if (warp < 2 * NT) {
      const float* from = reinterpret_cast<const float*>(&red[turn][0][n][lane]) + k;
      float gv = 0.f, uv = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        gv += from[w * NT * 128];
        uv += from[w * NT * 128 + 2];
      }
      const float act = a.act ? act_apply<2>(gv) : act_apply<5>(gv);
      // rows behind the last are zeros (their sums are)
      float v = pair >= 0 && f < a.inner ? act * uv * weight : 0.f;
      if constexpr (Scaled<T>::kIs) {
        float largest = fabsf(v);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(~0u, largest, o));
        const int e = exponent_for(largest);
        if (e != 0 && e != kZeros) {
          v *= __uint_as_float((unsigned)(127 - e) << 23);
          if (g == 0 && told != i) {
            a.parts[1 + i].w = 1;
            told = i;
          }
        }
        if (g == 0 && pair >= 0) {
          signed char* to = a.e + pair * a.e_row + (unit - i * blocks);
          *to = (signed char)e;
          if (unit - i * blocks == blocks - 1)  // up to whole pieces
            for (int c = blocks; c < a.e_row; ++c) *++to = kZeros;
        }
      }
      if (pair >= 0) {
        T* to = reinterpret_cast<T*>(a.h + pair * a.h_row) + f;
        if constexpr (sizeof(T) == 4) {
          *to = v;
        } else {
          T hi, lo;
          two_parts(v, hi, lo);
          *to = hi;
          *reinterpret_cast<T*>(reinterpret_cast<char*>(to) + a.h_part) = lo;
        }
      }
    }
  }
}

// WARPS of a CTA: with few blocks of rows, all of a block's in one CTA.
template <typename T, int NT, int WARPS>
struct Down {
  static constexpr int kDepth = NT == 1 ? 6 : 4;
  using R = Ring<NT * Parts<T>::kH, kDepth>;
  static constexpr int kResident = WARPS > 4 ? (NT == 1 ? 16 : 8) / WARPS : NT == 1 ? 4 : 3;
  static constexpr size_t smem(int parts, int pairs, int tokens) {
    return (size_t)WARPS * (R::kBytes + tokens * 64) + (size_t)parts * 16 + (size_t)((pairs + 3) / 4) * 16;
  }
};

template <typename T, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (Down<T, NT, WARPS>::kResident)) down_kernel(Args a) {
  using D = Down<T, NT, WARPS>;
  constexpr int PARTS = Parts<T>::kH;
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / ranks) * 16, cells = a.tokens * 16;
  float* tables = reinterpret_cast<float*>(smem + WARPS * D::R::kBytes);  // [warps][tokens][16]
  int4* parts = reinterpret_cast<int4*>(tables + WARPS * cells);
  int* pairs = reinterpret_cast<int*>(parts + a.most_parts);
  typename D::R ring(smem + warp * D::R::kBytes);
  for (int i = tid; i < WARPS * cells; i += (WARPS * 32)) tables[i] = 0.f;
  begin();
  for (int i = tid; i < a.most_parts; i += (WARPS * 32)) parts[i] = a.parts[1 + i];
  for (int i = tid; i < a.tokens * a.top; i += (WARPS * 32)) pairs[i] = a.pairs[i];
  const int bytes = (int)min(a.h_row, a.down_row), pieces = (bytes + 63) / 64;
  const int total = a.parts[0].x * pieces, q = rank * WARPS + warp, of = ranks * WARPS;
  const int p0 = (int)((long long)total * q / of), p1 = (int)((long long)total * (q + 1) / of);
  __syncthreads();

  struct {
    int left, part, at;
    const char *row0, *row1, *vec[NT];
    int rows0, rows1, vecs[NT];  // sizes, as above
    bool second;
  } ahead = {};
  auto aim = [&](int piece) {
    const int4 p = parts[ahead.part];
    ahead.at = piece * 64 + t * 16;
    ahead.rows0 = row + g < a.width ? 16 : 0;
    ahead.rows1 = row + g + 8 < a.width ? 16 : 0;
    const char* base = a.down + p.x * a.down_expert + ahead.at;
    ahead.row0 = base + min(row + g, a.width - 1) * a.down_row;
    ahead.row1 = base + min(row + g + 8, a.width - 1) * a.down_row;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int slot = n * 8 + g;
      ahead.vecs[n] = slot < p.z ? 16 : 0;
      ahead.vec[n] = a.h + (long long)pairs[p.y + min(slot, p.z - 1)] * a.h_row + ahead.at;
    }
    ahead.second = p.z > 8;
  };
  auto copy = [&](uint32_t to) {
    if (ahead.left) {
      const bool in = ahead.at < bytes;
      copy_async(to, ahead.row0, in ? ahead.rows0 : 0);
      copy_async(to + 512, ahead.row1, in ? ahead.rows1 : 0);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (n == 0 || ahead.second) {
#pragma unroll
          for (int p = 0; p < PARTS; ++p) copy_async(to + 1024 + (p * NT + n) * 512, ahead.vec[n] + p * a.h_part, in ? ahead.vecs[n] : 0);
        }
      ahead.at += 64;
      ahead.row0 += 64;
      ahead.row1 += 64;
#pragma unroll
      for (int n = 0; n < NT; ++n) ahead.vec[n] += 64;
      --ahead.left;
      if (ahead.at - t * 16 >= bytes) {
        ++ahead.part;
        if (ahead.left) aim(0);
      }
    }
    copy_commit();
  };
  ahead.left = p1 - p0;
  if (p0 < p1) {
    ahead.part = p0 / pieces;
    aim(p0 - ahead.part * pieces);
  }
  float* table = tables + warp * cells;
  uint32_t at = ring.base;
#pragma unroll
  for (int s = 0; s < D::kDepth; ++s) copy(at + s * D::R::kStage);
  for (int p = p0; p < p1;) {
    const int i = p / pieces, end = min(p1, (i + 1) * pieces);
    const int4 e = parts[i];
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    auto run = [&](auto scaled) {
      constexpr bool SCALED = decltype(scaled)::value;
      int exponents[NT] = {};
      const signed char* from[NT];
      if constexpr (SCALED) {
#pragma unroll
        for (int n = 0; n < NT; ++n) from[n] = a.e + (long long)pairs[e.y + min(n * 8 + g, e.z - 1)] * a.e_row + (p - i * pieces) * 4;
      }
      for (; p < end; ++p) {
        if constexpr (SCALED) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            exponents[n] = *reinterpret_cast<const int*>(from[n]);
            from[n] += 4;
          }
        }
        copy_wait<D::kDepth - 1>();
        take_piece<T, NT, PARTS, SCALED, typename D::R>(acc, at, e.z > 8, exponents);
        copy(at);
        at = at == ring.base + (D::kDepth - 1) * D::R::kStage ? ring.base : at + D::R::kStage;
      }
    };
    if constexpr (Scaled<T>::kIs) e.w ? run(std::true_type()) : run(std::false_type());
    else run(std::false_type());
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int slot = n * 8 + 2 * t + k;
        if (slot < e.z) {
          float* to = table + pairs[e.y + slot] / a.top * 16;
          to[g] += acc[n][k];
          to[g + 8] += acc[n][k + 2];
        }
      }
    __syncwarp();
  }
  __syncthreads();
  for (int i = tid; i < cells; i += (WARPS * 32)) {
    float s = tables[i];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) s += tables[w * cells + i];
    tables[i] = s;
  }
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  for (int i = rank * (WARPS * 32) + tid; i < cells; i += (WARPS * 32) * ranks) {
    float s = 0.f;
    for (int r = 0; r < ranks; ++r) s += cluster.map_shared_rank(tables, r)[i];
    const int n = i >> 4, d = row + (i & 15);
    if (d < a.width) ((T*)a.y)[n * a.y_st + d] = from_float<T>(s * (1.f / Scaled<T>::kTimes));
  }
  if (ranks > 1) cluster.sync();  // the others' reads of this CTA's table are over
}

// ---------------------------------------------------------------------------

int64_t size_of(int dtype) { return dtype == PFC_DTYPE_FLOAT32 ? 4 : 2; }

void check(const pfk_experts_params& p) {
  check_decode_dtype(p.dtype);
  const int64_t es = size_of(p.dtype);
  PFB_CHECK_ARG(p.tokens >= 0 && p.tokens <= INT32_MAX / kMostTop, "experts: bad number of tokens");
  PFB_CHECK_ARG(p.width >= 1 && p.width <= 65536 && p.inner >= 1 && p.inner <= 65536, "experts: width and inner must be 1 to 65536");
  PFB_CHECK_ARG(p.experts >= 1 && p.experts <= kMostExperts, "experts: their number must be 1 to 1024");
  PFB_CHECK_ARG(p.top >= 1 && p.top <= kMostTop && p.top <= p.experts, "experts: top must be 1 to 32 and at most their number");
  PFB_CHECK_ARG(p.activation == 0 || p.activation == 1, "experts: activation must be 0 (SiLU) or 1 (GELU)");
  PFB_CHECK_ARG(p.renormalize == 0 || p.renormalize == 1, "experts: renormalize must be 0 or 1");
  PFB_CHECK_ARG(p.x_st >= 0 && p.y_st >= 0, "experts: negative stride");
  PFB_CHECK_ARG(p.router_st >= p.width && p.router_st % 4 == 0 && p.gate_up_st >= p.width && p.gate_up_st * es % 16 == 0 &&
                    p.down_st >= p.inner && p.down_st * es % 16 == 0,
                "experts: rows of the weights must be padded to multiples of 16 bytes");
}

struct Plan {
  int64_t block, x_row, h_row, h_part, e_row;  // of a pass
  int64_t most_parts, h_at, e_at, parts_at, pairs_at, chosen_at, weights_at, bytes;
};

// At most so many parts of experts' pairs.
int64_t parts_of(const pfk_experts_params& p, int64_t tokens) {
  const int64_t pairs = tokens * p.top;
  return std::min(pairs, p.experts) + (tokens > 8 ? pairs / 16 : 0);
}

Plan plan_of(const pfk_experts_params& p) {
  Plan w;
  const int64_t es = size_of(p.dtype);
  w.block = std::min<int64_t>(p.tokens, kBlockTokens);
  const int64_t pairs = w.block * p.top;
  w.most_parts = parts_of(p, w.block);
  w.x_row = round_up(p.width * es, 16);
  w.h_row = round_up(round_up(p.inner, 8) * es, 16);
  w.h_part = pairs * w.h_row;
  w.h_at = round_up(w.block * w.x_row, 128);
  w.e_row = p.dtype == PFC_DTYPE_FLOAT16 ? round_up(ceil_div(p.inner, 8), 4) : 0;
  w.e_at = round_up(w.h_at + w.h_part * (es == 2 ? 2 : 1), 128);
  w.parts_at = round_up(w.e_at + pairs * w.e_row, 128);
  w.pairs_at = round_up(w.parts_at + (w.most_parts + 1) * (int64_t)sizeof(int4), 128);
  w.chosen_at = round_up(w.pairs_at + pairs * 4, 128);
  w.weights_at = round_up(w.chosen_at + pairs * 4, 128);
  w.bytes = w.weights_at + pairs * 4;
  return w;
}

// Sets what a kernel may take of shared memory, once per device, and asks how
// many of its CTAs share an SM (with the usual amount).
template <typename F>
int resident(F kernel, size_t most, size_t usual, std::once_flag* once, int* per) {
  const int dev = current_device();
  std::call_once(once[dev], [&] {
    PFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    PFB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per[dev], kernel, kThreads, usual));
    per[dev] = std::max(1, per[dev]);
  });
  return per[dev];
}

constexpr size_t kSharedOfSm = 228 * 1024;
constexpr int kMostPairs = kBlockTokens * kMostTop, kMostParts = kMostExperts + kMostPairs / 16;

template <typename T, int NT, int WARPS>
void launch_down(const Args& a, cudaStream_t stream) {
  using D = Down<T, NT, WARPS>;
  static std::once_flag once[64];
  constexpr size_t most = D::smem(kMostParts, NT == 1 ? 8 * kMostTop : kMostPairs, NT == 1 ? 8 : kBlockTokens);
  static_assert(most <= 227 * 1024, "more than a CTA may have");
  std::call_once(once[current_device()], [] {
    PFB_CUDA(cudaFuncSetAttribute(down_kernel<T, NT, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  });
  const int pairs = a.tokens * a.top;
  // as many CTAs as the device holds at once (a second round of few would take as
  // long as the first), but runs of at least 8 pieces for a warp
  const size_t smem = D::smem(a.most_parts, pairs, a.tokens);
  const int64_t blocks = ceil_div(a.width, 16), pieces = a.most_parts * ceil_div(a.h_row, 64);
  const int64_t slots = std::min<int64_t>(D::kResident, (int64_t)(kSharedOfSm / (smem + 1024))) * device_sm_count(current_device());
  int ranks = 1;
  while (ranks < kMostRanks && blocks * (ranks + 1) <= slots && pieces >= 8 * WARPS * (ranks + 1)) ++ranks;
  launch_following<Args>(down_kernel<T, NT, WARPS>, dim3((unsigned)(blocks * ranks)), WARPS * 32, smem, stream, a, ranks);
}

template <typename T, int NT>
void launch_products(const Args& a, cudaStream_t stream) {
  using U = Up<T, NT>;
  const int sms = device_sm_count(current_device()), pairs = a.tokens * a.top;
  static std::once_flag once_up[64];
  static int per_up[64];
  const int per = resident(up_kernel<T, NT>, U::smem(kMostParts, kMostPairs), U::smem(64, 64), once_up, per_up);
  const int64_t units = (int64_t)a.most_parts * ceil_div(a.inner, 8);
  launch_following<Args>(up_kernel<T, NT>, dim3((unsigned)std::min<int64_t>(units, (int64_t)per * sms)), kThreads, U::smem(a.most_parts, pairs),
                         stream, a);
  const int64_t blocks = ceil_div(a.width, 16);
  // Where CTAs of 16 warps fill the device, and nearly all of it, a block's sums
  // need no cluster (one token, width 2048: 10.5 us for 11.4; of width 2560, 8
  // warps without a cluster took 4 us longer, with 48 blocks 16 did 9 longer).
  // Where the widest clusters leave a quarter of the device idle, 8 warps in a
  // CTA hide more of the memory's latency than 4 (whole calls: fp32, 24 tokens,
  // 64 experts, 128 x 1400: 37.0 us with 4, 32.8 with 8; fp16, 128 tokens, 4 of
  // 128, 200 x 889: 85.4 and 75.5); with more blocks they cost more than they
  // give (fp16, 41 tokens, 4 of 64, 304 x 1024: 55.3 and 61.7).
  if (NT == 1 && 5 * blocks > 4 * sms && blocks <= sms) launch_down<T, NT, NT == 1 ? 16 : 8>(a, stream);
  else if (4 * blocks * kMostRanks <= 3 * sms) launch_down<T, NT, 8>(a, stream);
  else launch_down<T, NT, 4>(a, stream);
}

template <int TB>
size_t route_smem(int64_t experts) {
  const int64_t doubles = TB * (experts + ceil_div(experts, kRouteRanks));
  return (size_t)((doubles + (doubles & 1)) * 8 + TB * kRouteBlock * 4);
}

template <typename T, int TB>
void launch_route(const Args& a, size_t list, cudaStream_t stream) {
  static std::once_flag once[64];
  std::call_once(once[current_device()], [] {
    PFB_CUDA(cudaFuncSetAttribute(route_kernel<T, TB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)std::max(route_smem<TB>(kMostExperts), list_ints(kMostExperts, TB * kMostTop) * sizeof(int))));
  });
  launch_following<Args>(route_kernel<T, TB>, dim3((unsigned)(ceil_div(a.tokens, TB) * kRouteRanks)), kRouteThreads,
                         a.tokens <= TB ? std::max(route_smem<TB>(a.experts), list) : route_smem<TB>(a.experts), stream, a, kRouteRanks);
}

template <typename T>
void launch_typed(const pfk_experts_params& p, const Plan& w, Args a, cudaStream_t stream) {
  for (int64_t first = 0; first < p.tokens; first += w.block) {
    a.tokens = (int)std::min(w.block, p.tokens - first);
    a.x = (const T*)p.x + first * p.x_st;
    a.y = (T*)p.y + first * p.y_st;
    if (p.chosen) a.chosen = p.chosen + first * p.top;
    if (p.weights) a.weights = p.weights + first * p.top;
    const int pairs = a.tokens * a.top;
    a.h_part = pairs * w.h_row;
    a.most_parts = (int)parts_of(p, a.tokens);
    const size_t list = list_ints(a.experts, pairs) * sizeof(int);
    if (a.tokens == 1) launch_route<T, 1>(a, list, stream);
    else if (a.tokens <= 4 || a.tokens > 8) launch_route<T, 4>(a, list, stream);
    else launch_route<T, 8>(a, list, stream);  // one cluster, which lists the pairs
    if (a.tokens > 8) {
      static std::once_flag once[64];
      std::call_once(once[current_device()], [] {
        PFB_CUDA(cudaFuncSetAttribute(list_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(list_ints(kMostExperts, kMostPairs) * sizeof(int))));
      });
      launch_following<Args>(list_kernel, dim3(1), kRouteThreads, list, stream, a);
    }
    a.tokens <= 8 ? launch_products<T, 1>(a, stream) : launch_products<T, 2>(a, stream);
  }
}

}  // namespace

size_t experts_workspace(const pfk_experts_params& p) {
  check(p);
  return p.tokens ? (size_t)plan_of(p).bytes : 0;
}

void launch_experts(const pfk_experts_params& p, cudaStream_t stream) {
  check(p);
  if (p.tokens == 0) return;
  PFB_CHECK_ARG(p.x && p.y && p.router && p.gate_up && p.down, "experts: null pointer");
  PFB_CHECK_ARG(p.y != p.x || p.tokens == 1 || p.y_st == p.x_st, "experts: y shares x's memory with another stride");
  PFB_CHECK_ARG((uintptr_t)p.router % 16 == 0 && (uintptr_t)p.gate_up % 16 == 0 && (uintptr_t)p.down % 16 == 0,
                "experts: weights must be 16-byte aligned");
  const Plan w = plan_of(p);
  PFB_CHECK_ARG(p.workspace && p.workspace_bytes >= (size_t)w.bytes && (uintptr_t)p.workspace % 16 == 0,
                "experts: workspace missing, too small or not 16-byte aligned");
  const int64_t es = size_of(p.dtype);
  Args a = {};
  a.width = (int)p.width;
  a.inner = (int)p.inner;
  a.experts = (int)p.experts;
  a.top = (int)p.top;
  a.renormalize = p.renormalize;
  a.act = p.activation;
  a.x_st = p.x_st;
  a.router = p.router;
  a.router_st = p.router_st;
  a.gate_up = (const char*)p.gate_up;
  a.up_row = p.gate_up_st * es;
  a.up_expert = 2 * p.inner * a.up_row;
  a.down = (const char*)p.down;
  a.down_row = p.down_st * es;
  a.down_expert = p.width * a.down_row;
  a.y_st = p.y_st;
  char* ws = (char*)p.workspace;
  a.xs = ws;
  a.x_row = w.x_row;
  a.h = ws + w.h_at;
  a.h_row = w.h_row;
  a.e = (signed char*)(ws + w.e_at);
  a.e_row = w.e_row;
  a.parts = (int4*)(ws + w.parts_at);
  a.pairs = (int*)(ws + w.pairs_at);
  a.chosen = (int*)(ws + w.chosen_at);
  a.weights = (float*)(ws + w.weights_at);
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_typed<float>(p, w, a, stream);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_typed<__half>(p, w, a, stream);
  else launch_typed<__nv_bfloat16>(p, w, a, stream);
}

}  // namespace pfb
