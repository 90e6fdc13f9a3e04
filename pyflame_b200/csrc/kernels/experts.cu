// experts.cu — a mixture-of-experts layer for a few tokens.
//
//   logits = R x, the `top` largest of them, w = their softmax
//   y = sum_j w_j D_j (act(G_j x) * (U_j x))
//
// The weights of the chosen experts are the work: 3 * width * inner values
// each, read once for all the tokens that chose the expert, and with a few
// tokens memory is the bound.  Three kernels, each launched as a programmatic
// dependent of the one before:
//
// 1. route: a cluster of 8 CTAs for each token, or for four of many: each CTA
//    an eighth of the experts' logits, in 64 bits, since which expert a token
//    takes is a decision that no rounding should make; the first CTA gathers
//    them through distributed shared memory and picks.  Copies x, aligned and
//    padded, for the next kernel.
// 2. up: a CTA of 4 warps for 8 gate rows and their 8 up rows of an expert,
//    which share the 16 rows of a matrix instruction, so that a lane ends with
//    a gate and its up value.  The warps share the summed axis, 64 bytes of a
//    row at a time (256 consecutive bytes a CTA).  What leaves is w act(g) u
//    in two 16-bit parts (one fp32 value): a single one would round as
//    coarsely as the output does.
// 3. down: a cluster for 16 rows of the output.  All (used expert, 64 bytes)
//    pieces of those rows form one list, of which each warp of the cluster
//    takes an equal run; at an expert's end it adds what it has to its own
//    table of tokens in shared memory.  The tables are added in the order of
//    warps and ranks: no atomics, the same bits each time.
//
// Rows come straight from memory into operand registers (streamed.cuh).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>

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
constexpr int kRouteRanks = 8;
constexpr int kRouteThreads = 256;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRouteBlock = 1024;  // values of x that the router's kernel holds of a token at a time

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
  int4* used;  // how many, then of each: expert, first of its pairs, their number
  int* pairs;  // [tokens * top] by expert
};

// ---------------------------------------------------------------------------
// route
// ---------------------------------------------------------------------------

// TB tokens a cluster
template <typename T, int TB>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(Args a) {
  extern __shared__ double shared[];
  double* xd = shared;                               // [TB][kRouteBlock]
  double* logits = shared + TB * kRouteBlock;        // [TB][experts of a rank]
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int share = (a.experts + kRouteRanks - 1) / kRouteRanks;
  double* all = logits + TB * share;                 // rank 0: [TB][experts]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = (int)(blockIdx.x / kRouteRanks) * TB;
  const int mine = min(TB, a.tokens - first);
  const int e0 = rank * share, e1 = min(a.experts, e0 + share);
  begin();

  // x for the next kernel: the cluster's CTAs share the row
  const int padded = (int)(a.x_row / (int)sizeof(T));
  for (int i = rank * kRouteThreads + tid; i < mine * padded; i += kRouteRanks * kRouteThreads) {
    const int n = i / padded, d = i - n * padded;
    reinterpret_cast<T*>(a.xs + (first + n) * a.x_row)[d] =
        d < a.width ? ((const T*)a.x)[(first + n) * a.x_st + d] : from_float<T>(0.f);
  }

  for (int i = tid; i < TB * share; i += kRouteThreads) logits[i] = 0.0;
  for (int base = 0; base < a.width; base += kRouteBlock) {
    const int len = min(kRouteBlock, a.width - base);
    const int len4 = (len + 3) & ~3;  // rows of the router are padded with zeros to a multiple of 4
    __syncthreads();
    for (int i = tid; i < TB * len4; i += kRouteThreads) {
      const int n = i / len4, d = i - n * len4;
      xd[n * kRouteBlock + d] =
          n < mine && d < len ? (double)to_float<T>(((const T*)a.x)[(first + n) * a.x_st + base + d]) : 0.0;
    }
    __syncthreads();
    for (int e = e0 + warp; e < e1; e += kRouteThreads / 32) {
      const float4* row = reinterpret_cast<const float4*>(a.router + e * a.router_st + base);
      double sum[TB];
#pragma unroll
      for (int n = 0; n < TB; ++n) sum[n] = 0.0;
#pragma unroll 4
      for (int d = lane; d < len4 / 4; d += 32) {
        const float4 r = row[d];
        const double r0 = r.x, r1 = r.y, r2 = r.z, r3 = r.w;
#pragma unroll
        for (int n = 0; n < TB; ++n) {
          const double2 u = *reinterpret_cast<const double2*>(xd + n * kRouteBlock + 4 * d);
          const double2 v = *reinterpret_cast<const double2*>(xd + n * kRouteBlock + 4 * d + 2);
          sum[n] = fma(r0, u.x, fma(r1, u.y, fma(r2, v.x, fma(r3, v.y, sum[n]))));
        }
      }
#pragma unroll
      for (int n = 0; n < TB; ++n) {
#pragma unroll
        for (int o = 16; o; o >>= 1) sum[n] += __shfl_xor_sync(~0u, sum[n], o);
        if (lane == 0) logits[n * share + e - e0] += sum[n];
      }
    }
  }
  __syncthreads();
  cluster.sync();  // rank 0 has started, and its memory can be written
  double* to = cluster.map_shared_rank(all, 0);
  for (int i = tid; i < TB * (e1 - e0); i += kRouteThreads) {
    const int n = i / (e1 - e0), e = i - n * (e1 - e0);
    to[n * a.experts + e0 + e] = logits[n * share + e];
  }
  cluster.sync();
  if (rank != 0 || warp >= mine) return;

  // a warp picks for a token; NaN counts as the lowest
  const int n = warp;
  double* l = all + n * a.experts;
  double best = -INFINITY;
  for (int e = lane; e < a.experts; e += 32) {
    if (!(l[e] >= -1.7976931348623157e308)) l[e] = -INFINITY;
    best = fmax(best, l[e]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) best = fmax(best, __shfl_xor_sync(~0u, best, o));
  float total = 0.f;
  if (!a.renormalize) {
    for (int e = lane; e < a.experts; e += 32) total += expf((float)(l[e] - best));
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
  }
  unsigned taken = 0;  // of the lane's experts lane + 32 i
  float part = 0.f;    // of the choice that the lane keeps: the lane-th
  int kept = 0;
  for (int j = 0; j < a.top; ++j) {
    double m = -INFINITY;
    int at = INT_MAX;
    for (int e = lane, i = 0; e < a.experts; e += 32, ++i) {
      if (!(taken >> i & 1) && (at == INT_MAX || l[e] > m)) {
        m = l[e];
        at = e;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const double om = __shfl_xor_sync(~0u, m, o);
      const int oat = __shfl_xor_sync(~0u, at, o);
      if (oat != INT_MAX && (at == INT_MAX || om > m || (om == m && oat < at))) {
        m = om;
        at = oat;
      }
    }
    if ((at & 31) == lane) taken |= 1u << (at >> 5);
    const float w = expf((float)(m - best));
    if (a.renormalize) total += w;
    if (lane == j) {
      part = w;
      kept = at;
    }
  }
  if (lane < a.top) {
    a.chosen[(long long)(first + n) * a.top + lane] = kept;
    a.weights[(long long)(first + n) * a.top + lane] = part / total;
  }
}

// ---------------------------------------------------------------------------
// up
// ---------------------------------------------------------------------------

// acc[n] += 16 rows of this warp x its vectors, over the rows' pieces of 64
// bytes c = first, first + step, ... below `pieces`.  Bytes from `bytes` on
// belong to no row.  PARTS: of the vectors, which add up.
// UNROLL pieces are in flight, and share accumulators that are added to acc in
// fp32, rounded to nearest: the tensor cores truncate what they add.
template <typename T, int NT, int PARTS, int UNROLL>
__device__ __forceinline__ void stream_rows(float (&acc)[NT][4], const char* row0, const char* row1, const char* const (&vec)[NT],
                                            long long part, int first, int step, int pieces, int bytes, int t) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int c0 = first; c0 < pieces; c0 += step * UNROLL) {
    uint4 a0[UNROLL], a1[UNROLL], b[UNROLL][PARTS][NT];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int at = (c0 + u * step) * 64 + t * 16;
      const bool in = c0 + u * step < pieces && at < bytes;
      a0[u] = in && row0 ? load_stream(row0 + at) : zero;
      a1[u] = in && row1 ? load_stream(row1 + at) : zero;
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          b[u][p][n] = in && vec[n] ? *reinterpret_cast<const uint4*>(vec[n] + p * part + at) : zero;
    }
    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p) chunk_product<T, NT>(sum, a0[u], a1[u], b[u][p]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[n][r] += sum[n][r];
  }
}

template <typename T>
struct Parts {
  static constexpr int kH = sizeof(T) == 2 ? 2 : 1;  // of an intermediate value
};

template <typename T, int NT, int UNROLL>
__device__ __forceinline__ void up_block(const Args& a, int expert, int row, const int* list, int count, float4* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const char* base = a.gate_up + expert * a.up_expert;
  const int f = row + g;
  const char* gate = f < a.inner ? base + f * a.up_row : nullptr;
  const char* up = f < a.inner ? base + (a.inner + (long long)f) * a.up_row : nullptr;
  const char* vec[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) vec[n] = n * 8 + g < count ? a.xs + (long long)(list[n * 8 + g] / a.top) * a.x_row : nullptr;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  const int bytes = (int)min(a.x_row, a.up_row);
  stream_rows<T, NT, 1, UNROLL>(acc, gate, up, vec, 0, warp, kWarps, (bytes + 63) / 64, bytes, t);
#pragma unroll
  for (int n = 0; n < NT; ++n) red[(warp * NT + n) * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
  __syncthreads();
  static_assert(NT <= kWarps, "a warp finishes a block of vectors");
  if (warp < NT) {
    float4 s = red[warp * 32 + lane];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float4 v = red[(w * NT + warp) * 32 + lane];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int slot = warp * 8 + 2 * t + i;
      if (slot >= count) continue;
      const int pair = list[slot];
      const float gv = i ? s.y : s.x, uv = i ? s.w : s.z;
      const float act = a.act ? act_apply<2>(gv) : act_apply<5>(gv);
      // rows behind the last are zeros (their sums are)
      const float v = act * uv * a.weights[pair];
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
  __syncthreads();
}

// grid: (blocks of 8 rows + 1, experts or pairs).  The extra block of the
// first row lists the pairs by expert for the next kernel.
template <typename T>
__global__ void __launch_bounds__(kThreads) up_kernel(Args a) {
  __shared__ float4 red[kWarps * 4 * 32];
  extern __shared__ int list[];  // [pairs]
  __shared__ int counts[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  begin();
  const int pairs = a.tokens * a.top;

  if (blockIdx.x == gridDim.x - 1) {
    if (blockIdx.y) return;
    __shared__ int hist[kMostExperts];
    for (int e = tid; e < a.experts; e += kThreads) hist[e] = 0;
    __syncthreads();
    // the order of an expert's pairs has no effect: a token has one of them
    // at most, and their sums are apart
    for (int p = tid; p < pairs; p += kThreads) list[p] = atomicAdd(&hist[a.chosen[p]], 1);
    __syncthreads();
    if (warp == 0) {  // starts of the used experts
      int start = 0, used = 0;
      for (int base = 0; base < a.experts; base += 32) {
        const int e = base + lane, n = e < a.experts ? hist[e] : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += up;
        }
        const unsigned some = __ballot_sync(~0u, n > 0);
        if (n) a.used[1 + used + __popc(some & ((1u << lane) - 1))] = make_int4(e, start + sum - n, n, 0);
        if (e < a.experts) hist[e] = start + sum - n;
        start += __shfl_sync(~0u, sum, 31);
        used += __popc(some);
      }
      if (lane == 0) a.used[0] = make_int4(used, 0, 0, 0);
    }
    __syncthreads();
    for (int p = tid; p < pairs; p += kThreads) a.pairs[hist[a.chosen[p]] + list[p]] = p;
    return;
  }

  // the block's expert and the pairs that chose it: with fewer pairs than
  // experts, the expert of pair y where that is the first of its pairs
  const bool by_pair = pairs < a.experts;
  const int expert = by_pair ? a.chosen[blockIdx.y] : (int)blockIdx.y;
  int count = 0;
  for (int base = 0; base < pairs; base += kThreads) {
    const int p = base + tid;
    const bool match = p < pairs && a.chosen[p] == expert;
    const unsigned some = __ballot_sync(~0u, match);
    if (lane == 0) counts[warp] = __popc(some);
    __syncthreads();
    int at = count;
    for (int w = 0; w < warp; ++w) at += counts[w];
    if (match) list[at + __popc(some & ((1u << lane) - 1))] = p;
    for (int w = 0; w < kWarps; ++w) count += counts[w];
    __syncthreads();
  }
  if (count == 0 || (by_pair && list[0] != (int)blockIdx.y)) return;
  const int row = blockIdx.x * 8;
  for (int at = 0; at < count; at += 32) {
    const int some = min(32, count - at);
    if (some <= 8) up_block<T, 1, 8>(a, expert, row, list + at, some, red);
    else if (some <= 16) up_block<T, 2, 4>(a, expert, row, list + at, some, red);
    else up_block<T, 4, 2>(a, expert, row, list + at, some, red);
  }
}

// ---------------------------------------------------------------------------
// down
// ---------------------------------------------------------------------------

// One expert's pieces [c0, c1) for some of its pairs, added to the warp's table.
template <typename T, int NT, int UNROLL>
__device__ __forceinline__ void down_run(const Args& a, const char* row0, const char* row1, int bytes, int first, int count, int c0,
                                         int c1, float* table) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const char* vec[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) vec[n] = n * 8 + g < count ? a.h + (long long)a.pairs[first + n * 8 + g] * a.h_row : nullptr;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  stream_rows<T, NT, Parts<T>::kH, UNROLL>(acc, row0, row1, vec, a.h_part, c0, 1, c1, bytes, t);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int slot = n * 8 + 2 * t + i;
      if (slot < count) {
        float* to = table + a.pairs[first + slot] / a.top * 16;
        to[g] += acc[n][i];
        to[g + 8] += acc[n][i + 2];
      }
    }
  __syncwarp();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) down_kernel(Args a) {
  extern __shared__ float tables[];  // [warps][tokens][16]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / ranks) * 16;
  const int cells = a.tokens * 16;
  for (int i = tid; i < kWarps * cells; i += kThreads) tables[i] = 0.f;
  begin();
  const int bytes = (int)min(a.h_row, a.down_row), pieces = (bytes + 63) / 64;
  const int used = a.used[0].x;
  const int total = used * pieces, q = rank * kWarps + warp, of = ranks * kWarps;
  const int p0 = (int)((long long)total * q / of), p1 = (int)((long long)total * (q + 1) / of);
  __syncthreads();
  float* table = tables + warp * cells;
  for (int p = p0; p < p1;) {
    const int i = p / pieces, c0 = p - i * pieces, c1 = min(pieces, c0 + p1 - p);
    const int4 u = a.used[1 + i];
    const char* base = a.down + u.x * a.down_expert;
    const char* row0 = row + g < a.width ? base + (row + g) * a.down_row : nullptr;
    const char* row1 = row + g + 8 < a.width ? base + (row + g + 8) * a.down_row : nullptr;
    for (int at = 0; at < u.z; at += 32) {
      const int some = min(32, u.z - at);
      if (some <= 8) down_run<T, 1, sizeof(T) == 2 ? 4 : 8>(a, row0, row1, bytes, u.y + at, some, c0, c1, table);
      else if (some <= 16) down_run<T, 2, 4>(a, row0, row1, bytes, u.y + at, some, c0, c1, table);
      else down_run<T, 4, 2>(a, row0, row1, bytes, u.y + at, some, c0, c1, table);
    }
    p += c1 - c0;
  }
  __syncthreads();
  for (int i = tid; i < cells; i += kThreads) {
    float s = tables[i];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s += tables[w * cells + i];
    tables[i] = s;
  }
  cluster.sync();
  for (int i = rank * kThreads + tid; i < cells; i += kThreads * ranks) {
    float s = 0.f;
    for (int r = 0; r < ranks; ++r) s += cluster.map_shared_rank(tables, r)[i];
    const int n = i >> 4, d = row + (i & 15);
    if (d < a.width) ((T*)a.y)[n * a.y_st + d] = from_float<T>(s);
  }
  cluster.sync();  // the others' reads of this CTA's table are over
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
  int64_t block, x_row, h_row, h_part;  // of a pass
  int64_t h_at, used_at, pairs_at, chosen_at, weights_at, bytes;
};

Plan plan_of(const pfk_experts_params& p) {
  Plan w;
  const int64_t es = size_of(p.dtype);
  w.block = std::min<int64_t>(p.tokens, kBlockTokens);
  const int64_t pairs = w.block * p.top;
  w.x_row = round_up(p.width * es, 16);
  w.h_row = round_up(round_up(p.inner, 8) * es, 16);
  w.h_part = pairs * w.h_row;
  w.h_at = round_up(w.block * w.x_row, 128);
  w.used_at = round_up(w.h_at + w.h_part * (es == 2 ? 2 : 1), 128);
  w.pairs_at = round_up(w.used_at + (std::min(pairs, p.experts) + 1) * (int64_t)sizeof(int4), 128);
  w.chosen_at = round_up(w.pairs_at + pairs * 4, 128);
  w.weights_at = round_up(w.chosen_at + pairs * 4, 128);
  w.bytes = w.weights_at + pairs * 4;
  return w;
}

template <int TB>
size_t route_smem(int64_t experts) {
  return (size_t)TB * (kRouteBlock + ceil_div(experts, kRouteRanks) + experts) * sizeof(double);
}

template <typename T, int TB>
void launch_route(const Args& a, cudaStream_t stream) {
  static std::once_flag once[64];
  std::call_once(once[current_device()], [] {
    PFB_CUDA(cudaFuncSetAttribute(route_kernel<T, TB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)route_smem<TB>(kMostExperts)));
  });
  const size_t smem = route_smem<TB>(a.experts);
  launch_following<Args>(route_kernel<T, TB>, dim3((unsigned)(ceil_div(a.tokens, TB) * kRouteRanks)), kRouteThreads, smem, stream, a,
                         kRouteRanks);
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
    a.tokens <= 16 ? launch_route<T, 1>(a, stream) : launch_route<T, 4>(a, stream);
    const size_t list = (size_t)pairs * 4;
    launch_following<Args>(up_kernel<T>, dim3((unsigned)(ceil_div(p.inner, 8) + 1), (unsigned)std::min<int64_t>(pairs, p.experts)),
                           kThreads, list, stream, a);
    // enough CTAs for the device, but runs of at least 8 pieces for a warp
    const int64_t blocks = ceil_div(p.width, 16), pieces = std::min<int64_t>(pairs, p.experts) * ceil_div(w.h_row, 64);
    const int sms = device_sm_count(current_device());
    int ranks = 1;
    while (ranks < 8 && blocks * ranks < 4 * sms && pieces >= 8 * kWarps * 2 * ranks) ranks *= 2;
    const size_t tables = (size_t)kWarps * a.tokens * 16 * sizeof(float);
    launch_following<Args>(down_kernel<T>, dim3((unsigned)(blocks * ranks)), kThreads, tables, stream, a, ranks);
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
  a.used = (int4*)(ws + w.used_at);
  a.pairs = (int*)(ws + w.pairs_at);
  a.chosen = (int*)(ws + w.chosen_at);
  a.weights = (float*)(ws + w.weights_at);
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_typed<float>(p, w, a, stream);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_typed<__half>(p, w, a, stream);
  else launch_typed<__nv_bfloat16>(p, w, a, stream);
}

}  // namespace pfb
