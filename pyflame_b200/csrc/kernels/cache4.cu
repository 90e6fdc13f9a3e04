// cache4.cu — filling a paged key-value cache held in 4 bits, and reading its
// values back.
//
// A group of a head's values x becomes 16 even steps from its least value on:
//   low = bf16(min x), step = bf16((max x - low) * (1 / 15)),
//   code = clamp(rint((x - low) * (1 / step)), 0, 15),
// in single fp32 operations, so that a value's code depends on the group
// alone.  Which code a value next to a border gets changes it by a whole step:
// keys are therefore rotated in 64 bits and rounded to fp32 once.  bfloat16
// steps and lows reach as far as fp32 does; their own rounding moves the steps
// by 2^-9 of the range, far below half a step, 1/30 of it.
//
// A row (a head of a token) takes a lane for 16 of its values: minima and
// maxima meet by shuffles, and a lane's 16 codes are two words of a key row or
// four halves of value words.  k, v and q are read once, codes and q written
// once, but instructions bound it: a prompt of 8191 tokens, 32 query and 8
// key-value heads of 128 in fp16, 176 MB, takes 47 us (27 at 6.56 TB/s) with
// 63 % of the issue slots in use; a lane for 8 values took 52.  Reading it back
// takes 14 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../common.hpp"
#include "cache4.cuh"
#include "decode.cuh"
#include "kernels.hpp"

namespace pfb {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTokens = 8;  // a CTA takes at most

struct Args {
  uint32_t *k, *v, *k_scales, *v_scales;
  int heads, head_dim, group, blocks, groups;  // blocks of 32 values, words of a record's scales
  FastDiv by_page, by_chunks;
  long long num_slots;
  int* err;
  const void* src[3];  // k, v, q
  long long st[3], sh[3];
  int wide;  // rows may be read, and q written, 16 bytes at a time
  void* q_out;
  long long qo_st, qo_sh;
  int q_heads;
  int tokens, per_cta, split;
  const int64_t* slots;
  const int64_t* positions;
  const double* inv_freq;
  int rot, interleaved;
  double factor;
  void* out[2];  // of a read: k, v
};

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <> __device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T of_float(float v);
template <> __device__ __forceinline__ float of_float(float v) { return v; }
template <> __device__ __forceinline__ __half of_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 of_float(float v) { return __float2bfloat16_rn(v); }

template <typename T>
union Eight {
  uint4 raw[sizeof(T) / 2];
  T v[8];
  __device__ Eight() {}
};

template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p, bool wide) {
  Eight<T> e;
  if (wide) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.raw[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e.v[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = as_float<T>(e.v[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], bool wide) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = of_float<T>(x[i]);
  if (wide) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, e.raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e.v[i];
  }
}

// Cosine and sine of pos * w in 64 bits.  pos * w is a + b exactly, 2 / pi is
// kHigh + kLow, and the quarter turns n + r, |r| <= 1/2, come from their
// products, rounded only after n is subtracted.  The rest, |x| <= pi/4, goes
// through the two Taylor series up to x^17 and x^18, whose next terms are
// below 10^-19 (a third of the time of the library's function, which takes any
// argument: 5 us less for a prompt of 8191 tokens).
__device__ __forceinline__ double2 cos_sin(long long pos, double w) {
  constexpr double kHigh = 0x1.45f306dc9c883p-1, kLow = -0x1.6b01ec5417056p-55;
  const double p = (double)pos, a = p * w, b = fma(p, w, -a);
  const double n = rint(a * kHigh);
  const double r = fma(a, kHigh, -n) + fma(b, kHigh, a * kLow);
  const double x = r * 1.5707963267948966, z = x * x;
  double s = 1. / 355687428096000.;  // 1 / 17!
  s = fma(s, z, -1. / 1307674368000.);
  s = fma(s, z, 1. / 6227020800.);
  s = fma(s, z, -1. / 39916800.);
  s = fma(s, z, 1. / 362880.);
  s = fma(s, z, -1. / 5040.);
  s = fma(s, z, 1. / 120.);
  s = fma(s, z, -1. / 6.);
  s = fma(s, z * x, x);
  double c = -1. / 6402373705728000.;  // 1 / 18!
  c = fma(c, z, 1. / 20922789888000.);
  c = fma(c, z, -1. / 87178291200.);
  c = fma(c, z, 1. / 479001600.);
  c = fma(c, z, -1. / 3628800.);
  c = fma(c, z, 1. / 40320.);
  c = fma(c, z, -1. / 720.);
  c = fma(c, z, 1. / 24.);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.);
  const int quarter = (int)((long long)n & 3);
  if (quarter & 1) {
    const double t = c;
    c = -s;
    s = t;
  }
  return quarter & 2 ? make_double2(-c, -s) : make_double2(c, s);
}

// The larger and the smaller of two numbers, NaN if one is.
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// Codes of a row's group, of which each of `lanes` lanes has 16 values; `in`: how
// many are inside the head (of a last lane 8, with the other 8 the same again,
// or none), `some`: whether any of the group are.  Returns the group's scales;
// codes: words of 8 values.
__device__ __forceinline__ unsigned quantize(const float (&x)[16], int in, bool some, int lanes, unsigned (&codes)[2]) {
  float least = x[0], most = x[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) {
    least = min_nan(least, x[e]);
    most = max_nan(most, x[e]);
  }
  if (in <= 0) {
    least = INFINITY;
    most = -INFINITY;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    if (o >= lanes) break;  // the same in all lanes
    least = min_nan(least, __shfl_xor_sync(~0u, least, o));
    most = max_nan(most, __shfl_xor_sync(~0u, most, o));
  }
  const float low = __bfloat162float(__float2bfloat16_rn(least));
  float step = __bfloat162float(__float2bfloat16_rn((most - low) * (1.f / 15.f)));
  if (!(step >= 0x1p-126f)) step = 0.f;
  const float times = step > 0.f ? __frcp_rn(step) : 0.f;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    // The addition rounds to a whole number, ties to even: its bits are
    // 0x4b000000 + code.  What the eight constants add up to is taken off.
    unsigned sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = fminf(fmaxf((x[8 * s + e] - low) * times, 0.f), 15.f) + 0x1p23f;
      sum += __float_as_uint(t) << (4 * e);
    }
    codes[s] = 8 * s < in ? sum - 0x4b000000u * 0x11111111u : 0;
  }
  // (a group behind the head's end is kept as zeros)
  const bool fine = least >= -0x1p126f && most <= 0x1p126f;
  const unsigned word = (__float_as_uint(step) & 0xffff0000u) | __float_as_uint(low) >> 16;
  return !some ? 0 : fine ? word : 0x7fc07fc0u;
}

// A slot's token: head 0 of its page, and its offset there; page -1: none.
struct Place {
  int page, offset;
};
__device__ __forceinline__ Place place_of(const Args& a, long long slot) {
  if (slot >= a.num_slots && a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
  if (slot < 0 || slot >= a.num_slots) return {-1, 0};
  const unsigned page = a.by_page.div((unsigned)slot);
  return {(int)page, (int)((unsigned)slot - page * a.by_page.d)};
}
__device__ __forceinline__ long long record_of(const Args& a, const Place& p, int head) {
  return ((long long)p.page * a.heads + head) * a.by_page.d + p.offset;
}
// The place of 16 bits `half` of a token's values.
__device__ __forceinline__ long long value_at(const Args& a, const Place& p, int head, int blocks, int half) {
  const long long pair = ((long long)p.page * a.heads + head) * ((a.by_page.d + 1) >> 1) + (p.offset >> 1);
  return (pair * (8 * blocks) + half) * 2 + (p.offset & 1);
}

// Where the angle of pair p lies among a token's half: lanes that turn chunks
// of 8 values next to each other read places next to each other.  (In the order
// of the pairs, 16 lanes' reads met in one bank: 99 us for a prompt of 8191
// tokens.)
__device__ __forceinline__ int spread_of(int half, int interleaved) {
  const int angles = interleaved ? 4 : 8;  // of a chunk
  return half % angles == 0 ? angles : 1;
}
__device__ __forceinline__ int angle_at(int p, int half, int spread) { return p % spread * (half / spread) + p / spread; }

// Lanes of a row of BLOCKS blocks of 32 values, 16 each.
constexpr int lanes_of(int blocks) { return blocks <= 2 ? 4 : blocks <= 4 ? 8 : 16; }

// Keys and values.
template <typename T, int BLOCKS, bool KEYS, bool WIDE>
__device__ __forceinline__ void store_rows(const Args& a, const double2* turns, const Place* places, int first, int mine,
                                           int head_first, int head_last) {
  constexpr int LANES = lanes_of(BLOCKS), ROWS = 32 / LANES;  // rows of a warp at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = a.rot >> 1, part = lane % LANES, d0 = part * 16;
  const int in = min(16, a.head_dim - d0);  // values inside the head; not above 0: none
  const int lanes = min(a.group / 16, LANES), group = part / lanes;
  const bool some = group * lanes * 16 < a.head_dim;
  const int spread = spread_of(half, a.interleaved);
  const int heads = head_last - head_first, rows = mine * heads;
  const long long st = a.st[KEYS ? 0 : 1], sh = a.sh[KEYS ? 0 : 1];
  int i = warp * ROWS + lane / LANES, tok = i / heads, head = head_first + i - tok * heads;
  for (int i0 = warp * ROWS; i0 < rows; i0 += kWarps * ROWS, i += kWarps * ROWS) {
    const Place place = i < rows ? places[tok] : Place{-1, 0};
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
    if (place.page >= 0) {
      const T* src = (const T*)a.src[KEYS ? 0 : 1] + (long long)(first + tok) * st + head * sh;
      const double2* cs = turns + tok * half;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int d = d0 + 8 * s;
        if (8 * s >= in) continue;
        float v[8];
        load8<T>(v, src + d, WIDE);
        if (KEYS && d < a.rot) {
          if (a.interleaved) {  // pairs (2i, 2i + 1), inside the lane
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              if (d + e >= a.rot) continue;
              const double2 t = cs[spread == 4 ? e / 2 * (half / 4) + d / 8 : (d + e) >> 1];
              const double u = v[e], w = v[e + 1];
              v[e] = (float)fma(u, t.x, -(w * t.y));
              v[e + 1] = (float)fma(u, t.y, w * t.x);
            }
          } else if (spread == 8) {  // with the values half a rotation on or back
            const bool second = d >= half;
            float w[8];
            load8<T>(w, src + (second ? d - half : d + half), WIDE);
            const double2* at = cs + (second ? d - half : d) / 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const double2 t = at[e * (half / 8)];
              v[e] = (float)fma((double)v[e], t.x, (double)(second ? w[e] : -w[e]) * t.y);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (d + e >= a.rot) continue;
              const bool second = d + e >= half;
              const int p = second ? d + e - half : d + e;
              const double2 t = cs[p];
              const float w = as_float<T>(src[second ? p : p + half]);
              v[e] = (float)fma((double)v[e], t.x, (double)(second ? w : -w) * t.y);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[8 * s + e] = v[e];
          if (s == 0) x[8 + e] = v[e];
        }
      }
    }
    unsigned codes[2];
    const unsigned scales = quantize(x, in, some, lanes, codes);
    if (place.page >= 0 && part < 2 * BLOCKS) {
      const long long at = record_of(a, place, head);
      if constexpr (KEYS) {
#pragma unroll
        for (int s = 0; s < 2; ++s) a.k[at * (4 * BLOCKS) + cache4_key_word(2 * part + s, BLOCKS)] = codes[s];
      } else {
        unsigned short* v = reinterpret_cast<unsigned short*>(a.v) + value_at(a, place, head, BLOCKS, 0);
#pragma unroll
        for (int s = 0; s < 4; ++s) v[2 * cache4_value_half(4 * part + s, BLOCKS)] = (unsigned short)(codes[s >> 1] >> (16 * (s & 1)));
      }
      if (part % lanes == 0) (KEYS ? a.k_scales : a.v_scales)[at * a.groups + group] = scales;
    }
    for (head += kWarps * ROWS; head >= head_last && tok < mine; ++tok) head -= heads;
  }
}

// Queries, whose roundings decide nothing, in fp32 with cosines and sines
// rounded to it: three roundings of 2^-24 of a pair's size.  A thread turns two
// chunks of 8 values that turn together, or copies two.  Both are read before
// either is written: q_out may be q.
template <typename T, bool WIDE>
__device__ __forceinline__ void turn_queries(const Args& a, const float2* turns, const Place* places, int first, int mine,
                                             int head_first, int head_last) {
  const int half = a.rot >> 1, chunks = a.head_dim / 8;
  const bool by_chunk = a.interleaved || half % 8 == 0;  // a turned chunk's partner is a chunk, or itself
  const int heads = head_last - head_first;
  if (!by_chunk) {  // a value pair at a time
    const int items = half + (a.head_dim - a.rot);
    for (int i = threadIdx.x; i < mine * heads * items; i += kThreads) {
      const int row = i / items, p = i - row * items, tok = row / heads, head = head_first + row - tok * heads;
      if (places[tok].page < 0) continue;
      const T* src = (const T*)a.src[2] + (long long)(first + tok) * a.st[2] + head * a.sh[2];
      T* to = (T*)a.q_out + (long long)(first + tok) * a.qo_st + head * a.qo_sh;
      if (p < half) {
        const float2 cs = turns[tok * half + p];
        const float u = as_float<T>(src[p]), v = as_float<T>(src[p + half]);
        to[p] = of_float<T>(fmaf(u, cs.x, -(v * cs.y)));
        to[p + half] = of_float<T>(fmaf(u, cs.y, v * cs.x));
      } else {
        to[p + half] = src[p + half];
      }
    }
    return;
  }
  const int pairs = a.interleaved ? 0 : half / 8;  // items that turn two chunks with each other
  const int items = pairs + (chunks - 2 * pairs + 1) / 2;
  const int step = kThreads / items ? kThreads / items : 1;  // items: at most 16
  const int row_first = threadIdx.x / items, j = threadIdx.x - row_first * items;
  if (row_first >= step) return;
  const bool turn = j < pairs;
  const int c1 = turn ? j : 2 * pairs + 2 * (j - pairs), c2 = turn ? j + pairs : c1 + 1;
  int tok = row_first / heads, head = head_first + row_first - tok * heads;
  for (int i = row_first; i < mine * heads; i += step) {
    if (places[tok].page >= 0) {
      const T* src = (const T*)a.src[2] + (long long)(first + tok) * a.st[2] + head * a.sh[2];
      T* to = (T*)a.q_out + (long long)(first + tok) * a.qo_st + head * a.qo_sh;
      float x[8], y[8];
      load8<T>(x, src + 8 * c1, WIDE);
      if (c2 < chunks) load8<T>(y, src + 8 * c2, WIDE);
      const float2* cs = turns + tok * half;
      if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = cs[e * pairs + j];
          const float u = x[e];
          x[e] = fmaf(u, t.x, -(y[e] * t.y));
          y[e] = fmaf(u, t.y, y[e] * t.x);
        }
      } else if (a.interleaved) {
        const int spread = spread_of(half, 1);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          if (8 * c1 + e < a.rot) {
            const float2 t = cs[spread == 4 ? e / 2 * (half / 4) + c1 : 4 * c1 + e / 2];
            const float u = x[e];
            x[e] = fmaf(u, t.x, -(x[e + 1] * t.y));
            x[e + 1] = fmaf(u, t.y, x[e + 1] * t.x);
          }
          if (8 * c2 + e < a.rot && c2 < chunks) {
            const float2 t = cs[spread == 4 ? e / 2 * (half / 4) + c2 : 4 * c2 + e / 2];
            const float u = y[e];
            y[e] = fmaf(u, t.x, -(y[e + 1] * t.y));
            y[e + 1] = fmaf(u, t.y, y[e + 1] * t.x);
          }
        }
      }
      store8<T>(to + 8 * c1, x, WIDE);
      if (c2 < chunks) store8<T>(to + 8 * c2, y, WIDE);
    }
    for (head += step; head >= head_last && tok < mine; ++tok) head -= heads;
  }
}

// CTA (i, j): tokens i * per_cta on, and the j-th part of their heads
template <typename T, int BLOCKS, bool WIDE>
__global__ void __launch_bounds__(kThreads, 8) append_kernel(Args a) {
  extern __shared__ double2 turns[];  // [per_cta][rot / 2], then the same as float2
  __shared__ Place places[kTokens];
  const int tid = threadIdx.x, half = a.rot >> 1;
  begin();
  const int first = blockIdx.x * a.per_cta, mine = min(a.per_cta, a.tokens - first);
  float2* turns32 = reinterpret_cast<float2*>(turns + a.per_cta * half);
  const int spread = spread_of(half, a.interleaved);
  for (int i = tid; i < mine * half; i += kThreads) {
    const int tok = i / half, p = i - tok * half, at = tok * half + angle_at(p, half, spread);
    double2 cs = cos_sin(a.positions[first + tok], a.inv_freq[p]);
    cs.x *= a.factor;
    cs.y *= a.factor;
    turns[at] = cs;
    turns32[at] = make_float2((float)cs.x, (float)cs.y);
  }
  if (tid < mine) places[tid] = place_of(a, a.slots[first + tid]);
  __syncthreads();
  const int part = blockIdx.y;
  const int h0 = a.heads * part / a.split, h1 = a.heads * (part + 1) / a.split;
  const int q0 = a.q_heads * part / a.split, q1 = a.q_heads * (part + 1) / a.split;
  // queries are bound by memory, keys and values by their instructions: every
  // other CTA begins with the latter
  const bool late = blockIdx.x & 1;
  if (!late && q0 < q1) turn_queries<T, WIDE>(a, turns32, places, first, mine, q0, q1);
  if (h0 < h1) {
    store_rows<T, BLOCKS, true, WIDE>(a, turns, places, first, mine, h0, h1);
    store_rows<T, BLOCKS, false, WIDE>(a, turns, places, first, mine, h0, h1);
  }
  if (late && q0 < q1) turn_queries<T, WIDE>(a, turns32, places, first, mine, q0, q1);
}

// CTA (i, j): tokens i * per_cta on, and the j-th part of their keys' and
// values' chunks of 8 values, one a thread at a time.
constexpr int kReadThreads = 256;
constexpr int kReadTokens = 8;

template <typename T>
__global__ void __launch_bounds__(kReadThreads) read_kernel(Args a) {
  __shared__ Place places[kReadTokens];
  begin();
  const int tid = threadIdx.x, first = blockIdx.x * a.per_cta, mine = min(a.per_cta, a.tokens - first);
  if (tid < mine) places[tid] = place_of(a, a.slots[first + tid]);
  __syncthreads();
  const int chunks = a.head_dim / 8, items = 2 * a.heads * chunks, each = items / a.split, rest = items % a.split;
  const int part = blockIdx.y, from = each * part + min(part, rest), to = from + each + (part < rest);
  for (int i = from + tid; i < to; i += kReadThreads) {
    const int row = (int)a.by_chunks.div((unsigned)i), chunk = i - row * chunks;
    const bool value = row >= a.heads;
    const int head = value ? row - a.heads : row;
    // words of the codes, or halves of them, and of the scales
    const uint32_t* codes = value ? a.v : a.k;
    const uint32_t* scales = (value ? a.v_scales : a.k_scales) + chunk * 8 / a.group;
    const int at = value ? cache4_value_half(2 * chunk, a.blocks) : cache4_key_word(chunk, a.blocks);
    const int next = value ? cache4_value_half(2 * chunk + 1, a.blocks) : 0;
    T* out = (T*)a.out[value] + (((long long)first * a.heads + head) * chunks + chunk) * 8;
#pragma unroll 4
    for (int tok = 0; tok < mine; ++tok) {
      const bool there = places[tok].page >= 0;
      const Place place = there ? places[tok] : Place{0, 0};
      const long long record = record_of(a, place, head);
      unsigned c;
      if (value) {
        const unsigned short* v = reinterpret_cast<const unsigned short*>(codes) + value_at(a, place, head, a.blocks, 0);
        c = v[2 * at] | (unsigned)v[2 * next] << 16;
      } else {
        c = codes[record * (4 * a.blocks) + at];
      }
      const unsigned word = scales[record * a.groups];
      const float step = __uint_as_float(word & 0xffff0000u), low = __uint_as_float(word << 16);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = there ? fmaf(step, (float)(c >> (4 * e) & 15), low) : 0.f;
      store8<T>(out + (long long)tok * a.heads * a.head_dim, x, true);
    }
  }
}

void take_cache(Args& a, const pfk_cache4& c) {
  a.k = c.k;
  a.v = c.v;
  a.k_scales = c.k_scales;
  a.v_scales = c.v_scales;
  a.heads = (int)c.heads;
  a.head_dim = (int)c.head_dim;
  a.group = (int)c.group;
  a.blocks = cache4_width(c.head_dim) / 32;
  a.groups = cache4_groups(c.head_dim, c.group);
  a.by_page = FastDiv((unsigned)c.page_size);
  a.num_slots = c.num_pages * c.page_size;
  a.err = c.err;
}

template <typename T>
void launch_append(Args& a, cudaStream_t stream) {
  const int64_t sms = device_sm_count(current_device()), at_once = kWarps * (32 / lanes_of(a.blocks));
  // few tokens: a part of a token's heads each, a row for each lane; many:
  // what fills the device once, its 8 CTAs an SM
  const int64_t per = std::min<int64_t>(kTokens, ceil_div(a.tokens, 8 * sms));
  a.per_cta = (int)per;
  const int64_t ctas = ceil_div(a.tokens, per);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(std::max(a.heads, a.q_heads), at_once), 4 * sms / ctas, a.heads}));
  const size_t smem = (size_t)per * (a.rot / 2) * (sizeof(double2) + sizeof(float2));
  const dim3 grid((unsigned)ctas, (unsigned)a.split);
  auto launch = [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value;
    if (a.blocks == 2) launch_following<Args>(append_kernel<T, 2, WIDE>, grid, kThreads, smem, stream, a);
    else if (a.blocks == 3) launch_following<Args>(append_kernel<T, 3, WIDE>, grid, kThreads, smem, stream, a);
    else if (a.blocks == 4) launch_following<Args>(append_kernel<T, 4, WIDE>, grid, kThreads, smem, stream, a);
    else launch_following<Args>(append_kernel<T, 8, WIDE>, grid, kThreads, smem, stream, a);
  };
  a.wide ? launch(std::true_type()) : launch(std::false_type());
}

}  // namespace

void cache4_words(int64_t head_dim, int64_t group, int64_t* codes, int64_t* scales) {
  PFB_CHECK_ARG(codes && scales, "null argument");
  PFB_CHECK_ARG(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 256, "4-bit cache: head_dim must be a multiple of 8, at most 256");
  PFB_CHECK_ARG(group == 32 || group == 64 || group == 128, "4-bit cache: group must be 32, 64 or 128");
  *codes = cache4_width(head_dim) / 8;
  *scales = cache4_groups(head_dim, group);
}

void launch_cache4_append(const pfk_cache4_append_params& p, cudaStream_t stream) {
  check_cache4(p.cache);
  check_decode_dtype(p.dtype);
  PFB_CHECK_ARG(p.tokens >= 0 && p.tokens <= INT32_MAX - kTokens, "4-bit append: bad number of tokens");
  PFB_CHECK_ARG(p.q_heads >= 0 && p.q_heads <= 65536, "4-bit append: q_heads must be 0 to 65536");
  PFB_CHECK_ARG(!p.q == !p.q_out, "4-bit append: q and q_out go together");
  const pfk_rotary& r = p.rotary;
  PFB_CHECK_ARG(r.rotary_dim >= 0 && r.rotary_dim % 2 == 0 && r.rotary_dim <= p.cache.head_dim, "rotary_dim must be even and at most head_dim");
  PFB_CHECK_ARG(r.rotary_dim == 0 || r.inv_freq, "rotary: null inv_freq");
  PFB_CHECK_ARG(r.interleaved == 0 || r.interleaved == 1, "rotary: interleaved must be 0 or 1");
  if (p.tokens == 0) return;
  PFB_CHECK_ARG(p.k && p.v && p.slots, "4-bit append: null pointer");
  PFB_CHECK_ARG(!p.q || p.q != p.q_out || ((p.tokens == 1 || p.q_st == p.qo_st) && (p.q_heads <= 1 || p.q_sh == p.qo_sh)),
                "4-bit append: q_out shares q's memory with other strides");
  PFB_CHECK_ARG(r.rotary_dim == 0 || p.positions, "4-bit append: null positions");
  PFB_CHECK_ARG(p.k_st >= 0 && p.k_sh >= 0 && p.v_st >= 0 && p.v_sh >= 0 && p.q_st >= 0 && p.q_sh >= 0 && p.qo_st >= 0 && p.qo_sh >= 0,
                "4-bit append: negative stride");
  Args a = {};
  take_cache(a, p.cache);
  const int64_t es = p.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  const void* src[3] = {p.k, p.v, p.q};
  const int64_t st[3] = {p.k_st, p.v_st, p.q_st}, sh[3] = {p.k_sh, p.v_sh, p.q_sh};
  a.q_heads = p.q ? (int)p.q_heads : 0;
  a.wide = 1;
  for (int f = 0; f < 3; ++f) {
    a.src[f] = src[f];
    // an axis of length one is never stepped along: its stride says nothing about alignment
    a.st[f] = p.tokens > 1 ? st[f] : 0;
    a.sh[f] = (f == 2 ? a.q_heads : a.heads) > 1 ? sh[f] : 0;
    if (f < 2 || a.q_heads) a.wide = a.wide && (uintptr_t)src[f] % 16 == 0 && a.st[f] * es % 16 == 0 && a.sh[f] * es % 16 == 0;
  }
  a.q_out = p.q_out;
  a.qo_st = p.tokens > 1 ? p.qo_st : 0;
  a.qo_sh = a.q_heads > 1 ? p.qo_sh : 0;
  if (a.q_heads) a.wide = a.wide && (uintptr_t)p.q_out % 16 == 0 && a.qo_st * es % 16 == 0 && a.qo_sh * es % 16 == 0;
  a.tokens = (int)p.tokens;
  a.slots = p.slots;
  a.positions = p.positions;
  a.inv_freq = r.inv_freq;
  a.rot = (int)r.rotary_dim;
  a.interleaved = r.interleaved;
  a.factor = p.factor;
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_append<float>(a, stream);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_append<__half>(a, stream);
  else launch_append<__nv_bfloat16>(a, stream);
}

void launch_cache4_read(const pfk_cache4_read_params& p, cudaStream_t stream) {
  check_cache4(p.cache);
  check_decode_dtype(p.dtype);
  PFB_CHECK_ARG(p.tokens >= 0 && p.tokens <= INT32_MAX, "4-bit read: bad number of tokens");
  if (p.tokens == 0) return;
  PFB_CHECK_ARG(p.slots && p.k && p.v, "4-bit read: null pointer");
  PFB_CHECK_ARG((uintptr_t)p.k % 16 == 0 && (uintptr_t)p.v % 16 == 0, "4-bit read: k and v must be 16-byte aligned");
  Args a = {};
  take_cache(a, p.cache);
  a.tokens = (int)p.tokens;
  a.slots = p.slots;
  a.out[0] = p.k;
  a.out[1] = p.v;
  a.by_chunks = FastDiv((unsigned)(p.cache.head_dim / 8));
  const int64_t sms = device_sm_count(current_device());
  a.per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(kReadTokens, p.tokens / (8 * sms)));
  const int64_t ctas = ceil_div(p.tokens, a.per_cta);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(2 * p.cache.heads * (p.cache.head_dim / 8), kReadThreads), 4 * sms / ctas));
  const dim3 grid((unsigned)ctas, (unsigned)a.split);
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_following<Args>(read_kernel<float>, grid, kReadThreads, 0, stream, a);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_following<Args>(read_kernel<__half>, grid, kReadThreads, 0, stream, a);
  else launch_following<Args>(read_kernel<__nv_bfloat16>, grid, kReadThreads, 0, stream, a);
}

}  // namespace pfb
