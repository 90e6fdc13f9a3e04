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
// A row (a head of a token) takes a lane for 8 of its values: minima and
// maxima meet by shuffles, and a lane's 8 codes are a word of a key row or two
// halves of value words.  Memory is the bound: k, v and q are read once, codes
// and q written once.
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
constexpr int kTokens = 16;  // a CTA takes at most

struct Args {
  uint32_t *k, *v, *k_scales, *v_scales;
  int heads, head_dim, group, blocks, groups;  // blocks of 32 values, words of a record's scales
  FastDiv by_page;
  long long num_slots;
  int* err;
  const void* src[3];  // k, v, q
  long long st[3], sh[3];
  int wide[3];  // rows may be read (and q written) 16 bytes at a time
  void* q_out;
  long long qo_st, qo_sh;
  int q_heads;
  int tokens, per_cta, split;
  const int64_t* slots;
  const int64_t* positions;
  const double* inv_freq;
  int rot, interleaved;
  float factor;
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
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.raw[i] = reinterpret_cast<const uint4*>(p)[i];
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
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = e.raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e.v[i];
  }
}

// Cosine and sine of pos * w in 64 bits.  pos * w is a + b exactly, 2 / pi is
// kHigh + kLow, and the quarter turns n + r, |r| <= 1/2, come from their
// products, rounded only after n is subtracted.
__device__ __forceinline__ double2 cos_sin(long long pos, double w) {
  constexpr double kHigh = 0x1.45f306dc9c883p-1, kLow = -0x1.6b01ec5417056p-55;
  const double p = (double)pos, a = p * w, b = fma(p, w, -a);
  const double n = rint(a * kHigh);
  const double r = fma(a, kHigh, -n) + fma(b, kHigh, a * kLow);
  double s, c;
  sincospi(0.5 * r, &s, &c);
  const int quarter = (int)((long long)n & 3);
  if (quarter & 1) {
    const double t = c;
    c = -s;
    s = t;
  }
  return quarter & 2 ? make_double2(-c, -s) : make_double2(c, s);
}

// LANES a row: head_dim / 8, rounded up to a power of two
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) append_kernel(Args a) {
  extern __shared__ double2 turns[];  // [per_cta][rot / 2], then the same as float2
  __shared__ long long places[kTokens];  // slot, -1 for a token that is skipped
  constexpr int ROWS = 32 / LANES;       // of a warp at a time
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int half = a.rot >> 1;
  begin();
  const int first = blockIdx.x * a.per_cta, mine = min(a.per_cta, a.tokens - first);
  float2* turns32 = reinterpret_cast<float2*>(turns + a.per_cta * half);
  for (int i = tid; i < mine * half; i += kThreads) {
    const int tok = i / half, p = i - tok * half;
    double2 cs = cos_sin(a.positions[first + tok], a.inv_freq[p]);
    cs.x *= a.factor;
    cs.y *= a.factor;
    turns[i] = cs;
    turns32[i] = make_float2((float)cs.x, (float)cs.y);
  }
  for (int tok = tid; tok < mine; tok += kThreads) {
    const long long slot = a.slots[first + tok];
    if (slot >= a.num_slots && a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
    places[tok] = slot < a.num_slots ? slot : -1;
  }
  __syncthreads();

  const int all = 2 * a.heads + a.q_heads;
  const int row_first = (int)((long long)all * blockIdx.y / a.split), rows = (int)((long long)all * (blockIdx.y + 1) / a.split) - row_first;
  const int chunk = lane % LANES;
  const bool in_head = chunk * 8 < a.head_dim;
  const int lanes_of_group = min(a.group / 8, LANES);
  for (int i0 = warp * ROWS; i0 < mine * rows; i0 += kWarps * ROWS) {
    const int i = i0 + lane / LANES;
    const int tok = i < mine * rows ? i / rows : 0, row = row_first + i - tok * rows;
    const long long slot = i < mine * rows ? places[tok] : -1;
    const int family = row < a.heads ? 0 : row < 2 * a.heads ? 1 : 2;
    const int head = family == 0 ? row : family == 1 ? row - a.heads : row - 2 * a.heads;
    const bool live = slot >= 0 && in_head;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
      const T* src = (const T*)a.src[family] + (long long)(first + tok) * a.st[family] + head * a.sh[family];
      load8<T>(x, src + chunk * 8, a.wide[family]);
      const int d0 = chunk * 8;
      if (family != 1 && d0 < a.rot) {
        float y[8];  // the values that turn with them
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
        } else if (half % 8 == 0) {
          load8<T>(y, src + (d0 < half ? d0 + half : d0 - half), a.wide[family]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = d0 + e;
            y[e] = d < half ? as_float<T>(src[d + half]) : d < a.rot ? as_float<T>(src[d - half]) : 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = d0 + e;
          if (d >= a.rot) continue;
          const bool second = a.interleaved ? (d & 1) : d >= half;
          const int at = tok * half + (a.interleaved ? d >> 1 : second ? d - half : d);
          if (family == 0) {
            const double2 cs = turns[at];
            x[e] = (float)fma((double)x[e], cs.x, second ? (double)y[e] * cs.y : -((double)y[e] * cs.y));
          } else {
            const float2 cs = turns32[at];
            x[e] = fmaf(x[e], cs.x, second ? y[e] * cs.y : -(y[e] * cs.y));
          }
        }
      }
    }
    __syncwarp();  // q_out may be q: the row is read before any of it is written
    if (family == 2 && live) {
      T* to = (T*)a.q_out + (long long)(first + tok) * a.qo_st + head * a.qo_sh + chunk * 8;
      store8<T>(to, x, a.wide[2]);
    }
    float least = INFINITY, most = -INFINITY;
    int bad = 0;
    if (in_head) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        least = fminf(least, x[e]);
        most = fmaxf(most, x[e]);
        bad |= !(fabsf(x[e]) <= 0x1p126f);
      }
    }
    for (int o = 1; o < lanes_of_group; o <<= 1) {
      least = fminf(least, __shfl_xor_sync(~0u, least, o));
      most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
      bad |= __shfl_xor_sync(~0u, bad, o);
    }
    if (slot < 0 || family == 2 || chunk >= 4 * a.blocks) continue;
    // (a group behind the head's end is kept as zeros)
    const float low = __bfloat162float(__float2bfloat16_rn(chunk / lanes_of_group * lanes_of_group * 8 < a.head_dim ? least : 0.f));
    float step = __bfloat162float(__float2bfloat16_rn((most - low) * (1.f / 15.f)));
    if (!(step >= 0x1p-126f)) step = 0.f;
    const float times = step > 0.f ? 1.f / step : 0.f;
    unsigned codes = 0;
    if (in_head && !bad) {
#pragma unroll
      for (int e = 0; e < 8; ++e) codes |= (unsigned)fminf(fmaxf(rintf((x[e] - low) * times), 0.f), 15.f) << (4 * e);
    }
    const unsigned page = a.by_page.div((unsigned)slot);
    const long long record = ((long long)page * a.heads + head) * a.by_page.d + (slot - (long long)page * a.by_page.d);
    if (family == 0) {
      a.k[record * (4 * a.blocks) + cache4_key_word(chunk, a.blocks)] = codes;
    } else {
      unsigned short* v = reinterpret_cast<unsigned short*>(a.v + record * (4 * a.blocks));
      v[cache4_value_half(2 * chunk, a.blocks)] = (unsigned short)codes;
      v[cache4_value_half(2 * chunk + 1, a.blocks)] = (unsigned short)(codes >> 16);
    }
    if (chunk % lanes_of_group == 0) {
      const unsigned word = bad ? 0x7fc07fc0u : (__float_as_uint(step) & 0xffff0000u) | __float_as_uint(low) >> 16;
      (family == 0 ? a.k_scales : a.v_scales)[record * a.groups + chunk / lanes_of_group] = word;
    }
  }
}

// A thread for 8 values of a head, keys and then values.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(Args a) {
  begin();
  const int chunks = a.head_dim / 8;
  const long long each = (long long)a.tokens * a.heads * chunks;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < 2 * each; i += gridDim.x * 256ll) {
    const bool value = i >= each;
    const long long j = value ? i - each : i;
    const int chunk = (int)(j % chunks);
    const long long row = j / chunks, tok = row / a.heads;
    const int head = (int)(row - tok * a.heads);
    const long long slot = a.slots[tok];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= a.num_slots) {
      if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
    } else if (slot >= 0) {
      const unsigned page = a.by_page.div((unsigned)slot);
      const long long record = ((long long)page * a.heads + head) * a.by_page.d + (slot - (long long)page * a.by_page.d);
      unsigned codes;
      if (value) {
        const unsigned short* v = reinterpret_cast<const unsigned short*>(a.v + record * (4 * a.blocks));
        codes = v[cache4_value_half(2 * chunk, a.blocks)] | (unsigned)v[cache4_value_half(2 * chunk + 1, a.blocks)] << 16;
      } else {
        codes = a.k[record * (4 * a.blocks) + cache4_key_word(chunk, a.blocks)];
      }
      const unsigned word = (value ? a.v_scales : a.k_scales)[record * a.groups + chunk * 8 / a.group];
      const float step = __uint_as_float(word & 0xffff0000u), low = __uint_as_float(word << 16);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fmaf(step, (float)(codes >> (4 * e) & 15), low);
    }
    store8<T>((T*)a.out[value] + j * 8, x, true);
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
  const int lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32;
  const int64_t rows = 2ll * a.heads + a.q_heads, sms = device_sm_count(current_device());
  // a token or more for a CTA, about four rows for each of its lanes, as long
  // as the device is filled; with few tokens several CTAs share one
  const int64_t at_once = kWarps * (32 / lanes);
  int64_t per = std::max<int64_t>(1, std::min<int64_t>({4 * at_once / rows, a.tokens / (8 * sms), kTokens}));
  a.per_cta = (int)per;
  const int64_t ctas = ceil_div(a.tokens, per);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, at_once), 4 * sms / ctas));
  const size_t smem = (size_t)per * (a.rot / 2) * (sizeof(double2) + sizeof(float2));
  const dim3 grid((unsigned)ctas, (unsigned)a.split);
  if (lanes == 8) launch_following<Args>(append_kernel<T, 8>, grid, kThreads, smem, stream, a);
  else if (lanes == 16) launch_following<Args>(append_kernel<T, 16>, grid, kThreads, smem, stream, a);
  else launch_following<Args>(append_kernel<T, 32>, grid, kThreads, smem, stream, a);
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
  for (int f = 0; f < 3; ++f) {
    a.src[f] = src[f];
    // an axis of length one is never stepped along: its stride says nothing about alignment
    a.st[f] = p.tokens > 1 ? st[f] : 0;
    a.sh[f] = (f == 2 ? a.q_heads : a.heads) > 1 ? sh[f] : 0;
    a.wide[f] = (uintptr_t)src[f] % 16 == 0 && a.st[f] * es % 16 == 0 && a.sh[f] * es % 16 == 0;
  }
  a.q_out = p.q_out;
  a.qo_st = p.tokens > 1 ? p.qo_st : 0;
  a.qo_sh = a.q_heads > 1 ? p.qo_sh : 0;
  a.wide[2] = a.wide[2] && (uintptr_t)p.q_out % 16 == 0 && a.qo_st * es % 16 == 0 && a.qo_sh * es % 16 == 0;
  a.tokens = (int)p.tokens;
  a.slots = p.slots;
  a.positions = p.positions;
  a.inv_freq = r.inv_freq;
  a.rot = (int)r.rotary_dim;
  a.interleaved = r.interleaved;
  a.factor = r.factor;
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
  const int64_t work = 2 * p.tokens * p.cache.heads * (p.cache.head_dim / 8);
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(work, 256), 1 << 20));
  if (p.dtype == PFC_DTYPE_FLOAT32) launch_following<Args>(read_kernel<float>, grid, 256, 0, stream, a);
  else if (p.dtype == PFC_DTYPE_FLOAT16) launch_following<Args>(read_kernel<__half>, grid, 256, 0, stream, a);
  else launch_following<Args>(read_kernel<__nv_bfloat16>, grid, 256, 0, stream, a);
}

}  // namespace pfb
