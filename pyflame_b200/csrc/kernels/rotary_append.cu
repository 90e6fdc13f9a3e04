// rotary_append.cu — rotary positions, and appending new tokens to a paged
// key-value cache with the rotation applied on the way.
//
// Pair i of a head's first r values is turned by a = position * w_i:
//   (y1, y2) = (x1 cos a - x2 sin a, x1 sin a + x2 cos a),
// cosine and sine multiplied by a factor (1 unless the frequencies were
// rescaled).  The gradient is the same kernel with -a.  The angle is formed
// and reduced in two 64-bit numbers: at position 10^6 an angle in 32 bits is
// off by up to 0.03 radian, and the nearer a quarter turn's multiple, the more
// a single 64-bit number loses of the small sine or cosine there.  What is
// left, at most an eighth of a turn, goes through sincospif in fp32: cosines
// and sines, however small, are within 2 ulp of those of position * w_i at
// positions below 2^53.
//
// The work is bound by memory: every value is read once and written once, in
// accesses of up to 16 bytes that are marked as streaming (two prompts of
// 4096 tokens, 32 heads of 128 in bf16, 134 MB: 21.2 us, 6.3 TB/s, for 23.9
// without the marks).  A CTA takes a few tokens, computes their r/2 cosines
// and sines once into shared memory (they are shared by all heads), and its
// threads then turn pairs of chunks, the rows of q, k and v of a token in one
// list, so that one launch stores keys, values and queries (8191 tokens with
// 32 query and 8 key-value heads of 128 in fp16, 201 MB: 34.2 us, 5.9 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../common.hpp"
#include "decode.cuh"
#include "kernels.hpp"

namespace pfb {
namespace {

constexpr int kThreads = 128;
constexpr int kTokens = 64;     // a CTA takes at most
constexpr int kTableMax = 2048;  // cosine-sine pairs a CTA keeps (16 KB)

// One family of rows: `heads` rows a token, read at
// src + b*sb + t*st + h*sh, written at dst + b*db + (t*dt, or the slot's
// place in the cache) + h*dh.
struct Rows {
  const void* src = nullptr;
  void* dst = nullptr;
  long long sb = 0, st = 0, sh = 0, db = 0, dt = 0, dh = 0;
  int heads = 0;
  int rotate = 0;
  int paged = 0;
};

struct Args {
  Rows rows[3];
  int families = 0;
  int tokens = 0;              // of one batch entry
  long long total = 0;         // batch * tokens
  int per_cta = 1;             // tokens a CTA takes
  int head_dim = 0, rot = 0;   // values of a head, and how many are turned
  int items = 0;               // chunk pairs of a row
  FastDiv by_tokens, by_page;
  int all_heads = 0;
  int split = 1;  // CTAs that share a token's rows
  int interleaved = 0;
  int inverse = 0;
  float factor = 1.f;
  const double* inv_freq = nullptr;
  const int64_t* positions = nullptr;
  long long p_sb = 0, p_st = 0;
  const int64_t* slots = nullptr;
  long long num_slots = 0, page_stride = 0, token_stride = 0;
  int* err = nullptr;
};

// Cosine and sine of pos * w.  pos * w is a + b exactly (b the product's
// rounding error, by fma), 2 / pi is kHigh + kLow, and the quarter turns
// n + r, |r| <= 1/2, come from their products with the leading one, a * kHigh,
// rounded only after n is subtracted.
__device__ __forceinline__ float2 cos_sin(long long pos, double w) {
  constexpr double kHigh = 0x1.45f306dc9c883p-1, kLow = -0x1.6b01ec5417056p-55;
  const double p = (double)pos, a = p * w, b = fma(p, w, -a);
  const double n = rint(a * kHigh);
  const double r = fma(a, kHigh, -n) + fma(b, kHigh, a * kLow);
  float s, c;
  sincospif((float)(0.5 * r), &s, &c);
  const int quarter = (int)((long long)n & 3);
  if (quarter & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  return quarter & 2 ? make_float2(-c, -s) : make_float2(c, s);
}

__device__ __forceinline__ float2 turned(float u1, float u2, float2 cs) {
  return make_float2(fmaf(u1, cs.x, -(u2 * cs.y)), fmaf(u1, cs.y, u2 * cs.x));
}

// An access of VEC values as plain words: structs of __half or __nv_bfloat16
// are copied value by value.
template <int BYTES> struct Raw;
template <> struct Raw<16> { using R = uint4; };
template <> struct Raw<8> { using R = uint2; };
template <> struct Raw<4> { using R = unsigned; };
template <> struct Raw<2> { using R = unsigned short; };

// Two values of a chunk, e and e + 1, as floats, and back.
template <typename T>
struct Two;
template <>
struct Two<float> {
  static __device__ __forceinline__ float2 get(const unsigned* w, int e) { return make_float2(__uint_as_float(w[e]), __uint_as_float(w[e + 1])); }
  static __device__ __forceinline__ void put(unsigned* w, int e, float2 f) { w[e] = __float_as_uint(f.x), w[e + 1] = __float_as_uint(f.y); }
  static __device__ __forceinline__ float one(unsigned r) { return __uint_as_float(r); }
  static __device__ __forceinline__ unsigned one_of(float f) { return __float_as_uint(f); }
};
template <>
struct Two<__half> {
  static __device__ __forceinline__ float2 get(const unsigned* w, int e) {
    return __half22float2(*reinterpret_cast<const __half2*>(w + e / 2));
  }
  static __device__ __forceinline__ void put(unsigned* w, int e, float2 f) {
    const __half2 h = __float22half2_rn(f);
    w[e / 2] = *reinterpret_cast<const unsigned*>(&h);
  }
  static __device__ __forceinline__ float one(unsigned short r) { return __half2float(__ushort_as_half(r)); }
  static __device__ __forceinline__ unsigned short one_of(float f) { return __half_as_ushort(__float2half_rn(f)); }
};
template <>
struct Two<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(const unsigned* w, int e) {
    return make_float2(__uint_as_float(w[e / 2] << 16), __uint_as_float(w[e / 2] & 0xffff0000u));
  }
  static __device__ __forceinline__ void put(unsigned* w, int e, float2 f) {
    const __nv_bfloat162 h = __float22bfloat162_rn(f);
    w[e / 2] = *reinterpret_cast<const unsigned*>(&h);
  }
  static __device__ __forceinline__ float one(unsigned short r) { return __bfloat162float(__ushort_as_bfloat16(r)); }
  static __device__ __forceinline__ unsigned short one_of(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
};

// VEC: values of one access.  A row is `items` pairs of chunks: the first
// rot / (2 VEC) of them are pairs that turn together (chunks j and j + r/2
// values on, or 2j and 2j + 1), the rest are neighbouring chunks that are
// copied.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Args a) {
  extern __shared__ float2 table[];  // [per_cta][rot / 2]
  // of a token's rows in each family: where they are read (in elements), and
  // where they are written, -1 for a token that is skipped
  __shared__ long long from[3][kTokens], to[3][kTokens];
  using R = typename Raw<sizeof(T) * VEC>::R;
  using P = Two<T>;
  begin();
  const long long first = (long long)blockIdx.x * a.per_cta;
  const int mine = (int)min((long long)a.per_cta, a.total - first);
  const int half = a.rot >> 1;
  const int pairs = half / VEC;

  for (int i = threadIdx.x; i < mine * half; i += kThreads) {
    const int tok = i / half, p = i - tok * half;
    const unsigned n = (unsigned)(first + tok), b = a.by_tokens.div(n);
    const long long pos = a.positions[(long long)b * a.p_sb + (long long)(n - b * a.tokens) * a.p_st];
    const float2 cs = cos_sin(pos, a.inv_freq[p]);
    // angle j*VEC + e at [e][j]: neighbouring lanes, with neighbouring j, read neighbouring places
    table[tok * half + p % VEC * pairs + p / VEC] = make_float2(cs.x * a.factor, (a.inverse ? -cs.y : cs.y) * a.factor);
  }
  for (int tok = threadIdx.x; tok < mine; tok += kThreads) {
    const unsigned n = (unsigned)(first + tok), b = a.by_tokens.div(n);
    const long long t = n - b * a.tokens;
    long long place = 0;
    if (a.slots) {
      const long long slot = a.slots[n];
      place = -1;
      if (slot >= a.num_slots) {
        if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
      } else if (slot >= 0) {
        const unsigned page = a.by_page.div((unsigned)slot);
        place = (long long)page * a.page_stride + (slot - (long long)page * a.by_page.d) * a.token_stride;
      }
    }
    for (int f = 0; f < a.families; ++f) {
      const Rows& r = a.rows[f];
      from[f][tok] = b * r.sb + t * r.st;
      to[f][tok] = place < 0 ? -1 : r.paged ? place : b * r.db + t * r.dt;
    }
  }
  __syncthreads();

  // a thread keeps its place j in the rows and walks over them; rows wider
  // than the CTA take several passes
  const int chunks = a.head_dim / VEC;
  const int head_first = a.all_heads * blockIdx.y / a.split, head_last = a.all_heads * (blockIdx.y + 1) / a.split;
  const int wide = min(a.items, kThreads), stride = kThreads / wide;
  const int start = threadIdx.x / wide;
  if (start >= stride) return;
  for (int j = threadIdx.x - start * wide; j < a.items; j += wide) {
    int tok = 0, head = head_first + start;
    for (;; head += stride) {
      while (head >= head_last) {
        head -= head_last - head_first;
        ++tok;
      }
      if (tok >= mine) break;
      int h = head, f = 0;
      while (h >= a.rows[f].heads) h -= a.rows[f++].heads;
      const Rows& r = a.rows[f];
      const long long at = to[f][tok];
      if (at < 0) continue;
      const T* src = (const T*)r.src + from[f][tok] + h * r.sh;
      T* dst = (T*)r.dst + at + h * r.dh;
      const bool turn = r.rotate && j < pairs;
      int c1 = 2 * j, c2 = 2 * j + 1;  // the item's chunks; 2 * pairs is the first behind the turned ones
      if (turn && !a.interleaved) {
        c1 = j;
        c2 = j + pairs;
      }
      if (c1 >= chunks) continue;
      const bool two = c2 < chunks;
      R r1 = __ldcs(reinterpret_cast<const R*>(src + c1 * VEC)), r2{};
      if (two) r2 = __ldcs(reinterpret_cast<const R*>(src + c2 * VEC));
      if (turn) {
        const float2* cs = table + tok * half + j;
        if constexpr (VEC == 1) {
          const float2 y = turned(P::one(r1), P::one(r2), cs[0]);
          r1 = P::one_of(y.x);
          r2 = P::one_of(y.y);
        } else {
          unsigned* x1 = reinterpret_cast<unsigned*>(&r1);
          unsigned* x2 = reinterpret_cast<unsigned*>(&r2);
          if (a.interleaved) {  // chunk c1 holds the pairs of angles j*VEC ... , c2 those of the VEC/2 behind
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              const float2 u = P::get(x1, e), w = P::get(x2, e);
              P::put(x1, e, turned(u.x, u.y, cs[(e / 2) * pairs]));
              P::put(x2, e, turned(w.x, w.y, cs[(VEC / 2 + e / 2) * pairs]));
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              const float2 u = P::get(x1, e), w = P::get(x2, e);
              const float2 y = turned(u.x, w.x, cs[(e) * pairs]), z = turned(u.y, w.y, cs[(e + 1) * pairs]);
              P::put(x1, e, make_float2(y.x, z.x));
              P::put(x2, e, make_float2(y.y, z.y));
            }
          }
        }
      }
      __stcs(reinterpret_cast<R*>(dst + c1 * VEC), r1);
      if (two) __stcs(reinterpret_cast<R*>(dst + c2 * VEC), r2);
    }
  }
}

template <typename T, int VEC>
void launch_vec(Args& a, cudaStream_t stream) {
  const int half = a.rot / 2;
  const int copied = (int)ceil_div((a.head_dim - a.rot) / VEC, 2);
  a.items = half / VEC + copied;
  bool copies = false;
  for (int f = 0; f < a.families; ++f) copies |= !a.rows[f].rotate;
  if (copies) a.items = std::max(a.items, (int)ceil_div(a.head_dim / VEC, 2));
  a.by_tokens = FastDiv((unsigned)a.tokens);
  // about four items a thread, as long as the table fits (two: 22.5 us, eight:
  // 21.4, sixteen: 27 for the prompts' 21.2), fewer where that would leave
  // less than four CTAs an SM
  const int64_t per_token = (int64_t)a.all_heads * a.items;
  const int64_t filled = a.total / (4 * (int64_t)device_sm_count(current_device()));
  int64_t per = std::max<int64_t>(1, std::min<int64_t>(4 * kThreads / per_token, filled));
  per = std::min<int64_t>({per, kTokens, a.total});
  if (half) per = std::max<int64_t>(1, std::min<int64_t>(per, kTableMax / half));
  a.per_cta = (int)per;
  const size_t smem = (size_t)per * half * sizeof(float2);
  // with few tokens several CTAs share one's rows, an item a thread
  const int64_t sms = device_sm_count(current_device());
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(per_token, kThreads), 2 * sms / a.total, a.all_heads}));
  launch_following<Args>(rotary_kernel<T, VEC>, dim3((unsigned)ceil_div(a.total, per), (unsigned)a.split), kThreads, smem, stream, a);
}

// The widest access that every pointer, stride and boundary of the rows allows.
int widest(const Args& a, int64_t es) {
  for (int64_t vec = 16 / es; vec > 1; vec /= 2) {
    const int64_t bytes = vec * es;
    bool ok = (a.rot / 2) % vec == 0 && (a.head_dim - a.rot) % vec == 0 && a.head_dim % vec == 0;
    for (int f = 0; f < a.families && ok; ++f) {
      const Rows& r = a.rows[f];
      ok = (uintptr_t)r.src % bytes == 0 && (uintptr_t)r.dst % bytes == 0;
      for (long long s : {r.sb, r.st, r.sh, r.db, r.dt, r.dh}) ok = ok && s % vec == 0;
      if (r.paged) ok = ok && a.page_stride % vec == 0 && a.token_stride % vec == 0;
    }
    if (ok) return (int)vec;
  }
  return 1;
}

void launch(Args& a, int dtype, cudaStream_t stream) {
  a.all_heads = 0;
  for (int f = 0; f < a.families; ++f) {
    Rows& r = a.rows[f];
    a.all_heads += r.heads;
    // an axis of length one is never stepped along: its stride says nothing about alignment
    if (r.heads <= 1) r.sh = r.dh = 0;
    if (a.tokens <= 1) r.st = r.dt = 0;
    if (a.total <= a.tokens) r.sb = r.db = 0;
  }
  if (a.total == 0 || a.all_heads == 0 || a.head_dim == 0) return;
  const int vec = widest(a, dtype == PFC_DTYPE_FLOAT32 ? 4 : 2);
  if (dtype == PFC_DTYPE_FLOAT32) {
    if (vec == 4) launch_vec<float, 4>(a, stream);
    else if (vec == 2) launch_vec<float, 2>(a, stream);
    else launch_vec<float, 1>(a, stream);
  } else if (dtype == PFC_DTYPE_FLOAT16) {
    if (vec == 8) launch_vec<__half, 8>(a, stream);
    else if (vec == 4) launch_vec<__half, 4>(a, stream);
    else if (vec == 2) launch_vec<__half, 2>(a, stream);
    else launch_vec<__half, 1>(a, stream);
  } else {
    if (vec == 8) launch_vec<__nv_bfloat16, 8>(a, stream);
    else if (vec == 4) launch_vec<__nv_bfloat16, 4>(a, stream);
    else if (vec == 2) launch_vec<__nv_bfloat16, 2>(a, stream);
    else launch_vec<__nv_bfloat16, 1>(a, stream);
  }
}

void take_rotary(Args& a, const pfk_rotary& r, int64_t head_dim) {
  PFB_CHECK_ARG(r.rotary_dim >= 0 && r.rotary_dim % 2 == 0 && r.rotary_dim <= head_dim,
                "rotary_dim must be even and at most head_dim");
  PFB_CHECK_ARG(r.rotary_dim == 0 || r.inv_freq, "rotary: null inv_freq");
  PFB_CHECK_ARG(r.interleaved == 0 || r.interleaved == 1, "rotary: interleaved must be 0 or 1");
  a.rot = (int)r.rotary_dim;
  a.inv_freq = r.inv_freq;
  a.interleaved = r.interleaved;
  a.factor = r.factor;
}

}  // namespace

void launch_rope(const void* x, void* y, const pfk_rope_params& p, cudaStream_t stream) {
  check_decode_dtype(p.dtype);
  PFB_CHECK_ARG(p.batch >= 0 && p.tokens >= 0 && p.heads >= 0, "rope: negative size");
  PFB_CHECK_ARG(p.head_dim >= 1 && p.head_dim <= 1024, "rope: head_dim must be 1 to 1024");
  PFB_CHECK_ARG(p.heads <= 65536, "rope: more than 65536 heads");
  PFB_CHECK_ARG(p.batch <= INT32_MAX && p.tokens <= INT32_MAX && p.batch * p.tokens <= INT32_MAX,
                "rope: more than 2^31 - 1 tokens");
  PFB_CHECK_ARG(p.inverse == 0 || p.inverse == 1, "rope: inverse must be 0 or 1");
  Args a;
  take_rotary(a, p.rotary, p.head_dim);
  if (p.batch * p.tokens * p.heads == 0) return;
  PFB_CHECK_ARG(x && y, "rope: null pointer");
  // in place a row is read and written by the same threads
  PFB_CHECK_ARG(x != y || ((p.batch == 1 || p.x_sb == p.y_sb) && (p.tokens == 1 || p.x_st == p.y_st) && (p.heads == 1 || p.x_sh == p.y_sh)),
                "rope: y shares x's memory with other strides");
  PFB_CHECK_ARG(p.rotary.rotary_dim == 0 || p.positions, "rope: null positions");
  Rows& r = a.rows[0];
  r.src = x;
  r.dst = y;
  r.sb = p.x_sb; r.st = p.x_st; r.sh = p.x_sh;
  r.db = p.y_sb; r.dt = p.y_st; r.dh = p.y_sh;
  r.heads = (int)p.heads;
  r.rotate = 1;
  a.families = 1;
  a.tokens = (int)p.tokens;
  a.total = p.batch * p.tokens;
  a.head_dim = (int)p.head_dim;
  a.inverse = p.inverse;
  a.positions = p.positions;
  a.p_sb = p.p_sb;
  a.p_st = p.p_st;
  launch(a, p.dtype, stream);
}

void launch_paged_append(const pfk_paged_append_params& p, cudaStream_t stream) {
  check_paged_cache(p.cache);
  PFB_CHECK_ARG(p.cache.head_dim <= 1024, "paged append: head_dim above 1024");
  PFB_CHECK_ARG(p.tokens >= 0 && p.tokens <= INT32_MAX, "paged append: tokens must be 0 to 2^31 - 1");
  PFB_CHECK_ARG(p.q_heads >= 0 && p.q_heads <= 65536, "paged append: q_heads must be 0 to 65536");
  PFB_CHECK_ARG(!p.q == !p.q_out, "paged append: q and q_out go together");
  Args a;
  take_rotary(a, p.rotary, p.cache.head_dim);
  if (p.tokens == 0) return;
  PFB_CHECK_ARG(p.k && p.v && p.slots, "paged append: null pointer");
  PFB_CHECK_ARG(!p.q || p.q != p.q_out || ((p.tokens == 1 || p.q_st == p.qo_st) && (p.q_heads <= 1 || p.q_sh == p.qo_sh)),
                "paged append: q_out shares q's memory with other strides");
  PFB_CHECK_ARG(p.rotary.rotary_dim == 0 || p.positions, "paged append: null positions");
  Rows& k = a.rows[0];
  k.src = p.k;
  k.dst = p.cache.k;
  k.st = p.k_st; k.sh = p.k_sh; k.dh = p.cache.head_stride;
  k.heads = (int)p.cache.heads;
  k.rotate = 1;
  k.paged = 1;
  Rows& v = a.rows[1];
  v.src = p.v;
  v.dst = p.cache.v;
  v.st = p.v_st; v.sh = p.v_sh; v.dh = p.cache.head_stride;
  v.heads = (int)p.cache.heads;
  v.paged = 1;
  a.families = 2;
  if (p.q && p.q_heads) {
    Rows& q = a.rows[2];
    q.src = p.q;
    q.dst = p.q_out;
    q.st = p.q_st; q.sh = p.q_sh; q.dt = p.qo_st; q.dh = p.qo_sh;
    q.heads = (int)p.q_heads;
    q.rotate = 1;
    a.families = 3;
  }
  a.tokens = (int)p.tokens;
  a.total = p.tokens;
  a.head_dim = (int)p.cache.head_dim;
  a.positions = p.positions;
  a.p_st = 1;
  a.slots = p.slots;
  a.num_slots = p.cache.num_pages * p.cache.page_size;
  a.page_stride = p.cache.page_stride;
  a.token_stride = p.cache.token_stride;
  a.by_page = FastDiv((unsigned)p.cache.page_size);
  a.err = p.cache.err;
  launch(a, p.cache.dtype, stream);
}

}  // namespace pfb
