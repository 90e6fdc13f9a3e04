// rotary_append.cu — rotary positions, and appending new tokens to a paged
// key-value cache with the rotation applied on the way.
//
// Pair i of a head's first r values is turned by a = position * w_i:
//   (y1, y2) = (x1 cos a - x2 sin a, x1 sin a + x2 cos a),
// cosine and sine multiplied by a factor (1 unless the frequencies were
// rescaled).  The gradient is the same kernel with -a.  The angle is formed
// and reduced in 64 bits: at position 10^6 an angle in 32 bits is off by up
// to 0.03 radian.  What is left of it, in half-turns within [-1, 1], goes
// through sincospif, so cosines and sines are within 2 ulp at any position.
//
// The work is bound by memory: every value is read once and written once, in
// accesses of up to 16 bytes.  A CTA takes a few tokens, computes their r/2
// cosines and sines once into shared memory (they are shared by all heads),
// and its threads then turn pairs of chunks, the rows of q, k and v of a
// token in one list, so that one launch stores keys, values and queries.
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

constexpr int kThreads = 256;
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
  FastDiv by_items, by_heads, by_tokens, by_page;
  int all_heads = 0;
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

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
  T v[VEC];
};

// VEC: values of one access.  A row is `items` pairs of chunks: the first
// rot / (2 VEC) of them are pairs that turn together (chunks j and j + r/2
// values on, or 2j and 2j + 1), the rest are neighbouring chunks that are
// copied.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(Args a) {
  extern __shared__ float2 table[];  // [per_cta][rot / 2]
  __shared__ long long place[64];    // of a token's row in the cache; -1: skipped
  using C = Chunk<T, VEC>;
  begin();
  const long long first = (long long)blockIdx.x * a.per_cta;
  const int mine = (int)min((long long)a.per_cta, a.total - first);
  const int half = a.rot >> 1;

  for (int i = threadIdx.x; i < mine * half; i += kThreads) {
    const int tok = i / half, p = i - tok * half;
    const unsigned n = (unsigned)(first + tok);
    const unsigned b = a.by_tokens.div(n);
    const long long pos = a.positions[(long long)b * a.p_sb + (long long)(n - b * a.tokens) * a.p_st];
    const double turns = (double)pos * a.inv_freq[p] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    table[i] = make_float2(c * a.factor, (a.inverse ? -s : s) * a.factor);
  }
  if (a.slots) {
    for (int i = threadIdx.x; i < mine; i += kThreads) {
      const long long slot = a.slots[first + i];
      long long at = -1;
      if (slot >= a.num_slots) {
        if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
      } else if (slot >= 0) {
        const unsigned page = a.by_page.div((unsigned)slot);
        at = (long long)page * a.page_stride + (slot - (long long)page * a.by_page.d) * a.token_stride;
      }
      place[i] = at;
    }
  }
  __syncthreads();

  const int pairs = half / VEC;
  const int chunks = a.head_dim / VEC;
  const unsigned count = (unsigned)mine * a.all_heads * a.items;
  for (unsigned it = threadIdx.x; it < count; it += kThreads) {
    const unsigned row = a.by_items.div(it);
    const int j = (int)(it - row * a.items);
    const unsigned tok = a.by_heads.div(row);
    int h = (int)(row - tok * a.all_heads);
    int f = 0;
    while (h >= a.rows[f].heads) h -= a.rows[f++].heads;
    const Rows& r = a.rows[f];
    if (a.slots && place[tok] < 0) continue;
    const unsigned n = (unsigned)(first + tok);
    const unsigned b = a.by_tokens.div(n);
    const long long t = n - b * a.tokens;
    const T* src = (const T*)r.src + b * r.sb + t * r.st + h * r.sh;
    T* dst = (T*)r.dst + b * r.db + (r.paged ? place[tok] : t * r.dt) + h * r.dh;
    const bool turn = r.rotate && j < pairs;
    int c1, c2;  // the item's chunks
    if (turn) {
      c1 = a.interleaved ? 2 * j : j;
      c2 = a.interleaved ? 2 * j + 1 : j + pairs;
    } else {
      c1 = r.rotate ? 2 * pairs + 2 * (j - pairs) : 2 * j;
      c2 = c1 + 1;
      if (c1 >= chunks) continue;
    }
    const bool two = c2 < chunks;
    C x1 = *reinterpret_cast<const C*>(src + c1 * VEC), x2{};
    if (two) x2 = *reinterpret_cast<const C*>(src + c2 * VEC);
    if (turn) {
      const float2* cs = table + tok * half;
      if (a.interleaved && VEC > 1) {
        // pairs are neighbours: chunk c1 holds angles j*VEC ... , c2 the rest
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const float2 p = cs[j * VEC + e / 2], q = cs[j * VEC + VEC / 2 + e / 2];
          const float u1 = to_f(x1.v[e]), u2 = to_f(x1.v[(e + 1) % VEC]);
          const float w1 = to_f(x2.v[e]), w2 = to_f(x2.v[(e + 1) % VEC]);
          x1.v[e] = from_f<T>(fmaf(u1, p.x, -(u2 * p.y)));
          x1.v[(e + 1) % VEC] = from_f<T>(fmaf(u1, p.y, u2 * p.x));
          x2.v[e] = from_f<T>(fmaf(w1, q.x, -(w2 * q.y)));
          x2.v[(e + 1) % VEC] = from_f<T>(fmaf(w1, q.y, w2 * q.x));
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float2 p = cs[j * VEC + e];
          const float u1 = to_f(x1.v[e]), u2 = to_f(x2.v[e]);
          x1.v[e] = from_f<T>(fmaf(u1, p.x, -(u2 * p.y)));
          x2.v[e] = from_f<T>(fmaf(u1, p.y, u2 * p.x));
        }
      }
    }
    *reinterpret_cast<C*>(dst + c1 * VEC) = x1;
    if (two) *reinterpret_cast<C*>(dst + c2 * VEC) = x2;
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
  a.by_items = FastDiv((unsigned)a.items);
  a.by_heads = FastDiv((unsigned)a.all_heads);
  a.by_tokens = FastDiv((unsigned)a.tokens);
  // about four items a thread, as long as the table fits
  const int64_t per_token = (int64_t)a.all_heads * a.items;
  int64_t per = std::max<int64_t>(1, 4 * kThreads / per_token);
  per = std::min<int64_t>({per, 64, a.total});
  if (half) per = std::max<int64_t>(1, std::min<int64_t>(per, kTableMax / half));
  a.per_cta = (int)per;
  const size_t smem = (size_t)per * half * sizeof(float2);
  launch_following<Args>(rotary_kernel<T, VEC>, dim3((unsigned)ceil_div(a.total, per)), kThreads, smem, stream, a);
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
