// paged_attention.cu — attention of one new token per sequence over a paged
// key-value cache.
//
//   s_j = scale q.k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// Every key and value is read once: 2 * D values for 4 * D * G operations (G
// query heads share a key-value head), so memory bounds it as long as the
// products run on the tensor cores and the loads never pause.
//
// Work.  A unit is one sequence, one key-value head and 8 or 16 of its query
// heads; its keys are cut into tiles of 64.  The tiles of all units form one
// list, and each of a fixed number of CTAs (one wave) takes an equal run of
// it, whatever the sequences' lengths: lengths are device data, so the host
// could not balance them.  A CTA that has a whole unit writes its output; a
// unit that is shared leaves (m, sum, o) of each share in the workspace, and
// a second small kernel joins the shares in the order of the list, so that
// results do not depend on timing.
//
// Tile.  Each of a CTA's 4 warps takes 16 keys at a time, straight from
// global memory into the registers of mma.sync operands, without shared
// memory: S^T = K Q^T has the keys as its rows, and since the order of the
// summed axis is free as long as both operands agree, a lane's fragment of K
// is 16 consecutive bytes of two key rows.  O^T = V^T P^T has the values'
// axis as its rows: a lane loads 16 bytes of each of its 4 keys and pairs
// them with byte permutes.  P is turned from the first product's accumulator
// layout into the second's operand layout by movmatrix.  A group of 8 query
// heads fills the 8 columns of the instruction; tcgen05 would need 128 rows
// of one operand in shared memory for the same, and the products are far from
// being the limit.
//
// Types.  16-bit: Q, K, V enter exactly; P is split into a high and a low
// part, so its rounding (2^-16 and less) stays below that of the output. fp16
// P is scaled by 2^14 to keep small weights out of its subnormal range.
// fp32: both operands are split into tf32 high and low parts, three products
// (the dropped low-low term is below 2^-22 of the product).  Scores, maxima,
// sums and outputs are held in fp32.
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
constexpr int kTile = 16 * kWarps;  // keys
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
  // workspace: [0] tile count, then each unit's first tile, the shares'
  // maxima and sums [ctas][2][heads], and their outputs [ctas][2][heads][D]
  long long* starts;
  float* stats;
  float* parts;
  int ctas;
  int heads;  // of a full unit: min(group, unit_heads)
};

struct Span {
  int begin, end, tiles;  // seen keys, and the tiles that cover them
};

__device__ __forceinline__ Span span_of(const Args& a, int b) {
  long long n = a.seq_lens[b];
  if (n < 0 || n > a.most) {
    if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
    n = n < 0 ? 0 : a.most;
  }
  Span s;
  s.end = (int)n;
  s.begin = a.window > 0 && n > a.window ? (int)n - a.window : 0;
  s.tiles = n ? (s.end + kTile - 1) / kTile - s.begin / kTile : 0;
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

// DP: head_dim rounded up to the size that the registers are laid out for.
// NT: 8-column blocks of query heads.
template <typename T, int DP, int NT>
struct Layout {
  static constexpr int kVec = Traits<T>::kVec;
  static constexpr int kQ = DP / (4 * kVec);  // 16-byte chunks of a K row that a lane holds
  static constexpr int kV = DP / (8 * kVec);  // of a V row
  static constexpr int kPitch = DP + 4;
  static constexpr size_t q_bytes = (size_t)kQ * NT * 32 * 16 * (sizeof(T) == 4 ? 2 : 1);
  static constexpr size_t o_bytes = (size_t)kWarps * NT * 8 * kPitch * 4;
  static constexpr size_t m_bytes = (size_t)2 * kWarps * NT * 8 * 4;
  static constexpr size_t smem = q_bytes + o_bytes + m_bytes;
};

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kThreads) attend_kernel(const Args a) {
  using L = Layout<T, DP, NT>;
  using Tr = Traits<T>;
  constexpr int VEC = L::kVec;
  constexpr bool k32 = sizeof(T) == 4;
  extern __shared__ __align__(16) char smem[];
  uint4* qs = reinterpret_cast<uint4*>(smem);  // [split][nt][chunk][lane]
  float* os = reinterpret_cast<float*>(smem + L::q_bytes);
  float* ms = reinterpret_cast<float*>(smem + L::q_bytes + L::o_bytes);  // [warp][head] maxima, then sums
  float* ls = ms + kWarps * NT * 8;
  __shared__ long long scan[kWarps + 1];
  __shared__ int found_row;
  __shared__ long long found_before;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;");

  // the list of tiles: its length, and the row that holds this CTA's first
  const int per_row = a.kv_heads * a.chunks;
  long long total = 0;
  for (int b = tid; b < a.batch; b += kThreads) total += (long long)span_of(a, b).tiles * per_row;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
  if (lane == 0) scan[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += scan[w];
  if (blockIdx.x == 0 && tid == 0) a.starts[0] = total;
  const long long t0 = total * blockIdx.x / a.ctas, t1 = total * (blockIdx.x + 1) / a.ctas;
  if (t0 >= t1) return;
  long long before = 0;
  for (int base = 0;; base += kThreads) {
    __syncthreads();
    const int b = base + tid;
    const long long mine = b < a.batch ? (long long)span_of(a, b).tiles * per_row : 0;
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    long long start = before;
    for (int w = 0; w < warp; ++w) start += scan[w];
    start += sum - mine;
    if (mine > 0 && t0 >= start && t0 < start + mine) {
      found_row = b;
      found_before = start;
    }
    for (int w = 0; w < kWarps; ++w) before += scan[w];
    if (before > t0) break;  // total > t0: some block of rows gets there
  }
  __syncthreads();
  int row = found_row;
  Span sp = span_of(a, row);
  int unit = (int)((t0 - found_before) / sp.tiles);  // of the row
  int tile = (int)((t0 - found_before) - (long long)unit * sp.tiles);

  const float scale2 = a.scale * kLog2e;
  for (long long at = t0; at < t1;) {
    while (sp.tiles == 0) sp = span_of(a, ++row);
    const int count = (int)min((long long)(sp.tiles - tile), t1 - at);
    const int head = unit / a.chunks;
    const int first_q = head * a.group + (unit - head * a.chunks) * a.unit_heads;
    const int heads = min(a.unit_heads, (head + 1) * a.group - first_q);

    // Q in the order of the second operand's registers
    __syncthreads();  // the previous piece's reads of shared memory are over
    {
      const T* qp = (const T*)a.q + (long long)row * a.q_sb + (long long)first_q * a.q_sh;
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
          T x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = h < heads && d0 + e < a.head_dim ? qp[h * a.q_sh + d0 + e] : Tr::from(0.f);
          qs[i] = *reinterpret_cast<uint4*>(x);
        }
      }
    }
    __syncthreads();

    const char* kp = a.k + head * a.head_bytes;
    const char* vp = a.v + head * a.head_bytes;
    const int* table = a.table + (long long)row * a.table_stride;
    const int lo_key = sp.begin, hi_key = sp.end;
    const int first_key = (sp.begin / kTile + tile) * kTile + warp * 16;

    // place of one of a step's 16 keys (lane & 15) in the cache, in units
    auto place = [&](int step) -> unsigned {
      if (step >= count) return kNone;
      const int key = first_key + step * kTile + (lane & 15);
      if (key < lo_key || key >= hi_key) return kNone;
      const unsigned p = a.by_page.div((unsigned)key);
      const unsigned page = (unsigned)table[p];
      if (page >= a.num_pages) {
        if (a.err) *a.err = PFC_ERR_INVALID_ARGUMENT;
        return kNone;
      }
      return page * a.page_units + ((unsigned)key - p * a.by_page.d) * a.token_units;
    };
    uint4 kr[2][L::kQ], vr[4][L::kV];
    auto load_k = [&](unsigned where, bool (&seen)[2]) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const unsigned u = __shfl_sync(~0u, where, g + 8 * r);
        seen[r] = u != kNone;
        const char* p = kp + (unsigned long long)u * a.unit_bytes + t * 16;
#pragma unroll
        for (int c = 0; c < L::kQ; ++c) {
          kr[r][c] = make_uint4(0, 0, 0, 0);
          if (seen[r] && (c * 4 + t) * VEC < a.head_dim) kr[r][c] = load16(p + c * 64);
        }
      }
    };
    auto load_v = [&](unsigned where) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned u = __shfl_sync(~0u, where, 2 * t + (r & 1) + 8 * (r >> 1));
        const char* p = vp + (unsigned long long)u * a.unit_bytes + g * 16;
#pragma unroll
        for (int c = 0; c < L::kV; ++c) {
          vr[r][c] = make_uint4(0, 0, 0, 0);
          if (u != kNone && (c * 8 + g) * VEC < a.head_dim) vr[r][c] = load16(p + c * 128);
        }
      }
    };

    // per lane: query heads nt*8 + 2t and + 1
    float m[NT][2], l[NT][2], o[NT][L::kV][VEC / 2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int c = 0; c < L::kV; ++c)
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[nt][c][j][r] = 0.f;
    }
    bool seen[2];
    unsigned here = place(0);
    load_k(here, seen);
    load_v(here);
    unsigned next = place(1);
    for (int step = 0; step < count; ++step) {
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[nt][r] = 0.f;
#pragma unroll
        for (int c = 0; c < L::kQ; ++c) {
          const uint4 b = qs[(nt * L::kQ + c) * 32 + lane];
          if constexpr (k32) {
            const uint4 bl = qs[(NT * L::kQ + nt * L::kQ + c) * 32 + lane];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              unsigned h0, h1, h2, h3, l0, l1, l2, l3;
              split(__uint_as_float(word(kr[0][c], 2 * e)), h0, l0);
              split(__uint_as_float(word(kr[1][c], 2 * e)), h1, l1);
              split(__uint_as_float(word(kr[0][c], 2 * e + 1)), h2, l2);
              split(__uint_as_float(word(kr[1][c], 2 * e + 1)), h3, l3);
              mma_tf32(s[nt], l0, l1, l2, l3, word(b, 2 * e), word(b, 2 * e + 1));
              mma_tf32(s[nt], h0, h1, h2, h3, word(bl, 2 * e), word(bl, 2 * e + 1));
              mma_tf32(s[nt], h0, h1, h2, h3, word(b, 2 * e), word(b, 2 * e + 1));
            }
          } else {
            Tr::mma(s[nt], kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, b.x, b.y);
            Tr::mma(s[nt], kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, b.z, b.w);
          }
        }
      }
      const bool seen0 = seen[0], seen1 = seen[1];
      if (step + 1 < count) load_k(next, seen);

      unsigned pt[NT][4];  // P as the second operand: 16-bit hi, lo of keys 0-7 and 8-15; fp32 its four values
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = (r < 2 ? seen0 : seen1) ? s[nt][r] * scale2 : -INFINITY;
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
                mma_tf32(o[nt][c][j], l0, l1, l2, l3, bh[nt][0], bh[nt][1]);
                mma_tf32(o[nt][c][j], h0, h1, h2, h3, bl[nt][0], bl[nt][1]);
                mma_tf32(o[nt][c][j], h0, h1, h2, h3, bh[nt][0], bh[nt][1]);
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned a0 = __byte_perm(word(vr[0][c], j), word(vr[1][c], j), 0x5410);
            const unsigned a1 = __byte_perm(word(vr[0][c], j), word(vr[1][c], j), 0x7632);
            const unsigned a2 = __byte_perm(word(vr[2][c], j), word(vr[3][c], j), 0x5410);
            const unsigned a3 = __byte_perm(word(vr[2][c], j), word(vr[3][c], j), 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              Tr::mma(o[nt][c][j], a0, a1, a2, a3, pt[nt][1], pt[nt][3]);
              Tr::mma(o[nt][c][j], a0, a1, a2, a3, pt[nt][0], pt[nt][2]);
            }
          }
        }
      }
      if (step + 1 < count) {
        load_v(next);
        next = place(step + 2);
      }
    }

    // join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], off);
        if (g == 0) {
          ms[warp * NT * 8 + nt * 8 + 2 * t + i] = m[nt][i];
          ls[warp * NT * 8 + nt * 8 + 2 * t + i] = l[nt][i];
        }
#pragma unroll
        for (int c = 0; c < L::kV; ++c)
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j)
            *reinterpret_cast<float2*>(os + (size_t)(warp * NT * 8 + nt * 8 + 2 * t + i) * L::kPitch + (c * 8 + g) * VEC + 2 * j) =
                make_float2(o[nt][c][j][i], o[nt][c][j][i + 2]);
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
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ms[w * NT * 8 + h]);
      float v = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = ms[w * NT * 8 + h];
        const float f = mw == -INFINITY ? (top == -INFINITY ? 1.f : 0.f) : exp2_fast(mw - top);
        v += f * os[(size_t)(w * NT * 8 + h) * L::kPitch + d];
        sum += f * ls[w * NT * 8 + h];
      }
      if (whole) {
        ((T*)a.out)[(long long)row * a.o_sb + (first_q + h) * a.o_sh + d] = Tr::from(sum == 0.f ? 0.f : v / sum);
        if (d == 0 && a.lse)
          a.lse[(long long)row * a.q_heads + first_q + h] = sum == 0.f ? -INFINITY : (top + log2f(sum) - Tr::kShift) * kLn2;
      } else {
        a.parts[(share + h) * a.head_dim + d] = v;
        if (d == 0) {
          a.stats[2 * (share + h)] = top;
          a.stats[2 * (share + h) + 1] = sum;
        }
      }
    }
    if (tile == 0 && tid == 0) a.starts[1 + (long long)row * per_row + unit] = at;
    at += count;
    tile = 0;
    if (++unit == per_row) {
      unit = 0;
      sp.tiles = 0;
      if (at < t1) sp = span_of(a, ++row);
    }
  }
}

// One CTA per sequence and query head: joins the shares of a unit that
// several CTAs had, in the order of the list; writes empty sequences.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(const Args a) {
  using Tr = Traits<T>;
  __shared__ float tops[kWarps], sums[kWarps];
  __shared__ float acc[kWarps][256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.q_heads, qh = blockIdx.x % a.q_heads;
  T* out = (T*)a.out + (long long)b * a.o_sb + (long long)qh * a.o_sh;
  const Span sp = span_of(a, b);
  if (sp.tiles == 0) {
    for (int d = tid; d < a.head_dim; d += kThreads) out[d] = Tr::from(0.f);
    if (tid == 0 && a.lse) a.lse[(long long)b * a.q_heads + qh] = -INFINITY;
    return;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int head = qh / a.group, in_group = qh - head * a.group;
  const int unit = head * a.chunks + in_group / a.unit_heads, h = in_group % a.unit_heads;
  const long long total = a.starts[0];
  const long long first = a.starts[1 + (long long)b * a.kv_heads * a.chunks + unit];
  const long long last = first + sp.tiles - 1;
  // the CTA that has tile x: the largest c with floor(total * c / ctas) <= x
  const int c0 = (int)(((first + 1) * a.ctas + total - 1) / total) - 1;
  const int c1 = (int)(((last + 1) * a.ctas + total - 1) / total) - 1;
  if (c0 == c1) return;  // written whole
  auto share_of = [&](int c) -> long long {
    const long long t0 = total * c / a.ctas, t1 = total * (c + 1) / a.ctas;
    return t0 == t1 ? -1 : ((long long)c * 2 + (t0 <= first ? 1 : 0)) * a.heads + h;
  };
  float top = -INFINITY;
  for (int c = c0 + tid; c <= c1; c += kThreads) {
    const long long s = share_of(c);
    if (s >= 0) top = fmaxf(top, a.stats[2 * s]);
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, off));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, tops[w]);
  float sum = 0.f, v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  for (int c = c0 + warp; c <= c1; c += kWarps) {
    const long long s = share_of(c);
    if (s < 0) continue;
    const float mc = a.stats[2 * s];
    const float f = mc == -INFINITY ? (top == -INFINITY ? 1.f : 0.f) : exp2_fast(mc - top);
    sum += f * a.stats[2 * s + 1];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < a.head_dim) v[e] += f * a.parts[s * a.head_dim + lane + 32 * e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[warp][lane + 32 * e] = v[e];
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += sums[w];
  for (int d = tid; d < a.head_dim; d += kThreads) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += acc[w][d];
    out[d] = Tr::from(sum == 0.f ? 0.f : x / sum);
  }
  if (tid == 0 && a.lse) a.lse[(long long)b * a.q_heads + qh] = sum == 0.f ? -INFINITY : (top + log2f(sum) - Tr::kShift) * kLn2;
}

// CTAs of one wave of a kernel on the current device, asked once per device.
template <typename T, int DP, int NT>
int wave() {
  static std::once_flag once[64];
  static int ctas[64];
  const int dev = current_device();
  std::call_once(once[dev], [dev] {
    using L = Layout<T, DP, NT>;
    PFB_CUDA(cudaFuncSetAttribute(attend_kernel<T, DP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem));
    int per = 0;
    PFB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, attend_kernel<T, DP, NT>, kThreads, L::smem));
    ctas[dev] = std::max(1, per) * device_sm_count(dev);
  });
  return ctas[dev];
}

template <typename T, int DP, int NT>
void launch_sized(Args& a, cudaStream_t stream) {
  attend_kernel<T, DP, NT><<<(unsigned)a.ctas, kThreads, Layout<T, DP, NT>::smem, stream>>>(a);
  PFB_CUDA(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.batch * a.q_heads));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PFB_CUDA(cudaLaunchKernelEx(&cfg, join_kernel<T>, (const Args&)a));
}

template <typename T_, int DP_, int NT_>
struct Kernel {
  using T = T_;
  static constexpr int DP = DP_, NT = NT_;
};

// Query heads of a unit: two column blocks hold 16, but their accumulators
// fit the registers only with 16-bit types and head_dim up to 128.
int unit_heads(const pfk_paged_attention_params& p) {
  return p.q_heads / p.cache.heads > 8 && p.cache.dtype != PFC_DTYPE_FLOAT32 && p.cache.head_dim <= 128 ? 16 : 8;
}

// Calls f(Kernel<T, DP, NT>()) for the call's type and sizes.
template <class F>
void dispatch(const pfk_paged_attention_params& p, F&& f) {
  const bool wide = unit_heads(p) == 16;
  const int64_t d = p.cache.head_dim;
  switch (p.cache.dtype) {
    case PFC_DTYPE_FLOAT32:
      if (d <= 64) f(Kernel<float, 64, 1>());
      else if (d <= 128) f(Kernel<float, 128, 1>());
      else f(Kernel<float, 256, 1>());
      break;
    case PFC_DTYPE_FLOAT16:
      if (d <= 64) wide ? f(Kernel<__half, 64, 2>()) : f(Kernel<__half, 64, 1>());
      else if (d <= 128) wide ? f(Kernel<__half, 128, 2>()) : f(Kernel<__half, 128, 1>());
      else f(Kernel<__half, 256, 1>());
      break;
    default:
      if (d <= 64) wide ? f(Kernel<__nv_bfloat16, 64, 2>()) : f(Kernel<__nv_bfloat16, 64, 1>());
      else if (d <= 128) wide ? f(Kernel<__nv_bfloat16, 128, 2>()) : f(Kernel<__nv_bfloat16, 128, 1>());
      else f(Kernel<__nv_bfloat16, 256, 1>());
  }
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

struct Plan {
  int ctas, heads;
  int64_t units, stats_at, parts_at, bytes;
};

Plan plan_of(const pfk_paged_attention_params& p) {
  Plan w;
  const int64_t group = p.q_heads / p.cache.heads;
  const int most = unit_heads(p);
  w.heads = (int)std::min<int64_t>(group, most);
  dispatch(p, [&](auto k) { w.ctas = wave<typename decltype(k)::T, decltype(k)::DP, decltype(k)::NT>(); });
  w.units = p.batch * p.cache.heads * ceil_div(group, most);
  w.stats_at = round_up((1 + w.units) * 8, 16);
  w.parts_at = round_up(w.stats_at + (int64_t)w.ctas * 2 * w.heads * 2 * 4, 16);
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
  const pfk_paged_cache& c = p.cache;
  const int64_t es = c.dtype == PFC_DTYPE_FLOAT32 ? 4 : 2;
  Args a = {};
  // places in the cache fit 32 bits in units of the strides' common divisor
  const int64_t page_bytes = c.num_pages > 1 ? c.page_stride * es : 0, token_bytes = c.page_size > 1 ? c.token_stride * es : 0;
  const int64_t unit = std::max<int64_t>(16, gcd(page_bytes, token_bytes));
  const int64_t span = (c.num_pages - 1) * (page_bytes / unit) + (c.page_size - 1) * (token_bytes / unit);
  PFB_CHECK_ARG(span < 0xffffffffll, "paged attention: the cache spans more than 2^32 - 1 of its strides' common divisor");
  const Plan w = plan_of(p);
  PFB_CHECK_ARG(p.workspace && p.workspace_bytes >= (size_t)w.bytes && (uintptr_t)p.workspace % 16 == 0,
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
  a.most = std::min<int64_t>(p.table_width * c.page_size, INT32_MAX - kTile);
  a.window = (int)std::min<int64_t>(p.window, INT32_MAX);
  a.scale = p.scale;
  char* ws = (char*)p.workspace;
  a.starts = (long long*)ws;
  a.stats = (float*)(ws + w.stats_at);
  a.parts = (float*)(ws + w.parts_at);
  a.ctas = w.ctas;
  a.heads = w.heads;
  dispatch(p, [&](auto k) { launch_sized<typename decltype(k)::T, decltype(k)::DP, decltype(k)::NT>(a, stream); });
}

}  // namespace pfb
