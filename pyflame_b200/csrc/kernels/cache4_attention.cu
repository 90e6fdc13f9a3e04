// cache4_attention.cu — attention of one new token per sequence over a paged
// key-value cache held in 4 bits: checks, plans and launches of the kernels of
// cache4_attention.cuh.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "cache4_attention.cuh"

namespace pfb {
namespace {

using cache4::Args;
using cache4::kHeads;
using cache4::kMostRanks;

// Calls f with a value of the call's type.
template <class F>
auto typed(int dtype, F&& f) {
  if (dtype == PFC_DTYPE_FLOAT16) return f(__half());
  if (dtype == PFC_DTYPE_BFLOAT16) return f(__nv_bfloat16());
  return f(float());
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

constexpr int64_t kClusterTiles = 64;  // of 64 keys: the longest sequences that clusters take

struct Plan {
  int ctas, heads;
  bool runs;    // pages of whole runs of 16 tokens
  bool beside;  // units whose heads fill at most half of an instruction
  int ranks;  // CTAs of a unit's cluster; 0: runs of the list of all tiles
  int64_t stats_at, parts_at, bytes;
};

Plan plan_of(const pfk_cache4_attention_params& p) {
  Plan w;
  const int64_t group = p.q_heads / p.cache.heads;
  w.heads = (int)std::min<int64_t>(group, kHeads);
  w.runs = p.cache.page_size % 16 == 0;
  w.beside = w.heads <= kHeads / 2;
  w.ctas = typed(p.dtype, [&](auto t) { return cache4::wave_of<decltype(t)>(cache4_width(p.cache.head_dim), p.cache.group, w.runs, w.beside); });
  int64_t seen = std::min<int64_t>(p.table_width * p.cache.page_size, INT32_MAX);
  if (p.window) seen = std::min<int64_t>(seen, std::min<int64_t>(p.window, INT32_MAX) + 64);
  const int64_t units = p.batch * p.cache.heads * ceil_div(group, kHeads), tiles = ceil_div(seen, 64);
  w.ranks = 0;
  w.stats_at = w.parts_at = w.bytes = 0;
  // Few units with tables for short sequences: a cluster takes each, with no
  // list, no workspace and no second launch.
  int ranks = 1;
  while (ranks < kMostRanks && ranks < tiles) ranks *= 2;
  if (tiles <= kClusterTiles && units * ranks <= 2 * device_sm_count(current_device())) {
    w.ranks = ranks;
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
  a.head_pairs = (unsigned)((c.page_size + 1) / 2);
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
  typed(p.dtype, [&](auto t) { cache4::launch_of<decltype(t)>(a, cache4_width(c.head_dim), c.group, w.runs, w.beside, w.ranks, stream); });
}

}  // namespace pfb
