// Eviction from a paged key/value cache by accumulated attention weight.
//
// Per (request, kv head): a context of at most `budget` positions stays as it
// is; of a longer one the first `sinks` and the last `recent` positions stay,
// and of those between the budget - sinks - recent with the largest sums (the
// lowest position among equal sums; a sum that is no number ranks last).  The
// kept rows move, in order of position, to the first slots of the request: in
// place, or in the pages of another table.
//
// evict_select_kernel finds the kept positions: the threshold is the k-th
// largest 32-bit key, found eight bits at a time from histograms; then one
// ordered pass writes the kept positions.  evict_move_kernel moves the rows.
// Both are bound by memory: the sums are read once from HBM and again from L2.
#include "paged_cache.cuh"

namespace fm {
namespace {

constexpr int EV_THREADS = 512;

struct EvictArgs {
  CacheRef c;
  const float* sums;
  long long s_rs, s_hs;
  int budget, sinks, recent;
  int* kept;        // [R][KH][budget]
  int* lengths;     // [R]
  float* out_sums;  // [R][KH][budget]
  const int* out_table;
  long long ot_stride;
  int out_cap;  // slots that a row of out_table covers
  int row_bytes;
  int* err;
};

// larger sum, larger key; -0 equals +0, and no number is below every number
__device__ __forceinline__ uint32_t sum_key(float v) {
  if (v != v) return 0u;
  const uint32_t b = v == 0.0f ? 0u : __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int wsum[2][EV_THREADS / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / a.c.KH, h = blockIdx.x % a.c.KH;
  const int len = cache_length(a.c, r, a.err, tid == 0 && h == 0);
  const int n = min(len, a.budget);
  if (h == 0 && tid == 0) a.lengths[r] = n;
  const float* sums = a.sums + (long long)r * a.s_rs + (long long)h * a.s_hs;
  int* kept = a.kept + (long long)blockIdx.x * a.budget;
  float* out = a.out_sums + (long long)blockIdx.x * a.budget;
  for (int i = n + tid; i < a.budget; i += EV_THREADS) {
    kept[i] = -1;
    out[i] = 0.0f;
  }
  if (len <= a.budget) {
    for (int i = tid; i < n; i += EV_THREADS) {
      kept[i] = i;
      out[i] = sums[i];
    }
    return;
  }
  const int lo = a.sinks, hi = len - a.recent;  // the positions that compete
  int need = a.budget - a.sinks - a.recent;     // and how many of them stay (fewer than there are)
  uint32_t prefix = 0, mask = 0;
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += EV_THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += EV_THREADS) {
        const uint32_t k = sum_key(sums[i]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = need, b = 255;
        while (b > 0 && hist[b] < left) left -= hist[b--];
        s_need = left;
        s_prefix = prefix | ((uint32_t)b << shift);
      }
      __syncthreads();
      need = s_need;
      prefix = s_prefix;
      mask |= 255u << shift;
    }
  }
  // prefix is the smallest kept key, and `need` of the positions that hold it stay
  int base_keep = 0, base_tie = 0;
  for (int i0 = 0; i0 < len; i0 += EV_THREADS) {
    const int i = i0 + tid;
    bool sure = false, tie = false;
    float v = 0.0f;
    if (i < len) {
      v = sums[i];
      sure = i < lo || i >= hi;
      if (!sure && need > 0) {
        const uint32_t k = sum_key(v);
        sure = k > prefix;
        tie = k == prefix;
      }
    }
    // ties before this position decide whether it stays, kept positions before it where it goes
    const unsigned below = (1u << lane) - 1u;
    const unsigned tb = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) wsum[0][warp] = __popc(tb);
    __syncthreads();
    int tbefore = base_tie, ttotal = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) {
      if (w < warp) tbefore += wsum[0][w];
      ttotal += wsum[0][w];
    }
    const bool stay = sure || (tie && tbefore + __popc(tb & below) < need);
    const unsigned kb = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) wsum[1][warp] = __popc(kb);
    __syncthreads();
    int kbefore = base_keep, ktotal = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) {
      if (w < warp) kbefore += wsum[1][w];
      ktotal += wsum[1][w];
    }
    if (stay) {
      const int at = kbefore + __popc(kb & below);
      if (at < a.budget) {
        kept[at] = i;
        out[at] = v;
      }
    }
    base_tie += ttotal;
    base_keep += ktotal;
    __syncthreads();
  }
}

// One CTA per (request, kv head, keys or values).  A row only moves down
// (kept[i] >= i), so in place the CTA reads a block of rows before it writes
// the slots of that block: no later block reads a slot below its own first.
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a) {
  const int part = blockIdx.x & 1, item = blockIdx.x >> 1;
  const int r = item / a.c.KH, h = item % a.c.KH;
  const int len = cache_length(a.c, r, a.err, false);
  const int n = min(len, a.budget);
  const bool in_place = a.out_table == nullptr;
  if (in_place && len <= a.budget) return;
  const int* kept = a.kept + (long long)item * a.budget;
  uint8_t* base = (part ? a.c.v + (long long)h * a.c.vhs : a.c.k + (long long)h * a.c.khs);
  const long long ps = part ? a.c.vps : a.c.kps, ts = part ? a.c.vts : a.c.kts;
  const int* src_table = a.c.table + (long long)r * a.c.tstride;
  const int* dst_table = in_place ? src_table : a.out_table + (long long)r * a.ot_stride;
  auto row_at = [&](const int* table, int i) -> uint8_t* {
    const int page = table[i / a.c.page];
    if (page < 0 || page >= a.c.num_pages) {
      record_error(a.err, DEV_BAD_INDEX);
      return nullptr;
    }
    return base + page * ps + (i % a.c.page) * ts;
  };
  const int per_row = a.row_bytes / 16, rows = 256 / per_row;
  const int slot = threadIdx.x / per_row, off = (threadIdx.x % per_row) * 16;
  constexpr int U = 4;
  for (int i0 = 0; i0 < n; i0 += rows * U) {
    uint4 v[U];
    uint8_t* to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * rows + slot;
      to[u] = nullptr;
      if (i >= n) continue;
      const int from = kept[i];
      if (from < 0 || from >= len || (in_place && from == i)) continue;
      const uint8_t* src = row_at(src_table, from);
      uint8_t* dst = i < a.out_cap || in_place ? row_at(dst_table, i) : nullptr;
      if (src == nullptr || dst == nullptr) continue;
      v[u] = *reinterpret_cast<const uint4*>(src + off);
      to[u] = dst + off;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] != nullptr) *reinterpret_cast<uint4*>(to[u]) = v[u];
    __syncthreads();
  }
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" fm_status fm_paged_evict(const fm_paged_cache* cache, const fm_evict* p, fm_stream stream) {
  EvictArgs a{};
  fm_status st = cache_ref(cache, "paged_evict", &a.c);
  if (st != FM_OK) return st;
  if (!p) return set_error(FM_ERR_INVALID, "paged_evict: null arguments");
  if (p->budget < 1 || p->sinks < 0 || p->recent < 0 || p->budget > 0x7ffffff0 || p->sinks > p->budget ||
      p->recent > p->budget - p->sinks)
    return set_error(FM_ERR_SHAPE, "paged_evict: sinks + recent must lie within the budget");
  if (cache->requests == 0) return FM_OK;
  if (!p->weight_sums || !p->kept || !p->lengths || !p->out_sums)
    return set_error(FM_ERR_INVALID, "paged_evict: null pointer");
  if (p->out_page_table && p->out_page_table_cols < (p->budget + cache->page_size - 1) / cache->page_size)
    return set_error(FM_ERR_SHAPE, "paged_evict: the new page table does not cover the budget");
  if (p->lengths == cache->lengths)
    return set_error(FM_ERR_INVALID, "paged_evict: the new lengths must not overwrite the old");
  if (p->out_page_table == cache->page_table)
    return set_error(FM_ERR_INVALID, "paged_evict: pass no new page table to evict in place");
  a.sums = p->weight_sums;
  a.s_rs = p->sums_request_stride;
  a.s_hs = p->sums_head_stride;
  a.budget = (int)p->budget;
  a.sinks = (int)p->sinks;
  a.recent = (int)p->recent;
  a.kept = p->kept;
  a.lengths = p->lengths;
  a.out_sums = p->out_sums;
  a.out_table = p->out_page_table;
  a.ot_stride = p->out_page_table_stride;
  a.out_cap = a.budget;
  a.row_bytes = (int)cache->head_dim * (cache->dtype == FM_DT_E4M3 ? 1 : 2);
  a.err = p->err;
  const int64_t items = cache->requests * cache->kv_heads;
  if (items > 0x3fffffff) return set_error(FM_ERR_SHAPE, "paged_evict: grid too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = launch_kernel(evict_select_kernel, dim3((unsigned)items), dim3(EV_THREADS), 0, s, false, a);
  if (st != FM_OK) return st;
  return launch_kernel(evict_move_kernel, dim3((unsigned)items * 2), dim3(256), 0, s, false, a);
}
