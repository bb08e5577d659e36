// Eviction from a paged key/value cache by accumulated attention weight.
//
// Per (request, kv head): a context of at most `budget` positions stays as it
// is; of a longer one the first `sinks` and the last `recent` positions stay,
// and of those between the budget - sinks - recent with the largest sums (the
// lowest position among equal sums; a sum that is no number ranks last).  The
// kept rows move, in order of position, to the first slots of the request: in
// place, or in the pages of another table.
//
// evict_select_kernel finds the kept positions: one cluster of CTAs per
// (request, kv head), each with a slice of the positions whose keys it holds in
// shared memory.  The smallest kept key is found 11, 11 and 10 bits at a time,
// or until a bin stays whole, from histograms that the cluster adds up; then an
// ordered count gives every kept position its slot.  The rows are moved by
// evict_move_kernel, or, where there are CTAs enough, by the CTA that chose
// them (64 requests, 8 kv heads, 2000 .. 8192 to 2048 positions: 201 us in two
// launches, 197 us in one, of which 166 us are the rows' bytes; 8 e4m3 contexts
// of 20000 .. 65000 copied to 8192: 82 and 81 us).  A few rows are bound by latency: one request of 4096
// to 2048, 16 us, half of it choosing, in rounds of counting and meeting.
#include <cooperative_groups.h>

#include "paged_cache.cuh"

namespace fm {
namespace {

namespace cg = cooperative_groups;

constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_KEYS = 49152;  // keys of a slice that shared memory holds; longer slices read theirs from L2 again
constexpr int EV_FUSE = 148;    // CTAs that choose from which on they move the rows, too
// Sums that a thread of the choosing kernel has in flight (8 contexts of 20000 .. 65000: 82.5 us, with 8 83.5 us)
constexpr int EV_LOADS = 16;
constexpr int EV_UNROLL = 4;    // rows that a thread of the moving kernel has in flight

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
  int2* from;       // [R][KH][budget] (page, token) of the kept rows
  int row_bytes, slices, chunk;
  int* err;
};

// larger sum, larger key; -0 equals +0, and no number is below every number
__device__ __forceinline__ uint32_t sum_key(float v) {
  if (v != v) return 0u;
  const uint32_t b = v == 0.0f ? 0u : __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Moves rows begin .. end - 1 of (r, h)'s keys or values, `slice` of their
// bytes, by 256 threads.  In place a row only moves down (kept[i] >= i): the
// CTA reads a block of rows, all its threads meet, and it writes them.  No later
// block reads a slot below its own first one, so one meeting a block is all
// that is needed.
template <bool IN_PLACE>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int r, int h, int part, int slice, int begin, int end,
                                          int tid) {
  const int bytes = a.row_bytes / a.slices, per_row = bytes / 16;
  const int rows = 256 / per_row, mine = tid / per_row;
  uint8_t* base = (part ? a.c.v + (long long)h * a.c.vhs : a.c.k + (long long)h * a.c.khs) + slice * bytes +
                  (tid % per_row) * 16;
  const long long ps = part ? a.c.vps : a.c.kps, ts = part ? a.c.vts : a.c.kts;
  const int2* from = a.from + ((long long)r * a.c.KH + h) * a.budget;
  const int* to = IN_PLACE ? a.c.table + (long long)r * a.c.tstride : a.out_table + (long long)r * a.ot_stride;
  int2 src[EV_UNROLL];
  int dst[EV_UNROLL];
  auto look = [&](int i0) {
#pragma unroll
    for (int u = 0; u < EV_UNROLL; ++u) {
      const int i = i0 + u * rows + mine;
      src[u] = i < end ? from[i] : make_int2(-1, 0);
      dst[u] = i < end ? to[a.c.by_page.div(i)] : 0;
    }
  };
  look(begin);
  for (int i0 = begin; i0 < end; i0 += rows * EV_UNROLL) {
    uint4 v[EV_UNROLL];
    uint8_t* at[EV_UNROLL];
#pragma unroll
    for (int u = 0; u < EV_UNROLL; ++u) {
      const int i = i0 + u * rows + mine, tok = i - a.c.by_page.div(i) * a.c.page;
      at[u] = nullptr;
      if (src[u].x < 0 || (IN_PLACE && src[u].x == dst[u] && src[u].y == tok)) continue;
      if (dst[u] < 0 || dst[u] >= a.c.num_pages) {
        record_error(a.err, DEV_BAD_INDEX);
        continue;
      }
      at[u] = base + dst[u] * ps + tok * ts;
      v[u] = *reinterpret_cast<const uint4*>(base + src[u].x * ps + src[u].y * ts);
    }
    look(i0 + rows * EV_UNROLL);
    if (IN_PLACE) __syncthreads();
#pragma unroll
    for (int u = 0; u < EV_UNROLL; ++u)
      if (at[u] != nullptr) *reinterpret_cast<uint4*>(at[u]) = v[u];
  }
}

// MOVE: what the CTA does with the rows that it has chosen.
enum { EV_LEAVE, EV_IN_PLACE, EV_COPY };
template <int MOVE>
__global__ void __launch_bounds__(EV_THREADS, 2) evict_select_kernel(EvictArgs a) {
  extern __shared__ __align__(16) uint32_t ev_keys[];
  __shared__ alignas(16) int hist[2][EV_BINS];  // read four bins at a time
  __shared__ int wsum[EV_WARPS], wtie[EV_WARPS];
  __shared__ int s_total[2];  // this slice's sure positions and ties
  __shared__ int s_bin, s_left, s_whole;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int item = blockIdx.x / cs, r = item / a.c.KH, h = item % a.c.KH;
  pdl_wait();
  const int len = cache_length(a.c, r, a.err, tid == 0 && h == 0 && rank == 0);
  const int n = min(len, a.budget);
  if (h == 0 && rank == 0 && tid == 0) a.lengths[r] = n;
  const float* sums = a.sums + (long long)r * a.s_rs + (long long)h * a.s_hs;
  const int* table = a.c.table + (long long)r * a.c.tstride;
  const long long row0 = (long long)item * a.budget;
  for (int i = n + rank * EV_THREADS + tid; i < a.budget; i += cs * EV_THREADS) {
    a.kept[row0 + i] = -1;
    a.out_sums[row0 + i] = 0.0f;
  }
  // slots b .. e - 1: the kept positions at(slot), and what goes with them
  auto fill = [&](int b, int e, auto at) {
#pragma unroll 4
    for (int slot = b + tid; slot < e; slot += EV_THREADS) {
      const int i = at(slot), pg = a.c.by_page.div(i);
      const int page = table[pg];
      const bool ok = page >= 0 && page < a.c.num_pages;
      if (!ok) record_error(a.err, DEV_BAD_INDEX);
      a.kept[row0 + slot] = i;
      a.out_sums[row0 + slot] = sums[i];
      a.from[row0 + slot] = make_int2(ok ? page : -1, i - pg * a.c.page);
    }
  };
  if (len <= a.budget) {
    const int part = (n + cs - 1) / cs, b = min(n, rank * part), e = min(n, b + part);
    fill(b, e, [](int slot) { return slot; });
    if constexpr (MOVE == EV_COPY) {
      __syncthreads();
      move_rows<false>(a, r, h, tid >> 8, 0, b, e, tid & 255);
    }
    return;
  }
  // The first and the last positions get a key above every sum's: what stays are
  // then simply the `budget` largest keys.
  const int lo = a.sinks, hi = len - a.recent;  // the positions that compete
  const int per = ((len + cs - 1) / cs + 31) & ~31;
  const int begin = min(len, rank * per), count = min(len, begin + per) - begin;
  const bool held = count <= EV_KEYS;
  auto keyed = [&](int i, float v) { return begin + i < lo || begin + i >= hi ? 0xffffffffu : sum_key(v); };
  auto keys = [&](int i, uint32_t* k) {  // those of positions i .. i + 3 of the slice, i a multiple of 4
    if (held) {
      if (i < count) *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(ev_keys + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < count) k[e] = keyed(i + e, sums[begin + i + e]);
    }
  };
  // equal sums are common (positions that were never looked at): one addition for a whole warp's
  auto add = [&](int* hp, int bin) {
    const int lead = __shfl_sync(0xffffffffu, bin, 0);
    if (__all_sync(0xffffffffu, bin == lead)) {
      if (lane == 0 && bin >= 0) atomicAdd(&hp[bin], 32);
    } else if (bin >= 0) {
      atomicAdd(&hp[bin], 1);
    }
  };

  auto meet = [&]() {
    if (cs > 1)
      cluster.sync();
    else
      __syncthreads();
  };

  uint32_t prefix = 0, mask = 0;
  int need = a.budget;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 1023u : 2047u;
    int* hp = hist[pass & 1];
    for (int i = tid; i < EV_BINS; i += EV_THREADS) hp[i] = 0;
    __syncthreads();
    if (pass == 0) {  // as the sums come in
      for (int i0 = warp * 32; i0 < count; i0 += EV_LOADS * EV_THREADS) {
        float v[EV_LOADS];
#pragma unroll
        for (int u = 0; u < EV_LOADS; ++u) {
          const int i = i0 + u * EV_THREADS + lane;
          v[u] = i < count ? sums[begin + i] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < EV_LOADS; ++u) {
          const int i = i0 + u * EV_THREADS + lane;
          if (i - lane >= count) break;
          const uint32_t k = keyed(i, v[u]);
          if (held && i < count) ev_keys[i] = k;
          add(hp, i < count ? (int)(k >> shift) : -1);
        }
      }
    } else {
      for (int i0 = warp * 128; i0 < count; i0 += 4 * EV_THREADS) {  // four keys to a lane
        const int i = i0 + 4 * lane;
        uint32_t k[4] = {};
        keys(i, k);
        bool hit[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) hit[e] = i + e < count && (k[e] & mask) == prefix;
        if (!__any_sync(0xffffffffu, hit[0] || hit[1] || hit[2] || hit[3])) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) add(hp, hit[e] ? (int)((k[e] >> shift) & digit) : -1);
      }
    }
    meet();
    // thread t: bins 4 t .. 4 t + 3 over the cluster, and the count in all higher bins
    int4 mine = make_int4(0, 0, 0, 0);
    for (int q = 0; q < cs; ++q) {
      const int4 x = reinterpret_cast<const int4*>(cluster.map_shared_rank(hp, q))[tid];
      mine.x += x.x;
      mine.y += x.y;
      mine.z += x.z;
      mine.w += x.w;
    }
    const int all = mine.x + mine.y + mine.z + mine.w;
    int above = all;  // inclusive suffix sum over lanes
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_down_sync(0xffffffffu, above, off);
      if (lane + off < 32) above += v;
    }
    if (lane == 0) wsum[warp] = above;
    __syncthreads();
    above += __reduce_add_sync(0xffffffffu, lane > warp && lane < EV_WARPS ? wsum[lane] : 0) - all;
    // the bin in which the need-th largest lies belongs to exactly one thread
    const int c4[4] = {mine.w, mine.z, mine.y, mine.x};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (above < need && need <= above + c4[e]) {
        s_bin = 4 * tid + 3 - e;
        s_left = need - above;
        s_whole = need == above + c4[e];
      }
      above += c4[e];
    }
    __syncthreads();
    need = s_left;
    prefix |= (uint32_t)s_bin << shift;
    mask |= digit << shift;
    if (s_whole) {  // the whole bin stays: the next lower key is the first that does not
      prefix -= 1;  // not below 0: there are more positions than stay
      need = 0;
      break;
    }
  }
  // what is above prefix stays, and the first `need` positions that hold it
  const int seg = ((count + EV_WARPS - 1) / EV_WARPS + 127) & ~127;  // a warp's run of positions
  const int s0 = warp * seg, s1 = min(count, s0 + seg);
  auto look = [&](int i, bool* yes, bool* tie) {  // whether i .. i + 3 stay for sure, or hold prefix
    uint32_t k[4] = {};
    keys(i, k);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      yes[e] = i + e < count && k[e] > prefix;
      tie[e] = i + e < count && k[e] == prefix;
    }
  };
  int sure = 0, ties = 0;
#pragma unroll 2
  for (int i0 = s0; i0 < s1; i0 += 128) {
    bool yes[4], tie[4];
    look(i0 + 4 * lane, yes, tie);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sure += yes[e];
      ties += tie[e];
    }
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) {
    wsum[warp] = sure;
    wtie[warp] = ties;
  }
  __syncthreads();
  // before this warp, and of the slice
  const int ws = lane < EV_WARPS ? wsum[lane] : 0, wt = lane < EV_WARPS ? wtie[lane] : 0;
  int sb = __reduce_add_sync(0xffffffffu, lane < warp ? ws : 0), tb = __reduce_add_sync(0xffffffffu, lane < warp ? wt : 0);
  const int st = __reduce_add_sync(0xffffffffu, ws), tt = __reduce_add_sync(0xffffffffu, wt);
  if (tid == 0) {
    s_total[0] = st;
    s_total[1] = tt;
  }
  meet();
  int slice_sure = 0, slice_ties = 0;  // before this slice
  for (int q = 0; q < rank; ++q) {
    const int* other = cluster.map_shared_rank(s_total, q);
    slice_sure += other[0];
    slice_ties += other[1];
  }
  const int slot0 = min(a.budget, slice_sure + min(slice_ties, need));
  const int slot1 = min(a.budget, slice_sure + st + min(slice_ties + tt, need));
  // the positions of this slice's slots, by way of shared memory where they fit
  int* found = slot1 - slot0 <= 2 * EV_BINS ? &hist[0][0] - slot0 : a.kept + row0;
  sb += slice_sure;
  tb += slice_ties;
  if (cs > 1) cluster.barrier_arrive();
#pragma unroll 2
  for (int i0 = s0; i0 < s1; i0 += 128) {
    const int i = i0 + 4 * lane;
    bool yes[4], tie[4];
    look(i, yes, tie);
    // sure positions in the low half, ties in the high one; then what comes before this lane's
    int mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) mine += (int)yes[e] + ((int)tie[e] << 16);
    int x = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += v;
    }
    const int all = __shfl_sync(0xffffffffu, x, 31);
    x -= mine;
    int sy = sb + (x & 0xffff), t = tb + (x >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = sy + min(t, need);
      if ((yes[e] || (tie[e] && t < need)) && at < a.budget) found[at] = begin + i + e;
      sy += yes[e];
      t += tie[e];
    }
    sb += all & 0xffff;
    tb += all >> 16;
  }
  __syncthreads();
  fill(slot0, slot1, [&](int slot) { return found[slot]; });
  if (cs > 1) cluster.barrier_wait();  // no CTA ends while another reads its totals
  if constexpr (MOVE != EV_LEAVE) {
    __syncthreads();
    move_rows<MOVE == EV_IN_PLACE>(a, r, h, tid >> 8, 0, slot0, slot1, tid & 255);
  }
}

// One CTA per (request, kv head, keys or values, slice of the row's bytes), and
// for a copy to other pages per `chunk` rows.
template <bool IN_PLACE>
__global__ void __launch_bounds__(256, 4) evict_move_kernel(EvictArgs a) {
  pdl_wait();
  int b = blockIdx.x;
  const int slice = b % a.slices;
  b /= a.slices;
  const int part = b & 1, item = b >> 1;
  const int r = item / a.c.KH, h = item % a.c.KH;
  const int len = cache_length(a.c, r, a.err, false);
  if (IN_PLACE && len <= a.budget) return;
  const int begin = blockIdx.y * a.chunk, end = min(min(len, a.budget), begin + a.chunk);
  move_rows<IN_PLACE>(a, r, h, part, slice, begin, end, threadIdx.x);
}

// CTAs of a cluster: as many as run at once, two to an SM, with 2048 positions each at least
// (1 request of 16000, 8 kv heads: 31.6 us against 36.1 us with 4096 and 31.4 us with 1024; 8 of 8000: 36.6, 38.1, 38.0).
// With three to an SM, 5 requests of 16500 .. 33000 take 79 us against 65 us, 10 of 8200 .. 16000 65 us against 58 us,
// 20 of 4200 .. 8000, where that means two CTAs against one, 91 us against 92 us.
int evict_cluster(int64_t items, int64_t positions) {
  const int64_t resident = 2 * num_sms();
  int cs = 1;
  while (cs < 8 && items * cs * 2 <= resident && positions >= 2048 * 2 * cs) cs *= 2;
  return cs;
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_paged_evict_workspace_size(int64_t requests, int64_t kv_heads, int64_t budget) {
  return requests < 1 || kv_heads < 1 || budget < 1 ? 0 : (size_t)requests * kv_heads * budget * sizeof(int2);
}

extern "C" fm_status fm_paged_evict(const fm_paged_cache* cache, const fm_evict* p, fm_stream stream) {
  EvictArgs a{};
  fm_status st = cache_ref(cache, "paged_evict", &a.c);
  if (st != FM_OK) return st;
  if (!p) return set_error(FM_ERR_INVALID, "paged_evict: null arguments");
  if (p->budget < 1 || p->sinks < 0 || p->recent < 0 || p->budget > 0x7ffffff0 || p->sinks > p->budget ||
      p->recent > p->budget - p->sinks)
    return set_error(FM_ERR_SHAPE, "paged_evict: sinks + recent must lie within the budget");
  if (cache->requests == 0) return FM_OK;
  if ((!p->weight_sums && cache->max_length > 0) || !p->kept || !p->lengths || !p->out_sums)
    return set_error(FM_ERR_INVALID, "paged_evict: null pointer");
  if (p->out_page_table && p->out_page_table_cols < (p->budget + cache->page_size - 1) / cache->page_size)
    return set_error(FM_ERR_SHAPE, "paged_evict: the new page table does not cover the budget");
  if (p->lengths == cache->lengths)
    return set_error(FM_ERR_INVALID, "paged_evict: the new lengths must not overwrite the old");
  if (p->out_page_table && p->out_page_table == cache->page_table)
    return set_error(FM_ERR_INVALID, "paged_evict: pass no new page table to evict in place");
  const size_t need = fm_paged_evict_workspace_size(cache->requests, cache->kv_heads, p->budget);
  if (!p->workspace || p->workspace_bytes < need)
    return set_error(FM_ERR_WORKSPACE, "paged_evict: workspace %zu < %zu", p->workspace_bytes, need);
  if ((uintptr_t)p->workspace % 8) return set_error(FM_ERR_ALIGN, "paged_evict: workspace not 8-byte aligned");
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
  a.from = static_cast<int2*>(p->workspace);
  a.row_bytes = (int)cache->head_dim * (cache->dtype == FM_DT_E4M3 ? 1 : 2);
  a.err = p->err;
  const int64_t items = cache->requests * cache->kv_heads;
  if (items > 0x3ffffff) return set_error(FM_ERR_SHAPE, "paged_evict: grid too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  const int cs = evict_cluster(items, cache->max_length);
  int64_t keys = (cache->max_length + cs - 1) / cs + 32;
  if (keys > EV_KEYS) keys = EV_KEYS;
  const size_t smem = (size_t)keys * 4;
  auto select = [&](auto kernel, fm_status allowed) {
    if (allowed != FM_OK) return allowed;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * cs));
    cfg.blockDim = dim3(EV_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)cs, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) return set_error(FM_ERR_LAUNCH, "paged_evict: %s", cudaGetErrorString(e));
    ++launch_counter();
    return (fm_status)FM_OK;
  };
  constexpr int most = EV_KEYS * 4;
  // Where there is a CTA to every SM that can move what it has chosen, it does
  // so at once: the moving of some runs beside the choosing of others.  In
  // place only one CTA may move a (request, kv head)'s rows.
  a.slices = 1;
  if (a.out_table && items * cs >= EV_FUSE)
    return select(evict_select_kernel<EV_COPY>, allow_smem<evict_select_kernel<EV_COPY>>(most, "paged_evict"));
  if (!a.out_table && cs == 1 && items >= EV_FUSE)
    return select(evict_select_kernel<EV_IN_PLACE>, allow_smem<evict_select_kernel<EV_IN_PLACE>>(most, "paged_evict"));
  st = select(evict_select_kernel<EV_LEAVE>, allow_smem<evict_select_kernel<EV_LEAVE>>(most, "paged_evict"));
  if (st != FM_OK) return st;

  // Rows are cut into slices of 32 bytes at least while there are fewer than
  // two CTAs to an SM; a copy is cut along the rows instead.
  a.chunk = a.budget;
  unsigned chunks = 1;
  if (a.out_table) {
    a.chunk = 256;
    chunks = (unsigned)((a.budget + a.chunk - 1) / a.chunk);
    if (chunks > 65535) {
      a.chunk = (a.budget + 65534) / 65535;
      chunks = (unsigned)((a.budget + a.chunk - 1) / a.chunk);
    }
  } else {
    while (items * 2 * a.slices < 2 * 148 && a.row_bytes / a.slices > 32) a.slices *= 2;
  }
  const dim3 grid((unsigned)(items * 2 * a.slices), chunks);
  if (a.out_table) return launch_kernel(evict_move_kernel<false>, grid, dim3(256), 0, s, true, a);
  return launch_kernel(evict_move_kernel<true>, grid, dim3(256), 0, s, true, a);
}
