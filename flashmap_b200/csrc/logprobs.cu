// Log probabilities of given tokens, the entropy and the largest alternatives
// of rows of logits, without writing probabilities.
//
// With c = log2(e) / T, m = c max x (rounded) and d_i = c x_i - m:
//   S = sum 2^d,  U = sum 2^d d,  log p_i = ln 2 (d_i - log2 S),
//   entropy = ln 2 (log2 S - U / S).
// One pass over the row: every thread keeps (m, S, U) of what it has seen and
// rescales when its maximum grows,
//   d' = d + a, a = m - m':  S' = 2^a S,  U' = 2^a (U + a S).
// d is formed with one rounding and every m is the same rounded product
// wherever it is used, so that the rounding of m cancels.
//
// Alternatives.  The pass also leaves the maximum of every group of one or more
// warp loads (512 bytes each).  The k largest values, equal ones by the lowest id, lie in the
// k groups that come first by (maximum, lowest group): an element of another
// group is preceded by the k maxima of those.  Those groups are read once more
// (from L2), what reaches the k-th maximum is kept, and sorted.
//
// The row's bytes bound it (one exponential, and five other operations to a value).
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"

namespace fm {
namespace {

constexpr int LP_T = 256;
constexpr int LP_LOADS = 4;        // warp loads in flight
constexpr int LP_GROUPS = 1024;    // groups of a row at most
constexpr int LP_LIST = 2048;      // candidates that are sorted at once
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

struct LogprobArgs {
  const void* x;
  long long ld;  // elements between rows
  int V, rows;
  const long long* tokens;
  float c;         // log2(e) / T
  int k, gs;       // 2^gs warp loads make a group
  int groups;      // room for a row's group maxima
  int slices, per; // CTAs of a row, warp loads of each
  float* logprob;
  float* entropy;
  long long* ids;
  float* top;
  float4* part;  // [rows][slices] (m, S, U)
  float* gmax;   // [rows][groups]
  int* err;
};

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lp_warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// A row as 16-byte pieces: piece v has values v * N - shift .. of the row
// (shift: how far the row starts behind a 16-byte boundary).
template <typename T>
struct LpRow {
  static constexpr int N = 16 / (int)sizeof(T);
  const T* x;
  int V, shift, pieces;
  __device__ __forceinline__ LpRow(const LogprobArgs& a, int row) {
    x = static_cast<const T*>(a.x) + row * a.ld;
    V = a.V;
    shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    pieces = (V + shift + N - 1) / N;
  }
  __device__ __forceinline__ int first(int piece) const { return piece * N - shift; }
  // piece `p` as it lies in memory; values outside the row are -inf
  __device__ __forceinline__ uint4 load(int p) const {
    const int i0 = first(p);
    if (i0 >= 0 && i0 + N <= V) return __ldg(reinterpret_cast<const uint4*>(x + i0));
    T v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = i0 + e >= 0 && i0 + e < V ? x[i0 + e] : (T)(-INFINITY);
    return *reinterpret_cast<const uint4*>(v);
  }
};
template <typename T>
__device__ __forceinline__ void lp_unpack(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      x[i] = __uint_as_float(w[i]);
    }
  }
}
// the largest and the least of a piece, NaN left out
template <typename T>
__device__ __forceinline__ float2 lp_range(const uint4& u) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const __nv_bfloat162 l = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));
    return make_float2(fmaxf(__low2float(m), __high2float(m)), fminf(__low2float(l), __high2float(l)));
  } else {
    const float x[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w)};
    return make_float2(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fminf(fminf(x[0], x[1]), fminf(x[2], x[3])));
  }
}

struct LpSum {
  float m, s, u;
};
// both of one row
__device__ __forceinline__ LpSum lp_join(const LpSum& a, const LpSum& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return LpSum{m, a.s + b.s, a.u + b.u};  // sums of nothing, or NaN
  LpSum r{m, 0.0f, 0.0f};
  auto add = [&](const LpSum& v) {
    if (v.m == -INFINITY && v.s == 0.0f) return;  // saw nothing
    const float d = fmaxf(v.m - m, -1000.0f), f = lp_ex2(d);
    r.s += f * v.s;
    r.u += f * (v.u + d * v.s);
  };
  add(a);
  add(b);
  return r;
}

template <typename K>
__device__ __forceinline__ void lp_sort(K* keys, int n) {  // descending, n a power of two, by the block
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += LP_T) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const K a = keys[lo], b = keys[hi];
        if ((a < b) == ((lo & size) == 0)) {
          keys[lo] = b;
          keys[hi] = a;
        }
      }
    }
  __syncthreads();
}
__device__ __forceinline__ float lp_key_value(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t i) { return argmax_key(v != v ? -INFINITY : v, i); }

struct LpShared {
  unsigned long long keys[LP_LIST];  // the warps' first groups, then candidates
  float gmax[LP_GROUPS];
  int chosen[32];
  float least;
  LpSum warp[LP_T / 32];
  unsigned long long best[LP_T / 32];
  int count;
};

// What a row's sums and group maxima say; by one block.
template <typename T>
__device__ void lp_finish(const LogprobArgs& a, int row, const LpSum& all, const float* gmax, LpShared& sh) {
  const LpRow<T> x(a, row);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float log_s = log2f(all.s);
  const bool none = all.m == -INFINITY && all.s == 0.0f;  // -inf alone
  auto logprob = [&](float v) { return none ? -INFINITY : LP_LN2 * (fmaf(v, a.c, -all.m) - log_s); };
  if (tid == 0) {
    const long long t = a.tokens[row];
    float lp = -INFINITY;
    if (t >= 0 && t < a.V)
      lp = logprob((float)x.x[t]);
    else
      record_error(a.err, DEV_BAD_INDEX);
    a.logprob[row] = lp;
    a.entropy[row] = none ? 0.0f : LP_LN2 * (log_s - all.u / all.s);
  }
  if (a.k == 0) return;
  const int loads = (x.pieces + 31) / 32, groups = (loads + (1 << a.gs) - 1) >> a.gs;
  // Every warp draws the k first of its 128 groups, four to a lane; of those the k first stand behind fewer than k others.
  constexpr int W = LP_T / 32, PER = LP_GROUPS / LP_T;
  uint32_t mine[PER];  // orderable maxima of groups (warp * PER + j) * 32 + lane; 0: none
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int g = (warp * PER + j) * 32 + lane;
    mine[j] = g < groups ? (uint32_t)(lp_key(gmax[g], 0) >> 32) : 0u;
  }
  for (int i = 0; i < a.k; ++i) {
    uint32_t best = mine[0];
#pragma unroll
    for (int j = 1; j < PER; ++j) best = max(best, mine[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    uint32_t at = 0xffffffffu;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j) at = mine[j] == best ? (uint32_t)((warp * PER + j) * 32 + lane) : at;
    at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (at == (uint32_t)((warp * PER + j) * 32 + lane)) mine[j] = 0u;
    if (lane == 0) sh.keys[warp * a.k + i] = best ? (unsigned long long)best << 32 | (0xffffffffu - at) : 0ull;
  }
  __syncthreads();
  const int take = min(a.k, groups);
  for (int i = tid; i < W * a.k; i += LP_T) {
    const unsigned long long key = sh.keys[i];
    int before = 0;
    for (int j = 0; j < W * a.k; ++j) before += sh.keys[j] > key;
    if (key && before < take) {
      sh.chosen[before] = (int)argmax_key_index(key);
      if (before == take - 1) sh.least = lp_key_value(key);
    }
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  const float least = take < a.k ? -INFINITY : sh.least;
  // the chosen groups once more: values that reach the k-th maximum
  auto each = [&](auto&& f) {
    for (int i = warp; i < take << a.gs; i += LP_T / 32) {
      const int p = ((sh.chosen[i >> a.gs] << a.gs) + (i & ((1 << a.gs) - 1))) * 32 + lane;
      if (p >= x.pieces) continue;
      float v[LpRow<T>::N];
      lp_unpack<T>(x.load(p), v);
      const int i0 = x.first(p);
#pragma unroll
      for (int e = 0; e < LpRow<T>::N; ++e)
        if (i0 + e >= 0 && i0 + e < a.V) f(v[e] != v[e] ? -INFINITY : v[e], i0 + e);
    }
  };
  each([&](float v, int i) {
    if (v >= least) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < LP_LIST) sh.keys[at] = lp_key(v, (uint32_t)i);
    }
  });
  __syncthreads();
  const int count = sh.count;
  if (count <= LP_T) {  // as a rule: a candidate to a thread, which counts those before it
    const unsigned long long key = tid < count ? sh.keys[tid] : 0ull;
    int before = 0;
    for (int j = 0; j < count; ++j) before += sh.keys[j] > key;
    if (tid < count && before < a.k) {
      a.ids[(long long)row * a.k + before] = argmax_key_index(key);
      a.top[(long long)row * a.k + before] = logprob(lp_key_value(key));
    }
    return;
  }
  if (count <= LP_LIST) {
    int n = 2;
    while (n < count) n <<= 1;
    for (int i = count + tid; i < n; i += LP_T) sh.keys[i] = 0ull;
    lp_sort(sh.keys, n);
    if (tid < a.k) {
      const unsigned long long key = sh.keys[tid];
      a.ids[(long long)row * a.k + tid] = argmax_key_index(key);
      a.top[(long long)row * a.k + tid] = logprob(lp_key_value(key));
    }
    return;
  }
  // a great many equal values: one alternative after the other
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    unsigned long long best = 0;
    each([&](float v, int i) {
      const unsigned long long key = lp_key(v, (uint32_t)i);
      if (key < last && key > best) best = key;
    });
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (lane == 0) sh.best[warp] = best;
    __syncthreads();
    for (int w = 0; w < LP_T / 32; ++w) best = sh.best[w] > best ? sh.best[w] : best;
    last = best;
    if (tid == 0) {
      a.ids[(long long)row * a.k + j] = argmax_key_index(best);
      a.top[(long long)row * a.k + j] = logprob(lp_key_value(best));
    }
  }
}

__device__ __forceinline__ LpSum lp_block_join(LpSum v, LpShared& sh) {
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    const LpSum o{__shfl_xor_sync(0xffffffffu, v.m, off), __shfl_xor_sync(0xffffffffu, v.s, off),
                  __shfl_xor_sync(0xffffffffu, v.u, off)};
    // the lower lane's first, so that both get the same bits
    v = (threadIdx.x & off) ? lp_join(o, v) : lp_join(v, o);
  }
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh.warp[0];
  for (int w = 1; w < LP_T / 32; ++w) v = lp_join(v, sh.warp[w]);
  return v;
}

// Block (row, slice): warp loads slice * per .. of the row.  ONE: a warp load is
// a group of its own.
template <typename T, bool TOP, bool ONE>
__global__ void __launch_bounds__(LP_T, 4) logprob_scan_kernel(LogprobArgs a) {
  __shared__ LpShared sh;
  pdl_wait();
  const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const LpRow<T> x(a, row);
  constexpr int N = LpRow<T>::N;
  const int loads = (x.pieces + 31) / 32, end = min(loads, (slice + 1) * a.per);
  const int span = ONE ? LP_LOADS : max(LP_LOADS, 1 << a.gs);  // a warp's loads at a time hold whole groups
  float* gmax = a.slices == 1 ? sh.gmax : a.gmax + (long long)row * a.groups;
  const uint4 nothing = sizeof(T) == 2 ? make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u)
                                       : make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
  const int whole = x.shift ? 1 : 0, whole_end = (a.V + x.shift) / N;  // pieces that lie in the row altogether
  const uint4* base = reinterpret_cast<const uint4*>(x.x - x.shift) + lane;
  auto fetch = [&](uint4* u, int l1) {
    if (l1 * 32 >= whole && (l1 + LP_LOADS) * 32 <= whole_end) {
#pragma unroll
      for (int q = 0; q < LP_LOADS; ++q) u[q] = __ldcs(base + (l1 + q) * 32);
    } else {
#pragma unroll
      for (int q = 0; q < LP_LOADS; ++q) {
        const int p = (l1 + q) * 32 + lane;
        u[q] = p < x.pieces ? x.load(p) : nothing;
      }
    }
  };
  // the warp's batches: LP_LOADS loads each, span after span
  auto after = [&](int l1) { return ((l1 + LP_LOADS) & (span - 1)) ? l1 + LP_LOADS : l1 + LP_LOADS + (LP_T / 32 - 1) * span; };
  LpSum v{-INFINITY, 0.0f, 0.0f};
  const float2 c2 = make_float2(a.c, a.c);
  uint4 next[LP_LOADS];
  float gm = -INFINITY;
  // A span is gone through to its end: behind the row there is nothing, but a group is still closed.
  const int stop = (end + span - 1) & ~(span - 1);
  int l1 = slice * a.per + warp * span;
  if (l1 < stop) fetch(next, l1);
  while (l1 < stop) {
    uint4 u[LP_LOADS];
#pragma unroll
    for (int q = 0; q < LP_LOADS; ++q) u[q] = next[q];
    const int l2 = after(l1);
    if (l2 < stop) fetch(next, l2);
    float mx[LP_LOADS], top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int q = 0; q < LP_LOADS; ++q) {
      const float2 range = lp_range<T>(u[q]);
      mx[q] = range.x;
      top = fmaxf(top, range.x);
      low = fminf(low, range.y);
    }
    top *= a.c;
    if (top > v.m) {
      if (v.m != -INFINITY) {
        const float d = fmaxf(v.m - top, -1000.0f), f = lp_ex2(d);
        v.u = f * (v.u + d * v.s);
        v.s *= f;
      }
      v.m = top;
    }
    const float off = v.m == -INFINITY ? 0.0f : v.m;
    // 2^d d is 0 where d is -inf; where no value is so low that d could be, it needs no guard
    const bool guard = __any_sync(0xffffffffu, !(low * a.c - off > -1e30f));
    float2 s2 = make_float2(v.s, 0.0f), u2 = make_float2(v.u, 0.0f);
    const float2 o2 = make_float2(-off, -off);
    auto add = [&](auto guarded) {
#pragma unroll
      for (int q = 0; q < LP_LOADS; ++q) {
        float y[N];
        lp_unpack<T>(u[q], y);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          float2 d = __ffma2_rn(make_float2(y[e], y[e + 1]), c2, o2);
          const float2 p = make_float2(lp_ex2(d.x), lp_ex2(d.y));
          s2 = __fadd2_rn(s2, p);
          if constexpr (decltype(guarded)::value) d = make_float2(fmaxf(d.x, -1000.0f), fmaxf(d.y, -1000.0f));
          u2 = __ffma2_rn(p, d, u2);
        }
      }
    };
    if (guard)
      add(std::true_type{});
    else
      add(std::false_type{});
    v.s = s2.x + s2.y;
    v.u = u2.x + u2.y;
    if constexpr (TOP && ONE) {
      float mine = lp_warp_max(mx[0]);
#pragma unroll
      for (int q = 1; q < LP_LOADS; ++q) {
        const float g = lp_warp_max(mx[q]);
        mine = lane == q ? g : mine;
      }
      if (lane < LP_LOADS && l1 + lane < loads) gmax[l1 + lane] = mine;
    } else if constexpr (TOP) {
#pragma unroll
      for (int q = 0; q < LP_LOADS; ++q) {
        gm = fmaxf(gm, mx[q]);
        if (((l1 + q + 1) & ((1 << a.gs) - 1)) == 0) {
          const float g = lp_warp_max(gm);
          if (lane == 0 && l1 + q + 1 - (1 << a.gs) < loads) gmax[(l1 + q) >> a.gs] = g;
          gm = -INFINITY;
        }
      }
    }
    l1 = l2;
  }
  v = lp_block_join(v, sh);
  if (a.slices > 1) {
    if (threadIdx.x == 0) a.part[(long long)row * a.slices + slice] = make_float4(v.m, v.s, v.u, 0.0f);
    return;
  }
  lp_finish<T>(a, row, v, sh.gmax, sh);
}

template <typename T>
__global__ void __launch_bounds__(LP_T) logprob_join_kernel(LogprobArgs a) {
  __shared__ LpShared sh;
  pdl_wait();
  const int row = blockIdx.x;
  LpSum v{-INFINITY, 0.0f, 0.0f};
  for (int s = threadIdx.x; s < a.slices; s += LP_T) {
    const float4 p = a.part[(long long)row * a.slices + s];
    v = lp_join(v, LpSum{p.x, p.y, p.z});
  }
  v = lp_block_join(v, sh);
  lp_finish<T>(a, row, v, a.gmax + (long long)row * a.groups, sh);
}

struct LogprobPlan {
  int gs, groups, slices, per;
  size_t part, total;
};
LogprobPlan logprob_plan(int64_t rows, int64_t V, int64_t esz, int64_t k) {
  LogprobPlan p{};
  const int64_t load = 512 / esz, loads = (V + 16 / esz - 1 + load - 1) / load + 1;
  while (((loads - 1) >> p.gs) + 1 > LP_GROUPS) ++p.gs;
  p.groups = (int)(((loads - 1) >> p.gs) + 1);
  const int64_t span = 1 << p.gs > LP_LOADS ? 1 << p.gs : LP_LOADS, least = span * (LP_T / 32);
  int64_t slices = (4 * num_sms() + rows - 1) / rows;
  const int64_t most = (loads + least - 1) / least;
  if (slices > most) slices = most;
  p.per = (int)(((loads + slices - 1) / slices + span - 1) / span * span);
  p.slices = (int)((loads + p.per - 1) / p.per);
  p.part = p.slices > 1 ? (size_t)rows * p.slices * sizeof(float4) : 0;
  p.total = p.part + (p.slices > 1 && k ? ((size_t)rows * p.groups * 4 + 15) / 16 * 16 : 0);
  return p;
}

template <typename T>
fm_status launch_logprobs(const LogprobArgs& a, cudaStream_t s) {
  auto kernel = a.k == 0 ? logprob_scan_kernel<T, false, true> : a.gs == 0 ? logprob_scan_kernel<T, true, true> : logprob_scan_kernel<T, true, false>;
  const fm_status st = launch_kernel(kernel, dim3((unsigned)(a.rows * (int64_t)a.slices)), dim3(LP_T), 0, s, true, a);
  if (st != FM_OK || a.slices == 1) return st;
  return launch_kernel(logprob_join_kernel<T>, dim3((unsigned)a.rows), dim3(LP_T), 0, s, true, a);
}

bool logprob_sizes(int64_t rows, int64_t V, int32_t dtype, int64_t k) {
  return rows >= 0 && rows <= 0x3fffffff && V >= 1 && V <= 0x40000000 && k >= 0 && k <= FM_TOKEN_LOGPROBS_MAX_TOP && k <= V &&
         (dtype == FM_DT_BF16 || dtype == FM_DT_F32);
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_token_logprobs_workspace_size(int64_t rows, int64_t V, int32_t dtype, int64_t top_k) {
  if (rows < 1 || !logprob_sizes(rows, V, dtype, top_k)) return 0;
  return logprob_plan(rows, V, dtype == FM_DT_F32 ? 4 : 2, top_k).total;
}

extern "C" fm_status fm_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, const int64_t* tokens,
                                       int64_t rows, int64_t V, float temperature, int64_t top_k, float* logprobs,
                                       float* entropy, int64_t* top_ids, float* top_logprobs, void* workspace,
                                       size_t workspace_bytes, int32_t* err, fm_stream stream) {
  if (!logprob_sizes(rows, V, dtype, top_k)) return set_error(FM_ERR_SHAPE, "token_logprobs: bad shape");
  if (!(temperature > 0.0f && temperature < INFINITY))
    return set_error(FM_ERR_INVALID, "token_logprobs: the temperature must be positive");
  if (rows == 0) return FM_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top_k && (!top_ids || !top_logprobs)))
    return set_error(FM_ERR_INVALID, "token_logprobs: null pointer");
  const int64_t esz = dtype == FM_DT_F32 ? 4 : 2;
  if ((uintptr_t)logits % esz) return set_error(FM_ERR_ALIGN, "token_logprobs: logits must be aligned to their type");
  const LogprobPlan pl = logprob_plan(rows, V, esz, top_k);
  if (pl.total > workspace_bytes || (pl.total && !workspace))
    return set_error(FM_ERR_WORKSPACE, "token_logprobs: workspace %zu < %zu", workspace_bytes, pl.total);
  if ((uintptr_t)workspace % 16) return set_error(FM_ERR_ALIGN, "token_logprobs: workspace not 16-byte aligned");
  if (rows * pl.slices > 0x7fffffff) return set_error(FM_ERR_SHAPE, "token_logprobs: grid too large");
  LogprobArgs a{};
  a.x = logits;
  a.ld = rows == 1 ? 0 : row_stride;
  a.V = (int)V;
  a.rows = (int)rows;
  a.tokens = reinterpret_cast<const long long*>(tokens);
  a.c = LP_LOG2E / temperature;
  a.k = (int)top_k;
  a.gs = pl.gs;
  a.groups = pl.groups;
  a.slices = pl.slices;
  a.per = pl.per;
  a.logprob = logprobs;
  a.entropy = entropy;
  a.ids = reinterpret_cast<long long*>(top_ids);
  a.top = top_logprobs;
  a.part = static_cast<float4*>(workspace);
  a.gmax = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pl.part);
  a.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FM_DT_F32 ? launch_logprobs<float>(a, s) : launch_logprobs<__nv_bfloat16>(a, s);
}
