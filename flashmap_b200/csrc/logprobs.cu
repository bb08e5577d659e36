// Log probabilities of given tokens, the entropy and the largest alternatives
// of rows of logits, without writing probabilities.
//
// With c = log2(e) / T, m near max x and d_i = c (x_i - m):
//   S = sum 2^d,  U = sum 2^d d,  log p_i = ln 2 (d_i - log2 S),
//   entropy = ln 2 (log2 S - U / S).
// One pass over the row: every thread keeps (m, S, U) of what it has seen, m
// any value near the maximum, and rescales when m moves,
//   d' = d + a, a = c (m - m'):  S' = 2^a S,  U' = 2^a (U + a S).
// d is formed as c x - round(c m), one multiplication and addition, and c (m - m')
// as the difference of the same rounded products, so that their rounding
// cancels; only where |c m| is 2^24 or more (rows of a mask's value, tiny T) as
// c (x - m), since a rounding of 2^7 and more would be past the exponentials' range.
//
// Alternatives.  The pass also leaves the maximum of every group of two or more
// warp loads (512 bytes each).  The k largest values, equal ones by the lowest id, lie in the
// k groups that come first by (maximum, lowest group): an element of another
// group is preceded by the k maxima of those.  Those groups are read once more
// (from L2), what reaches the k-th maximum is kept, and sorted.
//
// The row's bytes bound it, and beside them one exponential and about eight other
// instructions to a value: 1088 bf16 rows of 151936, 56 us (5.9 TB/s), 81 to 84 us
// with 20 alternatives, whose own launch is bound by instructions (13 million);
// 1999 fp32 rows of 32003, half of it -inf, 44 to 46 us (5.6 to 5.8 TB/s);
// one bf16 row of 151936, 8.4 us with 5 alternatives, 10 us with 20.
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"

namespace fm {
namespace {

constexpr int LP_T = 256;
constexpr int LP_SLICES = 8;       // of a row at most: a cluster
constexpr int LP_LOADS = 4;        // warp loads in flight
constexpr int LP_GROUPS = 256;     // groups of a row at most: one to a thread
constexpr int LP_HITS = 512;
constexpr int LP_LIST = 2048;      // candidates that are sorted at once
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

struct LogprobArgs {
  const void* x;
  long long ld;  // elements between rows
  int V, rows;
  const long long* tokens;
  float t, c, lag; // T, log2(e) / T, 8 / c
  int k, gs;       // 2^gs warp loads make a group
  int groups;      // room for a row's group maxima
  int slices, per; // CTAs of a row, warp loads of each
  float* logprob;
  float* entropy;
  long long* ids;
  float* top;
  float4* part;  // [rows] (m, S, U)
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

// Eight bf16 or four fp32 values from x[i0] on, -inf where the row has none.
template <typename T>
__device__ __noinline__ uint4 lp_edge(const T* x, int i0, int V) {
  constexpr int N = 16 / (int)sizeof(T);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 2) {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
      const int i = i0 + 2 * q;
      const uint32_t lo = i >= 0 && i < V ? h[i] : 0xff80u, hi = i + 1 >= 0 && i + 1 < V ? h[i + 1] : 0xff80u;
      w[q] = lo | hi << 16;
    } else {
      const int i = i0 + q;
      w[q] = i >= 0 && i < V ? reinterpret_cast<const uint32_t*>(x)[i] : 0xff800000u;
    }
  }
  static_assert(N == 8 || N == 4, "bf16 or fp32");
  return make_uint4(w[0], w[1], w[2], w[3]);
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
    const int i0 = min(first(p), V);
    if (i0 >= 0 && i0 + N <= V) return __ldg(reinterpret_cast<const uint4*>(x + i0));
    return lp_edge(x, i0, V);
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
// A running m stands for the power c m: as the rounded product where that is
// within a half (|c m| < 2^24: what it is off by goes into every term and out with
// log2 S), else as c m itself, whose differences are formed as c (x - m).
__device__ __forceinline__ bool lp_fast(float m, float c) { return fabsf(m * c) < 16777216.0f; }
// the power of x less that of m
__device__ __forceinline__ float lp_diff(float x, float m, float c) {
  const bool fx = lp_fast(x, c), fm = lp_fast(m, c);
  return fx && fm ? __fsub_rn(__fmul_rn(x, c), __fmul_rn(m, c))
         : fm     ? fmaf(x, c, -__fmul_rn(m, c))
         : fx     ? -fmaf(m, c, -__fmul_rn(x, c))
                  : (x - m) * c;
}
// to the same place in the first CTA of the cluster
__device__ __forceinline__ void lp_store_first(const float* at, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(at), 0)), "f"(v) : "memory");
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

template <bool TOP>
struct LpShared {
  alignas(16) unsigned long long keys[TOP ? LP_LIST : 2];  // candidates
  alignas(16) uint32_t group[TOP ? LP_GROUPS : 4];  // orderable maxima
  int hit[TOP ? LP_HITS : 1];  // pieces that hold a candidate
  int chosen[32];
  int hits;
  uint32_t least;
  LpSum warp[LP_T / 32];
  unsigned long long best[LP_T / 32];
  int count;
};

// What a row's sums and group maxima say; by one block.
template <typename T, bool TOP>
__device__ void lp_finish(const LogprobArgs& a, int row, const LpSum& all, const float* gmax, LpShared<TOP>& sh) {
  const LpRow<T> x(a, row);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float log_s = log2f(all.s);
  const bool none = all.m == -INFINITY && all.s == 0.0f;  // -inf alone
  auto logprob = [&](float v) {
    if (none) return -INFINITY;
    const float d = lp_fast(all.m, a.c) ? fmaf(v, a.c, -__fmul_rn(all.m, a.c)) : (v - all.m) * a.c;
    // c (v - m) can be past fp32's range where (v - m) / T is not (masks of the type's lowest value); v - m can be, too,
    // where T brings it back
    if (d == -INFINITY && v > -INFINITY) return (a.t < 1.0f ? (v - all.m) / a.t : v / a.t - all.m / a.t) - LP_LN2 * log_s;
    const float lp = LP_LN2 * (d - log_s);
    return lp > 0.0f ? 0.0f : lp;  // d and log2 S of a token that is nearly certain agree but for their rounding
  };
  if (tid == 0) {
    const long long t = a.tokens[row];
    float lp = -INFINITY;
    if (t >= 0 && t < a.V)
      lp = logprob((float)x.x[t]);
    else
      record_error(a.err, DEV_BAD_INDEX);
    a.logprob[row] = lp;
    const float entropy = none ? 0.0f : LP_LN2 * (log_s - all.u / all.s);
    a.entropy[row] = entropy < 0.0f ? 0.0f : entropy;
  }
  if (!TOP || a.k == 0) return;
  const int loads = (x.pieces + 31) / 32, groups = (loads + (1 << a.gs) - 1) >> a.gs;
  // The groups that stand behind fewer than k others.
  static_assert(LP_GROUPS == LP_T, "a group to a thread");
  if (tid < LP_GROUPS) sh.group[tid] = tid < groups ? (uint32_t)(lp_key(gmax[tid], 0) >> 32) : 0u;
  if (tid == 0) {
    sh.count = sh.hits = 0;
    sh.least = 0xffffffffu;
  }
  __syncthreads();
  if (tid < groups) {
    const uint32_t mine = sh.group[tid];  // 1 at least
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < groups; j += 4) {
      const uint4 g = *reinterpret_cast<const uint4*>(sh.group + j);
      before += (g.x > mine - (j < tid)) + (g.y > mine - (j + 1 < tid)) + (g.z > mine - (j + 2 < tid)) + (g.w > mine - (j + 3 < tid));
    }
    if (before < a.k) {
      sh.chosen[before] = tid;
      atomicMin(&sh.least, mine);
    }
  }
  __syncthreads();
  const int take = min(a.k, groups);
  const float least = take < a.k ? -INFINITY : lp_key_value((unsigned long long)sh.least << 32);
  // the chosen groups once more: values that reach the k-th maximum
  const int again = take << a.gs;  // warp loads
  auto piece = [&](int i) { return ((sh.chosen[i >> a.gs] << a.gs) + (i & ((1 << a.gs) - 1))) * 32 + lane; };
  auto values = [&](int p, const uint4& u, auto&& f) {  // those of a piece, NaN as -inf
    const int first = x.first(p);
    float v[LpRow<T>::N];
    lp_unpack<T>(u, v);
#pragma unroll
    for (int e = 0; e < LpRow<T>::N; ++e)
      if (first + e >= 0 && first + e < a.V) f(v[e] != v[e] ? -INFINITY : v[e], first + e);
  };
  constexpr int W = LP_T / 32;
  {
    constexpr int U = 5;
    for (int i0 = warp; i0 < again; i0 += U * W) {
      uint4 u[U];
#pragma unroll
      for (int q = 0; q < U; ++q) u[q] = x.load(piece(min(i0 + q * W, again - 1)));
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (i0 + q * W < again && !(lp_range<T>(u[q]).x < least)) {
          const int at = atomicAdd(&sh.hits, 1);
          if (at < LP_HITS) sh.hit[at] = piece(i0 + q * W);
        }
    }
  }
  __syncthreads();
  const int hits = sh.hits;
  if (hits <= LP_HITS) {  // as a rule: the few pieces that hold such a value, one to a thread
    for (int i = tid; i < hits; i += LP_T)
      values(sh.hit[i], x.load(sh.hit[i]), [&](float v, int id) {
        if (v >= least) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < LP_LIST) sh.keys[at] = lp_key(v, (uint32_t)id);
        }
      });
  } else if (tid == 0) {
    sh.count = LP_LIST + 1;
  }
  __syncthreads();
  const int count = sh.count;
  if (count <= LP_T) {  // as a rule: a candidate to a thread, which counts those before it
    if (tid >= count) return;
    const unsigned long long key = sh.keys[tid];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j + 1 < count; j += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(sh.keys + j);
      before += (two.x > key) + (two.y > key);
    }
    if (count & 1) before += sh.keys[count - 1] > key;
    if (before < a.k) {
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
  // More candidates than are sorted: a great many equal values, but also rows that no threshold thins out, since they have
  // fewer groups than alternatives, or fewer groups with a value above -inf.  One alternative after the other, each a
  // pass over the chosen groups: a bf16 row of 8000 values takes 7.4 us with 5 alternatives, 54 us with 20 (2000 rows 24
  // and 410 us); one of 151936 of which 5 values are open 17 and 111 us.
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    unsigned long long best = 0;
    for (int i = warp; i < again; i += W)
      values(piece(i), x.load(piece(i)), [&](float v, int id) {
        const unsigned long long key = lp_key(v, (uint32_t)id);
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
    for (int w = 0; w < W; ++w) best = sh.best[w] > best ? sh.best[w] : best;
    last = best;
    if (tid == 0) {
      a.ids[(long long)row * a.k + j] = argmax_key_index(best);
      a.top[(long long)row * a.k + j] = logprob(lp_key_value(best));
    }
  }
}

// The sum of all lanes', in every lane.
__device__ __forceinline__ LpSum lp_warp_join(LpSum v, float c) {
  const float m = lp_warp_max(v.m);
  if (m != -INFINITY) {  // a lane that saw nothing gets a factor of 0, one with NaN keeps it
    const float d = v.m == m ? 0.0f : fmaxf(lp_diff(v.m, m, c), -1000.0f), f = lp_ex2(d);
    v.u = f * (v.u + d * v.s);
    v.s *= f;
  }
  v.m = m;
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    v.s += __shfl_xor_sync(0xffffffffu, v.s, off);
    v.u += __shfl_xor_sync(0xffffffffu, v.u, off);
  }
  return v;
}
template <bool TOP>
__device__ __forceinline__ LpSum lp_block_join(LpSum v, float c, LpShared<TOP>& sh) {
  const int lane = threadIdx.x & 31;
  v = lp_warp_join(v, c);
  if (lane == 0) sh.warp[threadIdx.x >> 5] = v;
  __syncthreads();
  return lp_warp_join(lane < LP_T / 32 ? sh.warp[lane] : LpSum{-INFINITY, 0.0f, 0.0f}, c);
}

// Block (row, slice): warp loads slice * per .. of the row, LP_LOADS of them at a
// time to a warp (a batch), the next batch on its way meanwhile.  Batches that
// do not lie in the row altogether come last.
// LONG: groups of more than a batch.  CLUSTER: a row's slices are a cluster of
// CTAs, which hand their sums and maxima to the first, and that finishes the row.
template <typename T, bool TOP, bool LONG, bool CLUSTER>
__global__ void __launch_bounds__(LP_T, 4) logprob_scan_kernel(LogprobArgs a) {
  __shared__ LpShared<CLUSTER && TOP> sh;
  __shared__ float row_gmax[CLUSTER && TOP ? LP_GROUPS : 1];
  __shared__ LpSum row_part[CLUSTER ? LP_SLICES : 1];
  if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  const int row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const LpRow<T> x(a, row);
  constexpr int N = LpRow<T>::N, W = LP_T / 32;
  const int loads = (x.pieces + 31) / 32, end = min(loads, (slice + 1) * a.per);
  float* gmax = CLUSTER ? row_gmax : a.gmax + (long long)row * a.groups;
  LpSum v{-INFINITY, 0.0f, 0.0f};
  const float2 c2 = make_float2(a.c, a.c);

  auto add = [&](const uint4* u, int l1) {
    float mx[LP_LOADS], top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int q = 0; q < LP_LOADS; ++q) {
      const float2 range = lp_range<T>(u[q]);
      mx[q] = range.x;
      top = fmaxf(top, range.x);
      low = fminf(low, range.y);
    }
    // m need not be the maximum: it follows when that is 2^8 ahead of it
    if (top > v.m && (v.m == -INFINITY || top > v.m + a.lag)) {
      if (v.m != -INFINITY) {
        const float d = fmaxf(lp_diff(v.m, top, a.c), -1000.0f), f = lp_ex2(d);
        v.u = f * (v.u + d * v.s);
        v.s *= f;
      }
      v.m = top;
    }
    const float off = v.m == -INFINITY ? 0.0f : __fmul_rn(v.m, a.c);
    float2 s2 = make_float2(v.s, 0.0f), u2 = make_float2(v.u, 0.0f);
    // 2^d d is 0 where d is -inf; where no value is so low that d could be, and c m goes by its rounded product, nothing is guarded
    const bool fast = fabsf(off) < 16777216.0f;
    if (__any_sync(0xffffffffu, !(fast && low * a.c > -1e30f))) {
      const float m = v.m == -INFINITY ? 0.0f : v.m;
#pragma unroll
      for (int q = 0; q < LP_LOADS; ++q) {
        float y[N];
        lp_unpack<T>(u[q], y);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float d = fast ? fmaf(y[e], a.c, -off) : (y[e] - m) * a.c, p = lp_ex2(d);
          s2.x += p;
          u2.x = fmaf(p, fmaxf(d, -1000.0f), u2.x);
        }
      }
    } else {
      const float2 o2 = make_float2(-off, -off);
#pragma unroll
      for (int q = 0; q < LP_LOADS; ++q) {
        float y[N];
        lp_unpack<T>(u[q], y);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 d = __ffma2_rn(make_float2(y[e], y[e + 1]), c2, o2);
          const float2 p = make_float2(lp_ex2(d.x), lp_ex2(d.y));
          s2 = __fadd2_rn(s2, p);
          u2 = __ffma2_rn(p, d, u2);
        }
      }
    }
    v.s = s2.x + s2.y;
    v.u = u2.x + u2.y;
    if constexpr (TOP) {
      if constexpr (!LONG) {  // groups of two or four loads
        if (a.gs == 1) {
          mx[0] = fmaxf(mx[0], mx[1]);
          mx[1] = fmaxf(mx[2], mx[3]);
        } else {
          mx[0] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        }
        float mine = lp_warp_max(mx[0]);
        if (a.gs == 1) {
          const float g = lp_warp_max(mx[1]);
          mine = lane == 1 ? g : mine;
        }
        const int g0 = (l1 >> a.gs) + lane;
        if (lane < LP_LOADS >> a.gs && g0 << a.gs < loads) gmax[g0] = mine;
      } else {  // a group is one warp's, batch after batch
        const float g = lp_warp_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
        if (lane == 0) {
          float* at = gmax + (l1 >> a.gs);
          *at = (l1 & ((1 << a.gs) - 1)) == 0 ? g : fmaxf(*at, g);
        }
      }
    }
  };
  const uint4* base = reinterpret_cast<const uint4*>(x.x - x.shift) + lane;
  const uint4* at = base;  // of the batch that comes next
  auto fetch = [&](uint4* u, int l1) {
    if constexpr (LONG) at = base + l1 * 32;
#pragma unroll
    for (int q = 0; q < LP_LOADS; ++q) u[q] = __ldcs(at + q * 32);
    at += W * LP_LOADS * 32;
  };
  // Batches of the warp: span after span, so that a group is one warp's.
  const int span = LONG ? 1 << a.gs : LP_LOADS;
  auto after = [&](int l1) {
    if constexpr (!LONG) return l1 + W * LP_LOADS;
    return ((l1 + LP_LOADS) & (span - 1)) ? l1 + LP_LOADS : l1 + LP_LOADS + (W - 1) * span;
  };
  const int first = slice * a.per + warp * span;
  const int whole_end = (a.V + x.shift) / N / (32 * LP_LOADS) * LP_LOADS;  // batches below this one are whole, but for
  const bool ragged = x.shift != 0 && first == 0;                          // the row's first where it starts between two pieces
  auto edge = [&](int l1) {
    uint4 u[LP_LOADS];
#pragma unroll
    for (int q = 0; q < LP_LOADS; ++q) u[q] = x.load((l1 + q) * 32 + lane);
    add(u, l1);
  };
  int l1 = first;
  if (ragged && l1 < end) {
    edge(l1);
    l1 = after(l1);
  }
  const int stop = min(end, whole_end);
  if (l1 < stop) {
    uint4 u[LP_LOADS], w[LP_LOADS];
    at = base + l1 * 32;
    fetch(u, l1);
    while (true) {
      const int l2 = after(l1);
      if (l2 < stop) fetch(w, l2);
      add(u, l1);
      l1 = l2;
      if (l1 >= stop) break;
      const int l3 = after(l1);
      if (l3 < stop) fetch(u, l3);
      add(w, l1);
      l1 = l3;
      if (l1 >= stop) break;
    }
  }
  for (; l1 < end; l1 = after(l1)) edge(l1);
  v = lp_block_join(v, a.c, sh);
  if constexpr (CLUSTER) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all have begun: their shared memory is there
    if (TOP && slice > 0) {
      const int g1 = min((loads + (1 << a.gs) - 1) >> a.gs, ((slice + 1) * a.per) >> a.gs);
      for (int g = ((slice * a.per) >> a.gs) + (int)threadIdx.x; g < g1; g += LP_T) lp_store_first(&row_gmax[g], row_gmax[g]);
    }
    if (threadIdx.x == 0) {
      lp_store_first(&row_part[slice].m, v.m);
      lp_store_first(&row_part[slice].s, v.s);
      lp_store_first(&row_part[slice].u, v.u);
    }
    cluster_sync();
    if (slice > 0) return;
    v = lp_warp_join(lane < a.slices ? row_part[lane] : LpSum{-INFINITY, 0.0f, 0.0f}, a.c);
    lp_finish<T, TOP>(a, row, v, row_gmax, sh);
  } else if (TOP) {
    if (threadIdx.x == 0) a.part[row] = make_float4(v.m, v.s, v.u, 0.0f);
  } else {
    lp_finish<T, false>(a, row, v, nullptr, sh);
  }
}

template <typename T>
__global__ void __launch_bounds__(LP_T, 6) logprob_join_kernel(LogprobArgs a) {
  __shared__ LpShared<true> sh;
  pdl_wait();
  const int row = blockIdx.x;
  const float4 p = a.part[row];
  const LpSum v{p.x, p.y, p.z};
  lp_finish<T, true>(a, row, v, a.gmax + (long long)row * a.groups, sh);
}

// Rows for four blocks to an SM: a block to a row, and where alternatives are
// wanted a second launch for them (1088 rows, 20 alternatives: 81 us; in the same
// launch 83 us, since all blocks come to that at once).  Fewer rows are cut into up
// to eight slices, a cluster to a row, in one launch: as fast on the device as with
// partial sums in memory and a second launch (1 row 8.4 and 8.2 us, 32 rows with
// 20 alternatives 11.4 and 12.2), and a call costs the host 4 us less.  As many
// slices as are at work at once, no more (200 rows: 2 slices 22 us, 3 slices 24 us;
// 300 rows of 32003: 1 slice 13 us, 2 slices 18 us).
struct LogprobPlan {
  int gs, groups, slices, per;
  bool cluster;
  size_t part, total;
};
LogprobPlan logprob_plan(int64_t rows, int64_t V, int64_t esz, int64_t k) {
  LogprobPlan p{};
  const int64_t load = 512 / esz, loads = (V + 16 / esz - 1 + load - 1) / load + 1, fill = 4 * num_sms();
  p.gs = 1;  // of two loads or more: what is read again is little, and there are fewer to draw from
  while (((loads - 1) >> p.gs) + 1 > LP_GROUPS) ++p.gs;
  p.groups = (int)(((loads - 1) >> p.gs) + 1);
  const int64_t span = 1 << p.gs > LP_LOADS ? 1 << p.gs : LP_LOADS, least = span * (LP_T / 32);
  p.cluster = rows < fill;
  int64_t slices = std::max<int64_t>(fill / rows, 1);
  slices = std::min<int64_t>(std::min<int64_t>(slices, LP_SLICES), (loads + least - 1) / least);
  p.per = (int)(((loads + slices - 1) / slices + span - 1) / span * span);
  p.slices = (int)((loads + p.per - 1) / p.per);
  p.part = !p.cluster && k ? (size_t)rows * sizeof(float4) : 0;
  p.total = p.part + (p.part ? ((size_t)rows * p.groups * 4 + 15) / 16 * 16 : 0);
  return p;
}

template <typename T, bool CLUSTER>
fm_status launch_logprobs(const LogprobArgs& a, cudaStream_t s) {
  auto kernel = a.k == 0      ? logprob_scan_kernel<T, false, false, CLUSTER>
                : a.gs <= 2 ? logprob_scan_kernel<T, true, false, CLUSTER>
                            : logprob_scan_kernel<T, true, true, CLUSTER>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * (int64_t)a.slices));
  cfg.blockDim = dim3(LP_T);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.slices;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return set_error(FM_ERR_LAUNCH, "token_logprobs: launch failed: %s", cudaGetErrorString(e));
  ++launch_counter();
  if (CLUSTER || a.k == 0) return FM_OK;
  return launch_kernel(logprob_join_kernel<T>, dim3((unsigned)a.rows), dim3(LP_T), 0, s, true, a);
}
template <typename T>
fm_status launch_logprobs(const LogprobArgs& a, bool cluster, cudaStream_t s) {
  return cluster ? launch_logprobs<T, true>(a, s) : launch_logprobs<T, false>(a, s);
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
  if (!(LP_LOG2E / temperature < INFINITY))
    return set_error(FM_ERR_INVALID, "token_logprobs: the temperature's reciprocal is past fp32's range");
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
  a.t = temperature;
  a.c = LP_LOG2E / temperature;
  a.lag = 8.0f / a.c;
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
  return dtype == FM_DT_F32 ? launch_logprobs<float>(a, pl.cluster, s) : launch_logprobs<__nv_bfloat16>(a, pl.cluster, s);
}
