// Causal attention of chunks of query rows (a prompt, a verified draft) over a
// paged key/value cache, with a sliding window and first tokens that stay
// visible.
//
// The queries of request r are its last positions: row i of n stands at
// p = length - n + i and sees the keys j <= p with p - j < window or j < sinks
// (every j <= p without a window).  Query head h reads kv head h / G.
//   out = sum_j w_j v_j,  w_j = exp(s_j - max s) / sum exp(s - max s)
#include "paged_cache.cuh"

namespace fm {
namespace {

constexpr int WA_ROWS = 256;  // (token, head of the group) rows of a CTA, in two tiles
constexpr int WA_KEYS = 128;  // keys of a tile

struct WindowArgs {
  CacheRef c;
  const uint8_t* q;  // bf16
  long long q_ts, q_hs;
  const int* cu;
  int T, H, G;
  float scale;  // softmax_scale * log2(e)
  int window, sinks;
  __nv_bfloat16* out;
  long long o_ts, o_hs;
  int tiles, splits;
  float* part;    // [splits][T][H][HD] unnormalised outputs, when splits > 1
  float2* stats;  // [splits][T][H] (maximum, sum), base-2 scores
  int* err;
};

// Row tile `tile` of the flattened batch: request and its tile, or request -1.
// Request r has ceil(n_r G / ROWS) tiles; the search runs by one warp.
__device__ __forceinline__ int2 find_tile(const int* cu, int R, int G, int rows, int tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int r0 = 0; r0 < R; r0 += 32) {
    const int r = r0 + lane;
    int n = r < R ? (int)(((long long)max(0, cu[r + 1] - cu[r]) * G + rows - 1) / rows) : 0;
    int scan = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, off);
      if (lane >= off) scan += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + scan > tile);
    if (hit) {
      const int w = __ffs(hit) - 1;
      const int first = __shfl_sync(0xffffffffu, before + scan - n, w);
      return make_int2(r0 + w, tile - first);
    }
    before += __shfl_sync(0xffffffffu, scan, 31);
  }
  return make_int2(-1, 0);
}

// ----------------------------------------------------------------- tensor memory
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] B[smem], 16-bit operands, fp32 accumulate
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of a B operand stored row by row of K (a key's values): rows of
// 128 bytes (64 columns of N) with 128-byte swizzling, 8 keys to a 1024-byte
// atom; the next 64 columns follow `block` bytes on.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t block) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(block >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16 with both operands f16 (half) or both bf16, D fp32
__host__ __device__ constexpr uint32_t wa_idesc(bool half, int M, int N, bool b_mn) {
  return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Shared memory: two row tiles of Q, a ring of K and V tiles (16-bit, 128-byte
// swizzled in blocks of 64 columns), for e4m3 caches two tiles of raw bytes.
template <int HD, bool KV8>
struct WaLayout {
  static constexpr int TILE = 128 * HD * 2;  // Q, K or V tile
  static constexpr int SLOTS = HD == 64 ? 8 : KV8 ? 4 : 5;
  static constexpr int RAW = KV8 ? 128 * HD : 0;
  static constexpr int RAWS = KV8 ? 2 : 0;
  static constexpr int LAG = KV8 ? 0 : 2;  // tiles of copies in flight behind the newest
  static constexpr int CTRL = 2 * TILE + SLOTS * TILE + RAWS * RAW;
  static constexpr int SMEM = 1024 + CTRL + 2048;
};

struct WaCtrl {
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_ready[2], o_done[2], q_full, drain;
  int abort;
  uint32_t tmem;
  uint32_t valid[8][4];  // keys of tile j (mod 8) whose page exists
  float qinv[256];       // e4m3: what a row's query was multiplied with, inverted
};

// 16 warps: two warpgroups of softmax (one to a row tile of 128), one that
// loads, and one whose first warp issues the products.  S = Q K^T goes to
// tensor memory; the softmax threads (one to a row) turn it into P in place,
// which is the next product's A operand.  While one row tile is in softmax the
// tensor cores work on the other.
template <int HD, bool KV8>
__global__ void __launch_bounds__(512, 1) window_attn_kernel(WindowArgs a) {
  using Lay = WaLayout<HD, KV8>;
  constexpr int TILE = Lay::TILE, SLOTS = Lay::SLOTS;
  constexpr int CPR = HD / 8;  // 16-byte chunks of a 16-bit row
  extern __shared__ __align__(1024) uint8_t wa_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // the row tile, the latest rows (those with the most keys) first
  const int bid = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int c = bid % a.c.KH;
  const int2 at = find_tile(a.cu, a.c.R, a.G, WA_ROWS, a.tiles - 1 - bid / a.c.KH);
  if (at.x < 0) return;
  const int r = at.x, q0 = a.cu[r], nq = a.cu[r + 1] - q0;
  if (q0 < 0 || nq < 0 || q0 + nq > a.T) {
    if (tid == 0) record_error(a.err, DEV_BAD_INDEX);
    return;
  }
  const int len = cache_length(a.c, r, a.err, tid == 0);
  const int row0 = at.y * WA_ROWS, rows = min(WA_ROWS, nq * a.G - row0);
  const int pos0 = len - nq;  // position of the request's first query row (negative: it sees nothing)
  const int p_lo = pos0 + row0 / a.G, p_hi = pos0 + (row0 + rows - 1) / a.G;
  const int mt = rows > 128 ? 2 : 1;

  // key tiles: those of the first tokens, then those from the first row's window on
  const int lo = a.window > 0 ? max(0, p_lo - a.window + 1) : 0;
  const int t_end = p_hi < 0 ? 0 : p_hi / WA_KEYS + 1;
  const int t_lo = lo / WA_KEYS;
  const int t_head = min((min(a.sinks, lo) + WA_KEYS - 1) / WA_KEYS, t_lo);
  const int total = max(0, t_head + t_end - t_lo);
  const int t_first = (int)((long long)total * split / a.splits);
  const int n = (int)((long long)total * (split + 1) / a.splits) - t_first;
  auto key0 = [&](int j) {  // first key of this CTA's tile j
    const int t = t_first + j;
    return (t < t_head ? t : t - t_head + t_lo) * WA_KEYS;
  };
  if (n <= 0) {  // nothing is seen
    if (a.splits == 1) {
      for (int i = tid; i < rows * CPR; i += 512) {
        const int row = row0 + i / CPR;
        *reinterpret_cast<uint4*>(a.out + (long long)(q0 + row / a.G) * a.o_ts +
                                  (long long)(c * a.G + row % a.G) * a.o_hs + (i % CPR) * 8) = make_uint4(0, 0, 0, 0);
      }
    } else {
      for (int i = tid; i < rows; i += 512) {
        const int row = row0 + i;
        a.stats[((long long)split * a.T + q0 + row / a.G) * a.H + c * a.G + row % a.G] = make_float2(-INFINITY, 0.0f);
      }
    }
    return;
  }

  uint8_t* base = wa_smem + ((1024 - (smem_u32(wa_smem) & 1023)) & 1023);
  uint8_t* sQ = base;
  uint8_t* sKV = base + 2 * TILE;
  uint8_t* sRaw = sKV + SLOTS * TILE;
  WaCtrl* ctl = reinterpret_cast<WaCtrl*>(base + Lay::CTRL);
  volatile int* abort = &ctl->abort;
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&ctl->full[i], 128);
      mbar_init(&ctl->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 2);
      mbar_init(&ctl->p_ready[i], 128);
      mbar_init(&ctl->o_done[i], 1);
    }
    mbar_init(&ctl->q_full, 256);
    mbar_init(&ctl->drain, 1);
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&ctl->tmem, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;

  float kd = 1.0f, vd = 1.0f;
  if (a.c.descales) {
    kd = a.c.descales[(long long)r * a.c.KH + c];
    vd = a.c.descales[(long long)(a.c.R + r) * a.c.KH + c];
  }
  // |scale| goes with the scores; its sign (or a zero scale) with the queries
  const float fscale = a.scale * kd;
  const float sgn = fscale > 0.0f ? 1.0f : fscale < 0.0f ? -1.0f : 0.0f;

  if (warp < 8) {
    regs_inc<192>();
    // ------------------------------------------------------------- queries
    {
      constexpr int RPI = 256 / CPR;  // rows at a time
      const int ch = tid % CPR;
#pragma unroll 4
      for (int i = 0; i < 256; i += RPI) {
        const int lr = i + tid / CPR;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (lr < rows) {
          const int row = row0 + lr;
          v = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) +
                                              (long long)(q0 + row / a.G) * a.q_ts +
                                              (long long)(c * a.G + row % a.G) * a.q_hs + ch * 8);
        }
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
        if constexpr (KV8) {
          float amax = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
#pragma unroll
          for (int off = 1; off < CPR; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
          const float f = half_row_scale(amax);
          if (ch == 0) ctl->qinv[lr] = 1.0f / f;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pack16(__uint_as_float(w[e] << 16) * f, __uint_as_float(w[e] & 0xffff0000u) * f, true);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = sgn > 0.0f ? w[e] : sgn < 0.0f ? w[e] ^ 0x80008000u : 0u;
        const int r128 = lr & 127;
        *reinterpret_cast<uint4*>(sQ + (lr >> 7) * TILE + (ch >> 3) * 16384 + r128 * 128 +
                                  (((ch & 7) ^ (r128 & 7)) << 4)) = v;
      }
      fence_async_smem();
      mbar_arrive(&ctl->q_full);
    }
    // ------------------------------------------------------------- softmax
    const int i = warp >> 2;  // row tile
    if (i < mt) {
      const int lr = i * 128 + (tid & 127), row = row0 + lr;
      const bool live = lr < rows;
      // sees keys up to p (a row past the end stands where the last one does, and is not written),
      const int p = pos0 + (live ? row : row0 + rows - 1) / a.G;
      const int wlo = a.window > 0 ? p - a.window + 1 : 0;  // from wlo on or below sinks
      float sc = sgn == 0.0f ? 1.0f : fabsf(fscale);
      if constexpr (KV8) {
        if (!mbar_wait(&ctl->q_full, 0, abort)) *abort = 1;  // the rows' factors are written
        sc *= ctl->qinv[lr];
      }
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const uint32_t tS = tmem + lanes + i * 128, tO = tmem + lanes + 256 + i * 128;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        if (!mbar_wait(&ctl->s_full[i], j & 1, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_x32(tS + q * 32, s + q * 32);
        const int j0 = key0(j);
        uint32_t vm[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) vm[q] = ctl->valid[j & 7][q];
        tmem_wait_ld();
        const bool all = p >= j0 + 127 && (j0 >= wlo || j0 + 127 < a.sinks) && (vm[0] & vm[1] & vm[2] & vm[3]) == ~0u;
        if (!__all_sync(0xffffffffu, all)) {
          const int np = p - j0 + 1, nw = wlo - j0, ns = a.sinks - j0;  // seen: c < np, and c >= nw or c < ns
          auto low = [](int x) { return x <= 0 ? 0u : x >= 32 ? ~0u : (1u << x) - 1u; };
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t bits = low(np - 32 * q) & (~low(nw - 32 * q) | low(ns - 32 * q)) & vm[q];
#pragma unroll
            for (int e = 0; e < 32; ++e) s[q * 32 + e] = (bits >> e) & 1u ? s[q * 32 + e] : -INFINITY;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 128; ++e) mx[e & 3] = fmaxf(mx[e & 3], s[e]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        // The subtracted maximum may lag behind the true one by a factor 2^8:
        // the numerators stay far inside their type's range, the division by
        // the sum takes the factor out, and O is seldom rescaled.
        const float mn = top > m + 8.0f || m == -INFINITY ? fmaxf(m, top) : m;
        if (__any_sync(0xffffffffu, mn != m)) {
          const float f = m == mn ? 1.0f : ex2(m - mn);
          if (j > 0) {  // S is complete, so the product before it, P V of tile j - 1, is too
#pragma unroll
            for (int q = 0; q < HD / 16; ++q) {
              float o[16];
              tmem_ld_x16(tO + q * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              tmem_st_x16(tO + q * 16, o);
            }
          }
          l *= f;
          m = mn;
        }
        const float neg = m == -INFINITY ? 0.0f : -m;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float p0 = ex2(fmaf(s[q * 64 + 2 * e], sc, neg)), p1 = ex2(fmaf(s[q * 64 + 2 * e + 1], sc, neg));
            acc[2 * (e & 1)] += p0;
            acc[2 * (e & 1) + 1] += p1;
            w[e] = pack16(p0, p1, KV8);
          }
          tmem_st_x32(tS + q * 32, w);
        }
        l += (acc[0] + acc[1]) + (acc[2] + acc[3]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->p_ready[i]);
      }
      if (ok && !mbar_wait(&ctl->o_done[i], 0, abort)) ok = false;
      if (!ok) {
        *abort = 1;
        record_error(a.err, DEV_TIMEOUT_ACC);
      } else {
        tc_fence_after();
        const int tok = q0 + (live ? row / a.G : 0), h = c * a.G + (live ? row % a.G : 0);
        const float inv = l == 0.0f ? 0.0f : vd / l;  // a row that sees nothing is zero
        const bool whole = a.splits == 1;
        float* part = whole ? nullptr : a.part + (((long long)split * a.T + tok) * a.H + h) * HD;
        __nv_bfloat16* out = a.out + (long long)tok * a.o_ts + (long long)h * a.o_hs;
        if (live && !whole) a.stats[((long long)split * a.T + tok) * a.H + h] = make_float2(m, l);
#pragma unroll
        for (int q = 0; q < HD / 32; ++q) {
          float o[32];
          tmem_ld_x32(tO + q * 32, o);
          tmem_wait_ld();
          if (!live) continue;
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 w;
              w.x = pack16(o[e] * inv, o[e + 1] * inv, false);
              w.y = pack16(o[e + 2] * inv, o[e + 3] * inv, false);
              w.z = pack16(o[e + 4] * inv, o[e + 5] * inv, false);
              w.w = pack16(o[e + 6] * inv, o[e + 7] * inv, false);
              *reinterpret_cast<uint4*>(out + q * 32 + e) = w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + q * 32 + e) =
                  make_float4(o[e] * vd, o[e + 1] * vd, o[e + 2] * vd, o[e + 3] * vd);
          }
        }
        tc_fence_before();
      }
    }
  } else if (warp < 12) {
    regs_dec<64>();
    // ------------------------------------------------------------- keys and values
    const int lw = warp - 8;  // rows 32 lw .. 32 lw + 31 of every tile
    const long long trow = (long long)r * a.c.tstride;
    auto lookup = [&](int j, int* tok) {  // page of this lane's key of tile j; -1: none, -2: a bad one
      if (j >= n) return -1;
      const int k = key0(j) + lw * 32 + lane;
      if (k > p_hi || !(k >= lo || k < a.sinks)) return -1;
      const int pg = k / a.c.page;
      *tok = k - pg * a.c.page;
      const int page = a.c.table[trow + pg];
      if (page >= 0 && page < a.c.num_pages) return page;
      record_error(a.err, DEV_BAD_INDEX);
      return -2;
    };
    int tok = 0, tok_next = 0, page = -1, page_next = lookup(0, &tok_next);
    bool ok = true;
    const int items = 2 * n;
    for (int q = 0; q < items + Lay::LAG + (KV8 ? 1 : 0); ++q) {
      // ---- issue item q (K and V of a tile in turn)
      if (q < items) {
        const int slot = q % SLOTS;
        if (!KV8 && q >= SLOTS && ok && !mbar_wait(&ctl->empty[slot], (q / SLOTS - 1) & 1, abort)) ok = false;
        if (!ok) break;
        const bool is_v = q & 1;
        if (!is_v) {
          page = page_next;
          tok = tok_next;
          page_next = lookup(q / 2 + 1, &tok_next);
          const uint32_t good = __ballot_sync(0xffffffffu, page != -2);
          if (lane == 0) ctl->valid[(q / 2) & 7][lw] = good;
        }
        const uint8_t* src = is_v ? a.c.v : a.c.k;
        long long off = -1;
        if (page >= 0)
          off = is_v ? page * a.c.vps + (long long)c * a.c.vhs + (long long)tok * a.c.vts
                     : page * a.c.kps + (long long)c * a.c.khs + (long long)tok * a.c.kts;
        constexpr int RC = KV8 ? HD / 16 : CPR;  // 16-byte chunks of a cache row
        constexpr int RPI = 32 / RC;
        const int ch = lane % RC;
        const uint32_t dst = KV8 ? smem_u32(sRaw) + (q & 1) * Lay::RAW + lw * 32 * HD
                                 : smem_u32(sKV) + slot * TILE + (ch >> 3) * 16384 + lw * 32 * 128;
#pragma unroll 4
        for (int u = 0; u < 32 / RPI; ++u) {
          const int row = u * RPI + lane / RC;
          const long long o = __shfl_sync(0xffffffffu, off, row);
          // keys that no row sees are zero: what the cache holds there may be no number
          pc_cp_async16(KV8 ? dst + row * HD + ch * 16 : dst + row * 128 + (((ch & 7) ^ (row & 7)) << 4),
                        src + (o < 0 ? 0 : o + ch * 16), o < 0 ? 0u : 16u);
        }
      }
      pc_cp_commit();
      if constexpr (KV8) {
        // ---- widen item q - 1, which this warp copied: e4m3 is exact in f16
        const int d = q - 1;
        if (d >= 0) {
          const int slot = d % SLOTS;
          pc_cp_wait<1>();
          __syncwarp();
          if (d >= SLOTS && !mbar_wait(&ctl->empty[slot], (d / SLOTS - 1) & 1, abort)) {
            ok = false;
            break;
          }
          constexpr int RC = HD / 16, RPI = 32 / RC;
          const int ch = lane % RC, odd = (ch >> 2) & 1;  // which half first: no two lanes of a row share a bank
          const uint8_t* raw = sRaw + (d & 1) * Lay::RAW + lw * 32 * HD;
          uint8_t* dst = sKV + slot * TILE + (ch >> 2) * 16384;
#pragma unroll 4
          for (int u = 0; u < 32 / RPI; ++u) {
            const int row = u * RPI + lane / RC, r128 = lw * 32 + row;
            const uint4 x = *reinterpret_cast<const uint4*>(raw + row * HD + ch * 16);
            const uint4 h0 = make_uint4(e4m3x2_h(x.x & 0xffffu), e4m3x2_h(x.x >> 16), e4m3x2_h(x.y & 0xffffu),
                                        e4m3x2_h(x.y >> 16));
            const uint4 h1 = make_uint4(e4m3x2_h(x.z & 0xffffu), e4m3x2_h(x.z >> 16), e4m3x2_h(x.w & 0xffffu),
                                        e4m3x2_h(x.w >> 16));
            uint8_t* drow = dst + r128 * 128;
            const int c0 = (2 * ch) & 7;
            *reinterpret_cast<uint4*>(drow + (((c0 + odd) ^ (r128 & 7)) << 4)) = odd ? h1 : h0;
            *reinterpret_cast<uint4*>(drow + (((c0 + 1 - odd) ^ (r128 & 7)) << 4)) = odd ? h0 : h1;
          }
          __syncwarp();  // the raw rows may be overwritten from here on
          fence_async_smem();
          mbar_arrive(&ctl->full[slot]);
        }
      } else {
        // ---- item q - LAG has arrived: hand it to the tensor cores
        const int d = q - Lay::LAG;
        if (d >= 0) {
          pc_cp_wait<Lay::LAG>();
          fence_async_smem();
          mbar_arrive(&ctl->full[d % SLOTS]);
        }
      }
    }
    pc_cp_wait<0>();
    if (!ok) {
      *abort = 1;
      record_error(a.err, DEV_TIMEOUT_EMPTY);
    }
  } else {
    regs_dec<64>();
    if (warp == 12 && lane == 0) {
      // ------------------------------------------------------------- products
      constexpr uint32_t ID_S = wa_idesc(KV8, 128, 128, false), ID_O = wa_idesc(KV8, 128, HD, true);
      auto product_s = [&](int i, int slot) {
        const uint32_t qa = smem_u32(sQ) + i * TILE, kb = smem_u32(sKV) + slot * TILE;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
          umma_bf16(tmem + i * 128, sdesc_k_sw128(qa + off), sdesc_k_sw128(kb + off), ID_S, k > 0);
        }
        mbar_arrive(&ctl->s_full[i]);  // the keys' validity words, too, are there
        umma_commit(&ctl->s_full[i]);
      };
      auto product_o = [&](int i, int slot, bool first) {
        const uint32_t vb = smem_u32(sKV) + slot * TILE;
#pragma unroll
        for (int k = 0; k < WA_KEYS / 16; ++k)
          umma_ts(tmem + 256 + i * 128, tmem + i * 128 + k * 8, sdesc_mn_sw128(vb + k * 2048, 16384), ID_O,
                  !first || k > 0);
      };
      int code = 0;
      if (!mbar_wait(&ctl->q_full, 0, abort) || !mbar_wait(&ctl->full[0], 0, abort)) code = DEV_TIMEOUT_FULL;
      if (!code) {
        tc_fence_after();
        for (int i = 0; i < mt; ++i) product_s(i, 0);
        umma_commit(&ctl->empty[0]);
      }
      for (int j = 0; j < n && !code; ++j) {
        const int qv = 2 * j + 1, qk = 2 * j + 2;
        const bool more = j + 1 < n;
        if (!mbar_wait(&ctl->full[qv % SLOTS], (qv / SLOTS) & 1, abort)) code = DEV_TIMEOUT_FULL;
        for (int i = 0; i < mt && !code; ++i) {
          if (!mbar_wait(&ctl->p_ready[i], j & 1, abort)) {
            code = DEV_TIMEOUT_ACC;
            break;
          }
          tc_fence_after();
          product_o(i, qv % SLOTS, j == 0);
          if (i == mt - 1) umma_commit(&ctl->empty[qv % SLOTS]);
          if (!more) {
            umma_commit(&ctl->o_done[i]);
            continue;
          }
          if (i == 0 && !mbar_wait(&ctl->full[qk % SLOTS], (qk / SLOTS) & 1, abort)) {
            code = DEV_TIMEOUT_FULL;
            break;
          }
          product_s(i, qk % SLOTS);
          if (i == mt - 1) umma_commit(&ctl->empty[qk % SLOTS]);
        }
      }
      if (code) {
        *abort = 1;
        record_error(a.err, code);
        umma_commit(&ctl->drain);  // nothing of this CTA may be in flight when it ends
        mbar_wait(&ctl->drain, 0, nullptr);
      }
    }
  }
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// A row's splits joined, one warp to a row (token, head).
template <int HD>
__global__ void __launch_bounds__(128) window_join_kernel(WindowArgs a) {
  pdl_wait();
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), rows = (long long)a.T * a.H;
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float top = -INFINITY;
  for (int z = 0; z < a.splits; ++z) top = fmaxf(top, a.stats[z * rows + row].x);
  const float u = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, o[HD / 32];
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) o[e] = 0.0f;
  for (int z = 0; z < a.splits; ++z) {
    const float2 st = a.stats[z * rows + row];
    if (st.x == -INFINITY && st.y == 0.0f) continue;  // saw nothing: its output was not written
    const float f = ex2(st.x - u);
    sum += st.y * f;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) o[e] += a.part[(z * rows + row) * HD + lane * (HD / 32) + e] * f;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  __nv_bfloat16* out = a.out + (row / a.H) * a.o_ts + (row % a.H) * a.o_hs + lane * (HD / 32);
#pragma unroll
  for (int e = 0; e < HD / 32; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack16(o[e] * inv, o[e + 1] * inv, false);
}

struct WindowPlan {
  int64_t tiles;
  int splits;
  size_t part, total;
};
// Row tiles (every request ends in one of its own at most), and the splits of
// their keys: as many as give two CTAs to an SM, of 512 keys at least.
WindowPlan window_plan(int64_t R, int64_t T, int64_t H, int64_t KH, int64_t HD, int64_t max_q, int64_t max_len,
                       int64_t window, int64_t sinks) {
  WindowPlan p{};
  p.tiles = (T * (H / KH) + WA_ROWS - 1) / WA_ROWS + R;
  int64_t span = max_len;
  if (window > 0 && window + max_q + sinks < span) span = window + max_q + sinks;
  const int64_t want = (2 * 148 + p.tiles * KH - 1) / (p.tiles * KH), most = span / 512;
  p.splits = (int)(want < most ? want : most);
  if (p.splits < 1) p.splits = 1;
  if (p.splits > 1) {
    p.part = (size_t)p.splits * T * H * HD * 4;
    p.total = p.part + (size_t)p.splits * T * H * 8;
  }
  return p;
}

template <int HD, bool KV8>
fm_status launch_window(const WindowArgs& a, cudaStream_t s) {
  constexpr int smem = WaLayout<HD, KV8>::SMEM;
  static_assert(sizeof(WaCtrl) <= 2048 && smem <= 232448, "shared memory");
  fm_status st = check_cuda(
      cudaFuncSetAttribute(window_attn_kernel<HD, KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
      "paged_window_attn");
  if (st != FM_OK) return st;
  st = launch_kernel(window_attn_kernel<HD, KV8>, dim3((unsigned)(a.tiles * a.c.KH * a.splits)), dim3(512), smem, s,
                     false, a);
  if (st != FM_OK || a.splits == 1) return st;
  return launch_kernel(window_join_kernel<HD>, dim3((unsigned)(((long long)a.T * a.H + 3) / 4)), dim3(128), 0, s, true,
                       a);
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_paged_window_attn_workspace_size(int64_t requests, int64_t rows, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_q, int64_t max_length,
                                                      int64_t window, int64_t sinks) {
  if (requests < 1 || rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || max_q < 0 || max_length < 0 ||
      window < 0 || sinks < 0)
    return 0;
  return window_plan(requests, rows, heads, kv_heads, head_dim, max_q, max_length, window, sinks).total;
}

extern "C" fm_status fm_paged_window_attn(const fm_paged_cache* cache, const fm_window_attn* p, fm_stream stream) {
  WindowArgs a{};
  fm_status st = cache_ref(cache, "paged_window_attn", &a.c);
  if (st != FM_OK) return st;
  if (!p) return set_error(FM_ERR_INVALID, "paged_window_attn: null arguments");
  if (p->heads < 1 || p->heads % cache->kv_heads || p->heads > 65535)
    return set_error(FM_ERR_SHAPE, "paged_window_attn: query heads must be a multiple of the kv heads");
  if (p->window < 0 || p->sinks < 0 || p->window > 0x7ffffff0 || p->sinks > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "paged_window_attn: window and sinks must not be negative");
  if (p->rows < 0 || p->rows * p->heads > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "paged_window_attn: too many query rows");
  if (cache->requests == 0 || p->rows == 0) return FM_OK;
  if (!p->q || !p->out || !p->cu_seqlens_q) return set_error(FM_ERR_INVALID, "paged_window_attn: null pointer");
  if ((uintptr_t)p->q % 16 || p->q_token_stride % 8 || p->q_head_stride % 8 || (uintptr_t)p->out % 16 ||
      p->out_token_stride % 8 || p->out_head_stride % 8)
    return set_error(FM_ERR_ALIGN, "paged_window_attn: query and output rows must be 16-byte aligned");
  a.q = static_cast<const uint8_t*>(p->q);
  a.q_ts = p->q_token_stride;
  a.q_hs = p->q_head_stride;
  a.cu = p->cu_seqlens_q;
  a.T = (int)p->rows;
  a.H = (int)p->heads;
  a.G = (int)(p->heads / cache->kv_heads);
  a.scale = p->softmax_scale * kLog2e;
  a.window = (int)p->window;
  a.sinks = (int)p->sinks;
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.o_ts = p->out_token_stride;
  a.o_hs = p->out_head_stride;
  a.err = p->err;
  const WindowPlan pl = window_plan(cache->requests, p->rows, p->heads, cache->kv_heads, cache->head_dim, p->max_q,
                                    cache->max_length, p->window, p->sinks);
  if (pl.total > p->workspace_bytes || (pl.total && !p->workspace))
    return set_error(FM_ERR_WORKSPACE, "paged_window_attn: workspace %zu < %zu", p->workspace_bytes, pl.total);
  if ((uintptr_t)p->workspace % 16) return set_error(FM_ERR_ALIGN, "paged_window_attn: workspace not 16-byte aligned");
  if (pl.tiles * cache->kv_heads * pl.splits > 0x7fffffff)
    return set_error(FM_ERR_SHAPE, "paged_window_attn: grid too large");
  a.tiles = (int)pl.tiles;
  a.splits = pl.splits;
  a.part = static_cast<float*>(p->workspace);
  a.stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(p->workspace) + pl.part);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool kv8 = cache->dtype == FM_DT_E4M3;
  if (cache->head_dim == 128) return kv8 ? launch_window<128, true>(a, s) : launch_window<128, false>(a, s);
  return kv8 ? launch_window<64, true>(a, s) : launch_window<64, false>(a, s);
}
