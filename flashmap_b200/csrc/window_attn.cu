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

constexpr int WA_ROWS = 64;  // (token, head of the group) rows of a CTA, 16 to a warp
constexpr int WA_KEYS = 64;  // keys of a tile

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

template <int HD, bool KV8>
__global__ void __launch_bounds__(128) window_attn_kernel(WindowArgs a) {
  constexpr int RB = HD * (KV8 ? 1 : 2), PART = WA_KEYS * RB, KS = HD / 16, NT = HD / 8;
  extern __shared__ __align__(1024) uint8_t wa_smem[];
  __shared__ int spage[2][WA_KEYS], stok[2][WA_KEYS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int c = blockIdx.y;
  const int2 at = find_tile(a.cu, a.c.R, a.G, WA_ROWS, blockIdx.x);
  if (at.x < 0) return;
  const int r = at.x, q0 = a.cu[r], nq = a.cu[r + 1] - q0;
  if (q0 < 0 || nq < 0 || q0 + nq > a.T) {
    if (threadIdx.x == 0) record_error(a.err, DEV_BAD_INDEX);
    return;
  }
  const int len = cache_length(a.c, r, a.err, threadIdx.x == 0);
  const int row0 = at.y * WA_ROWS, rows = nq * a.G;
  const int pos0 = len - nq;  // position of the request's first query row (negative: it sees nothing)
  const int p_lo = pos0 + row0 / a.G, p_hi = pos0 + (min(row0 + WA_ROWS, rows) - 1) / a.G;

  float kd = 1.0f, vd = 1.0f;
  if (a.c.descales) {
    kd = a.c.descales[(long long)r * a.c.KH + c];
    vd = a.c.descales[(long long)(a.c.R + r) * a.c.KH + c];
  }
  // this lane's two rows, gid and gid + 8 of the warp's sixteen
  int p[2];
  bool live[2];
  long long qoff[2], ooff[2];
  float sscale[2];
  uint32_t qa[KS][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = row0 + warp * 16 + gid + 8 * e;
    live[e] = row < rows;
    const int tok = live[e] ? row / a.G : 0, h = c * a.G + (live[e] ? row % a.G : 0);
    p[e] = live[e] ? pos0 + tok : -1;
    qoff[e] = (long long)(q0 + tok) * a.q_ts + (long long)h * a.q_hs;
    ooff[e] = (long long)(q0 + tok) * a.o_ts + (long long)h * a.o_hs;
    const __nv_bfloat16* qr = reinterpret_cast<const __nv_bfloat16*>(a.q) + qoff[e];
    float amax = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int col = ks * 16 + (KV8 ? tig * 4 + f * 2 : tig * 2 + f * 8);
        const uint32_t v = live[e] ? *reinterpret_cast<const uint32_t*>(qr + col) : 0u;
        qa[ks][e + 2 * f] = v;
        if constexpr (KV8)
          amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(v << 16)), fabsf(__uint_as_float(v & 0xffff0000u))));
      }
    sscale[e] = a.scale * kd;
    if constexpr (KV8) {
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float f = half_row_scale(amax);
      sscale[e] = sscale[e] / f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t v = qa[ks][e + 2 * g];
          qa[ks][e + 2 * g] = pack16(__uint_as_float(v << 16) * f, __uint_as_float(v & 0xffff0000u) * f, true);
        }
    }
  }

  // key tiles: those of the first tokens, then those from the first row's window on
  const int lo = a.window > 0 ? max(0, p_lo - a.window + 1) : 0;
  const int t_end = p_hi < 0 ? 0 : p_hi / WA_KEYS + 1;
  const int t_lo = lo / WA_KEYS;
  const int t_head = min((min(a.sinks, lo) + WA_KEYS - 1) / WA_KEYS, t_lo);
  const int ntiles = max(0, t_head + t_end - t_lo);
  auto tile_at = [&](int t) { return t < t_head ? t : t - t_head + t_lo; };

  const uint32_t sbase = smem_u32(wa_smem);
  auto lookup = [&](int t) {  // pages of tile t's keys, 64 threads
    if (t < ntiles && threadIdx.x < WA_KEYS) {
      const int j = tile_at(t) * WA_KEYS + threadIdx.x;
      int page = -1, tok = 0;
      if (j < len && j <= p_hi && (j >= lo || j < a.sinks)) {
        const int pg = j / a.c.page;
        tok = j - pg * a.c.page;
        page = a.c.table[(long long)r * a.c.tstride + pg];
        if (page < 0 || page >= a.c.num_pages) {
          record_error(a.err, DEV_BAD_INDEX);
          page = -1;
        }
      }
      spage[t & 1][threadIdx.x] = page;
      stok[t & 1][threadIdx.x] = tok;
    }
  };
  auto issue = [&](int t) {
    if (t < ntiles) {
      const uint32_t dst0 = sbase + (t & 1) * 2 * PART;
      constexpr int CPR = RB / 16;
      for (int i = threadIdx.x; i < WA_KEYS * CPR; i += 128) {
        const int row = i / CPR, ch = i % CPR;
        const long long pg = spage[t & 1][row], tk = stok[t & 1][row];
        const uint8_t* ks = a.c.k;
        const uint8_t* vs = a.c.v;
        if (pg >= 0) {
          ks += pg * a.c.kps + (long long)c * a.c.khs + tk * a.c.kts + ch * 16;
          vs += pg * a.c.vps + (long long)c * a.c.vhs + tk * a.c.vts + ch * 16;
        }
        const uint32_t dst = dst0 + row_sw<RB>(row, ch);
        pc_cp_async16(dst, ks, pg >= 0 ? 16u : 0u);
        pc_cp_async16(dst + PART, vs, pg >= 0 ? 16u : 0u);
      }
    }
    pc_cp_commit();
  };

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  lookup(0);
  __syncthreads();
  issue(0);
  lookup(1);
  for (int t = 0; t < ntiles; ++t) {
    __syncthreads();  // tile t - 1 is consumed, tile t + 1's pages are known
    issue(t + 1);
    pc_cp_wait<1>();
    __syncthreads();
    const uint32_t kb0 = sbase + (t & 1) * 2 * PART, vb0 = kb0 + PART;
    float sc[WA_KEYS / 8][4];
#pragma unroll
    for (int nt = 0; nt < WA_KEYS / 8; ++nt) {
      sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
      const int kr = nt * 8 + (lane & 7);
      if constexpr (KV8) {
#pragma unroll
        for (int k4 = 0; k4 < KS; k4 += 4) {
          uint32_t b[4];
          ldsm4(kb0 + row_sw<RB>(kr, k4 + (lane >> 3)), b);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mma16816<true>(sc[nt], qa[k4 + e][0], qa[k4 + e][1], qa[k4 + e][2], qa[k4 + e][3],
                           e4m3x2_h(b[e] & 0xffffu), e4m3x2_h(b[e] >> 16));
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          uint32_t b[4];
          ldsm4(kb0 + row_sw<RB>(kr, 2 * ks + (lane >> 3)), b);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            mma16816<false>(sc[nt], qa[ks + e][0], qa[ks + e][1], qa[ks + e][2], qa[ks + e][3], b[2 * e],
                            b[2 * e + 1]);
        }
      }
    }
    const int j0 = tile_at(t) * WA_KEYS;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < WA_KEYS / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + nt * 8 + tig * 2 + (e & 1), pe = p[e >> 1];
        const bool see = j <= pe && (a.window <= 0 || pe - j < a.window || j < a.sinks) &&
                         spage[t & 1][nt * 8 + tig * 2 + (e & 1)] >= 0;
        sc[nt][e] = see ? sc[nt][e] * sscale[e >> 1] : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], sc[nt][e]);
      }
    uint32_t pa[WA_KEYS / 16][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
      mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      const float mn = fmaxf(m[e], mx[e]), u = mn == -INFINITY ? 0.0f : mn;
      const float al = exp2f(m[e] - u);
      m[e] = mn;
      l[e] *= al;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][2 * e] *= al;
        o[i][2 * e + 1] *= al;
      }
#pragma unroll
      for (int nt = 0; nt < WA_KEYS / 8; ++nt) {
        const float p0 = exp2f(sc[nt][2 * e] - u), p1 = exp2f(sc[nt][2 * e + 1] - u);
        l[e] += p0 + p1;
        pa[nt / 2][e + 2 * (nt & 1)] = pack16(p0, p1, KV8);
      }
    }
#pragma unroll
    for (int k = 0; k < WA_KEYS / 16; ++k) {
      const int vr = k * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
      if constexpr (KV8) {
        // byte pairs: columns 2 gid and 2 gid + 1 of a sixteen go to its two products
#pragma unroll
        for (int i = 0; i < HD / 16; i += 2) {
          uint32_t b[4];
          ldsm4_t(vb0 + row_sw<RB>(vr, i + (lane >> 4)), b);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t x = b[2 * e], y = b[2 * e + 1];
            mma16816<true>(o[2 * (i + e)], pa[k][0], pa[k][1], pa[k][2], pa[k][3],
                           e4m3x2_h(__byte_perm(x, 0, 0x4420)), e4m3x2_h(__byte_perm(y, 0, 0x4420)));
            mma16816<true>(o[2 * (i + e) + 1], pa[k][0], pa[k][1], pa[k][2], pa[k][3],
                           e4m3x2_h(__byte_perm(x, 0, 0x4431)), e4m3x2_h(__byte_perm(y, 0, 0x4431)));
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
          uint32_t b[4];
          ldsm4_t(vb0 + row_sw<RB>(vr, i + (lane >> 4)), b);
          mma16816<false>(o[i], pa[k][0], pa[k][1], pa[k][2], pa[k][3], b[0], b[1]);
          mma16816<false>(o[i + 1], pa[k][0], pa[k][1], pa[k][2], pa[k][3], b[2], b[3]);
        }
      }
    }
    __syncthreads();  // spage of tile t is read
    lookup(t + 2);
  }
  pc_cp_wait<0>();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (!live[e]) continue;
    const float inv = l[e] == 0.0f ? 0.0f : vd / l[e];  // a row that sees nothing is zero
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if constexpr (KV8) {
        // products 2 i and 2 i + 1 hold the even and odd columns of a sixteen
        const int col = (i >> 1) * 16 + 2 * (tig * 2) + (i & 1);
        a.out[ooff[e] + col] = f2bf(o[i][2 * e] * inv);
        a.out[ooff[e] + col + 2] = f2bf(o[i][2 * e + 1] * inv);
      } else {
        *reinterpret_cast<uint32_t*>(a.out + ooff[e] + i * 8 + tig * 2) =
            pack16(o[i][2 * e] * inv, o[i][2 * e + 1] * inv, false);
      }
    }
  }
}

template <int HD, bool KV8>
fm_status launch_window(const WindowArgs& a, unsigned tiles, cudaStream_t s) {
  constexpr int smem = 4 * WA_KEYS * HD * (KV8 ? 1 : 2);
  fm_status st = check_cuda(
      cudaFuncSetAttribute(window_attn_kernel<HD, KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
      "paged_window_attn");
  if (st != FM_OK) return st;
  return launch_kernel(window_attn_kernel<HD, KV8>, dim3(tiles, a.c.KH), dim3(128), smem, s, false, a);
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_paged_window_attn_workspace_size(int64_t requests, int64_t rows, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_q, int64_t max_length,
                                                      int64_t window, int64_t sinks) {
  (void)requests, (void)rows, (void)heads, (void)kv_heads, (void)head_dim, (void)max_q, (void)max_length;
  (void)window, (void)sinks;
  return 0;
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
  // every request ends in one tile of its own at most
  const int64_t tiles = (p->rows * a.G + WA_ROWS - 1) / WA_ROWS + cache->requests;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool kv8 = cache->dtype == FM_DT_E4M3;
  if (cache->head_dim == 128)
    return kv8 ? launch_window<128, true>(a, (unsigned)tiles, s) : launch_window<128, false>(a, (unsigned)tiles, s);
  return kv8 ? launch_window<64, true>(a, (unsigned)tiles, s) : launch_window<64, false>(a, (unsigned)tiles, s);
}
