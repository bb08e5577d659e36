// Attention of one new token per request over a paged key/value cache.
//
// For request r and query head h of the group that shares kv head c, over the
// positions j that the token sees:
//   s_j = scale q_h . k_j,  w_j = exp(s_j - max s) / sum exp(s - max s),
//   out_h = sum_j w_j v_j,  and, when asked for, sums[r, c, j] += sum over the
// group's heads of w_j.
//
// The keys and values are read once and each takes part in 4 G operations a
// byte at most (G query heads to a kv head), so the cache's bytes bound it.
// A request's visible positions are cut into equal chunks, one CTA per (chunk,
// request, kv head, 8 or 16 query heads), so that one long request fills the
// GPU.  Each of a CTA's four warps streams its own 16-key tiles through a
// cp.async pipeline, with its own running maximum and sum, and the warps are
// merged at the end.  Chunks are joined by a second kernel
// (decode_join_kernel), which also turns the scores that the first one left
// into weights, since only then are a row's maximum and sum known.
//
// Measured, 32 heads on 8 of 128: 1 request of 49157, 44 us (4.6 TB/s, of which
// 6 us are the join); 64 requests of 1024 .. 8192 with sums, 225 us (5.5 TB/s,
// the scores and the join included); 40 heads on 8, e4m3, 192 requests of
// 512 .. 4096, 192 us (4.7 TB/s: no unit is full, each warp waits on its own chain);
// 64 heads on 8 of 64, a window of 2048, 92 us (5.6 TB/s).
#include "paged_cache.cuh"

namespace fm {
namespace {

constexpr int DA_STAGES = 2;
constexpr int DA_TILE = 16;  // keys of a warp's tile

struct DecodeArgs {
  CacheRef c;
  const uint8_t* q;  // bf16
  long long q_rs, q_hs;  // elements
  int H, G, hgroups;     // heads, heads per kv head, CTAs' head groups per kv head
  float scale;           // softmax_scale * log2(e)
  int window, sinks;
  int least, chunks;     // keys of a chunk at least, chunks of an item at most
  __nv_bfloat16* out;
  long long o_rs, o_hs;
  float* sums;
  long long s_rs, s_hs;
  float* part;    // [R * H][chunks][HD] unnormalised outputs
  float2* stats;  // [R * H][chunks] (maximum, sum), base-2 scores
  float* scores;  // [R * H][pitch] base-2 scores, when sums are wanted
  int pitch;
  int* err;
};

// Keys of a chunk of n visible positions.  Up to DA_WHOLE stay one chunk, which
// needs no join (201 positions, 1 request: 5.2 us against 6.3 us in chunks of 128).
constexpr int DA_WHOLE = 256;
__device__ __forceinline__ int chunk_of(const DecodeArgs& a, int n) {
  if (n <= DA_WHOLE) return DA_WHOLE;
  const int even = (((n + a.chunks - 1) / a.chunks) + 63) & ~63;
  return even > a.least ? even : a.least;
}

template <int HD, bool KV8>
struct DaLayout {
  static constexpr int RB = HD * (KV8 ? 1 : 2);       // bytes of a key row
  static constexpr int PART = DA_TILE * RB;           // K or V of a tile
  static constexpr int WARP = DA_STAGES * 2 * PART;
  static constexpr int PIPE = 4 * WARP;
};

template <int HD, bool KV8, int NG>
constexpr int da_smem() {
  constexpr int merge = 4 * 8 * NG * (HD + 4) * 4 + 4 * 8 * NG * 8 + 8 * NG * 8;
  return (DaLayout<HD, KV8>::PIPE > merge ? DaLayout<HD, KV8>::PIPE : merge) + 4 * DA_STAGES * 4;
}

// NG: groups of 8 query heads (1 or 2).  Scores: S[heads][keys] = Q K^T with
// the heads as the 16 rows of the product; then O^T[d][heads] = V^T P^T, whose
// B operand is the scores' accumulator layout as it stands.
template <int HD, bool KV8, int NG>
__global__ void __launch_bounds__(128) decode_attn_kernel(DecodeArgs a) {
  using Lay = DaLayout<HD, KV8>;
  constexpr int RB = Lay::RB, MT = HD / 16, KS = HD / 16;
  extern __shared__ __align__(1024) uint8_t da_smem_buf[];
  // a uniform warp number spares the e4m3 kernel the registers that keep a fourth CTA off the SM
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  pdl_wait();
  const int items = a.c.R * a.c.KH * a.hgroups;
  const int chunk = blockIdx.x / items;
  int rest = blockIdx.x % items;
  const int hg = rest % a.hgroups;
  rest /= a.hgroups;
  const int c = rest % a.c.KH, r = rest / a.c.KH;
  const int h0 = c * a.G + hg * 8 * NG;                 // first query head
  const int nh = min(8 * NG, a.G - hg * 8 * NG);        // query heads of this CTA
  const int len = cache_length(a.c, r, a.err, threadIdx.x == 0 && chunk == 0);
  const Span sp = visible_span(len, a.window, a.sinks);
  const int size = chunk_of(a, sp.n);
  if ((long long)chunk * size >= sp.n) {
    if (chunk == 0)  // nothing to attend to: zero rows
      for (int i = threadIdx.x; i < nh * HD; i += 128)
        a.out[(long long)r * a.o_rs + (long long)(h0 + i / HD) * a.o_hs + i % HD] = f2bf(0.0f);
    return;
  }
  const int begin = chunk * size, end = min(sp.n, begin + size);

  float kd = 1.0f, vd = 1.0f;
  if (a.c.descales) {
    kd = a.c.descales[(long long)r * a.c.KH + c];
    vd = a.c.descales[(long long)(a.c.R + r) * a.c.KH + c];
  }

  // Query fragments: head h0 + gid (and + 8).  An 8-bit key row is read four
  // bytes to a lane, so there a lane holds columns 4 tig .. 4 tig + 3 of each
  // sixteen, and for 16-bit rows columns 2 tig, 2 tig + 1 and those plus 8.
  uint32_t qa[NG][KS][2];
  float sscale[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const bool live = gid + 8 * n < nh;
    const __nv_bfloat16* row =
        reinterpret_cast<const __nv_bfloat16*>(a.q) + (long long)r * a.q_rs + (long long)(h0 + (live ? gid + 8 * n : 0)) * a.q_hs;
    float amax = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int col = ks * 16 + (KV8 ? tig * 4 + f * 2 : tig * 2 + f * 8);
        qa[n][ks][f] = live ? *reinterpret_cast<const uint32_t*>(row + col) : 0u;
        if constexpr (KV8) {
          amax = fmaxf(amax, fabsf(__uint_as_float(qa[n][ks][f] << 16)));
          amax = fmaxf(amax, fabsf(__uint_as_float(qa[n][ks][f] & 0xffff0000u)));
        }
      }
    sscale[n] = a.scale * kd;
    if constexpr (KV8) {
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float f = half_row_scale(amax);
      sscale[n] = sscale[n] / f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qa[n][ks][e] = pack16(__uint_as_float(qa[n][ks][e] << 16) * f,
                                __uint_as_float(qa[n][ks][e] & 0xffff0000u) * f, true);
    }
  }

  const uint32_t wbase = smem_u32(da_smem_buf) + warp * Lay::WARP;
  uint32_t* wok = reinterpret_cast<uint32_t*>(da_smem_buf + da_smem<HD, KV8, NG>() - 4 * DA_STAGES * 4) + warp * DA_STAGES;
  const int ntiles = (end - begin + 4 * DA_TILE - 1) / (4 * DA_TILE);
  const long long trow = (long long)r * a.c.tstride;
  // page and token of this lane's key of tile t (lanes 0 .. 15), read one tile ahead of its copies
  auto lookup = [&](int t, int* tok) {
    const int i = begin + (t * 4 + warp) * DA_TILE + lane;
    if (lane >= DA_TILE || i >= end) return -1;
    const int p = sp.pos(i), pg = a.c.by_page.div(p);
    *tok = p - pg * a.c.page;
    const int page = a.c.table[trow + pg];
    if (page >= 0 && page < a.c.num_pages) return page;
    record_error(a.err, DEV_BAD_INDEX);
    return -1;
  };
  int tok_next = 0, page_next = lookup(0, &tok_next);
  constexpr int CPR = RB / 16, RPI = 32 / CPR;  // copies per row, rows per instruction
  const int ch = lane % CPR, sub = lane / CPR;
  const uint8_t* kbase = a.c.k + (long long)c * a.c.khs + ch * 16;
  const uint8_t* vbase = a.c.v + (long long)c * a.c.vhs + ch * 16;
  auto issue = [&](int t) {
    if (t < ntiles) {
      const int page = page_next, tok = tok_next;
      page_next = lookup(t + 1, &tok_next);
      const int st = t % DA_STAGES;
      const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0) wok[st] = ok;
      const uint32_t sbase = wbase + st * 2 * Lay::PART;
      const long long koff = page >= 0 ? page * a.c.kps + tok * a.c.kts : 0;
      const uint32_t mine = ok >> sub;
      // rows that no position stands for are zero: what the cache holds there may be no number
      if (a.c.same) {
#pragma unroll
        for (int u = 0; u < DA_TILE / RPI; ++u) {
          const long long o = __shfl_sync(0xffffffffu, koff, u * RPI + sub);
          const uint32_t dst = sbase + row_sw<RB>(u * RPI + sub, ch), n = (mine >> (u * RPI)) & 1u ? 16u : 0u;
          pc_cp_async16(dst, kbase + o, n);
          pc_cp_async16(dst + Lay::PART, vbase + o, n);
        }
      } else {
        const long long voff = page >= 0 ? page * a.c.vps + tok * a.c.vts : 0;
#pragma unroll
        for (int u = 0; u < DA_TILE / RPI; ++u) {
          const long long o = __shfl_sync(0xffffffffu, koff, u * RPI + sub);
          const long long w = __shfl_sync(0xffffffffu, voff, u * RPI + sub);
          const uint32_t dst = sbase + row_sw<RB>(u * RPI + sub, ch), n = (mine >> (u * RPI)) & 1u ? 16u : 0u;
          pc_cp_async16(dst, kbase + o, n);
          pc_cp_async16(dst + Lay::PART, vbase + w, n);
        }
      }
    }
    pc_cp_commit();
  };
#pragma unroll
  for (int t = 0; t < DA_STAGES - 1; ++t) issue(t);

  float o[NG][MT][4];
  float m[NG], l[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
  }

  for (int t = 0; t < ntiles; ++t) {
    issue(t + DA_STAGES - 1);
    pc_cp_wait<DA_STAGES - 1>();
    __syncwarp();
    const uint32_t kb0 = wbase + (t % DA_STAGES) * 2 * Lay::PART, vb0 = kb0 + Lay::PART;
    const uint32_t ok = wok[t % DA_STAGES];
    float sc[2][4];  // keys 8 nt + 2 tig (+ 1) of heads gid, gid + 8
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
      const int kr = nt * 8 + (lane & 7);
      if constexpr (KV8) {
#pragma unroll
        for (int k4 = 0; k4 < KS; k4 += 4) {
          uint32_t b[4];
          ldsm4(kb0 + row_sw<RB>(kr, k4 + (lane >> 3)), b);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t b0, b1;
            e4m3x4_h(b[e], b0, b1);
            mma16816<true>(sc[nt], qa[0][k4 + e][0], NG == 2 ? qa[NG - 1][k4 + e][0] : 0u, qa[0][k4 + e][1],
                           NG == 2 ? qa[NG - 1][k4 + e][1] : 0u, b0, b1);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          uint32_t b[4];
          ldsm4(kb0 + row_sw<RB>(kr, 2 * ks + (lane >> 3)), b);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            mma16816<false>(sc[nt], qa[0][ks + e][0], NG == 2 ? qa[NG - 1][ks + e][0] : 0u, qa[0][ks + e][1],
                            NG == 2 ? qa[NG - 1][ks + e][1] : 0u, b[2 * e], b[2 * e + 1]);
        }
      }
    }
    const int key0 = begin + (t * 4 + warp) * DA_TILE;
    uint32_t pb[NG][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& s = sc[nt][2 * n + e];
          s = (ok >> (nt * 8 + tig * 2 + e)) & 1u ? s * sscale[n] : -INFINITY;
          mx = fmaxf(mx, s);
        }
      if (a.scores != nullptr && gid + 8 * n < nh) {
        float* dst = a.scores + ((long long)r * a.H + h0 + gid + 8 * n) * a.pitch + key0 + tig * 2;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)  // the pitch is even and past every chunk's last whole tile
          if (key0 + nt * 8 + tig * 2 < end)
            *reinterpret_cast<float2*>(dst + nt * 8) = make_float2(sc[nt][2 * n], sc[nt][2 * n + 1]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[n], mx);
      const float u = mn == -INFINITY ? 0.0f : mn;
      if (__any_sync(0xffffffffu, mn != m[n])) {
        const float al = ex2(m[n] - u);
        l[n] *= al;
        // the outputs' columns are heads 2 tig, 2 tig + 1
        const float a0 = __shfl_sync(0xffffffffu, al, tig * 8), a1 = __shfl_sync(0xffffffffu, al, tig * 8 + 4);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[n][i][0] *= a0;
          o[n][i][1] *= a1;
          o[n][i][2] *= a0;
          o[n][i][3] *= a1;
        }
        m[n] = mn;
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const float p0 = ex2(sc[nt][2 * n] - u), p1 = ex2(sc[nt][2 * n + 1] - u);
        l[n] += p0 + p1;
        pb[n][nt] = pack16(p0, p1, KV8);
      }
    }
    if constexpr (KV8) {
      // one transposed load of byte pairs holds columns 2 gid and 2 gid + 1 of
      // two keys: rows gid and gid + 8 of the product stand for those columns
#pragma unroll
      for (int i = 0; i < MT; i += 2) {
        uint32_t b[4];
        ldsm4_t(vb0 + row_sw<RB>((lane & 7) + ((lane >> 3) & 1) * 8, i + (lane >> 4)), b);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_h(__byte_perm(b[2 * e], 0, 0x3120), a0, a1);
          e4m3x4_h(__byte_perm(b[2 * e + 1], 0, 0x3120), a2, a3);
#pragma unroll
          for (int n = 0; n < NG; ++n) mma16816<true>(o[n][i + e], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t b[4];  // (keys 0-7, d 0-7), (keys 0-7, d 8-15), (keys 8-15, d 0-7), (keys 8-15, d 8-15)
        ldsm4_t(vb0 + row_sw<RB>((lane & 7) + (lane >> 4) * 8, 2 * i + ((lane >> 3) & 1)), b);
#pragma unroll
        for (int n = 0; n < NG; ++n) mma16816<false>(o[n][i], b[0], b[1], b[2], b[3], pb[n][0], pb[n][1]);
      }
    }
    __syncwarp();  // the stage may be refilled from here on
  }
  pc_cp_wait<0>();
  __syncthreads();  // every warp's pipeline is drained: its shared memory is free

  // merge the four warps: each head's maximum, sum and output
  float* mO = reinterpret_cast<float*>(da_smem_buf);  // [4][8 NG][HD + 4]
  float2* mS = reinterpret_cast<float2*>(mO + 4 * 8 * NG * (HD + 4));
  float2* mR = mS + 4 * 8 * NG;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
    if (tig == 0) mS[warp * 8 * NG + n * 8 + gid] = make_float2(m[n], l[n]);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = i * 16 + (KV8 ? 2 * gid + (e >> 1) : gid + (e >> 1) * 8);
        mO[(warp * 8 * NG + n * 8 + tig * 2 + (e & 1)) * (HD + 4) + d] = o[n][i][e];
      }
  }
  __syncthreads();
  const bool single = sp.n <= chunk_of(a, sp.n);
  if (threadIdx.x < nh) {
    float mm = -INFINITY, ll = 0.0f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mS[w * 8 * NG + threadIdx.x].x);
    const float u = mm == -INFINITY ? 0.0f : mm;
    for (int w = 0; w < 4; ++w) {
      float2& s = mS[w * 8 * NG + threadIdx.x];
      s.x = ex2(s.x - u);  // from here on the warp's factor
      ll += s.y * s.x;
    }
    mR[threadIdx.x] = make_float2(mm, ll);
    if (!single || a.scores != nullptr)
      a.stats[((long long)r * a.H + h0 + threadIdx.x) * a.chunks + chunk] = make_float2(mm, ll);
  }
  __syncthreads();
  for (int v = threadIdx.x; v < nh * (HD / 4); v += 128) {
    const int h = v / (HD / 4), d = (v % (HD / 4)) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = mS[w * 8 * NG + h].x;
      const float4 x = *reinterpret_cast<const float4*>(&mO[(w * 8 * NG + h) * (HD + 4) + d]);
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
    acc.x *= vd;
    acc.y *= vd;
    acc.z *= vd;
    acc.w *= vd;
    if (single) {
      const float ll = mR[h].y, inv = ll == 0.0f ? 0.0f : 1.0f / ll;  // a row whose scores are all -inf is zero
      uint2 w2 = make_uint2(pack16(acc.x * inv, acc.y * inv, false), pack16(acc.z * inv, acc.w * inv, false));
      *reinterpret_cast<uint2*>(a.out + (long long)r * a.o_rs + (long long)(h0 + h) * a.o_hs + d) = w2;
    } else {
      *reinterpret_cast<float4*>(a.part + (((long long)r * a.H + h0 + h) * a.chunks + chunk) * HD + d) = acc;
    }
  }
}

// (maximum, sum) of a row over its n chunks, by one warp; the maximum of a row
// whose scores are all -inf comes back as 0.
__device__ __forceinline__ float2 row_stats(const float2* stats, int n) {
  const int lane = threadIdx.x & 31;
  float2 first = lane < n ? stats[lane] : make_float2(-INFINITY, 0.0f);
  float mm = first.x;
  for (int c = lane + 32; c < n; c += 32) mm = fmaxf(mm, stats[c].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
  const float u = mm == -INFINITY ? 0.0f : mm;
  float ll = first.y * ex2(first.x - u);
  for (int c = lane + 32; c < n; c += 32) {
    const float2 s = stats[c];
    ll += s.y * ex2(s.x - u);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
  return make_float2(u, ll);
}

constexpr int DJ_HEADS = 8;  // heads whose scores a thread has in flight

// Blocks [0, row_blocks): (request, head) rows whose chunks are joined, one row
// to a block, or to a warp where a row has few chunks (WARP_ROWS).
// Blocks from there on: 4 NT visible positions of one (request, kv head),
// whose weights are added to the sums; every sum has one writer, so repeated
// runs agree bit for bit.
template <int HD, bool WARP_ROWS, int NT>
__global__ void __launch_bounds__(NT) decode_join_kernel(DecodeArgs a, int row_blocks, int key_blocks) {
  constexpr int DJ_KEYS = 4 * NT;
  static_assert(NT / 32 >= DJ_HEADS, "a warp to a head's statistics");
  __shared__ float4 sred[NT / 32][HD / 4];
  __shared__ float2 sst[DJ_HEADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.c.R * a.H;
  pdl_wait();
  if (WARP_ROWS && (int)blockIdx.x < row_blocks) {
    const int row = blockIdx.x * (NT / 32) + warp, r = row / a.H, h = row % a.H;
    if (row >= rows) return;
    const Span sp = visible_span(cache_length(a.c, r, a.err, false), a.window, a.sinks);
    const int size = chunk_of(a, sp.n), n = (sp.n + size - 1) / size;
    if (n <= 1) return;  // written by its only chunk
    const float2* stats = a.stats + (long long)row * a.chunks;
    const float* part = a.part + (long long)row * a.chunks * HD + lane * (HD / 32);
    float o[HD / 32] = {};
    const float2 st = row_stats(stats, n);
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      float x[HD / 32];
      if constexpr (HD == 128)
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(part + (long long)c * HD);
      else
        *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(part + (long long)c * HD);
      const float f = ex2(stats[c].x - st.x);
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) o[e] += x[e] * f;
    }
    const float inv = st.y == 0.0f ? 0.0f : 1.0f / st.y;
    __nv_bfloat16* out = a.out + (long long)r * a.o_rs + (long long)h * a.o_hs + lane * (HD / 32);
#pragma unroll
    for (int e = 0; e < HD / 32; e += 2)
      *reinterpret_cast<uint32_t*>(out + e) = pack16(o[e] * inv, o[e + 1] * inv, false);
    return;
  }
  if (!WARP_ROWS && (int)blockIdx.x < row_blocks) {
    const int row = blockIdx.x, r = row / a.H, h = row % a.H;
    const Span sp = visible_span(cache_length(a.c, r, a.err, false), a.window, a.sinks);
    const int size = chunk_of(a, sp.n), n = (sp.n + size - 1) / size;
    if (n <= 1) return;  // written by its only chunk
    const float2* stats = a.stats + (long long)row * a.chunks;
    const float2 st = row_stats(stats, n);
    constexpr int V = HD / 4, PER = NT / V;  // threads per chunk's row, chunks at a time
    const float4* part = reinterpret_cast<const float4*>(a.part + (long long)row * a.chunks * HD) + tid % V;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = tid / V; c < n; c += PER) {
      const float4 x = part[(long long)c * V];
      const float f = ex2(stats[c].x - st.x);
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
    if constexpr (V == 16) {  // two groups of a warp hold the same columns
      acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16);
      acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
      acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16);
      acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
    }
    if (lane < V) sred[warp][lane] = acc;
    __syncthreads();
    if (tid < V) {
      const float inv = st.y == 0.0f ? 0.0f : 1.0f / st.y;
      float4 o = sred[0][tid];
#pragma unroll 8
      for (int w = 1; w < NT / 32; ++w) {
        const float4 x = sred[w][tid];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
      }
      *reinterpret_cast<uint2*>(a.out + (long long)r * a.o_rs + (long long)h * a.o_hs + tid * 4) =
          make_uint2(pack16(o.x * inv, o.y * inv, false), pack16(o.z * inv, o.w * inv, false));
    }
    return;
  }
  const int item = (blockIdx.x - row_blocks) / key_blocks, kb = (blockIdx.x - row_blocks) % key_blocks;
  const int r = item / a.c.KH, c = item % a.c.KH;
  const Span sp = visible_span(cache_length(a.c, r, a.err, false), a.window, a.sinks);
  const int begin = kb * DJ_KEYS;
  if (begin >= sp.n) return;
  const int size = chunk_of(a, sp.n), n = (sp.n + size - 1) / size;
  const long long row0 = (long long)r * a.H + c * a.G;
  float* dst = a.sums + (long long)r * a.s_rs + (long long)c * a.s_hs;
  const int i = begin + tid * 4;  // this thread's four positions (the pitch is a multiple of 16)
  float old[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) old[e] = i + e < sp.n ? dst[sp.pos(i + e)] : 0.0f;
  float4 add = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int g0 = 0; g0 < a.G; g0 += DJ_HEADS) {
    float4 s[DJ_HEADS];
#pragma unroll
    for (int g = 0; g < DJ_HEADS; ++g)
      if (g0 + g < a.G && i < sp.n) s[g] = *reinterpret_cast<const float4*>(a.scores + (row0 + g0 + g) * a.pitch + i);
    if (warp < DJ_HEADS && g0 + warp < a.G) {
      const float2 st = row_stats(a.stats + (row0 + g0 + warp) * a.chunks, n);
      if (lane == 0) sst[warp] = make_float2(st.x, st.y == 0.0f ? 0.0f : 1.0f / st.y);
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < DJ_HEADS; ++g)
      if (g0 + g < a.G && i < sp.n) {
        const float2 st = sst[g];
        add.x += ex2(s[g].x - st.x) * st.y;
        add.y += ex2(s[g].y - st.x) * st.y;
        add.z += ex2(s[g].z - st.x) * st.y;
        add.w += ex2(s[g].w - st.x) * st.y;
      }
    __syncthreads();
  }
  const float w[4] = {add.x, add.y, add.z, add.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < sp.n) dst[sp.pos(i + e)] = old[e] + w[e];
}
struct DecodePlan {
  int ng, hgroups, least, chunks, pitch;
  size_t part, stats, scores, total;
};

// Every request is cut into equal chunks, so many that the launch has DA_CTAS
// CTAs; the kernel finds their size from the request's own length, so that a
// call sized for far longer contexts than it meets still uses the whole GPU.
// Chunks have DA_CHUNK keys at least (500 positions, 1 request: 6.0 us against
// 7.8 us in chunks of 256 and 6.0 us in chunks of 64), and more where there are
// enough (request, kv head) pairs to fill the GPU without cutting, three CTAs
// to an SM: then a cut only makes a join.
constexpr int DA_CTAS = 148 * 12;
constexpr int DA_CHUNK = 128;
constexpr int DA_ENOUGH = 1536;

DecodePlan decode_plan(int64_t R, int64_t H, int64_t KH, int64_t HD, int64_t max_len, int64_t window, bool sums,
                       int64_t sinks) {
  DecodePlan p{};
  const int64_t G = H / KH;
  p.ng = G > 8 ? 2 : 1;
  p.hgroups = (int)((G + 8 * p.ng - 1) / (8 * p.ng));
  const int64_t span = visible_span((int)max_len, (int)window, (int)sinks).n;
  const int64_t items = R * KH * p.hgroups, cut = (DA_CTAS + items - 1) / items;
  int64_t least = DA_ENOUGH * items / (3 * 148) / 64 * 64;
  least = least < DA_CHUNK ? DA_CHUNK : least > DA_ENOUGH ? DA_ENOUGH : least;
  p.least = (int)least;
  const int64_t most = span <= DA_WHOLE ? 1 : (span + least - 1) / least;
  p.chunks = (int)(cut < most ? cut : most);
  if (p.chunks < 1) p.chunks = 1;
  p.pitch = (int)((span + 15) / 16 * 16);
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const bool join = p.chunks > 1;
  p.part = join ? up((size_t)(R * H) * p.chunks * HD * 4) : 0;
  p.stats = join || sums ? up((size_t)(R * H) * p.chunks * 8) : 0;
  p.scores = sums ? up((size_t)(R * H) * p.pitch * 4) : 0;
  p.total = p.part + p.stats + p.scores;
  return p;
}

template <int HD, bool KV8, int NG>
fm_status launch_decode(const DecodeArgs& a, unsigned grid, cudaStream_t s) {
  constexpr int smem = da_smem<HD, KV8, NG>();
  const fm_status st = allow_smem<decode_attn_kernel<HD, KV8, NG>>(smem, "paged_decode_attn");
  if (st != FM_OK) return st;
  return launch_kernel(decode_attn_kernel<HD, KV8, NG>, dim3(grid), dim3(128), smem, s, true, a);
}

template <int HD>
fm_status launch_decode_hd(const DecodeArgs& a, bool kv8, int ng, unsigned grid, cudaStream_t s) {
  if (kv8) return ng == 2 ? launch_decode<HD, true, 2>(a, grid, s) : launch_decode<HD, true, 1>(a, grid, s);
  return ng == 2 ? launch_decode<HD, false, 2>(a, grid, s) : launch_decode<HD, false, 1>(a, grid, s);
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_paged_decode_attn_workspace_size(int64_t requests, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_length, int64_t window,
                                                      int64_t sinks, int32_t with_sums) {
  if (requests < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_length < 0 ||
      max_length > 0x7ffffff0 || window < 0 || window > 0x7ffffff0 || sinks < 0 || sinks > 0x7ffffff0)
    return 0;
  return decode_plan(requests, heads, kv_heads, head_dim, max_length, window, with_sums != 0, sinks).total;
}

extern "C" fm_status fm_paged_decode_attn(const fm_paged_cache* cache, const fm_decode_attn* p, fm_stream stream) {
  DecodeArgs a{};
  fm_status st = cache_ref(cache, "paged_decode_attn", &a.c);
  if (st != FM_OK) return st;
  if (!p) return set_error(FM_ERR_INVALID, "paged_decode_attn: null arguments");
  if (p->heads < 1 || p->heads % cache->kv_heads || p->heads > 65535)
    return set_error(FM_ERR_SHAPE, "paged_decode_attn: query heads must be a multiple of the kv heads");
  if (p->window < 0 || p->sinks < 0 || p->window > 0x7ffffff0 || p->sinks > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "paged_decode_attn: window and sinks must not be negative");
  if (cache->requests == 0) return FM_OK;
  if (!p->q || !p->out) return set_error(FM_ERR_INVALID, "paged_decode_attn: null pointer");
  // one request or one head is not stepped through: its stride may be anything
  a.q_rs = cache->requests == 1 ? 0 : p->q_request_stride;
  a.q_hs = p->heads == 1 ? 0 : p->q_head_stride;
  a.o_rs = cache->requests == 1 ? 0 : p->out_request_stride;
  a.o_hs = p->heads == 1 ? 0 : p->out_head_stride;
  if ((uintptr_t)p->q % 4 || a.q_rs % 2 || a.q_hs % 2 || (uintptr_t)p->out % 8 || a.o_rs % 4 || a.o_hs % 4)
    return set_error(FM_ERR_ALIGN, "paged_decode_attn: query rows must be 4-byte, output rows 8-byte aligned");
  const bool sums = p->weight_sums != nullptr;
  const DecodePlan pl = decode_plan(cache->requests, p->heads, cache->kv_heads, cache->head_dim, cache->max_length,
                                    p->window, sums, p->sinks);
  if (pl.total > p->workspace_bytes || (pl.total && !p->workspace))
    return set_error(FM_ERR_WORKSPACE, "paged_decode_attn: workspace %zu < %zu", p->workspace_bytes, pl.total);
  if ((uintptr_t)p->workspace % 16) return set_error(FM_ERR_ALIGN, "paged_decode_attn: workspace not 16-byte aligned");
  a.q = static_cast<const uint8_t*>(p->q);
  a.H = (int)p->heads;
  a.G = (int)(p->heads / cache->kv_heads);
  a.hgroups = pl.hgroups;
  a.scale = p->softmax_scale * kLog2e;
  a.window = (int)p->window;
  a.sinks = (int)p->sinks;
  a.least = pl.least;
  a.chunks = pl.chunks;
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.sums = p->weight_sums;
  a.s_rs = p->sums_request_stride;
  a.s_hs = p->sums_head_stride;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.part = reinterpret_cast<float*>(ws);
  a.stats = reinterpret_cast<float2*>(ws + pl.part);
  a.scores = sums ? reinterpret_cast<float*>(ws + pl.part + pl.stats) : nullptr;
  a.pitch = pl.pitch;
  a.err = p->err;
  const int64_t items = cache->requests * cache->kv_heads * pl.hgroups;
  // a warp to a row where that leaves no warp more than 16 chunks
  const bool warp_rows = pl.chunks <= 16;
  const int nt = warp_rows ? 256 : 1024;
  const int64_t per = warp_rows ? nt / 32 : 1, key_blocks = sums ? (pl.pitch + 4 * nt - 1) / (4 * nt) : 0;
  const int64_t row_blocks = pl.chunks > 1 ? (cache->requests * p->heads + per - 1) / per : 0;
  const int64_t join = row_blocks + cache->requests * cache->kv_heads * key_blocks;
  if (items * pl.chunks > 0x7fffffff || join > 0x7fffffff)
    return set_error(FM_ERR_SHAPE, "paged_decode_attn: grid too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool kv8 = cache->dtype == FM_DT_E4M3;
  const unsigned grid = (unsigned)(items * pl.chunks);
  st = cache->head_dim == 128 ? launch_decode_hd<128>(a, kv8, pl.ng, grid, s)
                              : launch_decode_hd<64>(a, kv8, pl.ng, grid, s);
  if (st != FM_OK || join == 0) return st;  // one chunk, and no sums or no positions
  const dim3 grid2((unsigned)join), block(nt);
  auto join_launch = [&](auto kernel) {
    return launch_kernel(kernel, grid2, block, 0, s, true, a, (int)row_blocks, (int)key_blocks);
  };
  if (cache->head_dim == 128)
    return warp_rows ? join_launch(decode_join_kernel<128, true, 256>) : join_launch(decode_join_kernel<128, false, 1024>);
  return warp_rows ? join_launch(decode_join_kernel<64, true, 256>) : join_launch(decode_join_kernel<64, false, 1024>);
}
