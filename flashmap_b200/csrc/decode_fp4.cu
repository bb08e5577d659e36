// Attention of one new token per request over a paged cache held in 4 bits.
//
// The rows' values are e2m1 codes times an e4m3 factor for each sixteen: 6
// significant bits, which f16 holds exactly, so the products' operands carry no
// rounding but the numerators'.  Formulas, chunks and the join are those of the
// wider caches (decode_parts.cuh).
//
// A key and value of 128 are 144 bytes for 8 to 16 heads, so what a key costs
// in instructions is near what it costs in bytes: a multiplication and a
// conversion to two values.  Each warp streams 32-key tiles through cp.async;
// keys are the rows of S[keys][heads] = K Q^T and the columns of O^T[d][heads] =
// V^T P^T, so that eight heads waste nothing of a product, and any order of d
// (in S) and of d (in O) may be chosen: a thread takes 16 consecutive
// bytes of a key, and 8 of a value, as they lie.  Values of two keys
// are paired for V^T by exchanging half bytes before the conversion.
//
// Measured, 32 heads on 8 of 128: 128 requests of 1024 .. 8192, 165 to 174 us (3.9 to 4.1 TB/s);
// 1 request of 100003, 32 us (3.6 TB/s, of which 5 us are the join); 201
// positions, 4.8 us.  No unit is full: the arithmetic pipe that converts is at 53
// percent and issue slots at 59, with four warps to a scheduler (registers);
// five, and a third stage of copies, measured the same, six spill.  More than 8
// heads to a group take 230 to 240 registers, two CTAs to an SM: 64 heads on 4 read
// the same bytes in 280 us, 2.5 TB/s.  At head_dim 64 and 32 heads on 8: 108 us, 3.2 TB/s.
#include <type_traits>

#include "decode_parts.cuh"

namespace fm {
namespace {

constexpr int D4_TILE = 32;  // keys of a warp's tile
constexpr int D4_STAGES = 2;
// A CTA's first copies and its merge weigh more against 4-bit keys: one long
// request is cut into 148 * 4 chunks, the CTAs that are resident at head_dim 128 and up to
// 8 heads to a group (100003 positions, 8 kv heads: 34 us, and 40 us in three times as many, both with a join slower by 2 us), and a batch into chunks
// of 2048 keys (128 requests of 1024 .. 8192, on one GPU: 163 us; of 1024 keys 173 us, of 4096 170 us).  Wider
// groups, of which two CTAs are resident, and head_dim 64 go by the same numbers; others were not tried there.
constexpr DecodeRule D4_RULE{148 * 4, 128, 1536, 2048, 148 * 32};

// P goes to f16 times 2^11, and the subtracted maximum may lag behind the true
// one by a factor 2^4: numerators stay below 2^15, and only those under 2^-25 of
// the largest meet f16's coarsest steps.
constexpr float D4_LIFT = 11.0f, D4_LAG = 4.0f;

template <int HD>
struct D4Layout {
  static constexpr int RB = HD / 2, SB = HD / 16;  // bytes of a row's codes, of its factors
  static constexpr int V = D4_TILE * RB, KF = 2 * V, VF = KF + D4_TILE * SB;
  static constexpr int STAGE = 2 * D4_TILE * (RB + SB);
  static constexpr int WARP = D4_STAGES * STAGE;
};
template <int HD, int NG>
constexpr int d4_smem() {
  constexpr int merge = 4 * 8 * NG * (HD + 4) * 4 + 4 * 8 * NG * 8 + 8 * NG * 8, pipe = 4 * D4Layout<HD>::WARP;
  return (pipe > merge ? pipe : merge) + 4 * D4_STAGES * 4;
}

// Where 16-byte chunk `ch` of a tile's row lies.  A thread's rows are those of
// key_row(): together, four rows' halves of V and eight rows' quarters of K fall into different banks.
template <int RB>
__device__ __forceinline__ uint32_t d4_sw(int row, int ch) {
  return (uint32_t)(row * RB + ch * 16) ^ (uint32_t)((row & 4) << 3);
}
// The tile's row that stands as row g of a group of eight in the products.
__device__ __forceinline__ int key_row(int g) { return g ^ ((g >> 1) & 1); }

__device__ __forceinline__ void d4_cp_async(uint32_t dst, const void* src, uint32_t bytes, bool wide) {
  if (wide)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t d4_lds8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t d4_lds16(uint32_t at) {
  uint32_t v;
  asm volatile("{.reg .u16 h; ld.shared.u16 h, [%1]; cvt.u32.u16 %0, h;}" : "=r"(v) : "r"(at) : "memory");
  return v;
}
template <int W>
__device__ __forceinline__ void d4_lds(uint32_t at, uint32_t* v) {
  if constexpr (W == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
  else if constexpr (W == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(at) : "memory");
}
// the transpose of an 8 x 8 matrix of 16-bit values, two to a lane
__device__ __forceinline__ uint32_t d4_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// NG: groups of 8 query heads (1 or 2).  WIDE: offsets past 32 bits in NarrowRef's units.
template <int HD, int NG, bool WIDE>
__global__ void __launch_bounds__(128) decode_fp4_kernel(DecodeArgs a, ScaleRef f, NarrowRef nr) {
  using Lay = D4Layout<HD>;
  constexpr int STAGES = D4_STAGES;
  constexpr int RB = Lay::RB, SB = Lay::SB;
  constexpr int KW = HD / 32, VW = HD / 64;  // words of a thread's piece of a key, of a value
  constexpr int KS = HD / 16;                // products along d, and rows of sixteen d of the output
  extern __shared__ __align__(1024) uint8_t d4_smem_buf[];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  pdl_wait();
  const int items = a.c.R * a.c.KH * a.hgroups;
  const int chunk = blockIdx.x / items;
  int rest = blockIdx.x % items;
  const int hg = rest % a.hgroups;
  rest /= a.hgroups;
  const int c = rest % a.c.KH, r = rest / a.c.KH;
  const int h0 = c * a.G + hg * 8 * NG;           // first query head
  const int nh = min(8 * NG, a.G - hg * 8 * NG);  // query heads of this CTA
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

  const uint32_t wbase = smem_u32(d4_smem_buf) + warp * Lay::WARP;
  uint32_t* wok = reinterpret_cast<uint32_t*>(d4_smem_buf + d4_smem<HD, NG>() - 4 * STAGES * 4) + warp * STAGES;
  const int ntiles = (end - begin + 4 * D4_TILE - 1) / (4 * D4_TILE);
  const long long trow = (long long)r * a.c.tstride;
  // page and token of this lane's key of tile t, read one tile ahead of its copies
  auto lookup = [&](int t, int* tok) {
    const int i = begin + (t * 4 + warp) * D4_TILE + lane;
    if (i >= end) return -1;
    const int p = sp.pos(i), pg = a.c.by_page.div(p);
    *tok = p - pg * a.c.page;
    const int page = a.c.table[trow + pg];
    if (page >= 0 && page < a.c.num_pages) return page;
    record_error(a.err, DEV_BAD_INDEX);
    return -1;
  };
  int tok_next = 0, page_next = lookup(0, &tok_next);
  constexpr int CPR = RB / 16, RPI = 32 / CPR;  // chunks of a row, rows per instruction
  const int ch = lane % CPR, sub = lane / CPR;
  const uint8_t* kbase = a.c.k + (long long)c * a.c.khs + ch * 16;
  const uint8_t* vbase = a.c.v + (long long)c * a.c.vhs + ch * 16;
  const uint8_t* kfbase = f.k + (long long)c * f.khs;
  const uint8_t* vfbase = f.v + (long long)c * f.vhs;
  auto issue = [&](int t, int st) {
    if (t < ntiles) {
      const int page = page_next, tok = tok_next;
      page_next = lookup(t + 1, &tok_next);
      const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0) wok[st] = ok;
      const uint32_t sbase = wbase + st * Lay::STAGE, dst = sbase + d4_sw<RB>(sub, ch);
      // Codes are numbers whatever they are, so rows that no position stands for may be any row; their factors are zero.
      const uint32_t own = page >= 0 ? SB : 0u;
      if constexpr (WIDE) {
        const long long koff = page >= 0 ? page * a.c.kps + tok * a.c.kts : 0;
        const long long voff = page >= 0 ? page * a.c.vps + tok * a.c.vts : 0;
        d4_cp_async(sbase + Lay::KF + lane * SB, page >= 0 ? kfbase + page * f.kps + tok * f.kts : kfbase, own, SB == 8);
        d4_cp_async(sbase + Lay::VF + lane * SB, page >= 0 ? vfbase + page * f.vps + tok * f.vts : vfbase, own, SB == 8);
#pragma unroll
        for (int u = 0; u < D4_TILE / RPI; ++u) {
          const long long o = __shfl_sync(0xffffffffu, koff, u * RPI + sub), w = __shfl_sync(0xffffffffu, voff, u * RPI + sub);
          pc_cp_async16(dst + u * RPI * RB, kbase + o, 16u);
          pc_cp_async16(dst + Lay::V + u * RPI * RB, vbase + w, 16u);
        }
      } else {
        const uint32_t pg = page >= 0 ? page : 0, tk = page >= 0 ? tok : 0;
        const uint32_t koff = pg * nr.kp + tk * nr.kt, kfoff = pg * nr.kfp + tk * nr.kft;
        const uint32_t voff = nr.same ? koff : pg * nr.vp + tk * nr.vt, vfoff = nr.same ? kfoff : pg * nr.vfp + tk * nr.vft;
        d4_cp_async(sbase + Lay::KF + lane * SB, kfbase + (unsigned long long)kfoff * SB, own, SB == 8);
        d4_cp_async(sbase + Lay::VF + lane * SB, vfbase + (unsigned long long)vfoff * SB, own, SB == 8);
#pragma unroll
        for (int u = 0; u < D4_TILE / RPI; ++u) {
          const uint32_t o = __shfl_sync(0xffffffffu, koff, u * RPI + sub);
          const uint32_t w = nr.same ? o : __shfl_sync(0xffffffffu, voff, u * RPI + sub);
          pc_cp_async16(dst + u * RPI * RB, kbase + (unsigned long long)o * 16, 16u);
          pc_cp_async16(dst + Lay::V + u * RPI * RB, vbase + (unsigned long long)w * 16, 16u);
        }
      }
    }
    pc_cp_commit();
  };
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) issue(t, t);

  // while the first tile is on its way
  float kd = 1.0f, vd = 1.0f;
  if (a.c.descales) {
    kd = a.c.descales[(long long)r * a.c.KH + c];
    vd = a.c.descales[(long long)(a.c.R + r) * a.c.KH + c];
  }
  // Query operand: head h0 + gid (and + 8), d = HD / 4 tig .. as a key's piece holds them; f16 times a power of two.
  const float scale = a.scale * kd;
  uint32_t qb[NG][KS][2];
  float sscale[NG][2];  // of heads 2 tig, 2 tig + 1
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const bool live = gid + 8 * n < nh;
    const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(a.q) + (long long)r * a.q_rs +
                               (long long)(h0 + (live ? gid + 8 * n : 0)) * a.q_hs + tig * (HD / 4);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t w = live ? *reinterpret_cast<const uint32_t*>(row + 4 * i + 2 * e) : 0u;
        qb[n][i][e] = w;
        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
      }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float up = half_row_scale(amax), sign = scale < 0.0f ? -up : scale == 0.0f ? 0.0f : up;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qb[n][i][e] = pack16(__uint_as_float(qb[n][i][e] << 16) * sign, __uint_as_float(qb[n][i][e] & 0xffff0000u) * sign, true);
    // |scale| goes with the scores, its sign (or a zero) with the queries
    sscale[n][0] = (scale == 0.0f ? 1.0f : fabsf(scale)) / __shfl_sync(0xffffffffu, up, tig * 8);
    sscale[n][1] = (scale == 0.0f ? 1.0f : fabsf(scale)) / __shfl_sync(0xffffffffu, up, tig * 8 + 4);
  }

  float o[NG][KS][4];
  float m[NG][2], l[NG][2];  // of heads 2 tig, 2 tig + 1: the reference and, of this lane's keys, the sum
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
  }

  // where this thread's pieces lie in a stage: of keys key_row(gid) (+ 8, 16, 24), of values key_row(2 tig), key_row(2 tig + 1)
  constexpr int KB = 4 * KW, VB = 4 * VW;  // bytes of a piece
  const int krow = key_row(gid), va = key_row(2 * tig), vb = key_row(2 * tig + 1);
  const uint32_t k_at = d4_sw<RB>(krow, tig * KB / 16) + (tig * KB) % 16;
  const uint32_t va_at = d4_sw<RB>(va, gid * VB / 16) + (gid * VB) % 16;
  const uint32_t vb_at = d4_sw<RB>(vb, gid * VB / 16) + (gid * VB) % 16;
  const uint32_t kf_at = Lay::KF + krow * SB + tig * (SB / 4);
  const uint32_t vfa_at = Lay::VF + va * SB + gid * HD / 128, vfb_at = Lay::VF + vb * SB + gid * HD / 128;

  auto tile = [&](int t, auto stage_at) {
    constexpr int stage = decltype(stage_at)::value;
    issue(t + STAGES - 1, (stage + STAGES - 1) % STAGES);
    pc_cp_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t sb = wbase + stage * Lay::STAGE;
    const uint32_t ok = wok[stage];
    float sc[2][NG][4];  // of 16 keys each: keys gid, gid, gid + 8, gid + 8 of heads 2 tig, 2 tig + 1
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int n = 0; n < NG; ++n) sc[half][n][0] = sc[half][n][1] = sc[half][n][2] = sc[half][n][3] = 0.0f;
      uint32_t ka[KW], kb[KW], fa[2], fb[2];
      d4_lds<KW>(sb + k_at + half * 16 * RB, ka);
      d4_lds<KW>(sb + k_at + (half * 16 + 8) * RB, kb);
      if constexpr (HD == 128) {  // two factors to a piece
        const uint32_t ea = e4m3x2_h(d4_lds16(sb + kf_at + half * 16 * SB));
        const uint32_t eb = e4m3x2_h(d4_lds16(sb + kf_at + (half * 16 + 8) * SB));
        fa[0] = __byte_perm(ea, 0, 0x1010);
        fa[1] = __byte_perm(ea, 0, 0x3232);
        fb[0] = __byte_perm(eb, 0, 0x1010);
        fb[1] = __byte_perm(eb, 0, 0x3232);
      } else {
        fa[0] = fa[1] = e4m3x2_h(d4_lds8(sb + kf_at + half * 16 * SB) * 0x101u);
        fb[0] = fb[1] = e4m3x2_h(d4_lds8(sb + kf_at + (half * 16 + 8) * SB) * 0x101u);
      }
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        uint32_t xa[4], xb[4];
        e2m1x8_h(ka[w], xa);
        e2m1x8_h(kb[w], xb);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          xa[e] = mul_h2(xa[e], fa[w * 2 / KW]);
          xb[e] = mul_h2(xb[e], fb[w * 2 / KW]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int n = 0; n < NG; ++n)
            mma16816<true>(sc[half][n], xa[2 * e], xb[2 * e], xa[2 * e + 1], xb[2 * e + 1], qb[n][2 * w + e][0],
                           qb[n][2 * w + e][1]);
      }
    }
    if (ok != 0xffffffffu) {
      const uint32_t seen = ok >> krow;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[half][n][e] = (seen >> (half * 16 + (e & 2) * 4)) & 1u ? sc[half][n][e] : -INFINITY;
    }
    uint32_t pb[2][NG][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const float top0 = fmaxf(fmaxf(sc[0][n][0], sc[0][n][2]), fmaxf(sc[1][n][0], sc[1][n][2])) * sscale[n][0];
      const float top1 = fmaxf(fmaxf(sc[0][n][1], sc[0][n][3]), fmaxf(sc[1][n][1], sc[1][n][3])) * sscale[n][1];
      // m is the maximum less the lift, and moves when a score outgrows it by the lag
      if (__any_sync(0xffffffffu, top0 > m[n][0] + (D4_LIFT + D4_LAG) || top1 > m[n][1] + (D4_LIFT + D4_LAG))) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = e ? top1 : top0;
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[n][e], mx - D4_LIFT);
          const float al = mn == -INFINITY ? 1.0f : ex2(m[n][e] - mn);
          m[n][e] = mn;
          l[n][e] *= al;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[n][i][e] *= al;
            o[n][i][2 + e] *= al;
          }
        }
      }
      const float u0 = m[n][0] == -INFINITY ? 0.0f : -m[n][0], u1 = m[n][1] == -INFINITY ? 0.0f : -m[n][1];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float p0 = ex2(fmaf(sc[half][n][0], sscale[n][0], u0)), p1 = ex2(fmaf(sc[half][n][1], sscale[n][1], u1));
        const float p2 = ex2(fmaf(sc[half][n][2], sscale[n][0], u0)), p3 = ex2(fmaf(sc[half][n][3], sscale[n][1], u1));
        l[n][0] += p0 + p2;
        l[n][1] += p1 + p3;
        pb[half][n][0] = d4_transpose(pack16(p0, p1, true));  // keys 2 tig, 2 tig + 1 of head gid
        pb[half][n][1] = d4_transpose(pack16(p2, p3, true));
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t x[2][4 * VW], y[2][4 * VW];  // values 2 i, and 2 i + 1, of a pair of keys
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t wa[VW], wb[VW];
        d4_lds<VW>(sb + Lay::V + va_at + (half * 16 + q * 8) * RB, wa);
        d4_lds<VW>(sb + Lay::V + vb_at + (half * 16 + q * 8) * RB, wb);
        const uint32_t s2 = e4m3x2_h(d4_lds8(sb + vfa_at + (half * 16 + q * 8) * SB) | d4_lds8(sb + vfb_at + (half * 16 + q * 8) * SB) << 8);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          e2m1x8_h((wa[w] & 0x0f0f0f0fu) | ((wb[w] << 4) & 0xf0f0f0f0u), &x[q][4 * w]);
          e2m1x8_h(((wa[w] >> 4) & 0x0f0f0f0fu) | (wb[w] & 0xf0f0f0f0u), &y[q][4 * w]);
        }
#pragma unroll
        for (int i = 0; i < 4 * VW; ++i) {
          x[q][i] = mul_h2(x[q][i], s2);
          y[q][i] = mul_h2(y[q][i], s2);
        }
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int n = 0; n < NG; ++n) mma16816<true>(o[n][i], x[0][i], y[0][i], x[1][i], y[1][i], pb[half][n][0], pb[half][n][1]);
    }
    __syncwarp();  // the stage may be refilled from here on
  };
  static_assert(STAGES == 2, "the loop goes by twos");
  for (int t = 0; t < ntiles; t += 2) {
    tile(t, std::integral_constant<int, 0>{});
    if (t + 1 < ntiles) tile(t + 1, std::integral_constant<int, 1>{});
  }
  pc_cp_wait<0>();
  __syncthreads();  // every warp's pipeline is drained: its shared memory is free

  // merge the four warps: each head's reference, sum and output
  float* mO = reinterpret_cast<float*>(d4_smem_buf);  // [4][8 NG][HD + 4]
  float2* mS = reinterpret_cast<float2*>(mO + 4 * 8 * NG * (HD + 4));
  float2* mR = mS + 4 * 8 * NG;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = l[n][e];
      s += __shfl_xor_sync(0xffffffffu, s, 4);
      s += __shfl_xor_sync(0xffffffffu, s, 8);
      s += __shfl_xor_sync(0xffffffffu, s, 16);
      if (gid == 0) mS[warp * 8 * NG + n * 8 + tig * 2 + e] = make_float2(m[n][e], s);
    }
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mO[(warp * 8 * NG + n * 8 + tig * 2 + (e & 1)) * (HD + 4) + gid * (HD / 8) + 2 * i + (e >> 1)] = o[n][i][e];
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
    if (!single) a.stats[((long long)r * a.H + h0 + threadIdx.x) * a.chunks + chunk] = make_float2(mm, ll);
  }
  __syncthreads();
  for (int v = threadIdx.x; v < nh * (HD / 4); v += 128) {
    const int h = v / (HD / 4), d = (v % (HD / 4)) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float g = mS[w * 8 * NG + h].x;
      const float4 x = *reinterpret_cast<const float4*>(&mO[(w * 8 * NG + h) * (HD + 4) + d]);
      acc.x += x.x * g;
      acc.y += x.y * g;
      acc.z += x.z * g;
      acc.w += x.w * g;
    }
    acc.x *= vd;
    acc.y *= vd;
    acc.z *= vd;
    acc.w *= vd;
    if (single) {
      const float ll = mR[h].y, inv = ll == 0.0f ? 0.0f : 1.0f / ll;  // a row whose scores are all -inf is zero
      *reinterpret_cast<uint2*>(a.out + (long long)r * a.o_rs + (long long)(h0 + h) * a.o_hs + d) =
          make_uint2(pack16(acc.x * inv, acc.y * inv, false), pack16(acc.z * inv, acc.w * inv, false));
    } else {
      *reinterpret_cast<float4*>(a.part + (((long long)r * a.H + h0 + h) * a.chunks + chunk) * HD + d) = acc;
    }
  }
}

template <int HD, int NG, bool WIDE>
fm_status launch_decode_fp4(const DecodeArgs& a, const ScaleRef& f, const NarrowRef& nr, unsigned grid, cudaStream_t s) {
  constexpr int smem = d4_smem<HD, NG>();
  const fm_status st = allow_smem<decode_fp4_kernel<HD, NG, WIDE>>(smem, "paged_decode_attn_fp4");
  if (st != FM_OK) return st;
  return launch_kernel(decode_fp4_kernel<HD, NG, WIDE>, dim3(grid), dim3(128), smem, s, true, a, f, nr);
}
template <int HD, bool WIDE>
fm_status launch_decode_fp4(const DecodeArgs& a, const ScaleRef& f, const NarrowRef& nr, int ng, unsigned grid, cudaStream_t s) {
  return ng == 2 ? launch_decode_fp4<HD, 2, WIDE>(a, f, nr, grid, s) : launch_decode_fp4<HD, 1, WIDE>(a, f, nr, grid, s);
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_paged_decode_attn_fp4_workspace_size(int64_t requests, int64_t heads, int64_t kv_heads,
                                                          int64_t head_dim, int64_t max_length, int64_t window,
                                                          int64_t sinks) {
  if (requests < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || max_length < 0 ||
      max_length > 0x7ffffff0 || window < 0 || window > 0x7ffffff0 || sinks < 0 || sinks > 0x7ffffff0)
    return 0;
  return decode_plan(requests, heads, kv_heads, head_dim, max_length, window, false, sinks, D4_RULE).total;
}

extern "C" fm_status fm_paged_decode_attn_fp4(const fm_paged_cache* cache, const fm_block_scales* scales,
                                              const fm_decode_attn* p, fm_stream stream) {
  const char* who = "paged_decode_attn_fp4";
  DecodeArgs a{};
  ScaleRef f{};
  fm_status st = cache_ref(cache, who, &a.c, true);
  if (st == FM_OK) st = scale_ref(cache, scales, who, &f);
  DecodePlan pl{};
  if (st == FM_OK) st = decode_args(cache, p, who, &a, &pl, D4_RULE);
  if (st != FM_OK) return st;
  if (p->weight_sums) return set_error(FM_ERR_UNSUPPORTED, "%s: a 4-bit cache gathers no weights", who);
  if (cache->requests == 0) return FM_OK;
  const DecodeJoin join = decode_join(cache, p, pl);
  const int64_t items = cache->requests * cache->kv_heads * pl.hgroups;
  if (items * pl.chunks > 0x7fffffff || join.blocks > 0x7fffffff) return set_error(FM_ERR_SHAPE, "%s: grid too large", who);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(items * pl.chunks);
  const NarrowRef nr = narrow_ref(a.c, f, cache->head_dim);
  if (cache->head_dim == 128)
    st = nr.fits ? launch_decode_fp4<128, false>(a, f, nr, pl.ng, grid, s) : launch_decode_fp4<128, true>(a, f, nr, pl.ng, grid, s);
  else
    st = nr.fits ? launch_decode_fp4<64, false>(a, f, nr, pl.ng, grid, s) : launch_decode_fp4<64, true>(a, f, nr, pl.ng, grid, s);
  return st != FM_OK ? st : launch_decode_join(a, join, cache->head_dim, s);
}
