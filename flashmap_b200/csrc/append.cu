// New tokens' keys and values into a paged cache, rotated on the way, and
// their queries rotated.
//
// With (c, s) the cosine and sine of a pair at the token's position:
//   (a, b) -> (a c - b s, b c + a s)
// in fp32, each product and sum rounded, then one rounding to the cache's type.
// A 4-bit row's 16 values share the factor f = e4m3(max |x| / 6) and become the
// e2m1 codes of x / f, both to nearest even.
//
// Every value is read and written once, so its bytes bound a prompt: 16504 tokens
// of 32 query heads on 8 of 128 into 4 bits, 72 to 75 us (4.9 to 5.1 TB/s), where a row to a
// thread, each looking its request up, took 150 us, and 113 us with three rows to
// a thread.  What is left is a warp's wait for its next four slots and the
// roundings' instructions (issue slots 59 percent; 64 registers to a thread, of
// which rotated rows into narrow caches spill 4 to 24 bytes).  A few tokens cost the chain
// of row bounds, position and cosines: 2.5 us on the GPU, less than the call's
// host time.
#include <algorithm>
#include <type_traits>

#include "paged_cache.cuh"

namespace fm {
namespace {

enum { AP_BF16 = 0, AP_E4M3 = 1, AP_FP4 = 2 };
enum { AP_PLAIN = 0, AP_HALVES = 1, AP_PAIRS = 2 };

struct AppendArgs {
  CacheRef c;
  ScaleRef f;
  const __nv_bfloat16 *k, *v, *q;
  long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs;
  __nv_bfloat16* out;
  long long o_ts, o_hs;
  int T, H;  // H: query heads, 0 without queries
  const int* cu;
  const void* pos;
  bool pos64;
  const float2* rope;
  long long rope_rows;
  int rot;
  int per, chunks;  // slots of a warp, warps of a token
  int* err;
};

// NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t y;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(y) : "f"(hi), "f"(lo));
  return y;
}
// eight values as e2m1 codes, the first in the lowest four bits
__device__ __forceinline__ uint32_t to_e2m1x8(const float* x) {
  uint32_t y;
  asm("{.reg .b8 a, b, c, d; cvt.rn.satfinite.e2m1x2.f32 a, %2, %1; cvt.rn.satfinite.e2m1x2.f32 b, %4, %3; "
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5; cvt.rn.satfinite.e2m1x2.f32 d, %8, %7; mov.b32 %0, {a, b, c, d};}"
      : "=r"(y)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return y;
}
__device__ __forceinline__ void unpack8(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Request of token t (the first whose rows end behind it), or -1; by one warp,
// which narrows the requests down to a 32nd at a time.
__device__ __forceinline__ int append_request(const AppendArgs& a, int t) {
  if (a.cu == nullptr) return t;
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.c.R;  // it is one of lo .. hi - 1, or none
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) / 32, last = min(lo + (lane + 1) * step, hi) - 1;
    const unsigned hit = __ballot_sync(0xffffffffu, a.cu[last + 1] > t);
    if (!hit) return -1;
    const int w = __ffs(hit) - 1;
    hi = min(lo + (w + 1) * step, hi);
    lo = lo + w * step;
  }
  const unsigned hit = __ballot_sync(0xffffffffu, lo + lane < hi && a.cu[lo + lane + 1] > t);
  return hit ? lo + __ffs(hit) - 1 : -1;
}

// x / d to the last bit where neither is out of range, r = 1 / d rounded: the
// rounded product is off by at most an ulp, and one step with the exact
// remainder rounds to nearest (Markstein).  inf and NaN do not come through.
__device__ __forceinline__ float ap_divide(float x, float d, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-q, d, x), r, q);
}
__device__ __forceinline__ uint4 ap_bf16x8(const float* x) {
  return make_uint4(pack16(x[0], x[1], false), pack16(x[2], x[3], false), pack16(x[4], x[5], false), pack16(x[6], x[7], false));
}

// Eight values to a thread, RPW rows to a warp at a time (a slot: rows of one
// kind, the last of a kind may be fewer).  A warp takes `per` slots of one token,
// its queries, then keys, then values: the token's request, place and cosines are
// found once for all of them, and addresses step from slot to slot.
template <int HD, int KIND, int ROPE>
__global__ void __launch_bounds__(256, 4) append_kernel(AppendArgs a) {
  constexpr int LPR = HD / 8, RPW = 32 / LPR, U = 4;  // U: slots whose rows are read at a time
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int at = lane % LPR, sub = lane / LPR, d0 = at * 8;
  const int QW = (a.H + RPW - 1) / RPW, KW = (a.c.KH + RPW - 1) / RPW, slots = QW + 2 * KW;
  const long long item = (long long)blockIdx.x * 8 + warp;
  const int t = (int)(item / a.chunks), s0 = (int)(item - (long long)t * a.chunks) * a.per, s1 = min(slots, s0 + a.per);
  const bool turned = ROPE != AP_PLAIN && d0 < a.rot;
  const int half = a.rot / 2;
  const bool first = d0 < half;  // of the two halves that are rotated into one another
  pdl_wait();
  if (a.cu != nullptr && blockIdx.x == 0)  // one block looks at all bounds: those that run back give rows to nobody
    for (int i = threadIdx.x; i < a.c.R; i += 256)
      if (a.cu[i + 1] < a.cu[i]) record_error(a.err, DEV_BAD_INDEX);
  if (t >= a.T) return;
  const int r = append_request(a, t);
  if (r < 0) return;
  const int len = a.c.lengths[r];
  int j = len - 1;  // place in the cache
  bool ok = true;
  if (a.cu != nullptr) {
    const int q0 = a.cu[r], n = a.cu[r + 1] - q0;
    ok = q0 >= 0 && n <= a.T - q0 && t >= q0 && t < q0 + n;
    j = len - n + (t - q0);
  }
  ok = ok && len >= 0 && len <= a.c.max_len;
  bool bad = !ok;
  ok = ok && j >= 0;
  long long pos = j;
  if (ROPE != AP_PLAIN && ok) {
    if (a.pos != nullptr) pos = a.pos64 ? static_cast<const long long*>(a.pos)[t] : static_cast<const int*>(a.pos)[t];
    if (pos < 0 || pos >= a.rope_rows) {
      bad = true;
      ok = false;
    }
  }
  if (bad && lane == 0) record_error(a.err, DEV_BAD_INDEX);
  if (!ok) {
    for (int s = s0; s < min(s1, QW); ++s)
      if (s * RPW + sub < a.H)
        *reinterpret_cast<uint4*>(a.out + t * a.o_ts + (s * RPW + sub) * a.o_hs + d0) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int pg = a.c.by_page.div(j), tok = j - pg * a.c.page;
  const int page = a.c.table[(long long)r * a.c.tstride + pg];
  constexpr int PAIRS = ROPE == AP_HALVES ? 8 : 4;  // of this thread's values
  float4 cs[PAIRS / 2];
  if (turned) {
    const float4* c4 = reinterpret_cast<const float4*>(a.rope + pos * half + (ROPE == AP_PAIRS ? d0 / 2 : first ? d0 : d0 - half));
#pragma unroll
    for (int i = 0; i < PAIRS / 2; ++i) {
      cs[i] = c4[i];
      if (ROPE == AP_HALVES && first) {  // a c - b s as a c + b (-s): the same bits
        cs[i].y = -cs[i].y;
        cs[i].w = -cs[i].w;
      }
    }
  }
  auto rotate = [&](float* x, const uint4& mate) {
    if (!turned) return;
    if constexpr (ROPE == AP_HALVES) {
      float y[8];
      unpack8(mate, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __fadd_rn(__fmul_rn(x[2 * i], cs[i].x), __fmul_rn(y[2 * i], cs[i].y));
        x[2 * i + 1] = __fadd_rn(__fmul_rn(x[2 * i + 1], cs[i].z), __fmul_rn(y[2 * i + 1], cs[i].w));
      }
    } else if constexpr (ROPE == AP_PAIRS) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float* z = x + 4 * i;
        const float a0 = z[0], a1 = z[2];
        z[0] = __fsub_rn(__fmul_rn(a0, cs[i].x), __fmul_rn(z[1], cs[i].y));
        z[1] = __fadd_rn(__fmul_rn(z[1], cs[i].x), __fmul_rn(a0, cs[i].y));
        z[2] = __fsub_rn(__fmul_rn(a1, cs[i].z), __fmul_rn(z[3], cs[i].w));
        z[3] = __fadd_rn(__fmul_rn(z[3], cs[i].z), __fmul_rn(a1, cs[i].w));
      }
    }
  };
  const int mate_lane = ROPE == AP_HALVES && turned ? lane + (first ? half : -half) / 8 : lane;  // holds the values that this lane's are rotated with
  // rows s .. of a kind with `heads` heads, U slots at a time: f(x, head) for each, the last slot's lanes without a row left out
  auto rows = [&](const __nv_bfloat16* src, long long hs, int from, int to, int heads, auto with_mate, auto&& f) {
    const __nv_bfloat16* row = src + (from * RPW + sub) * hs + d0;
    const long long step = RPW * hs;
    for (int s = from; s < to; s += U) {
      uint4 own[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u < to && (s + u) * RPW + sub < heads) own[u] = *reinterpret_cast<const uint4*>(row);
        row += step;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u >= to) break;
        float x[8];
        unpack8(own[u], x);
        if constexpr (decltype(with_mate)::value) {
          uint4 mate = own[u];
          if constexpr (ROPE == AP_HALVES) {
            mate.x = __shfl_sync(0xffffffffu, own[u].x, mate_lane);
            mate.y = __shfl_sync(0xffffffffu, own[u].y, mate_lane);
            mate.z = __shfl_sync(0xffffffffu, own[u].z, mate_lane);
            mate.w = __shfl_sync(0xffffffffu, own[u].w, mate_lane);
          }
          rotate(x, mate);
        }
        f(x, (s + u) * RPW + sub);
      }
    }
  };
  if (s0 < QW)
    rows(a.q + t * a.q_ts, a.q_hs, s0, min(s1, QW), a.H, std::true_type{}, [&](const float* x, int h) {
      if (h < a.H) *reinterpret_cast<uint4*>(a.out + t * a.o_ts + h * a.o_hs + d0) = ap_bf16x8(x);
    });
  if (s1 <= QW) return;
  if (page < 0 || page >= a.c.num_pages) {
    if (lane == 0) record_error(a.err, DEV_BAD_INDEX);
    return;
  }
  // a key or value row as the cache holds it
  auto put = [&](float* x, int h, uint8_t* to, long long hs, uint8_t* factors, long long fhs, const float* descales) {
    if (KIND != AP_BF16 && descales != nullptr) {
      const float d = descales[min(h, a.c.KH - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(x[i], d);
    }
    const bool live = h < a.c.KH;
    uint8_t* dst = to + h * hs;
    if constexpr (KIND == AP_BF16) {
      if (live) *reinterpret_cast<uint4*>(dst + d0 * 2) = ap_bf16x8(x);
    } else if constexpr (KIND == AP_E4M3) {
      if (live)
        *reinterpret_cast<uint2*>(dst + d0) = make_uint2(to_e4m3x2(x[0], x[1]) | to_e4m3x2(x[2], x[3]) << 16,
                                                         to_e4m3x2(x[4], x[5]) | to_e4m3x2(x[6], x[7]) << 16);
    } else {
      float top = fabsf(x[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
      constexpr float FINITE = 3.40282347e38f, SIXTH = 1.0f / 6.0f;
      if (top > FINITE) {  // an infinity counts as the largest finite value: both end at the largest factor and code
        top = FINITE;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -FINITE), FINITE);
      }
      const uint32_t factor = to_e4m3x2(ap_divide(top, 6.0f, SIXTH), 0.0f);
      const float f = __half2float(__ushort_as_half((unsigned short)(e4m3x2_h(factor) & 0xffffu)));
      const float inverse = f == 0.0f ? 0.0f : __frcp_rn(f);  // a factor of zero: codes of zero, with their sign
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = ap_divide(x[i], f, inverse);
      if (live) {
        *reinterpret_cast<uint32_t*>(dst + d0 / 2) = to_e2m1x8(x);
        if ((at & 1) == 0) factors[h * fhs + (at >> 1)] = (uint8_t)factor;
      }
    }
  };
  const float* descales = KIND != AP_BF16 && a.c.descales ? a.c.descales + (long long)r * a.c.KH : nullptr;
  if (s0 < QW + KW)
    rows(a.k + t * a.k_ts, a.k_hs, max(s0 - QW, 0), min(s1 - QW, KW), a.c.KH, std::true_type{}, [&](float* x, int h) {
      put(x, h, a.c.k + page * a.c.kps + tok * a.c.kts, a.c.khs, a.f.k + page * a.f.kps + tok * a.f.kts, a.f.khs, descales);
    });
  if (s1 > QW + KW)
    rows(a.v + t * a.v_ts, a.v_hs, max(s0 - QW - KW, 0), s1 - QW - KW, a.c.KH, std::false_type{}, [&](float* x, int h) {
      put(x, h, a.c.v + page * a.c.vps + tok * a.c.vts, a.c.vhs, a.f.v + page * a.f.vps + tok * a.f.vts, a.f.vhs,
          descales ? descales + (long long)a.c.R * a.c.KH : nullptr);
    });
}

template <int HD, int KIND, int ROPE>
fm_status launch_append(AppendArgs a, cudaStream_t s) {
  constexpr int RPW = 32 / (HD / 8);
  const int slots = (a.H + RPW - 1) / RPW + 2 * ((a.c.KH + RPW - 1) / RPW);
  // as many slots to a warp as leave every SM 32 warps
  const long long room = 148ll * 32 / a.T;
  const int chunks = (int)std::max(1ll, std::min<long long>(slots, room));
  a.per = (slots + chunks - 1) / chunks;
  a.chunks = (slots + a.per - 1) / a.per;
  const long long blocks = ((long long)a.T * a.chunks + 7) / 8;
  return launch_kernel(append_kernel<HD, KIND, ROPE>, dim3((unsigned)blocks), dim3(256), 0, s, true, a);
}
template <int HD, int KIND>
fm_status launch_append(const AppendArgs& a, int rope, cudaStream_t s) {
  return rope == AP_PLAIN    ? launch_append<HD, KIND, AP_PLAIN>(a, s)
         : rope == AP_HALVES ? launch_append<HD, KIND, AP_HALVES>(a, s)
                             : launch_append<HD, KIND, AP_PAIRS>(a, s);
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" fm_status fm_paged_append(const fm_paged_cache* cache, const fm_block_scales* scales, const fm_append* p,
                                     fm_stream stream) {
  AppendArgs a{};
  const bool fp4 = cache && cache->dtype == FM_DT_E2M1;
  fm_status st = cache_ref(cache, "paged_append", &a.c, fp4);
  if (st != FM_OK) return st;
  if (fp4 && (st = scale_ref(cache, scales, "paged_append", &a.f)) != FM_OK) return st;
  if (!p) return set_error(FM_ERR_INVALID, "paged_append: null arguments");
  if (p->tokens < 0 || p->tokens > 0x7fffffff || (p->query && (p->heads < 1 || p->heads > 65535)))
    return set_error(FM_ERR_SHAPE, "paged_append: bad shape");
  if (!p->cu_seqlens_q && p->tokens != cache->requests)
    return set_error(FM_ERR_SHAPE, "paged_append: without row bounds there is one token to a request");
  if (p->rope && (p->rotary_dim < 16 || p->rotary_dim % 16 || p->rotary_dim > cache->head_dim || p->rope_rows < 0))
    return set_error(FM_ERR_SHAPE, "paged_append: rotary_dim must be a multiple of 16 up to head_dim");
  if (p->query && !p->rope) return set_error(FM_ERR_INVALID, "paged_append: queries are taken to be rotated");
  if (p->positions && p->positions_dtype != FM_DT_I32 && p->positions_dtype != FM_DT_I64)
    return set_error(FM_ERR_INVALID, "paged_append: positions are int32 or int64");
  if (cache->dtype == FM_DT_BF16 && cache->descales)
    return set_error(FM_ERR_INVALID, "paged_append: descales go with an e4m3 or 4-bit cache");
  if (cache->requests == 0 || p->tokens == 0) return FM_OK;
  if (!p->key || !p->value || (p->query && !p->out)) return set_error(FM_ERR_INVALID, "paged_append: null pointer");
  // one token or one head is not stepped through: its stride may be anything
  const bool one = p->tokens == 1, lone = cache->kv_heads == 1;
  a.k_ts = one ? 0 : p->k_token_stride;
  a.v_ts = one ? 0 : p->v_token_stride;
  a.k_hs = lone ? 0 : p->k_head_stride;
  a.v_hs = lone ? 0 : p->v_head_stride;
  if (p->query) {
    a.q_ts = one ? 0 : p->q_token_stride;
    a.o_ts = one ? 0 : p->out_token_stride;
    a.q_hs = p->heads == 1 ? 0 : p->q_head_stride;
    a.o_hs = p->heads == 1 ? 0 : p->out_head_stride;
  }
  if ((uintptr_t)p->key % 16 || (uintptr_t)p->value % 16 || a.k_ts % 8 || a.k_hs % 8 || a.v_ts % 8 || a.v_hs % 8 ||
      (p->query && ((uintptr_t)p->query % 16 || (uintptr_t)p->out % 16 || a.q_ts % 8 || a.q_hs % 8 || a.o_ts % 8 || a.o_hs % 8)) ||
      (uintptr_t)p->rope % 16)
    return set_error(FM_ERR_ALIGN, "paged_append: rows must be 16-byte aligned");
  a.k = static_cast<const __nv_bfloat16*>(p->key);
  a.v = static_cast<const __nv_bfloat16*>(p->value);
  a.q = static_cast<const __nv_bfloat16*>(p->query);
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.T = (int)p->tokens;
  a.H = p->query ? (int)p->heads : 0;
  a.cu = p->cu_seqlens_q;
  a.pos = p->positions;
  a.pos64 = p->positions_dtype == FM_DT_I64;
  a.rope = reinterpret_cast<const float2*>(p->rope);
  a.rope_rows = p->rope_rows;
  a.rot = (int)p->rotary_dim;
  a.err = p->err;
  const int rope = !p->rope ? AP_PLAIN : p->interleaved ? AP_PAIRS : AP_HALVES;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = cache->head_dim == 128;
  if (cache->dtype == FM_DT_BF16) return wide ? launch_append<128, AP_BF16>(a, rope, s) : launch_append<64, AP_BF16>(a, rope, s);
  if (cache->dtype == FM_DT_E4M3) return wide ? launch_append<128, AP_E4M3>(a, rope, s) : launch_append<64, AP_E4M3>(a, rope, s);
  return wide ? launch_append<128, AP_FP4>(a, rope, s) : launch_append<64, AP_FP4>(a, rope, s);
}
