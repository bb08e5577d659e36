// What the operators on a paged key/value cache share (decode_attn.cu,
// window_attn.cu, evict.cu): the cache as the kernels see it, the positions a
// query row sees, and the mma.sync fragments of bf16 and e4m3 cache rows.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "launch.cuh"

namespace fm {

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and
// m = ceil(2^(31 + s) / d), n m / 2^(31 + s) exceeds n / d by n (m d - 2^(31 + s)) /
// (d 2^(31 + s)) < 1 / d, too little to reach the next whole number.
struct Divider {
  uint32_t d, m, s;
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> (s - 1)); }
};
inline Divider make_divider(uint32_t d) {
  Divider v{d, 0, 0};
  while ((1ull << v.s) < d) ++v.s;
  v.m = (uint32_t)(((1ull << (31 + v.s)) + d - 1) / d);
  return v;
}

// Strides in bytes: a pool's offsets pass 32 bits, so every one is 64-bit.
struct CacheRef {
  uint8_t* k;
  uint8_t* v;
  long long kps, khs, kts, vps, vhs, vts;  // page, head, token
  const int* table;
  long long tstride;
  const int* lengths;
  const float* descales;  // (2, R, KH) or null
  int page, num_pages, max_len;
  int R, KH;
  Divider by_page;
  bool same;  // keys and values have the same strides: one offset serves both
};

// The length of request r, cut to what the call was sized for.
__device__ __forceinline__ int cache_length(const CacheRef& c, int r, int* err, bool report) {
  const int len = c.lengths[r];
  if (len >= 0 && len <= c.max_len) return len;
  if (report) record_error(err, DEV_BAD_INDEX);
  return len < 0 ? 0 : c.max_len;
}

// Factors of a 4-bit cache; strides in bytes.
struct ScaleRef {
  uint8_t* k;
  uint8_t* v;
  long long kps, khs, kts, vps, vhs, vts;
};

// fm_paged_cache -> CacheRef; FM_OK or the error of the first bad field.  A
// 4-bit cache is one where `fp4` says that the caller takes its factors.
inline fm_status cache_ref(const fm_paged_cache* p, const char* who, CacheRef* c, bool fp4 = false) {
  if (!p) return set_error(FM_ERR_INVALID, "%s: null cache", who);
  if (p->requests < 0 || p->kv_heads < 1 || p->page_size < 1 || p->num_pages < 0 || p->page_table_cols < 0 ||
      p->max_length < 0)
    return set_error(FM_ERR_SHAPE, "%s: bad cache shape", who);
  if (p->requests > 0x7fffffff || p->kv_heads > 65535 || p->num_pages > 0x7fffffff || p->page_size > 0x7fffffff ||
      p->max_length > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "%s: cache too large", who);
  if (p->head_dim != 64 && p->head_dim != 128) return set_error(FM_ERR_UNSUPPORTED, "%s: head_dim 64 or 128", who);
  if (fp4 ? p->dtype != FM_DT_E2M1 : p->dtype != FM_DT_BF16 && p->dtype != FM_DT_E4M3)
    return set_error(FM_ERR_INVALID, "%s: the cache is %s", who, fp4 ? "e2m1" : "bf16 or e4m3");
  if (p->requests == 0) return FM_OK;
  // a cache without a page, a table column or a position has no address to give, and none is used
  const bool holds = p->num_pages > 0 && p->page_table_cols > 0 && p->max_length > 0;
  if (!p->lengths || (holds && (!p->k || !p->v || !p->page_table)))
    return set_error(FM_ERR_INVALID, "%s: null pointer", who);
  const long long esz = p->dtype == FM_DT_BF16 ? 2 : 1;
  *c = CacheRef{static_cast<uint8_t*>(p->k), static_cast<uint8_t*>(p->v),
                p->k_page_stride * esz, p->k_head_stride * esz, p->k_token_stride * esz,
                p->v_page_stride * esz, p->v_head_stride * esz, p->v_token_stride * esz,
                p->page_table, p->page_table_stride, p->lengths, p->descales,
                (int)p->page_size, (int)p->num_pages, 0, (int)p->requests, (int)p->kv_heads,
                make_divider((uint32_t)p->page_size), false};
  // what has one page, head or token is not stepped through: its stride may be anything
  if (c->num_pages == 1) c->kps = c->vps = 0;
  if (c->KH == 1) c->khs = c->vhs = 0;
  if (c->page == 1) c->kts = c->vts = 0;
  c->same = c->kps == c->vps && c->khs == c->vhs && c->kts == c->vts;
  const long long cap = p->page_table_cols > p->max_length / p->page_size ? p->max_length
                                                                           : p->page_table_cols * p->page_size;
  c->max_len = !holds ? 0 : (int)(p->max_length < cap ? p->max_length : cap);
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || c->kps % 16 || c->khs % 16 || c->kts % 16 || c->vps % 16 ||
      c->vhs % 16 || c->vts % 16)
    return set_error(FM_ERR_ALIGN, "%s: cache rows must be 16-byte aligned", who);
  return FM_OK;
}

// fm_block_scales -> ScaleRef, of a cache that cache_ref has accepted.
inline fm_status scale_ref(const fm_paged_cache* p, const fm_block_scales* f, const char* who, ScaleRef* s) {
  if (!f) return set_error(FM_ERR_INVALID, "%s: a 4-bit cache needs its factors", who);
  if (p->requests == 0) return FM_OK;
  if (p->num_pages > 0 && p->page_table_cols > 0 && p->max_length > 0 && (!f->k || !f->v))
    return set_error(FM_ERR_INVALID, "%s: null pointer", who);
  *s = ScaleRef{static_cast<uint8_t*>(f->k), static_cast<uint8_t*>(f->v),
                f->k_page_stride, f->k_head_stride, f->k_token_stride, f->v_page_stride, f->v_head_stride, f->v_token_stride};
  if (p->num_pages == 1) s->kps = s->vps = 0;
  if (p->kv_heads == 1) s->khs = s->vhs = 0;
  if (p->page_size == 1) s->kts = s->vts = 0;
  const long long n = p->head_dim / 16;
  if ((uintptr_t)s->k % n || (uintptr_t)s->v % n || s->kps % n || s->khs % n || s->kts % n || s->vps % n || s->vhs % n ||
      s->vts % n)
    return set_error(FM_ERR_ALIGN, "%s: rows of factors must be aligned to their %d bytes", who, (int)n);
  return FM_OK;
}

// Page and token strides of a 4-bit cache in units of 16 bytes (codes) and of a
// row (factors): where offsets in these units fit 32 bits.
struct NarrowRef {
  uint32_t kp, kt, vp, vt, kfp, kft, vfp, vft;
  bool fits;
  bool same;  // one offset serves keys and values, and one their factors
};
inline NarrowRef narrow_ref(const CacheRef& c, const ScaleRef& f, long long head_dim) {
  NarrowRef n{};
  auto fits = [&](long long ps, long long ts, long long unit, uint32_t* p, uint32_t* t) {
    if (ps < 0 || ts < 0 || ps / unit > 0xffffffffll || ts / unit > 0xffffffffll) return false;
    const double most = (double)(c.num_pages > 0 ? c.num_pages - 1 : 0) * (double)ps + (double)(c.page - 1) * (double)ts;
    *p = (uint32_t)(ps / unit);
    *t = (uint32_t)(ts / unit);
    return most / (double)unit < 4.0e9;
  };
  const long long row = head_dim / 16;
  n.fits = fits(c.kps, c.kts, 16, &n.kp, &n.kt) && fits(c.vps, c.vts, 16, &n.vp, &n.vt) && fits(f.kps, f.kts, row, &n.kfp, &n.kft) &&
           fits(f.vps, f.vts, row, &n.vfp, &n.vft);
  n.same = n.kp == n.vp && n.kt == n.vt && n.kfp == n.vfp && n.kft == n.vft;
  return n;
}

// Lets kernel K have `bytes` of dynamic shared memory, once per device.
template <auto K>
inline fm_status allow_smem(int bytes, const char* who) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return FM_OK;
  const fm_status st = check_cuda(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), who);
  if (st == FM_OK) done.fetch_or(bit, std::memory_order_release);
  return st;
}

// The positions of a context of `len` that its last token sees, numbered
// 0 .. n - 1 without the gap that a window leaves after the first tokens.
struct Span {
  int head;  // positions 0 .. head - 1 come first,
  int lo;    // then lo .. lo + n - head - 1
  int n;
  __device__ __forceinline__ int pos(int i) const { return i < head ? i : i - head + lo; }
};
__host__ __device__ inline Span visible_span(int len, int window, int sinks) {
  if (window <= 0 || len <= window) return Span{0, 0, len};
  const int lo = len - window;
  const int head = sinks < lo ? sinks : lo;
  return Span{head, lo, head + window};
}

// ----------------------------------------------------------------- asynchronous copies
__device__ __forceinline__ void pc_cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void pc_cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pc_cp_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// Byte offset of 16-byte chunk `ch` of row `row` in a tile of rows of RB
// bytes, swizzled so that eight rows' same chunk, and eight chunks of a row,
// fall into different banks.
template <int RB>
__device__ __forceinline__ uint32_t row_sw(int row, int ch) {
  if constexpr (RB >= 128) return (uint32_t)(row * RB + ((ch ^ (row & 7)) << 4));
  return (uint32_t)(row * RB + ((ch ^ ((row >> 1) & 3)) << 4));  // 64-byte rows: two per 128 bytes
}

// ----------------------------------------------------------------- fragments
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// D += A B, m16n8k16; operands bf16, or f16 where HALF (an e4m3 value is exact in f16)
template <bool HALF>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (HALF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e4m3 values (low byte first) as two f16x2
__device__ __forceinline__ void e4m3x4_h(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
// four bytes of two e2m1 codes each (low half first) as f16x2; the conversion
// takes a half's low byte, so one shift brings the other two into place
__device__ __forceinline__ void e2m1x8_h(uint32_t bytes, uint32_t* h) {
  asm("{.reg .b8 a, b, c, d; .reg .b32 u; mov.b32 {a, b, c, d}, %4; cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %2, c; "
      "shr.u32 u, %4, 8; mov.b32 {a, b, c, d}, u; cvt.rn.f16x2.e2m1x2 %1, a; cvt.rn.f16x2.e2m1x2 %3, c;}"
      : "=&r"(h[0]), "=r"(h[1]), "=&r"(h[2]), "=r"(h[3])
      : "r"(bytes));
}
// two e4m3 values (low byte first) as f16x2
__device__ __forceinline__ uint32_t e4m3x2_h(uint32_t two) {
  uint32_t y;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %1; cvt.rn.f16x2.e4m3x2 %0, a;}" : "=r"(y) : "r"(two));
  return y;
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
// 2^x; results under 2^-126 are zero
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool half) {
  if (half) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&b);
}

// A query row goes to f16 times a power of two that brings its largest value
// to [2^13, 2^14): its bf16 significands fit in f16, values under 2^-38 of the
// largest round to f16's smallest steps, and with cache values of at most 448
// no fp32 score overflows.  Rows of zeros, infinities or NaN keep a factor 1.
__device__ __forceinline__ float half_row_scale(float amax) {
  if (!(amax > 0.0f && amax < INFINITY)) return 1.0f;
  int e = 13 - (int)((__float_as_uint(amax) >> 23) & 0xff) + 127;  // bf16 and fp32 share the exponent
  e = e < -126 ? -126 : e > 126 ? 126 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace fm
