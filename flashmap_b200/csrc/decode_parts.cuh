// What the kernels of one new token per request share (decode_attn.cu,
// decode_fp4.cu): their arguments, how a request is cut into chunks, and the
// launch that joins the chunks.
#pragma once

#include <algorithm>

#include "paged_cache.cuh"

namespace fm {
namespace {

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

// (maximum, sum) of a row over its n chunks, by one warp, of which the first
// 32 F have been read: those of chunks lane + 32 f.  The maximum of a row whose
// scores are all -inf comes back as 0.
template <int F>
__device__ __forceinline__ float2 row_stats(const float2* stats, int n, float2 (&first)[F]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int f = 0; f < F; ++f)
    if (lane + 32 * f >= n) first[f] = make_float2(-INFINITY, 0.0f);
  float mm = first[0].x;
#pragma unroll
  for (int f = 1; f < F; ++f) mm = fmaxf(mm, first[f].x);
  for (int c = lane + 32 * F; c < n; c += 32) mm = fmaxf(mm, stats[c].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
  const float u = mm == -INFINITY ? 0.0f : mm;
  float ll = first[0].y * ex2(first[0].x - u);
#pragma unroll
  for (int f = 1; f < F; ++f) ll += first[f].y * ex2(first[f].x - u);
  for (int c = lane + 32 * F; c < n; c += 32) {
    const float2 s = stats[c];
    ll += s.y * ex2(s.x - u);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
  return make_float2(u, ll);
}
__device__ __forceinline__ float2 row_stats(const float2* stats, int n) {
  const int lane = threadIdx.x & 31;
  float2 first[1] = {lane < n ? stats[lane] : make_float2(-INFINITY, 0.0f)};
  return row_stats(stats, n, first);
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
  // A row's length is read while the chunks are still at work: they do not write it, and since this launch's CTAs begin
  // when all of theirs have passed their own wait, nothing before them does any more.
  int row_n = 0;  // chunks of a block's row
  if (!WARP_ROWS && (int)blockIdx.x < row_blocks) {
    const Span sp = visible_span(cache_length(a.c, (int)blockIdx.x / a.H, a.err, false), a.window, a.sinks);
    const int size = chunk_of(a, sp.n);
    row_n = (sp.n + size - 1) / size;
  }
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
    const int n = row_n;
    if (n <= 1) return;  // written by its only chunk
    const int row = blockIdx.x, r = row / a.H, h = row % a.H;
    const float2* stats = a.stats + (long long)row * a.chunks;
    constexpr int V = HD / 4, PER = NT / V;  // threads per chunk's row, chunks at a time
    const float4* part = reinterpret_cast<const float4*>(a.part + (long long)row * a.chunks * HD) + tid % V;
    // The first chunks are all read at once (100003 positions of 4 bits in 74 chunks: 34.1 us, and 32.3 us so).  Reading
    // them before the length is known gains 0.3 us more, but requests of one chunk in a call that is sized for many
    // then read for nothing (8 of 200 positions sized for 131072, bf16: 8.6 us, and 7.9 us so).
    constexpr int F = 4, U = 4;
    float2 first[F];
    float4 x[U];
    float m[U];
#pragma unroll
    for (int f = 0; f < F; ++f)
      if (lane + 32 * f < n) first[f] = stats[lane + 32 * f];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (tid / V + u * PER < n) {
        x[u] = part[(long long)(tid / V + u * PER) * V];
        m[u] = stats[tid / V + u * PER].x;
      }
    const float2 st = row_stats(stats, n, first);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float top) {
      const float f = ex2(top - st.x);
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (tid / V + u * PER < n) add(x[u], m[u]);
#pragma unroll 4
    for (int c = tid / V + U * PER; c < n; c += PER) add(part[(long long)c * V], stats[c].x);
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

struct DecodeRule {
  int64_t ctas, chunk, enough;  // as above
  int64_t most, cap;            // keys of a chunk at most where that takes no more than `cap` CTAs; 0: no such bound
};
constexpr DecodeRule DA_RULE{DA_CTAS, DA_CHUNK, DA_ENOUGH, 0, 0};

DecodePlan decode_plan(int64_t R, int64_t H, int64_t KH, int64_t HD, int64_t max_len, int64_t window, bool sums,
                       int64_t sinks, const DecodeRule& rule = DA_RULE) {
  DecodePlan p{};
  const int64_t G = H / KH;
  p.ng = G > 8 ? 2 : 1;
  p.hgroups = (int)((G + 8 * p.ng - 1) / (8 * p.ng));
  const int64_t span = visible_span((int)max_len, (int)window, (int)sinks).n;
  const int64_t items = R * KH * p.hgroups;
  int64_t cut = (rule.ctas + items - 1) / items;
  if (rule.most) {
    const int64_t fine = (span + rule.most - 1) / rule.most, room = rule.cap / items;
    cut = std::max(cut, std::min(fine, room));
  }
  int64_t least = rule.enough * items / (3 * 148) / 64 * 64;
  least = least < rule.chunk ? rule.chunk : least > rule.enough ? rule.enough : least;
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

// The arguments of a call on a cache that cache_ref has accepted.
inline fm_status decode_args(const fm_paged_cache* cache, const fm_decode_attn* p, const char* who, DecodeArgs* out,
                             DecodePlan* plan, const DecodeRule& rule = DA_RULE) {
  DecodeArgs& a = *out;
  if (!p) return set_error(FM_ERR_INVALID, "%s: null arguments", who);
  if (p->heads < 1 || p->heads % cache->kv_heads || p->heads > 65535)
    return set_error(FM_ERR_SHAPE, "%s: query heads must be a multiple of the kv heads", who);
  if (p->window < 0 || p->sinks < 0 || p->window > 0x7ffffff0 || p->sinks > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "%s: window and sinks must not be negative", who);
  if (cache->requests == 0) return FM_OK;  // the caller stops here, too
  if (!p->q || !p->out) return set_error(FM_ERR_INVALID, "%s: null pointer", who);
  // one request or one head is not stepped through: its stride may be anything
  a.q_rs = cache->requests == 1 ? 0 : p->q_request_stride;
  a.q_hs = p->heads == 1 ? 0 : p->q_head_stride;
  a.o_rs = cache->requests == 1 ? 0 : p->out_request_stride;
  a.o_hs = p->heads == 1 ? 0 : p->out_head_stride;
  if ((uintptr_t)p->q % 4 || a.q_rs % 2 || a.q_hs % 2 || (uintptr_t)p->out % 8 || a.o_rs % 4 || a.o_hs % 4)
    return set_error(FM_ERR_ALIGN, "%s: query rows must be 4-byte, output rows 8-byte aligned", who);
  const bool sums = p->weight_sums != nullptr;
  *plan = decode_plan(cache->requests, p->heads, cache->kv_heads, cache->head_dim, cache->max_length,
                      p->window, sums, p->sinks, rule);
  const DecodePlan& pl = *plan;
  if (pl.total > p->workspace_bytes || (pl.total && !p->workspace))
    return set_error(FM_ERR_WORKSPACE, "%s: workspace %zu < %zu", who, p->workspace_bytes, pl.total);
  if ((uintptr_t)p->workspace % 16) return set_error(FM_ERR_ALIGN, "%s: workspace not 16-byte aligned", who);
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
  return FM_OK;
}

struct DecodeJoin {
  int64_t row_blocks, key_blocks, blocks;
  bool warp_rows;  // a warp to a row where that leaves no warp more than 16 chunks
};
inline DecodeJoin decode_join(const fm_paged_cache* cache, const fm_decode_attn* p, const DecodePlan& pl) {
  DecodeJoin j{};
  j.warp_rows = pl.chunks <= 16;
  const int nt = j.warp_rows ? 256 : 1024;
  const int64_t per = j.warp_rows ? nt / 32 : 1;
  j.key_blocks = p->weight_sums ? (pl.pitch + 4 * nt - 1) / (4 * nt) : 0;
  j.row_blocks = pl.chunks > 1 ? (cache->requests * p->heads + per - 1) / per : 0;
  j.blocks = j.row_blocks + cache->requests * cache->kv_heads * j.key_blocks;
  return j;
}
inline fm_status launch_decode_join(const DecodeArgs& a, const DecodeJoin& j, int64_t head_dim, cudaStream_t s) {
  if (j.blocks == 0) return FM_OK;  // one chunk, and no sums or no positions
  auto go = [&](auto kernel, int nt) {
    return launch_kernel(kernel, dim3((unsigned)j.blocks), dim3(nt), 0, s, true, a, (int)j.row_blocks, (int)j.key_blocks);
  };
  if (head_dim == 128)
    return j.warp_rows ? go(decode_join_kernel<128, true, 256>, 256) : go(decode_join_kernel<128, false, 1024>, 1024);
  return j.warp_rows ? go(decode_join_kernel<64, true, 256>, 256) : go(decode_join_kernel<64, false, 1024>, 1024);
}

}  // namespace
}  // namespace fm
