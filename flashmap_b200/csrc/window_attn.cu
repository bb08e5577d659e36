// Causal attention of chunks of query rows (a prompt, a verified draft) over a
// paged key/value cache, with a sliding window and first tokens that stay
// visible.
//
// The queries of request r are its last positions: row i of n stands at
// p = length - n + i and sees the keys j <= p with p - j < window or j < sinks
// (every j <= p without a window).  Query head h reads kv head h / G.
//   out = sum_j w_j v_j,  w_j = exp(s_j - max s) / sum exp(s - max s)
//
// One kernel (window_attn_kernel) of persistent CTAs, one to an SM, on the
// tcgen05 tensor cores: 256 rows of (token, query head of the group) share the
// keys and values of their kv head, so a cache row is read once for the whole
// group.  Chunks of prompts are bound by the chain S -> softmax -> P -> P V of
// the two row tiles in flight and by the exponentials (4096 rows of 32 heads on
// 12300 positions with a window of 4000: 308 us, 874 TFLOP/s of the visible
// pairs, 52 percent of a large matrix product's rate; 32768 positions without a
// window: 1040 at clocks that the power limit sets).  Calls with few rows are
// bound by the cache's bytes and the latency of a CTA's first tiles (24 x 17 rows
// on 512 .. 4096 positions: 64 us, 3.65 TB/s).
//
// A cache of 4 bits halves or quarters the bytes and adds their widening, so it
// is no faster than one of bf16: 24 x 17 rows take 68 us, of which 27 are a CTA's
// first and last tiles and 1.9 us each key tile, the chain of a loading warp over
// its 32 rows; 2 x 2048 rows on 4100 .. 6200 positions 280 to 299 us (925 to 990
// TFLOP/s of the visible pairs; a tenth less without the loading warps' work).
// The kernels of narrow caches spill 44 to 68 bytes of a thread's registers; those
// of bf16 none.
#include "paged_cache.cuh"

namespace fm {
namespace {

constexpr int WA_ROWS = 256;  // (token, head of the group) rows of a CTA, in two tiles
constexpr int WA_KEYS = 128;  // keys of a tile
constexpr int WA_LAG = 1;     // 16-bit tiles whose copies are in flight behind the newest

// What a CTA says of the items that are cut at the ends of its share.
enum { WA_NONE = 0, WA_MORE = 1, WA_LAST = 2, WA_EMPTY = 3 };
struct WaCutItem {
  int starts;              // its last item goes on in the next CTA: slot 2 b + 1
  int q0, row0, rows, c;   // which item that is
  int goes_on;             // its first item began before (slot 2 b): WA_MORE also goes on after, WA_LAST ends here
};

struct WindowArgs {
  CacheRef c;
  const uint8_t* q;  // bf16
  long long q_ts, q_hs;
  const int* cu;
  int T, H, G;
  Divider by_g;
  float scale;  // softmax_scale * log2(e)
  int window, sinks;
  __nv_bfloat16* out;
  long long o_ts, o_hs;
  float* part;    // [2 CTAs][256][HD] outputs of items that are cut, not yet divided by their sums
  float2* stats;  // [2 CTAs][256] (maximum, sum), base-2 scores
  WaCutItem* cuts;  // [CTAs], or null: items are not cut
  int row_tiles;    // no fewer than there are
  int* err;
  ScaleRef f;       // of a 4-bit cache
  NarrowRef nr;
};

// The key tiles that rows row0 .. of request r see: those of the first tokens,
// then those from the first row's window on.
struct WaKeys {
  int pos0, p_hi, lo;       // position of the request's first row, of the last row here; first key of the window
  int t_head, t_lo, tiles;  // tiles 0 .. t_head - 1, then t_lo on
};
__device__ __forceinline__ WaKeys wa_keys(const WindowArgs& a, int len, int nq, int row0) {
  WaKeys k;
  const int rows = min(WA_ROWS, nq * a.G - row0);
  k.pos0 = len - nq;  // negative: the first rows see nothing
  k.p_hi = k.pos0 + a.by_g.div(row0 + rows - 1);
  k.lo = a.window > 0 ? max(0, k.pos0 + a.by_g.div(row0) - a.window + 1) : 0;
  const int t_end = k.p_hi < 0 ? 0 : k.p_hi / WA_KEYS + 1;
  k.t_lo = k.lo / WA_KEYS;
  k.t_head = min((min(a.sinks, k.lo) + WA_KEYS - 1) / WA_KEYS, k.t_lo);
  k.tiles = max(0, k.t_head + t_end - k.t_lo);
  return k;
}
// Query rows of request r; 0 where its bounds make no sense.
__device__ __forceinline__ int wa_queries(const WindowArgs& a, int r, bool report) {
  const int q0 = a.cu[r], nq = a.cu[r + 1] - q0;
  if (q0 >= 0 && nq >= 0 && nq <= a.T - q0) return nq;
  if (report) record_error(a.err, DEV_BAD_INDEX);
  return 0;
}
__device__ __forceinline__ int wa_row_tiles(const WindowArgs& a, int nq) {
  return (int)(((long long)nq * a.G + WA_ROWS - 1) / WA_ROWS);
}

// Request and row tile that come at `tile` in the batch, or request -1; by one warp.
__device__ __forceinline__ int2 wa_find(const WindowArgs& a, int tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int r0 = 0; r0 < a.c.R; r0 += 32) {
    const int r = r0 + lane, n = r < a.c.R ? wa_row_tiles(a, wa_queries(a, r, true)) : 0;
    int scan = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, off);
      if (lane >= off) scan += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + scan > tile);
    if (hit) {
      const int w = __ffs(hit) - 1;
      return make_int2(r0 + w, tile - __shfl_sync(0xffffffffu, before + scan - n, w));
    }
    before += __shfl_sync(0xffffffffu, scan, 31);
  }
  return make_int2(-1, 0);
}

// Work is dealt out by key tiles: the items (row tile by row tile, kv head by
// kv head) lie end to end, each as long as its key tiles plus WA_ITEM for what
// an item costs besides, and every CTA takes an equal length.  An item that
// lies across a border is cut there and joined by window_join_kernel, unless
// less than WA_CUT tiles would be cut off.
constexpr int WA_ITEM = 2;
constexpr int WA_CUT = 2;
constexpr int WA_SHARE = WA_ITEM + 4;  // the least length of a CTA's share
//
// Where there are as many items as CTAs and none has WA_LONG key tiles, CTA b
// simply takes items b, b + CTAs, .. from the last row tile on (the longest of a
// prompt): no shares, no join.  Whole items fill the CTAs unevenly, which costs
// more the longer they are; shares cost their sums and the join.  Us one by one
// and in shares, 32 heads on 8 of 128, requests of one length, 64 rows each:
//   requests          500    900     1200     1600     2400     6000 positions
//         20        37 41  51 51    59 55    71 63    94 77  199 136
//         40        51 56  75 81    86 85   102 99  137 124  303 243
//         80        80 93 120 138  137 151  166 169  225 220       -
// Lengths spread over a factor of 8, and 17 rows each, part ways near there, too; 24
// prompts of 500 .. 1400 take 289 us one by one, 364 us in shares.  An item taken by
// itself is looked up among all requests, so above WA_MANY of them it is shares again
// (17 rows on 100 .. 900 positions: 300 requests 214 and 286 us, 600 438 and 527, 1200
// 1330 and 891).
constexpr int WA_LONG = 14;
constexpr int WA_MANY = 800;
struct WaBorder {
  int r, y, c, t;  // request, row tile, kv head, and the first tile after the border
};
// Where a border `o` into an item of n tiles (one, if it has none) cuts it.
__device__ __forceinline__ int wa_cut(int o, int n) {
  if (o <= 0) return 0;
  const int t = o - WA_ITEM;
  if (n < 2 * WA_CUT) return o < (n + WA_ITEM + 1) / 2 ? 0 : n;
  return t < WA_CUT ? 0 : t > n - WA_CUT ? n : t;
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
__device__ __forceinline__ void tmem_st_x2(uint32_t taddr, float x, float y) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(taddr), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void tmem_ld_x2(uint32_t taddr, float& x, float& y) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=f"(x), "=f"(y) : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A B, 16-bit operands, fp32 accumulate; A from shared memory or
// from tensor memory.  Descriptors come as their low word (address and leading
// offset in units of 16 bytes); the high word is the same for every operand
// here: stride 1024 bytes between 8-row atoms, descriptor version 1, 128-byte
// swizzling.
constexpr uint32_t WA_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(WA_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(WA_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void wa_cp_async4(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
// (loads and stores of one thread's own place or of a tile that a barrier hands over: no compiler fence between them)
__device__ __forceinline__ void wa_lds8(uint32_t at, uint32_t* v) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
}
__device__ __forceinline__ void wa_lds4(uint32_t at, uint32_t* v) { asm volatile("ld.shared.u32 %0, [%1];" : "=r"(*v) : "r"(at)); }
__device__ __forceinline__ void wa_sts16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Low descriptor words.  K-major (Q, K): the leading offset is unused.  A B
// operand stored key by key (V, 64 columns of N to a 128-byte row): the next 64
// columns follow 16384 bytes on.
__device__ __forceinline__ uint32_t desc_lo_k(uint32_t saddr) { return (saddr >> 4) | 1u << 16; }
__device__ __forceinline__ uint32_t desc_lo_mn(uint32_t saddr) { return (saddr >> 4) | (16384u >> 4) << 16; }
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p)
      :
      : "memory");
  return p != 0;
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Shared memory: two row tiles of Q and a ring of K and V tiles (16-bit,
// 128-byte swizzled in blocks of 64 columns).  Rows of 4 bits arrive in a ring of
// their own, AHEAD tiles of K or V (a tile's codes and factors for each loading
// lane) that are in flight beside the one that is widened.
template <int HD, int BITS, bool DUO>
struct WaLayout {
  static constexpr int TILE = 128 * HD * 2;  // Q, K or V tile
  static constexpr int QT = BITS == 4 && DUO ? 1 : 2;  // calls of 128 rows have one row tile
  static constexpr int SLOTS = HD == 64 ? 8 : BITS == 4 && !DUO ? 4 : 5;
  static constexpr int AHEAD = BITS == 4 ? 3 : 0;
  static constexpr int RAW = 128 * (HD / 32) * 20;  // 16 bytes of codes and 4 of factors for each of a lane's rows
  static constexpr int RING = QT * TILE + SLOTS * TILE;
  static constexpr int CTRL = RING + AHEAD * RAW;
  static constexpr int SMEM = CTRL + 3072;  // 227 KB at head_dim 128: all that a CTA may have
};

// One unit of work: 256 rows of a request and kv head, and a range of key tiles.
struct WaItem {
  int r, c;         // r < 0: no more work
  int slot;         // where its output goes if it is cut, or -1
  int q0;           // the request's first query row
  int row0, rows;   // rows row0 .. row0 + rows - 1 of its nq G
  int pos0;         // position of its first query row
  int p_hi, lo;     // the last row's position; the first key of the first row's window
  int t_first, t_head, t_lo, n;
  float scale, vd;

  __device__ __forceinline__ int key0(int j) const {  // first key of tile j
    const int t = t_first + j;
    return (t < t_head ? t : t - t_head + t_lo) * WA_KEYS;
  }
  __device__ __forceinline__ int mt() const { return rows > 128 ? 2 : 1; }
  __device__ __forceinline__ bool duo() const { return rows <= 128 && n >= 2; }
};

constexpr int WA_ITEMS = 4;              // ring of work items
constexpr int WA_REQUESTS = 16384;       // requests of a call
constexpr int WA_ROW_TILES = 4096 * 512;  // row tiles of a call

struct WaCtrl {
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_ready[2][2], o_done[2], o_empty[2], other, q_raw, q_full, q_empty, drain;
  uint64_t item_full[WA_ITEMS], item_empty[WA_ITEMS];
  int abort;
  uint32_t tmem;
  alignas(16) uint32_t valid[8][4];  // keys of tile j (mod 8) whose page exists
  float qinv[2][256];                // e4m3: what a row's query was multiplied with, inverted (items in turn)
  WaItem item[WA_ITEMS];
  WaBorder border[2];
  int scan[16];
};

// 16 warps, persistent over work items: two warpgroups of
// softmax (one to a row tile of 128), one that loads keys and values, and one
// whose warps issue the products (12), hand out work items and load queries
// (13 to 15).  S = Q K^T goes to tensor memory; the softmax threads (one to a
// row) turn it into P in place, which is the next product's A operand.  While
// one row tile is in softmax the tensor cores work on the other, and the next
// item's loads run beside the current one's products.
//
// DUO is the kernel for calls whose requests have 128 rows at most, so that an
// item has one row tile: both softmax warpgroups take its rows, each every
// other key tile, so that here, too, one is in softmax while the other's
// products run, and join their halves at the end (24 x 17 rows on 512 .. 4096
// positions: 70 us with one warpgroup, 64 us with both; in the same kernel as
// the rest it costs that 4 percent).
//
// BITS: of a cache value (16, 8 or 4).  8 and 4 bits go through the loading
// warps' registers and on as f16, which holds them exactly.
template <int HD, int BITS, bool DUO>
__global__ void __launch_bounds__(512, 1) window_attn_kernel(WindowArgs a) {
  constexpr bool KV8 = BITS < 16;
  using Lay = WaLayout<HD, BITS, DUO>;
  constexpr int TILE = Lay::TILE, SLOTS = Lay::SLOTS;
  constexpr int CPR = HD / 8;  // 16-byte chunks of a 16-bit row
  // registers: 2 x 184 + 64 + 80, or 2 x 176 + 96 + 64 where narrow rows pass
  // through the loading warps, is what 4 x 128 threads are launched with
  extern __shared__ __align__(1024) uint8_t wa_smem[];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  uint8_t* sQ = wa_smem;
  uint8_t* sKV = wa_smem + Lay::QT * TILE;
  WaCtrl* ctl = reinterpret_cast<WaCtrl*>(wa_smem + Lay::CTRL);
  if (smem_u32(wa_smem) & 1023) {  // the swizzled tiles need the alignment that the declaration asks for
    pdl_wait();
    if (tid == 0) {
      record_error(a.err, DEV_BAD_COPY);
      if (a.cuts != nullptr) a.cuts[blockIdx.x] = WaCutItem{0, 0, 0, 0, 0, WA_NONE};
    }
    return;
  }
  volatile int* abort = &ctl->abort;
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&ctl->full[i], 128);
      mbar_init(&ctl->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 2);
      mbar_init(&ctl->p_ready[i][0], 128);
      mbar_init(&ctl->p_ready[i][1], 128);
      mbar_init(&ctl->o_done[i], 1);
      mbar_init(&ctl->o_empty[i], 128);
    }
    mbar_init(&ctl->other, 128);
    mbar_init(&ctl->q_raw, 96);
    mbar_init(&ctl->q_full, KV8 ? 256 : 96);
    mbar_init(&ctl->q_empty, 1);
    mbar_init(&ctl->drain, 1);
    for (int i = 0; i < WA_ITEMS; ++i) {
      mbar_init(&ctl->item_full[i], 1);
      mbar_init(&ctl->item_empty[i], 15);  // every warp but the one that hands out
    }
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
  const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem, 0);
  pdl_wait();

  // ------------------------------------------------------------- this CTA's share
  // sum over the CTA of the values before this thread's, and of all
  // (a key tile count is under 2^24, so a warp's sum fits 32 bits)
  auto scan = [&](int v, long long* all) {
    int x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) ctl->scan[warp] = x;
    __syncthreads();
    long long before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const int y = ctl->scan[w];
      before += w < warp ? y : 0;
      sum += y;
    }
    *all = sum;
    return before + x - v;
  };
  if (a.cuts != nullptr) {
    int* pre = reinterpret_cast<int*>(sKV);                                // row tiles before request r
    long long* chunk = reinterpret_cast<long long*>(sKV + WA_REQUESTS * 4);  // length of 512 row tiles
    long long row_tiles = 0;
    for (int r0 = 0; r0 < a.c.R; r0 += 512) {
      const int r = r0 + tid;
      const int m = r < a.c.R ? wa_row_tiles(a, wa_queries(a, r, blockIdx.x == 0)) : 0;
      long long all;
      const long long before = scan(m, &all);
      if (r < a.c.R) pre[r] = (int)(row_tiles + before);
      row_tiles += all;
    }
    if (row_tiles > a.row_tiles) {  // bounds that run back, so that requests share rows: nothing is done
      if (blockIdx.x == 0 && tid == 0) record_error(a.err, DEV_BAD_INDEX);
      row_tiles = 0;
    }
    __syncthreads();
    auto tiles_of = [&](int idx, int* req, int* y) {  // key tiles of row tile idx (one, if it has none)
      int lo = 0, hi = a.c.R - 1;                     // the last request with pre[r] <= idx has it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= idx)
          lo = mid;
        else
          hi = mid - 1;
      }
      *req = lo;
      *y = idx - pre[lo];
      return max(1, wa_keys(a, cache_length(a.c, lo, a.err, false), a.cu[lo + 1] - a.cu[lo], *y * WA_ROWS).tiles);
    };
    long long total = 0, before = 0;
    int r = 0, y = 0, n = 0;  // this thread's row tile of the newest 512
    for (int i0 = 0; i0 < row_tiles; i0 += 512) {
      n = i0 + tid < row_tiles ? tiles_of(i0 + tid, &r, &y) : 0;
      long long all;
      before = scan(n ? n + WA_ITEM : 0, &all);
      if (tid == 0) chunk[i0 >> 9] = all;
      total += all;
    }
    total *= a.c.KH;
    const int shares = (int)min((long long)gridDim.x, (total + WA_SHARE - 1) / WA_SHARE);
    if (tid < 2) ctl->border[tid] = WaBorder{a.c.R, 0, 0, 0};
    __syncthreads();
    for (int e = 0; e < 2; ++e) {
      const int b = blockIdx.x + e;
      const long long x = b >= shares ? total
                          : total < (1 << 20) ? (long long)((unsigned)total * (unsigned)b / (unsigned)shares)
                                              : total * b / shares;
      if (x >= total) continue;
      int i0 = 0;
      long long at = 0;
      if (row_tiles > 512) {
        while (at + chunk[i0] * a.c.KH <= x) at += chunk[i0++] * a.c.KH;
        i0 <<= 9;
        n = i0 + tid < row_tiles ? tiles_of(i0 + tid, &r, &y) : 0;
        long long all;
        before = scan(n ? n + WA_ITEM : 0, &all);
      }
      const long long into = x - at - before * a.c.KH;
      const int w = n + WA_ITEM;
      if (n && into >= 0 && into < (long long)w * a.c.KH) {
        const int c = into < 0x7fffffff ? (int)into / w : (int)(into / w);
        ctl->border[e] = WaBorder{r, y, c, wa_cut((int)(into - (long long)c * w), n)};
      }
    }
    __syncthreads();
  }

  // item k of this CTA; r < 0 after the last, or when a wait ran out
  auto take = [&](int k) {
    WaItem w;
    if (!mbar_wait(&ctl->item_full[k % WA_ITEMS], (k / WA_ITEMS) & 1, abort)) {
      *abort = 1;
      record_error(a.err, DEV_TIMEOUT_OTHER);
      w.r = -1;
    } else {
      w = ctl->item[k % WA_ITEMS];
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl->item_empty[k % WA_ITEMS]);
    return w;
  };

  if (warp < 8) {
    regs_inc<KV8 ? 176 : 184>();
    // ------------------------------------------------------------- softmax
    const int i = warp >> 2;  // row tile
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t tS = tmem + lanes + i * 128, tO = tmem + lanes + 256 + i * 128;
    uint32_t s_phase = 0, o_phase = 0, other_phase = 0;
    int tiles = 0, worked = 0;  // key tiles and items with keys so far
    for (int k = 0;; ++k) {
      const WaItem w = take(k);
      if (w.r < 0) break;
      const bool duo = DUO && w.duo();
      const int lr = (duo ? 0 : i * 128) + (tid & 127), row = w.row0 + lr;
      const bool live = lr < w.rows;
      auto out_row = [&](int at) {
        const int tok = a.by_g.div(at);
        return a.out + (long long)(w.q0 + tok) * a.o_ts + (long long)(w.c * a.G + at - tok * a.G) * a.o_hs;
      };
      if (w.n <= 0) {  // nothing is seen
        if (live)
          for (int e = 0; e < CPR; ++e) reinterpret_cast<uint4*>(out_row(row))[e] = make_uint4(0, 0, 0, 0);
        continue;
      }
      const int tile0 = tiles, par = worked & 1;
      tiles += w.n;
      ++worked;
      if constexpr (KV8) {  // this row tile's queries to f16, each row with a power of two of its own
        if (!mbar_wait(&ctl->q_raw, par, abort)) {
          *abort = 1;
          record_error(a.err, DEV_TIMEOUT_FULL);
          break;
        }
        if (i < w.mt()) {
          const int r128 = tid & 127;
          uint8_t* qrow = sQ + i * TILE + r128 * 128;
          auto piece = [&](int e) { return reinterpret_cast<uint4*>(qrow + (e >> 3) * 16384 + (((e & 7) ^ (r128 & 7)) << 4)); };
          float amax = 0.0f;
#pragma unroll 4
          for (int e = 0; e < CPR; ++e) {
            const uint4 v = *piece(e);
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
              amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(x[q] << 16)), fabsf(__uint_as_float(x[q] & 0xffff0000u))));
          }
          const float up = half_row_scale(amax), f = w.scale > 0.0f ? up : w.scale < 0.0f ? -up : 0.0f;
#pragma unroll 4
          for (int e = 0; e < CPR; ++e) {
            const uint4 v = *piece(e);
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
            uint32_t y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              y[q] = pack16(__uint_as_float(x[q] << 16) * f, __uint_as_float(x[q] & 0xffff0000u) * f, true);
            *piece(e) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          ctl->qinv[par][i * 128 + r128] = 1.0f / up;
        }
        fence_async_smem();
        mbar_arrive(&ctl->q_full);
      }
      if (!duo && i >= w.mt()) continue;
      // Numerators in f16: the row's largest lies between 2^11 and 2^15, so that only those under 2^-25 of it meet f16's
      // coarsest steps (bf16 has fp32's range).  Without the lift 1600 keys of 2^-23 beside one with a value of 0 came
      // out 10 to 20 percent off; the shorter lag costs rescalings (12 windowed prompts on 4 bits 65 -> 67 us, long
      // chunks 278 -> 280 us).
      constexpr float LIFT = KV8 ? 11.0f : 0.0f, LAG = KV8 ? 4.0f : 8.0f;
      // sees keys up to p (a row past the end stands where the last one does, and is not written),
      const int p = w.pos0 + a.by_g.div(live ? row : w.row0 + w.rows - 1);
      const int wlo = a.window > 0 ? p - a.window + 1 : 0;  // from wlo on or below sinks
      // |scale| goes with the scores, its sign (or a zero) with the queries
      float sc = w.scale == 0.0f ? 1.0f : fabsf(w.scale);
      float m = -INFINITY, l = 0.0f;
      bool ok = true, nan = false;
      const int first = duo ? i : 0, step = duo ? 2 : 1;
      for (int j = first; j < w.n; j += step) {
        if (!mbar_wait(&ctl->s_full[i], s_phase, abort)) {
          ok = false;
          break;
        }
        s_phase ^= 1;
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld_x32(tS + q * 32, s + q * 32);
        if (KV8 && j == first) sc *= ctl->qinv[par][lr];
        const int j0 = w.key0(j);
        const uint4 vm4 = *reinterpret_cast<const uint4*>(ctl->valid[(tile0 + j) & 7]);
        const uint32_t vm[4] = {vm4.x, vm4.y, vm4.z, vm4.w};
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
        for (int e = 0; e < 128; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], s[e], s[e + 1]);
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY) * sc;
        nan |= top != top;
        // The subtracted maximum may lag behind the true one by a factor 2^LAG:
        // the numerators stay far inside their type's range, the division by
        // the sum takes the factor (and the lift) out, and O is seldom rescaled.
        const float mn = top > m + LAG || m == -INFINITY ? fmaxf(m, top) : m;
        if (__any_sync(0xffffffffu, mn != m)) {
          const float f = m == mn ? 1.0f : ex2(m - mn);
          if (j > first) {  // S is complete, so the product with the V before it is too
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
        const float neg = m == -INFINITY ? 0.0f : LIFT - m;
        const float2 sc2 = make_float2(sc, sc), neg2 = make_float2(neg, neg);
        float2 acc[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float2 x = __ffma2_rn(make_float2(s[q * 64 + 2 * e], s[q * 64 + 2 * e + 1]), sc2, neg2);
            const float2 pr = make_float2(ex2(x.x), ex2(x.y));
            acc[e & 1] = __fadd2_rn(acc[e & 1], pr);
            pk[e] = pack16(pr.x, pr.y, KV8);
          }
          tmem_st_x32(tS + q * 32, pk);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&ctl->p_ready[i][q]);  // the product may start on these 64 keys
        }
        l += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
      }
      if (!ok || !mbar_wait(&ctl->o_done[i], o_phase, abort)) {
        *abort = 1;
        record_error(a.err, DEV_TIMEOUT_ACC);
        break;
      }
      o_phase ^= 1;
      tc_fence_after();
      if (m == -INFINITY) l = 0.0f;  // no score above -inf: zero
      if (nan) l = NAN;              // a score that is no number: nor is the row
      if (duo && i == 1) {  // the other warpgroup joins the two halves; S is free by now
        tmem_st_x2(tS, m, l);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->other);
        continue;
      }
      float o[HD];
#pragma unroll
      for (int q = 0; q < HD / 32; ++q) tmem_ld_x32(tO + q * 32, o + q * 32);
      if (duo) {
        if (!mbar_wait(&ctl->other, other_phase, abort)) {
          *abort = 1;
          record_error(a.err, DEV_TIMEOUT_ACC);
          break;
        }
        other_phase ^= 1;
        tc_fence_after();
        float m1, l1;
        tmem_ld_x2(tS + 128, m1, l1);
        tmem_wait_ld();
        const float mm = fmaxf(m, m1), u = mm == -INFINITY ? 0.0f : mm, f = ex2(m - u), g = ex2(m1 - u);
        l = l * f + l1 * g;
        m = mm;
#pragma unroll
        for (int q = 0; q < HD / 16; ++q) {
          float x[16];
          tmem_ld_x16(tO + 128 + q * 16, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[q * 16 + e] = o[q * 16 + e] * f + x[e] * g;
        }
      } else {
        tmem_wait_ld();
      }
      tc_fence_before();
      mbar_arrive(&ctl->o_empty[i]);  // the next item's product may overwrite it
      if (duo) mbar_arrive(&ctl->o_empty[1]);
      if (m == -INFINITY) {  // whatever 0 times the values was
#pragma unroll
        for (int e = 0; e < HD; ++e) o[e] = 0.0f;
      }
      if (w.slot < 0) {
        const float inv = l == 0.0f ? 0.0f : w.vd / l;
        // Four lanes hand one another 16-byte pieces, so that they write 64
        // consecutive bytes of one row at a time instead of 16 of four rows.
        uint4 x[CPR];
#pragma unroll
        for (int e = 0; e < CPR; ++e) {
          x[e].x = pack16(o[8 * e] * inv, o[8 * e + 1] * inv, false);
          x[e].y = pack16(o[8 * e + 2] * inv, o[8 * e + 3] * inv, false);
          x[e].z = pack16(o[8 * e + 4] * inv, o[8 * e + 5] * inv, false);
          x[e].w = pack16(o[8 * e + 6] * inv, o[8 * e + 7] * inv, false);
        }
        auto trade = [&](uint4& lo, uint4& hi, int bit) {  // the lane with the bit gives lo, the one without hi
          const bool up = lane & bit;
          const uint4 give = up ? lo : hi;
          uint4 got;
          got.x = __shfl_xor_sync(0xffffffffu, give.x, bit);
          got.y = __shfl_xor_sync(0xffffffffu, give.y, bit);
          got.z = __shfl_xor_sync(0xffffffffu, give.z, bit);
          got.w = __shfl_xor_sync(0xffffffffu, give.w, bit);
          (up ? lo : hi) = got;
        };
#pragma unroll
        for (int e = 0; e < CPR; e += 4) {
          trade(x[e], x[e + 1], 1);
          trade(x[e + 2], x[e + 3], 1);
          trade(x[e], x[e + 2], 2);
          trade(x[e + 1], x[e + 3], 2);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // x[e + u] is piece e + lane % 4 of row u of the four
          const int at = (lr & ~3) + u;
          if (at >= w.rows) continue;
          uint4* dst = reinterpret_cast<uint4*>(out_row(w.row0 + at)) + (lane & 3);
#pragma unroll
          for (int e = 0; e < CPR; e += 4) dst[e] = x[e + u];
        }
      } else {  // piece by piece of four columns, rows side by side
        a.stats[w.slot * WA_ROWS + lr] = make_float2(m, l);
        float4* part = reinterpret_cast<float4*>(a.part) + (long long)w.slot * WA_ROWS * (HD / 4) + lr;
#pragma unroll
        for (int e = 0; e < HD / 4; ++e)
          part[e * WA_ROWS] =
              make_float4(o[4 * e] * w.vd, o[4 * e + 1] * w.vd, o[4 * e + 2] * w.vd, o[4 * e + 3] * w.vd);
      }
    }
  } else if (warp < 12) {
    regs_dec<KV8 ? 96 : 64>();
    // ------------------------------------------------------------- keys and values
    const int lw = warp - 8;  // rows 32 lw .. 32 lw + 31 of every tile
    bool ok = true;
    int slot = 0, tiles = 0;
    uint32_t phase = 1;  // an empty slot's first wait succeeds at once
    constexpr int RC = HD * BITS / 128, RPI = 32 / RC, U = 32 / RPI;  // 16-byte chunks of a cache row, rows at a time
    const int ch = lane % RC, sub = lane / RC;
    auto advance = [&]() {
      if (++slot == SLOTS) {
        slot = 0;
        phase ^= 1;
      }
    };
    int behind = 0, oldest = 0;  // entries whose copies are not handed over, and the first of them
    auto hand_over = [&]() {
      fence_async_smem();
      mbar_arrive(&ctl->full[oldest]);
      oldest = oldest + 1 == SLOTS ? 0 : oldest + 1;
      --behind;
    };
    if constexpr (BITS == 4) {
      // A stream of tiles, K and V in turn, item after item: copies run AHEAD tiles before the widening.
      constexpr int AHEAD = Lay::AHEAD;
      const uint32_t raw = smem_u32(wa_smem) + Lay::RING + (lw * 32 + lane) * 16;  // [tile][row][lane], codes and then factors
      constexpr int CODES = 128 * 16;                                              // of a row of all lanes
      const int half = (ch & 1) * 16;  // where in a word of four factors this lane's two are
      const int turn = (ch >> 1) & 1;
      const uint32_t near = turn ? 0x3232u : 0x1010u, far = 0x4242u - near;  // the factors of the half that goes first, second
      const uint32_t dst0 = smem_u32(sKV) + (ch >> 1) * 16384 + (lw * 32 + sub) * 128;
      uint32_t quarter[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) quarter[q] = (uint32_t)((((ch & 1) * 4 + (q ^ (turn * 2))) ^ (sub & 7)) << 4);
      WaItem w;
      w.n = 0;
      int k = 0, j = 0, staged = 0, in = 0, out = 0;  // next item, key tile of w, tiles in flight, places in the ring
      bool is_v = false, more = true;
      int page = -1, tok = 0, page_next = -1, tok_next = 0;  // of this key tile and the next
      const uint8_t *kcodes = nullptr, *vcodes = nullptr, *kfactors = nullptr, *vfactors = nullptr;  // of w's head, this lane's piece
      uint32_t at[U] = {}, fat[U] = {}, there = 0;  // where this lane's rows are, in NarrowRef's units
      auto lookup = [&](int t, int* at) {  // page of this lane's key of tile t; -1: none, -2: a bad one
        if (t >= w.n) return -1;
        const int key = w.key0(t) + lw * 32 + lane;
        if (key > w.p_hi || !(key >= w.lo || key < a.sinks)) return -1;
        const int pg = a.c.by_page.div(key);
        *at = key - pg * a.c.page;
        const int id = a.c.table[(long long)w.r * a.c.tstride + pg];
        if (id >= 0 && id < a.c.num_pages) return id;
        record_error(a.err, DEV_BAD_INDEX);
        return -2;
      };
      auto fetch = [&]() {  // the tile's copies; what the cache holds of rows that are not seen may be no number
        if (!is_v) {
          page = page_next;
          tok = tok_next;
          page_next = lookup(j + 1, &tok_next);
          const uint32_t good = __ballot_sync(0xffffffffu, page != -2);
          if (lane == 0) ctl->valid[tiles & 7][lw] = good;
        }
        // codes are numbers whatever they are: of a row that is not seen the first row's are as good, its factors are zero
        const uint32_t dst = raw + in * Lay::RAW, fdst = dst + U * CODES - (lw * 32 + lane) * 12;
        if (a.nr.fits) {
          if (!is_v || !a.nr.same) {
            const uint32_t pg = max(page, 0), tk = page < 0 ? 0 : tok;
            const uint32_t o = is_v ? pg * a.nr.vp + tk * a.nr.vt : pg * a.nr.kp + tk * a.nr.kt;
            const uint32_t f = is_v ? pg * a.nr.vfp + tk * a.nr.vft : pg * a.nr.kfp + tk * a.nr.kft;
            there = __ballot_sync(0xffffffffu, page >= 0) >> sub;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              at[u] = __shfl_sync(0xffffffffu, o, u * RPI + sub);
              fat[u] = __shfl_sync(0xffffffffu, f, u * RPI + sub);
            }
          }
          const uint8_t* codes = is_v ? vcodes : kcodes;
          const uint8_t* factors = is_v ? vfactors : kfactors;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            pc_cp_async16(dst + u * CODES, codes + (unsigned long long)at[u] * 16, 16u);
            wa_cp_async4(fdst + u * 512, factors + (unsigned long long)fat[u] * (HD / 16), (there >> (u * RPI)) & 1u ? 4u : 0u);
          }
        } else {
          const unsigned long long off = page < 0 ? 0ull
                                         : is_v   ? page * a.c.vps + tok * a.c.vts
                                                  : page * a.c.kps + tok * a.c.kts;
          const unsigned long long foff = page < 0 ? 0ull
                                          : is_v   ? page * a.f.vps + tok * a.f.vts
                                                   : page * a.f.kps + tok * a.f.kts;
          const uint32_t some = __ballot_sync(0xffffffffu, page >= 0) >> sub;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const unsigned long long o = __shfl_sync(0xffffffffu, off, u * RPI + sub), fo = __shfl_sync(0xffffffffu, foff, u * RPI + sub);
            pc_cp_async16(dst + u * CODES, (is_v ? vcodes : kcodes) + o, 16u);
            wa_cp_async4(fdst + u * 512, (is_v ? vfactors : kfactors) + fo, (some >> (u * RPI)) & 1u ? 4u : 0u);
          }
        }
        pc_cp_commit();
        in = in + 1 == AHEAD ? 0 : in + 1;
        ++staged;
        if (is_v) {
          ++j;
          ++tiles;
        }
        is_v = !is_v;
      };
      while (ok) {
        while (more && staged < AHEAD) {
          if (j >= w.n) {  // the next item; tiles that are in flight are handed on before this warp waits for one
            if (staged > 0 && !__all_sync(0xffffffffu, mbar_try_wait(&ctl->item_full[k % WA_ITEMS], (k / WA_ITEMS) & 1))) break;
            w = take(k++);
            if (w.r < 0) {
              more = false;
              break;
            }
            j = 0;
            kcodes = a.c.k + w.c * a.c.khs + ch * 16;
            vcodes = a.c.v + w.c * a.c.vhs + ch * 16;
            kfactors = a.f.k + w.c * a.f.khs + (ch >> 1) * 4;
            vfactors = a.f.v + w.c * a.f.vhs + (ch >> 1) * 4;
            page_next = lookup(0, &tok_next);
            continue;
          }
          fetch();
        }
        if (staged == 0) {
          if (!more) break;
          continue;
        }
        if (staged == AHEAD)
          pc_cp_wait<AHEAD - 1>();
        else
          pc_cp_wait<0>();
        if (!mbar_wait(&ctl->empty[slot], phase, abort)) {
          ok = false;
          break;
        }
        // A lane's 32 values are half of a 64-column block; which of its halves goes first (`turn`): no two lanes of two
        // rows share a bank then.
        uint32_t words[U][4], factor[U];
        const uint32_t src = raw + out * Lay::RAW;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          wa_lds8(src + u * CODES + turn * 8, words[u]);
          wa_lds8(src + u * CODES + 8 - turn * 8, words[u] + 2);
          wa_lds4(src + U * CODES - (lw * 32 + lane) * 12 + u * 512, factor + u);
        }
        const uint32_t dst = dst0 + slot * TILE;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t f2 = e4m3x2_h(factor[u] >> half), f[2] = {__byte_perm(f2, 0, near), __byte_perm(f2, 0, far)};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t h[4];
            e2m1x8_h(words[u][q], h);
            wa_sts16(dst + u * RPI * 128 + quarter[q], mul_h2(h[0], f[q >> 1]), mul_h2(h[1], f[q >> 1]), mul_h2(h[2], f[q >> 1]),
                     mul_h2(h[3], f[q >> 1]));
          }
        }
        fence_async_smem();
        mbar_arrive(&ctl->full[slot]);
        advance();
        out = out + 1 == AHEAD ? 0 : out + 1;
        --staged;
      }
    } else
    for (int k = 0; ok; ++k) {
      const WaItem w = take(k);
      if (w.r < 0) break;
      const long long trow = (long long)w.r * a.c.tstride;
      auto lookup = [&](int j, int* tok) {  // page of this lane's key of tile j; -1: none, -2: a bad one
        if (j >= w.n) return -1;
        const int key = w.key0(j) + lw * 32 + lane;
        if (key > w.p_hi || !(key >= w.lo || key < a.sinks)) return -1;
        const int pg = a.c.by_page.div(key);
        *tok = key - pg * a.c.page;
        const int page = a.c.table[trow + pg];
        if (page >= 0 && page < a.c.num_pages) return page;
        record_error(a.err, DEV_BAD_INDEX);
        return -2;
      };
      // byte offsets of this lane's key and value, -1 where there is none:
      // rows that are not seen are zero, what the cache holds there may be no number
      auto k_off = [&](int page, int tok) {
        return page < 0 ? -1ll : page * a.c.kps + (long long)w.c * a.c.khs + tok * a.c.kts;
      };
      auto v_off = [&](int page, int tok) {
        return page < 0 ? -1ll : page * a.c.vps + (long long)w.c * a.c.vhs + tok * a.c.vts;
      };
      int tok_next = 0, page_next = lookup(0, &tok_next);
      if constexpr (KV8) {
        // e4m3 rows come into registers, one tile ahead, and go on as f16, which holds them exactly
        uint4 xk[U], xv[U];
        auto fetch = [&](uint4* x, const uint8_t* from, long long off) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const long long o = __shfl_sync(0xffffffffu, off, u * RPI + sub);
            x[u] = o < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(from + o + ch * 16);
          }
        };
        auto widen = [&](const uint4* x) {
          if (!mbar_wait(&ctl->empty[slot], phase, abort)) {
            ok = false;
            return;
          }
          uint8_t* dst = sKV + slot * TILE + (ch >> 2) * 16384 + (lw * 32 + sub) * 128;
          const int c0 = (2 * ch) & 7, odd = (ch >> 2) & 1;  // which half first: no two lanes of a row share a bank
#pragma unroll
          for (int u = 0; u < U; ++u) {
            uint4 h0, h1;
            e4m3x4_h(x[u].x, h0.x, h0.y);
            e4m3x4_h(x[u].y, h0.z, h0.w);
            e4m3x4_h(x[u].z, h1.x, h1.y);
            e4m3x4_h(x[u].w, h1.z, h1.w);
            const int sw = (u * RPI + sub) & 7;
            *reinterpret_cast<uint4*>(dst + u * RPI * 128 + (((c0 + odd) ^ sw) << 4)) = odd ? h1 : h0;
            *reinterpret_cast<uint4*>(dst + u * RPI * 128 + (((c0 + 1 - odd) ^ sw) << 4)) = odd ? h0 : h1;
          }
          fence_async_smem();
          mbar_arrive(&ctl->full[slot]);
          advance();
        };
        int page = page_next, tok = tok_next;
        if (w.n > 0) fetch(xk, a.c.k, k_off(page, tok));
        for (int j = 0; j < w.n && ok; ++j, ++tiles) {
          page_next = lookup(j + 1, &tok_next);
          const uint32_t good = __ballot_sync(0xffffffffu, page != -2);
          if (lane == 0) ctl->valid[tiles & 7][lw] = good;
          fetch(xv, a.c.v, v_off(page, tok));
          widen(xk);
          page = page_next;
          tok = tok_next;
          if (j + 1 < w.n) fetch(xk, a.c.k, k_off(page, tok));
          if (ok) widen(xv);
        }
      } else {
        if (w.n <= 0) {
          // No copy of this item hands over what is behind, and the warps that wait for that take no further
          // items: without this, a run of items that see no key would fill the ring of items and stop here.
          pc_cp_wait<0>();
          while (behind > 0) hand_over();
        }
        for (int j = 0; j < w.n && ok; ++j, ++tiles) {
          const int page = page_next, tok = tok_next;
          page_next = lookup(j + 1, &tok_next);
          const uint32_t good = __ballot_sync(0xffffffffu, page != -2);
          if (lane == 0) ctl->valid[tiles & 7][lw] = good;
#pragma unroll
          for (int is_v = 0; is_v < 2; ++is_v) {
            const long long off = is_v ? v_off(page, tok) : k_off(page, tok);
            const uint8_t* from = (is_v ? a.c.v : a.c.k) + ch * 16;
            if (!mbar_wait(&ctl->empty[slot], phase, abort)) {
              ok = false;
              break;
            }
            const uint32_t dst = smem_u32(sKV) + slot * TILE + (ch >> 3) * 16384 + (lw * 32 + sub) * 128;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const long long o = __shfl_sync(0xffffffffu, off, u * RPI + sub);
              pc_cp_async16(dst + u * RPI * 128 + (((ch & 7) ^ ((u * RPI + sub) & 7)) << 4), from + (o < 0 ? 0 : o),
                            o < 0 ? 0u : 16u);
            }
            pc_cp_commit();
            advance();
            // the entry WA_LAG before this one has arrived: hand it to the tensor cores
            if (++behind > WA_LAG) {
              pc_cp_wait<WA_LAG>();
              hand_over();
            }
          }
        }
      }
    }
    pc_cp_wait<0>();  // nothing of this CTA may be in flight when it ends
    while (!KV8 && ok && behind > 0) hand_over();
    if (!ok) {
      *abort = 1;
      record_error(a.err, DEV_TIMEOUT_EMPTY);
    }
  } else {
    regs_dec<KV8 ? 64 : 80>();
    if (warp == 12) {
      // ------------------------------------------------------------- products
      // The whole warp goes through the loop, so that the operands' addresses
      // are uniform values; one lane issues.
      constexpr uint32_t ID_S = wa_idesc(KV8, 128, 128, false), ID_O = wa_idesc(KV8, 128, HD, true);
      const bool leader = elect_one();
      const uint32_t q_lo = desc_lo_k(smem_u32(sQ)), kv = smem_u32(sKV);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort)); };
      auto product_s = [&](int i, int rows_of, int slot) {
        const uint32_t qa = q_lo + rows_of * (TILE >> 4), kb = desc_lo_k(kv + slot * TILE), d = tmem + i * 128;
        if (leader) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint32_t off = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
            umma_ss(d, qa + off, kb + off, ID_S, k > 0);
          }
          mbar_arrive(&ctl->s_full[i]);  // the keys' validity words and the rows' factors, too, are there
          umma_commit(&ctl->s_full[i]);
        }
      };
      auto product_o = [&](int i, int slot, int half, uint32_t accumulate) {  // 64 keys
        const uint32_t vb = desc_lo_mn(kv + slot * TILE) + half * 512, d = tmem + 256 + i * 128;
        const uint32_t pa = tmem + i * 128 + half * 32;
        if (leader) {
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_ts(d, pa + k * 8, vb + k * 128, ID_O, k > 0 ? 1u : accumulate);
        }
      };
      auto release = [&](uint64_t* bar) {
        if (leader) umma_commit(bar);
      };
      int code = 0, slot = 0;  // slot and phase: the ring's entry that comes next in this item
      uint32_t phase = 0, q_phase = 0, p_phase[2] = {0, 0}, o_phase[2] = {1, 1};
      bool s1_read = false;  // the second S holds what the last item's epilogue still reads
      auto slot_of = [&](int e) { return slot + e >= SLOTS ? slot + e - SLOTS : slot + e; };  // e < SLOTS
      // entry e from the next one on is in shared memory
      auto filled = [&](int e) {
        if (!wait(&ctl->full[slot_of(e)], slot + e >= SLOTS ? phase ^ 1 : phase)) code = DEV_TIMEOUT_FULL;
        return !code;
      };
      auto skip = [&](int e) {
        slot += e;
        if (slot >= SLOTS) {
          slot -= SLOTS;
          phase ^= 1;
        }
      };
      auto emptied = [&](int i) {  // what row tile i of the item before left in tensor memory is read
        if (!wait(&ctl->o_empty[i], o_phase[i])) code = DEV_TIMEOUT_ACC;
        o_phase[i] ^= 1;
        return !code;
      };
      // O_i += P_i V, as P's halves arrive
      auto add_pv = [&](int i, int sv, bool fresh) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait(&ctl->p_ready[i][half], p_phase[i])) {
            code = DEV_TIMEOUT_ACC;
            return false;
          }
          tc_fence_after();
          product_o(i, sv, half, !fresh || half > 0);
        }
        p_phase[i] ^= 1;
        return true;
      };
      for (int k = 0; !code; ++k) {
        const WaItem w = take(k);
        const int r = __shfl_sync(0xffffffffu, w.r, 0), n = __shfl_sync(0xffffffffu, w.n, 0);
        const int mt = __shfl_sync(0xffffffffu, w.mt(), 0);
        const bool duo = DUO && __shfl_sync(0xffffffffu, (int)w.duo(), 0);
        if (r < 0) break;
        if (n <= 0) continue;
        if (!wait(&ctl->q_full, q_phase)) code = DEV_TIMEOUT_FULL;
        q_phase ^= 1;
        if (code || !filled(0)) break;
        tc_fence_after();
        bool early = false;  // emptied(1) is done
        if ((duo || mt == 2) && s1_read) {
          if (!emptied(1)) break;
          early = true;
          s1_read = false;
        }
        if (duo) {
          // ring entries from here: K0 V0 K1 V1 ...; warpgroup i has the key tiles j with j % 2 == i
          product_s(0, 0, slot);
          release(&ctl->empty[slot]);
          if (!filled(2)) break;
          product_s(1, 0, slot_of(2));
          release(&ctl->empty[slot_of(2)]);
          if (n == 2) release(&ctl->q_empty);
          skip(1);
          for (int j = 0; j < n; j += 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // the next entry is the V of tile j + i
              if (j + i >= n || code) break;
              if (j == 0 && !(i == 1 && early) && !emptied(i)) break;
              if (!filled(0) || !add_pv(i, slot, j == 0)) break;
              release(&ctl->empty[slot]);
              if (j + i + 2 < n) {
                if (!filled(3)) break;
                product_s(i, 0, slot_of(3));
                release(&ctl->empty[slot_of(3)]);
                if (j + i + 3 == n) release(&ctl->q_empty);
              } else {
                release(&ctl->o_done[i]);
              }
              skip(j + i + 1 < n ? 2 : 1);
            }
            if (code) break;
          }
          s1_read = true;
        } else {
          for (int i = 0; i < mt; ++i) product_s(i, i, slot);
          release(&ctl->empty[slot]);
          if (n == 1) release(&ctl->q_empty);
          skip(1);
          for (int j = 0; j < n && !code; ++j) {
            const bool more = j + 1 < n;
            if (!filled(0)) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (i >= mt || code) break;
              if (j == 0 && !(i == 1 && early) && !emptied(i)) break;
              if (!add_pv(i, slot, j == 0)) break;
              if (i == mt - 1) release(&ctl->empty[slot]);
              if (!more) {
                release(&ctl->o_done[i]);
                continue;
              }
              if (i == 0 && !filled(1)) break;
              product_s(i, i, slot_of(1));
              if (i == mt - 1) {
                release(&ctl->empty[slot_of(1)]);
                if (j + 2 == n) release(&ctl->q_empty);
              }
            }
            skip(more ? 2 : 1);
          }
        }
      }
      if (leader) {
        if (code) {
          *abort = 1;
          record_error(a.err, code);
        }
        umma_commit(&ctl->drain);  // nothing of this CTA may be in flight when it ends, whichever wait ran out
      }
      mbar_wait(&ctl->drain, 0, nullptr);
    } else {
      // ------------------------------------------------------------- work items and queries
      const bool shares = a.cuts != nullptr;
      const long long items = (long long)a.row_tiles * a.c.KH;
      long long id = blockIdx.x;  // the next item, where there are no shares
      WaBorder cur{0, 0, 0, 0}, end{a.c.R, 0, 0, 0};
      if (shares) {
        cur = ctl->border[0];
        end = ctl->border[1];
      }
      WaCutItem cut{0, 0, 0, 0, 0, WA_NONE};
      if (shares && warp == 13 && lane == 0) a.cuts[blockIdx.x] = cut;  // what the join reads where a wait runs out
      uint32_t q_phase = 1;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        WaItem w;
        if (warp == 13) {
          w.r = -1;
          while (w.r < 0 && cur.r < a.c.R) {
            if (!shares) {
              if (id >= items) break;
              const int back = (int)(id / a.c.KH);
              const int2 at = wa_find(a, a.row_tiles - 1 - back);
              cur = WaBorder{at.x, at.y, (int)(id - (long long)back * a.c.KH), 0};
              id += gridDim.x;
              if (at.x < 0) {  // the bound on the row tiles was above their number
                cur.r = 0;
                continue;
              }
            }
            const int nq = wa_queries(a, cur.r, false), row0 = cur.y * WA_ROWS;
            if (cur.y >= wa_row_tiles(a, nq)) {
              cur = WaBorder{cur.r + 1, 0, 0, 0};
              continue;
            }
            const int len = cache_length(a.c, cur.r, a.err, lane == 0);
            const WaKeys keys = wa_keys(a, len, nq, row0);
            const int tiles = max(1, keys.tiles);
            const bool last = cur.r == end.r && cur.y == end.y && cur.c == end.c;
            const int t1 = last ? end.t : tiles;
            if (cur.t < t1) {
              w.r = cur.r;
              w.c = cur.c;
              w.q0 = a.cu[cur.r];
              w.row0 = row0;
              w.rows = min(WA_ROWS, nq * a.G - row0);
              if (Lay::QT == 1 && w.rows > 128) {  // more rows than the call was sized for: there is no room for their queries
                if (lane == 0) record_error(a.err, DEV_BAD_INDEX);
                w.rows = 128;
              }
              w.pos0 = keys.pos0;
              w.p_hi = keys.p_hi;
              w.lo = keys.lo;
              w.t_first = cur.t;
              w.t_head = keys.t_head;
              w.t_lo = keys.t_lo;
              w.n = keys.tiles ? t1 - cur.t : 0;
              w.slot = cur.t > 0 ? 2 * (int)blockIdx.x : t1 < tiles ? 2 * (int)blockIdx.x + 1 : -1;
              w.scale = a.scale;
              w.vd = 1.0f;
              if (a.c.descales) {
                w.scale *= a.c.descales[(long long)w.r * a.c.KH + w.c];
                w.vd = a.c.descales[(long long)(a.c.R + w.r) * a.c.KH + w.c];
              }
              if (cur.t > 0) cut.goes_on = t1 < tiles ? WA_MORE : WA_LAST;
              if (cur.t == 0 && t1 < tiles) cut = WaCutItem{1, w.q0, w.row0, w.rows, w.c, cut.goes_on};
            } else if (cur.t > 0 && cur.t < tiles) {
              cut.goes_on = WA_EMPTY;
            }
            cur.t = 0;
            if (!shares) continue;
            if (last) {
              cur.r = a.c.R;
            } else if (++cur.c == a.c.KH) {
              cur.c = 0;
              ++cur.y;
            }
          }
          if (w.r < 0 && shares && lane == 0) a.cuts[blockIdx.x] = cut;
          if (!mbar_wait(&ctl->item_empty[k % WA_ITEMS], ((k / WA_ITEMS) & 1) ^ 1, abort)) {
            *abort = 1;
            record_error(a.err, DEV_TIMEOUT_OTHER);
            break;
          }
          if (lane == 0) {
            ctl->item[k % WA_ITEMS] = w;
            mbar_arrive(&ctl->item_full[k % WA_ITEMS]);
          }
        } else {
          w = take(k);
        }
        if (w.r < 0) break;
        if (w.n <= 0) continue;
        // the item's queries, once the one before has no product with its own to come
        if (!mbar_wait(&ctl->q_empty, q_phase, abort)) {
          *abort = 1;
          record_error(a.err, DEV_TIMEOUT_EMPTY);
          break;
        }
        q_phase ^= 1;
        constexpr int RPI = 4;  // rows of a warp at a time: eight lanes to a row, CPR / 8 pieces to a lane
        const int ch = lane & 7, rows = w.mt() * 128;
        auto chunk = [&](int lr, int blk) {
          return sQ + (lr >> 7) * TILE + blk * 16384 + (lr & 127) * 128 + ((ch ^ (lr & 7)) << 4);
        };
        const uint8_t* qbase = a.q + 2 * ((long long)w.q0 * a.q_ts + (long long)w.c * a.G * a.q_hs + ch * 8);
#pragma unroll 4
        for (int lr = (warp - 13) * RPI + (lane >> 3); lr < rows; lr += 3 * RPI) {
          const bool live = lr < w.rows;
          const int row = w.row0 + (live ? lr : 0), tok = a.by_g.div(row);
          const uint8_t* src = qbase + 2 * (tok * a.q_ts + (row - tok * a.G) * a.q_hs);
#pragma unroll
          for (int blk = 0; blk < CPR / 8; ++blk) pc_cp_async16(smem_u32(chunk(lr, blk)), src + blk * 128, live ? 16u : 0u);
        }
        pc_cp_commit();
        pc_cp_wait<0>();
        if constexpr (KV8) {  // the softmax threads turn them into f16
          mbar_arrive(&ctl->q_raw);
        } else {
          if (!(w.scale > 0.0f))
            for (int lr = (warp - 13) * RPI + (lane >> 3); lr < rows; lr += 3 * RPI)
              for (int blk = 0; blk < CPR / 8; ++blk) {
                uint4* at = reinterpret_cast<uint4*>(chunk(lr, blk));
                const uint32_t keep = w.scale < 0.0f ? ~0u : 0u, flip = w.scale < 0.0f ? 0x80008000u : 0u;
                *at = make_uint4((at->x & keep) ^ flip, (at->y & keep) ^ flip, (at->z & keep) ^ flip, (at->w & keep) ^ flip);
              }
          fence_async_smem();
          mbar_arrive(&ctl->q_full);
        }
      }
      pc_cp_wait<0>();
    }
  }
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Rows of items that were cut: block (b, y) joins columns 16 y .. 16 y + 15 of
// the item that CTA b began and left to the next ones, one thread to a row.
template <int HD>
__global__ void __launch_bounds__(WA_ROWS) window_join_kernel(WindowArgs a, int ctas) {
  pdl_wait();
  const int b = blockIdx.x, lr = threadIdx.x;
  const WaCutItem cut = a.cuts[b];
  if (!cut.starts || lr >= cut.rows) return;
  float top = -INFINITY, sum = 0.0f;
  float4 o[4] = {};
  auto add = [&](int slot) {
    const float2 st = a.stats[slot * WA_ROWS + lr];
    const float4* part = reinterpret_cast<const float4*>(a.part) + (long long)slot * WA_ROWS * (HD / 4) + lr;
    const float m = fmaxf(top, st.x), u = m == -INFINITY ? 0.0f : m, f = ex2(top - u), g = ex2(st.x - u);
    sum = sum * f + st.y * g;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 x = part[(blockIdx.y * 4 + e) * WA_ROWS];
      o[e] = make_float4(o[e].x * f + x.x * g, o[e].y * f + x.y * g, o[e].z * f + x.z * g, o[e].w * f + x.w * g);
    }
    top = m;
  };
  add(2 * b + 1);
  for (int q = b + 1; q < ctas; ++q) {
    const int goes_on = a.cuts[q].goes_on;
    if (goes_on != WA_EMPTY) add(2 * q);
    if (goes_on == WA_LAST) break;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int row = cut.row0 + lr, tok = a.by_g.div(row);
  uint4* out = reinterpret_cast<uint4*>(a.out + (long long)(cut.q0 + tok) * a.o_ts +
                                        (long long)(cut.c * a.G + row - tok * a.G) * a.o_hs + blockIdx.y * 16);
#pragma unroll
  for (int e = 0; e < 2; ++e)
    out[e] = make_uint4(pack16(o[2 * e].x * inv, o[2 * e].y * inv, false), pack16(o[2 * e].z * inv, o[2 * e].w * inv, false),
                        pack16(o[2 * e + 1].x * inv, o[2 * e + 1].y * inv, false),
                        pack16(o[2 * e + 1].z * inv, o[2 * e + 1].w * inv, false));
}

struct WindowPlan {
  int ctas;
  bool cuts;  // whether an item can be long enough to be cut
  size_t part, stats, total;
};
WindowPlan window_plan(int64_t R, int64_t T, int64_t H, int64_t KH, int64_t HD, int64_t max_q, int64_t max_len,
                       int64_t window, int64_t sinks) {
  WindowPlan p{};
  const int64_t items = (T * (H / KH) / WA_ROWS + R) * KH, sms = num_sms();
  int64_t span = max_len;
  const int64_t per = WA_ROWS / (H / KH) + 2, tokens = max_q < per ? max_q : per;  // that a row tile touches
  if (window > 0 && window + tokens + sinks < span) span = window + tokens + sinks;
  const int64_t tiles = span / WA_KEYS + 3;
  p.cuts = tiles >= (items >= sms && R <= WA_MANY ? WA_LONG : 2 * WA_CUT);
  // an item that can be cut gives work to as many CTAs as it has tiles at most
  const int64_t most = p.cuts ? items * tiles : items;
  p.ctas = (int)(most < sms ? most : sms);
  p.part = p.cuts ? (size_t)p.ctas * 2 * WA_ROWS * HD * 4 : 0;
  p.stats = p.cuts ? (size_t)p.ctas * 2 * WA_ROWS * 8 : 0;
  p.total = p.part + p.stats + (p.cuts ? (size_t)p.ctas * sizeof(WaCutItem) : 0);
  return p;
}

template <int HD, int BITS, bool DUO>
fm_status launch_window(const WindowArgs& a, const WindowPlan& pl, cudaStream_t s) {
  constexpr int smem = WaLayout<HD, BITS, DUO>::SMEM;
  static_assert(sizeof(WaCtrl) <= 3072 && smem <= 232448, "shared memory");
  fm_status st = allow_smem<window_attn_kernel<HD, BITS, DUO>>(smem, "paged_window_attn");
  if (st != FM_OK) return st;
  st = launch_kernel(window_attn_kernel<HD, BITS, DUO>, dim3((unsigned)pl.ctas), dim3(512), smem, s, true, a);
  if (st != FM_OK || !pl.cuts) return st;
  return launch_kernel(window_join_kernel<HD>, dim3((unsigned)pl.ctas, HD / 16), dim3(WA_ROWS), 0, s, true, a, pl.ctas);
}

template <int HD, int BITS>
fm_status launch_window(const WindowArgs& a, const WindowPlan& pl, bool duo, cudaStream_t s) {
  return duo ? launch_window<HD, BITS, true>(a, pl, s) : launch_window<HD, BITS, false>(a, pl, s);
}

// The arguments of a call on a cache that cache_ref has accepted.
fm_status window_args(const fm_paged_cache* cache, const fm_window_attn* p, const char* who, WindowArgs* out,
                      WindowPlan* plan) {
  WindowArgs& a = *out;
  if (!p) return set_error(FM_ERR_INVALID, "%s: null arguments", who);
  if (p->heads < 1 || p->heads % cache->kv_heads || p->heads > 65535)
    return set_error(FM_ERR_SHAPE, "%s: query heads must be a multiple of the kv heads", who);
  if (p->window < 0 || p->sinks < 0 || p->window > 0x7ffffff0 || p->sinks > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "%s: window and sinks must not be negative", who);
  if (p->rows < 0 || p->rows > 0x7ffffff0 || p->rows * p->heads > 0x7ffffff0)
    return set_error(FM_ERR_SHAPE, "%s: too many query rows", who);
  if (cache->requests == 0 || p->rows == 0) return FM_OK;  // the caller stops here, too
  if (!p->q || !p->out || !p->cu_seqlens_q) return set_error(FM_ERR_INVALID, "%s: null pointer", who);
  // one row or one head is not stepped through: its stride may be anything
  a.q_ts = p->rows == 1 ? 0 : p->q_token_stride;
  a.q_hs = p->heads == 1 ? 0 : p->q_head_stride;
  a.o_ts = p->rows == 1 ? 0 : p->out_token_stride;
  a.o_hs = p->heads == 1 ? 0 : p->out_head_stride;
  if ((uintptr_t)p->q % 16 || a.q_ts % 8 || a.q_hs % 8 || (uintptr_t)p->out % 16 || a.o_ts % 8 || a.o_hs % 8)
    return set_error(FM_ERR_ALIGN, "%s: query and output rows must be 16-byte aligned", who);
  a.q = static_cast<const uint8_t*>(p->q);
  a.cu = p->cu_seqlens_q;
  a.T = (int)p->rows;
  a.H = (int)p->heads;
  a.G = (int)(p->heads / cache->kv_heads);
  a.by_g = make_divider((uint32_t)a.G);
  a.scale = p->softmax_scale * kLog2e;
  a.window = p->window >= cache->max_length ? 0 : (int)p->window;  // so wide that it hides nothing
  a.sinks = (int)p->sinks;
  a.out = static_cast<__nv_bfloat16*>(p->out);
  a.err = p->err;
  const WindowPlan pl = *plan = window_plan(cache->requests, p->rows, p->heads, cache->kv_heads, cache->head_dim, p->max_q,
                                    cache->max_length, p->window, p->sinks);
  if (pl.total > p->workspace_bytes || (pl.total && !p->workspace))
    return set_error(FM_ERR_WORKSPACE, "%s: workspace %zu < %zu", who, p->workspace_bytes, pl.total);
  if ((uintptr_t)p->workspace % 16) return set_error(FM_ERR_ALIGN, "%s: workspace not 16-byte aligned", who);
  if (cache->requests > WA_REQUESTS || p->rows * a.G / WA_ROWS + cache->requests > WA_ROW_TILES)
    return set_error(FM_ERR_SHAPE, "%s: more than %d requests or %d row tiles", who, WA_REQUESTS, WA_ROW_TILES);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.part = reinterpret_cast<float*>(ws);
  a.stats = reinterpret_cast<float2*>(ws + pl.part);
  a.cuts = pl.cuts ? reinterpret_cast<WaCutItem*>(ws + pl.part + pl.stats) : nullptr;
  a.row_tiles = (int)(p->rows * a.G / WA_ROWS + cache->requests);
  return FM_OK;
}

}  // namespace
}  // namespace fm

using namespace fm;

extern "C" size_t fm_paged_window_attn_workspace_size(int64_t requests, int64_t rows, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_q, int64_t max_length,
                                                      int64_t window, int64_t sinks) {
  if (requests < 1 || rows < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || max_q < 0 || max_length < 0 ||
      window < 0 || window > 0x7ffffff0 || sinks < 0 || sinks > 0x7ffffff0)
    return 0;
  return window_plan(requests, rows, heads, kv_heads, head_dim, max_q, max_length, window, sinks).total;
}

extern "C" fm_status fm_paged_window_attn(const fm_paged_cache* cache, const fm_window_attn* p, fm_stream stream) {
  WindowArgs a{};
  WindowPlan pl{};
  fm_status st = cache_ref(cache, "paged_window_attn", &a.c);
  if (st == FM_OK) st = window_args(cache, p, "paged_window_attn", &a, &pl);
  if (st != FM_OK || cache->requests == 0 || p->rows == 0) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool kv8 = cache->dtype == FM_DT_E4M3, duo = p->max_q * a.G <= 128;
  if (cache->head_dim == 128) return kv8 ? launch_window<128, 8>(a, pl, duo, s) : launch_window<128, 16>(a, pl, duo, s);
  return kv8 ? launch_window<64, 8>(a, pl, duo, s) : launch_window<64, 16>(a, pl, duo, s);
}

extern "C" fm_status fm_paged_window_attn_fp4(const fm_paged_cache* cache, const fm_block_scales* scales,
                                              const fm_window_attn* p, fm_stream stream) {
  const char* who = "paged_window_attn_fp4";
  WindowArgs a{};
  WindowPlan pl{};
  fm_status st = cache_ref(cache, who, &a.c, true);
  if (st == FM_OK) st = scale_ref(cache, scales, who, &a.f);
  if (st == FM_OK) st = window_args(cache, p, who, &a, &pl);
  if (st != FM_OK || cache->requests == 0 || p->rows == 0) return st;
  a.nr = narrow_ref(a.c, a.f, cache->head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool duo = p->max_q * a.G <= 128;
  return cache->head_dim == 128 ? launch_window<128, 4>(a, pl, duo, s) : launch_window<64, 4>(a, pl, duo, s);
}
