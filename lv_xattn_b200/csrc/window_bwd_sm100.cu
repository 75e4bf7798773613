// Backward of causal attention with a sliding window and sinks (window.cuh says which keys a query sees), 16-bit types.
//
//     S^T = K Q^T, P^T = exp2(S^T c - lse[col]), dP^T = V dO^T, dS^T = P^T o (dP^T - delta[col])
//     dV += P^T dO,  dK += dS^T Q,  dQ^T = K^T dS^T
// A work item is one 128-row key tile of one KV head; its CTA walks the 128-row query tiles that see some of its keys
// (window.cuh: the heads of a group side by side, so that few tiles are seen in part) and leaves all others alone. The
// frame, the TMEM plan (dK, dV, X: S^T -> P^T, Y: dP^T -> dQ^T, 128 columns each), the issue order and the roles are those
// of the backward block, for its measured reasons (bwd_sm100.cu): sixteen compute warps, eight drain warps for the
// reduce-adds of dQ^T (64 KB a tile, the bound of a tile: 4,900 of its 5,600 cycles), a TMA producer, an issuer. What bounds a whole
// text is its longest CTA, since a key tile is walked by one: 72 query tiles where an even share is 60 for 4,096 tokens with a window of
// 1,024, 64 where it is 29 for 2,048 causal ones (32 + 8 heads). What differs:
//   * items go out heaviest first (the first key tiles are seen by the most queries: all of them where they are sinks or
//     there is no window), forwards and backwards in turn, so that a CTA's share evens out;
//   * an item knows its own number of query tiles, possibly none;
//   * every query sees the sinks, so their key tiles would be walked long after all others are done (4,096 tokens with a
//     window of 1,024: 128 query tiles against 36). They are shared out over several items, each with a run of the queries
//     and fp32 dK and dV of its own, which the last kernel adds up in a fixed order (backward kernel of that case 400 -> 257 us);
//   * dQ is accumulated in the order of the tiles ([slab][chunk][token][head of the chunk][128]: a tile's rows are one
//     run of memory), and brought into [B, Hq, Sq, 128] by the kernel that rounds it;
//   * a thread's key is seen by a run of a tile's columns, so a masked tile costs two comparisons a tile and a select a
//     value; tiles seen whole cost none;
//   * rows of K and V behind the last valid key are cleared in shared memory: they may hold anything, and zero times
//     that would reach dQ. (A key inside must be finite: in a backward there is no other answer than NaN.)
//   * in fp16 P is made 2^14 times as large (SoftmaxRef): at most 1 as it is, behind 100,000 keys most of it is subnormal there, and
//     dV erred by 1.0e-3 instead of 3e-4;
//   * P is rounded to 16 bits for its product with dO, but dS is made from the fp32 P (dQ and dK then err by 2.4e-3 in bf16,
//     1.7e-3 of which is their own rounding; with P taken back from its 16 bits 3.0e-3). That P has to outlive the wait for
//     dP^T, 16 registers more in the compute warps. They come from the producer's and the issuer's warpgroup: 896 threads
//     are launched with 72 registers each, 512 x 80 + 256 x 72 + 128 x 40 is the same number of them. The issuer makes its
//     descriptors anew for every product, or it would not fit 40 (spilled, that cost 11 %; the drain warps with 64 instead of
//     72 cost 60 %). 258 -> 252 us for 4,096 tokens with a window of 1,024.
#include "lvx_internal.h"
#include "sm100_prims.cuh"
#include "window.cuh"
#include <math.h>
#include <algorithm>

namespace lvx {

constexpr int WB_TILE = 128 * 128 * 2;
constexpr int WB_HALF = WB_TILE / 2;
constexpr int WB_OFF_K = 0;
constexpr int WB_OFF_V = WB_TILE;
constexpr int WB_OFF_Q = 2 * WB_TILE;                     // stage s: Q at +s*2*TILE, dO right after
constexpr int WB_OFF_DS = WB_OFF_Q + 4 * WB_TILE;
constexpr int WB_OFF_STAT = WB_OFF_DS + WB_TILE;          // [2][lse2 128 | delta 128]
constexpr int WB_OFF_BAR = WB_OFF_STAT + 2 * 256 * 4;
constexpr int WB_SMEM = WB_OFF_BAR + 256;
constexpr int WB_COMPUTE = 16, WB_DRAIN_WARPS = 8;
constexpr int WB_WARP_TMA = WB_COMPUTE + WB_DRAIN_WARPS, WB_WARP_MMA = WB_WARP_TMA + 1;
constexpr int WB_THREADS = (WB_WARP_MMA + 3) * 32;      // two idle warps make the last warpgroup whole (setmaxnreg)
static_assert(WB_SMEM <= 232448, "shared memory budget");
constexpr uint32_t WB_DK = 0, WB_DV = 128, WB_X = 256, WB_Y = 384;

enum {
  WBB_KV_FULL = 0,
  WBB_KV_CLEAN,                         // rows behind the last valid key are cleared (items that have such rows)
  WBB_Q_FULL,                           // x2
  WBB_Q_EMPTY = WBB_Q_FULL + 2,         // x2
  WBB_S_FULL = WBB_Q_EMPTY + 2,
  WBB_DP_FULL,
  WBB_X_LOADED,
  WBB_P_FULL,
  WBB_DS_FREE,
  WBB_PDS_FULL,
  WBB_DQ_FULL,
  WBB_DQ_FREE,
  WBB_ACC_DONE,
  WBB_DRAIN,
  WBB_STAT_FULL,                        // x2
  WBB_COUNT = WBB_STAT_FULL + 2
};
#define WB_CODE(role, bar) (LVX_DEV_TIMEOUT_BASE | 0x500 | ((role) << 5) | (bar))

// Key tiles [0, tiles) are walked by `parts` items each.
struct SinkParts {
  int tiles, parts;
};

struct WinBwdParams {
  int sq, skv, hkv, g, slabs, nitems;
  SinkParts sp;
  float* parts;                        // [slab][sink tile][part][dK, dV][128][128]
  QTiles qt;
  WindowMask mask;
  const int32_t* kv_valid_len;
  const float *lse, *delta;            // [B*Hq, Sq]
  float scale, scale_log2;
  float* dq_acc;
  uint16_t *dk, *dv;                   // dense [B, Hkv, Skv, 128]
  int* status;
};

template <bool IS_BF16>
__global__ void __launch_bounds__(WB_THREADS, 1)
window_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                  const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const WinBwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WB_OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + WBB_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_stat = reinterpret_cast<float*>(smem + WB_OFF_STAT);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dep_wait();      // delta and the cleared accumulator, and what packs the rows of a shared prefix
  grid_dep_launch();
  const int heads = p.qt.heads, tile_rows = heads * p.qt.tokens;
  struct Item {
    int slab, kv0, valid, start;
    int blk0, ntot;          // first block of tokens, tiles to walk
    int part;                // index into `parts`, or -1: the item makes dK and dV itself
  };
  // the CTA's round-th item: forwards and backwards through the list in turn
  auto index_of = [&](int round) {
    return round * int(gridDim.x) + ((round & 1) ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x));
  };
  auto item_of = [&](int w) {
    Item it;
    it.slab = w % p.slabs;
    int tile = w / p.slabs;
    it.part = -1;
    const int shared_out = p.sp.tiles * p.sp.parts;
    if (tile < shared_out) {
      it.part = it.slab * shared_out + tile;
      tile /= p.sp.parts;
    } else {
      tile += p.sp.tiles - shared_out;
    }
    it.kv0 = tile * 128;
    it.valid = p.skv;
    if (p.kv_valid_len) it.valid = min(it.valid, max(0, p.kv_valid_len[it.slab / p.hkv]));
    it.start = p.mask.start >= 0 ? p.mask.start : it.valid - p.sq;
    const int ta = max(0, it.kv0 - it.start);
    const int tb = it.kv0 < p.mask.sinks ? p.sq : min(p.sq, it.kv0 + 127 - it.start + p.mask.window);
    it.blk0 = ta / p.qt.tokens;
    int blocks = it.kv0 < it.valid && ta < tb ? (tb - 1) / p.qt.tokens + 1 - it.blk0 : 0;
    if (it.part >= 0) {
      const int each = (blocks + p.sp.parts - 1) / p.sp.parts, first = it.part % p.sp.parts * each;
      it.blk0 += first;
      blocks = max(0, min(each, blocks - first));
    }
    it.ntot = blocks * p.qt.chunks;
    return it;
  };
  // first token and chunk of an item's j-th tile
  auto tile_tok = [&](const Item& it, int j) { return (it.blk0 + j / p.qt.chunks) * p.qt.tokens; };
  auto tile_chunk = [&](int j) { return j % p.qt.chunks; };

  const bool misaligned = (smem_u32(smem) & 1023u) != 0;      // the operand descriptors assume 1024-byte aligned tiles
  if (misaligned && tid == 0) atomicCAS(p.status, 0, WB_CODE(7, 0));
  // the status word may be set at any moment: one thread reads it, and the CTA leaves or stays as a whole
  int word = misaligned;
  if (tid == 0) word |= *reinterpret_cast<volatile int*>(p.status);

  if (tid == 0) {
    for (int b = 0; b < WBB_COUNT; ++b)
      mbar_init(&bars[b], b == WBB_X_LOADED || b == WBB_P_FULL || b == WBB_PDS_FULL || b == WBB_KV_CLEAN ? WB_COMPUTE
                          : b == WBB_DQ_FREE                                                             ? WB_DRAIN_WARPS
                          : b >= WBB_STAT_FULL                                                           ? 8
                                                                                                         : 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // the rows of Q and dO tiles that no box fills (groups whose size does not divide 128)
  for (int i = tid; i < (128 - tile_rows) * 8 * 8; i += WB_THREADS)
    reinterpret_cast<uint4*>(smem + WB_OFF_Q + (i & 7) * WB_HALF)[tile_rows * 8 + (i >> 3)] = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  if (warp == WB_WARP_MMA) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  const bool poisoned = __syncthreads_or(word) != 0;
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Every role walks the same items in the same order and keeps the same counters: `it` = items with tiles done, `jj0` =
  // tiles done before the current item, `cleaned` = items whose K and V were cleared in part.
  if (warp < WB_COMPUTE) {
    // =========================== compute warps ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 80;" ::: "memory");
    const int quarter = warp & 3;                         // TMEM lane quarter
    const int cg = warp >> 2;                             // 32-column group of the query tile
    const int r = quarter * 32 + lane;                    // key inside the tile
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tX = tmem_base + WB_X + lane_sel, tY = tmem_base + WB_Y + lane_sel;
    const float c = p.scale_log2;
    using Ref = SoftmaxRef<IS_BF16>;
    // dS = P (dP - delta): in fp16 P is grad_gain times as large as it is, and the statistics' delta as much smaller
    auto ds = [](uint32_t pv, uint32_t dp, float dl) {
      const float x = __uint_as_float(dp);
      return __uint_as_float(pv) * (IS_BF16 ? x - dl : fmaf(x, 1.f / Ref::grad_gain, -dl));
    };
    bool alive = !poisoned;
    int it = 0, jj0 = 0;
    for (int round = 0, w; alive && (w = index_of(round)) < p.nitems; ++round) {
      const Item I = item_of(w);
      if (I.ntot == 0) {      // nothing sees these keys (or they are not valid): their gradients are zero
        if (I.part >= 0) {
          float4* dst = reinterpret_cast<float4*>(p.parts + size_t(I.part) * 2 * 128 * 128);
          for (int i = tid; i < 2 * 128 * 32; i += WB_COMPUTE * 32) dst[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else if (warp < 8 && I.kv0 + (tid & 127) < p.skv) {
          uint4* dst = reinterpret_cast<uint4*>((warp < 4 ? p.dk : p.dv) + (size_t(I.slab) * p.skv + I.kv0 + (tid & 127)) * 128);
#pragma unroll
          for (int i = 0; i < 16; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        continue;
      }
      // Statistics of a tile's columns: threads 0-127 fetch lse, 128-255 delta.
      auto fetch_stat = [&](int j) -> float {
        if (tid >= 256) return 0.f;
        const int col = tid & 127, tok = tile_tok(I, j) + col / heads, head = tile_chunk(j) * heads + col % heads;
        const bool exists = col < tile_rows && tok < p.sq && head < p.g;
        const size_t at = (size_t(I.slab) * p.g + head) * p.sq + tok;
        if (tid >= 128) return exists ? p.delta[at] * (1.f / Ref::grad_gain) : 0.f;
        float v = INFINITY;       // +inf => P = 0: a query that does not exist, or that sees nothing
        if (exists) {
          v = p.lse[at] * 1.4426950408889634f;
          v = v == -INFINITY ? INFINITY : v - Ref::grad_bits;
        }
        return v;
      };
      auto put_stat = [&](int jj, float v) {
        if (tid >= 256) return;
        s_stat[(jj & 1) * 256 + tid] = v;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[WBB_STAT_FULL + (jj & 1)]);
      };
      put_stat(jj0, fetch_stat(0));
      float stat_next = I.ntot > 1 ? fetch_stat(1) : 0.f;
      if (I.valid < min(p.skv, I.kv0 + 128)) {      // rows that are there but not valid
        if (!mbar_wait(&bars[WBB_KV_FULL], it & 1, abort_flag, p.status, WB_CODE(0, WBB_KV_FULL))) {
          alive = false;
          break;
        }
        const int left = I.valid - I.kv0;
        for (int i = tid; i < (128 - left) * 8 * 4; i += WB_COMPUTE * 32)
          reinterpret_cast<uint4*>(smem + WB_OFF_K + (i & 3) * WB_HALF)[left * 8 + (i >> 2)] = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[WBB_KV_CLEAN]);
      }
      // The queries that see this thread's key: tokens from `from` on, up to `to`.
      const int key = I.kv0 + r;
      const int from = key < I.valid ? key - I.start : kNoWindow;
      const int to = key < p.mask.sinks ? kNoWindow : key - I.start + p.mask.window;
      for (int j = 0; j < I.ntot; ++j) {
        const int jj = jj0 + j;
        float stat_after = 0.f;
        if (j + 2 < I.ntot) stat_after = fetch_stat(j + 2);
        // ---------------- P^T half: needs S^T only ----------------
        if (!mbar_wait(&bars[WBB_S_FULL], jj & 1, abort_flag, p.status, WB_CODE(0, WBB_S_FULL))) {
          alive = false;
          break;
        }
        tc_fence_after();
        uint32_t s[32];
        tmem_ld32(tX + cg * 32, s);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[WBB_X_LOADED]);
        if (!mbar_wait(&bars[WBB_STAT_FULL + (jj & 1)], (jj >> 1) & 1, abort_flag, p.status, WB_CODE(0, WBB_STAT_FULL))) {
          alive = false;
          break;
        }
        // of the warp's 32 columns, those that see the key; a tile that all see is not masked
        uint32_t seen;
        {
          const int tok0 = tile_tok(I, j);
          const int c0 = min(max(from - tok0, 0), 128) * heads - cg * 32, c1 = min(max(to - tok0, 0), 128) * heads - cg * 32;
          seen = low_bits(clamp32(c1)) & ~low_bits(clamp32(c0));
        }
        const bool masked = __any_sync(0xffffffffu, seen != 0xffffffffu);
        const float4* sl = reinterpret_cast<const float4*>(s_stat + (jj & 1) * 256 + cg * 32);
        const float4* sd = reinterpret_cast<const float4*>(s_stat + (jj & 1) * 256 + 128 + cg * 32);
#pragma unroll
        for (int i = 0; i < 8; ++i) {      // s becomes P, which stays in fp32 for dS
          const float4 l2 = sl[i];
          s[4 * i] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[4 * i]), c, -l2.x)));
          s[4 * i + 1] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[4 * i + 1]), c, -l2.y)));
          s[4 * i + 2] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[4 * i + 2]), c, -l2.z)));
          s[4 * i + 3] = __float_as_uint(ex2f(fmaf(__uint_as_float(s[4 * i + 3]), c, -l2.w)));
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen & (1u << i))) s[i] = 0u;
        }
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          pk[i] = IS_BF16 ? pack_bf16x2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]))
                          : pack_f16x2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
        // P^T overwrites S^T in X: wait until every warp has taken its S^T columns out.
        if (!mbar_wait(&bars[WBB_X_LOADED], jj & 1, abort_flag, p.status, WB_CODE(0, WBB_X_LOADED))) {
          alive = false;
          break;
        }
        tmem_st16(tX + cg * 16, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[WBB_P_FULL]);      // dV of this tile may start
        // ---------------- dS^T half: needs dP^T ----------------
        if (!mbar_wait(&bars[WBB_DP_FULL], jj & 1, abort_flag, p.status, WB_CODE(0, WBB_DP_FULL))) {
          alive = false;
          break;
        }
        tc_fence_after();
        uint32_t dsk[16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t dp[16];
          tmem_ld16(tY + cg * 32 + h * 16, dp);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 dl = sd[h * 4 + i];
            const float d0 = ds(s[h * 16 + 4 * i], dp[4 * i], dl.x), d1 = ds(s[h * 16 + 4 * i + 1], dp[4 * i + 1], dl.y);
            const float d2 = ds(s[h * 16 + 4 * i + 2], dp[4 * i + 2], dl.z), d3 = ds(s[h * 16 + 4 * i + 3], dp[4 * i + 3], dl.w);
            dsk[h * 8 + 2 * i] = IS_BF16 ? pack_bf16x2(d0, d1) : pack_f16x2(d0, d1);
            dsk[h * 8 + 2 * i + 1] = IS_BF16 ? pack_bf16x2(d2, d3) : pack_f16x2(d2, d3);
          }
        }
        tc_fence_before();
        if (jj > 0 && !mbar_wait(&bars[WBB_DS_FREE], (jj - 1) & 1, abort_flag, p.status, WB_CODE(0, WBB_DS_FREE))) {
          alive = false;
          break;
        }
        {
          uint8_t* rowp = smem + WB_OFF_DS + (cg >> 1) * WB_HALF + r * 128;
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
            *reinterpret_cast<uint4*>(rowp + ((((cg & 1) * 4 + ch) ^ (r & 7)) << 4)) =
                make_uint4(dsk[4 * ch], dsk[4 * ch + 1], dsk[4 * ch + 2], dsk[4 * ch + 3]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[WBB_PDS_FULL]);
        if (j + 1 < I.ntot) put_stat(jj + 1, stat_next);
        stat_next = stat_after;
      }
      // ------------------------------- dK / dV of the item -------------------------------
      if (alive) alive = mbar_wait(&bars[WBB_ACC_DONE], it & 1, abort_flag, p.status, WB_CODE(0, WBB_ACC_DONE));
      alive = __all_sync(0xffffffffu, alive);
      tc_fence_after();
      if (alive) {
        // A thread's 64 bytes of a row go through the warp's own part of the dS^T tile (which nothing reads until this warp
        // writes it again), so that a store covers whole sectors. Written by row they were 16-byte pieces 256 bytes apart,
        // and the write-out took 12,000 cycles beside the reduce-adds instead of 3,000.
        uint8_t* stage = smem + WB_OFF_DS + (cg >> 1) * WB_HALF + quarter * 32 * 128;
        const size_t off = (size_t(I.slab) * p.skv + I.kv0 + quarter * 32) * 128 + cg * 32;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          uint32_t a[32];
          tmem_ld32(tmem_base + (which ? WB_DV : WB_DK) + lane_sel + cg * 32, a);
          tc_wait_ld();
          const float mul = which ? 1.f / Ref::grad_gain : p.scale;
          if (I.part >= 0) {
            float4* dst = reinterpret_cast<float4*>(p.parts + ((size_t(I.part) * 2 + which) * 128 + r) * 128 + cg * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i] = make_float4(__uint_as_float(a[4 * i]) * mul, __uint_as_float(a[4 * i + 1]) * mul,
                                   __uint_as_float(a[4 * i + 2]) * mul, __uint_as_float(a[4 * i + 3]) * mul);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t wd[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float lo = __uint_as_float(a[8 * i + 2 * e]) * mul, hi = __uint_as_float(a[8 * i + 2 * e + 1]) * mul;
                wd[e] = IS_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
              }
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((((cg & 1) * 4 + i) ^ (lane & 7)) << 4)) = make_uint4(wd[0], wd[1], wd[2], wd[3]);
            }
            __syncwarp();
            uint16_t* dst = (which ? p.dv : p.dk) + off;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rr = i * 8 + (lane >> 2), piece = lane & 3;
              if (I.kv0 + quarter * 32 + rr < p.skv)
                *reinterpret_cast<uint4*>(dst + rr * 128 + piece * 8) =
                    *reinterpret_cast<const uint4*>(stage + rr * 128 + ((((cg & 1) * 4 + piece) ^ (rr & 7)) << 4));
            }
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      ++it;
      jj0 += I.ntot;
    }
  } else if (warp < WB_WARP_TMA) {
    // =========================== dQ drain warps ===========================
    const int quarter = warp & 3;
    const int ch = (warp - WB_COMPUTE) >> 2;              // which 64 query columns
    const int d = quarter * 32 + lane;                    // head-dim index = TMEM lane of dQ^T
    const uint32_t tY = tmem_base + WB_Y + (static_cast<uint32_t>(quarter * 32) << 16);
    bool alive = !poisoned;
    int jj0 = 0;
    for (int round = 0, w; alive && (w = index_of(round)) < p.nitems; ++round) {
      const Item I = item_of(w);
      for (int j = 0; j < I.ntot; ++j) {
        const int jj = jj0 + j;
        if (!mbar_wait(&bars[WBB_DQ_FULL], jj & 1, abort_flag, p.status, WB_CODE(1, WBB_DQ_FULL))) {
          alive = false;
          break;
        }
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld32(tY + ch * 64, v[0]);
        tmem_ld32(tY + ch * 64 + 32, v[1]);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[WBB_DQ_FREE]);     // Y is free for the next tile's dP^T
        const int tok0 = tile_tok(I, j);
        const int ncols = min(tile_rows, (p.sq - tok0) * heads) - ch * 64;
        float* dst = p.dq_acc + ((size_t(I.slab) * p.qt.chunks + tile_chunk(j)) * p.sq * heads + size_t(tok0) * heads + ch * 64) * 128 + d;
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (i < ncols) atomicAdd(dst + size_t(i) * 128, __uint_as_float(v[i >> 5][i & 31]) * p.scale);
      }
      jj0 += I.ntot;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;" ::: "memory");
    if (warp == WB_WARP_TMA) {
      // =========================== TMA producer ===========================
      if (lane == 0 && !poisoned) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmDO);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        int issued = 0, kv_loads = 0;
        bool alive = true;
        int it = 0, jj0 = 0;
        for (int round = 0, w; alive && (w = index_of(round)) < p.nitems; ++round) {
          const Item I = item_of(w);
          if (I.ntot == 0) continue;
          const int kvh = I.slab % p.hkv, batch = I.slab / p.hkv;
          for (int j = 0; j < I.ntot; ++j) {
            const int jj = jj0 + j;
            const int s = jj & 1;
            if (!mbar_wait(&bars[WBB_Q_EMPTY + s], ((jj >> 1) & 1) ^ 1, abort_flag, p.status, WB_CODE(2, WBB_Q_EMPTY))) {
              alive = false;
              break;
            }
            uint8_t* dst = smem + WB_OFF_Q + s * 2 * WB_TILE;
            const int tok0 = tile_tok(I, j), head0 = tile_chunk(j) * heads;
            mbar_arrive_expect_tx(&bars[WBB_Q_FULL + s], 2 * tile_rows * 256);
            for (int h = 0; h < 2; ++h) {
              tma_load_5d(dst + h * WB_HALF, &tmQ, &bars[WBB_Q_FULL + s], h * 64, head0, tok0, kvh, batch);
              tma_load_5d(dst + WB_TILE + h * WB_HALF, &tmDO, &bars[WBB_Q_FULL + s], h * 64, head0, tok0, kvh, batch);
            }
            issued = jj + 1;
            if (j == 0) {
              // the item's K and V go in once the previous item's products have all completed
              if (it > 0 && !mbar_wait(&bars[WBB_ACC_DONE], (it - 1) & 1, abort_flag, p.status, WB_CODE(2, WBB_ACC_DONE))) {
                alive = false;
                break;
              }
              mbar_arrive_expect_tx(&bars[WBB_KV_FULL], 2 * WB_TILE);
              for (int h = 0; h < 2; ++h) {
                tma_load_4d(smem + WB_OFF_K + h * WB_HALF, &tmK, &bars[WBB_KV_FULL], h * 64, I.kv0, kvh, batch);
                tma_load_4d(smem + WB_OFF_V + h * WB_HALF, &tmV, &bars[WBB_KV_FULL], h * 64, I.kv0, kvh, batch);
              }
              ++kv_loads;
            }
          }
          ++it;
          jj0 += I.ntot;
        }
        if (*abort_flag) {      // let the copies in flight land before the CTA's shared memory goes away
          auto drain = [&](uint64_t* bar, uint32_t ph) {
            const long long t0 = clock64();
            while (!mbar_try_wait(bar, ph) && clock64() - t0 < LVX_SPIN_LIMIT_CYCLES) {}
          };
          if (kv_loads > 0) drain(&bars[WBB_KV_FULL], (kv_loads - 1) & 1);
          for (int jj = max(0, issued - 2); jj < issued; ++jj) drain(&bars[WBB_Q_FULL + (jj & 1)], (jj >> 1) & 1);
        }
      }
    } else if (warp == WB_WARP_MMA) {
      // =========================== MMA issuer ===========================
      if (lane == 0 && !poisoned) {
        constexpr uint32_t FMT = IS_BF16 ? UMMA_BF16 : UMMA_F16;
        constexpr uint32_t IDESC_ST = umma_idesc(FMT, UMMA_K_MAJOR, UMMA_K_MAJOR, 128, 128);
        constexpr uint32_t IDESC_ACC = umma_idesc(FMT, UMMA_K_MAJOR, UMMA_MN_MAJOR, 128, 128);
        constexpr uint32_t IDESC_DQ = umma_idesc(FMT, UMMA_MN_MAJOR, UMMA_MN_MAJOR, 128, 128);
        constexpr uint32_t HI = umma_desc_hi(1024);
        const uint32_t sK = smem_u32(smem + WB_OFF_K), sV = smem_u32(smem + WB_OFF_V);
        const uint32_t sQ0 = smem_u32(smem + WB_OFF_Q), sDS = smem_u32(smem + WB_OFF_DS);
        auto q_at = [&](int jj) { return sQ0 + (jj & 1) * 2 * WB_TILE; };
        // The descriptors are made anew for every product (one addition an instruction): kept over the loop, as the compiler
        // would have them, they do not fit this warp's registers.
        auto desc = [](uint32_t smem_addr, uint32_t lead) {
          uint32_t lo = umma_desc_lo(smem_addr, lead);
          asm volatile("" : "+r"(lo));
          return lo;
        };
        // D[128 kv, 128 q] = A[128 kv, 128 d] * B[128 q, 128 d]^T, both K-major
        auto issue_st = [&](uint32_t d_tmem, uint32_t a_smem, uint32_t b_smem) {
          const uint32_t a_lo = desc(a_smem, 16), b_lo = desc(b_smem, 16);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = ((kk >> 2) * WB_HALF + (kk & 3) * 32) >> 4;
            umma_ss_f16(d_tmem, umma_desc_join(a_lo + off, HI), umma_desc_join(b_lo + off, HI), IDESC_ST, kk > 0);
          }
        };
        // dV[128 kv, 128 d] += P^T (TMEM) * dO (MN-major: rows are q)
        auto issue_dv = [&](uint32_t b_smem, bool first) {
          const uint32_t b_lo = desc(b_smem, WB_HALF);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ts_f16(tmem_base + WB_DV, tmem_base + WB_X + kk * 8, umma_desc_join(b_lo + ((kk * 2048) >> 4), HI), IDESC_ACC,
                        (!first) || kk > 0);
        };
        // dK[128 kv, 128 d] += dS^T (shared memory, K-major) * Q (MN-major)
        auto issue_dk = [&](uint32_t b_smem, bool first) {
          const uint32_t a_lo = desc(sDS, 16), b_lo = desc(b_smem, WB_HALF);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ss_f16(tmem_base + WB_DK, umma_desc_join(a_lo + (((kk >> 2) * WB_HALF + (kk & 3) * 32) >> 4), HI),
                        umma_desc_join(b_lo + ((kk * 2048) >> 4), HI), IDESC_ACC, (!first) || kk > 0);
        };
        // dQ^T[128 d, 128 q] = K^T * dS^T (both MN-major: rows are kv)
        auto issue_dq = [&]() {
          const uint32_t kT_lo = desc(sK, WB_HALF), ds_lo = desc(sDS, WB_HALF);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ss_f16(tmem_base + WB_Y, umma_desc_join(kT_lo + ((kk * 2048) >> 4), HI),
                        umma_desc_join(ds_lo + ((kk * 2048) >> 4), HI), IDESC_DQ, kk > 0);
        };
        auto wait = [&](int bar, int n) { return mbar_wait(&bars[bar], n & 1, abort_flag, p.status, WB_CODE(3, bar)); };

        bool ok = true;
        int it = 0, jj0 = 0, cleaned = 0;
        for (int round = 0, w; ok && (w = index_of(round)) < p.nitems; ++round) {
          const Item I = item_of(w);
          if (I.ntot == 0) continue;
          // X is free (the tensor pipe runs in order behind the last dV); Y still holds the previous item's last dQ^T
          // until the drain warps have taken it.
          ok = wait(WBB_KV_FULL, it);
          if (ok && I.valid < min(p.skv, I.kv0 + 128)) ok = wait(WBB_KV_CLEAN, cleaned++);
          ok = ok && wait(WBB_Q_FULL + (jj0 & 1), jj0 >> 1);
          if (ok && jj0 > 0) ok = wait(WBB_DQ_FREE, jj0 - 1);
          if (!ok) break;
          tc_fence_after();
          issue_st(tmem_base + WB_X, sK, q_at(jj0));
          tc_commit(&bars[WBB_S_FULL]);
          issue_st(tmem_base + WB_Y, sV, q_at(jj0) + WB_TILE);
          tc_commit(&bars[WBB_DP_FULL]);
          for (int j = 0; ok && j < I.ntot; ++j) {
            const int jj = jj0 + j;
            const uint32_t sQ = q_at(jj);
            ok = wait(WBB_P_FULL, jj);
            if (!ok) break;
            tc_fence_after();
            issue_dv(sQ + WB_TILE, j == 0);
            if (j + 1 < I.ntot) {
              ok = wait(WBB_Q_FULL + ((jj + 1) & 1), (jj + 1) >> 1);
              if (!ok) break;
              tc_fence_after();
              issue_st(tmem_base + WB_X, sK, q_at(jj + 1));
              tc_commit(&bars[WBB_S_FULL]);
            }
            ok = wait(WBB_PDS_FULL, jj);
            if (!ok) break;
            tc_fence_after();
            issue_dq();                                   // Y: every warp took dP^T out before publishing dS^T
            tc_commit(&bars[WBB_DQ_FULL]);
            issue_dk(sQ, j == 0);
            tc_commit(&bars[WBB_Q_EMPTY + (jj & 1)]);
            tc_commit(&bars[WBB_DS_FREE]);
            if (j + 1 < I.ntot) {
              ok = wait(WBB_DQ_FREE, jj);
              if (!ok) break;
              tc_fence_after();
              issue_st(tmem_base + WB_Y, sV, q_at(jj + 1) + WB_TILE);
              tc_commit(&bars[WBB_DP_FULL]);
            }
          }
          if (ok) tc_commit(&bars[WBB_ACC_DONE]);
          ++it;
          jj0 += I.ntot;
        }
        if (!ok) {
          tc_commit(&bars[WBB_DRAIN]);
          const long long t0 = clock64();
          while (!mbar_try_wait(&bars[WBB_DRAIN], 0) && clock64() - t0 < LVX_SPIN_LIMIT_CYCLES) {}
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == WB_WARP_MMA) tmem_dealloc(tmem_base, 512);
}

// ---------------------------------------------------------------------------------------------
// dq[B, Hq, Sq, 128] = cast of the accumulator in tile order: the grid's second axis walks (slab, chunk), and a warp takes four
// rows of it at a time (16 bytes of fp32 a lane each). Then the sinks' dK and dV: the sum of their parts.
template <bool IS_BF16>
__global__ void __launch_bounds__(256)
window_dq_kernel(const float* __restrict__ acc, uint16_t* __restrict__ dq, int g, int sq, int heads, int chunks, int slabs, const SinkParts sp,
                 const float* __restrict__ parts, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, int skv, const int* status) {
  grid_dep_wait();
  grid_dep_read(acc);
  grid_dep_read(parts);
  if (status && *reinterpret_cast<const volatile int*>(status) != 0) {
    if ((threadIdx.x & 31) == 0) publish_status(status);
    return;
  }
  auto cast = [](float4 v) {
    return IS_BF16 ? make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)) : make_uint2(pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w));
  };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int y = blockIdx.y; y < slabs * chunks; y += gridDim.y) {
    const int chunk = y % chunks, slab = y / chunks, rows = sq * heads;
    const float4* src = reinterpret_cast<const float4*>(acc) + size_t(y) * rows * 32;
    for (int row0 = (blockIdx.x * 8 + warp) * 4; row0 < rows; row0 += gridDim.x * 32) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = src[size_t(min(row0 + u, rows - 1)) * 32 + lane];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int row = row0 + u, tok = row / heads, head = chunk * heads + row % heads;
        if (row < rows && head < g) reinterpret_cast<uint2*>(dq)[((size_t(slab) * g + head) * sq + tok) * 32 + lane] = cast(v[u]);
      }
    }
    const int sink_rows = chunk == 0 ? sp.tiles * 128 * 2 : 0;      // of this slab
    for (int i = blockIdx.x * 8 + warp; i < sink_rows; i += gridDim.x * 8) {
      const int r = i & 127, which = (i >> 7) & 1, tile = i >> 8;
      if (tile * 128 + r >= skv) continue;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = 0; c < sp.parts; ++c) {
        const float4 w = reinterpret_cast<const float4*>(parts)[((((size_t(slab) * sp.tiles + tile) * sp.parts + c) * 2 + which) * 128 + r) * 32 + lane];
        v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
      }
      reinterpret_cast<uint2*>(which ? dv : dk)[(size_t(slab) * skv + tile * 128 + r) * 32 + lane] = cast(v);
    }
  }
}

// The key tiles of the sinks that are shared out over several items, and over how many: as many as make an item about as long
// as those of the other keys.
static SinkParts sink_parts(const lvx_shape& s, const lvx_window& w) {
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  const WindowMask m = make_window_mask(w);
  SinkParts sp = {0, 1};
  if (m.window == kNoWindow || m.sinks == 0 || s.Skv == 0) return sp;
  const long all = (long(s.Sq) + qt.tokens - 1) / qt.tokens, usual = (long(m.window) + 127) / qt.tokens + 1;
  const long tiles = (std::min<long>(m.sinks, s.Skv) + 127) / 128;
  // (and no more than fill the GPU four times over: many sinks are many items as it is, and every part is 128 KB of scratch)
  const long enough = (4 * 148 + s.B * s.Hkv * tiles - 1) / (s.B * s.Hkv * tiles);
  const long parts = std::min((all + usual - 1) / usual, enough);
  if (parts < 2) return sp;
  sp.tiles = int(tiles);
  sp.parts = int(parts);
  return sp;
}

size_t window_sink_floats(const lvx_shape& s, const lvx_window& w) {
  const SinkParts sp = sink_parts(s, w);
  return size_t(s.B) * s.Hkv * sp.tiles * sp.parts * 2 * 128 * 128;
}

size_t window_dq_floats(const lvx_shape& s) {
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  return size_t(s.B) * s.Hkv * qt.chunks * s.Sq * qt.heads * 128;
}

// dq_acc (window_dq_floats, zeroed), then dk and dv; `parts`: window_sink_floats.
int launch_window_bwd(const lvx_shape& s, const lvx_window& w, const lvx_view& q, const lvx_view& d_o, const lvx_view& k,
                      const lvx_view& v, const float* lse, const float* delta, const int32_t* kv_valid_len, float sm_scale,
                      float* dq_acc, float* parts, void* dk, void* dv, int* status, Order order, cudaStream_t st) {
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  CUtensorMap tmQ, tmDO, tmK, tmV;
  int rc = make_q_map(&tmQ, s, qt, q);
  if (!rc) rc = make_q_map(&tmDO, s, qt, d_o);
  if (!rc) rc = make_kv_map(&tmK, s, k, q);
  if (!rc) rc = make_kv_map(&tmV, s, v, q);
  if (rc) return rc;
  WinBwdParams p;
  p.sq = s.Sq;
  p.skv = s.Skv;
  p.hkv = s.Hkv;
  p.g = s.Hq / s.Hkv;
  p.slabs = s.B * s.Hkv;
  p.sp = sink_parts(s, w);
  p.parts = parts;
  p.nitems = ((s.Skv + 127) / 128 + p.sp.tiles * (p.sp.parts - 1)) * p.slabs;
  p.qt = qt;
  p.mask = make_window_mask(w);
  p.kv_valid_len = kv_valid_len;
  p.lse = lse;
  p.delta = delta;
  p.scale = sm_scale;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.dq_acc = dq_acc;
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  p.status = status;
  const int grid = std::min(p.nitems, num_sms());
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kern) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WB_SMEM);
    if (e == cudaSuccess) e = launch_kernel(order, kern, grid, WB_THREADS, WB_SMEM, st, tmQ, tmDO, tmK, tmV, p);
  };
  if (s.dtype == LVX_BF16) go(window_bwd_kernel<true>);
  else go(window_bwd_kernel<false>);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(window bwd)");
  e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "window_bwd_kernel launch");
}

int launch_window_dq(const lvx_shape& s, const lvx_window& w, const float* acc, const float* parts, void* dq, void* dk, void* dv,
                     const int* status, cudaStream_t st) {
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  const long all = long(s.B) * s.Hkv * qt.chunks, rows = long(s.Sq) * qt.heads;
  const dim3 grid(unsigned(std::min<long>((rows + 31) / 32, (148 * 16 + all - 1) / all)), unsigned(std::min<long>(all, 65535)));
  auto go = [&](auto kern) {
    return launch_kernel(ORDER_OVERLAP, kern, grid, 256, 0, st, acc, static_cast<uint16_t*>(dq), s.Hq / s.Hkv, s.Sq, qt.heads, qt.chunks,
                         s.B * s.Hkv, sink_parts(s, w), parts, static_cast<uint16_t*>(dk), static_cast<uint16_t*>(dv), s.Skv, status);
  };
  const cudaError_t e = s.dtype == LVX_BF16 ? go(window_dq_kernel<true>) : go(window_dq_kernel<false>);
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "window_dq launch");
}

}  // namespace lvx
