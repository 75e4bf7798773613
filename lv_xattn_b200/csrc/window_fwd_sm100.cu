// Forward of causal attention with a sliding window and sinks, for more than a few query rows.
//
// Softmax(scale Q K^T) V over the keys that window.cuh describes, with the running maximum and sum of an online softmax.
// A CTA owns two 128-row query tiles of one KV head (neighbours, so that both see nearly the same keys: the heads of a
// group lie side by side in a tile, and with four heads two tiles span 64 tokens) and walks the key tiles that either of
// them sees: those of the sinks, then those of the window. Only a tile that some row sees in part is masked. What lies
// outside costs nothing.
//
// The anatomy is that of the forward block (two softmax warpgroups, thread = row = TMEM lane; a TMA producer; a tcgen05
// issuer that interleaves the two tiles, P overwriting S in TMEM): scores, softmax and product with V of a tile follow one
// another, so that a tile waits for its softmax and the two tiles take turns in the tensor core. What differs:
//   * P is handed over in halves, the first while the second is made, and the reference maximum is settled before the
//     exponentials (three-operand maxima: 64 instructions a row), so that no half has to be taken back. A tile pair then
//     takes 3,390 cycles instead of 3,720 (2,048 of which the tensor core and the exponentials need each): 304 K rows on 4,096
//     keys 540 -> 490 us, 1,300 TFLOP/s. A quarter of the exponentials as polynomials beside the others: no change;
//   * the epilogue and the rescaling work through fewer columns at a time than fit the registers of a loop of their own: what
//     does not spill around the tile loop, and a shorter way through the instruction cache, is worth more (the same rows with
//     a window of 9.4 tiles: 203 us before, 190 with halves, 178 without the spills, 174 with the short epilogue);
//   * CTAs are persistent, and the producer fetches the next item's Q and keys while the last softmax of this one runs;
//   * tiles come through tensor maps of rank 5 and 4, so that q, k and v may have any strides (a cache of more rows
//     than are valid, the projections' [B, S, H, 128]);
//   * key ranges are short, so that a CTA normally sees all of its keys and writes O (rounded once) and lse itself;
//     only where the tiles do not fill the GPU are they split, and the combine kernel merges the parts;
//   * the items with the latest queries, which see the most keys, come first, and CTAs walk the list forwards and backwards
//     in turn;
//   * what lies behind the last valid key may hold anything: scores are replaced, and the rows of V that the last valid
//     tile shares with it are cleared before they are multiplied with a probability of zero. A key inside that a row
//     does not see, but another row of the tile does, may hold an infinity or a NaN too: such a row ends with NaN
//     although its sum is finite, and is made again from the keys that it sees (window_plain_row; nothing else pays for it).
// P is rounded to 16 bits for its product, as in the forward block (O then errs by 2.3e-3 in bf16, 1.7e-3 of which is the
// rounding of O itself); the sum is taken before that.
#include "lvx_internal.h"
#include "sm100_prims.cuh"
#include "window.cuh"
#include <math.h>
#include <algorithm>
#include <limits>

namespace lvx {

constexpr int WF_NS = 2;                         // K/V pipeline stages
constexpr int WF_TILE = 128 * 128 * 2;
constexpr int WF_HALF = WF_TILE / 2;
constexpr int WF_OFF_K = 2 * WF_TILE;            // after the two Q tiles
constexpr int WF_OFF_V = WF_OFF_K + WF_NS * WF_TILE;
constexpr int WF_OFF_OUT = WF_OFF_V + WF_NS * WF_TILE;      // 4 KB per softmax warp: its rows of O on their way out
constexpr int WF_OFF_BAR = WF_OFF_OUT + 8 * 4096;
constexpr int WF_SMEM = WF_OFF_BAR + 256 + 1024;  // + barriers + alignment slack
constexpr int WF_THREADS = 384;
static_assert(WF_SMEM <= 232448, "shared memory budget");
// PAIR from this many key tiles on. us a call, one warpgroup per query tile -> PAIR, 32 tokens of 32 heads on 8 KV heads, over
// 512 / 2,048 / 4,096 / 16,384 keys, combine kernel included where there is one:
//    1 entry      15.0 -> 15.1    16.7 -> 16.7    19.0 -> 17.7     30 ->  25
//    8 entries    15.5 -> 18.0    28.8 -> 29.5    44.8 -> 40.3    128 -> 107
//   32 entries    28.6 -> 39.5      74 ->   78     140 ->  121    482 -> 370
constexpr int kPairTiles = 32;
// CTAs of the few-row kernel, one an SM, that run at once as clusters of n: what cudaOccupancyMaxActiveClusters says on this GPU's
// groups of SMs, one of which has fewer than 16. (As 16 clusters of eight, of which 15 fit, two tokens behind 4,096 keys on 8 KV
// heads took 19.0 us, as clusters of six 12.8, behind 16,384 41.6 and 27.2.)
constexpr int kClusterCtas[kRowCluster + 1] = {0, 148, 148, 135, 132, 130, 132, 105, 120};

enum {
  WFB_Q_FULL = 0,
  WFB_Q_EMPTY,
  WFB_K_FULL,
  WFB_K_EMPTY = WFB_K_FULL + WF_NS,
  WFB_V_FULL = WFB_K_EMPTY + WF_NS,
  WFB_V_EMPTY = WFB_V_FULL + WF_NS,
  WFB_S_FULL = WFB_V_EMPTY + WF_NS,
  WFB_P_FULL = WFB_S_FULL + 2,
  WFB_O_DONE = WFB_P_FULL + 4,
  WFB_DRAIN = WFB_O_DONE + 2,
  WFB_COUNT = WFB_DRAIN + 1
};
#define WF_CODE(role, bar) (LVX_DEV_TIMEOUT_BASE | 0x400 | ((role) << 5) | (bar))

struct WinFwdParams {
  int sq, skv, hkv, g, m_blocks;
  int slabs, splits, nitems;      // an item: a pair of query tiles of a slab, and a share of its keys
  int run_tiles;                  // > 0: items are shared out as runs of key tiles, run_tiles to a pair of query tiles
  QTiles qt;
  WindowMask mask;
  const int32_t* kv_valid_len;
  float scale_log2;
  int nsplit;
  bool beside;          // ORDER_BESIDE
  void* o;              // [B, Hq, Sq, 128] in the input type, with lse; nullptr: partials
  uint16_t* o_low;      // LOW: with low_rows rows a head
  int low_rows;
  float* lse;
  float *o_part, *ml_part;
  const uint16_t *q, *k, *v;      // for window_plain_row
  long long q_b, q_h, q_s, k_b, k_h, k_s, v_b, v_h, v_s;
  int* status;
};

// (ignores NaN, like fmaxf)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// One row's O as plain fp32 sums over its keys in tiles j = first, first + step, ... < n of `kt` from j0 on, written where the
// row belongs: in the input type and divided by l (`out16`), or as it is.
struct PlainRow {
  const uint16_t *q, *k, *v;
  uint16_t *out16, *low16;
  float* out;
  int first, step, n, j0, lo, hi, sink_end;
  float m, l;
};
template <bool IS_BF16>
__device__ __noinline__ void window_plain_row(const WinFwdParams& p, const KeyTiles& kt, const PlainRow& x) {
  for (int d = 0; d < 128; d += 32) {
    float o[32];
    for (int i = 0; i < 32; ++i) o[i] = 0.f;
    for (int j = x.first; j < x.n; j += x.step) {
      const int key0 = kt.tile(x.j0 + j) * 128, cut = min(key0 + 128, x.sink_end);
      for (int key = key0; key < min(key0 + 128, x.hi + 1); ++key)
        if (key < cut || key >= x.lo)
          axpy32<IS_BF16>(o, ex2f(dot128<IS_BF16>(x.q, x.k + key * p.k_s) * p.scale_log2 - x.m), x.v + key * p.v_s + d);
    }
    for (int i = 0; i < 32; i += 2) {
      if (x.out16 != nullptr) {
        const float inv = x.l > 0.f ? 1.f / x.l : 0.f;
        const uint32_t high = pack16x2<IS_BF16>(o[i] * inv, o[i + 1] * inv);
        reinterpret_cast<uint32_t*>(x.out16 + d)[i / 2] = high;
        if (x.low16 != nullptr) reinterpret_cast<uint32_t*>(x.low16 + d)[i / 2] = rest16x2<IS_BF16>(o[i] * inv, o[i + 1] * inv, high);
      } else {
        x.out[d + i] = o[i];
        x.out[d + i + 1] = o[i + 1];
      }
    }
  }
}

// PAIR: the slab has a single query tile (65 to 128 rows: a token each of 32 requests that share a prefix), and the two
// warpgroups take turns at its key tiles instead of one of them idling: each has an accumulator and a partial result of its
// own, and a key tile costs half of the softmax' time, which is then below that of its bytes.
// LOW: what O's rounding drops of early rows is kept (LowRows); a form of its own, since the mere question costs the others 2 %.
template <bool IS_BF16, bool PAIR, bool LOW = false>
__global__ void __launch_bounds__(WF_THREADS, 1)
window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ WinFwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WF_OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + WFB_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  GridDep dep(p.beside);
  const int heads = p.qt.heads, tile_rows = heads * p.qt.tokens;
  struct Item {
    int mb, slab, split, valid, start;      // split: number of the partial result
    KeyTiles kt;
    int j0, n;               // its share of the key tiles
    bool last;               // runs: the last share of its query tiles (partial results that nobody makes are up to it)
  };
  // block of tokens and chunk of heads of a tile (an integer division costs the roles' common start of an item dearly)
  auto block_of = [&](int tile) { return p.qt.chunks == 1 ? tile : tile / p.qt.chunks; };
  auto chunk_of = [&](int tile) { return p.qt.chunks == 1 ? 0 : tile % p.qt.chunks; };
  // Runs: the key tiles of all pairs of query tiles in one row, of which every CTA takes an equal stretch [run0, run1).
  const long long run_all = static_cast<long long>(p.nitems) * p.run_tiles;
  long long run0 = 0, run1 = 0;
  int run_first = 0, run_end = 0;
  if (p.run_tiles > 0) {
    run0 = blockIdx.x * run_all / gridDim.x;
    run1 = (blockIdx.x + 1) * run_all / gridDim.x;
    run_first = int(run0 / p.run_tiles);
    run_end = int((run1 - 1) / p.run_tiles);
  }
  // the CTA's round-th item: forwards and backwards through the list in turn
  auto index_of = [&](int round) {
    if (p.run_tiles > 0) return run_first + round <= run_end ? run_first + round : p.nitems;
    return round * int(gridDim.x) + ((round & 1) ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x));
  };
  auto item_of = [&](int w) {
    Item it;
    const int rest = w / p.slabs;
    it.slab = w - rest * p.slabs;
    it.split = p.splits == 1 ? 0 : rest / p.m_blocks;
    it.mb = p.m_blocks - 1 - (rest - it.split * p.m_blocks);
    it.valid = p.skv;
    if (p.kv_valid_len) it.valid = min(it.valid, max(0, p.kv_valid_len[it.slab / p.hkv]));
    it.start = p.mask.start >= 0 ? p.mask.start : it.valid - p.sq;
    // token range of the two tiles (the second may not exist: its rows do not then, and its tile is loaded as zeros)
    const int tok0 = block_of(2 * it.mb) * p.qt.tokens;
    const int tok1 = min(p.sq, (block_of(min(2 * it.mb + 1, p.qt.count - 1)) + 1) * p.qt.tokens) - 1;
    it.kt = key_tiles(p.mask, it.valid, it.start + tok0, it.start + tok1, 7);
    it.last = false;
    if (p.run_tiles > 0) {
      // the stretch's part of this item, in proportion to the tiles that there turn out to be
      const long long at = static_cast<long long>(w) * p.run_tiles;
      const int a = int(max(run0 - at, 0ll)), b = int(min(run1 - at, static_cast<long long>(p.run_tiles)));
      it.j0 = int(static_cast<long long>(a) * it.kt.n / p.run_tiles);
      it.n = int(static_cast<long long>(b) * it.kt.n / p.run_tiles) - it.j0;
      it.last = b == p.run_tiles;
      // its number: CTAs since the one whose stretch holds the item's first tile (CTA c's begins at floor(c * all / CTAs))
      it.split = a == 0 ? 0 : int(blockIdx.x) - int(((at + 1) * gridDim.x + run_all - 1) / run_all - 1);
      return it;
    }
    const int per_split = p.splits == 1 ? it.kt.n : (it.kt.n + p.splits - 1) / p.splits;
    it.j0 = min(it.kt.n, it.split * per_split);
    it.n = min(it.kt.n, it.j0 + per_split) - it.j0;
    return it;
  };

  // the status word may be set at any moment: one thread reads it, and the CTA leaves or stays as a whole
  int word = 0;
  if (tid == 0) word = *reinterpret_cast<volatile int*>(p.status);

  if (tid == 0) {
    mbar_init(&bars[WFB_Q_FULL], 1);
    mbar_init(&bars[WFB_Q_EMPTY], 1);
    for (int s = 0; s < WF_NS; ++s) {
      mbar_init(&bars[WFB_K_FULL + s], 1);
      mbar_init(&bars[WFB_K_EMPTY + s], 1);
      mbar_init(&bars[WFB_V_FULL + s], 1);
      mbar_init(&bars[WFB_V_EMPTY + s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[WFB_S_FULL + i], 1);
      for (int h = 0; h < 2; ++h) mbar_init(&bars[WFB_P_FULL + 2 * i + h], 4);      // one arrival per softmax warp
      mbar_init(&bars[WFB_O_DONE + i], 1);
    }
    mbar_init(&bars[WFB_DRAIN], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // the rows of a Q tile that no box fills (groups whose size does not divide 128)
  for (int i = tid; i < (128 - tile_rows) * 8 * 4; i += WF_THREADS) {
    const int part = i & 3, at = tile_rows * 8 + (i >> 2);
    reinterpret_cast<uint4*>(smem + part * WF_HALF)[at] = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_async_smem();
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  const bool poisoned = __syncthreads_or(word) != 0;
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Every role walks the same items in the same order and keeps the same counters: `it` = items with key tiles done, `jj0` =
  // key tiles done before the current item (PAIR: t0, those of one warpgroup). All barrier phases follow from them.
  // Registers: 384 threads are launched with 168 each; 256 x 208 + 128 x 88 is the same number of them.
  if (warp < 8) {
    // =========================== softmax warpgroups ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
    const int wg = warp >> 2;
    const int r = (warp & 3) * 32 + lane;            // row of the tile, TMEM lane
    const int r_tok = r / heads, r_head = r - r_tok * heads;
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + wg * 128 + lane_sel;
    const uint32_t tO = tmem_base + 256 + wg * 128 + lane_sel;
    const float c = p.scale_log2;
    using Ref = SoftmaxRef<IS_BF16>;
    // this warpgroup's key tiles: all of an item's, or every other one
    constexpr int STEP = PAIR ? 2 : 1;
    const int first = PAIR ? wg : 0;
    auto hand_over = [&](int half) {      // of P, to the tensor core
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[WFB_P_FULL + 2 * wg + half]);
    };
    bool alive = !poisoned;
    int done_items = 0, t0 = 0;      // items with tiles of this warpgroup, and those tiles
    for (int round = 0, w; alive && (w = index_of(round)) < p.nitems; ++round) {
      const Item I = item_of(w);
      const int tile = PAIR ? 0 : 2 * I.mb + wg;
      const int tok = block_of(tile) * p.qt.tokens + r_tok, head = chunk_of(tile) * heads + r_head;
      const bool exists = tile < p.qt.count && r < tile_rows && tok < p.sq && head < p.g;
      // this row's keys: [0, sink_end) and [lo, hi]. A row that does not exist sees everything against a reference of 0 (its
      // scores are zeros), so that it never holds up its warp.
      const int hi = exists ? min(I.start + tok, I.valid - 1) : I.valid - 1;
      const int lo = exists ? max(0, I.start + tok - p.mask.window + 1) : 0;
      const int sink_end = min(p.mask.sinks, hi + 1);
      // keys that every row of the warp sees: [0, all_sinks) and [all_lo, all_hi]
      const int all_hi = __reduce_min_sync(0xffffffffu, hi), all_lo = __reduce_max_sync(0xffffffffu, lo);
      const int all_sinks = min(p.mask.sinks, all_hi + 1);
      float m = exists ? -INFINITY : 0.f, high = m, l = 0.f;
      int t = 0;                       // tiles of this warpgroup in the item
      for (int j = first; j < I.n; j += STEP, ++t) {
        const int key0 = I.kt.tile(I.j0 + j) * 128;
        const bool full = key0 + 127 <= all_hi && (key0 >= all_lo || key0 + 128 <= all_sinks);
        if (!mbar_wait(&bars[WFB_S_FULL + wg], (t0 + t) & 1, abort_flag, p.status, WF_CODE(wg, WFB_S_FULL))) {
          alive = false;
          break;
        }
        tc_fence_after();
        // The usual tile: exponentials against the running maximum as it stands (it is only a reference point). The first half
        // of P is handed to the tensor core while the second is made.
        bool done = false;
        if (t > 0 && full) {
          uint32_t sv[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, sv[q]);
          tc_wait_ld();
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx[i & 3] = max3(mx[i & 3], __uint_as_float(sv[q][2 * i]), __uint_as_float(sv[q][2 * i + 1]));
          const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * c;
          if (!__any_sync(0xffffffffu, Ref::off(top, m))) {
            const float moff = m == -INFINITY ? 0.f : m;
            uint64_t sum_a = f32x2(0.f, 0.f), sum_b = f32x2(0.f, 0.f);
            const uint64_t c2 = f32x2(c, c), nm2 = f32x2(-moff, -moff);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[32];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t* b = &sv[2 * h + i / 8][4 * (i % 8)];
                float x0, x1, x2, x3;
                f32x2_get(fma2(f32x2(__uint_as_float(b[0]), __uint_as_float(b[1])), c2, nm2), x0, x1);
                f32x2_get(fma2(f32x2(__uint_as_float(b[2]), __uint_as_float(b[3])), c2, nm2), x2, x3);
                const float e0 = ex2f(x0), e1 = ex2f(x1), e2 = ex2f(x2), e3 = ex2f(x3);
                sum_a = add2(sum_a, f32x2(e0, e1));
                sum_b = add2(sum_b, f32x2(e2, e3));
                pk[2 * i] = IS_BF16 ? pack_bf16x2(e0, e1) : pack_f16x2(e0, e1);
                pk[2 * i + 1] = IS_BF16 ? pack_bf16x2(e2, e3) : pack_f16x2(e2, e3);
              }
              tmem_st32(tS + h * 32, pk);
              hand_over(h);
            }
            float s0, s1, s2, s3;
            f32x2_get(sum_a, s0, s1);
            f32x2_get(sum_b, s2, s3);
            l += (s0 + s1) + (s2 + s3);
            done = true;
          }
        }
        if (!done) {
          // The first tile, tiles that are seen in part, and scores that jumped: with the row maximum. A warp's rows are few
          // tokens, so of a partly seen tile's four groups of 32 keys all but one or two are seen by all of its rows or by none;
          // those that none sees are zeros without an exponential, and only the mixed ones are masked.
          uint32_t s[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, s[q]);
          uint32_t none = 0;      // bit q: group q is seen by no row of the warp
          if (!full) {
            uint32_t seen[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              seen[q] = visible_bits(key0 + q * 32, lo, hi, sink_end);
              if (!__any_sync(0xffffffffu, seen[q] != 0u)) none |= 1u << q;
            }
            tc_wait_ld();
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (!(none >> q & 1) && !__all_sync(0xffffffffu, seen[q] == 0xffffffffu)) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!(seen[q] & (1u << i))) s[q][i] = 0xff800000u;  // -inf
              }
          } else {
            tc_wait_ld();
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (!(none >> q & 1)) {
#pragma unroll
              for (int i = 0; i < 16; ++i) mx[i & 3] = max3(mx[i & 3], __uint_as_float(s[q][2 * i]), __uint_as_float(s[q][2 * i + 1]));
            }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
          const bool move = Ref::moves(top, m, high);
          float alpha = 1.f;
          if (move) {
            alpha = ex2f(m - (top - Ref::under));
            m = top - Ref::under;
            high = fmaxf(high, m);
            l *= alpha;
          }
          if (t > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {      // (32 columns at a time do not fit beside the scores)
              uint32_t o[16];
              tmem_ld16(tO + q * 16, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(tO + q * 16, o);
            }
          }
          const float moff = (m == -INFINITY) ? 0.f : m;
          const uint64_t c2 = f32x2(c, c), nm2 = f32x2(-moff, -moff);
          uint64_t sum = f32x2(0.f, 0.f);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t pk[16];
            if (none >> q & 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = 0u;
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float x0, x1;
                f32x2_get(fma2(f32x2(__uint_as_float(s[q][2 * i]), __uint_as_float(s[q][2 * i + 1])), c2, nm2), x0, x1);
                const float e0 = ex2f(x0), e1 = ex2f(x1);
                sum = add2(sum, f32x2(e0, e1));
                pk[i] = IS_BF16 ? pack_bf16x2(e0, e1) : pack_f16x2(e0, e1);
              }
            }
            tmem_st16(tS + q * 16, pk);
            if (q == 1) hand_over(0);
          }
          float sum0, sum1;
          f32x2_get(sum, sum0, sum1);
          l += sum0 + sum1;
          hand_over(1);
        }
      }
      // ------------------------------- epilogue -------------------------------
      if (alive && t > 0) alive = mbar_wait(&bars[WFB_O_DONE + wg], done_items & 1, abort_flag, p.status, WF_CODE(wg, WFB_O_DONE));
      alive = __all_sync(0xffffffffu, alive);
      tc_fence_after();
      if (alive) {
        // The warp's rows go through shared memory, 128 bytes of each at a time (16-byte pieces, rotated by row against bank
        // conflicts), so that a store covers whole sectors: written by row they are 32 pieces of 16 bytes, 256 bytes apart.
        const int row = head * p.sq + tok;         // of the slab
        const unsigned here = __ballot_sync(0xffffffffu, exists);
        uint8_t* out = smem + WF_OFF_OUT + warp * 4096;
        const bool direct = p.o != nullptr;
        const size_t slab_rows = size_t(p.g) * p.sq;
        uint8_t* base;
        int row_bytes;
        if (direct) {
          base = static_cast<uint8_t*>(p.o) + size_t(I.slab) * slab_rows * 256;
          row_bytes = 256;
        } else {
          base = reinterpret_cast<uint8_t*>(p.o_part) + (size_t(I.slab) * p.nsplit + (PAIR ? 2 * I.split + wg : I.split)) * slab_rows * 512;
          row_bytes = 512;
        }
        auto store = [&](int at) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = i * 4 + (lane >> 3), piece = lane & 7;
            const int to = __shfl_sync(0xffffffffu, row, rr);
            if (here >> rr & 1)
              *reinterpret_cast<uint4*>(base + size_t(to) * row_bytes + at + piece * 16) =
                  *reinterpret_cast<const uint4*>(out + rr * 128 + ((piece ^ (rr & 7)) << 4));
          }
          __syncwarp();
        };
        auto load = [&](int col, uint32_t (&o)[32]) {
          if (t > 0) {
            tmem_ld32(tO + col, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
        };
        uint64_t sum2 = 0ull;
        auto bad = [&](const uint32_t (&o)[32]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sum2 = add2(sum2, f32x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])));
        };
        auto low_row = [&] {
          const int at = LOW && exists ? LowRows::place(I.start + tok, I.start, p.low_rows) : -1;
          return at >= 0 ? p.o_low + ((size_t(I.slab) * p.g + head) * p.low_rows + at) * 128 : nullptr;
        };
        if (direct) {
          const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;      // (NaN stays)
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            uint32_t o[2][32];
            load(h * 64, o[0]);
            load(h * 64 + 32, o[1]);
            tc_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t w4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float x = __uint_as_float(o[q][8 * i + 2 * e]) * inv, y = __uint_as_float(o[q][8 * i + 2 * e + 1]) * inv;
                  w4[e] = pack16x2<IS_BF16>(x, y);
                }
                *reinterpret_cast<uint4*>(out + lane * 128 + (((q * 4 + i) ^ (lane & 7)) << 4)) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
              }
              bad(o[q]);
            }
            store(h * 128);
            if constexpr (LOW) {
              if (uint16_t* low = low_row()) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    uint32_t w4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      const float x = __uint_as_float(o[q][8 * i + 2 * e]) * inv, y = __uint_as_float(o[q][8 * i + 2 * e + 1]) * inv;
                      w4[e] = rest16x2<IS_BF16>(x, y, pack16x2<IS_BF16>(x, y));
                    }
                    reinterpret_cast<uint4*>(low + h * 64)[q * 4 + i] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
                  }
              }
            }
          }
          if (exists) p.lse[size_t(I.slab) * slab_rows + row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        } else {
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            uint32_t o[32];
            load(q * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(out + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            bad(o);
            store(q * 128);
          }
          if (exists) {
            float2* ml = reinterpret_cast<float2*>(p.ml_part) + size_t(I.slab) * p.nsplit * slab_rows + row;
            ml[(PAIR ? 2 * I.split + wg : I.split) * slab_rows] = make_float2(m, l);
            if (I.last)      // the partial results that no CTA makes
              for (int k = PAIR ? 2 * I.split + 2 + wg : I.split + 1; k < p.nsplit; k += STEP) ml[k * slab_rows] = make_float2(-INFINITY, 0.f);
          }
        }
        tc_fence_before();
        float sum_a, sum_b;
        f32x2_get(sum2, sum_a, sum_b);
        if (exists && isnan(sum_a + sum_b) && l < INFINITY) {
          const int batch = I.slab / p.hkv, kvh = I.slab % p.hkv;
          PlainRow x;
          x.q = p.q + batch * p.q_b + (kvh * p.g + head) * p.q_h + tok * p.q_s;
          x.k = p.k + batch * p.k_b + kvh * p.k_h;
          x.v = p.v + batch * p.v_b + kvh * p.v_h;
          x.low16 = low_row();
          x.out16 = direct ? reinterpret_cast<uint16_t*>(base + size_t(row) * 256) : nullptr;
          x.out = reinterpret_cast<float*>(base + size_t(row) * 512);
          x.first = first;
          x.step = STEP;
          x.n = I.n;
          x.j0 = I.j0;
          x.lo = lo;
          x.hi = hi;
          x.sink_end = sink_end;
          x.m = m == -INFINITY ? 0.f : m;
          x.l = l;
          const KeyTiles kt = I.kt;
          window_plain_row<IS_BF16>(p, kt, x);
        }
        __syncwarp();
      }
      done_items += t > 0;
      t0 += t;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
    if (warp == 8 && lane == 0 && !poisoned) {
      // =========================== TMA producer ===========================
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      int it = 0, jj0 = 0, k_issued = 0, v_issued = 0;
      bool alive = true;
      for (int round = 0, w; alive && (w = index_of(round)) < p.nitems; ++round) {
        const Item I = item_of(w);
        if (I.n == 0) continue;
        const int batch = I.slab / p.hkv, kvh = I.slab % p.hkv;
        // the previous item's last scores have been made: its Q is done with, while its last softmax still runs
        if (it > 0 && !mbar_wait(&bars[WFB_Q_EMPTY], (it - 1) & 1, abort_flag, p.status, WF_CODE(2, WFB_Q_EMPTY))) break;
        mbar_arrive_expect_tx(&bars[WFB_Q_FULL], (PAIR ? 1 : 2) * tile_rows * 256);
        for (int t = 0; t < (PAIR ? 1 : 2); ++t) {
          const int tile = 2 * I.mb + t;
          for (int h = 0; h < 2; ++h)
            tma_load_5d(smem + t * WF_TILE + h * WF_HALF, &tmQ, &bars[WFB_Q_FULL], h * 64, chunk_of(tile) * heads,
                        block_of(tile) * p.qt.tokens, kvh, batch);
        }
        ++it;
        for (int j = 0; j < I.n; ++j) {
          const int jj = jj0 + j, s = jj % WF_NS;
          const uint32_t ph = (jj / WF_NS) & 1;
          const int y = I.kt.tile(I.j0 + j) * 128;
          alive = mbar_wait(&bars[WFB_K_EMPTY + s], ph ^ 1, abort_flag, p.status, WF_CODE(2, WFB_K_EMPTY));
          if (!alive) break;
          mbar_arrive_expect_tx(&bars[WFB_K_FULL + s], WF_TILE);
          tma_load_4d(smem + WF_OFF_K + s * WF_TILE, &tmK, &bars[WFB_K_FULL + s], 0, y, kvh, batch);
          tma_load_4d(smem + WF_OFF_K + s * WF_TILE + WF_HALF, &tmK, &bars[WFB_K_FULL + s], 64, y, kvh, batch);
          k_issued = jj + 1;
          alive = mbar_wait(&bars[WFB_V_EMPTY + s], ph ^ 1, abort_flag, p.status, WF_CODE(2, WFB_V_EMPTY));
          if (!alive) break;
          mbar_arrive_expect_tx(&bars[WFB_V_FULL + s], WF_TILE);
          tma_load_4d(smem + WF_OFF_V + s * WF_TILE, &tmV, &bars[WFB_V_FULL + s], 0, y, kvh, batch);
          tma_load_4d(smem + WF_OFF_V + s * WF_TILE + WF_HALF, &tmV, &bars[WFB_V_FULL + s], 64, y, kvh, batch);
          v_issued = jj + 1;
        }
        jj0 += I.n;
      }
      if (*abort_flag) {      // a CTA that is giving up must not leave while a copy into its shared memory is in flight
        auto drain = [&](uint64_t* bar, uint32_t ph) {
          const long long t0 = clock64();
          while (!mbar_try_wait(bar, ph) && clock64() - t0 < LVX_SPIN_LIMIT_CYCLES) {}
        };
        if (it > 0) drain(&bars[WFB_Q_FULL], (it - 1) & 1);
        for (int j = max(0, k_issued - WF_NS); j < k_issued; ++j) drain(&bars[WFB_K_FULL + j % WF_NS], (j / WF_NS) & 1);
        for (int j = max(0, v_issued - WF_NS); j < v_issued; ++j) drain(&bars[WFB_V_FULL + j % WF_NS], (j / WF_NS) & 1);
      }
    }
    if (warp == 9 && !poisoned) {
      // =========================== MMA issuer (the whole warp walks, one elected lane issues) ===========================
      constexpr uint32_t FMT = IS_BF16 ? UMMA_BF16 : UMMA_F16;
      constexpr uint32_t IDESC_QK = umma_idesc(FMT, UMMA_K_MAJOR, UMMA_K_MAJOR, 128, 128);
      constexpr uint32_t IDESC_PV = umma_idesc(FMT, UMMA_K_MAJOR, UMMA_MN_MAJOR, 128, 128);
      constexpr uint32_t HI = umma_desc_hi(1024);
      const uint32_t sQ = smem_u32(smem), sK = smem_u32(smem + WF_OFF_K), sV = smem_u32(smem + WF_OFF_V);
      auto issue_qk = [&](int i, int stage) {
        const uint32_t a_lo = umma_desc_lo(sQ + (PAIR ? 0 : i * WF_TILE), 16);
        const uint32_t b_lo = umma_desc_lo(sK + stage * WF_TILE, 16);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = ((kk >> 2) * WF_HALF + (kk & 3) * 32) >> 4;
            umma_ss_f16(tmem_base + i * 128, umma_desc_join(a_lo + off, HI), umma_desc_join(b_lo + off, HI), IDESC_QK, kk > 0);
          }
        }
        __syncwarp();
      };
      auto issue_pv = [&](int i, int stage, int h, bool first) {
        const uint32_t b_lo = umma_desc_lo(sV + stage * WF_TILE, WF_HALF);
        if (elect_one()) {
#pragma unroll
          for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
            umma_ts_f16(tmem_base + 256 + i * 128, tmem_base + i * 128 + kk * 8, umma_desc_join(b_lo + ((kk * 2048) >> 4), HI),
                        IDESC_PV, (!first) || kk > 0);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc_commit(bar);
        __syncwarp();
      };
      auto wait = [&](int bar, uint32_t ph) {
        return __all_sync(0xffffffffu, mbar_wait(&bars[bar], ph, abort_flag, p.status, WF_CODE(3, bar)));
      };
      bool ok = true;
      int it = 0, jj0 = 0, t0[2] = {0, 0};      // t0: tiles of each warpgroup done
      for (int round = 0, w; ok && (w = index_of(round)) < p.nitems; ++round) {
        const Item I = item_of(w);
        const int n = I.n;
        if (n == 0) continue;
        auto k_full = [&](int j) { return wait(WFB_K_FULL + (jj0 + j) % WF_NS, (jj0 + j) / WF_NS & 1); };
        auto v_full = [&](int j) { return wait(WFB_V_FULL + (jj0 + j) % WF_NS, (jj0 + j) / WF_NS & 1); };
        auto stage = [&](int j) { return (jj0 + j) % WF_NS; };
        // rows of V behind the last valid key: whatever they hold is multiplied with zeros
        auto clear_v = [&](int j) {
          const int left = I.valid - I.kt.tile(I.j0 + j) * 128;
          if (left >= 128) return;
          for (int at = lane; at < (128 - left) * 16; at += 32)
            *reinterpret_cast<uint4*>(smem + WF_OFF_V + stage(j) * WF_TILE + ((at >> 3) & 1) * WF_HALF + (left + (at >> 4)) * 128 +
                                      (at & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_async_smem();
          __syncwarp();
        };
        // the item's first scores: S is free (the tensor pipe runs in order behind the last product with P)
        ok = wait(WFB_Q_FULL, it & 1) && k_full(0);
        if constexpr (PAIR) {
          // tile j is warpgroup j % 2's; its scores come two tiles ahead
          for (int j = 0; ok && j < min(n, 2); ++j) {
            if (j > 0) ok = k_full(j);
            if (!ok) break;
            tc_fence_after();
            issue_qk(j, stage(j));
            commit(&bars[WFB_S_FULL + j]);
            commit(&bars[WFB_K_EMPTY + stage(j)]);
            if (j == n - 1) commit(&bars[WFB_Q_EMPTY]);
          }
          for (int j = 0; ok && j < n; ++j) {
            const int i = j & 1;
            ok = v_full(j);
            if (ok) clear_v(j);
            for (int h = 0; h < 2; ++h) {
              ok = ok && wait(WFB_P_FULL + 2 * i + h, (t0[i] + (j >> 1)) & 1);
              if (!ok) break;
              tc_fence_after();
              issue_pv(i, stage(j), h, j < 2);
            }
            if (!ok) break;
            commit(&bars[WFB_V_EMPTY + stage(j)]);
            if (j + 2 < n) {
              ok = k_full(j + 2);
              if (!ok) break;
              tc_fence_after();
              issue_qk(i, stage(j + 2));
              commit(&bars[WFB_S_FULL + i]);
              commit(&bars[WFB_K_EMPTY + stage(j + 2)]);
              if (j + 2 == n - 1) commit(&bars[WFB_Q_EMPTY]);
            } else {
              commit(&bars[WFB_O_DONE + i]);
            }
          }
          t0[0] += (n + 1) / 2;
          t0[1] += n / 2;
        } else {
          if (ok) {
            tc_fence_after();
            issue_qk(0, stage(0));
            commit(&bars[WFB_S_FULL + 0]);
            issue_qk(1, stage(0));
            commit(&bars[WFB_S_FULL + 1]);
            commit(&bars[WFB_K_EMPTY + stage(0)]);
            if (n == 1) commit(&bars[WFB_Q_EMPTY]);
          }
          for (int j = 0; ok && j < n; ++j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (!ok) break;
              if (i == 0) {
                ok = v_full(j);
                if (ok) clear_v(j);
              }
              for (int h = 0; h < 2; ++h) {
                ok = ok && wait(WFB_P_FULL + 2 * i + h, (jj0 + j) & 1);
                if (!ok) break;
                tc_fence_after();
                issue_pv(i, stage(j), h, j == 0);
              }
              if (!ok) break;
              if (i == 1) commit(&bars[WFB_V_EMPTY + stage(j)]);
              if (j + 1 < n) {
                if (i == 0) ok = k_full(j + 1);
                if (!ok) break;
                tc_fence_after();
                issue_qk(i, stage(j + 1));
                commit(&bars[WFB_S_FULL + i]);
                if (i == 1) {
                  commit(&bars[WFB_K_EMPTY + stage(j + 1)]);
                  if (j + 1 == n - 1) commit(&bars[WFB_Q_EMPTY]);
                }
              } else {
                commit(&bars[WFB_O_DONE + i]);
              }
            }
          }
        }
        ++it;
        jj0 += n;
      }
      if (!ok) {      // wind down: let every MMA already issued finish before TMEM is released
        commit(&bars[WFB_DRAIN]);
        const long long t0 = clock64();
        while (!mbar_try_wait(&bars[WFB_DRAIN], 0) && clock64() - t0 < LVX_SPIN_LIMIT_CYCLES) {}
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem_base, 512);
  // this may be the last kernel of its call: the host is told of results that were not made
  if (tid == 0 && (poisoned || *abort_flag)) publish_status(p.status);
}

// ---------------------------------------------------------------------------------------------
static bool window_pair(const lvx_shape& s, long tiles, bool few) {
  return !few && tiles >= kPairTiles && make_q_tiles(s.Hq / s.Hkv, s.Sq).count == 1;
}
// key tiles that a CTA of this call sees at most: its tokens' windows, and the sinks
static long window_tiles(const lvx_shape& s, const lvx_window& w, bool few) {
  const int span = few ? s.Sq : 2 * make_q_tiles(s.Hq / s.Hkv, s.Sq).tokens;
  const WindowMask m = make_window_mask(w);
  const long all = (long(s.Skv) + 127) / 128;
  if (m.window == kNoWindow) return all;
  return std::min<long>(all, (long(m.window) + span + 126) / 128 + 1 + (long(m.sinks) + 127) / 128);
}

// Whether all pairs of query tiles see about the same number of key tiles: a prefix, a few tokens behind a long cache.
static bool window_even(const lvx_shape& s, const lvx_window& w, long tiles) {
  return w.query_start >= s.Skv || 8l * s.Sq <= tiles * 128;
}

// `merged`: the parts are merged with others in any case.
FwdPlan plan_window(const lvx_shape& s, const lvx_window& w, bool* few, bool merged) {
  *few = false;
  if (s.dtype == LVX_FP32) return plan_fwd(s);
  const int g = s.Hq / s.Hkv;
  FwdPlan p;
  p.rows = g * s.Sq;
  p.kv_tiles = (s.Skv + 127) / 128;
  *few = p.rows <= kFewRows;
  p.m_blocks = *few ? 1 : (make_q_tiles(g, s.Sq).count + 1) / 2;
  long tiles = window_tiles(s, w, *few);
  const long base = long(p.m_blocks) * s.B * s.Hkv;
  const bool pair = window_pair(s, tiles, *few);
  if (pair) tiles = (tiles + 1) / 2;      // what a CTA walks takes half as long
  const long most = std::min<long>(tiles > 0 ? tiles : 1, *few ? 148 : 64);
  // Splits that fill whole rounds of 148 SMs, eight rounds at most (the fixed cost then outweighs what a partly filled last round
  // wastes): 3 tiles' worth of fixed cost per item, and 4 for a second kernel where one would do without. Few rows do without it
  // as a cluster, which lies within one of the eight groups of SMs, of which fewer than all are then in use (kClusterCtas: 32 tokens
  // behind 8,192 keys as 256 clusters of four take 172 us instead of 152 as 256 CTAs).
  long best_cost = std::numeric_limits<long>::max();
  p.nsplit = 1;
  for (long ns = 1; ns <= most && (ns == 1 || base * ns <= 148 * 8); ++ns) {
    const bool cluster = *few && !merged && ns > 1 && ns <= kRowCluster;
    const long at_once = cluster ? kClusterCtas[ns] : 148;
    const long rounds = (base * ns + at_once - 1) / at_once, per = (tiles + ns - 1) / ns;
    const long cost = rounds * (per + 3) + (ns == 1 || cluster || (*few && merged) ? 0 : 4);
    if (cost < best_cost) {
      best_cost = cost;
      p.nsplit = int(ns);
    }
  }
  p.tiles_per_split = 0;          // the kernels share out what each CTA turns out to see
  // Runs, where the pairs of query tiles see about the same number of keys: equal stretches for 148 CTAs instead of whole
  // rounds of equal shares, which leave the last round partly filled, pay the fixed cost for every share and write as many
  // partial results. (168 pairs of 201 tiles: 547 -> 535 us, and their merge 48 -> 30; 80 pairs: 285 -> 270 and 23 -> 16; 8
  // pairs, which are 18 or 19 shares each way: even.) A pair is met by 148 / pairs CTAs, and one more where it does not divide.
  if (!*few && tiles > 0 && window_even(s, w, tiles) && base * tiles >= 148) {
    const long cost = (base * tiles + 147) / 148 + 3 * (base / 148 + 2) + 4;
    if (cost < best_cost) {
      p.tiles_per_split = int(tiles);
      p.nsplit = int((148 + base - 1) / base + (148 % base != 0 || 148 < base));
    }
  }
  if (pair) p.nsplit *= 2;        // partial results; there are half as many items
  p.o_part_bytes = (size_t(s.B) * s.Hkv * p.nsplit * p.rows * 512 + 255) & ~size_t(255);
  p.ml_part_bytes = (size_t(s.B) * s.Hkv * p.nsplit * p.rows * 8 + 255) & ~size_t(255);
  return p;
}

int make_q_map(CUtensorMap* out, const lvx_shape& s, const QTiles& qt, const lvx_view& v) {
  const uint64_t es = elt_size(s.dtype), g = s.Hq / s.Hkv;
  // the stride of a dimension of one is never used, but has to be a valid one
  auto stride = [&](int64_t st, uint64_t n) { return n > 1 ? uint64_t(st) * es : uint64_t(256); };
  const uint64_t dims[5] = {128, g, uint64_t(s.Sq), uint64_t(s.Hkv), uint64_t(s.B)};
  const uint64_t strides[4] = {stride(v.stride_h, g), stride(v.stride_s, s.Sq), stride(v.stride_h * int64_t(g), s.Hkv), stride(v.stride_b, s.B)};
  const uint32_t box[5] = {64, uint32_t(qt.heads), uint32_t(qt.tokens), 1, 1};
  return make_tmap_nd(out, s.dtype, v.data, 5, dims, strides, box);
}

int make_kv_map(CUtensorMap* out, const lvx_shape& s, const lvx_view& v, const lvx_view& dummy) {
  const uint64_t es = elt_size(s.dtype);
  auto stride = [&](int64_t st, uint64_t n) { return n > 1 ? uint64_t(st) * es : uint64_t(256); };
  // no keys: the map describes one row of q and nothing is loaded through it
  const uint64_t rows = s.Skv > 0 ? s.Skv : 1;
  const uint64_t dims[4] = {128, rows, s.Skv > 0 ? uint64_t(s.Hkv) : 1, s.Skv > 0 ? uint64_t(s.B) : 1};
  const uint64_t strides[3] = {stride(v.stride_s, dims[1]), stride(v.stride_h, dims[2]), stride(v.stride_b, dims[3])};
  const uint32_t box[4] = {64, 128, 1, 1};
  return make_tmap_nd(out, s.dtype, s.Skv > 0 ? v.data : dummy.data, 4, dims, strides, box);
}

int launch_window_fwd(const lvx_shape& s, const lvx_window& w, const FwdPlan& pl, const lvx_view& q, const lvx_view& k,
                      const lvx_view& v, const int32_t* kv_valid_len, float sm_scale, float* o_part, float* ml_part, void* o,
                      void* o_low, float* lse, int* status, Order order, cudaStream_t st) {
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  CUtensorMap tmQ, tmK, tmV;
  int rc = make_q_map(&tmQ, s, qt, q);
  if (!rc) rc = make_kv_map(&tmK, s, k, q);
  if (!rc) rc = make_kv_map(&tmV, s, v, q);
  if (rc) return rc;
  WinFwdParams p;
  p.sq = s.Sq;
  p.skv = s.Skv;
  p.hkv = s.Hkv;
  p.g = s.Hq / s.Hkv;
  p.m_blocks = pl.m_blocks;
  p.qt = qt;
  p.mask = make_window_mask(w);
  p.kv_valid_len = kv_valid_len;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.nsplit = pl.nsplit;
  p.beside = order == ORDER_BESIDE;
  p.o = o;
  p.o_low = static_cast<uint16_t*>(o_low);
  p.low_rows = low_rows_of(w);
  p.lse = lse;
  p.o_part = o_part;
  p.ml_part = ml_part;
  p.q = static_cast<const uint16_t*>(q.data);
  p.k = static_cast<const uint16_t*>(k.data);
  p.v = static_cast<const uint16_t*>(v.data);
  p.q_b = q.stride_b; p.q_h = q.stride_h; p.q_s = q.stride_s;
  p.k_b = k.stride_b; p.k_h = k.stride_h; p.k_s = k.stride_s;
  p.v_b = v.stride_b; p.v_h = v.stride_h; p.v_s = v.stride_s;
  p.status = status;
  const bool pair = window_pair(s, window_tiles(s, w, false), false);
  p.slabs = s.B * s.Hkv;
  p.run_tiles = pl.tiles_per_split;
  p.splits = p.run_tiles > 0 ? 1 : pair ? pl.nsplit / 2 : pl.nsplit;
  const long items = long(p.slabs) * pl.m_blocks * p.splits;
  if (items >= (1l << 30)) return fail(LVX_ERR_LIMIT, "window_fwd: %ld work items", items);
  p.nitems = int(items);
  // persistent: one CTA per SM; runs are planned for 148
  const unsigned grid = p.run_tiles > 0 ? 148 : unsigned(std::min<long>(items, num_sms()));
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kern) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WF_SMEM);
    if (e == cudaSuccess) e = launch_kernel(order, kern, grid, WF_THREADS, WF_SMEM, st, tmQ, tmK, tmV, p);
  };
  auto pick = [&](auto one, auto two, auto low) {
    if (pair) go(two);
    else if (o != nullptr && o_low != nullptr) go(low);
    else go(one);
  };
  if (s.dtype == LVX_BF16) pick(window_fwd_kernel<true, false>, window_fwd_kernel<true, true>, window_fwd_kernel<true, false, true>);
  else pick(window_fwd_kernel<false, false>, window_fwd_kernel<false, true>, window_fwd_kernel<false, false, true>);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(window fwd)");
  e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "window_fwd_kernel launch");
}

}  // namespace lvx
