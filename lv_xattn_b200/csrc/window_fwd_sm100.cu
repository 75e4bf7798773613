// Forward of causal attention with a sliding window and sinks, for more than a few query rows.
//
// Softmax(scale Q K^T) V over the keys that window.cuh describes, with the running maximum and sum of an online softmax.
// A CTA owns two 128-row query tiles of one KV head (neighbours, so that both see nearly the same keys: the heads of a
// group lie side by side in a tile, and with four heads two tiles span 64 tokens) and walks the key tiles that either of
// them sees: those of the sinks, then those of the window. Only a tile that some row sees in part is masked; the others
// take the path without a mask and without a row maximum. What lies outside costs nothing.
//
// The anatomy is that of the forward block (320 threads: two softmax warpgroups, thread = row = TMEM lane; a TMA
// producer; a tcgen05 issuer that interleaves the two tiles, P overwriting S in TMEM), with its measured reasons: the
// softmax is what a tile waits for, so that the two tiles take turns in the tensor core. What differs:
//   * tiles come through tensor maps of rank 5 and 4, so that q, k and v may have any strides (a cache of more rows
//     than are valid, the projections' [B, S, H, 128]);
//   * key ranges are short, so that a CTA normally sees all of its keys and writes O (rounded once) and lse itself;
//     only where the tiles do not fill the GPU are they split, and the combine kernel merges the parts;
//   * CTAs with the latest queries, which see the most keys, are started first;
//   * what lies behind the last valid key may hold anything: scores are replaced, and the rows of V that the last valid
//     tile shares with it are cleared before they are multiplied with a probability of zero. A key inside that a row
//     does not see, but another row of the tile does, may hold an infinity or a NaN too: such a row ends with NaN
//     although its sum is finite, and is made again from the keys that it sees (plain_values; nothing else pays for it).
// P is rounded to 16 bits for its product, as in the forward block (O then errs by 2.3e-3 in bf16, 1.7e-3 of which is the
// rounding of O itself); the sum is taken before that.
#include "lvx_internal.h"
#include "sm100_prims.cuh"
#include "window.cuh"
#include <math.h>
#include <algorithm>

namespace lvx {

constexpr int WF_NS = 2;                         // K/V pipeline stages
constexpr int WF_TILE = 128 * 128 * 2;
constexpr int WF_HALF = WF_TILE / 2;
constexpr int WF_OFF_K = 2 * WF_TILE;            // after the two Q tiles
constexpr int WF_OFF_V = WF_OFF_K + WF_NS * WF_TILE;
constexpr int WF_OFF_BAR = WF_OFF_V + WF_NS * WF_TILE;
constexpr int WF_SMEM = WF_OFF_BAR + 256 + 1024;  // + barriers + alignment slack
constexpr int WF_THREADS = 320;
// PAIR from this many key tiles on. us a call, one warpgroup per query tile -> PAIR, 32 tokens of 32 heads on 8 KV heads, over
// 512 / 2,048 / 4,096 / 16,384 keys, combine kernel included where there is one:
//    1 entry      15.7 ->  17.5    16.7 -> 18.9    19.2 ->  19.7     31 ->  27
//    8 entries    15.9 ->  20.4    30.7 -> 32.3    47.4 ->  42.0    139 -> 103
//   32 entries    40.5 ->  58.5     101 ->   98     161 ->   142    547 -> 402
constexpr int kPairTiles = 32;

enum {
  WFB_Q_FULL = 0,
  WFB_K_FULL = 1,
  WFB_K_EMPTY = WFB_K_FULL + WF_NS,
  WFB_V_FULL = WFB_K_EMPTY + WF_NS,
  WFB_V_EMPTY = WFB_V_FULL + WF_NS,
  WFB_S_FULL = WFB_V_EMPTY + WF_NS,
  WFB_P_FULL = WFB_S_FULL + 2,
  WFB_O_DONE = WFB_P_FULL + 2,
  WFB_DRAIN = WFB_O_DONE + 2,
  WFB_COUNT = WFB_DRAIN + 1
};
#define WF_CODE(role, bar) (LVX_DEV_TIMEOUT_BASE | 0x400 | ((role) << 5) | (bar))

struct WinFwdParams {
  int sq, skv, hkv, g, m_blocks;
  QTiles qt;
  WindowMask mask;
  const int32_t* kv_valid_len;
  float scale_log2;
  int nsplit;
  void* o;              // [B, Hq, Sq, 128] in the input type, with lse; nullptr: partials
  float* lse;
  float *o_part, *ml_part;
  const uint16_t *q, *k, *v;      // for plain_values
  long long q_b, q_h, q_s, k_b, k_h, k_s, v_b, v_h, v_s;
  int* status;
};

// 32 columns of one row's O over keys [key0, key1), as plain fp32 sums.
template <bool IS_BF16>
__device__ __noinline__ void window_plain_values(float* o, const uint16_t* q, const uint16_t* k, const uint16_t* v, long long ks,
                                                 long long vs, int key0, int key1, float c, float m) {
  for (int key = key0; key < key1; ++key)
    axpy32<IS_BF16>(o, ex2f(dot128<IS_BF16>(q, k + key * ks) * c - m), v + key * vs);
}

// PAIR: the slab has a single query tile (65 to 128 rows: a token each of 32 requests that share a prefix), and the two
// warpgroups take turns at its key tiles instead of one of them idling: each has an accumulator and a partial result of its
// own, and a key tile costs half of the softmax' time, which is then below that of its bytes.
template <bool IS_BF16, bool PAIR>
__global__ void __launch_bounds__(WF_THREADS, 1)
window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const WinFwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WF_OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + WFB_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slab = blockIdx.x, mb = p.m_blocks - 1 - int(blockIdx.y), split = blockIdx.z;
  const int batch = slab / p.hkv, kvh = slab % p.hkv;
  const int heads = p.qt.heads, tile_rows = heads * p.qt.tokens;

  int valid = p.skv;
  if (p.kv_valid_len) valid = min(valid, max(0, p.kv_valid_len[batch]));
  const int start = p.mask.start >= 0 ? p.mask.start : valid - p.sq;
  // token range of the CTA's two tiles (the second may not exist: its rows do not then, and its tile is loaded as zeros)
  const int tok0 = (2 * mb / p.qt.chunks) * p.qt.tokens;
  const int tok1 = min(p.sq, (min(2 * mb + 1, p.qt.count - 1) / p.qt.chunks + 1) * p.qt.tokens) - 1;
  const KeyTiles kt = key_tiles(p.mask, valid, start + tok0, start + tok1, 7);
  const int per_split = (kt.n + gridDim.z - 1) / gridDim.z;
  const int j0 = min(kt.n, split * per_split);
  const int n = min(kt.n, j0 + per_split) - j0;

  const bool poisoned = (*reinterpret_cast<volatile int*>(p.status) != 0);

  if (tid == 0) {
    mbar_init(&bars[WFB_Q_FULL], 1);
    for (int s = 0; s < WF_NS; ++s) {
      mbar_init(&bars[WFB_K_FULL + s], 1);
      mbar_init(&bars[WFB_K_EMPTY + s], 1);
      mbar_init(&bars[WFB_V_FULL + s], 1);
      mbar_init(&bars[WFB_V_EMPTY + s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[WFB_S_FULL + i], 1);
      mbar_init(&bars[WFB_P_FULL + i], 4);      // one arrival per softmax warp
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
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (!poisoned && warp < 8) {
    // =========================== softmax warpgroups ===========================
    const int wg = warp >> 2;
    const int r = (warp & 3) * 32 + lane;            // row of the tile, TMEM lane
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + wg * 128 + lane_sel;
    const uint32_t tO = tmem_base + 256 + wg * 128 + lane_sel;
    const float c = p.scale_log2;
    const int tile = PAIR ? 0 : 2 * mb + wg, tile_tok = (tile / p.qt.chunks) * p.qt.tokens;
    const int tok = tile_tok + r / heads, head = (tile % p.qt.chunks) * heads + r % heads;
    const bool exists = tile < p.qt.count && r < tile_rows && tok < p.sq && head < p.g;
    // this row's keys: [0, sink_end) and [lo, hi]. A row that does not exist sees everything against a reference of 0 (its
    // scores are zeros), so that it never holds up its warp.
    const int pos = start + tok;
    const int hi = exists ? min(pos, valid - 1) : valid - 1;
    const int lo = exists ? max(0, pos - p.mask.window + 1) : 0;
    const int sink_end = min(p.mask.sinks, hi + 1);
    // keys that every row of the warp sees: [0, all_sinks) and [all_lo, all_hi]
    const int all_hi = __reduce_min_sync(0xffffffffu, hi), all_lo = __reduce_max_sync(0xffffffffu, lo);
    const int all_sinks = min(p.mask.sinks, all_hi + 1);
    float m = exists ? -INFINITY : 0.f, l = 0.f;
    bool alive = true;
    // this warpgroup's key tiles: all of the CTA's, or every other one
    constexpr int STEP = PAIR ? 2 : 1;
    const int first = PAIR ? wg : 0;
    for (int j = first, t = 0; j < n; j += STEP, ++t) {
      const int key0 = kt.tile(j0 + j) * 128;
      const bool full = key0 + 127 <= all_hi && (key0 >= all_lo || key0 + 128 <= all_sinks);
      if (!mbar_wait(&bars[WFB_S_FULL + wg], t & 1, abort_flag, p.status, WF_CODE(wg, WFB_S_FULL))) {
        alive = false;
        break;
      }
      tc_fence_after();
      // The usual tile: exponentials against the running maximum as it stands (it is only a reference point), P held in
      // registers until the row sums are known to be small. (See fwd_sm100.cu for what each of these costs.)
      bool done = false;
      if (t > 0 && full) {
        uint32_t pk[2][32];
        uint64_t sum_a = f32x2(0.f, 0.f), sum_b = f32x2(0.f, 0.f);
        const uint64_t c2 = f32x2(c, c), nm2 = f32x2(-m, -m);
        auto chunk = [&](const uint32_t (&b)[32], uint32_t* out) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float x0, x1, x2, x3;
            f32x2_get(fma2(f32x2(__uint_as_float(b[4 * i]), __uint_as_float(b[4 * i + 1])), c2, nm2), x0, x1);
            f32x2_get(fma2(f32x2(__uint_as_float(b[4 * i + 2]), __uint_as_float(b[4 * i + 3])), c2, nm2), x2, x3);
            const float e0 = ex2f(x0), e1 = ex2f(x1), e2 = ex2f(x2), e3 = ex2f(x3);
            sum_a = add2(sum_a, f32x2(e0, e1));
            sum_b = add2(sum_b, f32x2(e2, e3));
            out[2 * i] = IS_BF16 ? pack_bf16x2(e0, e1) : pack_f16x2(e0, e1);
            out[2 * i + 1] = IS_BF16 ? pack_bf16x2(e2, e3) : pack_f16x2(e2, e3);
          }
        };
        {
          uint32_t sv[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, sv[q]);
          tc_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) chunk(sv[q], &pk[0][0] + q * 16);
        }
        float t0, t1, t2, t3;
        f32x2_get(sum_a, t0, t1);
        f32x2_get(sum_b, t2, t3);
        const float tile_sum = (t0 + t1) + (t2 + t3);
        if (__all_sync(0xffffffffu, tile_sum <= 16384.f)) {      // bounds each P; false for infinities and NaN
          tmem_st32(tS + 0, pk[0]);
          tmem_st32(tS + 32, pk[1]);
          l += tile_sum;
          done = true;
        }
      }
      if (!done) {
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, s[q]);
        tc_wait_ld();
        if (!full) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t seen = visible_bits(key0 + q * 32, lo, hi, sink_end);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(seen & (1u << i))) s[q][i] = 0xff800000u;  // -inf
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], __uint_as_float(s[q][i]));
        const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c);
        const bool grow = m_new > m + 8.f;       // raised only when it would grow by more than 2^8: P stays below 256
        float alpha = 1.f;
        if (grow) {
          alpha = ex2f(m - m_new);
          m = m_new;
          l *= alpha;
        }
        if (t > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[32];
            tmem_ld32(tO + q * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + q * 32, o);
          }
        }
        const float moff = (m == -INFINITY) ? 0.f : m;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float a0 = ex2f(fmaf(__uint_as_float(s[2 * h + e][2 * i]), c, -moff));
              const float a1 = ex2f(fmaf(__uint_as_float(s[2 * h + e][2 * i + 1]), c, -moff));
              sum0 += a0;
              sum1 += a1;
              pk[e * 16 + i] = IS_BF16 ? pack_bf16x2(a0, a1) : pack_f16x2(a0, a1);
            }
          tmem_st32(tS + h * 32, pk);
        }
        l += sum0 + sum1;
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[WFB_P_FULL + wg]);
    }
    // ------------------------------- epilogue -------------------------------
    if (alive && n > first) alive = mbar_wait(&bars[WFB_O_DONE + wg], 0, abort_flag, p.status, WF_CODE(wg, WFB_O_DONE));
    alive = __all_sync(0xffffffffu, alive);
    tc_fence_after();
    if (alive) {
      const int qh = kvh * p.g + head;
      const long long row = (static_cast<long long>(batch) * p.hkv * p.g + qh) * p.sq + tok;      // of [B, Hq, Sq]
      const long long prow = (static_cast<long long>(slab) * p.nsplit + (PAIR ? 2 * split + wg : split)) * p.g * p.sq + static_cast<long long>(head) * p.sq + tok;
      const float inv = p.o == nullptr ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;      // (NaN stays)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t o[32];
        float sum = 0.f;
        if (n > first) {
          tmem_ld32(tO + q * 32, o);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) sum += __uint_as_float(o[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (exists && isnan(sum) && l < INFINITY) {
          float again[32];
          for (int i = 0; i < 32; ++i) again[i] = 0.f;
          const uint16_t* qrow = p.q + batch * p.q_b + qh * p.q_h + tok * p.q_s;
          const uint16_t* kb = p.k + batch * p.k_b + kvh * p.k_h;
          const uint16_t* vb = p.v + batch * p.v_b + kvh * p.v_h + q * 32;
          for (int j = first; j < n; j += STEP) {
            const int key0 = kt.tile(j0 + j) * 128, key1 = key0 + 128;
            const int cut = min(key1, sink_end);          // the sinks, then what of the window lies behind them
            window_plain_values<IS_BF16>(again, qrow, kb, vb, p.k_s, p.v_s, key0, cut, c, m == -INFINITY ? 0.f : m);
            window_plain_values<IS_BF16>(again, qrow, kb, vb, p.k_s, p.v_s, max(max(key0, cut), lo), min(key1, hi + 1), c,
                                         m == -INFINITY ? 0.f : m);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(again[i]);
        }
        if (exists && p.o != nullptr) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + row * 128 + q * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = __uint_as_float(o[8 * i + 2 * e]) * inv, b = __uint_as_float(o[8 * i + 2 * e + 1]) * inv;
              w[e] = IS_BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
            }
            dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (exists) {
          float4* dst = reinterpret_cast<float4*>(p.o_part + prow * 128 + q * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                 __uint_as_float(o[4 * i + 3]));
        }
        __syncwarp();      // the next load of TMEM wants the whole warp
      }
      if (exists) {
        if (p.o != nullptr) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        else *reinterpret_cast<float2*>(p.ml_part + prow * 2) = make_float2(m, l);
      }
    }
  } else if (!poisoned && warp == 8 && n > 0) {
    // =========================== TMA producer ===========================
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      mbar_arrive_expect_tx(&bars[WFB_Q_FULL], (PAIR ? 1 : 2) * tile_rows * 256);
      for (int t = 0; t < (PAIR ? 1 : 2); ++t) {
        const int tile = 2 * mb + t;
        for (int h = 0; h < 2; ++h)
          tma_load_5d(smem + t * WF_TILE + h * WF_HALF, &tmQ, &bars[WFB_Q_FULL], h * 64, (tile % p.qt.chunks) * heads,
                      (tile / p.qt.chunks) * p.qt.tokens, kvh, batch);
      }
      int k_issued = 0, v_issued = 0;
      for (int j = 0; j < n; ++j) {
        const int s = j % WF_NS;
        const uint32_t ph = (j / WF_NS) & 1;
        const int y = kt.tile(j0 + j) * 128;
        if (!mbar_wait(&bars[WFB_K_EMPTY + s], ph ^ 1, abort_flag, p.status, WF_CODE(2, WFB_K_EMPTY))) break;
        mbar_arrive_expect_tx(&bars[WFB_K_FULL + s], WF_TILE);
        tma_load_4d(smem + WF_OFF_K + s * WF_TILE, &tmK, &bars[WFB_K_FULL + s], 0, y, kvh, batch);
        tma_load_4d(smem + WF_OFF_K + s * WF_TILE + WF_HALF, &tmK, &bars[WFB_K_FULL + s], 64, y, kvh, batch);
        k_issued = j + 1;
        if (!mbar_wait(&bars[WFB_V_EMPTY + s], ph ^ 1, abort_flag, p.status, WF_CODE(2, WFB_V_EMPTY))) break;
        mbar_arrive_expect_tx(&bars[WFB_V_FULL + s], WF_TILE);
        tma_load_4d(smem + WF_OFF_V + s * WF_TILE, &tmV, &bars[WFB_V_FULL + s], 0, y, kvh, batch);
        tma_load_4d(smem + WF_OFF_V + s * WF_TILE + WF_HALF, &tmV, &bars[WFB_V_FULL + s], 64, y, kvh, batch);
        v_issued = j + 1;
      }
      if (*abort_flag) {      // a CTA that is giving up must not leave while a copy into its shared memory is in flight
        auto drain = [&](uint64_t* bar, uint32_t ph) {
          const long long t0 = clock64();
          while (!mbar_try_wait(bar, ph) && clock64() - t0 < LVX_SPIN_LIMIT_CYCLES) {}
        };
        drain(&bars[WFB_Q_FULL], 0);
        for (int j = max(0, k_issued - WF_NS); j < k_issued; ++j) drain(&bars[WFB_K_FULL + j % WF_NS], (j / WF_NS) & 1);
        for (int j = max(0, v_issued - WF_NS); j < v_issued; ++j) drain(&bars[WFB_V_FULL + j % WF_NS], (j / WF_NS) & 1);
      }
    }
  } else if (!poisoned && warp == 9 && n > 0) {
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
    auto issue_pv = [&](int i, int stage, bool first) {
      const uint32_t b_lo = umma_desc_lo(sV + stage * WF_TILE, WF_HALF);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
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
    // rows of V behind the last valid key: whatever they hold is multiplied with zeros
    auto clear_v = [&](int j, int s) {
      const int left = valid - kt.tile(j0 + j) * 128;
      if (left >= 128) return;
      for (int at = lane; at < (128 - left) * 16; at += 32)
        *reinterpret_cast<uint4*>(smem + WF_OFF_V + s * WF_TILE + ((at >> 3) & 1) * WF_HALF + (left + (at >> 4)) * 128 + (at & 7) * 16) =
            make_uint4(0u, 0u, 0u, 0u);
      fence_async_smem();
      __syncwarp();
    };
    bool ok = wait(WFB_Q_FULL, 0) && wait(WFB_K_FULL, 0);
    if constexpr (PAIR) {
      // tile j is warpgroup j % 2's; its scores come two tiles ahead
      for (int j = 0; ok && j < min(n, 2); ++j) {
        if (j > 0) ok = wait(WFB_K_FULL + j % WF_NS, j / WF_NS & 1);
        if (!ok) break;
        tc_fence_after();
        issue_qk(j, j % WF_NS);
        commit(&bars[WFB_S_FULL + j]);
        commit(&bars[WFB_K_EMPTY + j % WF_NS]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int i = j & 1, s = j % WF_NS, s2 = (j + 2) % WF_NS;
        ok = wait(WFB_P_FULL + i, j >> 1 & 1) && wait(WFB_V_FULL + s, j / WF_NS & 1);
        if (!ok) break;
        clear_v(j, s);
        tc_fence_after();
        issue_pv(i, s, j < 2);
        commit(&bars[WFB_V_EMPTY + s]);
        if (j + 2 < n) {
          ok = wait(WFB_K_FULL + s2, (j + 2) / WF_NS & 1);
          if (!ok) break;
          tc_fence_after();
          issue_qk(i, s2);
          commit(&bars[WFB_S_FULL + i]);
          commit(&bars[WFB_K_EMPTY + s2]);
        } else {
          commit(&bars[WFB_O_DONE + i]);
        }
      }
    } else if (ok) {
      tc_fence_after();
      issue_qk(0, 0);
      commit(&bars[WFB_S_FULL + 0]);
      issue_qk(1, 0);
      commit(&bars[WFB_S_FULL + 1]);
      commit(&bars[WFB_K_EMPTY + 0]);
    }
    for (int j = 0; !PAIR && ok && j < n; ++j) {
      const int s = j % WF_NS, s1 = (j + 1) % WF_NS;
      const uint32_t ph = (j / WF_NS) & 1, ph1 = ((j + 1) / WF_NS) & 1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!ok) break;
        ok = wait(WFB_P_FULL + i, j & 1);
        if (ok && i == 0) {
          ok = wait(WFB_V_FULL + s, ph);
          if (ok) clear_v(j, s);
        }
        if (!ok) break;
        tc_fence_after();
        issue_pv(i, s, j == 0);
        if (i == 1) commit(&bars[WFB_V_EMPTY + s]);
        if (j + 1 < n) {
          if (i == 0) ok = wait(WFB_K_FULL + s1, ph1);
          if (!ok) break;
          tc_fence_after();
          issue_qk(i, s1);
          commit(&bars[WFB_S_FULL + i]);
          if (i == 1) commit(&bars[WFB_K_EMPTY + s1]);
        } else {
          commit(&bars[WFB_O_DONE + i]);
        }
      }
    }
    if (!ok) {      // wind down: let every MMA already issued finish before TMEM is released
      commit(&bars[WFB_DRAIN]);
      const long long t0 = clock64();
      while (!mbar_try_wait(&bars[WFB_DRAIN], 0) && clock64() - t0 < LVX_SPIN_LIMIT_CYCLES) {}
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

FwdPlan plan_window(const lvx_shape& s, const lvx_window& w, bool* few) {
  FwdPlan p = plan_fwd(s);          // (fp32: as it is)
  const int g = s.Hq / s.Hkv;
  *few = s.dtype != LVX_FP32 && p.rows <= kFewRows;
  bool pair = false;
  if (s.dtype != LVX_FP32) {
    const QTiles qt = make_q_tiles(g, s.Sq);
    p.m_blocks = *few ? 1 : (qt.count + 1) / 2;
    long tiles = window_tiles(s, w, *few);
    const long base = long(p.m_blocks) * s.B * s.Hkv;
    pair = window_pair(s, tiles, *few);
    if (pair) tiles = (tiles + 1) / 2;      // what a CTA walks takes half as long
    const long most = std::min<long>(tiles > 0 ? tiles : 1, *few ? 148 : 64);
    double best_cost = 1e300;
    for (int ns = 1; ns <= most; ++ns) {
      const long waves = (base * ns + 147) / 148, per = (tiles + ns - 1) / ns;
      // 3 tiles' worth of fixed cost per CTA, and 4 for a second kernel where one would do without
      const double cost = double(waves) * (per + 3.0) + (ns > 1 && !*few ? 4.0 : 0.0);
      if (cost < best_cost * 0.995) {
        best_cost = cost;
        p.nsplit = ns;
      }
    }
    p.tiles_per_split = 0;          // the kernels share out what each CTA turns out to see
    if (pair) p.nsplit *= 2;        // partial results; the grid has half as many splits
  }
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
                      float* lse, int* status, cudaStream_t st) {
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
  p.o = o;
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
  dim3 grid(s.B * s.Hkv, pl.m_blocks, pair ? pl.nsplit / 2 : pl.nsplit);
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kern) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WF_SMEM);
    if (e == cudaSuccess) kern<<<grid, WF_THREADS, WF_SMEM, st>>>(tmQ, tmK, tmV, p);
  };
  auto pick = [&](auto one, auto two) {
    if (pair) go(two);
    else go(one);
  };
  if (s.dtype == LVX_BF16) pick(window_fwd_kernel<true, false>, window_fwd_kernel<true, true>);
  else pick(window_fwd_kernel<false, false>, window_fwd_kernel<false, true>);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(window fwd)");
  e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "window_fwd_kernel launch");
}

}  // namespace lvx
