// Which keys a query sees in causal attention with a sliding window and sinks, and how the rows of the queries are packed
// into tiles. Shared by the kernels of window_fwd_sm100.cu, window_bwd_sm100.cu, fwd_rows_sm100.cu and general_tf32.cu.
//
// Query i of batch entry b sits at position p = first_b + i, first_b = n_b - Sq or given, and sees key j where
//     j < n_b  and  j <= p  and  (j > p - window  or  j < sinks).
#pragma once
#include "lvx_internal.h"

namespace lvx {

// Lengths and positions stay below 2^28 (checked on the host), so that sums of a few of them and a window fit an int.
constexpr int kWindowMaxLen = 1 << 28;
constexpr int kNoWindow = 1 << 29;

struct WindowMask {
  int window, sinks;     // window: keys that a query sees, its own included; kNoWindow
  int start;             // position of the first query, or -1: the last query sits on the last valid key
};
inline WindowMask make_window_mask(const lvx_window& w) {
  WindowMask m;
  m.window = w.window > 0 && w.window < kNoWindow ? w.window : kNoWindow;
  m.sinks = w.sinks < kWindowMaxLen ? w.sinks : kWindowMaxLen;
  m.start = w.query_start;
  return m;
}

// The softmax' reference m, in base 2: P of a tile is 2^(score - m), and O and the sum, in fp32, are rescaled when m moves. In bf16,
// which has fp32's range, m is raised to the maximum when that has outgrown it by 2^8. In fp16 P has to stay below 2^16, and what is
// below 2^-14 loses bits (2^-25: all of them), although the row's sum counts it: beside a sink of small value that outweighs the other
// keys by 2^18 O was off by 10 % in places. There m moves to 2^7 under the maximum of the tile at hand when that is above m by 2^15 or
// below it by 2^2, as long as it stays within 2^60 of the highest it was: what lies further down adds nothing. (m only ever raised, to
// 2^12 under the maximum, cost a window with sinks 23 %: the rows see few keys of their first tile, and outgrow it in the next.)
// The backward's P is at most 1 and is rounded 2^14 larger in fp16.
template <bool IS_BF16>
struct SoftmaxRef {
  static constexpr float under = IS_BF16 ? 0.f : 7.f;
  static constexpr float grad_bits = IS_BF16 ? 0.f : 14.f, grad_gain = IS_BF16 ? 1.f : 16384.f;
#ifdef __CUDACC__
  // whether a tile of maximum `top` may move m, and whether it does; `high`: the highest m (-inf, as `top` and m may be: no move)
  static __device__ __forceinline__ bool off(float top, float m) { return IS_BF16 ? top > m + 8.f : fabsf(top - m - 6.5f) > 8.5f; }
  static __device__ __forceinline__ bool moves(float top, float m, float high) {
    return IS_BF16 ? top > m + 8.f : top > m + 15.f || (top < m - 2.f && top - under > high - 60.f);
  }
#endif
};

// The key tiles that queries at positions p0..p1 see: [0, ns) for the sinks, then w0 >= ns onwards; n in all.
struct KeyTiles {
  int ns, w0, n;
  __host__ __device__ int tile(int j) const { return j < ns ? j : w0 + j - ns; }
};
__host__ __device__ inline KeyTiles key_tiles(const WindowMask& m, int valid, int p0, int p1, int tile_shift) {
  const int round = (1 << tile_shift) - 1;
  const int hi = p1 < valid - 1 ? p1 : valid - 1;                  // last key that any of them sees
  const int lo = p0 - m.window + 1 > 0 ? p0 - m.window + 1 : 0;    // first key of the first one's window
  const int sink_end = (m.sinks < hi + 1 ? m.sinks : hi + 1);
  KeyTiles t;
  t.ns = sink_end > 0 ? (sink_end + round) >> tile_shift : 0;
  t.w0 = lo >> tile_shift;
  int nw = 0;
  if (hi >= lo) {
    nw = (hi >> tile_shift) + 1 - t.w0;
    if (t.ns > t.w0) t.ns = t.w0;
  } else if (t.w0 < t.ns) {
    t.w0 = t.ns;
  }
  t.n = t.ns + nw;
  return t;
}

// Tiles of 128 query rows for one KV head: the heads of a group that share it side by side for each token, so that a
// tile spans few tokens and its keys are nearly the same for all of its rows. Row r of tile t is token
// (t / chunks) * tokens + r / heads, head (t % chunks) * heads + r % heads of the group; rows from heads * tokens on,
// heads past the group's last and tokens past Sq do not exist. One TMA box fetches a tile from a tensor of any strides.
struct QTiles {
  int heads, tokens;     // of a tile
  int chunks;            // tiles that a group of more than 128 heads takes
  int count;             // tiles of a KV head
};
inline QTiles make_q_tiles(int g, int sq) {
  QTiles q;
  q.heads = g < 128 ? g : 128;
  q.tokens = 128 / q.heads;
  q.chunks = (g + q.heads - 1) / q.heads;
  q.count = int(((long long)sq + q.tokens - 1) / q.tokens * q.chunks);
  return q;
}

#ifdef __CUDACC__
// x low bits set (0 <= x <= 32)
__device__ __forceinline__ uint32_t low_bits(int x) { return x >= 32 ? 0xffffffffu : (1u << x) - 1u; }
__device__ __forceinline__ int clamp32(int x) { return min(max(x, 0), 32); }
// Of the 32 keys from key0 on, those that lie in [0, sink_end) or [lo, hi]; sink_end <= hi + 1.
__device__ __forceinline__ uint32_t visible_bits(int key0, int lo, int hi, int sink_end) {
  return (low_bits(clamp32(hi + 1 - key0)) & ~low_bits(clamp32(lo - key0))) | low_bits(clamp32(sink_end - key0));
}
#endif

// Split of the key tiles over CTAs, and the layout of the partial results (FwdPlan's, with rows in the order of
// [B, Hq, Sq]); shared by the launchers and the workspace query. nsplit == 1 and not `few`: results are written directly.
FwdPlan plan_window(const lvx_shape& s, const lvx_window& w, bool* few, bool merged = false);

// SMs of the current device.
inline int num_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0)
    return n;
  return 148;
}

// Tensor map of up to five dimensions over 128-byte wide boxes with the 128-byte swizzle; strides in bytes, from the second
// dimension on.
int make_tmap_nd(CUtensorMap* out, int dtype, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                 const uint32_t* box);
// Q / dO tiles (rank 5: d, head of the group, token, KV head, batch entry) and K / V tiles (rank 4: d, key, KV head, batch
// entry) of tensors of any strides.
int make_q_map(CUtensorMap* out, const lvx_shape& s, const QTiles& qt, const lvx_view& v);
int make_kv_map(CUtensorMap* out, const lvx_shape& s, const lvx_view& v, const lvx_view& dummy);

}  // namespace lvx
