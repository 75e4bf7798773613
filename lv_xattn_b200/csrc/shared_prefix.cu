// Attention for a batch that shares a long prefix (a video's tokens), with keys of each request's own behind it: one softmax
// over both. The B / P requests of a prefix put all of their query rows (heads of the group, tokens) side by side as the rows
// of one KV head, so that the prefix is read once for all of them and its products are as tall as the batch; the own keys
// are a causal attention of each request. Both are the windowed attention kernels (the prefix: rows that stand behind all of
// its keys) and leave partial results that one kernel merges here. The backward is the same the other way round: with the
// merged log-sum-exp and delta each side's gradients are those of an attention of its own, and dQ is their sum.
//
// What is here are the small kernels around them, all bound by memory and small next to the prefix:
//   pack      rows of q (dO, lse, delta) from [B, Hq, Sq] to [P, Hkv, B / P, Hq / Hkv, Sq]: one copy of the queries, against a
//             prefix that is 100 to 100,000 times as long. Not done where the two orders are the same (one request per
//             prefix, or one KV head), nor in the forward of single tokens in 16 bits, where the requests are the tokens of
//             a view of q (eight tokens behind 6,404 keys 32 -> 29 us a call, 32 behind 102,464 128 -> 126 on the GPU).
//   combine   partials of the prefix (packed rows) and of the own keys (rows of a request) -> O and lse
//   dq        sum of the two fp32 accumulators, rounded once
#include "combine.cuh"
#include "window.cuh"
#include <algorithm>

namespace lvx {

// A row of [B, Hq, Sq] in the packed order [P, Hkv, per, g, Sq], per = B / P, or with `by_head` (Sq = 1) [P, Hkv, g, per]. Rows are
// counted in 32 bits (checked on the host): 64-bit divisions are most of what these kernels would execute.
struct PackOrder {
  int hkv, g, sq, per;
  bool by_head;
  __device__ __forceinline__ void split(int row, int& slab, int& in_slab) const {      // (KV head of a request, row in it)
    const int rows = g * sq;
    slab = row / rows;
    in_slab = row - slab * rows;
  }
  // packed row: of slab p * hkv + kvh
  __device__ __forceinline__ void packed(int slab, int in_slab, int& pslab, int& prow) const {
    const int b = slab / hkv, kvh = slab - b * hkv, p = b / per;
    pslab = p * hkv + kvh;
    prow = by_head ? in_slab * per + b - p * per : (b - p * per) * g * sq + in_slab;
  }
  __device__ __forceinline__ int packed_rows() const { return per * g * sq; }
};
static PackOrder pack_order(const lvx_shape& s, int prefixes, bool by_head = false) {
  return PackOrder{s.Hkv, s.Hq / s.Hkv, s.Sq, s.B / prefixes, by_head};
}

// ROW16: 16-byte pieces of a row (16: 16-bit types, 32: fp32), one a thread; a thread takes that piece of four rows, which are
// in flight together (42,624 rows of bf16: 10 -> 6 us against one row a thread and 64-bit arithmetic).
template <int ROW16>
__global__ void __launch_bounds__(256)
pack_rows_kernel(const char* __restrict__ q, long long q_b, long long q_h, long long q_s, const uint4* __restrict__ d_o,
                 const float* __restrict__ lse, const float* __restrict__ delta, uint4* __restrict__ q_out, uint4* __restrict__ do_out,
                 float* __restrict__ lse_out, float* __restrict__ delta_out, PackOrder order, int rows, const int* status) {
  grid_dep_wait();
  grid_dep_launch();
  grid_dep_read(delta);
  if (poisoned(status)) return;
  constexpr int U = 4, PER = 256 / ROW16;      // rows of a thread, rows of a block at a time
  const int piece = threadIdx.x % ROW16, row0 = blockIdx.x * PER * U + threadIdx.x / ROW16;
  uint4 v[U], w[U];
  int to[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = min(row0 + u * PER, rows - 1);
    int slab, in_slab, pslab, prow;
    order.split(row, slab, in_slab);
    order.packed(slab, in_slab, pslab, prow);
    to[u] = pslab * order.packed_rows() + prow;
    const int b = slab / order.hkv, head = in_slab / order.sq, tok = in_slab - head * order.sq;
    const int h = (slab - b * order.hkv) * order.g + head;
    v[u] = *reinterpret_cast<const uint4*>(q + b * q_b + h * q_h + tok * q_s + piece * 16);
    if (d_o != nullptr) w[u] = d_o[size_t(row) * ROW16 + piece];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + u * PER;
    if (row >= rows) return;
    q_out[size_t(to[u]) * ROW16 + piece] = v[u];
    if (d_o != nullptr) {
      do_out[size_t(to[u]) * ROW16 + piece] = w[u];
      if (piece == 0) {
        lse_out[to[u]] = lse[row];
        delta_out[to[u]] = delta[row];
      }
    }
  }
}

template <int OUT, int WPR>
__global__ void __launch_bounds__(256)
shared_combine_kernel(const float* __restrict__ o_pre, const float* __restrict__ ml_pre, int ns_pre, const float* __restrict__ o_own,
                      const float* __restrict__ ml_own, int ns_own, PackOrder order, void* __restrict__ o_out,
                      float* __restrict__ lse_out, int rows, const int* status) {
  grid_dep_wait();
  grid_dep_read(o_pre);
  grid_dep_read(ml_pre);
  grid_dep_read(o_own);
  grid_dep_read(ml_own);
  const int bad = status ? *reinterpret_cast<const volatile int*>(status) : 0;
  const int lane = threadIdx.x & 31, part = (threadIdx.x >> 5) % WPR;
  const int row = (blockIdx.x * 8 + (threadIdx.x >> 5)) / WPR;
  if (row >= rows) return;                 // WPR > 1: a block is one row, so its warps leave together
  int slab, in_slab, pslab, prow;
  order.split(row, slab, in_slab);
  order.packed(slab, in_slab, pslab, prow);
  RowAcc a;
  a.m = -INFINITY;
  a.l = 0.f;
  a.v = make_float4(0.f, 0.f, 0.f, 0.f);
  // four partials at a time in flight (eight: 53 -> 73 us for 42,624 rows of seven and one, with half the warps an SM)
  const int groups = (ns_pre + 3) >> 2, own_groups = (ns_own + 3) >> 2;
  for (int i = part; i < groups + own_groups; i += WPR) {
    if (i < groups) row_four(a, o_pre, ml_pre, pslab, ns_pre, order.packed_rows(), prow, i * 4, lane, true);
    else row_four(a, o_own, ml_own, slab, ns_own, order.g * order.sq, in_slab, (i - groups) * 4, lane, true);
  }
  if constexpr (WPR > 1) {
    __shared__ float4 s_v[WPR][32];
    __shared__ float2 s_ml[WPR];
    s_v[part][lane] = a.v;
    if (lane == 0) s_ml[part] = make_float2(a.m, a.l);
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      RowAcc b;
      b.m = s_ml[w].x;
      b.l = s_ml[w].y;
      b.v = s_v[w][lane];
      row_merge(a, b);
    }
  }
  if (bad) {
    if (lane == 0) publish_status(status);
    return;
  }
  const float inv = a.l == 0.f ? 0.f : 1.f / a.l;      // a row without keys: zeros and -inf
  store4<OUT>(o_out, size_t(row) * 32 + lane, make_float4(a.v.x * inv, a.v.y * inv, a.v.z * inv, a.v.w * inv));
  if (lane == 0) lse_out[row] = a.l == 0.f ? -INFINITY : (a.m + log2f(a.l)) * kLn2;
}

// dq = cast(acc_pre (packed rows) + acc_own). The prefix' accumulator is in tiles of `pre_tile` rows for each slab, the own
// one in the order of window_bwd_sm100.cu's tiles (heads of a tile, chunks).
template <int OUT>
__global__ void __launch_bounds__(256)
shared_dq_kernel(const float* __restrict__ acc_pre, int pre_slab_rows, const float* __restrict__ acc_own, int heads, int chunks,
                 PackOrder order, void* __restrict__ dq, int rows, const int* status) {
  grid_dep_wait();
  grid_dep_read(acc_pre);
  grid_dep_read(acc_own);
  if (poisoned(status)) {
    if ((threadIdx.x & 31) == 0) publish_status(status);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int row = blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8) {
    int slab, in_slab, pslab, prow;
    order.split(row, slab, in_slab);
    order.packed(slab, in_slab, pslab, prow);
    float4 v = reinterpret_cast<const float4*>(acc_pre)[(size_t(pslab) * pre_slab_rows + prow) * 32 + lane];
    if (acc_own != nullptr) {
      const int head = in_slab / order.sq, tok = in_slab - head * order.sq;
      const size_t at = ((size_t(slab) * chunks + head / heads) * order.sq + tok) * heads + head % heads;
      const float4 w = reinterpret_cast<const float4*>(acc_own)[at * 32 + lane];
      v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
    }
    store4<OUT>(dq, size_t(row) * 32 + lane, v);
  }
}

int launch_pack_rows(const lvx_shape& s, int prefixes, const lvx_view& q, const void* d_o, const float* lse, const float* delta,
                     void* q_out, void* do_out, float* lse_out, float* delta_out, Order order, cudaStream_t st) {
  const int rows = s.B * s.Hq * s.Sq;
  const int es = elt_size(s.dtype), pieces = es * 8;
  auto go = [&](auto kern) {
    return launch_kernel(order, kern, dim3((rows + 1024 / pieces - 1) / (1024 / pieces)), 256, 0, st, static_cast<const char*>(q.data),
                         q.stride_b * es, q.stride_h * es, q.stride_s * es, static_cast<const uint4*>(d_o), lse, delta,
                         static_cast<uint4*>(q_out), static_cast<uint4*>(do_out), lse_out, delta_out, pack_order(s, prefixes), rows,
                         device_status_ptr());
  };
  const cudaError_t e = es == 2 ? go(pack_rows_kernel<16>) : go(pack_rows_kernel<32>);
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "pack_rows launch");
}

int launch_shared_combine(const lvx_shape& s, int prefixes, bool by_head, const float* o_pre, const float* ml_pre, int ns_pre, const float* o_own,
                          const float* ml_own, int ns_own, void* o, float* lse, cudaStream_t st) {
  const int rows = s.B * s.Hq * s.Sq;
  // as in launch_fwd_combine: eight warps a row while the rows alone leave SMs empty and one warp's walk is long
  const bool wide = rows <= 148 * 8 && ns_pre + ns_own > 8;
  auto go = [&](auto one, auto eight) {
    return launch_kernel(ORDER_OVERLAP, wide ? eight : one, dim3(wide ? rows : (rows - 1) / 8 + 1), 256, 0, st, o_pre, ml_pre, ns_pre, o_own, ml_own,
                         ns_own, pack_order(s, prefixes, by_head), o, lse, rows, device_status_ptr());
  };
  const cudaError_t e = s.dtype == LVX_BF16   ? go(shared_combine_kernel<0, 1>, shared_combine_kernel<0, 8>)
                        : s.dtype == LVX_FP16 ? go(shared_combine_kernel<1, 1>, shared_combine_kernel<1, 8>)
                                              : go(shared_combine_kernel<2, 1>, shared_combine_kernel<2, 8>);
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "shared_combine launch");
}

int launch_shared_dq(const lvx_shape& s, int prefixes, const float* acc_pre, int pre_slab_rows, const float* acc_own, void* dq,
                     cudaStream_t st) {
  const int rows = s.B * s.Hq * s.Sq;
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  // the general kernel accumulates in the order of [B, Hq, Sq]: one head a chunk
  const int heads = s.dtype == LVX_FP32 ? 1 : qt.heads, chunks = s.dtype == LVX_FP32 ? s.Hq / s.Hkv : qt.chunks;
  const int blocks = std::min((rows - 1) / 8 + 1, 148 * 16);
  auto go = [&](auto kern) {
    return launch_kernel(ORDER_OVERLAP, kern, dim3(blocks), 256, 0, st, acc_pre, pre_slab_rows, acc_own, heads, chunks, pack_order(s, prefixes), dq,
                         rows, device_status_ptr());
  };
  const cudaError_t e = s.dtype == LVX_BF16   ? go(shared_dq_kernel<0>)
                        : s.dtype == LVX_FP16 ? go(shared_dq_kernel<1>)
                                              : go(shared_dq_kernel<2>);
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "shared_dq launch");
}

}  // namespace lvx
