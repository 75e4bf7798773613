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
//             prefix, or one KV head).
//   combine   partials of the prefix (packed rows) and of the own keys (rows of a request) -> O and lse
//   dq        sum of the two fp32 accumulators, rounded once
#include "combine.cuh"
#include "window.cuh"
#include <algorithm>

namespace lvx {

// A row of [B, Hq, Sq] in the packed order [P, Hkv, per, g, Sq], per = B / P.
struct PackOrder {
  int hkv, g, sq, per;
  __device__ __forceinline__ void split(long row, long& slab, int& in_slab) const {      // (KV head of a request, row in it)
    const int rows = g * sq;
    slab = row / rows;
    in_slab = int(row - slab * rows);
  }
  // packed row: of slab p * hkv + kvh
  __device__ __forceinline__ void packed(long slab, int in_slab, long& pslab, int& prow) const {
    const long b = slab / hkv;
    const int kvh = int(slab - b * hkv);
    const long p = b / per;
    pslab = p * hkv + kvh;
    prow = int(b - p * per) * g * sq + in_slab;
  }
  __device__ __forceinline__ long packed_rows() const { return long(per) * g * sq; }
};
static PackOrder pack_order(const lvx_shape& s, int prefixes) { return PackOrder{s.Hkv, s.Hq / s.Hkv, s.Sq, s.B / prefixes}; }

// ROW16: 16-byte pieces of a row (16: 16-bit types, 32: fp32). One piece a thread.
template <int ROW16>
__global__ void __launch_bounds__(256)
pack_rows_kernel(const char* __restrict__ q, long long q_b, long long q_h, long long q_s, const uint4* __restrict__ d_o,
                 const float* __restrict__ lse, const float* __restrict__ delta, uint4* __restrict__ q_out, uint4* __restrict__ do_out,
                 float* __restrict__ lse_out, float* __restrict__ delta_out, PackOrder order, long rows, const int* status) {
  if (poisoned(status)) return;
  const long at = long(blockIdx.x) * 256 + threadIdx.x;
  const long row = at / ROW16;
  const int piece = int(at % ROW16);
  if (row >= rows) return;
  long slab, pslab;
  int in_slab, prow;
  order.split(row, slab, in_slab);
  order.packed(slab, in_slab, pslab, prow);
  const long to = pslab * order.packed_rows() + prow;
  const long bh = row / order.sq, b = slab / order.hkv;
  const int h = int(bh - b * order.hkv * order.g), tok = int(row - bh * order.sq);
  q_out[to * ROW16 + piece] = *reinterpret_cast<const uint4*>(q + b * q_b + h * q_h + tok * q_s + piece * 16);
  if (d_o != nullptr) {
    do_out[to * ROW16 + piece] = d_o[at];
    if (piece == 0) {
      lse_out[to] = lse[row];
      delta_out[to] = delta[row];
    }
  }
}

template <int OUT, int WPR>
__global__ void __launch_bounds__(256)
shared_combine_kernel(const float* __restrict__ o_pre, const float* __restrict__ ml_pre, int ns_pre, const float* __restrict__ o_own,
                      const float* __restrict__ ml_own, int ns_own, PackOrder order, void* __restrict__ o_out,
                      float* __restrict__ lse_out, long rows, const int* status) {
  const int bad = status ? *reinterpret_cast<const volatile int*>(status) : 0;
  const int lane = threadIdx.x & 31, part = (threadIdx.x >> 5) % WPR;
  const long row = ((long(blockIdx.x) * blockDim.x + threadIdx.x) >> 5) / WPR;
  if (row >= rows) return;                 // WPR > 1: a block is one row, so its warps leave together
  long slab, pslab;
  int in_slab, prow;
  order.split(row, slab, in_slab);
  order.packed(slab, in_slab, pslab, prow);
  RowAcc a;
  a.m = -INFINITY;
  a.l = 0.f;
  a.v = make_float4(0.f, 0.f, 0.f, 0.f);
  const int groups = (ns_pre + 3) >> 2, own_groups = (ns_own + 3) >> 2;
  for (int i = part; i < groups + own_groups; i += WPR) {
    if (i < groups) row_four(a, o_pre, ml_pre, size_t(pslab), ns_pre, int(order.packed_rows()), prow, i * 4, lane);
    else row_four(a, o_own, ml_own, size_t(slab), ns_own, order.g * order.sq, in_slab, (i - groups) * 4, lane);
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
shared_dq_kernel(const float* __restrict__ acc_pre, long pre_slab_rows, const float* __restrict__ acc_own, int heads, int chunks,
                 PackOrder order, void* __restrict__ dq, long rows, const int* status) {
  if (poisoned(status)) {
    if ((threadIdx.x & 31) == 0) publish_status(status);
    return;
  }
  const int lane = threadIdx.x & 31;
  for (long row = (long(blockIdx.x) * 256 + threadIdx.x) >> 5; row < rows; row += long(gridDim.x) * 8) {
    long slab, pslab;
    int in_slab, prow;
    order.split(row, slab, in_slab);
    order.packed(slab, in_slab, pslab, prow);
    float4 v = reinterpret_cast<const float4*>(acc_pre)[(pslab * pre_slab_rows + prow) * 32 + lane];
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
                     void* q_out, void* do_out, float* lse_out, float* delta_out, cudaStream_t st) {
  const long rows = long(s.B) * s.Hq * s.Sq;
  const int es = elt_size(s.dtype), pieces = es * 8;
  auto go = [&](auto kern) {
    kern<<<(rows * pieces + 255) / 256, 256, 0, st>>>(static_cast<const char*>(q.data), q.stride_b * es, q.stride_h * es,
                                                      q.stride_s * es, static_cast<const uint4*>(d_o), lse, delta,
                                                      static_cast<uint4*>(q_out), static_cast<uint4*>(do_out), lse_out, delta_out,
                                                      pack_order(s, prefixes), rows, device_status_ptr());
  };
  if (es == 2) go(pack_rows_kernel<16>);
  else go(pack_rows_kernel<32>);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "pack_rows launch");
}

int launch_shared_combine(const lvx_shape& s, int prefixes, const float* o_pre, const float* ml_pre, int ns_pre, const float* o_own,
                          const float* ml_own, int ns_own, void* o, float* lse, cudaStream_t st) {
  const long rows = long(s.B) * s.Hq * s.Sq;
  // as in launch_fwd_combine: eight warps a row while the rows alone leave SMs empty and one warp's walk is long
  const bool wide = rows <= 148 * 8 && ns_pre + ns_own > 8;
  auto go = [&](auto one, auto eight) {
    if (wide) eight<<<rows, 256, 0, st>>>(o_pre, ml_pre, ns_pre, o_own, ml_own, ns_own, pack_order(s, prefixes), o, lse, rows, device_status_ptr());
    else one<<<(rows + 7) / 8, 256, 0, st>>>(o_pre, ml_pre, ns_pre, o_own, ml_own, ns_own, pack_order(s, prefixes), o, lse, rows, device_status_ptr());
  };
  if (s.dtype == LVX_BF16) go(shared_combine_kernel<0, 1>, shared_combine_kernel<0, 8>);
  else if (s.dtype == LVX_FP16) go(shared_combine_kernel<1, 1>, shared_combine_kernel<1, 8>);
  else go(shared_combine_kernel<2, 1>, shared_combine_kernel<2, 8>);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "shared_combine launch");
}

int launch_shared_dq(const lvx_shape& s, int prefixes, const float* acc_pre, long pre_slab_rows, const float* acc_own, void* dq,
                     cudaStream_t st) {
  const long rows = long(s.B) * s.Hq * s.Sq;
  const QTiles qt = make_q_tiles(s.Hq / s.Hkv, s.Sq);
  // the general kernel accumulates in the order of [B, Hq, Sq]: one head a chunk
  const int heads = s.dtype == LVX_FP32 ? 1 : qt.heads, chunks = s.dtype == LVX_FP32 ? s.Hq / s.Hkv : qt.chunks;
  const long blocks = std::min<long>((rows + 7) / 8, 148 * 16);
  auto go = [&](auto kern) {
    kern<<<blocks, 256, 0, st>>>(acc_pre, pre_slab_rows, acc_own, heads, chunks, pack_order(s, prefixes), dq, rows, device_status_ptr());
  };
  if (s.dtype == LVX_BF16) go(shared_dq_kernel<0>);
  else if (s.dtype == LVX_FP16) go(shared_dq_kernel<1>);
  else go(shared_dq_kernel<2>);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "shared_dq launch");
}

}  // namespace lvx
