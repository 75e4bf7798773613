// RMSNorm of every query and key head and the rotary embedding, in one pass, from the projections' layout (any strides,
// usually [B, S, H, 128]) to the attention kernels' [B, H, S, 128]; and its backward.
//
//   forward   r = rsqrt(mean_d(x^2) + eps), y = x r w;   out_d = y_d cos_d - y_{d+64} sin_d,
//             out_{d+64} = y_{d+64} cos_{d+64} + y_d sin_{d+64}   (d < 64)
//   backward  dy = the rotation's transpose of the gradient; xh = x r;
//             dx = r (w dy - xh mean_d(w dy xh)),   dw = sum over rows of dy xh
// All of it in fp32, rounded once when it is stored. r is computed again in the backward: x is read there anyway.
//
// Bound by memory (a row of 128 values in and out, two in and one out in the backward). Sixteen lanes work on a row; a
// lane holds d = 4l..4l+3 and the same of the other half, so that the rotation needs no exchange between lanes. A lane
// group takes four heads of one token (a unit): four rows in flight, and the token's cos and sin, which are as wide as
// two rows in fp32, are fetched once for them. The units of a block are neighbours, mostly of one token, so the tables
// come from L1. dw is kept in registers over a walk through the units, summed per block and then by a second kernel in a
// fixed order: atomics on its 128 addresses would cost both time and the same result twice.
#include "lvx_internal.h"
#include "sm100_prims.cuh"
#include <algorithm>

namespace lvx {

constexpr int HN_U = 4;             // heads of a unit
constexpr int HN_GROUPS = 16;       // lane groups of a block
constexpr int HN_BWD_BLOCKS = 148 * 4;
static_assert(HN_BWD_BLOCKS * 256 * sizeof(float) == LVX_HEAD_NORM_SCRATCH, "the header names the scratch's size");

struct HeadNormParams {
  int S, heads[2], chunks[2];       // [0] queries, [1] keys; chunks: units of a token
  long units;
  const void* x[2];
  long long x_b[2], x_h[2], x_s[2];
  const void* w[2];                 // nullptr: no norm
  int w_fp32, table_fp32;
  float eps;
  const void *cos, *sin;            // nullptr: no rotation
  long long t_b, t_s;
  void* out[2];                     // forward: [B, H, S, 128]; backward: dx [B, S, H, 128], nullptr: not wanted
  const void* g[2];                 // backward: gradient of `out`
  long long g_b[2], g_h[2], g_s[2];
  float* dw_part;                   // backward: [blocks][2][128], nullptr: no weight wants its gradient
  const int* status;
};

// four values of either type
template <int T>      // 0 bf16, 1 fp16, 2 fp32
__device__ __forceinline__ float4 hn_load(const void* base, long long at) {
  if (T == 2) return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + at);
  const float2 a = unpack16x2<T == 0>(u.x), b = unpack16x2<T == 0>(u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
template <int T>
__device__ __forceinline__ float4 hn_load_either(const void* base, long long at, int fp32) {
  return T == 2 || fp32 ? hn_load<2>(base, at) : hn_load<T>(base, at);
}
template <int T>
__device__ __forceinline__ void hn_store(void* base, long long at, float4 v) {
  if (T == 2) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = v;
  } else {
    const uint2 u = T == 0 ? make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)) : make_uint2(pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = u;
  }
}
__device__ __forceinline__ float4 hn_mul(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float4 hn_scale(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
__device__ __forceinline__ float4 hn_fma(float4 a, float4 b, float4 c) {
  return make_float4(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y), fmaf(a.z, b.z, c.z), fmaf(a.w, b.w, c.w));
}
__device__ __forceinline__ float4 hn_neg(float4 a) { return make_float4(-a.x, -a.y, -a.z, -a.w); }
__device__ __forceinline__ float hn_dot(float4 a, float4 b) { return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, a.w * b.w))); }

struct Half2 {        // a lane's share of a row: d = 4l.. and 64 + 4l..
  float4 a, b;
};
// sum over the sixteen lanes of a group, of HN_U values at a time
__device__ __forceinline__ void hn_sum(float (&v)[HN_U]) {
#pragma unroll
  for (int off = 8; off > 0; off >>= 1)
#pragma unroll
    for (int u = 0; u < HN_U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], off);
}

template <int T, bool BWD>
__global__ void __launch_bounds__(HN_GROUPS * 16)
head_norm_kernel(const HeadNormParams p) {
  __shared__ float s_dw[BWD ? HN_GROUPS : 1][128];
  int bad = 0;
  if (p.status) bad = *reinterpret_cast<const volatile int*>(p.status);
  const int group = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4;
  Half2 dw[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) dw[i].a = dw[i].b = make_float4(0.f, 0.f, 0.f, 0.f);
  const int per_token = p.chunks[0] + p.chunks[1];
  // The two groups of a warp walk together (their sums are exchanged with the whole warp's mask): the last unit may be
  // done twice, by a group that then stores nothing.
  for (long u0 = long(blockIdx.x) * HN_GROUPS + (group & ~1); u0 < p.units; u0 += long(gridDim.x) * HN_GROUPS) {
    const long unit = min(u0 + (group & 1), p.units - 1);
    const bool mine = u0 + (group & 1) < p.units;
    const long token = unit / per_token;
    int chunk = int(unit - token * per_token);
    const int which = chunk >= p.chunks[0];
    if (which) chunk -= p.chunks[0];
    const long b = token / p.S, s = token - b * p.S;
    const int h0 = chunk * HN_U, heads = p.heads[which];
    const void* xw = p.x[which];
    const void* ww = p.w[which];
    Half2 x[HN_U], g[BWD ? HN_U : 1];
#pragma unroll
    for (int u = 0; u < HN_U; ++u) {
      const int h = min(h0 + u, heads - 1);
      const long long at = b * p.x_b[which] + h * p.x_h[which] + s * p.x_s[which] + d;
      if (!BWD || ww != nullptr) {
        x[u].a = hn_load<T>(xw, at);
        x[u].b = hn_load<T>(xw, at + 64);
      }
      if constexpr (BWD) {
        const long long ga = b * p.g_b[which] + h * p.g_h[which] + s * p.g_s[which] + d;
        g[u].a = hn_load<T>(p.g[which], ga);
        g[u].b = hn_load<T>(p.g[which], ga + 64);
      }
    }
    Half2 c, sn, w;
    if (p.cos != nullptr) {
      const long long at = b * p.t_b + s * p.t_s + d;
      c.a = hn_load_either<T>(p.cos, at, p.table_fp32);
      c.b = hn_load_either<T>(p.cos, at + 64, p.table_fp32);
      sn.a = hn_load_either<T>(p.sin, at, p.table_fp32);
      sn.b = hn_load_either<T>(p.sin, at + 64, p.table_fp32);
    }
    // The sums are exchanged between lanes whether this group has a norm or not: the warp's other group may.
    float r[HN_U];
    if (ww != nullptr) {
      w.a = hn_load_either<T>(ww, d, p.w_fp32);
      w.b = hn_load_either<T>(ww, d + 64, p.w_fp32);
    }
#pragma unroll
    for (int u = 0; u < HN_U; ++u) r[u] = ww != nullptr ? hn_dot(x[u].a, x[u].a) + hn_dot(x[u].b, x[u].b) : 0.f;
    hn_sum(r);
#pragma unroll
    for (int u = 0; u < HN_U; ++u) r[u] = rsqrtf(r[u] * (1.f / 128.f) + p.eps);
    if constexpr (!BWD) {
#pragma unroll
      for (int u = 0; u < HN_U; ++u) {
        Half2 y = x[u];
        if (ww != nullptr) {
          y.a = hn_mul(hn_scale(y.a, r[u]), w.a);
          y.b = hn_mul(hn_scale(y.b, r[u]), w.b);
        }
        if (p.cos != nullptr) {
          const Half2 z = y;
          y.a = hn_fma(z.a, c.a, hn_neg(hn_mul(z.b, sn.a)));
          y.b = hn_fma(z.b, c.b, hn_mul(z.a, sn.b));
        }
        if (mine && !bad && h0 + u < heads) {
          const long long at = ((b * heads + h0 + u) * p.S + s) * 128 + d;
          hn_store<T>(p.out[which], at, y.a);
          hn_store<T>(p.out[which], at + 64, y.b);
        }
      }
    } else {
      float m[HN_U];
#pragma unroll
      for (int u = 0; u < HN_U; ++u) {
        if (p.cos != nullptr) {
          const Half2 z = g[u];
          g[u].a = hn_fma(z.a, c.a, hn_mul(z.b, sn.b));
          g[u].b = hn_fma(z.b, c.b, hn_neg(hn_mul(z.a, sn.a)));
        }
        m[u] = 0.f;
        if (ww != nullptr) {
          x[u].a = hn_scale(x[u].a, r[u]);
          x[u].b = hn_scale(x[u].b, r[u]);
          if (mine && h0 + u < heads) {
            // (selected, not indexed: an array of registers has no run-time index)
            if (which) {
              dw[1].a = hn_fma(g[u].a, x[u].a, dw[1].a);
              dw[1].b = hn_fma(g[u].b, x[u].b, dw[1].b);
            } else {
              dw[0].a = hn_fma(g[u].a, x[u].a, dw[0].a);
              dw[0].b = hn_fma(g[u].b, x[u].b, dw[0].b);
            }
          }
          g[u].a = hn_mul(g[u].a, w.a);
          g[u].b = hn_mul(g[u].b, w.b);
          m[u] = hn_dot(g[u].a, x[u].a) + hn_dot(g[u].b, x[u].b);
        }
      }
      hn_sum(m);
#pragma unroll
      for (int u = 0; u < HN_U; ++u) {
        if (ww != nullptr) {
          const float mean = -m[u] * (1.f / 128.f);
          g[u].a = hn_scale(hn_fma(x[u].a, make_float4(mean, mean, mean, mean), g[u].a), r[u]);
          g[u].b = hn_scale(hn_fma(x[u].b, make_float4(mean, mean, mean, mean), g[u].b), r[u]);
        }
        if (mine && !bad && p.out[which] != nullptr && h0 + u < heads) {
          const long long at = ((b * p.S + s) * heads + h0 + u) * 128 + d;
          hn_store<T>(p.out[which], at, g[u].a);
          hn_store<T>(p.out[which], at + 64, g[u].b);
        }
      }
    }
  }
  if (bad && (threadIdx.x & 31) == 0) publish_status(p.status);
  if constexpr (BWD) {
    if (p.dw_part == nullptr || __syncthreads_or(bad)) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __syncthreads();
      *reinterpret_cast<float4*>(&s_dw[group][d]) = dw[i].a;
      *reinterpret_cast<float4*>(&s_dw[group][d + 64]) = dw[i].b;
      __syncthreads();
      if (threadIdx.x < 128) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < HN_GROUPS; ++k) a += s_dw[k][threadIdx.x];
        p.dw_part[(size_t(blockIdx.x) * 2 + i) * 128 + threadIdx.x] = a;
      }
    }
  }
}

// dw[i][d] = sum over blocks of dw_part[block][i][d], in a fixed order: a block of this kernel takes 32 columns with 32
// slices of the blocks each.
template <int T>
__global__ void __launch_bounds__(1024)
head_norm_dw_kernel(const float* __restrict__ part, int blocks, void* dwq, void* dwk, int w_fp32, const int* status) {
  if (status && *reinterpret_cast<const volatile int*>(status) != 0) {
    if ((threadIdx.x & 31) == 0) publish_status(status);
    return;
  }
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float a = 0.f;
  for (int k = slice; k < blocks; k += 32) a += part[size_t(k) * 256 + col];
  s[slice][threadIdx.x & 31] = a;
  __syncthreads();
  a = s[threadIdx.x & 31][slice];           // lane = slice, warp = column
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
  if ((threadIdx.x & 31) == 0) {
    const int c = blockIdx.x * 32 + slice;
    void* dst = c < 128 ? dwq : dwk;
    if (dst == nullptr) return;
    if (T == 2 || w_fp32) static_cast<float*>(dst)[c & 127] = a;
    else static_cast<uint16_t*>(dst)[c & 127] = uint16_t(T == 0 ? pack_bf16x2(a, 0.f) : pack_f16x2(a, 0.f));
  }
}

static HeadNormParams head_norm_params(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k) {
  HeadNormParams p{};
  p.S = c.S;
  const lvx_view* v[2] = {q, k};
  const int heads[2] = {q ? c.Hq : 0, k ? c.Hkv : 0};
  for (int i = 0; i < 2; ++i) {
    p.heads[i] = heads[i];
    p.chunks[i] = (heads[i] + HN_U - 1) / HN_U;
    if (!v[i]) continue;
    p.x[i] = v[i]->data;
    p.x_b[i] = v[i]->stride_b;
    p.x_h[i] = v[i]->stride_h;
    p.x_s[i] = v[i]->stride_s;
  }
  p.units = long(c.B) * c.S * (p.chunks[0] + p.chunks[1]);
  p.w[0] = c.wq;
  p.w[1] = c.wk;
  p.w_fp32 = c.weight_fp32;
  p.table_fp32 = c.table_fp32;
  p.eps = c.eps;
  p.cos = c.cos;
  p.sin = c.sin;
  p.t_b = c.table_stride_b;
  p.t_s = c.table_stride_s;
  p.status = device_status_ptr();
  return p;
}

int launch_head_norm(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, void* q_out, void* k_out, cudaStream_t st) {
  HeadNormParams p = head_norm_params(c, q, k);
  p.out[0] = q_out;
  p.out[1] = k_out;
  const long blocks = std::min<long>((p.units + HN_GROUPS - 1) / HN_GROUPS, 148 * 32);
  if (c.dtype == LVX_BF16) head_norm_kernel<0, false><<<blocks, HN_GROUPS * 16, 0, st>>>(p);
  else if (c.dtype == LVX_FP16) head_norm_kernel<1, false><<<blocks, HN_GROUPS * 16, 0, st>>>(p);
  else head_norm_kernel<2, false><<<blocks, HN_GROUPS * 16, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "head_norm_kernel launch");
}

int launch_head_norm_bwd(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, const lvx_view* gq, const lvx_view* gk,
                         void* dq, void* dk, float* scratch, void* dwq, void* dwk, cudaStream_t st) {
  HeadNormParams p = head_norm_params(c, q, k);
  p.out[0] = dq;
  p.out[1] = dk;
  const lvx_view* g[2] = {gq, gk};
  for (int i = 0; i < 2; ++i) {
    if (!g[i]) continue;
    p.g[i] = g[i]->data;
    p.g_b[i] = g[i]->stride_b;
    p.g_h[i] = g[i]->stride_h;
    p.g_s[i] = g[i]->stride_s;
  }
  const bool with_dw = dwq || dwk;
  p.dw_part = with_dw ? scratch : nullptr;
  const int blocks = int(std::min<long>((p.units + HN_GROUPS - 1) / HN_GROUPS, with_dw ? HN_BWD_BLOCKS : 148 * 32));
  auto go = [&](auto kern, auto sum) {
    kern<<<blocks, HN_GROUPS * 16, 0, st>>>(p);
    if (with_dw) sum<<<8, 1024, 0, st>>>(scratch, blocks, dwq, dwk, c.weight_fp32, p.status);
  };
  if (c.dtype == LVX_BF16) go(head_norm_kernel<0, true>, head_norm_dw_kernel<0>);
  else if (c.dtype == LVX_FP16) go(head_norm_kernel<1, true>, head_norm_dw_kernel<1>);
  else go(head_norm_kernel<2, true>, head_norm_dw_kernel<2>);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "head_norm_bwd launch");
}

}  // namespace lvx
