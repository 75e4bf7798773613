// The pieces that kernels merging split-KV partials share (elementwise.cu, shared_prefix.cu).
#pragma once
#include "lvx_internal.h"
#include "sm100_prims.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

namespace lvx {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

// While the device status word is set (a bounded wait ran out somewhere) every kernel returns at once, so that
// nothing is computed from buffers an aborted kernel left unwritten.
__device__ __forceinline__ bool poisoned(const int* status) {
  return status != nullptr && *reinterpret_cast<const volatile int*>(status) != 0;
}

template <int OUT>  // 0 bf16, 1 fp16, 2 fp32
__device__ __forceinline__ void store4(void* base, size_t idx4, float4 v) {
  if (OUT == 2) {
    reinterpret_cast<float4*>(base)[idx4] = v;
  } else if (OUT == 0) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    uint2 u;
    u.x = *reinterpret_cast<uint32_t*>(&a);
    u.y = *reinterpret_cast<uint32_t*>(&b);
    reinterpret_cast<uint2*>(base)[idx4] = u;
  } else {
    __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    uint2 u;
    u.x = *reinterpret_cast<uint32_t*>(&a);
    u.y = *reinterpret_cast<uint32_t*>(&b);
    reinterpret_cast<uint2*>(base)[idx4] = u;
  }
}

struct RowAcc {
  float m, l;      // running max (base 2, already scaled) and sum
  float4 v;
};
__device__ __forceinline__ void row_merge(RowAcc& a, const RowAcc& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) {
    a.l += b.l;      // zeros, or the NaN of a side whose scores all are (row_four)
    return;
  }
  const float wa = exp2f(a.m - m), wb = exp2f(b.m - m);      // an empty side (max -inf) gets weight 0
  a.m = m;
  a.l = a.l * wa + b.l * wb;
  a.v.x = a.v.x * wa + b.v.x * wb;
  a.v.y = a.v.y * wa + b.v.y * wb;
  a.v.z = a.v.z * wa + b.v.z * wb;
  a.v.w = a.v.w * wa + b.v.w * wb;
}

// Four splits of a row from s0 on (those below nsplit), added to `a`. The maxima ignore NaN, so that a split whose scores all are
// NaN has the maximum of an empty one, -inf, and a sum of NaN; with `keep_nan` the row is NaN then, without it the split counts as empty.
__device__ __forceinline__ void row_four(RowAcc& a, const float* __restrict__ o_part, const float* __restrict__ ml_part, size_t slab,
                                         int nsplit, int rows_per_slab, int r, int s0, int lane, bool keep_nan) {
  float2 ml[4];
  float4 v[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int s = min(s0 + u, nsplit - 1);
    const size_t prow = (slab * nsplit + s) * rows_per_slab + r;
    ml[u] = *reinterpret_cast<const float2*>(ml_part + prow * 2);
    v[u] = reinterpret_cast<const float4*>(o_part + prow * 128)[lane];
    if (s0 + u >= nsplit) ml[u] = make_float2(-INFINITY, 0.f);
  }
  if (keep_nan) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (ml[u].x == -INFINITY) a.l += ml[u].y;
  }
  const float m = fmaxf(fmaxf(a.m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
  if (m == -INFINITY) return;
  const float wa = exp2f(a.m - m);
  a.m = m;
  a.l *= wa;
  a.v.x *= wa; a.v.y *= wa; a.v.z *= wa; a.v.w *= wa;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (ml[u].x == -INFINITY) continue;
    const float w = exp2f(ml[u].x - m);
    a.l += ml[u].y * w;
    a.v.x += v[u].x * w;
    a.v.y += v[u].y * w;
    a.v.z += v[u].z * w;
    a.v.w += v[u].w * w;
  }
}

}  // namespace lvx
