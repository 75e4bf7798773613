// RMSNorm of every query and key head and the rotary embedding, in one pass, from the projections' layout (any strides,
// usually [B, S, H, 128]) to the attention kernels' [B, H, S, 128]; and its backward.
//
//   forward   r = rsqrt(mean_d(x^2) + eps), y = x r w;   out_d = y_d cos_d - y_{d+64} sin_d,
//             out_{d+64} = y_{d+64} cos_{d+64} + y_d sin_{d+64}   (d < 64)
//   backward  dy = the rotation's transpose of the gradient; xh = x r;
//             dx = r (w dy - xh mean_d(w dy xh)),   dw = sum over rows of dy xh
// All of it in fp32, rounded once when it is stored. r is computed again in the backward: x is read there anyway.
//
// Bound by memory (a row of 128 values in and out, two in and one out in the backward), and close behind it by the issue of
// instructions: values go through the packed fp32 unit two at a time, the weight is multiplied into cos and sin once for all
// heads of a unit, and index arithmetic is 32 bits wide. Sixteen lanes work on a row; a lane holds d = 4l..4l+3 and the same of
// the other half, so that the rotation needs no exchange between lanes. A lane group takes a few heads of one token (a unit):
// its rows are in flight together, and the token's cos and sin, which are as wide as two rows in fp32, are fetched once for
// them. The units of a block are neighbours, mostly of one token, so the tables come from L1.
// Measured, bf16, 2 x 4,096 tokens of 32 + 8 heads (176 and 260 MB): forward 50 -> 38 us, backward 115 -> 68 us against one
// value an instruction and 64-bit divisions. Registers are what decides: four heads a unit and two blocks an SM in the
// backward 68 us (three blocks, which spill: 79 with two heads, 113 with four; one block 108), eight lanes a row 82; forward
// 38 us with four heads and four blocks (eight heads and three blocks 35, but a call of four tokens then takes 4.3 us instead of
// 3.3, on fewer SMs; five blocks, which spill, 52). A block works on queries or on keys; dw is kept in registers over its walk
// through the units, summed per block and then by a second kernel in a fixed order: atomics on its 128 addresses would cost
// time, and another result every time.
#include "lvx_internal.h"
#include "sm100_prims.cuh"
#include <algorithm>

namespace lvx {

constexpr int HN_LANES = 16;                    // lanes that work on a row
constexpr int HN_GROUPS = 256 / HN_LANES;       // lane groups of a block
constexpr int HN_V = 64 / HN_LANES;             // values of each half that a lane holds
constexpr int HN_P = HN_V / 2;                  // in pairs
constexpr int HN_BWD_BLOCKS = 148 * 8;
static_assert(HN_BWD_BLOCKS * 128 * sizeof(float) == LVX_HEAD_NORM_SCRATCH, "the header names the scratch's size");
constexpr int hn_unit(int t) { return t == 2 ? 2 : 4; }      // heads of a unit

struct HeadNormParams {
  int S;
  int blocks_q;                     // blocks that work on queries; the others on keys
  int heads[2], chunks[2];          // [0] queries, [1] keys; chunks: units of a token
  unsigned units[2];                // B * S * chunks
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
  float* dw_part;                   // backward: [blocks][128], nullptr: no weight wants its gradient
  const int* status;
};

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }

// A lane's share of half a row, of either type, as it lies in memory, and as pairs of floats.
template <int T>      // 0 bf16, 1 fp16, 2 fp32
struct RawHalf {
  static constexpr int WORDS = HN_V * (T == 2 ? 4 : 2) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const void* base, long long at) {
    const char* p = static_cast<const char*>(base) + at * (T == 2 ? 4 : 2);
    if constexpr (WORDS == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void get(uint64_t (&f)[HN_P]) const {
#pragma unroll
    for (int i = 0; i < HN_P; ++i) {
      if constexpr (T == 2) {
        f[i] = f32x2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      } else {
        const float2 t = unpack16x2<T == 0>(w[i]);
        f[i] = f32x2(t.x, t.y);
      }
    }
  }
};
template <int T>
__device__ __forceinline__ void hn_load_either(uint64_t (&f)[HN_P], const void* base, long long at, int fp32) {
  if (T == 2 || fp32) {
    RawHalf<2> r;
    r.load(base, at);
    r.get(f);
  } else {
    RawHalf<T> r;
    r.load(base, at);
    r.get(f);
  }
}
template <int T>
__device__ __forceinline__ void hn_store(void* base, long long at, const uint64_t (&f)[HN_P]) {
  constexpr int WORDS = RawHalf<T>::WORDS;
  uint32_t w[WORDS];
#pragma unroll
  for (int i = 0; i < HN_P; ++i) {
    float a, b;
    f32x2_get(f[i], a, b);
    if constexpr (T == 2) {
      w[2 * i] = __float_as_uint(a);
      w[2 * i + 1] = __float_as_uint(b);
    } else {
      w[i] = T == 0 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
    }
  }
  char* p = static_cast<char*>(base) + at * (T == 2 ? 4 : 2);
  if constexpr (WORDS == 2) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}
__device__ __forceinline__ float hn_add(uint64_t v) {
  float a, b;
  f32x2_get(v, a, b);
  return a + b;
}
// sum over the lanes of a group
__device__ __forceinline__ float hn_sum(float v) {
#pragma unroll
  for (int off = HN_LANES / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

template <int T, bool BWD>
__global__ void __launch_bounds__(256, BWD ? 2 : 4)
head_norm_kernel(const HeadNormParams p) {
  constexpr int U = hn_unit(T), PER = 32 / HN_LANES;      // lane groups of a warp
  __shared__ float s_dw[BWD ? HN_GROUPS : 1][BWD ? 132 : 1];
  int bad = 0;
  if (p.status) bad = *reinterpret_cast<const volatile int*>(p.status);
  const int group = threadIdx.x / HN_LANES, d = (threadIdx.x % HN_LANES) * HN_V;
  const int which = int(blockIdx.x) >= p.blocks_q;
  const unsigned block = which ? blockIdx.x - p.blocks_q : blockIdx.x, blocks = which ? gridDim.x - p.blocks_q : p.blocks_q;
  const unsigned units = p.units[which], chunks = p.chunks[which];
  const int heads = p.heads[which];
  const void* ww = p.w[which];
  const bool norm = ww != nullptr, rope = p.cos != nullptr;
  uint64_t dwa[HN_P], dwb[HN_P];
#pragma unroll
  for (int i = 0; i < HN_P; ++i) dwa[i] = dwb[i] = 0ull;
  // The lane groups of a warp walk together (their sums are exchanged under the whole warp's mask): the last unit may be
  // done more than once, by groups that then store nothing.
  for (unsigned u0 = block * HN_GROUPS + (group & ~(PER - 1)); u0 < units; u0 += blocks * HN_GROUPS) {
    const unsigned unit = min(u0 + (group & (PER - 1)), units - 1);
    const bool mine = u0 + (group & (PER - 1)) < units && !bad;
    const unsigned token = unit / chunks, b = token / unsigned(p.S);
    const int h0 = int(unit - token * chunks) * U, s = int(token - b * unsigned(p.S));
    RawHalf<T> xa[U], xb[U], ga[BWD ? U : 1], gb[BWD ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = min(h0 + u, heads - 1);
      if (!BWD || norm) {
        const long long at = b * p.x_b[which] + h * p.x_h[which] + s * p.x_s[which] + d;
        xa[u].load(p.x[which], at);
        xb[u].load(p.x[which], at + 64);
      }
      if constexpr (BWD) {
        const long long at = b * p.g_b[which] + h * p.g_h[which] + s * p.g_s[which] + d;
        ga[u].load(p.g[which], at);
        gb[u].load(p.g[which], at + 64);
      }
    }
    uint64_t ca[HN_P], cb[HN_P], sa[HN_P], sb[HN_P], wa[HN_P], wb[HN_P];
    if (rope) {
      const long long at = b * p.t_b + s * p.t_s + d;
      hn_load_either<T>(ca, p.cos, at, p.table_fp32);
      hn_load_either<T>(cb, p.cos, at + 64, p.table_fp32);
      hn_load_either<T>(sa, p.sin, at, p.table_fp32);
      hn_load_either<T>(sb, p.sin, at + 64, p.table_fp32);
#pragma unroll
      for (int i = 0; i < HN_P; ++i) sa[i] = neg2(sa[i]);
    }
    if (norm) {
      hn_load_either<T>(wa, ww, d, p.w_fp32);
      hn_load_either<T>(wb, ww, d + 64, p.w_fp32);
    }
    if constexpr (!BWD) {
      if (norm && rope) {
#pragma unroll
        for (int i = 0; i < HN_P; ++i) {
          ca[i] = mul2(ca[i], wa[i]);
          sa[i] = mul2(sa[i], wb[i]);
          cb[i] = mul2(cb[i], wb[i]);
          sb[i] = mul2(sb[i], wa[i]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint64_t a[HN_P], c[HN_P];
        xa[u].get(a);
        xb[u].get(c);
        uint64_t r2 = f32x2(1.f, 1.f);
        if (norm) {
          uint64_t q = mul2(a[0], a[0]);
#pragma unroll
          for (int i = 1; i < HN_P; ++i) q = fma2(a[i], a[i], q);
#pragma unroll
          for (int i = 0; i < HN_P; ++i) q = fma2(c[i], c[i], q);
          const float r = rsqrtf(hn_sum(hn_add(q)) * (1.f / 128.f) + p.eps);
          r2 = f32x2(r, r);
        }
#pragma unroll
        for (int i = 0; i < HN_P; ++i) {
          const uint64_t x = a[i], y = c[i];
          if (rope) {
            a[i] = mul2(fma2(x, ca[i], mul2(y, sa[i])), r2);
            c[i] = mul2(fma2(y, cb[i], mul2(x, sb[i])), r2);
          } else if (norm) {
            a[i] = mul2(mul2(x, wa[i]), r2);
            c[i] = mul2(mul2(y, wb[i]), r2);
          }
        }
        if (mine && h0 + u < heads) {
          const long long at = ((static_cast<long long>(b) * heads + h0 + u) * p.S + s) * 128 + d;
          hn_store<T>(p.out[which], at, a);
          hn_store<T>(p.out[which], at + 64, c);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint64_t ya[HN_P], yb[HN_P];      // dy, then dx
        ga[u].get(ya);
        gb[u].get(yb);
        if (rope) {
#pragma unroll
          for (int i = 0; i < HN_P; ++i) {
            const uint64_t e = ya[i], f = yb[i];
            ya[i] = fma2(e, ca[i], mul2(f, sb[i]));
            yb[i] = fma2(f, cb[i], mul2(e, sa[i]));
          }
        }
        if (norm) {
          uint64_t a[HN_P], c[HN_P];
          xa[u].get(a);
          xb[u].get(c);
          uint64_t q = 0ull, t = 0ull;
#pragma unroll
          for (int i = 0; i < HN_P; ++i) {
            q = fma2(c[i], c[i], fma2(a[i], a[i], q));
            t = fma2(c[i], mul2(yb[i], wb[i]), fma2(a[i], mul2(ya[i], wa[i]), t));
          }
          const float r = rsqrtf(hn_sum(hn_add(q)) * (1.f / 128.f) + p.eps);
          const float mean = hn_sum(hn_add(t)) * r * (1.f / 128.f);
          const uint64_t r2 = f32x2(r, r), nm = f32x2(-mean * r, -mean * r);
          const bool add = mine && h0 + u < heads;
#pragma unroll
          for (int i = 0; i < HN_P; ++i) {
            const uint64_t xha = mul2(a[i], r2), xhb = mul2(c[i], r2);
            if (add) {
              dwa[i] = fma2(ya[i], xha, dwa[i]);
              dwb[i] = fma2(yb[i], xhb, dwb[i]);
            }
            ya[i] = fma2(xha, nm, mul2(mul2(ya[i], wa[i]), r2));
            yb[i] = fma2(xhb, nm, mul2(mul2(yb[i], wb[i]), r2));
          }
        }
        if (mine && p.out[which] != nullptr && h0 + u < heads) {
          const long long at = ((static_cast<long long>(b) * p.S + s) * heads + h0 + u) * 128 + d;
          hn_store<T>(p.out[which], at, ya);
          hn_store<T>(p.out[which], at + 64, yb);
        }
      }
    }
  }
  if (bad && (threadIdx.x & 31) == 0) publish_status(p.status);
  if constexpr (BWD) {
    if (p.dw_part == nullptr || __syncthreads_or(bad)) return;
#pragma unroll
    for (int i = 0; i < HN_P; ++i) {
      f32x2_get(dwa[i], s_dw[group][d + 2 * i], s_dw[group][d + 2 * i + 1]);
      f32x2_get(dwb[i], s_dw[group][d + 64 + 2 * i], s_dw[group][d + 64 + 2 * i + 1]);
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < HN_GROUPS; ++k) a += s_dw[k][threadIdx.x];
      p.dw_part[size_t(blockIdx.x) * 128 + threadIdx.x] = a;
    }
  }
}

// dw[d] = sum over blocks of dw_part[block][d], in a fixed order: a block of this kernel takes 32 columns of the queries' or the
// keys' weight, with 32 slices of the blocks each.
template <int T>
__global__ void __launch_bounds__(1024)
head_norm_dw_kernel(const float* __restrict__ part, int blocks_q, int blocks, void* dwq, void* dwk, int w_fp32, const int* status) {
  if (status && __syncthreads_or(*reinterpret_cast<const volatile int*>(status) != 0)) {
    if ((threadIdx.x & 31) == 0) publish_status(status);
    return;
  }
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, which = blockIdx.x >> 2, col0 = (blockIdx.x & 3) * 32;
  void* dst = which ? dwk : dwq;
  if (dst == nullptr) return;
  const int first = which ? blocks_q : 0, end = which ? blocks : blocks_q;
  float a = 0.f;
  for (int k = first + slice; k < end; k += 32) a += part[size_t(k) * 128 + col0 + lane];
  s[slice][lane] = a;
  __syncthreads();
  a = s[lane][slice];           // lane = slice, warp = column
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
  if (lane == 0) {
    if (T == 2 || w_fp32) static_cast<float*>(dst)[col0 + slice] = a;
    else static_cast<uint16_t*>(dst)[col0 + slice] = uint16_t(T == 0 ? pack_bf16x2(a, 0.f) : pack_f16x2(a, 0.f));
  }
}

// `most`: blocks at most, 0: one unit a lane group. Returns the number of blocks.
static int head_norm_params(HeadNormParams& p, const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, int unit, long most) {
  p.S = c.S;
  const lvx_view* v[2] = {q, k};
  const int heads[2] = {q ? c.Hq : 0, k ? c.Hkv : 0};
  long blocks[2];
  for (int i = 0; i < 2; ++i) {
    p.heads[i] = heads[i];
    p.chunks[i] = (heads[i] + unit - 1) / unit;
    p.units[i] = unsigned(long(c.B) * c.S * p.chunks[i]);
    blocks[i] = (long(p.units[i]) + HN_GROUPS - 1) / HN_GROUPS;
    if (!v[i]) continue;
    p.x[i] = v[i]->data;
    p.x_b[i] = v[i]->stride_b;
    p.x_h[i] = v[i]->stride_h;
    p.x_s[i] = v[i]->stride_s;
  }
  if (most > 0 && blocks[0] + blocks[1] > most) {      // shared out in proportion, one at least for who has units
    long bq = most * blocks[0] / (blocks[0] + blocks[1]);
    bq = blocks[0] == 0 ? 0 : blocks[1] == 0 ? most : std::min(std::max(bq, 1l), most - 1);
    blocks[1] = most - bq;
    blocks[0] = bq;
  }
  p.blocks_q = int(blocks[0]);
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
  return int(blocks[0] + blocks[1]);
}

int launch_head_norm(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, void* q_out, void* k_out, cudaStream_t st) {
  HeadNormParams p{};
  const int blocks = head_norm_params(p, c, q, k, hn_unit(c.dtype), 0);
  p.out[0] = q_out;
  p.out[1] = k_out;
  if (c.dtype == LVX_BF16) head_norm_kernel<0, false><<<blocks, 256, 0, st>>>(p);
  else if (c.dtype == LVX_FP16) head_norm_kernel<1, false><<<blocks, 256, 0, st>>>(p);
  else head_norm_kernel<2, false><<<blocks, 256, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "head_norm_kernel launch");
}

int launch_head_norm_bwd(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, const lvx_view* gq, const lvx_view* gk,
                         void* dq, void* dk, float* scratch, void* dwq, void* dwk, cudaStream_t st) {
  const bool with_dw = dwq || dwk;
  HeadNormParams p{};
  const int blocks = head_norm_params(p, c, q, k, hn_unit(c.dtype), with_dw ? HN_BWD_BLOCKS : 0);
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
  p.dw_part = with_dw ? scratch : nullptr;
  auto go = [&](auto kern, auto sum) {
    kern<<<blocks, 256, 0, st>>>(p);
    if (with_dw) sum<<<8, 1024, 0, st>>>(scratch, p.blocks_q, blocks, dwq, dwk, c.weight_fp32, p.status);
  };
  if (c.dtype == LVX_BF16) go(head_norm_kernel<0, true>, head_norm_dw_kernel<0>);
  else if (c.dtype == LVX_FP16) go(head_norm_kernel<1, true>, head_norm_dw_kernel<1>);
  else go(head_norm_kernel<2, true>, head_norm_dw_kernel<2>);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LVX_OK : cuda_fail(e, "head_norm_bwd launch");
}

}  // namespace lvx
