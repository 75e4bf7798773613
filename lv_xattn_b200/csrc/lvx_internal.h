// Host-side declarations shared by the translation units of liblvx.so.
#pragma once
#include <cuda_runtime.h>
#include <cuda.h>
#include <stdint.h>
#include <stddef.h>
#include "../../include/lvx.h"

namespace lvx {

// printf-style setter of the thread-local error text returned by lvx_last_error(); returns `code`.
int fail(int code, const char* fmt, ...);
// Maps a cudaError_t to the ABI's positive return code and records its text.
int cuda_fail(cudaError_t e, const char* what);

// Encodes a 3-D tiled tensor map with 128-byte swizzle. dims/strides are given innermost first;
// stride[0] is implied by the element size. box2 is always 1. Returns an ABI status code.
int make_tmap_3d(CUtensorMap* out, int dtype, const void* base, uint64_t dim0, uint64_t dim1, uint64_t dim2,
                 uint64_t stride1_bytes, uint64_t stride2_bytes, uint32_t box0, uint32_t box1,
                 bool swizzle_atom_32b = false);

// Device status word of the current device (nullptr if it cannot be resolved), and the ABI's argument checks.
int* device_status_ptr();
int validate_shape(const lvx_shape* s, const char* who);
int validate_arch();

inline int q_blocks_of(const lvx_shape& s) { return s.q_blocks > 1 ? s.q_blocks : 1; }
inline int elt_size(int dtype) { return dtype == LVX_FP32 ? 4 : 2; }

// Dense additive bias on the scores: value for (query block, batch, query head, query row, key) at
// base[blk*s_blk + b*s_b + h*s_h + i*s_q + j*s_kv] (strides in floats; 0 broadcasts). nullptr = no bias.
struct BiasView {
  const float* base;
  long long s_blk, s_b, s_h, s_q, s_kv;
  int sq, g;          // query rows per head, query heads per KV head (to unpack a packed row)
};
inline BiasView make_bias(const lvx_shape& s, const lvx_bias* b) {
  BiasView v;
  v.base = b ? b->bias : nullptr;
  v.s_blk = b ? b->stride_block : 0;
  v.s_b = b ? b->stride_b : 0;
  v.s_h = b ? b->stride_h : 0;
  v.s_q = b ? b->stride_q : 0;
  v.s_kv = b ? b->stride_kv : 0;
  v.sq = s.Sq;
  v.g = s.Hq / s.Hkv;
  return v;
}

// Split-KV plan of the forward block; shared by the kernel launcher, the combine kernel and
// lvx_query_workspace so that all three agree on the workspace layout.
struct FwdPlan {
  int rows;          // g * Sq : packed query rows per (batch, kv head)
  int m_blocks;      // CTAs along the packed rows (256 rows each)
  int kv_tiles;      // ceil(Skv / 128)
  int nsplit;        // CTAs along the K/V range
  int tiles_per_split;
  size_t o_part_bytes;   // fp32 [B*Hkv][nsplit][rows][D]
  size_t ml_part_bytes;  // fp32 [B*Hkv][nsplit][rows][2]
};
FwdPlan plan_fwd(const lvx_shape& s);

// Launchers (one per .cu). `status` is the device status word.
int launch_fwd_block(const lvx_shape& s, const FwdPlan& p, const void* q, const void* k, const void* v,
                     const int32_t* kv_valid_len, float sm_scale, float* o_part, float* ml_part, int* status,
                     cudaStream_t st, const lvx_block_wait* bw = nullptr, const lvx_bias* bias = nullptr);
// The forward block for few packed query rows (fwd_rows_sm100.cu); same plan and partials layout.
constexpr int kFewRows = 64;
int launch_fwd_rows(const lvx_shape& s, const FwdPlan& p, const void* q, const void* k, const void* v,
                    const int32_t* kv_valid_len, float sm_scale, float* o_part, float* ml_part, int* status,
                    cudaStream_t st);
// What the rounding of O to 16 bits dropped, of the rows at the first kLowRows positions of a text: [B * Hq][kLowRows][128], by
// position, in O's type. The backward makes delta from both parts there: such rows see few keys, and in dS the error of a rounded
// O is then as large as the rounding of dS itself (texts of 16 tokens, bf16: gradients off by 2.80e-3 -> 2.41e-3, of 300
// 2.49e-3 -> 2.38e-3). Rows behind that many positions hardly change it, and the parts of all rows cost 4 to 6 % of a training pass.
// With fewer rows a head than kLowRows, [B * Hq][rows][128], they lie from the entry's first position on: a batch of 16-token texts
// keeps as much as its O that way, and sixteen times as much by position.
constexpr int kLowRows = LVX_LOW_ROWS;
struct LowRows {
  uint16_t* data;                // nullptr: not kept
  const int32_t* kv_valid_len;
  int start, skv, sq, heads;     // start: query_start; heads: Hq
  int rows;                      // of a head in `data`
  // where the row at position `pos` lies in its head's, if the entry's first query is at `first`; -1: not kept
  static __device__ __forceinline__ int place(int pos, int first, int rows) {
    const int at = rows < kLowRows ? pos - max(0, first) : pos;
    return pos >= 0 && pos < kLowRows && at < rows ? at : -1;
  }
  // the part of row `tok` of (batch entry, head) `bh`, or nullptr
  __device__ __forceinline__ uint16_t* row(int bh, int tok) const {
    if (data == nullptr) return nullptr;
    const int valid = kv_valid_len ? min(skv, max(0, kv_valid_len[bh / heads])) : skv;
    const int first = start >= 0 ? start : valid - sq, at = place(first + tok, first, rows);
    return at >= 0 ? data + (size_t(bh) * rows + at) * 128 : nullptr;
  }
};
inline int low_rows_of(const lvx_window& w) { return w.low_rows > 0 ? w.low_rows : kLowRows; }
inline LowRows low_rows(const lvx_shape& s, const lvx_window& w, void* o_low, const int32_t* kv_valid_len) {
  return {static_cast<uint16_t*>(o_low), kv_valid_len, w.query_start, s.Skv, s.Sq, s.Hq, low_rows_of(w)};
}
// How a kernel stands to the one before it in the stream: it starts when that one is complete; or comes onto the SMs while that
// one, of the same call, still runs, and waits for it itself, at its start or, needing none of its results, at its end
// (sm100_prims.cuh). The kernels of own keys and of a shared prefix stand beside each other: one token of 32 requests with 2,048
// own keys behind 102,464 134 -> 128 us, 77 tokens of eight requests behind 25,616 274 -> 270, 333 of four even.
enum Order { ORDER_AFTER, ORDER_OVERLAP, ORDER_BESIDE };
template <class... P, class... A>
inline cudaError_t launch_kernel(Order order, void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  c.attrs = &attr;
  c.numAttrs = order == ORDER_AFTER ? 0 : 1;
  return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}
// Windowed causal attention (window.cuh): few packed rows (partials; or O and lse, where plan_window has a slab's keys shared out over
// a cluster of at most kRowCluster CTAs), and the kernel for more (partials, or O and lse).
constexpr int kRowCluster = 8;
int launch_window_rows(const lvx_shape& s, const lvx_window& w, const FwdPlan& p, const lvx_view& q, const lvx_view& k,
                       const lvx_view& v, const int32_t* kv_valid_len, float sm_scale, float* o_part, float* ml_part, void* o,
                       void* o_low, float* lse, int* status, Order order, cudaStream_t st);
int launch_window_fwd(const lvx_shape& s, const lvx_window& w, const FwdPlan& p, const lvx_view& q, const lvx_view& k,
                      const lvx_view& v, const int32_t* kv_valid_len, float sm_scale, float* o_part, float* ml_part, void* o,
                      void* o_low, float* lse, int* status, Order order, cudaStream_t st);
// Its backward for 16-bit types: dq_acc (window_dq_floats of them, zeroed) is in tile order, launch_window_dq rounds it and
// adds up the parts (window_sink_floats of them) of the sinks' dK and dV.
size_t window_dq_floats(const lvx_shape& s);
size_t window_sink_floats(const lvx_shape& s, const lvx_window& w);
int launch_window_bwd(const lvx_shape& s, const lvx_window& w, const lvx_view& q, const lvx_view& d_o, const lvx_view& k,
                      const lvx_view& v, const float* lse, const float* delta, const int32_t* kv_valid_len, float sm_scale,
                      float* dq_acc, float* parts, void* dk, void* dv, int* status, Order order, cudaStream_t st);
int launch_window_dq(const lvx_shape& s, const lvx_window& w, const float* acc, const float* parts, void* dq, void* dk, void* dv,
                     const int* status, cudaStream_t st);
// Around the windowed kernels for a batch that shares prefixes (shared_prefix.cu).
int launch_pack_rows(const lvx_shape& s, int prefixes, const lvx_view& q, const void* d_o, const float* lse, const float* delta,
                     void* q_out, void* do_out, float* lse_out, float* delta_out, Order order, cudaStream_t st);
int launch_shared_combine(const lvx_shape& s, int prefixes, bool by_head, const float* o_pre, const float* ml_pre, int ns_pre, const float* o_own,
                          const float* ml_own, int ns_own, void* o, float* lse, cudaStream_t st);
int launch_shared_dq(const lvx_shape& s, int prefixes, const float* acc_pre, int pre_slab_rows, const float* acc_own, void* dq,
                     cudaStream_t st);
int launch_fwd_combine(const lvx_shape& s, const FwdPlan& p, const float* o_part, const float* ml_part,
                       const float* o_in, const float* lse_in, void* o_out, float* lse_out, int out_is_final,
                       cudaStream_t st, Order order = ORDER_AFTER, const LowRows& low = {});
int launch_bwd_prep(const lvx_shape& s, const void* o, const void* d_o, float* delta, cudaStream_t st, const LowRows& low = {},
                    void* zero = nullptr, size_t zero_bytes = 0);      // memory to be cleared on the way, a multiple of 16 bytes
int launch_bwd_block(const lvx_shape& s, const void* q, const void* d_o, const float* lse, const float* delta,
                     const void* k, const void* v, const int32_t* kv_valid_len, float sm_scale, float* dq_acc,
                     float* dk_acc, float* dv_acc, int accumulate_dkdv, int* status, cudaStream_t st,
                     const lvx_block_wait* bw = nullptr, const lvx_bias* bias = nullptr);
// Limit of the in-kernel waits for a peer's flag, in SM cycles (lvx_p2p_set_timeout).
long long p2p_wait_limit_cycles();
// The general block kernels (general_tf32.cu; same workspace layout and masking rules as the 16-bit path): fp32 (forward)
// and fp32 or fp16 (backward), optional dense additive bias.
int launch_fwd_block_general(const lvx_shape& s, const FwdPlan& p, const void* q, const void* k, const void* v,
                          const int32_t* kv_valid_len, const lvx_bias* bias, float sm_scale, float* o_part,
                          float* ml_part, cudaStream_t st, const lvx_window* win = nullptr);
int launch_bwd_block_general(const lvx_shape& s, const void* q, const void* d_o, const float* lse, const float* delta,
                          const void* k, const void* v, const int32_t* kv_valid_len, const lvx_bias* bias,
                          float sm_scale, float* dq_acc, void* dk_acc, void* dv_acc, int accumulate_dkdv,
                          cudaStream_t st, const lvx_window* win = nullptr);
// K/V projection with fused per-head RMSNorm (kvproj_sm100.cu) and the backward of that norm.
int launch_kv_project(int dtype, const void* x, const void* wk, const void* wv, const void* norm_w, float eps,
                      int batch, int s, int kd, int hkv, void* k_out, void* v_out, float* rstd, int* status,
                      cudaStream_t st);
int launch_knorm_bwd(int dtype, const void* k, const void* dk, const float* rstd, const void* norm_w, void* dkpre,
                     float* dw, long rows, cudaStream_t st);
int launch_kvproj_grad_rows(int dtype, const void* k, const void* dk, const void* dv, const float* rstd, const void* norm_w,
                            void* dk_rows, void* dv_rows, float* dw, int batch, int hkv, int s, cudaStream_t st);
// Head norms and rotary embedding (head_norm.cu).
int launch_head_norm(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, void* q_out, void* k_out, cudaStream_t st);
int launch_head_norm_bwd(const lvx_head_norm& c, const lvx_view* q, const lvx_view* k, const lvx_view* gq, const lvx_view* gk,
                         void* dq, void* dk, float* scratch, void* dwq, void* dwk, cudaStream_t st);
int launch_fwd_merge_parts(const lvx_shape& s, const float* o_parts, const float* lse_parts, int count,
                           size_t stride_o, size_t stride_lse, void* o_out, float* lse_out, cudaStream_t st);
int launch_sum_cast(const float* parts, int count, size_t stride, void* out, int out_dtype, size_t n, cudaStream_t st);
int launch_add_cast(const float* a, const float* b, void* out, int out_dtype, size_t n, cudaStream_t st);
int launch_selftest(int mode, const void* a, const void* b, float* d_out, int* status, cudaStream_t st);

}  // namespace lvx
