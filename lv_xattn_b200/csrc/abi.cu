// extern "C" surface of liblvx.so (see include/lvx.h): argument validation, error text,
// tensor-map encoding through the driver entry point, and the device status word.
#include "lvx_internal.h"
#include "window.cuh"
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

namespace lvx {

static thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int cuda_fail(cudaError_t e, const char* what) {
  snprintf(g_err, sizeof(g_err), "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
  return static_cast<int>(e) > 0 ? static_cast<int>(e) : 1;
}

// Device status word: one per device that loads the library, written by bounded waits that ran out. Words 2-3 hold the
// address of the host's copy (publish_status in elementwise.cu), once there is one.
__device__ __align__(16) int g_status_word[4];

static int* status_ptr() {
  static int* ptrs[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!ptrs[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_status_word) != cudaSuccess) return nullptr;
    ptrs[dev] = static_cast<int*>(p);
  }
  return ptrs[dev];
}

// The host's copy of the current device's status word: mapped pinned memory, set up by the first call that asks for it
// and kept for the process. nullptr while `st` is being captured and there is none yet (its set-up is not capturable).
static int* g_host_status[64];
static int* host_status_word(cudaStream_t st) {
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (g_host_status[dev]) return g_host_status[dev];
  int* sp = status_ptr();
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  // what fails here must not show up as the error of a later launch: the host word is a convenience
  if (!sp || cudaStreamIsCapturing(st, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    (void)cudaGetLastError();
    return nullptr;
  }
  void *h = nullptr, *d = nullptr;
  if (cudaHostAlloc(&h, 64, cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  *static_cast<volatile int*>(h) = 0;
  if (cudaHostGetDevicePointer(&d, h, 0) != cudaSuccess ||
      cudaMemcpy(sp + 2, &d, sizeof(d), cudaMemcpyHostToDevice) != cudaSuccess) {
    cudaFreeHost(h);
    (void)cudaGetLastError();
    return nullptr;
  }
  g_host_status[dev] = static_cast<int*>(h);
  return g_host_status[dev];
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

int make_tmap_3d(CUtensorMap* out, int dtype, const void* base, uint64_t dim0, uint64_t dim1, uint64_t dim2,
                 uint64_t stride1_bytes, uint64_t stride2_bytes, uint32_t box0, uint32_t box1, bool swizzle_atom_32b) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(LVX_ERR_DRIVER, "cuTensorMapEncodeTiled could not be resolved");
  CUtensorMapDataType dt = dtype == LVX_BF16   ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                           : dtype == LVX_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  if ((reinterpret_cast<uintptr_t>(base) & 15u) != 0)
    return fail(LVX_ERR_ALIGN, "tensor base %p is not 16-byte aligned", base);
  if (box0 * elt_size(dtype) != 128) return fail(LVX_ERR_SHAPE, "tensor-map box must be 128 bytes wide");
  cuuint64_t dims[3] = {dim0, dim1, dim2 ? dim2 : 1};
  cuuint64_t strides[2] = {stride1_bytes, stride2_bytes};
  cuuint32_t box[3] = {box0, box1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(out, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle_atom_32b ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(LVX_ERR_SHAPE, "cuTensorMapEncodeTiled failed with CUresult %d (dims %llu,%llu,%llu box %u,%u)",
                int(r), (unsigned long long)dim0, (unsigned long long)dim1, (unsigned long long)dim2, box0, box1);
  return LVX_OK;
}

int make_tmap_nd(CUtensorMap* out, int dtype, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                 const uint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(LVX_ERR_DRIVER, "cuTensorMapEncodeTiled could not be resolved");
  cuuint64_t d[5], st[4];
  cuuint32_t b[5], one[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    if (i + 1 < rank) st[i] = strides[i];
  }
  CUresult r = fn(out, dtype == LVX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                  const_cast<void*>(base), d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(LVX_ERR_SHAPE, "cuTensorMapEncodeTiled failed with CUresult %d (rank %d, dims %llu,%llu,%llu)", int(r), rank,
                (unsigned long long)dims[0], (unsigned long long)dims[1], (unsigned long long)dims[2]);
  return LVX_OK;
}

static int check_arch() {
  static int cached[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev >= 0 && dev < 64 && cached[dev] == 1) return LVX_OK;
  int major = 0;
  e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
  if (major != 10) return fail(LVX_ERR_ARCH, "device %d has compute capability %d.x; this library is sm_100a only", dev, major);
  if (dev >= 0 && dev < 64) cached[dev] = 1;
  return LVX_OK;
}

static int check_shape(const lvx_shape* s, const char* who) {
  if (!s) return fail(LVX_ERR_NULL, "%s: shape is NULL", who);
  if (s->D != 128) return fail(LVX_ERR_SHAPE, "%s: head dimension %d unsupported (128 only)", who, s->D);
  if (s->B <= 0 || s->Hq <= 0 || s->Hkv <= 0 || s->Sq <= 0 || s->Skv < 0)
    return fail(LVX_ERR_SHAPE, "%s: non-positive dimension (B=%d Hq=%d Hkv=%d Sq=%d Skv=%d)", who, s->B, s->Hq, s->Hkv,
                s->Sq, s->Skv);
  if (s->Hq % s->Hkv) return fail(LVX_ERR_SHAPE, "%s: Hq=%d is not a multiple of Hkv=%d", who, s->Hq, s->Hkv);
  if (s->dtype != LVX_BF16 && s->dtype != LVX_FP16 && s->dtype != LVX_FP32)
    return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported", who, s->dtype);
  if (s->q_blocks < 0 || s->q_blocks > 4096) return fail(LVX_ERR_SHAPE, "%s: q_blocks %d out of range", who, s->q_blocks);
  if (int64_t(s->Hq / s->Hkv) * s->Sq > (int64_t(1) << 30) ||
      int64_t(s->q_blocks > 1 ? s->q_blocks : 1) * s->B * s->Hkv > 65535)
    return fail(LVX_ERR_SHAPE, "%s: dimension too large", who);
  return LVX_OK;
}

// Non-static doors for the other translation units of the library.
int* device_status_ptr() { return status_ptr(); }
int validate_shape(const lvx_shape* s, const char* who) { return check_shape(s, who); }
int validate_arch() { return check_arch(); }

#define LVX_REQUIRE_PTR(p, who)                                           \
  do {                                                                    \
    if (!(p)) return lvx::fail(LVX_ERR_NULL, "%s: %s is NULL", who, #p);  \
    if (reinterpret_cast<uintptr_t>(p) & 15u)                             \
      return lvx::fail(LVX_ERR_ALIGN, "%s: %s is not 16-byte aligned", who, #p); \
  } while (0)

}  // namespace lvx

using namespace lvx;

extern "C" {

int lvx_version(void) { return LVX_ABI_VERSION; }

const char* lvx_last_error(void) { return g_err; }

int lvx_device_status(void* stream, int* status_out) {
  if (!status_out) return fail(LVX_ERR_NULL, "lvx_device_status: status_out is NULL");
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "lvx_device_status: status word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(status_out, sp, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyAsync(status)");
  e = cudaMemsetAsync(sp, 0, sizeof(int), st);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(status)");
  e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return cuda_fail(e, "cudaStreamSynchronize(status)");
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 && g_host_status[dev])
    *reinterpret_cast<volatile int*>(g_host_status[dev]) = 0;
  return LVX_OK;
}

int lvx_device_status_host(void* stream, const int** host_word) {
  if (!host_word) return fail(LVX_ERR_NULL, "lvx_device_status_host: host_word is NULL");
  *host_word = host_status_word(static_cast<cudaStream_t>(stream));
  return LVX_OK;
}

// Key-padding lengths given by the host, handed to the kernel by value: no copy, no synchronisation, capturable.
struct ValidLens {
  int64_t v[256];
};
__global__ void local_valid_kernel(const __grid_constant__ ValidLens lens, int n, int64_t base, int skv, int32_t* out) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t left = lens.v[i] - base;
  out[i] = int32_t(left < 0 ? 0 : left > skv ? skv : left);
}

int lvx_local_valid(const int64_t* valid_len, int count, int64_t first_key, int skv, int32_t* out, void* stream) {
  const char* who = "lvx_local_valid";
  if (count < 0 || skv < 0) return fail(LVX_ERR_SHAPE, "%s: negative count or skv", who);
  if (count == 0) return LVX_OK;
  if (!valid_len) return fail(LVX_ERR_NULL, "%s: valid_len is NULL", who);
  LVX_REQUIRE_PTR(out, who);
  for (int i0 = 0; i0 < count; i0 += 256) {
    ValidLens lens;
    const int n = count - i0 < 256 ? count - i0 : 256;
    memset(&lens, 0, sizeof(lens));
    memcpy(lens.v, valid_len + i0, size_t(n) * sizeof(int64_t));
    local_valid_kernel<<<1, 256, 0, static_cast<cudaStream_t>(stream)>>>(lens, n, first_key, skv, out + i0);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "local_valid launch");
  }
  return LVX_OK;
}

int lvx_device_status_peek(void* stream, int* host_out) {
  if (!host_out) return fail(LVX_ERR_NULL, "lvx_device_status_peek: host_out is NULL");
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "lvx_device_status_peek: status word unavailable");
  cudaError_t e = cudaMemcpyAsync(host_out, sp, sizeof(int), cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyAsync(status peek)");
  return LVX_OK;
}

int lvx_query_workspace(const lvx_shape* s, size_t* fwd_bytes, size_t* bwd_bytes) {
  int rc = check_shape(s, "lvx_query_workspace");
  if (rc) return rc;
  FwdPlan p = plan_fwd(*s);
  if (fwd_bytes) *fwd_bytes = p.o_part_bytes + p.ml_part_bytes;
  if (bwd_bytes) *bwd_bytes = 0;
  return LVX_OK;
}

static int check_block_wait(const lvx_shape* s, const lvx_block_wait* w, const char* who) {
  if (!w) return LVX_OK;
  if (s->dtype == LVX_FP32) return fail(LVX_ERR_DTYPE, "%s: the fp32 kernels do not take a block wait", who);
  const int qb = s->q_blocks > 1 ? s->q_blocks : 1;
  if (w->first_block < 0 || w->first_block >= qb) return fail(LVX_ERR_SHAPE, "%s: first_block %d outside [0, %d)", who, w->first_block, qb);
  if (w->my_flags) {
    if (w->slot < 0 || w->slot >= LVX_P2P_SLOTS) return fail(LVX_ERR_SHAPE, "%s: slot %d out of range", who, w->slot);
    if (qb > LVX_MAX_PEERS) return fail(LVX_ERR_SHAPE, "%s: %d blocks but only %d flag words per slot", who, qb, LVX_MAX_PEERS);
    if (reinterpret_cast<uintptr_t>(w->my_flags) & 3u) return fail(LVX_ERR_ALIGN, "%s: my_flags is misaligned", who);
  }
  return LVX_OK;
}

int lvx_fwd_block(const lvx_shape* s, const void* q, const void* k, const void* v, const int32_t* kv_valid_len,
                  float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  return lvx_fwd_block_gathered(s, q, k, v, kv_valid_len, sm_scale, workspace, workspace_bytes, nullptr, stream);
}

int lvx_fwd_block_gathered(const lvx_shape* s, const void* q, const void* k, const void* v, const int32_t* kv_valid_len,
                           float sm_scale, void* workspace, size_t workspace_bytes, const lvx_block_wait* wait,
                           void* stream) {
  const char* who = wait ? "lvx_fwd_block_gathered" : "lvx_fwd_block";
  int rc = check_shape(s, who);
  if (!rc) rc = check_block_wait(s, wait, who);
  if (rc) return rc;
  if ((rc = check_arch())) return rc;
  LVX_REQUIRE_PTR(q, who);
  LVX_REQUIRE_PTR(workspace, who);
  if (s->Skv > 0) {
    LVX_REQUIRE_PTR(k, who);
    LVX_REQUIRE_PTR(v, who);
  }
  FwdPlan p = plan_fwd(*s);
  if (workspace_bytes < p.o_part_bytes + p.ml_part_bytes)
    return fail(LVX_ERR_WORKSPACE, "%s: workspace has %zu bytes, %zu needed", who, workspace_bytes,
                p.o_part_bytes + p.ml_part_bytes);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_part_bytes);
  return launch_fwd_block(*s, p, q, k, v, kv_valid_len, sm_scale, o_part, ml_part, sp,
                          static_cast<cudaStream_t>(stream), wait);
}

int lvx_fwd_combine_merge(const lvx_shape* s, const void* workspace, const float* o_in, const float* lse_in,
                          void* o_out, float* lse_out, int out_is_final, void* stream) {
  const char* who = "lvx_fwd_combine_merge";
  int rc = check_shape(s, who);
  if (rc) return rc;
  LVX_REQUIRE_PTR(workspace, who);
  LVX_REQUIRE_PTR(o_out, who);
  LVX_REQUIRE_PTR(lse_out, who);
  if ((o_in == nullptr) != (lse_in == nullptr))
    return fail(LVX_ERR_NULL, "%s: o_in and lse_in must both be given or both be NULL", who);
  FwdPlan p = plan_fwd(*s);
  const float* o_part = static_cast<const float*>(workspace);
  const float* ml_part = reinterpret_cast<const float*>(static_cast<const char*>(workspace) + p.o_part_bytes);
  return launch_fwd_combine(*s, p, o_part, ml_part, o_in, lse_in, o_out, lse_out, out_is_final,
                            static_cast<cudaStream_t>(stream));
}

int lvx_bwd_prep(const lvx_shape* s, const void* o, const void* d_o, float* delta, void* stream) {
  const char* who = "lvx_bwd_prep";
  int rc = check_shape(s, who);
  if (rc) return rc;
  LVX_REQUIRE_PTR(o, who);
  LVX_REQUIRE_PTR(d_o, who);
  LVX_REQUIRE_PTR(delta, who);
  return launch_bwd_prep(*s, o, d_o, delta, static_cast<cudaStream_t>(stream));
}

int lvx_bwd_block(const lvx_shape* s, const void* q, const void* d_o, const float* lse, const float* delta,
                  const void* k, const void* v, const int32_t* kv_valid_len, float sm_scale, float* dq_acc,
                  float* dk_acc, float* dv_acc, int accumulate_dkdv, void* workspace, size_t workspace_bytes,
                  void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  return lvx_bwd_block_gathered(s, q, d_o, lse, delta, k, v, kv_valid_len, sm_scale, dq_acc, dk_acc, dv_acc,
                                accumulate_dkdv, nullptr, stream);
}

int lvx_bwd_block_gathered(const lvx_shape* s, const void* q, const void* d_o, const float* lse, const float* delta,
                           const void* k, const void* v, const int32_t* kv_valid_len, float sm_scale, float* dq_acc,
                           float* dk_acc, float* dv_acc, int accumulate_dkdv, const lvx_block_wait* wait, void* stream) {
  const char* who = wait ? "lvx_bwd_block_gathered" : "lvx_bwd_block";
  int rc = check_shape(s, who);
  if (!rc) rc = check_block_wait(s, wait, who);
  if (rc) return rc;
  if ((rc = check_arch())) return rc;
  LVX_REQUIRE_PTR(q, who);
  LVX_REQUIRE_PTR(d_o, who);
  LVX_REQUIRE_PTR(lse, who);
  LVX_REQUIRE_PTR(delta, who);
  LVX_REQUIRE_PTR(dq_acc, who);
  if (s->Skv == 0) return LVX_OK;
  LVX_REQUIRE_PTR(k, who);
  LVX_REQUIRE_PTR(v, who);
  LVX_REQUIRE_PTR(dk_acc, who);
  LVX_REQUIRE_PTR(dv_acc, who);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  return launch_bwd_block(*s, q, d_o, lse, delta, k, v, kv_valid_len, sm_scale, dq_acc, dk_acc, dv_acc,
                          accumulate_dkdv, sp, static_cast<cudaStream_t>(stream), wait);
}

int lvx_fwd_block_bias(const lvx_shape* s, const void* q, const void* k, const void* v, const int32_t* kv_valid_len,
                       const lvx_bias* bias, float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "lvx_fwd_block_bias";
  int rc = check_shape(s, who);
  if (rc) return rc;
  if ((rc = check_arch())) return rc;
  LVX_REQUIRE_PTR(q, who);
  LVX_REQUIRE_PTR(workspace, who);
  if (!bias || !bias->bias) return fail(LVX_ERR_NULL, "%s: bias is NULL (use lvx_fwd_block)", who);
  if (reinterpret_cast<uintptr_t>(bias->bias) & 3u) return fail(LVX_ERR_ALIGN, "%s: bias is not 4-byte aligned", who);
  if (!(sm_scale > 0.f)) return fail(LVX_ERR_SHAPE, "%s: sm_scale must be positive", who);
  if (s->Skv > 0) {
    LVX_REQUIRE_PTR(k, who);
    LVX_REQUIRE_PTR(v, who);
  }
  FwdPlan p = plan_fwd(*s);
  if (workspace_bytes < p.o_part_bytes + p.ml_part_bytes)
    return fail(LVX_ERR_WORKSPACE, "%s: workspace has %zu bytes, %zu needed", who, workspace_bytes,
                p.o_part_bytes + p.ml_part_bytes);
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_part_bytes);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  return launch_fwd_block(*s, p, q, k, v, kv_valid_len, sm_scale, o_part, ml_part, sp, static_cast<cudaStream_t>(stream),
                          nullptr, bias);
}

int lvx_bwd_block_bias(const lvx_shape* s, const void* q, const void* d_o, const float* lse, const float* delta,
                       const void* k, const void* v, const int32_t* kv_valid_len, const lvx_bias* bias, float sm_scale,
                       float* dq_acc, void* dk_acc, void* dv_acc, int accumulate_dkdv, void* stream) {
  const char* who = "lvx_bwd_block_bias";
  int rc = check_shape(s, who);
  if (rc) return rc;
  if ((rc = check_arch())) return rc;
  LVX_REQUIRE_PTR(q, who);
  LVX_REQUIRE_PTR(d_o, who);
  LVX_REQUIRE_PTR(lse, who);
  LVX_REQUIRE_PTR(delta, who);
  LVX_REQUIRE_PTR(dq_acc, who);
  if (!bias || !bias->bias) return fail(LVX_ERR_NULL, "%s: bias is NULL (use lvx_bwd_block)", who);
  if (!(sm_scale > 0.f)) return fail(LVX_ERR_SHAPE, "%s: sm_scale must be positive", who);
  if (accumulate_dkdv < 0 || accumulate_dkdv > 2)
    return fail(LVX_ERR_SHAPE, "%s: accumulate_dkdv must be 0, 1 or 2 (got %d)", who, accumulate_dkdv);
  if (s->Skv == 0) return LVX_OK;
  LVX_REQUIRE_PTR(k, who);
  LVX_REQUIRE_PTR(v, who);
  LVX_REQUIRE_PTR(dk_acc, who);
  LVX_REQUIRE_PTR(dv_acc, who);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  return launch_bwd_block(*s, q, d_o, lse, delta, k, v, kv_valid_len, sm_scale, dq_acc, static_cast<float*>(dk_acc),
                          static_cast<float*>(dv_acc), accumulate_dkdv, sp, static_cast<cudaStream_t>(stream), nullptr, bias);
}

int lvx_attn_forward(const lvx_shape* s, const void* q, const void* k, const void* v, const int32_t* kv_valid_len,
                     const lvx_bias* bias, float sm_scale, void* workspace, size_t workspace_bytes, void* o, float* lse,
                     void* stream) {
  const int rc = bias ? lvx_fwd_block_bias(s, q, k, v, kv_valid_len, bias, sm_scale, workspace, workspace_bytes, stream)
                      : lvx_fwd_block(s, q, k, v, kv_valid_len, sm_scale, workspace, workspace_bytes, stream);
  return rc ? rc : lvx_fwd_combine_merge(s, workspace, nullptr, nullptr, o, lse, 1, stream);
}

int lvx_attn_backward(const lvx_shape* s, const void* d_o, const void* q, const void* k, const void* v, const void* o,
                      const float* lse, const int32_t* kv_valid_len, const lvx_bias* bias, float sm_scale, void* scratch,
                      size_t scratch_bytes, void* dq, void* dk, void* dv, void* stream) {
  const char* who = "lvx_attn_backward";
  int rc = check_shape(s, who);
  if (rc) return rc;
  LVX_REQUIRE_PTR(o, who);
  LVX_REQUIRE_PTR(d_o, who);
  LVX_REQUIRE_PTR(dq, who);
  LVX_REQUIRE_PTR(scratch, who);
  const size_t rows = size_t(q_blocks_of(*s)) * s->B * s->Hq * s->Sq, n_q = rows * 128;
  if (scratch_bytes < n_q * sizeof(float) + rows * sizeof(float))
    return fail(LVX_ERR_WORKSPACE, "%s: scratch has %zu bytes, %zu needed", who, scratch_bytes,
                n_q * sizeof(float) + rows * sizeof(float));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // fp32: dQ is accumulated where it is wanted; otherwise in the scratch, and cast at the end
  const bool direct = s->dtype == LVX_FP32;
  float* dq_acc = direct ? static_cast<float*>(dq) : static_cast<float*>(scratch);
  float* delta = static_cast<float*>(scratch) + n_q;
  if ((rc = launch_bwd_prep(*s, o, d_o, delta, st))) return rc;
  const cudaError_t e = cudaMemsetAsync(dq_acc, 0, n_q * sizeof(float), st);
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(dq)");
  rc = bias ? lvx_bwd_block_bias(s, q, d_o, lse, delta, k, v, kv_valid_len, bias, sm_scale, dq_acc, dk, dv, 2, stream)
            : lvx_bwd_block(s, q, d_o, lse, delta, k, v, kv_valid_len, sm_scale, dq_acc, static_cast<float*>(dk),
                            static_cast<float*>(dv), 2, nullptr, 0, stream);
  if (rc || direct) return rc;
  return launch_add_cast(dq_acc, nullptr, dq, s->dtype, n_q, st);
}

int lvx_kv_project(int dtype, const void* x, const void* wk, const void* wv, const void* norm_w, float eps, int batch,
                   int S, int Kd, int Hkv, void* k_out, void* v_out, float* rstd, void* stream) {
  const char* who = "lvx_kv_project";
  int rc = check_arch();
  if (rc) return rc;
  if (dtype != LVX_BF16 && dtype != LVX_FP16) return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported (bf16 or fp16)", who, dtype);
  if (batch <= 0 || S <= 0 || Kd <= 0 || Hkv <= 0) return fail(LVX_ERR_SHAPE, "%s: non-positive dimension", who);
  if (Kd % 64) return fail(LVX_ERR_SHAPE, "%s: Kd=%d is not a multiple of 64", who, Kd);
  if (Hkv % 2) return fail(LVX_ERR_SHAPE, "%s: Hkv=%d is odd (tiles hold two heads)", who, Hkv);
  if (int64_t(batch) * S > (int64_t(1) << 31) - 512) return fail(LVX_ERR_SHAPE, "%s: batch*S too large", who);
  if (!(eps >= 0.f)) return fail(LVX_ERR_SHAPE, "%s: eps must be non-negative", who);
  LVX_REQUIRE_PTR(x, who);
  LVX_REQUIRE_PTR(wk, who);
  LVX_REQUIRE_PTR(wv, who);
  LVX_REQUIRE_PTR(k_out, who);
  LVX_REQUIRE_PTR(v_out, who);
  if (norm_w && (reinterpret_cast<uintptr_t>(norm_w) & 1u)) return fail(LVX_ERR_ALIGN, "%s: norm_w is misaligned", who);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  return launch_kv_project(dtype, x, wk, wv, norm_w, eps, batch, S, Kd, Hkv, k_out, v_out, rstd, sp,
                           static_cast<cudaStream_t>(stream));
}

int lvx_knorm_bwd(int dtype, const void* k, const void* dk, const float* rstd, const void* norm_w, void* dkpre,
                  float* dw, size_t rows, void* stream) {
  const char* who = "lvx_knorm_bwd";
  if (dtype != LVX_BF16 && dtype != LVX_FP16) return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported (bf16 or fp16)", who, dtype);
  if (rows == 0) return LVX_OK;
  LVX_REQUIRE_PTR(k, who);
  LVX_REQUIRE_PTR(dk, who);
  LVX_REQUIRE_PTR(rstd, who);
  LVX_REQUIRE_PTR(dkpre, who);
  LVX_REQUIRE_PTR(dw, who);
  if (!norm_w || (reinterpret_cast<uintptr_t>(norm_w) & 7u)) return fail(LVX_ERR_ALIGN, "%s: norm_w must be given, 8-byte aligned", who);
  return launch_knorm_bwd(dtype, k, dk, rstd, norm_w, dkpre, dw, long(rows), static_cast<cudaStream_t>(stream));
}

int lvx_kv_project_grad_rows(int dtype, const void* k, const void* dk, const void* dv, const float* rstd,
                             const void* norm_w, void* dk_rows, void* dv_rows, float* dw, int batch, int Hkv, int S,
                             void* stream) {
  const char* who = "lvx_kv_project_grad_rows";
  if (dtype != LVX_BF16 && dtype != LVX_FP16) return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported", who, dtype);
  if (batch < 0 || Hkv <= 0 || S < 0) return fail(LVX_ERR_SHAPE, "%s: negative dimension", who);
  if (batch == 0 || S == 0) return LVX_OK;
  LVX_REQUIRE_PTR(k, who);
  LVX_REQUIRE_PTR(dk, who);
  LVX_REQUIRE_PTR(dv, who);
  LVX_REQUIRE_PTR(rstd, who);
  if (dk_rows) LVX_REQUIRE_PTR(dk_rows, who);
  if (dv_rows) LVX_REQUIRE_PTR(dv_rows, who);
  if (norm_w) {
    if (dw) LVX_REQUIRE_PTR(dw, who);
    if (reinterpret_cast<uintptr_t>(norm_w) & 7u) return fail(LVX_ERR_ALIGN, "%s: norm_w is not 8-byte aligned", who);
  }
  return launch_kvproj_grad_rows(dtype, k, dk, dv, rstd, norm_w, dk_rows, dv_rows, dw, batch, Hkv, S,
                                 static_cast<cudaStream_t>(stream));
}

int lvx_fwd_merge_parts(const lvx_shape* s, const float* o_parts, const float* lse_parts, int count,
                        size_t part_stride_o, size_t part_stride_lse, void* o_out, float* lse_out, void* stream) {
  const char* who = "lvx_fwd_merge_parts";
  int rc = check_shape(s, who);
  if (rc) return rc;
  LVX_REQUIRE_PTR(o_parts, who);
  LVX_REQUIRE_PTR(lse_parts, who);
  LVX_REQUIRE_PTR(o_out, who);
  LVX_REQUIRE_PTR(lse_out, who);
  if (count < 1 || (part_stride_o & 3) != 0) return fail(LVX_ERR_SHAPE, "%s: count must be >= 1 and the O stride a multiple of 4 floats", who);
  return launch_fwd_merge_parts(*s, o_parts, lse_parts, count, part_stride_o, part_stride_lse, o_out, lse_out,
                                static_cast<cudaStream_t>(stream));
}

int lvx_sum_cast(const float* parts, int count, size_t part_stride, void* out, int out_dtype, size_t n, void* stream) {
  const char* who = "lvx_sum_cast";
  if (n == 0) return LVX_OK;
  LVX_REQUIRE_PTR(parts, who);
  LVX_REQUIRE_PTR(out, who);
  if (count < 1 || (part_stride & 3) != 0 || (n & 3) != 0)
    return fail(LVX_ERR_SHAPE, "%s: count >= 1, stride and n multiples of 4 floats are required", who);
  if (out_dtype != LVX_BF16 && out_dtype != LVX_FP16 && out_dtype != LVX_FP32)
    return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported", who, out_dtype);
  return launch_sum_cast(parts, count, part_stride, out, out_dtype, n, static_cast<cudaStream_t>(stream));
}

int lvx_add_cast(const float* a, const float* b, void* out, int out_dtype, size_t n, void* stream) {
  const char* who = "lvx_add_cast";
  if (n == 0) return LVX_OK;
  LVX_REQUIRE_PTR(a, who);
  LVX_REQUIRE_PTR(out, who);
  if (b && (reinterpret_cast<uintptr_t>(b) & 15u)) return fail(LVX_ERR_ALIGN, "%s: b is not 16-byte aligned", who);
  if (out_dtype != LVX_BF16 && out_dtype != LVX_FP16 && out_dtype != LVX_FP32)
    return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported", who, out_dtype);
  return launch_add_cast(a, b, out, out_dtype, n, static_cast<cudaStream_t>(stream));
}

static int check_view(const lvx_view* v, int elt, int align, const char* who, const char* name) {
  if (!v) return LVX_OK;
  if (!v->data) return fail(LVX_ERR_NULL, "%s: %s is NULL", who, name);
  if ((reinterpret_cast<uintptr_t>(v->data) & (align - 1)) ||
      ((v->stride_b | v->stride_h | v->stride_s) * elt) & (align - 1))
    return fail(LVX_ERR_ALIGN, "%s: rows of %s are not %d-byte aligned", who, name, align);
  return LVX_OK;
}

static int64_t head_norm_rows(const lvx_head_norm* c, const lvx_view* q, const lvx_view* k) {
  return int64_t(c->B) * c->S * ((q ? c->Hq : 0) + (k ? c->Hkv : 0));
}

static int check_head_norm(const lvx_head_norm* c, const lvx_view* q, const lvx_view* k, const char* who) {
  if (!c) return fail(LVX_ERR_NULL, "%s: the description is NULL", who);
  if (c->dtype != LVX_BF16 && c->dtype != LVX_FP16 && c->dtype != LVX_FP32) return fail(LVX_ERR_DTYPE, "%s: dtype %d unsupported", who, c->dtype);
  if (c->B < 0 || c->S < 0 || c->Hq < 0 || c->Hkv < 0) return fail(LVX_ERR_SHAPE, "%s: negative dimension", who);
  if (!q && !k) return fail(LVX_ERR_NULL, "%s: neither q nor k is given", who);
  if (!(c->eps >= 0.f)) return fail(LVX_ERR_SHAPE, "%s: eps must be non-negative", who);
  if ((c->cos == nullptr) != (c->sin == nullptr)) return fail(LVX_ERR_NULL, "%s: cos and sin go together", who);
  // units (two heads of a token at least) are counted in 32 bits
  if (int64_t(c->B) * c->S * std::max((c->Hq + 1) / 2, (c->Hkv + 1) / 2) >= (int64_t(1) << 31))
    return fail(LVX_ERR_LIMIT, "%s: B*S*heads too large", who);
  const int es = elt_size(c->dtype), align = 16;
  if (head_norm_rows(c, q, k) == 0) return LVX_OK;      // nothing is read, and nothing need be there
  int rc = check_view(q, es, align, who, "q");
  if (!rc) rc = check_view(k, es, align, who, "k");
  if (rc) return rc;
  const int ts = c->table_fp32 ? 4 : es;
  if ((reinterpret_cast<uintptr_t>(c->wq) | reinterpret_cast<uintptr_t>(c->wk)) & 15u)
    return fail(LVX_ERR_ALIGN, "%s: a weight is not 16-byte aligned", who);
  if ((reinterpret_cast<uintptr_t>(c->cos) | reinterpret_cast<uintptr_t>(c->sin) |
       (c->cos ? uintptr_t(c->table_stride_b | c->table_stride_s) * ts : 0)) & 15u)
    return fail(LVX_ERR_ALIGN, "%s: rows of cos and sin are not 16-byte aligned", who);
  return validate_arch();
}

int lvx_head_norm_rope(const lvx_head_norm* c, const lvx_view* q, const lvx_view* k, void* q_out, void* k_out, void* stream) {
  const char* who = "lvx_head_norm_rope";
  const int rc = check_head_norm(c, q, k, who);
  if (rc) return rc;
  if (head_norm_rows(c, q, k) == 0) return LVX_OK;
  if (q) LVX_REQUIRE_PTR(q_out, who);
  if (k) LVX_REQUIRE_PTR(k_out, who);
  return launch_head_norm(*c, q, k, q_out, k_out, static_cast<cudaStream_t>(stream));
}

int lvx_head_norm_rope_bwd(const lvx_head_norm* c, const lvx_view* q, const lvx_view* k, const lvx_view* gq, const lvx_view* gk,
                           void* dq, void* dk, void* dwq, void* dwk, void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "lvx_head_norm_rope_bwd";
  int rc = check_head_norm(c, q, k, who);
  if (rc) return rc;
  if ((q == nullptr) != (gq == nullptr) || (k == nullptr) != (gk == nullptr))
    return fail(LVX_ERR_NULL, "%s: q and gq, k and gk go together", who);
  const int es = elt_size(c->dtype), align = 16;
  const bool rows = head_norm_rows(c, q, k) > 0;
  if (rows && ((rc = check_view(gq, es, align, who, "gq")) || (rc = check_view(gk, es, align, who, "gk")))) return rc;
  if ((dwq && !(q && c->wq)) || (dwk && !(k && c->wk))) return fail(LVX_ERR_NULL, "%s: a gradient of a weight that is not there", who);
  if ((dq && !q) || (dk && !k)) return fail(LVX_ERR_NULL, "%s: a gradient of an input that is not there", who);
  if (dq && rows) LVX_REQUIRE_PTR(dq, who);
  if (dk && rows) LVX_REQUIRE_PTR(dk, who);
  if (!dq && !dk && !dwq && !dwk) return LVX_OK;
  if (dwq || dwk) {
    LVX_REQUIRE_PTR(scratch, who);
    if (scratch_bytes < LVX_HEAD_NORM_SCRATCH)
      return fail(LVX_ERR_WORKSPACE, "%s: scratch has %zu bytes, %d needed", who, scratch_bytes, LVX_HEAD_NORM_SCRATCH);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!rows) {      // no rows: the sums are empty
    const size_t n = 128 * (c->weight_fp32 ? 4 : es);
    cudaError_t e = cudaSuccess;
    if (dwq) e = cudaMemsetAsync(dwq, 0, n, st);
    if (e == cudaSuccess && dwk) e = cudaMemsetAsync(dwk, 0, n, st);
    return e == cudaSuccess ? LVX_OK : cuda_fail(e, "cudaMemsetAsync(dw)");
  }
  return launch_head_norm_bwd(*c, q, k, gq, gk, dq, dk, static_cast<float*>(scratch), dwq, dwk, st);
}

static lvx_view dense_view(const void* data, int heads, int rows) {
  return lvx_view{const_cast<void*>(data), int64_t(heads) * rows * 128, int64_t(rows) * 128, 128};
}

static int check_window(const lvx_shape* s, const lvx_window* w, const char* who) {
  const int rc = check_shape(s, who);
  if (rc) return rc;
  if (!w) return fail(LVX_ERR_NULL, "%s: the window is NULL", who);
  if (s->q_blocks > 1) return fail(LVX_ERR_SHAPE, "%s: one query block only", who);
  if (w->window < 0 || w->sinks < 0 || w->query_start < -1)
    return fail(LVX_ERR_SHAPE, "%s: window %d, sinks %d, query_start %d: negative", who, w->window, w->sinks, w->query_start);
  if (w->low_rows < 0 || w->low_rows > LVX_LOW_ROWS) return fail(LVX_ERR_SHAPE, "%s: low_rows %d outside 0..%d", who, w->low_rows, LVX_LOW_ROWS);
  if (s->Sq >= kWindowMaxLen || s->Skv >= kWindowMaxLen || w->query_start >= kWindowMaxLen)
    return fail(LVX_ERR_SHAPE, "%s: lengths and positions must be below %d", who, kWindowMaxLen);
  // the contract of the entry points: the kernels' item lists would take more
  if (s->dtype != LVX_FP32 && make_q_tiles(s->Hq / s->Hkv, s->Sq).count > 2 * 65535)
    return fail(LVX_ERR_LIMIT, "%s: %d query rows per KV head are more than 2 x 65,535 tiles", who, s->Hq / s->Hkv * s->Sq);
  return LVX_OK;
}

// q, k, v of a windowed call: rows that start on 16 bytes, and dense tensors for the fp32 kernels
static int check_qkv_views(const lvx_shape* s, const lvx_view* q, const lvx_view* k, const lvx_view* v, const char* who) {
  if (!q || !k || !v) return fail(LVX_ERR_NULL, "%s: q, k or v is NULL", who);
  const int es = elt_size(s->dtype);
  int rc = check_view(q, es, 16, who, "q");
  if (!rc && s->Skv > 0) rc = check_view(k, es, 16, who, "k");
  if (!rc && s->Skv > 0) rc = check_view(v, es, 16, who, "v");
  if (rc || s->dtype != LVX_FP32) return rc;
  auto dense = [](const lvx_view* t, int b, int h, int n) {
    return (n < 2 || t->stride_s == 128) && (h < 2 || t->stride_h == int64_t(n) * 128) && (b < 2 || t->stride_b == int64_t(h) * n * 128);
  };
  if (!dense(q, s->B, s->Hq, s->Sq) || (s->Skv > 0 && (!dense(k, s->B, s->Hkv, s->Skv) || !dense(v, s->B, s->Hkv, s->Skv))))
    return fail(LVX_ERR_SHAPE, "%s: fp32 tensors must be dense", who);
  return LVX_OK;
}

static size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
static size_t window_fwd_bytes(const lvx_shape* s, const FwdPlan& p, bool few) {
  const bool direct = p.nsplit <= (few ? kRowCluster : 1) && s->dtype != LVX_FP32;
  return direct ? 0 : p.o_part_bytes + p.ml_part_bytes;
}
static size_t window_bwd_bytes(const lvx_shape* s, const lvx_window* w) {
  return round256(size_t(s->B) * s->Hq * s->Sq * 4) +
         (s->dtype == LVX_FP32 ? 0 : (window_dq_floats(*s) + window_sink_floats(*s, *w)) * 4);
}

int lvx_window_workspace(const lvx_shape* s, const lvx_window* w, size_t* fwd_bytes, size_t* bwd_bytes) {
  const int rc = check_window(s, w, "lvx_window_workspace");
  if (rc) return rc;
  bool few;
  const FwdPlan p = plan_window(*s, *w, &few);
  if (fwd_bytes) *fwd_bytes = window_fwd_bytes(s, p, few);
  if (bwd_bytes) *bwd_bytes = window_bwd_bytes(s, w);
  return LVX_OK;
}

// The partials of a windowed forward, or where they are not needed (and o is given) its results.
static int window_forward(const lvx_shape* s, const lvx_window* w, const FwdPlan& p, bool few, const lvx_view* q, const lvx_view* k,
                          const lvx_view* v, const int32_t* kv_valid_len, float sm_scale, float* o_part, float* ml_part, void* o,
                          void* o_low, float* lse, int* sp, Order order, cudaStream_t st) {
  if (s->dtype == LVX_FP32)
    return launch_fwd_block_general(*s, p, q->data, k->data, v->data, kv_valid_len, nullptr, sm_scale, o_part, ml_part, st, w);
  if (few) return launch_window_rows(*s, *w, p, *q, *k, *v, kv_valid_len, sm_scale, o_part, ml_part, o, o_low, lse, sp, order, st);
  return launch_window_fwd(*s, *w, p, *q, *k, *v, kv_valid_len, sm_scale, o_part, ml_part, o, o_low, lse, sp, order, st);
}

int lvx_window_forward(const lvx_shape* s, const lvx_window* w, const lvx_view* q, const lvx_view* k, const lvx_view* v,
                       const int32_t* kv_valid_len, float sm_scale, void* workspace, size_t workspace_bytes, void* o, void* o_low,
                       float* lse, void* stream) {
  const char* who = "lvx_window_forward";
  int rc = check_window(s, w, who);
  if (!rc) rc = check_qkv_views(s, q, k, v, who);
  if (!rc) rc = check_arch();
  if (rc) return rc;
  if (!(sm_scale > 0.f)) return fail(LVX_ERR_SHAPE, "%s: sm_scale must be positive", who);
  LVX_REQUIRE_PTR(o, who);
  if (o_low && s->dtype == LVX_FP32) return fail(LVX_ERR_DTYPE, "%s: nothing of O is dropped in fp32", who);
  LVX_REQUIRE_PTR(lse, who);
  bool few;
  const FwdPlan p = plan_window(*s, *w, &few);
  const size_t need = window_fwd_bytes(s, p, few);
  if (need) LVX_REQUIRE_PTR(workspace, who);
  if (workspace_bytes < need) return fail(LVX_ERR_WORKSPACE, "%s: workspace has %zu bytes, %zu needed", who, workspace_bytes, need);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (need == 0) return window_forward(s, w, p, few, q, k, v, kv_valid_len, sm_scale, nullptr, nullptr, o, o_low, lse, sp, ORDER_AFTER, st);
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_part_bytes);
  rc = window_forward(s, w, p, few, q, k, v, kv_valid_len, sm_scale, o_part, ml_part, nullptr, nullptr, nullptr, sp, ORDER_AFTER, st);
  return rc ? rc : launch_fwd_combine(*s, p, o_part, ml_part, nullptr, nullptr, o, lse, 1, st, ORDER_OVERLAP, low_rows(*s, *w, o_low, kv_valid_len));
}

int lvx_window_backward(const lvx_shape* s, const lvx_window* w, const void* d_o, const lvx_view* q, const lvx_view* k,
                        const lvx_view* v, const void* o, const void* o_low, const float* lse, const int32_t* kv_valid_len,
                        float sm_scale, void* workspace, size_t workspace_bytes, void* dq, void* dk, void* dv, void* stream) {
  const char* who = "lvx_window_backward";
  int rc = check_window(s, w, who);
  if (!rc) rc = check_qkv_views(s, q, k, v, who);
  if (!rc) rc = check_arch();
  if (rc) return rc;
  if (!(sm_scale > 0.f)) return fail(LVX_ERR_SHAPE, "%s: sm_scale must be positive", who);
  LVX_REQUIRE_PTR(d_o, who);
  LVX_REQUIRE_PTR(o, who);
  if (o_low && s->dtype == LVX_FP32) return fail(LVX_ERR_DTYPE, "%s: nothing of O is dropped in fp32", who);
  LVX_REQUIRE_PTR(lse, who);
  LVX_REQUIRE_PTR(dq, who);
  LVX_REQUIRE_PTR(workspace, who);
  if (s->Skv > 0) {
    LVX_REQUIRE_PTR(dk, who);
    LVX_REQUIRE_PTR(dv, who);
  }
  const size_t need = window_bwd_bytes(s, w);
  if (workspace_bytes < need) return fail(LVX_ERR_WORKSPACE, "%s: workspace has %zu bytes, %zu needed", who, workspace_bytes, need);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool direct = s->dtype == LVX_FP32;      // dQ is accumulated where it is wanted
  const size_t rows = size_t(s->B) * s->Hq * s->Sq;
  float* delta = static_cast<float*>(workspace);
  float* dq_acc = direct ? static_cast<float*>(dq) : reinterpret_cast<float*>(static_cast<char*>(workspace) + round256(rows * 4));
  float* parts = direct ? nullptr : dq_acc + window_dq_floats(*s);
  if ((rc = launch_bwd_prep(*s, o, d_o, delta, st, low_rows(*s, *w, const_cast<void*>(o_low), kv_valid_len), dq_acc,
                            direct ? rows * 512 : window_dq_floats(*s) * 4)))
    return rc;
  if (s->Skv > 0) {
    const lvx_view dov = dense_view(d_o, s->Hq, s->Sq);
    rc = direct ? launch_bwd_block_general(*s, q->data, d_o, lse, delta, k->data, v->data, kv_valid_len, nullptr, sm_scale, dq_acc,
                                           dk, dv, 2, st, w)
                : launch_window_bwd(*s, *w, *q, dov, *k, *v, lse, delta, kv_valid_len, sm_scale, dq_acc, parts, dk, dv, sp, ORDER_OVERLAP, st);
  }
  return rc || direct ? rc : launch_window_dq(*s, *w, dq_acc, parts, dq, dk, dv, sp, st);
}

// The pieces of a call with shared prefixes: the prefix as an attention of packed rows, and the layout of the scratch.
struct SharedCall {
  lvx_shape pre;            // B = prefixes, one "head" per packed row, Sq = 1
  lvx_shape fwd;            // the same for the forward, which reads a single token's rows where they are: a "token" per request
  bool in_place;            // that it does
  lvx_window pre_win, own_win;
  FwdPlan pre_plan, own_plan;
  bool pre_few, own_few;
  bool packed;              // the packed order is another one than q's
  size_t rows;              // B * Hq * Sq
};
static int shared_call(SharedCall* c, const lvx_shape* s, int prefixes, int prefix_len, const char* who) {
  c->own_win = lvx_window{0, 0, -1, 0};
  int rc = check_window(s, &c->own_win, who);
  if (rc) return rc;
  if (prefixes < 1 || s->B % prefixes) return fail(LVX_ERR_SHAPE, "%s: %d requests are not a multiple of %d prefixes", who, s->B, prefixes);
  if (prefix_len < 1 || prefix_len >= kWindowMaxLen) return fail(LVX_ERR_SHAPE, "%s: a prefix of %d keys", who, prefix_len);
  const int64_t rows = int64_t(s->B / prefixes) * (s->Hq / s->Hkv) * s->Sq;      // of a prefix' KV head
  // all rows are counted in 32 bits, with room for a tile's last ones
  if (rows * s->Hkv * prefixes > (int64_t(1) << 30)) return fail(LVX_ERR_SHAPE, "%s: dimension too large", who);
  c->pre = *s;
  c->pre.B = prefixes;
  c->pre.Hq = int32_t(rows * s->Hkv);
  c->pre.Sq = 1;
  c->pre.Skv = prefix_len;
  c->pre_win = lvx_window{0, 0, prefix_len, 0};      // every row stands behind all keys
  if ((rc = check_window(&c->pre, &c->pre_win, who))) return rc;
  c->packed = s->B != prefixes && s->Hkv > 1;
  c->rows = size_t(s->B) * s->Hq * s->Sq;
  return LVX_OK;
}

// Forward: its plans, and the scratch.
static size_t shared_fwd_plan(SharedCall* c, const lvx_shape* s) {
  c->fwd = c->pre;
  c->in_place = c->packed && s->Sq == 1 && s->dtype != LVX_FP32;      // (the fp32 kernels read dense rows)
  if (c->in_place) {
    c->fwd.Hq = s->Hq;
    c->fwd.Sq = s->B / c->pre.B;
  }
  c->pre_plan = plan_window(c->fwd, c->pre_win, &c->pre_few, true);
  size_t n = c->pre_plan.o_part_bytes + c->pre_plan.ml_part_bytes + (c->in_place ? 0 : round256(c->rows * 128 * elt_size(s->dtype)));
  if (s->Skv > 0) {
    c->own_plan = plan_window(*s, c->own_win, &c->own_few, true);
    n += c->own_plan.o_part_bytes + c->own_plan.ml_part_bytes;
  }
  return n;
}
static size_t shared_bwd_bytes(const SharedCall& c, const lvx_shape* s) {
  const bool f32 = s->dtype == LVX_FP32;
  const size_t acc = f32 ? c.rows * 512 : window_dq_floats(c.pre) * 4;
  const size_t acc_own = s->Skv == 0 ? 0 : f32 ? c.rows * 512 : window_dq_floats(*s) * 4;
  return 3 * round256(c.rows * 4) + 2 * round256(c.rows * 128 * elt_size(s->dtype)) + round256(acc) + acc_own;
}

int lvx_shared_workspace(const lvx_shape* s, int prefixes, int prefix_len, size_t* fwd_bytes, size_t* bwd_bytes) {
  SharedCall c;
  const int rc = shared_call(&c, s, prefixes, prefix_len, "lvx_shared_workspace");
  if (rc) return rc;
  if (fwd_bytes) *fwd_bytes = shared_fwd_plan(&c, s);
  if (bwd_bytes) *bwd_bytes = shared_bwd_bytes(c, s);
  return LVX_OK;
}

int lvx_shared_forward(const lvx_shape* s, int prefixes, int prefix_len, const lvx_view* q, const lvx_view* pk, const lvx_view* pv,
                       const int32_t* prefix_valid_len, const lvx_view* k, const lvx_view* v, const int32_t* kv_valid_len,
                       float sm_scale, void* workspace, size_t workspace_bytes, void* o, float* lse, void* stream) {
  const char* who = "lvx_shared_forward";
  SharedCall c;
  int rc = shared_call(&c, s, prefixes, prefix_len, who);
  if (!rc) rc = check_qkv_views(s, q, s->Skv > 0 ? k : q, s->Skv > 0 ? v : q, who);
  if (rc) return rc;
  const size_t need = shared_fwd_plan(&c, s);
  const lvx_view packed_q = c.in_place ? lvx_view{q->data, (s->B / prefixes) * q->stride_b, q->stride_h, q->stride_b}
                                       : dense_view(c.packed ? workspace : q->data, c.pre.Hq, 1);
  if ((rc = check_qkv_views(&c.fwd, &packed_q, pk, pv, who)) || (rc = check_arch())) return rc;
  if (!(sm_scale > 0.f)) return fail(LVX_ERR_SHAPE, "%s: sm_scale must be positive", who);
  LVX_REQUIRE_PTR(o, who);
  LVX_REQUIRE_PTR(lse, who);
  LVX_REQUIRE_PTR(workspace, who);
  if (workspace_bytes < need) return fail(LVX_ERR_WORKSPACE, "%s: workspace has %zu bytes, %zu needed", who, workspace_bytes, need);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* at = static_cast<char*>(workspace) + (c.in_place ? 0 : round256(c.rows * 128 * elt_size(s->dtype)));
  auto take = [&](size_t n) {
    float* p = reinterpret_cast<float*>(at);
    at += n;
    return p;
  };
  float* o_pre = take(c.pre_plan.o_part_bytes);
  float* ml_pre = take(c.pre_plan.ml_part_bytes);
  float *o_own = nullptr, *ml_own = nullptr;
  // q as it lies serves where the orders agree, if it is dense
  const bool dense = q->stride_s == 128 && q->stride_h == int64_t(s->Sq) * 128 && q->stride_b == int64_t(s->Hq) * s->Sq * 128;
  lvx_view pq = packed_q;
  const bool pack = !c.in_place && (c.packed || !dense);
  if (pack) {
    pq.data = workspace;
    if ((rc = launch_pack_rows(*s, prefixes, *q, nullptr, nullptr, nullptr, workspace, nullptr, nullptr, nullptr, ORDER_AFTER, st))) return rc;
  }
  if (s->Skv > 0) {
    o_own = take(c.own_plan.o_part_bytes);
    ml_own = take(c.own_plan.ml_part_bytes);
  }
  auto own_keys = [&](Order order) {
    return s->Skv == 0 ? LVX_OK
                       : window_forward(s, &c.own_win, c.own_plan, c.own_few, q, k, v, kv_valid_len, sm_scale, o_own, ml_own, nullptr, nullptr,
                                        nullptr, sp, order, st);
  };
  auto prefix = [&](Order order) {
    return window_forward(&c.fwd, &c.pre_win, c.pre_plan, c.pre_few, &pq, pk, pv, prefix_valid_len, sm_scale, o_pre, ml_pre, nullptr,
                          nullptr, nullptr, sp, order, st);
  };
  // Packed rows are read by the kernel that waits for the packing. The own keys' kernel reads the caller's tensors alone, and without
  // packing so does the prefix' one: the second of them may stand beside the first. (The own keys first, which fill SMs faster, would
  // take 53 us instead of 57 for four tokens of 32 requests behind 6,404 shared and 512 own keys, 77 tokens of eight are even; but then
  // the packed rows' reader would not have waited for them.)
  if (pack) {
    if ((rc = prefix(ORDER_OVERLAP)) || (rc = own_keys(ORDER_BESIDE))) return rc;
  } else {
    if ((rc = own_keys(ORDER_AFTER)) || (rc = prefix(s->Skv > 0 ? ORDER_BESIDE : ORDER_AFTER))) return rc;
  }
  return launch_shared_combine(*s, prefixes, c.in_place, o_pre, ml_pre, c.pre_plan.nsplit, o_own, ml_own, o_own ? c.own_plan.nsplit : 0, o, lse, st);
}

int lvx_shared_backward(const lvx_shape* s, int prefixes, int prefix_len, const void* d_o, const lvx_view* q, const lvx_view* pk,
                        const lvx_view* pv, const int32_t* prefix_valid_len, const lvx_view* k, const lvx_view* v,
                        const int32_t* kv_valid_len, const void* o, const float* lse, float sm_scale, void* workspace,
                        size_t workspace_bytes, void* dq, void* dpk, void* dpv, void* dk, void* dv, void* stream) {
  const char* who = "lvx_shared_backward";
  SharedCall c;
  int rc = shared_call(&c, s, prefixes, prefix_len, who);
  if (!rc) rc = check_qkv_views(s, q, s->Skv > 0 ? k : q, s->Skv > 0 ? v : q, who);
  if (rc) return rc;
  const lvx_view packed_q = dense_view(c.packed ? workspace : q->data, c.pre.Hq, 1);
  if ((rc = check_qkv_views(&c.pre, &packed_q, pk, pv, who)) || (rc = check_arch())) return rc;
  if (!(sm_scale > 0.f)) return fail(LVX_ERR_SHAPE, "%s: sm_scale must be positive", who);
  LVX_REQUIRE_PTR(d_o, who);
  LVX_REQUIRE_PTR(o, who);
  LVX_REQUIRE_PTR(lse, who);
  LVX_REQUIRE_PTR(dq, who);
  LVX_REQUIRE_PTR(dpk, who);
  LVX_REQUIRE_PTR(dpv, who);
  LVX_REQUIRE_PTR(workspace, who);
  if (s->Skv > 0) {
    LVX_REQUIRE_PTR(dk, who);
    LVX_REQUIRE_PTR(dv, who);
  }
  const size_t need = shared_bwd_bytes(c, s);
  if (workspace_bytes < need) return fail(LVX_ERR_WORKSPACE, "%s: workspace has %zu bytes, %zu needed", who, workspace_bytes, need);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f32 = s->dtype == LVX_FP32;
  const size_t row_bytes = round256(c.rows * 128 * elt_size(s->dtype)), stat = round256(c.rows * 4);
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t n) {
    char* p = at;
    at += n;
    return p;
  };
  float* delta = reinterpret_cast<float*>(take(stat));
  float* lse_p = reinterpret_cast<float*>(take(stat));
  float* delta_p = reinterpret_cast<float*>(take(stat));
  char* q_p = take(row_bytes);
  char* do_p = take(row_bytes);
  float* acc = reinterpret_cast<float*>(at);
  const size_t acc_bytes = round256(f32 ? c.rows * 512 : window_dq_floats(c.pre) * 4);
  float* acc_own = s->Skv > 0 ? reinterpret_cast<float*>(at + acc_bytes) : nullptr;
  if ((rc = launch_bwd_prep(*s, o, d_o, delta, st, {}, acc, static_cast<char*>(workspace) + need - at))) return rc;
  const bool dense = q->stride_s == 128 && q->stride_h == int64_t(s->Sq) * 128 && q->stride_b == int64_t(s->Hq) * s->Sq * 128;
  const bool pack = c.packed || !dense;
  if (pack && (rc = launch_pack_rows(*s, prefixes, *q, d_o, lse, delta, q_p, do_p, lse_p, delta_p, ORDER_OVERLAP, st))) return rc;
  const lvx_view pq = dense_view(pack ? q_p : q->data, c.pre.Hq, 1), pdo = dense_view(pack ? do_p : d_o, c.pre.Hq, 1);
  const float *pl = pack ? lse_p : lse, *pd = pack ? delta_p : delta;
  const lvx_view dov = dense_view(d_o, s->Hq, s->Sq);
  rc = f32 ? launch_bwd_block_general(c.pre, pq.data, pdo.data, pl, pd, pk->data, pv->data, prefix_valid_len, nullptr, sm_scale, acc,
                                      dpk, dpv, 2, st, &c.pre_win)
           : launch_window_bwd(c.pre, c.pre_win, pq, pdo, *pk, *pv, pl, pd, prefix_valid_len, sm_scale, acc, nullptr, dpk, dpv, sp,
                               ORDER_OVERLAP, st);
  if (!rc && s->Skv > 0)
    rc = f32 ? launch_bwd_block_general(*s, q->data, d_o, lse, delta, k->data, v->data, kv_valid_len, nullptr, sm_scale, acc_own, dk,
                                        dv, 2, st, &c.own_win)
             : launch_window_bwd(*s, c.own_win, *q, dov, *k, *v, lse, delta, kv_valid_len, sm_scale, acc_own, nullptr, dk, dv, sp, ORDER_OVERLAP, st);
  if (rc) return rc;
  const QTiles pt = make_q_tiles(c.pre.Hq / c.pre.Hkv, 1);
  const int pre_slab_rows = f32 ? c.pre.Hq / c.pre.Hkv : pt.chunks * pt.heads;
  return launch_shared_dq(*s, prefixes, acc, pre_slab_rows, acc_own, dq, st);
}

int lvx_selftest_key_tiles(const lvx_window* w, int valid, int p0, int p1, int tile_shift, int* tiles, int capacity, int* count) {
  const char* who = "lvx_selftest_key_tiles";
  if (!w || !count || (!tiles && capacity > 0)) return fail(LVX_ERR_NULL, "%s: w, tiles or count is NULL", who);
  if (valid < 0 || valid >= kWindowMaxLen || p0 > p1 || p0 <= -kWindowMaxLen || p1 >= 2 * kWindowMaxLen || tile_shift < 0 || tile_shift > 20)
    return fail(LVX_ERR_SHAPE, "%s: a length, position or tile size out of range", who);
  const KeyTiles kt = key_tiles(make_window_mask(*w), valid, p0, p1, tile_shift);
  for (int j = 0; j < kt.n && j < capacity; ++j) tiles[j] = kt.tile(j);
  *count = kt.n;
  return LVX_OK;
}

int lvx_selftest_mma(int mode, const void* a, const void* b, float* d_out, void* stream) {
  const char* who = "lvx_selftest_mma";
  int rc = check_arch();
  if (rc) return rc;
  LVX_REQUIRE_PTR(a, who);
  LVX_REQUIRE_PTR(b, who);
  LVX_REQUIRE_PTR(d_out, who);
  int* sp = status_ptr();
  if (!sp) return fail(LVX_ERR_DRIVER, "%s: status word unavailable", who);
  return launch_selftest(mode, a, b, d_out, sp, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
