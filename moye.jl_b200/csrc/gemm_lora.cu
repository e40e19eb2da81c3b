// Low-rank adapters of many requests beside a shared projection:
//
//   D[i] = C[i] + s[a] * (X[i] . A[a]^T) . B[a]^T        X (rows, K), A (adapters, R, K), B (adapters, N, R), C, D (rows, N)
//
// where a = adapters[q] is the adapter of the request q that row i belongs to: offsets[q] <= i < offsets[q+1], or
// q = i when no offsets are given (a decoding step).  An adapter number outside 0..adapters-1 means none: D[i] = C[i].
// Rows outside every request are left as they were.  No counterpart in the reference.
//
// The product of rank R between the two factors never leaves the chip: a thread-block cluster takes a row, CTA c of it
// a slice of K for the first factor; the partial R-vectors meet through distributed shared memory (fp32, summed in CTA
// order, so the result does not depend on timing); then CTA c takes a slice of N for the second factor.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "ptx.cuh"

namespace moye {

constexpr int kLoraCtas = 8;         // cluster size
constexpr int kLoraThreads = 256;
constexpr int kMaxLoraRank = 128;

struct LoraArgs {
  int rows, requests, adapters, rank, n, k;
  const void *X, *A, *B, *C;
  void* D;
  long long x_pitch, a_pitch, a_stride, b_pitch, b_stride, c_pitch, d_pitch;  // elements
  const int *which, *offsets;
  const float* scales;
};

template <typename T>
__device__ __forceinline__ float2 lora_pair(uint32_t v);
template <>
__device__ __forceinline__ float2 lora_pair<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <>
__device__ __forceinline__ float2 lora_pair<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }

template <typename T>
__device__ __forceinline__ void lora_unpack(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = lora_pair<T>(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}

__device__ __forceinline__ float lora_load(const float* p) { return *p; }
__device__ __forceinline__ float lora_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float lora_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void lora_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void lora_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void lora_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float ld_remote_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

template <typename T, typename OutT>
__global__ void __launch_bounds__(kLoraThreads)
lora_row_kernel(const LoraArgs g) {
  __shared__ float part[kMaxLoraRank], v[kMaxLoraRank];
  __shared__ int found;
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / kLoraCtas, rank = (int)cluster_ctarank();
  if (g.offsets) {
    if (tid == 0) found = -1;
    __syncthreads();
    for (int q = tid; q < g.requests; q += kLoraThreads)
      if (g.offsets[q] <= row && row < g.offsets[q + 1]) atomicMax(&found, q);
    __syncthreads();
  } else if (tid == 0) {
    found = row;
  }
  __syncthreads();
  const int q = found;
  if (q < 0) return;  // the same in every CTA of the cluster
  const int a = g.which[q];
  const int n0 = (int)((long long)g.n * rank / kLoraCtas), n1 = (int)((long long)g.n * (rank + 1) / kLoraCtas);
  const OutT* c_row = static_cast<const OutT*>(g.C) + row * g.c_pitch;
  OutT* d_row = static_cast<OutT*>(g.D) + row * g.d_pitch;
  if (a < 0 || a >= g.adapters) {
    if (g.C != g.D)
      for (int n = n0 + tid; n < n1; n += kLoraThreads) d_row[n] = c_row[n];
    return;
  }
  {
    const int kv = g.k / 8, v0 = (int)((long long)kv * rank / kLoraCtas), v1 = (int)((long long)kv * (rank + 1) / kLoraCtas);
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(g.X) + row * g.x_pitch);
    for (int r = warp; r < g.rank; r += kLoraThreads / 32) {
      const uint4* ar = reinterpret_cast<const uint4*>(static_cast<const T*>(g.A) + a * g.a_stride + r * g.a_pitch);
      float s = 0.f;
      for (int i = v0 + lane; i < v1; i += 32) {
        float xf[8], af[8];
        lora_unpack<T>(x[i], xf);
        lora_unpack<T>(ar[i], af);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += xf[e] * af[e];
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      if (lane == 0) part[r] = s;
    }
  }
  cluster_arrive();
  cluster_wait();  // every CTA's partial vector is in place
  if (tid < g.rank) {
    float s = 0.f;
    for (int c = 0; c < kLoraCtas; ++c) s += ld_remote_f32(mapa_shared(smem_u32(part + tid), c));
    v[tid] = s * (g.scales ? g.scales[a] : 1.f);
  }
  cluster_arrive();  // this CTA has read the others' parts; it leaves only after they have read its own (below)
  __syncthreads();
  for (int n = n0 + tid; n < n1; n += kLoraThreads) {
    const uint4* b = reinterpret_cast<const uint4*>(static_cast<const T*>(g.B) + a * g.b_stride + n * g.b_pitch);
    float s = 0.f;
    for (int i = 0; i < g.rank / 8; ++i) {
      float bf[8];
      lora_unpack<T>(b[i], bf);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += bf[e] * v[i * 8 + e];
    }
    lora_store(d_row + n, lora_load(c_row + n) + s);
  }
  cluster_wait();
}

// ---------------------------------------------------------------------------------------------- host side
static int check_lora_factor(const char* what, const moye_tensor_t* t) {
  if ((t->shape[2] > 1 && t->stride[2] != 1) || (t->shape[1] > 1 && t->stride[1] < t->shape[2]) ||
      (t->shape[0] > 1 && t->stride[0] < (t->shape[1] - 1) * t->stride[1] + t->shape[2]))
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "gemm_lora: %s needs contiguous rows, and rows and adapters that do not overlap", what);
  if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) != 0 || (t->shape[1] > 1 && t->stride[1] % 8 != 0) ||
      (t->shape[0] > 1 && t->stride[0] % 8 != 0))
    MOYE_FAIL(MOYE_ERR_MISALIGNED, "gemm_lora: %s needs a base and pitches that are multiples of 16 bytes", what);
  return MOYE_OK;
}

int launch_gemm_lora(moye_b200_ctx* h, const moye_tensor_t* D, const moye_tensor_t* X, const moye_tensor_t* A, const moye_tensor_t* B,
                     const moye_tensor_t* C, const int* which, const int* offsets, int requests, const float* scales,
                     cudaStream_t stream) {
  if (!C) C = D;
  if (D->rank != 2 || X->rank != 2 || C->rank != 2 || A->rank != 3 || B->rank != 3)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "gemm_lora: D, X and C must be rank 2, A and B rank 3");
  const int64_t T = X->shape[0], K = X->shape[1], N = D->shape[1], R = A->shape[1], L = A->shape[0];
  if (A->shape[2] != K || B->shape[0] != L || B->shape[1] != N || B->shape[2] != R || D->shape[0] != T || C->shape[0] != T || C->shape[1] != N)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "gemm_lora: shape mismatch: X (%lld,%lld) A (%lld,%lld,%lld) B (%lld,%lld,%lld) C (%lld,%lld) D (%lld,%lld)",
              (long long)T, (long long)K, (long long)L, (long long)R, (long long)A->shape[2], (long long)B->shape[0],
              (long long)B->shape[1], (long long)B->shape[2], (long long)C->shape[0], (long long)C->shape[1],
              (long long)D->shape[0], (long long)D->shape[1]);
  if ((X->dtype != MOYE_F16 && X->dtype != MOYE_BF16) || A->dtype != X->dtype || B->dtype != X->dtype)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "gemm_lora: X, A and B must all be f16 or all bf16");
  if ((D->dtype != MOYE_F32 && D->dtype != X->dtype) || C->dtype != D->dtype)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "gemm_lora: C and D must both be f32 or both the operands' type");
  if (T < 0 || N <= 0 || K <= 0 || L <= 0) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "gemm_lora: empty product");
  if (R < 8 || R > kMaxLoraRank || R % 8 != 0)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "gemm_lora: the rank must be a multiple of 8, 8 to %d (got %lld): pad A and B with zeros", kMaxLoraRank, (long long)R);
  if (K % 8 != 0) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "gemm_lora: K must be a multiple of 8 (got %lld)", (long long)K);
  if (T > INT32_MAX / 16 || N > INT32_MAX / 2 || K > INT32_MAX / 2 || L > INT32_MAX / 2) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "gemm_lora: extent too large");
  if (requests < 0 || (!offsets && requests != T))
    MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gemm_lora: without offsets there is one request per row (%lld rows, %d requests)", (long long)T, requests);
  if (T == 0 || requests == 0) return MOYE_OK;
  if (!D->ptr || !C->ptr || !X->ptr || !A->ptr || !B->ptr || !which) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gemm_lora: null pointer");
  if (int rc = check_lora_factor("A", A)) return rc;
  if (int rc = check_lora_factor("B", B)) return rc;
  if ((K > 1 && X->stride[1] != 1) || (T > 1 && X->stride[0] < K)) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "gemm_lora: rows of X must be contiguous and must not overlap");
  if ((reinterpret_cast<uintptr_t>(X->ptr) & 15) != 0 || (T > 1 && X->stride[0] % 8 != 0))
    MOYE_FAIL(MOYE_ERR_MISALIGNED, "gemm_lora: X needs a base and a row pitch that are multiples of 16 bytes");
  for (const moye_tensor_t* t : {D, C})
    if ((N > 1 && t->stride[1] != 1) || (T > 1 && t->stride[0] < N))
      MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "gemm_lora: rows of C and D must be contiguous and must not overlap");
  if (C->ptr == D->ptr && T > 1 && C->stride[0] != D->stride[0])
    MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gemm_lora: C at D's address must be D");
  LoraArgs g = {};
  g.rows = (int)T;
  g.requests = requests;
  g.adapters = (int)L;
  g.rank = (int)R;
  g.n = (int)N;
  g.k = (int)K;
  g.X = X->ptr; g.A = A->ptr; g.B = B->ptr; g.C = C->ptr; g.D = D->ptr;
  g.x_pitch = X->stride[0];
  g.a_pitch = A->stride[1]; g.a_stride = A->stride[0];
  g.b_pitch = B->stride[1]; g.b_stride = B->stride[0];
  g.c_pitch = C->stride[0]; g.d_pitch = D->stride[0];
  g.which = which;
  g.offsets = offsets;
  g.scales = scales;
  auto go = [&](auto kern) -> int {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)T * kLoraCtas);
    cfg.blockDim = dim3(kLoraThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kLoraCtas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = launch_without_pdl() ? 1 : 2;
    MOYE_CUDA(cudaLaunchKernelEx(&cfg, kern, g));
    return MOYE_OK;
  };
  if (X->dtype == MOYE_F16) return D->dtype == MOYE_F32 ? go(lora_row_kernel<__half, float>) : go(lora_row_kernel<__half, __half>);
  return D->dtype == MOYE_F32 ? go(lora_row_kernel<__nv_bfloat16, float>) : go(lora_row_kernel<__nv_bfloat16, __nv_bfloat16>);
}

}  // namespace moye
