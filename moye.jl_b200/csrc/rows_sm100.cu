// Rows sorted by the group they choose, and back: `group_rows`, `gather_rows`, `combine_rows` and its gradient.
// No counterpart in the reference, whose copies (src/algorithm/copy.jl:4-64) move tiles whose place the layout alone
// decides; here the place of a row is data.
//
// T tokens choose `c` groups each (a choice outside 0..G-1 is dropped).  With the n = T*c choices numbered t*c + j:
//   order    the kept choices, stably sorted by group           (order[p] = choice at position p; -1 behind the last)
//   offsets  offsets[g] = first position of group g, offsets[G] = number of kept choices
//   inverse  inverse[order[p]] = p, -1 for a dropped choice
//   gather   dst[p] = src[order[p] / c]
//   combine  dst[t] = sum_j w[t,j] * src[inverse[t,j]]          (w = 1: the gradient of gather)
//   grad     dsrc[inverse[t,j]] = w[t,j] * ddst[t],  dw[t,j] = <ddst[t], src[inverse[t,j]]>
// All three data movements walk the TOKENS and go through `inverse`: a token's row is then read (or written) once and
// not once a choice, every output element has one writer, and sums run in the order of the choices: no atomics, the
// same bits on every run.  They are bound by memory: (T + n) rows for gather and combine, (T + 2n) for the gradient.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "ptx.cuh"

namespace moye {

// ---------------------------------------------------------------------------------------------- group_rows
// A counting sort in one launch of one cluster.  CTA r of C owns a contiguous run of choices, warp w of it a
// contiguous part of that: counting per warp in shared memory, a prefix over warps (per CTA), over CTAs (the other
// CTAs' totals through distributed shared memory) and over groups gives the first position of every (group, warp),
// and a second walk in the same order hands positions out, 32 choices at a time.  The order inside a warp's 32 is the
// lanes', so the sort is stable.  Latency-bound: the data is a few bytes per choice.
constexpr int kGroupThreads = 1024;
constexpr int kGroupWarps = kGroupThreads / 32;
constexpr int kMaxGroups = 1024;  // one thread per group in the scans; 32 counters a group fill 128 KB

struct IdSource {
  const void* ptr;
  int is64;
  long long s_token, s_choice;
  int choices;
};

__device__ __forceinline__ int load_id(const IdSource& ids, int i, int groups) {
  const int t = i / ids.choices, j = i - t * ids.choices;
  const long long at = t * ids.s_token + j * ids.s_choice;
  const long long v = ids.is64 ? static_cast<const long long*>(ids.ptr)[at] : static_cast<const int*>(ids.ptr)[at];
  return v >= 0 && v < groups ? static_cast<int>(v) : -1;
}

__device__ __forceinline__ int ld_remote_i32(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__global__ void __launch_bounds__(kGroupThreads, 1)
group_rows_kernel(const IdSource ids, int n, int groups, int* order, int* offsets, int* inverse) {
  extern __shared__ int sm[];
  int* hist = sm;                           // [warp][group]: counts, then positions relative to the CTA's first
  int* total = sm + kGroupWarps * groups;   // [group]: this CTA's count
  int* base = total + groups;               // [group]: first position of this CTA's members
  __shared__ int warp_sum[kGroupWarps];
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const long long blocks = ((long long)n + 31) / 32;  // runs of 32 choices, dealt to warps in order
  const long long w_all = (long long)C * kGroupWarps, me = (long long)rank * kGroupWarps + warp;
  const int b0 = (int)(blocks * me / w_all), b1 = (int)(blocks * (me + 1) / w_all);
  int* mine = hist + warp * groups;

  for (int g = lane; g < groups; g += 32) mine[g] = 0;
  __syncwarp();
  for (int b = b0; b < b1; ++b) {
    const int i = b * 32 + lane;
    const int id = i < n ? load_id(ids, i, groups) : -1;
    if (id >= 0) atomicAdd(&mine[id], 1);
  }
  __syncthreads();
  for (int g = tid; g < groups; g += kGroupThreads) {
    int run = 0;
    for (int w = 0; w < kGroupWarps; ++w) {
      const int v = hist[w * groups + g];
      hist[w * groups + g] = run;
      run += v;
    }
    total[g] = run;
  }
  cluster_arrive();
  cluster_wait();  // every CTA's totals are in place
  int before = 0, all = 0;
  if (tid < groups) {
    const uint32_t at = smem_u32(total + tid);
    for (int r = 0; r < C; ++r) {
      const int v = ld_remote_i32(mapa_shared(at, r));
      if (r < rank) before += v;
      all += v;
    }
  }
  cluster_arrive();  // this CTA has read the others' totals; it must not leave before they have read its own (below)
  // exclusive prefix of `all` over the groups, one group per thread
  int incl = all;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(~0u, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sum[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, s, d);
      if (lane >= d) s += up;
    }
    warp_sum[lane] = s;
  }
  __syncthreads();
  const int first = incl - all + (warp ? warp_sum[warp - 1] : 0);
  const int kept = warp_sum[kGroupWarps - 1];
  if (tid < groups) {
    base[tid] = first + before;
    if (rank == 0) offsets[tid] = first;
  }
  if (rank == 0 && tid == 0) offsets[groups] = kept;
  __syncthreads();
  for (int b = b0; b < b1; ++b) {
    const int i = b * 32 + lane;
    const int id = i < n ? load_id(ids, i, groups) : -1;
    const unsigned peers = __match_any_sync(~0u, id);
    const int ahead = __popc(peers & ((1u << lane) - 1));
    int pos = -1;
    if (id >= 0) pos = base[id] + mine[id] + ahead;
    __syncwarp();
    if (id >= 0 && ahead == 0) mine[id] += __popc(peers);
    __syncwarp();
    if (i < n) {
      inverse[i] = pos;
      if (pos >= 0) order[pos] = i;
    }
  }
  for (int p = kept + rank * kGroupThreads + tid; p < n; p += C * kGroupThreads) order[p] = -1;
  cluster_wait();
}

int launch_group_rows(moye_b200_ctx* h, const moye_tensor_t* ids, int groups, int* order, int* offsets, int* inverse,
                      cudaStream_t stream) {
  if (ids->dtype != MOYE_S32 && ids->dtype != MOYE_U64)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "group_rows: ids must be 32- or 64-bit integers (got dtype %d)", ids->dtype);
  if (ids->rank != 1 && ids->rank != 2) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "group_rows: ids must be (tokens) or (tokens, choices)");
  const long long tokens = ids->shape[0], choices = ids->rank == 2 ? ids->shape[1] : 1;
  if (groups < 1 || groups > kMaxGroups)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "group_rows: 1 to %d groups (got %d)", kMaxGroups, groups);
  if (tokens < 0 || choices < 1) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "group_rows: ids are (%lld, %lld)", tokens, choices);
  if (tokens > INT32_MAX / 2 / choices) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "group_rows: more than 2^30 choices");
  const int n = (int)(tokens * choices);
  if (!offsets || (n > 0 && (!ids->ptr || !order || !inverse))) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "group_rows: null pointer");
  const IdSource src{ids->ptr, ids->dtype == MOYE_U64, ids->stride[0], ids->rank == 2 ? ids->stride[1] : 0, (int)choices};
  const int smem = (kGroupWarps + 2) * groups * 4;
  if (int rc = configure_once(h, group_rows_kernel, (kGroupWarps + 2) * kMaxGroups * 4)) return rc;
  cudaLaunchConfig_t cfg = {};
  const unsigned ctas = n > 4096 ? 8 : 1;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kGroupThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = launch_without_pdl() ? 1 : 2;
  MOYE_CUDA(cudaLaunchKernelEx(&cfg, group_rows_kernel, src, n, groups, order, offsets, inverse));
  return MOYE_OK;
}

// ---------------------------------------------------------------------------------------------- rows there and back
template <typename T>
__device__ __forceinline__ float row_elem_to_float(T v);
template <>
__device__ __forceinline__ float row_elem_to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float row_elem_to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float row_elem_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T float_to_row_elem(float f);
template <>
__device__ __forceinline__ float float_to_row_elem<float>(float f) { return f; }
template <>
__device__ __forceinline__ __half float_to_row_elem<__half>(float f) { return __float2half_rn(f); }
template <>
__device__ __forceinline__ __nv_bfloat16 float_to_row_elem<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }

// `V` elements moved as one access: 16 bytes where every row starts on a 16-byte boundary, single elements otherwise.
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T e[V];
};

__device__ __forceinline__ float load_weight(const void* w, int dtype, long long i) {
  if (dtype == MOYE_F32) return static_cast<const float*>(w)[i];
  if (dtype == MOYE_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}
__device__ __forceinline__ void store_weight(void* w, int dtype, long long i, float v) {
  if (dtype == MOYE_F32) static_cast<float*>(w)[i] = v;
  else if (dtype == MOYE_F16) static_cast<__half*>(w)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
}

struct RowArgs {
  int tokens, choices, positions;  // positions: rows of the sorted side; an `inverse` outside them counts as dropped
  long long packs;                 // packs per row
  long long pitch_token, pitch_sorted, pitch_dsorted;  // elements
  const int* inverse;
  const void* weights;
  int w_dtype;
  long long ws_token, ws_choice;
  void* dweights;
  long long dws_token, dws_choice;
};

constexpr int kRowPacks = 4;  // packs a lane holds at once

// One warp takes kRowPacks * 32 packs of one token's row.
template <typename T, int V>
__global__ void __launch_bounds__(256)
gather_rows_kernel(T* dst, const T* src, const RowArgs g) {
  using P = Pack<T, V>;
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long parts = (g.packs + 32 * kRowPacks - 1) / (32 * kRowPacks);
  const long long items = parts * g.tokens, step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long it = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += step) {
    const long long t = it / parts, p0 = (it - t * parts) * (32 * kRowPacks) + lane;
    const P* row = reinterpret_cast<const P*>(src + t * g.pitch_token);
    P v[kRowPacks];
#pragma unroll
    for (int i = 0; i < kRowPacks; ++i)
      if (p0 + i * 32 < g.packs) v[i] = row[p0 + i * 32];
    for (int j = 0; j < g.choices; ++j) {
      const int pos = __ldg(g.inverse + t * g.choices + j);
      if (static_cast<unsigned>(pos) >= static_cast<unsigned>(g.positions)) continue;
      P* out = reinterpret_cast<P*>(dst + pos * g.pitch_sorted);
#pragma unroll
      for (int i = 0; i < kRowPacks; ++i)
        if (p0 + i * 32 < g.packs) out[p0 + i * 32] = v[i];
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(256)
combine_rows_kernel(T* dst, const T* src, const RowArgs g) {
  using P = Pack<T, V>;
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long parts = (g.packs + 32 * kRowPacks - 1) / (32 * kRowPacks);
  const long long items = parts * g.tokens, step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long it = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += step) {
    const long long t = it / parts, p0 = (it - t * parts) * (32 * kRowPacks) + lane;
    float acc[kRowPacks][V];
#pragma unroll
    for (int i = 0; i < kRowPacks; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[i][e] = 0.f;
    for (int j = 0; j < g.choices; ++j) {
      const int pos = __ldg(g.inverse + t * g.choices + j);
      if (static_cast<unsigned>(pos) >= static_cast<unsigned>(g.positions)) continue;
      const float w = g.weights ? load_weight(g.weights, g.w_dtype, t * g.ws_token + j * g.ws_choice) : 1.f;
      const P* in = reinterpret_cast<const P*>(src + pos * g.pitch_sorted);
      P v[kRowPacks];
#pragma unroll
      for (int i = 0; i < kRowPacks; ++i)
        if (p0 + i * 32 < g.packs) v[i] = in[p0 + i * 32];
#pragma unroll
      for (int i = 0; i < kRowPacks; ++i)
        if (p0 + i * 32 < g.packs)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[i][e] += w * row_elem_to_float<T>(v[i].e[e]);
    }
    P* out = reinterpret_cast<P*>(dst + t * g.pitch_token);
#pragma unroll
    for (int i = 0; i < kRowPacks; ++i)
      if (p0 + i * 32 < g.packs) {
        P v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.e[e] = float_to_row_elem<T>(acc[i][e]);
        out[p0 + i * 32] = v;
      }
  }
}

// One CTA of 128 threads per token: the dot products run over the whole row.
template <typename T, int V>
__global__ void __launch_bounds__(128)
combine_rows_grad_kernel(T* dsrc, const T* ddst, const T* src, const RowArgs g) {
  using P = Pack<T, V>;
  constexpr int NW = 4, CH = 8;  // choices taken at once
  __shared__ float part[NW][CH];
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int t = blockIdx.x; t < g.tokens; t += gridDim.x) {
    const P* dy = reinterpret_cast<const P*>(ddst + t * g.pitch_token);
    for (int j0 = 0; j0 < g.choices; j0 += CH) {
      float dot[CH];
#pragma unroll
      for (int j = 0; j < CH; ++j) dot[j] = 0.f;
      for (long long p0 = tid; p0 < g.packs; p0 += 128) {
        const P d = dy[p0];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          if (j0 + j >= g.choices) break;
          const int pos = __ldg(g.inverse + (long long)t * g.choices + j0 + j);
          if (static_cast<unsigned>(pos) >= static_cast<unsigned>(g.positions)) continue;
          const float w = g.weights ? load_weight(g.weights, g.w_dtype, t * g.ws_token + (j0 + j) * g.ws_choice) : 1.f;
          const P y = reinterpret_cast<const P*>(src + pos * g.pitch_sorted)[p0];
          P o;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float de = row_elem_to_float<T>(d.e[e]);
            dot[j] += de * row_elem_to_float<T>(y.e[e]);
            o.e[e] = float_to_row_elem<T>(w * de);
          }
          reinterpret_cast<P*>(dsrc + pos * g.pitch_dsorted)[p0] = o;
        }
      }
#pragma unroll
      for (int j = 0; j < CH; ++j) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(~0u, dot[j], d);
        if (lane == 0) part[warp][j] = dot[j];
      }
      __syncthreads();
      if (tid < CH && j0 + tid < g.choices) {
        const float s = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
        store_weight(g.dweights, g.w_dtype, t * g.dws_token + (j0 + tid) * g.dws_choice, s);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------- host side
static int check_rows(const char* who, const moye_tensor_t* token_side, const moye_tensor_t* sorted_side, int choices) {
  if (token_side->rank != 2 || sorted_side->rank != 2) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: arrays must be rank 2", who);
  if (token_side->dtype != sorted_side->dtype) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "%s: element types differ", who);
  const long long tokens = token_side->shape[0], width = token_side->shape[1];
  if (tokens < 0 || width < 0 || choices < 1) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: negative extent", who);
  if (tokens > INT32_MAX / 2 / choices) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "%s: more than 2^30 choices", who);
  if (sorted_side->shape[0] != tokens * choices || sorted_side->shape[1] != width)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: %lld tokens of width %lld with %d choices need a sorted side of (%lld, %lld), got (%lld, %lld)",
              who, tokens, width, choices, tokens * choices, width, (long long)sorted_side->shape[0], (long long)sorted_side->shape[1]);
  for (const moye_tensor_t* t : {token_side, sorted_side}) {
    if (t->shape[1] > 1 && t->stride[1] != 1) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows must be contiguous", who);
    if (t->shape[0] > 1 && t->stride[0] < t->shape[1]) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows overlap", who);
  }
  return MOYE_OK;
}

static bool overlap(const moye_tensor_t* a, const moye_tensor_t* b) {
  auto span = [](const moye_tensor_t* t) { return ((t->shape[0] - 1) * t->stride[0] + t->shape[1]) * (long long)dtype_bytes(t->dtype); };
  const char *pa = static_cast<const char*>(a->ptr), *pb = static_cast<const char*>(b->ptr);
  return pa < pb + span(b) && pb < pa + span(a);
}

static bool rows_on_16_bytes(const moye_tensor_t* t) {
  const int eb = dtype_bytes(t->dtype);
  return (reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && (t->shape[1] * eb) % 16 == 0 &&
         (t->shape[0] <= 1 || (t->stride[0] * eb) % 16 == 0);
}

static unsigned row_grid(moye_b200_ctx* h, const RowArgs& g) {
  const long long items = (g.packs + 32 * kRowPacks - 1) / (32 * kRowPacks) * g.tokens;
  const long long cap = (long long)h->num_sms * 8, blocks = (items + 7) / 8;
  return (unsigned)(blocks < cap ? blocks : cap);
}

int launch_gather_rows(moye_b200_ctx* h, const moye_tensor_t* dst, const moye_tensor_t* src, const int* inverse, int choices,
                       cudaStream_t stream) {
  if (int rc = check_rows("gather_rows", src, dst, choices)) return rc;
  const int eb = dtype_bytes(src->dtype);
  if (eb != 1 && eb != 2 && eb != 4 && eb != 8) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "gather_rows: elements of 1, 2, 4 or 8 bytes");
  if (src->shape[0] == 0 || src->shape[1] == 0) return MOYE_OK;
  if (!dst->ptr || !src->ptr || !inverse) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gather_rows: null pointer");
  if (overlap(dst, src)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gather_rows: dst and src overlap");
  RowArgs g = {};
  g.tokens = (int)src->shape[0];
  g.choices = choices;
  g.positions = (int)dst->shape[0];
  g.inverse = inverse;
  auto go = [&](auto elem, auto v) -> int {
    using T = decltype(elem);
    constexpr int V = decltype(v)::value;
    g.packs = src->shape[1] / V;
    g.pitch_token = src->stride[0];
    g.pitch_sorted = dst->stride[0];
    MOYE_CUDA(launch_dependent(gather_rows_kernel<T, V>, dim3(row_grid(h, g)), dim3(256), 0, stream, static_cast<T*>(dst->ptr),
                               static_cast<const T*>(src->ptr), g));
    return MOYE_OK;
  };
  const bool wide = rows_on_16_bytes(src) && rows_on_16_bytes(dst);
  switch (eb) {
    case 1: return wide ? go(uint8_t(), std::integral_constant<int, 16>()) : go(uint8_t(), std::integral_constant<int, 1>());
    case 2: return wide ? go(uint16_t(), std::integral_constant<int, 8>()) : go(uint16_t(), std::integral_constant<int, 1>());
    case 4: return wide ? go(uint32_t(), std::integral_constant<int, 4>()) : go(uint32_t(), std::integral_constant<int, 1>());
    default: return wide ? go(uint64_t(), std::integral_constant<int, 2>()) : go(uint64_t(), std::integral_constant<int, 1>());
  }
}

static int check_weights(const char* who, const moye_tensor_t* w, long long tokens, int choices) {
  if (w->dtype != MOYE_F32 && w->dtype != MOYE_F16 && w->dtype != MOYE_BF16)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "%s: weights must be f32, f16 or bf16", who);
  if (w->rank != 2 || w->shape[0] != tokens || w->shape[1] != choices)
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "%s: weights must be (%lld, %d)", who, tokens, choices);
  if (!w->ptr && tokens > 0) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "%s: null pointer", who);
  return MOYE_OK;
}

// Calls f(T(), integral_constant<int, V>()) for a float element type.
template <typename F>
static int for_float_rows(const char* who, int dtype, bool wide, F f) {
  switch (dtype) {
    case MOYE_F32: return wide ? f(float(), std::integral_constant<int, 4>()) : f(float(), std::integral_constant<int, 1>());
    case MOYE_F16: return wide ? f(__half(), std::integral_constant<int, 8>()) : f(__half(), std::integral_constant<int, 1>());
    case MOYE_BF16:
      return wide ? f(__nv_bfloat16(), std::integral_constant<int, 8>()) : f(__nv_bfloat16(), std::integral_constant<int, 1>());
    default: MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "%s: element type %d is not supported (f32, f16, bf16)", who, dtype);
  }
}

int launch_combine_rows(moye_b200_ctx* h, const moye_tensor_t* dst, const moye_tensor_t* src, const moye_tensor_t* weights,
                        const int* inverse, int choices, cudaStream_t stream) {
  if (int rc = check_rows("combine_rows", dst, src, choices)) return rc;
  if (weights)
    if (int rc = check_weights("combine_rows", weights, dst->shape[0], choices)) return rc;
  if (dst->shape[0] == 0 || dst->shape[1] == 0) return MOYE_OK;
  if (!dst->ptr || !src->ptr || !inverse) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows: null pointer");
  if (overlap(dst, src)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows: dst and src overlap");
  RowArgs g = {};
  g.tokens = (int)dst->shape[0];
  g.choices = choices;
  g.positions = (int)src->shape[0];
  g.inverse = inverse;
  g.pitch_token = dst->stride[0];
  g.pitch_sorted = src->stride[0];
  if (weights) {
    g.weights = weights->ptr;
    g.w_dtype = weights->dtype;
    g.ws_token = weights->stride[0];
    g.ws_choice = weights->stride[1];
  }
  return for_float_rows("combine_rows", dst->dtype, rows_on_16_bytes(dst) && rows_on_16_bytes(src), [&](auto elem, auto v) -> int {
    using T = decltype(elem);
    constexpr int V = decltype(v)::value;
    g.packs = dst->shape[1] / V;
    MOYE_CUDA(launch_dependent(combine_rows_kernel<T, V>, dim3(row_grid(h, g)), dim3(256), 0, stream, static_cast<T*>(dst->ptr),
                               static_cast<const T*>(src->ptr), g));
    return MOYE_OK;
  });
}

int launch_combine_rows_grad(moye_b200_ctx* h, const moye_tensor_t* dsrc, const moye_tensor_t* dweights, const moye_tensor_t* ddst,
                             const moye_tensor_t* src, const moye_tensor_t* weights, const int* inverse, int choices,
                             cudaStream_t stream) {
  if (int rc = check_rows("combine_rows_grad", ddst, src, choices)) return rc;
  if (int rc = check_rows("combine_rows_grad", ddst, dsrc, choices)) return rc;
  if (int rc = check_weights("combine_rows_grad", weights, ddst->shape[0], choices)) return rc;
  if (int rc = check_weights("combine_rows_grad", dweights, ddst->shape[0], choices)) return rc;
  if (weights->dtype != dweights->dtype) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "combine_rows_grad: weights and dweights differ in type");
  if (ddst->shape[0] == 0) return MOYE_OK;
  if (ddst->shape[1] == 0) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_SHAPE, "combine_rows_grad: rows of width 0");
  if (!dsrc->ptr || !ddst->ptr || !src->ptr || !inverse) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows_grad: null pointer");
  if (overlap(dsrc, src) || overlap(dsrc, ddst)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows_grad: dsrc overlaps an input");
  RowArgs g = {};
  g.tokens = (int)ddst->shape[0];
  g.choices = choices;
  g.positions = (int)src->shape[0];
  g.inverse = inverse;
  g.pitch_token = ddst->stride[0];
  g.pitch_sorted = src->stride[0];
  g.pitch_dsorted = dsrc->stride[0];
  g.weights = weights->ptr;
  g.w_dtype = weights->dtype;
  g.ws_token = weights->stride[0];
  g.ws_choice = weights->stride[1];
  g.dweights = dweights->ptr;
  g.dws_token = dweights->stride[0];
  g.dws_choice = dweights->stride[1];
  const bool wide = rows_on_16_bytes(ddst) && rows_on_16_bytes(src) && rows_on_16_bytes(dsrc);
  return for_float_rows("combine_rows_grad", ddst->dtype, wide, [&](auto elem, auto v) -> int {
    using T = decltype(elem);
    constexpr int V = decltype(v)::value;
    g.packs = ddst->shape[1] / V;
    const long long cap = (long long)h->num_sms * 16;
    const unsigned blocks = (unsigned)(g.tokens < cap ? g.tokens : cap);
    MOYE_CUDA(launch_dependent(combine_rows_grad_kernel<T, V>, dim3(blocks), dim3(128), 0, stream, static_cast<T*>(dsrc->ptr),
                               static_cast<const T*>(ddst->ptr), static_cast<const T*>(src->ptr), g));
    return MOYE_OK;
  });
}

}  // namespace moye
