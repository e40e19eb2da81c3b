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
// same bits on every run.  They are bound by memory: (T + n) rows for gather and combine, (T + 2n) for the gradient
// (16384 tokens x 8, width 2048 bf16: gather 6.0 TB/s, combine 5.9; 8192 x 2, width 4096: gradient 5.8).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdlib>
#include <numeric>

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
  int packed;  // entry i lies at i * s_choice
  long long s_token, s_choice;
  int choices;
};
constexpr int kIdBatch = 8;   // ids a lane requests at once: the walk is bound by the latency of these loads

__device__ __forceinline__ int load_id(const IdSource& ids, int i, int groups) {
  long long at = i * ids.s_choice;
  if (!ids.packed) {
    const int t = i / ids.choices, j = i - t * ids.choices;
    at = t * ids.s_token + j * ids.s_choice;
  }
  const long long v = ids.is64 ? static_cast<const long long*>(ids.ptr)[at] : static_cast<const int*>(ids.ptr)[at];
  return v >= 0 && v < groups ? static_cast<int>(v) : -1;
}

__device__ __forceinline__ int ld_remote_i32(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// The lanes whose key equals this lane's, a ballot per bit of the key (11 at most).  `__match_any_sync` does the same in
// one instruction whose time grows with the number of different keys: 131072 choices among 128 groups took 29 us with it.
__device__ __forceinline__ unsigned same_key(int key, int bits) {
  unsigned peers = ~0u;
  for (int b = 0; b < bits; ++b) {
    const bool one = (key >> b) & 1;
    const unsigned set = __ballot_sync(~0u, one);
    peers &= one ? set : ~set;
  }
  return peers;
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
  const int key_bits = 32 - __clz(groups);
  int id[kIdBatch];
  for (int b = b0; b < b1; b += kIdBatch) {
#pragma unroll
    for (int u = 0; u < kIdBatch; ++u) {
      const int i = (b + u) * 32 + lane;
      id[u] = b + u < b1 && i < n ? load_id(ids, i, groups) : -1;
    }
#pragma unroll
    for (int u = 0; u < kIdBatch; ++u)
      if (id[u] >= 0) atomicAdd(&mine[id[u]], 1);
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
  for (int b = b0; b < b1; b += kIdBatch) {
    if (b1 - b0 > kIdBatch) {  // else the counting walk has left them in place
#pragma unroll
      for (int u = 0; u < kIdBatch; ++u) {
        const int i = (b + u) * 32 + lane;
        id[u] = b + u < b1 && i < n ? load_id(ids, i, groups) : -1;
      }
    }
#pragma unroll
    for (int u = 0; u < kIdBatch; ++u) {
      if (b + u >= b1) break;
      const int i = (b + u) * 32 + lane;
      const unsigned peers = same_key(id[u] < 0 ? groups : id[u], key_bits);
      const int ahead = __popc(peers & ((1u << lane) - 1));
      int pos = -1;
      if (id[u] >= 0) pos = base[id[u]] + mine[id[u]] + ahead;
      __syncwarp();
      if (id[u] >= 0 && ahead == 0) mine[id[u]] += __popc(peers);
      __syncwarp();
      if (i < n) {
        inverse[i] = pos;
        if (pos >= 0) order[pos] = i;
      }
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
  IdSource src;
  src.ptr = ids->ptr;
  src.is64 = ids->dtype == MOYE_U64;
  src.s_token = ids->stride[0];
  src.s_choice = choices > 1 ? ids->stride[1] : ids->stride[0];
  src.packed = choices == 1 || src.s_token == choices * src.s_choice;
  src.choices = (int)choices;
  const int smem = (kGroupWarps + 2) * groups * 4;
  if (int rc = configure_once(h, group_rows_kernel, (kGroupWarps + 2) * kMaxGroups * 4)) return rc;
  cudaLaunchConfig_t cfg = {};
  // One CTA while its warps have at most 4 batches of 32 choices each, then 8; beyond 32768 choices 16, if the device holds
  // a cluster of 16 (131072 choices, 128 groups, launch included: 25 us with 8 CTAs, 18 with 16, bound by their own instructions:
  // issue slots 54 % used)
  unsigned ctas = n > 4096 ? 8 : 1;
  if (n > 32768 && clusters_that_fit(h, group_rows_kernel, 16, kGroupThreads, (kGroupWarps + 2) * kMaxGroups * 4) > 0) ctas = 16;
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
struct Pack {
  using Raw = typename std::conditional<V != 1, uint4,
              typename std::conditional<sizeof(T) == 8, uint2,
              typename std::conditional<sizeof(T) == 4, uint32_t,
              typename std::conditional<sizeof(T) == 2, uint16_t, uint8_t>::type>::type>::type>::type;
  static_assert(V == 1 || V * sizeof(T) == 16, "an access is one element or 16 bytes");
  Raw raw;
  __device__ __forceinline__ void load(const T* row, long long i) { raw = reinterpret_cast<const Raw*>(row)[i]; }
  __device__ __forceinline__ void store(T* row, long long i) const { reinterpret_cast<Raw*>(row)[i] = raw; }
  __device__ __forceinline__ float at(int e) const { return row_elem_to_float<T>(reinterpret_cast<const T*>(&raw)[e]); }
  __device__ __forceinline__ void set(int e, float f) { reinterpret_cast<T*>(&raw)[e] = float_to_row_elem<T>(f); }
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

// Accesses a lane has under way: kept near 8 of 16 bytes, which at the resident warps covers the latency of memory.
template <int V>
__host__ __device__ constexpr int gather_packs() { return V == 1 ? 8 : 4; }  // packs of a token's row a lane holds
// combine and its gradient request the rows of U choices at once, 2 for one or two choices and 4 for more, N accesses of
// each per thread.  Requests of missing choices are wasted (2 choices, 8192 rows of 4096 bf16: combine 58 us with U = 4);
// more accesses in flight than this cost more in resident CTAs than they hide (the same with U = 2: 39 us with N = 2, 52
// with 4, 59 with 8; 8 choices, 16384 rows of 2048: 103 us with U x N = 8, 105 with 4, 130 with 16).  The gradient reads
// one row more and takes N = 4 (58 us, 59 with 2, 74 with 8).
template <int V>
__host__ __device__ constexpr int combine_packs() { return V == 1 ? 4 : 2; }
template <int V, int U>
__host__ __device__ constexpr int grad_packs() { return (V == 1 ? 16 : 8) / U; }

// Position and weight of up to 32 choices of a token, one per lane; a dropped choice has position -1.
struct Choices {
  int pos;
  float w;
  __device__ __forceinline__ Choices(const RowArgs& g, long long t, int j0, int lane) : pos(-1), w(1.f) {
    const int j = j0 + lane;
    if (j < g.choices && t < g.tokens) {
      pos = __ldg(g.inverse + t * g.choices + j);
      if (g.weights) w = load_weight(g.weights, g.w_dtype, t * g.ws_token + j * g.ws_choice);
    }
    if (static_cast<unsigned>(pos) >= static_cast<unsigned>(g.positions)) pos = -1;
  }
};

// One warp takes N * 32 packs of one token's row.
template <typename T, int V>
__global__ void __launch_bounds__(256)
gather_rows_kernel(T* dst, const T* src, const RowArgs g) {
  using P = Pack<T, V>;
  constexpr int N = gather_packs<V>();
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int parts = (int)((g.packs + 32 * N - 1) / (32 * N));
  const int it = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long t = it / parts, p0 = (long long)(it - (int)t * parts) * (32 * N) + lane;
  if (t >= g.tokens) return;
  P v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i].load(src + t * g.pitch_token, min(p0 + i * 32, g.packs - 1));
  for (int j0 = 0; j0 < g.choices; j0 += 32) {
    const Choices c(g, t, j0, lane);
    for (int j = 0; j < 32 && j0 + j < g.choices; ++j) {
      const int pos = __shfl_sync(~0u, c.pos, j);
      if (pos < 0) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (p0 + i * 32 < g.packs) v[i].store(dst + pos * g.pitch_sorted, p0 + i * 32);
    }
  }
}

// One CTA of 128 threads per token, a thread N packs of its row at a time.
template <typename T, int V, int U>
__global__ void __launch_bounds__(128)
combine_rows_kernel(T* dst, const T* src, const RowArgs g) {
  using P = Pack<T, V>;
  constexpr int N = combine_packs<V>();
  griddep_launch();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long t = blockIdx.x;
  const Choices first(g, t, 0, lane);
  for (long long base = 0; base < g.packs; base += 128 * N) {
    const long long p0 = base + threadIdx.x;
    float acc[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[i][e] = 0.f;
    for (int j0 = 0; j0 < g.choices; j0 += 32) {
      Choices c = first;
      if (j0) c = Choices(g, t, j0, lane);
      const int here = min(32, g.choices - j0);
      for (int j = 0; j < here; j += U) {
        P v[U][N];
        int pos[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          pos[u] = __shfl_sync(~0u, c.pos, (j + u) & 31);
          if (j + u >= here) pos[u] = -1;
          // no branch around a load: a dropped choice reads row 0 and a lane behind the row its last pack, for nothing
          const T* in = src + max(pos[u], 0) * g.pitch_sorted;
#pragma unroll
          for (int i = 0; i < N; ++i) v[u][i].load(in, min(p0 + i * 128, g.packs - 1));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float w = __shfl_sync(~0u, c.w, (j + u) & 31);
          if (pos[u] < 0) continue;
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[i][e] += w * v[u][i].at(e);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (p0 + i * 128 < g.packs) {
        P v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.set(e, acc[i][e]);
        v.store(dst + t * g.pitch_token, p0 + i * 128);
      }
  }
}

// One CTA of 128 threads per token: the dot products run over the whole row.
template <typename T, int V, int U>
__global__ void __launch_bounds__(128)
combine_rows_grad_kernel(T* dsrc, const T* ddst, const T* src, const RowArgs g) {
  using P = Pack<T, V>;
  constexpr int N = grad_packs<V, U>(), NW = 4;
  __shared__ float part[NW][U];
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long t = blockIdx.x;
  const T* dy = ddst + t * g.pitch_token;
  for (int j0 = 0; j0 < g.choices; j0 += 32) {
    const Choices c(g, t, j0, lane);
    const int here = min(32, g.choices - j0);
    for (int j = 0; j < here; j += U) {
      float dot[U], w[U];
      int pos[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        dot[u] = 0.f;
        pos[u] = __shfl_sync(~0u, c.pos, (j + u) & 31);
        w[u] = __shfl_sync(~0u, c.w, (j + u) & 31);
        if (j + u >= here) pos[u] = -1;
      }
      for (long long p0 = tid; p0 < g.packs; p0 += 128 * N) {
        P d[N], y[U][N];
#pragma unroll
        for (int i = 0; i < N; ++i) d[i].load(dy, min(p0 + i * 128, g.packs - 1));
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) y[u][i].load(src + max(pos[u], 0) * g.pitch_sorted, min(p0 + i * 128, g.packs - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (pos[u] < 0) continue;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (p0 + i * 128 >= g.packs) continue;
            P o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float de = d[i].at(e);
              dot[u] += de * y[u][i].at(e);
              o.set(e, w[u] * de);
            }
            o.store(dsrc + pos[u] * g.pitch_dsorted, p0 + i * 128);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[u] += __shfl_xor_sync(~0u, dot[u], d);
        if (lane == 0) part[warp][u] = dot[u];
      }
      __syncthreads();
      if (tid < U && j + tid < here) {
        const float s = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
        store_weight(g.dweights, g.w_dtype, t * g.dws_token + (j0 + j + tid) * g.dws_choice, s);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------- host side
// Rows of an array that is only read may lie on one another (a broadcast gradient); `written` is the one that is not.
static int check_rows(const char* who, const moye_tensor_t* token_side, const moye_tensor_t* sorted_side, const moye_tensor_t* written,
                      int choices) {
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
    if (t->shape[0] > 1 && t->stride[0] < (t == written ? t->shape[1] : 0))
      MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "%s: rows %s", who, t == written ? "of an output overlap" : "with a negative pitch");
  }
  return MOYE_OK;
}

static bool rows_on_16_bytes(const moye_tensor_t* t) {
  const int eb = dtype_bytes(t->dtype);
  return (reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && (t->shape[1] * eb) % 16 == 0 &&
         (t->shape[0] <= 1 || (t->stride[0] * eb) % 16 == 0);
}

// CTAs of 8 warps, a warp per `packs_per_lane * 32` packs of a row.  More tokens than a grid holds are refused.
static int row_grid(const char* who, const RowArgs& g, int packs_per_lane, unsigned* grid) {
  const long long warps = (g.packs + 32 * packs_per_lane - 1) / (32 * packs_per_lane) * g.tokens, blocks = (warps + 7) / 8;
  if (warps > INT32_MAX / 2) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "%s: too many rows of this width", who);
  *grid = (unsigned)blocks;
  return MOYE_OK;
}

int launch_gather_rows(moye_b200_ctx*, const moye_tensor_t* dst, const moye_tensor_t* src, const int* inverse, int choices,
                       cudaStream_t stream) {
  if (int rc = check_rows("gather_rows", src, dst, dst, choices)) return rc;
  const int eb = dtype_bytes(src->dtype);
  if (eb != 1 && eb != 2 && eb != 4 && eb != 8) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "gather_rows: elements of 1, 2, 4 or 8 bytes");
  if (src->shape[0] == 0 || src->shape[1] == 0) return MOYE_OK;
  if (!dst->ptr || !src->ptr || !inverse) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gather_rows: null pointer");
  if (rows_overlap(dst, src)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gather_rows: dst and src overlap");
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
    unsigned grid;
    if (int rc = row_grid("gather_rows", g, gather_packs<V>(), &grid)) return rc;
    MOYE_CUDA(launch_dependent(gather_rows_kernel<T, V>, dim3(grid), dim3(256), 0, stream, static_cast<T*>(dst->ptr),
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

int launch_combine_rows(moye_b200_ctx*, const moye_tensor_t* dst, const moye_tensor_t* src, const moye_tensor_t* weights,
                        const int* inverse, int choices, cudaStream_t stream) {
  if (int rc = check_rows("combine_rows", dst, src, dst, choices)) return rc;
  if (weights)
    if (int rc = check_weights("combine_rows", weights, dst->shape[0], choices)) return rc;
  if (dst->shape[0] == 0 || dst->shape[1] == 0) return MOYE_OK;
  if (!dst->ptr || !src->ptr || !inverse) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows: null pointer");
  if (rows_overlap(dst, src)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows: dst and src overlap");
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
    auto run = [&](auto u) -> int {
      constexpr int U = decltype(u)::value;
      MOYE_CUDA(launch_dependent(combine_rows_kernel<T, V, U>, dim3((unsigned)g.tokens), dim3(128), 0, stream, static_cast<T*>(dst->ptr),
                                 static_cast<const T*>(src->ptr), g));
      return MOYE_OK;
    };
    return choices <= 2 ? run(std::integral_constant<int, 2>()) : run(std::integral_constant<int, 4>());
  });
}

int launch_combine_rows_grad(moye_b200_ctx*, const moye_tensor_t* dsrc, const moye_tensor_t* dweights, const moye_tensor_t* ddst,
                             const moye_tensor_t* src, const moye_tensor_t* weights, const int* inverse, int choices,
                             cudaStream_t stream) {
  if (int rc = check_rows("combine_rows_grad", ddst, src, nullptr, choices)) return rc;
  if (int rc = check_rows("combine_rows_grad", ddst, dsrc, dsrc, choices)) return rc;
  if (int rc = check_weights("combine_rows_grad", weights, ddst->shape[0], choices)) return rc;
  if (int rc = check_weights("combine_rows_grad", dweights, ddst->shape[0], choices)) return rc;
  // any strides that give every choice an element of its own (no broadcast output): two meet at the least common multiple
  const long long T = dweights->shape[0], st = std::llabs(dweights->stride[0]), sc = std::llabs(dweights->stride[1]), both = std::gcd(st, sc);
  if ((T > 1 && st == 0) || (choices > 1 && sc == 0) || (T > 1 && choices > 1 && sc / both < T && st / both < choices))
    MOYE_FAIL(MOYE_ERR_UNSUPPORTED_LAYOUT, "combine_rows_grad: elements of dweights overlap");
  if (weights->dtype != dweights->dtype) MOYE_FAIL(MOYE_ERR_UNSUPPORTED_DTYPE, "combine_rows_grad: weights and dweights differ in type");
  if (ddst->shape[0] == 0) return MOYE_OK;
  const bool empty = ddst->shape[1] == 0;  // no rows to read or write: the weights' gradients are empty sums
  if (!inverse || (!empty && (!dsrc->ptr || !ddst->ptr || !src->ptr))) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows_grad: null pointer");
  if (!empty && (rows_overlap(dsrc, src) || rows_overlap(dsrc, ddst))) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "combine_rows_grad: dsrc overlaps an input");
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
    auto run = [&](auto u) -> int {
      MOYE_CUDA(launch_dependent(combine_rows_grad_kernel<T, V, decltype(u)::value>, dim3((unsigned)g.tokens), dim3(128), 0, stream,
                                 static_cast<T*>(dsrc->ptr), static_cast<const T*>(ddst->ptr), static_cast<const T*>(src->ptr), g));
      return MOYE_OK;
    };
    return choices <= 2 ? run(std::integral_constant<int, 2>()) : run(std::integral_constant<int, 4>());
  });
}

}  // namespace moye
