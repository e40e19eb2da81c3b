// Low-rank adapters of many requests beside a shared projection:
//
//   D[i] = C[i] + s[a] * (X[i] . A[a]^T) . B[a]^T        X (rows, K), A (adapters, R, K), B (adapters, N, R), C, D (rows, N)
//
// where a = adapters[q] is the adapter of the request q that row i belongs to: offsets[q] <= i < offsets[q+1], or
// q = i when no offsets are given (a decoding step).  An adapter number outside 0..adapters-1 means none: D[i] = C[i].
// Rows outside every request are left as they were.  A border below an earlier one counts as that one, so that requests
// never share a row: both kernels then take a row once, by the same request.  No counterpart in the reference.
//
// The product of rank R between the two factors never leaves the chip: a thread-block cluster takes a row, CTA c of it
// a slice of K for the first factor; the partial R-vectors meet through distributed shared memory (fp32, summed in CTA
// order, so the result does not depend on timing); then CTA c takes a slice of N for the second factor.  82 to 86 clusters
// are resident at once (5 CTAs per SM by registers): K = N = 4096, R = 16, up to 82 rows 5.5 us, 128 rows two waves, 9.5.
#include "gemm_common.cuh"

namespace moye {

constexpr int kLoraCtas = 8;         // cluster size of the row kernel
constexpr int kLoraThreads = 256;
constexpr int kLoraRowChunk = 512;   // columns of a CTA's slice that meet in shared memory before they are stored
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
__global__ void __launch_bounds__(kLoraThreads, 5)
lora_row_kernel(const LoraArgs g) {
  __shared__ float part[kMaxLoraRank], v[kMaxLoraRank], out[kLoraRowChunk];
  __shared__ int found;
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / kLoraCtas, rank = (int)cluster_ctarank();
  if (g.offsets) {
    // the first request that ends behind the row, unless the row lies before all of them
    if (tid == 0) found = g.requests;
    const int first = __ldg(g.offsets);
    __syncthreads();
    for (int q = tid; q < g.requests; q += kLoraThreads)
      if (row < g.offsets[q + 1]) atomicMin(&found, first <= row ? q : g.requests);
    __syncthreads();
  } else if (tid == 0) {
    found = row;
  }
  __syncthreads();
  const int q = found;
  if (q >= g.requests) return;  // the same in every CTA of the cluster
  const int a = g.which[q];
  const int n0 = (int)((long long)g.n * rank / kLoraCtas), n1 = (int)((long long)g.n * (rank + 1) / kLoraCtas);
  const OutT* c_row = static_cast<const OutT*>(g.C) + row * g.c_pitch;
  OutT* d_row = static_cast<OutT*>(g.D) + row * g.d_pitch;
  if (a < 0 || a >= g.adapters) {
    if (g.C != g.D)
      for (int n = n0 + tid; n < n1; n += kLoraThreads) d_row[n] = c_row[n];
    return;
  }
  const T* b_rows = static_cast<const T*>(g.B) + a * g.b_stride;
  {
    // a warp takes 2 rows of A[a] at a time, two words of 16 bytes of each per lane
    const int kv = g.k / 8, v0 = (int)((long long)kv * rank / kLoraCtas), v1 = (int)((long long)kv * (rank + 1) / kLoraCtas);
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(g.X) + row * g.x_pitch);
    for (int r0 = warp * 2; r0 < g.rank; r0 += kLoraThreads / 16) {  // R is a multiple of 8: both rows exist
      const T* ar = static_cast<const T*>(g.A) + a * g.a_stride + r0 * g.a_pitch;
      float s[2] = {0.f, 0.f};
      for (int i0 = v0; i0 < v1; i0 += 64) {
        uint4 xw[2], aw[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = min(i0 + h * 32 + lane, v1 - 1);
          xw[h] = x[i];
#pragma unroll
          for (int r = 0; r < 2; ++r) aw[r][h] = reinterpret_cast<const uint4*>(ar + r * g.a_pitch)[i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (i0 + h * 32 + lane >= v1) continue;
          float xf[8];
          lora_unpack<T>(xw[h], xf);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float af[8];
            lora_unpack<T>(aw[r][h], af);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[r] += xf[e] * af[e];
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s[r] += __shfl_xor_sync(~0u, s[r], d);
        if (lane == 0) part[r0 + r] = s[r];
      }
    }
  }
  cluster_arrive();
  cluster_wait();  // every CTA's partial vector is in place
  if (tid < kMaxLoraRank) {
    float s = 0.f;
    if (tid < g.rank) {
      for (int c = 0; c < kLoraCtas; ++c) s += ld_remote_f32(mapa_shared(smem_u32(part + tid), c));
      s *= g.scales ? g.scales[a] : 1.f;
    }
    v[tid] = s;
  }
  cluster_arrive();  // this CTA has read the others' parts; it leaves only after they have read its own (below)
  __syncthreads();
  const int words = g.rank / 8;
  if (words <= 4) {  // short rows: one per thread (128 requests, R = 16: 8 us against 11 with the rows shared)
    for (int n = n0 + tid; n < n1; n += kLoraThreads) {
      const uint4* b = reinterpret_cast<const uint4*>(b_rows + n * g.b_pitch);
      const float c = lora_load(c_row + n);
      uint4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = b[min(i, words - 1)];
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= words) break;
        float bf[8];
        lora_unpack<T>(w[i], bf);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += bf[e] * v[i * 8 + e];
      }
      lora_store(d_row + n, c + s);
    }
    cluster_wait();
    return;
  }
  // long rows: `lanes` neighbouring lanes share one, 16 bytes each, so that a warp reads whole rows, 4 batches of them
  // under way (128 requests, R = 64: 28 us against 34 with a row per thread)
  int lanes = 1;
  while (lanes < words) lanes *= 2;
  const int sub = lane & (lanes - 1), per_warp = 32 / lanes, mine = lane / lanes;
  float vf[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) vf[e] = v[sub * 8 + e];
  for (int c0 = n0; c0 < n1; c0 += kLoraRowChunk) {
    const int c1 = min(c0 + kLoraRowChunk, n1);
    // the loop is the warp's, not the lane's: all 32 lanes meet in its shuffles
    for (int nw = c0 + warp * per_warp; nw < c1; nw += 4 * (kLoraThreads / 32) * per_warp) {
      const int n = nw + mine;
      uint4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        w[u] = reinterpret_cast<const uint4*>(b_rows + min(n + u * (kLoraThreads / 32) * per_warp, c1 - 1) * g.b_pitch)[min(sub, words - 1)];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float bf[8], s = 0.f;
        lora_unpack<T>(w[u], bf);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += bf[e] * vf[e];
        if (sub >= words) s = 0.f;
        for (int d = lanes / 2; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        const int at = n + u * (kLoraThreads / 32) * per_warp;
        if (sub == 0 && at < c1) out[at - c0] = s;
      }
    }
    __syncthreads();
    for (int n = c0 + tid; n < c1; n += kLoraThreads) lora_store(d_row + n, lora_load(c_row + n) + out[n - c0]);
    __syncthreads();
  }
  cluster_wait();
}

// ---------------------------------------------------------------------------------------------- requests of several rows
// A cluster of C CTAs takes up to 128 rows of one request.  CTA c multiplies its K blocks of X (128 lanes of tensor
// memory) with A[a] (R columns); with C > 1 the fp32 parts meet through distributed shared memory, CTA c summing 1 / C of
// the rows in CTA order and handing the result to all; every CTA then multiplies it with its 128-column chunks of B[a] and
// adds C.  The product of rank R enters the second multiplication as a sum of 16-bit parts: two parts carry 16 (bf16)
// or 22 (f16) bits, off by 2^-17 of a product where the output's rounding takes 2^-9 (a third part moves 0.04 % of bf16
// outputs by a step, for 9 % of the time); bf16 operands with a Float32 output take three (24 bits).
// A Float32 output also has its sums over K taken out of tensor memory every 512 products, as in gemm_grouped.cu.
// f16 has not the range of the fp32 sums (65504, and steps of 2^-24 near zero): a row is brought to magnitude 1 by a power
// of two first, which the epilogue takes back.
//
// Warp 0 producer, warp 1 MMA issuer, warps 4-11 move the parts and run the epilogue.  The kernel is bound by memory (X and
// C in, D out) and lives on bytes in flight.  The first product has all of shared memory for its ring of K blocks (9 at
// rank 64; with 4 it took 34 us of 16384 rows x 4096); the second has it for chunks of B, the rank-R product and boxes of C:
// the epilogue keeps one to five boxes of 4 KB ahead per warp, a thread holds one row of the accumulator and adds it to the same
// row of the box, which goes out by TMA again.  (C through registers and D by vector stores, on two CTAs per SM: 16384 rows
// of 24 requests, rank 64, 4096 x 4096: 115 us.)
//
// Measured: those 16384 rows 80 us (X streams at 6.3 TB/s, C and D at 5.6; 4 us of start-up, 1.5 of exchange between them),
// 64 requests of 16 rows, R = 64: 43 us against 215 row by row.
//
// Tiles of at most 32 rows turn the second product round: the lanes are the columns of D and the rows its columns, so
// that all warps have work and nothing crosses shared memory.
constexpr int kLoraTileThreads = 384;
enum : int { SITEL_PROD_EMPTY = 171, SITEL_MMA_FULL = 172, SITEL_MMA_V = 173, SITEL_MMA_ACC = 174, SITEL_EPI_V = 175, SITEL_EPI_PARTS = 176, SITEL_EPI_ACC = 177, SITEL_SMEM_BASE = 178, SITEL_EPI_C = 179 };

struct LoraTileArgs {
  LoraArgs g;
  uint32_t idesc1, idesc2;
  int* status;
  int k_stages, k_bytes;                                    // first product: ring of K blocks from offset 0
  int b_stages, b_bytes, v_off, c_off, c_bufs, bar_off;     // second: ring of chunks from 0, then the rest; bytes
};

__device__ __forceinline__ float4 ld_remote_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_remote_u32x2(uint32_t cluster_addr, uint32_t x, uint32_t y) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(cluster_addr), "r"(x), "r"(y) : "memory");
}
// The epilogue's 256 threads meet, all going on or giving up together.
__device__ __forceinline__ bool lora_epi_all(bool mine) { return all_of<256>(1, mine); }

// One 16-byte word of outputs: the input word plus `up` times EPV accumulators.
__device__ __forceinline__ uint4 lora_add(const uint4& c, const uint32_t* v, float up, float*) {
  return make_uint4(__float_as_uint(fmaf(__uint_as_float(v[0]), up, __uint_as_float(c.x))), __float_as_uint(fmaf(__uint_as_float(v[1]), up, __uint_as_float(c.y))),
                    __float_as_uint(fmaf(__uint_as_float(v[2]), up, __uint_as_float(c.z))), __float_as_uint(fmaf(__uint_as_float(v[3]), up, __uint_as_float(c.w))));
}
template <typename T>
__device__ __forceinline__ uint4 lora_add(const uint4& c, const uint32_t* v, float up, T*) {
  float f[8];
  lora_unpack<T>(c, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = fmaf(__uint_as_float(v[e]), up, f[e]);
  return make_uint4(pack_pair<T>(f[0], f[1]), pack_pair<T>(f[2], f[3]), pack_pair<T>(f[4], f[5]), pack_pair<T>(f[6], f[7]));
}

// The powers of two that bring a row whose magnitudes stay below `m` to magnitude 1 (`down`) and back (`up`); 1 where m
// is no number.
__device__ __forceinline__ void lora_range(float m, float& down, float& up) {
  const int e = static_cast<int>(__float_as_uint(m) >> 23);  // m >= 0: the biased exponent
  const int x = min(e, 252);
  down = e == 255 ? 1.f : __uint_as_float(static_cast<uint32_t>(253 - x) << 23);  // 2^(126 - x): m * down is in [1/2, 1)
  up = e == 255 ? 1.f : __uint_as_float(static_cast<uint32_t>(x + 1) << 23);
}

// The request and first row of tile `want`; q = -1 when there are fewer tiles.  All threads of the CTA; `sums` holds one
// int per warp.
__device__ __forceinline__ void lora_find_tile(const LoraArgs& g, int want, int* sums, int* result) {
  const int tid = threadIdx.x, per = (g.requests + kLoraTileThreads - 1) / kLoraTileThreads;
  const int q0 = min(tid * per, g.requests), q1 = min(q0 + per, g.requests);
  auto border = [&](int q) { return min(max(__ldg(g.offsets + q), 0), g.rows); };
  int high = 0;  // the largest border before q0, where that is not border(q0) itself
  auto tiles_of = [&](int q, int& lo, int& hi) {  // in the order of q, from q0 on
    if (q == q0) lo = max(border(q), high);
    else lo = hi;
    hi = max(border(q + 1), lo);
    return (hi - lo + 127) >> 7;
  };
  int before = 0, mine = 0, lo = 0, hi = 0;
  bool back = false;
  auto count = [&]() {  // tiles of this thread's requests, and of its warp's threads before it
    mine = 0;
    for (int q = q0; q < q1; ++q) {
      mine += tiles_of(q, lo, hi);
      back |= hi != border(q + 1);
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(~0u, incl, d);
      if ((tid & 31) >= d) incl += up;
    }
    if ((tid & 31) == 31) sums[tid >> 5] = incl;
    before = incl - mine;
  };
  if (tid == 0) result[0] = -1;
  count();
  if (__syncthreads_or(back)) {
    // a border runs backwards: the largest before each thread's requests, then again
    int top = 0;
    for (int q = q0; q < q1; ++q) top = max(top, border(q));
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) top = max(top, __shfl_up_sync(~0u, top, d));
    if ((tid & 31) == 31) sums[tid >> 5] = top;
    high = __shfl_up_sync(~0u, top, 1);
    if ((tid & 31) == 0) high = 0;
    __syncthreads();
    for (int w = 0; w < (tid >> 5); ++w) high = max(high, sums[w]);
    __syncthreads();
    count();
    __syncthreads();
  }
  for (int w = 0; w < (tid >> 5); ++w) before += sums[w];
  if (before <= want && want < before + mine) {
    for (int q = q0; q < q1; ++q) {
      const int n = tiles_of(q, lo, hi);
      if (want < before + n) {
        result[0] = q;
        result[1] = lo + (want - before) * 128;
        result[2] = min(128, hi - result[1]);
        break;
      }
      before += n;
    }
  }
  __syncthreads();
}

template <typename T, typename OutT, bool VEC, int PARTS>
__global__ void __launch_bounds__(kLoraTileThreads, 1)
lora_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmD, const LoraTileArgs p) {
  const LoraArgs& g = p.g;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // the plan has no slack to align the base by hand
    if (threadIdx.x == 0) atomicCAS(p.status, 0, SITEL_SMEM_BASE);
    return;
  }
  uint8_t* vparts = smem + p.v_off;                          // [part][64-wide block of R][128 rows][128 bytes], swizzled
  uint8_t* cboxes = smem + p.c_off;                          // [8 warps][c_bufs][32 rows][128 bytes], swizzled
  float* parts = reinterpret_cast<float*>(cboxes);           // before that (C > 1): [128][R] fp32
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.bar_off);
  uint64_t *k_full = bars, *k_empty = bars + 12, *b_full = bars + 24, *b_empty = bars + 28, *acc_full = bars + 32, *acc_empty = bars + 34,
           *v_acc = bars + 36, *p_ready = bars + 37, *v_ready = bars + 38, *c_full = bars + 40,  // c_full[8 warps][c_bufs <= 6]
           *v_full = bars + 88, *v_empty = bars + 90;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 39);
  int* scratch = reinterpret_cast<int*>(bars + 92);          // 12 warp sums, then the tile
  float* row_max = reinterpret_cast<float*>(bars + 128);     // [2 sets][128 rows]
  float* row_up = row_max + 256;                             // [128 rows]
  constexpr uint32_t TMEM_COLS = 256;
  constexpr bool RANGE = std::is_same<T, __half>::value, PROMOTE = sizeof(OutT) == 4;
  constexpr int RUN = 8;  // K blocks summed in tensor memory

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  griddep_wait();
  lora_find_tile(g, blockIdx.x / C, scratch, scratch + 12);
  const int q = scratch[12], row0 = scratch[13], nrows = scratch[14];
  if (q < 0) return;  // fewer tiles than clusters; the same in the whole cluster
  // debug build: a tile inside the arrays
  if (!MOYE_DBG_OK(q < g.requests && row0 >= 0 && nrows > 0 && nrows <= 128 && row0 + nrows <= g.rows, p.status, 984)) return;
  const int a = g.which[q];
  const int chunks = (g.n + 127) / 128, kbs = (g.k + 63) / 64;
  const int ch0 = chunks * rank / C, ch1 = chunks * (rank + 1) / C;
  const OutT* c_base = static_cast<const OutT*>(g.C) + row0 * g.c_pitch;
  OutT* d_base = static_cast<OutT*>(g.D) + row0 * g.d_pitch;
  if (a < 0 || a >= g.adapters) {
    if (g.C != g.D) {
      const int n0 = ch0 * 128, n1 = min(ch1 * 128, g.n);
      if constexpr (VEC) {
        constexpr int EPV = 16 / (int)sizeof(OutT);
        for (int r = warp; r < nrows; r += kLoraTileThreads / 32) {
          const OutT* from = c_base + r * g.c_pitch;
          OutT* to = d_base + r * g.d_pitch;
          for (int n = n0 + lane * EPV; n < n1; n += 8 * 32 * EPV) {
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + i * 32 * EPV < n1) v[i] = *reinterpret_cast<const uint4*>(from + n + i * 32 * EPV);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + i * 32 * EPV < n1) *reinterpret_cast<uint4*>(to + n + i * 32 * EPV) = v[i];
          }
        }
      } else {
        for (int r = warp; r < nrows; r += kLoraTileThreads / 32)
          for (int n = n0 + lane; n < n1; n += 32) d_base[r * g.d_pitch + n] = c_base[r * g.c_pitch + n];
      }
    }
    return;
  }
  const int kb0 = kbs * rank / C, kb1 = kbs * (rank + 1) / C;  // at least one block: C <= kbs
  const int rblocks = (g.rank + 63) / 64, rsteps = (g.rank + 15) / 16;
  const int a_bytes = rsteps * 16 * 128;
  const bool turned = nrows <= 32;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < p.k_stages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < p.b_stages; ++s) {
      mbar_init(&b_full[s], 1);
      mbar_init(&b_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], turned ? 4 : 8);
      mbar_init(&v_full[b], 1);
      mbar_init(&v_empty[b], 8);
    }
    mbar_init(v_acc, 1);
    mbar_init(p_ready, C);
    mbar_init(v_ready, C);
    for (int i = 0; i < 8 * p.c_bufs; ++i) mbar_init(&c_full[i], 1);
    fence_mbar_init();
    prefetch_tensormap(&tmX);
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (C > 1) {
    cluster_arrive();
    cluster_wait();  // every CTA's barriers are set up
  }
  tc_fence_after_sync();
  // Only now, with this CTA's tensor memory allocated: a dependent grid that came to sit on this SM earlier could take
  // the columns and hold them while it waits for this grid.
  griddep_launch();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_holder);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer: K blocks, then chunks of B
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait(&k_empty[stage], phase ^ 1, p.status, SITEL_PROD_EMPTY);
        if (!ok) break;
        uint8_t* s = smem + stage * p.k_bytes;
        mbar_arrive_expect_tx(&k_full[stage], 128 * 128 + a_bytes);
        tma_load_2d(s, &tmX, &k_full[stage], kb * 64, row0);
        tma_load_3d(s + 128 * 128, &tmA, &k_full[stage], kb * 64, 0, a);
        if (++stage == p.k_stages) { stage = 0; phase ^= 1; }
      }
      // the chunks lie where the K blocks did
      ok = ok && mbar_wait(v_acc, 0, p.status, SITEL_PROD_EMPTY);
      stage = 0;
      phase = 0;
      for (int ch = ch0; ch < ch1 && ok; ++ch) {
        ok = mbar_wait(&b_empty[stage], phase ^ 1, p.status, SITEL_PROD_EMPTY);
        if (!ok) break;
        mbar_arrive_expect_tx(&b_full[stage], p.b_bytes);
        for (int b = 0; b < rblocks; ++b)
          tma_load_3d(smem + stage * p.b_bytes + b * 128 * 128, &tmB, &b_full[stage], b * 64, ch * 128, a);
        if (++stage == p.b_stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0, run = 0; kb < kb1 && ok; ++run) {
        const int end = PROMOTE ? min(kb + RUN, kb1) : kb1;
        const uint32_t v_tmem = tmem_base + (run & 1) * 128;
        ok = mbar_wait(&v_empty[run & 1], ((run >> 1) & 1) ^ 1, p.status, SITEL_MMA_ACC);
        tc_fence_after_sync();
        for (const int first = kb; kb < end && ok; ++kb) {
          ok = mbar_wait(&k_full[stage], phase, p.status, SITEL_MMA_FULL);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t s = smem_u32(smem + stage * p.k_bytes);
          const uint64_t xd = umma_desc_k_sw128(s), ad = umma_desc_k_sw128(s + 128 * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) tc_mma_ss<KIND_F16>(v_tmem, xd + 2 * k, ad + 2 * k, p.idesc1, (kb > first || k > 0) ? 1u : 0u);
          tc_commit(&k_empty[stage]);
          if (++stage == p.k_stages) { stage = 0; phase ^= 1; }
        }
        if (ok) tc_commit(&v_full[run & 1]);
      }
      if (ok) tc_commit(v_acc);
      stage = 0;
      phase = 0;
      if (ok && ch1 > ch0) ok = mbar_wait_cluster(v_ready, 0, p.status, SITEL_MMA_V);
      fence_proxy_async_smem();
      const uint32_t vs = smem_u32(vparts);
      const uint32_t idesc = p.idesc2 | ((uint32_t)(turned ? (nrows + 15) / 16 * 2 : 16) << 17);
      for (int i = 0; i < ch1 - ch0 && ok; ++i) {
        const int buf = i & 1;
        ok = mbar_wait(&acc_empty[buf], ((i >> 1) & 1) ^ 1, p.status, SITEL_MMA_ACC) && mbar_wait(&b_full[stage], phase, p.status, SITEL_MMA_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t s = smem_u32(smem + stage * p.b_bytes);
        for (int part = 0; part < PARTS; ++part)
          for (int k = 0; k < rsteps; ++k) {
            const uint32_t at = (k >> 2) * (128 * 128) + (k & 3) * 32;  // block of 64, step of 16 inside it
            const uint64_t vd = umma_desc_k_sw128(vs + part * rblocks * (128 * 128) + at), bd = umma_desc_k_sw128(s + at);
            tc_mma_ss<KIND_F16>(tmem_base + buf * 128, turned ? bd : vd, turned ? vd : bd, idesc, (part | k) != 0 ? 1u : 0u);
          }
        tc_commit(&b_empty[stage]);
        tc_commit(&acc_full[buf]);
        if (++stage == p.b_stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ warps 4-11: the rank-R product, then the epilogue
    constexpr int BW = 128 / (int)sizeof(OutT), EPV = 16 / (int)sizeof(OutT);  // columns of a box; elements of 16 bytes
    constexpr int BPC = 64 / BW;                                                // boxes of a warp's 64 columns of a chunk
    const int qd = warp & 3, set = (warp - 4) >> 2, et = (warp - 4) * 32 + lane;  // tensor-memory quarter; half of a chunk's columns
    const int my_row = qd * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(qd * 32) << 16);
    const float scale = g.scales ? __ldg(g.scales + a) : 1.f;
    uint8_t* my_boxes = cboxes + (warp - 4) * p.c_bufs * 4096;
    uint64_t* my_full = c_full + (warp - 4) * p.c_bufs;
    const int nboxes = VEC && !turned && qd * 32 < nrows ? (ch1 - ch0) * BPC : 0;
    auto box_col = [&](int k) { return (ch0 + k / BPC) * 128 + set * 64 + (k % BPC) * BW; };
    auto request = [&](int k, int slot) {  // one lane
      mbar_arrive_expect_tx(&my_full[slot], 4096);
      tma_load_2d(my_boxes + slot * 4096, &tmC, &my_full[slot], box_col(k), row0 + qd * 32);
    };
    // Scale first, then the power of two: their product leaves fp32 where a row is zero or tiny (2^126 * 4), and would make
    // the row's zeros undefined.
    auto scaled = [&](const float4& x, float down) {
      return make_float4(x.x * scale * down, x.y * scale * down, x.z * scale * down, x.w * scale * down);
    };
    // the value of `x` as PARTS 16-bit numbers, the largest first
    auto write_parts = [&](int row, int col, float4 x, auto&& store) {  // 4 columns at once
      float r[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const uint32_t w0 = pack_pair<T>(r[0], r[1]), w1 = pack_pair<T>(r[2], r[3]);
        const float2 f0 = lora_pair<T>(w0), f1 = lora_pair<T>(w1);
        const float f[4] = {f0.x, f0.y, f1.x, f1.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = isinf(f[i]) ? 0.f : r[i] - f[i];  // an infinity has no rest
        store((part * rblocks + (col >> 6)) * (128 * 128) + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 4) * 2, w0, w1);
      }
    };
    // this set's columns of the rank-R product, 16 at a time from 16 set on
    float sums[4][16];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[i][j] = 0.f;
    bool ok = true;
    for (int kb = kb0, run = 0; kb < kb1 && ok; kb += PROMOTE ? RUN : kb1 - kb0, ++run) {
      ok = lora_epi_all(mbar_wait(&v_full[run & 1], (run >> 1) & 1, p.status, SITEL_EPI_V));
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (set + 2 * i < rsteps) {
          uint32_t v[16];
          tmem_ld_x16(t_lane + (run & 1) * 128 + (set + 2 * i) * 16, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[i][j] += __uint_as_float(v[j]);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_empty[run & 1]);
    }
    // A rank that ends inside 16 columns: the products with rows of zeros behind it, undefined where X is infinite, are zero
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((set + 2 * i) * 16 + 8 == g.rank)
#pragma unroll
        for (int j = 8; j < 16; ++j) sums[i][j] = 0.f;
    // the boxes of C lie where the K blocks did
    ok = ok && lora_epi_all(mbar_wait(v_acc, 0, p.status, SITEL_EPI_V));
    if (ok) {
      if (C == 1 && lane == 0)
        for (int k = 0; k < p.c_bufs - 1 && k < nboxes; ++k) request(k, k);
      auto each_4 = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (set + 2 * i < rsteps)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              f((set + 2 * i) * 16 + j, make_float4(sums[i][j], sums[i][j + 1], sums[i][j + 2], sums[i][j + 3]));
      };
      const int turn = my_row % (rsteps * 4);  // of this row's units in `parts`
      float down = 1.f, most = 0.f;
      // of the finite values: beside an infinity they have to stay finite, or their signs would meet the infinity's
      auto finite = [](float x) { return isinf(x) ? 0.f : fabsf(x); };
      auto largest = [&](const float4& x) { most = fmaxf(most, fmaxf(fmaxf(finite(x.x), finite(x.y)), fmaxf(finite(x.z), finite(x.w)))); };
      if (RANGE && C == 1) {
        each_4([&](int, const float4& x) { largest(x); });
        row_max[set * 128 + my_row] = most;
        lora_epi_all(true);
        float up;
        lora_range(fmaxf(row_max[my_row], row_max[128 + my_row]) * fabsf(scale), down, up);
        if (set == 0) row_up[my_row] = up;
      }
      each_4([&](int c, const float4& x) {
        if (C == 1) {
          write_parts(my_row, c, scaled(x, down),
                      [&](int at, uint32_t w0, uint32_t w1) { *reinterpret_cast<uint2*>(vparts + at) = make_uint2(w0, w1); });
        } else {
          // 16-byte units of a row rotated by the row: neighbouring rows fall on different banks
          const int units = rsteps * 4, u = (c >> 2) + turn;
          *reinterpret_cast<float4*>(parts + my_row * units * 4 + (u < units ? u : u - units) * 4) = x;
          if (RANGE) largest(x);
        }
      });
      if (RANGE && C > 1) row_max[set * 128 + my_row] = most;
      if (C == 1) {
        fence_proxy_async_smem();
        lora_epi_all(true);
        if (et == 0) mbar_arrive(v_ready);
      } else {
        lora_epi_all(true);
        if (et == 0)
          for (int c = 0; c < C; ++c) mbar_arrive_remote_release(mapa_shared(smem_u32(p_ready), c));
        ok = lora_epi_all(mbar_wait_cluster(p_ready, 0, p.status, SITEL_EPI_PARTS));
        if (ok) {
          // rows of the instruction behind the tile's own stay whatever they are: nothing reads their products
          const int units = rsteps * 4, r0 = nrows * rank / C, r1 = nrows * (rank + 1) / C;
          auto range_of = [&](int row, float& down, float& up) {  // by the sum of the CTAs' largest: cheaper than the sums' own
            const uint32_t at = smem_u32(row_max + row);
            float m = 0.f;
            for (int c = 0; c < C; ++c) m += fmaxf(ld_remote_f32(mapa_shared(at, c)), ld_remote_f32(mapa_shared(at + 512, c)));
            lora_range(m * fabsf(scale), down, up);
          };
          if (RANGE && et < nrows) {
            float down, up;
            range_of(et, down, up);
            row_up[et] = up;
          }
          for (int i = et; i < (r1 - r0) * units; i += 256) {
            const int row = r0 + i / units, u = i - (row - r0) * units;
            const uint32_t at = smem_u32(parts + row * units * 4 + ((u + row) % units) * 4);
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < C; ++c) {
              const float4 x = ld_remote_f32x4(mapa_shared(at, c));
              s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
            }
            float down = 1.f, up;
            if (RANGE) range_of(row, down, up);
            write_parts(row, u * 4, scaled(s, down), [&](int off, uint32_t w0, uint32_t w1) {
              const uint32_t to = smem_u32(vparts + off);
              for (int c = 0; c < C; ++c) st_remote_u32x2(mapa_shared(to, c), w0, w1);
            });
          }
          fence_proxy_async_all();
          lora_epi_all(true);
          if (et == 0)
            for (int c = 0; c < C; ++c) mbar_arrive_remote_release(mapa_shared(smem_u32(v_ready), c));
          // the boxes lie where the parts were: only when every CTA has read them
          ok = lora_epi_all(mbar_wait_cluster(v_ready, 0, p.status, SITEL_EPI_PARTS));
          fence_proxy_async_smem();
          if (ok && lane == 0)
            for (int k = 0; k < p.c_bufs - 1 && k < nboxes; ++k) request(k, k);
        }
      }
    }
    if (turned) {
      // lanes: 128 columns of D; columns: its rows.  The two sets of four warps take every other chunk; C of the next one
      // is on its way.  No branch around a single load: rows behind the last read that one again.
      using Raw = typename std::conditional<sizeof(OutT) == 4, float, uint16_t>::type;
      auto fetch = [&](int i, Raw (&c)[32]) {
        const Raw* from = reinterpret_cast<const Raw*>(c_base) + min((ch0 + i) * 128 + my_row, g.n - 1);
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 8)
          if (j0 < nrows) {
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j0 + j] = from[min(j0 + j, nrows - 1) * g.c_pitch];
          }
      };
      Raw c[32], ahead[32];
      if (set < ch1 - ch0) fetch(set, c);
      for (int i = set; i < ch1 - ch0 && ok; i += 2) {
        const int n = (ch0 + i) * 128 + my_row;
        if (i + 2 < ch1 - ch0) fetch(i + 2, ahead);
        ok = mbar_wait(&acc_full[set], (i >> 1) & 1, p.status, SITEL_EPI_ACC);
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t v[32];
        tmem_ld_x32(t_lane + set * 128, v);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[set]);
        if (n < g.n) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j < nrows) lora_store(d_base + j * g.d_pitch + n, fmaf(__uint_as_float(v[j]), RANGE ? row_up[j] : 1.f, lora_load(reinterpret_cast<const OutT*>(&c[j]))));
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) c[j] = ahead[j];
      }
    } else {
      const bool live = qd * 32 < nrows, whole = qd * 32 + 32 <= nrows;  // this warp's 32 rows
      int slot = 0;  // of the next box, and the parity of its barrier
      uint32_t box_phase = 0;
      const float up = RANGE && my_row < nrows ? row_up[my_row] : 1.f;
      for (int i = 0; i < ch1 - ch0 && ok; ++i) {
        const int buf = i & 1;
        ok = mbar_wait(&acc_full[buf], (i >> 1) & 1, p.status, SITEL_EPI_ACC);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t t_half = t_lane + buf * 128 + set * 64;
        auto release = [&]() {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
        };
        if (!live) {
          release();
          continue;
        }
        if constexpr (VEC) {
          for (int b = 0; b < BPC; ++b) {
            const int k = i * BPC + b, col = box_col(k);
            uint32_t v[BW];
#pragma unroll
            for (int c = 0; c < BW; c += 32) tmem_ld_x32(t_half + b * BW + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
            ok = mbar_wait(&my_full[slot], box_phase, p.status, SITEL_EPI_C);
            tmem_ld_wait();
            if (b == BPC - 1) release();
            if (!ok) break;
            uint8_t* row = my_boxes + slot * 4096 + lane * 128;
            uint4 w[8];  // all reads before the first write: the compiler cannot know that they do not overlap
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = *reinterpret_cast<const uint4*>(row + ((u ^ (lane & 7)) << 4));
#pragma unroll
            for (int u = 0; u < 8; ++u)
              *reinterpret_cast<uint4*>(row + ((u ^ (lane & 7)) << 4)) = lora_add(w[u], v + u * EPV, up, static_cast<OutT*>(nullptr));
            fence_proxy_async_smem();
            __syncwarp();
            if (whole) {
              if (lane == 0) {
                if (col < g.n) tma_store_2d(&tmD, my_boxes + slot * 4096, col, row0 + qd * 32);
                tma_store_commit();
                tma_store_wait_read<1>();  // the box before this one is free again
              }
            } else {  // the last rows of a request: vector stores of whole 128-byte rows
              const int n = col + (lane & 7) * EPV;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + (lane >> 3);
                if (qd * 32 + r < nrows && n < g.n)
                  *reinterpret_cast<uint4*>(d_base + (qd * 32 + r) * g.d_pitch + n) =
                      *reinterpret_cast<const uint4*>(my_boxes + slot * 4096 + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
              }
            }
            // box k + c_bufs - 1 goes where box k - 1 was
            if (lane == 0 && k + p.c_bufs - 1 < nboxes) request(k + p.c_bufs - 1, slot == 0 ? p.c_bufs - 1 : slot - 1);
            if (++slot == p.c_bufs) { slot = 0; box_phase ^= 1; }
          }
        } else {
          float* st = reinterpret_cast<float*>(my_boxes);  // 32 rows of 32 columns, 16-byte units swizzled by the row
          for (int h = 0; h < 64; h += 32) {
            uint32_t v[32];
            tmem_ld_x32(t_half + h, v);
            tmem_ld_wait();
            if (h == 32) release();
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(st + lane * 32 + ((j ^ (lane & 7)) << 2)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            __syncwarp();
            const int n = (ch0 + i) * 128 + set * 64 + h + lane;
            for (int r = 0; r < 32 && qd * 32 + r < nrows; ++r) {
              const long long at = qd * 32 + r;
              if (n < g.n) {
                const float x = st[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)];
                lora_store(d_base + at * g.d_pitch + n, fmaf(x, RANGE ? row_up[at] : 1.f, lora_load(c_base + at * g.c_pitch + n)));
              }
            }
            __syncwarp();  // the staging is read: the next step may overwrite it
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }

  // ---------------------------------------------------------------- teardown
  if (*reinterpret_cast<volatile int*>(p.status) != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // a wait gave up: copies in flight get time to land
  }
  tc_fence_before_sync();
  __syncthreads();
  if (C > 1) {
    cluster_arrive();
    cluster_wait();  // no CTA leaves while another may still reach into its shared memory
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename T, typename OutT, bool VEC>
static int launch_lora_tile(moye_b200_ctx* h, const LoraArgs& g, int dtype, int out, cudaStream_t stream) {
  constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value && sizeof(OutT) == 4 ? 3 : 2;
  const int rsteps = (g.rank + 15) / 16, rblocks = (g.rank + 63) / 64, kbs = (g.k + 63) / 64;
  const long long live = g.requests < g.rows ? g.requests : g.rows, tiles = live + (g.rows - live) / 128;  // at most
  if (tiles > INT32_MAX / 16) MOYE_FAIL(MOYE_ERR_TOO_LARGE, "gemm_lora: too many rows and requests");
  auto kern = lora_tile_kernel<T, OutT, VEC, PARTS>;
  if (int rc = configure_once(h, kern, 227 * 1024)) return rc;
  const int total = 224 * 1024, smem = 227 * 1024;  // the last 3 KB: barriers, row ranges
  // CTAs of a tile: as many as let all tiles run at once, one CTA per SM (a cluster has to find its SMs in one part of the
  // GPU: 16 clusters of 8 do not fit on 148 SMs); each needs a K block
  int ctas = kLoraCtas < kbs ? kLoraCtas : kbs;
  for (; ctas > 1; --ctas) {
    if (tiles * ctas > h->num_sms) continue;
    if (clusters_that_fit(h, kern, ctas, kLoraTileThreads, smem) >= tiles) break;
  }
  LoraTileArgs p = {};
  p.g = g;
  const uint32_t fmt = dtype == MOYE_BF16 ? 1u : 0u;
  p.idesc1 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(rsteps * 2) << 17) | (8u << 24);
  p.idesc2 = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
  p.status = h->d_status;
  const int block = 128 * 128;
  p.k_bytes = (block + rsteps * 16 * 128 + 1023) & ~1023;
  p.k_stages = total / p.k_bytes < 12 ? total / p.k_bytes : 12;
  p.b_bytes = rblocks * block;
  const int v_bytes = PARTS * rblocks * block;
  // boxes of C per warp: what two chunks of B leave room for (2 at rank 128 in three parts, 5 at rank 64)
  p.c_bufs = (total - v_bytes - 2 * p.b_bytes) / (8 * 4096);
  if (p.c_bufs > 6) p.c_bufs = 6;
  p.b_stages = (total - v_bytes - p.c_bufs * 8 * 4096) / p.b_bytes;
  if (p.b_stages > 4) p.b_stages = 4;
  p.v_off = p.b_stages * p.b_bytes;
  p.c_off = p.v_off + v_bytes;
  p.bar_off = total;
  CUtensorMap tx, ta, tb, tc, td;
  if (int rc = encode_tmap_2d_uncached(&tx, g.X, dtype, g.k, g.rows, (uint64_t)g.x_pitch * 2, 64, 128, true)) return rc;
  const uint64_t a_pitch = g.a_pitch * 2, a_stride = g.adapters > 1 ? g.a_stride * 2 : g.rank * a_pitch;
  const uint64_t b_pitch = g.n > 1 ? g.b_pitch * 2 : g.rank * 2, b_stride = g.adapters > 1 ? g.b_stride * 2 : g.n * b_pitch;
  if (int rc = encode_tmap_3d(&ta, g.A, dtype, g.k, g.rank, g.adapters, a_pitch, a_stride, 64, rsteps * 16, true)) return rc;
  if (int rc = encode_tmap_3d(&tb, g.B, dtype, g.rank, g.n, g.adapters, b_pitch, b_stride, 64, 128, true)) return rc;
  if constexpr (VEC) {
    if (int rc = encode_tmap_2d_uncached(&tc, g.C, out, g.n, g.rows, (uint64_t)g.c_pitch * sizeof(OutT), 128 / sizeof(OutT), 32, true)) return rc;
    if (int rc = encode_tmap_2d_uncached(&td, g.D, out, g.n, g.rows, (uint64_t)g.d_pitch * sizeof(OutT), 128 / sizeof(OutT), 32, true)) return rc;
  } else {  // not used
    tc = tx;
    td = tx;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * ctas));
  cfg.blockDim = dim3(kLoraTileThreads);
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
  log_line("gemm_lora %d rows, %d requests, rank %d, %d x %d  in %d  -> tiles of 128 rows on %d CTAs", g.rows, g.requests, g.rank, g.n,
           g.k, dtype, ctas);
  MOYE_CUDA(cudaLaunchKernelEx(&cfg, kern, tx, ta, tb, tc, td, p));
  return MOYE_OK;
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
  if (rows_overlap(C, D) && !(C->ptr == D->ptr && (T == 1 || C->stride[0] == D->stride[0])))
    MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gemm_lora: C and D overlap without being the same");
  if (rows_overlap(X, D)) MOYE_FAIL(MOYE_ERR_INVALID_ARG, "gemm_lora: X and D overlap");
  LoraArgs g = {};
  g.rows = (int)T;
  g.requests = requests;
  g.adapters = (int)L;
  g.rank = (int)R;
  g.n = (int)N;
  g.k = (int)K;
  g.X = X->ptr; g.A = A->ptr; g.B = B->ptr; g.C = C->ptr; g.D = D->ptr;
  g.x_pitch = T > 1 ? X->stride[0] : K;  // the pitch of a single row says nothing
  g.a_pitch = A->stride[1]; g.a_stride = A->stride[0];
  g.b_pitch = B->stride[1]; g.b_stride = B->stride[0];
  g.c_pitch = T > 1 ? C->stride[0] : N;
  g.d_pitch = T > 1 ? D->stride[0] : N;
  g.which = which;
  g.offsets = offsets;
  g.scales = scales;
  // Requests of several rows share their adapter's factors on the tensor cores.  A row by itself costs its factors' bytes
  // from L2, 3e-7 to 4e-7 us x R (K + N) (512 rows, K = N = 4096: R = 16 28 us, R = 64 86 us); the tile kernel starts
  // 10 us later and takes about 3.6e-5 us x (K + N) per tile (256 tiles, R = 16: 93 us; R = 64: 109).  64 requests of
  // 4 / 8 / 16 rows, R = 16: rows 22 / 37 / 64 us, tiles 33 / 35 / 35.
  const double tiles = (double)T / 128 + (requests < T ? requests : T);
  if (offsets && (double)T * R > 84 * tiles + 2.3e7 / (double)(K + N)) {
    auto on16 = [](const moye_tensor_t* t) {
      const int eb = dtype_bytes(t->dtype);
      return (reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && (t->shape[1] * eb) % 16 == 0 &&
             (t->shape[0] <= 1 || (t->stride[0] * eb) % 16 == 0);
    };
    const bool vec = on16(C) && on16(D), wide = D->dtype == MOYE_F32;
    if (X->dtype == MOYE_F16) {
      if (wide) return vec ? launch_lora_tile<__half, float, true>(h, g, X->dtype, D->dtype, stream) : launch_lora_tile<__half, float, false>(h, g, X->dtype, D->dtype, stream);
      return vec ? launch_lora_tile<__half, __half, true>(h, g, X->dtype, D->dtype, stream) : launch_lora_tile<__half, __half, false>(h, g, X->dtype, D->dtype, stream);
    }
    if (wide)
      return vec ? launch_lora_tile<__nv_bfloat16, float, true>(h, g, X->dtype, D->dtype, stream) : launch_lora_tile<__nv_bfloat16, float, false>(h, g, X->dtype, D->dtype, stream);
    return vec ? launch_lora_tile<__nv_bfloat16, __nv_bfloat16, true>(h, g, X->dtype, D->dtype, stream)
               : launch_lora_tile<__nv_bfloat16, __nv_bfloat16, false>(h, g, X->dtype, D->dtype, stream);
  }
  log_line("gemm_lora %lld rows, %d requests, rank %lld, %lld x %lld  in %d  -> a cluster per row", (long long)T, requests, (long long)R,
           (long long)N, (long long)K, X->dtype);
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
