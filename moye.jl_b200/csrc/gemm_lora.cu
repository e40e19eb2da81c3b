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
#include "gemm_common.cuh"

namespace moye {

constexpr int kLoraCtas = 8;         // cluster size of the row kernel
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

// ---------------------------------------------------------------------------------------------- long requests
// A cluster of C CTAs takes up to 128 rows of one request.  CTA c multiplies its K blocks of X (128 lanes of tensor
// memory) with A[a] (R columns); with C > 1 the fp32 parts meet through distributed shared memory, CTA c summing 128 / C
// rows in CTA order and handing the result to all; every CTA then multiplies it with its 128-column chunks of B[a] and
// adds C.  The product of rank R enters the second multiplication as a sum of 16-bit parts: two parts carry 16 (bf16)
// or 22 (f16) bits, a sixteenth of an output step or less; bf16 operands with a Float32 output take three (24 bits).
//
// Warp 0 producer, warp 1 MMA issuer, warps 2-5 move the parts and run the epilogue.  The producer's ring carries first
// the K blocks, then the chunks of B, which therefore arrive while the parts meet.  The output is bound by memory: the
// accumulator crosses shared memory so that a warp reads C and writes D in 16-byte accesses of whole sectors, and the
// next 4 KB of C per warp are on their way while these are added.
// Two CTAs fit on an SM (256 tensor-memory columns each, at most 113 KB); three never do, their shared memory is too large.
constexpr int kLoraTileThreads = 192;
enum : int { SITEL_PROD_EMPTY = 171, SITEL_MMA_FULL = 172, SITEL_MMA_V = 173, SITEL_MMA_ACC = 174, SITEL_EPI_V = 175, SITEL_EPI_PARTS = 176, SITEL_EPI_ACC = 177, SITEL_SMEM_BASE = 178 };

struct LoraTileArgs {
  LoraArgs g;
  uint32_t idesc1, idesc2;
  int* status;
  int stages, stage_bytes, v_off, stage_out_off, bar_off;  // shared-memory plan, bytes
};

__device__ __forceinline__ float4 ld_remote_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_remote_u32x2(uint32_t cluster_addr, uint32_t x, uint32_t y) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(cluster_addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void lora_epi_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t lora_pack2(float a, float b) {
  const T lo = cvt_out<T>(a), hi = cvt_out<T>(b);
  return (uint32_t)(*reinterpret_cast<const uint16_t*>(&lo)) | ((uint32_t)(*reinterpret_cast<const uint16_t*>(&hi)) << 16);
}

// The request and first row of tile `want`; q = -1 when there are fewer tiles.  All threads of the CTA; `sums` holds one
// int per thread.
__device__ __forceinline__ void lora_find_tile(const LoraArgs& g, int want, int* sums, int* result) {
  const int tid = threadIdx.x, per = (g.requests + kLoraTileThreads - 1) / kLoraTileThreads;
  const int q0 = min(tid * per, g.requests), q1 = min(q0 + per, g.requests);
  auto tiles_of = [&](int q, int& lo, int& hi) {
    lo = min(max(__ldg(g.offsets + q), 0), g.rows);
    hi = min(max(__ldg(g.offsets + q + 1), 0), g.rows);
    return hi > lo ? (hi - lo + 127) >> 7 : 0;
  };
  int mine = 0, lo, hi;
  for (int q = q0; q < q1; ++q) mine += tiles_of(q, lo, hi);
  if (tid == 0) result[0] = -1;
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(~0u, incl, d);
    if ((tid & 31) >= d) incl += up;
  }
  if ((tid & 31) == 31) sums[tid >> 5] = incl;
  __syncthreads();
  int before = incl - mine;
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
__global__ void __launch_bounds__(kLoraTileThreads, 2)
lora_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA,
                 const __grid_constant__ CUtensorMap tmB, const LoraTileArgs p) {
  const LoraArgs& g = p.g;
  // No slack for aligning the base by hand: two CTAs at rank 64 leave 700 bytes of an SM's shared memory.
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, SITEL_SMEM_BASE);
    return;
  }
  uint8_t* vparts = smem + p.v_off;                                // [part][64-wide block of R][128 rows][128 bytes], swizzled
  float* parts = reinterpret_cast<float*>(smem + p.stage_out_off);  // [128][R] fp32; later the epilogue's staging
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.bar_off);
  uint64_t *full = bars, *empty = bars + 8, *acc_full = bars + 16, *acc_empty = bars + 18, *v_acc = bars + 20, *p_ready = bars + 21,
           *v_ready = bars + 22;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 23);
  int* scratch = reinterpret_cast<int*>(bars + 24);  // 8 warp sums, then the tile
  constexpr uint32_t TMEM_COLS = 256;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  griddep_wait();
  lora_find_tile(g, blockIdx.x / C, scratch, scratch + 8);
  const int q = scratch[8], row0 = scratch[9], nrows = scratch[10];
  if (q < 0) return;  // fewer tiles than CTAs; the same in the whole cluster
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

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    mbar_init(v_acc, 1);
    mbar_init(p_ready, C);
    mbar_init(v_ready, C);
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
      for (int i = 0; i < (kb1 - kb0) + (ch1 - ch0); ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1, p.status, SITEL_PROD_EMPTY)) break;
        uint8_t* s = smem + stage * p.stage_bytes;
        if (i < kb1 - kb0) {
          const int k = (kb0 + i) * 64;
          mbar_arrive_expect_tx(&full[stage], 128 * 128 + a_bytes);
          tma_load_2d(s, &tmX, &full[stage], k, row0);
          tma_load_3d(s + 128 * 128, &tmA, &full[stage], k, 0, a);
        } else {
          const int n = (ch0 + i - (kb1 - kb0)) * 128;
          mbar_arrive_expect_tx(&full[stage], rblocks * 128 * 128);
          for (int b = 0; b < rblocks; ++b) tma_load_3d(s + b * 128 * 128, &tmB, &full[stage], b * 64, n, a);
        }
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(&full[stage], phase, p.status, SITEL_MMA_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t s = smem_u32(smem + stage * p.stage_bytes);
        const uint64_t xd = umma_desc_k_sw128(s), ad = umma_desc_k_sw128(s + 128 * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_ss<KIND_F16>(tmem_base, xd + 2 * k, ad + 2 * k, p.idesc1, (kb > kb0 || k > 0) ? 1u : 0u);
        tc_commit(&empty[stage]);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      if (ok) tc_commit(v_acc);
      if (ok && ch1 > ch0) ok = mbar_wait_cluster(v_ready, 0, p.status, SITEL_MMA_V);
      fence_proxy_async_smem();
      const uint32_t vs = smem_u32(vparts);
      for (int i = 0; i < ch1 - ch0 && ok; ++i) {
        const int buf = i & 1;
        ok = mbar_wait(&acc_empty[buf], ((i >> 1) & 1) ^ 1, p.status, SITEL_MMA_ACC) && mbar_wait(&full[stage], phase, p.status, SITEL_MMA_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t s = smem_u32(smem + stage * p.stage_bytes);
        for (int part = 0; part < PARTS; ++part)
          for (int k = 0; k < rsteps; ++k) {
            const uint32_t at = (k >> 2) * (128 * 128) + (k & 3) * 32;  // block of 64, step of 16 inside it
            tc_mma_ss<KIND_F16>(tmem_base + buf * 128, umma_desc_k_sw128(vs + part * rblocks * (128 * 128) + at), umma_desc_k_sw128(s + at),
                                p.idesc2, (part | k) != 0 ? 1u : 0u);
          }
        tc_commit(&empty[stage]);
        tc_commit(&acc_full[buf]);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ warps 2-5: the rank-R product, then the epilogue
    constexpr int EPV = 16 / (int)sizeof(OutT);  // elements of 16 bytes
    constexpr int LPR = 32 / EPV;                // lanes side by side in one row of a step of 32 columns
    constexpr int STEPS = 8 / LPR;               // steps whose C is on its way: 8 accesses of 16 bytes a lane
    const int qd = warp & 3, et = (warp - 2) * 32 + lane;  // tensor-memory quarter; thread among the 128
    const int my_row = qd * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>(qd * 32) << 16;
    const float scale = g.scales ? __ldg(g.scales + a) : 1.f;
    const int sub_row = lane / LPR, sub_col = (lane % LPR) * EPV;  // access i of a step: row i * EPV + sub_row
    uint4 cpre[STEPS][LPR];
    auto prefetch = [&](uint4 (&to)[LPR], int n) {
      n += sub_col;
#pragma unroll
      for (int i = 0; i < LPR; ++i) {
        const int r = qd * 32 + i * EPV + sub_row;
        if (r < nrows && n < g.n) to[i] = *reinterpret_cast<const uint4*>(c_base + r * g.c_pitch + n);
      }
    };
    if (VEC && ch0 < ch1) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) prefetch(cpre[s], ch0 * 128 + s * 32);
    }
    // the value of `x` as PARTS 16-bit numbers, the largest first
    auto write_parts = [&](int row, int col, float4 x, auto&& store) {  // 4 columns at once
      float r[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const uint32_t w0 = lora_pack2<T>(r[0], r[1]), w1 = lora_pack2<T>(r[2], r[3]);
        const float2 f0 = lora_pair<T>(w0), f1 = lora_pair<T>(w1);
        r[0] -= f0.x; r[1] -= f0.y; r[2] -= f1.x; r[3] -= f1.y;
        store((part * rblocks + (col >> 6)) * (128 * 128) + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 4) * 2, w0, w1);
      }
    };
    // the four warps go on or give up together: they meet at barriers
    bool ok = all_of_128(1, mbar_wait(v_acc, 0, p.status, SITEL_EPI_V));
    if (ok) {
      tc_fence_after_sync();
      for (int c = 0; c < rsteps * 16; c += 16) {  // columns behind R are products with zero rows: zero
        uint32_t v[16];
        tmem_ld_x16(tmem_base + t_lane + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 x = make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
          if (C == 1) {
            write_parts(my_row, c + j, make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale),
                        [&](int at, uint32_t w0, uint32_t w1) { *reinterpret_cast<uint2*>(vparts + at) = make_uint2(w0, w1); });
          } else {
            // 16-byte units of a row rotated by the row: neighbouring rows fall on different banks
            const int units = rsteps * 4, u = ((c + j) >> 2) + my_row;
            *reinterpret_cast<float4*>(parts + my_row * units * 4 + (u % units) * 4) = x;
          }
        }
      }
      tc_fence_before_sync();
      if (C == 1) {
        fence_proxy_async_smem();
        lora_epi_sync();
        if (et == 0) mbar_arrive(v_ready);
      } else {
        lora_epi_sync();
        if (et == 0)
          for (int c = 0; c < C; ++c) mbar_arrive_remote_release(mapa_shared(smem_u32(p_ready), c));
        ok = all_of_128(1, mbar_wait_cluster(p_ready, 0, p.status, SITEL_EPI_PARTS));
        if (ok) {
          const int units = rsteps * 4, r0 = 128 * rank / C, r1 = 128 * (rank + 1) / C;
          for (int i = et; i < (r1 - r0) * units; i += 128) {
            const int row = r0 + i / units, u = i - (row - r0) * units;
            const uint32_t at = smem_u32(parts + row * units * 4 + ((u + row) % units) * 4);
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < C; ++c) {
              const float4 x = ld_remote_f32x4(mapa_shared(at, c));
              s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
            }
            write_parts(row, u * 4, make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale), [&](int off, uint32_t w0, uint32_t w1) {
              const uint32_t to = smem_u32(vparts + off);
              for (int c = 0; c < C; ++c) st_remote_u32x2(mapa_shared(to, c), w0, w1);
            });
          }
          fence_proxy_async_all();
          lora_epi_sync();
          if (et == 0)
            for (int c = 0; c < C; ++c) mbar_arrive_remote_release(mapa_shared(smem_u32(v_ready), c));
        }
      }
    }
    float* st = parts + (warp - 2) * 32 * 32;  // this warp's staging: 32 rows of 32 columns, 16-byte units swizzled by the row
    for (int i = 0; i < ch1 - ch0 && ok; ++i) {
      const int buf = i & 1, n0 = (ch0 + i) * 128;
      ok = mbar_wait(&acc_full[buf], (i >> 1) & 1, p.status, SITEL_EPI_ACC);
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll 1
      for (int h = 0; h < 128; h += 32 * STEPS) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int col = h + s * 32;
          {
            uint32_t v[32];
            tmem_ld_x32(tmem_base + t_lane + buf * 128 + col, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(st + lane * 32 + ((j ^ (lane & 7)) << 2)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
          if (col + 32 >= 128) tc_fence_before_sync();
          __syncwarp();
          if (col + 32 >= 128 && lane == 0) mbar_arrive(&acc_empty[buf]);
          if constexpr (VEC) {
            const int n = n0 + col + sub_col;
#pragma unroll
            for (int k = 0; k < LPR; ++k) {
              const int r = k * EPV + sub_row;
              OutT o[EPV];
              const OutT* cin = reinterpret_cast<const OutT*>(&cpre[s][k]);
#pragma unroll
              for (int e = 0; e < EPV; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(st + r * 32 + ((((sub_col + e) >> 2) ^ (r & 7)) << 2));
                o[e] = cvt_out<OutT>(lora_load(cin + e) + x.x);
                o[e + 1] = cvt_out<OutT>(lora_load(cin + e + 1) + x.y);
                o[e + 2] = cvt_out<OutT>(lora_load(cin + e + 2) + x.z);
                o[e + 3] = cvt_out<OutT>(lora_load(cin + e + 3) + x.w);
              }
              if (qd * 32 + r < nrows && n < g.n)
                *reinterpret_cast<uint4*>(d_base + (qd * 32 + r) * g.d_pitch + n) = *reinterpret_cast<const uint4*>(o);
            }
            const int next = n0 + col + 32 * STEPS;  // the same step of the next round, maybe in the next chunk
            if (next < ch1 * 128) prefetch(cpre[s], next);
          } else {
            for (int r = 0; r < 32 && qd * 32 + r < nrows; ++r) {
              const long long row = qd * 32 + r;
              if (n0 + col + lane < g.n) {
                const float x = st[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)];
                lora_store(d_base + row * g.d_pitch + n0 + col + lane, lora_load(c_base + row * g.c_pitch + n0 + col + lane) + x);
              }
            }
          }
          __syncwarp();  // the staging is read: the next step may overwrite it
        }
      }
    }
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
static int launch_lora_tile(moye_b200_ctx* h, const LoraArgs& g, int dtype, cudaStream_t stream) {
  constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value && sizeof(OutT) == 4 ? 3 : 2;
  const int rsteps = (g.rank + 15) / 16, rblocks = (g.rank + 63) / 64, kbs = (g.k + 63) / 64;
  const long long tiles = ((long long)g.rows + 127) / 128 + (g.requests < g.rows ? g.requests : g.rows);  // at most
  // CTAs of a tile: as few as fill the GPU with two CTAs per SM; each needs a K block
  int ctas = 1;
  while (ctas < kLoraCtas && ctas * 2 <= kbs && tiles * ctas < 2 * h->num_sms) ctas *= 2;
  LoraTileArgs p = {};
  p.g = g;
  const uint32_t fmt = dtype == MOYE_BF16 ? 1u : 0u;
  p.idesc1 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(rsteps * 2) << 17) | (8u << 24);
  p.idesc2 = (1u << 4) | (fmt << 7) | (fmt << 10) | (16u << 17) | (8u << 24);
  p.status = h->d_status;
  const int block = 128 * 128;
  p.stage_bytes = block + rsteps * 16 * 128 > rblocks * block ? block + rsteps * 16 * 128 : rblocks * block;
  p.stage_bytes = (p.stage_bytes + 1023) & ~1023;
  const int v_bytes = PARTS * rblocks * block;
  int out_bytes = 4 * 32 * 32 * 4;
  if (ctas > 1 && 128 * rsteps * 16 * 4 > out_bytes) out_bytes = 128 * rsteps * 16 * 4;
  const int rest = v_bytes + out_bytes + 512, half_sm = 113 * 1024;
  // two CTAs per SM if three (two) stages fit into half of its shared memory, else one with as many as fit
  p.stages = rest + 3 * p.stage_bytes <= half_sm ? 3 : rest + 2 * p.stage_bytes <= half_sm ? 2 : 4;
  while (p.stages > 2 && rest + p.stages * p.stage_bytes > 227 * 1024) --p.stages;
  p.v_off = p.stages * p.stage_bytes;
  p.stage_out_off = p.v_off + v_bytes;
  p.bar_off = p.stage_out_off + out_bytes;
  const int smem = p.bar_off + 512;
  CUtensorMap tx, ta, tb;
  if (int rc = encode_tmap_2d_uncached(&tx, g.X, dtype, g.k, g.rows, (uint64_t)g.x_pitch * 2, 64, 128, true)) return rc;
  const uint64_t a_pitch = g.a_pitch * 2, a_stride = g.adapters > 1 ? g.a_stride * 2 : g.rank * a_pitch;
  const uint64_t b_pitch = g.n > 1 ? g.b_pitch * 2 : g.rank * 2, b_stride = g.adapters > 1 ? g.b_stride * 2 : g.n * b_pitch;
  if (int rc = encode_tmap_3d(&ta, g.A, dtype, g.k, g.rank, g.adapters, a_pitch, a_stride, 64, rsteps * 16, true)) return rc;
  if (int rc = encode_tmap_3d(&tb, g.B, dtype, g.rank, g.n, g.adapters, b_pitch, b_stride, 64, 128, true)) return rc;
  auto kern = lora_tile_kernel<T, OutT, VEC, PARTS>;
  if (int rc = configure_once(h, kern, 227 * 1024)) return rc;
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
  log_line("gemm_lora %d rows, %d requests, rank %d, %d x %d  in %d  -> tiles of 128 rows on %d CTAs, %d stages", g.rows, g.requests,
           g.rank, g.n, g.k, dtype, ctas, p.stages);
  MOYE_CUDA(cudaLaunchKernelEx(&cfg, kern, tx, ta, tb, p));
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
  // Requests of several rows share their adapter's factors on the tensor cores; single rows do not.
  if (offsets && T >= 4ll * requests) {
    auto on16 = [](const moye_tensor_t* t) {
      const int eb = dtype_bytes(t->dtype);
      return (reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && (t->shape[1] * eb) % 16 == 0 &&
             (t->shape[0] <= 1 || (t->stride[0] * eb) % 16 == 0);
    };
    const bool vec = on16(C) && on16(D), wide = D->dtype == MOYE_F32;
    if (X->dtype == MOYE_F16) {
      if (wide) return vec ? launch_lora_tile<__half, float, true>(h, g, X->dtype, stream) : launch_lora_tile<__half, float, false>(h, g, X->dtype, stream);
      return vec ? launch_lora_tile<__half, __half, true>(h, g, X->dtype, stream) : launch_lora_tile<__half, __half, false>(h, g, X->dtype, stream);
    }
    if (wide)
      return vec ? launch_lora_tile<__nv_bfloat16, float, true>(h, g, X->dtype, stream) : launch_lora_tile<__nv_bfloat16, float, false>(h, g, X->dtype, stream);
    return vec ? launch_lora_tile<__nv_bfloat16, __nv_bfloat16, true>(h, g, X->dtype, stream)
               : launch_lora_tile<__nv_bfloat16, __nv_bfloat16, false>(h, g, X->dtype, stream);
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
