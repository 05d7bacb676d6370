// 8-bit projection on the tcgen05 tensor cores (sm_100a): e4m3 weights with
// a scale per output channel, e4m3 activations with a scale per token row.
//
//   out[m][j] = epilogue( (sum_k W[j][k] X[m][k]) * sx[m] * sw[j] )
//
// Weight rows j fill the MMA's M = 128, token rows m are its N (at most 256
// per block), K goes in blocks of 128 bytes.  Few token rows make the
// weights' bytes the cost, so they have to stream through every SM at once:
// a weight tile's K range is split over a cluster of C CTAs, C as large as
// keeps all CTAs of the launch resident.  Each CTA sums its share in TMEM; at
// the end every CTA stores its fp32 partial in its own shared memory and, after
// one cluster barrier, finishes 1/C of the tile from all C partials, read
// over distributed shared memory in rank order.  No partial goes through
// global memory, there is no workspace, no counter and no atomic, and the
// result of a call is always the same bits.
//
// Warp 0 requests the tiles (TMA, 128-byte swizzle), warp 1 issues
// tcgen05.mma kind::f8f6f4 (fp32 accumulators in TMEM), warps 2-5 move the
// accumulators to shared memory; all six finish the outputs.  Before the
// dependency wait the first weight tiles are only prefetched into L2: the
// weights may come from an earlier kernel of the stream (tsds_quant_fp8), so
// they are read after it.
// Every mbarrier wait is bounded; a CTA that gives up records TSDS_E_TIMEOUT
// and still takes part in the cluster's barriers.
#include "common.cuh"
#include "linear.cuh"
#include "tc_core.cuh"

using namespace tsds;
using namespace tsds::tc;

namespace {

constexpr int THREADS = 192;
constexpr int KB = 128;                  // bytes (elements) of K per stage: one swizzle row
constexpr int A_BYTES = TILE_J * KB;     // 16 KB of weights per stage
constexpr int MAX_ROWS = 256;            // token rows per block: the widest MMA
constexpr int RING = 8;                  // most stages
constexpr int MAX_C = 8;                 // largest portable cluster
constexpr int SMEM_SM = 233472;          // 228 KB per SM
constexpr int SMEM_CTA = 220 * 1024;     // dynamic shared memory a CTA may ask for
constexpr int SMEM_SIDE = 2048;          // static shared memory + the system's 1 KB per CTA

struct F8Args {
  int M, n_out, KT, C, blocks;  // blocks of MAX_ROWS token rows
  int npad, stages, b_bytes, chunk;
  int ldo, res_ld;
  const float *sx, *sw;
  const bf16* res;
  bf16* out;
  int32_t* status;
  uint32_t idesc;
  int tmem_cols;
  uint64_t wait_ns;
};

struct F8Shared {
  uint64_t full[RING], empty[RING], done, drain;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void umma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum));
}

__device__ __forceinline__ float4 ld_peer(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// every thread of the cluster (or of the CTA, when it is alone)
__device__ __forceinline__ void unit_barrier(int C) {
  __syncwarp();
  if (C > 1)
    cluster_sync_all();
  else
    __syncthreads();
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

template <int EPI>
__global__ void __launch_bounds__(THREADS)
    f8_gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap, F8Args p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ F8Shared sh;
  constexpr bool SW = EPI == EPI_SWIGLU;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.C > 1 ? (int)cluster_ctarank() : 0;
  const int unit = blockIdx.x / p.C;            // (weight tile, token block), token blocks fastest:
  const int tile = unit / p.blocks;             // the tiles in flight share their weights through L2
  const int m_base = (unit - tile * p.blocks) * MAX_ROWS;
  const int k_lo = rank * p.KT / p.C, nk = (rank + 1) * p.KT / p.C - k_lo;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    mbar_init(&sh.done, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                 "r"(p.tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  uint8_t* a_smem = smem;
  uint8_t* b_smem = smem + p.stages * A_BYTES;
  pdl_trigger();
  int issued = 0;
  // a stage's weight rows: 128 of one matrix, or 64 gate and 64 up rows
  const int row0 = SW ? tile * 64 : tile * TILE_J;
  const int row1 = SW ? p.n_out + tile * 64 : row0 + 64;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&amap);
      prefetch_tmap(&bmap);
      for (int i = 0; i < nk && i < p.stages; ++i) {
        tma_prefetch_l2_2d(&amap, (k_lo + i) * KB, row0);
        tma_prefetch_l2_2d(&amap, (k_lo + i) * KB, row1);
      }
      pdl_wait();
      for (int i = 0; i < nk; ++i) {
        const int s = i % p.stages;
        if (i >= p.stages && !mbar_wait(&sh.empty[s], (i / p.stages - 1) & 1, p.wait_ns)) {
          atomicExch(p.status, TSDS_E_TIMEOUT);
          *(volatile int*)&sh.abort = 1;
          break;
        }
        mbar_arrive_expect_tx(&sh.full[s], A_BYTES + p.b_bytes);
        const int x = (k_lo + i) * KB;
        tma_load_2d(a_smem + s * A_BYTES, &amap, &sh.full[s], x, row0);
        tma_load_2d(a_smem + s * A_BYTES + A_BYTES / 2, &amap, &sh.full[s], x, row1);
        tma_load_2d(b_smem + s * p.b_bytes, &bmap, &sh.full[s], x, m_base);
        issued = i + 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      for (int i = 0; i < nk; ++i) {
        const int s = i % p.stages;
        if (!mbar_wait(&sh.full[s], (i / p.stages) & 1, p.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = smem_u32(a_smem + s * A_BYTES), b = smem_u32(b_smem + s * p.b_bytes);
#pragma unroll
        for (int kk = 0; kk < KB / 32; ++kk)
          umma_f8(tmem, sdesc_sw128(a + kk * 32), sdesc_sw128(b + kk * 32), p.idesc, (i | kk) != 0);
        umma_commit(&sh.empty[s]);
        issued = i + 1;
      }
      if (ok) {
        umma_commit(&sh.done);
      } else {
        atomicExch(p.status, TSDS_E_TIMEOUT);
        *(volatile int*)&sh.abort = 1;
      }
    }
  }
  pdl_wait();
  __syncwarp();
  // done completes when every MMA has, so the ring is free for the partials
  if (!mbar_wait(&sh.done, 0, p.wait_ns)) {
    if (lane == 0) atomicExch(p.status, TSDS_E_TIMEOUT);
    *(volatile int*)&sh.abort = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const bool alive = !*(volatile int*)&sh.abort;
  if (!alive) {  // uniform: copies and MMAs in flight finish (bounded) before TMEM is freed
    if (warp == 0 && lane == 0) drain_tma_ring(sh.full, p.stages, issued);
    if (warp == 1 && lane == 0 && issued > 0) drain_mma<1>(&sh.drain);
    __syncthreads();
  }

  float* part = reinterpret_cast<float*>(smem);
  const uint32_t part_addr = smem_u32(part);
  const int rows = p.M - m_base < MAX_ROWS ? p.M - m_base : MAX_ROWS;
  constexpr int G = SW ? 16 : 32;   // groups of four output channels per token row
  const int j_base = SW ? tile * 64 : tile * TILE_J;
  const bool wide = (p.ldo % 4) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 &&
                    (EPI != EPI_RESIDUAL || ((p.res_ld % 4) == 0 && (reinterpret_cast<uintptr_t>(p.res) & 7) == 0));
  // token rows in chunks that fit the ring: partials [chunk][128] fp32
  for (int c0 = 0; c0 < rows; c0 += p.chunk) {
    const int cn = rows - c0 < p.chunk ? rows - c0 : p.chunk;
    if (alive && warp >= 2) {
      const int quarter = warp & 3;   // the TMEM lanes this warp may read
      const int r = quarter * 32 + lane;
      for (int c = 0; c < cn; c += 16) {
        float v[16];
        tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c0 + c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < cn) part[(c + i) * TILE_J + r] = v[i];
      }
    }
    unit_barrier(p.C);
    const int total = cn * G, lo = rank * total / p.C, hi = (rank + 1) * total / p.C;
    for (int e = lo + (int)threadIdx.x; alive && e < hi; e += THREADS) {
      const int mc = e / G, g = e - mc * G;
      const int m = m_base + c0 + mc, j = j_base + g * 4;
      const uint32_t at = part_addr + (uint32_t)(mc * TILE_J + g * 4) * 4;
      float4 acc[2];
#pragma unroll
      for (int h = 0; h < (SW ? 2 : 1); ++h) {
        if (p.C == 1) {
          acc[h] = *reinterpret_cast<const float4*>(part + mc * TILE_J + g * 4 + h * 64);
        } else {
          float4 f[MAX_C];
#pragma unroll
          for (int q = 0; q < MAX_C; ++q)
            if (q < p.C) f[q] = ld_peer(mapa_shared(at + h * 256, q));
          acc[h] = f[0];
#pragma unroll
          for (int q = 1; q < MAX_C; ++q)
            if (q < p.C) acc[h] = add4(acc[h], f[q]);
        }
      }
      const float sx = p.sx[m];
      float o[4];
      const float a4[4] = {acc[0].x, acc[0].y, acc[0].z, acc[0].w};
      const float b4[4] = {acc[1].x, acc[1].y, acc[1].z, acc[1].w};
      const int left = p.n_out - j;   // channels of this group inside the output
      if (left <= 0) continue;
      const bool vec = wide && left >= 4;
      float rv[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (EPI == EPI_RESIDUAL) {
        const bf16* rp = p.res + (int64_t)m * p.res_ld + j;
        if (vec) {
          const uint2 u = *reinterpret_cast<const uint2*>(rp);
          rv[0] = bf_lo(u.x), rv[1] = bf_hi(u.x), rv[2] = bf_lo(u.y), rv[3] = bf_hi(u.y);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < left) rv[i] = bf2f(rp[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int jj = i < left ? j + i : j;
        o[i] = a4[i] * sx * p.sw[jj];
        if constexpr (SW) o[i] = silu(o[i]) * (b4[i] * sx * p.sw[p.n_out + jj]);
        if constexpr (EPI == EPI_RESIDUAL) o[i] += rv[i];
      }
      bf16* op = p.out + (int64_t)m * p.ldo + j;
      if (vec) {
        *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < left) op[i] = f2bf(o[i]);
      }
    }
    unit_barrier(p.C);   // the peers are done with this CTA's partials
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols));
  }
}

// Clusters of C CTAs with `smem` bytes each that the device holds at once
// (0 if the query fails); cached per (C, smem), the devices of one process
// assumed alike.
template <int EPI>
int resident_clusters(int C, size_t smem) {
  struct Entry {
    int C;
    size_t smem;
    int n;
  };
  static Entry cache[64];
  static int used = 0;
  std::lock_guard<std::mutex> hold(tsds_host_cache_lock());
  for (int i = 0; i < used; ++i)
    if (cache[i].C == C && cache[i].smem == smem) return cache[i].n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, f8_gemm_kernel<EPI>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (used < 64) cache[used++] = {C, smem, n};
  return n;
}

template <int EPI>
int run(const uint8_t* x, int ldx, const uint8_t* w, F8Args p, int K, cudaStream_t stream) {
  static tsds_device_flags limit_set;
  int st = tsds_smem_limit_once(f8_gemm_kernel<EPI>, SMEM_CTA, limit_set);
  if (st != TSDS_OK) return st;
  constexpr bool SW = EPI == EPI_SWIGLU;
  const int tiles = SW ? (p.n_out + 63) / 64 : (p.n_out + TILE_J - 1) / TILE_J;
  p.KT = (K + KB - 1) / KB;
  p.blocks = (p.M + MAX_ROWS - 1) / MAX_ROWS;
  const int widest = p.M < MAX_ROWS ? p.M : MAX_ROWS;
  p.npad = (widest + 15) / 16 * 16;
  p.b_bytes = p.npad * KB;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.npad) p.tmem_cols *= 2;
  // CTAs per SM: three while three accumulators fit in TMEM's 512 columns and
  // three stages in a third of the shared memory
  int ctas = p.npad <= 64 ? 3 : 2;
  const int stage = A_BYTES + p.b_bytes;
  p.stages = (SMEM_SM / ctas - SMEM_SIDE - 1024) / stage;
  if (p.stages > RING) p.stages = RING;
  const size_t smem = (size_t)p.stages * stage + 1024;
  p.chunk = p.stages * stage / (TILE_J * 4) / 16 * 16;
  if (p.chunk > p.npad) p.chunk = p.npad;
  const long long units = (long long)tiles * p.blocks;
  p.C = 1;
  for (int c = MAX_C; c > 1; --c) {
    if (p.KT < 2 * c || units * c > (long long)tsds_tc_num_sms() * ctas) continue;
    if (resident_clusters<EPI>(c, smem) >= units) {
      p.C = c;
      break;
    }
  }
  TSDS_RETURN_IF(units * p.C > 0x7fffffffll, TSDS_E_UNSUPPORTED);
  p.idesc = (1u << 4) | ((uint32_t)(p.npad >> 3) << 17) | ((uint32_t)(TILE_J >> 4) << 24);
  p.wait_ns = tsds_get_wait_limit_ns();
  CUtensorMap amap, bmap;
  st = tsds_make_tmap_2d_u8(&amap, w, K, SW ? 2 * (uint64_t)p.n_out : p.n_out, K, KB, 64);
  if (st != TSDS_OK) return st;
  st = tsds_make_tmap_2d_u8(&bmap, x, K, p.M, ldx, KB, p.npad);
  if (st != TSDS_OK) return st;
  const dim3 grid((unsigned)(units * p.C));
  if (p.C > 1)
    tsds_launch_cluster(f8_gemm_kernel<EPI>, grid, dim3(THREADS), smem, stream, p.C, amap, bmap, p);
  else
    tsds_launch(f8_gemm_kernel<EPI>, grid, dim3(THREADS), smem, stream, amap, bmap, p);
  return tsds_launch_status();
}

int check(const void* x, int ldx, const float* sx, const void* w, const float* sw, const void* out, int ldo, int M,
          int n_out, int K, const int32_t* status) {
  TSDS_RETURN_IF(M < 0 || n_out <= 0 || K <= 0 || (K % 16) != 0 || ldx < K || ldo < n_out || n_out > (1 << 29),
                 TSDS_E_INVALID);
  if (M == 0) return TSDS_OK;
  TSDS_RETURN_IF(!x || !sx || !w || !sw || !out || !status, TSDS_E_INVALID);
  TSDS_RETURN_IF(!tsds_aligned16(x) || !tsds_aligned16(w) || (ldx % 16), TSDS_E_ALIGN);
  return TSDS_OK;
}

F8Args args_of(const float* sx, const float* sw, void* out, int ldo, int M, int n_out, int32_t* status) {
  F8Args p = {};
  p.M = M;
  p.n_out = n_out;
  p.ldo = ldo;
  p.sx = sx;
  p.sw = sw;
  p.out = (bf16*)out;
  p.status = status;
  return p;
}

}  // namespace

extern "C" int tsds_linear_fp8(const void* x, int ldx, const float* x_scale, const void* W, const float* w_scale,
                               void* out, int ldo, int M, int n_out, int K, int32_t* status, tsds_stream_t stream) {
  const int st = check(x, ldx, x_scale, W, w_scale, out, ldo, M, n_out, K, status);
  if (st != TSDS_OK || M == 0) return st;
  return run<EPI_STORE>((const uint8_t*)x, ldx, (const uint8_t*)W,
                        args_of(x_scale, w_scale, out, ldo, M, n_out, status), K, stream);
}

extern "C" int tsds_linear_residual_fp8(const void* x, int ldx, const float* x_scale, const void* W,
                                        const float* w_scale, const void* res, int res_ld, void* out, int ldo, int M,
                                        int n_out, int K, int32_t* status, tsds_stream_t stream) {
  const int st = check(x, ldx, x_scale, W, w_scale, out, ldo, M, n_out, K, status);
  if (st != TSDS_OK) return st;
  TSDS_RETURN_IF(res_ld < n_out, TSDS_E_INVALID);
  if (M == 0) return TSDS_OK;
  TSDS_RETURN_IF(!res || (res == out && res_ld != ldo), TSDS_E_INVALID);
  F8Args p = args_of(x_scale, w_scale, out, ldo, M, n_out, status);
  p.res = (const bf16*)res;
  p.res_ld = res_ld;
  return run<EPI_RESIDUAL>((const uint8_t*)x, ldx, (const uint8_t*)W, p, K, stream);
}

extern "C" int tsds_linear_swiglu_fp8(const void* x, int ldx, const float* x_scale, const void* W,
                                      const float* w_scale, void* out, int ldo, int M, int n_out, int K,
                                      int32_t* status, tsds_stream_t stream) {
  const int st = check(x, ldx, x_scale, W, w_scale, out, ldo, M, n_out, K, status);
  if (st != TSDS_OK || M == 0) return st;
  return run<EPI_SWIGLU>((const uint8_t*)x, ldx, (const uint8_t*)W,
                         args_of(x_scale, w_scale, out, ldo, M, n_out, status), K, stream);
}
