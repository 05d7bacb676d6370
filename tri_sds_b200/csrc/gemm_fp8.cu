// 8-bit projection on the tcgen05 tensor cores (sm_100a): e4m3 weights with
// a scale per output channel, e4m3 activations with a scale per token row.
//
//   out[m][j] = epilogue( (sum_k W[j][k] X[m][k]) * sx[m] * sw[j] )
//
// Weight rows j fill the MMA's M = 128, token rows m are its N (at most 256
// per block), K goes in blocks of 128 bytes.  A unit is one weight tile times
// one token block; two schedules, by the number of units:
//
// * Few units (at most the CTAs that are resident at once): a unit's K range is
//   split over a cluster of C CTAs, C as large as keeps the launch resident, so
//   that the weights stream through every SM at once.  Each CTA sums its share
//   in TMEM; at the end every CTA stores its fp32 partial in its own shared
//   memory and, after one cluster barrier, finishes 1/C of the token rows
//   from all C partials, read over distributed shared memory in rank order.
//   No partial goes through global memory, there is no workspace, no counter
//   and no atomic, and a call always gives the same bits.
// * Many units: persistent CTAs take whole units in turn (C = 1) with two
//   accumulators in TMEM, so the epilogue of one unit runs under the main
//   loop of the next and the ring never drains.
//
// Above 128 token rows a tile's X bytes outweigh its weights', and two CTAs
// form a pair (tcgen05 cta_group::2): a unit is 256 weight rows, each CTA stages
// its 128 of them and half of the token rows, one thread of the leader issues
// the MMAs of both, and each CTA finishes the 128 rows in its own TMEM.
//
// Warp 0 requests the tiles (TMA, 128-byte swizzle), warp 1 issues
// tcgen05.mma kind::f8f6f4 (fp32 accumulators in TMEM), warps 2-5 drain the
// accumulators.  Before the dependency wait the first weight tiles are only
// prefetched into L2: the weights may come from an earlier kernel of the
// stream (tsds_quant_fp8), so they are read after it.
// Every mbarrier wait is bounded; a CTA that gives up records TSDS_E_TIMEOUT
// and still takes part in the cluster's barriers.
#include "common.cuh"
#include "linear.cuh"
#include "tc_core.cuh"

#include <type_traits>

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
constexpr int STAGING = 32 * TILE_J * 4;   // output staging of a persistent CTA
constexpr int SMEM_SIDE = 2048;          // static shared memory + the system's 1 KB per CTA

struct F8Args {
  int M, n_out, KT, C, blocks, rows;  // blocks of token rows, rows of each but the last
  int units, bufs;              // units of the launch; accumulators per CTA
  int npad, stages, b_bytes, chunk;
  int out_off;                  // C == 1: offset of the output staging (0: the ring, free by then)
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
  uint64_t full[RING], empty[RING], tfull[2], tempty[2], drain;
  uint32_t tmem;
  int abort;
  int given_up, peer_issued;   // pairs: a CTA of the cluster gave up; blocks that the leader's peer requested
};

template <int CG>
__device__ __forceinline__ void umma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum));
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum));
}

// Arrival on `bar` when every MMA issued so far is done: of this CTA, or (a
// pair) of both CTAs of the pair whose cluster ranks `pair` has set.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t pair) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)pair)
        : "memory");
  else
    umma_commit(bar);
}

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// whether `ok` holds in all 128 threads of the epilogue warps
__device__ __forceinline__ bool epi_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.red.and.pred q, 1, 128, p;\n"
      " selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.0f + expf(-g)); }

// CG: CTAs per unit; SPLIT: a unit's K over a cluster.  One CTA per SM as the
// register target: with ptxas's own choice (56 registers for the residual
// epilogue) the loads of the split epilogue no longer go out together (O at 128
// rows 17.6 us instead of 15.9).  Whole units of one CTA, which have few rows,
// must leave room for three CTAs per SM (gate/up at 26 rows 48 us with two).
template <int EPI, int CG, bool SPLIT>
__global__ void __launch_bounds__(THREADS, SPLIT || CG == 2 ? 1 : 3)
    f8_gemm_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap, F8Args p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ F8Shared sh;
  constexpr bool SW = EPI == EPI_SWIGLU;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int crank = p.C * CG > 1 ? (int)cluster_ctarank() : 0;
  const int half = crank % CG, rank = crank / CG;            // of the pair; of the K split
  const int first_unit = blockIdx.x / (p.C * CG), unit_step = gridDim.x / (p.C * CG);
  const uint32_t lead = crank - half, pair = 3u << lead;     // a pair's leader, and both its CTAs
  constexpr int ROWS = SW ? 64 : TILE_J;                     // output channels per CTA of a unit
  const int k_lo = rank * p.KT / p.C, nk = (rank + 1) * p.KT / p.C - k_lo;
  // unit -> this CTA's weight tile and first token row; token blocks fastest, so
  // that the units in flight share their weights through L2
  auto tile_of = [&](int u) { return u / p.blocks * CG + half; };
  auto row_of = [&](int u) { return (u - u / p.blocks * p.blocks) * p.rows; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], 4 * CG);   // one arrival per epilogue warp
    }
    mbar_init(&sh.drain, 1);
    sh.abort = sh.given_up = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                   "r"(p.bufs * p.tmem_cols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                   "r"(p.bufs * p.tmem_cols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_barrier();   // both CTAs' barriers and TMEM exist
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  uint8_t* a_smem = smem;
  uint8_t* b_smem = smem + p.stages * A_BYTES;
  pdl_trigger();
  int issued = 0;
  // What a thread of the epilogue works on: four channels of the tile (their
  // scales in registers) and every token row that is its turn.  The channels
  // are adjacent (8-byte accesses) where the buffers' alignment allows; else
  // `spread` apart, so that neighbouring threads' 2-byte accesses still are.
  struct Out {
    int j, step;      // first channel, distance of the next
    int count;        // channels inside the output
    bool vec;         // 8-byte accesses
    float sw[SW ? 2 : 1][4];
  };
  auto out_of = [&](int tile, int first, int t, int spread) {
    Out w;
    const int base = tile * ROWS, inside = p.n_out - base < ROWS ? p.n_out - base : ROWS;
    w.vec = (p.ldo % 4) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && inside % 4 == 0 &&
            (EPI != EPI_RESIDUAL || ((p.res_ld % 4) == 0 && (reinterpret_cast<uintptr_t>(p.res) & 7) == 0));
    w.step = w.vec ? 1 : spread;
    w.j = base + first + (spread == 1 || w.vec ? t * 4 : t);
    const int left = base + inside - w.j;
    w.count = left <= 0 ? 0 : ((left + w.step - 1) / w.step < 4 ? (left + w.step - 1) / w.step : 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w.sw[0][i] = i < w.count ? p.sw[w.j + i * w.step] : 0.f;
      if constexpr (SW) w.sw[1][i] = i < w.count ? p.sw[p.n_out + w.j + i * w.step] : 0.f;
    }
    return w;
  };
  // A row's residual, loaded ahead of its sums: the residual may be the output,
  // so a load cannot pass an earlier row's store.  FULL: all four channels are
  // inside the output; a warp alone on its scheduler pays each branch in full.
  auto load_res = [&](auto full, auto vec, const Out& w, int m) {
    uint2 v = make_uint2(0, 0);
    if constexpr (EPI == EPI_RESIDUAL) {
      const bf16* rp = p.res + (int64_t)m * p.res_ld + w.j;
      if (vec) {
        if (full || w.count > 0) v = *reinterpret_cast<const uint2*>(rp);
      } else {
        const uint16_t* r16 = reinterpret_cast<const uint16_t*>(rp);
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = full || i < w.count ? r16[i * w.step] : 0;
        v = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
      }
    }
    return v;
  };
  auto finish = [&](auto full, auto vec, const Out& w, int m, const float4 (&acc)[2], float sx, uint2 res) {
    const float a4[4] = {acc[0].x, acc[0].y, acc[0].z, acc[0].w};
    const float rv[4] = {bf_lo(res.x), bf_hi(res.x), bf_lo(res.y), bf_hi(res.y)};
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = a4[i] * sx * w.sw[0][i];
      if constexpr (SW) {
        const float b4[4] = {acc[1].x, acc[1].y, acc[1].z, acc[1].w};
        o[i] = silu(o[i]) * (b4[i] * sx * w.sw[1][i]);
      }
      if constexpr (EPI == EPI_RESIDUAL) o[i] += rv[i];
    }
    bf16* op = p.out + (int64_t)m * p.ldo + w.j;
    if (vec) {
      if (full || w.count > 0) *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (full || i < w.count) op[i * w.step] = f2bf(o[i]);
    }
  };
  using Yes = std::true_type;
  using No = std::false_type;

  // The residual's lines of rows m .. m + rows - 1 of a tile into L2, by the 128
  // epilogue threads while the tensor cores work
  auto prefetch_res = [&](int tile, int m, int rows) {
    if constexpr (EPI == EPI_RESIDUAL) {
      const int j = tile * TILE_J + (threadIdx.x & 1) * 64;
      if (j >= p.n_out) return;
      for (int i = ((int)threadIdx.x - 64) >> 1; i < rows; i += 64)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.res + (int64_t)(m + i) * p.res_ld + j));
    }
  };

  // Warps 0 and 1 run their loops as whole warps with one elected lane issuing:
  // ptxas keeps warp-uniform operands in uniform registers then (a loop inside
  // one lane's branch costs 300 ns per block for the MMAs alone, this one
  // 205 ns).  Ring position and phase are counted, not divided out of the block number.
  if (warp == 0) {
    if (elect_one()) {
      prefetch_tmap(&amap);
      prefetch_tmap(&bmap);
      const int tile = tile_of(first_unit);
      for (int i = 0; i < nk && i < p.stages; ++i) {
        tma_prefetch_l2_2d(&amap, (k_lo + i) * KB, tile * ROWS);
        if (SW) tma_prefetch_l2_2d(&amap, (k_lo + i) * KB, p.n_out + tile * ROWS);
      }
    }
    __syncwarp();
    pdl_wait();
    const int bytes = CG * (A_BYTES + p.b_bytes);   // a pair's land on the leader's barrier
    int s = 0;
    uint32_t phase = 1;   // a fresh barrier's previous phase counts as complete
    bool ok = true;
    for (int u = first_unit; ok && u < p.units; u += unit_step) {
      // a stage's weight rows: 128 of one matrix, or 64 gate and 64 up rows
      const int row0 = tile_of(u) * ROWS, row1 = p.n_out + row0;
      const int m0 = row_of(u) + half * (p.npad / CG);   // of a pair, half of the token rows each
      int x = k_lo * KB;
      for (int i = 0; i < nk; ++i, x += KB) {
        ok = warp_wait(&sh.empty[s], phase, p.wait_ns);
        if (!ok) break;
        if (elect_one()) {
          if (half == 0) mbar_arrive_expect_tx(&sh.full[s], bytes);
          uint8_t* a = a_smem + s * A_BYTES;
          if constexpr (CG == 2) {
            const uint32_t bar = mapa_shared(smem_u32(&sh.full[s]), lead);
            tma_load_2d_pair(a, &amap, bar, x, row0);
            if (SW) tma_load_2d_pair(a + A_BYTES / 2, &amap, bar, x, row1);
            tma_load_2d_pair(b_smem + s * p.b_bytes, &bmap, bar, x, m0);
          } else {
            tma_load_2d(a, &amap, &sh.full[s], x, row0);
            if (SW) tma_load_2d(a + A_BYTES / 2, &amap, &sh.full[s], x, row1);
            tma_load_2d(b_smem + s * p.b_bytes, &bmap, &sh.full[s], x, m0);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == p.stages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) {
      if (lane == 0) atomicExch(p.status, TSDS_E_TIMEOUT);
      *(volatile int*)&sh.abort = 1;
    }
  } else if (warp == 1) {
    bool ok = true;
    const uint64_t a0 = sdesc_sw128(smem_u32(a_smem)), b0 = sdesc_sw128(smem_u32(b_smem));
    int s = 0, buf = 0;
    uint32_t phase = 0, tphase = 1;
    for (int u = first_unit; half == 0 && ok && u < p.units; u += unit_step) {
      ok = warp_wait(&sh.tempty[buf], tphase, p.wait_ns);
      const uint32_t d = tmem + buf * p.tmem_cols;
      if (ok && elect_one()) tc_fence_after();
      for (int i = 0; ok && i < nk; ++i) {
        ok = warp_wait(&sh.full[s], phase, p.wait_ns);
        if (!ok) break;
        if (elect_one()) {
          tc_fence_after();
          const uint64_t a = a0 + (uint32_t)(s * A_BYTES >> 4), b = b0 + (uint32_t)(s * p.b_bytes >> 4);
#pragma unroll
          for (int kk = 0; kk < KB / 32; ++kk) umma_f8<CG>(d, a + kk * 2, b + kk * 2, p.idesc, (i | kk) != 0);
          commit<CG>(&sh.empty[s], pair);
        }
        __syncwarp();
        ++issued;
        if (++s == p.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      if (ok && elect_one()) commit<CG>(&sh.tfull[buf], pair);
      __syncwarp();
      if (++buf == p.bufs) {
        buf = 0;
        tphase ^= 1;
      }
    }
    if (!ok) {
      if (lane == 0) atomicExch(p.status, TSDS_E_TIMEOUT);
      *(volatile int*)&sh.abort = 1;
    }
  } else if constexpr (!SPLIT) {
    // ---- epilogue of whole units: each warp transposes 32 token rows at a time of
    // its 32 channels through 4 KB of its own, so that stores are 64-byte runs
    // and no warp waits for another (SwiGLU: a gate warp and its up warp share
    // 8 KB and take half of the rows each).  The next 32 columns of TMEM and
    // the residuals of the next 32 rows are on their way meanwhile.  With one
    // staging area for the block and a block barrier per 16 rows a unit of 256
    // rows took 8 us, more than its main loop up to K = 4096. ----
    pdl_wait();
    constexpr int PASS = SW ? 4 : 8;   // of 4 rows each, 8 threads to a row
    constexpr int BATCH = CG == 2 ? 4 : 1;   // passes whose sums a thread holds at once
    const int quarter = warp & 3;      // the TMEM lanes this warp may read
    const int strip = SW ? quarter & 1 : quarter;
    const int mine = SW ? (quarter >> 1) * 16 + lane / 8 : lane / 8;   // row of the first pass
    float* from = reinterpret_cast<float*>(smem + p.out_off) + strip * (SW ? 2048 : 1024);
    float* to = from + (SW ? (quarter >> 1) * 1024 : 0) + lane;
    auto strip_sync = [&] {
      if (!SW)
        __syncwarp();
      else if (strip == 0)
        asm volatile("bar.sync 2, 64;" ::: "memory");
      else
        asm volatile("bar.sync 3, 64;" ::: "memory");
    };
    int buf = 0;
    uint32_t tphase = 0;
    for (int u = first_unit; u < p.units; u += unit_step) {
      const Out w = out_of(tile_of(u), strip * 32, lane % 8, 8);
      const int m0 = row_of(u), rows = p.M - m0 < p.rows ? p.M - m0 : p.rows;
      prefetch_res(tile_of(u), m0, rows);
      const bool full = __all_sync(0xffffffffu, w.count == 4);
      struct Rows {   // what 32 rows take from global memory
        float sx;     // of row `lane`
        uint2 res[PASS];
      } in0, in1;
      auto load_rows = [&](Rows& in, int c) {
        in.sx = c + lane < rows ? p.sx[m0 + c + lane] : 0.f;
        const int m = m0 + c + mine;
        if (full && w.vec && c + 32 <= rows) {
#pragma unroll
          for (int i = 0; i < PASS; ++i) in.res[i] = load_res(Yes(), Yes(), w, m + i * 4);
        } else if (full && c + 32 <= rows) {
#pragma unroll
          for (int i = 0; i < PASS; ++i) in.res[i] = load_res(Yes(), No(), w, m + i * 4);
        } else {
#pragma unroll
          for (int i = 0; i < PASS; ++i)
            if (c + mine + i * 4 < rows) in.res[i] = load_res(No(), w.vec, w, m + i * 4);
        }
      };
      load_rows(in0, 0);
      // the four warps go on together or not at all
      const bool ok = mbar_wait(&sh.tfull[buf], tphase, p.wait_ns);
      if (!ok) {
        atomicExch(p.status, TSDS_E_TIMEOUT);
        *(volatile int*)&sh.abort = 1;
      }
      if (!epi_all(ok)) break;
      __syncwarp();
      tc_fence_after();
      const uint32_t at = tmem + buf * p.tmem_cols + ((uint32_t)(quarter * 32) << 16);
      uint32_t v[32];
      tmem_request32(at, v);
      // (TMEM columns come in powers of two from 32: those past the last row are there)
      auto do_rows = [&](const Rows& in, Rows& next, int c) {
        tmem_wait32(v);
        if (c + 32 >= rows) {   // this warp has read its part of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2)
              mbar_arrive_remote(mapa_shared(smem_u32(&sh.tempty[buf]), lead));   // the leader's MMAs reuse it
            else
              mbar_arrive(&sh.tempty[buf]);
          }
        }
        strip_sync();   // the rows before have been read
#pragma unroll
        for (int i = 0; i < 32; ++i) to[i * 32] = __uint_as_float(v[i]);
        strip_sync();
        if (c + 32 < rows) {
          tmem_request32(at + c + 32, v);
          load_rows(next, c + 32);
        }
        auto rest = [&](auto whole, auto vec) {
#pragma unroll
          for (int i0 = 0; i0 < PASS; i0 += BATCH) {
            float4 acc[BATCH][2];
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
#pragma unroll
              for (int h = 0; h < (SW ? 2 : 1); ++h) {
                const float* a = from + h * 1024 + (mine + (i0 + i) * 4) * 32 + (vec ? lane % 8 * 4 : lane % 8);
                acc[i][h] = vec ? *reinterpret_cast<const float4*>(a) : make_float4(a[0], a[8], a[16], a[24]);
              }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
              const int mc = mine + (i0 + i) * 4;
              const float sx = __shfl_sync(0xffffffffu, in.sx, mc);
              if (whole || c + mc < rows) finish(whole, vec, w, m0 + c + mc, acc[i], sx, in.res[i0 + i]);
            }
          }
        };
        if (full && w.vec && c + 32 <= rows)
          rest(Yes(), Yes());
        else if (full && c + 32 <= rows)
          rest(Yes(), No());
        else
          rest(No(), w.vec);
        __syncwarp();
      };
      for (int c = 0; c < rows; c += 64) {
        do_rows(in0, in1, c);
        if (c + 32 < rows) do_rows(in1, in0, c + 32);
      }
      if (++buf == p.bufs) {
        buf = 0;
        tphase ^= 1;
      }
    }
  }
  if constexpr (SPLIT) {
    pdl_wait();
    if (warp >= 2) {   // this CTA's share of the rows (of the first chunk)
      const int m0 = row_of(first_unit), rows = p.M - m0 < p.rows ? p.M - m0 : p.rows;
      const int cn = rows < p.chunk ? rows : p.chunk, lo = rank * cn / p.C;
      prefetch_res(tile_of(first_unit), m0 + lo, (rank + 1) * cn / p.C - lo);
    }
    __syncwarp();
    // tfull completes when every MMA has, so the ring is free for the partials
    if (!mbar_wait(&sh.tfull[0], 0, p.wait_ns)) {
      if (lane == 0) atomicExch(p.status, TSDS_E_TIMEOUT);
      *(volatile int*)&sh.abort = 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const bool alive = !*(volatile int*)&sh.abort;
  if (!alive) {  // uniform: copies and MMAs in flight finish (bounded) before TMEM is freed
    // (a pair's copies at the end, when neither CTA requests any more)
    if (CG == 1 && warp == 0 && lane == 0) drain_tma_ring(sh.full, p.stages, issued);
    if (warp == 1 && lane == 0 && issued > 0) {
      commit<CG>(&sh.drain, pair);
      mbar_wait(&sh.drain, 0, 20000000ull);
    }
    __syncthreads();
  }
  if constexpr (SPLIT) {
    // ---- epilogue of a split unit: token rows in chunks that fit the ring, partials [chunk][128] fp32 ----
    float* part = reinterpret_cast<float*>(smem);
    constexpr int G = SW ? 16 : 32, STEP = THREADS / G;
    const int g4 = threadIdx.x % G * 4;
    const Out w = out_of(tile_of(first_unit), 0, threadIdx.x % G, 1);
    const int m0 = row_of(first_unit), rows = p.M - m0 < p.rows ? p.M - m0 : p.rows;
    for (int c0 = 0; c0 < rows; c0 += p.chunk) {
      const int cn = rows - c0 < p.chunk ? rows - c0 : p.chunk;
      if (alive && warp >= 2) {
        const int quarter = warp & 3;
        float* mine = part + quarter * 32 + lane;
        for (int c = 0; c < cn; c += 16) {
          float v[16];
          tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c0 + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < cn) mine[(c + i) * TILE_J] = v[i];
        }
      }
      cluster_barrier();
      if (alive && w.count > 0) {
        // this CTA's token rows, from every CTA's partials in rank order; of pairs
        // so many rows at once that eight loads are on their way
        const int hi = (rank + 1) * cn / p.C;
        auto join = [&](auto at_once, auto most) {
          constexpr int NR = decltype(at_once)::value, MC = decltype(most)::value;
          for (int m1 = rank * cn / p.C + (int)threadIdx.x / G; m1 < hi; m1 += STEP * NR) {
            uint2 res[NR];
            float sx[NR];
            float4 acc[NR][2];
#pragma unroll
            for (int r = 0; r < NR; ++r)
              if (m1 + r * STEP < hi) {
                res[r] = load_res(No(), w.vec, w, m0 + c0 + m1 + r * STEP);
                sx[r] = p.sx[m0 + c0 + m1 + r * STEP];
              }
#pragma unroll
            for (int h = 0; h < (SW ? 2 : 1); ++h) {
              float4 f[NR][MC];
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                const uint32_t at = smem_u32(part + (m1 + r * STEP) * TILE_J + g4) + h * 256;
#pragma unroll
                for (int q = 0; q < MC; ++q)
                  if (q < p.C && m1 + r * STEP < hi) f[r][q] = ld_peer(mapa_shared(at, q * CG + half));
              }
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                acc[r][h] = f[r][0];
#pragma unroll
                for (int q = 1; q < MC; ++q)
                  if (q < p.C) acc[r][h] = add4(acc[r][h], f[r][q]);
              }
            }
#pragma unroll
            for (int r = 0; r < NR; ++r)
              if (m1 + r * STEP < hi) finish(No(), w.vec, w, m0 + c0 + m1 + r * STEP, acc[r], sx[r], res[r]);
          }
        };
        // (of one-CTA units, which run up to three to an SM, one row: more would
        // take the registers of the third)
        if constexpr (CG == 1)
          join(std::integral_constant<int, 1>(), std::integral_constant<int, MAX_C>());
        else if (p.C <= 2)
          join(std::integral_constant<int, 4>(), std::integral_constant<int, 2>());
        else
          join(std::integral_constant<int, 2>(), std::integral_constant<int, 4>());
      }
      cluster_barrier();   // the peers are done with this CTA's partials
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) {
    if (!alive && threadIdx.x < p.C * CG) st_peer(mapa_shared(smem_u32(&sh.given_up), threadIdx.x), 1);
  }
  __syncthreads();
  if constexpr (CG == 2) {
    cluster_barrier();   // the pair is done with both TMEM halves and barriers
    if (*(volatile int*)&sh.given_up) {
      // (the same in every CTA of the cluster)  A pair's copies all land on the leader's
      // barriers, but each CTA requested its own: what the peer requested beyond the
      // leader's count is expected now, so that the drain waits for it too.  What it
      // requested less never comes, and costs the drain its limit.
      if (half == 1 && warp == 0 && lane == 0) st_peer(mapa_shared(smem_u32(&sh.peer_issued), lead), issued);
      cluster_barrier();
      if (half == 0 && warp == 0 && lane == 0) {
        const int peer = *(volatile int*)&sh.peer_issued;
        for (int j = issued; j < peer; ++j) mbar_arrive_expect_tx(&sh.full[j % p.stages], A_BYTES + p.b_bytes);
        drain_tma_ring(sh.full, p.stages, peer > issued ? peer : issued);
      }
      cluster_barrier();
    }
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.bufs * p.tmem_cols));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.bufs * p.tmem_cols));
  }
}

// One way to place a launch: CTAs per unit, CTAs per SM, K split, ring depth.
struct Shape {
  int CG = 1, C = 1, stages = 0;
  bool persistent = false;
  long long grid = 0;
  double cost = 1e30;   // estimated time, us
};

size_t smem_budget(int ctas) {
  const int budget = SMEM_SM / ctas - SMEM_SIDE;
  return budget < SMEM_CTA ? budget : SMEM_CTA;
}

// Clusters of `size` CTAs resident at once, `ctas` CTAs per SM.  Asked of a kernel
// with the same threads and shared memory, never launched: of one that allocates
// TMEM the runtime says one CTA per SM.
__global__ void __launch_bounds__(THREADS) occupancy_kernel() {}
int resident(int dev, int ctas, int size) {
  static tsds_cluster_counts known[3];
  return tsds_resident_clusters(dev, occupancy_kernel, THREADS, smem_budget(ctas), size, known[ctas - 1]);
}

// What bounds the kernel up to 256 token rows is how many bytes of weights are
// in flight: an SM holds a few hundred open requests, and a DRAM access
// takes about a microsecond, so the rate grows with (CTAs x stages x 16 KB) up to
// about 16 MB: 0.4 bytes per us for each in flight.  A launch whose units are not
// all resident at once goes in rounds, and its last round lasts at least as long
// as one unit on one SM.  Joining the parts of a split unit takes a microsecond
// and 20 ns per row.  Measured: q/k/v (80 tiles) at 26 rows 13.1 us on one CTA per
// SM (C = 1, 10 MB in flight), 12.0 on two (C = 3, 16 MB and more); at 200 rows
// (40 pairs) 18.2 on one (C = 1), 21.4 on two (C = 3); gate/up (400 tiles) at 128
// rows 49.7 us on one persistent CTA per SM, 60.4 on two.
Shape shape_of(int dev, int tiles, int blocks, int KT, int npad, int tmem_cols, int ctas, int CG) {
  Shape h;
  h.CG = CG;
  const int sms = tsds_tc_num_sms();
  const long long units = (long long)((tiles + CG - 1) / CG) * blocks;
  const long long places = (long long)sms * ctas / CG;   // units resident at once
  h.persistent = units > places;
  if (ctas * tmem_cols * (h.persistent ? 2 : 1) > 512) return h;
  const int budget = (int)smem_budget(ctas);
  h.stages = (budget - 1024 - (h.persistent ? STAGING : 0)) / (A_BYTES + npad / CG * KB);
  if (h.stages > RING) h.stages = RING;
  // K over as many CTAs as keep the whole launch resident, with a tenth of the
  // places to spare for the next one: a cluster that has to wait for a place
  // doubles the time (26 rows, 6144 -> 2048: 12.5 us with 16 clusters of 8, of
  // which 15 fit, 6.8 with 16 of 6)
  while ((h.C + 1) * CG <= MAX_C && KT >= 2 * (h.C + 1) && units * (h.C + 1) * 10 <= places * 9 &&
         units <= resident(dev, ctas, (h.C + 1) * CG))
    ++h.C;
  h.grid = h.persistent ? places : units * h.C;   // in units' CTAs, CG of them each
  double waste = 1.0;
  if (h.persistent) {
    const long long full = (units - 1) / places;   // rounds before the last
    const double last = (double)(units - full * places) * CG / sms;
    waste = (full * ctas + (last > 1.0 ? last : 1.0)) * sms / (units * CG);
  }
  double flight = (double)h.grid * CG * h.stages * A_BYTES;
  if (flight > 16e6) flight = 16e6;
  const double bytes = (double)units * CG * KT * A_BYTES;
  h.cost = waste * bytes / (0.4 * flight);   // us
  if (h.C > 1) h.cost += 1 + 0.02 * (npad + h.C);
  return h;
}

// Token rows per block, a multiple of 32 above 256 rows: what takes least by this
// estimate, 0.34 us for a block of K and 256 rows on a pair of CTAs, the epilogue's share of
// 32 rows, units in rounds or, all resident, their K over several pairs, whose
// parts then have to be joined.  2048 rows into 5120 (20 pairs of tiles) are 3 rounds of 74
// units with blocks of 256 rows, and 3 rounds of three quarters the length with
// blocks of 192.
int block_rows(int M, int tiles, int KT) {
  if (M <= MAX_ROWS) return MAX_ROWS;
  const long long pairs = (tiles + 1) / 2, places = tsds_tc_num_sms() / 2;
  int best = MAX_ROWS;
  double least = 0;
  for (int r = MAX_ROWS; r > TILE_J; r -= 32) {   // (128 rows and fewer are not for pairs)
    const long long units = pairs * ((M + r - 1) / r), rounds = (units + places - 1) / places;
    long long C = places * 9 / (units * 10);
    C = C < 1 ? 1 : (C > MAX_C / 2 ? MAX_C / 2 : C);
    const double t = rounds * (r + 32) * KT * (0.34 / 256) / C + (C > 1 ? 1 + 0.02 * r : 0);
    if (least == 0 || t < least) {
      least = t;
      best = r;
    }
  }
  return best;
}

template <int EPI, int CG, bool SPLIT>
int launch(const CUtensorMap& amap, const CUtensorMap& bmap, const F8Args& p, unsigned grid, size_t smem,
           cudaStream_t stream) {
  static tsds_device_flags limit_set;
  const int st = tsds_smem_limit_once(f8_gemm_kernel<EPI, CG, SPLIT>, SMEM_CTA, limit_set);
  if (st != TSDS_OK) return st;
  if (p.C * CG > 1)
    tsds_launch_cluster(f8_gemm_kernel<EPI, CG, SPLIT>, dim3(grid), dim3(THREADS), smem, stream, p.C * CG, amap, bmap,
                        p);
  else
    tsds_launch(f8_gemm_kernel<EPI, CG, SPLIT>, dim3(grid), dim3(THREADS), smem, stream, amap, bmap, p);
  return tsds_launch_status();
}

template <int EPI>
int run(const uint8_t* x, int ldx, const uint8_t* w, F8Args p, int K, cudaStream_t stream) {
  constexpr bool SW = EPI == EPI_SWIGLU;
  const int tiles = SW ? (p.n_out + 63) / 64 : (p.n_out + TILE_J - 1) / TILE_J;
  p.KT = (K + KB - 1) / KB;
  p.rows = block_rows(p.M, tiles, p.KT);
  p.blocks = (p.M + p.rows - 1) / p.rows;
  TSDS_RETURN_IF((long long)tiles * p.blocks > 0x3fffffffll, TSDS_E_UNSUPPORTED);
  const int widest = p.M < p.rows ? p.M : p.rows;
  p.npad = (widest + 15) / 16 * 16;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.npad) p.tmem_cols *= 2;
  const int dev = tsds_device();
  TSDS_RETURN_IF(dev < 0, TSDS_E_DEVICE);
  Shape best;
  for (int CG = 1; CG <= (p.npad > TILE_J ? 2 : 1); ++CG)
    for (int ctas = 1; ctas <= 3; ++ctas) {
      const Shape h = shape_of(dev, tiles, p.blocks, p.KT, p.npad, p.tmem_cols, ctas, CG);
      if (h.stages >= 2 && h.cost <= best.cost) best = h;
    }
  TSDS_RETURN_IF(best.stages < 2, TSDS_E_UNSUPPORTED);
  p.units = (tiles + best.CG - 1) / best.CG * p.blocks;
  p.C = best.C;
  p.bufs = best.persistent ? 2 : 1;
  p.stages = best.stages;
  p.b_bytes = p.npad / best.CG * KB;
  const int ring = p.stages * (A_BYTES + p.b_bytes);
  p.out_off = best.persistent ? ring : 0;
  size_t smem = (size_t)ring + (best.persistent ? STAGING : 0) + 1024;
  // A CTA's part of the SM's shared memory is at least its part of TMEM's 512
  // columns, so CTAs that fit an SM never wait for columns there: a cluster
  // whose CTA waited for another stream's, and that one for this, would hang both.
  const size_t least = (size_t)p.bufs * p.tmem_cols * SMEM_SM / 512 - SMEM_SIDE;
  if (smem < least) smem = least < SMEM_CTA ? least : SMEM_CTA;
  p.chunk = ring / (TILE_J * 4) / 16 * 16;
  if (p.chunk > p.npad) p.chunk = p.npad;
  p.idesc = (1u << 4) | ((uint32_t)(p.npad >> 3) << 17) | ((uint32_t)(TILE_J * best.CG >> 4) << 24);
  p.wait_ns = tsds_get_wait_limit_ns();
  CUtensorMap amap, bmap;
  int st = tsds_make_tmap_2d_u8(&amap, w, K, SW ? 2 * (uint64_t)p.n_out : p.n_out, K, KB, SW ? 64 : TILE_J);
  if (st != TSDS_OK) return st;
  st = tsds_make_tmap_2d_u8(&bmap, x, K, p.M, ldx, KB, p.npad / best.CG);
  if (st != TSDS_OK) return st;
  const unsigned grid = (unsigned)(best.grid * best.CG);
  if (best.CG == 2)
    return p.C > 1 ? launch<EPI, 2, true>(amap, bmap, p, grid, smem, stream)
                   : launch<EPI, 2, false>(amap, bmap, p, grid, smem, stream);
  return p.C > 1 ? launch<EPI, 1, true>(amap, bmap, p, grid, smem, stream)
                 : launch<EPI, 1, false>(amap, bmap, p, grid, smem, stream);
}

// w_rows: rows of W
int check(const void* x, int ldx, const float* sx, const void* w, int64_t w_rows, const float* sw, const void* out,
          int ldo, int M, int n_out, int K, const int32_t* status) {
  TSDS_RETURN_IF(M < 0 || n_out <= 0 || K <= 0 || (K % 16) != 0 || ldx < K || ldo < n_out || n_out > (1 << 29),
                 TSDS_E_INVALID);
  // rows and K are rounded up to whole blocks in 32 bits
  TSDS_RETURN_IF(M > (1 << 30) || K > (1 << 30), TSDS_E_UNSUPPORTED);
  if (M == 0) return TSDS_OK;
  TSDS_RETURN_IF(!x || !sx || !w || !sw || !out || !status, TSDS_E_INVALID);
  TSDS_RETURN_IF(!tsds_aligned16(x) || !tsds_aligned16(w) || (ldx % 16), TSDS_E_ALIGN);
  // (a block's rows are stored while others still read theirs)
  const tsds_rows o = {out, M, ldo * (int64_t)2, n_out * (int64_t)2};
  TSDS_RETURN_IF(tsds_overlap(o, {x, M, ldx, K}) || tsds_overlap(o, {w, 1, 0, w_rows * K}), TSDS_E_INVALID);
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
  const int st = check(x, ldx, x_scale, W, n_out, w_scale, out, ldo, M, n_out, K, status);
  if (st != TSDS_OK || M == 0) return st;
  return run<EPI_STORE>((const uint8_t*)x, ldx, (const uint8_t*)W,
                        args_of(x_scale, w_scale, out, ldo, M, n_out, status), K, stream);
}

extern "C" int tsds_linear_residual_fp8(const void* x, int ldx, const float* x_scale, const void* W,
                                        const float* w_scale, const void* res, int res_ld, void* out, int ldo, int M,
                                        int n_out, int K, int32_t* status, tsds_stream_t stream) {
  const int st = check(x, ldx, x_scale, W, n_out, w_scale, out, ldo, M, n_out, K, status);
  if (st != TSDS_OK) return st;
  TSDS_RETURN_IF(res_ld < n_out, TSDS_E_INVALID);
  if (M == 0) return TSDS_OK;
  TSDS_RETURN_IF(!res || (res == out && res_ld != ldo), TSDS_E_INVALID);
  TSDS_RETURN_IF(res != out && tsds_overlap({out, M, ldo * (int64_t)2, n_out * (int64_t)2},
                                            {res, M, res_ld * (int64_t)2, n_out * (int64_t)2}),
                 TSDS_E_INVALID);
  F8Args p = args_of(x_scale, w_scale, out, ldo, M, n_out, status);
  p.res = (const bf16*)res;
  p.res_ld = res_ld;
  return run<EPI_RESIDUAL>((const uint8_t*)x, ldx, (const uint8_t*)W, p, K, stream);
}

extern "C" int tsds_linear_swiglu_fp8(const void* x, int ldx, const float* x_scale, const void* W,
                                      const float* w_scale, void* out, int ldo, int M, int n_out, int K,
                                      int32_t* status, tsds_stream_t stream) {
  const int st = check(x, ldx, x_scale, W, 2 * (int64_t)n_out, w_scale, out, ldo, M, n_out, K, status);
  if (st != TSDS_OK || M == 0) return st;
  return run<EPI_SWIGLU>((const uint8_t*)x, ldx, (const uint8_t*)W,
                         args_of(x_scale, w_scale, out, ldo, M, n_out, status), K, stream);
}
