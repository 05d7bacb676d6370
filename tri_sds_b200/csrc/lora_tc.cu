// Low-rank adapters beside a shared projection, for many token rows, on the
// tcgen05 tensor cores (sm_100a); the formula and the one-launch kernel for few
// rows are in lora.cu.  Two launches:
//
// * shrink: t[m][u] = scale * sum_k A[u][k] x[m][k].  A cluster of 8 CTAs takes
//   a block of token rows and one adapter of those that occur in it, a CTA 1/8
//   of K.  Rank rows fill the MMA's M, token rows are its N; x and A stream
//   through a TMA ring.  The partial sums meet over distributed shared memory
//   (rank order: always the same bits), and t is stored as two bf16 words
//   (hi + lo, 16 bits of it), so its rounding is far below the output's.
// * expand: out = y + B t^T.  A block is 128 token rows, which fill the MMA's M, so a
//   lane of TMEM is a row; channels are its N.  The CTAs of a block take its channel
//   tiles in turn: the y tile comes by TMA, the products of every adapter of the block
//   (both words of t into one accumulator, two of which alternate) are added to
//   their rows in shared memory, and the tile leaves by TMA once.
//
// The bytes of x and y bound both (B and A come from L2 after their first
// use); the MMAs are a few percent of the tensor cores' rate.  2048 rows, K 5120,
// rank 32 into q/k/v of 10240 columns: 30.0 us, shrink about 13 of them (21 MB of x, the
// rest the chain from launch to reduction) and expand 17 (84 MB of y and out,
// 5 TB/s).  Asking for y from shrink already, into L2, cost 7 us.
//
// shrink lets its successor start only after its own dependency wait, so
// everything before shrink is complete when expand begins, and expand may
// read y, B and the indices before its wait; only t comes after it.  With one CTA of expand
// per SM that starts where shrink has left an SM: their shared memory does not fit together.
#include "common.cuh"
#include "linear.cuh"
#include "lora.cuh"
#include "tc_core.cuh"

using namespace tsds;
using namespace tsds::tc;
using namespace tsds::lora;

namespace {

constexpr int CL = 8;               // CTAs per shrink cluster
constexpr int THREADS = 192;        // TMA warp, MMA warp, four epilogue warps
constexpr int BKE = 64;             // elements of K (or ranks) per block: a 128-byte swizzle row
constexpr int RING = 8;             // most stages
constexpr int SHRINK_SMEM = 110 * 1024;   // two CTAs per SM, with their static shared memory

struct ShrinkArgs {
  LoraArgs l;
  bf16* t;             // [M][2][ld_t]: hi, lo
  int ld_t, Rp;        // columns of t; columns per slice
  int nt, blocks;      // token rows per block, blocks
  int arows, bx;       // rank rows per pass; rows of a small box
  int KT, stages, stage_bytes;
  uint32_t idesc;
  int tmem_cols;
  uint64_t wait_ns;
};

struct ShrinkShared {
  Tile tile;
  uint64_t full[RING], empty[RING], tfull, drain;
  uint32_t tmem;
  int abort;
};

// TMEM columns for the CTA, by one whole warp, before anything else: the SM's
// next CTA does not start until this one has given its permit to allocate back
// (taken after the rows' grouping it held every second CTA up for 5 us).
__device__ __forceinline__ void tmem_take(uint32_t* to, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(to)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_give(uint32_t tmem, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}

// A tile of shared memory to global memory, by one thread; stores are waited for in groups.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* smem_src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// all but the last N groups have read their shared memory
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void give_up(int32_t* status, int* abort, int lane) {
  if (lane == 0) atomicExch(status, TSDS_E_TIMEOUT);
  *(volatile int*)abort = 1;
}

__global__ void __launch_bounds__(THREADS)
    shrink_kernel(const __grid_constant__ CUtensorMap a_all, const __grid_constant__ CUtensorMap a_box,
                  const __grid_constant__ CUtensorMap xmap, ShrinkArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ ShrinkShared sh;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  if (warp == 1) tmem_take(&sh.tmem, p.tmem_cols);
  // every block's first adapter before any block's second: clusters without one come last
  const int unit = blockIdx.x / CL, slot = unit / p.blocks, row0 = (unit - slot * p.blocks) * p.nt;
  if (warp == 0 && elect_one()) {
    prefetch_tmap(&a_all);
    prefetch_tmap(&xmap);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    mbar_init(&sh.tfull, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  pdl_wait();
  pdl_trigger();   // after the wait: expand reads what comes before this kernel without one
  group_rows(p.l, sh.tile, row0, p.nt, rank == 0 && slot == 0, false);
  tc_fence_after();   // (group_rows ends with a barrier)
  const uint32_t tmem = sh.tmem;
  int adapters = 0;
#pragma unroll
  for (int w = 0; w < MAX_TILE / 32; ++w) adapters += __popc(sh.tile.leads[w]);
  if (adapters <= slot) {   // a cluster whose turn never comes
    if (warp == 1) tmem_give(tmem, p.tmem_cols);
    return;
  }
  float* part = reinterpret_cast<float*>(smem);   // [nt][128], in the ring once it is free
  const int k_lo = rank * p.KT / CL, nk = (rank + 1) * p.KT / CL - k_lo;
  int s = 0, issued = 0;                 // ring position, blocks so far (warps 0 and 1)
  uint32_t phase = warp == 0 ? 1 : 0, tphase = 0;
  bool alive = true;

  uint32_t leads = sh.tile.leads[0];
  for (int gi = 0, word = 0; gi < adapters; ++gi, leads &= leads - 1) {
    while (leads == 0) leads = sh.tile.leads[++word];
    if (gi % p.l.slots != slot) continue;
    const Adapter ad = adapter_of(p.l, sh.tile, sh.tile.id[word * 32 + __ffs(leads) - 1]);
    const int ra16 = (ad.ra + 15) / 16 * 16;
    for (int u0 = 0; ad.ra > 0 && u0 < p.l.S * p.l.R; u0 += p.arows) {   // rank rows u0 .. u0 + arows - 1
      const bool all = ad.ra == p.l.R;
      if (warp == 0 && alive) {
        // small boxes of this pass: only the ranks that the adapter uses
        uint32_t boxes = 0;
        if (!all)
          for (int i = 0, u = u0; u < u0 + p.arows && u < p.l.S * p.l.R; ++i, u += p.bx)
            if (u % p.l.R < ad.ra) boxes |= 1u << i;
        const int bytes = p.nt * 128 + (all ? p.arows : __popc(boxes) * p.bx) * 128;
        for (int i = 0; i < nk; ++i) {
          alive = warp_wait(&sh.empty[s], phase, p.wait_ns);
          if (!alive) break;
          if (elect_one()) {
            uint8_t* a = smem + s * p.stage_bytes;
            const int k = (k_lo + i) * BKE, a_row = ad.id * p.l.S * p.l.R;
            mbar_arrive_expect_tx(&sh.full[s], bytes);
            tma_load_2d(a + p.arows * 128, &xmap, &sh.full[s], k, row0);
            if (all) {
              tma_load_2d(a, &a_all, &sh.full[s], k, a_row + u0);
            } else {
              for (uint32_t b = boxes; b; b &= b - 1) {
                const int u = (__ffs(b) - 1) * p.bx;
                tma_load_2d(a + u * 128, &a_box, &sh.full[s], k, a_row + u0 + u);
              }
            }
          }
          __syncwarp();
          ++issued;
          if (++s == p.stages) {
            s = 0;
            phase ^= 1;
          }
        }
        if (!alive) give_up(p.l.status, &sh.abort, lane);
      } else if (warp == 1 && alive) {
        for (int i = 0; i < nk; ++i) {
          alive = warp_wait(&sh.full[s], phase, p.wait_ns);
          if (!alive) break;
          if (elect_one()) {
            tc_fence_after();
            const uint64_t a = sdesc_sw128(smem_u32(smem + s * p.stage_bytes));
            const uint64_t b = sdesc_sw128(smem_u32(smem + s * p.stage_bytes + p.arows * 128));
#pragma unroll
            for (int kk = 0; kk < BKE / 16; ++kk) umma_bf16(tmem, a + kk * 2, b + kk * 2, p.idesc, (i | kk) != 0);
            umma_commit(&sh.empty[s]);
          }
          __syncwarp();
          ++issued;
          if (++s == p.stages) {
            s = 0;
            phase ^= 1;
          }
        }
        if (alive && elect_one()) umma_commit(&sh.tfull);
        __syncwarp();
        if (!alive) give_up(p.l.status, &sh.abort, lane);
      }
      __syncwarp();
      // a CTA without a block of K (K short of 8 blocks) has nothing to wait for
      if (nk > 0) {
        if (alive && !mbar_wait(&sh.tfull, tphase, p.wait_ns)) give_up(p.l.status, &sh.abort, lane);
        tphase ^= 1;
      }
      __syncwarp();
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
      alive = !*(volatile int*)&sh.abort;
      if (alive && warp >= 2) {
        const int quarter = warp & 3;
        float* mine = part + quarter * 32 + lane;
        for (int c = 0; c < p.nt; c += 16) {
          float v[16];
          if (nk > 0) {
            tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) mine[(c + i) * TILE_J] = v[i];
        }
        tc_fence_before();
      }
      cluster_barrier();
      // this CTA's token rows: four ranks at a time, from every CTA's partials
      const int share = p.nt / CL, groups = p.l.S * (ra16 / 4);
      for (int e = threadIdx.x; alive && e < share * groups; e += THREADS) {
        const int i = rank * share + e / groups, gq = e % groups, sl = gq / (ra16 / 4), r = (gq - sl * (ra16 / 4)) * 4;
        const int u = sl * p.l.R + r - u0;
        // columns past the rank are zeros, written with the pass their slice begins in
        const bool sum = r < ad.ra && u >= 0 && u < p.arows;
        const int u_first = sl * p.l.R;
        if (!sum && !(r >= ad.ra && u_first >= u0 && u_first < u0 + p.arows)) continue;
        if (sh.tile.id[i] != ad.id) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (sum) {
          const uint32_t at = smem_u32(part + i * TILE_J + u);
          float4 f[CL];
#pragma unroll
          for (int k = 0; k < CL; ++k) f[k] = ld_peer(mapa_shared(at, k));
          float4 a = f[0];
#pragma unroll
          for (int k = 1; k < CL; ++k) a = make_float4(a.x + f[k].x, a.y + f[k].y, a.z + f[k].z, a.w + f[k].w);
          const float w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = r + k < ad.ra ? w[k] * ad.scale : 0.f;
        }
        float h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) two_words(v[k], h[k], l[k]);
        bf16* to = p.t + (int64_t)(row0 + i) * 2 * p.ld_t + sl * p.Rp + r;
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf2(h[0], h[1]), pack_bf2(h[2], h[3]));
        *reinterpret_cast<uint2*>(to + p.ld_t) =
            make_uint2(pack_bf2(l[0], l[1]), pack_bf2(l[2], l[3]));
      }
      // the peers are done with this CTA's partials; the ring may be loaded again
      fence_proxy_async();
      cluster_barrier();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (sh.abort) {
    if (warp == 0 && lane == 0 && issued > 0) drain_tma_ring(sh.full, p.stages, issued);
    if (warp == 1 && lane == 0 && issued > 0) drain_mma<1>(&sh.drain);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_give(tmem, p.tmem_cols);
  }
}

constexpr int XM = 128;                     // token rows of an expand block: the MMA's M
constexpr int X_THREADS = 384;              // B/t warp, MMA warp, y/out warp, an idle one, eight epilogue warps
constexpr int BOX = XM * 128;               // 128 rows of 128 bytes: of t (64 ranks), B or y (64 channels)
constexpr int X_SMEM = 208 * 1024 + 1024;   // 1 KB to align
constexpr int X_BUFS = 2;                   // accumulators
constexpr int X_RING = 8;                   // most stages of B

struct ExpandArgs {
  LoraArgs l;
  int ld_t, Rp, tiles, step, kb, tn;        // step: CTAs that share a block's tiles; kb: blocks of 64 ranks; tn: channels per tile
  int b_stages, y_stages;
  int first_tile[MAX_SLICES + 1];           // channel tiles where the slices begin
  uint64_t wait_ns;
};

// out, a map per slice: a tile that reaches past its slice's end is cut there
struct OutMaps {
  CUtensorMap of[MAX_SLICES];
};

struct ExpandShared {
  alignas(16) int32_t id[XM];   // adapter of each row; -1: none; -2: past the last row
  int32_t group[XM];            // its place among the block's adapters; -1: nothing to add
  int32_t gid[XM], grank[XM];   // the block's adapters: index, rank
  int32_t rank[NEAR];           // rank of the first adapters
  uint32_t leads[4];            // bits of the rows that are the first of their adapter
  int plain;                    // a row without an adapter
  uint64_t full[X_RING], empty[X_RING], t_full, t_empty, tfull[X_BUFS], tempty[X_BUFS], yfull[4], ydone[4], drain;
  uint32_t tmem;
  int abort;
};

// A channel tile: its slice, first channel, and the end of its slice.
struct Channels {
  int sl, lo, end;
};
__device__ __forceinline__ Channels channels_of(const ExpandArgs& p, int tile) {
  Channels c;
  c.sl = 0;
#pragma unroll
  for (int i = 1; i < MAX_SLICES; ++i)
    if (i < p.l.S && tile >= p.first_tile[i]) c.sl = i;
  c.lo = p.l.first_col[c.sl] + (tile - p.first_tile[c.sl]) * p.tn;
  c.end = p.l.first_col[c.sl + 1];
  return c;
}

// The block's rows by adapter, by the first 128 threads (the next 64 read ranks
// meanwhile); returns how many adapters have something to add.
__device__ __forceinline__ int group_block(const ExpandArgs& p, ExpandShared& sh, int row0) {
  const LoraArgs& l = p.l;
  const int tid = threadIdx.x, lane = tid & 31;
  int id = -2, m = row0 + tid;
  if (tid < XM) {
    if (m < l.M) {
      id = l.adapter[m];
      if (id < 0 || id >= l.n_adapters) id = -1;   // (shrink has reported an index past the last)
    }
    sh.id[tid] = id;
  } else if (tid < XM + NEAR) {
    const int a = tid - XM;
    sh.rank[a] = l.ranks && a < l.n_adapters ? l.ranks[a] : l.R;
  }
  if (tid == 0) sh.plain = 0;
  __syncthreads();
  int ra = 0, first = tid;
  if (tid < XM) {
    if (id >= 0) ra = id < NEAR ? sh.rank[id] : (l.ranks ? l.ranks[id] : l.R);
    ra = ra < 0 ? 0 : (ra > l.R ? l.R : ra);
#pragma unroll 4
    for (int j = XM - 4; j >= 0; j -= 4) {   // without a branch; the smallest row comes last
      const int4 v = *reinterpret_cast<const int4*>(sh.id + j);
      first = v.w == id ? j + 3 : first;
      first = v.z == id ? j + 2 : first;
      first = v.y == id ? j + 1 : first;
      first = v.x == id ? j : first;
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, ra > 0 && first == tid);
    if (lane == 0) sh.leads[tid >> 5] = bits;
    if (id != -2 && ra == 0) sh.plain = 1;
  }
  __syncthreads();
  auto before = [&](int row) {
    int n = __popc(sh.leads[row >> 5] & ((1u << (row & 31)) - 1));
#pragma unroll
    for (int w = 0; w < 3; ++w)
      if (w < row >> 5) n += __popc(sh.leads[w]);
    return n;
  };
  if (tid < XM) {
    const int g = before(first);
    sh.group[tid] = ra > 0 ? g : -1;
    if (ra > 0 && first == tid) {
      sh.gid[g] = id;
      sh.grank[g] = ra;
    }
  }
  __syncthreads();
  return __popc(sh.leads[0]) + __popc(sh.leads[1]) + __popc(sh.leads[2]) + __popc(sh.leads[3]);
}

template <int PER_SM>   // CTAs per SM
__global__ void __launch_bounds__(X_THREADS, PER_SM)
    expand_kernel(const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap tmap,
                  const __grid_constant__ CUtensorMap ymap, const __grid_constant__ OutMaps omap, ExpandArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ ExpandShared sh;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 1) tmem_take(&sh.tmem, X_BUFS * p.tn);
  const int block = blockIdx.x / p.step, row0 = block * XM, tile0 = blockIdx.x - block * p.step;
  const int items = (p.tiles - tile0 + p.step - 1) / p.step, boxes = p.tn / 64;
  uint8_t *t_smem = smem, *b_smem = t_smem + p.kb * 2 * BOX, *y_smem = b_smem + p.b_stages * p.kb * p.tn * 128;
  auto load_y = [&](int i) {   // by one thread
    const int s = i % p.y_stages, lo = channels_of(p, tile0 + i * p.step).lo;
    mbar_arrive_expect_tx(&sh.yfull[s], boxes * BOX);
    for (int h = 0; h < boxes; ++h) tma_load_2d(y_smem + (s * boxes + h) * BOX, &ymap, &sh.yfull[s], lo + h * 64, row0);
  };
  if (warp == 2 && lane == 0) {
    for (int i = 0; i < X_RING; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.yfull[i], 1);
      mbar_init(&sh.ydone[i], 8);    // one arrival per epilogue warp
    }
    for (int i = 0; i < X_BUFS; ++i) {
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], 8);
    }
    mbar_init(&sh.t_full, 1);
    mbar_init(&sh.t_empty, 1);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_barrier_init();
    fence_proxy_async();
    for (int i = 0; i < items && i < p.y_stages; ++i) load_y(i);   // y is complete before shrink starts
  }
  tc_fence_before();
  pdl_trigger();
  const int groups = group_block(p, sh, row0);
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // rows without an adapter stay as they are where out is y: then rows are
  // stored one by one
  const bool in_place = p.l.out == p.l.y, by_row = in_place && sh.plain;
  const bool any = groups > 0 || !in_place;
  int issued = 0, slices = 0;   // blocks of the B ring (warps 0 and 1), loads of t (warp 0)
  int y_issued = items < p.y_stages ? items : p.y_stages;
  bool ok = true;

  if (warp == 0) {
    int s = 0, sl = -1;
    uint32_t phase = 1;
    for (int i = 0; ok && i < items && groups > 0; ++i) {
      const Channels c = channels_of(p, tile0 + i * p.step);
      for (int g = 0; g < groups; ++g) {
        ok = warp_wait(&sh.empty[s], phase, p.wait_ns);
        if (!ok) break;
        const int id = sh.gid[g], kb = (sh.grank[g] + BKE - 1) / BKE;
        if (elect_one()) {
          mbar_arrive_expect_tx(&sh.full[s], kb * p.tn * 128);
          for (int k = 0; k < kb; ++k)
            tma_load_2d(b_smem + (s * p.kb + k) * p.tn * 128, &bmap, &sh.full[s], k * BKE, id * p.l.N + c.lo);
        }
        __syncwarp();
        ++issued;
        if (++s == p.b_stages) {
          s = 0;
          phase ^= 1;
        }
        if (sl != c.sl) {   // the slice's t; the first read that waits for shrink
          if (slices == 0)
            pdl_wait();
          else
            ok = warp_wait(&sh.t_empty, (slices - 1) & 1, p.wait_ns);
          if (!ok) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&sh.t_full, p.kb * 2 * BOX);
            for (int k = 0; k < p.kb * 2; ++k)   // hi, lo of each 64 ranks
              tma_load_2d(t_smem + k * BOX, &tmap, &sh.t_full, (k & 1) * p.ld_t + c.sl * p.Rp + (k >> 1) * BKE, row0);
          }
          __syncwarp();
          sl = c.sl;
          ++slices;
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc =
        (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.tn >> 3) << 17) | ((uint32_t)(XM >> 4) << 24);
    const uint64_t t0 = sdesc_sw128(smem_u32(t_smem));
    int s = 0, sl = -1, buf = 0;
    uint32_t phase = 0, tphase = 1, slice_phase = 1;
    for (int i = 0; ok && i < items && groups > 0; ++i) {
      const Channels c = channels_of(p, tile0 + i * p.step);
      if (sl != c.sl) {
        if (sl >= 0 && elect_one()) umma_commit(&sh.t_empty);   // the old slice's products are done
        __syncwarp();
        sl = c.sl;
        slice_phase ^= 1;
        ok = warp_wait(&sh.t_full, slice_phase, p.wait_ns);
      }
      for (int g = 0; ok && g < groups; ++g) {
        ok = warp_wait(&sh.tempty[buf], tphase, p.wait_ns) && warp_wait(&sh.full[s], phase, p.wait_ns);
        if (!ok) break;
        const int ra = sh.grank[g], steps = (ra + 15) / 16;   // of 16 ranks
        uint8_t* bs = b_smem + s * p.kb * p.tn * 128;
        if (ra & 15) {
          // the last step's ranks past the adapter's: B's columns there are not
          // part of it, whatever they hold
          const int from = ra & 63, to = ((ra + 15) & ~15) - (ra & ~63);
          uint8_t* b = bs + (ra / 64) * p.tn * 128;
          for (int row = lane; row < p.tn; row += 32)
            for (int k = from; k < to; ++k)
              *reinterpret_cast<uint16_t*>(b + row * 128 + (((k >> 3) ^ (row & 7)) << 4) + (k & 7) * 2) = 0;
          fence_proxy_async();
        }
        __syncwarp();
        if (elect_one()) {
          tc_fence_after();
          const uint64_t b0 = sdesc_sw128(smem_u32(bs));
          for (int k = 0; k < steps; ++k) {
            const uint64_t b = b0 + (uint32_t)((k >> 2) * p.tn * 128 >> 4) + (k & 3) * 2;
            const uint64_t t = t0 + (uint32_t)((k >> 2) * 2 * BOX >> 4) + (k & 3) * 2;
            umma_bf16(tmem + buf * p.tn, t + (BOX >> 4), b, idesc, k != 0);   // lo
            umma_bf16(tmem + buf * p.tn, t, b, idesc, 1);                     // hi
          }
          umma_commit(&sh.empty[s]);
          umma_commit(&sh.tfull[buf]);
        }
        __syncwarp();
        ++issued;
        if (++s == p.b_stages) {
          s = 0;
          phase ^= 1;
        }
        if (++buf == X_BUFS) {
          buf = 0;
          tphase ^= 1;
        }
      }
    }
  } else if (warp == 2) {
    if (any) {
      pdl_wait();   // what is stored may be what an earlier kernel still reads
      for (int i = 0; i < items; ++i) {
        ok = warp_wait(&sh.ydone[i % p.y_stages], (i / p.y_stages) & 1, p.wait_ns);
        if (!ok) break;
        if (lane == 0) {
          const Channels c = channels_of(p, tile0 + i * p.step);
          for (int h = 0; h < boxes && !by_row; ++h) {
            const int x = c.lo + h * 64;
            if (x < c.end)
              tma_store_2d(&omap.of[c.sl], x - p.l.first_col[c.sl], row0,
                           y_smem + (i % p.y_stages * boxes + h) * BOX);
          }
          bulk_commit();
          if (i > 0 && i - 1 + p.y_stages < items) {
            bulk_wait_read<1>();   // the item before has left its stage
            load_y(i - 1 + p.y_stages);
          }
        }
        __syncwarp();
        if (i > 0 && i - 1 + p.y_stages < items) ++y_issued;
      }
    }
  } else if (warp >= 4 && any) {
    // A lane is a token row: it adds its adapter's products to its row of the
    // y tile in shared memory, half of the tile's channels, 32 at a time.
    const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane, cols = p.tn / 2;
    const int mine = sh.group[row];
    bf16* out_row = p.l.out + (int64_t)(row0 + row) * p.l.ldo;
    int buf = 0;
    uint32_t tphase = 0;
    for (int i = 0; ok && i < items; ++i) {
      const int st = i % p.y_stages;
      ok = warp_wait(&sh.yfull[st], (i / p.y_stages) & 1, p.wait_ns);
      const Channels ch = channels_of(p, tile0 + i * p.step);
      for (int g = 0; ok && g < groups; ++g) {
        ok = warp_wait(&sh.tfull[buf], tphase, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        if (__any_sync(0xffffffffu, mine == g)) {
          for (int c = 0; c < cols; c += 32) {
            const int col = half * cols + c;   // of the tile
            uint32_t v[32];
            tmem_request32(tmem + buf * p.tn + ((uint32_t)(quarter * 32) << 16) + col, v);
            uint8_t* box = y_smem + (st * boxes + (col >> 6)) * BOX + row * 128;
            uint4* at[4];
            uint4 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              at[k] = reinterpret_cast<uint4*>(box + (((((col & 63) >> 3) + k) ^ (row & 7)) << 4));
              y[k] = *at[k];
            }
            tmem_wait32(v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float* d = reinterpret_cast<const float*>(v) + k * 8;
              y[k] = make_uint4(pack_bf2(bf_lo(y[k].x) + d[0], bf_hi(y[k].x) + d[1]),
                                pack_bf2(bf_lo(y[k].y) + d[2], bf_hi(y[k].y) + d[3]),
                                pack_bf2(bf_lo(y[k].z) + d[4], bf_hi(y[k].z) + d[5]),
                                pack_bf2(bf_lo(y[k].w) + d[6], bf_hi(y[k].w) + d[7]));
            }
            if (mine == g) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (!by_row)
                  *at[k] = y[k];
                else if (ch.lo + col + k * 8 < ch.end)
                  *reinterpret_cast<uint4*>(out_row + ch.lo + col + k * 8) = y[k];
              }
            }
            __syncwarp();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.tempty[buf]);
        if (++buf == X_BUFS) {
          buf = 0;
          tphase ^= 1;
        }
      }
      fence_proxy_async();   // the store reads what this warp wrote
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(&sh.ydone[st]);
    }
  }
  if (!ok) {
    if (lane == 0) atomicExch(p.l.status, TSDS_E_TIMEOUT);
    *(volatile int*)&sh.abort = 1;
  }
  __syncwarp();
  pdl_wait();
  if (warp == 2 && lane == 0) {
    bulk_wait_read<0>();
    if (!any) drain_tma_ring(sh.yfull, p.y_stages, y_issued);   // nothing waited for them
  }
  tc_fence_before();
  __syncthreads();
  if (sh.abort) {   // uniform: copies and MMAs in flight finish (bounded) before TMEM is freed
    if (warp == 0 && lane == 0) {
      drain_tma_ring(sh.full, p.b_stages, issued);
      if (slices > 0) mbar_wait(&sh.t_full, (slices - 1) & 1, 20000000ull);
    }
    if (warp == 2 && lane == 0) drain_tma_ring(sh.yfull, p.y_stages, y_issued);
    if (warp == 1 && lane == 0 && issued > 0) drain_mma<1>(&sh.drain);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_give(tmem, X_BUFS * p.tn);
  }
}

int launch_shrink(const CUtensorMap& a_all, const CUtensorMap& a_box, const CUtensorMap& xmap, const ShrinkArgs& p,
                  cudaStream_t stream) {
  static tsds_device_flags limit_set;
  const int st = tsds_smem_limit_once(shrink_kernel, SHRINK_SMEM, limit_set);
  if (st != TSDS_OK) return st;
  // more of the SM's shared memory than of TMEM's columns (110 KB for up to 128; expand:
  // 190 KB or more for 256, 89 KB or more for 128), so CTAs that fit an SM never wait for columns
  const int smem = SHRINK_SMEM;
  tsds_launch_cluster(shrink_kernel, dim3((unsigned)(p.blocks * p.l.slots * CL)), dim3(THREADS), smem, stream, CL,
                      a_all, a_box, xmap, p);
  return tsds_launch_status();
}

template <int PER_SM>
int launch_expand(const CUtensorMap& bmap, const CUtensorMap& tmap, const CUtensorMap& ymap, const OutMaps& omap,
                  const ExpandArgs& p, int blocks, int smem, cudaStream_t stream) {
  static tsds_device_flags limit_set;
  const int st = tsds_smem_limit_once(expand_kernel<PER_SM>, X_SMEM, limit_set);
  if (st != TSDS_OK) return st;
  tsds_launch(expand_kernel<PER_SM>, dim3((unsigned)(blocks * p.step)), dim3(X_THREADS), smem, stream, bmap, tmap, ymap,
              omap, p);
  return tsds_launch_status();
}

int rank_columns(int R) { return (R + BKE - 1) / BKE * BKE; }

}  // namespace

size_t tsds_lora_tc_workspace_bytes(int M, int R, int S) {
  return (size_t)M * 2 * S * rank_columns(R) * sizeof(bf16);
}

int tsds_lora_tc(const LoraArgs& l, void* workspace, cudaStream_t stream) {
  ShrinkArgs p = {};
  p.l = l;
  p.t = (bf16*)workspace;
  p.Rp = rank_columns(l.R);
  p.ld_t = l.S * p.Rp;
  // Token rows per shrink block: 32 for few rows (more clusters; 8 x 26 rows at
  // rank 64 into q/k/v 23.6 us, with 64 26.2), 64 above (an adapter's A is read
  // less often; 16 x 26 rows, K 25600, rank 16 26 us, with 32 37), 128 from 3584 rows on,
  // where even one adapter per block makes 28 clusters, 1.5 CTAs per SM (4096 rows at
  // rank 16 into q/k/v 47.7 us, with 64 52.7; 2048 rows, 16 clusters, at rank 32 32.3 and 30.4)
  p.nt = l.M <= 256 ? 32 : (l.M < 3584 ? 64 : 128);
  p.blocks = (l.M + p.nt - 1) / p.nt;
  const int SR = l.S * l.R;
  p.arows = SR < TILE_J ? SR : TILE_J;
  p.bx = l.R % 16 ? 8 : 16;
  p.KT = (l.K + BKE - 1) / BKE;
  p.stage_bytes = (p.arows + p.nt) * 128;
  // the MMA reads 128 rows from a stage's first, which may reach past its end
  const int slack = p.arows + p.nt < TILE_J ? (TILE_J - p.arows - p.nt) * 128 : 0;
  p.stages = (SHRINK_SMEM - 1024 - slack) / p.stage_bytes;
  if (p.stages > RING) p.stages = RING;
  p.tmem_cols = p.nt;
  p.idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.nt >> 3) << 17) | ((uint32_t)(TILE_J >> 4) << 24);
  p.wait_ns = tsds_get_wait_limit_ns();
  // A cluster per adapter of a block of rows as long as all are resident at
  // once; beyond that each takes several in turn.  One without an adapter
  // holds the next launch up: with twice as many the q/k/v adapters of 256 rows
  // that alternate between 8 adapters of rank 64 take 43.5 us instead of 40.9.
  const int sms = tsds_tc_num_sms();
  p.l.slots = 2 * sms / CL / p.blocks;
  p.l.slots = p.l.slots < 1 ? 1 : (p.l.slots > p.nt ? p.nt : p.l.slots);
  if (p.l.slots > l.n_adapters) p.l.slots = l.n_adapters;
  CUtensorMap a_all, a_box, xmap, bmap, tmap, ymap;
  const uint64_t a_rows = (uint64_t)l.n_adapters * SR;
  int st = tsds_make_tmap_2d_bf16(&a_all, l.a, l.K, a_rows, (uint64_t)l.K * 2, BKE, p.arows, 1);
  if (st == TSDS_OK) st = tsds_make_tmap_2d_bf16(&a_box, l.a, l.K, a_rows, (uint64_t)l.K * 2, BKE, p.bx, 1);
  if (st == TSDS_OK) st = tsds_make_tmap_2d_bf16(&xmap, l.x, l.K, l.M, (uint64_t)l.ldx * 2, BKE, p.nt, 1);
  ExpandArgs q = {};
  q.l = l;
  q.ld_t = p.ld_t;
  q.Rp = p.Rp;
  q.kb = p.Rp / BKE;
  q.wait_ns = p.wait_ns;
  // 128 channels per tile and one CTA per SM with deep rings; but 64 and two
  // CTAs per SM (where their t leaves room) with few tiles and several adapters in a
  // block: they follow one another in a tile (64 rows that alternate between 8 adapters
  // of rank 64 into q/k/v 23.3 us instead of 25.5; of one adapter it is 13.4 instead of 12.7).
  const int blocks = (l.M + XM - 1) / XM;
  auto shape = [&](int tn, int places) {
    q.tn = tn;
    for (int i = 0; i < l.S; ++i)
      q.first_tile[i + 1] = q.first_tile[i] + (l.first_col[i + 1] - l.first_col[i] + tn - 1) / tn;
    q.tiles = q.first_tile[l.S];
    int step = places / blocks;
    step = step < 1 ? 1 : (step > q.tiles ? q.tiles : step);
    const int per = (q.tiles + step - 1) / step;
    q.step = (q.tiles + per - 1) / per;   // the tiles evenly among the CTAs
    return per;
  };
  int budget = X_SMEM, per = shape(128, sms);
  bool two = false;
  if (per <= 2 && l.n_adapters > 2 * blocks) {
    two = q.kb == 1;
    per = shape(64, two ? 2 * sms : sms);
    if (two) budget = 112 * 1024;
  }
  const int b_stage = q.kb * q.tn * 128, y_stage = q.tn / 64 * BOX;
  budget -= 1024 + q.kb * 2 * BOX;
  q.y_stages = (budget - 2 * b_stage) / y_stage;
  q.y_stages = q.y_stages > 4 ? 4 : q.y_stages;
  if (q.y_stages > per) q.y_stages = per < 2 ? 2 : per;
  q.b_stages = (budget - q.y_stages * y_stage) / b_stage;
  if (q.b_stages > X_RING) q.b_stages = X_RING;
  const int smem = 1024 + q.kb * 2 * BOX + q.b_stages * b_stage + q.y_stages * y_stage;
  OutMaps omap;
  if (st == TSDS_OK)
    st = tsds_make_tmap_2d_bf16(&bmap, l.b, l.R, (uint64_t)l.n_adapters * l.N, (uint64_t)l.R * 2, BKE, q.tn, 1);
  if (st == TSDS_OK)
    st = tsds_make_tmap_2d_bf16(&tmap, workspace, 2 * (uint64_t)p.ld_t, l.M, 4 * (uint64_t)p.ld_t, BKE, XM, 1);
  if (st == TSDS_OK) st = tsds_make_tmap_2d_bf16(&ymap, l.y, l.N, l.M, (uint64_t)l.ldy * 2, 64, XM, 1);
  for (int i = 0; i < l.S && st == TSDS_OK; ++i)
    st = tsds_make_tmap_2d_bf16(&omap.of[i], l.out + l.first_col[i], l.first_col[i + 1] - l.first_col[i], l.M,
                                (uint64_t)l.ldo * 2, 64, XM, 1);
  if (st != TSDS_OK) return st;

  st = launch_shrink(a_all, a_box, xmap, p, stream);
  if (st != TSDS_OK) return st;

  return two ? launch_expand<2>(bmap, tmap, ymap, omap, q, blocks, smem, stream)
             : launch_expand<1>(bmap, tmap, ymap, omap, q, blocks, smem, stream);
}
