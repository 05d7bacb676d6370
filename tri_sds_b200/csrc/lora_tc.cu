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
// * expand: out = y + B t^T.  An item is 128 output channels x 64 token rows x
//   adapter; two CTAs per SM share a block's items and take theirs in one
//   sequence, with B and y of the next items on their way.  The products of
//   both words of t go into one TMEM accumulator, two of which alternate, and
//   each epilogue warp adds its 32 channels of 32 rows to y by itself.
//
// The bytes of x and y bound both (B and A come from L2 after their first
// use); the MMAs are a few percent of the tensor cores' rate.  2048 rows, K 5120,
// rank 32 into q/k/v of 10240 columns: 36 us, shrink about 13 of them (21 MB of x, the
// rest the chain from launch to reduction) and expand 21 (84 MB of y and out,
// 4 TB/s).  Asking for y from shrink already, into L2, made it 43.
// shrink lets its successor start only after its own dependency wait, so
// everything before shrink is complete when expand begins, and expand may
// read y, B and the indices before its wait; only t comes after it.
#include "common.cuh"
#include "linear.cuh"
#include "lora.cuh"
#include "tc_core.cuh"

#include <type_traits>

using namespace tsds;
using namespace tsds::tc;
using namespace tsds::lora;

namespace {

constexpr int CL = 8;               // CTAs per shrink cluster
constexpr int THREADS = 192;        // TMA warp, MMA warp, four epilogue warps
constexpr int BKE = 64;             // elements of K (or ranks) per block: a 128-byte swizzle row
constexpr int RING = 8;             // most stages
constexpr int A_SLACK = TILE_J * 128;   // the MMA reads 128 rows of A, a stage may hold fewer

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
  if (__popcll(sh.tile.leads) <= slot) {   // a cluster whose turn never comes
    if (warp == 1) tmem_give(tmem, p.tmem_cols);
    return;
  }
  float* part = reinterpret_cast<float*>(smem);   // [nt][128], in the ring once it is free
  const int k_lo = rank * p.KT / CL, nk = (rank + 1) * p.KT / CL - k_lo;
  int s = 0, issued = 0;                 // ring position, blocks so far (warps 0 and 1)
  uint32_t phase = warp == 0 ? 1 : 0, tphase = 0;
  bool alive = true;

  unsigned long long leads = sh.tile.leads;
  for (int gi = 0; leads; ++gi, leads &= leads - 1) {
    if (gi % p.l.slots != slot) continue;
    const Adapter ad = adapter_of(p.l, sh.tile, sh.tile.id[__ffsll((long long)leads) - 1]);
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
        float h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = rbf(v[k]);
        bf16* to = p.t + (int64_t)(row0 + i) * 2 * p.ld_t + sl * p.Rp + r;
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf2(h[0], h[1]), pack_bf2(h[2], h[3]));
        *reinterpret_cast<uint2*>(to + p.ld_t) =
            make_uint2(pack_bf2(v[0] - h[0], v[1] - h[1]), pack_bf2(v[2] - h[2], v[3] - h[3]));
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

constexpr int XN = 64;                      // token rows of an expand unit
constexpr int X_THREADS = 320;              // TMA warp, MMA warp, two groups of four epilogue warps
constexpr int B_TILE = TILE_J * 128;        // 128 channels x 64 ranks
constexpr int T_TILE = XN * 128;            // 64 token rows x 64 ranks
constexpr int X_LD = 36;                    // padded row of 32 staged channels: 16-byte reads of two rows in all banks
constexpr int X_STAGING = 8 * 16 * X_LD * (int)sizeof(float);

struct ExpandArgs {
  LoraArgs l;
  int ld_t, Rp, blocks, tiles, step, kb;    // step: CTAs that share a block's items; kb: blocks of 64 ranks
  int first_tile[MAX_SLICES + 1];           // channel tiles where the slices begin
  uint64_t wait_ns;
};

struct ExpandShared {
  Tile tile;
  Adapter group[XN];   // what this CTA adds or copies, in turn
  uint64_t t_full, full[2], empty[2], tfull[2], tempty[2], drain;
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
  c.lo = p.l.first_col[c.sl] + (tile - p.first_tile[c.sl]) * TILE_J;
  c.end = p.l.first_col[c.sl + 1];
  return c;
}

// An item of expand's work: one adapter of the block and a channel tile.  The CTA
// of index c takes items c, c + step, ... of all of them, adapter by adapter.
struct Item {
  int g, tile;
};
__device__ __forceinline__ Item next_item(const ExpandArgs& p, Item it) {
  for (it.tile += p.step; it.tile >= p.tiles; it.tile -= p.tiles) ++it.g;
  return it;
}

__global__ void __launch_bounds__(X_THREADS, 2)
    expand_kernel(const __grid_constant__ CUtensorMap bmap, const __grid_constant__ CUtensorMap tmap, ExpandArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ ExpandShared sh;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 1) tmem_take(&sh.tmem, 2 * XN);
  const int block = blockIdx.x / p.step, row0 = block * XN;
  const int index = blockIdx.x - block * p.step;
  const Item first = {index / p.tiles, index % p.tiles};
  if (warp == 0 && elect_one()) {
    prefetch_tmap(&bmap);
    prefetch_tmap(&tmap);
    mbar_init(&sh.t_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
      mbar_init(&sh.tfull[i], 1);
      mbar_init(&sh.tempty[i], 8);   // one arrival per epilogue warp
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  pdl_trigger();
  group_rows(p.l, sh.tile, row0, XN, false, p.l.out != p.l.y);
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const int groups = __popcll(sh.tile.leads);
  if (groups <= first.g) {   // nothing for this CTA
    if (warp == 1) tmem_give(tmem, 2 * XN);
    pdl_wait();
    return;
  }
  if (threadIdx.x < XN && (sh.tile.leads >> threadIdx.x & 1)) {
    const int i = __popcll(sh.tile.leads & ((1ull << threadIdx.x) - 1)), id = sh.tile.id[threadIdx.x];
    sh.group[i] = id >= 0 ? adapter_of(p.l, sh.tile, id) : Adapter{id, 0, 0.f};
  }
  __syncthreads();
  const int b_bytes = p.kb * B_TILE;
  uint8_t *b_smem = smem, *t_smem = smem + 2 * b_bytes;   // t: [slice][kb][hi, lo]
  float* stg = reinterpret_cast<float*>(t_smem + p.l.S * p.kb * 2 * T_TILE);
  int buf = 0, issued = 0;     // ring position = accumulator: one B tile per output tile
  uint32_t phase = 0;
  bool ok = true;

  // every warp goes through the same items, group by group and tile by tile,
  // without a barrier between groups
  if (warp == 0) {
    for (Item it = first; it.g < groups; it = next_item(p, it)) {
      const Adapter ad = sh.group[it.g];
      if (ad.ra == 0) continue;
      ok = warp_wait(&sh.empty[buf], phase ^ 1, p.wait_ns);
      if (!ok) break;
      if (elect_one()) {
        const int kb = (ad.ra + BKE - 1) / BKE;
        mbar_arrive_expect_tx(&sh.full[buf], kb * B_TILE);
        for (int i = 0; i < kb; ++i)
          tma_load_2d(b_smem + buf * b_bytes + i * B_TILE, &bmap, &sh.full[buf], i * BKE,
                      ad.id * p.l.N + channels_of(p, it.tile).lo);
      }
      __syncwarp();
      if (issued == 0) {   // every slice's t of these rows, once; the first read that waits for shrink
        pdl_wait();
        if (elect_one()) {
          mbar_arrive_expect_tx(&sh.t_full, p.l.S * p.kb * 2 * T_TILE);
          for (int i = 0; i < p.l.S * p.kb; ++i) {
            uint8_t* t = t_smem + i * 2 * T_TILE;
            tma_load_2d(t, &tmap, &sh.t_full, i * BKE, row0);
            tma_load_2d(t + T_TILE, &tmap, &sh.t_full, p.ld_t + i * BKE, row0);
          }
        }
        __syncwarp();
      }
      ++issued;
      phase ^= buf;
      buf ^= 1;
    }
  } else if (warp == 1) {
    for (Item it = first; it.g < groups; it = next_item(p, it)) {
      const Adapter ad = sh.group[it.g];
      const int steps = (ad.ra + 15) / 16;   // of 16 ranks
      if (steps == 0) continue;
      ok = warp_wait(&sh.tempty[buf], phase ^ 1, p.wait_ns) && warp_wait(&sh.full[buf], phase, p.wait_ns) &&
           warp_wait(&sh.t_full, 0, p.wait_ns);
      if (!ok) break;
      uint8_t* bs = b_smem + buf * b_bytes;
      if (ad.ra & 15) {
        // the last step's ranks past the adapter's: B's columns there are not
        // part of it, whatever they hold
        const int from = ad.ra & 63, to = ((ad.ra + 15) & ~15) - (ad.ra & ~63);
        uint8_t* b = bs + (ad.ra / 64) * B_TILE;
        for (int row = lane; row < TILE_J; row += 32)
          for (int c = from; c < to; ++c)
            *reinterpret_cast<uint16_t*>(b + row * 128 + (((c >> 3) ^ (row & 7)) << 4) + (c & 7) * 2) = 0;
        fence_proxy_async();
      }
      __syncwarp();
      if (elect_one()) {
        tc_fence_after();
        const uint32_t idesc =
            (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(XN >> 3) << 17) | ((uint32_t)(TILE_J >> 4) << 24);
        const uint64_t b0 = sdesc_sw128(smem_u32(bs));
        const uint64_t t0 = sdesc_sw128(smem_u32(t_smem + channels_of(p, it.tile).sl * p.kb * 2 * T_TILE));
        for (int i = 0; i < steps; ++i) {
          const uint64_t b = b0 + (uint32_t)((i >> 2) * B_TILE >> 4) + (i & 3) * 2;
          const uint64_t t = t0 + (uint32_t)((i >> 2) * 2 * T_TILE >> 4) + (i & 3) * 2;
          umma_bf16(tmem + buf * XN, b, t + (T_TILE >> 4), idesc, i != 0);   // lo
          umma_bf16(tmem + buf * XN, b, t, idesc, 1);                        // hi
        }
        umma_commit(&sh.empty[buf]);
        umma_commit(&sh.tfull[buf]);
      }
      __syncwarp();
      ++issued;
      phase ^= buf;
      buf ^= 1;
    }
  } else {
    // A warp takes 32 channels (its lanes of TMEM) of 32 token rows, a thread
    // eight channels of every eighth row, so a warp accesses rows in runs of 64
    // bytes.  It transposes 16 rows at a time through staging of its own: with
    // 128 threads on one staging area and a branch per row an item took twice as long.
    const int half = (warp - 2) >> 2, quarter = warp & 3;
    const int tr = half * 32 + (lane >> 2), j0 = quarter * 32 + (lane & 3) * 8;
    float* to = stg + (warp - 2) * 16 * X_LD + lane;
    const float* from = stg + (warp - 2) * 16 * X_LD + (lane >> 2) * X_LD + (lane & 3) * 8;
    using Yes = std::true_type;
    using No = std::false_type;
    const int row_id = sh.tile.id[half * 32 + lane];
    struct Part {   // an item's part of this warp
      int id, lo;
      bool whole, in;   // all 32 x 32 outputs, any of this thread's channels
    };
    auto part_of = [&](Item it) {
      const Channels c = channels_of(p, it.tile);
      Part w;
      w.id = sh.group[it.g].id;
      w.lo = c.lo;
      w.in = c.lo + j0 < c.end;
      w.whole = __all_sync(0xffffffffu, row_id == w.id && w.in);
      return w;
    };
    auto load_y = [&](Item it, uint4 (&y)[4]) {
      if (it.g >= groups) return;
      const Part w = part_of(it);
      const bf16* at = p.l.y + (int64_t)(row0 + tr) * p.l.ldy + w.lo + j0;
      if (w.whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = *reinterpret_cast<const uint4*>(at + i * 8 * p.l.ldy);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (w.in && sh.tile.id[tr + i * 8] == w.id) y[i] = *reinterpret_cast<const uint4*>(at + i * 8 * p.l.ldy);
      }
    };
    // an item further ahead: its lines into L2, one per thread of every other warp
    auto prefetch_y = [&](Item it) {
      if (it.g >= groups || (quarter & 1) || row_id != sh.group[it.g].id) return;
      const Channels c = channels_of(p, it.tile);
      if (c.lo + quarter * 32 < c.end)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.l.y + (int64_t)(row0 + half * 32 + lane) * p.l.ldy + c.lo +
                                                      quarter * 32));
    };
    auto finish = [&](Item it, const uint4 (&y)[4]) {
      const Part w = part_of(it);
      bf16* out = p.l.out + (int64_t)(row0 + tr) * p.l.ldo + w.lo + j0;
      if (sh.group[it.g].ra == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (w.in && sh.tile.id[tr + i * 8] == w.id) *reinterpret_cast<uint4*>(out + i * 8 * p.l.ldo) = y[i];
        return;
      }
      ok = warp_wait(&sh.tfull[buf], phase, p.wait_ns);
      if (!ok) return;
      tc_fence_after();
      uint32_t v[32];
      tmem_request32(tmem + buf * XN + ((uint32_t)(quarter * 32) << 16) + half * 32, v);
      tmem_wait32(v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.tempty[buf]);   // this warp has read its part of the accumulator
      auto rest = [&](auto whole) {
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
#pragma unroll
          for (int i = 0; i < 16; ++i) to[i * X_LD] = __uint_as_float(v[c + i]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = c / 8 + i;
            const float4 a = *reinterpret_cast<const float4*>(from + i * 8 * X_LD);
            const float4 b = *reinterpret_cast<const float4*>(from + i * 8 * X_LD + 4);
            const uint4 o = y[k];
            if (whole || (w.in && sh.tile.id[tr + k * 8] == w.id))
              *reinterpret_cast<uint4*>(out + k * 8 * p.l.ldo) = make_uint4(
                  pack_bf2(bf_lo(o.x) + a.x, bf_hi(o.x) + a.y), pack_bf2(bf_lo(o.y) + a.z, bf_hi(o.y) + a.w),
                  pack_bf2(bf_lo(o.z) + b.x, bf_hi(o.z) + b.y), pack_bf2(bf_lo(o.w) + b.z, bf_hi(o.w) + b.w));
          }
          __syncwarp();
        }
      };
      if (w.whole)
        rest(Yes());
      else
        rest(No());
      phase ^= buf;
      buf ^= 1;
    };
    // the next item's y is requested before this one's is used, in a register
    // set of its own: loads are awaited by set, so one set would be awaited
    // with the requests just made (5 us a tile instead of 1.2)
    uint4 y0[4], y1[4];
    Item now = first, next = next_item(p, now), ahead = next_item(p, next);
    load_y(now, y0);
    prefetch_y(next);
    prefetch_y(ahead);
    pdl_wait();   // a copied row may be what an earlier kernel still reads
    while (now.g < groups) {
      ahead = next_item(p, ahead);
      load_y(next, y1);
      prefetch_y(ahead);
      finish(now, y0);
      if (!ok || next.g >= groups) break;
      now = next_item(p, next);
      ahead = next_item(p, ahead);
      load_y(now, y0);
      prefetch_y(ahead);
      finish(next, y1);
      if (!ok) break;
      next = next_item(p, now);
    }
  }
  if (!ok) {
    if (lane == 0) atomicExch(p.l.status, TSDS_E_TIMEOUT);
    *(volatile int*)&sh.abort = 1;
  }
  __syncwarp();
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (sh.abort) {   // uniform: copies and MMAs in flight finish (bounded) before TMEM is freed
    if (warp == 0 && lane == 0) {
      drain_tma_ring(sh.full, 2, issued);
      if (issued > 0) mbar_wait(&sh.t_full, 0, 20000000ull);   // requested behind the first tile
    }
    if (warp == 1 && lane == 0 && issued > 0) drain_mma<1>(&sh.drain);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_give(tmem, 2 * XN);
  }
}

int launch_shrink(const CUtensorMap& a_all, const CUtensorMap& a_box, const CUtensorMap& xmap, const ShrinkArgs& p,
                  cudaStream_t stream) {
  static tsds_device_flags limit_set;
  const int st = tsds_smem_limit_once(shrink_kernel, 97 * 1024, limit_set);
  if (st != TSDS_OK) return st;
  // more of the SM's shared memory than of TMEM's columns (at least 57 KB for 64;
  // expand: 65 KB for 128), so CTAs that fit an SM never wait for columns
  const int smem = p.stages * p.stage_bytes + A_SLACK + 1024;
  tsds_launch_cluster(shrink_kernel, dim3((unsigned)(p.blocks * p.l.slots * CL)), dim3(THREADS), smem, stream, CL,
                      a_all, a_box, xmap, p);
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
  // rank 64 into q/k/v 23.7 us, with 64 26.6), 64 above (an adapter's A is read
  // less often; 16 x 26 rows, K 25600, rank 16 25.0 us, with 32 37.7)
  p.nt = l.M <= 256 ? 32 : 64;
  p.blocks = (l.M + p.nt - 1) / p.nt;
  const int SR = l.S * l.R;
  p.arows = SR < TILE_J ? SR : TILE_J;
  p.bx = l.R % 16 ? 8 : 16;
  p.KT = (l.K + BKE - 1) / BKE;
  p.stage_bytes = (p.arows + p.nt) * 128;
  p.stages = (96 * 1024 - A_SLACK) / p.stage_bytes;
  if (p.stages > RING) p.stages = RING;
  p.tmem_cols = p.nt;
  p.idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.nt >> 3) << 17) | ((uint32_t)(TILE_J >> 4) << 24);
  p.wait_ns = tsds_get_wait_limit_ns();
  // A cluster per adapter of a block of rows as long as all are resident at
  // once; beyond that each takes several in turn.  One without an adapter
  // holds the next launch up: with twice as many the q/k/v adapters of 256 rows
  // that alternate between 8 adapters of rank 64 take 47 us instead of 44.
  const int sms = tsds_tc_num_sms();
  p.l.slots = 2 * sms / CL / p.blocks;
  p.l.slots = p.l.slots < 1 ? 1 : (p.l.slots > p.nt ? p.nt : p.l.slots);
  if (p.l.slots > l.n_adapters) p.l.slots = l.n_adapters;
  CUtensorMap a_all, a_box, xmap, bmap, tmap;
  const uint64_t a_rows = (uint64_t)l.n_adapters * SR;
  int st = tsds_make_tmap_2d_bf16(&a_all, l.a, l.K, a_rows, (uint64_t)l.K * 2, BKE, p.arows, 1);
  if (st == TSDS_OK) st = tsds_make_tmap_2d_bf16(&a_box, l.a, l.K, a_rows, (uint64_t)l.K * 2, BKE, p.bx, 1);
  if (st == TSDS_OK) st = tsds_make_tmap_2d_bf16(&xmap, l.x, l.K, l.M, (uint64_t)l.ldx * 2, BKE, p.nt, 1);
  if (st == TSDS_OK)
    st = tsds_make_tmap_2d_bf16(&bmap, l.b, l.R, (uint64_t)l.n_adapters * l.N, (uint64_t)l.R * 2, BKE, TILE_J, 1);
  if (st == TSDS_OK)
    st = tsds_make_tmap_2d_bf16(&tmap, workspace, 2 * (uint64_t)p.ld_t, l.M, 4 * (uint64_t)p.ld_t, BKE, XN, 1);
  if (st != TSDS_OK) return st;

  st = launch_shrink(a_all, a_box, xmap, p, stream);
  if (st != TSDS_OK) return st;

  ExpandArgs q = {};
  q.l = l;
  q.ld_t = p.ld_t;
  q.Rp = p.Rp;
  q.blocks = (l.M + XN - 1) / XN;
  q.kb = p.Rp / BKE;
  for (int i = 0; i < l.S; ++i)
    q.first_tile[i + 1] = q.first_tile[i] + (l.first_col[i + 1] - l.first_col[i] + TILE_J - 1) / TILE_J;
  q.tiles = q.first_tile[l.S];
  q.wait_ns = p.wait_ns;
  const int smem = 2 * q.kb * B_TILE + l.S * q.kb * 2 * T_TILE + X_STAGING + 1024;
  // a block's items over as many CTAs as are resident at once
  const int places = sms * (smem <= 112 * 1024 ? 2 : 1), most = q.tiles * (l.n_adapters < XN ? l.n_adapters + 1 : XN);
  q.step = places / q.blocks;
  q.step = q.step < 1 ? 1 : (q.step > most ? most : q.step);
  static tsds_device_flags expand_set;
  st = tsds_smem_limit_once(expand_kernel, 220 * 1024, expand_set);
  if (st != TSDS_OK) return st;
  tsds_launch(expand_kernel, dim3((unsigned)(q.blocks * q.step)), dim3(X_THREADS), smem, stream, bmap, tmap,
              q);
  return tsds_launch_status();
}
