// Low-rank adapters of many requests beside a shared projection (sm_100a):
//
//   out[m][j] = bf16( y[m][j] + scale[a] * sum_{r < rank[a]} B[a][j][r] * t[m][s(j)*R + r] ),
//   t[m][u]   = sum_k A[a][u][k] x[m][k],          a = adapter[m]
//
// y is the projection's output and s(j) the slice (q, k, v) of column j.  The
// work is the adapters' bytes (few rows) or x and y (many rows): the two
// products are small, and the tensor cores are fed from registers
// (mma.sync, fp32 accumulators) at a small part of their rate.
//
// One launch.  A cluster of 8 CTAs takes a tile of consecutive token rows and
// one adapter of those that occur in it: each CTA computes t over 1/8 of K,
// 1/8 of t's rows is summed by each CTA from all partials (over distributed
// shared memory, in rank order, so the result is always the same bits) and
// handed to all, and each CTA then adds t B^T to 1/8 of the columns.  t is
// computed for every row of the tile; only the adapter's own rows are written,
// the others belong to another cluster (or a later pass of this one).  Rows
// without an adapter are left alone, or copied when out is not y.
// What a CTA needs for the second product (its part of B and y) is
// prefetched into L2 before the first.
// t stays in fp32 until the second product, which reads it as the sum of two
// bf16 words (16 bits of it instead of 8), so t's rounding is far below
// that of the output.
//
// This file's kernel is for few rows, where the adapters' bytes are the cost and
// the chain of latencies the time: every warp takes its own part of K straight
// into registers, all loads in flight at once.  Many rows: lora_tc.cu.
#include "common.cuh"
#include "linear.cuh"
#include "lora.cuh"
#include "tc_core.cuh"

using namespace tsds;
using namespace tsds::lora;

namespace {

constexpr int CL = 8;         // CTAs per cluster
constexpr int TR = 16;        // rows per tile: one m16 tile
constexpr int RANKS = 64;     // columns of t, at most: 8 n8 tiles

// Whether one launch of this file's kernel runs, or the two of lora_tc.cu.  A
// cluster here reads all ranks of every slice for 16 rows, so the columns of t,
// the rows' bytes and the (tile, adapter) pairs decide; how many pairs occur is known
// only up to tiles x min(adapters, 16).  Measured, here and there (K 5120 into
// q/k/v of 10240, or K 8192 -> 5120): 8 rows of 8 adapters, rank 16 in three slices
// 10.8 and 14.9 us, rank 64 in one 13.1 and 15.2; 32 rows, rank 64 in one 13.0 and
// 13.4; 8 x 26 rows, rank 16 in three 14.8 and 15.9, rank 32 in one 14.0 and 14.2; 512
// rows of one adapter, rank 16 in three 15.2 and 15.5, rank 16 in one 13.1 and 13.7, rank
// 32 in one 16.7 and 14.1, 1024 rows 24.2 and 18.4; 128 rows that alternate between 16
// adapters, rank 16 in one 44 and 29.  K 25600 -> 5120: 8 rows, rank 16 10.3 and 21.3;
// 208 rows, rank 48 28.8 and 21.3; 512 rows, rank 64 42.8 and 21.3.  (Taken with read-only loads of A
// and B; with the plain ones the first case takes 10.1 us here, 8 x 26 rows 14.2 and 13.8.)
bool few_rows(int M, int K, int R, int S, int n_adapters) {
  const int tiles = (M + TR - 1) / TR, SR = S * R;
  if (M > 512 || tiles * (n_adapters < TR ? n_adapters : TR) > 104) return false;
  return SR <= 16 || (SR <= 48 && (int64_t)tiles * K <= 200000) || (SR <= RANKS && M <= TR);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void st_peer8(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}

// (a plain load for A and B too: an adapter's may have been written by the kernel before,
// whose end this one waits for after its own start)
__device__ __forceinline__ uint4 ld16(const bf16* p) { return *reinterpret_cast<const uint4*>(p); }

// `bytes` (a multiple of 16) from a 16-byte aligned address into L2
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// The adapter at hand, and its layout: n8 tiles and chunks of 16 of a slice's
// ranks, columns of t per slice.
struct Ranks : Adapter {
  int nr8, nch, Rp;
};

// Rows without an adapter: this CTA's columns copied from y.
__device__ __forceinline__ void copy_rows(const LoraArgs& p, const Tile& sh, int row0, int rank) {
  const int nv = p.N / 8;
  for (int i = 0; i < TR; ++i) {
    if (sh.id[i] != -1) continue;
    const int64_t m = row0 + i;
    for (int c = rank * (int)blockDim.x + (int)threadIdx.x; c < nv; c += CL * (int)blockDim.x)
      *reinterpret_cast<uint4*>(p.out + m * p.ldo + c * 8) = ld16(p.y + m * p.ldy + c * 8);
  }
}

// This CTA's groups of 32 columns: [lo, hi).
__device__ __forceinline__ void column_groups(const LoraArgs& p, int rank, int& lo, int& hi) {
  const int groups = (p.N + 31) / 32;
  lo = rank * groups / CL;
  hi = (rank + 1) * groups / CL;
}

// The CTA's part of B, and of y in the adapter's rows, into L2.
__device__ __forceinline__ void prefetch_second(const LoraArgs& p, const Tile& sh, const Ranks& ad, int row0,
                                                int rank) {
  int lo, hi;
  column_groups(p, rank, lo, hi);
  const int c0 = lo * 32, c1 = hi * 32 < p.N ? hi * 32 : p.N, tid = threadIdx.x;
  if (c1 <= c0) return;
  if (tid < TR) {
    if (sh.id[tid] == ad.id) prefetch_l2(p.y + (int64_t)(row0 + tid) * p.ldy + c0, (uint32_t)(c1 - c0) * 2);
  } else if (ad.ra * 2 > p.R) {   // most of every row of B: 4 KB at a time
    const char* b = reinterpret_cast<const char*>(p.b + ((int64_t)ad.id * p.N + c0) * p.R);
    const int64_t bytes = (int64_t)(c1 - c0) * p.R * 2;
    for (int64_t o = (int64_t)(tid - TR) * 4096; o < bytes; o += ((int64_t)blockDim.x - TR) * 4096)
      prefetch_l2(b + o, (uint32_t)(bytes - o < 4096 ? bytes - o : 4096));
  }
}

// t's columns (nt rank tiles): the cluster's partial sums (part: [TR][ldr] in
// every CTA) of this CTA's share of the rows, scaled, as two bf16 words into
// every CTA's t_hi / t_lo.
__device__ __forceinline__ void exchange(const LoraArgs& p, const Ranks& ad, float* part, int ldr, bf16* t_hi,
                                         bf16* t_lo, int nt, int rank) {
  tc::cluster_barrier();   // every CTA's part is complete
  constexpr int SHARE = TR / CL;
  const int n4 = nt * 2;
  for (int e = threadIdx.x; e < SHARE * n4; e += blockDim.x) {
    const int m = rank * SHARE + e / n4, c4 = e % n4;
    const uint32_t at = smem_u32(part + m * ldr + c4 * 4);
    float4 f[CL];
#pragma unroll
    for (int k = 0; k < CL; ++k) f[k] = tc::ld_peer(tc::mapa_shared(at, k));
    float4 s = f[0];
#pragma unroll
    for (int k = 1; k < CL; ++k) s = make_float4(s.x + f[k].x, s.y + f[k].y, s.z + f[k].z, s.w + f[k].w);
    const int ti = c4 / 2, sl = ti / ad.nr8;
    const int to = m * p.ld_t + sl * ad.Rp + (ti - sl * ad.nr8) * 8 + (c4 & 1) * 4;
    // ranks past the adapter's are zeros: an infinite x or scale would make NaN of them
    const int left = ad.ra - (ti - sl * ad.nr8) * 8 - (c4 & 1) * 4;
    const float v[4] = {s.x, s.y, s.z, s.w};
    float h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) two_words(k < left ? v[k] * ad.scale : 0.f, h[k], l[k]);
    const uint32_t h0 = pack_bf2(h[0], h[1]), h1 = pack_bf2(h[2], h[3]);
    const uint32_t l0 = pack_bf2(l[0], l[1]), l1 = pack_bf2(l[2], l[3]);
    const uint32_t ah = smem_u32(t_hi + to), al = smem_u32(t_lo + to);
#pragma unroll
    for (int k = 0; k < CL; ++k) {
      st_peer8(tc::mapa_shared(ah, k), h0, h1);
      st_peer8(tc::mapa_shared(al, k), l0, l1);
    }
  }
  tc::cluster_barrier();   // t is complete everywhere, part may be overwritten
}

// out = y + t B^T over this CTA's columns, in the adapter's rows.  A warp takes
// 32 columns at a time; the four n8 tiles interleave their columns so that a
// thread ends up with eight adjacent ones (n0 + 8q ..): column c of tile i is
// n0 + 8 (c / 2) + 2 i + c % 2.
template <int CH>   // chunks of 16 ranks loaded together
__device__ __forceinline__ void expand(const LoraArgs& p, const Tile& sh, const Ranks& ad, const bf16* t_hi,
                                       const bf16* t_lo, int row0, int rank) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const bf16* b_id = p.b + (int64_t)ad.id * p.N * p.R + 4 * q;
  bool mine[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) mine[h] = sh.id[g + 8 * h] == ad.id;
  int lo, hi;
  column_groups(p, rank, lo, hi);
  for (int gr = lo + (int)(threadIdx.x >> 5); gr < hi; gr += blockDim.x >> 5) {
    const int n0 = gr * 32, n = n0 + 8 * q;
    int sl = 0;
#pragma unroll
    for (int s = 1; s < MAX_SLICES; ++s)
      if (s < p.S && n0 >= p.first_col[s]) sl = s;
    uint4 yv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n < p.N && mine[h]) yv[h] = ld16(p.y + (int64_t)(row0 + g + 8 * h) * p.ldy + n);
    float acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const int col = n0 + 8 * (g >> 1);   // this lane's rows of B: col + (g & 1) + 2 i
    const bf16* b_col = b_id + (int64_t)(col + (g & 1)) * p.R;
    for (int c0 = 0; c0 < ad.nch; c0 += CH) {
      uint2 bv[CH][4];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int left = ad.ra - (c0 + c) * 16 - 4 * q;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bv[c][i] = make_uint2(0, 0);
          if (col < p.N && left > 0)
            bv[c][i] = *reinterpret_cast<const uint2*>(b_col + 2 * i * p.R + (c0 + c) * 16);
        }
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (c0 + c >= ad.nch) break;
        const int r = (c0 + c) * 16 + 4 * q, left = ad.ra - r;
        if (left < 4) {   // ranks past the adapter's are not part of it, whatever they hold
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (left < 1) bv[c][i].x = 0;
            else if (left < 2) bv[c][i].x &= 0xffffu;
            if (left < 3) bv[c][i].y = 0;
            else bv[c][i].y &= 0xffffu;
          }
        }
        __syncwarp();
        const int at = g * p.ld_t + sl * ad.Rp + r;
        const uint2 h0 = *reinterpret_cast<const uint2*>(t_hi + at);
        const uint2 h8 = *reinterpret_cast<const uint2*>(t_hi + at + 8 * p.ld_t);
        const uint2 l0 = *reinterpret_cast<const uint2*>(t_lo + at);
        const uint2 l8 = *reinterpret_cast<const uint2*>(t_lo + at + 8 * p.ld_t);
        const uint32_t fh[4] = {h0.x, h8.x, h0.y, h8.y}, fl[4] = {l0.x, l8.x, l0.y, l8.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) mma16816(acc[i], fl, bv[c][i].x, bv[c][i].y);
#pragma unroll
        for (int i = 0; i < 4; ++i) mma16816(acc[i], fh, bv[c][i].x, bv[c][i].y);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n < p.N && mine[h]) {
        const uint32_t u[4] = {yv[h].x, yv[h].y, yv[h].z, yv[h].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = pack_bf2(bf_lo(u[k]) + acc[k][2 * h], bf_hi(u[k]) + acc[k][2 * h + 1]);
        *reinterpret_cast<uint4*>(p.out + (int64_t)(row0 + g + 8 * h) * p.ldo + n) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    __syncwarp();
  }
}

// The first product.  NT: most n8 rank tiles, U: chunks of 32 k loaded
// together, PER_SM: CTAs per SM.
template <int NT, int U, int WARPS, int PER_SM>
struct First {
  static constexpr int CTAS = PER_SM, THREADS = WARPS * 32, LDR = NT * 8 + 4;   // LDR: padded row of partial sums
  static constexpr int PART = WARPS * TR * LDR * (int)sizeof(float);   // the CTA's sum, behind those of its warps
  static constexpr int WORK = PART + TR * LDR * (int)sizeof(float);

  static __device__ __forceinline__ void run(const LoraArgs& p, const Ranks& ad, uint8_t* work, float* part, int row0,
                                             int rank, int nt) {
    float* red = reinterpret_cast<float*>(work);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const bf16* a_id = p.a + (int64_t)ad.id * p.S * p.R * p.K + 8 * q;
    const bf16* x_row = p.x + (int64_t)(row0 + g) * p.ldx + 8 * q;
    int ar[NT];   // rank row of each tile, -1: none
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int s = i / ad.nr8, r = (i - s * ad.nr8) * 8 + g;
      ar[i] = i < nt && r < ad.ra ? s * p.R + r : -1;
    }
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    // k is summed in the order the 16-byte loads give it: lane q of a row
    // holds k = 8q .. 8q+7 of a chunk, elements 0-3 in the first step and 4-7
    // in the second, the same for both operands
    const int chunks = (p.K + 31) / 32, lo = rank * chunks / CL, hi = (rank + 1) * chunks / CL;
    if (hi - lo > WARPS * U && hi * 32 <= p.K) {
      // several rounds of loads: this CTA's part of every row goes to L2 at once, so
      // that only the first round waits for DRAM
      const uint32_t bytes = (uint32_t)(hi - lo) * 64;
      for (int i = tid; i < nt * 8 + TR; i += THREADS) {
        const int u = i / 8, s = u / ad.nr8, r = (u - s * ad.nr8) * 8 + i % 8, m = row0 + i - nt * 8;
        if (i < nt * 8 && r < ad.ra)
          prefetch_l2(p.a + ((int64_t)ad.id * p.S * p.R + s * p.R + r) * p.K + lo * 32, bytes);
        else if (i >= nt * 8 && m < p.M)
          prefetch_l2(p.x + (int64_t)m * p.ldx + lo * 32, bytes);
      }
      __syncwarp();
    }
    for (int c0 = lo + warp; c0 < hi; c0 += WARPS * U) {
      uint4 xv[U][2], av[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * WARPS, k = c * 32;
        const bool in = c < hi && k + 8 * q < p.K;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          av[u][i] = in && ar[i] >= 0 ? ld16(a_id + (int64_t)ar[i] * p.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          xv[u][h] = in && row0 + g + 8 * h < p.M ? ld16(x_row + 8 * h * p.ldx + k) : make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint4 xa = xv[u][0], xb = xv[u][1];
        const uint32_t f0[4] = {xa.x, xb.x, xa.y, xb.y}, f1[4] = {xa.z, xb.z, xa.w, xb.w};
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < nt) mma16816(acc[i], f0, av[u][i].x, av[u][i].y);
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < nt) mma16816(acc[i], f1, av[u][i].z, av[u][i].w);
      }
    }
    // the CTA's sum, warps in order
    float* mine = red + warp * TR * LDR;
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (i < nt) {
        *reinterpret_cast<float2*>(mine + g * LDR + i * 8 + 2 * q) = make_float2(acc[i][0], acc[i][1]);
        *reinterpret_cast<float2*>(mine + (g + 8) * LDR + i * 8 + 2 * q) = make_float2(acc[i][2], acc[i][3]);
      }
    __syncthreads();
    const int n4 = nt * 2;
    for (int e = tid; e < TR * n4; e += THREADS) {
      const int at = e / n4 * LDR + e % n4 * 4;
      float4 s = *reinterpret_cast<const float4*>(red + at);
#pragma unroll
      for (int k = 1; k < WARPS; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(red + k * TR * LDR + at);
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
      }
      *reinterpret_cast<float4*>(part + at) = s;
    }
  }
};

template <typename F>
__global__ void __launch_bounds__(F::THREADS, F::CTAS) lora_kernel(LoraArgs p) {
  __shared__ Tile sh;
  extern __shared__ __align__(128) uint8_t dyn[];
  float* part = reinterpret_cast<float*>(dyn + F::PART);   // [TR][LDR] this CTA's sum, read by the cluster
  bf16* t_hi = reinterpret_cast<bf16*>(dyn + F::WORK);
  bf16* t_lo = t_hi + TR * p.ld_t;
  const int rank = (int)tc::cluster_ctarank();
  // every tile's first adapter before any tile's second: clusters without one come last
  const int tiles = (p.M + TR - 1) / TR, unit = blockIdx.x / CL, slot = unit / tiles, row0 = (unit - slot * tiles) * TR;
  pdl_trigger();
  pdl_wait();
  group_rows(p, sh, row0, TR, rank == 0, p.out != p.y);
  uint32_t leads = sh.leads[0];   // TR rows
  for (int gi = 0; leads; ++gi, leads &= leads - 1) {
    if (gi % p.slots != slot) continue;
    const int id = sh.id[__ffs(leads) - 1];
    if (id < 0) {
      copy_rows(p, sh, row0, rank);
      continue;
    }
    Ranks ad;
    static_cast<Adapter&>(ad) = adapter_of(p, sh, id);
    ad.nr8 = (ad.ra + 7) / 8;
    ad.nch = (ad.ra + 15) / 16;
    ad.Rp = (p.R + 15) / 16 * 16;
    prefetch_second(p, sh, ad, row0, rank);
    const int nt = p.S * ad.nr8;
    if (nt > 0) {
      F::run(p, ad, dyn, part, row0, rank, nt);
      exchange(p, ad, part, F::LDR, t_hi, t_lo, nt, rank);
    }
    // an odd number of rank tiles: the last chunk of 16 ends in zeros
    if (ad.nr8 & 1) {
      for (int e = threadIdx.x; e < TR * p.S * 8; e += F::THREADS) {
        const int at = e / (p.S * 8) * p.ld_t + e / 8 % p.S * ad.Rp + ad.nr8 * 8 + e % 8;
        t_hi[at] = t_lo[at] = f2bf(0.f);
      }
      __syncthreads();
    }
    if (ad.nch <= 1)
      expand<1>(p, sh, ad, t_hi, t_lo, row0, rank);
    else
      expand<2>(p, sh, ad, t_hi, t_lo, row0, rank);
    __syncthreads();   // t is read; a peer writes the next adapter's after the next cluster barrier
  }
}

// shared memory of the largest call
template <typename F>
constexpr int most_smem() {
  return F::WORK + 2 * TR * (RANKS + 16) * (int)sizeof(bf16);
}

// Clusters of the larger CTAs, one CTA per SM, that are resident at once.
using Large = First<8, 2, 12, 1>;
int resident_large() {
  static tsds_cluster_counts known;
  const int dev = tsds_device();
  return dev < 0 ? 0 : tsds_resident_clusters(dev, lora_kernel<Large>, Large::THREADS, most_smem<Large>(), CL, known);
}

template <typename F>
int launch_lora(LoraArgs p, cudaStream_t stream) {
  static tsds_device_flags limit_set;
  const int smem = F::WORK + 2 * TR * p.ld_t * (int)sizeof(bf16);
  constexpr int most = most_smem<F>();
  static_assert(most <= 226 * 1024, "shared memory of a CTA");
  const int st = tsds_smem_limit_once(lora_kernel<F>, most, limit_set);
  if (st != TSDS_OK) return st;
  const int tiles = (p.M + TR - 1) / TR;
  // a cluster per adapter of a tile while the grid stays within ~500 CTAs
  // (clusters without one leave at once); beyond that a cluster takes several
  int slots = 60 / tiles;
  slots = slots < 1 ? 1 : (slots > TR + 1 ? TR + 1 : slots);
  if (slots > p.n_adapters + 1) slots = p.n_adapters + 1;
  p.slots = slots;
  tsds_launch_cluster(lora_kernel<F>, dim3((unsigned)(tiles * slots * CL)), dim3(F::THREADS), smem, stream, CL, p);
  return tsds_launch_status();
}

}  // namespace

extern "C" size_t tsds_lora_workspace_bytes(int M, int R, int n_slices) {
  // whatever K and the number of adapters are
  if (M <= 0 || R <= 0 || n_slices <= 0 || (M <= TR && n_slices * R <= RANKS)) return 0;
  return tsds_lora_tc_workspace_bytes(M, R, n_slices);
}

extern "C" int tsds_lora_add(const void* y, int ldy, const void* x, int ldx, const void* lora_a, const void* lora_b,
                             const int32_t* adapter, const float* scale, const int32_t* ranks, void* out, int ldo,
                             int M, int K, int N, int n_adapters, int R, int n_slices, const int32_t* slice_widths,
                             void* workspace, size_t workspace_bytes, int32_t* status, tsds_stream_t stream) {
  TSDS_RETURN_IF(M < 0 || K <= 0 || (K % 8) != 0 || N <= 0 || (N % 8) != 0 || n_adapters <= 0 || R <= 0 ||
                     (R % 8) != 0 || ldx < K || ldy < N || ldo < N,
                 TSDS_E_INVALID);
  TSDS_RETURN_IF(n_slices < 1 || (n_slices > 1 && !slice_widths), TSDS_E_INVALID);
  TSDS_RETURN_IF(R > MAX_RANK || n_slices > MAX_SLICES || M > (1 << 26) || K > (1 << 30) || N > (1 << 30),
                 TSDS_E_UNSUPPORTED);
  LoraArgs p = {};
  p.S = n_slices;
  if (n_slices > 1) {
    int64_t at = 0;
    for (int s = 0; s < n_slices; ++s) {
      // a group of 32 columns lies in one slice
      TSDS_RETURN_IF(slice_widths[s] <= 0 || (slice_widths[s] % 32) != 0, TSDS_E_INVALID);
      p.first_col[s] = (int)at;
      at += slice_widths[s];
      TSDS_RETURN_IF(at > N, TSDS_E_INVALID);
    }
    TSDS_RETURN_IF(at != N, TSDS_E_INVALID);
  } else {
    TSDS_RETURN_IF(slice_widths && slice_widths[0] != N, TSDS_E_INVALID);
  }
  p.first_col[n_slices] = N;
  if (M == 0) return TSDS_OK;
  TSDS_RETURN_IF(!y || !x || !lora_a || !lora_b || !adapter || !out || !status, TSDS_E_INVALID);
  TSDS_RETURN_IF(!tsds_aligned16(y) || !tsds_aligned16(x) || !tsds_aligned16(lora_a) || !tsds_aligned16(lora_b) ||
                     !tsds_aligned16(out) || (ldx % 8) || (ldy % 8) || (ldo % 8),
                 TSDS_E_ALIGN);
  TSDS_RETURN_IF((out == y && ldo != ldy) || out == x, TSDS_E_INVALID);
  p.x = (const bf16*)x;
  p.y = (const bf16*)y;
  p.a = (const bf16*)lora_a;
  p.b = (const bf16*)lora_b;
  p.out = (bf16*)out;
  p.adapter = adapter;
  p.ranks = ranks;
  p.scale = scale;
  p.status = status;
  p.ldx = ldx;
  p.ldy = ldy;
  p.ldo = ldo;
  p.M = M;
  p.K = K;
  p.N = N;
  p.R = R;
  p.n_adapters = n_adapters;
  // rows of t: 16 elements past a multiple of 64, so that the fragments'
  // 8-byte reads of four rows cover all banks
  p.ld_t = (n_slices * ((R + 15) / 16 * 16) + 63) / 64 * 64 + 16;
  const bool few = few_rows(M, K, R, n_slices, n_adapters);
  if (!few) {
    // rows of A and B are tensor-map coordinates there
    TSDS_RETURN_IF((int64_t)n_adapters * (N > n_slices * R ? N : n_slices * R) > 0x7fffffff, TSDS_E_UNSUPPORTED);
    TSDS_RETURN_IF(!workspace || workspace_bytes < tsds_lora_tc_workspace_bytes(M, R, n_slices), TSDS_E_WORKSPACE);
    TSDS_RETURN_IF(!tsds_aligned16(workspace), TSDS_E_ALIGN);
  }
  // what is read while out is written: everything but y, and y too unless each element is out's own
  const int64_t r = (int64_t)n_adapters * R * 2;
  const tsds_rows o = {out, M, ldo * (int64_t)2, N * (int64_t)2};
  TSDS_RETURN_IF(tsds_overlap(o, {x, M, ldx * (int64_t)2, K * (int64_t)2}) ||
                     (out != y && tsds_overlap(o, {y, M, ldy * (int64_t)2, N * (int64_t)2})) ||
                     tsds_overlap(o, {lora_a, 1, 0, r * n_slices * K}) || tsds_overlap(o, {lora_b, 1, 0, r * N}),
                 TSDS_E_INVALID);
  if (!few) return tsds_lora_tc(p, workspace, stream);
  // Where a cluster for every adapter of every tile fits the SMs at once the call
  // is a matter of latency: many warps and loads per CTA (q/k/v adapters of 8
  // one-token requests 10.8 us, 14.2 with the smaller CTAs).  With more of them two
  // smaller CTAs per SM overlap (8 x 26 rows 14.8 us, 21.7 with the larger ones).
  const int most = (M + TR - 1) / TR * (n_adapters < TR ? n_adapters : TR);
  if (most > resident_large()) return launch_lora<First<8, 1, 8, 2>>(p, stream);
  if (n_slices * R <= 16) return launch_lora<First<2, 4, 16, 1>>(p, stream);
  return launch_lora<Large>(p, stream);
}
