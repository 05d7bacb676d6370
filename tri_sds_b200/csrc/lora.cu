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
// Two kernels for the first product.  Few rows (tiles of 16 or 32): the
// adapter's bytes are the cost; every warp takes its own part of K straight
// into registers, all loads in flight at once.  Many rows (tiles of 64): x is
// the cost, and warps share operands; x and A go through a cp.async ring.
#include "common.cuh"
#include "tc_core.cuh"

using namespace tsds;

namespace {

constexpr int MAX_SLICES = 4;
constexpr int MAX_RANK = 128;
constexpr int MAX_TILE = 64;   // rows per tile, at most
constexpr int NEAR = 64;       // adapters whose rank and scale every CTA reads

struct LoraArgs {
  const bf16 *x, *y, *a, *b;
  bf16* out;
  const int32_t *adapter, *ranks;
  const float* scale;
  int32_t* status;
  int64_t ldx, ldy, ldo;
  int M, K, N, R, S, n_adapters, slots, ld_t;
  int first_col[MAX_SLICES + 1];   // columns where the slices begin
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// 16 bytes to shared memory, or zeros where `in` is false
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

__device__ __forceinline__ float4 ld_peer4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ void st_peer8(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}

__device__ __forceinline__ uint4 ld16(const bf16* p) { return *reinterpret_cast<const uint4*>(p); }

// `bytes` (a multiple of 16) from a 16-byte aligned address into L2
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  tc::cluster_sync_all();
}

struct Tile {
  int32_t id[MAX_TILE];      // adapter of each row; -1: none; -2: past the last row
  unsigned long long leads;  // rows that are the first of their adapter
  // rank and scale of the first adapters, read beside the rows' indices rather than after them
  int32_t rank[NEAR];
  float scale[NEAR];
};

// The adapter at hand.
struct Adapter {
  int id, ra, nr8, nch, Rp;   // index, rank, n8 tiles and chunks of 16 of a slice's ranks, columns of t per slice
  float scale;
};

// The tile's rows by adapter.
template <int TR>
__device__ __forceinline__ void group_rows(const LoraArgs& p, Tile& sh, int row0, int rank) {
  const int tid = threadIdx.x;
  if (tid == 0) sh.leads = 0;
  if (tid >= 64 && tid < 64 + NEAR) {
    const int a = tid - 64;
    sh.rank[a] = p.ranks && a < p.n_adapters ? p.ranks[a] : p.R;
    sh.scale[a] = p.scale && a < p.n_adapters ? p.scale[a] : 1.0f;
  }
  if (tid < TR) {
    const int m = row0 + tid;
    int id = m < p.M ? p.adapter[m] : -2;
    if (m < p.M && id < 0) id = -1;
    if (id >= p.n_adapters) {   // never followed: the row keeps its projection
      id = -1;
      if (rank == 0) atomicExch(p.status, TSDS_E_INDEX);
    }
    sh.id[tid] = id;
  }
  __syncthreads();
  if (tid < TR) {
    const int id = sh.id[tid];
    bool first = true;
#pragma unroll
    for (int j = 0; j < TR; ++j) first = first && !(j < tid && sh.id[j] == id);
    // rows without an adapter are a group of their own (copied) unless in place
    if (first && (id >= 0 || (id == -1 && p.out != p.y))) atomicOr(&sh.leads, 1ull << tid);
  }
  __syncthreads();
}

// Rows without an adapter: this CTA's columns copied from y.
template <int TR, int CL>
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
template <int CL>
__device__ __forceinline__ void column_groups(const LoraArgs& p, int rank, int& lo, int& hi) {
  const int groups = (p.N + 31) / 32;
  lo = rank * groups / CL;
  hi = (rank + 1) * groups / CL;
}

// The CTA's part of B, and of y in the adapter's rows, into L2.
template <int TR, int CL>
__device__ __forceinline__ void prefetch_second(const LoraArgs& p, const Tile& sh, const Adapter& ad, int row0,
                                                int rank) {
  int lo, hi;
  column_groups<CL>(p, rank, lo, hi);
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

// t's columns for rank tiles t0 .. t0 + nt - 1: the cluster's partial sums
// (part: [TR][ldr] in every CTA) of this CTA's share of the rows, scaled, as
// two bf16 words into every CTA's t_hi / t_lo.
template <int TR, int CL>
__device__ __forceinline__ void exchange(const LoraArgs& p, const Adapter& ad, float* part, int ldr, bf16* t_hi,
                                         bf16* t_lo, int t0, int nt, int rank) {
  cluster_barrier();   // every CTA's part is complete
  constexpr int SHARE = TR / CL;
  const int n4 = nt * 2;
  for (int e = threadIdx.x; e < SHARE * n4; e += blockDim.x) {
    const int m = rank * SHARE + e / n4, c4 = e % n4;
    const uint32_t at = smem_u32(part + m * ldr + c4 * 4);
    float4 f[CL];
#pragma unroll
    for (int k = 0; k < CL; ++k) f[k] = ld_peer4(tc::mapa_shared(at, k));
    float4 s = f[0];
#pragma unroll
    for (int k = 1; k < CL; ++k) s = make_float4(s.x + f[k].x, s.y + f[k].y, s.z + f[k].z, s.w + f[k].w);
    const int ti = t0 + c4 / 2, sl = ti / ad.nr8;
    const int to = m * p.ld_t + sl * ad.Rp + (ti - sl * ad.nr8) * 8 + (c4 & 1) * 4;
    const float v[4] = {s.x * ad.scale, s.y * ad.scale, s.z * ad.scale, s.w * ad.scale};
    float h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = rbf(v[k]);
    const uint32_t h0 = pack_bf2(h[0], h[1]), h1 = pack_bf2(h[2], h[3]);
    const uint32_t l0 = pack_bf2(v[0] - h[0], v[1] - h[1]), l1 = pack_bf2(v[2] - h[2], v[3] - h[3]);
    const uint32_t ah = smem_u32(t_hi + to), al = smem_u32(t_lo + to);
#pragma unroll
    for (int k = 0; k < CL; ++k) {
      st_peer8(tc::mapa_shared(ah, k), h0, h1);
      st_peer8(tc::mapa_shared(al, k), l0, l1);
    }
  }
  cluster_barrier();   // t is complete everywhere, part may be overwritten
}

// out = y + t B^T over this CTA's columns, in the adapter's rows among row
// tiles m0 .. m0 + MT - 1.  A warp takes
// 32 columns at a time; the four n8 tiles interleave their columns so that a
// thread ends up with eight adjacent ones (n0 + 8q ..): column c of tile i is
// n0 + 8 (c / 2) + 2 i + c % 2.
template <int MT, int CH, int CL>   // CH: chunks of 16 ranks loaded together
__device__ __forceinline__ void expand(const LoraArgs& p, const Tile& sh, const Adapter& ad, const bf16* t_hi,
                                       const bf16* t_lo, int row0, int rank, unsigned mtiles, int m0) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const bf16* b_id = p.b + (int64_t)ad.id * p.N * p.R + 4 * q;
  bool mine[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) mine[m][h] = sh.id[(m0 + m) * 16 + g + 8 * h] == ad.id;
  int lo, hi;
  column_groups<CL>(p, rank, lo, hi);
  for (int gr = lo + (int)(threadIdx.x >> 5); gr < hi; gr += blockDim.x >> 5) {
    const int n0 = gr * 32, n = n0 + 8 * q;
    int sl = 0;
#pragma unroll
    for (int s = 1; s < MAX_SLICES; ++s)
      if (s < p.S && n0 >= p.first_col[s]) sl = s;
    uint4 yv[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (n < p.N && mine[m][h]) yv[m][h] = ld16(p.y + (int64_t)(row0 + (m0 + m) * 16 + g + 8 * h) * p.ldy + n);
    float acc[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i][0] = acc[m][i][1] = acc[m][i][2] = acc[m][i][3] = 0.f;
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
            bv[c][i] = __ldg(reinterpret_cast<const uint2*>(b_col + 2 * i * p.R + (c0 + c) * 16));
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
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (!(mtiles >> (m0 + m) & 1)) continue;
          const int at = ((m0 + m) * 16 + g) * p.ld_t + sl * ad.Rp + r;
          const uint2 h0 = *reinterpret_cast<const uint2*>(t_hi + at);
          const uint2 h8 = *reinterpret_cast<const uint2*>(t_hi + at + 8 * p.ld_t);
          const uint2 l0 = *reinterpret_cast<const uint2*>(t_lo + at);
          const uint2 l8 = *reinterpret_cast<const uint2*>(t_lo + at + 8 * p.ld_t);
          const uint32_t fh[4] = {h0.x, h8.x, h0.y, h8.y}, fl[4] = {l0.x, l8.x, l0.y, l8.y};
#pragma unroll
          for (int i = 0; i < 4; ++i) mma16816(acc[m][i], fl, bv[c][i].x, bv[c][i].y);
#pragma unroll
          for (int i = 0; i < 4; ++i) mma16816(acc[m][i], fh, bv[c][i].x, bv[c][i].y);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (n < p.N && mine[m][h]) {
          const uint32_t u[4] = {yv[m][h].x, yv[m][h].y, yv[m][h].z, yv[m][h].w};
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o[k] = pack_bf2(bf_lo(u[k]) + acc[m][k][2 * h], bf_hi(u[k]) + acc[m][k][2 * h + 1]);
          *reinterpret_cast<uint4*>(p.out + (int64_t)(row0 + (m0 + m) * 16 + g + 8 * h) * p.ldo + n) =
              make_uint4(o[0], o[1], o[2], o[3]);
        }
    __syncwarp();
  }
}

// Few rows.  MT: m16 tiles of the tile's rows, NT: n8 rank tiles per pass
// over K, U: chunks of 32 k loaded together.
template <int MT, int NT, int U, int WARPS>
struct FewRows {
  static constexpr int THREADS = WARPS * 32;
  static constexpr int TR = 16 * MT, LDR = NT * 8 + 4;   // padded row of partial sums
  static constexpr int PASS = NT;
  static constexpr int PART = WARPS * TR * LDR * (int)sizeof(float);   // the CTA's sum, behind those of its warps
  static constexpr int WORK = PART + TR * LDR * (int)sizeof(float);
  static constexpr int CTAS = 1;

  template <int CL>
  static __device__ __forceinline__ void first(const LoraArgs& p, const Adapter& ad, uint8_t* work, float* part,
                                               int row0, int rank, unsigned, int t0, int nt) {
    float* red = reinterpret_cast<float*>(work);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const bf16* a_id = p.a + (int64_t)ad.id * p.S * p.R * p.K + 8 * q;
    const bf16* x_row = p.x + (int64_t)(row0 + g) * p.ldx + 8 * q;
    int ar[NT];   // rank row of each tile, -1: none
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int s = (t0 + i) / ad.nr8, r = (t0 + i - s * ad.nr8) * 8 + g;
      ar[i] = i < nt && r < ad.ra ? s * p.R + r : -1;
    }
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[m][i][0] = acc[m][i][1] = acc[m][i][2] = acc[m][i][3] = 0.f;
    // k is summed in the order the 16-byte loads give it: lane q of a row
    // holds k = 8q .. 8q+7 of a chunk, elements 0-3 in the first step and 4-7
    // in the second, the same for both operands
    const int chunks = (p.K + 31) / 32;
    for (int c0 = rank * WARPS + warp; c0 < chunks; c0 += CL * WARPS * U) {
      uint4 xv[U][MT][2], av[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (c0 + u * CL * WARPS) * 32;
        const bool in = k + 8 * q < p.K;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          av[u][i] = in && ar[i] >= 0 ? ldg16(a_id + (int64_t)ar[i] * p.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            xv[u][m][h] = in && row0 + m * 16 + g + 8 * h < p.M ? ld16(x_row + (m * 16 + 8 * h) * p.ldx + k)
                                                                 : make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 xa = xv[u][m][0], xb = xv[u][m][1];
          const uint32_t f0[4] = {xa.x, xb.x, xa.y, xb.y}, f1[4] = {xa.z, xb.z, xa.w, xb.w};
#pragma unroll
          for (int i = 0; i < NT; ++i)
            if (i < nt) mma16816(acc[m][i], f0, av[u][i].x, av[u][i].y);
#pragma unroll
          for (int i = 0; i < NT; ++i)
            if (i < nt) mma16816(acc[m][i], f1, av[u][i].z, av[u][i].w);
        }
    }
    // the CTA's sum, warps in order
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float* mine = red + (warp * TR + m * 16) * LDR;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (i < nt) {
          *reinterpret_cast<float2*>(mine + g * LDR + i * 8 + 2 * q) = make_float2(acc[m][i][0], acc[m][i][1]);
          *reinterpret_cast<float2*>(mine + (g + 8) * LDR + i * 8 + 2 * q) = make_float2(acc[m][i][2], acc[m][i][3]);
        }
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

// Many rows.  x and A in blocks of 64 k (rows of 128 bytes, 16-byte pieces
// XORed with the row so that ldmatrix meets no bank conflict) through a ring
// of STAGES; a warp takes one row tile and its share of the rank tiles.
template <int TILE_ROWS, int RING>
struct ManyRows {
  static constexpr int THREADS = 256;
  static constexpr int TR = TILE_ROWS, MT = TR / 16, NT = 12, LDR = NT * 8 + 4;
  static constexpr int NW = 8 / MT, NP = NT / NW;   // warps that share a row tile, rank tiles of each
  static constexpr int PASS = NT;
  static constexpr int STAGES = RING, ROWS = TR + NT * 8, STAGE = ROWS * 128;
  static constexpr int PART = 0;   // the CTA's sum: in the ring, free by then
  static constexpr int WORK = STAGES * STAGE;
  static constexpr int CTAS = 2;

  template <int CL>
  static __device__ __forceinline__ void first(const LoraArgs& p, const Adapter& ad, uint8_t* work, float* part,
                                               int row0, int rank, unsigned mtiles, int t0, int nt) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const uint32_t base = smem_u32(work);
    const int blocks = (p.K + 63) / 64, b0 = rank * blocks / CL, b1 = (rank + 1) * blocks / CL;
    // a thread's rows: tid / 8 + 32 i (x rows first, then rank rows), piece tid % 8 of each
    constexpr int PER = ROWS * 8 / THREADS;
    const int piece = tid % 8, rows = TR + nt * 8;
    const bf16* src[PER];
    uint32_t dst[PER];
    bool in[PER];
    const bf16* a_id = p.a + (int64_t)ad.id * p.S * p.R * p.K;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int row = tid / 8 + i * (THREADS / 8);
      dst[i] = base + row * 128 + ((piece ^ (row & 7)) << 4);
      if (row < TR) {
        in[i] = row0 + row < p.M;
        src[i] = p.x + (int64_t)(in[i] ? row0 + row : 0) * p.ldx;
      } else {
        const int u = row - TR, ti = t0 + u / 8, s = ti / ad.nr8, r = (ti - s * ad.nr8) * 8 + u % 8;
        in[i] = row < rows && r < ad.ra;
        src[i] = a_id + (int64_t)(in[i] ? s * p.R + r : 0) * p.K;
      }
    }
    auto load = [&](int b, int s) {
      const int k = b * 64 + piece * 8;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (tid / 8 + i * (THREADS / 8) < rows)
          cp16(dst[i] + s * STAGE, src[i] + (k < p.K ? k : 0), in[i] && k < p.K);
    };
    float acc[NP][4];
#pragma unroll
    for (int i = 0; i < NP; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const int mt = warp % MT, n_lo = warp / MT * nt / NW, n_hi = (warp / MT + 1) * nt / NW;
    for (int i = 0; i < STAGES - 1; ++i) {
      if (b0 + i < b1) load(b0 + i, i);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int b = b0, i = 0; b < b1; ++b, ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncthreads();   // block b has landed for all; the stage of block b - 1 is free
      if (b + STAGES - 1 < b1) load(b + STAGES - 1, (i + STAGES - 1) % STAGES);
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (!(mtiles >> mt & 1)) continue;
      const uint32_t st = base + i % STAGES * STAGE;
      // ldmatrix rows: x: lane % 16 of the row tile, k half lane / 16; A: two n8
      // tiles, row lane % 8 of tile lane / 16, k half (lane / 8) % 2
      const int xrow = mt * 16 + lane % 16;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t f[4];
        ldmatrix4(f, st + xrow * 128 + (((kk * 2 + lane / 16) ^ (xrow & 7)) << 4));
#pragma unroll
        for (int i2 = 0; i2 < (NP + 1) / 2; ++i2) {
          const int n = n_lo + i2 * 2;
          if (n < n_hi) {
            const int arow = TR + (n + lane / 16) * 8 + lane % 8;
            uint32_t w[4];
            // of an odd last tile's partner nothing is used: read the tile itself twice
            const int safe = n + 1 < n_hi ? arow : TR + n * 8 + lane % 8;
            ldmatrix4(w, st + safe * 128 + (((kk * 2 + lane / 8 % 2) ^ (safe & 7)) << 4));
            mma16816(acc[i2 * 2], f, w[0], w[1]);
            if (i2 * 2 + 1 < NP && n + 1 < n_hi) mma16816(acc[i2 * 2 + 1 < NP ? i2 * 2 + 1 : 0], f, w[2], w[3]);
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();   // every warp is done with the ring
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (n_lo + i < n_hi) {
        float* at = part + (mt * 16 + g) * LDR + (n_lo + i) * 8 + 2 * q;
        *reinterpret_cast<float2*>(at) = make_float2(acc[i][0], acc[i][1]);
        *reinterpret_cast<float2*>(at + 8 * LDR) = make_float2(acc[i][2], acc[i][3]);
      }
  }
};

template <typename First, int CL>
__global__ void __launch_bounds__(First::THREADS, First::CTAS) lora_kernel(LoraArgs p) {
  constexpr int TR = First::TR, MT = TR / 16, LDR = First::LDR, ET = MT < 2 ? MT : 2;
  __shared__ Tile sh;
  extern __shared__ __align__(128) uint8_t dyn[];
  float* part = reinterpret_cast<float*>(dyn + First::PART);   // [TR][LDR] this CTA's sum, read by the cluster
  bf16* t_hi = reinterpret_cast<bf16*>(dyn + First::WORK);
  bf16* t_lo = t_hi + TR * p.ld_t;
  const int rank = (int)tc::cluster_ctarank();
  // every tile's first adapter before any tile's second: clusters without one come last
  const int tiles = (p.M + TR - 1) / TR, unit = blockIdx.x / CL, slot = unit / tiles, tile = unit - slot * tiles;
  const int row0 = tile * TR;
  pdl_trigger();
  pdl_wait();
  group_rows<TR>(p, sh, row0, rank);
  unsigned long long leads = sh.leads;
  for (int gi = 0; leads; ++gi, leads &= leads - 1) {
    if (gi % p.slots != slot) continue;
    Adapter ad;
    ad.id = sh.id[__ffsll((long long)leads) - 1];
    if (ad.id < 0) {
      copy_rows<TR, CL>(p, sh, row0, rank);
      continue;
    }
    if (ad.id < NEAR) {
      ad.ra = sh.rank[ad.id];
      ad.scale = sh.scale[ad.id];
    } else {
      ad.ra = p.ranks ? p.ranks[ad.id] : p.R;
      ad.scale = p.scale ? p.scale[ad.id] : 1.0f;
    }
    ad.ra = ad.ra < 0 ? 0 : (ad.ra > p.R ? p.R : ad.ra);
    ad.nr8 = (ad.ra + 7) / 8;
    ad.nch = (ad.ra + 15) / 16;
    ad.Rp = (p.R + 15) / 16 * 16;
    unsigned mtiles = 0;   // row tiles that hold a row of this adapter
#pragma unroll
    for (int i = 0; i < TR; ++i)
      if (sh.id[i] == ad.id) mtiles |= 1u << (i / 16);
    prefetch_second<TR, CL>(p, sh, ad, row0, rank);
    const int tiles8 = p.S * ad.nr8;
    for (int t0 = 0; t0 < tiles8; t0 += First::PASS) {
      const int nt = tiles8 - t0 < First::PASS ? tiles8 - t0 : First::PASS;
      First::template first<CL>(p, ad, dyn, part, row0, rank, mtiles, t0, nt);
      exchange<TR, CL>(p, ad, part, LDR, t_hi, t_lo, t0, nt, rank);
    }
    // an odd number of rank tiles: the last chunk of 16 ends in zeros
    if (ad.nr8 & 1) {
      for (int e = threadIdx.x; e < TR * p.S * 8; e += blockDim.x) {
        const int at = e / (p.S * 8) * p.ld_t + e / 8 % p.S * ad.Rp + ad.nr8 * 8 + e % 8;
        t_hi[at] = t_lo[at] = f2bf(0.f);
      }
      __syncthreads();
    }
    for (int m0 = 0; m0 < MT; m0 += ET) {   // two row tiles at a time keep the sums in registers
      if (!(mtiles >> m0 & ((1u << ET) - 1))) continue;
      if (ad.nch <= 1)
        expand<ET, 1, CL>(p, sh, ad, t_hi, t_lo, row0, rank, mtiles, m0);
      else
        expand<ET, 2, CL>(p, sh, ad, t_hi, t_lo, row0, rank, mtiles, m0);
    }
    __syncthreads();   // t is read; a peer writes the next adapter's after the next cluster barrier
  }
}

template <typename First, int CL>
int launch_lora(LoraArgs p, cudaStream_t stream) {
  constexpr int TR = First::TR;
  static tsds_device_flags limit_set;
  const int smem = First::WORK + 2 * TR * p.ld_t * (int)sizeof(bf16);
  constexpr int most = First::WORK + 2 * TR * (MAX_SLICES * MAX_RANK + 16) * (int)sizeof(bf16);
  static_assert(most <= 226 * 1024, "shared memory of a CTA");
  const int st = tsds_smem_limit_once(lora_kernel<First, CL>, most, limit_set);
  if (st != TSDS_OK) return st;
  const int tiles = (p.M + TR - 1) / TR;
  // a cluster per adapter of a tile while the grid stays within ~1000 CTAs
  // (clusters without one leave at once); beyond that a cluster takes several
  int slots = 128 / tiles;
  slots = slots < 1 ? 1 : (slots > TR + 1 ? TR + 1 : slots);
  if (slots > p.n_adapters + 1) slots = p.n_adapters + 1;
  p.slots = slots;
  tsds_launch_cluster(lora_kernel<First, CL>, dim3((unsigned)(tiles * slots * CL)), dim3(First::THREADS), smem, stream, CL, p);
  return tsds_launch_status();
}

}  // namespace

extern "C" int tsds_lora_add(const void* y, int ldy, const void* x, int ldx, const void* lora_a, const void* lora_b,
                             const int32_t* adapter, const float* scale, const int32_t* ranks, void* out, int ldo,
                             int M, int K, int N, int n_adapters, int R, int n_slices, const int32_t* slice_widths,
                             int32_t* status, tsds_stream_t stream) {
  TSDS_RETURN_IF(M < 0 || K <= 0 || (K % 8) != 0 || N <= 0 || (N % 8) != 0 || n_adapters <= 0 || R <= 0 ||
                     (R % 8) != 0 || ldx < K || ldy < N || ldo < N,
                 TSDS_E_INVALID);
  TSDS_RETURN_IF(n_slices < 1 || (n_slices > 1 && !slice_widths), TSDS_E_INVALID);
  TSDS_RETURN_IF(R > MAX_RANK || n_slices > MAX_SLICES || M > (1 << 26), TSDS_E_UNSUPPORTED);
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
  }
  if (M == 0) return TSDS_OK;
  TSDS_RETURN_IF(!y || !x || !lora_a || !lora_b || !adapter || !out || !status, TSDS_E_INVALID);
  TSDS_RETURN_IF(!tsds_aligned16(y) || !tsds_aligned16(x) || !tsds_aligned16(lora_a) || !tsds_aligned16(lora_b) ||
                     !tsds_aligned16(out) || (ldx % 8) || (ldy % 8) || (ldo % 8),
                 TSDS_E_ALIGN);
  TSDS_RETURN_IF(out == y && ldo != ldy, TSDS_E_INVALID);
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
  if (M > 512) return launch_lora<ManyRows<64, 3>, 8>(p, stream);
  if (M > 256) return launch_lora<ManyRows<32, 4>, 8>(p, stream);
  if (M > 16) return launch_lora<FewRows<2, 8, 2, 8>, 8>(p, stream);
  if (n_slices * R <= 16) return launch_lora<FewRows<1, 2, 4, 16>, 8>(p, stream);
  return launch_lora<FewRows<1, 8, 2, 12>, 8>(p, stream);
}
