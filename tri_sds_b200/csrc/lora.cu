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
// the partial sums are exchanged through distributed shared memory (rank
// order, so the result is always the same bits), and each CTA then adds
// t B^T to 1/8 of the columns.  Rows of a tile with another adapter belong to
// another cluster (or a later pass of this one); rows without an adapter are
// left alone, or copied when out is not y.
// t stays in fp32 until the second product, which reads it as the sum of two
// bf16 words (16 bits of it instead of 8), so t's rounding is far below
// that of the output.
#include "common.cuh"
#include "tc_core.cuh"

using namespace tsds;

namespace {

constexpr int CL = 8;          // CTAs per cluster
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int MAX_SLICES = 4;
constexpr int MAX_RANK = 128;
constexpr int MAX_TILE = 64;   // rows per tile, at most

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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float4 ld_peer4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint4 ld16(const bf16* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  tc::cluster_sync_all();
}

struct Tile {
  int32_t id[MAX_TILE];      // adapter of each row; -1: none; -2: past the last row
  int32_t first[MAX_TILE];   // first row of the tile with the same adapter
  int32_t pos[MAX_TILE];     // rows before it with the same adapter
  int32_t row[MAX_TILE];     // the rows of the adapter at hand
  unsigned long long leads;  // rows that are the first of their adapter
  int count;
};

// MW: m16 row tiles per tile of rows, each on WARPS / MW warps that share K.
// NT: n8 rank tiles per pass over K.  U: chunks of 32 k loaded together.
template <int MW, int NT, int U>
__global__ void __launch_bounds__(THREADS, MW == 1 ? 2 : 1) lora_kernel(LoraArgs p) {
  constexpr int TR = 16 * MW, KW = WARPS / MW;
  constexpr int LDR = NT * 8 + 4;   // padded row of partial sums
  __shared__ Tile sh;
  extern __shared__ __align__(16) uint8_t dyn[];
  float* red = reinterpret_cast<float*>(dyn);          // [KW][TR][LDR] partial sums of the warps
  float* part = red + KW * TR * LDR;                   // [TR][LDR] this CTA's sum, read by the cluster
  bf16* t_hi = reinterpret_cast<bf16*>(part + TR * LDR);
  bf16* t_lo = t_hi + TR * p.ld_t;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;
  const int rank = (int)tc::cluster_ctarank();
  const int unit = blockIdx.x / CL, tile = unit / p.slots, slot = unit - tile * p.slots;
  const int row0 = tile * TR;
  pdl_trigger();
  pdl_wait();

  // the tile's rows by adapter
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
  if (tid == 0) sh.leads = 0;
  __syncthreads();
  if (tid < TR) {
    const int id = sh.id[tid];
    int n = 0, f = tid;
#pragma unroll 16
    for (int j = TR - 1; j >= 0; --j)
      if (j < tid && sh.id[j] == id) {
        ++n;
        f = j;
      }
    sh.first[tid] = f;
    sh.pos[tid] = n;
    // rows without an adapter are a group of their own (copied) unless in place
    if (f == tid && (id >= 0 || (id == -1 && p.out != p.y))) atomicOr(&sh.leads, 1ull << tid);
  }
  __syncthreads();
  unsigned long long leads = sh.leads;
  bool first_group = true;
  for (int gi = 0; leads; ++gi, leads &= leads - 1) {
    if (gi % p.slots != slot) continue;
    const int lead = __ffsll((long long)leads) - 1;
    const int id = sh.id[lead];
    if (!first_group) __syncthreads();   // the last group's rows and t are read
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (tid < TR && sh.first[tid] == lead && sh.id[tid] == id) {
      sh.row[sh.pos[tid]] = row0 + tid;
      atomicMax(&sh.count, sh.pos[tid] + 1);
    }
    __syncthreads();
    const int cnt = sh.count;
    if (id < 0) {
      // copy: this CTA's 16-byte columns of each row
      const int nv = p.N / 8;
      for (int i = 0; i < cnt; ++i) {
        const int64_t m = sh.row[i];
        for (int c = rank * THREADS + tid; c < nv; c += CL * THREADS)
          *reinterpret_cast<uint4*>(p.out + m * p.ldo + c * 8) = ld16(p.y + m * p.ldy + c * 8);
      }
      first_group = false;
      continue;
    }
    int ra = p.ranks ? p.ranks[id] : p.R;
    ra = ra < 0 ? 0 : (ra > p.R ? p.R : ra);
    const float scale = p.scale ? p.scale[id] : 1.0f;
    const int nr8 = (ra + 7) / 8, nch = (ra + 15) / 16, Rp = (p.R + 15) / 16 * 16;
    const int mtiles = (cnt + 15) / 16;
    // odd number of rank tiles: the second product's last chunk of 16 ends in zeros
    if (nr8 & 1)
      for (int e = tid; e < TR * p.S * 8; e += THREADS) {
        const int at = (e / (p.S * 8)) * p.ld_t + (e / 8 % p.S) * Rp + nr8 * 8 + e % 8;
        t_hi[at] = t_lo[at] = f2bf(0.f);
      }

    // ---- t = x A^T, NT rank tiles per pass over this CTA's part of K ----
    const int mt = warp % MW, kp = warp / MW;
    const bf16* a_id = p.a + (int64_t)id * p.S * p.R * p.K;
    const bf16 *xg = nullptr, *xg8 = nullptr;
    if (mt * 16 + g < cnt) xg = p.x + (int64_t)sh.row[mt * 16 + g] * p.ldx;
    if (mt * 16 + g + 8 < cnt) xg8 = p.x + (int64_t)sh.row[mt * 16 + g + 8] * p.ldx;
    const int tiles8 = p.S * nr8, chunks = (p.K + 31) / 32;
    for (int t0 = 0; t0 < tiles8; t0 += NT) {
      const int nt = tiles8 - t0 < NT ? tiles8 - t0 : NT;
      float acc[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      if (mt < mtiles) {
        const bf16* ar[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int s = (t0 + i) / nr8, r = (t0 + i - s * nr8) * 8 + g;
          ar[i] = i < nt && r < ra ? a_id + (int64_t)(s * p.R + r) * p.K : nullptr;
        }
        // k is summed in the order the 16-byte loads give it: lane q of a row
        // holds k = 8q .. 8q+7 of a chunk, elements 0-3 in the first step
        // and 4-7 in the second, the same for both operands
        for (int c0 = rank * KW + kp; c0 < chunks; c0 += CL * KW * U) {
          uint4 xa[U], xb[U], av[U][NT];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int k = (c0 + u * CL * KW) * 32 + 8 * q;
            const bool in = k < p.K;
            xa[u] = in && xg ? ld16(xg + k) : make_uint4(0, 0, 0, 0);
            xb[u] = in && xg8 ? ld16(xg8 + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < NT; ++i) av[u][i] = in && ar[i] ? ldg16(ar[i] + k) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint32_t f0[4] = {xa[u].x, xb[u].x, xa[u].y, xb[u].y};
            const uint32_t f1[4] = {xa[u].z, xb[u].z, xa[u].w, xb[u].w};
#pragma unroll
            for (int i = 0; i < NT; ++i)
              if (i < nt) {
                mma16816(acc[i], f0, av[u][i].x, av[u][i].y);
                mma16816(acc[i], f1, av[u][i].z, av[u][i].w);
              }
          }
        }
      }
      // partial sums: warps of this CTA, then the cluster
      float* mine = red + (kp * TR + mt * 16) * LDR;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (i < nt && mt < mtiles) {
          *reinterpret_cast<float2*>(mine + g * LDR + i * 8 + 2 * q) = make_float2(acc[i][0], acc[i][1]);
          *reinterpret_cast<float2*>(mine + (g + 8) * LDR + i * 8 + 2 * q) = make_float2(acc[i][2], acc[i][3]);
        }
      __syncthreads();
      const int n4 = nt * 2, total = mtiles * 16 * n4;
      for (int e = tid; e < total; e += THREADS) {
        const int at = (e / n4) * LDR + e % n4 * 4;
        float4 s = *reinterpret_cast<const float4*>(red + at);
#pragma unroll
        for (int k = 1; k < KW; ++k) {
          const float4 v = *reinterpret_cast<const float4*>(red + k * TR * LDR + at);
          s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
        }
        *reinterpret_cast<float4*>(part + at) = s;
      }
      cluster_barrier();
      for (int e = tid; e < total; e += THREADS) {
        const int m = e / n4, c4 = e - m * n4;
        const uint32_t at = smem_u32(part + m * LDR + c4 * 4);
        float4 f[CL];
#pragma unroll
        for (int k = 0; k < CL; ++k) f[k] = ld_peer4(tc::mapa_shared(at, k));
        float4 s = f[0];
#pragma unroll
        for (int k = 1; k < CL; ++k) s = make_float4(s.x + f[k].x, s.y + f[k].y, s.z + f[k].z, s.w + f[k].w);
        const int ti = t0 + c4 / 2, sl = ti / nr8;
        const int to = m * p.ld_t + sl * Rp + (ti - sl * nr8) * 8 + (c4 & 1) * 4;
        const float v[4] = {s.x * scale, s.y * scale, s.z * scale, s.w * scale};
        float h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = rbf(v[k]);
        *reinterpret_cast<uint2*>(t_hi + to) = make_uint2(pack_bf2(h[0], h[1]), pack_bf2(h[2], h[3]));
        *reinterpret_cast<uint2*>(t_lo + to) =
            make_uint2(pack_bf2(v[0] - h[0], v[1] - h[1]), pack_bf2(v[2] - h[2], v[3] - h[3]));
      }
      cluster_barrier();   // part may be overwritten (or the CTA leave), t is complete
    }
    if (tiles8 == 0) __syncthreads();

    // ---- out = y + t B^T over this CTA's groups of 32 columns ----
    const bf16* b_id = p.b + (int64_t)id * p.N * p.R;
    const int groups = (p.N + 31) / 32;
    for (int gr = rank * WARPS + warp; gr < groups; gr += CL * WARPS) {
      const int n0 = gr * 32;
      int sl = 0;
#pragma unroll
      for (int s = 1; s < MAX_SLICES; ++s)
        if (s < p.S && n0 >= p.first_col[s]) sl = s;
      float acc[MW][4][4];
#pragma unroll
      for (int m = 0; m < MW; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i][0] = acc[m][i][1] = acc[m][i][2] = acc[m][i][3] = 0.f;
      // the four n8 tiles interleave their columns so that a thread ends up
      // with eight adjacent ones (n0 + 8q ..): column c of tile i is
      // n0 + 8 (c / 2) + 2 i + c % 2
      for (int ch = 0; ch < nch; ++ch) {
        const int r = ch * 16 + 4 * q, left = ra - r;
        uint2 bv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = n0 + 8 * (g >> 1) + 2 * i + (g & 1);
          bv[i] = make_uint2(0, 0);
          if (n < p.N && left > 0) bv[i] = __ldg(reinterpret_cast<const uint2*>(b_id + (int64_t)n * p.R + r));
          if (left < 4) {   // ranks past the adapter's are not part of it, whatever they hold
            if (left < 1) bv[i].x = 0;
            else if (left < 2) bv[i].x &= 0xffffu;
            if (left < 3) bv[i].y = 0;
            else bv[i].y &= 0xffffu;
          }
        }
#pragma unroll
        for (int m = 0; m < MW; ++m) {
          if (m >= mtiles) break;
          const int at = (m * 16 + g) * p.ld_t + sl * Rp + r;
          const uint2 h0 = *reinterpret_cast<const uint2*>(t_hi + at);
          const uint2 h8 = *reinterpret_cast<const uint2*>(t_hi + at + 8 * p.ld_t);
          const uint2 l0 = *reinterpret_cast<const uint2*>(t_lo + at);
          const uint2 l8 = *reinterpret_cast<const uint2*>(t_lo + at + 8 * p.ld_t);
          const uint32_t fh[4] = {h0.x, h8.x, h0.y, h8.y}, fl[4] = {l0.x, l8.x, l0.y, l8.y};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mma16816(acc[m][i], fl, bv[i].x, bv[i].y);
            mma16816(acc[m][i], fh, bv[i].x, bv[i].y);
          }
        }
      }
      const int n = n0 + 8 * q;
      if (n < p.N) {
#pragma unroll
        for (int m = 0; m < MW; ++m) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int i = m * 16 + g + 8 * h;
            if (i < cnt) {
              const int64_t row = sh.row[i];
              const uint4 yv = ld16(p.y + row * p.ldy + n);
              const uint32_t u[4] = {yv.x, yv.y, yv.z, yv.w};
              uint32_t o[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                o[k] = pack_bf2(bf_lo(u[k]) + acc[m][k][2 * h], bf_hi(u[k]) + acc[m][k][2 * h + 1]);
              *reinterpret_cast<uint4*>(p.out + row * p.ldo + n) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
        }
      }
    }
    first_group = false;
  }
}

template <int MW, int NT, int U>
int launch_lora(LoraArgs p, cudaStream_t stream) {
  constexpr int TR = 16 * MW;
  static tsds_device_flags limit_set;
  constexpr int fixed = (WARPS / MW + 1) * TR * (NT * 8 + 4) * (int)sizeof(float);
  const int smem = fixed + 2 * TR * p.ld_t * (int)sizeof(bf16);
  constexpr int most = fixed + 2 * TR * (MAX_SLICES * MAX_RANK + 16) * (int)sizeof(bf16);
  const int st = tsds_smem_limit_once(lora_kernel<MW, NT, U>, most, limit_set);
  if (st != TSDS_OK) return st;
  const int tiles = (p.M + TR - 1) / TR;
  // a cluster per adapter of a tile while the grid stays within ~1000 CTAs
  // (clusters without one leave at once); beyond that a cluster takes several
  int slots = 128 / tiles;
  slots = slots < 1 ? 1 : (slots > TR + 1 ? TR + 1 : slots);
  if (slots > p.n_adapters + 1) slots = p.n_adapters + 1;
  p.slots = slots;
  tsds_launch_cluster(lora_kernel<MW, NT, U>, dim3((unsigned)(tiles * slots * CL)), dim3(THREADS), smem, stream, CL,
                      p);
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
  if (M > 1024) return launch_lora<4, 8, 1>(p, stream);
  if (n_slices * R <= 16) return launch_lora<1, 2, 4>(p, stream);
  return launch_lora<1, 8, 2>(p, stream);
}
