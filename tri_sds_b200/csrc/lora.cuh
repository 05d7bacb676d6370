// What the two forms of the per-request adapters (lora.cu, lora_tc.cu) share: the
// call's arguments and the grouping of a tile's token rows by adapter.
#pragma once

#include "common.cuh"

namespace tsds {
namespace lora {

constexpr int MAX_SLICES = 4;
constexpr int MAX_RANK = 128;
constexpr int MAX_TILE = 128;   // rows per tile, at most
constexpr int NEAR = 64;       // adapters whose rank and scale every CTA reads

struct LoraArgs {
  const bf16 *x, *y, *a, *b;
  bf16* out;
  const int32_t *adapter, *ranks;
  const float* scale;
  int32_t* status;
  int64_t ldx, ldy, ldo;
  int M, K, N, R, S, n_adapters, slots, ld_t;
  int first_col[MAX_SLICES + 1];   // columns where the slices begin, and N
};

struct Tile {
  alignas(16) int32_t id[MAX_TILE];   // adapter of each row; -1: none; -2: past the last row
  uint32_t leads[MAX_TILE / 32];      // bits of the rows that are the first of their adapter
  // rank and scale of the first adapters, read beside the rows' indices rather than after them
  int32_t rank[NEAR];
  float scale[NEAR];
};

struct Adapter {
  int id, ra;   // index, rank
  float scale;
};

// The rows row0 .. row0 + rows - 1 by adapter (rows: a multiple of 4, at most
// MAX_TILE; at least MAX_TILE + NEAR threads).  Rows without an adapter are a
// group of their own where `copies`.  An index past the last adapter is never
// followed: the row keeps its projection, and the status says so where `report`.
// Ends with a barrier.
__device__ __forceinline__ void group_rows(const LoraArgs& p, Tile& sh, int row0, int rows, bool report,
                                           bool copies) {
  const int tid = threadIdx.x;
  int id = -2;
  if (tid < MAX_TILE) {
    const int m = row0 + tid;
    if (tid < rows && m < p.M) {
      id = p.adapter[m];
      if (id >= p.n_adapters && report) atomicExch(p.status, TSDS_E_INDEX);
      if (id < 0 || id >= p.n_adapters) id = -1;
    }
    sh.id[tid] = id;
  } else if (tid < MAX_TILE + NEAR) {
    const int a = tid - MAX_TILE;
    sh.rank[a] = p.ranks && a < p.n_adapters ? p.ranks[a] : p.R;
    sh.scale[a] = p.scale && a < p.n_adapters ? p.scale[a] : 1.0f;
  }
  __syncthreads();
  if (tid < MAX_TILE) {
    // without a branch: with one per row 64 rows took 3 us
    bool seen = false;
#pragma unroll 4
    for (int j = 0; j < rows; j += 4) {
      const int4 v = *reinterpret_cast<const int4*>(sh.id + j);
      seen |= ((v.x == id) & (j < tid)) | ((v.y == id) & (j + 1 < tid)) | ((v.z == id) & (j + 2 < tid)) |
              ((v.w == id) & (j + 3 < tid));
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, !seen && (id >= 0 || (id == -1 && copies)));
    if ((tid & 31) == 0) sh.leads[tid >> 5] = bits;
  }
  __syncthreads();
}

__device__ __forceinline__ Adapter adapter_of(const LoraArgs& p, const Tile& sh, int id) {
  Adapter ad;
  ad.id = id;
  if (id < NEAR) {
    ad.ra = sh.rank[id];
    ad.scale = sh.scale[id];
  } else {
    ad.ra = p.ranks ? p.ranks[id] : p.R;
    ad.scale = p.scale ? p.scale[id] : 1.0f;
  }
  ad.ra = ad.ra < 0 ? 0 : (ad.ra > p.R ? p.R : ad.ra);
  return ad;
}

// v as the sum of two bf16 words.  An infinity is in the first alone (its
// remainder would be a NaN), and a number that bf16 would round to one has the largest
// bf16 there and the rest in the second.
__device__ __forceinline__ void two_words(float v, float& hi, float& lo) {
  constexpr float most = 3.38953139e38f;   // the largest bf16
  hi = rbf(v);
  lo = v - hi;
  if (fabsf(hi) > most) {
    const bool inf = fabsf(v) > 3.40282347e38f;
    hi = inf ? v : copysignf(most, v);
    lo = inf ? 0.f : v - hi;
  }
}

}  // namespace lora
}  // namespace tsds

// The two-launch form (lora_tc.cu) and the bytes of the workspace that holds its t.
size_t tsds_lora_tc_workspace_bytes(int M, int R, int S);
int tsds_lora_tc(const tsds::lora::LoraArgs& args, void* workspace, cudaStream_t stream);
