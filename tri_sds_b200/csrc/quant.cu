// Rows to 8 bits (sm_100a): e4m3 with one fp32 scale per row, plain
// (tsds_quant_fp8) or after the residual addition and RMSNorm
// (tsds_add_rms_norm_fp8).
//
// For a row p (p = x, or p = r * w with r = bf16(x + res) and the norm's
// weights w) and c the row's norm factor (1, or rstd = 1/sqrt(mean r^2 + eps)):
//
//   s = max(c * max|p|, 2^-100) / 448,     q = e4m3((c * p) / s)
//
// c cancels in q = e4m3(p * 448 / max|p|), so one pass over the row gives
// both reductions (sum of squares and max) and q needs neither c nor a
// second look at y = c * p.  A product of two bf16 values is exact in fp32,
// and 448 / max|p| is held as two fp32 words, so p * 448 / max|p| is rounded
// once: a value half-way between two e4m3 numbers goes to the even one, as in
// exact arithmetic, instead of to the side that the scale's rounding picks.
// Sums and maxima are fp32; max.NaN keeps a NaN, so a row that holds one
// gets a NaN scale and NaN values.
//
// A row stays in one CTA's registers, so each of its bytes moves once and HBM
// bounds many rows: 10240 rows of 5120 quantised in 25.4 us (6.2 TB/s), 4096 rows
// of 5120 with residual, norm and both outputs in 30.0 us (6.3 TB/s).  Few rows are a
// launch, the row's loads and the CTA's two reductions: 26 rows of 25600 in 2.8 us.
#include "common.cuh"
#include "linear.cuh"

using namespace tsds;

namespace {

constexpr float kTop = 448.0f;              // largest e4m3 value
constexpr float kTiny = 7.88860905e-31f;    // 2^-100: smallest magnitude a row is scaled to
constexpr float kSmall = 8.67361738e-19f;   // 2^-60: products below it are moved up first,
constexpr float kUp = 1.84467441e19f;       // by 2^64

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (lo, hi) -> two e4m3 in a 16-bit word, round to nearest even, saturating
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint4 ld16(const bf16* p) { return *reinterpret_cast<const uint4*>(p); }

// bf16(a + b) of eight pairs
__device__ __forceinline__ uint4 add8(uint4 a, uint4 b) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack_bf2(bf_lo(u[i]) + bf_lo(v[i]), bf_hi(u[i]) + bf_hi(v[i]));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

struct QuantArgs {
  const bf16 *x, *res, *w;
  bf16 *res_out, *norm_out;
  uint8_t* q;
  float* scale;
  int n;
  int64_t ldx, ld_res, ld_res_out, ldq, ld_norm;
  float eps;
};

// sum += r^2, top = max|p| over a vector's eight elements
template <bool NORM>
__device__ __forceinline__ void reduce8(uint4 r, uint4 g, float& sum, float& top) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w}, w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = bf_lo(u[i]), b = bf_hi(u[i]);
    if constexpr (NORM) {
      sum = fmaf(a, a, sum);
      sum = fmaf(b, b, sum);
      top = max_nan(top, fabsf(a * bf_lo(w[i])));
      top = max_nan(top, fabsf(b * bf_hi(w[i])));
    } else {
      top = max_nan(top, max_nan(fabsf(a), fabsf(b)));
    }
  }
}

// eight elements times the row's power of two quantised (hi + lo: the two words of the
// multiplier), and with norm_out their normed values (r * rstd) * w rounded to bf16
template <bool NORM>
__device__ __forceinline__ void store8(const QuantArgs& a, uint8_t* qrow, bf16* nrow, int c, uint4 r, uint4 g, float pre,
                                       float hi, float lo, float rstd) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w}, w[4] = {g.x, g.y, g.z, g.w};
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float p0 = bf_lo(u[i]), p1 = bf_hi(u[i]);
    if constexpr (NORM) {
      p0 *= bf_lo(w[i]);
      p1 *= bf_hi(w[i]);
      p0 *= pre;
      p1 *= pre;
    }
    h[i] = pack_e4m3x2(fmaf(p0, hi, p0 * lo), fmaf(p1, hi, p1 * lo));
  }
  *reinterpret_cast<uint2*>(qrow + c * 8) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  if constexpr (NORM) {
    if (nrow) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = pack_bf2(bf_lo(u[i]) * rstd * bf_lo(w[i]), bf_hi(u[i]) * rstd * bf_hi(w[i]));
      *reinterpret_cast<uint4*>(nrow + c * 8) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// One CTA of NT threads per row.  Rows of at most NT * VMAX 16-byte vectors are read
// once and kept in registers; longer ones are read a second time (from
// res_out when there is a residual).
template <bool NORM, int NT, int VMAX>
__global__ void __launch_bounds__(NT) quant_rows_kernel(QuantArgs a) {
  __shared__ float red_s[NT / 32], red_m[NT / 32];
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const int nv = a.n / 8, t = threadIdx.x;
  const bf16* xr = a.x + row * a.ldx;
  const bf16* rr = a.res ? a.res + row * a.ld_res : nullptr;
  bf16* ro = a.res ? a.res_out + row * a.ld_res_out : nullptr;
  uint8_t* qr = a.q + row * a.ldq;
  bf16* nr = a.norm_out ? a.norm_out + row * a.ld_norm : nullptr;
  const bool keep = nv <= NT * VMAX;
  uint4 v[VMAX], g[VMAX];
  // the weights too may come from the kernel before (1 + gamma, say), so nothing is read
  // earlier, and by plain loads: 4.18 us instead of 4.10 at 208 rows of 5120
  pdl_wait();
  float sum = 0.f, top = 0.f;
  if (keep) {
    uint4 b[VMAX];
#pragma unroll
    for (int i = 0; i < VMAX; ++i) {
      const int c = t + i * NT;
      v[i] = c < nv ? ld16(xr + c * 8) : make_uint4(0, 0, 0, 0);
      if (NORM && rr && c < nv) b[i] = ld16(rr + c * 8);
      if constexpr (NORM) g[i] = c < nv ? ld16(a.w + c * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VMAX; ++i) {
      const int c = t + i * NT;
      if (c < nv) {
        if (NORM && rr) {
          v[i] = add8(v[i], b[i]);
          *reinterpret_cast<uint4*>(ro + c * 8) = v[i];
        }
        reduce8<NORM>(v[i], g[i], sum, top);
      }
    }
  } else {
    for (int c = t; c < nv; c += NT) {
      uint4 r = ld16(xr + c * 8);
      uint4 w = make_uint4(0, 0, 0, 0);
      if constexpr (NORM) {
        w = ld16(a.w + c * 8);
        if (rr) {
          r = add8(r, ld16(rr + c * 8));
          *reinterpret_cast<uint4*>(ro + c * 8) = r;
        }
      }
      reduce8<NORM>(r, w, sum, top);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if constexpr (NORM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if ((t & 31) == 0) {
    red_s[t >> 5] = sum;
    red_m[t >> 5] = top;
  }
  __syncthreads();
  sum = 0.f;
  top = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    sum += red_s[i];
    top = max_nan(top, red_m[i]);
  }
  const float rstd = NORM ? 1.0f / sqrtf(sum / (float)a.n + a.eps) : 1.0f;
  const float amax = rstd * top;
  // Where rstd lifts a row of tiny products the multiplier could pass the largest fp32
  // number (a row of zeros with eps = 1e-12: 0 * inf): the products are
  // moved up by a power of two, exactly, and the multiplier is as much smaller.
  const float pre = NORM && top < kSmall ? kUp : 1.0f;
  float hi, lo = 0.f;
  if (amax >= kTiny) {
    const float m = top * pre;
    hi = kTop / m;
    lo = fmaf(-hi, m, kTop) / m;
  } else {  // an (almost) empty row, or a NaN
    hi = amax != amax ? amax : rstd * (kTop / kTiny / pre);
  }
  if (t == 0) a.scale[row] = (amax < kTiny ? kTiny : amax) / kTop;
  if (keep) {
#pragma unroll
    for (int i = 0; i < VMAX; ++i) {
      const int c = t + i * NT;
      if (c < nv) store8<NORM>(a, qr, nr, c, v[i], g[i], pre, hi, lo, rstd);
    }
  } else {
    const bf16* src = NORM && rr ? ro : xr;
    for (int c = t; c < nv; c += NT) {
      const uint4 w = NORM ? ld16(a.w + c * 8) : make_uint4(0, 0, 0, 0);
      store8<NORM>(a, qr, nr, c, ld16(src + c * 8), w, pre, hi, lo, rstd);
    }
  }
}

template <bool NORM, int NT, int VMAX>
int launch(const QuantArgs& a, int rows, cudaStream_t stream) {
  tsds_launch(quant_rows_kernel<NORM, NT, VMAX>, dim3(rows), dim3(NT), 0, stream, a);
  return tsds_launch_status();
}

// Rows of up to 8192 elements: 256 threads.  Longer ones: 1024 threads where
// the rows are few and one row's time is what counts; with many rows half as
// many threads with twice the vectors each keep more loads in flight per SM
// (quantising 5809 rows of 9024: 28.8 us, 55 with 1024 threads).  The threads set the
// order in which a norm's squares are summed, so above 8192 elements a row's last
// bits may differ between calls of few and of many rows.
template <bool NORM>
int launch_rows(const QuantArgs& a, int rows, cudaStream_t stream) {
  if (a.n <= 8192) return launch<NORM, 256, 4>(a, rows, stream);
  if (rows < 2 * tsds_tc_num_sms() || a.n > 32768) return launch<NORM, 1024, 4>(a, rows, stream);
  if (a.n <= 16384) return launch<NORM, NORM ? 512 : 256, NORM ? 4 : 8>(a, rows, stream);
  return launch<NORM, 512, 8>(a, rows, stream);
}

tsds_rows rows_bf16(const void* p, int rows, int ld, int n) { return {p, rows, ld * (int64_t)2, n * (int64_t)2}; }

// Whether an output may lie where it does beside a bf16 operand of the same rows: apart from it, or
// exactly on it.
bool apart_or_same(const tsds_rows& out, const tsds_rows& in) {
  return (out.base == in.base && out.ld == in.ld) || !tsds_overlap(out, in);
}

}  // namespace

extern "C" int tsds_quant_fp8(const void* x, void* q, float* scale, int rows, int n, int ldx, int ldq,
                              tsds_stream_t stream) {
  TSDS_RETURN_IF(rows < 0 || n <= 0 || (n % 16) != 0 || ldx < n || ldq < n, TSDS_E_INVALID);
  if (rows == 0) return TSDS_OK;
  TSDS_RETURN_IF(!x || !q || !scale, TSDS_E_INVALID);
  TSDS_RETURN_IF(!tsds_aligned16(x) || !tsds_aligned16(q) || (ldx % 8) || (ldq % 16), TSDS_E_ALIGN);
  // (a long row is read twice, the second time after its first bytes are written)
  TSDS_RETURN_IF(tsds_overlap({q, rows, ldq, n}, rows_bf16(x, rows, ldx, n)), TSDS_E_INVALID);
  QuantArgs a = {};
  a.x = (const bf16*)x;
  a.q = (uint8_t*)q;
  a.scale = scale;
  a.n = n;
  a.ldx = ldx;
  a.ldq = ldq;
  return launch_rows<false>(a, rows, stream);
}

extern "C" int tsds_add_rms_norm_fp8(const void* x, const void* res, const void* w, void* res_out, void* q,
                                     float* scale, void* norm_out, int rows, int n, int ldx, int ld_res,
                                     int ld_res_out, int ldq, int ld_norm, float eps, tsds_stream_t stream) {
  TSDS_RETURN_IF(rows < 0 || n <= 0 || (n % 16) != 0 || ldx < n || ldq < n, TSDS_E_INVALID);
  TSDS_RETURN_IF((res && (ld_res < n || ld_res_out < n)) || (norm_out && ld_norm < n), TSDS_E_INVALID);
  if (rows == 0) return TSDS_OK;
  TSDS_RETURN_IF(!x || !w || !q || !scale || (res && !res_out), TSDS_E_INVALID);
  TSDS_RETURN_IF(!tsds_aligned16(x) || !tsds_aligned16(w) || !tsds_aligned16(q) || (ldx % 8) || (ldq % 16),
                 TSDS_E_ALIGN);
  TSDS_RETURN_IF(res && (!tsds_aligned16(res) || !tsds_aligned16(res_out) || (ld_res % 8) || (ld_res_out % 8)),
                 TSDS_E_ALIGN);
  TSDS_RETURN_IF(res && ((res_out == res && ld_res_out != ld_res) || (res_out == x && ld_res_out != ldx)),
                 TSDS_E_INVALID);
  TSDS_RETURN_IF(norm_out && (!tsds_aligned16(norm_out) || (ld_norm % 8)), TSDS_E_ALIGN);
  const tsds_rows rx = rows_bf16(x, rows, ldx, n), rr = rows_bf16(res, rows, ld_res, n),
                  ro = rows_bf16(res ? res_out : nullptr, rows, ld_res_out, n),
                  rn = rows_bf16(norm_out, rows, ld_norm, n), rq = {q, rows, ldq, n};
  TSDS_RETURN_IF(tsds_overlap(rq, rx) || tsds_overlap(rq, rr) || tsds_overlap(rq, ro) || tsds_overlap(rq, rn) ||
                     tsds_overlap(rn, ro) || !apart_or_same(ro, rx) || !apart_or_same(ro, rr) ||
                     !apart_or_same(rn, rx) || !apart_or_same(rn, rr),
                 TSDS_E_INVALID);
  QuantArgs a = {};
  a.x = (const bf16*)x;
  a.res = (const bf16*)res;
  a.w = (const bf16*)w;
  a.res_out = (bf16*)res_out;
  a.norm_out = (bf16*)norm_out;
  a.q = (uint8_t*)q;
  a.scale = scale;
  a.n = n;
  a.ldx = ldx;
  a.ld_res = ld_res;
  a.ld_res_out = ld_res_out;
  a.ldq = ldq;
  a.ld_norm = ld_norm;
  a.eps = eps;
  return launch_rows<true>(a, rows, stream);
}
