// Root-mean-square norm over the last dimension with the residual's addition:
//   h = x + residual,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w
// y is written as fp32 or as 8-bit blocks (rtb_fp8.cuh: e4m3, a power-of-two scale
// for each 128 columns of a row), h as fp32 where it is wanted, rstd for the
// backward pass (rtb_norm_bwd.cu).  HBM-bound: x and the residual are read once, h
// and y written once.
//
// A row of up to 16384 columns lives in the registers of a group of 32..512
// threads: warp w of the group holds the 128-column blocks w, w + W, ..., so that
// an 8-bit block's maximum is one warp's.  Squares and their sum are double: fp32 ones
// leave its range from magnitudes of 2e19 on (and under 1e-23), and are off by more than
// the middle of two 8-bit codes forgives (up to 1e-7 of rstd; the conversions cost 0 to 8%,
// 65536 x 512 with the 8-bit output 41.2 -> 44.5 us).  1024 threads of 64 registers share an
// SM: that many rows in flight hide a row's chain of loads, sum and stores (with fp32
// squares, 16 values a thread of 512 and not 32 of 256, 4095 x 8191: 92 us, 96; 32 of 512
// and not 64 of 256, 2047 x 16383: 97 us, 142).  Wider rows take a CTA each and two passes,
// the second out of L2.
//
// Measured: 8192 x 4096 with a residual 89 us (6.0 TB/s, 92% of a copy), with the 8-bit
// output 71 (6.2 TB/s); 16384 x 2048 88 and 71 us, 2048 x 16384 92 and 90, 8192 x 4097 103
// and 107, 600 x 40000 97 and 99.
#include "rtb_fp8.cuh"
#include "rtb_internal.h"
#include "rtb_ptx.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 256;

struct RmsParams {
  int64_t rows;
  int d;
  const float* x;
  int64_t ldx;
  const float* r;  // residual, or null
  int64_t ldr;
  const float* w;  // null: 1
  float eps;
  double inv_d;
  float* h;        // null: not wanted
  int64_t ldh;
  float* y;        // fp32 output
  int64_t ldy;
  uint8_t* q;      // 8-bit output
  int64_t ldq;
  uint8_t* scale;
  int64_t lds;
  float* rstd;     // null: not wanted
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's four columns of the 128-column block that begins at c0 (4 lane + j, or
// lane + 32 j where rows are off the 16-byte boundaries); 0 past the row's d.
template <bool VEC>
__device__ __forceinline__ void load4(const float* row, int c0, int d, int lane, float (&v)[4]) {
  if (VEC) {
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c0 + 4 * lane < d) f = *reinterpret_cast<const float4*>(row + c0 + 4 * lane);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c0 + lane + 32 * j < d ? row[c0 + lane + 32 * j] : 0.0f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store4(float* row, int c0, int d, int lane, const float (&v)[4]) {
  if (VEC) {
    if (c0 + 4 * lane < d)
      __stcs(reinterpret_cast<float4*>(row + c0 + 4 * lane), make_float4(v[0], v[1], v[2], v[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + lane + 32 * j < d) __stcs(row + c0 + lane + 32 * j, v[j]);
  }
}

// The row's statistic, rounded, and its factors: rstd = scale (hi + lo), scale a power of
// two and hi in [1, 2) but at the ends of fp32's range.  A row's values times scale are of
// the order of 1, so that y is exact to its last place where rstd itself, of a row beyond
// 8e37 or under 3e-39, is no normal number of fp32.
struct Rstd {
  float value, scale, hi, lo;
};
__device__ __forceinline__ Rstd rstd_of(double total, double inv_d, float eps) {
  const double r = rsqrt(fma(total, inv_d, (double)eps));
  const int e = min(max((__double2hiint(r) >> 20 & 0x7FF) - 1023, -126), 127);
  const double unit = r * __hiloint2double((1023 - e) << 20, 0);
  const float hi = (float)unit;
  return {(float)r, __int_as_float((e + 127) << 23), hi, (float)(unit - (double)hi)};
}
// h (r.hi + r.lo) w in fp32 as the next rounding wants it: where the product is no fp32
// number, the one of its two neighbours with an odd last bit, which is never half way
// between two codes.
__device__ __forceinline__ float product_to_odd(float h, Rstd r, float w) {
  const float u = h * r.hi, ue = fmaf(h, r.lo, fmaf(h, r.hi, -u));
  const float y = u * w, ye = fmaf(ue, w, fmaf(u, w, -y));
  const float s = y + ye, rest = ye - (s - y);
  const uint32_t bits = __float_as_uint(s);
  if ((bits & 1u) || !(fabsf(rest) > 0.0f) || s == 0.0f) return s;  // (NaN: s is no number)
  return __uint_as_float((rest > 0.0f) == (s > 0.0f) ? bits + 1 : bits - 1);
}

// y of a block's four columns, from h times the row's scale, and its way out.
template <bool VEC, bool FP8>
__device__ __forceinline__ void finish4(const RmsParams& p, int64_t m, int c0, int lane, Rstd rstd,
                                        const float (&h)[4]) {
  float y[4], w[4] = {1.0f, 1.0f, 1.0f, 1.0f};
  if (p.w) load4<VEC>(p.w, c0, p.d, lane, w);
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = h[j] * rstd.hi * w[j];
  if (!FP8) {
    store4<VEC>(p.y + m * p.ldy, c0, p.d, lane, y);
    return;
  }
  // A value is to be rounded once, to 8 bits, and y has been three times, by 3 units of its
  // last place at most.  That changes a code only within as much of the middle of two codes
  // (or, the block's scale, of 448 times a power of two), numbers of five bits, whose last
  // 19 are zero: these few (1 in 60000) are multiplied again with twice the digits.
  constexpr uint32_t kNear = 8u << 13;
  auto off = [&](int j) { return (__float_as_uint(y[j]) << 13) + (kNear >> 1); };
  if (min(min(off(0), off(1)), min(off(2), off(3))) < kNear) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (off(j) < kNear && y[j] != 0.0f && fabsf(y[j]) <= 3.402823466e38f)
        y[j] = product_to_odd(h[j], rstd, w[j]);
  }
  // (magnitudes compare as their bits do)
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a = __float_as_uint(finite_abs(y[j]));
    top = a > top ? a : top;
  }
  const uint32_t sb = e8m0_of_amax(__uint_as_float(__reduce_max_sync(0xffffffffu, top)));
  const uint32_t four = e4m3x4(y[0], y[1], y[2], y[3], e8m0_inverse(sb));
  uint8_t* qr = p.q + m * p.ldq + c0;
  if (VEC) {
    if (c0 + 4 * lane < p.d) *reinterpret_cast<uint32_t*>(qr + 4 * lane) = four;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + lane + 32 * j < p.d) qr[lane + 32 * j] = (uint8_t)(four >> (8 * j));
  }
  if (lane == 0) p.scale[m * p.lds + c0 / kFp8Block] = (uint8_t)sb;
}

constexpr int cta(int T) { return T > kThreads ? T : kThreads; }

// T threads a row, NB blocks of 128 columns a warp.
template <int T, int NB, bool VEC, bool FP8>
__global__ void __launch_bounds__(cta(T), T == 512 ? 2 : 4) rms_rows_kernel(const RmsParams p) {
  constexpr int R = cta(T) / T;  // rows a CTA works on
  constexpr int W = T / 32;        // warps a row
  __shared__ double red[2][R][W];  // two buffers, so that one barrier a row is enough
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, grp = threadIdx.x / T, w = (threadIdx.x % T) >> 5;
  int phase = 0;
  for (int64_t m = (int64_t)blockIdx.x * R + grp; m < p.rows;
       m += (int64_t)gridDim.x * R, phase ^= 1) {
    float h[NB][4];
    const float* xr = p.x + m * p.ldx;
#pragma unroll
    for (int i = 0; i < NB; ++i) load4<VEC>(xr, 128 * (w + W * i), p.d, lane, h[i]);
    if (p.r) {
      const float* rr = p.r + m * p.ldr;
      float r[NB][4];
#pragma unroll
      for (int i = 0; i < NB; ++i) load4<VEC>(rr, 128 * (w + W * i), p.d, lane, r[i]);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) h[i][j] += r[i][j];
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = fma((double)h[i][j], (double)h[i][j], ss);
    double total = warp_sum(ss);
    if (W > 1) {
      if (lane == 0) red[phase][grp][w] = total;
      named_bar_sync(1 + grp, T);
      total = 0.0;
#pragma unroll
      for (int k = 0; k < W; ++k) total += red[phase][grp][k];
    }
    const Rstd rstd = rstd_of(total, p.inv_d, p.eps);
    if (p.rstd && lane == 0 && w == 0) p.rstd[m] = rstd.value;
    if (p.h) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
        store4<VEC>(p.h + m * p.ldh, 128 * (w + W * i), p.d, lane, h[i]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] *= rstd.scale;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (128 * (w + W * i) < p.d) finish4<VEC, FP8>(p, m, 128 * (w + W * i), lane, rstd, h[i]);
  }
}

// Any width: a CTA a row.  A column stays with one thread in both passes, so that
// outputs may lie where inputs do.
template <bool VEC, bool FP8>
__global__ void __launch_bounds__(kThreads) rms_wide_kernel(const RmsParams p) {
  constexpr int W = kThreads / 32;
  __shared__ double red[W];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int blocks = (p.d + 127) / 128;
  for (int64_t m = blockIdx.x; m < p.rows; m += gridDim.x) {
    auto input = [&](int c0, float (&h)[4]) {
      load4<VEC>(p.x + m * p.ldx, c0, p.d, lane, h);
      if (p.r) {
        float r[4];
        load4<VEC>(p.r + m * p.ldr, c0, p.d, lane, r);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] += r[j];
      }
    };
    double ss = 0.0;
#pragma unroll 4
    for (int b = w; b < blocks; b += W) {
      float h[4];
      input(128 * b, h);
      if (p.h) store4<VEC>(p.h + m * p.ldh, 128 * b, p.d, lane, h);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss += (double)h[j] * h[j];
    }
    const double part = warp_sum(ss);
    __syncthreads();  // red[] free from the previous row
    if (lane == 0) red[w] = part;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int k = 0; k < W; ++k) total += red[k];
    const Rstd rstd = rstd_of(total, p.inv_d, p.eps);
    if (p.rstd && threadIdx.x == 0) p.rstd[m] = rstd.value;
    for (int b = w; b < blocks; b += W) {
      float h[4];
      if (p.h) load4<VEC>(p.h + m * p.ldh, 128 * b, p.d, lane, h);
      else input(128 * b, h);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] *= rstd.scale;
      finish4<VEC, FP8>(p, m, 128 * b, lane, rstd, h);
    }
  }
}

int launch(rtb_ctx* ctx, void (*k)(const RmsParams), int64_t ctas, int threads, const RmsParams& p,
           cudaStream_t s) {
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  clear_stale_cuda_error();
  cudaError_t e = launch_pdl(k, dim3((unsigned)(ctas < cap ? ctas : cap)), dim3((unsigned)threads), 0, s, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "rms_norm launch");
}

template <int T, int NB, bool VEC, bool FP8>
int rows_as(rtb_ctx* ctx, const RmsParams& p, cudaStream_t s) {
  constexpr int R = cta(T) / T;
  return launch(ctx, rms_rows_kernel<T, NB, VEC, FP8>, (p.rows + R - 1) / R, cta(T), p, s);
}

template <bool VEC, bool FP8>
int run(rtb_ctx* ctx, const RmsParams& p, cudaStream_t s) {
  const int blocks = (p.d + 127) / 128;
  if (blocks <= 1) return rows_as<32, 1, VEC, FP8>(ctx, p, s);
  if (blocks <= 2) return rows_as<32, 2, VEC, FP8>(ctx, p, s);
  if (blocks <= 4) return rows_as<32, 4, VEC, FP8>(ctx, p, s);
  if (blocks <= 8) return rows_as<64, 4, VEC, FP8>(ctx, p, s);
  if (blocks <= 16) return rows_as<128, 4, VEC, FP8>(ctx, p, s);
  if (blocks <= 32) return rows_as<256, 4, VEC, FP8>(ctx, p, s);
  if (blocks <= 64) return rows_as<512, 4, VEC, FP8>(ctx, p, s);
  if (blocks <= 128) return rows_as<512, 8, VEC, FP8>(ctx, p, s);
  return launch(ctx, rms_wide_kernel<VEC, FP8>, p.rows, kThreads, p, s);
}

}  // namespace

int rms_norm_run(rtb_ctx* ctx, const RmsDesc& d, cudaStream_t s) {
  RmsParams p{};
  p.rows = d.rows;
  p.d = (int)d.d;
  p.x = d.x;
  p.ldx = d.ldx;
  p.r = d.residual;
  p.ldr = d.ldr;
  p.w = d.w;
  p.eps = d.eps;
  p.inv_d = 1.0 / (double)p.d;
  p.h = d.sum;
  p.ldh = d.ldsum;
  p.y = d.y;
  p.ldy = d.ldy;
  p.q = d.q;
  p.ldq = d.ldq;
  p.scale = d.scale;
  p.lds = d.lds;
  p.rstd = d.rstd;
  auto al = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n == 0; };
  const bool vec = d.d % 4 == 0 && al(d.x, 16) && d.ldx % 4 == 0 && al(d.w, 16) &&
                   (!d.residual || (al(d.residual, 16) && d.ldr % 4 == 0)) &&
                   (!d.sum || (al(d.sum, 16) && d.ldsum % 4 == 0)) &&
                   (d.q ? al(d.q, 4) && d.ldq % 4 == 0 : al(d.y, 16) && d.ldy % 4 == 0);
  if (d.q) return vec ? run<true, true>(ctx, p, s) : run<false, true>(ctx, p, s);
  return vec ? run<true, false>(ctx, p, s) : run<false, false>(ctx, p, s);
}

}  // namespace rtb
