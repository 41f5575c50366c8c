// LayerNorm backward over the last dimension (with the fused activation of
// rtb_layer_norm).  With u_j = (x_j - mean) rstd, z = u g + b and dz = dy
// act'(z):
//   dg = sum_rows dz u,  db = sum_rows dz
//   dx = rstd (h - mean_j(h) - u mean_j(h u)),  h = dz g
// x is fp32 or an 8-bit checkpoint (rtb_fp8.cuh); mean and rstd are the
// forward pass's.  HBM-bound: x and dy are read and dx written once (12 bytes
// an element, 9 from a checkpoint).
//
// One CTA per row, rows strided over the grid; every CTA sums dg and db of its
// rows column by column into a row of its own of a [CTA][2][d] workspace
// (fixed owners, no atomics: the result does not depend on timing), and a
// second kernel adds the CTAs' rows.
#include "rtb_act.cuh"
#include "rtb_fp8.cuh"
#include "rtb_internal.h"
#include "rtb_ptx.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 256;

struct NormBwdParams {
  int64_t rows;
  int d;
  const float* x;
  int64_t ldx;
  const uint8_t* q;
  int64_t ldq;
  const uint8_t* scale;
  int64_t lds;
  const float *mean, *rstd, *g, *b;
  int act;
  const float* dy;
  int64_t lddy;
  float* dx;
  int64_t lddx;
  float* part;  // [CTA][2][d] partial dg, db; null when neither is wanted
  int accumulate;
};

// act'(z) as a function of z; ReLU's derivative is 0 at 0 and for NaN, as its
// forward maps both to 0.
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == RTB_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == RTB_ACT_SIGMOID) {
    const float y = 1.0f / (1.0f + expf(-z));
    return y * (1.0f - y);
  }
  if (act == RTB_ACT_TANH) {
    const float y = tanhf(z);
    return 1.0f - y * y;
  }
  return 1.0f;
}

__device__ __forceinline__ float2 block_sum2(float a, float b, float (*red)[2]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();  // red[] free from the previous row
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5][0] = a;
    red[threadIdx.x >> 5][1] = b;
  }
  __syncthreads();
  a = b = 0.0f;
#pragma unroll
  for (int k = 0; k < kThreads / 32; ++k) {
    a += red[k][0];
    b += red[k][1];
  }
  return make_float2(a, b);
}

// Any width and alignment: three passes over the row's columns, the second and
// third out of L1/L2.
__global__ void __launch_bounds__(kThreads) norm_bwd_kernel(const NormBwdParams p) {
  __shared__ float red[kThreads / 32][2];
  griddep_wait();
  griddep_launch_dependents();
  float* pg = p.part ? p.part + (int64_t)blockIdx.x * 2 * p.d : nullptr;
  bool first = true;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, first = false) {
    const float mean = p.mean[r], rstd = p.rstd[r];
    const float* dyr = p.dy + r * p.lddy;
    auto at = [&](int j, float& u, float& dz, float& h) {
      float x;
      if (p.q) {
        const float s = e8m0_to_float(p.scale[r * p.lds + j / kFp8Block]);
        x = e4m3x2_to_float2(p.q[r * p.ldq + j]).x * s;
      } else {
        x = p.x[r * p.ldx + j];
      }
      u = (x - mean) * rstd;
      const float gv = p.g ? p.g[j] : 1.0f;
      dz = dyr[j];
      if (p.act != RTB_ACT_NONE) dz *= act_slope(fmaf(u, gv, p.b ? p.b[j] : 0.0f), p.act);
      h = dz * gv;
    };
    float s1 = 0.0f, s2 = 0.0f;
    for (int j = threadIdx.x; j < p.d; j += kThreads) {
      float u, dz, h;
      at(j, u, dz, h);
      s1 += h;
      s2 = fmaf(h, u, s2);
      if (pg) {
        pg[j] = first ? dz * u : fmaf(dz, u, pg[j]);
        pg[p.d + j] = first ? dz : pg[p.d + j] + dz;
      }
    }
    if (!p.dx) continue;
    const float2 t = block_sum2(s1, s2, red);
    const float m1 = t.x / p.d, m2 = t.y / p.d;
    float* dxr = p.dx + r * p.lddx;
    for (int j = threadIdx.x; j < p.d; j += kThreads) {
      float u, dz, h;
      at(j, u, dz, h);
      const float v = rstd * (h - m1 - u * m2);
      dxr[j] = p.accumulate ? dxr[j] + v : v;
    }
  }
}

// dg[j] (+)= sum over the CTAs' partial rows, db likewise (blockIdx.y picks
// one): 32 columns per CTA, 8 threads a column, in a fixed order.
__global__ void __launch_bounds__(kThreads) norm_bwd_reduce_kernel(const float* __restrict__ part,
                                                                   int ctas, int d, float* dg,
                                                                   float* db, int accumulate) {
  __shared__ float t[8][33];
  griddep_wait();
  griddep_launch_dependents();
  float* out = blockIdx.y ? db : dg;
  if (!out) return;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (j < d)
    for (int c = w; c < ctas; c += 8) s += part[((int64_t)c * 2 + blockIdx.y) * d + j];
  t[w][lane] = s;
  __syncthreads();
  if (w == 0 && j < d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += t[k][lane];
    out[j] = accumulate ? out[j] + s : s;
  }
}

}  // namespace

int norm_backward_run(rtb_ctx* ctx, const NormBwdDesc& d, cudaStream_t s) {
  NormBwdParams p{};
  p.rows = d.rows;
  p.d = (int)d.d;
  p.x = d.x;
  p.ldx = d.ldx;
  p.q = d.q;
  p.ldq = d.ldq;
  p.scale = d.scale;
  p.lds = d.lds;
  p.mean = d.mean;
  p.rstd = d.rstd;
  p.g = d.g;
  p.b = d.b;
  p.act = d.act;
  p.dy = d.dy;
  p.lddy = d.lddy;
  p.dx = d.dx;
  p.lddx = d.lddx;
  p.accumulate = d.accumulate;
  const int64_t cap = (int64_t)ctx->sm_count * 4;
  const int grid = (int)(d.rows < cap ? d.rows : cap);
  float* part = nullptr;
  int st;
  if (d.dg || d.db) {
    if ((st = ws_alloc(ctx, (void**)&part, (size_t)grid * 2 * d.d * sizeof(float), s))) return st;
    p.part = part;
  }
  clear_stale_cuda_error();
  cudaError_t e = launch_pdl(norm_bwd_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, p);
  if (e == cudaSuccess && part)
    e = launch_pdl(norm_bwd_reduce_kernel, dim3((unsigned)((d.d + 31) / 32), 2), dim3(kThreads), 0,
                   s, (const float*)part, grid, (int)d.d, d.dg, d.db, d.accumulate);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(part, s);
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "layer_norm_backward launch");
}

}  // namespace rtb
