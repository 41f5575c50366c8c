// LayerNorm backward over the last dimension (with the fused activation of
// rtb_layer_norm).  With u_j = (x_j - mean) rstd, z = u g + b and dz = dy
// act'(z):
//   dg = sum_rows dz u,  db = sum_rows dz
//   dx = rstd (h - mean_j(h) - u mean_j(h u)),  h = dz g
// x is fp32 or an 8-bit checkpoint (rtb_fp8.cuh); mean and rstd are the
// forward pass's.  HBM-bound: x and dy are read and dx written once (12 bytes
// an element, 9 from a checkpoint).
//
// A row belongs to a group of T threads that holds it in registers (E values of
// x and dy a thread; the loads of a row are all in flight before its one
// reduction of two sums), rows strided over the groups of the resident CTAs.
// dg and db are sums over rows, one column always with the same thread: E
// running sums each in registers (in shared memory for rows beyond 8192
// columns, where 1024 threads leave 64 registers a thread), added up over a
// CTA's groups in group order, left in a row of a [CTA][2][d] workspace, and
// the CTAs' rows are added by a second kernel.  No atomics: the order depends on
// the shape alone.  A single CTA writes its sums itself.  Rows beyond 16384
// columns take a CTA each and three passes.
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

// out (+)= v
__device__ __forceinline__ void put(float* out, float v, int accumulate) {
  *out = accumulate ? *out + v : v;
}

// VEC: thread t of the group holds the float4 units t + T i (d % 4 == 0,
// 16-byte aligned rows), else the columns t + T i.  SAVED: x from the
// checkpoint.  Partial sums over at most E values in fp32, then shuffles and
// the group's warps in order.
template <int T, int E, bool VEC, bool SAVED>
__global__ void __launch_bounds__(T > 256 ? T : 256, T > 512 ? 1 : (T > 256 ? 1 : 2))
    norm_bwd_rows_kernel(const NormBwdParams p, float* dg, float* db) {
  constexpr int kBlock = T > 256 ? T : 256;
  constexpr int G = VEC ? E / 4 : E;  // loads of x (and of dy) a thread
  constexpr int C = E / G;            // columns of a load
  constexpr int R = kBlock / T;       // rows a CTA works on
  constexpr int W = T / 32;
  constexpr bool kAccSmem = T == 1024;
  __shared__ float red[2][R][W][2];
  extern __shared__ float acc_s[];  // [2][d]: the CTA's sums (kAccSmem: running)
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x % T, grp = threadIdx.x / T;
  const int units = VEC ? p.d >> 2 : p.d;
  const bool sums = p.part || dg || db;
  float ag[kAccSmem ? 1 : E], ab[kAccSmem ? 1 : E];
#pragma unroll
  for (int i = 0; i < (kAccSmem ? 1 : E); ++i) ag[i] = ab[i] = 0.0f;
  if (kAccSmem && sums) {
    for (int j = threadIdx.x; j < 2 * p.d; j += kBlock) acc_s[j] = 0.0f;
    __syncthreads();
  }
  int phase = 0;
  for (int64_t r = (int64_t)blockIdx.x * R + grp; r < p.rows; r += (int64_t)gridDim.x * R, phase ^= 1) {
    float u[E], h[E];  // x, then u; dy, then h
    const float mean = __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
    const float* dyr = p.dy + r * p.lddy;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = t + T * i;
      const bool in = k < units;
      if (VEC) {
        float4 a = make_float4(mean, mean, mean, mean), g = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in) {
          if (SAVED) {
            const uint32_t four = __ldcs(reinterpret_cast<const uint32_t*>(p.q + r * p.ldq) + k);
            const float s = e8m0_to_float(__ldg(p.scale + r * p.lds + (k >> 5)));
            a = e4m3x4_to_float4(four);
            a.x *= s; a.y *= s; a.z *= s; a.w *= s;
          } else {
            a = __ldcs(reinterpret_cast<const float4*>(p.x + r * p.ldx) + k);
          }
          g = __ldcs(reinterpret_cast<const float4*>(dyr) + k);
        }
        u[4 * i] = a.x; u[4 * i + 1] = a.y; u[4 * i + 2] = a.z; u[4 * i + 3] = a.w;
        h[4 * i] = g.x; h[4 * i + 1] = g.y; h[4 * i + 2] = g.z; h[4 * i + 3] = g.w;
      } else {
        u[i] = mean;
        h[i] = 0.0f;
        if (in) {
          if (SAVED) {
            const float s = e8m0_to_float(__ldg(p.scale + r * p.lds + k / kFp8Block));
            u[i] = e4m3x2_to_float2(__ldcs(p.q + r * p.ldq + k)).x * s;
          } else {
            u[i] = __ldcs(p.x + r * p.ldx + k);
          }
          h[i] = __ldcs(dyr + k);
        }
      }
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = t + T * i;
      float gv[C], bv[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        gv[c] = 1.0f;
        bv[c] = 0.0f;
      }
      if (k < units) {
        if (VEC) {
          if (p.g) *reinterpret_cast<float4*>(gv) = __ldg(reinterpret_cast<const float4*>(p.g) + k);
          if (p.b && p.act != RTB_ACT_NONE)
            *reinterpret_cast<float4*>(bv) = __ldg(reinterpret_cast<const float4*>(p.b) + k);
        } else {
          if (p.g) gv[0] = __ldg(p.g + k);
          if (p.b && p.act != RTB_ACT_NONE) bv[0] = __ldg(p.b + k);
        }
      }
      float4 sg, sb;
      if (kAccSmem && sums && k < units && VEC) {
        sg = reinterpret_cast<const float4*>(acc_s)[k];
        sb = reinterpret_cast<const float4*>(acc_s + p.d)[k];
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = C * i + c;
        u[e] = (u[e] - mean) * rstd;
        float dz = h[e];
        if (p.act != RTB_ACT_NONE) dz *= act_slope(fmaf(u[e], gv[c], bv[c]), p.act);
        if (!kAccSmem) {
          ag[e] = fmaf(dz, u[e], ag[e]);
          ab[e] += dz;
        } else if (sums && k < units) {
          if (VEC) {
            (&sg.x)[c] = fmaf(dz, u[e], (&sg.x)[c]);
            (&sb.x)[c] += dz;
          } else {
            acc_s[k] = fmaf(dz, u[e], acc_s[k]);
            acc_s[p.d + k] += dz;
          }
        }
        h[e] = dz * gv[c];
        s1 += h[e];
        s2 = fmaf(h[e], u[e], s2);
      }
      if (kAccSmem && sums && k < units && VEC) {
        reinterpret_cast<float4*>(acc_s)[k] = sg;
        reinterpret_cast<float4*>(acc_s + p.d)[k] = sb;
      }
    }
    if (!p.dx) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    if (W > 1) {
      // two buffers, so that one barrier a row is enough
      if ((t & 31) == 0) {
        red[phase][grp][t >> 5][0] = s1;
        red[phase][grp][t >> 5][1] = s2;
      }
      named_bar_sync(1 + grp, T);
      s1 = s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k) {
        s1 += red[phase][grp][k][0];
        s2 += red[phase][grp][k][1];
      }
    }
    const float m1 = s1 / p.d, m2 = s2 / p.d;
    float* dxr = p.dx + r * p.lddx;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = t + T * i;
      if (k >= units) continue;
      float v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = rstd * (h[C * i + c] - m1 - u[C * i + c] * m2);
      if (VEC) {
        float4* o = reinterpret_cast<float4*>(dxr) + k;
        float4 w = *reinterpret_cast<const float4*>(v);
        if (p.accumulate) {
          const float4 q = *o;
          w.x += q.x; w.y += q.y; w.z += q.z; w.w += q.w;
        }
        __stcs(o, w);
      } else {
        put(dxr + k, v[0], p.accumulate);
      }
    }
  }
  if (!sums) return;
  // the CTA's sums over its groups, in group order
  if (!kAccSmem) {
    for (int gi = 0; gi < R; ++gi) {
      if (grp == gi) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const int k = t + T * i;
          if (k >= units) continue;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            put(acc_s + C * k + c, ag[C * i + c], gi > 0);
            put(acc_s + p.d + C * k + c, ab[C * i + c], gi > 0);
          }
        }
      }
      __syncthreads();
    }
  } else {
    __syncthreads();
  }
  for (int j = threadIdx.x; j < p.d; j += kBlock) {
    if (p.part) {
      float* pr = p.part + (int64_t)blockIdx.x * 2 * p.d;
      pr[j] = acc_s[j];
      pr[p.d + j] = acc_s[p.d + j];
    } else {
      if (dg) put(dg + j, acc_s[j], p.accumulate);
      if (db) put(db + j, acc_s[p.d + j], p.accumulate);
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

template <int T, int E, bool VEC, bool SAVED>
int launch_rows(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  constexpr int kBlock = T > 256 ? T : 256;
  constexpr int R = kBlock / T;
  auto* k = norm_bwd_rows_kernel<T, E, VEC, SAVED>;
  const size_t smem = (dg || db) ? (size_t)2 * p.d * sizeof(float) : 0;
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_status(e, "layer_norm_backward smem attribute");
  }
  int per_sm = 1;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, kBlock, smem);
  if (per_sm < 1) per_sm = 1;
  const int64_t need = (p.rows + R - 1) / R, cap = (int64_t)ctx->sm_count * per_sm;
  const int grid = (int)(need < cap ? need : cap);
  if (!dg && !db) {
    clear_stale_cuda_error();
    e = launch_pdl(k, dim3((unsigned)grid), dim3(kBlock), 0, s, (const NormBwdParams)p,
                   (float*)nullptr, (float*)nullptr);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? RTB_OK : cuda_status(e, "layer_norm_backward launch");
  }
  float* part = nullptr;
  if (grid > 1) {
    const int st = ws_alloc(ctx, (void**)&part, (size_t)grid * 2 * p.d * sizeof(float), s);
    if (st) return st;
  }
  p.part = part;
  clear_stale_cuda_error();
  e = launch_pdl(k, dim3((unsigned)grid), dim3(kBlock), smem, s, (const NormBwdParams)p, dg, db);
  if (e == cudaSuccess && part)
    e = launch_pdl(norm_bwd_reduce_kernel, dim3((unsigned)((p.d + 31) / 32), 2), dim3(kThreads), 0,
                   s, (const float*)part, grid, p.d, dg, db, p.accumulate);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(part, s);
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "layer_norm_backward launch");
}

template <bool VEC, bool SAVED>
int launch_width(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  if (p.d <= 128) return launch_rows<32, 4, VEC, SAVED>(ctx, p, dg, db, s);
  if (p.d <= 256) return launch_rows<32, 8, VEC, SAVED>(ctx, p, dg, db, s);
  if (p.d <= 512) return launch_rows<32, 16, VEC, SAVED>(ctx, p, dg, db, s);
  if (p.d <= 1024) return launch_rows<64, 16, VEC, SAVED>(ctx, p, dg, db, s);
  if (p.d <= 2048) return launch_rows<128, 16, VEC, SAVED>(ctx, p, dg, db, s);
  if (p.d <= 4096) return launch_rows<256, 16, VEC, SAVED>(ctx, p, dg, db, s);
  if (p.d <= 8192) return launch_rows<512, 16, VEC, SAVED>(ctx, p, dg, db, s);
  return launch_rows<1024, 16, VEC, SAVED>(ctx, p, dg, db, s);
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
  if (d.d <= 16384) {
    auto al = [](const void* q, uintptr_t n) { return (reinterpret_cast<uintptr_t>(q) % n) == 0; };
    const bool vec = d.d % 4 == 0 && al(d.dy, 16) && d.lddy % 4 == 0 &&
                     (!d.dx || (al(d.dx, 16) && d.lddx % 4 == 0)) && (!d.g || al(d.g, 16)) &&
                     (!d.b || al(d.b, 16)) &&
                     (d.q ? al(d.q, 4) && d.ldq % 4 == 0 : al(d.x, 16) && d.ldx % 4 == 0);
    if (d.q) return vec ? launch_width<true, true>(ctx, p, d.dg, d.db, s)
                        : launch_width<false, true>(ctx, p, d.dg, d.db, s);
    return vec ? launch_width<true, false>(ctx, p, d.dg, d.db, s)
               : launch_width<false, false>(ctx, p, d.dg, d.db, s);
  }
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
