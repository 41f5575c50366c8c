// LayerNorm backward over the last dimension (with the fused activation of
// rtb_layer_norm).  With u_j = (x_j - mean) rstd, z = u g + b and dz = dy
// act'(z):
//   dg = sum_rows dz u,  db = sum_rows dz
//   dx = rstd (h - mean_j(h) - u mean_j(h u)),  h = dz g
// x is fp32 or an 8-bit checkpoint (rtb_fp8.cuh); mean and rstd are the
// forward pass's.  HBM-bound: x and dy are read and dx written once (12 bytes
// an element, 9 from a checkpoint).
//
// A row belongs to a group of threads that holds it in registers, rows strided
// over the groups of the resident CTAs; one reduction of two sums a row.  dg and
// db are sums over rows, one column always with the same thread: running sums in
// registers (in shared memory for rows beyond 8192 columns, where 1024 threads
// leave 64 registers each), added up over a CTA's groups in group order, left in
// a row of a [CTA][2][d] workspace, and the CTAs' rows are added by a second
// kernel.  No atomics: the order depends on the shape alone.  A single CTA writes
// its sums itself.  Rows beyond 16384 columns take a CTA each and three passes.
//
// Measured: 8192 x 4096 80 us (5.0 TB/s of the 12 bytes an element, 77% of a copy),
// 16384 x 2048 from a checkpoint 77 us (3.9 TB/s of 9 bytes: the instructions of
// the row's fixed part count as much), 2048 x 16384 111 us, 8192 x 4097 140 us.
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

constexpr int kRing = 3;  // stages of the row ring: 96 KB for 512 threads of 8 values

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Up to 8192 columns: T threads a row (a multiple of 32), E values of x and of
// dy each: lane l of the group's warp w holds the units 32 G w + l + 32 i, i <
// G, where a unit is a float4 (VEC: d % 4 == 0, 16-byte aligned rows) or a
// column; the distances are constants, so that a row's addresses cost little.
// SAVED: x from the checkpoint.  ACT: an activation.
//
// VEC: each thread copies its own values of the group's next kRing rows into
// shared memory (cp.async), waits for its own copies alone and refills the slot
// once it has used the values: no barrier is needed for the ring.  Eight values
// a thread (five registers each) leave room for 1024 threads on an SM, whose
// number, not the bytes in flight, hides the row's chain of loads, sums,
// shuffles and one barrier; what bounds it then is HBM.  Other rows are loaded
// into registers directly: copies of 4 bytes cost more than they hide.
template <int kBlock, int E, bool VEC, bool SAVED, bool ACT>
__global__ void __launch_bounds__(kBlock, 1024 / kBlock)
    norm_bwd_rows_kernel(const NormBwdParams p, const int T, const float inv_d, float* dg,
                         float* db) {
  constexpr int G = VEC ? E / 4 : E;  // copies of x (and of dy) a thread
  constexpr int C = E / G;            // columns of a copy
  __shared__ float red[2][kBlock / 32][2];
  extern __shared__ float4 ring4[];   // the ring, then reused for the CTA's sums
  const int R = kBlock / T;           // rows a CTA works on
  const int grp = threadIdx.x / T, t = threadIdx.x - grp * T;
  const int units = VEC ? p.d >> 2 : p.d;
  const int k0 = (t >> 5) * (32 * G) + (t & 31);  // this thread's first unit
  const int rem = units - k0;                     // its unit i exists if 32 i < rem
  const bool sums = p.part || dg || db;
  // a slot: x, then dy, both on 16-byte boundaries
  const int xbytes = ((SAVED ? units * 4 : units * C * 4) + 15) & ~15;
  const int row_bytes = xbytes + ((units * C * 4 + 15) & ~15);
  const uint32_t slot0 = smem_u32(ring4) + (uint32_t)(grp * kRing * row_bytes);
  constexpr bool kKeep = VEC && !ACT;  // the weight stays in registers
  float ag[E], ab[E], gw[kKeep ? E : 1];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    ag[i] = ab[i] = 0.0f;
    if (kKeep) gw[i] = 1.0f;
  }
  griddep_wait();
  griddep_launch_dependents();
  if (kKeep && p.g) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (32 * (i / C) < rem) gw[i] = __ldg(p.g + C * (k0 + 32 * (i / C)) + i % C);
    }
  }
  // rows and leading dimensions fit 32 bits (checked by the host), so that a
  // row's address is one multiply-add
  const int rows = (int)p.rows, step = (int)gridDim.x * R;
  const int ldx = (int)p.ldx, ldq = (int)p.ldq, lds = (int)p.lds, lddy = (int)p.lddy,
            lddx = (int)p.lddx;
  auto fetch = [&](int r, int s) {
    if (r < rows) {
      const uint32_t xs = slot0 + (uint32_t)(s * row_bytes + (SAVED ? 4 : 16) * k0);
      const uint32_t ys = slot0 + (uint32_t)(s * row_bytes + xbytes + 16 * k0);
      const char* xr = SAVED ? reinterpret_cast<const char*>(p.q + (int64_t)r * ldq + 4 * k0)
                             : reinterpret_cast<const char*>(p.x + (int64_t)r * ldx + 4 * k0);
      const char* yr = reinterpret_cast<const char*>(p.dy + (int64_t)r * lddy + 4 * k0);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        if (32 * i < rem) {
          if (SAVED) cp_async_4(xs + 128 * i, xr + 128 * i);
          else cp_async_16_cg(xs + 512 * i, xr + 512 * i);
          cp_async_16_cg(ys + 512 * i, yr + 512 * i);
        }
      }
    }
    cp_async_commit();  // (an empty group behind the last row)
  };
  int r = grp < R ? (int)blockIdx.x * R + grp : rows;
  if (VEC)
    for (int s = 0; s < kRing; ++s) fetch(r + s * step, s);
  float mean = 0.0f, rstd = 0.0f;
  if (r < rows) {
    mean = __ldg(p.mean + r);
    rstd = __ldg(p.rstd + r);
  }
  int slot = 0, phase = 0;
  for (; r < rows; r += step, phase ^= 1) {
    // the next row's statistics and this row's block scales
    const int rn = r + step < rows ? r + step : r;
    const float mean_n = __ldg(p.mean + rn), rstd_n = __ldg(p.rstd + rn);
    uint32_t sb[VEC ? G : 1];
    if (SAVED && VEC) {
      const uint8_t* sr = p.scale + (int64_t)r * lds + (t >> 5) * G;  // one byte for 32 units
#pragma unroll
      for (int i = 0; i < G; ++i) sb[i] = 32 * i < rem ? __ldg(sr + i) : 0u;
    }
    float u[E], h[E];  // x, then u; dy, then h
    if (VEC) {
      cp_async_wait<kRing - 1>();  // this slot's copies, the oldest group, have landed
      const uint32_t xs = slot0 + (uint32_t)(slot * row_bytes + (SAVED ? 4 : 16) * k0);
      const uint32_t ys = slot0 + (uint32_t)(slot * row_bytes + xbytes + 16 * k0);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        float4 a = make_float4(mean, mean, mean, mean), g = make_float4(0.f, 0.f, 0.f, 0.f);
        if (32 * i < rem) {
          if (SAVED) {
            a = e4m3x4_to_float4(__float_as_uint(lds32(xs + 128 * i)));
            const float s = e8m0_to_float(sb[i]);
            a.x *= s; a.y *= s; a.z *= s; a.w *= s;
          } else {
            a = lds128(xs + 512 * i);
          }
          g = lds128(ys + 512 * i);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
          u[C * i + c] = (&a.x)[c];
          h[C * i + c] = (&g.x)[c];
        }
      }
    } else {
      const float* yr = p.dy + (int64_t)r * lddy + k0;
      const float* xr = p.x + (int64_t)r * ldx + k0;
      const uint8_t* qr = p.q + (int64_t)r * ldq + k0;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        u[i] = mean;
        h[i] = 0.0f;
        uint32_t code = 0, byte = 0;
        if (32 * i < rem) {
          if (SAVED) {
            code = __ldcs(qr + 32 * i);
            byte = __ldg(p.scale + (int64_t)r * lds + (k0 + 32 * i) / kFp8Block);
          } else {
            u[i] = __ldcs(xr + 32 * i);
          }
          h[i] = __ldcs(yr + 32 * i);
        }
        if (SAVED && 32 * i < rem) u[i] = e4m3x2_to_float2(code).x * e8m0_to_float(byte);
      }
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      u[i] = (u[i] - mean) * rstd;
      const int j = C * (k0 + 32 * (i / C)) + i % C;
      float gv = 1.0f;
      if (kKeep) gv = gw[i];
      else if (p.g && 32 * (i / C) < rem) gv = __ldg(p.g + j);
      if (ACT) {
        const float bv = p.b && 32 * (i / C) < rem ? __ldg(p.b + j) : 0.0f;
        h[i] *= act_slope(fmaf(u[i], gv, bv), p.act);
      }
      ag[i] = fmaf(h[i], u[i], ag[i]);
      ab[i] += h[i];
      h[i] *= gv;
      s1 += h[i];
      s2 = fmaf(h[i], u[i], s2);
    }
    if (VEC) {
      fetch(r + kRing * step, slot);  // every value of the slot is in registers
      if (++slot == kRing) slot = 0;
    }
    if (p.dx) {
      // Both sums at once: the half-warps exchange, then lanes 0..15 add up the
      // first sum and lanes 16..31 the second.
      const bool second = t & 16;
      float v = second ? s2 : s1;
      v += __shfl_xor_sync(0xffffffffu, second ? s1 : s2, 16);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (T > 32) {
        // two buffers, so that one barrier a row is enough; every warp adds the
        // warps' sums for itself, in the same order
        const int nw = T >> 5, w0 = grp * nw, l = t & 15;
        if (l == 0) red[phase][w0 + (t >> 5)][second] = v;
        named_bar_sync(1 + grp, T);
        v = l < nw ? red[phase][w0 + l][second] : 0.0f;
        if (kBlock > 512 && l + 16 < nw) v += red[phase][w0 + 16 + l][second];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      }
      s1 = __shfl_sync(0xffffffffu, v, 0);
      s2 = __shfl_sync(0xffffffffu, v, 16);
      const float m1 = s1 * inv_d, m2 = s2 * inv_d;
      float* dxr = p.dx + (int64_t)r * lddx + C * k0;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        if (32 * i >= rem) continue;
        float4 w;
#pragma unroll
        for (int c = 0; c < C; ++c)
          (&w.x)[c] = rstd * fmaf(-u[C * i + c], m2, h[C * i + c] - m1);
        if (VEC) {
          float4* o = reinterpret_cast<float4*>(dxr) + 32 * i;
          if (p.accumulate) {
            const float4 q = *o;
            w.x += q.x; w.y += q.y; w.z += q.z; w.w += q.w;
          }
          __stcs(o, w);
        } else {
          put(dxr + 32 * i, w.x, p.accumulate);
        }
      }
    }
    mean = mean_n;
    rstd = rstd_n;
  }
  cp_async_wait<0>();
  if (!sums) return;
  // the CTA's sums over its groups, in group order, where the ring was
  float* acc_s = reinterpret_cast<float*>(ring4);
  __syncthreads();
  for (int gi = 0; gi < R; ++gi) {
    if (grp == gi) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (32 * (i / C) >= rem) continue;
        const int j = C * (k0 + 32 * (i / C)) + i % C;
        put(acc_s + j, ag[i], gi > 0);
        put(acc_s + p.d + j, ab[i], gi > 0);
      }
    }
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

// Rows of 8193 to 16384 columns: 1024 threads with 16 values each, loaded
// straight into registers; the sums for dg and db, for which 64 registers a
// thread leave no room, in shared memory.
template <int T, int E, bool VEC, bool SAVED>
__global__ void __launch_bounds__(T > 256 ? T : 256, T > 512 ? 1 : (T > 256 ? 1 : 2))
    norm_bwd_direct_kernel(const NormBwdParams p, float* dg, float* db) {
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
// one): 8 columns per CTA (one 32-byte sector of a row), 32 threads a column
// with 8 rows in flight each, added in a fixed order.
__global__ void __launch_bounds__(kThreads) norm_bwd_reduce_kernel(const float* __restrict__ part,
                                                                   int ctas, int d, float* dg,
                                                                   float* db, int accumulate) {
  __shared__ float t[32][9];
  griddep_wait();
  griddep_launch_dependents();
  float* out = blockIdx.y ? db : dg;
  if (!out) return;
  const int col = threadIdx.x & 7, w = threadIdx.x >> 3;
  const int j = blockIdx.x * 8 + col;
  float s = 0.0f;
  if (j < d) {
    const float* p = part + (int64_t)blockIdx.y * d + j;
    for (int c0 = w; c0 < ctas; c0 += 256) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = c0 + 32 * i < ctas ? __ldg(p + (int64_t)(c0 + 32 * i) * 2 * d) : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  }
  t[w][col] = s;
  __syncthreads();
  if (w == 0 && j < d) {
#pragma unroll
    for (int k = 1; k < 32; ++k) s += t[k][col];
    out[j] = accumulate ? out[j] + s : s;
  }
}

// The sums' way out: a partial row for each CTA and the second kernel, or the
// only CTA's own stores.
template <typename Launch>
int launch_with_sums(NormBwdParams& p, int grid, float* dg, float* db, cudaStream_t s,
                     const Launch& launch) {
  float* part = nullptr;
  if (grid > 1 && (dg || db)) {
    const int st = ws_alloc(nullptr, (void**)&part, (size_t)grid * 2 * p.d * sizeof(float), s);
    if (st) return st;
  }
  p.part = part;
  clear_stale_cuda_error();
  cudaError_t e = launch();
  if (e == cudaSuccess && part)
    e = launch_pdl(norm_bwd_reduce_kernel, dim3((unsigned)((p.d + 7) / 8), 2), dim3(kThreads), 0,
                   s, (const float*)part, grid, p.d, dg, db, p.accumulate);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(part, s);
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "layer_norm_backward launch");
}

template <int T, int E, bool VEC, bool SAVED>
int launch_direct(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  constexpr int kBlock = T > 256 ? T : 256;
  constexpr int R = kBlock / T;
  auto* k = norm_bwd_direct_kernel<T, E, VEC, SAVED>;
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
  return launch_with_sums(p, grid, dg, db, s, [&] {
    return launch_pdl(k, dim3((unsigned)grid), dim3(kBlock), smem, s, (const NormBwdParams)p, dg,
                      db);
  });
}

template <int kBlock, int E, bool VEC, bool SAVED, bool ACT>
int launch_rows(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  constexpr int G = VEC ? E / 4 : E;
  constexpr int kPerSm = 1024 / kBlock;
  auto* k = norm_bwd_rows_kernel<kBlock, E, VEC, SAVED, ACT>;
  const int units = VEC ? p.d / 4 : p.d;
  const int T = (units + 32 * G - 1) / (32 * G) * 32, R = kBlock / T;
  const int row_bytes = (((SAVED ? p.d : 4 * p.d) + 15) & ~15) + ((4 * p.d + 15) & ~15);
  int smem = VEC ? R * kRing * row_bytes : 0;
  if (smem < 8 * p.d) smem = 8 * p.d;  // the CTA's sums
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cuda_status(e, "layer_norm_backward smem attribute");
  const int64_t need = (p.rows + R - 1) / R, cap = (int64_t)ctx->sm_count * kPerSm;
  const int grid = (int)(need < cap ? need : cap);
  return launch_with_sums(p, grid, dg, db, s, [&] {
    return launch_pdl(k, dim3((unsigned)grid), dim3(kBlock), (size_t)smem, s,
                      (const NormBwdParams)p, T, 1.0f / (float)p.d, dg, db);
  });
}

template <bool VEC, bool SAVED>
int launch_width(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  const bool act = p.act != RTB_ACT_NONE;
  if (p.d <= 128)
    return act ? launch_rows<512, 4, VEC, SAVED, true>(ctx, p, dg, db, s)
               : launch_rows<512, 4, VEC, SAVED, false>(ctx, p, dg, db, s);
  if (p.d <= 4096)
    return act ? launch_rows<512, 8, VEC, SAVED, true>(ctx, p, dg, db, s)
               : launch_rows<512, 8, VEC, SAVED, false>(ctx, p, dg, db, s);
  if (p.d <= 8192)
    return act ? launch_rows<1024, 8, VEC, SAVED, true>(ctx, p, dg, db, s)
               : launch_rows<1024, 8, VEC, SAVED, false>(ctx, p, dg, db, s);
  return launch_direct<1024, 16, VEC, SAVED>(ctx, p, dg, db, s);
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
  // (the row kernels index rows and rows' addresses with 32-bit factors)
  constexpr int64_t kMax32 = INT32_MAX - (1 << 20);
  if (d.d <= 16384 && d.rows <= kMax32 && d.ldx <= kMax32 && d.ldq <= kMax32 && d.lds <= kMax32 &&
      d.lddy <= kMax32 && d.lddx <= kMax32) {
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
    e = launch_pdl(norm_bwd_reduce_kernel, dim3((unsigned)((d.d + 7) / 8), 2), dim3(kThreads), 0,
                   s, (const float*)part, grid, (int)d.d, d.dg, d.db, d.accumulate);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(part, s);
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "layer_norm_backward launch");
}

}  // namespace rtb
