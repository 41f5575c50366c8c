// LayerNorm backward over the last dimension (with the fused activation of
// rtb_layer_norm).  With u_j = (x_j - mean) rstd, z = u g + b and dz = dy
// act'(z):
//   dg = sum_rows dz u,  db = sum_rows dz
//   dx = rstd (h - mean_j(h) - u mean_j(h u)),  h = dz g
// x is fp32 or an 8-bit checkpoint (rtb_fp8.cuh); mean and rstd are the
// forward pass's.
// RMS (rtb_rms.cu's backward pass): no mean, no bias, no activation, and the
// gradient that reaches x from elsewhere (the residual stream) is added:
//   u = x rstd,  dx = rstd (h - u mean_j(h u)) + dsum,  h = dy g,  dg = sum_rows dy u
// HBM-bound: x and dy are read and dx written once (12 bytes an element, 9 from a
// checkpoint; 4 more for dsum).
//
// A row belongs to a group of threads that holds it in registers, rows strided
// over the groups of the resident CTAs; one reduction of two sums a row.  dg and
// db are sums over rows, one column always with the same thread: running sums in
// registers (in shared memory for rows beyond 8192 columns, where 1024 threads
// leave 64 registers each), added up over a CTA's groups in group order, left in
// a row of a [CTA][2][d] workspace, and the CTAs' rows are added by a second
// kernel.  No atomics: the order depends on the sizes, the alignment (which kernel)
// and the device (how many CTAs) alone.  A single CTA writes
// its sums itself.  Rows beyond 16384 columns take a CTA each and two passes.
//
// Measured: 8192 x 4096 75 us (5.4 TB/s of the 12 bytes an element, 82% of a copy),
// 16384 x 2048 from a checkpoint 67 us (4.5 TB/s of 9 bytes: the instructions of
// the row's fixed part count as much), 2048 x 16384 102 us, 8192 x 4097 130 us;
// 8192 x 4096 with sigmoid 99 us, with tanh 101.  RMS, 8192 x 4096: 73 us, with dsum 90
// (6.0 TB/s), from a checkpoint 74 and 83; 16384 x 2048 from one 68; 2048 x 16384 with dsum
// 112, 8192 x 4097 154; 1531 x 1001 from a checkpoint 12.5; 600 x 40000, the kernel of any
// width, with dsum 579.
#include "rtb_act.cuh"
#include "rtb_f32x2.cuh"
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
  const float* dsum;  // RMS: added to dx; or null
  int64_t ldds;
  float* dx;
  int64_t lddx;
  float* part;  // [CTA][2][d] partial dg, db; null when neither is wanted
  int accumulate;
};

// e / (1 + e)^2 of two values in [0, 1], as e / (1 + e (2 + e)), which rounds less.
// The reciprocal is the instruction's own (1 ulp; with correctly rounded quotients
// 8192 x 4096 takes 112 us for sigmoid and not 99).
__device__ __forceinline__ unsigned long long bell2(float e0, float e1) {
  const unsigned long long e = pack2(e0, e1);
  const float2 d = unpack2(fma2(e, add2(e, pack2(2.0f, 2.0f)), pack2(1.0f, 1.0f)));
  float r0, r1;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(d.y));
  return mul2(e, pack2(r0, r1));
}
// act'(z) as a function of z, of two values; ReLU's derivative is 0 at 0 and for
// NaN, as its forward maps both to 0.  With e = exp(-|z|) sigmoid's is e / (1 +
// e)^2 and, with e = exp(-2 |z|), tanh's 4 e / (1 + e)^2: no difference of values
// near 1, so that a few ulp hold where the activation is saturated too.
__device__ __forceinline__ unsigned long long act_slope2(float2 z, int act) {
  if (act == RTB_ACT_RELU) return pack2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
  if (act == RTB_ACT_SIGMOID) return bell2(expf(-fabsf(z.x)), expf(-fabsf(z.y)));
  if (act == RTB_ACT_TANH)
    return mul2(bell2(expf(-2.0f * fabsf(z.x)), expf(-2.0f * fabsf(z.y))), pack2(4.0f, 4.0f));
  return pack2(1.0f, 1.0f);
}
__device__ __forceinline__ float act_slope(float z, int act) {
  return unpack2(act_slope2(make_float2(z, z), act)).x;
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

// Any width and alignment: two passes over the row's columns, the second out of L1 or
// L2.  bias: the sums for db are wanted too.
__global__ void __launch_bounds__(kThreads) norm_bwd_kernel(const NormBwdParams p, const int bias) {
  __shared__ float red[kThreads / 32][2];
  griddep_wait();
  griddep_launch_dependents();
  float* pg = p.part ? p.part + (int64_t)blockIdx.x * 2 * p.d : nullptr;
  float* pb = pg && bias ? pg + p.d : nullptr;  // (an index p.d + j would pass 32 bits)
  bool first = true;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, first = false) {
    const float mean = p.mean ? p.mean[r] : 0.0f, rstd = p.rstd[r];  // (RMS: no mean)
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
        if (pb) pb[j] = first ? dz : pb[j] + dz;
      }
    }
    if (!p.dx) continue;
    const float2 t = block_sum2(s1, s2, red);
    const float m1 = p.mean ? t.x / p.d : 0.0f, m2 = t.y / p.d;
    float* dxr = p.dx + r * p.lddx;
    const float* dsr = p.dsum ? p.dsum + r * p.ldds : nullptr;
    for (int j = threadIdx.x; j < p.d; j += kThreads) {
      float u, dz, h;
      at(j, u, dz, h);
      float v = rstd * (h - m1 - u * m2);
      if (dsr) v += dsr[j];
      dxr[j] = p.accumulate ? dxr[j] + v : v;
    }
  }
}

// out (+)= v
__device__ __forceinline__ void put(float* out, float v, int accumulate) {
  *out = accumulate ? *out + v : v;
}

constexpr int kRing = 3;  // stages of the row ring: 96 KB for 512 threads of 8 values

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts_u8(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// A row of `bytes` bytes at any address into shared memory, at the same offset
// from a 16-byte boundary: T threads take its 16-byte chunks (N each at most) in
// turn.  Chunks that reach over [lo, hi), the tensor, go byte by byte.
template <int N>
__device__ __forceinline__ void copy_row(uint32_t dst, const void* row, int bytes, const void* lo,
                                         const void* hi, int t, int T) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(row), a0 = a & ~uintptr_t(15);
  const uintptr_t l = reinterpret_cast<uintptr_t>(lo), h = reinterpret_cast<uintptr_t>(hi);
  const int chunks = ((int)(a - a0) + bytes + 15) >> 4;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = t + i * T;
    if (c >= chunks) continue;
    const uintptr_t g = a0 + 16 * c;
    if (g >= l && g + 16 <= h) {
      cp_async_16_cg(dst + 16 * c, reinterpret_cast<const void*>(g));
    } else {
#pragma unroll 1
      for (int b = 0; b < 16; ++b)
        if (g + b >= l && g + b < h)
          sts_u8(dst + 16 * c + b, *reinterpret_cast<const uint8_t*>(g + b));
    }
  }
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
// shuffles and one barrier.  The arithmetic is packed, two values an
// instruction; FULL: every thread has all of its units, and nothing asks (8192 x
// 4096 78 -> 75 us, from a checkpoint 84 -> 71, 4096 x 8192 83 -> 74 by both).
//
// Rows off the 16-byte boundaries: the threads copy the row's aligned chunks for
// one another, and the barrier of a row's sums also publishes the next row (from
// a checkpoint 8192 x 4097: 349 us by direct loads, 160 here; 65536 x 301: 167,
// 102; fp32 x 8192 x 4097, one group on an SM: 133, 129).  fp32 rows of up to 4096
// columns are loaded into registers directly: with more groups on an SM the
// copies cost more than they hide (65536 x 301: 62 us, 87 by copies; 1531 x 1001
// with tanh 13.2, 15.6).
template <int kBlock, bool VEC, bool SAVED>
constexpr bool kRows = VEC || SAVED || kBlock > 512;  // rows through the ring

template <int kBlock, int E, bool VEC, bool SAVED, bool ACT, bool FULL, bool RMS>
__global__ void __launch_bounds__(kBlock, 1024 / kBlock)
    norm_bwd_rows_kernel(const NormBwdParams p, const int T, const float inv_d, float* dg,
                         float* db) {
  constexpr int G = VEC ? E / 4 : E;  // copies of x (and of dy) a thread
  constexpr int C = E / G;            // columns of a copy
  constexpr int P = E / 2;            // pairs of values
  constexpr bool RING = kRows<kBlock, VEC, SAVED>, SHARED = RING && !VEC;
  constexpr bool kAhead = SAVED && (kBlock > 512 || !VEC);  // block scales a row ahead
  __shared__ float red[2][kBlock / 32][2];
  extern __shared__ float4 ring4[];   // the ring, then reused for the CTA's sums
  const int R = kBlock / T;           // rows a CTA works on
  const int grp = threadIdx.x / T, t = threadIdx.x - grp * T;
  const int units = VEC ? p.d >> 2 : p.d;
  const int k0 = (t >> 5) * (32 * G) + (t & 31);  // this thread's first unit
  const int rem = FULL ? 32 * G : units - k0;     // its unit i exists if 32 i < rem
  const bool sums = p.part || dg || db;
  // a slot: x, then dy, both on 16-byte boundaries
  const int xrow = SAVED ? units * C : units * C * 4, yrow = units * C * 4;  // bytes of a row
  const int xbytes = (xrow + (VEC ? 15 : 30)) & ~15;
  const int row_bytes = xbytes + ((yrow + (VEC ? 15 : 30)) & ~15);
  const uint32_t slot0 = smem_u32(ring4) + (uint32_t)(grp * kRing * row_bytes);
  constexpr bool kKeep = VEC && !ACT;  // the weight stays in registers
  unsigned long long ag[P], ab[RMS ? 1 : P], gw[kKeep ? P : 1];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    ag[i] = ab[RMS ? 0 : i] = 0ull;
    if (kKeep) gw[i] = pack2(1.0f, 1.0f);
  }
  // the pair of a column vector's values that belongs to values 2 i, 2 i + 1
  auto columns = [&](const float* v, int i, float none) {
    const bool in0 = 32 * (2 * i / C) < rem, in1 = 32 * ((2 * i + 1) / C) < rem;
    return pack2(v && in0 ? __ldg(v + C * (k0 + 32 * (2 * i / C)) + 2 * i % C) : none,
                 v && in1 ? __ldg(v + C * (k0 + 32 * ((2 * i + 1) / C)) + (2 * i + 1) % C) : none);
  };
  griddep_wait();
  griddep_launch_dependents();
  if (kKeep && p.g) {
#pragma unroll
    for (int i = 0; i < P; ++i) gw[i] = columns(p.g, i, 1.0f);
  }
  // rows and leading dimensions fit 32 bits (checked by the host), so that a
  // row's address is one multiply-add
  const int rows = (int)p.rows, step = (int)gridDim.x * R;
  const int ldx = (int)p.ldx, ldq = (int)p.ldq, lds = (int)p.lds, lddy = (int)p.lddy,
            lddx = (int)p.lddx, ldds = (int)p.ldds;
  auto xrow_at = [&](int r) {
    return SAVED ? reinterpret_cast<const char*>(p.q + (int64_t)r * ldq)
                 : reinterpret_cast<const char*>(p.x + (int64_t)r * ldx);
  };
  auto yrow_at = [&](int r) { return reinterpret_cast<const char*>(p.dy + (int64_t)r * lddy); };
  auto fetch = [&](int r, int s) {
    if (r < rows) {
      if (VEC) {
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
      } else {
        const uint32_t xs = slot0 + (uint32_t)(s * row_bytes), ys = xs + (uint32_t)xbytes;
        const char *xr = xrow_at(r), *yr = yrow_at(r);
        copy_row<SAVED ? 1 : E / 4 + 1>(xs, xr, xrow, xrow_at(0), xrow_at(rows - 1) + xrow, t, T);
        copy_row<E / 4 + 1>(ys, yr, yrow, yrow_at(0), yrow_at(rows - 1) + yrow, t, T);
      }
    }
    cp_async_commit();  // (an empty group behind the last row)
  };
  int r = grp < R ? (int)blockIdx.x * R + grp : rows;
  if (RING)
    for (int s = 0; s < kRing; ++s) fetch(r + s * step, s);
  // a thread's block scales of a row
  constexpr int NS = !SAVED ? 1 : VEC ? G : G / 4;
  auto scales = [&](int r, uint32_t (&sb)[NS]) {
    const uint8_t* sr = p.scale + (int64_t)r * lds + (t >> 5) * NS;
#pragma unroll
    for (int i = 0; i < NS; ++i) sb[i] = SAVED && (VEC ? 32 : 128) * i < rem ? __ldg(sr + i) : 0u;
  };
  float mean = 0.0f, rstd = 0.0f;
  uint32_t sb[NS] = {};
  if (r < rows) {
    if (!RMS) mean = __ldg(p.mean + r);
    rstd = __ldg(p.rstd + r);
    if (kAhead) scales(r, sb);
    if (SHARED) {
      cp_async_wait<kRing - 1>();
      if (T > 32) named_bar_sync(1 + grp, T);
      else __syncwarp();
    }
  }
  int slot = 0, phase = 0;
  for (; r < rows; r += step, phase ^= 1) {
    // the next row's statistics and block scales
    const int rn = r + step < rows ? r + step : r;
    // (its dsum, which no ring takes, into L2 at least: 8192 x 4097 170 -> 153 us, from a
    // checkpoint x 4096 90 -> 83; rows without a ring, 65536 x 301, 64.5 -> 70.7)
    if (RING && RMS && p.dsum && p.dx && 32 * t < p.d) prefetch_l2(p.dsum + (int64_t)rn * ldds + 32 * t);
    const float mean_n = RMS ? 0.0f : __ldg(p.mean + rn), rstd_n = __ldg(p.rstd + rn);
    uint32_t sb_n[NS] = {};
    if (kAhead) scales(rn, sb_n);
    else if (SAVED) scales(r, sb);
    unsigned long long u[P], h[P];  // x, then u; dy, then h
    if (VEC) {
      cp_async_wait<kRing - 1>();  // this slot's copies, the oldest group, have landed
      const uint32_t xs = slot0 + (uint32_t)(slot * row_bytes + (SAVED ? 4 : 16) * k0);
      const uint32_t ys = slot0 + (uint32_t)(slot * row_bytes + xbytes + 16 * k0);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        float4 a = make_float4(mean, mean, mean, mean), g = make_float4(0.f, 0.f, 0.f, 0.f);
        if (32 * i < rem) {
          if (SAVED) a = e4m3x4_to_float4(__float_as_uint(lds32(xs + 128 * i)));
          else a = lds128(xs + 512 * i);
          g = lds128(ys + 512 * i);
        }
        u[2 * i] = pack2(a.x, a.y);
        u[2 * i + 1] = pack2(a.z, a.w);
        if (SAVED && 32 * i < rem) {
          const float s = e8m0_to_float(sb[i]);
          u[2 * i] = mul2(u[2 * i], pack2(s, s));
          u[2 * i + 1] = mul2(u[2 * i + 1], pack2(s, s));
        }
        h[2 * i] = pack2(g.x, g.y);
        h[2 * i + 1] = pack2(g.z, g.w);
      }
    } else {
      const float* xr = p.x + (int64_t)r * ldx + k0;
      const float* yr = p.dy + (int64_t)r * lddy + k0;
      uint32_t xs = 0, ys = 0;
      if (SHARED) {
        xs = slot0 + (uint32_t)(slot * row_bytes) + (SAVED ? 1 : 4) * k0;
        ys = slot0 + (uint32_t)(slot * row_bytes + xbytes) + 4 * k0;
        xs += (uint32_t)(reinterpret_cast<uintptr_t>(xrow_at(r)) & 15u);
        ys += (uint32_t)(reinterpret_cast<uintptr_t>(yrow_at(r)) & 15u);
      }
      float a[E], g[E];
#pragma unroll
      for (int i = 0; i < G; ++i) {
        a[i] = mean;
        g[i] = 0.0f;
        if (32 * i < rem) {
          if (SAVED) a[i] = e4m3x2_to_float2(lds_u8(xs + 32 * i)).x * e8m0_to_float(sb[i / 4 % NS]);
          else a[i] = SHARED ? lds32(xs + 128 * i) : __ldcs(xr + 32 * i);
          g[i] = SHARED ? lds32(ys + 128 * i) : __ldcs(yr + 32 * i);
        }
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        u[i] = pack2(a[2 * i], a[2 * i + 1]);
        h[i] = pack2(g[2 * i], g[2 * i + 1]);
      }
    }
    // (RMS: the registers that the bias's sums have otherwise; loaded here, so that
    // the row's sums hide the latency)
    unsigned long long ds[RMS ? P : 1];
    if (RMS) {
      const float* dsr = p.dsum + (int64_t)r * ldds + C * k0;
#pragma unroll
      for (int i = 0; i < P; ++i) ds[RMS ? i : 0] = 0ull;
      if (p.dsum && p.dx) {
#pragma unroll
        for (int i = 0; i < G; i += VEC ? 1 : 2) {
          if (VEC) {
            if (32 * i < rem) {
              const float4 f = __ldcs(reinterpret_cast<const float4*>(dsr) + 32 * i);
              ds[RMS ? 2 * i : 0] = pack2(f.x, f.y);
              ds[RMS ? 2 * i + 1 : 0] = pack2(f.z, f.w);
            }
          } else {
            ds[RMS ? i / 2 : 0] = pack2(32 * i < rem ? __ldcs(dsr + 32 * i) : 0.0f,
                                        32 * (i + 1) < rem ? __ldcs(dsr + 32 * (i + 1)) : 0.0f);
          }
        }
      }
    }
    unsigned long long t1 = 0ull, t2 = 0ull;
    const unsigned long long rs = pack2(rstd, rstd), nm = pack2(-mean, -mean);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      u[i] = RMS ? mul2(u[i], rs) : mul2(add2(u[i], nm), rs);
      const unsigned long long gv = kKeep ? gw[kKeep ? i : 0] : columns(p.g, i, 1.0f);
      if (ACT) {
        const float2 z = unpack2(fma2(u[i], gv, columns(p.b, i, 0.0f)));
        h[i] = mul2(h[i], act_slope2(z, p.act));
      }
      ag[i] = fma2(h[i], u[i], ag[i]);
      if (!RMS) ab[RMS ? 0 : i] = add2(ab[RMS ? 0 : i], h[i]);
      h[i] = mul2(h[i], gv);
      if (!RMS) t1 = add2(t1, h[i]);
      t2 = fma2(h[i], u[i], t2);
    }
    float s1 = unpack2(t1).x + unpack2(t1).y, s2 = unpack2(t2).x + unpack2(t2).y;
    auto refill = [&] {
      fetch(r + kRing * step, slot);
      if (++slot == kRing) slot = 0;
    };
    if (VEC) refill();  // every value of the slot is in registers
    if (p.dx || SHARED) {
      // Both sums at once: the half-warps exchange, then lanes 0..15 add up the
      // first sum and lanes 16..31 the second.
      const bool second = t & 16;
      float v = second ? s2 : s1;
      v += __shfl_xor_sync(0xffffffffu, second ? s1 : s2, 16);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (SHARED) cp_async_wait<kRing - 2>();  // this thread's copies of the next row
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
      } else if (SHARED) {
        __syncwarp();
      }
      if (SHARED) refill();  // every thread of the group has used the slot
      s1 = __shfl_sync(0xffffffffu, v, 0);
      s2 = __shfl_sync(0xffffffffu, v, 16);
      const unsigned long long m1 = pack2(-s1 * inv_d, -s1 * inv_d), m2 = pack2(-s2 * inv_d, -s2 * inv_d);
      float* dxr = p.dx + (int64_t)r * lddx + C * k0;
#pragma unroll
      for (int i = 0; i < P; ++i)
        u[i] = RMS ? fma2(rs, fma2(u[i], m2, h[i]), ds[RMS ? i : 0])
                   : mul2(rs, fma2(u[i], m2, add2(h[i], m1)));
      if (SHARED && !p.dx) {
        // (only the sums were asked for)
      } else if (VEC) {
        float4* o = reinterpret_cast<float4*>(dxr);
        if (p.accumulate) {
#pragma unroll
          for (int i = 0; i < G; ++i) {
            if (32 * i >= rem) continue;
            const float4 q = o[32 * i];
            u[2 * i] = add2(pack2(q.x, q.y), u[2 * i]);
            u[2 * i + 1] = add2(pack2(q.z, q.w), u[2 * i + 1]);
          }
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float2 a = unpack2(u[2 * i]), b = unpack2(u[2 * i + 1]);
          if (32 * i < rem) __stcs(o + 32 * i, make_float4(a.x, a.y, b.x, b.y));
        }
      } else {
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float2 a = unpack2(u[i / 2]);
          if (32 * i < rem) put(dxr + 32 * i, i % 2 ? a.y : a.x, p.accumulate);
        }
      }
    }
    mean = mean_n;
    rstd = rstd_n;
#pragma unroll
    for (int i = 0; i < (kAhead ? NS : 0); ++i) sb[i] = sb_n[i];
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
        const float2 a = unpack2(ag[i / 2]), b = unpack2(ab[RMS ? 0 : i / 2]);
        put(acc_s + j, i % 2 ? a.y : a.x, gi > 0);
        if (!RMS) put(acc_s + p.d + j, i % 2 ? b.y : b.x, gi > 0);
      }
    }
    __syncthreads();
  }
  for (int j = threadIdx.x; j < p.d; j += kBlock) {
    if (p.part) {
      float* pr = p.part + (int64_t)blockIdx.x * 2 * p.d;
      pr[j] = acc_s[j];
      if (!RMS) pr[p.d + j] = acc_s[p.d + j];
    } else {
      if (dg) put(dg + j, acc_s[j], p.accumulate);
      if (!RMS && db) put(db + j, acc_s[p.d + j], p.accumulate);
    }
  }
}

// Rows of 8193 to 16384 columns: a CTA of 1024 threads with 16 values each, loaded
// straight into registers; the sums for dg and db, for which 64 registers a
// thread leave no room, in shared memory.
constexpr int kWide = 1024;

template <bool VEC, bool SAVED, bool RMS>
__global__ void __launch_bounds__(kWide, 1)
    norm_bwd_direct_kernel(const NormBwdParams p, float* dg, float* db) {
  constexpr int E = 16, G = VEC ? E / 4 : E;  // values, loads of x (and of dy) a thread
  constexpr int C = E / G;                    // columns of a load
  constexpr int W = kWide / 32;
  __shared__ float red[2][W][2];
  extern __shared__ float acc_s[];  // [2][d] (RMS [d]): the CTA's running sums
  griddep_wait();
  griddep_launch_dependents();
  const int t = threadIdx.x;
  const int units = VEC ? p.d >> 2 : p.d;
  const bool sums = p.part || dg || db;
  if (sums) {
    for (int j = t; j < (RMS ? 1 : 2) * p.d; j += kWide) acc_s[j] = 0.0f;
    __syncthreads();
  }
  int phase = 0;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, phase ^= 1) {
    float u[E], h[E];  // x, then u; dy, then h
    const float mean = RMS ? 0.0f : __ldg(p.mean + r), rstd = __ldg(p.rstd + r);
    const float* dyr = p.dy + r * p.lddy;
    // The next row into L2 (2048 x 16384 110 -> 102 us, RMS with dsum from a checkpoint 128 ->
    // 107).  fp32 rows off the 16-byte boundaries, whose single loads are many, do not gain
    // (2048 x 16383 163 -> 170) but by dsum, which is loaded last (229 -> 204).
    const int64_t rn = r + gridDim.x;
    if (rn < p.rows && 32 * t < p.d) {
      if (VEC || SAVED) {
        prefetch_l2(p.dy + rn * p.lddy + 32 * t);
        if (!SAVED) prefetch_l2(p.x + rn * p.ldx + 32 * t);
        else if (128 * t < p.d) prefetch_l2(p.q + rn * p.ldq + 128 * t);
      }
      if (RMS && p.dsum && p.dx) prefetch_l2(p.dsum + rn * p.ldds + 32 * t);
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = t + kWide * i;
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
      const int k = t + kWide * i;
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
      const bool add = sums && k < units;
      float4 sg, sb;
      if (add && VEC) {
        sg = reinterpret_cast<const float4*>(acc_s)[k];
        if (!RMS) sb = reinterpret_cast<const float4*>(acc_s + p.d)[k];
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = C * i + c;
        u[e] = (u[e] - mean) * rstd;
        float dz = h[e];
        if (p.act != RTB_ACT_NONE) dz *= act_slope(fmaf(u[e], gv[c], bv[c]), p.act);
        if (add && VEC) {
          (&sg.x)[c] = fmaf(dz, u[e], (&sg.x)[c]);
          if (!RMS) (&sb.x)[c] += dz;
        } else if (add) {
          acc_s[k] = fmaf(dz, u[e], acc_s[k]);
          if (!RMS) acc_s[p.d + k] += dz;
        }
        h[e] = dz * gv[c];
        s1 += h[e];
        s2 = fmaf(h[e], u[e], s2);
      }
      if (add && VEC) {
        reinterpret_cast<float4*>(acc_s)[k] = sg;
        if (!RMS) reinterpret_cast<float4*>(acc_s + p.d)[k] = sb;
      }
    }
    if (!p.dx) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    // two buffers, so that one barrier a row is enough
    if ((t & 31) == 0) {
      red[phase][t >> 5][0] = s1;
      red[phase][t >> 5][1] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      s1 += red[phase][k][0];
      s2 += red[phase][k][1];
    }
    const float m1 = RMS ? 0.0f : s1 / p.d, m2 = s2 / p.d;
    float* dxr = p.dx + r * p.lddx;
    const float* dsr = RMS && p.dsum ? p.dsum + r * p.ldds : nullptr;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int k = t + kWide * i;
      if (k >= units) continue;
      float v[C];
#pragma unroll
      for (int c = 0; c < C; ++c) v[c] = rstd * (h[C * i + c] - m1 - u[C * i + c] * m2);
      if (RMS && dsr) {
        float e[C];
        if (VEC) *reinterpret_cast<float4*>(e) = __ldcs(reinterpret_cast<const float4*>(dsr) + k);
        else e[0] = __ldcs(dsr + k);
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] += e[c];
      }
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
  __syncthreads();
  for (int j = t; j < p.d; j += kWide) {
    if (p.part) {
      float* pr = p.part + (int64_t)blockIdx.x * 2 * p.d;
      pr[j] = acc_s[j];
      if (!RMS) pr[p.d + j] = acc_s[p.d + j];
    } else {
      if (dg) put(dg + j, acc_s[j], p.accumulate);
      if (!RMS && db) put(db + j, acc_s[p.d + j], p.accumulate);
    }
  }
}

// dg[j] (+)= sum over the CTAs' partial rows, db likewise (blockIdx.y picks
// one): 32 columns per CTA, 32 threads a column with 8 rows in flight each, added
// in a fixed order.
constexpr int kReduceThreads = 1024;

__global__ void __launch_bounds__(kReduceThreads) norm_bwd_reduce_kernel(const float* __restrict__ part,
                                                                   int ctas, int d, float* dg,
                                                                   float* db, int accumulate) {
  __shared__ float t[32][33];
  griddep_wait();
  griddep_launch_dependents();
  float* out = blockIdx.y ? db : dg;
  if (!out) return;
  const int col = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + col;
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

// What an error is reported as, by the entry point (RMS: no mean).
int failed(const NormBwdParams& p, cudaError_t e) {
  return cuda_status(e, p.mean ? "layer_norm_backward launch" : "rms_norm_backward launch");
}

// The sums' way out: a partial row for each CTA and the second kernel, or the
// only CTA's own stores.
template <typename Launch>
int launch_with_sums(rtb_ctx* ctx, NormBwdParams& p, int grid, float* dg, float* db,
                     cudaStream_t s, const Launch& launch) {
  float* part = nullptr;
  if (grid > 1 && (dg || db)) {
    const int st = ws_alloc(ctx, (void**)&part, (size_t)grid * 2 * p.d * sizeof(float), s);
    if (st) return st;
  }
  p.part = part;
  clear_stale_cuda_error();
  cudaError_t e = launch();
  if (e == cudaSuccess && part)
    e = launch_pdl(norm_bwd_reduce_kernel, dim3((unsigned)((p.d + 31) / 32), db ? 2 : 1), dim3(kReduceThreads), 0,
                   s, (const float*)part, grid, p.d, dg, db, p.accumulate);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(part, s);
  return e == cudaSuccess ? RTB_OK : failed(p, e);
}

template <bool VEC, bool SAVED, bool RMS>
int launch_direct(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  auto* k = norm_bwd_direct_kernel<VEC, SAVED, RMS>;
  const size_t smem = (dg || db) ? (size_t)(RMS ? 1 : 2) * p.d * sizeof(float) : 0;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       2 * 16384 * (int)sizeof(float));
  if (e != cudaSuccess) return failed(p, e);
  const int grid = (int)(p.rows < ctx->sm_count ? p.rows : ctx->sm_count);
  return launch_with_sums(ctx, p, grid, dg, db, s, [&] {
    return launch_pdl(k, dim3((unsigned)grid), dim3(kWide), smem, s, (const NormBwdParams)p, dg, db);
  });
}

// RMS: rows that one CTA takes in so many rounds are one CTA's, which needs no workspace and
// no second kernel (two rounds, 16 x 512: 5.3 -> 4.6 us, 10.4 -> 6.3 with the host's time of
// the call; 8 x 1001 6.0 -> 5.4, 9.2 -> 6.1; 2 x 8192 7.1 both, 8.3 for 9.5; four rounds, 16
// x 1024: 5.1 -> 6.1, 4 x 8192 7.3 -> 10.9).  (Layer norm keeps its order of sums.)
constexpr int kAlone = 2;

template <int kBlock, int E, bool VEC, bool SAVED, bool ACT, bool FULL, bool RMS>
int launch_rows_as(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  constexpr int G = VEC ? E / 4 : E;
  constexpr int kPerSm = 1024 / kBlock;
  auto* k = norm_bwd_rows_kernel<kBlock, E, VEC, SAVED, ACT, FULL, RMS>;
  const int units = VEC ? p.d / 4 : p.d;
  const int T = (units + 32 * G - 1) / (32 * G) * 32, R = kBlock / T;
  constexpr int kPad = VEC ? 15 : 30;
  const int row_bytes = (((SAVED ? p.d : 4 * p.d) + kPad) & ~15) + ((4 * p.d + kPad) & ~15);
  int smem = kRows<kBlock, VEC, SAVED> ? R * kRing * row_bytes : 0;
  if (smem < (RMS ? 4 : 8) * p.d) smem = (RMS ? 4 : 8) * p.d;  // the CTA's sums
  // The limit belongs to the kernel and not to the launch, and another thread may
  // be between its own two: so it is one number, that of the widest launch.  Groups
  // of T threads hold at most E values a thread, R d <= kBlock E, and R is at most
  // kBlock / 32.
  constexpr int kRingMax = kRing * (kBlock * E * (SAVED ? 5 : 8) + kBlock / 32 * 2 * kPad);
  constexpr int kSumsMax = 8 * kBlock * E;
  constexpr int kMost = kRows<kBlock, VEC, SAVED> && kRingMax > kSumsMax ? kRingMax : kSumsMax;
  static_assert(kMost + 1024 <= 232448, "shared memory");
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  if (e != cudaSuccess) return failed(p, e);
  const int64_t need = (p.rows + R - 1) / R, cap = (int64_t)ctx->sm_count * kPerSm;
  const int grid = RMS && dg && need <= kAlone ? 1 : (int)(need < cap ? need : cap);
  return launch_with_sums(ctx, p, grid, dg, db, s, [&] {
    return launch_pdl(k, dim3((unsigned)grid), dim3(kBlock), (size_t)smem, s,
                      (const NormBwdParams)p, T, 1.0f / (float)p.d, dg, db);
  });
}

template <int kBlock, int E, bool VEC, bool SAVED, bool ACT, bool RMS = false>
int launch_rows(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  if (VEC && p.d % (32 * E) == 0)
    return launch_rows_as<kBlock, E, VEC, SAVED, ACT, VEC, RMS>(ctx, p, dg, db, s);
  return launch_rows_as<kBlock, E, VEC, SAVED, ACT, false, RMS>(ctx, p, dg, db, s);
}

template <bool VEC, bool SAVED>
int launch_width(rtb_ctx* ctx, NormBwdParams& p, float* dg, float* db, cudaStream_t s) {
  const bool act = p.act != RTB_ACT_NONE;
  if (!p.mean) {  // RMS
    if (p.d <= 128) return launch_rows<512, 4, VEC, SAVED, false, true>(ctx, p, dg, db, s);
    if (p.d <= 4096) return launch_rows<512, 8, VEC, SAVED, false, true>(ctx, p, dg, db, s);
    if (p.d <= 8192) return launch_rows<1024, 8, VEC, SAVED, false, true>(ctx, p, dg, db, s);
    return launch_direct<VEC, SAVED, true>(ctx, p, dg, db, s);
  }
  if (p.d <= 128)
    return act ? launch_rows<512, 4, VEC, SAVED, true>(ctx, p, dg, db, s)
               : launch_rows<512, 4, VEC, SAVED, false>(ctx, p, dg, db, s);
  if (p.d <= 4096)
    return act ? launch_rows<512, 8, VEC, SAVED, true>(ctx, p, dg, db, s)
               : launch_rows<512, 8, VEC, SAVED, false>(ctx, p, dg, db, s);
  if (p.d <= 8192)
    return act ? launch_rows<1024, 8, VEC, SAVED, true>(ctx, p, dg, db, s)
               : launch_rows<1024, 8, VEC, SAVED, false>(ctx, p, dg, db, s);
  return launch_direct<VEC, SAVED, false>(ctx, p, dg, db, s);
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
  p.dsum = d.dsum;
  p.ldds = d.ldds;
  p.dx = d.dx;
  p.lddx = d.lddx;
  p.accumulate = d.accumulate;
  // (the row kernels index rows and rows' addresses with 32-bit factors)
  constexpr int64_t kMax32 = INT32_MAX - (1 << 20);
  if (d.d <= 16384 && d.rows <= kMax32 && d.ldx <= kMax32 && d.ldq <= kMax32 && d.lds <= kMax32 &&
      d.lddy <= kMax32 && d.lddx <= kMax32 && d.ldds <= kMax32) {
    auto al = [](const void* q, uintptr_t n) { return (reinterpret_cast<uintptr_t>(q) % n) == 0; };
    const bool vec = d.d % 4 == 0 && al(d.dy, 16) && d.lddy % 4 == 0 &&
                     (!d.dx || (al(d.dx, 16) && d.lddx % 4 == 0)) && (!d.g || al(d.g, 16)) &&
                     (!d.b || al(d.b, 16)) &&
                     (!d.dsum || (al(d.dsum, 16) && d.ldds % 4 == 0)) &&
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
  cudaError_t e = launch_pdl(norm_bwd_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, p, (int)(d.db != nullptr));
  if (e == cudaSuccess && part)
    e = launch_pdl(norm_bwd_reduce_kernel, dim3((unsigned)((d.d + 31) / 32), d.db ? 2 : 1), dim3(kReduceThreads), 0,
                   s, (const float*)part, grid, (int)d.d, d.dg, d.db, d.accumulate);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(part, s);
  return e == cudaSuccess ? RTB_OK : failed(p, e);
}

}  // namespace rtb
