// The 4-bit product for few rows of A (a generation step's tokens): a stream over the
// weight on the CUDA cores,
//   C[m,n] = act( sum_b 2^(sa[m,b] + sb[n,b] - 254) sum_{k in b} qa[m,k] qb[n,k] + bias[n] )
// over blocks b of 32 elements.  A code's value is a half-precision number as it
// stands, so two codes become one register by one conversion (a PRMT lookup of bytes for
// integer dot products takes 4.7 clocks a warp and eight codes, this 2.5), and the
// products are packed half-precision multiply-adds that are exact: a chain of eight
// products is a multiple of 1/4 of at most 288, eleven bits.  A block's four chains are
// added in fp32, exactly too, then multiplied by the smaller scale (exactly) and by the
// larger in a multiply-add: fp32 rounds once for each block.
//
// A warp takes four weight rows, a lane a block (16 bytes) of each at a time, so that A
// out of shared memory serves four; with few weight rows several warps share a
// contraction, their sums added in a fixed order.  A CTA keeps A for all of its rows.
//
// Measured (in a graph): a row by 4096 x 4096 in 4.1 us out of L2 and 4.4 from memory (two
// rows 5.3, four by 2048 x 2048 3.4); by 1000 x 1000, rows of 500 bytes, 3.7.  Bound by the conversions and
// products, 2.5 of the 4.4 clocks that a warp takes for eight codes, and a short call by its
// start and end.
#include <type_traits>

#include "rtb_act.cuh"
#include "rtb_fp4.cuh"
#include "rtb_fp4_load.cuh"
#include "rtb_internal.h"
#include "rtb_ptx.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = 4;      // weight rows of a warp
// Blocks of a weight row that a warp takes at a time.  Rows on 16-byte boundaries: one a
// lane.  Else a lane loads the 16 aligned bytes in which its block begins, the rest are
// the next lane's, and the last lane is there for its neighbour only.
constexpr int lanes(bool vec) { return vec ? 32 : 31; }
// Blocks of A in shared memory at a time (68 KB): whole turns of a warp.
constexpr int chunk(int rows, bool vec) { return 1024 / rows / 32 * lanes(vec); }

// Eight codes -> four pairs of half-precision values, exactly.
__device__ __forceinline__ void codes_to_halves(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ void fma_halves(uint32_t& d, uint32_t a, uint32_t b) {
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(d) : "r"(a), "r"(b));
}
// The smaller of two scales and the larger; NaN where one of them is.
__device__ __forceinline__ float2 ordered(float a, float b) {
  float2 f;
  asm("min.NaN.f32 %0, %2, %3;\n\tmax.NaN.f32 %1, %2, %3;" : "=f"(f.x), "=f"(f.y) : "f"(a), "f"(b));
  return f;
}
__device__ __forceinline__ float sum_of_halves(uint32_t h) {
  float lo, hi;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(lo), "=f"(hi)
      : "r"(h));
  return lo + hi;
}

// The 16 bytes that begin `off` (0..15, the same in all lanes) behind this lane's 16,
// which the next lane's follow.
__device__ __forceinline__ uint4 behind(uint4 w, int off) {
  if (off == 0) return w;
  uint32_t v[8] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[4 + i] = __shfl_down_sync(0xffffffffu, v[i], 1);
#pragma unroll
  for (int i = 0; i < 6; ++i) v[i] = off & 8 ? v[i + 2] : v[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = off & 4 ? v[i + 1] : v[i];
  const int s = 8 * (off & 3);
  return make_uint4(__funnelshift_r(v[0], v[1], s), __funnelshift_r(v[1], v[2], s),
                    __funnelshift_r(v[2], v[3], s), __funnelshift_r(v[3], v[4], s));
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

struct RowsParams {
  int64_t N;
  int M, half, blocks, split;  // split: warps that share a contraction
  int64_t groups;              // of weight rows
  const uint8_t *A, *B, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb;
  const float* bias;
  int act;
  int16_t front, back;         // ENDS: weight rows in front of the first and behind the N-th
  float* C;
  int64_t ldc;
};
static_assert(sizeof(RowsParams) <= 128, "more: other registers, a row by 4096 x 4096 4.4 -> 4.8 us");

// A block of a row of A, 0 where the row has ended.  (The large kernel has these lines in
// its loop: with this call it takes other registers, a row by 4096 x 4096 4.4 -> 4.6 us.)
__device__ __forceinline__ uint4 load_a(const RowsParams& p, int m, int b) {
  uint4 q = load_block(p.A + m * p.lda, b, p.half);
  const int left = p.half - 16 * b;  // bytes behind the row are none of its own
  if (left < 16) {
    uint32_t* e = &q.x;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      e[j] = left >= 4 * j + 4 ? e[j] : left <= 4 * j ? 0u : e[j] & ((1u << (8 * (left - 4 * j))) - 1u);
  }
  return q;
}

// The weight's ends: the first and last rows, whose 16-byte loads would reach over the
// matrix, by words, a row at a time for the whole CTA.  (One CTA more for them: a row by
// 1000 x 1000 3.7 us as before, by 28672 x 8190 49.3 -> 47.7.  Both kinds of loads in one
// loop cost every row, 28672 x 8190 64 us.)
template <int MT>
__device__ __forceinline__ void end_rows(const RowsParams& p, float (*red)[kRows * MT]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int e = 0; e < p.front + p.back; ++e) {
    const int64_t n = e < p.front ? e - p.front : p.N + e - p.front;
    float acc[MT] = {};
#pragma unroll 1
    for (int b = threadIdx.x; b < p.blocks; b += kThreads) {
      const uint4 q = load_block(p.B + n * p.ldb, b, p.half);
      const float fb = e8m0_to_float(__ldg(p.sb + n * p.ldsb + b));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= p.M) break;
        const uint4 x = load_a(p, m, b);
        const float2 f = ordered(e8m0_to_float(__ldg(p.sa + m * p.ldsa + b)), fb);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t hq[4], hx[4], d = 0u;
          codes_to_halves(j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w, hq);
          codes_to_halves(j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w, hx);
#pragma unroll
          for (int k = 0; k < 4; ++k) fma_halves(d, hq[k], hx[k]);
          sum += sum_of_halves(d);
        }
        acc[m] = fmaf(sum * f.x, f.y, acc[m]);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
      if (lane == 0) red[warp][m] = acc[m];
    }
    __syncthreads();
    if ((int)threadIdx.x < p.M) {
      float sum = 0.0f;
      for (int k = 0; k < kWarps; ++k) sum += red[k][threadIdx.x];
      p.C[threadIdx.x * p.ldc + n] = activate(sum + (p.bias ? __ldg(p.bias + n) : 0.0f), p.act);
    }
    __syncthreads();  // red[] is free
  }
}

// MT: rows of A in the registers (M of them exist).  Shared memory: A's halves
// [MT][4 words][kChunk][16 bytes], then [MT][kChunk] scales.
// ENDS: a CTA more, for the weight's ends.
template <int MT, bool VEC, bool ENDS>
__global__ void __launch_bounds__(kThreads, 2) fp4_rows_kernel(const RowsParams p) {
  constexpr int kChunk = chunk(MT, VEC), kLanes = lanes(VEC);
  extern __shared__ uint4 a_s[];
  float* scale_s = reinterpret_cast<float*>(a_s + MT * 4 * kChunk);
  __shared__ float red[kWarps][kRows * MT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = p.split, part = warp % split, per = kWarps / split;  // per: groups of a CTA
  // The first of the weight into L2, while the kernel before ends (a hint, which reads
  // nothing: the weight may still be written; a row by 4096 x 4096 5.2 -> 4.4 us).
  {
    const int64_t n0 = ((int64_t)blockIdx.x * per + warp / split) * kRows;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t at = (int64_t)16 * (kLanes * (part + k * split) + lane);
        if (n0 + r < p.N && at < p.half) prefetch_l2(p.B + (n0 + r) * p.ldb + at);
      }
  }
  griddep_wait();
  griddep_launch_dependents();
  const unsigned ctas = gridDim.x - ENDS;
  if (ENDS && blockIdx.x == ctas) {
    end_rows<MT>(p, red);
    return;
  }
  for (int64_t g0 = (int64_t)blockIdx.x * per; g0 < p.groups; g0 += (int64_t)ctas * per) {
    const int64_t n0 = (g0 + warp / split) * kRows;
    float acc[kRows * MT];
#pragma unroll
    for (int i = 0; i < kRows * MT; ++i) acc[i] = 0.0f;
    uint4 w[kRows];
    uint32_t sb[kRows];
    auto load = [&](int b) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        w[r] = make_uint4(0u, 0u, 0u, 0u);
        sb[r] = 127u;
        if (n0 + r < p.N) {
          const uint8_t* row = p.B + (n0 + r) * p.ldb;
          if (VEC) {
            if (b < p.blocks) w[r] = __ldg(reinterpret_cast<const uint4*>(row) + b);
          } else {
            w[r] = load_chunk(row, b, p.half);
          }
          if (b < p.blocks) sb[r] = __ldg(p.sb + (n0 + r) * p.ldsb + b);
        }
      }
    };
    int b = kLanes * part + lane;
    load(b);  // on its way while A is laid out
    for (int c0 = 0; c0 < p.blocks; c0 += kChunk) {
      const int cn = p.blocks - c0 < kChunk ? p.blocks - c0 : kChunk;
      // (A that fits stays for all of the CTA's groups)
      if (p.blocks > kChunk || g0 == (int64_t)blockIdx.x * per) {
        if (p.blocks > kChunk) __syncthreads();  // the chunk before has been read
        for (int i = threadIdx.x; i < MT * cn; i += kThreads) {
          const int m = i / cn, k = i - m * cn;
          uint4 q = make_uint4(0u, 0u, 0u, 0u);
          uint32_t s = 127u;
          if (m < p.M) {
            q = load_block(p.A + m * p.lda, c0 + k, p.half);
            s = __ldg(p.sa + m * p.ldsa + c0 + k);
            const int left = p.half - 16 * (c0 + k);  // bytes behind the row are none of its own
            if (left < 16) {
              uint32_t* e = &q.x;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                e[j] = left >= 4 * j + 4 ? e[j] : left <= 4 * j ? 0u : e[j] & ((1u << (8 * (left - 4 * j))) - 1u);
            }
          }
          const uint32_t e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t h[4];
            codes_to_halves(e[j], h);
            a_s[(4 * m + j) * kChunk + k] = make_uint4(h[0], h[1], h[2], h[3]);
          }
          scale_s[m * kChunk + k] = e8m0_to_float(s);
        }
        __syncthreads();
      }
      while (b - lane < c0 + cn) {  // (a warp's lanes stay together)
        const bool mine = lane < kLanes && b < c0 + cn;
        const int k = mine ? b - c0 : 0;
        uint4 u[kRows];
        float fb[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          u[r] = VEC ? w[r] : behind(w[r], (int)((reinterpret_cast<uintptr_t>(p.B) + (n0 + r) * p.ldb) & 15));
          fb[r] = e8m0_to_float(sb[r]);
        }
        b += kLanes * split;
        load(b);  // the next block's, while this one's are multiplied
        uint32_t d[kRows * MT][2];  // two chains: words 0 and 1, 2 and 3
#pragma unroll
        for (int i = 0; i < kRows * MT; ++i) d[i][0] = d[i][1] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 x[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) x[m] = a_s[(4 * m + j) * kChunk + k];
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            uint32_t h[4];
            codes_to_halves(j == 0 ? u[r].x : j == 1 ? u[r].y : j == 2 ? u[r].z : u[r].w, h);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              fma_halves(d[r * MT + m][j / 2], h[0], x[m].x);
              fma_halves(d[r * MT + m][j / 2], h[1], x[m].y);
              fma_halves(d[r * MT + m][j / 2], h[2], x[m].z);
              fma_halves(d[r * MT + m][j / 2], h[3], x[m].w);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const float fa = scale_s[m * kChunk + k];
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            // (the smaller scale first: exact, and finite where the product of the sum and
            // both is, which the product of the two need not be)
            const float2 f = ordered(fa, fb[r]);
            const float sum = sum_of_halves(d[r * MT + m][0]) + sum_of_halves(d[r * MT + m][1]);
            if (mine) acc[r * MT + m] = fmaf(sum * f.x, f.y, acc[r * MT + m]);
          }
        }
      }
    }
    // The lanes' sums: halves of the values change places until each lane has one, then
    // the rest of the lanes that share it.
    int index = 0;
#pragma unroll
    for (int step = 0; step < 5; ++step) {
      const int o = 16 >> step, n = (kRows * MT) >> (step + 1);  // a constant each
      if (n > 0) {
        const bool upper = lane & o;
        index = 2 * index + upper;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float send = upper ? acc[i] : acc[i + n], keep = upper ? acc[i + n] : acc[i];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      } else {
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
      }
    }
    const bool mine = (lane & (32 / (kRows * MT) - 1)) == 0;
    const int m = index % MT;
    if (split == 1) {
      const int64_t n = n0 + index / MT;
      if (mine && m < p.M && n < p.N)
        p.C[m * p.ldc + n] = activate(acc[0] + (p.bias ? __ldg(p.bias + n) : 0.0f), p.act);
      continue;
    }
    if (mine) red[warp][index] = acc[0];
    __syncthreads();
    for (int i = threadIdx.x; i < per * kRows * MT; i += kThreads) {
      const int g = i / (kRows * MT), v = i % (kRows * MT), mm = v % MT;
      const int64_t n = (g0 + g) * kRows + v / MT;
      if (mm >= p.M || n >= p.N) continue;
      float sum = red[g * split][v];
      for (int k = 1; k < split; ++k) sum += red[g * split + k][v];
      p.C[mm * p.ldc + n] = activate(sum + (p.bias ? __ldg(p.bias + n) : 0.0f), p.act);
    }
    __syncthreads();  // red[] is free
  }
}

template <int MT, bool VEC, bool ENDS>
int launch(rtb_ctx* ctx, RowsParams& p, cudaStream_t s) {
  auto* k = fp4_rows_kernel<MT, VEC, ENDS>;
  constexpr int kSmem = MT * chunk(MT, VEC) * 68;
  {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return cuda_status(e, "fp4_matmul smem attribute");
  }
  p.groups = (p.N + kRows - 1) / kRows;
  // Two CTAs on an SM at once; warps that share a contraction while that many have work
  // and each lane a block.
  const int64_t warps = (int64_t)2 * ctx->sm_count * kWarps;
  p.split = 1;
  while (p.split < kWarps && p.groups * p.split * 2 <= warps && p.split * 2 * lanes(VEC) <= p.blocks)
    p.split *= 2;
  const int64_t per = kWarps / p.split, need = (p.groups + per - 1) / per;
  const int64_t most = 2 * ctx->sm_count - ENDS;
  const int64_t ctas = need < most ? need : most;
  clear_stale_cuda_error();
  cudaError_t e = launch_pdl(k, dim3((unsigned)(ctas + ENDS)), dim3(kThreads), (size_t)kSmem, s, (const RowsParams)p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "fp4_matmul launch");
}

}  // namespace

int fp4_rows_run(rtb_ctx* ctx, const Fp4Desc& d, cudaStream_t s) {
  RowsParams p{};
  p.M = (int)d.M;
  p.half = (int)(d.K / 2);
  p.blocks = (int)((d.K + 31) / 32);
  int front, back;
  end_rows_of(d.B, d.N, d.ldb, p.half, &front, &back);
  p.front = (int16_t)front;
  p.back = (int16_t)back;
  p.N = d.N - front - back;
  p.A = d.A;
  p.lda = d.lda;
  p.B = d.B + front * d.ldb;
  p.ldb = d.ldb;
  p.sa = d.sa;
  p.ldsa = d.ldsa;
  p.sb = d.sb + front * d.ldsb;
  p.ldsb = d.ldsb;
  p.bias = d.bias ? d.bias + front : nullptr;
  p.act = d.act;
  p.C = d.C + front;
  p.ldc = d.ldc;
  const bool vec = (reinterpret_cast<uintptr_t>(d.B) & 15u) == 0 && d.ldb % 16 == 0;
  const bool ends = front + back > 0;
  auto as = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    if (vec) return ends ? launch<MT, true, true>(ctx, p, s) : launch<MT, true, false>(ctx, p, s);
    return ends ? launch<MT, false, true>(ctx, p, s) : launch<MT, false, false>(ctx, p, s);
  };
  if (d.M == 1) return as(std::integral_constant<int, 1>());
  if (d.M == 2) return as(std::integral_constant<int, 2>());
  return as(std::integral_constant<int, 4>());
}

}  // namespace rtb
