// The 4-bit product for few rows of A (a generation step's tokens): a stream over the
// weight on the CUDA cores,
//   C[m,n] = act( sum_b 2^(sa[m,b] + sb[n,b] - 254) sum_{k in b} qa[m,k] qb[n,k] + bias[n] )
// over blocks b of 32 elements.  Twice a code's value is a whole number of at most 12,
// so a block's sum is exact in integers: four products an instruction (dp4a).  A code
// becomes a byte by table lookup: PRMT's selector takes a code's three magnitude bits as
// they lie, and a selector with the sign bit set gives 0 where the table's bytes are
// positive; so the tables 16 + v and 16 - v, the latter asked with the signs turned,
// together give 16 + value, and the 16 times the sum of the row's values is taken off
// the block's sum, where it starts.  Then one conversion, one multiply-add by the two
// scales: fp32 sees exact block sums.
//
// A warp takes four weight rows, a lane a block (16 bytes) of each at a time, so that A
// out of shared memory serves four; with few rows several warps share a contraction,
// their sums added in a fixed order.
//
// Measured: XX
#include "rtb_act.cuh"
#include "rtb_fp4.cuh"
#include "rtb_internal.h"
#include "rtb_ptx.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRows = 4;      // weight rows of a warp
// Blocks of A in shared memory at a time (40 KB, 80 for eight rows).
constexpr int chunk(int rows) { return rows == 1 ? 1024 : rows == 2 ? 512 : 256; }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
// Eight codes -> bytes of 16 + twice the value, the first four and the last four.
__device__ __forceinline__ void codes_to_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t x = w ^ 0x88888888u;
  lo = prmt(0x13121110u, 0x1C181614u, w) | prmt(0x0D0E0F10u, 0x04080A0Cu, x);
  hi = prmt(0x13121110u, 0x1C181614u, w >> 16) | prmt(0x0D0E0F10u, 0x04080A0Cu, x >> 16);
}
// c + the dot product of four unsigned and four signed bytes
__device__ __forceinline__ int dot4(uint32_t u, uint32_t s, int c) {
  int d;
  asm("dp4a.u32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(u), "r"(s), "r"(c));
  return d;
}

// The 16 bytes of block b of a row of `half` bytes, 0 behind the row.  VEC: the row is on
// a 16-byte boundary.  Else aligned words, each read only where one of its bytes exists.
template <bool VEC>
__device__ __forceinline__ uint4 load_block(const uint8_t* row, int b, int half) {
  const uint8_t* p = row + (int64_t)16 * b;
  if (VEC) return __ldg(reinterpret_cast<const uint4*>(p));  // (a row's last block: its own 16 bytes)
  const int off = (int)(reinterpret_cast<uintptr_t>(p) & 3u);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p - off);
  const int left = half - 16 * b;
  uint32_t v[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = 4 * i - off < left && (i < 4 || off) ? __ldg(w + i) : 0u;
  return make_uint4(__funnelshift_r(v[0], v[1], 8 * off), __funnelshift_r(v[1], v[2], 8 * off),
                    __funnelshift_r(v[2], v[3], 8 * off), __funnelshift_r(v[3], v[4], 8 * off));
}

struct RowsParams {
  int64_t N;
  int M, half, blocks, split;  // split: warps that share a contraction
  const uint8_t *A, *B, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb;
  const float* bias;
  int act;
  float* C;
  int64_t ldc;
};

// MT: rows of A in the registers (M of them exist).  Shared memory: A's bytes
// [MT][2 halves][kChunk][16], then [MT][kChunk] pairs of what a block's sum starts from
// and half of half of its scale.
template <int MT, bool VEC>
__global__ void __launch_bounds__(kThreads) fp4_rows_kernel(const RowsParams p) {
  constexpr int kChunk = chunk(MT);
  extern __shared__ uint4 a_s[];
  int2* start_s = reinterpret_cast<int2*>(a_s + MT * 2 * kChunk);
  __shared__ float red[kWarps][kRows * MT];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = p.split, part = warp % split;
  const int64_t n0 = ((int64_t)blockIdx.x * (kWarps / split) + warp / split) * kRows;
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
      if (b < p.blocks && n0 + r < p.N) {
        w[r] = load_block<VEC>(p.B + (n0 + r) * p.ldb, b, p.half);
        sb[r] = __ldg(p.sb + (n0 + r) * p.ldsb + b);
      }
    }
  };
  int b = 32 * part + lane;
  load(b);  // on its way while A is laid out
  for (int c0 = 0; c0 < p.blocks; c0 += kChunk) {
    const int cn = p.blocks - c0 < kChunk ? p.blocks - c0 : kChunk;
    if (c0) __syncthreads();  // the chunk before has been read
    for (int i = threadIdx.x; i < MT * cn; i += kThreads) {
      const int m = i / cn, k = i - m * cn;
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      uint32_t s = 127u;
      if (m < p.M) {
        q = load_block<false>(p.A + m * p.lda, c0 + k, p.half);
        s = __ldg(p.sa + m * p.ldsa + c0 + k);
        const int left = p.half - 16 * (c0 + k);  // bytes behind the row are none of its own
        if (left < 16) {
          uint32_t* e = &q.x;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            e[j] = left >= 4 * j + 4 ? e[j] : left <= 4 * j ? 0u : e[j] & ((1u << (8 * (left - 4 * j))) - 1u);
        }
      }
      uint32_t v[8];
      codes_to_bytes(q.x, v[0], v[1]);
      codes_to_bytes(q.y, v[2], v[3]);
      codes_to_bytes(q.z, v[4], v[5]);
      codes_to_bytes(q.w, v[6], v[7]);
      int sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __vsub4(v[j], 0x10101010u);
        sum = __dp4a((int)v[j], 0x01010101, sum);
      }
      a_s[(2 * m) * kChunk + k] = make_uint4(v[0], v[1], v[2], v[3]);
      a_s[(2 * m + 1) * kChunk + k] = make_uint4(v[4], v[5], v[6], v[7]);
      start_s[m * kChunk + k] = make_int2(-16 * sum, __float_as_int(0.25f * e8m0_to_float(s)));
    }
    __syncthreads();
    while (b < c0 + cn) {
      uint32_t u[kRows][8];
      float fb[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        codes_to_bytes(w[r].x, u[r][0], u[r][1]);
        codes_to_bytes(w[r].y, u[r][2], u[r][3]);
        codes_to_bytes(w[r].z, u[r][4], u[r][5]);
        codes_to_bytes(w[r].w, u[r][6], u[r][7]);
        fb[r] = e8m0_to_float(sb[r]);
      }
      const int k = b - c0;
      b += 32 * split;
      load(b);  // the next block's, while this one's are multiplied
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 x = a_s[(2 * m) * kChunk + k], y = a_s[(2 * m + 1) * kChunk + k];
        const int2 st = start_s[m * kChunk + k];
        const float fa = __int_as_float(st.y);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          int d = st.x;
          d = dot4(u[r][0], x.x, d);
          d = dot4(u[r][1], x.y, d);
          d = dot4(u[r][2], x.z, d);
          d = dot4(u[r][3], x.w, d);
          d = dot4(u[r][4], y.x, d);
          d = dot4(u[r][5], y.y, d);
          d = dot4(u[r][6], y.z, d);
          d = dot4(u[r][7], y.w, d);
          acc[r * MT + m] = fmaf((float)d, fa * fb[r], acc[r * MT + m]);
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
  if ((lane & (32 / (kRows * MT) - 1)) == 0) red[warp][index] = acc[0];
  __syncthreads();
  for (int i = threadIdx.x; i < kWarps / split * kRows * MT; i += kThreads) {
    const int g = i / (kRows * MT), v = i % (kRows * MT), m = v % MT;
    const int64_t n = ((int64_t)blockIdx.x * (kWarps / split) + g) * kRows + v / MT;
    if (m >= p.M || n >= p.N) continue;
    float sum = red[g * split][v];
    for (int k = 1; k < split; ++k) sum += red[g * split + k][v];
    p.C[m * p.ldc + n] = activate(sum + (p.bias ? __ldg(p.bias + n) : 0.0f), p.act);
  }
}

template <int MT, bool VEC>
int launch(rtb_ctx* ctx, RowsParams& p, cudaStream_t s) {
  auto* k = fp4_rows_kernel<MT, VEC>;
  constexpr int kSmem = MT * chunk(MT) * 40;
  if (kSmem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return cuda_status(e, "fp4_matmul smem attribute");
  }
  const int64_t groups = (p.N + kRows - 1) / kRows;
  // warps that share a contraction: until 16 warps an SM have work, each a block a lane
  p.split = 1;
  while (p.split < kWarps && groups * p.split < (int64_t)16 * ctx->sm_count && p.split * 64 <= p.blocks)
    p.split *= 2;
  const int64_t per = kWarps / p.split, grid = (groups + per - 1) / per;
  clear_stale_cuda_error();
  cudaError_t e = launch_pdl(k, dim3((unsigned)grid), dim3(kThreads), (size_t)kSmem, s, (const RowsParams)p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "fp4_matmul launch");
}

}  // namespace

int fp4_rows_run(rtb_ctx* ctx, const Fp4Desc& d, cudaStream_t s) {
  RowsParams p{};
  p.N = d.N;
  p.M = (int)d.M;
  p.half = (int)(d.K / 2);
  p.blocks = (int)((d.K + 31) / 32);
  p.A = d.A;
  p.lda = d.lda;
  p.B = d.B;
  p.ldb = d.ldb;
  p.sa = d.sa;
  p.ldsa = d.ldsa;
  p.sb = d.sb;
  p.ldsb = d.ldsb;
  p.bias = d.bias;
  p.act = d.act;
  p.C = d.C;
  p.ldc = d.ldc;
  const bool vec = (reinterpret_cast<uintptr_t>(d.B) & 15u) == 0 && d.ldb % 16 == 0;
  if (d.M == 1) return vec ? launch<1, true>(ctx, p, s) : launch<1, false>(ctx, p, s);
  if (d.M == 2) return vec ? launch<2, true>(ctx, p, s) : launch<2, false>(ctx, p, s);
  if (d.M <= 4) return vec ? launch<4, true>(ctx, p, s) : launch<4, false>(ctx, p, s);
  return vec ? launch<8, true>(ctx, p, s) : launch<8, false>(ctx, p, s);
}

}  // namespace rtb
