// Writing, restoring and laying out 8-bit block-scaled tensors (rtb_fp8.cuh).
//   save:    s = 2^ceil(log2(max|x| / 448)) over the block, q = e4m3(x / s)
//   restore: x' = q * s
// Both stream their operands once (5 bytes a value): HBM-bound, 16384 x 4096
// saved and restored in 132 us (5.1 TB/s, 78% of a copy); saved alone 77 us, in 128 x
// 128 blocks 100 us (3.4 TB/s), a CTA a block.
#include <cuda_bf16.h>

#include "rtb_fp8.cuh"
#include "rtb_internal.h"
#include "rtb_ptx.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 256;

inline bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

int grid_for(rtb_ctx* ctx, int64_t blocks, int per_sm) {
  const int64_t cap = (int64_t)ctx->sm_count * per_sm;
  return (int)(blocks < cap ? (blocks > 0 ? blocks : 1) : cap);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One warp per 1 x 128 block, four columns a lane (VEC: one 16-byte load and
// one 4-byte store; else columns lane + 32 j, so that the byte stores of a
// warp are contiguous), kBlocks consecutive blocks at a time: their loads are
// all in flight before the first maximum.  
constexpr int kBlocks = 4;
template <bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const float* __restrict__ x,
                                                                 int64_t ldx, int64_t total,
                                                                 int cols, int cblocks, uint8_t* q,
                                                                 int64_t ldq, uint8_t* scale,
                                                                 int64_t lds) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kBlocks;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kBlocks; w < total;
       w += step) {
    int64_t r = w / cblocks;
    int cb = (int)(w - r * cblocks);
    int64_t row[kBlocks];
    int col[kBlocks];
    float v[kBlocks][4];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      row[n] = r;
      col[n] = cb * kFp8Block;
      const bool in = w + n < total;
      const float* xr = x + r * ldx;
      if (VEC) {
        const int c = col[n] + 4 * lane;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in && c < cols) f = __ldcs(reinterpret_cast<const float4*>(xr + c));  // cols % 4 == 0
        v[n][0] = f.x; v[n][1] = f.y; v[n][2] = f.z; v[n][3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = col[n] + lane + 32 * j;
          v[n][j] = in && c < cols ? __ldcs(xr + c) : 0.0f;
        }
      }
      if (++cb == cblocks) {
        cb = 0;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      if (w + n >= total) break;
      const float amax = warp_max(fmaxf(fmaxf(finite_abs(v[n][0]), finite_abs(v[n][1])),
                                        fmaxf(finite_abs(v[n][2]), finite_abs(v[n][3]))));
      const uint32_t sb = e8m0_of_amax(amax);
      const uint32_t four = e4m3x4(v[n][0], v[n][1], v[n][2], v[n][3], e8m0_inverse(sb));
      uint8_t* qr = q + row[n] * ldq;
      if (VEC) {
        const int c = col[n] + 4 * lane;
        if (c < cols) *reinterpret_cast<uint32_t*>(qr + c) = four;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = col[n] + lane + 32 * j;
          if (c < cols) qr[c] = (uint8_t)(four >> (8 * j));
        }
      }
      if (lane == 0) scale[row[n] * lds + col[n] / kFp8Block] = (uint8_t)sb;
    }
  }
}

// One CTA per 128 x 128 block: warp w holds rows w, w + 8, ... of the block in
// registers (16 rows, four columns a lane), the maximum goes through shared
// memory.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const float* __restrict__ x,
                                                                   int64_t ldx, int64_t rows,
                                                                   int cols, int cblocks,
                                                                   int64_t total, uint8_t* q,
                                                                   int64_t ldq, uint8_t* scale,
                                                                   int64_t lds) {
  __shared__ float red[2][kThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int phase = 0;
  for (int64_t b = blockIdx.x; b < total; b += gridDim.x, phase ^= 1) {
    const int64_t rb = b / cblocks;
    const int c0 = (int)(b - rb * cblocks) * kFp8Block;
    const int64_t r0 = rb * kFp8Block;
    float v[16][4];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t r = r0 + warp + 8 * i;
      const float* xr = x + r * ldx;
      if (VEC) {
        const int c = c0 + 4 * lane;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && c < cols) f = __ldcs(reinterpret_cast<const float4*>(xr + c));
        v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = c0 + lane + 32 * j;
          v[i][j] = (r < rows && c < cols) ? __ldcs(xr + c) : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = fmaxf(amax, finite_abs(v[i][j]));
    amax = warp_max(amax);
    if (lane == 0) red[phase][warp] = amax;
    __syncthreads();  // two buffers: the next block's writes do not meet this block's readers
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k) amax = fmaxf(amax, red[phase][k]);
    const uint32_t sb = e8m0_of_amax(amax);
    const float inv = e8m0_inverse(sb);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t r = r0 + warp + 8 * i;
      if (r >= rows) continue;
      uint8_t* qr = q + r * ldq;
      const uint32_t four = e4m3x4(v[i][0], v[i][1], v[i][2], v[i][3], inv);
      if (VEC) {
        const int c = c0 + 4 * lane;
        if (c < cols) *reinterpret_cast<uint32_t*>(qr + c) = four;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = c0 + lane + 32 * j;
          if (c < cols) qr[c] = (uint8_t)(four >> (8 * j));
        }
      }
    }
    if (threadIdx.x == 0) scale[rb * lds + c0 / kFp8Block] = (uint8_t)sb;
  }
}

// Aligned rows: four columns a thread, four such quads at a time (their loads
// in flight together).
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ q,
                                                              int64_t ldq, int64_t rows, int cols,
                                                              const uint8_t* __restrict__ scale,
                                                              int64_t lds, int row_shift, float* y,
                                                              int64_t ldy) {
  griddep_wait();
  griddep_launch_dependents();
  const int quads = cols / 4;
  const int64_t total = rows * quads;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t i0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; i0 < total; i0 += 4 * step) {
    uint32_t four[4], sb[4];
    int64_t at[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t i = i0 + n * step;
      four[n] = sb[n] = 0;
      at[n] = -1;
      if (i < total) {
        const int64_t r = i / quads;
        const int c = (int)(i - r * quads) * 4;
        at[n] = r * ldy + c;
        sb[n] = __ldg(scale + (r >> row_shift) * lds + c / kFp8Block);
        four[n] = __ldcs(reinterpret_cast<const uint32_t*>(q + r * ldq + c));
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (at[n] < 0) break;
      const float s = e8m0_to_float(sb[n]);
      const float4 f = e4m3x4_to_float4(four[n]);
      __stcs(reinterpret_cast<float4*>(y + at[n]), make_float4(f.x * s, f.y * s, f.z * s, f.w * s));
    }
  }
}

// Any rows: a warp per 1 x 128 block, columns lane + 32 j, so that the byte
// loads and the stores of a warp are contiguous; kBlocks blocks at a time.
__global__ void __launch_bounds__(kThreads) dequantize_any_kernel(const uint8_t* __restrict__ q,
                                                                  int64_t ldq, int64_t total,
                                                                  int cols, int cblocks,
                                                                  const uint8_t* __restrict__ scale,
                                                                  int64_t lds, int row_shift,
                                                                  float* y, int64_t ldy) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kBlocks;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kBlocks; w < total;
       w += step) {
    int64_t r = w / cblocks;
    int cb = (int)(w - r * cblocks);
    uint32_t code[kBlocks][4], sb[kBlocks];
    float* out[kBlocks];
    int left[kBlocks];  // columns of the block from this lane's first one on
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      left[n] = w + n < total ? cols - cb * kFp8Block - lane : 0;
      const int64_t c = (int64_t)cb * kFp8Block + lane;
      sb[n] = 0;
      if (w + n < total) sb[n] = __ldg(scale + (r >> row_shift) * lds + cb);
      out[n] = y + r * ldy + c;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        code[n][j] = 32 * j < left[n] ? (uint32_t)__ldcs(q + r * ldq + c + 32 * j) : 0u;
      if (++cb == cblocks) {
        cb = 0;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const float s = e8m0_to_float(sb[n]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * j < left[n]) __stcs(out[n] + 32 * j, e4m3x2_to_float2(code[n][j]).x * s);
    }
  }
}

// dst[r][c] = c < cols ? src[r * rs + c * cs] : 0, for c < ldd, of up to two
// matrices in one launch (blockIdx.y).  Rows that are only misaligned (cs ==
// 1): four bytes a thread out of two aligned words.  Transposed (rs == 1):
// through a 64 x 64 tile so that both sides are read and written along their
// rows.
struct PackSide {
  const uint8_t* src;
  int64_t rows, cols, rs, cs;
  uint8_t* dst;
  int64_t ldd;  // a multiple of 16
};
__global__ void __launch_bounds__(kThreads) pack_bytes_kernel(const PackSide a, const PackSide b) {
  __shared__ uint8_t t[64][65];
  griddep_wait();
  griddep_launch_dependents();
  const PackSide& p = blockIdx.y ? b : a;
  if (p.cs == 1) {
    const int64_t words = p.ldd / 4, total = p.rows * words;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * kThreads) {
      const int64_t r = i / words, c = (i - r * words) * 4;
      const uint8_t* sp = p.src + r * p.rs + c;
      const int64_t n = p.cols - c;  // bytes of the word that exist
      uint32_t v = 0;
      if (n > 0) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(sp) & 3);
        const uint32_t* w = reinterpret_cast<const uint32_t*>(sp - off);
        const uint32_t lo = __ldg(w);
        // the second word only where one of the wanted bytes lies in it
        const uint32_t hi = off + (n < 4 ? (uint32_t)n : 4u) > 4u ? __ldg(w + 1) : 0u;
        v = __funnelshift_r(lo, hi, 8 * off);
        if (n < 4) v &= (1u << (8 * n)) - 1u;
      }
      *reinterpret_cast<uint32_t*>(p.dst + r * p.ldd + c) = v;
    }
    return;
  }
  const int64_t tiles_c = (p.ldd + 63) / 64, tiles = (p.rows + 63) / 64 * tiles_c;
  for (int64_t k = blockIdx.x; k < tiles; k += gridDim.x) {
    const int64_t r0 = k / tiles_c * 64, c0 = k % tiles_c * 64;
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kThreads) {
      const int lr = i & 63, lc = i >> 6;
      const int64_t r = r0 + lr, c = c0 + lc;
      t[lr][lc] = (r < p.rows && c < p.cols) ? p.src[r * p.rs + c * p.cs] : (uint8_t)0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kThreads) {
      const int lc = i & 63, lr = i >> 6;
      const int64_t r = r0 + lr, c = c0 + lc;
      if (r < p.rows && c < p.ldd) p.dst[r * p.ldd + c] = t[lr][lc];
    }
  }
}

// The weight gradient's operands, in one launch (eight columns a thread).
//
// X: the checkpoint's values in bf16: q * s has four significant bits, so the
// conversion is exact (down to bf16's smallest subnormal, 2^-133).
// Y: dC as a sum of `pieces` bf16 terms: 8 significant bits each, truncated (a
// value above bf16's largest would round to infinity) but for the last, which is
// rounded, so three hold an fp32 value exactly (24 bits) as long as the last
// term is in bf16's range.  An infinity or NaN is the first term alone, so that
// it meets the product as it would in fp32.
// Rows [rows, rows_pad) and the columns up to ldx and ldy are zero.
struct OperandsParams {
  const uint8_t* q;
  int64_t ldq;
  const uint8_t* scale;
  int64_t lds;
  int row_shift, K, qvec;
  const float* dc;
  int64_t lddc;
  int N, yvec;
  int64_t rows, rows_pad;
  __nv_bfloat16 *x, *y;
  int64_t ldx, ldy;
  int pieces;
};
__global__ void __launch_bounds__(kThreads) wgrad_operands_kernel(const OperandsParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t xu = p.ldx / 8, yu = p.ldy / 8;
  const int64_t nx = p.rows_pad * xu, total = nx + p.rows_pad * yu;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    if (i < nx) {
      const int64_t r = i / xu;
      const int c = (int)(i - r * xu) * 8;
      uint32_t w[4] = {0, 0, 0, 0};
      if (r < p.rows) {
        const uint8_t* qr = p.q + r * p.ldq + c;
        const float s = e8m0_to_float(p.scale[(r >> p.row_shift) * p.lds + c / kFp8Block]);
        uint32_t b[2] = {0, 0};
        if (p.qvec && c + 8 <= p.K) {
          const uint2 v = __ldcs(reinterpret_cast<const uint2*>(qr));
          b[0] = v.x; b[1] = v.y;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j < p.K) b[j >> 2] |= (uint32_t)qr[j] << (8 * (j & 3));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 f = e4m3x4_to_float4(b[h]);
          const __nv_bfloat162 a = __floats2bfloat162_rn(f.x * s, f.y * s);
          const __nv_bfloat162 d = __floats2bfloat162_rn(f.z * s, f.w * s);
          w[2 * h] = *reinterpret_cast<const uint32_t*>(&a);
          w[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&d);
        }
      }
      *reinterpret_cast<uint4*>(p.x + r * p.ldx + c) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      const int64_t k = i - nx, r = k / yu;
      const int c = (int)(k - r * yu) * 8;
      float v[8];
      const float* xr = p.dc + r * p.lddc + c;
      if (p.yvec && r < p.rows && c + 8 <= p.N) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(xr));
        const float4 b = __ldcs(reinterpret_cast<const float4*>(xr) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (r < p.rows && c + j < p.N) ? xr[j] : 0.0f;
      }
      for (int n = 0; n < p.pieces; ++n) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (n + 1 < p.pieces)
            asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(v[2 * j + 1]), "f"(v[2 * j]));
          else
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(v[2 * j + 1]), "f"(v[2 * j]));
          // (an infinity or NaN leaves nothing for the next term)
          const float lo = __uint_as_float(w[j] << 16), hi = __uint_as_float(w[j] & 0xFFFF0000u);
          v[2 * j] = finite_abs(v[2 * j]) > 0.0f ? v[2 * j] - lo : 0.0f;
          v[2 * j + 1] = finite_abs(v[2 * j + 1]) > 0.0f ? v[2 * j + 1] - hi : 0.0f;
        }
        *reinterpret_cast<uint4*>(p.y + ((int64_t)n * p.rows_pad + r) * p.ldy + c) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <typename... KArgs, typename... Args>
int run(const char* what, void (*k)(KArgs...), int grid, cudaStream_t s, Args... args) {
  clear_stale_cuda_error();
  cudaError_t e = launch_pdl(k, dim3((unsigned)grid), dim3(kThreads), 0, s, args...);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, what);
}

}  // namespace

int launch_fp8_quantize(rtb_ctx* ctx, const float* x, int64_t ldx, int64_t rows, int64_t cols,
                        int block_rows, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds,
                        cudaStream_t s) {
  const int cblocks = (int)((cols + kFp8Block - 1) / kFp8Block);
  const bool vec = cols % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 && aligned(x, 16) && aligned(q, 4);
  if (block_rows == 1) {
    const int64_t total = rows * cblocks;
    const int grid = grid_for(ctx, (total + 8 * kBlocks - 1) / (8 * kBlocks), 8);
    return vec ? run("fp8_quantize launch", quantize_rows_kernel<true>, grid, s, x, ldx, total,
                     (int)cols, cblocks, q, ldq, scale, lds)
               : run("fp8_quantize launch", quantize_rows_kernel<false>, grid, s, x, ldx, total,
                     (int)cols, cblocks, q, ldq, scale, lds);
  }
  const int64_t total = (rows + kFp8Block - 1) / kFp8Block * cblocks;
  const int grid = grid_for(ctx, total, 2);
  return vec ? run("fp8_quantize launch", quantize_blocks_kernel<true>, grid, s, x, ldx, rows,
                   (int)cols, cblocks, total, q, ldq, scale, lds)
             : run("fp8_quantize launch", quantize_blocks_kernel<false>, grid, s, x, ldx, rows,
                   (int)cols, cblocks, total, q, ldq, scale, lds);
}

int launch_fp8_dequantize(rtb_ctx* ctx, const uint8_t* q, int64_t ldq, int64_t rows, int64_t cols,
                          const uint8_t* scale, int64_t lds, int block_rows, float* y, int64_t ldy,
                          cudaStream_t s) {
  const bool vec = cols % 4 == 0 && ldy % 4 == 0 && ldq % 4 == 0 && aligned(y, 16) && aligned(q, 4);
  const int shift = block_rows == 1 ? 0 : 7;
  if (vec)
    return run("fp8_dequantize launch", dequantize_kernel,
               grid_for(ctx, (rows * (cols / 4) + kThreads - 1) / kThreads, 8), s, q, ldq, rows,
               (int)cols, scale, lds, shift, y, ldy);
  const int cblocks = (int)((cols + kFp8Block - 1) / kFp8Block);
  const int64_t total = rows * cblocks;
  return run("fp8_dequantize launch", dequantize_any_kernel,
             grid_for(ctx, (total + 8 * kBlocks - 1) / (8 * kBlocks), 8), s, q, ldq, total, (int)cols,
             cblocks, scale, lds, shift, y, ldy);
}

int launch_pack_bytes(rtb_ctx* ctx, const PackDesc& a, const PackDesc& b, cudaStream_t s) {
  const PackDesc* d[2] = {&a, &b};
  PackSide side[2];
  int n = 0;
  int64_t most = 1;
  for (const PackDesc* p : d) {
    if (!p->dst) continue;
    side[n++] = {p->src, p->rows, p->cols, p->rs, p->cs, p->dst, p->ldd};
    const int64_t ctas = p->cs == 1 ? (p->rows * (p->ldd / 4) + kThreads - 1) / kThreads
                                    : (p->rows + 63) / 64 * ((p->ldd + 63) / 64);
    most = ctas > most ? ctas : most;
  }
  if (n == 0) return RTB_OK;
  if (n == 1) side[1] = side[0];
  clear_stale_cuda_error();
  cudaError_t e = launch_pdl(pack_bytes_kernel, dim3((unsigned)grid_for(ctx, most, 8), (unsigned)n),
                             dim3(kThreads), 0, s, (const PackSide)side[0], (const PackSide)side[1]);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "fp8 pack launch");
}

int launch_wgrad_operands(rtb_ctx* ctx, const uint8_t* q, int64_t ldq, const uint8_t* scale,
                          int64_t lds, int block_rows, const float* dc, int64_t rows, int64_t K,
                          int64_t N, void* x, int64_t ldx, void* y, int64_t ldy, int64_t rows_pad,
                          int pieces, cudaStream_t s) {
  OperandsParams p{};
  p.q = q;
  p.ldq = ldq;
  p.scale = scale;
  p.lds = lds;
  p.row_shift = block_rows == 1 ? 0 : 7;
  p.K = (int)K;
  p.qvec = ldq % 8 == 0 && aligned(q, 8);
  p.dc = dc;
  p.lddc = N;
  p.N = (int)N;
  p.yvec = N % 4 == 0 && aligned(dc, 16);
  p.rows = rows;
  p.rows_pad = rows_pad;
  p.x = static_cast<__nv_bfloat16*>(x);
  p.y = static_cast<__nv_bfloat16*>(y);
  p.ldx = ldx;
  p.ldy = ldy;
  p.pieces = pieces;
  const int64_t units = rows_pad * ((ldx + ldy) / 8);
  return run("wgrad operands launch", wgrad_operands_kernel,
             grid_for(ctx, (units + kThreads - 1) / kThreads, 8), s, (const OperandsParams)p);
}

}  // namespace rtb
