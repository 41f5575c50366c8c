// Writing, restoring and laying out 8-bit block-scaled tensors (rtb_fp8.cuh).
//   save:    s = 2^ceil(log2(max|x| / 448)) over the block, q = e4m3(x / s)
//   restore: x' = q * s
// Both stream their operands once (5 bytes a value): HBM-bound.
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
// warp are contiguous).
template <bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const float* __restrict__ x,
                                                                 int64_t ldx, int64_t rows, int cols,
                                                                 int cblocks, uint8_t* q,
                                                                 int64_t ldq, uint8_t* scale,
                                                                 int64_t lds) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t total = rows * cblocks;
  for (int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
    const int64_t r = w / cblocks;
    const int c0 = (int)(w - r * cblocks) * kFp8Block;
    const float* xr = x + r * ldx;
    uint8_t* qr = q + r * ldq;
    float v[4];
    if (VEC) {
      const int c = c0 + 4 * lane;
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < cols) f = __ldcs(reinterpret_cast<const float4*>(xr + c));  // cols % 4 == 0
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + lane + 32 * j;
        v[j] = c < cols ? __ldcs(xr + c) : 0.0f;
      }
    }
    const float amax = warp_max(fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])),
                                      fmaxf(finite_abs(v[2]), finite_abs(v[3]))));
    const uint32_t sb = e8m0_of_amax(amax);
    const uint32_t four = e4m3x4(v[0], v[1], v[2], v[3], e8m0_inverse(sb));
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
    if (lane == 0) scale[r * lds + c0 / kFp8Block] = (uint8_t)sb;
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

// Four columns a thread.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ q,
                                                              int64_t ldq, int64_t rows, int cols,
                                                              const uint8_t* __restrict__ scale,
                                                              int64_t lds, int row_shift, float* y,
                                                              int64_t ldy) {
  griddep_wait();
  griddep_launch_dependents();
  const int quads = (cols + 3) / 4;
  const int64_t total = rows * quads;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const int64_t r = i / quads;
    const int c = (int)(i - r * quads) * 4;
    const uint8_t* qr = q + r * ldq + c;
    const float s = e8m0_to_float(scale[(r >> row_shift) * lds + c / kFp8Block]);
    uint32_t four = 0;
    if (VEC) {
      four = __ldcs(reinterpret_cast<const uint32_t*>(qr));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) four |= (uint32_t)qr[j] << (8 * j);
    }
    const float4 f = e4m3x4_to_float4(four);
    float* yr = y + r * ldy + c;
    if (VEC) {
      __stcs(reinterpret_cast<float4*>(yr), make_float4(f.x * s, f.y * s, f.z * s, f.w * s));
    } else {
      const float e[4] = {f.x * s, f.y * s, f.z * s, f.w * s};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) yr[j] = e[j];
    }
  }
}

// dst[r][c] = c < cols ? src[r * rs + c * cs] : 0, for c < ldd, through a 64 x
// 64 tile so that both sides are read and written along their rows.
__global__ void __launch_bounds__(kThreads) pack_bytes_kernel(const uint8_t* __restrict__ src,
                                                              int64_t rows, int64_t cols, int64_t rs,
                                                              int64_t cs, uint8_t* dst, int64_t ldd,
                                                              int64_t tiles_c, int64_t tiles) {
  __shared__ uint8_t t[64][65];
  griddep_wait();
  griddep_launch_dependents();
  for (int64_t b = blockIdx.x; b < tiles; b += gridDim.x) {
    const int64_t r0 = b / tiles_c * 64, c0 = b % tiles_c * 64;
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kThreads) {
      const int fast = i & 63, slow = i >> 6;
      const int lr = cs == 1 ? slow : fast, lc = cs == 1 ? fast : slow;
      const int64_t r = r0 + lr, c = c0 + lc;
      t[lr][lc] = (r < rows && c < cols) ? src[r * rs + c * cs] : (uint8_t)0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kThreads) {
      const int lc = i & 63, lr = i >> 6;
      const int64_t r = r0 + lr, c = c0 + lc;
      if (r < rows && c < ldd) dst[r * ldd + c] = t[lr][lc];
    }
  }
}

// The checkpoint's values in bf16: q * s has four significant bits, so the
// conversion is exact (down to bf16's smallest subnormal, 2^-133).  Rows
// [rows, rows_pad) and columns [cols, ldo) are zero.
__global__ void __launch_bounds__(kThreads) decode_bf16_kernel(const uint8_t* __restrict__ q,
                                                               int64_t ldq, int64_t rows, int cols,
                                                               const uint8_t* __restrict__ scale,
                                                               int64_t lds, int row_shift,
                                                               __nv_bfloat16* out, int64_t ldo,
                                                               int64_t rows_pad, int vec) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t units = ldo / 8;
  const int64_t total = rows_pad * units;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const int64_t r = i / units;
    const int c = (int)(i - r * units) * 8;
    uint32_t w[4] = {0, 0, 0, 0};
    if (r < rows) {
      const uint8_t* qr = q + r * ldq + c;
      const float s = e8m0_to_float(scale[(r >> row_shift) * lds + c / kFp8Block]);
      uint32_t b[2] = {0, 0};
      if (vec && c + 8 <= cols) {
        const uint2 v = __ldcs(reinterpret_cast<const uint2*>(qr));
        b[0] = v.x; b[1] = v.y;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < cols) b[j >> 2] |= (uint32_t)qr[j] << (8 * (j & 3));
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
    *reinterpret_cast<uint4*>(out + r * ldo + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// x as a sum of `pieces` bf16 terms, each the rounding of what the ones before
// left: 8 significant bits a term, so three hold an fp32 value exactly (24
// bits) as long as the last term is in bf16's range.  An infinity or NaN is the
// first term alone, so that it meets the product as it would in fp32.
__global__ void __launch_bounds__(kThreads) split_bf16_kernel(const float* __restrict__ x,
                                                              int64_t ldx, int64_t rows, int cols,
                                                              __nv_bfloat16* out, int64_t ldo,
                                                              int64_t rows_pad, int pieces, int vec) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t units = ldo / 8;
  const int64_t total = rows_pad * units;
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const int64_t r = i / units;
    const int c = (int)(i - r * units) * 8;
    float v[8];
    const float* xr = x + r * ldx + c;
    if (vec && r < rows && c + 8 <= cols) {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(xr));
      const float4 b = __ldcs(reinterpret_cast<const float4*>(xr) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (r < rows && c + j < cols) ? xr[j] : 0.0f;
    }
    for (int p = 0; p < pieces; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&t);
        // (an infinity or NaN leaves nothing for the next term)
        v[2 * j] = finite_abs(v[2 * j]) > 0.0f ? v[2 * j] - __low2float(t) : 0.0f;
        v[2 * j + 1] = finite_abs(v[2 * j + 1]) > 0.0f ? v[2 * j + 1] - __high2float(t) : 0.0f;
      }
      *reinterpret_cast<uint4*>(out + ((int64_t)p * rows_pad + r) * ldo + c) =
          make_uint4(w[0], w[1], w[2], w[3]);
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
    const int grid = grid_for(ctx, (rows * cblocks + 7) / 8, 8);
    return vec ? run("fp8_quantize launch", quantize_rows_kernel<true>, grid, s, x, ldx, rows,
                     (int)cols, cblocks, q, ldq, scale, lds)
               : run("fp8_quantize launch", quantize_rows_kernel<false>, grid, s, x, ldx, rows,
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
  const int64_t quads = (cols + 3) / 4;
  const int grid = grid_for(ctx, (rows * quads + kThreads - 1) / kThreads, 8);
  const int shift = block_rows == 1 ? 0 : 7;
  return vec ? run("fp8_dequantize launch", dequantize_kernel<true>, grid, s, q, ldq, rows,
                   (int)cols, scale, lds, shift, y, ldy)
             : run("fp8_dequantize launch", dequantize_kernel<false>, grid, s, q, ldq, rows,
                   (int)cols, scale, lds, shift, y, ldy);
}

int launch_pack_bytes(rtb_ctx* ctx, const uint8_t* src, int64_t rows, int64_t cols, int64_t rs,
                      int64_t cs, uint8_t* dst, int64_t ldd, cudaStream_t s) {
  const int64_t tiles_c = (ldd + 63) / 64, tiles = (rows + 63) / 64 * tiles_c;
  return run("fp8 pack launch", pack_bytes_kernel, grid_for(ctx, tiles, 8), s, src, rows, cols, rs,
             cs, dst, ldd, tiles_c, tiles);
}

int launch_decode_bf16(rtb_ctx* ctx, const uint8_t* q, int64_t ldq, int64_t rows, int64_t cols,
                       const uint8_t* scale, int64_t lds, int block_rows, void* out, int64_t ldo,
                       int64_t rows_pad, cudaStream_t s) {
  const int vec = ldq % 8 == 0 && aligned(q, 8);
  const int grid = grid_for(ctx, (rows_pad * (ldo / 8) + kThreads - 1) / kThreads, 8);
  return run("fp8 decode launch", decode_bf16_kernel, grid, s, q, ldq, rows, (int)cols, scale, lds,
             block_rows == 1 ? 0 : 7, static_cast<__nv_bfloat16*>(out), ldo, rows_pad, vec);
}

int launch_split_bf16(rtb_ctx* ctx, const float* x, int64_t ldx, int64_t rows, int64_t cols,
                      void* out, int64_t ldo, int64_t rows_pad, int pieces, cudaStream_t s) {
  const int vec = ldx % 4 == 0 && aligned(x, 16);
  const int grid = grid_for(ctx, (rows_pad * (ldo / 8) + kThreads - 1) / kThreads, 8);
  return run("split launch", split_bf16_kernel, grid, s, x, ldx, rows, (int)cols,
             static_cast<__nv_bfloat16*>(out), ldo, rows_pad, pieces, vec);
}

}  // namespace rtb
