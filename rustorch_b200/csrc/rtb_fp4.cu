// Writing and restoring 4-bit block-scaled tensors (rtb_fp4.cuh).
//   save:    s = 2^ceil(log2(max|x| / 6)) over the block, q = e2m1(x / s)
//   restore: x' = q * s
// Both stream their operands once (4.53 bytes a value): HBM-bound.
#include "rtb_fp4.cuh"
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

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Aligned rows: eight columns a lane, 256 columns a warp and kChunks such chunks at a
// time, whose loads are all in flight before the first maximum; four lanes share a
// block.
constexpr int kChunks = 2;
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const float* __restrict__ x, int64_t ldx,
                                                                int64_t total, int cols, int chunks,
                                                                uint8_t* q, int64_t ldq, uint8_t* scale,
                                                                int64_t lds) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kChunks;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kChunks; w < total;
       w += step) {
    int64_t row[kChunks];
    int col[kChunks];
    float v[kChunks][8];
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      row[n] = (w + n) / chunks;
      col[n] = (int)((w + n) - row[n] * chunks) * 256 + 8 * lane;
      if (w + n >= total) col[n] = cols;  // (past the last row)
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (col[n] < cols) {  // cols % 8 == 0
        const float4* p = reinterpret_cast<const float4*>(x + row[n] * ldx + col[n]);
        a = __ldcs(p);
        b = __ldcs(p + 1);
      }
      v[n][0] = a.x; v[n][1] = a.y; v[n][2] = a.z; v[n][3] = a.w;
      v[n][4] = b.x; v[n][5] = b.y; v[n][6] = b.z; v[n][7] = b.w;
    }
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[n][j]));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t sb = fp4_scale_byte(top);
      const uint32_t eight = e2m1x8(v[n], fp4_inverse(sb));
      if (col[n] < cols) {
        *reinterpret_cast<uint32_t*>(q + row[n] * ldq + col[n] / 2) = sb == 255 ? 0u : eight;
        if ((lane & 3) == 0) scale[row[n] * lds + col[n] / kFp4Block] = (uint8_t)sb;
      }
    }
  }
}

// Any rows: a warp a block, a column a lane, kBlocks blocks at a time.
constexpr int kBlocks = 8;
__global__ void __launch_bounds__(kThreads) fp4_quantize_any_kernel(const float* __restrict__ x,
                                                                    int64_t ldx, int64_t total, int cols,
                                                                    int cblocks, uint8_t* q, int64_t ldq,
                                                                    uint8_t* scale, int64_t lds) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kBlocks;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kBlocks; w < total;
       w += step) {
    int64_t r = w / cblocks;
    int cb = (int)(w - r * cblocks);
    int64_t row[kBlocks];
    int block[kBlocks];
    float v[kBlocks];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      row[n] = r;
      block[n] = cb;
      const int left = cols - cb * kFp4Block;  // columns from the block's first one on
      v[n] = w + n < total && lane < left ? __ldcs(x + r * ldx + cb * kFp4Block + lane) : 0.0f;
      if (++cb == cblocks) {
        cb = 0;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      if (w + n >= total) break;
      const uint32_t sb = fp4_scale_byte(__reduce_max_sync(0xffffffffu, magnitude(v[n])));
      const float next = __shfl_down_sync(0xffffffffu, v[n], 1);
      const float two[8] = {v[n], next};
      const uint32_t byte = sb == 255 ? 0u : e2m1x8(two, fp4_inverse(sb)) & 0xFFu;
      if ((lane & 1) == 0 && lane < cols - block[n] * kFp4Block)
        q[row[n] * ldq + block[n] * (kFp4Block / 2) + lane / 2] = (uint8_t)byte;
      if (lane == 0) scale[row[n] * lds + block[n]] = (uint8_t)sb;
    }
  }
}

// The transpose of a row-major matrix [cols, rows] (row stride ldx): a CTA takes 256
// columns of 32 rows, warp w the w-th block of 32 columns, lane l the l-th row, so that
// loads run along the stored rows and a block's maximum is one thread's.  The codes
// pass through shared memory and leave along the result's rows, 128 bytes each.
template <typename Word>  // how the result's rows are aligned
__global__ void __launch_bounds__(kThreads) fp4_quantize_columns_kernel(const float* __restrict__ x,
                                                                        int64_t ldx, int64_t rows, int64_t cols,
                                                                        int64_t row_tiles, int64_t tiles,
                                                                        uint8_t* q, int64_t ldq, uint8_t* scale,
                                                                        int64_t lds) {
  __shared__ __align__(16) uint8_t codes[32][128 + 16];
  __shared__ uint8_t bytes[32][8];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t r0 = t % row_tiles * 32, c0 = t / row_tiles * 256;
    const int64_t cw = c0 + 32 * w;
    float v[32];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      v[j] = r0 + lane < rows && cw + j < cols ? __ldcs(x + (cw + j) * ldx + r0 + lane) : 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) top = max(top, magnitude(v[j]));
    const uint32_t sb = fp4_scale_byte(top);
    const float inv = fp4_inverse(sb);
    uint32_t word[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = v[8 * k + j];
      word[k] = sb == 255 ? 0u : e2m1x8(e, inv);
    }
    __syncthreads();  // the tile before has left
    *reinterpret_cast<uint4*>(&codes[lane][16 * w]) = make_uint4(word[0], word[1], word[2], word[3]);
    bytes[lane][w] = (uint8_t)sb;
    __syncthreads();
    constexpr int kWords = 128 / sizeof(Word);
    const int64_t qcols = (cols + 1) / 2, scols = (cols + kFp4Block - 1) / kFp4Block;
    for (int i = threadIdx.x; i < 32 * kWords; i += kThreads) {
      const int r = i / kWords, k = i % kWords;
      const int64_t at = c0 / 2 + k * (int)sizeof(Word);
      if (r0 + r >= rows) break;
      uint8_t* o = q + (r0 + r) * ldq + at;
      if (at + (int)sizeof(Word) <= qcols) {
        *reinterpret_cast<Word*>(o) = *reinterpret_cast<const Word*>(&codes[r][k * sizeof(Word)]);
      } else {
        for (int b = 0; b < (int)sizeof(Word) && at + b < qcols; ++b) o[b] = codes[r][k * sizeof(Word) + b];
      }
    }
    const int r = threadIdx.x >> 3, k = threadIdx.x & 7;
    if (r0 + r < rows && c0 / kFp4Block + k < scols) scale[(r0 + r) * lds + c0 / kFp4Block + k] = bytes[r][k];
  }
}

// Aligned rows: eight columns a thread, four such groups at a time (their loads in
// flight together).
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                                  int64_t rows, int cols,
                                                                  const uint8_t* __restrict__ scale, int64_t lds,
                                                                  float* y, int64_t ldy) {
  griddep_wait();
  griddep_launch_dependents();
  const int groups = cols / 8;
  const int64_t total = rows * groups, step = (int64_t)gridDim.x * kThreads;
  for (int64_t i0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; i0 < total; i0 += 4 * step) {
    uint32_t eight[4], sb[4];
    int64_t at[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t i = i0 + n * step;
      eight[n] = sb[n] = 0;
      at[n] = -1;
      if (i < total) {
        const int64_t r = i / groups;
        const int c = (int)(i - r * groups) * 8;
        at[n] = r * ldy + c;
        sb[n] = __ldg(scale + r * lds + c / kFp4Block);
        eight[n] = __ldcs(reinterpret_cast<const uint32_t*>(q + r * ldq + c / 2));
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (at[n] < 0) break;
      const float s = e8m0_to_float(sb[n]);
      float v[8];
      e2m1x8_to_float(eight[n], v);
      float4* o = reinterpret_cast<float4*>(y + at[n]);
      __stcs(o, make_float4(v[0] * s, v[1] * s, v[2] * s, v[3] * s));
      __stcs(o + 1, make_float4(v[4] * s, v[5] * s, v[6] * s, v[7] * s));
    }
  }
}

// Any rows: a warp a block, a column a lane, kBlocks blocks at a time.
__global__ void __launch_bounds__(kThreads) fp4_dequantize_any_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                                      int64_t total, int cols, int cblocks,
                                                                      const uint8_t* __restrict__ scale,
                                                                      int64_t lds, float* y, int64_t ldy) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kBlocks;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kBlocks; w < total;
       w += step) {
    int64_t r = w / cblocks;
    int cb = (int)(w - r * cblocks);
    uint32_t code[kBlocks], sb[kBlocks];
    float* out[kBlocks];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      out[n] = nullptr;
      code[n] = sb[n] = 0;
      if (w + n < total && lane < cols - cb * kFp4Block) {
        const int64_t c = (int64_t)cb * kFp4Block + lane;
        out[n] = y + r * ldy + c;
        sb[n] = __ldg(scale + r * lds + cb);
        code[n] = __ldcs(q + r * ldq + c / 2);
      }
      if (++cb == cblocks) {
        cb = 0;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      float v[8];
      e2m1x8_to_float(code[n] >> (lane & 1 ? 4 : 0), v);
      if (out[n]) __stcs(out[n], v[0] * e8m0_to_float(sb[n]));
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

int launch_fp4_quantize(rtb_ctx* ctx, const float* x, int64_t ldx, int trans, int64_t rows,
                        int64_t cols, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds,
                        cudaStream_t s) {
  const char* what = "fp4_quantize launch";
  if (trans) {
    const int64_t row_tiles = (rows + 31) / 32, tiles = row_tiles * ((cols + 255) / 256);
    const int grid = grid_for(ctx, tiles, 32);
    if (aligned(q, 16) && ldq % 16 == 0)
      return run(what, fp4_quantize_columns_kernel<uint4>, grid, s, x, ldx, rows, cols, row_tiles, tiles,
                 q, ldq, scale, lds);
    if (aligned(q, 4) && ldq % 4 == 0)
      return run(what, fp4_quantize_columns_kernel<uint32_t>, grid, s, x, ldx, rows, cols, row_tiles, tiles,
                 q, ldq, scale, lds);
    return run(what, fp4_quantize_columns_kernel<uint8_t>, grid, s, x, ldx, rows, cols, row_tiles, tiles,
               q, ldq, scale, lds);
  }
  if (cols % 8 == 0 && ldx % 4 == 0 && aligned(x, 16) && ldq % 4 == 0 && aligned(q, 4)) {
    const int chunks = (int)((cols + 255) / 256);
    const int64_t total = rows * chunks;
    return run(what, fp4_quantize_kernel, grid_for(ctx, (total + 8 * kChunks - 1) / (8 * kChunks), 8), s, x,
               ldx, total, (int)cols, chunks, q, ldq, scale, lds);
  }
  const int cblocks = (int)((cols + kFp4Block - 1) / kFp4Block);
  const int64_t total = rows * cblocks;
  return run(what, fp4_quantize_any_kernel, grid_for(ctx, (total + 8 * kBlocks - 1) / (8 * kBlocks), 8), s,
             x, ldx, total, (int)cols, cblocks, q, ldq, scale, lds);
}

int launch_fp4_dequantize(rtb_ctx* ctx, const uint8_t* q, int64_t ldq, int64_t rows, int64_t cols,
                          const uint8_t* scale, int64_t lds, float* y, int64_t ldy, cudaStream_t s) {
  if (cols % 8 == 0 && ldy % 4 == 0 && aligned(y, 16) && ldq % 4 == 0 && aligned(q, 4))
    return run("fp4_dequantize launch", fp4_dequantize_kernel,
               grid_for(ctx, (rows * (cols / 8) + kThreads - 1) / kThreads, 8), s, q, ldq, rows, (int)cols,
               scale, lds, y, ldy);
  const int cblocks = (int)((cols + kFp4Block - 1) / kFp4Block);
  const int64_t total = rows * cblocks;
  return run("fp4_dequantize launch", fp4_dequantize_any_kernel,
             grid_for(ctx, (total + 8 * kBlocks - 1) / (8 * kBlocks), 8), s, q, ldq, total, (int)cols,
             cblocks, scale, lds, y, ldy);
}

}  // namespace rtb
