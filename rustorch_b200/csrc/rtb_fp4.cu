// Writing and restoring 4-bit block-scaled tensors (rtb_fp4.cuh).
//   save:    s = 2^ceil(log2(max|x| / 6)) over the block, q = e2m1(x / s)
//   restore: x' = q * s
// Both stream their operands once (4.53 bytes a value): HBM-bound.  8192 x 4096 saved in
// 24.8 us (6.1 TB/s, 94% of a copy), as its transpose in 29.5, restored in 28.4; rows off
// the 16-byte boundaries, 8192 x 4100, 36.5, 36.7 and 35 us (a block a warp and byte stores:
// 126 and 84; words shifted between the lanes 40 and, transposed, 47).
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

// 32 bytes at once (a lane's eight columns), past L1: a value is used once.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]),
               "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// Aligned rows: eight columns a lane, 256 columns a warp and kChunks such chunks at a
// time, whose loads are all in flight before the first maximum; four lanes share a
// block.  WIDE: rows on 32-byte boundaries.
constexpr int kChunks = 4;
template <bool WIDE>
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
    int64_t r = w / chunks;
    int c = (int)(w - r * chunks) * 256 + 8 * lane;
    int64_t row[kChunks];
    int col[kChunks];
    float v[kChunks][8];
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      row[n] = r;
      col[n] = w + n < total ? c : cols;  // (past the last row)
      if (col[n] < cols) {  // cols % 8 == 0
        const float* p = x + r * ldx + c;
        if (WIDE) {
          load8(p, v[n]);
        } else {
          const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
          const float4 b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
          v[n][0] = a.x; v[n][1] = a.y; v[n][2] = a.z; v[n][3] = a.w;
          v[n][4] = b.x; v[n][5] = b.y; v[n][6] = b.z; v[n][7] = b.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[n][j] = 0.0f;
      }
      c += 256;
      if (c >= chunks * 256) {
        c -= chunks * 256;
        ++r;
      }
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

// n (at most 128) bytes in shared memory, on a 4-byte boundary and with four readable ones
// behind the 128, to a row of any alignment by a warp: whole words of memory, and the bytes
// at the two ends by lanes of their own.
__device__ __forceinline__ void store_bytes(uint8_t* q, const uint8_t* from, int n, int lane) {
  const int head = (int)(-reinterpret_cast<uintptr_t>(q) & 3u);  // bytes before the first whole word
  const int words = n > head ? (n - head) >> 2 : 0;
  const uint32_t* in = reinterpret_cast<const uint32_t*>(from);
  if (lane < words)
    *reinterpret_cast<uint32_t*>(q + head + 4 * lane) = __funnelshift_r(in[lane], in[lane + 1], 8 * head);
  const int k = lane < 4 ? lane : head + 4 * words + lane - 4;
  if (lane < 8 && k < (lane < 4 && head < n ? head : n)) q[k] = from[k];
}
// A chunk's codes, four bytes a lane, from a row of any alignment: n bytes, 0 behind them.  (No word is read that holds none of them.)
__device__ __forceinline__ uint32_t load_codes(const uint8_t* q, int n, int lane) {
  const int off = (int)(reinterpret_cast<uintptr_t>(q) & 3u);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(q - off);
  const int left = n - 4 * lane;  // bytes from this lane's first one on
  if (left <= 0) return 0u;
  const uint32_t lo = __ldg(w + lane);
  const uint32_t hi = off + (left < 4 ? left : 4) > 4 ? __ldg(w + lane + 1) : 0u;
  const uint32_t v = __funnelshift_r(lo, hi, 8 * off);
  return left < 4 ? v & ((1u << (8 * left)) - 1u) : v;
}

// Any rows: chunks of 256 columns a warp, loaded a column a lane and turned through
// shared memory, so that a lane has eight columns side by side as above.
constexpr int kAny = 2;  // chunks at a time (4: 8192 x 4100 38 and 35 us for 36.5 and 35, 4096 x 1001 7.3 and 7.0 for 6.5 and 6.2)
__global__ void __launch_bounds__(kThreads) fp4_quantize_any_kernel(const float* __restrict__ x,
                                                                    int64_t ldx, int64_t total, int cols,
                                                                    int chunks, uint8_t* q, int64_t ldq,
                                                                    uint8_t* scale, int64_t lds) {
  __shared__ __align__(16) float turn[kThreads / 32][256];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  float* mine = turn[threadIdx.x >> 5];
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kAny;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kAny; w < total; w += step) {
    int64_t r = w / chunks;
    int c = (int)(w - r * chunks) * 256;
    int64_t row[kAny];
    int col[kAny];
    float v[kAny][8];
#pragma unroll
    for (int n = 0; n < kAny; ++n) {
      row[n] = r;
      col[n] = c;
      const float* p = x + r * ldx + c + lane;
      const int left = w + n < total ? cols - c - lane : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[n][j] = 32 * j < left ? __ldcs(p + 32 * j) : 0.0f;
      c += 256;
      if (c >= chunks * 256) {
        c = 0;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kAny; ++n) {
      if (w + n >= total) break;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) mine[32 * j + lane] = v[n][j];
      __syncwarp();
      float e[8];
      *reinterpret_cast<float4*>(e) = *reinterpret_cast<const float4*>(mine + 8 * lane);
      *reinterpret_cast<float4*>(e + 4) = *reinterpret_cast<const float4*>(mine + 8 * lane + 4);
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude(e[j]));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t sb = fp4_scale_byte(top);
      const uint32_t eight = e2m1x8(e, fp4_inverse(sb));
      const int left = cols - col[n];
      __syncwarp();  // the values have been read
      *reinterpret_cast<uint32_t*>(mine + lane) = sb == 255 ? 0u : eight;
      __syncwarp();
      store_bytes(q + row[n] * ldq + col[n] / 2, reinterpret_cast<const uint8_t*>(mine),
                  left < 256 ? (left + 1) / 2 : 128, lane);
      if ((lane & 3) == 0 && 8 * lane < left)
        scale[row[n] * lds + col[n] / kFp4Block + lane / 4] = (uint8_t)sb;
    }
  }
}

// The transpose of a row-major matrix [cols, rows] (row stride ldx): a CTA takes 256
// columns of 32 rows, warp w the w-th block of 32 columns, lane l the l-th row, so that
// loads run along the stored rows and a block's maximum is one thread's.  The codes
// pass through shared memory and leave along the result's rows, 128 bytes each.  Five
// CTAs on an SM: 8192 x 4096 in 29.5 us; four 32.3, three 37.8, six, whose registers do
// not hold the 32 values, 37.
template <bool VEC>  // the result's rows are on 16-byte boundaries
__global__ void __launch_bounds__(kThreads, 5) fp4_quantize_columns_kernel(const float* __restrict__ x,
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
    const int64_t qcols = (cols + 1) / 2, scols = (cols + kFp4Block - 1) / kFp4Block;
    if (VEC) {
      const int r = threadIdx.x >> 3, k = threadIdx.x & 7;
      const int64_t at = c0 / 2 + 16 * k;
      if (r0 + r < rows) {
        uint8_t* o = q + (r0 + r) * ldq + at;
        if (at + 16 <= qcols) {
          *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(&codes[r][16 * k]);
        } else {
          for (int b = 0; b < 16 && at + b < qcols; ++b) o[b] = codes[r][16 * k + b];
        }
      }
    } else {
      const int n = qcols - c0 / 2 < 128 ? (int)(qcols - c0 / 2) : 128;  // bytes of a row here
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = w + 8 * i;
        if (r0 + r >= rows) break;
        store_bytes(q + (r0 + r) * ldq + c0 / 2, codes[r], n, lane);
      }
    }
    const int r = threadIdx.x >> 3, k = threadIdx.x & 7;
    if (r0 + r < rows && c0 / kFp4Block + k < scols) scale[(r0 + r) * lds + c0 / kFp4Block + k] = bytes[r][k];
  }
}

// Aligned rows, the same way: kChunks chunks of 256 columns a warp.
template <bool WIDE>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                                  int64_t total, int cols, int chunks,
                                                                  const uint8_t* __restrict__ scale, int64_t lds,
                                                                  float* y, int64_t ldy) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kChunks;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kChunks; w < total;
       w += step) {
    int64_t r = w / chunks;
    int c = (int)(w - r * chunks) * 256 + 8 * lane;
    float* out[kChunks];
    uint32_t eight[kChunks], sb[kChunks];
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      out[n] = nullptr;
      eight[n] = sb[n] = 0;
      if (w + n < total && c < cols) {  // cols % 8 == 0
        out[n] = y + r * ldy + c;
        sb[n] = __ldg(scale + r * lds + c / kFp4Block);
        eight[n] = __ldcs(reinterpret_cast<const uint32_t*>(q + r * ldq + c / 2));
      }
      c += 256;
      if (c >= chunks * 256) {
        c -= chunks * 256;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      if (!out[n]) continue;
      const float s = e8m0_to_float(sb[n]);
      float v[8];
      e2m1x8_to_float(eight[n], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= s;
      if (WIDE) {
        store8(out[n], v);
      } else {
        float4* o = reinterpret_cast<float4*>(out[n]);
        __stcs(o, make_float4(v[0], v[1], v[2], v[3]));
        __stcs(o + 1, make_float4(v[4], v[5], v[6], v[7]));
      }
    }
  }
}

// Any rows: chunks of 256 columns a warp, turned through shared memory.
__global__ void __launch_bounds__(kThreads) fp4_dequantize_any_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                                      int64_t total, int cols, int chunks,
                                                                      const uint8_t* __restrict__ scale,
                                                                      int64_t lds, float* y, int64_t ldy) {
  __shared__ __align__(16) float turn[kThreads / 32][256];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  float* mine = turn[threadIdx.x >> 5];
  const int64_t step = (int64_t)gridDim.x * (kThreads / 32) * kAny;
  for (int64_t w = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kAny; w < total; w += step) {
    int64_t r = w / chunks;
    int c = (int)(w - r * chunks) * 256;
    int64_t row[kAny];
    int col[kAny];
    uint32_t eight[kAny], sb[kAny];
#pragma unroll
    for (int n = 0; n < kAny; ++n) {
      row[n] = r;
      col[n] = c;
      const int left = w + n < total ? cols - c : 0;
      eight[n] = load_codes(q + r * ldq + c / 2, left < 256 ? (left + 1) / 2 : 128, lane);
      sb[n] = 8 * lane < left ? __ldg(scale + r * lds + c / kFp4Block + lane / 4) : 0u;
      c += 256;
      if (c >= chunks * 256) {
        c = 0;
        ++r;
      }
    }
#pragma unroll
    for (int n = 0; n < kAny; ++n) {
      if (w + n >= total) break;
      const float s = e8m0_to_float(sb[n]);
      float v[8];
      e2m1x8_to_float(eight[n], v);
      __syncwarp();
      *reinterpret_cast<float4*>(mine + 8 * lane) = make_float4(v[0] * s, v[1] * s, v[2] * s, v[3] * s);
      *reinterpret_cast<float4*>(mine + 8 * lane + 4) = make_float4(v[4] * s, v[5] * s, v[6] * s, v[7] * s);
      __syncwarp();
      float* out = y + row[n] * ldy + col[n] + lane;
      const int left = cols - col[n] - lane;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (32 * j < left) __stcs(out + 32 * j, mine[32 * j + lane]);
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
    const bool vec = aligned(q, 16) && ldq % 16 == 0;
    return run(what, vec ? fp4_quantize_columns_kernel<true> : fp4_quantize_columns_kernel<false>, grid, s, x, ldx,
               rows, cols, row_tiles, tiles, q, ldq, scale, lds);
  }
  const int chunks = (int)((cols + 255) / 256);
  const int64_t total = rows * chunks;
  if (cols % 8 == 0 && ldx % 4 == 0 && aligned(x, 16) && ldq % 4 == 0 && aligned(q, 4)) {
    const bool wide = aligned(x, 32) && ldx % 8 == 0;
    return run(what, wide ? fp4_quantize_kernel<true> : fp4_quantize_kernel<false>,
               grid_for(ctx, (total + 8 * kChunks - 1) / (8 * kChunks), 8), s, x, ldx, total, (int)cols, chunks,
               q, ldq, scale, lds);
  }
  return run(what, fp4_quantize_any_kernel, grid_for(ctx, (total + 8 * kAny - 1) / (8 * kAny), 8), s, x, ldx,
             total, (int)cols, chunks, q, ldq, scale, lds);
}

int launch_fp4_dequantize(rtb_ctx* ctx, const uint8_t* q, int64_t ldq, int64_t rows, int64_t cols,
                          const uint8_t* scale, int64_t lds, float* y, int64_t ldy, cudaStream_t s) {
  const int chunks = (int)((cols + 255) / 256);
  const int64_t total = rows * chunks;
  if (cols % 8 == 0 && ldy % 4 == 0 && aligned(y, 16) && ldq % 4 == 0 && aligned(q, 4)) {
    const bool wide = aligned(y, 32) && ldy % 8 == 0;
    return run("fp4_dequantize launch", wide ? fp4_dequantize_kernel<true> : fp4_dequantize_kernel<false>,
               grid_for(ctx, (total + 8 * kChunks - 1) / (8 * kChunks), 8), s, q, ldq, total, (int)cols, chunks,
               scale, lds, y, ldy);
  }
  return run("fp4_dequantize launch", fp4_dequantize_any_kernel,
             grid_for(ctx, (total + 8 * kAny - 1) / (8 * kAny), 8), s, q, ldq, total, (int)cols, chunks, scale,
             lds, y, ldy);
}

}  // namespace rtb
