// Shared by the block-scaled product kernels (rtb_blockgemm.cu: one CTA a tile;
// rtb_pairgemm.cu, rtb_mxgemm.cu: two CTAs a tile): parameters, scales, instruction
// descriptors.
#pragma once
#include <cuda.h>

#include "rtb_act.cuh"
#include "rtb_f32x2.cuh"
#include "rtb_fp8.cuh"
#include "rtb_internal.h"
#include "rtb_ptx.cuh"

namespace rtb {

struct BlockParams {
  int64_t xrows, ycols;  // output extents along X and Y
  int depth;             // contraction length
  int stages_total;      // ceil(depth / kDepth)
  int tiles_x, tiles_y;
  float* out;            // row-major, leading dimension ldo
  int64_t ldo;
  int swap;              // 0: X rows are the output's rows; 1: its columns (few rows)
  const float* bias;     // per output column
  int act;
  int accumulate;
  int pieces;            // MODE 1
  int64_t piece_rows;    // MODE 1: contraction rows between Y's pieces
  ScaleRef scx, scy;     // MODE 0
  // MODE 0, CTA pairs: the scales as fp32, [block][row], zero past the operand
  // (launch_scale_tables)
  const float *tabx, *taby;
  int64_t pitchx, pitchy;
  int c_tma;             // CTA pairs: rows of the output leave through TMA stores
  int parts;             // CTAs that share a tile (a cluster)
  int vec_ok;            // 16-byte aligned output rows and bias
  int* err;
  unsigned long long timeout_ns;
};

// A scale as it lies in memory, and its value.  They are apart so that a load
// can be issued blocks ahead of its use: decoding at the load waits for it
// (451 -> 364 us on 8192 x 4096 x 8192, float scales).
__device__ __forceinline__ uint32_t load_scale(const ScaleRef& s, int64_t i) {
  return s.is_f32 ? __ldg(static_cast<const uint32_t*>(s.p) + i)
                  : (uint32_t)__ldg(static_cast<const uint8_t*>(s.p) + i);
}
__device__ __forceinline__ float scale_value(const ScaleRef& s, uint32_t raw) {
  return s.is_f32 ? __uint_as_float(raw) : e8m0_to_float(raw);
}

// Instruction descriptor, fp32 accumulate, dense.  Bits: D format [4,6) = 1;
// A format [7,10), B format [10,13): e4m3 = 0 (kind::f8f6f4), bf16 = 1
// (kind::f16); A MN-major [15], B MN-major [16]; N >> 3 [17,23); M >> 4 [24,29).
constexpr __host__ __device__ uint32_t block_idesc(int mode, int m, int n) {
  return (1u << 4) | (mode == 0 ? 0u : (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16)) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Waits for the TMEM loads issued so far; the registers go through the
// statement, so that their uses stay behind it.
__device__ __forceinline__ void tmem_wait_x16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// Blocks in a scale table of `units` blocks: whole quads and one more, so that
// a quad can be loaded ahead without a check.
inline int64_t table_blocks(int64_t units) { return (units + 3) / 4 * 4 + 4; }

// Products on CTA pairs (rtb_pairgemm.cu); yvec as in rtb_blockgemm.cu.
int launch_mx(rtb_ctx* ctx, const uint8_t* X, int64_t ldx, const uint8_t* Y, int64_t ldy,
              BlockParams& p, cudaStream_t s);  // e8m0 scales (rtb_mxgemm.cu)
int launch_pair(rtb_ctx* ctx, int mode, bool yvec, const CUtensorMap& tmX, const CUtensorMap& tmY,
                BlockParams& p, cudaStream_t s);

}  // namespace rtb
