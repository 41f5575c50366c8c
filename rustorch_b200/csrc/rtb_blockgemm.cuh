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
  int depth;             // contraction length (4-bit operands: bytes of a row)
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
  ScaleRef scx, scy;
  int sc_bytes, sc_vec;  // 4-bit operands: scales of a row, and whether their rows are 8-byte aligned
  // MODE 0, CTA pairs: the scales as fp32, [block][row], zero past the operand
  // (launch_scale_tables)
  const float *tabx, *taby;
  int64_t pitchx, pitchy;
  int c_tma;             // CTA pairs: rows of the output leave through TMA stores
  int parts;             // CTAs that share a tile (a cluster)
  int vec_ok;            // 16-byte aligned output rows
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

// 4-bit operands: four scales, for blocks of 32 columns each, from byte 4 j on of a row of
// `bytes` that begins anywhere: aligned words of memory, `lo` and `hi`.  A word that
// holds none of the row's bytes is not read but the row's first one in its place, without
// a branch, so that many are in flight at once.
struct ScaleWord {
  uint32_t lo, hi;
};
__device__ __forceinline__ ScaleWord fp4_load_scales(const uint8_t* row, int j, int bytes) {
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 3u);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(row - off);
  ScaleWord v;
  v.lo = __ldg(w + (4 * j < bytes ? j : 0));
  v.hi = __ldg(w + (4 * j + 4 - off < bytes && off ? j + 1 : 0));
  return v;
}
// ... their four bytes; 2^0 past the row's last.
__device__ __forceinline__ uint32_t fp4_scale_word(const ScaleWord& v, const uint8_t* row, int j, int bytes) {
  const uint32_t word = __funnelshift_r(v.lo, v.hi, 8 * (uint32_t)(reinterpret_cast<uintptr_t>(row) & 3u));
  const int n = bytes - 4 * j;
  const uint32_t mask = n >= 4 ? 0xFFFFFFFFu : n > 0 ? (1u << (8 * n)) - 1u : 0u;
  return (word & mask) | (0x7F7F7F7Fu & ~mask);
}
// Instruction descriptor of kind::mxf4: e2m1 operands ([7,10), [10,12) = 1), K-major,
// N >> 3 at [17,23), scales e8m0 [23], M >> 4 at [24,29); the scales' place in their
// word, byte 0 or 2, at [4,6) (B) and [29,31) (A).
constexpr __host__ __device__ uint32_t mx4_idesc(int m, int n, int byte) {
  return ((uint32_t)byte << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
         ((uint32_t)(m >> 4) << 24) | ((uint32_t)byte << 29);
}

// Products on CTA pairs (rtb_pairgemm.cu); yvec as in rtb_blockgemm.cu.
int launch_mx(rtb_ctx* ctx, const uint8_t* X, int64_t ldx, const uint8_t* Y, int64_t ldy,
              BlockParams& p, bool fp4, cudaStream_t s);  // e8m0 scales (rtb_mxgemm.cu)
int launch_pair(rtb_ctx* ctx, int mode, bool yvec, const CUtensorMap& tmX, const CUtensorMap& tmY,
                BlockParams& p, cudaStream_t s);

}  // namespace rtb
