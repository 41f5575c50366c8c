// Loads out of 4-bit rows at any address for the product of few rows (rtb_fp4_rows.cu).
// (tests/cpp/fp4_load.cpp runs them on the host.)
#pragma once
#include <cstdint>

namespace rtb {

// The 16 bytes of block b of a row of `half` bytes at any address, by aligned words, each
// read only where one of its bytes exists.
__device__ __forceinline__ uint4 load_block(const uint8_t* row, int b, int half) {
  const uint8_t* p = row + (int64_t)16 * b;
  const int off = (int)(reinterpret_cast<uintptr_t>(p) & 3u);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p - off);
  const int left = half - 16 * b;
  uint32_t v[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = 4 * i - off < left && (i < 4 || off) ? __ldg(w + i) : 0u;
  return make_uint4(__funnelshift_r(v[0], v[1], 8 * off), __funnelshift_r(v[1], v[2], 8 * off),
                    __funnelshift_r(v[2], v[3], 8 * off), __funnelshift_r(v[3], v[4], 8 * off));
}
// The 16 aligned bytes of memory in which block b of a row of `half` bytes begins: what of
// them belongs to other rows, or to the gaps between, comes along; 0 where the row has ended.
__device__ __forceinline__ uint4 load_chunk(const uint8_t* row, int b, int half) {
  const uintptr_t at = (reinterpret_cast<uintptr_t>(row) + (int64_t)16 * b) & ~uintptr_t(15);
  return at < reinterpret_cast<uintptr_t>(row) + half ? __ldg(reinterpret_cast<const uint4*>(at))
                                                      : make_uint4(0u, 0u, 0u, 0u);
}
// The first and last rows of a matrix of n, in some 16 bytes of which (as above) lies memory
// in front of the matrix, or behind it.
inline void end_rows_of(const uint8_t* b, int64_t n, int64_t ldb, int half, int* front, int* back) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(b), end = first + (n - 1) * ldb + half;
  const int64_t before = (int64_t)((0 - first) & 15), behind = (int64_t)(end & 15);
  const int64_t f = (before + ldb - 1) / ldb, k = (behind + ldb - 1) / ldb;
  *front = (int)(f < n ? f : n);
  *back = (int)(k < n - *front ? k : n - *front);
}

}  // namespace rtb
