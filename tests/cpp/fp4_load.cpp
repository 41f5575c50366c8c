// The loads of the 4-bit product of few rows (csrc/rtb_fp4_load.cuh) on the host: every
// address they read, and every byte they return, for matrices at each byte of 16 with rows
// of every length and gap.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

struct uint4 {
  uint32_t x, y, z, w;
};
static uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }
static uint32_t __funnelshift_r(uint32_t lo, uint32_t hi, uint32_t s) {
  return (uint32_t)(((uint64_t)hi << 32 | lo) >> (s & 31));
}
static const uint8_t *g_front, *g_end;  // the matrix; loads may touch `g_slack` bytes around it
static int g_slack, g_bad, g_misaligned;
template <typename T>
static T __ldg(const T* p) {
  const uint8_t* b = reinterpret_cast<const uint8_t*>(p);
  if (b < g_front - g_slack || b + sizeof(T) > g_end + g_slack) ++g_bad;
  if (b >= g_end || b + sizeof(T) <= g_front) ++g_bad;  // none of the matrix's bytes
  if (reinterpret_cast<uintptr_t>(b) % sizeof(T)) ++g_misaligned;
  T v;
  memcpy(&v, p, sizeof(T));
  return v;
}
#define __device__
#define __forceinline__ inline
#include "../../rustorch_b200/csrc/rtb_fp4_load.cuh"

int main() {
  std::vector<uint8_t> memory(1 << 16);
  for (size_t i = 0; i < memory.size(); ++i) memory[i] = (uint8_t)(i * 131 + (i >> 8) * 17 + 1);
  uint8_t* base = memory.data() + (64 - reinterpret_cast<uintptr_t>(memory.data()) % 64);
  int wrong = 0;
  long calls = 0;
  for (int offset = 0; offset < 16; ++offset)
    for (int half = 1; half <= 50; ++half)
      for (int gap = 0; gap <= 17; ++gap)
        for (int rows = 1; rows <= 20; rows += rows < 3 ? 1 : 17) {
          const uint8_t* front = base + 64 + offset;
          const int64_t ld = half + gap;
          g_front = front;
          g_end = front + (rows - 1) * ld + half;
          const int blocks = (half + 15) / 16;
          int before, behind;
          rtb::end_rows_of(front, rows, ld, half, &before, &behind);
          if (before < 0 || behind < 0 || before + behind > rows) ++wrong;
          for (int r = 0; r < rows; ++r) {
            const uint8_t* row = front + r * ld;
            const bool whole = r >= before && r < rows - behind;  // loaded by 16 bytes
            for (int b = 0; b <= blocks + 1; ++b) {
              ++calls;
              uint8_t got[16];
              if (whole) {
                g_slack = 0;
                const uint4 c = rtb::load_chunk(row, b, half);
                memcpy(got, &c, 16);
                const uint8_t* at = reinterpret_cast<const uint8_t*>((reinterpret_cast<uintptr_t>(row) + 16 * b) & ~uintptr_t(15));
                for (int i = 0; i < 16; ++i)
                  if (at + i >= row && at + i < row + half && got[i] != at[i]) ++wrong;
              }
              if (b >= blocks) continue;
              g_slack = 3;  // words, each of which holds some of the row's bytes
              const uint4 q = rtb::load_block(row, b, half);
              memcpy(got, &q, 16);
              for (int i = 0; i < 16 && 16 * b + i < half; ++i)
                if (got[i] != row[16 * b + i]) ++wrong;
            }
          }
        }
  if (g_bad || g_misaligned || wrong) {
    printf("%d loads out of the matrix, %d misaligned, %d wrong bytes of %ld calls\n", g_bad, g_misaligned, wrong, calls);
    return 1;
  }
  printf("fine\n");
  return 0;
}
