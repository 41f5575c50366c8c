// The products of rtb_blockgemm.cu on CTA pairs (tcgen05 cta_group::2): a
// persistent kernel whose two CTAs compute one 256 x 256 tile.  Each CTA loads
// its own 128 X rows and half of the 256 Y columns, the pair's tensor cores
// read both halves, and each CTA's TMEM holds its 128 rows x 256 columns of
// the accumulator, twice.
//
// Why pairs: a stage of 128 contraction bytes takes 512 clocks of MMAs and 32
// KB of loads per SM, 64 bytes a clock; one CTA alone needs 48 KB for a 128 x
// 256 tile in the same time, more than L2 feeds an SM.
//
// Promotion: after every 128 contraction elements the epilogue warps add the
// finished partial sum into registers (128 a thread: 8 warps, each 32 TMEM
// lanes x 128 columns) while the MMAs fill the other half of TMEM.  In MODE 0
// that is 32768 multiply-adds per 512 clocks of MMAs, half of the SM's fp32
// lanes; packed f32x2 instructions halve the issue slots.
//
// Measured: MODE 0 (f32 scales, one for each 128 columns) 8192 x 4096 x 8192 in 381
// us alone, 392 in a loop, 1400 TFLOP/s, bound by the epilogue's chain of barrier,
// TMEM loads and adds (about 1150 clocks a block); with a scale for each column 547,
// its epilogue multiplies twice.  MODE 1 8192 x 4096 x 4096 in 633 us alone, 707 to
// 733 in a loop (the power cap), 60 of them for its operands: 1.1 to 1.4 PFLOP/s of
// bf16 MMAs, bound by them.  Outputs that TMA cannot store (N or ldc off a multiple of 4)
// leave by scalar stores: 8192 x 4097 x 8192 777 us against 547, MODE 1 8192 x 4097
// x 4096 849 against 707.
//
// Roles (warps of each CTA): 0, 2, 3 TMA producers; 1 TMEM allocation, and in the
// pair's first CTA the MMA issue for both; 4..11 epilogue (lanes 32 (w % 4)..,
// columns 128 ((w - 4) / 4)..).  The first warpgroup hands registers to the
// epilogue's two (384 threads x 168 at launch = 128 x (40 + 232 + 232)): at 168
// the accumulators spill.  Barriers: `full` and `tempty` live in the
// first CTA (the producers' bytes and the epilogues' arrivals of both CTAs),
// `empty` and `tfull` in each (the MMA's commits go to both).
#include "rtb_pair.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 384;
constexpr int kTile = 256;
constexpr int kChunk = 128 * 32 * 4;  // a staged 128 x 32 fp32 piece of the output
constexpr int kSmemBytes = 232448;

template <int MODE, bool YVEC>
struct PairCfg {
  static constexpr int kDepth = MODE == 0 ? 128 : 64;
  static constexpr int kYPieces = MODE == 0 ? 1 : 3;
  static constexpr int kStageBytes = 16384 * (1 + kYPieces);
  // two staging chunks; the column scales take a stage's place
  static constexpr int kStages = MODE == 0 ? (YVEC ? 5 : 6) : 3;
  static constexpr int kPerUnit = 128 / kDepth;
  static_assert(1024 + kStages * kStageBytes + 2 * kChunk + 512 + (YVEC ? 8192 : 0) <= kSmemBytes,
                "shared memory");
};

// The scales of both operands as fp32 tables [block][row]: the epilogue then
// takes a block's scales of 32 rows with one coalesced, unconditional load that
// nothing has to decode (a conditional load of whatever type the caller has
// waits for its value where the branches meet: 1000 clocks every time).
// blockIdx.z picks the operand; rows [rows, pitch) and blocks [units, blocks)
// are zero.  32 x 32 tiles through shared memory.
struct TableSide {
  ScaleRef s;
  int64_t rows, pitch;
  float* out;
};
__global__ void __launch_bounds__(256) scale_table_kernel(const TableSide x, const TableSide y,
                                                          int units, int blocks) {
  __shared__ float t[32][33];
  griddep_wait();
  griddep_launch_dependents();
  const TableSide& d = blockIdx.z ? y : x;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int k0 = blockIdx.y * 32;
  for (int64_t r0 = (int64_t)blockIdx.x * 32; r0 < d.pitch; r0 += (int64_t)gridDim.x * 32) {
    __syncthreads();
    for (int i = w; i < 32; i += 8) {
      const int64_t r = r0 + i;
      const int k = k0 + lane;
      float v = 0.0f;
      if (r < d.rows && k < units)
        v = scale_value(d.s, load_scale(d.s, (r >> d.s.row_shift) * d.s.ld_row + k * d.s.ld_col));
      t[i][lane] = v;
    }
    __syncthreads();
    for (int i = w; i < 32; i += 8)
      if (k0 + i < blocks && r0 + lane < d.pitch)
        d.out[(int64_t)(k0 + i) * d.pitch + r0 + lane] = t[lane][i];
  }
}

template <int MODE>
__device__ __forceinline__ void mma_pair_e(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                           uint32_t acc) {
  if (MODE == 0) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
  }
}
// Tiles in bands of 8 X tiles, so that the 74 pairs' working set is about
// square.
__device__ __forceinline__ void pair_tile(const BlockParams& p, int t, int& tx, int& ty) {
  const int band = 8 * p.tiles_y;
  const int g = t / band;
  int h = p.tiles_x - 8 * g;
  h = h < 8 ? h : 8;
  const int r = t - g * band;
  tx = 8 * g + r % h;
  ty = r / h;
}

template <int MODE, bool YVEC>
__global__ void __launch_bounds__(kThreads, 1)
    pair_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmY,
                     const __grid_constant__ CUtensorMap tmC, const BlockParams p) {
  using C = PairCfg<MODE, YVEC>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* staging = base + S * C::kStageBytes;  // 2 x kChunk, 1024-byte aligned
  uint8_t* tail = staging + 2 * kChunk;
  uint64_t* full = reinterpret_cast<uint64_t*>(tail);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sy_s = reinterpret_cast<float*>(tail + 512);  // YVEC: [2][4 blocks][256]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmY);
    if (p.c_tma) tma_prefetch_desc(&tmC);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers and TMEM are ready
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
  const int tiles = p.tiles_x * p.tiles_y;
  const int nst = p.stages_total;
  const int units = (nst + C::kPerUnit - 1) / C::kPerUnit;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp != 1 && lane == 0) {
      // three producers take the stages in turn: one thread's wait and issue of a
      // stage's loads takes about as long as its MMAs
      const int turn = warp ? warp - 1 : 0;
      int q = 0;
      const uint32_t bytes = 2u * 16384u * (uint32_t)(1 + (MODE == 0 ? 1 : p.pieces));
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int tx, ty;
        pair_tile(p, t, tx, ty);
        const int x0 = tx * kTile + 128 * (int)rank, y0 = ty * kTile + 128 * (int)rank;
        for (int i = 0; i < nst; ++i, q = q == 2 ? 0 : q + 1) {
          if (q != turn) {
            if (++s == S) { s = 0; ph ^= 1; }
            continue;
          }
          if (!(ok = mbar_wait_bounded(&empty[s], ph ^ 1, abort_flag, p.err, DEV_TIMEOUT_EMPTY,
                                  p.timeout_ns)))
            break;
          const uint32_t st = smem_u32(base + s * C::kStageBytes);
          // the first CTA expects both CTAs' bytes; the second's may land first
          const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
          if (MODE == 0) {
            tma_load_2d_pair(st, &tmX, bar, i * 128, x0);
            tma_load_2d_pair(st + 16384, &tmY, bar, i * 128, y0);
          } else {
            for (int b = 0; b < 2; ++b)
              tma_load_2d_pair(st + 8192 * b, &tmX, bar, x0 + 64 * b, 64 * i);
            for (int q = 0; q < p.pieces; ++q)
              for (int b = 0; b < 2; ++b)
                tma_load_2d_pair(st + 16384 * (1 + q) + 8192 * b, &tmY, bar, y0 + 64 * b,
                                 (int)(q * p.piece_rows) + 64 * i);
          }
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t id = block_idesc(MODE, 256, 256);
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        int got = 0;
        if (lane == 0) got = mbar_wait_bounded(bar, parity, abort_flag, p.err, code, p.timeout_ns);
        return __shfl_sync(0xffffffffu, got, 0) != 0;
      };
      int s = 0, g = 0;
      uint32_t ph = 0;
      bool ok = true;
      // Lane 0: whether the next stage's operands and the next accumulator were
      // found ready before this stage's last MMA.  A wait costs this warp 200
      // clocks of latency even when its barrier is complete, so the tests run
      // behind the MMAs issued before them.
      int next_full = 0, next_empty = 0;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int i = 0;
        for (int u = 0; u < units && ok; ++u, ++g) {
          const int b = g & 1;
          const uint32_t d = tmem + (uint32_t)(b * 256);
          for (int j = 0; j < C::kPerUnit && i < nst; ++j, ++i) {
            if (!__shfl_sync(0xffffffffu, next_full, 0) &&
                !(ok = wait(&full[s], ph, DEV_TIMEOUT_FULL)))
              break;
            if (j == 0 && !__shfl_sync(0xffffffffu, next_empty, 0) &&
                !(ok = wait(&tempty[b], ((g >> 1) & 1) ^ 1, DEV_TIMEOUT_TMEM_EMPTY)))
              break;
            tc_fence_after();
            const int sn = s + 1 == S ? 0 : s + 1;
            const uint32_t phn = s + 1 == S ? ph ^ 1u : ph;
            const bool last = j + 1 == C::kPerUnit || i + 1 == nst;
            const uint32_t xa = smem_u32(base + s * C::kStageBytes), ya = xa + 16384;
            if (MODE == 0) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (k == 2 && lane == 0) {
                  next_full = mbar_test_wait(&full[sn], phn);
                  next_empty = mbar_test_wait(&tempty[b ^ 1], (((g + 1) >> 1) & 1) ^ 1);
                }
                mma_pair_e<0>(d, umma_desc(xa + 32 * k, 16, 1024, kLayoutSW128),
                              umma_desc(ya + 32 * k, 16, 1024, kLayoutSW128), id, k > 0);
              }
            } else {
              for (int q = p.pieces - 1; q >= 0; --q) {
                if (q == 0 && lane == 0) {
                  next_full = mbar_test_wait(&full[sn], phn);
                  if (last) next_empty = mbar_test_wait(&tempty[b ^ 1], (((g + 1) >> 1) & 1) ^ 1);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_pair_e<1>(d, umma_desc(xa + 2048 * k, 8192, 1024, kLayoutSW128),
                                umma_desc(ya + 16384 * q + 2048 * k, 8192, 1024, kLayoutSW128), id,
                                j > 0 || k > 0 || q < p.pieces - 1);
              }
            }
            commit_pair_e(&empty[s]);
            if (last) commit_pair_e(&tfull[b]);
            s = sn;
            ph = phn;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int row = 32 * (warp & 3) + lane;
    const int half = (warp - 4) >> 2;
    const int et = threadIdx.x - 128 - 128 * half;  // 0..127 within the half
    const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)(128 * half);
    const uint32_t tempty0[2] = {map_rank(smem_u32(&tempty[0]), 0), map_rank(smem_u32(&tempty[1]), 0)};
    uint8_t* stg = staging + half * kChunk;
    int g = 0;
    int quad = 0;  // quads of blocks so far, over all tiles: the buffer of a quad's column scales
    bool ok = true;
    for (int t = pair; t < tiles; t += pairs) {
      int tx, ty;
      pair_tile(p, t, tx, ty);
      const int64_t x = (int64_t)tx * kTile + 128 * rank + row;
      const int64_t y0 = (int64_t)ty * kTile + 128 * half;
      unsigned long long acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0ull;
      // this thread's scales of the next four blocks, loaded four blocks ahead
      const float* px = MODE == 0 ? p.tabx + x : nullptr;
      const float* py = MODE == 0 ? p.taby + (YVEC ? y0 + et : 2 * ty + half) : nullptr;
      float nx[4] = {}, ny[4] = {};
      if (MODE == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          nx[i] = __ldg(px + i * p.pitchx);
          ny[i] = __ldg(py + i * p.pitchy);
        }
      }
      for (int v = 0; v < units; v += 4, ++quad) {
        float sc[4];
        float* sy = sy_s + 1024 * (quad & 1) + 128 * half;
        if (MODE == 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sc[i] = YVEC ? nx[i] : nx[i] * ny[i];
            if (YVEC) sy[256 * i + et] = ny[i];
          }
          px += 4 * p.pitchx;
          py += 4 * p.pitchy;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            nx[i] = __ldg(px + i * p.pitchx);
            ny[i] = __ldg(py + i * p.pitchy);
          }
          // Two buffers, taken in turn across tiles too: a buffer is written again
          // two quads later, behind the barrier of the quad between, which every
          // reader of this one has passed.  (The stores of a finished tile need
          // have no barrier.)
          if (YVEC) named_bar_sync(1 + half, 128);
        }
        const int n = units - v < 4 ? units - v : 4;
#pragma unroll 1
        for (int i = 0; i < n; ++i, ++g) {
          const int b = g & 1;
          if (ok) {
            int got = 0;
            if (lane == 0)
              got = mbar_wait_bounded(&tfull[b], (g >> 1) & 1, abort_flag, p.err,
                                                    DEV_TIMEOUT_TMEM_FULL, p.timeout_ns);
            ok = __shfl_sync(0xffffffffu, got, 0) != 0;
          }
          tc_fence_after();
          float f = 1.0f;
          if (MODE == 0) {
            f = sc[0];
            sc[0] = sc[1];
            sc[1] = sc[2];
            sc[2] = sc[3];
          }
          const unsigned long long s2 = pack2(f, f);
          const uint32_t ta = t_lane + (uint32_t)(256 * b);
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 64 columns at a time
            uint32_t r[4][16];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld_x16(ta + 64 * h + 16 * c, r[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_wait_x16(r[c]);
            if (h == 1) {  // the last of this buffer is in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) arrive_pair(tempty0[b]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const unsigned long long w = pack2(r[c][2 * j], r[c][2 * j + 1]);
                unsigned long long& a = acc[32 * h + 8 * c + j];
                if (MODE == 1) a = add2(a, w);
                else if (YVEC)
                  a = fma2(mul2(w, s2),
                           *reinterpret_cast<const unsigned long long*>(sy + 256 * i + 64 * h +
                                                                        16 * c + 2 * j), a);
                else a = fma2(w, s2, a);
              }
          }
        }
      }
      // the finished rows, 32 columns at a time
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t yc = y0 + 32 * c;
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 f = unpack2(acc[16 * c + j]);
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += yc + j < p.ycols ? __ldg(p.bias + yc + j) : 0.0f;
        }
        float* o = p.out + x * p.ldo + yc;
        if (p.accumulate && x < p.xrows) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (yc + j < p.ycols) v[j] += o[j];
        }
        activate_n<32>(v, p.act);
        if (p.c_tma) {
          // the store before has read the chunk (its issuing thread waits)
          if (et == 0) bulk_wait_group_read<0>();
          named_bar_sync(1 + half, 128);
          const uint32_t dst = smem_u32(stg) + row * 128;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            sts128(dst + ((j ^ (row & 7)) << 4),
                   make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
          fence_proxy_async_smem();
          named_bar_sync(1 + half, 128);
          const int xs = tx * kTile + 128 * (int)rank;
          if (et == 0 && yc < p.ycols && xs < p.xrows) {
            tma_store_2d(&tmC, stg, (int)yc, xs);
            bulk_commit_group();
          }
        } else if (x < p.xrows) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (yc + j < p.ycols) o[j] = v[j];
        }
      }
    }
    if (p.c_tma && et == 0) bulk_wait_group<0>();
  }

  // ------------------------------------------------------------ teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // copies in flight land before the CTA's shared memory is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    __syncthreads();
  }
  cluster_sync_all();  // no commit or arrival for this CTA is under way any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

template <int MODE, bool YVEC>
int launch(rtb_ctx* ctx, const CUtensorMap& tmX, const CUtensorMap& tmY, BlockParams& p,
           cudaStream_t s) {
  using C = PairCfg<MODE, YVEC>;
  auto* k = pair_gemm_kernel<MODE, YVEC>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return cuda_status(e, "pair gemm smem attribute");
  p.tiles_x = (int)((p.xrows + kTile - 1) / kTile);
  p.tiles_y = (int)((p.ycols + kTile - 1) / kTile);
  p.stages_total = (p.depth + C::kDepth - 1) / C::kDepth;
  const int64_t tiles = (int64_t)p.tiles_x * p.tiles_y;
  if (tiles > INT32_MAX / 2) return set_error(RTB_E_UNSUPPORTED, "pair gemm: too many tiles");
  CUtensorMap tmC = tmX;
  // (A TMA store clips a box at the tensor's columns in units of 16 bytes: up to three
  // floats behind a row whose length is no multiple of 4 would be overwritten.  A test
  // for each chunk makes the epilogue with column scales spill: 8192 x 4096 x 8192 547
  // -> 596 us.)
  p.c_tma = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && p.ldo % 4 == 0 && p.ycols % 4 == 0;
  if (p.c_tma) {
    const int st = make_tmap_2d(&tmC, p.out, (uint64_t)p.ycols, (uint64_t)p.xrows, (uint64_t)p.ldo,
                                32, 128, false);
    if (st) return st;
  }
  const int64_t pairs = ctx->sm_count / 2 < tiles ? ctx->sm_count / 2 : tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  clear_stale_cuda_error();
  e = cudaLaunchKernelEx(&cfg, k, tmX, tmY, tmC, (const BlockParams)p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "pair gemm launch");
}

}  // namespace

int launch_pair(rtb_ctx* ctx, int mode, bool yvec, const CUtensorMap& tmX, const CUtensorMap& tmY,
                BlockParams& p, cudaStream_t s) {
  if (mode == 0) {
    const int64_t units = (p.depth + 127) / 128, blocks = table_blocks(units);
    TableSide x = {p.scx, p.xrows, (p.xrows + kTile - 1) / kTile * kTile, nullptr};
    TableSide y = {p.scy, p.ycols, (p.ycols + kTile - 1) / kTile * kTile, nullptr};
    if (!yvec) {  // one entry for each 128 columns
      y.s.row_shift = 0;
      y.rows = (p.ycols + 127) / 128;
      y.pitch /= 128;
    }
    float* ws = nullptr;
    int st = ws_alloc(ctx, (void**)&ws, (size_t)((x.pitch + y.pitch) * blocks) * sizeof(float), s);
    if (st) return st;
    x.out = ws;
    y.out = ws + x.pitch * blocks;
    const int64_t longer = x.pitch > y.pitch ? x.pitch : y.pitch;
    const int64_t gx = (longer + 31) / 32;
    clear_stale_cuda_error();
    cudaError_t e = launch_pdl(scale_table_kernel,
                               dim3((unsigned)(gx < 512 ? gx : 512), (unsigned)((blocks + 31) / 32), 2),
                               dim3(256), 0, s, (const TableSide)x, (const TableSide)y, (int)units,
                               (int)blocks);
    if (e == cudaSuccess) e = cudaGetLastError();
    st = e == cudaSuccess ? RTB_OK : cuda_status(e, "scale table launch");
    p.tabx = x.out;
    p.taby = y.out;
    p.pitchx = x.pitch;
    p.pitchy = y.pitch;
    if (st == RTB_OK)
      st = yvec ? launch<0, true>(ctx, tmX, tmY, p, s) : launch<0, false>(ctx, tmX, tmY, p, s);
    ws_free(ws, s);
    return st;
  }
  return launch<1, false>(ctx, tmX, tmY, p, s);
}

}  // namespace rtb
