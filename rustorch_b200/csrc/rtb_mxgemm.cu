// C[m,n] = act( sum_k A[m,k] 2^ea B[n,k] 2^eb + bias[n] ) for e4m3 operands with
// power-of-two (e8m0) block scales, on CTA pairs with the tensor core's own block
// scaling (tcgen05 kind::mxf8f6f4, one scale for 32 contraction elements; a
// block of 128 gives its scale to four of them).
//
// The scales enter inside the MMA, so a partial sum has to leave the tensor core
// only for the accumulation's sake, every 1024 or 2048 elements (the tensor core
// does not round each addition to nearest: the error grows with the chain, 9e-8
// relative after 32 steps) instead of every 128: the epilogue's chain of barrier,
// TMEM loads and adds, 1150 clocks against 512 of MMAs in rtb_pairgemm.cu, is out
// of the way.
//
// Tile 256 x 256 with one accumulator or 256 x 224 with two (the scales need
// columns of TMEM too), whichever takes less time in whole rounds of the pairs.
// Roles (warps of each CTA): 0, 2, 3 TMA producers; 1 TMEM allocation, and in the
// pair's first CTA the issue for both; 4..11 epilogue (lanes 32 (w % 4).., one
// half of the columns).
//
// Scales: a kernel before lays them out once per call as 512-byte groups of 128
// rows for each block (row r: the 32-bit word at 16 (r % 32) + 4 (r / 32), its
// byte repeated four times).  A stage's groups (X: one, Y: two) come with its
// operands by TMA, and tcgen05.cp spreads them over the TMEM lanes: word column r
// / 32, lane r % 32, the same in all four lane quarters.  (Two warps writing the
// groups into shared memory: 522 us on 8192 x 4096 x 8192, every stage waiting
// for their loads and fences.)
//
// Measured: 8192 x 4096 x 8192 in 212 us alone, 262 to 273 in a loop (the power cap),
// 2.1 PFLOP/s; 8192 x 8192 x 1024 in 97 and 105.  Outputs that TMA cannot store (N or
// ldc off a multiple of 4) leave by scalar stores, 32 rows an instruction: 8192 x 4097
// x 8192 429 us.
#include "rtb_pair.cuh"

namespace rtb {

namespace {

constexpr int kThreads = 384;
constexpr int kTileX = 256;
constexpr int kStages = 5;
constexpr int kStageBytes = 16384 + 16384 + 2048;  // X, Y (half of the tile's rows), scales
constexpr int kChunk = 128 * 16 * 4;               // a staged 128 x 16 fp32 piece of the output
constexpr int kBufs = 3;                           // staging chunks of an epilogue half
constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 2 * kBufs * kChunk + 512 + 1024;
constexpr uint32_t kScaleCol = 448;                // TMEM: two buffers of 4 + 8 columns
static_assert(kSmemBytes <= 232448, "shared memory");

// Instruction descriptor of kind::mxf8f6f4: scale ids 0 ([4,6) and [29,31)),
// e4m3 operands, K-major, N >> 3 at [17,23), scales e8m0 [23], M >> 4 at [24,29).
constexpr __host__ __device__ uint32_t mx_idesc(int tn) {
  return ((uint32_t)(tn >> 3) << 17) | (1u << 23) | ((uint32_t)(kTileX >> 4) << 24);
}

// One stage, issued by one elected lane: the three scale groups into TMEM (32
// rows of 16 bytes of shared memory each -> 32 lanes x 4 columns, in every lane
// quarter, in both CTAs), four MMAs of 32 contraction elements (32 bytes further
// on in the operands' rows: 2 in the descriptors), the stage's release.  One
// election for all: with one for each instruction the issue of a stage took
// longer than its MMAs.
__device__ __forceinline__ void mx_stage_e(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                           uint32_t sa, uint64_t sc, uint32_t acc, uint64_t* empty) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 r, sb, sb2;\n\t.reg .b16 m;\n\t"
      ".reg .b64 a1, a2, a3, b1, b2, b3, c1, c2;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "mov.b16 m, 3;\n\t"
      "add.u32 sb, %4, 4;\n\tadd.u32 sb2, %4, 8;\n\t"
      "add.s64 c1, %5, 32;\n\tadd.s64 c2, %5, 64;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%4], %5;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [sb], c1;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [sb2], c2;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [sb], p;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a1, b1, %3, [%4], [sb], t;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a2, b2, %3, [%4], [sb], t;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a3, b3, %3, [%4], [sb], t;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%7], m;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(sa), "l"(sc), "r"(acc), "r"(smem_u32(empty))
      : "memory");
}

// The scale groups: X's of 128 rows each, then Y's, two for each of its tiles of
// tn rows.  blockIdx.x picks the group, blockIdx.y 32 blocks of the contraction;
// rows past the operand or the tile get 2^0.
struct ScaleGroups {
  ScaleRef x, y;
  int64_t xrows, yrows;
  int xgroups, tn, blocks;
  uint32_t* out;  // [xgroups][blocks][128], then [y tiles][blocks][2][128]
};
__global__ void __launch_bounds__(256) scale_groups_kernel(const ScaleGroups p) {
  __shared__ uint8_t t[128][33];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int g = blockIdx.x, k0 = blockIdx.y * 32;
  const bool isx = g < p.xgroups;
  const int yg = g - p.xgroups, tile = yg >> 1, part = yg & 1;
  const ScaleRef& s = isx ? p.x : p.y;
  const int64_t first = isx ? (int64_t)g * 128 : (int64_t)tile * p.tn + part * 128;
  const int64_t end = isx ? p.xrows : ((int64_t)(tile + 1) * p.tn < p.yrows ? (int64_t)(tile + 1) * p.tn : p.yrows);
  const int k = k0 + lane;
#pragma unroll 4
  for (int i = w; i < 128; i += 8) {
    const int64_t r = first + i;
    uint8_t v = 127;
    if (r < end && k < p.blocks)
      v = __ldg(static_cast<const uint8_t*>(s.p) + (r >> s.row_shift) * s.ld_row + k * s.ld_col);
    t[i][lane] = v;
  }
  __syncthreads();
  // word q of a group is row q / 4 + 32 (q % 4)
  const int64_t base = isx ? (int64_t)g * p.blocks : (int64_t)p.xgroups * p.blocks + (int64_t)tile * p.blocks * 2 + part;
  const int step = isx ? 1 : 2;
  for (int i = threadIdx.x; i < 32 * 128; i += 256) {
    const int kk = i >> 7, q = i & 127;
    if (k0 + kk < p.blocks)
      p.out[(base + (int64_t)(k0 + kk) * step) * 128 + q] = t[(q >> 2) + 32 * (q & 3)][kk] * 0x01010101u;
  }
}

// Tiles in bands of 8 X tiles, so that the 74 pairs' working set is about
// square.
__device__ __forceinline__ void mx_tile(const BlockParams& p, int t, int& tx, int& ty) {
  const int band = 8 * p.tiles_y;
  const int g = t / band;
  int h = p.tiles_x - 8 * g;
  h = h < 8 ? h : 8;
  const int r = t - g * band;
  tx = 8 * g + r % h;
  ty = r / h;
}

template <int TN>
__global__ void __launch_bounds__(kThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmY,
                   const __grid_constant__ CUtensorMap tmSx, const __grid_constant__ CUtensorMap tmSy,
                   const __grid_constant__ CUtensorMap tmC, const BlockParams p) {
  constexpr int S = kStages;
  constexpr int kHalf = TN / 2;  // columns of an epilogue half, Y rows of a CTA
  // two accumulators where the scales leave room for them; one is promoted half
  // as often, since its MMAs wait for the promotion
  constexpr int kAccBufs = 2 * TN <= (int)kScaleCol ? 2 : 1;
  constexpr int kPerUnit = kAccBufs == 2 ? 8 : 16;  // blocks of 128 between promotions
  static_assert(TN % 32 == 0 && TN <= 256, "tile width");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* staging = base + S * kStageBytes;  // [2][kBufs] x kChunk, 1024-byte aligned
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + 2 * kBufs * kChunk);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* bias_s = reinterpret_cast<float*>(staging + 2 * kBufs * kChunk + 512);  // [2][128]

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
    tma_prefetch_desc(&tmSx);
    tma_prefetch_desc(&tmSy);
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
  const int units = (nst + kPerUnit - 1) / kPerUnit;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp != 1 && lane == 0) {
      // three producers take the stages in turn: one thread's wait and issue of a
      // stage's four loads takes about 600 clocks, longer than its MMAs
      const int turn = warp ? warp - 1 : 0;
      int q = 0;
      // X 128 rows, half of the Y rows and three scale groups, of both CTAs
      const uint32_t bytes = 2u * (16384u + (uint32_t)kHalf * 128u + 3u * 512u);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int tx, ty;
        mx_tile(p, t, tx, ty);
        const int x0 = tx * kTileX + 128 * (int)rank, y0 = ty * TN + kHalf * (int)rank;
        for (int i = 0; i < nst; ++i, q = q == 2 ? 0 : q + 1) {
          if (q != turn) {
            if (++s == S) { s = 0; ph ^= 1; }
            continue;
          }
          if (!(ok = mbar_wait_bounded(&empty[s], ph ^ 1, abort_flag, p.err, DEV_TIMEOUT_EMPTY,
                                       p.timeout_ns)))
            break;
          const uint32_t st = smem_u32(base + s * kStageBytes);
          // the first CTA expects both CTAs' bytes; the second's may land first
          const uint32_t bar = map_rank(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
          tma_load_2d_pair(st, &tmX, bar, i * 128, x0);
          tma_load_2d_pair(st + 16384, &tmY, bar, i * 128, y0);
          tma_load_2d_pair(st + 32768, &tmSx, bar, 0, (2 * tx + (int)rank) * nst + i);
          tma_load_2d_pair(st + 32768 + 512, &tmSy, bar, 0, 2 * (ty * nst + i));
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
    } else if (warp == 1 && rank == 0) {
      auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        int got = 0;
        if (lane == 0) got = mbar_wait_bounded(bar, parity, abort_flag, p.err, code, p.timeout_ns);
        return __shfl_sync(0xffffffffu, got, 0) != 0;
      };
      int s = 0, g = 0, q = 0;
      uint32_t ph = 0;
      bool ok = true;
      // Lane 0: whether the next stage's operands and the next unit's accumulator
      // were found ready before this stage's MMAs were issued.  A wait costs this
      // warp 200 clocks of latency even when its barrier is complete; the tests
      // run behind the issue.
      int next_full = 0, next_empty = 0;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int i = 0;
        for (int u = 0; u < units && ok; ++u, ++g) {
          const int b = kAccBufs == 2 ? g & 1 : 0, use = kAccBufs == 2 ? g >> 1 : g;
          const uint32_t d = tmem + (uint32_t)(b * TN);
          for (int j = 0; j < kPerUnit && i < nst; ++j, ++i, q ^= 1) {
            const int ready = __shfl_sync(0xffffffffu, next_full | (next_empty << 1), 0);
            if (!(ready & 1) && !(ok = wait(&full[s], ph, DEV_TIMEOUT_FULL))) break;
            if (j == 0 && !(ready & 2) &&
                !(ok = wait(&tempty[b], (use & 1) ^ 1, DEV_TIMEOUT_TMEM_EMPTY)))
              break;
            tc_fence_after();
            const int sn = s + 1 == S ? 0 : s + 1;
            const uint32_t phn = s + 1 == S ? ph ^ 1u : ph;
            const bool last = j + 1 == kPerUnit || i + 1 == nst;
            if (lane == 0) {
              next_full = mbar_test_wait(&full[sn], phn);
              next_empty = kAccBufs == 2 && last ? mbar_test_wait(&tempty[b ^ 1], (((g + 1) >> 1) & 1) ^ 1) : 0;
            }
            // operands K-major in 128-byte swizzled rows; scale groups unswizzled,
            // 8-row groups 128 bytes apart
            const uint32_t xa = smem_u32(base + s * kStageBytes);
            mx_stage_e(d, umma_desc(xa, 16, 1024, kLayoutSW128),
                       umma_desc(xa + 16384, 16, 1024, kLayoutSW128), mx_idesc(TN),
                       tmem + kScaleCol + 12u * (uint32_t)q, umma_desc(xa + 32768, 128, 128, 0), j > 0,
                       &empty[s]);
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
    const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)(kHalf * half);
    const uint32_t tempty0[2] = {map_rank(smem_u32(&tempty[0]), 0), map_rank(smem_u32(&tempty[1]), 0)};
    uint8_t* stg0 = staging + half * kBufs * kChunk;
    int g = 0, buf = 0;
    bool ok = true;
    for (int t = pair; t < tiles; t += pairs) {
      int tx, ty;
      mx_tile(p, t, tx, ty);
      const int64_t x = (int64_t)tx * kTileX + 128 * rank + row;
      const int64_t y0 = (int64_t)ty * TN + kHalf * half;
      if (p.bias) {
        // the tile's bias: loaded here, its latency passes behind the MMAs; the
        // barriers of the stores below keep its readers and writers apart
        named_bar_sync(1 + half, 128);
        if (et < kHalf) bias_s[128 * half + et] = y0 + et < p.ycols ? __ldg(p.bias + y0 + et) : 0.0f;
        named_bar_sync(1 + half, 128);
      }
      unsigned long long acc[kHalf / 2];
#pragma unroll
      for (int j = 0; j < kHalf / 2; ++j) acc[j] = 0ull;
      for (int u = 0; u < units; ++u, ++g) {
        const int b = kAccBufs == 2 ? g & 1 : 0, use = kAccBufs == 2 ? g >> 1 : g;
        if (ok) {
          int got = 0;
          if (lane == 0)
            got = mbar_wait_bounded(&tfull[b], use & 1, abort_flag, p.err,
                                    DEV_TIMEOUT_TMEM_FULL, p.timeout_ns);
          ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        }
        tc_fence_after();
        const uint32_t ta = t_lane + (uint32_t)(TN * b);
#pragma unroll
        for (int c = 0; c < kHalf / 16; ++c) {
          uint32_t r[16];
          tmem_ld_x16(ta + 16 * c, r);
          tmem_wait_x16(r);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            acc[8 * c + j] = add2(acc[8 * c + j], pack2(r[2 * j], r[2 * j + 1]));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_pair(tempty0[b]);
      }
      // the finished rows, 16 columns at a time
#pragma unroll
      for (int c = 0; c < kHalf / 16; ++c) {
        const int64_t yc = y0 + 16 * c;
        float v[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = unpack2(acc[8 * c + j]);
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += bias_s[128 * half + 16 * c + j];
        }
        activate_n<16>(v, p.act);
        if (p.c_tma) {
          // this chunk's store before has read it (its issuing thread waits): with
          // one chunk a half the waits made a tile's epilogue 6 us long
          uint8_t* stg = stg0 + buf * kChunk;
          if (et == 0) bulk_wait_group_read<kBufs - 1>();
          named_bar_sync(1 + half, 128);
          // 64-byte rows, 16-byte units swizzled by (row / 2) % 4
          const uint32_t dst = smem_u32(stg) + row * 64;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sts128(dst + ((j ^ ((row >> 1) & 3)) << 4),
                   make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
          fence_proxy_async_smem();
          named_bar_sync(1 + half, 128);
          const int xs = tx * kTileX + 128 * (int)rank;
          if (et == 0 && yc < p.ycols && xs < p.xrows) {
            tma_store_2d(&tmC, stg, (int)yc, xs);
          }
          if (et == 0) bulk_commit_group();  // (an empty group where nothing is stored)
          buf = buf + 1 == kBufs ? 0 : buf + 1;
        } else if (x < p.xrows) {
          float* o = p.out + x * p.ldo + yc;
#pragma unroll
          for (int j = 0; j < 16; ++j)
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

template <int TN>
int launch(rtb_ctx* ctx, const uint8_t* X, int64_t ldx, const uint8_t* Y, int64_t ldy,
           BlockParams& p, cudaStream_t s) {
  auto* k = mx_gemm_kernel<TN>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return cuda_status(e, "block-scaled gemm smem attribute");
  p.tiles_x = (int)((p.xrows + kTileX - 1) / kTileX);
  p.tiles_y = (int)((p.ycols + TN - 1) / TN);
  p.stages_total = (p.depth + 127) / 128;
  const int64_t tiles = (int64_t)p.tiles_x * p.tiles_y;
  if (tiles > INT32_MAX / 2) return set_error(RTB_E_UNSUPPORTED, "block-scaled gemm: too many tiles");
  CUtensorMap tmX, tmY;
  int st;
  if ((st = make_tmap_2d_bytes(&tmX, X, 1, (uint64_t)p.depth, (uint64_t)p.xrows, (uint64_t)ldx, 128,
                               128)))
    return st;
  if ((st = make_tmap_2d_bytes(&tmY, Y, 1, (uint64_t)p.depth, (uint64_t)p.ycols, (uint64_t)ldy, 128,
                               TN / 2)))
    return st;
  CUtensorMap tmC = tmX;
  // (A TMA store clips a box at the tensor's columns in units of 16 bytes: up to three
  // floats behind a row whose length is no multiple of 4 would be overwritten.  A test
  // for each chunk, so that only a row's last one is stored directly, costs the others
  // 2 us of 97 on 8192 x 8192 x 1024.)
  p.c_tma = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && p.ldo % 4 == 0 && p.ycols % 4 == 0;
  if (p.c_tma && (st = make_tmap_2d_swz(&tmC, p.out, (uint64_t)p.ycols, (uint64_t)p.xrows,
                                        (uint64_t)p.ldo, 16, 128, kTmapSwizzle64)))
    return st;
  // the scale groups: X's tiles of 256 rows have two, whole or not
  ScaleGroups sg = {p.scx, p.scy, p.xrows, p.ycols, 2 * p.tiles_x, TN, p.stages_total, nullptr};
  const int64_t groups = (int64_t)sg.xgroups + 2 * p.tiles_y;
  const int64_t rows = groups * p.stages_total;
  if (rows > INT32_MAX / 2) return set_error(RTB_E_UNSUPPORTED, "block-scaled gemm: too many scales");
  if ((st = ws_alloc(ctx, (void**)&sg.out, (size_t)rows * 512, s))) return st;
  const float* fx = reinterpret_cast<const float*>(sg.out);
  const int64_t xr = (int64_t)sg.xgroups * p.stages_total;
  CUtensorMap tmSx, tmSy;
  st = make_tmap_2d_swz(&tmSx, fx, 128, (uint64_t)xr, 128, 128, 1, kTmapSwizzleNone);
  if (st == RTB_OK)
    st = make_tmap_2d_swz(&tmSy, fx + xr * 128, 128, (uint64_t)(rows - xr), 128, 128, 2,
                          kTmapSwizzleNone);
  if (st != RTB_OK) {
    ws_free(sg.out, s);
    return st;
  }
  clear_stale_cuda_error();
  e = launch_pdl(scale_groups_kernel,
                 dim3((unsigned)groups, (unsigned)((p.stages_total + 31) / 32)), dim3(256), 0, s,
                 (const ScaleGroups)sg);
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
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, k, tmX, tmY, tmSx, tmSy, tmC, (const BlockParams)p);
  if (e == cudaSuccess) e = cudaGetLastError();
  ws_free(sg.out, s);
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "block-scaled gemm launch");
}

}  // namespace

int launch_mx(rtb_ctx* ctx, const uint8_t* X, int64_t ldx, const uint8_t* Y, int64_t ldy,
              BlockParams& p, cudaStream_t s) {
  // 256 columns move fewer bytes for a product, 224 have room for a second
  // accumulator, behind which a tile's epilogue (and the promotions) pass.  In
  // whole rounds of the pairs, from the measured times of a round: 0.37 us a
  // stage, and 6 or 4 us a tile (8192 x 4096 x 8192: 225 us against 261; 8192 x
  // 8192 x 1024: 123 against 106).
  auto cost = [&](int64_t tn, double tile_us) {
    const int64_t tiles = ((p.xrows + kTileX - 1) / kTileX) * ((p.ycols + tn - 1) / tn);
    const int64_t pairs = ctx->sm_count / 2;
    return (double)((tiles + pairs - 1) / pairs) * (0.37 * ((p.depth + 127) / 128) + tile_us);
  };
  return cost(224, 4.0) < 0.95 * cost(256, 6.0) ? launch<224>(ctx, X, ldx, Y, ldy, p, s)
                                                : launch<256>(ctx, X, ldx, Y, ldy, p, s);
}

}  // namespace rtb
