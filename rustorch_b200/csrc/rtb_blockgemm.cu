// Products whose partial sums leave the tensor core every 128 elements of the
// contraction (tcgen05, sm_100a):
//
//   MODE 0  C[m,n] = act( sum_kb sa[m,kb] sb[n,kb] sum_{k in kb} A[m,k] B[n,k]
//                         + bias[n] ),  A and B e4m3 (kind::f8f6f4)
//   MODE 1  D[k,n] (+)= sum_m X[m,k] Y[m,n],  X bf16, Y a sum of bf16 terms
//                       (kind::f16): the weight gradient from a checkpoint
//
// In both the MMAs of one 128-element block accumulate in TMEM and the
// epilogue warps add the block's partial sum into fp32 registers on the CUDA
// cores: MODE 0 because each block has scales of its own (one fused
// multiply-add an element applies both), MODE 1 because the tensor core's own
// accumulation does not round every addition to nearest, so its error grows
// with the length of the chain.
//
// A CTA computes a 128 x BN tile: X rows (MMA M side, TMEM lanes) by Y columns
// (MMA N side).  Roles (warp index): 0 TMA producer, 1 TMEM allocator + MMA
// issuer, 2..5 epilogue (TMEM lanes 32 (w % 4)..).  The accumulator is double
// buffered in TMEM, so the promotion of one block overlaps the MMAs of the
// next.  Every wait is bounded: after a timeout a role goes on without waiting
// (no thread leaves early, so that barriers still meet), the output is
// undefined and the error word tells the host.
//
// Shared memory (128-byte swizzle throughout):
//   MODE 0, K-major: row r at r * 128 B holds 128 e4m3 of the contraction.
//   MODE 1, MN-major: boxes of 64 contraction rows x 64 bf16 (8 KB).
#include <cstdlib>

#include "rtb_blockgemm.cuh"

namespace rtb {

namespace {

constexpr int kX = 128;                // tile rows
constexpr int kXBytes = 128 * 128;     // X bytes of a stage (16 KB, both modes)
constexpr int kSmemMax = 232448;       // dynamic shared memory per CTA
constexpr int kReserve = 4096;         // barriers, scales, alignment slack
constexpr int kThreads = 192;

template <int MODE, int BN>
struct Cfg {
  static constexpr int kDepth = MODE == 0 ? 128 : 64;  // contraction elements of a stage
  static constexpr int kPieces = MODE == 0 ? 1 : 3;
  static constexpr int kYPiece = BN * 128;             // one Y piece of a stage (BN x 128 B)
  static constexpr int kStageBytes = kXBytes + kPieces * kYPiece;
  static constexpr int kStagesRaw = (kSmemMax - kReserve) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kSmemBytes = kStages * kStageBytes + kReserve;
  static constexpr int kPerUnit = 128 / kDepth;        // stages of a promotion unit
  static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
  static_assert(kStages >= 2, "two stages");
};

template <int MODE>
__device__ __forceinline__ void mma_e(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                      uint32_t acc) {
  if (MODE == 0) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
  }
}

// YVEC (MODE 0): a scale for every Y column (block_rows 1); otherwise the
// tile's columns lie in one 128-row block and share one.
template <int MODE, int BN, bool YVEC>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap tmX,
                      const __grid_constant__ CUtensorMap tmY, const BlockParams p) {
  using C = Cfg<MODE, BN>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* tail = base + S * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(tail);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* sy_s = reinterpret_cast<float*>(tail + 512);  // YVEC: [2][BN] column scales

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 128);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmY);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int tx = blockIdx.x % p.tiles_x, ty = blockIdx.x / p.tiles_x;
  const int nst = p.stages_total;
  const int units = (nst + C::kPerUnit - 1) / C::kPerUnit;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t tx_bytes = kXBytes + (MODE == 0 ? 1 : p.pieces) * C::kYPiece;
      for (int i = 0; i < nst; ++i) {
        const int s = i % S;
        if (!mbar_wait_bounded(&empty[s], ((i / S) & 1) ^ 1, abort_flag, p.err, DEV_TIMEOUT_EMPTY,
                               p.timeout_ns))
          break;
        uint8_t* st = base + s * C::kStageBytes;
        mbar_arrive_expect_tx(&full[s], tx_bytes);
        if (MODE == 0) {
          tma_load_2d(st, &tmX, &full[s], i * 128, tx * kX);
          tma_load_2d(st + kXBytes, &tmY, &full[s], i * 128, ty * BN);
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b)
            tma_load_2d(st + b * 8192, &tmX, &full[s], tx * kX + 64 * b, i * 64);
          for (int q = 0; q < p.pieces; ++q)
#pragma unroll
            for (int b = 0; b < BN / 64; ++b)
              tma_load_2d(st + kXBytes + q * C::kYPiece + b * 8192, &tmY, &full[s],
                          ty * BN + 64 * b, (int)(q * p.piece_rows) + i * 64);
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t id = block_idesc(MODE, kX, BN);
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      int got = 0;
      if (lane == 0) got = mbar_wait_bounded(bar, parity, abort_flag, p.err, code, p.timeout_ns);
      return __shfl_sync(0xffffffffu, got, 0) != 0;
    };
    for (int u = 0, i = 0; u < units && ok; ++u) {
      const int b = u & 1;
      if (!(ok = wait(&tempty[b], ((u >> 1) & 1) ^ 1, DEV_TIMEOUT_TMEM_EMPTY))) break;
      tc_fence_after();
      const uint32_t d = tmem + (uint32_t)(b * BN);
      for (int j = 0; j < C::kPerUnit && i < nst; ++j, ++i) {
        const int s = i % S;
        if (!(ok = wait(&full[s], (i / S) & 1, DEV_TIMEOUT_FULL))) break;
        tc_fence_after();
        const uint32_t xa = smem_u32(base + s * C::kStageBytes), ya = xa + kXBytes;
        if (MODE == 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 e4m3 (32 bytes of the swizzled row) a step
            mma_e<0>(d, umma_desc(xa + 32 * k, 16, 1024, kLayoutSW128),
                     umma_desc(ya + 32 * k, 16, 1024, kLayoutSW128), id, k > 0);
        } else {
          // the smallest terms first; 16 contraction rows (2 KB) a step, 8 KB
          // between 64-column boxes, 1 KB per 8 rows
          for (int q = p.pieces - 1; q >= 0; --q)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_e<1>(d, umma_desc(xa + 2048 * k, 8192, 1024, kLayoutSW128),
                       umma_desc(ya + q * C::kYPiece + 2048 * k, 8192, 1024, kLayoutSW128), id,
                       j > 0 || k > 0 || q < p.pieces - 1);
        }
        umma_commit_e(&empty[s]);
      }
      if (!ok) break;
      umma_commit_e(&tfull[b]);
    }
  } else {
    const int row = 32 * (warp & 3) + lane;
    const int et = threadIdx.x - 64;  // 0..127
    const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const int64_t x = (int64_t)tx * kX + row;
    const int64_t y0 = (int64_t)ty * BN;
    float acc[BN];
#pragma unroll
    for (int j = 0; j < BN; ++j) acc[j] = 0.0f;
    bool ok = true;
    const int64_t xi = MODE == 0 && x < p.xrows ? (x >> p.scx.row_shift) * p.scx.ld_row : -1;
    const int64_t yr = y0 + (YVEC ? et : 0);
    const int64_t yi = MODE == 0 && yr < p.ycols && (!YVEC || et < BN)
                           ? (yr >> p.scy.row_shift) * p.scy.ld_row : -1;
    auto scale_x = [&](int u) -> uint32_t {
      return xi >= 0 && u < units ? load_scale(p.scx, xi + u * p.scx.ld_col) : 0u;
    };
    auto scale_y = [&](int u) -> uint32_t {
      return yi >= 0 && u < units ? load_scale(p.scy, yi + u * p.scy.ld_col) : 0u;
    };
    uint32_t rx[2] = {0, 0}, ry[2] = {0, 0};  // the scales of the next two blocks
    if (MODE == 0) {
      rx[0] = scale_x(0);
      ry[0] = scale_y(0);
      rx[1] = scale_x(1);
      ry[1] = scale_y(1);
    }
    for (int u = 0; u < units; ++u) {
      const int b = u & 1;
      float cx = 0.0f, cy = 0.0f;
      if (MODE == 0) {
        cx = scale_value(p.scx, rx[0]);
        cy = scale_value(p.scy, ry[0]);
        rx[0] = rx[1];
        ry[0] = ry[1];
        rx[1] = scale_x(u + 2);
        ry[1] = scale_y(u + 2);
      }
      if (YVEC) {
        // two buffers: the block after next's write comes behind the next barrier
        if (et < BN) sy_s[b * BN + et] = cy;
        named_bar_sync(1, 128);
      }
      if (ok) {
        int got = 0;
        if (lane == 0)
          got = mbar_wait_bounded(&tfull[b], (u >> 1) & 1, abort_flag, p.err,
                                  DEV_TIMEOUT_TMEM_FULL, p.timeout_ns);
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
      }
      tc_fence_after();
      const float s = MODE == 0 ? (YVEC ? cx : cx * cy) : 1.0f;
#pragma unroll
      for (int c = 0; c < BN; c += 16) {
        uint32_t r[16];
        tmem_ld_x16(t_lane + (uint32_t)(b * BN + c), r);
        tmem_wait_x16(r);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float t = __uint_as_float(r[j]);
          if (MODE == 1) acc[c + j] += t;
          else if (YVEC) acc[c + j] = fmaf(t, s * sy_s[b * BN + c + j], acc[c + j]);
          else acc[c + j] = fmaf(t, s, acc[c + j]);
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty[b]);
    }
    if (x < p.xrows) {
      float* o = p.out + x * p.sx + y0 * p.sy;
      const float bx = p.bias && p.bias_on_x ? p.bias[x] : 0.0f;
#pragma unroll
      for (int j = 0; j < BN; ++j) {
        if (y0 + j >= p.ycols) break;
        float v = acc[j] + bx;
        if (p.bias && !p.bias_on_x) v += __ldg(p.bias + y0 + j);
        if (p.accumulate) v += o[j * p.sy];
        o[j * p.sy] = activate(v, p.act);
      }
    }
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
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <int MODE, int BN, bool YVEC>
int launch(const CUtensorMap& tmX, const CUtensorMap& tmY, BlockParams& p, cudaStream_t s) {
  using C = Cfg<MODE, BN>;
  auto* k = block_gemm_kernel<MODE, BN, YVEC>;
  cudaError_t e =
      cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return cuda_status(e, "block gemm smem attribute");
  p.tiles_x = (int)((p.xrows + kX - 1) / kX);
  p.tiles_y = (int)((p.ycols + BN - 1) / BN);
  p.stages_total = (p.depth + C::kDepth - 1) / C::kDepth;
  const int64_t tiles = (int64_t)p.tiles_x * p.tiles_y;
  if (tiles > INT32_MAX) return set_error(RTB_E_UNSUPPORTED, "block gemm: too many tiles");
  clear_stale_cuda_error();
  e = launch_pdl(k, dim3((unsigned)tiles), dim3(kThreads), C::kSmemBytes, s, tmX, tmY,
                 (const BlockParams)p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "block gemm launch");
}

// CTA pairs where their 256 x 256 tiles occupy most of the SMs.
bool use_pairs(const rtb_ctx* ctx, const BlockParams& p) {
  static const int env = [] {
    const char* v = std::getenv("RTB_PAIR");
    return v ? std::atoi(v) : -1;
  }();
  if (env >= 0) return env != 0;
  const int64_t tiles = ((p.xrows + 255) / 256) * ((p.ycols + 255) / 256);
  return tiles * 2 > ctx->sm_count / 2;
}

int check_extents(int64_t a, int64_t b, int64_t c) {
  if (a > INT32_MAX - 512 || b > INT32_MAX - 512 || c > INT32_MAX - 512)
    return set_error(RTB_E_UNSUPPORTED, "block gemm: dimension exceeds 2^31-513");
  return RTB_OK;
}

}  // namespace

int fp8_gemm_run(rtb_ctx* ctx, const Fp8Desc& d, cudaStream_t s) {
  int st;
  if ((st = check_extents(d.M, d.N, d.K))) return st;
  // Few rows of A: the weight's rows fill the 128-row tile and A is the narrow
  // side (C^T = B . A^T), so little of the tile is padding.
  const bool swap = d.M <= 64;
  BlockParams p{};
  p.xrows = swap ? d.N : d.M;
  p.ycols = swap ? d.M : d.N;
  p.depth = (int)d.K;
  p.out = d.C;
  p.sx = swap ? 1 : d.ldc;
  p.sy = swap ? d.ldc : 1;
  p.bias = d.bias;
  p.bias_on_x = swap;
  p.act = d.act;
  p.scx = swap ? d.sb : d.sa;
  p.scy = swap ? d.sa : d.sb;
  p.err = ctx->d_err;
  p.timeout_ns = ctx->timeout_ns;
  const bool yvec = p.scy.row_shift == 0;
  const int bn = swap ? (d.M <= 16 ? 16 : d.M <= 32 ? 32 : 64) : 128;
  const uint8_t* X = swap ? d.B : d.A;
  const uint8_t* Y = swap ? d.A : d.B;
  CUtensorMap tmX, tmY;
  if ((st = make_tmap_2d_bytes(&tmX, X, 1, (uint64_t)d.K, (uint64_t)p.xrows,
                               (uint64_t)(swap ? d.ldb : d.lda), 128, kX)))
    return st;
  if ((st = make_tmap_2d_bytes(&tmY, Y, 1, (uint64_t)d.K, (uint64_t)p.ycols,
                               (uint64_t)(swap ? d.lda : d.ldb), 128, (uint32_t)bn)))
    return st;
  if (!swap && use_pairs(ctx, p)) return launch_pair(ctx, 0, yvec, tmX, tmY, p, s);
  if (bn == 16) return yvec ? launch<0, 16, true>(tmX, tmY, p, s) : launch<0, 16, false>(tmX, tmY, p, s);
  if (bn == 32) return yvec ? launch<0, 32, true>(tmX, tmY, p, s) : launch<0, 32, false>(tmX, tmY, p, s);
  if (bn == 64) return yvec ? launch<0, 64, true>(tmX, tmY, p, s) : launch<0, 64, false>(tmX, tmY, p, s);
  return yvec ? launch<0, 128, true>(tmX, tmY, p, s) : launch<0, 128, false>(tmX, tmY, p, s);
}

int wgrad_run(rtb_ctx* ctx, const WgradDesc& d, cudaStream_t s) {
  int st;
  if ((st = check_extents(d.rows_pad * d.pieces, d.N, d.K))) return st;
  BlockParams p{};
  p.xrows = d.K;
  p.ycols = d.N;
  p.depth = (int)d.rows;
  p.out = d.D;
  p.sx = d.ldd;
  p.sy = 1;
  p.accumulate = d.accumulate;
  p.pieces = d.pieces;
  p.piece_rows = d.rows_pad;
  p.err = ctx->d_err;
  p.timeout_ns = ctx->timeout_ns;
  CUtensorMap tmX, tmY;
  if ((st = make_tmap_2d_bytes(&tmX, d.X, 2, (uint64_t)d.ldx, (uint64_t)d.rows_pad,
                               (uint64_t)d.ldx, 64, 64)))
    return st;
  if ((st = make_tmap_2d_bytes(&tmY, d.Y, 2, (uint64_t)d.ldy, (uint64_t)(d.rows_pad * d.pieces),
                               (uint64_t)d.ldy, 64, 64)))
    return st;
  if (use_pairs(ctx, p)) return launch_pair(ctx, 1, false, tmX, tmY, p, s);
  return launch<1, 128, false>(tmX, tmY, p, s);
}

}  // namespace rtb
