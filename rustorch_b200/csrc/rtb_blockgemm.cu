// Products whose partial sums leave the tensor core every 128 elements of the
// contraction (tcgen05, sm_100a):
//
//   MODE 0  C[m,n] = act( sum_kb sa[m,kb] sb[n,kb] sum_{k in kb} A[m,k] B[n,k]
//                         + bias[n] ),  A and B e4m3 (kind::f8f6f4)
//   MODE 1  D[k,n] (+)= sum_m X[m,k] Y[m,n],  X bf16, Y a sum of bf16 terms
//                       (kind::f16): the weight gradient from a checkpoint
//   MODE 2  as MODE 0 with e8m0 scales, applied by the tensor core
//                       (kind::mxf8f6f4, see rtb_mxgemm.cu): a promotion every
//                       1024 elements.  MODE 0 takes 1500 clocks a block, the
//                       epilogue's chain of barrier, TMEM loads and adds.
//
// In the first two the MMAs of one 128-element block accumulate in TMEM and the
// epilogue warps add the block's partial sum into fp32 registers on the CUDA
// cores: MODE 0 because each block has scales of its own (one fused
// multiply-add an element applies both), MODE 1 because the tensor core's own
// accumulation does not round every addition to nearest, so its error grows
// with the length of the chain.
//
// A CTA computes a 128 x BN tile: X rows (MMA M side, TMEM lanes) by Y columns
// (MMA N side).  Few tiles: a cluster of 2, 4 or 8 CTAs shares a tile, each a
// part of the contraction, and adds the parts out of one another's shared
// memory in rank order (no workspace, no counters, the same bits every time).
// Roles (warp index): 0, 6, 7 TMA producers, 1 TMEM allocator + MMA issuer, 2..5
// epilogue (TMEM lanes 32 (w % 4)..; MODE 2: they also lay out the scales).  The
// accumulator is double buffered in TMEM, so the promotion of one block overlaps the MMAs of the next.  The
// finished tile goes through shared memory (the idle load ring), so that its
// stores run along the output's rows and bias, activation and the sum of the
// parts are one short loop.  Every wait is bounded: after a timeout a role goes
// on without waiting (no thread leaves early, so that barriers still meet), the
// output is undefined and the error word tells the host.
//
// Shared memory (128-byte swizzle throughout):
//   MODE 0, 2, K-major: row r at r * 128 B holds 128 e4m3 of the contraction.
//   MODE 1, MN-major: boxes of 64 contraction rows x 64 bf16 (8 KB).
#include "rtb_blockgemm.cuh"
#include "rtb_per_device.h"

namespace rtb {

namespace {

constexpr int kX = 128;                // tile rows
constexpr int kXBytes = 128 * 128;     // X bytes of a stage (16 KB, both modes)
constexpr int kSmemMax = 232448;       // dynamic shared memory per CTA
constexpr int kSmemHalf = 115712;      // of two CTAs on an SM
constexpr int kReserve = 2048;         // barriers, alignment slack
constexpr int kScaleUnits = 32;        // blocks whose scales are staged at a time
constexpr int kThreads = 256;

template <int MODE, int BN, bool YVEC>
struct Cfg {
  static constexpr int kDepth = MODE == 1 ? 64 : 128;  // contraction elements of a stage
  static constexpr int kPieces = MODE == 1 ? 3 : 1;
  static constexpr int kYPiece = BN * 128;             // one Y piece of a stage (BN x 128 B)
  static constexpr int kStageBytes = kXBytes + kPieces * kYPiece;
  // Narrow tiles, two CTAs on an SM: one's loads pass behind the other's start and
  // end (a token row by 8192 x 8192: 19.9 us with one CTA of eight stages, 18.8).
  static constexpr int kPerSm = MODE == 2 && BN <= 32 ? 2 : 1;
  static constexpr int kSf = kPerSm == 2 ? 8 : 16;     // MODE 2: blocks of a scale buffer, of two
  static constexpr int kBudget = kPerSm == 2 ? kSmemHalf : kSmemMax;
  static constexpr int kSy = YVEC ? BN : 1;            // column scales of a block
  static constexpr int kScaleBytes =
      MODE == 0 ? kScaleUnits * (128 + kSy) * 4 : (MODE == 2 ? 2 * kSf * 1024 : 0);
  static constexpr int kStagesRaw = (kBudget - kReserve - kScaleBytes) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 8 ? 8 : kStagesRaw;
  static constexpr int kSmemBytes = kStages * kStageBytes + kScaleBytes + kReserve;
  // the finished tile: [128][BN + 4] floats, or [BN][132] where X is the
  // output's columns
  static_assert(kStages * kStageBytes >= 128 * (BN + 4) * 4 &&
                    kStages * kStageBytes >= BN * 132 * 4, "the ring holds the finished tile");
  static constexpr int kPerUnit = MODE == 0 ? 1 : (MODE == 1 ? 2 : 8);  // stages between promotions
  static constexpr int kGrain = MODE == 1 ? 2 : 1;     // stages that parts are cut at
  // MODE 2: two buffers of 4 + 4 scale columns behind the accumulators
  static constexpr int kTmemNeed = 2 * BN + (MODE == 2 ? 16 : 0);
  static constexpr int kTmemCols =
      kTmemNeed <= 32 ? 32 : kTmemNeed <= 64 ? 64 : kTmemNeed <= 128 ? 128 : kTmemNeed <= 256 ? 256 : 512;
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

// MODE 2: a stage's two scale groups into TMEM, its four MMAs and its release,
// by one elected lane (mx_stage_e in rtb_mxgemm.cu is the same for a pair).
__device__ __forceinline__ void mx_stage1_e(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                            uint32_t sa, uint64_t cx, uint64_t cy, uint32_t acc,
                                            uint64_t* empty) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 r, sb;\n\t"
      ".reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "setp.ne.b32 p, %7, 0;\n\t"
      "setp.eq.b32 t, 0, 0;\n\t"
      "add.u32 sb, %4, 4;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%4], %5;\n\t"
      "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [sb], %6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [sb], p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a1, b1, %3, [%4], [sb], t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a2, b2, %3, [%4], [sb], t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a3, b3, %3, [%4], [sb], t;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%8];\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(sa), "l"(cx), "l"(cy), "r"(acc), "r"(smem_u32(empty))
      : "memory");
}

// MODE 2: the scale bytes of blocks u .. u + n - 1 (n <= N) of row r; 2^0 for rows
// past the operand.
template <int N>
__device__ __forceinline__ void load_scale_bytes(const ScaleRef& s, int64_t r, int64_t rows, int u,
                                                 int n, uint32_t (&raw)[N]) {
  const bool in = r < rows;
  const uint8_t* p = static_cast<const uint8_t*>(s.p) +
                     (in ? (r >> s.row_shift) * s.ld_row + (int64_t)u * s.ld_col : 0);
#pragma unroll
  for (int k = 0; k < N; ++k) raw[k] = in && k < n ? __ldg(p + (int64_t)k * s.ld_col) : 127u;
}
// ... as words of the 512-byte groups that the tensor core takes (row l of a group:
// the word at 16 (l % 32) + 4 (l / 32), its byte four times).
template <int N>
__device__ __forceinline__ void store_scale_words(const uint32_t (&raw)[N], uint8_t* group, int l) {
#pragma unroll
  for (int k = 0; k < N; ++k)
    *reinterpret_cast<uint32_t*>(group + 512 * k + 16 * (l & 31) + 4 * (l >> 5)) = raw[k] * 0x01010101u;
}

// The scales of blocks u .. u + n - 1 of row r, decoded, to dst[0], dst[step],
// ...; zero for rows past the operand.
__device__ __forceinline__ void stage_scales(const ScaleRef& s, int64_t r, int64_t rows, int u,
                                             int n, float* dst, int step) {
  const bool in = r < rows;
  const int64_t at = in ? (r >> s.row_shift) * s.ld_row + (int64_t)u * s.ld_col : 0;
  for (int k = 0; k < n; k += 8) {
    uint32_t raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      raw[i] = load_scale(s, at + (int64_t)(k + i < n ? k + i : k) * s.ld_col);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < n) dst[(k + i) * step] = in ? scale_value(s, raw[i]) : 0.0f;
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// Without an order of memory: behind reads whose values have been used, when the
// stores since need not be seen (a release would wait for them).
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" :::
                   "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// YVEC (MODE 0): a scale for every Y column (block_rows 1); otherwise the
// tile's columns lie in one 128-row block and share one.
template <int MODE, int BN, bool YVEC>
__global__ void __launch_bounds__(kThreads, Cfg<MODE, BN, YVEC>::kPerSm)
    block_gemm_kernel(const __grid_constant__ CUtensorMap tmX,
                      const __grid_constant__ CUtensorMap tmY, const BlockParams p) {
  using C = Cfg<MODE, BN, YVEC>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* sx = reinterpret_cast<float*>(base + S * C::kStageBytes);  // [kScaleUnits][128]
  float* sy = sx + (MODE == 0 ? kScaleUnits * 128 : 0);             // [kScaleUnits][kSy]
  uint8_t* tail = base + S * C::kStageBytes + C::kScaleBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(tail);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* sfull = tempty + 2;   // MODE 2: scale buffers
  uint64_t* sempty = sfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* sf = reinterpret_cast<uint8_t*>(sx);  // MODE 2: [2][X, Y][kSf][512]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 128);
      mbar_init(&sfull[b], 128);
      mbar_init(&sempty[b], 1);
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

  // the cluster's tile, and this CTA's part of the contraction
  const int parts = p.parts, rank = (int)blockIdx.x % parts, tile = (int)blockIdx.x / parts;
  const int tx = tile % p.tiles_x, ty = tile / p.tiles_x;
  const int all = (p.stages_total + C::kGrain - 1) / C::kGrain;
  const int i0 = (int)((int64_t)rank * all / parts) * C::kGrain;
  const int i1g = (int)((int64_t)(rank + 1) * all / parts) * C::kGrain;
  const int i1 = i1g < p.stages_total ? i1g : p.stages_total;
  const int nst = i1 - i0;
  const int units = (nst + C::kPerUnit - 1) / C::kPerUnit;

  if (warp == 0 || warp >= 6) {
    if (lane == 0) {
      // three producers take the stages in turn: one thread's wait and issue
      // takes longer than a stage's MMAs
      const uint32_t tx_bytes = kXBytes + (MODE == 1 ? p.pieces : 1) * C::kYPiece;
      for (int i = i0 + (warp ? warp - 5 : 0); i < i1; i += 3) {
        const int s = (i - i0) % S;
        if (!mbar_wait_bounded(&empty[s], (((i - i0) / S) & 1) ^ 1, abort_flag, p.err,
                               DEV_TIMEOUT_EMPTY, p.timeout_ns))
          break;
        uint8_t* st = base + s * C::kStageBytes;
        mbar_arrive_expect_tx(&full[s], tx_bytes);
        if (MODE != 1) {
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
    // (lane 0) the next stage's operands were found ready before this stage's
    // MMAs: a wait costs 200 clocks even when its barrier is complete
    int next_full = 0;
    for (int u = 0, i = 0; u < units && ok; ++u) {
      const int b = u & 1;
      const uint32_t d = tmem + (uint32_t)(b * BN);
      for (int j = 0; j < C::kPerUnit && i < nst; ++j, ++i) {
        const int s = i % S;
        if (!__shfl_sync(0xffffffffu, next_full, 0) &&
            !(ok = wait(&full[s], (i / S) & 1, DEV_TIMEOUT_FULL)))
          break;
        if (j == 0 && !(ok = wait(&tempty[b], ((u >> 1) & 1) ^ 1, DEV_TIMEOUT_TMEM_EMPTY))) break;
        const int c = i / C::kSf, k = i % C::kSf;  // MODE 2: scale buffer c & 1, its block k
        if (MODE == 2 && k == 0 && !(ok = wait(&sfull[c & 1], (c >> 1) & 1, DEV_TIMEOUT_LOADED)))
          break;
        tc_fence_after();
        if (lane == 0) next_full = mbar_test_wait(&full[(i + 1) % S], ((i + 1) / S) & 1);
        const uint32_t xa = smem_u32(base + s * C::kStageBytes), ya = xa + kXBytes;
        if (MODE == 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q)  // 32 e4m3 (32 bytes of the swizzled row) a step
            mma_e<0>(d, umma_desc(xa + 32 * q, 16, 1024, kLayoutSW128),
                     umma_desc(ya + 32 * q, 16, 1024, kLayoutSW128), id, q > 0);
          umma_commit_e(&empty[s]);
        } else if (MODE == 1) {
          // the smallest terms first; 16 contraction rows (2 KB) a step, 8 KB
          // between 64-column boxes, 1 KB per 8 rows
          for (int q = p.pieces - 1; q >= 0; --q)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              mma_e<1>(d, umma_desc(xa + 2048 * r, 8192, 1024, kLayoutSW128),
                       umma_desc(ya + q * C::kYPiece + 2048 * r, 8192, 1024, kLayoutSW128), id,
                       j > 0 || r > 0 || q < p.pieces - 1);
          umma_commit_e(&empty[s]);
        } else {
          const uint32_t g = smem_u32(sf) + (uint32_t)((c & 1) * C::kSf * 1024 + 512 * k);
          mx_stage1_e(d, umma_desc(xa, 16, 1024, kLayoutSW128), umma_desc(ya, 16, 1024, kLayoutSW128),
                      ((uint32_t)(BN >> 3) << 17) | (1u << 23) | ((uint32_t)(kX >> 4) << 24),
                      tmem + 2 * BN + 8u * (uint32_t)(i & 1), umma_desc(g, 128, 128, 0),
                      umma_desc(g + C::kSf * 512, 128, 128, 0), j > 0, &empty[s]);
          if (k == C::kSf - 1) umma_commit_e(&sempty[c & 1]);
        }
      }
      if (!ok) break;
      umma_commit_e(&tfull[b]);
    }
  } else {
    const int row = 32 * (warp & 3) + lane;
    const int et = threadIdx.x - 64;  // 0..127
    const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    unsigned long long acc[BN / 2];
#pragma unroll
    for (int j = 0; j < BN / 2; ++j) acc[j] = 0ull;
    bool ok = true;
    // MODE 2: the scales of blocks kSf c .. into buffer c & 1
    auto scale_words = [&](int c) {
      const int first = c * C::kSf;
      if (first >= nst) return;
      if (c >= 2 && ok) {  // the buffer's MMAs before are done
        int got = 0;
        if (lane == 0)
          got = mbar_wait_bounded(&sempty[c & 1], ((c >> 1) - 1) & 1, abort_flag, p.err,
                                  DEV_TIMEOUT_EMPTY, p.timeout_ns);
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
      }
      const int n = nst - first < C::kSf ? nst - first : C::kSf;
      uint8_t* g = sf + (c & 1) * C::kSf * 1024;
      // (both operands' loads before the first store: one latency, not two)
      uint32_t rx[C::kSf], ry[C::kSf];
      load_scale_bytes(p.scx, (int64_t)tx * kX + et, p.xrows, i0 + first, n, rx);
      load_scale_bytes(p.scy, (int64_t)ty * BN + et, et < BN ? p.ycols : 0, i0 + first, n, ry);
      store_scale_words(rx, g, et);
      store_scale_words(ry, g + C::kSf * 512, et);
      fence_proxy_async_smem();  // the tensor core's copies read them
      mbar_arrive(&sfull[c & 1]);
    };
    if (MODE == 2) scale_words(0);
    for (int u = 0; u < units; ++u) {
      const int b = u & 1;
      // the next buffer, while this one's blocks are multiplied
      if (MODE == 2 && u * C::kPerUnit % C::kSf == 0) scale_words(u * C::kPerUnit / C::kSf + 1);
      if (MODE == 0 && u % kScaleUnits == 0) {
        // the next blocks' scales, decoded, eight loads in flight a thread
        const int n = units - u < kScaleUnits ? units - u : kScaleUnits;
        named_bar_sync(1, 128);  // the blocks before are done with theirs
        stage_scales(p.scx, (int64_t)tx * kX + et, p.xrows, i0 + u, n, sx + et, 128);
        if (YVEC) {
          if (et < BN)
            stage_scales(p.scy, (int64_t)ty * BN + et, p.ycols, i0 + u, n, sy + et, C::kSy);
        } else if (et < n) {
          stage_scales(p.scy, (int64_t)ty * BN, p.ycols, i0 + u + et, 1, sy + et, 1);
        }
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
      const int us = u % kScaleUnits;
      float f = 1.0f;
      if (MODE == 0) f = YVEC ? sx[us * 128 + row] : sx[us * 128 + row] * sy[us];
      const unsigned long long s2 = pack2(f, f);
#pragma unroll
      for (int c = 0; c < BN / 16; ++c) {
        uint32_t r[16];
        tmem_ld_x16(t_lane + (uint32_t)(b * BN + 16 * c), r);
        tmem_wait_x16(r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned long long v = pack2(r[2 * j], r[2 * j + 1]);
          unsigned long long& a = acc[8 * c + j];
          if (MODE != 0) a = add2(a, v);
          else if (YVEC)
            a = fma2(mul2(v, s2), *reinterpret_cast<const unsigned long long*>(
                                      sy + us * C::kSy + 16 * c + 2 * j), a);
          else a = fma2(v, s2, a);
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty[b]);
    }
    // The finished tile into the ring: every load has been used by an MMA that
    // has completed.  Rows are the output's rows.
    const uint32_t tb = smem_u32(base);
    if (p.swap) {
#pragma unroll
      for (int j = 0; j < BN / 2; ++j) {
        const float2 v = unpack2(acc[j]);
        sts32(tb + (uint32_t)((2 * j) * 132 + row) * 4, v.x);
        sts32(tb + (uint32_t)((2 * j + 1) * 132 + row) * 4, v.y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < BN / 4; ++j) {
        const float2 v = unpack2(acc[2 * j]), w = unpack2(acc[2 * j + 1]);
        sts128(tb + (uint32_t)(row * (BN + 4) + 4 * j) * 4, make_float4(v.x, v.y, w.x, w.y));
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  if (parts > 1) cluster_sync();
  else __syncthreads();
  tc_fence_after();

  // Each CTA of the cluster adds its share of the rows over all parts, in rank
  // order, and writes them.
  {
    const int trows = p.swap ? BN : kX, tcols = p.swap ? kX : BN;
    const int pitch = tcols + 4, quads = tcols / 4, share = trows / parts;
    const int64_t m0 = p.swap ? (int64_t)ty * BN : (int64_t)tx * kX;
    const int64_t n0 = p.swap ? (int64_t)tx * kX : (int64_t)ty * BN;
    const int64_t M = p.swap ? p.ycols : p.xrows, N = p.swap ? p.xrows : p.ycols;
    const uint32_t tb = smem_u32(base);
    // four quads at a time: a load out of another CTA takes longer than the
    // whole of the work on it
    const int total = share * quads;
    for (int e0 = threadIdx.x; e0 < total; e0 += 4 * kThreads) {
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kThreads;
        if (e < total) {
          const uint32_t at =
              tb + (uint32_t)((rank * share + e / quads) * pitch + e % quads * 4) * 4;
          v[i] = parts == 1 ? lds128(at) : ld_cluster(map_rank(at, 0));
        }
      }
      for (int q = 1; q < parts; ++q) {
        float4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e0 + i * kThreads;
          if (e < total)
            w[i] = ld_cluster(map_rank(
                tb + (uint32_t)((rank * share + e / quads) * pitch + e % quads * 4) * 4, (uint32_t)q));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i].x += w[i].x; v[i].y += w[i].y; v[i].z += w[i].z; v[i].w += w[i].w;
        }
      }
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kThreads;
        if (e >= total) break;
        const int64_t m = m0 + rank * share + e / quads, n = n0 + e % quads * 4;
        if (m >= M || n >= N) continue;
        float4 x = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
        float* o = p.out + m * p.ldo + n;
        if (p.vec_ok && n + 4 <= N) {
          if (p.bias) {
            const float4 b4 = __ldg(reinterpret_cast<const float4*>(p.bias + n));
            x.x += b4.x; x.y += b4.y; x.z += b4.z; x.w += b4.w;
          }
          if (p.accumulate) {
            const float4 q = *reinterpret_cast<const float4*>(o);
            x.x += q.x; x.y += q.y; x.z += q.z; x.w += q.w;
          }
          *reinterpret_cast<float4*>(o) = activate4(x, p.act);
        } else {
          const float ve[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (n + j >= N) break;
            float w = ve[j];
            if (p.bias) w += __ldg(p.bias + n + j);
            if (p.accumulate) w += o[j];
            o[j] = activate(w, p.act);
          }
        }
      }
    }
  }

  // ------------------------------------------------------------ teardown
  __syncthreads();
  if (*abort_flag) {
    // copies in flight land before the CTA's shared memory is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (parts > 1) cluster_sync_relaxed();  // the other CTAs have read this one's part
  if (warp == 1) tmem_dealloc(tmem, C::kTmemCols);
}

// Clusters of `parts` CTAs that the GPU holds at once (a cluster lies in one GPC, so
// that there are fewer than SMs / parts).  The shared memory limit of k is set.
template <int MODE, int BN, bool YVEC>
int max_clusters(const rtb_ctx* ctx, int parts) {
  static PerDevice<4> known;  // by log2 of parts
  const int n = known.get(ctx->device, parts == 1 ? 0 : parts == 2 ? 1 : parts == 4 ? 2 : 3, [&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)parts);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<MODE, BN, YVEC>::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int most = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveClusters(&most, block_gemm_kernel<MODE, BN, YVEC>, &cfg);
    return e == cudaSuccess ? most : 0;
  });
  return n < 1 ? 1 : n;
}

// CTAs that share a tile: a power of two up to 8 with at least two blocks of the
// contraction each, such that all clusters run at once (16 tiles of 8 CTAs, one on
// an SM, take a second round for the last one: 128 x 2048 x 4096 22.8 us, 12.4 with
// four; 512 x 512 x 4096 23.0, 12.4).  With two CTAs on an SM (the query counts one)
// and eight blocks for each a few clusters may follow: a token row by 4096 x
// 4096 10.7 us with eight, 10.0 with four; 32 x 4096 x 14336 18.6, 20.8.
template <int MODE, int BN, bool YVEC>
int pick_parts(const rtb_ctx* ctx, int64_t tiles, int64_t units) {
  constexpr int kPerSm = Cfg<MODE, BN, YVEC>::kPerSm;
  int parts = 1;
  while (parts < 8 && units >= parts * 4 && tiles * parts * 2 <= kPerSm * ctx->sm_count &&
         (tiles <= (int64_t)kPerSm * max_clusters<MODE, BN, YVEC>(ctx, parts * 2) ||
          (kPerSm == 2 && units >= parts * 16)))
    parts *= 2;
  return parts;
}

template <int MODE, int BN, bool YVEC>
int launch(rtb_ctx* ctx, const CUtensorMap& tmX, const CUtensorMap& tmY, BlockParams& p,
           cudaStream_t s) {
  using C = Cfg<MODE, BN, YVEC>;
  auto* k = block_gemm_kernel<MODE, BN, YVEC>;
  cudaError_t e =
      cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return cuda_status(e, "block gemm smem attribute");
  p.tiles_x = (int)((p.xrows + kX - 1) / kX);
  p.tiles_y = (int)((p.ycols + BN - 1) / BN);
  p.stages_total = (p.depth + C::kDepth - 1) / C::kDepth;
  const int64_t tiles = (int64_t)p.tiles_x * p.tiles_y;
  if (tiles > INT32_MAX / 8) return set_error(RTB_E_UNSUPPORTED, "block gemm: too many tiles");
  p.parts = pick_parts<MODE, BN, YVEC>(ctx, tiles, (p.stages_total + C::kGrain - 1) / C::kGrain);
  p.vec_ok = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && p.ldo % 4 == 0 &&
             (!p.bias || (reinterpret_cast<uintptr_t>(p.bias) & 15u) == 0);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.parts;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  clear_stale_cuda_error();
  e = cudaLaunchKernelEx(&cfg, k, tmX, tmY, (const BlockParams)p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? RTB_OK : cuda_status(e, "block gemm launch");
}

// CTA pairs where their 256 x 256 tiles occupy more than half of the SMs.
// Measured, one CTA a tile against pairs: 512 x 4096 x 4096 (32 tiles) 23.1 us,
// 24.9; 1024 x 2048 x 1024 (32) 13.8, 14.7; 1024 x 4096 x 4096 (64) 44.3, 26.0;
// 2048 x 2048 x 512 (64) 23.2, 14.0; weight gradients with 32 and 64 tiles, 4096
// rows, 72 us, 85, and 130, 92.
bool use_pairs(const rtb_ctx* ctx, const BlockParams& p) {
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
  // side (C^T = B . A^T), so that at most 15 rows of 16, 31 of 64 are padding and
  // not 64 of 128 (16 x 8192 x 8192: 19.3 us in a loop, 3.5 TB/s of the weight).
  const bool swap = d.M <= 64;
  BlockParams p{};
  p.xrows = swap ? d.N : d.M;
  p.ycols = swap ? d.M : d.N;
  p.depth = (int)d.K;
  p.out = d.C;
  p.ldo = d.ldc;
  p.swap = swap;
  p.bias = d.bias;
  p.act = d.act;
  p.scx = swap ? d.sb : d.sa;
  p.scy = swap ? d.sa : d.sb;
  p.err = ctx->d_err;
  p.timeout_ns = ctx->timeout_ns;
  const bool yvec = p.scy.row_shift == 0;
  const int bn = swap ? (d.M <= 16 ? 16 : d.M <= 32 ? 32 : 64) : 128;
  const uint8_t* X = swap ? d.B : d.A;
  const uint8_t* Y = swap ? d.A : d.B;
  const bool pairs = !swap && use_pairs(ctx, p);
  if (pairs && !p.scx.is_f32 && !p.scy.is_f32)
    return launch_mx(ctx, X, d.lda, Y, d.ldb, p, s);
  CUtensorMap tmX, tmY;
  if ((st = make_tmap_2d_bytes(&tmX, X, 1, (uint64_t)d.K, (uint64_t)p.xrows,
                               (uint64_t)(swap ? d.ldb : d.lda), 128, kX)))
    return st;
  if ((st = make_tmap_2d_bytes(&tmY, Y, 1, (uint64_t)d.K, (uint64_t)p.ycols,
                               (uint64_t)(swap ? d.lda : d.ldb), 128, (uint32_t)bn)))
    return st;
  if (pairs) return launch_pair(ctx, 0, yvec, tmX, tmY, p, s);
  if (!p.scx.is_f32 && !p.scy.is_f32) {
    if (bn == 16) return launch<2, 16, false>(ctx, tmX, tmY, p, s);
    if (bn == 32) return launch<2, 32, false>(ctx, tmX, tmY, p, s);
    if (bn == 64) return launch<2, 64, false>(ctx, tmX, tmY, p, s);
    return launch<2, 128, false>(ctx, tmX, tmY, p, s);
  }
  if (bn == 16) return yvec ? launch<0, 16, true>(ctx, tmX, tmY, p, s) : launch<0, 16, false>(ctx, tmX, tmY, p, s);
  if (bn == 32) return yvec ? launch<0, 32, true>(ctx, tmX, tmY, p, s) : launch<0, 32, false>(ctx, tmX, tmY, p, s);
  if (bn == 64) return yvec ? launch<0, 64, true>(ctx, tmX, tmY, p, s) : launch<0, 64, false>(ctx, tmX, tmY, p, s);
  return yvec ? launch<0, 128, true>(ctx, tmX, tmY, p, s) : launch<0, 128, false>(ctx, tmX, tmY, p, s);
}

int wgrad_run(rtb_ctx* ctx, const WgradDesc& d, cudaStream_t s) {
  int st;
  if ((st = check_extents(d.rows_pad * d.pieces, d.N, d.K))) return st;
  BlockParams p{};
  p.xrows = d.K;
  p.ycols = d.N;
  p.depth = (int)d.rows;
  p.out = d.D;
  p.ldo = d.ldd;
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
  // few tiles: narrower ones, twice as many (4096 x 512 x 512, 16 tiles: 38.9 ->
  // 26.0 us; 1024^3, 64 tiles, which two CTAs share anyway: 20.7 -> 23.0)
  const int64_t tiles = ((p.xrows + 127) / 128) * ((p.ycols + 127) / 128);
  if (tiles * 3 <= ctx->sm_count) return launch<1, 64, false>(ctx, tmX, tmY, p, s);
  return launch<1, 128, false>(ctx, tmX, tmY, p, s);
}

}  // namespace rtb
