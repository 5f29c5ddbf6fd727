// 8-bit linear: Y[m][n] = (sum_k Q[m][k] W[n][k]) * (s[m] * t[n]) + b[n]
// with 8-bit codes Q (tokens) and W (output channels), FP32 scales s and t,
// the sum in 32-bit integers on the 5th-generation tensor cores
// (tcgen05.mma.kind::i8), so it is exact for K <= 131071.
//
// Tiles are transposed: the MMA's 128 rows (TMEM lanes) are output channels
// and its columns are tokens.  A few tokens then cost a few columns instead of
// a padded 128-row tile, t[n] and b[n] are one register a lane, and a warp
// writes 32 consecutive outputs of one token, whatever N, ldc or the alignment
// of Y (no vector store to fall back from).
//
// One CTA, persistent over the tiles:
//   warp 0      TMA producer: a 128 x 128 box of W and a tok x 128 box of Q a
//               stage (128-byte swizzle; what lies outside reads as zero).
//   warp 1      MMA issuer: 4 x m128 n<tok> k32 a stage; owns TMEM.
//   warps 2..5  epilogue: tcgen05.ld 32 lanes x 32 columns, scale, bias, one
//               rounding, 64-byte row segments.
// Every wait is bounded (mbar_wait_bounded).
#pragma once

#include "fmm_common.cuh"

namespace fmm {

constexpr int kI8TileN = 128;    // output channels of a tile
constexpr int kI8BlockK = 128;   // k of a stage: one 128-byte swizzle row
constexpr int kI8Threads = 192;
constexpr uint32_t kI8WBytes = kI8TileN * kI8BlockK;
constexpr int kI8MaxStages = 8;

struct Int8LinearParams {
  int64_t M, N, K;
  int64_t ldc;
  const float* token_scales;
  const float* channel_scales;
  const void* bias;  // output type, may be null
  void* out;
  int32_t tok;       // tokens of a tile, a multiple of 16, <= 256
  int32_t stages;
  int32_t tiles_m, tiles_n;
  uint32_t tmem_cols;
  uint64_t timeout_ns;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* tmap, uint32_t bar, int32_t c0,
                                            int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T in 32-bit integers, one elected thread.
__device__ __forceinline__ void tc_mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor, kind::i8: signed 8-bit A and B (both K-major), S32 D.
__host__ __device__ constexpr uint32_t idesc_i8_s32(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// One 16-bit output: scaled sum, bias, one rounding.
template <bool kBf16>
__device__ __forceinline__ uint16_t int8_output(uint32_t sum, float token_scale, float channel_scale, float bias) {
  const float v = fmaf(static_cast<float>(static_cast<int32_t>(sum)), token_scale * channel_scale, bias);
  return static_cast<uint16_t>(pack2_rn<kBf16>(v, 0.0f) & 0xffffu);
}

template <bool kBf16>
__device__ __forceinline__ float load_bias(const void* bias, int64_t n) {
  if (bias == nullptr) return 0.0f;
  if constexpr (kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
  return __half2float(static_cast<const __half*>(bias)[n]);
}

template <bool kBf16>
__global__ void __launch_bounds__(kI8Threads, 1)
    int8_linear_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_q,
                       const Int8LinearParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  const uint32_t tok_bytes = static_cast<uint32_t>(p.tok) * kI8BlockK;
  const uint32_t stage_bytes = kI8WBytes + tok_bytes;
  uint8_t* ctrl = smem_raw + (base - raw_addr) + p.stages * stage_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ctrl);
  const uint32_t full_bar = smem_u32(bars);
  const uint32_t empty_bar = smem_u32(bars + kI8MaxStages);
  const uint32_t tfull_bar = smem_u32(bars + 2 * kI8MaxStages);
  const uint32_t tempty_bar = smem_u32(bars + 2 * kI8MaxStages + 1);
  const uint32_t drain_bar = smem_u32(bars + 2 * kI8MaxStages + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kI8MaxStages + 3);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    mbar_init(tfull_bar, 1);
    mbar_init(tempty_bar, 4);  // one arrival per epilogue warp
    mbar_init(drain_bar, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_q);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int total = p.tiles_m * p.tiles_n;
  const int k_blocks = static_cast<int>((p.K + kI8BlockK - 1) / kI8BlockK);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const int tm = t / p.tiles_n, tn = t - tm * p.tiles_n;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(empty_bar + 8 * stage, phase ^ 1u, abort, p.timeout_ns, 21)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + stage * stage_bytes;
          mbar_arrive_expect_tx(full_bar + 8 * stage, stage_bytes);
          tma_load_2d(dst, &tmap_w, full_bar + 8 * stage, kb * kI8BlockK, tn * kI8TileN);
          tma_load_2d(dst + kI8WBytes, &tmap_q, full_bar + 8 * stage, kb * kI8BlockK, tm * p.tok);
          ++issued;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        // the last min(stages, issued) loads may still be landing
        int s = stage;
        uint32_t ph = phase;
        for (int n = 0; n < p.stages && n < issued; ++n) {
          if (--s < 0) {
            s = p.stages - 1;
            ph ^= 1u;
          }
          volatile int no_abort = 0;
          mbar_wait_bounded(full_bar + 8 * s, ph, &no_abort, p.timeout_ns, 25);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true, issued_any = false;
      const uint32_t idesc = idesc_i8_s32(kI8TileN, static_cast<uint32_t>(p.tok));
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        if (!mbar_wait_bounded(tempty_bar, acc_phase ^ 1u, abort, p.timeout_ns, 22)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(full_bar + 8 * stage, phase, abort, p.timeout_ns, 23)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t src = base + stage * stage_bytes;
#pragma unroll
          for (int kk = 0; kk < kI8BlockK / 32; ++kk)
            tc_mma_i8(tmem_base, smem_desc_k_sw128(src + kk * 32), smem_desc_k_sw128(src + kI8WBytes + kk * 32),
                      idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          issued_any = true;
          tc_commit(empty_bar + 8 * stage);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit(tfull_bar);
        acc_phase ^= 1u;
      }
      if (!ok && issued_any) {
        tc_commit(drain_bar);
        volatile int no_abort = 0;
        mbar_wait_bounded(drain_bar, 0, &no_abort, p.timeout_ns, 26);
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    uint32_t acc_phase = 0;
    uint16_t* out = static_cast<uint16_t*>(p.out);
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const int tm = t / p.tiles_n, tn = t - tm * p.tiles_n;
      const int64_t n = static_cast<int64_t>(tn) * kI8TileN + quarter * 32 + lane;
      const int64_t m0 = static_cast<int64_t>(tm) * p.tok;
      const int tokens = static_cast<int>(p.M - m0 < p.tok ? p.M - m0 : p.tok);
      const float channel_scale = n < p.N ? p.channel_scales[n] : 0.0f;
      const float bias = n < p.N ? load_bias<kBf16>(p.bias, n) : 0.0f;
      int ready = 0;
      if (lane == 0) ready = mbar_wait_bounded(tfull_bar, acc_phase, abort, p.timeout_ns, 24) ? 1 : 0;
      ready = __shfl_sync(0xffffffffu, ready, 0);
      if (!ready) break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < tokens; c += 32) {
        uint32_t v[32];
        tc_ld_32x32b_x32(t_addr + c, v);
        tc_wait_ld();
        const float token_scale = c + lane < tokens ? p.token_scales[m0 + c + lane] : 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float ts = __shfl_sync(0xffffffffu, token_scale, j);
          if (c + j < tokens && n < p.N)
            out[(m0 + c + j) * p.ldc + n] = int8_output<kBf16>(v[j], ts, channel_scale, bias);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty_bar);
      acc_phase ^= 1u;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, p.tmem_cols);
  }
}

}  // namespace fmm
