// 8-bit linear: Y[m][n] = (sum_k Q[m][k] W[n][k]) * (s[m] * t[n]) + b[n]
// with 8-bit codes Q (tokens) and W (output channels), FP32 scales s and t,
// the sum in 32-bit integers on the 5th-generation tensor cores
// (tcgen05.mma.kind::i8), so it is exact for K <= 131071.
//
// Tiles lie one of two ways.  With channels in the MMA's rows (TMEM lanes) and
// tokens in its columns, a few tokens cost a few columns instead of a padded
// 128-row tile, t[n] and b[n] are one register a lane, and a warp writes 32
// consecutive outputs of one token, whatever N, ldc or the alignment of Y.
// With tokens in the rows (kTokens) a lane holds 32 consecutive outputs of a
// token, which leave by TMA stores; that needs rows of Y on 16-byte boundaries
// and pays where many outputs meet a short K (50000 x 64 x 304: 31 us, 17).
//
// Three kernels:
//   int8_linear_few_kernel   a few tokens: bound by reading the weight
//   int8_linear_kernel       one SM a tile, either way
//   int8_linear_pair_kernel  two SMs a tile of 256 x 256 (many tokens)
// Every wait is bounded (mbar_wait_bounded); on a timeout all roles unwind.
#pragma once

#include "fmm_common.cuh"
#include "int8_rows.cuh"

namespace fmm {

constexpr int kI8Lanes = 128;    // MMA rows of an SM's tile
constexpr int kI8BlockK = 128;   // k of one 128-byte swizzle row
constexpr int kI8EpilogueWarps = 8;  // at most; two for each 32 TMEM lanes, every other 32 columns each
constexpr int kI8Threads = 64 + 32 * kI8EpilogueWarps;
constexpr int kI8MaxStages = 24;

struct Int8LinearParams {
  int64_t M, N, K;
  int64_t ldc;
  const float* token_scales;
  const float* channel_scales;
  const void* bias;  // output type, may be null
  void* out;
  int32_t lanes;     // MMA rows of a tile: channels (a multiple of 8, <= 128), or 128 tokens
  int32_t cols;      // MMA columns of a tile, a multiple of 16, <= 256: tokens, or channels
  int32_t stages;
  int32_t tiles_m, tiles_n;  // token tiles, channel tiles
  int32_t group_m;   // token tiles of a group, which sweeps the channel tiles together
  int32_t atoms;     // 128-deep columns of a stage
  uint32_t tmem_cols;  // columns of one of the two accumulators
  uint64_t timeout_ns;
};

// True in one lane of a converged warp.  The loops around it are run by the
// whole warp: with a single lane in them the compiler moves every descriptor
// into uniform registers by loops of its own (4096-deep tiles of 64 channels x
// 16 tokens: 13.7 us, 11.8 this way).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// Tile t -> (token tile, channel tile): groups of `group_m` token tiles sweep
// the channel tiles, so that tiles in flight share tokens and weights in L2.
__device__ __forceinline__ void int8_tile_coords(const Int8LinearParams& p, int t, int& tm, int& tn) {
  const int per_group = p.group_m * p.tiles_n;
  const int group = t / per_group, in_group = t - group * per_group;
  const int first = group * p.group_m, rows = min(p.tiles_m - first, p.group_m);
  tn = in_group / rows;
  tm = first + in_group - tn * rows;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* tmap, uint32_t bar, int32_t c0,
                                            int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T in 32-bit integers, by the lane where
// `leader` holds.  The whole warp comes here: operands that are the same in
// every lane stay in uniform registers, where the instruction reads them.
__device__ __forceinline__ void tc_mma_i8(uint32_t leader, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}

// 2-SM form, issued by one thread of the even CTA.
__device__ __forceinline__ void tc_mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, uint32_t bar_cluster, int32_t c0,
                                                 int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar_cluster), "r"(c0), "r"(c1)
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

// Scaled outputs of 32 token columns for one lane's channel: column c + j of
// the tile is token m0 + c + j, lane j holds its scale.  Instructions count: whole blocks of 32 tokens x 32 channels take two
// columns to a conversion and no predicates (9 instructions a column; 25 with a
// branch a store, which held the 256 x 256 tiles back: 4096 x 4096 x 12288
// 176 us).
template <bool kBf16>
__device__ __forceinline__ void store_columns(const Int8LinearParams& p, const uint32_t (&v)[32], int64_t m0, int c,
                                              int tokens, int64_t n, float token_scale, float channel_scale, float bias) {
  uint16_t* out = static_cast<uint16_t*>(p.out) + (m0 + c) * p.ldc + n;
  const int64_t ldc = p.ldc;
  if (c + 32 <= tokens && __all_sync(0xffffffffu, n < p.N)) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const float a = __shfl_sync(0xffffffffu, token_scale, j), b = __shfl_sync(0xffffffffu, token_scale, j + 1);
      const uint32_t two =
          pack2_rn<kBf16>(fmaf(static_cast<float>(static_cast<int32_t>(v[j])), a * channel_scale, bias),
                          fmaf(static_cast<float>(static_cast<int32_t>(v[j + 1])), b * channel_scale, bias));
      out[0] = static_cast<uint16_t>(two);
      out[ldc] = static_cast<uint16_t>(two >> 16);
      out += 2 * ldc;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float ts = __shfl_sync(0xffffffffu, token_scale, j);
    if (c + j < tokens && n < p.N) out[j * ldc] = int8_output<kBf16>(v[j], ts, channel_scale, bias);
  }
}

// Tiled TMA store (shared -> global) of one box.  Rows outside are not written,
// nor 16-byte units of a row; the unit that holds a row's end is written whole,
// so the host takes this form for rows of whole units.
__device__ __forceinline__ void tma_store_2d(const void* tmap, uint32_t src, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(src), "r"(c0), "r"(c1)
               : "memory");
}

// kTokens: 32 outputs of one lane's token, of channels n0 .. n0 + 31 (lane j
// holds the scale and bias of channel n0 + j), into this lane's row of a 32 x
// 32 block (64-byte swizzle: 16-byte unit j of row l sits at l * 64 + ((j ^ ((l
// >> 1) & 3)) << 4)), which a TMA store writes.
constexpr uint32_t kI8BlockBytes = 32 * 32 * 2;
template <bool kBf16>
__device__ __forceinline__ void store_block(const void* tmap, uint32_t buffer, const uint32_t (&v)[32], int64_t m,
                                            int64_t n0, float token_scale, float channel_scale, float bias,
                                            bool has_bias, int lane) {
  uint32_t w[16];
  if (has_bias) {
#pragma unroll
    for (int j = 0; j < 32; j += 2)
      w[j / 2] = pack2_rn<kBf16>(
          fmaf(static_cast<float>(static_cast<int32_t>(v[j])),
               token_scale * __shfl_sync(0xffffffffu, channel_scale, j), __shfl_sync(0xffffffffu, bias, j)),
          fmaf(static_cast<float>(static_cast<int32_t>(v[j + 1])),
               token_scale * __shfl_sync(0xffffffffu, channel_scale, j + 1), __shfl_sync(0xffffffffu, bias, j + 1)));
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 2)
      w[j / 2] = pack2_rn<kBf16>(static_cast<float>(static_cast<int32_t>(v[j])) *
                                     (token_scale * __shfl_sync(0xffffffffu, channel_scale, j)),
                                 static_cast<float>(static_cast<int32_t>(v[j + 1])) *
                                     (token_scale * __shfl_sync(0xffffffffu, channel_scale, j + 1)));
  }
  // the store issued from this buffer two blocks ago must have read it
  if (lane == 0) bulk_wait_group_read<1>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j)
    st_shared_v4(buffer + static_cast<uint32_t>(lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)), w[4 * j], w[4 * j + 1],
                 w[4 * j + 2], w[4 * j + 3]);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(tmap, buffer, static_cast<int32_t>(n0), static_cast<int32_t>(m));
    bulk_commit_group();
  }
}

// One accumulator of 128 lanes x `columns` (of them `count` exist) at t_addr,
// by one epilogue warp: its 32 lanes, blocks of 32 columns.  row: what the lane
// stands for; column0: what column 0 does.
template <bool kBf16, bool kTokens>
struct Int8Epilogue {
  const Int8LinearParams& p;
  const void* tmap_c;
  uint32_t buffers;  // kTokens: two blocks of this warp
  int lane, first, step;  // columns first, first + step, ... in blocks of 32
  int turn = 0;

  // scale and bias of lane's row, and the scale (and bias) of column first + lane
  float row_scale, row_bias, col_scale, col_bias;
  __device__ __forceinline__ void load_column(int64_t column0, int c, int count) {
    const bool in = c + lane < count;
    if constexpr (kTokens) {
      col_scale = in ? p.channel_scales[column0 + c + lane] : 0.0f;
      col_bias = in ? load_bias<kBf16>(p.bias, column0 + c + lane) : 0.0f;
    } else {
      col_scale = in ? p.token_scales[column0 + c + lane] : 0.0f;
    }
  }
  __device__ __forceinline__ void prepare(int64_t row, int64_t column0, int count) {
    if constexpr (kTokens) {
      row_scale = row < p.M ? p.token_scales[row] : 0.0f;
    } else {
      row_scale = row < p.N ? p.channel_scales[row] : 0.0f;
      row_bias = row < p.N ? load_bias<kBf16>(p.bias, row) : 0.0f;
    }
    load_column(column0, first, count);
  }
  __device__ __forceinline__ void drain(uint32_t t_addr, int64_t row, int64_t column0, int count) {
#pragma unroll 1
    for (int c = first; c < count; c += step) {
      uint32_t v[32];
      tc_ld_32x32b_x32(t_addr + c, v);
      const float scale = col_scale, bias = col_bias;
      load_column(column0, c + step, count);  // the next ones, before these are waited for
      tc_wait_ld();
      if constexpr (kTokens) {
        if (row - lane < p.M)  // the warp's first token
          store_block<kBf16>(tmap_c, buffers + (turn++ & 1) * kI8BlockBytes, v, row - lane, column0 + c, row_scale, scale,
                             bias, p.bias != nullptr, lane);
      } else {
        store_columns<kBf16>(p, v, column0, c, count, row, scale, row_scale, row_bias);
      }
    }
  }
  __device__ __forceinline__ void finish() {
    // the blocks must have been written before the CTA leaves
    if constexpr (kTokens) {
      if (lane == 0) bulk_wait_group_all();
      __syncwarp();
    }
  }
};

// Structure (persistent over the tiles; 2 x tmem_cols accumulator columns, so
// that the epilogue of a tile runs beside the next one's products):
//   warp 0      TMA producer: `atoms` lanes x 128 and cols x 128 boxes a stage
//               (128-byte swizzle; what lies outside reads as zero).
//   warp 1      MMA issuer: 4 x m128 n<cols> k32 a box; owns TMEM.
//   warps 2..9  epilogue: tcgen05.ld 32 lanes x 32 columns, scale, bias, one
//               rounding, 64-byte row segments.  Eight warps, because one to
//               a scheduler waits for its own results (20000 x 256 x 1000:
//               35 us with four).
// A tile may have fewer than 128 channels, so that a few tokens' tiles, which
// cost the weight's bytes and little else, come out even over the SMs; the
// product runs over 128 rows of shared memory all the same and the sums of the
// rows behind the tile, whatever they are, are not read.
template <bool kBf16, bool kTokens>
__global__ void __launch_bounds__(kI8Threads, 1)
    int8_linear_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                       const __grid_constant__ CUtensorMap tmap_c, const Int8LinearParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  const uint32_t b_bytes = static_cast<uint32_t>(p.cols) * kI8BlockK;
  const uint32_t a_bytes = static_cast<uint32_t>(p.lanes) * kI8BlockK;
  const uint32_t stage_bytes = p.atoms * (a_bytes + b_bytes);
  // columns first: the products read 128 rows of the other operand, into the
  // next stage or, at the end, into what the host adds behind the last one
  const uint32_t blocks = base + p.stages * stage_bytes + (kI8Lanes - p.lanes) * kI8BlockK;
  uint8_t* ctrl = smem_raw + (blocks - raw_addr) + (kTokens ? kI8EpilogueWarps * 2 * kI8BlockBytes : 0);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ctrl);
  const uint32_t full_bar = smem_u32(bars);
  const uint32_t empty_bar = smem_u32(bars + kI8MaxStages);
  const uint32_t tfull_bar = smem_u32(bars + 2 * kI8MaxStages);       // [2]
  const uint32_t tempty_bar = smem_u32(bars + 2 * kI8MaxStages + 2);  // [2]
  const uint32_t drain_bar = smem_u32(bars + 2 * kI8MaxStages + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kI8MaxStages + 5);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int total = p.tiles_m * p.tiles_n;
  const int columns = static_cast<int>((p.K + kI8BlockK - 1) / kI8BlockK);  // 128 codes each

  // the producer's place: tile, column, stage; one call waits for a stage, loads it and moves on
  int load_t = blockIdx.x, load_kb = 0, load_stage = 0, issued = 0, load_m = 0, load_n = 0;
  uint32_t load_phase = 0;
  bool load_ok = true;
  if (load_t < total) int8_tile_coords(p, load_t, load_m, load_n);
  auto load_stage_next = [&] {
    load_ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty_bar + 8 * load_stage, load_phase ^ 1u, abort,
                                                        p.timeout_ns, 21));
    if (!load_ok) return;
    if (elect_one()) {
      const int atoms = min(p.atoms, columns - load_kb);
      const uint32_t bar = full_bar + 8 * load_stage;
      uint32_t dst = base + load_stage * stage_bytes;
      mbar_arrive_expect_tx(bar, atoms * (a_bytes + b_bytes));
      for (int at = 0; at < atoms; ++at) {
        tma_load_2d(dst + b_bytes, &tmap_a, bar, (load_kb + at) * kI8BlockK, (kTokens ? load_m : load_n) * p.lanes);
        tma_load_2d(dst, &tmap_b, bar, (load_kb + at) * kI8BlockK, (kTokens ? load_n : load_m) * p.cols);
        dst += a_bytes + b_bytes;
      }
    }
    __syncwarp();
    ++issued;
    if (++load_stage == p.stages) {
      load_stage = 0;
      load_phase ^= 1u;
    }
    if ((load_kb += p.atoms) >= columns) {
      load_kb = 0;
      load_t += gridDim.x;
      if (load_t < total) int8_tile_coords(p, load_t, load_m, load_n);
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar + 8 * b, 1);
      mbar_init(tempty_bar + 8 * b, kI8EpilogueWarps);  // one arrival each
    }
    mbar_init(drain_bar, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    if (kTokens) prefetch_tmap(&tmap_c);
  }
  if (warp == 0) {
    // the ring is filled while tensor memory is being allocated
    __syncwarp();
    wait_for_previous_kernel();
    while (issued < p.stages && load_t < total && load_ok) load_stage_next();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 2 * p.tmem_cols);
    tmem_relinquish();
  }
  wait_for_previous_kernel();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Behind the barrier that follows the allocation: a CTA of the next kernel
  // allocates before it waits for this one, and must not take the columns first
  // if it ever fits beside this CTA.
  let_next_kernel_start();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    while (load_t < total && load_ok) load_stage_next();
    if (!load_ok) {
      // the last min(stages, issued) loads may still be landing
      for (int n = 0; n < p.stages && n < issued; ++n) {
        if (--load_stage < 0) {
          load_stage = p.stages - 1;
          load_phase ^= 1u;
        }
        volatile int no_abort = 0;
        mbar_wait_bounded(full_bar + 8 * load_stage, load_phase, &no_abort, p.timeout_ns, 25);
      }
    }
  } else if (warp == 1) {
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true, issued_any = false;
    const uint32_t idesc = idesc_i8_s32(kI8Lanes, static_cast<uint32_t>(p.cols));
    const uint64_t b_desc0 = smem_desc_k_sw128(base), a_desc0 = smem_desc_k_sw128(base + b_bytes);
    const uint32_t atom_step = (a_bytes + b_bytes) >> 4, stage_step = stage_bytes >> 4;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(tempty_bar + 8 * acc, acc_phase ^ 1u, abort, p.timeout_ns, 22));
      if (!ok) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * p.tmem_cols;
      for (int kb = 0; kb < columns; kb += p.atoms) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(full_bar + 8 * stage, phase, abort, p.timeout_ns, 23));
        if (!ok) break;
        tc_fence_after();
        const int atoms = min(p.atoms, columns - kb);
        const uint32_t leader = elect_one();
        uint64_t b_desc = b_desc0 + stage * stage_step, a_desc = a_desc0 + stage * stage_step;
        for (int at = 0; at < atoms; ++at) {
#pragma unroll
          for (int kk = 0; kk < kI8BlockK / 32; ++kk)  // 32 codes on, 32 bytes on
            tc_mma_i8(leader, d_tmem, a_desc + kk * 2, b_desc + kk * 2, idesc, (kb > 0 || at > 0 || kk > 0) ? 1u : 0u);
          b_desc += atom_step;
          a_desc += atom_step;
        }
        if (leader) tc_commit(empty_bar + 8 * stage);
        __syncwarp();
        issued_any = true;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if (elect_one()) tc_commit(tfull_bar + 8 * acc);
      __syncwarp();
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (!ok && issued_any) {
      if (elect_one()) tc_commit(drain_bar);
      __syncwarp();
      volatile int no_abort = 0;
      mbar_wait_bounded(drain_bar, 0, &no_abort, p.timeout_ns, 26);
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    const int block = warp - 2;
    Int8Epilogue<kBf16, kTokens> epilogue{p, &tmap_c, blocks + block * 2 * kI8BlockBytes, lane, block / 4 * 32,
                                           kI8EpilogueWarps / 4 * 32};
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      int tm, tn;
      int8_tile_coords(p, t, tm, tn);
      // lanes behind the tile or the operand stand for its end
      const int64_t lane_end = kTokens ? p.M : p.N, lane0 = static_cast<int64_t>(kTokens ? tm : tn) * p.lanes;
      const int64_t row = quarter * 32 + lane < p.lanes ? lane0 + quarter * 32 + lane : lane_end;
      const int64_t column0 = static_cast<int64_t>(kTokens ? tn : tm) * p.cols;
      const int64_t rest = (kTokens ? p.N : p.M) - column0;
      const int count = static_cast<int>(rest < p.cols ? rest : p.cols);
      epilogue.prepare(row, column0, count);
      int ready = 0;
      if (lane == 0) ready = mbar_wait_bounded(tfull_bar + 8 * acc, acc_phase, abort, p.timeout_ns, 24) ? 1 : 0;
      ready = __shfl_sync(0xffffffffu, ready, 0);
      if (!ready) break;
      tc_fence_after();
      if (quarter * 32 < p.lanes)
        epilogue.drain(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * p.tmem_cols, row, column0, count);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty_bar + 8 * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    epilogue.finish();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * p.tmem_cols);
  }
}

// ---------------------------------------------------------------------------
// 2-SM form: a cluster of two CTAs computes a tile of 256 channels x 256 tokens
// with tcgen05.mma.cta_group::2.  CTA r holds channels [128 r, 128 r + 128) and
// its half of the tokens, so an SM loads 32 KB a 128-deep block
// for twice the products that the same bytes give one SM alone: at the full
// rate L2 and shared memory are what bounds the product, not the tensor cores.
// Roles as above; the even CTA issues the products, loads complete on its
// barriers, and each CTA's epilogue drains its own 128 channels.
struct Int8PairConfig {
  static constexpr int kTile = 256;
  static constexpr int kAtoms = 2;  // 128-deep columns of swizzle atoms a stage
  static constexpr int kBK = kAtoms * kI8BlockK;
  static constexpr int kStages = 3;
  static constexpr uint32_t kAtomBytes = 128 * kI8BlockK;      // this CTA's half of an operand
  static constexpr uint32_t kABytes = kAtoms * kAtomBytes;     // 32 KB
  static constexpr uint32_t kStageBytes = 2 * kABytes;         // 64 KB
  static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + 1024 + 8 * (2 * kStages + 8);
};

template <bool kBf16>
__global__ void __launch_bounds__(kI8Threads, 1)
    int8_linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                            const __grid_constant__ CUtensorMap tmap_b16, const Int8LinearParams p) {
  using Cfg = Int8PairConfig;
  constexpr int STAGES = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + (base - raw_addr) + STAGES * Cfg::kStageBytes);
  const uint32_t full_bar = smem_u32(bars);                     // [STAGES], used in CTA 0
  const uint32_t empty_bar = smem_u32(bars + STAGES);           // [STAGES], each CTA
  const uint32_t tfull_bar = smem_u32(bars + 2 * STAGES);       // [2], each CTA
  const uint32_t tempty_bar = smem_u32(bars + 2 * STAGES + 2);  // [2], used in CTA 0
  const uint32_t drain_bar = smem_u32(bars + 2 * STAGES + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 5);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int epilogue_warps = blockDim.x / 32 - 2;  // 4 or 8
  const uint32_t cta = cluster_cta_rank();  // 0 = even CTA (issues the MMAs)
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar + 8 * b, 1);
      mbar_init(tempty_bar + 8 * b, 2 * epilogue_warps);  // of both CTAs
    }
    mbar_init(drain_bar, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    prefetch_tmap(&tmap_b16);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 2 * Cfg::kTile);
    tmem_relinquish_pair();
  }
  wait_for_previous_kernel();
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  let_next_kernel_start();  // behind the allocation, as above
  const uint32_t tmem_base = *tmem_slot;

  const int total = p.tiles_m * p.tiles_n;
  const int k_blocks = static_cast<int>((p.K + Cfg::kBK - 1) / Cfg::kBK);
  // columns of tile tm: the MMA's N, 16 from each CTA at least
  auto columns = [&](int tm) {
    const int64_t rest = p.M - static_cast<int64_t>(tm) * Cfg::kTile;
    return rest >= Cfg::kTile ? Cfg::kTile : static_cast<int>((rest + 31) / 32 * 32);
  };

  if (warp == 0) {
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = pair; t < total && ok; t += pairs) {
      int tm, tn;
      int8_tile_coords(p, t, tm, tn);
      // each CTA supplies half of the tokens; a ragged last tile loads
      // exactly its half in 16-row boxes, since a 128-row box would fetch
      // rows that belong to the other half
      const int n_cols = columns(tm), half = n_cols / 2;
      const int a_row = tn * Cfg::kTile + static_cast<int>(cta) * 128;
      const int b_row = tm * Cfg::kTile + static_cast<int>(cta) * half;
      const uint32_t stage_tx = 2u * (Cfg::kABytes + static_cast<uint32_t>(half) * Cfg::kBK);
      for (int kb = 0; kb < k_blocks; ++kb) {
        ok = __all_sync(0xffffffffu,
                        mbar_wait_bounded_cluster(empty_bar + 8 * stage, phase ^ 1u, abort, p.timeout_ns, 41));
        if (!ok) break;
        if (elect_one()) {
          const uint32_t full_even = map_to_cta(full_bar + 8 * stage, 0);
          if (cta == 0) mbar_arrive_expect_tx(full_bar + 8 * stage, stage_tx);
#pragma unroll
          for (int at = 0; at < Cfg::kAtoms; ++at) {
            const int k0 = kb * Cfg::kBK + at * kI8BlockK;
            const uint32_t a_dst = base + stage * Cfg::kStageBytes + at * Cfg::kAtomBytes;
            const uint32_t b_dst = a_dst + Cfg::kABytes;
            tma_load_2d_pair(a_dst, &tmap_a, full_even, k0, a_row);
            if (n_cols == Cfg::kTile) {
              tma_load_2d_pair(b_dst, &tmap_b, full_even, k0, b_row);
            } else {
              for (int j = 0; j < half; j += 16)
                tma_load_2d_pair(b_dst + static_cast<uint32_t>(j) * kI8BlockK, &tmap_b16, full_even, k0, b_row + j);
            }
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && issued > 0) {
      // loads may still be landing in this CTA's shared memory (they complete
      // on the even CTA's barrier): give them time before the CTA unwinds
      const uint64_t start = globaltimer_ns();
      while (globaltimer_ns() - start < 200000ull) {
      }
    }
  } else if (warp == 1) {
    if (cta == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true, issued_any = false;
      const uint64_t a_desc0 = smem_desc_k_sw128(base), b_desc0 = smem_desc_k_sw128(base + Cfg::kABytes);
      for (int t = pair; t < total && ok; t += pairs) {
        int tm, tn;
        int8_tile_coords(p, t, tm, tn);
        const uint32_t idesc = idesc_i8_s32(Cfg::kTile, static_cast<uint32_t>(columns(tm)));
        ok = __all_sync(0xffffffffu,
                        mbar_wait_bounded_cluster(tempty_bar + 8 * acc, acc_phase ^ 1u, abort, p.timeout_ns, 42));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * Cfg::kTile);
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait_bounded_cluster(full_bar + 8 * stage, phase, abort, p.timeout_ns, 43));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t a_desc = a_desc0 + stage * (Cfg::kStageBytes >> 4);
            const uint64_t b_desc = b_desc0 + stage * (Cfg::kStageBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < Cfg::kBK / 32; ++kk) {
              const uint32_t at = (kk / 4) * (Cfg::kAtomBytes >> 4) + (kk % 4) * 2;
              tc_mma_i8_pair(d_tmem, a_desc + at, b_desc + at, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
            }
            tc_commit_pair_multicast(empty_bar + 8 * stage, 0x3);
          }
          __syncwarp();
          issued_any = true;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (elect_one()) tc_commit_pair_multicast(tfull_bar + 8 * acc, 0x3);
        __syncwarp();
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok && issued_any) {
        if (elect_one()) tc_commit_pair_multicast(drain_bar, 0x1);
        __syncwarp();
        volatile int no_abort = 0;
        mbar_wait_bounded(drain_bar, 0, &no_abort, p.timeout_ns, 46);
      }
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t tempty_even = map_to_cta(tempty_bar, 0);
    Int8Epilogue<kBf16, false> epilogue{p, nullptr, 0u, lane, (warp - 2) / 4 * 32, epilogue_warps / 4 * 32};
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = pair; t < total; t += pairs) {
      int tm, tn;
      int8_tile_coords(p, t, tm, tn);
      const int64_t row = static_cast<int64_t>(tn) * Cfg::kTile + static_cast<int>(cta) * 128 + quarter * 32 + lane;
      const int64_t column0 = static_cast<int64_t>(tm) * Cfg::kTile;
      const int count = static_cast<int>(p.M - column0 < Cfg::kTile ? p.M - column0 : Cfg::kTile);
      epilogue.prepare(row, column0, count);
      int ready = 0;
      if (lane == 0)
        ready = mbar_wait_bounded_cluster(tfull_bar + 8 * acc, acc_phase, abort, p.timeout_ns, 44) ? 1 : 0;
      ready = __shfl_sync(0xffffffffu, ready, 0);
      if (!ready) break;
      tc_fence_after();
      epilogue.drain(
          tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * Cfg::kTile), row, column0,
          count);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(tempty_even + 8 * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
  }

  tc_fence_before();
  cluster_sync_all();  // nobody leaves while the pair may still touch its memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * Cfg::kTile);
  }
}

// ---------------------------------------------------------------------------
// Few tokens: Y = Q W^T is bound by reading W once, and by the time from the
// launch to the last store.  Nothing is shared between warps: each takes units
// of four channels in turn, whose rows come through a ring of its own in shared
// memory by bulk copies (issued by the warp itself, running on across units),
// against the tokens' codes, which the CTA keeps in shared memory.  Products
// are dot products of four codes; a lane sums every 32nd 16-code piece of a
// row, and the lanes' 32-bit sums are added at the row's end.  Units of four
// channels spread W over all SMs (tiles of 128 leave a third of them idle at
// N = 12288), and neither tensor maps nor tensor memory are set up first.
//   MT: tokens, rounded up.
constexpr int kI8FewK = 1024;  // codes of a row in a stage
constexpr int kI8FewMaxWarps = 16, kI8FewMaxStages = 8;

struct Int8FewParams {
  const int8_t* codes;
  const int8_t* weight;
  int64_t ldq, ldw, ldc, N;
  const float* token_scales;
  const float* channel_scales;
  const void* bias;
  void* out;
  int32_t M, K;
  int32_t units, stages;
  uint64_t timeout_ns;
};

// 16 codes of a row from `k` on; what lies past K is zero and not read.
__device__ __forceinline__ uint4 load_codes(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
  if (k < K) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k + i < K) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i % 4));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int c) {
  c = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), c);
  c = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), c);
  c = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), c);
  return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), c);
}

template <bool kBf16, int MT, int R>
__global__ void __launch_bounds__(32 * kI8FewMaxWarps, 1) int8_linear_few_kernel(const Int8FewParams p) {
  constexpr uint32_t kStageBytes = R * kI8FewK;
  static_assert(MT * R <= 32, "an output a lane");
  __shared__ __align__(8) uint64_t s_full[kI8FewMaxWarps * kI8FewMaxStages];
  __shared__ int s_abort[kI8FewMaxWarps];
  extern __shared__ __align__(128) uint8_t s_few[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
  const uint32_t full_bar = smem_u32(s_full + warp * kI8FewMaxStages);
  const int pitch = (p.K + 15) / 16 * 16;  // of a token's codes
  uint8_t* ring = s_few + warp * p.stages * kStageBytes;
  uint8_t* tokens = s_few + warps * p.stages * kStageBytes;
  const int k_stages = (p.K + kI8FewK - 1) / kI8FewK;
  const int whole = p.K & ~15;  // codes that copies move; the rest of a row is read in place

  // this warp's units and stages, in the order in which they are copied
  const int unit0 = warp * gridDim.x + blockIdx.x, unit_step = warps * gridDim.x;
  int copy_unit = unit0, copy_ks = 0;
  auto copy = [&](int stage) {
    if (copy_unit >= p.units) return;
    const int64_t n0 = static_cast<int64_t>(copy_unit) * R;
    const int rows = static_cast<int>(p.N - n0 < R ? p.N - n0 : R), k0 = copy_ks * kI8FewK;
    const int bytes = max(0, min(kI8FewK, whole - k0));
    const uint32_t bar = full_bar + 8 * stage;
    if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(rows * bytes));
    __syncwarp();
    if (lane < rows && bytes > 0)
      bulk_load(smem_u32(ring) + stage * kStageBytes + lane * kI8FewK, p.weight + (n0 + lane) * p.ldw + k0,
                static_cast<uint32_t>(bytes), bar);
    if (++copy_ks == k_stages) {
      copy_ks = 0;
      copy_unit += unit_step;
    }
  };
  if (lane == 0) {
    s_abort[warp] = 0;
    for (int s = 0; s < p.stages; ++s) mbar_init(full_bar + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  let_next_kernel_start();
  wait_for_previous_kernel();
  for (int s = 0; s < p.stages; ++s) copy(s);
  // the tokens, zero past K
  for (int i = threadIdx.x; i < p.M * (pitch / 16); i += blockDim.x) {
    const int m = i / (pitch / 16), k = (i - m * (pitch / 16)) * 16;
    *reinterpret_cast<uint4*>(tokens + m * pitch + k) = load_codes(p.codes + m * p.ldq, k, p.K);
  }
  // lane m * R + r stores the output of token m and channel r of the unit
  const int out_m = lane / R, out_r = lane % R;
  const float token_scale = out_m < p.M ? p.token_scales[out_m] : 0.0f;
  __syncthreads();

  int stage = 0;
  uint32_t phase = 0;
  for (int unit = unit0; unit < p.units; unit += unit_step) {
    const int64_t n0 = static_cast<int64_t>(unit) * R, n = n0 + out_r;
    const float channel_scale = n < p.N ? p.channel_scales[n] : 0.0f;
    const float bias = n < p.N ? load_bias<kBf16>(p.bias, n) : 0.0f;
    int sum[MT][R];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) sum[m][r] = 0;
    for (int ks = 0; ks < k_stages; ++ks) {
      mbar_wait_bounded(full_bar + 8 * stage, phase, &s_abort[warp], p.timeout_ns, 51);
      const uint8_t* from = ring + stage * kStageBytes;
#pragma unroll
      for (int i = 0; i < kI8FewK / 512; ++i) {
        const int at = i * 512 + lane * 16, k = ks * kI8FewK + at;
        if (k >= p.K) continue;
        uint4 w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = *reinterpret_cast<const uint4*>(from + r * kI8FewK + at);
        if (k >= whole) {
#pragma unroll
          for (int r = 0; r < R; ++r)
            w[r] = n0 + r < p.N ? load_codes(p.weight + (n0 + r) * p.ldw, k, p.K) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (m >= p.M) break;
          const uint4 q = *reinterpret_cast<const uint4*>(tokens + m * pitch + k);
#pragma unroll
          for (int r = 0; r < R; ++r) sum[m][r] = dot16(w[r], q, sum[m][r]);
        }
      }
      // all lanes hold their pieces: the stage may be filled again
      if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&s_abort[warp]) != 0)) break;
      copy(stage);
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (__any_sync(0xffffffffu, *static_cast<volatile int*>(&s_abort[warp]) != 0)) break;
    int mine = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int all = __reduce_add_sync(0xffffffffu, sum[m][r]);
        mine = lane == m * R + r ? all : mine;
      }
    if (out_m < p.M && n < p.N)
      static_cast<uint16_t*>(p.out)[out_m * p.ldc + n] =
          int8_output<kBf16>(static_cast<uint32_t>(mine), token_scale, channel_scale, bias);
  }
  if (s_abort[warp] != 0 && lane == 0) {
    // copies into this warp's ring may still be landing: give each its limit
    volatile int no_abort = 0;
    for (int s = 0; s < p.stages; ++s)
      mbar_wait_bounded(full_bar + 8 * s, s < stage ? phase ^ 1u : phase, &no_abort, p.timeout_ns, 52);
  }
}

}  // namespace fmm
