// Rows to 8-bit codes: symmetric integers with one FP32 scale a row.
//
//   quantize_rows   p = x                              s = a / 127
//   rms_norm_int8   h = rnd(x + r), p = h * g          s = a * rstd / 127
//                   rstd = 1 / sqrt(mean(h^2) + eps)
//   a = max |p| over the row,  q = round_half_even(127 p / a)
//
// rstd cancels in q, so one reduction (sum of squares and maximum together)
// separates the read of a row from its write: a row stays on the chip in
// between and every element crosses HBM once.
//
// Codes are those of exact arithmetic.  p is exact in FP32 where x and g have
// 16 bits (at most 22 significant bits); with an FP32 gain the threads that
// hold the largest rounded p look its FP64 value up.  Rows whose products or
// squares leave FP32's range, below or above, are taken once more in FP64
// (take_row_wide).  127 / a is rounded, so each product is taken by the FP32
// numbers on either side of it; where the two codes differ (1 product in 10^5),
// 254 p and (2c + 1) a are compared in FP64, exact on both sides.
//
// A row with an infinity or a NaN (or, in the norm, with a square or a scale
// beyond FP32) has codes 0 and a NaN scale: whatever is computed from it is NaN.
// A row of zeros has codes 0 and scale 0.
//
// Two kernels.  Few rows: a block (or a warp) a row, the row in registers, for
// the shortest way from the first byte to the last.  Many rows: bound by HBM,
// so rows arrive by bulk copies in a ring of shared memory and instructions are
// counted (see int8_rows_streamed_kernel).
#pragma once

#include <type_traits>

#include "fmm_common.cuh"

namespace fmm {

// Launches of the 8-bit kernels overlap the end of the kernel before them in
// the stream (programmatic stream serialisation): a CTA may be set up early, and
// waits here until that kernel has finished and its writes can be seen.  Every
// thread calls it before it reads or writes global memory, and before any wait
// with a limit, which would count the other kernel's time.
__device__ __forceinline__ void wait_for_previous_kernel() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// From here on the next kernel's CTAs may be set up where there is room; a kernel
// with tensor memory calls it once its own allocation is made.
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;"); }

constexpr int kRowsMaxThreads = 1024;
constexpr int kRowsNormThreads = 768;  // streamed norms: 80 registers a thread (65536 x 4608: 349 us with 64, 334)

struct Int8RowsParams {
  const void* x;
  const void* residual;  // null: no addition
  void* residual_out;
  const void* gain;
  int8_t* codes;
  float* scales;
  int64_t rows;
  int64_t ldx, ldr, ldo, ldq;
  int32_t cols;
  float eps;
  float eps_sum;  // eps * cols
  // register form: > 1: the block is one row's; 1: every warp has a row of its own.
  // Streamed form: the warps of a group
  int32_t warps_per_row;
  // streamed form: rows of a block at work, ring stages of each, and the waits' limit
  int32_t groups, stages;
  uint64_t timeout_ns;
};

// 8 consecutive elements as FP32, from a 16-byte aligned address (two for FP32).
template <class T>
struct RowVec;
template <>
struct RowVec<float> {
  static __device__ __forceinline__ void load(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct RowVec<__nv_bfloat16> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2_rn<true>(a, b); }
  static __device__ __forceinline__ __nv_bfloat16 rnd(float a) { return __float2bfloat16_rn(a); }
  static __device__ __forceinline__ float wide(__nv_bfloat16 a) { return __bfloat162float(a); }
};
template <>
struct RowVec<__half> {
  static __device__ __forceinline__ void load(const __half* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      f[2 * e] = t.x;
      f[2 * e + 1] = t.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2_rn<false>(a, b); }
  static __device__ __forceinline__ __half rnd(float a) { return __float2half_rn(a); }
  static __device__ __forceinline__ float wide(__half a) { return __half2float(a); }
};

// round_half_even(127 P / M) where it is `below` or `below + 1`, M > 0, P and M
// of at most 44 significant bits: both sides of the comparison are exact.
__device__ __forceinline__ int exact_code(double P, double M, int below) {
  const double value = 254.0 * P, border = (2 * below + 1) * M;
  return value > border || (value == border && (below & 1)) ? below + 1 : below;
}

// The larger of m and |a|, |b|; NaN if one of them is.
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
  return m;
}

// What the row reduction gives: the sum of squares (norm only) and the bits of
// the largest |p|, which compare as the values do, infinities and NaN above
// all finite ones.
struct RowTotals {
  float square;
  uint32_t peak;
};

template <bool kNorm>
__device__ __forceinline__ RowTotals warp_totals(RowTotals t) {
  if constexpr (kNorm) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) t.square += __shfl_xor_sync(0xffffffffu, t.square, d);
  }
  t.peak = __reduce_max_sync(0xffffffffu, t.peak);
  return t;
}

// What a row's totals say about its codes.  A plain row multiplies by 127 / a,
// computed from both sides: by `low` and by `high`, a few steps of FP32 apart
// with the exact quotient between them.  Where both give the same code it is
// the exact one; where they differ, the product is next to a border.  Rows that
// are not plain are zeros, not finite, or so small or large that FP32's products,
// squares, 127 / a or the scale lose digits.
struct RowScale {
  bool plain;
  float low, high;
};
// 2^low <= the positive number of these bits < 2^high
__device__ __forceinline__ bool within(uint32_t bits, int low, int high) {
  return bits - (static_cast<uint32_t>(low + 127) << 23) < static_cast<uint32_t>(high - low) << 23;
}
// kPair: the product and the peak are rounded too
template <bool kNorm, bool kPair>
__device__ __forceinline__ RowScale row_scale(const RowTotals& total, float eps_sum) {
  RowScale s;
  const float peak = __uint_as_float(total.peak);
  // false for NaN; a norm's scale, at most 2^50 a / 127, stays in FP32
  s.plain = within(total.peak, -100, kNorm ? 50 : 100);
  // Squares lose digits below 2^-126, 2^-150 each at most: nothing beside a mean and
  // epsilon of 2^-100 and more (rows have up to 2^30 elements)
  if (kNorm) s.plain = s.plain && within(__float_as_uint(total.square + eps_sum), -70, 128);
  // the quotient is at most half a step off, the pair's other two roundings a step more each
  constexpr uint32_t kSteps = kPair ? 3 : 1;
  const uint32_t middle = __float_as_uint(127.0f / peak);
  s.low = __uint_as_float(middle - kSteps);
  s.high = __uint_as_float(middle + kSteps);
  return s;
}
template <bool kNorm>
__device__ __forceinline__ float stored_scale(const RowTotals& total, int cols, float eps) {
  float scale = __uint_as_float(total.peak);
  if (kNorm) scale = scale / sqrtf(total.square / static_cast<float>(cols) + eps);
  return scale / 127.0f;
}

// x + kMagic rounds x to an integer, the low byte of the sum: no conversions,
// which run at an eighth of the rate.
constexpr float kMagic = 0x1.8p23f;

// Codes (low bytes) of 8 products of a plain row; the result has a bit set
// where a product is next to a border.
__device__ __forceinline__ uint32_t codes_of(const float (&p)[8], const RowScale& s, float (&code)[8],
                                            float (&other)[8]) {
  uint32_t differ = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    code[e] = fmaf(p[e], s.low, kMagic);
    other[e] = fmaf(p[e], s.high, kMagic);
    differ |= __float_as_uint(code[e]) ^ __float_as_uint(other[e]);
  }
  return differ;
}
__device__ __forceinline__ uint32_t border_mask(const float (&code)[8], const float (&other)[8]) {
  uint32_t mask = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) mask |= code[e] != other[e] ? 1u << e : 0u;
  return mask;
}

// Four codes: the low bytes of four words.
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  const uint32_t low = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t high = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(low, high, 0x5410);
}
__device__ __forceinline__ uint2 pack_codes(const float (&code)[8]) {
  return make_uint2(pack_codes(code[0], code[1], code[2], code[3]), pack_codes(code[4], code[5], code[6], code[7]));
}

// h + f rounded to the stream's type: the 8 elements as stored, and in h.
template <class T>
__device__ __forceinline__ uint4 add_vec(float (&h)[8], const float (&f)[8]) {
  uint4 w;
  w.x = RowVec<T>::pack(h[0] + f[0], h[1] + f[1]);
  w.y = RowVec<T>::pack(h[2] + f[2], h[3] + f[3]);
  w.z = RowVec<T>::pack(h[4] + f[4], h[5] + f[5]);
  w.w = RowVec<T>::pack(h[6] + f[6], h[7] + f[7]);
  RowVec<T>::load(reinterpret_cast<const T*>(&w), h);
  return w;
}

// The code of a plain row's product next to a border, P its FP64 value.
__device__ __forceinline__ int8_t settled_code(double P, double exact_peak, const RowScale& s) {
  const int below = static_cast<int>(floorf(static_cast<float>(P) * s.low));
  return static_cast<int8_t>(exact_code(P, exact_peak, below));
}

// round_half_even(127 P / M) without a guess at hand, 0 < M, |P| <= M.  The floor may
// be one off next to an integer: both codes that it leaves are looked at.
__device__ __forceinline__ int8_t wide_code(double P, double M) {
  return static_cast<int8_t>(exact_code(P, M, static_cast<int>(floor(127.0 * P / M))));
}

// One row in FP64, where its products are exact (48 bits at most, between 2^-282
// and 2^256), by the `width` threads that had it: a warp, or those of named
// barrier `barrier` with a word of `squares` and `peaks` for each warp.  Reads
// h, the stream in memory, in the order in which its own threads wrote it.
template <class T, class G, bool kNorm, bool kVec>
__device__ __forceinline__ void take_row_wide(const T* h, const G* gain, int8_t* codes, float* scale, int cols, float eps,
                                              int t, int width, int barrier, double* squares, unsigned long long* peaks) {
  constexpr int kRun = kVec ? 8 : 1;  // consecutive elements of a thread
  auto product = [&](int c) {
    double P = static_cast<double>(RowVec<T>::one(h + c));
    if constexpr (kNorm) P *= static_cast<double>(RowVec<G>::one(gain + c));
    return P;
  };
  double square = 0.0;
  unsigned long long bits = 0;  // of the largest |p|, which compare as the values do, NaN above infinities
#pragma unroll 1
  for (int c0 = kRun * t; c0 < cols; c0 += kRun * width)
#pragma unroll 1
    for (int c = c0; c < min(c0 + kRun, cols); ++c) {
      const float v = RowVec<T>::one(h + c);
      if (kNorm) {
        // a square beyond FP32 makes the row one that is not finite
        const float low = v * v;
        square += __float_as_uint(low) < 0x7f800000u ? static_cast<double>(v) * v : static_cast<double>(low);
      }
      const unsigned long long mine = static_cast<unsigned long long>(__double_as_longlong(fabs(product(c))));
      bits = mine > bits ? mine : bits;
    }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    square += __shfl_xor_sync(0xffffffffu, square, d);
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
  }
  if (width > 32) {
    if (t % 32 == 0) {
      squares[t / 32] = square;
      peaks[t / 32] = bits;
    }
    named_barrier_sync(barrier, width);
    square = 0.0;
#pragma unroll 1
    for (int w = 0; w < width / 32; ++w) {
      square += squares[w];
      bits = max(bits, peaks[w]);
    }
    named_barrier_sync(barrier, width);  // the next row writes them
  }
  const double peak = __longlong_as_double(static_cast<long long>(bits));
  double s = peak / 127.0;
  if (kNorm && peak > 0.0) s /= sqrt(square / cols + static_cast<double>(eps));
  // a scale beyond FP32 is not finite either
  const bool finite = s <= static_cast<double>(3.402823466e38f) && (!kNorm || square < static_cast<double>(INFINITY));
  const bool zero = !finite || peak == 0.0;
  if (t == 0) *scale = finite ? static_cast<float>(s) : __uint_as_float(0x7fc00000u);
#pragma unroll 1
  for (int c0 = kRun * t; c0 < cols; c0 += kRun * width)
#pragma unroll 1
    for (int c = c0; c < min(c0 + kRun, cols); ++c) codes[c] = zero ? 0 : wide_code(product(c), peak);
}

// ---------------------------------------------------------------- few rows
// V: vectors of 8 elements a thread holds in registers (0: the row is read
// twice in a loop, for rows beyond the registers of a block).  kVec: rows of
// every tensor start on 16-byte boundaries (8 for the codes), a thread's 8
// elements are consecutive; otherwise they are a block's width apart, so that
// 2-byte and 4-byte accesses still coalesce.
template <class T, class G, bool kNorm, int V, bool kVec>
__global__ void __launch_bounds__(kRowsMaxThreads, 1) int8_rows_kernel(const Int8RowsParams p) {
  constexpr bool kPair = kNorm && std::is_same<G, float>::value;
  constexpr int kHeld = V > 0 ? V : 1;
  __shared__ float s_square[2][32];
  __shared__ uint32_t s_peak[2][32];
  __shared__ unsigned long long s_exact[2];
  __shared__ double s_wide_square[32];
  __shared__ unsigned long long s_wide_peak[32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool block_row = p.warps_per_row > 1;
  const int rows_per_block = block_row ? 1 : blockDim.x / 32;
  const int width = block_row ? blockDim.x : 32;  // threads of a row
  const int t = block_row ? threadIdx.x : lane;
  const int cols = p.cols;
  const bool add = kNorm && p.residual != nullptr;
  const G* gain = static_cast<const G*>(p.gain);
  // first element of this thread's vector v, and the step between its elements
  const int step = kVec ? 1 : width;
  auto first = [&](int v) { return kVec ? (v * width + t) * 8 : v * 8 * width + t; };
  const int loops = V > 0 ? V : (cols + 8 * width - 1) / (8 * width);
  if (kPair && threadIdx.x < 2) s_exact[threadIdx.x] = 0;
  let_next_kernel_start();
  wait_for_previous_kernel();

  int parity = 0;
  for (int64_t row = int64_t(blockIdx.x) * rows_per_block + (block_row ? 0 : warp); row < p.rows;
       row += int64_t(gridDim.x) * rows_per_block) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = add ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    T* ro = add ? static_cast<T*>(p.residual_out) + row * p.ldo : nullptr;
    const T* stream = add ? ro : x;  // h in memory, once this thread has read its elements
    int8_t* q = p.codes + row * p.ldq;

    // h of vector v: x, or x + r rounded to the stream's type; past the end 0
    auto read = [&](int v, const T* a, const T* b, float (&h)[8]) {
      const int c0 = first(v);
      if (kVec && c0 + 8 <= cols) {
        RowVec<T>::load(a + c0, h);
        if constexpr (kNorm) {
          if (b != nullptr) {
            float f[8];
            RowVec<T>::load(b + c0, f);
            *reinterpret_cast<uint4*>(ro + c0) = add_vec<T>(h, f);
          }
        }
        return;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = c0 + e * step;
        h[e] = 0.0f;
        if (c < cols) {
          h[e] = RowVec<T>::one(a + c);
          if constexpr (kNorm) {
            if (b != nullptr) {
              const T s = RowVec<T>::rnd(h[e] + RowVec<T>::one(b + c));
              ro[c] = s;
              h[e] = RowVec<T>::wide(s);
            }
          }
        }
      }
    };
    // h -> p in place
    auto times_gain = [&](int v, float (&h)[8]) {
      if constexpr (kNorm) {
        const int c0 = first(v);
        float g[8];
        if (kVec && c0 + 8 <= cols) {
          RowVec<G>::load(gain + c0, g);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = c0 + e * step < cols ? RowVec<G>::one(gain + c0 + e * step) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] *= g[e];
      }
    };
    float square = 0.0f, most = 0.0f;
    uint32_t seen = 0;  // of the bits of h
    auto take = [&](int v, float (&h)[8]) {
      if constexpr (kNorm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          square = fmaf(h[e], h[e], square);
          seen |= __float_as_uint(h[e]);
        }
      }
      times_gain(v, h);
#pragma unroll
      for (int e = 0; e < 8; e += 2) most = max_abs(most, h[e], h[e + 1]);
    };
    // p of one element in FP64, exact, from memory
    auto exact = [&](int c) {
      double P = static_cast<double>(RowVec<T>::one(stream + c));
      if constexpr (kNorm) P *= static_cast<double>(RowVec<G>::one(gain + c));
      return P;
    };

    float held[kHeld][8];
    if constexpr (V > 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) read(v, x, r, held[v]);
#pragma unroll
      for (int v = 0; v < V; ++v) take(v, held[v]);
    } else {
      for (int v = 0; v < loops; ++v) {
        read(v, x, r, held[0]);
        take(v, held[0]);
      }
    }
    const uint32_t mine = __float_as_uint(most);
    RowTotals total = warp_totals<kNorm>({square, mine});
    if (block_row) {
      if (lane == 0) {
        s_square[parity][warp] = total.square;
        s_peak[parity][warp] = total.peak;
      }
      // one barrier a row: the other half of the arrays is written next
      __syncthreads();
      const bool in = lane < p.warps_per_row;
      total.square = in ? s_square[parity][lane] : 0.0f;
      total.peak = in ? s_peak[parity][lane] : 0u;
      total = warp_totals<kNorm>(total);
    }
    const RowScale scale = row_scale<kNorm, kPair>(total, p.eps_sum);
    if (kNorm && !scale.plain) {
      // a row of zeros has codes 0 and scale 0, without an epsilon too; its
      // products may be 0 without it
      bool zeros = total.peak == 0u;
      if (zeros) {
        const bool mine_zero = (seen & 0x7fffffffu) == 0;
        zeros = block_row ? named_barrier_and(0, width, mine_zero) : __all_sync(0xffffffffu, mine_zero);
      }
      if (!zeros) {
        take_row_wide<T, G, kNorm, kVec>(stream, gain, q, p.scales + row, cols, p.eps, t, width, 0, s_wide_square,
                                         s_wide_peak);
      } else {
        if (t == 0) p.scales[row] = 0.0f;
#pragma unroll 1
        for (int v = 0; v < loops; ++v) {
          const int c0 = first(v);
          if (kVec && c0 + 8 <= cols) {
            *reinterpret_cast<uint2*>(q + c0) = make_uint2(0u, 0u);
            continue;
          }
#pragma unroll 1
          for (int c = c0; c < min(c0 + 8 * step, cols); c += step) q[c] = 0;
        }
      }
      if (kPair && block_row && threadIdx.x == 0) s_exact[parity ^ 1] = 0;  // as below
      parity ^= 1;
      continue;
    }
    const bool finite = kNorm || total.peak < 0x7f800000u;
    if (t == 0) p.scales[row] = finite ? stored_scale<kNorm>(total, cols, p.eps) : __uint_as_float(0x7fc00000u);
    double exact_peak = __uint_as_float(total.peak);
    if constexpr (kPair) {
      // p is rounded here: those who hold the largest look it up in FP64
      unsigned long long bits = 0;
      if (mine == total.peak) {
        double value = 0.0;
        if constexpr (V > 0) {
          uint32_t largest = 0;
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              largest |= __float_as_uint(fabsf(held[v][e])) == total.peak ? 1u << (8 * v + e) : 0u;
#pragma unroll 1
          for (; largest != 0; largest &= largest - 1) {
            const int i = __ffs(largest) - 1, c = first(i >> 3) + (i & 7) * step;
            if (c < cols) value = fmax(value, fabs(exact(c)));
          }
        } else {
          for (int v = 0; v < loops; ++v)
            for (int c = first(v); c < min(first(v) + 8 * step, cols); c += step) value = fmax(value, fabs(exact(c)));
        }
        bits = static_cast<unsigned long long>(__double_as_longlong(value));
      }
      if (block_row) {
        if (bits != 0) atomicMax(&s_exact[parity], bits);
        if (threadIdx.x == 0) s_exact[parity ^ 1] = 0;  // nobody reads it before the next row's first barrier
        __syncthreads();
        bits = s_exact[parity];
      } else {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
      }
      exact_peak = __longlong_as_double(static_cast<long long>(bits));
    }
    parity ^= 1;

#pragma unroll
    for (int v = 0; v < loops; ++v) {
      const int c0 = first(v);
      if (V == 0) {
        // second reading: the stream as stored, or x
        read(v, stream, nullptr, held[0]);
        times_gain(v, held[0]);
      }
      if (!kNorm && !scale.plain) {
        // without a norm the peak is exact, and codes are all that is left
        const bool zero = !finite || total.peak == 0u;
        if (kVec && zero && c0 + 8 <= cols) {
          *reinterpret_cast<uint2*>(q + c0) = make_uint2(0u, 0u);
          continue;
        }
        for (int c = c0; c < min(c0 + 8 * step, cols); c += step) q[c] = zero ? 0 : wide_code(exact(c), exact_peak);
        continue;
      }
      float code[8], other[8];
      const uint32_t differ = codes_of(held[V > 0 ? v : 0], scale, code, other);
      if (kVec && c0 + 8 <= cols) {
        *reinterpret_cast<uint2*>(q + c0) = pack_codes(code);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e * step < cols) q[c0 + e * step] = static_cast<int8_t>(__float_as_uint(code[e]));
      }
      if (differ != 0) {
        uint32_t near = border_mask(code, other);
#pragma unroll 1
        for (; near != 0; near &= near - 1) {
          const int c = c0 + (__ffs(near) - 1) * step;
          if (c < cols) q[c] = settled_code(exact(c), exact_peak, scale);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- many rows
// The scale of a streamed row that waits for take_row_wide, a NaN that nothing
// computes.  Such rows are rare, and are taken behind the loop over the rows:
// inside it, the registers cost the others 5 to 10 % (8214 x 4608: 39.7 us, 44.8).
constexpr uint32_t kRowWaits = 0x7fffffffu;
// It finds its place from the parameters: nothing of the loop's stays in registers for it.
template <class T, class G, bool kNorm, bool kVec>
__device__ __noinline__ void take_waiting_rows(const Int8RowsParams& p) {
  __shared__ double squares[32];
  __shared__ unsigned long long peaks[32];
  const int width = p.warps_per_row * 32, group = threadIdx.x / width, t = threadIdx.x - group * width;
  const bool add = kNorm && p.residual != nullptr;
  if (width == 32) __syncwarp();
  else named_barrier_sync(1 + group, width);
  for (int64_t row = int64_t(group) * gridDim.x + blockIdx.x; row < p.rows; row += int64_t(gridDim.x) * p.groups) {
    if (*reinterpret_cast<const volatile uint32_t*>(p.scales + row) != kRowWaits) continue;
    const T* stream = add ? static_cast<const T*>(p.residual_out) + row * p.ldo : static_cast<const T*>(p.x) + row * p.ldx;
    take_row_wide<T, G, kNorm, kVec>(stream, static_cast<const G*>(p.gain), p.codes + row * p.ldq, p.scales + row, p.cols,
                                     p.eps, t, width, 1 + group, squares + group * p.warps_per_row,
                                     peaks + group * p.warps_per_row);
  }
}

// Bulk copy of 16-byte units (both addresses aligned) into this CTA's shared
// memory, completing on the mbarrier at `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

// The 16-byte units of a row: `count` elements from element `head` on.
struct RowBody {
  int head, count;
};
template <class T>
__device__ __forceinline__ RowBody row_body(const T* row, int cols) {
  constexpr int kUnit = 16 / sizeof(T);
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int head = min((kUnit - off) & (kUnit - 1), cols);
  return {head, (cols - head) & ~(kUnit - 1)};
}

constexpr int kRowsMaxGroups = 32;
constexpr int kRowsMaxStages = 4;

// One CTA an SM; `groups` groups of `warps_per_row` warps, each with rows of
// its own and a ring of `stages` rows of shared memory that bulk copies fill,
// so HBM is busy while rows are reduced and converted.  A row is read from its
// stage twice (totals, then codes): nothing is held in registers, few warps
// share a row (a reduction costs each of them some 100 instructions whatever
// the row's length), and groups wait for nobody but their own warps.  With a
// residual the sum goes back into the stage, and to memory; the gain has an FP32
// copy in shared memory.
//
// kVec: rows and leading dimensions are whole 16-byte units.  Otherwise copies
// move the whole units inside a row and the few elements at its ends are put
// into the stage by threads; accesses are one element wide, `width` threads
// apart, and codes are collected in shared memory.
template <class T, class G, bool kNorm, bool kVec>
__global__ void __launch_bounds__(kVec && kNorm ? kRowsNormThreads : kRowsMaxThreads, 1)
    int8_rows_streamed_kernel(const __grid_constant__ Int8RowsParams p) {
  constexpr bool kPair = kNorm && std::is_same<G, float>::value;
  __shared__ __align__(8) uint64_t s_full[kRowsMaxGroups * kRowsMaxStages];
  __shared__ float s_square[kRowsMaxGroups];
  __shared__ uint32_t s_peak[kRowsMaxGroups];
  __shared__ unsigned long long s_exact[kRowsMaxGroups];
  __shared__ int s_abort[kRowsMaxGroups];
  extern __shared__ __align__(128) uint8_t s_ring[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int warps = p.warps_per_row, width = warps * 32;
  const int group = warp / warps, t = threadIdx.x - group * width;
  const int cols = p.cols;
  const bool add = kNorm && p.residual != nullptr;
  float* gain = reinterpret_cast<float*>(s_ring);
  const uint32_t gain_bytes = kNorm ? (static_cast<uint32_t>(cols) * 4u + 15u) / 16u * 16u : 0u;
  const uint32_t slot = (static_cast<uint32_t>(cols) * sizeof(T) + 15u) / 16u * 16u + (kVec ? 0u : 16u);
  const uint32_t stage_bytes = slot * (add ? 2u : 1u);
  const uint32_t code_bytes = kVec ? 0u : (static_cast<uint32_t>(cols) + 15u) / 16u * 16u;
  uint8_t* ring = s_ring + gain_bytes + static_cast<size_t>(group) * (p.stages * stage_bytes + code_bytes);
  int8_t* s_codes = reinterpret_cast<int8_t*>(ring + p.stages * stage_bytes);
  const uint32_t full_bar = smem_u32(s_full + group * kRowsMaxStages);
  // consecutive rows go to consecutive SMs, so that SMs differ by a row at most
  const int64_t row0 = int64_t(group) * gridDim.x + blockIdx.x, row_step = int64_t(gridDim.x) * p.groups;
  // kVec: the first halves of the gain's vectors, then the second halves, so
  // that lanes read 16 bytes apart (32 apart, two of them share a bank)
  auto gain_at = [&](int c) { return kVec ? gain[((c & 4) ? cols / 2 : 0) + c / 8 * 4 + (c & 3)] : gain[c]; };
  auto load_gain = [&](int c, float (&g)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(gain + c / 2);
    const float4 b = *reinterpret_cast<const float4*>(gain + (cols + c) / 2);
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w;
    g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
  };
  auto group_sync = [&] {
    if (warps == 1) __syncwarp();
    else named_barrier_sync(1 + group, width);
  };
  // where element 0 of a row is in its slot: bodies start on 16-byte boundaries
  auto origin = [&](const T* row) { return kVec ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u); };
  // thread 0 of the group: fetch `row` into `stage`
  auto fetch = [&](int64_t row, int stage) {
    const uint32_t bar = full_bar + 8 * stage, dst = smem_u32(ring + stage * stage_bytes);
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = add ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    const RowBody a = kVec ? RowBody{0, cols} : row_body(x, cols);
    const RowBody b = !add ? RowBody{0, 0} : kVec ? RowBody{0, cols} : row_body(r, cols);
    mbar_arrive_expect_tx(bar, static_cast<uint32_t>((a.count + b.count) * sizeof(T)));
    if (a.count > 0) bulk_load(dst + origin(x) + a.head * sizeof(T), x + a.head, a.count * sizeof(T), bar);
    if (b.count > 0) bulk_load(dst + slot + origin(r) + b.head * sizeof(T), r + b.head, b.count * sizeof(T), bar);
  };
  let_next_kernel_start();
  if (t == 0) {
    s_abort[group] = 0;
    for (int s = 0; s < p.stages; ++s) mbar_init(full_bar + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  wait_for_previous_kernel();
  if (t == 0) {
    for (int s = 0; s < p.stages; ++s)
      if (row0 + s * row_step < p.rows) fetch(row0 + s * row_step, s);
  }
  if (threadIdx.x < kRowsMaxGroups) s_exact[threadIdx.x] = 0;
  if constexpr (kNorm) {
    const G* source = static_cast<const G*>(p.gain);
    if constexpr (kVec) {
      for (int c = 8 * threadIdx.x; c < cols; c += 8 * blockDim.x) {
        float g[8];
        RowVec<G>::load(source + c, g);
        *reinterpret_cast<float4*>(gain + c / 2) = make_float4(g[0], g[1], g[2], g[3]);
        *reinterpret_cast<float4*>(gain + (cols + c) / 2) = make_float4(g[4], g[5], g[6], g[7]);
      }
    } else {
      for (int c = threadIdx.x; c < cols; c += blockDim.x) gain[c] = RowVec<G>::one(source + c);
    }
  }
  __syncthreads();

  int stage = 0;
  uint32_t phase = 0;
  bool waits = false;  // some row is left to take_row_wide
  for (int64_t row = row0; row < p.rows; row += row_step) {
    int8_t* q = p.codes + row * p.ldq;
    T* ro = add ? static_cast<T*>(p.residual_out) + row * p.ldo : nullptr;
    // a wait that runs out is noticed by the whole group behind its barrier
    mbar_wait_bounded(full_bar + 8 * stage, phase, &s_abort[group], p.timeout_ns, 31);
    uint8_t* bytes = ring + stage * stage_bytes;
    T* h = reinterpret_cast<T*>(bytes);
    const T* f = reinterpret_cast<const T*>(bytes + slot);
    if constexpr (!kVec) {
      const T* x = static_cast<const T*>(p.x) + row * p.ldx;
      const RowBody a = row_body(x, cols);
      h = reinterpret_cast<T*>(bytes + origin(x));
      // what the copies leave out: fewer than 16 elements at each end
      for (int c = t; c < cols - a.count; c += width) {
        const int at = c < a.head ? c : c + a.count;
        h[at] = x[at];
      }
      if (add) {
        const T* r = static_cast<const T*>(p.residual) + row * p.ldr;
        const RowBody b = row_body(r, cols);
        T* left = reinterpret_cast<T*>(bytes + slot + origin(r));
        for (int c = t; c < cols - b.count; c += width) {
          const int at = c < b.head ? c : c + b.count;
          left[at] = r[at];
        }
        f = left;
      }
      group_sync();
    }

    // ---- totals
    float square = 0.0f, square_b = 0.0f, most = 0.0f;
    // FP32 gain: where this thread's largest product was, and whether a later
    // vector had one as large
    int at = 0;
    bool again = false;
    auto take = [&](float largest, int c) {
      if constexpr (kPair) {
        again = largest > most ? false : again || largest == most;
        at = largest > most ? c : at;
      }
      most = max_abs(most, largest, largest);
    };
    if constexpr (kVec) {
#pragma unroll 4
      for (int c = 8 * t; c < cols; c += 8 * width) {
        float v[8];
        RowVec<T>::load(h + c, v);
        if constexpr (kNorm) {
          if (add) {
            float w[8];
            RowVec<T>::load(f + c, w);
            const uint4 sum = add_vec<T>(v, w);
            *reinterpret_cast<uint4*>(h + c) = sum;
            *reinterpret_cast<uint4*>(ro + c) = sum;
          }
          float g[8];
          load_gain(c, g);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            square = fmaf(v[e], v[e], square);
            square_b = fmaf(v[e + 1], v[e + 1], square_b);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= g[e];
        }
        if constexpr (kPair) {
          float largest = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e += 2) largest = max_abs(largest, v[e], v[e + 1]);
          take(largest, c);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 2) most = max_abs(most, v[e], v[e + 1]);
        }
      }
    } else {
#pragma unroll 4
      for (int c = t; c < cols; c += width) {
        float v = RowVec<T>::one(h + c);
        if constexpr (kNorm) {
          if (add) {
            const T s = RowVec<T>::rnd(v + RowVec<T>::one(f + c));
            h[c] = s;
            ro[c] = s;
            v = RowVec<T>::wide(s);
          }
          square = fmaf(v, v, square);
          v *= gain[c];
        }
        take(fabsf(v), c);
      }
    }
    const uint32_t mine = __float_as_uint(most);
    RowTotals total = warp_totals<kNorm>({square + square_b, mine});
    if (warps > 1) {
      if (lane == 0) {
        s_square[warp] = total.square;
        s_peak[warp] = total.peak;
      }
      group_sync();
      total.square = 0.0f;
      total.peak = 0u;
      for (int w = group * warps; w < (group + 1) * warps; ++w) {
        total.square += s_square[w];
        total.peak = max(total.peak, s_peak[w]);
      }
    }
    if (warps == 1 ? __any_sync(0xffffffffu, *static_cast<volatile int*>(&s_abort[group]) != 0)
                   : *static_cast<volatile int*>(&s_abort[group]) != 0)
      break;
    const RowScale scale = row_scale<kNorm, kPair>(total, p.eps_sum);
    if (scale.plain && t == 0) p.scales[row] = stored_scale<kNorm>(total, cols, p.eps);
    // p of one element in FP64, exact
    auto exact = [&](int c) {
      double P = static_cast<double>(RowVec<T>::one(h + c));
      if constexpr (kNorm) P *= static_cast<double>(gain_at(c));
      return P;
    };
    double exact_peak = __uint_as_float(total.peak);
    if (kPair && scale.plain) {
      // p is rounded here: those who hold the largest look it up in FP64
      unsigned long long bits = 0;
      if (mine == total.peak) {
        double value = 0.0;
        auto look = [&](int c0) {
#pragma unroll
          for (int e = 0; e < (kVec ? 8 : 1); ++e) {
            const float a = RowVec<T>::one(h + c0 + e), g = gain_at(c0 + e);
            if (__float_as_uint(fabsf(a * g)) == total.peak)
              value = fmax(value, fabs(static_cast<double>(a) * static_cast<double>(g)));
          }
        };
        if (!again) {
          look(at);
        } else {
          const int step = kVec ? 8 : 1;
          for (int c = step * t; c < cols; c += step * width) look(c);
        }
        bits = static_cast<unsigned long long>(__double_as_longlong(value));
      }
      if (warps > 1) {
        if (bits != 0) atomicMax(&s_exact[group], bits);
        group_sync();
        bits = s_exact[group];
      } else {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
      }
      exact_peak = __longlong_as_double(static_cast<long long>(bits));
    }

    // ---- codes
    if (!scale.plain) {
      // a row of zeros has codes 0 and scale 0, without an epsilon too; a norm's
      // products may be 0 without it.  Elements as above: with a residual the
      // stage holds sums that only the thread which wrote them is sure to see (a
      // group of one warp has no barrier in between)
      bool zeros = total.peak == 0u;
      if (kNorm && zeros) {
        uint32_t seen = 0;
        if constexpr (kVec) {
#pragma unroll 1
          for (int c = 8 * t; c < cols; c += 8 * width) {
            const uint4 v = *reinterpret_cast<const uint4*>(h + c);
            seen |= (v.x | v.y | v.z | v.w) & 0x7fff7fffu;  // 16-bit elements
          }
        } else {
#pragma unroll 1
          for (int c = t; c < cols; c += width) seen |= RowVec<T>::one(h + c) != 0.0f ? 1u : 0u;
        }
        zeros = warps == 1 ? __all_sync(0xffffffffu, seen == 0) : named_barrier_and(1 + group, width, seen == 0);
      }
      if (t == 0) p.scales[row] = zeros ? 0.0f : __uint_as_float(kRowWaits);
      waits = waits || !zeros;
      if constexpr (kVec) {
#pragma unroll 1
        for (int c = 8 * t; c < cols; c += 8 * width) *reinterpret_cast<uint2*>(q + c) = make_uint2(0u, 0u);
      } else {
#pragma unroll 1
        for (int c = t; c < cols; c += width) s_codes[c] = 0;
      }
    } else if constexpr (kVec) {
#pragma unroll 4
      for (int c = 8 * t; c < cols; c += 8 * width) {
        float v[8];
        RowVec<T>::load(h + c, v);
        if constexpr (kNorm) {
          float g[8];
          load_gain(c, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= g[e];
        }
        float code[8], other[8];
        const uint32_t differ = codes_of(v, scale, code, other);
        *reinterpret_cast<uint2*>(q + c) = pack_codes(code);
        if (differ != 0) {
          uint32_t near = border_mask(code, other);
#pragma unroll 1
          for (; near != 0; near &= near - 1) {
            const int at = c + __ffs(near) - 1;
            q[at] = settled_code(exact(at), exact_peak, scale);
          }
        }
      }
    } else {
#pragma unroll 4
      for (int c = t; c < cols; c += width) {
        float v = RowVec<T>::one(h + c);
        if constexpr (kNorm) v *= gain[c];
        const float code = fmaf(v, scale.low, kMagic);
        int8_t byte = static_cast<int8_t>(__float_as_uint(code));
        if (code != fmaf(v, scale.high, kMagic)) byte = settled_code(exact(c), exact_peak, scale);
        s_codes[c] = byte;
      }
    }
    // this thread's writes to the stage come before the copy that refills it
    if (add || !kVec) fence_proxy_async_smem();
    group_sync();
    if (t == 0) {
      if (kPair) s_exact[group] = 0;  // read by all; the next row's first barrier comes before its use
      if (row + p.stages * row_step < p.rows) fetch(row + p.stages * row_step, stage);
    }
    if constexpr (!kVec) {
      // collected codes, 16 at a time where the row allows it; the next row
      // writes them behind a barrier that follows
      const bool whole = (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
      const int units = whole ? cols / 16 : 0;
      for (int u = t; u < units; u += width)
        *reinterpret_cast<uint4*>(q + 16 * u) = *reinterpret_cast<const uint4*>(s_codes + 16 * u);
      for (int c = 16 * units + t; c < cols; c += width) q[c] = s_codes[c];
    }
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (s_abort[group] != 0 && t == 0) {
    // copies into this group's ring may still be landing: give each its limit
    volatile int no_abort = 0;
    for (int s = 0; s < p.stages; ++s)
      if (row0 + s * row_step < p.rows)
        mbar_wait_bounded(full_bar + 8 * s, s < stage ? phase ^ 1u : phase, &no_abort, p.timeout_ns, 32);
  }
  if (waits) take_waiting_rows<T, G, kNorm, kVec>(p);
}

}  // namespace fmm
