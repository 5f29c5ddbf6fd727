// Rows to 8-bit codes: symmetric integers with one FP32 scale a row.
//
//   quantize_rows   p = x                              s = a / 127
//   rms_norm_int8   h = rnd(x + r), p = h * g          s = a * rstd / 127
//                   rstd = 1 / sqrt(mean(h^2) + eps)
//   a = max |p| over the row,  q = round_half_even(127 p / a)
//
// rstd cancels in q, so one reduction (sum of squares and maximum together)
// separates the read of a row from its write: the row stays in registers and
// every element crosses HBM once.
//
// Codes are those of exact arithmetic.  p is exact in FP32 where x and g have
// 16 bits (at most 22 significant bits); with an FP32 gain it is the pair
// hi + lo, lo = fma(h, g, -hi), and the maximum compares pairs.  p * (127 / a)
// carries at most four roundings, 4 * 2^-24 * 127 < 2^-15, so only a quotient
// within 2^-14 of a half can round the wrong way; those (1 in 8000) compare
// 254 |p| with (2c + 1) a in FP64, where both products are exact.
//
// A row with an infinity or a NaN (or, in the norm, with a square beyond FP32)
// has codes 0 and a NaN scale: whatever is computed from it is NaN.  A row of
// zeros has codes 0 and scale 0.
#pragma once

#include <type_traits>

#include "fmm_common.cuh"

namespace fmm {

constexpr int kRowsMaxThreads = 512;

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
  int32_t warps_per_row;  // > 1: the block is one row's; 1: every warp has a row of its own
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

// round_half_even(127 |P| / M) with the sign of P, for 0 <= |P| <= M, M > 0,
// P and M of at most 44 significant bits: 254 |P| and (2c +- 1) M are exact.
__device__ __forceinline__ int exact_code(double P, double M) {
  const double a = 254.0 * fabs(P);
  int c = static_cast<int>(floor((a / M + 1.0) * 0.5));
  const double low = (2 * c - 1) * M, high = (2 * c + 1) * M;
  if (a < low || (a == low && (c & 1))) --c;
  else if (a > high || (a == high && (c & 1))) ++c;
  return P < 0.0 ? -c : c;
}

// What the row reduction gives: the sum of squares (norm only) and the
// largest |p| as (bits of hi, lo).  Bits compare as the values do, infinities
// and NaN above all finite ones.
struct RowTotals {
  float square;
  uint32_t hi;
  float lo;
};

// Order-preserving map of a finite FP32 to unsigned, and back.
__device__ __forceinline__ uint32_t float_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <bool kNorm, bool kPair>
__device__ __forceinline__ RowTotals warp_totals(RowTotals t) {
  RowTotals r = t;
  if constexpr (kNorm) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) r.square += __shfl_xor_sync(0xffffffffu, r.square, d);
  }
  r.hi = __reduce_max_sync(0xffffffffu, t.hi);
  if constexpr (kPair)
    r.lo = key_float(__reduce_max_sync(0xffffffffu, t.hi == r.hi ? float_key(t.lo) : 0u));
  return r;
}

// V: vectors of 8 elements a thread holds in registers (0: the row is read
// twice in a loop, for rows beyond the registers of a block).  kVec: rows of
// every tensor start on 16-byte boundaries (8 for the codes), a thread's 8
// elements are consecutive; otherwise they are a block's width apart, so that
// 2-byte and 4-byte accesses still coalesce.
template <class T, class G, bool kNorm, int V, bool kVec>
__global__ void __launch_bounds__(kRowsMaxThreads) int8_rows_kernel(const Int8RowsParams p) {
  constexpr bool kPair = kNorm && std::is_same<G, float>::value;
  constexpr int kHeld = V > 0 ? V : 1;
  __shared__ float s_square[2][32];
  __shared__ uint32_t s_hi[2][32];
  __shared__ float s_lo[2][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool block_row = p.warps_per_row > 1;
  const int rows_per_block = block_row ? 1 : blockDim.x / 32;
  const int width = block_row ? blockDim.x : 32;           // threads of a row
  const int t = block_row ? threadIdx.x : lane;
  const int cols = p.cols;
  const G* gain = static_cast<const G*>(p.gain);
  // first element of this thread's vector v, and the step between its elements
  const int step = kVec ? 1 : width;
  auto first = [&](int v) { return kVec ? (v * width + t) * 8 : v * 8 * width + t; };
  const int loops = V > 0 ? V : (cols + 8 * width - 1) / (8 * width);

  int parity = 0;
  for (int64_t row = int64_t(blockIdx.x) * rows_per_block + (block_row ? 0 : warp); row < p.rows;
       row += int64_t(gridDim.x) * rows_per_block) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = (kNorm && p.residual != nullptr) ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    T* ro = r != nullptr ? static_cast<T*>(p.residual_out) + row * p.ldo : nullptr;
    int8_t* q = p.codes + row * p.ldq;

    // h of vector v: x, or x + r rounded to the stream's type; past the end 0
    auto read = [&](int v, const T* a, const T* b, T* out, float (&h)[8]) {
      const int c0 = first(v);
      if (kVec && c0 + 8 <= cols) {
        RowVec<T>::load(a + c0, h);
        if constexpr (kNorm) {
          if (b != nullptr) {
            float f[8];
            RowVec<T>::load(b + c0, f);
            uint4 w;
            w.x = RowVec<T>::pack(h[0] + f[0], h[1] + f[1]);
            w.y = RowVec<T>::pack(h[2] + f[2], h[3] + f[3]);
            w.z = RowVec<T>::pack(h[4] + f[4], h[5] + f[5]);
            w.w = RowVec<T>::pack(h[6] + f[6], h[7] + f[7]);
            *reinterpret_cast<uint4*>(out + c0) = w;
            RowVec<T>::load(reinterpret_cast<const T*>(&w), h);
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
              out[c] = s;
              h[e] = RowVec<T>::wide(s);
            }
          }
        }
      }
    };
    auto read_gain = [&](int v, float (&g)[8]) {
      const int c0 = first(v);
      if (kVec && c0 + 8 <= cols) {
        RowVec<G>::load(gain + c0, g);
        return;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = c0 + e * step < cols ? RowVec<G>::one(gain + c0 + e * step) : 0.0f;
    };
    // h -> p in place, taking part in the totals
    auto take = [&](int v, float (&h)[8], RowTotals& total) {
      float g[8];
      if constexpr (kNorm) read_gain(v, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float was = h[e];
        if constexpr (kNorm) {
          total.square = fmaf(was, was, total.square);
          h[e] = was * g[e];
        }
        const uint32_t hi = __float_as_uint(fabsf(h[e]));
        if constexpr (kPair) {
          const float rest = fmaf(was, g[e], -h[e]);
          const float lo = h[e] < 0.0f ? -rest : rest;
          if (hi > total.hi || (hi == total.hi && lo > total.lo)) total.lo = lo;
        }
        total.hi = max(total.hi, hi);
      }
    };

    float held[kHeld][8];
    RowTotals total = {0.0f, 0u, 0.0f};
    if constexpr (V > 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) read(v, x, r, ro, held[v]);
#pragma unroll
      for (int v = 0; v < V; ++v) take(v, held[v], total);
    } else {
      for (int v = 0; v < loops; ++v) {
        read(v, x, r, ro, held[0]);
        take(v, held[0], total);
      }
    }
    total = warp_totals<kNorm, kPair>(total);
    if (block_row) {
      if (lane == 0) {
        s_square[parity][warp] = total.square;
        s_hi[parity][warp] = total.hi;
        s_lo[parity][warp] = total.lo;
      }
      // one barrier a row: the other half of the arrays is written next
      __syncthreads();
      const bool in = lane < p.warps_per_row;
      total.square = in ? s_square[parity][lane] : 0.0f;
      total.hi = in ? s_hi[parity][lane] : 0u;
      total.lo = in ? s_lo[parity][lane] : 0.0f;
      total = warp_totals<kNorm, kPair>(total);
      parity ^= 1;
    }

    const float peak = __uint_as_float(total.hi);
    bool finite = total.hi < 0x7f800000u;
    float scale = peak;
    if constexpr (kNorm) {
      const float mean = total.square / static_cast<float>(cols);
      finite = finite && __float_as_uint(mean) < 0x7f800000u;
      scale = peak / sqrtf(mean + p.eps);
    }
    scale = finite ? scale / 127.0f : __uint_as_float(0x7fc00000u);
    if (t == 0) p.scales[row] = scale;
    const bool zero = !finite || total.hi == 0u;
    // 127 / peak leaves FP32 below 2^-121; such rows take the exact codes
    const bool tiny = peak < 0x1p-100f;
    const float inverse = zero || tiny ? 0.0f : 127.0f / peak;
    const double exact_peak = static_cast<double>(peak) + (kPair ? static_cast<double>(total.lo) : 0.0);

#pragma unroll
    for (int v = 0; v < loops; ++v) {
      const int c0 = first(v);
      if (V == 0) {
        // second reading: the stream as stored, or x
        RowTotals unused = {0.0f, 0u, 0.0f};
        read(v, ro != nullptr ? ro : x, nullptr, nullptr, held[0]);
        take(v, held[0], unused);
      }
      float(&pv)[8] = held[V > 0 ? v : 0];
      int code[8];
      bool border = tiny && !zero;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = zero ? 0.0f : pv[e] * inverse;
        code[e] = __float2int_rn(d);
        border = border || fabsf(d - static_cast<float>(code[e])) > 0.5f - 0x1p-14f;
      }
      if (kVec && c0 + 8 <= cols) {
        uint2 w;
        w.x = (code[0] & 255) | (code[1] & 255) << 8 | (code[2] & 255) << 16 | code[3] << 24;
        w.y = (code[4] & 255) | (code[5] & 255) << 8 | (code[6] & 255) << 16 | code[7] << 24;
        *reinterpret_cast<uint2*>(q + c0) = w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e * step < cols) q[c0 + e * step] = static_cast<int8_t>(code[e]);
      }
      if (border) {
        // once more from memory (this thread's own elements), in FP64
        const T* h = ro != nullptr ? ro : x;
#pragma unroll 1
        for (int c = c0; c < min(c0 + 8 * step, cols); c += step) {
          double P = static_cast<double>(RowVec<T>::one(h + c));
          if constexpr (kNorm) P *= static_cast<double>(RowVec<G>::one(gain + c));
          q[c] = static_cast<int8_t>(exact_code(P, exact_peak));
        }
      }
    }
  }
}

}  // namespace fmm
