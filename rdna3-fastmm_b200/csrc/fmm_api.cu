// C ABI of libfmm_sm100.so: argument checking, launch geometry, TMA tensor
// maps, and the per-scheme dispatch of the generated transforms.
//
// Nothing here allocates device memory or synchronises the stream (except
// fmm_device_status, whose job is to synchronise and read the status word).

#include <cuda.h>
#include <cudaTypedefs.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>
#include <vector>

#include "fmm_common.cuh"
#include "transforms.cuh"
#include "generated/fmm_schemes.cuh"
#include "leaf_gemm.cuh"
#include "reconstruct_tc.cuh"
#include "reconstruct_staged.cuh"
#include "int8_rows.cuh"
#include "int8_gemm.cuh"

// Scratch of fmm_linear_noalloc: the L, Rt and P planes of one call live in
// this array instead of caller-provided buffers.  It is part of the module, so
// every GPU that loads this library holds it until the process exits.
static __device__ __align__(256) unsigned char g_noalloc_scratch[FMM_NOALLOC_SCRATCH_BYTES];

namespace fmm {

namespace {

thread_local std::string t_last_error;
uint64_t g_timeout_ns = 2000000000ull;  // 2 s per wait
int g_sm_budget = 0;                     // 0: every SM; else the most SMs one launch may fill

int fail(int code, const std::string& what) {
  t_last_error = what;
  return code;
}

int cuda_fail(cudaError_t e, const char* where) {
  return fail(FMM_ERR_CUDA, std::string(where) + ": " + cudaGetErrorString(e));
}

bool aligned(const void* p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

int scheme_size(int scheme) {
  switch (scheme) {
    case FMM_SCHEME_RANK7: return 2;
    case FMM_SCHEME_RANK48: return 4;
    case FMM_SCHEME_RANK49: return 4;
    case FMM_SCHEME_RANK343: return 8;
    default: return 0;
  }
}

int dims_for(int scheme, int64_t M, int64_t K, int64_t N, fmm_dims* d) {
  const int s = scheme_size(scheme);
  if (s == 0) return fail(FMM_ERR_UNSUPPORTED, "unknown scheme id " + std::to_string(scheme));
  if (M < 1 || K < 1 || N < 1) return fail(FMM_ERR_INVALID_ARGUMENT, "matrix dimensions must be positive");
  d->scheme_size = s;
  d->rank = scheme;
  d->bm = ceil_div(M, s);
  d->bk = ceil_div(K, s);
  d->bn = ceil_div(N, s);
  d->ldk = round_up(d->bk, 8);
  d->ldp = round_up(d->bn, 8);
  d->left_elements = d->rank * d->bm * d->ldk;
  d->right_elements = d->rank * d->bn * d->ldk;
  d->product_elements = d->rank * d->bm * d->ldp;
  // 32-bit per-plane vector indices in the streaming kernels; TMA coordinates
  if (d->bm * d->ldk > (int64_t(1) << 31) || d->bn * d->ldk > (int64_t(1) << 31) ||
      d->bm * d->ldp > (int64_t(1) << 31) || d->bm > (int64_t(1) << 30) ||
      d->bn > (int64_t(1) << 30))
    return fail(FMM_ERR_TOO_LARGE, "transform planes exceed 2^31 elements");
  return FMM_OK;
}

struct DeviceInfo {
  int sm_count = 0;
  bool gemm_configured = false;
  bool pair256_configured = false;
  bool pair128_configured = false;
  bool pair192_configured = false;
  bool pair256k128_configured = false;
  void* noalloc_scratch = nullptr;  // device address of g_noalloc_scratch
  void* rank343_wt = nullptr;       // device address of g_rank343_wt, once uploaded
  bool reconstruct_tc_configured = false;
};

constexpr int kMaxDevices = 64;
DeviceInfo g_devices[kMaxDevices];
std::mutex g_device_mutex;

int device_info(DeviceInfo** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(FMM_ERR_UNSUPPORTED, "device index out of range");
  std::lock_guard<std::mutex> lock(g_device_mutex);
  DeviceInfo& info = g_devices[dev];
  if (info.sm_count == 0) {
    int major = 0, minor = 0, sms = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    if (major != 10 || minor != 0)
      return fail(FMM_ERR_UNSUPPORTED, "libfmm_sm100 needs an sm_100 (B200) device; found sm_" +
                                           std::to_string(major) + std::to_string(minor));
    info.sm_count = sms;
  }
  *out = &info;
  return FMM_OK;
}

// SMs a launch may fill: all of them, or the budget set by fmm_set_sm_budget
// (kept even so that SM pairs of the 2-SM GEMM stay whole).
int usable_sms(const DeviceInfo* info) {
  int sms = info->sm_count;
  if (g_sm_budget > 0 && g_sm_budget < sms) sms = g_sm_budget & ~1;
  return sms < 2 ? 2 : sms;
}

// ------------------------------------------------------------------ dispatch
// Launch shapes were swept on B200 with random data (threads per block,
// minimum resident blocks, grid cap in blocks per SM); with every input
// preloaded these reach 91-98 % of the measured copy bandwidth.  The K x N
// right transform (plain-mm API) was swept separately: small 32 (k) x 8 (n)
// tiles with two k per thread and many resident blocks won for every scheme
// (16384^2: rank 7 4.8, rank 48/49 4.2, rank 343 2.4 TB/s).  The rank-48/49
// reconstruct runs TMA-staged (kOutStages > 0): timed right after the leaf
// GEMM that writes its products, 2 stages of 256 positions and 4 CTAs per SM
// beat the register kernel by 12-25 % (3 stages x 2 CTAs, fewer compute warps
// per SM, lost to it; 128-position tiles and single stages were slower).
template <int SCHEME>
struct SchemeTraits;
template <>
struct SchemeTraits<FMM_SCHEME_RANK7> {
  using Left = gen::Rank7Left;
  using Right = gen::Rank7Right;
  using Output = gen::Rank7Output;
  static constexpr int S = 2;
  static constexpr int VEC = 8;
  static constexpr int kInThreads = 256, kInBlocks = 1, kInGrid = 64;
  static constexpr int kOutVec = 8, kOutThreads = 128, kOutBlocks = 4, kOutGrid = 64;
  static constexpr int kOutStages = 0;
  static constexpr bool kTensorCoreOutput = false;
  static constexpr int kKnTK = 32, kKnTN = 8, kKnVec = 2, kKnThreads = 128, kKnBlocks = 4;
};
template <>
struct SchemeTraits<FMM_SCHEME_RANK48> {
  using Left = gen::Rank48Left;
  using Right = gen::Rank48Right;
  using Output = gen::Rank48Output;
  static constexpr int S = 4;
  static constexpr int VEC = 4;
  static constexpr int kInThreads = 128, kInBlocks = 4, kInGrid = 64;
  static constexpr int kOutVec = 4, kOutThreads = 128, kOutBlocks = 3, kOutGrid = 16;
  static constexpr int kOutStages = 2, kOutStagedBlocks = 4;
  static constexpr bool kTensorCoreOutput = false;
  static constexpr int kKnTK = 32, kKnTN = 8, kKnVec = 2, kKnThreads = 128, kKnBlocks = 4;
};
template <>
struct SchemeTraits<FMM_SCHEME_RANK49> {
  using Left = gen::Rank49Left;
  using Right = gen::Rank49Right;
  using Output = gen::Rank49Output;
  static constexpr int S = 4;
  static constexpr int VEC = 4;
  static constexpr int kInThreads = 128, kInBlocks = 4, kInGrid = 64;
  static constexpr int kOutVec = 4, kOutThreads = 128, kOutBlocks = 3, kOutGrid = 64;
  static constexpr int kOutStages = 2, kOutStagedBlocks = 4;
  static constexpr bool kTensorCoreOutput = false;
  static constexpr int kKnTK = 32, kKnTN = 8, kKnVec = 2, kKnThreads = 128, kKnBlocks = 4;
};
// Rank 343: 64 inputs and 343 planes per position.  The input side keeps two
// elements per thread (64 packed inputs plus the circuit fit in registers);
// the output side is a tensor-core product with the coefficient matrix
// (reconstruct_tc.cuh).
template <>
struct SchemeTraits<FMM_SCHEME_RANK343> {
  using Left = gen::Rank343Left;
  using Right = gen::Rank343Right;
  using Output = gen::Rank343OutputCoefficients;
  static constexpr int S = 8;
  static constexpr int VEC = 2;
  static constexpr int kInThreads = 128, kInBlocks = 1, kInGrid = 16;
  static constexpr bool kTensorCoreOutput = true;
  static constexpr int kKnTK = 32, kKnTN = 8, kKnVec = 2, kKnThreads = 128, kKnBlocks = 1;
};

int streaming_grid(const DeviceInfo* info, int64_t work_items, int threads, int blocks_per_sm) {
  const int64_t blocks = ceil_div(work_items, threads);
  const int64_t cap = int64_t(usable_sms(info)) * blocks_per_sm;
  return static_cast<int>(blocks < cap ? (blocks > 0 ? blocks : 1) : cap);
}

template <int SCHEME>
TransformArgs transform_args(const void* src, int64_t rows, int64_t cols, int64_t ld, void* dst,
                             int64_t brows, int64_t bcols, int64_t ldd) {
  using T = SchemeTraits<SCHEME>;
  const bool vec = (bcols % T::VEC == 0) && (ld % T::VEC == 0) && aligned(src, 2 * T::VEC);
  TransformArgs a;
  a.src = static_cast<const uint16_t*>(src);
  a.rows = rows;
  a.cols = cols;
  a.ld = ld;
  a.dst = static_cast<uint16_t*>(dst);
  a.brows = brows;
  a.bcols = bcols;
  a.ldd = ldd;
  a.vector_loads = vec ? 1 : 0;
  return a;
}

// Precision of one launch (the dtype argument of the C ABI): operand and
// output elements FP16 or BF16, plane elements BF16 only for
// FMM_DTYPE_BF16_BF16 (FP16 otherwise).
template <int PREC>
struct Precision {
  static constexpr bool kHalf = PREC == FMM_DTYPE_F16;
  static constexpr bool kBfPlanes = PREC == FMM_DTYPE_BF16_BF16;
};

template <int SCHEME, bool kWeight, int PREC>
int launch_input_transform(const void* src, int64_t rows, int64_t cols, int64_t ld, void* dst,
                           int64_t brows, int64_t bcols, int64_t ldd, cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  constexpr bool kHalf = Precision<PREC>::kHalf, kBf = Precision<PREC>::kBfPlanes;
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  const TransformArgs a = transform_args<SCHEME>(src, rows, cols, ld, dst, brows, bcols, ldd);
  const int64_t items = brows * (ldd / T::VEC);
  using Prog = typename std::conditional<kWeight, typename T::Right, typename T::Left>::type;
  block_transform_kernel<Prog, T::S, T::VEC, kWeight, T::kInThreads, T::kInBlocks, kHalf, kBf>
      <<<streaming_grid(info, items, T::kInThreads, T::kInGrid), T::kInThreads, 0, stream>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, kWeight ? "weight transform launch" : "left transform launch");
  return FMM_OK;
}

// Left and weight transform of a dynamic linear in one launch; each gets a
// share of the CTAs proportional to its vectors (at least one).
template <int SCHEME, int PREC>
int launch_paired_transform(const void* A, int64_t M, int64_t K, int64_t lda, void* L, const void* W,
                            int64_t N, int64_t ldw, void* Rt, const fmm_dims& d, cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  constexpr bool kHalf = Precision<PREC>::kHalf, kBf = Precision<PREC>::kBfPlanes;
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  const TransformArgs left = transform_args<SCHEME>(A, M, K, lda, L, d.bm, d.bk, d.ldk);
  const TransformArgs weight = transform_args<SCHEME>(W, N, K, ldw, Rt, d.bn, d.bk, d.ldk);
  const int64_t left_items = d.bm * (d.ldk / T::VEC);
  const int64_t weight_items = d.bn * (d.ldk / T::VEC);
  int total = streaming_grid(info, left_items + weight_items, T::kInThreads, T::kInGrid);
  if (total < 2) total = 2;
  int64_t left_blocks = (int64_t(total) * left_items) / (left_items + weight_items);
  if (left_blocks < 1) left_blocks = 1;
  if (left_blocks > total - 1) left_blocks = total - 1;
  paired_transform_kernel<typename T::Left, typename T::Right, T::S, T::VEC, T::kInThreads,
                          T::kInBlocks, kHalf, kBf>
      <<<total, T::kInThreads, 0, stream>>>(left, weight, static_cast<uint32_t>(left_blocks));
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paired transform launch");
  return FMM_OK;
}

template <class Coefs, bool kHalf>
int launch_reconstruct_tc(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                          void* C, int64_t ldc, DeviceInfo* info, cudaStream_t stream);

template <int SCHEME, int PREC>
int launch_reconstruct_staged(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                              void* C, int64_t ldc, DeviceInfo* info, cudaStream_t stream);

template <int SCHEME, int PREC>
int launch_reconstruct_staged_gather(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                                     const GatherDests& dests, int64_t ldc, DeviceInfo* info,
                                     cudaStream_t stream);

// FMM_RECONSTRUCT_VARIANT=register keeps the circuit schemes on the register
// reconstruct (the TMA-staged one is the default where a scheme has stages).
bool staged_reconstruct_enabled() {
  const char* v = std::getenv("FMM_RECONSTRUCT_VARIANT");
  return v == nullptr || std::string(v) != "register";
}

template <int SCHEME, int PREC>
int launch_reconstruct(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                       void* C, int64_t ldc, cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  constexpr bool kHalf = Precision<PREC>::kHalf, kBf = Precision<PREC>::kBfPlanes;
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  if constexpr (T::kTensorCoreOutput) {
    return launch_reconstruct_tc<typename T::Output, kHalf>(P, d, M, N, bias, C, ldc, info, stream);
  } else {
    if constexpr (T::kOutStages > 0) {
      if (staged_reconstruct_enabled() && aligned(P, 16) && d.ldp % 8 == 0)
        return launch_reconstruct_staged<SCHEME, PREC>(P, d, M, N, bias, C, ldc, info, stream);
    }
    constexpr int V = T::kOutVec;
    const bool vec = (d.bn % V == 0) && (ldc % V == 0) && aligned(C, 2 * V);
    const bool vec_bias = (d.bn % V == 0) && bias != nullptr && aligned(bias, 2 * V);
    const int64_t items = d.bm * ceil_div(d.bn, V);
    const int grid = streaming_grid(info, items, T::kOutThreads, T::kOutGrid);
    reconstruct_kernel<typename T::Output, T::S, V, T::kOutThreads, T::kOutBlocks, kHalf, kBf>
        <<<grid, T::kOutThreads, 0, stream>>>(
            static_cast<const uint16_t*>(P), d.bm, d.bn, d.ldp, static_cast<const uint16_t*>(bias),
            static_cast<uint16_t*>(C), M, N, ldc, (vec ? 1 : 0) | (vec_bias ? 2 : 0));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "reconstruct launch");
    return FMM_OK;
  }
}

template <int SCHEME, int PREC>
int launch_reconstruct_gather(const void* P, const fmm_dims& d, int64_t M, int64_t N,
                              const void* bias, const GatherDests& dests, int64_t ldc,
                              cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  constexpr bool kHalf = Precision<PREC>::kHalf, kBf = Precision<PREC>::kBfPlanes;
  if constexpr (T::kTensorCoreOutput) {
    return fail(FMM_ERR_UNSUPPORTED, "the gathering reconstruct covers the circuit schemes (7, 48, 49)");
  } else {
    constexpr int V = T::kOutVec;
    DeviceInfo* info = nullptr;
    if (int rc = device_info(&info)) return rc;
    if constexpr (T::kOutStages > 0) {
      // staged tiles with bulk-copy stores: every output row segment starts on
      // a 16-byte boundary and moves a multiple of 16 bytes
      bool bulk = staged_reconstruct_enabled() && aligned(P, 16) && d.ldp % 8 == 0 && d.bn % 8 == 0 &&
                  N % 8 == 0 && ldc % 8 == 0;
      for (int k = 0; k < dests.n; ++k) bulk = bulk && aligned(dests.p[k], 16);
      if (bulk)
        return launch_reconstruct_staged_gather<SCHEME, PREC>(P, d, M, N, bias, dests, ldc, info, stream);
    }
    bool vec = (d.bn % V == 0) && (ldc % V == 0);
    for (int k = 0; k < dests.n; ++k) vec = vec && aligned(dests.p[k], 2 * V);
    const bool vec_bias = (d.bn % V == 0) && bias != nullptr && aligned(bias, 2 * V);
    const int64_t items = d.bm * ceil_div(d.bn, V);
    const int grid = streaming_grid(info, items, T::kOutThreads, T::kOutGrid);
    reconstruct_gather_kernel<typename T::Output, T::S, V, T::kOutThreads, T::kOutBlocks, kHalf, kBf>
        <<<grid, T::kOutThreads, 0, stream>>>(static_cast<const uint16_t*>(P), d.bm, d.bn, d.ldp,
                                              static_cast<const uint16_t*>(bias), dests, M, N, ldc,
                                              (vec ? 1 : 0) | (vec_bias ? 2 : 0));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "gathering reconstruct launch");
    return FMM_OK;
  }
}

template <class Kernel>
int ensure_smem_attribute(bool& done, Kernel kernel, size_t bytes);

template <int SCHEME, int PREC>
int launch_right_kn(const void* B, int64_t K, int64_t N, int64_t ldb, void* dst, const fmm_dims& d,
                    cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  constexpr bool kHalf = Precision<PREC>::kHalf, kBf = Precision<PREC>::kBfPlanes;
  constexpr int TK = T::kKnTK, TN = T::kKnTN;
  using Tile = KnTile<T::S, TK, TN>;
  auto kernel = right_transform_kn_kernel<typename T::Right, T::S, kHalf, TK, TN, T::kKnVec, T::kKnThreads,
                                           T::kKnBlocks, kBf>;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (Tile::kBytes > 48 * 1024 && dev >= 0 && dev < kMaxDevices) {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], kernel, Tile::kBytes)) return rc;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(d.ldk, TK)), static_cast<unsigned>(ceil_div(d.bn, TN)));
  const bool vec = (ldb % 8 == 0) && (d.bn % 8 == 0) && aligned(B, 16);
  kernel<<<grid, T::kKnThreads, Tile::kBytes, stream>>>(static_cast<const uint16_t*>(B), K, N, ldb,
                                                        static_cast<uint16_t*>(dst), d.bk, d.bn, d.ldk,
                                                        vec ? 1 : 0);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "right transform (K x N) launch");
  return FMM_OK;
}

// Runtime (scheme, dtype) -> template instance.  BF16 planes exist for rank 49
// only, the one scheme whose reference plan offers them (Rank49Plan's
// (bfloat16, bfloat16) precision pair).
template <template <int, int> class F, class... Args>
int dispatch(int scheme, int dtype, Args... args) {
  const bool half = dtype == FMM_DTYPE_F16;
  if (dtype == FMM_DTYPE_BF16_BF16 && scheme != FMM_SCHEME_RANK49)
    return fail(FMM_ERR_UNSUPPORTED, "BF16 planes (FMM_DTYPE_BF16_BF16) are offered for rank 49 only");
  switch (scheme) {
    case FMM_SCHEME_RANK7:
      return half ? F<FMM_SCHEME_RANK7, FMM_DTYPE_F16>::run(args...)
                  : F<FMM_SCHEME_RANK7, FMM_DTYPE_BF16>::run(args...);
    case FMM_SCHEME_RANK48:
      return half ? F<FMM_SCHEME_RANK48, FMM_DTYPE_F16>::run(args...)
                  : F<FMM_SCHEME_RANK48, FMM_DTYPE_BF16>::run(args...);
    case FMM_SCHEME_RANK343:
      // FP16 inputs and output only, as the reference plan (precision_pairs)
      if (!half) return fail(FMM_ERR_UNSUPPORTED, "rank 343 takes FP16 operands only");
      return F<FMM_SCHEME_RANK343, FMM_DTYPE_F16>::run(args...);
    default:
      if (dtype == FMM_DTYPE_BF16_BF16) return F<FMM_SCHEME_RANK49, FMM_DTYPE_BF16_BF16>::run(args...);
      return half ? F<FMM_SCHEME_RANK49, FMM_DTYPE_F16>::run(args...)
                  : F<FMM_SCHEME_RANK49, FMM_DTYPE_BF16>::run(args...);
  }
}
template <int SC, int H>
struct LeftOp {
  static int run(const void* A, int64_t M, int64_t K, int64_t lda, void* L, const fmm_dims* d,
                 cudaStream_t s) {
    return launch_input_transform<SC, false, H>(A, M, K, lda, L, d->bm, d->bk, d->ldk, s);
  }
};
template <int SC, int H>
struct PairedOp {
  static int run(const void* A, int64_t M, int64_t K, int64_t lda, void* L, const void* W, int64_t N,
                 int64_t ldw, void* Rt, const fmm_dims* d, cudaStream_t s) {
    return launch_paired_transform<SC, H>(A, M, K, lda, L, W, N, ldw, Rt, *d, s);
  }
};
template <int SC, int H>
struct WeightOp {
  static int run(const void* W, int64_t N, int64_t K, int64_t ldw, void* Rt, const fmm_dims* d,
                 cudaStream_t s) {
    return launch_input_transform<SC, true, H>(W, N, K, ldw, Rt, d->bn, d->bk, d->ldk, s);
  }
};
template <int SC, int H>
struct RightKnOp {
  static int run(const void* B, int64_t K, int64_t N, int64_t ldb, void* Rt, const fmm_dims* d,
                 cudaStream_t s) {
    return launch_right_kn<SC, H>(B, K, N, ldb, Rt, *d, s);
  }
};
template <int SC, int H>
struct ReconstructGatherOp {
  static int run(const void* P, const fmm_dims* d, int64_t M, int64_t N, const void* bias,
                 const GatherDests* dests, int64_t ldc, cudaStream_t s) {
    return launch_reconstruct_gather<SC, H>(P, *d, M, N, bias, *dests, ldc, s);
  }
};
template <int SC, int H>
struct ReconstructOp {
  static int run(const void* P, const fmm_dims* d, int64_t M, int64_t N, const void* bias, void* C,
                 int64_t ldc, cudaStream_t s) {
    return launch_reconstruct<SC, H>(P, *d, M, N, bias, C, ldc, s);
  }
};

int check_dtype(int dtype) {
  if (dtype != FMM_DTYPE_BF16 && dtype != FMM_DTYPE_F16 && dtype != FMM_DTYPE_BF16_BF16)
    return fail(FMM_ERR_UNSUPPORTED,
                "dtype must be FMM_DTYPE_BF16, FMM_DTYPE_F16 or FMM_DTYPE_BF16_BF16");
  return FMM_OK;
}

// ------------------------------------------------------------------ TMA maps
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

int tensor_map_encoder(PFN_cuTensorMapEncodeTiled_v12000* out) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (g_encode == nullptr) return fail(FMM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  *out = g_encode;
  return FMM_OK;
}

// Stacked 16-bit planes [batch][plane_rows][pitch] as a 3-D map over (k, row,
// batch), covering the first `rows` rows of every plane (rows <= plane_rows;
// `base` may point into a plane to start the band further down); box = 64
// K-elements (128 B, swizzled) x box_rows rows x 1 plane.  TMA copies the
// 2-byte elements without conversion, so the FP16 map serves BF16 planes too.
int plane_map(CUtensorMap* map, const void* base, int64_t k, int64_t rows, int64_t pitch,
              int64_t batch, uint32_t box_rows, int64_t plane_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (int rc = tensor_map_encoder(&encode)) return rc;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows),
                        static_cast<cuuint64_t>(batch)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch * 2),
                           static_cast<cuuint64_t>(pitch * 2 * plane_rows)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(kGemmBK), box_rows, 1};
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims,
                      strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return FMM_OK;
}

// Generic 3-D FP16 tiled map (128-byte swizzle); strides in bytes.
int tiled_map_3d(CUtensorMap* map, const void* base, const int64_t (&dims)[3],
                 const int64_t (&strides)[2], const uint32_t (&box)[3],
                 CUtensorMapSwizzle swizzle) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (int rc = tensor_map_encoder(&encode)) return rc;
  cuuint64_t d[3] = {static_cast<cuuint64_t>(dims[0]), static_cast<cuuint64_t>(dims[1]),
                     static_cast<cuuint64_t>(dims[2])};
  cuuint64_t st[2] = {static_cast<cuuint64_t>(strides[0]), static_cast<cuuint64_t>(strides[1])};
  cuuint32_t b[3] = {box[0], box[1], box[2]};
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), d, st, b,
                      elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return FMM_OK;
}

using GemmCfg = LeafGemmConfig<256, 4>;
using PairCfg256 = LeafGemmPairConfig<256, 7>;
using PairCfg192 = LeafGemmPairConfig<192, 7>;
using PairCfg128 = LeafGemmPairConfig<128, 8>;
using PairCfg256K128 = LeafGemmPairConfig<256, 3, 128>;
// the same two tiles with the TMA-store epilogue (one stage fewer for the
// epilogue's 16 KiB of shared-memory store buffers)
using PairCfg256Tma = LeafGemmPairConfig<256, 6, 64, true>;
using PairCfg256K128Tma = LeafGemmPairConfig<256, 3, 128, true>;
// narrower pair tiles with 128-deep k-blocks (TMA-store epilogue only): 3
// stages of 56 KiB at BN = 192, 4 of 48 KiB at BN = 128
using PairCfg192K128Tma = LeafGemmPairConfig<192, 3, 128, true>;
using PairCfg128K128Tma = LeafGemmPairConfig<128, 4, 128, true>;

enum GemmVariant {
  kVariantSingle = 0,
  kVariantPair256 = 1,
  kVariantPair128 = 2,
  kVariantPair192 = 3,
  kVariantPair256K128 = 4,  // 256x256 pair tile, 128-deep k-blocks in 3 stages
  kVariantPair192K128 = 5,  // 256x192 pair tile, 128-deep k-blocks in 3 stages
  kVariantPair128K128 = 6,  // 256x128 pair tile, 128-deep k-blocks in 4 stages
};

bool deep_k_variant(int variant) {
  return variant == kVariantPair256K128 || variant == kVariantPair192K128 || variant == kVariantPair128K128;
}

// Estimated relative cost of a variant: whole waves of full-tile equivalents
// over the SMs (or SM pairs), times the padded work one SM does per tile,
// divided by the variant's measured throughput relative to the 1-SM 128x256
// tile on B200 leaf shapes (a pair stages half of B per SM; 256x192 pairs
// measured 0.90 - 0.97 of one SM, 256x128 pairs slower still and only used
// when forced).  The ragged last N tile counts only the columns its MMA
// computes (the remainder rounded up to 16, or 32 for a pair).
double variant_cost(int variant, int64_t rank, int64_t bm, int64_t bn, int sms) {
  const bool pair = variant != kVariantSingle;
  const int64_t tm = pair ? 256 : 128;
  const int64_t tn = variant == kVariantPair128 ? 128 : (variant == kVariantPair192 ? 192 : 256);
  const int64_t granule = pair ? 32 : 16;
  const int64_t units = pair ? sms / 2 : sms;
  const double efficiency = variant == kVariantSingle    ? 1.0
                            : variant == kVariantPair256 ? 1.15
                            : variant == kVariantPair192 ? 0.95
                                                         : 0.70;
  const int64_t full_n = bn / tn;
  const int64_t last_cols = round_up(bn - full_n * tn, granule);
  const double n_tiles = double(full_n) + double(last_cols) / double(tn);
  const double waves = std::ceil(double(rank * ceil_div(bm, tm)) * n_tiles / double(units));
  return waves * double(tm * tn / (pair ? 2 : 1)) / efficiency;
}

int choose_variant(int64_t rank, int64_t bm, int64_t bn, int sms) {
  if (const char* forced = std::getenv("FMM_LEAF_GEMM_VARIANT")) {
    const std::string v(forced);
    if (v == "single") return kVariantSingle;
    if (v == "pair256") return kVariantPair256;
    if (v == "pair192") return kVariantPair192;
    if (v == "pair128") return kVariantPair128;
    if (v == "pair256k128") return kVariantPair256K128;
    if (v == "pair192k128") return kVariantPair192K128;
    if (v == "pair128k128") return kVariantPair128K128;
  }
  int best = kVariantSingle;
  double best_cost = variant_cost(kVariantSingle, rank, bm, bn, sms);
  for (int v : {kVariantPair256, kVariantPair192}) {
    const double c = variant_cost(v, rank, bm, bn, sms);
    if (c < best_cost) {
      best = v;
      best_cost = c;
    }
  }
  return best;
}

// Epilogue of the 256 x 256 pair GEMM: per-lane row stores, or shared-memory
// staged TMA stores (16 KiB of buffers).  The 128-deep configuration keeps its
// 3 stages either way and takes the TMA stores; the 64-deep one would lose one
// of its 7 stages and keeps the row stores.  FMM_LEAF_GEMM_EPILOGUE=rows|tma
// forces either.
bool tma_store_epilogue(int variant) {
  if (const char* v = std::getenv("FMM_LEAF_GEMM_EPILOGUE")) {
    if (std::string(v) == "tma") return true;
    if (std::string(v) == "rows") return false;
  }
  return deep_k_variant(variant);
}

template <class Kernel>
int ensure_smem_attribute(bool& done, Kernel kernel, size_t bytes) {
  if (done) return FMM_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(bytes));
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(leaf GEMM)");
  done = true;
  return FMM_OK;
}

template <class Cfg, bool kBf16>
int launch_pair(const void* L, const void* Rt, const LeafGemmParams& prm, int64_t ldk, int sms,
                cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(FMM_ERR_UNSUPPORTED, "device index out of range");
  CUtensorMap map_l, map_r, map_r16;
  if (int rc = plane_map(&map_l, L, prm.bk, prm.bm, ldk, prm.rank, kGemmBM, prm.plane_rows)) return rc;
  if (int rc = plane_map(&map_r, Rt, prm.bk, prm.bn, ldk, prm.rank, Cfg::kBN / 2, prm.bn)) return rc;
  // 16-row boxes for the ragged last N tile's halves
  if (int rc = plane_map(&map_r16, Rt, prm.bk, prm.bn, ldk, prm.rank, 16, prm.bn)) return rc;
  // P[rank][bm][ldp] for the TMA-store epilogue: boxes of 32 columns x 32 rows,
  // 64-byte swizzle (unused by the row-store epilogue)
  // 16-row boxes of L for the transposed tail tiles' B operand (rows past bm
  // read as zeros)
  CUtensorMap map_l16 = map_l;
  if (prm.tail_rows > 0) {
    if (int rc = plane_map(&map_l16, L, prm.bk, prm.bm, ldk, prm.rank, 16, prm.plane_rows)) return rc;
  }
  CUtensorMap map_p = map_l;
  if constexpr (Cfg::kTmaStore) {
    if (int rc = tiled_map_3d(&map_p, prm.P, {prm.ldp, prm.bm, int64_t(prm.rank)},
                              {prm.ldp * 2, prm.plane_rows * prm.ldp * 2}, {32u, 32u, 1u},
                              CU_TENSOR_MAP_SWIZZLE_64B))
      return rc;
  }
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], leaf_gemm_pair_kernel<Cfg, kBf16>, Cfg::kSmemBytes))
      return rc;
  }
  const int64_t tiles =
      int64_t(prm.rank) * (ceil_div(prm.bm - prm.tail_rows, Cfg::kTileM) * ceil_div(prm.bn, Cfg::kBN) + prm.tail_tiles);
  const int64_t pairs = tiles < sms / 2 ? tiles : sms / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs), 1, 1);
  cfg.blockDim = dim3(kGemmThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, leaf_gemm_pair_kernel<Cfg, kBf16>, map_l, map_r, map_r16, map_p, map_l16, prm);
  if (e != cudaSuccess) return cuda_fail(e, "leaf GEMM (pair) launch");
  return FMM_OK;
}

// ------------------------------------------------------------------ rank-343 output
// W^T of the rank-343 scheme as FP16 [64 outputs][384 products] (+-1 / 0,
// zero past product 343): one copy per device in static device memory,
// uploaded on the first rank-343 reconstruct on that device.
static __device__ __align__(1024) uint16_t g_rank343_wt[kRcN * kRcKPadded];

using RcCfg = ReconstructTcConfig<6>;

template <class Coefs>
int upload_coefficients(DeviceInfo* info) {
  static_assert(Coefs::kOutputs == kRcN && Coefs::kInputs == kRcRank, "rank-343 coefficient table");
  std::lock_guard<std::mutex> lock(g_device_mutex);
  if (info->rank343_wt != nullptr) return FMM_OK;
  std::vector<uint16_t> host(size_t(kRcN) * kRcKPadded, 0);
  for (int o = 0; o < kRcN; ++o)
    for (int r = 0; r < kRcRank; ++r)
      host[size_t(o) * kRcKPadded + r] =
          Coefs::kW[o][r] > 0 ? uint16_t(0x3C00) : (Coefs::kW[o][r] < 0 ? uint16_t(0xBC00) : uint16_t(0));
  cudaError_t e = cudaMemcpyToSymbol(g_rank343_wt, host.data(), host.size() * sizeof(uint16_t));
  if (e != cudaSuccess) return cuda_fail(e, "upload of the rank-343 coefficients");
  void* addr = nullptr;
  e = cudaGetSymbolAddress(&addr, g_rank343_wt);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress(g_rank343_wt)");
  info->rank343_wt = addr;
  return FMM_OK;
}

template <class Coefs, bool kHalf>
int launch_reconstruct_tc(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                          void* C, int64_t ldc, DeviceInfo* info, cudaStream_t stream) {
  if (int rc = upload_coefficients<Coefs>(info)) return rc;
  CUtensorMap map_p, map_w;
  // P[343][bm][ldp] as (position, row, product); box 64 positions x 1 row x 64 products
  if (int rc = tiled_map_3d(&map_p, P, {d.ldp, d.bm, kRcRank}, {d.ldp * 2, d.bm * d.ldp * 2},
                            {64u, 1u, static_cast<uint32_t>(kRcK)}, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int rc = tiled_map_3d(&map_w, info->rank343_wt, {kRcKPadded, kRcN, 1},
                            {int64_t(kRcKPadded) * 2, int64_t(kRcKPadded) * kRcN * 2},
                            {static_cast<uint32_t>(kRcK), static_cast<uint32_t>(kRcN), 1u},
                            CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(info->reconstruct_tc_configured,
                                       reconstruct_tc_kernel<RcCfg, kHalf>, RcCfg::kSmemBytes))
      return rc;
  }
  ReconstructTcParams prm;
  prm.bm = d.bm;
  prm.bn = d.bn;
  prm.M = M;
  prm.N = N;
  prm.ldc = ldc;
  const int64_t per_row = ceil_div(d.bn, kRcM);
  if (d.bm * per_row > 0x7fffffff) return fail(FMM_ERR_TOO_LARGE, "too many reconstruct tiles");
  prm.tiles_per_row = static_cast<int32_t>(per_row);
  prm.total_tiles = static_cast<int32_t>(d.bm * per_row);
  prm.vector_stores = (d.bn % 8 == 0 && ldc % 8 == 0 && aligned(C, 16)) ? 1 : 0;
  prm.bias = static_cast<const uint16_t*>(bias);
  prm.C = static_cast<uint16_t*>(C);
  prm.timeout_ns = g_timeout_ns;
  const int sms = usable_sms(info);
  const int grid = prm.total_tiles < sms ? prm.total_tiles : sms;
  reconstruct_tc_kernel<RcCfg, kHalf><<<grid, kRcThreads, RcCfg::kSmemBytes, stream>>>(map_p, map_w, prm);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "rank-343 reconstruct launch");
  return FMM_OK;
}

// TMA-staged reconstruct of a circuit scheme: persistent CTAs, one box of
// 256 positions x R products per tile (unswizzled, so plane r of a tile sits at
// r * 256 elements in shared memory), two positions a compute thread.
template <int SCHEME, int PREC>
int launch_reconstruct_staged(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                              void* C, int64_t ldc, DeviceInfo* info, cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  using Prog = typename T::Output;
  using Cfg = StagedReconstructConfig<Prog, T::kOutStages>;
  auto kernel = reconstruct_staged_kernel<Prog, T::S, T::kOutStages, Precision<PREC>::kHalf, Cfg::kTP,
                                          T::kOutStagedBlocks, Precision<PREC>::kBfPlanes>;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(FMM_ERR_UNSUPPORTED, "device index out of range");
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], kernel, Cfg::kSmemBytes)) return rc;
  }
  CUtensorMap map_p;
  if (int rc = tiled_map_3d(&map_p, P, {d.ldp, d.bm, int64_t(Cfg::kR)}, {d.ldp * 2, d.bm * d.ldp * 2},
                            {uint32_t(Cfg::kTP), 1u, uint32_t(Cfg::kR)}, CU_TENSOR_MAP_SWIZZLE_NONE))
    return rc;
  StagedReconstructParams prm;
  prm.bm = d.bm;
  prm.bn = d.bn;
  prm.M = M;
  prm.N = N;
  prm.ldc = ldc;
  const int64_t per_row = ceil_div(d.bn, Cfg::kTP);
  if (d.bm * per_row > 0x7fffffff) return fail(FMM_ERR_TOO_LARGE, "too many reconstruct tiles");
  prm.tiles_per_row = static_cast<int32_t>(per_row);
  prm.total_tiles = static_cast<int32_t>(d.bm * per_row);
  const bool vec = (d.bn % Cfg::kVec == 0) && (ldc % Cfg::kVec == 0) && aligned(C, 2 * Cfg::kVec);
  const bool vec_bias = (d.bn % Cfg::kVec == 0) && bias != nullptr && aligned(bias, 2 * Cfg::kVec);
  prm.vector_flags = (vec ? 1 : 0) | (vec_bias ? 2 : 0);
  prm.bias = static_cast<const uint16_t*>(bias);
  prm.C = static_cast<uint16_t*>(C);
  prm.timeout_ns = g_timeout_ns;
  const int64_t cap = int64_t(usable_sms(info)) * T::kOutStagedBlocks;
  const int grid = static_cast<int>(prm.total_tiles < cap ? prm.total_tiles : cap);
  kernel<<<grid, Cfg::kThreads, Cfg::kSmemBytes, stream>>>(map_p, prm);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "staged reconstruct launch");
  return FMM_OK;
}

// The staged reconstruct fused with the gather (bulk-copy stores into every
// destination): 512-position tiles (two TMA boxes) in 3 stages, 8 compute
// warps, one CTA per SM, the grid the SM budget in force (fmm_set_sm_budget),
// so a leaf GEMM launched beside it with the complementary budget keeps its
// SMs whole.
constexpr int kGatherStages = 3;

template <int SCHEME, int PREC>
int launch_reconstruct_staged_gather(const void* P, const fmm_dims& d, int64_t M, int64_t N, const void* bias,
                                     const GatherDests& dests, int64_t ldc, DeviceInfo* info,
                                     cudaStream_t stream) {
  using T = SchemeTraits<SCHEME>;
  using Prog = typename T::Output;
  using Cfg = StagedGatherConfig<Prog, kGatherStages>;
  auto kernel = reconstruct_staged_gather_kernel<Prog, T::S, kGatherStages, Precision<PREC>::kHalf, Cfg::kTP,
                                                 Precision<PREC>::kBfPlanes>;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(FMM_ERR_UNSUPPORTED, "device index out of range");
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], kernel, Cfg::kSmemBytes)) return rc;
  }
  CUtensorMap map_p;
  if (int rc = tiled_map_3d(&map_p, P, {d.ldp, d.bm, int64_t(Cfg::kR)}, {d.ldp * 2, d.bm * d.ldp * 2},
                            {uint32_t(Cfg::kBoxTP), 1u, uint32_t(Cfg::kR)}, CU_TENSOR_MAP_SWIZZLE_NONE))
    return rc;
  StagedReconstructParams prm;
  prm.bm = d.bm;
  prm.bn = d.bn;
  prm.M = M;
  prm.N = N;
  prm.ldc = ldc;
  const int64_t per_row = ceil_div(d.bn, Cfg::kTP);
  if (d.bm * per_row > 0x7fffffff) return fail(FMM_ERR_TOO_LARGE, "too many reconstruct tiles");
  prm.tiles_per_row = static_cast<int32_t>(per_row);
  prm.total_tiles = static_cast<int32_t>(d.bm * per_row);
  const bool vec_bias = (d.bn % Cfg::kVec == 0) && bias != nullptr && aligned(bias, 2 * Cfg::kVec);
  prm.vector_flags = vec_bias ? 2 : 0;  // bit 0 (vector stores into C) is unused: copies write C
  prm.bias = static_cast<const uint16_t*>(bias);
  prm.C = nullptr;
  prm.timeout_ns = g_timeout_ns;
  const int64_t cap = usable_sms(info);
  const int grid = static_cast<int>(prm.total_tiles < cap ? prm.total_tiles : cap);
  kernel<<<grid, Cfg::kThreads, Cfg::kSmemBytes, stream>>>(map_p, prm, dests);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "staged gathering reconstruct launch");
  return FMM_OK;
}

// The 1-SM GEMM (small or ragged leaves).
template <bool kBf16>
int launch_single(const void* L, const void* Rt, const LeafGemmParams& prm, int64_t ldk, int sms,
                  cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(FMM_ERR_UNSUPPORTED, "device index out of range");
  CUtensorMap map_l, map_r;
  if (int rc = plane_map(&map_l, L, prm.bk, prm.bm, ldk, prm.rank, kGemmBM, prm.plane_rows)) return rc;
  if (int rc = plane_map(&map_r, Rt, prm.bk, prm.bn, ldk, prm.rank, GemmCfg::kBN, prm.bn)) return rc;
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], leaf_gemm_kernel<GemmCfg, kBf16>, GemmCfg::kSmemBytes))
      return rc;
  }
  const int64_t tiles = int64_t(prm.rank) * prm.tiles_m * prm.tiles_n;
  const int grid = static_cast<int>(tiles < sms ? tiles : sms);
  leaf_gemm_kernel<GemmCfg, kBf16><<<grid, kGemmThreads, GemmCfg::kSmemBytes, stream>>>(map_l, map_r, prm);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "leaf GEMM launch");
  return FMM_OK;
}

// M-tiles per group of the tile order (a group sweeps all N-tiles of its
// M-tiles before the next group starts, so the group's L rows and the
// weight planes' N-tiles are reused from L2): 16, or FMM_LEAF_GEMM_GROUP_M.
int leaf_group_m() {
  if (const char* v = std::getenv("FMM_LEAF_GEMM_GROUP_M")) {
    const int g = std::atoi(v);
    if (g >= 1 && g <= 4096) return g;
  }
  return 16;
}

// Serpentine N order across tile groups (on; FMM_LEAF_GEMM_SERPENTINE=0 turns
// it off): a group starts on the weight-plane columns its predecessor used
// last, which cut the c5b launch's DRAM reads from 4.87 to 4.19 GB (ncu, one
// full-size launch); its time moved less than the run-to-run noise.
int leaf_serpentine() {
  const char* v = std::getenv("FMM_LEAF_GEMM_SERPENTINE");
  return (v != nullptr && std::string(v) == "0") ? 0 : 1;
}

// One GEMM launch over rows [row0, row0 + rows) of every plane (planes of
// `plane_rows` rows), with the given variant and epilogue.
template <bool kBf16>
int launch_leaf_band(int variant, bool tma_store, int rank, const uint16_t* L, const void* Rt,
                     int64_t row0, int64_t rows, int64_t plane_rows, int64_t bn, int64_t bk,
                     uint16_t* P, int sms, cudaStream_t stream, int64_t transposed_tail = 0) {
  const int64_t ldk = round_up(bk, 8), ldp = round_up(bn, 8);
  const uint16_t* band_l = L + row0 * ldk;
  LeafGemmParams prm;
  prm.bm = rows;
  prm.bn = bn;
  prm.bk = bk;
  prm.ldp = ldp;
  prm.plane_rows = plane_rows;
  prm.rank = rank;
  prm.tiles_m = static_cast<int32_t>(ceil_div(rows, kGemmBM));
  prm.tiles_n = static_cast<int32_t>(ceil_div(bn, GemmCfg::kBN));
  prm.group_m = leaf_group_m();
  prm.serpentine = leaf_serpentine();
  prm.tail_rows = static_cast<int32_t>(transposed_tail);
  prm.tail_tiles = transposed_tail > 0 ? static_cast<int32_t>(ceil_div(bn, 256)) : 0;
  prm.P = P + row0 * ldp;
  prm.timeout_ns = g_timeout_ns;
  if (variant == kVariantPair256) {
    return tma_store ? launch_pair<PairCfg256Tma, kBf16>(band_l, Rt, prm, ldk, sms, stream)
                     : launch_pair<PairCfg256, kBf16>(band_l, Rt, prm, ldk, sms, stream);
  }
  if (variant == kVariantPair256K128) {
    return tma_store ? launch_pair<PairCfg256K128Tma, kBf16>(band_l, Rt, prm, ldk, sms, stream)
                     : launch_pair<PairCfg256K128, kBf16>(band_l, Rt, prm, ldk, sms, stream);
  }
  // the narrow 128-deep configurations exist with the TMA-store epilogue only
  if (variant == kVariantPair192K128) return launch_pair<PairCfg192K128Tma, kBf16>(band_l, Rt, prm, ldk, sms, stream);
  if (variant == kVariantPair128K128) return launch_pair<PairCfg128K128Tma, kBf16>(band_l, Rt, prm, ldk, sms, stream);
  if constexpr (!kBf16) {
    if (variant == kVariantPair192) return launch_pair<PairCfg192, false>(band_l, Rt, prm, ldk, sms, stream);
    if (variant == kVariantPair128) return launch_pair<PairCfg128, false>(band_l, Rt, prm, ldk, sms, stream);
  }
  return launch_single<kBf16>(band_l, Rt, prm, ldk, sms, stream);
}

// Rows of a short last M tile of the 2-SM GEMM, run as a second, 1-SM launch
// of 128-row tiles over the planes' last rows (one SM instead of two for each
// of their tiles) when FMM_LEAF_GEMM_TAIL=1 and the planes' last 256-row tile
// holds at most 128 rows.  Off by default: on c4 (bm = 2054, a 6-row last
// tile) the two launches measured 0.7 % slower than one (0.591 vs 0.587 ms,
// GEMM alone, three interleaved rounds) -- the second launch's partial waves
// cost what the narrower tiles save.
int64_t split_tail_rows(int variant, int64_t bm) {
  if (variant == kVariantSingle) return 0;
  const int64_t tail = bm % 256;
  if (bm < 256 || tail == 0 || tail > 128) return 0;
  const char* v = std::getenv("FMM_LEAF_GEMM_TAIL");
  return (v != nullptr && std::string(v) == "1") ? tail : 0;
}

// Rows of a short last M tile (1..32 rows) that the 256 x 256 pair kernels
// compute transposed inside the same launch: P^T = Rt * L_tail^T in 256 x 32
// tiles over bn, an eighth of a regular tile's MMA work, instead of padding
// the rows to a whole 256-row tile (c4: bm = 2054, 6 rows).
// FMM_LEAF_GEMM_TAIL=0 pads them as before; =1 selects the 1-SM band above.
int64_t transposed_tail_rows(int variant, int64_t bm) {
  if (variant != kVariantPair256 && variant != kVariantPair256K128) return 0;
  const int64_t tail = bm % 256;
  if (bm < 256 || tail == 0 || tail > 32) return 0;
  const char* v = std::getenv("FMM_LEAF_GEMM_TAIL");
  if (v != nullptr && (std::string(v) == "0" || std::string(v) == "1")) return 0;
  return tail;
}

// FP16 planes (kBf16 = false) or BF16 planes.  The BF16 form carries the
// 1-SM configuration and every 128-deep pair configuration; a forced narrower
// 64-deep pair variant runs as the 256 x 256 pair there.
template <bool kBf16>
int launch_leaf_gemm(int rank, const void* L, const void* Rt, int64_t bm, int64_t bn, int64_t bk,
                     void* P, cudaStream_t stream) {
  if (rank < 1 || bm < 1 || bn < 1 || bk < 1)
    return fail(FMM_ERR_INVALID_ARGUMENT, "leaf GEMM dimensions must be positive");
  if (!aligned(L, 16) || !aligned(Rt, 16) || !aligned(P, 16))
    return fail(FMM_ERR_MISALIGNED, "leaf GEMM planes must be 16-byte aligned");
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  if (int64_t(rank) * ceil_div(bm, kGemmBM) * ceil_div(bn, 128) > (int64_t(1) << 30))
    return fail(FMM_ERR_TOO_LARGE, "too many GEMM tiles");
  const int sms = usable_sms(info);
  int variant = choose_variant(rank, bm, bn, sms);
  // 128-deep k-blocks with the TMA-store epilogue, from bk = 1024 up (at most
  // 6 % of the last k-block's MMA work is zero padding there): measured
  // against 64-deep k-blocks in 7 stages with row stores (GEMM alone, full
  // clock, L2 flushed, 3 interleaved rounds): c2 0.256 -> 0.240 ms, c5a
  // 0.594 -> 0.557, c5b 4.11-4.17 -> 3.95-4.09 (against 64-deep k-blocks with
  // the TMA stores there, the previous choice).  A forced
  // FMM_LEAF_GEMM_VARIANT keeps its own k-depth.
  if (bk >= 1024 && std::getenv("FMM_LEAF_GEMM_VARIANT") == nullptr) {
    if (variant == kVariantPair256) variant = kVariantPair256K128;
    if (variant == kVariantPair192) variant = kVariantPair192K128;
    if (variant == kVariantPair128) variant = kVariantPair128K128;
  }
  if (kBf16 && (variant == kVariantPair192 || variant == kVariantPair128)) variant = kVariantPair256;
  const bool tma_store = tma_store_epilogue(variant);
  const uint16_t* l16 = static_cast<const uint16_t*>(L);
  uint16_t* p16 = static_cast<uint16_t*>(P);
  const int64_t tail = split_tail_rows(variant, bm);
  const int64_t transposed = tail == 0 ? transposed_tail_rows(variant, bm) : 0;
  if (int rc = launch_leaf_band<kBf16>(variant, tma_store, rank, l16, Rt, 0, bm - tail, bm, bn, bk, p16, sms,
                                       stream, transposed))
    return rc;
  if (tail == 0) return FMM_OK;
  // the short last band: same stream, after the 2-SM launch
  return launch_leaf_band<kBf16>(kVariantSingle, false, rank, l16, Rt, bm - tail, tail, bm, bn, bk, p16, sms,
                                 stream);
}

// ------------------------------------------------------------------ 8-bit integer linear
// Launch that may overlap the end of the kernel before it in the stream
// (wait_for_previous_kernel), in clusters of `cluster` CTAs.
template <class... P, class... A>
int launch_int8(void (*kernel)(P...), const char* what, int64_t grid, int threads, size_t shared, int cluster,
                cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  return FMM_OK;
}

template <class T, class G, bool kNorm, int V, bool kVec>
int launch_int8_rows(const Int8RowsParams& p, int threads, const DeviceInfo* info, cudaStream_t stream) {
  const int rows_per_block = p.warps_per_row > 1 ? 1 : threads / 32;
  const int64_t blocks = ceil_div(p.rows, rows_per_block);
  // the blocks that an SM is sure to hold at once (64 registers a thread); each takes row after row
  const int64_t cap = int64_t(usable_sms(info)) * (kRowsMaxThreads / threads);
  const int grid = static_cast<int>(blocks < cap ? blocks : cap);
  return launch_int8(int8_rows_kernel<T, G, kNorm, V, kVec>,
                     kNorm ? "RMS norm (8-bit) launch" : "row quantisation launch", grid, threads, 0, 1, stream, p);
}

constexpr size_t kRowsRingBytes = 216 * 1024;  // rings of the streamed form

// Streamed form: as many groups as the rings of two stages leave room for (32
// at most; 15 where groups have several warps, and so a barrier each), more
// stages where there is room.  A lane takes about eight vectors of a row, so
// that the reduction is a small part of its work, but 15 warps are at work at
// least.  Measured (us, bf16): 16384 elements, three groups of 5, 8, 10 warps
// 48.2, 43.0, 48.2 (4992 rows); norm of 4608 with residual, five groups of 2,
// 3, 4, 6 warps 391, 334, 362, 385 (65536 rows); 32768 elements, one group of
// 12, 16, 24, 32 warps 169, 156, 169, 182 (8192 rows).  Rows that are not
// aligned have many more instructions: all 32 warps (12288 x 4607 in FP32, five
// groups of 1, 2, 6 warps: 159, 101, 70).  Returns false where two stages of a row do not fit.
bool plan_streamed_rows(Int8RowsParams* p, size_t slot, size_t code_bytes, size_t gain_bytes) {
  if (gain_bytes >= kRowsRingBytes) return false;
  const size_t room = kRowsRingBytes - gain_bytes;
  const size_t stage = slot * (p->residual != nullptr ? 2 : 1);
  int64_t groups = static_cast<int64_t>(room / (2 * stage + code_bytes));
  if (groups < 1) return false;
  if (groups > kRowsMaxGroups) groups = kRowsMaxGroups;
  const int64_t vectors = ceil_div(p->cols, 8);
  int64_t warps = 32 / groups;
  if (code_bytes == 0) {
    const int64_t enough = ceil_div(15, groups);
    warps = (vectors + 128) / 256;
    if (warps < enough) warps = enough;
  }
  if (warps > ceil_div(vectors, 32)) warps = ceil_div(vectors, 32);
  if (warps < 1) warps = 1;
  if (warps > 1 && groups > 15) groups = 15;
  const int64_t total = (code_bytes == 0 && gain_bytes > 0 ? kRowsNormThreads : kRowsMaxThreads) / 32;
  if (groups * warps > total) groups = total / warps;
  p->groups = static_cast<int32_t>(groups);
  p->warps_per_row = static_cast<int32_t>(warps);
  p->stages = kRowsMaxStages;
  while (p->stages > 2 && groups * (p->stages * stage + code_bytes) > room) --p->stages;
  return true;
}

template <class T, class G, bool kNorm, bool kVec>
int launch_int8_rows_streamed(Int8RowsParams p, size_t shared, const DeviceInfo* info, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  p.timeout_ns = g_timeout_ns;
  auto kernel = int8_rows_streamed_kernel<T, G, kNorm, kVec>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], kernel, kRowsRingBytes)) return rc;
  }
  const int64_t blocks = ceil_div(p.rows, p.groups);
  const int sms = usable_sms(info);
  const int grid = static_cast<int>(blocks < sms ? blocks : sms);
  return launch_int8(kernel, kNorm ? "RMS norm (8-bit) launch" : "row quantisation launch", grid,
                     32 * p.warps_per_row * p.groups, shared, 1, stream, p);
}

// Many rows of more than one vector a lane are streamed (65536 BF16 rows, us
// streamed and from registers: 256 elements 23.6, 17.2; 512: 30.2, 29.5; 1024:
// 41.4, 46.9; norms with a residual of 256: 40.3, 32.2, of 1024: 79.5, 112; FP32
// rows of 256: 22.6, 17.9).  Otherwise a row of up to 1024 elements is one warp's (four vectors of
// 8 a lane), four rows a block; longer rows are a block's, with the fewest
// vectors a thread that 1024 threads cover; beyond 32768 elements the row is
// read twice.
template <class T, class G, bool kNorm, bool kVec>
int dispatch_int8_rows(Int8RowsParams p, const DeviceInfo* info, cudaStream_t stream) {
  const int64_t vectors = ceil_div(p.cols, 8);
  const int64_t row_bytes = p.cols * int64_t(sizeof(T));
  if (vectors > 32) {
    // the streamed form takes vectors of 8 elements where rows are whole ones
    // (FP32 rows of 4 n elements are aligned, but need not be), else elements
    const bool whole = kVec && p.cols % 8 == 0;
    const size_t slot = static_cast<size_t>(round_up(row_bytes, 16)) + (whole ? 0 : 16);
    const size_t code_bytes = whole ? 0 : static_cast<size_t>(round_up(p.cols, 16));
    const size_t gain_bytes = kNorm ? static_cast<size_t>(round_up(p.cols * int64_t(4), 16)) : 0;
    Int8RowsParams streamed = p;
    if (plan_streamed_rows(&streamed, slot, code_bytes, gain_bytes) &&
        p.rows > 2 * int64_t(usable_sms(info)) * streamed.groups) {
      const size_t shared =
          gain_bytes + streamed.groups * (streamed.stages * slot * (p.residual != nullptr ? 2 : 1) + code_bytes);
      if constexpr (kVec) {
        if (whole) return launch_int8_rows_streamed<T, G, kNorm, true>(streamed, shared, info, stream);
      }
      return launch_int8_rows_streamed<T, G, kNorm, false>(streamed, shared, info, stream);
    }
  }
  if (vectors <= 128) {
    p.warps_per_row = 1;
    if (vectors <= 32) return launch_int8_rows<T, G, kNorm, 1, kVec>(p, 128, info, stream);
    if (vectors <= 64) return launch_int8_rows<T, G, kNorm, 2, kVec>(p, 128, info, stream);
    return launch_int8_rows<T, G, kNorm, 4, kVec>(p, 128, info, stream);
  }
  auto warps = [&](int v) { return static_cast<int>(ceil_div(ceil_div(vectors, v), 32)); };
  const int most = kRowsMaxThreads / 32;
  if (warps(1) <= most) {
    p.warps_per_row = warps(1);
    return launch_int8_rows<T, G, kNorm, 1, kVec>(p, 32 * p.warps_per_row, info, stream);
  }
  if (warps(2) <= most) {
    p.warps_per_row = warps(2);
    return launch_int8_rows<T, G, kNorm, 2, kVec>(p, 32 * p.warps_per_row, info, stream);
  }
  if (warps(4) <= most) {
    p.warps_per_row = warps(4);
    return launch_int8_rows<T, G, kNorm, 4, kVec>(p, 32 * p.warps_per_row, info, stream);
  }
  p.warps_per_row = most;
  return launch_int8_rows<T, G, kNorm, 0, kVec>(p, kRowsMaxThreads, info, stream);
}

// kVec: every row of every tensor starts on a vector's boundary.
template <class T, class G, bool kNorm>
int run_int8_rows(const Int8RowsParams& p, cudaStream_t stream) {
  if (p.rows == 0) return FMM_OK;
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  constexpr int64_t kPer16 = 16 / sizeof(T);
  bool vec = aligned(p.x, 16) && p.ldx % kPer16 == 0 && aligned(p.codes, 8) && p.ldq % 8 == 0;
  if (kNorm) vec = vec && aligned(p.gain, 16);
  if (p.residual != nullptr)
    vec = vec && aligned(p.residual, 16) && p.ldr % kPer16 == 0 && aligned(p.residual_out, 16) && p.ldo % kPer16 == 0;
  return vec ? dispatch_int8_rows<T, G, kNorm, true>(p, info, stream)
             : dispatch_int8_rows<T, G, kNorm, false>(p, info, stream);
}

int check_rows(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) return fail(FMM_ERR_INVALID_ARGUMENT, "rows must not be negative and columns positive");
  if (cols > (int64_t(1) << 30)) return fail(FMM_ERR_TOO_LARGE, "rows of more than 2^30 elements");
  return FMM_OK;
}

// 8-bit codes [rows][ld] as a 2-D map over (k, row); box = 128 codes (one
// swizzled 128-byte row) x box_rows.
int codes_map(CUtensorMap* map, const void* base, int64_t k, int64_t rows, int64_t ld, uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (int rc = tensor_map_encoder(&encode)) return rc;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kI8BlockK), box_rows};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return FMM_OK;
}

constexpr size_t kI8MaxSmem = 232448;

// Y[M][N] (16-bit) as a 2-D map over (channel, token); box 32 x 32, 64-byte swizzle.
int output_map(CUtensorMap* map, void* base, int64_t M, int64_t N, int64_t ld) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (int rc = tensor_map_encoder(&encode)) return rc;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(M)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * 2)};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, dims, strides, box, elem,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return FMM_OK;
}

// How a product is taken: which way the tiles lie (two SMs a tile: channels in
// the lanes; with tokens there its outputs were no faster, 65536 x 4608 x 12288
// 2.54 ms to 2.24), two SMs a tile or one, and an SM's tile.
struct Int8Shape {
  bool tokens, pair;
  int lanes, cols;
};

// Measured (one B200, us): a 128-deep column of K costs a tile of 128 lanes
// 0.15 + 0.0011 cols (64, 128, 192, 256: 0.20, 0.28, 0.36, 0.43), one of 64 lanes
// about an eighth less, a 256 x 256 tile of two SMs 0.37 however many of its
// columns exist.  The outputs of an SM's tile take 0.5 + 0.0097 cols beside the
// next tile's products, 0.0076 by TMA; every launch costs some 4 more.
double int8_cost(int64_t M, int64_t K, int64_t N, const Int8Shape& s, int sms) {
  const int64_t lane_end = s.tokens ? M : N, col_end = s.tokens ? N : M;
  const double columns = double(ceil_div(K, kI8BlockK));
  const double out = 0.5 + (s.tokens ? 0.0076 : 0.0097) * s.cols;
  double tile = 0;
  int64_t tiles = 0, units = 0;
  if (s.pair) {
    tiles = ceil_div(lane_end, 256) * ceil_div(col_end, 256);
    units = sms / 2;
    tile = columns * 0.37;
  } else {
    tiles = ceil_div(lane_end, s.lanes) * ceil_div(col_end, s.cols);
    units = sms;
    tile = columns * (0.15 + 0.0011 * s.cols) * (s.lanes < kI8Lanes ? 0.875 : 1.0);
  }
  return (s.pair ? 5.0 : 4.0) + double(ceil_div(tiles, units)) * (tile > out ? tile : out);
}

// The least estimate over tokens in equal tiles and tiles of the usual widths;
// `aligned`: the outputs may leave by TMA.
Int8Shape choose_int8_shape(int64_t M, int64_t K, int64_t N, bool aligned, int sms) {
  Int8Shape best = {false, false, kI8Lanes, 16};
  double least = 1e30;
  auto consider = [&](bool tokens, bool pair, int lanes, int64_t cols) {
    const Int8Shape s = {tokens, pair, lanes, static_cast<int>(cols)};
    const double c = int8_cost(M, K, N, s, sms);
    if (c < least) {
      least = c;
      best = s;
    }
  };
  for (int lanes : {kI8Lanes, kI8Lanes / 2}) {
    for (int64_t pieces = ceil_div(M, 256); pieces <= 16; ++pieces)
      consider(false, false, lanes, round_up(ceil_div(M, pieces), 16));
    if (M > 256)
      for (int64_t tok : {64, 96, 128, 192, 256}) consider(false, false, lanes, tok);
  }
  consider(false, true, kI8Lanes, 256);
  if (aligned && M > 64) {
    for (int64_t cols : {64, 96, 128, 192, 256}) consider(true, false, kI8Lanes, cols);
  }
  return best;
}

template <bool kBf16, bool kTokens>
int launch_int8_single(const int8_t* codes, int64_t ldq, const int8_t* weight_codes, int64_t ldw, Int8LinearParams p,
                       const Int8Shape& shape, int sms, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  p.lanes = shape.lanes;
  p.cols = shape.cols;
  p.tmem_cols = 32;
  while (p.tmem_cols < static_cast<uint32_t>(p.cols)) p.tmem_cols *= 2;
  p.tiles_m = static_cast<int32_t>(ceil_div(p.M, kTokens ? p.lanes : p.cols));
  p.tiles_n = static_cast<int32_t>(ceil_div(p.N, kTokens ? p.cols : p.lanes));
  // 128-deep columns of a stage: as many as keep it at 64 KB (three stages), up
  // to four.  64 channels x 16 tokens, K = 4096, with 1, 2, 4: 13.4, 10.7, 10.0
  // us; 128 x 128: 14.3, 13.5; 128 x 192 with 1, 2: 27.1, 32.8
  p.atoms = p.lanes + p.cols <= 128 ? 4 : p.lanes + p.cols <= 256 ? 2 : 1;
  const size_t stage = p.atoms * size_t(p.lanes + p.cols) * kI8BlockK;
  // alignment, barriers, blocks of outputs, and the rows that products read
  // behind the last stage's
  const size_t control = 1024 + 8 * (2 * kI8MaxStages + 6) + size_t(kI8Lanes - p.lanes) * kI8BlockK +
                         (kTokens ? size_t(kI8EpilogueWarps) * 2 * kI8BlockBytes : 0);
  p.stages = kI8MaxStages;
  while (p.stages > 1 && p.stages * stage + control > kI8MaxSmem) --p.stages;
  const size_t smem = p.stages * stage + control;
  CUtensorMap map_a, map_b;
  if (int rc = codes_map(&map_a, kTokens ? codes : weight_codes, p.K, kTokens ? p.M : p.N, kTokens ? ldq : ldw,
                         static_cast<uint32_t>(p.lanes)))
    return rc;
  if (int rc = codes_map(&map_b, kTokens ? weight_codes : codes, p.K, kTokens ? p.N : p.M, kTokens ? ldw : ldq,
                         static_cast<uint32_t>(p.cols)))
    return rc;
  CUtensorMap map_c = map_a;  // not read where tokens are columns
  if (kTokens) {
    if (int rc = output_map(&map_c, p.out, p.M, p.N, p.ldc)) return rc;
  }
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], int8_linear_kernel<kBf16, kTokens>, kI8MaxSmem)) return rc;
  }
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
  const int grid = static_cast<int>(tiles < sms ? tiles : sms);
  return launch_int8(int8_linear_kernel<kBf16, kTokens>, "8-bit linear launch", grid, kI8Threads, smem, 1, stream,
                     map_a, map_b, map_c, p);
}

template <bool kBf16>
int launch_int8_pair(const int8_t* codes, int64_t ldq, const int8_t* weight_codes, int64_t ldw, Int8LinearParams p,
                     int sms, cudaStream_t stream) {
  using Cfg = Int8PairConfig;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  p.tiles_m = static_cast<int32_t>(ceil_div(p.M, Cfg::kTile));
  p.tiles_n = static_cast<int32_t>(ceil_div(p.N, Cfg::kTile));
  CUtensorMap map_a, map_b, map_b16;
  if (int rc = codes_map(&map_a, weight_codes, p.K, p.N, ldw, 128)) return rc;
  if (int rc = codes_map(&map_b, codes, p.K, p.M, ldq, 128)) return rc;
  if (int rc = codes_map(&map_b16, codes, p.K, p.M, ldq, 16)) return rc;
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], int8_linear_pair_kernel<kBf16>, Cfg::kSmemBytes)) return rc;
  }
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
  const int64_t pairs = tiles < sms / 2 ? tiles : sms / 2;
  // four epilogue warps keep up with a long K, and leave it more power
  // (65536 x 4608 x 12288: 2305 us with eight, 2268)
  const int threads = p.K >= 2048 ? 64 + 32 * 4 : kI8Threads;
  return launch_int8(int8_linear_pair_kernel<kBf16>, "8-bit linear (pair) launch", 2 * pairs, threads,
                     Cfg::kSmemBytes, 2, stream, map_a, map_b, map_b16, p);
}

constexpr size_t kI8FewShared = 216 * 1024;

bool int8_few_fits(int64_t M, int64_t K) { return M * round_up(K, 16) <= int64_t(kI8FewShared / 2); }

// Warps and stages of the few-token kernel beside the tokens' codes.
void plan_int8_few(int64_t M, int64_t K, int64_t N, int channels, int sms, int* warps, int* stages, size_t* shared) {
  const size_t tokens = static_cast<size_t>(M * round_up(K, 16));
  // units of an SM, and as many warps as take an equal number of them
  const int64_t each = ceil_div(ceil_div(N, channels), sms);
  *warps = static_cast<int>(ceil_div(each, ceil_div(each, kI8FewMaxWarps)));
  const size_t stage = size_t(channels) * kI8FewK, room = (kI8FewShared - tokens) / stage;
  *stages = static_cast<int>(room / *warps);
  if (*stages > kI8FewMaxStages) *stages = kI8FewMaxStages;
  if (*stages < 2) {
    *warps = static_cast<int>(room / 2);
    *stages = 2;
  }
  *shared = *warps * *stages * stage + tokens;
}

template <bool kBf16, int MT, int R>
int launch_int8_few(Int8FewParams p, int sms, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  auto kernel = int8_linear_few_kernel<kBf16, MT, R>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  {
    std::lock_guard<std::mutex> lock(g_device_mutex);
    if (int rc = ensure_smem_attribute(configured[dev], kernel, kI8FewShared)) return rc;
  }
  int warps = 0;
  size_t shared = 0;
  plan_int8_few(p.M, p.K, p.N, R, sms, &warps, &p.stages, &shared);
  const int64_t units = ceil_div(p.N, R);
  p.units = static_cast<int32_t>(units);
  const int grid = static_cast<int>(units < sms ? units : sms);
  return launch_int8(kernel, "8-bit linear (few tokens) launch", grid, 32 * warps, shared, 1, stream, p);
}

// Channels of a unit of the few-token kernel: the most (4, 2, 1) that leave an
// SM 12 units, so that enough warps have rows in flight.  One token, us for 1,
// 2, 4: N = 12288, K = 4608: 19.5, 13.9, 12.8; N = 4096, K = 4096: 8.4, 6.8,
// 7.1; N = 512, K = 4096: 4.3, 4.9, 6.2.
int int8_few_channels(int64_t N, int sms) {
  return N >= int64_t(48) * sms ? 4 : N >= int64_t(24) * sms ? 2 : 1;
}

template <bool kBf16, int MT>
int launch_int8_few_tokens(const Int8FewParams& p, int channels, int sms, cudaStream_t stream) {
  if (channels == 1) return launch_int8_few<kBf16, MT, 1>(p, sms, stream);
  if (MT == 4 || channels == 2) return launch_int8_few<kBf16, MT, 2>(p, sms, stream);
  if constexpr (MT < 4) return launch_int8_few<kBf16, MT, 4>(p, sms, stream);
  return FMM_OK;
}

// Dot products for one or two tokens, and for three and four where the unit
// has fewer than four channels (N = 4096, K = 4096, four tokens: 8.8 us, 9.6 on
// the tensor cores; N = 12288, K = 4608: 16.7, 14.2); beyond that tensor cores,
// by the estimates above.
template <bool kBf16>
int launch_linear_int8(const int8_t* codes, int64_t ldq, const int8_t* weight_codes, int64_t ldw,
                       Int8LinearParams p, cudaStream_t stream) {
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  const int sms = usable_sms(info);
  p.group_m = 16;
  p.timeout_ns = g_timeout_ns;
  if (ceil_div(p.M, 16) * ceil_div(p.N, 64) > (int64_t(1) << 30))
    return fail(FMM_ERR_TOO_LARGE, "too many tiles");
  const int channels = int8_few_channels(p.N, sms);
  if ((p.M <= 2 || (p.M <= 4 && channels < 4)) && int8_few_fits(p.M, p.K)) {
    Int8FewParams f = {};
    f.codes = codes;
    f.weight = weight_codes;
    f.ldq = ldq;
    f.ldw = ldw;
    f.ldc = p.ldc;
    f.N = p.N;
    f.token_scales = p.token_scales;
    f.channel_scales = p.channel_scales;
    f.bias = p.bias;
    f.out = p.out;
    f.M = static_cast<int32_t>(p.M);
    f.K = static_cast<int32_t>(p.K);
    f.timeout_ns = g_timeout_ns;
    if (p.M == 1) return launch_int8_few_tokens<kBf16, 1>(f, channels, sms, stream);
    if (p.M == 2) return launch_int8_few_tokens<kBf16, 2>(f, channels, sms, stream);
    return launch_int8_few_tokens<kBf16, 4>(f, channels, sms, stream);
  }
  // a box store ends at a whole 16 bytes of a row: a row that ends inside them
  // would take up to 7 of the elements behind it along
  const bool rows16 = aligned(p.out, 16) && p.ldc % 8 == 0 && p.N % 8 == 0;
  const Int8Shape shape = choose_int8_shape(p.M, p.K, p.N, rows16, sms);
  if (shape.pair) return launch_int8_pair<kBf16>(codes, ldq, weight_codes, ldw, p, sms, stream);
  return shape.tokens ? launch_int8_single<kBf16, true>(codes, ldq, weight_codes, ldw, p, shape, sms, stream)
                      : launch_int8_single<kBf16, false>(codes, ldq, weight_codes, ldw, p, shape, sms, stream);
}

// Device address of g_noalloc_scratch on the current device.  In host code the
// array's name is only a host-side stand-in, so the address is looked up once
// per device (with that device current) and cached.
int noalloc_scratch(void** out) {
  DeviceInfo* info = nullptr;
  if (int rc = device_info(&info)) return rc;
  std::lock_guard<std::mutex> lock(g_device_mutex);
  if (info->noalloc_scratch == nullptr) {
    void* address = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&address, g_noalloc_scratch);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress(no-alloc scratch)");
    info->noalloc_scratch = address;
  }
  *out = info->noalloc_scratch;
  return FMM_OK;
}

__global__ void bounded_wait_probe_kernel(uint64_t timeout_ns) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    // nothing ever arrives: the wait must give up after timeout_ns
    mbar_wait_bounded(smem_u32(&bar), 0, &abort_flag, timeout_ns, 7);
  }
  __syncthreads();
}

}  // namespace
}  // namespace fmm

using namespace fmm;

extern "C" {

int fmm_version(void) { return 100; }

const char* fmm_last_error_string(void) { return t_last_error.c_str(); }

int fmm_plan_dims(int scheme, int64_t M, int64_t K, int64_t N, fmm_dims* out) {
  if (out == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null output");
  return dims_for(scheme, M, K, N, out);
}

int fmm_transform_a(int scheme, int dtype, const void* A, int64_t M, int64_t K, int64_t lda,
                    void* L, fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, M, K, 1, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (A == nullptr || L == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (lda < K) return fail(FMM_ERR_INVALID_ARGUMENT, "lda < K");
  if (!aligned(L, 16)) return fail(FMM_ERR_MISALIGNED, "L must be 16-byte aligned");
  return dispatch<LeftOp>(scheme, dtype, A, M, K, lda, L, &d, reinterpret_cast<cudaStream_t>(stream));
}

int fmm_transform_w(int scheme, int dtype, const void* W, int64_t N, int64_t K, int64_t ldw,
                    void* Rt, fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, 1, K, N, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (W == nullptr || Rt == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldw < K) return fail(FMM_ERR_INVALID_ARGUMENT, "ldw < K");
  if (!aligned(Rt, 16)) return fail(FMM_ERR_MISALIGNED, "Rt must be 16-byte aligned");
  return dispatch<WeightOp>(scheme, dtype, W, N, K, ldw, Rt, &d, reinterpret_cast<cudaStream_t>(stream));
}

int fmm_transform_aw(int scheme, int dtype, const void* A, int64_t M, int64_t K, int64_t lda,
                     void* L, const void* W, int64_t N, int64_t ldw, void* Rt, fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, M, K, N, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (A == nullptr || L == nullptr || W == nullptr || Rt == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (lda < K || ldw < K) return fail(FMM_ERR_INVALID_ARGUMENT, "lda or ldw < K");
  if (!aligned(L, 16) || !aligned(Rt, 16))
    return fail(FMM_ERR_MISALIGNED, "L and Rt must be 16-byte aligned");
  return dispatch<PairedOp>(scheme, dtype, A, M, K, lda, L, W, N, ldw, Rt, &d,
                            reinterpret_cast<cudaStream_t>(stream));
}

int fmm_transform_b(int scheme, int dtype, const void* B, int64_t K, int64_t N, int64_t ldb,
                    void* Rt, fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, 1, K, N, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (B == nullptr || Rt == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldb < N) return fail(FMM_ERR_INVALID_ARGUMENT, "ldb < N");
  if (!aligned(Rt, 16)) return fail(FMM_ERR_MISALIGNED, "Rt must be 16-byte aligned");
  return dispatch<RightKnOp>(scheme, dtype, B, K, N, ldb, Rt, &d, reinterpret_cast<cudaStream_t>(stream));
}

int fmm_leaf_gemm(int rank, const void* L, const void* Rt, int64_t bm, int64_t bn, int64_t bk,
                  void* P, fmm_stream_t stream) {
  if (L == nullptr || Rt == nullptr || P == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  return launch_leaf_gemm<false>(rank, L, Rt, bm, bn, bk, P, reinterpret_cast<cudaStream_t>(stream));
}

int fmm_leaf_gemm_bf16(int rank, const void* L, const void* Rt, int64_t bm, int64_t bn, int64_t bk,
                       void* P, fmm_stream_t stream) {
  if (L == nullptr || Rt == nullptr || P == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  return launch_leaf_gemm<true>(rank, L, Rt, bm, bn, bk, P, reinterpret_cast<cudaStream_t>(stream));
}

int fmm_reconstruct(int scheme, int dtype, const void* P, int64_t M, int64_t N, const void* bias,
                    void* C, int64_t ldc, fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, M, 1, N, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (P == nullptr || C == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldc < N) return fail(FMM_ERR_INVALID_ARGUMENT, "ldc < N");
  if (!aligned(P, 16)) return fail(FMM_ERR_MISALIGNED, "P must be 16-byte aligned");
  return dispatch<ReconstructOp>(scheme, dtype, P, &d, M, N, bias, C, ldc,
                                 reinterpret_cast<cudaStream_t>(stream));
}

int fmm_reconstruct_gather(int scheme, int dtype, const void* P, int64_t M, int64_t N,
                           const void* bias, void* const* dests, int ndest, int64_t ldc,
                           fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, M, 1, N, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (P == nullptr || dests == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (ndest < 1 || ndest > kMaxGatherDests)
    return fail(FMM_ERR_INVALID_ARGUMENT, "ndest must be in [1, 8]");
  if (ldc < N) return fail(FMM_ERR_INVALID_ARGUMENT, "ldc < N");
  if (!aligned(P, 16)) return fail(FMM_ERR_MISALIGNED, "P must be 16-byte aligned");
  GatherDests list = {};
  list.n = ndest;
  for (int k = 0; k < ndest; ++k) {
    if (dests[k] == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null destination");
    list.p[k] = static_cast<uint16_t*>(dests[k]);
  }
  return dispatch<ReconstructGatherOp>(scheme, dtype, P, &d, M, N, bias, &list, ldc,
                                       reinterpret_cast<cudaStream_t>(stream));
}

int fmm_linear(int scheme, int dtype, const void* A, const void* W, const void* bias, void* C,
               int64_t M, int64_t K, int64_t N, void* L, void* Rt, void* P, unsigned int flags,
               fmm_stream_t stream) {
  fmm_dims d;
  if (int rc = dims_for(scheme, M, K, N, &d)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (A == nullptr || C == nullptr || L == nullptr || Rt == nullptr || P == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  const bool prepacked = (flags & FMM_LINEAR_PREPACKED) != 0;
  if (!prepacked && W == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null weight");
  if (!prepacked && !(flags & FMM_RIGHT_KN)) {
    // native [N, K] weight: both input-side transforms in one launch
    if (int rc = fmm_transform_aw(scheme, dtype, A, M, K, K, L, W, N, K, Rt, stream)) return rc;
  } else {
    if (int rc = fmm_transform_a(scheme, dtype, A, M, K, K, L, stream)) return rc;
    if (!prepacked) {
      if (int rc = fmm_transform_b(scheme, dtype, W, K, N, N, Rt, stream)) return rc;
    }
  }
  const int gemm = dtype == FMM_DTYPE_BF16_BF16
                       ? fmm_leaf_gemm_bf16(static_cast<int>(d.rank), L, Rt, d.bm, d.bn, d.bk, P, stream)
                       : fmm_leaf_gemm(static_cast<int>(d.rank), L, Rt, d.bm, d.bn, d.bk, P, stream);
  if (gemm != FMM_OK) return gemm;
  return fmm_reconstruct(scheme, dtype, P, M, N, bias, C, N, stream);
}

int fmm_linear_noalloc(int scheme, const void* A, const void* W, const void* bias, void* C,
                       int64_t M, int64_t K, int64_t N, fmm_stream_t stream) {
  // BF16 linears only: rank 343 takes FP16 operands, so it has no BF16 form to run here
  if (scheme != FMM_SCHEME_RANK7 && scheme != FMM_SCHEME_RANK48 && scheme != FMM_SCHEME_RANK49)
    return fail(FMM_ERR_UNSUPPORTED, "fmm_linear_noalloc: scheme " + std::to_string(scheme) +
                                         " is not a BF16 linear scheme (7, 48 or 49)");
  fmm_dims d;
  if (int rc = dims_for(scheme, M, K, N, &d)) return rc;
  if (A == nullptr || W == nullptr || C == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t left = round_up(d.left_elements * 2, 256);
  const int64_t right = round_up(d.right_elements * 2, 256);
  const int64_t products = round_up(d.product_elements * 2, 256);
  const int64_t needed = left + right + products;
  if (needed > static_cast<int64_t>(FMM_NOALLOC_SCRATCH_BYTES))
    return fail(FMM_ERR_TOO_LARGE,
                "fmm_linear_noalloc: this shape needs " + std::to_string(needed) +
                    " bytes of scratch, more than its fixed " +
                    std::to_string(static_cast<long long>(FMM_NOALLOC_SCRATCH_BYTES)) +
                    "; use fmm_linear with caller-provided planes");
  void* base = nullptr;
  if (int rc = noalloc_scratch(&base)) return rc;
  unsigned char* bytes = static_cast<unsigned char*>(base);
  // Every plane element the GEMM and the reconstruct read is written earlier
  // in the same call (pitch padding included), so nothing is cleared first.
  return fmm_linear(scheme, FMM_DTYPE_BF16, A, W, bias, C, M, K, N, bytes, bytes + left,
                    bytes + left + right, 0u, stream);
}

// ------------------------------------------------------------------ 8-bit integer linear
int fmm_quantize_rows(int dtype, const void* X, int64_t rows, int64_t cols, int64_t ldx, int8_t* codes,
                      int64_t ldq, float* scales, fmm_stream_t stream) {
  if (dtype != FMM_DTYPE_BF16 && dtype != FMM_DTYPE_F16 && dtype != FMM_DTYPE_F32)
    return fail(FMM_ERR_UNSUPPORTED, "dtype must be FMM_DTYPE_BF16, FMM_DTYPE_F16 or FMM_DTYPE_F32");
  if (int rc = check_rows(rows, cols)) return rc;
  if (rows > 0 && (X == nullptr || codes == nullptr || scales == nullptr))
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (ldx < cols || ldq < cols) return fail(FMM_ERR_INVALID_ARGUMENT, "ldx or ldq < cols");
  if (!aligned(X, dtype == FMM_DTYPE_F32 ? 4 : 2) || !aligned(scales, 4))
    return fail(FMM_ERR_MISALIGNED, "X and scales must be aligned to their elements");
  Int8RowsParams p = {};
  p.x = X;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.ldx = ldx;
  p.ldq = ldq;
  p.cols = static_cast<int32_t>(cols);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FMM_DTYPE_F32) return run_int8_rows<float, float, false>(p, s);
  if (dtype == FMM_DTYPE_F16) return run_int8_rows<__half, __half, false>(p, s);
  return run_int8_rows<__nv_bfloat16, __nv_bfloat16, false>(p, s);
}

int fmm_rms_norm_int8(int dtype, int gain_dtype, const void* X, int64_t ldx, const void* residual, int64_t ldr,
                      const void* gain, int64_t rows, int64_t cols, float eps, void* residual_out, int64_t ldo,
                      int8_t* codes, int64_t ldq, float* scales, fmm_stream_t stream) {
  if (dtype != FMM_DTYPE_BF16 && dtype != FMM_DTYPE_F16)
    return fail(FMM_ERR_UNSUPPORTED, "dtype must be FMM_DTYPE_BF16 or FMM_DTYPE_F16");
  if (gain_dtype != dtype && gain_dtype != FMM_DTYPE_F32)
    return fail(FMM_ERR_UNSUPPORTED, "the gain has the dtype of X or FMM_DTYPE_F32");
  if (int rc = check_rows(rows, cols)) return rc;
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(FMM_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  if (rows > 0 && (X == nullptr || gain == nullptr || codes == nullptr || scales == nullptr))
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (residual != nullptr && residual_out == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "a residual needs residual_out");
  if (ldx < cols || ldq < cols || (residual != nullptr && (ldr < cols || ldo < cols)))
    return fail(FMM_ERR_INVALID_ARGUMENT, "a leading dimension is less than cols");
  if (!aligned(X, 2) || !aligned(residual, 2) || !aligned(residual_out, 2) || !aligned(scales, 4) ||
      !aligned(gain, gain_dtype == FMM_DTYPE_F32 ? 4 : 2))
    return fail(FMM_ERR_MISALIGNED, "operands must be aligned to their elements");
  Int8RowsParams p = {};
  p.x = X;
  p.residual = residual;
  p.residual_out = residual != nullptr ? residual_out : nullptr;
  p.gain = gain;
  p.codes = codes;
  p.scales = scales;
  p.rows = rows;
  p.ldx = ldx;
  p.ldr = ldr;
  p.ldo = ldo;
  p.ldq = ldq;
  p.cols = static_cast<int32_t>(cols);
  p.eps = eps;
  p.eps_sum = eps * static_cast<float>(cols);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (gain_dtype == FMM_DTYPE_F32)
    return dtype == FMM_DTYPE_F16 ? run_int8_rows<__half, float, true>(p, s)
                                  : run_int8_rows<__nv_bfloat16, float, true>(p, s);
  return dtype == FMM_DTYPE_F16 ? run_int8_rows<__half, __half, true>(p, s)
                                : run_int8_rows<__nv_bfloat16, __nv_bfloat16, true>(p, s);
}

int fmm_linear_int8(int dtype, const int8_t* codes, int64_t ldq, const float* scales,
                    const int8_t* weight_codes, int64_t ldw, const float* weight_scales, const void* bias,
                    void* C, int64_t ldc, int64_t M, int64_t K, int64_t N, fmm_stream_t stream) {
  if (dtype != FMM_DTYPE_BF16 && dtype != FMM_DTYPE_F16)
    return fail(FMM_ERR_UNSUPPORTED, "dtype must be FMM_DTYPE_BF16 or FMM_DTYPE_F16");
  if (M < 0 || K < 1 || N < 1)
    return fail(FMM_ERR_INVALID_ARGUMENT, "M must not be negative, K and N positive");
  if (K > 131071) return fail(FMM_ERR_TOO_LARGE, "K beyond 131071 could leave the 32-bit sum");
  if (M > (int64_t(1) << 30) || N > (int64_t(1) << 30)) return fail(FMM_ERR_TOO_LARGE, "M or N beyond 2^30");
  if (ldq < K || ldw < K || ldc < N) return fail(FMM_ERR_INVALID_ARGUMENT, "a leading dimension is too small");
  if (M == 0) return FMM_OK;
  if (codes == nullptr || scales == nullptr || weight_codes == nullptr || weight_scales == nullptr || C == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (!aligned(codes, 16) || !aligned(weight_codes, 16) || ldq % 16 != 0 || ldw % 16 != 0)
    return fail(FMM_ERR_MISALIGNED, "code rows must start on 16-byte boundaries");
  if (!aligned(scales, 4) || !aligned(weight_scales, 4) || !aligned(bias, 2) || !aligned(C, 2))
    return fail(FMM_ERR_MISALIGNED, "operands must be aligned to their elements");
  Int8LinearParams p = {};
  p.M = M;
  p.N = N;
  p.K = K;
  p.ldc = ldc;
  p.token_scales = scales;
  p.channel_scales = weight_scales;
  p.bias = bias;
  p.out = C;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == FMM_DTYPE_BF16 ? launch_linear_int8<true>(codes, ldq, weight_codes, ldw, p, s)
                                 : launch_linear_int8<false>(codes, ldq, weight_codes, ldw, p, s);
}

// ------------------------------------------------------------------ peer memory (IPC)
static_assert(sizeof(cudaIpcMemHandle_t) == FMM_IPC_HANDLE_BYTES, "IPC handle size");

int fmm_ipc_export(const void* ptr, unsigned char* handle, uint64_t* offset) {
  if (ptr == nullptr || handle == nullptr || offset == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  static PFN_cuMemGetAddressRange_v3020 range = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuMemGetAddressRange", &fn, 3020, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      range = reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(fn);
  });
  if (range == nullptr) return fail(FMM_ERR_CUDA, "cuMemGetAddressRange is unavailable");
  CUdeviceptr base = 0;
  size_t size = 0;
  if (range(&base, &size, reinterpret_cast<CUdeviceptr>(ptr)) != CUDA_SUCCESS)
    return fail(FMM_ERR_INVALID_ARGUMENT, "pointer is not device memory of this context");
  cudaIpcMemHandle_t h;
  cudaError_t e = cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base));
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcGetMemHandle");
  std::memcpy(handle, &h, sizeof(h));
  *offset = static_cast<uint64_t>(reinterpret_cast<CUdeviceptr>(ptr) - base);
  return FMM_OK;
}

int fmm_ipc_import(const unsigned char* handle, uint64_t offset, void** base, void** ptr) {
  if (handle == nullptr || base == nullptr || ptr == nullptr)
    return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  cudaIpcMemHandle_t h;
  std::memcpy(&h, handle, sizeof(h));
  void* mapped = nullptr;
  cudaError_t e = cudaIpcOpenMemHandle(&mapped, h, cudaIpcMemLazyEnablePeerAccess);
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcOpenMemHandle");
  *base = mapped;
  *ptr = static_cast<unsigned char*>(mapped) + offset;
  return FMM_OK;
}

int fmm_ipc_close(void* base) {
  if (base == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  cudaError_t e = cudaIpcCloseMemHandle(base);
  if (e != cudaSuccess) return cuda_fail(e, "cudaIpcCloseMemHandle");
  return FMM_OK;
}

int fmm_copy_async(void* dst, const void* src, uint64_t bytes, fmm_stream_t stream) {
  if (dst == nullptr || src == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null pointer");
  if (bytes == 0) return FMM_OK;
  cudaError_t e = cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToDevice,
                                  reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyAsync (device to device)");
  return FMM_OK;
}

int fmm_set_sm_budget(int sms) {
  if (sms < 0) return fail(FMM_ERR_INVALID_ARGUMENT, "SM budget must be >= 0");
  g_sm_budget = sms;
  return FMM_OK;
}

int fmm_set_wait_timeout_ns(uint64_t timeout_ns) {
  if (timeout_ns == 0) return fail(FMM_ERR_INVALID_ARGUMENT, "timeout must be positive");
  g_timeout_ns = timeout_ns;
  return FMM_OK;
}

int fmm_device_status(int device, uint32_t* status, uint32_t* site, int reset) {
  if (status == nullptr) return fail(FMM_ERR_INVALID_ARGUMENT, "null status");
  int previous = 0;
  cudaError_t e = cudaGetDevice(&previous);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (device != previous && (e = cudaSetDevice(device)) != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
  int rc = FMM_OK;
  unsigned int value = 0, where = 0;
  if ((e = cudaDeviceSynchronize()) != cudaSuccess) rc = cuda_fail(e, "cudaDeviceSynchronize");
  if (rc == FMM_OK && (e = cudaMemcpyFromSymbol(&value, g_status, sizeof(value))) != cudaSuccess)
    rc = cuda_fail(e, "read status");
  if (rc == FMM_OK && (e = cudaMemcpyFromSymbol(&where, g_timeout_site, sizeof(where))) != cudaSuccess)
    rc = cuda_fail(e, "read timeout site");
  if (rc == FMM_OK && reset) {
    const unsigned int zero = 0;
    if ((e = cudaMemcpyToSymbol(g_status, &zero, sizeof(zero))) != cudaSuccess ||
        (e = cudaMemcpyToSymbol(g_timeout_site, &zero, sizeof(zero))) != cudaSuccess)
      rc = cuda_fail(e, "clear status");
  }
  if (device != previous) cudaSetDevice(previous);
  *status = value;
  if (site != nullptr) *site = where;
  return rc;
}

int fmm_test_bounded_wait(uint64_t timeout_ns, fmm_stream_t stream) {
  if (timeout_ns == 0 || timeout_ns > 10000000000ull)
    return fail(FMM_ERR_INVALID_ARGUMENT, "probe timeout must be in (0, 10 s]");
  bounded_wait_probe_kernel<<<1, 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(timeout_ns);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "bounded wait probe launch");
  return FMM_OK;
}

}  // extern "C"
