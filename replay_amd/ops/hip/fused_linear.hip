// y = act(x W^T + bias) + residual and its gradients (gfx950).
//
//   z = x W^T + bias      y = act(z) + residual
//   dz = dy act'(z)       dx = dz W      dW = dz^T x      db = sum_rows dz
//
// Three products over one tile kernel: their operands differ only in which
// index is contiguous in memory, and in where the contraction runs (over the
// rows, M, for dW: it is split over workgroups and joined in a fixed order).
// z is kept for the backward pass in the input's type, rounded once: act' is
// as exact as the gradient's own rounding needs.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if (act == ACT_SILU) return z / (1.f + expf(-z));
  return z;
}

__device__ __forceinline__ float act_slope(int act, float z) {
  if (act == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == ACT_GELU)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
           z * 0.39894228040143268f * expf(-0.5f * z * z);
  if (act == ACT_SILU) {
    const float s = 1.f / (1.f + expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

struct Gemm {
  const void *a, *b;
  int64_t lda, ldb;
  int M, N;
  int64_t K, k_part;      // contraction, and how much of it one part covers
  // epilogue (one part only)
  const void *bias, *residual;
  int64_t ldr;
  void *y, *z;            // [M, N] contiguous; z or nullptr
  int act;
  float* part;            // [parts, M, N] instead of y
};

// Element (r, k) of an operand: r * ld + k where the contraction is
// contiguous (KM), else k * ld + r.  64 x BK of it into LDS as [r][k].
template <typename T, bool KM, int BK, int LDK>
__device__ __forceinline__ void stage(T* dst, const T* src, int64_t ld, int r0, int R, int64_t k0,
                                      int64_t k_end) {
  for (int i = threadIdx.x; i < 64 * BK; i += 256) {
    const int r = KM ? i / BK : i % 64, k = KM ? i % BK : i / 64;
    T v = from_f32<T>(0.f);
    if (r0 + r < R && k0 + k < k_end) v = src[KM ? (r0 + r) * ld + k0 + k : (k0 + k) * ld + r0 + r];
    dst[r * LDK + k] = v;
  }
}

template <typename T>
struct Tile;  // one 16 x 16 product step of depth DEPTH from LDS rows
template <>
struct Tile<float> {
  static constexpr int DEPTH = 4;
  static __device__ __forceinline__ f32x4 step(const float* a, const float* b, int g, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a[g], b[g], c, 0, 0, 0);
  }
};
template <>
struct Tile<__hip_bfloat16> {
  static constexpr int DEPTH = 32;
  static __device__ __forceinline__ f32x4 step(const __hip_bfloat16* a, const __hip_bfloat16* b,
                                               int g, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(a + 8 * g),
                                                   *reinterpret_cast<const bf16x8*>(b + 8 * g), c, 0,
                                                   0, 0);
  }
};
template <>
struct Tile<__half> {
  static constexpr int DEPTH = 32;
  static __device__ __forceinline__ f32x4 step(const __half* a, const __half* b, int g, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const f16x8*>(a + 8 * g),
                                                  *reinterpret_cast<const f16x8*>(b + 8 * g), c, 0,
                                                  0, 0);
  }
};

// 64 x 64 tile, 4 waves of 32 x 32.
template <typename T, bool A_KM, bool B_KM>
__global__ __launch_bounds__(256) void gemm64(Gemm p) {
  constexpr int BK = 32, LDK = BK + 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) T a_s[64 * LDK];
  __shared__ __attribute__((aligned(16))) T b_s[64 * LDK];
  const int tiles_n = (p.N + 63) / 64;
  const int m0 = (blockIdx.x / tiles_n) * 64, n0 = (blockIdx.x % tiles_n) * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lo = lane & 15, g = lane >> 4;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const int64_t k_begin = blockIdx.y * p.k_part, k_end = min(p.K, k_begin + p.k_part);
  f32x4 acc[2][2] = {};
  for (int64_t k0 = k_begin; k0 < k_end; k0 += BK) {
    __syncthreads();
    stage<T, A_KM, BK, LDK>(a_s, reinterpret_cast<const T*>(p.a), p.lda, m0, p.M, k0, k_end);
    stage<T, B_KM, BK, LDK>(b_s, reinterpret_cast<const T*>(p.b), p.ldb, n0, p.N, k0, k_end);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < BK; s += Tile<T>::DEPTH) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = Tile<T>::step(a_s + (wm + 16 * i + lo) * LDK + s,
                                    b_s + (wn + 16 * j + lo) * LDK + s, g, acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + wn + 16 * j + lo;
      if (n >= p.N) continue;
      const float bias = p.bias ? to_f32<T>(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + wm + 16 * i + 4 * g + r;
        if (m >= p.M) continue;
        const int64_t at = (int64_t)m * p.N + n;
        if (p.part) {
          p.part[(int64_t)blockIdx.y * p.M * p.N + at] = acc[i][j][r];
          continue;
        }
        const float z = acc[i][j][r] + bias;
        float y = act_of(p.act, z);
        if (p.z) reinterpret_cast<T*>(p.z)[at] = from_f32<T>(z);
        if (p.residual) y += to_f32<T>(reinterpret_cast<const T*>(p.residual)[m * p.ldr + n]);
        reinterpret_cast<T*>(p.y)[at] = from_f32<T>(y);
      }
    }
  }
}

// out[i] = sum over parts, in order
template <typename T>
__global__ void join_parts(const float* part, T* out, int64_t size, int parts) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < size;
       i += (int64_t)gridDim.x * blockDim.x) {
    float sum = 0.f;
    for (int s = 0; s < parts; ++s) sum += part[s * size + i];
    out[i] = from_f32<T>(sum);
  }
}

template <typename T>
__global__ void slope_product(const T* dy, int64_t ldy, const T* z, T* dz, int64_t M, int N, int act) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < M * N;
       i += (int64_t)gridDim.x * blockDim.x) {
    const float d = to_f32<T>(dy[(i / N) * ldy + i % N]);
    dz[i] = from_f32<T>(d * act_slope(act, to_f32<T>(z[i])));
  }
}

// part[y][n] = sum of rows [y * rows, ...) of column n
template <typename T>
__global__ void column_sums(const T* dz, int64_t ld, float* part, int64_t M, int N, int64_t rows) {
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= N) return;
  float sum = 0.f;
  const int64_t end = min(M, (blockIdx.y + 1) * rows);
  for (int64_t m = blockIdx.y * rows; m < end; ++m) sum += to_f32<T>(dz[m * ld + n]);
  part[(int64_t)blockIdx.y * N + n] = sum;
}

template <typename T, bool A_KM, bool B_KM>
void launch_gemm(const Gemm& p, int parts, hipStream_t stream) {
  const int64_t tiles = (int64_t)((p.M + 63) / 64) * ((p.N + 63) / 64);
  TORCH_CHECK(tiles < (int64_t(1) << 31), "fused_linear: too many tiles");
  if (tiles == 0) return;
  hipLaunchKernelGGL((gemm64<T, A_KM, B_KM>), dim3((unsigned)tiles, parts), dim3(256), 0, stream, p);
  HIP_CHECK(hipGetLastError());
}

unsigned flat_blocks(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, 16384); }

void check_rows(const torch::Tensor& t, const torch::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device() && t.scalar_type() == x.scalar_type(), "fused_linear: ", name,
              " must share type and device with x");
  TORCH_CHECK(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), "fused_linear: ", name,
              " needs two dimensions, the last contiguous");
  TORCH_CHECK(t.size(0) < (int64_t(1) << 31) - 256 && t.size(1) < (int64_t(1) << 31) - 256,
              "fused_linear: ", name, " is too large");
}

void check_x(const torch::Tensor& x, const torch::Tensor& weight) {
  const auto dt = x.scalar_type();
  TORCH_CHECK(x.is_cuda(), "fused_linear: x must be on the GPU");
  TORCH_CHECK(dt == torch::kBFloat16 || dt == torch::kHalf || dt == torch::kFloat32,
              "fused_linear: x must be bfloat16, float16 or float32");
  check_rows(x, x, "x");
  check_rows(weight, x, "weight");
  TORCH_CHECK(weight.size(1) == x.size(1), "fused_linear: x and weight differ in their last dimension");
}

template <typename T>
void forward_t(const torch::Tensor& x, const torch::Tensor& w, Gemm p, hipStream_t stream) {
  p.a = x.data_ptr();
  p.lda = x.stride(0);
  p.b = w.data_ptr();
  p.ldb = w.stride(0);
  p.M = x.size(0);
  p.N = w.size(0);
  p.K = p.k_part = x.size(1);
  launch_gemm<T, true, true>(p, 1, stream);
}

template <typename T>
void backward_t(const torch::Tensor& dz, const torch::Tensor& x, const torch::Tensor& w,
                torch::Tensor& dx, torch::Tensor& dw, torch::Tensor& db, hipStream_t stream) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  auto f32 = x.options().dtype(torch::kFloat32);
  if (dx.defined()) {
    Gemm p = {};
    p.a = dz.data_ptr();
    p.lda = dz.stride(0);
    p.b = w.data_ptr();
    p.ldb = w.stride(0);
    p.M = M;
    p.N = K;
    p.K = p.k_part = N;
    p.y = dx.data_ptr();
    launch_gemm<T, true, false>(p, 1, stream);
  }
  if (dw.defined()) {
    Gemm p = {};
    p.a = dz.data_ptr();
    p.lda = dz.stride(0);
    p.b = x.data_ptr();
    p.ldb = x.stride(0);
    p.M = N;
    p.N = K;
    p.K = M;
    const int64_t tiles = ((N + 63) / 64) * ((K + 63) / 64);
    int64_t parts = std::max<int64_t>(1, std::min<int64_t>(1024 / std::max<int64_t>(tiles, 1), M / 256));
    p.k_part = std::max<int64_t>(32, ((M + parts - 1) / parts + 31) / 32 * 32);
    parts = std::max<int64_t>(1, (M + p.k_part - 1) / p.k_part);
    auto part = torch::empty({parts, N, K}, f32);
    p.part = part.data_ptr<float>();
    launch_gemm<T, false, false>(p, (int)parts, stream);
    if (N * K) {
      hipLaunchKernelGGL((join_parts<T>), dim3(flat_blocks(N * K)), dim3(256), 0, stream, p.part,
                         reinterpret_cast<T*>(dw.data_ptr()), N * K, (int)parts);
      HIP_CHECK(hipGetLastError());
    }
  }
  if (db.defined() && N) {
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(256, M / 64));
    const int64_t rows = (M + parts - 1) / parts;
    auto part = torch::empty({parts, N}, f32);
    hipLaunchKernelGGL((column_sums<T>), dim3((unsigned)((N + 255) / 256), (unsigned)parts), dim3(256),
                       0, stream, reinterpret_cast<const T*>(dz.data_ptr()), dz.stride(0),
                       part.data_ptr<float>(), M, (int)N, rows);
    HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((join_parts<T>), dim3(flat_blocks(N)), dim3(256), 0, stream,
                       part.data_ptr<float>(), reinterpret_cast<T*>(db.data_ptr()), N, (int)parts);
    HIP_CHECK(hipGetLastError());
  }
}

}  // namespace

// -> {y, z or empty}
std::vector<torch::Tensor> fused_linear_fwd(torch::Tensor x, torch::Tensor weight,
                                            c10::optional<torch::Tensor> bias,
                                            c10::optional<torch::Tensor> residual, int64_t act,
                                            bool want_z) {
  check_x(x, weight);
  const int64_t M = x.size(0), N = weight.size(0);
  TORCH_CHECK(act >= 0 && act <= 3, "fused_linear: unknown activation");
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == x.device() && bias->scalar_type() == x.scalar_type() &&
                    bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous(),
                "fused_linear: bias must be [N], of x's type and device");
  }
  if (residual.has_value()) {
    check_rows(*residual, x, "residual");
    TORCH_CHECK(residual->size(0) == M && residual->size(1) == N, "fused_linear: residual must be [M, N]");
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto stream = at::cuda::getCurrentHIPStream();
  auto y = torch::empty({M, N}, x.options());
  auto z = torch::empty({want_z ? M : 0, N}, x.options());
  Gemm p = {};
  p.bias = bias.has_value() ? bias->data_ptr() : nullptr;
  p.residual = residual.has_value() ? residual->data_ptr() : nullptr;
  p.ldr = residual.has_value() ? residual->stride(0) : 0;
  p.y = y.data_ptr();
  p.z = want_z ? z.data_ptr() : nullptr;
  p.act = (int)act;
  if (x.scalar_type() == torch::kBFloat16) forward_t<__hip_bfloat16>(x, weight, p, stream);
  else if (x.scalar_type() == torch::kHalf) forward_t<__half>(x, weight, p, stream);
  else forward_t<float>(x, weight, p, stream);
  return {y, z};
}

// -> {dx, dw, db}, empty where not needed.  z: what the slope is taken at
// (for relu the output serves as well); unused without an activation.
std::vector<torch::Tensor> fused_linear_bwd(torch::Tensor dy, torch::Tensor x, torch::Tensor weight,
                                            torch::Tensor z, int64_t act, bool need_x, bool need_w,
                                            bool need_b) {
  check_x(x, weight);
  check_rows(dy, x, "dy");
  const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
  TORCH_CHECK(act >= 0 && act <= 3, "fused_linear: unknown activation");
  TORCH_CHECK(dy.size(0) == M && dy.size(1) == N, "fused_linear: dy must be [M, N]");
  TORCH_CHECK(act == ACT_NONE || (z.is_contiguous() && z.dim() == 2 && z.size(0) == M &&
                                  z.size(1) == N && z.scalar_type() == x.scalar_type() &&
                                  z.device() == x.device()),
              "fused_linear: z must be [M, N], of x's type and device");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto stream = at::cuda::getCurrentHIPStream();
  torch::Tensor dx, dw, db, dz = dy;
  if (need_x) dx = torch::empty({M, K}, x.options());
  if (need_w) dw = torch::empty({N, K}, x.options());
  if (need_b) db = torch::empty({N}, x.options());
  if (act != ACT_NONE) dz = torch::empty({M, N}, x.options());
#define FL_BACKWARD(T)                                                                            \
  do {                                                                                            \
    if (act != ACT_NONE && M * N) {                                                               \
      hipLaunchKernelGGL((slope_product<T>), dim3(flat_blocks(M * N)), dim3(256), 0, stream,      \
                         reinterpret_cast<const T*>(dy.data_ptr()), dy.stride(0),                 \
                         reinterpret_cast<const T*>(z.data_ptr()),                                \
                         reinterpret_cast<T*>(dz.data_ptr()), M, (int)N, (int)act);               \
      HIP_CHECK(hipGetLastError());                                                               \
    }                                                                                             \
    backward_t<T>(dz, x, weight, dx, dw, db, stream);                                             \
  } while (0)
  if (x.scalar_type() == torch::kBFloat16) FL_BACKWARD(__hip_bfloat16);
  else if (x.scalar_type() == torch::kHalf) FL_BACKWARD(__half);
  else FL_BACKWARD(float);
#undef FL_BACKWARD
  auto none = torch::empty({0}, x.options());
  return {need_x ? dx : none, need_w ? dw : none, need_b ? db : none};
}
