// y = act(x W^T + bias) + residual and its gradients (gfx950).
//
//   z = x W^T + bias      y = act(z) + residual
//   dz = dy act'(z)       dx = dz W      dW = dz^T x      db = sum_rows dz
//
// Three products over one tile kernel: their operands differ only in which
// index is contiguous in memory, and in where the contraction runs (over the
// rows, M, for dW: it is split over workgroups and joined in a fixed order).
// z is kept for the backward pass in the input's type, rounded once: act' is
// as exact as the gradient's own rounding needs.  dz is rounded to it too, since
// the matrix instructions take it so (db sums it before): gradients of bfloat16
// inputs with gelu are then off by 2.4e-3 of their norm, 1.7e-3 with one rounding.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;

enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// phi(z) sqrt(2 pi) = e^{-z^2/2}, and the normal distribution's Phi(z).
// Phi(-|z|) = erfc(x) / 2 = e^{-x^2} w(x) / 2 with x = |z| / sqrt 2, and w as a
// polynomial in t = 1 / (1 + 0.4 x), fitted to relative error over x >= 0
// (1.3e-7; 5e-7 as evaluated in float).  The tail keeps its relative accuracy,
// and it takes a third of the instructions of erff, whose two branches a wave
// mostly runs both (25601 x 1024 by K 256 with gelu: 50 -> 39 us).
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  const float x = fabsf(z);
  bell = __expf(-0.5f * z * z);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.28284271f * x);
  float w = 0.05027306452393532f;
  w = w * t - 0.18294541537761688f;
  w = w * t + 0.16915756464004517f;
  w = w * t - 0.005669722333550453f;
  w = w * t + 0.1414615660905838f;
  w = w * t + 0.16853384673595428f;
  w = w * t + 0.2078438252210617f;
  w = w * t + 0.22566953301429749f;
  w = w * t + 0.22567586600780487f;
  const float tail = 0.5f * w * t * bell;
  return z < 0.f ? tail : 1.f - tail;
}

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == ACT_GELU) {
    float bell;
    return z * normal_cdf(z, bell);
  }
  if (act == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  return z;
}

__device__ __forceinline__ float act_slope(int act, float z) {
  if (act == ACT_RELU) return z <= 0.f ? 0.f : 1.f;  // a NaN lets the gradient pass, as it passes itself
  if (act == ACT_GELU) {
    float bell;
    const float cdf = normal_cdf(z, bell);
    return cdf + z * 0.39894228040143268f * bell;
  }
  if (act == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
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
  float* row_part;        // [parts, M] sums of A over the contraction, or nullptr
  unsigned tiles;         // of one part
};

__device__ __attribute__((aligned(16))) const unsigned zero_chunk[4] = {0, 0, 0, 0};

// How an operand lies in memory and in LDS.  Element (r, k) is at r * ld + k
// where the contraction is contiguous (KM), else at k * ld + r.  A stage holds
// R rows by BK = 128 bytes of contraction in 16-byte chunks, in the operand's
// own order, with the chunks permuted so that neither the fragment reads nor
// the writes of a wave meet in the same banks:
//   KM:     [r][chunk]   chunk ^ (r >> 1)
//   not KM: [k][unit]    units of 16 rows; permuted by the bits of k in which
//                        the lanes of one fragment read differ
// Fragments are 16 bytes a lane: 8 (4) contraction steps of row (lane & 15).
// Which steps is up to us as long as A and B agree: group g = lane >> 4 holds
// k = 8 g .. 8 g + 7 (16 bits) or 4 g .. 4 g + 3 (float).
template <typename T, bool KM, int R>
struct Operand {
  static constexpr int CH = 16 / sizeof(T), BK = 128 / sizeof(T), BYTES = R * 128;
  static constexpr int ROW = KM ? 128 : R * sizeof(T);  // bytes of a row in LDS
  static constexpr int UNIT = sizeof(T) * 16;           // bytes of 16 rows

  // (bits 2 and 5 of k, 16 bits, and 0, 1 and 4, float, may not count: they
  // are the constants of a lane's reads)
  static __device__ __forceinline__ int unit_mix(int k) {
    if (sizeof(T) == 4) return (k >> 2) & 3;
    if (R == 64) return ((k >> 1) & 1) | (((k >> 3) & 1) << 1);
    return ((k & 3) | (((k >> 3) & 1) << 2)) & (R / 16 - 1);
  }
  // slot (16-byte place in the stage) -> its chunk's row and contraction step
  static __device__ __forceinline__ void source_of(int slot, int& r, int& k) {
    if (KM) {
      r = slot >> 3;
      k = ((slot & 7) ^ ((r >> 1) & 7)) * CH;
    } else {
      constexpr int PER = ROW / 16, SUB = UNIT / 16;
      k = slot / PER;
      const int p = slot % PER;
      r = ((((p / SUB) ^ unit_mix(k)) * SUB) + p % SUB) * CH;
    }
  }
  // A wave's fragments, CNT blocks of 16 rows from row w0 (a multiple of 16 CNT).
  // What differs between lanes is worked out once; the rest of each address is
  // a constant.
  template <int CNT>
  struct Fragments {
    unsigned off[KM ? 2 : CNT];

    __device__ __forceinline__ Fragments(int w0, int lane) {
      const int lo = lane & 15, g = lane >> 4;
      if (KM) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) off[kb & (KM ? 1 : 0)] = (w0 + lo) * 128 + (((kb * 4 + g) ^ ((lo >> 1) & 7)) << 4);
      } else {
        const int k = sizeof(T) == 2 ? 8 * g + (lo >> 2) : 4 * g;
        const int in = sizeof(T) == 2 ? (lo & 3) * 8 : lo * 4;
#pragma unroll
        for (int i = 0; i < CNT; ++i)
          off[i & (KM ? 1 : CNT - 1)] = k * ROW + (((w0 >> 4) + i) ^ unit_mix(k)) * UNIT + in;
      }
    }
    // block i, 64 bytes kb of the contraction
    __device__ __forceinline__ uint4 get(const char* stage, int i, int kb) const {
      if constexpr (KM) {
        return *reinterpret_cast<const uint4*>(stage + off[kb] + i * 2048);
      } else if constexpr (sizeof(T) == 2) {
        uint2 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          auto v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(stage + off[i] + (kb * 32 + 4 * h) * ROW));
          half[h] = __builtin_bit_cast(uint2, v);
        }
        return uint4{half[0].x, half[0].y, half[1].x, half[1].y};
      } else {
        unsigned v[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
          v[s] = *reinterpret_cast<const unsigned*>(stage + off[i] + (kb * 16 + s) * ROW);
        return uint4{v[0], v[1], v[2], v[3]};
      }
    }
  };
  // Bytes from the tile's first element to a slot's chunk; rows past the end
  // repeat the last ones (their results are not stored).  Whole, aligned
  // chunks only, and strides that stay within 32 bits over a tile.
  static __device__ __forceinline__ unsigned offset_of(int slot, int r0, int R_all, int64_t ld) {
    int r, k;
    source_of(slot, r, k);
    const unsigned row = min(r0 + r, KM ? R_all - 1 : R_all - CH) - r0;
    return (KM ? row * (unsigned)ld + k : k * (unsigned)ld + row) * (unsigned)sizeof(T);
  }
  // A chunk of any size and alignment; zero outside.
  static __device__ __forceinline__ uint4 load_chunk(const T* src, int64_t ld, int r, int R_all,
                                                     int64_t k, int64_t k_end) {
    alignas(16) T t[CH];
    const int64_t in = KM ? k_end - k : R_all - r;  // elements of it that exist
    if ((KM ? r < R_all : k < k_end) && in > 0) {
      const T* at = KM ? src + r * ld + k : src + k * ld + r;
      if (in >= CH) {
        __builtin_memcpy(t, at, 16);
      } else {
#pragma unroll
        for (int i = 0; i < CH; ++i) t[i] = i < in ? at[i] : from_f32<T>(0.f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < CH; ++i) t[i] = from_f32<T>(0.f);
    }
    return *reinterpret_cast<const uint4*>(t);
  }
};

template <typename T>
__device__ __forceinline__ f32x4 mfma_block(uint4 a, uint4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma_block<__hip_bfloat16>(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_block<__half>(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_block<float>(uint4 a, uint4 b, f32x4 c) {
  const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s], y[s], c, 0, 0, 0);
  return c;
}

template <typename T>
__device__ __forceinline__ uint4 ones_chunk();
template <>
__device__ __forceinline__ uint4 ones_chunk<__hip_bfloat16>() {
  return uint4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
}
template <>
__device__ __forceinline__ uint4 ones_chunk<__half>() {
  return uint4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
}
template <>
__device__ __forceinline__ uint4 ones_chunk<float>() {
  return uint4{0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u};
}

// V neighbours of a row, of which n exist; no alignment is asked for.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, int n, float* o) {
  alignas(16) T t[V];
  if (n >= V) {
    __builtin_memcpy(t, p, V * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = to_f32<T>(t[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, int n, const float* v) {
  alignas(16) T t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = from_f32<T>(v[i]);
  if (n >= V) {
    __builtin_memcpy(p, t, V * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = t[i];
  }
}

// What becomes of a wave's 16 x WN block of z - bias, which lies in LDS as
// float [16][WN + 4]: whole rows of it are read back, so that memory sees runs
// of full lines.  (Straight from the accumulators, 8 bytes a lane in 16 rows at
// once, the narrow products' stores ran at a third of the card's rate.)
template <typename T, int WN, int ACT>
__device__ __forceinline__ void finish_block(const Gemm& p, const float* block, int lane, int m, int n0,
                                             const float* bias) {
  constexpr int V = 16 / sizeof(T), ACROSS = WN / V, DOWN = 64 / ACROSS;
  const int col = (lane % ACROSS) * V, n = n0 + col, left = p.N - n;
#pragma unroll
  for (int r0 = 0; r0 < 16; r0 += DOWN) {
    const int row = r0 + lane / ACROSS;
    if (m + row >= p.M || left <= 0) continue;
    const int64_t at = (int64_t)(m + row) * p.N + n;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i += 4)
      *reinterpret_cast<f32x4*>(v + i) = *reinterpret_cast<const f32x4*>(block + row * (WN + 4) + col + i);
    if (p.part) {
      store_row<float, V>(p.part + at, left, v);
      continue;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += bias[i];
    if (p.z) store_row<T, V>(reinterpret_cast<T*>(p.z) + at, left, v);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = act_of(ACT, v[i]);
    if (p.residual) {
      float add[V];
      load_row<T, V>(reinterpret_cast<const T*>(p.residual) + (m + row) * p.ldr + n, left, add);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += add[i];
    }
    store_row<T, V>(reinterpret_cast<T*>(p.y) + at, left, v);
  }
}

// BM x BN tile, WM x WN waves.  The products are taken transposed (rows of the
// accumulator run along N), so that a lane holds four neighbours of one output
// row.  DIRECT: chunks go from memory to LDS without registers; else through
// registers, any size and alignment.  Either way a stage ahead of the products
// where there are two (STAGES): two arrays of their own and a loop over pairs,
// since only so can the compiler tell that reading one need not wait for the
// loads into the other.
template <typename T, bool A_KM, bool B_KM, int BM, int BN, int WM, int WN, bool DIRECT, int STAGES>
__global__ __launch_bounds__(WM * WN * 64) void gemm_tile(Gemm p) {
  using A = Operand<T, A_KM, BM>;
  using B = Operand<T, B_KM, BN>;
  constexpr int BK = A::BK, NT = WM * WN * 64;
  constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  constexpr int SA = BM * 8 / NT, SB = BN * 8 / NT, STAGE = A::BYTES + B::BYTES;
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0, "whole chunks for each thread");
  static_assert(WM * WN * 16 * (BN / WN + 4) * 4 <= STAGE, "the waves' output blocks fit in a stage");
  __shared__ __attribute__((aligned(16))) char stage0[STAGE];
  __shared__ __attribute__((aligned(16))) char stage1[STAGES == 2 ? STAGE : 16];

  // Workgroups go round the 8 dies in turn: give each die one run of tiles,
  // ordered in bands of 8 tile rows, so that its own L2 serves the operands; of
  // a contraction in parts, the tiles of one part after the other.
  const unsigned all = gridDim.x, id = blockIdx.x;
  const unsigned die = id & 7, per = all >> 3, more = all & 7;
  const unsigned u = die * per + min(die, more) + (id >> 3);
  const unsigned at_part = u / p.tiles, t = u - at_part * p.tiles;
  p.part += (int64_t)at_part * p.M * p.N;
  const unsigned tn = (p.N + BN - 1) / BN, tm = (p.M + BM - 1) / BM;
  const unsigned band = t / (8 * tn), rows = min(8u, tm - band * 8), in = t - band * 8 * tn;
  const int m0 = (int)(band * 8 + in % rows) * BM, n0 = (int)(in / rows) * BN;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // the same for its lanes
  const int lo = lane & 15, g = lane >> 4;
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  const T* a_src = reinterpret_cast<const T*>(p.a);
  const T* b_src = reinterpret_cast<const T*>(p.b);
  const int64_t k_begin = at_part * p.k_part, k_end = min(p.K, k_begin + p.k_part);
  const int iters = k_end > k_begin ? (int)((k_end - k_begin + BK - 1) / BK) : 0;

  // where this thread's chunks of the first stage lie
  const char* a_base = reinterpret_cast<const char*>(a_src + (A_KM ? m0 * p.lda + k_begin : k_begin * p.lda + m0));
  const char* b_base = reinterpret_cast<const char*>(b_src + (B_KM ? n0 * p.ldb + k_begin : k_begin * p.ldb + n0));
  const int64_t a_step = (A_KM ? 1 : p.lda) * (int64_t)(BK * sizeof(T));
  const int64_t b_step = (B_KM ? 1 : p.ldb) * (int64_t)(BK * sizeof(T));
  unsigned a_off[SA], b_off[SB];
  if constexpr (DIRECT) {
#pragma unroll
    for (int i = 0; i < SA; ++i) a_off[i] = A::offset_of(i * NT + tid, m0, p.M, p.lda);
#pragma unroll
    for (int i = 0; i < SB; ++i) b_off[i] = B::offset_of(i * NT + tid, n0, p.N, p.ldb);
  }
  uint4 ra[DIRECT ? 1 : SA], rb[DIRECT ? 1 : SB];
  auto fetch = [&](int it, char* stage) {
    const int64_t k0 = k_begin + (int64_t)it * BK;
    if constexpr (DIRECT) {
      const char* ab = a_base + it * a_step;
      const char* bb = b_base + it * b_step;
      // the bases stay scalar, so that a load's address is these and one offset
      // register; the compiler would step a pointer of two for each load
      asm volatile("" : "+s"(ab), "+s"(bb));
      const bool whole = k0 + BK <= k_end;  // the same for all
      auto load = [&](const char* src, char* dst) {
        __builtin_amdgcn_global_load_lds((const void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
      };
      char* dst = stage + wave * 1024;
      if (whole) {
#pragma unroll
        for (int i = 0; i < SA; ++i) load(ab + a_off[i], dst + i * NT * 16);
#pragma unroll
        for (int i = 0; i < SB; ++i) load(bb + b_off[i], dst + A::BYTES + i * NT * 16);
      } else {  // chunks past the end of the contraction read as zero
        const int in = (int)(k_end - k0);
        int r, k;
#pragma unroll
        for (int i = 0; i < SA; ++i) {
          A::source_of(i * NT + tid, r, k);
          load(k < in ? ab + a_off[i] : reinterpret_cast<const char*>(zero_chunk), dst + i * NT * 16);
        }
#pragma unroll
        for (int i = 0; i < SB; ++i) {
          B::source_of(i * NT + tid, r, k);
          load(k < in ? bb + b_off[i] : reinterpret_cast<const char*>(zero_chunk), dst + A::BYTES + i * NT * 16);
        }
      }
    } else {
      int r, k;
#pragma unroll
      for (int i = 0; i < SA; ++i) {
        A::source_of(i * NT + tid, r, k);
        ra[i] = A::load_chunk(a_src, p.lda, m0 + r, p.M, k0 + k, k_end);
      }
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        B::source_of(i * NT + tid, r, k);
        rb[i] = B::load_chunk(b_src, p.ldb, n0 + r, p.N, k0 + k, k_end);
      }
    }
  };
  auto put = [&](char* stage) {
    if constexpr (!DIRECT) {
      char* dst = stage + tid * 16;
#pragma unroll
      for (int i = 0; i < SA; ++i) *reinterpret_cast<uint4*>(dst + i * NT * 16) = ra[i];
#pragma unroll
      for (int i = 0; i < SB; ++i) *reinterpret_cast<uint4*>(dst + A::BYTES + i * NT * 16) = rb[i];
    }
  };

  f32x4 acc[MI][NI] = {};
  // sums of A's rows over the contraction: a product with ones, for the first
  // column of tiles
  constexpr bool SUMS = !A_KM;
  f32x4 sums[SUMS ? MI : 1] = {};
  const bool want_sums = SUMS && p.row_part != nullptr && n0 == 0 && wn == 0;
  const typename A::template Fragments<MI> a_frag(wm, lane);
  const typename B::template Fragments<NI> b_frag(wn, lane);
  auto multiply = [&](const char* a_s) {
    const char* b_s = a_s + A::BYTES;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      uint4 fb[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = b_frag.get(b_s, j, kb);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const uint4 fa = a_frag.get(a_s, i, kb);
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mfma_block<T>(fb[j], fa, acc[i][j]);
        if constexpr (SUMS) {
          if (want_sums) sums[i] = mfma_block<T>(ones_chunk<T>(), fa, sums[i]);
        }
      }
    }
  };
  // The stage has arrived (each wave waits for its own part, then for the
  // others), and every wave is done with what is loaded into next.
  auto arrive = [&] {
    if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  if (iters) {
    fetch(0, stage0);
    put(stage0);
  }
  if constexpr (STAGES == 1) {
    for (int it = 0; it < iters; ++it) {
      arrive();
      multiply(stage0);
      if (it + 1 < iters) {
        __syncthreads();
        fetch(it + 1, stage0);
        put(stage0);
      }
    }
  } else {
    int it = 0;
    for (; it + 1 < iters; it += 2) {
      arrive();
      fetch(it + 1, stage1);
      multiply(stage0);
      put(stage1);
      arrive();
      const bool on = it + 2 < iters;
      if (on) fetch(it + 2, stage0);
      multiply(stage1);
      if (on) put(stage0);
    }
    if (it < iters) {
      arrive();
      multiply(stage0);
    }
  }
  __syncthreads();  // the stages now hold the output blocks

  constexpr int WNC = BN / WN, V = 16 / sizeof(T);
  // worked out anew: kept through the loop, what follows takes registers there
  int lane_out = threadIdx.x & 63;
  asm volatile("" : "+v"(lane_out));
  const int lo_out = lane_out & 15, g_out = lane_out >> 4;
  float* block = reinterpret_cast<float*>(stage0) + wave * 16 * (WNC + 4);
  float bias[V];
  const int n_lane = n0 + wn + (lane_out % (WNC / V)) * V;
  if (p.bias) {
    load_row<T, V>(reinterpret_cast<const T*>(p.bias) + n_lane, p.N - n_lane, bias);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = 0.f;
  }
  auto finish = [&](auto act) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + wm + 16 * i;
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<f32x4*>(block + lo_out * (WNC + 4) + 16 * j + 4 * g_out) = acc[i][j];
      finish_block<T, WNC, decltype(act)::value>(p, block, lane_out, m, n0 + wn, bias);
      if constexpr (SUMS) {
        if (want_sums && g_out == 0 && m + lo_out < p.M) p.row_part[(int64_t)at_part * p.M + m + lo_out] = sums[i][0];
      }
    }
  };
  if constexpr (A_KM && B_KM) {  // the forward product
    if (p.act == ACT_RELU) return finish(std::integral_constant<int, ACT_RELU>{});
    if (p.act == ACT_GELU) return finish(std::integral_constant<int, ACT_GELU>{});
    if (p.act == ACT_SILU) return finish(std::integral_constant<int, ACT_SILU>{});
  }
  finish(std::integral_constant<int, ACT_NONE>{});
}

// out[i] = sum of the parts' element i, in a fixed order: 16 lanes by 4 elements
// across, 16 groups down the parts, whose sums meet in LDS (256 parts of 64 x 64,
// 4 MB: 5 us).  The elements from size on lie apart, as another array of the same
// number of parts.
template <typename T>
__global__ __launch_bounds__(256) void join_parts(const float* part, T* out, int64_t size, const float* part2,
                                                  T* out2, int64_t size2, int64_t blocks, int parts) {
  constexpr int X = 16, Y = 16;
  __shared__ __attribute__((aligned(16))) f32x4 group[Y][X];
  const int x = threadIdx.x % X, y = threadIdx.x / X;
  int64_t block = blockIdx.x;
  if (block >= blocks) {
    block -= blocks;
    part = part2;
    out = out2;
    size = size2;
  }
  const int64_t i = (block * X + x) * 4;
  const int left = (int)min((int64_t)4, size - i);
  float sum[4] = {};
  if (left > 0) {
#pragma unroll 4
    for (int s = y; s < parts; s += Y) {
      float v[4];
      load_row<float, 4>(part + s * size + i, left, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r] += v[r];
    }
  }
  group[y][x] = f32x4{sum[0], sum[1], sum[2], sum[3]};
  __syncthreads();
  // the groups in pairs, halving
#pragma unroll
  for (int half = Y / 2; half > 0; half /= 2) {
    if (y < half) group[y][x] += group[y + half][x];
    __syncthreads();
  }
  if (y == 0 && left > 0) {
    const f32x4 all = group[0][x];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) out[i + r] = from_f32<T>(all[r]);
  }
}

// dz = dy act'(z), and the column sums of it before its rounding, for db;
// without z the sums of dy alone.
// LC threads (a power of two) with a chunk of columns each, 256 / LC rows at a
// time; part[blockIdx.y][n] = sums over the rows of this workgroup.
template <typename T>
__global__ __launch_bounds__(256) void slope_product(const T* dy, int64_t ldy, const T* z, T* dz,
                                                     float* part, int64_t M, int N, int act, int LC,
                                                     int64_t rows) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float sums[256 * V];
  const int c = (blockIdx.x * LC + threadIdx.x % LC) * V, step = 256 / LC;
  const int left = min(V, N - c);
  const int64_t end = min(M, (blockIdx.y + 1) * rows);
  float sum[V] = {};
  if (left > 0) {
    for (int64_t m = blockIdx.y * rows + threadIdx.x / LC; m < end; m += step) {
      alignas(16) T d[V], s[V];
      const T* dp = dy + m * ldy + c;
      if (left == V) {
        __builtin_memcpy(d, dp, 16);
        if (z) __builtin_memcpy(s, z + m * N + c, 16);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[i] = i < left ? dp[i] : from_f32<T>(0.f);
          if (z) s[i] = i < left ? z[m * N + c + i] : from_f32<T>(0.f);
        }
      }
      if (!z) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += to_f32<T>(d[i]);
        continue;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float v = to_f32<T>(d[i]) * act_slope(act, to_f32<T>(s[i]));
        sum[i] += v;
        d[i] = from_f32<T>(v);
      }
      T* out = dz + m * N + c;
      if (left == V) {
        __builtin_memcpy(out, d, 16);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < left) out[i] = d[i];
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < V; ++i) sums[i * 256 + threadIdx.x] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < LC * V; i += 256) {
    const int lane = i / V, n = (blockIdx.x * LC + lane) * V + i % V;
    if (n >= N) continue;
    float all = 0.f;
    for (int r = 0; r < step; ++r) all += sums[(i % V) * 256 + r * LC + lane];
    part[(int64_t)blockIdx.y * N + n] = all;
  }
}

// Which tile a product runs on.
enum Tile { T256, T128, T128x64, T64 };

int64_t tile_count(Tile t, int64_t M, int64_t N) {
  const int64_t bm = t == T256 ? 256 : t == T64 ? 64 : 128, bn = t == T256 ? 256 : t == T128 ? 128 : 64;
  return ((M + bm - 1) / bm) * ((N + bn - 1) / bn);
}

// The largest tile that still gives every CU a workgroup and has a contraction
// long enough for it: one workgroup of the large tiles fills a CU, so nothing
// hides its first loads and its stores.  bfloat16, us: 16384 x 4096 by K 4096:
// 543 (T256), 666 (T128), 755 (T128x64); 25601 x 256 by K 1024: 38, 25, 31;
// 25601 x 1024 by K 256 (erff): 60, 58, 50; 409600 x 64 by K 64: 84, 51, 30, 39 (T64).
Tile pick_tile(int64_t M, int64_t N, int64_t K, bool wide) {
  if (wide && K >= 1024 && tile_count(T256, M, N) >= 256) return T256;
  if (N > 64 && K >= 512 && tile_count(T128, M, N) >= 256) return T128;
  if (M > 64 && tile_count(T128x64, M, N) >= 256) return T128x64;
  return T64;
}

// Whole 16-byte chunks, and offsets over a tile within 32 bits: what the path
// without registers needs.
template <typename T>
bool chunks_aligned(const void* p, int64_t ld, int64_t inner) {
  constexpr int CH = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % CH == 0 && ld < (1 << 21) &&
         inner % CH == 0;
}

template <typename T, bool A_KM, bool B_KM, int BM, int BN, int WM, int WN, bool DIRECT, int STAGES>
void launch_tile(Gemm p, int parts, hipStream_t stream) {
  const int64_t tiles = (int64_t)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  TORCH_CHECK(tiles * parts < (int64_t(1) << 31), "fused_linear: too many tiles");
  p.tiles = (unsigned)tiles;
  hipLaunchKernelGGL((gemm_tile<T, A_KM, B_KM, BM, BN, WM, WN, DIRECT, STAGES>),
                     dim3((unsigned)(tiles * parts)), dim3(WM * WN * 64), 0, stream, p);
  HIP_CHECK(hipGetLastError());
}

template <typename T, bool A_KM, bool B_KM>
void launch_gemm(const Gemm& p, Tile tile, int parts, hipStream_t stream) {
  if (p.M == 0 || p.N == 0) return;
  const bool direct = chunks_aligned<T>(p.a, p.lda, A_KM ? p.K : p.M) &&
                      chunks_aligned<T>(p.b, p.ldb, B_KM ? p.K : p.N);
  // a contraction of one stage needs no second: more workgroups fit a CU
  const bool one = A_KM && p.K * (int64_t)sizeof(T) <= 128;
#define FL_TILE(...) return launch_tile<T, A_KM, B_KM, __VA_ARGS__>(p, parts, stream)
  if (direct) {
    if constexpr (sizeof(T) == 2 && A_KM) {
      if (tile == T256) FL_TILE(256, 256, 2, 4, true, 2);
    }
    // where dW has one workgroup a CU: in 8 waves, two a SIMD hide each other's
    // transposing reads (1024 x 256 by 25601: 36 us in 4 waves, 31; all gradients of
    // 8192 x 8192 by 8192, with db, whose sums weigh more in narrower waves: 2590, 2650)
    if constexpr (sizeof(T) == 2 && !A_KM) {
      if (tile == T128 && tile_count(T128, p.M, p.N) < 128) FL_TILE(128, 128, 2, 4, true, 2);
    }
    if (tile == T256 || tile == T128) FL_TILE(128, 128, 2, 2, true, 2);
    if constexpr (A_KM) {
      if (tile == T128x64 && one) FL_TILE(128, 64, 4, 1, true, 1);
      if (tile == T128x64) FL_TILE(128, 64, 4, 1, true, 2);
      if (one) FL_TILE(64, 64, 2, 2, true, 1);
    }
    FL_TILE(64, 64, 2, 2, true, 2);
  }
  // through registers the larger tile only pays where the products bound
  // (20001 x 501 by K 1001: 131 us with T128, 101 with T64)
  if constexpr (A_KM) {
    if (tile == T256) FL_TILE(128, 128, 2, 2, false, 2);
  }
  FL_TILE(64, 64, 2, 2, false, 2);
#undef FL_TILE
}

// Parts of out, and where given of out2, joined in one launch.
template <typename T>
void join(const torch::Tensor& part, torch::Tensor& out, const torch::Tensor& part2, torch::Tensor out2,
          int parts, hipStream_t stream) {
  const int64_t size = out.numel(), size2 = out2.defined() ? out2.numel() : 0;
  const int64_t blocks = (size + 63) / 64, all = blocks + (size2 + 63) / 64;
  if (all == 0) return;
  TORCH_CHECK(all < (int64_t(1) << 31), "fused_linear: weight too large");
  const float* p2 = size2 ? part2.data_ptr<float>() : nullptr;
  T* o2 = size2 ? reinterpret_cast<T*>(out2.data_ptr()) : nullptr;
  hipLaunchKernelGGL((join_parts<T>), dim3((unsigned)all), dim3(256), 0, stream, part.data_ptr<float>(),
                     reinterpret_cast<T*>(out.data_ptr()), size, p2, o2, size2, blocks, parts);
  HIP_CHECK(hipGetLastError());
}

// [..., D] as rows of D, the last dimension contiguous.
torch::Tensor rows_of(const torch::Tensor& t) {
  auto r = t;
  if (t.dim() != 2) {
    TORCH_CHECK(t.dim() >= 1, "fused_linear: needs at least one dimension");
    int64_t rows = 1;
    for (int i = 0; i < t.dim() - 1; ++i) rows *= t.size(i);
    r = t.reshape({rows, t.size(-1)});
  }
  return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}

void check_rows(const torch::Tensor& t, const torch::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device() && t.scalar_type() == x.scalar_type(), "fused_linear: ", name,
              " must share type and device with x");
  TORCH_CHECK(t.dim() == 2, "fused_linear: ", name, " needs two dimensions");
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
  launch_gemm<T, true, true>(p, pick_tile(p.M, p.N, p.K, sizeof(T) == 2), 1, stream);
}

template <typename T>
void backward_t(const torch::Tensor& dy, const torch::Tensor& x, const torch::Tensor& w,
                const torch::Tensor& z, int act, torch::Tensor& dx, torch::Tensor& dw,
                torch::Tensor& db, hipStream_t stream) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  constexpr bool wide = sizeof(T) == 2;
  auto f32 = x.options().dtype(torch::kFloat32);
  torch::Tensor dz = dy;
  const bool slope = act != ACT_NONE;
  // without a slope dz is exact, and its column sums ride on the product for dW
  const bool sums = db.defined() && !slope && dw.defined() && M && N && K;
  if (db.defined() && (M == 0 || N == 0)) db.zero_();
  if (M && N && (slope || (db.defined() && !sums))) {
    if (slope) dz = torch::empty({M, N}, x.options());
    constexpr int V = 16 / sizeof(T);
    int LC = 1;
    while (LC < 64 && LC * V < N) LC *= 2;
    const int64_t across = (N + LC * V - 1) / (LC * V);
    const int64_t down = std::max<int64_t>(1, std::min<int64_t>(2048 / across, M / (4 * (256 / LC))));
    const int64_t rows = (M + down - 1) / down;
    auto part = torch::empty({db.defined() ? down : 0, N}, f32);
    hipLaunchKernelGGL((slope_product<T>), dim3((unsigned)across, (unsigned)down), dim3(256), 0, stream,
                       reinterpret_cast<const T*>(dy.data_ptr()), dy.stride(0),
                       slope ? reinterpret_cast<const T*>(z.data_ptr()) : nullptr,
                       slope ? reinterpret_cast<T*>(dz.data_ptr()) : nullptr,
                       db.defined() ? part.data_ptr<float>() : nullptr, M, (int)N, act, LC, rows);
    HIP_CHECK(hipGetLastError());
    if (db.defined()) join<T>(part, db, {}, {}, (int)down, stream);
  }
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
    launch_gemm<T, true, false>(p, pick_tile(M, K, N, wide), 1, stream);
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
    // The rows are cut into parts, of 256 rows at least, until there is a
    // workgroup a CU: more parts are more float partials to write and read back.
    // us by workgroups 128, 256, 512, 1024, before a part's tiles shared a die:
    // 1024 x 256 by 25601 rows 46, 37 (now 31), 42, 56; 64 x 64 by 409600 (T64)
    // 30, 21, 24, 27.  Where the tiles alone fill
    // half the card, two a CU (2048 x 2048 by 8192: 131, 118).  (T256's registers
    // are full already: 849 us against 647 for 4096 x 4096 by 16384.)  Through
    // registers, small tiles and many: 500 x 1000 by 20000, 154 with T128, 89.
    const bool direct = chunks_aligned<T>(p.a, p.lda, N) && chunks_aligned<T>(p.b, p.ldb, K);
    const Tile dw_tile = !direct || N <= 64 || K <= 64 ? T64 : T128;
    const int64_t tiles = std::max<int64_t>(tile_count(dw_tile, N, K), 1);
    const int64_t most = std::max<int64_t>(1, M / 256), want = !direct ? 1024 : tiles >= 128 ? 512 : 256;
    int64_t parts = std::max<int64_t>(1, std::min<int64_t>(want / tiles, most));
    p.k_part = std::max<int64_t>(64, ((M + parts - 1) / parts + 63) / 64 * 64);
    parts = std::max<int64_t>(1, (M + p.k_part - 1) / p.k_part);
    auto part = torch::empty({parts, N, K}, f32);
    auto row_part = torch::empty({sums ? parts : 0, N}, f32);
    p.part = part.data_ptr<float>();
    p.row_part = sums ? row_part.data_ptr<float>() : nullptr;
    launch_gemm<T, false, false>(p, dw_tile, (int)parts, stream);
    join<T>(part, dw, row_part, sums ? db : torch::Tensor(), (int)parts, stream);
  }
}

}  // namespace

// -> {y, of x's leading dimensions, z or empty, as rows}
std::vector<torch::Tensor> fused_linear_fwd(torch::Tensor x_in, torch::Tensor weight,
                                            c10::optional<torch::Tensor> bias,
                                            c10::optional<torch::Tensor> residual, int64_t act,
                                            bool want_z) {
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(
      x_in.is_cuda() ? c10::optional<c10::Device>(x_in.device()) : c10::nullopt);
  auto x = rows_of(x_in);
  check_x(x, weight);
  weight = rows_of(weight);
  const int64_t M = x.size(0), N = weight.size(0);
  TORCH_CHECK(act >= 0 && act <= 3, "fused_linear: unknown activation");
  // a dual tensor's tangent would be lost
  auto dual = [](const c10::optional<torch::Tensor>& t) { return t.has_value() && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!dual(x_in) && !dual(weight) && !dual(bias) && !dual(residual),
              "fused_linear: not differentiable in forward mode on the GPU");
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == x.device() && bias->scalar_type() == x.scalar_type() &&
                    bias->dim() == 1 && bias->size(0) == N,
                "fused_linear: bias must be [N], of x's type and device");
    bias = bias->contiguous();
  }
  auto shape = x_in.sizes().vec();
  shape.back() = N;
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == c10::IntArrayRef(shape), "fused_linear: residual must be [..., N]");
    residual = rows_of(*residual);
    check_rows(*residual, x, "residual");
  }
  auto stream = at::cuda::getCurrentHIPStream();
  auto y = torch::empty(shape, x.options());
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

// -> {dx, dw, db}, empty where not needed.  z: what the slope is taken at (for
// relu the output serves as well); unused without an activation.
std::vector<torch::Tensor> fused_linear_bwd(torch::Tensor dy_in, torch::Tensor x_in, torch::Tensor weight,
                                            torch::Tensor z, int64_t act, bool need_x, bool need_w,
                                            bool need_b) {
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(
      x_in.is_cuda() ? c10::optional<c10::Device>(x_in.device()) : c10::nullopt);
  auto x = rows_of(x_in), dy = rows_of(dy_in);
  check_x(x, weight);
  weight = rows_of(weight);
  check_rows(dy, x, "dy");
  const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
  TORCH_CHECK(act >= 0 && act <= 3, "fused_linear: unknown activation");
  TORCH_CHECK(dy.size(0) == M && dy.size(1) == N, "fused_linear: dy must be [..., N]");
  TORCH_CHECK(act == ACT_NONE || (z.is_contiguous() && z.numel() == M * N &&
                                  z.scalar_type() == x.scalar_type() && z.device() == x.device()),
              "fused_linear: z must be [..., N], of x's type and device");
  auto stream = at::cuda::getCurrentHIPStream();
  torch::Tensor dx, dw, db;
  if (need_x) dx = torch::empty(x_in.sizes(), x.options());
  if (need_w) dw = torch::empty({N, K}, x.options());
  if (need_b) db = torch::empty({N}, x.options());
#define FL_BACKWARD(T) backward_t<T>(dy, x, weight, z, (int)act, dx, dw, db, stream)
  if (x.scalar_type() == torch::kBFloat16) FL_BACKWARD(__hip_bfloat16);
  else if (x.scalar_type() == torch::kHalf) FL_BACKWARD(__half);
  else FL_BACKWARD(float);
#undef FL_BACKWARD
  auto none = torch::empty({0}, x.options());
  return {need_x ? dx : none, need_w ? dw : none, need_b ? db : none};
}
