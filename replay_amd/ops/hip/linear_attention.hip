// Linear attention with a decay for each head (gfx950).
//
// For the valid positions t of one (batch, head), with l = exp(log_decay):
//
//   S_t = l S_{t-1} + k_t v_t^T          o_t = scale q_t^T S_t
//
// A masked position takes no part: it neither decays nor writes the state,
// and its output is zero.  Over a chunk of C positions with the start state S
// and n_i = the number of valid positions among the chunk's first i+1,
//
//   o_i = scale [ l^{n_i} q_i^T S + sum_{j<=i} l^{n_i-n_j} (q_i.k_j) v_j ]
//   S  <- l^N S + sum_j l^{N-n_j} k_j v_j^T                    (N = n_last)
//
// Every gradient but the decay's is another linear attention, so ONE pass
// kernel serves all of them (dO = the output's gradient):
//
//   dq = forward pass over (q, k, v) := (dO, v, k), state transposed
//   dk = REVERSED pass over (v, dO, q), dv = reversed pass over (k, q, dO):
//        position j sees the later ones i >= j; the state is dL/dS, the
//        query-side weight is l^{N-n_j} and the update's is scale l^{n_i}
//
// The decay's gradient is taken forward: S' = dS/dlog l obeys
//   S' <- l^N (S' + N S) + sum_j (N-n_j) l^{N-n_j} k_j v_j^T
// and rides on the dq pass as sum_i q_i . dq'_i.  (The shorter formula
// sum_t t (q_t.dq_t - k_t.dk_t) cancels nearly everything on long histories.)
// In a cut history each segment takes its start state as constant; what that
// state's own derivative adds is <S'_start, V>, V = the segment's contribution
// to dL/dS, which a scan sums up over the segments.
//
// Where batch x heads alone cannot fill the card, the history is cut into
// segments: a state-only pass gives each segment's own contribution, a scan
// over the segments turns these into start states, and the full pass then
// runs all segments at once.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;

struct Rows {  // [B, H, L, D] with unit stride in D
  const void* p;
  int64_t b, h, l;
};

struct ShortArgs {
  Rows q, k, v, out;       // forward: out
  Rows dout, dq, dk, dv;   // backward
  const float* log_decay;  // [H]
  const bool* mask;        // [B, L] or nullptr, true = valid
  int64_t mask_b, mask_l;
  float* decay_part;       // [B, H] or nullptr
  float scale;
  int H, L, Dk, Dv;
};

struct PassArgs {
  Rows q, k, v, x;       // x: the query whose product with dq' is the decay's gradient
  void* out;
  int64_t out_b, out_h, out_l;
  const float* log_decay;            // [H]
  const bool* mask;                  // [B, L] or nullptr, true = valid
  int64_t mask_b, mask_l;
  const float* state_in;             // [B, H, Dk, Dv] or nullptr
  float* state_out;                  // same or nullptr: the state after the last chunk
  const float* state_end_grad;       // same or nullptr: for <S'_end, dS_end>
  float* seg;                        // [B, H, G, Dk, Dv]: contributions, then start states
  float* seg_d;                      // of each segment: S' at its end, for a constant start
  int* seg_count;                    // [B, H, G] valid positions
  float* decay_part;                 // [B, H, parts] partial sums of the decay's gradient
  int parts;
  int64_t st_c, st_e;                // strides of a state's (contraction, value) axes
  int B, H, L, Dc, De, G, seg_chunks;
  float c_pair, c_inter, c_update;   // where the scale goes
};

// dk's and dv's passes run in one launch, by turns of 8 workgroups, so that the
// two for the same rows are on one die at about the same time: both read q and
// dO, and few heads fill the card better.  us, of the whole backward pass, in two
// launches and in one: 2 x 8 heads of 16384 at 128, 365 and 343; 33 x 3 of 333
// (float32, 48) 98 and 83; 64 x 8 of 500 (40 and 56) 124 and 113; 1024 x 2 of
// 200 at 64, 184 and 179.
template <int N>
struct Passes {
  PassArgs a[N];
};
constexpr int passes_of(bool rev, bool state_only, bool deriv) { return rev && !state_only && !deriv ? 2 : 1; }

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// V neighbours of a row, of which n exist; no alignment is asked for
template <typename T, int V>
__device__ __forceinline__ uint4 load_piece(const T* p, int n) {
  alignas(16) T t[V];
  if (n >= V) {
    __builtin_memcpy(t, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
  return *reinterpret_cast<const uint4*>(t);
}

// One operand's 32 positions on their way from memory to LDS, where they are
// float: 16-byte pieces, DP / V of 4 DP threads a row.
template <typename T, int DP>
struct Rows32 {
  static constexpr int V = 16 / sizeof(T), ACROSS = DP / V, DOWN = DP * 4 / ACROSS, PIECES = 32 / DOWN;
  static constexpr int LD = DP + 4;  // rows then start 4 banks apart

  const T* at;
  int64_t l;
  int left;
  uint4 r[PIECES];

  __device__ __forceinline__ Rows32(const Rows& src, int b, int h, int D) {
    const int d = (threadIdx.x % ACROSS) * V;
    l = src.l;
    left = D - d;
    at = reinterpret_cast<const T*>(src.p) + b * src.b + h * src.h + (threadIdx.x / ACROSS) * l + d;
  }
  __device__ __forceinline__ void fetch(int l0, unsigned bits) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      r[i] = uint4{0, 0, 0, 0};
      if (((bits >> (threadIdx.x / ACROSS + i * DOWN)) & 1) && left > 0)
        r[i] = load_piece<T, V>(at + (l0 + i * DOWN) * l, left);
    }
  }
  __device__ __forceinline__ void put(float* dst) const {
    dst += (threadIdx.x / ACROSS) * LD + (threadIdx.x % ACROSS) * V;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      alignas(16) T t[V];
      *reinterpret_cast<uint4*>(t) = r[i];
#pragma unroll
      for (int j = 0; j < V; j += 4)
        *reinterpret_cast<f32x4*>(dst + i * DOWN * LD + j) =
            f32x4{to_f32<T>(t[j]), to_f32<T>(t[j + 1]), to_f32<T>(t[j + 2]), to_f32<T>(t[j + 3])};
    }
  }
};

// One segment of one (batch, head) on the float32 matrix instructions: 16
// positions a chunk (the pair products grow with it, and these instructions
// have a sixteenth of the 16-bit ones' rate), 32 a load.  DP/16 waves; each
// owns 16 value columns and the whole contraction axis of the state, in the
// accumulator layout (column = lane & 15, row = 4 (lane >> 4) + r), which is
// also the layout of an operand whose contraction index is visited in that
// order: neither the state nor the pair weights leave the registers between
// products.  (Launch bounds as in la_pass_bf16: none that need spills.)
template <typename T, int DP, bool REV, bool STATE_ONLY, bool DERIV>
__global__ __launch_bounds__(DP * 4, 2) void la_pass_f32(Passes<passes_of(REV, STATE_ONLY, DERIV)> all_passes) {
  constexpr bool PAIR = passes_of(REV, STATE_ONLY, DERIV) == 2;
  unsigned id = blockIdx.x;
  const PassArgs& a = all_passes.a[PAIR ? (id >> 3) & 1 : 0];
  if (PAIR) {
    id = (id >> 4) * 8 + (id & 7);
    if (id >= (unsigned)(a.B * a.H * a.G)) return;  // the same for a whole workgroup
  }
  using Ch = Rows32<T, DP>;
  constexpr int C = 16, ROWS = 32, LD = Ch::LD, NT = DP / 16, WAVES = DP / 16;
  constexpr bool FULL = !STATE_ONLY, X = DERIV && FULL;
  __shared__ __attribute__((aligned(16))) float q_s[FULL ? ROWS * LD : 4];
  __shared__ __attribute__((aligned(16))) float k_s[ROWS * LD];
  __shared__ __attribute__((aligned(16))) float v_s[ROWS * LD];
  __shared__ __attribute__((aligned(16))) float o_s[FULL ? ROWS * LD : 4];
  __shared__ __attribute__((aligned(16))) float x_s[X ? ROWS * LD : 4];
  // of each position, within its chunk: the valid ones up to it, and its
  // weights in the product with the start state and in the state's update
  __shared__ __attribute__((aligned(16))) float n_s[ROWS], inter_s[ROWS], update_s[ROWS];
  __shared__ float lam[C + 1];
  __shared__ float red[WAVES];

  const int seg = id % (unsigned)a.G;
  const int64_t bh = id / (unsigned)a.G;
  const int b = bh / a.H, h = bh % a.H;
  // the wave's index is the same for its lanes, which the compiler cannot see:
  // what depends on it alone then needs no vector registers and no masks
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo = lane & 15, g = lane >> 4;
  const int e0 = wave * 16, e = e0 + lo;
  const bool busy = e0 < a.De;
  const int64_t state_size = (int64_t)a.Dc * a.De;
  // seg_chunks counts loads of 32 positions here
  const int n_loads = (a.L + ROWS - 1) / ROWS;
  const int first = seg * a.seg_chunks, last = min(n_loads, first + a.seg_chunks);
  auto start_of = [&](int step) { return (REV ? first + last - 1 - step : step) * ROWS; };
  Ch q_r(a.q, b, h, a.Dc), k_r(a.k, b, h, a.Dc), v_r(a.v, b, h, a.De), x_r(a.x, b, h, a.De);
  // The mask is read a load ahead of the rows that it says to read.
  const bool* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
  auto look = [&](int step) {
    const int pos = start_of(step) + lane;
    return lane < ROWS && step < last && pos < a.L && (!mask || mask[pos * a.mask_l]);
  };
  auto fetch = [&](int step, unsigned bits) {
    const int l0 = start_of(step);
    if (FULL) q_r.fetch(l0, bits);
    k_r.fetch(l0, bits);
    v_r.fetch(l0, bits);
    if (X) x_r.fetch(l0, bits);
  };
  // the first loads are on their way while the rest is prepared
  unsigned bits = (unsigned)__ballot(look(first));
  fetch(first, bits);
  bool ahead = look(first + 1);
  const float ld = a.log_decay[h];
  // a decay of zero (log -inf) keeps l^0 = 1
  if (threadIdx.x <= C) lam[threadIdx.x] = threadIdx.x ? expf(ld * threadIdx.x) : 1.f;

  // whether the state after the last chunk is asked for
  const bool at_end = REV ? seg == 0 : seg == a.G - 1;
  const bool want_end = STATE_ONLY || (at_end && a.state_out) || (DERIV && (a.G > 1 || a.state_end_grad));
  // false while the state is known to be zero, as a history's first chunk has it
  bool started = FULL && (a.G > 1 || a.state_in);
  f32x4 S[NT], Sd[DERIV ? NT : 1];
  {
    const float* src = nullptr;
    if (FULL) {
      if (a.G > 1) src = a.seg + (bh * a.G + seg) * state_size;
      else if (a.state_in) src = a.state_in + bh * state_size;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // the addresses of a tile at a time: worked out together, they take two
      // registers for each element of the state
      int g_t = g;
      asm volatile("" : "+v"(g_t)::"memory");
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int c = 16 * t + 4 * g_t + r;
        const bool in = c < a.Dc && e < a.De;
        S[t][r] = (src && in) ? src[c * a.st_c + e * a.st_e] : 0.f;
        if (DERIV) Sd[t][r] = 0.f;
      }
    }
  }
  __syncthreads();  // lam
  // the pair weights of a chunk without gaps
  f32x4 full = {};
  if (FULL) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int gap = REV ? 4 * g + r - lo : lo - 4 * g - r;
      full[r] = gap >= 0 ? a.c_pair * lam[max(gap, 0)] : 0.f;
    }
  }

  T* out = nullptr;
  if (FULL)
    out = reinterpret_cast<T*>(a.out) + b * a.out_b + h * a.out_h +
          (threadIdx.x / Ch::ACROSS) * a.out_l + (threadIdx.x % Ch::ACROSS) * Ch::V;
  // outputs of the rows at l0 in whole rows, from LDS or zeros
  auto store = [&](int l0, bool zero) {
    const int row = threadIdx.x / Ch::ACROSS, left = v_r.left;
    const float* from = o_s + row * LD + (threadIdx.x % Ch::ACROSS) * Ch::V;
#pragma unroll
    for (int i = 0; i < Ch::PIECES; ++i) {
      if (l0 + row + Ch::DOWN * i >= a.L || left <= 0) continue;
      alignas(16) T t[Ch::V];
#pragma unroll
      for (int j = 0; j < Ch::V; j += 4) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (!zero) v = *reinterpret_cast<const f32x4*>(from + i * Ch::DOWN * LD + j);
#pragma unroll
        for (int r = 0; r < 4; ++r) t[j + r] = from_f32<T>(v[r]);
      }
      T* p = out + (l0 + Ch::DOWN * i) * a.out_l;
      if (left >= Ch::V) {
        __builtin_memcpy(p, t, 16);
      } else {
#pragma unroll
        for (int j = 0; j < Ch::V; ++j)
          if (j < left) p[j] = t[j];
      }
    }
  };

  int total = 0;
  float d_decay = 0.f;
#pragma unroll 1
  for (int step = first; step < last; ++step) {
    const int l0 = start_of(step);
    const unsigned now = bits;
    total += __popc(now);
    // without valid positions nothing is seen, added or forgotten.  (One way
    // round the loop for both cases: a second one, with a continue, kept copies
    // of the state.)
    if (now) {
      if (FULL) q_r.put(q_s);
      k_r.put(k_s);
      v_r.put(v_s);
      if (X) x_r.put(x_s);
      if (threadIdx.x < ROWS) {
        const unsigned own = (now >> (lane & 16)) & 0xffffu;
        const int n = __popc(own & ((2u << (lane & 15)) - 1)), N = __popc(own);
        n_s[lane] = (float)n;
        inter_s[lane] = a.c_inter * lam[REV ? N - n : n];
        update_s[lane] = a.c_update * lam[REV ? n : N - n];
      }
      __syncthreads();
    }
    bits = (unsigned)__ballot(ahead);
    fetch(step + 1, bits);
    ahead = look(step + 2);

    if (busy && now) {
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int r0 = (REV ? 1 - half : half) * C;
        const unsigned own = (now >> r0) & 0xffffu;
        const int N = __popc(own);
        // (an empty half: its products are of zeros, and decay by l^0)
        const float* k_c = k_s + r0 * LD;
        float vr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) vr[r] = v_s[(r0 + 4 * g + r) * LD + e0 + lo];
        const f32x4 n_j = *reinterpret_cast<const f32x4*>(n_s + r0 + 4 * g);
        if (FULL) {
          const float* q_c = q_s + (r0 + lo) * LD;
          const float n_i = n_s[r0 + lo], w_i = inter_s[r0 + lo];
          f32x4 pt = {0.f, 0.f, 0.f, 0.f}, o = pt, od = pt;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (DERIV) asm volatile("" ::: "memory");
            const f32x4 qv = *reinterpret_cast<const f32x4*>(q_c + 16 * t + 4 * g);
            const f32x4 kv = *reinterpret_cast<const f32x4*>(k_c + lo * LD + 16 * t + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) pt = mfma4(kv[r], qv[r], pt);
            if (started) {
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                o = mfma4(S[t][r], qv[r], o);
                if (DERIV) od = mfma4(Sd[t][r], qv[r], od);
              }
            }
          }
          if (DERIV) od = w_i * (od + n_i * o);
          o = w_i * o;
          // valid positions in one run: n_i - n_j = i - j wherever a pair counts
          const unsigned run = own >> __builtin_ctz(own | 0x10000u);
          const bool whole = (run & (run + 1)) == 0;
          const f32x4 gaps = REV ? n_j - n_i : n_i - n_j;
          f32x4 p = pt * full;
          if (!whole) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool seen = REV ? 4 * g + r >= lo : 4 * g + r <= lo;
              p[r] = seen ? pt[r] * (a.c_pair * lam[max((int)gaps[r], 0)]) : 0.f;
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            o = mfma4(vr[r], p[r], o);
            if (DERIV) od = mfma4(vr[r], p[r] * gaps[r], od);
          }
          if (DERIV) {
            const f32x4 xv = *reinterpret_cast<const f32x4*>(x_s + (r0 + lo) * LD + e0 + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) d_decay += xv[r] * od[r];
          }
          *reinterpret_cast<f32x4*>(o_s + (r0 + lo) * LD + e0 + 4 * g) = o;
        }
        const bool update = want_end || step + 1 < last || half == 0;
        started = true;
        if (update) {
          const float lN = lam[N];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (DERIV) Sd[t] = lN * (Sd[t] + (float)N * S[t]);
            S[t] = lN * S[t];
          }
          const f32x4 w = *reinterpret_cast<const f32x4*>(update_s + r0 + 4 * g);
          const f32x4 left = REV ? n_j : (float)N - n_j;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (DERIV) asm volatile("" ::: "memory");
            const float weighted = vr[r] * w[r];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const float kv = k_c[(4 * g + r) * LD + 16 * t + lo];
              S[t] = mfma4(kv, weighted, S[t]);
              if (DERIV) Sd[t] = mfma4(kv, weighted * left[r], Sd[t]);
            }
          }
        }
      }
    }
    if (now) __syncthreads();  // the rows are read and their outputs are in LDS
    if (FULL) store(l0, now == 0);
  }

  float* dst = nullptr;
  float* dst_d = nullptr;
  if (STATE_ONLY) {
    dst = a.seg + (bh * a.G + seg) * state_size;
    if (threadIdx.x == 0) a.seg_count[bh * a.G + seg] = total;
  } else if (at_end && a.state_out) {
    dst = a.state_out + bh * state_size;
  }
  // the derivative of the end state: for the scan, or here if it ends the history
  if (X && a.G > 1) dst_d = a.seg_d + (bh * a.G + seg) * state_size;
  const float* end_grad = (X && a.G == 1 && a.state_end_grad) ? a.state_end_grad + bh * state_size : nullptr;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    int g_t = g;
    asm volatile("" : "+v"(g_t)::"memory");
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = 16 * t + 4 * g_t + r;
      if (c < a.Dc && e < a.De) {
        const int64_t at = c * a.st_c + e * a.st_e;
        if (dst) dst[at] = S[t][r];
        if (DERIV && dst_d) dst_d[at] = Sd[t][r];
        if (DERIV && end_grad) d_decay += Sd[t][r] * end_grad[at];
      }
    }
  }
  if (X) {
    d_decay = wave_reduce_sum(d_decay);
    if (lane == 0) red[wave] = d_decay;
    __syncthreads();
    if (threadIdx.x == 0) {
      float sum = 0.f;
      for (int w = 0; w < WAVES; ++w) sum += red[w];
      a.decay_part[bh * a.parts + seg] = sum;
    }
  }
}

// ---------------------------------------------------------------------------
// The same pass for bfloat16 on the 16-bit matrix instructions, 64 positions a
// chunk.  Pair weights and states go from one product's result into the next
// one's operand without leaving the registers: a contraction over positions is
// visited in the order that two accumulator tiles have it, {4g .. 4g+3,
// 16+4g .. 16+4g+3} for lane group g; one over the head size in memory's order,
// 8g .. 8g+7, to which the rows of the state's tiles are permuted.  Everything
// comes from row-major LDS tiles, the transposed operands by transposing reads.
//
// The pair weights of a chunk are 6 units of a tile row by 32 keys (those on
// one side of the diagonal), shared out among the waves and handed round through
// LDS in operand layout.  (Each wave computing all of them took 90 more vector
// and 14 more matrix instructions a chunk at head size 64, and at 128, where 8
// waves did so, twice the time.)
//
// Roundings to bfloat16: the pair weights, once (half a step of each term).
// The state goes into the outputs as the sum of two bfloat16s (2^-17), into
// the decay's float32 gradient as three; the values weighted into the float32
// states go in as three, so that these are no coarser than their sums.

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;

__device__ __forceinline__ f32x4 mfma32(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 join8(uint2 a, uint2 b) {
  return __builtin_bit_cast(bf16x8, uint4{a.x, a.y, b.x, b.y});
}

__device__ __forceinline__ bf16x8 pack8(f32x4 a, f32x4 b) {
  const bf16x4 x = __builtin_convertvector(a, bf16x4), y = __builtin_convertvector(b, bf16x4);
  return join8(__builtin_bit_cast(uint2, x), __builtin_bit_cast(uint2, y));
}

__device__ __forceinline__ f32x4 widen(bf16x4 a) { return __builtin_convertvector(a, f32x4); }

// A float operand as a sum of N bfloat16s: to 2^-17 with two, exact with three
// (but for what underflows).
template <int N>
struct Split8 {
  bf16x8 part[N];
  __device__ __forceinline__ Split8(f32x4 a, f32x4 b) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bf16x4 x = __builtin_convertvector(a, bf16x4), y = __builtin_convertvector(b, bf16x4);
      part[i] = join8(__builtin_bit_cast(uint2, x), __builtin_bit_cast(uint2, y));
      a = a - widen(x);
      b = b - widen(y);
    }
  }
  // c + this . other, the small parts first; this as the left operand or the right
  __device__ __forceinline__ f32x4 times(bf16x8 other, f32x4 c) const {
#pragma unroll
    for (int i = N - 1; i >= 0; --i) c = mfma32(part[i], other, c);
    return c;
  }
  __device__ __forceinline__ f32x4 after(bf16x8 other, f32x4 c) const {
#pragma unroll
    for (int i = N - 1; i >= 0; --i) c = mfma32(other, part[i], c);
    return c;
  }
};

// 8 neighbours of a row, of which n exist (all of them unless EDGE); no
// alignment is asked for
template <bool EDGE>
__device__ __forceinline__ uint4 load8(const __hip_bfloat16* p, int n) {
  alignas(16) __hip_bfloat16 t[8];
  if (!EDGE || n >= 8) {
    __builtin_memcpy(t, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = i < n ? p[i] : __hip_bfloat16(0.f);
  }
  return *reinterpret_cast<const uint4*>(t);
}

template <bool EDGE>
__device__ __forceinline__ void store8(__hip_bfloat16* p, int n, uint4 v) {
  if (!EDGE || n >= 8) {
    __builtin_memcpy(p, &v, 16);
  } else {
    alignas(16) __hip_bfloat16 t[8];
    *reinterpret_cast<uint4*>(t) = v;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = t[i];
  }
}

// One operand's 64 positions on their way from memory to LDS: 16-byte pieces,
// DP / 8 threads a row.
template <int DP, bool EDGE, bool ROWS, int THREADS = DP * 4>
struct Chunk {
  static constexpr int C = 64, ACROSS = DP / 8, DOWN = THREADS / ACROSS, PIECES = C / DOWN;
  // rows 16 bytes apart from a power of two: the fragment reads of 16 rows
  // then start in banks 4 words apart.  Without such reads, 32 bytes: the
  // transposing reads of 8 rows then fill the banks.
  static constexpr int LD = DP * 2 + (ROWS ? 16 : 32), BYTES = C * LD;

  const __hip_bfloat16* at;  // this thread's first piece of position 0
  int64_t l;
  int left;                  // columns from d on that exist
  uint4 r[PIECES];

  __device__ __forceinline__ Chunk(const Rows& src, int b, int h, int D) {
    const int d = (threadIdx.x % ACROSS) * 8;
    l = src.l;
    left = D - d;
    at = reinterpret_cast<const __hip_bfloat16*>(src.p) + b * src.b + h * src.h +
         (threadIdx.x / ACROSS) * l + d;
  }
  __device__ __forceinline__ void fetch(int l0, uint64_t bits) {
    const uint64_t mine = bits >> (threadIdx.x / ACROSS);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      r[i] = uint4{0, 0, 0, 0};
      if (((mine >> (i * DOWN)) & 1) && left > 0) r[i] = load8<EDGE>(at + (l0 + i * DOWN) * l, left);
    }
  }
  __device__ __forceinline__ void put(char* dst) const {
    dst += (threadIdx.x / ACROSS) * LD + (threadIdx.x % ACROSS) * 16;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) *reinterpret_cast<uint4*>(dst + i * DOWN * LD) = r[i];
  }
  // operand rows row0 + (lane & 15), contraction block s of the head size
  static __device__ __forceinline__ bf16x8 rows(const char* t, int row0, int s, int lo, int g) {
    return *reinterpret_cast<const bf16x8*>(t + (row0 + lo) * LD + s * 64 + g * 16);
  }
  // operand columns, contraction block s of the positions: col0 + (lane & 15),
  // or, for tile t of the state, state_row(t, .) of it
  static __device__ __forceinline__ bf16x8 columns(const char* t, int col0, int apart, int s, int lo, int g) {
    uint2 half[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* p = t + (32 * s + 16 * i + 4 * g + (lo >> 2)) * LD + col0 * 2 + (lo & 3) * apart * 2;
      auto v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      half[i] = __builtin_bit_cast(uint2, v);
    }
    return join8(half[0], half[1]);
  }
};

// The contraction index of row 4 g + r of the state's tile t; in memory's order
// (the state-only pass, whose state is no operand) or permuted.
template <bool PERMUTED>
__device__ __forceinline__ int state_row(int t, int g, int r) {
  return PERMUTED ? 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r : 16 * t + 4 * g + r;
}

// DP / 16 waves, each with 16 value columns and the whole contraction axis.  The
// launch bounds are the tightest that spill no vector registers, and the build
// refuses kernels here that do: an earlier form of this pass with 53 spilled
// registers at head size 128 gave wrong first chunks now and then.  Why is not
// known.  Read in full, its assembly waits for every load before its use; a load
// is there before younger stores, to scratch memory too (0 of 168 million early);
// and no two waves share LDS without a barrier between.
// AHEAD: a chunk's rows are loaded while the one before is worked on.  At head
// size 128 two workgroups a CU (128 registers) without that hide the loads better
// than one with it, where there are as many: 64 x 8 heads of 512, 57 us against
// 80; 2 x 8 of 16384 in 256 workgroups, 147 against 122.
template <int DP, bool REV, bool STATE_ONLY, bool DERIV, bool EDGE, bool AHEAD>
__global__ __launch_bounds__(DP * 4, DERIV ? 2 : AHEAD ? 3 : 4) void la_pass_bf16(Passes<passes_of(REV, STATE_ONLY, DERIV)> all_passes) {
  constexpr bool PAIR = passes_of(REV, STATE_ONLY, DERIV) == 2;
  unsigned id = blockIdx.x;
  const PassArgs& a = all_passes.a[PAIR ? (id >> 3) & 1 : 0];
  if (PAIR) {
    id = (id >> 4) * 8 + (id & 7);
    if (id >= (unsigned)(a.B * a.H * a.G)) return;  // the same for a whole workgroup
  }
  using Ch = Chunk<DP, EDGE, !STATE_ONLY>;
  constexpr int C = 64, NS = DP / 32, NT = DP / 16, LD = Ch::LD, WAVES = DP / 16;
  constexpr bool FULL = !STATE_ONLY, X = DERIV && FULL;
  __shared__ __attribute__((aligned(16))) char q_s[FULL ? Ch::BYTES : 16];
  __shared__ __attribute__((aligned(16))) char k_s[Ch::BYTES];
  __shared__ __attribute__((aligned(16))) char v_s[Ch::BYTES];
  __shared__ uint4 p_s[FULL ? 6 : 1][64];    // pair weights, as operands
  // those of a chunk without gaps, by tile distance (at head size 32 not worth
  // their room: a workgroup less a CU)
  constexpr bool TABLE = FULL && DP > 32;
  __shared__ f32x4 full_s[TABLE ? 4 : 1][64];
  __shared__ __attribute__((aligned(16))) char x_s[X ? Ch::BYTES : 16];
  // of each position: the valid ones up to it, and its weights in the product
  // with the start state and in the state's update
  __shared__ __attribute__((aligned(16))) float n_s[C], inter_s[C], update_s[C];
  __shared__ float lam[C + 1];
  __shared__ float red[WAVES];

  const int seg = id % (unsigned)a.G;
  const int64_t bh = id / (unsigned)a.G;
  const int b = bh / a.H, h = bh % a.H;
  // the wave's index is the same for its lanes, which the compiler cannot see:
  // what depends on it alone then needs no vector registers and no masks
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo = lane & 15, g = lane >> 4;
  const int e0 = wave * 16, e = e0 + lo;
  const bool busy = e0 < a.De;
  const int64_t state_size = (int64_t)a.Dc * a.De;
  const int n_chunks = (a.L + C - 1) / C;
  const int first = seg * a.seg_chunks, last = min(n_chunks, first + a.seg_chunks);
  auto start_of = [&](int step) { return (REV ? first + last - 1 - step : step) * C; };
  Ch q_r(a.q, b, h, a.Dc), k_r(a.k, b, h, a.Dc), v_r(a.v, b, h, a.De), x_r(a.x, b, h, a.De);
  // The mask is read a chunk ahead of the rows that it says to read.
  const bool* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
  auto look = [&](int step) {
    const int pos = start_of(step) + lane;
    return step < last && pos < a.L && (!mask || mask[pos * a.mask_l]);
  };
  auto fetch = [&](int step, uint64_t bits) {
    const int l0 = start_of(step);
    if (FULL) q_r.fetch(l0, bits);
    k_r.fetch(l0, bits);
    v_r.fetch(l0, bits);
    if (X) x_r.fetch(l0, bits);
  };
  // the first loads are on their way while the rest is prepared
  uint64_t bits = __ballot(look(first));
  if (AHEAD) fetch(first, bits);
  bool ahead = look(first + 1);
  const float ld = a.log_decay[h];
  // a decay of zero (log -inf) keeps l^0 = 1
  for (int i = threadIdx.x; i <= C; i += DP * 4) lam[i] = i ? expf(ld * i) : 1.f;

  // false while the state is known to be zero, as a history's first chunk has it
  bool started = FULL && (a.G > 1 || a.state_in);
  // whether the state after the last chunk is asked for
  const bool at_end = REV ? seg == 0 : seg == a.G - 1;
  const bool want_end = STATE_ONLY || (at_end && a.state_out) || (DERIV && (a.G > 1 || a.state_end_grad));
  f32x4 S[NT], Sd[DERIV ? NT : 1];
  {
    const float* src = nullptr;
    if (FULL) {
      if (a.G > 1) src = a.seg + (bh * a.G + seg) * state_size;
      else if (a.state_in) src = a.state_in + bh * state_size;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // the addresses of a tile at a time: worked out together, they take two
      // registers for each element of the state
      int g_t = g;
      asm volatile("" : "+v"(g_t)::"memory");
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int c = state_row<FULL>(t, g_t, r);
        const bool in = c < a.Dc && e < a.De;
        S[t][r] = (src && in) ? src[c * a.st_c + e * a.st_e] : 0.f;
        if (DERIV) Sd[t][r] = 0.f;
      }
    }
  }
  __syncthreads();  // lam

  if (TABLE) {
    for (int d = wave; d < 4; d += WAVES) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int gap = 16 * d + (REV ? 4 * g + r - lo : lo - 4 * g - r);
        full_s[d][lane][r] = gap >= 0 ? a.c_pair * lam[max(gap, 0)] : 0.f;
      }
    }
  }
  // Unit u: tile row it by key block s; the first four have two tiles each, the
  // last two one.  Mirrored in the reversed pass.
  auto unit_it = [](int u) { const int it = (0x203321 >> (4 * u)) & 15; return REV ? 3 - it : it; };
  auto unit_s = [](int u) { const int s = (0x101000 >> (4 * u)) & 15; return REV ? 1 - s : s; };

  __hip_bfloat16* out = nullptr;
  if (FULL)
    out = reinterpret_cast<__hip_bfloat16*>(a.out) + b * a.out_b + h * a.out_h +
          (threadIdx.x / Ch::ACROSS) * a.out_l + (threadIdx.x % Ch::ACROSS) * 8;
  // outputs of the chunk at l0 in whole rows, from LDS (where they take v's
  // place: a thread reads what it alone will overwrite) or zeros
  auto store = [&](int l0, bool zero) {
    const int row = threadIdx.x / Ch::ACROSS, left = v_r.left;
    const char* from = v_s + row * LD + (threadIdx.x % Ch::ACROSS) * 16;
#pragma unroll
    for (int i = 0; i < Ch::PIECES; ++i) {
      if (l0 + row + Ch::DOWN * i >= a.L || left <= 0) continue;
      uint4 v = {0, 0, 0, 0};
      if (!zero) v = *reinterpret_cast<const uint4*>(from + i * Ch::DOWN * LD);
      store8<EDGE>(out + (l0 + Ch::DOWN * i) * a.out_l, left, v);
    }
  };

  int total = 0;
  float d_decay = 0.f;
#pragma unroll 1
  for (int step = first; step < last; ++step) {
    const int l0 = start_of(step);
    const uint64_t now = bits;
    const int N = __popcll(now);
    total += N;
    // without valid positions nothing is seen, added or forgotten.  (One way
    // round the loop for both cases: a second one, with a continue, kept copies
    // of the state, 50 registers of it at head size 64.)
    if (N) {
      if (!AHEAD) fetch(step, now);
      if (FULL) q_r.put(q_s);
      k_r.put(k_s);
      v_r.put(v_s);
      if (X) x_r.put(x_s);
      if (wave == 0) {
        const int n = __popcll(now & ((2ull << lane) - 1));
        n_s[lane] = (float)n;
        inter_s[lane] = a.c_inter * lam[REV ? N - n : n];
        update_s[lane] = a.c_update * lam[REV ? n : N - n];
      }
      __syncthreads();
    }
    bits = __ballot(ahead);
    if (AHEAD) fetch(step + 1, bits);
    ahead = look(step + 2);

    if (N) {
      const float all = (float)N;
      if (FULL) {
        // valid positions in one run: n_i - n_j = i - j wherever a pair counts
        const uint64_t run = now >> __builtin_ctzll(now);
        const bool whole = (run & (run + 1)) == 0;
#pragma unroll 1
        for (int unit = wave; unit < 6; unit += WAVES) {
          const int it = unit_it(unit), s = unit_s(unit), i = 16 * it + lo;
          const float n_i = n_s[i];
          bf16x8 qf[NS];
#pragma unroll
          for (int c = 0; c < NS; ++c) qf[c] = Ch::rows(q_s, 16 * it, c, lo, g);
          f32x4 p[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int jt = 2 * s + u, apart = REV ? jt - it : it - jt;
            p[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (apart < 0) continue;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NS; ++c) acc = mfma32(Ch::rows(k_s, 16 * jt, c, lo, g), qf[c], acc);
            f32x4 gaps;
            if (DERIV || !TABLE || !whole) {
              const f32x4 n_j = *reinterpret_cast<const f32x4*>(n_s + 16 * jt + 4 * g);
              gaps = REV ? n_j - n_i : n_i - n_j;
            }
            if (TABLE && whole) {
              p[u] = acc * full_s[apart][lane];
            } else {
              f32x4 w;
#pragma unroll
              for (int r = 0; r < 4; ++r) w[r] = lam[max((int)gaps[r], 0)];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const bool seen = apart > 0 || (REV ? 4 * g + r >= lo : 4 * g + r <= lo);
                p[u][r] = seen ? acc[r] * (a.c_pair * w[r]) : 0.f;
              }
            }
            if (DERIV) {  // sum of gap weight (q_i.k_j) (x_i.v_j)
              asm volatile("" ::: "memory");
              f32x4 other = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int c = 0; c < NS; ++c)
                other = mfma32(Ch::rows(v_s, 16 * jt, c, lo, g), Ch::rows(x_s, 16 * it, c, lo, g), other);
#pragma unroll
              for (int r = 0; r < 4; ++r) d_decay += p[u][r] * gaps[r] * other[r];
            }
          }
          p_s[unit][lane] = __builtin_bit_cast(uint4, pack8(p[0], p[1]));
        }
      }

      bf16x8 vf[2];
      f32x4 o[FULL ? 4 : 1];
      if (busy) {
#pragma unroll
        for (int s = 0; s < 2; ++s) vf[s] = Ch::columns(v_s, e0, 4, s, lo, g);

        if (FULL) {
          // the start state's part, a block of the contraction at a time: so the
          // split state needs registers for one block only
#pragma unroll
          for (int it = 0; it < 4; ++it) o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (started) {
            f32x4 od[DERIV ? 4 : 1];
            if (DERIV) {
#pragma unroll
              for (int it = 0; it < 4; ++it) od[it] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int s = 0; s < NS; ++s) {
              asm volatile("" ::: "memory");
              const Split8<DERIV ? 3 : 2> state(S[2 * s], S[2 * s + 1]);
              const Split8<3> state_d(Sd[DERIV ? 2 * s : 0], Sd[DERIV ? 2 * s + 1 : 0]);
#pragma unroll
              for (int it = 0; it < 4; ++it) {
                if (DERIV) asm volatile("" ::: "memory");
                const bf16x8 qf = Ch::rows(q_s, 16 * it, s, lo, g);
                o[it] = state.times(qf, o[it]);
                if (DERIV) od[it] = state_d.times(qf, od[it]);
              }
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
              const int i = 16 * it + lo;
              const float w_i = inter_s[i];
              if (DERIV) {  // of the decay's gradient, x . (S' + n S) q w
                od[it] = w_i * (od[it] + n_s[i] * o[it]);
                const f32x4 xv = widen(*reinterpret_cast<const bf16x4*>(x_s + i * LD + (e0 + 4 * g) * 2));
#pragma unroll
                for (int r = 0; r < 4; ++r) d_decay += xv[r] * od[it][r];
              }
              o[it] = w_i * o[it];
            }
          }
        }
      }

      if (FULL) {
        __syncthreads();  // the pair weights are there, and v is read
        if (busy) {
#pragma unroll
          for (int u = 0; u < 6; ++u) {
            const int it = unit_it(u), s = unit_s(u);
            o[it] = mfma32(vf[s], __builtin_bit_cast(bf16x8, p_s[u][lane]), o[it]);
          }
#pragma unroll
          for (int it = 0; it < 4; ++it)
            *reinterpret_cast<bf16x4*>(v_s + (16 * it + lo) * LD + (e0 + 4 * g) * 2) =
                __builtin_convertvector(o[it], bf16x4);
        }
      }
      if (busy) {
        const bool update = want_end || step + 1 < last;
        started = true;
        if (update) {
          const float lN = lam[N];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (DERIV) Sd[t] = lN * (Sd[t] + all * S[t]);
            S[t] = lN * S[t];
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            asm volatile("" ::: "memory");
            f32x4 w[2];
            const uint4 raw = __builtin_bit_cast(uint4, vf[s]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              w[i] = widen(__builtin_bit_cast(bf16x4, i ? uint2{raw.z, raw.w} : uint2{raw.x, raw.y})) *
                     *reinterpret_cast<const f32x4*>(update_s + 32 * s + 16 * i + 4 * g);
            auto add = [&](f32x4* state) {
              const Split8<3> weighted(w[0], w[1]);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                if (!AHEAD) __builtin_amdgcn_sched_barrier(0);  // in order: fewer registers
                if (DERIV && t % 2 == 0) asm volatile("" ::: "memory");
                const bf16x8 kf = Ch::columns(k_s, state_row<FULL>(t, 0, 0), FULL ? 8 : 4, s, lo, g);
                state[t] = weighted.after(kf, state[t]);
              }
            };
            add(S);
            if (DERIV) {
              asm volatile("" ::: "memory");
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const f32x4 n_j = *reinterpret_cast<const f32x4*>(n_s + 32 * s + 16 * i + 4 * g);
                w[i] = w[i] * (REV ? n_j : all - n_j);
              }
              add(Sd);
            }
          }
        }
      }
      __syncthreads();  // the chunk is read and its outputs are in LDS
    }
    if (FULL) store(l0, N == 0);
  }

  float* dst = nullptr;
  float* dst_d = nullptr;
  if (STATE_ONLY) {
    dst = a.seg + (bh * a.G + seg) * state_size;
    if (threadIdx.x == 0) a.seg_count[bh * a.G + seg] = total;
  } else if (at_end && a.state_out) {
    dst = a.state_out + bh * state_size;
  }
  // the derivative of the end state: for the scan, or here if it ends the history
  if (X && a.G > 1) dst_d = a.seg_d + (bh * a.G + seg) * state_size;
  const float* end_grad = (X && a.G == 1 && a.state_end_grad) ? a.state_end_grad + bh * state_size : nullptr;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    int g_t = g;
    asm volatile("" : "+v"(g_t)::"memory");
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = state_row<FULL>(t, g_t, r);
      if (c < a.Dc && e < a.De) {
        const int64_t at = c * a.st_c + e * a.st_e;
        if (dst) dst[at] = S[t][r];
        if (DERIV && dst_d) dst_d[at] = Sd[t][r];
        if (DERIV && end_grad) d_decay += Sd[t][r] * end_grad[at];
      }
    }
  }
  if (X) {
    d_decay = wave_reduce_sum(d_decay);
    if (lane == 0) red[wave] = d_decay;
    __syncthreads();
    if (threadIdx.x == 0) {
      float sum = 0.f;
      for (int w = 0; w < WAVES; ++w) sum += red[w];
      a.decay_part[bh * a.parts + seg] = sum;
    }
  }
}

// Histories of at most one chunk without a state on either side, where nothing is
// carried: with w_ij = scale l^{n_i-n_j}, j <= i.  Wave w has 16 positions.
//   out_i = sum_j w_ij (x_i.y_j) z_j for the positions of wave w
template <int DP, class Ch>
__device__ __forceinline__ void short_rows(const char* x_s, const char* y_s, const char* z_s, const float* n_s,
                                           const float* lam, int wave, int lo, int g, bf16x4* out) {
  constexpr int NS = DP / 32, NT = DP / 16;
  const int own = 16 * wave;
  const float n_own = n_s[own + lo];
  f32x4 o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16x8 xf[NS];
#pragma unroll
  for (int c = 0; c < NS; ++c) xf[c] = Ch::rows(x_s, own, c, lo, g);
#pragma unroll 1
  for (int s = 0; 2 * s <= wave; ++s) {
    f32x4 p[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j0 = 16 * (2 * s + u);
      p[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (j0 > own) continue;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NS; ++c) acc = mfma32(Ch::rows(y_s, j0, c, lo, g), xf[c], acc);
      const f32x4 gaps = n_own - *reinterpret_cast<const f32x4*>(n_s + j0 + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        p[u][r] = j0 < own || 4 * g + r <= lo ? acc[r] * lam[max((int)gaps[r], 0)] : 0.f;
    }
    const bf16x8 pf = pack8(p[0], p[1]);
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = mfma32(Ch::columns(z_s, 16 * t, 4, s, lo, g), pf, o[t]);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) out[t] = __builtin_convertvector(o[t], bf16x4);
}

// rows [0, L) of an LDS tile to [B, H, L, D] memory, 16 bytes a thread
template <bool EDGE, class Ch>
__device__ __forceinline__ void short_store(const char* from, const Rows& dst, int b, int h, int L, int D) {
  const int row = threadIdx.x / Ch::ACROSS, d = (threadIdx.x % Ch::ACROSS) * 8;
  __hip_bfloat16* out = reinterpret_cast<__hip_bfloat16*>(const_cast<void*>(dst.p)) + b * dst.b + h * dst.h + d;
#pragma unroll
  for (int i = 0; i < Ch::PIECES; ++i) {
    const int l = row + i * Ch::DOWN;
    if (l < L && d < D)
      store8<EDGE>(out + l * dst.l, D - d, *reinterpret_cast<const uint4*>(from + l * Ch::LD + d * 2));
  }
}

// The forward pass of them, out = (w o q k^T) v.
template <int DP, bool EDGE>
__global__ __launch_bounds__(256, 4) void la_short_fwd(ShortArgs a) {
  using Ch = Chunk<DP, EDGE, true, 256>;
  constexpr int NT = DP / 16;
  // the outputs take the place of q, whose rows a wave reads alone
  __shared__ __attribute__((aligned(16))) char q_s[Ch::BYTES], k_s[Ch::BYTES], v_s[Ch::BYTES];
  __shared__ __attribute__((aligned(16))) float n_s[Ch::C];
  __shared__ float lam[Ch::C];
  const int64_t bh = blockIdx.x;
  const int b = bh / a.H, h = bh % a.H;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo = lane & 15, g = lane >> 4;
  const uint64_t bits = __ballot(lane < a.L && (!a.mask || a.mask[b * a.mask_b + lane * a.mask_l]));
  {
    Ch q_r(a.q, b, h, a.Dk), k_r(a.k, b, h, a.Dk), v_r(a.v, b, h, a.Dv);
    q_r.fetch(0, bits);
    k_r.fetch(0, bits);
    v_r.fetch(0, bits);
    if (wave == 0) {
      n_s[lane] = (float)__popcll(bits & ((2ull << lane) - 1));
      lam[lane] = a.scale * (lane ? expf(a.log_decay[h] * lane) : 1.f);
    }
    q_r.put(q_s);
    k_r.put(k_s);
    v_r.put(v_s);
  }
  __syncthreads();
  if (16 * wave < a.L) {
    bf16x4 o[NT];
    short_rows<DP, Ch>(q_s, k_s, v_s, n_s, lam, wave, lo, g, o);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      *reinterpret_cast<bf16x4*>(q_s + (16 * wave + lo) * Ch::LD + (16 * t + 4 * g) * 2) = o[t];
  }
  __syncthreads();
  short_store<EDGE, Ch>(q_s, a.out, b, h, a.L, a.Dv);
}

// All gradients of them, each tensor read once:
//   A_ij = w_ij q_i.k_j          B_ij = w_ij dO_i.v_j
//   dq = B k       dk = B^T q       dv = A^T dO
//   the decay's: sum (n_i - n_j) A_ij (dO_i.v_j)
// A wave has its positions as queries for dq and as keys for dk and dv, so that
// no pair weight is another wave's and the work is about even (w + 1 and 4 - w
// tiles of pairs).  The products that a transposed operand needs are worked out
// again, transposed.
template <int DP, bool EDGE>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 4) void la_short_bwd(ShortArgs a) {
  using Ch = Chunk<DP, EDGE, true, 256>;
  constexpr int C = 64, NS = DP / 32, NT = DP / 16, LD = Ch::LD;
  // dq, dk and dv take the places of q, k and v
  __shared__ __attribute__((aligned(16))) char q_s[Ch::BYTES], k_s[Ch::BYTES], v_s[Ch::BYTES], g_s[Ch::BYTES];
  __shared__ __attribute__((aligned(16))) float n_s[C];
  __shared__ float lam[C];
  __shared__ float red[4];

  const int64_t bh = blockIdx.x;
  const int b = bh / a.H, h = bh % a.H;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo = lane & 15, g = lane >> 4;
  const uint64_t bits = __ballot(lane < a.L && (!a.mask || a.mask[b * a.mask_b + lane * a.mask_l]));
  {
    Ch q_r(a.q, b, h, a.Dk), k_r(a.k, b, h, a.Dk), v_r(a.v, b, h, a.Dv), g_r(a.dout, b, h, a.Dv);
    q_r.fetch(0, bits);
    k_r.fetch(0, bits);
    v_r.fetch(0, bits);
    g_r.fetch(0, bits);
    if (wave == 0) {
      n_s[lane] = (float)__popcll(bits & ((2ull << lane) - 1));
      lam[lane] = a.scale * (lane ? expf(a.log_decay[h] * lane) : 1.f);
    }
    q_r.put(q_s);
    k_r.put(k_s);
    v_r.put(v_s);
    g_r.put(g_s);
  }
  __syncthreads();

  const int tiles = (a.L + 15) / 16, own = 16 * wave;
  bf16x4 dq[NT], dk[NT], dv[NT];
  float d_decay = 0.f;
  if (wave < tiles) {
    const float n_own = n_s[own + lo];
    short_rows<DP, Ch>(g_s, v_s, k_s, n_s, lam, wave, lo, g, dq);
    f32x4 o[NT], o2[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = o2[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    bf16x8 kf[NS], vf[NS];
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      kf[c] = Ch::rows(k_s, own, c, lo, g);
      vf[c] = Ch::rows(v_s, own, c, lo, g);
    }
#pragma unroll 1
    for (int s = wave / 2; 2 * s < tiles; ++s) {
      f32x4 p[2], p2[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i0 = 16 * (2 * s + u);
        p[u] = p2[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (i0 < own) continue;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f}, acc2 = acc;
#pragma unroll
        for (int c = 0; c < NS; ++c) {
          acc = mfma32(Ch::rows(q_s, i0, c, lo, g), kf[c], acc);
          acc2 = mfma32(Ch::rows(g_s, i0, c, lo, g), vf[c], acc2);
        }
        const f32x4 gaps = *reinterpret_cast<const f32x4*>(n_s + i0 + 4 * g) - n_own;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = i0 > own || 4 * g + r >= lo ? lam[max((int)gaps[r], 0)] : 0.f;
          p[u][r] = acc[r] * w;
          p2[u][r] = acc2[r] * w;
          d_decay += p[u][r] * gaps[r] * acc2[r];
        }
      }
      const bf16x8 pf = pack8(p[0], p[1]), pf2 = pack8(p2[0], p2[1]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        o[t] = mfma32(Ch::columns(g_s, 16 * t, 4, s, lo, g), pf, o[t]);
        o2[t] = mfma32(Ch::columns(q_s, 16 * t, 4, s, lo, g), pf2, o2[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      dv[t] = __builtin_convertvector(o[t], bf16x4);
      dk[t] = __builtin_convertvector(o2[t], bf16x4);
    }
  }
  d_decay = wave_reduce_sum(d_decay);
  if (lane == 0) red[wave] = d_decay;
  __syncthreads();  // q, k, v are read
  if (wave < tiles) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int at = (own + lo) * LD + (16 * t + 4 * g) * 2;
      *reinterpret_cast<bf16x4*>(q_s + at) = dq[t];
      *reinterpret_cast<bf16x4*>(k_s + at) = dk[t];
      *reinterpret_cast<bf16x4*>(v_s + at) = dv[t];
    }
  }
  __syncthreads();
  short_store<EDGE, Ch>(q_s, a.dq, b, h, a.L, a.Dk);
  short_store<EDGE, Ch>(k_s, a.dk, b, h, a.L, a.Dk);
  short_store<EDGE, Ch>(v_s, a.dv, b, h, a.L, a.Dv);
  if (threadIdx.x == 0 && a.decay_part) a.decay_part[bh] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Contributions of the segments -> start states, in place, one thread for
// each element of a state.
template <bool REV>
__global__ void la_scan(float* seg, const int* count, const float* state_in, const float* log_decay,
                        int H, int G, int64_t state_size) {
  const int64_t bh = blockIdx.x;
  const float ld = log_decay[bh % H];
  for (int64_t at = threadIdx.x + (int64_t)blockIdx.y * blockDim.x; at < state_size;
       at += (int64_t)gridDim.y * blockDim.x) {
    float run = state_in ? state_in[bh * state_size + at] : 0.f;
    for (int s = 0; s < G; ++s) {
      const int64_t i = bh * G + (REV ? G - 1 - s : s);
      const int N = count[i];
      const float own = seg[i * state_size + at];
      seg[i * state_size + at] = run;
      run = (N ? expf(ld * N) : 1.f) * run + own;
    }
  }
}

// What the start states' own derivatives add to the decay's gradient: the sum
// over the segments of <S'_start, V>, and <S'_end, dL/dS_end>; a partial sum for
// each workgroup of 256 elements.  seg_v: the contributions V.
__global__ __launch_bounds__(256) void la_scan_decay(const float* seg_d, const float* seg_v,
                                                     const int* count, const float* end_grad,
                                                     const float* log_decay, float* part, int parts,
                                                     int first_part, int H, int G, int64_t state_size) {
  __shared__ float red[4];
  const int64_t bh = blockIdx.x, at = threadIdx.x + (int64_t)blockIdx.y * 256;
  const float ld = log_decay[bh % H];
  float run = 0.f, sum = 0.f;
  if (at < state_size) {
    for (int s = 0; s < G; ++s) {
      const int64_t i = bh * G + s;
      const int N = count[i];
      sum += run * seg_v[i * state_size + at];
      run = (N ? expf(ld * N) : 1.f) * run + seg_d[i * state_size + at];
    }
    if (end_grad) sum += run * end_grad[bh * state_size + at];
  }
  sum = wave_reduce_sum(sum);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[bh * parts + first_part + blockIdx.y] = (red[0] + red[1]) + (red[2] + red[3]);
}

// part [B, H, parts] -> [H]; a fixed order, in 64 bits (the parts may cancel).
__global__ __launch_bounds__(1024) void la_decay_sum(const float* part, float* out, int B, int H, int parts) {
  __shared__ double red[16];
  const int h = blockIdx.x;
  const int64_t n = (int64_t)B * parts;
  double sum = 0.0;
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += 8 * 1024) {
    float v[8];  // in flight together: this is all latency
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = i0 + j * 1024;
      v[j] = i < n ? part[((i / parts) * H + h) * parts + i % parts] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, WAVE);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < 16; ++w) all += red[w];
    out[h] = (float)all;
  }
}

// One position for each row: the state is read, updated and written once, and
// that is the bound.  A wave takes 4 LE columns of one (batch, head): LE lanes
// with four neighbours each across, 64 / LE groups of rows down, BATCH rows of
// a group in flight; the groups' outputs meet in two or three shuffles.  No
// LDS and no barrier: 4096 x 4 states of 64 x 64 in 80 us (6.7 TB/s, the
// last-level cache keeping a part of the 268 MB; a loop of one column a
// thread: 253).  EDGE: any head sizes, else whole batches.
template <typename T, int LE, int BATCH, bool EDGE>
__global__ __launch_bounds__(256) void la_step_kernel(Rows q, Rows k, Rows v, const float* log_decay,
                                                      float* state, int64_t st_b, int64_t st_h,
                                                      const bool* active, int64_t act_b, T* out,
                                                      int64_t waves, int H, int Dk, int Dv, float scale) {
  constexpr int RG = 64 / LE;
  const int lane = threadIdx.x & 63, rg = lane / LE;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wave >= waves) return;
  const int across = (Dv + 4 * LE - 1) / (4 * LE);
  const int64_t bh = wave / across;
  const int b = bh / H, h = bh % H;
  const int e = (int)(wave % across) * 4 * LE + (lane % LE) * 4, n = EDGE ? Dv - e : 4;
  T* o = out + bh * Dv + e;
  float sum[4] = {};
  if (!active || active[b * act_b]) {
    const float l = expf(log_decay[h]);
    const T* qr = reinterpret_cast<const T*>(q.p) + b * q.b + h * q.h;
    const T* kr = reinterpret_cast<const T*>(k.p) + b * k.b + h * k.h;
    const T* vr = reinterpret_cast<const T*>(v.p) + b * v.b + h * v.h;
    float* S = state + b * st_b + h * st_h + e;
    float ve[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ve[i] = i < n ? to_f32<T>(vr[e + i]) : 0.f;
    const int rows = (Dk + RG - 1) / RG, row0 = rg * rows, row_end = min(Dk, row0 + rows);
    if (n > 0) {
      for (int c0 = row0; c0 < row_end; c0 += BATCH) {
        f32x4 st[BATCH];
        T kc[BATCH], qc[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const float* at = S + (int64_t)(c0 + i) * Dv;
          if (!EDGE || (c0 + i < row_end && n >= 4)) {
            __builtin_memcpy(&st[i], at, 16);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) st[i][j] = (c0 + i < row_end && j < n) ? at[j] : 0.f;
          }
        }
        if (!EDGE) {
          __builtin_memcpy(kc, kr + c0, BATCH * sizeof(T));
          __builtin_memcpy(qc, qr + c0, BATCH * sizeof(T));
        } else {
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            kc[i] = c0 + i < row_end ? kr[c0 + i] : from_f32<T>(0.f);
            qc[i] = c0 + i < row_end ? qr[c0 + i] : from_f32<T>(0.f);
          }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          if (EDGE && c0 + i >= row_end) continue;
          const float ki = to_f32<T>(kc[i]), qi = to_f32<T>(qc[i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            st[i][j] = l * st[i][j] + ki * ve[j];
            sum[j] += qi * st[i][j];
          }
          float* at = S + (int64_t)(c0 + i) * Dv;
          if (!EDGE || n >= 4) {
            __builtin_memcpy(at, &st[i], 16);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < n) at[j] = st[i][j];
          }
        }
      }
    }
#pragma unroll
    for (int off = LE; off < 64; off *= 2)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += __shfl_xor(sum[j], off, WAVE);
  }
  if (rg == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!EDGE || j < n) o[j] = from_f32<T>(scale * sum[j]);
  }
}

// ---------------------------------------------------------------------------

Rows rows_of(const torch::Tensor& t) {
  return {t.data_ptr(), t.stride(0), t.stride(1), t.dim() == 4 ? t.stride(2) : 0};
}

int padded(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

struct Split {
  int G, seg_chunks;
};

// Positions of one load: bfloat16's pass takes 64; float16 shares float32's, which
// holds everything in float32 (a state is past float16's own range).
int chunk_of(torch::ScalarType dt) { return dt == torch::kBFloat16 ? 64 : 32; }

// One workgroup for each (batch, head) where these alone fill the card (two a
// CU; one, of 8 waves, of bfloat16's at head sizes past 64); else the history is
// cut until there are about that many, in segments of at least 256 positions (64
// of the slower float32 pass), so that the state-only pass and the scan stay
// small beside the work they split.  Forward / backward, by segments: 2 x 8 heads
// of 16384 at head size 128 in 4, 380 us, 8, 203, 16 (taken), 124 / 360, 32, 117 /
// 372, 64, 135 / 464; 8 x 8 of 4096 at 64 in 4, 70 / 166, 8 (taken), 53 / 145, 16,
// 59 / 157; float32, 33 x 3 of 333 at 48 in 1, 57, 2, 54, 4 (taken), 37, 11, 38;
// float16, 6 x 2 of 12878 at 88 in 22, 375 / 1038, 41 (taken), 216 / 655, 81,
// 232 / 703.
Split split_of(int64_t BH, int64_t L, int64_t D, int C) {
  const int64_t chunks = (L + C - 1) / C, want = D > 64 && C == 64 ? 256 : 512;
  int64_t G = BH ? std::min<int64_t>((want + BH - 1) / BH, chunks / (C == 64 ? 4 : 2)) : 1;
  G = std::max<int64_t>(G, 1);
  const int64_t per = std::max<int64_t>((chunks + G - 1) / G, 1);
  return {(int)std::max<int64_t>((chunks + per - 1) / per, 1), (int)per};
}

template <bool REV, bool STATE_ONLY, bool DERIV>
void launch_pass(torch::ScalarType dt, const Passes<passes_of(REV, STATE_ONLY, DERIV)>& p, hipStream_t stream) {
  const PassArgs& a = p.a[0];
  int64_t blocks = (int64_t)a.B * a.H * a.G;
  if (passes_of(REV, STATE_ONLY, DERIV) == 2) blocks = (blocks + 7) / 8 * 16;
  TORCH_CHECK(blocks < (int64_t(1) << 31), "linear attention: too many (batch, head, segment)s");
  const int dp = padded(std::max(a.Dc, a.De));
  const bool edge = a.Dc % 8 || a.De % 8;
#define LA_LAUNCH(DP, ...)                                                                     \
  hipLaunchKernelGGL((__VA_ARGS__), dim3((unsigned)blocks), dim3(DP * 4), 0, stream, p)
#define LA_BF16(DP, AHEAD)                                                                     \
  do {                                                                                         \
    if (edge) LA_LAUNCH(DP, la_pass_bf16<DP, REV, STATE_ONLY, DERIV, true, AHEAD>);            \
    else LA_LAUNCH(DP, la_pass_bf16<DP, REV, STATE_ONLY, DERIV, false, AHEAD>);                \
  } while (0)
#define LA_F32(DP)                                                                             \
  do {                                                                                         \
    if (dt == torch::kHalf) LA_LAUNCH(DP, la_pass_f32<__half, DP, REV, STATE_ONLY, DERIV>);    \
    else LA_LAUNCH(DP, la_pass_f32<float, DP, REV, STATE_ONLY, DERIV>);                        \
  } while (0)
  if (dt == torch::kBFloat16) {
    if (dp == 32) LA_BF16(32, true);
    else if (dp == 64) LA_BF16(64, true);
    else if (STATE_ONLY || DERIV || edge || blocks <= 256) LA_BF16(128, true);
    else if constexpr (!STATE_ONLY && !DERIV)
      LA_LAUNCH(128, la_pass_bf16<128, REV, false, false, false, false>);
  } else {
    if (dp == 32) LA_F32(32);
    else if (dp == 64) LA_F32(64);
    else LA_F32(128);
  }
#undef LA_BF16
#undef LA_F32
#undef LA_LAUNCH
  HIP_CHECK(hipGetLastError());
}

template <bool REV>
void launch_scan(const PassArgs& a, const float* state_in, hipStream_t stream) {
  const int64_t size = (int64_t)a.Dc * a.De;
  hipLaunchKernelGGL((la_scan<REV>), dim3((unsigned)(a.B * a.H), (unsigned)((size + 255) / 256)),
                     dim3(256), 0, stream, a.seg, a.seg_count, state_in, a.log_decay, a.H, a.G, size);
  HIP_CHECK(hipGetLastError());
}

// The kernels read any strides but the last dimension's.
torch::Tensor unit_stride(const torch::Tensor& t) {
  return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

void check_inputs(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                  const torch::Tensor& log_decay, const c10::optional<torch::Tensor>& mask,
                  const c10::optional<torch::Tensor>& state, int dim) {
  const auto dt = q.scalar_type();
  TORCH_CHECK(q.is_cuda(), "linear attention: q must be on the GPU");
  TORCH_CHECK(dt == torch::kBFloat16 || dt == torch::kHalf || dt == torch::kFloat32,
              "linear attention: q, k, v must be bfloat16, float16 or float32");
  TORCH_CHECK(q.dim() == dim && k.dim() == dim && v.dim() == dim, "linear attention: q, k, v need ",
              dim, " dimensions");
  for (const auto& t : {q, k, v}) {
    TORCH_CHECK(t.scalar_type() == dt && t.device() == q.device(),
                "linear attention: q, k, v must share type and device");
    for (int i = 0; i < dim - 1; ++i)
      TORCH_CHECK(t.size(i) == q.size(i), "linear attention: q, k, v differ in dimension ", i);
  }
  TORCH_CHECK(k.size(-1) == q.size(-1), "linear attention: q and k differ in head size");
  TORCH_CHECK(q.size(-1) >= 1 && q.size(-1) <= 128 && v.size(-1) >= 1 && v.size(-1) <= 128,
              "linear attention: head sizes from 1 to 128");
  for (int i = 0; i < dim - 1; ++i)
    TORCH_CHECK(q.size(i) < (int64_t(1) << 31) - 256, "linear attention: dimension ", i, " is too large");
  TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == q.size(1) &&
                  log_decay.scalar_type() == torch::kFloat32 && log_decay.device() == q.device(),
              "linear attention: log_decay must be float32 [H] on the same device");
  if (mask.has_value()) {
    TORCH_CHECK(mask->scalar_type() == torch::kBool && mask->device() == q.device() &&
                    mask->size(0) == q.size(0) && mask->dim() == dim - 2 &&
                    (dim == 3 || mask->size(1) == q.size(2)),
                "linear attention: the mask must be bool over the positions, on the same device");
  }
  if (state.has_value()) {
    TORCH_CHECK(state->scalar_type() == torch::kFloat32 && state->device() == q.device() &&
                    state->dim() == 4 && state->size(0) == q.size(0) && state->size(1) == q.size(1) &&
                    state->size(2) == q.size(-1) && state->size(3) == v.size(-1),
                "linear attention: the state must be float32 [B, H, Dk, Dv] on the same device");
  }
}

// The kernels carry no forward-mode tangents: a dual tensor is refused, since its
// tangent would be lost.
template <typename... Ts>
void check_no_tangent(const Ts&... given) {
  auto has = [](const c10::optional<torch::Tensor>& t) { return t.has_value() && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!(has(given) || ...), "linear attention: not differentiable in forward mode on the GPU");
}

// [B, L, H, D] memory behind a [B, H, L, D] view: what the next projection
// reads needs no copy.
torch::Tensor heads_last(const torch::Tensor& q, int64_t D) {
  return torch::empty({q.size(0), q.size(2), q.size(1), D}, q.options()).transpose(1, 2);
}

PassArgs args_of(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                 const torch::Tensor& log_decay, const c10::optional<torch::Tensor>& mask, bool flip) {
  PassArgs a = {};
  a.q = rows_of(q);
  a.k = rows_of(k);
  a.v = rows_of(v);
  a.log_decay = log_decay.data_ptr<float>();
  if (mask.has_value()) {
    a.mask = mask->data_ptr<bool>();
    a.mask_b = mask->stride(0);
    a.mask_l = mask->stride(1);
  }
  a.B = q.size(0);
  a.H = q.size(1);
  a.L = q.size(2);
  a.Dc = q.size(3);
  a.De = v.size(3);
  // a state lies in memory as [Dk, Dv]; flipped passes contract over Dv
  a.st_c = flip ? 1 : a.De;
  a.st_e = flip ? a.Dc : 1;
  a.G = 1;
  return a;
}

void set_out(PassArgs& a, const torch::Tensor& out) {
  a.out = out.data_ptr();
  a.out_b = out.stride(0);
  a.out_h = out.stride(1);
  a.out_l = out.stride(2);
}

// One chunk and no state: nothing to carry.  us, with the general passes and
// without: 8192 x 2 heads of 50 at head size 32, forward 47 and 33, backward 183 (10
// tensors read and 3 written in three passes; 4 and 3 here) and 80.
bool is_short(const torch::Tensor& q, bool states) {
  return q.scalar_type() == torch::kBFloat16 && q.size(2) <= 64 && !states;
}

ShortArgs short_args(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                     const torch::Tensor& log_decay, const c10::optional<torch::Tensor>& mask, double scale) {
  TORCH_CHECK(q.size(0) * q.size(1) < (int64_t(1) << 31), "linear attention: too many (batch, head)s");
  ShortArgs a = {};
  a.q = rows_of(q);
  a.k = rows_of(k);
  a.v = rows_of(v);
  a.log_decay = log_decay.data_ptr<float>();
  if (mask.has_value()) {
    a.mask = mask->data_ptr<bool>();
    a.mask_b = mask->stride(0);
    a.mask_l = mask->stride(1);
  }
  a.scale = (float)scale;
  a.H = q.size(1);
  a.L = q.size(2);
  a.Dk = q.size(3);
  a.Dv = v.size(3);
  return a;
}

#define LA_SHORT_DP(KERNEL, DP)                                                                      \
  do {                                                                                               \
    const dim3 grid((unsigned)(B * H));                                                              \
    if (Dk % 8 || Dv % 8) hipLaunchKernelGGL((KERNEL<DP, true>), grid, dim3(256), 0, stream, a);     \
    else hipLaunchKernelGGL((KERNEL<DP, false>), grid, dim3(256), 0, stream, a);                     \
  } while (0)
#define LA_SHORT(KERNEL)                                   \
  do {                                                     \
    const int dp = padded(std::max(Dk, Dv));               \
    if (dp == 32) LA_SHORT_DP(KERNEL, 32);                 \
    else if (dp == 64) LA_SHORT_DP(KERNEL, 64);            \
    else LA_SHORT_DP(KERNEL, 128);                         \
    HIP_CHECK(hipGetLastError());                          \
  } while (0)

}  // namespace

// -> {out, state or empty, start states of the segments or empty}
std::vector<torch::Tensor> linear_attention_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                                torch::Tensor log_decay,
                                                c10::optional<torch::Tensor> mask,
                                                c10::optional<torch::Tensor> state, double scale,
                                                bool want_state) {
  check_inputs(q, k, v, log_decay, mask, state, 4);
  check_no_tangent(q, k, v, log_decay, state);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto stream = at::cuda::getCurrentHIPStream();
  q = unit_stride(q);
  k = unit_stride(k);
  v = unit_stride(v);
  log_decay = log_decay.contiguous();
  if (state.has_value()) state = state->contiguous();
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), Dk = q.size(3), Dv = v.size(3);
  auto f32 = q.options().dtype(torch::kFloat32);
  auto out = heads_last(q, Dv);
  auto end = want_state ? torch::empty({B, H, Dk, Dv}, f32) : torch::empty({0}, f32);
  auto seg = torch::empty({0}, f32);
  if (B * H == 0) return {out, end, seg};
  if (is_short(q, state.has_value() || want_state)) {
    ShortArgs a = short_args(q, k, v, log_decay, mask, scale);
    a.out = rows_of(out);
    LA_SHORT(la_short_fwd);
    return {out, end, seg};
  }

  PassArgs a = args_of(q, k, v, log_decay, mask, false);
  set_out(a, out);
  const Split s = split_of(B * H, L, std::max(Dk, Dv), chunk_of(q.scalar_type()));
  a.G = s.G;
  a.seg_chunks = s.seg_chunks;
  a.state_in = state.has_value() ? state->data_ptr<float>() : nullptr;
  a.state_out = want_state ? end.data_ptr<float>() : nullptr;
  a.c_pair = a.c_inter = (float)scale;
  a.c_update = 1.f;
  torch::Tensor count;
  if (a.G > 1) {
    seg = torch::empty({B, H, a.G, Dk, Dv}, f32);
    count = torch::empty({B, H, a.G}, q.options().dtype(torch::kInt32));
    a.seg = seg.data_ptr<float>();
    a.seg_count = count.data_ptr<int>();
    launch_pass<false, true, false>(q.scalar_type(), {{a}}, stream);
    launch_scan<false>(a, a.state_in, stream);
  }
  launch_pass<false, false, false>(q.scalar_type(), {{a}}, stream);
  return {out, end, seg};
}

// -> {dq, dk, dv, dlog_decay or empty, dstate0 or empty}; seg: what the
// forward pass returned (start states of the segments), or empty
std::vector<torch::Tensor> linear_attention_bwd(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor log_decay,
    c10::optional<torch::Tensor> mask, c10::optional<torch::Tensor> state, torch::Tensor dout,
    c10::optional<torch::Tensor> dstate, torch::Tensor seg, double scale, bool need_decay,
    bool need_state) {
  check_inputs(q, k, v, log_decay, mask, state, 4);
  check_inputs(q, k, dout, log_decay, mask, dstate, 4);
  TORCH_CHECK(dout.size(3) == v.size(3), "linear attention: dout differs from v in head size");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto stream = at::cuda::getCurrentHIPStream();
  q = unit_stride(q);
  k = unit_stride(k);
  v = unit_stride(v);
  dout = unit_stride(dout);
  log_decay = log_decay.contiguous();
  if (state.has_value()) state = state->contiguous();
  if (dstate.has_value()) dstate = dstate->contiguous();
  const int64_t B = q.size(0), H = q.size(1), L = q.size(2), Dk = q.size(3), Dv = v.size(3);
  const auto dt = q.scalar_type();
  auto f32 = q.options().dtype(torch::kFloat32);
  auto dq = heads_last(q, Dk), dk = heads_last(q, Dk), dv = heads_last(q, Dv);
  auto ddecay = need_decay ? torch::empty({H}, f32) : torch::empty({0}, f32);
  auto ds0 = need_state ? torch::empty({B, H, Dk, Dv}, f32) : torch::empty({0}, f32);
  if (B * H == 0) {
    if (need_decay) ddecay.zero_();
    return {dq, dk, dv, ddecay, ds0};
  }
  if (is_short(q, state.has_value() || dstate.has_value() || need_state)) {
    ShortArgs a = short_args(q, k, v, log_decay, mask, scale);
    a.dout = rows_of(dout);
    a.dq = rows_of(dq);
    a.dk = rows_of(dk);
    a.dv = rows_of(dv);
    auto part = torch::empty({need_decay ? B * H : 0}, f32);
    a.decay_part = need_decay ? part.data_ptr<float>() : nullptr;
    LA_SHORT(la_short_bwd);
    if (need_decay) {
      hipLaunchKernelGGL(la_decay_sum, dim3((unsigned)H), dim3(1024), 0, stream, a.decay_part,
                         ddecay.data_ptr<float>(), (int)B, (int)H, 1);
      HIP_CHECK(hipGetLastError());
    }
    return {dq, dk, dv, ddecay, ds0};
  }
  const Split s = split_of(B * H, L, std::max(Dk, Dv), chunk_of(q.scalar_type()));
  const bool split = s.G > 1;
  TORCH_CHECK(!split || (seg.dim() == 5 && seg.size(2) == s.G && seg.is_contiguous()),
              "linear attention: the forward pass's segment states are missing");
  const float* state_in = state.has_value() ? state->data_ptr<float>() : nullptr;
  const float* dstate_in = dstate.has_value() ? dstate->data_ptr<float>() : nullptr;
  torch::Tensor count, part, seg_d, seg_r;
  if (split) count = torch::empty({B, H, s.G}, q.options().dtype(torch::kInt32));

  // the reversed passes: dv with the state's gradient, and dk
  PassArgs v_args = args_of(k, q, dout, log_decay, mask, false);
  set_out(v_args, dv);
  v_args.G = s.G;
  v_args.seg_chunks = s.seg_chunks;
  v_args.state_in = dstate_in;
  v_args.state_out = need_state ? ds0.data_ptr<float>() : nullptr;
  v_args.c_pair = v_args.c_update = (float)scale;
  v_args.c_inter = 1.f;
  if (split) {
    seg_r = torch::empty_like(seg);
    v_args.seg = seg_r.data_ptr<float>();
    v_args.seg_count = count.data_ptr<int>();
    launch_pass<true, true, false>(dt, {{v_args}}, stream);
  }

  {  // dq, and the decay's gradient
    PassArgs a = args_of(dout, v, k, log_decay, mask, true);
    set_out(a, dq);
    a.G = s.G;
    a.seg_chunks = s.seg_chunks;
    a.state_in = state_in;
    a.state_end_grad = dstate_in;
    a.c_pair = a.c_inter = (float)scale;
    a.c_update = 1.f;
    a.x = rows_of(q);
    if (split) a.seg = seg.data_ptr<float>();
    if (need_decay) {
      // partial sums: one for each workgroup of the pass and of the scan
      const int64_t blocks = split ? (Dk * Dv + 255) / 256 : 0;
      a.parts = (int)(s.G + blocks);
      part = torch::empty({B, H, a.parts}, f32);
      a.decay_part = part.data_ptr<float>();
      if (split) {
        seg_d = torch::empty_like(seg);
        a.seg_d = seg_d.data_ptr<float>();
      }
      launch_pass<false, false, true>(dt, {{a}}, stream);
      if (split) {
        hipLaunchKernelGGL(la_scan_decay, dim3((unsigned)(B * H), (unsigned)blocks), dim3(256), 0, stream,
                           a.seg_d, v_args.seg, v_args.seg_count, dstate_in, a.log_decay, a.decay_part,
                           a.parts, s.G, (int)H, s.G, Dk * Dv);
        HIP_CHECK(hipGetLastError());
      }
      hipLaunchKernelGGL(la_decay_sum, dim3((unsigned)H), dim3(1024), 0, stream,
                         part.data_ptr<float>(), ddecay.data_ptr<float>(), (int)B, (int)H, a.parts);
      HIP_CHECK(hipGetLastError());
    } else {
      launch_pass<false, false, false>(dt, {{a}}, stream);
    }
  }

  if (split) launch_scan<true>(v_args, dstate_in, stream);
  PassArgs c = args_of(v, dout, q, log_decay, mask, true);
  set_out(c, dk);
  c.G = s.G;
  c.seg_chunks = s.seg_chunks;
  c.state_in = dstate_in;
  c.seg = v_args.seg;
  c.c_pair = c.c_update = (float)scale;
  c.c_inter = 1.f;
  launch_pass<true, false, false>(dt, {{v_args, c}}, stream);
  return {dq, dk, dv, ddecay, ds0};
}

torch::Tensor linear_attention_step(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                    torch::Tensor log_decay, torch::Tensor state,
                                    c10::optional<torch::Tensor> active, double scale) {
  check_inputs(q, k, v, log_decay, active, state, 3);
  check_no_tangent(q, k, v, log_decay, state);
  const int64_t B = q.size(0), H = q.size(1), Dk = q.size(2), Dv = v.size(2);
  TORCH_CHECK((Dv <= 1 || state.stride(3) == 1) && (Dk <= 1 || state.stride(2) == Dv),
              "linear attention: each head's state must be contiguous");
  if (!state.is_contiguous() && state.numel()) {
    // the blocks in the order of the smaller stride, then the larger: each step
    // has to pass what lies below it
    const int in = B > 1 && (H <= 1 || state.stride(0) < state.stride(1)) ? 0 : 1, outer = 1 - in;
    int64_t reach = Dk * Dv;
    for (int i : {in, outer}) {
      if (state.size(i) <= 1) continue;
      TORCH_CHECK(state.stride(i) >= reach, "linear attention: blocks of the state overlap in memory");
      reach += state.stride(i) * (state.size(i) - 1);
    }
  }
  TORCH_CHECK(B * H < (int64_t(1) << 31), "linear attention: too many (batch, head)s");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  auto stream = at::cuda::getCurrentHIPStream();
  q = unit_stride(q);
  k = unit_stride(k);
  v = unit_stride(v);
  log_decay = log_decay.contiguous();
  auto out = torch::empty({B, H, Dv}, q.options());
  if (B * H == 0) return out;
  const bool* act = active.has_value() ? active->data_ptr<bool>() : nullptr;
  const int64_t act_b = active.has_value() ? active->stride(0) : 0;
  // 16 lanes across, 8 for heads of up to 32 values; batches of 16 rows where
  // the rows of a group fill them, else 4
  const int LE = Dv > 32 ? 16 : 8, RG = 64 / LE;
  const int64_t waves = B * H * ((Dv + 4 * LE - 1) / (4 * LE));
  const bool cols = Dv % (4 * LE) == 0;
  const bool whole16 = cols && Dk % (RG * 16) == 0, whole4 = cols && Dk % (RG * 4) == 0;
  TORCH_CHECK(waves / 4 < (int64_t(1) << 31), "linear attention: too many (batch, head)s");
#define LA_STEP(T, LE, BATCH, EDGE)                                                              \
  hipLaunchKernelGGL((la_step_kernel<T, LE, BATCH, EDGE>), dim3((unsigned)((waves + 3) / 4)),    \
                     dim3(256), 0, stream, rows_of(q), rows_of(k), rows_of(v),                   \
                     log_decay.data_ptr<float>(), state.data_ptr<float>(), state.stride(0),      \
                     state.stride(1), act, act_b, reinterpret_cast<T*>(out.data_ptr()), waves,   \
                     (int)H, (int)Dk, (int)Dv, (float)scale)
#define LA_STEP_T(T)                                                                             \
  do {                                                                                           \
    if (LE == 16 && whole16) LA_STEP(T, 16, 16, false);                                          \
    else if (LE == 16 && whole4) LA_STEP(T, 16, 4, false);                                       \
    else if (LE == 16) LA_STEP(T, 16, 8, true);                                                  \
    else if (whole16) LA_STEP(T, 8, 16, false);                                                  \
    else if (whole4) LA_STEP(T, 8, 4, false);                                                    \
    else LA_STEP(T, 8, 8, true);                                                                 \
  } while (0)
  if (q.scalar_type() == torch::kBFloat16) LA_STEP_T(__hip_bfloat16);
  else if (q.scalar_type() == torch::kHalf) LA_STEP_T(__half);
  else LA_STEP_T(float);
#undef LA_STEP_T
#undef LA_STEP
  HIP_CHECK(hipGetLastError());
  // as every operation in place does: a backward pass that saved this state as
  // its initial_state then raises instead of reading the new one (tensors made in
  // inference mode have no such count)
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return out;
}
