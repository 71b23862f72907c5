// Operators on logits [rows][cols]: the policy's answers and the learner's loss.
//
//   k_adjust_wave, k_adjust   penalties for repeated actions, a bias, a legal-move mask
//   k_adjust_grad             its backward pass; k_bias_join joins the gradient of a bias that rows share
//   k_loss_wave, k_loss_block, k_loss_part + k_loss_row   the policy/value loss, with or without its gradient
//   k_loss_grad               the gradient alone, from the rows' statistics
//   k_loss_mean               the mean of the rows
//
// All are bound by memory or, for small calls, by latency: every element is read and written once, 16 bytes at a time
// and before anything that does not need it, and arithmetic is in float.  (A copy of 1 GiB reaches 5.2 TB/s here.)
#include "ops.h"

#include <math.h>

namespace mtaz {
namespace {

// elements of 16 bytes
template <int DT> constexpr int PER = DT == MTAZ_F32 ? 4 : 8;

struct Legal {
  const uint32_t* bits;
  int64_t stride;
  // bits of columns v .. v + N - 1 (v a multiple of N, N 4 or 8), 0 behind the last column (n of them are left)
  template <int N> __device__ __forceinline__ uint32_t some(int64_t row, int v, int n) const {
    const uint32_t all = n >= N ? (1u << N) - 1 : n > 0 ? (1u << n) - 1 : 0u;
    return bits && n > 0 ? (bits[row * stride + (v >> 5)] >> (v & 31)) & all : all;
  }
};

struct Taken {
  const int32_t* actions;
  int64_t stride;
  const int32_t* lengths;
  int history;
  float repetition, inverse, frequency, presence;       // inverse: 1 / repetition
  const float* per_row;
};
struct Penalty {
  float repetition, inverse, frequency, presence;
};
__device__ __forceinline__ Penalty penalty_of(const Taken& t, int64_t row) {
  if (t.per_row) {
    const float* p = t.per_row + 3 * row;
    return {p[0], 1.f / p[0], p[1], p[2]};
  }
  return {t.repetition, t.inverse, t.frequency, t.presence};
}
// calls f for every action that the row has taken, THREADS threads in steps of four entries; the first entries are
// asked for before the length is there.  Entries outside [0, cols) lie outside every tile.
template <int THREADS, typename F> __device__ __forceinline__ void each_taken(const Taken& t, int64_t row, int thread, F f) {
  const int32_t* a = t.actions + row * t.stride;
  const int len = t.lengths ? min(max(t.lengths[row], 0), t.history) : t.history;
  for (int i = 4 * thread; i < t.history; i += 4 * THREADS) {
    Pack<int32_t, 4> q;
    if (i + 4 <= t.history) {
      q = *reinterpret_cast<const Pack<int32_t, 4>*>(a + i);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) q.v[j] = i + j < t.history ? a[i + j] : -1;
    }
    if (i >= len) break;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < len) f(q.v[j]);
  }
}

// An address that the compiler does not know to be p: it joins the first of a row's last few elements with the wide
// access of the other path, which then falls into two or three.
template <typename T> __device__ __forceinline__ T* apart(T* p) {
  asm("" : "+v"(p));
  return p;
}
// N elements packed in 32-bit words: 16-bit values of their own would take a register each, and where two paths join,
// the wide load's words would be taken apart as soon as they are there.
template <int DT, int N> struct Words {
  typedef typename Elem<DT>::T T;
  static constexpr int W = N * (int)sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void fetch(const T* p, int n) {   // n of them there, the others 0
    if (n >= N) {
      __builtin_memcpy(w, p, sizeof(w));
    } else {
      p = apart(p);
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) put(j, p[j]);
      forget();
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (DT == MTAZ_F32) return __builtin_bit_cast(float, w[j]);
    if constexpr (DT == MTAZ_BF16) return __builtin_bit_cast(float, j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    if constexpr (DT == MTAZ_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j / 2] >> (16 * (j & 1))));
  }
  __device__ __forceinline__ void put(int j, T x) {
    if constexpr (DT == MTAZ_F32) w[j] = __builtin_bit_cast(uint32_t, x);
    else {
      const uint32_t half = __builtin_bit_cast(uint16_t, x);
      w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | half << 16 : (w[j / 2] & 0xffff0000u) | half;
    }
  }
  __device__ __forceinline__ void leave(T* p, int n) const {
    if (n >= N) {
      __builtin_memcpy(p, w, sizeof(w));
      return;
    }
    p = apart(p);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= n) continue;
      if constexpr (sizeof(T) == 4) p[j] = __builtin_bit_cast(T, w[j]);
      else p[j] = __builtin_bit_cast(T, (uint16_t)(w[j / 2] >> (16 * (j & 1))));
    }
  }
  // what lies under the bits of ok, and `other` elsewhere (a value's bits, twice where they are 16)
  __device__ __forceinline__ void keep(uint32_t ok, uint32_t other) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      uint32_t m;
      if constexpr (DT == MTAZ_F32) m = bits_of(ok, i);
      else m = (bits_of(ok, 2 * i) & 0xffffu) | (bits_of(ok, 2 * i + 1) << 16);
      w[i] = (w[i] & m) | (other & ~m);
    }
  }
  static __device__ __forceinline__ uint32_t bits_of(uint32_t ok, int j) { return 0u - ((ok >> j) & 1u); }
  // The compiler forgets how the words came about: else it keeps every value as a float from one phase to the next.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[i]));
  }
};

// ---- penalties, bias, mask -----------------------------------------------------------------------------------
template <int DT> constexpr uint32_t NEVER = DT == MTAZ_F32 ? 0xff800000u : DT == MTAZ_F16 ? 0xfc00fc00u : 0xff80ff80u;
// One access: N logits, the counts of their actions (none: nullptr), their bias and legality.  Without a branch and
// with the reciprocal of the repetition penalty, because a few taken actions among many others are enough to send
// every wave through all branches.  The reciprocal is a rounded float itself, so that x times it is off by up to 2^-23 of
// the result, where x / repetition would be by 2^-24.
template <int DT, int N>
__device__ __forceinline__ void adjust(Words<DT, N>& q, const uint32_t* cnt, const Words<MTAZ_F32, N>& bias, uint32_t ok,
                                       const Penalty& p) {
  typedef Elem<DT> E;
  float f[N];
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = q.get(j);
  if (cnt) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 four = *reinterpret_cast<const uint4*>(cnt + i);
      const uint32_t c[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = f[i + j], y = fmaf(-p.frequency, (float)c[j], x * (x > 0.f ? p.inverse : p.repetition)) - p.presence;
        f[i + j] = c[j] ? y : x;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) q.put(j, E::put(f[j] + bias.get(j)));
  q.keep(ok, NEVER<DT>);
}

// Rows of up to WAVE_COLS columns: a wave each, with the counts of its actions in its own piece of LDS.  4096 x 554 f32
// with 60 actions a row and masks: 6.8 us (19 MB, 2.9 TB/s, most of it from the caches).
constexpr int WAVE_COLS = 1024;
template <int DT>
__global__ __launch_bounds__(256) void k_adjust_wave(const typename Elem<DT>::T* x, int64_t x_stride,
                                                     typename Elem<DT>::T* y, int64_t y_stride, int64_t rows, int cols,
                                                     Legal legal, const float* bias, int64_t bias_stride, Taken taken) {
  constexpr int N = PER<DT>, REP = WAVE_COLS / (64 * N);
  __shared__ __attribute__((aligned(16))) uint32_t counts[4][WAVE_COLS];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= rows) return;
  Words<DT, N> q[REP];
#pragma unroll
  for (int k = 0; k < REP; ++k) {
    const int v = N * (lane + 64 * k);
    if (v < cols) q[k].fetch(x + row * x_stride + v, cols - v);
  }
  Penalty p = {};
  uint32_t* cnt = counts[wave];
  const bool counted = taken.actions != nullptr;
  if (counted) {                                        // LDS serves one wave's accesses in order
    p = penalty_of(taken, row);
#pragma unroll
    for (int k = 0; k < WAVE_COLS / 256; ++k) *reinterpret_cast<uint4*>(cnt + 4 * (lane + 64 * k)) = make_uint4(0, 0, 0, 0);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    each_taken<64>(taken, row, lane, [&](int v) {
      if ((uint32_t)v < (uint32_t)cols) atomicAdd(&cnt[v], 1u);
    });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
#pragma unroll
  for (int k = 0; k < REP; ++k) {
    const int v = N * (lane + 64 * k), n = cols - v;
    if (n <= 0) continue;
    const uint32_t ok = legal.some<N>(row, v, n);
    Words<MTAZ_F32, N> b = {};
    if (bias && ok) b.fetch(bias + row * bias_stride + v, n);
    adjust<DT, N>(q[k], counted ? cnt + v : nullptr, b, ok, p);
    q[k].leave(y + row * y_stride + v, n);
  }
}

// Longer rows in tiles, so that one long row fills the chip as well as many: a workgroup counts the actions in its
// columns.  Integer adds, so their order does not matter.  One access a thread and four workgroups on a CU hide each
// other's phases; two accesses take 84 registers, only two workgroups fit, and it took a fifth longer.  1024 x 50021 f16
// with everything (205 MB): 60 us in a training step, where the logits come from memory, 43 call after call, where
// the last-level cache has them; without actions 33.  A workgroup takes `per` rows one after the other, more than one
// only where they share mask and bias, which it then reads once.
constexpr int NT = 512;
template <int DT, bool COUNTED>
__global__ __launch_bounds__(NT) void k_adjust(const typename Elem<DT>::T* x, int64_t x_stride,
                                               typename Elem<DT>::T* y, int64_t y_stride, int64_t rows, int per, int cols,
                                               int tiles, Legal legal, const float* bias, int64_t bias_stride,
                                               Taken taken) {
  constexpr int N = PER<DT>, TILE = NT * N;
  __shared__ __attribute__((aligned(16))) uint32_t cnt[COUNTED ? TILE : 4];
  const int64_t r0 = (int64_t)(blockIdx.x / tiles) * per, r1 = min(rows, r0 + per);
  const int v0 = (int)(blockIdx.x % tiles) * TILE, i = N * threadIdx.x, v = v0 + i, n = cols - v;
  Words<DT, N> q;
  Words<MTAZ_F32, N> b = {};
  if (n > 0) q.fetch(x + r0 * x_stride + v, n);
  const uint32_t ok = legal.some<N>(r0, v, n);
  if (bias && ok) b.fetch(bias + r0 * bias_stride + v, n);
  for (int64_t row = r0; row < r1; ++row) {
    if (row > r0 && n > 0) q.fetch(x + row * x_stride + v, n);
    Penalty p = {};
    if (COUNTED) {
      p = penalty_of(taken, row);
#pragma unroll
      for (int k = 0; k < N / 4; ++k) *reinterpret_cast<uint4*>(cnt + 4 * (threadIdx.x + NT * k)) = make_uint4(0, 0, 0, 0);
      __syncthreads();
      each_taken<NT>(taken, row, threadIdx.x, [&](int a) {
        const uint32_t at = (uint32_t)a - (uint32_t)v0;
        if (at < (uint32_t)TILE) atomicAdd(&cnt[at], 1u);
      });
      __syncthreads();
    }
    if (n > 0) {
      adjust<DT, N>(q, COUNTED ? cnt + i : nullptr, b, ok, p);
      q.leave(y + row * y_stride + v, n);
    }
    if (COUNTED && row + 1 < r1) __syncthreads();       // all have read their counts
  }
}

// d x = d y where legal, else 0; gb: the same in float, per row; part: its sums over the columns of the workgroup's rows,
// for a bias that all rows share.  A workgroup takes `per` rows one after the other, four of them under way.  1024 x 50021
// f16 with a shared bias: 51 us (205 MB, 4.0 TB/s).
template <int DT>
__global__ __launch_bounds__(NT) void k_adjust_grad(const typename Elem<DT>::T* gy, int64_t gy_stride,
                                                    typename Elem<DT>::T* gx, int64_t gx_stride, float* gb,
                                                    int64_t gb_stride, float* part, int64_t rows, int per, int cols,
                                                    int tiles, Legal legal) {
  constexpr int N = PER<DT>;
  const int64_t chunk = blockIdx.x / tiles, r0 = chunk * per, r1 = min(rows, r0 + per);
  const int v = ((int)(blockIdx.x % tiles) * NT + threadIdx.x) * N, n = cols - v;
  if (n <= 0) return;
  float sum[N] = {};
  const uint32_t first = legal.some<N>(r0, v, n);
  auto take = [&](int64_t row, Words<DT, N>& g) {
    g.keep(legal.stride == 0 ? first : legal.some<N>(row, v, n), 0);
    if (gx) g.leave(gx + row * gx_stride + v, n);
    Words<MTAZ_F32, N> f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      f.put(j, g.get(j));
      sum[j] += g.get(j);
    }
    if (gb) f.leave(gb + row * gb_stride + v, n);
  };
  constexpr int AHEAD = 4;                              // rows under way at once
  Words<DT, N> g[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (r0 + k < r1) g[k].fetch(gy + (r0 + k) * gy_stride + v, n);
  for (int64_t row = r0; row < r1; row += AHEAD)
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (row + k >= r1) break;
      take(row + k, g[k]);
      if (row + k + AHEAD < r1) g[k].fetch(gy + (row + k + AHEAD) * gy_stride + v, n);
    }
  if (part) {
    Words<MTAZ_F32, N> f;
#pragma unroll
    for (int j = 0; j < N; ++j) f.put(j, sum[j]);
    f.leave(part + chunk * cols + v, n);
  }
}
// Afterwards the few places of taken actions: d x = d y * slope, the slope 1 / repetition (x > 0) or repetition.  A
// thread per entry of the list; an action that is in it twice is written twice alike.
template <int DT>
__global__ __launch_bounds__(256) void k_taken_grad(const typename Elem<DT>::T* gy, int64_t gy_stride,
                                                    const typename Elem<DT>::T* x, int64_t x_stride,
                                                    typename Elem<DT>::T* gx, int64_t gx_stride, int64_t rows, int cols,
                                                    int groups, Legal legal, Taken taken) {
  typedef Elem<DT> E;
  const int64_t id = (int64_t)blockIdx.x * 4 + threadIdx.x / 64, row = id / groups;
  const int i = (int)(id % groups) * 64 + threadIdx.x % 64;
  if (row >= rows || i >= taken.history) return;
  const int v = taken.actions[row * taken.stride + i];
  if (taken.lengths && i >= taken.lengths[row]) return;
  if ((uint32_t)v >= (uint32_t)cols || !legal.some<1>(row, v, 1)) return;
  const Penalty p = penalty_of(taken, row);
  const float g = E::get(gy[row * gy_stride + v]);
  gx[row * gx_stride + v] = E::put(E::get(x[row * x_stride + v]) > 0.f ? g * p.inverse : g * p.repetition);
}
// the workgroups' sums, in order
__global__ __launch_bounds__(256) void k_bias_join(const float* part, int chunks, int cols, float* gb) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= cols) return;
  float s = 0.f;
#pragma unroll 8
  for (int c = 0; c < chunks; ++c) s += part[(int64_t)c * cols + v];
  gb[v] = s;
}

// ---- policy/value loss -------------------------------------------------------------------------------------
// With top the largest legal logit, total = sum exp(z - top), pi = sum of the targets, dot = sum pi (z - top):
//   row = pi log(total) - dot,   d row / d z = exp(z - top) / total * pi - target.
// exp by the instruction for 2^x.  The product with log2(e) is off by 2^-24 of z - top (and the factor by a third of that),
// which a term e^(z - top) turns into at most 0.5 * 2^-24 of the largest, but |z - top| 2^-24 of itself: for float
// logits, whose small gradients would show it, the product's remainder goes into the term.  Five operations more a
// logit: 4096 x 554 with targets 7.7 us in place of 7.2.  (0 stays 0: the remainder of a product past -FLT_MAX is no number.)
__device__ __forceinline__ float soft_exp(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }
template <int DT> __device__ __forceinline__ float soft_exp_of(float d) {
  if constexpr (DT != MTAZ_F32) return soft_exp(d);
  constexpr double LOG2E = 1.44269504088896341;
  constexpr float HIGH = (float)LOG2E, LOW = (float)(LOG2E - (double)HIGH);
  const float p = d * HIGH, rest = fmaf(d, LOW, fmaf(d, HIGH, -p)), e = __builtin_amdgcn_exp2f(p);
  return e > 0.f ? fmaf(e, rest * 0.693147180559945309f, e) : e;
}

struct Row {
  float loss;          // without the value term
  float top, inv, pi;  // inv = 1 / total, 0 where nothing is legal
};
__device__ __forceinline__ Row row_of(float top, float total, float pi, float dot) {
  const bool some = top != -INFINITY || total != 0.f;   // a NaN among the logits is no empty row
  return {some ? pi * logf(total) - dot : 0.f, top, some ? 1.f / total : 0.f, pi};
}
// what exp is taken relative to: nothing in a row without a finite logit
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.f : top; }
// the value term, the row's statistics for k_loss_mean and k_loss_grad, the value's gradient
__device__ __forceinline__ float finish_row(const Row& r, int64_t row, const float* value, const float* reward, float k,
                                            float* stats, float* value_grad) {
  float loss = r.loss;
  if (value) {
    const float d = value[row] - reward[row];
    loss += d * d;
    if (value_grad) value_grad[row] = 2.f * k * d;
  }
  *reinterpret_cast<float4*>(stats + 4 * row) = make_float4(r.top, r.inv, r.pi, loss);
  return loss;
}
__device__ __forceinline__ float wave_sum(float x) {
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

// A row in registers, THREADS threads with REP times PER logits each.  What is not legal, or not there, is held as a
// logit of -inf with a target of 0, which adds nothing anywhere.  KEEP: the exponentials stay in registers from the sums
// to the gradient; else they are taken twice.
template <int DT, int DP, int THREADS, int REP, bool KEEP = true> struct Held {
  static constexpr int N = PER<DT>;
  typedef typename Elem<DT>::T Z;
  typedef typename Elem<DP>::T W;
  Words<DT, N> z[REP];
  Words<DP, N> w[REP];
  float e[KEEP ? REP : 1][N];   // exp(z - top), after sums()
  uint32_t ok[REP];
  __device__ __forceinline__ void fetch(const Z* logits, const W* target, int64_t row, int cols, const Legal& legal,
                                        int thread) {
#pragma unroll
    for (int k = 0; k < REP; ++k) {
      const uint32_t v = N * (thread + THREADS * k);
      const int n = cols - (int)v;
      ok[k] = legal.some<N>(row, v, n);
      if (n > 0) z[k].fetch(logits + v, n), w[k].fetch(target + v, n);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < REP; ++k)
      if (ok[k] != (1u << N) - 1)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (!((ok[k] >> j) & 1u)) z[k].put(j, Elem<DT>::put(-INFINITY)), w[k].put(j, Elem<DP>::put(0.f));
  }
  __device__ __forceinline__ float top() const {
    float t = -INFINITY;
#pragma unroll
    for (int k = 0; k < REP; ++k) {
#pragma unroll
      for (int j = 0; j < N; ++j) t = fmaxf(t, z[k].get(j));
    }
    return t;
  }
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int k = 0; k < REP; ++k) z[k].forget(), w[k].forget();
  }
  // A logit of -inf makes the loss infinite if it has a target, and a target of 0 adds nothing.
  __device__ __forceinline__ void sums(float base, float& total, float& pi, float& dot) {
    if (!KEEP) forget();
    total = pi = dot = 0.f;
#pragma unroll
    for (int k = 0; k < REP; ++k) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = z[k].get(j) - base, t = w[k].get(j);
        const float x = soft_exp_of<DT>(d);
        if (KEEP) e[k][j] = x;
        total += x;
        pi += t;
        dot += t != 0.f ? t * d : 0.f;
      }
    }
  }
  __device__ __forceinline__ void leave(Z* g, int cols, const Row& r, float k, int thread) {
    if (!KEEP) forget();
    const float soft = k * r.inv * r.pi, kt = r.inv == 0.f ? 0.f : k, base = base_of(r.top);
#pragma unroll
    for (int q = 0; q < REP; ++q) {
      const int v = N * (thread + THREADS * q), n = cols - v;
      if (n <= 0) continue;
      Words<DT, N> o;
#pragma unroll
      for (int j = 0; j < N; ++j) o.put(j, Elem<DT>::put(fmaf(KEEP ? e[q][j] : soft_exp_of<DT>(z[q].get(j) - base), soft,
                                      -kt * w[q].get(j))));
      if (ok[q] != (1u << N) - 1)                       // 0 there in a row of NaN too
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (!((ok[q] >> j) & 1u)) o.put(j, Elem<DT>::put(0.f));
      o.leave(g + v, n);
    }
  }
};

// Rows of up to WAVE_COLS columns: a wave each, and everything stays in its registers.  4096 x 554 f32 with targets:
// 8 us (18 MB).  ONE: a single workgroup takes all rows and their mean (32 x 554 with the gradient 9.2 us).
template <int DT, int DP, bool ONE>
__global__ __launch_bounds__(ONE ? 1024 : 256) void k_loss_wave(const typename Elem<DT>::T* z, int64_t z_stride,
                                                                const typename Elem<DP>::T* pi, int64_t pi_stride,
                                                                int64_t rows, int cols, Legal legal, const float* value,
                                                                const float* reward, float* stats, float* loss,
                                                                typename Elem<DT>::T* grad, int64_t grad_stride,
                                                                float* value_grad, float k) {
  constexpr int WAVES = ONE ? 16 : 4;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  double mean = 0.;
  for (int64_t row = ONE ? wave : (int64_t)blockIdx.x * WAVES + wave; row < rows; row += ONE ? WAVES : rows) {
    Held<DT, DP, 64, WAVE_COLS / (64 * PER<DT>)> h;
    h.fetch(z + row * z_stride, pi + row * pi_stride, row, cols, legal, lane);
    h.clear();
    const float top = wave_max(h.top());
    float total, sum, dot;
    h.sums(base_of(top), total, sum, dot);
    const Row r = row_of(top, wave_sum(total), wave_sum(sum), wave_sum(dot));
    if (grad) h.leave(grad + row * grad_stride, cols, r, k, lane);
    if (lane == 0) mean += (double)finish_row(r, row, value, reward, k, stats, value_grad);
  }
  if (!ONE) return;
  __shared__ double ws[WAVES];
  if (lane == 0) ws[wave] = mean;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < WAVES; ++w) mean += ws[w];
    *loss = (float)(mean / (double)rows);
  }
}

// Rows that fit into a workgroup's registers: one workgroup each.  With 32 logits a thread and more the exponentials are
// taken twice; 64 of 16 bits and their targets still leave room for two workgroups of 512 on a CU, so that one loads
// while the other computes.  2048 x 32003 bf16 with the gradient: 106 us (393 MB, 3.7 TB/s); its 26 operations a logit
// take 44 us, and two workgroups hide half of them.
template <int DT, int DP, int THREADS, int REP>
__global__ __launch_bounds__(THREADS, 4) void k_loss_block(const typename Elem<DT>::T* z, int64_t z_stride,
                                                           const typename Elem<DP>::T* pi, int64_t pi_stride, int cols,
                                                           Legal legal, const float* value, const float* reward,
                                                           float* stats, typename Elem<DT>::T* grad, int64_t grad_stride,
                                                           float* value_grad, float k) {
  constexpr int WAVES = THREADS / 64;
  __shared__ float ws[4][WAVES];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  Held<DT, DP, THREADS, REP, (REP * PER<DT> < 32)> h;
  h.fetch(z + row * z_stride, pi + row * pi_stride, row, cols, legal, threadIdx.x);
  h.clear();
  float top = wave_max(h.top());
  if (lane == 0) ws[0][wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ws[0][w]);
  float total, sum, dot;
  h.sums(base_of(top), total, sum, dot);
  total = wave_sum(total), sum = wave_sum(sum), dot = wave_sum(dot);
  if (lane == 0) ws[1][wave] = total, ws[2][wave] = sum, ws[3][wave] = dot;
  __syncthreads();
  total = sum = dot = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += ws[1][w], sum += ws[2][w], dot += ws[3][w];
  const Row r = row_of(top, total, sum, dot);
  if (grad) h.leave(grad + row * grad_stride, cols, r, k, threadIdx.x);
  if (threadIdx.x == 0) finish_row(r, row, value, reward, k, stats, value_grad);
}

// Longer rows in tiles: the statistics of a tile, then of the row from its tiles'.  The gradient reads logits and targets
// again, since a row does not fit into a workgroup's registers: 512 x 131072 bf16 takes 56 us for the statistics (268 MB,
// 4.8 TB/s) and 67 for the gradient (403 MB, 6.0 TB/s, some of it from the last-level cache), 128 with the mean; one pass
// over what has to move would take 78 at the rate of a copy.
struct Soft {
  float top, total, pi, dot;
};
// The statistics of two pieces joined: each sum moves from its own top to the larger one.  A piece whose
// top is -inf has no finite logit: its total is 0 (or NaN) and its dot 0 (no target there) or infinite already.
__device__ __forceinline__ Soft join(const Soft& a, const Soft& b) {
  Soft r;
  r.top = fmaxf(a.top, b.top);
  const float da = a.top == -INFINITY ? 0.f : a.top - r.top, db = b.top == -INFINITY ? 0.f : b.top - r.top;
  r.total = a.total * soft_exp(da) + b.total * soft_exp(db);
  r.pi = a.pi + b.pi;
  r.dot = (a.dot + da * a.pi) + (b.dot + db * b.pi);
  return r;
}
constexpr int TILE_REP = 2;
template <int DT> constexpr int LOSS_TILE = NT * PER<DT> * TILE_REP;
template <int DT, int DP>
__global__ __launch_bounds__(NT) void k_loss_part(const typename Elem<DT>::T* z, int64_t z_stride,
                                                  const typename Elem<DP>::T* pi, int64_t pi_stride, int cols,
                                                  int tiles, Legal legal, Soft* part) {
  constexpr int WAVES = NT / 64;
  __shared__ float ws[4][WAVES];
  const int64_t row = blockIdx.x / tiles;
  const int v0 = (int)(blockIdx.x % tiles) * LOSS_TILE<DT>;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  Held<DT, DP, NT, TILE_REP> h;
  const Legal here = {legal.bits ? legal.bits + v0 / 32 : nullptr, legal.stride};
  h.fetch(z + row * z_stride + v0, pi + row * pi_stride + v0, row, cols - v0, here, threadIdx.x);
  h.clear();
  float top = wave_max(h.top());
  if (lane == 0) ws[0][wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ws[0][w]);
  float total, sum, dot;
  h.sums(base_of(top), total, sum, dot);
  total = wave_sum(total), sum = wave_sum(sum), dot = wave_sum(dot);
  if (lane == 0) ws[1][wave] = total, ws[2][wave] = sum, ws[3][wave] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = sum = dot = 0.f;
    for (int w = 0; w < WAVES; ++w) total += ws[1][w], sum += ws[2][w], dot += ws[3][w];
    part[blockIdx.x] = {top, total, sum, dot};
  }
}

// One tile of the gradient from the row's statistics
template <int DT, int DP>
__device__ __forceinline__ void grad_tile(const typename Elem<DT>::T* z, const typename Elem<DP>::T* pi,
                                          typename Elem<DT>::T* g, int64_t row, int v0, int cols, const Legal& legal,
                                          const Row& r, float k) {
  Held<DT, DP, NT, TILE_REP, false> h;
  const Legal here = {legal.bits ? legal.bits + v0 / 32 : nullptr, legal.stride};
  h.fetch(z + v0, pi + v0, row, cols - v0, here, threadIdx.x);
  h.clear();
  h.leave(g + v0, cols - v0, r, k, threadIdx.x);
}

// Joins the row's tiles, every workgroup of a row in the same order, and writes its own tile of the gradient; the row's
// first workgroup writes its statistics.
template <int DT, int DP>
__global__ __launch_bounds__(NT) void k_loss_row(const typename Elem<DT>::T* z, int64_t z_stride,
                                                 const typename Elem<DP>::T* pi, int64_t pi_stride, int cols,
                                                 int tiles, Legal legal, const Soft* part, const float* value,
                                                 const float* reward, float* stats, typename Elem<DT>::T* grad,
                                                 int64_t grad_stride, float* value_grad, float k) {
  const int per_row = grad ? tiles : 1;                 // workgroups
  const int64_t row = blockIdx.x / per_row;
  const int tile = (int)(blockIdx.x % per_row);
  __shared__ Row joined;
  if (threadIdx.x < 64) {
    Soft s = {-INFINITY, 0.f, 0.f, 0.f};
    for (int t = threadIdx.x; t < tiles; t += 64) s = join(s, part[row * tiles + t]);
    for (int o = 32; o; o >>= 1) {
      const Soft t = {__shfl_xor(s.top, o), __shfl_xor(s.total, o), __shfl_xor(s.pi, o), __shfl_xor(s.dot, o)};
      s = (threadIdx.x & o) ? join(t, s) : join(s, t);   // the lower lane first on both sides: the same sums
    }
    if (threadIdx.x == 0) {
      joined = row_of(s.top, s.total, s.pi, s.dot);
      if (tile == 0) finish_row(joined, row, value, reward, k, stats, value_grad);
    }
  }
  if (!grad) return;
  __syncthreads();
  grad_tile<DT, DP>(z + row * z_stride, pi + row * pi_stride, grad + row * grad_stride, row, tile * LOSS_TILE<DT>, cols, legal,
                    joined, k);
}

// The gradient from the statistics: rows of up to WAVE_COLS a wave each, longer ones in tiles (2048 x 32003 bf16 73 us, 393
// MB, 5.4 TB/s; 512 x 131072 59 us)
template <int DT, int DP>
__global__ __launch_bounds__(256) void k_loss_grad_wave(const typename Elem<DT>::T* z, int64_t z_stride,
                                                        const typename Elem<DP>::T* pi, int64_t pi_stride, int64_t rows,
                                                        int cols, Legal legal, const float* value, const float* reward,
                                                        const float* stats, const float* grad_out,
                                                        typename Elem<DT>::T* grad, int64_t grad_stride,
                                                        float* value_grad) {
  const int lane = threadIdx.x % 64;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (row >= rows) return;
  const float k = *grad_out / (float)rows;
  if (value_grad && lane == 0) value_grad[row] = 2.f * k * (value[row] - reward[row]);
  if (!grad) return;
  const float4 st = *reinterpret_cast<const float4*>(stats + 4 * row);
  Held<DT, DP, 64, WAVE_COLS / (64 * PER<DT>), false> h;
  h.fetch(z + row * z_stride, pi + row * pi_stride, row, cols, legal, lane);
    h.clear();
  h.leave(grad + row * grad_stride, cols, Row{0.f, st.x, st.y, st.z}, k, lane);
}
template <int DT, int DP>
__global__ __launch_bounds__(NT) void k_loss_grad(const typename Elem<DT>::T* z, int64_t z_stride,
                                                  const typename Elem<DP>::T* pi, int64_t pi_stride, int64_t rows,
                                                  int cols, int tiles, Legal legal, const float* value,
                                                  const float* reward, const float* stats, const float* grad_out,
                                                  typename Elem<DT>::T* grad, int64_t grad_stride, float* value_grad) {
  const int64_t row = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x % tiles);
  const float k = *grad_out / (float)rows;
  if (value_grad && tile == 0 && threadIdx.x == 0) value_grad[row] = 2.f * k * (value[row] - reward[row]);
  if (!grad) return;
  const float4 st = *reinterpret_cast<const float4*>(stats + 4 * row);
  grad_tile<DT, DP>(z + row * z_stride, pi + row * pi_stride, grad + row * grad_stride, row, tile * LOSS_TILE<DT>, cols, legal,
                    Row{0.f, st.x, st.y, st.z}, k);
}

// The mean of the rows' losses by one workgroup, in a fixed order and in 64 bits.  A few rows are added like k_loss_wave's
// one workgroup adds them, 16 waves' sums one after the other: a captured call, which takes this way, gives the same bits.
constexpr int64_t FEW_ROWS = 32;
__global__ __launch_bounds__(1024) void k_loss_mean(const float* stats, int64_t rows, float* loss) {
  if (rows <= FEW_ROWS) {
    if (threadIdx.x >= 64) return;
    double s = 0.;
    for (int64_t r = threadIdx.x; threadIdx.x < 16 && r < rows; r += 16) s += (double)stats[4 * r + 3];
    double mean = __shfl(s, 0);
    for (int w = 1; w < 16; ++w) mean += __shfl(s, w);
    if (threadIdx.x == 0) *loss = (float)(mean / (double)rows);
    return;
  }
  double s = 0.;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < rows; r += 1024) s += (double)stats[4 * r + 3];
  __shared__ double ws[16];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if (threadIdx.x % 64 == 0) ws[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += ws[w];
    *loss = (float)(s / (double)rows);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------
constexpr int64_t MOST_COLS = 1 << 24;
constexpr int64_t MOST_WAVES = (1 << 26) - 4;

int64_t tiles_of(int64_t cols, int tile) { return (cols + tile - 1) / tile; }
const char* bad_shape(int64_t rows, int64_t cols, int dtype) {
  if (rows < 0) return "rows must not be negative";
  if (cols < 1 || cols > MOST_COLS) return "cols must be in [1, 2^24]";
  // a launch has fewer than 2^32 threads: 64 a row in the kernels for short rows, 512 a tile in the others
  // (rounded up to four rows, or four times 64 entries, a workgroup)
  if (rows > MOST_WAVES || (cols > WAVE_COLS && rows * tiles_of(cols, 512 * 4) >= 1 << 23)) return "too many rows for one call";
  if (dtype < MTAZ_F32 || dtype > MTAZ_BF16) return "unknown element type";
  return nullptr;
}
// `rows` rows of cols elements of type dtype in memory
struct Place {
  const char* at;
  int64_t step, width;                                  // bytes from row to row, and of a row
  Place(const void* p, int64_t stride, int64_t cols, int dtype)
      : at((const char*)p), step(stride * elem_size(dtype)), width(cols * elem_size(dtype)) {}
};
// Whether two places overlap.  The very same rows are allowed where `same` says so, and so are rows that interleave
// (columns of one matrix).
bool tangled(const Place& a, const Place& b, int64_t rows, bool same) {
  if (!a.at || !b.at || rows == 0) return false;
  if (a.at == b.at && a.width == b.width && (a.step == b.step || rows == 1)) return !same;
  if (a.at + (rows - 1) * a.step + a.width <= b.at || b.at + (rows - 1) * b.step + b.width <= a.at) return false;
  if (a.step != b.step || a.step <= 0) return true;
  const int64_t off = ((b.at - a.at) % a.step + a.step) % a.step;   // from a row of a to the next of b
  return off < a.width || a.step - off < b.width;
}
// Whether an output lies over what is read for other places than the one that is written: a mask, or the actions taken,
// their lengths and penalties
bool over_inputs(const Place& out, int64_t rows, int64_t cols, const uint32_t* legal, int64_t legal_stride,
                 const int32_t* actions = nullptr, int64_t actions_stride = 0, int history = 0,
                 const int32_t* lengths = nullptr, const float* per_row = nullptr) {
  auto over = [&](const void* p, int64_t stride, int64_t width) {
    return tangled({p, stride, width, MTAZ_F32}, out, rows, false);
  };
  return over(legal, legal_stride, (cols + 31) / 32) ||
         (actions && history && (over(actions, actions_stride, history) || over(lengths, 1, 1) || over(per_row, 3, 3)));
}
const char* bad_taken(const int32_t* actions, int64_t stride, int history, const double* penalties,
                      const float* per_row) {
  if (history < 0 || history > 1 << 30) return "history must be in [0, 2^30]";
  if (!actions || history == 0) return nullptr;
  if (stride < 0) return "actions_stride must not be negative";
  if (!penalties && !per_row) return "actions without penalties";
  if (!per_row && !(penalties[0] > 0.)) return "repetition must be positive";
  return nullptr;
}
Taken taken_of(const int32_t* actions, int64_t stride, int history, const int32_t* lengths, const double* penalties,
               const float* per_row) {
  Taken t = {};
  if (!actions || history == 0) return t;
  if (!per_row && penalties[0] == 1. && penalties[1] == 0. && penalties[2] == 0.) return t;   // nothing to do
  t.actions = actions, t.stride = stride, t.lengths = lengths, t.history = history, t.per_row = per_row;
  if (!per_row) t.repetition = (float)penalties[0], t.inverse = (float)(1. / penalties[0]), t.frequency = (float)penalties[1], t.presence = (float)penalties[2];
  return t;
}
// Longest row that stays in the registers of one workgroup
constexpr int BLOCK_COLS = 32768;
int64_t loss_workspace(int64_t rows, int64_t cols) {
  return cols <= BLOCK_COLS ? 256 : (int64_t)sizeof(Soft) * rows * tiles_of(cols, LOSS_TILE<MTAZ_F32>);
}
const char* bad_work(const void* work, int64_t bytes, int64_t needed) {
  return !work || ((uintptr_t)work & 255) || bytes < needed ? "workspace too small or not aligned to 256 bytes" : nullptr;
}
// Whether the stream records a graph.  (The stream of nullptr cannot, and asked beside another's capture it would end that.)
bool capturing(hipStream_t s) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return s && hipStreamIsCapturing(s, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}
int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(e));
}
// Rows a workgroup of k_adjust_grad takes one after the other: so many that all workgroups are on the CUs at once.
int64_t rows_each(int64_t rows, int64_t cols) {
  const int64_t across = tiles_of(cols, 512 * 8), chunks = across >= 1024 ? 1 : 1024 / across;
  return rows <= chunks ? 1 : (rows + chunks - 1) / chunks;
}
int64_t bias_chunks(int64_t rows, int64_t cols) {
  const int64_t each = rows_each(rows, cols);
  return (rows + each - 1) / each;
}

}  // namespace
}  // namespace mtaz

using namespace mtaz;

// the statement that follows the type, with DT = the element type (DP = the targets')
#define FOR_TYPE(dtype, ...)                                             \
  if (dtype == MTAZ_F32) { constexpr int DT = MTAZ_F32; __VA_ARGS__; }     \
  else if (dtype == MTAZ_F16) { constexpr int DT = MTAZ_F16; __VA_ARGS__; } \
  else { constexpr int DT = MTAZ_BF16; __VA_ARGS__; }
#define FOR_TYPES(dtype, target, ...)                                         \
  FOR_TYPE(dtype, if (target == MTAZ_F32) { constexpr int DP = MTAZ_F32; __VA_ARGS__; } \
                  else { constexpr int DP = DT; __VA_ARGS__; })

extern "C" int mtaz_adjust_logits(int device, int64_t rows, int64_t cols, int dtype, const void* d_logits,
                                  int64_t logits_stride, void* d_out, int64_t out_stride, const uint32_t* d_legal,
                                  int64_t legal_stride, const float* d_bias, int64_t bias_stride,
                                  const int32_t* d_actions, int64_t actions_stride, int history,
                                  const int32_t* d_lengths, const double* penalties, const float* d_penalties,
                                  void* stream) {
  const char* bad = bad_shape(rows, cols, dtype);
  if (!bad) bad = bad_taken(d_actions, actions_stride, history, penalties, d_penalties);
  if (!bad && (!d_logits || !d_out) && rows) bad = "no logits or no output";
  if (!bad && out_stride < cols && rows > 1) bad = "rows of the output overlap";
  if (!bad && tangled({d_logits, logits_stride, cols, dtype}, {d_out, out_stride, cols, dtype}, rows, true))
    bad = "the output overlaps the logits and is not in place";
  const Place to(d_out, out_stride, cols, dtype);
  if (!bad && (over_inputs(to, rows, cols, d_legal, legal_stride, d_actions, actions_stride, history, d_lengths, d_penalties) ||
               tangled({d_bias, bias_stride, cols, MTAZ_F32}, to, rows, true)))
    bad = "the output overlaps the mask, the bias or the actions";
  if (bad) return ops_error(MTAZ_E_FAIL, "adjust_logits", bad);
  if (rows == 0) return 0;
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, "adjust_logits", hipGetErrorString(on.status));
  const Taken t = taken_of(d_actions, actions_stride, history, d_lengths, penalties, d_penalties);
  const Legal legal{d_legal, legal_stride};
  const hipStream_t s = (hipStream_t)stream;
  const int nc = (int)cols;
  FOR_TYPE(dtype, {
    const auto* x = (const Elem<DT>::T*)d_logits;
    auto* y = (Elem<DT>::T*)d_out;
    if (cols <= WAVE_COLS) {
      k_adjust_wave<DT><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(x, logits_stride, y, out_stride, rows, nc, legal, d_bias,
                                                                 bias_stride, t);
    } else {
      const int64_t tiles = tiles_of(cols, NT * PER<DT>);
      // Two rows a workgroup where they share what it would read again, a float's bias for each logit, and the chip is
      // full twice over all the same (call after call, 512 actions: 1024 x 50021 f16 43 us, with one row 48, f32 90 and 99,
      // 4096 x 5000 f16 24 and 28; from memory 2 to 3 us less with two rows, and without actions as much more).
      const bool two = d_bias && bias_stride == 0 && (!d_legal || legal_stride == 0) && rows * tiles >= 4096;
      const unsigned grid = (unsigned)((two ? (rows + 1) / 2 : rows) * tiles);
      if (t.actions) k_adjust<DT, true><<<grid, NT, 0, s>>>(x, logits_stride, y, out_stride, rows, two ? 2 : 1, nc, (int)tiles,
                                                            legal, d_bias, bias_stride, t);
      else k_adjust<DT, false><<<grid, NT, 0, s>>>(x, logits_stride, y, out_stride, rows, two ? 2 : 1, nc, (int)tiles, legal,
                                                   d_bias, bias_stride, t);
    }
  });
  return launched("adjust_logits");
}

extern "C" int64_t mtaz_adjust_logits_grad_workspace(int64_t rows, int64_t cols) {
  if (const char* bad = bad_shape(rows, cols, MTAZ_F32)) return ops_error(MTAZ_E_FAIL, "adjust_logits_grad", bad);
  return 4 * cols * bias_chunks(rows, cols);
}

extern "C" int mtaz_adjust_logits_grad(int device, int64_t rows, int64_t cols, int dtype, const void* d_grad_out,
                                       int64_t grad_out_stride, const void* d_logits, int64_t logits_stride,
                                       void* d_grad, int64_t grad_stride, float* d_bias_grad, int64_t bias_grad_stride,
                                       const uint32_t* d_legal, int64_t legal_stride, const int32_t* d_actions,
                                       int64_t actions_stride, int history, const int32_t* d_lengths,
                                       const double* penalties, const float* d_penalties, void* d_work,
                                       int64_t work_bytes, void* stream) {
  const char* what = "adjust_logits_grad";
  const char* bad = bad_shape(rows, cols, dtype);
  if (!bad) bad = bad_taken(d_actions, actions_stride, history, penalties, d_penalties);
  // the frequency and presence penalties are constants: without a repetition penalty the slope is 1 everywhere
  const bool bends = !bad && (d_penalties || (penalties && penalties[0] != 1.));
  const Taken t = bends ? taken_of(d_actions, actions_stride, history, d_lengths, penalties, d_penalties) : Taken{};
  const bool shared = d_bias_grad && bias_grad_stride == 0;
  if (!bad && rows && !d_grad_out) bad = "no incoming gradient";
  if (!bad && rows && t.actions && d_grad && !d_logits) bad = "the penalties' gradient needs the logits";
  if (!bad && rows * ((history + 63) / 64) > MOST_WAVES) bad = "too many rows for one call";
  if (!bad && rows > 1 && ((d_grad && grad_stride < cols) || (d_bias_grad && !shared && bias_grad_stride < cols)))
    bad = "rows of an output overlap";
  if (!bad && shared && rows) bad = bad_work(d_work, work_bytes, 4 * cols * bias_chunks(rows, cols));
  if (!bad && tangled({d_grad_out, grad_out_stride, cols, dtype}, {d_grad, grad_stride, cols, dtype}, rows, !t.actions))
    bad = "the gradient overlaps the incoming one (in place is allowed without a repetition penalty)";
  if (!bad && t.actions && tangled({d_logits, logits_stride, cols, dtype}, {d_grad, grad_stride, cols, dtype}, rows, false))
    bad = "the gradient overlaps the logits";
  for (const Place& to : {Place(d_grad, grad_stride, cols, dtype), Place(d_bias_grad, bias_grad_stride, cols, MTAZ_F32)})
    if (!bad && over_inputs(to, rows, cols, d_legal, legal_stride, d_actions, actions_stride, history, d_lengths, d_penalties))
      bad = "a gradient overlaps the mask or the actions";
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const hipStream_t s = (hipStream_t)stream;
  const int nc = (int)cols;
  const Legal legal{d_legal, legal_stride};
  const int64_t groups = (t.history + 63) / 64;         // of 64 entries
  const int64_t each = rows_each(rows, cols), chunks = rows ? (rows + each - 1) / each : 0;
  if (rows && (d_grad || d_bias_grad)) {
    FOR_TYPE(dtype, {
      const auto* gy = (const Elem<DT>::T*)d_grad_out;
      auto* gx = (Elem<DT>::T*)d_grad;
      const int tiles = (int)tiles_of(cols, NT * PER<DT>);
      k_adjust_grad<DT><<<(unsigned)(chunks * tiles), NT, 0, s>>>(gy, grad_out_stride, gx, grad_stride,
                                                                shared ? nullptr : d_bias_grad, bias_grad_stride,
                                                                shared ? (float*)d_work : nullptr, rows, (int)each, nc,
                                                                tiles, legal);
      if (gx && t.actions)
        k_taken_grad<DT><<<(unsigned)((rows * groups + 3) / 4), 256, 0, s>>>(gy, grad_out_stride,
                                                                           (const Elem<DT>::T*)d_logits, logits_stride, gx,
                                                                           grad_stride, rows, nc, (int)groups, legal, t);
    });
  }
  if (shared) k_bias_join<<<(nc + 255) / 256, 256, 0, s>>>((const float*)d_work, (int)chunks, nc, d_bias_grad);
  return launched(what);
}

extern "C" int64_t mtaz_policy_loss_workspace(int64_t rows, int64_t cols) {
  if (const char* bad = bad_shape(rows, cols, MTAZ_F32)) return ops_error(MTAZ_E_FAIL, "policy_loss", bad);
  return loss_workspace(rows, cols);
}

static const char* bad_loss(int64_t rows, int64_t cols, int dtype, int target_dtype, const void* logits,
                            const void* target, const float* value, const float* reward, const float* stats,
                            const void* grad, int64_t grad_stride, const float* value_grad) {
  if (const char* bad = bad_shape(rows, cols, dtype)) return bad;
  if (rows < 1) return "the mean of no rows";
  if (target_dtype != MTAZ_F32 && target_dtype != dtype) return "targets are float32 or of the logits' type";
  if (!logits || !target || !stats) return "no logits, targets or statistics";
  if ((uintptr_t)stats & 15) return "statistics must be aligned to 16 bytes";
  if (!value != !reward) return "a value without a reward, or a reward without a value";
  if (value_grad && !value) return "the gradient of a value that is not there";
  if (grad && grad_stride < cols && rows > 1) return "rows of the gradient overlap";
  return nullptr;
}
// A gradient over its own logits is written where a thread has read them; over the targets likewise.
static const char* bad_place(int64_t rows, int64_t cols, int dtype, int target_dtype, const void* logits,
                             int64_t logits_stride, const void* target, int64_t target_stride, const uint32_t* legal,
                             int64_t legal_stride, const void* grad, int64_t grad_stride) {
  const Place g(grad, grad_stride, cols, dtype);
  if (over_inputs(g, rows, cols, legal, legal_stride)) return "the gradient overlaps the mask";
  if (tangled({logits, logits_stride, cols, dtype}, g, rows, true) ||
      tangled({target, target_stride, cols, target_dtype}, g, rows, true))
    return "the gradient overlaps the logits or the targets and is not in place";
  return nullptr;
}

extern "C" int mtaz_policy_loss(int device, int64_t rows, int64_t cols, int dtype, int target_dtype,
                                const void* d_logits, int64_t logits_stride, const void* d_target,
                                int64_t target_stride, const uint32_t* d_legal, int64_t legal_stride,
                                const float* d_value, const float* d_reward, float* d_loss, float* d_stats,
                                void* d_grad, int64_t grad_stride, float* d_value_grad, double scale, void* d_work,
                                int64_t work_bytes, void* stream) {
  const char* what = "policy_loss";
  const char* bad = bad_loss(rows, cols, dtype, target_dtype, d_logits, d_target, d_value, d_reward, d_stats, d_grad,
                             grad_stride, d_value_grad);
  if (!bad && !d_loss) bad = "no place for the loss";
  if (!bad) bad = bad_work(d_work, work_bytes, loss_workspace(rows, cols));
  if (!bad) bad = bad_place(rows, cols, dtype, target_dtype, d_logits, logits_stride, d_target, target_stride, d_legal, legal_stride,
                             d_grad, grad_stride);
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const hipStream_t s = (hipStream_t)stream;
  const int nc = (int)cols;
  const Legal legal{d_legal, legal_stride};
  const float k = (float)(scale / (double)rows);
  // A handful of short rows: one launch, mean included.  With 8, 16, 24, 32 and 64 rows of 554 it takes 4.6, 5.7, 7.6, 9.0 and
  // 16.3 us in a graph, and the two launches 5.9 to 6.5; called one by one, where the host's launches bound them, 7.8, 7.9,
  // 8.2, 9.3 and 16.4 against 10.4.  So up to 16 rows, and up to 32 outside a capture: the means are added in the same
  // order on both sides.
  const bool one = cols <= WAVE_COLS && (rows <= FEW_ROWS / 2 || (rows <= FEW_ROWS && !capturing(s)));
  FOR_TYPES(dtype, target_dtype, {
    const auto* z = (const Elem<DT>::T*)d_logits;
    const auto* pi = (const Elem<DP>::T*)d_target;
    auto* g = (Elem<DT>::T*)d_grad;
    const unsigned n = (unsigned)rows;
    constexpr int N = PER<DT>;
    if (one) {
      k_loss_wave<DT, DP, true><<<1, 1024, 0, s>>>(z, logits_stride, pi, target_stride, rows, nc, legal, d_value, d_reward,
                                                  d_stats, d_loss, g, grad_stride, d_value_grad, k);
    } else if (cols <= WAVE_COLS) {
      k_loss_wave<DT, DP, false><<<(n + 3) / 4, 256, 0, s>>>(z, logits_stride, pi, target_stride, rows, nc, legal, d_value,
                                                           d_reward, d_stats, d_loss, g, grad_stride, d_value_grad, k);
    } else if (cols <= BLOCK_COLS) {
      auto launch = [&](auto kernel, int threads) {
        kernel<<<n, threads, 0, s>>>(z, logits_stride, pi, target_stride, nc, legal, d_value, d_reward, d_stats, g,
                                     grad_stride, d_value_grad, k);
      };
      constexpr int LONG = DP == MTAZ_F32 ? 1024 : 512;
      // 16 logits a thread while that fits: 16384 x 4096 f32 takes 153 us with 256 threads, 290 with 1024
      if (cols <= 2048) launch(k_loss_block<DT, DP, 128, 16 / N>, 128);
      else if (cols <= 4096) launch(k_loss_block<DT, DP, 256, 16 / N>, 256);
      else if (cols <= 8192) launch(k_loss_block<DT, DP, 512, 16 / N>, 512);
      else if (cols <= 16384) launch(k_loss_block<DT, DP, 1024, 16 / N>, 1024);
      else launch(k_loss_block<DT, DP, LONG, BLOCK_COLS / (LONG * N)>, LONG);
    } else {
      const int tiles = (int)tiles_of(cols, LOSS_TILE<DT>);
      k_loss_part<DT, DP><<<n * tiles, NT, 0, s>>>(z, logits_stride, pi, target_stride, nc, tiles, legal, (Soft*)d_work);
      k_loss_row<DT, DP><<<g ? n * tiles : n, NT, 0, s>>>(z, logits_stride, pi, target_stride, nc, tiles, legal,
                                                        (const Soft*)d_work, d_value, d_reward, d_stats, g, grad_stride,
                                                        d_value_grad, k);
    }
  });
  if (!one) k_loss_mean<<<1, 1024, 0, s>>>(d_stats, rows, d_loss);
  return launched(what);
}

extern "C" int mtaz_policy_loss_grad(int device, int64_t rows, int64_t cols, int dtype, int target_dtype,
                                     const void* d_logits, int64_t logits_stride, const void* d_target,
                                     int64_t target_stride, const uint32_t* d_legal, int64_t legal_stride,
                                     const float* d_value, const float* d_reward, const float* d_stats,
                                     const float* d_grad_out, void* d_grad, int64_t grad_stride, float* d_value_grad,
                                     void* stream) {
  const char* what = "policy_loss_grad";
  const char* bad = bad_loss(rows, cols, dtype, target_dtype, d_logits, d_target, d_value, d_reward, d_stats, d_grad,
                             grad_stride, d_value_grad);
  if (!bad && !d_grad_out) bad = "no incoming gradient";
  if (!bad) bad = bad_place(rows, cols, dtype, target_dtype, d_logits, logits_stride, d_target, target_stride, d_legal, legal_stride,
                             d_grad, grad_stride);
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  if (!d_grad && !d_value_grad) return 0;
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const int nc = (int)cols;
  const Legal legal{d_legal, legal_stride};
  const hipStream_t s = (hipStream_t)stream;
  FOR_TYPES(dtype, target_dtype, {
    const auto* z = (const Elem<DT>::T*)d_logits;
    const auto* pi = (const Elem<DP>::T*)d_target;
    auto* g = (Elem<DT>::T*)d_grad;
    if (cols <= WAVE_COLS) {
      k_loss_grad_wave<DT, DP><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(z, logits_stride, pi, target_stride, rows, nc, legal,
                                                                        d_value, d_reward, d_stats, d_grad_out, g,
                                                                        grad_stride, d_value_grad);
    } else {
      const int tiles = (int)tiles_of(cols, LOSS_TILE<DT>);
      k_loss_grad<DT, DP><<<(unsigned)(rows * tiles), NT, 0, s>>>(z, logits_stride, pi, target_stride, rows, nc, tiles, legal,
                                                                d_value, d_reward, d_stats, d_grad_out, g, grad_stride,
                                                                d_value_grad);
    }
  });
  return launched(what);
}
