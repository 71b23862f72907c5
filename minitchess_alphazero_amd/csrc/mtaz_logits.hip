// Operators on logits [rows][cols]: the policy's answers and the learner's loss.
//
//   k_adjust        penalties for repeated actions, a bias, a legal-move mask
//   k_adjust_grad   its backward pass (per row), k_bias_sum / k_bias_join for a shared bias
//   k_loss_part, k_loss_row, k_loss_mean   the policy/value loss and its gradient
//
// All are bound by memory: every element is read and written once with wide accesses, arithmetic is
// in float.  A row is cut into tiles of TILE columns, one workgroup each, so that a single long row
// fills the chip as well as many short ones do; what a tile needs of its row (the counts of the actions taken
// in its columns, the softmax statistics of the other tiles) is rebuilt by its workgroup.
#include "ops.h"

#include <math.h>

namespace mtaz {
namespace {

constexpr int TILE = 4096;    // columns per workgroup
constexpr int NT = 256;
constexpr int PER = 4;        // elements per access (16 B of float, 8 B of a 16-bit type)

struct Legal {
  const uint32_t* bits;
  int64_t stride;
  // bits of columns v .. v + 3 (v a multiple of 4)
  __device__ __forceinline__ uint32_t four(int64_t row, int v) const {
    return bits ? (bits[row * stride + (v >> 5)] >> (v & 31)) & 15u : 15u;
  }
};

struct Taken {
  const int32_t* actions;
  int64_t stride;
  const int32_t* lengths;
  int history;
  float repetition, frequency, presence;
  const float* per_row;
};

struct Penalty {
  float repetition, frequency, presence;
};

__device__ __forceinline__ Penalty penalty_of(const Taken& t, int64_t row) {
  if (t.per_row) return {t.per_row[3 * row], t.per_row[3 * row + 1], t.per_row[3 * row + 2]};
  return {t.repetition, t.frequency, t.presence};
}

// counts of the row's actions in columns [v0, v0 + nv) into cnt (LDS); integer adds, so their order does
// not matter.  Entries outside [0, cols) fall outside every tile.
__device__ __forceinline__ void count_taken(const Taken& t, int64_t row, int v0, int nv, uint32_t* cnt) {
  for (int i = threadIdx.x; i < nv; i += NT) cnt[i] = 0;
  __syncthreads();
  const int len = t.lengths ? min(max(t.lengths[row], 0), t.history) : t.history;
  const int32_t* a = t.actions + row * t.stride;
  for (int i = threadIdx.x; i < len; i += NT) {
    const uint32_t v = (uint32_t)(a[i] - v0);
    if (v < (uint32_t)nv) atomicAdd(&cnt[v], 1u);
  }
  __syncthreads();
}

template <typename T> __device__ __forceinline__ Pack<T, PER> load4(const T* p, int n) {
  Pack<T, PER> r;
  if (n >= PER) return *reinterpret_cast<const Pack<T, PER>*>(p);
#pragma unroll
  for (int j = 0; j < PER; ++j) r.v[j] = j < n ? p[j] : (T)0.f;
  return r;
}
template <typename T> __device__ __forceinline__ void store4(T* p, const Pack<T, PER>& r, int n) {
  if (n >= PER) {
    *reinterpret_cast<Pack<T, PER>*>(p) = r;
    return;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (j < n) p[j] = r.v[j];
}

template <int DT>
__global__ __launch_bounds__(NT) void k_adjust(const typename Elem<DT>::T* x, int64_t x_stride,
                                               typename Elem<DT>::T* y, int64_t y_stride, int cols, int tiles,
                                               Legal legal, const float* bias, int64_t bias_stride, Taken taken) {
  typedef Elem<DT> E;
  __shared__ uint32_t cnt[TILE];
  const int64_t row = blockIdx.x / tiles;
  const int v0 = (int)(blockIdx.x % tiles) * TILE;
  const int nv = min(TILE, cols - v0);
  const bool counted = taken.actions != nullptr;
  Penalty p = {1.f, 0.f, 0.f};
  if (counted) {
    count_taken(taken, row, v0, nv, cnt);
    p = penalty_of(taken, row);
  }
  for (int i = PER * threadIdx.x; i < nv; i += PER * NT) {
    const int v = v0 + i, n = nv - i;
    const uint32_t ok = legal.four(row, v);
    Pack<typename E::T, PER> q = load4(x + row * x_stride + v, n);
    Pack<float, PER> b = {};
    if (bias) b = load4(bias + row * bias_stride + v, n);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      float s = E::get(q.v[j]);
      const uint32_t c = counted && j < n ? cnt[i + j] : 0u;
      if (c) s = (s > 0.f ? s / p.repetition : s * p.repetition) - p.frequency * (float)c - p.presence;
      s += b.v[j];
      q.v[j] = E::put((ok >> j) & 1u ? s : -INFINITY);
    }
    store4(y + row * y_stride + v, q, n);
  }
}

// d x = d y * slope, slope = 1, or 1 / repetition (x > 0) or repetition (x <= 0) of a taken action; 0 where
// not legal.  gb: the same without the slope, per row, in float.
template <int DT>
__global__ __launch_bounds__(NT) void k_adjust_grad(const typename Elem<DT>::T* gy, int64_t gy_stride,
                                                    const typename Elem<DT>::T* x, int64_t x_stride,
                                                    typename Elem<DT>::T* gx, int64_t gx_stride, float* gb,
                                                    int64_t gb_stride, int cols, int tiles, Legal legal, Taken taken) {
  typedef Elem<DT> E;
  __shared__ uint32_t cnt[TILE];
  const int64_t row = blockIdx.x / tiles;
  const int v0 = (int)(blockIdx.x % tiles) * TILE;
  const int nv = min(TILE, cols - v0);
  const bool counted = taken.actions != nullptr;
  float rep = 1.f, inv = 1.f;
  if (counted) {
    count_taken(taken, row, v0, nv, cnt);
    rep = penalty_of(taken, row).repetition;
    inv = 1.f / rep;
  }
  for (int i = PER * threadIdx.x; i < nv; i += PER * NT) {
    const int v = v0 + i, n = nv - i;
    const uint32_t ok = legal.four(row, v);
    Pack<typename E::T, PER> g = load4(gy + row * gy_stride + v, n);
    Pack<float, PER> f;
#pragma unroll
    for (int j = 0; j < PER; ++j) f.v[j] = (ok >> j) & 1u ? E::get(g.v[j]) : 0.f;
    if (gb) store4(gb + row * gb_stride + v, f, n);
    if (!gx) continue;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (counted && j < n && cnt[i + j] && ((ok >> j) & 1u)) f.v[j] *= E::get(x[row * x_stride + v + j]) > 0.f ? inv : rep;
      g.v[j] = E::put(f.v[j]);
    }
    store4(gx + row * gx_stride + v, g, n);
  }
}

// Shared bias: columns summed over rows in a fixed order, chunk by chunk of rows, then over the chunks.
constexpr int BIAS_COLS = NT * PER;
template <int DT>
__global__ __launch_bounds__(NT) void k_bias_sum(const typename Elem<DT>::T* gy, int64_t gy_stride, int64_t rows,
                                                 int64_t per_chunk, int cols, Legal legal, float* part) {
  typedef Elem<DT> E;
  const int v = blockIdx.x * BIAS_COLS + PER * threadIdx.x, n = cols - v;
  if (n <= 0) return;
  const int64_t r0 = blockIdx.y * per_chunk, r1 = min(rows, r0 + per_chunk);
  Pack<float, PER> s = {};
  for (int64_t row = r0; row < r1; ++row) {
    const uint32_t ok = legal.four(row, v);
    const Pack<typename E::T, PER> g = load4(gy + row * gy_stride + v, n);
#pragma unroll
    for (int j = 0; j < PER; ++j) s.v[j] += (ok >> j) & 1u ? E::get(g.v[j]) : 0.f;
  }
  store4(part + (int64_t)blockIdx.y * cols + v, s, n);
}
__global__ __launch_bounds__(NT) void k_bias_join(const float* part, int chunks, int cols, float* gb) {
  const int v = blockIdx.x * NT + threadIdx.x;
  if (v >= cols) return;
  float s = 0.f;
  for (int c = 0; c < chunks; ++c) s += part[(int64_t)c * cols + v];
  gb[v] = s;
}
int bias_chunks(int64_t rows) { return (int)(rows < 64 ? rows : 64); }

// ---- policy/value loss -------------------------------------------------------------------------------------
// Statistics of a row or a piece of it: the largest logit, sum exp(z - top), sum pi, sum pi (z - top).
struct Soft {
  float top, total, pi, dot;
};

// The statistics of two pieces joined: each sum moves from its own top to the larger one.  A piece whose
// top is -inf has no finite logit: its total is 0 (or NaN) and its dot 0 (no target there) or infinite already.
__device__ __forceinline__ Soft join(const Soft& a, const Soft& b) {
  Soft r;
  r.top = fmaxf(a.top, b.top);
  const float da = a.top == -INFINITY ? 0.f : a.top - r.top, db = b.top == -INFINITY ? 0.f : b.top - r.top;
  r.total = a.total * expf(da) + b.total * expf(db);
  r.pi = a.pi + b.pi;
  r.dot = (a.dot + da * a.pi) + (b.dot + db * b.pi);
  return r;
}
__device__ __forceinline__ Soft wave_join(Soft s) {
  for (int o = 32; o; o >>= 1) {
    const Soft t = {__shfl_xor(s.top, o), __shfl_xor(s.total, o), __shfl_xor(s.pi, o), __shfl_xor(s.dot, o)};
    s = (threadIdx.x & o) ? join(t, s) : join(s, t);   // lower lane first on both sides: the same sums
  }
  return s;
}

template <int DT, int DP>
__global__ __launch_bounds__(NT) void k_loss_part(const typename Elem<DT>::T* z, int64_t z_stride,
                                                  const typename Elem<DP>::T* pi, int64_t pi_stride, int cols,
                                                  int tiles, Legal legal, Soft* part) {
  const int64_t row = blockIdx.x / tiles;
  const int v0 = (int)(blockIdx.x % tiles) * TILE;
  const int nv = min(TILE, cols - v0);
  constexpr int REP = TILE / (PER * NT);
  Pack<typename Elem<DT>::T, PER> q[REP];
  uint32_t ok[REP];
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < REP; ++k) {
    const int i = PER * (threadIdx.x + NT * k), n = nv - i;
    ok[k] = 0;
    if (n <= 0) continue;
    ok[k] = legal.four(row, v0 + i) & (n < PER ? (1u << n) - 1u : 15u);
    q[k] = load4(z + row * z_stride + v0 + i, n);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if ((ok[k] >> j) & 1u) top = fmaxf(top, Elem<DT>::get(q[k].v[j]));
  }
  Soft s = {top, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < REP; ++k) {
    const int i = PER * (threadIdx.x + NT * k), n = nv - i;
    if (!ok[k]) continue;
    const Pack<typename Elem<DP>::T, PER> t = load4(pi + row * pi_stride + v0 + i, n);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if ((ok[k] >> j) & 1u) {
        const float w = Elem<DP>::get(t.v[j]), x = Elem<DT>::get(q[k].v[j]);
        const float d = x == -INFINITY ? -INFINITY : x - top;
        s.total += d == -INFINITY ? 0.f : expf(d);
        s.pi += w;
        if (w != 0.f) s.dot += w * d;
      }
  }
  __shared__ Soft ws[NT / 64];
  s = wave_join(s);
  if (threadIdx.x % 64 == 0) ws[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NT / 64; ++w) s = join(s, ws[w]);
    part[blockIdx.x] = s;
  }
}

// The gradient of one element from the row's statistics {top, 1 / total, sum pi}
__device__ __forceinline__ float loss_slope(float x, float w, const float* st, float k) {
  const float e = x == -INFINITY ? 0.f : expf(x - st[0]) * st[1];
  return k * (st[1] == 0.f ? 0.f : e * st[2] - w);
}

template <int DT, int DP>
__device__ __forceinline__ void loss_grad_tile(const typename Elem<DT>::T* z, const typename Elem<DP>::T* pi,
                                               typename Elem<DT>::T* g, int64_t row, int v0, int nv, const Legal& legal,
                                               const float* st, float k) {
  for (int i = PER * threadIdx.x; i < nv; i += PER * NT) {
    const int n = nv - i;
    const uint32_t ok = legal.four(row, v0 + i);
    Pack<typename Elem<DT>::T, PER> q = load4(z + i, n);
    const Pack<typename Elem<DP>::T, PER> t = load4(pi + i, n);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      q.v[j] = Elem<DT>::put((ok >> j) & 1u ? loss_slope(Elem<DT>::get(q.v[j]), Elem<DP>::get(t.v[j]), st, k) : 0.f);
    store4(g + i, q, n);
  }
}

// Joins the row's tiles (every workgroup of a row the same way), writes its own tile of the gradient; the
// row's first workgroup writes its statistics and loss.
template <int DT, int DP>
__global__ __launch_bounds__(NT) void k_loss_row(const typename Elem<DT>::T* z, int64_t z_stride,
                                                 const typename Elem<DP>::T* pi, int64_t pi_stride, int cols,
                                                 int tiles, Legal legal, const Soft* part, const float* value,
                                                 const float* reward, float* stats, typename Elem<DT>::T* grad,
                                                 int64_t grad_stride, float* value_grad, float k) {
  const int64_t row = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x % tiles), v0 = tile * TILE;
  __shared__ float st[4];
  if (threadIdx.x < 64) {
    Soft s = {-INFINITY, 0.f, 0.f, 0.f};
    for (int t = threadIdx.x; t < tiles; t += 64) s = join(s, part[row * tiles + t]);
    s = wave_join(s);
    if (threadIdx.x == 0) {
      const bool some = s.top != -INFINITY || s.total != 0.f;   // a NaN among the logits is no empty row
      float loss = some ? s.pi * logf(s.total) - s.dot : 0.f;
      st[0] = s.top;
      st[1] = some ? 1.f / s.total : 0.f;
      st[2] = s.pi;
      if (tile == 0) {
        if (value) {
          const float d = value[row] - reward[row];
          loss += d * d;
          if (value_grad) value_grad[row] = 2.f * k * d;
        }
        float* o = stats + 4 * row;
        o[0] = st[0], o[1] = st[1], o[2] = st[2], o[3] = loss;
      }
    }
  }
  if (!grad) return;
  __syncthreads();
  loss_grad_tile<DT, DP>(z + row * z_stride + v0, pi + row * pi_stride + v0, grad + row * grad_stride + v0, row, v0,
                         min(TILE, cols - v0), legal, st, k);
}

template <int DT, int DP>
__global__ __launch_bounds__(NT) void k_loss_grad(const typename Elem<DT>::T* z, int64_t z_stride,
                                                  const typename Elem<DP>::T* pi, int64_t pi_stride, int64_t rows,
                                                  int cols, int tiles, Legal legal, const float* value,
                                                  const float* reward, const float* stats, const float* grad_out,
                                                  typename Elem<DT>::T* grad, int64_t grad_stride, float* value_grad) {
  const int64_t row = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x % tiles), v0 = tile * TILE;
  const float k = *grad_out / (float)rows;
  if (value_grad && tile == 0 && threadIdx.x == 0) value_grad[row] = 2.f * k * (value[row] - reward[row]);
  if (!grad) return;
  const float st[3] = {stats[4 * row], stats[4 * row + 1], stats[4 * row + 2]};
  loss_grad_tile<DT, DP>(z + row * z_stride + v0, pi + row * pi_stride + v0, grad + row * grad_stride + v0, row, v0,
                         min(TILE, cols - v0), legal, st, k);
}

// The mean of the rows' losses by one workgroup, in a fixed order and in 64 bits
__global__ __launch_bounds__(1024) void k_loss_mean(const float* stats, int64_t rows, float* loss) {
  double s = 0.;
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

const char* bad_shape(int64_t rows, int64_t cols, int dtype) {
  if (rows < 0) return "rows must not be negative";
  if (cols < 1 || cols > MOST_COLS) return "cols must be in [1, 2^24]";
  if (rows * ((cols + TILE - 1) / TILE) > INT32_MAX || rows > INT32_MAX) return "too many rows for one call";
  if (dtype < MTAZ_F32 || dtype > MTAZ_BF16) return "unknown element type";
  return nullptr;
}
const char* bad_taken(const int32_t* actions, int64_t stride, int history, const double* penalties,
                      const float* per_row) {
  if (history < 0) return "history must not be negative";
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
  if (!per_row) t.repetition = (float)penalties[0], t.frequency = (float)penalties[1], t.presence = (float)penalties[2];
  return t;
}
int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(e));
}
int tiles_of(int64_t cols) { return (int)((cols + TILE - 1) / TILE); }

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
  if (!bad && d_out == d_logits && out_stride != logits_stride && rows > 1) bad = "in place needs equal strides";
  if (bad) return ops_error(MTAZ_E_FAIL, "adjust_logits", bad);
  if (rows == 0) return 0;
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, "adjust_logits", hipGetErrorString(on.status));
  const int tiles = tiles_of(cols);
  const Taken t = taken_of(d_actions, actions_stride, history, d_lengths, penalties, d_penalties);
  FOR_TYPE(dtype, (k_adjust<DT><<<(unsigned)(rows * tiles), NT, 0, (hipStream_t)stream>>>(
                      (const Elem<DT>::T*)d_logits, logits_stride, (Elem<DT>::T*)d_out, out_stride, (int)cols, tiles,
                      Legal{d_legal, legal_stride}, d_bias, bias_stride, t)));
  return launched("adjust_logits");
}

extern "C" int64_t mtaz_adjust_logits_grad_workspace(int64_t rows, int64_t cols) {
  if (const char* bad = bad_shape(rows, cols, MTAZ_F32)) return ops_error(MTAZ_E_FAIL, "adjust_logits_grad", bad);
  return 4 * cols * bias_chunks(rows);
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
  const Taken t = bad ? Taken{} : taken_of(d_actions, actions_stride, history, d_lengths, penalties, d_penalties);
  const bool shared = d_bias_grad && bias_grad_stride == 0;
  if (!bad && rows && !d_grad_out) bad = "no incoming gradient";
  if (!bad && rows && t.actions && d_grad && !d_logits) bad = "the penalties' gradient needs the logits";
  if (!bad && rows > 1 && ((d_grad && grad_stride < cols) || (d_bias_grad && !shared && bias_grad_stride < cols)))
    bad = "rows of an output overlap";
  if (!bad && shared && rows && (!d_work || work_bytes < 4 * cols * bias_chunks(rows))) bad = "workspace too small";
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const hipStream_t s = (hipStream_t)stream;
  const int tiles = tiles_of(cols), nc = (int)cols;
  const Legal legal{d_legal, legal_stride};
  float* row_bias = shared ? nullptr : d_bias_grad;
  const int chunks = bias_chunks(rows);
  const int64_t per_chunk = chunks ? (rows + chunks - 1) / chunks : 0;
  FOR_TYPE(dtype, {
    if (rows && (d_grad || row_bias))
      k_adjust_grad<DT><<<(unsigned)(rows * tiles), NT, 0, s>>>((const Elem<DT>::T*)d_grad_out, grad_out_stride,
                                                              (const Elem<DT>::T*)d_logits, logits_stride,
                                                              (Elem<DT>::T*)d_grad, grad_stride, row_bias,
                                                              bias_grad_stride, nc, tiles, legal, t);
    if (shared && rows)
      k_bias_sum<DT><<<dim3((nc + BIAS_COLS - 1) / BIAS_COLS, chunks), NT, 0, s>>>(
          (const Elem<DT>::T*)d_grad_out, grad_out_stride, rows, per_chunk, nc, legal, (float*)d_work);
  });
  if (shared) k_bias_join<<<(nc + NT - 1) / NT, NT, 0, s>>>((const float*)d_work, chunks, nc, d_bias_grad);
  return launched(what);
}

extern "C" int64_t mtaz_policy_loss_workspace(int64_t rows, int64_t cols) {
  if (const char* bad = bad_shape(rows, cols, MTAZ_F32)) return ops_error(MTAZ_E_FAIL, "policy_loss", bad);
  return (int64_t)sizeof(Soft) * rows * tiles_of(cols);
}

static const char* bad_loss(int64_t rows, int64_t cols, int dtype, int target_dtype, const void* logits,
                            const void* target, const float* value, const float* reward, const float* stats,
                            const void* grad, int64_t grad_stride, const float* value_grad) {
  if (const char* bad = bad_shape(rows, cols, dtype)) return bad;
  if (rows < 1) return "the mean of no rows";
  if (target_dtype != MTAZ_F32 && target_dtype != dtype) return "targets are float32 or of the logits' type";
  if (!logits || !target || !stats) return "no logits, targets or statistics";
  if (!value != !reward) return "a value without a reward, or a reward without a value";
  if (value_grad && !value) return "the gradient of a value that is not there";
  if (grad && grad_stride < cols && rows > 1) return "rows of the gradient overlap";
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
  if (!bad && (!d_work || work_bytes < (int64_t)sizeof(Soft) * rows * tiles_of(cols))) bad = "workspace too small";
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const hipStream_t s = (hipStream_t)stream;
  const int tiles = tiles_of(cols), nc = (int)cols;
  const unsigned grid = (unsigned)(rows * tiles);
  const Legal legal{d_legal, legal_stride};
  const float k = (float)(scale / (double)rows);
  FOR_TYPES(dtype, target_dtype, {
    const auto* z = (const Elem<DT>::T*)d_logits;
    const auto* pi = (const Elem<DP>::T*)d_target;
    k_loss_part<DT, DP><<<grid, NT, 0, s>>>(z, logits_stride, pi, target_stride, nc, tiles, legal, (Soft*)d_work);
    // without a gradient one workgroup per row joins its tiles
    k_loss_row<DT, DP><<<grid, NT, 0, s>>>(z, logits_stride, pi, target_stride, nc, tiles, legal, (const Soft*)d_work,
                                          d_value, d_reward, d_stats, (Elem<DT>::T*)d_grad, grad_stride, d_value_grad,
                                          k);
  });
  k_loss_mean<<<1, 1024, 0, s>>>(d_stats, rows, d_loss);
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
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  if (!d_grad && !d_value_grad) return 0;
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const int tiles = tiles_of(cols), nc = (int)cols;
  FOR_TYPES(dtype, target_dtype,
            (k_loss_grad<DT, DP><<<(unsigned)(rows * tiles), NT, 0, (hipStream_t)stream>>>(
                (const Elem<DT>::T*)d_logits, logits_stride, (const Elem<DP>::T*)d_target, target_stride, rows, nc,
                tiles, Legal{d_legal, legal_stride}, d_value, d_reward, d_stats, d_grad_out, (Elem<DT>::T*)d_grad,
                grad_stride, d_value_grad)));
  return launched(what);
}
