// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step around it.
//
// With r the shorter and L the longer side, X [r][L] (a tall matrix transposed) and the coefficients a, b, c:
//   X <- G / (|G|_F + eps);    steps times:  S = X X^T,  B = b S + c S S,  X <- a X + B X.
//
// The products run on the f16 matrix cores and keep 32-bit accuracy: a value x is held as two f16 numbers,
// hi = f16(2^e x) and lo = f16(2^e x - hi), together 22 bits, and a product is hi hi + hi lo + lo hi with
// float sums (lo lo is below the last bit kept).  2^e brings the largest value the matrix can hold below
// 2^14: all entries of X, S and B are bounded by their spectral norms, and those follow from the
// coefficients alone, since the first X has norm at most 1 (bounds()).  Against the f32 matrix instruction
// (157 TFLOP/s) the split has a third of the f16 rate, about 5 times as much.
//
// X, S and B lie in the workspace as hi and lo planes, padded with zeros to whole tiles, so that the product
// kernel checks no bounds; a padded row or column stays zero through every step.
#include "ops.h"

#include <math.h>

namespace mtaz {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NT = 256;
constexpr int MOST = 64;      // matrices per launch: their pointers travel as kernel arguments
constexpr int PAD = 64;       // rows and columns of the planes are multiples of it
constexpr int PARTS = 64;     // workgroups per matrix for the sum of squares

struct Matrices {
  const void* grad[MOST];
  void* out[MOST];            // the result, or the parameter
  float* momentum[MOST];      // null: no momentum
};
struct Shape {
  int rows, cols;             // of the matrix as it lies in memory
  int r, L;                   // short and long side
  int rp, Lp;                 // padded
};
struct Update {
  float momentum, keep, step;   // m <- momentum m + (1 - momentum) g;  w <- keep w - step O
  int nesterov;
};
// hi and lo planes of n matrices [rows][pitch], one after the other
struct Planes {
  _Float16 *hi, *lo;
  int64_t each;               // elements of one matrix
  int pitch;
};

// ---- the matrix to orthogonalise: sum of squares, then the planes of X -----------------------------------------
template <int DT, bool MUON>
__device__ __forceinline__ float update_of(float g, float m, const Update& u) {
  return MUON ? (u.nesterov ? fmaf(u.momentum, m, (1.f - u.momentum) * g) : m) : g;
}

// Partial sums of squares in 64 bits: neither large nor tiny gradients leave the range.  With momentum, the
// pass also brings it up to date.
template <int DT, bool MUON>
__global__ __launch_bounds__(NT) void k_squares(Matrices ms, int64_t count, Update u, double* part) {
  typedef Elem<DT> E;
  const int i = blockIdx.y;
  const typename E::T* g = (const typename E::T*)ms.grad[i];
  float* mom = ms.momentum[i];
  double s = 0.;
  for (int64_t k = 4 * ((int64_t)blockIdx.x * NT + threadIdx.x); k < count; k += 4 * NT * PARTS) {
    const int n = (int)min((int64_t)4, count - k);
    for (int j = 0; j < n; ++j) {
      const float gv = E::get(g[k + j]);
      float mv = 0.f;
      if (MUON) {
        mv = fmaf(u.momentum, mom[k + j], (1.f - u.momentum) * gv);
        mom[k + j] = mv;
      }
      const double x = (double)update_of<DT, MUON>(gv, mv, u);
      s += x * x;
    }
  }
  __shared__ double ws[NT / 64];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if (threadIdx.x % 64 == 0) ws[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[i * PARTS + blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

__device__ __forceinline__ void split(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// X = matrix * 2^e / (norm + eps) in planes, transposed where the matrix is tall; 64 x 64 elements per workgroup
template <int DT, bool MUON>
__global__ __launch_bounds__(NT) void k_planes(Matrices ms, Shape sh, Update u, const double* part, double eps,
                                               double unit, Planes X) {
  typedef Elem<DT> E;
  const int i = blockIdx.z;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;   // of X
  __shared__ double inv;
  __shared__ float tile[64][65];
  if (threadIdx.x < 64) {
    double s = part[i * PARTS + threadIdx.x];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if (threadIdx.x == 0) inv = unit / (sqrt(s) + eps);
  }
  __syncthreads();
  const bool tall = sh.rows > sh.cols;
  const typename E::T* g = (const typename E::T*)ms.grad[i];
  const float* mom = ms.momentum[i];
  for (int k = threadIdx.x; k < 64 * 64; k += NT) {
    const int a = k >> 6, b = k & 63;                     // b runs along the memory of the matrix
    const int row = tall ? c0 + a : r0 + a, col = tall ? r0 + b : c0 + b;
    float x = 0.f;
    if (row < sh.rows && col < sh.cols) {
      const int64_t at = (int64_t)row * sh.cols + col;
      x = (float)((double)update_of<DT, MUON>(E::get(g[at]), MUON ? mom[at] : 0.f, u) * inv);
    }
    if (tall) tile[b][a] = x; else tile[a][b] = x;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 64 * 8; k += NT) {
    const int a = k >> 3, b = (k & 7) * 8;
    f16x8 h, l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      _Float16 hj, lj;
      split(tile[a][b + j], hj, lj);
      h[j] = hj, l[j] = lj;
    }
    const int64_t at = i * X.each + (int64_t)(r0 + a) * X.pitch + c0 + b;
    *reinterpret_cast<f16x8*>(X.hi + at) = h;
    *reinterpret_cast<f16x8*>(X.lo + at) = l;
  }
}

// ---- products --------------------------------------------------------------------------------------------------
// One workgroup: D[m][n] = sum_k P[m][k] Q[n][k] for a T x T tile, 4 waves of T/2 x T/2 on the 32x32x16 instruction.
//   GRAM    P = Q = X:  S, the tiles on and below the diagonal, each written twice
//   POLY    P = Q = S:  B = b S + c S S, likewise
//   APPLY   P = X transposed while it is read from LDS, Q = B:  X <- a X + B X (m runs along X's rows in memory)
//   LAST_*  APPLY whose result leaves the planes: orthogonalised, or subtracted from the parameter
enum Kind { GRAM, POLY, APPLY, LAST_OUT, LAST_MUON };
constexpr int BK = 32;

struct Product {
  Planes P, Q, D;
  int k;                // depth, a multiple of BK
  int tiles_m;          // tiles along m (APPLY)
  float self, acc;      // D = self * (the element of S or X) + acc * sum
};

// 16 bytes a lane straight into LDS; the wave's 64 pieces lie there in lane order
__device__ __forceinline__ void to_lds(const _Float16* from, _Float16* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// T rows of BK elements (64 B): 4 pieces a row, piece p of row m at p ^ (m >> 2 & 3), so that the 16 lanes that
// read one piece of 16 rows meet 16 different bank groups
template <int T>
__device__ __forceinline__ void load_rows(const _Float16* g, int pitch, int k0, _Float16* lds, int wave, int lane) {
  for (int c = wave; c < T / 16; c += 4) {
    const int m = c * 16 + (lane >> 2), p = (lane & 3) ^ ((m >> 2) & 3);
    to_lds(g + (int64_t)m * pitch + k0 + p * 8, lds + c * 512);
  }
}
template <int T>
__device__ __forceinline__ f16x8 read_rows(const _Float16* lds, int m, int p) {
  return *reinterpret_cast<const f16x8*>(lds + m * BK + ((p ^ ((m >> 2) & 3)) * 8));
}
// BK rows of T elements; piece p of row k lies at p ^ swz(k): the four rows one transposing read touches lie in
// different banks
template <int T> __device__ __forceinline__ int swz(int k) { return T == 128 ? (k & 3) << 2 : ((k >> 1) & 1) << 2; }
template <int T>
__device__ __forceinline__ void load_cols(const _Float16* g, int pitch, int k0, _Float16* lds, int wave, int lane) {
  constexpr int PR = T / 8, RW = 64 / PR;               // pieces a row, rows a wave
  for (int c = wave; c < BK / RW; c += 4) {
    const int k = c * RW + lane / PR, p = (lane % PR) ^ swz<T>(k);
    to_lds(g + (int64_t)(k0 + k) * pitch + p * 8, lds + c * 512);
  }
}
// elements k .. k + 7 of column m (k a multiple of 8, m = the lane's): two transposing reads of 4 rows x 16 columns
template <int T>
__device__ __forceinline__ f16x8 read_cols(const _Float16* lds, int m0, int k0, int lane) {
  const int q = lane & 15, col = m0 + ((lane >> 4) & 1) * 16 + (q & 3) * 4;
  f16x8 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = k0 + (lane >> 5) * 8 + h * 4 + (q >> 2);
    const _Float16* at = lds + k * T + ((((col >> 3) ^ swz<T>(k)) << 3) | (col & 7));
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)const_cast<_Float16*>(at));
    const f16x4 f = __builtin_bit_cast(f16x4, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[4 * h + j] = f[j];
  }
  return r;
}

template <int T, int KIND, int DT>
__global__ __launch_bounds__(NT) void k_product(Product pr, Matrices ms, Shape sh, Update u) {
  constexpr bool COLS = KIND >= APPLY;
  constexpr int W = T / 2, F = W / 32;
  __shared__ __attribute__((aligned(16))) _Float16 lds[4 * T * BK];
  _Float16 *ph = lds, *pl = lds + T * BK, *qh = lds + 2 * T * BK, *ql = lds + 3 * T * BK;
  const int i = blockIdx.y, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int bm, bn;
  if (COLS) {
    bm = blockIdx.x % pr.tiles_m, bn = blockIdx.x / pr.tiles_m;
  } else {                                              // lower triangle, row by row
    bm = (int)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
    if ((bm + 1) * (bm + 2) / 2 <= (int)blockIdx.x) ++bm;
    if (bm * (bm + 1) / 2 > (int)blockIdx.x) --bm;
    bn = blockIdx.x - bm * (bm + 1) / 2;
  }
  const _Float16* gph = pr.P.hi + i * pr.P.each + (COLS ? (int64_t)bm * T : (int64_t)bm * T * pr.P.pitch);
  const _Float16* gpl = pr.P.lo + i * pr.P.each + (COLS ? (int64_t)bm * T : (int64_t)bm * T * pr.P.pitch);
  const _Float16* gqh = pr.Q.hi + i * pr.Q.each + (int64_t)bn * T * pr.Q.pitch;
  const _Float16* gql = pr.Q.lo + i * pr.Q.each + (int64_t)bn * T * pr.Q.pitch;
  const int m0 = (wave & 1) * W, n0 = (wave >> 1) * W;

  f32x16 acc[F][F] = {};
  for (int k0 = 0; k0 < pr.k; k0 += BK) {
    if (COLS) {
      load_cols<T>(gph, pr.P.pitch, k0, ph, wave, lane);
      load_cols<T>(gpl, pr.P.pitch, k0, pl, wave, lane);
    } else {
      load_rows<T>(gph, pr.P.pitch, k0, ph, wave, lane);
      load_rows<T>(gpl, pr.P.pitch, k0, pl, wave, lane);
    }
    load_rows<T>(gqh, pr.Q.pitch, k0, qh, wave, lane);
    load_rows<T>(gql, pr.Q.pitch, k0, ql, wave, lane);
    __builtin_amdgcn_s_waitcnt(0x0f70);                 // vmcnt(0): this wave's pieces are in LDS
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < BK; kk += 16) {
      f16x8 ah[F], al[F], bh[F], bl[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        if (COLS) {
          ah[f] = read_cols<T>(ph, m0 + 32 * f, kk, lane);
          al[f] = read_cols<T>(pl, m0 + 32 * f, kk, lane);
        } else {
          ah[f] = read_rows<T>(ph, m0 + 32 * f + (lane & 31), kk / 8 + (lane >> 5));
          al[f] = read_rows<T>(pl, m0 + 32 * f + (lane & 31), kk / 8 + (lane >> 5));
        }
        bh[f] = read_rows<T>(qh, n0 + 32 * f + (lane & 31), kk / 8 + (lane >> 5));
        bl[f] = read_rows<T>(ql, n0 + 32 * f + (lane & 31), kk / 8 + (lane >> 5));
      }
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < F; ++g) {
          acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[f], bh[g], acc[f][g], 0, 0, 0);
          acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[f], bl[g], acc[f][g], 0, 0, 0);
          acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[f], bh[g], acc[f][g], 0, 0, 0);
        }
    }
    __syncthreads();
  }

  // a lane holds column n and, four at a time, consecutive rows m
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int g = 0; g < F; ++g)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = bm * T + m0 + 32 * f + 8 * q + 4 * (lane >> 5);
        const int n = bn * T + n0 + 32 * g + (lane & 31);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = pr.acc * acc[f][g][4 * q + j];
        if (KIND != GRAM) {
          const Planes& A = pr.P;                       // S, or X
          const int64_t at = i * A.each + (int64_t)n * A.pitch + m;
          const f16x4 h = *reinterpret_cast<const f16x4*>(A.hi + at), l = *reinterpret_cast<const f16x4*>(A.lo + at);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = fmaf(pr.self, (float)h[j] + (float)l[j], v[j]);
        }
        if (KIND <= APPLY) {
          f16x4 h, l;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            _Float16 hj, lj;
            split(v[j], hj, lj);
            h[j] = hj, l[j] = lj;
          }
          const int64_t at = i * pr.D.each + (int64_t)n * pr.D.pitch + m;
          *reinterpret_cast<f16x4*>(pr.D.hi + at) = h;
          *reinterpret_cast<f16x4*>(pr.D.lo + at) = l;
          if (KIND != APPLY && bm != bn) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int64_t to = i * pr.D.each + (int64_t)(m + j) * pr.D.pitch + n;
              pr.D.hi[to] = h[j], pr.D.lo[to] = l[j];
            }
          }
        } else {
          typedef Elem<DT> E;
          typename E::T* o = (typename E::T*)ms.out[i];
          const bool tall = sh.rows > sh.cols;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (n >= sh.r || m + j >= sh.L) continue;
            const int64_t at = tall ? (int64_t)(m + j) * sh.cols + n : (int64_t)n * sh.cols + m + j;
            o[at] = E::put(KIND == LAST_MUON ? fmaf(u.keep, E::get(o[at]), -u.step * v[j]) : v[j]);
          }
        }
      }
}

// ---- host --------------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

struct Work {
  double* part;
  Planes X[2], S, B;
  int64_t bytes;
};
Work layout(int n, const Shape& sh, char* base) {
  Work w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = base ? base + at : nullptr;
    at += up(bytes, 256);
    return p;
  };
  auto planes = [&](int rows, int pitch) {
    Planes p;
    p.each = (int64_t)rows * pitch, p.pitch = pitch;
    p.hi = (_Float16*)take(2 * p.each * n);
    p.lo = (_Float16*)take(2 * p.each * n);
    return p;
  };
  w.part = (double*)take(8 * PARTS * n);
  w.X[0] = planes(sh.rp, sh.Lp);
  w.X[1] = planes(sh.rp, sh.Lp);
  w.S = planes(sh.rp, sh.rp);
  w.B = planes(sh.rp, sh.rp);
  w.bytes = at;
  return w;
}

Shape shape_of(int64_t rows, int64_t cols) {
  Shape s;
  s.rows = (int)rows, s.cols = (int)cols;
  s.r = (int)(rows < cols ? rows : cols), s.L = (int)(rows < cols ? cols : rows);
  s.rp = (int)up(s.r, PAD), s.Lp = (int)up(s.L, PAD);
  return s;
}

const char* bad_shape(int n, int64_t rows, int64_t cols, int dtype) {
  if (n < 0) return "n must not be negative";
  if (rows < 1 || cols < 1 || rows > 65536 || cols > 65536 || rows * cols > (1 << 30))
    return "rows and cols must be in [1, 65536] and their product at most 2^30";
  if (dtype < MTAZ_F32 || dtype > MTAZ_BF16) return "unknown element type";
  return nullptr;
}

// Exponents that keep every entry below 2^14: of X before each step and after the last, of S and of B.
// Singular values start in [0, 1]; after a step they lie below the largest |s (a + b s^2 + c s^4)| over the range
// before it, S below its square and B below the largest |b s^2 + c s^4|.  The maxima are taken over a grid that holds
// the range's end, where a polynomial between two of 4096 points exceeds the larger one by some 10^-7 of its
// maximum, with a thousandth on top for that and for roundings; f16 has room for twice 2^14 besides.
struct Exponents {
  int x[MTAZ_MAX_STEPS + 1], s[MTAZ_MAX_STEPS], b[MTAZ_MAX_STEPS];
};
const char* bounds(int steps, const double* co, Exponents& e) {
  double top = 1.;
  auto unit = [](double bound) {
    const int k = 14 - (int)ceil(log2(bound));
    return k > 40 ? 40 : k;
  };
  for (int t = 0; t <= steps; ++t) {
    if (!(top <= 1e6)) return "the coefficients let the singular values grow past 10^6";
    e.x[t] = unit(top > 1e-9 ? top : 1e-9);
    if (t == steps) break;
    double next = 0., poly = 0.;
    for (int k = 0; k <= 4096; ++k) {
      const double s = top * k / 4096., q = co[1] * s * s + co[2] * s * s * s * s;
      next = fmax(next, fabs(s * (co[0] + q))), poly = fmax(poly, fabs(q));
    }
    e.s[t] = unit(fmax(1.001 * top * top, 1e-9));
    e.b[t] = unit(fmax(1.001 * poly, 1e-9));
    top = 1.001 * next;
  }
  return nullptr;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(e));
}

template <int T, int KIND, int DT>
void product(const Product& pr, int tiles, int n, const Matrices& ms, const Shape& sh, const Update& u, hipStream_t s) {
  k_product<T, KIND, DT><<<dim3(tiles, n), NT, 0, s>>>(pr, ms, sh, u);
}

template <int DT, bool MUON>
void iterate(const Matrices& ms, int n, const Shape& sh, const Update& u, int steps, const double* co, double eps,
             const Exponents& e, char* base, hipStream_t s) {
  constexpr int T = 64;
  const Work w = layout(n, sh, base);
  const int64_t count = (int64_t)sh.rows * sh.cols;
  k_squares<DT, MUON><<<dim3(PARTS, n), NT, 0, s>>>(ms, count, u, w.part);
  k_planes<DT, MUON><<<dim3(sh.Lp / 64, sh.rp / 64, n), NT, 0, s>>>(ms, sh, u, w.part, eps, ldexp(1., e.x[0]), w.X[0]);
  const int tr = sh.rp / T, tL = sh.Lp / T, tri = tr * (tr + 1) / 2;
  for (int t = 0; t < steps; ++t) {
    const Planes &X = w.X[t & 1], &Y = w.X[(t + 1) & 1];
    Product p = {X, X, w.S, sh.Lp, 0, 0.f, (float)ldexp(1., e.s[t] - 2 * e.x[t])};
    product<T, GRAM, MTAZ_F32>(p, tri, n, ms, sh, u, s);
    p = {w.S, w.S, w.B, sh.rp, 0, (float)ldexp(co[1], e.b[t] - e.s[t]), (float)ldexp(co[2], e.b[t] - 2 * e.s[t])};
    product<T, POLY, MTAZ_F32>(p, tri, n, ms, sh, u, s);
    const int ex = t + 1 < steps ? e.x[t + 1] : 0;
    p = {X, w.B, Y, sh.rp, tL, (float)ldexp(co[0], ex - e.x[t]), (float)ldexp(1., ex - e.x[t] - e.b[t])};
    if (t + 1 < steps)
      product<T, APPLY, MTAZ_F32>(p, tr * tL, n, ms, sh, u, s);
    else
      product<T, MUON ? LAST_MUON : LAST_OUT, DT>(p, tr * tL, n, ms, sh, u, s);
  }
}

// All checks, then the matrices in groups of at most MOST over the same workspace
template <bool MUON>
int run(const char* what, int device, int n, int64_t rows, int64_t cols, int dtype, const void* const* grad,
        void* const* out, float* const* momenta, const Update& u, int steps, const double* co, double eps, void* work,
        int64_t work_bytes, void* stream) {
  Exponents e;
  const char* bad = bad_shape(n, rows, cols, dtype);
  if (!bad && n && (!grad || !out || (MUON && !momenta))) bad = "no matrices";
  if (!bad && (steps < 1 || steps > MTAZ_MAX_STEPS)) bad = "steps must be in [1, 32]";
  if (!bad && (!co || !isfinite(co[0]) || !isfinite(co[1]) || !isfinite(co[2]))) bad = "coefficients must be finite";
  if (!bad && !(eps >= 0.)) bad = "eps must not be negative";
  if (!bad) bad = bounds(steps, co, e);
  if (bad) return ops_error(MTAZ_E_FAIL, what, bad);
  for (int i = 0; i < n; ++i)
    if (!grad[i] || !out[i] || (MUON && !momenta[i])) return ops_error(MTAZ_E_FAIL, what, "a null matrix");
  if (n == 0) return 0;
  const Shape sh = shape_of(rows, cols);
  if (!work || ((uintptr_t)work & 255) || work_bytes < layout(n < MOST ? n : MOST, sh, nullptr).bytes)
    return ops_error(MTAZ_E_FAIL, what, "workspace too small or not aligned to 256 bytes");
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  for (int first = 0; first < n; first += MOST) {
    const int m = n - first < MOST ? n - first : MOST;
    Matrices ms = {};
    for (int i = 0; i < m; ++i) {
      ms.grad[i] = grad[first + i], ms.out[i] = out[first + i];
      if (MUON) ms.momentum[i] = momenta[first + i];
    }
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == MTAZ_F32) iterate<MTAZ_F32, MUON>(ms, m, sh, u, steps, co, eps, e, (char*)work, s);
    else if (dtype == MTAZ_F16) iterate<MTAZ_F16, MUON>(ms, m, sh, u, steps, co, eps, e, (char*)work, s);
    else iterate<MTAZ_BF16, MUON>(ms, m, sh, u, steps, co, eps, e, (char*)work, s);
  }
  return launched(what);
}

}  // namespace
}  // namespace mtaz

using namespace mtaz;

extern "C" int64_t mtaz_orthogonalize_workspace(int n, int64_t rows, int64_t cols, int dtype) {
  if (const char* bad = bad_shape(n, rows, cols, dtype)) return ops_error(MTAZ_E_FAIL, "orthogonalize", bad);
  return layout(n < MOST ? n : MOST, shape_of(rows, cols), nullptr).bytes;
}

extern "C" int mtaz_orthogonalize(int device, int n, int64_t rows, int64_t cols, int dtype, const void* const* d_grad,
                                  void* const* d_out, int steps, const double* coefficients, double eps, void* d_work,
                                  int64_t work_bytes, void* stream) {
  return run<false>("orthogonalize", device, n, rows, cols, dtype, d_grad, d_out, nullptr, Update{}, steps,
                    coefficients, eps, d_work, work_bytes, stream);
}

extern "C" int mtaz_muon_step(int device, int n, int64_t rows, int64_t cols, int dtype, void* const* d_params,
                              const void* const* d_grads, float* const* d_momenta, double lr, double momentum,
                              int nesterov, double weight_decay, double scale, int steps, const double* coefficients,
                              double eps, void* d_work, int64_t work_bytes, void* stream) {
  if (!(momentum >= 0. && momentum < 1.)) return ops_error(MTAZ_E_FAIL, "muon_step", "momentum must be in [0, 1)");
  if (!isfinite(lr) || !isfinite(weight_decay) || !isfinite(scale))
    return ops_error(MTAZ_E_FAIL, "muon_step", "lr, weight_decay and scale must be finite");
  const Update u = {(float)momentum, (float)(1. - lr * weight_decay), (float)(lr * scale), nesterov};
  return run<true>("muon_step", device, n, rows, cols, dtype, d_grads, d_params, d_momenta, u, steps, coefficients,
                   eps, d_work, work_bytes, stream);
}
