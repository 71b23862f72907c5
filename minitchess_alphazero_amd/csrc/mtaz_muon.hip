// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step around it.
//
// With r the shorter and L the longer side, X [r][L] (a tall matrix transposed) and the coefficients a, b, c:
//   X <- G / (|G|_F + eps);    steps times:  S = X X^T,  B = a I + b S + c S S,  X <- B X.
//
// The products run on the f16 matrix cores with factors of 22 bits: a value x is held as two f16 numbers,
// hi = f16(2^e x) and lo = f16(2^e x - hi), off by at most 2^-23 of x, and a product is hi hi + hi lo + lo hi with
// float sums (lo lo is below the last bit kept).  A float would hold 24 bits; the result is about as near to the
// definition all the same, because the sums are what loses most: against 64 bits, in shares of the error of the library's
// float products, 256 x 300 0.4 to 0.6, 509 x 1021 0.5 to 0.6, 1000 x 1536 0.3 to 0.5, 256 x 2304 0.6 to 0.7, 64 x 3000
// 1.0 to 1.4 (Gaussian matrices and gradients of few strong directions).  2^e brings the largest value the matrix can hold below
// 2^14: all entries of X, S and B are bounded by their spectral norms, and those follow from the
// coefficients alone, since the first X has norm at most 1 (bounds()).  Against the f32 matrix instruction
// (157 TFLOP/s) the split has a third of the f16 rate, about 5 times as much.
//
// X, S and B lie in the workspace as such pairs: a row is a run of 128-byte lines, each the hi and then the lo
// halves of 32 consecutive elements, so that one line is what a product reads of a row at a time.  They are padded
// with zeros to whole tiles, so that the product kernel checks no bounds; a padded row or column stays zero through
// every step.
//
// The products bound the large matrices: 1140 / 3 = 380 TFLOP/s at the rate that a large f16 product of the library
// reaches here, counting a symmetric product once.  2048 x 8192 bf16 with five steps takes 1311 us (404 GFLOP: 308),
// 18 x 256 x 2304 f32 270 us (35 GFLOP: 130; its products are 256 deep or 2304 long and wait for memory and for each
// other), and a matrix that fits into one CU's LDS is bound by the latency of its 15 products (554 x 61: 50 us).
//
// One factor of f16 alone would take a third of the products, and be off by 2^-12 in every X, S and B: a gradient with
// few strong directions has its weak ones, noise included, made up to 3.4 times larger a step, and five steps turn that
// into several per cent of the result.  So 16-bit matrices are computed like 32-bit ones, and rounded once.
#include "ops.h"

#include <math.h>

namespace mtaz {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int NT = 256;
constexpr int MOST = 64;      // matrices per launch: their pointers travel as kernel arguments
constexpr int PARTS = 256;    // most workgroups per matrix for the sum of squares

struct Matrices {
  const void* grad[MOST];
  void* out[MOST];            // the result, or the parameter
  float* momentum[MOST];      // null: no momentum
};
struct Shape {
  int rows, cols;             // of the matrix as it lies in memory
  int r, L;                   // short and long side
  int rp, Lp;                 // padded to whole tiles over r x L
  int tile_r, tile_L;         // tile of the products over r x r (64, 96 or 128) and over r x L (64 or 128)
  int height;                 // rows of X, S, B and C in memory: rp, padded to whole tiles over r x r; what lies behind
                              // rp is read, but by nothing that is kept
  int parts;                  // workgroups for the sum of squares
};
struct Update {
  float momentum, fresh, keep, step;   // m <- momentum m + fresh g, fresh = 1 - momentum;  w <- keep w - step O
  int nesterov;
};
// n matrices of pairs, one after the other
struct Pairs {
  _Float16* at;
  int64_t each;               // halves of one matrix
  int pitch;                  // halves of one row: twice the padded columns
  // the hi half of (row, col); its lo half lies 32 behind it
  __device__ __forceinline__ _Float16* hi(int i, int row, int col) const {
    return at + i * each + (int64_t)row * pitch + (col >> 5) * 64 + (col & 31);
  }
};

// ---- the matrix to orthogonalise: sum of squares, then the pairs of X -----------------------------------------
template <int DT, bool MUON>
__device__ __forceinline__ float update_of(float g, float m, const Update& u) {
  return MUON ? (u.nesterov ? fmaf(u.momentum, m, u.fresh * g) : m) : g;
}

// Partial sums of squares in 64 bits: neither large nor tiny gradients leave the range.  With momentum, the
// pass also brings it up to date.  Bound by memory: 18 x 256 x 2304 f32 8.4 us (42 MB, 5.0 TB/s), with momentum 22 us
// (127 MB, 5.8 TB/s).
template <int DT, bool MUON>
__global__ __launch_bounds__(NT) void k_squares(Matrices ms, int64_t count, Update u, double* part) {
  const int parts = gridDim.x;
  typedef Elem<DT> E;
  const int i = blockIdx.y;
  const typename E::T* g = (const typename E::T*)ms.grad[i];
  float* mom = ms.momentum[i];
  double s = 0.;
  constexpr int N = 8;
  for (int64_t k = N * ((int64_t)blockIdx.x * NT + threadIdx.x); k < count; k += (int64_t)N * NT * parts) {
    const int n = (int)min((int64_t)N, count - k);
    Pack<typename E::T, N> gv;
    Pack<float, N> mv;
    if (n == N) {
      gv = *reinterpret_cast<const Pack<typename E::T, N>*>(g + k);
      if (MUON) mv = *reinterpret_cast<const Pack<float, N>*>(mom + k);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) gv.v[j] = j < n ? g[k + j] : (typename E::T)0.f, mv.v[j] = MUON && j < n ? mom[k + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = E::get(gv.v[j]);
      if (MUON) mv.v[j] = fmaf(u.momentum, mv.v[j], u.fresh * x);
      const double y = (double)update_of<DT, MUON>(x, mv.v[j], u);
      s = fma(y, y, s);
    }
    if (MUON) {
      if (n == N) *reinterpret_cast<Pack<float, N>*>(mom + k) = mv;
      else
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < n) mom[k + j] = mv.v[j];
    }
  }
  __shared__ double ws[NT / 64];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if (threadIdx.x % 64 == 0) ws[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[i * parts + blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

__device__ __forceinline__ void split(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// eight consecutive elements (a multiple of 8 into the row) as pairs
__device__ __forceinline__ void store_pairs(_Float16* to, const float* x) {
  f32x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x[j];
  const f16x8 h = __builtin_convertvector(v, f16x8);
  const f16x8 l = __builtin_convertvector(v - __builtin_convertvector(h, f32x8), f16x8);
  *reinterpret_cast<f16x8*>(to) = h;
  *reinterpret_cast<f16x8*>(to + 32) = l;
}

// X = matrix * 2^e / (norm + eps) in pairs, transposed where the matrix is tall; 64 x 64 elements per workgroup, through
// LDS, since either side may run along memory.  18 x 256 x 2304 f32: 21 us (85 MB, 4.0 TB/s).
template <int DT, bool MUON>
__global__ __launch_bounds__(NT) void k_pairs(Matrices ms, Shape sh, Update u, const double* part, double eps,
                                               double unit, Pairs X) {
  typedef Elem<DT> E;
  const int i = blockIdx.z;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;   // of X
  __shared__ double inv;
  __shared__ float tile[64][65];
  if (threadIdx.x < 64) {
    double s = 0.;
    for (int p = threadIdx.x; p < sh.parts; p += 64) s += part[i * sh.parts + p];
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
    store_pairs(X.hi(i, r0 + a, c0 + b), &tile[a][b]);
  }
}

// ---- products --------------------------------------------------------------------------------------------------
// One workgroup: D[m][n] = sum_k P[m][k] Q[n][k] for a tile of T x T on the 32x32x16 instruction.
//   GRAM    P = Q = X:  S, the tiles on and below the diagonal, each written twice
//   POLY    P = Q = S:  B = a I + b S + c S S, likewise (a in B and not in the next product: X is read once less there)
//   APPLY   P = X transposed while it is read from LDS, Q = B:  X <- B X (m runs along X's rows in memory)
//   LAST_*  APPLY whose result leaves the pairs: orthogonalised, or subtracted from the parameter
//
// A round is DEPTH elements deep.  It goes straight from memory into LDS, in a ring of RING rounds: all but one are
// under way while one is multiplied, and a round costs one barrier.  SIDE x SIDE waves share the tile, GROUPS such
// sets share the depth of a round, and their sums are added at the end in a fixed order.
//
// APPLY of 2048 x 8192 (128-tiles, two workgroups a CU): 200 us, 1030 TFLOP/s of f16 products against the library's 1140
// for one large product; the matrix cores are busy two thirds of the time, at the clock that the power limit leaves.
// GRAM 2048 x 2048 x 8192 (96-tiles, half the square): 118 us, 970 TFLOP/s.  Small ones are bound by what a launch costs
// besides, about 6 us for the first loads, the sums through LDS and the stores: 18 x 256 x 256 x 256 takes 7.5 us.
enum Kind { GRAM, POLY, APPLY, LAST_OUT, LAST_MUON };

struct Product {
  Pairs P, Q, D;
  int k;                // depth, a multiple of 64
  int n;                // matrices
  int tiles, tiles_m;   // tiles of one matrix, and along m (APPLY)
  float acc, self, one; // D = acc * sum, and in POLY + self * the element of S + one on the diagonal
};
struct Leave {          // what LAST_* needs besides
  Matrices ms;
  Shape sh;
  Update u;
};
struct Stay {};
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// 16 bytes a lane straight into LDS; the wave's 64 pieces lie there in lane order
__device__ __forceinline__ void to_lds(const char* from, uint32_t lane_offset, _Float16* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + lane_offset),
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// Waits until at most PENDING of the wave's loads are under way (and all its LDS reads are done), then for the
// workgroup: after it every wave's older pieces are in LDS, and nobody reads the round before any more.
template <int PENDING> __device__ __forceinline__ void ready() {
  __builtin_amdgcn_s_waitcnt((PENDING & 15) | ((PENDING >> 4) << 14) | 0x0070);   // vmcnt(PENDING) lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Rows in LDS: blocks of T lines, 8 pieces of 16 B each (hi 0-3, lo 4-7), piece p of row m at p ^ (m >> 1 & 7), so that the
// 16 lanes that read one piece of 16 rows meet 16 different bank groups.
__device__ __forceinline__ int row_piece(int m, int p) { return p ^ ((m >> 1) & 7); }
__device__ __forceinline__ f16x8 read_rows(const _Float16* lds, int m, int p) {
  return *reinterpret_cast<const f16x8*>(lds + m * 64 + row_piece(m, p) * 8);
}
// Columns in LDS: rows of T / 32 lines; piece p of row k at p ^ ((k & 3) << 2), so that the four rows that a
// transposing read touches (64 B each) lie in different banks.
__device__ __forceinline__ int col_piece(int k, int p) { return p ^ ((k & 3) << 2); }
// For F groups of 32 columns from m0 on: elements k .. k + 7 (k = k0 + 8 for the upper half wave) of the lane's column,
// their hi halves and their lo halves; each is two transposing reads of 4 rows x 16 columns.  In one block of
// assembly that ends with its own wait, because the compiler would have every such read wait for all loads on
// their way into LDS.
template <int T, int F>
__device__ __forceinline__ void read_cols(const _Float16* lds, int m0, int k0, int lane, f16x8* hi, f16x8* lo) {
  const int q = lane & 15, col = ((lane >> 4) & 1) * 16 + (q & 3) * 4;   // within a group
  const int k = k0 + (lane >> 5) * 8 + (q >> 2);                        // k & 3 is that of k + 4 too
  const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds +
                        k * 4 * T + (col & 7) * 2;
  f16x4 v[F][4];
#pragma unroll
  for (int f = 0; f < F; f += 2) {
    const int p = ((m0 >> 5) + f) * 8 + (col >> 3);
    const uint32_t h0 = base + col_piece(k, p) * 16, l0 = base + col_piece(k, p + 4) * 16;
    const uint32_t h1 = base + col_piece(k, p + 8) * 16, l1 = base + col_piece(k, p + 12) * 16;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
        "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[f][0]), "=&v"(v[f][1]), "=&v"(v[f][2]), "=&v"(v[f][3]), "=&v"(v[f + 1][0]), "=&v"(v[f + 1][1]),
          "=&v"(v[f + 1][2]), "=&v"(v[f + 1][3])
        : "v"(h0), "v"(l0), "v"(h1), "v"(l1), "n"(16 * T)
        : "memory");
  }
#pragma unroll
  for (int f = 0; f < F; ++f) {
    hi[f] = __builtin_shufflevector(v[f][0], v[f][1], 0, 1, 2, 3, 4, 5, 6, 7);
    lo[f] = __builtin_shufflevector(v[f][2], v[f][3], 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// the row of element t of a lower triangle, row by row
__device__ __forceinline__ int triangle_row(int t) {
  int row = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  if ((row + 1) * (row + 2) / 2 <= t) ++row;
  if (row * (row + 1) / 2 > t) --row;
  return row;
}
__device__ __forceinline__ bool tall(const Stay&) { return false; }
__device__ __forceinline__ bool tall(const Leave& l) { return l.sh.rows > l.sh.cols; }
// up to eight consecutive results into the output or the parameter
template <int DT, bool MUON>
__device__ __forceinline__ void leave(typename Elem<DT>::T* o, const float* v, int n, const Update& u) {
  typedef Elem<DT> E;
  Pack<typename E::T, 8> q;
  if (n >= 8) {
    if (MUON) q = *reinterpret_cast<const Pack<typename E::T, 8>*>(o);
#pragma unroll
    for (int j = 0; j < 8; ++j) q.v[j] = E::put(MUON ? fmaf(u.keep, E::get(q.v[j]), -u.step * v[j]) : v[j]);
    *reinterpret_cast<Pack<typename E::T, 8>*>(o) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) o[j] = E::put(MUON ? fmaf(u.keep, E::get(o[j]), -u.step * v[j]) : v[j]);
  }
}

template <int T, int SIDE, int GROUPS, int DEPTH, int RING, int KIND, int DT, typename Out>
__global__ __launch_bounds__(64 * SIDE * SIDE * GROUPS, 160 * 1024 / (RING * T * DEPTH * 8) * SIDE * SIDE * GROUPS / 4)
void k_product(Product pr, Out out) {
  constexpr bool COLS = KIND >= APPLY;
  constexpr int WAVES = SIDE * SIDE * GROUPS;
  constexpr int W = T / SIDE, F = W / 32;               // a wave's part of the tile, in 32 x 32 sums
  constexpr int STEPS = DEPTH / 16 / GROUPS;            // instructions deep a wave goes per round
  constexpr int CH = T * DEPTH / 256 / WAVES;           // pieces of 1 KiB a wave loads of P, and of Q, per round
  constexpr int HALF = T * DEPTH * 2;                   // halves of one operand's round
  constexpr int PITCH = W + 4, PART = W * PITCH;        // floats of a wave's sums in LDS
  constexpr int LOOP = RING * 2 * HALF * 2, END = WAVES * PART * 4;
  static_assert(T * DEPTH % (256 * WAVES) == 0 && DEPTH % (16 * GROUPS) == 0 && 64 % DEPTH == 0, "round");
  static_assert(!COLS || F % 2 == 0, "read_cols");
  __shared__ __attribute__((aligned(1024))) char shared[LOOP > END ? LOOP : END];
  _Float16* lds = reinterpret_cast<_Float16*>(shared);
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int part = wave % (SIDE * SIDE), group = wave / (SIDE * SIDE);
  // Workgroups go round the 8 XCDs in turn; give each XCD one contiguous run of tiles, and order the tiles in bands,
  // so that those an XCD works on at a time share rows and columns in its L2.
  const int total = pr.tiles * pr.n, xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
  const int id = xcd * (total / 8) + min(xcd, total % 8) + nth;
  const int i = id / pr.tiles, t = id % pr.tiles;
  int bm, bn;
  if (COLS) {                                           // bands of 8 tiles along n, n the faster within a band
    const int band = t / (8 * pr.tiles_m), in = t - band * 8 * pr.tiles_m;
    const int high = min(8, pr.tiles / pr.tiles_m - band * 8);
    bm = in / high, bn = band * 8 + in % high;
  } else {                                              // lower triangle in bands of 8 rows: a band's square columns,
    const int first = triangle_row(t) & ~7, in = t - first * (first + 1) / 2;   // then its triangle
    const int high = min(8, triangle_row(pr.tiles - 1) + 1 - first);
    if (in < first * high) {
      bm = first + in % high, bn = in / high;
    } else {
      const int rest = in - first * high, row = triangle_row(rest);
      bm = first + row, bn = first + rest - row * (row + 1) / 2;
    }
  }
  const char* const from_p = (const char*)(COLS ? pr.P.hi(i, 0, bm * T) : pr.P.hi(i, bm * T, 0));
  const char* const from_q = (const char*)pr.Q.hi(i, bn * T, 0);
  // where in a round this lane's 16 bytes come from (bytes)
  uint32_t at_p[CH], at_q[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int chunk = wave + WAVES * c;
    const int line = chunk / (T / 8), m = chunk % (T / 8) * 8 + (lane >> 3);
    const uint32_t in_row = (uint32_t)(line * 128 + row_piece(m, lane & 7) * 16);
    at_q[c] = (uint32_t)m * pr.Q.pitch * 2 + in_row;
    if (COLS) {
      constexpr int PR = T / 4, RW = 64 / PR;           // pieces a row, rows a wave
      const int k = chunk * RW + lane / PR;
      at_p[c] = (uint32_t)k * pr.P.pitch * 2 + (uint32_t)col_piece(k, lane % PR) * 16;
    } else {
      at_p[c] = (uint32_t)m * pr.P.pitch * 2 + in_row;
    }
  }
  const int64_t step_p = COLS ? (int64_t)DEPTH * pr.P.pitch * 2 : DEPTH * 4, step_q = DEPTH * 4;
  auto load = [&](int round, int buf, int c) {          // one piece of P and one of Q
    const int chunk = wave + WAVES * c;
    to_lds(from_p + round * step_p, at_p[c], lds + buf * 2 * HALF + chunk * 512);
    to_lds(from_q + round * step_q, at_q[c], lds + buf * 2 * HALF + HALF + chunk * 512);
  };
  const int m0 = part % SIDE * W, n0 = part / SIDE * W;
  const int rounds = pr.k / DEPTH;
  // Where each wave has a tile to itself, a round's operands are read during the products of the round before (2048 x 8192
  // bf16, five steps: 1311 us, without 1350); with four waves a tile 1024 deep that takes 35 us and without 32.
  constexpr bool EARLY = !COLS && STEPS == 1 && SIDE == 1;
  f32x16 acc[F][F] = {};
  struct Operands { f16x8 ah[F], al[F], bh[F], bl[F]; };
  auto read = [&](int buf, int step, Operands& x) {
    const _Float16 *p = lds + buf * 2 * HALF, *q = p + HALF;
    const int kk = (group * STEPS + step) * 16;
    const int line = kk / 32 * T * 64, piece = kk % 32 / 8 + (lane >> 5);   // rows: block of lines, piece
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int m = m0 + 32 * f + (lane & 31), n = n0 + 32 * f + (lane & 31);
      if (!COLS) {
        x.ah[f] = read_rows(p + line, m, piece);
        x.al[f] = read_rows(p + line, m, piece + 4);
      }
      x.bh[f] = read_rows(q + line, n, piece);
      x.bl[f] = read_rows(q + line, n, piece + 4);
    }
    if constexpr (COLS) read_cols<T, F>(p, m0, kk, lane, x.ah, x.al);
  };
  // One step's products.  A round's loads are issued between its products: a wave issues in order, and the address path
  // takes 1 KiB pieces too slowly to have them ahead of everything.
  auto multiply = [&](const Operands& x, int step, auto loads, int r, int over) {
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int g = 0; g < F; ++g) {
        acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.al[f], x.bh[g], acc[f][g], 0, 0, 0);
        acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ah[f], x.bl[g], acc[f][g], 0, 0, 0);
        acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ah[f], x.bh[g], acc[f][g], 0, 0, 0);
        if constexpr (decltype(loads)::value) {
          constexpr int ALL = STEPS * F * F;
          const int at = (step * F + f) * F + g;
#pragma unroll
          for (int c = at * CH / ALL; c < (at + 1) * CH / ALL; ++c) load(r, over, c);
          __builtin_amdgcn_sched_barrier(EARLY ? 0 : 0x7);   // these loads stay here; 0x7: arithmetic may pass
        }
      }
  };
  constexpr int AHEAD = EARLY ? RING : RING - 1;        // rounds under way beside the one that is multiplied
#pragma unroll
  for (int r = 0; r < AHEAD; ++r)
    if (r < rounds)
#pragma unroll
      for (int c = 0; c < CH; ++c) load(r, r, c);
  if constexpr (EARLY) {
    Operands even, odd;
    int buf = 0;                                        // of round r, free once everybody has its operands
    if (rounds >= RING) ready<2 * CH * (RING - 1)>();
    else ready<0>();
    read(0, 0, even);
    auto round = [&](int r, auto loads, const Operands& now, Operands& next) {
      constexpr bool more = decltype(loads)::value;
      const int over = buf;
      buf = buf + 1 == RING ? 0 : buf + 1;
      ready<more ? 2 * CH * (RING - 2) : 0>();          // round r + 1 is there
      read(buf, 0, next);                               // (of the last round nothing that is used)
      __builtin_amdgcn_sched_barrier(0);
      multiply(now, 0, loads, r + RING, over);
    };
    int r = 0;
    for (; r + RING + 1 < rounds; r += 2) {
      round(r, Yes{}, even, odd);
      round(r + 1, Yes{}, odd, even);
    }
    if (r + RING < rounds) {
      round(r, Yes{}, even, odd);
      even = odd, ++r;
    }
    for (; r < rounds; ++r) {
      round(r, No{}, even, odd);
      even = odd;
    }
  } else {
    int buf = 0;
    auto round = [&](int r, auto loads) {
      const int over = buf == 0 ? RING - 1 : buf - 1;   // the round read last
#pragma unroll
      for (int step = 0; step < STEPS; ++step) {
        Operands x;
        read(buf, step, x);
        multiply(x, step, loads, r + AHEAD, over);
      }
      buf = buf + 1 == RING ? 0 : buf + 1;
    };
    int r = 0;
    for (; r + AHEAD < rounds; ++r) {
      ready<2 * CH * (AHEAD - 1)>();                    // all rounds loaded so far but the newest AHEAD - 1
      round(r, Yes{});
    }
    for (; r < rounds; ++r) {
      ready<0>();
      round(r, No{});
    }
  }

  // The sums through LDS as [n][m], so that memory is read and written along rows: a lane holds column n and, four
  // at a time, consecutive m.  Group g then finishes the g-th share of the rows.
  ready<0>();
  float* const sums = reinterpret_cast<float*>(shared) + part * PART;         // of group 0; the next lies SIDE^2 PART on
  float* const mine = sums + group * SIDE * SIDE * PART;
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int g = 0; g < F; ++g)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float4 v;
        v.x = acc[f][g][4 * q], v.y = acc[f][g][4 * q + 1], v.z = acc[f][g][4 * q + 2], v.w = acc[f][g][4 * q + 3];
        *reinterpret_cast<float4*>(mine + (32 * g + (lane & 31)) * PITCH + 32 * f + 8 * q + 4 * (lane >> 5)) = v;
      }
  ready<0>();
  constexpr int PER_ROW = W / 8, SHARE = W / GROUPS;    // lanes a row, 8 elements each; rows a wave
  constexpr int ROWS = 64 / PER_ROW;                    // rows at a time; lanes behind the last whole row have none
  const int row0 = lane < ROWS * PER_ROW ? group * SHARE + lane / PER_ROW : W;
  const bool turn = KIND < APPLY ? bm != bn : KIND > APPLY && tall(out);   // leaves transposed (too), below
#pragma unroll 4
  for (int row = row0; row < (group + 1) * SHARE; row += ROWS) {
    const int col = lane % PER_ROW * 8, n = bn * T + n0 + row, m = bm * T + m0 + col;
    float* at = sums + row * PITCH + col;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = at[j];
#pragma unroll
    for (int g = 1; g < GROUPS; ++g)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += at[g * SIDE * SIDE * PART + j];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= pr.acc;
    if constexpr (KIND == POLY) {
      const _Float16* self = pr.P.hi(i, n, m);
      const f16x8 h = *reinterpret_cast<const f16x8*>(self), l = *reinterpret_cast<const f16x8*>(self + 32);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = fmaf(pr.self, (float)h[j] + (float)l[j], v[j]);
        if (m + j == n) v[j] += pr.one;
      }
    }
    if (turn) {
#pragma unroll
      for (int j = 0; j < 8; ++j) at[j] = v[j];
    }
    if constexpr (KIND <= APPLY) {
      store_pairs(pr.D.hi(i, n, m), v);
    } else {
      const Shape& sh = out.sh;
      if (!turn && n < sh.r)
        leave<DT, KIND == LAST_MUON>((typename Elem<DT>::T*)out.ms.out[i] + (int64_t)n * sh.cols + m, v, sh.L - m, out.u);
    }
  }
  if (!turn) return;
  ready<0>();
#pragma unroll 4
  for (int row = row0; row < (group + 1) * SHARE; row += ROWS) {
    const int col = lane % PER_ROW * 8, m = bm * T + m0 + row, n = bn * T + n0 + col;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = sums[(col + j) * PITCH + row];
    if constexpr (KIND < APPLY) store_pairs(pr.D.hi(i, m, n), v);
    if constexpr (KIND > APPLY) {
      const Shape& sh = out.sh;
      if (m < sh.L)
        leave<DT, KIND == LAST_MUON>((typename Elem<DT>::T*)out.ms.out[i] + (int64_t)m * sh.cols + n, v, sh.r - n, out.u);
    }
  }
}

// ---- small matrices ------------------------------------------------------------------------------------------------
// A matrix that fits into one CU's LDS together with its r x r products is taken through all steps there, by one
// workgroup of 16 waves in one launch: memory is read once and the result written.  X lies in LDS as hi and lo planes
// [r16][pitch], S and then B as [r16][pitch_s]; the 16-byte piece p of row m is at p ^ (m >> 1 & 7), and the pitches are
// odd multiples of 128 bytes where there is room, so that the 16 rows of an operand lie in different banks.  Products
// are 16 x 16 x 32: a wave takes whole tiles of S and B (on and below the diagonal, written twice) and whole strips of
// 16 columns of X, which it reads before it overwrites them.  554 x 61 f32 takes 50 us, 8 a step, where the general
// kernels' 17 launches take 86; above SMALL_ROWS and where X does not fit those are taken.
constexpr int SMALL_WAVES = 16;
constexpr int SMALL_LDS = 160 * 1024;
constexpr int SMALL_ROWS = 128;                         // r at most: three tiles of S a wave
struct Small {
  int r16, strips;                                      // padded short side; 16 columns each of the long side
  int depth, depth_s, pitch, pitch_s;                   // of X and of S: columns up to a multiple of 64; from row to row
};
struct Factors {                                        // of GRAM, POLY (S S, S, diagonal) and APPLY, per step
  float gram[MTAZ_MAX_STEPS], square[MTAZ_MAX_STEPS], self[MTAZ_MAX_STEPS], one[MTAZ_MAX_STEPS], apply[MTAZ_MAX_STEPS];
};
// where column c of row m lies in its row
__device__ __forceinline__ int small_at(int m, int c) { return row_piece(m, c >> 3) * 8 + (c & 7); }

typedef float f32x4 __attribute__((ext_vector_type(4)));
// 16 x 16 sums of hi hi, hi lo and lo hi over one instruction's depth
struct Sums {
  f32x4 main = {}, cross = {}, cross2 = {};
  __device__ __forceinline__ void add(f16x8 ah, f16x8 al, f16x8 bh, f16x8 bl) {
    main = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, main, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, cross, 0, 0, 0);
    cross2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, cross2, 0, 0, 0);
  }
  __device__ __forceinline__ f32x4 sum() const { return main + (cross + cross2); }
};

// P P^T for rows [16 a, +16) and [16 b, +16) of the planes at hi: k runs along the rows, `depth` a multiple of 64.
// A lane's rows 16 a + j and 16 b + j are swizzled alike, and 64 columns are one full turn of the swizzle: the lane's
// places for the two instructions of a turn stay the same from turn to turn.
__device__ __forceinline__ f32x4 gram_tile(const _Float16* hi, int lo, int pitch, int depth, int a, int b, int lane) {
  const int j = lane & 15, first = small_at(j, (lane >> 4) * 8);
  const _Float16 *pa = hi + (16 * a + j) * pitch + first, *pb = hi + (16 * b + j) * pitch + first;
  const int second = first & 32 ? -32 : 32;
  auto at = [](const _Float16* p) { return *reinterpret_cast<const f16x8*>(p); };
  Sums s;
  if (a == b) {
    for (int k = 0; k < depth; k += 64, pa += 64) {
      const f16x8 ah = at(pa), al = at(pa + lo), ch = at(pa + second), cl = at(pa + lo + second);
      s.add(ah, al, ah, al);
      s.add(ch, cl, ch, cl);
    }
  } else {
    for (int k = 0; k < depth; k += 64, pa += 64, pb += 64) {
      const f16x8 ah = at(pa), al = at(pa + lo), bh = at(pb), bl = at(pb + lo);
      const f16x8 ch = at(pa + second), cl = at(pa + lo + second), dh = at(pb + second), dl = at(pb + lo + second);
      s.add(ah, al, bh, bl);
      s.add(ch, cl, dh, dl);
    }
  }
  return s.sum();
}

__device__ __forceinline__ void split4(f32x4 v, f16x4& h, f16x4& l) {
  h = __builtin_convertvector(v, f16x4);
  l = __builtin_convertvector(v - __builtin_convertvector(h, f32x4), f16x4);
}
// a tile's result into the symmetric planes: a lane holds column 16 b + (lane & 15), rows 16 a + 4 (lane >> 4) + j
__device__ __forceinline__ void put_tile(_Float16* hi, int lo, int pitch, int a, int b, f32x4 v, int lane) {
  f16x4 h, l;
  split4(v, h, l);
  const int m = 16 * a + 4 * (lane >> 4), n = 16 * b + (lane & 15);
  _Float16* to = hi + n * pitch + small_at(n, m);
  *reinterpret_cast<f16x4*>(to) = h;
  *reinterpret_cast<f16x4*>(to + lo) = l;
  if (a != b)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      to = hi + (m + j) * pitch + small_at(m + j, n);
      to[0] = h[j], to[lo] = l[j];
    }
}

// DEEP: instructions deep that B X goes at most, r16 / 32 rounded up to 1, 2 or 4; a wave takes up to WIDE strips of X at
// a time, so that a part of B once read serves them all.
template <int DT, bool MUON, int DEEP>
__global__ __launch_bounds__(64 * SMALL_WAVES) void k_small(Matrices ms, Shape sh, Small sm, Update u, int steps,
                                                            double eps, double unit, Factors fa) {
  typedef Elem<DT> E;
  constexpr int ALL = 64 * SMALL_WAVES;
  __shared__ __attribute__((aligned(1024))) char shared[SMALL_LDS];
  const int i = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int lane = threadIdx.x % 64;
  const typename E::T* g = (const typename E::T*)ms.grad[i];
  float* mom = ms.momentum[i];
  typename E::T* out = (typename E::T*)ms.out[i];
  const bool tall = sh.rows > sh.cols;

  // the steps' factors, lane t those of step t
  const int mine = min(lane, MTAZ_MAX_STEPS - 1);
  const float f_gram = fa.gram[mine], f_square = fa.square[mine], f_self = fa.self[mine], f_one = fa.one[mine],
              f_apply = fa.apply[mine];

  // The matrix, eight elements at a time: all of a thread's share (LDS holds 40 Ki pairs) is under way at once and
  // stays in registers until the norm, summed in 64 bits, is known.  Momentum is brought up to date on the way.
  constexpr int N = 8, PACKS = SMALL_LDS / 4 / (ALL * N);
  const int count = sh.rows * sh.cols;
  Pack<typename E::T, N> gv[PACKS];
  Pack<float, N> mv[PACKS];
#pragma unroll
  for (int c = 0; c < PACKS; ++c) {
    const int k = N * (threadIdx.x + ALL * c), n = count - k;
    if (n >= N) {
      gv[c] = *reinterpret_cast<const Pack<typename E::T, N>*>(g + k);
      if (MUON) mv[c] = *reinterpret_cast<const Pack<float, N>*>(mom + k);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) gv[c].v[j] = j < n ? g[k + j] : (typename E::T)0.f, mv[c].v[j] = MUON && j < n ? mom[k + j] : 0.f;
    }
  }
  _Float16* const X = reinterpret_cast<_Float16*>(shared);
  const int lo = sm.r16 * sm.pitch, lo_s = sm.r16 * sm.pitch_s;
  _Float16* const S = X + 2 * lo;
  for (int k = threadIdx.x; k < (lo + lo_s) / 4; k += ALL) reinterpret_cast<f16x8*>(X)[k] = f16x8{};   // the padding
  __syncthreads();
  double sq = 0.;
#pragma unroll
  for (int c = 0; c < PACKS; ++c) {
    const int k = N * (threadIdx.x + ALL * c), n = count - k;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = E::get(gv[c].v[j]);
      float m = mv[c].v[j];
      if (MUON) {
        m = fmaf(u.momentum, m, u.fresh * x);
        if (j < n) mom[k + j] = m;
      }
      mv[c].v[j] = update_of<DT, MUON>(x, m, u);
      const double y = (double)mv[c].v[j];
      sq = fma(y, y, sq);
    }
  }
  double* sums = reinterpret_cast<double*>(S);
  for (int o = 32; o; o >>= 1) sq += __shfl_xor(sq, o);
  if (lane == 0) sums[wave] = sq;
  __syncthreads();
  double norm = 0.;
  for (int w = 0; w < SMALL_WAVES; ++w) norm += sums[w];
  const double inv = unit / (sqrt(norm) + eps);
  int twos;                                             // as a float below 1 and a power of two: in range for any norm
  const float ones = (float)frexp(inv, &twos);
  __syncthreads();
  if (threadIdx.x < SMALL_WAVES) sums[threadIdx.x] = 0.;
#pragma unroll
  for (int c = 0; c < PACKS; ++c) {
    const int k = N * (threadIdx.x + ALL * c);
    int row = k / sh.cols, col = k - row * sh.cols;     // in memory
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (k + j < count) {
        const int m = tall ? col : row, n = tall ? row : col, to = m * sm.pitch + small_at(m, n);
        _Float16 h, l;
        split(ldexpf(mv[c].v[j] * ones, twos), h, l);
        X[to] = h, X[to + lo] = l;
      }
      if (++col == sh.cols) col = 0, ++row;
    }
  }
  __syncthreads();

  const int R = sm.r16 / 16, tiles = R * (R + 1) / 2;
  constexpr int MINE = (SMALL_ROWS / 16) * (SMALL_ROWS / 16 + 1) / 2 / SMALL_WAVES + 1;   // tiles of S a wave
  for (int step = 0; step < steps; ++step) {
    asm volatile("" : "+v"(lane));                      // addresses are computed in each step, not kept (and spilled) over all
    const float k_gram = __shfl(f_gram, step), k_square = __shfl(f_square, step), k_self = __shfl(f_self, step),
                k_one = __shfl(f_one, step), k_apply = __shfl(f_apply, step);
    for (int t = wave; t < tiles; t += SMALL_WAVES) {
      const int a = triangle_row(t), b = t - a * (a + 1) / 2;
      put_tile(S, lo_s, sm.pitch_s, a, b, k_gram * gram_tile(X, lo, sm.pitch, sm.depth, a, b, lane), lane);
    }
    __syncthreads();
    f32x4 v[MINE];
#pragma unroll
    for (int c = 0; c < MINE; ++c) {
      const int t = wave + SMALL_WAVES * c;
      if (t >= tiles) continue;
      const int a = triangle_row(t), b = t - a * (a + 1) / 2, m = 16 * a + 4 * (lane >> 4), n = 16 * b + (lane & 15);
      const f32x4 ss = gram_tile(S, lo_s, sm.pitch_s, sm.depth_s, a, b, lane);
      const _Float16* self = S + n * sm.pitch_s + small_at(n, m);
      const f16x4 h = *reinterpret_cast<const f16x4*>(self), l = *reinterpret_cast<const f16x4*>(self + lo_s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[c][j] = fmaf(k_self, (float)h[j] + (float)l[j], k_square * ss[j]);
        if (m + j == n) v[c][j] += k_one;
      }
    }
    __syncthreads();                                    // S is read; B takes its place
#pragma unroll
    for (int c = 0; c < MINE; ++c) {
      const int t = wave + SMALL_WAVES * c;
      if (t >= tiles) continue;
      const int a = triangle_row(t), b = t - a * (a + 1) / 2;
      put_tile(S, lo_s, sm.pitch_s, a, b, v[c], lane);
    }
    __syncthreads();
    const bool last = step + 1 == steps;
    constexpr int WIDE = DEEP == 4 ? 1 : 2;
    const int q = lane & 15, g8 = (lane >> 4) * 8;
    for (int strip = wave * WIDE; strip < sm.strips; strip += SMALL_WAVES * WIDE) {
      // The strips' columns as the first operand, k = rows of X: two transposing reads of 4 rows x 16 columns for 8 rows
      // a lane.  A transposing read runs in all lanes, whatever the mask: the lanes behind the last row read rows that are
      // there (r16 is a multiple of 16) and drop what they got, and so do strips behind the last.
      f16x8 ah[WIDE][DEEP], al[WIDE][DEEP];
#pragma unroll
      for (int w = 0; w < WIDE; ++w) {
        const int first = 16 * min(strip + w, sm.strips - 1) + (q & 3) * 4;
        const int turn[2] = {small_at(g8 + (q >> 2), first), small_at(g8 + (q >> 2) + 4, first)};   // 32 rows on the same
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
          const bool there = 32 * d + g8 < sm.r16;
          const _Float16* at = X + (there ? 32 * d + g8 + (q >> 2) : q >> 2) * sm.pitch;
          f16x4 part[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)                   // hi of rows row, row + 4; lo
            part[e] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(at + (e >> 1) * lo + 4 * (e & 1) * sm.pitch + turn[e & 1])));
          const f16x8 h = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
          const f16x8 l = __builtin_shufflevector(part[2], part[3], 0, 1, 2, 3, 4, 5, 6, 7);
          ah[w][d] = there ? h : f16x8{}, al[w][d] = there ? l : f16x8{};
        }
      }
      for (int tile = 0; tile < R; ++tile) {
        const int row = 16 * tile + q;
        const int first = small_at(q, g8);              // 16 rows on the same, 64 columns on too
        const _Float16* pb = S + row * sm.pitch_s;
        Sums s[WIDE];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {                // behind r16 X is 0 here, and B in its padding
          const _Float16* at = pb + (32 * d < sm.r16 ? 64 * (d / 2) + (d & 1 ? first ^ 32 : first) : 0);
          const f16x8 bh = *reinterpret_cast<const f16x8*>(at), bl = *reinterpret_cast<const f16x8*>(at + lo_s);
#pragma unroll
          for (int w = 0; w < WIDE; ++w) s[w].add(ah[w][d], al[w][d], bh, bl);
        }
#pragma unroll
        for (int w = 0; w < WIDE; ++w) {
          const int col = 16 * (strip + w) + (lane >> 4) * 4;
          if (strip + w >= sm.strips) continue;
          const f32x4 x = k_apply * s[w].sum();
          if (!last) {
            f16x4 h, l;
            split4(x, h, l);
            _Float16* to = X + row * sm.pitch + small_at(row, col);
            *reinterpret_cast<f16x4*>(to) = h;
            *reinterpret_cast<f16x4*>(to + lo) = l;
          } else if (row < sh.r) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (col + j >= sh.L) continue;
              typename E::T* o = out + (tall ? (col + j) * sh.cols + row : row * sh.cols + col + j);
              *o = E::put(MUON ? fmaf(u.keep, E::get(*o), -u.step * x[j]) : x[j]);
            }
          }
        }
      }
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

struct Work {
  double* part;
  Pairs X[2], S, B, C;
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
  auto pairs = [&](int rows, int cols) {
    Pairs p;
    p.pitch = 2 * cols, p.each = (int64_t)rows * p.pitch;
    p.at = (_Float16*)take(2 * p.each * n);
    return p;
  };
  w.part = (double*)take(8 * PARTS * n);
  w.X[0] = pairs(sh.height, sh.Lp);
  w.X[1] = pairs(sh.height, sh.Lp);
  w.S = pairs(sh.height, sh.height);
  w.B = pairs(sh.height, sh.height);
  w.C = pairs(sh.height, sh.height);
  w.bytes = at;
  return w;
}

// Tiles over r x L: 128 where the matrices have enough of them to occupy half of the 256 CUs, else 64 (B X of 18 x 256 x
// 2304, 648 tiles of 128: 27.7 us, of 64 36.0; of 3 x 512 x 1021, 96 tiles of 128: 14.8, of 64 11.3).  Over r x r, on
// and below the diagonal: the size that takes the fewest rounds of 256, each in proportion to its area; a tile of 64
// reads twice as much a product as one of 128 and counts for a third more.  (2048 x 2048: 136 tiles of 128 leave half
// of the chip without work and take 47 us a square; 253 of 96 fill it and take 36.)
Shape shape_of(int n, int64_t rows, int64_t cols) {
  Shape s;
  s.rows = (int)rows, s.cols = (int)cols;
  s.r = (int)(rows < cols ? rows : cols), s.L = (int)(rows < cols ? cols : rows);
  s.tile_L = n * (up(s.r, 128) / 128) * (up(s.L, 128) / 128) >= 128 ? 128 : 64;
  s.rp = (int)up(s.r, s.tile_L), s.Lp = (int)up(s.L, s.tile_L);
  double best = 0.;
  for (int T : {128, 96, 64}) {
    const int64_t t = up(s.rp, T) / T, tiles = n * t * (t + 1) / 2;
    const double cost = (double)T * T * (double)((tiles + 255) / 256) * (T == 64 ? 4. / 3. : T == 96 ? 1.05 : 1.);
    if (T == 128 || cost < best) best = cost, s.tile_r = T;
  }
  s.height = (int)up(s.rp, s.tile_r);
  const int64_t parts = up(rows * cols, 8 * NT * 2) / (8 * NT * 2);   // two rounds each at least
  s.parts = (int)(parts < PARTS ? parts : PARTS);
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
// before it, S below its square and B below the largest |a + b s^2 + c s^4|: both are taken at the range's ends and
// where the derivative vanishes, with a thousandth on top for roundings; f16 has room for twice 2^14 besides.
struct Exponents {
  int x[MTAZ_MAX_STEPS + 1], s[MTAZ_MAX_STEPS], b[MTAZ_MAX_STEPS];
  double end[MTAZ_MAX_STEPS], poly[MTAZ_MAX_STEPS];     // the bounds of S and of B
};
int exponent(double bound) {
  const int k = 14 - (int)ceil(log2(1.001 * fmax(bound, 1e-9)));
  return k > 40 ? 40 : k;
}
const char* bounds(int steps, const double* co, Exponents& e) {
  const double a = co[0], b = co[1], c = co[2];
  auto q = [&](double t) { return fabs(a + t * (b + t * c)); };   // of t = s^2
  // of s q(s^2): a + 3 b t + 5 c t^2 = 0 (one of the two forms of each root is exact where c is small or 0)
  const double disc = 9. * b * b - 20. * a * c, root = disc > 0. ? sqrt(disc) : 0., z = -3. * b - copysign(root, b);
  const double at[2] = {disc >= 0. && c != 0. ? z / (10. * c) : -1., disc >= 0. && z != 0. ? 2. * a / z : -1.};
  double top = 1.;
  for (int t = 0; t <= steps; ++t) {
    if (!(top <= 1e6)) return "the coefficients let the singular values grow past 10^6";
    e.x[t] = exponent(top);
    if (t == steps) break;
    const double end = top * top;
    double next = top * q(end), poly = fmax(q(0.), q(end));
    for (double s2 : at)
      if (s2 > 0. && s2 < end) next = fmax(next, sqrt(s2) * q(s2));
    if (c != 0. && -b / (2. * c) > 0. && -b / (2. * c) < end) poly = fmax(poly, q(-b / (2. * c)));
    e.s[t] = exponent(end), e.b[t] = exponent(poly);
    e.end[t] = end, e.poly[t] = poly;
    top = 1.001 * next;
  }
  return nullptr;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(e));
}

bool small(const Shape& sh, Small& sm) {
  sm.r16 = (int)up(sh.r, 16), sm.strips = (int)up(sh.L, 16) / 16;
  if (sm.r16 > SMALL_ROWS) return false;
  auto fits = [&](int a, int b) {
    sm.pitch = a, sm.pitch_s = b;
    return 4ll * sm.r16 * (a + b) <= SMALL_LDS;
  };
  const int a = sm.depth = (int)up(sh.L, 64), b = sm.depth_s = (int)up(sh.r, 64);
  return fits(a | 64, b | 64) || fits(a | 64, b) || fits(a, b | 64) || fits(a, b);
}

// Up to one tile a CU: the whole LDS for the ring, and waves that share the depth, so that each SIMD has work while
// another wave waits (216 tiles of 128, 1024 deep: 34 us, in the other form 40; 180 of 64, 2304 deep: 20 and 27).  More tiles: two workgroups a CU, of which
// one multiplies while the other begins or ends.
template <int KIND, int DT, typename Out>
void product(Product pr, int T, const Out& out, hipStream_t s) {
  const unsigned grid = (unsigned)(pr.tiles * pr.n);
  if (T == 128) {
    if (grid <= 256) k_product<128, 2, 2, 32, 4, KIND, DT, Out><<<grid, 512, 0, s>>>(pr, out);
    else k_product<128, 2, 1, 32, 2, KIND, DT, Out><<<grid, 256, 0, s>>>(pr, out);
  } else if (T == 96) {
    if constexpr (KIND < APPLY) k_product<96, 1, 4, 64, 3, KIND, DT, Out><<<grid, 256, 0, s>>>(pr, out);
  } else {
    if (grid <= 256) k_product<64, 1, 4, 64, 4, KIND, DT, Out><<<grid, 256, 0, s>>>(pr, out);
    else k_product<64, 1, 4, 64, 2, KIND, DT, Out><<<grid, 256, 0, s>>>(pr, out);
  }
}

template <int DT, bool MUON>
void iterate(const Matrices& ms, int n, const Shape& sh, const Update& u, int steps, const double* co, double eps,
             const Exponents& e, char* base, hipStream_t s) {
  Small sm;
  if (small(sh, sm)) {
    Factors fa = {};
    for (int t = 0; t < steps; ++t) {
      fa.gram[t] = (float)ldexp(1., e.s[t] - 2 * e.x[t]);
      fa.square[t] = (float)ldexp(co[2], e.b[t] - 2 * e.s[t]), fa.self[t] = (float)ldexp(co[1], e.b[t] - e.s[t]);
      fa.one[t] = (float)ldexp(co[0], e.b[t]);
      fa.apply[t] = (float)ldexp(1., (t + 1 < steps ? e.x[t + 1] : 0) - e.x[t] - e.b[t]);
    }
    const double unit = ldexp(1., e.x[0]);
    if (sm.r16 <= 32) k_small<DT, MUON, 1><<<n, 64 * SMALL_WAVES, 0, s>>>(ms, sh, sm, u, steps, eps, unit, fa);
    else if (sm.r16 <= 64) k_small<DT, MUON, 2><<<n, 64 * SMALL_WAVES, 0, s>>>(ms, sh, sm, u, steps, eps, unit, fa);
    else k_small<DT, MUON, 4><<<n, 64 * SMALL_WAVES, 0, s>>>(ms, sh, sm, u, steps, eps, unit, fa);
    return;
  }
  const Work w = layout(n, sh, base);
  const int64_t count = (int64_t)sh.rows * sh.cols;
  k_squares<DT, MUON><<<dim3(sh.parts, n), NT, 0, s>>>(ms, count, u, w.part);
  k_pairs<DT, MUON><<<dim3(sh.Lp / 64, sh.rp / 64, n), NT, 0, s>>>(ms, sh, u, w.part, eps, ldexp(1., e.x[0]), w.X[0]);
  const int tr = sh.height / sh.tile_r, tri = tr * (tr + 1) / 2;
  const int tL = sh.Lp / sh.tile_L, tall = sh.rp / sh.tile_L * tL;
  auto two = [](int k) { return (float)ldexp(1., k); };
  auto gram = [&](const Pairs& P, const Pairs& Q, const Pairs& D, int depth, int shift) {   // D = 2^shift P Q^T, symmetric
    product<GRAM, MTAZ_F32>({P, Q, D, depth, n, tri, 0, two(shift), 0.f, 0.f}, sh.tile_r, Stay{}, s);
  };
  auto poly = [&](const Pairs& S, const Pairs& D, int t) {                                    // D = a I + b S + c S S
    product<POLY, MTAZ_F32>({S, S, D, sh.rp, n, tri, 0, (float)ldexp(co[2], e.b[t] - 2 * e.s[t]),
                             (float)ldexp(co[1], e.b[t] - e.s[t]), (float)ldexp(co[0], e.b[t])}, sh.tile_r, Stay{}, s);
  };
  // Two steps in one where the long side is long against the short one: with M = a I + b S + c S S the second step's S
  // is M S M, and X <- M' M X; three products r x r more, and one product over the long side and one with X less
  // (2048 x 8192 bf16 1902 us without, 1577 with it).  That is a gain from L = 3 r on (16 bits, four and eighteen
  // matrices: 4 x 512 x 1536 209 us without and 202 with it, 18 x 256 x 1024 190 and 178, 3 x 200 x 4000 230 and 199; the
  // loss where it is none is small: 18 x 128 x 512 109 and 116), and from 1.5 r on where the square products fill the
  // chip, which takes about three million elements in them (6 x 1000 x 1536 731 and 681, 1 x 2048 x 3200 865 and 802, 6 x
  // 768 x 1152 399 and 395; but 1 x 768 x 1152 171 and 192, 6 x 640 x 960 296 and 309).
  // S loses accuracy by that in its small eigenvalues, a^2 = 12 times the rounding of its large ones: not visible
  // where the result is rounded to 16 bits, and in 32 bits not when it is done for the first two steps alone and r is not
  // small (against 64 bits, gradients of few strong directions: 6 x 1000 x 1536 2.5e-6 without and 1.9e-6 with it, 18 x 256
  // x 1024 1.4e-6 and 1.3e-6; 64 x 5000 of falling spectrum 8e-7 either way, but 15 x 5000 4e-7 and 9e-7).
  const bool joinable = sh.L >= 3ll * sh.r || (2ll * sh.L >= 3ll * sh.r && (int64_t)n * sh.r * sh.r >= 3 << 20);
  int now = 0;
  for (int t = 0; t < steps;) {
    const bool join = joinable && t + 1 < steps && (DT != MTAZ_F32 || (t == 0 && sh.r >= 64));
    const Pairs &X = w.X[now], &Y = w.X[now ^ 1];
    gram(X, X, w.S, sh.Lp, e.s[t] - 2 * e.x[t]);
    poly(w.S, w.B, t);
    const Pairs* M = &w.B;
    int em = e.b[t];
    if (join) {
      const int et = exponent(e.poly[t] * e.end[t]), eq = exponent(e.poly[t] * e.poly[t + 1]);
      gram(w.B, w.S, w.C, sh.rp, et - e.b[t] - e.s[t]);
      gram(w.C, w.B, w.S, sh.rp, e.s[t + 1] - et - e.b[t]);
      poly(w.S, w.C, t + 1);
      gram(w.C, w.B, w.S, sh.rp, eq - e.b[t + 1] - e.b[t]);
      M = &w.S, em = eq;
    }
    const int next = t + (join ? 2 : 1), ex = next < steps ? e.x[next] : 0;
    const Product last = {X, *M, Y, sh.rp, n, tall, tL, two(ex - e.x[t] - em), 0.f, 0.f};
    if (next < steps) product<APPLY, MTAZ_F32>(last, sh.tile_L, Stay{}, s);
    else product<MUON ? LAST_MUON : LAST_OUT, DT>(last, sh.tile_L, Leave{ms, sh, u}, s);
    t = next, now ^= 1;
  }
}

// Matrices that go through the kernels together: up to MOST, and fewer where they are so large that one fills the chip,
// so that the workspace stays near 2 GiB
int group_of(int64_t rows, int64_t cols) {
  const int64_t m = (2ll << 30) / layout(1, shape_of(1, rows, cols), nullptr).bytes;
  return m < 1 ? 1 : m < MOST ? (int)m : MOST;
}
// of the whole groups or of the last one, which may choose other tiles
int64_t workspace(int n, int64_t rows, int64_t cols) {
  auto of = [&](int m) {
    const Shape sh = shape_of(m, rows, cols);
    Small sm;
    return m == 0 || small(sh, sm) ? 256 : layout(m, sh, nullptr).bytes;
  };
  const int most = group_of(rows, cols);
  const int64_t whole = of(n < most ? n : most), rest = of(n % most);
  return whole > rest ? whole : rest;
}

// All checks, then the matrices in groups over the same workspace
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
  if (!work || ((uintptr_t)work & 255) || work_bytes < workspace(n, rows, cols))
    return ops_error(MTAZ_E_FAIL, what, "workspace too small or not aligned to 256 bytes");
  DeviceScope on(device);
  if (on.status != hipSuccess) return ops_error(MTAZ_E_DEVICE, what, hipGetErrorString(on.status));
  const int most = group_of(rows, cols);
  for (int first = 0; first < n; first += most) {
    const int m = n - first < most ? n - first : most;
    Matrices ms = {};
    for (int i = 0; i < m; ++i) {
      ms.grad[i] = grad[first + i], ms.out[i] = out[first + i];
      if (MUON) ms.momentum[i] = momenta[first + i];
    }
    const hipStream_t s = (hipStream_t)stream;
    const Shape sh = shape_of(m, rows, cols);
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
  return workspace(n, rows, cols);
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
  const Update u = {(float)momentum, (float)(1. - momentum), (float)(1. - lr * weight_decay), (float)(lr * scale), nesterov};
  return run<true>("muon_step", device, n, rows, cols, dtype, d_grads, d_params, d_momenta, u, steps, coefficients,
                   eps, d_work, work_bytes, stream);
}
