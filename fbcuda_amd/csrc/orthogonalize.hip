// Newton-Schulz products: X = G / (|G| + eps), then for each (a, b, c)
//
//   A = X X^T,  B = b A + c A A,  X = a X + B X
//
// X, A and B lie in the workspace as pairs: a value times 2^10 is the sum of two float16 numbers, its leading 11 bits and the
// next ones.  22 bits of typical values (an entry of an orthogonal matrix of 4096 columns is about 1 / 64: 16, whose second
// piece is about 2^-8, far above the smallest normal float16, 2^-14), and the largest are below 64 * 2^10.  A product of
// pairs is three products of pieces on the 16-bit matrix instructions; that of the second pieces, below 2^-22, is left out.
// (One 16-bit piece would not do: bfloat16 between the products leaves results 1e-2 to 5e-2 off the formula, float16 1e-3
// to 6e-3, pairs about 2e-6, as 32-bit arithmetic does: the first steps multiply small singular values by 3.4 each, and what
// rounding put beside them, too.)
//
// Two ways:
//   whole     one launch, a workgroup to a matrix in LDS: up to 96 rows (or columns) and 156 KB of pairs.  16 of 131 x 81 bf16
//             46 us, 64 x 64 f32 19; step by step 80 and 52, of which each launch's way through memory is 2.5 to 4
//   steps()   three products a step.  What bounds them: launches and latency below about 10^9 operations a product (192 x 1600
//             f32 104 us, 17 launches), above it the matrix instructions, three for what one 16-bit product takes (8192 x 2048 f32
//             1.63 ms, 1.03 PFLOP/s of the three; bf16, whose first step has fewer pieces, 1.55)
//             (The P x P matrices of all steps first, every A from the first, and X met by them once at the end, took 0.92 ms for
//             8192 x 2048 bf16.  But a rounding of the first A grows by up to a^2 with every step that only looks at A, where X
//             itself would have set it right: five times the error of 32-bit arithmetic there, and up to half a rounding to bfloat16
//             on matrices of one strong direction.)
//
// A pair matrix has rows of a multiple of 32 columns, 32 leading pieces and then their 32 second pieces, 128 bytes: what a
// matrix instruction takes of a row.  Rows and columns are filled up with zeros.
#include "pair_plan.h"
#include "product.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace fbfft_amd {
namespace {

typedef half16 halfx4 __attribute__((ext_vector_type(4)));

constexpr float kUnit = 1024.f;  // what stands for 1 in pieces

struct Pairs {
  half16* data;
  long cols;   // a multiple of 32; a row has 2 cols pieces
  long batch;  // pieces from a matrix to the next
};

__device__ __forceinline__ long placeOf(const Pairs& m, long i, long j) { return 2 * (i * m.cols + j / 32 * 32) + j % 32; }
// eight values as their leading and second pieces
__device__ __forceinline__ void splitEight(const float (&z)[8], halfx8& lead, halfx8& rest) {
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    lead[v] = (half16)z[v];
    rest[v] = (half16)(z[v] - (float)lead[v]);
  }
}

template <class T>
struct Given {
  T* data;
  long row, col, batch;
};

constexpr int kShares = 256;  // parts of a matrix whose squares are summed

__device__ __forceinline__ double groupSum(double v, double* space) {
  v = waveSum(v);
  if (threadIdx.x % 64 == 0) space[threadIdx.x / 64] = v;
  __syncthreads();
  return space[0] + space[1] + space[2] + space[3];
}

// Eight neighbours of a line of `count` elements, from element j: zeros behind the last.
template <class T>
__device__ __forceinline__ void loadEight(const T* line, long stride, long j, long count, float (&v)[8]) {
  if (stride == 1 && j + 8 <= count) {
    loadPack<T, 8>(line + j, v);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = j + q < count ? (float)line[(j + q) * stride] : 0.f;
  }
}

// Squares are summed in 64 bits: those of float32 values pass its range.  (Lines are rows or columns, whichever elements are
// neighbours; words: of eight elements to a line.)
template <class T>
__global__ __launch_bounds__(256) void squares(Given<const T> g, long lines, long count, Divisor words, double* sums) {
  __shared__ double space[4];
  const T* const from = g.data + blockIdx.y * g.batch;
  const int total = (int)(lines * words.value);
  double sum = 0;
#pragma unroll 2
  for (int at = (int)blockIdx.x * 256 + threadIdx.x; at < total; at += kShares * 256) {
    const int i = quotient(at, words);
    float v[8];
    loadEight(from + i * g.row, g.col, 8l * (at - i * (int)words.value), count, v);
#pragma unroll
    for (int q = 0; q < 8; ++q) sum += (double)v[q] * (double)v[q];
  }
  sum = groupSum(sum, space);
  if (threadIdx.x == 0) sums[blockIdx.y * kShares + blockIdx.x] = sum;
}

// X and its transpose from G, as pairs of a power of two times G; factors: what that leaves to 1 / (|G| + eps), from 1 to 2.  (So
// the leading pieces hold 16-bit values by themselves.)  A workgroup: 64 x 64 elements, through LDS; LINES: columns are the
// lines of neighbours.
template <class T, bool LINES>
__global__ __launch_bounds__(256) void begin(Given<const T> g, long rows, long cols, const double* sums, float eps, Pairs x, Pairs xt,
                                             float* factors) {
  constexpr int PITCH = 68;
  __shared__ double space[4];
  __shared__ __attribute__((aligned(16))) float tile[64 * PITCH];
  const double by = (double)kUnit / (__builtin_sqrt(groupSum(sums[blockIdx.y * kShares + threadIdx.x], space)) + (double)eps);
  // (0 and what is not finite leave no exponent: they go with the factor)
  const bool normal = by > 0x1p-1000 && by < 0x1p1000;
  const double power = normal ? __builtin_bit_cast(double, __builtin_bit_cast(unsigned long, by) & 0x7ff0000000000000ul) : 1.0;
  if (blockIdx.x == 0 && threadIdx.x == 0) factors[blockIdx.y] = (float)(by / power);
  const int across = (int)((x.cols + 63) / 64), down = (int)blockIdx.x / across;
  const long i0 = 64l * down, j0 = 64l * ((int)blockIdx.x - down * across);
  const T* const from = g.data + blockIdx.y * g.batch;
#pragma unroll
  for (int at = threadIdx.x; at < 512; at += 256) {
    const int line = at / 8, in = at % 8 * 8;
    float v[8];
    if (LINES) {
      const long j = min(j0 + line, cols - 1);
      loadEight(from + j * g.col, g.row, i0 + in, rows, v);
    } else {
      const long i = min(i0 + line, rows - 1);
      loadEight(from + i * g.row, g.col, j0 + in, cols, v);
    }
    const bool there = LINES ? j0 + line < cols : i0 + line < rows;
#pragma unroll
    for (int q = 0; q < 8; ++q) tile[LINES ? (in + q) * PITCH + line : line * PITCH + in + q] = there ? (float)((double)v[q] * power) : 0.f;
  }
  __syncthreads();
  x.data += blockIdx.y * x.batch, xt.data += blockIdx.y * xt.batch;
#pragma unroll
  for (int at = threadIdx.x; at < 512; at += 256) {
    const int line = at / 8, in = at % 8 * 8;
    halfx8 lead, rest;
    float z[8];
    if (i0 + line < xt.cols && j0 + in < x.cols) {
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = tile[line * PITCH + in + q];
      splitEight(z, lead, rest);
      half16* const to = x.data + placeOf(x, i0 + line, j0 + in);
      *reinterpret_cast<halfx8*>(to) = lead;
      *reinterpret_cast<halfx8*>(to + 32) = rest;
    }
    if (j0 + line < x.cols && i0 + in < xt.cols) {
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = tile[(in + q) * PITCH + line];
      splitEight(z, lead, rest);
      half16* const to = xt.data + placeOf(xt, j0 + line, i0 + in);
      *reinterpret_cast<halfx8*>(to) = lead;
      *reinterpret_cast<halfx8*>(to + 32) = rest;
    }
  }
}

// Of four neighbours those from `first` up to `end`, as pieces.
__device__ __forceinline__ void storeFour(half16* to, const float (&z)[4], int first, int end) {
  halfx4 lead, rest;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    lead[v] = (half16)z[v];
    rest[v] = (half16)(z[v] - (float)lead[v]);
  }
  if (first <= 0 && end >= 4) {
    *reinterpret_cast<halfx4*>(to) = lead;
    *reinterpret_cast<halfx4*>(to + 32) = rest;
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (v >= first && v < end) to[v] = lead[v], to[v + 32] = rest[v];
  }
}

// ---- products ----

__device__ __forceinline__ floatx4 multiply(uintx4 a, uintx4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}

// a b^T of two pair matrices, and what becomes of it: z = by sum + beta old, to out, and to turned the other way round.
struct PairArgs {
  Pairs a, b;
  long M, N, K, range;  // multiples of 32; k per range
  float by, beta;
  const float* factors;  // not null: of each matrix; `power` times in by, once in beta
  int power;
  Pairs old, out, turned;  // old, turned: data may be null
  // out is: what lies on and below the diagonal, and its mirror image.  (Exactly: A A is computed as A A^T.)
  bool symmetric;
  float* parts;            // not null: sums of each range of a symmetric product, [matrix][range][tile][BM][BN], in place of results
};

// where the last product leaves its results, times a factor
template <class T>
struct Result {
  Given<T> y;
  long rows, cols;
  float scale;
};
struct Nothing {};

// Of eight neighbours those from `first` up to `end`.
__device__ __forceinline__ void storeEight(half16* to, const float (&z)[8], int first, int end) {
  halfx8 lead, rest;
  splitEight(z, lead, rest);
  if (first <= 0 && end >= 8) {
    *reinterpret_cast<halfx8*>(to) = lead;
    *reinterpret_cast<halfx8*>(to + 32) = rest;
  } else {
#pragma unroll
    for (int v = 0; v < 8; ++v)
      if (v >= first && v < end) to[v] = lead[v], to[v + 32] = rest[v];
  }
}

// 32 rows by COLS columns of results from row m0 and column n0, both multiples of 32, by WAVES waves, one or a workgroup's:
// eight(row, column, v) gives eight neighbouring sums.  What stands beside them is on its way for all rows at once (a row after the
// other, each waits for memory).  Results that go the other way round meet in LDS, 32 x (COLS + 4) numbers.
template <int COLS, int WAVES, class RESULT, class EIGHT>
__device__ __forceinline__ void leavePairs(const PairArgs& g, const RESULT& result, long matrix, long m0, long n0, bool mirror,
                                           float* space, EIGHT eight) {
  constexpr int LANES = COLS / 8, ROWS = WAVES * 64 / LANES, TIMES = ROWS < 32 ? 32 / ROWS : 1, PITCH = COLS + 4;
  constexpr bool LAST = !__is_same(RESULT, Nothing);
  const int lane = threadIdx.x % (WAVES * 64), c = lane % LANES * 8;
  bool turns = mirror;
  if constexpr (LAST) turns = result.y.row == 1 && result.y.col != 1;
  const long n = n0 + c;
  const bool inside = n < g.N;  // (N is a multiple of 32)
  const float factor = g.factors ? g.factors[matrix] : 1.f, by = g.by * factor * (g.power == 2 ? factor : 1.f), beta = g.beta * factor;
  halfx8 old[TIMES][2] = {};
  if (g.old.data && inside) {
#pragma unroll
    for (int t = 0; t < TIMES; ++t) {
      const int row = t * ROWS + lane / LANES;
      if (row >= 32 || m0 + row >= g.M) continue;
      const half16* const from = g.old.data + matrix * g.old.batch + placeOf(g.old, m0 + row, n);
      old[t][0] = *reinterpret_cast<const halfx8*>(from), old[t][1] = *reinterpret_cast<const halfx8*>(from + 32);
    }
  }
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const int row = t * ROWS + lane / LANES;
    if (row >= 32) continue;
    const long m = m0 + row;
    float z[8];
    eight(row, c, z);
#pragma unroll
    for (int v = 0; v < 8; ++v) z[v] = z[v] * by + beta * ((float)old[t][0][v] + (float)old[t][1][v]);
    if (inside && m < g.M) {
      if constexpr (LAST) {
#pragma unroll
        for (int v = 0; v < 8; ++v) z[v] *= result.scale;
        auto* const to = result.y.data + matrix * result.y.batch + m * result.y.row + n * result.y.col;
        if (!turns && m < result.rows) {
          if (result.y.col == 1 && n + 8 <= result.cols) {
            storePack(to, z);
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              if (n + v < result.cols) storePack(to + v * result.y.col, {z[v]});
          }
        }
      } else {
        storeEight(g.out.data + matrix * g.out.batch + placeOf(g.out, m, n), z, 0, g.symmetric ? (int)min(m - n + 1, 8l) : 8);
      }
    }
    if (turns) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<floatx4*>(space + row * PITCH + c + 4 * h) = floatx4{z[4 * h], z[4 * h + 1], z[4 * h + 2], z[4 * h + 3]};
    }
  }
  if (!turns) return;
  if constexpr (WAVES == 1)
    waveExchange();
  else
    __syncthreads();
#pragma unroll 4
  for (int at = lane; at < COLS * 4; at += WAVES * 64) {
    const int column = at % COLS, q = at / COLS;
    const long n = n0 + column;
    if (n >= g.N || m0 >= g.M) continue;
    float z[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) z[v] = space[(8 * q + v) * PITCH + column];
    if constexpr (LAST) {
      auto* const to = result.y.data + matrix * result.y.batch + n * result.y.col + m0 + 8 * q;
      if (n < result.cols) {
        if (m0 + 8 * q + 8 <= result.rows) {
          storePack(to, z);
        } else {
#pragma unroll
          for (int v = 0; v < 8; ++v)
            if (m0 + 8 * q + v < result.rows) storePack(to + v, {z[v]});
        }
      }
    } else {
      storeEight(g.turned.data + matrix * g.turned.batch + placeOf(g.turned, n, m0) + 8 * q, z,
                 g.symmetric ? (int)max(n + 1 - (m0 + 8 * q), 0l) : 0, 8);
    }
  }
}

// Tile `tile` of those on and below the diagonal of `down` rows of tiles: in strips of four rows, column after column, so that
// those that run together share lines of both operands.
__device__ __forceinline__ void belowDiagonal(int tile, int down, int& i, int& j) {
  // (strip s begins with tile 8 s^2 + 2 s)
  int s = (int)((__builtin_sqrtf(32.f * tile + 4.f) - 2.f) * 0.0625f);
  while (s > 0 && 8 * s * s + 2 * s > tile) --s;
  while (8 * (s + 1) * (s + 1) + 2 * (s + 1) <= tile) ++s;
  tile -= 8 * s * s + 2 * s;
  const int height = min(4, down - 4 * s);
  if (tile < 4 * s * height) {
    i = 4 * s + tile % height;
    j = tile / height;
    return;
  }
  tile -= 4 * s * height;
  i = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3;
  j = 4 * s + tile - i * (i + 1) / 2;
  i += 4 * s;
}

template <int BM, int BN>
struct PairTile {
  long m0, n0;
  int index;  // among the tiles of a symmetric product
  bool any, mirror;

  __device__ __forceinline__ PairTile(const PairArgs& g) {
    const int turn = gridDim.x < 8 ? 0 : (int)(blockIdx.y + blockIdx.z) % 8;
    if (g.symmetric) {
      const int side = (int)((g.M + BM - 1) / BM), total = side * (side + 1) / 2, per = (total + 7) / 8;
      index = ((int)blockIdx.x + turn) % 8 * per + (int)blockIdx.x / 8;
      any = (int)blockIdx.x / 8 < per && index < total;
      int i, j;
      belowDiagonal(any ? index : 0, side, i, j);
      m0 = (long)i * BM, n0 = (long)j * BN;
      mirror = true;
    } else {
      const Tile<BM, BN> t(g.M, g.N, turn);
      m0 = t.m0, n0 = t.n0, any = t.any, index = 0;
      mirror = g.turned.data != nullptr;
    }
  }
};

// A workgroup: BM x BN results over one range of k, a wave WM x WN of them.  ONE: operands (1: b, 3: both) whose second pieces
// are all zeros.  LDS holds the operands of DEPTH steps of 32 k,
// lines of 128 bytes with both pieces.  A step is RM groups of 3 RN matrix instructions: the smaller products first.
template <class RESULT, int ONE, int BM, int BN, int WM, int WN, int DEPTH>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void product(PairArgs g, RESULT result) {
  constexpr int WAVES = BM / WM * (BN / WN), RM = WM / 16, RN = WN / 16;
  typedef Direct<BM, 64, true, WAVES> A;
  typedef Direct<BN, 64, true, WAVES> B;
  constexpr int STEP = A::bytes + B::bytes, LOADS = A::loads + B::loads;
  __shared__ __attribute__((aligned(1024))) char space[DEPTH * STEP];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
  const PairTile<BM, BN> tile(g);
  if (!tile.any) return;
  const long m0 = tile.m0, n0 = tile.n0, first = blockIdx.y * g.range, end = min(first + g.range, g.K), matrix = blockIdx.z;

  A a;
  B b;
  a.setup(g.a.data + matrix * g.a.batch + 2 * (m0 * g.a.cols + first), 2 * g.a.cols, g.M - m0);
  b.setup(g.b.data + matrix * g.b.batch + 2 * (n0 * g.b.cols + first), 2 * g.b.cols, g.N - n0);
  floatx4 sum[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  int left = (int)(end - first) * 2;  // pieces of a row that are not on their way yet
  auto load = [&](int q, char* to) __attribute__((always_inline)) {
    if (q < A::loads)
      a.load(q, left, to);
    else
      b.load(q - A::loads, left, to + A::bytes);
  };
  auto loaded = [&]() __attribute__((always_inline)) {
    a.base += a.advance;
    b.base += b.advance;
    left -= 64;
  };
  // (behind the last step too, without a word, so that as many loads are always on their way)
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
    for (int q = 0; q < LOADS; ++q) load(q, space + d * STEP);
    loaded();
  }
  const int laneA = A::laneAt(wm), laneB = B::laneAt(wn);
  uintx4 fa[2][2], fb[2][2][RN];  // [turn][piece]
  auto readA = [&](int turn, int i, int d) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < (ONE == 3 ? 1 : 2); ++p) fa[turn][p] = A::fragment(space + d * STEP, laneA, p, i);
  };
  auto readB = [&](int d) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < (ONE ? 1 : 2); ++p)
#pragma unroll
      for (int j = 0; j < RN; ++j) fb[d % 2][p][j] = B::fragment(space + d * STEP + A::bytes, laneB, p, j);
  };
  static_assert(RM % 2 == 0 && DEPTH % 2 == 0, "two turns of fragments");
  arrive<(DEPTH - 1) * LOADS>();
  readB(0);
  readA(0, 0, 0);
  auto round = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        const int turn = i % 2;
        if (i + 1 < RM) {
          readA(turn ^ 1, i + 1, d);
        } else {
          // every wave has this step's fragments, so that its place is free, and the next step's operands are there
          arrive<(DEPTH - 2) * LOADS>();
          readB((d + 1) % DEPTH);
          readA(turn ^ 1, 0, (d + 1) % DEPTH);
        }
        if (!ONE) {
#pragma unroll
          for (int j = 0; j < RN; ++j) sum[i][j] = multiply(fb[d % 2][1][j], fa[turn][0], sum[i][j]);
        }
        if (ONE != 3) {
#pragma unroll
          for (int j = 0; j < RN; ++j) sum[i][j] = multiply(fb[d % 2][0][j], fa[turn][1], sum[i][j]);
        }
#pragma unroll
        for (int j = 0; j < RN; ++j) sum[i][j] = multiply(fb[d % 2][0][j], fa[turn][0], sum[i][j]);
        if (i + 1 == RM) {
#pragma unroll
          for (int q = 0; q < LOADS; ++q) load(q, space + d * STEP);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      loaded();
      if (left <= -DEPTH * 64) return false;  // that was the last step
    }
    return true;
  };
  while (round()) {
  }

  // (the loads requested behind the last step write zeros to LDS, which the results now go through)
  arrive<0>();
  constexpr int PITCH = WN + 4;
  static_assert(32 * PITCH * 4 <= DEPTH * STEP / WAVES, "a wave's share of LDS holds 32 rows");
  float* const mine = reinterpret_cast<float*>(space + wave * (DEPTH * STEP / WAVES));
  auto eight = [&](int row, int c, float(&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const floatx4 q = *reinterpret_cast<const floatx4*>(mine + row * PITCH + c + 4 * h);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * h + k] = q[k];
    }
  };
#pragma unroll
  for (int i0 = 0; i0 < RM; i0 += 2) {
    waveExchange();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < RN; ++j) *reinterpret_cast<floatx4*>(mine + (16 * i + lane % 16) * PITCH + 16 * j + lane / 16 * 4) = sum[i0 + i][j];
    waveExchange();
    const int row0 = wm + 16 * i0;
    if (__is_same(RESULT, Nothing) && g.parts) {
      const long tiles = gridDim.x;
      float* const to = g.parts + (((matrix * gridDim.y + blockIdx.y) * tiles + tile.index) * BM + row0) * BN + wn;
#pragma unroll 1
      for (int row = lane / (WN / 8); row < 32; row += 512 / WN) {
        float v[8];
        eight(row, lane % (WN / 8) * 8, v);
        storePack(to + row * BN + lane % (WN / 8) * 8, v);
      }
    } else {
      leavePairs<WN, 1>(g, result, matrix, m0 + row0, n0 + wn, tile.mirror, mine, eight);
    }
  }
}

// Results of a symmetric product from the sums of `ranges` ranges of k, in their order: a workgroup to 32 rows of up to 64 columns
// of a tile, eight ranges' sums on their way at once (60 x 60 in 13 ranges 5.5 us, by a wave and range after range 11.9).
template <int BM, int BN>
__global__ __launch_bounds__(256) void join(PairArgs g, int ranges, int tiles) {
  constexpr int COLS = BN < 64 ? BN : 64, ACROSS = BN / COLS, BLOCKS = BM / 32 * ACROSS, AHEAD = 8;  // BLOCKS: of a tile
  __shared__ __attribute__((aligned(16))) float space[32 * (COLS + 4)];
  const int index = (int)blockIdx.x / BLOCKS, block = (int)blockIdx.x % BLOCKS;
  const long matrix = blockIdx.z;
  int i, j;
  belowDiagonal(index, (int)((g.M + BM - 1) / BM), i, j);
  const int row0 = block / ACROSS * 32, col0 = block % ACROSS * COLS;
  const long m0 = (long)i * BM + row0, n0 = (long)j * BN + col0;
  if (m0 >= g.M || n0 >= g.N) return;
  const long far = (long)tiles * BM * BN;  // from a range to the next
  const float* const from = g.parts + matrix * ranges * far + ((long)index * BM + row0) * BN + col0;
  leavePairs<COLS, 4>(g, Nothing{}, matrix, m0, n0, true, space, [&](int row, int c, float(&v)[8]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.f;
    for (int first = 0; first < ranges; first += AHEAD) {
      float u[AHEAD][8];
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) loadPack<float, 8>(from + min(first + r, ranges - 1) * far + row * BN + c, u[r]);
#pragma unroll
      for (int r = 0; r < AHEAD; ++r)
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] += first + r < ranges ? u[r][q] : 0.f;
    }
  });
}

// Small products.  A workgroup: SIDE x SIDE results over one range of k, its waves a part of that each, straight from memory to
// the matrix instructions; their sums meet in LDS.
template <class RESULT, int SIDE, int WAVES, int AHEAD>
__global__ __launch_bounds__(WAVES * 64) void small(PairArgs g, RESULT result) {
  constexpr int PITCH = SIDE + 4, R = SIDE / 16, LANES = SIDE / 4;
  constexpr bool LAST = !__is_same(RESULT, Nothing);
  __shared__ __attribute__((aligned(16))) float sums[WAVES][SIDE * PITCH];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const PairTile<SIDE, SIDE> tile(g);
  if (!tile.any) return;
  const long m0 = tile.m0, n0 = tile.n0, matrix = blockIdx.z;
  // (four neighbouring results to a lane of the first ones, which what stands beside them is on its way to already)
  const int row = threadIdx.x / LANES, c = threadIdx.x % LANES * 4;
  const long m = m0 + row, n = n0 + c;
  halfx4 oldLead{}, oldRest{};
  if (row < SIDE && g.old.data && (LAST || !g.parts)) {
    const half16* const from = g.old.data + matrix * g.old.batch + placeOf(g.old, m, n);
    oldLead = *reinterpret_cast<const halfx4*>(from), oldRest = *reinterpret_cast<const halfx4*>(from + 32);
  }
  const float factor = g.factors ? g.factors[matrix] : 1.f;
  const long begin = blockIdx.y * g.range, stop = min(begin + g.range, g.K);
  const long share = ((stop - begin) / 32 + WAVES - 1) / WAVES * 32, first = begin + wave * share, end = min(first + share, stop);
  const half16* a[R];
  const half16* b[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    a[i] = g.a.data + matrix * g.a.batch + 2 * (m0 + 16 * i + lane % 16) * g.a.cols + lane / 16 * 8;
    b[i] = g.b.data + matrix * g.b.batch + 2 * (n0 + 16 * i + lane % 16) * g.b.cols + lane / 16 * 8;
  }
  floatx4 sum[R][R] = {};
  for (long k0 = first; k0 < end; k0 += 32 * AHEAD) {
    uintx4 fa[AHEAD][R][2], fb[AHEAD][R][2];  // [step][rows][piece]
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const long k = min(k0 + 32 * s, end - 32);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          fa[s][i][p] = *reinterpret_cast<const uintx4*>(a[i] + 2 * k + 32 * p);
          fb[s][i][p] = *reinterpret_cast<const uintx4*>(b[i] + 2 * k + 32 * p);
        }
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      if (k0 + 32 * s >= end) break;
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) sum[i][j] = multiply(fb[s][j][1], fa[s][i][0], sum[i][j]);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) sum[i][j] = multiply(fb[s][j][0], fa[s][i][1], sum[i][j]);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) sum[i][j] = multiply(fb[s][j][0], fa[s][i][0], sum[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j)
      *reinterpret_cast<floatx4*>(&sums[wave][(16 * i + lane % 16) * PITCH + 16 * j + lane / 16 * 4]) = sum[i][j];
  __syncthreads();
  bool turns = tile.mirror && !g.parts;
  if constexpr (LAST) turns = result.y.row == 1 && result.y.col != 1;
  float z[4] = {};
  if (row < SIDE) {
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const floatx4 q = *reinterpret_cast<const floatx4*>(&sums[w][row * PITCH + c]);
#pragma unroll
      for (int v = 0; v < 4; ++v) z[v] += q[v];
    }
    if (!LAST && g.parts) {
      storePack(g.parts + (((matrix * gridDim.y + blockIdx.y) * gridDim.x + tile.index) * SIDE + row) * SIDE + c, z);
      return;
    }
    const float by = g.by * factor * (g.power == 2 ? factor : 1.f), beta = g.beta * factor;
#pragma unroll
    for (int v = 0; v < 4; ++v) z[v] *= by;
    if (g.old.data) {
#pragma unroll
      for (int v = 0; v < 4; ++v) z[v] += beta * ((float)oldLead[v] + (float)oldRest[v]);
    }
    if constexpr (LAST) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        z[v] *= result.scale;
        if (!turns && m < result.rows && n + v < result.cols)
          storePack(result.y.data + matrix * result.y.batch + m * result.y.row + (n + v) * result.y.col, {z[v]});
      }
    } else {
      storeFour(g.out.data + matrix * g.out.batch + placeOf(g.out, m, n), z, 0, g.symmetric ? (int)min(m - n + 1, 4l) : 4);
    }
    if (turns) *reinterpret_cast<floatx4*>(&sums[0][row * PITCH + c]) = floatx4{z[0], z[1], z[2], z[3]};
  }
  if (!turns) return;
  __syncthreads();
  if (row < SIDE) {
    // now a column, four of its rows
#pragma unroll
    for (int v = 0; v < 4; ++v) z[v] = sums[0][(c + v) * PITCH + row];
    if constexpr (LAST) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (n0 + row < result.cols && m0 + c + v < result.rows)
          storePack(result.y.data + matrix * result.y.batch + (n0 + row) * result.y.col + (m0 + c + v) * result.y.row, {z[v]});
    } else {
      storeFour(g.turned.data + matrix * g.turned.batch + placeOf(g.turned, n0 + row, m0 + c), z,
                g.symmetric ? (int)max(n0 + row + 1 - (m0 + c), 0l) : 0, 4);
    }
  }
}

// ---- small matrices: all steps in one launch ----

// A workgroup to a matrix, whose X, A and B stay in LDS: pair lines of 32 columns as in memory, rows 16 bytes further apart, so that
// the 16 rows of a fragment take all banks.  Waves take blocks of 16 x 16 results in turn; X's columns, which the last product
// of a step sums over X's rows, come by the transposing read.
constexpr int kWholeLanes = 1024;
constexpr int kWholeBlocks = 2;        // of a symmetric matrix to a wave
constexpr int kWholeSmall = 64 << 10;  // bytes of LDS

struct WholeArgs {
  long rows, cols;
  int P, Q, steps;
  float eps, scale;
  float coefficients[96];
};

// Eight k from 32 kb + 8 (lane / 16) of row first + lane % 16.
__device__ __forceinline__ uintx4 wholeFragment(const char* m, int pitch, int first, int kb, int piece) {
  const int lane = threadIdx.x % 64;
  return *reinterpret_cast<const uintx4*>(m + (first + lane % 16) * pitch + kb * 128 + piece * 64 + lane / 16 * 16);
}
// The same of a matrix that lies the other way round, [k][row].  (Of sixteen lanes, lane l gives the address of four rows (l % 4)
// of k (l / 4) and gets four k of row l.)
__device__ __forceinline__ uintx4 wholeTurned(const char* m, int pitch, int first, int kb, int piece) {
  const int lane = threadIdx.x % 64, at = first + lane % 4 * 4;
  uintx4 f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = 32 * kb + lane / 16 * 8 + lane % 16 / 4 + 4 * h;
    const char* const from = m + k * pitch + at / 32 * 128 + piece * 64 + at % 32 * 2;
    const uintx2 u = __builtin_bit_cast(
        uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)const_cast<char*>(from)));
    f[2 * h] = u[0];
    f[2 * h + 1] = u[1];
  }
  return f;
}

// a block's sums, of kbs steps: a(kb, piece) and b(kb, piece) give the fragments.  (Three sums, which do not wait for each other.)
template <class A, class B>
__device__ __forceinline__ floatx4 wholeSums(int kbs, A a, B b) {
  floatx4 s0{0.f, 0.f, 0.f, 0.f}, s1 = s0, s2 = s0;
  for (int kb = 0; kb < kbs; ++kb) {
    const uintx4 a0 = a(kb, 0), a1 = a(kb, 1), b0 = b(kb, 0), b1 = b(kb, 1);
    s1 = multiply(b1, a0, s1);
    s2 = multiply(b0, a1, s2);
    s0 = multiply(b0, a0, s0);
  }
  return s0 + (s1 + s2);
}

__device__ __forceinline__ void wholePair(char* m, int pitch, int i, int j, half16& lead, half16& rest) {
  const half16* const at = reinterpret_cast<const half16*>(m + i * pitch + j / 32 * 128) + j % 32;
  lead = at[0], rest = at[32];
}

// This lane's four results of block (i, j), of row m = 16 i + lane % 16 and columns from n = 16 j + 4 (lane / 16), of a symmetric
// matrix: what lies on and below the diagonal, and its mirror image.
__device__ __forceinline__ void wholeSymmetric(char* to, int pitch, int i, int j, const float (&z)[4]) {
  const int lane = threadIdx.x % 64, m = 16 * i + lane % 16, n = 16 * j + lane / 16 * 4;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    if (n + v > m) continue;
    const half16 lead = (half16)z[v], rest = (half16)(z[v] - (float)lead);
    half16* const here = reinterpret_cast<half16*>(to + m * pitch + (n + v) / 32 * 128) + (n + v) % 32;
    half16* const there = reinterpret_cast<half16*>(to + (n + v) * pitch + m / 32 * 128) + m % 32;
    here[0] = lead, here[32] = rest;
    there[0] = lead, there[32] = rest;
  }
}

template <class T, int BYTES>
__global__ __launch_bounds__(kWholeLanes) void whole(Given<const T> g, Given<T> y, WholeArgs w) {
  constexpr int WAVES = kWholeLanes / 64;
  __shared__ __attribute__((aligned(128))) char space[BYTES];
  __shared__ double sums[WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, P = w.P, Q = w.Q;
  const int pitchX = 4 * Q + 16, pitchA = 4 * P + 16;
  char *const x = space, *const gram = x + P * pitchX, *const poly = gram + P * pitchA;
  const T* const from = g.data + blockIdx.x * g.batch;
  T* const to = y.data + blockIdx.x * y.batch;

  // G as numbers of 32 bits, in the place of their pairs, and its squares
  double sum = 0;
  const bool lines = g.row == 1 && g.col != 1;  // columns are the lines of neighbours
  const int words = (lines ? P : Q) / 8, total = (lines ? Q : P) * words;
  for (int at = threadIdx.x; at < total; at += kWholeLanes) {
    const int line = at / words, in = (at - line * words) * 8;
    const long here = lines ? w.cols : w.rows, count = lines ? w.rows : w.cols;
    float v[8] = {};
    if (line < here) loadEight(from + line * (lines ? g.col : g.row), lines ? g.row : g.col, in, count, v);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      sum += (double)v[q] * (double)v[q];
      const int i = lines ? in + q : line, j = lines ? line : in + q;
      *reinterpret_cast<float*>(x + i * pitchX + 4 * j) = v[q];
    }
  }
  sum = waveSum(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int q = 0; q < WAVES; ++q) sum += sums[q];
  const double by = (double)kUnit / (__builtin_sqrt(sum) + (double)w.eps);
  // (eight lanes to a line of 32 numbers, all of a wave's before any of its pairs)
  for (int first = 0; first < P * (Q / 32); first += kWholeLanes / 8) {
    const int at = first + threadIdx.x / 8, i = at / (Q / 32), in = threadIdx.x % 8 * 4;
    char* const line = x + i * pitchX + (at - i * (Q / 32)) * 128;
    float z[4] = {};
    if (i < P) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(line + in * 4);
#pragma unroll
      for (int q = 0; q < 4; ++q) z[q] = (float)((double)v[q] * by);
    }
    waveExchange();
    if (i < P) storeFour(reinterpret_cast<half16*>(line) + in, z, 0, 4);
    waveExchange();
  }
  __syncthreads();

  const float one = 1.f / kUnit;
  const int down = P / 16, triangle = down * (down + 1) / 2, across = Q / 16;
  int rows[kWholeBlocks], cols[kWholeBlocks];  // of this wave's blocks of a symmetric matrix
#pragma unroll
  for (int q = 0; q < kWholeBlocks; ++q) {
    const int t = wave + WAVES * q;
    belowDiagonal(t < triangle ? t : 0, down, rows[q], cols[q]);
  }
  // waves that share 16 columns of X, where there are fewer of those than waves
  const int shares = across >= WAVES ? 1 : across >= WAVES / 2 ? 2 : 4, rounds = (across * shares + WAVES - 1) / WAVES;
  for (int step = 0; step < w.steps; ++step) {
    const float a = w.coefficients[3 * step], b = w.coefficients[3 * step + 1], c = w.coefficients[3 * step + 2];
#pragma unroll
    for (int q = 0; q < kWholeBlocks; ++q) {
      if (wave + WAVES * q >= triangle) break;
      const int i = rows[q], j = cols[q];
      const floatx4 s = wholeSums(
          Q / 32, [&](int kb, int p) { return wholeFragment(x, pitchX, 16 * i, kb, p); },
          [&](int kb, int p) { return wholeFragment(x, pitchX, 16 * j, kb, p); });
      wholeSymmetric(gram, pitchA, i, j, {s[0] * one, s[1] * one, s[2] * one, s[3] * one});
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kWholeBlocks; ++q) {
      if (wave + WAVES * q >= triangle) break;
      const int i = rows[q], j = cols[q];
      const floatx4 s = wholeSums(
          P / 32, [&](int kb, int p) { return wholeFragment(gram, pitchA, 16 * i, kb, p); },
          [&](int kb, int p) { return wholeFragment(gram, pitchA, 16 * j, kb, p); });
      const int m = 16 * i + lane % 16, n = 16 * j + lane / 16 * 4;
      float z[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        half16 lead, rest;
        wholePair(gram, pitchA, m, n + v, lead, rest);
        z[v] = c * one * s[v] + b * ((float)lead + (float)rest);
      }
      wholeSymmetric(poly, pitchA, i, j, z);
    }
    __syncthreads();
    // 16 columns of X at a time, overwritten where they lie, when all that they are summed from is in registers
    const bool last = step + 1 == w.steps;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
      const int task = wave + WAVES * round, j = task / shares;
      uintx4 columns[kWholeSteps][2];
      if (j < across) {
#pragma unroll
        for (int kb = 0; kb < kWholeSteps; ++kb)
          if (kb < P / 32)
#pragma unroll
            for (int piece = 0; piece < 2; ++piece) columns[kb][piece] = wholeTurned(x, pitchX, 16 * j, kb, piece);
      }
      if (shares > 1)
        __syncthreads();
      else
        waveExchange();
      if (j >= across) continue;
      for (int i = task % shares; i < down; i += shares) {
        floatx4 s0{0.f, 0.f, 0.f, 0.f}, s1 = s0, s2 = s0;
#pragma unroll
        for (int kb = 0; kb < kWholeSteps; ++kb)
          if (kb < P / 32) {
            const uintx4 a0 = wholeFragment(poly, pitchA, 16 * i, kb, 0), a1 = wholeFragment(poly, pitchA, 16 * i, kb, 1);
            s1 = multiply(columns[kb][1], a0, s1);
            s2 = multiply(columns[kb][0], a1, s2);
            s0 = multiply(columns[kb][0], a0, s0);
          }
        const int m = 16 * i + lane % 16, n = 16 * j + lane / 16 * 4;
        half16* const here = reinterpret_cast<half16*>(x + m * pitchX + n / 32 * 128) + n % 32;
        const halfx4 lead = *reinterpret_cast<const halfx4*>(here), rest = *reinterpret_cast<const halfx4*>(here + 32);
        float z[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) z[v] = one * (s0[v] + (s1[v] + s2[v])) + a * ((float)lead[v] + (float)rest[v]);
        if (!last) {
          storeFour(here, z, 0, 4);
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (m < w.rows && n + v < w.cols) storePack(to + m * y.row + (n + v) * y.col, {z[v] * w.scale});
        }
      }
    }
    if (!last) __syncthreads();
  }
}

size_t partsBytes(const PairPlan& p, long batch) {
  return p.ranges > 1 ? (size_t)batch * p.ranges * p.tiles * p.side * p.side * sizeof(float) : 0;
}

template <class RESULT, int SIDE>
void launchSmall(const PairArgs& g, const RESULT& result, dim3 grid, hipStream_t s) {
  // (as many waves as there are steps for, two steps of each ahead)
  if (g.range <= 256)
    small<RESULT, SIDE, 4, 2><<<grid, 256, 0, s>>>(g, result);
  else if (g.range <= 512)
    small<RESULT, SIDE, 8, 2><<<grid, 512, 0, s>>>(g, result);
  else
    small<RESULT, SIDE, 16, 2><<<grid, 1024, 0, s>>>(g, result);
}

// one: see product's ONE (float32 matrices have second pieces everywhere, the last product's first operand always has)
template <class RESULT>
void launchProduct(PairArgs g, const RESULT& result, const PairPlan& plan, int one, float* parts, unsigned batch, hipStream_t s) {
  const dim3 grid((unsigned)plan.tiles, (unsigned)plan.ranges, batch);
  g.range = plan.range;
  if (plan.ranges > 1) g.parts = parts;
  auto tiles = [&](auto pieces) {
    constexpr int ONE = decltype(pieces)::value;
    if (plan.kind == Deep64)
      product<RESULT, ONE, 64, 64, 32, 32, 4><<<grid, 256, 0, s>>>(g, result);
    else if (plan.kind == Wide64)
      product<RESULT, ONE, 64, 64, 32, 32, 2><<<grid, 256, 0, s>>>(g, result);
    else if (plan.kind == Deep128)
      product<RESULT, ONE, 128, 128, 32, 64, 4><<<grid, 512, 0, s>>>(g, result);
    else if (plan.kind == Wide128)
      product<RESULT, ONE, 128, 128, 64, 32, 2><<<grid, 512, 0, s>>>(g, result);
    else
      product<RESULT, ONE, 256, 256, 128, 64, 2><<<grid, 512, 0, s>>>(g, result);
  };
  if (plan.kind == Small16)
    launchSmall<RESULT, 16>(g, result, grid, s);
  else if (plan.kind == Small32)
    launchSmall<RESULT, 32>(g, result, grid, s);
  else if (one == 0)
    tiles(std::integral_constant<int, 0>());
  else if constexpr (!__is_same(RESULT, Result<float>)) {
    if (one == 1) tiles(std::integral_constant<int, 1>());
    if constexpr (__is_same(RESULT, Nothing))
      if (one == 3) tiles(std::integral_constant<int, 3>());
  }
  if (plan.ranges > 1) {  // (symmetric products)
    const long down = ceilDivLong(g.M, plan.side), count = down * (down + 1) / 2;
    const dim3 blocks((unsigned)(count * (plan.side / 32) * (plan.side > 32 ? plan.side / 64 : 1)), 1, batch);
    const int ranges = (int)plan.ranges, rounded = (int)plan.tiles;
    if (plan.side == 32)
      join<32, 32><<<blocks, 256, 0, s>>>(g, ranges, rounded);
    else if (plan.side == 64)
      join<64, 64><<<blocks, 256, 0, s>>>(g, ranges, rounded);
    else if (plan.side == 128)
      join<128, 128><<<blocks, 256, 0, s>>>(g, ranges, rounded);
    else
      join<256, 256><<<blocks, 256, 0, s>>>(g, ranges, rounded);
  }
}

// What lies in the workspace, for so many matrices of P x Q, and how the products run: of X with its transpose, of the P x P
// matrices, and of them with X.
struct Space {
  double* sums;
  float* factors;
  Pairs x, xt[2], gram, poly;
  float* parts;
  size_t bytes;
  PairPlan gramPlan, polyPlan, lastPlan;

  Space(void* workspace, long batch, long P, long Q)
      : gramPlan(planOf(true, batch, P, P, Q, computeUnits())), polyPlan(planOf(true, batch, P, P, P, computeUnits())),
        lastPlan(planOf(false, batch, P, Q, P, computeUnits())) {
    char* at = static_cast<char*>(workspace);
    auto take = [&](size_t size) {
      char* const from = at;
      at += rounded(size);
      return from;
    };
    sums = reinterpret_cast<double*>(take((size_t)batch * kShares * sizeof(double)));
    factors = reinterpret_cast<float*>(take((size_t)batch * sizeof(float)));
    auto pairs = [&](long rows, long cols) {
      return Pairs{reinterpret_cast<half16*>(take((size_t)batch * 2 * rows * cols * sizeof(half16))), cols, 2 * rows * cols};
    };
    x = pairs(P, Q), xt[0] = pairs(Q, P), xt[1] = pairs(Q, P), gram = pairs(P, P), poly = pairs(P, P);
    size_t most = 0;
    for (const PairPlan* p : {&gramPlan, &polyPlan, &lastPlan}) most = std::max(most, partsBytes(*p, batch));
    parts = reinterpret_cast<float*>(take(most));
    bytes = at - static_cast<char*>(workspace);
  }

  bool fits(long batch) const {
    for (const PairPlan* p : {&gramPlan, &polyPlan, &lastPlan})
      // (workgroups of up to 1024 lanes, or of 256 to 32 x 32 or 32 x 64 of the results)
      if (!launches((double)p->tiles * std::max(p->ranges, p->ranges > 1 ? p->side * p->side / 4096 + 1l : 1l) * batch, 1024)) return false;
    return true;
  }
};

// One call: the matrices, and its launches.
template <class T>
struct Call {
  const OrthogonalProblem& p;
  hipStream_t s;
  bool turn;
  long rows, cols, P, Q;  // X has no more rows than columns; filled up
  Given<const T> g;
  Given<T> y;
  Space w;

  Call(const OrthogonalProblem& problem, hipStream_t stream)
      : p(problem), s(stream), turn(p.rows > p.cols), rows(turn ? p.cols : p.rows), cols(turn ? p.rows : p.cols), P(padded(rows)),
        Q(padded(cols)), g{static_cast<const T*>(p.x.data), turn ? p.x.col : p.x.row, turn ? p.x.row : p.x.col, p.xBatch},
        y{static_cast<T*>(p.y.data), turn ? p.y.col : p.y.row, turn ? p.y.row : p.y.col, p.yBatch}, w(p.workspace, p.batch, P, Q) {}

  static constexpr bool SHORT = sizeof(T) == 2;  // X is single pieces at first
  static constexpr float one = 1.f / kUnit;
  unsigned batch() const { return (unsigned)p.batch; }
  float coefficient(int step, int i) const { return p.coefficients[3 * step + i]; }
  Result<T> result() const { return {y, rows, cols, p.scale / kUnit}; }

  void squaresAndX(long squared) {
    // lines of neighbours, for the squares
    const bool lines = g.row == 1 && g.col != 1;
    const Given<const T> by{g.data, lines ? g.col : g.row, lines ? g.row : g.col, g.batch};
    const long count = lines ? rows : cols;
    squares<T><<<dim3(kShares, batch()), 256, 0, s>>>(by, lines ? cols : rows, count, divisorOf(ceilDivLong(count, 8)), w.sums);
    const dim3 grid((unsigned)squared, batch());
    if (lines)
      begin<T, true><<<grid, 256, 0, s>>>(g, rows, cols, w.sums, p.eps, w.x, w.xt[0], w.factors);
    else
      begin<T, false><<<grid, 256, 0, s>>>(g, rows, cols, w.sums, p.eps, w.x, w.xt[0], w.factors);
  }

  void steps() {
    for (int i = 0; i < p.steps; ++i) {
      const float a = coefficient(i, 0), b = coefficient(i, 1), c = coefficient(i, 2);
      const bool first = i == 0;
      launchProduct(PairArgs{w.x, w.x, P, P, Q, 0, one, 0.f, first ? w.factors : nullptr, 2, Pairs{}, w.gram, w.gram, true, nullptr}, Nothing{},
                    w.gramPlan, SHORT && first ? 3 : 0, w.parts, batch(), s);
      launchProduct(PairArgs{w.gram, w.gram, P, P, P, 0, c * one, b, nullptr, 0, w.gram, w.poly, w.poly, true, nullptr}, Nothing{}, w.polyPlan, 0,
                    w.parts, batch(), s);
      const PairArgs x{w.poly, w.xt[i % 2], P, Q, P, 0, one, a, first ? w.factors : nullptr, 1, w.x, w.x, w.xt[(i + 1) % 2], false, nullptr};
      if (i + 1 < p.steps)
        launchProduct(x, Nothing{}, w.lastPlan, SHORT && first ? 1 : 0, w.parts, batch(), s);
      else
        launchProduct(x, result(), w.lastPlan, SHORT && first ? 1 : 0, w.parts, batch(), s);
    }
  }
};

template <class T>
void launchWhole(const OrthogonalProblem& p, hipStream_t s) {
  const bool turn = p.rows > p.cols;
  const long rows = turn ? p.cols : p.rows, cols = turn ? p.rows : p.cols, P = padded(rows), Q = padded(cols), bytes = wholeBytes(P, Q);
  Given<const T> g{static_cast<const T*>(p.x.data), turn ? p.x.col : p.x.row, turn ? p.x.row : p.x.col, p.xBatch};
  Given<T> y{static_cast<T*>(p.y.data), turn ? p.y.col : p.y.row, turn ? p.y.row : p.y.col, p.yBatch};
  WholeArgs w{rows, cols, (int)P, (int)Q, p.steps, p.eps, p.scale / kUnit, {}};
  for (int i = 0; i < 3 * p.steps; ++i) w.coefficients[i] = p.coefficients[i];
  // (as many matrices at a time as a launch, which counts its lanes in 32 bits, holds)
  constexpr long most = 0xffffffffl / kWholeLanes;
  for (long first = 0; first < p.batch; first += most, g.data += most * g.batch, y.data += most * y.batch) {
    const dim3 grid((unsigned)std::min(most, p.batch - first));
    if (bytes <= kWholeSmall)
      whole<T, kWholeSmall><<<grid, kWholeLanes, 0, s>>>(g, y, w);
    else
      whole<T, kWholeLarge><<<grid, kWholeLanes, 0, s>>>(g, y, w);
  }
}

template <class T>
int run(const OrthogonalProblem& p, hipStream_t s) {
  if (inOneLaunch(padded(std::min(p.rows, p.cols)), padded(std::max(p.rows, p.cols)))) {
    launchWhole<T>(p, s);
    return launchStatus();
  }
  Call<T> call(p, s);
  const long squared = ceilDivLong(call.P, 64) * ceilDivLong(call.Q, 64);
  if (p.batch > 65535 || !launches((double)squared * p.batch, 256) || !call.w.fits(p.batch)) return FBFFT_UNSUPPORTED_SIZE;
  call.squaresAndX(squared);
  call.steps();
  return launchStatus();
}

}  // namespace

size_t orthogonalWorkspaceBytes(long batch, long rows, long cols) {
  const long P = padded(std::min(rows, cols)), Q = padded(std::max(rows, cols));
  // (matrices in LDS leave it alone, whatever their number: one matrix's)
  return Space(nullptr, inOneLaunch(P, Q) ? 1 : batch, P, Q).bytes;
}

int launchOrthogonalize(const OrthogonalProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return run<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? run<half16>(p, s) : run<brain16>(p, s);
}

}  // namespace fbfft_amd
