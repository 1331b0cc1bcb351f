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
// A pair matrix has rows of a multiple of 32 columns, 32 leading pieces and then their 32 second pieces, 128 bytes: what a
// matrix instruction takes of a row.  Rows and columns are filled up with zeros.
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef half16 halfx8 __attribute__((ext_vector_type(8)));

constexpr float kUnit = 1024.f;  // what stands for 1 in pieces

struct Pairs {
  half16* data;
  long cols;   // a multiple of 32; a row has 2 cols pieces
  long batch;  // pieces from a matrix to the next
};

__device__ __forceinline__ long placeOf(const Pairs& m, long i, long j) { return 2 * (i * m.cols + j / 32 * 32) + j % 32; }
__device__ __forceinline__ void storePair(const Pairs& m, long i, long j, float v) {
  half16* const to = m.data + placeOf(m, i, j);
  const half16 lead = (half16)v;
  to[0] = lead;
  to[32] = (half16)(v - (float)lead);
}
__device__ __forceinline__ float loadPair(const Pairs& m, long i, long j) {
  const half16* const from = m.data + placeOf(m, i, j);
  return (float)from[0] + (float)from[32];
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

// Squares are summed in 64 bits: those of float32 values pass its range.
template <class T>
__global__ __launch_bounds__(256) void squares(Given<const T> g, long rows, long cols, double* sums) {
  __shared__ double space[4];
  const T* const from = g.data + blockIdx.y * g.batch;
  double sum = 0;
  for (long i = blockIdx.x; i < rows; i += kShares)
    for (long j = threadIdx.x; j < cols; j += 256) {
      const double v = (double)(float)from[i * g.row + j * g.col];
      sum += v * v;
    }
  sum = groupSum(sum, space);
  if (threadIdx.x == 0) sums[blockIdx.y * kShares + blockIdx.x] = sum;
}

// X and its transpose from G: rows <= cols of them, up to the padded sizes.
template <class T>
__global__ __launch_bounds__(256) void begin(Given<const T> g, long rows, long cols, const double* sums, float eps, Pairs x, Pairs xt) {
  __shared__ double space[4];
  const double norm = __builtin_sqrt(groupSum(sums[blockIdx.y * kShares + threadIdx.x], space));
  const double by = (double)kUnit / (norm + (double)eps);
  x.data += blockIdx.y * x.batch, xt.data += blockIdx.y * xt.batch;
  const long tall = xt.cols;  // rows of x
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < tall * x.cols; at += (long)gridDim.x * 256) {
    const long i = at / x.cols, j = at - i * x.cols;
    const float v = i < rows && j < cols ? (float)((double)(float)g.data[blockIdx.y * g.batch + i * g.row + j * g.col] * by) : 0.f;
    storePair(x, i, j, v);
    storePair(xt, j, i, v);
  }
}

__device__ __forceinline__ floatx4 multiply(halfx8 a, halfx8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

struct PairProduct {
  Pairs a, b;       // rows of both, k contiguous: a b^T
  long M, N, K;     // padded
  float by, beta;   // result: by (sum in units of 2^20) + beta old
  Pairs old, out, turned;  // old, turned: data may be null
};

// A wave: 32 x 32 results, straight from memory to the matrix instructions.  LAST: the result goes to the caller's matrix.
template <class T, bool LAST>
__global__ __launch_bounds__(256) void product(PairProduct p, Given<T> y, long rows, long cols, float scale) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const long across = p.N / 32, tile = blockIdx.x * 4l + wave, m0 = tile / across * 32, n0 = tile % across * 32;
  if (m0 >= p.M) return;
  const half16 *const a = p.a.data + blockIdx.y * p.a.batch, *const b = p.b.data + blockIdx.y * p.b.batch;
  floatx4 sum[2][2] = {};
  for (long k = 0; k < p.K; k += 32) {
    halfx8 fa[2][2], fb[2][2];  // [block of rows][piece]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const long in = 2 * k + 32 * q + lane / 16 * 8;
        fa[i][q] = *reinterpret_cast<const halfx8*>(a + 2 * (m0 + 16 * i + lane % 16) * p.a.cols + in);
        fb[i][q] = *reinterpret_cast<const halfx8*>(b + 2 * (n0 + 16 * i + lane % 16) * p.b.cols + in);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sum[i][j] = multiply(fb[j][1], fa[i][0], sum[i][j]);
        sum[i][j] = multiply(fb[j][0], fa[i][1], sum[i][j]);
        sum[i][j] = multiply(fb[j][0], fa[i][0], sum[i][j]);
      }
  }
  Pairs old = p.old, out = p.out, turned = p.turned;
  old.data += blockIdx.y * old.batch, out.data += blockIdx.y * out.batch, turned.data += blockIdx.y * turned.batch;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const long m = m0 + 16 * i + lane % 16, n = n0 + 16 * j + lane / 16 * 4 + v;
        float z = sum[i][j][v] * p.by;
        if (p.old.data) z += p.beta * loadPair(old, m, n);
        if (LAST) {
          if (m < rows && n < cols) y.data[blockIdx.y * y.batch + m * y.row + n * y.col] = (T)(z * scale);
        } else {
          storePair(out, m, n, z);
          if (p.turned.data) storePair(turned, n, m, z);
        }
      }
}

long padded(long n) { return (n + 31) / 32 * 32; }
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// What lies in the workspace, for so many matrices of P x Q.
struct Space {
  double* sums;
  Pairs x, xt[2], gram, poly;
  size_t bytes;

  Space(void* workspace, long batch, long P, long Q) {
    char* at = static_cast<char*>(workspace);
    sums = reinterpret_cast<double*>(at);
    at += rounded((size_t)batch * kShares * sizeof(double));
    auto pairs = [&](long rows, long cols) {
      const Pairs m{reinterpret_cast<half16*>(at), cols, 2 * rows * cols};
      at += rounded((size_t)batch * 2 * rows * cols * sizeof(half16));
      return m;
    };
    x = pairs(P, Q), xt[0] = pairs(Q, P), xt[1] = pairs(Q, P), gram = pairs(P, P), poly = pairs(P, P);
    bytes = at - static_cast<char*>(workspace);
  }
};

template <class T>
int run(const OrthogonalProblem& p, hipStream_t s) {
  // (X has no more rows than columns)
  const bool turn = p.rows > p.cols;
  const long rows = turn ? p.cols : p.rows, cols = turn ? p.rows : p.cols, P = padded(rows), Q = padded(cols);
  const Given<const T> g{static_cast<const T*>(p.x.data), turn ? p.x.col : p.x.row, turn ? p.x.row : p.x.col, p.xBatch};
  const Given<T> y{static_cast<T*>(p.y.data), turn ? p.y.col : p.y.row, turn ? p.y.row : p.y.col, p.yBatch};
  Space w(p.workspace, p.batch, P, Q);
  const long most = 65535;
  if (p.batch > most || !launches((double)p.batch * (P / 32 * (Q / 32) / 4 + 1), 256)) return FBFFT_UNSUPPORTED_SIZE;
  const unsigned batch = (unsigned)p.batch;
  auto blocks = [&](long M, long N) { return dim3((unsigned)((M / 32 * (N / 32) + 3) / 4), batch); };
  squares<T><<<dim3(kShares, batch), 256, 0, s>>>(g, rows, cols, w.sums);
  begin<T><<<dim3((unsigned)std::min((P * Q + 255) / 256, 4096l), batch), 256, 0, s>>>(g, rows, cols, w.sums, p.eps, w.x, w.xt[0]);
  const float one = 1.f / kUnit;
  for (int i = 0; i < p.steps; ++i) {
    const float a = p.coefficients[3 * i], b = p.coefficients[3 * i + 1], c = p.coefficients[3 * i + 2];
    const Pairs from = w.xt[i % 2], to = w.xt[(i + 1) % 2], none{};
    product<T, false><<<blocks(P, P), 256, 0, s>>>(PairProduct{w.x, w.x, P, P, Q, one, 0.f, none, w.gram, none}, y, 0, 0, 0.f);
    product<T, false><<<blocks(P, P), 256, 0, s>>>(PairProduct{w.gram, w.gram, P, P, P, c * one, b, w.gram, w.poly, none}, y, 0, 0, 0.f);
    const PairProduct last{w.poly, from, P, Q, P, one, a, w.x, w.x, to};
    if (i + 1 < p.steps)
      product<T, false><<<blocks(P, Q), 256, 0, s>>>(last, y, 0, 0, 0.f);
    else
      product<T, true><<<blocks(P, Q), 256, 0, s>>>(last, y, rows, cols, p.scale / kUnit);
  }
  return launchStatus();
}

}  // namespace

size_t orthogonalWorkspaceBytes(long batch, long rows, long cols) {
  return Space(nullptr, batch, padded(std::min(rows, cols)), padded(std::max(rows, cols))).bytes;
}

int launchOrthogonalize(const OrthogonalProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return run<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? run<half16>(p, s) : run<brain16>(p, s);
}

}  // namespace fbfft_amd
