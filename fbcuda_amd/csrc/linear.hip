// Rows times a weight matrix with bias, activation and residual, and its gradients.
//
//   forward    z = x w^T + bias,  y = activation(z) + residual
//   backward   dz = dy activation'(z);  dx = dz w,  dw = dz^T x,  dbias = sum of dz's rows
//
// All three products are sum_k A[i][k] B[j][k] for operands whose unit stride lies along k or along the row, on the
// 16-bit matrix instructions with fp32 sums.  float32 operands are cut into three bf16 pieces of 8 bits each (exactly:
// the pieces are the leading, middle and last bits), of whose nine products the six largest are summed; what is left
// out is below 2^-23 of a product.
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef half16 halfx8 __attribute__((ext_vector_type(8)));
typedef brain16 brainx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct Epilogue {
  Matrix out, residual, z;  // data null: none of it
  Line bias;
  int activation;
  float* parts;  // not null: fp32 sums of each range of k, [range][M][N], in place of results
};

struct ProductArgs {
  Matrix a, b;
  long M, N, K, range;  // k per range
  Epilogue e;
};

__device__ __forceinline__ floatx4 multiply(uintx4 a, uintx4 b, floatx4 c, half16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 multiply(uintx4 a, uintx4 b, floatx4 c, brain16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(brainx8, a), __builtin_bit_cast(brainx8, b), c, 0, 0, 0);
}

template <class T>
struct Pieces {
  static constexpr int count = 1;
  typedef T type;
};
template <>
struct Pieces<float> {
  static constexpr int count = 3;
  typedef brain16 type;
};

// the leading 16 bits of each of two floats, one above the other
__device__ __forceinline__ unsigned leading(float low, float high) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, high), __builtin_bit_cast(unsigned, low), 0x07060302);
}
__device__ __forceinline__ float withoutLeading(float v) {
  return v - __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & 0xFFFF0000u);
}

constexpr int kTile = 128, kStep = 32;  // rows of either operand and k of a step

// One step of an operand, [row][k] or [k][row], as 16-bit pieces in LDS: 16-byte words that are permuted so that the
// lanes of a fragment's read spread over the banks.  KC: k is contiguous.
template <class T, bool KC>
struct Stage {
  static constexpr int per = 16 / sizeof(T), words = kTile * kStep / per / 256, pieceBytes = kTile * kStep * 2;
  typename Pack<T, per>::type v[words];

  __device__ __forceinline__ void load(const Matrix& m, long row0, long rows, long k0, long end) {
    const T* const data = static_cast<const T*>(m.data);
#pragma unroll
    for (int i = 0; i < words; ++i) {
      const int w = threadIdx.x + 256 * i;
      const long row = row0 + (KC ? w / (kStep / per) : w % (kTile / per) * per);
      const long k = k0 + (KC ? w % (kStep / per) * per : w / (kTile / per));
      const long inner = KC ? m.col : m.row;
      if (inner == 1 && (KC ? row < rows && k + per <= end : k < end && row + per <= rows)) {
        v[i] = *reinterpret_cast<const typename Pack<T, per>::type*>(data + row * m.row + k * m.col);
      } else {
#pragma unroll
        for (int j = 0; j < per; ++j) {
          const long r = KC ? row : row + j, c = KC ? k + j : k;
          v[i][j] = r < rows && c < end ? data[r * m.row + c * m.col] : (T)0.f;
        }
      }
    }
  }

  // where element `at` (a multiple of `per`) of line `line` lies: bytes
  static __device__ __forceinline__ int place(int line, int at) {
    if (KC) return line * 64 + ((at / 8 ^ line / 4 % 4) * 16) + at % 8 * 2;
    return line * 256 + ((at / 16 ^ (line % 4 + line / 8 % 2 * 4)) * 32) + at % 16 * 2;
  }

  __device__ __forceinline__ void store(char* space) const {
#pragma unroll
    for (int i = 0; i < words; ++i) {
      const int w = threadIdx.x + 256 * i;
      const int line = KC ? w / (kStep / per) : w / (kTile / per);
      const int at = KC ? w % (kStep / per) * per : w % (kTile / per) * per;
      char* const to = space + place(line, at);
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uintx4*>(to) = __builtin_bit_cast(uintx4, v[i]);
      } else {
        float r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = v[i][j];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          *reinterpret_cast<uintx2*>(to + p * pieceBytes) = uintx2{leading(r[0], r[1]), leading(r[2], r[3])};
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] = withoutLeading(r[j]);
        }
      }
    }
  }

  // eight k of row `row` + lane % 16: k from 8 (lane / 16)
  static __device__ __forceinline__ uintx4 fragment(const char* space, int row) {
    const int lane = threadIdx.x % 64;
    if (KC) return *reinterpret_cast<const uintx4*>(space + place(row + lane % 16, lane / 16 * 8));
    // the transposing read: of sixteen lanes, lane l gives the address of four rows (l % 4) of k (l / 4) and gets four k of row l
    const int k = lane / 16 * 8 + lane % 16 / 4, at = row + lane % 4 * 4;
    uintx4 f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* const from = space + place(k + 4 * h, at);
      const shortx4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) shortx4*)const_cast<char*>(from));
      const uintx2 u = __builtin_bit_cast(uintx2, q);
      f[2 * h] = u[0];
      f[2 * h + 1] = u[1];
    }
    return f;
  }
};

// one result from its sum
template <class T>
__device__ __forceinline__ void finish(const Epilogue& e, long i, long j, float z) {
  z += lineOr(e.bias, j, 0.f);
  if (e.z.data) static_cast<T*>(e.z.data)[i * e.z.row + j * e.z.col] = (T)z;
  float v = activate(z, e.activation);
  if (e.residual.data) v += (float)static_cast<const T*>(e.residual.data)[i * e.residual.row + j * e.residual.col];
  static_cast<T*>(e.out.data)[i * e.out.row + j * e.out.col] = (T)v;
}

// A workgroup: 128 x 128 results over one range of k; a wave a quarter of them.  B's rows lie along the rows of the
// matrix instruction, so that a lane ends with four neighbouring results of one row.
template <class T, bool AK, bool BK>
__global__ __launch_bounds__(256) void product(ProductArgs g) {
  typedef typename Pieces<T>::type P;
  constexpr int PIECES = Pieces<T>::count, BYTES = kTile * kStep * 2;
  __shared__ __attribute__((aligned(16))) char space[2 * PIECES * BYTES];
  char *const sa = space, *const sb = space + PIECES * BYTES;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int wm = wave / 2 * 64, wn = wave % 2 * 64;
  const long m0 = (long)blockIdx.y * kTile, n0 = (long)blockIdx.x * kTile;
  const long first = blockIdx.z * g.range, end = min(first + g.range, g.K);

  floatx4 sum[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  Stage<T, AK> a;
  Stage<T, BK> b;
  a.load(g.a, m0, g.M, first, end);
  b.load(g.b, n0, g.N, first, end);
  for (long k = first; k < end; k += kStep) {
    __syncthreads();
    a.store(sa);
    b.store(sb);
    __syncthreads();
    a.load(g.a, m0, g.M, k + kStep, end);
    b.load(g.b, n0, g.N, k + kStep, end);
    uintx4 fb[PIECES][4];
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) fb[p][j] = Stage<T, BK>::fragment(sb + p * BYTES, wn + 16 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uintx4 fa[PIECES];
#pragma unroll
      for (int p = 0; p < PIECES; ++p) fa[p] = Stage<T, AK>::fragment(sa + p * BYTES, wm + 16 * i);
      // the products of pieces p and q, the smallest first
#pragma unroll
      for (int order = PIECES - 1; order >= 0; --order)
#pragma unroll
        for (int p = 0; p <= order; ++p)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[i][j] = multiply(fb[order - p][j], fa[p], sum[i][j], P());
    }
  }

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long m = m0 + wm + 16 * i + lane % 16;
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const long n = n0 + wn + 16 * j + lane / 16 * 4 + v;
        if (n >= g.N) continue;
        if (g.e.parts)
          g.e.parts[(blockIdx.z * g.M + m) * g.N + n] = sum[i][j][v];
        else
          finish<T>(g.e, m, n, sum[i][j][v]);
      }
  }
}

// Results from the sums of `ranges` ranges of k, in their order.
template <class T>
__global__ __launch_bounds__(256) void joinRanges(Epilogue e, long M, long N, int ranges) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * N) return;
  float z = 0.f;
  for (int r = 0; r < ranges; ++r) z += e.parts[(long)r * M * N + i];
  finish<T>(e, i / N, i % N, z);
}

// Results without any k.
template <class T>
__global__ __launch_bounds__(256) void noProduct(Epilogue e, long M, long N) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < M * N) finish<T>(e, i / N, i % N, 0.f);
}

constexpr int kBiasRows = 64;  // rows of dz that a workgroup sums

// dz = dy activation'(z), dense, and its columns' sums over kBiasRows rows each
template <class T>
__global__ __launch_bounds__(256) void preactivationGradient(Matrix dy, Matrix z, T* dz, float* parts, long M, long N, int activation) {
  const long n = (long)blockIdx.x * 256 + threadIdx.x, m0 = (long)blockIdx.y * kBiasRows;
  if (n >= N) return;
  float sum = 0.f;
  for (long m = m0; m < min(m0 + kBiasRows, M); ++m) {
    float v = (float)static_cast<const T*>(dy.data)[m * dy.row + n * dy.col];
    if (activation != FBFFT_ACTIVATION_NONE) v *= slope((float)static_cast<const T*>(z.data)[m * z.row + n * z.col], activation);
    if (dz) dz[m * N + n] = (T)v;
    sum += v;
  }
  if (parts) parts[blockIdx.y * N + n] = sum;
}

__global__ __launch_bounds__(256) void biasGradient(const float* parts, Line out, long N, long count) {
  const long n = (long)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  double sum = 0;
  for (long r = 0; r < count; ++r) sum += parts[r * N + n];
  storeAny(out.data, out.type, n * out.stride, (float)sum);
}

long ceilDivLong(long a, long b) { return (a + b - 1) / b; }
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// ranges of k: enough workgroups for two on each compute unit, at least 8 steps in a range
long rangesOf(long M, long N, long K) {
  const long tiles = ceilDivLong(M, kTile) * ceilDivLong(N, kTile);
  return std::max(1L, std::min({512 / std::max(tiles, 1L), K / (8 * kStep), 64L}));
}

size_t partsBytes(long M, long N, long K) {
  const long ranges = rangesOf(M, N, K);
  return ranges > 1 ? rounded((size_t)ranges * M * N * sizeof(float)) : 0;
}

template <class T>
int multiplyAll(const Matrix& a, const Matrix& b, long M, long N, long K, Epilogue e, float* parts, hipStream_t s) {
  const dim3 flat((unsigned)ceilDivLong(M * N, 256));
  if (K == 0) {
    noProduct<T><<<flat, 256, 0, s>>>(e, M, N);
    return launchStatus();
  }
  ProductArgs g{a, b, M, N, K, K, e};
  const long ranges = rangesOf(M, N, K);
  g.range = ceilDivLong(ceilDivLong(K, ranges), kStep) * kStep;
  if (ranges > 1) g.e.parts = parts;
  const dim3 grid((unsigned)ceilDivLong(N, kTile), (unsigned)ceilDivLong(M, kTile), (unsigned)ranges);
  const bool ak = a.col == 1 || a.row != 1, bk = b.col == 1 || b.row != 1;
  if (ak && bk)
    product<T, true, true><<<grid, 256, 0, s>>>(g);
  else if (ak)
    product<T, true, false><<<grid, 256, 0, s>>>(g);
  else if (bk)
    product<T, false, true><<<grid, 256, 0, s>>>(g);
  else
    product<T, false, false><<<grid, 256, 0, s>>>(g);
  if (ranges > 1) joinRanges<T><<<flat, 256, 0, s>>>(g.e, M, N, (int)ranges);
  return launchStatus();
}

template <class T>
int forward(const LinearProblem& p, hipStream_t s) {
  Epilogue e{p.y, p.residual, p.z, p.bias, p.activation, nullptr};
  return multiplyAll<T>(p.x, p.w, p.M, p.N, p.K, e, static_cast<float*>(p.workspace), s);
}

template <class T>
int backward(const LinearProblem& p, hipStream_t s) {
  char* space = static_cast<char*>(p.workspace);
  Matrix dz = p.dy;
  const long chunks = ceilDivLong(p.M, kBiasRows);
  float* const parts = reinterpret_cast<float*>(space);
  space += rounded((size_t)chunks * p.N * sizeof(float));
  const bool products = p.dx.data || p.dw.data, apart = products && p.activation != FBFFT_ACTIVATION_NONE;
  if (p.activation != FBFFT_ACTIVATION_NONE) {
    if (apart) dz = Matrix{space, p.N, 1};
    space += rounded((size_t)p.M * p.N * sizeof(T));
  }
  if (p.M > 0 && p.N > 0 && (apart || p.gradBias.data)) {
    const dim3 grid((unsigned)ceilDivLong(p.N, 256), (unsigned)chunks);
    preactivationGradient<T><<<grid, 256, 0, s>>>(p.dy, p.z, apart ? static_cast<T*>(dz.data) : nullptr,
                                                  p.gradBias.data ? parts : nullptr, p.M, p.N, p.activation);
  }
  if (p.gradBias.data && p.N > 0)
    biasGradient<<<dim3((unsigned)ceilDivLong(p.N, 256)), 256, 0, s>>>(parts, p.gradBias, p.N, p.M > 0 ? chunks : 0);
  int rc = launchStatus();
  if (rc == FBFFT_SUCCESS && p.dx.data && p.M > 0 && p.K > 0)
    rc = multiplyAll<T>(dz, Matrix{p.w.data, p.w.col, p.w.row}, p.M, p.K, p.N, Epilogue{p.dx, {}, {}, {}, 0, nullptr},
                        reinterpret_cast<float*>(space), s);
  if (rc == FBFFT_SUCCESS && p.dw.data && p.N > 0 && p.K > 0)
    rc = multiplyAll<T>(Matrix{dz.data, dz.col, dz.row}, Matrix{p.x.data, p.x.col, p.x.row}, p.N, p.K, p.M,
                        Epilogue{p.dw, {}, {}, {}, 0, nullptr}, reinterpret_cast<float*>(space), s);
  return rc;
}

}  // namespace

size_t linearWorkspaceBytes(int pass, long M, long K, long N, int type) {
  if (pass == 0) return partsBytes(M, N, K);
  return rounded((size_t)ceilDivLong(M, kBiasRows) * N * sizeof(float)) +
         rounded((size_t)M * N * (type == FBFFT_FLOAT32 ? 4 : 2)) + std::max(partsBytes(M, K, N), partsBytes(N, K, M));
}

int launchLinearForward(const LinearProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return forward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? forward<half16>(p, s) : forward<brain16>(p, s);
}

int launchLinearBackward(const LinearProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return backward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? backward<half16>(p, s) : backward<brain16>(p, s);
}

}  // namespace fbfft_amd
