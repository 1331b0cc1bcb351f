// Rows in microscaled 4-bit floating point, and their product with an epilogue.
//
//   a block of 32 neighbours v of a row:  e = floor(log2(max |v|)) - 2, at least -127;  code = nearest of v / 2^e, ties to even
//   product                               y = activation(sum_k x w + bias) + residual
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

// The scale's byte of a block from the bits of its largest magnitude (as numbers without sign, which order like the values),
// 255 for what is not finite.  floor(log2) is the exponent's field; numbers without one have their leading bit looked up, but
// all of them are below 2^-125 and take the least scale.
__device__ __forceinline__ int scaleOf(unsigned most) {
  const int exponent = (int)(most >> 23);
  return exponent == 255 ? 255 : max(exponent - 2, 0);
}

// Eight values, of a block with this scale, as codes.  (v / 2^e is a product with 2^-e, which is exact: a finite value's scale
// is at most 252, so 2^-e a normal number.)
__device__ __forceinline__ unsigned codesOf(const float (&v)[8], int scale) {
  if (scale == 255) return 0;
  const float by = __builtin_bit_cast(float, (unsigned)(254 - scale) << 23);
  unsigned codes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __builtin_fabsf(v[j] * by);
    // ties to the even code
    const unsigned code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
    codes |= (code | (__builtin_bit_cast(unsigned, v[j]) >> 28 & 8u)) << 4 * j;
  }
  return codes;
}

__device__ __forceinline__ float powerOf(int scale) {  // 2^(scale - 127); NaN for 255
  return __builtin_bit_cast(float, scale == 255 ? 0x7fc00000u : scale == 0 ? 0x00400000u : (unsigned)scale << 23);
}

__device__ __forceinline__ float valueOf(unsigned code, float scale) {
  const unsigned size = code & 7;
  const float v = size < 2 ? 0.5f * size : __builtin_bit_cast(float, (size + 252u) << 22);  // exponent of two bits from 127 - 1, a bit of mantissa
  return (code & 8 ? -v : v) * scale;
}

// the greatest over four neighbouring lanes
__device__ __forceinline__ unsigned mostOfFour(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xF, 0xF, false));
  return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xF, 0xF, false));
}

template <class T>
__device__ __forceinline__ void loadEight(const T* row, long stride, long k, long K, float (&v)[8]) {
  if (stride == 1 && k + 8 <= K) {
    loadPack<T, 8>(row + k, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? (float)row[(k + j) * stride] : 0.f;
  }
}

// Eight values to a lane, a block to four neighbouring lanes.
template <class T>
__global__ __launch_bounds__(256) void quantize(Matrix x, long M, long K, Mx4 to, Divisor perRow) {
  const int i = blockIdx.x * 256 + threadIdx.x, m = quotient(i, perRow), word = i - m * (int)perRow.value;
  if (m >= M) return;  // (a block's four lanes together)
  float v[8];
  loadEight(static_cast<const T*>(x.data) + m * x.row, x.col, 8l * word, K, v);
  unsigned most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
  const int scale = scaleOf(mostOfFour(most));
  *reinterpret_cast<unsigned*>(to.codes + m * to.codeStride + 4l * word) = codesOf(v, scale);
  if (word % 4 == 0) to.scales[m * to.scaleStride + word / 4] = (unsigned char)scale;
}

template <class T>
__global__ __launch_bounds__(256) void dequantize(Mx4 from, Matrix y, long M, long K, Divisor perRow) {
  const int i = blockIdx.x * 256 + threadIdx.x, m = quotient(i, perRow), word = i - m * (int)perRow.value;
  const long k = 8l * word;
  if (m >= M || k >= K) return;
  const unsigned codes = *reinterpret_cast<const unsigned*>(from.codes + m * from.codeStride + 4l * word);
  const float scale = powerOf(from.scales[m * from.scaleStride + word / 4]);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = valueOf(codes >> 4 * j & 15, scale);
  T* const to = static_cast<T*>(y.data) + m * y.row;
  if (y.col == 1 && k + 8 <= K) {
    storePack<T, 8>(to + k, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) to[(k + j) * y.col] = (T)v[j];
  }
}

// f(first row, rows, workgroups, words to a row) for as many rows at a time as a launch counts in 31 bits
template <class F>
int inLaunches(long M, long blocks, F f) {
  const long words = 4 * blocks, most = std::max(1l, (1l << 30) / words);
  for (long m = 0; m < M; m += most) {
    const long rows = std::min(most, M - m);
    f(m, rows, dim3((unsigned)((rows * words + 255) / 256)), divisorOf(words));
  }
  return launchStatus();
}

__device__ __forceinline__ floatx4 multiply(uintx4 a, int scaleA, uintx4 b, int scaleB, floatx4 c) {
  const intx8 x{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, y{(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, scaleA, 0, scaleB);
}

// A wave: 16 x 16 results, straight from memory to the matrix instructions: lane l has block l / 16 of four of row l % 16.
template <class T>
__global__ __launch_bounds__(256) void product(LinearMx4Problem p) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const long down = (p.M + 15) / 16, tile = blockIdx.x * 4l + wave, m0 = tile % down * 16, n0 = tile / down * 16;
  if (n0 >= p.N) return;
  const long xm = min(m0 + lane % 16, p.M - 1), wn = min(n0 + lane % 16, p.N - 1);
  const unsigned char *const x = p.xq.codes + xm * p.xq.codeStride, *const w = p.w.codes + wn * p.w.codeStride;
  const unsigned char *const xs = p.xq.scales + xm * p.xq.scaleStride, *const ws = p.w.scales + wn * p.w.scaleStride;
  floatx4 sum{0.f, 0.f, 0.f, 0.f};
  for (long b0 = 0; b0 < p.blocks; b0 += 4) {
    const long b = b0 + lane / 16;
    uintx4 a{}, c{};
    int sa = 0, sc = 0;  // (a block behind the last: zeros times 2^-127)
    if (b < p.blocks) {
      a = *reinterpret_cast<const uintx4*>(w + 16 * b), c = *reinterpret_cast<const uintx4*>(x + 16 * b);
      sa = ws[b], sc = xs[b];
    }
    sum = multiply(a, sa, c, sc, sum);
  }
  const long m = m0 + lane % 16;
  if (m >= p.M) return;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const long n = n0 + lane / 16 * 4 + v;
    if (n >= p.N) break;
    float z = activate(sum[v] + lineOr(p.bias, n, 0.f), p.activation);
    if (p.residual.data) z += (float)static_cast<const T*>(p.residual.data)[m * p.residual.row + n * p.residual.col];
    static_cast<T*>(p.y.data)[m * p.y.row + n * p.y.col] = (T)z;
  }
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

template <class T>
int run(LinearMx4Problem p, hipStream_t s) {
  const double groups = (double)((p.M + 15) / 16) * ((p.N + 15) / 16) / 4 + 1;
  if (!launches(groups, 256)) return FBFFT_UNSUPPORTED_SIZE;
  if (p.x.data && p.blocks > 0) {
    p.xq = Mx4{static_cast<unsigned char*>(p.workspace), static_cast<unsigned char*>(p.workspace) + rounded((size_t)p.M * p.blocks * 16),
               16 * p.blocks, p.blocks};
    const int rc = launchMx4Quantize(p.x, p.type, p.M, p.K, p.xq, s);
    if (rc != FBFFT_SUCCESS) return rc;
  }
  product<T><<<dim3((unsigned)groups), 256, 0, s>>>(p);
  return launchStatus();
}

}  // namespace

int launchMx4Quantize(const Matrix& x, int type, long M, long K, const Mx4& to, hipStream_t s) {
  return inLaunches(M, (K + 31) / 32, [&](long m, long rows, dim3 grid, Divisor perRow) {
    Matrix from = x;
    from.data = static_cast<char*>(x.data) + m * x.row * (type == FBFFT_FLOAT32 ? 4 : 2);
    const Mx4 q{to.codes + m * to.codeStride, to.scales + m * to.scaleStride, to.codeStride, to.scaleStride};
    if (type == FBFFT_FLOAT32)
      quantize<float><<<grid, 256, 0, s>>>(from, rows, K, q, perRow);
    else if (type == FBFFT_FLOAT16)
      quantize<half16><<<grid, 256, 0, s>>>(from, rows, K, q, perRow);
    else
      quantize<brain16><<<grid, 256, 0, s>>>(from, rows, K, q, perRow);
  });
}

int launchMx4Dequantize(const Mx4& from, const Matrix& y, int type, long M, long K, hipStream_t s) {
  return inLaunches(M, (K + 31) / 32, [&](long m, long rows, dim3 grid, Divisor perRow) {
    Matrix to = y;
    to.data = static_cast<char*>(y.data) + m * y.row * (type == FBFFT_FLOAT32 ? 4 : 2);
    const Mx4 q{from.codes + m * from.codeStride, from.scales + m * from.scaleStride, from.codeStride, from.scaleStride};
    if (type == FBFFT_FLOAT32)
      dequantize<float><<<grid, 256, 0, s>>>(q, to, rows, K, perRow);
    else if (type == FBFFT_FLOAT16)
      dequantize<half16><<<grid, 256, 0, s>>>(q, to, rows, K, perRow);
    else
      dequantize<brain16><<<grid, 256, 0, s>>>(q, to, rows, K, perRow);
  });
}

size_t linearMx4WorkspaceBytes(long M, long blocks, long) { return rounded((size_t)M * blocks * 16) + rounded((size_t)M * blocks); }

int launchLinearMx4(const LinearMx4Problem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return run<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? run<half16>(p, s) : run<brain16>(p, s);
}

}  // namespace fbfft_amd
