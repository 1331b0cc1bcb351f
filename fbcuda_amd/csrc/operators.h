// Shared by the operators around convolution and linear layers: group and layer norm, products with an epilogue, dropout,
// orthogonalised updates, 4-bit rows.
#pragma once

#include "common.h"

namespace fbfft_amd {

typedef _Float16 half16;
typedef __bf16 brain16;

template <class T, int N>
struct Pack {
  // N neighbouring elements that start at any element
  typedef T __attribute__((ext_vector_type(N), aligned(sizeof(T)))) type;
};
template <class T>
struct Pack<T, 1> {
  typedef T type;
};

template <class T, int N>
__device__ __forceinline__ void loadPack(const T* p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = (float)*p;
  } else {
    const auto w = *reinterpret_cast<const typename Pack<T, N>::type*>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)w[j];
  }
}

template <class T, int N>
__device__ __forceinline__ void storePack(T* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    *p = (T)v[0];
  } else {
    typename Pack<T, N>::type w;
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = (T)v[j];
    *reinterpret_cast<typename Pack<T, N>::type*>(p) = w;
  }
}

// storePack, STREAM: of results that are not read again soon, past the caches.  (A choice at run time would not do: the
// compiler makes one plain store of the two.)
template <bool STREAM, class T, int N>
__device__ __forceinline__ void leavePack(T* p, const float (&v)[N]) {
  if constexpr (!STREAM || N == 1) {
    storePack<T, N>(p, v);
  } else {
    typename Pack<T, N>::type w;
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = (T)v[j];
    __builtin_nontemporal_store(w, reinterpret_cast<typename Pack<T, N>::type*>(p));
  }
}

// Results of 48 MiB and more are such (us, past the caches / through them: group norm of 16 x 32 x 256 x 256 bf16
// 43.9 / 48.9 forward and 74.5 / 78.8 backward, of 128 x 192 x 23 x 23 fp32 22.3 / 26.1; dropout of 67 MB 36.9 / 38.4);
// smaller ones are likely read from there next (32 x 192 x 23 x 23 fp32 13.5 / 9.7, dropout of 19 MB 11.0 / 10.7).
inline bool streams(double elements, int type) { return elements * (type == FBFFT_FLOAT32 ? 4 : 2) >= (double)(48 << 20); }

// Whether one launch holds so many workgroups: it counts its lanes in 32 bits.
inline bool launches(double blocks, int lanes) { return blocks * lanes < 4294967296.0; }

// element i of an array of a type that is known at run time
__device__ __forceinline__ float loadAny(const void* p, int type, long i) {
  if (type == FBFFT_FLOAT32) return static_cast<const float*>(p)[i];
  if (type == FBFFT_FLOAT16) return (float)static_cast<const half16*>(p)[i];
  return (float)static_cast<const brain16*>(p)[i];
}
__device__ __forceinline__ void storeAny(void* p, int type, long i, float v) {
  if (type == FBFFT_FLOAT32)
    static_cast<float*>(p)[i] = v;
  else if (type == FBFFT_FLOAT16)
    static_cast<half16*>(p)[i] = (half16)v;
  else
    static_cast<brain16*>(p)[i] = (brain16)v;
}

// Division of numbers below 2^31 by one that is fixed before the launch: one product and a shift.
struct Divisor {
  unsigned magic, shift, value;
};
inline Divisor divisorOf(long value) {
  Divisor d{0, 0, (unsigned)value};
  if (value < 2) return d;
  unsigned bits = 1;
  while ((1ul << bits) < (unsigned long)value) ++bits;
  d.magic = (unsigned)(((1ul << (31 + bits)) + value - 1) / value);  // at least 2^31: the value is over 2^(bits - 1)
  d.shift = bits - 1;
  return d;
}
__device__ __forceinline__ int quotient(int n, const Divisor& d) {
  return d.value < 2 ? n : (int)(__umulhi((unsigned)n, d.magic) >> d.shift);
}

// Sums over the 64 lanes of a wave, in every lane: four steps among 16 lanes by data-parallel moves, then rows and
// halves of the wave swapped against themselves.  Nothing goes through LDS.
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CONTROL, 0xF, 0xF, false));
}
template <int CONTROL>
__device__ __forceinline__ double moved(double v) {
  const long i = __builtin_bit_cast(long, v);
  const int low = (int)i, high = (int)(i >> 32);
  const unsigned l = __builtin_amdgcn_update_dpp(low, low, CONTROL, 0xF, 0xF, false);
  const unsigned h = __builtin_amdgcn_update_dpp(high, high, CONTROL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (unsigned long)h << 32 | l);
}
template <bool HALVES>
__device__ __forceinline__ float swappedSum(float v) {
  const unsigned i = __builtin_bit_cast(unsigned, v);
  const auto r = HALVES ? __builtin_amdgcn_permlane32_swap(i, i, false, false) : __builtin_amdgcn_permlane16_swap(i, i, false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
template <bool HALVES>
__device__ __forceinline__ double swappedSum(double v) {
  const unsigned long i = __builtin_bit_cast(unsigned long, v);
  const unsigned low = (unsigned)i, high = (unsigned)(i >> 32);
  const auto l = HALVES ? __builtin_amdgcn_permlane32_swap(low, low, false, false) : __builtin_amdgcn_permlane16_swap(low, low, false, false);
  const auto h = HALVES ? __builtin_amdgcn_permlane32_swap(high, high, false, false) : __builtin_amdgcn_permlane16_swap(high, high, false, false);
  return __builtin_bit_cast(double, (unsigned long)(unsigned)h[0] << 32 | (unsigned)l[0]) +
         __builtin_bit_cast(double, (unsigned long)(unsigned)h[1] << 32 | (unsigned)l[1]);
}
template <class S>
__device__ __forceinline__ S waveSum(S v) {
  v += moved<0xB1>(v);   // lanes 1 0 3 2
  v += moved<0x4E>(v);   // lanes 2 3 0 1
  v += moved<0x141>(v);  // eight lanes, reversed
  v += moved<0x140>(v);  // sixteen lanes, reversed
  return swappedSum<true>(swappedSum<false>(v));
}

// The same over the lanes whose numbers leave one remainder on division by `period`, a power of two up to 32.
template <class S>
__device__ __forceinline__ S waveSumEvery(S v, int period) {
  if (period <= 8) v += moved<0x128>(v);  // rotations among 16 lanes, by 8
  if (period <= 4) v += moved<0x124>(v);
  if (period <= 2) v += moved<0x122>(v);
  if (period <= 1) v += moved<0x121>(v);
  if (period <= 16) v = swappedSum<false>(v);
  return swappedSum<true>(v);
}

// The same over `lanes` neighbours, a power of two up to 64.
template <class S>
__device__ __forceinline__ S waveSumOf(S v, int lanes) {
  if (lanes > 1) v += moved<0xB1>(v);
  if (lanes > 2) v += moved<0x4E>(v);
  if (lanes > 4) v += moved<0x141>(v);
  if (lanes > 8) v += moved<0x140>(v);
  if (lanes > 16) v = swappedSum<false>(v);
  return lanes > 32 ? swappedSum<true>(v) : v;
}

// a vector of parameters, or nothing
struct Line {
  void* data;
  long stride;
  int type;
};
__device__ __forceinline__ float lineOr(const Line& l, long i, float otherwise) {
  return l.data ? loadAny(l.data, l.type, i * l.stride) : otherwise;
}

// exp(v) and 1 / v from the hardware's instructions.  The quotient is within about one unit in the last place; of exp the
// product with log2 e is rounded first, so that its relative error grows with v, to about (1 + |v|) 2^-24.
__device__ __forceinline__ float expOf(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float inverse(float v) { return __builtin_amdgcn_rcpf(v); }

// The normal distribution function and density.  The tail is exp(-a^2 / 2) times a polynomial in 1 / (1 + 0.3 a),
// fitted here to erfc's definition by least squares reweighted towards the least greatest relative error (the polynomial's
// 2e-7 up to a = 14; the exponential adds its own, so that the tail is within 7e-7 up to a = 3, 4e-6 up to 9 and 8e-6 up to
// 13).  In absolute terms the function is within 2.5e-7.  The library's erff takes two ways that a wave walks both: about
// 45 instructions, this 17.
__device__ __forceinline__ void normalOf(float z, float& cdf, float& density) {
  const float a = __builtin_fabsf(z), t = inverse(__builtin_fmaf(0.3f, a, 1.f));
  float q = 0.0356752947f;
  q = __builtin_fmaf(q, t, -0.15720516f);
  q = __builtin_fmaf(q, t, 0.20635691f);
  q = __builtin_fmaf(q, t, -0.0536866151f);
  q = __builtin_fmaf(q, t, 0.128563106f);
  q = __builtin_fmaf(q, t, 0.0999130756f);
  q = __builtin_fmaf(q, t, 0.120754018f);
  q = __builtin_fmaf(q, t, 0.119629294f);
  const float e = expOf(-0.5f * a * a), tail = e * (q * t);
  cdf = z < 0.f ? tail : 1.f - tail;
  density = 0.398942280f * e;
}

// z times the normal distribution function, where the density is not wanted: log2(cdf / (1 - cdf)) is z times a
// polynomial in z^2, fitted the same way up to |z| = 5.6 (and constant behind it) for the least greatest error of the
// result, 6.6e-8: half of what 32-bit arithmetic loses in z (1 + erf(z / sqrt 2)) / 2.  (An absolute error: of the results
// below -3, which go to 0, it is as much as half at -5.6 and more than all farther out.)
__device__ __forceinline__ float gelu(float z) {
  const float u = __builtin_fminf(z * z, 31.36f);
  float q = 5.2339035e-09f;
  q = __builtin_fmaf(q, u, -3.86017405e-07f);
  q = __builtin_fmaf(q, u, 1.14667555e-05f);
  q = __builtin_fmaf(q, u, -0.000159485367f);
  q = __builtin_fmaf(q, u, -9.52946357e-05f);
  q = __builtin_fmaf(q, u, 0.104838192f);
  q = __builtin_fmaf(q, u, 2.30220747f);
  return z * inverse(1.f + __builtin_amdgcn_exp2f(-z * q));
}

__device__ __forceinline__ float activate(float z, int activation) {
  // (a comparison that keeps NaN)
  if (activation == FBFFT_ACTIVATION_RELU) return z < 0.f ? 0.f : z;
  if (activation == FBFFT_ACTIVATION_SILU) return z * inverse(1.f + expOf(-z));
  if (activation == FBFFT_ACTIVATION_GELU) return gelu(z);
  return z;
}

template <int N>
__device__ __forceinline__ void activateAll(float (&v)[N], int activation) {
  if (activation == FBFFT_ACTIVATION_NONE) return;
  if (activation == FBFFT_ACTIVATION_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate(v[j], FBFFT_ACTIVATION_RELU);
  } else if (activation == FBFFT_ACTIVATION_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate(v[j], FBFFT_ACTIVATION_SILU);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate(v[j], FBFFT_ACTIVATION_GELU);
  }
}

__device__ __forceinline__ float slope(float z, int activation) {
  if (activation == FBFFT_ACTIVATION_RELU) return z > 0.f ? 1.f : 0.f;
  if (activation == FBFFT_ACTIVATION_SILU) {
    const float u = inverse(1.f + expOf(-z));
    return u * (1.f + z * (1.f - u));
  }
  if (activation == FBFFT_ACTIVATION_GELU) {
    float cdf, density;
    normalOf(z, cdf, density);
    return __builtin_fmaf(z, density, cdf);
  }
  return 1.f;
}

// g[j] times the slope at z[j]
template <int N>
__device__ __forceinline__ void slopeAll(const float (&z)[N], float (&g)[N], int activation) {
  if (activation == FBFFT_ACTIVATION_NONE) return;
  if (activation == FBFFT_ACTIVATION_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] *= slope(z[j], FBFFT_ACTIVATION_RELU);
  } else if (activation == FBFFT_ACTIVATION_SILU) {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] *= slope(z[j], FBFFT_ACTIVATION_SILU);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] *= slope(z[j], FBFFT_ACTIVATION_GELU);
  }
}

// ---- launchers (each returns an fbfft_error; shapes are checked by the caller) ----

// one [B][C][H][W] operand
struct Image {
  void* data;
  long b, c, h, w;  // strides in elements
};

struct NormProblem {
  Image x, y, g;  // forward: x, y.  backward: x, g (gradOutput), y (gradInput; data may be null)
  Line weight, bias, gradWeight, gradBias;
  float *mean, *rstd;
  long meanB, meanG, rstdB, rstdG;
  long B, C, G, H, W;
  int type, activation;
  float eps;
  void* workspace;
};
size_t normWorkspaceBytes(int pass, long B, long C, long P, long G);
int launchNormForward(const NormProblem& p, hipStream_t s);
int launchNormBackward(const NormProblem& p, hipStream_t s);

// one matrix operand: element (i, j) at i * row + j * col
struct Matrix {
  void* data;
  long row, col;
};

struct LinearProblem {
  Matrix x, w, residual, y, z, dy, dx, dw;  // forward: x, w, residual, y, z.  backward: x, w, dy, z, dx, dw
  Line bias, gradBias;
  long M, K, N;
  int type, activation;
  void* workspace;
};
size_t linearWorkspaceBytes(int pass, long M, long K, long N, int type);
int launchLinearForward(const LinearProblem& p, hipStream_t s);
int launchLinearBackward(const LinearProblem& p, hipStream_t s);

struct DropoutProblem {
  const void *x, *residual;
  void* y;
  long size[FBFFT_MAX_DIM], xs[FBFFT_MAX_DIM], rs[FBFFT_MAX_DIM], ys[FBFFT_MAX_DIM];  // right-aligned, size 1 in front
  long total;
  int type;
  unsigned threshold;
  unsigned long long seed, offset;
  const unsigned long long* step;
};
int launchDropout(const DropoutProblem& p, hipStream_t s);

// rows of a matrix: 2-d operands of layer norm
struct LayerNormProblem {
  Matrix x, y, g;  // forward: x, y.  backward: x, g (gradOutput), y (gradInput; data may be null)
  Line weight, bias, gradWeight, gradBias;
  float *mean, *rstd;
  long meanStride, rstdStride;
  long M, N;
  int type;
  float eps;
  void* workspace;
};
size_t layerNormWorkspaceBytes(int pass, long M, long N);
int launchLayerNormForward(const LayerNormProblem& p, hipStream_t s);
int launchLayerNormBackward(const LayerNormProblem& p, hipStream_t s);

struct OrthogonalProblem {
  Matrix x, y;  // of the first matrix
  long xBatch, yBatch;
  long batch, rows, cols;
  int type;
  const float* coefficients;
  int steps;
  float eps, scale;
  void* workspace;
};
size_t orthogonalWorkspaceBytes(long batch, long rows, long cols);
int launchOrthogonalize(const OrthogonalProblem& p, hipStream_t s);

// rows in the 4-bit format
struct Mx4 {
  unsigned char *codes, *scales;
  long codeStride, scaleStride;
};
int launchMx4Quantize(const Matrix& x, int type, long M, long K, const Mx4& to, hipStream_t s);
int launchMx4Dequantize(const Mx4& from, const Matrix& y, int type, long M, long K, hipStream_t s);

struct LinearMx4Problem {
  Matrix x;  // data null: xq instead
  Mx4 xq, w;
  Matrix residual, y;
  Line bias;
  long M, K, blocks, N;
  int type, activation;
  void* workspace;
};
size_t linearMx4WorkspaceBytes(long M, long blocks, long N);
int launchLinearMx4(const LinearMx4Problem& p, hipStream_t s);

}  // namespace fbfft_amd
