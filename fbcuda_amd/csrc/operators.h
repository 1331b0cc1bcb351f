// Shared by the operators around a convolution layer: group norm, products with an epilogue, dropout.
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

// a vector of parameters, or nothing
struct Line {
  void* data;
  long stride;
  int type;
};
__device__ __forceinline__ float lineOr(const Line& l, long i, float otherwise) {
  return l.data ? loadAny(l.data, l.type, i * l.stride) : otherwise;
}

// exp(-a) for a >= 0 and 1 / v from the hardware's instructions, each within about one unit in the last place
__device__ __forceinline__ float expOf(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ float inverse(float v) { return __builtin_amdgcn_rcpf(v); }

// The normal distribution function and density.  The tail is exp(-a^2 / 2) times a polynomial in 1 / (1 + 0.3 a),
// fitted here to erfc's definition by least squares reweighted towards the least greatest relative error (1.5e-7 up
// to a = 14).  The library's erff takes two ways that a wave walks both: about 45 instructions, this 17.
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

__device__ __forceinline__ float activate(float z, int activation) {
  // (a comparison that keeps NaN)
  if (activation == FBFFT_ACTIVATION_RELU) return z < 0.f ? 0.f : z;
  if (activation == FBFFT_ACTIVATION_SILU) return z * inverse(1.f + expOf(-z));
  if (activation == FBFFT_ACTIVATION_GELU) {
    float cdf, density;
    normalOf(z, cdf, density);
    return z * cdf;
  }
  return z;
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

// dense: every operand is one run of elements in logical order
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

}  // namespace fbfft_amd
