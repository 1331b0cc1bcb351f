// Layer norm of rows, and its gradients.
//
//   forward    y = (x - mean) rstd w + b,  rstd = 1 / sqrt(var + eps)
//   backward   xh = (x - mean) rstd, h = w g;  dx = rstd (h - mean(h) - xh mean(h xh)),  dw = sum g xh,  db = sum g over rows
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

constexpr int kLanes = 256;

// the sum over a workgroup, in every lane
__device__ __forceinline__ float groupSum(float v, float* space) {
  v = waveSum(v);
  if (threadIdx.x % 64 == 0) space[threadIdx.x / 64] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int q = 0; q < kLanes / 64; ++q) v += space[q];
  __syncthreads();
  return v;
}

template <class T>
__device__ __forceinline__ float valueOf(const Matrix& m, long i, long j) {
  return (float)static_cast<const T*>(m.data)[i * m.row + j * m.col];
}

// any strides: a workgroup to a row
template <class T>
__global__ __launch_bounds__(kLanes) void anyForward(LayerNormProblem p) {
  __shared__ float space[kLanes / 64];
  for (long i = blockIdx.x; i < p.M; i += gridDim.x) {
    float sum = 0.f;
    for (long j = threadIdx.x; j < p.N; j += kLanes) sum += valueOf<T>(p.x, i, j);
    const float mean = groupSum(sum, space) / p.N;
    sum = 0.f;
    for (long j = threadIdx.x; j < p.N; j += kLanes) {
      const float d = valueOf<T>(p.x, i, j) - mean;
      sum += d * d;
    }
    const float rstd = 1.f / __builtin_sqrtf(groupSum(sum, space) / p.N + p.eps);
    for (long j = threadIdx.x; j < p.N; j += kLanes)
      static_cast<T*>(p.y.data)[i * p.y.row + j * p.y.col] =
          (T)((valueOf<T>(p.x, i, j) - mean) * rstd * lineOr(p.weight, j, 1.f) + lineOr(p.bias, j, 0.f));
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[i * p.meanStride] = mean;
      if (p.rstd) p.rstd[i * p.rstdStride] = rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(kLanes) void anyBackward(LayerNormProblem p) {
  __shared__ float space[kLanes / 64];
  for (long i = blockIdx.x; i < p.M; i += gridDim.x) {
    const float mean = p.mean[i * p.meanStride], rstd = p.rstd[i * p.rstdStride];
    float s1 = 0.f, s2 = 0.f;
    for (long j = threadIdx.x; j < p.N; j += kLanes) {
      const float h = valueOf<T>(p.g, i, j) * lineOr(p.weight, j, 1.f);
      s1 += h;
      s2 += h * ((valueOf<T>(p.x, i, j) - mean) * rstd);
    }
    s1 = groupSum(s1, space) / p.N;
    s2 = groupSum(s2, space) / p.N;
    for (long j = threadIdx.x; j < p.N; j += kLanes) {
      const float h = valueOf<T>(p.g, i, j) * lineOr(p.weight, j, 1.f), xh = (valueOf<T>(p.x, i, j) - mean) * rstd;
      static_cast<T*>(p.y.data)[i * p.y.row + j * p.y.col] = (T)(rstd * (h - s1 - xh * s2));
    }
  }
}

// Columns' sums over a band of rows; parts: [band][2][N].
template <class T>
__global__ __launch_bounds__(kLanes) void anyParameters(LayerNormProblem p, float* parts, long bands) {
  const long across = (p.N + kLanes - 1) / kLanes, band = blockIdx.x / across, j = blockIdx.x % across * kLanes + threadIdx.x;
  if (j >= p.N) return;
  float w = 0.f, b = 0.f;
  for (long i = band; i < p.M; i += bands) {
    const float g = valueOf<T>(p.g, i, j);
    w += g * ((valueOf<T>(p.x, i, j) - p.mean[i * p.meanStride]) * p.rstd[i * p.rstdStride]);
    b += g;
  }
  parts[2 * band * p.N + j] = w;
  parts[(2 * band + 1) * p.N + j] = b;
}

__global__ __launch_bounds__(kLanes) void joinParameters(LayerNormProblem p, const float* parts, long bands) {
  const long j = (long)blockIdx.x * kLanes + threadIdx.x;
  if (j >= p.N) return;
  float w = 0.f, b = 0.f;
  for (long i = 0; i < bands; ++i) {
    w += parts[2 * i * p.N + j];
    b += parts[(2 * i + 1) * p.N + j];
  }
  if (p.gradWeight.data) storeAny(p.gradWeight.data, p.gradWeight.type, j * p.gradWeight.stride, w);
  if (p.gradBias.data) storeAny(p.gradBias.data, p.gradBias.type, j * p.gradBias.stride, b);
}

long bandsOf(long M) { return std::min(M, 256L); }

template <class T>
int forward(const LayerNormProblem& p, hipStream_t s) {
  anyForward<T><<<dim3((unsigned)std::min(p.M, 1L << 20)), kLanes, 0, s>>>(p);
  return launchStatus();
}

template <class T>
int backward(const LayerNormProblem& p, hipStream_t s) {
  float* const parts = static_cast<float*>(p.workspace);
  const long bands = p.M > 0 ? bandsOf(p.M) : 0, across = (p.N + kLanes - 1) / kLanes;
  // (before gradInput, which may be one of the operands)
  if (p.gradWeight.data || p.gradBias.data) {
    if (!launches((double)across * std::max(bands, 1L), kLanes)) return FBFFT_UNSUPPORTED_SIZE;
    if (bands > 0) anyParameters<T><<<dim3((unsigned)(across * bands)), kLanes, 0, s>>>(p, parts, bands);
    joinParameters<<<dim3((unsigned)across), kLanes, 0, s>>>(p, parts, bands);
  }
  if (p.y.data && p.M > 0) anyBackward<T><<<dim3((unsigned)std::min(p.M, 1L << 20)), kLanes, 0, s>>>(p);
  return launchStatus();
}

}  // namespace

size_t layerNormWorkspaceBytes(int pass, long M, long N) { return pass == 0 ? 0 : (size_t)bandsOf(M) * 2 * N * sizeof(float); }

int launchLayerNormForward(const LayerNormProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return forward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? forward<half16>(p, s) : forward<brain16>(p, s);
}

int launchLayerNormBackward(const LayerNormProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return backward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? backward<half16>(p, s) : backward<brain16>(p, s);
}

}  // namespace fbfft_amd
