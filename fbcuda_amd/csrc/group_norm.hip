// Group norm with an activation, forward and backward.
//
//   mean, var over the n = D P values of a group (D channels, P = H W pixels), xh = (x - mean) / sqrt(var + eps)
//   y  = activation(xh w[c] + b[c])
//   dz = dy activation'(xh w[c] + b[c]);  db[c] = sum dz,  dw[c] = sum dz xh
//   dx = rstd (w dz - sum(w dz) / n - xh sum(w dz xh) / n)
//
// Sums of x and x^2 are taken in 64 bits: their difference then keeps a variance that is far smaller than the
// squared mean, without a second pass over the data.
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

struct NormArgs {
  Image x, y, g;
  Line weight, bias, gradWeight, gradBias;
  float *mean, *rstd;
  long meanB, meanG, rstdB, rstdG;
  long B, C, G, D, H, W, P;
  int activation;
  float eps;
  float2* channels;  // backward: sums of dz and dz xh of each image and channel
};

__device__ __forceinline__ long pixelAt(const Image& i, long p, long W) { return p / W * i.h + p % W * i.w; }

// The activation's argument, from a product and a sum that are rounded apart: both passes, and a program that writes
// the formula down, then agree on which values a ReLU lets through.
__device__ __forceinline__ float affine(float xh, float w, float shift) {
#pragma clang fp contract(off)
  return xh * w + shift;
}

// the sum over the workgroup's 256 lanes, in every lane
__device__ __forceinline__ double groupSum(double v, double* space) {
#pragma unroll
  for (int k = 32; k > 0; k /= 2) v += __shfl_xor(v, k);
  __syncthreads();
  if (threadIdx.x % 64 == 0) space[threadIdx.x / 64] = v;
  __syncthreads();
  return space[0] + space[1] + space[2] + space[3];
}

// A workgroup takes one group of one image, whatever the strides.
template <class T>
__global__ __launch_bounds__(256) void normAny(NormArgs a) {
  __shared__ double space[4];
  const long b = blockIdx.x / a.G, g = blockIdx.x % a.G, n = a.D * a.P;
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + g * a.D * a.x.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + g * a.D * a.y.c;
  double s1 = 0, s2 = 0;
  for (long e = threadIdx.x; e < n; e += 256) {
    const double v = (float)x[e / a.P * a.x.c + pixelAt(a.x, e % a.P, a.W)];
    s1 += v;
    s2 += v * v;
  }
  s1 = groupSum(s1, space);
  s2 = groupSum(s2, space);
  const double centre = s1 / n, variance = fmax(s2 / n - centre * centre, 0.0);
  const float mean = (float)centre, rstd = (float)(1.0 / sqrt(variance + a.eps));
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[b * a.meanB + g * a.meanG] = mean;
    if (a.rstd) a.rstd[b * a.rstdB + g * a.rstdG] = rstd;
  }
  for (long e = threadIdx.x; e < n; e += 256) {
    const long c = e / a.P, p = e % a.P;
    const float v = (float)x[c * a.x.c + pixelAt(a.x, p, a.W)];
    const float w = lineOr(a.weight, g * a.D + c, 1.f), shift = lineOr(a.bias, g * a.D + c, 0.f);
    y[c * a.y.c + pixelAt(a.y, p, a.W)] = (T)activate(affine((v - mean) * rstd, w, shift), a.activation);
  }
}

// A workgroup sums one channel of one image.
template <class T>
__global__ __launch_bounds__(256) void normSumsAny(NormArgs a) {
  __shared__ double space[4];
  const long b = blockIdx.x / a.C, c = blockIdx.x % a.C, group = c / a.D;
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  const float w = lineOr(a.weight, c, 1.f), shift = lineOr(a.bias, c, 0.f);
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + c * a.x.c;
  const T* const g = static_cast<const T*>(a.g.data) + b * a.g.b + c * a.g.c;
  double s1 = 0, s2 = 0;
  for (long p = threadIdx.x; p < a.P; p += 256) {
    const float xh = ((float)x[pixelAt(a.x, p, a.W)] - mean) * rstd;
    const float dz = (float)g[pixelAt(a.g, p, a.W)] * slope(affine(xh, w, shift), a.activation);
    s1 += dz;
    s2 += (double)dz * xh;
  }
  s1 = groupSum(s1, space);
  s2 = groupSum(s2, space);
  if (threadIdx.x == 0) a.channels[b * a.C + c] = float2{(float)s1, (float)s2};
}

// A workgroup takes one group of one image.
template <class T>
__global__ __launch_bounds__(256) void normGradAny(NormArgs a) {
  const long b = blockIdx.x / a.G, group = blockIdx.x % a.G, n = a.D * a.P;
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  double s1 = 0, s2 = 0;
  for (long c = group * a.D; c < (group + 1) * a.D; ++c) {
    const float2 s = a.channels[b * a.C + c];
    const float w = lineOr(a.weight, c, 1.f);
    s1 += (double)s.x * w;
    s2 += (double)s.y * w;
  }
  const float m1 = (float)(s1 / n), m2 = (float)(s2 / n);
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + group * a.D * a.x.c;
  const T* const g = static_cast<const T*>(a.g.data) + b * a.g.b + group * a.D * a.g.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + group * a.D * a.y.c;
  for (long e = threadIdx.x; e < n; e += 256) {
    const long c = e / a.P, p = e % a.P;
    const float w = lineOr(a.weight, group * a.D + c, 1.f), shift = lineOr(a.bias, group * a.D + c, 0.f);
    const float xh = ((float)x[c * a.x.c + pixelAt(a.x, p, a.W)] - mean) * rstd;
    const float dz = (float)g[c * a.g.c + pixelAt(a.g, p, a.W)] * slope(affine(xh, w, shift), a.activation);
    y[c * a.y.c + pixelAt(a.y, p, a.W)] = (T)(rstd * (dz * w - m1 - xh * m2));
  }
}

// The gradients of weight and bias: the sums over the images, in their order.
__global__ __launch_bounds__(64) void normParameters(NormArgs a) {
  const long c = (long)blockIdx.x * 64 + threadIdx.x;
  if (c >= a.C) return;
  double s1 = 0, s2 = 0;
  for (long b = 0; b < a.B; ++b) {
    const float2 s = a.channels[b * a.C + c];
    s1 += s.x;
    s2 += s.y;
  }
  if (a.gradBias.data) storeAny(a.gradBias.data, a.gradBias.type, c * a.gradBias.stride, (float)s1);
  if (a.gradWeight.data) storeAny(a.gradWeight.data, a.gradWeight.type, c * a.gradWeight.stride, (float)s2);
}

NormArgs argsOf(const NormProblem& p) {
  NormArgs a{};
  a.x = p.x, a.y = p.y, a.g = p.g;
  a.weight = p.weight, a.bias = p.bias, a.gradWeight = p.gradWeight, a.gradBias = p.gradBias;
  a.mean = p.mean, a.rstd = p.rstd;
  a.meanB = p.meanB, a.meanG = p.meanG, a.rstdB = p.rstdB, a.rstdG = p.rstdG;
  a.B = p.B, a.C = p.C, a.G = p.G, a.D = p.C / p.G, a.H = p.H, a.W = p.W, a.P = p.H * p.W;
  a.activation = p.activation, a.eps = p.eps;
  a.channels = static_cast<float2*>(p.workspace);
  return a;
}

template <class T>
int forward(const NormProblem& p, hipStream_t s) {
  const NormArgs a = argsOf(p);
  normAny<T><<<dim3((unsigned)(a.B * a.G)), 256, 0, s>>>(a);
  return launchStatus();
}

template <class T>
int backward(const NormProblem& p, hipStream_t s) {
  NormArgs a = argsOf(p);
  if (a.P == 0) a.B = 0;  // no pixels: the gradients are sums of nothing
  if (a.B > 0) normSumsAny<T><<<dim3((unsigned)(a.B * a.C)), 256, 0, s>>>(a);
  if (a.B > 0 && a.y.data) normGradAny<T><<<dim3((unsigned)(a.B * a.G)), 256, 0, s>>>(a);
  if (a.gradWeight.data || a.gradBias.data)
    normParameters<<<dim3((unsigned)((a.C + 63) / 64)), 64, 0, s>>>(a);
  return launchStatus();
}

}  // namespace

size_t normWorkspaceBytes(int pass, long B, long C, long P, long G) {
  return pass == 0 ? 0 : (size_t)(B * C) * sizeof(float2);
}

int launchNormForward(const NormProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return forward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? forward<half16>(p, s) : forward<brain16>(p, s);
}

int launchNormBackward(const NormProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return backward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? backward<half16>(p, s) : backward<brain16>(p, s);
}

}  // namespace fbfft_amd
