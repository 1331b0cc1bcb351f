// Layer norm of rows, and its gradients.
//
//   forward    y = (x - mean) rstd w + b,  rstd = 1 / sqrt(var + eps)
//   backward   xh = (x - mean) rstd, h = w g;  dx = rstd (h - mean(h) - xh mean(h xh)),  dw = sum g xh,  db = sum g over rows
//
// Memory bounds all of it: every operand is read once, rows stay in registers between their sums and their results.  (16384 x 2048
// bf16 forward 23.6 us, 5.7 TB/s; 8192 x 2048 bf16 backward 24.5, where 101 MB take 19 at the rate of a copy and the join of the
// columns' sums is a launch of 3 to 4; 67712 x 192 f32 backward 33.1, 156 MB 29.)  Few rows are a launch: 1 x 2048 4.1 us.
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

constexpr int kLanes = 256;

// the sum over a workgroup, in every lane
template <int LANES>
__device__ __forceinline__ float groupSum(float v, float* space) {
  v = waveSum(v);
  if (threadIdx.x % 64 == 0) space[threadIdx.x / 64] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int q = 0; q < LANES / 64; ++q) v += space[q];
  __syncthreads();
  return v;
}

template <class T>
__device__ __forceinline__ float valueOf(const Matrix& m, long i, long j) {
  return (float)static_cast<const T*>(m.data)[i * m.row + j * m.col];
}

// any strides and lengths: a workgroup to a row
template <class T, int LANES>
__global__ __launch_bounds__(LANES) void anyForward(LayerNormProblem p) {
  __shared__ float space[LANES / 64];
  for (long i = blockIdx.x; i < p.M; i += gridDim.x) {
    float sum = 0.f;
#pragma unroll 4
    for (long j = threadIdx.x; j < p.N; j += LANES) sum += valueOf<T>(p.x, i, j);
    const float mean = groupSum<LANES>(sum, space) / p.N;
    sum = 0.f;
#pragma unroll 4
    for (long j = threadIdx.x; j < p.N; j += LANES) {
      const float d = valueOf<T>(p.x, i, j) - mean;
      sum += d * d;
    }
    const float rstd = 1.f / __builtin_sqrtf(groupSum<LANES>(sum, space) / p.N + p.eps);
#pragma unroll 4
    for (long j = threadIdx.x; j < p.N; j += LANES)
      static_cast<T*>(p.y.data)[i * p.y.row + j * p.y.col] =
          (T)((valueOf<T>(p.x, i, j) - mean) * rstd * lineOr(p.weight, j, 1.f) + lineOr(p.bias, j, 0.f));
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[i * p.meanStride] = mean;
      if (p.rstd) p.rstd[i * p.rstdStride] = rstd;
    }
  }
}

template <class T, int LANES>
__global__ __launch_bounds__(LANES) void anyBackward(LayerNormProblem p) {
  __shared__ float space[LANES / 64];
  for (long i = blockIdx.x; i < p.M; i += gridDim.x) {
    const float mean = p.mean[i * p.meanStride], rstd = p.rstd[i * p.rstdStride];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
    for (long j = threadIdx.x; j < p.N; j += LANES) {
      const float h = valueOf<T>(p.g, i, j) * lineOr(p.weight, j, 1.f);
      s1 += h;
      s2 += h * ((valueOf<T>(p.x, i, j) - mean) * rstd);
    }
    s1 = groupSum<LANES>(s1, space) / p.N;
    s2 = groupSum<LANES>(s2, space) / p.N;
#pragma unroll 4
    for (long j = threadIdx.x; j < p.N; j += LANES) {
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

// ---- rows of neighbours that lanes hold in registers ----

// A row's words of VEC values, WORDS to a lane, LANES lanes to a row.
template <class T, int VEC, int LANES, int WORDS>
struct Row {
  typename Pack<T, VEC>::type v[WORDS];

  static __device__ __forceinline__ long at(int w) { return (long)(w * LANES + threadIdx.x % LANES) * VEC; }
  // SKIP: lanes behind a row's end pass by (of rows that reach all lanes that costs 2 %)
  template <bool SKIP>
  __device__ __forceinline__ void load(const Matrix& m, long i, long N) {
    const T* const from = static_cast<const T*>(m.data) + i * m.row;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const long j = at(w);
      if (j + VEC <= N) {
        v[w] = *reinterpret_cast<const typename Pack<T, VEC>::type*>(from + j);
      } else {
        if (SKIP) v[w] = typename Pack<T, VEC>::type{};
        if (!SKIP || j < N) {
#pragma unroll
          for (int q = 0; q < VEC; ++q) v[w][q] = j + q < N ? from[j + q] : (T)0.f;
        }
      }
    }
  }
};

template <bool STREAM, class T, int VEC>
__device__ __forceinline__ void leaveWord(T* to, long j, long N, const float (&v)[VEC]) {
  if (j + VEC <= N) {
    leavePack<STREAM, T, VEC>(to + j, v);
  } else {
#pragma unroll
    for (int q = 0; q < VEC; ++q)
      if (j + q < N) to[j + q] = (T)v[q];
  }
}

// VEC parameters from j
template <int VEC>
__device__ __forceinline__ void loadLine(const Line& l, long j, long N, float otherwise, float (&v)[VEC]) {
  if (l.data && l.type == FBFFT_FLOAT32 && l.stride == 1 && j + VEC <= N) {
    loadPack<float, VEC>(static_cast<const float*>(l.data) + j, v);
  } else {
#pragma unroll
    for (int q = 0; q < VEC; ++q) v[q] = j + q < N ? lineOr(l, j + q, otherwise) : 0.f;
  }
}

// The same number, from which the compiler computes nothing in front of a loop: the addresses of all words' parameters, of three
// types, take hundreds of registers there.
__device__ __forceinline__ long hidden(long j) {
  asm volatile("" : "+v"(j));
  return j;
}

// The sums of two values over the lanes of a row, in every lane.  Rows of more than a wave meet in LDS, `turn` in turn two parts
// of it, so that one barrier is enough.
template <int LANES, int THREADS>
__device__ __forceinline__ void rowSums(float& s1, float& s2, float (*space)[THREADS / 64][2], int turn) {
  if constexpr (LANES <= 64) {
    s1 = waveSumOf(s1, LANES);
    s2 = waveSumOf(s2, LANES);
  } else {
    s1 = waveSum(s1);
    s2 = waveSum(s2);
    if (threadIdx.x % 64 == 0) space[turn][threadIdx.x / 64][0] = s1, space[turn][threadIdx.x / 64][1] = s2;
    __syncthreads();
    s1 = s2 = 0.f;
    const int first = threadIdx.x / LANES * (LANES / 64);
#pragma unroll
    for (int q = 0; q < LANES / 64; ++q) {
      s1 += space[turn][first + q][0];
      s2 += space[turn][first + q][1];
    }
  }
}

// A workgroup takes THREADS / LANES rows at a time, the next ones on their way where registers allow it.  The variance is that of the values in registers
// around their mean: nothing cancels.
template <class T, int VEC, int LANES, int WORDS, int THREADS, bool STREAM>
__global__ __launch_bounds__(THREADS) void rowsForward(LayerNormProblem p) {
  constexpr int GROUPS = THREADS / LANES;
  constexpr bool HOLDS = WORDS * VEC <= 16;  // the parameters, and the next row
  __shared__ float space[2][THREADS / 64][2];
  typedef Row<T, VEC, LANES, WORDS> R;
  float weight[HOLDS ? WORDS : 1][VEC], bias[HOLDS ? WORDS : 1][VEC];
  if constexpr (HOLDS) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      loadLine(p.weight, R::at(w), p.N, 1.f, weight[w]);
      loadLine(p.bias, R::at(w), p.N, 0.f, bias[w]);
    }
  }
  const long step = (long)gridDim.x * GROUPS, first = (long)blockIdx.x * GROUPS + threadIdx.x / LANES;
  const float each = 1.f / (float)p.N;
  R next;
  if constexpr (HOLDS) next.template load<false>(p.x, min(first, p.M - 1), p.N);
  for (long i = first; i - threadIdx.x / LANES < p.M; i += step) {  // (as often for all rows of a workgroup)
    R x;
    if constexpr (HOLDS) {
      x = next;
      if (i - threadIdx.x / LANES + step < p.M) next.template load<false>(p.x, min(i + step, p.M - 1), p.N);
    } else {
      x.template load<false>(p.x, min(i, p.M - 1), p.N);
    }
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int w = 0; w < WORDS; ++w)
#pragma unroll
      for (int q = 0; q < VEC; ++q) sum += (float)x.v[w][q];
    rowSums<LANES, THREADS>(sum, none, space, 0);
    const float mean = sum * each;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < WORDS; ++w)
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        const float d = R::at(w) + q < p.N ? (float)x.v[w][q] - mean : 0.f;
        sum = __builtin_fmaf(d, d, sum);
      }
    rowSums<LANES, THREADS>(sum, none, space, 1);
    const float rstd = 1.f / __builtin_sqrtf(sum * each + p.eps);
    if (i < p.M) {
      T* const to = static_cast<T*>(p.y.data) + i * p.y.row;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        float y[VEC];
        if constexpr (!HOLDS) {
          const long j = hidden(R::at(w));
          loadLine(p.weight, j, p.N, 1.f, weight[0]);
          loadLine(p.bias, j, p.N, 0.f, bias[0]);
        }
        constexpr int last = HOLDS ? WORDS - 1 : 0;
#pragma unroll
        for (int q = 0; q < VEC; ++q) y[q] = __builtin_fmaf(((float)x.v[w][q] - mean) * rstd, weight[min(w, last)][q], bias[min(w, last)][q]);
        leaveWord<STREAM, T, VEC>(to, R::at(w), p.N, y);
      }
      if (threadIdx.x % LANES == 0) {
        if (p.mean) p.mean[i * p.meanStride] = mean;
        if (p.rstd) p.rstd[i * p.rstdStride] = rstd;
      }
    }
  }
}

// The columns' sums of all rows over LANES words of a row (up to 64) from word `first`, by a workgroup of 1024 lanes, to the
// gradients.
template <class T, int VEC, int LANES>
__device__ __forceinline__ void leaveColumns(const LayerNormProblem& p, long first, float* space) {
  constexpr int GROUPS = 1024 / LANES, COLUMNS = LANES * VEC;
  typedef Row<T, VEC, LANES, 1> R;
  const long from = first * VEC;
  Matrix x = p.x, g = p.g;
  x.data = static_cast<T*>(x.data) + from, g.data = static_cast<T*>(g.data) + from;
  float sumW[VEC] = {}, sumB[VEC] = {};
#pragma unroll 4
  for (long i = threadIdx.x / LANES; i < p.M; i += GROUPS) {
    R a, b;
    a.template load<true>(x, i, p.N - from);
    b.template load<true>(g, i, p.N - from);
    const float mean = p.mean[i * p.meanStride], rstd = p.rstd[i * p.rstdStride];
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const float dy = (float)b.v[0][q];
      sumB[q] += dy;
      sumW[q] = __builtin_fmaf(dy, ((float)a.v[0][q] - mean) * rstd, sumW[q]);
    }
  }
  // over a wave's rows, then over the waves
#pragma unroll
  for (int q = 0; q < VEC; ++q)
#pragma unroll
    for (int far = LANES; far < 64; far *= 2) {
      sumW[q] += __shfl_xor(sumW[q], far);
      sumB[q] += __shfl_xor(sumB[q], far);
    }
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    __syncthreads();
    if (lane < LANES) {
#pragma unroll
      for (int q = 0; q < VEC; ++q) space[wave * COLUMNS + lane * VEC + q] = part ? sumB[q] : sumW[q];
    }
    __syncthreads();
    const Line& to = part ? p.gradBias : p.gradWeight;
    for (int j = threadIdx.x; j < COLUMNS && from + j < p.N; j += 1024) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 16; ++w) v += space[w * COLUMNS + j];
      if (to.data) storeAny(to.data, to.type, (from + j) * to.stride, v);
    }
  }
}

// Rows as above, 1024 lanes to a workgroup; SUMS: the columns' sums of its rows stay in registers, meet in LDS and go to parts
// [workgroup][2][N], where parts is not null.  Else the workgroups behind the first `groups` take the columns' sums of all rows, 64
// words of a row each.
template <class T, int VEC, int LANES, int WORDS, bool STREAM, bool SUMS>
__global__ __launch_bounds__(1024) void rowsBackward(LayerNormProblem p, float* parts, int groups) {
  constexpr int GROUPS = 1024 / LANES, ACROSS = LANES < 64 ? LANES : 64;
  if constexpr (!SUMS) {
    __shared__ __attribute__((aligned(16))) float columns[16 * ACROSS * VEC];
    if ((int)blockIdx.x >= groups) {
      leaveColumns<T, VEC, ACROSS>(p, (long)((int)blockIdx.x - groups) * ACROSS, columns);
      return;
    }
  }
  __shared__ float space[2][16][2];
  typedef Row<T, VEC, LANES, WORDS> R;
  constexpr bool HOLDS = WORDS == 1;  // the parameters, and the next row
  float weight[VEC], sumW[WORDS][VEC] = {}, sumB[WORDS][VEC] = {};
  if constexpr (HOLDS) loadLine(p.weight, R::at(0), p.N, 1.f, weight);
  const long step = (long)groups * GROUPS, first = (long)blockIdx.x * GROUPS + threadIdx.x / LANES;
  const float each = 1.f / (float)p.N;
  R nextX, nextG;
  float nextMean, nextRstd;
  auto load = [&](long row) __attribute__((always_inline)) {
    const long i = min(row, p.M - 1);
    nextX.template load<true>(p.x, i, p.N);
    nextG.template load<true>(p.g, i, p.N);
    nextMean = p.mean[i * p.meanStride], nextRstd = p.rstd[i * p.rstdStride];
  };
  if constexpr (HOLDS) load(first);
  int turn = 0;
  for (long i = first; i - threadIdx.x / LANES < p.M; i += step) {
    if constexpr (!HOLDS) load(i);
    const R x = nextX, g = nextG;
    const float mean = nextMean, rstd = nextRstd;
    if (HOLDS && i - threadIdx.x / LANES + step < p.M) load(i + step);
    float s1 = 0.f, s2 = 0.f;
    if (i < p.M) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        if constexpr (!HOLDS) {
          loadLine(p.weight, hidden(R::at(w)), p.N, 1.f, weight);
        }
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const float dy = (float)g.v[w][q], xh = ((float)x.v[w][q] - mean) * rstd, h = dy * weight[q];
          s1 += h;
          s2 = __builtin_fmaf(h, xh, s2);
          if constexpr (SUMS) {
            sumB[w][q] += dy;
            sumW[w][q] = __builtin_fmaf(dy, xh, sumW[w][q]);
          }
        }
      }
    }
    if (p.y.data) {
      rowSums<LANES, 1024>(s1, s2, space, turn);
      s1 *= each;
      s2 *= each;
      if (i < p.M) {
        T* const to = static_cast<T*>(p.y.data) + i * p.y.row;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          float d[VEC];
          if constexpr (!HOLDS) {
            loadLine(p.weight, hidden(R::at(w)), p.N, 1.f, weight);
          }
#pragma unroll
          for (int q = 0; q < VEC; ++q) {
            const float xh = ((float)x.v[w][q] - mean) * rstd, h = (float)g.v[w][q] * weight[q];
            d[q] = rstd * (h - s1 - xh * s2);
          }
          leaveWord<STREAM, T, VEC>(to, R::at(w), p.N, d);
        }
      }
    }
    turn ^= 1;
  }
  if (!SUMS || !parts) return;
  float* const to = parts + (long)blockIdx.x * 2 * p.N;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      leaveWord<false, float, VEC>(to, R::at(w), p.N, sumW[w]);
      leaveWord<false, float, VEC>(to + p.N, R::at(w), p.N, sumB[w]);
    }
  } else {
    static_assert(WORDS == 1, "a word to a lane");
    __shared__ __attribute__((aligned(16))) float sums[GROUPS][LANES * VEC];
    const int group = threadIdx.x / LANES, column = threadIdx.x % LANES * VEC;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < VEC; ++q) sums[group][column + q] = part ? sumB[0][q] : sumW[0][q];
      __syncthreads();
      for (int j = threadIdx.x; j < LANES * VEC && j < p.N; j += 1024) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) v += sums[q][j];
        to[part * p.N + j] = v;
      }
    }
  }
}

// Columns' sums by themselves: a wave takes 64 words of a row and every kColumnWaves-th row of a band.  A band's go to parts
// [band][2][N], those of one band to the gradients.
constexpr int kColumnWaves = 8;

template <class T, int VEC>
__global__ __launch_bounds__(kColumnWaves * 64) void columnSums(LayerNormProblem p, float* parts, long rows) {
  __shared__ __attribute__((aligned(16))) float sums[kColumnWaves][64 * VEC];
  typedef Row<T, VEC, 64, 1> R;
  const long from = (long)blockIdx.x * 64 * VEC, first = (long)blockIdx.y * rows, end = min(first + rows, p.M);
  Matrix x = p.x, g = p.g;
  x.data = static_cast<T*>(x.data) + from, g.data = static_cast<T*>(g.data) + from;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  float sumW[VEC] = {}, sumB[VEC] = {};
#pragma unroll 4
  for (long i = first + wave; i < end; i += kColumnWaves) {
    R a, b;
    a.template load<true>(x, i, p.N - from);
    b.template load<true>(g, i, p.N - from);
    const float mean = p.mean[i * p.meanStride], rstd = p.rstd[i * p.rstdStride];
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
      const float dy = (float)b.v[0][q];
      sumB[q] += dy;
      sumW[q] = __builtin_fmaf(dy, ((float)a.v[0][q] - mean) * rstd, sumW[q]);
    }
  }
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < VEC; ++q) sums[wave][threadIdx.x % 64 * VEC + q] = part ? sumB[q] : sumW[q];
    __syncthreads();
    const Line& to = part ? p.gradBias : p.gradWeight;
    for (int j = threadIdx.x; j < 64 * VEC && from + j < p.N; j += kColumnWaves * 64) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kColumnWaves; ++q) v += sums[q][j];
      if (parts)
        parts[(2 * blockIdx.y + part) * p.N + from + j] = v;
      else if (to.data)
        storeAny(to.data, to.type, (from + j) * to.stride, v);
    }
  }
}

// Parts' sums, joined in their order, from column `first` of [2][N] on: 1024 / SLICES columns to a workgroup, SLICES lanes to each.
template <int SLICES>
__global__ __launch_bounds__(1024) void joinRows(LayerNormProblem p, const float* parts, int bands, long first) {
  constexpr int COLUMNS = 1024 / SLICES;
  __shared__ float sums[SLICES][COLUMNS + 1];
  const int column = threadIdx.x % COLUMNS, slice = threadIdx.x / COLUMNS;
  const long j = first + (long)blockIdx.x * COLUMNS + column;
  float sum = 0.f;
  if (j < 2 * p.N)
#pragma unroll 8
    for (int r = slice; r < bands; r += SLICES) sum += parts[r * 2 * p.N + j];
  sums[slice][column] = sum;
  __syncthreads();
  if (slice > 0 || j >= 2 * p.N) return;
  sum = 0.f;
#pragma unroll
  for (int q = 0; q < SLICES; ++q) sum += sums[q][column];
  const Line& to = j < p.N ? p.gradWeight : p.gradBias;
  if (to.data) storeAny(to.data, to.type, (j < p.N ? j : j - p.N) * to.stride, sum);
}

// Parts of the rows whose columns' sums are joined: a workgroup to a compute unit, or two to narrow rows, whose sums are little (us
// of 256, 512 and 1024 parts: 8192 x 2048 bf16 25.0, 29.4, 37.6; 4096 x 8192 bf16 43.5, 54.4, 71.8; 67712 x 192 f32 33.6, 29.1,
// 30.8).
long bandsOf(long M, long N) { return std::min(M, N < 256 ? 512L : 256L); }

// Whether a workgroup may sum its columns of all rows in twelve turns: then workgroups for rows and for columns run in one launch,
// without parts (128 x 2048 bf16 5.6 us, 7.6 in two launches; 128 x 8192 6.0, 10.4; 256 x 512 7.2 either way).
bool together(long M, long N, size_t valueBytes) {
  const long words = (N * (long)valueBytes + 15) / 16;
  long lanes = 8;
  while (lanes < 64 && lanes < words) lanes *= 2;
  return N <= 16384 && M * lanes <= 12288;
}

// Whether the columns are summed by themselves, from x and g once more: for few long rows, of which each workgroup has one or two
// and leaves sums as long as they are (us apart and together: 256 x 16384 bf16 13.9, 28.3; 64 x 8192 f16 10.0, 11.0; 512 x 8192 bf16
// 13.6, 18.1; 1024 x 8192 bf16 21.2, 20.5; 512 x 4096 f32 13.1, 14.5; 64 x 8192 f32 11.6, 10.6).
// Rows that no workgroup holds are read again as it is.
bool apart(long M, long N, size_t valueBytes) {
  return N > 16384 || (std::min(M, 256L) * N >= 3 << 18 && M * (long)valueBytes <= 1024);
}

// Lanes to a row: as many as it has words, so that a lane holds one; wider rows take more words to a lane.
template <class T, bool STREAM>
bool launchRows(const LayerNormProblem& p, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const long words = (p.N + V - 1) / V;
  const unsigned most = 2048;
  auto grid = [&](int groups) { return dim3((unsigned)std::min((p.M + groups - 1) / groups, (long)most)); };
#define FBFFT_ROWS(LANES, WORDS, THREADS)                                                        \
  if (words <= LANES * WORDS) {                                                                  \
    rowsForward<T, V, LANES, WORDS, THREADS, STREAM><<<grid(THREADS / LANES), THREADS, 0, s>>>(p); \
    return true;                                                                                 \
  }
  FBFFT_ROWS(4, 1, 256)
  FBFFT_ROWS(8, 1, 256)
  FBFFT_ROWS(16, 1, 256)
  FBFFT_ROWS(32, 1, 256)
  FBFFT_ROWS(64, 1, 256)
  if (p.M >= 4 * computeUnits()) {
    FBFFT_ROWS(64, 2, 256)
    FBFFT_ROWS(64, 4, 256)
  }
  if constexpr (!STREAM) {  // (so few rows of that length are no 48 MiB)
    FBFFT_ROWS(256, 1, 256)
  }
  FBFFT_ROWS(256, 2, 256)
  FBFFT_ROWS(256, 4, 256)
  FBFFT_ROWS(1024, 2, 1024)
  FBFFT_ROWS(1024, 4, 1024)
  if constexpr (sizeof(T) == 4) {
    FBFFT_ROWS(1024, 8, 1024)
  }
#undef FBFFT_ROWS
  return false;
}

// Workgroups for the rows of a backward pass, with the columns' sums of each in parts (SUMS), or without them and `columns` more for
// the columns of all rows; 0 where no registers hold a row.  rows: whether gradInput is wanted, or not yet.
template <class T, bool STREAM, bool SUMS>
int launchRowsBack(const LayerNormProblem& p, float* parts, bool rows, bool columns, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const long words = (p.N + V - 1) / V, bands = bandsOf(p.M, p.N);
#define FBFFT_ROWS(LANES, WORDS)                                                                                   \
  if (words <= LANES * WORDS) {                                                                                    \
    const long most = (p.M + 1024 / LANES - 1) / (1024 / LANES), groups = rows ? std::min(SUMS ? bands : 65536L, most) : 0; \
    const long more = columns ? (words + 63) / 64 : 0;                                                             \
    rowsBackward<T, V, LANES, WORDS, STREAM, SUMS><<<dim3((unsigned)(groups + more)), 1024, 0, s>>>(p, parts, (int)groups); \
    return (int)(groups + more);                                                                                   \
  }
  FBFFT_ROWS(8, 1)
  FBFFT_ROWS(16, 1)
  FBFFT_ROWS(32, 1)
  FBFFT_ROWS(64, 1)
  FBFFT_ROWS(128, 1)
  FBFFT_ROWS(256, 1)
  FBFFT_ROWS(512, 1)
  FBFFT_ROWS(1024, 1)
  FBFFT_ROWS(1024, 2)
  if constexpr (sizeof(T) == 4) {
    FBFFT_ROWS(1024, 4)
  }
#undef FBFFT_ROWS
  return 0;
}

// Lanes of the workgroups that read a row several times: 1024 for few long rows (gradients of 1 x 20000 bf16 15.5 us and by 256
// lanes 36.4, 1024 x 20000 80.6 and 91.2, 2048 x 20000 150 and 138).
bool manyLanes(const LayerNormProblem& p) { return p.N > 4096 && p.M <= 4 * computeUnits(); }

template <class T>
int forward(const LayerNormProblem& p, hipStream_t s) {
  if (p.x.col == 1 && p.y.col == 1 && (streams((double)p.M * p.N, p.type) ? launchRows<T, true>(p, s) : launchRows<T, false>(p, s)))
    return launchStatus();
  const dim3 grid((unsigned)std::min(p.M, 1L << 20));
  if (!manyLanes(p))
    anyForward<T, 256><<<grid, 256, 0, s>>>(p);
  else
    anyForward<T, 1024><<<grid, 1024, 0, s>>>(p);
  return launchStatus();
}

constexpr long kMostLanes = 0xffffffffl;  // of a launch

void launchJoinRows(const LayerNormProblem& p, const float* parts, int bands, hipStream_t s) {
  const long columns = bands > 32 ? 16 : 128, most = kMostLanes / 1024;  // of a workgroup; workgroups of a launch
  for (long first = 0; first < 2 * p.N; first += most * columns) {
    const dim3 grid((unsigned)std::min(most, (2 * p.N - first + columns - 1) / columns));
    if (bands > 32)
      joinRows<64><<<grid, 1024, 0, s>>>(p, parts, bands, first);
    else
      joinRows<8><<<grid, 1024, 0, s>>>(p, parts, bands, first);
  }
}

template <class T>
int backward(const LayerNormProblem& p, hipStream_t s) {
  float* const parts = static_cast<float*>(p.workspace);
  bool sums = p.gradWeight.data || p.gradBias.data;
  const long across = (p.N + kLanes - 1) / kLanes;
  long bands = p.M > 0 ? std::min(bandsOf(p.M, p.N), kMostLanes / kLanes / across) : 0;  // (of the element by element way)
  bool done = p.M == 0;
  if (!done && p.x.col == 1 && p.g.col == 1 && (!p.y.data || p.y.col == 1)) {
    if (sums && together(p.M, p.N, sizeof(T))) {
      const bool over = p.y.data && (p.y.data == p.x.data || p.y.data == p.g.data);  // (what the columns read)
      launchRowsBack<T, false, false>(p, nullptr, p.y.data && !over, true, s);
      if (over) launchRowsBack<T, false, false>(p, nullptr, true, false, s);
      return launchStatus();
    }
    constexpr int V = 16 / sizeof(T);
    const long over = (p.N + 64 * V - 1) / (64 * V);
    // (one band where there are 512 workgroups across; of float32 rows of 2^31 - 256 values and more they do not fit a launch)
    if (sums && apart(p.M, p.N, sizeof(T)) && launches((double)over, kColumnWaves * 64)) {
      const long most = std::min(std::max(512 / over, 1L), (p.M + 31) / 32);
      const long rows = (p.M + most - 1) / most;
      bands = (p.M + rows - 1) / rows;
      columnSums<T, V><<<dim3((unsigned)over, (unsigned)bands), kColumnWaves * 64, 0, s>>>(p, bands > 1 ? parts : nullptr, rows);
      if (bands > 1) launchJoinRows(p, parts, (int)bands, s);
      if (!p.y.data) return launchStatus();
      sums = false;
      done = launchRowsBack<T, false, false>(p, nullptr, true, false, s) > 0;
    } else {
      float* const to = sums ? parts : nullptr;
      const int groups = streams((double)p.M * p.N, p.type) ? launchRowsBack<T, true, true>(p, to, true, false, s)
                                                            : launchRowsBack<T, false, true>(p, to, true, false, s);
      if (groups) done = true, bands = groups;
    }
  }
  // (before gradInput, which may be one of the operands)
  if (!done && sums) anyParameters<T><<<dim3((unsigned)(across * bands)), kLanes, 0, s>>>(p, parts, bands);
  const dim3 grid((unsigned)std::min(p.M, 1L << 20));
  if (!done && p.y.data && !manyLanes(p))
    anyBackward<T, 256><<<grid, 256, 0, s>>>(p);
  else if (!done && p.y.data)
    anyBackward<T, 1024><<<grid, 1024, 0, s>>>(p);
  if (sums) launchJoinRows(p, parts, (int)bands, s);
  return launchStatus();
}

}  // namespace

size_t layerNormWorkspaceBytes(int pass, long M, long N) { return pass == 0 ? 0 : (size_t)bandsOf(M, N) * 2 * N * sizeof(float); }

int launchLayerNormForward(const LayerNormProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return forward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? forward<half16>(p, s) : forward<brain16>(p, s);
}

int launchLayerNormBackward(const LayerNormProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return backward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? backward<half16>(p, s) : backward<brain16>(p, s);
}

}  // namespace fbfft_amd
