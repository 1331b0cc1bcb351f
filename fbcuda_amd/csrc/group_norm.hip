// Group norm with an activation, forward and backward.
//
//   mean, var over the n = D P values of a group (D channels, P = H W pixels), xh = (x - mean) / sqrt(var + eps)
//   y  = activation(xh w[c] + b[c])
//   dz = dy activation'(xh w[c] + b[c]);  db[c] = sum dz,  dw[c] = sum dz xh
//   dx = rstd (w dz - sum(w dz) / n - xh sum(w dz xh) / n)
//
// Sums of x and x^2 are taken in 64 bits: their difference then keeps a variance that is far smaller than the
// squared mean, without a second pass over the data (64-bit additions run at the rate of 32-bit ones here).
//
// Three sets of kernels:
//   Last    a lane holds a few neighbouring channels and walks over pixels (channels contiguous, or any strides)
//   Planes  a lane walks over the contiguous values of a group (planes without gaps)
//   Any     a group, or 64 channels, to a workgroup, element by element: groups wider than Last's lanes
// The first two hold what a workgroup reads in registers where that suffices for a whole group, so that memory sees
// one read and one write in one launch; else a first launch leaves sums of pieces of a group, and a second one joins
// them and reads again, backwards, what the last-level cache still holds.
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
  Divisor byW, byP, byD, byLanes, byPieces, byCuts, byBands;
  double share;  // 1 / (D P)
  int activation;
  float eps;
  // channels-last plan: channels of a workgroup, rows of lanes and lanes of a row, pixels of a piece; planes: values of one
  int band, rows, rowsSecond, lanes, pieces, cuts;
  long piece, cut;  // of the first launch's pieces, and of the second one's
  double2* sums;     // forward: of x and x^2, [image][group][piece]
  float2* groups;    // backward: sums of w dz and w dz xh, [image][group][piece]
  float2* channels;  // backward: sums of dz and dz xh, [image][piece][channel]
};

__device__ __forceinline__ long pixelAt(const NormArgs& a, const Image& i, int p) {
  // (rows without gaps: the second term is 0; a branch would cost more)
  return (long)p * i.w + (long)quotient(p, a.byW) * (i.h - a.W * i.w);
}

// The activation's argument, from a product and a sum that are rounded apart: both passes, and a program that writes
// the formula down, then agree on which values a ReLU lets through.
__device__ __forceinline__ float affine(float xh, float w, float shift) {
#pragma clang fp contract(off)
  return xh * w + shift;
}

struct Moments {
  float mean, rstd;
};
__device__ __forceinline__ Moments momentsOf(const NormArgs& a, double s1, double s2) {
  const double centre = s1 * a.share, variance = s2 * a.share - centre * centre;
  // (not a maximum: a group that holds NaN keeps it)
  return {(float)centre, 1.f / sqrtf((float)((variance < 0.0 ? 0.0 : variance) + a.eps))};
}

// the sum over a workgroup of NT lanes, in every lane
template <int NT, class S>
__device__ __forceinline__ S teamSum(S v, S* space) {
  v = waveSum(v);
  if (NT == 64) return v;
  __syncthreads();
  if (threadIdx.x % 64 == 0) space[threadIdx.x / 64] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) v += space[k];
  return v;
}

// A workgroup's lanes shared out among its groups, up to NT of them: neighbours, as many to each, a power of two up to a
// wave, as there are and as have a term to add, so that all groups are summed at once (a wave to one group after the
// other: 4 x 64 x 199 x 199 f16, 32 groups of 64 pieces, 30 us instead of 21.6; 80 x 32 x 107 x 106, 60 and 45).
struct Share {
  int lanes, group, place;
};
template <int NT>
__device__ __forceinline__ Share shareOf(int groups, int terms) {
  int lanes = 64;
  while (lanes > 1 && (lanes * groups > NT || lanes / 2 >= terms)) lanes /= 2;
  return {lanes, (int)threadIdx.x / lanes, (int)threadIdx.x & (lanes - 1)};
}

// The gradients of weight and bias: the sums over images and pieces.  256 lanes: eight channels, 32 lanes to each.
constexpr int kParameters = 8;
__device__ __forceinline__ void parameterGradients(const NormArgs& a, int block, float2 (&part)[32][kParameters]) {
  const int lane = threadIdx.x % kParameters, slice = threadIdx.x / kParameters;
  const long c = (long)block * kParameters + lane, rows = a.B * a.pieces;
  float s1 = 0, s2 = 0;
  if (c < a.C)
#pragma unroll 8
    for (long r = slice; r < rows; r += 32) {
      const float2 s = a.channels[r * a.C + c];
      s1 += s.x;
      s2 += s.y;
    }
  part[slice][lane] = float2{s1, s2};
  __syncthreads();
  if (slice > 0 || c >= a.C) return;
  s1 = s2 = 0;
  for (int r = 0; r < 32; ++r) {
    s1 += part[r][lane].x;
    s2 += part[r][lane].y;
  }
  if (a.gradBias.data) storeAny(a.gradBias.data, a.gradBias.type, c * a.gradBias.stride, s1);
  if (a.gradWeight.data) storeAny(a.gradWeight.data, a.gradWeight.type, c * a.gradWeight.stride, s2);
}

__global__ __launch_bounds__(256) void normParameters(NormArgs a) {
  __shared__ float2 part[32][kParameters];
  parameterGradients(a, blockIdx.x, part);
}

// ---- Last ----

constexpr int kBand = 1024;   // channels of a workgroup at most
constexpr int kFirst = 512;   // lanes of the first of two launches: few pieces, which every workgroup of the second one joins
constexpr int kAhead = 4, kAheadTwo = 2;  // pixels of one and of each of two operands that a lane has on their way

template <int NT, int VEC, class S>
struct Columns {
  S lane[NT * VEC], part[NT];
};

// A workgroup's band of whole groups: lane t holds VEC channels from VEC (t % lanes) of every rows-th pixel.  Adds what
// each lane has of its channels over the rows of lanes; sums[i] is then that of lane column i (several values of a lane
// side by side).  Where rows of lanes divide a wave its rows meet in registers first (64 sums by one lane from LDS
// took 7 us of the smallest call's 14), and what waits in LDS is summed in two stages.
// `step` of a lane's channels, 1 or a power of two that divides VEC, are added up before that: those of one group.
template <int NT, int VEC, class S>
__device__ __forceinline__ void joinRows(const NormArgs& a, int lanes, int column, int r, int step, S (&v)[VEC],
                                         Columns<NT, VEC, S>& space, S* sums) {
#pragma unroll
  for (int d = 1; d < VEC; d *= 2)
    if (step > d)
#pragma unroll
      for (int j = 0; j < VEC; j += 2 * d) v[j] += v[j + d];
  const int t = threadIdx.x, shift = 31 - __builtin_clz(step), slots = VEC >> shift, columns = lanes * slots;
  const bool divides = a.lanes <= 32 && (a.lanes & (a.lanes - 1)) == 0;
  const int rows = divides ? NT / 64 : a.rows, row = divides ? t / 64 : r;
  if (divides)
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if ((j & (step - 1)) == 0) v[j] = waveSumEvery(v[j], a.lanes);
  __syncthreads();
  if (column < lanes && (divides ? t % 64 < a.lanes : r < a.rows))
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if ((j & (step - 1)) == 0) space.lane[row * columns + column * slots + (j >> shift)] = v[j];
  __syncthreads();
  if (rows <= 16 || columns > NT / 2) {
    for (int i = t; i < columns; i += NT) {
      S sum = 0;
#pragma unroll 4
      for (int k = 0; k < rows; ++k) sum += space.lane[k * columns + i];
      sums[i] = sum;
    }
    return;
  }
  const int parts = min(NT / columns, 16), part = t / columns, i = t - part * columns;
  if (part < parts) {
    S sum = 0;
#pragma unroll 4
    for (int k = part; k < rows; k += parts) sum += space.lane[k * columns + i];
    space.part[t] = sum;
  }
  __syncthreads();
  if (t < columns) {
    S sum = 0;
#pragma unroll 4
    for (int k = 0; k < parts; ++k) sum += space.part[k * columns + t];
    sums[t] = sum;
  }
}

// What a workgroup of Last, and a lane of it, work on.
struct Band {
  int b, piece, first, firstGroup;  // image, piece, channels and groups in front of the band
  int channels, lanes, groups;      // of the band; lanes: of a row, with channels
  int column, r;                    // of this lane: its place in a row of lanes, and the row
  int rows, p, end;                 // rows of lanes; first pixel, and the one behind the last
  bool live;
};
// (SECOND: of the second launch, of 256 lanes)
template <int VEC, bool SECOND = false>
__device__ __forceinline__ Band bandOf(const NormArgs& a, int index) {
  Band w;
  const int row = quotient(index, SECOND ? a.byCuts : a.byPieces);
  w.piece = index - row * (SECOND ? a.cuts : a.pieces);
  w.p = w.piece * (int)(SECOND ? a.cut : a.piece);
  w.end = (int)min(w.p + (SECOND ? a.cut : a.piece), a.P);
  w.b = quotient(row, a.byBands);
  w.first = (row - w.b * (int)a.byBands.value) * a.band;
  w.channels = min(a.band, (int)a.C - w.first);
  w.lanes = w.channels / VEC;
  w.firstGroup = quotient(w.first, a.byD);
  w.groups = quotient(w.channels, a.byD);
  w.r = quotient(threadIdx.x, a.byLanes);
  w.column = threadIdx.x - w.r * a.lanes;
  w.rows = SECOND ? a.rowsSecond : a.rows;
  w.live = w.r < w.rows && w.column < w.lanes;
  return w;
}
template <class T>
__device__ __forceinline__ T* laneOf(const NormArgs& a, const Image& i, const Band& band, int vec) {
  return static_cast<T*>(i.data) + band.b * i.b + (long)(band.first + band.column * vec) * i.c;
}

// weight and bias of the band's channels, into LDS
__device__ __forceinline__ void bandParameters(const NormArgs& a, const Band& band, float2* to, int threads) {
  for (int c = threadIdx.x; c < band.channels; c += threads)
    to[c] = float2{lineOr(a.weight, band.first + c, 1.f), lineOr(a.bias, band.first + c, 0.f)};
}

template <int VEC>
struct Channel {
  float mean[VEC], rstd[VEC], w[VEC], shift[VEC];

  __device__ __forceinline__ void load(const NormArgs& a, const Band& band, const Moments* stats, const float2* params) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = min(band.column * VEC + j, band.channels - 1);
      const Moments m = stats[quotient(c, a.byD)];
      const float2 p = params[c];
      mean[j] = m.mean;
      rstd[j] = m.rstd;
      w[j] = p.x;
      shift[j] = p.y;
    }
  }
  // The activation's arguments in the place of x.  (One multiply-add of x by rstd w would round at the size of mean rstd w,
  // which in a group of nearly constant values is far above the result: 0.5 at 30000.)
  __device__ __forceinline__ void apply(float (&x)[VEC]) const {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = affine((x[j] - mean[j]) * rstd[j], w[j], shift[j]);
  }
  // x is replaced by the normalised values, z by the activation's arguments
  __device__ __forceinline__ void arguments(float (&x)[VEC], float (&z)[VEC]) const {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[j] = (x[j] - mean[j]) * rstd[j];
      z[j] = affine(x[j], w[j], shift[j]);
    }
  }
};

// the statistics of the band's groups from sums over their columns; space holds 64-bit sums
template <int NT, int VEC>
__device__ __forceinline__ void joinMoments(const NormArgs& a, const Band& band, double (&s1)[VEC], double (&s2)[VEC],
                                            Columns<NT, VEC, double>& space, double* sums, Moments* stats, bool raw) {
  const int D = (int)a.D;
  // a lane's channels of one group, where groups and words start together
  const int step = D % VEC == 0 ? VEC : VEC % D == 0 ? D : 1, wide = D / step;
  const Share share = shareOf<NT>(band.groups, wide);
  auto one = [&](double(&s)[VEC]) __attribute__((always_inline)) {
    joinRows<NT, VEC>(a, band.lanes, band.column, band.r, step, s, space, sums);
    __syncthreads();
    double v = 0;
    if (share.group < band.groups)
#pragma unroll 4
      for (int i = share.place; i < wide; i += share.lanes) v += sums[share.group * wide + i];
    return waveSumOf(v, share.lanes);
  };
  const double first = one(s1), second = one(s2);
  const int g = share.group;
  if (g < band.groups && share.place == 0) {
    const long group = band.firstGroup + g;
    if (raw) {
      a.sums[(band.b * a.G + group) * a.pieces + band.piece] = double2{first, second};
    } else {
      const Moments m = momentsOf(a, first, second);
      stats[g] = m;
      if (a.mean) a.mean[band.b * a.meanB + group * a.meanG] = m.mean;
      if (a.rstd) a.rstd[band.b * a.rstdB + group * a.rstdG] = m.rstd;
    }
  }
  __syncthreads();
}

template <int VEC>
__device__ __forceinline__ void moments(const float (&v)[VEC], double (&s1)[VEC], double (&s2)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const double x = v[j];
    s1[j] += x;
    s2[j] = __builtin_fma(x, x, s2[j]);
  }
}

// N elements of one word
template <int VEC, class R>
__device__ __forceinline__ void unpack(const R raw, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = (float)raw;
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)raw[j];
  }
}

// Workgroups are dealt out to the eight XCDs in turn; those of one XCD take neighbouring work, so that lines that two
// bands of an image share are read into one L2.
__device__ __forceinline__ int nearWork(int total) {
  const int per = (total + 7) / 8;
  const int index = (int)blockIdx.x % 8 * per + (int)blockIdx.x / 8;
  return (int)blockIdx.x / 8 < per && index < total ? index : -1;
}

// All pixels of a band in registers: one read, one write.  One image of 64 x 27 x 27 bf16: 7.0 us, most of it the launch,
// one trip to memory and the joins in LDS.
template <class T, int VEC, int NT, int ITEMS, bool STREAM>
__global__ __launch_bounds__(NT) void lastForward(NormArgs a, int total) {
  __shared__ Columns<NT, VEC, double> space;
  __shared__ double sums[kBand];
  __shared__ Moments stats[NT];
  __shared__ float2 params[kBand];
  const int index = nearWork(total);
  if (index < 0) return;
  const Band band = bandOf<VEC>(a, index);
  const T* const x = laneOf<const T>(a, a.x, band, VEC);
  T* const y = laneOf<T>(a, a.y, band, VEC);
  const int P = (int)a.P;
  typename Pack<T, VEC>::type raw[ITEMS];
  if (band.live)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int p = band.r + i * a.rows;
      if (p < P) raw[i] = *reinterpret_cast<const typename Pack<T, VEC>::type*>(x + pixelAt(a, a.x, p));
    }
  bandParameters(a, band, params, NT);
  double s1[VEC] = {}, s2[VEC] = {};
  if (band.live)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (band.r + i * a.rows < P) {
        float v[VEC];
        unpack(raw[i], v);
        moments(v, s1, s2);
      }
  joinMoments<NT, VEC>(a, band, s1, s2, space, sums, stats, false);
  if (!band.live) return;
  Channel<VEC> ch;
  ch.load(a, band, stats, params);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int p = band.r + i * a.rows;
    if (p >= P) break;
    float v[VEC];
    unpack(raw[i], v);
    ch.apply(v);
    activateAll(v, a.activation);
    leavePack<STREAM, T, VEC>(y + pixelAt(a, a.y, p), v);
  }
}

// Where a lane walks over the pixels of a piece: AHEAD of them are on their way from memory, requested before what has
// to be known to use them, and in the loop before the ones in hand are used.
template <class T, int VEC, int AHEAD>
struct Walk {
  typedef typename Pack<T, VEC>::type Word;
  const T* from;
  int p, end, rows;
  Word coming[AHEAD], now[AHEAD];

  __device__ __forceinline__ void request(const NormArgs& a, const Image& i) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) coming[k] = *reinterpret_cast<const Word*>(from + pixelAt(a, i, min(p + k * rows, end - 1)));
  }
  __device__ __forceinline__ Walk(const NormArgs& a, const Image& i, const Band& band)
      : from(laneOf<const T>(a, i, band, VEC)), p(band.p + band.r), end(band.end), rows(band.rows) {
    if (band.live && p < end) request(a, i);
  }
  __device__ __forceinline__ void next(const NormArgs& a, const Image& i) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) now[k] = coming[k];
    p += AHEAD * rows;
    if (p < end) request(a, i);
  }
};

// The sums of a piece of each group.  16 x 32 x 256 x 256 bf16: 18-19 us for 67 MB, 3.6 TB/s; bound by memory and by the
// start of one round of workgroups.
template <class T, int VEC>
__global__ __launch_bounds__(kFirst) void lastSums(NormArgs a) {
  __shared__ Columns<kFirst, VEC, double> space;
  __shared__ double sums[kBand];
  const Band band = bandOf<VEC>(a, blockIdx.x);
  Walk<T, VEC, kAhead> x(a, a.x, band);
  double s1[VEC] = {}, s2[VEC] = {};
  if (band.live)
    for (int p = x.p; p < x.end; p += kAhead * x.rows) {
      x.next(a, a.x);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (p + k * x.rows < x.end) {
          float v[VEC];
          unpack(x.now[k], v);
          moments(v, s1, s2);
        }
    }
  joinMoments<kFirst, VEC>(a, band, s1, s2, space, sums, nullptr, true);
}

// 16 x 32 x 256 x 256 bf16, GELU: 28 us for 134 MB, 4.8 TB/s (half of it still in the last-level cache; one multiply-add a value
// in place of affine(): 26).
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void lastApply(NormArgs a) {
  __shared__ Moments stats[256];
  __shared__ float2 params[kBand];
  const Band band = bandOf<VEC, true>(a, gridDim.x - 1 - blockIdx.x);
  Walk<T, VEC, kAhead> x(a, a.x, band);
  bandParameters(a, band, params, 256);
  const Share share = shareOf<256>(band.groups, a.pieces);
  const long group = band.firstGroup + share.group;
  double s1 = 0, s2 = 0;
  if (share.group < band.groups)
#pragma unroll 4
    for (int i = share.place; i < a.pieces; i += share.lanes) {
      const double2 s = a.sums[(band.b * a.G + group) * a.pieces + i];
      s1 += s.x;
      s2 += s.y;
    }
  s1 = waveSumOf(s1, share.lanes);
  s2 = waveSumOf(s2, share.lanes);
  if (share.group < band.groups && share.place == 0) {
    const Moments m = momentsOf(a, s1, s2);
    stats[share.group] = m;
    if (band.piece == 0 && a.mean) a.mean[band.b * a.meanB + group * a.meanG] = m.mean;
    if (band.piece == 0 && a.rstd) a.rstd[band.b * a.rstdB + group * a.rstdG] = m.rstd;
  }
  __syncthreads();
  if (!band.live) return;
  Channel<VEC> ch;
  ch.load(a, band, stats, params);
  T* const y = laneOf<T>(a, a.y, band, VEC);
  for (int p = x.p; p < x.end; p += kAhead * x.rows) {
    x.next(a, a.x);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (p + k * x.rows < x.end) {
        float v[VEC];
        unpack(x.now[k], v);
        ch.apply(v);
        activateAll(v, a.activation);
        leavePack<STREAM, T, VEC>(y + pixelAt(a, a.y, p + k * x.rows), v);
      }
  }
}

// the statistics that the forward pass kept
__device__ __forceinline__ void keptMoments(const NormArgs& a, const Band& band, Moments* stats, int threads) {
  for (int g = threadIdx.x; g < band.groups; g += threads) {
    const long group = band.firstGroup + g;
    stats[g] = Moments{a.mean[band.b * a.meanB + group * a.meanG], a.rstd[band.b * a.rstdB + group * a.rstdG]};
  }
  __syncthreads();
}

// Sums of dz and dz xh per channel of the band, kept for the gradients of weight and bias; then those of w dz and
// w dz xh per group: done(group of the band, sum, sum) in one lane.
template <int NT, int VEC, class F>
__device__ __forceinline__ void joinGradients(const NormArgs& a, const Band& band, float (&s1)[VEC], float (&s2)[VEC],
                                              Columns<NT, VEC, float>& space, float (&sums)[2][kBand], const float2* params, F done) {
  joinRows<NT, VEC>(a, band.lanes, band.column, band.r, 1, s1, space, sums[0]);
  joinRows<NT, VEC>(a, band.lanes, band.column, band.r, 1, s2, space, sums[1]);
  // (a lane reads what it has written)
  for (int c = threadIdx.x; c < band.channels; c += NT) {
    const float2 s{sums[0][c], sums[1][c]};
    a.channels[((long)band.b * a.pieces + band.piece) * a.C + band.first + c] = s;
    const float w = params[c].x;
    sums[0][c] = s.x * w;
    sums[1][c] = s.y * w;
  }
  __syncthreads();
  const int D = (int)a.D;
  const Share share = shareOf<NT>(band.groups, D);
  float m1 = 0, m2 = 0;
  if (share.group < band.groups)
#pragma unroll 4
    for (int i = share.place; i < D; i += share.lanes) {
      m1 += sums[0][share.group * D + i];
      m2 += sums[1][share.group * D + i];
    }
  m1 = waveSumOf(m1, share.lanes);
  m2 = waveSumOf(m2, share.lanes);
  if (share.group < band.groups && share.place == 0) done(share.group, m1, m2);
}

// dx in the place of dz, from xh
template <int VEC>
__device__ __forceinline__ void inputGradient(const Channel<VEC>& ch, const float (&m1)[VEC], const float (&m2)[VEC],
                                              const float (&xh)[VEC], float (&dz)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) dz[j] = ch.rstd[j] * (dz[j] * ch.w[j] - m1[j] - xh[j] * m2[j]);
}

// All pixels of a band of input and gradient in registers: two reads, one write.  128 x 192 x 23 x 23 bf16, groups of six:
// 32-34 us for 78 MB, 2.4 TB/s.  164 registers leave three workgroups to a compute unit; the 1024 of this shape are four to each,
// so a round of three and one of one, and a workgroup's read, join and write do not overlap (capped at 128 registers
// they spill: 58 us).
template <class T, int VEC, int NT, int ITEMS, bool STREAM>
__global__ __launch_bounds__(NT) void lastBackward(NormArgs a, int total) {
  __shared__ Columns<NT, VEC, float> space;
  __shared__ float sums[2][kBand];
  __shared__ Moments stats[NT], means[NT];
  __shared__ float2 params[kBand];
  const int index = nearWork(total);
  if (index < 0) return;
  const Band band = bandOf<VEC>(a, index);
  const T* const x = laneOf<const T>(a, a.x, band, VEC);
  const T* const g = laneOf<const T>(a, a.g, band, VEC);
  const int P = (int)a.P;
  typename Pack<T, VEC>::type rx[ITEMS], rg[ITEMS];
  if (band.live)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int p = band.r + i * a.rows;
      if (p < P) {
        rx[i] = *reinterpret_cast<const typename Pack<T, VEC>::type*>(x + pixelAt(a, a.x, p));
        rg[i] = *reinterpret_cast<const typename Pack<T, VEC>::type*>(g + pixelAt(a, a.g, p));
      }
    }
  bandParameters(a, band, params, NT);
  keptMoments(a, band, stats, NT);
  float s1[VEC] = {}, s2[VEC] = {};
  Channel<VEC> ch;
  ch.load(a, band, stats, params);
  if (band.live)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (band.r + i * a.rows < P) {
        float v[VEC], dz[VEC], z[VEC];
        unpack(rx[i], v);
        unpack(rg[i], dz);
        ch.arguments(v, z);
        slopeAll(z, dz, a.activation);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s1[j] += dz[j];
          s2[j] = __builtin_fmaf(dz[j], v[j], s2[j]);
        }
      }
  joinGradients<NT, VEC>(a, band, s1, s2, space, sums, params,
                         [&](int k, float m1, float m2) { means[k] = Moments{m1 * (float)a.share, m2 * (float)a.share}; });
  if (!a.y.data) return;
  __syncthreads();
  if (!band.live) return;
  T* const y = laneOf<T>(a, a.y, band, VEC);
  float m1[VEC], m2[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const Moments m = means[quotient(band.column * VEC + j, a.byD)];
    m1[j] = m.mean;
    m2[j] = m.rstd;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int p = band.r + i * a.rows;
    if (p >= P) break;
    float v[VEC], dz[VEC], z[VEC];
    unpack(rx[i], v);
    unpack(rg[i], dz);
    ch.arguments(v, z);
    slopeAll(z, dz, a.activation);
    inputGradient(ch, m1, m2, v, dz);
    leavePack<STREAM, T, VEC>(y + pixelAt(a, a.y, p), dz);
  }
}

template <class T, int VEC>
__global__ __launch_bounds__(kFirst) void lastGradSums(NormArgs a) {
  __shared__ Columns<kFirst, VEC, float> space;
  __shared__ float sums[2][kBand];
  __shared__ Moments stats[kFirst];
  __shared__ float2 params[kBand];
  const Band band = bandOf<VEC>(a, blockIdx.x);
  Walk<T, VEC, kAheadTwo> x(a, a.x, band), g(a, a.g, band);
  bandParameters(a, band, params, kFirst);
  keptMoments(a, band, stats, kFirst);
  Channel<VEC> ch;
  ch.load(a, band, stats, params);
  float s1[VEC] = {}, s2[VEC] = {};
  if (band.live)
    for (int p = x.p; p < x.end; p += kAheadTwo * x.rows) {
      x.next(a, a.x);
      g.next(a, a.g);
#pragma unroll
      for (int k = 0; k < kAheadTwo; ++k)
        if (p + k * x.rows < x.end) {
          float v[VEC], dz[VEC], z[VEC];
          unpack(x.now[k], v);
          unpack(g.now[k], dz);
          ch.arguments(v, z);
          slopeAll(z, dz, a.activation);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            s1[j] += dz[j];
            s2[j] = __builtin_fmaf(dz[j], v[j], s2[j]);
          }
        }
    }
  joinGradients<kFirst, VEC>(a, band, s1, s2, space, sums, params, [&](int k, float m1, float m2) {
    a.groups[(band.b * a.G + band.firstGroup + k) * a.pieces + band.piece] = float2{m1, m2};
  });
}

// (The first `before` workgroups add up the gradients of weight and bias.)  16 x 32 x 256 x 256 f16: 36 us for 201 MB, the
// sums before it 35 us for 134 MB: 5.6 and 3.8 TB/s, beside an exponential and 20 other operations for each value.
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void lastGradApply(NormArgs a, int before) {
  __shared__ Moments stats[256], means[256];
  __shared__ union {
    float2 params[kBand], part[32][kParameters];
  } space;
  if ((int)blockIdx.x < before) return parameterGradients(a, blockIdx.x, space.part);
  float2* const params = space.params;
  const Band band = bandOf<VEC, true>(a, gridDim.x - 1 - blockIdx.x);
  Walk<T, VEC, kAheadTwo> x(a, a.x, band), g(a, a.g, band);
  bandParameters(a, band, params, 256);
  const Share share = shareOf<256>(band.groups, a.pieces);
  float f1 = 0, f2 = 0;
  if (share.group < band.groups)
#pragma unroll 4
    for (int i = share.place; i < a.pieces; i += share.lanes) {
      const float2 s = a.groups[(band.b * a.G + band.firstGroup + share.group) * a.pieces + i];
      f1 += s.x;
      f2 += s.y;
    }
  f1 = waveSumOf(f1, share.lanes);
  f2 = waveSumOf(f2, share.lanes);
  if (share.group < band.groups && share.place == 0) means[share.group] = Moments{f1 * (float)a.share, f2 * (float)a.share};
  keptMoments(a, band, stats, 256);
  if (!band.live) return;
  T* const y = laneOf<T>(a, a.y, band, VEC);
  Channel<VEC> ch;
  ch.load(a, band, stats, params);
  float m1[VEC], m2[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const Moments m = means[quotient(band.column * VEC + j, a.byD)];
    m1[j] = m.mean;
    m2[j] = m.rstd;
  }
  for (int p = x.p; p < x.end; p += kAheadTwo * x.rows) {
    x.next(a, a.x);
    g.next(a, a.g);
#pragma unroll
    for (int k = 0; k < kAheadTwo; ++k)
      if (p + k * x.rows < x.end) {
        float v[VEC], dz[VEC], z[VEC];
        unpack(x.now[k], v);
        unpack(g.now[k], dz);
        ch.arguments(v, z);
        slopeAll(z, dz, a.activation);
        inputGradient(ch, m1, m2, v, dz);
        leavePack<STREAM, T, VEC>(y + pixelAt(a, a.y, p + k * x.rows), dz);
      }
  }
}

// ---- Planes ----

// Elements e ... e + VEC - 1 of the n of a group: neighbours (VEC > 1), or one by its strides.
template <class T, int VEC>
struct Words {
  typename Pack<T, VEC>::type raw;

  static __device__ __forceinline__ long offset(const NormArgs& a, const Image& i, int e) {
    const int c = quotient(e, a.byP);
    return c * i.c + pixelAt(a, i, e - c * (int)a.P);
  }
  __device__ __forceinline__ void load(const NormArgs& a, const Image& i, const T* base, int e, int n) {
    if constexpr (VEC == 1) {
      raw = e < n ? base[offset(a, i, e)] : (T)0.f;
    } else if (e + VEC <= n) {
      raw = *reinterpret_cast<const typename Pack<T, VEC>::type*>(base + e);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) raw[j] = e + j < n ? base[e + j] : (T)0.f;
    }
  }
  template <bool STREAM>
  static __device__ __forceinline__ void store(const NormArgs& a, const Image& i, T* base, int e, int n, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
      if (e < n) base[offset(a, i, e)] = (T)v[0];
    } else if (e + VEC <= n) {
      leavePack<STREAM, T, VEC>(base + e, v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (e + j < n) base[e + j] = (T)v[j];
    }
  }
};

// weight and bias of elements e ... of group g: of one channel or, over the end of a plane, of two (planes are no
// smaller than a word)
template <int VEC>
struct Along {
  float w[VEC], shift[VEC];

  __device__ __forceinline__ void load(const NormArgs& a, long group, int e) {
    const int P = (int)a.P, c = quotient(e, a.byP), left = (c + 1) * P - e;
    const long first = group * a.D + c, second = c + 1 < a.D ? first + 1 : first;
    const float w0 = lineOr(a.weight, first, 1.f), shift0 = lineOr(a.bias, first, 0.f);
    float w1 = w0, shift1 = shift0;
    if (VEC > 1 && left < VEC) {
      w1 = lineOr(a.weight, second, 1.f);
      shift1 = lineOr(a.bias, second, 0.f);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      w[j] = j < left ? w0 : w1;
      shift[j] = j < left ? shift0 : shift1;
    }
  }
};

// A team of TEAM lanes holds a group in registers; teams of 64 share a workgroup of 256.  128 x 192 x 23 x 23 fp32: 21 us
// for 104 MB, 5.0 TB/s, against 18 us for a copy.
template <class T, int VEC, int TEAM, int ITEMS, bool STREAM>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void planesForward(NormArgs a) {
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  __shared__ double space[TEAM / 64];
  const int t = threadIdx.x % TEAM, n = (int)(a.D * a.P);
  const long index = (long)blockIdx.x * TEAMS + threadIdx.x / TEAM;
  if (index >= a.B * a.G) return;  // (a whole wave: teams of more are a workgroup each)
  const long b = index / a.G, g = index % a.G;
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + g * a.D * a.x.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + g * a.D * a.y.c;
  Words<T, VEC> v[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) v[i].load(a, a.x, x, (i * TEAM + t) * VEC, n);
  double s1[VEC] = {}, s2[VEC] = {};
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {  // (zeros behind the end)
    float f[VEC];
    unpack(v[i].raw, f);
    moments(f, s1, s2);
  }
#pragma unroll
  for (int j = 1; j < VEC; ++j) s1[0] += s1[j], s2[0] += s2[j];
  s1[0] = teamSum<TEAM>(s1[0], space);
  s2[0] = teamSum<TEAM>(s2[0], space);
  const Moments m = momentsOf(a, s1[0], s2[0]);
  if (t == 0) {
    if (a.mean) a.mean[b * a.meanB + g * a.meanG] = m.mean;
    if (a.rstd) a.rstd[b * a.rstdB + g * a.rstdG] = m.rstd;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int e = (i * TEAM + t) * VEC;
    if (e >= n) break;
    Along<VEC> p;
    p.load(a, g, e);
    float out[VEC];
    unpack(v[i].raw, out);
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = affine((out[j] - m.mean) * m.rstd, p.w[j], p.shift[j]);
    activateAll(out, a.activation);
    Words<T, VEC>::template store<STREAM>(a, a.y, y, e, n, out);
  }
}

// A workgroup sums a piece of a group whose planes are small: 64 x 64 x 40 x 40 fp32, one group: 6.7 us for 26 MB.
template <class T, int VEC>
__global__ __launch_bounds__(256) void planesSums(NormArgs a) {
  __shared__ double space[4];
  const long piece = blockIdx.x % a.pieces, index = blockIdx.x / a.pieces, b = index / a.G, g = index % a.G;
  const int n = (int)(a.D * a.P), end = (int)min((piece + 1) * a.piece, (long)n);
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + g * a.D * a.x.c;
  double s1[VEC] = {}, s2[VEC] = {};
#pragma unroll 4
  for (long e = piece * a.piece + threadIdx.x * VEC; e < end; e += 256 * VEC) {
    Words<T, VEC> v;
    v.load(a, a.x, x, (int)e, end);
    float f[VEC];
    unpack(v.raw, f);
    moments(f, s1, s2);
  }
#pragma unroll
  for (int j = 1; j < VEC; ++j) s1[0] += s1[j], s2[0] += s2[j];
  s1[0] = teamSum<256>(s1[0], space);
  s2[0] = teamSum<256>(s2[0], space);
  if (threadIdx.x == 0) a.sums[index * a.pieces + piece] = double2{s1[0], s2[0]};
}

// (the same shape: 12.6 us for 52 MB, each word's channel by a division)
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void planesApply(NormArgs a) {
  __shared__ double space[4];
  const long block = gridDim.x - 1 - blockIdx.x;
  const long piece = block % a.pieces, index = block / a.pieces, b = index / a.G, g = index % a.G;
  const int n = (int)(a.D * a.P), end = (int)min((piece + 1) * a.piece, (long)n);
  double s1 = 0, s2 = 0;
  for (int i = threadIdx.x; i < a.pieces; i += 256) {
    const double2 s = a.sums[index * a.pieces + i];
    s1 += s.x;
    s2 += s.y;
  }
  s1 = teamSum<256>(s1, space);
  s2 = teamSum<256>(s2, space);
  const Moments m = momentsOf(a, s1, s2);
  if (threadIdx.x == 0 && piece == 0) {
    if (a.mean) a.mean[b * a.meanB + g * a.meanG] = m.mean;
    if (a.rstd) a.rstd[b * a.rstdB + g * a.rstdG] = m.rstd;
  }
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + g * a.D * a.x.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + g * a.D * a.y.c;
#pragma unroll 4
  for (long e = piece * a.piece + threadIdx.x * VEC; e < end; e += 256 * VEC) {
    Words<T, VEC> v;
    v.load(a, a.x, x, (int)e, end);
    Along<VEC> p;
    p.load(a, g, (int)e);
    float out[VEC];
    unpack(v.raw, out);
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = affine((out[j] - m.mean) * m.rstd, p.w[j], p.shift[j]);
    activateAll(out, a.activation);
    Words<T, VEC>::template store<STREAM>(a, a.y, y, (int)e, end, out);
  }
}

// A team sums a piece of one plane.  16 x 32 x 256 x 256 fp32: 50 us for 268 MB, 5.4 TB/s.
template <class T, int VEC, int TEAM>
__global__ __launch_bounds__(256) void planesGradSums(NormArgs a) {
  constexpr int TEAMS = 256 / TEAM;
  __shared__ float space[TEAM / 64];
  const long block = (long)blockIdx.x * TEAMS + threadIdx.x / TEAM;
  if (block >= a.B * a.C * a.pieces) return;  // (a whole wave)
  const long piece = block % a.pieces, index = block / a.pieces, b = index / a.C, c = index % a.C, group = c / a.D;
  const int t = threadIdx.x % TEAM, end = (int)min((piece + 1) * a.piece, a.P);
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  const float w = lineOr(a.weight, c, 1.f), shift = lineOr(a.bias, c, 0.f);
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + c * a.x.c;
  const T* const g = static_cast<const T*>(a.g.data) + b * a.g.b + c * a.g.c;
  float s1 = 0, s2 = 0;
#pragma unroll 2
  for (long e = piece * a.piece + t * VEC; e < end; e += TEAM * VEC) {
    Words<T, VEC> vx, vg;
    vx.load(a, a.x, x, (int)e, end);
    vg.load(a, a.g, g, (int)e, end);
    float fx[VEC], fg[VEC];
    unpack(vx.raw, fx);
    unpack(vg.raw, fg);
    float z[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      fx[j] = (fx[j] - mean) * rstd;
      z[j] = affine(fx[j], w, shift);
    }
    slopeAll(z, fg, a.activation);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      // (behind the end nothing, whatever the slope is there)
      const float dz = e + j < end ? fg[j] : 0.f;
      s1 += dz;
      s2 = __builtin_fmaf(dz, fx[j], s2);
    }
  }
  s1 = teamSum<TEAM>(s1, space);
  s2 = teamSum<TEAM>(s2, space);
  if (t == 0) a.channels[(b * a.pieces + piece) * a.C + c] = float2{s1, s2};
}

// A workgroup: 256 VEC elements, times `each`, of a group.  The first `before` of them add up the gradients of weight
// and bias.  92 x 176 x 27 x 26 f16, whose planes no words fit: 21 us for 68 MB, the sums before it 23 for 45 MB.
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void planesGradApply(NormArgs a, long blocks, int each, int before) {
  __shared__ float space[4];
  __shared__ float2 sums[32][kParameters];
  if ((int)blockIdx.x < before) return parameterGradients(a, blockIdx.x, sums);
  const long block = gridDim.x - 1 - blockIdx.x, part = block % blocks, index = block / blocks, b = index / a.G, group = index % a.G;
  const int n = (int)(a.D * a.P);
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  float m1 = 0, m2 = 0;
  for (long i = threadIdx.x; i < a.D * a.pieces; i += 256) {
    const long c = group * a.D + i % a.D;
    const float2 s = a.channels[(b * a.pieces + i / a.D) * a.C + c];
    const float w = lineOr(a.weight, c, 1.f);
    m1 += s.x * w;
    m2 += s.y * w;
  }
  const float scale = 1.f / (float)n;
  m1 = teamSum<256>(m1, space) * scale;
  m2 = teamSum<256>(m2, space) * scale;
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + group * a.D * a.x.c;
  const T* const g = static_cast<const T*>(a.g.data) + b * a.g.b + group * a.D * a.g.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + group * a.D * a.y.c;
#pragma unroll 2
  for (int i = 0; i < each; ++i) {
    const long at = ((part * each + i) * 256 + threadIdx.x) * VEC;
    if (at >= n) break;
    const int e = (int)at;
    Words<T, VEC> vx, vg;
    vx.load(a, a.x, x, e, n);
    vg.load(a, a.g, g, e, n);
    Along<VEC> p;
    p.load(a, group, e);
    float fx[VEC], out[VEC], z[VEC];
    unpack(vx.raw, fx);
    unpack(vg.raw, out);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      fx[j] = (fx[j] - mean) * rstd;
      z[j] = affine(fx[j], p.w[j], p.shift[j]);
    }
    slopeAll(z, out, a.activation);
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = rstd * (out[j] * p.w[j] - m1 - fx[j] * m2);
    Words<T, VEC>::template store<STREAM>(a, a.y, y, e, n, out);
  }
}

// Large planes: a workgroup to a piece of one plane, whose weight and bias it knows.  (The pieces and cuts are of a
// plane here.)  What a lane has on its way: four words of one operand, two of each of two.
template <class T, int VEC, int AHEAD>
struct Run {
  Words<T, VEC> coming[AHEAD], now[AHEAD];
  const T* from;
  int e, end;

  __device__ __forceinline__ void request(const NormArgs& a, const Image& i) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (e + k * 256 * VEC < end) coming[k].load(a, i, from, e + k * 256 * VEC, end);
  }
  __device__ __forceinline__ Run(const NormArgs& a, const Image& i, long b, long c, long first, long size)
      : from(static_cast<const T*>(i.data) + b * i.b + c * i.c), e((int)first + threadIdx.x * VEC), end((int)min(first + size, a.P)) {
    request(a, i);
  }
  __device__ __forceinline__ void next(const NormArgs& a, const Image& i) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) now[k] = coming[k];
    e += AHEAD * 256 * VEC;
    request(a, i);
  }
};

// A workgroup sums a piece of one plane: 16 x 32 x 256 x 256 fp32 28 us for 134 MB, 4.8 TB/s.
template <class T, int VEC>
__global__ __launch_bounds__(256) void planeSums(NormArgs a) {
  __shared__ double space[4];
  const int index = quotient(blockIdx.x, a.byPieces), piece = blockIdx.x - index * a.pieces;
  const long b = index / (int)a.C, c = index % (int)a.C;
  Run<T, VEC, kAhead> x(a, a.x, b, c, piece * a.piece, a.piece);
  double s1[VEC] = {}, s2[VEC] = {};
  for (int e = x.e; e < x.end; e += kAhead * 256 * VEC) {
    x.next(a, a.x);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (e + k * 256 * VEC < x.end) {  // (zeros behind the end of a word)
        float v[VEC];
        unpack(x.now[k].raw, v);
        moments(v, s1, s2);
      }
  }
#pragma unroll
  for (int j = 1; j < VEC; ++j) s1[0] += s1[j], s2[0] += s2[j];
  s1[0] = teamSum<256>(s1[0], space);
  s2[0] = teamSum<256>(s2[0], space);
  if (threadIdx.x == 0) a.sums[(long)index * a.pieces + piece] = double2{s1[0], s2[0]};
}

// A workgroup writes a piece of one plane: the same shape, 42 us for 268 MB, 6.4 TB/s (the cache holds a part).
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void planeApply(NormArgs a) {
  __shared__ double space[4];
  const int block = gridDim.x - 1 - blockIdx.x, index = quotient(block, a.byCuts), cut = block - index * a.cuts;
  const long b = index / (int)a.C, c = index % (int)a.C, g = quotient((int)c, a.byD);
  Run<T, VEC, kAhead> x(a, a.x, b, c, cut * a.cut, a.cut);
  const float w = lineOr(a.weight, c, 1.f), shift = lineOr(a.bias, c, 0.f);
  const double2* const sums = a.sums + (b * a.C + g * a.D) * a.pieces;
  double s1 = 0, s2 = 0;
  for (long i = threadIdx.x; i < a.D * a.pieces; i += 256) {
    s1 += sums[i].x;
    s2 += sums[i].y;
  }
  s1 = teamSum<256>(s1, space);
  s2 = teamSum<256>(s2, space);
  const Moments m = momentsOf(a, s1, s2);
  if (threadIdx.x == 0 && cut == 0 && c == g * a.D) {
    if (a.mean) a.mean[b * a.meanB + g * a.meanG] = m.mean;
    if (a.rstd) a.rstd[b * a.rstdB + g * a.rstdG] = m.rstd;
  }
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + c * a.y.c;
  for (int e = x.e; e < x.end; e += kAhead * 256 * VEC) {
    x.next(a, a.x);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (e + k * 256 * VEC < x.end) {
        float v[VEC];
        unpack(x.now[k].raw, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = affine((v[j] - m.mean) * m.rstd, w, shift);
        activateAll(v, a.activation);
        Words<T, VEC>::template store<STREAM>(a, a.y, y, e + k * 256 * VEC, x.end, v);
      }
  }
}

// The same backward, 62 us for 403 MB, 6.5 TB/s.
template <class T, int VEC, bool STREAM>
__global__ __launch_bounds__(256) void planeGradApply(NormArgs a, int before) {
  __shared__ float space[4];
  __shared__ float2 sums[32][kParameters];
  if ((int)blockIdx.x < before) return parameterGradients(a, blockIdx.x, sums);
  const int block = gridDim.x - 1 - blockIdx.x, index = quotient(block, a.byCuts), cut = block - index * a.cuts;
  const long b = index / (int)a.C, c = index % (int)a.C, group = quotient((int)c, a.byD);
  Run<T, VEC, kAheadTwo> x(a, a.x, b, c, cut * a.cut, a.cut), g(a, a.g, b, c, cut * a.cut, a.cut);
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  const float w = lineOr(a.weight, c, 1.f), shift = lineOr(a.bias, c, 0.f);
  float m1 = 0, m2 = 0;
  for (long i = threadIdx.x; i < a.D * a.pieces; i += 256) {
    const long other = group * a.D + i % a.D;
    const float2 s = a.channels[(b * a.pieces + i / a.D) * a.C + other];
    const float v = lineOr(a.weight, other, 1.f);
    m1 += s.x * v;
    m2 += s.y * v;
  }
  m1 = teamSum<256>(m1, space) * (float)a.share;
  m2 = teamSum<256>(m2, space) * (float)a.share;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + c * a.y.c;
  for (int e = x.e; e < x.end; e += kAheadTwo * 256 * VEC) {
    x.next(a, a.x);
    g.next(a, a.g);
#pragma unroll
    for (int k = 0; k < kAheadTwo; ++k)
      if (e + k * 256 * VEC < x.end) {
        float v[VEC], out[VEC], z[VEC];
        unpack(x.now[k].raw, v);
        unpack(g.now[k].raw, out);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[j] = (v[j] - mean) * rstd;
          z[j] = affine(v[j], w, shift);
        }
        slopeAll(z, out, a.activation);
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = rstd * (out[j] * w - m1 - v[j] * m2);
        Words<T, VEC>::template store<STREAM>(a, a.y, y, e + k * 256 * VEC, x.end, out);
      }
  }
}

// ---- Any ----

// Groups wider than a row of lanes, whose pixels lie farther apart than their channels: neighbouring lanes take
// neighbouring channels (64 x 2048 x 7 x 7 bf16 channels last, one group, 13 MB: forward 101 us, backward 114;
// with neighbouring pixels, 256 lanes and every lane adding up all channels' sums 281 and 720).  A workgroup to a group
// leaves most of the card idle where groups are few: the form for shapes that no net here has.
constexpr int kAny = 1024;

// A workgroup takes one group of one image.
template <class T>
__global__ __launch_bounds__(kAny) void normAny(NormArgs a) {
  __shared__ double space[kAny / 64];
  const long b = blockIdx.x / a.G, g = blockIdx.x % a.G, n = a.D * a.P;
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + g * a.D * a.x.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + g * a.D * a.y.c;
  double s1 = 0, s2 = 0;
#pragma unroll 4
  for (long e = threadIdx.x; e < n; e += kAny) {
    const int p = quotient((int)e, a.byD);
    const double v = (float)x[(e - p * a.D) * a.x.c + pixelAt(a, a.x, p)];
    s1 += v;
    s2 += v * v;
  }
  s1 = teamSum<kAny>(s1, space);
  s2 = teamSum<kAny>(s2, space);
  const Moments m = momentsOf(a, s1, s2);
  const float mean = m.mean, rstd = m.rstd;
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[b * a.meanB + g * a.meanG] = mean;
    if (a.rstd) a.rstd[b * a.rstdB + g * a.rstdG] = rstd;
  }
#pragma unroll 2
  for (long e = threadIdx.x; e < n; e += kAny) {
    const int p = quotient((int)e, a.byD);
    const long c = e - p * a.D;
    const float v = (float)x[c * a.x.c + pixelAt(a, a.x, p)];
    const float w = lineOr(a.weight, g * a.D + c, 1.f), shift = lineOr(a.bias, g * a.D + c, 0.f);
    y[c * a.y.c + pixelAt(a, a.y, p)] = (T)activate(affine((v - mean) * rstd, w, shift), a.activation);
  }
}

// A workgroup sums 64 channels of one image.
template <class T>
__global__ __launch_bounds__(256) void normSumsAny(NormArgs a, int blocks) {
  __shared__ double2 space[4][64];
  const int lane = threadIdx.x % 64, r = threadIdx.x / 64;
  const long b = blockIdx.x / blocks, own = (blockIdx.x % blocks) * 64L + lane, c = min(own, a.C - 1), group = c / a.D;
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  const float w = lineOr(a.weight, c, 1.f), shift = lineOr(a.bias, c, 0.f);
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + c * a.x.c;
  const T* const g = static_cast<const T*>(a.g.data) + b * a.g.b + c * a.g.c;
  double s1 = 0, s2 = 0;
#pragma unroll 2
  for (int p = r; p < a.P; p += 4) {
    const float xh = ((float)x[pixelAt(a, a.x, p)] - mean) * rstd;
    const float dz = (float)g[pixelAt(a, a.g, p)] * slope(affine(xh, w, shift), a.activation);
    s1 += dz;
    s2 += (double)dz * xh;
  }
  space[r][lane] = double2{s1, s2};
  __syncthreads();
  if (r > 0 || own >= a.C) return;
  s1 = s2 = 0;
  for (int k = 0; k < 4; ++k) {
    s1 += space[k][lane].x;
    s2 += space[k][lane].y;
  }
  a.channels[b * a.C + c] = float2{(float)s1, (float)s2};
}

// A workgroup takes one group of one image.
template <class T>
__global__ __launch_bounds__(kAny) void normGradAny(NormArgs a) {
  __shared__ double space[kAny / 64];
  const long b = blockIdx.x / a.G, group = blockIdx.x % a.G, n = a.D * a.P;
  const float mean = a.mean[b * a.meanB + group * a.meanG], rstd = a.rstd[b * a.rstdB + group * a.rstdG];
  double s1 = 0, s2 = 0;
  for (long c = group * a.D + threadIdx.x; c < (group + 1) * a.D; c += kAny) {
    const float2 s = a.channels[b * a.C + c];
    const float w = lineOr(a.weight, c, 1.f);
    s1 += (double)s.x * w;
    s2 += (double)s.y * w;
  }
  const float m1 = (float)(teamSum<kAny>(s1, space) / n), m2 = (float)(teamSum<kAny>(s2, space) / n);
  const T* const x = static_cast<const T*>(a.x.data) + b * a.x.b + group * a.D * a.x.c;
  const T* const g = static_cast<const T*>(a.g.data) + b * a.g.b + group * a.D * a.g.c;
  T* const y = static_cast<T*>(a.y.data) + b * a.y.b + group * a.D * a.y.c;
#pragma unroll 2
  for (long e = threadIdx.x; e < n; e += kAny) {
    const int p = quotient((int)e, a.byD);
    const long c = e - p * a.D;
    const float w = lineOr(a.weight, group * a.D + c, 1.f), shift = lineOr(a.bias, group * a.D + c, 0.f);
    const float xh = ((float)x[c * a.x.c + pixelAt(a, a.x, p)] - mean) * rstd;
    const float dz = (float)g[c * a.g.c + pixelAt(a, a.g, p)] * slope(affine(xh, w, shift), a.activation);
    y[c * a.y.c + pixelAt(a, a.y, p)] = (T)(rstd * (dz * w - m1 - xh * m2));
  }
}

// ---- what runs ----

enum Family { Last, Planes, Any };

// The kernels of a problem: elements of a word, lanes of a workgroup or team and words of a lane where a group stays in
// registers (items 0: two launches), and the pieces that the first of two launches cuts a group into.
struct NormPlan {
  Family family;
  int vec, threads, items, band, lanes, rows;
  bool large;  // Planes: a workgroup to a piece of one plane
  long pieces, piece, cuts, cut;
};

bool unitPixels(const Image& i, long C, long H, long W) {
  return (W == 1 || i.w == 1) && (H == 1 || i.h == W) && (C == 1 || i.c == H * W);
}
bool wordsFit(const Image& i, long vec, size_t size) {
  return i.b % vec == 0 && i.h % vec == 0 && i.w % vec == 0 && aligned(i.data, vec * size);
}

constexpr long kMostPieces = 64, kLargePlane = 2048;
// (of each image's pixels, or of a group's values; the bound that the workspace is made for)
long piecesOf(long units, long images) {
  return std::max(1L, std::min({kMostPieces, 1024 / std::max(1L, images), units}));
}

NormPlan planOf(const NormProblem& p, bool backward) {
  const size_t size = p.type == FBFFT_FLOAT32 ? 4 : 2;
  const int most = 16 / (int)size;
  const long P = p.H * p.W, D = p.C / p.G, n = D * P;
  const Image* const used[3] = {&p.x, &p.y, &p.g};
  const int count = backward ? 3 : 2;
  bool unit = true, channels = true, nearer = true;
  for (int i = 0; i < count; ++i) {
    if (!used[i]->data) continue;
    unit = unit && unitPixels(*used[i], p.C, p.H, p.W);
    channels = channels && (p.C == 1 || used[i]->c == 1);
    nearer = nearer && std::abs(used[i]->w) < std::abs(used[i]->c);
  }
  NormPlan plan{};
  if (unit || (nearer && !channels)) {
    plan.family = Planes;
    plan.vec = unit && P >= most ? most : 1;
    const long held = (n + plan.vec - 1) / plan.vec;
    if (!backward) {
      plan.threads = held <= 64 * 4 ? 64 : held <= 256 * 4 ? 256 : 1024;
      plan.items = held <= plan.threads * 4L ? 4 : held <= plan.threads * 8L ? 8 : 0;
      plan.large = plan.items == 0 && P >= kLargePlane;
      if (plan.items == 0 && !plan.large) {
        plan.pieces = piecesOf((n + 4095) / 4096, p.B * p.G);
        plan.piece = ((n + plan.pieces - 1) / plan.pieces + plan.vec - 1) / plan.vec * plan.vec;
        return plan;
      }
    } else {
      plan.threads = P <= 64 * 4 * plan.vec ? 64 : 256;
      plan.large = P >= kLargePlane;
    }
    // (pieces and cuts begin with whole words)
    const auto words = [&](long size) { return (size + plan.vec - 1) / plan.vec * plan.vec; };
    plan.pieces = piecesOf((P + 4095) / 4096, p.B * p.C);
    plan.piece = words((P + plan.pieces - 1) / plan.pieces);
    plan.cuts = std::max(1L, std::min(2048 / (p.B * p.C), (P + 4095) / 4096));
    plan.cut = words((P + plan.cuts - 1) / plan.cuts);
    return plan;
  }
  plan.family = Last;
  for (plan.vec = channels ? most : 1; plan.vec > 1; plan.vec = plan.vec > 2 ? 2 : 1) {
    bool fit = p.C % plan.vec == 0;
    for (int i = 0; i < count; ++i) fit = fit && (!used[i]->data || wordsFit(*used[i], plan.vec, size));
    if (fit) break;
  }
  const long vec = plan.vec;
  long least = D;  // channels of the smallest band: whole groups and whole words
  while (least % vec != 0) least += D;
  if (least / vec > 256 || least > kBand || (D % vec != 0 && least > 256)) {
    plan.family = Any;
    plan.pieces = 1;
    return plan;
  }
  auto setBand = [&](long band, int threads) {
    plan.band = (int)std::min(band, p.C), plan.threads = threads;
    plan.lanes = (int)(plan.band / vec), plan.rows = threads / plan.lanes;
  };
  // A group in registers: workgroups of 256 lanes, several to a compute unit, before larger ones (128 x 192 x 23 x 23 bf16,
  // us: 20.0 and 32.5, backward 36.5 and 40), and of the bands of channels that fit them the widest that leaves a
  // workgroup for each unit.  16-bit types go down to bands of 32 bytes before larger workgroups, float32 does not (the
  // same shape, backward: 83 and 58); whatever a group has comes last.
  struct Choice {
    int threads, items, bytes;
  };
  const bool narrow = size == 2;
  const Choice choices[] = {{256, 4, 128}, {256, 8, 128}, {256, 4, 64},  {256, 8, 64},  {256, 4, narrow ? 32 : 0}, {256, 8, narrow ? 32 : 0},
                            {512, 8, 128}, {512, 8, 64},  {1024, 8, 64}, {256, 4, 1},   {256, 8, 1},               {512, 8, 1},
                            {1024, 8, 1}};
  const long bytes = least * (long)size;
  for (const Choice& c : choices) {
    if (c.bytes == 0 || (backward && c.threads == 1024)) continue;  // (two operands of 1024 lanes would not fit their registers)
    const long band = std::min(p.C, (c.bytes + bytes - 1) / bytes * least), lanes = band / vec, bands = (p.C + band - 1) / band;
    if (c.bytes > 1 && p.B * bands < 256 && band > least) continue;
    if (lanes > c.threads || band / D > c.threads || band > kBand || P > c.threads / lanes * (long)c.items) continue;
    setBand(band, c.threads);
    plan.items = c.items;
    plan.pieces = 1, plan.piece = P;
    return plan;
  }
  // two launches: bands as wide as they may be, of which a pixel's values fill whole lines (69 x 160 x 66 x 69 f16, 63 us;
  // bands of 256 and 128 bytes: 93 and 133)
  long band = least;
  while (band + least <= p.C && (band + least) / vec <= 256 && band + least <= kBand && (band + least) / D <= 256 &&
         (D % vec == 0 || band + least <= 256))
    band += least;
  setBand(band, kFirst);
  const long images = p.B * ((p.C + plan.band - 1) / plan.band), second = 256 / plan.lanes;
  plan.pieces = piecesOf((P + 4 * plan.rows - 1) / (4 * plan.rows), images);
  plan.piece = (P + plan.pieces - 1) / plan.pieces;
  plan.cuts = std::max(1L, std::min(2048 / images, (P + 4 * second - 1) / (4 * second)));
  plan.cut = (P + plan.cuts - 1) / plan.cuts;
  return plan;
}

NormArgs argsOf(const NormProblem& p, const NormPlan& plan, bool backward) {
  NormArgs a{};
  a.x = p.x, a.y = p.y, a.g = p.g;
  a.weight = p.weight, a.bias = p.bias, a.gradWeight = p.gradWeight, a.gradBias = p.gradBias;
  a.mean = p.mean, a.rstd = p.rstd;
  a.meanB = p.meanB, a.meanG = p.meanG, a.rstdB = p.rstdB, a.rstdG = p.rstdG;
  a.B = p.B, a.C = p.C, a.G = p.G, a.D = p.C / p.G, a.H = p.H, a.W = p.W, a.P = p.H * p.W;
  a.activation = p.activation, a.eps = p.eps;
  a.share = 1.0 / ((double)a.D * a.P);
  a.byW = divisorOf(a.W), a.byP = divisorOf(a.P), a.byD = divisorOf(a.D), a.byLanes = divisorOf(plan.lanes);
  a.byPieces = divisorOf(plan.pieces), a.byBands = divisorOf(plan.band ? (p.C + plan.band - 1) / plan.band : 1);
  a.band = plan.band, a.rows = plan.rows, a.lanes = plan.lanes, a.pieces = (int)plan.pieces, a.piece = plan.piece;
  a.rowsSecond = plan.lanes ? 256 / plan.lanes : 0, a.cuts = (int)plan.cuts, a.cut = plan.cut, a.byCuts = divisorOf(plan.cuts);
  char* const space = static_cast<char*>(p.workspace);
  if (!backward) {
    a.sums = reinterpret_cast<double2*>(space);
  } else {
    a.groups = reinterpret_cast<float2*>(space);
    a.channels = a.groups + (p.B * kMostPieces < 1024 ? p.B * kMostPieces : std::max(1024L, p.B)) * p.G;
  }
  return a;
}

long blocksOf(const NormArgs& a) { return a.B * ((a.C + a.band - 1) / a.band) * a.pieces; }

// the parts that planesGradApply cuts a group into, and the words of a lane of each
struct Parts {
  long blocks, each;
};
Parts partsOf(const NormPlan& plan, const NormArgs& a) {
  const long words = (a.D * a.P + plan.vec - 1) / plan.vec, each = std::max(1L, std::min(8L, words * a.B * a.G / (256 * 4096)));
  return {(words + 256 * each - 1) / (256 * each), each};
}

// Whether each launch of a pass holds its lanes (`before`: workgroups that add up the gradients of weight and bias).
bool fits(const NormPlan& plan, const NormArgs& a, bool backward, long before) {
  const double groups = (double)a.B * a.G, planes = (double)a.B * a.C;
  if (plan.family == Last) {
    const double total = (double)blocksOf(a);
    if (plan.items > 0) return launches(total + 8, plan.threads);
    return launches(total, kFirst) && launches(total / a.pieces * a.cuts + before, 256);
  }
  if (plan.family == Any) return launches(groups, kAny) && (!backward || launches((double)a.B * ((a.C + 63) / 64), 256));
  if (plan.large) return launches(planes * a.pieces, 256) && launches(planes * a.cuts + before, 256);
  if (backward)
    return launches(plan.threads == 64 ? (planes * a.pieces + 3) / 4 : planes * a.pieces, 256) &&
           launches(groups * partsOf(plan, a).blocks + before, 256);
  if (plan.items == 0) return launches(groups * a.pieces, 256);
  return plan.threads == 64 ? launches((groups + 3) / 4, 256) : launches(groups, plan.threads);
}

// images `first` ... `first` + count - 1 of a problem
NormProblem imagesOf(NormProblem p, long first, long count) {
  const long size = p.type == FBFFT_FLOAT32 ? 4 : 2;
  for (Image* i : {&p.x, &p.y, &p.g})
    if (i->data) i->data = static_cast<char*>(i->data) + first * i->b * size;
  if (p.mean) p.mean += first * p.meanB;
  if (p.rstd) p.rstd += first * p.rstdB;
  p.B = count;
  return p;
}

// How many images go into one set of launches where all of them do not: of 2^22 and more planes or groups, whose lanes pass
// what a launch holds.  0: not even one.
long imagesAtOnce(const NormProblem& p, bool backward, long before) {
  for (long images = p.B; images > 1;) {
    images = (images + 1) / 2;
    const NormProblem q = imagesOf(p, 0, images);
    const NormPlan plan = planOf(q, backward);
    if (fits(plan, argsOf(q, plan, backward), backward, before)) return images;
  }
  return 0;
}

template <class T, int VEC, bool S>
int forwardLast(const NormPlan& plan, const NormArgs& a, hipStream_t s) {
  const int total = (int)blocksOf(a);
  const dim3 grid((unsigned)total), dealt((unsigned)((total + 7) / 8 * 8)), second((unsigned)(total / a.pieces * a.cuts));
  if (plan.items == 0) {
    lastSums<T, VEC><<<grid, kFirst, 0, s>>>(a);
    lastApply<T, VEC, S><<<second, 256, 0, s>>>(a);
  } else if (plan.items == 4) {
    lastForward<T, VEC, 256, 4, S><<<dealt, 256, 0, s>>>(a, total);
  } else if (plan.threads == 256) {
    lastForward<T, VEC, 256, 8, S><<<dealt, 256, 0, s>>>(a, total);
  } else if (plan.threads == 512) {
    lastForward<T, VEC, 512, 8, S><<<dealt, 512, 0, s>>>(a, total);
  } else {
    lastForward<T, VEC, 1024, 8, S><<<dealt, 1024, 0, s>>>(a, total);
  }
  return launchStatus();
}

template <class T, int VEC, bool S>
int forwardPlanes(const NormPlan& plan, const NormArgs& a, hipStream_t s) {
  const long groups = a.B * a.G;
  if (plan.large) {
    planeSums<T, VEC><<<dim3((unsigned)(a.B * a.C * a.pieces)), 256, 0, s>>>(a);
    planeApply<T, VEC, S><<<dim3((unsigned)(a.B * a.C * a.cuts)), 256, 0, s>>>(a);
  } else if (plan.items == 0) {
    planesSums<T, VEC><<<dim3((unsigned)(groups * a.pieces)), 256, 0, s>>>(a);
    planesApply<T, VEC, S><<<dim3((unsigned)(groups * a.pieces)), 256, 0, s>>>(a);
  } else if (plan.threads == 64) {
    planesForward<T, VEC, 64, 4, S><<<dim3((unsigned)((groups + 3) / 4)), 256, 0, s>>>(a);
  } else if (plan.threads == 256) {
    planesForward<T, VEC, 256, 4, S><<<dim3((unsigned)groups), 256, 0, s>>>(a);
  } else if (plan.items == 4) {
    planesForward<T, VEC, 1024, 4, S><<<dim3((unsigned)groups), 1024, 0, s>>>(a);
  } else {
    planesForward<T, VEC, 1024, 8, S><<<dim3((unsigned)groups), 1024, 0, s>>>(a);
  }
  return launchStatus();
}

// (both: whether the gradients of weight and bias are done, by `before` workgroups)
template <class T, int VEC, bool S>
bool backwardLast(const NormPlan& plan, const NormArgs& a, int before, hipStream_t s) {
  const int total = (int)blocksOf(a);
  const dim3 grid((unsigned)total), dealt((unsigned)((total + 7) / 8 * 8)), second((unsigned)(total / a.pieces * a.cuts));
  if (plan.items == 0) {
    lastGradSums<T, VEC><<<grid, kFirst, 0, s>>>(a);
    if (!a.y.data) return false;
    lastGradApply<T, VEC, S><<<dim3(second.x + (unsigned)before), 256, 0, s>>>(a, before);
    return true;
  }
  if (plan.items == 4)
    lastBackward<T, VEC, 256, 4, S><<<dealt, 256, 0, s>>>(a, total);
  else if (plan.threads == 256)
    lastBackward<T, VEC, 256, 8, S><<<dealt, 256, 0, s>>>(a, total);
  else
    lastBackward<T, VEC, 512, 8, S><<<dealt, 512, 0, s>>>(a, total);
  return false;
}

template <class T, int VEC, bool S>
bool backwardPlanes(const NormPlan& plan, const NormArgs& a, int before, hipStream_t s) {
  const long planes = a.B * a.C * a.pieces;
  if (plan.threads == 64)
    planesGradSums<T, VEC, 64><<<dim3((unsigned)((planes + 3) / 4)), 256, 0, s>>>(a);
  else
    planesGradSums<T, VEC, 256><<<dim3((unsigned)planes), 256, 0, s>>>(a);
  if (!a.y.data) return false;
  if (plan.large) {
    planeGradApply<T, VEC, S><<<dim3((unsigned)(a.B * a.C * a.cuts + before)), 256, 0, s>>>(a, before);
    return true;
  }
  const Parts parts = partsOf(plan, a);
  planesGradApply<T, VEC, S><<<dim3((unsigned)(a.B * a.G * parts.blocks + before)), 256, 0, s>>>(a, parts.blocks, (int)parts.each, before);
  return true;
}

template <class T>
int forwardImages(const NormPlan& plan, const NormArgs& a, bool stream, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (plan.family == Planes) {
    if (plan.vec == 1) return forwardPlanes<T, 1, false>(plan, a, s);
    return stream ? forwardPlanes<T, W, true>(plan, a, s) : forwardPlanes<T, W, false>(plan, a, s);
  }
  if (plan.family == Last) {
    if (plan.vec == 1) return forwardLast<T, 1, false>(plan, a, s);
    if (plan.vec == 2) return forwardLast<T, 2, false>(plan, a, s);
    return stream ? forwardLast<T, W, true>(plan, a, s) : forwardLast<T, W, false>(plan, a, s);
  }
  normAny<T><<<dim3((unsigned)(a.B * a.G)), kAny, 0, s>>>(a);
  return launchStatus();
}

template <class T>
int forward(const NormProblem& p, hipStream_t s) {
  const NormPlan plan = planOf(p, false);
  const NormArgs a = argsOf(p, plan, false);
  const bool stream = streams((double)p.B * p.C * a.P, p.type);
  if (fits(plan, a, false, 0)) return forwardImages<T>(plan, a, stream, s);
  const long images = imagesAtOnce(p, false, 0);
  if (images == 0) return FBFFT_UNSUPPORTED_SIZE;
  int rc = FBFFT_SUCCESS;
  for (long first = 0; first < p.B && rc == FBFFT_SUCCESS; first += images) {
    const NormProblem q = imagesOf(p, first, std::min(images, p.B - first));
    const NormPlan part = planOf(q, false);
    rc = forwardImages<T>(part, argsOf(q, part, false), stream, s);
  }
  return rc;
}

// (whether the gradients of weight and bias are done, by `before` workgroups)
template <class T>
bool backwardImages(const NormPlan& plan, const NormArgs& a, int before, bool stream, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (plan.family == Planes) {
    if (plan.vec == 1) return backwardPlanes<T, 1, false>(plan, a, before, s);
    return stream ? backwardPlanes<T, W, true>(plan, a, before, s) : backwardPlanes<T, W, false>(plan, a, before, s);
  }
  if (plan.family == Last) {
    if (plan.vec == 1) return backwardLast<T, 1, false>(plan, a, before, s);
    if (plan.vec == 2) return backwardLast<T, 2, false>(plan, a, before, s);
    return stream ? backwardLast<T, W, true>(plan, a, before, s) : backwardLast<T, W, false>(plan, a, before, s);
  }
  const long blocks = (a.C + 63) / 64;
  normSumsAny<T><<<dim3((unsigned)(a.B * blocks)), 256, 0, s>>>(a, (int)blocks);
  if (a.y.data) normGradAny<T><<<dim3((unsigned)(a.B * a.G)), kAny, 0, s>>>(a);
  return false;
}

template <class T>
int backward(const NormProblem& p, hipStream_t s) {
  NormPlan plan{Any};
  NormArgs a = argsOf(p, plan, true);
  const long parameters = a.gradWeight.data || a.gradBias.data ? (a.C + kParameters - 1) / kParameters : 0;
  if (!launches(parameters, 256)) return FBFFT_UNSUPPORTED_SIZE;
  bool done = parameters == 0;
  if (a.B == 0 || a.P == 0) {
    a.B = 0;  // the gradients of weight and bias are sums of nothing
  } else {
    plan = planOf(p, true);
    a = argsOf(p, plan, true);
    const bool stream = streams((double)p.B * p.C * a.P, p.type);
    if (fits(plan, a, true, parameters)) {
      done |= backwardImages<T>(plan, a, (int)parameters, stream, s);
    } else {
      const long images = imagesAtOnce(p, true, 0);
      if (images == 0) return FBFFT_UNSUPPORTED_SIZE;
      a.pieces = 1;  // the channels' sums of one image after the other
      for (long first = 0; first < p.B; first += images) {
        const NormProblem q = imagesOf(p, first, std::min(images, p.B - first));
        NormPlan part = planOf(q, true);
        part.pieces = 1, part.piece = a.P;
        NormArgs some = argsOf(q, part, true);
        some.channels = a.channels + first * a.C;
        backwardImages<T>(part, some, 0, stream, s);
      }
    }
  }
  if (!done) normParameters<<<dim3((unsigned)parameters), 256, 0, s>>>(a);
  return launchStatus();
}

}  // namespace

size_t normWorkspaceBytes(int pass, long B, long C, long P, long G) {
  // images times pieces: of any plan
  const long rows = B * kMostPieces < 1024 ? B * kMostPieces : std::max(1024L, B);
  if (pass == 0) return (size_t)(rows * G + std::max(B * C, 1024L)) * sizeof(double2);
  return (size_t)rows * (G + C) * sizeof(float2);
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
