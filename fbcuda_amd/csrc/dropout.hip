// Dropout whose mask is drawn from a counter-based generator, forward and backward.
//
//   y[i] = (u(i) >= T ? x[i] * 65536 / (65536 - T) : 0) + residual[i]
//
// u(i): 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) at the counter (i / 8, offset).  Sixteen bits per
// element instead of 32 halve the generator, whose 20 products of 32 x 32 bits per counter run at a quarter of the
// rate of other vector instructions; T is the probability rounded to 16 bits, and the factor is that of T, so the
// expectation is exact.  1048576 x 32 bf16 with a residual: 35.6 us for 201 MB, 5.65 TB/s, the rate of a copy; 2000 f16: a
// launch, 1.7 us of 4.1.
#include "operators.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

struct DropoutArgs {
  const void *x, *residual;
  void* y;
  long size[FBFFT_MAX_DIM], xs[FBFFT_MAX_DIM], rs[FBFFT_MAX_DIM], ys[FBFFT_MAX_DIM];
  // from an element to the next one, which lies in the next place of dimension d and the first of those after it
  long xn[FBFFT_MAX_DIM], rn[FBFFT_MAX_DIM], yn[FBFFT_MAX_DIM];
  int outer;  // the first dimension of more than one
  long total;
  Divisor byInner;  // the innermost extent, where places are counted in 31 bits
  bool counted, words;  // whether they are; whether neighbours of a row are neighbours in every operand
  unsigned threshold, seedLow, seedHigh;
  unsigned long long offset;
  const unsigned long long* step;
  float factor;
};

struct Words {
  unsigned w[4];
};

// The multipliers and key increments are those of the published generator.
__device__ __forceinline__ Words philox(unsigned long long block, unsigned long long offset, unsigned k0, unsigned k1) {
  unsigned a = (unsigned)block, b = (unsigned)(block >> 32), c = (unsigned)offset, d = (unsigned)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p = (unsigned long long)a * 0xD2511F53u, q = (unsigned long long)c * 0xCD9E8D57u;
    a = (unsigned)(q >> 32) ^ b ^ k0;
    b = (unsigned)q;
    c = (unsigned)(p >> 32) ^ d ^ k1;
    d = (unsigned)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{a, b, c, d}};
}

// A thread takes the eight elements of one counter.  DENSE: they are neighbours in every operand.  Otherwise they still
// move as words where they lie in one row of neighbours: 8192 rows of 2048 fp32 with 8 more between the rows, with a
// residual, 152 us element by element, 39 as words (5.2 TB/s).  What lies across the end of a row goes by steps from place to
// place, all reads before the writes: 9403 rows of 2087 bf16 with 5 between them 24 us, 9683847 of 3 f16 with 5 148 us (each
// place computed from its index, one element after the other: 35 and 446).
template <class T, bool DENSE, bool STREAM>
__global__ __launch_bounds__(256) void dropout(DropoutArgs g) {
  const long block = (long)blockIdx.x * 256 + threadIdx.x, first = block * 8;
  if (first >= g.total) return;
  const Words words = philox(block, g.offset + (g.step ? *g.step : 0), g.seedLow, g.seedHigh);
  const T* const x = static_cast<const T*>(g.x);
  const T* const residual = static_cast<const T*>(g.residual);
  T* const y = static_cast<T*>(g.y);
  auto result = [&](int j, float v, float r) __attribute__((always_inline)) {
    const unsigned u = j % 2 ? words.w[j / 2] >> 16 : words.w[j / 2] & 0xFFFFu;
    return (u >= g.threshold ? v * g.factor : 0.f) + r;
  };
  if (DENSE) {
    if (first + 8 > g.total) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (first + j < g.total) y[first + j] = (T)result(j, (float)x[first + j], residual ? (float)residual[first + j] : 0.f);
      return;
    }
    float v[8], r[8] = {};
    loadPack<T, 8>(x + first, v);
    if (residual) loadPack<T, 8>(residual + first, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = result(j, v[j], r[j]);
    leavePack<STREAM, T, 8>(y + first, v);
    return;
  }
  constexpr int INNER = FBFFT_MAX_DIM - 1;
  long at[FBFFT_MAX_DIM];
  long rest = g.counted ? quotient((int)first, g.byInner) : first / g.size[INNER];
  at[INNER] = first - rest * g.size[INNER];
#pragma unroll
  for (int d = INNER - 1; d > 0; --d) {
    const long next = d <= g.outer ? 0 : rest / g.size[d];
    at[d] = rest - next * g.size[d];
    rest = next;
  }
  at[0] = rest;
  long xo = 0, ro = 0, yo = 0;
#pragma unroll
  for (int d = 0; d <= INNER; ++d) xo += at[d] * g.xs[d], ro += at[d] * g.rs[d], yo += at[d] * g.ys[d];
  if (g.words && at[INNER] + 8 <= g.size[INNER]) {
    float v[8], r[8] = {};
    loadPack<T, 8>(x + xo, v);
    if (residual) loadPack<T, 8>(residual + ro, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = result(j, v[j], r[j]);
    storePack<T, 8>(y + yo, v);
    return;
  }
  const int count = (int)min(8l, g.total - first);
  long from[8], by[8], to[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    from[j] = xo, by[j] = ro, to[j] = yo;
    bool carry = j + 1 < count;  // (behind the last element the places stay those of the last)
#pragma unroll
    for (int d = INNER; d >= 0; --d) {
      if (!carry) continue;
      carry = ++at[d] == g.size[d];
      if (carry)
        at[d] = 0;
      else
        xo += g.xn[d], ro += g.rn[d], yo += g.yn[d];
    }
  }
  // (all reads before the first write, for which nobody then waits)
  float v[8], r[8] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)x[from[j]];
  if (residual)
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (float)residual[by[j]];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) y[to[j]] = (T)result(j, v[j], r[j]);
}

template <class T>
void launch(const DropoutArgs& g, bool dense, bool stream, hipStream_t s) {
  const dim3 grid((unsigned)((g.total + 2047) / 2048));
  if (!dense)
    dropout<T, false, false><<<grid, 256, 0, s>>>(g);
  else if (stream)
    dropout<T, true, true><<<grid, 256, 0, s>>>(g);
  else
    dropout<T, true, false><<<grid, 256, 0, s>>>(g);
}

}  // namespace

int launchDropout(const DropoutProblem& p, hipStream_t s) {
  if (!launches((double)((p.total + 2047) / 2048), 256)) return FBFFT_UNSUPPORTED_SIZE;
  DropoutArgs g{};
  g.x = p.x, g.residual = p.residual, g.y = p.y, g.total = p.total;
  std::copy(p.size, p.size + FBFFT_MAX_DIM, g.size);
  std::copy(p.xs, p.xs + FBFFT_MAX_DIM, g.xs);
  std::copy(p.rs, p.rs + FBFFT_MAX_DIM, g.rs);
  std::copy(p.ys, p.ys + FBFFT_MAX_DIM, g.ys);
  g.threshold = p.threshold;
  // (65536 dropped of 65536: no element is kept, and the factor is never used)
  g.factor = p.threshold < 65536u ? (float)(65536.0 / (65536.0 - p.threshold)) : 0.f;
  g.seedLow = (unsigned)p.seed, g.seedHigh = (unsigned)(p.seed >> 32), g.offset = p.offset, g.step = p.step;
  // neighbouring dimensions that are one run in every operand become one; what is left lies to the right
  int last = FBFFT_MAX_DIM - 1;
  for (int d = FBFFT_MAX_DIM - 2; d >= 0; --d) {
    if (g.size[d] == 1) continue;
    const long n = g.size[last];
    if (n == 1 || (g.xs[d] == g.xs[last] * n && g.ys[d] == g.ys[last] * n && (!g.residual || g.rs[d] == g.rs[last] * n))) {
      if (n == 1) g.xs[last] = g.xs[d], g.ys[last] = g.ys[d], g.rs[last] = g.rs[d];
      g.size[last] = n * g.size[d];
    } else {
      --last;
      g.size[last] = g.size[d], g.xs[last] = g.xs[d], g.ys[last] = g.ys[d], g.rs[last] = g.rs[d];
    }
  }
  for (int d = 0; d < last; ++d) g.size[d] = 1;
  g.outer = last;
  for (int d = 0; d < FBFFT_MAX_DIM; ++d) {
    g.xn[d] = g.xs[d], g.rn[d] = g.rs[d], g.yn[d] = g.ys[d];
    for (int e = d + 1; e < FBFFT_MAX_DIM; ++e) {
      g.xn[d] -= (g.size[e] - 1) * g.xs[e];
      g.rn[d] -= (g.size[e] - 1) * g.rs[e];
      g.yn[d] -= (g.size[e] - 1) * g.ys[e];
    }
  }
  g.words = g.xs[FBFFT_MAX_DIM - 1] == 1 && g.ys[FBFFT_MAX_DIM - 1] == 1 && (!g.residual || g.rs[FBFFT_MAX_DIM - 1] == 1);
  g.words = g.words || g.total == 1;
  const bool dense = g.words && last == FBFFT_MAX_DIM - 1;
  g.counted = g.total <= 0x7fffffff;
  g.byInner = divisorOf(g.counted ? g.size[FBFFT_MAX_DIM - 1] : 1);
  const bool stream = streams((double)p.total, p.type);
  if (p.type == FBFFT_FLOAT32)
    launch<float>(g, dense, stream, s);
  else if (p.type == FBFFT_FLOAT16)
    launch<half16>(g, dense, stream, s);
  else
    launch<brain16>(g, dense, stream, s);
  return launchStatus();
}

}  // namespace fbfft_amd
