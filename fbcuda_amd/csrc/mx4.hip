// Rows in microscaled 4-bit floating point, and their product with an epilogue.
//
//   a block of 32 neighbours v of a row:  e = floor(log2(max |v|)) - 2, at least -127;  code = nearest of v / 2^e, ties to even
//   product                               y = activation(sum_k x w + bias) + residual
//
// The scaled matrix instruction takes 128 k of 16 rows of both operands: a lane a whole block, 16 bytes, and the byte of its scale.
#include "mx4_plan.h"
#include "product.h"

#include <algorithm>

namespace fbfft_amd {
namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));

// The scale's byte of a block from the bits of its largest magnitude as float32 (numbers without sign, which order like the
// values), 255 for what is not finite.  floor(log2) is the exponent's field; the least scale is that of all numbers below 2^-124,
// those without an exponent of their own among them.
__device__ __forceinline__ int scaleOf(unsigned most) {
  const int exponent = (int)(most >> 23);
  return exponent == 255 ? 255 : max(exponent - 2, 0);
}

// N neighbours of a row, N a multiple of eight; behind `left` of them zeros.
template <class T, int N>
struct Values {
  static constexpr int per = 16 / sizeof(T), words = N / per;
  typename Pack<T, per>::type v[words];

  __device__ __forceinline__ void load(const T* from, long left) {
    if (left >= N) {
#pragma unroll
      for (int i = 0; i < words; ++i) v[i] = *reinterpret_cast<const typename Pack<T, per>::type*>(from + i * per);
    } else {
#pragma unroll
      for (int i = 0; i < words; ++i)
#pragma unroll
        for (int j = 0; j < per; ++j) v[i][j] = i * per + j < left ? from[i * per + j] : (T)0.f;
    }
  }
  __device__ __forceinline__ void gather(const T* from, long stride, long left) {
#pragma unroll
    for (int i = 0; i < words; ++i)
#pragma unroll
      for (int j = 0; j < per; ++j) v[i][j] = i * per + j < left ? from[(i * per + j) * stride] : (T)0.f;
  }

  // the bits of the largest magnitude, as float32
  __device__ __forceinline__ unsigned most() const {
    if constexpr (sizeof(T) == 4) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < words; ++i)
#pragma unroll
        for (int j = 0; j < per; ++j) m = max(m, __builtin_bit_cast(unsigned, (float)v[i][j]) & 0x7fffffffu);
      return m;
    } else {
      typedef unsigned short __attribute__((ext_vector_type(8))) Bits;
      Bits m = __builtin_bit_cast(Bits, v[0]) & (unsigned short)0x7fff;
#pragma unroll
      for (int i = 1; i < words; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(Bits, v[i]) & (unsigned short)0x7fff);
      unsigned short one = m[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) one = max(one, m[j]);
      return __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(T, one));
    }
  }

  // The codes of eight of them from 8 q.  The instruction takes the scale as the exponent of a float32 and divides exactly,
  // rounds to the nearest, ties to even, and saturates; a block whose scale is NaN has codes of zeros.
  __device__ __forceinline__ unsigned codes(int q, int scale) const {
    const float by = __builtin_bit_cast(float, (unsigned)scale << 23);
    unsigned c = 0;
#define FBFFT_PAIR(J, BYTE)                                                                                                       \
  if constexpr (sizeof(T) == 4) {                                                                                                 \
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2 * q + J / 4][J % 4], v[2 * q + J / 4][J % 4 + 1], by, BYTE);              \
  } else if constexpr (__is_same(T, half16)) {                                                                                    \
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, Two{v[q][J % per], v[q][J % per + 1]}, by, BYTE);                             \
  } else {                                                                                                                        \
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, Two{v[q][J % per], v[q][J % per + 1]}, by, BYTE);                            \
  }
    typedef T __attribute__((ext_vector_type(2))) Two;
    FBFFT_PAIR(0, 0)
    FBFFT_PAIR(2, 1)
    FBFFT_PAIR(4, 2)
    FBFFT_PAIR(6, 3)
#undef FBFFT_PAIR
    return scale == 255 ? 0 : c;
  }
};

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

// Eight values to a lane, a block to four neighbouring lanes: loads of 16 bytes and one pass, which memory bounds.  (8192 x 2048
// bf16, 85 MB there and back, 18.1 us, 15.5 at the rate of a copy and two launches.)
template <class T>
__global__ __launch_bounds__(256) void quantize(Matrix x, long M, long K, Mx4 to, Divisor perRow) {
  const int i = blockIdx.x * 256 + threadIdx.x, m = quotient(i, perRow), word = i - m * (int)perRow.value;
  if (m >= M) return;  // (a block's four lanes together)
  Values<T, 8> v;
  const T* const from = static_cast<const T*>(x.data) + m * x.row + 8l * word * x.col;
  if (x.col == 1)
    v.load(from, K - 8l * word);
  else
    v.gather(from, x.col, K - 8l * word);
  const int scale = scaleOf(mostOfFour(v.most()));
  *reinterpret_cast<unsigned*>(to.codes + m * to.codeStride + 4l * word) = v.codes(0, scale);
  if (word % 4 == 0) to.scales[m * to.scaleStride + word / 4] = (unsigned char)scale;
}

// The same lanes the other way: a word of eight codes, one store of 16 bytes.
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

// ---- products ----

struct Mx4Args {
  Mx4 x, w;
  long M, N, blocks, range;  // blocks per range of k
  Epilogue e;
};

// c + a b^T, with bytes OA and OB of the scales
template <int OA, int OB>
__device__ __forceinline__ floatx4 multiply(uintx4 a, int scaleA, uintx4 b, int scaleB, floatx4 c) {
  const intx8 x{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}, y{(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, OA, scaleA, OB, scaleB);
}
// bytes 2 a + H and 2 b + H, a and b 0 or 1 and known where this is compiled
template <int H>
__device__ __forceinline__ floatx4 multiplyAt(int a, int b, uintx4 fa, int scaleA, uintx4 fb, int scaleB, floatx4 c) {
  if (a) return b ? multiply<2 + H, 2 + H>(fa, scaleA, fb, scaleB, c) : multiply<2 + H, H>(fa, scaleA, fb, scaleB, c);
  return b ? multiply<H, 2 + H>(fa, scaleA, fb, scaleB, c) : multiply<H, H>(fa, scaleA, fb, scaleB, c);
}

// One step of an operand: eight blocks of each row, lines of 128 bytes.  A lane takes two neighbouring blocks of its row in
// two instructions, so that their scales are two neighbouring bytes.
template <int ROWS, int WAVES>
struct Packed : Direct<ROWS, 64, true, WAVES> {
  static __device__ __forceinline__ int laneAt(int first) {
    const int lane = threadIdx.x % 64, line = first + lane % 16;
    return line * 128 + Packed::permuted(line, lane / 16 * 2) * 16;
  }
  static __device__ __forceinline__ uintx4 fragment(const char* step, int lane, int h, int i) {
    return *reinterpret_cast<const uintx4*>(step + (lane ^ h * 16) + i * (16 * 128));
  }
};

// A workgroup: BM x BN results over one range of k, a wave WM x WN of them.  LDS holds the operands of two steps of 256 k; a
// thread moves the eight scales of one row of one operand through its registers.  In LDS the scales of rows r and r + 16 lie
// side by side for each pair of blocks: a lane's scales of two fragments in both instructions are one word.
// Bound by the matrix instructions and their fragments' way from LDS where k is long (4096 x 16384 x 4096 125 to 146 us, 3.8 to
// 4.4 PFLOP/s), and by the results where it is not: 8192 x 2048 x 8192 88 us without an activation, of which the products are 62;
// GELU adds 18, whose exponentials wait on nothing but find two waves to a SIMD, a bias and the residual of 134 MB 26 to 44 more.  Tiles
// of 256 need half of the operands' way from L2 that those of 128 do, and fill the chip only with large products.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void product(Mx4Args g) {
  constexpr int WAVES = BM / WM * (BN / WN), RM = WM / 16, RN = WN / 16;
  typedef Packed<BM, WAVES> A;
  typedef Packed<BN, WAVES> B;
  constexpr int SCALES = (BM + BN) * 8, STEP = A::bytes + B::bytes, LOADS = A::loads + B::loads;
  static_assert(BM + BN == WAVES * 64 && BM % 32 == 0 && WM % 32 == 0 && WN % 32 == 0, "a row's scales to a thread");
  // (one array: of two, the compiler makes every read of LDS wait for the loads on their way to it)
  __shared__ __attribute__((aligned(1024))) char space[2 * STEP + 2 * SCALES];
  char* const scales = space + 2 * STEP;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
  const Tile<BM, BN> tile(g.M, g.N, gridDim.x < 8 ? 0 : (int)blockIdx.y);
  if (!tile.any) return;
  const long m0 = tile.m0, n0 = tile.n0, first = blockIdx.y * g.range, end = min(first + g.range, g.blocks);

  A a;
  B b;
  a.setup(g.x.codes + m0 * g.x.codeStride + 16 * first, g.x.codeStride / 2, g.M - m0);
  b.setup(g.w.codes + n0 * g.w.codeStride + 16 * first, g.w.codeStride / 2, g.N - n0);

  // this thread's row of scales: of A, then of B (behind the last: the last again, whose results nobody takes)
  const bool ofA = threadIdx.x < BM;
  const int row = ofA ? threadIdx.x : threadIdx.x - BM;
  const unsigned char* from = ofA ? g.x.scales + min(m0 + row, g.M - 1) * g.x.scaleStride + first
                                  : g.w.scales + min(n0 + row, g.N - 1) * g.w.scaleStride + first;
  const int place = (ofA ? 0 : BM * 8) + row / 32 * 256 + row % 16 * 4 + row / 16 % 2 * 2;
  int ahead = (int)(end - first);  // blocks whose scales are not loaded yet
  typedef unsigned long __attribute__((aligned(1))) Eight;
  // The next eight scales; behind the last block 2^-127 (whose codes are zeros).  Of the first step there may be fewer than eight;
  // later ones, if there is anything left, have eight in front of the end.  (Without a branch, which the order of the loop's
  // instructions would not outlive: what is not wanted is read from the codes.)
  auto firstScales = [&]() __attribute__((always_inline)) {
    unsigned long v = 0;
    if (ahead >= 8) {
      v = *reinterpret_cast<const Eight*>(from);
    } else {
#pragma unroll 1
      for (int j = 0; j < ahead; ++j) v |= (unsigned long)from[j] << 8 * j;
    }
    from += 8;
    ahead -= 8;
    return v;
  };
  unsigned long coming;  // scales of the step after the one that is multiplied, so many of them behind the end
  int behind;
  auto nextScales = [&]() __attribute__((always_inline)) {
    behind = min(max(8 - ahead, 0), 7);
    coming = *reinterpret_cast<const Eight*>(ahead > 0 ? from - behind : g.x.codes);
    from += 8;
    ahead -= 8;
  };
  auto storeScales = [&](unsigned long v, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<unsigned short*>(scales + to * SCALES + place + q * 64) = (unsigned short)(v >> 16 * q);
  };

  floatx4 sum[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  int left = (int)(end - first) * 8;  // 16-bit words of a row that are not on their way yet
  auto load = [&](int q, char* to) __attribute__((always_inline)) {
    if (q < A::loads)
      a.load(q, left, to);
    else
      b.load(q - A::loads, left, to + A::bytes);
  };
  auto loaded = [&]() __attribute__((always_inline)) {
    a.base += a.advance;
    b.base += b.advance;
    left -= 64;
  };
#pragma unroll
  for (int q = 0; q < LOADS; ++q) load(q, space);
  loaded();
  const unsigned long scales0 = firstScales();
#pragma unroll
  for (int q = 0; q < LOADS; ++q) load(q, space + STEP);
  loaded();
  nextScales();
  storeScales(scales0, 0);

  const int laneA = A::laneAt(wm), laneB = B::laneAt(wn);
  const int scaleA = wm / 32 * 256 + lane / 16 * 64 + lane % 16 * 4, scaleB = BM * 8 + wn / 32 * 256 + lane / 16 * 64 + lane % 16 * 4;
  // A step is 2 RM groups of RN matrix instructions, of one fragment of x each, which is read two groups ahead
  constexpr int GROUPS = 2 * RM, AHEAD = 2, RING = 4;
  static_assert(GROUPS % RING == 0 && RN <= RM && RN % AHEAD == 0 && LOADS % AHEAD == 0, "whole turns");
  uintx4 fa[RING], fb[2][RN];
  int sa[2][RM / 2], sb[2][RN / 2];
  auto readA = [&](int t, int d) __attribute__((always_inline)) { fa[t % RING] = A::fragment(space + d * STEP, laneA, t / RM, t % RM); };
  auto readB = [&](int j, int h, int d) __attribute__((always_inline)) { fb[h][j] = B::fragment(space + d * STEP + A::bytes, laneB, h, j); };
  auto readScales = [&](int d) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RM / 2; ++i) sa[d][i] = *reinterpret_cast<const int*>(scales + d * SCALES + scaleA + i * 256);
#pragma unroll
    for (int j = 0; j < RN / 2; ++j) sb[d][j] = *reinterpret_cast<const int*>(scales + d * SCALES + scaleB + j * 256);
  };
  // (the first step's words are there; at most the second's are on their way)
  arrive<LOADS>();
  readScales(0);
#pragma unroll
  for (int j = 0; j < RN; ++j) readB(j, 0, 0);
#pragma unroll
  for (int t = 0; t < AHEAD; ++t) readA(t, 0);
  auto round = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
#pragma unroll
      for (int t = 0; t < GROUPS; ++t) {
        const int last = t - (GROUPS - AHEAD);  // of the step's last groups
        if (last == 0) {
          // every wave has this step's fragments, so that its place is free, and the next step's operands are there
          storeScales(coming >> 8 * behind, d ^ 1);
          arrive<0>();
          readScales(d ^ 1);
        }
        if (last < 0) {
          readA(t + AHEAD, d);
          if (t < RN) readB(t, 1, d);
        } else {
          readA(last, d ^ 1);
#pragma unroll
          for (int j = last * (RN / AHEAD); j < (last + 1) * (RN / AHEAD); ++j) readB(j, 0, d ^ 1);
        }
#pragma unroll
        for (int j = 0; j < RN; ++j) {
          const int i = t % RM;
          if (t < RM)
            sum[i][j] = multiplyAt<0>(j % 2, i % 2, fb[0][j], sb[d][j / 2], fa[t % RING], sa[d][i / 2], sum[i][j]);
          else
            sum[i][j] = multiplyAt<1>(j % 2, i % 2, fb[1][j], sb[d][j / 2], fa[t % RING], sa[d][i / 2], sum[i][j]);
        }
        if (last >= 0) {
#pragma unroll
          for (int q = last * (LOADS / AHEAD); q < (last + 1) * (LOADS / AHEAD); ++q) load(q, space + d * STEP);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      nextScales();
      loaded();
      if (left <= -128) return false;  // that was the last step
    }
    return true;
  };
  while (round()) {
  }

  // (the loads requested behind the last step write zeros to LDS, which the results now go through)
  arrive<0>();
  constexpr int SHARE = 2 * STEP / WAVES, FIT = SHARE / (WN * 64);  // of LDS, to a wave; blocks of rows
  constexpr int TURN = FIT >= RM ? RM : FIT >= 4 ? 4 : FIT >= 2 ? 2 : 1;
  static_assert(FIT > 0 && RM % TURN == 0, "a wave's share of LDS holds whole rows of blocks");
  leave<T, RM, RN, TURN>(g, blockIdx.y, m0 + wm, n0 + wn, sum, space + wave * SHARE);
}

// Few rows.  A workgroup: 16 NB rows of w and 16 RB of x, its waves a range of k each, w straight from memory to the matrix
// instructions (rows behind the last are the last again, and nobody takes their results); their sums meet in LDS.  WAY (RB =
// 1): the workgroup quantises x to LDS by itself, while the first of w are on their way; else x is quantised already.
constexpr int kFewWaves = 8;

struct FewArgs {
  Mx4Args g;
  Matrix x;
  long K;
  Divisor across, words;  // workgroups to a band of rows; of eight values to a row of x
  int pitch, scales;      // of x in LDS: bytes from a row to the next, and in front of the scales
};

// Bound by w's way from memory, which needs many loads under way and no tile, and by the launch: 1 x 2048 x 8192 4.6 us, of which
// the bytes are 1.6 at the rate of a copy and an empty launch 3.5.  Quantising on the way saves a launch, 2.5 us there.
template <class T, bool WAY, int RB, int NB, int AHEAD>
__global__ __launch_bounds__(kFewWaves * 64) void fewRows(FewArgs f) {
  static_assert(!WAY || RB == 1, "quantised on the way: 16 rows at most");
  extern __shared__ __attribute__((aligned(16))) char space[];  // x, then the sums
  const Mx4Args& g = f.g;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, band = quotient(blockIdx.x, f.across);
  const long n0 = (long)(blockIdx.x - band * f.across.value) * (16 * NB), m0 = (long)band * (16 * RB);
  const unsigned char *w[NB], *ws[NB], *x[RB], *xs[RB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const long n = min(n0 + 16 * j + lane % 16, g.N - 1);
    w[j] = g.w.codes + n * g.w.codeStride, ws[j] = g.w.scales + n * g.w.scaleStride;
  }
  const int share = (int)((g.blocks + kFewWaves * 4 - 1) / (kFewWaves * 4) * 4), first = wave * share, end = min(first + share, (int)g.blocks);
  uintx4 cw[AHEAD][NB];
  int sw[AHEAD][NB];
  // (blocks behind the last: the last again, and then zeros times 2^-127)
  auto load = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int b = min(b0 + 4 * s + lane / 16, end - 1);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        cw[s][j] = *reinterpret_cast<const uintx4*>(w[j] + 16 * b);
        sw[s][j] = ws[j][b];
      }
    }
  };
  if (first < end) load(first);
  if constexpr (WAY) {
    const int words = (int)(g.M - m0 < 16 ? g.M - m0 : 16) * (int)f.words.value;
    for (int i = threadIdx.x; i < words; i += kFewWaves * 64) {  // (a block's four lanes together: f.words is a multiple of four)
      const int m = quotient(i, f.words), word = i - m * (int)f.words.value;
      Values<T, 8> v;
      v.load(static_cast<const T*>(f.x.data) + (m0 + m) * f.x.row + 8l * word, f.K - 8l * word);
      const int scale = scaleOf(mostOfFour(v.most()));
      *reinterpret_cast<unsigned*>(space + m * f.pitch + 4 * word) = v.codes(0, scale);
      if (word % 4 == 0) space[f.scales + m * (f.pitch / 16) + word / 4] = (char)scale;
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const long m = min(m0 + 16 * i + lane % 16, g.M - 1);
    x[i] = WAY ? reinterpret_cast<unsigned char*>(space) + (m - m0) * f.pitch : g.x.codes + m * g.x.codeStride;
    xs[i] = WAY ? reinterpret_cast<unsigned char*>(space) + f.scales + (m - m0) * (f.pitch / 16) : g.x.scales + m * g.x.scaleStride;
  }
  floatx4 sum[RB][NB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int b0 = first; b0 < end;) {
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int at = b0 + 4 * s + lane / 16, b = min(at, end - 1);
      const bool there = at < end;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const uintx4 c = *reinterpret_cast<const uintx4*>(x[i] + 16 * b);
        const int sx = there ? xs[i][b] : 0;
#pragma unroll
        for (int j = 0; j < NB; ++j)
          sum[i][j] = multiply<0, 0>(there ? cw[s][j] : uintx4{0, 0, 0, 0}, there ? sw[s][j] : 0, c, sx, sum[i][j]);
      }
    }
    b0 += 4 * AHEAD;
    if (b0 < end) load(b0);
  }
  if (WAY) __syncthreads();
  // (lane: row lane % 16 of x, four rows of w)
  float* const sums = reinterpret_cast<float*>(space);
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) sums[wave * (RB * NB * 256) + (16 * i + lane % 16) * (16 * NB) + 16 * j + lane / 16 * 4 + q] = sum[i][j][q];
  __syncthreads();
  for (int at = threadIdx.x; at < RB * NB * 256; at += kFewWaves * 64) {
    const long m = m0 + at / (16 * NB), n = n0 + at % (16 * NB);
    if (m >= g.M || n >= g.N) continue;
    float z = lineOr(g.e.bias, n, 0.f);
#pragma unroll
    for (int q = 0; q < kFewWaves; ++q) z += sums[q * (RB * NB * 256) + at];
    z = activate(z, g.e.activation);
    if (g.e.residual.data) z += (float)static_cast<const T*>(g.e.residual.data)[m * g.e.residual.row + n * g.e.residual.col];
    static_cast<T*>(g.e.out.data)[m * g.e.out.row + n * g.e.out.col] = (T)z;
  }
}

template <class T, bool WAY, int RB, int NB>
void launchFew(FewArgs f, hipStream_t s) {
  const long across = ceilDivLong(f.g.N, 16 * NB);
  f.across = divisorOf(across), f.words = divisorOf(4 * f.g.blocks);
  f.pitch = (int)(16 * f.g.blocks + 16), f.scales = (int)std::min(f.g.M, 16l) * f.pitch;
  const size_t rows = WAY ? fewBytes(f.g.M, f.g.blocks) : 0, bytes = std::max(rows, sizeof(float) * kFewWaves * RB * NB * 256);
  const dim3 grid((unsigned)(across * ceilDivLong(f.g.M, 16 * RB)));
  constexpr int most = RB * NB > 2 ? 2 : 4;
  const int steps = (int)ceilDivLong(f.g.blocks, 4 * kFewWaves);
  if (steps <= 1)
    fewRows<T, WAY, RB, NB, 1><<<grid, kFewWaves * 64, bytes, s>>>(f);
  else if (steps <= 2)
    fewRows<T, WAY, RB, NB, 2><<<grid, kFewWaves * 64, bytes, s>>>(f);
  else
    fewRows<T, WAY, RB, NB, most><<<grid, kFewWaves * 64, bytes, s>>>(f);
}

// ---- what runs ----

template <class T>
int run(const LinearMx4Problem& p, hipStream_t s) {
  const Mx4Plan plan = planOf(p.M, p.blocks, p.N, p.x.data && p.x.col == 1, computeUnits());
  Mx4Args g{p.xq, p.w, p.M, p.N, p.blocks, plan.range, Epilogue{p.y, p.residual, {}, p.bias, p.activation, false, nullptr}};
  g.e.dense = p.y.col == 1 && (!p.residual.data || p.residual.col == 1);
  char* space = static_cast<char*>(p.workspace);
  const bool tiles = plan.kind == Mx4Plan::Tiles;
  const long rows = tiles ? plan.rows : 16 * plan.rows, cols = tiles ? plan.cols : 16 * plan.cols;
  const long groups = ceilDivLong(p.M, rows) * ceilDivLong(p.N, cols), blocks = tiles && groups >= 8 ? (groups + 7) / 8 * 8 : groups;
  const JoinPlan join = plan.ranges > 1 ? joinOf(g.e.dense, p.M, p.N, plan.ranges) : JoinPlan{};
  const int lanes = tiles ? plan.rows * 2 : kFewWaves * 64;
  if (!launches((double)blocks * plan.ranges, lanes) || !launches(join.blocks, 256)) return FBFFT_UNSUPPORTED_SIZE;
  if (p.x.data && p.blocks > 0 && plan.kind != Mx4Plan::Way) {
    g.x = Mx4{reinterpret_cast<unsigned char*>(space), reinterpret_cast<unsigned char*>(space) + rounded((size_t)p.M * p.blocks * 16),
              16 * p.blocks, p.blocks};
    space += rounded((size_t)p.M * p.blocks * 16) + rounded((size_t)p.M * p.blocks);
    const int rc = launchMx4Quantize(p.x, p.type, p.M, p.K, g.x, s);
    if (rc != FBFFT_SUCCESS) return rc;
  }
  if (!tiles) {
    const FewArgs f{g, p.x, p.K, {}, {}, 0, 0};
    const bool two = plan.cols == 2;
    if (plan.kind == Mx4Plan::Way)
      two ? launchFew<T, true, 1, 2>(f, s) : launchFew<T, true, 1, 1>(f, s);
    else if (plan.rows == 1)
      two ? launchFew<T, false, 1, 2>(f, s) : launchFew<T, false, 1, 1>(f, s);
    else if (plan.rows == 2)
      two ? launchFew<T, false, 2, 2>(f, s) : launchFew<T, false, 2, 1>(f, s);
    else
      two ? launchFew<T, false, 4, 2>(f, s) : launchFew<T, false, 4, 1>(f, s);
    return launchStatus();
  }
  if (plan.ranges > 1) g.e.parts = reinterpret_cast<float*>(space);
  const dim3 grid((unsigned)blocks, (unsigned)plan.ranges);
  if (plan.rows == 256)
    product<T, 256, 256, 128, 64><<<grid, 512, 0, s>>>(g);
  else
    product<T, 128, 128, 64, 64><<<grid, 256, 0, s>>>(g);
  if (plan.ranges > 1) launchJoin<T>(join, g.e, p.M, p.N, (int)plan.ranges, s);
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

size_t linearMx4WorkspaceBytes(long M, long blocks, long N) {
  // (x, quantised in front of the product, and ranges' sums, whichever way x comes)
  const int units = computeUnits();
  const long ranges = std::max(planOf(M, blocks, N, true, units).ranges, planOf(M, blocks, N, false, units).ranges);
  return rounded((size_t)M * blocks * 16) + rounded((size_t)M * blocks) + (ranges > 1 ? rounded((size_t)ranges * M * N * sizeof(float)) : 0);
}

int launchLinearMx4(const LinearMx4Problem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return run<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? run<half16>(p, s) : run<brain16>(p, s);
}

}  // namespace fbfft_amd
