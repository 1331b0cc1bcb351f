// What products on the matrix instructions share: an epilogue, results on their way through LDS, tiles, operands that go straight
// from memory to LDS, ranges of k and how their sums meet.
#pragma once

#include "linear_step.h"
#include "operators.h"

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
  bool dense;    // rows of out, residual and z without gaps between neighbours
  float* parts;  // not null: fp32 sums of each range of k, [range][M][N], in place of results
};

// the biases from j
__device__ __forceinline__ void loadBias(const Line& bias, long j, float (&b)[8]) {
  if (bias.stride == 1 && bias.type == FBFFT_FLOAT32) {
    loadPack<float, 8>(static_cast<const float*>(bias.data) + j, b);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) b[q] = bias.data ? loadAny(bias.data, bias.type, (j + q) * bias.stride) : 0.f;
  }
}

// Eight neighbouring results of row i, or the `count` of them that are inside, from their sums: all of them at once
// where neighbours are neighbours in memory, else one by one.
template <class T, class Eight, class One>
__device__ __forceinline__ void finish(const Epilogue& e, long i, long j, long count, Eight eight, One one) {
  T* const out = static_cast<T*>(e.out.data) + i * e.out.row + j * e.out.col;
  const T* const residual = static_cast<const T*>(e.residual.data) + i * e.residual.row + j * e.residual.col;
  T* const kept = static_cast<T*>(e.z.data) + i * e.z.row + j * e.z.col;
  if (e.dense && count >= 8) {
    float z[8];
    eight(z);
    float b[8];
    loadBias(e.bias, j, b);
#pragma unroll
    for (int v = 0; v < 8; ++v) z[v] += b[v];
    if (e.z.data) storePack<T, 8>(kept, z);
    activateAll(z, e.activation);
    if (e.residual.data) {
      float r[8];
      loadPack<T, 8>(residual, r);
#pragma unroll
      for (int v = 0; v < 8; ++v) z[v] += r[v];
    }
    storePack<T, 8>(out, z);
    return;
  }
#pragma unroll 1
  for (int v = 0; v < min(count, 8L); ++v) {
    const float z = one(v) + lineOr(e.bias, j + v, 0.f);
    if (e.z.data) kept[v * e.z.col] = (T)z;
    float y = activate(z, e.activation);
    if (e.residual.data) y += (float)residual[v * e.residual.col];
    out[v * e.out.col] = (T)y;
  }
}

// A wave's sums, RM x RN blocks of 16 x 16 (a lane: four neighbours of row lane % 16 of each), go through its own
// `space` in LDS, TURN rows of blocks at a time, so that a lane then has eight neighbouring results, and rows of them
// are whole lines.  The 16-byte words of a row are permuted, so that 16 rows' writes take all banks.
// (ARGS: with M and N, the results' extents, and e, their epilogue.)
template <class T, int RM, int RN, int TURN, class ARGS>
__device__ __forceinline__ void leave(const ARGS& g, long range, long m0, long n0, const floatx4 (&sum)[RM][RN], char* space) {
  constexpr int COLS = RN * 16, WORDS = COLS / 4, LANES = COLS / 8, MASK = WORDS < 16 ? WORDS - 1 : 15;
  const int lane = threadIdx.x % 64;
#pragma unroll
  for (int i0 = 0; i0 < RM; i0 += TURN) {
    waveExchange();
#pragma unroll
    for (int i = 0; i < TURN; ++i)
#pragma unroll
      for (int j = 0; j < RN; ++j) {
        const int row = 16 * i + lane % 16, word = (4 * j + lane / 16) ^ (row & MASK);
        *reinterpret_cast<floatx4*>(space + (row * WORDS + word) * 16) = sum[i0 + i][j];
      }
    waveExchange();
    const long n = n0 + lane % LANES * 8, count = g.N - n;
    const int word = lane % LANES * 2;
    auto eight = [&](int row, float(&v)[8]) __attribute__((always_inline)) {
      const char* const line = space + row * (WORDS * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const floatx4 q = *reinterpret_cast<const floatx4*>(line + ((word + h) ^ (row & MASK)) * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * h + k] = q[k];
      }
    };
    auto one = [&](int row, int v) __attribute__((always_inline)) {
      return *reinterpret_cast<const float*>(space + row * (WORDS * 16) + ((word + v / 4) ^ (row & MASK)) * 16 + v % 4 * 4);
    };
    constexpr int ROWS = 64 / LANES, TIMES = 16 * TURN / ROWS, AT_ONCE = TIMES < 4 ? TIMES : 4;
    const long m1 = m0 + 16 * i0;
    if (g.e.parts) {
#pragma unroll 1
      for (int row = lane / LANES; row < 16 * TURN; row += ROWS) {
        const long m = m1 + row;
        if (m >= g.M || count <= 0) continue;
        float* const to = g.e.parts + (range * g.M + m) * g.N + n;
        if (count >= 8) {
          float v[8];
          eight(row, v);
          storePack<float, 8>(to, v);
        } else {
#pragma unroll 1
          for (int v = 0; v < count; ++v) to[v] = one(row, v);
        }
      }
    } else if (g.e.dense && n0 + COLS <= g.N) {
      // whole rows: a few rows' residuals on their way at once (one by one, each of them waits for memory: 8192 x 8192 x
      // 2048 with residual and preactivation 333 us instead of 298-309)
      float bias[8];
      loadBias(g.e.bias, n, bias);
      const T* const residual = static_cast<const T*>(g.e.residual.data);
#pragma unroll 1
      for (int t = 0; t < TIMES; t += AT_ONCE) {
        typename Pack<T, 8>::type r[AT_ONCE];
        if (residual)
#pragma unroll
          for (int q = 0; q < AT_ONCE; ++q)
            r[q] = *reinterpret_cast<const typename Pack<T, 8>::type*>(
                residual + min(m1 + lane / LANES + (t + q) * ROWS, g.M - 1) * g.e.residual.row + n);
#pragma unroll
        for (int q = 0; q < AT_ONCE; ++q) {
          const int row = lane / LANES + (t + q) * ROWS;
          const long m = m1 + row;
          if (m >= g.M) break;
          float z[8];
          eight(row, z);
#pragma unroll
          for (int v = 0; v < 8; ++v) z[v] += bias[v];
          if (g.e.z.data) storePack<T, 8>(static_cast<T*>(g.e.z.data) + m * g.e.z.row + n, z);
          activateAll(z, g.e.activation);
          if (residual)
#pragma unroll
            for (int v = 0; v < 8; ++v) z[v] += (float)r[q][v];
          storePack<T, 8>(static_cast<T*>(g.e.out.data) + m * g.e.out.row + n, z);
        }
      }
    } else {
#pragma unroll 1
      for (int row = lane / LANES; row < 16 * TURN; row += ROWS) {
        const long m = m1 + row;
        if (m >= g.M || count <= 0) continue;
        finish<T>(
            g.e, m, n, count, [&](float(&v)[8]) __attribute__((always_inline)) { eight(row, v); },
            [&](int v) __attribute__((always_inline)) { return one(row, v); });
      }
    }
  }
}

// Where a workgroup's tile lies.  Neighbouring tiles go to one XCD (workgroups are dealt out to the eight in turn), in
// strips of four rows of tiles, so that those that run together share lines of both operands in its L2.  `turn`: by so much
// further XCDs, for what else than a tile a grid's workgroups differ in, so that a few tiles' ranges and matrices go to all eight.
template <int BM, int BN>
struct Tile {
  long m0, n0;
  bool any;

  __device__ __forceinline__ Tile(long M, long N, int turn = 0) {
    constexpr int tall = 4;
    const int across = (int)((N + BN - 1) / BN), down = (int)((M + BM - 1) / BM), total = across * down, per = (total + 7) / 8;
    int tile = ((int)blockIdx.x + turn) % 8 * per + (int)blockIdx.x / 8;
    any = (int)blockIdx.x / 8 < per && tile < total;
    const int strip = tile / (tall * across), height = max(1, min(tall, down - strip * tall));
    tile -= strip * tall * across;
    m0 = (long)(strip * tall + tile % height) * BM;
    n0 = (long)(tile / height) * BN;
  }
};

typedef __attribute__((address_space(3))) void* LdsAddress;

// One step of an operand on its way to LDS, in the words of linear_step.h.  The buffer's own bounds are of no use for what
// lies behind an operand (they hold for one length only, while lines of a step end in different places): a word is read
// where its row and its k are inside.
template <int ROWS, int DEEP, bool KC, int WAVES>
struct Direct : StepWords<ROWS, DEEP, KC, WAVES> {
  typedef StepWords<ROWS, DEEP, KC, WAVES> Places;
  using Places::loads, Places::permuted;
  typename Places::Word word[loads];  // of each load
  const char* base;                   // the next step's first word
  long advance;                       // bytes from a step to the next

  // rows: from the tile's first, inside
  __device__ __forceinline__ void setup(const void* first, long step, long rows) {
#pragma unroll
    for (int i = 0; i < loads; ++i) word[i] = Places::wordOf(threadIdx.x, i, step, rows);
    base = static_cast<const char*>(first);
    advance = KC ? DEEP * 2 : DEEP * 2 * step;
  }

  // Load i of the next step, of which `left` k are inside (perhaps none): what is not inside reads as zeros.
  __device__ __forceinline__ void load(int i, int left, char* space) const {
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, kReach, 0x00020000);
    char* const to = space + (threadIdx.x / 64 * loads + i) * 1024;
    const unsigned place = Places::placeOf(word[i], left);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (LdsAddress)to, 16, place, 0, 0, 0);
  }

  // Where this lane's part of the fragments from row `first` (a multiple of 16 times their number) lies in a step, and
  // fragment i of half h: eight k from 32 h + 8 (lane / 16) of row first + 16 i + lane % 16.
  static __device__ __forceinline__ int laneAt(int first) {
    const int lane = threadIdx.x % 64;
    if (KC) {
      const int line = first + lane % 16;
      return line * (DEEP * 2) + permuted(line, lane / 16) * 16;
    }
    const int line = lane / 16 * 8 + lane % 16 / 4, row = first + lane % 4 * 4;
    return line * (ROWS * 2) + permuted(line, row / 8) * 16 + row % 8 * 2;
  }
  static __device__ __forceinline__ uintx4 fragment(const char* step, int lane, int h, int i) {
    if (KC) return *reinterpret_cast<const uintx4*>(step + (lane ^ h * 64) + i * (16 * DEEP * 2));
    uintx4 f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      // (four and 32 lines on, the words of a line are permuted the same way)
      const char* const from = step + (lane ^ i * 32) + (32 * h + 4 * q) * (ROWS * 2);
      const uintx2 u = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (__attribute__((address_space(3))) shortx4*)const_cast<char*>(from)));
      f[2 * q] = u[0];
      f[2 * q + 1] = u[1];
    }
    return f;
  }
};

// Waits until at most PENDING of this wave's loads are on their way, and its reads of LDS have arrived, then for the
// workgroup's other waves.  (In instructions that the compiler counts with, so that it adds no waits of its own.)
template <int PENDING>
__device__ __forceinline__ void arrive() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(PENDING % 16 | 0x70 | PENDING / 16 << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Results from the sums of `ranges` ranges of k, in their order (of none: from 0).  A lane: eight neighbours.
template <class T>
__global__ __launch_bounds__(256) void joinWords(Epilogue e, long M, long N, int ranges) {
  const long words = N / 8, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= M * words) return;
  const long m = i / words, n = i % words * 8;
  const float* const from = e.parts + m * N + n;
  auto eight = [&](float(&z)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 8; ++q) z[q] = 0.f;
#pragma unroll 4
    for (int r = 0; r < ranges; ++r) {
      float v[8];
      loadPack<float, 8>(from + r * M * N, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] += v[q];
    }
  };
  auto one = [&](int v) __attribute__((always_inline)) {
    float z = 0.f;
    for (int r = 0; r < ranges; ++r) z += from[r * M * N + v];
    return z;
  };
  finish<T>(e, m, n, 8, eight, one);
}

// The same, a result to a lane, or to GROUPS of them that take the ranges in turn: for few results, or rows that no
// words fit.
template <class T, int GROUPS>
__global__ __launch_bounds__(256) void joinRanges(Epilogue e, long M, long N, int ranges) {
  constexpr int SIDE = 256 / GROUPS;
  __shared__ float sums[256];
  const int group = threadIdx.x / SIDE;
  const long i = (long)blockIdx.x * SIDE + threadIdx.x % SIDE;
  float z = 0.f;
  if (i < M * N)
#pragma unroll 8
    for (int r = group; r < ranges; r += GROUPS) z += e.parts[r * M * N + i];
  if (GROUPS > 1) {
    sums[threadIdx.x] = z;
    __syncthreads();
    if (group > 0) return;
    z = 0.f;
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) z += sums[q * SIDE + threadIdx.x];
  }
  if (i >= M * N) return;
  const long m = i / N, n = i - m * N;
  z += lineOr(e.bias, n, 0.f);
  if (e.z.data) static_cast<T*>(e.z.data)[m * e.z.row + n * e.z.col] = (T)z;
  z = activate(z, e.activation);
  if (e.residual.data) z += (float)static_cast<const T*>(e.residual.data)[m * e.residual.row + n * e.residual.col];
  static_cast<T*>(e.out.data)[m * e.out.row + n * e.out.col] = (T)z;
}

// How the sums of `ranges` ranges become results: words of eight, or a lane or eight to a result.
struct JoinPlan {
  int kind;  // 0: words; 1, 8: joinRanges' groups
  long blocks;
};
JoinPlan joinOf(bool dense, long M, long N, long ranges) {
  if (N % 8 == 0 && dense && M * N >= 1 << 18) return {0, (M * (N / 8) + 255) / 256};
  return ranges < 8 ? JoinPlan{1, (M * N + 255) / 256} : JoinPlan{8, (M * N + 31) / 32};
}

template <class T>
void launchJoin(const JoinPlan& plan, const Epilogue& e, long M, long N, int ranges, hipStream_t s) {
  const dim3 grid((unsigned)plan.blocks);
  if (plan.kind == 0)
    joinWords<T><<<grid, 256, 0, s>>>(e, M, N, ranges);
  else if (plan.kind == 1)
    joinRanges<T, 1><<<grid, 256, 0, s>>>(e, M, N, ranges);
  else
    joinRanges<T, 8><<<grid, 256, 0, s>>>(e, M, N, ranges);
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace
}  // namespace fbfft_amd
