// Rows times a weight matrix with bias, activation and residual, and its gradients.
//
//   forward    z = x w^T + bias,  y = activation(z) + residual
//   backward   dz = dy activation'(z);  dx = dz w,  dw = dz^T x,  dbias = sum of dz's rows
//
// All three products are sum_k A[i][k] B[j][k] for operands whose unit stride lies along k or along the row, on the
// 16-bit matrix instructions with fp32 sums.  float32 operands are cut into three bf16 pieces of 8 bits each (exactly:
// the pieces are the leading, middle and last bits), of whose nine products the six largest are summed; what is left
// out is below 2^-21 of a product (the second piece is below 2^-7 of a value, the third below 2^-15), 2^-24 on average.
#include "linear_step.h"
#include "operators.h"

#include <algorithm>

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

struct ProductArgs {
  Matrix a, b;
  long M, N, K, range;  // k per range
  Epilogue e;
};

__device__ __forceinline__ floatx4 multiply(uintx4 a, uintx4 b, floatx4 c, half16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 multiply(uintx4 a, uintx4 b, floatx4 c, brain16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(brainx8, a), __builtin_bit_cast(brainx8, b), c, 0, 0, 0);
}

template <class T>
struct Pieces {
  static constexpr int count = 1;
  typedef T type;
};
template <>
struct Pieces<float> {
  static constexpr int count = 3;
  typedef brain16 type;
};

// the leading 16 bits of each of two floats, one above the other
__device__ __forceinline__ unsigned leading(float low, float high) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, high), __builtin_bit_cast(unsigned, low), 0x07060302);
}
__device__ __forceinline__ float withoutLeading(float v) {
  return v - __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & 0xFFFF0000u);
}

constexpr int kStep = 32;  // k of a step

// One step of an operand, ROWS rows by kStep of k, [row][k] or [k][row], as 16-bit pieces in LDS: 16-byte words that
// are permuted so that the lanes of a fragment's read spread over the banks.  KC: k is contiguous.
template <class T, bool KC, int ROWS>
struct Stage {
  static constexpr int per = 16 / sizeof(T), words = ROWS * kStep / per / 256, pieceBytes = ROWS * kStep * 2;
  typename Pack<T, per>::type v[words];
  const T* from[words];  // of each word at k = 0
  bool whole[words];     // its elements are neighbours, and inside

  static __device__ __forceinline__ int lineOf(int i) { return (threadIdx.x + 256 * i) / ((KC ? kStep : ROWS) / per); }
  static __device__ __forceinline__ int firstOf(int i) { return (threadIdx.x + 256 * i) % ((KC ? kStep : ROWS) / per) * per; }

  __device__ __forceinline__ void setup(const Matrix& m, long row0, long rows) {
#pragma unroll
    for (int i = 0; i < words; ++i) {
      const long row = row0 + (KC ? lineOf(i) : firstOf(i)), k = KC ? firstOf(i) : lineOf(i);
      // (rows behind the last: the last again, whose results nobody takes)
      from[i] = static_cast<const T*>(m.data) + min(row, rows - 1) * m.row + k * m.col;
      whole[i] = KC ? m.col == 1 : m.row == 1 && row + per <= rows;
    }
  }

  __device__ __forceinline__ void load(const Matrix& m, long row0, long rows, long k0, long end) {
#pragma unroll
    for (int i = 0; i < words; ++i) {
      const long k = k0 + (KC ? firstOf(i) : lineOf(i));
      const T* const p = from[i] + k0 * m.col;
      if (whole[i] && (KC ? k + per <= end : k < end)) {
        v[i] = *reinterpret_cast<const typename Pack<T, per>::type*>(p);
      } else {
        const long left = KC ? end - k : rows - row0 - firstOf(i), step = KC ? m.col : m.row;
        const bool some = KC || k < end;
#pragma unroll
        for (int j = 0; j < per; ++j) v[i][j] = some && j < left ? p[j * step] : (T)0.f;
      }
    }
  }

  // where element `at` (a multiple of `per`) of line `line` lies: bytes
  static __device__ __forceinline__ int place(int line, int at) {
    if (KC) return line * 64 + ((at / 8 ^ line / 4 % 4) * 16) + at % 8 * 2;
    const int spread = line % 4 + line / 8 % 2 * 4;
    return line * (ROWS * 2) + ((at / 16 ^ (ROWS >= 128 ? spread : spread % 4)) * 32) + at % 16 * 2;
  }

  __device__ __forceinline__ void store(char* space) const {
#pragma unroll
    for (int i = 0; i < words; ++i) {
      char* const to = space + place(lineOf(i), firstOf(i));
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uintx4*>(to) = __builtin_bit_cast(uintx4, v[i]);
      } else {
        float r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = v[i][j];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          *reinterpret_cast<uintx2*>(to + p * pieceBytes) = uintx2{leading(r[0], r[1]), leading(r[2], r[3])};
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] = withoutLeading(r[j]);
        }
      }
    }
  }

  // eight k of row `row` + lane % 16: k from 8 (lane / 16)
  static __device__ __forceinline__ uintx4 fragment(const char* space, int row) {
    const int lane = threadIdx.x % 64;
    if (KC) return *reinterpret_cast<const uintx4*>(space + place(row + lane % 16, lane / 16 * 8));
    // the transposing read: of sixteen lanes, lane l gives the address of four rows (l % 4) of k (l / 4) and gets four k of row l
    const int k = lane / 16 * 8 + lane % 16 / 4, at = row + lane % 4 * 4;
    uintx4 f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* const q = space + place(k + 4 * h, at);
      const uintx2 u = __builtin_bit_cast(
          uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)const_cast<char*>(q)));
      f[2 * h] = u[0];
      f[2 * h + 1] = u[1];
    }
    return f;
  }
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
template <class T, int RM, int RN, int TURN>
__device__ __forceinline__ void leave(const ProductArgs& g, long range, long m0, long n0, const floatx4 (&sum)[RM][RN], char* space) {
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
// strips of four rows of tiles, so that those that run together share lines of both operands in its L2.
template <int BM, int BN>
struct Tile {
  long m0, n0;
  bool any;

  __device__ __forceinline__ Tile(long M, long N) {
    constexpr int tall = 4;
    const int across = (int)((N + BN - 1) / BN), down = (int)((M + BM - 1) / BM), total = across * down, per = (total + 7) / 8;
    int tile = (int)blockIdx.x % 8 * per + (int)blockIdx.x / 8;
    any = (int)blockIdx.x / 8 < per && tile < total;
    const int strip = tile / (tall * across), height = max(1, min(tall, down - strip * tall));
    tile -= strip * tall * across;
    m0 = (long)(strip * tall + tile % height) * BM;
    n0 = (long)(tile / height) * BN;
  }
};

// A workgroup: BM x BN results over one range of k; a wave WM x WN of them.  B's rows lie along the rows of the
// matrix instruction, so that a lane ends with four neighbouring results of one row.  The next step's words are in
// registers while this one's pieces are multiplied.  67712 x 192 x 64 fp32 with GELU, residual and preactivation: 30 us for
// 104 MB, 3.5 TB/s, where cutting operands into pieces, LDS and memory take turns; 5330 x 1920 x 208: 43 us, 98 TFLOP/s of
// fp32, six times that in matrix instructions (two steps ahead in registers: 34 and more us instead of 30; rows of x straight
// from memory: 36.5).  The bound of three workgroups to a compute unit leaves the float32 kernels of 128 x 64 168 registers, and
// 12 to 24 values of a lane in scratch memory.
template <class T, bool AK, bool BK, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(256, BM * BN == 8192 ? 3 : 1) void product(ProductArgs g) {
  typedef typename Pieces<T>::type P;
  typedef Stage<T, AK, BM> A;
  typedef Stage<T, BK, BN> B;
  constexpr int PIECES = Pieces<T>::count, RM = WM / 16, RN = WN / 16, BYTES = PIECES * (A::pieceBytes + B::pieceBytes);
  constexpr int SHARE = BYTES / 4 > WN * 64 ? BYTES / 4 : WN * 64;  // of LDS, to a wave
  static_assert(BM / WM * (BN / WN) == 4, "four waves");
  __shared__ __attribute__((aligned(16))) char space[4 * SHARE];
  char *const sa = space, *const sb = space + PIECES * A::pieceBytes;
  const int wave = threadIdx.x / 64, wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
  const Tile<BM, BN> tile(g.M, g.N);
  if (!tile.any) return;
  const long first = blockIdx.y * g.range, end = min(first + g.range, g.K);

  floatx4 sum[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  A a;
  B b;
  a.setup(g.a, tile.m0, g.M);
  b.setup(g.b, tile.n0, g.N);
  a.load(g.a, tile.m0, g.M, first, end);
  b.load(g.b, tile.n0, g.N, first, end);
  for (long k = first; k < end; k += kStep) {
    __syncthreads();
    a.store(sa);
    b.store(sb);
    __syncthreads();
    if (k + kStep < end) {
      a.load(g.a, tile.m0, g.M, k + kStep, end);
      b.load(g.b, tile.n0, g.N, k + kStep, end);
    }
    uintx4 fb[PIECES][RN];
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int j = 0; j < RN; ++j) fb[p][j] = B::fragment(sb + p * B::pieceBytes, wn + 16 * j);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      uintx4 fa[PIECES];
#pragma unroll
      for (int p = 0; p < PIECES; ++p) fa[p] = A::fragment(sa + p * A::pieceBytes, wm + 16 * i);
      // the products of pieces p and q, the smallest first
#pragma unroll
      for (int order = PIECES - 1; order >= 0; --order)
#pragma unroll
        for (int p = 0; p <= order; ++p)
#pragma unroll
          for (int j = 0; j < RN; ++j) sum[i][j] = multiply(fb[order - p][j], fa[p], sum[i][j], P());
    }
  }
  __syncthreads();
  constexpr int FIT = SHARE / (WN * 64), TURN = FIT >= RM ? RM : FIT >= 2 ? 2 : 1;  // blocks of rows
  static_assert(FIT > 0 && RM % TURN == 0, "a wave's share of LDS holds whole rows of blocks");
  leave<T, RM, RN, TURN>(g, blockIdx.y, tile.m0 + wm, tile.n0 + wn, sum, space + wave * SHARE);
}

// ---- operands of 16 bits that go straight from memory to LDS ----

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

// A workgroup: BM x BN results over one range of k, a wave WM x WN of them.  LDS holds the operands of DEPTH steps of
// DEEP k; the fragments of the next 32 k are on their way from LDS while a wave multiplies those of these, and waves
// meet once a step.  Steps of 64 k take rows whose k are contiguous in whole lines of 128 bytes (8192 x 8192 x 2048, us:
// 268, steps of 32: 307); where rows are contiguous instead, more and shorter steps are better (both: 283, 331).  Bound by the
// matrix instructions and the reads of LDS between them: 8192 x 8192 x 2048 bf16 251 us, 1.09 PFLOP/s.
template <class T, bool AK, bool BK, int BM, int BN, int WM, int WN, int DEEP, int DEPTH>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void productDirect(ProductArgs g) {
  constexpr int WAVES = BM / WM * (BN / WN), RM = WM / 16, RN = WN / 16;
  typedef Direct<BM, DEEP, AK, WAVES> A;
  typedef Direct<BN, DEEP, BK, WAVES> B;
  constexpr int STEP = A::bytes + B::bytes, LOADS = A::loads + B::loads;
  __shared__ __attribute__((aligned(1024))) char space[DEPTH * STEP];
  const int wave = threadIdx.x / 64;
  const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
  const Tile<BM, BN> tile(g.M, g.N);
  if (!tile.any) return;
  const long m0 = tile.m0, n0 = tile.n0, first = blockIdx.y * g.range, end = min(first + g.range, g.K);

  A a;
  B b;
  a.setup(static_cast<const T*>(g.a.data) + m0 * g.a.row + first * g.a.col, AK ? g.a.row : g.a.col, g.M - m0);
  b.setup(static_cast<const T*>(g.b.data) + n0 * g.b.row + first * g.b.col, BK ? g.b.row : g.b.col, g.N - n0);

  floatx4 sum[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) sum[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

  auto load = [&](int q, int left, char* to) __attribute__((always_inline)) {
    if (q < A::loads)
      a.load(q, left, to);
    else
      b.load(q - A::loads, left, to + A::bytes);
  };
  int left = (int)(end - first);  // k that are not on their way yet
  auto loaded = [&]() __attribute__((always_inline)) {
    a.base += a.advance;
    b.base += b.advance;
    left -= DEEP;
  };
  // (behind the last step too, without a word, so that as many loads are always on their way)
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
    for (int q = 0; q < LOADS; ++q) load(q, left, space + d * STEP);
    loaded();
  }
  const int laneA = A::laneAt(wm), laneB = B::laneAt(wn);
  uintx4 fa[2][RM], fb[2][RN];
  constexpr int READS = RM + RN;
  auto read = [&](int q, int set, const char* from, int half) __attribute__((always_inline)) {
    if (q < RN)
      fb[set][q] = B::fragment(from + A::bytes, laneB, half, q);
    else
      fa[set][q - RN] = A::fragment(from, laneA, half, q - RN);
  };
  auto row = [&](int set, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < RN; ++j) sum[i][j] = multiply(fb[set][j], fa[set][i], sum[i][j], T());
  };
  // Reads and loads go between matrix instructions a few at a time: a wave waits where it issues them (8192 x 8192 x
  // 2048, us: 251, all reads first 268).  Not the transposing reads, which the compiler holds back until none of the wave's loads
  // is on its way: all of them first (280, between matrix instructions 328).  Behind every barrier of those forms stands
  // that wait, so of their four steps in LDS no more than one is in flight while a wave reads.
  constexpr bool SPREAD = AK && BK;
  auto reads = [&](int i, int set, const char* from, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < READS; ++q)
      if (SPREAD ? q >= i * READS / RM && q < (i + 1) * READS / RM : i == 0) read(q, set, from, half);
  };
  constexpr int HALVES = DEEP / 32;
  static_assert(DEPTH * HALVES % 2 == 0, "two sets of fragments, in turn");
  arrive<(DEPTH - 1) * LOADS>();
#pragma unroll
  for (int q = 0; q < READS; ++q) read(q, 0, space, 0);
  auto round = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int set = d * HALVES % 2, last = (set + HALVES - 1) % 2;
      if constexpr (HALVES == 2) {
#pragma unroll
        for (int i = 0; i < RM; ++i) {
          reads(i, last, space + d * STEP, 1);
          row(set, i);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // the next step's operands are there, and this one's place is free: every wave has its fragments
      arrive<(DEPTH - 2) * LOADS>();
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        reads(i, last ^ 1, space + (d + 1) % DEPTH * STEP, 0);
        row(last, i);
#pragma unroll
        for (int q = i * LOADS / RM; q < (i + 1) * LOADS / RM; ++q) load(q, left, space + d * STEP);
        __builtin_amdgcn_sched_barrier(0);
      }
      loaded();
      if (left <= -DEPTH * DEEP) return false;  // that was the last step
    }
    return true;
  };
  while (round()) {
  }

  // (the loads requested behind the last step write zeros to LDS, which the results now go through)
  arrive<0>();
  constexpr int SHARE = DEPTH * STEP / WAVES, FIT = SHARE / (WN * 64);  // of LDS, to a wave; blocks of rows
  constexpr int TURN = FIT >= RM ? RM : FIT >= 4 ? 4 : FIT >= 2 ? 2 : 1;
  static_assert(FIT > 0 && RM % TURN == 0, "a wave's share of LDS holds whole rows of blocks");
  leave<T, RM, RN, TURN>(g, blockIdx.y, m0 + wm, n0 + wn, sum, space + wave * SHARE);
}

// ---- a few rows: as fast as the weights can be read ----

constexpr int kFew = 16;

// Eight neighbouring k of a row from memory to the matrix instructions, as pieces.
template <class T>
struct Slice {
  static constexpr int PIECES = Pieces<T>::count;
  typename Pack<T, 8>::type v;

  __device__ __forceinline__ void load(const T* row, long k, long end) {
    if (k + 8 <= end) {
      v = *reinterpret_cast<const typename Pack<T, 8>::type*>(row + k);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < end ? row[k + j] : (T)0.f;
    }
  }
  __device__ __forceinline__ void pieces(uintx4 (&to)[PIECES]) const {
    if constexpr (PIECES == 1) {
      to[0] = __builtin_bit_cast(uintx4, v);
    } else {
      float r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = v[j];
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        to[p] = uintx4{leading(r[0], r[1]), leading(r[2], r[3]), leading(r[4], r[5]), leading(r[6], r[7])};
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = withoutLeading(r[j]);
      }
    }
  }
};

// Up to 16 rows of x.  A workgroup: 16 rows of w, its waves a range of k each, straight from memory to the matrix
// instructions (rows of x behind the last are the last again, and nobody takes their results); their sums meet in LDS.
// Bound by reading w: 16 x 4096 x 8192 bf16 17.8 us for 67 MB, 3.8 TB/s; 1 x 2048 x 2048 4.4 us, most of it the launch and
// one trip to memory.
template <class T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void fewRows(ProductArgs g) {
  typedef typename Pieces<T>::type P;
  constexpr int PIECES = Pieces<T>::count, AHEAD = sizeof(T) == 2 ? 8 : 4;
  __shared__ float sums[WAVES][256];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const long n0 = (long)blockIdx.x * 16;
  const T* const w = static_cast<const T*>(g.b.data) + min(n0 + lane % 16, g.N - 1) * g.b.row;
  const T* const x = static_cast<const T*>(g.a.data) + min((long)lane % 16, g.M - 1) * g.a.row;
  const long share = (g.K + WAVES * 32 - 1) / (WAVES * 32) * 32, first = wave * share, end = min(first + share, g.K);
  floatx4 sum{0.f, 0.f, 0.f, 0.f};
  for (long k0 = first; k0 < end; k0 += AHEAD * 32) {
    Slice<T> sw[AHEAD], sx[AHEAD];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const long k = k0 + 32 * s + lane / 16 * 8;
      sw[s].load(w, k, end);
      sx[s].load(x, k, end);
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      uintx4 pw[PIECES], px[PIECES];
      sw[s].pieces(pw);
      sx[s].pieces(px);
#pragma unroll
      for (int order = PIECES - 1; order >= 0; --order)
#pragma unroll
        for (int p = 0; p <= order; ++p) sum = multiply(pw[order - p], px[p], sum, P());
    }
  }
  // (lane: row lane % 16 of x, four rows of w)
#pragma unroll
  for (int v = 0; v < 4; ++v) sums[wave][lane % 16 * 16 + lane / 16 * 4 + v] = sum[v];
  __syncthreads();
  const long m = threadIdx.x / 16, n = n0 + threadIdx.x % 16;
  if (threadIdx.x >= 256 || m >= g.M || n >= g.N) return;
  float z = lineOr(g.e.bias, n, 0.f);
#pragma unroll
  for (int q = 0; q < WAVES; ++q) z += sums[q][threadIdx.x];
  if (g.e.z.data) static_cast<T*>(g.e.z.data)[m * g.e.z.row + n * g.e.z.col] = (T)z;
  z = activate(z, g.e.activation);
  if (g.e.residual.data) z += (float)static_cast<const T*>(g.e.residual.data)[m * g.e.residual.row + n * g.e.residual.col];
  static_cast<T*>(g.e.out.data)[m * g.e.out.row + n * g.e.out.col] = (T)z;
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

// Rows of dz that a workgroup sums: all of a few, whose sums are then the bias's gradient (60 x 64 x 128 f32: all three
// gradients 17.7 us, in two parts that are joined 20.3), else 32, four for a lane at once (of 64: 5952 x 64 x 800 f16 40.8 us
// instead of 37.5).
constexpr long kBiasRows = 32, kBiasFew = 64;
inline long biasRows(long M) { return M <= kBiasFew ? std::max(M, 1L) : kBiasRows; }

// dz = dy activation'(z), dense, and its columns' sums over `rows` rows each, or, of all rows, the bias's gradient.  A
// workgroup: 32 words of VEC columns, eight rows of lanes.  (All workgroups along x, `across` of them to a part of the
// rows: the other axes count to 65535 only, fewer than the parts of 32 rows from 2097121 rows on.)  dz is rounded to the
// operands' type, which the matrix instructions take, after its sum: what a program does whose activation returns a gradient of
// that type.  It costs gradients half again of what rounding them costs (4096 x 1024 x 4096 bf16: 2.35e-3 from the sums in 64 bits
// instead of 1.66e-3); two pieces of dz would keep it and double both products.
template <class T, int VEC>
__global__ __launch_bounds__(256) void preactivationGradient(Matrix dy, Matrix z, T* dz, float* parts, Line bias, long M, long N,
                                                             int activation, long rows, Divisor across) {
  typedef typename Pack<T, VEC>::type Word;
  constexpr int AHEAD = 4;
  __shared__ float sums[8][32 * VEC];
  const int column = threadIdx.x % 32, r = threadIdx.x / 32, part = quotient(blockIdx.x, across);
  const int block = blockIdx.x - part * (int)across.value;
  const long first = ((long)block * 32 + column) * VEC, m0 = part * rows, end = min(m0 + rows, M);
  // (the last word of a row ends with it, and repeats what the one before it has: N is no less than a word)
  const long n = min(first, N - VEC);
  const int repeats = (int)min(first - n, (long)VEC);
  auto load = [&](const Matrix& from, long m) __attribute__((always_inline)) {
    return *reinterpret_cast<const Word*>(static_cast<const T*>(from.data) + min(m, end - 1) * from.row + n * from.col);
  };
  auto unpacked = [&](const Word& w, float(&v)[VEC]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (VEC == 1)
        v[j] = (float)w;
      else
        v[j] = (float)w[j];
    }
  };
  float sum[VEC] = {};
  if (repeats < VEC)
    for (long m = m0 + r; m < end; m += 8 * AHEAD) {
      Word wg[AHEAD], wz[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        wg[q] = load(dy, m + 8 * q);
        if (activation != FBFFT_ACTIVATION_NONE) wz[q] = load(z, m + 8 * q);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        if (m + 8 * q >= end) break;
        float v[VEC], a[VEC];
        unpacked(wg[q], v);
        if (activation != FBFFT_ACTIVATION_NONE) {
          unpacked(wz[q], a);
          slopeAll(a, v, activation);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] += v[j];
        if (dz) storePack<T, VEC>(dz + (m + 8 * q) * N + n, v);
      }
    }
  if (!parts && !bias.data) return;
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    if (j >= repeats) sums[r][column * VEC + j - repeats] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    const long at = (long)block * 32 * VEC + i;
    if (at >= N) continue;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) v += sums[q][i];
    if (parts)
      parts[part * N + at] = v;
    else
      storeAny(bias.data, bias.type, at * bias.stride, v);
  }
}

// A workgroup: eight columns, 32 lanes to each.
__global__ __launch_bounds__(256) void biasGradient(const float* parts, Line out, long N, long count) {
  __shared__ float sums[32][8];
  const int column = threadIdx.x % 8, slice = threadIdx.x / 8;
  const long n = (long)blockIdx.x * 8 + column;
  float sum = 0.f;
  if (n < N)
#pragma unroll 4
    for (long r = slice; r < count; r += 32) sum += parts[r * N + n];
  sums[slice][column] = sum;
  __syncthreads();
  if (slice > 0 || n >= N) return;
  sum = 0.f;
#pragma unroll
  for (int q = 0; q < 32; ++q) sum += sums[q][column];
  storeAny(out.data, out.type, n * out.stride, sum);
}

long ceilDivLong(long a, long b) { return (a + b - 1) / b; }
size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// ---- what runs ----

// The kernel of a product, the rows and columns of its tile and the ranges that k is cut into.
struct ProductPlan {
  enum Kind { Staged, Straight };
  int kind, rows, cols;
  long ranges, range;
};

bool contiguousK(const Matrix& m) { return m.col == 1 || m.row != 1; }

// an operand of 16 bits whose 16-byte words can go straight to LDS: aligned, no word over the end of a line, a tile's
// lines within 31 bits
bool goesStraight(const Matrix& m, long rows, long K) {
  const bool kc = contiguousK(m);
  const long inner = kc ? m.col : m.row, step = kc ? m.row : m.col, line = kc ? K : rows;
  return inner == 1 && line % 8 == 0 && step % 8 == 0 && step >= line && step < (1l << 21) && aligned(m.data, 16);
}

// The kernel with the least expected time, from what each takes for a step of k and for its results (us, measured on
// products of 8192 x 8192 x 2048, 4096 x 1024 x 4096 and single tiles: 256 x 256 tiles, one to a compute unit, 1.75 a step of
// 64 and 12 for the results; 128 x 128 ones 0.85 alone and 1.1 for two; the staged ones' are estimates).  A range of k more
// costs its sums' way to memory and back.  (`together` is a number of the model, no occupancy: registers leave a compute unit
// three float32 workgroups of 64 x 64, or four where k is contiguous in neither operand, and two of 128 x 128, or one where it
// is in one of them only: 128 to 140 registers, 256 to 272.)
// What the estimates cost, on random products timed with every staged tile and 1 to 64 ranges, in times of the fastest's
// (geometric mean of 25 to 30, greatest): float32 x w^T 1.02, 1.26, of odd sizes 1.00, 1.29, dz w 1.05, 1.36, dz^T x 1.06,
// 1.34; 16 bits of odd sizes 0.99, 1.25 and 1.00, 1.25 and 1.04, 1.36 (below 1 by chance).  Farthest off are mostly products that
// tiles of 64 x 64 would serve better.
template <class T>
ProductPlan planOf(long M, long N, long K, bool straight) {
  struct Option {
    int kind, rows, cols, step, together;  // together: workgroups that share a compute unit
    double alone, shared, results;
  };
  static const Option wide[] = {{ProductPlan::Straight, 256, 256, 64, 1, 1.75, 1.75, 12}, {ProductPlan::Straight, 128, 128, 64, 2, 0.85, 1.1, 5}};
  static const Option pieces[] = {{ProductPlan::Staged, 128, 128, 32, 2, 2.0, 2.6, 5}, {ProductPlan::Staged, 128, 64, 32, 3, 1.2, 2.0, 3},
                                  {ProductPlan::Staged, 64, 64, 32, 4, 0.8, 1.6, 2}};
  static const Option staged[] = {{ProductPlan::Staged, 128, 128, 32, 2, 0.9, 1.2, 5}, {ProductPlan::Staged, 128, 64, 32, 3, 0.7, 1.2, 3},
                                  {ProductPlan::Staged, 64, 64, 32, 4, 0.5, 1.0, 2}};
  const Option* const options = straight ? wide : sizeof(T) == 4 ? pieces : staged;
  const int count = straight ? 2 : 3, units = computeUnits();
  ProductPlan best{};
  double least = 0;
  for (int o = 0; o < count; ++o) {
    const Option& a = options[o];
    const long tiles = ceilDivLong(M, a.rows) * ceilDivLong(N, a.cols);
    for (long ranges = 1; ranges <= 64; ranges *= 2) {
      const long range = ceilDivLong(ceilDivLong(K, ranges), a.step) * a.step, used = ceilDivLong(K, range);
      if (ranges > 1 && range < 2 * a.step) break;
      const long groups = tiles * used, slots = (long)units * a.together;
      const double step = groups <= units ? a.alone : a.shared;
      const double rounds = groups <= slots ? 1.0 : std::max((double)groups / slots, groups < 4 * slots ? (double)ceilDivLong(groups, slots) : 1.0);
      double time = rounds * (range / a.step * step + a.results);
      if (used > 1) time += 4.0 + 0.15 * used + (double)M * N * used * 8 / 6e6;
      if (least == 0 || time < least) {
        least = time;
        best = ProductPlan{a.kind, a.rows, a.cols, used, range};
      }
    }
  }
  return best;
}

size_t partsBytes(long M, long N, long K, int type) {
  // (whichever way the operands lie)
  const ProductPlan plans[] = {type == FBFFT_FLOAT32 ? planOf<float>(M, N, K, false) : planOf<half16>(M, N, K, true), planOf<half16>(M, N, K, false)};
  long ranges = plans[0].ranges;
  if (type != FBFFT_FLOAT32) ranges = std::max(ranges, plans[1].ranges);
  return ranges > 1 ? rounded((size_t)ranges * M * N * sizeof(float)) : 0;
}

template <class T, bool AK, bool BK>
void launchProduct(const ProductPlan& plan, long blocks, const ProductArgs& g, hipStream_t s) {
  const dim3 grid((unsigned)blocks, (unsigned)plan.ranges);
  if constexpr (sizeof(T) == 2) {
    if (plan.kind == ProductPlan::Straight) {
      constexpr int DEEP = AK && BK ? 64 : 32, DEPTH = 128 / DEEP;
      if (plan.rows == 256)
        productDirect<T, AK, BK, 256, 256, 128, 64, DEEP, DEPTH><<<grid, 512, 0, s>>>(g);
      else
        productDirect<T, AK, BK, 128, 128, 64, 32, DEEP, DEPTH><<<grid, 512, 0, s>>>(g);
      return;
    }
  }
  if (plan.cols == 128)
    product<T, AK, BK, 128, 128, 64, 64><<<grid, 256, 0, s>>>(g);
  else if (plan.rows == 128)
    product<T, AK, BK, 128, 64, 32, 64><<<grid, 256, 0, s>>>(g);
  else
    product<T, AK, BK, 64, 64, 32, 32><<<grid, 256, 0, s>>>(g);
}

// A product and the launches that it takes, known before anything is enqueued.
template <class T>
struct Product {
  Matrix a, b;
  long M, N, K;
  Epilogue e;
  bool few;          // few rows, straight from memory
  ProductPlan plan;  // else (K = 0: of no ranges)
  JoinPlan join;
  long blocks;

  Product(const Matrix& a, const Matrix& b, long M, long N, long K, const Epilogue& epilogue)
      : a(a), b(b), M(M), N(N), K(K), e(epilogue), few(false), plan{}, join{}, blocks(0) {
    e.dense = e.out.col == 1 && (!e.residual.data || e.residual.col == 1) && (!e.z.data || e.z.col == 1);
    few = K > 0 && M <= kFew && a.col == 1 && b.col == 1;
    if (few) {
      blocks = ceilDivLong(N, 16);
      return;
    }
    if (K > 0) {
      plan = planOf<T>(M, N, K, sizeof(T) == 2 && goesStraight(a, M, K) && goesStraight(b, N, K));
      blocks = (ceilDivLong(M, plan.rows) * ceilDivLong(N, plan.cols) + 7) / 8 * 8;
    }
    if (plan.ranges != 1) join = joinOf(e.dense, M, N, plan.ranges);
  }

  // (as many waves as there are steps of k for)
  int fewLanes() const { return K <= 2048 ? 512 : 1024; }
  bool fits() const {
    return launches(blocks, few ? fewLanes() : plan.kind == ProductPlan::Straight ? 512 : 256) && launches(join.blocks, 256);
  }

  int run(float* parts, hipStream_t s) const {
    ProductArgs g{a, b, M, N, K, few ? K : plan.range, e};
    if (few) {
      if (K <= 2048)
        fewRows<T, 8><<<dim3((unsigned)blocks), 512, 0, s>>>(g);
      else
        fewRows<T, 16><<<dim3((unsigned)blocks), 1024, 0, s>>>(g);
      return launchStatus();
    }
    if (plan.ranges > 1) g.e.parts = parts;
    if (K > 0) {
      const bool ak = contiguousK(a), bk = contiguousK(b);
      if (ak && bk)
        launchProduct<T, true, true>(plan, blocks, g, s);
      else if (ak)
        launchProduct<T, true, false>(plan, blocks, g, s);
      else if (bk)
        launchProduct<T, false, true>(plan, blocks, g, s);
      else
        launchProduct<T, false, false>(plan, blocks, g, s);
    }
    if (plan.ranges != 1) launchJoin<T>(join, g.e, M, N, (int)plan.ranges, s);
    return launchStatus();
  }
};

template <class T>
int forward(const LinearProblem& p, hipStream_t s) {
  const Product<T> y(p.x, p.w, p.M, p.N, p.K, Epilogue{p.y, p.residual, p.z, p.bias, p.activation, false, nullptr});
  return y.fits() ? y.run(static_cast<float*>(p.workspace), s) : FBFFT_UNSUPPORTED_SIZE;
}

template <class T>
int backward(const LinearProblem& p, hipStream_t s) {
  char* space = static_cast<char*>(p.workspace);
  Matrix dz = p.dy;
  const long chunks = ceilDivLong(p.M, biasRows(p.M));
  float* const parts = reinterpret_cast<float*>(space);
  space += rounded((size_t)chunks * p.N * sizeof(float));
  const bool products = p.dx.data || p.dw.data, apart = products && p.activation != FBFFT_ACTIVATION_NONE;
  if (p.activation != FBFFT_ACTIVATION_NONE) {
    if (apart) dz = Matrix{space, p.N, 1};
    space += rounded((size_t)p.M * p.N * sizeof(T));
  }
  constexpr int W = 16 / sizeof(T);
  const bool words = p.N >= W && p.dy.col == 1 && (p.activation == FBFFT_ACTIVATION_NONE || p.z.col == 1);
  const long across = ceilDivLong(p.N, 32 * (words ? W : 1));
  const bool first = p.M > 0 && p.N > 0 && (apart || p.gradBias.data), hasX = p.dx.data && p.M > 0 && p.K > 0;
  const bool hasW = p.dw.data && p.N > 0 && p.K > 0, hasBias = p.gradBias.data && p.N > 0 && chunks != 1;
  const Product<T> dx(dz, Matrix{p.w.data, p.w.col, p.w.row}, p.M, p.K, p.N, Epilogue{p.dx, {}, {}, {}, 0, false, nullptr});
  const Product<T> dw(Matrix{dz.data, dz.col, dz.row}, Matrix{p.x.data, p.x.col, p.x.row}, p.N, p.K, p.M,
                      Epilogue{p.dw, {}, {}, {}, 0, false, nullptr});
  if ((first && !launches(across * chunks, 256)) || (hasBias && !launches(ceilDivLong(p.N, 8), 256)) || (hasX && !dx.fits()) ||
      (hasW && !dw.fits()))
    return FBFFT_UNSUPPORTED_SIZE;
  if (first) {
    const dim3 grid((unsigned)(across * chunks));
    T* const to = apart ? static_cast<T*>(dz.data) : nullptr;
    float* const sums = p.gradBias.data && chunks > 1 ? parts : nullptr;
    const Line bias = chunks > 1 ? Line{} : p.gradBias;
    if (words)
      preactivationGradient<T, W><<<grid, 256, 0, s>>>(p.dy, p.z, to, sums, bias, p.M, p.N, p.activation, biasRows(p.M), divisorOf(across));
    else
      preactivationGradient<T, 1><<<grid, 256, 0, s>>>(p.dy, p.z, to, sums, bias, p.M, p.N, p.activation, biasRows(p.M), divisorOf(across));
  }
  if (hasBias) biasGradient<<<dim3((unsigned)ceilDivLong(p.N, 8)), 256, 0, s>>>(parts, p.gradBias, p.N, p.M > 0 ? chunks : 0);
  int rc = launchStatus();
  if (rc == FBFFT_SUCCESS && hasX) rc = dx.run(reinterpret_cast<float*>(space), s);
  if (rc == FBFFT_SUCCESS && hasW) rc = dw.run(reinterpret_cast<float*>(space), s);
  return rc;
}

}  // namespace

size_t linearWorkspaceBytes(int pass, long M, long K, long N, int type) {
  if (pass == 0) return K > 0 ? partsBytes(M, N, K, type) : 0;
  return rounded((size_t)ceilDivLong(M, biasRows(M)) * N * sizeof(float)) +
         rounded((size_t)M * N * (type == FBFFT_FLOAT32 ? 4 : 2)) + std::max(partsBytes(M, K, N, type), partsBytes(N, K, M, type));
}

int launchLinearForward(const LinearProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return forward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? forward<half16>(p, s) : forward<brain16>(p, s);
}

int launchLinearBackward(const LinearProblem& p, hipStream_t s) {
  if (p.type == FBFFT_FLOAT32) return backward<float>(p, s);
  return p.type == FBFFT_FLOAT16 ? backward<half16>(p, s) : backward<brain16>(p, s);
}

}  // namespace fbfft_amd
