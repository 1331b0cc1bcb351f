// Where the 16-byte words of one step of an operand lie, in memory and in LDS, when they go straight from the one to the
// other (product.h).  Arithmetic only, which a host compiler runs, too.
#pragma once

#include <hip/hip_runtime.h>

namespace fbfft_amd {

inline long ceilDivLong(long a, long b) { return (a + b - 1) / b; }

constexpr unsigned kOutside = 0x80000000u;  // the place of a word that is not there: behind every buffer
constexpr int kReach = 0x7fffffff;          // bytes of a buffer, which ends in front of it

// One step of an operand, ROWS rows by DEEP (32 or 64) of k, in words of eight 16-bit elements.  A wave's load fills 1024
// neighbouring bytes of LDS, so the words are permuted where they are read from memory.  KC: k is contiguous, a line is a
// row, of eight words; else a line is a k, of ROWS / 8.
template <int ROWS, int DEEP, bool KC, int WAVES>
struct StepWords {
  static constexpr int words = DEEP * ROWS / 8, loads = words / 64 / WAVES, perLine = KC ? DEEP / 8 : ROWS / 8;
  static constexpr int bytes = words * 16;
  static_assert(loads * 64 * WAVES == words, "whole loads");

  // which word lies where: KC: so that 16 rows of one k take all places of 256 bytes; else four k and two halves of
  // a fragment do
  static __host__ __device__ __forceinline__ int permuted(int line, int word) {
    if (KC) return word ^ (DEEP == 64 ? line / 2 % 8 : line / 4 % 4);
    return word ^ ((line % 4 + line / 8 % 2 * 4) * 2);
  }

  // The word of a thread's load i, from an operand whose lines lie `step` elements apart and of whose rows `inside` are left
  // (rows, or k where they are contiguous, are a multiple of eight: no word is inside in part).
  struct Word {
    unsigned at;  // bytes from the step's first word; kOutside behind the last row
    int k;        // of its first element
  };
  static __host__ __device__ __forceinline__ Word wordOf(int thread, int i, long step, long inside) {
    const int place = (thread / 64 * loads + i) * 64 + thread % 64, line = place / perLine;
    const int word = permuted(line, place % perLine);
    const bool there = (KC ? line : word * 8) < inside;
    return {there ? (unsigned)(line * step + word * 8) * 2 : kOutside, KC ? word * 8 : line};
  }
  // where it is read from while `left` k are inside (perhaps none): a word behind them reads as zeros, too
  static __host__ __device__ __forceinline__ unsigned placeOf(const Word& w, int left) { return w.k >= left ? kOutside : w.at; }
};

}  // namespace fbfft_amd
