// places.h -- a matrix's packs of elements shared out among threads by their
// number, so that rows of any length keep every lane at work.
#pragma once
#include <hip/hip_runtime.h>

namespace {

// Places of a [rows][packs] grid by their number: item `first` + j, j < 2^20.
struct Places {
  long row; int in, packs; float rate;
  __device__ __forceinline__ Places(long first, int packs_) : row(first / packs_), in((int)(first - row * packs_)), packs(packs_), rate(1.0f / packs_) {}
  __device__ __forceinline__ void of(int j, long& r, int& pack) const {
    const int i = in + j;
    int q = (int)(i * rate);   // within one of i / packs, which is at most j / packs + 1: i and rate are off by 2^-24 of themselves
    int left = i - q * packs;
    if (left < 0) { q--; left += packs; }
    if (left >= packs) { q++; left -= packs; }
    r = row + q;
    pack = left;
  }
};

}  // namespace
