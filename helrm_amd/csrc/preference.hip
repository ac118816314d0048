// preference.hip -- a loss of pairs of sequences, of which the first is
// preferred, from their tokens' losses and those of a reference model.
//
//   r[s] = sum over the tokens of s that count of (reference - loss), or its mean
//   m = beta (r[0] - r[1]) - margin
//   logistic: (1 - e) log(1 + exp(-m)) + e log(1 + exp(m)),  hinge: max(0, 1 - m)
//   d/d loss[t] = -+ beta d/dm (/ the number of tokens that count)
//
// Sums are of 64 bits: long sequences differ by little of their sums.  A token is
// read once in each direction.  Bound by memory where there are many (512 pairs of
// 2 x 8,192, 134 MB read, 23 us = 5.8 TB/s; backward 100 MB, 16 us, from the
// caches; four tokens a load, a token a load 34 and 16), by launches otherwise
// (128 pairs of 1,700 tokens in a line: 7 + 4 us, and 23 with the host's time).  In a
// line the forward pass shares out a sequence by the mean length: one of 10,000
// tokens among 300 pairs of 2 x 40 takes it from 7 to 58 us.
#include <algorithm>
#include "plan.h"
#include "preference.h"

namespace {

struct Sum { double sum; long count; };
constexpr int WAVE = 64, MOST = 1024;
constexpr int MOST_SPLITS = 64;
constexpr int EACH = 4;   // tokens a thread at once

// Over `lanes` lanes beside one another, a power of two.
__device__ __forceinline__ Sum wave_sum(Sum s, int lanes = WAVE) {
  for (int o = lanes / 2; o; o >>= 1) {
    s.sum += __shfl_xor(s.sum, o);
    s.count += __shfl_xor(s.count, o);
  }
  return s;
}

// Where a sequence's tokens are: elements of a line, or from a row's first one.
struct Tokens { long from, to; };
__device__ __forceinline__ Tokens tokens_of(const PairArgs& a, long sequence) {
  if (!a.offsets) return {0, a.length};
  // (whatever the offsets say, within the line)
  const long from = min(max((long)a.offsets[sequence], 0L), a.length);
  return {from, min(max((long)a.offsets[sequence + 1], from), a.length)};
}
__device__ __forceinline__ Tokens share_of(Tokens t, int split, int splits) {
  const long n = t.to - t.from;
  return {t.from + n / splits * split + min((long)split, n % splits), t.from + n / splits * (split + 1) + min((long)split + 1, n % splits)};
}

// What `threads` threads have of a sequence's share.
__device__ __forceinline__ Sum sum_of(const PairArgs& a, long sequence, int split, int thread, int threads) {
  const Tokens t = share_of(tokens_of(a, sequence), split, a.splits);
  const long row = a.offsets ? 0 : sequence;
  const float* loss = a.loss + row * a.ldloss;
  const float* reference = a.reference ? a.reference + row * a.ldreference : nullptr;
  const long long* target = a.target ? a.target + row * a.ldtarget : nullptr;
  Sum s{0.0, 0};
  auto add = [&](float l, float r, long long t) {
    const bool counts = !target || t != a.ignore;
    s.sum += counts ? (double)r - (double)l : 0.0;
    s.count += counts;
  };
  // four tokens at a time (loads of 16 bytes need no alignment)
  const long whole = t.from + (t.to - t.from) / EACH * EACH;
#pragma unroll 2
  for (long i = t.from + thread * EACH; i < whole; i += threads * EACH) {
    float l[EACH], r[EACH] = {};
    long long k[EACH] = {};
    __builtin_memcpy(l, loss + i, sizeof(l));
    if (reference) __builtin_memcpy(r, reference + i, sizeof(r));
    if (target) __builtin_memcpy(k, target + i, sizeof(k));
#pragma unroll
    for (int e = 0; e < EACH; e++) add(l[e], r[e], k[e]);
  }
  const long i = whole + thread;
  if (i < t.to) add(loss[i], reference ? reference[i] : 0.0f, target ? target[i] : 0);
  return s;
}

// softplus(m) = log(1 + exp m)
__device__ __forceinline__ double softplus(double m) { return fmax(m, 0.0) + log1p(exp(-fabs(m))); }
__device__ __forceinline__ double sigmoid(double m) { return 1.0 / (1.0 + exp(-m)); }

__device__ __forceinline__ void finish(const PairArgs& a, long pair, Sum first, Sum second) {
  const bool any = first.count + second.count > 0;
  const double each[2] = {a.average ? 1.0 / (double)max(first.count, 1L) : 1.0, a.average ? 1.0 / (double)max(second.count, 1L) : 1.0};
  double r[2] = {first.sum * each[0], second.sum * each[1]};
  if (a.offsets) {   // sequences that leave the line, or run backwards
    const long long o[3] = {a.offsets[2 * pair], a.offsets[2 * pair + 1], a.offsets[2 * pair + 2]};
    if (o[0] < 0 || o[1] < o[0] || o[2] < o[1] || o[2] > a.length) r[0] = r[1] = NAN;
  }
  const double m = a.beta * (r[0] - r[1]) - a.margin;
  double value, slope;
  if (a.kind == PAIR_HINGE) {
    value = m < 1.0 ? 1.0 - m : m >= 1.0 ? 0.0 : NAN;
    slope = m < 1.0 ? -1.0 : m >= 1.0 ? 0.0 : NAN;
  } else {
    const double e = a.smoothing;   // (0 and 1: one of the two alone, or its infinity would be 0 * inf)
    value = e < 1.0 ? softplus(-m) * (1.0 - e) : 0.0;
    slope = -sigmoid(-m) * (1.0 - e);
    if (e > 0.0) {
      value += softplus(m) * e;
      slope += sigmoid(m) * e;
    }
  }
  const bool none = !any && r[0] == 0.0;
  if (a.kept) a.kept[pair] = none ? 0 : 1;
  a.value[pair] = none ? 0.0f : (float)value;
  a.ratio[2 * pair] = (float)r[0];
  a.ratio[2 * pair + 1] = (float)r[1];
  a.slope[2 * pair] = (float)(-slope * a.beta * each[0]);
  a.slope[2 * pair + 1] = (float)(slope * a.beta * each[1]);
}

// `lanes` lanes of a wave a pair.
__global__ __launch_bounds__(256) void pair_lanes_kernel(const PairArgs a, int lanes, long base) {
  const long pair = (base + blockIdx.x) * (256 / lanes) + threadIdx.x / lanes;
  if (pair >= a.pairs) return;
  const int lane = threadIdx.x % lanes;
  Sum s[2];
  for (int k = 0; k < 2; k++) s[k] = wave_sum(sum_of(a, 2 * pair + k, 0, lane, lanes), lanes);
  if (lane == 0) finish(a, pair, s[0], s[1]);
}

// A workgroup a pair, or a share of one.
__global__ __launch_bounds__(MOST) void pair_kernel(const PairArgs a, long base) {
  __shared__ Sum lds[2][MOST / WAVE];
  const long block = base + blockIdx.x, pair = block / a.splits;
  const int split = (int)(block - pair * a.splits);
  for (int k = 0; k < 2; k++) {
    const Sum s = wave_sum(sum_of(a, 2 * pair + k, split, threadIdx.x, blockDim.x));
    if (threadIdx.x % WAVE == 0) lds[k][threadIdx.x / WAVE] = s;
  }
  __syncthreads();
  if (threadIdx.x) return;
  Sum s[2] = {lds[0][0], lds[1][0]};
  for (int w = 1; w < (int)blockDim.x / WAVE; w++)
    for (int k = 0; k < 2; k++) {
      s[k].sum += lds[k][w].sum;
      s[k].count += lds[k][w].count;
    }
  if (a.splits == 1) return finish(a, pair, s[0], s[1]);
  for (int k = 0; k < 2; k++) ((Sum*)a.workspace)[block * 2 + k] = s[k];
}
// The shares of a pair, a wave each.
__global__ __launch_bounds__(256) void pair_join_kernel(const PairArgs a) {
  const long pair = blockIdx.x * (256L / WAVE) + threadIdx.x / WAVE;
  if (pair >= a.pairs) return;
  const int lane = threadIdx.x % WAVE;
  Sum s[2];
  for (int k = 0; k < 2; k++) s[k] = wave_sum(lane < a.splits ? ((const Sum*)a.workspace)[(pair * a.splits + lane) * 2 + k] : Sum{0.0, 0});
  if (lane == 0) finish(a, pair, s[0], s[1]);
}

// The gradient in rows, `threads` threads a share of a sequence.
__global__ __launch_bounds__(256) void pair_grad_kernel(const PairArgs a, int threads, long base) {
  const long team = (base + blockIdx.x) * (256 / threads) + threadIdx.x / threads, sequence = team / a.splits;
  const int split = (int)(team - sequence * a.splits), thread = threadIdx.x % threads;
  if (sequence >= 2 * a.pairs) return;
  const Tokens t = share_of({0, a.length}, split, a.splits);
  const long long* target = a.target ? a.target + sequence * a.ldtarget : nullptr;
  float* d = a.dloss + sequence * a.lddloss;
  const float v = a.dvalue[sequence / 2] * a.slope[sequence];
  const long whole = t.from + (t.to - t.from) / EACH * EACH;
#pragma unroll 2
  for (long i = t.from + thread * EACH; i < whole; i += threads * EACH) {
    long long k[EACH];
    float o[EACH];
    if (target) __builtin_memcpy(k, target + i, sizeof(k));
#pragma unroll
    for (int e = 0; e < EACH; e++) o[e] = !target || k[e] != a.ignore ? v : 0.0f;
    __builtin_memcpy(d + i, o, sizeof(o));
  }
  const long i = whole + thread;
  if (i < t.to) d[i] = !target || target[i] != a.ignore ? v : 0.0f;
}

// The gradient in a line.  A workgroup has tokens beside one another, EACH of a
// thread, marks where sequences begin among them and takes the running maximum of
// the marks, so that a token is written once whatever the offsets say (a sequence
// that wrote its own tokens would meet others' where offsets descend), and a long
// sequence is as parallel as short ones.  Bound by the four loads that wait for
// one another: 128 pairs of 2 x 1,500 tokens on average 4.1 us (3.5 a sequence by
// itself), 300 of 2 x 40 with one of 10,000 among them 3.4 (32).
constexpr int MARKED = 1024;
template <int EACH> __global__ __launch_bounds__(256) void line_grad_kernel(const PairArgs a, long base) {
  constexpr int LINE = 256 * EACH;
  __shared__ __align__(16) unsigned marks[LINE];
  __shared__ unsigned tops[256 / WAVE];
  const long all = 2 * a.pairs, first = (base + blockIdx.x) * LINE, last = min(first + LINE, a.length) - 1;
  const int at = threadIdx.x * EACH;
  const long i = first + at;
  const bool whole = i + EACH <= a.length;
  long long k[EACH] = {};
  if (a.target) {
    if (whole) __builtin_memcpy(k, a.target + i, sizeof(k));
    else
      for (int e = 0; e < EACH; e++) if (i + e < a.length) k[e] = a.target[i + e];
  }
#pragma unroll
  for (int e = 0; e < EACH; e += 4) *(uint4*)(marks + at + e) = make_uint4(0, 0, 0, 0);
  // How many offsets are at most the first token's place, and the last one's: from ..
  // to of them, narrowed with as many probes at a time as there are threads until
  // few are between.  (Of offsets that descend, some number.)
  long from[2] = {0, 0}, to[2] = {all + 1, all + 1};
  while (to[1] - from[0] > MARKED && (from[0] < to[0] || from[1] < to[1])) {   // (the same of all threads)
    bool below[2];
    long step[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
      step[w] = (to[w] - from[w] + 255) / 256;
      const long probe = from[w] + (threadIdx.x + 1) * step[w] - 1;
      below[w] = from[w] < to[w] && probe < to[w] && a.offsets[probe] <= (w ? last : first);
    }
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const int count = __syncthreads_count(below[w]);
      if (from[w] == to[w]) continue;
      from[w] = min(from[w] + count * step[w], to[w]);
      to[w] = min(from[w] + step[w] - 1, to[w]);
    }
  }
  __syncthreads();
#pragma unroll 4
  for (long j = from[0] + threadIdx.x; j < to[1]; j += 256) {
    const long o = a.offsets[j];
    if (o <= last) atomicMax(&marks[o <= first ? 0 : o - first], (unsigned)(j - from[0]) + 1);   // (any number may be an offset)
  }
  __syncthreads();
  unsigned m[EACH];
  __builtin_memcpy(m, __builtin_assume_aligned(marks + at, 16), sizeof(m));
#pragma unroll
  for (int e = 1; e < EACH; e++) m[e] = max(m[e], m[e - 1]);
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
  unsigned top = m[EACH - 1];
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) {
    const unsigned t = __shfl_up(top, o);
    if (lane >= o) top = max(top, t);
  }
  if (lane == WAVE - 1) tops[wave] = top;
  __syncthreads();
  top = __shfl_up(top, 1);
  if (lane == 0) top = 0;
  for (int w = 0; w < wave; w++) top = max(top, tops[w]);
#pragma unroll
  for (int e = 0; e < EACH; e++) m[e] = max(m[e], top);
  // of token t, behind m offsets
  auto value = [&](long t, unsigned m) {
    const long s = from[0] + m;   // in sequence s - 1
    const long begin = s > 0 ? a.offsets[s - 1] : 0, end = s <= all ? a.offsets[s] : a.length;
    const float v = s > 0 && s <= all ? a.dvalue[(s - 1) / 2] * a.slope[s - 1] : 0.0f;
    return t < begin || t >= end ? NAN : v;   // (not in it: offsets that descend)
  };
  if (i > last) return;
  float o[EACH];
  if (m[0] == m[EACH - 1] && whole) {
    const long s = from[0] + m[0];
    const long end = s <= all ? a.offsets[s] : a.length;
    const float v = value(i, m[0]);
#pragma unroll
    for (int e = 0; e < EACH; e++) o[e] = i + e < end ? v : NAN;
  } else {
#pragma unroll
    for (int e = 0; e < EACH; e++) o[e] = value(i + e, m[e]);
  }
#pragma unroll
  for (int e = 0; e < EACH; e++) if (a.target && k[e] == a.ignore) o[e] = 0.0f;
  if (whole) __builtin_memcpy(a.dloss + i, o, sizeof(o));
  else
    for (int e = 0; e < EACH; e++) if (i + e < a.length) a.dloss[i + e] = o[e];
}

long mean_length(long pairs, long length, bool packed) { return packed ? clr::ceil_div(length, std::max(2 * pairs, 1L)) : length; }
// Threads of a sequence, which take four tokens each at once; in a line, where
// one may be much longer than the mean, more for the shortest.  50,000 pairs of
// 2 x 16 tokens, forward and backward: 7 + 5 us with 4 lanes, 18 + 10 with 16, 51 + 28
// with 64.  Of long sequences, forward: 512 pairs of 2 x 8,192 tokens 22.8 us
// with 256 threads, 23.3 with 1,024; 300 of 3,000 9.5 and 11.3; 8 of 100,000 15.1 and 11.6.
int lanes_of(long mean, bool packed) { return mean <= 16 && !packed ? 4 : mean <= 64 ? 16 : mean <= 256 ? WAVE : 256; }
// Shares of a pair: where pairs are few and long, as many as give 256 workgroups,
// of 8,192 tokens at the least (8 pairs of 2 x 100,000 tokens 12 us, 32 with one share; backward 5 and 25).
int splits_of(long pairs, long length, bool packed) {
  const long most = 2 * mean_length(pairs, length, packed) / 8192;
  return (int)std::max(1L, std::min({clr::ceil_div(256, pairs), most, (long)MOST_SPLITS}));
}

}  // namespace

size_t preference_workspace(long pairs, long length, bool packed) {
  const int splits = pairs ? splits_of(pairs, length, packed) : 1;
  return splits > 1 ? (size_t)pairs * splits * 2 * sizeof(Sum) : 0;
}
void preference_launch(PairArgs a, hipStream_t st) {
  const long mean = mean_length(a.pairs, a.length, a.offsets);
  a.splits = splits_of(a.pairs, a.length, a.offsets);
  const int lanes = lanes_of(mean, a.offsets);
  if (lanes <= WAVE && a.pairs >= 256) {
    clr::in_launches(clr::ceil_div(a.pairs, 256 / lanes), 256, [&](long base, unsigned n) { pair_lanes_kernel<<<n, 256, 0, st>>>(a, lanes, base); });
    return;
  }
  const int threads = a.pairs >= 256 || mean <= 2048 ? 256 : MOST;
  clr::in_launches(a.pairs * a.splits, threads, [&](long base, unsigned n) { pair_kernel<<<n, threads, 0, st>>>(a, base); });
  if (a.splits > 1) pair_join_kernel<<<clr::groups_of(clr::ceil_div(a.pairs, 256 / WAVE), 256), 256, 0, st>>>(a);
}
void preference_grad_launch(PairArgs a, hipStream_t st) {
  if (a.offsets) {
    // (512 pairs of 2 x 8,192 tokens on average 23.1 us with 4 a thread, 21.4 with 8; 128 of 2 x 1,500 4.1 and 4.8)
    auto go = [&](auto each) {
      constexpr int N = decltype(each)::value;
      clr::in_launches(clr::ceil_div(a.length, 256 * N), 256, [&](long base, unsigned n) { line_grad_kernel<N><<<n, 256, 0, st>>>(a, base); });
    };
    if (a.length < 1L << 20) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
    return;
  }
  const int threads = lanes_of(a.length, false);
  a.splits = (int)std::max(1L, std::min(a.length / 2048, 1L << 20));
  clr::in_launches(clr::ceil_div(2 * a.pairs * a.splits, 256 / threads), 256, [&](long base, unsigned n) { pair_grad_kernel<<<n, 256, 0, st>>>(a, threads, base); });
}
