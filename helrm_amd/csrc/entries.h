// entries.h -- device functions of a row's entries in a distillation: the
// teacher's probabilities and the entries' scores.
#pragma once
#include "teacher.h"

namespace {

constexpr int AT_ONCE = 4;   // entries of a wave

// V elements from p[k] on, 0 past the end.
template <class T, int V> __device__ __forceinline__ void load_part(const T* p, int k, int width, float (&v)[V]) {
  T t[V] = {};
  if (k + V <= width) __builtin_memcpy(t, p + k, sizeof(t));   // (global loads of 16 bytes need no alignment)
  else
#pragma unroll
    for (int e = 0; e < V; e++) if (k + e < width) t[e] = p[k + e];
#pragma unroll
  for (int e = 0; e < V; e++) v[e] = (float)t[e];
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// A row's entries in LDS, `top` of them and as many more as make a multiple of 4:
// the table's row or one of these, a teacher's logit and then what it weighs.
constexpr int NOTHING = -1, OUTSIDE = -2;
constexpr int ENTRY_WAVES = 16;   // the most of a workgroup
struct Entries {
  int* ids; float* weights; float* sums;
  int top, padded;
  __device__ __forceinline__ Entries(char* lds, int top_) : top(top_), padded((top_ + 3) & ~3) {
    ids = (int*)lds;
    weights = (float*)(ids + padded);
    sums = weights + padded;
  }
  __device__ __forceinline__ char* behind() const { return (char*)(sums + ENTRY_WAVES); }
};

template <class L> __device__ __forceinline__ int entry_of(const TeachArgs& a, long at, float& logit) {
  logit = (float)((const L*)a.logits)[at];
  const long long id = a.ids[at];
  return id == a.ignore || logit == -INFINITY ? NOTHING : id < 0 || id >= a.vocab ? OUTSIDE : (int)id;
}
// Reads them; the largest logit, of each thread, is the result, and `any` 1 if it has an entry, 3 one outside the table.
template <class L> __device__ __forceinline__ float read_entries(const TeachArgs& a, long row, const Entries& e, int& any) {
  float top = -INFINITY;
  any = 0;
  for (int j = threadIdx.x; j < e.padded; j += blockDim.x) {
    float t = -INFINITY;
    const int id = j < e.top ? entry_of<L>(a, row * e.top + j, t) : NOTHING;
    e.ids[j] = id;
    e.weights[j] = t;
    if (id == NOTHING) continue;
    any |= id == OUTSIDE ? 3 : 1;
    top = fmaxf(top, t);
  }
  return top;
}
// The weights become exponentials; the result is their sum.  All the threads of a workgroup.
__device__ __forceinline__ float weigh(const TeachArgs& a, float top, const Entries& e) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  top = wave_max(top);
  if (waves > 1) {
    if (lane == 0) e.sums[wave] = top;
    __syncthreads();
    for (int w = 0; w < waves; w++) top = fmaxf(top, e.sums[w]);
    __syncthreads();
  }
  float sum = 0;
  for (int j = threadIdx.x; j < e.padded; j += blockDim.x) {
    // (the difference first: of lowest values alone it is 0, whatever the temperature)
    const float v = e.ids[j] == NOTHING ? 0.0f : expf((e.weights[j] - top) / a.temperature);
    e.weights[j] = v;
    sum += v;
  }
  sum = wave_sum(sum);
  if (waves > 1) {
    if (lane == 0) e.sums[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < waves; w++) sum += e.sums[w];
  }
  return sum;
}
// What entry j and those with the same id weigh together, and whether it is the first of them.
__device__ __forceinline__ float together(const Entries& e, int j, bool& first) {
  const int id = e.ids[j];
  float p = 0;
  first = true;
  for (int k = 0; k < e.padded; k += 4) {
    const int4 ids = *(const int4*)(e.ids + k);
    const float4 w = *(const float4*)(e.weights + k);
    const int i[4] = {ids.x, ids.y, ids.z, ids.w};
    const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int n = 0; n < 4; n++) {
      if (i[n] != id) continue;
      if (k + n < j) first = false;
      p += v[n];
    }
  }
  return p;
}

// A workgroup has a row's entries, or where there are few rows a share of them,
// the teacher's probabilities among them.  lds: entries_bytes.
template <class T, class L> __device__ __forceinline__ void row_entries(const TeachArgs& a, long block, char* lds) {
  constexpr int V = 16 / sizeof(T);
  const Entries e(lds, a.top);
  const long row = block / a.parts;
  const int part = (int)(block - row * a.parts), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const long first = row * a.top;
  int any;
  const float top = read_entries<L>(a, row, e, any);
  const int found = __syncthreads_or(any);
  const bool outside = __syncthreads_or(any & 2);
  const float sum = weigh(a, top, e);
  __syncthreads();
  for (int j = part * blockDim.x + threadIdx.x; j < a.top; j += a.parts * blockDim.x) {
    bool leads;
    const float p = together(e, j, leads);
    const int id = e.ids[j];
    a.probs[first + j] = id == OUTSIDE ? NAN : id == NOTHING || !leads ? -1.0f : p / sum;
    a.cols[first + j] = id >= 0 && leads ? id : -1;
  }
  if (part == 0 && threadIdx.x == 0) a.kept[row] = !found ? TEACH_NONE : outside ? TEACH_OUTSIDE : TEACH_FINE;
  const T* x = (const T*)a.x + row * a.ldx;
  for (int j0 = (part * waves + wave) * AT_ONCE; j0 < a.top; j0 += a.parts * waves * AT_ONCE) {
    int id[AT_ONCE];
    float sum[AT_ONCE] = {};
    bool some = false;
#pragma unroll
    for (int n = 0; n < AT_ONCE; n++) {
      id[n] = j0 + n < a.top ? e.ids[j0 + n] : NOTHING;
      some |= id[n] >= 0;
    }
    if (some)
      for (int k = lane * V; k < a.width; k += 64 * V) {
        float u[V], w[AT_ONCE][V];
        load_part<T, V>(x, k, a.width, u);
#pragma unroll
        for (int n = 0; n < AT_ONCE; n++) load_part<T, V>((const T*)a.table + max(id[n], 0) * a.ldtable, k, a.width, w[n]);
#pragma unroll
        for (int n = 0; n < AT_ONCE; n++)
#pragma unroll
          for (int i = 0; i < V; i++) sum[n] = __builtin_fmaf(u[i], w[n][i], sum[n]);
      }
#pragma unroll
    for (int n = 0; n < AT_ONCE; n++) sum[n] = wave_sum(sum[n]);
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < AT_ONCE; n++)
        if (j0 + n < a.top) a.scores[first + j0 + n] = id[n] >= 0 ? sum[n] / a.temperature : 0.0f;
  }
}

}  // namespace
