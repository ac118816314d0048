// teacher.hip -- a row's entries in a distillation from a teacher's top logits.
//
//   p = softmax(t / T) over the entries j, s[j] = <x, table[k[j]]> / T, lse = log sum over the table of exp <x, table[v]> / T
//   loss = T^2 sum_j p[j] (log p[j] - (s[j] - lse)),  dl[v] = T (exp(<x, table[v]> / T - lse) - p of v) dloss
//
// The softmax over the table and the products with dl are those of the cross
// entropy (products.hip, skinny.hip).  Here the entries' scores are computed from
// the table's rows, which are few of them and mostly common ones; a tile of the
// product would have to find them among its columns.  The scores are kept for the
// gradient, whose places of the entries are written again from them: the
// difference of two probabilities is taken in float32 and rounded once.
#include <algorithm>
#include "teacher.h"
#include "tiles.h"

namespace {

constexpr int BLOCK = 256;
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

// A workgroup has a row, or where there are few rows a share of its entries,
// and the first of them the teacher's probabilities.  L: the type of its logits.
template <class T, class L>
__global__ __launch_bounds__(BLOCK) void entries_kernel(const TeachArgs a, long base) {
  constexpr int V = 16 / sizeof(T), WAVES = BLOCK / 64;
  __shared__ long long ids[MOST_TOP];   // a.ignore of what is no entry
  __shared__ float probs[MOST_TOP];
  __shared__ float sums[WAVES];
  const long block = base + blockIdx.x, row = block / a.parts;
  const int part = (int)(block - row * a.parts), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long first = row * a.top;
  float top = -INFINITY;
  int any = 0;
  for (int j = threadIdx.x; j < a.top; j += BLOCK) {
    const float t = (float)((const L*)a.logits)[first + j];
    const long long id = t == -INFINITY ? a.ignore : a.ids[first + j];
    ids[j] = id;
    probs[j] = t;
    if (id == a.ignore) continue;
    any |= id < 0 || id >= a.vocab ? 3 : 1;
    top = fmaxf(top, t);
  }
  const int found = __syncthreads_or(any);
  const bool outside = __syncthreads_or(any & 2);
  if (part == 0) {
    top = wave_max(top);
    if (lane == 0) sums[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) top = fmaxf(top, sums[w]);
    __syncthreads();
    float sum = 0;
    for (int j = threadIdx.x; j < a.top; j += BLOCK) {
      // (the difference first: of lowest values alone it is 0, whatever the temperature)
      const float e = ids[j] == a.ignore ? 0.0f : expf((probs[j] - top) / a.temperature);
      probs[j] = e;
      sum += e;
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) sum += sums[w];
    for (int j = threadIdx.x; j < a.top; j += BLOCK) {
      const long long id = ids[j];
      float p = 0;
      bool again = false;
      for (int k = 0; k < a.top; k++) {
        if (ids[k] != id) continue;
        again |= k < j;
        p += probs[k];
      }
      a.probs[first + j] = id == a.ignore || again ? -1.0f : id < 0 || id >= a.vocab ? NAN : p / sum;
    }
    if (threadIdx.x == 0) a.kept[row] = !found ? TEACH_NONE : outside ? TEACH_OUTSIDE : TEACH_FINE;
  }
  const T* x = (const T*)a.x + row * a.ldx;
  for (int j0 = (part * WAVES + wave) * AT_ONCE; j0 < a.top; j0 += a.parts * WAVES * AT_ONCE) {
    long long id[AT_ONCE];
    bool in[AT_ONCE];
    float sum[AT_ONCE] = {};
    bool some = false;
#pragma unroll
    for (int e = 0; e < AT_ONCE; e++) {
      id[e] = j0 + e < a.top ? ids[j0 + e] : a.ignore;
      in[e] = id[e] != a.ignore && id[e] >= 0 && id[e] < a.vocab;
      some |= in[e];
    }
    if (some)
      for (int k = lane * V; k < a.width; k += 64 * V) {
        float u[V], w[AT_ONCE][V];
        load_part<T, V>(x, k, a.width, u);
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++) load_part<T, V>((const T*)a.table + (in[e] ? id[e] : 0) * a.ldtable, k, a.width, w[e]);
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++)
#pragma unroll
          for (int i = 0; i < V; i++) sum[e] = __builtin_fmaf(u[i], w[e][i], sum[e]);
      }
#pragma unroll
    for (int e = 0; e < AT_ONCE; e++) sum[e] = wave_sum(sum[e]);
    if (lane == 0)
#pragma unroll
      for (int e = 0; e < AT_ONCE; e++)
        if (j0 + e < a.top) a.scores[first + j0 + e] = in[e] ? sum[e] / a.temperature : id[e] == a.ignore ? 0.0f : NAN;
  }
}

// WAVES of a workgroup join a row's pieces and add its entries' terms.
template <int WAVES>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void finish_kernel(const TeachFinish a, long base) {
  constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1, N = WAVES * 64;
  __shared__ float2 pieces[WAVES];
  __shared__ float sums[WAVES];
  const long i = (base + blockIdx.x) * ROWS + (WAVES == 1 ? threadIdx.x >> 6 : 0);
  const int at = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, wave = at >> 6;
  if (i >= (a.count ? *a.count : a.n)) return;
  const long row = a.rows ? a.rows[i] : i;
  float2 run = make_float2(-INFINITY, 0.0f);
#pragma unroll 4
  for (int k = at; k < a.parts; k += N) run = join(run, a.part[i * a.parts + k]);
#pragma unroll
  for (int o = 32; o; o >>= 1) run = join(run, make_float2(__shfl_xor(run.x, o), __shfl_xor(run.y, o)));
  if constexpr (WAVES > 1) {
    if ((at & 63) == 0) pieces[wave] = run;
    __syncthreads();
    run = pieces[0];
    for (int w = 1; w < WAVES; w++) run = join(run, pieces[w]);
  }
  const float lse = run.x + logf(run.y);
  float sum = 0;
  for (int j = at; j < a.top; j += N) {
    const float p = a.probs[row * a.top + j];
    if (p < 0.0f || p == 0.0f) continue;   // (a NaN is added)
    sum += p * (logf(p) - (a.scores[row * a.top + j] - lse));
  }
  sum = wave_sum(sum);
  if constexpr (WAVES > 1) {
    if ((at & 63) == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < WAVES; w++) sum += sums[w];
  }
  if (at) return;
  const bool none = !a.rows && a.kept[row] == TEACH_NONE;
  a.lse[row] = none ? 0.0f : lse;
  a.loss[row] = none ? 0.0f : sum * a.temperature * a.temperature;
}

// `lanes` threads a row.
template <class T>
__global__ __launch_bounds__(BLOCK) void patch_kernel(const TeachPatch a, int lanes, long base) {
  const long i = (base + blockIdx.x) * (BLOCK / lanes) + threadIdx.x / lanes;
  if (i >= *a.count) return;
  const long first = a.rows[i] * (long)a.top;
  const float grad = a.tgt[i] < 0 ? NAN : a.grad[i] * (a.scale ? *a.scale : 1.0f), lse = a.lse[i];
  for (int j = threadIdx.x % lanes; j < a.top; j += lanes) {
    const long col = a.ids[first + j] - a.v0;
    const float p = a.probs[first + j];
    if (p < 0.0f || col < 0 || col >= a.len) continue;
    const float v = (__expf(a.scores[first + j] - lse) - p) * grad;
    uint16_t* o = a.dl + i * a.ld + col;
    if constexpr (sizeof(T) == 4) {
      __bf16 s[3];
      split3(v, s);
#pragma unroll
      for (int k = 0; k < 3; k++) o[k * a.part] = __builtin_bit_cast(uint16_t, s[k]);
    } else {
      const T one = (T)v;
      o[0] = __builtin_bit_cast(uint16_t, one);
      if (a.part) o[a.part] = __builtin_bit_cast(uint16_t, (T)(fabsf((float)one) < INFINITY ? v - (float)one : 0.0f));
    }
  }
}

}  // namespace

void teach_entries(TeachArgs a, hipStream_t st) {
  // 512 workgroups, if there are as many times the entries that one takes at once
  a.parts = (int)std::max<long>(1, std::min<long>(clr::ceil_div(512, a.rows), clr::ceil_div(a.top, AT_ONCE * (BLOCK / 64))));
  clr::with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    clr::in_launches(a.rows * a.parts, BLOCK, [&](long base, unsigned n) {
      if (a.teacher_type == DT_F32) entries_kernel<T, float><<<n, BLOCK, 0, st>>>(a, base);
      else entries_kernel<T, T><<<n, BLOCK, 0, st>>>(a, base);
    });
  });
}
void teach_finish(const TeachFinish& a, hipStream_t st) {
  if (a.rows) clr::in_launches(clr::ceil_div(a.n, 4), BLOCK, [&](long base, unsigned n) { finish_kernel<1><<<n, BLOCK, 0, st>>>(a, base); });
  else finish_kernel<16><<<(unsigned)a.n, 1024, 0, st>>>(a, 0);
}
void teach_patch(const TeachPatch& a, hipStream_t st) {
  int lanes = 1;
  while (lanes < BLOCK && lanes < a.top) lanes *= 2;
  clr::with_type(a.dtype, [&](auto t) {
    clr::in_launches(clr::ceil_div(a.n, BLOCK / lanes), BLOCK, [&](long base, unsigned n) { patch_kernel<decltype(t)><<<n, BLOCK, 0, st>>>(a, lanes, base); });
  });
}
