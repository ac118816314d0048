// norm.hip -- layer norm, forward and backward.
//
//   mu = mean(x), r = (mean((x - mu)^2) + eps)^-1/2, h = (x - mu) r, y = h w + b
//   dx = r (w dy - mean(w dy) - h mean(w dy h)), dw = sum_rows dy h, db = sum_rows dy
//
// All sums are float32.  The variance is the mean square about the mean, so
// rows far from zero lose nothing.  Bound by memory: a row is read once, by 1
// to 8 waves that hold 16 values a lane, and the backward pass adds its rows
// to the weights' gradients in registers while it has them.
//
// Measured (a copy here: 4.95 TB/s): 32,768 x 4,096 bfloat16 forward 110 us =
// 4.9 TB/s, backward 176 us = 4.6 TB/s and 8 us for the sums of the weights'
// gradients; 8,192 x 1,024 bfloat16 9 + 13 + 4 us; 4,097 x 1,001 float32, an
// element a load, 8 + 15 + 4 us; 1 x 512 2 us.
#include <algorithm>
#include "cleartext.h"
#include "norm.h"

namespace {

constexpr int BLOCK = 256;
constexpr int HOLD = 16;             // values a lane
constexpr int MOST_WAVES = 8;        // of a row: 8,192 values; longer rows are read again for every sum

template <class T, int V> struct Pack { T v[V]; };

// A row's values, V neighbours at a time: lane l of n takes packs l, l + n, ...
// ODD: rows start anywhere and the last pack may be cut short.
template <class T, int V, int N, bool ODD>
__device__ __forceinline__ void load_row(const T* p, int lane, int n, int width, float (&v)[N * V]) {
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int i = (j * n + lane) * V;
    Pack<T, V> t{};
    if constexpr (ODD) {
      if (i + V <= width) __builtin_memcpy(&t, p + i, sizeof(t));   // (global loads of 16 bytes need no alignment)
      else
#pragma unroll
        for (int e = 0; e < V; e++) if (i + e < width) t.v[e] = p[i + e];
    } else if (i < width) {
      const uint4 raw = *(const uint4*)(p + i);
      t = __builtin_bit_cast(decltype(t), raw);
    }
#pragma unroll
    for (int e = 0; e < V; e++) v[j * V + e] = (float)t.v[e];
  }
}
template <class T, int V, int N, bool ODD>
__device__ __forceinline__ void store_row(T* p, int lane, int n, int width, const float (&v)[N * V]) {
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int i = (j * n + lane) * V;
    if (i >= width) continue;
    Pack<T, V> t;
#pragma unroll
    for (int e = 0; e < V; e++) t.v[e] = (T)v[j * V + e];
    if constexpr (!ODD) *(uint4*)(p + i) = __builtin_bit_cast(uint4, t);
    else if (i + V <= width) __builtin_memcpy(p + i, &t, sizeof(t));
    else
#pragma unroll
      for (int e = 0; e < V; e++) if (i + e < width) p[i + e] = t.v[e];
  }
}
// The weights of the same places, 0 past the end of the row.
template <class P, int V, int N, bool ODD>
__device__ __forceinline__ void load_param(const P* p, int lane, int n, int width, float (&v)[N * V]) {
#pragma unroll
  for (int j = 0; j < N; j++) {
    const int i = (j * n + lane) * V;
    Pack<P, V> t{};
    if (i < width) {
      if constexpr (!ODD && V * sizeof(P) % 16 == 0) {
        uint4 raw[V * sizeof(P) / 16];
#pragma unroll
        for (int k = 0; k < (int)(V * sizeof(P) / 16); k++) raw[k] = ((const uint4*)(p + i))[k];
        __builtin_memcpy(&t, raw, sizeof(t));
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) if (!ODD || i + e < width) t.v[e] = p[i + e];
      }
    }
#pragma unroll
    for (int e = 0; e < V; e++) v[j * V + e] = (float)t.v[e];
  }
}

__device__ __forceinline__ float2 wave_sum(float2 v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) { v.x += __shfl_xor(v.x, o); v.y += __shfl_xor(v.y, o); }
  return v;
}
// The sums over the waves of a row, in the same order every time.  `lds`: MOST_WAVES pairs, not those of the call before.
template <bool MANY> __device__ __forceinline__ float2 row_sum(float2 v, int wave, int waves, float2* lds) {
  v = wave_sum(v);
  if (!MANY) return v;
  if ((threadIdx.x & 63) == 0) lds[wave] = v;
  __syncthreads();
  float2 s = lds[0];
  for (int i = 1; i < waves; i++) { s.x += lds[i].x; s.y += lds[i].y; }
  return s;
}

// MANY: the workgroup has one row at a time; otherwise each of its waves has
// one.  It takes every gridDim.x-th (of four): the weights stay in registers,
// where 32-bit ones of their own would be twice the traffic of a 16-bit row.
template <class T, class P, int V, int N, bool ODD, bool MANY>
__global__ __launch_bounds__(MANY ? 512 : BLOCK) void norm_forward(const T* x, long ldx, const P* w, const P* b, T* y, long ldy, float* mean,
                                                                     float* rstd, long rows, int width, float eps) {
  __shared__ float2 lds[4][MOST_WAVES];
  const int wave = MANY ? threadIdx.x >> 6 : 0, waves = MANY ? blockDim.x >> 6 : 1;
  const int lane = MANY ? threadIdx.x : threadIdx.x & 63, n = waves * 64;
  const long per = MANY ? 1 : BLOCK / 64;
  float c[N * V], o[N * V];
  load_param<P, V, N, ODD>(w, lane, n, width, c);
  if (b) load_param<P, V, N, ODD>(b, lane, n, width, o);
  else {
#pragma unroll
    for (int i = 0; i < N * V; i++) o[i] = 0.0f;
  }
  int turn = 0;
  for (long row = blockIdx.x * per + (MANY ? 0 : threadIdx.x >> 6); row < rows; row += gridDim.x * per, turn ^= 2) {
    float v[N * V];
    load_row<T, V, N, ODD>(x + row * ldx, lane, n, width, v);
    float s = 0;
#pragma unroll
    for (int i = 0; i < N * V; i++) s += v[i];
    const float mu = row_sum<MANY>(make_float2(s, 0), wave, waves, lds[turn]).x / width;
    float q = 0;
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float d = (j * n + lane) * V + (ODD ? e : 0) < width ? v[j * V + e] - mu : 0.0f;
        v[j * V + e] = d;
        q += d * d;
      }
    const float r = 1.0f / sqrtf(row_sum<MANY>(make_float2(q, 0), wave, waves, lds[turn + 1]).x / width + eps);
#pragma unroll
    for (int i = 0; i < N * V; i++) v[i] = v[i] * r * c[i] + o[i];
    store_row<T, V, N, ODD>(y + row * ldy, lane, n, width, v);
    if (lane == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
  }
}

// A workgroup takes every gridDim.x-th row (MANY), or four of them at a time,
// one a wave, and leaves the sums of dy h and dy over its rows in
// part[blockIdx.x][2][width].
template <class T, class P, int V, int N, bool ODD, bool MANY>
__global__ __launch_bounds__(MANY ? 512 : BLOCK) void norm_backward(const T* dy, long lddy, const T* x, long ldx, const P* w, const float* mean,
                                                                     const float* rstd, T* dx, long lddx, float* part, long rows, int width) {
  constexpr int E = N * V;
  __shared__ float2 lds[2][MOST_WAVES];
  __shared__ float sums[MANY ? 1 : BLOCK / 64][MANY ? 1 : 64 * E];
  const int wave = MANY ? threadIdx.x >> 6 : 0, waves = MANY ? blockDim.x >> 6 : 1;
  const int lane = MANY ? threadIdx.x : threadIdx.x & 63, n = waves * 64;
  const int mine = MANY ? 0 : threadIdx.x >> 6;
  const long per = MANY ? 1 : BLOCK / 64;
  float c[E], sw[E], sb[E];
  load_param<P, V, N, ODD>(w, lane, n, width, c);
#pragma unroll
  for (int i = 0; i < E; i++) sw[i] = sb[i] = 0;
  int turn = 0;
  for (long row = blockIdx.x * per + mine; row < rows; row += gridDim.x * per, turn ^= 1) {
    float h[E], d[E];
    load_row<T, V, N, ODD>(x + row * ldx, lane, n, width, h);
    load_row<T, V, N, ODD>(dy + row * lddy, lane, n, width, d);
    const float mu = mean[row], r = rstd[row];
    float2 s = make_float2(0, 0);
#pragma unroll
    for (int j = 0; j < N; j++) {
#pragma unroll
      for (int i = j * V; i < (j + 1) * V; i++) {
        // past the end of the row d, c and h are 0, also where mu r overflows
        const float m = (j * n + lane) * V + (ODD ? i - j * V : 0) < width ? mu : 0.0f;
        h[i] = (h[i] - m) * r;
        sw[i] += d[i] * h[i];
        sb[i] += d[i];
        d[i] *= c[i];
        s.x += d[i];
        s.y += d[i] * h[i];
      }
    }
    s = row_sum<MANY>(s, wave, waves, lds[turn]);
    s.x /= width;
    s.y /= width;
#pragma unroll
    for (int i = 0; i < E; i++) d[i] = r * (d[i] - s.x - h[i] * s.y);
    store_row<T, V, N, ODD>(dx + row * lddx, lane, n, width, d);
  }
  float* out = part + (long)blockIdx.x * 2 * width;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    if (MANY) {
#pragma unroll
      for (int j = 0; j < N; j++)
#pragma unroll
        for (int e = 0; e < V; e++) {
          const int i = (j * n + lane) * V + e;
          if (i < width) out[(long)k * width + i] = k ? sb[j * V + e] : sw[j * V + e];
        }
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < N; j++)
#pragma unroll
        for (int e = 0; e < V; e++) sums[mine][(j * 64 + lane) * V + e] = k ? sb[j * V + e] : sw[j * V + e];
      __syncthreads();
      for (int i = threadIdx.x; i < width; i += BLOCK) {
        float t = 0;
        for (int u = 0; u < BLOCK / 64; u++) t += sums[u][i];
        out[(long)k * width + i] = t;
      }
    }
  }
}

// dw and db: the sums over the workgroups' parts, 16 columns a workgroup, in
// a fixed order (no atomics: the gradient is the same on every run).  Bound by
// latency: 512 parts of 4,096 columns, 17 MB from the last-level cache, 8 us.
constexpr int SUM_COLS = 16, SUM_ROWS = 64;
template <class P>
__global__ __launch_bounds__(SUM_COLS* SUM_ROWS) void norm_param_sum(const float* part, P* dw, P* db, int parts, int width, long first) {
  __shared__ float lds[SUM_ROWS][SUM_COLS + 1];
  const int c = threadIdx.x % SUM_COLS, r = threadIdx.x / SUM_COLS;
  const long i = (first + blockIdx.x) * SUM_COLS + c;
  P* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0;
  if (i < width)
#pragma unroll 8
    for (int k = r; k < parts; k += SUM_ROWS) s += part[((long)k * 2 + blockIdx.y) * width + i];
  lds[r][c] = s;
  __syncthreads();
  if (r || i >= width) return;
  for (int k = 1; k < SUM_ROWS; k++) s += lds[k][c];
  out[i] = (P)s;
}

// ---- rows of more than MOST_WAVES * 64 * HOLD values: one workgroup a row, which it reads once for every sum (from its
// caches after the first: a row is at least 16 KiB).  The simple form: no model here has rows that long. ----
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(make_float2(v, 0)).x;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0;
  for (int i = 0; i < BLOCK / 64; i++) s += lds[i];
  return s;
}
template <class T, class P>
__global__ __launch_bounds__(BLOCK) void norm_forward_long(const T* x, long ldx, const P* w, const P* b, T* y, long ldy, float* mean,
                                                           float* rstd, int width, float eps, long first) {
  __shared__ float lds[BLOCK / 64];
  const long row = first + blockIdx.x;
  x += row * ldx;
  y += row * ldy;
  float s = 0;
  for (int i = threadIdx.x; i < width; i += BLOCK) s += (float)x[i];
  const float mu = block_sum(s, lds) / width;
  float q = 0;
  for (int i = threadIdx.x; i < width; i += BLOCK) { const float d = (float)x[i] - mu; q += d * d; }
  const float r = 1.0f / sqrtf(block_sum(q, lds) / width + eps);
  for (int i = threadIdx.x; i < width; i += BLOCK)
    y[i] = (T)(((float)x[i] - mu) * r * (float)w[i] + (b ? (float)b[i] : 0.0f));
  if (threadIdx.x == 0) {
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = r;
  }
}
template <class T, class P>
__global__ __launch_bounds__(BLOCK) void norm_backward_long(const T* dy, long lddy, const T* x, long ldx, const P* w, const float* mean,
                                                            const float* rstd, T* dx, long lddx, int width, long first) {
  __shared__ float lds[BLOCK / 64];
  const long row = first + blockIdx.x;
  dy += row * lddy;
  x += row * ldx;
  dx += row * lddx;
  const float mu = mean[row], r = rstd[row];
  float s = 0, t = 0;
  for (int i = threadIdx.x; i < width; i += BLOCK) {
    const float d = (float)dy[i] * (float)w[i];
    s += d;
    t += d * ((float)x[i] - mu) * r;
  }
  s = block_sum(s, lds) / width;
  t = block_sum(t, lds) / width;
  for (int i = threadIdx.x; i < width; i += BLOCK) {
    const float d = (float)dy[i] * (float)w[i];
    dx[i] = (T)(r * (d - s - ((float)x[i] - mu) * r * t));
  }
}
// A span of rows, one thread a column.  It reads dx's place before nobody: it runs ahead of norm_backward_long.
template <class T>
__global__ __launch_bounds__(BLOCK) void norm_param_long(const T* dy, long lddy, const T* x, long ldx, const float* mean, const float* rstd,
                                                         float* part, long rows, int width, long span) {
  const int i = blockIdx.x * BLOCK + threadIdx.x;
  if (i >= width) return;
  const long r0 = blockIdx.y * span, r1 = min(rows, r0 + span);
  float sw = 0, sb = 0;
  for (long row = r0; row < r1; row++) {
    const float d = (float)dy[row * lddy + i];
    sw += d * ((float)x[row * ldx + i] - mean[row]) * rstd[row];
    sb += d;
  }
  part[(long)blockIdx.y * 2 * width + i] = sw;
  part[(long)blockIdx.y * 2 * width + width + i] = sb;
}

bool is_long(int width) { return width > MOST_WAVES * 64 * HOLD; }
int row_waves(int width) { return (int)clr::ceil_div(width, 64 * HOLD); }
constexpr long MOST_GROUPS = 2048;   // of the forward pass: eight a CU
// Workgroups of the backward pass: two a CU, and at least four rows for each
// wave or row, so that the parts are little beside the rows.
int part_count(long rows, int width) {
  const long per = is_long(width) ? 32 : row_waves(width) > 1 ? 8 : 4 * (BLOCK / 64);
  return (int)std::max<long>(1, std::min<long>(512, clr::ceil_div(rows, per)));
}

// f(V, N, ODD): how a row is loaded -- V elements at a time, N times a lane -- and whether not every row of every tensor
// (and the weights) starts at a multiple of 16 bytes and holds a whole number of them.  Then 16-bit rows are still read 16
// bytes at a time (32,768 x 4,095 bfloat16 forward 204 us, 335 an element at a time, backward 327 and 966; 4,097 x 1,001
// backward 19 and 38), except forward with a whole row of 513 to 1,024 in one wave, where the cut pack holds the wave up
// (4,097 x 1,001 14 us, 10 an element at a time), and float32 an element at a time (4,097 x 1,001 10 + 18.7 us, 14 + 18.7 in
// packs; 32,768 x 1,535 79 + 151 and 89 + 215; 32,768 x 4,095 202 + 313 and 224 + 324).  Not the faster at every size: 32,768 x
// 333 float32 backward 39 us, 34.5 in packs; 32,768 x 767 bfloat16 forward 50 us, 41 in packs.
template <int V> struct Int { static constexpr int value = V; };
template <class T, class F> void with_packs(bool aligned, bool forward, int width, int waves, F&& f) {
  constexpr int V = 16 / sizeof(T);
  const bool half = clr::ceil_div(width, waves * 64 * V) <= HOLD / V / 2;
  auto go = [&](auto odd) {
    if (half) f(Int<V>{}, Int<HOLD / V / 2>{}, odd);
    else f(Int<V>{}, Int<HOLD / V>{}, odd);
  };
  if (aligned) return go(std::false_type{});
  if constexpr (sizeof(T) == 2)
    if (!forward || waves > 1 || half) return go(std::true_type{});
  f(Int<1>{}, Int<HOLD>{}, std::true_type{});
}
bool packs(const void* p, long ld, long rows, int width, int dtype) {
  const int v = 16 / dtype_size(dtype);
  return (uintptr_t)p % 16 == 0 && width % v == 0 && (rows <= 1 || ld % v == 0);
}

}  // namespace

void norm_forward_launch(const NormArgs& a, hipStream_t st) {
  if (!a.rows) return;
  const bool aligned = packs(a.x, a.ldx, a.rows, a.width, a.dtype) && packs(a.y, a.ldy, a.rows, a.width, a.dtype) &&
                       ((uintptr_t)a.weight | (uintptr_t)a.bias) % 16 == 0;
  const int waves = row_waves(a.width);
  clr::with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      if (is_long(a.width)) {
        clr::in_launches(a.rows, BLOCK, [&](long first, unsigned k) {
          norm_forward_long<T, P><<<k, BLOCK, 0, st>>>((const T*)a.x, a.ldx, (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.ldy, a.mean, a.rstd,
                                                       a.width, a.eps, first);
        });
        return;
      }
      with_packs<T>(aligned, true, a.width, waves, [&](auto v, auto n, auto odd) {
        if (waves > 1)
          norm_forward<T, P, decltype(v)::value, decltype(n)::value, decltype(odd)::value, true><<<(unsigned)std::min<long>(a.rows, MOST_GROUPS), waves * 64, 0, st>>>(
              (const T*)a.x, a.ldx, (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.ldy, a.mean, a.rstd, a.rows, a.width, a.eps);
        else
          norm_forward<T, P, decltype(v)::value, decltype(n)::value, decltype(odd)::value, false><<<(unsigned)std::min(clr::ceil_div(a.rows, BLOCK / 64), MOST_GROUPS), BLOCK, 0, st>>>(
              (const T*)a.x, a.ldx, (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.ldy, a.mean, a.rstd, a.rows, a.width, a.eps);
      });
    };
    if (a.param_dtype == DT_F32) go(float{});
    else go(t);
  });
}

size_t norm_backward_workspace(long rows, int width) { return (size_t)part_count(rows, width) * 2 * width * sizeof(float); }

void norm_backward_launch(const NormArgs& a, hipStream_t st) {
  const bool aligned = packs(a.x, a.ldx, a.rows, a.width, a.dtype) && packs(a.y, a.ldy, a.rows, a.width, a.dtype) &&
                       packs(a.dx, a.lddx, a.rows, a.width, a.dtype) && (uintptr_t)a.weight % 16 == 0;
  const int parts = part_count(a.rows, a.width), waves = row_waves(a.width);
  float* part = (float*)a.workspace;
  clr::with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      if (is_long(a.width)) {
        norm_param_long<T><<<dim3(clr::groups_of(clr::ceil_div(a.width, BLOCK), BLOCK), parts), BLOCK, 0, st>>>(
            (const T*)a.y, a.ldy, (const T*)a.x, a.ldx, a.mean, a.rstd, part, a.rows, a.width, clr::ceil_div(a.rows, parts));
        clr::in_launches(a.rows, BLOCK, [&](long first, unsigned k) {
          norm_backward_long<T, P><<<k, BLOCK, 0, st>>>((const T*)a.y, a.ldy, (const T*)a.x, a.ldx, (const P*)a.weight, a.mean, a.rstd, (T*)a.dx, a.lddx,
                                                        a.width, first);
        });
      } else {
        with_packs<T>(aligned, false, a.width, waves, [&](auto v, auto n, auto odd) {
          if (waves > 1)
            norm_backward<T, P, decltype(v)::value, decltype(n)::value, decltype(odd)::value, true><<<parts, waves * 64, 0, st>>>(
                (const T*)a.y, a.ldy, (const T*)a.x, a.ldx, (const P*)a.weight, a.mean, a.rstd, (T*)a.dx, a.lddx, part, a.rows, a.width);
          else
            norm_backward<T, P, decltype(v)::value, decltype(n)::value, decltype(odd)::value, false><<<parts, BLOCK, 0, st>>>(
                (const T*)a.y, a.ldy, (const T*)a.x, a.ldx, (const P*)a.weight, a.mean, a.rstd, (T*)a.dx, a.lddx, part, a.rows, a.width);
        });
      }
      clr::in_launches(clr::ceil_div(a.width, SUM_COLS), SUM_COLS * SUM_ROWS, [&](long first, unsigned k) {
        norm_param_sum<P><<<dim3(k, 2), SUM_COLS * SUM_ROWS, 0, st>>>(part, (P*)a.dweight, (P*)a.dbias, parts, a.width, first);
      });
    };
    if (a.param_dtype == DT_F32) go(float{});
    else go(t);
  });
}
