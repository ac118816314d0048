// norm.hip -- layer norm, forward and backward.
//
//   mu = mean(x), r = (mean((x - mu)^2) + eps)^-1/2, h = (x - mu) r, y = h w + b
//   dx = r (w dy - mean(w dy) - h mean(w dy h)), dw = sum_rows dy h, db = sum_rows dy
//
// All sums are float32.  The variance is the mean square about the mean, in a
// second reading of the row, so rows far from zero lose nothing.
#include "cleartext.h"
#include "norm.h"

namespace {

constexpr int BLOCK = 256;

// The sum over the workgroup, in the same order every time; `lds` holds one
// float a wave.
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0;
#pragma unroll
  for (int i = 0; i < BLOCK / 64; i++) s += lds[i];
  return s;
}

// One workgroup a row.
template <class T, class P>
__global__ __launch_bounds__(BLOCK) void norm_forward(const T* x, long ldx, const P* w, const P* b, T* y, long ldy, float* mean,
                                                      float* rstd, int width, float eps) {
  __shared__ float lds[BLOCK / 64];
  const long row = blockIdx.x;
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
__global__ __launch_bounds__(BLOCK) void norm_backward(const T* dy, long lddy, const T* x, long ldx, const P* w, const float* mean,
                                                       const float* rstd, T* dx, long lddx, int width) {
  __shared__ float lds[BLOCK / 64];
  const long row = blockIdx.x;
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

// dw and db of a span of rows, one thread a column: float32 partial sums,
// which the next kernel adds in the order of the spans (no atomics: the
// gradient is the same on every run).
template <class T>
__global__ __launch_bounds__(BLOCK) void norm_param_partial(const T* dy, long lddy, const T* x, long ldx, const float* mean,
                                                            const float* rstd, float* part, long rows, int width, long span) {
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
template <class P>
__global__ __launch_bounds__(BLOCK) void norm_param_sum(const float* part, P* dw, P* db, int spans, int width) {
  const int i = blockIdx.x * BLOCK + threadIdx.x;
  if (i >= width) return;
  float sw = 0, sb = 0;
  for (int s = 0; s < spans; s++) {
    sw += part[(long)s * 2 * width + i];
    sb += part[(long)s * 2 * width + width + i];
  }
  dw[i] = (P)sw;
  if (db) db[i] = (P)sb;
}

int param_spans(long rows) { return (int)std::max<long>(1, std::min<long>(256, clr::ceil_div(rows, 32))); }

}  // namespace

void norm_forward_launch(const NormArgs& a, hipStream_t st) {
  if (!a.rows) return;
  clr::with_type(a.dtype, [&](auto t) {
    clr::with_type(a.param_dtype, [&](auto p) {
      using T = decltype(t); using P = decltype(p);
      norm_forward<T, P><<<dim3(a.rows), BLOCK, 0, st>>>((const T*)a.x, a.ldx, (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.ldy,
                                                         a.mean, a.rstd, a.width, a.eps);
    });
  });
}

size_t norm_backward_workspace(long rows, int width) { return (size_t)param_spans(rows) * 2 * width * sizeof(float); }

void norm_backward_launch(const NormArgs& a, hipStream_t st) {
  const int spans = param_spans(a.rows), cols = (int)clr::ceil_div(a.width, BLOCK);
  float* part = (float*)a.workspace;
  clr::with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    clr::with_type(a.param_dtype, [&](auto p) {
      using P = decltype(p);
      if (a.rows)
        norm_backward<T, P><<<dim3(a.rows), BLOCK, 0, st>>>((const T*)a.y, a.ldy, (const T*)a.x, a.ldx, (const P*)a.weight, a.mean, a.rstd,
                                                            (T*)a.dx, a.lddx, a.width);
      norm_param_partial<T><<<dim3(cols, spans), BLOCK, 0, st>>>((const T*)a.y, a.ldy, (const T*)a.x, a.ldx, a.mean, a.rstd, part, a.rows,
                                                                 a.width, clr::ceil_div(a.rows, spans));
      norm_param_sum<P><<<dim3(cols), BLOCK, 0, st>>>(part, (P*)a.dweight, (P*)a.dbias, spans, a.width);
    });
  });
}
