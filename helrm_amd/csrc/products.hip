// products.hip -- matrix products of the gated block and the cross entropy.
//
// The factors are float32 in LDS and multiply on v_mfma_f32_16x16x4_f32, so
// every product of 16-bit elements is exact and every sum float32.
#include "products.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int TM = 64, TN = 64, TK = 16, THREADS = 256;
constexpr int PAD = 4;

enum Epi { EPI_STORE, EPI_GATE, EPI_GATE_GRAD, EPI_SOFTMAX, EPI_SOFTMAX_GRAD };

__device__ __forceinline__ float act_of(int act, const float* c, float g) {
  if (act == ACT_SILU) return g / (1.0f + __expf(-g));
  if (act == ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
  return ((c[3] * g + c[2]) * g + c[1]) * g + c[0];
}
__device__ __forceinline__ float act_grad(int act, const float* c, float g) {
  if (act == ACT_SILU) { const float s = 1.0f / (1.0f + __expf(-g)); return s * (1.0f + g * (1.0f - s)); }
  if (act == ACT_GELU) return 0.5f * (1.0f + erff(g * 0.70710678118654752f)) + g * __expf(-0.5f * g * g) * 0.39894228040143268f;
  return (3.0f * c[3] * g + 2.0f * c[2]) * g + c[1];
}

// (maximum, sum of exponentials about it) of two pieces of a row.  Where both
// hold nothing above -inf there is nothing to rescale; a NaN stays one.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = a.x > b.x || a.x != a.x ? a.x : b.x;
  if (m == -INFINITY) return make_float2(m, a.y + b.y);
  return make_float2(m, a.y * __expf(a.x - m) + b.y * __expf(b.x - m));
}

__device__ __forceinline__ void put(void* c, int type, long i, float v) {
  if (type == DT_F32) ((float*)c)[i] = v;
  else if (type == DT_BF16) ((__bf16*)c)[i] = (__bf16)v;
  else ((_Float16*)c)[i] = (_Float16)v;
}

// A tile of a factor, float32, k-major: dst[k][row].  Outside it is 0.
template <class T>
__device__ __forceinline__ void load_tile(const Factor& f, long r0, long rows, int k0, int K, float (*dst)[TM + PAD]) {
  const T* p = (const T*)f.p;
  if (f.t == 1) {
    for (int i = threadIdx.x; i < TM * TK; i += THREADS) {
      const int r = i / TK, k = i % TK;
      dst[k][r] = r0 + r < rows && k0 + k < K ? (float)p[(r0 + r) * f.s + k0 + k] : 0.0f;
    }
  } else {
    for (int i = threadIdx.x; i < TM * TK; i += THREADS) {
      const int r = i % TM, k = i / TM;
      dst[k][r] = r0 + r < rows && k0 + k < K ? (float)p[(r0 + r) * f.s + (k0 + k) * f.t] : 0.0f;
    }
  }
}

// One 64 x 64 tile a workgroup, 32 x 32 a wave.  The matrix instruction takes
// the table's side first, so that a lane holds four neighbouring columns n of
// one row m.  EPI_GATE: B rows of the tile alternate, 16 of the gate and 16
// of the up projection, so both values of a column are in one lane.
template <class T, int EPI>
__global__ __launch_bounds__(THREADS) void product_kernel(ProductArgs p) {
  __shared__ float A[TK][TM + PAD], B[TK][TN + PAD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  const long m0 = (long)blockIdx.y * TM, n0 = (long)blockIdx.x * (EPI == EPI_GATE ? TN / 2 : TN);
  long M = p.M;
  int K = p.K;
  if (p.count) { if (p.count_k) K = *p.count; else M = *p.count; }
  if (m0 >= M) return;
  f32x4 acc[2][2] = {};
  for (int pair = 0; pair < (EPI == EPI_GATE ? 1 : p.pairs); pair++)
    for (int k0 = 0; k0 < K; k0 += TK) {
      load_tile<T>(p.a[pair], m0, M, k0, K, A);
      if (EPI == EPI_GATE) {
        for (int i = threadIdx.x; i < TN * TK; i += THREADS) {
          const int r = i / TK, k = i % TK;
          const long n = n0 + (r >> 5) * 16 + (r & 15);
          const Factor& f = p.b[(r >> 4) & 1];
          B[k][r] = n < p.N && k0 + k < K ? (float)((const T*)f.p)[n * f.s + k0 + k] : 0.0f;
        }
      } else {
        load_tile<T>(p.b[pair], n0, p.N, k0, K, B);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < TK; k += 4) {
        float a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          a[i] = A[k + (lane >> 4)][wm * 32 + i * 16 + (lane & 15)];
          b[i] = B[k + (lane >> 4)][wn * 32 + i * 16 + (lane & 15)];
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j], a[i], acc[i][j], 0, 0, 0);
      }
      __syncthreads();
    }
  // acc[i][j][e] is (m, n) = (m0 + wm 32 + i 16 + lane % 16, n0 + wn 32 + j 16 + 4 (lane / 16) + e)
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const long m = m0 + wm * 32 + i * 16 + (lane & 15);
    if (EPI == EPI_SOFTMAX) {
      float2 run = make_float2(-INFINITY, 0.0f);
      const int t = m < M ? p.target[m] : -1;
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const long n = n0 + wn * 32 + j * 16 + 4 * (lane >> 4) + e;
          if (n < p.N) run = join(run, make_float2(acc[i][j][e], 1.0f));
          if (m < M && n == t) p.picked[m] = acc[i][j][e];
        }
      for (int o = 16; o < 64; o <<= 1) run = join(run, make_float2(__shfl_xor(run.x, o), __shfl_xor(run.y, o)));
      if (m < M && lane < 16) p.part[m * p.parts + blockIdx.x * 2 + wn] = run;
      continue;
    }
    if (m >= M) continue;
    if (EPI == EPI_GATE) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const long n = n0 + wn * 16 + 4 * (lane >> 4) + e;
        if (n >= p.N) continue;
        const float g = acc[i][0][e], u = acc[i][1][e];
        if (p.g) { p.g[m * p.N + n] = g; p.u[m * p.N + n] = u; }
        put(p.h, p.dtype, m * p.N + n, act_of(p.act, p.coef, g) * u);
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const long n = n0 + wn * 32 + j * 16 + 4 * (lane >> 4) + e;
        if (n >= p.N) continue;
        float v = acc[i][j][e];
        if (EPI == EPI_STORE) {
          if (p.unscale) v /= *p.unscale;
          if (p.add) v += ((float*)p.c)[m * p.ldc + n];
          put(p.c, p.ctype, m * p.ldc + n, v);
        } else if (EPI == EPI_GATE_GRAD) {
          const long at = m * p.N + n;
          const float g = p.g[at], u = p.u[at], a = act_of(p.act, p.coef, g);
          put(p.dg, p.dtype, at, v * u * act_grad(p.act, p.coef, g));
          put(p.du, p.dtype, at, v * a);
          put(p.h, p.dtype, at, a * u);
        } else {
          const int row = p.rows[m], t = p.target[m];
          float d = __expf(v - p.lse[row]);
          if (t == p.n0 + n) d -= 1.0f;
          if (t < 0) d = NAN;
          put(p.c, p.ctype, m * p.ldc + n, d * p.grad[row] * (p.scale ? *p.scale : 1.0f));
        }
      }
  }
}

template <int EPI> void launch(const ProductArgs& p, hipStream_t st) {
  if (!p.M || !p.N) return;
  const dim3 grid((unsigned)clr::ceil_div(p.N, EPI == EPI_GATE ? TN / 2 : TN), (unsigned)clr::ceil_div(p.M, TM));
  clr::with_type(p.dtype, [&](auto t) { product_kernel<decltype(t), EPI><<<grid, THREADS, 0, st>>>(p); });
}

constexpr int ROWS_BLOCK = 1024;

// One workgroup: the rows that count, in order.
__global__ __launch_bounds__(ROWS_BLOCK) void kept_rows_kernel(RowsArgs a) {
  __shared__ int sums[ROWS_BLOCK / 64];
  __shared__ float tops[ROWS_BLOCK / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  float top = 0;
  for (long r0 = 0; r0 < a.n; r0 += ROWS_BLOCK) {
    const long r = r0 + threadIdx.x;
    const long long t = r < a.n ? a.target[r] : a.ignore;
    const bool keep = r < a.n && t != a.ignore;
    const unsigned long long mask = __ballot(keep);
    if (lane == 0) sums[wave] = __popcll(mask);
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < ROWS_BLOCK / 64; w++) { if (w < wave) before += sums[w]; all += sums[w]; }
    if (keep) {
      const int i = before + __popcll(mask & ((1ull << lane) - 1));
      a.rows[i] = (int)r;
      a.tgt[i] = t >= 0 && t < a.vocab ? (int)t : -1;
      if (a.picked) a.picked[i] = NAN;
      if (a.scale) top = fmaxf(top, fabsf(a.grad[r]));
    } else if (r < a.n) {
      if (a.loss) a.loss[r] = 0.0f;
      if (a.lse) a.lse[r] = 0.0f;
    }
    base += all;
    __syncthreads();
  }
  if (a.scale) {
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 0; w < ROWS_BLOCK / 64; w++) top = fmaxf(top, tops[w]);
      int e = 0;
      if (top > 0.0f && top < INFINITY) { frexpf(top, &e); e = min(max(14 - e, -100), 100); }
      *a.scale = ldexpf(1.0f, e);
    }
  }
  if (threadIdx.x == 0) *a.count = base;
}

template <class T>
__global__ void gather_kernel(const T* from, long ld, T* to, long ldto, const int* rows, const int* count, int width) {
  const long i = blockIdx.x;
  if (i >= *count) return;
  const T* f = from + (long)rows[i] * ld;
  for (int k = threadIdx.x; k < width; k += blockDim.x) to[i * ldto + k] = f[k];
}

__global__ void finish_kernel(const float2* part, int parts, const float* picked, const int* rows, const int* count, float* loss, float* lse) {
  const long i = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (i >= *count) return;
  const int lane = threadIdx.x & 63;
  float2 run = make_float2(-INFINITY, 0.0f);
  for (int k = lane; k < parts; k += 64) run = join(run, part[i * parts + k]);
  for (int o = 32; o; o >>= 1) run = join(run, make_float2(__shfl_xor(run.x, o), __shfl_xor(run.y, o)));
  if (lane == 0) {
    const float l = run.x + logf(run.y);
    lse[rows[i]] = l;
    loss[rows[i]] = l - picked[i];
  }
}


template <class T>
__global__ void scatter_kernel(const float* acc, long ldacc, const int* rows, const int* count, const float* scale, T* out, long ldout, long n, int width) {
  // the rows between one kept row and the next belong to the first of them
  const long i = blockIdx.x;
  const int kept = *count;
  if (i > kept) return;
  const long first = i < kept ? rows[i] : n, before = i ? rows[i - 1] + 1 : 0;
  for (long r = before; r < first; r++)
    for (int k = threadIdx.x; k < width; k += blockDim.x) out[r * ldout + k] = (T)0.0f;
  if (i == kept) return;
  const float s = scale ? 1.0f / *scale : 1.0f;
  for (int k = threadIdx.x; k < width; k += blockDim.x) out[first * ldout + k] = (T)(acc[i * ldacc + k] * s);
}

__global__ void zero_kernel(uint16_t* p, size_t n) {
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0;
}

}  // namespace

int softmax_parts(int N) { return 2 * (int)clr::ceil_div(N, TN); }
void product_gate(const ProductArgs& p, hipStream_t st) { launch<EPI_GATE>(p, st); }
void product_gate_grad(const ProductArgs& p, hipStream_t st) { launch<EPI_GATE_GRAD>(p, st); }
void product_store(const ProductArgs& p, hipStream_t st) { launch<EPI_STORE>(p, st); }
void product_softmax(const ProductArgs& p, hipStream_t st) { launch<EPI_SOFTMAX>(p, st); }
void product_softmax_grad(const ProductArgs& p, hipStream_t st) { launch<EPI_SOFTMAX_GRAD>(p, st); }

void kept_rows(const RowsArgs& a, hipStream_t st) { kept_rows_kernel<<<1, ROWS_BLOCK, 0, st>>>(a); }
void gather_rows(const void* from, long ld, void* to, long ldto, const int* rows, const int* count, long n, int width, int dtype, hipStream_t st) {
  if (!n) return;
  clr::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    gather_kernel<T><<<(unsigned)n, 256, 0, st>>>((const T*)from, ld, (T*)to, ldto, rows, count, width);
  });
}
void softmax_finish(const float2* part, int parts, const float* picked, const int* rows, const int* count, long n, float* loss, float* lse, hipStream_t st) {
  if (n) finish_kernel<<<(unsigned)clr::ceil_div(n, 4), 256, 0, st>>>(part, parts, picked, rows, count, loss, lse);
}
void scatter_rows(const float* acc, long ldacc, const int* rows, const int* count, const float* scale, void* out, long ldout, long n, int width, int dtype,
                  hipStream_t st) {
  clr::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    scatter_kernel<T><<<(unsigned)(n + 1), 256, 0, st>>>(acc, ldacc, rows, count, scale, (T*)out, ldout, n, width);
  });
}
void fill_zero(void* p, size_t bytes, hipStream_t st) {
  const size_t n = bytes / 2;
  if (n) zero_kernel<<<(unsigned)std::min<size_t>(2048, (n + 255) / 256), 256, 0, st>>>((uint16_t*)p, n);
}
