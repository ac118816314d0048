// products.hip -- matrix products of the gated block and the cross entropy.
//
// C[m][n] = sum_k A(m, k) B(n, k) on v_mfma_f32_16x16x32_{bf16,f16}: products
// of 16-bit elements are exact and every sum is float32.  A float32 factor
// is three bfloat16 parts of 8 bits each, x = x0 + x1 + x2, and a product the
// six of their nine products above 2^-24 of it, smallest first; that is as
// exact as a float32 multiplication, on a unit 16 times as fast.
//
// A workgroup has a BM x BN tile of C, k advances by 64.  Both factors' tiles
// go from memory to LDS directly (16 bytes a lane, no registers), into one of
// two buffers while the other is multiplied; one barrier a step.  Elements
// outside a factor are read as 0 through the bounds of its buffer
// descriptor, so no tile has a special case.
//
// LDS layout.  A factor whose rows run along k is held as [row][64 k], its
// 16-byte chunk c of row r at chunk c ^ (r & 7): the 16 rows that a wave reads
// at once lie in all banks.  A factor whose rows run along m (or n) is held
// as [64 k][row] and read through the transposing LDS load, four k of 16 rows
// for 16 lanes; 32 bytes p of row k are at p ^ h(k), h(k) = (k & 3) | (k >> 1 & 4),
// so that the eight k rows that 32 lanes read lie in all banks.
#include "products.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16;

constexpr int STEP = 64;                 // k of a step
constexpr int XCDS = 8;
constexpr unsigned OUTSIDE = 0x80000000u;  // an offset past every descriptor's bound

enum Epi { EPI_STORE, EPI_GATE, EPI_GATE_GRAD, EPI_SOFTMAX, EPI_SOFTMAX_GRAD };

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <class T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };

// a = act(g) and d = act'(g) of four values
__device__ __forceinline__ void act4(int act, const float* c, const float g[4], float a[4], float d[4]) {
  if (act == ACT_SILU) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float s = 1.0f / (1.0f + __expf(-g[e]));
      a[e] = g[e] * s;
      d[e] = s * (1.0f + g[e] * (1.0f - s));
    }
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float cdf = 0.5f * (1.0f + erff(g[e] * 0.70710678118654752f));
      a[e] = g[e] * cdf;
      d[e] = cdf + g[e] * __expf(-0.5f * g[e] * g[e]) * 0.39894228040143268f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      a[e] = ((c[3] * g[e] + c[2]) * g[e] + c[1]) * g[e] + c[0];
      d[e] = (3.0f * c[3] * g[e] + 2.0f * c[2]) * g[e] + c[1];
    }
  }
}

// (maximum, sum of exponentials about it) of two pieces of a row.  Where both
// hold nothing above -inf there is nothing to rescale; a NaN stays one.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = a.x > b.x || a.x != a.x ? a.x : b.x;
  if (m == -INFINITY) return make_float2(m, a.y + b.y);
  return make_float2(m, a.y * __expf(a.x - m) + b.y * __expf(b.x - m));
}

// The parts of a float32 value; what is not finite is in the first alone.
__device__ __forceinline__ void split3(float v, __bf16 out[3]) {
  out[0] = (__bf16)v;
  const float r = fabsf((float)out[0]) < INFINITY ? v - (float)out[0] : 0.0f;
  out[1] = (__bf16)r;
  out[2] = (__bf16)(r - (float)out[1]);
}

// Four neighbouring elements into an intermediate in the layout of a factor
// (8-byte aligned; a float32 operator's: three parts, `part` elements apart).
__device__ __forceinline__ u16 bits(__bf16 v) { return __builtin_bit_cast(u16, v); }
__device__ __forceinline__ u16 bits(_Float16 v) { return __builtin_bit_cast(u16, v); }
__device__ __forceinline__ void put8(u16* c, u16 a, u16 b, u16 d, u16 e) {
  *(uint2*)c = make_uint2((unsigned)a | (unsigned)b << 16, (unsigned)d | (unsigned)e << 16);
}
template <class T> __device__ __forceinline__ void put_held(void* c, int type, long part, long at, const float v[4]) {
  u16* o = (u16*)c + at;
  put8(o, bits((T)v[0]), bits((T)v[1]), bits((T)v[2]), bits((T)v[3]));
  if (sizeof(T) == 2 && type == DT_F32) {
    __bf16 s[4][3];
#pragma unroll
    for (int e = 0; e < 4; e++) split3(v[e], s[e]);
#pragma unroll
    for (int k = 1; k < 3; k++) put8(o + k * part, bits(s[0][k]), bits(s[1][k]), bits(s[2][k]), bits(s[3][k]));
  }
}
// The first n of four neighbouring elements of a tensor of the caller's.
template <class T> __device__ __forceinline__ void put_out(void* c, int type, long at, const float v[4], int n) {
  if (type == DT_F32) {
    float* o = (float*)c + at;
    if (n >= 4 && ((uintptr_t)o & 15) == 0) *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
    else {
#pragma unroll
      for (int e = 0; e < 4; e++) if (e < n) o[e] = v[e];
    }
  } else {
    u16* o = (u16*)c + at;
    if (n >= 4 && ((uintptr_t)o & 7) == 0) put8(o, bits((T)v[0]), bits((T)v[1]), bits((T)v[2]), bits((T)v[3]));
    else {
#pragma unroll
      for (int e = 0; e < 4; e++) if (e < n) o[e] = bits((T)v[e]);
    }
  }
}
__device__ __forceinline__ void get4(const float* c, float v[4]) {
  const float4 t = *(const float4*)c;
  v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}

// One factor's loads of a step.  ALONG_K: its rows run along k.  R rows of the
// tile, W waves; every wave issues R / 8 / W loads of 1 KiB.
template <bool ALONG_K, int R, int W> struct Loader {
  static constexpr int N = R / 8 / W;
  unsigned off[N];   // of the lane's 16 bytes, from the step's first element
  int kk;            // the lane's first k (ALONG_K) -- or, of load j, kk + j * PER
  static constexpr int PER = 512 / R;

  // row(r): row r of the tile from the tile's first one, or negative outside
  template <class F> __device__ __forceinline__ void init(long ld, int wave, int lane, F&& row) {
    if (ALONG_K) {
      kk = ((lane & 7) ^ (lane >> 3)) * 8;
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int r = row((wave * N + j) * 8 + (lane >> 3));
        off[j] = r < 0 ? OUTSIDE : (unsigned)(r * ld * 2) + kk * 2;
      }
    } else {
      kk = wave * N * PER + lane / (R / 8);
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int k = kk + j * PER, h = (k & 3) | (k >> 1 & 4);
        const int r = row(((lane % (R / 8)) ^ (h << 1)) * 8);
        off[j] = r < 0 ? OUTSIDE : (unsigned)(k * ld * 2) + r * 2;
      }
    }
  }
  // `left`: k that the factor still has from here on
  template <int J> __device__ __forceinline__ void one(const u16* p, int left, u16* lds, int wave) const {
    __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00027000);
    const unsigned o = kk + (ALONG_K ? 0 : J * PER) < left ? off[J] : OUTSIDE;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(lds + (wave * N + J) * 512), 16, o, 0, 0, 0);
  }
};

// A lane's fragments: 8 k of one of 16 rows, for MFMA's k = 8 (lane / 16) + 0..7.
template <class T, bool ALONG_K, int R> struct Reader {
  typedef typename Vec8<T>::type V;
  unsigned at, flip;
  __device__ __forceinline__ void init(int row0, int lane) {
    if (ALONG_K) {
      at = (row0 + (lane & 15)) * 128;
      flip = ((lane >> 4) ^ (lane & 7)) * 16;
    } else {
      const int g = lane >> 4, i = lane & 15, h = (i >> 2) | (g & 1) << 2;
      at = (g * 8 + (i >> 2)) * R * 2 + (i & 1) * 8 + (i >> 1 & 1) * 16;
      flip = ((row0 / 16) ^ h) * 32;
    }
  }
  // fragment i (rows row0 + 16 i ..) of half-step s (k 32 s ..)
  __device__ __forceinline__ V get(const u16* lds, int i, int s) const {
    typedef __attribute__((address_space(3))) const char* P;
    if (ALONG_K) {
      P p = (P)(const char*)lds + at + i * 2048 + (flip ^ (s * 64));
      return *(__attribute__((address_space(3))) const V*)p;
    } else {
      P p = (P)(const char*)lds + at + s * 32 * R * 2 + (flip ^ (i * 32));
      s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * R * 2));
      return __builtin_bit_cast(V, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Workgroups of one XCD share its L2: consecutive ids go round the XCDs, so
// each XCD is given a run of tiles, 8 rows of tiles wide.
__device__ __forceinline__ void tile_of(int id, int total, int nm, int nn, int& m, int& n) {
  const int x = id % XCDS, q = total / XCDS, r = total % XCDS;
  id = id / XCDS + (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q);
  const int group = id / (8 * nn), first = group * 8, rows = min(8, nm - first), in = id - group * 8 * nn;
  m = first + in % rows;
  n = in / rows;
}

// The wave's accumulators, and what becomes of them.  acc[i][j][e] is
// (m, n) = (mw + 16 i + lane % 16, nw + 16 j + 4 (lane / 16) + e).
template <class T, int EPI, int FM, int FN, int WAVES_N>
__device__ __forceinline__ void finish(const ProductArgs& p, f32x4 (&acc)[FM][FN], long M, long mw, long nw, int lane, int wave_n, int wave_m, int tile_n,
                                       float2* lds) {
  const int quad = lane >> 4;
  if (EPI == EPI_SOFTMAX) {
    // a row's maximum and sum over the tile's columns: over the lane's, over the four lanes that share the row, over
    // the waves beside one another
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const long m = mw + 16 * i + (lane & 15);
      const int t = m < M ? p.target[m] : -1;
      float top = -INFINITY;
      bool nan = false;
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const long n = nw + 16 * j + 4 * quad + e;
          const float v = acc[i][j][e];
          if (n < p.N) { top = fmaxf(top, v); nan |= v != v; }
          if (n < p.N && n == t) p.picked[m] = v;
        }
      if (nan) top = NAN;
      float sum = 0;
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (nw + 16 * j + 4 * quad + e < p.N) sum += top == -INFINITY ? 1.0f : __expf(acc[i][j][e] - top);
      float2 run = make_float2(top, sum);
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) run = join(run, make_float2(__shfl_xor(run.x, o), __shfl_xor(run.y, o)));
      if (lane < 16) lds[((wave_m * FM + i) * 16 + lane) * WAVES_N + wave_n] = run;
    }
    __syncthreads();
    const int rows = blockDim.x / 64 / WAVES_N * FM * 16;
    for (int r = threadIdx.x; r < rows; r += blockDim.x) {
      const long m = mw - wave_m * FM * 16 + r;
      if (m >= M) break;
      float2 run = lds[r * WAVES_N];
#pragma unroll
      for (int k = 1; k < WAVES_N; k++) run = join(run, lds[r * WAVES_N + k]);
      p.part[m * p.parts + tile_n] = run;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const long m = mw + 16 * i + (lane & 15);
    if (m >= M) continue;
    if (EPI == EPI_GATE) {
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        const long n = nw + 8 * j + 4 * quad;
        if (n >= p.ldh) continue;
        float g[4], u[4], h[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {   // the columns that fill a row up are 0
          const bool in = n + e < p.N;
          g[e] = in ? acc[i][j][e] : 0.0f;
          u[e] = in ? acc[i][j + 1][e] : 0.0f;
        }
        act4(p.act, p.coef, g, h, d);
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] *= u[e];
        const long at = m * p.ldh + n;
        if (p.g) { *(float4*)(p.g + at) = make_float4(g[0], g[1], g[2], g[3]); *(float4*)(p.u + at) = make_float4(u[0], u[1], u[2], u[3]); }
        put_held<T>(p.h, p.dtype, p.hpart, at, h);
      }
      continue;
    }
    const int row = EPI == EPI_SOFTMAX_GRAD ? p.rows[m] : 0, t = EPI == EPI_SOFTMAX_GRAD ? p.target[m] : 0;
    const float lse = EPI == EPI_SOFTMAX_GRAD ? p.lse[row] : 0.0f;
    const float grad = EPI == EPI_SOFTMAX_GRAD ? p.grad[row] * (p.scale ? *p.scale : 1.0f) : 0.0f;
    const float factor = EPI == EPI_STORE && p.unscale ? 1.0f / *p.unscale : 1.0f;
#pragma unroll
    for (int j = 0; j < FN; j++) {
      const long n = nw + 16 * j + 4 * quad;
      const int left = (int)(p.N - n);
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = acc[i][j][e];
      if (EPI == EPI_STORE) {
        if (left <= 0) continue;
        if (p.add) {
          const float* c = (const float*)p.c + m * p.ldc + n;
#pragma unroll
          for (int e = 0; e < 4; e++) if (e < left) v[e] += c[e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] *= factor;
        put_out<T>(p.c, p.ctype, m * p.ldc + n, v, left);
      } else if (EPI == EPI_GATE_GRAD) {
        if (n >= p.ldh) continue;
        const long at = m * p.ldh + n;
        float g[4], u[4], a[4], d[4];
        get4(p.g + at, g);
        get4(p.u + at, u);
        act4(p.act, p.coef, g, a, d);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (e >= left) v[e] = 0.0f;   // with g and u of 0, the columns that fill a row up are 0
          d[e] *= v[e] * u[e];
          v[e] *= a[e];
          a[e] *= u[e];
        }
        put_held<T>(p.dg, p.dtype, p.hpart, at, d);
        put_held<T>(p.du, p.dtype, p.hpart, at, v);
        put_held<T>(p.h, p.dtype, p.hpart, at, a);
      } else if (EPI == EPI_SOFTMAX_GRAD) {
        if (n >= ((p.N + 7) & ~7)) continue;   // the row is filled up with zeros to a multiple of 8
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float d = __expf(v[e] - lse);
          if (t == p.n0 + n + e) d -= 1.0f;
          if (t < 0) d = NAN;
          v[e] = e < left ? d * grad : 0.0f;
        }
        put_held<T>(p.c, p.dtype, p.hpart, m * p.ldc + n, v);
      }
    }
  }
}

template <class T, int BM, int BN, int WM, int WN, bool A_K, bool B_K, int EPI>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(const ProductArgs p) {
  constexpr int W = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int COLS = EPI == EPI_GATE ? BN / 2 : BN;   // columns of C in a tile
  __shared__ __align__(1024) u16 a0[BM * STEP], b0[BN * STEP], a1[BM * STEP], b1[BN * STEP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave / WN, wave_n = wave % WN;
  int tile_m, tile_n;
  tile_of(blockIdx.x, gridDim.x, (int)((p.M + BM - 1) / BM), (int)((p.N + COLS - 1) / COLS), tile_m, tile_n);
  const long m0 = (long)tile_m * BM, n0 = (long)tile_n * COLS;
  int M = p.M, K = p.K;
  if (p.count) { if (p.count_k) K = *p.count; else M = *p.count; }
  if (m0 >= M) return;
  // a row along k is filled up with zeros to a multiple of 8
  const int KA = A_K ? (K + 7) & ~7 : K, KB = B_K ? (K + 7) & ~7 : K;

  Loader<A_K, BM, W> la;
  Loader<B_K, BN, W> lb;
  Reader<T, A_K, BM> ra;
  Reader<T, B_K, BN> rb;
  la.init(p.lda, wave, lane, [&](int r) { return m0 + r < (A_K ? M : (p.M + 7) & ~7) ? r : -1; });
  // the gate's rows and the up projection's alternate by 16, so that a lane has both values of a column
  lb.init(p.ldb, wave, lane, [&](int r) {
    if (EPI == EPI_GATE) r = (r >> 5) * 16 + (r & 15);
    return n0 + r < (B_K ? p.N : (p.N + 7) & ~7) ? r : -1;
  });
  ra.init(wave_m * FM * 16, lane);
  rb.init(wave_n * FN * 16, lane);

  const int steps_of = (K + STEP - 1) / STEP, steps = steps_of * p.pairs;
  int pair = 0, k = 0;   // of the next load
  const long arow = A_K ? m0 * p.lda : m0, brow = B_K ? n0 * p.ldb : n0;
  auto load = [&](u16* a, u16* b) {
    const u16* pa = p.a[pair] + arow + (A_K ? k : k * p.lda);
    const u16* pb = p.b[pair] + brow + (B_K ? k : k * p.ldb);
    const int left_a = KA - k, left_b = KB - k;
    la.template one<0>(pa, left_a, a, wave);
    la.template one<1>(pa, left_a, a, wave);
    la.template one<2>(pa, left_a, a, wave);
    la.template one<3>(pa, left_a, a, wave);
    const u16* pu = EPI == EPI_GATE ? p.b2[pair] + brow + k : pb;
    lb.template one<0>(pb, left_b, b, wave);
    lb.template one<1>(pb, left_b, b, wave);
    lb.template one<2>(pu, left_b, b, wave);
    lb.template one<3>(pu, left_b, b, wave);
    k += STEP;
    if (k >= K) { k = 0; pair++; }
  };
  static_assert(Loader<A_K, BM, W>::N == 4 && Loader<B_K, BN, W>::N == 4, "four loads a wave and factor");

  f32x4 acc[FM][FN] = {};
  auto multiply = [&](const u16* a, const u16* b) {
    // the addresses of the fragments are computed anew in every step: kept, they would not fit in the registers
    asm volatile("" : "+v"(ra.flip), "+v"(rb.flip));
#pragma unroll
    for (int s = 0; s < 2; s++) {
      typename Vec8<T>::type fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FN; j++) fb[j] = rb.get(b, j, s);
#pragma unroll
      for (int i = 0; i < FM; i++) fa[i] = ra.get(a, i, s);
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mfma(fb[j], fa[i], acc[i][j]);
    }
  };
  // One step is multiplied while the next one arrives.  The barrier says both that a buffer has arrived and that
  // nobody reads the other one any more.  An odd step comes first, then the two buffers take turns.
  if (steps & 1) {
    load(a1, b1);
    __syncthreads();
    if (steps > 1) load(a0, b0);
    multiply(a1, b1);
  } else if (steps) {
    load(a0, b0);
  }
  for (int t = steps >> 1; t > 0; t--) {
    __syncthreads();
    load(a1, b1);
    multiply(a0, b0);
    __syncthreads();
    if (t > 1) load(a0, b0);
    multiply(a1, b1);
  }
  if (EPI == EPI_SOFTMAX) __syncthreads();
  finish<T, EPI, FM, FN, WN>(p, acc, M, m0 + wave_m * FM * 16, n0 + wave_n * FN * (EPI == EPI_GATE ? 8 : 16), lane, wave_n, wave_m, tile_n, (float2*)a0);
}

template <class T, bool A_K, bool B_K, int EPI> void launch_type(const ProductArgs& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0) return;
  constexpr int half = EPI == EPI_GATE ? 2 : 1;
  // 256 x 256 has half the memory traffic; a launch that would leave most of the 256 CUs without a tile takes 128 x 128
  const long big = clr::ceil_div(p.M, 256) * clr::ceil_div(p.N, 256 / half);
  if (big >= 192 || EPI == EPI_SOFTMAX) {
    product_kernel<T, 256, 256, 2, 4, A_K, B_K, EPI><<<(unsigned)big, 512, 0, st>>>(p);
  } else {
    const long n = clr::ceil_div(p.M, 128) * clr::ceil_div(p.N, 128 / half);
    product_kernel<T, 128, 128, 2, 2, A_K, B_K, EPI><<<(unsigned)n, 256, 0, st>>>(p);
  }
}
template <bool A_K, bool B_K, int EPI> void launch(const ProductArgs& p, hipStream_t st) {
  if (p.dtype == DT_F16) launch_type<_Float16, A_K, B_K, EPI>(p, st);
  else launch_type<__bf16, A_K, B_K, EPI>(p, st);
}

// A factor in the layout that the tiles are loaded from: rows[i] (or i) of
// `from` to row i, filled up with zeros to ldto; float32 as three parts.
template <class T>
__global__ __launch_bounds__(256) void lay_out_kernel(const T* from, long ld, u16* to, long ldto, long part, const int* rows, const int* count, int width) {
  const long i = blockIdx.x;
  if (count && i >= *count) return;
  const T* f = from + (rows ? (long)rows[i] : i) * ld;
  for (int k = blockIdx.y * 256 + threadIdx.x; k < ldto; k += gridDim.y * 256) {
    const T v = k < width ? f[k] : (T)0.0f;
    if constexpr (sizeof(T) == 4) {
      __bf16 s[3];
      split3(v, s);
      for (int j = 0; j < 3; j++) to[j * part + i * ldto + k] = bits(s[j]);
    } else {
      to[i * ldto + k] = bits(v);
    }
  }
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

int softmax_parts(int N) { return (int)clr::ceil_div(N, 256); }
void product_gate(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_GATE>(p, st); }
void product_gate_grad(const ProductArgs& p, hipStream_t st) { launch<true, false, EPI_GATE_GRAD>(p, st); }
void product_nt(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_STORE>(p, st); }
void product_nn(const ProductArgs& p, hipStream_t st) { launch<true, false, EPI_STORE>(p, st); }
void product_tn(const ProductArgs& p, hipStream_t st) { launch<false, false, EPI_STORE>(p, st); }
void product_softmax(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_SOFTMAX>(p, st); }
void product_softmax_grad(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_SOFTMAX_GRAD>(p, st); }

void kept_rows(const RowsArgs& a, hipStream_t st) { kept_rows_kernel<<<1, ROWS_BLOCK, 0, st>>>(a); }
void lay_out(const void* from, long ld, int dtype, void* to, long ldto, long part, const int* rows, const int* count, long n, int width, hipStream_t st) {
  if (!n) return;
  const dim3 grid((unsigned)n, (unsigned)std::min<long>(16, clr::ceil_div(ldto, 256)));
  clr::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    lay_out_kernel<T><<<grid, 256, 0, st>>>((const T*)from, ld, (u16*)to, ldto, part, rows, count, width);
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
