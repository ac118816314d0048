// skinny.hip -- products of a few rows with a matrix: the block and the scores
// of single vectors, where the matrix is read once and nothing else counts.
//
// C[t][n] = sum_k X(t, k) W(n, k) for up to 16 rows t, 64 of float32 (more of
// 16 bits are faster through the tiles: 33 rows against 65,536 x 1,024 bfloat16
// 71 us here and 35 there; of float32, which the tiles need laid out, 148 us
// here and 339 there).  Bound by memory: 16
// rows of W go straight from memory to the registers of a wave, 128 bytes a
// row and turn, and multiply up to four groups of 16 rows of X there
// (v_mfma_f32_16x16x32).  The waves of a workgroup share out k and add their
// sums through LDS, so that a short matrix still keeps every CU loading.
// Nothing is laid out first: rows of any alignment are read 16 bytes at a time,
// but for a row's last odd elements (one row against 65,536 x 1,001: bfloat16 46
// us, 98 an element at a time; float32 60 and 124), and float32 ones are split
// into three bfloat16 parts in registers and multiplied as in products.hip.
//
// Measured: one row against 65,536 x 1,024 bfloat16, 134 MB, 28 us = 4.8 TB/s
// (a copy: 4.95); the gate and up projections of one row of 1,024 to 4,096, 17
// MB, 6.5 us; the down projection, 8 MB, 10.7 us: its 1,024 results are 64
// workgroups, on a quarter of the CUs.
#include "entries.h"
#include "skinny.h"
#include "tiles.h"

namespace {

enum Epi { SKINNY_STORE, SKINNY_GATE, SKINNY_SOFTMAX, SKINNY_TEACH };
constexpr bool is_softmax(int epi) { return epi == SKINNY_SOFTMAX || epi == SKINNY_TEACH; }

// Eight k of a row for one matrix instruction, or the parts of eight float32.
template <class T> struct Eight {
  typename Vec8<T>::type v[1];
};
template <> struct Eight<float> {
  bf16x8 v[3];
};
template <class T> struct Raw { T e[8]; };

template <class T, bool ALIGNED> __device__ __forceinline__ Raw<T> load8(const T* p, int k, int K, bool in) {
  Raw<T> r{};
  if (ALIGNED) {
    if (in && k < K) {
      uint4 q[sizeof(T) / 2];
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; i++) q[i] = ((const uint4*)(p + k))[i];
      __builtin_memcpy(&r, q, sizeof(r));
    }
  } else if (in && k + 8 <= K) {
    __builtin_memcpy(&r, p + k, sizeof(r));   // (global loads of 16 bytes need no alignment)
  } else if (in) {
#pragma unroll
    for (int e = 0; e < 8; e++) if (k + e < K) r.e[e] = p[k + e];
  }
  return r;
}
template <class T> __device__ __forceinline__ Eight<T> eight(const Raw<T>& r) {
  Eight<T> o;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      __bf16 s[3];
      split3(r.e[e], s);
      o.v[0][e] = s[0]; o.v[1][e] = s[1]; o.v[2][e] = s[2];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) o.v[0][e] = r.e[e];
  }
  return o;
}
// The first parts' products are added to c, the corrections to r (settled at the end).
template <class T> __device__ __forceinline__ void dot8(const Eight<T>& w, const Eight<T>& x, f32x4& c, f32x4& r) {
  if constexpr (sizeof(T) == 4) {
    r = mfma(w.v[0], x.v[2], r);
    r = mfma(w.v[1], x.v[1], r);
    r = mfma(w.v[2], x.v[0], r);
    r = mfma(w.v[0], x.v[1], r);
    r = mfma(w.v[1], x.v[0], r);
  }
  c = mfma(w.v[0], x.v[0], c);
}

// The hidden values of a 16-bit block stay float32 here: they are few, and in
// two parts of 8 (11) bits they multiply as exactly as the weights deserve.
template <class T> struct Two {
  typename Vec8<T>::type v[2];
};
template <class T> __device__ __forceinline__ Two<T> two(const Raw<float>& r) {
  Two<T> o;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const T first = (T)r.e[e];
    o.v[0][e] = first;
    o.v[1][e] = (T)(fabsf((float)first) < INFINITY ? r.e[e] - (float)first : 0.0f);
  }
  return o;
}
template <class T> __device__ __forceinline__ void dot8(const Eight<T>& w, const Two<T>& x, f32x4& c, f32x4& r) {
  r = mfma(w.v[0], x.v[1], r);
  c = mfma(w.v[0], x.v[0], c);
}

// A workgroup takes `groups` times 16 rows of W; or, where there are rows
// enough to keep every wave loading, each of its waves does (`alone`), which
// saves the exchange of sums.  Lane l of a wave holds, of a
// group, row l % 16 and the k 16 (l / 16) + 0..15 of 64; its sums are row t = l % 16
// of X and the columns 4 (l / 16) + 0..3.
// What a launch does beside its product.
struct Nothing {};
template <int EPI> using Beside = std::conditional_t<EPI == SKINNY_TEACH, TeachArgs, Nothing>;
template <class T, bool ALIGNED, int NB> constexpr int most_waves() { return sizeof(T) == 2 && ALIGNED && NB == 1 ? 16 : 8; }
// X: the type of x, T or float.
template <class T, class X, bool ALIGNED, int NB, int EPI>
__global__ __launch_bounds__((most_waves<T, ALIGNED, NB>()) * 64) void skinny_kernel(const SkinnyArgs p, const Beside<EPI> beside) {
  constexpr int MATS = EPI == SKINNY_GATE ? 2 : 1, TURNS = !ALIGNED || sizeof(T) == 4 ? 2 : 4;
  extern __shared__ __align__(16) float lds[];   // [waves][MATS * NB][64][4]
  int block = blockIdx.x;
  if constexpr (EPI == SKINNY_TEACH) {
    block -= p.T * beside.parts;
    if (block < 0) {   // the first workgroups (the memory holds up the others meanwhile)
      if (beside.teacher_type == DT_F32) row_entries<T, float>(beside, blockIdx.x, (char*)lds);
      else row_entries<T, T>(beside, blockIdx.x, (char*)lds);
      return;
    }
  }
  const int lane = threadIdx.x & 63, own = threadIdx.x >> 6;
  const int wave = p.alone ? 0 : own, waves = p.alone ? 1 : blockDim.x >> 6;   // of those that share k
  const long team = p.alone ? (long)block * (blockDim.x >> 6) + own : block;
  const int t = lane & 15, quad = lane >> 4;
  float2 run[NB];   // softmax: the team's piece of row t (of wave b)
#pragma unroll
  for (int b = 0; b < NB; b++) run[b] = make_float2(-INFINITY, 0.0f);
  for (int group = 0; group < p.groups; group++) {
    const long n0 = (team * p.groups + group) * 16;
    if (n0 >= p.N) break;
    const bool in = n0 + t < p.N;
    const T* w[2] = {(const T*)p.w + (n0 + t) * p.ldw, MATS == 2 ? (const T*)p.w2 + (n0 + t) * p.ldw2 : nullptr};
    f32x4 acc[MATS][NB] = {}, rest[MATS][NB] = {};
    for (int k0 = wave * 64; k0 < p.K; k0 += waves * 64 * TURNS) {
      Raw<T> raw[MATS][TURNS][2];
#pragma unroll
      for (int u = 0; u < TURNS; u++)
#pragma unroll
        for (int m = 0; m < MATS; m++)
#pragma unroll
          for (int s = 0; s < 2; s++) raw[m][u][s] = load8<T, ALIGNED>(w[m], k0 + u * waves * 64 + quad * 16 + s * 8, p.K, in);
#pragma unroll
      for (int u = 0; u < TURNS; u++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          Eight<T> f[MATS];
#pragma unroll
          for (int m = 0; m < MATS; m++) f[m] = eight(raw[m][u][s]);
#pragma unroll
          for (int b = 0; b < NB; b++) {
            const int row = b * 16 + t;
            const Raw<X> rx = load8<X, ALIGNED>((const X*)p.x + (long)row * p.ldx, k0 + u * waves * 64 + quad * 16 + s * 8, p.K, row < p.T);
            if constexpr (sizeof(X) == sizeof(T)) {
              const Eight<T> x = eight(rx);
#pragma unroll
              for (int m = 0; m < MATS; m++) dot8(f[m], x, acc[m][b], rest[m][b]);
            } else {
              const Two<T> x = two<T>(rx);
#pragma unroll
              for (int m = 0; m < MATS; m++) dot8(f[m], x, acc[m][b], rest[m][b]);
            }
          }
        }
    }
    if constexpr (sizeof(X) == 4) {
#pragma unroll
      for (int m = 0; m < MATS; m++)
#pragma unroll
        for (int b = 0; b < NB; b++) acc[m][b] += settled(rest[m][b]);
    }
    if (waves > 1) {
      if (group) __syncthreads();   // the sums of the group before have been read
#pragma unroll
      for (int m = 0; m < MATS; m++)
#pragma unroll
        for (int b = 0; b < NB; b++) *(f32x4*)(lds + (((wave * MATS + m) * NB + b) * 64 + lane) * 4) = acc[m][b];
      __syncthreads();
    }
#pragma unroll
    for (int b = 0; b < NB; b++) {
      if (b % waves != wave) continue;
      f32x4 sum[MATS];
#pragma unroll
      for (int m = 0; m < MATS; m++) {
        sum[m] = waves > 1 ? f32x4{} : acc[m][b];
        if (waves > 1)
          for (int k = 0; k < waves; k++) sum[m] += *(const f32x4*)(lds + (((k * MATS + m) * NB + b) * 64 + lane) * 4);
      }
      const int row = b * 16 + t;
      const long n = n0 + 4 * quad;
      const int left = (int)min((long)p.N - n, 4L);
      if (is_softmax(EPI)) {
        float top = -INFINITY, s = 0;
        const long long target = EPI == SKINNY_SOFTMAX && row < p.T ? p.target[row] : -1;
        if (EPI == SKINNY_TEACH) sum[0] *= p.rate;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (e < left) top = fmaxf(top, sum[0][e]);
          if (EPI == SKINNY_SOFTMAX && e < left && n + e == target) p.picked[row] = sum[0][e];
        }
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int e = 0; e < 4; e++) if (e < left) s += __expf(sum[0][e] - base);
        float2 piece = make_float2(top, s);
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) piece = join(piece, make_float2(__shfl_xor(piece.x, o), __shfl_xor(piece.y, o)));
        run[b] = join(run[b], piece);
        continue;
      }
      if (row >= p.T) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = sum[0][e];
      if (EPI == SKINNY_GATE) {
        float u[4], a[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          u[e] = e < left ? sum[MATS - 1][e] : 0.0f;
          v[e] = e < left ? v[e] : 0.0f;
        }
        if (p.g && n < p.ldg) {
          *(float4*)(p.g + row * p.ldg + n) = make_float4(v[0], v[1], v[2], v[3]);
          *(float4*)(p.u + row * p.ldg + n) = make_float4(u[0], u[1], u[2], u[3]);
        }
        act4(p.act, p.coef, v, a, d);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = a[e] * u[e];
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (e >= left) continue;
        if (EPI == SKINNY_GATE) ((float*)p.out)[row * p.ldout + n + e] = v[e];
        else ((T*)p.out)[row * p.ldout + n + e] = (T)v[e];
      }
    }
  }
  if (is_softmax(EPI)) {
#pragma unroll
    for (int b = 0; b < NB; b++)
      if (b % waves == wave && lane < 16 && b * 16 + t < p.T && team < p.parts) p.part[(long)(b * 16 + t) * p.parts + team] = run[b];
  }
}

// A workgroup a row: the loss and lse of its pieces, 0 for an ignored row.
constexpr int FINISH = 1024;
__global__ __launch_bounds__(FINISH) void skinny_finish_kernel(const float2* part, int parts, const float* picked, const long long* target, long long ignore,
                                                            int vocab, float* loss, float* lse) {
  __shared__ float2 lds[FINISH / 64];
  const int row = blockIdx.x;
  part += (long)row * parts;
  float2 run = make_float2(-INFINITY, 0.0f);
#pragma unroll 4
  for (int k = threadIdx.x; k < parts; k += FINISH) run = join(run, part[k]);
  for (int o = 32; o; o >>= 1) run = join(run, make_float2(__shfl_xor(run.x, o), __shfl_xor(run.y, o)));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = run;
  __syncthreads();
  if (threadIdx.x) return;
  for (int k = 1; k < FINISH / 64; k++) run = join(run, lds[k]);
  const long long t = target[row];
  const float l = run.x + logf(run.y);
  lse[row] = t == ignore ? 0.0f : l;
  loss[row] = t == ignore ? 0.0f : t < 0 || t >= vocab ? NAN : l - picked[row];
}

// Waves of a workgroup: enough that 2,048 of them are at work where the
// matrix has so few rows, of at least one turn of loads (256 k) each.
int waves_of(int N, int K, int type, int most) {
  int w = 4;
  const int turn = type == DT_F32 ? 128 : 256;
  while (w < most && (long)clr::ceil_div(N, 16) * w < 2048 && K > w * turn) w *= 2;
  return w;
}

template <int EPI> void launch(SkinnyArgs p, hipStream_t st, const Beside<EPI>& beside = {}) {
  if (p.T <= 0 || p.N <= 0) return;
  const long teams = clr::ceil_div(p.N, 16L * p.groups);
  p.alone = teams >= 2048;
  clr::with_type(p.dtype, [&](auto type) {
    using T = decltype(type);
    const long v = 16 / sizeof(T);
    using X = std::conditional_t<EPI == SKINNY_STORE, float, T>;
    auto fits = [&](const void* q, long ld) { return (uintptr_t)q % 16 == 0 && ld % v == 0; };
    const bool aligned = p.K % 8 == 0 && fits(p.x, p.ldx) && fits(p.w, p.ldw) && (EPI != SKINNY_GATE || fits(p.w2, p.ldw2));
    auto go = [&](auto nb) {
      constexpr int NB = decltype(nb)::value;
      const int waves = p.alone ? 4 : waves_of(p.N, p.K, p.dtype, aligned ? most_waves<T, true, NB>() : most_waves<T, false, NB>());
      long groups = p.alone ? clr::ceil_div(teams, 4) : teams;
      size_t lds = (size_t)waves * (EPI == SKINNY_GATE ? 2 : 1) * NB * 1024;
      if constexpr (EPI == SKINNY_TEACH) {
        groups += (long)p.T * beside.parts;
        lds = std::max(lds, entries_bytes(beside.top));
      }
      const unsigned grid = clr::groups_of(groups, waves * 64);
      if (aligned) skinny_kernel<T, X, true, NB, EPI><<<grid, waves * 64, lds, st>>>(p, beside);
      else skinny_kernel<T, X, false, NB, EPI><<<grid, waves * 64, lds, st>>>(p, beside);
    };
    if (p.T <= 16) go(std::integral_constant<int, 1>{});
    if constexpr (sizeof(T) == 4) {
      if (p.T > 16 && p.T <= 32) go(std::integral_constant<int, 2>{});
      else if (p.T > 32) go(std::integral_constant<int, 4>{});
    }
  });
}

}  // namespace

void skinny_gate(SkinnyArgs p, hipStream_t st) { p.groups = 1; launch<SKINNY_GATE>(p, st); }
void skinny_store(SkinnyArgs p, hipStream_t st) { p.groups = 1; launch<SKINNY_STORE>(p, st); }
// Groups of 16 rows a team takes one after another: as many as leave 4,096 teams.
static int softmax_groups(int N) { return (int)std::max<long>(1, N / 16 / 4096); }
int skinny_softmax_parts(int N) { return (int)clr::ceil_div(N, 16L * softmax_groups(N)); }
void skinny_softmax(SkinnyArgs p, long long ignore, float* loss, float* lse, hipStream_t st) {
  p.groups = softmax_groups(p.N);
  p.parts = skinny_softmax_parts(p.N);
  launch<SKINNY_SOFTMAX>(p, st);
  skinny_finish_kernel<<<(unsigned)p.T, FINISH, 0, st>>>(p.part, p.parts, p.picked, p.target, ignore, p.N, loss, lse);
}
void skinny_teach(SkinnyArgs p, const TeachArgs& entries, hipStream_t st) {
  p.groups = softmax_groups(p.N);
  p.parts = skinny_softmax_parts(p.N);
  launch<SKINNY_TEACH>(p, st, entries);
}
