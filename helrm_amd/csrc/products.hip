// products.hip -- matrix products of the gated block and the cross entropy.
//
// C[m][n] = sum_k A(m, k) B(n, k) on v_mfma_f32_16x16x32_{bf16,f16}: products
// of 16-bit elements are exact and every sum is float32.  A float32 factor
// is three bfloat16 parts of 8 bits each, x = x0 + x1 + x2, and a product the
// six of their nine products above 2^-24 of it, smallest first; that is as
// exact as a float32 multiplication, on a unit 16 times as fast.  Infinite
// factors and overflows come out as float32's do: the sums of the five smaller
// products are left out where they are not finite, before x0 y0 is added
// (a product within 2^-7 of the largest float32 may already be infinite).
// That takes 1 to 3 % of a float32 product, in kernels of its own.
//
// A workgroup has a BM x BN tile of C, k advances by 64.  Both factors' tiles
// go from memory to LDS directly (16 bytes a lane, no registers), into one of
// two buffers while the other one is multiplied.
// Elements outside a factor are read as 0 through the bounds of its buffer
// descriptor, so no tile has a special case.  Products whose tiles would
// leave CUs idle are split along k into float32 sums that a second kernel adds
// in order.
//
// LDS layout.  A factor whose rows run along k is held as [row][64 k], its
// 16-byte chunk c of row r at chunk c ^ (r & 7): the 16 rows that a wave reads
// at once lie in all banks.  A factor whose rows run along m (or n) is held
// as [64 k][row] and read through the transposing LDS load, four k of 16 rows
// for 16 lanes; 32 bytes p of row k are at p ^ h(k), h(k) = (k & 3) | (k >> 1 & 4),
// so that the eight k rows that 32 lanes read lie in all banks.
//
// Measured, bfloat16, random values (a library product of 8192 x 8192 x 2048
// here: 1364 TFLOP/s of A B^T, 1180 of A B):
//   A B^T    8192 x 2048 x 8192           204 us   1350 TFLOP/s
//   A B      8192 x 2048 x (8192 + 8192)  412      1335
//   A^T B    3 of 8192 x 2048 x 8192      649      1271
//   gate     8192 x 8192 x 2048, twice    534      1029 (670 MB of results)
//   its gradient  8192 x 8192 x 2048      425       647 (940 MB in and out: 190 us of a copy)
//   softmax  8192 x 131072 x 2048        3555      1237
// Bound by power first: with zeros for data the same instructions reach 1500
// TFLOP/s, with random values the clock falls to 1.57 GHz and the matrix units
// are busy 64 % of the time.  The gate and its gradient are bound by memory at
// the end of a tile, when a CU does nothing else.
#include "products.h"
#include "tiles.h"

namespace {

using clr::STEP;
constexpr int XCDS = 8;
// Products of one launch, in the order of their workgroups.
struct Batch {
  ProductArgs p[3];
  int first[3];
  int count;
  __device__ __forceinline__ int which(int block) const { return count > 2 && block >= first[2] ? 2 : count > 1 && block >= first[1] ? 1 : 0; }
};
constexpr unsigned OUTSIDE = 0x80000000u;  // an offset past every descriptor's bound

enum Epi { EPI_STORE, EPI_GATE, EPI_GATE_GRAD, EPI_SOFTMAX, EPI_SOFTMAX_GRAD };

__device__ __forceinline__ u16 bits(__bf16 v) { return __builtin_bit_cast(u16, v); }
__device__ __forceinline__ u16 bits(_Float16 v) { return __builtin_bit_cast(u16, v); }
template <class T> __device__ __forceinline__ uint2 pack4(const float v[4]) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const f32x4 f = {v[0], v[1], v[2], v[3]};
  return __builtin_bit_cast(uint2, __builtin_convertvector(f, T4));
}
// Four neighbouring elements into an intermediate in the layout of a factor
// (8-byte aligned; a float32 operator's: three parts, `part` elements apart; of
// 16 bits: two parts, or one and no `part`).
template <class T> __device__ __forceinline__ void put_held(u16* o, int type, long part, const float v[4]) {
  if (type == DT_F32) {
    float r[3][4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      __bf16 s[3];
      split3(v[e], s);
#pragma unroll
      for (int k = 0; k < 3; k++) r[k][e] = (float)s[k];
    }
#pragma unroll
    for (int k = 0; k < 3; k++) *(uint2*)(o + k * part) = pack4<__bf16>(r[k]);
    return;
  }
  *(uint2*)o = pack4<T>(v);
  if (part) {
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float first = (float)(T)v[e];
      r[e] = isfinite(first) ? v[e] - first : 0.0f;
    }
    *(uint2*)(o + part) = pack4<T>(r);
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
    if (n >= 4 && ((uintptr_t)o & 7) == 0) *(uint2*)o = pack4<T>(v);
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

// The first `left` of four neighbouring columns of a product, at element `at` of c.
template <class T> __device__ __forceinline__ void store4(const ProductArgs& p, long at, int left, float v[4]) {
  if (p.add) {
    const float* c = (const float*)p.c + at;
#pragma unroll
    for (int e = 0; e < 4; e++) if (e < left) v[e] += c[e];
  }
  if (p.unscale) {
    const float factor = 1.0f / *p.unscale;   // a power of two
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= factor;
  }
  put_out<T>(p.c, p.ctype, at, v, left);
}

// One factor's loads of a step.  ALONG_K: its rows run along k.  R rows of the
// tile, W waves; every wave issues R / 8 / W loads of 1 KiB.
template <bool ALONG_K, int R, int W> struct Loader {
  static constexpr int N = R / 8 / W;
  unsigned off[N];   // of the lane's 16 bytes, from the step's first element: under 2^31, since factors' rows are under 2^21
                     // elements apart, or (dl) all within 2^28 bytes
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
  __device__ __forceinline__ void one(int j, const u16* p, int left, u16* lds, int wave) const {
    __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00027000);
    const unsigned o = kk + (ALONG_K ? 0 : j * PER) < left ? off[j] : OUTSIDE;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(lds + (wave * N + j) * 512), 16, o, 0, 0, 0);
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

// A row's maximum and sum over the tile's columns: over the lane's, over the
// four lanes that share the row, over the waves beside one another.  acc[i][j][e]
// is (m, n) = (mw + 16 i + lane % 16, n_wave + 16 j + 4 (lane / 16) + e).
template <int FM, int FN, int WAVES_M, int WAVES_N>
__device__ __forceinline__ void softmax_piece(const ProductArgs& p, const f32x4 (&acc)[FM][FN], int M, long m0, long n0, int wave_m, int wave_n, int tile_n,
                                              float2* lds) {
  const int lane = threadIdx.x & 63, quad = lane >> 4;
  const int left = (int)min((long)p.N - n0 - wave_n * FN * 16, 1L << 20) - 4 * quad;   // columns from the lane's first one on
  const bool whole = (long)p.N - n0 - wave_n * FN * 16 >= FN * 16;   // of the wave: no bounds
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const int r = (wave_m * FM + i) * 16 + (lane & 15);
    const long m = m0 + r;
    const int t = m < M ? p.target[m] - (int)(p.n0 + n0 + wave_n * FN * 16 + 4 * quad) : -1;   // the target's place from there
    if (t >= 0 && t < FN * 16) {   // (seldom: one tile has it)
#pragma unroll
      for (int c = 0; c < FN * 4; c++) if (16 * (c >> 2) + (c & 3) == t) p.picked[m] = acc[i][c >> 2][c & 3];
    }
    float top = -INFINITY, sum = 0;
    // fmaxf passes over a NaN; its exponential is one again
    if (whole) {
#pragma unroll
      for (int c = 0; c < FN * 4; c++) top = fmaxf(top, acc[i][c >> 2][c & 3]);
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int c = 0; c < FN * 4; c++) sum += __expf(acc[i][c >> 2][c & 3] - base);
    } else {
#pragma unroll
      for (int c = 0; c < FN * 4; c++) if (16 * (c >> 2) + (c & 3) < left) top = fmaxf(top, acc[i][c >> 2][c & 3]);
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int c = 0; c < FN * 4; c++) if (16 * (c >> 2) + (c & 3) < left) sum += __expf(acc[i][c >> 2][c & 3] - base);
    }
    float2 run = make_float2(top, sum);
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) run = join(run, make_float2(__shfl_xor(run.x, o), __shfl_xor(run.y, o)));
    if (lane < 16) lds[r * WAVES_N + wave_n] = run;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < WAVES_M * FM * 16 && m0 + r < M; r += WAVES_M * WAVES_N * 64) {
    float2 run = lds[r * WAVES_N];
#pragma unroll
    for (int k = 1; k < WAVES_N; k++) run = join(run, lds[r * WAVES_N + k]);
    p.part[(m0 + r) * p.parts + tile_n] = run;
  }
}

// What becomes of four neighbouring columns of a row, n columns from the end
// of the matrix (`left`), at element first + at of the results (gate: v of the
// gate, u of the up projection).
// WHOLE: all four columns are there and, of a store, the place takes one vector.
struct RowValues { float lse, grad; int target; };
template <class T, int EPI, bool WHOLE>
__device__ __forceinline__ void emit4(const ProductArgs& p, long first, unsigned at, int left, const RowValues& row, float v[4], float u[4],
                                      const float (&held)[2][4]) {
  if (!WHOLE && left < 4) {
#pragma unroll
    for (int e = 0; e < 4; e++) if (e >= left) v[e] = u[e] = 0.0f;   // the columns that fill a row up are 0
  }
  if (EPI == EPI_STORE) {
    if (!WHOLE) store4<T>(p, first + at, left, v);
    else if (p.ctype == DT_F32) *(float4*)((float*)p.c + first + at) = make_float4(v[0], v[1], v[2], v[3]);
    else *(uint2*)((u16*)p.c + first + at) = pack4<T>(v);
  } else if (EPI == EPI_GATE) {
    float a[4], d[4];
    act4(p.act, p.coef, v, a, d);
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] *= u[e];
    if (p.g) {   // (read again in the backward pass only: past the caches they are written twice as fast)
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, (f32x4*)(p.g + first + at));
      __builtin_nontemporal_store(f32x4{u[0], u[1], u[2], u[3]}, (f32x4*)(p.u + first + at));
    }
    put_held<T>((u16*)p.h + first + at, p.dtype, p.hpart, a);
  } else if (EPI == EPI_GATE_GRAD) {
    float a[4], d[4];
    act4(p.act, p.coef, held[0], a, d);
#pragma unroll
    for (int e = 0; e < 4; e++) {   // (g, u and v are 0 in the columns that fill a row up)
      d[e] *= v[e] * held[1][e];
      v[e] *= a[e];
      a[e] *= held[1][e];
    }
    put_held<T>((u16*)p.dg + first + at, p.dtype, p.hpart, d);
    put_held<T>((u16*)p.du + first + at, p.dtype, p.hpart, v);
    put_held<T>((u16*)p.h + first + at, p.dtype, p.hpart, a);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = __expf(v[e] - row.lse);
    if (row.target >= 0 && row.target < 4) {   // (seldom)
#pragma unroll
      for (int e = 0; e < 4; e++) if (row.target == e) v[e] -= 1.0f;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= row.grad;
    if (!WHOLE && left < 4) {
#pragma unroll
      for (int e = 0; e < 4; e++) if (e >= left) v[e] = 0.0f;
    }
    put_held<T>((u16*)p.c + first + at, p.dtype, p.hpart, v);
  }
}

// Elements from one row of the results to the next, and of a split product's sums (gate: the gate's, then the up projection's).
template <int EPI> __device__ __host__ __forceinline__ long result_ld(const ProductArgs& p) {
  return EPI == EPI_STORE || EPI == EPI_SOFTMAX_GRAD ? p.ldc : p.ldh;
}
template <int EPI> __device__ __host__ __forceinline__ long sum_cols(const ProductArgs& p) { return EPI == EPI_STORE ? (p.N + 3) & ~3 : p.ldh; }
template <int EPI> __device__ __host__ __forceinline__ long sum_ld(const ProductArgs& p) { return sum_cols<EPI>(p) * (EPI == EPI_GATE ? 2 : 1); }

// A wave's accumulators go through its own part of LDS, 64 rows of 64 float32
// columns at a time (16 bytes c of row r at c ^ (r & 15)), so that what is
// stored are whole lines of a row and the code of it is there once.  A place is
// a 32-bit offset from the wave's first element: of up to 128 rows, which are
// under 2^24 elements apart in a caller's result, 2^21 in an intermediate, 2^22
// in split sums; all the rows of a loss's dl are under 2^27 elements, or 2^10
// apart.
template <class T, int EPI, int FM, int FN>
__device__ __forceinline__ void emit(const ProductArgs& p, const f32x4 (&acc)[FM][FN], int M, long mw, long n_wave, int split, float* own) {
  constexpr int LANES = EPI == EPI_GATE ? 8 : 16, ROWS = 64 / LANES;   // of a row; rows a time
  constexpr int GROUP = 4;   // places a lane reads before it writes them: its waits are shared
  const int lane = threadIdx.x & 63, col = lane % LANES;
  // gate: the columns are 16 of the gate, the same 16 of the up projection, 16 of the gate, ...
  const int c = EPI == EPI_GATE ? (col >> 2) * 8 + (col & 3) : col;
  const bool sums = EPI != EPI_SOFTMAX_GRAD && p.splits > 1;
  const unsigned ld = (unsigned)(sums ? sum_ld<EPI>(p) : result_ld<EPI>(p));
  const unsigned second = EPI == EPI_GATE ? (unsigned)sum_cols<EPI>(p) : 0;
  // a store of whole vectors, nothing to add or divide by
  const bool plain = EPI != EPI_STORE || sums || (!p.add && !p.unscale && p.ldc % 4 == 0 && (uintptr_t)p.c % 16 == 0);
  static_assert(FN == 4 && FM % 4 == 0, "64 x 64 a time");
#pragma unroll
  for (int part = 0; part < FM / 4; part++) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = i * 16 + (lane & 15), at = j * 4 + (lane >> 4);
        *(f32x4*)(own + r * 64 + ((at ^ (r & 15)) * 4)) = acc[part * 4 + i][j];
      }
    const long first = (sums ? (long)split * p.M * ld : 0) + mw * ld + n_wave;
    // columns that there are from the lane's first one on, and columns with the zeros that fill an intermediate's row up
    const int left = (int)min((long)p.N - n_wave, 64L) - col * 4;
    const int room = EPI == EPI_STORE ? left : (int)min(((p.N + 7L) & ~7L) - n_wave, 64L) - col * 4;
    const int rows = (int)min(M - mw - part * 64, 64L);
    RowValues mine{};   // of row `lane` of the 64
    if (EPI == EPI_SOFTMAX_GRAD && lane < rows) {
      const long m = mw + part * 64 + lane;
      mine.target = p.target[m];
      mine.lse = p.lse[m];
      mine.grad = mine.target < 0 ? NAN : p.grad[m] * (p.scale ? *p.scale : 1.0f);
    }
    auto places = [&](auto whole_) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole_)::value;
#pragma unroll 1
      for (int r0 = 0; r0 < 64; r0 += ROWS * GROUP) {
        float v[GROUP][4], u[GROUP][4] = {}, held[GROUP][2][4] = {};
        RowValues row[GROUP] = {};
#pragma unroll
        for (int g = 0; g < GROUP; g++) {
          const int r = r0 + g * ROWS + lane / LANES;
          get4(own + r * 64 + ((c ^ (r & 15)) * 4), v[g]);
          if (EPI == EPI_GATE) get4(own + r * 64 + (((c + 4) ^ (r & 15)) * 4), u[g]);
          if (EPI == EPI_SOFTMAX_GRAD)
            row[g] = {__shfl(mine.lse, r), __shfl(mine.grad, r), __shfl(mine.target, r) - (int)(p.n0 + n_wave) - col * 4};
          if (EPI == EPI_GATE_GRAD && !sums && (WHOLE || (r < rows && room > 0))) {
            const unsigned at = (part * 64 + r) * ld + col * 4;
            get4(p.g + first + at, held[g][0]);
            get4(p.u + first + at, held[g][1]);
          }
        }
#pragma unroll
        for (int g = 0; g < GROUP; g++) {
          const int r = r0 + g * ROWS + lane / LANES;
          if (!WHOLE && (r >= rows || room <= 0)) continue;
          const unsigned at = (part * 64 + r) * ld + col * 4;
          if (sums) {
            *(float4*)(p.partial + first + at) = make_float4(v[g][0], v[g][1], v[g][2], v[g][3]);
            if (EPI == EPI_GATE) *(float4*)(p.partial + first + second + at) = make_float4(u[g][0], u[g][1], u[g][2], u[g][3]);
          } else {
            emit4<T, EPI, WHOLE>(p, first, at, left, row[g], v[g], u[g], held[g]);
          }
        }
      }
    };
    if (plain && rows == 64 && p.N - n_wave >= (EPI == EPI_GATE ? 32 : 64)) places(std::true_type{});
    else places(std::false_type{});
  }
}

// Waits until the wave's LDS reads are done, and all but its newest `LEFT`
// loads have arrived, then for the other waves.
__device__ __forceinline__ void everybody() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// Tells the compiler to issue LDS reads one by one between matrix
// instructions, over the first three quarters of them, and to keep both here:
// left to itself it bunches the reads before the barrier that waits for them.
template <int READS, int MULS> __device__ __forceinline__ void spread() {
  constexpr int OVER = MULS * 3 / 4;
  if constexpr (READS > 0) {
#pragma unroll
    for (int i = 0; i < READS; i++) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
#pragma unroll
      for (int m = i * OVER / READS; m < (i + 1) * OVER / READS; m++) __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, MULS - OVER, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// PARTS: the first pairs of factors are corrections.
template <class T, int BM, int BN, int WM, int WN, bool A_K, bool B_K, int EPI, bool PARTS>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(const Batch batch) {
  const int which = batch.which(blockIdx.x);
  const ProductArgs& p = batch.p[which];
  const int id = blockIdx.x - batch.first[which];
  constexpr int W = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int COLS = EPI == EPI_GATE ? BN / 2 : BN;   // columns of C in a tile
  // Arrays of their own, not one: only so does the compiler see that a load into one does not concern reads of another.
  __shared__ __align__(1024) u16 a0[BM * STEP], b0[BN * STEP], a1[BM * STEP], b1[BN * STEP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave / WN, wave_n = wave % WN;
  const int nm = (p.M + BM - 1) / BM, nn = (p.N + COLS - 1) / COLS;
  const int split = id / (nm * nn);
  int tile_m, tile_n;
  tile_of(id - split * nm * nn, nm * nn, nm, nn, tile_m, tile_n);
  const long m0 = (long)tile_m * BM, n0 = (long)tile_n * COLS;
  int M = p.M, K = p.K;
  if (p.count) { if (p.count_k) K = *p.count; else M = *p.count; }
  if (m0 >= M) return;
  // a row along k is filled up with zeros to a multiple of 8
  const int KA = A_K ? (K + 7) & ~7 : K, KB = B_K ? (K + 7) & ~7 : K;

  constexpr int LA = Loader<A_K, BM, W>::N, LB = Loader<B_K, BN, W>::N;
  static_assert(LA == 4 && LB == 4, "the steps below");
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

  const int steps_of = (K + STEP - 1) / STEP;
  const int from = (int)((long)steps_of * p.pairs * split / p.splits), to = (int)((long)steps_of * p.pairs * (split + 1) / p.splits);
  // The place of the loads.  Without a step left every address is outside: nothing is read, the load only counts.
  const long arow = A_K ? m0 * p.lda : m0, brow = B_K ? n0 * p.ldb : n0;
  int pair = steps_of ? from / steps_of : 0, k = (from - pair * steps_of) * STEP, left = to - from;
  const u16 *pa = p.a[0], *pb = p.b[0], *pu = pb;
  auto seek = [&] {
    pa = p.a[pair] + arow + (A_K ? k : k * p.lda);
    pb = p.b[pair] + brow + (B_K ? k : k * p.ldb);
    if (EPI == EPI_GATE) pu = p.b2[pair] + brow + k;
  };
  if (left > 0) seek();
  auto load_a = [&](u16* a, int j) { la.one(j, pa, left > 0 ? KA - k : 0, a, wave); };
  // (the tile's rows by 16: gate, up, gate, ...)
  auto load_b = [&](u16* b, int j) { lb.one(j, EPI == EPI_GATE && (j >> 1 & 1) ? pu : pb, left > 0 ? KB - k : 0, b, wave); };
  auto next = [&] {
    left--;
    k += STEP;
    pa += A_K ? STEP : STEP * p.lda;
    pb += B_K ? STEP : STEP * p.ldb;
    pu += STEP;
    if (k >= K && left > 0) { k = 0; pair++; seek(); }
  };

  // Quarter q of a step multiplies the fragments of A rows' half q / 2 and of k's half q & 1, while those of the next
  // quarter are read; B's fragments of both halves of k stay.
  constexpr int HALF = FM / 2;
  f32x4 acc[FM][FN] = {};
  typename Vec8<T>::type fa[2][HALF], fb[2][FN];
  auto read_b = [&](const u16* b, int q) {
    // the addresses of the fragments are computed anew: kept, they would not fit in the registers
    asm volatile("" : "+v"(rb.flip));
#pragma unroll
    for (int j = 0; j < FN; j++) fb[q & 1][j] = rb.get(b, j, q & 1);
  };
  auto read_a = [&](const u16* a, int q) {
    asm volatile("" : "+v"(ra.flip));
#pragma unroll
    for (int i = 0; i < HALF; i++) fa[q & 1][i] = ra.get(a, (q >> 1) * HALF + i, q & 1);
  };
  auto multiply = [&](int q, int part) {   // of two parts
#pragma unroll
    for (int i = part * HALF / 2; i < (part + 1) * HALF / 2; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) {
        f32x4& c = acc[(q >> 1) * HALF + i][j];
        c = mfma(fb[q & 1][j], fa[q & 1][i], c);
      }
  };
  constexpr int MULS = HALF / 2 * FN, READ_A = HALF * (A_K ? 1 : 2), READ_B = FN * (B_K ? 1 : 2);
  // Step t is in buffer t % 2.  Its eight loads a wave go out one by one among the matrix instructions: sent together
  // they would hold the wave up until the last one is taken.  B of step t + 2 is loaded into step t's place once
  // everybody has step t's fragments of B (the first barrier), half of A once everybody has those of A (the second) and
  // the other half at the beginning of step t + 1.  An odd number of steps is filled up with one of zeros.
  auto step = [&](u16* a, u16* b, u16* na, u16* nb) {
    load_a(na, 2);
    read_b(b, 1);
    multiply(0, 0);
    spread<READ_B, MULS>();
    load_a(na, 3);
    read_a(a, 1);
    multiply(0, 1);
    spread<READ_A, MULS>();
    everybody();
    next();
    load_b(b, 0);
    read_a(a, 2);
    multiply(1, 0);
    spread<READ_A, MULS>();
    load_b(b, 1);
    multiply(1, 1);
    spread<0, MULS>();
    load_b(b, 2);
    read_a(a, 3);
    multiply(2, 0);
    spread<READ_A, MULS>();
    load_b(b, 3);
    multiply(2, 1);
    spread<0, MULS>();
    arrive<4>();   // the next step's loads are there (those of B since are not its), and everybody has this one's fragments
    load_a(a, 0);
    read_a(na, 0);
    multiply(3, 0);
    spread<READ_A, MULS>();
    load_a(a, 1);
    read_b(nb, 0);
    multiply(3, 1);
    spread<READ_B, MULS>();
  };
  // steps of corrections, from the first one here
  const int corrections = steps_of * p.corrections - from;
  auto settle = [&] {
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = settled(acc[i][j]);
  };
  const int total = (to - from + 1) / 2;
  if (total) {
#pragma unroll
    for (int j = 0; j < 4; j++) { load_b(b0, j); load_a(a0, j); }
    next();
#pragma unroll
    for (int j = 0; j < 4; j++) load_b(b1, j);
    load_a(a1, 0);
    load_a(a1, 1);
    arrive<6>();
    read_a(a0, 0);
    read_b(b0, 0);
  }
  for (int t = 0; t < total; t++) {
    if (PARTS && t > 0 && corrections == 2 * t) settle();
    step(a0, b0, a1, b1);
    if (PARTS && corrections == 2 * t + 1) settle();
    step(a1, b1, a0, b0);
  }
  if (PARTS && corrections >= to - from) settle();
  arrive<0>();   // no load may still write LDS when it is used again, or given away
  if constexpr (EPI == EPI_SOFTMAX) {
    softmax_piece<FM, FN, WM, WN>(p, acc, M, m0, n0, wave_m, wave_n, tile_n, (float2*)a0);
  } else {
    const int q = BM == 256 ? wave >> 1 : wave;   // 16 KiB a wave
    u16* mine = (q == 0 ? a0 : q == 1 ? b0 : q == 2 ? a1 : b1) + (BM == 256 ? (wave & 1) * 8192 : 0);
    emit<T, EPI, FM, FN>(p, acc, M, m0 + wave_m * FM * 16, n0 + wave_n * FN * (EPI == EPI_GATE ? 8 : 16), split, (float*)mine);
  }
}

// The sums of split products, four columns a thread, and what becomes of them.
// In the order of the splits, so that a result does not depend on which
// workgroup ends first.  Bound by memory and its launch: 1537 x 1000 over k =
// 2 x 2736 takes 56 us in one piece, 38 in two, 5 of them here.
template <class T, int EPI>
__global__ __launch_bounds__(256) void join_kernel(const Batch batch) {
  const int which = batch.which(blockIdx.x);
  const ProductArgs& p = batch.p[which];
  const long cols = sum_cols<EPI>(p) / 4, i = (blockIdx.x - batch.first[which]) * 256L + threadIdx.x;
  const long m = i / cols, n = (i - m * cols) * 4;
  if (m >= (p.count && !p.count_k ? *p.count : p.M)) return;
  float v[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < p.splits; s++) {
    const float* at = p.partial + ((long)s * p.M + m) * sum_ld<EPI>(p) + n;
    float t[4];
    get4(at, t);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += t[e];
    if (EPI == EPI_GATE) {
      get4(at + cols * 4, t);
#pragma unroll
      for (int e = 0; e < 4; e++) u[e] += t[e];
    }
  }
  const long at = m * result_ld<EPI>(p) + n;
  float held[2][4] = {};
  if (EPI == EPI_GATE_GRAD) {
    get4(p.g + at, held[0]);
    get4(p.u + at, held[1]);
  }
  emit4<T, EPI, false>(p, at, 0, (int)min(p.N - n, 4L), RowValues{}, v, u, held);
}

using clr::Plan;
using clr::plan_of;
using clr::steps_of;

template <class T, bool A_K, bool B_K, int EPI> void launch_type(Batch b, const Plan& plan, hipStream_t st) {
  const long size = plan.tile();
  long tiles = 0, sums = 0;
  Batch j = b;
  for (int i = 0; i < b.count; i++) {
    ProductArgs& p = b.p[i];
    p.splits = j.p[i].splits = plan.splits;
    b.first[i] = (int)tiles;
    j.first[i] = (int)sums;
    tiles += clr::ceil_div(p.M, size) * clr::ceil_div(p.N, EPI == EPI_GATE ? size / 2 : size) * p.splits;
    sums += clr::ceil_div((long)p.M * (sum_cols<EPI>(p) / 4), 256);
  }
  auto go = [&](auto parts) {
    constexpr bool PARTS = decltype(parts)::value;
    if (plan.big) product_kernel<T, 256, 256, 2, 4, A_K, B_K, EPI, PARTS><<<clr::groups_of(tiles, 512), 512, 0, st>>>(b);
    else product_kernel<T, 128, 128, 2, 2, A_K, B_K, EPI, PARTS><<<clr::groups_of(tiles, 256), 256, 0, st>>>(b);
  };
  // (float16 factors have two parts only where the product is stored)
  bool parts = false;
  for (int i = 0; i < b.count; i++) parts |= b.p[i].corrections > 0;
  if constexpr (EPI == EPI_STORE || std::is_same_v<T, __bf16>) {
    if (parts) go(std::true_type{});
    else go(std::false_type{});
  } else {
    go(std::false_type{});
  }
  if constexpr (EPI == EPI_STORE || EPI == EPI_GATE || EPI == EPI_GATE_GRAD)
    if (plan.splits > 1) join_kernel<T, EPI><<<clr::groups_of(sums, 256), 256, 0, st>>>(j);
}
template <bool A_K, bool B_K, int EPI> void launch(std::initializer_list<ProductArgs> products, const Plan& plan, hipStream_t st) {
  Batch b{};
  for (const ProductArgs& p : products) if (p.M > 0 && p.N > 0) b.p[b.count++] = p;
  if (!b.count) return;
  if (b.p[0].dtype == DT_F16) launch_type<_Float16, A_K, B_K, EPI>(b, plan, st);
  else launch_type<__bf16, A_K, B_K, EPI>(b, plan, st);
}
template <bool A_K, bool B_K, int EPI> void launch(const ProductArgs& p, hipStream_t st) {
  constexpr bool may_split = EPI == EPI_STORE || EPI == EPI_GATE || EPI == EPI_GATE_GRAD;
  launch<A_K, B_K, EPI>({p}, plan_of({{p.M, p.N}}, steps_of(p.K, p.pairs), EPI == EPI_GATE, may_split), st);
}

// Up to 8 matrices into the layout that the tiles are loaded from, one launch:
// rows[i] (or i) of `from` to row i of `to`, filled up with zeros to ldto;
// float32 as three parts.  Bound by memory: 50,021 x 416 float32, 208 MB read
// and written, 45 us = 4.7 TB/s.
struct LayOuts { LayOut j[8]; long first[8]; int count; };
template <class T>
__global__ __launch_bounds__(256) void lay_out_kernel(const LayOuts all, long base) {
  const long id = base + blockIdx.x;
  int which = 0;
  while (which + 1 < all.count && id >= all.first[which + 1]) which++;
  const LayOut& j = all.j[which];
  const long i = id - all.first[which];
  if (j.count && i >= *j.count) return;
  const T* f = (const T*)j.from + (j.rows ? (long)j.rows[i] : i) * j.ld;
  u16* to = (u16*)j.to + i * j.ldto;
  constexpr int V = 16 / sizeof(T);
  if (((uintptr_t)f & 15) == 0 && j.width % V == 0) {
    for (int k = threadIdx.x * V; k < j.ldto; k += 256 * V) {
      T v[V];
      if (k < j.width) __builtin_memcpy(v, __builtin_assume_aligned(f + k, 16), 16);
      else for (int e = 0; e < V; e++) v[e] = (T)0.0f;
      if constexpr (sizeof(T) == 4) {
        float q[3][4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          __bf16 s[3];
          split3(v[e], s);
#pragma unroll
          for (int t = 0; t < 3; t++) q[t][e] = (float)s[t];
        }
#pragma unroll
        for (int t = 0; t < 3; t++) *(uint2*)(to + t * j.part + k) = pack4<__bf16>(q[t]);
      } else {
        __builtin_memcpy(__builtin_assume_aligned(to + k, 16), v, 16);
      }
    }
    return;
  }
  for (int k = threadIdx.x; k < j.ldto; k += 256) {
    const T v = k < j.width ? f[k] : (T)0.0f;
    if constexpr (sizeof(T) == 4) {
      __bf16 s[3];
      split3(v, s);
      for (int t = 0; t < 3; t++) to[t * j.part + k] = bits(s[t]);
    } else {
      to[k] = bits(v);
    }
  }
}

constexpr int ROWS_BLOCK = 1024;

// One workgroup: the rows that count, in order.  Bound by latency (a loop of 1,024 rows a turn): 14 us for 8,192 rows,
// 0.1 % of the loss that so leaves the others out of its products.
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
      if (a.lse_kept) { a.lse_kept[i] = a.lse[r]; a.grad_kept[i] = a.grad[r]; }
      if (a.picked) a.picked[i] = NAN;
      if (a.scale) top = fmaxf(top, fabsf(a.grad[r]));
      if (a.place) a.place[r] = i;
    } else if (r < a.n) {
      if (a.loss) { a.loss[r] = 0.0f; a.lse[r] = 0.0f; }
      if (a.place) a.place[r] = -1;
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

// A wave a row joins its tiles' pieces: 8,192 rows of 512 pieces, 34 MB, 11 us (twice its memory time; one launch of the loss).
__global__ void finish_kernel(const float2* part, int parts, const float* picked, const int* rows, const int* count, float* loss, float* lse, long first) {
  const long i = (first + blockIdx.x) * 4 + (threadIdx.x >> 6);
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

// A workgroup a row, its sums from where kept_rows put it, or zeros: a run of ignored rows is as parallel as any.
// Bound by memory: 8,192 x 2,048 from float32 to bfloat16, 100 MB, 18 us = 5.4 TB/s.
template <class T>
__global__ __launch_bounds__(256) void scatter_kernel(const float* acc, long ldacc, long second, const int* place, const float* scale, T* out, long ldout,
                                                      int width, long base) {
  const long r = base + blockIdx.x, i = place[r];
  const float s = scale ? 1.0f / *scale : 1.0f;
  T* o = out + r * ldout;
  const float* v = acc + i * ldacc;
  if (width % 4 == 0 && (uintptr_t)o % (4 * sizeof(T)) == 0) {   // (ldacc is the width)
    for (int k = threadIdx.x * 4; k < width; k += 1024) {
      float t[4] = {0, 0, 0, 0};
      if (i >= 0) get4(v + k, t);
      if (i >= 0 && second) {
        float l[4];
        get4(v + second + k, l);
#pragma unroll
        for (int e = 0; e < 4; e++) t[e] += settled(l[e]);
      }
      T q[4];
#pragma unroll
      for (int e = 0; e < 4; e++) q[e] = (T)(t[e] * s);
      __builtin_memcpy(__builtin_assume_aligned(o + k, 4 * sizeof(T)), q, sizeof(q));
    }
  } else {
    for (int k = threadIdx.x; k < width; k += 256) o[k] = i < 0 ? (T)0.0f : (T)((v[k] + (second ? settled(v[second + k]) : 0.0f)) * s);
  }
}

// The sum of the losses and the number of rows that have a target: a share of
// them a workgroup, joined in order by a second launch where there are several
// (no atomics, and nothing has to be cleared first).  In 64 bits, so that
// millions of losses cost a mean nothing.  Bound by launches up to 2^20 rows (14
// us a call, with the host's time), by loads in flight beyond: 2^25 rows, 400 MB,
// 139 us = 2.9 TB/s, beside a table's products with each of them.
struct Total { double sum; long count; };
constexpr int TOTAL_BLOCK = 512, TOTAL_ROWS = 4096, TOTAL_MOST = 256;   // rows a workgroup at the least, and workgroups at the most
__device__ __forceinline__ Total total_of(Total t) {
  __shared__ Total lds[TOTAL_BLOCK / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) { t.sum += __shfl_xor(t.sum, o); t.count += __shfl_xor(t.count, o); }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = t;
  __syncthreads();
  t = lds[0];
  for (int k = 1; k < TOTAL_BLOCK / 64; k++) { t.sum += lds[k].sum; t.count += lds[k].count; }
  return t;
}
__device__ __forceinline__ void put_total(Total t, bool mean, float* total, float* factor) {
  const double n = mean ? (double)max(t.count, 1L) : 1.0;
  *total = (float)(t.sum / n);
  *factor = (float)(1.0 / n);
}
__global__ __launch_bounds__(TOTAL_BLOCK) void total_kernel(const float* loss, const long long* target, long long ignore, long n, Total* part, float* total,
                                                           float* factor) {
  Total t{0.0, 0};
#pragma unroll 4
  for (long i = blockIdx.x * (long)TOTAL_BLOCK + threadIdx.x; i < n; i += gridDim.x * (long)TOTAL_BLOCK) {
    t.sum += loss[i];
    if (target) t.count += target[i] != ignore;
  }
  t = total_of(t);
  if (threadIdx.x) return;
  if (gridDim.x > 1) part[blockIdx.x] = t;
  else put_total(t, target, total, factor);
}
__global__ __launch_bounds__(TOTAL_BLOCK) void total_join_kernel(const Total* part, int parts, bool mean, float* total, float* factor) {
  const Total t = total_of((int)threadIdx.x < parts ? part[threadIdx.x] : Total{0.0, 0});
  if (threadIdx.x == 0) put_total(t, mean, total, factor);
}
int total_groups(long n) { return (int)std::max<long>(1, std::min<long>(TOTAL_MOST, n / TOTAL_ROWS)); }

__global__ void zero_kernel(uint16_t* p, size_t n) {
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0;
}

}  // namespace

size_t product_scratch(std::initializer_list<Shape> shapes, long K, int pairs, bool gate) {
  const Plan plan = plan_of(shapes, steps_of(K, pairs), gate, true);
  size_t n = 0;
  if (plan.splits > 1)
    for (const Shape& s : shapes) n += (size_t)plan.splits * s.M * ((s.N + 7) & ~7L) * (gate ? 2 : 1);
  return n * sizeof(float);
}
void product_gate(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_GATE>(p, st); }
void product_gate_grad(const ProductArgs& p, hipStream_t st) { launch<true, false, EPI_GATE_GRAD>(p, st); }
void product_nt(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_STORE>(p, st); }
void product_nn(const ProductArgs& p, hipStream_t st) { launch<true, false, EPI_STORE>(p, st); }
void product_tn(const ProductArgs& p, hipStream_t st) { launch<false, false, EPI_STORE>(p, st); }
void product_tn(ProductArgs a, ProductArgs b, ProductArgs c, hipStream_t st) {
  const Plan plan = plan_of({{a.M, a.N}, {b.M, b.N}, {c.M, c.N}}, steps_of(a.K, a.pairs), false, true);
  auto sums = [&](const ProductArgs& p) { return (size_t)plan.splits * p.M * ((p.N + 7) & ~7L); };
  b.partial = a.partial + (plan.splits > 1 ? sums(a) : 0);
  c.partial = b.partial + (plan.splits > 1 ? sums(b) : 0);
  launch<false, false, EPI_STORE>({a, b, c}, plan, st);
}
void product_softmax(const ProductArgs& p, const clr::SoftmaxPlan& plan, hipStream_t st) {
  for (long v0 = 0; v0 < p.N; v0 += plan.columns) {
    ProductArgs q = p;
    q.n0 = (int)v0;
    q.N = (int)std::min(plan.columns, p.N - v0);
    for (int k = 0; k < q.pairs; k++) q.b[k] += v0 * q.ldb;
    q.parts = plan.parts;
    q.part += v0 / plan.plan.tile();
    launch<true, true, EPI_SOFTMAX>({q}, plan.plan, st);
  }
}
void product_softmax_grad(const ProductArgs& p, hipStream_t st) { launch<true, true, EPI_SOFTMAX_GRAD>(p, st); }

void lay_out(const LayOut* jobs, int n, int dtype, hipStream_t st) {
  LayOuts all{};
  long blocks = 0;
  for (int i = 0; i < n; i++)
    if (jobs[i].n > 0) {
      all.first[all.count] = blocks;
      all.j[all.count++] = jobs[i];
      blocks += jobs[i].n;
    }
  clr::with_type(dtype, [&](auto t) {
    clr::in_launches(blocks, 256, [&](long base, unsigned n) { lay_out_kernel<decltype(t)><<<n, 256, 0, st>>>(all, base); });
  });
}
void kept_rows(const RowsArgs& a, hipStream_t st) { kept_rows_kernel<<<1, ROWS_BLOCK, 0, st>>>(a); }
void softmax_finish(const float2* part, int parts, const float* picked, const int* rows, const int* count, long n, float* loss, float* lse, hipStream_t st) {
  clr::in_launches(clr::ceil_div(n, 4), 256, [&](long first, unsigned k) {
    finish_kernel<<<k, 256, 0, st>>>(part, parts, picked, rows, count, loss, lse, first);
  });
}
void scatter_rows(const float* acc, long ldacc, long second, const int* place, const float* scale, void* out, long ldout, long n, int width, int dtype,
                  hipStream_t st) {
  clr::with_type(dtype, [&](auto t) {
    using T = decltype(t);
    clr::in_launches(n, 256, [&](long base, unsigned k) { scatter_kernel<T><<<k, 256, 0, st>>>(acc, ldacc, second, place, scale, (T*)out, ldout, width, base); });
  });
}
size_t loss_total_bytes(long n) { return total_groups(n) > 1 ? total_groups(n) * sizeof(Total) : 0; }
void loss_total(const float* loss, const long long* target, long long ignore, long n, void* workspace, float* total, float* factor, hipStream_t st) {
  const int groups = total_groups(n);
  total_kernel<<<groups, TOTAL_BLOCK, 0, st>>>(loss, target, ignore, n, (Total*)workspace, total, factor);
  if (groups > 1) total_join_kernel<<<1, TOTAL_BLOCK, 0, st>>>((const Total*)workspace, groups, target, total, factor);
}
void fill_zero(void* p, size_t bytes, hipStream_t st) {
  const size_t n = bytes / 2;
  if (n) zero_kernel<<<(unsigned)std::min<size_t>(2048, (n + 255) / 256), 256, 0, st>>>((uint16_t*)p, n);
}
