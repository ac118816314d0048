// teacher.hip -- a row's entries in a distillation from a teacher's top logits.
//
//   p = softmax(t / T) over the entries j, s[j] = <x, table[k[j]]> / T, lse = log sum over the table of exp <x, table[v]> / T
//   loss = T^2 sum_j p[j] (log p[j] - (s[j] - lse)),  dl[v] = T (exp(<x, table[v]> / T - lse) - p of v) dloss
//
// The softmax over the table and the products with dl are those of the cross
// entropy (products.hip, skinny.hip).  The entries' scores come out of the
// product's tiles, which are told which of their columns each row wants; or,
// where a row has few of them, from the table's rows themselves.  They are kept for
// the gradient, whose places of the entries are written again from them: the
// difference of two probabilities is taken in float32 and rounded once.
//
// Measured, of 4,096 x 1,024 against 65,536 rows, 64 entries, bfloat16, both
// directions 1,890 us (the cross entropy's 1,880): the entries' order 26 us, the
// product's tiles 25 us more for the scores picked out of them (158 from the
// table's rows, at 3.4 TB/s), the places written again 7 us a piece of the table.
// One row against 65,536 x 1,024: 28 us for the table and, beside it, the entries; 6 to join.
#include <algorithm>
#include "entries.h"
#include "teacher.h"
#include "tiles.h"

namespace {

constexpr int BLOCK = 256;

template <class T, class L>
__global__ __launch_bounds__(BLOCK) void teach_entries_kernel(const TeachArgs a, long base) {
  extern __shared__ __align__(16) char lds[];
  row_entries<T, L>(a, base + blockIdx.x, lds);
}

// A wave a row.  Bound by its launch: 8,192 x 64, 6 MB, 5 us.
template <class L>
__global__ __launch_bounds__(BLOCK) void teach_kept_kernel(const TeachArgs a, long base) {
  const long row = (base + blockIdx.x) * (BLOCK / 64) + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  bool found = false, outside = false;
  for (int j = threadIdx.x & 63; j < a.top; j += 64) {
    float t;
    const int id = entry_of<L>(a, row * a.top + j, t);
    found |= id != NOTHING;
    outside |= id == OUTSIDE;
  }
  const bool any = __ballot(found), out = __ballot(outside);
  if ((threadIdx.x & 63) == 0) a.kept[row] = !any ? TEACH_NONE : out ? TEACH_OUTSIDE : TEACH_FINE;
}

// A workgroup a row that counts: its entries in the order of the table's rows,
// each one's place from a comparison with all.  Bound by those comparisons: 8,192
// rows of 64, a wave a row, 39 us (four waves, three of them idle: 93); 520 of 200,
// four waves, 29.  WAVES: 1 where there are few entries.
constexpr int order_most(int waves) { return waves == 1 ? 64 : MOST_TOP; }
template <class L, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void teach_order_kernel(const TeachArgs a, long base) {
  extern __shared__ __align__(16) char lds[];
  const Entries e(lds, a.top);
  int* leads = (int*)e.behind();     // the table's row of an entry that is the first of its id, else -1
  int* tiles = leads + e.padded;     // of the entries, in order
  const long i = base + blockIdx.x;
  if (i >= *a.count) return;
  const long row = a.which[i], first = row * a.top;
  int any;
  const float top = read_entries<L>(a, row, e, any);
  __syncthreads();
  const float sum = weigh(a, top, e);
  __syncthreads();
  constexpr int MINE = order_most(WAVES) / 64 / WAVES;
  float probs[MINE];
#pragma unroll
  for (int n = 0; n < MINE; n++) {
    const int j = threadIdx.x + n * WAVES * 64;
    if (j >= e.padded) break;
    bool l;
    const float p = together(e, j, l);
    const int id = e.ids[j];
    leads[j] = id >= 0 && l ? id : -1;
    probs[n] = id == OUTSIDE ? NAN : id == NOTHING || !l ? -1.0f : p / sum;
  }
  __syncthreads();
  int entries = 0;   // all of them, of a thread that has a place
#pragma unroll
  for (int n = 0; n < MINE; n++) {
    const int j = threadIdx.x + n * WAVES * 64;
    if (j >= e.padded) break;
    const int id = leads[j];
    int below = 0, others = 0;   // entries of rows before; places that are none before
    entries = 0;
    for (int k = 0; k < e.padded; k += 4) {
      const int4 at = *(const int4*)(leads + k);
      const int q[4] = {at.x, at.y, at.z, at.w};
#pragma unroll
      for (int m = 0; m < 4; m++) {
        entries += q[m] >= 0;
        below += q[m] >= 0 && q[m] < id;
        others += q[m] < 0 && k + m < j;
      }
    }
    const int at = id >= 0 ? below : entries + others;
    if (j < e.top) {
      a.probs[first + at] = probs[n];
      a.cols[first + at] = id;
    }
    if (id >= 0) tiles[at] = id >> a.shift;
  }
  __shared__ int all;   // (waves whose threads have no place have not counted)
  if (threadIdx.x == 0) all = entries;
  __syncthreads();
  uint16_t* starts = a.starts + i * (a.tiles + 1L);
  for (int k = threadIdx.x >> 6; k <= all; k += WAVES) {   // tiles whose first entry is number k
    const int from = k ? tiles[k - 1] + 1 : 0, to = k < all ? tiles[k] : a.tiles;
    for (int t = from + (int)(threadIdx.x & 63); t <= to; t += 64) starts[t] = (uint16_t)k;
  }
}

// WAVES of a workgroup join a row's pieces and add its entries' terms.
template <int WAVES>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void teach_finish_kernel(const TeachFinish a, long base) {
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
__global__ __launch_bounds__(BLOCK) void teach_patch_kernel(const TeachPatch a, int lanes, long base) {
  const long i = (base + blockIdx.x) * (BLOCK / lanes) + threadIdx.x / lanes;
  if (i >= *a.count) return;
  const long first = a.rows[i] * (long)a.top;
  const float grad = a.tgt[i] < 0 ? NAN : a.grad[i] * (a.scale ? *a.scale : 1.0f), lse = a.lse[i];
  for (int j = threadIdx.x % lanes; j < a.top; j += lanes) {
    const long col = a.cols[first + j] - a.v0;
    if (a.cols[first + j] < 0 || col < 0 || col >= a.len) continue;
    const float p = a.probs[first + j];
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

void teach_entries(const TeachArgs& a, hipStream_t st) {
  clr::with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    clr::in_launches(a.rows * a.parts, BLOCK, [&](long base, unsigned n) {
      if (a.teacher_type == DT_F32) teach_entries_kernel<T, float><<<n, BLOCK, entries_bytes(a.top), st>>>(a, base);
      else teach_entries_kernel<T, T><<<n, BLOCK, entries_bytes(a.top), st>>>(a, base);
    });
  });
}
// f(L{}): of the type of the teacher's logits
template <class F> static void with_teacher(const TeachArgs& a, F&& f) { clr::with_type(a.teacher_type, f); }
void teach_kept(const TeachArgs& a, hipStream_t st) {
  with_teacher(a, [&](auto l) {
    clr::in_launches(clr::ceil_div(a.rows, BLOCK / 64), BLOCK, [&](long base, unsigned n) { teach_kept_kernel<decltype(l)><<<n, BLOCK, 0, st>>>(a, base); });
  });
}
void teach_order(const TeachArgs& a, hipStream_t st) {
  const size_t bytes = entries_bytes(a.top) + (size_t)((a.top + 3) & ~3) * 8;
  with_teacher(a, [&](auto l) {
    clr::in_launches(a.rows, BLOCK, [&](long base, unsigned n) {
      if (a.top <= order_most(1)) teach_order_kernel<decltype(l), 1><<<n, 64, bytes, st>>>(a, base);
      else teach_order_kernel<decltype(l), 4><<<n, BLOCK, bytes, st>>>(a, base);
    });
  });
}
void teach_finish(const TeachFinish& a, hipStream_t st) {
  if (a.rows) clr::in_launches(clr::ceil_div(a.n, 4), BLOCK, [&](long base, unsigned n) { teach_finish_kernel<1><<<n, BLOCK, 0, st>>>(a, base); });
  else teach_finish_kernel<16><<<(unsigned)a.n, 1024, 0, st>>>(a, 0);
}
void teach_patch(const TeachPatch& a, hipStream_t st) {
  int lanes = 1;
  while (lanes < BLOCK && lanes < a.top) lanes *= 2;
  clr::with_type(a.dtype, [&](auto t) {
    clr::in_launches(clr::ceil_div(a.n, BLOCK / lanes), BLOCK, [&](long base, unsigned n) { teach_patch_kernel<decltype(t)><<<n, BLOCK, 0, st>>>(a, lanes, base); });
  });
}
