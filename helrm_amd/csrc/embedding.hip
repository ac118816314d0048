// embedding.hip -- rows of a table for ids, and the table's gradient.
//
//   y[i] = scale table[ids[i]],  dtable[v] = scale sum over i with ids[i] = v of dy[i]
//
// The gradient has no atomics: ids are sorted (a stable radix sort, so that
// equal ids keep their order), the sorted ids are cut into pieces of equal
// length, and each piece adds the rows of its runs of equal ids in registers.  A
// run inside a piece is a row of the gradient; what a run has in each of several
// pieces is added in order by a second launch.  So a frequent id is as parallel
// as any, and a result is the same on every run.  Sums are float32, scaled and
// rounded once.
#include <algorithm>
#include "embedding.h"

namespace {

constexpr int BLOCK = 256;

// V neighbouring elements of a row, 16 bytes or one element (rows of any
// alignment: global accesses of 16 bytes need none).
template <class T, int V> struct Pack { T v[V]; };
template <class T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> t;
  __builtin_memcpy(&t, p, sizeof(t));
  return t;
}
template <class T, int V> __device__ __forceinline__ void store_pack(T* p, const float (&v)[V]) {
  Pack<T, V> t;
#pragma unroll
  for (int e = 0; e < V; e++) t.v[e] = (T)v[e];
  __builtin_memcpy(p, &t, sizeof(t));
}
// First element of a row's pack: the last one begins earlier, where the width is not a multiple, and holds some elements again.
template <int V> __device__ __forceinline__ int pack_at(int pack, int width) { return min(pack * V, width - V); }

// Places of a [rows][packs] grid by their number: item `first` + j, j < 2^30.
struct Places {
  long row; int in, packs; float rate;
  __device__ __forceinline__ Places(long first, int packs_) : row(first / packs_), in((int)(first - row * packs_)), packs(packs_), rate(1.0f / packs_) {}
  __device__ __forceinline__ void of(int j, long& r, int& pack) const {
    const int i = in + j;
    int q = (int)(i * rate);   // within one of i / packs: it is under 1,025 unless packs is 1
    int left = i - q * packs;
    if (left < 0) { q--; left += packs; }
    if (left >= packs) { q++; left -= packs; }
    r = row + q;
    pack = left;
  }
};

constexpr int TURNS = 4;   // packs a thread

template <class T, int V>
__global__ __launch_bounds__(BLOCK) void embed_kernel(const EmbedArgs a, int packs, long items, long base) {
  const long first = (base + blockIdx.x) * (BLOCK * TURNS);
  const Places places(first, packs);
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const int j = u * BLOCK + threadIdx.x;
    if (first + j >= items) break;
    long row;
    int pack;
    places.of(j, row, pack);
    const int at = pack_at<V>(pack, a.width);
    const long long id = a.ids[row];
    const bool in = id >= 0 && id < a.vocab && id != a.ignore;
    const Pack<T, V> t = load_pack<T, V>((const T*)a.table + (in ? id : 0) * a.ldtable + at);
    float v[V];
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = in ? (float)t.v[e] * a.scale : id == a.ignore ? 0.0f : NAN;
    store_pack<T, V>((T*)a.y + row * a.ldy + at, v);
  }
}

// ---- the sort ----
// Keys are ids, `vocab` of an id that has no row (sorted last); values are the ids' places.

constexpr int SORT = 1024, WAVES = SORT / 64, MOST_BITS = 9, MOST_DIGITS = 1 << MOST_BITS;
constexpr int ONE_ITEMS = 8, TILE_ITEMS = 4;
constexpr long ONE = SORT * ONE_ITEMS, TILE = SORT * TILE_ITEMS;   // the most that one workgroup sorts alone; a workgroup's share otherwise

struct SortArgs {
  const long long* ids;                     // of the first pass
  const unsigned* from; const unsigned* from_at;
  unsigned* to; unsigned* to_at;
  int* counts;                              // [tiles][digits]
  long long ignore;
  int n, vocab, bits, passes, shift, tiles;
};
__device__ __forceinline__ unsigned key_of(const SortArgs& a, int i) {
  const long long id = a.ids[i];
  return id >= 0 && id < a.vocab && id != a.ignore ? (unsigned)id : (unsigned)a.vocab;
}

// Item j of a lane is number wave * 64 ITEMS + 64 j + lane of the tile; the
// first n of them are there.  rank[j]: how many items of the wave with the same
// digit are before it; counts[wave][digit]: how many the wave has.
template <int ITEMS>
__device__ __forceinline__ void rank_items(const unsigned (&key)[ITEMS], int n, int shift, int bits, int (&rank)[ITEMS], int (*counts)[MOST_DIGITS]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int k = lane; k < 1 << bits; k += 64) counts[wave][k] = 0;
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < ITEMS; j++) {
    const bool there = (wave * ITEMS + j) * 64 + lane < n;
    const unsigned digit = key[j] >> shift & ((1u << bits) - 1);
    unsigned long long same = __ballot(there);
    for (int b = 0; b < bits; b++) {
      const bool bit = digit >> b & 1;
      const unsigned long long set = __ballot(bit);
      same &= bit ? set : ~set;
    }
    const int before = __popcll(same & ((1ull << lane) - 1));
    rank[j] = 0;
    if (there) rank[j] = counts[wave][digit] + before;
    // (a wave's accesses to LDS are in order; the compiler may not keep a count that another lane writes)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (there && before == 0) counts[wave][digit] += __popcll(same);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}
// counts[wave][digit] becomes what the waves before have; the result, of thread `digit`, what all have.
__device__ __forceinline__ int over_waves(int digits, int (*counts)[MOST_DIGITS]) {
  int sum = 0;
  if ((int)threadIdx.x < digits)
    for (int w = 0; w < WAVES; w++) {
      const int c = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = sum;
      sum += c;
    }
  return sum;
}
// The sum of v over the threads before this one.  Two barriers.
__device__ __forceinline__ int before_me(int v, int* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(s, o);
    if (lane >= o) s += t;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  for (int w = 0; w < wave; w++) s += lds[w];
  __syncthreads();
  return s - v;
}

// The whole sort of up to ONE ids.
__global__ __launch_bounds__(SORT) void sort_one_kernel(const SortArgs a) {
  __shared__ int counts[WAVES][MOST_DIGITS], start[MOST_DIGITS], sums[WAVES];
  __shared__ unsigned keys[ONE], ats[ONE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned key[ONE_ITEMS], at[ONE_ITEMS];
  int rank[ONE_ITEMS];
#pragma unroll
  for (int j = 0; j < ONE_ITEMS; j++) {
    const int i = (wave * ONE_ITEMS + j) * 64 + lane;
    key[j] = i < a.n ? key_of(a, i) : 0;
    at[j] = i;
  }
  for (int pass = 0; pass < a.passes; pass++) {
    const int shift = pass * a.bits;
    rank_items<ONE_ITEMS>(key, a.n, shift, a.bits, rank, counts);
    __syncthreads();
    const int base = before_me(over_waves(1 << a.bits, counts), sums);
    if ((int)threadIdx.x < 1 << a.bits) start[threadIdx.x] = base;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ONE_ITEMS; j++)
      if ((wave * ONE_ITEMS + j) * 64 + lane < a.n) {
        const unsigned digit = key[j] >> shift & ((1u << a.bits) - 1);
        const int to = start[digit] + counts[wave][digit] + rank[j];
        keys[to] = key[j];
        ats[to] = at[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ONE_ITEMS; j++) {
      const int i = (wave * ONE_ITEMS + j) * 64 + lane;
      key[j] = i < a.n ? keys[i] : 0;
      at[j] = i < a.n ? ats[i] : 0;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < ONE_ITEMS; j++) {
    const int i = (wave * ONE_ITEMS + j) * 64 + lane;
    if (i < a.n) {
      a.to[i] = key[j];
      a.to_at[i] = at[j];
    }
  }
}

// One pass over many tiles: how often each digit is in a tile, ...
__global__ __launch_bounds__(SORT) void count_kernel(const SortArgs a) {
  __shared__ int counts[MOST_DIGITS];
  const int digits = 1 << a.bits, first = blockIdx.x * (int)TILE;
  for (int k = threadIdx.x; k < digits; k += SORT) counts[k] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < TILE_ITEMS; j++) {
    const int i = first + j * SORT + threadIdx.x;
    if (i < a.n) atomicAdd(&counts[(a.shift ? a.from[i] : key_of(a, i)) >> a.shift & (digits - 1)], 1);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < digits; k += SORT) a.counts[(long)blockIdx.x * digits + k] = counts[k];
}
// ... (of many tiles) in the tiles before, and in all, in a row behind the last; 64 digits a workgroup, ...
constexpr int FEW_TILES = 128;   // the most that every workgroup adds up by itself
__global__ __launch_bounds__(SORT) void scan_kernel(const SortArgs a) {
  __shared__ int sums[WAVES][64];
  const int digits = 1 << a.bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digit = blockIdx.x * 64 + lane;
  const int from = (int)((long)a.tiles * wave / WAVES), to = (int)((long)a.tiles * (wave + 1) / WAVES);
  const bool in = digit < digits;
  int sum = 0;
  if (in)
#pragma unroll 8
    for (int t = from; t < to; t++) sum += a.counts[(long)t * digits + digit];
  sums[wave][lane] = sum;
  __syncthreads();
  sum = 0;
  for (int w = 0; w < wave; w++) sum += sums[w][lane];
  if (!in) return;
#pragma unroll 8
  for (int t = from; t < to; t++) {
    const int c = a.counts[(long)t * digits + digit];
    a.counts[(long)t * digits + digit] = sum;
    sum += c;
  }
  if (wave == WAVES - 1) a.counts[(long)a.tiles * digits + digit] = sum;
}
// ... and every item to its place.
__global__ __launch_bounds__(SORT) void scatter_kernel(const SortArgs a) {
  __shared__ int counts[WAVES][MOST_DIGITS], start[MOST_DIGITS], sums[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << a.bits, tile = blockIdx.x, first = tile * (int)TILE;
  unsigned key[TILE_ITEMS], at[TILE_ITEMS];
  int rank[TILE_ITEMS];
  const int n = min((int)TILE, a.n - first);
#pragma unroll
  for (int j = 0; j < TILE_ITEMS; j++) {
    const int i = (wave * TILE_ITEMS + j) * 64 + lane;
    key[j] = i >= n ? 0 : a.shift ? a.from[first + i] : key_of(a, first + i);
    at[j] = i >= n ? 0 : a.shift ? a.from_at[first + i] : first + i;
  }
  rank_items<TILE_ITEMS>(key, n, a.shift, a.bits, rank, counts);
  int before = 0, all = 0;
  if ((int)threadIdx.x < digits) {
    if (a.tiles > FEW_TILES) {
      before = a.counts[(long)tile * digits + threadIdx.x];
      all = a.counts[(long)a.tiles * digits + threadIdx.x];
    } else {
#pragma unroll 8
      for (int t = 0; t < a.tiles; t++) {
        const int c = a.counts[t * digits + threadIdx.x];
        all += c;
        if (t < tile) before += c;
      }
    }
  }
  __syncthreads();
  over_waves(digits, counts);
  const int base = before_me(all, sums);
  if ((int)threadIdx.x < digits) start[threadIdx.x] = base + before;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < TILE_ITEMS; j++)
    if ((wave * TILE_ITEMS + j) * 64 + lane < n) {
      const unsigned digit = key[j] >> a.shift & (digits - 1);
      const int to = start[digit] + counts[wave][digit] + rank[j];
      a.to[to] = key[j];
      a.to_at[to] = at[j];
    }
}

// ---- the sums ----

struct SumArgs {
  const unsigned* keys; const unsigned* ats;   // sorted
  const void* dy; long lddy;
  void* dtable;
  float* partial;              // [pieces][2][width]: what a run that began in a piece before has in this one, and one that goes on behind
  int n, vocab, width, packs;
  int piece, pieces;           // length and number
  int lanes, blocks;           // of a team, which adds `lanes` packs of the rows of a piece; teams beside one another
  float scale;
};

// WAVE: a team is a wave.
template <class T, int V, bool WAVE>
__global__ __launch_bounds__(BLOCK) void sum_kernel(const SumArgs a, long base) {
  constexpr int AHEAD = 8;
  const int lane = WAVE ? threadIdx.x & 63 : threadIdx.x & (a.lanes - 1);
  unsigned team = (unsigned)(((base + blockIdx.x) * BLOCK + threadIdx.x) / (WAVE ? 64 : a.lanes));
  if (WAVE) team = __builtin_amdgcn_readfirstlane(team);
  const unsigned piece = team / a.blocks;
  const int pack = (int)(team - piece * a.blocks) * a.lanes + lane;
  if (piece >= (unsigned)a.pieces) return;
  const int from = (int)piece * a.piece, to = min(from + a.piece, a.n);
  unsigned cur = a.keys[from];
  if (cur >= (unsigned)a.vocab || pack >= a.packs) return;
  bool before = from > 0 && a.keys[from - 1] == cur;   // the run began in a piece before
  const int at = pack_at<V>(pack, a.width);
  float sum[V] = {};
  auto held = [&](int which) {
    float* p = a.partial + ((long)piece * 2 + which) * a.width + at;
    __builtin_memcpy(p, sum, sizeof(sum));
  };
  auto done = [&] {
    if (before) held(0);
    else {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; e++) v[e] = sum[e] * a.scale;
      store_pack<T, V>((T*)a.dtable + (long)cur * a.width + at, v);
    }
  };
  for (int i = from; i < to; i += AHEAD) {
    unsigned key[AHEAD];
    Pack<T, V> t[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      const int k = min(i + u, to - 1);
      key[u] = a.keys[k];
      t[u] = load_pack<T, V>((const T*)a.dy + a.ats[k] * a.lddy + at);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      if (i + u >= to) break;
      if (key[u] != cur) {
        done();
        if (key[u] >= (unsigned)a.vocab) return;
        cur = key[u];
        before = false;
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] = 0;
      }
#pragma unroll
      for (int e = 0; e < V; e++) sum[e] += (float)t[u].v[e];
    }
  }
  if (!before && to < a.n && a.keys[to] == cur) held(1);
  else done();
}

// The runs that go on over pieces, each by the workgroups of the piece that it begins in: a column block each.
template <class T, int V>
__global__ __launch_bounds__(BLOCK) void join_kernel(const SumArgs a, long base) {
  __shared__ float lds[BLOCK * V];
  const unsigned id = (unsigned)(base + blockIdx.x), piece = id / a.blocks;
  const int from = (int)piece * a.piece, to = from + a.piece;
  if (to >= a.n) return;
  const unsigned key = a.keys[to];
  if (key >= (unsigned)a.vocab || a.keys[to - 1] != key || (from > 0 && a.keys[from - 1] == key)) return;
  // pieces that begin with the run: those behind this one, as long as there are any
  int more = 0;
  for (int q = (int)piece + 1;; q += BLOCK) {
    const int mine = q + threadIdx.x;
    const int n = __syncthreads_count(mine < a.pieces && a.keys[(long)mine * a.piece] == key);
    more += n;
    if (n < BLOCK) break;
  }
  const int lane = threadIdx.x & (a.lanes - 1), team = threadIdx.x / a.lanes, teams = BLOCK / a.lanes;
  const int pack = (int)(id - piece * a.blocks) * a.lanes + lane, at = pack_at<V>(pack, a.width);
  float sum[V] = {};
  if (pack < a.packs)
#pragma unroll 4
    for (int i = team; i <= more; i += teams) {
      float v[V];
      __builtin_memcpy(v, a.partial + (((long)piece + i) * 2 + (i == 0)) * a.width + at, sizeof(v));
#pragma unroll
      for (int e = 0; e < V; e++) sum[e] += v[e];
    }
#pragma unroll
  for (int e = 0; e < V; e++) lds[threadIdx.x * V + e] = sum[e];
  __syncthreads();
  if (team || pack >= a.packs) return;
  for (int t = 1; t < min(teams, more + 1); t++)
#pragma unroll
    for (int e = 0; e < V; e++) sum[e] += lds[(t * a.lanes + lane) * V + e];
#pragma unroll
  for (int e = 0; e < V; e++) sum[e] *= a.scale;
  store_pack<T, V>((T*)a.dtable + (long)key * a.width + at, sum);
}

template <class T, int V>
__global__ __launch_bounds__(BLOCK) void clear_kernel(T* table, int width, int packs, long items, long base) {
  const long first = (base + blockIdx.x) * (BLOCK * TURNS);
  const Places places(first, packs);
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const int j = u * BLOCK + threadIdx.x;
    if (first + j >= items) break;
    long row;
    int pack;
    places.of(j, row, pack);
    const float v[V] = {};
    store_pack<T, V>(table + row * width + pack_at<V>(pack, width), v);
  }
}

// f(T{}, V): packs of 16 bytes, or single elements of rows that have no 16 bytes
template <class F> void with_packs(int dtype, int width, F&& f) {
  clr::with_type(dtype, [&](auto t) {
    constexpr int V = 16 / sizeof(t);
    if (width >= V) f(t, std::integral_constant<int, V>{});
    else f(t, std::integral_constant<int, 1>{});
  });
}
int packs_of(int width, int dtype) {
  const int v = 16 / dtype_size(dtype);
  return width >= v ? (int)clr::ceil_div(width, v) : width;
}

// The pieces of the workspace, or only their bytes.
struct Space {
  unsigned *keys[2], *ats[2];
  int* counts;
  float* partial;
  size_t bytes = 0;
};
// Ids of a piece: as few as leave 2,048 teams, of 16 to 64.
int piece_of(long tokens, int blocks, int lanes) {
  const long teams = tokens * blocks * lanes / 64 / 2048;
  return teams >= 64 ? 64 : teams >= 32 ? 32 : 16;
}
int lanes_of(int packs) {
  int n = 1;
  while (n < 64 && n < packs) n *= 2;
  return n;
}
Space space_of(char* base, long tokens, int width, int vocab, int dtype) {
  Space s;
  auto take = [&](size_t n) {
    char* p = base ? base + s.bytes : nullptr;
    s.bytes += clr::align256(n);
    return p;
  };
  const int packs = packs_of(width, dtype), lanes = lanes_of(packs), blocks = (int)clr::ceil_div(packs, lanes);
  const bool one = tokens <= ONE;
  for (int i = 0; i < 2; i++) {
    s.keys[i] = i && one ? s.keys[0] : (unsigned*)take(tokens * 4);
    s.ats[i] = i && one ? s.ats[0] : (unsigned*)take(tokens * 4);
  }
  s.counts = one ? nullptr : (int*)take((clr::ceil_div(tokens, TILE) + 1) * MOST_DIGITS * 4);
  s.partial = (float*)take(clr::ceil_div(tokens, piece_of(tokens, blocks, lanes)) * 2 * width * sizeof(float));
  return s;
}

}  // namespace

void embedding_launch(const EmbedArgs& a, hipStream_t st) {
  const int packs = packs_of(a.width, a.dtype);
  const long items = a.tokens * packs;
  with_packs(a.dtype, a.width, [&](auto t, auto v) {
    clr::in_launches(clr::ceil_div(items, BLOCK * TURNS), BLOCK,
                     [&](long base, unsigned n) { embed_kernel<decltype(t), decltype(v)::value><<<n, BLOCK, 0, st>>>(a, packs, items, base); });
  });
}

size_t embedding_grad_workspace(long tokens, int width, int vocab, int dtype) { return space_of(nullptr, tokens, width, vocab, dtype).bytes; }

void embedding_grad_launch(const EmbedArgs& a, hipStream_t st) {
  const Space space = space_of((char*)a.workspace, a.tokens, a.width, a.vocab, a.dtype);
  const int packs = packs_of(a.width, a.dtype);
  const long items = (long)a.vocab * packs;
  with_packs(a.dtype, a.width, [&](auto t, auto v) {
    clr::in_launches(clr::ceil_div(items, BLOCK * TURNS), BLOCK, [&](long base, unsigned n) {
      using T = decltype(t);
      clear_kernel<T, decltype(v)::value><<<n, BLOCK, 0, st>>>((T*)a.dtable, a.width, packs, items, base);
    });
  });
  if (!a.tokens) return;
  SortArgs s{};
  s.ids = a.ids;
  s.ignore = a.ignore;
  s.n = (int)a.tokens;
  s.vocab = a.vocab;
  int bits = 1;
  while (a.vocab >> bits) bits++;
  s.passes = (int)clr::ceil_div(bits, MOST_BITS);
  s.bits = (int)clr::ceil_div(bits, s.passes);
  int out = 0;
  if (a.tokens <= ONE) {
    s.to = space.keys[0];
    s.to_at = space.ats[0];
    sort_one_kernel<<<1, SORT, 0, st>>>(s);
  } else {
    s.tiles = (int)clr::ceil_div(a.tokens, TILE);
    s.counts = space.counts;
    for (int pass = 0; pass < s.passes; pass++) {
      out = pass & 1;
      s.shift = pass * s.bits;
      s.from = space.keys[1 - out];
      s.from_at = space.ats[1 - out];
      s.to = space.keys[out];
      s.to_at = space.ats[out];
      count_kernel<<<s.tiles, SORT, 0, st>>>(s);
      if (s.tiles > FEW_TILES) scan_kernel<<<(unsigned)clr::ceil_div(1 << s.bits, 64), SORT, 0, st>>>(s);
      scatter_kernel<<<s.tiles, SORT, 0, st>>>(s);
    }
  }
  SumArgs m{};
  m.keys = space.keys[out];
  m.ats = space.ats[out];
  m.dy = a.y; m.lddy = a.ldy;
  m.dtable = a.dtable;
  m.partial = space.partial;
  m.n = (int)a.tokens; m.vocab = a.vocab; m.width = a.width; m.packs = packs;
  m.lanes = lanes_of(packs);
  m.blocks = (int)clr::ceil_div(packs, m.lanes);
  m.piece = piece_of(a.tokens, m.blocks, m.lanes);
  m.pieces = (int)clr::ceil_div(a.tokens, m.piece);
  m.scale = a.scale;
  with_packs(a.dtype, a.width, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const long teams = (long)m.pieces * m.blocks;
    clr::in_launches(clr::ceil_div(teams * m.lanes, BLOCK), BLOCK, [&](long base, unsigned n) {
      if (m.lanes == 64) sum_kernel<T, V, true><<<n, BLOCK, 0, st>>>(m, base);
      else sum_kernel<T, V, false><<<n, BLOCK, 0, st>>>(m, base);
    });
    if (m.pieces > 1)
      clr::in_launches(teams, BLOCK, [&](long base, unsigned n) { join_kernel<T, V><<<n, BLOCK, 0, st>>>(m, base); });
  });
}
