// embedding.hip -- rows of a table for ids, and the table's gradient.
//
//   y[i] = scale table[ids[i]],  dtable[v] = scale sum over i with ids[i] = v of dy[i]
//
// The gradient adds nothing atomically: ids are sorted (a stable radix sort, so
// that equal ids keep their order), the sorted ids are cut into pieces of equal
// length, and each piece adds the rows of its runs of equal ids in registers.  A
// run inside a piece is a row of the gradient; what a run has in each of several
// pieces is added in a fixed order by a second launch.  So a common id is as parallel
// as any, and the same call gives the same result on every run (the length of the
// pieces goes by the row's width and type too: a column beside others of another
// width may differ in its last bit).  Sums are float32, scaled and rounded once.
// The whole table is cleared by workgroups beside the sort's, which hide it
// where it is small and are hidden by it where it is large; rows that an id names
// are so written twice.  (Up to 256 ids, only the rows that no id names are cleared.)
//
// Bound by memory where rows are long (a copy here: 5.0 TB/s), by launches where
// they are few.  131,072 ids x 2,048 against 131,072 rows bfloat16: rows 120-186
// us (537 MB written, the common ids' rows come from the caches), gradient
// 244: 90 for 537 MB cleared beside the sort, 132 for the sums (537 MB read, 155
// written), 22 for the runs over several pieces.  16,384 x 1,024 against 65,536
// rows: rows 11 us, gradient 44: 13 + 10 for the sort with 134 MB cleared beside
// it, 13 and 10 for the sums.  53,248 x 16 float32: 3 us, and 24 + 7 + 6 of short
// launches.
#include <algorithm>
#include "embedding.h"
#include "places.h"

namespace {

constexpr int BLOCK = 256;

// V neighbouring elements of a row, 16 bytes or one element (rows of any
// alignment: global accesses of 16 bytes need none).
typedef unsigned Wide __attribute__((ext_vector_type(4), aligned(2)));
template <class T, int V> struct Pack { T v[V]; };
template <class T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> t;
  __builtin_memcpy(&t, p, sizeof(t));
  return t;
}
// ... that are read once
template <class T, int V> __device__ __forceinline__ Pack<T, V> stream_pack(const T* p) {
  if constexpr (V == 1) return load_pack<T, V>(p);
  else return __builtin_bit_cast(Pack<T, V>, __builtin_nontemporal_load((const Wide*)p));
}
// STREAM: past the caches
template <bool STREAM, class T, int V> __device__ __forceinline__ void store_pack(T* p, const float (&v)[V]) {
  Pack<T, V> t;
#pragma unroll
  for (int e = 0; e < V; e++) t.v[e] = (T)v[e];
  if constexpr (V == 1 || !STREAM) __builtin_memcpy(p, &t, sizeof(t));
  else __builtin_nontemporal_store(__builtin_bit_cast(Wide, t), (Wide*)p);
}
// Results larger than the last-level cache go past it, so that it keeps the
// common ids' rows: 131,072 x 2,048 bfloat16, both directions, 424 us, 433 with
// ordinary stores, 2^20 x 512 498 and 610.  Smaller ones stay for their reader, which costs
// 40,000 x 1,024, 82 MB, 4 us here (91, 87 past the cache).
bool streams(long rows, int width, int dtype) { return (double)rows * width * dtype_size(dtype) > 256L << 20; }

// First element of a row's pack: the last one begins earlier, where the width is not a multiple, and holds some elements again.
template <int V> __device__ __forceinline__ int pack_at(int pack, int width) { return min(pack * V, width - V); }

constexpr int TURNS = 4;   // packs a thread

template <class A> __device__ __forceinline__ bool inside(const A& a, long long id) { return id >= 0 && id < a.vocab && id != a.ignore; }

template <class T, int V, bool STREAM>
__global__ __launch_bounds__(BLOCK) void embed_kernel(const EmbedArgs a, int packs, long items, long base) {
  const long first = (base + blockIdx.x) * (BLOCK * TURNS);
  const Places places(first, packs);
  const int last = (int)min(items - first, (long)BLOCK * TURNS) - 1;   // (the last workgroup's threads do that one again)
  long row[TURNS], id[TURNS];
  int at[TURNS];
  Pack<T, V> t[TURNS];
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    places.of(min(u * BLOCK + (int)threadIdx.x, last), row[u], at[u]);
    at[u] = pack_at<V>(at[u], a.width);
    id[u] = a.ids[row[u]];
  }
#pragma unroll
  for (int u = 0; u < TURNS; u++) t[u] = load_pack<T, V>((const T*)a.table + (inside(a, id[u]) ? id[u] : 0) * a.ldtable + at[u]);
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const bool in = inside(a, id[u]);
    float v[V];
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = in ? (float)t[u].v[e] * a.scale : id[u] == a.ignore ? 0.0f : NAN;
    store_pack<STREAM, T, V>((T*)a.y + row[u] * a.ldy + at[u], v);
  }
}

// ---- the sort ----
// Keys are ids, `vocab` of an id that has no row (sorted last); values are the ids' places.

constexpr int SORT = 1024, WAVES = SORT / 64, MOST_BITS = 9, MOST_DIGITS = 1 << MOST_BITS;
// The most ids that one workgroup sorts alone, and the most whose tiles of SORT
// are sorted each by itself and merged.  Gradient against 65,536 rows, alone and
// merged: 5,120 x 64 25.1 and 23.5 us, 5,120 x 1,024 31.3 and 32.3, 6,144 x 64
// 27.2 and 23.5; merged and by tiles' counts: 16,384 x 1,024 43.5 and 49.8,
// 32,768 x 1,024 56.9 and 59.1 (more ids do not fit into LDS).
constexpr long ONE = SORT * 5, MERGED = SORT * 32;
// Ids a thread of a workgroup's share of more: fewer are done sooner, but every
// workgroup adds up the counts of all (up to FEW_TILES) tiles.  Gradient against
// 65,536 rows x 64 with two and four: 40,000 ids 36.5 and 43.6 us, 65,536 40.7 and
// 45.8, 131,072 53 and 57, 2^20 123 and 119.
int items_of(long tokens) { return tokens <= 64 * SORT ? 2 : 4; }

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
  return inside(a, id) ? (unsigned)id : (unsigned)a.vocab;
}

// Item j < per of a lane is number (wave * per + j) * 64 + lane of the tile; the
// first n of them are there.  rank[j]: how many items of the wave with the same
// digit are before it; counts[wave][digit]: how many the wave has.
template <int ITEMS>
__device__ __forceinline__ void rank_items(const unsigned (&key)[ITEMS], int per, int n, int shift, int bits, int (&rank)[ITEMS], int (*counts)[MOST_DIGITS]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int k = lane; k < 1 << bits; k += 64) counts[wave][k] = 0;
  asm volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < ITEMS; j++) {
    if (j >= per) break;
    const bool there = (wave * per + j) * 64 + lane < n;
    const unsigned digit = key[j] >> shift & ((1u << bits) - 1);
    const unsigned long long all = __ballot(there);
    unsigned low = (unsigned)all, high = (unsigned)(all >> 32);   // lanes with the same digit
#pragma unroll
    for (int b = 0; b < MOST_BITS; b++) {   // (bits that no digit has are equal)
      const int bit = __builtin_amdgcn_sbfe(digit, b, 1);
      const unsigned long long set = __ballot(bit);
      low &= ~((unsigned)set ^ bit);
      high &= ~((unsigned)(set >> 32) ^ bit);
    }
    const int before = __builtin_amdgcn_mbcnt_hi(high, __builtin_amdgcn_mbcnt_lo(low, 0));
    rank[j] = 0;
    if (there) rank[j] = counts[wave][digit] + before;
    // (a wave's accesses to LDS are in order; the compiler may not keep a count that another lane writes)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (there && before == 0) counts[wave][digit] += __popc(low) + __popc(high);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}
// What the waves have of a digit, of thread `digit`.
struct Column {
  int count[WAVES];
  __device__ __forceinline__ int read(int digits, const int (*counts)[MOST_DIGITS]) {
    int sum = 0;
    if ((int)threadIdx.x < digits)
#pragma unroll
      for (int w = 0; w < WAVES; w++) sum += count[w] = counts[w][threadIdx.x];
    return sum;
  }
  // counts[wave][digit] becomes where the wave's first one goes, where those of the digit begin at `first`
  __device__ __forceinline__ void place(int digits, int first, int (*counts)[MOST_DIGITS]) const {
    if ((int)threadIdx.x < digits)
#pragma unroll
      for (int w = 0; w < WAVES; w++) {
        counts[w][threadIdx.x] = first;
        first += count[w];
      }
  }
};
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
#pragma unroll
  for (int w = 0; w < WAVES; w++) s += w < wave ? lds[w] : 0;
  __syncthreads();
  return s - v;
}

// What a launch of the sort does beside it: workgroups behind those of the sort
// clear a share of the table's gradient, which takes longer than the sort where
// the table is large.
struct Clear {
  char* table;
  long first, last;   // places of 16 bytes, or of 2 where a row has less than 16; the last ones of a row overlap
  int packs, groups;
  long row;           // bytes of a row
  bool stream;
};
template <int BYTES> __device__ __forceinline__ void clear_places(const Clear& c, int group) {
  constexpr int EACH = 4;
  for (long first = c.first + (long)group * SORT * EACH; first < c.last; first += (long)c.groups * SORT * EACH) {
    const Places places(first, c.packs);
#pragma unroll
    for (int u = 0; u < EACH; u++) {
      const int j = u * SORT + threadIdx.x;
      if (first + j >= c.last) continue;
      long r;
      int pack;
      places.of(j, r, pack);
      char* p = c.table + r * c.row;
      if constexpr (BYTES == 2) *(uint16_t*)(p + pack * 2) = 0;
      else {
        Wide* to = (Wide*)(p + min((long)pack * 16, c.row - 16));
        if (c.stream) __builtin_nontemporal_store(Wide{0, 0, 0, 0}, to);
        else *to = Wide{0, 0, 0, 0};
      }
    }
  }
}
__device__ __forceinline__ void clear_share(const Clear& c, int group) {
  if (c.row >= 16) clear_places<16>(c, group);
  else clear_places<2>(c, group);
}

// The whole sort of up to SORT * ITEMS ids, or of each of several tiles of so many by itself.
template <int ITEMS>
__global__ __launch_bounds__(SORT) void sort_tile_kernel(const SortArgs a, const Clear c) {
  __shared__ int counts[WAVES][MOST_DIGITS], sums[WAVES];
  __shared__ unsigned keys[SORT * ITEMS], ats[SORT * ITEMS];
  if ((int)blockIdx.x >= a.tiles) return clear_share(c, blockIdx.x - a.tiles);
  const int first = blockIdx.x * SORT * ITEMS, n = min(SORT * ITEMS, a.n - first);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (n + SORT - 1) / SORT;   // (as many for every wave)
  unsigned key[ITEMS], at[ITEMS];
  int rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; j++) {
    const int i = (wave * per + j) * 64 + lane;
    key[j] = j < per && i < n ? key_of(a, first + i) : 0;
    at[j] = first + i;
  }
  for (int pass = 0; pass < a.passes; pass++) {
    const int shift = pass * a.bits;
    rank_items<ITEMS>(key, per, n, shift, a.bits, rank, counts);
    __syncthreads();
    Column column;
    const int all = column.read(1 << a.bits, counts);
    column.place(1 << a.bits, before_me(all, sums), counts);
    __syncthreads();
    const bool last = pass == a.passes - 1;
#pragma unroll
    for (int j = 0; j < ITEMS; j++)
      if (j < per && (wave * per + j) * 64 + lane < n) {
        const unsigned digit = key[j] >> shift & ((1u << a.bits) - 1);
        const int to = counts[wave][digit] + rank[j];
        (last ? a.to + first : keys)[to] = key[j];
        (last ? a.to_at + first : ats)[to] = at[j];
      }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
      const int i = (wave * per + j) * 64 + lane;
      key[j] = j < per && i < n ? keys[i] : 0;
      at[j] = j < per && i < n ? ats[i] : 0;
    }
    // (the next pass writes them after three barriers)
  }
}

// Up to TILES sorted tiles of SORT ids into one: an id goes behind the smaller
// ones of every tile, found by bisection in LDS, and the equal ones of the tiles
// before.  Four threads an id, which share the tiles out.
template <int TILES>
__global__ __launch_bounds__(SORT) void sort_merge_kernel(const SortArgs a, const Clear c) {
  __shared__ __align__(16) unsigned keys[TILES * SORT];
  constexpr int EACH = SORT / 4, MINE = TILES / 4;
  const int groups = (a.n + EACH - 1) / EACH;
  if ((int)blockIdx.x >= groups) return clear_share(c, blockIdx.x - groups);
#pragma unroll
  for (int u = 0; u < MINE; u++) {
    const int i = (u * SORT + threadIdx.x) * 4;
    uint4 v = make_uint4(~0u, ~0u, ~0u, ~0u);   // behind every key
    if (i + 4 <= a.n) v = *(const uint4*)(a.from + i);
    else {
      if (i < a.n) v.x = a.from[i];
      if (i + 1 < a.n) v.y = a.from[i + 1];
      if (i + 2 < a.n) v.z = a.from[i + 2];
    }
    *(uint4*)(keys + i) = v;
  }
  __syncthreads();
  const int e = blockIdx.x * EACH + threadIdx.x / 4, part = threadIdx.x & 3, own = e / SORT;
  const unsigned key = keys[e];
  int at[MINE] = {}, to = 0;
#pragma unroll
  for (int step = SORT / 2; step; step /= 2)
#pragma unroll
    for (int u = 0; u < MINE; u++) {
      const int tile = u * 4 + part;
      at[u] += keys[tile * SORT + at[u] + step - 1] < key + (tile < own) ? step : 0;
    }
#pragma unroll
  for (int u = 0; u < MINE; u++) {
    const int tile = u * 4 + part;
    to += tile == own ? e % SORT : at[u] + (keys[tile * SORT + at[u]] < key + (tile < own));
  }
  to += __shfl_xor(to, 1);
  to += __shfl_xor(to, 2);
  if (part || e >= a.n) return;
  a.to[to] = key;
  a.to_at[to] = a.from_at[e];
}

// One pass over many tiles: how often each digit is in a tile, ...
template <int ITEMS>
__global__ __launch_bounds__(SORT) void sort_count_kernel(const SortArgs a, const Clear c) {
  __shared__ int counts[MOST_DIGITS];
  if ((int)blockIdx.x >= a.tiles) return clear_share(c, blockIdx.x - a.tiles);
  const int digits = 1 << a.bits, first = blockIdx.x * SORT * ITEMS;
  for (int k = threadIdx.x; k < digits; k += SORT) counts[k] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; j++) {
    const int i = first + j * SORT + threadIdx.x;
    if (i < a.n) atomicAdd(&counts[(a.shift ? a.from[i] : key_of(a, i)) >> a.shift & (digits - 1)], 1);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < digits; k += SORT) a.counts[(long)blockIdx.x * digits + k] = counts[k];
}
// ... (of many tiles) in the tiles before, and in all, in a row behind the last; 64 digits a workgroup, ...
constexpr int FEW_TILES = 128;   // the most that every workgroup adds up by itself
__global__ __launch_bounds__(SORT) void sort_scan_kernel(const SortArgs a) {
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
template <int ITEMS>
__global__ __launch_bounds__(SORT) void sort_scatter_kernel(const SortArgs a, const Clear c) {
  __shared__ int counts[WAVES][MOST_DIGITS], sums[WAVES], others[2][MOST_DIGITS];
  if ((int)blockIdx.x >= a.tiles) return clear_share(c, blockIdx.x - a.tiles);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << a.bits, tile = blockIdx.x, first = tile * SORT * ITEMS;
  unsigned key[ITEMS], at[ITEMS];
  int rank[ITEMS];
  const int n = min(SORT * ITEMS, a.n - first);
#pragma unroll
  for (int j = 0; j < ITEMS; j++) {
    const int i = (wave * ITEMS + j) * 64 + lane;
    key[j] = i >= n ? 0 : a.shift ? a.from[first + i] : key_of(a, first + i);
    at[j] = i >= n ? 0 : a.shift ? a.from_at[first + i] : first + i;
  }
  // of thread t's digit t % 512: how many there are in half of the tiles, and in those of them before this one
  const int digit = threadIdx.x & (MOST_DIGITS - 1), half = threadIdx.x / MOST_DIGITS;
  int before = 0, all = 0;
  if (digit < digits) {
    if (a.tiles > FEW_TILES) {
      if (!half) {
        before = a.counts[(long)tile * digits + digit];
        all = a.counts[(long)a.tiles * digits + digit];
      }
    } else {
#pragma unroll 8
      for (int t = half; t < a.tiles; t += 2) {
        const int k = a.counts[t * digits + digit];
        all += k;
        if (t < tile) before += k;
      }
    }
  }
  if (half) {
    others[0][digit] = before;
    others[1][digit] = all;
  }
  rank_items<ITEMS>(key, ITEMS, n, a.shift, a.bits, rank, counts);
  __syncthreads();
  Column column;
  column.read(digits, counts);
  const int base = before_me(half ? 0 : all + others[1][digit], sums);
  column.place(digits, half ? 0 : base + before + others[0][digit], counts);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; j++)
    if ((wave * ITEMS + j) * 64 + lane < n) {
      const unsigned d = key[j] >> a.shift & (digits - 1);
      const int to = counts[wave][d] + rank[j];
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
  int across;                  // lanes of a team that joins
  int group;                   // pieces whose shares of one run are added beforehand, where there are so many pieces
  float scale;
};

// WAVE: a team is a wave.
template <class T, int V, bool WAVE>
__global__ __launch_bounds__(BLOCK) void run_sum_kernel(const SumArgs a, long base) {
  constexpr int AHEAD = 8;   // rows on their way (the gradient of 131,072 x 2,048: 257 us; 268 with 4, 391 with 16, for which there are too few registers)
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
      store_pack<false, T, V>((T*)a.dtable + (long)cur * a.width + at, v);
    }
  };
  for (int i = from; i < to; i += AHEAD) {
    unsigned key[AHEAD];
    Pack<T, V> t[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      const int k = min(i + u, to - 1);
      key[u] = a.keys[k];
      t[u] = stream_pack<T, V>((const T*)a.dy + a.ats[k] * a.lddy + at);
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

// Sums of `items` partial sums, number i of them item(i), a column of packs a
// lane, by the teams of a workgroup; put(at, sum) of each pack.
template <int V, class I, class F> __device__ __forceinline__ void add_partials(const SumArgs& a, int items, float* lds, I&& item, F&& put) {
  const int lane = threadIdx.x & (a.across - 1), team = threadIdx.x / a.across, teams = blockDim.x / a.across;
  for (int first = 0; first < a.packs; first += a.across) {
    const int pack = first + lane, at = pack_at<V>(pack, a.width);
    float sum[V] = {};
    if (pack < a.packs)
#pragma unroll 8
      for (int i = team; i < items; i += teams) {
        float v[V];
        __builtin_memcpy(v, a.partial + item(i) * a.width + at, sizeof(v));
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] += v[e];
      }
    if (first) __syncthreads();
#pragma unroll
    for (int e = 0; e < V; e++) lds[threadIdx.x * V + e] = sum[e];
    __syncthreads();
    if (team || pack >= a.packs) continue;
    for (int t = 1; t < min(teams, items); t++)
#pragma unroll
      for (int e = 0; e < V; e++) sum[e] += lds[(t * a.across + lane) * V + e];
    put(at, sum);
  }
}
// How many of the pieces from, from + step, ... before `end` begin with `key`: those in front, as long as they do.
__device__ __forceinline__ int beginning_with(const SumArgs& a, unsigned key, int from, int step, int end) {
  int count = 0;
  for (long q = from; q < end; q += (long)step * blockDim.x) {
    const long mine = q + (long)step * threadIdx.x;
    const int n = __syncthreads_count(mine < end && a.keys[mine * a.piece] == key);
    count += n;
    if (n < (int)blockDim.x) break;
  }
  return count;
}
// A run that goes on over groups of pieces: what it has in several pieces of one
// is added up, a workgroup a group, into the second place of the first of
// them, which no other run can need: that piece is the run's from end to end.
constexpr int JOIN = 1024;   // the most threads
template <int V>
__global__ __launch_bounds__(JOIN) void run_group_kernel(const SumArgs a, long base) {
  extern __shared__ float lds[];   // [threads][V]
  const int piece = (int)(base + blockIdx.x) * a.group, from = piece * a.piece;
  if (!from) return;
  const unsigned key = a.keys[from];
  if (key >= (unsigned)a.vocab || a.keys[from - 1] != key) return;
  const int items = beginning_with(a, key, piece, 1, min(piece + a.group, a.pieces));
  if (items == 1) return;
  add_partials<V>(a, items, lds, [&](int i) { return ((long)piece + i) * 2; }, [&](int at, const float(&sum)[V]) {
    __builtin_memcpy(a.partial + ((long)piece * 2 + 1) * a.width + at, sum, sizeof(sum));
  });
}
// The runs that go on over pieces, a workgroup for the piece that one begins in:
// most pieces have none.
template <class T, int V>
__global__ __launch_bounds__(JOIN) void run_join_kernel(const SumArgs a, long base) {
  extern __shared__ float lds[];   // [threads][V]
  const int piece = (int)(base + blockIdx.x), from = piece * a.piece, to = from + a.piece;
  if (to >= a.n) return;
  const unsigned key = a.keys[to];
  if (key >= (unsigned)a.vocab || a.keys[to - 1] != key || (from > 0 && a.keys[from - 1] == key)) return;
  // the pieces that it goes on in: the rest of the group, then groups
  const int next = (int)min((piece / a.group + 1L) * a.group, (long)a.pieces);
  const int own = beginning_with(a, key, piece + 1, 1, next), groups = piece + 1 + own == next ? beginning_with(a, key, next, a.group, a.pieces) : 0;
  add_partials<V>(a, 1 + own + groups, lds,
                  [&](int i) {
                    if (i <= own) return ((long)piece + i) * 2 + (i == 0);
                    const long first = next + (i - own - 1L) * a.group;   // of a group
                    return first * 2 + (first + 1 < a.pieces && a.keys[(first + 1) * a.piece] == key);
                  },
                  [&](int at, float(&sum)[V]) {
#pragma unroll
                    for (int e = 0; e < V; e++) sum[e] *= a.scale;
                    store_pack<false, T, V>((T*)a.dtable + (long)key * a.width + at, sum);
                  });
}

template <class F> void with_items(int n, F&& f) {
  if (n <= 1) f(std::integral_constant<int, 1>{});
  else if (n <= 2) f(std::integral_constant<int, 2>{});
  else if (n <= 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

// ---- few ids ----
// One launch: a workgroup an id (and column block), which adds the rows of all
// that are equal if it is the first of them, and others that clear rows of the
// table that no id names.  A workgroup compares all ids, and one id's rows are
// added by one: more ids are sorted.  64 ids x 408 against 960 rows float32, both
// directions, 24 us in four launches, 18 in two (the host's time).
constexpr int FEW = 256;
struct FewArgs {
  EmbedArgs e;
  int packs, blocks, chunk;   // packs of a row; column blocks of BLOCK of them; rows that a workgroup clears
};
constexpr int MOST_CHUNK = 4096;
template <class T, int V>
__global__ __launch_bounds__(BLOCK) void few_kernel(const FewArgs a, long base) {
  __shared__ int ids[FEW], list[FEW];
  __shared__ unsigned named[MOST_CHUNK / 32];
  __shared__ int sums[BLOCK / 64];
  const int n = (int)a.e.tokens, mine = threadIdx.x;
  const long long id = mine < n ? a.e.ids[mine] : a.e.ignore;
  const bool in = mine < n && inside(a.e, id);
  const long block = base + blockIdx.x;
  if (block >= (long)n * a.blocks) {
    const long first = (block - (long)n * a.blocks) * a.chunk;
    const int rows = (int)min((long)a.chunk, a.e.vocab - first);
    for (int k = threadIdx.x; k < MOST_CHUNK / 32; k += BLOCK) named[k] = 0;
    __syncthreads();
    if (in && id >= first && id < first + rows) atomicOr(&named[(id - first) >> 5], 1u << ((id - first) & 31));
    __syncthreads();
    const Places places(0, a.packs);
    const int items = rows * a.packs;   // (under 2^20, or a single row)
    for (int j = threadIdx.x; j < items; j += BLOCK) {
      long r;
      int pack;
      if (rows == 1) { r = 0; pack = j; }
      else places.of(j, r, pack);
      if (named[r >> 5] >> (r & 31) & 1) continue;
      const float zero[V] = {};
      store_pack<false, T, V>((T*)a.e.dtable + (first + r) * a.e.width + pack_at<V>(pack, a.e.width), zero);
    }
    return;
  }
  const int token = (int)(block / a.blocks);
  ids[mine] = in ? (int)id : -1;
  __syncthreads();
  const int key = ids[token];
  const bool same = key >= 0 && ids[mine] == key;
  if (__syncthreads_or((same && mine < token) || key < 0)) return;
  // the equal ones, in order
  const unsigned long long mask = __ballot(same);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) sums[wave] = __popcll(mask);
  __syncthreads();
  int before = __popcll(mask & ((1ull << lane) - 1)), all = 0;
#pragma unroll
  for (int w = 0; w < BLOCK / 64; w++) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  if (same) list[before] = mine;
  __syncthreads();
  const int pack = (int)(block - (long)token * a.blocks) * BLOCK + threadIdx.x;
  if (pack >= a.packs) return;
  const int at = pack_at<V>(pack, a.e.width);
  float sum[V] = {};
#pragma unroll 8
  for (int k = 0; k < all; k++) {
    const Pack<T, V> t = load_pack<T, V>((const T*)a.e.y + list[k] * a.e.ldy + at);
#pragma unroll
    for (int e = 0; e < V; e++) sum[e] += (float)t.v[e];
  }
#pragma unroll
  for (int e = 0; e < V; e++) sum[e] *= a.e.scale;
  store_pack<false, T, V>((T*)a.e.dtable + (long)key * a.e.width + at, sum);
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

// Pieces from which on a launch adds up groups of them before each run is joined
// by a workgroup: 5 us more where runs are short (53,248 x 16, 3,328 pieces, gradient
// 35 us, 41 with it; 2^20 x 64 113 and 120); 2^20 equal ids x 512, 16,384 pieces, 337 us with it and 1,773 without.
constexpr int MANY_PIECES = 4096;
// The pieces of the workspace, or only their bytes.
struct Space {
  unsigned *keys[2], *ats[2];
  int* counts;
  float* partial;
  size_t bytes = 0;
};
// Ids of a piece: as many as leave 2,048 waves, of 16 to 64.  A longer piece has
// fewer sums that are joined, a shorter one keeps more waves at work: gradient of
// 16,384 x 1,024 44 us with 2,048 or 1,024 waves, 50 with 512; of 131,072 x 2,048
// 257 us with pieces of 64, 261 of 128, 270 of 256.
int piece_of(long tokens, int blocks, int lanes) {
  const long waves = tokens * blocks * lanes / 64;
  return waves >= 64 * 2048 ? 64 : waves >= 32 * 2048 ? 32 : 16;
}
int lanes_of(int packs, int most) {
  int n = 1;
  while (n < most && n < packs) n *= 2;
  return n;
}
Space space_of(char* base, long tokens, int width, int vocab, int dtype) {
  Space s;
  auto take = [&](size_t n) {
    char* p = base ? base + s.bytes : nullptr;
    s.bytes += clr::align256(n);
    return p;
  };
  const int packs = packs_of(width, dtype), lanes = lanes_of(packs, 64), blocks = (int)clr::ceil_div(packs, lanes);
  const bool one = tokens <= ONE;
  for (int i = 0; i < 2; i++) {
    s.keys[i] = i && one ? s.keys[0] : (unsigned*)take(tokens * 4);
    s.ats[i] = i && one ? s.ats[0] : (unsigned*)take(tokens * 4);
  }
  s.counts = tokens <= MERGED ? nullptr : (int*)take((clr::ceil_div(tokens, SORT * items_of(tokens)) + 1) * MOST_DIGITS * 4);
  s.partial = (float*)take(clr::ceil_div(tokens, piece_of(tokens, blocks, lanes)) * 2 * width * sizeof(float));
  return s;
}

}  // namespace

void embedding_launch(const EmbedArgs& a, hipStream_t st) {
  const int packs = packs_of(a.width, a.dtype);
  const long items = a.tokens * packs;
  with_packs(a.dtype, a.width, [&](auto t, auto v) {
    clr::in_launches(clr::ceil_div(items, BLOCK * TURNS), BLOCK,
                     [&](long base, unsigned n) {
                       using T = decltype(t);
                       constexpr int V = decltype(v)::value;
                       if (streams(a.tokens, a.width, a.dtype)) embed_kernel<T, V, true><<<n, BLOCK, 0, st>>>(a, packs, items, base);
                       else embed_kernel<T, V, false><<<n, BLOCK, 0, st>>>(a, packs, items, base);
                     });
  });
}

size_t embedding_grad_workspace(long tokens, int width, int vocab, int dtype) { return tokens <= FEW ? 0 : space_of(nullptr, tokens, width, vocab, dtype).bytes; }

static void few_launch(const EmbedArgs& e, hipStream_t st) {
  FewArgs a{e};
  a.packs = packs_of(e.width, e.dtype);
  a.blocks = (int)clr::ceil_div(a.packs, BLOCK);
  a.chunk = std::max(1, std::min(MOST_CHUNK, 4096 / a.packs));   // 64 KiB of packs
  const long groups = e.tokens * a.blocks + clr::ceil_div(e.vocab, a.chunk);
  with_packs(e.dtype, e.width, [&](auto t, auto v) {
    clr::in_launches(groups, BLOCK, [&](long base, unsigned n) { few_kernel<decltype(t), decltype(v)::value><<<n, BLOCK, 0, st>>>(a, base); });
  });
}

void embedding_grad_launch(const EmbedArgs& a, hipStream_t st) {
  if (a.tokens <= FEW) return few_launch(a, st);
  const Space space = space_of((char*)a.workspace, a.tokens, a.width, a.vocab, a.dtype);
  SortArgs s{};
  s.ids = a.ids;
  s.ignore = a.ignore;
  s.n = (int)a.tokens;
  s.vocab = a.vocab;
  int bits = 1;
  while (a.vocab >> bits) bits++;
  s.passes = (int)clr::ceil_div(bits, MOST_BITS);
  s.bits = (int)clr::ceil_div(bits, s.passes);
  const bool one = a.tokens <= ONE, merged = !one && a.tokens <= MERGED;
  const int items = items_of(a.tokens);
  s.tiles = one ? 1 : (int)clr::ceil_div(a.tokens, merged ? SORT : SORT * items);
  // the table's places, shared out by how long the launches take: a scatter twice as long as a count, 6 to 4 of tiles and their merging
  Clear c{};
  c.table = (char*)a.dtable;
  c.row = (long)a.width * dtype_size(a.dtype);
  c.packs = (int)(c.row >= 16 ? clr::ceil_div(c.row, 16) : c.row / 2);
  c.stream = streams(a.vocab, a.width, a.dtype);
  const long places = (long)a.vocab * c.packs;
  auto clearing = [&](int part, int parts, int of) {
    c.first = places * part / of;
    c.last = places * (part + parts) / of;
    c.groups = (int)std::min<long>(clr::ceil_div(c.last - c.first, SORT * 4), 1024);
    return c.groups;
  };
  int out = 0;
  if (one) {
    s.to = space.keys[0];
    s.to_at = space.ats[0];
    const unsigned groups = s.tiles + clearing(0, 1, 1);
    with_items((int)clr::ceil_div(a.tokens, SORT), [&](auto n) { sort_tile_kernel<decltype(n)::value><<<groups, SORT, 0, st>>>(s, c); });
  } else if (merged) {
    s.to = space.keys[0];
    s.to_at = space.ats[0];
    unsigned groups = s.tiles + clearing(0, 6, 10);
    sort_tile_kernel<1><<<groups, SORT, 0, st>>>(s, c);
    out = 1;
    s.from = s.to;
    s.from_at = s.to_at;
    s.to = space.keys[1];
    s.to_at = space.ats[1];
    groups = (unsigned)clr::ceil_div(a.tokens, SORT / 4) + clearing(6, 4, 10);
    if (s.tiles <= 16) sort_merge_kernel<16><<<groups, SORT, 0, st>>>(s, c);
    else sort_merge_kernel<32><<<groups, SORT, 0, st>>>(s, c);
  } else {
    s.counts = space.counts;
    for (int pass = 0; pass < s.passes; pass++) {
      out = pass & 1;
      s.shift = pass * s.bits;
      s.from = space.keys[1 - out];
      s.from_at = space.ats[1 - out];
      s.to = space.keys[out];
      s.to_at = space.ats[out];
      unsigned groups = s.tiles + clearing(3 * pass, 1, 3 * s.passes);
      if (items == 2) sort_count_kernel<2><<<groups, SORT, 0, st>>>(s, c);
      else sort_count_kernel<4><<<groups, SORT, 0, st>>>(s, c);
      if (s.tiles > FEW_TILES) sort_scan_kernel<<<(unsigned)clr::ceil_div(1 << s.bits, 64), SORT, 0, st>>>(s);
      groups = s.tiles + clearing(3 * pass + 1, 2, 3 * s.passes);
      if (items == 2) sort_scatter_kernel<2><<<groups, SORT, 0, st>>>(s, c);
      else sort_scatter_kernel<4><<<groups, SORT, 0, st>>>(s, c);
    }
  }
  const int packs = packs_of(a.width, a.dtype);
  SumArgs m{};
  m.keys = space.keys[out];
  m.ats = space.ats[out];
  m.dy = a.y; m.lddy = a.ldy;
  m.dtable = a.dtable;
  m.partial = space.partial;
  m.n = (int)a.tokens; m.vocab = a.vocab; m.width = a.width; m.packs = packs;
  m.lanes = lanes_of(packs, 64);
  m.across = lanes_of(packs, JOIN);
  const int threads = std::min(std::max(4 * m.across, 256), JOIN);   // (the gradient of 53,248 x 16, rows of 4 packs: 50 us with 1,024, 37 with 256)
  m.blocks = (int)clr::ceil_div(packs, m.lanes);
  m.piece = piece_of(a.tokens, m.blocks, m.lanes);
  m.pieces = (int)clr::ceil_div(a.tokens, m.piece);
  m.group = m.pieces > MANY_PIECES ? 32 : m.pieces;
  m.scale = a.scale;
  with_packs(a.dtype, a.width, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const long teams = (long)m.pieces * m.blocks;
    clr::in_launches(clr::ceil_div(teams * m.lanes, BLOCK), BLOCK, [&](long base, unsigned n) {
      if (m.lanes == 64) run_sum_kernel<T, V, true><<<n, BLOCK, 0, st>>>(m, base);
      else run_sum_kernel<T, V, false><<<n, BLOCK, 0, st>>>(m, base);
    });
    if (m.group < m.pieces)
      clr::in_launches(clr::ceil_div(m.pieces, m.group), threads,
                       [&](long base, unsigned n) { run_group_kernel<V><<<n, threads, threads * V * sizeof(float), st>>>(m, base); });
    if (m.pieces > 1)
      clr::in_launches(m.pieces, threads, [&](long base, unsigned n) { run_join_kernel<T, V><<<n, threads, threads * V * sizeof(float), st>>>(m, base); });
  });
}
