// The embedding of a vocabulary that may be sharded over ranks: lookup with
// scaling, and its gradient by sorted tokens.
//
//   lookup:   out[i]  = scale * table[id_i - first]            (0: not here)
//   gradient: d[r]    = scale * sum of grad[i] over id_i - first == r
//   sum_rows: the rows r that occur, ascending, each with that sum
//
// All of it moves data; nothing is computed that a memory pass does not hide.
// Lookup of 16385 tokens of 4096 bf16, a quarter of them here: 23 us, 6.5 TB/s.
// Gradient of 16384 tokens into 131072 x 4096 bf16: 236 us, 5.1 TB/s, of which
// 192 are the zeros of rows that no token names (with the sort in their shadow),
// 33 the sums and 5 their joining. 32768 rows of 1024 fp32 into one set: 84 us,
// of which 33 are the sort, 32 the sums (at the rate of a copy) and 10 counting
// and joining: few launches' worth of work, bound by their latency.
// The gradient orders the tokens first, by a stable radix sort of (row, place)
// pairs, so that every row of the result has one owner that adds its tokens'
// gradients in the order of their places: no atomics on values, and the same
// bits from every run.
#include <hip/hip_runtime.h>
#include "../common/tensor_ops.hpp"
#include "ops_device.hpp"

namespace accl {
namespace ops {

// ------------------------------------------------------------- row of a token
template <class I>
__device__ inline u32 shard_row(I id, i64 first, u64 rows) {
  u64 r = u64(i64(id)) - u64(first);  // wraps far above rows if id < first
  return i64(id) >= first && r < rows ? u32(r) : u32(rows);
}

// ------------------------------------------------------------------- columns
// Eight columns of a lane. The last of a width that is no multiple of eight are
// read as the last eight, of which the first `skip` are the lane's before, and
// lanes behind the width read those as well and own none: loads of all lanes are
// whole and can be ahead of their use. (With loads of single elements, 1228 rows
// of 286 fp32 took 20.9 us instead of 19.3, their gradient of 16000 x 128 37.6
// instead of 32.9.)
struct Columns {
  u64 at;
  int n, skip;  // columns skip .. n - 1 are this lane's
  __device__ Columns(u64 c, u64 width) {
    n = int(width < VEC ? width : VEC);
    at = c + VEC <= width ? c : width - n;
    skip = c < width ? int(c - at) : n;
  }
};

template <class T>
__device__ inline void store_own(T* p, const Columns& cols, const Eight<T>& v) {
  if (cols.n == VEC && cols.skip == 0) {
    store8(p, VEC, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= cols.skip && i < cols.n) p[i] = v.e[i];
  }
}

// --------------------------------------------------------------------- lookup
// One wave takes SPAN elements of four tokens' rows, whose loads go out
// together.
constexpr u32 AT_ONCE = 4;

template <class T, class I>
__global__ void __launch_bounds__(256) lookup_kernel(
    const I* ids, u64 tokens, i64 first, u64 rows, u64 width, float scale,
    const T* table, i64 table_stride, T* out, i64 out_stride, int past_caches) {
  const u32 lane = threadIdx.x & 63;
  const Columns cols(u64(blockIdx.x) * SPAN + lane * VEC, width);
  for (u64 i = (u64(blockIdx.y) * 4 + (threadIdx.x >> 6)) * AT_ONCE; i < tokens;
       i += u64(gridDim.y) * 4 * AT_ONCE) {
    u32 r[AT_ONCE];
#pragma unroll
    for (u32 a = 0; a < AT_ONCE; ++a)
      r[a] = __builtin_amdgcn_readfirstlane(
          i + a < tokens ? shard_row(ids[i + a], first, rows) : u32(rows));
    Eight<T> v[AT_ONCE];
#pragma unroll
    for (u32 a = 0; a < AT_ONCE; ++a)
      load8(table + i64(r[a]) * table_stride + i64(cols.at),
            r[a] < rows ? cols.n : 0, v[a]);
#pragma unroll
    for (u32 a = 0; a < AT_ONCE; ++a) {
      if (i + a >= tokens) break;
      // tokens without a row: zeros, whatever the scale
      const float by = r[a] < rows ? scale : 0.0f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[a].e[j] = T(float(v[a].e[j]) * by);
      T* to = out + i64(i + a) * out_stride + i64(cols.at);
      if (past_caches && cols.skip == 0) stream8(to, cols.n, v[a]);
      else store_own(to, cols, v[a]);
    }
  }
}

void gpu_lookup(const EmbeddingArgs& a, void* stream) {
  if (!a.tokens || !a.width) return;
  if (a.rows >= (1ull << 31)) throw accl_error("embedding: too many rows");
  dim3 grid(blocks_of(a.width, SPAN),
            u32(a.tokens / (4 * AT_ONCE) < 65535
                    ? blocks_of(a.tokens, 4 * AT_ONCE) : 65535));
  // A result that no cache of the chip's parts holds goes past them (16385
  // tokens of 4096 bf16: 36 us into the caches, 23 past them), unless its rows
  // end inside 16 bytes (16001 of 1003: 11.9 and 12.2).
  const u64 row_bytes = a.width * dtype_size(a.dst_dtype);
  const int past_caches =
      a.tokens * row_bytes > (32u << 20) && row_bytes % 16 == 0;
  with_type(a.src_dtype, "embedding", [&](auto t) {
    using T = decltype(t);
    if (a.ids_dtype == DataType::int64)
      hipLaunchKernelGGL((lookup_kernel<T, i64>), grid, dim3(256), 0,
                         (hipStream_t)stream, (const i64*)a.ids, a.tokens,
                         a.first_row, a.rows, a.width, a.scale,
                         (const T*)a.src, a.src_stride, (T*)a.dst,
                         a.dst_stride, past_caches);
    else
      hipLaunchKernelGGL((lookup_kernel<T, i32>), grid, dim3(256), 0,
                         (hipStream_t)stream, (const i32*)a.ids, a.tokens,
                         a.first_row, a.rows, a.width, a.scale,
                         (const T*)a.src, a.src_stride, (T*)a.dst,
                         a.dst_stride, past_caches);
  });
  launched("embedding");
}

// ----------------------------------------------------------------------- fill
// Zeros for a gradient, of which no token may name most rows. They are far more
// than the sort reads, so each launch of the sort takes a share of them along,
// in workgroups behind its own. The stores do not stay in the caches: those
// keep the tokens' gradients, which are read next (16384 tokens into
// 131072 x 4096 bf16: 253 us with ordinary stores, 236 with these). A wave
// writes 8 KiB in a row: 271 us with 1, 241 with 4, 260 with 16.
constexpr u32 FILL_RUN = 8192;
struct Fill {
  char* out;
  u64 bytes;
  u32 share, shares, groups;  // groups: workgroups of a launch
};

template <bool PAST_CACHES>
__device__ inline void fill_run(char* at) {
  at += (threadIdx.x & 63) * 16;
#pragma unroll
  for (u32 k = 0; k < FILL_RUN; k += 1024)
    if (PAST_CACHES)
      __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, (u32x4_any*)(at + k));
    else
      *(u32x4_any*)(at + k) = u32x4{0, 0, 0, 0};
}

__device__ inline void fill_share(const Fill& f, u32 group, u32 threads) {
  const u64 lines = f.bytes / FILL_RUN;
  const u64 from = lines * f.share / f.shares;
  const u64 to = lines * (f.share + 1) / f.shares;
  const u32 waves = threads / 64;
  for (u64 i = from + u64(group) * waves + (threadIdx.x >> 6); i < to;
       i += u64(f.groups) * waves)
    fill_run<true>(f.out + i * FILL_RUN);
  // what is left, in pairs of bytes
  if (f.share + 1 == f.shares && group == 0)
    for (u64 c = lines * FILL_RUN + threadIdx.x * 2; c < f.bytes; c += threads * 2)
      *(u16*)(f.out + c) = 0;
}

static u32 fill_groups(u64 bytes, u32 shares) {
  const u64 n = bytes / shares / (4 * FILL_RUN) + 1;
  return u32(n < 2048 ? n : 2048);
}

// ----------------------------------------------------------------------- sort
// Stable least-significant-digit radix sort of (row, place). Digits have at
// most 9 bits, so that a vocabulary of fewer than 2^18 rows takes two passes
// (tokens without a row have the number behind the last as theirs). Up to 4096
// tokens are sorted by one workgroup in LDS, in one launch (a gradient of 2048
// tokens took 25 us in tiles and 19 so, of 4096 28 and 27, of 8192, if allowed,
// 36 and 43). More of them are cut in tiles: for each pass a histogram of each
// tile, then a scatter in which a workgroup finds its place for every digit from
// the histograms of all tiles. (Counting the next digit with atomics inside the
// scatter saved a launch and cost more: 18 us against 5 + 8 at 32768 tokens, for
// tokens that are frequent.)
constexpr int DIGIT_BITS = 9, DIGITS = 1 << DIGIT_BITS;
constexpr int ALONE_THREADS = 512, ALONE_ROUNDS = 8;
constexpr int ALONE = ALONE_THREADS * ALONE_ROUNDS;  // tokens of one workgroup
constexpr int SORT_THREADS = 256;
constexpr int SORT_WAVES = SORT_THREADS / 64;
constexpr int ROUNDS = 4;                     // tokens of a lane at once
constexpr int PIECE = SORT_THREADS * ROUNDS;  // tokens of a workgroup at once
constexpr u32 SORT_BLOCKS = 256;

struct SortPlan {
  u32 n, tile, blocks, passes, bits;
};

static SortPlan sort_plan(u64 tokens, u64 rows) {
  SortPlan p{};
  p.n = u32(tokens);
  u32 pieces = blocks_of(tokens, PIECE);
  u32 per = (pieces + SORT_BLOCKS - 1) / SORT_BLOCKS;
  p.tile = tokens <= ALONE ? ALONE : per * PIECE;
  p.blocks = blocks_of(tokens, p.tile);
  u32 need = 1;
  while (rows >> need) ++need;  // rows itself marks a token without a row
  p.passes = (need + DIGIT_BITS - 1) / DIGIT_BITS;
  p.bits = (need + p.passes - 1) / p.passes;
  return p;
}

// Where a pass reads its tokens: the ids themselves first, sorted pairs later.
template <class I>
struct FromIds {
  const I* ids;
  i64 first;
  u64 rows;
  __device__ u32 key(u32 i) const { return shard_row(ids[i], first, rows); }
  __device__ u32 place(u32 i) const { return i; }
};
struct FromPairs {
  const u32* keys;
  const u32* places;
  __device__ u32 key(u32 i) const { return keys[i]; }
  __device__ u32 place(u32 i) const { return places[i]; }
};

template <int WAVES>
struct SortShared {
  u32 count[WAVES][DIGITS];
  u32 base[DIGITS];
  u32 per_wave[WAVES];
};

// exclusive sum over the block's threads
__device__ inline u32 scan_exclusive(u32 v, u32* per_wave) {
  const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u32 s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    u32 o = __shfl_up(s, d);
    if (lane >= u32(d)) s += o;
  }
  if (lane == 63) per_wave[wave] = s;
  __syncthreads();
  u32 before = 0;
  for (u32 w = 0; w < wave; ++w) before += per_wave[w];
  __syncthreads();
  return before + s - v;
}

template <int WAVES>
__device__ inline void clear_counts(SortShared<WAVES>& sh) {
  for (u32 d = threadIdx.x; d < WAVES * DIGITS; d += WAVES * 64)
    (&sh.count[0][0])[d] = 0;
  __syncthreads();
}

// Rank of a lane's token among its wave's tokens of the same digit so far: those
// of earlier rounds, and the lanes before it. Lanes with the same digit find each
// other bit by bit, and the first of them counts them all. LDS takes a wave's
// operations in their order, so that no round waits for the one before.
// Unrolled, 32768 rows of 1024 fp32 take 84.7 us instead of 85.9; but where one
// workgroup sorts, which has eight copies of it, 4000 tokens take 24.2 instead of
// 23.4.
typedef volatile u32 __attribute__((address_space(3))) lds_u32;
struct Rank {
  u32 earlier, before;
  __device__ operator u32() const { return earlier + before; }
};
template <bool UNROLL>
__device__ inline Rank rank_in_wave(lds_u32* count, u32 digit, u32 bits,
                                    bool here) {
  u64 same = __builtin_amdgcn_ballot_w64(here);
  auto among = [&](u32 b) {
    const bool set = (digit >> b) & 1;
    const u64 m = __builtin_amdgcn_ballot_w64(set);
    same &= set ? m : ~m;
  };
  if constexpr (UNROLL) {
#pragma unroll
    for (u32 b = 0; b < DIGIT_BITS; ++b) among(b);
  } else {
#pragma unroll 1
    for (u32 b = 0; b < bits; ++b) among(b);
  }
  Rank rank;
  rank.before = __builtin_amdgcn_mbcnt_hi(
      u32(same >> 32), __builtin_amdgcn_mbcnt_lo(u32(same), 0));
  rank.earlier = here ? count[digit] : 0;
  if (here && rank.before == 0)
    __hip_atomic_fetch_add((u32 __attribute__((address_space(3)))*)&count[digit],
                           u32(__popcll(same)), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_WAVEFRONT);
  return rank;
}

// Turns each wave's counts into where its tokens of a digit begin, from the
// block's places in base, which move on behind this piece. A thread owns the
// same neighbouring digits everywhere.
template <int WAVES>
__device__ inline void place_waves(SortShared<WAVES>& sh) {
  constexpr int OWN = DIGITS / (WAVES * 64);
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const u32 d = threadIdx.x * OWN + i;
    u32 at = sh.base[d];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const u32 c = sh.count[w][d];
      sh.count[w][d] = at;
      at += c;
    }
    sh.base[d] = at;
  }
  __syncthreads();
}

// For sum_rows (ids_out) it counts heads of runs too, as count_kernel does: 1228
// tokens of 286 fp32 23.6 us with that kernel, 20.9 so.
template <class I>
__global__ void __launch_bounds__(ALONE_THREADS) sort_alone_kernel(
    FromIds<I> src, u32 n, u32 passes, u32 bits, u32* keys, u32* places,
    u32* before, u32* tiles, I* ids_out, Fill fill) {
  if (blockIdx.x > 0) return fill_share(fill, blockIdx.x - 1, ALONE_THREADS);
  __shared__ SortShared<ALONE_THREADS / 64> sh;
  __shared__ __align__(16) u32 moved[2][ALONE];
  const u32 t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const u32 mask = (1u << bits) - 1;
  const u32 rounds = (n + ALONE_THREADS - 1) / ALONE_THREADS;
  const u32 mine = wave * rounds * 64 + lane;
  for (u32 pass = 0; pass < passes; ++pass) {
    const u32 shift = pass * bits;
    u32 key[ALONE_ROUNDS], place[ALONE_ROUNDS];
    Rank rank[ALONE_ROUNDS];
#pragma unroll
    for (int r = 0; r < ALONE_ROUNDS; ++r) {
      const u32 i = mine + r * 64;
      key[r] = place[r] = 0;
      if (u32(r) < rounds && i < n) {
        key[r] = pass ? moved[0][i] : src.key(i);
        place[r] = pass ? moved[1][i] : src.place(i);
      }
    }
    clear_counts(sh);
#pragma unroll
    for (int r = 0; r < ALONE_ROUNDS; ++r)
      if (u32(r) < rounds)
        rank[r] = rank_in_wave<false>((lds_u32*)sh.count[wave],
                                      (key[r] >> shift) & mask, bits,
                                      mine + r * 64 < n);
    __syncthreads();
    u32 total = 0;
#pragma unroll
    for (int w = 0; w < ALONE_THREADS / 64; ++w) total += sh.count[w][t];
    sh.base[t] = scan_exclusive(total, sh.per_wave);
    place_waves(sh);
#pragma unroll
    for (int r = 0; r < ALONE_ROUNDS; ++r) {
      if (u32(r) >= rounds || mine + r * 64 >= n) continue;
      const u32 to = sh.count[wave][(key[r] >> shift) & mask] + rank[r];
      moved[0][to] = key[r];
      moved[1][to] = place[r];
    }
    __syncthreads();
  }
  for (u32 i = t; i < n; i += ALONE_THREADS) {
    keys[i] = moved[0][i];
    places[i] = moved[1][i];
  }
  if (!ids_out) return;
  const u32 from = t * 8, rows = u32(src.rows);
  u32 left = t ? moved[0][from - 1] : rows, heads = 0;
#pragma unroll
  for (u32 i = 0; i < 8; ++i) {
    const u32 key = moved[0][from + i];
    heads += from + i < n && key < rows && key != left;
    left = key;
  }
  const u32 at = scan_exclusive(heads, sh.per_wave);
  if (from < n) before[t] = at;
  if (t + 1 == ALONE_THREADS) tiles[0] = at + heads;
  for (u32 i = t; i < n; i += ALONE_THREADS) ids_out[i] = I(-1);
}

// Counts of a digit in every tile.
template <class S>
__global__ void __launch_bounds__(SORT_THREADS) histogram_kernel(
    S src, u32 n, u32 tile, u32 blocks, u32 shift, u32 mask, u32* hist,
    Fill fill) {
  if (blockIdx.x >= blocks)
    return fill_share(fill, blockIdx.x - blocks, SORT_THREADS);
  __shared__ u32 count[DIGITS];
  for (u32 d = threadIdx.x; d < DIGITS; d += SORT_THREADS) count[d] = 0;
  __syncthreads();
  const u32 from = blockIdx.x * tile;
  const u32 to = n - from < tile ? n : from + tile;
  for (u32 i = from + threadIdx.x; i < to; i += SORT_THREADS)
    atomicAdd(&count[(src.key(i) >> shift) & mask], 1u);
  __syncthreads();
  for (u32 d = threadIdx.x; d < DIGITS; d += SORT_THREADS)
    hist[blockIdx.x * DIGITS + d] = count[d];
}

template <class S>
__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(
    S src, u32 n, u32 tile, u32 blocks, u32 shift, u32 bits, const u32* hist,
    u32* keys, u32* places, Fill fill) {
  if (blockIdx.x >= blocks)
    return fill_share(fill, blockIdx.x - blocks, SORT_THREADS);
  __shared__ SortShared<SORT_WAVES> sh;
  const u32 t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const u32 mask = (1u << bits) - 1;

  const u32 from = blockIdx.x * tile;
  const u32 to = n - from < tile ? n : from + tile;
  u32 key[ROUNDS], place[ROUNDS];
  Rank rank[ROUNDS];
  auto load = [&](u32 mine) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const u32 i = mine + r * 64;
      key[r] = i < to ? src.key(i) : 0;
      place[r] = i < to ? src.place(i) : 0;
    }
  };
  u32 mine = from + wave * (PIECE / SORT_WAVES) + lane;
  load(mine);

  // all tokens of this thread's digits, and those of earlier tiles
  u32x2 total = {0, 0}, before = {0, 0};
#pragma unroll 16
  for (u32 b = 0; b < blocks; ++b) {
    const u32x2 h = *(const u32x2*)&hist[b * DIGITS + t * 2];
    total += h;
    if (b < blockIdx.x) before += h;
  }
  const u32 at = scan_exclusive(total.x + total.y, sh.per_wave);
  sh.base[t * 2] = at + before.x;
  sh.base[t * 2 + 1] = at + total.x + before.y;

  for (u32 piece = from; piece < to; piece += PIECE) {
    clear_counts(sh);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
      rank[r] = rank_in_wave<true>((lds_u32*)sh.count[wave],
                                   (key[r] >> shift) & mask, bits,
                                   mine + r * 64 < to);
    __syncthreads();
    place_waves(sh);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if (mine + r * 64 >= to) continue;
      const u32 p = sh.count[wave][(key[r] >> shift) & mask] + rank[r];
      keys[p] = key[r];
      places[p] = place[r];
    }
    __syncthreads();
    mine += PIECE;
    load(mine);
  }
}

// ----------------------------------------------------------------------- sums
// The sorted tokens are cut in chunks. One wave adds a chunk's gradients over
// SPAN columns; a run of one row that lies inside the chunk goes to its row at
// once. Runs that cross chunks leave their part of each chunk in the workspace,
// and a second kernel adds those in their order: however often one token
// occurs, no wave adds more than a chunk's rows.
constexpr u32 LONG_CHUNK = 32, SHORT_CHUNK = 8;
constexpr u32 COUNT_PIECE = 1024;  // tokens whose heads a workgroup counts at once
constexpr u32 COUNT_BLOCKS = 1024;

static u32 chunk_of(u64 tokens, u64 width) {
  const u64 waves = u64(blocks_of(tokens, LONG_CHUNK)) * blocks_of(width, SPAN);
  return waves < 2048 ? SHORT_CHUNK : LONG_CHUNK;
}
static u32 count_tile(u64 tokens) {
  const u32 pieces = blocks_of(tokens, COUNT_PIECE);
  return (pieces + COUNT_BLOCKS - 1) / COUNT_BLOCKS * COUNT_PIECE;
}

// A grid's second dimension ends at 65535.
static dim3 long_grid(u32 columns, u32 n) {
  return dim3(columns, n < 65535 ? n : 65535, (n + 65534) / 65535);
}
__device__ inline u32 long_index() { return blockIdx.z * 65535 + blockIdx.y; }

struct Runs {
  const u32 *keys, *places;
  u32 n, rows;
  float *heads, *tails;  // [chunks][width]: a run from before, a run to behind
  // sum_rows: runs that begin in a tile, and before each eight tokens in it
  const u32 *tiles, *before;
  u32 tile;
  u32 chunk;
};

// Heads of runs (first tokens of a row) are counted to give every row its
// place in the result of sum_rows, whose places without a row hold -1.
template <class I>
__global__ void __launch_bounds__(256) count_kernel(
    const u32* keys, u32 n, u32 rows, u32 tile, u32* before, u32* tiles,
    I* ids_out) {
  __shared__ u32 per_wave[4];
  const u32 from = blockIdx.x * tile, to = n - from < tile ? n : from + tile;
  const u32 lane = threadIdx.x & 63;
  u32 so_far = 0;
  for (u32 piece = from; piece < to; piece += COUNT_PIECE) {
    // a wave takes 256 neighbours; eight lanes hold 32 counts of eight tokens
    u32 mine = 0;
    const u32 first = piece + (threadIdx.x >> 6) * 256;
#pragma unroll
    for (u32 k = 0; k < 4; ++k) {
      const u32 i = first + k * 64 + lane;
      const u32 key = i < n ? keys[i] : rows;
      const bool head = key < rows && (i == 0 || keys[i - 1] != key);
      if (i < n) ids_out[i] = I(-1);
      const u64 m = __builtin_amdgcn_ballot_w64(head);
      if (lane / 8 == k) mine = __popc(u32(m >> (lane % 8 * 8)) & 0xFF);
    }
    const u32 at = so_far + scan_exclusive(mine, per_wave);
    if (lane < 32 && first + lane * 8 < n) before[first / 8 + lane] = at;
    __shared__ u32 last;
    if (threadIdx.x == 255) last = at + mine;
    __syncthreads();
    so_far = last;
    __syncthreads();
  }
  if (threadIdx.x == 0) tiles[blockIdx.x] = so_far;
}

// runs that begin in the first n tiles; for all lanes of a wave
__device__ inline u32 runs_of_tiles(const u32* tiles, u32 n) {
  u32 v = 0;
  for (u32 i = threadIdx.x & 63; i < n; i += 64) v += tiles[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return __builtin_amdgcn_readfirstlane(v);
}

template <class O>
__device__ inline void put_sum(O* to, const Columns& cols, const float sum[VEC],
                               float scale, int accumulate) {
  Eight<O> v;
  if (accumulate) load8(to, cols.n, v);
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    v.e[e] = O((accumulate ? float(v.e[e]) : 0.0f) + sum[e] * scale);
  store_own(to, cols, v);
}

__device__ inline void put_part(float* to, const Columns& cols,
                                const float sum[VEC]) {
  Eight<float> v;
#pragma unroll
  for (int e = 0; e < VEC; ++e) v.e[e] = sum[e];
  store_own(to, cols, v);
}

// A chunk's tokens, one a lane: `ends` has the lanes whose run does not go on
// in the next lane, `heads` those whose run begins there.
struct Chunk {
  u32 key, place, tokens;
  u64 heads, ends;
  bool from_before, to_behind;
  __device__ Chunk(const Runs& runs, u32 c) {
    const u32 lane = threadIdx.x & 63, i = c * runs.chunk + lane;
    const bool in = lane < runs.chunk && i < runs.n;
    key = in ? runs.keys[i] : runs.rows;
    place = in ? runs.places[i] : 0;
    const u32 left = in && i > 0 ? runs.keys[i - 1] : runs.rows;
    const u32 right = in && i + 1 < runs.n ? runs.keys[i + 1] : runs.rows;
    const bool has = key < runs.rows;
    tokens = u32(__popcll(__builtin_amdgcn_ballot_w64(has)));
    heads = __builtin_amdgcn_ballot_w64(has && left != key);
    ends = __builtin_amdgcn_ballot_w64(has && right != key);
    from_before = tokens && !(heads & 1);
    to_behind = tokens && !((ends >> (tokens - 1)) & 1);
  }
};

// place of the first run that begins in chunk c among all runs
__device__ inline u32 runs_before(const Runs& runs, u32 c) {
  const u32 i = c * runs.chunk;
  return runs.before[i / 8] + runs_of_tiles(runs.tiles, i / runs.tile);
}

template <class T, class O, class I>
__global__ void __launch_bounds__(256) sum_kernel(
    Runs runs, u32 chunks, u64 width, float scale, const T* grad,
    i64 grad_stride, O* out, i64 out_stride, int accumulate, I* ids_out,
    i64* count_out) {
  const u32 lane = threadIdx.x & 63;
  const Columns cols(u64(blockIdx.x) * SPAN + lane * VEC, width);
  const u32 unit =
      long_index() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= chunks) return;
  if (count_out && unit == 0 && blockIdx.x == 0) {
    const u32 count =
        runs_of_tiles(runs.tiles, (runs.n + runs.tile - 1) / runs.tile);
    if (lane == 0) *count_out = count;
  }
  const Chunk chunk(runs, unit);
  u32 run = ids_out ? runs_before(runs, unit) : 0;
  if (ids_out && blockIdx.x == 0 && (chunk.heads >> lane & 1))
    ids_out[run + u32(__popcll(chunk.heads & ((1ull << lane) - 1)))] =
        I(chunk.key);
  // the run that comes from before has its place already
  if (chunk.from_before) --run;
  float sum[VEC] = {};
  constexpr u32 AHEAD = 4;
  Eight<T> v[2][AHEAD];
  auto load = [&](u32 j, Eight<T>(&to)[AHEAD]) {
#pragma unroll
    for (u32 a = 0; a < AHEAD; ++a) {
      const u32 k = j + a < chunk.tokens ? j + a : chunk.tokens - 1;
      load8(grad + i64(u32(__builtin_amdgcn_readlane(int(chunk.place), int(k)))) *
                       grad_stride + i64(cols.at), cols.n, to[a]);
    }
  };
  auto add = [&](u32 j, const Eight<T>(&from)[AHEAD]) {
#pragma unroll
    for (u32 a = 0; a < AHEAD; ++a) {
      const u32 k = j + a;
      if (k >= chunk.tokens) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += float(from[a].e[e]);
      const bool last = k + 1 == chunk.tokens;
      if (!last && !(chunk.ends >> k & 1)) continue;
      // a whole run, or this chunk's part of one
      const bool first = (chunk.heads & ((2ull << k) - 1)) == 0;
      if (first) {  // begins before this chunk
        put_part(runs.heads + u64(unit) * width + cols.at, cols, sum);
      } else if (last && chunk.to_behind) {
        put_part(runs.tails + u64(unit) * width + cols.at, cols, sum);
      } else {
        const u32 row = ids_out
                            ? run
                            : u32(__builtin_amdgcn_readlane(int(chunk.key), int(k)));
        put_sum(out + i64(row) * out_stride + i64(cols.at), cols, sum, scale,
                accumulate);
      }
      ++run;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
    }
  };
  if (!chunk.tokens) return;
  load(0, v[0]);
  for (u32 j = 0; j < chunk.tokens; j += 2 * AHEAD) {
    load(j + AHEAD, v[1]);
    add(j, v[0]);
    load(j + 2 * AHEAD, v[0]);
    add(j + AHEAD, v[1]);
  }
}

// Joins the parts of the run that begins in a chunk and goes on behind it: its
// waves add a quarter of them each.
template <class O, class I>
__global__ void __launch_bounds__(256) join_kernel(
    Runs runs, u32 chunks, u64 width, float scale, O* out, i64 out_stride,
    int accumulate, I* ids_out) {
  const u32 c = long_index();
  if (c + 1 >= chunks) return;
  const Chunk chunk(runs, c);
  if (!chunk.to_behind || !chunk.heads) return;
  const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u32 key =
      u32(__builtin_amdgcn_readlane(int(chunk.key), int(chunk.tokens - 1)));
  const u32 row =
      ids_out ? runs_before(runs, c) + u32(__popcll(chunk.heads)) - 1 : key;
  // the last chunk with a part is the first whose last token has another row,
  // or the one before if that chunk begins with another row
  u32 end = c + 1;
  for (;; end += 64) {
    const u32 d = end + lane;
    const u32 first = d * runs.chunk;  // the run goes on into chunk d
    const bool on = d < chunks && runs.keys[first] == key;
    const u64 m = __builtin_amdgcn_ballot_w64(on);
    if (~m) {
      end += u32(__builtin_ctzll(~m));
      break;
    }
  }
  const u32 parts = end - (c + 1), per = (parts + 3) / 4;
  const Columns cols(u64(blockIdx.x) * SPAN + lane * VEC, width);
  float sum[VEC] = {};
  Eight<float> v;
  if (wave == 0) {
    load8(runs.tails + u64(c) * width + cols.at, cols.n, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = v.e[e];
  }
  const u32 from = c + 1 + wave * per;
  const u32 to = from + per < end ? from + per : end;
#pragma unroll 4
  for (u32 d = from; d < to; ++d) {
    load8(runs.heads + u64(d) * width + cols.at, cols.n, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += v.e[e];
  }
  __shared__ float shared[3][VEC][64];
  if (wave) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) shared[wave - 1][e][lane] = sum[e];
  }
  __syncthreads();
  if (wave || cols.skip == cols.n) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += shared[w][e][lane];
  put_sum(out + i64(row) * out_stride + i64(cols.at), cols, sum, scale,
          accumulate);
}

// ----------------------------------------------------------------- few tokens
// Up to FEW tokens need no sort. A workgroup takes a token over SPAN columns,
// sees whether its row occurs before, and if not adds all tokens of that row:
// each wave those among its 64, in the order of their places, then the waves'
// sums in theirs. For sum_rows it also counts the rows below its own, and clears
// the row of the result with its token's number if that has none.
// One launch instead of four: 64 tokens into 4096 x 512 bf16 14.9 -> 7.3 us
// (10.8 with the zeros of other rows in a launch of their own), into their rows
// 19.2 -> 8.8; 256 of one row of 4096 fp32 14.8 -> 9.2, into 10000 x 4096 bf16
// 22.8 -> 13.7. With 512 tokens a gradient of one row gained 2 us and rows of
// 4096 nothing.
constexpr u32 FEW = 256;

// Zeros in the rows that no token names, by workgroups behind those of the
// tokens: `per` rows at once. Nothing else needs the caches here, so the stores
// go into them (200 tokens into 32768 x 2048 bf16: 19.2 us, 26.3 past them; 31
// into 131072 x 4096: 184 and 195). Runs begin at whole lines (107 into
// 77926 x 1283 fp32: 76 us, from any 16 bytes on 86).
constexpr u32 FEW_ROWS = 1024;

template <class O>
__device__ inline void fill_others(u32 key, u64 rows, u64 width, O* out, u32 per,
                                   u32 group, u32 groups) {
  __shared__ u32 named[FEW_ROWS];
  const u32 t = threadIdx.x, lane = t & 63;
  const u32 wave = __builtin_amdgcn_readfirstlane(t >> 6);
  for (u64 from = u64(group) * per; from < rows; from += u64(groups) * per) {
    const u32 n = u32(rows - from < per ? rows - from : per);
    const u32 mine = key - u32(from);  // far above n for other rows
    if (!__syncthreads_or(mine < n)) {
      char* at = (char*)(out + from * width);
      char* end = (char*)(out + (from + n) * width);
      const u32 odd = u32(-u64(at)) % 256;  // in front of whole lines
      if (u64(end - at) >= odd) {
        if (t < odd / 2) ((u16*)at)[t] = 0;
        at += odd;
        const u64 runs = u64(end - at) / FILL_RUN;
        for (u64 i = wave; i < runs; i += FEW / 64)
          fill_run<false>(at + i * FILL_RUN);
        at += runs * FILL_RUN;
      }
      for (at += t * 16; at + 16 <= end; at += FEW * 16)
        *(u32x4_any*)at = u32x4{0, 0, 0, 0};
      for (; at < end; at += 2) *(u16*)at = 0;
      continue;
    }
    for (u32 r = t; r < n; r += FEW) named[r] = 0;
    __syncthreads();
    if (mine < n) named[mine] = 1;
    __syncthreads();
    for (u32 r = 0; r < n; r += 64) {
      const bool other = r + lane < n && !named[r + lane];
      u64 others = __builtin_amdgcn_ballot_w64(other && lane % 4 == wave);
      for (; others; others &= others - 1) {
        O* row = out + (from + r + u32(__builtin_ctzll(others))) * width;
        u64 c = lane * VEC;
        for (; c + VEC <= width; c += SPAN)
          store8(row + c, VEC, Eight<O>{});
        for (; c < width; ++c) row[c] = O(0.0f);
      }
    }
  }
}

template <class T, class O, class I>
__global__ void __launch_bounds__(FEW) few_kernel(
    const I* ids, u32 n, i64 first, u64 rows, u64 width, float scale,
    const T* grad, i64 grad_stride, O* out, i64 out_stride, int accumulate,
    I* ids_out, i64* count_out, u32 per) {
  __shared__ u32 keys[FEW];
  __shared__ u64 begins[FEW / 64];  // tokens whose row does not occur before
  __shared__ float sums[FEW / 64 - 1][VEC][64];
  const u32 t = threadIdx.x, lane = t & 63;
  const u32 wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const u32 mine = blockIdx.y;
  const u32 key = t < n ? shard_row(ids[t], first, rows) : u32(rows);
  if (mine >= n)
    return fill_others(key, rows, width, out, per,
                       (mine - n) * gridDim.x + blockIdx.x,
                       (gridDim.y - n) * gridDim.x);
  keys[t] = key;
  __syncthreads();
  const u32 row = keys[mine];
  const u64 same = __builtin_amdgcn_ballot_w64(key == row);
  const bool held = row < u32(rows);
  const Columns cols(u64(blockIdx.x) * SPAN + lane * VEC, width);

  u32 place = row, count = 0;
  bool begin;
  if (ids_out) {
    // a table in which each row finds the first of its tokens; twice as many
    // slots as tokens, so that every search ends
    __shared__ u32 slots[2 * FEW], firsts[2 * FEW];
    slots[t] = slots[t + FEW] = firsts[t] = firsts[t + FEW] = ~0u;
    __syncthreads();
    u32 h = key * 2654435761u / (0x80000000u / FEW);
    if (key < u32(rows)) {
      for (;; h = (h + 1) % (2 * FEW)) {
        const u32 had = atomicCAS(&slots[h], ~0u, key);
        if (had == ~0u || had == key) break;
      }
      atomicMin(&firsts[h], t);
    }
    __syncthreads();
    const bool b = key < u32(rows) && firsts[h] == t;
    const u64 m = __builtin_amdgcn_ballot_w64(b);
    const u64 below = __builtin_amdgcn_ballot_w64(b && key < row);
    __shared__ u32 lower[FEW / 64];
    if (lane == 0) {
      begins[wave] = m;
      lower[wave] = u32(__popcll(below));
    }
    __syncthreads();
    place = 0;
    for (u32 w = 0; w < FEW / 64; ++w) {
      place += lower[w];
      count += u32(__popcll(begins[w]));
    }
    begin = begins[mine / 64] >> (mine % 64) & 1;
    if (t == 0 && blockIdx.x == 0) {
      if (mine >= count) ids_out[mine] = I(-1);
      if (begin) ids_out[place] = I(row);
      if (mine == 0) *count_out = count;
    }
    if (mine >= count && wave == 0) {
      const float none[VEC] = {};
      put_sum(out + i64(mine) * out_stride + i64(cols.at), cols, none, 0.0f, 0);
    }
  } else {
    // lanes of earlier tokens
    const u32 from = wave * 64;
    const u64 earlier =
        mine >= from + 64 ? ~0ull : mine > from ? (1ull << (mine - from)) - 1 : 0;
    if (lane == 0) begins[wave] = same & earlier;
    __syncthreads();
    begin = held;
    for (u32 w = 0; w < FEW / 64; ++w) begin = begin && !begins[w];
  }
  if (!begin) return;

  float sum[VEC] = {};
  u64 left = same;
  constexpr u32 AHEAD = 4;
  while (left) {
    Eight<T> v[AHEAD];
    u32 have = 0;
#pragma unroll
    for (u32 a = 0; a < AHEAD; ++a) {
      if (!left) break;
      const u32 i = wave * 64 + u32(__builtin_ctzll(left));
      left &= left - 1;
      load8(grad + i64(i) * grad_stride + i64(cols.at), cols.n, v[a]);
      ++have;
    }
#pragma unroll
    for (u32 a = 0; a < AHEAD; ++a) {
      if (a >= have) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += float(v[a].e[e]);
    }
  }
  if (wave) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) sums[wave - 1][e][lane] = sum[e];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (u32 w = 0; w < FEW / 64 - 1; ++w)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] += sums[w][e][lane];
  put_sum(out + i64(place) * out_stride + i64(cols.at), cols, sum, scale,
          accumulate);
}

// ------------------------------------------------------------------ workspace
struct Workspace {
  u32 *keys[2], *places[2], *hist, *before, *tiles;
  float *heads, *tails;
  u64 bytes;
  Workspace(void* p, u64 tokens, u64 rows, u64 width, bool to_rows) {
    char* at = (char*)p;
    auto take = [&](u64 n) {
      u32* q = (u32*)at;
      at += (n * 4 + 255) / 256 * 256;
      return q;
    };
    const SortPlan plan = sort_plan(tokens, rows);
    const u64 chunks = blocks_of(tokens, chunk_of(tokens, width));
    for (int i = 0; i < 2; ++i) {
      keys[i] = take(tokens);
      places[i] = take(tokens);
    }
    hist = take(plan.blocks > 1 ? u64(plan.blocks) * DIGITS : 0);
    before = take(to_rows ? blocks_of(tokens, 8) : 0);
    tiles = take(to_rows ? COUNT_BLOCKS : 0);
    heads = (float*)take(chunks * width);
    tails = (float*)take(chunks * width);
    bytes = u64(at - (char*)p);
  }
};

u64 gpu_gradient_workspace(u64 tokens, u64 rows, u64 width, bool to_rows) {
  return tokens <= FEW ? 0 : Workspace(nullptr, tokens, rows, width, to_rows).bytes;
}

__global__ void __launch_bounds__(256) zero_kernel(Fill fill) {
  fill_share(fill, blockIdx.x, 256);
}

static void zero(const EmbeddingArgs& a, hipStream_t st) {
  Fill fill{(char*)a.dst, a.rows * a.width * dtype_size(a.dst_dtype), 0, 1, 0};
  fill.groups = fill_groups(fill.bytes, 1);
  hipLaunchKernelGGL(zero_kernel, dim3(fill.groups), dim3(256), 0, st, fill);
}

template <class I>
static void gradient_of_few(const EmbeddingArgs& a, bool to_rows,
                            hipStream_t st) {
  const char* what = to_rows ? "sum_rows" : "embedding_grad";
  const u32 columns = a.width ? blocks_of(a.width, SPAN) : 1;
  u32 per = 1, fills = 0;  // of the second dimension
  if (!to_rows && !a.accumulate) {
    const u32 groups =
        fill_groups(a.rows * a.width * dtype_size(a.dst_dtype), 1);
    if (a.rows < groups) {
      zero(a, st);
    } else {
      const u64 n = (a.rows + groups - 1) / groups;
      per = u32(n < FEW_ROWS ? n : FEW_ROWS);
      fills = (groups + columns - 1) / columns;
    }
  }
  with_type(a.dst_dtype, what, [&](auto o) {
    using O = decltype(o);
    with_type(a.src_dtype, what, [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((few_kernel<T, O, I>),
                         dim3(columns, u32(a.tokens) + fills), dim3(FEW), 0, st,
                         (const I*)a.ids, u32(a.tokens), a.first_row, a.rows,
                         a.width, a.scale, (const T*)a.src, a.src_stride,
                         (O*)a.dst, a.dst_stride, int(a.accumulate),
                         to_rows ? (I*)a.ids_out : nullptr,
                         to_rows ? a.count_out : nullptr, per);
    });
  });
  launched(what);
}

template <class I>
static void gradient(const EmbeddingArgs& a, bool to_rows, hipStream_t st) {
  if (a.tokens <= FEW) return gradient_of_few<I>(a, to_rows, st);
  const char* what = to_rows ? "sum_rows" : "embedding_grad";
  Workspace w(a.workspace, a.tokens, a.rows, a.width, to_rows);
  const SortPlan p = sort_plan(a.tokens, a.rows);
  const dim3 threads(SORT_THREADS);
  Fill fill{(char*)a.dst, 0, 0, p.blocks == 1 ? 1 : 2 * p.passes, 0};
  if (!a.accumulate) {
    fill.bytes = (to_rows ? a.tokens : a.rows) * a.width * dtype_size(a.dst_dtype);
    fill.groups = fill_groups(fill.bytes, fill.shares);
  }
  const FromIds<I> ids{(const I*)a.ids, a.first_row, a.rows};
  const u32 mask = (1u << p.bits) - 1;
  int side = 0;
  I* ids_out = to_rows ? (I*)a.ids_out : nullptr;
  const u32 tile = p.blocks == 1 ? ALONE : count_tile(a.tokens);
  if (p.blocks == 1) {
    hipLaunchKernelGGL((sort_alone_kernel<I>), dim3(1 + fill.groups),
                       dim3(ALONE_THREADS), 0, st, ids, p.n, p.passes, p.bits,
                       w.keys[0], w.places[0], w.before, w.tiles, ids_out, fill);
  } else {
    const dim3 grid(p.blocks + fill.groups);
    for (u32 pass = 0; pass < p.passes; ++pass) {
      const u32 shift = pass * p.bits;
      auto go = [&](auto src) {
        using S = decltype(src);
        hipLaunchKernelGGL((histogram_kernel<S>), grid, threads, 0, st, src,
                           p.n, p.tile, p.blocks, shift, mask, w.hist, fill);
        ++fill.share;
        hipLaunchKernelGGL((scatter_kernel<S>), grid, threads, 0, st, src, p.n,
                           p.tile, p.blocks, shift, p.bits, w.hist,
                           w.keys[pass % 2], w.places[pass % 2], fill);
        ++fill.share;
      };
      if (pass == 0) go(ids);
      else go(FromPairs{w.keys[side], w.places[side]});
      side = pass % 2;
    }
  }
  const u32 chunk = chunk_of(a.tokens, a.width);
  const u32 chunks = blocks_of(a.tokens, chunk);
  const Runs runs{w.keys[side], w.places[side], p.n, u32(a.rows), w.heads,
                  w.tails, w.tiles, w.before, tile, chunk};
  if (to_rows && p.blocks > 1)
    hipLaunchKernelGGL((count_kernel<I>), dim3(blocks_of(a.tokens, tile)),
                       dim3(256), 0, st, runs.keys, p.n, u32(a.rows), tile,
                       w.before, w.tiles, ids_out);
  const u32 columns = a.width ? blocks_of(a.width, SPAN) : 1;
  with_type(a.dst_dtype, what, [&](auto o) {
    using O = decltype(o);
    with_type(a.src_dtype, what, [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((sum_kernel<T, O, I>), long_grid(columns, (chunks + 3) / 4),
                         dim3(256), 0, st, runs, chunks, a.width, a.scale,
                         (const T*)a.src, a.src_stride, (O*)a.dst, a.dst_stride,
                         int(a.accumulate), ids_out,
                         to_rows ? a.count_out : nullptr);
    });
    if (chunks > 1 && a.width)
      hipLaunchKernelGGL((join_kernel<O, I>), long_grid(columns, chunks - 1),
                         dim3(256), 0, st, runs, chunks, a.width, a.scale,
                         (O*)a.dst, a.dst_stride, int(a.accumulate), ids_out);
  });
  launched(what);
}

static void check(const EmbeddingArgs& a, const char* what, bool to_rows) {
  // places and rows are 32-bit numbers
  if (a.tokens >= (1ull << 31) || a.rows >= (1ull << 31))
    throw accl_error(std::string(what) + ": too many tokens or rows");
  if (a.workspace_bytes <
      gpu_gradient_workspace(a.tokens, a.rows, a.width, to_rows))
    throw accl_error(std::string(what) + ": workspace too small");
}

void gpu_gradient(const EmbeddingArgs& a, void* stream) {
  check(a, "embedding_grad", false);
  if (!a.accumulate && a.dst_stride != i64(a.width))
    throw accl_error("embedding_grad: a new result has no gaps");
  if (!a.rows || !a.width) return;
  if (!a.tokens) {
    if (!a.accumulate) {
      zero(a, (hipStream_t)stream);
      launched("embedding_grad");
    }
    return;
  }
  if (a.ids_dtype == DataType::int64)
    gradient<i64>(a, false, (hipStream_t)stream);
  else
    gradient<i32>(a, false, (hipStream_t)stream);
}

__global__ void no_rows_kernel(i64* count_out) { *count_out = 0; }

void gpu_sum_rows(const EmbeddingArgs& a, void* stream) {
  check(a, "sum_rows", true);
  if (!a.tokens) {
    hipLaunchKernelGGL(no_rows_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream,
                       a.count_out);
    launched("sum_rows");
    return;
  }
  if (a.ids_dtype == DataType::int64)
    gradient<i64>(a, true, (hipStream_t)stream);
  else
    gradient<i32>(a, true, (hipStream_t)stream);
}

}  // namespace ops
}  // namespace accl
