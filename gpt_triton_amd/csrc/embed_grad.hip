// Gradients of the embedding's tables: row v of the token table's is the sum of dz over the positions of token v, row l of the
// position table's the sum over the batch, both dense, rows without a token zeros.
//
// The sums are formed in fp32, each in one order, in the order of the positions and without atomics, so the same call
// gives the same bits.  That takes each token's positions one behind the other:
//   up to 256 tokens, one launch: every workgroup has a range of the vocabulary and looks all tokens through;
//   more, a stable radix sort of the tokens with their positions, by one workgroup up to 16384 tokens, else a workgroup a tile of
//   them (from 1.6 million tokens on with two launches a digit that add the tiles' counts), whose launches also write the zero
//   rows and form the position table's sums; then runs of the sorted positions are summed, whoever has a
//   token to itself writes its row, and what a token has in several runs is joined in a last launch.
// Bound by memory: dz twice (once for each table), the tables' gradients once.  us, 512 x 300 tokens, fp16, 768 wide (236 MB of dz, 77 MB of
// zero rows and sums): 143, of which the positions' sums and the runs' 55 and 52 at 4.3 and 4.6 TB/s; with one token in all places 175.
// 16 x 1024, fp32: 57; 2 x 64, one launch: 15, zero rows.
#include "common.h"
#include "launch.h"

namespace gptmi {
namespace {

constexpr int kFew = 256;          // tokens of the single launch
constexpr int kTile = 4096;        // tokens a workgroup sorts
// Tokens that one workgroup sorts alone, in registers and 131 KB of LDS, beside the zero rows.  us, kernels / calls, this and by
// tiles: 16 x 1024 tokens, 768 wide, fp32 57 / 63 and 60 / 71; 8 x 2000, 64 wide, fp16 49 / 63 and 48 / 70.
constexpr int kOneTile = 16384;
constexpr int kSortThreads = 1024;
// Tiles whose counts each workgroup that moves adds by itself, work that grows with their square; more, and two launches a digit do
// it for all.  us, calls, 64 wide, fp16, by itself / by the launches: 256 tiles 155 / 182, 512 320 / 302, 1024 778 / 570; 4096, 16 wide
// 6140 / 2150.
constexpr int kManyTiles = 400;
constexpr int kGroupTiles = 256;   // of these a workgroup
constexpr int kMaxBits = 9;        // of a digit
constexpr int kFill = 65536;       // bytes of zero rows a workgroup

// VN elements of a row: 16 bytes, or one element where a row or an address is no multiple of that.
template <typename T, int VN>
__device__ __forceinline__ void add_chunk(const T* p, float (&sum)[VN]) {
  typedef T V __attribute__((ext_vector_type(VN)));
  const V x = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int i = 0; i < VN; ++i) sum[i] += (float)x[i];
}
template <typename T>
__device__ __forceinline__ void add_chunk(const T* p, float (&sum)[1]) {
  sum[0] += (float)*p;
}
template <typename T, int VN>
__device__ __forceinline__ void put_chunk(T* p, const float (&sum)[VN]) {
  if constexpr (VN == 1) {
    *p = (T)sum[0];
  } else {
    typedef T V __attribute__((ext_vector_type(VN)));
    V x;
#pragma unroll
    for (int i = 0; i < VN; ++i) x[i] = (T)sum[i];
    *reinterpret_cast<V*>(p) = x;
  }
}
template <int VN>
__device__ __forceinline__ void clear(float (&sum)[VN]) {
#pragma unroll
  for (int i = 0; i < VN; ++i) sum[i] = 0.f;
}

struct EmbedGradArgs {
  const int64_t* ids;
  const void* dz;
  void *d_wte, *d_wpe;  // one of them may be nullptr
  int64_t tokens, L, V, P;
  int H;
  DropoutArgs drop;
  // the sort's
  int tiles, bits;          // workgroups, bits of a digit
  int lanes, across, share;  // of the position table's parts: chunks each, parts a row, groups that share a batch
  // other work of a launch: workgroups of positions, and behind them zero rows, from which 64 KB on, the token table's first
  int64_t positions, fill, table_fills;
  int64_t behind;           // elements of the position table behind the first P rows, zeros
  unsigned *keys[2], *at[2];  // tokens (V: none) and positions
  unsigned* hist;           // [tiles][1 << bits]: counts, or the counts of the tiles in front
  unsigned* group_counts;   // [groups + 1][1 << bits] where there are many tiles: of kGroupTiles tiles each, and of all
  bool many;
  // the sums'
  const unsigned *sorted, *order;
  float* parts;             // [runs][2][H]: what a run has of a token that began in front of it, and of one that goes on behind
  int run;                  // tokens of a run
};

// A mask of dropout is one for all rows, so it comes behind the sums: which of a chunk's columns are kept, and the sums over
// 1 - p, by a reciprocal with the remainder's correction (subnormal remainders aside, correctly rounded).
template <int VN>
__device__ __forceinline__ unsigned kept_columns(const EmbedGradArgs& a, int chunk) {
  unsigned kept = ~0u;
  if (a.drop.p > 0.f) {
    unsigned column[VN];
    float u[VN];
#pragma unroll
    for (int i = 0; i < VN; ++i) column[i] = (unsigned)(chunk * VN + i);
    philox_uniform<VN>(a.drop, column, u);
    kept = 0;
#pragma unroll
    for (int i = 0; i < VN; ++i) kept |= u[i] > a.drop.p ? 1u << i : 0u;
  }
  return kept;
}
template <typename T, int VN>
__device__ __forceinline__ void put_sum(const EmbedGradArgs& a, T* row, int chunk, unsigned kept, float (&sum)[VN]) {
  if (a.drop.p > 0.f) {
    const KeepScale scale(a.drop.p);
#pragma unroll
    for (int i = 0; i < VN; ++i) sum[i] = kept >> i & 1 ? scale.of_half(sum[i]) : 0.f;
  }
  put_chunk<T, VN>(row + chunk * VN, sum);
}

// Adds rows place(first) .. place(last - 1) of chunk `chunk`, eight on their way at a time.
template <typename T, int VN, typename F>
__device__ __forceinline__ void add_rows(const T* dz, int H, int chunk, int64_t first, int64_t last, F place, float (&sum)[VN]) {
  typedef T V __attribute__((ext_vector_type(VN)));
  constexpr int U = 8;
  int64_t i = first;
  for (; i + U <= last; i += U) {
    if constexpr (VN == 1) {
      T x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) x[j] = dz[place(i + j) * H + chunk];
#pragma unroll
      for (int j = 0; j < U; ++j) sum[0] += (float)x[j];
    } else {
      V x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) x[j] = *reinterpret_cast<const V*>(dz + place(i + j) * H + chunk * VN);
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int n = 0; n < VN; ++n) sum[n] += (float)x[j][n];
    }
  }
  for (; i < last; ++i) add_chunk(dz + place(i) * H + chunk * VN, sum);
}

// Parts of rows of the position table's gradient, a.lanes chunks of each, by a workgroup in groups of as many threads: a.share
// of them share the batch of a row.
template <typename T, int VN, int NT>
__device__ __forceinline__ void position_parts(const EmbedGradArgs& a, int64_t item, float* lds) {
  const int tid = threadIdx.x, lanes = a.lanes, group = tid / lanes, lane = tid - group * lanes;
  const int rows = NT / lanes / a.share, in_block = group / a.share, part = group - in_block * a.share;
  const int64_t block = item / a.across, l = block * rows + in_block;
  const int chunk = (int)(item - block * a.across) * lanes + lane;
  const bool there = in_block < rows && l < a.P && chunk < a.H / VN;
  const int64_t batch = l < a.L ? a.tokens / a.L : 0, share = (batch + a.share - 1) / a.share;
  const int64_t first = min((int64_t)part * share, batch), last = min(first + share, batch);
  float sum[VN];
  clear(sum);
  if (there) add_rows<T, VN>((const T*)a.dz, a.H, chunk, first, last, [&](int64_t b) { return b * a.L + l; }, sum);
  if (a.share > 1) {
    if (in_block < rows)
#pragma unroll
      for (int i = 0; i < VN; ++i) lds[(group * VN + i) * lanes + lane] = sum[i];
    __syncthreads();
    if (there && part == 0)
      for (int n = 1; n < a.share; ++n)
#pragma unroll
        for (int i = 0; i < VN; ++i) sum[i] += lds[((group + n) * VN + i) * lanes + lane];
  }
  if (there && part == 0) put_sum<T, VN>(a, (T*)a.d_wpe + l * a.H, chunk, kept_columns<VN>(a, chunk), sum);
}

// Threads that share a row's chunks: a power of two below a wavefront, whole wavefronts beyond.
__host__ __device__ __forceinline__ int lanes_of(int chunks, int most) {
  if (chunks >= most) return most;
  if (chunks > 32) return (chunks + 63) & ~63;
  int n = 1;
  while (n < chunks) n *= 2;
  return n;
}

// ---------------------------------------------------------------------------
// Up to kFew tokens: workgroups of `rows_of` tokens of the vocabulary each, then one for each position.
// ---------------------------------------------------------------------------
template <typename T, int VN>
__global__ __launch_bounds__(256) void embed_grad_few_kernel(EmbedGradArgs a, int rows_of, int vocab_blocks) {
  __shared__ float lds[256 * VN];
  __shared__ unsigned found[kFew], sorted[kFew];
  __shared__ int counts[4], begin[64 + 1];
  const int tid = threadIdx.x, chunks = a.H / VN, lanes = lanes_of(chunks, 256);
  if ((int)blockIdx.x >= vocab_blocks) {
    position_parts<T, VN, 256>(a, blockIdx.x - vocab_blocks, lds);
    return;
  }
  const int64_t v0 = (int64_t)blockIdx.x * rows_of;
  const int rows = (int)min((int64_t)rows_of, a.V - v0);
  const int64_t token = tid < a.tokens ? a.ids[tid] - v0 : -1;
  const bool mine = token >= 0 && token < rows;
  const uint64_t have = __ballot(mine);
  if ((tid & 63) == 0) counts[tid >> 6] = __popcll(have);
  __syncthreads();
  int in_front = 0, all = 0;
  for (int w = 0; w < 4; ++w) {
    if (w == tid >> 6) in_front = all;
    all += counts[w];
  }
  if (mine) found[in_front + __popcll(have & ((1ull << (tid & 63)) - 1))] = (unsigned)token << 8 | tid;
  __syncthreads();
  // by token, then position: a few of them, ranked by counting
  if (tid < all) {
    const unsigned me = found[tid];
    int rank = 0;
    for (int i = 0; i < all; ++i) rank += found[i] < me;
    sorted[rank] = me;
  }
  if (tid <= rows) {
    int n = 0;
    for (int i = 0; i < all; ++i) n += (int)(found[i] >> 8) < tid;
    begin[tid] = n;
  }
  __syncthreads();
  const T* dz = (const T*)a.dz;
  const int groups = 256 / lanes, group = tid / lanes, lane = tid - group * lanes;
  if (group >= groups) return;
  for (int r = group; r < rows; r += groups) {
    T* row = (T*)a.d_wte + (v0 + r) * a.H;
    const int first = begin[r], last = begin[r + 1];
    for (int chunk = lane; chunk < chunks; chunk += lanes) {
      float sum[VN];
      clear(sum);
      if (first < last) {
        add_rows<T, VN>(dz, a.H, chunk, first, last, [&](int64_t i) { return (int64_t)(sorted[i] & 255); }, sum);
        put_sum<T, VN>(a, row, chunk, kept_columns<VN>(a, chunk), sum);
      } else {
        put_chunk<T, VN>(row + chunk * VN, sum);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// More: the sort.
// ---------------------------------------------------------------------------
constexpr int kWaves = kSortThreads / kWave, kEach = kTile / kSortThreads;
struct SortLds {
  unsigned counts[kWaves][1 << kMaxBits];
  unsigned sums[kWaves];
};

__host__ __device__ __forceinline__ int64_t groups_of(int64_t tiles) { return (tiles + kGroupTiles - 1) / kGroupTiles; }

// Lanes of the wavefront with the same digit.
__device__ __forceinline__ uint64_t same_digit(unsigned digit, int bits, bool valid) {
  const uint64_t all = __ballot(valid);
  unsigned low = (unsigned)all, high = (unsigned)(all >> 32);
  for (int b = 0; b < bits; ++b) {
    const int set = (int)(digit << (31 - b)) >> 31;  // all ones or none
    const uint64_t ones = __ballot(set < 0);
    low &= ~((unsigned)ones ^ (unsigned)set);
    high &= ~((unsigned)(ones >> 32) ^ (unsigned)set);
  }
  return (uint64_t)high << 32 | low;
}

__device__ __forceinline__ unsigned key_of(const EmbedGradArgs& a, int64_t i) {
  const int64_t id = a.ids[i];
  return (unsigned)((uint64_t)id < (uint64_t)a.V ? id : a.V);
}

// What fills the GPU beside the sort: zero rows of the token table's gradient in blocks of 64 KB, and rows of the position
// table's.  Every launch of the sort has a part of each, in workgroups behind its own.
template <typename T, int VN>
__device__ __forceinline__ void other_work(const EmbedGradArgs& a, int64_t item, float* lds) {
  if (item < a.positions) {
    position_parts<T, VN, kSortThreads>(a, item, lds);
    return;
  }
  item += a.fill - a.positions;
  T* table = (T*)a.d_wte;
  int64_t elements = a.V * (int64_t)a.H;
  if (item >= a.table_fills) {
    item -= a.table_fills;
    table = (T*)a.d_wpe + a.P * a.H;
    elements = a.behind;
  }
  constexpr int64_t PER = kFill / sizeof(T);
  const int64_t first = item * PER, last = min(first + PER, elements);
  float none[VN];
  clear(none);
  for (int64_t i = first + threadIdx.x * VN; i < last; i += kSortThreads * VN) put_chunk<T, VN>(table + i, none);
}

// Where this thread's tokens go by one digit: wavefront w has tokens 64 EACH w .. of the tile, 64 at a time.  place_of: the
// first place of each digit for this tile, by the threads of the digits.
template <int EACH, typename F>
__device__ __forceinline__ void rank_tile(SortLds& lds, int count, int bits, int shift, const unsigned (&key)[EACH],
                                          unsigned (&place)[EACH], F place_of) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, digits = 1 << bits, base = wave * (kWave * EACH);
  for (int i = tid; i < kWaves << bits; i += kSortThreads) lds.counts[i >> bits][i & (digits - 1)] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const bool valid = base + j * kWave + lane < count;
    const unsigned digit = key[j] >> shift & (digits - 1);
    const uint64_t same = same_digit(digit, bits, valid);
    const int in_front = __popcll(same & ((1ull << lane) - 1));
    volatile unsigned* counted = &lds.counts[wave][digit];
    place[j] = *counted + in_front;
    __builtin_amdgcn_wave_barrier();
    if (valid && in_front == 0) *counted = place[j] + __popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // behind all of smaller digits: the sum of what place_of counts of them
  unsigned mine = 0, before = 0;
  if (tid < digits)
    for (int w = 0; w < kWaves; ++w) mine += lds.counts[w][tid];
  const unsigned total = place_of(mine, &before);
  unsigned scan = total;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const unsigned other = __shfl_up(scan, step);
    scan += lane >= step ? other : 0;
  }
  if (lane == 63) lds.sums[wave] = scan;
  __syncthreads();
  for (int w = 0; w < wave; ++w) scan += lds.sums[w];
  if (tid < digits) {
    unsigned sum = scan - total + before;
    for (int w = 0; w < kWaves; ++w) {
      const unsigned n = lds.counts[w][tid];
      lds.counts[w][tid] = sum;
      sum += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j) place[j] += lds.counts[wave][key[j] >> shift & (digits - 1)];
}

// A single tile: all digits in one workgroup, EACH tokens a thread.
template <typename T, int VN, int EACH>
struct TileLds {
  union {
    SortLds s;
    float other[kSortThreads * VN];
  };
  unsigned keys[kSortThreads * EACH];
  uint16_t at[kSortThreads * EACH];
};
template <typename T, int VN, int EACH>
__global__ __launch_bounds__(kSortThreads) void embed_grad_sort_kernel(EmbedGradArgs a, int passes) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  TileLds<T, VN, EACH>& lds = *reinterpret_cast<TileLds<T, VN, EACH>*>(smem);
  if (blockIdx.x > 0) {
    other_work<T, VN>(a, blockIdx.x - 1, lds.other);
    return;
  }
  const int count = (int)a.tokens, base = (threadIdx.x >> 6) * (kWave * EACH) + (threadIdx.x & 63);
  unsigned key[EACH], from[EACH], place[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = base + j * kWave;
    key[j] = i < count ? key_of(a, i) : 0;
    from[j] = (unsigned)i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    rank_tile(lds.s, count, a.bits, pass * a.bits, key, place, [](unsigned mine, unsigned*) { return mine; });
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (base + j * kWave < count) {
        lds.keys[place[j]] = key[j];
        lds.at[place[j]] = (uint16_t)from[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = base + j * kWave;
      key[j] = i < count ? lds.keys[i] : 0;
      from[j] = i < count ? lds.at[i] : 0;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int i = base + j * kWave;
    if (i < count) {
      a.keys[0][i] = key[j];
      a.at[0][i] = from[j];
    }
  }
}

// More tiles, a launch to count and one to move for each digit.  How many tokens of each tile have each digit; FIRST: from the
// ids themselves.
template <typename T, int VN, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embed_grad_count_kernel(EmbedGradArgs a, int shift, int from) {
  __shared__ union {
    unsigned counts[1 << kMaxBits];
    float other[kSortThreads * VN];
  } lds;
  if ((int)blockIdx.x >= a.tiles) {
    other_work<T, VN>(a, (int64_t)blockIdx.x - a.tiles, lds.other);
    return;
  }
  const int tid = threadIdx.x, digits = 1 << a.bits;
  const int64_t base = (int64_t)blockIdx.x * kTile;
  unsigned key[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int64_t i = base + j * kSortThreads + tid;
    key[j] = 0;
    if (i < a.tokens) key[j] = FIRST ? key_of(a, i) : a.keys[from][i];
  }
  if (tid < digits) lds.counts[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (base + j * kSortThreads + tid < a.tokens) atomicAdd(&lds.counts[key[j] >> shift & (digits - 1)], 1u);
  __syncthreads();
  if (tid < digits) a.hist[(int64_t)blockIdx.x * digits + tid] = lds.counts[tid];
}

// Many tiles: the counts of kGroupTiles tiles together,
__global__ __launch_bounds__(kSortThreads) void embed_grad_group_kernel(EmbedGradArgs a) {
  __shared__ unsigned other[1 << kMaxBits];
  constexpr int HALF = kSortThreads / 2;
  const int digits = 1 << a.bits, digit = threadIdx.x % HALF, half = threadIdx.x / HALF;
  const int64_t first = (int64_t)blockIdx.x * kGroupTiles, last = min(first + kGroupTiles, (int64_t)a.tiles);
  unsigned sum = 0;
  if (digit < digits) {
#pragma unroll 16
    for (int64_t t = first + half; t < last; t += 2) sum += a.hist[t * digits + digit];
  }
  if (half == 1) other[digit] = sum;
  __syncthreads();
  if (half == 0 && digit < digits) a.group_counts[(int64_t)blockIdx.x * digits + digit] = sum + other[digit];
}
// and each tile's counts as those of the tiles in front of it.
__global__ __launch_bounds__(kSortThreads / 2) void embed_grad_in_front_kernel(EmbedGradArgs a) {
  static_assert(kSortThreads / 2 >= 1 << kMaxBits, "a thread a digit");
  constexpr int U = 16;
  const int digits = 1 << a.bits, digit = threadIdx.x, groups = gridDim.x;
  if (digit >= digits) return;
  unsigned in_front = 0, total = 0;
#pragma unroll 16
  for (int g = 0; g < groups; ++g) {
    const unsigned n = a.group_counts[(int64_t)g * digits + digit];
    in_front += g < (int)blockIdx.x ? n : 0;
    total += n;
  }
  if (blockIdx.x == 0) a.group_counts[(int64_t)groups * digits + digit] = total;  // behind what the other workgroups read
  const int64_t first = (int64_t)blockIdx.x * kGroupTiles, last = min(first + kGroupTiles, (int64_t)a.tiles);
  for (int64_t t = first; t < last; t += U) {
    unsigned n[U];
#pragma unroll
    for (int j = 0; j < U; ++j) n[j] = a.hist[min(t + j, last - 1) * digits + digit];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (t + j < last) a.hist[(t + j) * digits + digit] = in_front;
      in_front += n[j];
    }
  }
}

// Moves the tokens to their places by one digit.
template <typename T, int VN, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void embed_grad_move_kernel(EmbedGradArgs a, int shift, int from) {
  __shared__ union {
    SortLds s;
    float other[kSortThreads * VN];
  } lds;
  if ((int)blockIdx.x >= a.tiles) {
    other_work<T, VN>(a, (int64_t)blockIdx.x - a.tiles, lds.other);
    return;
  }
  const int tid = threadIdx.x, digits = 1 << a.bits;
  const int64_t first = (int64_t)blockIdx.x * kTile;
  const int count = (int)min((int64_t)kTile, a.tokens - first), base = (tid >> 6) * (kWave * kEach) + (tid & 63);
  unsigned key[kEach], at[kEach], place[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = base + j * kWave;
    key[j] = at[j] = 0;
    if (i < count) {
      key[j] = FIRST ? key_of(a, first + i) : a.keys[from][first + i];
      at[j] = FIRST ? (unsigned)(first + i) : a.at[from][first + i];
    }
  }
  // of each digit, the tokens of all tiles, and of those in front of this one
  unsigned total = 0, in_front = 0;
  if (a.many) {
    if (tid < digits) {
      in_front = a.hist[(int64_t)blockIdx.x * digits + tid];
      total = a.group_counts[(int64_t)groups_of(a.tiles) * digits + tid];
    }
  } else if (tid < digits) {
#pragma unroll 16
    for (int t = 0; t < a.tiles; ++t) {
      const unsigned n = a.hist[(int64_t)t * digits + tid];
      in_front += t < (int)blockIdx.x ? n : 0;
      total += n;
    }
  }
  rank_tile(lds.s, count, a.bits, shift, key, place, [&](unsigned, unsigned* before) {
    *before = in_front;
    return total;
  });
  unsigned* keys = a.keys[1 - from];
  unsigned* to = a.at[1 - from];
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (base + j * kWave < count) {
      keys[place[j]] = key[j];
      to[place[j]] = at[j];
    }
}

// ---------------------------------------------------------------------------
// The sums of runs of a.run sorted tokens, a group of threads a run.
// ---------------------------------------------------------------------------
template <typename T, int VN>
__global__ __launch_bounds__(256) void embed_grad_sum_kernel(EmbedGradArgs a) {
  typedef T V __attribute__((ext_vector_type(VN)));
  const int chunks = a.H / VN, lanes = lanes_of(chunks, 256), groups = 256 / lanes;
  const int group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes;
  const int64_t runs = (a.tokens + a.run - 1) / a.run, r = (int64_t)blockIdx.x * groups + group;
  if (group >= groups || r >= runs) return;
  const int64_t first = r * a.run;
  const int count = (int)min((int64_t)a.run, a.tokens - first);
  const T* dz = (const T*)a.dz;
  const unsigned *tokens = a.sorted + first, *rows = a.order + first;
  const unsigned none = (unsigned)a.V;
  const unsigned before = first > 0 ? tokens[-1] : ~0u, behind = first + count < a.tokens ? tokens[count] : ~0u;
  constexpr int U = 8;
  for (int chunk = blockIdx.y * 256 + lane; chunk < min(chunks, (int)(blockIdx.y + 1) * 256); chunk += lanes) {
    float sum[VN];
    clear(sum);
    const unsigned kept = kept_columns<VN>(a, chunk);
    bool began = tokens[0] != before;  // the token at hand began in this run
    unsigned row[U], token[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      row[j] = rows[min(j, count - 1)];
      token[j] = tokens[min(j, count - 1)];
    }
    for (int i0 = 0; i0 < count; i0 += U) {
      V x[U];
      unsigned now[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {  // rows behind the last token are rows all the same
        const T* from = dz + (int64_t)row[j] * a.H + chunk * VN;
        if constexpr (VN == 1) x[j][0] = *from;
        else x[j] = *reinterpret_cast<const V*>(from);
        now[j] = token[j];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        row[j] = rows[min(i0 + U + j, count - 1)];
        token[j] = tokens[min(i0 + U + j, count - 1)];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const bool there = i0 + j < count && now[j] != none, end = i0 + j == count - 1;
        const unsigned next = end ? behind : j + 1 < U ? now[j + 1 < U ? j + 1 : 0] : token[0];
        if (there) {
#pragma unroll
          for (int n = 0; n < VN; ++n) sum[n] += (float)x[j][n];
          if (next != now[j]) {
            if (began) put_sum<T, VN>(a, (T*)a.d_wte + (int64_t)now[j] * a.H, chunk, kept, sum);
            else put_chunk<float, VN>(a.parts + (r * 2) * a.H + chunk * VN, sum);
            clear(sum);
            began = true;
          } else if (end) {
            put_chunk<float, VN>(a.parts + (r * 2 + (began ? 1 : 0)) * a.H + chunk * VN, sum);
          }
        }
      }
    }
  }
}

// The tokens that go on behind the run in which they began: a workgroup each run, most of which have none.
template <typename T, int VN>
__global__ __launch_bounds__(256) void embed_grad_join_kernel(EmbedGradArgs a) {
  __shared__ float lds[256 * VN];
  const int64_t r = blockIdx.x, first = r * a.run, last = first + a.run;
  const unsigned token = a.sorted[last - 1];  // no workgroup has the last run
  if (a.sorted[last] != token || token == (unsigned)a.V) return;
  if (a.sorted[first] == token && first > 0 && a.sorted[first - 1] == token) return;
  // runs behind that begin with it
  const int64_t runs = (a.tokens + a.run - 1) / a.run;
  int64_t more = 0;
  for (;;) {
    const int64_t at = r + 1 + more + (threadIdx.x & 63);
    const int n = __popcll(__ballot(at < runs && a.sorted[min(at, runs - 1) * a.run] == token));
    more += n;
    if (n < kWave) break;
  }
  const int chunks = a.H / VN, lanes = lanes_of(chunks, 256), groups = 256 / lanes;
  const int group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes;
  const int64_t share = (more + groups - 1) / groups;
  const int64_t from = min((int64_t)group * share, more), to = group < groups ? min(from + share, more) : from;
  for (int c0 = blockIdx.y * 256; c0 < min(chunks, (int)(blockIdx.y + 1) * 256); c0 += lanes) {
    const int chunk = c0 + lane;
    float sum[VN];
    clear(sum);
    if (group < groups && chunk < chunks) {
      if (group == 0) add_chunk(a.parts + (r * 2 + 1) * a.H + chunk * VN, sum);
      add_rows<float, VN>(a.parts, a.H, chunk, from, to, [&](int64_t i) { return (r + 1 + i) * 2; }, sum);
    }
    if (groups > 1) {
      __syncthreads();
      if (group < groups)
#pragma unroll
        for (int i = 0; i < VN; ++i) lds[(group * VN + i) * lanes + lane] = sum[i];
      __syncthreads();
      if (group == 0)
        for (int n = 1; n < groups; ++n)
#pragma unroll
          for (int i = 0; i < VN; ++i) sum[i] += lds[(n * VN + i) * lanes + lane];
    }
    if (group == 0 && chunk < chunks) put_sum<T, VN>(a, (T*)a.d_wte + (int64_t)token * a.H, chunk, kept_columns<VN>(a, chunk), sum);
  }
}

// Only the position table's.
template <typename T, int VN>
__global__ __launch_bounds__(kSortThreads) void embed_grad_positions_kernel(EmbedGradArgs a) {
  __shared__ float lds[kSortThreads * VN];
  position_parts<T, VN, kSortThreads>(a, blockIdx.x, lds);
}

template <typename T, int VN, int EACH>
int launch_sort(const EmbedGradArgs& a, unsigned blocks, int passes, hipStream_t st) {
  const auto kernel = embed_grad_sort_kernel<T, VN, EACH>;
  constexpr int lds = sizeof(TileLds<T, VN, EACH>);
  static bool attr_done = false;  // idempotent; a race only repeats the call
  if (!attr_done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("hipFuncSetAttribute(%d bytes LDS): %s", lds, hipGetErrorString(e));
      return -4;
    }
    attr_done = true;
  }
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kSortThreads), lds, st, a, passes);
  return 0;
}

int run_of(int64_t tokens) { return tokens >= 1 << 17 ? 128 : tokens >= 1 << 15 ? 64 : 32; }

template <typename T, int VN>
int launch_as(EmbedGradArgs a, hipStream_t st) {
  const int chunks = a.H / VN;
  // The batch of a row of the position table is shared, by groups that are narrower then, where the rows alone would be few threads
  // (us, 583 x 11 tokens, 1280 wide, fp32: 126 as whole rows, 102 shared by 16 groups, 77 with the zero rows behind them filled as the
  // token table's are; 512 x 300 fp16, 768 wide, of which the launch with them: 57 by 8, 63 by 16).
  const int threads = a.d_wte && a.tokens <= kFew ? 256 : kSortThreads;
  int64_t positions = 0;  // workgroups
  if (a.d_wte && a.tokens > kFew) {  // rows of the position table that no token has are zero rows as the others
    a.behind = a.d_wpe ? (a.P - a.L) * a.H : 0;
    a.P = a.L;
  }
  const auto share_by = [&](int share) {
    a.share = share;
    a.lanes = lanes_of(chunks, threads / share);
    a.across = (chunks + a.lanes - 1) / a.lanes;
    const int rows = threads / a.lanes / share;
    positions = a.d_wpe ? (a.P + rows - 1) / rows * a.across : 0;
  };
  share_by(1);
  while (a.share < threads / 64 && a.share < a.tokens / a.L && a.L * chunks * a.share < 1 << 17 && positions < 1 << 19)
    share_by(2 * a.share);
  if (!a.d_wte) {
    hipLaunchKernelGGL((embed_grad_positions_kernel<T, VN>), dim3((unsigned)positions), dim3(kSortThreads), 0, st, a);
    return 0;
  }
  if (a.tokens <= kFew) {
    // up to 64 rows a workgroup, fewer where that leaves CUs without one
    int rows = 64;
    while (rows > 4 && (a.V + rows - 1) / rows < 512) rows /= 2;
    const int64_t blocks = (a.V + rows - 1) / rows;
    hipLaunchKernelGGL((embed_grad_few_kernel<T, VN>), dim3((unsigned)(blocks + positions)), dim3(256), 0, st, a, rows,
                       (int)blocks);
    return 0;
  }
  int width = 1;
  while (a.V >> width) ++width;  // bits of V, the key of no token
  const int passes = (width + kMaxBits - 1) / kMaxBits;
  a.bits = (width + passes - 1) / passes;
  a.tiles = (int)((a.tokens + kTile - 1) / kTile);
  a.many = a.tiles > kManyTiles;
  const auto fills_of = [](int64_t elements) { return (elements * (int64_t)sizeof(T) + kFill - 1) / kFill; };
  a.table_fills = fills_of(a.V * a.H);
  const int64_t fills = a.table_fills + fills_of(a.behind);
  if (a.tokens <= kOneTile) {
    a.positions = positions;
    const unsigned blocks = (unsigned)(1 + fills + positions);
    const int rc = a.tokens <= kTile ? launch_sort<T, VN, kEach>(a, blocks, passes, st)
                                     : launch_sort<T, VN, kOneTile / kSortThreads>(a, blocks, passes, st);
    if (rc) return rc;
    a.sorted = a.keys[0];
    a.order = a.at[0];
  } else {
    // The last launch has the position table's rows, few and long ones; a launch that counts takes about half as long as one
    // that moves, so the others divide the zero rows in thirds a pass.  us, 512 x 300 tokens fp16, the sort's launches with all
    // zero rows in the first and the positions in the second / all divided / this: 91 / 102 / 84.
    int64_t end = 0;
    const auto part = [&](int third, int pass) {
      const int64_t in = 3 * pass + third, of = 3 * passes - 2;
      a.fill = end;
      end = fills * (in < of ? in : of) / of;
      a.positions = in > of ? positions : 0;
      return dim3((unsigned)(a.tiles + a.positions + end - a.fill));
    };
    for (int pass = 0; pass < passes; ++pass) {
      const int shift = pass * a.bits, from = pass & 1;
      const dim3 count = part(1, pass);
      if (pass == 0)
        hipLaunchKernelGGL((embed_grad_count_kernel<T, VN, true>), count, dim3(kSortThreads), 0, st, a, shift, from);
      else
        hipLaunchKernelGGL((embed_grad_count_kernel<T, VN, false>), count, dim3(kSortThreads), 0, st, a, shift, from);
      if (a.many) {
        const dim3 groups((unsigned)groups_of(a.tiles));
        hipLaunchKernelGGL(embed_grad_group_kernel, groups, dim3(kSortThreads), 0, st, a);
        hipLaunchKernelGGL(embed_grad_in_front_kernel, groups, dim3(kSortThreads / 2), 0, st, a);
      }
      const dim3 move = part(3, pass);
      if (pass == 0)
        hipLaunchKernelGGL((embed_grad_move_kernel<T, VN, true>), move, dim3(kSortThreads), 0, st, a, shift, from);
      else
        hipLaunchKernelGGL((embed_grad_move_kernel<T, VN, false>), move, dim3(kSortThreads), 0, st, a, shift, from);
    }
    a.sorted = a.keys[passes & 1];
    a.order = a.at[passes & 1];
  }
  const int groups = 256 / lanes_of(chunks, 256);
  const int64_t runs = (a.tokens + a.run - 1) / a.run;
  const unsigned across = (unsigned)((chunks + 255) / 256);
  hipLaunchKernelGGL((embed_grad_sum_kernel<T, VN>), dim3((unsigned)((runs + groups - 1) / groups), across), dim3(256), 0, st, a);
  if (runs > 1)
    hipLaunchKernelGGL((embed_grad_join_kernel<T, VN>), dim3((unsigned)(runs - 1), across), dim3(256), 0, st, a);
  return 0;
}

int64_t up(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }
// Of the tiles' counts, and the groups' and all together.
int64_t hist_bytes(int64_t tokens) {
  const int64_t tiles = (tokens + kTile - 1) / kTile;
  return up(tiles * (4 << kMaxBits)) + (tiles > kManyTiles ? up((groups_of(tiles) + 1) * (4 << kMaxBits)) : 0);
}

}  // namespace

size_t embed_grad_bytes(int64_t tokens, int64_t H) {
  if (tokens <= kFew) return 0;
  const int64_t run = run_of(tokens), runs = (tokens + run - 1) / run;
  return (size_t)(4 * up(tokens * 4) + hist_bytes(tokens) + up(runs * 2 * H * 4));
}

int launch_embed_backward(const int64_t* ids, const void* dz, void* d_wte, void* d_wpe, int64_t tokens, int64_t L, int64_t V,
                          int64_t P, int H, Dropout drop, bool f16, void* workspace, hipStream_t st) {
  EmbedGradArgs a = {};
  a.ids = ids;
  a.dz = dz;
  a.d_wte = d_wte;
  a.d_wpe = d_wpe;
  a.tokens = tokens, a.L = L, a.V = V, a.P = P, a.H = H;
  a.drop = DropoutArgs{drop.p, (unsigned)drop.seed, (unsigned)(drop.seed >> 32)};
  a.run = run_of(tokens);
  char* ws = (char*)workspace;
  for (int i = 0; i < 2; ++i) {
    a.keys[i] = (unsigned*)(ws + (2 * i) * up(tokens * 4));
    a.at[i] = (unsigned*)(ws + (2 * i + 1) * up(tokens * 4));
  }
  a.hist = (unsigned*)(ws + 4 * up(tokens * 4));
  a.group_counts = (unsigned*)((char*)a.hist + up((tokens + kTile - 1) / kTile * (4 << kMaxBits)));
  a.parts = (float*)((char*)a.hist + hist_bytes(tokens));
  const uintptr_t all = (uintptr_t)dz | (uintptr_t)d_wte | (uintptr_t)d_wpe;
  if (f16) return H % 8 == 0 && (all & 15) == 0 ? launch_as<_Float16, 8>(a, st) : launch_as<_Float16, 1>(a, st);
  return H % 4 == 0 && (all & 15) == 0 ? launch_as<float, 4>(a, st) : launch_as<float, 1>(a, st);
}

}  // namespace gptmi
