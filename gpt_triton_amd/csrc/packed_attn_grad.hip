// Gradients of causal attention over packed sequences (packed_attn.hip).  With t = scale, w_ij = softmax_j(t q_i . k_j)
// over the keys j <= i of i's sequence, and e_i the gradient of the output o_i = sum_j w_ij v_j:
//   delta_i = sum_j w_ij (e_i . v_j) = e_i . o_i,   u_ij = w_ij (e_i . v_j - delta_i)
//   dq_i = t sum_j u_ij k_j,   dk_j = t sum_i u_ij q_i,   dv_j = sum_i w_ij e_i
// over the queries i >= j of all the heads that share a key head.  The weights are formed again from q, k and the
// statistic that the forward pass keeps of each row, so nothing of the size of the scores goes to memory.
//
// Launches: row sums (delta, and e's and v's squares); what goes by sequences (delta of the first queries as sums over their
// keys, in place of the row sums'; the largest rows of each key head); the walk of the keys (dk and dv: a workgroup has a block of keys and walks over the queries) and the
// walk of the queries (dq: a block of queries, over the keys), up to d = 64 in one launch; and, where the heads over a key head
// are divided among workgroups, their sums' join.  So each sum is formed by one workgroup in one order, without atomics, at the
// cost of forming w and u twice: 7 products instead of 5.
//
// u sums to 0 over a row's keys as far as delta is right: an error of delta is one of all of the row's u, and dq has it times
// the mean of the keys.  So delta comes from the output and what its rounding takes, which the forward pass keeps: 2-norms of dq's
// errors, 1 x 1024 tokens, 12 heads of 64, of which u's rounding has its part whatever delta is: 3.0e-4 for keys and
// values of unit spread, 4.0e-4, 8.4e-4 and 2.7e-3 where their channels have offsets of 1, 3 and 10 as well; from the rounded output
// 3.0e-4, 1.9e-3, 1.7e-2 and 0.19.  dk 2.9e-4 to 3.0e-4; 3.0e-4, 3.5e-4, 6.3e-4, 1.9e-3.  It costs 26 us of the forward pass of
// 1 x 8192 tokens below and 3 of its row sums.
//
// Both walks are one kernel: rows x in registers (k and v, or q and e), rows y that pass through LDS (q and e, or k and v).
// The products are Y . X^T with v_mfma_f32_16x16x32_f16, whose result lane (c, g), c = lane % 16, g = lane / 16, has
// row c of x and four rows of y; rows 4 g + r of the two 16-row blocks b of a group of 32 are y's rows 8 g + 4 b + r, so
// that w and u, rounded to fp16, are the second operand of the sums over y as they stand.
//
// What bounds it: the matrix pipe and the vector pipe in turn.  us, the row sums and the walks, causal:
//   25 heads of 64, 1 x 8192 tokens: 775 (7 products of L^2 d operations a head: 970 TFLOP/s, where a large library product
//     reaches 1212; MFMA 0.44 and VALU 0.51 busy at 2.1 GHz); two wavefronts a SIMD and two launches 13 % more
//   32 heads of 128 over 8, texts of 4096, 4095, 2049, 1933, 517 and 64: 1400 (855 TFLOP/s; the keys' walk with one wavefront a SIMD,
//     whose steps overlap; without overlap 18 % more); eight narrower wavefronts for it 844 where it took 834, tiles of 128 rows 949
//   12 heads of 64, 48 texts of up to 1024, 7276 rows: 62, 48 x 300: 81, of which the row sums 17, the sequences'
//     launch 4, and more than half of the rest workgroups' starts, finding their rows, first loads and results
//   12 heads of 32, 16 x 1024: 98, of which the walks 80 to 90; the vector pipe is busy for 45 of these (70 cycles for 64 pairs of a query
//     and a key in both walks, 32 of them exponentials), the matrix pipe for 18; of 16 91, 46 and 14
// Registers that are spilled (64 wide 32, 256 wide 13 and 81) are used row by row, which the next lines are about, and behind the walks' loops.
// A backward pass with an infinity or a NaN among the output's gradients goes row by row where that reaches, 10 to 50 times as long
// (12 heads of 64, 1 x 1024: 1400 us, 48 x 300: 560 for one of them, 2000 for nothing else): a step that a training loop skips.
#include <type_traits>
#include <utility>

#include "common.h"
#include "launch.h"
#include "packed_attn.h"

namespace gptmi {
namespace {

// The weights are formed as 2^kUp w and u as 2^kUp f u, f a power of two: fp16 numbers of the size of one that stay
// normal numbers down to 2^-28 of it.
constexpr int kUp = 14;
constexpr int kSums = 1024;         // workgroups of the row sums at most
constexpr int kSequenceBlocks = 1 << 16;  // of either part of the sequences' launch

struct SlotDeal {
  int slots, grid;
  bool longest_first;
};
struct GradArgs {
  const _Float16 *q, *k, *v, *out, *remainder, *d_out;  // remainder: the forward pass's, or nullptr
  _Float16 *dq, *dk, *dv;  // dense; dq, or dk and dv, may be nullptr
  const float2* stats;     // [heads][T], the forward pass's
  float *lse, *minus_delta;  // [heads][T]: 2^kUp w = 2^(s t log2(e) - lse); a NaN: see packed_sums_kernel
  float *e_squares, *v_squares;  // e . e [heads][T], v . v [kv_heads][T], 0 where it is no number; behind the launch of the sequences, the
                                 // first row of a sequence and key head has the largest of all of it
  int firsts;                    // workgroups of that launch for the first queries, behind them those for the largest rows
  bool whole;                    // each of which has a sequence and key head, else each wavefront
  const int64_t* starts;
  int64_t rows;  // T
  int sequences, heads, kv_heads;
  SlotDeal deal[2];  // of the blocks of queries, and of keys
  int shares;        // into which the heads that share a key head are divided
  float* parts;      // more than one: their sums, [shares][2][T][kv_heads][d], dk and dv
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // pitches in elements
  float scale;
};

// ---------------------------------------------------------------------------
// delta, lse, and squares of e's and v's rows.  Rows that belong to no sequence get gradients of 0 here.
// A row whose statistic is of scores key by key (infinities and NaN, scores of some thousands) gets lse = NaN: what meets it
// comes out as NaN, and is done again with the statistic itself.
// ---------------------------------------------------------------------------
template <int D>
__global__ __launch_bounds__(256) void packed_sums_kernel(GradArgs a) {
  constexpr int LPR = D / 8;          // lanes a row
  constexpr int RPP = 256 / LPR;      // rows a pass
  constexpr int BLOCK = RPP > 64 ? RPP : 64, PASSES = BLOCK / RPP;
  const int tid = threadIdx.x, in_row = tid % LPR, row_of = tid / LPR;
  const int64_t from = a.starts[0], to = a.starts[a.sequences];
  const int64_t items = (a.rows + BLOCK - 1) / BLOCK * a.heads;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t block = item / a.heads;
    const int head = (int)(item - block * a.heads);
    // all rows' loads first
    h8 e[PASSES], o[PASSES], rest[PASSES], v[PASSES];
    float2 stat[PASSES];
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int64_t row = block * BLOCK + pass * RPP + row_of, at = (row * a.heads + head) * D + in_row * 8;
      e[pass] = o[pass] = rest[pass] = v[pass] = h8(0);
      if (row < from || row >= to || row >= a.rows) continue;
      e[pass] = *reinterpret_cast<const h8*>(a.d_out + at);
      o[pass] = *reinterpret_cast<const h8*>(a.out + at);
      if (a.remainder) rest[pass] = *reinterpret_cast<const h8*>(a.remainder + at);
      if (head < a.kv_heads) v[pass] = *reinterpret_cast<const h8*>(a.v + row * a.v_row + head * a.v_head + in_row * 8);
      stat[pass] = a.stats[head * a.rows + row];
    }
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int64_t row = block * BLOCK + pass * RPP + row_of;
      if (row >= a.rows) break;
      if (row < from || row >= to) {
        const int64_t at = (row * a.heads + head) * D + in_row * 8, kv_at = (row * a.kv_heads + head) * D + in_row * 8;
        if (a.dq) *reinterpret_cast<h8*>(a.dq + at) = h8(0);
        if (a.dk && head < a.kv_heads) *reinterpret_cast<h8*>(a.dk + kv_at) = *reinterpret_cast<h8*>(a.dv + kv_at) = h8(0);
        continue;
      }
      float dot = 0.f, ee = 0.f, vv = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dot = fmaf((float)e[pass][i], fmaf((float)rest[pass][i], 0x1p-10f, (float)o[pass][i]), dot);
        ee = fmaf((float)e[pass][i], (float)e[pass][i], ee);
        vv = fmaf((float)v[pass][i], (float)v[pass][i], vv);
      }
#pragma unroll
      for (int step = 1; step < LPR; step *= 2) {
        dot += __shfl_xor(dot, step);
        ee += __shfl_xor(ee, step);
        vv += __shfl_xor(vv, step);
      }
      if (in_row == 0) {
        const int64_t place = head * a.rows + row;
        a.lse[place] = stat[pass].x - __builtin_amdgcn_logf(stat[pass].y) - kUp;  // to the base 2; NaN where .y < 0
        a.minus_delta[place] = -dot;
        // rows with an infinity or a NaN spoil only what they are part of
        a.e_squares[place] = ee < INFINITY ? ee : 0.f;
        if (head < a.kv_heads) a.v_squares[place] = vv < INFINITY ? vv : 0.f;
      }
    }
  }
}

// 4 bytes a lane, as load_lds16.
__device__ __forceinline__ void load_lds4(const void* base, unsigned lane_off, unsigned lds_off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds_off), "v"(lane_off), "s"(base)
               : "memory", "m0");
}

__device__ __forceinline__ h8 lds_read16(unsigned at) {
  return *(const __attribute__((address_space(3))) h8*)(uintptr_t)at;
}

// delta of a sequence's first 16 queries as the sum over their keys, a wavefront for a sequence and head.  e . o is off by what the
// forward pass's weights were rounded by, which few keys do not average out: dq of a text of 24 tokens is (2-norm, relative) 2.9e-4
// off with both, 8.6e-4 and this way 7.7e-4 where the channels of keys and values have offsets of 3.  3 us.
template <int D>
__device__ __forceinline__ void first_queries(const GradArgs& a, int block) {
  constexpr int KS = (D + 31) / 32;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t items = (int64_t)a.sequences * a.heads;
  for (int64_t item = (int64_t)block * 4 + wave; item < items; item += (int64_t)a.firsts * 4) {
    const int64_t sequence = item / a.heads;
    const int head = (int)(item - sequence * a.heads), kv_head = head / (a.heads / a.kv_heads);
    const int64_t begin = a.starts[sequence], end = a.starts[sequence + 1];
    const int64_t first = begin < 0 ? 0 : begin < a.rows ? begin : a.rows;
    const int64_t last = end < first ? first : end < a.rows ? end : a.rows;
    if (last - first < 2) continue;
    const int L = (int)min(last - first, (int64_t)16);
    const int64_t row = first + min(c, L - 1);
    const _Float16 *q = a.q + (row * a.q_row + head * a.q_head) + g * 8, *k = a.k + (row * a.k_row + kv_head * a.k_head) + g * 8;
    const _Float16 *v = a.v + (row * a.v_row + kv_head * a.v_head) + g * 8, *e = a.d_out + (row * a.heads + head) * D + g * 8;
    f4 s = f4(0.f), p = f4(0.f);  // of query c, keys 4 g + 0..3
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      h8 x[4] = {h8(0), h8(0), h8(0), h8(0)};
      if (D >= 32 || g < 2) {
        x[0] = *reinterpret_cast<const h8*>(k + ks * 32);
        x[1] = *reinterpret_cast<const h8*>(q + ks * 32);
        x[2] = *reinterpret_cast<const h8*>(v + ks * 32);
        x[3] = *reinterpret_cast<const h8*>(e + ks * 32);
      }
      s = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[0], x[1], s, 0, 0, 0);
      p = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[2], x[3], p, 0, 0, 0);
    }
    const int64_t place = head * a.rows + row;
    const float lse = a.lse[place];
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float w = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale * 1.4426950408889634f, -lse));
      sum = 4 * g + r <= c ? fmaf(w, p[r], sum) : sum;
    }
    const LanePair pair = row_swap(half_sum(sum));
    sum = (pair.a + pair.b) * 0x1p-14f;
    static_assert(kUp == 14, "of lse");
    if (g == 0 && c < L && fabsf(sum) < INFINITY) a.minus_delta[place] = -sum;  // else a row that is marked, or none
  }
}

// The largest of n numbers, 0 at least, in every thread of THREADS that share them: a wavefront, or the workgroup.
template <int THREADS>
__device__ __forceinline__ float largest_of(const float* x, int64_t pitch, int rows, unsigned n, float* lds) {
  constexpr int U = 8;
  float most = 0.f;
  for (int row = 0; row < rows; ++row, x += pitch)
    for (unsigned i = threadIdx.x % THREADS; i < n; i += U * THREADS) {
      float some[U];
#pragma unroll
      for (int j = 0; j < U; ++j) some[j] = x[min(i + j * THREADS, n - 1)];
#pragma unroll
      for (int j = 0; j < U; ++j) most = fmaxf(most, some[j]);
    }
  most = wave_max(most);
  if constexpr (THREADS > kWave) {
    __syncthreads();
    lds[threadIdx.x >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
  }
  return most;
}

// The largest rows of e and v of each sequence and key head, in its first row's places.
template <int THREADS>
__device__ __forceinline__ void largest_rows(const GradArgs& a, int block, int blocks, float* lds) {
  constexpr int TEAMS = 256 / THREADS;
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS), per_key = a.heads / a.kv_heads;
  const int64_t items = (int64_t)a.sequences * a.kv_heads;
  for (int64_t item = (int64_t)block * TEAMS + team; item < items; item += (int64_t)blocks * TEAMS) {
    const int64_t sequence = item / a.kv_heads;
    const int kv_head = (int)(item - sequence * a.kv_heads);
    const int64_t begin = a.starts[sequence], end = a.starts[sequence + 1];
    const int64_t first = begin < 0 ? 0 : begin < a.rows ? begin : a.rows;
    const int64_t last = end < first ? first : end < a.rows ? end : a.rows;
    if (first == last) continue;
    float* e = a.e_squares + ((int64_t)kv_head * per_key * a.rows + first);
    float* v = a.v_squares + (kv_head * a.rows + first);
    const float most_e = largest_of<THREADS>(e, a.rows, per_key, (unsigned)(last - first), lds);
    const float most_v = largest_of<THREADS>(v, a.rows, 1, (unsigned)(last - first), lds);
    if (threadIdx.x % THREADS == 0) *e = most_e, *v = most_v;  // all of them have been read
  }
}

// What goes by sequences: their first queries' deltas, and their largest rows.
template <int D>
__global__ __launch_bounds__(256) void packed_sequences_kernel(GradArgs a) {
  __shared__ float lds[4];
  const int block = blockIdx.x;
  if (block < a.firsts) first_queries<D>(a, block);
  else if (a.whole) largest_rows<256>(a, block - a.firsts, (int)gridDim.x - a.firsts, lds);
  else largest_rows<kWave>(a, block - a.firsts, (int)gridDim.x - a.firsts, lds);
}

// 2^n with 4 < 2^n bound <= 8 for bound = sqrt(ee vv), which |e . v| of the sequence does not pass: |u| is at most bound / 2, since what
// w leaves of 1 is the others' part of delta, so 2^kUp 2^n |u| is at most 2^16, which 65519 rounds to.  (A u that is off
// by more comes out as an infinity, and is done again.)
__device__ __forceinline__ float factor_of(float ee, float vv) {
  const float bound = sqrtf(ee) * sqrtf(vv);
  return bound > 0.f && bound < INFINITY ? ldexpf(1.f, min(ilogbf(7.99f / bound), 100)) : 1.f;
}

// f(0), .. f(N - 1), the numbers as types.
template <typename F, int... I>
__device__ __forceinline__ void for_each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each_of(F f) {
  for_each_of(f, std::make_integer_sequence<int, N>{});
}

constexpr int tile_rows(int d) { return d <= 128 ? 64 : 32; }  // of y
// Whether the steps of a walk overlap (see there): where the sums leave registers for one wavefront a SIMD, which has
// nothing else to hide its waits behind.
constexpr bool overlaps(int d, bool keys) { return keys && d >= 128; }
// Places of tiles in LDS, for the order of the steps.
constexpr int places_of(int d, bool keys) { return !overlaps(d, keys) ? 2 : tile_rows(d) == 64 ? 3 : 4; }
constexpr int lds_of(int d, bool keys) { return places_of(d, keys) * 2 * tile_rows(d) * (d * 2 + 4); }
// Wavefronts a SIMD that the registers are divided for.
constexpr int waves_of(int d, bool keys) { return d <= 64 ? 3 : keys ? 1 : 2; }

// One workgroup's rows of x against all its rows of y, 64 NB rows of x.  KEYS: x = k, v and y = q, e of all the key head's heads;
// else x = q, e and y = k, v.
template <int D, int NB, bool KEYS>
__device__ __forceinline__ void walk(const GradArgs& a, int id, int slots, bool longest_first) {
  constexpr int R = 64 * NB;
  constexpr int TY = tile_rows(D);
  constexpr int KS = (D + 31) / 32, DB = D / 16;
  constexpr int ROWB = D * 2, CH = D / 8, RPI = 1024 / ROWB;
  constexpr int TILE = TY * ROWB;
  constexpr bool OVERLAPS = overlaps(D, KEYS);
  constexpr int GROUPS = TY / 32, PLACES = places_of(D, KEYS);
  constexpr int ROWS = TY / 2, NDMA = ROWS / RPI;  // rows of a tile that a wavefront brings, and its load instructions
  // Unit u of row r of a tile lies at u ^ key(r).  A row read takes unit g of rows 8 (c / 4) + c % 4 (+ 4 b), served lanes
  // 0..3, 12..15, 20..27 first, a transposing one two units of rows 8 g + 0..3 (+ 4), two g at a time: in different banks both (but for D = 16).
  const auto key = [](int r) {
    return 2 * (CH >= 16 ? (r & 3) | (r >> 3 & 1) << 2 : CH == 8 ? (r >> 1 & 1) | (r >> 3 & 1) << 1 : CH == 4 ? r >> 3 & 1 : 0);
  };
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // PLACES of y's two tiles each, and of their rows' lse and delta
  float* rows_of = reinterpret_cast<float*>(smem + PLACES * 2 * TILE);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const unsigned smem_base = (unsigned)(uintptr_t)smem;

  const int per_key = a.heads / a.kv_heads, rep = KEYS ? per_key / a.shares : 1;  // heads over a key head, and of this walk
  Place place;
  if (!find_place(id, KEYS ? a.kv_heads * a.shares : a.heads, a.kv_heads, slots, longest_first, &place)) return;
  const Sequences in{a.starts, a.rows, a.sequences};
  const Block block = longest_first && a.sequences > 1 ? nth_longest<R>(in, place.slot) : find_block<R>(in, slots - 1 - place.slot);
  if (block.length == 0) return;
  const int L = block.length;
  // early keys have the most queries, late queries the most keys
  const int x0 = (KEYS ? (L - 1) / R - block.block : block.block) * R;
  const int xw0 = x0 + wave * 16 * NB;
  const bool active = xw0 < L;
  const int kv_head = __builtin_amdgcn_readfirstlane(place.head / (KEYS ? a.shares : per_key));
  const int head0 = __builtin_amdgcn_readfirstlane(place.head * rep);
  const int first_tile = KEYS ? x0 / TY : 0;
  const int tiles = (KEYS ? (L - 1) / TY : (min(x0 + R, L) - 1) / TY) + 1 - first_tile;
  const int all = KEYS ? tiles * rep : tiles;
  const _Float16* qp = a.q + (block.first * a.q_row + head0 * a.q_head);
  const _Float16* kp = a.k + (block.first * a.k_row + kv_head * a.k_head);
  const _Float16* vp = a.v + (block.first * a.v_row + kv_head * a.v_head);
  const _Float16* ep = a.d_out + (block.first * a.heads + head0) * D;
  const int64_t e_row = (int64_t)a.heads * D;
  const float* lse = a.lse + (head0 * a.rows + block.first);
  const float* minus_delta = a.minus_delta + (head0 * a.rows + block.first);

  // ---- x: lane (c, g) holds d = 32 ks + 8 g + 0..7; rows past the end repeat the last one and are not stored
  h8 xa[NB][KS], xb[NB][KS];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int64_t row = min(xw0 + 16 * n + c, L - 1);
    const _Float16* pa = (KEYS ? kp + row * a.k_row : qp + row * a.q_row) + g * 8;
    const _Float16* pb = (KEYS ? vp + row * a.v_row : ep + row * e_row) + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      xa[n][ks] = xb[n][ks] = h8(0);
      if (D >= 32 || g < 2) {
        xa[n][ks] = *reinterpret_cast<const h8*>(pa + ks * 32);
        xb[n][ks] = *reinterpret_cast<const h8*>(pb + ks * 32);
      }
    }
  }

  // ---- y: wavefronts 0 and 1 bring q or k, 2 and 3 e or v; a sequence's last tile repeats its last row
  const bool second = wave >= 2;
  const int first_row = (wave & 1) * ROWS;
  const int64_t pitch = (KEYS ? (second ? e_row : a.q_row) : (second ? a.v_row : a.k_row)) * 2;
  const int64_t head_pitch = KEYS ? (second ? (int64_t)D : a.q_head) * 2 : 0;
  const char* src = (const char*)(KEYS ? (second ? ep : qp) : (second ? vp : kp)) + first_row * pitch;
  const int lrow = lane / CH;
  const unsigned lane_unit = (unsigned)((lane % CH) ^ key(lrow) ^ key(first_row)) << 4;
  const unsigned lane_row = (unsigned)lrow * (unsigned)pitch;
  auto issue_tile = [&](int h, int t, int place_of) {
    const unsigned dst = smem_base + (unsigned)((place_of * 2 + (second ? 1 : 0)) * TILE + first_row * ROWB);
    const char* base = src + h * head_pitch + (int64_t)t * TY * pitch;
    const int rest = L - 1 - t * TY - first_row;  // the last row of this wavefront's
    if (rest >= ROWS - 1) {
#pragma unroll
      for (int j = 0; j < NDMA; ++j) {
        load_lds16(base, (lane_unit ^ ((unsigned)key(j * RPI) << 4)) + lane_row, dst + j * 1024);
        base += RPI * pitch;
      }
    } else {
      base += (int64_t)min(rest, 0) * pitch;  // of rows behind the end, row 0 is the sequence's last
      const int last = max(rest, 0);
#pragma unroll
      for (int j = 0; j < NDMA; ++j)
        load_lds16(base, (unsigned)min(j * RPI + lrow, last) * (unsigned)pitch + (lane_unit ^ ((unsigned)key(j * RPI) << 4)),
                   dst + j * 1024);
    }
    if (KEYS && (wave & 1) == 0 && lane < TY) {  // the rows' lse and -delta, too
      const float* from = (second ? minus_delta : lse) + h * a.rows + (int64_t)t * TY;
      load_lds4(from, (unsigned)min(lane, L - 1 - t * TY) * 4u,
                smem_base + (unsigned)(PLACES * 2 * TILE + (place_of * 2 + (second ? 1 : 0)) * TY * 4));
    }
  };

  // ---- the factor that keeps u in fp16's range, by the largest rows of this sequence and key head: one for all rows where rows
  // are summed over, each row's own otherwise
  const float most_v = a.v_squares[kv_head * a.rows + block.first];
  float x_lse[NB], x_less[NB], factor[NB];  // of row c of block n: lse, less the factor's exponent, and -delta
  if constexpr (KEYS) {
    factor[0] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, factor_of(a.e_squares[(int64_t)kv_head * per_key * a.rows + block.first], most_v))));
  } else {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int row = min(xw0 + 16 * n + c, L - 1);
      float ee = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) ee = fmaf((float)xb[n][ks][i], (float)xb[n][ks][i], ee);
      const LanePair pair = row_swap(half_sum(ee));
      factor[n] = factor_of(pair.a + pair.b, most_v);
      x_lse[n] = lse[row] - (float)ilogbf(factor[n]);
      x_less[n] = minus_delta[row];
    }
  }
  // ---- this lane's LDS addresses inside a tile: unit g of its row for the row reads, unit (c / 2) % 2 of its row for the
  // transposing ones.  Another k-slice or 16-column block is another unit, whose bits an xor sets, since the keys are xor'ed too.
  const int k_row = 8 * (c >> 2) + (c & 3), v_row = 8 * g + (c >> 2);
  const unsigned k_base = (unsigned)(k_row * ROWB + (((D >= 32 ? g : g & 1) ^ key(k_row)) << 4));
  const unsigned v_base = (unsigned)(v_row * ROWB + ((((c & 3) >> 1) ^ key(v_row)) << 4) + (c & 1) * 8);
  const float to_exp2 = a.scale * 1.4426950408889634f;

  f4 sa[NB][DB], sb[KEYS ? NB : 1][KEYS ? DB : 1];  // sums of u times q or k, and of w times e: d = 16 i + 4 g + 0..3 of row c
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      sa[n][i] = f4(0.f);
      if constexpr (KEYS) sb[n][i] = f4(0.f);
    }

  // y goes by in groups of 32 rows.  Without overlap a step is the scores and e . v of a group, its w and u, and the sums over
  // it; the SIMD's other wavefronts are at another of these.  With overlap it is w and u of one group, the scores and e . v of the
  // next and the sums over the one in front, which do not wait for each other; the LDS reads of each chunk of some 8 matrix
  // instructions are issued in front of the one before it, and a part of the vector instructions goes beside each.
  constexpr int C = KS < 2 ? KS : 2, NQ = 2 * KS / C;                        // score chunks: C k-slices of a 16-row block
  constexpr int CI = DB < (KEYS ? 1 : 2) ? DB : KEYS ? 1 : 2, NS = DB / CI;  // sum chunks: CI 16-column blocks
  constexpr int UNITS = 2 * NB;                                              // of four rows' w and u each
  struct Scores {
    f4 s[NB][2], p[NB][2], lse[2];
  };
  struct Weights {
    h8 w[NB], u[NB];
  };
  struct Rows {
    h8 a[C], b[C];
    f4 less;
  };
  struct Columns {
    h8 a[CI], b[KEYS ? CI : 1];
  };
  auto read_tr = [](unsigned at) { return lds_read_tr16((const char*)(uintptr_t)at); };
  auto read_rows = [&](auto chunk, Rows& to, Scores& next, unsigned at, const float* stat) {
    constexpr int b = decltype(chunk)::value / (KS / C), first = decltype(chunk)::value % (KS / C) * C;
    if constexpr (KEYS && first == 0) {
      to.less = *reinterpret_cast<const f4*>(stat + TY + 8 * g + 4 * b);
      if constexpr (OVERLAPS) next.lse[b] = *reinterpret_cast<const f4*>(stat + 8 * g + 4 * b);
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int ks = first + j;
      const unsigned from = ((at + k_base) ^ (ks << 6)) + b * 4 * ROWB;
      to.a[j] = lds_read16(from);
      to.b[j] = lds_read16(from + TILE);
      if (D < 32 && g >= 2) to.a[j] = to.b[j] = h8(0);
    }
  };
  auto scores = [&](auto chunk, const Rows& y, Scores& to) {  // s: q . k, p: e . v - delta
    constexpr int b = decltype(chunk)::value / (KS / C), first = decltype(chunk)::value % (KS / C) * C;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int ks = first + j;
        to.s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y.a[j], xa[n][ks], ks == 0 ? f4(0.f) : to.s[n][b], 0, 0, 0);
        to.p[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y.b[j], xb[n][ks], ks > 0 ? to.p[n][b] : KEYS ? y.less : f4(x_less[n]), 0, 0, 0);
      }
  };
  auto read_columns = [&](auto chunk, Columns& to, unsigned at) {
#pragma unroll
    for (int j = 0; j < CI; ++j) {
      const int i = decltype(chunk)::value * CI + j;
      const unsigned from = (at + v_base) ^ (i << 5);
      const h4 lo = read_tr(from), hi = read_tr(from + 4 * ROWB);
      to.a[j] = h8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if constexpr (KEYS) {
        const h4 lo2 = read_tr(from + TILE), hi2 = read_tr(from + TILE + 4 * ROWB);
        to.b[j] = h8{lo2[0], lo2[1], lo2[2], lo2[3], hi2[0], hi2[1], hi2[2], hi2[3]};
      }
    }
  };
  auto sums = [&](auto chunk, const Columns& y, const Weights& by) {
#pragma unroll
    for (int j = 0; j < CI; ++j)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int i = decltype(chunk)::value * CI + j;
        sa[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y.a[j], by.u[n], sa[n][i], 0, 0, 0);
        if constexpr (KEYS) sb[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y.b[j], by.w[n], sb[n][i], 0, 0, 0);
      }
  };
  auto weights = [&](int unit, const Scores& from, Weights& to, const float* stat = nullptr) {
    const int n = unit % NB, b = unit / NB;
    f4 lse;
    if constexpr (KEYS) lse = OVERLAPS ? from.lse[b] : *reinterpret_cast<const f4*>(stat + 8 * g + 4 * b);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float w = __builtin_amdgcn_exp2f(fmaf(from.s[n][b][r], to_exp2, -(KEYS ? lse[r] : x_lse[n])));
      if constexpr (KEYS) to.w[n][4 * b + r] = (_Float16)w;
      to.u[n][4 * b + r] = (_Float16)((KEYS ? w * factor[0] : w) * from.p[n][b][r]);
    }
  };
  auto some_scores = [&](auto block, Scores& to, unsigned at, const float* stat) {
    for_each_of<NQ / 2>([&](auto q) {
      constexpr std::integral_constant<int, decltype(block)::value * (NQ / 2) + decltype(q)::value> chunk{};
      Rows rows;
      read_rows(chunk, rows, to, at, stat);
      if constexpr (decltype(q)::value > 0) rows.less = f4(0.f);
      scores(chunk, rows, to);
    });
  };
  auto all_sums = [&](const Weights& by, unsigned at) {
    for_each_of<NS>([&](auto i) {
      Columns columns;
      read_columns(i, columns, at);
      sums(i, columns, by);
    });
  };
  auto hide = [&](Scores& now, int y0, int from, int to) {  // blocks from .. to - 1
    const int x_last = xw0 + 16 * NB - 1;
    if (KEYS ? y0 < x_last || y0 + 31 >= L : y0 + 31 > xw0) {  // the diagonal passes through, or the end, or nothing is seen
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int b = from; b < to; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int y = y0 + 8 * g + 4 * b + r, x = xw0 + 16 * n + c;
            now.s[n][b][r] = (KEYS ? x <= y && y < L : y <= x) ? now.s[n][b][r] : -INFINITY;
            if ((KEYS ? y : x) == 0) now.p[n][b][r] *= 0.f;  // a sequence's first query has one key, and no gradient
          }
    }
  };
  auto step = [&](Scores& now, Weights& made, int y0, Scores& next, unsigned next_at, const float* next_stat,
                  const Weights& last, unsigned last_at) {
    Rows rows[2];
    Columns columns[2];
    read_rows(std::integral_constant<int, 0>{}, rows[0], next, next_at, next_stat);
    hide(now, y0, 0, 2);
    constexpr int NC = NQ + NS;
    // unit u of the weights goes beside chunk u (NC + 1) / UNITS - 1, the first in front of all
    const auto some_weights = [&](int chunk) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
        if (u * (NC + 1) / UNITS == chunk) weights(u, now, made);
    };
    some_weights(0);
    for_each_of<NQ>([&](auto q) {
      constexpr int i = decltype(q)::value;
      if constexpr (i + 1 < NQ) read_rows(std::integral_constant<int, i + 1>{}, rows[(i + 1) & 1], next, next_at, next_stat);
      else read_columns(std::integral_constant<int, 0>{}, columns[0], last_at);
      scores(q, rows[i & 1], next);
      some_weights(i + 1);
    });
    for_each_of<NS>([&](auto q) {
      constexpr int i = decltype(q)::value;
      if constexpr (i + 1 < NS) read_columns(std::integral_constant<int, i + 1>{}, columns[(i + 1) & 1], last_at);
      sums(q, columns[i & 1], last);
      some_weights(NQ + i + 1);
    });
  };

  // Tile `it` is in place it % PLACES.  Without overlap the barrier in front of it says that it has landed, and that all are
  // done with tile it - 1, whose place tile it + 1 takes.  With overlap the barrier of tile `it`, in front of its last step, says
  // that tile it + 1 has landed, and that all are done with the tile whose place tile it + 2 takes (two groups a tile:
  // it - 1, last read by the step of the first half; one: it - 2).
  struct At {
    int h, t, place;
  };
  auto following = [&](At at) {
    At to = {at.h, at.t + 1, at.place + 1 == PLACES ? 0 : at.place + 1};
    if (to.t == first_tile + tiles) to.t = first_tile, ++to.h;
    return to;
  };
  auto tile_at = [&](const At& at) { return smem_base + (unsigned)(at.place * 2 * TILE); };
  auto stat_at = [&](const At& at) { return rows_of + at.place * 2 * TY; };
  auto arrive = [] { asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  At now = {0, first_tile, 0}, next = following(now), last = now;
  issue_tile(now.h, now.t, now.place);
  if constexpr (OVERLAPS) arrive();
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int n = 0; n < NB; ++n) {  // they have landed too: no wait at their uses, which would be one for the tiles
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(xa[n][ks]), "+v"(xb[n][ks]));
    if constexpr (!KEYS) asm volatile("" : "+v"(x_lse[n]), "+v"(x_less[n]));
  }
  if (OVERLAPS && all > 1) issue_tile(next.h, next.t, next.place);
  Scores even, odd;
  Weights front, back;  // of the group in front, by turns
#pragma unroll
  for (int n = 0; n < NB; ++n) front.w[n] = front.u[n] = back.w[n] = back.u[n] = h8(0);
  if (OVERLAPS && active) {
    some_scores(std::integral_constant<int, 0>{}, even, tile_at(now), stat_at(now));
    some_scores(std::integral_constant<int, 1>{}, even, tile_at(now), stat_at(now));
  }
  auto barrier = [&](int it) {
    if (it + 1 >= all) return;
    arrive();
    if (it + 2 < all) {
      const At then = following(next);
      issue_tile(then.h, then.t, then.place);
    }
  };
  if constexpr (!OVERLAPS) {
    for (int it = 0; it < all; ++it) {
      arrive();
      if (it + 1 < all) issue_tile(next.h, next.t, next.place);
      // the groups that this wavefront's rows see something of; one body, for the sums stay in place then
      const int seen = (KEYS ? xw0 : xw0 + 16 * NB - 1) - now.t * TY;
      const int begin = KEYS && seen > 0 ? seen >> 5 : 0, end = KEYS ? GROUPS : seen < 0 ? 0 : min(GROUPS, (seen >> 5) + 1);
#pragma unroll 1
      for (int group = active ? begin : end; group < end; ++group) {
        const unsigned at = tile_at(now) + group * 32 * ROWB;
        const float* stat = stat_at(now) + group * 32;
        for_each_of<2>([&](auto b) {  // 16 rows after the other: fewer registers at a time
          some_scores(b, even, at, stat);
          hide(even, now.t * TY + 32 * group, b, b + 1);
#pragma unroll
          for (int n = 0; n < NB; ++n) weights(b * NB + n, even, front, stat);
        });
        all_sums(front, at);
      }
      now = next;
      next = following(next);
    }
  } else if constexpr (GROUPS == 2) {
    for (int it = 0; it < all; ++it) {
      const unsigned at = tile_at(now), half = at + 32 * ROWB;
      if (active) step(even, front, now.t * TY, odd, half, stat_at(now) + 32, back, tile_at(last) + 32 * ROWB);
      barrier(it);
      if (active) step(odd, back, now.t * TY + 32, even, tile_at(next), stat_at(next), front, at);
      last = now;
      now = next;
      next = following(next);
    }
    if (active) all_sums(back, tile_at(last) + 32 * ROWB);
  } else {
    for (int it = 0; it < all; it += 2) {
      barrier(it);
      if (active) step(even, front, now.t * TY, odd, tile_at(next), stat_at(next), back, tile_at(last));
      last = now;
      now = next;
      next = following(next);
      if (it + 1 == all) {
        back = front;
        break;
      }
      barrier(it + 1);
      if (active) step(odd, back, now.t * TY, even, tile_at(next), stat_at(next), front, tile_at(last));
      last = now;
      now = next;
      next = following(next);
    }
    if (active) all_sums(back, tile_at(last));
  }
  if (!active) return;

  // ---- results.  An infinity or a NaN among them: an input is none, or a row is marked, or something has left fp16's
  // range on the way, and a hidden row may have spoilt others with its weight of 0.  Once more, row by row of y, in fp32.
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int x = xw0 + 16 * n + c;
    const float f = KEYS ? factor[0] : factor[n], by_a = a.scale * ldexpf(1.f, -kUp) / f, by_b = ldexpf(1.f, -kUp);
    f4 nones = f4(0.f);
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        nones[r] = fmaf(sa[n][i][r], 0.f, nones[r]);
        if constexpr (KEYS) nones[r] = fmaf(sb[n][i][r], 0.f, nones[r]);
      }
    const float none = (nones[0] + nones[1]) + (nones[2] + nones[3]);
    const int64_t row = block.first + x;
    const int64_t place_a = KEYS ? (row * a.kv_heads + kv_head) * D : (row * a.heads + head0) * D;
    // four numbers of the results, or of this walk's part of them
    const auto store = [&](int at, f4 ra, f4 rb) {
      if (x >= L) return;
      if (KEYS && a.shares > 1) {
        float* to = a.parts + (int64_t)(place.head % a.shares) * 2 * a.rows * a.kv_heads * D + place_a + at;
        *reinterpret_cast<f4*>(to) = ra;
        *reinterpret_cast<f4*>(to + a.rows * a.kv_heads * D) = rb;
        return;
      }
      *reinterpret_cast<h4*>((KEYS ? a.dk : a.dq) + place_a + at) = __builtin_convertvector(ra, h4);
      if constexpr (KEYS) *reinterpret_cast<h4*>(a.dv + place_a + at) = __builtin_convertvector(rb, h4);
    };
    if (!__any(none != 0.f && x < L)) {
      if (DB == 1 || (KEYS && a.shares > 1)) {
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          if constexpr (KEYS) store(16 * i + 4 * g, sa[n][i] * by_a, sb[n][i] * by_b);
          else store(16 * i + 4 * g, sa[n][i] * by_a, f4(0.f));
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i + 1 < DB; i += 2) {
        store_blocks((KEYS ? a.dk : a.dq) + place_a + 16 * i, g, __builtin_convertvector(sa[n][i] * by_a, h4),
                     __builtin_convertvector(sa[n][i + 1] * by_a, h4), x < L);
        if constexpr (KEYS)
          store_blocks(a.dv + place_a + 16 * i, g, __builtin_convertvector(sb[n][i] * by_b, h4),
                       __builtin_convertvector(sb[n][i + 1] * by_b, h4), x < L);
      }
      continue;
    }
    float va[KS][8], vb[KEYS ? KS : 1][8];  // d = 32 ks + 8 g + 0..7
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        va[ks][i] = 0.f;
        if constexpr (KEYS) vb[ks][i] = 0.f;
      }
    const int y_first = KEYS ? xw0 + 16 * n : 0, y_last = KEYS ? L - 1 : min(xw0 + 16 * n + 15, L - 1);
    for (int head = 0; head < (KEYS ? rep : 1); ++head)
      for (int y = y_first; y <= y_last; ++y) {
#pragma clang fp contract(off)
        const _Float16* ya = (KEYS ? qp + head * a.q_head + y * a.q_row : kp + y * a.k_row) + g * 8;
        const _Float16* yb = (KEYS ? ep + head * D + y * e_row : vp + y * a.v_row) + g * 8;
        const int query = KEYS ? y : min(x, L - 1);
        const float2 stat = a.stats[(int64_t)(head0 + head) * a.rows + block.first + query];
        const float less = minus_delta[head * a.rows + query];
        float s = 0.f, p = 0.f;  // the score as the forward pass forms it key by key
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (D < 32 && g >= 2) continue;
          const h8 fa = *reinterpret_cast<const h8*>(ya + ks * 32), fb = *reinterpret_cast<const h8*>(yb + ks * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            s = fmaf((float)xa[n][ks][i], (float)fa[i], s);
            p = fmaf((float)xb[n][ks][i], (float)fb[i], p);
          }
        }
        const LanePair sp = row_swap(half_sum(s)), pp = row_swap(half_sum(p));
        s = sp.a + sp.b;
        p = pp.a + pp.b;
        const float w = stat.y > 0.f ? __builtin_amdgcn_exp2f(fmaf(s, to_exp2, -stat.x)) * stat.y
                                     : __expf(s * a.scale - stat.x) * -stat.y;
        const float u = w * ((p + less) * (query == 0 ? 0.f : 1.f));
        const bool seen = KEYS ? x <= y : y <= x;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (D < 32 && g >= 2) continue;
          const h8 fa = *reinterpret_cast<const h8*>(ya + ks * 32), fb = *reinterpret_cast<const h8*>(yb + ks * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float more = fmaf(u, (float)fa[i], va[ks][i]);
            va[ks][i] = seen ? more : va[ks][i];
            if constexpr (KEYS) {
              const float more_b = fmaf(w, (float)fb[i], vb[ks][i]);
              vb[ks][i] = seen ? more_b : vb[ks][i];
            }
          }
        }
      }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f4 ra, rb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ra[i] = va[ks][4 * half + i] * a.scale;
          rb[i] = KEYS ? vb[KEYS ? ks : 0][4 * half + i] : 0.f;
        }
        if (D >= 32 || g < 2) store(ks * 32 + g * 8 + 4 * half, ra, rb);
      }
  }
}

// The parts of dk and dv, added in the order of the heads.
template <int D>
__global__ __launch_bounds__(256) void packed_join_kernel(GradArgs a) {
  const int64_t all = a.rows * a.kv_heads * D, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const int64_t row = at / (a.kv_heads * D);
  if (at >= all || row < a.starts[0] || row >= a.starts[a.sequences]) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    f4 sum = *reinterpret_cast<const f4*>(a.parts + which * all + at);
    for (int i = 1; i < a.shares; ++i) sum += *reinterpret_cast<const f4*>(a.parts + (2 * i + which) * all + at);
    *reinterpret_cast<h4*>((which ? a.dv : a.dk) + at) = __builtin_convertvector(sum, h4);
  }
}

template <int D, int NB, bool KEYS>
__global__ __launch_bounds__(256, waves_of(D, KEYS)) void packed_grad_kernel(GradArgs a) {
  walk<D, NB, KEYS>(a, (int)(blockIdx.y * kGridRow + blockIdx.x), a.deal[KEYS].slots, a.deal[KEYS].longest_first);
}

// Both walks in one launch: which workgroups start last decides when a launch ends, and one end is less than two.  Eight ids
// of the one, then eight of the other, as far as both go: the ids' place modulo 8 says which XCD has them.
template <int D, int NB>
__global__ __launch_bounds__(256, waves_of(D, true)) void packed_grads_kernel(GradArgs a) {
  const int id = (int)(blockIdx.y * kGridRow + blockIdx.x), keys = a.deal[1].grid, queries = a.deal[0].grid;
  const int both = 2 * min(keys, queries);
  const bool key = id < both ? (id >> 3 & 1) == 0 : keys > queries;
  const int own = id < both ? (id >> 4) * 8 + (id & 7) : id - both / 2;
  if (key) walk<D, NB, true>(a, own, a.deal[1].slots, a.deal[1].longest_first);
  else walk<D, NB, false>(a, own, a.deal[0].slots, a.deal[0].longest_first);
}

// How many slots of 64 NB rows, in which order, and the workgroups, a multiple of 8.
template <int NB>
bool deal_slots(const GradArgs& a, int heads, SlotDeal* deal) {
  const int64_t slots = a.rows / (64 * NB) + a.sequences, blocks = slots * heads;
  if (blocks > (1ll << 30) - kGridRow) {
    set_error("flash_attn_packed_backward: %lld rows in %d sequences of %d heads exceed the grid", (long long)a.rows,
              a.sequences, heads);
    return false;
  }
  const bool longest_first = a.sequences <= kMany * kWave && slots <= 512 && blocks <= 5120 && a.rows >= 128ll * a.sequences;
  const int64_t grid = longest_first ? (slots + 7) / 8 * 8 * heads : (blocks + 7) / 8 * 8;
  *deal = {(int)slots, (int)grid, longest_first};
  return true;
}

template <typename K>
int launch(K kernel, const GradArgs& a, int64_t grid, int lds, bool* attr_done, hipStream_t st) {
  if (!*attr_done) {  // idempotent; a race only repeats the call
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("hipFuncSetAttribute(%d bytes LDS): %s", lds, hipGetErrorString(e));
      return -4;
    }
    *attr_done = true;
  }
  const dim3 dims((unsigned)(grid < kGridRow ? grid : kGridRow), (unsigned)((grid + kGridRow - 1) / kGridRow));
  hipLaunchKernelGGL(kernel, dims, dim3(256), lds, st, a);
  return 0;
}

// Where the blocks of keys would not fill the GPU, the heads that share a key head are divided, into no more parts than needed.
template <int NB>
int shares_of(int64_t rows, int64_t sequences, int heads, int kv_heads) {
  const int64_t blocks = (rows / (64 * NB) + sequences) * kv_heads;
  const int rep = heads / kv_heads;
  int shares = 1;
  while (shares < rep && (rep % shares != 0 || blocks * shares < 512)) ++shares;
  return shares;
}
template <int D>
constexpr int blocks_of() {  // of 16 rows a wavefront
  return D <= 128 ? 2 : 1;
}

template <int D>
int launch_d(GradArgs a, hipStream_t st) {
  constexpr int NB = blocks_of<D>();
  constexpr int BLOCK = 256 / (D / 8) > 64 ? 256 / (D / 8) : 64;
  const int64_t items = (a.rows + BLOCK - 1) / BLOCK * a.heads;
  if (!deal_slots<NB>(a, a.heads, &a.deal[0]) || !deal_slots<NB>(a, a.kv_heads * a.shares, &a.deal[1])) return -2;
  hipLaunchKernelGGL((packed_sums_kernel<D>), dim3((unsigned)(items < kSums ? items : kSums)), dim3(256), 0, st, a);
  const int64_t firsts = ((int64_t)a.sequences * a.heads + 3) / 4, keys = (int64_t)a.sequences * a.kv_heads;
  a.firsts = (int)(firsts < kSequenceBlocks ? firsts : kSequenceBlocks);
  // us, the launch, a workgroup / a wavefront for each sequence and key head: 1 x 8192 tokens, 12 heads 5.5 / 12.9, 16 x 1024, 32
  // over 8 5.7 / 8.5, 48 x 300, 12 5.5 / 4.3, 400 x 40 14.1 / 10.2, 10000 x 3, 32 over 8 281 / 197
  a.whole = a.rows >= 512ll * a.sequences;
  const int64_t largest = a.whole ? keys : (keys + 3) / 4;
  hipLaunchKernelGGL((packed_sequences_kernel<D>), dim3((unsigned)(a.firsts + (largest < kSequenceBlocks ? largest : kSequenceBlocks))),
                     dim3(256), 0, st, a);
  static bool done[2];
  int rc = 0;
  if constexpr (D <= 64) {
    if (!a.dq) a.deal[0].grid = 0;
    if (!a.dk) a.deal[1].grid = 0;
    rc = launch(packed_grads_kernel<D, NB>, a, (int64_t)a.deal[0].grid + a.deal[1].grid, lds_of(D, true), &done[0], st);
  } else {
    if (a.dk) rc = launch(packed_grad_kernel<D, NB, true>, a, a.deal[1].grid, lds_of(D, true), &done[1], st);
    if (a.dq && !rc) rc = launch(packed_grad_kernel<D, NB, false>, a, a.deal[0].grid, lds_of(D, false), &done[0], st);
  }
  if (a.dk && a.shares > 1 && !rc)
    hipLaunchKernelGGL((packed_join_kernel<D>), dim3((unsigned)((a.rows * a.kv_heads * D + 1023) / 1024)), dim3(256), 0, st, a);
  return rc;
}

}  // namespace

// lse and -delta, e's and v's squares, and the parts of dk and dv.
static size_t row_bytes(int64_t rows, int64_t heads, int64_t kv_heads) {
  return ((size_t)rows * (size_t)(3 * heads + kv_heads) * sizeof(float) + 255) / 256 * 256;
}
size_t packed_attn_grad_bytes(int64_t rows, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t d) {
  const int shares = d <= 128 ? shares_of<blocks_of<128>()>(rows, sequences, (int)heads, (int)kv_heads)
                              : shares_of<blocks_of<256>()>(rows, sequences, (int)heads, (int)kv_heads);
  return row_bytes(rows, heads, kv_heads) + (shares > 1 ? (size_t)shares * 2 * (size_t)(rows * kv_heads * d) * sizeof(float) : 0);
}

int launch_flash_attn_packed_backward(const PackedAttention& p, const PackedGradients& d, int head_size, void* workspace,
                                      hipStream_t st) {
  GradArgs a;
  a.q = (const _Float16*)p.q;
  a.k = (const _Float16*)p.k;
  a.v = (const _Float16*)p.v;
  a.out = (const _Float16*)p.out;
  a.remainder = (const _Float16*)p.remainder;
  a.d_out = (const _Float16*)d.d_out;
  a.dq = (_Float16*)d.dq;
  a.dk = (_Float16*)d.dk;
  a.dv = (_Float16*)d.dv;
  a.stats = (const float2*)p.stats;
  a.lse = (float*)workspace;
  a.minus_delta = a.lse + p.rows * p.heads;
  a.e_squares = a.minus_delta + p.rows * p.heads;
  a.v_squares = a.e_squares + p.rows * p.heads;
  a.parts = (float*)((char*)workspace + row_bytes(p.rows, p.heads, p.kv_heads));
  a.shares = head_size <= 128 ? shares_of<blocks_of<128>()>(p.rows, p.sequences, (int)p.heads, (int)p.kv_heads)
                              : shares_of<blocks_of<256>()>(p.rows, p.sequences, (int)p.heads, (int)p.kv_heads);
  a.starts = p.starts;
  a.rows = p.rows;
  a.sequences = (int)p.sequences;
  a.heads = (int)p.heads;
  a.kv_heads = (int)p.kv_heads;
  a.q_row = p.q_row, a.q_head = p.q_head, a.k_row = p.k_row, a.k_head = p.k_head, a.v_row = p.v_row, a.v_head = p.v_head;
  a.scale = p.scale;
  switch (head_size) {
    case 16: return launch_d<16>(a, st);
    case 32: return launch_d<32>(a, st);
    case 64: return launch_d<64>(a, st);
    case 128: return launch_d<128>(a, st);
    case 256: return launch_d<256>(a, st);
  }
  set_error("flash_attn_packed_backward: head size %d (16, 32, 64, 128 and 256 are supported)", head_size);
  return -2;
}

}  // namespace gptmi
