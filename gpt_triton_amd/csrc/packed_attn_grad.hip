// Gradients of causal attention over packed sequences (packed_attn.hip).  With t = scale, w_ij = softmax_j(t q_i . k_j)
// over the keys j <= i of i's sequence, and e_i the gradient of the output o_i = sum_j w_ij v_j:
//   delta_i = sum_j w_ij (e_i . v_j) = e_i . o_i,   u_ij = w_ij (e_i . v_j - delta_i)
//   dq_i = t sum_j u_ij k_j,   dk_j = t sum_i u_ij q_i,   dv_j = sum_i w_ij e_i
// over the queries i >= j of all the heads that share a key head.  The weights are formed again from q, k and the
// statistic that the forward pass keeps of each row, so nothing of the size of the scores goes to memory.
//
// Three launches: row sums (delta, and the largest rows of e and v); dk and dv, a workgroup for a block of keys, which walks
// over the queries; dq, a workgroup for a block of queries, which walks over the keys.  So each sum is formed by one
// workgroup in one order, without atomics, at the cost of forming w and u twice: 7 products instead of 5.
//
// Both walks are one kernel: rows x in registers (k and v, or q and e), rows y that pass through LDS (q and e, or k and v).
// The products are Y . X^T with v_mfma_f32_16x16x32_f16, whose result lane (c, g), c = lane % 16, g = lane / 16, has
// row c of x and four rows of y; rows 4 g + r of the two 16-row blocks b of a group of 32 are y's rows 8 g + 4 b + r, so
// that w and u, rounded to fp16, are the second operand of the sums over y as they stand.
#include <type_traits>

#include "common.h"
#include "launch.h"
#include "packed_attn.h"

namespace gptmi {
namespace {

// The weights are formed as 2^kUp w and u as 2^kUp f u, f a power of two: fp16 numbers of the size of one that stay
// normal numbers down to 2^-28 of it.
constexpr int kUp = 14;
constexpr int kSums = 512;  // workgroups of the row sums at most

struct GradArgs {
  const _Float16 *q, *k, *v, *out, *d_out;
  _Float16 *dq, *dk, *dv;  // dense; dq, or dk and dv, may be nullptr
  const float2* stats;     // [heads][T], the forward pass's
  float *lse, *delta;      // [heads][T]: w = 2^(s t log2(e) - lse - kUp); a NaN: see packed_sums_kernel
  float2* most;            // the largest e . e and v . v of each workgroup of the row sums
  int mosts;
  const int64_t* starts;
  int64_t rows;  // T
  int sequences, heads, kv_heads, slots, longest_first;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // pitches in elements
  float scale;
};

// ---------------------------------------------------------------------------
// delta, lse and the largest rows.  Rows that belong to no sequence get gradients of 0 here.
// A row whose statistic is of scores key by key (infinities and NaN, scores of some thousands) gets lse = NaN: what meets it
// comes out as NaN, and is done again with the statistic itself.
// ---------------------------------------------------------------------------
template <int D>
__global__ __launch_bounds__(256) void packed_sums_kernel(GradArgs a) {
  constexpr int LPR = D / 8;          // lanes a row
  constexpr int RPP = 256 / LPR;      // rows a pass
  constexpr int BLOCK = RPP > 64 ? RPP : 64;
  __shared__ float2 largest[4];
  const int tid = threadIdx.x, in_row = tid % LPR, row_of = tid / LPR;
  const int64_t from = a.starts[0], to = a.starts[a.sequences];
  const int64_t items = (a.rows + BLOCK - 1) / BLOCK * a.heads;
  float most_e = 0.f, most_v = 0.f;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t block = item / a.heads;
    const int head = (int)(item - block * a.heads);
#pragma unroll
    for (int pass = 0; pass < BLOCK / RPP; ++pass) {
      const int64_t row = block * BLOCK + pass * RPP + row_of;
      if (row >= a.rows) break;
      const int64_t at = (row * a.heads + head) * D + in_row * 8, kv_at = (row * a.kv_heads + head) * D + in_row * 8;
      if (row < from || row >= to) {
        if (a.dq) *reinterpret_cast<h8*>(a.dq + at) = h8(0);
        if (a.dk && head < a.kv_heads) *reinterpret_cast<h8*>(a.dk + kv_at) = *reinterpret_cast<h8*>(a.dv + kv_at) = h8(0);
        continue;
      }
      const h8 e = *reinterpret_cast<const h8*>(a.d_out + at), o = *reinterpret_cast<const h8*>(a.out + at);
      float dot = 0.f, ee = 0.f, vv = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dot = fmaf((float)e[i], (float)o[i], dot);
        ee = fmaf((float)e[i], (float)e[i], ee);
      }
      if (head < a.kv_heads) {
        const h8 v = *reinterpret_cast<const h8*>(a.v + row * a.v_row + head * a.v_head + in_row * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i) vv = fmaf((float)v[i], (float)v[i], vv);
      }
#pragma unroll
      for (int step = 1; step < LPR; step *= 2) {
        dot += __shfl_xor(dot, step);
        ee += __shfl_xor(ee, step);
        vv += __shfl_xor(vv, step);
      }
      // rows with an infinity or a NaN spoil only what they are part of
      if (ee < INFINITY) most_e = fmaxf(most_e, ee);
      if (vv < INFINITY) most_v = fmaxf(most_v, vv);
      if (in_row == 0) {
        const int64_t place = head * a.rows + row;
        const float2 stat = a.stats[place];
        a.lse[place] = stat.x - __builtin_amdgcn_logf(stat.y) - kUp;  // to the base 2; NaN where stat.y < 0
        a.delta[place] = dot;
      }
    }
  }
  most_e = wave_max(most_e);
  most_v = wave_max(most_v);
  if ((tid & 63) == 0) largest[tid >> 6] = {most_e, most_v};
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      most_e = fmaxf(most_e, largest[i].x);
      most_v = fmaxf(most_v, largest[i].y);
    }
    a.most[blockIdx.x] = {most_e, most_v};
  }
}

// 2^n with 4 < 2^n bound <= 8 for bound = sqrt(ee vv), which |e . v| does not pass: |u| is at most bound / 2, since what
// w leaves of 1 is the others' part of delta, so 2^kUp 2^n |u| is at most 2^16, which 65519 rounds to.  (A u that is off
// by more comes out as an infinity, and is done again.)
__device__ __forceinline__ float factor_of(float ee, float vv) {
  const float bound = sqrtf(ee) * sqrtf(vv);
  return bound > 0.f && bound < INFINITY ? ldexpf(1.f, min(ilogbf(7.99f / bound), 100)) : 1.f;
}

// KEYS: x = k, v and y = q, e of all the key head's heads; else x = q, e and y = k, v.  A workgroup has 64 NB rows of x.
template <int D, int NB, bool KEYS>
__global__ __launch_bounds__(256, D <= 64 ? 2 : 1) void packed_grad_kernel(GradArgs a) {
  constexpr int R = 64 * NB;
  constexpr int TY = D <= 128 ? 64 : 32;  // rows of y a tile
  constexpr int KS = (D + 31) / 32, DB = D / 16;
  constexpr int ROWB = D * 2, CH = D / 8, RPI = 1024 / ROWB;
  constexpr int TILE = TY * ROWB;
  constexpr int ROWS = TY / 2, NDMA = ROWS / RPI;  // rows of a tile that a wavefront brings, and its load instructions
  // Unit u of row r of a tile lies at u ^ key(r).  Row reads take one unit of rows 8 i + 0..3 (+ 4 b), i = 0..3,
  // transposing ones two units of rows 8 g + 0..3 (+ 4), two g at a time: in different banks both.
  const auto key = [](int r) {
    return CH >= 16 ? (r >> 4 & 1) | (r & 3) << 1 | (r >> 3 & 1) << 3
           : CH == 8 ? (r >> 4 & 1) | (r >> 1 & 1) << 1 | (r >> 3 & 1) << 2
           : CH == 4 ? (r >> 4 & 1) | (r >> 3 & 1) << 1
                     : r >> 3 & 1;
  };
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // two places each for y's two tiles, and their rows' lse and delta
  float* rows_of = reinterpret_cast<float*>(smem + 4 * TILE);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const unsigned smem_base = (unsigned)(uintptr_t)smem;

  const int rep = a.heads / a.kv_heads;
  Place place;
  if (!find_place((int)(blockIdx.y * kGridRow + blockIdx.x), KEYS ? a.kv_heads : a.heads, a.kv_heads, a.slots,
                  a.longest_first, &place))
    return;
  const Sequences in{a.starts, a.rows, a.sequences};
  const Block block = a.longest_first && a.sequences > 1 ? nth_longest<R>(in, place.slot)
                                                         : find_block<R>(in, a.slots - 1 - place.slot);
  if (block.length == 0) return;
  const int L = block.length;
  // early keys have the most queries, late queries the most keys
  const int x0 = (KEYS ? (L - 1) / R - block.block : block.block) * R;
  const int xw0 = x0 + wave * 16 * NB;
  const bool active = xw0 < L;
  const int kv_head = KEYS ? place.head : place.head / rep;
  const int head0 = KEYS ? place.head * rep : place.head;
  const int first_tile = KEYS ? x0 / TY : 0;
  const int tiles = (KEYS ? (L - 1) / TY : (min(x0 + R, L) - 1) / TY) + 1 - first_tile;
  const int all = KEYS ? tiles * rep : tiles;
  const _Float16* qp = a.q + (block.first * a.q_row + head0 * a.q_head);
  const _Float16* kp = a.k + (block.first * a.k_row + kv_head * a.k_head);
  const _Float16* vp = a.v + (block.first * a.v_row + kv_head * a.v_head);
  const _Float16* ep = a.d_out + (block.first * a.heads + head0) * D;
  const int64_t e_row = (int64_t)a.heads * D;
  const float* lse = a.lse + (head0 * a.rows + block.first);
  const float* delta = a.delta + (head0 * a.rows + block.first);

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
  };

  // ---- the factor that keeps u in fp16's range: one for all rows where rows are summed over, each row's own otherwise
  float most_e = 0.f, most_v = 0.f;
  for (int i = lane; i < a.mosts; i += kWave) {
    const float2 m = a.most[i];
    most_e = fmaxf(most_e, m.x);
    most_v = fmaxf(most_v, m.y);
  }
  most_v = wave_max(most_v);
  float x_lse[NB], x_delta[NB], factor[NB];  // of row c of block n
  if constexpr (KEYS) {
    factor[0] = factor_of(wave_max(most_e), most_v);
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
      x_lse[n] = lse[row];
      x_delta[n] = delta[row] * factor[n];
    }
  }
  // lse of the rows of y's tile in the first TY threads, delta times the factor in the next; rows behind the end weigh 0
  auto stat_of = [&](int h, int t) {
    float x = INFINITY;
    if (KEYS && tid < 2 * TY) {
      const int row = t * TY + tid % TY;
      const float* from = (tid < TY ? lse : delta) + h * a.rows;
      x = from[min(row, L - 1)];
      x = tid >= TY ? x * factor[0] : row < L ? x : INFINITY;
    }
    return x;
  };

  // ---- LDS read offsets of this lane inside a tile
  const int k_row = 8 * (c >> 2) + (c & 3), v_row = 8 * g + (c >> 2);
  constexpr int KV = KS < 4 ? KS : 4, VV = DB < 8 ? DB : 8;
  int k_off[KV], v_off[VV];
#pragma unroll
  for (int ks = 0; ks < KV; ++ks) k_off[ks] = k_row * ROWB + (((4 * ks + (D >= 32 ? g : g & 1)) ^ key(k_row)) << 4);
#pragma unroll
  for (int i = 0; i < VV; ++i) v_off[i] = v_row * ROWB + (((2 * i + ((c & 3) >> 1)) ^ key(v_row)) << 4) + (c & 1) * 8;
  const float to_exp2 = a.scale * 1.4426950408889634f;

  f4 sa[NB][DB], sb[KEYS ? NB : 1][KEYS ? DB : 1];  // sums of u times q or k, and of w times e: d = 16 i + 4 g + 0..3 of row c
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      sa[n][i] = f4(0.f);
      if constexpr (KEYS) sb[n][i] = f4(0.f);
    }

  // 32 rows of y, from row y0 of the sequence, at `at` in LDS.  MASK: the diagonal passes through.
  auto group = [&](auto mask, int y0, const char* at, const float* stat) {
    constexpr bool MASK = decltype(mask)::value;
    f4 s[NB][2], p[NB][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const char* from = at + b * 4 * ROWB + k_off[ks % KV] + (ks / KV) * 256;
        h8 ya = *reinterpret_cast<const h8*>(from), yb = *reinterpret_cast<const h8*>(from + TILE);
        if (D < 32 && g >= 2) ya = yb = h8(0);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ya, xa[n][ks], ks == 0 ? f4(0.f) : s[n][b], 0, 0, 0);
          p[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(yb, xb[n][ks], ks == 0 ? f4(0.f) : p[n][b], 0, 0, 0);
        }
      }
    h8 w[NB], u[NB];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      f4 y_lse, y_delta;
      if constexpr (KEYS) {
        y_lse = *reinterpret_cast<const f4*>(stat + 8 * g + 4 * b);
        y_delta = *reinterpret_cast<const f4*>(stat + TY + 8 * g + 4 * b);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float e = fmaf(s[n][b][r], to_exp2, -(KEYS ? y_lse[r] : x_lse[n]));
          if constexpr (MASK) {
            const int y = y0 + 8 * g + 4 * b + r, x = xw0 + 16 * n + c;
            e = (KEYS ? x <= y : y <= x) ? e : -INFINITY;
          }
          const float weight = __builtin_amdgcn_exp2f(e);
          if constexpr (KEYS) w[n][4 * b + r] = (_Float16)weight;
          u[n][4 * b + r] = (_Float16)(weight * fmaf(p[n][b][r], KEYS ? factor[0] : factor[n], -(KEYS ? y_delta[r] : x_delta[n])));
        }
    }
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const char* from = at + v_off[i % VV] + (i / VV) * 256;
      const h4 lo = lds_read_tr16(from), hi = lds_read_tr16(from + 4 * ROWB);
      const h8 ya = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (int n = 0; n < NB; ++n) sa[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ya, u[n], sa[n][i], 0, 0, 0);
      if constexpr (KEYS) {
        const h4 lo2 = lds_read_tr16(from + TILE), hi2 = lds_read_tr16(from + TILE + 4 * ROWB);
        const h8 yb = {lo2[0], lo2[1], lo2[2], lo2[3], hi2[0], hi2[1], hi2[2], hi2[3]};
#pragma unroll
        for (int n = 0; n < NB; ++n) sb[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(yb, w[n], sb[n][i], 0, 0, 0);
      }
    }
  };

  issue_tile(0, first_tile, 0);
  float stat = stat_of(0, first_tile);
  int h = 0, t = first_tile;  // of tile `it`
  for (int it = 0; it < all; ++it) {
    if (KEYS && tid < 2 * TY) rows_of[(it & 1) * 2 * TY + tid] = stat;
    // what this wavefront requested has landed; behind the barrier that holds for everyone, and the last step's tiles are free
    asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    int next_t = t + 1, next_h = h;
    if (next_t == first_tile + tiles) next_t = first_tile, ++next_h;
    if (it + 1 < all) {
      issue_tile(next_h, next_t, (it + 1) & 1);
      stat = stat_of(next_h, next_t);
    }
    if (active) {
      const char* at = smem + (it & 1) * 2 * TILE;
      const float* stats = rows_of + (it & 1) * 2 * TY;
      const int x_last = xw0 + 16 * NB - 1;
#pragma unroll
      for (int half = 0; half < TY / 32; ++half) {
        const int y0 = t * TY + half * 32;
        const bool none = KEYS ? y0 + 31 < xw0 : y0 > x_last, full = KEYS ? y0 >= x_last : y0 + 31 <= xw0;
        if (none) continue;
        if (full) group(std::false_type{}, y0, at + half * 32 * ROWB, stats + half * 32);
        else group(std::true_type{}, y0, at + half * 32 * ROWB, stats + half * 32);
      }
    }
    t = next_t;
    h = next_h;
  }
  if (!active) return;

  // ---- results.  An infinity or a NaN among them: an input is none, or a row is marked, or something has left fp16's
  // range on the way, and a hidden row may have spoilt others with its weight of 0.  Once more, row by row of y, in fp32.
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int x = xw0 + 16 * n + c;
    const float f = KEYS ? factor[0] : factor[n], by_a = a.scale * ldexpf(1.f, -kUp) / f, by_b = ldexpf(1.f, -kUp);
    float none = 0.f;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        none = fmaf(sa[n][i][r], 0.f, none);
        if constexpr (KEYS) none = fmaf(sb[n][i][r], 0.f, none);
      }
    const int64_t row = block.first + x;
    _Float16* to_a = KEYS ? a.dk + (row * a.kv_heads + kv_head) * D : a.dq + (row * a.heads + head0) * D;
    _Float16* to_b = KEYS ? a.dv + (row * a.kv_heads + kv_head) * D : nullptr;
    if (!__any(none != 0.f && x < L)) {
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        h4 ra, rb;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ra[r] = (_Float16)(sa[n][i][r] * by_a);
          if constexpr (KEYS) rb[r] = (_Float16)(sb[n][i][r] * by_b);
        }
        if (x < L) {
          *reinterpret_cast<h4*>(to_a + 16 * i + 4 * g) = ra;
          if constexpr (KEYS) *reinterpret_cast<h4*>(to_b + 16 * i + 4 * g) = rb;
        }
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
        const float del = delta[head * a.rows + query];
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
        const float u = w * (p - del);
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
    for (int ks = 0; ks < KS; ++ks) {
      h8 ra, rb;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ra[i] = (_Float16)(va[ks][i] * a.scale);
        if constexpr (KEYS) rb[i] = (_Float16)vb[ks][i];
      }
      if (x < L && (D >= 32 || g < 2)) {
        *reinterpret_cast<h8*>(to_a + ks * 32 + g * 8) = ra;
        if constexpr (KEYS) *reinterpret_cast<h8*>(to_b + ks * 32 + g * 8) = rb;
      }
    }
  }
}

template <int D, int NB, bool KEYS>
int launch_as(GradArgs a, hipStream_t st) {
  constexpr int R = 64 * NB, TY = D <= 128 ? 64 : 32, lds = 4 * TY * D * 2 + 4 * TY * 4;
  const int heads = KEYS ? a.kv_heads : a.heads;
  const int64_t slots = a.rows / R + a.sequences, blocks = slots * heads;
  if (blocks > (1ll << 31) - kGridRow) {
    set_error("flash_attn_packed_backward: %lld rows in %d sequences of %d heads exceed the grid", (long long)a.rows,
              a.sequences, heads);
    return -2;
  }
  static bool attr_done = false;  // idempotent; a race only repeats the call
  if (!attr_done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(packed_grad_kernel<D, NB, KEYS>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("hipFuncSetAttribute(%d bytes LDS): %s", lds, hipGetErrorString(e));
      return -4;
    }
    attr_done = true;
  }
  a.slots = (int)slots;
  a.longest_first = a.sequences <= kMany * kWave && slots <= 512 && blocks <= 5120 && a.rows >= 128ll * a.sequences;
  const int64_t grid = a.longest_first ? (slots + 7) / 8 * 8 * heads : blocks;
  const dim3 dims((unsigned)(grid < kGridRow ? grid : kGridRow), (unsigned)((grid + kGridRow - 1) / kGridRow));
  hipLaunchKernelGGL((packed_grad_kernel<D, NB, KEYS>), dims, dim3(256), lds, st, a);
  return 0;
}

template <int D>
int launch_d(GradArgs a, hipStream_t st) {
  constexpr int BLOCK = 256 / (D / 8) > 64 ? 256 / (D / 8) : 64;
  const int64_t items = (a.rows + BLOCK - 1) / BLOCK * a.heads;
  a.mosts = (int)(items < kSums ? items : kSums);
  hipLaunchKernelGGL((packed_sums_kernel<D>), dim3(a.mosts), dim3(256), 0, st, a);
  constexpr int NB = D <= 128 ? 2 : 1;
  int rc = 0;
  if (a.dk) rc = launch_as<D, NB, true>(a, st);
  if (a.dq && !rc) rc = launch_as<D, NB, false>(a, st);
  return rc;
}

}  // namespace

size_t packed_attn_grad_bytes(int64_t rows, int64_t heads) {
  return (size_t)(kSums * sizeof(float2)) + (size_t)rows * (size_t)heads * 2 * sizeof(float);
}

int launch_flash_attn_packed_backward(const PackedAttention& p, const PackedGradients& d, int head_size, void* workspace,
                                      hipStream_t st) {
  GradArgs a;
  a.q = (const _Float16*)p.q;
  a.k = (const _Float16*)p.k;
  a.v = (const _Float16*)p.v;
  a.out = (const _Float16*)p.out;
  a.d_out = (const _Float16*)d.d_out;
  a.dq = (_Float16*)d.dq;
  a.dk = (_Float16*)d.dk;
  a.dv = (_Float16*)d.dv;
  a.stats = (const float2*)p.stats;
  a.most = (float2*)workspace;
  a.lse = (float*)(a.most + kSums);
  a.delta = a.lse + p.rows * p.heads;
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
