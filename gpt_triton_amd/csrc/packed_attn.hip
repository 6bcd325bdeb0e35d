// Causal attention over whole prompts that lie one behind the other without padding, with grouped heads, fp16:
//   out[i][n] = sum_{j <= i, same sequence} w_ij v[j][n / (N / G)],   w_i = softmax_j(scale q[i][n] . k[j][n / (N / G)])
// q [T][N][D], k, v [T][G][D] at row and head pitches of their own (the q, k, v product's rows as they are), out [T][N][D],
// sequence s the rows starts[s] .. starts[s + 1] - 1.
//
// One workgroup = 4 wavefronts = 64 QB queries of one sequence and head, QB blocks of 16 for each wavefront; or, in P = 2
// parts, half as many, two wavefronts for the key tiles of even number and two for the others, whose sums are joined at the
// end.  The products are the transposed ones, S^T = K . Q^T and O^T += V^T . P^T with v_mfma_f32_16x16x32_f16, so that a
// query's scores and sums are in the four lanes (c, g), c = lane % 16 its number in the block, g = lane / 16.  Rows 4 g +
// r of K's 16-row blocks b = 0, 1 are keys 8 g + 4 b + r of a group of 32, which makes a lane's weights the second operand
// of the next product as they stand: keys 8 g .. 8 g + 7.
#include <type_traits>

#include "common.h"
#include "launch.h"

namespace gptmi {
namespace {

constexpr int kKeys = 64;  // keys a tile
constexpr int kGridRow = 1 << 20;  // workgroups a row of the grid: threads of one dimension have to stay below 2^32

struct PackedArgs {
  const _Float16 *q, *k, *v;
  _Float16* out;
  const int64_t* starts;
  int64_t rows;               // T
  int sequences, heads, kv_heads, slots, longest_first;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // pitches in elements
  float scale;
};

// 16 bytes a lane from base + lane_off into LDS at lds_off + 16 lane.  Assembly, so that the compiler does not wait
// for these loads in front of each LDS read; the kernel waits by hand.
__device__ __forceinline__ void load_lds16(const void* base, unsigned lane_off, unsigned lds_off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_off), "v"(lane_off), "s"(base)
               : "memory", "m0");
}

// Without the compiler's quieting of NaNs in front; one makes a NaN of the row, which is looked for at the end.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A mean of finite fp16 values is at most the largest of them, 65504, but its weights as rounded may make up to 2^-11 more
// than 1, and what is above 65519 would be an infinity.
__device__ __forceinline__ float bounded(float x) {
  return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : x;
}

// Slots: sequence s, which starts at row a, has its blocks of R queries from slot a / R + s on, which leaves room for
// every sequence whatever the lengths are (floor(a / R) + floor(len / R) <= floor((a + len) / R)), needs no
// lengths on the host and no pass over them on the GPU.  Slots that are left over hold nothing.
struct Block {
  int64_t first;  // the sequence's first row
  int length;     // rows of it, 0: nothing to do
  int block;      // which R of them
};
template <int R>
__device__ __forceinline__ Block find_block(const PackedArgs& a, int slot) {
  // the last sequence whose first slot is not behind this one: 64 probes at a time
  const int lane = threadIdx.x & 63;
  int low = 0, left = a.sequences;
  while (left > 1) {
    const int step = (left + 63) >> 6, at = low + lane * step;
    bool in = false;
    if (lane * step < left) in = a.starts[at] / R + at <= slot;
    const int n = __popcll(__ballot(in));
    const int skip = (n > 1 ? n - 1 : 0) * step;
    low += skip;
    left = min(step, left - skip);
  }
  low = __builtin_amdgcn_readfirstlane(low);
  // whatever the starts are, rows stay inside [0, T)
  const int64_t begin = a.starts[low], end = a.starts[low + 1];
  const int64_t first = begin < 0 ? 0 : begin < a.rows ? begin : a.rows;
  const int64_t last = end < first ? first : end < a.rows ? end : a.rows;
  const int64_t length = last - first, block = slot - (begin / R + low);
  return {first, block >= 0 && block * R < length ? (int)length : 0, (int)block};
}

// The nth block of all sequences' blocks in the order of their keys, the most first, for up to 64 kMany sequences.
// Where all workgroups run at once or nearly, the last one to start decides when the launch ends.
constexpr int kMany = 4;
template <int R>
__device__ __forceinline__ Block nth_longest(const PackedArgs& a, int nth) {
  const int lane = threadIdx.x & 63;
  int first[kMany], length[kMany], most = 0;  // of sequence lane + 64 i; rows are below 2^31
#pragma unroll
  for (int i = 0; i < kMany; ++i) {
    const int s = lane + i * kWave;
    first[i] = length[i] = 0;
    if (i * kWave >= a.sequences) break;
    if (s < a.sequences) {
      const int64_t begin = a.starts[s], end = a.starts[s + 1];
      const int64_t from = begin < 0 ? 0 : begin < a.rows ? begin : a.rows;
      const int64_t to = end < from ? from : end < a.rows ? end : a.rows;
      first[i] = (int)from;
      length[i] = (int)(to - from);
    }
    most = max(most, length[i]);
  }
  most = __builtin_amdgcn_readfirstlane((int)wave_max((float)((most + R - 1) / R)));  // below 2^24: the host sees to it
  for (int block = most - 1; block >= 0; --block) {
    int all = 0;
#pragma unroll
    for (int i = 0; i < kMany; ++i) {
      if (i * kWave >= a.sequences) break;
      const uint64_t have = __ballot(length[i] > block * R);
      const int n = __popcll(have);
      if (nth >= all && nth < all + n) {  // the (nth - all)th of these
        const bool me = (have >> lane & 1) && __popcll(have & ((1ull << lane) - 1)) == nth - all;
        const int s = __ffsll((unsigned long long)__ballot(me)) - 1;
        return {__builtin_amdgcn_readlane(first[i], s), __builtin_amdgcn_readlane(length[i], s), block};
      }
      all += n;
    }
    nth -= all;
  }
  return {0, 0, 0};
}

template <int D, int QB, int P>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void packed_attn_kernel(PackedArgs a) {
  constexpr int R = 64 * QB / P;       // queries a workgroup
  constexpr int KS = (D + 31) / 32, DB = D / 16;
  constexpr int ROWB = D * 2;          // bytes of a row in LDS
  constexpr int CH = D / 8;            // 16-byte units of it
  constexpr int RPI = 1024 / ROWB;     // rows that a load instruction covers
  constexpr int TILE = kKeys * ROWB;   // bytes of a K (or V) tile
  constexpr int ROWS = 32 * P;         // rows of a tile that a wavefront brings
  constexpr int NDMA = ROWS / RPI;     // in so many load instructions
  // Unit u of K's row r lies at u ^ k_key(r), of V's at u ^ v_key(r).  A read of K takes one unit of rows 8 i + 0..3
  // (+ 4 b), i = 0..3, a transposing read of V two units of rows 8 g + 0..3, two g at a time: the keys put these into
  // different banks. Neither depends on bit 2 or 5 of the row, and both are made of its bits by or, so a sum of rows
  // has the keys' xor.
  const auto k_key = [](int r) {
    return CH >= 16 ? (r & 3) | (r >> 3 & 3) << 2 : CH == 8 ? (r >> 1 & 1) | (r >> 3 & 3) << 1 : (r >> 3 & 3) & (CH - 1);
  };
  const auto v_key = [](int r) {
    return 2 * (CH >= 16 ? (r & 3) | (r >> 3 & 1) << 2 : CH == 8 ? (r >> 1 & 1) | (r >> 3 & 1) << 1 : CH == 4 ? r >> 3 & 1 : 0);
  };
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // of each part: two places for K tiles, two for V
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const unsigned smem_base = (unsigned)(uintptr_t)smem;

  // ids that are equal modulo 8 run on one XCD, whose L2 then holds the K and V of its heads; the heads of up to 7
  // key heads beyond a multiple of 8, untied, are dealt to all.  Either an XCD's heads one behind the other (the
  // untied ones first), late blocks, which have the most keys, in front, or the late blocks of all its heads in
  // front, eight slots at a time.
  const int id = (int)(blockIdx.y * kGridRow + blockIdx.x), rep = a.heads / a.kv_heads, untied = (a.kv_heads & 7) * rep;
  int head, slot;
  const auto tied_head = [&](int nth) { return ((id & 7) + 8 * (nth / rep)) * rep + nth % rep; };
  if (a.longest_first) {
    // eight slots are a.heads rows of 8 ids, in the order of their slots: `untied` of them, spread among the others,
    // for the untied heads
    const int eight = id / (8 * a.heads), row = (id - eight * 8 * a.heads) >> 3, tied = a.heads - untied;
    const int u = row * untied / a.heads, t = row - u;  // rows of either kind in front
    if ((row + 1) * untied / a.heads > u) {
      slot = (8 * u + (id & 7)) / untied;
      const int at = 8 * u + (id & 7) - slot * untied, few = a.kv_heads & 7, nth = at / few;
      head = tied + (at - nth * few) * rep + nth;  // 1, 2 or 4 key heads each have XCDs of their own
    } else {
      slot = t / (tied >> 3);
      head = tied_head(t - slot * (tied >> 3));
    }
    slot += 8 * eight;
    if (slot >= a.slots) return;
  } else if (id >= a.slots * a.heads) {
    return;
  } else if (id < a.slots * untied) {
    slot = id / untied;
    head = a.heads - untied + (id - slot * untied);
  } else {
    const int at = (id - a.slots * untied) >> 3, nth = at / a.slots;
    slot = at - nth * a.slots;
    head = tied_head(nth);
  }
  const Block block = a.longest_first && a.sequences > 1 ? nth_longest<R>(a, slot) : find_block<R>(a, a.slots - 1 - slot);
  if (block.length == 0) return;
  const int L = block.length, q0 = block.block * R;
  // part p of P has the key tiles p, p + P, .., perhaps none
  const int part = P == 1 ? 0 : wave >> 1, in_part = P == 1 ? wave : wave & 1;
  const int qw0 = q0 + in_part * 16 * QB;
  const bool wave_active = qw0 < L;
  const int last_q = min(q0 + R, L) - 1;
  const int nt = last_q / kKeys + 1;  // key tiles
  const int own = (nt - part + P - 1) / P;  // of this part
  const int kv_head = head / rep;
  const _Float16* qp = a.q + (block.first * a.q_row + head * a.q_head);
  const _Float16* kp = a.k + (block.first * a.k_row + kv_head * a.k_head);
  const _Float16* vp = a.v + (block.first * a.v_row + kv_head * a.v_head);

  // ---- queries: lane (c, g) holds d = 32 ks + 8 g + 0..7 (nothing where there is no such d); rows past the end repeat
  // the last one and are not stored
  h8 qf[QB][KS];
#pragma unroll
  for (int n = 0; n < QB; ++n) {
    const _Float16* p = qp + (int64_t)min(qw0 + 16 * n + c, L - 1) * a.q_row + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[n][ks] = h8(0);
      if (D >= 32 || g < 2) qf[n][ks] = *reinterpret_cast<const h8*>(p + ks * 32);
    }
  }

  // ---- tile loads: wavefronts 0-1 bring K, 2-3 V, 32 rows each; with two parts one wavefront of each K and one V.
  // Load j's rows are RPI j further on, which the scalar base takes, and their keys differ by bits that are the same
  // for all lanes; a sequence's last tile repeats its last row.
  const bool brings_v = P == 1 ? wave >= 2 : wave & 1;
  const int first_row = P == 1 ? (wave & 1) * 32 : 0;
  const int64_t pitch = (brings_v ? a.v_row : a.k_row) * 2;
  const char* src = (const char*)(brings_v ? vp : kp) + first_row * pitch;
  const int lrow = lane / CH;
  const unsigned lane_unit = (unsigned)((lane % CH) ^ (brings_v ? v_key(lrow) : k_key(lrow))) << 4;
  const unsigned lane_row = (unsigned)lrow * (unsigned)pitch;
  auto issue_tile = [&](int nth) {  // of this part's tiles
    const int t = nth * P + part;
    const int place = part * 4 + (brings_v ? 2 : 0) + (nth & 1);
    const unsigned dst = smem_base + (unsigned)(place * TILE + first_row * ROWB);
    const char* base = src + (int64_t)t * kKeys * pitch;
    const int rest = L - 1 - t * kKeys - first_row;  // the last row of this wavefront's
    if (rest >= ROWS - 1) {
#pragma unroll
      for (int j = 0; j < NDMA; ++j) {
        const unsigned key = (unsigned)(brings_v ? v_key(j * RPI) : k_key(j * RPI));
        load_lds16(base, (lane_unit ^ (key << 4)) + lane_row, dst + j * 1024);
        base += RPI * pitch;
      }
    } else {
      base += (int64_t)min(rest, 0) * pitch;  // of rows behind the end, row 0 is the sequence's last
      const int last = max(rest, 0);
#pragma unroll
      for (int j = 0; j < NDMA; ++j) {
        const unsigned key = (unsigned)(brings_v ? v_key(j * RPI) : k_key(j * RPI));
        load_lds16(base, (unsigned)min(j * RPI + lrow, last) * (unsigned)pitch + (lane_unit ^ (key << 4)), dst + j * 1024);
      }
    }
  };

  // ---- LDS read offsets of this lane inside a tile
  const int k_row = 8 * (c >> 2) + (c & 3), v_row = 8 * g + (c >> 2);
  constexpr int KV = KS < 4 ? KS : 4, VV = DB < 8 ? DB : 8;
  int k_off[KV], v_off[VV];
#pragma unroll
  for (int ks = 0; ks < KV; ++ks) k_off[ks] = k_row * ROWB + (((4 * ks + (D >= 32 ? g : g & 1)) ^ k_key(k_row)) << 4);
#pragma unroll
  for (int i = 0; i < VV; ++i)
    v_off[i] = 2 * TILE + v_row * ROWB + (((2 * i + ((c & 3) >> 1)) ^ v_key(v_row)) << 4) + (c & 1) * 8;
  const float to_exp2 = a.scale * 1.4426950408889634f;

  f4 oacc[QB][DB];  // of query c of block n: d = 16 i + 4 g + 0..3
#pragma unroll
  for (int n = 0; n < QB; ++n)
#pragma unroll
    for (int i = 0; i < DB; ++i) oacc[n][i] = f4(0.f);
  // The weights are 2^(t s - base), t = scale log2(e), base = t ref - 6 as rounded, for a reference that the running
  // maximum may pass by 2^8 before it follows: the accumulator is rescaled in few tiles (by what the bases as rounded
  // differ by, so that tiles of different references agree), a weight is at most 2^14, and one is a subnormal fp16
  // number, which has fewer bits, below 2^-20 of the reference.  The denominator adds the weights in fp32, in the
  // four lanes of a query and across them at the end.  (us, this / dot products of the rounded pairs with ones, which
  // flush subnormal weights / a column of ones in the matrix product, which costs registers: 48 of up to 1024 rows
  // 23.2 / 23.1 / 26.0, 1 x 16384 995 / 988 / 1003.) The key that set the reference weighs 2^6, so a denominator
  // below 2^5 is one whose base was rounded by more than the weights reach, which the end looks for.
  float ref[QB], limit[QB], base[QB], den[QB];
#pragma unroll
  for (int n = 0; n < QB; ++n) ref[n] = limit[n] = base[n] = -INFINITY, den[n] = 0.f;
  const float room = 8.0f / to_exp2;

  // One 64-key tile.  MASK: the one that the diagonal cuts, in which query x of the wavefront sees keys 0 .. edge + x;
  // KG = 1: none of them the second 32 of it.
  const int edge = qw0 & 63;
  f4 s[QB][4];  // scores, [block][2 group + b]
  auto scores = [&](const char* buf) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int at = (kb >> 1) * 32 * ROWB + (kb & 1) * 4 * ROWB + k_off[ks % KV] + (ks / KV) * 256;
        h8 kf = *reinterpret_cast<const h8*>(buf + at);
        if (D < 32 && g >= 2) kf = h8(0);
#pragma unroll
        for (int n = 0; n < QB; ++n)
          s[n][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[n][ks], ks == 0 ? f4(0.f) : s[n][kb], 0, 0, 0);
      }
  };
  h8 pf[QB][2];
  auto softmax = [&](auto mask, auto key_groups) {
    constexpr bool MASK = decltype(mask)::value;
    constexpr int KG = decltype(key_groups)::value;
    float most[QB];
    bool higher = false;
#pragma unroll
    for (int n = 0; n < QB; ++n) {
      if constexpr (MASK) {
#pragma unroll
        for (int kb = 0; kb < 2 * KG; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[n][kb][r] = (kb >> 1) * 32 + (kb & 1) * 4 + r + 8 * g <= edge + 16 * n + c ? s[n][kb][r] : -INFINITY;
      }
      float m = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2 * KG; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = larger(m, s[n][kb][r]);
      const LanePair halves = half_swap(m);
      const LanePair p = row_swap(larger(halves.a, halves.b));
      most[n] = larger(p.a, p.b);
      higher |= most[n] > limit[n];
    }
    if (D > 128 || __any(higher)) {  // a branch there costs registers that there are none of
#pragma unroll
      for (int n = 0; n < QB; ++n) {
        const float to = larger(most[n], ref[n]), next = fmaf(to, to_exp2, -6.0f);
        const float mult = __builtin_amdgcn_exp2f(base[n] - next);
        ref[n] = to;
        limit[n] = to + room;
        base[n] = next;
        den[n] *= mult;
#pragma unroll
        for (int i = 0; i < DB; ++i) oacc[n][i] *= mult;
      }
    }
#pragma unroll
    for (int n = 0; n < QB; ++n)
#pragma unroll
      for (int kb = 0; kb < 2 * KG; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[n][kb][r], to_exp2, -base[n]));
          pf[n][kb >> 1][4 * (kb & 1) + r] = (_Float16)p;
          den[n] += p;
        }
#pragma unroll
    for (int n = 0; n < QB; ++n) asm volatile("" : "+v"(den[n]));  // here, not with copies of the weights behind the barrier
  };
  auto weighted = [&](auto key_groups, const char* buf) {
    constexpr int KG = decltype(key_groups)::value;
#pragma unroll
    for (int kg = 0; kg < KG; ++kg)
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        const char* vt = buf + kg * 32 * ROWB + v_off[i % VV] + (i / VV) * 256;
        const h4 lo = lds_read_tr16(vt), hi = lds_read_tr16(vt + 4 * ROWB);
        const h8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int n = 0; n < QB; ++n)
          oacc[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[n][kg], oacc[n][i], 0, 0, 0);
      }
  };
  const int nfull = qw0 >> 6;  // key tiles entirely below this wavefront's diagonal
  // The order inside a wavefront is softmax of tile t, the score products of tile t + 1, the P . V products of tile t,
  // which the matrix pipe works through under the softmax of tile t + 1 and other wavefronts'.  So step t has K of tile t + 1
  // and V of tile t, with K of t + 2 and V of t + 1 on their way: two places each.
  // What this wavefront requested has landed; behind the barrier that holds for everyone, and the last step's tiles are free.
  auto arrive = [&] { asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  auto request = [&](int k_tile) {  // and the V tile in front of it
    const int t = brings_v ? k_tile - 1 : k_tile;
    if (t < own) issue_tile(t);
  };
  auto tile = [&](int t) { return (const char*)smem + part * 4 * TILE + (t & 1) * TILE; };
  if (own > 0) issue_tile(0);
  if (!brings_v && own > 1) issue_tile(1);
  arrive();
#pragma unroll
  for (int n = 0; n < QB; ++n)  // they have landed too: no wait at their uses
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[n][ks]));
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  const bool has = wave_active && (P == 1 || nfull >= part);
  const int full = P == 1 ? nfull : (nfull - part) >> 1;  // tiles of this part in front of its last one
  const int steps = (nt + P - 1) / P - 1;                 // for all wavefronts
  if (has) scores(tile(0));
  if (steps > 0) {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone is done with K of tile 0
    request(2);
  }
  if (has) {
    for (int t = 0; t < full; ++t) {
      softmax(std::false_type{}, two);
      __builtin_amdgcn_sched_barrier(0);
      scores(tile(t + 1));
      weighted(two, tile(t));
      arrive();
      request(t + 3);
    }
    if (P > 1 && (nfull - part) % P != 0) {
      softmax(std::false_type{}, two);
      weighted(two, tile(full));
    } else if (D <= 64 && QB <= 2 && edge + 16 * QB <= 32) {
      softmax(std::true_type{}, one);
      weighted(one, tile(full));
    } else {
      softmax(std::true_type{}, two);
      weighted(two, tile(full));
    }
  }
  for (int t = has ? full : 0; t < steps; ++t) {
    arrive();
    request(t + 3);
  }
  if constexpr (P > 1) {
    // The second part's sums, scaled to the larger of both references, to the first's: by LDS, whose tiles are done with.
    f4* sums = reinterpret_cast<f4*>(smem) + in_part * QB * (DB + 1) * kWave + lane;
    __syncthreads();
    if (part == 1 && wave_active) {
#pragma unroll
      for (int n = 0; n < QB; ++n) {
#pragma unroll
        for (int i = 0; i < DB; ++i) sums[(n * (DB + 1) + i) * kWave] = oacc[n][i];
        sums[(n * (DB + 1) + DB) * kWave] = f4{base[n], den[n], 0.f, 0.f};
      }
    }
    __syncthreads();
    if (part == 1 || !wave_active) return;
#pragma unroll
    for (int n = 0; n < QB; ++n) {
      const f4 other = sums[(n * (DB + 1) + DB) * kWave];
      const float to = larger(base[n], other[0]);
      const float mine = __builtin_amdgcn_exp2f(base[n] - to), its = __builtin_amdgcn_exp2f(other[0] - to);
      den[n] = fmaf(den[n], mine, other[1] * its);
#pragma unroll
      for (int i = 0; i < DB; ++i) oacc[n][i] = oacc[n][i] * mine + sums[(n * (DB + 1) + i) * kWave] * its;
    }
  }
  if (!wave_active) return;

  // ---- an infinity or a NaN among the results: one of the inputs is none, and a hidden key's value, times its weight
  // of 0, may have spoilt queries in front of it; or scores are beyond what fp32 has of an exponent (some 2^25).  Once
  // more, key by key, for these 16 queries.  Then the output, 8 bytes a lane and 32 for the four of a query.
#pragma unroll
  for (int n = 0; n < QB; ++n) {
    const int q = qw0 + 16 * n + c;
    const LanePair pair = row_swap(half_sum(den[n]));
    const float sum = pair.a + pair.b, inv = 1.0f / sum;
    float none = sum >= 32.0f ? 0.f : 1.f;
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      oacc[n][i] *= inv;
#pragma unroll
      for (int r = 0; r < 4; ++r) none = fmaf(oacc[n][i][r], 0.f, none);
    }
    if (__any(none != 0.f && q < L)) {
      const int last = min(qw0 + 16 * n + 15, L - 1);
      // of query c with key j, from this lane's elements of both and the other three lanes': one rounded number
      auto score = [&](int j) {
#pragma clang fp contract(off)
        const _Float16* kj = kp + (int64_t)j * a.k_row + g * 8;
        float x = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (D < 32 && g >= 2) continue;
          const h8 kf = *reinterpret_cast<const h8*>(kj + ks * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) x = fmaf((float)qf[n][ks][i], (float)kf[i], x);
        }
        const LanePair pair = row_swap(half_sum(x));
        return (pair.a + pair.b) * a.scale;
      };
      float m = -INFINITY, total = 0.f;
#pragma unroll 4
      for (int j = 0; j <= last; ++j) {
        const float x = score(j), to = fmaxf(m, x), by = to == -INFINITY ? 0.f : to;
        const float more = fmaf(total, __expf(m - by), __expf(x - by));
        total = j <= q ? more : total;
        m = j <= q ? to : m;
      }
      const bool number = total == total && fabsf(m) < INFINITY;  // else there is no softmax
      const float inv_total = number ? 1.0f / total : NAN;
#pragma unroll
      for (int i = 0; i < DB; ++i) oacc[n][i] = f4(number ? 0.f : NAN);
      if (__any(number && q < L)) {
#pragma unroll 2
        for (int j = 0; j <= last; ++j) {
          const float w = __expf(score(j) - m) * inv_total;
          const _Float16* vj = vp + (int64_t)j * a.v_row + 4 * g;
#pragma unroll
          for (int i = 0; i < DB; ++i) {
            const h4 vf = *reinterpret_cast<const h4*>(vj + 16 * i);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float more = fmaf(w, (float)vf[r], oacc[n][i][r]);
              oacc[n][i][r] = j <= q ? more : oacc[n][i][r];
            }
          }
        }
      }
    }
    _Float16* o = a.out + ((block.first + q) * a.heads + head) * D + 4 * g;
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      h4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = (_Float16)bounded(oacc[n][i][r]);
      if (q < L) *reinterpret_cast<h4*>(o + 16 * i) = x;
    }
  }
}

template <int D, int QB, int P>
int launch_as(PackedArgs a, int64_t slots, hipStream_t st) {
  const int64_t blocks = slots * a.heads;
  if (blocks > (1ll << 31) - kGridRow) {
    set_error("flash_attn_packed: %lld rows in %d sequences of %d heads exceed the grid", (long long)a.rows, a.sequences,
              a.heads);
    return -2;
  }
  constexpr int lds = P * 2 * 2 * kKeys * D * 2;
  static bool attr_done = false;  // idempotent; a race only repeats the call
  if (!attr_done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(packed_attn_kernel<D, QB, P>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("hipFuncSetAttribute(%d bytes LDS): %s", lds, hipGetErrorString(e));
      return -4;
    }
    attr_done = true;
  }
  a.slots = (int)slots;
  // Up to 20 workgroups a CU the heaviest of all heads first: whichever starts last ends the launch.  Beyond, and
  // where there is hardly more than a block a sequence, a head's blocks one behind the other, whose K and V then come
  // from one XCD's L2. us, by slots / heaviest first: 2 x 8192 rows of 12 heads (1560 workgroups) 268 / 236, 16 x
  // 1024 (1728) 51.4 / 42.3, 8 x 4096 of 16 (4224) 349 / 336, 100 of up to 2048 (6064) 151 / 158, 64 x 1024 of 25
  // (14400) 337 / 441, 200 x 64 of 12 (3600) 22.0 / 23.6, 1 x 4096 (780) 62.6 / 58.3, 1 x 16384 of 25 (3225) 992 /
  // 926 (980 with the heads dealt to all XCDs, whose L2s then ask for seven times as much); d = 128, 32 heads over 8,
  // 6 of up to 4096 (3360) 394 / 375, 32 of up to 2048 (3680) 169 / 153, 16 x 1024 (4608) 211 / 202; d = 256, 4 x
  // 1024 of 12 (432) 108 / 69.
  a.longest_first = a.sequences <= kMany * kWave && slots <= 512 && blocks <= 5120 && a.rows >= 128ll * a.sequences;
  const int64_t grid = a.longest_first ? (slots + 7) / 8 * 8 * a.heads : blocks;
  const dim3 dims((unsigned)(grid < kGridRow ? grid : kGridRow), (unsigned)((grid + kGridRow - 1) / kGridRow));
  hipLaunchKernelGGL((packed_attn_kernel<D, QB, P>), dims, dim3(256), lds, st, a);
  return 0;
}

// While the workgroups run at once, the launch takes what a wavefront's chain through its key tiles takes: 0.5 us a
// tile for 16 queries, 0.8 for 32.  So up to 2.5 workgroups a CU of 32 queries, in two parts of the key tiles; up to 2
// of 64 in two parts, 3 or 4 the longer the sequences are, which then hide what a workgroup begins and ends with; up to
// 5 of 64 queries, 16 a wavefront; and 32 a wavefront beyond: K and V are read from LDS for more queries at a time.
// us, 16 / 32 / 16 in two parts / 32 in two parts: 1 x 1024 rows of 12 heads 15.8 / 18.7 / 10.4 / 12.7 (396 workgroups
// in two parts, 204 of 64 queries), 1 x 2500 34.1 / 39.5 / 25.3 / 27.5 (948, 480), 1 x 4096 56.3 / 64.6 / 57.5 / 44.0
// (1548, 780), 1 x 1024 of 25 heads 16.4 / 19.1 / 15.1 / 13.9 (825, 425), 1 x 2048 32.1 / 35.1 / 35.7 / 29.0 (1625,
// 825), 8 x 150 9.9 / 9.9 / 11.5 / 12.5 (1125, 650), 4 x 1024 of 12 19.8 / 22.6 / 32.3 / 23.3 (1584, 816), 16 x 300
// 11.3 / 13.0 / 23.7 / 16.3 (2184, 1092), 48 of up to 1024 (7558 rows) 24.0 / 22.3 / 53.8 / 34.1 (3408, 1992), 2 x 8192
// 293 / 245 / 361 / 320.  d = 128: two parts fill a CU's LDS, 1 x 1024 of 12 heads 20.5 / 27.1 / 19.4 / 19.7, 1 x 1024 of
// 32 over 8 23.1 / 28.2 / 42.1 / 27.1: not taken.  64 queries a wavefront were slower yet: 1 x 16384 of 25 heads 16 / 32 /
// 64 1046 / 969 / 997 in an earlier state.  d = 256 has one workgroup a CU either way.
template <int D>
int launch_d(const PackedArgs& a, hipStream_t st) {
  const int64_t slots32 = a.rows / 32 + a.sequences, slots = a.rows / 64 + a.sequences;
  if constexpr (D <= 64) {
    if (slots32 * a.heads <= 640) return launch_as<D, 1, 2>(a, slots32, st);
    const int64_t average = a.rows / a.sequences;
    if (slots * a.heads <= (average >= 2048 ? 1024 : average >= 256 ? 768 : 512)) return launch_as<D, 2, 2>(a, slots, st);
  }
  if constexpr (D <= 128)
    if (slots * a.heads <= 1280) return launch_as<D, 1, 1>(a, slots, st);
  return launch_as<D, 2, 1>(a, a.rows / 128 + a.sequences, st);
}

}  // namespace

int launch_flash_attn_packed(const PackedAttention& p, int d, hipStream_t st) {
  PackedArgs a;
  a.q = (const _Float16*)p.q;
  a.k = (const _Float16*)p.k;
  a.v = (const _Float16*)p.v;
  a.out = (_Float16*)p.out;
  a.starts = p.starts;
  a.rows = p.rows;
  a.sequences = (int)p.sequences;
  a.heads = (int)p.heads;
  a.kv_heads = (int)p.kv_heads;
  a.q_row = p.q_row, a.q_head = p.q_head, a.k_row = p.k_row, a.k_head = p.k_head, a.v_row = p.v_row, a.v_head = p.v_head;
  a.scale = p.scale;
  switch (d) {
    case 16: return launch_d<16>(a, st);
    case 32: return launch_d<32>(a, st);
    case 64: return launch_d<64>(a, st);
    case 128: return launch_d<128>(a, st);
    case 256: return launch_d<256>(a, st);
  }
  set_error("flash_attn_packed: head size %d (16, 32, 64, 128 and 256 are supported)", d);
  return -2;
}

}  // namespace gptmi
