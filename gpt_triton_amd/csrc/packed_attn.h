// What the kernels over packed sequences share: where a workgroup's rows are, and in which order the work is dealt.
#pragma once
#include <stdint.h>

#include "common.h"

namespace gptmi {

constexpr int kGridRow = 1 << 20;  // workgroups a row of the grid: threads of one dimension have to stay below 2^32

// Sequences one behind the other: sequence s is the rows starts[s] .. starts[s + 1] - 1 of `rows`.
struct Sequences {
  const int64_t* starts;
  int64_t rows;  // T
  int sequences;
};

// 16 bytes a lane from base + lane_off into LDS at lds_off + 16 lane.  Assembly, so that the compiler does not wait
// for these loads in front of each LDS read; the kernel waits by hand.
__device__ __forceinline__ void load_lds16(const void* base, unsigned lane_off, unsigned lds_off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_off), "v"(lane_off), "s"(base)
               : "memory", "m0");
}

// Lane (c, g) has columns 4 g + 0..3 of two blocks of 16 columns of row c.  Rows of lanes exchange halves, so that a lane stores 16
// bytes and four lanes 64 side by side, not 32 (us, gradients of 48 x 300 tokens, 12 heads of 64: 72, else 77).
__device__ __forceinline__ void store_blocks(_Float16* at, int g, h4 first, h4 second, bool there) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  const u2 p = __builtin_bit_cast(u2, first), q = __builtin_bit_cast(u2, second);
  const auto low = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
  const auto high = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
  if (there) *reinterpret_cast<u4*>(at + 16 * (g & 1) + 8 * (g >> 1)) = u4{low[0], high[0], low[1], high[1]};
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
__device__ __forceinline__ Block find_block(const Sequences& a, int slot) {
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
__device__ __forceinline__ Block nth_longest(const Sequences& a, int nth) {
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

// Which head, of `heads` over `kv_heads`, and which slot a workgroup has; false: none.
// ids that are equal modulo 8 run on one XCD, whose L2 then holds the K and V of its heads; the heads of up to 7
// key heads beyond a multiple of 8, untied, are dealt to all.  Either an XCD's heads one behind the other (the
// untied ones first), late blocks, which have the most keys, in front, or the late blocks of all its heads in
// front, eight slots at a time.
struct Place {
  int head, slot;
};
__device__ __forceinline__ bool find_place(int id, int heads, int kv_heads, int slots, bool longest_first, Place* place) {
  const int rep = heads / kv_heads, untied = (kv_heads & 7) * rep;
  const auto tied_head = [&](int nth) { return ((id & 7) + 8 * (nth / rep)) * rep + nth % rep; };
  int head, slot;
  if (longest_first) {
    // eight slots are `heads` rows of 8 ids, in the order of their slots: `untied` of them, spread among the others,
    // for the untied heads
    const int eight = id / (8 * heads), row = (id - eight * 8 * heads) >> 3, tied = heads - untied;
    const int u = row * untied / heads, t = row - u;  // rows of either kind in front
    if ((row + 1) * untied / heads > u) {
      slot = (8 * u + (id & 7)) / untied;
      const int at = 8 * u + (id & 7) - slot * untied, few = kv_heads & 7, nth = at / few;
      head = tied + (at - nth * few) * rep + nth;  // 1, 2 or 4 key heads each have XCDs of their own
    } else {
      slot = t / (tied >> 3);
      head = tied_head(t - slot * (tied >> 3));
    }
    slot += 8 * eight;
    if (slot >= slots) return false;
  } else if (id >= slots * heads) {
    return false;
  } else if (id < slots * untied) {
    slot = id / untied;
    head = heads - untied + (id - slot * untied);
  } else {
    const int at = (id - slots * untied) >> 3, nth = at / slots;
    slot = at - nth * slots;
    head = tied_head(nth);
  }
  *place = {head, slot};
  return true;
}

}  // namespace gptmi
