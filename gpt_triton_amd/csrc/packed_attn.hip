// Causal attention over whole prompts that lie one behind the other without padding, with grouped heads, fp16:
//   out[i][n] = sum_{j <= i, same sequence} w_ij v[j][n / (N / G)],   w_i = softmax_j(scale q[i][n] . k[j][n / (N / G)])
// q [T][N][D], k, v [T][G][D] at row and head pitches of their own (the q, k, v product's rows as they are), out [T][N][D],
// sequence s the rows starts[s] .. starts[s + 1] - 1.
//
// One workgroup = 4 wavefronts = 128 queries of one sequence and head; wavefront w has queries 32 w .. 32 w + 31 of
// them.  The products are the transposed ones of flash_attn.hip, one lane one query: S^T = K . Q^T, O^T += V^T . P^T
// with v_mfma_f32_32x32x16_f16, so that the maximum and the sum of a row stay in a lane (and lane ^ 32) and P's registers
// are the second operand as they stand.
#include <type_traits>

#include "common.h"
#include "launch.h"

namespace gptmi {
namespace {

constexpr int kRows = 128;  // queries a workgroup
constexpr int kKeys = 64;   // keys a tile

struct PackedArgs {
  const _Float16 *q, *k, *v;
  _Float16* out;
  const int64_t* starts;
  int64_t rows;               // T
  int sequences, heads, kv_heads, slots;
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

// Slots: a sequence that starts at row a has the 128-query blocks from slot a / 128 + s on, which leaves room for
// every sequence whatever the lengths are (floor(a / 128) + floor(len / 128) <= floor((a + len) / 128)), needs no
// lengths on the host and no pass over them on the GPU.  Slots that are left over hold nothing.
struct Block {
  int64_t first;  // the sequence's first row
  int length;     // rows of it, 0: nothing to do
  int block;      // which 128 of them
};
__device__ __forceinline__ Block find_block(const PackedArgs& a, int slot) {
  // the last sequence whose first slot is not behind this one: 64 probes at a time
  const int lane = threadIdx.x & 63;
  int low = 0, left = a.sequences;
  while (left > 1) {
    const int step = (left + 63) >> 6, at = low + lane * step;
    bool in = false;
    if (lane * step < left) in = (a.starts[at] >> 7) + at <= slot;
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
  const int64_t length = last - first, block = slot - ((begin >> 7) + low);
  return {first, block >= 0 && block * kRows < length ? (int)length : 0, (int)block};
}

template <int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void packed_attn_kernel(PackedArgs a) {
  constexpr int KS = D / 16, DB = (D + 31) / 32;
  constexpr int ROWB = D * 2;          // bytes of a row in LDS
  constexpr int CH = D / 8;            // 16-byte units of it
  constexpr int RPI = 1024 / ROWB;     // rows that a load instruction covers
  constexpr int TILE = kKeys * ROWB;   // bytes of a K (or V) tile
  constexpr int STAGE = 2 * TILE;
  constexpr int NDMA = D / 16;         // load instructions a wavefront and tile
  // K unit u of row r lies at u ^ k_key(r), V at u ^ v_key(r): reads of one unit of 16 rows, and transposing reads of 64
  // bytes of 4 rows, meet all banks
  constexpr int KSHIFT = CH == 2 ? 3 : CH == 4 ? 2 : CH == 8 ? 1 : 0, KMASK = CH < 16 ? CH - 1 : 15;
  constexpr int VMUL = CH >= 16 ? 4 : CH == 8 ? 2 : 0;
  extern __shared__ __attribute__((aligned(1024))) char smem[];  // 2 stages, 64 bytes more for D = 16
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ql = lane & 31, g = lane >> 5;
  const unsigned smem_base = (unsigned)(uintptr_t)smem;

  // ids that are equal modulo 8 run on one XCD, whose L2 then holds the K and V of its heads; the heads of up to 7 key
  // heads beyond a multiple of 8 are dealt to all, first, for they have no such order.  Late blocks, which have the most keys,
  // come first.
  const int id = (int)blockIdx.x, rep = a.heads / a.kv_heads, untied = (a.kv_heads & 7) * rep;
  int head, slot;
  if (id < a.slots * untied) {
    slot = id / untied;
    head = a.heads - untied + (id - slot * untied);
  } else {
    const int at = (id - a.slots * untied) >> 3, nth = at / a.slots;
    slot = at - nth * a.slots;
    head = ((id & 7) + 8 * (nth / rep)) * rep + nth % rep;
  }
  const Block block = find_block(a, a.slots - 1 - slot);
  if (block.length == 0) return;
  const int L = block.length, q0 = block.block * kRows;
  const int qw0 = q0 + wave * 32, q = qw0 + ql;
  const bool wave_active = qw0 < L;
  const int last_q = min(q0 + kRows, L) - 1;
  const int nt = last_q / kKeys + 1;  // key tiles
  const int kv_head = head / rep;
  const _Float16* qp = a.q + (block.first * a.q_row + head * a.q_head);
  const _Float16* kp = a.k + (block.first * a.k_row + kv_head * a.k_head);
  const _Float16* vp = a.v + (block.first * a.v_row + kv_head * a.v_head);

  // ---- queries: lane (ql, g) holds d = 16 ks + 8 g + 0..7; rows past the end repeat the last one and are not stored
  h8 qf[KS];
  {
    const _Float16* p = qp + (int64_t)min(q, L - 1) * a.q_row + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const h8*>(p + ks * 16);
  }

  // ---- tile loads: wavefronts 0-1 bring K, 2-3 V, 32 rows each.  Load j's rows are RPI j further on, which the scalar
  // base takes, and their keys differ by bits that are the same for all lanes; a sequence's last tile repeats its last row.
  const bool brings_v = wave >= 2;
  const int64_t pitch = (brings_v ? a.v_row : a.k_row) * 2;
  const char* src = (const char*)(brings_v ? vp : kp) + (wave & 1) * 32 * pitch;
  const int lrow = lane / CH;
  const unsigned lane_unit = (unsigned)((lane % CH) ^ (brings_v ? VMUL * (lrow & 3) : (lrow >> KSHIFT) & KMASK)) << 4;
  const unsigned lane_row = (unsigned)lrow * (unsigned)pitch;
  auto issue_tile = [&](int t) {
    const unsigned dst = smem_base + (unsigned)((t & 1) * STAGE) + (brings_v ? (unsigned)TILE : 0u) +
                         (unsigned)((wave & 1) * NDMA) * 1024u;
    const char* base = src + (int64_t)t * kKeys * pitch;
    const int rest = L - 1 - t * kKeys - (wave & 1) * 32;  // the last row of this wavefront's 32
    if (rest >= 31) {
#pragma unroll
      for (int j = 0; j < NDMA; ++j) {
        const unsigned key = brings_v ? (unsigned)(VMUL * ((j * RPI) & 3)) : (unsigned)(((j * RPI) >> KSHIFT) & KMASK);
        load_lds16(base, (lane_unit ^ (key << 4)) + lane_row, dst + j * 1024);
        base += RPI * pitch;
      }
    } else {
      base += (int64_t)min(rest, 0) * pitch;  // of 32 rows behind the end, row 0 is the sequence's last
      const int last = max(rest, 0);
#pragma unroll
      for (int j = 0; j < NDMA; ++j) {
        const unsigned key = brings_v ? (unsigned)(VMUL * ((j * RPI) & 3)) : (unsigned)(((j * RPI) >> KSHIFT) & KMASK);
        load_lds16(base, (unsigned)min(j * RPI + lrow, last) * (unsigned)pitch + (lane_unit ^ (key << 4)), dst + j * 1024);
      }
    }
  };

  // ---- LDS read offsets of this lane inside a tile
  const int tri_q = ql - 4 * g;
  constexpr int KV = KS < 8 ? KS : 8;
  int k_off[KV];
#pragma unroll
  for (int ks = 0; ks < KV; ++ks) k_off[ks] = ql * ROWB + (((ks * 2 + g) ^ ((ql >> KSHIFT) & KMASK)) << 4);
  const int sl = lane & 15, vrow = 4 * g + (sl >> 2);
  constexpr int VV = DB < 4 ? DB : 4;
  int v_off[VV];
#pragma unroll
  for (int i = 0; i < VV; ++i) {
    const int unit = (4 * i + 2 * ((lane >> 4) & 1) + ((sl & 3) >> 1)) ^ (VMUL * (vrow & 3));
    v_off[i] = TILE + vrow * ROWB + (unit << 4) + (sl & 1) * 8;
  }
  const float c = a.scale * 1.4426950408889634f;

  f16v oacc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[i][r] = 0.f;
  // The weights are 2^(c s - base), base = c ref - 6, for a reference that the running maximum may pass by 2^8 before it
  // follows: the accumulator is rescaled in few tiles, a weight is at most 2^14, and one is a subnormal fp16 number, which
  // has fewer bits, below 2^-20 of the reference.  The denominator adds the weights as rounded for the product with V.
  float ref = -INFINITY, limit = -INFINITY, base = 0.f, den = 0.f;
  const float room = 8.0f / c;

  // One 64-key tile.  MODE 0: both 32-key blocks entirely visible; 1: block 0 cut by the diagonal, block 1 hidden; 2:
  // block 0 visible, block 1 cut by the diagonal.
  auto step = [&](auto mode_tag, const char* buf) {
    constexpr int MODE = decltype(mode_tag)::value;
    constexpr int NKB = MODE == 1 ? 1 : 2;
    f16v s[NKB];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const h8 kf = *reinterpret_cast<const h8*>(buf + kb * 32 * ROWB + k_off[ks % KV] + (ks / KV) * 256);
        s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[ks], s[kb], 0, 0, 0);
      }
    }
    if constexpr (MODE != 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[NKB - 1][r] = 8 * (r >> 2) + (r & 3) <= tri_q ? s[NKB - 1][r] : -INFINITY;
    }
    float bmax = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) bmax = fmaxf(bmax, s[kb][r]);
    bmax = half_max(bmax);
    if (D > 128 || __any(bmax > limit)) {  // a branch there costs registers that there are none of
      const float higher = fmaxf(bmax, ref), mult = __builtin_amdgcn_exp2f((ref - higher) * c);
      ref = higher;
      limit = higher + room;
      base = fmaf(higher, c, -6.0f);
      den *= mult;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[i][r] *= mult;
    }
    h8 pf[NKB][2];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          h2 p;
          p[0] = (_Float16)__builtin_amdgcn_exp2f(fmaf(s[kb][8 * tt + j], c, -base));
          p[1] = (_Float16)__builtin_amdgcn_exp2f(fmaf(s[kb][8 * tt + j + 1], c, -base));
          pf[kb][tt][j] = p[0];
          pf[kb][tt][j + 1] = p[1];
          den = __builtin_amdgcn_fdot2(p, h2{1, 1}, den, false);
        }
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const char* vt = buf + (kb * 32 + tt * 16) * ROWB;
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const h4 lo = lds_read_tr16(vt + v_off[i % VV] + (i / VV) * 256);
          const h4 hi = lds_read_tr16(vt + v_off[i % VV] + (i / VV) * 256 + 8 * ROWB);
          const h8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          oacc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[kb][tt], oacc[i], 0, 0, 0);
        }
      }
  };

  const int nfull = qw0 >> 6;  // key tiles entirely below this wavefront's diagonal
  auto arrive = [&] { asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  auto request = [&](int t) {
    if (t + 1 < nt) issue_tile(t + 1);
  };
  issue_tile(0);
  arrive();
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));  // they have landed too: no wait at their uses
  request(0);
  if (wave_active) {
    for (int t = 0; t < nfull; ++t) {
      step(std::integral_constant<int, 0>{}, smem + (t & 1) * STAGE);
      arrive();
      request(t + 1);
    }
    const char* buf = smem + (nfull & 1) * STAGE;
    if ((qw0 & 32) == 0) step(std::integral_constant<int, 1>{}, buf);
    else step(std::integral_constant<int, 2>{}, buf);
  }
  for (int t = wave_active ? nfull + 1 : 1; t < nt; ++t) {
    arrive();
    request(t);
  }
  if (!wave_active) return;

  // ---- an infinity or a NaN among the results: one of the inputs is none, and a hidden key's value, times its weight
  // of 0, may have spoilt queries in front of it.  Once more, key by key, for this wavefront.
  const float inv = 1.0f / half_sum(den);
  float none = 0.f;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (32 * i + 8 * (r >> 2) < D) {
        oacc[i][r] *= inv;
        none = fmaf(oacc[i][r], 0.f, none);
      }
  if (__any(none != 0.f && q < L)) {
    const int last = min(qw0 + 31, L - 1), mine = min(q, L - 1);
    const _Float16* p = qp + (int64_t)mine * a.q_row;
    auto score = [&](int j) {
      const _Float16* kj = kp + (int64_t)j * a.k_row;
      float s = 0.f;
#pragma unroll 1
      for (int d = 0; d < D; ++d) s = fmaf((float)p[d], (float)kj[d], s);
      return j <= mine ? s * a.scale : -INFINITY;
    };
    float m = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int j = 0; j <= last; ++j) m = fmaxf(m, score(j));
#pragma unroll 1
    for (int j = 0; j <= last; ++j) sum += j <= mine ? __expf(score(j) - m) : 0.f;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[i][r] = 0.f;
#pragma unroll 1
    for (int j = 0; j <= last; ++j) {
      const float w = __expf(score(j) - m) / sum;
      const _Float16* vj = vp + (int64_t)j * a.v_row + 4 * g;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * i + 8 * (r >> 2) < D) {
            const float more = fmaf(w, (float)vj[32 * i + 8 * (r >> 2) + (r & 3)], oacc[i][r]);
            oacc[i][r] = j <= mine ? more : oacc[i][r];
          }
    }
  }

  // ---- output: the two lanes of a query trade halves and store 16 bytes each
  _Float16* o = a.out + ((block.first + q) * a.heads + head) * D + 8 * g;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      if (32 * i + 16 * pr >= D) continue;
      h4 x, y;  // d = 32 i + 16 pr + 4 g + 0..3 and the same + 8
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = (_Float16)oacc[i][8 * pr + j];
        y[j] = (_Float16)oacc[i][8 * pr + 4 + j];
      }
      const u2 xd = __builtin_bit_cast(u2, x), yd = __builtin_bit_cast(u2, y);
      const auto r0 = __builtin_amdgcn_permlane32_swap(xd[0], yd[0], false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(xd[1], yd[1], false, false);
      if (q < L) *reinterpret_cast<u4*>(o + i * 32 + 16 * pr) = u4{r0[0], r1[0], r0[1], r1[1]};
    }
}

template <int D>
int launch_d(const PackedArgs& a, hipStream_t st) {
  constexpr int lds = 2 * 2 * kKeys * D * 2 + 64;
  static bool attr_done = false;  // idempotent; a race only repeats the call
  if (!attr_done) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(packed_attn_kernel<D>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) {
      set_error("hipFuncSetAttribute(%d bytes LDS): %s", lds, hipGetErrorString(e));
      return -4;
    }
    attr_done = true;
  }
  hipLaunchKernelGGL(packed_attn_kernel<D>, dim3((unsigned)(a.slots * a.heads)), dim3(256), lds, st, a);
  return 0;
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
  const int64_t slots = p.rows / kRows + p.sequences;
  if (slots * p.heads >= 1ll << 31) {
    set_error("flash_attn_packed: %lld rows in %lld sequences of %lld heads exceed the grid", (long long)p.rows,
              (long long)p.sequences, (long long)p.heads);
    return -2;
  }
  a.slots = (int)slots;
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
