// Rows of logits: log probabilities of given tokens with the row's entropy and its most likely tokens, their
// gradient, and the distillation loss against a teacher's top logits with its gradient.
//
// One workgroup per row.  With z = x / temperature, m = max x and c = log2(e) / temperature, the logits are taken as
// e_j = 2^t_j, t_j = x_j c - b, b = m c rounded to fp32; one logit that equals m is left out of the sums
//   s = sum e_j,   u = sum e_j t_j       and is 2^d itself, d = m c - b (what the rounding left)
// so that, with S = 2^d + s and L = log1p(s 2^-d) = log(S) - d log 2,
//   log p_j = (x_j - m) / temperature - L       H = -sum p_j log p_j = L - log 2 (u - d s) / S       p_j = e_j / S
// L is the logarithm of a number near 1 where one token has nearly all the probability, and keeps its bits there (a log
// probability of -1e-5, say); H's two terms are both positive, so neither loses bits to the other.
// Maximum, sums and logarithms are fp32.
#include "common.h"

namespace gptmi {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 128;     // top tokens, and a teacher's entries

template <typename T> struct RowVec;
template <> struct RowVec<_Float16> {
  typedef h8 V;
  static constexpr int N = 8;
};
template <> struct RowVec<float> {
  typedef f4 V;
  static constexpr int N = 4;
};

// Maximum and minimum of which any NaN makes a NaN (one instruction each, two for the price of one in fp16).
template <typename A>
__device__ __forceinline__ A most_of(A a, A b) { return __builtin_elementwise_maximum(a, b); }
template <typename A>
__device__ __forceinline__ A least_of(A a, A b) { return __builtin_elementwise_minimum(a, b); }

// A row as the workgroup's threads share it: 16-byte chunks from the first aligned address on, dealt one behind
// the other, and in front and behind at most 2 (N - 1) single elements, one for each of the first threads.
// It is read once and stays in registers, CH chunks a thread (-infinity where it has ended); OPEN: what a longer row has
// behind those is read again by every pass.
template <typename T, int NT, int CH, bool OPEN>
struct Row {
  typedef typename RowVec<T>::V V;
  static constexpr int N = RowVec<T>::N;
  const T* x;
  int vocab, lead, chunks, loose;  // loose: the index of this thread's single element, or -1
  V held[CH > 0 ? CH : 1];
  T single;
  __device__ __forceinline__ Row(const T* row, int vocab_) : x(row), vocab(vocab_) {
    const int ahead = (int)((-(intptr_t)row & 15) / (int)sizeof(T));
    lead = ahead < vocab ? ahead : vocab;
    chunks = (vocab - lead) / N;
    loose = loose_of(threadIdx.x);
  }
  __device__ __forceinline__ int loose_of(int t) const {
    return t < lead ? t : t < vocab - chunks * N ? t + chunks * N : -1;
  }
  __device__ __forceinline__ V chunk(int c) const {
    V v = V((T)-INFINITY);
    if (c < chunks) v = reinterpret_cast<const V*>(x + lead)[c];
    return v;
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < CH; ++i) held[i] = chunk(threadIdx.x + i * NT);
    single = (T)-INFINITY;
    if (loose >= 0) single = x[loose];
  }
  // In front of a pass: what the last one converted is not kept for this one, which is a register for each element, and
  // the single element's index is formed again, two registers that the pass in between spilled (88 us instead of 82 for
  // the loss and gradient of 2048 rows of 50257 fp16 logits).
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int i = 0; i < CH; ++i) asm volatile("" : "+v"(held[i]));
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    loose = loose_of(t);
  }
  // whether a wavefront has any of chunk i
  __device__ __forceinline__ bool part(int i) const {
    return i == 0 || __builtin_amdgcn_readfirstlane((int)threadIdx.x & -kWave) + i * NT < chunks;
  }
  // f(chunks, the first one's number, how many: up to G) for this thread's part of the row but for the single element, the
  // first as soon as they are there, the others NT chunks further on each; -infinity for what is not there
  template <int G, typename F>
  __device__ __forceinline__ void groups(F f) const {
    constexpr int REST = CH % G;
#pragma unroll
    for (int i = 0; i + G <= CH; i += G)
      if (part(i)) f(held + i, (int)threadIdx.x + i * NT, std::integral_constant<int, G>{});
    if constexpr (REST > 0)
      if (part(CH - REST)) f(held + CH - REST, (int)threadIdx.x + (CH - REST) * NT, std::integral_constant<int, REST>{});
    if constexpr (OPEN) {
      for (int c = threadIdx.x + CH * NT; c < chunks; c += G * NT) {
        V v[G];
#pragma unroll
        for (int k = 0; k < G; ++k) v[k] = chunk(c + k * NT);
        f(v, c, std::integral_constant<int, G>{});
      }
    }
  }
  // f(values, index of the first of them, how many: N or 1) for this thread's part of the row; a single element that is
  // not there has index -1
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    groups<4>([&](const V* v, int c, auto n) {
#pragma unroll
      for (int k = 0; k < n.value; ++k)
        if (part_of(c + k * NT)) {
          float y[N];
#pragma unroll
          for (int j = 0; j < N; ++j) y[j] = (float)v[k][j];
          f(y, lead + (c + k * NT) * N, std::integral_constant<int, N>{});
        }
    });
    const float y[1] = {(float)single};
    f(y, loose, std::integral_constant<int, 1>{});
  }
  __device__ __forceinline__ bool part_of(int c) const {
    return __builtin_amdgcn_readfirstlane(c & -kWave) < chunks;
  }
  __device__ __forceinline__ float at(int64_t i) const { return (float)x[i]; }
};

// All threads of a row: a workgroup, or a wavefront of one, whose LDS operations are in order as they stand.
template <int NT>
__device__ __forceinline__ void sync_row() {
  if constexpr (NT == kWave) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}
// Rows of a workgroup, the one that a thread works on, and its part of an LDS array with an element a row.
template <int NT>
constexpr int kRowsOf = NT == kWave ? 4 : 1;
template <int NT>
__device__ __forceinline__ int row_in_group() {
  return NT == kWave ? __builtin_amdgcn_readfirstlane((int)threadIdx.y) : 0;
}

// 2^20 workgroups a row of the grid: threads of one dimension have to stay below 2^32.
constexpr int kGridRow = 1 << 20;
template <int NT>
__device__ __forceinline__ int64_t row_of_group(int in_group) {
  return ((int64_t)blockIdx.y * kGridRow + blockIdx.x) * kRowsOf<NT> + in_group;
}

template <int NT>
struct Shared {
  static constexpr int W = NT / kWave;
  float top[W], s[W], u[W], low[W];
  float groups[64], many[256];  // maxima of 64 groups of threads, and of 256 where there are so many
  int scan[W];
};

// The value of the lane that differs by D = 1, 2, 4 or 8; for 4 and 8 of one with the same bits above, which is as good
// where the lanes that differ by less have one value: a group's sum or maximum is formed with D = 1, 2, ..
template <int D, typename A>
__device__ __forceinline__ A from_lane(A v) {
  constexpr int control = D == 1 ? 0xb1 : D == 2 ? 0x4e : D == 4 ? 0x141 : 0x140;  // quad_perm, row_half_mirror, row_mirror
  return __builtin_bit_cast(A, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), control, 0xf, 0xf, true));
}

// op over the W values (a power of two up to 16) that lane l has the l % W-th of, for every lane.
template <int W, typename Op>
__device__ __forceinline__ float join(float v, Op op) {
  if constexpr (W >= 16) v = op(v, row_rotate<8>(v));
  if constexpr (W >= 8) v = op(v, row_rotate<4>(v));
  if constexpr (W >= 4) v = op(v, row_rotate<2>(v));
  if constexpr (W >= 2) v = op(v, row_rotate<1>(v));
  return v;
}

// t = x c - b.  fp16: one operation from the logit as it is, b rounded once for all of a row (by up to 32 for logits of 65504
// and a temperature of 1e-4, the least that the host lets through, where 2^32 is the largest exponential).  fp32, whose m c
// may overflow: the difference, which is 0 for m, and its multiple.
template <typename T>
struct Exponent {
  float c, ref, b;
  __device__ __forceinline__ Exponent(float c_, float ref_) : c(c_) { at(ref_); }
  __device__ __forceinline__ void at(float r) {  // 0 in the place of -infinity: nothing is above it
#pragma clang fp contract(off)  // b is the rounded product wherever it is used
    ref = r == -INFINITY ? 0.f : r;
    b = ref * c;
  }
  __device__ __forceinline__ float operator()(float x) const {
    if constexpr (sizeof(T) == 2) return fmaf(x, c, -b);
    else return (x - ref) * c;
  }
  // what the operator gives for the reference itself
  __device__ __forceinline__ float rest() const { return (*this)(ref); }
  // how far the exponents move when the reference goes from o's to this one: not above 0 once there is any sum, and
  // finite, so that nothing is left of one and not a NaN
  __device__ __forceinline__ float down(const Exponent& o) const {
#pragma clang fp contract(off)
    return fmaxf(fminf(sizeof(T) == 2 ? o.b - b : (o.ref - ref) * c, 0.f), -1e25f);
  }
};
// A number that is the same in all lanes, as a scalar: not a register of each thread.
__device__ __forceinline__ float uniform(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
// e t with 0 where e is: tokens that cannot occur
__device__ __forceinline__ float entropy_term(float e, float t, float u) { return fmaf(e, fmaxf(t, -1e30f), u); }

// What a row's softmax needs.
template <typename T>
struct Stats {
  float m, inv_tau;   // maximum, 1 / tau
  Exponent<T> t;      // with reference m
  float S, inv, log_s;  // S, 1 / S, L; S = 0 where no token has any probability
  float entropy;
  __device__ __forceinline__ float log_p(float x) const {
    return S == 0.f ? -INFINITY : (x - m) * inv_tau - log_s;
  }
};

// Sum of c over the threads in front of this one; total: over all.
template <int NT>
__device__ __forceinline__ int scan_exclusive(int c, Shared<NT>& sh, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = c;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(s, d);
    s += lane >= d ? o : 0;
  }
  sync_row<NT>();
  if (lane == 63) sh.scan[wave] = s;
  sync_row<NT>();
  int front = 0;
  total = 0;
#pragma unroll 1
  for (int w = 0; w < Shared<NT>::W; ++w) {
    front += w < wave ? sh.scan[w] : 0;
    total += sh.scan[w];
  }
  return front + s - c;
}

// Maximum and sums of the row, in an order that depends on nothing but its place in memory and its length.  One pass:
// a thread takes its logits in groups of G chunks, of each first the maximum, which is then the reference of what it has
// summed (so that no exponent is above 0 and u never changes sign), and keeps the largest logit so far out of the sums:
// where a larger one comes, the old one goes in.  The groups' sums start while later groups are on their way.
// TOP: the maxima of 64 and of 256 groups of threads go to sh.groups and sh.many, a thread with a NaN as -infinity there
// (its other logits may reach what the groups' bound is, which holds without them); low: the least of the latter above
// -infinity; mine: this thread's maximum, NaN where it has met one.
struct Tops {
  float low, mine;
};
template <bool ENTROPY, bool TOP, typename T, int NT, int CH, bool OPEN>
__device__ __forceinline__ Stats<T> row_stats(Row<T, NT, CH, OPEN>& row, float tau, Shared<NT>& sh, Tops* tops = nullptr) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int W = Shared<NT>::W;
  constexpr int E = sizeof(T) == 2 ? 2 : 1;  // largest logits kept out: one for each half of a register
  typedef T Top __attribute__((ext_vector_type(E)));
  const float inv_tau = 1.0f / tau, c = kLog2e * inv_tau;
  Top top = Top((T)-INFINITY);
  top[0] = row.single;
  Exponent<T> t(c, -INFINITY);
  float s[E] = {}, u[E] = {};
  row.template groups<4>([&](const auto* v, int, auto n) {
    constexpr int N = RowVec<T>::N;
    Top most = top;
#pragma unroll
    for (int k = 0; k < n.value; ++k)
#pragma unroll
      for (int j = 0; j < N; j += E) {
        Top x;
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = v[k][j + i];
        most = most_of(most, x);
      }
    const Exponent<T> old = t;
    float ref = (float)most[0];
#pragma unroll
    for (int i = 1; i < E; ++i) ref = most_of(ref, (float)most[i]);
    t.at(ref);
    const float d = t.down(old), f = __builtin_amdgcn_exp2f(d);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if constexpr (ENTROPY) u[i] = fmaf(d, s[i], u[i]) * f;
      s[i] *= f;
    }
#pragma unroll
    for (int k = 0; k < n.value; ++k)
#pragma unroll
      for (int j = 0; j < N; j += E) {
        Top x;
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = v[k][j + i];
        const Top less = least_of(top, x);
        top = most_of(top, x);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float y = t((float)less[i]), e = __builtin_amdgcn_exp2f(y);
          s[i] += e;
          if constexpr (ENTROPY) u[i] = entropy_term(e, y, u[i]);
        }
      }
  });
  // the thread's: one largest logit, one sum (its reference may be that of no group at all)
  float mine = (float)top[0];
  {
    const Exponent<T> old = t;
    float less = -INFINITY;
    if constexpr (E == 2) {
      less = least_of(mine, (float)top[1]);
      mine = most_of(mine, (float)top[1]);
    }
    t.at(mine);
    const float d = t.down(old), f = __builtin_amdgcn_exp2f(d), y = t(less), e = __builtin_amdgcn_exp2f(y);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if constexpr (ENTROPY) u[i] = fmaf(d, s[i], u[i]) * f;
      s[i] *= f;
    }
    if constexpr (E == 2) {
      s[0] += s[1] + e;
      if constexpr (ENTROPY) u[0] = entropy_term(e, y, u[0] + u[1]);
    }
  }
  // of this lane's (largest, s, u) and others' whose largest is m: the sums for reference m, all but the first largest
  auto rebase = [&](float& s, float& u, const Exponent<T>& from, const Exponent<T>& to, float largest, bool first) {
    const float d = to.down(from), f = __builtin_amdgcn_exp2f(d);
    const float y = to(largest), e = __builtin_amdgcn_exp2f(y);
    if constexpr (ENTROPY) u = fmaf(d, s, u) * f;
    s *= f;
    if (!first) {
      s += e;
      if constexpr (ENTROPY) u = entropy_term(e, y, u);
    }
  };
  if constexpr (TOP) {
    tops->mine = mine;
    float g = fmaxf(mine, -INFINITY);
    constexpr int SMALL = NT >= 256 ? NT / 256 : 1, LANES = NT / 64;
    if constexpr (SMALL > 1) g = fmaxf(g, from_lane<1>(g));
    if constexpr (SMALL > 2) g = fmaxf(g, from_lane<2>(g));
    const float least = group_reduce<kWave>(g > -INFINITY ? g : INFINITY, [](float a, float b) { return fminf(a, b); });
    if (lane == 0) sh.low[wave] = least;
    if (NT >= 256 && lane % SMALL == 0) sh.many[threadIdx.x / SMALL] = g;
    if constexpr (SMALL == 1 && LANES > 1) g = fmaxf(g, from_lane<1>(g));
    if constexpr (SMALL <= 2 && LANES > 2) g = fmaxf(g, from_lane<2>(g));
    if constexpr (LANES > 4) g = fmaxf(g, from_lane<4>(g));
    if constexpr (LANES > 8) g = fmaxf(g, from_lane<8>(g));
    if (lane % LANES == 0) sh.groups[threadIdx.x / LANES] = g;
  }
  const float m_wave = group_reduce<kWave>(mine, [](float a, float b) { return most_of(a, b); });
  {
    Exponent<T> to(c, m_wave);
    const uint64_t largest = __ballot(mine == m_wave);
    rebase(s[0], u[0], t, to, mine, largest != 0 && lane == __ffsll((unsigned long long)largest) - 1);
  }
  s[0] = wave_sum(s[0]);
  if constexpr (ENTROPY) u[0] = wave_sum(u[0]);
  if (lane == 0) {
    sh.top[wave] = m_wave;
    sh.s[wave] = s[0];
    sh.u[wave] = u[0];
  }
  sync_row<NT>();
  const int w = lane % W;
  auto add = [](float a, float b) { return a + b; };
  mine = sh.top[w];
  if constexpr (TOP) tops->low = uniform(join<W>(sh.low[w], [](float a, float b) { return fminf(a, b); }));
  const float m = uniform(join<W>(mine, [](float a, float b) { return most_of(a, b); }));
  Stats<T> st = {m, uniform(inv_tau), Exponent<T>(uniform(c), m)};
  st.t.b = uniform(st.t.b);
  st.t.ref = uniform(st.t.ref);
  float sum = sh.s[w], terms = sh.u[w];
  const uint64_t largest = __ballot(mine == m);
  rebase(sum, terms, Exponent<T>(c, mine), st.t, mine, largest != 0 && w == __ffsll((unsigned long long)largest) - 1);
  sum = join<W>(sum, add);
  if constexpr (ENTROPY) terms = join<W>(terms, add);
  if (m == INFINITY) sum = NAN;
  const float d = st.t.rest(), one = __builtin_amdgcn_exp2f(d);
  if (m == -INFINITY) {
    st.S = st.inv = st.log_s = st.entropy = 0.f;
  } else {
    st.S = uniform(one + sum);
    st.inv = uniform(1.0f / st.S);
    st.log_s = uniform(log1pf(sum * __builtin_amdgcn_exp2f(-d)));
    st.entropy = ENTROPY ? uniform(st.log_s - kLn2 * fmaf(-d, sum, terms) * st.inv) : 0.f;
  }
  return st;
}

// Logits in their order as unsigned numbers (-0 as +0, NaN as -infinity), the lower index first among equal ones.
__device__ __forceinline__ uint64_t top_key(float x, int index) {
  const unsigned u = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
  const unsigned o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const unsigned o = (unsigned)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)(0xffffffffu - (unsigned)key); }

template <int NT>
struct TopShared {
  static constexpr int kKeep = NT == 64 ? 512 : 1024;
  static constexpr int kBins = 256;
  uint64_t kept[kKeep], fewer[kKeep];
  int bins[kBins], count, count_fewer, cut, threads;
  short thread[NT];
  __device__ __forceinline__ void clear() {  // in front of a barrier in front of row_top
    for (int i = threadIdx.x; i < kBins; i += NT) bins[i] = 0;
    if (threadIdx.x == 0) count = count_fewer = threads = 0;
  }
};

// The k-th largest of the lanes' numbers, or a little below it: its upper 18 bits, one by one from the top.
__device__ __forceinline__ float kth_of_lanes(float v, int k) {
  const unsigned key = (unsigned)(top_key(v, 0) >> 32);
  unsigned kth = 0;
#pragma unroll
  for (int bit = 31; bit >= 14; --bit) {
    const unsigned trial = kth | 1u << bit;
    if (__popcll(__ballot(key >= trial)) >= k) kth = trial;
  }
  return kth < 0x007fffffu ? -INFINITY : key_value((uint64_t)kth << 32);  // below -infinity's there are NaNs
}

// found(r, key) of the k largest logits, r = 0 .. k - 1 in any order, by one thread each.  A bound that at least k of
// them reach is the k-th largest of the maxima of some groups of threads: of 64 groups up to k = 32, of 256, by a
// histogram, beyond.  The logits that reach it are gathered, little more than k (some 24 for k = 20, 180 for 128), from
// memory, since a row's registers held any longer are too many: the chunks of the few threads whose maximum reaches it
// or is NaN, one a thread, or the whole row.  A histogram leaves of more than 256 those from the k-th's bin on, and the
// rest is ranked by counting.  2048 rows of 50257 fp16 logits, us: no top tokens 41, 1 41, 5 42, 20 46, 64 57, 128 80; 16384 of
// 300: none 16, 20 33, 128, for which a row has 256 threads and most groups nothing, 123.
template <typename T, int NT, int CH, bool OPEN, typename F>
__device__ __forceinline__ void row_top(const Row<T, NT, CH, OPEN>& row, int k, Tops tops, float high, TopShared<NT>& top,
                                        Shared<NT>& sh, F found) {
  constexpr int kKeep = TopShared<NT>::kKeep, kBins = TopShared<NT>::kBins, N = RowVec<T>::N;
  const int tid = threadIdx.x, lane = tid & 63;
  // Bins of n keys between those of `from` and `high`, lower ones in the first: the lowest bin in which one of the k
  // largest is.
  unsigned base = 0;
  int shift = 0;
  auto bin_of = [&](unsigned key) { return key <= base ? 0u : min((key - base) >> shift, kBins - 1u); };
  auto cut_bins = [&](int n, auto key_of, float from) {
    base = (unsigned)(top_key(from, 0) >> 32);
    const unsigned range = (unsigned)(top_key(high, 0) >> 32) - base;
    shift = max(0, 24 - __clz((int)(range | 1)));
    for (int i = tid; i < n; i += NT) atomicAdd(&top.bins[bin_of(key_of(i))], 1);
    sync_row<NT>();
    if (tid < kWave) {
      int c[kBins / kWave], sum = 0;  // this lane's bins, the highest values first
#pragma unroll
      for (int i = 0; i < kBins / kWave; ++i) {
        int& bin = top.bins[kBins - 1 - (lane * (kBins / kWave) + i)];
        sum += c[i] = bin;
        bin = 0;
      }
      int front = sum;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(front, d);
        front += lane >= d ? o : 0;
      }
      front -= sum;
#pragma unroll
      for (int i = 0; i < kBins / kWave; ++i) {
        if (front < k && front + c[i] >= k) top.cut = kBins - 1 - (lane * (kBins / kWave) + i);
        front += c[i];
      }
    }
    sync_row<NT>();
    return (unsigned)top.cut;
  };
  float low = -INFINITY;
  if (NT < 256 || k <= 32) {  // a wavefront's row has no more
    low = kth_of_lanes(sh.groups[lane], k);
  } else if (NT >= 256 && tops.low < INFINITY) {
    const unsigned cut = cut_bins(256, [&](int i) { return (unsigned)(top_key(sh.many[i], 0) >> 32); }, tops.low);
    if (cut > 0) low = key_value((uint64_t)(base + (cut << shift)) << 32);  // some in the first bin may be below its edge
  }
  auto put = [&](int at, float y, int index) {
    if (at < kKeep) top.kept[at] = top_key(y, index);
  };
  const Row<T, NT, 0, true> again = [&] {
    Row<T, NT, 0, true> r(row.x, row.vocab);
    r.single = row.single;
    return r;
  }();
  auto recount = [&](auto reaches) {
    sync_row<NT>();
    if (tid == 0) top.count = 0;
    sync_row<NT>();
    again.each([&](const auto& y, int first, auto n) {
      int c = 0;
#pragma unroll
      for (int j = 0; j < n.value; ++j) c += reaches(y[j]);
      if (first < 0) c = 0;
      if (c > 0) {
        int at = atomicAdd(&top.count, c);
#pragma unroll
        for (int j = 0; j < n.value; ++j)
          if (reaches(y[j])) put(at++, y[j], first + j);
      }
    });
    sync_row<NT>();
    return top.count;
  };
  auto above = [&](float y) { return y > low; };
  int n = kKeep + 1;  // all logits reach -infinity: not gathered
  if (low > -INFINITY) {
    const uint64_t in = __ballot(!(tops.mine < low));  // NaN: others of the thread may reach it
    if (in) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&top.threads, __popcll(in));
      at = __builtin_amdgcn_readfirstlane(at);
      if (in >> lane & 1) top.thread[at + __popcll(in & ((1ull << lane) - 1))] = (short)tid;
    }
    sync_row<NT>();
    const int threads = top.threads;
    const int units = (row.chunks + NT - 1) / NT + 1;  // of a thread: its chunks and its single element
    if (threads * units * N <= 32 * NT) {
      const float per = 1.0f / (float)units;
      for (int f = tid; f < threads * units; f += NT) {
        const int nth = (int)(((float)f + 0.5f) * per), e = f - nth * units, t = top.thread[nth], chunk = t + e * NT;
        if (e < units - 1) {
          const auto v = row.chunk(chunk);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float y = (float)v[j];
            if (y >= low) put(atomicAdd(&top.count, 1), y, row.lead + chunk * N + j);
          }
        } else if (t < row.vocab - row.chunks * N) {
          const int index = t < row.lead ? t : t + row.chunks * N;
          const float y = row.at(index);
          if (y >= low) put(atomicAdd(&top.count, 1), y, index);
        }
      }
      sync_row<NT>();
      n = top.count;
    } else {
      n = recount([&](float y) { return y >= low; });
    }
  }
  if (n > kKeep) {
    n = recount(above);
    if (n > kKeep) {
      // the k-th largest value, bit by bit from the top: the largest that at least k reach
      unsigned kth = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = kth | 1u << bit;
        int c = 0;
        again.each([&](const auto& y, int first, auto m) {
          if (m.value == 1 && first < 0) return;
#pragma unroll
          for (int j = 0; j < m.value; ++j) c += first + j < row.vocab && (unsigned)(top_key(y[j], 0) >> 32) >= trial;
        });
        int total;
        scan_exclusive<NT>(c, sh, total);
        if (total >= k) kth = trial;
      }
      low = key_value((uint64_t)kth << 32);
      n = recount(above);  // fewer than k
    }
    if (n < k) {
      // the first k - n of the logits that equal `low`, in the order of their indices
      auto take = [&](bool one, int first, int elements) {
        int c = 0, total;
        if (one)
          for (int j = 0; j < elements; ++j) c += fmaxf(row.at(first + j), -INFINITY) == low;
        int at = n + scan_exclusive<NT>(c, sh, total);
        if (one)
          for (int j = 0; j < elements; ++j)
            if (fmaxf(row.at(first + j), -INFINITY) == low) {
              if (at < k) top.kept[at] = top_key(row.at(first + j), first + j);
              ++at;
            }
        n += total;
      };
      take(tid < row.lead, tid, 1);
      for (int c = 0; c < row.chunks && n < k; c += NT) take(c + tid < row.chunks, row.lead + (c + tid) * N, N);
      if (n < k) take(row.loose >= row.lead, row.loose, 1);
      n = k;
      sync_row<NT>();
    }
  }
  const uint64_t* list = top.kept;
  if (n > 256) {
    const unsigned cut = cut_bins(n, [&](int i) { return (unsigned)(top.kept[i] >> 32); }, low);
    for (int i = tid; i < n; i += NT) {
      const uint64_t key = top.kept[i];
      if (bin_of((unsigned)(key >> 32)) >= cut) top.fewer[atomicAdd(&top.count_fewer, 1)] = key;
    }
    sync_row<NT>();
    n = top.count_fewer;
    list = top.fewer;
  }
  // 2^split threads for a key, each for a part of the others
  int split = 0;
  while (split < 4 && (n << (split + 1)) <= NT) ++split;
  const int parts = 1 << split, part = tid & (parts - 1);
#pragma unroll 1
  for (int i = tid >> split; i < ((n << split) + 63 & -64) >> split; i += NT >> split) {
    const uint64_t key = list[i < n ? i : 0];
    int rank = 0;
#pragma unroll 8
    for (int j = part; j < n; j += parts) rank += list[j] > key;
    if (parts > 1) rank += from_lane<1>(rank);
    if (parts > 2) rank += from_lane<2>(rank);
    if (parts > 4) rank += from_lane<4>(rank);
    if (parts > 8) rank += from_lane<8>(rank);
    if (i < n && part == 0 && rank < k) found(rank, key);
  }
}

template <typename T, bool TOP, int NT, int CH, bool OPEN, int WAVES>
__global__ __launch_bounds__(NT * kRowsOf<NT>, WAVES) void token_log_probs_kernel(
    const T* __restrict__ x, int64_t ld, int64_t rows, int vocab, const int64_t* __restrict__ tokens, float tau, int k,
    float* __restrict__ log_probs, float* __restrict__ entropy, float* __restrict__ top_log_probs,
    int64_t* __restrict__ top_tokens) {
  __shared__ Shared<NT> sh_of[kRowsOf<NT>];
  const int in_group = row_in_group<NT>();
  const int64_t r = row_of_group<NT>(in_group);
  if (r >= rows) return;
  Shared<NT>& sh = sh_of[in_group];
  Row<T, NT, CH, OPEN> row(x + r * ld, vocab);
  row.load();
  TopShared<NT>* top_shared = nullptr;
  if constexpr (TOP) {
    __shared__ TopShared<NT> top[kRowsOf<NT>];
    top_shared = top + in_group;
    top_shared->clear();
  }
  Tops tops;
  const Stats<T> st = row_stats<true, TOP>(row, tau, sh, &tops);
  if (log_probs != nullptr) {
    const int64_t t = tokens[r];
    const bool in = t >= 0 && t < vocab;
    const float score = st.log_p(row.at(in ? t : 0));
    if (threadIdx.x == 0) log_probs[r] = in ? score : 0.f;
  }
  if (entropy != nullptr && threadIdx.x == 0) entropy[r] = st.entropy;
  if constexpr (TOP)
    row_top(row, k, tops, st.m, *top_shared, sh, [&](int rank, uint64_t key) {
      top_log_probs[r * k + rank] = st.log_p(key_value(key));
      top_tokens[r * k + rank] = key_index(key);
    });
}

// Tokens of a row whose gradient has a part of its own: the token, its logit, its part, and the sum of the parts of all
// entries of that token; first[t] and next[i] chain the entries whose logits thread t has.
template <int NT>
struct Special {
  int id[kMaxTop + 1], next[kMaxTop + 1], first[NT];
  float x[kMaxTop + 1], add[kMaxTop + 1], total[kMaxTop + 1];
};

// The entries lane, lane + 64, .. of a row, by the first wavefront and for all behind the next barrier: f(i, token,
// part, logit) gives entry i, token -1 for none.
template <typename T, int NT, int CH, bool OPEN, typename F>
__device__ __forceinline__ void set_special(const Row<T, NT, CH, OPEN>& row, Special<NT>& sp, int count, F f) {
  const int lane = threadIdx.x;
  for (int t = lane; t < NT; t += kWave) sp.first[t] = -1;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int e = 0; e <= kMaxTop / kWave; ++e) {
    const int i = lane + e * kWave;
    if (i >= count) break;
    int64_t token = -1;
    float part = 0.f, x = 0.f;
    f(e, i, token, part, x);
    const bool in = token >= 0 && token < row.vocab;
    const int id = in ? (int)token : -1, behind = id - row.lead;
    sp.id[i] = id;
    sp.add[i] = in ? part : 0.f;
    sp.x[i] = x;
    if (in) {
      const int owner = behind < 0 ? id : behind < row.chunks * row.N ? behind / row.N % NT : id - row.chunks * row.N;
      sp.next[i] = atomicExch(&sp.first[owner], i);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int i = lane; i < count; i += kWave) {
    const int id = sp.id[i];
    float sum = 0.f;
#pragma unroll 8
    for (int j = 0; j < count; ++j) sum += sp.id[j] == id ? sp.add[j] : 0.f;
    sp.total[i] = sum;
  }
}

// STREAM: past the caches.  (Not as a condition at the store, which the compiler makes one plain store of.)
template <bool STREAM, typename V>
__device__ __forceinline__ void store_chunk(V* at, V v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, at);
  else *at = v;
}

// Writes f(x_j) of every logit of the row, and of the special ones' f(x) + scale total: over what was written, by the thread
// that wrote it, so that nothing has to be waited for.  Entries of one token write one number.
template <typename T, int NT, int CH, bool OPEN, typename F>
__device__ __forceinline__ void write_gradient(Row<T, NT, CH, OPEN>& row, T* __restrict__ out, const Special<NT>& sp,
                                               bool special, float scale, bool stream, F f) {
  typedef typename RowVec<T>::V V;
  const bool whole = ((uintptr_t)out & 15) == ((uintptr_t)row.x & 15);
  row.renew();
  auto write = [&](auto past) {
    row.each([&](const auto& y, int first, auto n) {
      if constexpr (n.value > 1) {
        if (first >= row.lead + row.chunks * n.value) return;
        V v;
#pragma unroll
        for (int j = 0; j < n.value; ++j) v[j] = (T)f(y[j]);
        if (whole) {
          store_chunk<decltype(past)::value>(reinterpret_cast<V*>(out + first), v);
        } else {
#pragma unroll
          for (int j = 0; j < n.value; ++j) out[first + j] = v[j];
        }
      } else if (first >= 0) {
        out[first] = (T)f(y[0]);
      }
    });
  };
  if (OPEN || stream) write(std::true_type{});  // what is read again here stays in the L2
  else write(std::false_type{});
  asm volatile("" ::: "memory");
  if (special)
    for (int i = sp.first[threadIdx.x]; i >= 0; i = sp.next[i]) out[sp.id[i]] = (T)fmaf(scale, sp.total[i], f(sp.x[i]));
}

template <typename T, int NT>
__device__ __forceinline__ void write_zeros(T* __restrict__ out, int vocab, bool stream) {
  const Row<T, NT, 0, true> row(out, vocab);
  typedef typename RowVec<T>::V V;
  auto write = [&](auto past) {
    for (int c = threadIdx.x; c < row.chunks; c += NT)
      store_chunk<decltype(past)::value>(reinterpret_cast<V*>(out + row.lead) + c, V(0));
  };
  if (stream) write(std::true_type{});
  else write(std::false_type{});
  if (row.loose >= 0) out[row.loose] = (T)0;
}

// dx_j = ([j = token] g + sum_i u_i [j = id_i] - p_j (g + sum_i u_i + h (log p_j + H))) / tau for the gradients g of
// log p(token), h of the entropy and u_i of the top tokens' log probabilities.
template <typename T, int NT, int CH, bool OPEN, int WAVES>
__global__ __launch_bounds__(NT * kRowsOf<NT>, WAVES) void token_log_probs_backward_kernel(
    const T* __restrict__ x, int64_t ld, int64_t rows, int vocab, const int64_t* __restrict__ tokens, float tau,
    RowGradient d_log_probs, RowGradient d_entropy, int k, const int64_t* __restrict__ top_tokens,
    const float* __restrict__ d_top, T* __restrict__ out, int64_t ld_out, bool stream) {
  __shared__ Shared<NT> sh_of[kRowsOf<NT>];
  __shared__ Special<NT> sp_of[kRowsOf<NT>];
  const int in_group = row_in_group<NT>();
  const int64_t r = rows - 1 - row_of_group<NT>(in_group);  // the last first: the forward pass read them last
  if (r < 0) return;
  Shared<NT>& sh = sh_of[in_group];
  Special<NT>& sp = sp_of[in_group];
  const int count = k + 1;
  Row<T, NT, CH, OPEN> row(x + r * ld, vocab);
  // Where the condition is the same for all threads, and not in a thread's branch below: a load from one address is
  // a scalar one, which a wavefront executes in a branch that none of its lanes takes.
  int64_t token = -1;
  float d_token = 0.f, h = 0.f;
  if (d_log_probs.d != nullptr) {
    token = tokens[r];
    d_token = d_log_probs.d[r * d_log_probs.pitch];
  }
  if (d_entropy.d != nullptr) h = d_entropy.d[r * d_entropy.pitch];
  if (threadIdx.x < kWave)
    set_special(row, sp, count, [&](int, int i, int64_t& t, float& part, float& logit) {
      t = token;
      part = d_token;
      if (i < k) {
        t = top_tokens[r * k + i];
        part = d_top[r * k + i];
      }
      if (t >= 0 && t < vocab) logit = row.at(t);
    });
  sync_row<NT>();
  float g = 0.f;
  bool none = true;
#pragma unroll 8
  for (int i = 0; i < count; ++i) {
    g += sp.add[i];
    none &= sp.add[i] == 0.f;
  }
  g = uniform(g);
  T* o = out + r * ld_out;
  if (none && h == 0.f) {  // padding: whatever its logits are
    write_zeros<T, NT>(o, vocab, stream);
    return;
  }
  row.load();
  const Stats<T> st = row_stats<true, false>(row, tau, sh);
  const float scale = uniform(st.inv * st.inv_tau), lift = uniform(st.entropy - st.log_s - kLn2 * st.t.rest());
  write_gradient(row, o, sp, st.S != 0.f, st.inv_tau, stream, [&](float y) {
    const float t = st.t(y), p = __builtin_amdgcn_exp2f(t) * scale;
    // an exponent below -200 is as good as -200, where p is 0: h times an infinite one would make a NaN of that 0
    return -p * fmaf(h, fmaf(kLn2, fmaxf(t, -200.f), lift), g);
  });
}

// A row's entries: a register each of all wavefronts otherwise.  total: 1, or 0 where there are none.
struct Entries {
  float q[kMaxTop], log_q[kMaxTop], x[kMaxTop], total;
};

// q = softmax(teacher / tau) over the row's entries (an id outside the vocabulary is no entry), loss = w sum q (log q -
// log p); gradient w / tau (p_j - sum of q over the entries of token j).
template <typename T, bool GRAD, int NT, int CH, bool OPEN, int WAVES>
__global__ __launch_bounds__(NT * kRowsOf<NT>, WAVES) void distillation_kernel(
    const T* __restrict__ x, int64_t ld, int64_t rows, int vocab, const int64_t* __restrict__ teacher_tokens,
    const void* __restrict__ teacher, int teacher_f16, int k, float tau, const float* __restrict__ weights,
    RowGradient d_losses, float* __restrict__ losses, T* __restrict__ out, int64_t ld_out, bool stream) {
  __shared__ Shared<NT> sh_of[kRowsOf<NT>];
  __shared__ Special<NT> sp_of[kRowsOf<NT>];
  __shared__ Entries entries_of[kRowsOf<NT>];
  const int in_group = row_in_group<NT>();
  int64_t r = row_of_group<NT>(in_group);
  if (GRAD && losses == nullptr) r = rows - 1 - r;  // as in the gradient above
  if (r < 0 || r >= rows) return;
  Shared<NT>& sh = sh_of[in_group];
  Special<NT>& sp = sp_of[in_group];
  Entries& entries = entries_of[in_group];
  const int tid = threadIdx.x;
  const float w = weights != nullptr ? weights[r] : 1.f;
  float w_grad = w;
  if (d_losses.d != nullptr) w_grad = uniform(w * d_losses.d[r * d_losses.pitch]);
  if (w == 0.f || (losses == nullptr && w_grad == 0.f)) {  // padding: whatever its logits are
    if (tid == 0 && losses != nullptr) losses[r] = 0.f;
    if constexpr (GRAD) write_zeros<T, NT>(out + r * ld_out, vocab, stream);
    return;
  }
  Row<T, NT, CH, OPEN> row(x + r * ld, vocab);
  constexpr int E = kMaxTop / kWave;  // a lane's entries, for the first wavefront
  float q[E], log_q[E], student[E];
  // the entries and their logits are requested first, and worked on while the row is on its way
  int64_t entry[E];
  if (tid < kWave) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int at = tid + i * kWave;
      entry[i] = -1;
      log_q[i] = -INFINITY;
      if (at < k) {
        entry[i] = teacher_tokens[r * k + at];
        log_q[i] = teacher_f16 ? (float)((const _Float16*)teacher)[r * k + at] : ((const float*)teacher)[r * k + at];
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      student[i] = 0.f;
      if (entry[i] >= 0 && entry[i] < vocab) student[i] = row.at(entry[i]);
    }
  }
  row.load();
  if (tid < kWave) {
    const float inv_tau = 1.0f / tau;
    float most = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (entry[i] < 0 || entry[i] >= vocab) log_q[i] = -INFINITY;
      most = fmaxf(most, log_q[i]);
    }
    most = wave_max(most);
    if (most == -INFINITY) most = 0.f;  // no entry: q = 0
#pragma unroll
    for (int i = 0; i < E; ++i) {
      log_q[i] = (log_q[i] - most) * inv_tau;  // in this order: finite, however small tau is
      q[i] = expf(log_q[i]);
      sum += q[i];
    }
    sum = wave_sum(sum);
    const float log_sum = logf(sum), inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      q[i] *= inv;
      entries.q[tid + i * kWave] = q[i];
      entries.log_q[tid + i * kWave] = log_q[i] - log_sum;
      entries.x[tid + i * kWave] = student[i];
    }
    if (tid == 0) entries.total = sum == 0.f ? 0.f : 1.f;
    if constexpr (GRAD)
      set_special(row, sp, k, [&](int e, int, int64_t& token, float& part, float& logit) {
        if (e >= E) return;
        token = entry[e];
        part = -q[e];
        logit = student[e];
      });
  }
  const Stats<T> st = row_stats<false, false>(row, tau, sh);
  if (tid < kWave && losses != nullptr) {
    float loss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int at = tid + i * kWave;
      loss += entries.q[at] == 0.f ? 0.f : entries.q[at] * (entries.log_q[at] - st.log_p(entries.x[at]));
    }
    loss = wave_sum(loss);
    if (tid == 0) losses[r] = entries.total == 0.f ? 0.f : w * loss;
  }
  if constexpr (GRAD) {
    if (uniform(entries.total) == 0.f) {  // no entries: whatever the row's logits are, which a factor of 0 is not
      write_zeros<T, NT>(out + r * ld_out, vocab, stream);
      return;
    }
    const float scale = uniform(w_grad * st.inv * st.inv_tau);
    write_gradient(row, out + r * ld_out, sp, st.S != 0.f, w_grad * st.inv_tau, stream,
                   [&](float y) { return __builtin_amdgcn_exp2f(st.t(y)) * scale; });
  }
}

// f(threads, chunks a thread, wavefronts a SIMD) as integral constants for rows of this many chunks.  A row takes 4 CH
// registers a thread and some 26 more, so few threads with long parts keep the most rows on a CU: of 50257 fp16 logits
// (6283 chunks) 3 with 512 threads, 4 with 256, 2 with 1024; 1477 rows scored 31 / 32 / 38 us, with their top 20 37 /
// 41 / 43; of 50304 fp32 logits (12576 chunks), forward and backward of 2048 rows 216 with 512 threads, 225 with 1024,
// loss and gradient of 4096 324 and 427.  WIDE, for a loss' gradient, whose stores are what it waits for: 1024 threads
// where a thread then has up to 8 chunks; 2048 rows of 50257 fp16 logits 512 / 1024 threads 85 / 78, with the loss 90 /
// 83, of 65024 102 / 99 and 108 / 105, of 32000 fp32 99 / 97 and 105 / 102, but the gradient of log probabilities 86 /
// 90.  Rows of up to 256 chunks have a wavefront each, four a workgroup; the longest, beyond 20480 chunks, are read
// again behind those.  min_threads: what the call needs.
template <bool WIDE, typename F>
void pick(int chunks, int min_threads, F f) {
#define GPTMI_ROW(NT, CH, OPEN, WAVES)                                                                        \
  if (NT >= min_threads && (OPEN || chunks <= NT * CH))                                                       \
    return f(std::integral_constant<int, NT>(), std::integral_constant<int, CH>(), std::integral_constant<bool, OPEN>(), \
             std::integral_constant<int, WAVES>())
  GPTMI_ROW(64, 4, false, 4);
  GPTMI_ROW(256, 4, false, 4);
  GPTMI_ROW(256, 8, false, 4);
  GPTMI_ROW(512, 8, false, 4);
  if constexpr (WIDE) {
    GPTMI_ROW(1024, 8, false, 8);
  } else {
    GPTMI_ROW(512, 13, false, 6);
    GPTMI_ROW(512, 16, false, 4);
  }
  GPTMI_ROW(512, 25, false, 4);
  GPTMI_ROW(1024, 16, false, 4);
  GPTMI_ROW(1024, 20, true, 4);
#undef GPTMI_ROW
}

template <bool WIDE, typename F>
void pick_row(const LogitRows& a, int min_threads, F f) {
  if (a.f16)
    pick<WIDE>(a.vocab / 8, min_threads, [&](auto nt, auto ch, auto open, auto waves) { f(_Float16(), nt, ch, open, waves); });
  else
    pick<WIDE>(a.vocab / 4, min_threads, [&](auto nt, auto ch, auto open, auto waves) { f(float(), nt, ch, open, waves); });
}

template <int NT>
dim3 grid_of(const LogitRows& a) {
  const int64_t n = (a.rows + kRowsOf<NT> - 1) / kRowsOf<NT>;
  return dim3((unsigned)(n < kGridRow ? n : kGridRow), (unsigned)((n + kGridRow - 1) / kGridRow));
}
// A gradient goes past the caches where it would push out the logits that the forward pass left in the memory-side
// cache of 256 MB, whose last rows a backward pass therefore takes first, and a one-pass gradient where it would not
// stay there itself (what waits there for its way to memory is written while the next kernel reads); always where rows
// are so long that they are read again.  us, without / with, 50304 logits: forward and backward of 1024 fp32 rows (206
// MB) 129 / 115, with a sum that reads the gradient 171 / 167, of 2048 246 / 216 and 329 / 326 (the first rows first
// 250 and 342), of 768 rows (155 MB) with the sum 126 / 131; one pass of 2048 fp16 rows (206 MB) 89 / 84, but with the
// sum 139 / 149, of 1536 fp32 rows (309 MB) 129 / 121 and 210 / 207; of 512 rows of 128256 fp32 logits 129 / 108.
constexpr int64_t kStreamBehindForward = 192 << 20, kStreamOnePass = 256 << 20;
int64_t gradient_bytes(const LogitRows& a) { return a.rows * a.vocab * (a.f16 ? 2 : 4); }

template <int NT>
dim3 block_of() { return dim3(NT, kRowsOf<NT>); }

}  // namespace

void launch_token_log_probs(const LogitRows& a, const int64_t* tokens, int top, float* log_probs, float* entropy,
                            float* top_log_probs, int64_t* top_tokens, hipStream_t st) {
  // a wavefront has 64 groups to bound the top tokens with: no more than 32 of them
  pick_row<false>(a, top > 32 ? 256 : 0, [&](auto type, auto nt, auto ch, auto open, auto waves) {
    typedef decltype(type) T;
    auto kernel = top > 0 ? token_log_probs_kernel<T, true, nt.value, ch.value, open.value, waves.value>
                          : token_log_probs_kernel<T, false, nt.value, ch.value, open.value, waves.value>;
    hipLaunchKernelGGL(kernel, grid_of<nt.value>(a), block_of<nt.value>(), 0, st, (const T*)a.x, a.ld, a.rows, a.vocab,
                       tokens, a.temperature, top, log_probs, entropy, top_log_probs, top_tokens);
  });
}

void launch_token_log_probs_backward(const LogitRows& a, const int64_t* tokens, RowGradient d_log_probs,
                                     RowGradient d_entropy, int top, const int64_t* top_tokens, const float* d_top,
                                     void* grad, int64_t ld_grad, hipStream_t st) {
  const bool stream = gradient_bytes(a) > kStreamBehindForward;
  pick_row<false>(a, 0, [&](auto type, auto nt, auto ch, auto open, auto waves) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((token_log_probs_backward_kernel<T, nt.value, ch.value, open.value, waves.value>),
                       grid_of<nt.value>(a), block_of<nt.value>(), 0, st, (const T*)a.x, a.ld, a.rows, a.vocab, tokens,
                       a.temperature, d_log_probs, d_entropy, top, top_tokens, d_top, (T*)grad, ld_grad, stream);
  });
}

void launch_distillation(const LogitRows& a, const int64_t* teacher_tokens, const void* teacher, bool teacher_f16,
                         int k, const float* weights, RowGradient d_losses, float* losses, void* grad, int64_t ld_grad,
                         hipStream_t st) {
  const bool stream = gradient_bytes(a) > (losses == nullptr ? kStreamBehindForward : kStreamOnePass);
  const auto launch = [&](auto gradient) {
    pick_row<gradient.value>(a, 0, [&](auto type, auto nt, auto ch, auto open, auto waves) {
      typedef decltype(type) T;
      hipLaunchKernelGGL((distillation_kernel<T, gradient.value, nt.value, ch.value, open.value, waves.value>),
                         grid_of<nt.value>(a), block_of<nt.value>(), 0, st, (const T*)a.x, a.ld, a.rows, a.vocab,
                         teacher_tokens, teacher, (int)teacher_f16, k, a.temperature, weights, d_losses, losses, (T*)grad,
                         ld_grad, stream);
    });
  };
  if (grad != nullptr) launch(std::true_type{});
  else launch(std::false_type{});
}

}  // namespace gptmi
