// The norm of many gradients together, and the gradients at that norm or at a limit: norm = scale |g| over all elements of all
// tensors, out = scale min(1, limit / norm) g.
//
// Squares are summed in 64 bits, which vector units do at the rate of 32: no square is too large or too small, and the norm does
// not depend on how the tensors are divided but for its last bits.  Two launches for each kTensors tensors: workgroups' sums over their
// chunks, each in one order; then every workgroup adds all workgroups' sums (1024 numbers a launch, from the L2; kJoin) in one order and
// scales its chunks, the last first, which the memory-side cache still has.  Bound by memory: 148 tensors of a 124M model in fp32 (498 MB), below the limit,
// 93 us, 5.4 TB/s; 355M elements from fp16 to fp32, 589 us, the squares at 4.3 TB/s and the scaling at 5.0.
#include "common.h"
#include "launch.h"

namespace gptmi {
namespace {

constexpr int kTensors = 152;    // of one launch: what kernel arguments, 4 KB, have room for (a model of 12 layers has 148)
constexpr int kBlocks = 1024;    // workgroups of one launch at most
// More workgroups' sums than these are added by a launch of their own, else by every workgroup that scales, work that grows with
// the square of the launches.  us in a graph, fp32 in place, with that launch / without: 304 tensors of 110000 elements (2048 sums) 55 / 55,
// 608 102 / 107, 2432 443 / 549, 6000 1084 / 1759; 60000 of 100 2440 / 5190.
constexpr unsigned kJoin = 2 * kBlocks;
constexpr int kThreads = 256;
constexpr int kGroups = 8;       // of 8 elements a thread at a time
constexpr int64_t kChunk = kThreads * 8 * kGroups;  // elements

struct ClipArgs {
  const void* in[kTensors];
  void* out[kTensors];
  unsigned first[kTensors];     // this launch's first chunk of each
  unsigned size_low[kTensors];
  uint16_t size_high[kTensors];  // of the elements; and bit 14: in is fp16, bit 15: out is
  int tensors;
  bool in_place;                // all of them
  unsigned chunks, before;     // of this launch; sums of the launches in front
  double* sums;                // of all launches' workgroups
  unsigned all;                // of them
  float* norm;
  float scale, limit;
};
static_assert(sizeof(ClipArgs) <= 4096, "kernel arguments");
constexpr int kInHalf = 1, kOutHalf = 2;
__device__ __forceinline__ int types_of(const ClipArgs& a, int tensor) { return a.size_high[tensor] >> 14; }
__device__ __forceinline__ int64_t size_of(const ClipArgs& a, int tensor) {
  return (int64_t)(a.size_high[tensor] & 0x3fff) << 32 | a.size_low[tensor];
}

// Elements in front of the first that lies at a multiple of 16 bytes.
__host__ __device__ __forceinline__ int ragged(const void* p, bool f16, int64_t n) {
  const int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (f16 ? 2 : 4);
  return head < n ? head : (int)n;
}

// Chunk after chunk, in either direction: which tensor it is of, where its elements begin, at a multiple of 16 bytes, how many
// they are, and how many of the tensor lie in front of its first chunk.
struct Cursor {
  int tensor, count, front;
  int64_t begin;
  __device__ __forceinline__ explicit Cursor(const ClipArgs& a, unsigned chunk) {
    int low = 0, high = a.tensors;
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (a.first[mid] <= chunk) low = mid;
      else high = mid;
    }
    tensor = low;
    at(a, chunk);
  }
  __device__ __forceinline__ void at(const ClipArgs& a, unsigned chunk) {
    while (tensor + 1 < a.tensors && a.first[tensor + 1] <= chunk) ++tensor;
    while (a.first[tensor] > chunk) --tensor;
    const int64_t size = size_of(a, tensor);
    const int head = ragged(a.in[tensor], types_of(a, tensor) & kInHalf, size);
    begin = (int64_t)(chunk - a.first[tensor]) * kChunk + head;
    count = (int)min(kChunk, size - begin);
    front = chunk == a.first[tensor] ? head : 0;
  }
};

typedef float f8 __attribute__((ext_vector_type(8)));
template <typename T>
__device__ __forceinline__ f8 load8(const T* p) {
  typedef T V __attribute__((ext_vector_type(8)));
  return __builtin_convertvector(*reinterpret_cast<const V*>(p), f8);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, f8 x) {
  typedef T V __attribute__((ext_vector_type(8)));
  *reinterpret_cast<V*>(p) = __builtin_convertvector(x, V);
}

__device__ __forceinline__ double sum_of(double x, double* lds) {  // of the workgroup, in every thread
#pragma unroll
  for (int step = 32; step > 0; step /= 2) x += __shfl_xor(x, step);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename T>
__device__ __forceinline__ double squares(const T* p, int n, int front) {
  const int tid = threadIdx.x, groups = n / 8;
  double sum = 0.0;
  const auto add = [&](f8 x) {
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fma((double)x[k], (double)x[k], sum);
  };
  const auto add_one = [&](float x) { sum = fma((double)x, (double)x, sum); };
  if (n == kChunk) {
    f8 x[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) x[j] = load8(p + (tid + j * kThreads) * 8);
#pragma unroll
    for (int j = 0; j < kGroups; ++j) add(x[j]);
  } else {
    for (int i = tid; i < groups; i += kThreads) add(load8(p + i * 8));
    if (tid < n - groups * 8) add_one((float)p[groups * 8 + tid]);
  }
  if (tid < front) add_one((float)p[tid - front]);
  return sum;
}

__global__ __launch_bounds__(kThreads) void grad_squares_kernel(ClipArgs a) {
  __shared__ double lds[4];
  double sum = 0.0;
  Cursor cursor(a, blockIdx.x);
  for (unsigned chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    cursor.at(a, chunk);
    const void* in = a.in[cursor.tensor];
    sum += types_of(a, cursor.tensor) & kInHalf ? squares((const _Float16*)in + cursor.begin, cursor.count, cursor.front)
                                    : squares((const float*)in + cursor.begin, cursor.count, cursor.front);
  }
  sum = sum_of(sum, lds);
  if (threadIdx.x == 0) a.sums[a.before + blockIdx.x] = sum;
}

// x times a factor, in two steps where it is one that fp32 would round as a subnormal number.
struct Factor {
  float first, second;
  __device__ __forceinline__ explicit Factor(double by)
      : first((float)(by < 0x1p-100 ? by * 0x1p64 : by)), second(by < 0x1p-100 ? 0x1p-64f : 1.f) {}
  template <typename V>
  __device__ __forceinline__ V operator()(V x) const { return x * first * second; }
};

template <typename S, typename T>
__device__ __forceinline__ void scaled(const S* in, T* out, int n, int front, Factor by) {
  const int tid = threadIdx.x, groups = n / 8;
  if (tid < front) out[tid - front] = (T)by((float)in[tid - front]);
  if (((uintptr_t)out & 15) != 0) {  // aligned differently
    for (int i = tid; i < n; i += kThreads) out[i] = (T)by((float)in[i]);
  } else if (n == kChunk) {
    f8 x[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) x[j] = load8(in + (tid + j * kThreads) * 8);
#pragma unroll
    for (int j = 0; j < kGroups; ++j) store8(out + (tid + j * kThreads) * 8, by(x[j]));
  } else {
    for (int i = tid; i < groups; i += kThreads) store8(out + i * 8, by(load8(in + i * 8)));
    if (tid < n - groups * 8) out[groups * 8 + tid] = (T)by((float)in[groups * 8 + tid]);
  }
}

__device__ __forceinline__ double sum_of_all(const double* sums, unsigned all, double* lds) {
  double sum = 0.0;
#pragma unroll 8
  for (unsigned i = threadIdx.x; i < all; i += kThreads) sum += sums[i];
  return sum_of(sum, lds);
}

// The sum of all workgroups' in the first one's place, by one workgroup.
__global__ __launch_bounds__(kThreads) void grad_join_kernel(double* sums, unsigned all) {
  __shared__ double lds[4];
  const double sum = sum_of_all(sums, all, lds);  // behind a barrier: all have been read
  if (threadIdx.x == 0) sums[0] = sum;
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(ClipArgs a) {
  __shared__ double lds[4];
  const double sum = sum_of_all(a.sums, a.all, lds);
  const double norm = (double)a.scale * sqrt(sum);
  if (blockIdx.x == 0 && a.before == 0 && threadIdx.x == 0) *a.norm = (float)norm;
  if (a.chunks == 0) return;
  // a NaN is passed on, and an infinite norm leaves 0 or NaN whatever the limit is
  const Factor by((double)a.scale * (norm <= (double)a.limit && norm < (double)INFINITY ? 1.0 : (double)a.limit / norm));
  const bool same = by.first == 1.f;
  if (same && a.in_place) return;
  Cursor cursor(a, a.chunks - 1 - blockIdx.x);
  for (unsigned i = blockIdx.x; i < a.chunks; i += gridDim.x) {
    cursor.at(a, a.chunks - 1 - i);
    const void* in = a.in[cursor.tensor];
    void* out = a.out[cursor.tensor];
    if (in == out && same) continue;
    const int64_t at = cursor.begin;
    const int n = cursor.count, front = cursor.front;
    switch (types_of(a, cursor.tensor)) {
      case 0: scaled((const float*)in + at, (float*)out + at, n, front, by); break;
      case kInHalf: scaled((const _Float16*)in + at, (float*)out + at, n, front, by); break;
      case kOutHalf: scaled((const float*)in + at, (_Float16*)out + at, n, front, by); break;
      default: scaled((const _Float16*)in + at, (_Float16*)out + at, n, front, by); break;
    }
  }
}

}  // namespace

// The sums of the launches' workgroups: no more than a launch has, nor than there are chunks.
size_t clip_grad_bytes(int64_t tensors) { return (size_t)((tensors + kTensors - 1) / kTensors) * kBlocks * sizeof(double); }

void launch_clip_grad_norm(const Gradients& g, float scale, float limit, float* norm, void* workspace, hipStream_t st) {
  ClipArgs a;
  a.sums = (double*)workspace;
  a.all = 0;
  a.in_place = g.in_place;
  a.norm = norm;
  a.scale = scale;
  a.limit = limit;
  const bool nothing = g.in_place && scale == 1.f && limit == INFINITY;  // the norm alone
  for (int scale_them = 0; scale_them < 2; ++scale_them) {
    if (scale_them && (nothing || a.all == 0)) {
      a.tensors = 0;
      a.chunks = a.before = 0;
      hipLaunchKernelGGL(grad_scale_kernel, dim3(1), dim3(kThreads), 0, st, a);
      break;
    }
    if (scale_them && a.all > kJoin) {
      hipLaunchKernelGGL(grad_join_kernel, dim3(1), dim3(kThreads), 0, st, a.sums, a.all);
      a.all = 1;
    }
    int64_t next = 0;
    a.before = 0;
    while (next < g.tensors) {
      a.tensors = 0;
      int64_t chunks = 0;
      for (; next < g.tensors && a.tensors < kTensors; ++next) {
        if (g.sizes[next] == 0) continue;
        const int64_t aligned = g.sizes[next] - ragged(g.in[next], g.in_f16[next] != 0, g.sizes[next]);
        const int64_t more = aligned <= kChunk ? 1 : (aligned + kChunk - 1) / kChunk;
        const int n = a.tensors++;
        a.in[n] = g.in[next];
        a.out[n] = g.out[next];
        a.size_low[n] = (unsigned)g.sizes[next];
        a.size_high[n] = (uint16_t)(g.sizes[next] >> 32 | (int64_t)((g.in_f16[next] ? kInHalf : 0) | (g.out_f16[next] ? kOutHalf : 0)) << 14);
        a.first[n] = (unsigned)chunks;
        chunks += more;
      }
      if (chunks == 0) continue;
      a.chunks = (unsigned)chunks;
      const unsigned blocks = chunks < kBlocks ? (unsigned)chunks : kBlocks;
      if (scale_them) {
        hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kThreads), 0, st, a);
      } else {
        hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(kThreads), 0, st, a);
        a.all += blocks;
      }
      a.before += blocks;
    }
  }
}

}  // namespace gptmi
