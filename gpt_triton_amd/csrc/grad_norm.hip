// The norm of many gradients together, and the gradients at that norm or at a limit: norm = scale |g| over all elements of all
// tensors, out = scale min(1, limit / norm) g.
//
// Squares are summed in 64 bits, which vector units do at the rate of 32: no square is too large or too small, and the norm does
// not depend on how the tensors are divided but for its last bits.  Two launches for each kTensors tensors: chunks' sums, in an order
// of their own each; then every workgroup adds all chunks' sums (some 2000 numbers from the L2) in one order and scales its chunk,
// the last first, which the memory-side cache still has.  Bound by memory.
#include "common.h"
#include "launch.h"

namespace gptmi {
namespace {

constexpr int kTensors = 112;   // of one launch: what kernel arguments, 4 KB, have room for
constexpr int kChunks = 2048;   // of all tensors, and one more each
constexpr int kThreads = 256;

struct ClipArgs {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t size[kTensors];
  unsigned first[kTensors];    // this launch's first chunk of each
  unsigned char f16[kTensors];  // 1: in, 2: out
  int tensors;
  unsigned chunks, before;     // of this launch, of the launches in front
  int64_t chunk;               // elements, a multiple of 8
  double* sums;                // of all chunks
  unsigned all;                // chunks of all launches
  float* norm;
  float scale, limit;
};

struct Piece {
  int tensor;
  int64_t begin, count;
};
__device__ __forceinline__ Piece piece_of(const ClipArgs& a, unsigned chunk) {
  int low = 0, high = a.tensors;
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (a.first[mid] <= chunk) low = mid;
    else high = mid;
  }
  const int64_t begin = (int64_t)(chunk - a.first[low]) * a.chunk;
  return {low, begin, min(a.chunk, a.size[low] - begin)};
}

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

// Elements in front of the first that lies at a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ int64_t ragged(const T* p, int64_t n) {
  const int64_t head = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (int64_t)sizeof(T);
  return min(head, n);
}

__device__ __forceinline__ double sum_of(double x, double* lds) {  // of the workgroup, in every thread
#pragma unroll
  for (int step = 32; step > 0; step /= 2) x += __shfl_xor(x, step);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename T>
__device__ __forceinline__ double squares(const T* p, int64_t n) {
  const int tid = threadIdx.x;
  const int64_t head = ragged(p, n), groups = (n - head) / 8, tail = head + groups * 8;
  double sum = 0.0;
  const auto add = [&](float x) { sum = fma((double)x, (double)x, sum); };
  if (tid < head) add((float)p[tid]);
  if (tid < n - tail) add((float)p[tail + tid]);
  p += head;
  constexpr int U = 4;
  int64_t i = tid;
  for (; i + (U - 1) * kThreads < groups; i += U * kThreads) {
    f8 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = load8(p + (i + j * kThreads) * 8);
#pragma unroll
    for (int j = 0; j < U; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) add(x[j][k]);
  }
  for (; i < groups; i += kThreads) {
    const f8 x = load8(p + i * 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) add(x[k]);
  }
  return sum;
}

__global__ __launch_bounds__(kThreads) void grad_squares_kernel(ClipArgs a) {
  __shared__ double lds[4];
  const Piece piece = piece_of(a, blockIdx.x);
  const void* in = a.in[piece.tensor];
  const double sum = sum_of(a.f16[piece.tensor] & 1 ? squares((const _Float16*)in + piece.begin, piece.count)
                                                    : squares((const float*)in + piece.begin, piece.count), lds);
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
__device__ __forceinline__ void scaled(const S* in, T* out, int64_t n, Factor by) {
  const int tid = threadIdx.x;
  const int64_t head = ragged(in, n);
  if (((uintptr_t)(out + head) & 15) != 0) {  // aligned differently
    for (int64_t i = tid; i < n; i += kThreads) out[i] = (T)by((float)in[i]);
    return;
  }
  const int64_t groups = (n - head) / 8, tail = head + groups * 8;
  if (tid < head) out[tid] = (T)by((float)in[tid]);
  if (tid < n - tail) out[tail + tid] = (T)by((float)in[tail + tid]);
  in += head;
  out += head;
  constexpr int U = 4;
  int64_t i = tid;
  for (; i + (U - 1) * kThreads < groups; i += U * kThreads) {
    f8 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = load8(in + (i + j * kThreads) * 8);
#pragma unroll
    for (int j = 0; j < U; ++j) store8(out + (i + j * kThreads) * 8, by(x[j]));
  }
  for (; i < groups; i += kThreads) store8(out + i * 8, by(load8(in + i * 8)));
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(ClipArgs a) {
  __shared__ double lds[4];
  double sum = 0.0;
  for (unsigned i = threadIdx.x; i < a.all; i += kThreads) sum += a.sums[i];
  sum = sum_of(sum, lds);
  const double norm = (double)a.scale * sqrt(sum);
  if (blockIdx.x == 0 && a.before == 0 && threadIdx.x == 0) *a.norm = (float)norm;
  if (a.chunks == 0) return;
  // a NaN is passed on
  const Factor by((double)a.scale * (norm <= (double)a.limit ? 1.0 : (double)a.limit / norm));
  const Piece piece = piece_of(a, a.chunks - 1 - blockIdx.x);
  const void* in = a.in[piece.tensor];
  void* out = a.out[piece.tensor];
  if (in == out && by.first == 1.f) return;
  const int64_t at = piece.begin, n = piece.count;
  switch (a.f16[piece.tensor]) {
    case 0: return scaled((const float*)in + at, (float*)out + at, n, by);
    case 1: return scaled((const _Float16*)in + at, (float*)out + at, n, by);
    case 2: return scaled((const float*)in + at, (_Float16*)out + at, n, by);
    default: return scaled((const _Float16*)in + at, (_Float16*)out + at, n, by);
  }
}

}  // namespace

size_t clip_grad_bytes(int64_t tensors) { return (size_t)(kChunks + tensors) * sizeof(double); }

void launch_clip_grad_norm(const Gradients& g, float scale, float limit, float* norm, void* workspace, hipStream_t st) {
  int64_t elements = 0;
  for (int64_t i = 0; i < g.tensors; ++i) elements += g.sizes[i];
  ClipArgs a;
  a.chunk = ((elements + kChunks - 1) / kChunks + 4095) / 4096 * 4096;
  if (a.chunk < 8192) a.chunk = 8192;
  a.sums = (double*)workspace;
  a.norm = norm;
  a.scale = scale;
  a.limit = limit;
  int64_t all = 0;
  for (int64_t i = 0; i < g.tensors; ++i) all += (g.sizes[i] + a.chunk - 1) / a.chunk;
  a.all = (unsigned)all;
  const bool nothing = g.in_place && scale == 1.f && limit == INFINITY;  // the norm alone
  for (int scale_them = 0; scale_them < 2; ++scale_them) {
    if (scale_them && (nothing || all == 0)) {
      a.tensors = 0;
      a.chunks = a.before = 0;
      hipLaunchKernelGGL(grad_scale_kernel, dim3(1), dim3(kThreads), 0, st, a);
      break;
    }
    int64_t next = 0;
    a.before = 0;
    while (next < g.tensors) {
      a.tensors = 0;
      a.chunks = 0;
      for (; next < g.tensors && a.tensors < kTensors; ++next) {
        if (g.sizes[next] == 0) continue;
        const int n = a.tensors++;
        a.in[n] = g.in[next];
        a.out[n] = g.out[next];
        a.size[n] = g.sizes[next];
        a.f16[n] = (unsigned char)((g.in_f16[next] ? 1 : 0) | (g.out_f16[next] ? 2 : 0));
        a.first[n] = a.chunks;
        a.chunks += (unsigned)((g.sizes[next] + a.chunk - 1) / a.chunk);
      }
      if (a.chunks == 0) continue;
      if (scale_them) hipLaunchKernelGGL(grad_scale_kernel, dim3(a.chunks), dim3(kThreads), 0, st, a);
      else hipLaunchKernelGGL(grad_squares_kernel, dim3(a.chunks), dim3(kThreads), 0, st, a);
      a.before += a.chunks;
    }
  }
}

}  // namespace gptmi
