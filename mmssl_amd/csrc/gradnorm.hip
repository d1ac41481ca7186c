// The global norm of a list of gradients, and the list scaled down to a largest norm.
//
//   n = sqrt(sum over all tensors of |g|^2);   out = g * c,  c = min(1, max_norm / (n + eps))
//
// A launch takes up to MMSSL_CLIP_MAX_TENSORS tensors of any of the three types and any size as kernel arguments (nothing is
// uploaded, a captured graph replays them); its blocks share the tensors' chunks evenly and leave one partial sum each. The
// sums are in 64 bits: the square of every fp32 number is representable, nothing overflows or vanishes on the way, and the
// conversions hide behind the loads. The scaling launch adds the partial sums up again in every block (a few KB out of the
// cache) instead of waiting for a launch that would do it once, and walks the chunks from the back, where the norm's launch
// has just left them in the caches.
#include <algorithm>

#include "typed.hpp"

using namespace mmssl;

namespace {

constexpr int kMaxT = MMSSL_CLIP_MAX_TENSORS;
constexpr int kChunk = 8192;              // elements of a chunk
constexpr int kMaxBlocks = 1024;          // of one launch

struct List {
  const void* g[kMaxT];
  void* o[kMaxT];
  int64_t n[kMaxT];
  int32_t first[kMaxT + 1];               // first chunk of each tensor
  uint8_t dt[kMaxT];
  int32_t count;
};
struct NormList {                         // the same without outputs: half the arguments
  const void* g[kMaxT];
  int64_t n[kMaxT];
  int32_t first[kMaxT + 1];
  uint8_t dt[kMaxT];
  int32_t count;
};

template <class L>
__device__ __forceinline__ int tensor_of(const L& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
// the block's sum on every thread
__device__ __forceinline__ double block_sum(double v, double* red) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class T>
__device__ __forceinline__ double squares(const T* __restrict__ p, int left) {
  constexpr int N = Vec<T>::N, IT = kChunk / (kBlock * N);
  double a = 0.0;
  if (left >= kChunk) {
    typename Vec<T>::raw v[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) v[k] = load_raw<T, true>(p + (k * kBlock + threadIdx.x) * N, N);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const typename Vec<T>::f32 f = to_f32<T>(v[k]);
#pragma unroll
      for (int e = 0; e < N; ++e) a = fma((double)f[e], (double)f[e], a);
    }
  } else {
    for (int i = threadIdx.x * N; i < left; i += kBlock * N) {
      const typename Vec<T>::f32 f = to_f32<T>(load_raw<T>(p + i, left - i));
#pragma unroll
      for (int e = 0; e < N; ++e) a = fma((double)f[e], (double)f[e], a);
    }
  }
  return a;
}

__global__ __launch_bounds__(kBlock) void norm_kernel(NormList l, double* __restrict__ part) {
  __shared__ double red[4];
  const int chunks = l.first[l.count];
  double a = 0.0;
  for (int ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
    const int t = tensor_of(l, ch);
    const int64_t at = (int64_t)(ch - l.first[t]) * kChunk;
    const int left = (int)min((int64_t)kChunk, l.n[t] - at);
    if (l.dt[t] == MMSSL_F32) a += squares(static_cast<const float*>(l.g[t]) + at, left);
    else if (l.dt[t] == MMSSL_BF16) a += squares(static_cast<const bf16_t*>(l.g[t]) + at, left);
    else a += squares(static_cast<const f16_t*>(l.g[t]) + at, left);
  }
  a = block_sum(a, red);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

__device__ __forceinline__ double norm_of(const double* __restrict__ part, int nparts, double* red) {
  double a = 0.0;
  for (int i = threadIdx.x; i < nparts; i += kBlock) a += part[i];
  return sqrt(block_sum(a, red));
}

__global__ __launch_bounds__(kBlock) void norm_finish_kernel(const double* __restrict__ part, int nparts,
                                                             float* __restrict__ norm) {
  __shared__ double red[4];
  const double n = norm_of(part, nparts, red);
  if (threadIdx.x == 0) norm[0] = (float)n;
}

template <class T>
__device__ __forceinline__ void scaled(const T* p, T* o, int left, float c) {
  constexpr int N = Vec<T>::N, IT = kChunk / (kBlock * N);
  if (left >= kChunk) {
    typename Vec<T>::raw v[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k)
      v[k] = *reinterpret_cast<const typename Vec<T>::raw*>(p + (k * kBlock + threadIdx.x) * N);
#pragma unroll
    for (int k = 0; k < IT; ++k)
      *reinterpret_cast<typename Vec<T>::raw*>(o + (k * kBlock + threadIdx.x) * N) =
          __builtin_convertvector(to_f32<T>(v[k]) * c, typename Vec<T>::raw);
  } else {
    const int whole = left / N * N;
    for (int i = threadIdx.x * N; i < whole; i += kBlock * N) {
      const typename Vec<T>::raw v = *reinterpret_cast<const typename Vec<T>::raw*>(p + i);
      *reinterpret_cast<typename Vec<T>::raw*>(o + i) = __builtin_convertvector(to_f32<T>(v) * c, typename Vec<T>::raw);
    }
    if (whole + (int)threadIdx.x < left) o[whole + threadIdx.x] = (T)((float)p[whole + threadIdx.x] * c);
  }
}

// `out` may be the gradients themselves: every element is read and written by one thread
__global__ __launch_bounds__(kBlock) void clip_kernel(List l, const double* __restrict__ part, int nparts, float max_norm,
                                                      float eps, int same, float* __restrict__ norm) {
  __shared__ double red[4];
  const double n = norm_of(part, nparts, red);
  const double q = (double)max_norm / (n + (double)eps);
  const float c = q >= 1.0 ? 1.0f : (float)q;            // a NaN stays one
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
  if (same && c == 1.0f) return;                         // in place, below the largest norm: times 1
  const int chunks = l.first[l.count];
  for (int ch = chunks - 1 - (int)blockIdx.x; ch >= 0; ch -= gridDim.x) {
    const int t = tensor_of(l, ch);
    const int64_t at = (int64_t)(ch - l.first[t]) * kChunk;
    const int left = (int)min((int64_t)kChunk, l.n[t] - at);
    if (l.dt[t] == MMSSL_F32) scaled(static_cast<const float*>(l.g[t]) + at, static_cast<float*>(l.o[t]) + at, left, c);
    else if (l.dt[t] == MMSSL_BF16)
      scaled(static_cast<const bf16_t*>(l.g[t]) + at, static_cast<bf16_t*>(l.o[t]) + at, left, c);
    else scaled(static_cast<const f16_t*>(l.g[t]) + at, static_cast<f16_t*>(l.o[t]) + at, left, c);
  }
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// the tensors [a, b) of one launch; 0, or the error
template <class L>
int fill(L& l, const void* const* grads, const int64_t* numel, const int32_t* dtypes, int a, int b) {
  int64_t chunks = 0;
  l.count = b - a;
  for (int i = a; i < b; ++i) {
    l.g[i - a] = grads[i];
    l.n[i - a] = numel[i];
    l.dt[i - a] = (uint8_t)dtypes[i];
    l.first[i - a] = (int32_t)chunks;
    chunks += chunks_of(numel[i]);
    if (chunks > 0x3fffffff) return MMSSL_E_UNSUPP;
  }
  l.first[b - a] = (int32_t)chunks;
  return 0;
}

int check_list(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count) {
  if (count < 0 || (count > 0 && (!grads || !numel || !dtypes))) return MMSSL_E_BADARG;
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0 || !known_dtype(dtypes[i])) return MMSSL_E_BADARG;
    if (numel[i] > 0 && (!grads[i] || !aligned_to(grads[i], dtype_bytes(dtypes[i])))) return MMSSL_E_BADARG;
  }
  return 0;
}

int launches_of(int count) { return (count + kMaxT - 1) / kMaxT; }

// partial sums of all launches; blocks of launch k in *blocks (NULL: not wanted)
int norm_launches(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count, double* part,
                  hipStream_t s, int* nparts) {
  int used = 0;
  for (int a = 0; a < count; a += kMaxT) {
    const int b = std::min(count, a + kMaxT);
    NormList l;
    if (int rc = fill(l, grads, numel, dtypes, a, b)) return rc;
    const int blocks = std::min(l.first[l.count], kMaxBlocks);
    if (blocks == 0) continue;
    hipLaunchKernelGGL(norm_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, s, l, part + used);
    MMSSL_LAUNCH_CHECK();
    used += blocks;
  }
  *nparts = used;
  return 0;
}

}  // namespace

extern "C" size_t mmssl_grad_norm_workspace_bytes(int count) {
  return count < 0 ? 0 : (size_t)launches_of(count) * kMaxBlocks * 8 + 16;
}

extern "C" int mmssl_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count, float* norm,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_list(grads, numel, dtypes, count)) return rc;
  if (!norm) return MMSSL_E_BADARG;
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < mmssl_grad_norm_workspace_bytes(count))
    return MMSSL_E_WORKSPACE;
  double* part = static_cast<double*>(workspace);
  int nparts = 0;
  if (int rc = norm_launches(grads, numel, dtypes, count, part, as_stream(stream), &nparts)) return rc;
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kBlock), 0, as_stream(stream), (const double*)part, nparts, norm);
  MMSSL_LAUNCH_CHECK();
  return 0;
}

extern "C" int mmssl_clip_grads(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes,
                                int count, float max_norm, float eps, float* norm, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (int rc = check_list(grads, numel, dtypes, count)) return rc;
  if (!norm || !(max_norm >= 0.f) || !(eps >= 0.f) || (count > 0 && !outs)) return MMSSL_E_BADARG;
  for (int i = 0; i < count; ++i)
    if (numel[i] > 0 && (!outs[i] || !aligned_to(outs[i], dtype_bytes(dtypes[i])))) return MMSSL_E_BADARG;
  if (!workspace || !aligned_to(workspace, 8) || workspace_bytes < mmssl_grad_norm_workspace_bytes(count))
    return MMSSL_E_WORKSPACE;
  double* part = static_cast<double*>(workspace);
  const hipStream_t s = as_stream(stream);
  int nparts = 0;
  if (int rc = norm_launches(grads, numel, dtypes, count, part, s, &nparts)) return rc;
  if (nparts == 0) {
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kBlock), 0, s, (const double*)part, 0, norm);
    MMSSL_LAUNCH_CHECK();
    return 0;
  }
  bool told = false;
  for (int b = count; b > 0; b = (b - 1) / kMaxT * kMaxT) {            // the last tensors first: they were read last
    const int a = (b - 1) / kMaxT * kMaxT;
    List l;
    if (int rc = fill(l, grads, numel, dtypes, a, b)) return rc;
    int same = 1;
    for (int i = a; i < b; ++i) {
      l.o[i - a] = outs[i];
      same &= numel[i] == 0 || outs[i] == grads[i];
    }
    const int blocks = std::min(l.first[l.count], kMaxBlocks);
    if (blocks == 0) continue;
    hipLaunchKernelGGL(clip_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, s, l, (const double*)part, nparts, max_norm, eps,
                       same, told ? (float*)nullptr : norm);
    MMSSL_LAUNCH_CHECK();
    told = true;
  }
  return 0;
}
