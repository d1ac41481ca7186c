// The global norm of a list of gradients, and the list scaled down to a largest norm.
//
//   n = sqrt(sum over all tensors of |g|^2);   out = g * c,  c = min(1, max_norm / (n + eps))
//
// Up to MMSSL_CLIP_MAX_TENSORS tensors of any of the three types and any size are kernel arguments; longer lists are written by
// kernel arguments into a table in the workspace first, so that the norm and the scaling stay one launch each (600 tensors,
// 60 M bf16: 150 us as seven launches each). Nothing is uploaded from host memory, a captured graph replays the list. The
// blocks share the tensors' chunks evenly and leave one partial sum each. The
// sums are in 64 bits: the square of every fp32 number is representable, nothing overflows or vanishes on the way, and the
// conversions hide behind the loads. The scaling launch adds the partial sums up again in every block (a few KB out of the
// cache) instead of waiting for a launch that would do it once. With a list in the arguments it walks the chunks from the back,
// where the norm's launch has just left them in the caches; in a longer list each block walks its own run of chunks forwards.
#include <algorithm>

#include "typed.hpp"

using namespace mmssl;

namespace {

constexpr int kMaxT = MMSSL_CLIP_MAX_TENSORS;
// Elements of a chunk, blocks of a launch: 384 M fp32 in 9 tensors 864 us (8192 and 1024: 868; 16384: 881), 600 tensors of 60 M
// bf16 86 us (90; 93), 24 tensors of 0.3 M fp32 8.9 us (9.4; 11.1).
constexpr int kChunk = 4096;
constexpr int kMaxBlocks = 2048;

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

// one tensor of a list in the workspace
struct __attribute__((aligned(16))) Entry {
  const void* g;
  void* o;
  int64_t n;
  int32_t first;
  int32_t dt;
};

__global__ __launch_bounds__(128) void table_kernel(List l, int32_t from, Entry* __restrict__ table) {
  for (int i = threadIdx.x; i < l.count; i += 128) table[i] = {l.g[i], l.o[i], l.n[i], from + l.first[i], l.dt[i]};
}

// Where a chunk is: its tensor's type, first element of the chunk, elements from there on.
struct Place {
  const char* g;
  char* o;
  int64_t left;
  int dt;
};
__device__ __forceinline__ Place place_of(const void* g, void* o, int64_t n, int dt, int chunk) {
  const int64_t at = (int64_t)chunk * kChunk, size = dt == MMSSL_F32 ? 4 : 2;
  return {static_cast<const char*>(g) + at * size, static_cast<char*>(o) + at * size, n - at, dt};
}
__device__ __forceinline__ void* out_of(const List& l, int t) { return l.o[t]; }
__device__ __forceinline__ void* out_of(const NormList&, int) { return nullptr; }

// Lists in the arguments: a search through scalar registers for each chunk, the chunks dealt to the blocks in turn.
template <class L>
struct Walk {
  const L& l;
  __device__ __forceinline__ Walk(const L& list) : l(list) {}
  __device__ __forceinline__ int begin(int) const { return blockIdx.x; }
  __device__ __forceinline__ int end(int chunks) const { return chunks; }
  __device__ __forceinline__ int step() const { return gridDim.x; }
  __device__ __forceinline__ int from_back(int i, int chunks) const { return chunks - 1 - i; }
  __device__ __forceinline__ Place find(int chunk) const {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (l.first[mid] <= chunk) lo = mid;
      else hi = mid - 1;
    }
    return place_of(l.g[lo], out_of(l, lo), l.n[lo], l.dt[lo], chunk - l.first[lo]);
  }
};

// Lists in the workspace: a block's chunks follow each other. Where they are is worked out for kAhead of them at a time: each
// thread looks at its share of the entries and writes down the chunks that fall into its entries, so that the entries are one
// round of loads and not a chain of them in front of every tensor (600 tensors, 60 M bf16: both launches 86 us, so 80).
struct Table {
  const Entry* e;
  int32_t count, chunks;
};
constexpr int kAhead = 64;
template <>
struct Walk<Table> {
  const Table l;
  Place* at;                              // LDS, kAhead of them
  int from = 0, until = 0;                // the chunks that are there
  __device__ __forceinline__ Walk(const Table& table) : l(table) {
    __shared__ Place place[kAhead];
    at = place;
  }
  __device__ __forceinline__ int begin(int chunks) const { return (int)((int64_t)chunks * blockIdx.x / gridDim.x); }
  __device__ __forceinline__ int end(int chunks) const { return (int)((int64_t)chunks * (blockIdx.x + 1) / gridDim.x); }
  __device__ __forceinline__ int step() const { return 1; }
  __device__ __forceinline__ int from_back(int i, int) const { return i; }
  __device__ __forceinline__ Place find(int chunk) {             // the same chunk for every thread of the block
    if (chunk >= until) {
      from = chunk;
      until = min(chunk + kAhead, end(l.chunks));
      __syncthreads();
#pragma unroll 4
      for (int i = threadIdx.x; i < l.count; i += kBlock) {
        const Entry e = l.e[i];
        const int last = e.first + (int)((e.n + kChunk - 1) / kChunk);
        for (int c = max(e.first, from); c < min(last, until); ++c) at[c - from] = place_of(e.g, e.o, e.n, e.dt, c - e.first);
      }
      __syncthreads();
    }
    Place p = at[chunk - from];
    p.dt = __builtin_amdgcn_readfirstlane(p.dt);
    return p;
  }
};
template <class L>
__device__ __forceinline__ int chunks_in(const L& l) { return l.first[l.count]; }
__device__ __forceinline__ int chunks_in(const Table& l) { return l.chunks; }

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

// The elements of a chunk, `left` of them: all vectors are asked for before the first is used, also those of a tensor's last,
// shorter chunk (with a loop there, lists of many small tensors waited once per 4 KB: 600 of 60 M bf16, norm alone 54 -> 42 us).
template <class T>
struct Chunk {
  static constexpr int N = Vec<T>::N, IT = kChunk / (kBlock * N);
  typedef typename Vec<T>::raw R;
  R v[IT];
  T last;                                 // one of the elements behind the last whole vector
  int whole;
  bool has_last;
  __device__ __forceinline__ void load(const T* p, int left) {
    whole = left / N * N;
    has_last = whole + (int)threadIdx.x < left;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int i = (k * kBlock + threadIdx.x) * N;
      v[k] = (R)(T)0.0f;
      if (i < whole) v[k] = *reinterpret_cast<const R*>(p + i);
    }
    last = (T)0.0f;
    if (has_last) last = p[whole + threadIdx.x];
  }
};

template <class T>
__device__ __forceinline__ double squares(const T* __restrict__ p, int left) {
  Chunk<T> q;
  q.load(p, left);
  double a = 0.0;
#pragma unroll
  for (int k = 0; k < Chunk<T>::IT; ++k) {
    const typename Vec<T>::f32 f = to_f32<T>(q.v[k]);
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) a = fma((double)f[e], (double)f[e], a);
  }
  return fma((double)(float)q.last, (double)(float)q.last, a);
}

template <class L>
__global__ __launch_bounds__(kBlock) void norm_kernel(L l, double* __restrict__ part) {
  __shared__ double red[4];
  const int chunks = chunks_in(l);
  Walk<L> w(l);
  double a = 0.0;
  for (int ch = w.begin(chunks); ch < w.end(chunks); ch += w.step()) {
    const Place p = w.find(ch);
    const int left = (int)min((int64_t)kChunk, p.left);
    if (p.dt == MMSSL_F32) a += squares(reinterpret_cast<const float*>(p.g), left);
    else if (p.dt == MMSSL_BF16) a += squares(reinterpret_cast<const bf16_t*>(p.g), left);
    else a += squares(reinterpret_cast<const f16_t*>(p.g), left);
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
  Chunk<T> q;
  q.load(p, left);
#pragma unroll
  for (int k = 0; k < Chunk<T>::IT; ++k) {
    const int i = (k * kBlock + threadIdx.x) * Vec<T>::N;
    if (i < q.whole)
      *reinterpret_cast<typename Vec<T>::raw*>(o + i) =
          __builtin_convertvector(to_f32<T>(q.v[k]) * c, typename Vec<T>::raw);
  }
  if (q.has_last) o[q.whole + threadIdx.x] = (T)((float)q.last * c);
}

// `out` may be the gradients themselves: every element is read and written by one thread
template <class L>
__global__ __launch_bounds__(kBlock) void clip_kernel(L l, const double* __restrict__ part, int nparts, float max_norm,
                                                      float eps, int same, float* __restrict__ norm) {
  __shared__ double red[4];
  const double n = norm_of(part, nparts, red);
  const double q = (double)max_norm / (n + (double)eps);
  const float c = q >= 1.0 ? 1.0f : (float)q;            // a NaN stays one
  if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
  if (same && c == 1.0f) return;                         // in place, below the largest norm: times 1
  const int chunks = chunks_in(l);
  Walk<L> w(l);
  for (int i = w.begin(chunks); i < w.end(chunks); i += w.step()) {
    const Place p = w.find(w.from_back(i, chunks));
    const int left = (int)min((int64_t)kChunk, p.left);
    if (p.dt == MMSSL_F32) scaled(reinterpret_cast<const float*>(p.g), reinterpret_cast<float*>(p.o), left, c);
    else if (p.dt == MMSSL_BF16) scaled(reinterpret_cast<const bf16_t*>(p.g), reinterpret_cast<bf16_t*>(p.o), left, c);
    else scaled(reinterpret_cast<const f16_t*>(p.g), reinterpret_cast<f16_t*>(p.o), left, c);
  }
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// the tensors [a, b) as kernel arguments
template <class L>
void fill(L& l, const void* const* grads, const int64_t* numel, const int32_t* dtypes, int a, int b) {
  int64_t chunks = 0;
  l.count = b - a;
  for (int i = a; i < b; ++i) {
    l.g[i - a] = grads[i];
    l.n[i - a] = numel[i];
    l.dt[i - a] = (uint8_t)dtypes[i];
    l.first[i - a] = (int32_t)chunks;
    chunks += chunks_of(numel[i]);
  }
  l.first[b - a] = (int32_t)chunks;
}

int check_list(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count) {
  if (count < 0 || (count > 0 && (!grads || !numel || !dtypes))) return MMSSL_E_BADARG;
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0 || !known_dtype(dtypes[i])) return MMSSL_E_BADARG;
    if (numel[i] > 0 && (!grads[i] || !aligned_to(grads[i], dtype_bytes(dtypes[i])))) return MMSSL_E_BADARG;
  }
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (numel[i] > (int64_t)0x3fffffff * kChunk) return MMSSL_E_UNSUPP;
    chunks += chunks_of(numel[i]);
    if (chunks > 0x3fffffff) return MMSSL_E_UNSUPP;
  }
  return 0;
}

// workspace: the blocks' sums, then the table of a long list
constexpr size_t kPartBytes = (size_t)kMaxBlocks * 8;
size_t ws_bytes(int count) { return kPartBytes + (count > kMaxT ? (size_t)count * sizeof(Entry) : 0); }

int total_chunks(const int64_t* numel, int count) {
  int64_t c = 0;
  for (int i = 0; i < count; ++i) c += chunks_of(numel[i]);
  return (int)c;                          // check_list has seen it
}

// the long list's table; `outs` may be NULL
int write_table(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, int count,
                Entry* table, hipStream_t s) {
  int32_t from = 0;
  for (int a = 0; a < count; a += kMaxT) {
    const int b = std::min(count, a + kMaxT);
    List l;
    fill(l, grads, numel, dtypes, a, b);
    for (int i = a; i < b; ++i) l.o[i - a] = outs ? outs[i] : nullptr;
    hipLaunchKernelGGL(table_kernel, dim3(1), dim3(128), 0, s, l, from, table + a);
    MMSSL_LAUNCH_CHECK();
    from += l.first[l.count];
  }
  return 0;
}

template <class L>
int norm_launch(const L& l, int blocks, double* part, hipStream_t s) {
  hipLaunchKernelGGL(norm_kernel<L>, dim3((unsigned)blocks), dim3(kBlock), 0, s, l, part);
  MMSSL_LAUNCH_CHECK();
  return 0;
}

// grads -> the blocks' sums in `part`; a long list's table is written on the way
int sums_of(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes, int count, int chunks,
            void* workspace, hipStream_t s) {
  double* part = static_cast<double*>(workspace);
  const int blocks = std::min(chunks, kMaxBlocks);
  if (count > kMaxT) {
    Entry* table = reinterpret_cast<Entry*>(static_cast<char*>(workspace) + kPartBytes);
    if (int rc = write_table(grads, outs, numel, dtypes, count, table, s)) return rc;
    return norm_launch(Table{table, count, chunks}, blocks, part, s);
  }
  NormList l;
  fill(l, grads, numel, dtypes, 0, count);
  return norm_launch(l, blocks, part, s);
}

}  // namespace

extern "C" size_t mmssl_grad_norm_workspace_bytes(int count) { return count < 0 ? 0 : ws_bytes(count); }

extern "C" int mmssl_grad_norm(const void* const* grads, const int64_t* numel, const int32_t* dtypes, int count, float* norm,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_list(grads, numel, dtypes, count)) return rc;
  if (!norm) return MMSSL_E_BADARG;
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < ws_bytes(count)) return MMSSL_E_WORKSPACE;
  const hipStream_t s = as_stream(stream);
  const int chunks = total_chunks(numel, count);
  if (chunks)
    if (int rc = sums_of(grads, nullptr, numel, dtypes, count, chunks, workspace, s)) return rc;
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kBlock), 0, s, static_cast<const double*>(workspace),
                     std::min(chunks, kMaxBlocks), norm);
  MMSSL_LAUNCH_CHECK();
  return 0;
}

extern "C" int mmssl_clip_grads(const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes,
                                int count, float max_norm, float eps, float* norm, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (int rc = check_list(grads, numel, dtypes, count)) return rc;
  if (!norm || !(max_norm >= 0.f) || !(eps >= 0.f) || (count > 0 && !outs)) return MMSSL_E_BADARG;
  int same = 1;
  for (int i = 0; i < count; ++i) {
    if (numel[i] > 0 && (!outs[i] || !aligned_to(outs[i], dtype_bytes(dtypes[i])))) return MMSSL_E_BADARG;
    same &= numel[i] == 0 || outs[i] == grads[i];
  }
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < ws_bytes(count)) return MMSSL_E_WORKSPACE;
  const hipStream_t s = as_stream(stream);
  const int chunks = total_chunks(numel, count), blocks = std::min(chunks, kMaxBlocks);
  const double* part = static_cast<const double*>(workspace);
  if (chunks == 0) {
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kBlock), 0, s, part, 0, norm);
    MMSSL_LAUNCH_CHECK();
    return 0;
  }
  if (int rc = sums_of(grads, outs, numel, dtypes, count, chunks, workspace, s)) return rc;
  if (count > kMaxT) {
    const Table l{reinterpret_cast<const Entry*>(static_cast<const char*>(workspace) + kPartBytes), count, chunks};
    hipLaunchKernelGGL(clip_kernel<Table>, dim3((unsigned)blocks), dim3(kBlock), 0, s, l, part, blocks, max_norm, eps, same,
                       norm);
  } else {
    List l;
    fill(l, grads, numel, dtypes, 0, count);
    for (int i = 0; i < count; ++i) l.o[i] = outs[i];
    hipLaunchKernelGGL(clip_kernel<List>, dim3((unsigned)blocks), dim3(kBlock), 0, s, l, part, blocks, max_norm, eps, same,
                       norm);
  }
  MMSSL_LAUNCH_CHECK();
  return 0;
}
