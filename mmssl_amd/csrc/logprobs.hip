// Log probabilities of given columns of score rows X [rows, cols], the rows' entropy, their k best columns, and the gradient.
//
//   z = x / T, lp_j = z_j - log sum exp(z);  logp = lp_target, H = -sum p_j lp_j, top = the k largest x (ties: lowest column)
//   gx_j = (1/T) (g_target [j = target] + sum_i gtop_i [j = top_i] - p_j (g_target + sum_i gtop_i) - gH p_j (lp_j + H))
//
// Forward: one read of X. A block holds a slice of a row in its registers: the slice's maximum m, S = sum e_j and
// A = sum e_j y_j with y_j = (x_j - m) / T, e_j = exp(y_j); slices join by S = sum S_i 2^(d_i), A = sum 2^(d_i) (A_i + d_i S_i)
// with d_i the distance of the slice's maximum from the row's. H = log S - A / S: both parts are >= 0, nothing cancels.
// The best columns come out of the same registers: a lower bound of the k-th largest value from the threads' maxima leaves
// about 2 k candidates, which are ranked by counting.
// Backward: one read of X, one write of gx.
//
// Bound by memory from some ten million scores on: 8192 x 35598 bf16 forward 148 us (583 MB: 3.9 TB/s; best of 15 launches 129) and 5
// for the join, backward 214 us (1.17 GB, 5.5 TB/s; best 202). With alternatives by the phases that follow the loads in every block: 1024 x
// 18357 fp32 with 50 of them 27 us (75 MB) and 7 for the join; one row of 1 M columns with 20: 6.5 + 7.3, latency.
#include <algorithm>

#include "typed.hpp"

using namespace mmssl;

namespace {

constexpr int kTopMax = 128;          // most alternatives
constexpr int kCand = 1024;           // candidates of a slice that are ranked by counting
constexpr int kWaves = kBlock / 64;
constexpr float kLn2 = 0.69314718055994530942f, kLog2e = 1.4426950408889634074f;
constexpr float kFar = -1.0e4f;       // exp2 of this is 0; stands for -inf where 0 * -inf has to be 0

// a value's place in the order of values as a whole number: NaN above +inf, -0 equal to 0
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float((o >> 31) ? (o & 0x7fffffffu) : ~o);
}
// (value, column) as one number: larger is better, equal values by the lower column. Never 0 for a column.
__device__ __forceinline__ uint64_t pair_of(float x, int64_t col) {
  return ((uint64_t)order_of(x) << 32) | (uint64_t)(0xffffffffu - (uint32_t)col);
}
__device__ __forceinline__ int64_t col_of(uint64_t p) { return (int64_t)(0xffffffffu - (uint32_t)p); }
__device__ __forceinline__ float val_of(uint64_t p) { return value_of((uint32_t)(p >> 32)); }

struct RowOut {
  const int64_t* target64;
  const int32_t* target32;
  int64_t ignore;
  float* logp;
  float* entropy;
  float* top_logp;
  int64_t* top_idx;
  float4* stats;               // row maximum, log2 of the sum, entropy, - (NULL: no backward pass will follow)
};

struct Sums {
  float m, s, a;               // maximum, sum of e, sum of e * y in units of log2
};

// what a row's sums say: (log of the sum, entropy) in nats; the row without a finite maximum has no probabilities
struct RowStat {
  float m, l2, h;
  bool empty;
};
__device__ __forceinline__ RowStat stat_of(Sums q) {
  RowStat r;
  r.m = q.m;
  r.empty = q.s == 0.f;                          // every entry is -inf
  r.l2 = r.empty ? __builtin_inff() : log2f(q.s);
  r.h = r.empty ? 0.f : (r.l2 - q.a / q.s) * kLn2;
  return r;
}
__device__ __forceinline__ float logp_of(float x, RowStat r, float inv_t) {
  if (r.empty) return -__builtin_inff();
  return (x - r.m) * inv_t - r.l2 * kLn2;
}

__device__ __forceinline__ int64_t target_of(const RowOut& o, int64_t row) {
  return o.target64 ? o.target64[row] : (int64_t)o.target32[row];
}
// the score of the row's target; anything where it has none
template <class T>
__device__ __forceinline__ float target_score(const T* __restrict__ x, int64_t cols, int64_t row, const RowOut& o) {
  const int64_t t = target_of(o, row);
  return t >= 0 && t < cols ? (float)x[t] : 0.f;
}
__device__ __forceinline__ void write_row(float x, int64_t cols, int64_t row, RowStat r, float inv_t, const RowOut& o) {
  const int64_t t = target_of(o, row);
  float lp;
  if (t == o.ignore) lp = 0.f;
  else if (t < 0 || t >= cols) lp = __builtin_nanf("");
  else lp = logp_of(x, r, inv_t);
  o.logp[row] = lp;
  o.entropy[row] = r.h;
  if (o.stats) o.stats[row] = make_float4(r.m, r.l2, r.h, 0.f);
}

__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  // a side of nothing but -inf (s = 0) has no part; a NaN in s counts. Far below the other: factor 0, and 0 * -inf is kept out
  const float da = a.s == 0.f ? kFar : fmaxf((a.m - r.m) * c, kFar), db = b.s == 0.f ? kFar : fmaxf((b.m - r.m) * c, kFar);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  r.s = a.s * fa + b.s * fb;
  r.a = fmaf(da, a.s, a.a) * fa + fmaf(db, b.s, b.a) * fb;
  return r;
}

// A lower bound of the k-th largest of all entries from the maxima (as whole numbers) of the threads that hold entries, `held`
// of them: as many threads as alternatives have a maximum that is no smaller. Each full wave of such threads finds the q-th
// largest of its maxima by its bits, the smallest of these is the bound; 0 where there are too few threads. One value a wave.
__device__ __forceinline__ uint32_t wave_bound(uint32_t key, int held, int k) {
  const int w = threadIdx.x >> 6, full = max(1, held / 64), q = (k + full - 1) / full;
  if (w >= full) return 0xffffffffu;
  if (q > 64) return 0;
  uint32_t t = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cnd = t | (1u << bit);
    const int n = __popcll(__ballot(key >= cnd));
    if (n >= q) t = cnd;
    if (n == q) break;
  }
  return t;
}

// the k best of n pairs in LDS, in order, to out[0, k): a pair's place is the number of better ones
template <class PUT>
__device__ __forceinline__ void rank_pairs(const uint64_t* __restrict__ pairs, int n, int k, PUT put) {
  for (int j = threadIdx.x; j < n; j += kBlock) {
    const uint64_t mine = pairs[j];
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) r += pairs[i] > mine;
    if (r < k) put(r, mine);
  }
}

// Exactly the k best of the `mine` columns from x on, in no order: for slices in which the bound leaves more candidates than
// are ranked (many equal values, few finite ones). The k-th largest value by its bits, then, among the entries equal to it,
// the last column that is still taken; the columns are read again from the caches for each count.
template <class T>
__device__ __attribute__((noinline)) void pick_exactly(const T* __restrict__ x, int mine, int k, int64_t c0, uint64_t* pairs,
                                                       int* n_pairs, int* count) {
  int turn = 0;
  auto total = [&](int h) {                                     // over the block; the same for every thread
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) h += __shfl_xor(h, m, 64);
    if ((threadIdx.x & 63) == 0) count[turn * kWaves + (threadIdx.x >> 6)] = h;
    __syncthreads();
    const int* q = count + turn * kWaves;
    turn ^= 1;
    return (q[0] + q[1]) + (q[2] + q[3]);
  };
  uint32_t kth = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cnd = kth | (1u << bit);
    int h = 0;
    for (int at = threadIdx.x; at < mine; at += kBlock) h += order_of((float)x[at]) >= cnd;
    if (total(h) >= k) kth = cnd;
  }
  int above = 0;
  for (int at = threadIdx.x; at < mine; at += kBlock) above += order_of((float)x[at]) > kth;
  const int need = k - total(above);
  int last = 0;                                                 // the need-th of the equal ones stands at this column
  for (int bit = 16; bit >= 0; --bit) {
    const int cnd = last | (1 << bit);
    int h = 0;
    for (int at = threadIdx.x; at < min(mine, cnd); at += kBlock) h += order_of((float)x[at]) == kth;
    if (total(h) < need) last = cnd;
  }
  __syncthreads();
  if (threadIdx.x == 0) *n_pairs = 0;
  __syncthreads();
  for (int at = threadIdx.x; at < mine; at += kBlock) {
    const float f = (float)x[at];
    const uint32_t key = order_of(f);
    if (key > kth || (key == kth && at <= last)) pairs[atomicAdd(n_pairs, 1)] = pair_of(f, c0 + at);
  }
}

// ---- forward: slices --------------------------------------------------------------------------------------------------
// Block (row, slice): columns [slice * len, ...). NV vectors a thread; vector v of thread t starts at column
// (v * kBlock + t) * N of the slice. sums [rows][splits], cand [rows][k][splits]. With one slice a row the block writes the
// row's results itself.
template <class T, int NV, bool FULL, bool TOP>
__global__ __launch_bounds__(kBlock) void lp_slice_kernel(const T* __restrict__ X, int64_t ldx, int64_t cols, int len,
                                                          int splits, float c, float inv_t, int k, RowOut o,
                                                          Sums* __restrict__ sums, uint64_t* __restrict__ cand) {
  constexpr int N = Vec<T>::N;
  typedef typename Vec<T>::raw R;
  __shared__ float red[3 * kWaves];
  __shared__ uint32_t bound[kWaves];
  __shared__ uint64_t pairs[TOP ? kCand : 1];
  __shared__ int n_pairs;
  __shared__ int count[2 * kWaves];
  const int64_t row = blockIdx.x / splits;
  const int slice = (int)(blockIdx.x % splits);
  const int64_t c0 = (int64_t)slice * len;
  const int mine = (int)min((int64_t)len, cols - c0);           // columns of this slice
  const T* x = X + row * ldx;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;

  R raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * kBlock + threadIdx.x) * N;
    raw[v] = (R)(T)(-__builtin_inff());
    if (FULL) {
      if (at < mine) raw[v] = load_raw<T, true>(x + c0 + at, N);
    } else if (at + N <= mine) {
      raw[v] = load_raw<T, true>(x + c0 + at, N);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (at + e < mine) raw[v][e] = x[c0 + at + e];
    }
  }
  float tm = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < N; ++e) tm = fmaxf(tm, (float)raw[v][e]);
  float m = group_max<64>(tm);
  if (lane == 0) red[w] = m;
  if (threadIdx.x == 0) n_pairs = 0;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float base = m == -__builtin_inff() ? 0.f : m;          // nothing but -inf (and NaN): y = -inf, e = 0
  // y = (x - base) c as one fma around hi = base c: off by the same known lo = base c - hi in every term, which is taken
  // out of the sums below. Scores so large that lo is no longer small are subtracted first.
  const float hi = base * c;
  const bool fused = fabsf(hi) <= 1048576.f;
  const float lo = fused ? fmaf(base, c, -hi) : 0.f;
  float s = 0.f, a = 0.f;
  auto sweep = [&](auto dist) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float y = dist((float)raw[v][e]);
        const float p = __builtin_amdgcn_exp2f(y);
        s += p;
        a = fmaf(p, fmaxf(y, kFar), a);                         // a NaN is in p as well
      }
  };
  if (fused) sweep([&](float f) { return fmaf(f, c, -hi); });
  else sweep([&](float f) { return (f - base) * c; });
  const bool odd = s != s;                                      // this thread holds a NaN (or the row an infinity)
  a = fmaf(-lo, s, a);
  s = group_sum<64>(s);
  a = group_sum<64>(a);
  if (lane == 0) {
    red[kWaves + w] = s;
    red[2 * kWaves + w] = a;
  }
  if (TOP) {
    const uint32_t t = wave_bound(order_of(tm), min(kBlock, (mine + N - 1) / N), k);
    if (lane == 0) bound[w] = t;
  }
  __syncthreads();
  Sums z;
  z.m = m;
  const float back = exp2f(-lo);
  z.s = ((red[kWaves] + red[kWaves + 1]) + (red[kWaves + 2] + red[kWaves + 3])) * back;
  z.a = ((red[2 * kWaves] + red[2 * kWaves + 1]) + (red[2 * kWaves + 2] + red[2 * kWaves + 3])) * back;
  const RowStat r = stat_of(z);
  if (threadIdx.x == 0) {
    if (splits == 1) write_row(target_score(x, cols, row, o), cols, row, r, inv_t, o);
    else sums[blockIdx.x] = z;
  }
  if (!TOP) return;

  const uint32_t tb = min(min(bound[0], bound[1]), min(bound[2], bound[3]));
  const float tf = value_of(tb);
  int n;
  if (tb > order_of(-__builtin_inff())) {
    // Candidates: !(x < tf), which NaN is too. A wave takes its places at once; the lanes' shares come from the ballots, which
    // stay in scalar registers (a place for each lane or value from a counter in LDS: 27 against 22 us at 1024 x 18357 fp32
    // with 50 alternatives).
    if (__any(!(tm < tf) || odd)) {
      uint64_t hit[NV * N];
      int all = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          hit[v * N + e] = __ballot(!((float)raw[v][e] < tf));
          all += __popcll(hit[v * N + e]);
        }
      int i = 0;
      if (lane == 0) i = atomicAdd(&n_pairs, all);
      i = __builtin_amdgcn_readfirstlane(i);
      if (i + all <= kCand) {                                     // (what does not fit is picked below)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const uint64_t h = hit[v * N + e];
            if (h) {
              if (h >> lane & 1) {                                // value and column for now: few instructions a hit
                const int at = i + __builtin_amdgcn_mbcnt_hi((uint32_t)(h >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)h, 0));
                pairs[at] = ((uint64_t)__float_as_uint((float)raw[v][e]) << 32) | ((v * kBlock + threadIdx.x) * N + e);
              }
              i += __popcll(h);
            }
          }
      }
    }
    __syncthreads();
    n = n_pairs;
    if (n <= kCand) {
      for (int j = threadIdx.x; j < n; j += kBlock) {             // an entry is its thread's alone
        const uint64_t q = pairs[j];
        pairs[j] = pair_of(__uint_as_float((uint32_t)(q >> 32)), c0 + (uint32_t)q);
      }
      __syncthreads();
    }
  } else {
    n = kCand + 1;                                                // too few finite maxima for a bound
  }
  if (n > kCand) {
    if (mine <= kBlock) {                                         // all of a short slice
      if ((int)threadIdx.x < mine) pairs[threadIdx.x] = pair_of((float)x[c0 + threadIdx.x], c0 + threadIdx.x);
      n = mine;
    } else {
      n = min(k, mine);
      pick_exactly<T>(x + c0, mine, n, c0, pairs, &n_pairs, count);
    }
    __syncthreads();
  }
  if (splits == 1) {
    rank_pairs(pairs, n, k, [&](int i, uint64_t p) {
      o.top_idx[row * k + i] = col_of(p);
      o.top_logp[row * k + i] = logp_of(val_of(p), r, inv_t);
    });
  } else {
    uint64_t* out = cand + row * k * splits + slice;              // [rows][k][splits]: the slices' best, then their next ...
    rank_pairs(pairs, n, k, [&](int i, uint64_t p) { out[(int64_t)i * splits] = p; });
    for (int i = n + threadIdx.x; i < k; i += kBlock) out[(int64_t)i * splits] = 0;
  }
}

// ---- forward: short rows without alternatives: a wave a row, no barriers (100 K rows of 1000 fp32: 150 us with a block a row) ---
template <class T, int NV, bool FULL>
__global__ __launch_bounds__(kBlock) void lp_short_kernel(const T* __restrict__ X, int64_t ldx, int64_t rows, int cols, float c,
                                                          float inv_t, RowOut o) {
  constexpr int N = Vec<T>::N;
  typedef typename Vec<T>::raw R;
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  const T* x = X + row * ldx;
  R raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = (v * 64 + lane) * N;
    raw[v] = (R)(T)(-__builtin_inff());
    if (FULL ? at < cols : at + N <= cols) {
      raw[v] = load_raw<T, true>(x + at, N);
    } else if (!FULL) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (at + e < cols) raw[v][e] = x[at + e];
    }
  }
  const float at_target = lane == 0 ? target_score(x, cols, row, o) : 0.f;
  float m = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, (float)raw[v][e]);
  m = group_max<64>(m);
  const float base = m == -__builtin_inff() ? 0.f : m;
  Sums z = {m, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float y = ((float)raw[v][e] - base) * c;
      const float p = __builtin_amdgcn_exp2f(y);
      z.s += p;
      z.a = fmaf(p, fmaxf(y, kFar), z.a);
    }
  z.s = group_sum<64>(z.s);
  z.a = group_sum<64>(z.a);
  if (lane == 0) write_row(at_target, cols, row, stat_of(z), inv_t, o);
}

// ---- forward: the slices of a row -------------------------------------------------------------------------------------
// These kernels run once through little data: what they cost is misses, of data and of instructions. What can be asked for at
// once is, and their loops stay rolled (the same with 16 pairs a thread in unrolled registers: 20 us for one row of 1 M
// columns, of it 9 for code that had to come from memory).

// Sums of the `group` (a power of two, up to a wave) neighbouring lanes, joined in a fixed order; the first has them.
__device__ __forceinline__ Sums join_lanes(Sums z, int group, float c) {
#pragma unroll 1
  for (int m = 1; m < group; m <<= 1) {
    Sums y;
    y.m = __shfl_xor(z.m, m, 64);
    y.s = __shfl_xor(z.s, m, 64);
    y.a = __shfl_xor(z.a, m, 64);
    const bool second = threadIdx.x & m;                          // the same operands in the same order on both lanes
    z = join({second ? y.m : z.m, second ? y.s : z.s, second ? y.a : z.a},
             {second ? z.m : y.m, second ? z.s : y.s, second ? z.a : y.a}, c);
  }
  return z;
}

// `group` lanes a row
template <class T>
__global__ __launch_bounds__(kBlock) void lp_join_kernel(const T* __restrict__ X, int64_t ldx, int64_t rows, int64_t cols,
                                                         int splits, int group, float c, float inv_t, RowOut o,
                                                         const Sums* __restrict__ sums) {
  const int64_t row = (int64_t)blockIdx.x * (kBlock / group) + threadIdx.x / group;
  const int lane = threadIdx.x & (group - 1);
  Sums z = {-__builtin_inff(), 0.f, 0.f};
  float at_target = 0.f;
  if (row < rows) {
    if (lane < splits) z = sums[row * splits + lane];
    if (lane == 0) at_target = target_score(X + row * ldx, cols, row, o);
#pragma unroll 1
    for (int i = lane + group; i < splits; i += group) z = join(z, sums[row * splits + i], c);
  }
  z = join_lanes(z, group, c);
  if (row < rows && lane == 0) write_row(at_target, cols, row, stat_of(z), inv_t, o);
}

// ... with alternatives: one block a row. The slices' k best are pairs of distinct numbers, the slices' first ones before their
// second ones: the k-th largest of the first 256 bounds the row's k-th largest from below and leaves a few times k pairs, which
// are ranked. Up to `hold` pairs are all looked at (LDS); of longer lists each thread follows its slices' down to the bound.
// Where the bound leaves more than kCand, the k-th largest is found by its bits.
template <class T>
__global__ __launch_bounds__(kBlock) void lp_join_top_kernel(const T* __restrict__ X, int64_t ldx, int64_t cols, int splits,
                                                             float c, float inv_t, int k, RowOut o,
                                                             const Sums* __restrict__ sums,
                                                             const uint64_t* __restrict__ cand, int hold) {
  extern __shared__ uint64_t held[];
  __shared__ uint64_t best[kCand];
  __shared__ Sums part[kWaves];
  __shared__ uint32_t bound[kWaves];
  __shared__ int n_best;
  __shared__ int wsum[2][kWaves];
  constexpr int kAhead = 4;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, total = splits * k;
  const bool flat = total <= hold;
  const uint64_t* src = cand + row * total;
  const uint64_t first = tid < total ? src[tid] : 0;
  uint64_t next[kAhead];                             // of the thread's first slice, below its best
  if (!flat) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) next[j] = tid < splits && j + 1 < k ? src[(j + 1) * splits + tid] : 0;
  }
  Sums z = {-__builtin_inff(), 0.f, 0.f};
  if (tid < splits) z = sums[row * splits + tid];
  float at_target = 0.f;
  if (tid == kBlock - 1) at_target = target_score(X + row * ldx, cols, row, o);
  if (flat) {
    if (tid < total) held[tid] = first;
#pragma unroll 4
    for (int i = tid + kBlock; i < total; i += kBlock) held[i] = src[i];
  }
#pragma unroll 1
  for (int i = tid + kBlock; i < splits; i += kBlock) z = join(z, sums[row * splits + i], c);
  const uint32_t t = wave_bound((uint32_t)(first >> 32), min(kBlock, total), k);
  z = join_lanes(z, 64, c);
  if ((tid & 63) == 0) {
    bound[tid >> 6] = t;
    part[tid >> 6] = z;
  }
  if (tid == 0) n_best = 0;
  __syncthreads();
  z = part[0];
#pragma unroll 1
  for (int w = 1; w < kWaves; ++w) z = join(z, part[w], c);
  const RowStat r = stat_of(z);
  if (tid == kBlock - 1) write_row(at_target, cols, row, r, inv_t, o);
  auto put = [&](uint64_t p) {
    const int at = atomicAdd(&n_best, 1);
    if (at < kCand) best[at] = p;
  };
  auto take = [&](uint64_t from) {                                          // from >= 1: 0 is no pair
    if (flat) {
#pragma unroll 1
      for (int i = tid; i < total; i += kBlock)
        if (held[i] >= from) put(held[i]);
      return;
    }
#pragma unroll 1
    for (int s = tid; s < splits; s += kBlock) {
#pragma unroll 1
      for (int j = 0; j < k; ++j) {
        uint64_t p;
        if (s == tid && j <= kAhead) {
          p = first;
#pragma unroll
          for (int h = 0; h < kAhead; ++h)
            if (j == h + 1) p = next[h];
        } else {
          p = src[(int64_t)j * splits + s];
        }
        if (p < from) break;
        put(p);
      }
    }
  };
  const uint32_t tb = min(min(bound[0], bound[1]), min(bound[2], bound[3]));
  take(max((uint64_t)tb << 32, (uint64_t)1));
  __syncthreads();
  int n = n_best;
  if (n > kCand) {                                                          // the same on every thread
    uint64_t from = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t cnd = from | (1ull << bit);
      int h = 0;
      for (int i = tid; i < total; i += kBlock) h += src[i] >= cnd;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) h += __shfl_xor(h, m, 64);
      if ((tid & 63) == 0) wsum[bit & 1][tid >> 6] = h;
      __syncthreads();
      const int* q = wsum[bit & 1];
      const int above = (q[0] + q[1]) + (q[2] + q[3]);
      if (above >= k) from = cnd;
      if (above == k) break;
    }
    __syncthreads();
    if (tid == 0) n_best = 0;
    __syncthreads();
    take(max(from, (uint64_t)1));
    __syncthreads();
    n = n_best;
  }
  rank_pairs(best, n, k, [&](int i, uint64_t p) {
    o.top_idx[row * k + i] = col_of(p);
    o.top_logp[row * k + i] = logp_of(val_of(p), r, inv_t);
  });
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// LANES of a block a slice: a block, or a wave (short rows: 100 K rows of 1000 bf16 127 us with a block a row)
template <class T, int LANES, int NV, bool FULL>
__global__ __launch_bounds__(kBlock) void lp_bwd_kernel(const T* __restrict__ X, int64_t ldx, int64_t rows, int64_t cols,
                                                        int splits,
                                                        float c, float inv_t, int k, const int64_t* __restrict__ target64,
                                                        const int32_t* __restrict__ target32, int64_t ignore,
                                                        const int64_t* __restrict__ top_idx,
                                                        const float4* __restrict__ stats, const float* __restrict__ glogp,
                                                        const float* __restrict__ gent, const float* __restrict__ gtop,
                                                        T* __restrict__ GX) {
  constexpr int N = Vec<T>::N, LEN = LANES * NV * N;
  typedef typename Vec<T>::f32 F;
  const int tid = threadIdx.x & (LANES - 1);
  const int64_t part = (int64_t)blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
  const bool there = part < rows * splits;         // the last block of short rows holds fewer
  const int64_t row = there ? part / splits : 0;
  const int64_t c0 = there ? part % splits * LEN : cols;
  const T* x = X + row * ldx;
  T* gx = GX + row * cols;
  typename Vec<T>::raw raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t at = c0 + (v * LANES + tid) * N;
    if (at < cols) raw[v] = load_raw<T, FULL>(x + at, (int)min((int64_t)N, cols - at));
  }
  const float4 st = stats[row];
  const bool empty = st.y == __builtin_inff();
  const float m = empty ? 0.f : st.x, l2 = empty ? 0.f : st.y;
  const int64_t t = target64 ? target64[row] : (int64_t)target32[row];
  const bool asked = t != ignore && t >= 0 && t < cols;            // the target names a column
  const float gt = glogp && asked ? glogp[row] : 0.f;
  float g = gt;
  if (gtop)
    for (int i = 0; i < k; ++i) g += gtop[row * k + i];
  const float gh = gent ? gent[row] : 0.f;
  // gx = p (a + b log2 p) away from the named columns
  // (a row without probabilities: exp2(-inf) * 0)
  const float a = empty ? 0.f : -inv_t * (g + gh * st.z), b = empty ? 0.f : -inv_t * gh * kLn2;
  auto common = [&](float f) {
    const float q = fmaf(f - m, c, -l2);
    const float p = __builtin_amdgcn_exp2f(q);
    return p * fmaf(b, fmaxf(q, kFar), a);
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t at = c0 + (v * LANES + tid) * N;
    if (at < cols) {
      const F f = to_f32<T>(raw[v]);
      F y;
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = common(f[e]);
      store_f32<T, FULL>(gx + at, (int)min((int64_t)N, cols - at), y);
    }
  }
  // the named columns of this slice once more, with their own part: entry 0 is the target, the others the alternatives. One
  // thread a column: the first entry that names it adds up all that do.
  __threadfence_block();
  __syncthreads();
  const int named = 1 + (gtop ? k : 0);
  for (int i = tid; i < named; i += LANES) {
    const int64_t j = i ? top_idx[row * k + i - 1] : t;
    if (j < c0 || j >= min(cols, c0 + LEN) || empty || (i == 0 && !asked)) continue;
    if (i && j == t && asked) continue;
    float own = i ? gtop[row * k + i - 1] : gt;
    if (i == 0 && gtop)
      for (int h = 0; h < k; ++h)
        if (top_idx[row * k + h] == j) own += gtop[row * k + h];
    gx[j] = (T)(inv_t * own + common((float)x[j]));
  }
}

// ---- host -------------------------------------------------------------------------------------------------------------
struct Cut {
  int nv;          // vectors a thread
  int len;         // columns of a slice
  int64_t splits;
};

// Slices of 32 values a thread (with 64, two thirds of the waves fit: 8192 x 35598 bf16 forward 188 -> 150 us, 1024 x 18357 fp32
// with 50 alternatives 34 -> 28 us); shorter ones where that leaves fewer than 512 blocks: with 128 / 256 / 512 / 1024 instead, 1 x 1 M
// fp32 6.6 / 7.1 / 7.2 / 7.2 us and with 20 alternatives 12.3 / 13.5 / 13.6 / 13.4, 64 x 18357 6.6 / 6.6 / 6.7 / 7.3 and 12.2 / 11.3 / 11.9 /
// 12.2, 200 x 18357 7.2 / 7.1 / 7.1 / 7.4 and 13.6 / 13.6 / 13.7 / 14.5. Slices of a row are of equal length, to whole vectors.
Cut cut_for(int64_t rows, int64_t cols, int es) {
  const int n = 16 / es, most = 32 / n;
  Cut q{};
  for (q.nv = most; q.nv > 2; q.nv /= 2)
    if (rows * ((cols + kBlock * n * q.nv - 1) / (kBlock * n * q.nv)) >= 512) break;
  while (q.nv > 2 && (int64_t)kBlock * n * (q.nv / 2) >= cols) q.nv /= 2;
  const int64_t most_len = (int64_t)kBlock * n * q.nv;
  q.splits = (cols + most_len - 1) / most_len;
  q.len = (int)(((cols + q.splits - 1) / q.splits + n - 1) / n * n);
  q.splits = (cols + q.len - 1) / q.len;
  return q;
}

// Rows that a wave takes alone, 32 values a lane (50 000 x 500 bf16 forward 24 us, a block a row 88; x 2048 35 and 67; no slower
// for few rows).
bool short_rows(int64_t cols) { return cols <= 2048; }

size_t ws_bytes(int64_t rows, const Cut& q, int k) {
  if (q.splits == 1) return 16;
  const size_t sums = ((size_t)rows * q.splits * sizeof(Sums) + 15) / 16 * 16;
  return sums + (size_t)rows * q.splits * k * 8 + 16;
}

int check_common(int dtype, int64_t rows, int64_t cols, int target_bytes, int k, float temperature) {
  if (!known_dtype(dtype) || rows < 0 || cols < 1 || (target_bytes != 4 && target_bytes != 8) || k < 0) return MMSSL_E_BADARG;
  if (!(temperature > 0.f) || temperature > 3.0e38f || !(1.0f / temperature <= 3.0e38f)) return MMSSL_E_BADARG;
  if (k > kTopMax || k > cols || cols > 0x7ffffff0) return MMSSL_E_UNSUPP;
  // a row has at most ceil(cols / 2048) slices, so its pairs are counted in 32 bits
  if (rows > 0x7fffffff || !launchable(rows * ((cols + 2047) / 2048), kBlock)) return MMSSL_E_UNSUPP;
  return 0;
}

}  // namespace

extern "C" size_t mmssl_logprobs_rows_workspace_bytes(int dtype, int64_t rows, int64_t cols, int k) {
  if (check_common(dtype, rows, cols, 8, k, 1.0f)) return 0;
  return ws_bytes(rows, cut_for(rows, cols, dtype_bytes(dtype)), k);
}

extern "C" int mmssl_logprobs_rows(const void* X, int64_t ldx, int dtype, int64_t rows, int64_t cols, const void* target,
                                   int target_bytes, int64_t ignore_index, int k, float temperature, float* logp,
                                   float* entropy, float* top_logp, int64_t* top_idx, float* stats, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (int rc = check_common(dtype, rows, cols, target_bytes, k, temperature)) return rc;
  if (rows == 0) return 0;
  const size_t es = dtype_bytes(dtype);
  if (!X || !target || !logp || !entropy || ldx < 0 || (k > 0 && (!top_logp || !top_idx))) return MMSSL_E_BADARG;
  if (!aligned_to(X, es) || !aligned_to(target, target_bytes) || !aligned_to(stats, 16) || !aligned_to(top_idx, 8))
    return MMSSL_E_BADARG;
  const float c = (float)((double)kLog2e / temperature), inv_t = (float)(1.0 / (double)temperature);
  RowOut o{target_bytes == 8 ? static_cast<const int64_t*>(target) : nullptr,
           target_bytes == 4 ? static_cast<const int32_t*>(target) : nullptr,
           ignore_index, logp, entropy, top_logp, top_idx, reinterpret_cast<float4*>(stats)};
  const hipStream_t s = as_stream(stream);
  if (k == 0 && short_rows(cols)) {
    const dim3 grid((unsigned)((rows + kWaves - 1) / kWaves));
#define LP_SHORT_F(T, V, F)                                                                                              \
  hipLaunchKernelGGL((lp_short_kernel<T, V, F>), grid, dim3(kBlock), 0, s, (const T*)X, ldx, rows, (int)cols, c, inv_t, o)
#define LP_SHORT_V(T, V)                            \
  do {                                              \
    if (cols % Vec<T>::N == 0) LP_SHORT_F(T, V, true); \
    else LP_SHORT_F(T, V, false);                   \
  } while (0)
#define LP_SHORT(T)                                                       \
  do {                                                                    \
    if (cols <= 512) LP_SHORT_V(T, 8 / Vec<T>::N);                        \
    else if (cols <= 1024) LP_SHORT_V(T, 16 / Vec<T>::N);                 \
    else LP_SHORT_V(T, 32 / Vec<T>::N);                                   \
  } while (0)
    MMSSL_BY_DTYPE(dtype, LP_SHORT);
    MMSSL_LAUNCH_CHECK();
    return 0;
  }
  const Cut q = cut_for(rows, cols, (int)es);
  if (q.splits > 1 && (!workspace || !aligned_to(workspace, 16) || workspace_bytes < ws_bytes(rows, q, k)))
    return MMSSL_E_WORKSPACE;
  Sums* sums = static_cast<Sums*>(workspace);
  uint64_t* cand = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) +
                                               ((size_t)rows * q.splits * sizeof(Sums) + 15) / 16 * 16);
  const dim3 grid((unsigned)(rows * q.splits)), block(kBlock);
#define LP_SLICE_T(T, V, F, TOP)                                                                                         \
  hipLaunchKernelGGL((lp_slice_kernel<T, V, F, TOP>), grid, block, 0, s, (const T*)X, ldx, cols, q.len, (int)q.splits, c, \
                     inv_t, k, o, sums, cand)
#define LP_SLICE_V(T, V)                                         \
  if constexpr (V * Vec<T>::N <= 32) {                           \
    if (cols % Vec<T>::N == 0) {                                 \
      if (k) LP_SLICE_T(T, V, true, true);                       \
      else LP_SLICE_T(T, V, true, false);                        \
    } else {                                                     \
      if (k) LP_SLICE_T(T, V, false, true);                      \
      else LP_SLICE_T(T, V, false, false);                       \
    }                                                            \
  }
#define LP_SLICE(T)                      \
  switch (q.nv) {                        \
    case 8: LP_SLICE_V(T, 8); break;     \
    case 4: LP_SLICE_V(T, 4); break;     \
    default: LP_SLICE_V(T, 2); break;    \
  }
  MMSSL_BY_DTYPE(dtype, LP_SLICE);
  MMSSL_LAUNCH_CHECK();
  if (q.splits == 1) return 0;
#define LP_JOIN(T)                                                                                                       \
  if (k)                                                                                                                 \
    hipLaunchKernelGGL(lp_join_top_kernel<T>, dim3((unsigned)rows), block, (size_t)hold * 8, s, (const T*)X, ldx, cols,   \
                       (int)q.splits, c, inv_t, k, o, (const Sums*)sums, (const uint64_t*)cand, hold);                   \
  else                                                                                                                   \
    hipLaunchKernelGGL(lp_join_kernel<T>, dim3((unsigned)((rows * group + kBlock - 1) / kBlock)), block, 0, s,            \
                       (const T*)X, ldx, rows, cols, (int)q.splits, group, c, inv_t, o, (const Sums*)sums)
  const int hold = (int)std::min<int64_t>(q.splits * k, 2048);              // pairs in LDS: 16 KB at most
  int group = 1;
  while (group < 64 && group < q.splits) group *= 2;
  MMSSL_BY_DTYPE(dtype, LP_JOIN);
  MMSSL_LAUNCH_CHECK();
  return 0;
}

extern "C" int mmssl_logprobs_rows_bwd(const void* X, int64_t ldx, int dtype, int64_t rows, int64_t cols,
                                       const void* target, int target_bytes, int64_t ignore_index, int k,
                                       float temperature, const int64_t* top_idx, const float* stats, const float* glogp,
                                       const float* gentropy, const float* gtop, void* GX, void* stream) {
  if (int rc = check_common(dtype, rows, cols, target_bytes, k, temperature)) return rc;
  if (rows == 0) return 0;
  const size_t es = dtype_bytes(dtype);
  if (!X || !target || !stats || !GX || ldx < 0 || (gtop && (!top_idx || k < 1))) return MMSSL_E_BADARG;
  if (!aligned_to(X, es) || !aligned_to(GX, es) || !aligned_to(target, target_bytes) || !aligned_to(stats, 16) ||
      !aligned_to(top_idx, 8))
    return MMSSL_E_BADARG;
  const float c = (float)((double)kLog2e / temperature), inv_t = (float)(1.0 / (double)temperature);
  const int64_t* t64 = target_bytes == 8 ? static_cast<const int64_t*>(target) : nullptr;
  const int32_t* t32 = target_bytes == 4 ? static_cast<const int32_t*>(target) : nullptr;
  constexpr int NV = 4;
#define LP_BWD_F(T, L, F)                                                                                                \
  hipLaunchKernelGGL((lp_bwd_kernel<T, L, NV, F>), dim3((unsigned)((rows * splits + kBlock / L - 1) / (kBlock / L))),     \
                     dim3(kBlock), 0, as_stream(stream), (const T*)X, ldx, rows, cols, (int)splits, c, inv_t, k, t64,     \
                     t32, ignore_index, top_idx, (const float4*)stats, glogp, gentropy, gtop, (T*)GX)
#define LP_BWD_L(T, L)                                                          \
  do {                                                                          \
    const int64_t len = L * NV * Vec<T>::N, splits = (cols + len - 1) / len;    \
    if (cols % Vec<T>::N == 0) LP_BWD_F(T, L, true);                            \
    else LP_BWD_F(T, L, false);                                                 \
  } while (0)
  // a wave a row where one slice holds it (50 000 x 2048 bf16: 77 us, blocks 87; fp32, two slices: 144 against 137)
#define LP_BWD(T)                                        \
  do {                                                   \
    if (cols <= 64 * NV * Vec<T>::N) LP_BWD_L(T, 64);    \
    else LP_BWD_L(T, kBlock);                            \
  } while (0)
  MMSSL_BY_DTYPE(dtype, LP_BWD);
  MMSSL_LAUNCH_CHECK();
  return 0;
}
