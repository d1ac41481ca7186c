// Row lookup with scaling, and its gradient by sorted tokens.
//
//   out[i, :] = scale * table[idx[i], :]            gW[v, :] = scale * sum over i with idx[i] = v of g[i, :]
//
// The gradient adds the rows of equal tokens in a fixed order: the places are sorted by token (stable), the sorted list is cut
// into equal chunks, a lane group walks a chunk and keeps the running sum of the token it is at. A sum that lies inside a
// chunk is written at once; one that crosses a chunk's border leaves a partial row that a last launch joins, in the
// chunks' order or, over more than 16 of them, lane group by lane group. No float atomics: the same call gives the same bits.
//
// Both directions are bound by memory where they are large: 1 000 003 places of 1 M x 128 bf16 look up in 83 us (457 MB moved, 5.5
// TB/s), are summed in 127 us (590 MB, 4.6 TB/s, rows at random) after three radix passes of 23 us each (latency: the pairs are 8
// MB and come from the caches) and joined in 13. 1024 rows of 64 fp32 look up in 3.5 us, a launch.
#include <algorithm>

#include "typed.hpp"

using namespace mmssl;

namespace {

// Up to here the places are ranked by counting (one launch, quadratic work), above by radix passes. The whole gradient into 18357 x
// 64 fp32: 4096 places 18 against 21 us, 8192 24 against 23, 16384 35 against 25. Other tables, 2048 and 8192 places: 200 rows (one pass
// instead of two) 16 and 26 against 15 and 19, 18357 x 1024 26 and 38 against 30 and 36, 1 M x 64 (three) 45 and 54 against 56 and 59.
constexpr int kRankMax = 8192;
constexpr int kSortThreads = 1024;
constexpr int kSortBlocks = 256;
constexpr int kRankTile = 4096;
constexpr int kZeroRowsMax = 2048;
constexpr int kScanMax = 4096;       // places that a block looks through for rows without a token: 16 rounds

struct IdxRule {
  int rows;            // tokens in [0, rows) are looked up ...
  int has_pad;
  int64_t pad;         // ... but for this one
};

// the sort key of a token: the token, or `rows` for one without a row (padding, out of range)
template <class I>
__device__ __forceinline__ int key_of(I v, IdxRule q) {
  const int64_t x = (int64_t)v;
  return (x >= 0 && x < q.rows && !(q.has_pad && x == q.pad)) ? (int)x : q.rows;
}

// ---- lookup ---------------------------------------------------------------------------------------------------------
template <class T, class I, int LPR, int U, bool FULL>
__global__ __launch_bounds__(kBlock) void embed_fwd_kernel(const T* __restrict__ table, int64_t ldt, int d,
                                                           const I* __restrict__ idx, int64_t n, IdxRule q, float scale,
                                                           T* __restrict__ out, int64_t ldo) {
  constexpr int N = Vec<T>::N;
  const int lig = threadIdx.x & (LPR - 1);
  const int64_t first = ((int64_t)blockIdx.x * (kBlock / LPR) + threadIdx.x / LPR) * U;
  if (first >= n) return;
  int64_t row[U];
  float fill[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    row[u] = -1;
    fill[u] = 0.f;
    if (first + u < n) {
      const int64_t v = (int64_t)idx[first + u];
      if (!(q.has_pad && v == q.pad)) {
        if (v >= 0 && v < q.rows) row[u] = v;
        else fill[u] = __builtin_nanf("");
      }
    }
  }
  for (int c = lig * N; c < d; c += LPR * N) {
    typename Vec<T>::raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row[u] >= 0) v[u] = load_raw<T, FULL>(table + row[u] * ldt + c, d - c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u < n) {
        typename Vec<T>::f32 f;
        if (row[u] >= 0) f = to_f32<T>(v[u]) * scale;
        else f = fill[u];
        store_f32<T, FULL>(out + (first + u) * ldo + c, d - c, f);
      }
  }
}

// Rows of up to 64 vectors that do not fill a lane group of a power of two: a block's threads share the vectors of its tokens
// evenly (20 M fp32 values at width 65: lane groups 38 us, so 30; where the groups are full they are faster, 1 M rows of 128
// bf16: 82 against 93 us).
// magic = ceil(2^20 / vecs): (l * magic) >> 20 = l / vecs for every l < kFlat = 2^10 (the error l * 64 stays below 2^20, the
// product at or below 2^30).
constexpr int kFlatU = 4, kFlat = kBlock * kFlatU;

template <class T, class I, bool FULL>
__global__ __launch_bounds__(kBlock) void embed_fwd_flat_kernel(const T* __restrict__ table, int64_t ldt, int d, int vecs,
                                                                uint32_t magic, int tokens, const I* __restrict__ idx,
                                                                int64_t n, IdxRule q, float scale, T* __restrict__ out,
                                                                int64_t ldo) {
  constexpr int N = Vec<T>::N;
  const int64_t first = (int64_t)blockIdx.x * tokens;
  const int mine = (int)min((int64_t)tokens, n - first) * vecs;
  int64_t row[kFlatU], at[kFlatU];
  int col[kFlatU];
  float fill[kFlatU];
#pragma unroll
  for (int u = 0; u < kFlatU; ++u) {
    const uint32_t l = u * kBlock + threadIdx.x;
    const uint32_t t = (l * magic) >> 20;
    col[u] = (int)(l - t * vecs) * N;
    at[u] = first + t;
    row[u] = -1;
    fill[u] = 0.f;
    if ((int)l < mine) {
      const int64_t v = (int64_t)idx[at[u]];
      if (!(q.has_pad && v == q.pad)) {
        if (v >= 0 && v < q.rows) row[u] = v;
        else fill[u] = __builtin_nanf("");
      }
    }
  }
  typename Vec<T>::raw v[kFlatU];
#pragma unroll
  for (int u = 0; u < kFlatU; ++u)
    if (row[u] >= 0) v[u] = load_raw<T, FULL>(table + row[u] * ldt + col[u], d - col[u]);
#pragma unroll
  for (int u = 0; u < kFlatU; ++u)
    if ((int)(u * kBlock + threadIdx.x) < mine) {
      typename Vec<T>::f32 f;
      if (row[u] >= 0) f = to_f32<T>(v[u]) * scale;
      else f = fill[u];
      store_f32<T, FULL>(out + at[u] * ldo + col[u], d - col[u], f);
    }
}

// ---- places by token ------------------------------------------------------------------------------------------------
// KP: (key, place) pairs, one 8-byte access each.
// n <= kRankMax: a place's position in the sorted list is the number of places before it, (key, place) compared as a pair.
// One block ranks 64 places (a lane each), its 16 waves count a sixteenth of the list each.
template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_rank_kernel(const I* __restrict__ idx, int n, IdxRule q,
                                                                  int2* __restrict__ KP) {
  __shared__ int4 keys4[kRankTile / 4];
  __shared__ int cnt[64];
  int* keys = reinterpret_cast<int*>(keys4);
  constexpr int kSpan = kRankTile / (kSortThreads / 64);        // 256 keys of a tile for each wave
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int lo = blockIdx.x * 64, i = lo + lane;
  const int mine = i < n ? key_of(idx[i], q) : 0;
  if (threadIdx.x < 64) cnt[threadIdx.x] = 0;
  int c = 0;
  for (int t0 = 0; t0 < n; t0 += kRankTile) {
    __syncthreads();
    for (int j = threadIdx.x; j < kRankTile; j += kSortThreads)
      keys[j] = t0 + j < n ? key_of(idx[t0 + j], q) : 0x7fffffff;
    __syncthreads();
    const int base = t0 + w * kSpan;
    if (base < n) {
      const int4* p = keys4 + w * (kSpan / 4);
      if (base + kSpan <= lo || base > lo + 63) {
        const int bound = base > lo + 63 ? mine : mine + 1;     // behind: smaller keys; before: equal ones too
#pragma unroll 8
        for (int j = 0; j < kSpan / 4; ++j) {
          const int4 k = p[j];
          c += (k.x < bound) + (k.y < bound) + (k.z < bound) + (k.w < bound);
        }
      } else {
#pragma unroll 4
        for (int j = 0; j < kSpan / 4; ++j) {
          const int4 k = p[j];
          const int at = base + 4 * j;
          c += (k.x < mine + (at < i)) + (k.y < mine + (at + 1 < i)) + (k.z < mine + (at + 2 < i)) +
               (k.w < mine + (at + 3 < i));
        }
      }
    }
  }
  atomicAdd(&cnt[lane], c);
  __syncthreads();
  if (w == 0 && i < n) {
    const int r = cnt[lane];
    KP[r] = make_int2(mine, i);
  }
}

// Radix passes of up to 8 bits from the low end; block b owns the places [b * per, (b + 1) * per).
template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_hist_kernel(const I* __restrict__ idx, const int2* __restrict__ in,
                                                                  int64_t n, IdxRule q, int64_t per, int shift, int mask,
                                                                  int* __restrict__ H) {
  __shared__ int h[256];
  if (threadIdx.x < 256) h[threadIdx.x] = 0;
  __syncthreads();
  const int64_t a = (int64_t)blockIdx.x * per, b = min(n, a + per);
  for (int64_t i = a + threadIdx.x; i < b; i += kSortThreads) {
    const int k = in ? in[i].x : key_of(idx[i], q);
    atomicAdd(&h[(k >> shift) & mask], 1);
  }
  __syncthreads();
  if (threadIdx.x < 256) H[(int64_t)blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}

template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_scatter_kernel(const I* __restrict__ idx, const int2* __restrict__ in,
                                                                     int64_t n, IdxRule q, int64_t per, int shift, int mask,
                                                                     const int* __restrict__ H, int2* __restrict__ out) {
  constexpr int kWaves = kSortThreads / 64, kTile = kSortThreads;      // (four pairs a thread from 256 K places on: the same time)
  __shared__ int wc[kWaves][256];      // counts, then the next place of a wave's run of a digit
  __shared__ int base[256];
  __shared__ int wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t a = (int64_t)blockIdx.x * per, b = min(n, a + per);
  int2 e;                              // (key, place); key -1: behind the block's places
  auto load = [&](int64_t t0) {
    const int64_t i = t0 + tid;
    e = make_int2(-1, 0);
    if (i < b) e = in ? in[i] : make_int2(key_of(idx[i], q), (int)i);
  };
  load(a);                             // the first tile arrives under the counts
  // where this block's run of each digit begins: all smaller digits + this digit in the blocks before
  {
    const int dig = tid & 255, part = tid >> 8, nb = gridDim.x;
    const int k0 = part * nb / 4, k1 = (part + 1) * nb / 4;
    int tot = 0, pre = 0;
#pragma unroll 16
    for (int k = k0; k < k1; ++k) {
      const int c = H[(int64_t)k * 256 + dig];
      tot += c;
      pre += k < (int)blockIdx.x ? c : 0;
    }
    wc[part][dig] = tot;
    wc[part + 4][dig] = pre;
  }
  __syncthreads();
  if (tid < 256) {
    const int tot = (wc[0][tid] + wc[1][tid]) + (wc[2][tid] + wc[3][tid]);
    const int pre = (wc[4][tid] + wc[5][tid]) + (wc[6][tid] + wc[7][tid]);
    int s = tot;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(s, m, 64);
      if (lane >= m) s += o;
    }
    if (lane == 63) wsum[w] = s;
    base[tid] = s - tot + pre;
  }
  __syncthreads();
  if (tid < 256) {
    int add = 0;
    for (int k = 0; k < w; ++k) add += wsum[k];
    base[tid] += add;
  }
  for (int64_t t0 = a; t0 < b; t0 += kTile) {
    __syncthreads();
    for (int k = tid; k < kWaves * 256; k += kSortThreads) wc[k >> 8][k & 255] = 0;
    __syncthreads();
    const int dig = (e.x >> shift) & mask;
    uint64_t m = __ballot(e.x >= 0);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const uint64_t on = __ballot((dig >> bit) & 1);
      m &= ((dig >> bit) & 1) ? on : ~on;
    }
    // the wave's lanes with this lane's digit: their number is the digit's count, those before this lane its place among them
    const int off = __popcll(m & ((1ull << lane) - 1));
    if (e.x >= 0 && off == 0) wc[w][dig] = __popcll(m);
    __syncthreads();
    if (tid < 256) {
      int run = base[tid];
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const int c = wc[k][tid];
        wc[k][tid] = run;
        run += c;
      }
      base[tid] = run;
    }
    __syncthreads();
    if (e.x >= 0) out[wc[w][dig] + off] = e;
    if (t0 + kTile < b) load(t0 + kTile);
  }
}

// ---- sums of equal tokens -------------------------------------------------------------------------------------------
// first place in the sorted KP[0, n) whose key is >= x; 256 probes a round, three rounds for 16 M places
__device__ __forceinline__ int64_t block_lower_bound(const int2* __restrict__ KP, int64_t n, int x) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t s = (hi - lo + kBlock - 1) / kBlock;
    const int64_t p = lo + (threadIdx.x + 1) * s - 1;
    const int c = __syncthreads_count(p < hi && KP[p].x < x);
    lo += c * s;
    hi = min(hi, lo + s - 1);
  }
  return lo;
}

// Blocks [0, rblocks): chunks of the sorted list, LPR lanes a chunk, `ctiles` column tiles of LPR vectors.
// The others: zrows table rows each; rows without a token are written as zeros.
// part = [2][chunks][d] fp32: the sum of a chunk's first token where it began before the chunk, and of its last token where
// that began in the chunk and goes on behind it.
template <class T, int LPR, bool FULL>
__global__ __launch_bounds__(kBlock) void embed_grad_kernel(const int2* __restrict__ KP, int64_t n,
                                                            int rows, int d, const T* __restrict__ g, int64_t ldg,
                                                            float scale, T* __restrict__ gW, float* __restrict__ part,
                                                            int chunk, int64_t chunks, int ctiles, int64_t rblocks,
                                                            int zrows) {
  constexpr int N = Vec<T>::N, B = FULL ? 8 : 4;    // partial vectors cost registers: 240 with 8 rows in flight
  typedef typename Vec<T>::f32 F;
  const int lig = threadIdx.x & (LPR - 1);
  if ((int64_t)blockIdx.x < rblocks) {
    const int64_t w = (int64_t)(blockIdx.x / ctiles) * (kBlock / LPR) + threadIdx.x / LPR;
    if (w >= chunks) return;
    const int col = ((int)(blockIdx.x % ctiles) * LPR + lig) * N;
    const int left = d - col;
    if (left <= 0) return;
    const int64_t a = w * chunk, b = min(n, a + chunk);
    int cur = KP[a].x;
    if (cur >= rows) return;                       // the keys without a row come last
    bool head = a > 0 && KP[a - 1].x == cur;
    F acc = 0.f;
    for (int64_t p0 = a; p0 < b; p0 += B) {
      int key[B], pos[B];
#pragma unroll
      for (int u = 0; u < B; u += 2) {             // KP is padded to whole batches; chunks start at multiples of B
        const int4 two = *reinterpret_cast<const int4*>(KP + p0 + u);
        key[u] = two.x; pos[u] = two.y;
        key[u + 1] = two.z; pos[u + 1] = two.w;
      }
      typename Vec<T>::raw v[B];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (p0 + u >= b) key[u] = rows;
        if (key[u] < rows) v[u] = load_raw<T, FULL>(g + (int64_t)pos[u] * ldg + col, left);
      }
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (key[u] < rows) {
          if (key[u] != cur) {
            if (head) store_part<N, FULL>(part + w * d + col, left, acc);
            else store_f32<T, FULL>(gW + (int64_t)cur * d + col, left, acc * scale);
            head = false;
            cur = key[u];
            acc = 0.f;
          }
          acc += to_f32<T>(v[u]);
        }
      }
    }
    const bool on = b < n && KP[b].x == cur;
    if (head) store_part<N, FULL>(part + w * d + col, left, acc);
    else if (on) store_part<N, FULL>(part + (chunks + w) * d + col, left, acc);
    else store_f32<T, FULL>(gW + (int64_t)cur * d + col, left, acc * scale);
    return;
  }
  __shared__ uint32_t seen[kZeroRowsMax / 32];
  const int64_t r0 = ((int64_t)blockIdx.x - rblocks) * zrows;
  const int nr = (int)min((int64_t)zrows, (int64_t)rows - r0);
  for (int k = threadIdx.x; k < kZeroRowsMax / 32; k += kBlock) seen[k] = 0;
  const int64_t lo = block_lower_bound(KP, n, (int)r0), hi = block_lower_bound(KP, n, (int)(r0 + nr));
  __syncthreads();
  if (hi - lo <= kScanMax) {
    for (int64_t i = lo + threadIdx.x; i < hi; i += kBlock) {
      const int r = KP[i].x - (int)r0;
      atomicOr(&seen[r >> 5], 1u << (r & 31));
    }
  } else {                                         // popular tokens: each row is searched for instead
    for (int r = threadIdx.x; r < nr; r += kBlock) {
      const int x = (int)r0 + r;
      int64_t a = lo, b = hi;                      // the first place whose key is >= x
      while (a < b) {
        const int64_t mid = (a + b) >> 1;
        if (KP[mid].x < x) a = mid + 1;
        else b = mid;
      }
      if (a < hi && KP[a].x == x) atomicOr(&seen[r >> 5], 1u << (r & 31));
    }
  }
  __syncthreads();
  const F z = 0.f;
  for (int r = threadIdx.x / LPR; r < nr; r += kBlock / LPR)
    if (!(seen[r >> 5] >> (r & 31) & 1))
      for (int c = lig * N; c < d; c += LPR * N) store_f32<T, FULL>(gW + (r0 + r) * d + c, d - c, z);
}

// A chunk whose last token begins in it and goes on behind it joins that token's partial rows, in the chunks' order. Up to
// kShort following chunks: the chunk's lane group alone; more: the whole block, its groups taking every GPB-th chunk (131 072 places,
// popular tokens: 40 us with 2 or 16, 51 with 64).
template <class T, int LPR, bool FULL>
__global__ __launch_bounds__(kBlock) void embed_join_kernel(const int2* __restrict__ KP, int64_t n, int rows, int d,
                                                            float scale, T* __restrict__ gW,
                                                            const float* __restrict__ part, int chunk, int64_t chunks,
                                                            int ctiles) {
  constexpr int N = Vec<T>::N, GPB = kBlock / LPR, kShort = 16;
  typedef typename Vec<T>::f32 F;
  __shared__ F red[kBlock];
  __shared__ int64_t long_w[GPB];
  __shared__ int64_t long_m[GPB];
  __shared__ int n_long;
  const int lig = threadIdx.x & (LPR - 1), grp = threadIdx.x / LPR;
  const int64_t w = (int64_t)(blockIdx.x / ctiles) * GPB + grp;
  const int col = ((int)(blockIdx.x % ctiles) * LPR + lig) * N;
  const int left = d - col;
  if (threadIdx.x == 0) n_long = 0;
  bool mine = false;
  int cur = rows;
  if (w < chunks - 1) {
    const int64_t a = w * chunk, b = a + chunk;
    cur = KP[b - 1].x;
    mine = cur < rows && KP[b].x == cur && (KP[a].x != cur || a == 0 || KP[a - 1].x != cur);
  }
  // number of following chunks that begin with the token: the next LPR at once, then a search, LPR probes a round
  auto leading = [&](bool hit) {                 // how many lanes of the group from the first on
    const uint64_t bal = __ballot(hit) >> ((threadIdx.x & 63) / LPR * LPR);
    const uint64_t miss = LPR == 64 ? ~bal : (~bal & ((1ull << (LPR & 63)) - 1));
    return miss ? __ffsll((unsigned long long)miss) - 1 : LPR;
  };
  int64_t lo = w + 1, hi;
  {
    const int64_t c = lo + lig;
    const int run = leading(mine && c < chunks && KP[c * chunk].x == cur);
    lo += run;
    hi = mine && run == LPR ? chunks : lo;
  }
  while (__any(lo < hi)) {
    const int64_t step = (hi - lo + LPR - 1) / LPR, c = lo + (lig + 1) * step - 1;
    const int run = leading(lo < hi && c < hi && KP[c * chunk].x == cur);
    if (lo < hi) {
      lo += run * step;
      hi = min(hi, lo + step - 1);
    }
  }
  const int64_t m = mine ? lo - (w + 1) : 0;
  __syncthreads();
  if (mine && m > kShort) {
    if (lig == 0) {
      const int s = atomicAdd(&n_long, 1);
      long_w[s] = w;
      long_m[s] = m;
    }
  } else if (mine && left > 0) {
    F acc = load_part<N, F, FULL>(part + (chunks + w) * d + col, left);
    for (int64_t j = 1; j <= m; ++j) acc += load_part<N, F, FULL>(part + (w + j) * d + col, left);
    store_f32<T, FULL>(gW + (int64_t)cur * d + col, left, acc * scale);
  }
  __syncthreads();
  for (int s = 0; s < n_long; ++s) {
    const int64_t lw = long_w[s], lm = long_m[s];
    F acc = 0.f;
    if (left > 0) {
#pragma unroll 8
      for (int64_t j = 1 + grp; j <= lm; j += GPB) acc += load_part<N, F, FULL>(part + (lw + j) * d + col, left);
    }
    red[threadIdx.x] = acc;
    __syncthreads();
    if (grp == 0 && left > 0) {
      F sum = load_part<N, F, FULL>(part + (chunks + lw) * d + col, left);
#pragma unroll
      for (int k = 0; k < GPB; ++k) sum += red[k * LPR + lig];
      store_f32<T, FULL>(gW + (int64_t)KP[lw * chunk + chunk - 1].x * d + col, left, sum * scale);
    }
    __syncthreads();
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
int lanes_for(int vecs) { return vecs <= 8 ? 8 : vecs <= 16 ? 16 : vecs <= 32 ? 32 : 64; }

struct Plan {
  bool ranked;
  int passes, bits;          // radix: number of passes, bits of each
  int64_t per, blocks;       // radix: places of a block (whole tiles), blocks
  int chunk;
  int64_t chunks;
  int64_t npad;              // (key, place) pairs, whole batches
  size_t bytes, off_hist, off_part;
};

Plan plan_for(int64_t rows, int d, int64_t n) {
  Plan p{};
  p.ranked = n <= kRankMax;
  int bits = 1;
  while (bits < 31 && (rows >> bits)) ++bits;              // keys run from 0 to `rows`
  p.passes = (bits + 7) / 8;
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t tiles = (n + kSortThreads - 1) / kSortThreads;
  p.per = (tiles + kSortBlocks - 1) / kSortBlocks * kSortThreads;
  p.blocks = n ? (n + p.per - 1) / p.per : 0;
  // places of a chunk: longer ones leave fewer partial rows, shorter ones more lanes at work. The whole gradient into 18357 x 64
  // fp32 with 8 / 16 / 64: 8192 places 25 / 25 / 37 us, 51200 32 / 32 / 44, 524288 78 / 71 / 58. At other widths: 8 columns, 8192
  // places 29 / 30 / 41, 524287 88 / 83 / 81; 1024 columns 38 / 37 / 49 and 674 / 580 / 510 (65536 places 107 / 98 / 93: wide rows would
  // gain up to 12 % from 64 earlier, the rule does not look at the width).
  p.chunk = n >= (1 << 19) ? 64 : n >= (1 << 15) ? 16 : 8;
  p.chunks = (n + p.chunk - 1) / p.chunk;
  p.npad = (n + 15) / 16 * 16;
  const size_t lists = (size_t)p.npad * (p.ranked ? 8 : 16);
  p.off_hist = lists;
  p.off_part = p.off_hist + (p.ranked ? 0 : (size_t)p.blocks * 256 * 4);
  p.bytes = p.off_part + (size_t)p.chunks * 2 * d * 4 + 16;
  return p;
}

template <class I>
int sort_places(const I* idx, int64_t n, IdxRule q, const Plan& p, char* ws, const int2** sorted, hipStream_t s) {
  int2* KP[2] = {reinterpret_cast<int2*>(ws), reinterpret_cast<int2*>(ws) + p.npad};
  *sorted = KP[0];
  if (n == 0) return 0;
  if (p.ranked) {
    hipLaunchKernelGGL(embed_rank_kernel<I>, dim3((unsigned)((n + 63) / 64)), dim3(kSortThreads), 0, s, idx, (int)n, q, KP[0]);
    MMSSL_LAUNCH_CHECK();
    return 0;
  }
  int* H = reinterpret_cast<int*>(ws + p.off_hist);
  const int2* in = nullptr;
  const int mask = (1 << p.bits) - 1;
  for (int k = 0; k < p.passes; ++k) {
    const dim3 grid((unsigned)p.blocks), block(kSortThreads);
    hipLaunchKernelGGL(embed_hist_kernel<I>, grid, block, 0, s, idx, in, n, q, p.per, k * p.bits, mask, H);
    MMSSL_LAUNCH_CHECK();
    hipLaunchKernelGGL(embed_scatter_kernel<I>, grid, block, 0, s, idx, in, n, q, p.per, k * p.bits, mask, H, KP[k & 1]);
    MMSSL_LAUNCH_CHECK();
    in = *sorted = KP[k & 1];
  }
  return 0;
}

template <class T, int LPR, bool FULL>
int grad_launch(const int2* KP, int64_t n, int rows, int d, const T* g, int64_t ldg, float scale, T* gW,
                float* part, const Plan& p, hipStream_t s) {
  const int vecs = (d + Vec<T>::N - 1) / Vec<T>::N;
  const int ctiles = (vecs + LPR - 1) / LPR;
  const int64_t groups = (p.chunks + kBlock / LPR - 1) / (kBlock / LPR);
  const int64_t rblocks = groups * ctiles;
  const int zrows = (int)std::max<int64_t>(32, std::min<int64_t>(kZeroRowsMax, (64 << 10) / ((int64_t)d * sizeof(T))));
  const int64_t zblocks = ((int64_t)rows + zrows - 1) / zrows;
  if (!launchable(rblocks + zblocks, kBlock)) return MMSSL_E_UNSUPP;
  if (rblocks + zblocks == 0) return 0;
  hipLaunchKernelGGL((embed_grad_kernel<T, LPR, FULL>), dim3((unsigned)(rblocks + zblocks)), dim3(kBlock), 0, s, KP, n, rows, d,
                     g, ldg, scale, gW, part, p.chunk, p.chunks, ctiles, rblocks, zrows);
  MMSSL_LAUNCH_CHECK();
  if (p.chunks > 1) {
    hipLaunchKernelGGL((embed_join_kernel<T, LPR, FULL>), dim3((unsigned)rblocks), dim3(kBlock), 0, s, KP, n, rows, d, scale, gW,
                       (const float*)part, p.chunk, p.chunks, ctiles);
    MMSSL_LAUNCH_CHECK();
  }
  return 0;
}

int check_common(int dtype, int64_t rows, int d, int64_t n, int idx_bytes) {
  if (!known_dtype(dtype) || rows < 0 || d < 1 || n < 0 || (idx_bytes != 4 && idx_bytes != 8)) return MMSSL_E_BADARG;
  // rows and places are 32-bit keys; a row's columns are counted in 32 bits
  if (rows > 0x7ffffffe || n > 0x7ffffff0 || d > (1 << 24)) return MMSSL_E_UNSUPP;
  return 0;
}

}  // namespace

extern "C" int mmssl_embed_rows(const void* table, int64_t ldt, int dtype, int64_t rows, int d, const void* idx,
                                int idx_bytes, int64_t n, float scale, int has_padding, int64_t padding_idx, void* out,
                                int64_t ldo, void* stream) {
  if (int rc = check_common(dtype, rows, d, n, idx_bytes)) return rc;
  if (n == 0) return 0;
  if ((!table && rows > 0) || !idx || !out || ldt < 0 || ldo < d) return MMSSL_E_BADARG;
  const size_t es = dtype_bytes(dtype);
  if (!aligned_to(table, es) || !aligned_to(out, es) || !aligned_to(idx, idx_bytes)) return MMSSL_E_BADARG;
  const IdxRule q{(int)rows, has_padding ? 1 : 0, padding_idx};
  const int vecs = (int)((d + 16 / es - 1) / (16 / es)), lpr = lanes_for(vecs);
  const bool flat = vecs < lpr;
  constexpr int U = 4;
  const int tokens = flat ? kFlat / vecs : kBlock / lpr * U;                // of a block
  const int64_t blocks = (n + tokens - 1) / tokens;
  const uint32_t magic = ((1u << 20) + vecs - 1) / vecs;
#define EMBED_FWD_L(T, I, L, F)                                                                                          \
  hipLaunchKernelGGL((embed_fwd_kernel<T, I, L, U, F>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),       \
                     (const T*)table, ldt, d, (const I*)idx, n, q, scale, (T*)out, ldo)
#define EMBED_FWD_F(T, I, F)                                                                                             \
  if (flat)                                                                                                              \
    hipLaunchKernelGGL((embed_fwd_flat_kernel<T, I, F>), dim3((unsigned)blocks), dim3(kBlock), 0, as_stream(stream),      \
                       (const T*)table, ldt, d, vecs, magic, tokens, (const I*)idx, n, q, scale, (T*)out, ldo);          \
  else if (lpr == 8) EMBED_FWD_L(T, I, 8, F);                                                                            \
  else if (lpr == 16) EMBED_FWD_L(T, I, 16, F);                                                                          \
  else if (lpr == 32) EMBED_FWD_L(T, I, 32, F);                                                                          \
  else EMBED_FWD_L(T, I, 64, F)
#define EMBED_FWD(T)                                         \
  do {                                                       \
    const bool full = d % Vec<T>::N == 0;                    \
    if (idx_bytes == 8 && full) { EMBED_FWD_F(T, int64_t, true); } \
    else if (idx_bytes == 8) { EMBED_FWD_F(T, int64_t, false); }   \
    else if (full) { EMBED_FWD_F(T, int32_t, true); }        \
    else { EMBED_FWD_F(T, int32_t, false); }                 \
  } while (0)
  if (!launchable(blocks, kBlock)) return MMSSL_E_UNSUPP;
  MMSSL_BY_DTYPE(dtype, EMBED_FWD);
  MMSSL_LAUNCH_CHECK();
  return 0;
}

extern "C" size_t mmssl_embed_rows_bwd_workspace_bytes(int64_t rows, int d, int64_t n) {
  if (rows < 0 || rows > 0x7ffffffe || d < 1 || d > (1 << 24) || n < 0 || n > 0x7ffffff0) return 0;
  return plan_for(rows, d, n).bytes;
}

extern "C" int mmssl_embed_rows_bwd(const void* g, int64_t ldg, int dtype, const void* idx, int idx_bytes, int64_t n,
                                    int64_t rows, int d, float scale, int has_padding, int64_t padding_idx, void* grad,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_common(dtype, rows, d, n, idx_bytes)) return rc;
  if (rows == 0) return 0;
  if (!grad || ldg < 0 || (n > 0 && (!g || !idx))) return MMSSL_E_BADARG;
  const size_t es = dtype_bytes(dtype);
  if (!aligned_to(grad, es) || !aligned_to(g, es) || (n > 0 && !aligned_to(idx, idx_bytes))) return MMSSL_E_BADARG;
  const Plan p = plan_for(rows, d, n);
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < p.bytes) return MMSSL_E_WORKSPACE;
  const IdxRule q{(int)rows, has_padding ? 1 : 0, padding_idx};
  const hipStream_t s = as_stream(stream);
  char* ws = static_cast<char*>(workspace);
  const int2* KP = nullptr;
  const int rc = idx_bytes == 8 ? sort_places((const int64_t*)idx, n, q, p, ws, &KP, s)
                                : sort_places((const int32_t*)idx, n, q, p, ws, &KP, s);
  if (rc) return rc;
  float* part = reinterpret_cast<float*>(ws + p.off_part);
  const int lpr = lanes_for((d + (int)(16 / es) - 1) / (int)(16 / es));
#define EMBED_GRAD_L(T, L)                                                                                              \
  return d % Vec<T>::N == 0                                                                                              \
             ? grad_launch<T, L, true>(KP, n, (int)rows, d, (const T*)g, ldg, scale, (T*)grad, part, p, s)             \
             : grad_launch<T, L, false>(KP, n, (int)rows, d, (const T*)g, ldg, scale, (T*)grad, part, p, s)
#define EMBED_GRAD(T)               \
  switch (lpr) {                    \
    case 8: EMBED_GRAD_L(T, 8);     \
    case 16: EMBED_GRAD_L(T, 16);   \
    case 32: EMBED_GRAD_L(T, 32);   \
    default: EMBED_GRAD_L(T, 64);   \
  }
  MMSSL_BY_DTYPE(dtype, EMBED_GRAD);
  return 0;
}
