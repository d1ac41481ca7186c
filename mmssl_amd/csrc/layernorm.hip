// Layer norm over the rows of X [rows, d], its backward pass and the gradients of weight and bias.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b
//   gx = r (q - mean(q) - h mean(q h)),  q = gy w;      gw = sum over rows of gy h,  gb = sum over rows of gy
//
// All three directions stream their operands once: a row lives in the registers of a lane group (up to 16 values a lane;
// the variance is taken around the mean in a second sweep over the registers, so nothing cancels), the columns a lane holds
// are the same for every row, so the weight stays in registers and the weight's gradient adds up there over the rows of a
// block; the blocks' partial sums meet in a second launch in a fixed order. Rows longer than 16384 are swept from memory.
//
// Bound by memory: 65536 x 4096 bf16 forward 206 us (1.07 GB, 5.2 TB/s; best of 15 launches 199), backward 317 (1.61 GB, 5.1 TB/s;
// best 297) and 8 for the parameters' sums; 51197 x 256 fp32 21 + 27 + 4 us; 1024 x 64 fp32 3.2, a launch. Rows of 20000 fp32: 3.4 and 2.3 TB/s.
#include <algorithm>

#include "typed.hpp"

using namespace mmssl;

namespace {

constexpr int kMaxInRegs = 16384;

// How a row ends: with a whole vector; with a part of one, which is then the last N columns of the row (its first `skip`
// columns are the vector before's too: left out of the sums, written twice with the same values); or element by element: rows
// shorter than a vector, and fp32 backward, where three single elements cost less than the bookkeeping (233 K rows of 257: 155
// against 172 us; bf16, seven: 150 against 95 us, forward 84 against 72).
enum Tail { kWhole, kShared, kShort };

// LPR lanes a row (a power of two; above 64 whole waves of one block), NV vectors a lane: vector v of lane l holds the
// columns [(v * LPR + l) * N, + N). (As many waves as the row needs instead of a power of two: rows of 4097 bf16 backward 142 ->
// 113 us, but the row sums over a number of waves known only at run time cost every other width: 8192 91 -> 115, 6000 93 -> 120.)
template <class T, int LPR, int NV, Tail TAIL>
struct RowTile {
  static constexpr int N = Vec<T>::N;
  static constexpr int TPB = LPR > 64 ? LPR : kBlock;      // a row of several waves has its block to itself
  static constexpr int GPB = TPB / LPR;          // rows of a block at a time
  static constexpr int WPR = LPR > 64 ? LPR / 64 : 1;
  typedef typename Vec<T>::f32 F;
  typedef typename Vec<T>::raw R;

  // first column, moved back where the row ends inside the vector, and how many of its columns the vector before holds (N:
  // nothing of the row is here)
  __device__ static __forceinline__ int col(int v, int lig, int d) {
    const int c = (v * LPR + lig) * N;
    return TAIL == kShared ? min(c, d - N) : c;
  }
  __device__ static __forceinline__ int skip(int v, int lig, int d) {
    return TAIL == kShared ? min((v * LPR + lig) * N - col(v, lig, d), N) : 0;
  }
  __device__ static __forceinline__ bool there(int v, int lig, int d) { return (v * LPR + lig) * N < d; }
  // is element k the row's, and this vector's alone
  __device__ static __forceinline__ bool own(int v, int lig, int d, int k) {
    if (TAIL == kWhole) return there(v, lig, d);
    if (TAIL == kShort) return col(v, lig, d) + k < d;
    return k >= skip(v, lig, d);
  }

  __device__ static __forceinline__ void load(const T* __restrict__ p, int d, int lig, R (&x)[NV]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = col(v, lig, d);
      x[v] = (typename Vec<T>::raw)(T)0.0f;
      if (there(v, lig, d)) x[v] = load_raw<T, TAIL != kShort>(p + c, d - c);
    }
  }
  __device__ static __forceinline__ void store(T* __restrict__ p, int d, int v, int lig, F y) {
    const int c = col(v, lig, d);
    if (there(v, lig, d)) store_f32<T, TAIL != kShort>(p + c, d - c, y);
  }
};

// a weight / bias vector of type code dt as fp32, columns behind the row as 0
template <int N>
__device__ __forceinline__ void load_param(const void* __restrict__ w, int dt, int c, int d, float* out) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float f = 0.f;
    if (c + k < d) {
      if (dt == MMSSL_F32) f = static_cast<const float*>(w)[c + k];
      else if (dt == MMSSL_BF16) f = (float)static_cast<const bf16_t*>(w)[c + k];
      else f = (float)static_cast<const f16_t*>(w)[c + k];
    }
    out[k] = f;
  }
}

// Sums of NS values over the LPR lanes of a row; every lane ends with them. `red` = two copies of [NS][waves]: used in turn,
// one barrier a call is enough.
template <int LPR, int NS>
__device__ __forceinline__ void row_sum(float (&s)[NS], float* red, int& turn) {
#pragma unroll
  for (int k = 0; k < NS; ++k) s[k] = group_sum<(LPR < 64 ? LPR : 64)>(s[k]);
  if (LPR > 64) {
    constexpr int W = LPR / 64;
    float* r = red + turn * (NS * W);
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < NS; ++k) r[k * W + (threadIdx.x >> 6)] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) a += r[k * W + w];
      s[k] = a;
    }
  }
}

template <class T, int LPR, int NV, Tail TAIL>
__global__ __launch_bounds__((RowTile<T, LPR, NV, TAIL>::TPB)) void ln_fwd_kernel(const T* __restrict__ X, int64_t ldx,
                                                                                  int64_t rows, int d,
                                                                                  const void* __restrict__ w,
                                                                                  const void* __restrict__ b, int pdt,
                                                                                  float eps, T* __restrict__ Y,
                                                                                  float2* __restrict__ stats) {
  typedef RowTile<T, LPR, NV, TAIL> Q;
  constexpr int N = Q::N;
  __shared__ float red[2 * Q::WPR];
  int turn = 0;
  const int lig = threadIdx.x & (LPR - 1);
  const int64_t step = (int64_t)gridDim.x * Q::GPB;
  const float inv_d = 1.0f / (float)d;
  float W[NV][N], Bb[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = Q::col(v, lig, d);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      W[v][k] = 1.f;
      Bb[v][k] = 0.f;
    }
    if (w) load_param<N>(w, pdt, c, d, W[v]);
    if (b) load_param<N>(b, pdt, c, d, Bb[v]);
  }
  int64_t row = (int64_t)blockIdx.x * Q::GPB + threadIdx.x / LPR;
  typename Q::R raw[NV];
  if (row < rows) Q::load(X + row * ldx, d, lig, raw);
  for (; row < rows; row += step) {
    typename Q::F x[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v] = to_f32<T>(raw[v]);
    if (row + step < rows) Q::load(X + (row + step) * ldx, d, lig, raw);      // the next row, under this one's sums
    float s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) s[0] += TAIL != kShared || Q::own(v, lig, d, k) ? x[v][k] : 0.f;    // 0 behind the row
    row_sum<LPR, 1>(s, red, turn);
    const float mu = s[0] / (float)d;        // the mean itself, not its product with a rounded 1 / d: x - mu may cancel
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float t = x[v][k] - mu;
        x[v][k] = t;
        q[0] += Q::own(v, lig, d, k) ? t * t : 0.f;
      }
    row_sum<LPR, 1>(q, red, turn);
    const float r = 1.0f / sqrtf(q[0] * inv_d + eps);
    if (stats && lig == 0) stats[row] = make_float2(mu, r);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      typename Q::F y;
#pragma unroll
      for (int k = 0; k < N; ++k) y[k] = fmaf(x[v][k] * r, W[v][k], Bb[v][k]);
      Q::store(Y + row * d, d, v, lig, y);
    }
  }
}

// part [blocks][2][d]: this block's sums of gy h and gy (NULL: not wanted); GX may be NULL
template <class T, int LPR, int NV, Tail TAIL>
__global__ __launch_bounds__((RowTile<T, LPR, NV, TAIL>::TPB)) void ln_bwd_kernel(
    const T* __restrict__ X, int64_t ldx, const T* __restrict__ G, int64_t ldg, int64_t rows, int d,
    const void* __restrict__ w, int pdt, const float2* __restrict__ stats, T* __restrict__ GX, float* __restrict__ part) {
  typedef RowTile<T, LPR, NV, TAIL> Q;
  constexpr int N = Q::N;
  __shared__ float red[4 * Q::WPR];
  int turn = 0;
  const int lig = threadIdx.x & (LPR - 1);
  const int64_t step = (int64_t)gridDim.x * Q::GPB;
  const float inv_d = 1.0f / (float)d;
  float W[NV][N], aw[NV][N], ab[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int k = 0; k < N; ++k) W[v][k] = 1.f, aw[v][k] = 0.f, ab[v][k] = 0.f;
    if (w) load_param<N>(w, pdt, Q::col(v, lig, d), d, W[v]);
  }
  int64_t row = (int64_t)blockIdx.x * Q::GPB + threadIdx.x / LPR;
  constexpr bool AHEAD = NV * N <= 8;              // with 16 values a lane and 1024 lanes the next row would spill
  typename Q::R rx[NV], rg[NV];
  if (AHEAD && row < rows) {
    Q::load(X + row * ldx, d, lig, rx);
    Q::load(G + row * ldg, d, lig, rg);
  }
  for (; row < rows; row += step) {
    typename Q::F x[NV], g[NV];
    const float2 st = stats[row];
    if (!AHEAD) {
      Q::load(X + row * ldx, d, lig, rx);
      Q::load(G + row * ldg, d, lig, rg);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      x[v] = to_f32<T>(rx[v]);
      g[v] = to_f32<T>(rg[v]);
    }
    if (AHEAD && row + step < rows) {
      Q::load(X + (row + step) * ldx, d, lig, rx);
      Q::load(G + (row + step) * ldg, d, lig, rg);
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float h = (x[v][k] - st.x) * st.y;           // columns behind the row: g = 0, so every product is
        const float gg = g[v][k], q = gg * W[v][k];
        x[v][k] = h;
        aw[v][k] = fmaf(gg, h, aw[v][k]);
        ab[v][k] += gg;
        g[v][k] = q;
        const float once = TAIL != kShared || Q::own(v, lig, d, k) ? q : 0.f;
        s[0] += once;
        s[1] = fmaf(once, h, s[1]);
      }
    if (!GX) continue;                                     // uniform
    row_sum<LPR, 2>(s, red, turn);
    const float m1 = s[0] * inv_d, m2 = s[1] * inv_d;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      typename Q::F y;
#pragma unroll
      for (int k = 0; k < N; ++k) y[k] = st.y * (g[v][k] - m1 - x[v][k] * m2);
      Q::store(GX + row * d, d, v, lig, y);
    }
  }
  if (!part) return;
  // the groups of a block, in their order
  float* out = part + (int64_t)blockIdx.x * 2 * d;
  if (Q::GPB == 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int c = Q::col(v, lig, d) + k;
        if (Q::own(v, lig, d, k)) {
          out[c] = aw[v][k];
          out[d + c] = ab[v][k];
        }
      }
    return;
  }
  constexpr int kSlots = Q::TPB * N;              // one vector of every lane at a time
  __shared__ float slot[Q::GPB == 1 ? 1 : 2 * kSlots];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    __syncthreads();
    const int skip = Q::skip(v, lig, d);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k >= skip) {                            // (slots behind the row are not read)
        slot[threadIdx.x * N + k - skip] = aw[v][k];
        slot[kSlots + threadIdx.x * N + k - skip] = ab[v][k];
      }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * LPR * N; j += Q::TPB) {
      const int half = j / (LPR * N), at = j % (LPR * N);
      if (v * LPR * N + at >= d) continue;
      float a = 0.f;
#pragma unroll 4
      for (int gidx = 0; gidx < Q::GPB; ++gidx) a += slot[half * kSlots + gidx * LPR * N + at];
      out[half * d + v * LPR * N + at] = a;
    }
  }
}

// gw / gb from the blocks' partial sums: 16 columns a block, its 64 groups of 4 lanes take every 64th partial each
__global__ __launch_bounds__(kBlock) void ln_param_kernel(const float* __restrict__ part, int nparts, int d,
                                                          void* __restrict__ gw, void* __restrict__ gb, int pdt) {
  __shared__ float4 red[64][4];
  const int l = threadIdx.x & 3, gidx = threadIdx.x >> 2;
  const int64_t width = 2 * (int64_t)d;
  const int64_t c = (int64_t)blockIdx.x * 16 + l * 4;
  Vec<float>::f32 a = 0.f;
  if (c < width) {
    const int left = (int)min((int64_t)4, width - c);
#pragma unroll 8
    for (int p = gidx; p < nparts; p += 64) a += load_raw<float>(part + (int64_t)p * width + c, left);
  }
  red[gidx][l] = make_float4(a[0], a[1], a[2], a[3]);
  __syncthreads();
  if (threadIdx.x < 16) {
    const int64_t col = (int64_t)blockIdx.x * 16 + threadIdx.x;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 64; ++k) t += reinterpret_cast<const float*>(red[k])[threadIdx.x];
    if (col < width) {
      void* out = col < d ? gw : gb;
      const int64_t j = col < d ? col : col - d;
      if (out) {
        if (pdt == MMSSL_F32) static_cast<float*>(out)[j] = t;
        else if (pdt == MMSSL_BF16) static_cast<bf16_t*>(out)[j] = (bf16_t)t;
        else static_cast<f16_t*>(out)[j] = (f16_t)t;
      }
    }
  }
}

// ---- rows longer than the registers of a block hold: one block a row, three sweeps (the later ones from the caches) -------
constexpr int kWideThreads = 1024;

template <class T>
__global__ __launch_bounds__(kWideThreads) void ln_fwd_wide_kernel(const T* __restrict__ X, int64_t ldx, int d,
                                                                   const void* __restrict__ w, const void* __restrict__ b,
                                                                   int pdt, float eps, T* __restrict__ Y,
                                                                   float2* __restrict__ stats) {
  constexpr int N = Vec<T>::N;
  __shared__ float red[2 * (kWideThreads / 64)];
  int turn = 0;
  const T* x = X + (int64_t)blockIdx.x * ldx;
  T* y = Y + (int64_t)blockIdx.x * d;
  const float inv_d = 1.0f / (float)d;
  float s[1] = {0.f};
  for (int c = threadIdx.x * N; c < d; c += kWideThreads * N) {
    const typename Vec<T>::f32 f = to_f32<T>(load_raw<T>(x + c, d - c));
#pragma unroll
    for (int k = 0; k < N; ++k) s[0] += f[k];
  }
  row_sum<kWideThreads, 1>(s, red, turn);
  const float mu = s[0] / (float)d;        // the mean itself, not its product with a rounded 1 / d: x - mu may cancel
  float q[1] = {0.f};
  for (int c = threadIdx.x * N; c < d; c += kWideThreads * N) {
    const typename Vec<T>::f32 f = to_f32<T>(load_raw<T>(x + c, d - c));
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float t = c + k < d ? f[k] - mu : 0.f;
      q[0] += t * t;
    }
  }
  row_sum<kWideThreads, 1>(q, red, turn);
  const float r = 1.0f / sqrtf(q[0] * inv_d + eps);
  if (stats && threadIdx.x == 0) stats[blockIdx.x] = make_float2(mu, r);
  for (int c = threadIdx.x * N; c < d; c += kWideThreads * N) {
    typename Vec<T>::f32 f = to_f32<T>(load_raw<T>(x + c, d - c));
    float W[N], Bb[N];
#pragma unroll
    for (int k = 0; k < N; ++k) W[k] = 1.f, Bb[k] = 0.f;
    if (w) load_param<N>(w, pdt, c, d, W);
    if (b) load_param<N>(b, pdt, c, d, Bb);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = fmaf((f[k] - mu) * r, W[k], Bb[k]);
    store_f32<T>(y + c, d - c, f);
  }
}

template <class T>
__global__ __launch_bounds__(kWideThreads) void ln_gx_wide_kernel(const T* __restrict__ X, int64_t ldx,
                                                                  const T* __restrict__ G, int64_t ldg, int d,
                                                                  const void* __restrict__ w, int pdt,
                                                                  const float2* __restrict__ stats, T* __restrict__ GX) {
  constexpr int N = Vec<T>::N;
  __shared__ float red[4 * (kWideThreads / 64)];
  int turn = 0;
  const T* x = X + (int64_t)blockIdx.x * ldx;
  const T* g = G + (int64_t)blockIdx.x * ldg;
  T* gx = GX + (int64_t)blockIdx.x * d;
  const float2 st = stats[blockIdx.x];
  const float inv_d = 1.0f / (float)d;
  float s[2] = {0.f, 0.f};
#pragma unroll 1
  for (int sweep = 0; sweep < 2; ++sweep) {
    for (int c = threadIdx.x * N; c < d; c += kWideThreads * N) {
      const typename Vec<T>::f32 xf = to_f32<T>(load_raw<T>(x + c, d - c)), gf = to_f32<T>(load_raw<T>(g + c, d - c));
      float W[N];
#pragma unroll
      for (int k = 0; k < N; ++k) W[k] = 1.f;
      if (w) load_param<N>(w, pdt, c, d, W);
      typename Vec<T>::f32 o;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float h = (xf[k] - st.x) * st.y, q = gf[k] * W[k];
        if (sweep == 0) {
          s[0] += q;
          s[1] = fmaf(q, h, s[1]);
        }
        o[k] = st.y * (q - s[0] - h * s[1]);
      }
      if (sweep) store_f32<T>(gx + c, d - c, o);
    }
    if (sweep == 0) {
      row_sum<kWideThreads, 2>(s, red, turn);
      s[0] *= inv_d;
      s[1] *= inv_d;
    }
  }
}

// blockIdx.x: column tile of kBlock vectors; blockIdx.y: stripe of rows
template <class T>
__global__ __launch_bounds__(kBlock) void ln_gw_wide_kernel(const T* __restrict__ X, int64_t ldx, const T* __restrict__ G,
                                                            int64_t ldg, int64_t rows, int d,
                                                            const float2* __restrict__ stats, float* __restrict__ part) {
  constexpr int N = Vec<T>::N;
  const int c = (blockIdx.x * kBlock + threadIdx.x) * N;
  if (c >= d) return;
  typename Vec<T>::f32 aw = 0.f, ab = 0.f;
#pragma unroll 2
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const typename Vec<T>::f32 x = to_f32<T>(load_raw<T>(X + r * ldx + c, d - c));
    const typename Vec<T>::f32 g = to_f32<T>(load_raw<T>(G + r * ldg + c, d - c));
    const float2 st = stats[r];
    aw += g * ((x - st.x) * st.y);
    ab += g;
  }
  float* out = part + (int64_t)blockIdx.y * 2 * d;
  store_part<N>(out + c, d - c, aw);
  store_part<N>(out + d + c, d - c, ab);
}

// ---- host -----------------------------------------------------------------------------------------------------------
struct Shape {
  int lpr, nv;      // lpr 0: wide
};

// The fewest lanes that hold the row with `values` (16 or 8) of it a lane; what is over 1024 lanes' share doubles it.
Shape shape_for(int d, int es, int values) {
  const int n = 16 / es, vecs = (d + n - 1) / n;
  if (d > kMaxInRegs) return {0, 0};
  for (int l = 8; l <= 64; l *= 2)
    if (vecs <= l) return {l, 1};
  const int nv = values / n;
  for (int l = 64; l <= 1024; l *= 2) {
    if (values > 8 && vecs <= l * (nv / 2)) return {l, nv / 2};
    if (vecs <= l * nv) return {l, nv};
  }
  return {1024, 16 / n};
}
// Forward 16 values a lane, backward 8: there three more copies of them stay in registers. 65536 x 4096 bf16, 256 lanes with
// 16 values against 512 with 8: forward 199 against 230 us, backward 345 (3 waves a SIMD) against 302 us (4).
Shape fwd_shape(int d, int es) { return shape_for(d, es, 16); }
Shape bwd_shape(int d, int es) { return shape_for(d, es, 8); }

int tpb_of(Shape q) { return q.lpr > 64 ? q.lpr : kBlock; }
int gpb_of(Shape q) { return q.lpr > 64 ? 1 : kBlock / q.lpr; }

// Blocks of a launch over rows: `waves` of them on each of 256 CUs, no more than the rows need.
int64_t blocks_for(int64_t rows, Shape q, int waves) {
  return std::min<int64_t>((rows + gpb_of(q) - 1) / gpb_of(q), (int64_t)256 * waves / (tpb_of(q) / 64));
}

constexpr int kFwdWaves = 16, kBwdWaves = 16;
int64_t wide_stripes(int64_t rows) { return std::min<int64_t>(rows, 256); }
int64_t parts_for(int64_t rows, int d, int es) {
  const Shape q = bwd_shape(d, es);
  return q.lpr ? blocks_for(rows, q, kBwdWaves) : wide_stripes(rows);
}

int check_common(int dtype, int64_t rows, int d, int pdt, float eps) {
  if (!known_dtype(dtype) || !known_dtype(pdt) || rows < 0 || d < 1 || !(eps >= 0.f)) return MMSSL_E_BADARG;
  // one block a row where rows are wide; a row's columns are counted in 32 bits
  if (d > (1 << 24) || (d > kMaxInRegs && !launchable(rows, kWideThreads))) return MMSSL_E_UNSUPP;
  return 0;
}

// CALL(T, LPR, NV) for the shape q: vectors of 16 values, 8, 4 (rows of few vectors, fp32)
#define LN_LANES(T, CALL, L)                          \
  case L:                                             \
    if (q.nv == 1) { CALL(T, L, 1); }                 \
    else if (q.nv == 2) { CALL(T, L, 2); }            \
    else { CALL(T, L, 4); }                           \
    break
#define LN_SHAPES(T, CALL)                            \
  do {                                                \
    const Tail tail = d % Vec<T>::N == 0 ? kWhole : d > Vec<T>::N ? kShared : kShort; \
    switch (q.lpr) {                                  \
      LN_LANES(T, CALL, 8);                           \
      LN_LANES(T, CALL, 16);                          \
      LN_LANES(T, CALL, 32);                          \
      LN_LANES(T, CALL, 64);                          \
      LN_LANES(T, CALL, 128);                         \
      LN_LANES(T, CALL, 256);                         \
      LN_LANES(T, CALL, 512);                         \
      LN_LANES(T, CALL, 1024);                        \
    }                                                 \
  } while (0)
// the shapes that occur: one vector up to 64 lanes; above, 8 values a lane (backward) or 8 and 16 (forward); 16 at 1024 lanes
#define LN_FWD_HAS(T, L, V) (V == 1 ? (L <= 64 || Vec<T>::N == 8) : (L >= 64 && (V * Vec<T>::N == 8 || V * Vec<T>::N == 16)))
#define LN_BWD_HAS(T, L, V) (V == 1 ? (L <= 64 || Vec<T>::N == 8) \
                                    : (L >= 64 && (V * Vec<T>::N == 8 || (L == 1024 && V * Vec<T>::N == 16))))

}  // namespace

extern "C" int mmssl_layernorm_rows(const void* X, int64_t ldx, int dtype, int64_t rows, int d, const void* weight,
                                    const void* bias, int param_dtype, float eps, void* Y, float* stats, void* stream) {
  if (int rc = check_common(dtype, rows, d, param_dtype, eps)) return rc;
  if (rows == 0) return 0;
  const size_t es = dtype_bytes(dtype), ps = dtype_bytes(param_dtype);
  if (!X || !Y || ldx < 0 || !aligned_to(X, es) || !aligned_to(Y, es) || !aligned_to(weight, ps) || !aligned_to(bias, ps) ||
      !aligned_to(stats, 8))
    return MMSSL_E_BADARG;
  const hipStream_t s = as_stream(stream);
  const Shape q = fwd_shape(d, (int)es);
  if (!q.lpr) {
#define LN_FWD_WIDE(T)                                                                                                   \
  hipLaunchKernelGGL(ln_fwd_wide_kernel<T>, dim3((unsigned)rows), dim3(kWideThreads), 0, s, (const T*)X, ldx, d, weight,  \
                     bias, param_dtype, eps, (T*)Y, (float2*)stats)
    MMSSL_BY_DTYPE(dtype, LN_FWD_WIDE);
    MMSSL_LAUNCH_CHECK();
    return 0;
  }
  const dim3 grid((unsigned)blocks_for(rows, q, kFwdWaves)), block(tpb_of(q));
#define LN_FWD_F(T, L, V, F)                                                                                             \
  hipLaunchKernelGGL((ln_fwd_kernel<T, L, V, F>), grid, block, 0, s, (const T*)X, ldx, rows, d, weight, bias,             \
                     param_dtype, eps, (T*)Y, (float2*)stats)
#define LN_FWD_V(T, L, V)                                          \
  if constexpr (LN_FWD_HAS(T, L, V)) {                             \
    if (tail == kWhole) LN_FWD_F(T, L, V, kWhole);                 \
    else if (tail == kShared) LN_FWD_F(T, L, V, kShared);          \
    else if constexpr (L == 8) LN_FWD_F(T, L, V, kShort);          \
  }
#define LN_FWD(T) LN_SHAPES(T, LN_FWD_V)
  MMSSL_BY_DTYPE(dtype, LN_FWD);
  MMSSL_LAUNCH_CHECK();
  return 0;
}

extern "C" size_t mmssl_layernorm_rows_bwd_workspace_bytes(int dtype, int64_t rows, int d) {
  if (!known_dtype(dtype) || rows < 0 || d < 1 || d > (1 << 24)) return 0;
  return (size_t)parts_for(rows, d, dtype_bytes(dtype)) * 2 * d * 4 + 16;
}

extern "C" int mmssl_layernorm_rows_bwd(const void* X, int64_t ldx, const void* G, int64_t ldg, int dtype, int64_t rows,
                                        int d, const void* weight, int param_dtype, const float* stats, void* GX,
                                        void* gweight, void* gbias, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  if (int rc = check_common(dtype, rows, d, param_dtype, 0.f)) return rc;
  const size_t es = dtype_bytes(dtype), ps = dtype_bytes(param_dtype);
  const bool params = gweight || gbias;
  if (ldx < 0 || ldg < 0 || !aligned_to(X, es) || !aligned_to(G, es) || !aligned_to(GX, es) || !aligned_to(weight, ps) ||
      !aligned_to(gweight, ps) || !aligned_to(gbias, ps) || !aligned_to(stats, 8))
    return MMSSL_E_BADARG;
  if (rows > 0 && (!X || !G || !stats)) return MMSSL_E_BADARG;
  if (!GX && !params) return 0;
  float* part = static_cast<float*>(workspace);
  if (params && (!workspace || !aligned_to(workspace, 16) ||
                 workspace_bytes < mmssl_layernorm_rows_bwd_workspace_bytes(dtype, rows, d)))
    return MMSSL_E_WORKSPACE;
  const hipStream_t s = as_stream(stream);
  const Shape q = bwd_shape(d, (int)es);
  const int64_t nparts = parts_for(rows, d, (int)es);
  if (rows > 0 && q.lpr) {
    const dim3 grid((unsigned)nparts), block(tpb_of(q));
    float* pp = params ? part : nullptr;
#define LN_BWD_F(T, L, V, F)                                                                                             \
  hipLaunchKernelGGL((ln_bwd_kernel<T, L, V, F>), grid, block, 0, s, (const T*)X, ldx, (const T*)G, ldg, rows, d, weight, \
                     param_dtype, (const float2*)stats, (T*)GX, pp)
#define LN_BWD_V(T, L, V)                                          \
  if constexpr (LN_BWD_HAS(T, L, V)) {                             \
    if (tail == kWhole) LN_BWD_F(T, L, V, kWhole);                 \
    else if constexpr (Vec<T>::N == 4) LN_BWD_F(T, L, V, kShort);  \
    else if (tail == kShared) LN_BWD_F(T, L, V, kShared);          \
    else if constexpr (L == 8) LN_BWD_F(T, L, V, kShort);          \
  }
#define LN_BWD(T) LN_SHAPES(T, LN_BWD_V)
    MMSSL_BY_DTYPE(dtype, LN_BWD);
    MMSSL_LAUNCH_CHECK();
  } else if (rows > 0) {
#define LN_GX_WIDE(T)                                                                                                    \
  hipLaunchKernelGGL(ln_gx_wide_kernel<T>, dim3((unsigned)rows), dim3(kWideThreads), 0, s, (const T*)X, ldx, (const T*)G, \
                     ldg, d, weight, param_dtype, (const float2*)stats, (T*)GX)
#define LN_GW_WIDE(T)                                                                                                    \
  hipLaunchKernelGGL(ln_gw_wide_kernel<T>, dim3((unsigned)((d + kBlock * Vec<T>::N - 1) / (kBlock * Vec<T>::N)),          \
                                                (unsigned)nparts),                                                       \
                     dim3(kBlock), 0, s, (const T*)X, ldx, (const T*)G, ldg, rows, d, (const float2*)stats, part)
    if (GX) {
      MMSSL_BY_DTYPE(dtype, LN_GX_WIDE);
      MMSSL_LAUNCH_CHECK();
    }
    if (params) {
      MMSSL_BY_DTYPE(dtype, LN_GW_WIDE);
      MMSSL_LAUNCH_CHECK();
    }
  }
  if (params) {
    hipLaunchKernelGGL(ln_param_kernel, dim3((unsigned)((2 * (int64_t)d + 15) / 16)), dim3(kBlock), 0, s,
                       (const float*)part, (int)nparts, d, gweight, gbias, param_dtype);
    MMSSL_LAUNCH_CHECK();
  }
  return 0;
}
