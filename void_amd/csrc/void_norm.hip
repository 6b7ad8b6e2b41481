// void_norm.hip — layer norm over the last axis, forward and backward, for
// gfx950, declared in include/void_amd.h.
//
// Row x of C values, weight w and bias b:
//   mu = sum x / C,  v = sum (x - mu)^2 / C,  r = 1 / sqrt(v + eps),
//   xh = (x - mu) r,  y = xh w + b;
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),
//   dw = sum_rows dy xh,  db = sum_rows dy.
// Both passes are bound by memory: a row is read once into registers, so that
// the mean and the variance around it (two sums, no cancellation whatever the
// row's offset) cost no second read.  T threads share a row, NV pieces of 16
// bytes each, in a grid that walks over the rows; the next row's pieces load
// while the current one is reduced.  All sums and statistics are fp32; y and dx
// are rounded once, when stored.
//
// The backward pass sums dw and db for its own rows in registers and writes
// them once at the end, one partial row per workgroup; a second kernel adds
// the partial rows in order (no atomics: the same bits on every run).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "rows.h"
#include "void_amd.h"

extern "C" __attribute__((visibility("hidden"))) int void_internal_fail(int code, const char* msg);

namespace {

// Threads that a workgroup of rows of T threads has: whole rows, 256 at least.
constexpr int block_of(int T) { return T < 256 ? 256 : T; }

// One read of x, one write of y.  16384 x 8192 bf16 91 us, 5.9 TB/s; 2048 x 4096 bf16
// 10.7 us, in the caches; 5003 x 3001 fp32 28 us, 4.3 TB/s; one row of 4096 3.2 us, which
// is the launch and two sums.
template <class E, class W, int T, int NV, bool ODD>
__global__ __launch_bounds__(block_of(T)) void norm_kernel(const E* __restrict__ x, int64_t ldx,
                                                           const W* __restrict__ weight, const W* __restrict__ bias,
                                                           int64_t rows, int cols, float eps, E* __restrict__ y,
                                                           int64_t ldy, float2* __restrict__ stats) {
  constexpr int N = Piece<E>::n, kRows = block_of(T) / T;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ float2 red[2][16];
  RowSum<T> rs{red};
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / T;
  const float inv = 1.f / (float)cols;
  Loaded<E, ODD> v[NV];
  if (row < rows)
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i].load(x + row * ldx, (i * T + t) * N, cols);
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_params(w[i], weight, (i * T + t) * N, cols, 1.f);
    load_params(b[i], bias, (i * T + t) * N, cols, 0.f);
  }
  for (; row < rows; row += step) {
    F f[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) f[i] = __builtin_convertvector(v[i].take(x + row * ldx, (i * T + t) * N, cols), F);
    if (row + step < rows)
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i].load(x + (row + step) * ldx, (i * T + t) * N, cols);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) s += f[i][e];
    const float mu = rs.sum(s) * inv;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = (i * T + t) * N + e < cols ? f[i][e] - mu : 0.f;
        f[i][e] = d;
        q = fmaf(d, d, q);
      }
    const float r = 1.f / sqrtf(rs.sum(q) * inv + eps);
    if (stats && t == 0) stats[row] = make_float2(mu, r);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F o;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = fmaf(f[i][e] * r, w[i][e], b[i][e]);
      if ((i * T + t) * N < cols) store_piece(y + row * ldy, (i * T + t) * N, cols, __builtin_convertvector(o, V));
    }
  }
}

// Rows that no register variant holds (more than 16384 values): three passes over the
// row, which stays in the L2 between them; bound by those.  2048 x 32768 bf16 91 us, 2.9 TB/s
// of one read and one write; fp32 160 us, 3.4 TB/s.
template <class E, class W>
__global__ __launch_bounds__(1024) void norm_long_kernel(const E* __restrict__ x, int64_t ldx,
                                                         const W* __restrict__ weight, const W* __restrict__ bias,
                                                         int64_t rows, int cols, float eps, E* __restrict__ y,
                                                         int64_t ldy, float2* __restrict__ stats) {
  constexpr int N = Piece<E>::n;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ float2 red[2][16];
  RowSum<1024> rs{red};
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const E* xr = x + row * ldx;
    float s = 0.f;
    for (int64_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
      const F f = __builtin_convertvector(load_piece(xr, (int)c, cols), F);
#pragma unroll
      for (int e = 0; e < N; ++e) s += f[e];
    }
    const float mu = rs.sum(s) / (float)cols;
    float q = 0.f;
    for (int64_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
      const F f = __builtin_convertvector(load_piece(xr, (int)c, cols), F);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = c + e < cols ? f[e] - mu : 0.f;
        q = fmaf(d, d, q);
      }
    }
    const float r = 1.f / sqrtf(rs.sum(q) / (float)cols + eps);
    if (stats && threadIdx.x == 0) stats[row] = make_float2(mu, r);
    for (int64_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
      const F f = __builtin_convertvector(load_piece(xr, (int)c, cols), F);
      float w[N], b[N];
      load_params(w, weight, (int)c, cols, 1.f);
      load_params(b, bias, (int)c, cols, 0.f);
      F o;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = fmaf((f[e] - mu) * r, w[e], b[e]);
      store_piece(y + row * ldy, (int)c, cols, __builtin_convertvector(o, V));
    }
  }
}

// dx (unless null) and this workgroup's partial sums of dw and db (unless
// `part` is null) in part[2 blockIdx.x] and part[2 blockIdx.x + 1], rows of
// `cols` floats.  One read of x and dy, one write of dx: 16384 x 8192 bf16 156 us,
// 5.1 TB/s; 2048 x 4096 bf16 14.5 us; 5003 x 3001 fp32 43 us, 4.2 TB/s.
template <class E, class W, int T, int NV, bool ODD>
__global__ __launch_bounds__(block_of(T)) void norm_grad_kernel(
    const E* __restrict__ dy, int64_t lddy, const E* __restrict__ x, int64_t ldx, const W* __restrict__ weight,
    const float2* __restrict__ stats, int64_t rows, int cols, E* __restrict__ dx, int64_t lddx,
    float* __restrict__ part) {
  constexpr int N = Piece<E>::n, kBlock = block_of(T), kRows = kBlock / T;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ float2 red[2][16];
  RowSum<T> rs{red};
  const int t = threadIdx.x % T;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / T;
  const float inv = 1.f / (float)cols;
  // 1024 threads have 128 registers each: no room for the next row's pieces.
  constexpr bool kAhead = T < 1024;
  Loaded<E, ODD> vx[NV], vg[NV];
  float2 st = {};
  auto fetch = [&](int64_t r) {
    st = stats[r];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      vx[i].load(x + r * ldx, (i * T + t) * N, cols);
      vg[i].load(dy + r * lddy, (i * T + t) * N, cols);
    }
  };
  if (kAhead && row < rows) fetch(row);
  float w[NV][N];
  F aw[NV], ab[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_params(w[i], weight, (i * T + t) * N, cols, 1.f);
    aw[i] = ab[i] = 0.f;
  }
  for (; row < rows; row += step) {
    if (!kAhead) fetch(row);
    F h[NV], g[NV];
    float s1 = 0.f, s2 = 0.f;
    const float r = st.y;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      h[i] = __builtin_convertvector(vx[i].take(x + row * ldx, (i * T + t) * N, cols), F);
      g[i] = __builtin_convertvector(vg[i].take(dy + row * lddy, (i * T + t) * N, cols), F);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        // Past the row's end dy is zero, so only what is stored could see h there.
        h[i][e] = (h[i][e] - st.x) * r;
        aw[i][e] = fmaf(g[i][e], h[i][e], aw[i][e]);
        ab[i][e] += g[i][e];
        g[i][e] *= w[i][e];
        s1 += g[i][e];
        s2 = fmaf(g[i][e], h[i][e], s2);
      }
    }
    if (kAhead && row + step < rows) fetch(row + step);
    if (!dx) continue;
    const float2 m = rs.sum(s1, s2);
    const float c1 = m.x * inv, c2 = m.y * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F o;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = r * (g[i][e] - fmaf(h[i][e], c2, c1));
      if ((i * T + t) * N < cols) store_piece(dx + row * lddx, (i * T + t) * N, cols, __builtin_convertvector(o, V));
    }
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (kRows > 1) {
    // The workgroup's row groups added in order: lanes of one wave first, then
    // the four waves through LDS.
    __shared__ float sum[4][2][NV][(T < 64 ? T : 64) * N];
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        float a = aw[i][e], c = ab[i][e];
        for (int off = T; off < 64; off <<= 1) {
          a += __shfl_xor(a, off, 64);
          c += __shfl_xor(c, off, 64);
        }
        if ((threadIdx.x & 63) < T) {
          sum[wave][0][i][t * N + e] = a;
          sum[wave][1][i][t * N + e] = c;
        }
      }
    __syncthreads();
    for (int j = threadIdx.x; j < NV * T * N; j += kBlock) {
      const int i = j / (T * N), e = j % (T * N);
      if (j < cols) {
        pw[j] = (sum[0][0][i][e] + sum[1][0][i][e]) + (sum[2][0][i][e] + sum[3][0][i][e]);
        pw[cols + j] = (sum[0][1][i][e] + sum[1][1][i][e]) + (sum[2][1][i][e] + sum[3][1][i][e]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + t) * N;
#pragma unroll
      for (int e = 0; e < N; e += 4)
        if (c + e < cols) {
          store_piece<float>(pw, c + e, cols, Piece<float>::vec{aw[i][e], aw[i][e + 1], aw[i][e + 2], aw[i][e + 3]});
          store_piece<float>(pw + cols, c + e, cols,
                             Piece<float>::vec{ab[i][e], ab[i][e + 1], ab[i][e + 2], ab[i][e + 3]});
        }
    }
  }
}

// dx of rows that no register variant holds: two passes, the second in the L2.  2048 x
// 32768 bf16 101 us, 4.0 TB/s of x, dy and dx; fp32 213 us, 3.8 TB/s.
template <class E, class W>
__global__ __launch_bounds__(1024) void norm_long_grad_kernel(const E* __restrict__ dy, int64_t lddy,
                                                              const E* __restrict__ x, int64_t ldx,
                                                              const W* __restrict__ weight,
                                                              const float2* __restrict__ stats, int64_t rows, int cols,
                                                              E* __restrict__ dx, int64_t lddx) {
  constexpr int N = Piece<E>::n;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ float2 red[2][16];
  RowSum<1024> rs{red};
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float2 st = stats[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
      const F h = __builtin_convertvector(load_piece(x + row * ldx, (int)c, cols), F);
      const F g = __builtin_convertvector(load_piece(dy + row * lddy, (int)c, cols), F);
      float w[N];
      load_params(w, weight, (int)c, cols, 1.f);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        s1 = fmaf(g[e], w[e], s1);
        s2 = fmaf(g[e] * w[e], (h[e] - st.x) * st.y, s2);
      }
    }
    const float2 m = rs.sum(s1, s2);
    const float c1 = m.x / (float)cols, c2 = m.y / (float)cols;
    for (int64_t c = threadIdx.x * N; c < cols; c += 1024 * N) {
      const F h = __builtin_convertvector(load_piece(x + row * ldx, (int)c, cols), F);
      const F g = __builtin_convertvector(load_piece(dy + row * lddy, (int)c, cols), F);
      float w[N];
      load_params(w, weight, (int)c, cols, 1.f);
      F o;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = st.y * (g[e] * w[e] - fmaf((h[e] - st.x) * st.y, c2, c1));
      store_piece(dx + row * lddx, (int)c, cols, __builtin_convertvector(o, V));
    }
  }
}

// Their dw and db: 64 pieces of columns and 4 rows at a time, the rows dealt to
// blockIdx.y; one partial row per workgroup.  2048 x 32768 bf16 45 us, behind dx's kernel
// and partly in the caches; fp32 107 us, 5.0 TB/s.
template <class E>
__global__ __launch_bounds__(256) void norm_long_params_kernel(const E* __restrict__ dy, int64_t lddy,
                                                               const E* __restrict__ x, int64_t ldx,
                                                               const float2* __restrict__ stats, int64_t rows, int cols,
                                                               float* __restrict__ part) {
  constexpr int N = Piece<E>::n;
  typedef typename Piece<E>::fvec F;
  __shared__ float sum[4][2][64 * N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * N;
  F aw = 0.f, ab = 0.f;
  if (c < cols)
    for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < rows; row += (int64_t)gridDim.y * 4) {
      const float2 st = stats[row];
      const F h = __builtin_convertvector(load_piece(x + row * ldx, (int)c, cols), F);
      const F g = __builtin_convertvector(load_piece(dy + row * lddy, (int)c, cols), F);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        aw[e] = fmaf(g[e], (h[e] - st.x) * st.y, aw[e]);
        ab[e] += g[e];
      }
    }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    sum[wave][0][lane * N + e] = aw[e];
    sum[wave][1][lane * N + e] = ab[e];
  }
  __syncthreads();
  float* pw = part + (int64_t)blockIdx.y * 2 * cols;
  for (int j = threadIdx.x; j < 64 * N; j += 256) {
    const int64_t col = (int64_t)blockIdx.x * 64 * N + j;
    if (col < cols) {
      pw[col] = (sum[0][0][j] + sum[1][0][j]) + (sum[2][0][j] + sum[3][0][j]);
      pw[cols + col] = (sum[0][1][j] + sum[1][1][j]) + (sum[2][1][j] + sum[3][1][j]);
    }
  }
}

// dweight[c] and dbias[c]: the n partial rows of 2 cols floats added in order,
// 16 of them at a time (one a wave), and rounded once.  512 rows of 2 x 4096 4.0 us,
// 256 of 2 x 8192 5.8 us: the latency of a launch and of a few loads in a row.
template <class W>
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float* __restrict__ part, int n, int cols,
                                                        W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sum[16][64];
  const int64_t j = grid_block() * 64 + (threadIdx.x & 63);
  const float s = partial_rows_sum(part, n, 2 * (int64_t)cols, j, sum);
  if (threadIdx.x < 64) {
    if (j < cols) {
      if (dw) dw[j] = (W)s;
    } else if (j < 2 * (int64_t)cols && db) {
      db[j - cols] = (W)s;
    }
  }
}

constexpr int kCus = 256;

// The register variant for rows of `cols` values: at most 16 values a thread
// (the backward pass holds dw and db sums for each beside x and dy; 32 spilled),
// one wave a row up to 1024 values, where a sum needs no barrier, whole
// workgroups beyond.  Calls go(T, NV) as integral constants; false where the
// row is longer than any variant holds (16384 values).
template <class E, class Go>
bool by_width(int cols, Go go) {
  using std::integral_constant;
  constexpr int k8 = sizeof(E) == 4 ? 2 : 1;  // pieces of 8 values
#define VOID_ROW(T_, NV_) \
  if (cols <= T_ * NV_ * Piece<E>::n) return go(integral_constant<int, T_>{}, integral_constant<int, NV_>{}), true
  VOID_ROW(8, k8);
  VOID_ROW(16, k8);
  VOID_ROW(32, k8);
  VOID_ROW(64, k8);
  VOID_ROW(64, 2 * k8);
  VOID_ROW(256, k8);
  VOID_ROW(256, 2 * k8);
  VOID_ROW(512, 2 * k8);
  VOID_ROW(1024, 2 * k8);
#undef VOID_ROW
  return false;
}

// Partial rows of dw and db (workgroups of the backward pass).
template <class E>
int partials(int64_t rows, int cols) {
  int n = 0;
  if (!by_width<E>(cols, [&](auto t, auto) {
        constexpr int T = decltype(t)::value, kRows = block_of(T) / T;
        n = (int)std::min<int64_t>((rows + kRows - 1) / kRows, kCus * (T > 256 ? 1 : 2));
      }))
    n = (int)std::min<int64_t>((rows + 3) / 4, 64);
  return n;
}

template <class E, class W>
void forward(const void* x, int64_t ldx, const void* w, const void* b, int64_t rows, int cols, float eps, void* y,
             int64_t ldy, float* stats, hipStream_t stream) {
  auto args = [&](auto kernel, int64_t grid, int block) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(block), 0, stream, static_cast<const E*>(x), ldx,
                       static_cast<const W*>(w), static_cast<const W*>(b), rows, cols, eps, static_cast<E*>(y), ldy,
                       reinterpret_cast<float2*>(stats));
  };
  if (!by_width<E>(cols, [&](auto t, auto nv) {
        constexpr int T = decltype(t)::value, NV = decltype(nv)::value, kRows = block_of(T) / T;
        by_parity<E>(x, ldx, x, ldx, rows, [&](auto odd) {
          args(norm_kernel<E, W, T, NV, decltype(odd)::value>,
               std::min<int64_t>((rows + kRows - 1) / kRows, kCus * (T > 256 ? 2 : 4)), block_of(T));
        });
      }))
    args(norm_long_kernel<E, W>, std::min<int64_t>(rows, kCus * 2), 1024);
}

template <class E, class W>
void backward(const void* dy_, int64_t lddy, const void* x_, int64_t ldx, const void* w_, const float* stats_,
              int64_t rows, int cols, void* dx_, int64_t lddx, void* dw, void* db, float* part, hipStream_t stream) {
  const E *dy = static_cast<const E*>(dy_), *x = static_cast<const E*>(x_);
  const W* w = static_cast<const W*>(w_);
  E* dx = static_cast<E*>(dx_);
  const float2* stats = reinterpret_cast<const float2*>(stats_);
  const int n = partials<E>(rows, cols);
  if (!by_width<E>(cols, [&](auto t, auto nv) {
        constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
        by_parity<E>(dy, lddy, x, ldx, rows, [&](auto odd) {
          hipLaunchKernelGGL((norm_grad_kernel<E, W, T, NV, decltype(odd)::value>), dim3(n), dim3(block_of(T)), 0,
                             stream, dy, lddy, x, ldx, w, stats, rows, cols, dx, lddx, part);
        });
      })) {
    if (dx)
      hipLaunchKernelGGL((norm_long_grad_kernel<E, W>), dim3((unsigned)std::min<int64_t>(rows, kCus * 2)), dim3(1024),
                         0, stream, dy, lddy, x, ldx, w, stats, rows, cols, dx, lddx);
    if (part)
      hipLaunchKernelGGL(norm_long_params_kernel<E>,
                         dim3((unsigned)(((int64_t)cols + 64 * Piece<E>::n - 1) / (64 * Piece<E>::n)), n), dim3(256), 0,
                         stream, dy, lddy, x, ldx, stats, rows, cols, part);
  }
  if (part)
    hipLaunchKernelGGL(norm_sum_kernel<W>, grid_of((2 * (int64_t)cols + 63) / 64), dim3(1024), 0, stream, part,
                       n, cols, static_cast<W*>(dw), static_cast<W*>(db));
}

int check_rows(int64_t rows, int32_t cols, int32_t dtype, int32_t param_dtype) {
  if (rows < 0 || cols < 0) return void_internal_fail(VOID_ERR_ARG, "negative size");
  // A piece's end past the row's must not pass 31 bits.
  if (cols > INT_MAX / 2) return void_internal_fail(VOID_ERR_UNSUPPORTED, "rows are limited to 2^30 values");
  if (dtype != VOID_DT_F32 && dtype != VOID_DT_BF16 && dtype != VOID_DT_F16)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "values are fp32, bf16 or fp16");
  if (param_dtype != dtype && param_dtype != VOID_DT_F32)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "weight and bias have the values' type, or fp32");
  return 1;
}

bool unaligned(const void* p, int32_t dtype) { return (uintptr_t)p % (dtype == VOID_DT_F32 ? 4 : 2); }

// go(E, W) for the values' and the parameters' type.
template <class Go>
void by_type(int32_t dtype, int32_t param_dtype, Go go) {
  if (dtype == VOID_DT_F32) go(float{}, float{});
  else if (dtype == VOID_DT_BF16 && param_dtype == VOID_DT_F32) go(__bf16{}, float{});
  else if (dtype == VOID_DT_BF16) go(__bf16{}, __bf16{});
  else if (param_dtype == VOID_DT_F32) go(_Float16{}, float{});
  else go(_Float16{}, _Float16{});
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VOID_OK : void_internal_fail(VOID_ERR_HIP, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int void_layer_norm(const void* x, int64_t ldx, const void* weight, const void* bias, int32_t param_dtype, int64_t rows,
                    int32_t cols, float eps, int32_t dtype, void* y, int64_t ldy, float* stats, hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const int st = check_rows(rows, cols, dtype, param_dtype);
  if (st <= 0) return st;
  if (rows == 0 || cols == 0) return VOID_OK;
  if (!x || !y) return void_internal_fail(VOID_ERR_ARG, "null x or y");
  if ((rows > 1 && (ldx < 0 || ldy < cols)) || unaligned(x, dtype) || unaligned(y, dtype) ||
      unaligned(weight, param_dtype) || unaligned(bias, param_dtype) || (uintptr_t)stats % 8)
    return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements, rows must not overlap");
  by_type(dtype, param_dtype, [&](auto e, auto w) {
    forward<decltype(e), decltype(w)>(x, ldx, weight, bias, rows, cols, eps, y, ldy, stats, stream);
  });
  return launched();
}

size_t void_layer_norm_grad_workspace_bytes(int64_t rows, int32_t cols, int32_t dtype) {
  if (rows <= 0 || cols <= 0) return 0;
  const int n = dtype == VOID_DT_F32 ? partials<float>(rows, cols) : partials<__bf16>(rows, cols);
  return (size_t)n * 2 * cols * sizeof(float);
}

int void_layer_norm_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                         int32_t param_dtype, const float* stats, int64_t rows, int32_t cols, int32_t dtype, void* dx,
                         int64_t lddx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                         hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const int st = check_rows(rows, cols, dtype, param_dtype);
  if (st <= 0) return st;
  if (cols == 0 || (!dx && !dweight && !dbias)) return VOID_OK;
  const bool params = dweight || dbias;
  if (rows == 0 && !params) return VOID_OK;
  if (rows && (!dy || !x || !stats)) return void_internal_fail(VOID_ERR_ARG, "null dy, x or stats");
  if ((rows > 1 && (ldx < 0 || lddy < 0 || (dx && lddx < cols))) || unaligned(dy, dtype) || unaligned(x, dtype) ||
      unaligned(dx, dtype) || unaligned(weight, param_dtype) || unaligned(dweight, param_dtype) ||
      unaligned(dbias, param_dtype) || (uintptr_t)stats % 8)
    return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements, rows must not overlap");
  if (params && rows &&
      (!workspace || (uintptr_t)workspace % 4 ||
       workspace_bytes < void_layer_norm_grad_workspace_bytes(rows, cols, dtype)))
    return void_internal_fail(VOID_ERR_WORKSPACE, "layer norm gradient: workspace missing or too small");
  by_type(dtype, param_dtype, [&](auto e, auto w) {
    using E = decltype(e);
    using W = decltype(w);
    if (rows)
      backward<E, W>(dy, lddy, x, ldx, weight, stats, rows, cols, dx, lddx, dweight, dbias,
                     params ? static_cast<float*>(workspace) : nullptr, stream);
    else  // no rows: the parameters' gradients are sums of nothing
      hipLaunchKernelGGL(norm_sum_kernel<W>, grid_of((2 * (int64_t)cols + 63) / 64), dim3(1024), 0, stream,
                         nullptr, 0, cols, static_cast<W*>(dweight), static_cast<W*>(dbias));
  });
  return launched();
}

}  // extern "C"
