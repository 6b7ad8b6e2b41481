// void_distill.hip — distillation from a teacher's top logits, forward and
// backward, for gfx950, declared in include/void_amd.h.
//
// A row has V student logits s and k teacher entries (logit t_j, index i_j);
// an entry with a negative index or a logit of -inf does not count.  With the
// temperature T,
//   p = softmax(t / T) over the row's entries,  q = softmax(s / T) over all V,
//   loss = T^2 sum_j p_j (log p_j - log q_{i_j}),
//   dloss / ds_v = T (q_v - sum_{j: i_j = v} p_j).
// A row without entries has loss 0 and gradient 0, whatever its logits hold,
// and its logits are not read.  An index of V or more makes the row NaN.
//
// Everything is bound by reading s and writing its gradient.  exp(s / T) is
// taken as exp2((s - m) log2(e) / T) around the row's largest logit m: the
// difference first, so that logits of the type's lowest value, used as masks,
// neither overflow nor meet an infinity.  m and z = sum exp2(...) are fp32, the
// gradient is rounded once.  A row's entries live in LDS; their logits' few
// gradients are written again, with the p of equal indices added in order, behind
// the barrier that follows the row's (no atomics).
//
// Many rows: one workgroup of T threads a row.  Few rows: S slices of each row,
// whose (m, z) parts every reader joins for itself in slice order.  Loss and
// gradient in one call keep the row in registers between the sum and the
// gradient (up to 16 pieces of 16 bytes a thread): one read, one write.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "rows.h"
#include "void_amd.h"

extern "C" __attribute__((visibility("hidden"))) int void_internal_fail(int code, const char* msg);

namespace {

constexpr int kMaxEntries = VOID_DISTILL_MAX_ENTRIES;
constexpr int kMaxSlices = 64;  // a slice a lane where they are joined
constexpr float kLowest = -3.402823466e38f;

struct Args {
  const void* logits;
  const void* top;
  const void* index;
  int64_t ld, ldt, ldi, rows;
  int vocab, k, top_type, index_bytes;
  float temperature, c;  // c = log2(e) / T
};

// 2^x by the hardware's instruction (results below 2^-126 are 0).
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- reductions over the T threads of a workgroup -------------------------

template <int T>
__device__ __forceinline__ float max_over(float v, float* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  if constexpr (T > 64) {
    __syncthreads();  // red is free
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) v = fmaxf(v, red[w]);
  }
  return v;
}

template <int T>
__device__ __forceinline__ float sum_over(float v, float* red) {
  v = lanes_sum<64>(v);
  if constexpr (T > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += red[w];
  }
  return v;
}

// ---- the teacher's entries of a row ---------------------------------------

// In dynamic LDS, k of each.
struct Entries {
  float* p;     // probability; 0 where the entry does not count
  float* lp;    // its logarithm
  int32_t* at;  // index, -1 where the entry does not count
};

__device__ __forceinline__ Entries entries_of(float* lds, int k) {
  return Entries{lds, lds + k, reinterpret_cast<int32_t*>(lds + 2 * k)};
}

size_t entries_bytes(int k) { return (size_t)std::max(k, 1) * 12; }

__device__ __forceinline__ int64_t entry_index(const Args& a, int64_t row, int j) {
  return a.index_bytes == 8 ? static_cast<const int64_t*>(a.index)[row * a.ldi + j]
                            : (int64_t) static_cast<const int32_t*>(a.index)[row * a.ldi + j];
}

__device__ __forceinline__ float entry_logit(const Args& a, int64_t row, int j) {
  const int64_t o = row * a.ldt + j;
  if (a.top_type == VOID_DT_F32) return static_cast<const float*>(a.top)[o];
  if (a.top_type == VOID_DT_BF16) return (float)static_cast<const __bf16*>(a.top)[o];
  return (float)static_cast<const _Float16*>(a.top)[o];
}

__device__ __forceinline__ bool entry_counts(int64_t at, float t) { return at >= 0 && !(t == -INFINITY); }

// Whether the row has an entry that counts (the same for all T threads).
template <int T>
__device__ __forceinline__ bool has_entries(const Args& a, int64_t row) {
  int any = 0;
  for (int j = threadIdx.x; j < a.k; j += T) any |= entry_counts(entry_index(a, row, j), entry_logit(a, row, j));
  if constexpr (T == 64) return __ballot(any) != 0;
  else return __syncthreads_or(any) != 0;
}

// The row's entries into `en`; false (and nothing usable in en) where none
// counts.  Ends behind a barrier.
template <int T>
__device__ __forceinline__ bool load_entries(const Args& a, int64_t row, const Entries& en, float* red) {
  __syncthreads();  // en is free
  float top = -INFINITY;
  int bad = 0;
  for (int j = threadIdx.x; j < a.k; j += T) {
    const int64_t at = entry_index(a, row, j);
    const float t = entry_logit(a, row, j);
    const bool use = entry_counts(at, t);
    bad |= use && at >= a.vocab;
    en.at[j] = use ? (int32_t)(at < a.vocab ? at : 0) : -1;
    en.lp[j] = t;
    if (use) top = fmaxf(top, t == t ? t : kLowest);  // a NaN still counts
  }
  top = max_over<T>(top, red);
  if (top == -INFINITY) return false;
  float s = bad ? NAN : 0.f;
  for (int j = threadIdx.x; j < a.k; j += T) {
    const float d = (en.lp[j] - top) * a.c, e = en.at[j] >= 0 ? pow2(d) : 0.f;
    en.p[j] = e;
    en.lp[j] = d;
    s += e;
  }
  s = sum_over<T>(s, red);
  const float inv = 1.f / s, ls = logf(s);
  for (int j = threadIdx.x; j < a.k; j += T) {
    en.p[j] *= inv;
    en.lp[j] = en.lp[j] * 0.693147180559945309f - ls;
  }
  __syncthreads();
  return true;
}

// The row's loss from its entries and its m and z.
template <class E, int T>
__device__ __forceinline__ float row_loss(const Args& a, const E* s, const Entries& en, float m, float z, float* red) {
  const float lz = logf(z), t = a.temperature;
  float sum = 0.f;
  for (int j = threadIdx.x; j < a.k; j += T) {
    const float p = en.p[j];
    if (en.at[j] >= 0 && p != 0.f) sum += p * (en.lp[j] + (lz - ((float)s[en.at[j]] - m) / t));
  }
  return sum_over<T>(sum, red) * t * t;
}

// ---- sums over the vocabulary ----------------------------------------------

struct Part {  // largest logit and sum exp2((s - m) c) of a row or of a slice
  float m, z;
};

__device__ __forceinline__ Part join(Part x, Part y, float c) {
  const float m = fmaxf(x.m, y.m);
  return Part{m, x.z * pow2((x.m - m) * c) + y.z * pow2((y.m - m) * c)};
}

// (m, z) of pieces [first, last) of a row, for all T threads.  Each thread
// keeps its own largest logit and rescales its sum when a batch of kAhead
// pieces raises it.
template <class E, int T>
__device__ __forceinline__ Part row_part(const Args& a, const E* s, int first, int last, float* red) {
  constexpr int N = Piece<E>::n, kAhead = 4;
  typedef typename Piece<E>::fvec F;
  float m = kLowest, z = 0.f;
  for (int64_t q = first + threadIdx.x; q < last; q += kAhead * T) {
    typename Piece<E>::vec v[kAhead];
    bool whole[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t c0 = (q + u * T) * N;
      whole[u] = q + u * T < last && c0 + N <= a.vocab;
      if (whole[u]) v[u] = *reinterpret_cast<const typename Piece<E>::any*>(s + c0);
    }
    F f[kAhead];
    float top = m;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (whole[u]) f[u] = __builtin_convertvector(v[u], F);
      else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int64_t c = (q + u * T) * N + e;
          f[u][e] = q + u * T < last && c < a.vocab ? (float)s[c] : -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, f[u][e]);
    }
    z *= pow2((m - top) * a.c);
    m = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) z += pow2((f[u][e] - m) * a.c);
  }
  const float top = max_over<T>(m, red);
  z = sum_over<T>(z * pow2((m - top) * a.c), red);
  return Part{top, z};
}

// The S parts of a row joined; a wave at a time, every wave the same.
__device__ __forceinline__ Part join_parts(const float2* parts, int S, float c) {
  const int lane = threadIdx.x & 63;
  Part p{kLowest, 0.f};
  if (lane < S) {
    const float2 f = parts[lane];
    p = Part{f.x, f.y};
  }
  if (S > 1)
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) p = join(p, Part{__shfl_xor(p.m, off, 64), __shfl_xor(p.z, off, 64)}, c);
  return Part{__shfl(p.m, 0, 64), __shfl(p.z, 0, 64)};
}

// Pieces [first, last) of slice s of S.
__device__ __forceinline__ void slice(int pieces, int S, int s, int& first, int& last) {
  const int per = (pieces + S - 1) / S;
  first = (int)std::min<int64_t>((int64_t)s * per, pieces);
  last = std::min(first + per, pieces);
}

// ---- gradient --------------------------------------------------------------

// The gradient of the entries' logits with index in [lo, hi): the first of
// equal indices writes, with all their p.
template <class E, int T>
__device__ __forceinline__ void entry_grads(const Args& a, const E* s, const Entries& en, Part st, float gs, int64_t lo,
                                            int64_t hi, E* ds) {
  for (int j = threadIdx.x; j < a.k; j += T) {
    const int at = en.at[j];
    if (at < lo || at >= hi) continue;
    float p = 0.f;
    bool first = true;
    for (int i = 0; i < a.k; ++i)
      if (en.at[i] == at) {
        first &= i >= j;
        p += en.p[i];
      }
    if (first) ds[at] = (E)(gs * (pow2(((float)s[at] - st.m) * a.c) / st.z - p));
  }
}

template <class E, int T>
__device__ __forceinline__ void zero_pieces(E* ds, int vocab, int first, int last) {
  for (int q = first + threadIdx.x; q < last; q += T) store_piece<E>(ds, q * Piece<E>::n, vocab, {});
}

// ---- kernels ---------------------------------------------------------------

// Unit u = (row, slice).  Writes the slice's part; used[row] (slice 0).  With
// LOSS (S = 1) the row's loss too.
template <class E, int T, bool LOSS>
__global__ __launch_bounds__(T) void distill_parts_kernel(Args a, int S, int64_t units, float2* __restrict__ parts,
                                                          int32_t* __restrict__ used, float* __restrict__ loss) {
  __shared__ float red[16];
  extern __shared__ float lds[];
  const Entries en = entries_of(lds, a.k);
  const int pieces = (int)(((int64_t)a.vocab + Piece<E>::n - 1) / Piece<E>::n);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t row = u / S;
    const int sl = (int)(u - row * S);
    const E* s = static_cast<const E*>(a.logits) + row * a.ld;
    const bool some = LOSS ? load_entries<T>(a, row, en, red) : has_entries<T>(a, row);
    Part p{0.f, 1.f};
    float l = 0.f;
    if (some) {
      int first, last;
      slice(pieces, S, sl, first, last);
      p = row_part<E, T>(a, s, first, last, red);
      if constexpr (LOSS) l = row_loss<E, T>(a, s, en, p.m, p.z, red);
    }
    if (threadIdx.x == 0) {
      parts[u] = make_float2(p.m, p.z);
      if (sl == 0) used[row] = some;
      if constexpr (LOSS) loss[row] = l;
    }
  }
}

// The losses of rows whose parts were made in slices.
template <class E>
__global__ __launch_bounds__(256) void distill_loss_kernel(Args a, int S, const float2* __restrict__ parts,
                                                           float* __restrict__ loss) {
  __shared__ float red[16];
  extern __shared__ float lds[];
  const Entries en = entries_of(lds, a.k);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float l = 0.f;
    if (load_entries<256>(a, row, en, red)) {
      const Part p = join_parts(parts + row * S, S, a.c);
      l = row_loss<E, 256>(a, static_cast<const E*>(a.logits) + row * a.ld, en, p.m, p.z, red);
    }
    if (threadIdx.x == 0) loss[row] = l;
  }
}

// n counts of rows with entries, for all T threads.
template <int T>
__device__ __forceinline__ float total_count(const int32_t* counts, int n, float* red) {
  // Exact in fp32 sums of parts below 2^24 each; a mean over more rows rounds.
  int64_t c = 0;
  for (int i = threadIdx.x; i < n; i += T) c += counts[i];
  return sum_over<T>((float)c, red);
}

// Gradient, unit u = (row, slice) of G.  The upstream gradient is g[row * gstep],
// times *factor where that is not null, times scale; `counts` (n of them, or
// null) divides by the number of rows with entries.  With `loss`, slice 0
// writes the row's loss.
template <class E, int T>
__global__ __launch_bounds__(T) void distill_grad_kernel(Args a, int S, const float2* __restrict__ parts, int G,
                                                         int64_t units, const float* __restrict__ g, int64_t gstep,
                                                         const float* __restrict__ factor, float scale,
                                                         const int32_t* __restrict__ counts, int n_counts,
                                                         E* __restrict__ grad, int64_t ldg, float* __restrict__ loss) {
  constexpr int N = Piece<E>::n, kAhead = 4;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ float red[16];
  extern __shared__ float lds[];
  const Entries en = entries_of(lds, a.k);
  const int pieces = (int)(((int64_t)a.vocab + N - 1) / N);
  if (factor) scale *= *factor;
  if (counts) scale /= fmaxf(total_count<T>(counts, n_counts, red), 1.f);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t row = u / G;
    const int sl = (int)(u - row * G);
    const E* s = static_cast<const E*>(a.logits) + row * a.ld;
    E* ds = grad + row * ldg;
    int first, last;
    slice(pieces, G, sl, first, last);
    if (!load_entries<T>(a, row, en, red)) {
      zero_pieces<E, T>(ds, a.vocab, first, last);
      if (loss && sl == 0 && threadIdx.x == 0) loss[row] = 0.f;
      continue;
    }
    const Part st = join_parts(parts + row * S, S, a.c);
    if (loss && sl == 0) {
      const float l = row_loss<E, T>(a, s, en, st.m, st.z, red);
      if (threadIdx.x == 0) loss[row] = l;
    }
    const float gs = (g ? g[row * gstep] * scale : scale) * a.temperature;
    // A row made NaN by an index past the vocabulary shows it everywhere.
    const float f = en.p[0] == en.p[0] ? gs / st.z : NAN;
    for (int64_t q = first + threadIdx.x; q < last; q += kAhead * T) {
      V v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (q + i * T < last) v[i] = load_piece(s, (int)((q + i * T) * N), a.vocab);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (q + i * T < last) {
          F o = __builtin_convertvector(v[i], F);
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = pow2((o[e] - st.m) * a.c) * f;
          store_piece(ds, (int)((q + i * T) * N), a.vocab, __builtin_convertvector(o, V));
        }
    }
    __syncthreads();  // the entries' logits are written again
    entry_grads<E, T>(a, s, en, st, gs, (int64_t)first * N, (int64_t)last * N, ds);
  }
}

// counts[b]: rows with entries among those of workgroup b, a wave a row.
__global__ __launch_bounds__(1024) void distill_count_kernel(Args a, int32_t* __restrict__ counts) {
  __shared__ int32_t sum[16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int32_t n = 0;
  for (int64_t row = (int64_t)blockIdx.x * 16 + wave; row < a.rows; row += (int64_t)gridDim.x * 16) {
    bool any = false;
    for (int j = 0; j < a.k && !any; j += 64) {
      bool here = false;
      if (j + lane < a.k) here = entry_counts(entry_index(a, row, j + lane), entry_logit(a, row, j + lane));
      any = __ballot(here) != 0;
    }
    n += any;
  }
  if (lane == 0) sum[wave] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t t = 0;
    for (int w = 0; w < 16; ++w) t += sum[w];
    counts[blockIdx.x] = t;
  }
}

// Loss and gradient of whole rows, NV pieces a thread in registers between the
// two.
template <class E, int T, int NV>
__global__ __launch_bounds__(T) void distill_step_kernel(Args a, float scale, const int32_t* __restrict__ counts,
                                                         int n_counts, E* __restrict__ grad, int64_t ldg,
                                                         float* __restrict__ loss, int32_t* __restrict__ used) {
  constexpr int N = Piece<E>::n;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ float red[16];
  extern __shared__ float lds[];
  const Entries en = entries_of(lds, a.k);
  if (counts) scale /= fmaxf(total_count<T>(counts, n_counts, red), 1.f);
  const int pieces = (int)(((int64_t)a.vocab + N - 1) / N);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const E* s = static_cast<const E*>(a.logits) + row * a.ld;
    E* ds = grad + row * ldg;
    const bool some = load_entries<T>(a, row, en, red);
    if (threadIdx.x == 0) used[row] = some;
    if (!some) {
      zero_pieces<E, T>(ds, a.vocab, 0, pieces);
      if (threadIdx.x == 0) loss[row] = 0.f;
      continue;
    }
    V v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + (int)threadIdx.x) * N;
      if (c + N <= a.vocab) v[i] = *reinterpret_cast<const typename Piece<E>::any*>(s + c);
      else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[i][e] = c + e < a.vocab ? s[c + e] : (E)-INFINITY;
      }
    }
    // Without these the compiler keeps every value widened from one loop to the
    // next, at twice the registers.
    auto forget = [&] {
#pragma unroll
      for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i]));
    };
    float m = kLowest;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const F f = __builtin_convertvector(v[i], F);
#pragma unroll
      for (int e = 0; e < N; ++e) m = fmaxf(m, f[e]);
    }
    m = max_over<T>(m, red);
    forget();
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const F f = __builtin_convertvector(v[i], F);
#pragma unroll
      for (int e = 0; e < N; ++e) z += pow2((f[e] - m) * a.c);
    }
    z = sum_over<T>(z, red);
    forget();
    const float gs = scale * a.temperature, f0 = en.p[0] == en.p[0] ? gs / z : NAN;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * T + (int)threadIdx.x) * N;
      if (c < a.vocab) {
        F o = __builtin_convertvector(v[i], F);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = pow2((o[e] - m) * a.c) * f0;
        store_piece(ds, c, a.vocab, __builtin_convertvector(o, V));
      }
    }
    const float l = row_loss<E, T>(a, s, en, m, z, red);
    if (threadIdx.x == 0) loss[row] = l;
    __syncthreads();
    entry_grads<E, T>(a, s, en, Part{m, z}, gs, 0, a.vocab, ds);
  }
}

// out[0] = sum of the rows' losses, divided by the rows with entries for the
// mean; out[1] (unless factor is null) = what it was multiplied by.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ loss,
                                                           const int32_t* __restrict__ used, int64_t rows, int mean,
                                                           float* __restrict__ out, float* __restrict__ factor) {
  __shared__ float red[16];
  float s = 0.f;
  int64_t n = 0;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    s += loss[r];
    n += used[r];
  }
  s = sum_over<1024>(s, red);
  const float c = sum_over<1024>((float)n, red);
  const float f = mean ? 1.f / fmaxf(c, 1.f) : 1.f;
  if (threadIdx.x == 0) {
    *out = s * f;
    if (factor) *factor = f;
  }
}

// ---- host -------------------------------------------------------------------

constexpr int kCus = 256;
constexpr int64_t kMaxGrid = 1 << 20;

int pieces_of(int vocab, int esz) { return (int)(((int64_t)vocab * esz + 15) / 16); }

// Slices of a row: two workgroups a CU where the rows alone do not give them,
// slices of 4096 values at least.
int slices(int64_t rows, int vocab) {
  if (rows <= 0) return 1;
  const int64_t want = (2 * kCus + rows - 1) / rows, most = vocab / 4096;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, (int64_t)kMaxSlices}));
}

// go(T) for slices of `values` values: one wave up to 2048, 256 threads up to
// 32768, 1024 beyond.
template <class Go>
void by_length(int64_t values, Go go) {
  if (values <= 2048) go(std::integral_constant<int, 64>{});
  else if (values <= 32768) go(std::integral_constant<int, 256>{});
  else go(std::integral_constant<int, 1024>{});
}

template <class Go>
void by_type(int32_t dtype, Go go) {
  if (dtype == VOID_DT_F32) go(float{});
  else if (dtype == VOID_DT_BF16) go(__bf16{});
  else go(_Float16{});
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VOID_OK : void_internal_fail(VOID_ERR_HIP, hipGetErrorString(e));
}

// 1: go on, 0: nothing to do, negative: refused.
int check(const void_distill_args* d) {
  if (!d) return void_internal_fail(VOID_ERR_ARG, "null arguments");
  if (d->rows < 0 || d->vocab < 0 || d->k < 0) return void_internal_fail(VOID_ERR_ARG, "negative size");
  if (d->k > kMaxEntries) return void_internal_fail(VOID_ERR_UNSUPPORTED, "too many teacher entries a row");
  auto type = [](int32_t t) { return t == VOID_DT_F32 || t == VOID_DT_BF16 || t == VOID_DT_F16; };
  if (!type(d->dtype) || !type(d->teacher_dtype))
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "logits are fp32, bf16 or fp16");
  if (d->index_bytes != 4 && d->index_bytes != 8)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "indices are int32 or int64");
  if (!(d->temperature > 0.f) || std::isinf(d->temperature))
    return void_internal_fail(VOID_ERR_ARG, "the temperature must be positive");
  if (d->rows == 0 || d->vocab == 0) return 0;
  const int esz = d->dtype == VOID_DT_F32 ? 4 : 2, tsz = d->teacher_dtype == VOID_DT_F32 ? 4 : 2;
  if (!d->logits || (d->k && (!d->teacher || !d->index))) return void_internal_fail(VOID_ERR_ARG, "null array");
  if (d->ld < 0 || d->ldt < 0 || d->ldi < 0) return void_internal_fail(VOID_ERR_ARG, "negative pitch");
  if ((uintptr_t)d->logits % esz || (uintptr_t)d->teacher % tsz || (uintptr_t)d->index % d->index_bytes)
    return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements");
  return 1;
}

Args args_of(const void_distill_args* d) {
  return Args{d->logits, d->teacher, d->index, d->ld, d->ldt, d->ldi, d->rows, d->vocab, d->k, d->teacher_dtype,
              d->index_bytes, d->temperature, (float)(1.4426950408889634 / (double)d->temperature)};
}

template <class E>
void parts(const Args& a, int S, float2* part, int32_t* used, float* loss, hipStream_t stream) {
  const int64_t units = a.rows * S;
  by_length((a.vocab + S - 1) / S, [&](auto t) {
    constexpr int T = decltype(t)::value;
    const dim3 grid((unsigned)std::min(units, kMaxGrid));
    if (S == 1 && loss)
      hipLaunchKernelGGL((distill_parts_kernel<E, T, true>), grid, dim3(T), entries_bytes(a.k), stream, a, S, units, part, used, loss);
    else
      hipLaunchKernelGGL((distill_parts_kernel<E, T, false>), grid, dim3(T), entries_bytes(a.k), stream, a, S, units, part, used, loss);
  });
  if (S > 1 && loss)
    hipLaunchKernelGGL(distill_loss_kernel<E>, dim3((unsigned)std::min(a.rows, kMaxGrid)), dim3(256), entries_bytes(a.k), stream, a, S,
                       part, loss);
}

template <class E>
void gradient(const Args& a, int S, const float2* part, const float* g, int64_t gstep, const float* factor, float scale,
              const int32_t* counts, int n_counts, void* grad, int64_t ldg, float* loss, hipStream_t stream) {
  const int64_t units = a.rows * S;
  by_length((a.vocab + S - 1) / S, [&](auto t) {
    constexpr int T = decltype(t)::value;
    hipLaunchKernelGGL((distill_grad_kernel<E, T>), dim3((unsigned)std::min(units, kMaxGrid)), dim3(T), entries_bytes(a.k), stream, a, S,
                       part, S, units, g, gstep, factor, scale, counts, n_counts, static_cast<E*>(grad), ldg, loss);
  });
}

// Registers of the one-read kernel: calls go(T, NV), false where a row does not fit.
template <class E, class Go>
bool by_row(int vocab, Go go) {
  using std::integral_constant;
#define VOID_ROW(T_, NV_) \
  if (pieces <= T_ * NV_) return go(integral_constant<int, T_>{}, integral_constant<int, NV_>{}), true
  const int pieces = pieces_of(vocab, (int)sizeof(E));
  VOID_ROW(64, 2);
  VOID_ROW(64, 4);
  VOID_ROW(256, 2);
  VOID_ROW(256, 4);
  VOID_ROW(256, 8);
  VOID_ROW(256, 16);
  VOID_ROW(1024, 8);
  VOID_ROW(1024, 16);
#undef VOID_ROW
  return false;
}

constexpr int kCountGrid = 256;

int count_grid(int64_t rows) { return (int)std::min<int64_t>((rows + 15) / 16, kCountGrid); }

}  // namespace

extern "C" {

int32_t void_distill_slices(int64_t rows, int32_t vocab) { return slices(rows, vocab); }

int void_distill_loss(const void_distill_args* d, float* row_loss, float* parts_, int32_t* used, hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const int st = check(d);
  if (st <= 0) return st;
  if (!row_loss || !parts_ || !used || (uintptr_t)parts_ % 8) return void_internal_fail(VOID_ERR_ARG, "null output");
  const Args a = args_of(d);
  by_type(d->dtype, [&](auto e) {
    parts<decltype(e)>(a, slices(d->rows, d->vocab), reinterpret_cast<float2*>(parts_), used, row_loss, stream);
  });
  return launched();
}

int void_distill_reduce(const float* row_loss, const int32_t* used, int64_t rows, int32_t mean, float* loss,
                        float* factor, hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  if (rows < 0 || !loss || (rows && (!row_loss || !used))) return void_internal_fail(VOID_ERR_ARG, "null array");
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, row_loss, used, rows, mean, loss, factor);
  return launched();
}

int void_distill_grad(const void_distill_args* d, const float* parts_, const float* upstream, int64_t upstream_step,
                      const float* factor, void* grad, int64_t ldg, hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const int st = check(d);
  if (st <= 0) return st;
  if (!parts_ || (uintptr_t)parts_ % 8 || !upstream || !grad || (uintptr_t)grad % (d->dtype == VOID_DT_F32 ? 4 : 2) ||
      (d->rows > 1 && ldg < d->vocab))
    return void_internal_fail(VOID_ERR_ARG, "null or misaligned array, or rows that overlap");
  const Args a = args_of(d);
  by_type(d->dtype, [&](auto e) {
    gradient<decltype(e)>(a, slices(d->rows, d->vocab), reinterpret_cast<const float2*>(parts_), upstream,
                          upstream_step, factor, 1.f, nullptr, 0, grad, ldg, nullptr, stream);
  });
  return launched();
}

size_t void_distill_step_workspace_bytes(int64_t rows, int32_t vocab) {
  if (rows <= 0) return 0;
  // Parts (8 bytes each), then a loss and a flag per row and the counts.
  return (size_t)rows * slices(rows, vocab) * 8 + (size_t)rows * 8 + kCountGrid * 4;
}

int void_distill_step(const void_distill_args* d, int32_t mean, float grad_scale, float* loss, void* grad, int64_t ldg,
                      void* workspace, size_t workspace_bytes, hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const int st = check(d);
  if (st < 0) return st;
  if (!loss) return void_internal_fail(VOID_ERR_ARG, "null loss");
  if (st == 0) return void_distill_reduce(nullptr, nullptr, 0, mean, loss, nullptr, stream);
  if (!grad || (uintptr_t)grad % (d->dtype == VOID_DT_F32 ? 4 : 2) || (d->rows > 1 && ldg < d->vocab))
    return void_internal_fail(VOID_ERR_ARG, "null or misaligned gradient, or rows that overlap");
  if (!workspace || (uintptr_t)workspace % 8 ||
      workspace_bytes < void_distill_step_workspace_bytes(d->rows, d->vocab))
    return void_internal_fail(VOID_ERR_WORKSPACE, "distillation: workspace missing or too small");
  const Args a = args_of(d);
  const int S = slices(d->rows, d->vocab);
  float2* part = static_cast<float2*>(workspace);
  float* row_loss = reinterpret_cast<float*>(part + d->rows * S);
  int32_t* used = reinterpret_cast<int32_t*>(row_loss + d->rows);
  int32_t* counts = used + d->rows;
  by_type(d->dtype, [&](auto e) {
    using E = decltype(e);
    if (S == 1) {
      const int n = count_grid(d->rows);
      auto count = [&] {
        if (mean) hipLaunchKernelGGL(distill_count_kernel, dim3(n), dim3(1024), 0, stream, a, counts);
      };
      if (by_row<E>(d->vocab, [&](auto t, auto nv) {
            constexpr int T = decltype(t)::value, NV = decltype(nv)::value;
            count();
            hipLaunchKernelGGL((distill_step_kernel<E, T, NV>),
                               dim3((unsigned)std::min<int64_t>(d->rows, kCus * (2048 / T))), dim3(T), entries_bytes(a.k), stream, a,
                               grad_scale, mean ? counts : nullptr, n, static_cast<E*>(grad), ldg, row_loss, used);
          }))
        return;
    }
    parts<E>(a, S, part, used, nullptr, stream);
    int n = (int)d->rows;
    const int32_t* c = used;
    if (mean && S == 1) {
      n = count_grid(d->rows);
      hipLaunchKernelGGL(distill_count_kernel, dim3(n), dim3(1024), 0, stream, a, counts);
      c = counts;
    }
    gradient<E>(a, S, part, nullptr, 0, nullptr, grad_scale, mean ? c : nullptr, n, grad, ldg, row_loss, stream);
  });
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, row_loss, used, d->rows, mean, loss, nullptr);
  return launched();
}

}  // extern "C"
