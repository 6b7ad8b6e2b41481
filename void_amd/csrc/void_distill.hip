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
// gradient is rounded once.  A row's entries live in LDS; one wave makes their
// probabilities, the loss and their logits' few gradients, which it writes again,
// with the p of equal indices added in order, behind the barrier that follows the
// row's gradient (no atomics).
//
// Many rows: one workgroup of T threads a row.  Few rows: S slices of each row,
// whose (m, z) parts every reader joins for itself in slice order.  Loss and
// gradient in one call keep what they can of a row in registers between the sum and
// the gradient and read the rest again while it is in the caches: one read of the
// memory, one write.

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

// The gradient is not read again here: its stores leave the caches to the logits.
template <class E>
__device__ __forceinline__ void stream_out(E* p, typename Piece<E>::vec v) {
  __builtin_nontemporal_store(v, reinterpret_cast<typename Piece<E>::any*>(p));
}

// ---- reductions over the T threads of a workgroup -------------------------
//
// One barrier each: every kind has an area of its own in LDS, and an area is
// written again only behind another barrier that follows its reads.

struct Areas {
  float max[16], sum[16];
  int flags[16];
};

template <int T>
__device__ __forceinline__ float max_over(float v, Areas& r) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) r.max[threadIdx.x >> 6] = v;
    __syncthreads();
    v = r.max[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) v = fmaxf(v, r.max[w]);
  }
  return v;
}

template <int T>
__device__ __forceinline__ float sum_over(float v, Areas& r) {
  v = lanes_sum<64>(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) r.sum[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += r.sum[w];
  }
  return v;
}

// The two low bits of v, or-ed: put() before a barrier, get() behind it.
template <int T>
__device__ __forceinline__ int put_flags(int v, Areas& r) {
  const int f = (__ballot(v & 1) ? 1 : 0) | (__ballot(v & 2) ? 2 : 0);
  if (T > 64 && (threadIdx.x & 63) == 0) r.flags[threadIdx.x >> 6] = f;
  return f;
}
template <int T>
__device__ __forceinline__ int get_flags(int f, const Areas& r) {
  if constexpr (T > 64) {
    f = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) f |= r.flags[w];
  }
  return __builtin_amdgcn_readfirstlane(f);
}

// ---- the teacher's entries of a row ---------------------------------------

constexpr int kSome = 1, kBad = 2;  // the row has an entry; one is past the vocabulary

// In dynamic LDS, k of each.
struct Entries {
  int32_t* at;  // index, -1 where the entry does not count
  float* t;     // the teacher's logit, later its probability
  float* s;     // the student's logit there
  float* w;     // the probabilities of all entries of its index; -1 unless it is the first of them
};

constexpr int pad4(int k) { return (k + 3) & ~3; }

__device__ __forceinline__ Entries entries_of(float* lds, int k) {
  return Entries{reinterpret_cast<int32_t*>(lds), lds + pad4(k), lds + 2 * pad4(k), lds + 3 * pad4(k)};
}

size_t entries_bytes(int k) { return (size_t)pad4(std::max(k, 1)) * 16; }

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

// What a row's entries ask for, by one wave (the others go on), in two parts.  The
// first needs the teacher alone: p and, where the gradient is made, the p of equal
// indices, which the first of them takes.  Returns the lane's part of sum p log p.
__device__ __forceinline__ float teacher_by_wave(const Args& a, const Entries& en, int flags, int64_t lo,
                                                 int64_t hi) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  for (int j = lane; j < a.k; j += 64)
    if (en.at[j] >= 0) {
      const float t = en.t[j];
      top = fmaxf(top, t == t ? t : kLowest);  // a NaN still counts
    }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  float sum = 0.f;
  for (int j = lane; j < a.k; j += 64)
    if (en.at[j] >= 0) sum += pow2((en.t[j] - top) * a.c);
  sum = flags & kBad ? NAN : lanes_sum<64>(sum);
  const float inv = 1.f / sum, log_sum = logf(sum);
  float own = 0.f;
  for (int j = lane; j < a.k; j += 64) {
    const float d = en.t[j] - top, p = en.at[j] >= 0 ? pow2(d * a.c) * inv : 0.f;
    if (p != 0.f) own += p * (d / a.temperature - log_sum);  // log p
    en.t[j] = p;
  }
  lanes_in_order();  // equal indices' p are other lanes'
  for (int j = lane; j < a.k; j += 64) {
    const int at = en.at[j];
    if (at < lo || at >= hi) continue;
    float p = 0.f;
    bool first = true;
    for (int i = 0; i < a.k; i += 4) {
      const int4 q = *reinterpret_cast<const int4*>(en.at + i);
      if (q.x == at || q.y == at || q.z == at || q.w == at) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w) == at) {
            first &= i + e >= j;
            p += en.t[i + e];
          }
      }
    }
    en.w[j] = first ? p : -1.f;
  }
  return own;
}

// The second needs m and z = sum exp2((s - m) c): the loss (returned) and, unless ds
// is null, the gradients of the entries' logits with index in [lo, hi), behind a
// barrier that follows everything else of the row's gradient.
template <class E>
__device__ __forceinline__ float entries_by_wave(const Args& a, const Entries& en, float own, float m, float z, float gs,
                                                 int64_t lo, int64_t hi, E* ds) {
  const int lane = threadIdx.x & 63;
  const float back = logf(z), iz = 1.f / z;
  float loss = own;
  for (int j = lane; j < a.k; j += 64) {
    const float p = en.t[j], d = en.s[j] - m;
    if (p != 0.f) loss += p * (back - d / a.temperature);  // - log q
    if (ds) {
      const int at = en.at[j];
      const float w = en.w[j];
      if (at >= lo && at < hi && !(w < 0.f)) ds[at] = (E)(gs * (pow2(d * a.c) * iz - w));
    }
  }
  return lanes_sum<64>(loss) * a.temperature * a.temperature;
}

// ---- slices of a row ---------------------------------------------------------

struct Part {  // largest logit and sum exp2((s - m) c) of a row or of a slice
  float m, z;
};

// Slice s of S: whole pieces [first, last), and, the last slice, the row's `rest`
// values behind them.
template <class E>
struct Slice {
  static constexpr int N = Piece<E>::n;
  uint32_t first, last, rest;
  int64_t lo, hi;  // its columns
  __device__ __forceinline__ Slice(int vocab, int S, int s) {
    const uint32_t whole = (uint32_t)vocab / N, per = (whole + S - 1) / S;
    first = min(per * s, whole);
    last = min(first + per, whole);
    rest = s == S - 1 ? (uint32_t)vocab % N : 0;
    lo = (int64_t)first * N;
    hi = (int64_t)last * N + rest;
  }
};

__device__ __forceinline__ Part join(Part x, Part y, float c) {
  const float m = fmaxf(x.m, y.m);
  return Part{m, x.z * pow2((x.m - m) * c) + y.z * pow2((y.m - m) * c)};
}

// (m, z) of a slice, for all T threads.  Each thread keeps its own largest logit and
// rescales its sum when a batch of kAhead pieces raises it.
template <class E, int T, bool ODD>
__device__ __forceinline__ Part slice_part(const Args& a, const E* s, const Slice<E>& sl, Areas& red) {
  constexpr int N = Piece<E>::n, kAhead = 4;
  typedef typename Piece<E>::fvec F;
  float m = kLowest, z = 0.f;
  if (threadIdx.x < sl.rest) {
    const float x = (float)s[(int64_t)sl.last * N + threadIdx.x];
    m = fmaxf(m, x);
    z = pow2((x - m) * a.c);
  }
  for (uint32_t q = sl.first + threadIdx.x; q < sl.last; q += kAhead * T) {
    Loaded<E, ODD> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      v[u].lowest();
      if (q + u * T < sl.last) v[u].whole(s + (int64_t)(q + u * T) * N);
    }
    float top = m;
    F f[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      f[u] = __builtin_convertvector(v[u].take(s), F);
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

// The S parts of a row, one a lane, and joined; a wave at a time, every wave the same.
__device__ __forceinline__ Part lane_part(const float2* parts, int S) {
  const int lane = threadIdx.x & 63;
  const float2 f = lane < S ? parts[lane] : make_float2(kLowest, 0.f);
  return Part{f.x, f.y};
}
__device__ __forceinline__ Part join_parts(Part p, int S, float c) {
  if (S > 1)
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) p = join(p, Part{__shfl_xor(p.m, off, 64), __shfl_xor(p.z, off, 64)}, c);
  return Part{__shfl(p.m, 0, 64), __shfl(p.z, 0, 64)};
}

template <class E, int T>
__device__ __forceinline__ void zero_slice(E* ds, const Slice<E>& sl) {
  for (uint32_t q = sl.first + threadIdx.x; q < sl.last; q += T) stream_out(ds + (int64_t)q * Piece<E>::n, {});
  if (threadIdx.x < sl.rest) ds[(int64_t)sl.last * Piece<E>::n + threadIdx.x] = (E)0.f;
}

// A row's entries into LDS, with its logits there where it has any; its flags.  Every
// thread's entries stand before the barrier here, the logits (en.s) behind it: where other
// lanes read those, another barrier comes first.
template <class E, int T>
__device__ __forceinline__ int take_entries(const Args& a, int64_t row, const E* s, const Entries& en, Areas& red) {
  __syncthreads();  // en is free
  int flags = 0;
  for (int j = threadIdx.x; j < pad4(a.k); j += T) {
    int at = -1;
    if (j < a.k) {
      const int64_t v = entry_index(a, row, j);
      const float t = entry_logit(a, row, j);
      const bool use = entry_counts(v, t);
      at = !use ? -1 : v < a.vocab ? (int32_t)v : 0;
      flags |= !use ? 0 : v < a.vocab ? kSome : kSome | kBad;
      en.t[j] = t;
    }
    en.at[j] = at;
  }
  flags = put_flags<T>(flags, red);
  __syncthreads();
  flags = get_flags<T>(flags, red);
  if (flags & kSome)
    for (int j = threadIdx.x; j < a.k; j += T) en.s[j] = (float)s[max(en.at[j], 0)];
  return flags;
}

// ---- kernels ---------------------------------------------------------------

// Unit u = (row, slice).  Writes the slice's part; used[row] (slice 0).  With
// LOSS (S = 1) the row's loss too.  Clears `arrived` (unless null).  Bound by reading the
// logits: 4096 x 32768 bf16 63 us between other work, 4.2 TB/s (52 us call after call, partly
// from the caches); 730 x 50021 fp32 with a quarter of the rows without entries 24.5 us,
// 4.5 TB/s.
template <class E, int T, bool LOSS, bool ODD>
__global__ __launch_bounds__(T) void distill_parts_kernel(Args a, int S, int64_t units, float2* __restrict__ parts,
                                                          int32_t* __restrict__ used, float* __restrict__ loss,
                                                          int32_t* __restrict__ arrived) {
  __shared__ Areas red;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const Entries en = entries_of(lds, a.k);
  if (arrived && blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t row = u / S;
    const int sl = (int)(u - row * S);
    const E* s = static_cast<const E*>(a.logits) + row * a.ld;
    int flags;
    if constexpr (LOSS) {
      flags = take_entries<E, T>(a, row, s, en, red);
    } else {
      flags = 0;
      for (int j = threadIdx.x; j < a.k; j += T)
        flags |= entry_counts(entry_index(a, row, j), entry_logit(a, row, j)) ? kSome : 0;
      flags = put_flags<T>(flags, red);
      __syncthreads();
      flags = get_flags<T>(flags, red);
    }
    Part p{0.f, 1.f};
    if (flags & kSome) p = slice_part<E, T, ODD>(a, s, Slice<E>(a.vocab, S, sl), red);
    if (threadIdx.x < 64) {
      float l = 0.f;
      if constexpr (LOSS)
        if (flags & kSome)
          l = entries_by_wave<E>(a, en, teacher_by_wave(a, en, flags, 0, 0), p.m, p.z, 0.f, 0, 0, nullptr);
      if (threadIdx.x == 0) {
        parts[u] = make_float2(p.m, p.z);
        if (sl == 0) used[row] = flags & kSome;
        if constexpr (LOSS) loss[row] = l;
      }
    }
    if constexpr (!LOSS) __syncthreads();  // the areas are free
  }
}

// The losses of rows whose parts were made in slices; a wave a row.
template <class E>
__global__ __launch_bounds__(64) void distill_loss_kernel(Args a, int S, const float2* __restrict__ parts,
                                                          float* __restrict__ loss) {
  __shared__ Areas red;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const Entries en = entries_of(lds, a.k);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float l = 0.f;
    const int flags = take_entries<E, 64>(a, row, static_cast<const E*>(a.logits) + row * a.ld, en, red);
    if (flags & kSome) {
      const Part p = join_parts(lane_part(parts + row * S, S), S, a.c);
      l = entries_by_wave<E>(a, en, teacher_by_wave(a, en, flags, 0, 0), p.m, p.z, 0.f, 0, 0, nullptr);
    }
    if (threadIdx.x == 0) loss[row] = l;
  }
}

// The sum of n counts of rows with entries, by each wave for itself.
__device__ __forceinline__ float total_count(const int32_t* counts, int n) {
  int64_t c = 0;
  for (int i = threadIdx.x & 63; i < n; i += 64) c += counts[i];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) c += __shfl_xor(c, off, 64);
  return (float)c;
}

// A row's loss by one wave.  With `total` the wave that is last to come (the rows' count
// of them is in `arrived`) sums all losses in a fixed order, times `share`.
__device__ __forceinline__ void add_row_loss(const Args& a, int64_t row, float l, float* loss, float share,
                                             float* total, int32_t* arrived) {
  const int lane = threadIdx.x & 63;
  if (!total) {
    if (lane == 0) loss[row] = l;
    return;
  }
  int before = 0;
  if (lane == 0) {
    __hip_atomic_store(loss + row, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (__shfl(before, 0, 64) != (int)a.rows - 1) return;
  float s = 0.f;
  for (int64_t r = lane; r < a.rows; r += 64)
    s += __hip_atomic_load(loss + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s = lanes_sum<64>(s);
  if (lane == 0) *total = s * share;
}

// Gradient, unit u = (row, slice) of G.  The upstream gradient is g[row * gstep],
// times *factor where that is not null, times scale; `counts` (n of them, or
// null) divides by the number of rows with entries.  With `loss`, slice 0
// writes the row's loss; `total` (unless null) becomes their sum or mean.  Bound by
// one read of the logits and one write of as much: 4096 x 32768 bf16 102 us, 5.3 TB/s;
// 730 x 50021 fp32 with a quarter of the rows without entries 55 us, 4.7 TB/s.  What
// the entries need of the teacher is made while the logits come (300 x 131072 bf16,
// loss and gradient: 50.4 us, and 54.4 at the end).
template <class E, int T, bool ODD>
__global__ __launch_bounds__(T) void distill_grad_kernel(Args a, int S, const float2* __restrict__ parts, int G,
                                                         int64_t units, const float* __restrict__ g, int64_t gstep,
                                                         const float* __restrict__ factor, float scale,
                                                         const int32_t* __restrict__ counts, int n_counts,
                                                         E* __restrict__ grad, int64_t ldg, float* __restrict__ loss,
                                                         float* __restrict__ total, int32_t* __restrict__ arrived) {
  constexpr int N = Piece<E>::n, kAhead = 4;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ Areas red;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const Entries en = entries_of(lds, a.k);
  if (factor) scale *= *factor;
  const float share = counts ? 1.f / fmaxf(total_count(counts, n_counts), 1.f) : 1.f;
  scale *= share;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t row = u / G;
    const int n = (int)(u - row * G);
    const Slice<E> sl(a.vocab, G, n);
    const E* s = static_cast<const E*>(a.logits) + row * a.ld;
    E* ds = grad + row * ldg;
    const Part mine = lane_part(parts + row * S, S);
    const int flags = take_entries<E, T>(a, row, s, en, red);
    if (!(flags & kSome)) {
      zero_slice<E, T>(ds, sl);
      if (loss && n == 0 && threadIdx.x < 64) add_row_loss(a, row, 0.f, loss, share, total, arrived);
      continue;
    }
    const float gs = (g ? g[row * gstep] * scale : scale) * a.temperature;
    Loaded<E, ODD> v[kAhead];
    auto load = [&](uint32_t q) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (q + i * T < sl.last) v[i].whole(s + (int64_t)(q + i * T) * N);
    };
    uint32_t q = sl.first + threadIdx.x;
    load(q);
    float own = 0.f;
    if (threadIdx.x < 64) own = teacher_by_wave(a, en, flags, sl.lo, sl.hi);  // while they come
    const Part st = join_parts(mine, S, a.c);
    const float f = flags & kBad ? NAN : gs / st.z;
    while (q < sl.last) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (q + i * T < sl.last) {
          F o = __builtin_convertvector(v[i].take(s), F);
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = pow2((o[e] - st.m) * a.c) * f;
          stream_out(ds + (int64_t)(q + i * T) * N, __builtin_convertvector(o, V));
        }
      q += kAhead * T;
      load(q);
    }
    if (threadIdx.x < sl.rest) {
      const int64_t c = (int64_t)sl.last * N + threadIdx.x;
      ds[c] = (E)(pow2(((float)s[c] - st.m) * a.c) * f);
    }
    __syncthreads();  // the entries' logits are written again
    if (threadIdx.x < 64) {
      const float l = entries_by_wave<E>(a, en, own, st.m, st.z, gs, sl.lo, sl.hi, ds);
      if (loss && n == 0) add_row_loss(a, row, l, loss, share, total, arrived);
    }
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

// Loss and gradient of whole rows.  The first NV pieces a thread of a row stay in
// registers between its sums and its gradient; what a longer row has behind them is
// read again from the caches.  Four waves a SIMD: while one workgroup sums, others
// load and store.  Bound by the memory: 8192 x 65536 bf16 466 us, 4.6 TB/s of one read
// and one write; x 131072 967 us, 4.45, with a quarter of the rows without entries
// 820 to 870 us, 4.3 to 4.6 (a copy of 2 GiB: 4.94); 2048 x 65536 fp32 239 us, 4.5.
template <class E, int T, int NV, bool ODD>
__global__ __launch_bounds__(T, 4) void distill_step_kernel(Args a, float scale, const int32_t* __restrict__ counts,
                                                            int n_counts, E* __restrict__ grad, int64_t ldg,
                                                            float* __restrict__ loss, int32_t* __restrict__ used) {
  constexpr int N = Piece<E>::n, kAhead = 2;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  __shared__ Areas red;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const Entries en = entries_of(lds, a.k);
  if (counts) scale /= fmaxf(total_count(counts, n_counts), 1.f);
  const float gs = scale * a.temperature;
  const uint32_t whole = (uint32_t)a.vocab / N, rest = (uint32_t)a.vocab % N;
  const std::make_integer_sequence<int, NV> pieces_each;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const E* s = static_cast<const E*>(a.logits) + row * a.ld;
    E* ds = grad + row * ldg;
    const int flags = take_entries<E, T>(a, row, s, en, red);
    if (threadIdx.x == 0) used[row] = flags & kSome;
    if (!(flags & kSome)) {
      zero_slice<E, T>(ds, Slice<E>(a.vocab, 1, 0));
      if (threadIdx.x == 0) loss[row] = 0.f;
      continue;
    }
    V v[NV];
    // Else the compiler keeps every value widened from one loop to the next, at
    // twice the registers.
    auto forget = [&] {
#pragma unroll
      for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i]));
    };
    {
      Loaded<E, ODD> in[NV];
      each_of(
          [&](auto i) {
            const uint32_t q = (uint32_t)i.value * T + threadIdx.x;
            in[i.value].lowest();
            if (q < whole) in[i.value].whole(s + (int64_t)q * N);
          },
          pieces_each);
      each_of([&](auto i) { v[i.value] = in[i.value].take(s); }, pieces_each);
    }
    const float tail = threadIdx.x < rest ? (float)s[(int64_t)whole * N + threadIdx.x] : -INFINITY;
    // A thread's own largest logit first: what lies behind the registers, rescaling
    // its sum as it rises, then the registers.
    float m = kLowest, z = 0.f;
#pragma unroll 1
    for (uint32_t q = NV * T + threadIdx.x; q < whole; q += kAhead * T) {
      Loaded<E, ODD> w[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        w[u].lowest();
        if (q + u * T < whole) w[u].whole(s + (int64_t)(q + u * T) * N);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const F f = __builtin_convertvector(w[u].take(s), F);
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, f[e]);
      }
      z *= pow2((m - top) * a.c);
      m = top;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const F f = __builtin_convertvector(w[u].take(s), F);
#pragma unroll
        for (int e = 0; e < N; ++e) z += pow2((f[e] - m) * a.c);
      }
    }
    float top = fmaxf(m, tail);
    each_of(
        [&](auto i) {
          const F f = __builtin_convertvector(v[i.value], F);
#pragma unroll
          for (int e = 0; e < N; ++e) top = fmaxf(top, f[e]);
          __builtin_amdgcn_sched_barrier(0);
        },
        pieces_each);
    forget();
    z *= pow2((m - top) * a.c);
    m = top;
    z += pow2((tail - m) * a.c);
    each_of(
        [&](auto i) {
          const F f = __builtin_convertvector(v[i.value], F);
#pragma unroll
          for (int e = 0; e < N; ++e) z += pow2((f[e] - m) * a.c);
          __builtin_amdgcn_sched_barrier(0);
        },
        pieces_each);
    forget();
    top = max_over<T>(m, red);
    z = sum_over<T>(z * pow2((m - top) * a.c), red);
    m = top;
    const float f0 = flags & kBad ? NAN : gs / z;
    each_of(
        [&](auto i) {
          const uint32_t q = (uint32_t)i.value * T + threadIdx.x;
          if (q < whole) {
            F o = __builtin_convertvector(v[i.value], F);
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = pow2((o[e] - m) * a.c) * f0;
            stream_out(ds + (int64_t)q * N, __builtin_convertvector(o, V));
          }
          __builtin_amdgcn_sched_barrier(0);
        },
        pieces_each);
#pragma unroll 1
    for (uint32_t q = NV * T + threadIdx.x; q < whole; q += kAhead * T) {
      Loaded<E, ODD> w[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (q + u * T < whole) w[u].whole(s + (int64_t)(q + u * T) * N);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (q + u * T < whole) {
          F o = __builtin_convertvector(w[u].take(s), F);
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = pow2((o[e] - m) * a.c) * f0;
          stream_out(ds + (int64_t)(q + u * T) * N, __builtin_convertvector(o, V));
        }
    }
    if (threadIdx.x < rest) ds[(int64_t)whole * N + threadIdx.x] = (E)(pow2((tail - m) * a.c) * f0);
    __syncthreads();  // the entries' logits are written again
    // Both parts here: the other waves end now and make room for the next row's (with
    // the first part before the barrier 8192 x 16384 bf16 139 us against 125).
    if (threadIdx.x < 64) {
      const float own = teacher_by_wave(a, en, flags, 0, a.vocab);
      const float l = entries_by_wave<E>(a, en, own, m, z, gs, 0, a.vocab, ds);
      if (threadIdx.x == 0) loss[row] = l;
    }
  }
}

// out[0] = sum of the rows' losses, divided by the rows with entries for the
// mean; out[1] (unless factor is null) = what it was multiplied by.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ loss,
                                                           const int32_t* __restrict__ used, int64_t rows, int mean,
                                                           float* __restrict__ out, float* __restrict__ factor) {
  __shared__ Areas red;
  float s = 0.f;
  int64_t n = 0;
  // Four rows in flight; a thread's are added in order.
  for (int64_t r = threadIdx.x; r < rows; r += 4 * 1024) {
    float l[4];
    int u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = r + i * 1024 < rows;
      l[i] = in ? loss[r + i * 1024] : 0.f;
      u[i] = in ? used[r + i * 1024] : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s += l[i];
      n += u[i];
    }
  }
  s = sum_over<1024>(s, red);
  __syncthreads();
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

// Slices of a row: two workgroups a CU where the rows alone do not give them,
// slices of 4096 values at least.
int slices(int64_t rows, int vocab) {
  if (rows <= 0) return 1;
  const int64_t want = (2 * kCus + rows - 1) / rows, most = vocab / 4096;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, (int64_t)kMaxSlices}));
}

// go(T) for slices of `pieces` 16-byte pieces: few threads a slice, since each
// workgroup has its entries to see to (gradient of 8192 rows bf16: 2000 wide 19 us with
// 64 threads, 31 with 256; 8192 wide 60 and 52; 2048 x 131072 216 with 256, 208 with 512).
// With `few` rows to fill the chip 256 at least (loss and gradient of one row x 131072
// 13.3 us, and 14.4 with 64).
template <class Go>
void by_length(int64_t pieces, bool few, Go go) {
  if (!few && pieces <= 512) go(std::integral_constant<int, 64>{});
  else if (pieces <= 8192) go(std::integral_constant<int, 256>{});
  else go(std::integral_constant<int, 512>{});
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
  if (d->vocab > INT_MAX / 2) return void_internal_fail(VOID_ERR_UNSUPPORTED, "vocabularies are limited to 2^30 values");
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
void parts(const Args& a, int S, float2* part, int32_t* used, float* loss, int32_t* arrived, hipStream_t stream) {
  const int64_t units = a.rows * S;
  by_length(((int64_t)a.vocab / S + Piece<E>::n - 1) / Piece<E>::n, S > 1, [&](auto t) {
    by_parity<E>(a.logits, a.ld, nullptr, 0, a.rows, [&](auto odd) {
      constexpr int T = decltype(t)::value;
      constexpr bool ODD = decltype(odd)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(units, kMaxGrid)), dim3(T), entries_bytes(a.k), stream, a, S,
                           units, part, used, loss, arrived);
      };
      if (S == 1 && loss) go(distill_parts_kernel<E, T, true, ODD>);
      else go(distill_parts_kernel<E, T, false, ODD>);
    });
  });
  if (S > 1 && loss)
    hipLaunchKernelGGL(distill_loss_kernel<E>, dim3((unsigned)std::min(a.rows, kMaxGrid)), dim3(64), entries_bytes(a.k),
                       stream, a, S, part, loss);
}

template <class E>
void gradient(const Args& a, int S, const float2* part, const float* g, int64_t gstep, const float* factor, float scale,
              const int32_t* counts, int n_counts, void* grad, int64_t ldg, float* loss, float* total, int32_t* arrived,
              hipStream_t stream) {
  const int64_t units = a.rows * S;
  by_length(((int64_t)a.vocab / S + Piece<E>::n - 1) / Piece<E>::n, S > 1, [&](auto t) {
    by_parity<E>(a.logits, a.ld, nullptr, 0, a.rows, [&](auto odd) {
      constexpr int T = decltype(t)::value;
      hipLaunchKernelGGL((distill_grad_kernel<E, T, decltype(odd)::value>), dim3((unsigned)std::min(units, kMaxGrid)),
                         dim3(T), entries_bytes(a.k), stream, a, S, part, S, units, g, gstep, factor, scale, counts,
                         n_counts, static_cast<E*>(grad), ldg, loss, total, arrived);
    });
  });
}

// Threads and register pieces of the one-read kernel: calls go(T, NV).  Few threads a
// row, since each workgroup has its entries to see to, and eight pieces at most, with
// which four waves fit a SIMD (sixteen spill): 8192 x 32768 bf16 242 us with 256
// threads and 268 with 512; x 65536 461 and 463; x 131072 (a quarter of the rows
// without entries) 884 and 810, for all rows read by 1024 threads 16 pieces deep 1118.
template <class E, class Go>
void by_row(int vocab, Go go) {
  using std::integral_constant;
  const int pieces = vocab / Piece<E>::n;
  if (pieces <= 64 * 2) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (pieces <= 64 * 4) go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (pieces <= 64 * 8) go(integral_constant<int, 64>{}, integral_constant<int, 8>{});
  else if (pieces <= 128 * 8) go(integral_constant<int, 128>{}, integral_constant<int, 8>{});
  else if (pieces <= 8192) go(integral_constant<int, 256>{}, integral_constant<int, 8>{});
  else go(integral_constant<int, 512>{}, integral_constant<int, 8>{});
}

constexpr int kCountGrid = 256;

// Up to so many rows the gradient's kernel sums the losses itself, a launch less: 8 rows
// x 131072 bf16 12.7 us against 14.2 (15.2 and 18.2 with the host's part).  Each row that
// arrives writes an L2 back, so that more rows lose by it: 64 of the same 27 us and 19.5.
constexpr int64_t kJoinedRows = 16;

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
    parts<decltype(e)>(a, slices(d->rows, d->vocab), reinterpret_cast<float2*>(parts_), used, row_loss, nullptr,
                       stream);
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
                          upstream_step, factor, 1.f, nullptr, 0, grad, ldg, nullptr, nullptr, nullptr, stream);
  });
  return launched();
}

size_t void_distill_step_workspace_bytes(int64_t rows, int32_t vocab) {
  if (rows <= 0) return 0;
  // Parts (8 bytes each), then a loss and a flag per row and the counts (of the arrived, for few rows).
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
  auto sum = [&] {
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, row_loss, used, d->rows, mean, loss, nullptr);
  };
  by_type(d->dtype, [&](auto e) {
    using E = decltype(e);
    if (S == 1) {
      const int n = count_grid(d->rows);
      if (mean) hipLaunchKernelGGL(distill_count_kernel, dim3(n), dim3(1024), 0, stream, a, counts);
      by_row<E>(d->vocab, [&](auto t, auto nv) {
        by_parity<E>(d->logits, d->ld, nullptr, 0, d->rows, [&](auto odd) {
          constexpr int T = decltype(t)::value;
          constexpr int NV = decltype(nv)::value;
          constexpr bool ODD = decltype(odd)::value;
          hipLaunchKernelGGL((distill_step_kernel<E, T, NV, ODD>), dim3((unsigned)std::min(d->rows, kMaxGrid)), dim3(T),
                             entries_bytes(a.k), stream, a, grad_scale, mean ? counts : nullptr, n,
                             static_cast<E*>(grad), ldg, row_loss, used);
        });
      });
      sum();
      return;
    }
    // Few rows: the parts of their slices, then the gradient and each row's loss.
    const bool join = d->rows <= kJoinedRows;
    parts<E>(a, S, part, used, nullptr, join ? counts : nullptr, stream);
    gradient<E>(a, S, part, nullptr, 0, nullptr, grad_scale, mean ? used : nullptr, (int)d->rows, grad, ldg, row_loss,
                join ? loss : nullptr, counts, stream);
    if (!join) sum();
  });
  return launched();
}

}  // extern "C"
