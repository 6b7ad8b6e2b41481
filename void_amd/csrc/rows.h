// rows.h — 16-byte pieces of float rows and sums over the threads of a row,
// shared by the layer norm, distillation and dense layer kernels.
//
// A piece is 16 bytes of a row: 8 bf16 / fp16 values or 4 fp32 values.  Rows
// need no alignment past their elements': global memory takes 16-byte accesses
// at any element address, so a row of any width and pitch is read and written
// in whole pieces, and only the piece that the row ends in is put together.  Loads
// that start between two dwords are slow, so that rows of 16-bit values of odd
// widths have variants that load whole dwords (Loaded).

#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

namespace {

template <class E>
struct Piece {
  static constexpr int n = 16 / (int)sizeof(E);
  typedef E vec __attribute__((ext_vector_type(16 / sizeof(E))));
  typedef float fvec __attribute__((ext_vector_type(16 / sizeof(E))));
  typedef vec any __attribute__((aligned(sizeof(E))));
};

// The piece of a row of `cols` values that starts at column c; zeros past the end.
template <class E>
__device__ __forceinline__ typename Piece<E>::vec load_piece(const E* row, int c, int cols) {
  typename Piece<E>::vec v = {};
  if (c + Piece<E>::n <= cols) {
    v = *reinterpret_cast<const typename Piece<E>::any*>(row + c);
  } else if (sizeof(E) == 2 && cols >= Piece<E>::n) {
    // The row's last n values in one load, shifted down to where they belong: loads of
    // single values, each behind a branch, would wait for each other.  (fp32 has three
    // of them at most: layer norm of 5003 x 3001 took 3 % more this way.)
    const auto last = *reinterpret_cast<const typename Piece<E>::any*>(row + cols - Piece<E>::n);
    const uint32_t by = (uint32_t)(c + Piece<E>::n - cols);
    if (c < cols)
      v = __builtin_bit_cast(typename Piece<E>::vec, __builtin_bit_cast(unsigned __int128, last) >> (by * (8 * sizeof(E))));
  } else {
#pragma unroll
    for (int e = 0; e < Piece<E>::n; ++e)
      if (c + e < cols) v[e] = row[c + e];
  }
  return v;
}

template <class E>
__device__ __forceinline__ void store_piece(E* row, int c, int cols, typename Piece<E>::vec v) {
  if (c + Piece<E>::n <= cols) {
    *reinterpret_cast<typename Piece<E>::any*>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < Piece<E>::n; ++e)
      if (c + e < cols) row[c + e] = v[e];
  }
}

// A piece on its way from a row.  Where ODD, the row may start between two dwords: loads
// at such addresses run at half the rate, so the dwords that hold the piece are loaded
// as they lie, and take() shifts them into place when they are used (layer norm of
// 16384 x 8191 bf16 forward 109 us, and 165 without; backward 242 and 334).
template <class E, bool ODD>
struct Loaded {
  typename Piece<E>::vec v;
  __device__ __forceinline__ void load(const E* row, int c, int cols) { v = load_piece(row, c, cols); }
  __device__ __forceinline__ void whole(const E* p) { v = *reinterpret_cast<const typename Piece<E>::any*>(p); }
  __device__ __forceinline__ typename Piece<E>::vec take(const E*) const { return v; }
  __device__ __forceinline__ typename Piece<E>::vec take(const E*, int, int) const { return v; }
  __device__ __forceinline__ void lowest() { v = (E)-INFINITY; }
};
template <class E>
struct Loaded<E, true> {
  static_assert(sizeof(E) == 2);
  typedef uint32_t V4 __attribute__((ext_vector_type(4)));
  typedef V4 Any __attribute__((aligned(4)));
  V4 lo;
  uint32_t hi;
  __device__ __forceinline__ void lowest() {  // -inf wherever it is shifted to
    lo = hi = (uint32_t)__builtin_bit_cast(uint16_t, (E)-INFINITY) * 0x10001u;
  }
  // Every dword that is read holds some of the piece's values.
  __device__ __forceinline__ void whole(const E* p) {
    const uintptr_t a = (uintptr_t)p;
    lo = *reinterpret_cast<const Any*>(a & ~(uintptr_t)3);
    hi = *reinterpret_cast<const uint32_t*>((a + 14) & ~(uintptr_t)3);
  }
  __device__ __forceinline__ void load(const E* row, int c, int cols) {
    lo = 0;
    hi = 0;
    if (c + 8 <= cols) {
      whole(row + c);
    } else if (c < cols) {
      const uintptr_t first = (uintptr_t)(row + c) & ~(uintptr_t)3, last = (uintptr_t)(row + cols - 1) & ~(uintptr_t)3;
#pragma unroll
      for (int i = 0; i < 4; ++i) lo[i] = *reinterpret_cast<const uint32_t*>(first + 4 * i < last ? first + 4 * i : last);
      hi = *reinterpret_cast<const uint32_t*>(last);
    }
  }
  // Of a whole piece of a row (any address of the row's parity).
  __device__ __forceinline__ typename Piece<E>::vec take(const E* row) const {
    const uint32_t by = ((uint32_t)(uintptr_t)row & 2) * 8;
    V4 d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = __builtin_amdgcn_alignbit(i < 3 ? lo[i + 1] : hi, lo[i], by);
    return __builtin_bit_cast(typename Piece<E>::vec, d);
  }
  __device__ __forceinline__ typename Piece<E>::vec take(const E* row, int c, int cols) const {
    typename Piece<E>::vec v = take(row);
    if (c + 8 > cols)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? v[e] : (E)0.f;
    return v;
  }
};

// go(ODD) for arrays of rows at `a` and `b`: whether any of them may start between dwords.
template <class E, class Go>
void by_parity(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, Go go) {
  const uintptr_t at = (uintptr_t)a | (uintptr_t)b | (rows > 1 ? (uintptr_t)((lda | ldb) * (int64_t)sizeof(E)) : 0);
  if constexpr (sizeof(E) == 2)
    if (at & 3) return go(std::true_type{});
  go(std::false_type{});
}

// n values of a parameter vector (weight, bias) from column c, in fp32; `none`
// stands for each where there is no vector, zero past the end.
template <int N, class W>
__device__ __forceinline__ void load_params(float (&f)[N], const W* p, int c, int cols, float none) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = none;
  } else if (c + N <= cols) {
#pragma unroll
    for (int q = 0; q < N; q += Piece<W>::n <= N ? Piece<W>::n : N) {
      constexpr int n = Piece<W>::n <= N ? Piece<W>::n : N;
      typedef W vec __attribute__((ext_vector_type(n)));
      typedef vec any __attribute__((aligned(sizeof(W))));
      const vec v = *reinterpret_cast<const any*>(p + c + q);
#pragma unroll
      for (int e = 0; e < n; ++e) f[q + e] = (float)v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = c + e < cols ? (float)p[c + e] : 0.f;
  }
}

// f(0), f(1), ..., as integral constants: an unrolled loop whose indexes stay constants.
template <class F, int... Q>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, Q...>) {
  (f(std::integral_constant<int, Q>{}), ...);
}

// Between LDS writes of some lanes of a wave and reads of them by others: the wave's LDS
// operations run in order, this keeps the compiler to it.  Costs no instruction.
__device__ __forceinline__ void lanes_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Sum over the aligned group of T lanes (a power of two up to 64) that holds this lane.
template <int T>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int off = T / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Sums of a (and b) over the T threads of a row: T up to 64 lanes, or the whole
// workgroup of T threads through LDS.  Two areas of `red` in turn, so that one
// barrier a sum is enough: area i is written again only behind the barrier of
// the sum in between, which every thread reaches after its reads of area i.
template <int T>
struct RowSum {
  float2 (*red)[16];
  int turn = 0;
  __device__ __forceinline__ float2 sum(float a, float b) {
    a = lanes_sum<(T < 64 ? T : 64)>(a);
    b = lanes_sum<(T < 64 ? T : 64)>(b);
    if constexpr (T > 64) {
      if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = make_float2(a, b);
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < T / 64; ++w) {
        const float2 r = red[turn][w];
        a += r.x;
        b += r.y;
      }
      turn ^= 1;
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float sum(float a) {
    a = lanes_sum<(T < 64 ? T : 64)>(a);
    if constexpr (T > 64) {
      if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6].x = a;
      __syncthreads();
      a = 0.f;
#pragma unroll
      for (int w = 0; w < T / 64; ++w) a += red[turn][w].x;
      turn ^= 1;
    }
    return a;
  }
};

// Grids of any number of workgroups: along one axis their threads have to stay below 2^32
// (a launch of more runs what is left of that, without an error), so that from 2^20
// workgroups on they go on along the second.
constexpr int64_t kGridX = 1 << 20;
inline dim3 grid_of(int64_t blocks) {
  return dim3((unsigned)(blocks < kGridX ? blocks : kGridX), (unsigned)((blocks + kGridX - 1) / kGridX));
}
__device__ __forceinline__ int64_t grid_block() { return (int64_t)blockIdx.y * kGridX + blockIdx.x; }

// Column c of n rows of `pitch` floats, added in order by a workgroup of 1024: each
// wave every 16th row, eight of them in flight, then the waves in order.  The result
// is the first wave's (0 past the last column).
__device__ __forceinline__ float partial_rows_sum(const float* part, int n, int64_t pitch, int64_t c,
                                                  float (&sum)[16][64]) {
  constexpr int kAhead = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float a[kAhead] = {};
  if (c < pitch) {
    int k = wave;
    for (; k + 16 * (kAhead - 1) < n; k += 16 * kAhead)
#pragma unroll
      for (int u = 0; u < kAhead; ++u) a[u] += part[(k + 16 * u) * pitch + c];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (k + 16 * u < n) a[u] += part[(k + 16 * u) * pitch + c];
  }
  sum[wave][lane] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  __syncthreads();
  float s = 0.f;
  if (wave == 0)
#pragma unroll
    for (int w = 0; w < 16; ++w) s += sum[w][lane];
  return s;
}

}  // namespace
