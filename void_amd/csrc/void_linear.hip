// void_linear.hip — the dense layer with its epilogue, forward and backward,
// for gfx950, declared in include/void_amd.h:
//
//   Z = X W^T + b,  Y = act(Z) + R;   dZ = dY act'(Z),  dX = dZ W,  dW = dZ^T X,
//   db = sum_rows dZ.
//
// All three products are C[i][j] = sum_r A(i, r) B(j, r) with each operand
// stored along r ("plain": X, W in the forward pass, dZ in dX) or along i / j
// ("turned": W in dX; dZ and X in dW).  Products run on the matrix cores (exact
// products, fp32 sums).  Bound by them from some hundred tokens on, by reading W for
// few tokens.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "lds_dma.h"
#include "rows.h"
#include "void_amd.h"

extern "C" __attribute__((visibility("hidden"))) int void_internal_fail(int code, const char* msg);

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4h __attribute__((ext_vector_type(4)));
typedef short v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));

// ---- epilogue --------------------------------------------------------------

// act'(Z), kept for the backward pass: fp32 for fp32 values, else a 16-bit code.  s lies
// in [-0.13, 1.13] for every activation.  From 2^-5 on |s| is fixed point in steps of 2^-15
// (within 2^-16; 1 is exact), which takes 37000 codes of the positive side and 3200 of the
// negative; the others hold |s| from 2^-29 to 2^-5 with 9 bits behind its leading one
// (within 2^-10 of itself), so that saturated units, whose slopes are small, keep their
// gradients; below that it is 0.  Beside dZ's rounding (2^-8 of itself for bf16, 2^-11 for
// fp16) that is a quarter at most for bf16, and for fp16 a thirtieth near 1, as much at 2^-5
// and twice as much below.  NaN becomes 0, which no slope takes.  Packing costs 1.3 % of a
// training step of 8192 x 14336 x 4096 with GELU against fixed point alone, which rounds
// slopes below 2^-16 to 0 (2605 us and 2570).
template <class E>
struct Slope {
  typedef uint16_t type;
  static constexpr uint32_t kLow = 0x31000000;  // 2^-29
  static __device__ __forceinline__ uint16_t pack(float s) {
    const float a = fabsf(s);
    const uint32_t code = (max(__float_as_uint(a), kLow) - kLow + (1 << 13)) >> 14;  // 0 .. 12288 below 2^-5
    const float m = a < 0x1p-5f ? (float)code : fmaf(a, 32768.f, 11264.f);
    return (uint16_t)__float2uint_rz(16384.5f + copysignf(m, s));
  }
  static __device__ __forceinline__ float unpack(uint16_t u) {
    const int w = (int)u - 16384;
    const uint32_t m = (uint32_t)abs(w);
    const float small = m ? __uint_as_float((m << 14) + kLow) : 0.f;
    const float a = m < 12288 ? small : (float)((int)m - 11264) * 0x1p-15f;
    return u ? (w < 0 ? -a : a) : __builtin_nanf("");
  }
};
template <>
struct Slope<float> {
  typedef float type;
  static __device__ __forceinline__ float pack(float s) { return s; }
  static __device__ __forceinline__ float unpack(float s) { return s; }
};

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.442695040888963f));
}

// z <- activation(z) and, where `want` is set, slope <- activation'(z).  GELU is
// its tanh form z sigmoid(2 u), u = 0.7978845608 (z + 0.044715 z^3).  The slope's
// z^2 is kept finite: it stands beside s (1 - s), which is 0 there.
__device__ __forceinline__ void activate(float& z, float& slope, int act, bool want) {
  if (act == VOID_ACT_RELU) {
    slope = z > 0.f ? 1.f : 0.f;
    z = z < 0.f ? 0.f : z;
  } else if (act == VOID_ACT_GELU) {
    // sigmoid(2 u) = 1 / (1 + 2^-(2 log2(e) u)); 2 du/dz = 1.5957691 + 0.2140644 z^2.
    const float z2 = z * z;
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * fmaf(z2, -0.10294324f, -2.30220819f)));
    const float y = z * s;
    if (want) slope = fmaf(y * (1.f - s), fmaf(fminf(z2, 1e4f), 0.21406442f, 1.5957691216f), s);
    z = y;
  } else if (act == VOID_ACT_SILU) {
    const float s = sigmoid(z);
    if (want) slope = fmaf(z * s, 1.f - s, s);
    z *= s;
  }
}

struct Epilogue {
  void* out;             // [M, N] of E
  int64_t ldo;
  const void* bias;      // [N], or null
  const void* residual;  // [M, N] of E, or null
  int64_t ldr;
  void* slope;           // [M, N] of Slope<E>, or null
  int bias_f32, act;
};

template <class E>
__device__ __forceinline__ float bias_at(const Epilogue& p, int64_t n) {
  if (!p.bias) return 0.f;
  return p.bias_f32 ? static_cast<const float*>(p.bias)[n] : (float)static_cast<const E*>(p.bias)[n];
}

template <class E>
__device__ __forceinline__ void finish(const Epilogue& p, float sum, float bias, int64_t m, int64_t n, int64_t N) {
  float y = sum + bias, slope = 0.f;
  activate(y, slope, p.act, p.slope != nullptr);
  if (p.slope) static_cast<typename Slope<E>::type*>(p.slope)[m * N + n] = Slope<E>::pack(slope);
  if (p.residual) y += (float)static_cast<const E*>(p.residual)[m * p.ldr + n];
  static_cast<E*>(p.out)[m * p.ldo + n] = (E)y;
}

// The same for a piece of n values of a row from column c on; `res` is the
// residual's piece.
template <class E>
__device__ __forceinline__ void finish_piece(const Epilogue& p, typename Piece<E>::fvec z, const float (&bias)[Piece<E>::n],
                                             typename Piece<E>::vec res, int64_t m, int c, int N) {
  constexpr int n = Piece<E>::n;
  typedef typename Piece<E>::fvec F;
  typedef typename Slope<E>::type S;
  typedef S SV __attribute__((ext_vector_type(16 / sizeof(E))));
  typedef SV SAny __attribute__((aligned(sizeof(S))));
#pragma unroll
  for (int e = 0; e < n; ++e) z[e] += bias[e];
  if (p.act != VOID_ACT_NONE) {
    F slope = 0.f;
    auto all = [&](int act, bool want) {
#pragma unroll
      for (int e = 0; e < n; ++e) {
        float y = z[e], d = 0.f;
        activate(y, d, act, want);
        z[e] = y, slope[e] = d;
      }
    };
    if (p.act == VOID_ACT_RELU) all(VOID_ACT_RELU, true);
    else if (p.act == VOID_ACT_GELU) all(VOID_ACT_GELU, true);
    else all(VOID_ACT_SILU, true);
    if (p.slope) {
      S* sr = static_cast<S*>(p.slope) + m * N + c;
      SV v;
#pragma unroll
      for (int e = 0; e < n; ++e) v[e] = Slope<E>::pack(slope[e]);
      if (c + n <= N) {
        *reinterpret_cast<SAny*>(sr) = v;
      } else {
#pragma unroll
        for (int e = 0; e < n; ++e)
          if (c + e < N) sr[e] = v[e];
      }
    }
  }
  if (p.residual) z += __builtin_convertvector(res, F);
  store_piece(static_cast<E*>(p.out) + m * p.ldo, c, N, __builtin_convertvector(z, typename Piece<E>::vec));
}

template <class E>
__device__ __forceinline__ typename Piece<E>::vec residual_piece(const Epilogue& p, int64_t m, int c, int N) {
  if (!p.residual) return typename Piece<E>::vec{};
  return load_piece(static_cast<const E*>(p.residual) + m * p.ldr, c, N);
}

template <class E>
__device__ __forceinline__ void bias_piece(const Epilogue& p, int c, int N, float (&f)[Piece<E>::n]) {
  if (p.bias_f32) load_params(f, static_cast<const float*>(p.bias), c, N, 0.f);
  else load_params(f, static_cast<const E*>(p.bias), c, N, 0.f);
}

// ---- the tiled product -----------------------------------------------------

struct Product {
  const void* a;  // plain: [M, K] rows lda apart; turned: [K, M]
  const void* b;  // plain: [N, K]; turned: [K, N]
  int64_t lda, ldb;
  int64_t M, N, K;
  int tiles_m, tiles_n, splits, steps_per_split;
  float* part;  // splits > 1: [splits][M][N] fp32 sums instead of the epilogue
  Epilogue epi;
};

__device__ __forceinline__ v16f mfma(v4i a, v4i b, v16f c, __bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma(v4i a, v4i b, v16f c, _Float16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8hf, a), __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
}

__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8hf, a), __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
}

// One operand's B rows (of the tile) x 128 bytes along r, in LDS.
//
// Plain: row i at 128 i, its 16-byte chunks permuted by c ^ (i & 7), so that the
// rows of a fragment read hit different banks.  Turned: row r of B values, its
// chunks permuted by c ^ swizzle(r), which keeps the 64 bytes that a transposing read
// takes of each of 4 rows in different banks.  The LDS-DMA writes lane after lane, so
// the permutation is in what each lane loads.
template <class E, int B, int NW, bool TURNED>
struct Operand {
  static constexpr int kPer = 16 / (int)sizeof(E), kBK = 128 / (int)sizeof(E), kLoads = B * 128 / (NW * 1024);
  static constexpr int kCpr = B * (int)sizeof(E) / 16;  // chunks of a turned row

  // Of a turned row; only r & 3 counts.
  static __device__ __forceinline__ constexpr int swizzle(int r) {
    return kCpr >= 16 ? (r & 3) << 2 : kCpr == 8 ? (r & 2) << 1 : 0;
  }

  // From load to load a wave's rows go on by kRows, which leaves the permutation as it is.
  static constexpr int kRows = TURNED ? NW * 64 / kCpr : NW * 8;
  static_assert(kRows % (TURNED ? 4 : 8) == 0);

  const uint8_t* base;  // of the next step's first row / column
  int64_t step;         // bytes from step to step
  int voff[kLoads];
  int at;               // r of load 0's chunk within a step; turned: kRows more for each next

  // I - i0 rows (turned: columns) remain from i0 on.  Offsets to the rows that there are fit
  // 31 bits (checked by the host); those past them may wrap and are not used.
  __device__ __forceinline__ void init(const void* p, int64_t ld, int64_t i0, int64_t I, int64_t r0, int wave,
                                       int lane) {
    const int id = wave * 64 + lane;
    const uint32_t pitch = (uint32_t)ld * (uint32_t)sizeof(E);
    const int rows = (int)std::min<int64_t>(I - i0, B);
    if constexpr (!TURNED) {
      base = static_cast<const uint8_t*>(p) + (i0 * ld + r0) * (int64_t)sizeof(E);
      step = 128;
      const int row = id >> 3, c = (id & 7) ^ (row & 7);
      const uint32_t first = row * pitch + 16 * c;
#pragma unroll
      for (int q = 0; q < kLoads; ++q) voff[q] = row + q * kRows < rows ? (int)(first + q * kRows * pitch) : kOutOfRange;
      at = c * kPer;
    } else {
      base = static_cast<const uint8_t*>(p) + (r0 * ld + i0) * (int64_t)sizeof(E);
      step = ld * 128;
      const int row = id / kCpr, c = (id % kCpr) ^ swizzle(row);
      const uint32_t first = row * pitch + 16 * c;
#pragma unroll
      for (int q = 0; q < kLoads; ++q) voff[q] = c * kPer < rows ? (int)(first + q * kRows * pitch) : kOutOfRange;
      at = row;
    }
  }

  // Load Q of the next step into LDS, the last of them stepping on; `left` values
  // of r remain from it on.
  template <int Q>
  __device__ __forceinline__ void load_one(uint8_t* lds, int wave, int left) {
    dma_b128(sgpr_rsrc(base), lds + (Q * NW + wave) * 1024, at + (TURNED ? Q * kRows : 0) < left ? voff[Q] : kOutOfRange, 0);
    if (Q == kLoads - 1) base += step;
  }
  template <int... Q>
  __device__ __forceinline__ void load_all(std::integer_sequence<int, Q...>, uint8_t* lds, int wave, int left) {
    (load_one<Q>(lds, wave, left), ...);
  }
  __device__ __forceinline__ void load(uint8_t* lds, int wave, int left) {
    load_all(std::make_integer_sequence<int, kLoads>{}, lds, wave, left);
  }

  // Half kk (32 of r) of a plain operand's rows i0 .. i0 + 15 for the 16 x 16 x 32
  // instructions: lane (i, g) holds r = 8 g .. 8 g + 7 of row i.  16-bit values.
  static __device__ __forceinline__ v4i fragment16(const uint8_t* lds, int i0, int kk, int lane) {
    static_assert(!TURNED && sizeof(E) == 2);
    const int i = lane & 15, g = lane >> 4;
    return *reinterpret_cast<const v4i*>(lds + (i0 + i) * 128 + (((4 * kk + g) ^ (i & 7)) << 4));
  }

  // Chunk pair kk's fragment of rows i0 .. i0 + 31: 16 bytes along r a lane.
  static __device__ __forceinline__ v4i fragment(const uint8_t* lds, int i0, int kk, int lane) {
    const int j = lane & 31, g = lane >> 5;
    if constexpr (!TURNED) {
      return *reinterpret_cast<const v4i*>(lds + (i0 + j) * 128 + (((2 * kk + g) ^ (j & 7)) << 4));
    } else if constexpr (sizeof(E) == 4) {
      v4f f;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        f[s] = *reinterpret_cast<const float*>(lds + (8 * kk + 4 * g + s) * (B * 4) +
                                               ((((i0 + j) >> 2) ^ swizzle(s)) << 4) + (j & 3) * 4);
      return __builtin_bit_cast(v4i, f);
    } else {
      // Two ds_read_b64_tr_b16: the 16 lanes of a read fetch 4 rows x 16 columns,
      // 8 bytes each in row-major order, and lane t gets column t.
      const int i = j & 15;
      v4h t[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 16 * kk + 8 * g + 4 * r + (i >> 2);
        const int c = (i0 >> 3) + 2 * (j >> 4) + ((i & 3) >> 1);
        const uint8_t* p = lds + row * (B * 2) + ((c ^ swizzle(i >> 2)) << 4) + 8 * (i & 1);
        t[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4h*)(const_cast<uint8_t*>(p)));
      }
      return __builtin_bit_cast(v4i, v8h{t[0][0], t[0][1], t[0][2], t[0][3], t[1][0], t[1][1], t[1][2], t[1][3]});
    }
  }
};

// Which tile and split of the grid a workgroup takes.  Workgroups are dealt to the
// 8 XCDs in turn: each XCD gets a run of neighbouring tiles, whose operands its L2
// then holds.
template <int BM, int BN>
struct Place {
  int64_t m0, n0, r0, left;  // first row and column, first r and how many of them
  int split;
  __device__ __forceinline__ Place(const Product& p, int bk) {
    const int n = gridDim.x, x = blockIdx.x & 7, q = n >> 3;
    int t = x * q + min(x, n & 7) + (blockIdx.x >> 3);
    const int tiles = p.tiles_m * p.tiles_n;
    split = t / tiles;
    t -= split * tiles;
    constexpr int kGroup = 4;
    const int group = t / (kGroup * p.tiles_n), first = group * kGroup, size = min(kGroup, p.tiles_m - first);
    const int in = t - group * kGroup * p.tiles_n;
    m0 = (int64_t)(first + in % size) * BM;
    n0 = (int64_t)(in / size) * BN;
    r0 = (int64_t)split * p.steps_per_split * bk;
    left = std::min<int64_t>(p.K - r0, (int64_t)p.steps_per_split * bk);
  }
};

// ROWS rows x COLS columns of sums from the wave's strip in LDS: whole pieces of
// rows through the epilogue (or to the partial sums), four of them in flight.
template <class E, int COLS, int ROWS, int PITCH = COLS>
__device__ __forceinline__ void store_strip(const Product& p, int split, const float* strip, int64_t row0, int64_t col0,
                                            int lane) {
  lanes_in_order();  // the strip is other lanes' writing
  constexpr int n = Piece<E>::n, kLanes = COLS / n, kRows = 64 / kLanes, kAhead = ROWS / kRows < 4 ? ROWS / kRows : 4;
  static_assert(ROWS % (kAhead * kRows) == 0);
  typedef typename Piece<E>::fvec F;
  const int c = lane % kLanes * n, N = (int)p.N, col = (int)col0 + c;
  if (col >= N) return;
  float bias[n];
  bias_piece<E>(p.epi, col, N, bias);
  strip += lane / kLanes * PITCH + c;
  row0 += lane / kLanes;
#pragma unroll 1
  for (int q = 0; q < ROWS; q += kAhead * kRows) {
    F z[kAhead];
    typename Piece<E>::vec res[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      z[u] = *reinterpret_cast<const F*>(strip + (q + u * kRows) * PITCH);
      if (row0 + q + u * kRows < p.M) res[u] = residual_piece<E>(p.epi, row0 + q + u * kRows, col, N);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t row = row0 + q + u * kRows;
      if (row >= p.M) continue;
      if (p.part) {
        float* d = p.part + ((int64_t)split * p.M + row) * N;
#pragma unroll
        for (int e = 0; e < n; e += 4)
          if (col + e < N)
            store_piece<float>(d, col + e, N, Piece<float>::vec{z[u][e], z[u][e + 1], z[u][e + 2], z[u][e + 3]});
      } else {
        finish_piece<E>(p.epi, z[u], bias, res[u], row, col, N);
      }
    }
  }
}

// A 32 x 32 block of sums into a strip: lane (j, g) holds column j and rows
// (r & 3) + 8 (r >> 2) + 4 g.
template <int COLS>
__device__ __forceinline__ void to_strip(float* strip, int col, v16f acc, int lane) {
#pragma unroll
  for (int r = 0; r < 16; ++r) strip[((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * COLS + col + (lane & 31)] = acc[r];
}

// BM x 128 tiles, 4 waves, two workgroups a CU.  BM = 128: waves of 64 x 64, two
// steps in LDS.  BM = 64 and 32, for few rows: waves of BM x 32, three and four steps,
// since there the operand that streams past is what bounds it, and bytes in flight
// what that asks for.  fp32 runs at 137 TFLOP/s in its loop (the instructions' peak is
// 157): 730 x 5003 x 3001 199 us, 110 TFLOP/s with the tiles' ends.  32 tokens x 14336 x
// 4096 bf16 29 us, 4.0 TB/s of W; 16 tokens of the same fp32 44 us, 5.4 TB/s.  4096 x 4096 bf16:
// 128 tokens 21 us, 512 30, 1024 53 in whole calls, of which a join takes 4 to 8.
template <class E, int BM, bool TA, bool TB>
__global__ __launch_bounds__(256, 2) void product_kernel(Product p) {
  constexpr int BN = 128, NW = 4, kBK = 128 / (int)sizeof(E), kStages = BM == 128 ? 2 : BM == 64 ? 3 : 4;
  constexpr int RA = BM == 128 ? 2 : BM / 32, RB = BM == 128 ? 2 : 1;
  typedef Operand<E, BM, NW, TA> OpA;
  typedef Operand<E, BN, NW, TB> OpB;
  constexpr int kLoads = OpA::kLoads + OpB::kLoads;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kStages][(BM + BN) * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<BM, BN> at(p, kBK);
  const int steps = (int)((at.left + kBK - 1) / kBK);
  OpA a;
  OpB b;
  a.init(p.a, p.lda, at.m0, p.M, at.r0, wave, lane);
  b.init(p.b, p.ldb, at.n0, p.N, at.r0, wave, lane);
  const int wm = BM == 128 ? (wave >> 1) * 64 : 0, wn = BM == 128 ? (wave & 1) * 64 : wave * 32;
  v16f acc[RA][RB];
#pragma unroll
  for (int i = 0; i < RA; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j) acc[i][j] = 0.f;
  // Past the last step nothing is left of r: such loads bring zeros and ask for no
  // memory, and the waits can count.
  auto load = [&](int s, int slot) {
    const int l = (int)std::max<int64_t>(0, std::min<int64_t>(at.left - (int64_t)s * kBK, kBK));
    a.load(&lds[slot][0], wave, l);
    b.load(&lds[slot][BM * 128], wave, l);
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(s, s);
  int slot = 0, free = kStages - 1;
  for (int s = 0; s < steps; ++s) {
    wait_vm<(kStages - 2) * kLoads>();
    __syncthreads();  // step s has landed everywhere, step s - 1 is read
    load(s + kStages - 1, free);
    const uint8_t *la = &lds[slot][0], *lb = &lds[slot][BM * 128];
    free = slot;
    slot = slot + 1 == kStages ? 0 : slot + 1;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      v4i fa[RA], fb[RB];
#pragma unroll
      for (int i = 0; i < RA; ++i) fa[i] = OpA::fragment(la, wm + 32 * i, kk, lane);
#pragma unroll
      for (int j = 0; j < RB; ++j) fb[j] = OpB::fragment(lb, wn + 32 * j, kk, lane);
      // fp32: one of the chunk's four values at a time, so that products in a row are
      // of different sums.
#pragma unroll
      for (int u = 0; u < (sizeof(E) == 4 ? 4 : 1); ++u)
#pragma unroll
        for (int i = 0; i < RA; ++i)
#pragma unroll
          for (int j = 0; j < RB; ++j)
            if constexpr (sizeof(E) == 4)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(v4f, fa[i])[u],
                                                               __builtin_bit_cast(v4f, fb[j])[u], acc[i][j], 0, 0, 0);
            else
              acc[i][j] = mfma(fa[i], fb[j], acc[i][j], E{});
    }
  }
  wait_vm<0>();     // loads past the last step still write zeros
  __syncthreads();  // and the last step is read
  constexpr int kRows = 32 * RA, kCols = 32 * RB;
  float* strip = reinterpret_cast<float*>(&lds[0][0]) + wave * kRows * kCols;
#pragma unroll
  for (int i = 0; i < RA; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j) to_strip<kCols>(strip + i * 32 * kCols, 32 * j, acc[i][j], lane);
  store_strip<E, kCols, kRows>(p, at.split, strip, at.m0 + wm, at.n0 + wn, lane);
}

template <class F>
__device__ __forceinline__ void each8(F f) {
  each_of(f, std::make_integer_sequence<int, 8>{});
}

// 256 x 256 tiles of 16-bit operands, 4 waves of 128 x 128, one workgroup a CU: the
// fewest LDS bytes a product (a wave's fragments serve 16 matrix instructions from 8
// reads), with 256 accumulators a lane.
//
// A step (64 of r) is four fragment sets; each set is read while the matrix cores
// work on the one before it, across the steps too: the one barrier of a step stands
// before its last set, when all of the step has been read and the next step has
// landed.  LDS holds three steps of A and two of B (all 160 KB): the loads of a step
// are spread over the sets, four each, so that no wave waits to issue them, and the
// waits count those of A for the step after next, which stay in flight.  8192 x 4096 x 14336
// bf16 (dX) 717 to 790 us, 1220 to 1340 TFLOP/s; 14336 x 4096 x 8192 (dW, both turned) 780 to
// 810 us.  The matrix cores are busy 70 % (dX) and 59 % (dW) of the cycles, at 1.8 to 2.0 GHz
// with random operands: power takes the rest of the 2.4 GHz at which equal values run.
template <class E, bool TA, bool TB>
__global__ __launch_bounds__(256, 1) void wide_product_kernel(Product p) {
  constexpr int B = 256, NW = 4, kBK = 64, R = 4, kOperand = B * 128;
  typedef Operand<E, B, NW, TA> OpA;
  typedef Operand<E, B, NW, TB> OpB;
  static_assert(OpA::kLoads == 8 && OpB::kLoads == 8);
  __shared__ __attribute__((aligned(1024))) uint8_t lds[5][kOperand];  // A: 0 1 2, B: 3 4
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<B, B> at(p, kBK);
  const int steps = (int)((at.left + kBK - 1) / kBK);
  OpA a;
  OpB b;
  a.init(p.a, p.lda, at.m0, p.M, at.r0, wave, lane);
  b.init(p.b, p.ldb, at.n0, p.N, at.r0, wave, lane);
  const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;
  v16f acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = 0.f;
  // What is left of r at step s; past the last step nothing: such loads bring zeros
  // and ask for no memory.
  auto left = [&](int s) { return (int)std::max<int64_t>(0, std::min<int64_t>(at.left - (int64_t)s * kBK, kBK)); };
  v4i fa[2][R], fb[2][R];
  // Where A of this step, the next and the one after next are, and B of this and the next.
  const uint8_t *a0 = lds[0], *a1 = lds[1], *a2 = lds[2], *b0 = lds[3], *b1 = lds[4];
  // Set kk's products, two at a time behind one of the next set's eight reads and,
  // every second time, one of the phase's four loads.  The reads come in the order in
  // which the next set's products take them.
  auto phase = [&](auto kk_, const uint8_t* ra, const uint8_t* rb, auto load) {
    constexpr int kk = decltype(kk_)::value, next = (kk + 1) & 3, set = kk & 1, to = next & 1;
    auto two = [&](auto q_) {
      constexpr int q = decltype(q_)::value, i = q >> 1, j = (q & 1) * 2;
      if constexpr (q == 0) fb[to][0] = OpB::fragment(rb, wn, next, lane);
      else if constexpr (q == 1) fa[to][0] = OpA::fragment(ra, wm, next, lane);
      else if constexpr (q <= 4) fb[to][q - 1] = OpB::fragment(rb, wn + 32 * (q - 1), next, lane);
      else fa[to][q - 4] = OpA::fragment(ra, wm + 32 * (q - 4), next, lane);
      load(q_);
      acc[i][j] = mfma(fa[set][i], fb[set][j], acc[i][j], E{});
      acc[i][j + 1] = mfma(fa[set][i], fb[set][j + 1], acc[i][j + 1], E{});
      __builtin_amdgcn_sched_barrier(0);
    };
    each8(two);
  };
  a.load(const_cast<uint8_t*>(a0), wave, left(0));
  b.load(const_cast<uint8_t*>(b0), wave, left(0));
  a.load(const_cast<uint8_t*>(a1), wave, left(1));
  b.load(const_cast<uint8_t*>(b1), wave, left(1));
  wait_vm<16>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    fb[0][i] = OpB::fragment(b0, wn + 32 * i, 0, lane);
    fa[0][i] = OpA::fragment(a0, wm + 32 * i, 0, lane);
  }
  for (int s = 0; s < steps; ++s) {
    const int l2 = left(s + 2);
    phase(std::integral_constant<int, 0>{}, a0, b0, [&](auto q) {
      if constexpr (q.value % 2 == 0) a.template load_one<q.value / 2>(const_cast<uint8_t*>(a2), wave, l2);
    });
    phase(std::integral_constant<int, 1>{}, a0, b0, [&](auto q) {
      if constexpr (q.value % 2 == 0) a.template load_one<4 + q.value / 2>(const_cast<uint8_t*>(a2), wave, l2);
    });
    phase(std::integral_constant<int, 2>{}, a0, b0, [](auto) {});
    wait_vm<8>();     // A of step s + 2 stays in flight
    __syncthreads();  // step s is read, step s + 1 has landed
    phase(std::integral_constant<int, 3>{}, a1, b1,
          [&](auto q) { b.template load_one<q.value>(const_cast<uint8_t*>(b0), wave, l2); });
    const uint8_t *a3 = a0, *b2 = b0;
    a0 = a1, a1 = a2, a2 = a3;
    b0 = b1, b1 = b2;
  }
  wait_vm<0>();     // loads past the last step still write zeros
  __syncthreads();
  float* strip = reinterpret_cast<float*>(&lds[0][0]) + wave * 64 * 128;
  each_of(
      [&](auto h_) {
        constexpr int h = 2 * decltype(h_)::value;
        lanes_in_order();  // the strip is read
#pragma unroll
        for (int j = 0; j < R; ++j) {
          to_strip<128>(strip, 32 * j, acc[h][j], lane);
          to_strip<128>(strip + 32 * 128, 32 * j, acc[h + 1][j], lane);
        }
        store_strip<E, 128, 64>(p, at.split, strip, at.m0 + wm + 32 * h, at.n0 + wn, lane);
      },
      std::make_integer_sequence<int, 2>{});
}

// The same for two plain operands on the 16 x 16 x 32 instructions, whose sums cost
// the matrix cores less energy (they take half as many steps along r): 8192 x 14336 x 4096
// bf16 725 us, 1327 TFLOP/s, against 773; the matrix cores are busy 66 % of the cycles at
// 2.0 GHz, which power sets.  (Turned operands' fragments leave too few registers for it.)  A step is two
// fragment sets and takes 1.37 us; a tile's start and end take 12 to 16 us, with GELU and
// its slope 10 more, which one wave a SIMD spends on them alone.
template <class E>
__global__ __launch_bounds__(256, 1) void wide_plain_kernel(Product p) {
  constexpr int B = 256, NW = 4, kBK = 64, R = 8, kOperand = B * 128;
  typedef Operand<E, B, NW, false> OpA;
  typedef OpA OpB;
  static_assert(OpA::kLoads == 8 && OpB::kLoads == 8);
  __shared__ __attribute__((aligned(1024))) uint8_t lds[5][kOperand];  // A: 0 1 2, B: 3 4
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<B, B> at(p, kBK);
  const int steps = (int)((at.left + kBK - 1) / kBK);
  OpA a;
  OpB b;
  a.init(p.a, p.lda, at.m0, p.M, at.r0, wave, lane);
  b.init(p.b, p.ldb, at.n0, p.N, at.r0, wave, lane);
  const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;
  v4f acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = 0.f;
  // What is left of r at step s; past the last step nothing: such loads bring zeros
  // and ask for no memory.
  auto left = [&](int s) { return (int)std::max<int64_t>(0, std::min<int64_t>(at.left - (int64_t)s * kBK, kBK)); };
  v4i fa[2][R], fb[2][R];
  // Where A of this step, the next and the one after next are, and B of this and the next.
  const uint8_t *a0 = lds[0], *a1 = lds[1], *a2 = lds[2], *b0 = lds[3], *b1 = lds[4];
  // Set kk's products, four at a time behind one of the other set's sixteen reads and,
  // every second time, one of the phase's eight loads.  The reads come in the order in
  // which the next products take them.
  auto phase = [&](auto kk_, const uint8_t* ra, const uint8_t* rb, auto load) {
    constexpr int set = decltype(kk_)::value, to = set ^ 1;
    auto four = [&](auto q_) {
      constexpr int q = decltype(q_)::value, i = q >> 1, j = (q & 1) * 4;
      if constexpr (q == 0) fb[to][0] = OpB::fragment16(rb, wn, to, lane);
      else if constexpr (q == 1) fa[to][0] = OpA::fragment16(ra, wm, to, lane);
      else if constexpr (q <= 8) fb[to][q - 1] = OpB::fragment16(rb, wn + 16 * (q - 1), to, lane);
      else fa[to][q - 8] = OpA::fragment16(ra, wm + 16 * (q - 8), to, lane);
      if constexpr (q % 2 == 0) load(std::integral_constant<int, q / 2>{});
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[i][j + u] = mfma16(fa[set][i], fb[set][j + u], acc[i][j + u], E{});
      __builtin_amdgcn_sched_barrier(0);
    };
    each_of(four, std::make_integer_sequence<int, 16>{});
  };
  a.load(const_cast<uint8_t*>(a0), wave, left(0));
  b.load(const_cast<uint8_t*>(b0), wave, left(0));
  a.load(const_cast<uint8_t*>(a1), wave, left(1));
  b.load(const_cast<uint8_t*>(b1), wave, left(1));
  wait_vm<16>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    fb[0][i] = OpB::fragment16(b0, wn + 16 * i, 0, lane);
    fa[0][i] = OpA::fragment16(a0, wm + 16 * i, 0, lane);
  }
  for (int s = 0; s < steps; ++s) {
    const int l2 = left(s + 2);
    phase(std::integral_constant<int, 0>{}, a0, b0,
          [&](auto q) { a.template load_one<q.value>(const_cast<uint8_t*>(a2), wave, l2); });
    wait_vm<8>();     // A of step s + 2 stays in flight
    __syncthreads();  // step s is read, step s + 1 has landed
    phase(std::integral_constant<int, 1>{}, a1, b1,
          [&](auto q) { b.template load_one<q.value>(const_cast<uint8_t*>(b0), wave, l2); });
    const uint8_t *a3 = a0, *b2 = b0;
    a0 = a1, a1 = a2, a2 = a3;
    b0 = b1, b1 = b2;
  }
  wait_vm<0>();     // loads past the last step still write zeros
  __syncthreads();
  // Rows 144 floats apart: the four rows of a store then lie in different banks.
  constexpr int kPitch = 144;
  float* strip = reinterpret_cast<float*>(&lds[0][0]) + wave * 64 * kPitch;
  each_of(
      [&](auto h_) {
        constexpr int h = 4 * decltype(h_)::value;
        lanes_in_order();  // the strip is read
        // Lane (j, g) holds column j and rows 4 g .. 4 g + 3 of each 16 x 16.
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < R; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              strip[(16 * i + 4 * (lane >> 4) + r) * kPitch + 16 * j + (lane & 15)] = acc[h + i][j][r];
        store_strip<E, 128, 64, kPitch>(p, at.split, strip, at.m0 + wm + 16 * h, at.n0 + wn, lane);
      },
      std::make_integer_sequence<int, 2>{});
}

// The splits' sums added in order, then the epilogue.  Bound by reading them: two
// splits of 2048 x 4096 17 us, 6.0 TB/s with the residual and y (partly in the caches).
template <class E>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits, int64_t M, int N,
                                                   Epilogue epi) {
  constexpr int n = Piece<E>::n;
  const int per_row = (N + n - 1) / n;
  const int64_t total = M * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / per_row;
    const int c = (int)(i - m * per_row) * n;
    typename Piece<E>::fvec z = 0.f;
    for (int k = 0; k < splits; ++k) {
      float f[n];
      load_params(f, part + ((int64_t)k * M + m) * N, c, N, 0.f);
#pragma unroll
      for (int e = 0; e < n; ++e) z[e] += f[e];
    }
    float bias[n];
    bias_piece<E>(epi, c, N, bias);
    finish_piece<E>(epi, z, bias, residual_piece<E>(epi, m, c, N), m, c, N);
  }
}

// ---- few tokens -------------------------------------------------------------

// Up to 16 MT tokens: bound by reading W once.  A workgroup of NW waves takes 16
// rows of W, each wave a share of K straight from memory into fragments (no LDS:
// nothing of W is used twice), any alignment; the waves' sums are added in order.
// One token x 14336 x 4096 bf16 25.6 us, 4.6 TB/s; fp32 43.8 us, 5.4 TB/s; 16 tokens x 4096 x
// 4096 fp32 18.5 us, 3.6 TB/s.
template <class E, int MT, int NW, bool ODD>
__global__ __launch_bounds__(64 * NW) void few_kernel(const E* __restrict__ x, int64_t ldx, const E* __restrict__ w,
                                                      int64_t ldw, int M, int64_t N, int K, Epilogue epi) {
  constexpr int kPer = Piece<E>::n, kStep = 4 * kPer;  // 64 bytes of a row: a chunk each for 4 lanes
  constexpr int kAhead = ODD && MT == 4 ? 2 : 4;  // as much as fits the registers
  typedef typename Piece<E>::vec V;
  __shared__ v4f sum[NW][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int64_t n0 = grid_block() * 16;  // the last groups of a grid of two axes may lie past N
  // Rows past the end repeat the last one; their sums are not stored.
  const E* wr = w + std::min<int64_t>(n0 + i, N - 1) * ldw + g * kPer;
  const E* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x + (int64_t)min(16 * t + i, M - 1) * ldx + g * kPer;
  v4f acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = 0.f;
  auto multiply = [&](V wv, V xv, v4f c) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[s], wv[s], c, 0, 0, 0);
      return c;
    } else if constexpr (std::is_same_v<E, __bf16>) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv, wv, c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(xv, wv, c, 0, 0, 0);
    }
  };
  // Whole steps: the waves take groups of kAhead in turn.
  const int steps = K / kStep, groups = steps / kAhead;
  for (int q = wave; q < groups; q += NW) {
    const int k0 = q * kAhead * kStep;
    Loaded<E, ODD> wv[kAhead], xv[kAhead][MT];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      wv[u].whole(wr + k0 + u * kStep);
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[u][t].whole(xr[t] + k0 + u * kStep);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const V w4 = wv[u].take(wr);
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = multiply(w4, xv[u][t].take(xr[t]), acc[t]);
    }
  }
  // The rest, a step a wave; past K both operands are zero.
  for (int q = groups * kAhead + wave; q * kStep < K; q += NW) {
    const int k0 = q * kStep;
    const V wv = load_piece(wr - g * kPer, k0 + g * kPer, K);
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = multiply(wv, load_piece(xr[t] - g * kPer, k0 + g * kPer, K), acc[t]);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sum[wave][t][lane] = acc[t];
  __syncthreads();
  // Lane (i, g) of a sum holds column n0 + i and tokens 4 g .. 4 g + 3.
  for (int q = threadIdx.x; q < MT * 64; q += 64 * NW) {
    const int t = q >> 6, l = q & 63;
    v4f s = sum[0][t][l];
#pragma unroll
    for (int v = 1; v < NW; ++v) s += sum[v][t][l];
    const int64_t n = n0 + (l & 15);
    if (n >= N) continue;
    const float bias = bias_at<E>(epi, n);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = 16 * t + 4 * (l >> 4) + r;
      if (m < M) finish<E>(epi, s[r], bias, m, n, N);
    }
  }
}

// ---- dZ and db ----------------------------------------------------------------

// dz = dy act'(z) (unless dz is null), zero from N to ldz's next whole piece, and
// this workgroup's column sums in part[blockIdx.y][N] (unless part is null).  64
// pieces of columns, 4 rows at a time.  Bound by the memory: 8192 x 14336 bf16 154 us,
// 4.6 TB/s of dy, the slope and dz.
template <class E, bool ODD>
__global__ __launch_bounds__(256) void slope_kernel(const E* __restrict__ dy, int64_t lddy,
                                                    const typename Slope<E>::type* __restrict__ slope, int64_t M, int N,
                                                    E* __restrict__ dz, int64_t ldz, float* __restrict__ part) {
  constexpr int n = Piece<E>::n;
  typedef typename Piece<E>::vec V;
  typedef typename Piece<E>::fvec F;
  typedef typename Slope<E>::type S;
  typedef S SV __attribute__((ext_vector_type(16 / sizeof(E))));
  __shared__ float sum[4][64 * n];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c64 = ((int64_t)blockIdx.x * 64 + lane) * n;
  F s = 0.f;
  if (c64 < N) {
    const int c = (int)c64;
    for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < M; row += (int64_t)gridDim.y * 4) {
      const E* dr = dy + row * lddy;
      const S* sr = slope + row * N;
      Loaded<E, ODD> v;
      Loaded<S, ODD> sv;
      v.load(dr, c, N);
      if (slope) sv.load(sr, c, N);
      F f = __builtin_convertvector(v.take(dr, c, N), F);
      if (slope) {
        const SV s4 = sv.take(sr, c, N);
#pragma unroll
        for (int e = 0; e < n; ++e) f[e] = c + e < N ? f[e] * Slope<E>::unpack(s4[e]) : 0.f;
        if (dz) *reinterpret_cast<V*>(dz + row * ldz + c) = __builtin_convertvector(f, V);
      }
      s += f;
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < n; ++e) sum[wave][lane * n + e] = s[e];
  __syncthreads();
  for (int j = threadIdx.x; j < 64 * n; j += 256) {
    const int64_t col = (int64_t)blockIdx.x * 64 * n + j;
    if (col < N) part[(int64_t)blockIdx.y * N + col] = (sum[0][j] + sum[1][j]) + (sum[2][j] + sum[3][j]);
  }
}

// db: the n partial rows added in order, 16 at a time (one a wave), and rounded once
// (74 rows of 14336: 4.8 us).
template <class W>
__global__ __launch_bounds__(1024) void bias_sum_kernel(const float* __restrict__ part, int n, int N, W* __restrict__ db) {
  __shared__ float sum[16][64];
  const int64_t c = grid_block() * 64 + (threadIdx.x & 63);
  const float s = partial_rows_sum(part, n, N, c, sum);
  if (threadIdx.x < 64 && c < N) db[c] = (W)s;
}

// ---- host ---------------------------------------------------------------------

constexpr int kCus = 256;

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VOID_OK : void_internal_fail(VOID_ERR_HIP, hipGetErrorString(e));
}

bool float_type(int32_t t) { return t == VOID_DT_F32 || t == VOID_DT_BF16 || t == VOID_DT_F16; }
int size_of(int32_t t) { return t == VOID_DT_F32 ? 4 : 2; }

template <class Go>
void by_type(int32_t dtype, Go go) {
  if (dtype == VOID_DT_F32) go(float{});
  else if (dtype == VOID_DT_BF16) go(__bf16{});
  else go(_Float16{});
}

// Tile rows (the columns are 128, or 256 for 256) and the K splits of a product.
struct Plan {
  int tile, splits, steps_per_split;
};

// The plan of least estimated time, in microseconds, of those with at most kMaxTiles
// workgroups (of 256 threads: below 2^32 along a grid's axis); tile 0 where there is none.
// A CU takes one 256-row tile at a time, or two of the others: `fixed` is a tile's start
// and epilogue, `alone` and `full` a step of 128 bytes along r where a CU has one tile and,
// per tile, where it has two; splits add a launch and their sums' traffic.  The figures are fitted to 400
// timings of 18 bf16 and 8 fp32 products (17 to 8192 rows, 512 to 14336 columns, depths
// of 512 to 14336; the estimates are within 15 %, but for products of several rounds of
// 256-row tiles, which the chip's power makes up to a fifth slower; the plans chosen are
// 1 to 2 % and 0.4 % slower than each product's best).
struct Cost {
  int tile;
  double fixed, alone, full, join, traffic;
};

constexpr Cost kCost16[] = {{256, 11.7, 1.17, 1.17, 3.0, 1.2},
                            {128, 3.7, 0.77, 0.55, 3.2, 1.0},
                            {64, 0.8, 0.45, 0.39, 4.9, 1.3},
                            {32, 1.9, 0.35, 0.29, 5.0, 0.85}};
constexpr Cost kCost32[] = {{128, 1.3, 2.07, 1.96, 4.8, 1.0}, {64, 1.0, 1.12, 1.03, 4.5, 1.15}, {32, 2.7, 0.65, 0.57, 3.0, 1.0}};

constexpr int64_t kMaxTiles = (1 << 24) - 1;

Plan plan_of(int64_t M, int64_t N, int64_t K, int esz) {
  const int64_t steps = std::max<int64_t>(1, (K * esz + 127) / 128);
  Plan best{};
  double least = 1e300;
  auto consider = [&](const Cost& c) {
    const int64_t width = c.tile == 256 ? 256 : 128;
    const int64_t tiles = ((M + c.tile - 1) / c.tile) * ((N + width - 1) / width);
    for (int splits = 1; splits <= 32 && splits <= steps; ++splits) {
      const int64_t per = (steps + splits - 1) / splits;
      if (tiles * splits > kMaxTiles || (splits > 1 && ((steps + per - 1) / per != splits || per < 4))) continue;
      const int64_t each = (tiles * splits + kCus - 1) / kCus;  // tiles of the fullest CU
      const double one = c.fixed + per * c.alone, two = c.fixed + per * std::max(c.alone, 2 * c.full);
      double cost = c.tile == 256 ? each * one : each / 2 * two + each % 2 * (one - 0.3 * c.fixed);
      if (splits > 1) cost += c.join + c.traffic * splits * M * N / 1e6;
      if (cost < least) {
        least = cost;
        best = Plan{c.tile, splits, (int)per};
      }
    }
  };
  if (esz == 4)
    for (const Cost& c : kCost32) consider(c);
  else
    for (const Cost& c : kCost16) consider(c);
  return best;
}

template <class E, bool TA, bool TB>
void product(Product p, const Plan& plan, hipStream_t stream) {
  // The rows that lda and ldb lie between: of a single one the pitch may be anything.
  if ((TA ? p.K : p.M) <= 1) p.lda = 0;
  if ((TB ? p.K : p.N) <= 1) p.ldb = 0;
  p.splits = plan.splits;
  p.steps_per_split = plan.steps_per_split;
  p.tiles_m = (int)((p.M + plan.tile - 1) / plan.tile);
  p.tiles_n = (int)((p.N + (plan.tile == 256 ? 255 : 127)) / (plan.tile == 256 ? 256 : 128));
  const dim3 grid((unsigned)((int64_t)p.tiles_m * p.tiles_n * plan.splits));
  if constexpr (sizeof(E) == 2)
    if (plan.tile == 256) {
      if constexpr (!TA && !TB) hipLaunchKernelGGL(wide_plain_kernel<E>, grid, dim3(256), 0, stream, p);
      else hipLaunchKernelGGL((wide_product_kernel<E, TA, TB>), grid, dim3(256), 0, stream, p);
    }
  if (plan.tile == 128) hipLaunchKernelGGL((product_kernel<E, 128, TA, TB>), grid, dim3(256), 0, stream, p);
  if (plan.tile == 64) hipLaunchKernelGGL((product_kernel<E, 64, TA, TB>), grid, dim3(256), 0, stream, p);
  if (plan.tile == 32) hipLaunchKernelGGL((product_kernel<E, 32, TA, TB>), grid, dim3(256), 0, stream, p);
  if (plan.splits > 1)
    hipLaunchKernelGGL(join_kernel<E>, dim3((unsigned)std::min<int64_t>((p.M * ((p.N * (int64_t)sizeof(E) + 15) / 16) + 255) / 256, kCus * 16)),
                       dim3(256), 0, stream, p.part, plan.splits, p.M, (int)p.N, p.epi);
}

template <class E>
void few(const void_linear_args* d, const Epilogue& epi, hipStream_t stream) {
  auto go = [&](auto mt, auto nw) {
    constexpr int MT = decltype(mt)::value, NW = decltype(nw)::value;
    by_parity<E>(d->x, d->ldx, d->w, d->ldw, std::max(d->M, d->N), [&](auto odd) {
      hipLaunchKernelGGL((few_kernel<E, MT, NW, decltype(odd)::value>), grid_of((d->N + 15) / 16), dim3(64 * NW), 0,
                         stream, static_cast<const E*>(d->x), d->ldx, static_cast<const E*>(d->w), d->ldw, (int)d->M,
                         d->N, (int)d->K, epi);
    });
  };
  auto waves = [&](auto mt) {
    if (d->N >= 8192) go(mt, std::integral_constant<int, 4>{});
    else go(mt, std::integral_constant<int, 16>{});
  };
  if (d->M <= 16) waves(std::integral_constant<int, 1>{});
  else if (d->M <= 32) waves(std::integral_constant<int, 2>{});
  else waves(std::integral_constant<int, 4>{});
}

// Up to 64 tokens take operands of any alignment, through few_kernel.  Where the
// operands allow the tiles, more than 16 tokens take them (few_kernel's waves read X
// again and again: 32 tokens x 14336 x 4096 bf16 52 us, tiles 29), and two to 16 where
// the weight is larger than 64 MiB (16 tokens of the same 36.7 us, tiles 27.6; x 4096 x
// 4096 12.9, and 16.9 with the tiles' second launch).
bool few_tokens(int64_t M) { return M <= 64; }
bool few_by_rows(int64_t M, int64_t N, int64_t K, int esz, bool whole) {
  return M == 1 || (M <= 16 && N * K * esz <= (int64_t)64 << 20) || (M <= 64 && !whole);
}

// Rows that the LDS-DMA reads in whole chunks: aligned, of whole chunks.
bool whole_chunks(const void* p, int64_t ld, int64_t cols, int esz) {
  return (uintptr_t)p % 16 == 0 && ld * esz % 16 == 0 && cols * esz % 16 == 0;
}

int check(const void_linear_args* d) {
  if (!d) return void_internal_fail(VOID_ERR_ARG, "null arguments");
  if (d->M < 0 || d->N < 0 || d->K < 0) return void_internal_fail(VOID_ERR_ARG, "negative size");
  if (d->N > INT_MAX / 2 || d->K > INT_MAX / 2 || d->M > INT_MAX)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "sizes are limited to 2^30 features and 2^31 rows");
  if (!float_type(d->dtype)) return void_internal_fail(VOID_ERR_UNSUPPORTED, "values are fp32, bf16 or fp16");
  return 1;
}

// Whether 31-bit offsets reach the rows that a step of a tile takes: 256 at most of a
// plain operand, a step's depth of a turned one.  A single row's pitch is not looked at.
bool within_reach(int64_t rows, int64_t ld, int esz, bool turned = false) {
  return rows <= 1 || std::min<int64_t>(rows, turned ? 128 / esz : 256) * ld * esz <= INT_MAX - 65536;
}

int64_t padded(int64_t cols, int esz) { return (cols * esz + 15) / 16 * 16 / esz; }

}  // namespace

extern "C" {

int32_t void_linear_any_alignment(int64_t M) { return few_tokens(M); }

size_t void_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int32_t dtype) {
  if (M <= 0 || N <= 0 || few_by_rows(M, N, K, size_of(dtype), true)) return 0;
  const Plan p = plan_of(M, N, K, size_of(dtype));
  return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0;
}

int void_linear(const void_linear_args* d, hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const int st = check(d);
  if (st <= 0) return st;
  if (d->M == 0 || d->N == 0) return VOID_OK;
  const int esz = size_of(d->dtype);
  if (!d->y || (d->K && (!d->x || !d->w))) return void_internal_fail(VOID_ERR_ARG, "null x, w or y");
  if (d->bias && d->bias_dtype != d->dtype && d->bias_dtype != VOID_DT_F32)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "the bias has the values' type, or fp32");
  if (d->activation < VOID_ACT_NONE || d->activation > VOID_ACT_SILU)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "unknown activation");
  if (d->slope && d->activation == VOID_ACT_NONE) return void_internal_fail(VOID_ERR_ARG, "slope without an activation");
  if ((d->M > 1 && (d->ldx < d->K || d->ldy < d->N || (d->residual && d->ldr < 0))) || (d->N > 1 && d->ldw < d->K))
    return void_internal_fail(VOID_ERR_ARG, "leading dimension too small");
  if (((uintptr_t)d->x | (uintptr_t)d->w | (uintptr_t)d->y | (uintptr_t)d->residual | (uintptr_t)d->slope) % esz ||
      (d->bias && (uintptr_t)d->bias % size_of(d->bias_dtype)))
    return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements");
  const Epilogue epi{d->y, d->ldy, d->bias, d->residual, d->ldr, d->slope, d->bias_dtype == VOID_DT_F32, d->activation};
  const bool whole = d->K == 0 || (whole_chunks(d->x, d->ldx, d->K, esz) && whole_chunks(d->w, d->ldw, d->K, esz));
  const bool near = d->K == 0 || (within_reach(d->M, d->ldx, esz) && within_reach(d->N, d->ldw, esz));
  if (few_by_rows(d->M, d->N, d->K, esz, whole && near)) {
    by_type(d->dtype, [&](auto e) { few<decltype(e)>(d, epi, stream); });
    return launched();
  }
  if (!whole)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "more than 64 tokens need rows of whole 16-byte chunks");
  if (!near) return void_internal_fail(VOID_ERR_UNSUPPORTED, "rows are too far apart");
  const Plan plan = plan_of(d->M, d->N, d->K, esz);
  if (!plan.tile) return void_internal_fail(VOID_ERR_UNSUPPORTED, "more tiles than a grid holds");
  if (plan.splits > 1 && (!d->workspace || (uintptr_t)d->workspace % 4 ||
                          d->workspace_bytes < (size_t)plan.splits * d->M * d->N * 4))
    return void_internal_fail(VOID_ERR_WORKSPACE, "linear: workspace missing or too small");
  by_type(d->dtype, [&](auto e) {
    product<decltype(e), false, false>(Product{d->x, d->w, d->ldx, d->ldw, d->M, d->N, d->K, 0, 0, 0, 0,
                                               plan.splits > 1 ? static_cast<float*>(d->workspace) : nullptr, epi},
                                       plan, stream);
  });
  return launched();
}

int void_linear_grad_x(const void* dz, int64_t ldz, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K,
                       int32_t dtype, void* dx, int64_t ldx, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const void_linear_args d{.M = M, .N = N, .K = K, .dtype = dtype};
  const int st = check(&d);
  if (st <= 0) return st;
  if (M == 0 || K == 0) return VOID_OK;
  const int esz = size_of(dtype);
  if (!dx || (N && (!dz || !w))) return void_internal_fail(VOID_ERR_ARG, "null array");
  if (M > 1 && (ldz < N || ldx < K)) return void_internal_fail(VOID_ERR_ARG, "leading dimension too small");
  if ((uintptr_t)dx % esz) return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements");
  if (N && (!whole_chunks(dz, ldz, padded(N, esz), esz) || ldz < padded(N, esz) ||
            !whole_chunks(w, ldw, padded(K, esz), esz) || ldw < padded(K, esz)))
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "the products of the gradient need rows of whole 16-byte chunks");
  if (N && !(within_reach(M, ldz, esz) && within_reach(N, ldw, esz, true)))
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "rows are too far apart");
  const Plan plan = plan_of(M, K, N, esz);
  if (!plan.tile) return void_internal_fail(VOID_ERR_UNSUPPORTED, "more tiles than a grid holds");
  if (plan.splits > 1 && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < (size_t)plan.splits * M * K * 4))
    return void_internal_fail(VOID_ERR_WORKSPACE, "linear gradient: workspace missing or too small");
  by_type(dtype, [&](auto e) {
    product<decltype(e), false, true>(Product{dz, w, ldz, ldw, M, K, N, 0, 0, 0, 0,
                                              plan.splits > 1 ? static_cast<float*>(workspace) : nullptr,
                                              Epilogue{dx, ldx, nullptr, nullptr, 0, nullptr, 0, VOID_ACT_NONE}},
                                      plan, stream);
  });
  return launched();
}

int void_linear_grad_w(const void* dz, int64_t ldz, const void* x, int64_t ldx, int64_t M, int64_t N, int64_t K,
                       int32_t dtype, void* dw, int64_t ldw, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const void_linear_args d{.M = M, .N = N, .K = K, .dtype = dtype};
  const int st = check(&d);
  if (st <= 0) return st;
  if (N == 0 || K == 0) return VOID_OK;
  const int esz = size_of(dtype);
  if (!dw || (M && (!dz || !x))) return void_internal_fail(VOID_ERR_ARG, "null array");
  if (N > 1 && ldw < K) return void_internal_fail(VOID_ERR_ARG, "leading dimension too small");
  if ((uintptr_t)dw % esz) return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements");
  if (M && (!whole_chunks(dz, ldz, padded(N, esz), esz) || ldz < padded(N, esz) ||
            !whole_chunks(x, ldx, padded(K, esz), esz) || ldx < padded(K, esz)))
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "the products of the gradient need rows of whole 16-byte chunks");
  if (M && !(within_reach(M, ldz, esz, true) && within_reach(M, ldx, esz, true)))
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "rows are too far apart");
  const Plan plan = plan_of(N, K, M, esz);
  if (!plan.tile) return void_internal_fail(VOID_ERR_UNSUPPORTED, "more tiles than a grid holds");
  if (plan.splits > 1 && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < (size_t)plan.splits * N * K * 4))
    return void_internal_fail(VOID_ERR_WORKSPACE, "linear gradient: workspace missing or too small");
  by_type(dtype, [&](auto e) {
    product<decltype(e), true, true>(Product{dz, x, ldz, ldx, N, K, M, 0, 0, 0, 0,
                                             plan.splits > 1 ? static_cast<float*>(workspace) : nullptr,
                                             Epilogue{dw, ldw, nullptr, nullptr, 0, nullptr, 0, VOID_ACT_NONE}},
                                     plan, stream);
  });
  return launched();
}

size_t void_linear_grad_workspace_bytes(int64_t rows, int64_t cols, int64_t depth, int32_t dtype) {
  if (rows <= 0 || cols <= 0) return 0;
  const Plan p = plan_of(rows, cols, depth, size_of(dtype));
  return p.splits > 1 ? (size_t)p.splits * rows * cols * 4 : 0;
}

static int slope_grid(int64_t M, int64_t N, int32_t dtype) {
  const int64_t gx = (N * size_of(dtype) + 1023) / 1024;
  return (int)std::max<int64_t>(1, std::min<int64_t>((M + 3) / 4, (kCus * 8 + gx - 1) / gx));
}

size_t void_linear_grad_z_workspace_bytes(int64_t M, int64_t N, int32_t dtype) {
  return M <= 0 || N <= 0 ? 0 : (size_t)slope_grid(M, N, dtype) * N * 4;
}

int void_linear_grad_z(const void* dy, int64_t lddy, const void* slope, int64_t M, int64_t N, int32_t dtype, void* dz,
                       int64_t ldz, void* db, int32_t bias_dtype, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  void_internal_fail(VOID_OK, "");
  const void_linear_args d{.M = M, .N = N, .dtype = dtype};
  const int st = check(&d);
  if (st <= 0) return st;
  if (N == 0 || (!dz && !db)) return VOID_OK;
  const int esz = size_of(dtype);
  if (M && !dy) return void_internal_fail(VOID_ERR_ARG, "null dy");
  if (dz && (!slope || (uintptr_t)dz % 16 || ldz * esz % 16 || ldz < padded(N, esz)))
    return void_internal_fail(VOID_ERR_ARG, "dz needs the slope and rows of whole 16-byte chunks");
  if (db && bias_dtype != dtype && bias_dtype != VOID_DT_F32)
    return void_internal_fail(VOID_ERR_UNSUPPORTED, "the bias has the values' type, or fp32");
  if (((uintptr_t)dy | (uintptr_t)slope) % esz || (uintptr_t)db % size_of(bias_dtype) || (M > 1 && lddy < 0))
    return void_internal_fail(VOID_ERR_ARG, "arrays must be aligned to their elements");
  const int gy = M ? slope_grid(M, N, dtype) : 0;
  if (db && M && (!workspace || (uintptr_t)workspace % 4 || workspace_bytes < (size_t)gy * N * 4))
    return void_internal_fail(VOID_ERR_WORKSPACE, "linear gradient: workspace missing or too small");
  by_type(dtype, [&](auto e) {
    using E = decltype(e);
    if (M)
      by_parity<E>(dy, lddy, slope, slope ? N : 0, M, [&](auto odd) {
        hipLaunchKernelGGL((slope_kernel<E, decltype(odd)::value>), dim3((unsigned)((N * esz + 1023) / 1024), gy),
                           dim3(256), 0, stream, static_cast<const E*>(dy), lddy,
                           static_cast<const typename Slope<E>::type*>(slope), M, (int)N, static_cast<E*>(dz), ldz,
                           db ? static_cast<float*>(workspace) : nullptr);
      });
    if (db) {
      const dim3 grid = grid_of((N + 63) / 64);
      if (bias_dtype == VOID_DT_F32)
        hipLaunchKernelGGL(bias_sum_kernel<float>, grid, dim3(1024), 0, stream, static_cast<float*>(workspace), gy,
                           (int)N, static_cast<float*>(db));
      else
        hipLaunchKernelGGL(bias_sum_kernel<E>, grid, dim3(1024), 0, stream, static_cast<float*>(workspace), gy, (int)N,
                           static_cast<E*>(db));
    }
  });
  return launched();
}

}  // extern "C"
