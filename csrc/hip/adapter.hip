// Low-rank adapters beside a shared projection, and their gradients.
//
//   S = X A_i (T x r, fp32)    Y = X W + s_i S B_i
//   D = dY B_i^T (T x r)       dX = dY W^T + s_i D A_i^T
//   dA_i = s_i sum_t X_t^T D_t     dB_i = s_i sum_t S_t^T dY_t    (rows t of adapter i)
//
// Names: U (T x C) is the operand with a row per token, F_i the factor that
// brings it down to r columns, G_i the factor that brings those up again, so
// that dX is the same product as Y with the operands turned.
//
// Few rows (up to 64, a decoding step): bound by reading W once.  Two launches:
// partial sums of U W over pieces of C and of U F_i beside them, then their sums
// and the product with G_i.  32 rows, 64 adapters of rank 16, bf16 4096 x 4096:
// 10.9 + 5.2 us, W read at 3.1 TB/s (a large copy on this card: 4.95).
// Many rows: bound by the matrix units.  The rows are ordered by adapter, so a
// tile of the large product has few adapters; the factors are laid out for the
// matrix units once per call; U F_i is one pass over U; the accumulators of the
// large product begin with s_i (U F_i) G_i.  8192 rows, bf16 8192 x 8192, rank 64:
// 8 + 58 + 840 to 875 us, the large product at 1.26 to 1.31 PFLOP/s (a plain library product of
// that size: 1.27 to 1.56 by its layout).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <type_traits>
#include <utility>

#include "device_common.h"
#include "gelim/internal.h"

namespace gelim {
namespace {

using dev::f4;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// A matrix, or one matrix per adapter: element (i, j) of adapter a is p[a as + i rs + j cs]; rs or cs is 1.
struct View {
  const void* p;
  int64_t as, rs, cs;
};

// 16 bytes of a type, and the matrix instruction over them: lane l of a wave
// holds row (column) l % 16 and, of a step of kStep values along the sum, the
// kE ones from (l / 16) kE on.  In D lane l has column l % 16, rows 4 (l / 16) .. + 3.
template <class T>
struct Mma;
template <>
struct Mma<__bf16> {
  static constexpr int kE = 8, kStep = 32;
  using Frag = bf8;
  static __device__ __forceinline__ f4 mma(Frag a, Frag b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> {
  static constexpr int kE = 8, kStep = 32;
  using Frag = h8;
  static __device__ __forceinline__ f4 mma(Frag a, Frag b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  static constexpr int kE = 4, kStep = 16;
  using Frag = f4;
  static __device__ __forceinline__ f4 mma(Frag a, Frag b, f4 c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};

// The blocks of the large product: kB rows and columns; lane l has row (column) l % kB and, of a step along the sum,
// the kE values from (l / kB) kE on.  16-bit types as above: 32 x 32 x 16 instructions alone, from registers, reach 1670
// TFLOP/s at the clock that the card holds under them, 16 x 16 x 32 1800 (profiles/adapter_counters.txt).
template <class T>
struct Block {
  static constexpr int kB = 16;
  using Acc = f4;
  static __device__ __forceinline__ f4 mma(typename Mma<T>::Frag a, typename Mma<T>::Frag b, f4 c) {
    return Mma<T>::mma(a, b, c);
  }
};
// fp32: in D lane l has column l % 32 and the rows 8 (r / 4) + 4 (l / 32) + r % 4
template <>
struct Block<float> {
  static constexpr int kB = 32;
  typedef float Acc __attribute__((ext_vector_type(16)));
  static __device__ __forceinline__ Acc mma(f4 a, f4 b, Acc c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};

template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
  T v[4];
};
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned {
  typename Mma<T>::Frag v;
};
// 16 bytes from any element's address; with fewer than kE elements there, zeros in the others' place
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag load16(const T* p) {
  return ((const Unaligned<T>*)p)->v;
}
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag load_part(const T* p, int64_t have) {
  constexpr int E = Mma<T>::kE;
  if (have >= E) return load16(p);
  typename Mma<T>::Frag v = {};
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < have) v[e] = p[e];
  return v;
}

// The same without a branch, for waves of which all lanes are at an edge or may be: kE loads in flight.  The row's
// last element, have - 1 from p, exists also where have <= 0.
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag load_edge(const T* p, int have) {
  constexpr int E = Mma<T>::kE;
  typename Mma<T>::Frag v;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const T x = p[min(e, have - 1)];
    v[e] = e < have ? x : (T)0.f;
  }
  return v;
}

// kE rows (along the sum) of kE columns each, in registers, turned: out[j] holds column j's kE values.
// 16-bit types: 32 byte permutes for 64 elements.
template <class T>
__device__ __forceinline__ void turn(const typename Mma<T>::Frag (&in)[Mma<T>::kE],
                                     typename Mma<T>::Frag (&out)[Mma<T>::kE]) {
  if constexpr (sizeof(T) == 2) {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    u4 o[8];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const u4 a = __builtin_bit_cast(u4, in[2 * p]), b = __builtin_bit_cast(u4, in[2 * p + 1]);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        o[2 * d][p] = __builtin_amdgcn_perm(b[d], a[d], 0x05040100);
        o[2 * d + 1][p] = __builtin_amdgcn_perm(b[d], a[d], 0x07060302);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = __builtin_bit_cast(typename Mma<T>::Frag, o[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) out[j][k] = in[k][j];
  }
}

// What the rows are: adapter of each, its factor, and how many there are of both.
struct Rows {
  const int32_t* index;
  const float* scale;
  float scale_value;
  int n, T;
};
__device__ __forceinline__ int adapter_of(const Rows& g, int64_t t) { return g.index ? g.index[t] : 0; }
__device__ __forceinline__ float scale_of(const Rows& g, int i) { return g.scale ? g.scale[i] : g.scale_value; }

// ---- few rows -------------------------------------------------------------

struct Few {
  const void* U;
  int64_t ldu;
  View W, F;
  Rows rows;
  float *part, *low;  // part: splits x T x ldp, low: low_splits x T x r
  int C, N, r, ldp, splits, blocks, low_splits;
};

// The first of the kE columns that a lane takes where W's rows run along memory: at the end of a row the lane takes
// its last kE, some of them a neighbour's as well, who comes to the same sums.
__device__ __forceinline__ int few_column(int N, int n, int E) { return N >= E ? min(n, N - E) : n; }
// One wave: 16 kE columns of W, its steps of the sum; W_KC: W's sum runs along its rows in memory. Each 16-byte
// load of 16 neighbouring lanes covers 256 bytes of a row of W (64 where W_KC: two steps make the line). One step's
// loads in flight: with two, fewer waves fit a SIMD, and 32 rows of 4096 x 4096 took 14.2 instead of 10.9 us.
template <class T, bool W_KC, int TT, bool EDGE>
__device__ __forceinline__ void few_steps(const Few& a, int n0, int s0, int s1, f4 (&acc)[Mma<T>::kE][TT]) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr int E = M::kE;
  const int l16 = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
  const T* W = (const T*)a.W.p;
  const T* U = (const T*)a.U;
  for (int s = s0; s < s1; ++s) {
    const int k = s * M::kStep + g * E;
    Frag w[E], x[TT];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if constexpr (W_KC) {
        const T* col = W + (int64_t)min(n0 + j * 16 + l16, a.N - 1) * a.W.cs;
        if constexpr (EDGE) w[j] = load_edge(col + k, a.C - k);
        else w[j] = load16(col + k);
      } else {
        const int n = few_column(a.N, n0 + l16 * E, E);
        if constexpr (EDGE) {
          w[j] = load_edge(W + (int64_t)min(k + j, a.C - 1) * a.W.rs + n, a.N - n);
          if (k + j >= a.C) w[j] = Frag{};
        } else {
          w[j] = load16(W + (int64_t)(k + j) * a.W.rs + n);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const T* row = U + (int64_t)min(t * 16 + l16, a.rows.T - 1) * a.ldu;
      if constexpr (EDGE) x[t] = load_edge(row + k, a.C - k);
      else x[t] = load16(row + k);
    }
    if constexpr (!W_KC) {
      Frag v[E];
      turn<T>(w, v);
#pragma unroll
      for (int j = 0; j < E; ++j) w[j] = v[j];
    }
#pragma unroll
    for (int j = 0; j < E; ++j)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[j][t] = M::mma(w[j], x[t], acc[j][t]);
  }
}

constexpr int kLowPiece = 512;  // values of C: a wave's load of 16 bytes a lane, or two
// low (T x r) of one row over one piece of C, on the vector units: F_i is read once per row that uses it.
template <class T>
__device__ __forceinline__ void few_low(const Few& a, int t, int split, float* lds) {
  using M = Mma<T>;
  constexpr int E = M::kE;
  const int i = adapter_of(a.rows, t);
  if (i < 0 || i >= a.rows.n) return;
  const int piece = (a.C + a.low_splits * kLowPiece - 1) / (a.low_splits * kLowPiece) * kLowPiece;
  const int c0 = min(a.C, split * piece), c1 = min(a.C, c0 + piece);
  const T* u = (const T*)a.U + t * a.ldu;
  const T* f = (const T*)a.F.p + i * a.F.as;
  float* out = a.low + ((int64_t)split * a.rows.T + t) * a.r;
  if (a.F.rs != 1) {
    // r values side by side: thread (c, chunk of E ranks); what a chunk reads behind the last rank is not used
    const int chunks = (a.r + E - 1) / E, lanes = 256 / chunks;
    const int j0 = threadIdx.x % chunks * E, cl = threadIdx.x / chunks;
    const int64_t last = (int64_t)(a.C - 1) * a.F.rs + a.r - E - j0;  // the last offset that 16 bytes can be read from
    const int whole = last < 0 ? c0 : a.F.rs == 0 ? c1 : (int)min((int64_t)c1, last / a.F.rs + 1);
    float acc[E] = {};
    if (cl < lanes) {
      int c = c0 + cl;
#pragma unroll 4
      for (; c < whole; c += lanes) {
        const auto v = load16(f + c * a.F.rs + j0);
        const float x = (float)u[c];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += x * (float)v[e];
      }
      for (; c < c1; c += lanes) {
        const auto v = load_edge(f + c * a.F.rs + j0, a.r - j0);
        const float x = (float)u[c];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += x * (float)v[e];
      }
    }
    // thread layout [cl][chunk][e] is [cl][rank]: sum over cl in two steps
#pragma unroll
    for (int e = 0; e < E; ++e) lds[threadIdx.x * E + e] = acc[e];
    __syncthreads();
    const int width = chunks * E, shares = min(256 / width, 16);
    const int j = threadIdx.x % width, share = threadIdx.x / width;
    float s = 0.f;
    if (share < shares)
      for (int c = share; c < lanes; c += shares) s += lds[c * width + j];
    __syncthreads();
    if (share < shares) lds[share * width + j] = s;
    __syncthreads();
    if (share == 0 && j < a.r) {
      s = 0.f;
      for (int c = 0; c < shares; ++c) s += lds[c * width + j];
      out[j] = s;
    }
  } else {
    // the sum runs along memory: a wave per rank
    const int lane = threadIdx.x % 64;
    for (int j = threadIdx.x / 64; j < a.r; j += 4) {
      const T* fj = f + j * a.F.cs;
      float s = 0.f;
      for (int c = c0 + lane * E; c < c1; c += 64 * E) {
        const auto v = load_part(fj + c, c1 - c), x = load_part(u + c, c1 - c);
#pragma unroll
        for (int e = 0; e < E; ++e) s += (float)v[e] * (float)x[e];
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
      if (lane == 0) out[j] = s;
    }
  }
}

// The first launch: blocks x splits workgroups of the large product, then T x low_splits of the low one.
// Four waves share a block of 16 kE columns and cut its steps once more; their sums meet in LDS.
template <class T, bool W_KC, int TT>
__global__ __launch_bounds__(256, TT <= 2 ? 3 : 2) void few_kernel(Few a) {
  using M = Mma<T>;
  constexpr int E = M::kE, kCols = 16 * E;
  constexpr int kFrags = E * TT;
  __shared__ f4 lds[2 * kFrags * 64];
  const int b = blockIdx.x;
  if (b >= a.blocks * a.splits) {
    static_assert(sizeof(lds) >= 256 * E * sizeof(float), "few_low's sums");
    const int q = b - a.blocks * a.splits;
    few_low<T>(a, q / a.low_splits, q % a.low_splits, (float*)lds);
    return;
  }
  const int block = b % a.blocks, split = b / a.blocks, n0 = block * kCols;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int steps = (a.C + M::kStep - 1) / M::kStep, parts = a.splits * 4, part = split * 4 + wave;
  const int s0 = (int)((int64_t)steps * part / parts), s1 = (int)((int64_t)steps * (part + 1) / parts);
  f4 acc[E][TT] = {};
  const int whole = W_KC || a.N >= E ? min(s1, a.C / M::kStep) : s0;  // steps before one that ends behind the sum
  few_steps<T, W_KC, TT, false>(a, n0, s0, whole, acc);
  few_steps<T, W_KC, TT, true>(a, n0, max(s0, whole), s1, acc);
  // waves 2 and 3 hand theirs to 0 and 1, then 1 to 0
#pragma unroll
  for (int half = 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int j = 0; j < E; ++j)
#pragma unroll
        for (int t = 0; t < TT; ++t) lds[((wave - half) * kFrags + j * TT + t) * 64 + lane] = acc[j][t];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int j = 0; j < E; ++j)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[j][t] += lds[(wave * kFrags + j * TT + t) * 64 + lane];
    __syncthreads();
  }
  if (wave) return;
  const int l16 = lane % 16, g = lane / 16;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int row = t * 16 + l16;
    if (row >= a.rows.T) continue;
    float* out = a.part + ((int64_t)split * a.rows.T + row) * a.ldp;
    if constexpr (W_KC) {
#pragma unroll
      for (int j = 0; j < E; ++j) *(f4*)(out + n0 + j * 16 + g * 4) = acc[j][t];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < E; j += 4) {
          const Four<float> v = {acc[j][t][i], acc[j + 1][t][i], acc[j + 2][t][i], acc[j + 3][t][i]};
          *(Four<float>*)(out + few_column(a.N, n0 + (g * 4 + i) * E, E) + j) = v;
        }
    }
  }
}

// The second launch: sums of the pieces, the product with G_i (r = 0: it is in them), the result.
// A workgroup takes 256 columns of one row, its four waves sharing the pieces and the ranks, or (ONE_ROW false: with
// enough rows to fill the chip) of four rows, a wave each.
struct Finish {
  const float *part, *low;
  View G;
  Rows rows;
  const int32_t* perm;  // the row at each place of part and low; null: in order
  int N, r, ldp, splits, low_splits, ldl, blocks;
  void* Y;
  int64_t ldy;
};

template <class T, bool ONE_ROW>
__global__ __launch_bounds__(256) void finish_kernel(Finish a) {
  constexpr int kShare = ONE_ROW ? 4 : 1;
  __shared__ float s_all[ONE_ROW ? 1 : 4][GELIM_ADAPTER_MAX_RANK];
  __shared__ f4 sums[3][64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, part = ONE_ROW ? wave : 0;
  const int at = ONE_ROW ? blockIdx.x / a.blocks : blockIdx.x / a.blocks * 4 + wave;
  if (!ONE_ROW && at >= a.rows.T) return;
  float* s = s_all[ONE_ROW ? 0 : wave];
  const int64_t t = a.perm ? a.perm[at] : at;
  const int i = adapter_of(a.rows, t);
  const bool has = i >= 0 && i < a.rows.n;
  const int n = blockIdx.x % a.blocks * 256 + lane * 4;
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  if (n < a.N)
#pragma unroll 4
    for (int p = part; p < a.splits; p += kShare)
      acc += *(const f4*)(a.part + ((int64_t)p * a.rows.T + at) * a.ldp + n);
  if (has) {
    const float f = scale_of(a.rows, i);
    for (int j = ONE_ROW ? threadIdx.x : lane; j < a.r; j += ONE_ROW ? 256 : 64) {
      float v = 0.f;
      for (int p = 0; p < a.low_splits; ++p) v += a.low[((int64_t)p * a.rows.T + at) * a.ldl + j];
      s[j] = f * v;
    }
  }
  if constexpr (ONE_ROW) __syncthreads();
  else __builtin_amdgcn_wave_barrier();
  if (has && n < a.N) {
    const T* G = (const T*)a.G.p + i * a.G.as;
    const int have = min(4, a.N - n);
    if (a.G.cs == 1 && have == 4) {
#pragma unroll 4
      for (int j = part; j < a.r; j += kShare) {
        const Four<T> v = *(const Four<T>*)(G + j * a.G.rs + n);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += s[j] * (float)v.v[e];
      }
    } else if (a.G.rs == 1) {
      // ranks side by side: 16 bytes of them at a time
      constexpr int E = Mma<T>::kE;
      const int64_t last = (a.N - 1) * a.G.cs + a.r - E;
      for (int j = part * E; j < a.r; j += kShare * E)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t at = min(n + e, a.N - 1) * a.G.cs + j;
          const auto v = at <= last ? load16(G + at) : load_edge(G + at, a.r - j);
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (j + k < a.r) acc[e] += s[j + k] * (float)v[k];
        }
    } else {
      for (int j = part; j < a.r; j += kShare)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < have) acc[e] += s[j] * (float)G[j * a.G.rs + (n + e) * a.G.cs];
    }
  }
  if constexpr (ONE_ROW) {
    if (wave) sums[wave - 1][lane] = acc;
    __syncthreads();
    if (wave) return;
    acc += sums[0][lane] + sums[1][lane] + sums[2][lane];
  }
  if (n >= a.N) return;
  if (!has && i != -1) acc = acc * __builtin_nanf("");
  T* y = (T*)a.Y + t * a.ldy + n;
  if (n + 4 <= a.N) {
    *(Four<T>*)y = Four<T>{(T)acc[0], (T)acc[1], (T)acc[2], (T)acc[3]};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) y[e] = (T)acc[e];
  }
}

bool one_row(const Finish& e) { return (int64_t)e.rows.T * e.blocks < 2048; }
int64_t finish_groups(const Finish& e) { return (int64_t)(one_row(e) ? e.rows.T : (e.rows.T + 3) / 4) * e.blocks; }
template <class T>
void finish(const Finish& e, hipStream_t s) {
  const dim3 grid((unsigned)finish_groups(e));
  if (one_row(e)) hipLaunchKernelGGL((finish_kernel<T, true>), grid, dim3(256), 0, s, e);
  else hipLaunchKernelGGL((finish_kernel<T, false>), grid, dim3(256), 0, s, e);
}

// ---- many rows ------------------------------------------------------------
//
// The rows in order of their adapter: perm (T places), start (n + 1): adapter
// i's places are start[i] .. start[i + 1] - 1, rows without one come last.  With one adapter
// and no index both are null and the order is the rows' own.

struct Order {
  const int32_t *perm, *start;
  bool packed;  // the layouts of the factors have a slot for each row's adapter at most, not one for each resident one
};
__device__ __forceinline__ int64_t row_at(const Order& o, int64_t at) { return o.perm ? o.perm[at] : at; }
// adapter i's layout, if it has rows: both i and start grow from one adapter with rows to the next, and start < T
__device__ __forceinline__ int packed_slot(int i, int start) { return min(i, start); }

// Pieces of at most `size` places, each within one adapter.  Adapter i's pieces have the numbers from
// start[i] / size + min(i, start[i]) on: distinct for different adapters, as floor((s + c) / size) - floor(s / size) + 1
// >= ceil(c / size) and an adapter with rows moves both i and start on, and without a sum over the adapters.  So there
// are no more than T / size + min(n, T) numbers, however many adapters are resident.  Some stay empty (count 0).
struct Piece {
  int adapter, begin, count, slot;  // slot: where its factors are laid out
};
__device__ __forceinline__ int first_piece(int start, int i, int size) { return start / size + min(i, start); }
__device__ __forceinline__ Piece piece_of(const Piece* table, const Rows& g, int number, int size) {
  if (!table) return {0, number * size, max(0, min(size, g.T - number * size)), 0};
  return table[number];
}
int pieces(int64_t T, int64_t n, bool ordered, int size) {
  return (int)(T / size + std::min<int64_t>(ordered ? n : 1, T));
}

// A matrix (one per adapter) copied as rows x ld values, zeros behind the source's rows and columns; or in a matrix
// instruction's fragments, so that a wave's load of one is 1 KB without gaps: kFrag16 by steps along ld, blocks of 16
// rows, lanes, kE values; kFrag32 by blocks of 32 rows, 8 values along ld, lanes, kE values.
enum { kRows, kFrag16, kFrag32 };
struct Copy {
  View src;
  void* dst;
  int rows, cols, ld, count;  // of the copy (rows, ld) and how many matrices
  int have;                   // rows of the source; the others are zeros
  int order;  // kRows, or in fragments
  bool straight;
  int first;                  // workgroups before this copy's
  int tiles, per;             // of a matrix that is not straight, and of a workgroup
};
constexpr int kCopies = 6, kCopyTile = 64;
struct Prepare {
  Rows rows;
  int32_t *perm, *start;
  int order_groups;  // n + 1, or 0: the order is not needed
  bool packed;
  struct Pieces {
    Piece* table;
    int size;
  } pieces[2];
  Copy copy[kCopies];
  int copies;
  int* counter;  // set to zero for the launches behind this one
  int counters;
};

// Adapter i's rows (i = n: those without one), in order, by one workgroup:
// it counts the rows of lower adapters, then writes its own behind those.  A thread takes kOrder rows side by side.
constexpr int kOrder = 32, kPrepare = 256;
__device__ __forceinline__ void order_rows(const Prepare& p, int i) {
  __shared__ int sums[2][kPrepare / 64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = p.rows.n;
  int id[kOrder];
  auto fetch = [&](int64_t t0) {  // adapters of this thread's rows; behind the last row -1
#pragma unroll
    for (int q = 0; q < kOrder; q += 4) {
      const int64_t t = t0 + threadIdx.x * kOrder + q;
      Four<int> a = {{0, 0, 0, 0}};
      if (t + 4 <= p.rows.T) a = *(const Four<int>*)(p.rows.index + t);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t + e < p.rows.T) a.v[e] = p.rows.index[t + e];
#pragma unroll
      for (int e = 0; e < 4; ++e) id[q + e] = t + e >= p.rows.T ? -1 : a.v[e] < 0 || a.v[e] >= n ? n : a.v[e];
    }
  };
  int c = 0;
  for (int64_t t0 = 0; t0 < p.rows.T; t0 += kPrepare * kOrder) {
    fetch(t0);
#pragma unroll
    for (int q = 0; q < kOrder; ++q) c += id[q] >= 0 && id[q] < i;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
  if (lane == 0) sums[0][wave] = c;
  __syncthreads();
  int at = 0;
  for (int w = 0; w < kPrepare / 64; ++w) at += sums[0][w];
  const int begin = at;
  if (threadIdx.x == 0) p.start[i] = at;
  for (int64_t t0 = 0; t0 < p.rows.T; t0 += kPrepare * kOrder) {
    if (p.rows.T > kPrepare * kOrder) fetch(t0);  // otherwise they are still here
    int mine = 0;
#pragma unroll
    for (int q = 0; q < kOrder; ++q) mine += id[q] == i;
    int upto = mine;  // of this and the lower lanes
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 63) sums[1][wave] = upto;
    __syncthreads();
    int place = at + upto - mine;
    for (int w = 0; w < kPrepare / 64; ++w) {
      if (w < wave) place += sums[1][w];
      at += sums[1][w];
    }
#pragma unroll
    for (int q = 0; q < kOrder; ++q)
      if (id[q] == i) p.perm[place++] = (int32_t)(t0 + threadIdx.x * kOrder + q);
  }
  // this adapter's pieces, and empty ones up to the next adapter's; behind the last adapter empty ones to the
  // table's end
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int size = p.pieces[k].size;
    if (!p.pieces[k].table) continue;
    const int first = first_piece(begin, i, size);
    const int end = i < n ? first_piece(at, i + 1, size) : p.rows.T / size + min(n, p.rows.T);
    for (int q = first + threadIdx.x; q < end; q += kPrepare) {
      const int from = begin + (q - first) * size;
      p.pieces[k].table[q] = {i, from, i < n ? max(0, min(size, at - from)) : 0, p.packed ? packed_slot(i, begin) : i};
    }
  }
}

// 16 KB of a copy whose source runs along its rows: 16 bytes a thread, from any element's address.
constexpr int kStraight = 1024;  // chunks of 16 bytes
template <class T>
__device__ __forceinline__ void copy_straight(const Copy& c, int part) {
  constexpr int E = Mma<T>::kE;
  const int across = c.ld / E;
  const int64_t all = (int64_t)c.count * c.rows * across;
#pragma unroll
  for (int q = 0; q < kStraight / kPrepare; ++q) {
    const int64_t o = (int64_t)part * kStraight + q * kPrepare + threadIdx.x;
    if (o >= all) return;
    const int64_t row = o / across, m = row / c.rows, i = row % c.rows;
    const int j = (int)(o % across) * E;
    *((typename Mma<T>::Frag*)c.dst + o) =
        load_part((const T*)c.src.p + m * c.src.as + i * c.src.rs + j, i < c.have ? c.cols - j : 0);
  }
}

// One 64 x 64 tile of a copy, read along the source's memory and written along the destination's, 16 bytes a thread.
template <class T>
__device__ __forceinline__ void copy_tile(const Copy& c, int m, int slot, int tile) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr int E = M::kE, kAcross = kCopyTile / E, kChunks = kCopyTile * kAcross;
  __shared__ T lds[kCopyTile][kCopyTile + 2];
  const int across = (c.ld + kCopyTile - 1) / kCopyTile;
  const int r0 = tile / across * kCopyTile, c0 = tile % across * kCopyTile;
  const T* src = (const T*)c.src.p + m * c.src.as;
  T* dst = (T*)c.dst + (int64_t)slot * c.rows * c.ld;
  const bool along = c.src.cs == 1;
  Frag v[kChunks / kPrepare];
#pragma unroll
  for (int q = 0; q < kChunks / kPrepare; ++q) {
    const int o = q * kPrepare + threadIdx.x, slow = o / kAcross, fast = o % kAcross * E;
    const int i = r0 + (along ? slow : fast), j = c0 + (along ? fast : slow);
    const bool in = i < c.have && j < c.cols;
    v[q] = load_part(src + i * c.src.rs + j * c.src.cs, !in ? 0 : along ? c.cols - j : c.have - i);
  }
#pragma unroll
  for (int q = 0; q < kChunks / kPrepare; ++q) {
    const int o = q * kPrepare + threadIdx.x, slow = o / kAcross, fast = o % kAcross * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (along) lds[slow][fast + e] = v[q][e];
      else lds[fast + e][slow] = v[q][e];
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kChunks / kPrepare; ++q) {
    int o = q * kPrepare + threadIdx.x, i, j;
    T* to;
    if (c.order == kFrag16) {
      const int blocks = c.rows / 16, here = min(4, blocks - r0 / 16);  // of 16 rows, in all and in this tile
      const int step = o / (here * 64), rb = o / 64 % here, lane = o % 64;
      if (step >= kCopyTile / M::kStep) continue;
      i = rb * 16 + lane % 16, j = step * M::kStep + lane / 16 * E;
      to = dst + (((int64_t)(c0 / M::kStep + step) * blocks + r0 / 16 + rb) * 64 + lane) * E;
    } else {
      i = o / kAcross, j = o % kAcross * E;
      if (r0 + i >= c.rows || c0 + j >= c.ld) continue;
      to = dst + (int64_t)(r0 + i) * c.ld + c0 + j;
      if (c.order == kFrag32)
        to = dst + (((int64_t)(r0 + i) / 32 * (c.ld / 8) + (c0 + j) / 8) * (32 * 8 / E) + j % 8 / E * 32 + i % 32) * E;
    }
    Frag w;
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = lds[i][j + e];
    *(Frag*)to = w;
  }
}

// A workgroup's tiles of one matrix.  With more than a few adapters those that no row has are left out, as resident
// adapters may be many more than a batch uses (500 of rank 16, 7 of them in use, 4096 x 4096: 149 -> 29 us for this
// launch); beyond kScanRows rows, where looking for that would cost more than a tile's copy, all are laid out.  With
// more adapters than rows the same look finds the layout's slot.
constexpr int kScanAdapters = 8, kScanRows = 8192;
template <class T>
__device__ __forceinline__ void copy_tiles(const Copy& c, int part, const Rows& rows, bool packed) {
  const int parts = (c.tiles + c.per - 1) / c.per, m = part / parts, first = part % parts * c.per;
  int slot = m;
  if (c.count > kScanAdapters && rows.T <= kScanRows) {
    constexpr int kLoads = kScanRows / (kPrepare * 4);  // all under way at once
    Four<int> id[kLoads];
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int t = (q * kPrepare + threadIdx.x) * 4;
      id[q] = {{-1, -1, -1, -1}};
      if (t + 4 <= rows.T) id[q] = *(const Four<int>*)(rows.index + t);
    }
    const int rest = rows.T / 4 * 4 + threadIdx.x;
    bool used = rest < rows.T && rows.index[rest] == m;
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) used |= id[q].v[e] == m;
    if (!__syncthreads_or(used)) return;
    if (packed) {
      __shared__ int below[kPrepare / 64];
      int c = rest < rows.T && rows.index[rest] >= 0 && rows.index[rest] < m;  // rows of lower adapters
#pragma unroll
      for (int q = 0; q < kLoads; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) c += id[q].v[e] >= 0 && id[q].v[e] < m;
#pragma unroll
      for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
      if (threadIdx.x % 64 == 0) below[threadIdx.x / 64] = c;
      __syncthreads();
      int start = 0;
      for (int w = 0; w < kPrepare / 64; ++w) start += below[w];
      slot = packed_slot(m, start);
    }
  }
  for (int tile = first; tile < min(c.tiles, first + c.per); ++tile) {
    if (tile != first) __syncthreads();
    copy_tile<T>(c, m, slot, tile);
  }
}

// The first launch: counters cleared, the order, the factors laid out for the matrix units, and
// an operand whose rows do not begin at multiples of 16 bytes copied to where they do.  All parts run beside each
// other: 6 us where there is little to copy, X and W of 4096 x 4095 in bf16 26 us (5.1 TB/s).  Read in place by
// unaligned loads the rows would cost the low-rank pass alone 20 us there (12.5 -> 32.5), as each lane's 16 bytes and
// its neighbours' then lie in two lines.
template <class T>
__global__ __launch_bounds__(kPrepare) void prepare_kernel(Prepare p) {
  int b = blockIdx.x;
  for (int c = b * kPrepare + threadIdx.x; c < p.counters; c += gridDim.x * kPrepare) p.counter[c] = 0;
  if (b < p.order_groups) return order_rows(p, b);
  b -= p.order_groups;
  int k = p.copies - 1;
  while (k > 0 && b < p.copy[k].first) --k;
  if (p.copy[k].straight) copy_straight<T>(p.copy[k], b - p.copy[k].first);
  else copy_tiles<T>(p.copy[k], b - p.copy[k].first, p.rows, p.packed);
}

// low (place, rank) = U F_i, 32 places of one adapter by a workgroup, whose 8 waves cut the sum (16 waves were no
// faster at any size, 10.2 instead of 8.3 us for 150 rows of K 2048, rank 64). F is laid out in fragments, ldf values
// along the sum with zeros behind C.  Bound by what goes through the L2 caches, U once and F_i for every 32 rows
// (8192 x 8192, rank 64: 480 MB at 8.3 TB/s, more than half of it F_i); each wave keeps several steps' loads in
// flight.  With few rows several workgroups cut the sum once more; the last of them to end adds their parts, always
// in the same order. Measured, bf16: 2048 x 4096, rank 16, 8.8 us; 8192 x 8192, rank 64, 58 us (more loads under way,
// waves side by side along a row, or the pieces of an adapter on one XCD changed that by less than the noise). Also
// in fragments of 32 places and 8 ranks for the matrix units of the large product, with 16-bit types as the sum of
// three values of the type, which hold all 24 bits of the fp32 sum.  fp16: a row is first brought to below 2^14 by a
// power of two (`by`), as it may be beyond the type's range; small values of the row are off by 2^-38 of its largest
// at most.
struct Low {
  const void *U, *F;
  int64_t ldu;
  float *low, *by;
  void* split;
  int cu, ldf, pieces, splits;  // cu: values in a row of U, a multiple of 16 bytes
  float* part;                  // piece, split, fragment, lane, 4 values; with splits > 1
  int* arrived;                 // of each piece
};
struct LowPair {
  Low p[2];
  Rows rows;
  Order order;
  const Piece* table;
  int r;
};
constexpr int kLowRows = 32;
constexpr int kLowWaves = 8;
// steps whose loads are under way, by the registers of two workgroups a CU (rank 120, 4096 rows of 4096: 25 us, with
// one step 29)
constexpr int low_flight(int rank_blocks) { return rank_blocks <= 4 ? 4 : rank_blocks == 8 ? 2 : 1; }

// v as the sum of kTerms values of the type, all of its sign and none of them zero: each but the last is the largest
// one below what is left (in size), so that nothing is lost on the way (bf16: 8 + 8 + 8 bits).  Beside an infinite
// factor the terms then give v's infinity; with the nearest values a second term of 0 or of the other sign would give
// NaN.  0, infinities and NaN are all of their terms.
template <class T>
constexpr int kTerms = sizeof(T) == 2 ? 3 : 1;
template <class T>
__device__ __forceinline__ void terms(float v, T (&out)[kTerms<T>]) {
  const bool whole = !(fabsf(v) > 0.f && fabsf(v) <= 3.402823466e38f);
#pragma unroll
  for (int h = 0; h < kTerms<T> - 1; ++h) {
    const float below = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) - 1);
    T t = 0;
    if constexpr (std::is_same_v<T, _Float16>) t = (T)__builtin_amdgcn_cvt_pkrtz(below, 0.f)[0];
    else if constexpr (sizeof(T) == 2)
      t = __builtin_bit_cast(T, (unsigned short)(__builtin_bit_cast(unsigned, below) >> 16));
    out[h] = whole ? (T)v : t;
    v = whole ? v : v - (float)t;
  }
  out[kTerms<T> - 1] = (T)v;
}
// a power of two that brings fp16's `most` to [2^13, 2^14)
__device__ __forceinline__ int to_fp16_range(float most) {
  return most > 0.f ? min(max(13 - ilogbf(most), -100), 100) : 0;
}

template <class T, int RB>
__global__ __launch_bounds__(kLowWaves * 64) void low_kernel(LowPair both) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr int E = M::kE, rp = 16 * RB, kWaves = kLowWaves;
  __shared__ f4 lds[kWaves / 2][RB * 2][64];
  const Low& a = both.p[blockIdx.y];
  const int piece = blockIdx.x % a.pieces, split = blockIdx.x / a.pieces;
  if (split >= a.splits) return;
  const Piece pc = piece_of(both.table, both.rows, piece, kLowRows);
  if (pc.count == 0) return;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, l16 = lane % 16, g = lane / 16;
  const T* u[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
    u[t] = (const T*)a.U + row_at(both.order, pc.begin + min(t * 16 + l16, pc.count - 1)) * a.ldu;
  const Frag* f = (const Frag*)((const T*)a.F + (int64_t)pc.slot * rp * a.ldf) + lane;
  const int steps = (a.cu + M::kStep - 1) / M::kStep;
  const int shares = kWaves * a.splits, share = split * kWaves + wave;
  const int s0 = (int)((int64_t)steps * share / shares), s1 = (int)((int64_t)steps * (share + 1) / shares);
  f4 acc[RB][2] = {};
  constexpr int kFlight = low_flight(RB);
  for (int s = s0; s < s1; s += kFlight) {
    Frag x[kFlight][2], w[kFlight][RB];
#pragma unroll
    for (int q = 0; q < kFlight; ++q) {
      // a step behind the last one repeats it, with zeros for U
      const int step = min(s + q, s1 - 1), k = step * M::kStep + g * E;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        x[q][t] = Frag{};
        if (k < a.cu && s + q < s1) x[q][t] = *(const Frag*)(u[t] + k);
      }
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        w[q][j] = Frag{};
        if (s + q < s1) w[q][j] = f[((int64_t)step * RB + j) * 64];
      }
    }
#pragma unroll
    for (int q = 0; q < kFlight; ++q)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[j][t] = M::mma(w[q][j], x[q][t], acc[j][t]);
  }
#pragma unroll
  for (int half = kWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) lds[wave - half][j * 2 + t][lane] = acc[j][t];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[j][t] += lds[wave][j * 2 + t][lane];
    __syncthreads();
  }
  if (a.splits > 1) {
    // The parts go past the caches that other XCDs do not see (sc1: the scope of the whole device), so that none has to
    // be written back or dropped as by a fence; the count goes up when they have arrived (vmcnt 0).
    constexpr int kDevice = 16;
    typedef int i4 __attribute__((ext_vector_type(4)));
    float* mine = a.part + (int64_t)piece * a.splits * (RB * 2 * 64 * 4);
    auto parts = __builtin_amdgcn_make_buffer_rsrc(mine, 0, a.splits * RB * 2 * 1024, 0x00027000);
    __shared__ int last;
    if (wave == 0) {
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i4, acc[j][t]), parts,
                                                 ((split * RB + j) * 2 + t) * 1024 + lane * 16, 0, kDevice);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (lane == 0)
        last = __hip_atomic_fetch_add(a.arrived + piece, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.splits - 1;
    }
    __syncthreads();
    if (!last) return;
    for (int m = wave; m < RB * 2; m += kWaves) {
      f4 v = {0.f, 0.f, 0.f, 0.f};
      for (int p = 0; p < a.splits; p += 4) {
        f4 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          w[q] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
                     parts, (min(p + q, a.splits - 1) * RB * 2 + m) * 1024 + lane * 16, 0, kDevice));
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (p + q < a.splits) v += w[q];
      }
      lds[0][m][lane] = v;
    }
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[j][t] = lds[0][j * 2 + t][lane];
  }
  if (wave) return;
  // behind the last rank zeros, not an infinity times F's zeros there
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j * 16 + g * 4 + i >= both.r) acc[j][0][i] = acc[j][1][i] = 0.f;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const bool in = t * 16 + l16 < pc.count;
    const int64_t at = pc.begin + t * 16 + l16;
    float by = 1.f;
    if constexpr (std::is_same_v<T, _Float16>) {
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = fabsf(acc[j][t][i]);
          if (v > most && v <= 3.4e38f) most = v;
        }
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      const int e = to_fp16_range(most);
      by = ldexpf(1.f, e);
      if (in && g == 0) a.by[at] = ldexpf(1.f, -e);
    }
    if (!in) continue;
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      *(f4*)(a.low + at * rp + j * 16 + g * 4) = acc[j][t];
      // in fragments of 8 ranks (j * 2 + g / 2) and 32 places: 32 lanes for each term, fp32 two halves of the ranks
      T* out = (T*)a.split + ((at / 32 * (rp / 8) + j * 2 + g / 2) * (sizeof(T) == 2 ? 96 : 64) + at % 32) * E;
      if constexpr (sizeof(T) == 2) {
        Four<T> v[kTerms<T>];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          T one[kTerms<T>];
          terms(acc[j][t][i] * by, one);
#pragma unroll
          for (int h = 0; h < kTerms<T>; ++h) v[h].v[i] = one[h];
        }
#pragma unroll
        for (int h = 0; h < kTerms<T>; ++h) *(Four<T>*)(out + h * 32 * E + g % 2 * 4) = v[h];
      } else {
        *(f4*)(out + g % 2 * 32 * E) = acc[j][t];
      }
    }
  }
}

// The large product: (U W) of BT places x BN columns, sum in steps of 128 bytes.  Bound by the matrix units at the
// clock that the card holds under them, 1.6 to 1.85 GHz, and by the waits at the barriers (8192^3 in bf16: the units
// busy in 65% of the cycles at 1.57 GHz, fp32 4096^3 85% at 2.08, both under the profiler), so by what a product
// costs in power as well: 16 x 16 x 32 instructions instead of 32 x 32 x 16 took 876 instead of 909 us there.
// Against 8 waves of 128 x 64 on 256 x 256, 4 waves of 128 x 128 took 26% longer, 256 x 128 tiles alone 11%, and half
// steps with four or five tiles in LDS 3 to 6%.
struct Big {
  const void *U, *W, *G;
  int64_t ldu, ldw;
  int cu, cw;  // values of a row of U / of the sum in W that exist (W_KC: multiples of 16 bytes); zeros behind
  Rows rows;
  Order order;
  const float* by;
  const void* split;
  int N, nw, r, rp, splits, tiles_t, tiles_n;  // nw: columns of W as stored
  void* Y;
  int64_t ldy;
  float* part;  // splits > 1: partial sums instead of Y
  int ldp;
};

__device__ const uint4 g_zeros[1] = {};

// 16 bytes per lane from global memory to LDS, at `at` + 16 lane; s_waitcnt vmcnt waits for it.  In assembly, as
// the compiler waits for all such loads before a transposing read of LDS, whatever that reads.
__device__ __forceinline__ void to_lds(const void* from, unsigned at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from)
               : "memory", "m0");
}
template <class T>
__device__ __forceinline__ unsigned lds_address(T* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)p;
}

// Tiles in LDS, as chunks of 16 bytes.  Operands whose sum runs along memory:
// rows of 8 chunks, chunk c of row i at place c ^ (i / 2 % 8), so that any 16
// rows a fragment reads lie in 16 different places of 256 bytes.  Otherwise rows
// (of the sum) of all columns; the 32 (fp32: 128) bytes that a read takes from a
// row are moved by the row's number, so that the rows of one read fall on different banks.
template <class T, int kRowChunks>
__device__ __forceinline__ int swap_columns(int k) {  // in chunks
  if constexpr (sizeof(T) == 2) return ((k & 3) | (k >> 1 & 4)) * 2 % kRowChunks;
  else return (k >> 2 & 1) * 8 % kRowChunks;
}

// WT x WN waves share a tile in blocks of 16 x 16 (fp32: 32 x 32).  S tiles in
// LDS and two sets of fragments in registers: while one quarter of a tile is
// multiplied the next is read; when the last quarter is in registers the
// tile's place is loaded again, S - 1 tiles' time before the barrier that waits for it.
template <class T, bool W_KC, int BT, int BN, int WT, int WN, int S, bool SPLIT>
__global__ __launch_bounds__(WT * WN * 64) void big_kernel(Big a) {
  using Frag = typename Mma<T>::Frag;
  constexpr int E = Mma<T>::kE, BK = 8 * E;
  using Acc = typename Block<T>::Acc;
  constexpr int kB = Block<T>::kB, kLanes = 64 / kB, kParts = 8 / kLanes, kAcc = kB * kB / 64;
  constexpr int TT = BT / WT / kB, TN = BN / WN / kB;
  constexpr int kLoadU = BT / (WT * WN * 8), kLoadW = BN / (WT * WN * 8);
  constexpr int kRowChunks = BN / E;  // chunks in a row of W's tile if not W_KC
  __shared__ __attribute__((aligned(16))) T lds[S * (BT + BN) * BK];  // U's tiles, then W's

  // Workgroups go to the 8 XCDs in turn: each XCD gets neighbouring tiles, and those that run at a time (a 256 x
  // 256 tile or two smaller ones on each of 32 CUs) are kGroup tiles high and about as wide, so that its L2 reads few
  // operands for many tiles.
  constexpr int kGroup = BT == 256 ? 4 : 8;
  const int tiles = a.tiles_t * a.tiles_n, q = tiles / 8, rem = tiles % 8, xcd = blockIdx.x % 8;
  const int number = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + blockIdx.x / 8;
  const int band = number / (kGroup * a.tiles_n), in_band = number % (kGroup * a.tiles_n);
  const int high = min(kGroup, a.tiles_t - band * kGroup);
  const int t0 = (band * kGroup + in_band % high) * BT, n0 = in_band / high * BN;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, lb = lane % kB, g = lane / kB;
  const int wt = wave / WN * (BT / WT), wn = wave % WN * (BN / WN);

  const int nk = (max(a.cu, a.cw) + BK - 1) / BK;
  const int k0 = SPLIT ? (int)((int64_t)nk * blockIdx.y / a.splits) : 0;
  const int k1 = SPLIT ? (int)((int64_t)nk * (blockIdx.y + 1) / a.splits) : nk;

  // what each lane loads: row of U / chunk along the sum, and the same of W
  const T *up[kLoadU], *wp[kLoadW];
  int uk[kLoadU], wk[kLoadW];
#pragma unroll
  for (int q = 0; q < kLoadU; ++q) {
    const int i = (wave * kLoadU + q) * 8 + lane / 8;
    uk[q] = ((lane % 8) ^ (i >> 1 & 7)) * E;
    up[q] = (const T*)a.U + row_at(a.order, min(t0 + i, a.rows.T - 1)) * a.ldu + uk[q];
  }
#pragma unroll
  for (int q = 0; q < kLoadW; ++q) {
    if constexpr (W_KC) {
      const int i = (wave * kLoadW + q) * 8 + lane / 8;
      wk[q] = ((lane % 8) ^ (i >> 1 & 7)) * E;
      wp[q] = (const T*)a.W + (int64_t)min(n0 + i, a.N - 1) * a.ldw + wk[q];
    } else {
      const int place = (wave * kLoadW + q) * 64 + lane, k = place / kRowChunks;
      const int n = min(n0 + ((place % kRowChunks) ^ swap_columns<T, kRowChunks>(k)) * E, a.nw - E);
      wk[q] = k;
      wp[q] = (const T*)a.W + (int64_t)k * a.ldw + n;
    }
  }
  const int64_t w_step = W_KC ? BK : BK * a.ldw;
  // W not along the sum: loads whose rows' columns are swapped alike differ by whole rows, so one address serves them
  constexpr int kLoadRows = W_KC ? 1 : 64 / kRowChunks;
  auto twin = [](int q) constexpr {
    if (W_KC) return q;
    for (int p = 0; p < q; ++p)
      if (sizeof(T) == 2 ? ((p ^ q) * kLoadRows & 11) == 0 : ((p ^ q) * kLoadRows & 4) == 0) return p;
    return q;
  };
  // the q-th load of a tile; guard: with zeros behind the sum's end, also for tiles that nothing uses
  auto load = [&](auto guard, int kt, int stage, int q) {
    const int k = kt * BK;
    const void* from;
    unsigned to;
    if (q < kLoadU) {
      from = up[q] + k;
      if (decltype(guard)::value && k + uk[q] >= a.cu) from = g_zeros;
      to = lds_address(lds + stage * BT * BK + (wave * kLoadU + q) * 64 * E);
    } else {
      q -= kLoadU;
      from = wp[twin(q)] + (kt * w_step + (q - twin(q)) * kLoadRows * a.ldw);
      if (decltype(guard)::value && k + wk[q] >= a.cw) from = g_zeros;
      to = lds_address(lds + (S * BT + stage * BN) * BK + (wave * kLoadW + q) * 64 * E);
    }
    to_lds(from, __builtin_amdgcn_readfirstlane(to));
  };

  Acc acc[TN][TT] = {}, total[sizeof(T) == 4 ? TN : 1][TT] = {};
  // Where this lane's fragments begin in a tile.  A step along the sum (of kParts) moves the chunk's number by an
  // exclusive or, which the swap above leaves alone, or the row; a block of W's columns moves their number in the same
  // way, as a wave's columns begin at a multiple of their number; the rest are constant distances.
  const int u_at = (wt + lb) * BK + (g ^ (lb >> 1 & 7)) * E;
  int w_at;  // of the wave's first block
  if constexpr (W_KC) {
    w_at = (wn + lb) * BK + (g ^ (lb >> 1 & 7)) * E;
  } else {
    const int n = wn + (sizeof(T) == 2 ? lane % 4 * 4 : lb);
    const int k = sizeof(T) == 2 ? g * 8 + lane % 16 / 4 : g * 4;
    w_at = k * BN + ((n / E) ^ swap_columns<T, kRowChunks>(k)) * E + n % E;
  }
  w_at += S * BT * BK;
  asm("" : "+v"(w_at));  // one number: from U's first tile on, W's are too far away for an instruction's offset
  auto read_x = [&](int stage, int part, int t) {
    return *(const Frag*)&lds[stage * BT * BK + (u_at ^ (part * kLanes * E)) + t * kB * BK];
  };
  auto read_w = [&](int stage, int part, int j) {
    const int ws = stage * BN * BK;
    if constexpr (W_KC) {
      return *(const Frag*)&lds[ws + (w_at ^ (part * kLanes * E)) + j * kB * BK];
    } else if constexpr (sizeof(T) == 2) {
      // 16 lanes read 4 rows (of the sum) x 16 columns, 8 bytes each, and get their column's 4 values
      s8 v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4*)&lds[ws + (w_at ^ (j * kB)) + (part * kLanes * E + h * 4) * BN]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h * 4 + e] = r[e];
      }
      return __builtin_bit_cast(Frag, v);
    } else {
      Frag v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = lds[ws + (w_at ^ (j * kB)) + (part * kLanes * E + e) * BN];
      return v;
    }
  };
  // A step along the sum in one or two halves of the wave's rows, x[0] and x[1] in turn.  While one half is multiplied
  // the next is read; with the last half of a step each fragment of W is read for the next step right after its last
  // use (one half: into the other of two sets), so that it has as long to arrive.
  constexpr int kMma = TT * TN, kLoads = kLoadU + kLoadW;
  constexpr int TH = TT > 1 ? TT / 2 : 1, kHalves = TT / TH, kSetsW = kHalves == 1 ? 2 : 1, kSubs = kParts * kHalves;
  Frag x[2][TH], w[kSetsW][TN];
  // the sub-th half of a tile's; then, in this order, what follows is read, and with `loads` a tile is loaded
  auto half = [&](int sub, int stage, auto loads, auto guard, int kt, int to) {
    const int h = sub % kHalves, next = (sub + 1) % kSubs, part = next / kHalves;
    const int set = sub / kHalves % kSetsW, set_next = part % kSetsW;
#pragma unroll
    for (int m = 0; m < TN * TH; ++m) {
      constexpr int kAll = TN * TH, kSpan = (kAll + 1) / 2;
      const int j = m / TH, i = m % TH;
#pragma unroll
      for (int q = 0; q < TH; ++q)
        if (q * kSpan / TH == m) x[(sub + 1) % 2][q] = read_x(stage, part, next % kHalves * TH + q);
      if (kSetsW == 2)
#pragma unroll
        for (int q = 0; q < TN; ++q)
          if (q * kSpan / TN == m) w[set_next][q] = read_w(stage, part, q);
      if constexpr (decltype(loads)::value)
#pragma unroll
        for (int q = 0; q < kLoads; ++q)
          if (q * kAll / kLoads == m) load(guard, kt, to, q);
      acc[j][h * TH + i] = Block<T>::mma(w[set][j], x[sub % 2][i], acc[j][h * TH + i]);
      if (kSetsW == 1 && h == kHalves - 1 && i == TH - 1) w[0][j] = read_w(stage, part, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // one tile from its place in LDS; its first half and W are in registers, and the next tile's will be
  auto step = [&](auto guard, int kt, int stage) {
    constexpr std::false_type no{};
#pragma unroll
    for (int sub = 0; sub < kSubs - 1; ++sub) half(sub, stage, no, no, 0, 0);
    // this wave's loads of the next tile have landed (only S - 2 tiles' may be under way) and its reads are done,
    // then everybody's
    constexpr int kAway = (S - 2) * kLoads;
    static_assert(kAway < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt(0x0070 | (kAway & 15) | (kAway >> 4) << 14);
    __syncthreads();
    half(kSubs - 1, (stage + 1) % S, std::true_type{}, guard, kt + S, stage);
  };
#pragma unroll
  for (int st = 0; st < S; ++st)
#pragma unroll
    for (int q = 0; q < kLoads; ++q) load(std::true_type{}, k0 + st, st, q);
  unsigned wrong = 0;  // rows of this lane whose adapter does not exist
  {
    // this lane's rows, and their adapters
    int row[TT], mine[TT], slot[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) row[t] = (int)row_at(a.order, min(t0 + wt + t * kB + lb, a.rows.T - 1));
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      mine[t] = adapter_of(a.rows, row[t]);
      if (t0 + wt + t * kB + lb >= a.rows.T) mine[t] = -1;
      wrong |= (unsigned)(mine[t] < -1 || mine[t] >= a.rows.n) << t;
      slot[t] = mine[t];
    }
    if (a.order.packed)
#pragma unroll
      for (int t = 0; t < TT; ++t)
        if (mine[t] >= 0 && mine[t] < a.rows.n) slot[t] = packed_slot(mine[t], a.order.start[mine[t]]);
    // The accumulators begin with s_i (U F_i) G_i, while the first tiles load (SPLIT: each part of the sum with some
    // of the adapters and ranks).  U F_i comes as three values of the type (fp32: itself); the loads of kSets steps
    // are under way at a time.  A row without this adapter loads its own garbage, which reaches that row's
    // accumulators alone, and these are set afterwards.
    auto has = [&](int t) { return mine[t] >= 0 && mine[t] < a.rows.n; };
    auto place = [&](int t) { return (int64_t)min(t0 + wt + t * kB + lb, a.rows.T - 1); };
    // the fragments that the low-rank pass and the first launch wrote, of 32 places or columns and 8 ranks.  Such a
    // block is a slot, with 16-bit types one for each of its terms; these types' instructions take four slots, one by
    // each group of 16 lanes.  A slot behind the last is zeros on both sides.
    constexpr int kSlots = sizeof(T) == 2 ? 4 : 1;
    const int slots = (a.r + 7) / 8 * kTerms<T>;
    auto x_of = [&](int t, int b) {
      const int at = t0 + wt + t * kB;
      const int64_t first = (int64_t)min(at / 32, (a.rows.T - 1) / 32) * (a.rp / 8) * kTerms<T>;
      if constexpr (sizeof(T) == 2) {
        const Frag v = ((const Frag*)a.split)[(first + min(b + g, slots - 1)) * 32 + at % 32 + lb];
        return b + g < slots ? v : Frag{};
      } else return ((const Frag*)a.split)[(first + b) * 64 + lane];
    };
    auto w_of = [&](int slot, int j, int b) {
      const int n = n0 + wn + j * kB;
      const int64_t blocks = (a.N + 31) / 32, block = min((int64_t)n / 32, blocks - 1);
      const int64_t first = (slot * blocks + block) * (a.rp / 8);
      if constexpr (sizeof(T) == 2) {
        const Frag v = ((const Frag*)a.G)[(first + (unsigned)min(b + g, slots - 1) / kTerms<T>) * 32 + n % 32 + lb];
        return b + g < slots ? v : Frag{};
      } else return ((const Frag*)a.G)[(first + b) * 64 + lane];
    };
    auto factor = [&](int t, int cur) {
      float f = scale_of(a.rows, cur);
      if constexpr (std::is_same_v<T, _Float16>) f *= has(t) ? a.by[place(t)] : 0.f;
      return f;
    };
    constexpr int kSets = (sizeof(T) == 2 ? 1 : 2) * (TT * TN * kB * kB <= 1024 ? 2 : 1);  // by the registers
    const int shares = SPLIT ? a.splits : 1, share = SPLIT ? blockIdx.y : 0;
    uint64_t some[TT], any = 0;
    int first = -1, first_slot = 0;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      some[t] = __ballot(has(t));
      if (some[t] && !any) {
        first = __builtin_amdgcn_readlane(mine[t], __builtin_ctzll(some[t]));
        first_slot = __builtin_amdgcn_readlane(slot[t], __builtin_ctzll(some[t]));
      }
      any |= some[t];
    }
    bool one = true;
#pragma unroll
    for (int t = 0; t < TT; ++t) one = one && __ballot(has(t) && mine[t] != first) == 0;
    if (any && one) {
      // one adapter among all of the wave's rows: straight into the accumulators, zeros again where it is no row's
      Frag x[kSets][TT], w[kSets][TN];
      auto fetch = [&](int q, int b) {
        if (b >= slots) return;
#pragma unroll
        for (int t = 0; t < TT; ++t) x[q][t] = x_of(t, b);
#pragma unroll
        for (int j = 0; j < TN; ++j) w[q][j] = w_of(first_slot, j, b);
      };
#pragma unroll
      for (int q = 0; q < kSets; ++q) fetch(q, (share + q * shares) * kSlots);
      for (int b = share * kSlots; b < slots; b += kSets * shares * kSlots)
#pragma unroll
        for (int q = 0; q < kSets; ++q) {
          if (b + q * shares * kSlots < slots)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int t = 0; t < TT; ++t) acc[j][t] = Block<T>::mma(w[q][j], x[q][t], acc[j][t]);
          fetch(q, b + (kSets + q) * shares * kSlots);
        }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const float f = factor(t, first);
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < kAcc; ++r) acc[j][t][r] = has(t) ? f * acc[j][t][r] : 0.f;
      }
    } else if (any) {
      // for each adapter among a block's rows the product of all of them, kept where it is theirs
      int unit = shares - share;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        uint64_t left = some[t];
        while (left) {
          const int lead = __builtin_ctzll(left), cur = __builtin_amdgcn_readlane(mine[t], lead);
          const int cur_slot = __builtin_amdgcn_readlane(slot[t], lead);
          left &= ~__ballot(mine[t] == cur);
          Acc d[TN] = {};
          for (int b = 0; b < slots; b += kSlots * kSets) {
            if (SPLIT && unit++ % shares != 0) continue;
            Frag x[kSets], w[TN][kSets];
#pragma unroll
            for (int q = 0; q < kSets; ++q) {
              if (b + q * kSlots >= slots) continue;
              x[q] = x_of(t, b + q * kSlots);
#pragma unroll
              for (int j = 0; j < TN; ++j) w[j][q] = w_of(cur_slot, j, b + q * kSlots);
            }
#pragma unroll
            for (int q = 0; q < kSets; ++q)
              if (b + q * kSlots < slots)
#pragma unroll
                for (int j = 0; j < TN; ++j) d[j] = Block<T>::mma(w[j][q], x[q], d[j]);
          }
          const float f = factor(t, cur);
          if (mine[t] == cur)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[j][t] = f * d[j];
        }
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < TH; ++q) x[0][q] = read_x(0, 0, q);
#pragma unroll
  for (int q = 0; q < TN; ++q) w[0][q] = read_w(0, 0, q);
  const int whole = min(k1, min(a.cu, a.cw) / BK);  // tiles without a part behind the end
  int kt = k0;
  for (; kt + 2 * S - 1 < whole; kt += S) {
#pragma unroll
    for (int st = 0; st < S; ++st) step(std::false_type{}, kt + st, st);
    if constexpr (sizeof(T) == 4) {
      // fp32: sums of about 512 values, then of those, or the rounding of one long sum would grow with its length
      constexpr int kLong = 512 / (S * BK);
      if ((kt - k0) / S % kLong == kLong - 1)
#pragma unroll
        for (int m = 0; m < kMma; ++m) {
          total[m / TT][m % TT] += acc[m / TT][m % TT];
          acc[m / TT][m % TT] = Acc{};
        }
    }
  }
  for (; kt < k1; kt += S)
#pragma unroll
    for (int st = 0; st < S; ++st)
      if (kt + st < k1) step(std::true_type{}, kt + st, st);
  if constexpr (sizeof(T) == 4)
#pragma unroll
    for (int m = 0; m < kMma; ++m) acc[m / TT][m % TT] += total[m / TT][m % TT];
  // No load may land in LDS from here on.  Each wave turns its part of the tile there, in chunks of 16 bytes
  // moved by the row's number, and writes whole rows of it: straight from the accumulators a store would reach 16
  // bytes of each of 32 rows.
  __builtin_amdgcn_s_waitcnt(0x0070);
  __syncthreads();
  using Out = std::conditional_t<SPLIT, float, T>;
  constexpr int EO = 16 / sizeof(Out), kRowOut = BN / WN / EO, kHigh = BT / WT;  // chunks of a row, rows
  static_assert(WT * WN * kHigh * kRowOut * 16 <= (int)sizeof(lds), "turned tile");
  Out* mem = (Out*)lds + wave * kHigh * kRowOut * EO;
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int i = t * kB + lb;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      Acc v = acc[j][t];
      if (!SPLIT && (wrong >> t & 1)) v = v * __builtin_nanf("");
#pragma unroll
      for (int r = 0; r < kAcc; r += 4) {
        const int n = j * kB + r * 2 + g * 4;
        *(Four<Out>*)(mem + (i * kRowOut + ((n / EO) ^ (i % kRowOut))) * EO + n % EO) =
            Four<Out>{(Out)v[r], (Out)v[r + 1], (Out)v[r + 2], (Out)v[r + 3]};
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  constexpr int kAtOnce = 64 / kRowOut;  // rows of a store
#pragma unroll
  for (int q = 0; q < kHigh / kAtOnce; ++q) {
    const int i = q * kAtOnce + lane / kRowOut, c = lane % kRowOut;
    typedef Out Chunk __attribute__((ext_vector_type(EO)));
    const Chunk v = *(const Chunk*)(mem + (i * kRowOut + (c ^ (i % kRowOut))) * EO);
    const int at = t0 + wt + i, n = n0 + wn + c * EO;
    if (at >= a.rows.T) continue;
    if constexpr (SPLIT) {
      *(Chunk*)(a.part + ((int64_t)blockIdx.y * a.rows.T + at) * a.ldp + n) = v;
    } else {
      struct __attribute__((packed, aligned(sizeof(Out)))) Any {
        Chunk v;
      };
      Out* out = (Out*)a.Y + row_at(a.order, at) * a.ldy + n;
      if (n + EO <= a.N) ((Any*)out)->v = v;
      else
#pragma unroll
        for (int e = 0; e < EO; ++e)
          if (n + e < a.N) out[e] = v[e];
    }
  }
}

// The factors' gradients (4096 rows, 4096 + 4096 columns, rank 16, bf16: 22 us, U at 3.0 TB/s): sum over the
// places of an adapter of U_t^T V_t, V = S or D, in pieces of `size` places (32 to kGradRows: with few rows smaller
// ones, for enough workgroups, but not so small that the parts, a rank's 4 bytes a column each, outweigh U's).  A
// workgroup takes 64 kE columns of U, a wave 16 kE, whose rows it turns in registers.  V is turned on its way to
// LDS, as the sum of three values of the type (fp16: brought to below 2^14 by the piece's power of two).  Bound by
// reading U once: each wave keeps two steps' rows in flight.
constexpr int kGradRows = 128;
struct Outer {
  const void* U;
  int64_t ldu;
  const float* low;  // V
  float* part;       // part, rank, column
  int cu, ldp, blocks;
  // for adapters of one piece: the gradient itself, at adapter as + column cs + rank rs
  void* out;
  int64_t as, cs, rs;
  int cols;
};
struct OuterPair {
  Outer p[2];
  Rows rows;
  Order order;
  const Piece* table;
  int rp, pieces, size, r;
};
// Adapters of one piece write their gradients at once, the others parts that are added up.  Such an adapter i has more
// than `size` rows, so its parts have the numbers from start / size + min(i, start / size) on, as its pieces have theirs:
// no more than T / size + min(n, T / size).
__device__ __forceinline__ int first_part(int start, int i, int size) { return start / size + min(i, start / size); }
int parts_of(int64_t T, int64_t n, int size) { return (int)(T / size + std::min(n, std::max<int64_t>(1, T / size))); }
// all of adapter i's rows as one piece
__device__ __forceinline__ Piece whole_of(const Order& o, const Rows& g, int i) {
  if (!o.start) return {0, 0, g.T, 0};
  return {i, o.start[i], o.start[i + 1] - o.start[i], 0};
}

// BY_ADAPTER: with at most `size` rows a piece for each adapter, also for those without rows, whose gradients are zeros
template <class T, int RB, bool BY_ADAPTER>
__global__ __launch_bounds__(256) void outer_kernel(OuterPair both) {
  using M = Mma<T>;
  using Frag = typename M::Frag;
  constexpr int E = M::kE, kRanks = RB * 16, kPitch = kGradRows + 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) T vs[kTerms<T>][kRanks][kPitch];
  __shared__ int32_t row[kGradRows];
  __shared__ float wave_most[4];
  const Outer& a = both.p[blockIdx.y];
  const int piece = blockIdx.x % both.pieces, block = blockIdx.x / both.pieces;
  if (block >= a.blocks) return;
  const Piece pc =
      BY_ADAPTER ? whole_of(both.order, both.rows, piece) : piece_of(both.table, both.rows, piece, both.size);
  if (!BY_ADAPTER && pc.count == 0) return;
  const Piece all = whole_of(both.order, both.rows, pc.adapter);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, l16 = lane % 16, g = lane / 16;
  const int j0 = blockIdx.z * kRanks;
  if (threadIdx.x < kGradRows)
    row[threadIdx.x] = pc.count ? (int32_t)row_at(both.order, pc.begin + min((int)threadIdx.x, pc.count - 1)) : 0;
  __syncthreads();
  const int n0 = (block * 4 + wave) * 16 * E, n = n0 + l16 * E;
  const T* U = (const T*)a.U + n;
  constexpr int kFlight = 2;
  Frag in[kFlight][E];
  auto fetch = [&](int s) {
#pragma unroll
    for (int q = 0; q < kFlight; ++q)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int t = (s + q) * M::kStep + g * E + e;
        in[q][e] = Frag{};
        if (t < pc.count && n < a.cu) in[q][e] = *(const Frag*)(U + row[t] * a.ldu);
      }
  };
  fetch(0);  // while V is laid out
  // V: thread (place, every other 4 ranks)
  constexpr int kMine = kRanks / 8;
  const int t = threadIdx.x / 2;
  f4 v[kMine];
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    v[q] = f4{0.f, 0.f, 0.f, 0.f};
    if (t < pc.count) v[q] = *(const f4*)(a.low + (int64_t)(pc.begin + t) * both.rp + j0 + q * 8 + threadIdx.x % 2 * 4);
  }
  float by = 1.f, back = 1.f;
  if constexpr (std::is_same_v<T, _Float16>) {
    float most = 0.f;
#pragma unroll
    for (int q = 0; q < kMine; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = fabsf(v[q][e]);
        if (x > most && x <= 3.4e38f) most = x;
      }
#pragma unroll
    for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    if (lane == 0) wave_most[wave] = most;
    __syncthreads();
    most = fmaxf(fmaxf(wave_most[0], wave_most[1]), fmaxf(wave_most[2], wave_most[3]));
    const int e = to_fp16_range(most);
    by = ldexpf(1.f, e);
    back = ldexpf(1.f, -e);
  }
#pragma unroll
  for (int q = 0; q < kMine; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = q * 8 + threadIdx.x % 2 * 4 + e;
      T one[kTerms<T>];
      terms(v[q][e] * by, one);
#pragma unroll
      for (int h = 0; h < kTerms<T>; ++h) vs[h][j][t] = one[h];
    }
  __syncthreads();
  if (n0 >= a.cu) return;
  f4 acc[E][RB] = {};
  for (int s = 0;;) {
#pragma unroll
    for (int q = 0; q < kFlight; ++q) {
      Frag w[E];
      turn<T>(in[q], w);
#pragma unroll
      for (int h = 0; h < kTerms<T>; ++h)
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const Frag x = *(const Frag*)&vs[h][b * 16 + l16][(s + q) * M::kStep + g * E];
#pragma unroll
          for (int j = 0; j < E; ++j) acc[j][b] = M::mma(w[j], x, acc[j][b]);
        }
    }
    s += kFlight;
    if (s * M::kStep >= pc.count) break;
    fetch(s);
  }
  if (BY_ADAPTER || all.count <= both.size) {
    // an adapter without rows gets zeros, whatever its factor holds
    const float f = pc.count ? scale_of(both.rows, pc.adapter) * back : 0.f;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int j = j0 + b * 16 + l16;
      if (j >= both.r) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = n0 + (g * 4 + i) * E;
        T* out = (T*)a.out + pc.adapter * a.as + c * a.cs + j * a.rs;
        Unaligned<T> v;
#pragma unroll
        for (int e = 0; e < E; ++e) v.v[e] = (T)(f * acc[e][b][i]);
        if (a.cs == 1 && c + E <= a.cols) *(Unaligned<T>*)out = v;
        else
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (c + e < a.cols) out[e * a.cs] = v.v[e];
      }
    }
    return;
  }
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int part = first_part(all.begin, pc.adapter, both.size) + (pc.begin - all.begin) / both.size;
    float* out = a.part + ((int64_t)part * both.rp + j0 + b * 16 + l16) * a.ldp + n0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < E; j += 4)
        *(f4*)(out + (g * 4 + i) * E + j) =
            back * f4{acc[j][b][i], acc[j + 1][b][i], acc[j + 2][b][i], acc[j + 3][b][i]};
  }
}

// Last the sums of the parts, times s_i, in the factor's layout, and zeros for adapters without rows: 64 columns of
// one adapter by a workgroup, whose four waves share the pieces of 4 ranks or, where the adapters have few pieces,
// take 4 ranks each.
struct Sum {
  const float* part;
  void* out;
  int64_t as, cs, rs;  // adapter, column, rank
  int cols, ldp, blocks;
};
struct SumPair {
  Sum p[2];
  Rows rows;
  Order order;
  int r, rp, size;
};

template <class T, bool SHARE>
__global__ __launch_bounds__(256) void sum_kernel(SumPair both) {
  __shared__ f4 lds[3][64];
  const Sum& a = both.p[blockIdx.y];
  if ((int)blockIdx.x >= a.blocks) return;
  constexpr int kRanks = SHARE ? 4 : 16;
  const int groups = (both.r + kRanks - 1) / kRanks, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int c = blockIdx.x / groups * 64 + lane, j0 = blockIdx.x % groups * kRanks + (SHARE ? 0 : wave * 4);
  for (int i = blockIdx.z; i < both.rows.n; i += gridDim.z) {
    const Piece all = whole_of(both.order, both.rows, i);
    const int count = all.count, many = (count + both.size - 1) / both.size;
    if (many == 1) continue;  // written already
    const int first = first_part(all.begin, i, both.size);
    f4 s = {0.f, 0.f, 0.f, 0.f};
    if (j0 < both.rp)
#pragma unroll 4
      for (int p = SHARE ? wave : 0; p < many; p += SHARE ? 4 : 1) {
        const float* from = a.part + ((int64_t)(first + p) * both.rp + j0) * a.ldp + c;
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from[e * (int64_t)a.ldp];
        s += v;
      }
    if constexpr (SHARE) {
      if (wave) lds[wave - 1][lane] = s;
      __syncthreads();
      s += lds[0][lane] + lds[1][lane] + lds[2][lane];
    }
    if ((!SHARE || wave == 0) && c < a.cols) {
      s = s * (count ? scale_of(both.rows, i) : 0.f);  // without rows zeros, whatever the factor holds
      T* out = (T*)a.out + i * a.as + c * a.cs + j0 * a.rs;
      if (a.rs == 1 && j0 + 4 <= both.r) {
        *(Four<T>*)out = Four<T>{(T)s[0], (T)s[1], (T)s[2], (T)s[3]};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j0 + e < both.r) out[e * a.rs] = (T)s[e];
      }
    }
    if constexpr (SHARE) __syncthreads();
  }
}

// ---- host -----------------------------------------------------------------

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

int check_shape(const gelim_adapter_args& a) {
  if (a.dtype < GELIM_T_F32 || a.dtype > GELIM_T_F16) return GELIM_FAIL(GELIM_E_ARG, "adapter: unknown type");
  if (a.T < 0 || a.K <= 0 || a.N <= 0 || a.r <= 0 || a.n <= 0) return GELIM_FAIL(GELIM_E_ARG, "adapter: bad shape");
  if (a.T > GELIM_ADAPTER_MAX_DIM || a.K > GELIM_ADAPTER_MAX_DIM || a.N > GELIM_ADAPTER_MAX_DIM || a.n > 65535)
    return GELIM_FAIL(GELIM_E_ARG, "adapter: dimension too large");
  if (a.r > GELIM_ADAPTER_MAX_RANK) return GELIM_FAIL(GELIM_E_ARG, "adapter: rank above 256");
  return GELIM_OK;
}

int check(const gelim_adapter_args& a, bool grad) {
  GELIM_TRY(check_shape(a));
  if (!a.index && a.n != 1 && a.T)
    return GELIM_FAIL(GELIM_E_ARG, "adapter: an index is needed with more than one adapter");
  if (!a.W || !a.A || !a.B || (a.T && (!a.X || !a.Y))) return GELIM_FAIL(GELIM_E_ARG, "adapter: null matrix");
  const int64_t need = gelim_adapter_workspace(&a, grad);
  if (need < 0) return (int)need;
  if (a.ws_bytes < need) return GELIM_FAIL(GELIM_E_ARG, "adapter: workspace too small");
  return GELIM_OK;
}

// Hands out the workspace; with a null base it only counts.
struct Space {
  char* base;
  int64_t used = 0, threads = 0;  // threads: of the largest launch
  unsigned launch(int64_t groups, int64_t block, int64_t across = 1) {
    threads = std::max(threads, groups * block * across);
    return (unsigned)groups;
  }
  template <class P>
  P* take(int64_t count) {
    P* p = (P*)(base + used);
    used += up(count * (int64_t)sizeof(P), 256);
    return p;
  }
};

constexpr int kFewRows = 64;

// Y (T x N) = U (T x C) W (C x N) + s_i (U F_i) G_i
struct Problem {
  const void* U;
  int64_t ldu;
  int C, N;
  View W, F, G;
  bool w_kc;
  void* Y;
  int64_t ldy;
};

View turned(View v) { return {v.p, v.as, v.cs, v.rs}; }
View view_w(const gelim_adapter_args& a) { return {a.W, 0, a.w_trans ? 1 : a.ldw, a.w_trans ? a.ldw : 1}; }
View view_a(const gelim_adapter_args& a) { return {a.A, a.a_stride, a.a_trans ? 1 : a.lda, a.a_trans ? a.lda : 1}; }
View view_b(const gelim_adapter_args& a) { return {a.B, a.b_stride, a.b_trans ? 1 : a.ldb, a.b_trans ? a.ldb : 1}; }
Rows rows_of(const gelim_adapter_args& a) { return {a.index, a.scale, (float)a.scale_value, (int)a.n, (int)a.T}; }
Problem product_of(const gelim_adapter_args& a) {
  return {a.X, a.ldx, (int)a.K, (int)a.N, view_w(a), view_a(a), view_b(a), a.w_trans != 0, a.Y, a.ldy};
}
Problem back_of(const gelim_adapter_args& a) {
  return {a.Y, a.ldy, (int)a.N, (int)a.K, turned(view_w(a)), turned(view_b(a)), turned(view_a(a)), a.w_trans == 0,
          a.dX, a.lddx};
}

int rank_blocks(int64_t r) {  // of 16, a power of two
  int b = 1;
  while (16 * b < r) b *= 2;
  return b;
}

// -- few rows

template <class T>
int few_product(const Problem& p, const Rows& g, int r, Space& ws, hipStream_t s, bool run) {
  using M = Mma<T>;
  Few f{};
  f.U = p.U, f.ldu = p.ldu, f.W = p.W, f.F = p.F, f.rows = g, f.C = p.C, f.N = p.N, f.r = r;
  f.blocks = (int)((p.N + 16 * M::kE - 1) / (16 * M::kE));
  const int steps = (p.C + M::kStep - 1) / M::kStep;
  // workgroups: one a CU, as more cost the second launch what they save (32 rows of bf16 4096 x 4096: 16.2 us
  // with 256, 17.8 with 512); two for fp32 in rows of N, where a wave has half as many loads under way (8 x 2048
  // x 7168: 22.5 us with 256, 17.9 with 512; with W along the sum 60 x 1000 x 2000 takes 14.8 and 17.4)
  const int groups = sizeof(T) == 4 && !p.w_kc ? 512 : 256;
  f.splits = std::clamp(groups / f.blocks, 1, std::max(1, std::min(64, steps / 4)));
  f.low_splits = std::clamp(256 / g.T, 1, std::max(1, std::min(16, p.C / 256)));
  f.ldp = f.blocks * 16 * M::kE;
  f.part = ws.take<float>((int64_t)f.splits * g.T * f.ldp);
  f.low = ws.take<float>((int64_t)f.low_splits * g.T * r);
  const dim3 grid(ws.launch((int64_t)f.blocks * f.splits + g.T * f.low_splits, 256));
  Finish e{f.part, f.low, p.G, g, nullptr, p.N, r, f.ldp, f.splits, f.low_splits, r, (p.N + 255) / 256,
           p.Y, p.ldy};
  ws.launch(finish_groups(e), 256);
  if (!run) return GELIM_OK;
  const int tt = (g.T + 15) / 16;
  auto launch = [&](auto kc) {
    constexpr bool KC = decltype(kc)::value;
    if (tt == 1) hipLaunchKernelGGL((few_kernel<T, KC, 1>), grid, dim3(256), 0, s, f);
    else if (tt == 2) hipLaunchKernelGGL((few_kernel<T, KC, 2>), grid, dim3(256), 0, s, f);
    else hipLaunchKernelGGL((few_kernel<T, KC, 4>), grid, dim3(256), 0, s, f);
  };
  if (p.w_kc) launch(std::true_type{});
  else launch(std::false_type{});
  finish<T>(e, s);
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
}

// -- many rows

template <class T>
struct Many {
  static constexpr int E = Mma<T>::kE;
  const gelim_adapter_args& a;
  Rows g;
  int rb, rp;
  Prepare prep{};
  Order order{};
  int64_t groups = 0;
  Space& ws;

  Many(const gelim_adapter_args& args, Space& space) : a(args), g(rows_of(args)), ws(space) {
    rb = rank_blocks(a.r);
    rp = 16 * rb;
    prep.rows = g;
    if (a.index && a.T) {
      prep.perm = ws.template take<int32_t>(a.T);
      prep.start = ws.template take<int32_t>(a.n + 1);
      prep.order_groups = (int)a.n + 1;
      prep.packed = a.n > a.T && a.n > kScanAdapters && a.T <= kScanRows;
      order = {prep.perm, prep.start, prep.packed};
      set_pieces(0, kLowRows);
    }
    groups = prep.order_groups;
    prep.counter = ws.template take<int>(2 * pieces(a.T, a.n, a.index != nullptr, kLowRows));
  }

  // a table of pieces of that size, if there is an order at all
  void set_pieces(int k, int size) {
    if (a.index) prep.pieces[k] = {ws.template take<Piece>(pieces(a.T, a.n, true, size)), size};
  }
  T* copy(View src, int rows, int have, int cols, int ld, int count, int order = kRows) {
    Copy& c = prep.copy[prep.copies++];
    const int64_t tiles = (int64_t)((rows + kCopyTile - 1) / kCopyTile) * ((ld + kCopyTile - 1) / kCopyTile);
    const int64_t per = std::clamp<int64_t>(count * tiles / 4096, 1, tiles);  // tiles of a workgroup: 16 of them a CU
    const int64_t slots = prep.packed ? std::min<int64_t>(count, a.T) : count;
    c = {src, ws.template take<T>(slots * rows * ld), rows, cols, ld, count, have, order,
         order == kRows && src.cs == 1, (int)groups - prep.order_groups, (int)tiles, (int)per};
    groups += c.straight ? ((int64_t)count * rows * (ld / E) + kStraight - 1) / kStraight
                         : count * ((tiles + per - 1) / per);
    ws.launch(groups, kPrepare);
    return (T*)c.dst;
  }
  static bool aligned(const void* p, int64_t ld, int64_t len) {
    return (uintptr_t)p % 16 == 0 && ld % E == 0 && len % E == 0;
  }
  // rows of U as 16-byte chunks: as they are, or copied
  struct Wide {
    const void* p;
    int64_t ld;
    int cols;  // that may be read
  };
  Wide wide(const void* p, int64_t ld, int64_t rows, int cols) {
    if (aligned(p, ld, cols)) return {p, ld, cols};
    const int to = (int)up(cols, 64);
    return {copy({p, 0, ld, 1}, (int)rows, (int)rows, cols, to, 1), to, to};
  }

  // F laid out for the low product: ranks x the sum
  Low low_of(const Wide& U, View F, int C) {
    Low l{};
    l.ldf = (int)up(C, 64);
    l.F = copy(turned(F), rp, (int)a.r, C, l.ldf, (int)a.n, kFrag16);
    l.U = U.p, l.ldu = U.ld, l.cu = U.cols;
    l.pieces = pieces(a.T, a.n, a.index != nullptr, kLowRows);
    l.low = ws.template take<float>(a.T * rp);
    const int steps = (C + Mma<T>::kStep - 1) / Mma<T>::kStep;
    // cut the sum where that leaves a wave a round of loads or more
    l.splits = std::clamp(256 / std::max(1, l.pieces), 1, std::clamp(steps / (kLowWaves * low_flight(rb)), 1, 16));
    ws.launch((int64_t)l.pieces * l.splits, kLowWaves * 64);
    if (l.splits > 1) {
      l.part = ws.template take<float>((int64_t)l.pieces * l.splits * kLowRows * rp);
      l.arrived = prep.counter + prep.counters;
      prep.counters += l.pieces;
    }
    l.split = ws.template take<T>(up(a.T, 32) * rp * kTerms<T>);
    if (std::is_same_v<T, _Float16>) l.by = ws.template take<float>(a.T);
    return l;
  }
  int run_prepare(hipStream_t s) {
    if (groups) hipLaunchKernelGGL(prepare_kernel<T>, dim3((unsigned)groups), dim3(kPrepare), 0, s, prep);
    return GELIM_OK;
  }
  void run_low(const Low* l, int count, hipStream_t s) {
    LowPair both{};
    both.rows = g, both.order = order, both.table = prep.pieces[0].table, both.r = (int)a.r;
    unsigned most = 0;
    for (int k = 0; k < count; ++k) {
      both.p[k] = l[k];
      most = std::max(most, (unsigned)(l[k].pieces * l[k].splits));
    }
    const dim3 grid(most, (unsigned)count);
    auto launch = [&](auto blocks) {
      constexpr int RB = decltype(blocks)::value;
      hipLaunchKernelGGL((low_kernel<T, RB>), grid, dim3(kLowWaves * 64), 0, s, both);
    };
    if (rb == 1) launch(std::integral_constant<int, 1>{});
    else if (rb == 2) launch(std::integral_constant<int, 2>{});
    else if (rb == 4) launch(std::integral_constant<int, 4>{});
    else if (rb == 8) launch(std::integral_constant<int, 8>{});
    else launch(std::integral_constant<int, 16>{});
  }

  // the large product
  struct Plan {
    Big b;
    bool kc;
    int bt, bn;
    Problem p;
  };
  // The tile by what it is expected to take: the rounds of 256 workgroups, or of 512 where two fit a CU, each of
  // a fixed part (a launch's share, the first loads, the low-rank part, the end) and the tiles' steps of 128
  // bytes along the sum, both as measured (us) with one workgroup a CU and with two.
  void choose(Plan& q, int nk) {
    struct Shape {
      int bt, bn;
      double fixed, step, fixed2, step2;  // step2 0: one fits
    };
    static constexpr Shape k16[] = {{256, 256, 16.7, 1.55, 0, 0}, {256, 128, 11.9, 0.84, 0, 0},
                                    {128, 128, 9.4, 0.50, 0, 0}, {64, 64, 5.6, 0.26, 5.2, 0.39}};
    static constexpr Shape k32[] = {{128, 128, 12.3, 2.26, 0, 0}, {128, 64, 9.7, 1.17, 10.0, 2.37},
                                    {64, 64, 6.5, 0.65, 6.0, 1.30}};
    double best = 1e30;
    auto look = [&](const Shape& h) {
      const int64_t tiles = ((a.T + h.bt - 1) / h.bt) * ((q.p.N + h.bn - 1) / h.bn);
      for (int splits = 1; splits <= 16 && (splits == 1 || (h.bn < 256 && nk / splits >= 4)); ++splits) {
        const int64_t groups = tiles * splits, steps = (nk + splits - 1) / splits;
        const double one = h.fixed + h.step * steps, two = h.fixed2 + h.step2 * steps;
        const int64_t rest = groups % 512;
        double us = (double)((groups + 255) / 256) * one;
        // a last round of less than a workgroup a CU: some CUs get two of them all the same, unless it is the only one
        const double last = rest > 256 ? two : rest ? (groups < 512 ? one : (one + two) / 2) : 0;
        if (h.step2 > 0) us = (double)(groups / 512) * two + last;
        // joining the parts: a launch, and reading them
        if (splits > 1) us += 3 + 0.6e-6 * (double)splits * a.T * q.p.N;
        if (us < best) best = us, q.bt = h.bt, q.bn = h.bn, q.b.splits = splits;
      }
    };
    if (sizeof(T) == 2)
      for (const Shape& h : k16) look(h);
    else
      for (const Shape& h : k32) look(h);
  }
  Finish joined(const Plan& q) const {
    const Big& b = q.b;
    return {b.part, nullptr, View{}, g, order.perm, b.N, 0, b.ldp, b.splits, 0, 0, (b.N + 255) / 256, b.Y, b.ldy};
  }
  Plan big_of(const Problem& p, const Wide& U) {
    Plan q{};
    Big& b = q.b;
    q.kc = p.w_kc;
    q.p = p;
    b.U = U.p, b.ldu = U.ld, b.cu = U.cols, b.rows = g, b.order = order, b.N = p.N, b.r = (int)a.r, b.rp = rp;
    b.Y = p.Y, b.ldy = p.ldy;
    if (p.w_kc) {
      const Wide w = wide(p.W.p, p.W.cs, p.N, p.C);
      b.W = w.p, b.ldw = w.ld, b.cw = w.cols;
    } else {
      const Wide w = wide(p.W.p, p.W.rs, p.C, p.N);
      b.W = w.p, b.ldw = w.ld, b.cw = p.C, b.nw = w.cols;
    }
    const int nk = (std::max(b.cu, b.cw) + 8 * E - 1) / (8 * E);
    choose(q, nk);
    b.tiles_t = (int)((a.T + q.bt - 1) / q.bt);
    b.tiles_n = (p.N + q.bn - 1) / q.bn;
    if (b.splits > 1) {
      b.ldp = b.tiles_n * q.bn;
      b.part = ws.template take<float>((int64_t)b.splits * a.T * b.ldp);
    }
    ws.launch((int64_t)b.tiles_t * b.tiles_n, q.bt * q.bn >= 256 * 128 ? 512 : 256, b.splits);
    if (b.splits > 1) ws.launch(finish_groups(joined(q)), 256);
    b.G = copy(turned(p.G), (int)up(p.N, 32), p.N, (int)a.r, rp, (int)a.n, kFrag32);
    return q;
  }
  template <bool KC, int BT, int BN, int WT, int WN, int S>
  void launch(const Big& b, hipStream_t s) {
    const dim3 grid((unsigned)(b.tiles_t * b.tiles_n), (unsigned)b.splits);
    if constexpr (BN < 256)
      if (b.splits > 1) {
        hipLaunchKernelGGL((big_kernel<T, KC, BT, BN, WT, WN, S, true>), grid, dim3(WT * WN * 64), 0, s, b);
        return;
      }
    hipLaunchKernelGGL((big_kernel<T, KC, BT, BN, WT, WN, S, false>), grid, dim3(WT * WN * 64), 0, s, b);
  }
  void run_big(Plan& q, const Low& l, hipStream_t s) {
    Big& b = q.b;
    b.by = l.by, b.split = l.split;
    auto shape = [&](auto kc) {
      constexpr bool KC = decltype(kc)::value;
      if (q.bt == 64) launch<KC, 64, 64, 2, 2, 4>(b, s);
      else if (q.bt == 128 && q.bn == 128) launch<KC, 128, 128, 2, 2, 4>(b, s);
      else if constexpr (sizeof(T) == 4) launch<KC, 128, 64, 2, 2, 3>(b, s);
      else if constexpr (sizeof(T) == 2) {
        if (q.bn == 128) launch<KC, 256, 128, 4, 2, 3>(b, s);
        else launch<KC, 256, 256, 2, 4, 2>(b, s);
      }
    };
    if (q.kc) shape(std::true_type{});
    else shape(std::false_type{});
    if (b.splits > 1) finish<T>(joined(q), s);
  }
};

template <class T>
int product(const gelim_adapter_args& a, Space& ws, hipStream_t s, bool run) {
  const Problem p = product_of(a);
  if (a.T == 0) return GELIM_OK;
  if (a.T <= kFewRows) return few_product<T>(p, rows_of(a), (int)a.r, ws, s, run);
  Many<T> m(a, ws);
  const auto U = m.wide(p.U, p.ldu, a.T, p.C);
  Low l = m.low_of(U, p.F, p.C);
  auto q = m.big_of(p, U);
  if (!run) return GELIM_OK;
  m.run_prepare(s);
  m.run_low(&l, 1, s);
  m.run_big(q, l, s);
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
}

template <class T>
int gradient(const gelim_adapter_args& a, Space& ws, hipStream_t s, bool run) {
  if (!a.dX && !a.dA && !a.dB) return GELIM_OK;
  // what the wanted results need, and nothing else: S for dB, D for the others, X for the factors' gradients
  const bool need_s = a.T && a.dB, need_d = a.T && (a.dX || a.dA), need_x = a.T && (a.dA || a.dB);
  Many<T> m(a, ws);
  const int K = (int)a.K, N = (int)a.N;
  typename Many<T>::Wide X{}, dY{};
  if (need_x) X = m.wide(a.X, a.ldx, a.T, K);
  if (a.T) dY = m.wide(a.Y, a.ldy, a.T, N);
  const Problem back = back_of(a);
  typename Many<T>::Plan q{};
  Low low[2];  // D, S
  if (need_d) low[0] = m.low_of(dY, back.F, N);
  if (need_s) low[1] = m.low_of(X, view_a(a), K);
  if (a.dX && a.T) q = m.big_of(back, dY);
  // the sides: dA = X^T D, dB^T = dY^T S
  int size = kGradRows;
  const bool direct = a.T > 0 && a.T <= size;  // no adapter has more than one piece: no parts to add up
  while (!direct && size > std::max(32, 2 * m.rp) && a.T / size * ((K + N) / (64 * Mma<T>::kE)) < 256) size /= 2;
  const int pcs = direct ? (int)a.n : pieces(a.T, a.n, a.index != nullptr, size);
  if (!direct) m.set_pieces(1, size);
  OuterPair op{};
  SumPair sp{};
  op.rows = sp.rows = m.g, op.order = sp.order = m.order;
  op.rp = sp.rp = m.rp, sp.r = (int)a.r, op.pieces = pcs, op.size = sp.size = size, op.r = (int)a.r;
  op.table = m.prep.pieces[1].table;
  const bool share = pcs >= 4 * a.n;
  int sides = 0;
  int64_t outer_groups = 0, sum_groups = 0;
  for (int k = 0; k < 2; ++k) {
    if (!(k ? a.dB : a.dA)) continue;
    const auto& U = k ? dY : X;
    const int cols = k ? N : K;
    Outer& o = op.p[sides];
    Sum& u = sp.p[sides];
    ++sides;
    o.U = U.p, o.low = low[k].low, o.ldu = U.ld, o.cu = U.cols;
    o.blocks = (U.cols + 64 * Mma<T>::kE - 1) / (64 * Mma<T>::kE);
    o.ldp = (int)up(U.cols, 16 * Mma<T>::kE);
    if (!direct) o.part = ws.take<float>((int64_t)parts_of(a.T, a.n, size) * m.rp * o.ldp);
    u.part = o.part, u.out = k ? a.dB : a.dA, u.cols = cols, u.ldp = o.ldp;
    u.as = (int64_t)a.r * cols;
    const bool along = k ? !a.b_trans : a.a_trans;  // columns side by side
    u.cs = along ? 1 : a.r, u.rs = along ? cols : 1;
    const int64_t blocks = (cols + 63) / 64 * ((a.r + (share ? 3 : 15)) / (share ? 4 : 16));
    u.blocks = (int)blocks;
    o.out = u.out, o.as = u.as, o.cs = u.cs, o.rs = u.rs, o.cols = cols;
    outer_groups = std::max(outer_groups, (int64_t)pcs * o.blocks);
    sum_groups = std::max(sum_groups, blocks);
  }
  const unsigned sum_depth = (unsigned)std::min<int64_t>(a.n, 4096);
  ws.launch(outer_groups, 256, 2 * m.rb);
  ws.launch(sum_groups, 256, 2);
  if (!run) return GELIM_OK;
  m.run_prepare(s);
  if (a.T) {
    m.run_low(need_d ? low : low + 1, need_d + need_s, s);
    if (a.dX) m.run_big(q, low[0], s);
  }
  if (sides) {
    if (a.T) {
      int per = std::min(m.rb, 4);  // blocks of 16 ranks a workgroup, fewer where that fills the chip
      while (per > 1 && outer_groups * sides * (m.rb / per) < 384) per /= 2;
      const dim3 grid((unsigned)outer_groups, (unsigned)sides, (unsigned)(m.rb / per));
      auto launch = [&](auto direct) {
        constexpr bool D = decltype(direct)::value;
        if (per == 1) hipLaunchKernelGGL((outer_kernel<T, 1, D>), grid, dim3(256), 0, s, op);
        else if (per == 2) hipLaunchKernelGGL((outer_kernel<T, 2, D>), grid, dim3(256), 0, s, op);
        else hipLaunchKernelGGL((outer_kernel<T, 4, D>), grid, dim3(256), 0, s, op);
      };
      if (direct) launch(std::true_type{});
      else launch(std::false_type{});
    }
    if (direct) {
      HIP_TRY(hipGetLastError());
      return GELIM_OK;
    }
    const dim3 grid((unsigned)sum_groups, (unsigned)sides, sum_depth);
    if (share) hipLaunchKernelGGL((sum_kernel<T, true>), grid, dim3(256), 0, s, sp);
    else hipLaunchKernelGGL((sum_kernel<T, false>), grid, dim3(256), 0, s, sp);
  }
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
}

int run_or_count(const gelim_adapter_args& a, bool grad, Space& ws, hipStream_t s, bool run) {
  if (grad) {
    if (a.dtype == GELIM_T_F32) return gradient<float>(a, ws, s, run);
    if (a.dtype == GELIM_T_BF16) return gradient<__bf16>(a, ws, s, run);
    return gradient<_Float16>(a, ws, s, run);
  }
  if (a.dtype == GELIM_T_F32) return product<float>(a, ws, s, run);
  if (a.dtype == GELIM_T_BF16) return product<__bf16>(a, ws, s, run);
  return product<_Float16>(a, ws, s, run);
}

}  // namespace
}  // namespace gelim

extern "C" int64_t gelim_adapter_args_layout(int32_t which) {
  switch (which) {
    case 0: return sizeof(gelim_adapter_args);
    case 1: return offsetof(gelim_adapter_args, T);
    case 2: return offsetof(gelim_adapter_args, index);
    case 3: return offsetof(gelim_adapter_args, ws_bytes);
    default: return -1;
  }
}

extern "C" int64_t gelim_adapter_workspace(const gelim_adapter_args* a, int grad) {
  GELIM_TRY(gelim::check_shape(*a));
  gelim::Space ws{nullptr};
  gelim::run_or_count(*a, grad != 0, ws, nullptr, false);
  // a workgroup's number times its threads is an int in the kernels
  if (ws.threads > INT32_MAX) return GELIM_FAIL(GELIM_E_ARG, "adapter: too large for one launch");
  return ws.used;
}

extern "C" int gelim_adapter_matmul(const gelim_adapter_args* a, void* stream) {
  GELIM_TRY(gelim::check(*a, false));
  gelim::Space ws{(char*)a->ws};
  return gelim::run_or_count(*a, false, ws, (hipStream_t)stream, true);
}

extern "C" int gelim_adapter_matmul_grad(const gelim_adapter_args* a, void* stream) {
  GELIM_TRY(gelim::check(*a, true));
  gelim::Space ws{(char*)a->ws};
  return gelim::run_or_count(*a, true, ws, (hipStream_t)stream, true);
}
