// Low-rank adapters beside a shared projection, and their gradients.
//
//   S = X A_i (T x r, fp32)    Y = X W + s_i S B_i
//   D = dY B_i^T (T x r)       dX = dY W^T + s_i D A_i^T
//   dA_i = s_i sum_t X_t^T D_t     dB_i = s_i sum_t S_t^T dY_t    (rows t of adapter i)
//
// Plain form: every sum in fp32 on the vector units, any layout.
#include <hip/hip_runtime.h>

#include <cstddef>
#include <utility>

#include "device_common.h"
#include "gelim/internal.h"

namespace gelim {
namespace {

// a matrix, or one matrix per adapter: element (i, j) of adapter a at p[a * as + i * rs + j * cs]
template <class T>
struct View {
  T* p;
  int64_t as, rs, cs;
};

struct Rows {
  const int32_t* index;
  const float* scale;
  float scale_value;
  int n;
};

__device__ __forceinline__ int adapter_of(const Rows& g, int64_t t) { return g.index ? g.index[t] : 0; }
__device__ __forceinline__ float scale_of(const Rows& g, int i) { return g.scale ? g.scale[i] : g.scale_value; }

// low (T x r) = U (T x C) F_i (C x r); one workgroup per row
template <class T>
__global__ __launch_bounds__(256) void low_kernel(View<const T> U, View<const T> F, Rows g, float* low, int C, int r) {
  const int64_t t = blockIdx.x;
  const int i = adapter_of(g, t);
  if (i < 0 || i >= g.n) return;
  __shared__ float part[4];
  for (int j = 0; j < r; ++j) {
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += 256)
      s += (float)U.p[t * U.rs + c * U.cs] * (float)F.p[i * F.as + c * F.rs + j * F.cs];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
    __syncthreads();
    if (threadIdx.x == 0) low[t * r + j] = part[0] + part[1] + part[2] + part[3];
    __syncthreads();
  }
}

// Y (T x N) = X (T x K) W (K x N) + s_i low G_i (r x N); one thread per element of a 16 x 16 tile
template <class T>
__global__ __launch_bounds__(256) void product_kernel(View<const T> X, View<const T> W, View<const T> G, Rows g,
                                                      const float* low, View<T> Y, int64_t Tn, int K, int N, int r) {
  __shared__ float xs[16][17], ws[16][17];
  const int x = threadIdx.x % 16, y = threadIdx.x / 16;
  const int64_t t = (int64_t)blockIdx.y * 16 + y;
  const int64_t n = (int64_t)blockIdx.x * 16 + x;
  float acc = 0.f;
  for (int k0 = 0; k0 < K; k0 += 16) {
    xs[y][x] = t < Tn && k0 + x < K ? (float)X.p[t * X.rs + (k0 + x) * X.cs] : 0.f;
    ws[y][x] = n < N && k0 + y < K ? (float)W.p[(k0 + y) * W.rs + n * W.cs] : 0.f;
    __syncthreads();
    for (int k = 0; k < 16; ++k) acc += xs[y][k] * ws[k][x];
    __syncthreads();
  }
  if (t >= Tn || n >= N) return;
  const int i = adapter_of(g, t);
  if (i >= 0 && i < g.n) {
    float s = 0.f;
    for (int j = 0; j < r; ++j) s += low[t * r + j] * (float)G.p[i * G.as + j * G.rs + n * G.cs];
    acc += scale_of(g, i) * s;
  } else if (i != -1) {
    acc = __builtin_nanf("");
  }
  Y.p[t * Y.rs + n * Y.cs] = (T)acc;
}

// F_i (C x r) = s_i sum over the rows t of adapter i of U_t^T low_t; one thread per column of U
template <class T>
__global__ __launch_bounds__(256) void factor_grad_kernel(View<const T> U, const float* low, Rows g, View<T> F,
                                                          int64_t Tn, int C, int r) {
  const int c = blockIdx.x * 256 + threadIdx.x, i = blockIdx.y, j = blockIdx.z;
  if (c >= C) return;
  float s = 0.f;
  for (int64_t t = 0; t < Tn; ++t)
    if (adapter_of(g, t) == i) s += (float)U.p[t * U.rs + c * U.cs] * low[t * r + j];
  F.p[i * F.as + c * F.rs + j * F.cs] = (T)(scale_of(g, i) * s);
}

int check(const gelim_adapter_args& a, bool grad) {
  if (a.dtype < GELIM_T_F32 || a.dtype > GELIM_T_F16) return GELIM_FAIL(GELIM_E_ARG, "adapter: unknown type");
  if (a.T < 0 || a.K <= 0 || a.N <= 0 || a.r <= 0 || a.n <= 0) return GELIM_FAIL(GELIM_E_ARG, "adapter: bad shape");
  if (a.T > INT32_MAX || a.K > INT32_MAX || a.N > INT32_MAX || a.n > 65535)
    return GELIM_FAIL(GELIM_E_ARG, "adapter: dimension too large");
  if (a.r > GELIM_ADAPTER_MAX_RANK) return GELIM_FAIL(GELIM_E_ARG, "adapter: rank above 256");
  if (!a.W || !a.A || !a.B || (a.T && (!a.X || !a.Y))) return GELIM_FAIL(GELIM_E_ARG, "adapter: null matrix");
  if (a.ws_bytes < gelim_adapter_workspace(&a, grad)) return GELIM_FAIL(GELIM_E_ARG, "adapter: workspace too small");
  return GELIM_OK;
}

// A as K x r and B as r x N, or with `turn` their transposes
template <class T>
View<const T> view_w(const gelim_adapter_args& a, bool turn) {
  View<const T> v{(const T*)a.W, 0, a.w_trans ? 1 : a.ldw, a.w_trans ? a.ldw : 1};
  if (turn) std::swap(v.rs, v.cs);
  return v;
}
template <class T>
View<const T> view_a(const gelim_adapter_args& a, bool turn) {
  View<const T> v{(const T*)a.A, a.a_stride, a.a_trans ? 1 : a.lda, a.a_trans ? a.lda : 1};
  if (turn) std::swap(v.rs, v.cs);
  return v;
}
template <class T>
View<const T> view_b(const gelim_adapter_args& a, bool turn) {
  View<const T> v{(const T*)a.B, a.b_stride, a.b_trans ? 1 : a.ldb, a.b_trans ? a.ldb : 1};
  if (turn) std::swap(v.rs, v.cs);
  return v;
}

template <class T>
int product(const gelim_adapter_args& a, hipStream_t s) {
  const Rows g{a.index, a.scale, (float)a.scale_value, (int)a.n};
  const View<const T> X{(const T*)a.X, 0, a.ldx, 1};
  float* low = (float*)a.ws;
  hipLaunchKernelGGL(low_kernel<T>, dim3((unsigned)a.T), dim3(256), 0, s, X, view_a<T>(a, false), g, low, (int)a.K,
                     (int)a.r);
  const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.T + 15) / 16));
  hipLaunchKernelGGL(product_kernel<T>, grid, dim3(256), 0, s, X, view_w<T>(a, false), view_b<T>(a, false), g, low,
                     View<T>{(T*)a.Y, 0, a.ldy, 1}, a.T, (int)a.K, (int)a.N, (int)a.r);
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
}

template <class T>
int gradient(const gelim_adapter_args& a, hipStream_t s) {
  const Rows g{a.index, a.scale, (float)a.scale_value, (int)a.n};
  const View<const T> X{(const T*)a.X, 0, a.ldx, 1}, dY{(const T*)a.Y, 0, a.ldy, 1};
  float *S = (float*)a.ws, *D = S + a.T * a.r;
  if (a.T) {
    hipLaunchKernelGGL(low_kernel<T>, dim3((unsigned)a.T), dim3(256), 0, s, X, view_a<T>(a, false), g, S, (int)a.K,
                       (int)a.r);
    hipLaunchKernelGGL(low_kernel<T>, dim3((unsigned)a.T), dim3(256), 0, s, dY, view_b<T>(a, true), g, D, (int)a.N,
                       (int)a.r);
    if (a.dX) {
      const dim3 grid((unsigned)((a.K + 15) / 16), (unsigned)((a.T + 15) / 16));
      hipLaunchKernelGGL(product_kernel<T>, grid, dim3(256), 0, s, dY, view_w<T>(a, true), view_a<T>(a, true), g, D,
                         View<T>{(T*)a.dX, 0, a.lddx, 1}, a.T, (int)a.N, (int)a.K, (int)a.r);
    }
  }
  if (a.dA) {
    const View<T> dA{(T*)a.dA, a.K * a.r, a.a_trans ? 1 : a.r, a.a_trans ? a.K : 1};
    const dim3 grid((unsigned)((a.K + 255) / 256), (unsigned)a.n, (unsigned)a.r);
    hipLaunchKernelGGL(factor_grad_kernel<T>, grid, dim3(256), 0, s, X, D, g, dA, a.T, (int)a.K, (int)a.r);
  }
  if (a.dB) {
    const View<T> dBt{(T*)a.dB, a.r * a.N, a.b_trans ? a.r : 1, a.b_trans ? 1 : a.N};
    const dim3 grid((unsigned)((a.N + 255) / 256), (unsigned)a.n, (unsigned)a.r);
    hipLaunchKernelGGL(factor_grad_kernel<T>, grid, dim3(256), 0, s, dY, S, g, dBt, a.T, (int)a.N, (int)a.r);
  }
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
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
  return (grad ? 8 : 4) * a->T * a->r;
}

extern "C" int gelim_adapter_matmul(const gelim_adapter_args* a, void* stream) {
  GELIM_TRY(gelim::check(*a, false));
  if (a->T == 0) return GELIM_OK;
  if (a->dtype == GELIM_T_F32) return gelim::product<float>(*a, (hipStream_t)stream);
  if (a->dtype == GELIM_T_BF16) return gelim::product<__bf16>(*a, (hipStream_t)stream);
  return gelim::product<_Float16>(*a, (hipStream_t)stream);
}

extern "C" int gelim_adapter_matmul_grad(const gelim_adapter_args* a, void* stream) {
  GELIM_TRY(gelim::check(*a, true));
  if (a->dtype == GELIM_T_F32) return gelim::gradient<float>(*a, (hipStream_t)stream);
  if (a->dtype == GELIM_T_BF16) return gelim::gradient<__bf16>(*a, (hipStream_t)stream);
  return gelim::gradient<_Float16>(*a, (hipStream_t)stream);
}
