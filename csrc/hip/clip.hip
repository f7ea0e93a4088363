// 2-norm over many tensors, and their copies scaled by min(1, max_norm / (norm + 1e-6)).
//
// Memory-bound: every element is read twice (the factor needs all of them) and
// written once.  Two passes over the tensors; a pass is one launch per
// kPerLaunch tensors, whose table travels in the kernel's arguments, so a
// captured graph needs no table in device memory.  The tensors are cut into
// chunks and workgroup b takes the chunks b, b + grid, ...; its sum goes to its
// own slot of the workspace, onto that of the launch before, and every
// workgroup of the second pass adds the slots up in one fixed order: no
// atomics, the same bits every time.
// Squares are summed in fp64: bf16 and fp32 values above 1.8e19 have squares
// beyond fp32's range, and at 4 converted elements per clock and CU the fp64
// units keep up with the memory.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "device_common.h"
#include "gelim/internal.h"

namespace gelim {
namespace {

constexpr int kPerLaunch = 128, kSlots = 1024, kThreads = 256;
constexpr int64_t kChunk = 16384;  // elements

struct Table {
  const void* in[kPerLaunch];
  void* out[kPerLaunch];
  int64_t size[kPerLaunch];
  int32_t first[kPerLaunch];  // chunks before this tensor
  int8_t type[kPerLaunch];
  int32_t count, chunks;
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");

// 16 bytes at any element's address: the hardware takes unaligned vector accesses
template <class T>
struct Pack {
  static constexpr int kLen = 16 / sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Mem {
    T v[kLen];
  };
};

__device__ __forceinline__ int tensor_of(const Table& tb, int chunk) {
  int lo = 0, hi = tb.count - 1;  // the last tensor that begins at or before the chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tb.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <class T>
__device__ __forceinline__ double squares(const T* p, int64_t len) {
  constexpr int L = Pack<T>::kLen;
  double s = 0.0;
  int64_t e = (int64_t)threadIdx.x * L;
#pragma unroll 4
  for (; e + L <= len; e += kThreads * L) {
    const typename Pack<T>::Mem m = *(const typename Pack<T>::Mem*)(p + e);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const double v = (double)(float)m.v[i];
      s = fma(v, v, s);
    }
  }
  for (; e < len; ++e) {  // the one thread with a part of a pack
    const double v = (double)(float)p[e];
    s = fma(v, v, s);
  }
  return s;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 64];
  v = dev::wave_sum(v);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < kThreads / 64; ++i) s += part[i];
  return s;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(const Table tb, double* slots, int fresh) {
  double s = 0.0;
  for (int c = blockIdx.x; c < tb.chunks; c += gridDim.x) {
    const int i = tensor_of(tb, c);
    const int64_t at = (int64_t)(c - tb.first[i]) * kChunk, len = min(tb.size[i] - at, kChunk);
    if (tb.type[i] == GELIM_T_F32) s += squares((const float*)tb.in[i] + at, len);
    else if (tb.type[i] == GELIM_T_BF16) s += squares((const __bf16*)tb.in[i] + at, len);
    else s += squares((const _Float16*)tb.in[i] + at, len);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) slots[blockIdx.x] = fresh ? s : slots[blockIdx.x] + s;
}

template <class T>
__device__ __forceinline__ void scaled(const T* p, T* q, int64_t len, float f) {
  constexpr int L = Pack<T>::kLen;
  int64_t e = (int64_t)threadIdx.x * L;
#pragma unroll 4
  for (; e + L <= len; e += kThreads * L) {
    typename Pack<T>::Mem m = *(const typename Pack<T>::Mem*)(p + e);
#pragma unroll
    for (int i = 0; i < L; ++i) m.v[i] = (T)((float)m.v[i] * f);
    *(typename Pack<T>::Mem*)(q + e) = m;
  }
  for (; e < len; ++e) q[e] = (T)((float)p[e] * f);
}

__global__ __launch_bounds__(kThreads) void scale_kernel(const Table tb, const double* slots, int nslots,
                                                         double max_norm, float* norm_out) {
  double s = 0.0;
  for (int i = threadIdx.x; i < nslots; i += kThreads) s += slots[i];
  const double norm = sqrt(block_sum(s));
  // a NaN norm makes a NaN factor; an infinite max_norm leaves all as it is
  double f = isinf(max_norm) ? 1.0 : max_norm / (norm + 1e-6);
  if (f > 1.0) f = 1.0;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  for (int k = blockIdx.x; k < tb.chunks; k += gridDim.x) {
    const int c = tb.chunks - 1 - k;  // the first pass's last chunks are the likeliest in a cache
    const int i = tensor_of(tb, c);
    if (f == 1.0 && tb.in[i] == tb.out[i]) continue;
    const int64_t at = (int64_t)(c - tb.first[i]) * kChunk, len = min(tb.size[i] - at, kChunk);
    if (tb.type[i] == GELIM_T_F32) scaled((const float*)tb.in[i] + at, (float*)tb.out[i] + at, len, (float)f);
    else if (tb.type[i] == GELIM_T_BF16) scaled((const __bf16*)tb.in[i] + at, (__bf16*)tb.out[i] + at, len, (float)f);
    else scaled((const _Float16*)tb.in[i] + at, (_Float16*)tb.out[i] + at, len, (float)f);
  }
}

// An output may be its own input and must not touch any other tensor.
int check_overlap(const void* const* in, void* const* out, const int64_t* sizes, const int8_t* types, int64_t count) {
  struct Span {
    uintptr_t begin, end;
    int64_t i;
  };
  std::vector<Span> v;
  v.reserve(count);
  for (int64_t i = 0; i < count; ++i)
    if (sizes[i]) v.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + sizes[i] * (types[i] ? 2 : 4), i});
  std::sort(v.begin(), v.end(), [](const Span& x, const Span& y) { return x.begin < y.begin; });
  for (size_t k = 1; k < v.size(); ++k)
    if (v[k].begin < v[k - 1].end)
      return GELIM_FAIL(GELIM_E_ARG, "clip: tensors " + std::to_string(v[k - 1].i) + " and " +
                                         std::to_string(v[k].i) + " are written to the same memory");
  for (int64_t i = 0; i < count; ++i) {
    if (!sizes[i] || in[i] == out[i]) continue;
    const uintptr_t b = (uintptr_t)in[i], e = b + sizes[i] * (types[i] ? 2 : 4);
    auto k = std::upper_bound(v.begin(), v.end(), b, [](uintptr_t x, const Span& s) { return x < s.end; });
    if (k != v.end() && k->begin < e)
      return GELIM_FAIL(GELIM_E_ARG, "clip: output " + std::to_string(k->i) + " overlaps input " + std::to_string(i));
  }
  return GELIM_OK;
}

int clip(const void* const* in, void* const* out, const int64_t* sizes, const int8_t* types, int64_t count,
         double max_norm, float* d_norm, double* slots, hipStream_t s) {
  if (!(max_norm >= 0)) return GELIM_FAIL(GELIM_E_ARG, "clip: max_norm must be a number and not negative");
  if (!d_norm || !slots) return GELIM_FAIL(GELIM_E_ARG, "clip: null norm or workspace");
  std::vector<Table> tables(1);
  int64_t most = 0;
  tables[0].count = tables[0].chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || (sizes[i] && (!in[i] || !out[i])) || types[i] < GELIM_T_F32 || types[i] > GELIM_T_F16)
      return GELIM_FAIL(GELIM_E_ARG, "clip: bad tensor " + std::to_string(i));
    if (!sizes[i]) continue;
    const int64_t chunks = (sizes[i] + kChunk - 1) / kChunk;
    if (tables.back().count == kPerLaunch || tables.back().chunks + chunks > INT32_MAX) {
      tables.emplace_back();
      tables.back().count = tables.back().chunks = 0;
    }
    Table& t = tables.back();
    if (chunks > INT32_MAX) return GELIM_FAIL(GELIM_E_ARG, "clip: tensor too large");
    t.in[t.count] = in[i];
    t.out[t.count] = out[i];
    t.size[t.count] = sizes[i];
    t.type[t.count] = types[i];
    t.first[t.count++] = t.chunks;
    t.chunks += (int32_t)chunks;
    most = std::max<int64_t>(most, t.chunks);
  }
  GELIM_TRY(check_overlap(in, out, sizes, types, count));
  const int grid = (int)std::clamp<int64_t>(most, 1, kSlots);
  for (size_t k = 0; k < tables.size(); ++k)
    hipLaunchKernelGGL(squares_kernel, dim3(grid), dim3(kThreads), 0, s, tables[k], slots, k == 0);
  for (size_t k = tables.size(); k-- > 0;)
    hipLaunchKernelGGL(scale_kernel, dim3(grid), dim3(kThreads), 0, s, tables[k], slots, grid, max_norm,
                       k == 0 ? d_norm : nullptr);
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
}

}  // namespace
}  // namespace gelim

extern "C" int64_t gelim_clip_workspace(int64_t) { return gelim::kSlots * (int64_t)sizeof(double); }

extern "C" int gelim_clip_norm(const void* const* in, void* const* out, const int64_t* sizes, const int8_t* dtypes,
                               int64_t count, double max_norm, float* d_norm, void* ws, int64_t ws_bytes,
                               void* stream) {
  if (count < 0) return GELIM_FAIL(GELIM_E_ARG, "clip: negative count");
  if (ws_bytes < gelim_clip_workspace(count)) return GELIM_FAIL(GELIM_E_ARG, "clip: workspace too small");
  try {
    return gelim::clip(in, out, sizes, dtypes, count, max_norm, d_norm, (double*)ws, (hipStream_t)stream);
  } catch (const std::bad_alloc&) {
    return GELIM_FAIL(GELIM_E_NOMEM, "clip: out of host memory");
  }
}
