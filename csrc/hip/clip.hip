// 2-norm over many tensors, and their copies scaled by min(1, max_norm / (norm + 1e-6)).
//
// Memory-bound: every element is read twice (the factor needs all of them) and
// written once.  Two passes over the tensors; a pass is one launch per 264
// tensors (172 with outputs apart), whose table travels in the kernel's arguments, so a
// captured graph needs no table in device memory.  The tensors are cut into
// chunks and each workgroup takes a run of them; its sum goes to its
// own slot of the workspace, onto that of the launch before, and every
// workgroup of the second pass adds the slots up in one fixed order: no
// atomics, the same bits every time.
// Squares are summed in fp64: bf16 and fp32 values above 1.8e19 have squares
// beyond fp32's range, and at 4 converted elements per clock and CU the fp64
// units keep up with the memory.  The factor is rounded to fp32
// (off by 2^-24 at most), the product once more to the tensor's type; a factor
// below 2^-100, whose fp32 value may have lost bits or all of it, stays fp64.
// Measured: 290 tensors of together 1e9 bf16 values 1110 to 1170 us, 6 GB at 5.1 to 5.4 TB/s (a large copy: 4.95); 448
// tensors of 29e6 fp32 values, outputs apart, 65 us on the GPU under 230 us of the caller's time to name them all.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <climits>
#include <string>
#include <vector>

#include "device_common.h"
#include "gelim/internal.h"

namespace gelim {
namespace {

constexpr int kSlots = 1024, kThreads = 256;
constexpr int kChunk = 16384;  // elements

template <bool APART>
struct Table {
  static constexpr int kMost = APART ? 172 : 264;  // within 4 KB of arguments
  const void* in[kMost];
  void* out[APART ? kMost : 1];
  int32_t first[kMost + 1];  // chunks before this tensor
  uint16_t tail[kMost];      // elements of its last chunk
  int8_t type[kMost];
  int32_t count;
};
static_assert(sizeof(Table<true>) <= 4000 && sizeof(Table<false>) <= 4000, "kernel arguments");

// 16 bytes at any element's address: the hardware takes unaligned vector accesses
template <class T>
struct Pack {
  static constexpr int kLen = 16 / sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Mem {
    T v[kLen];
  };
};

// The chunks [begin, end) of one workgroup, one after the other: f(tensor, first element, elements, type).
template <bool APART, class F>
__device__ __forceinline__ void each_chunk(const Table<APART>& tb, F f) {
  const int all = tb.first[tb.count];
  const int begin = (int)((int64_t)all * blockIdx.x / gridDim.x);
  const int end = (int)((int64_t)all * (blockIdx.x + 1) / gridDim.x);
  if (begin == end) return;
  int lo = 0, hi = tb.count - 1;  // the last tensor that begins at or before `begin`
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tb.first[mid] <= begin) lo = mid;
    else hi = mid - 1;
  }
  for (int c = begin; c < end; ++c) {
    while (c >= tb.first[lo + 1]) ++lo;
    f(lo, (int64_t)(c - tb.first[lo]) * kChunk, c + 1 == tb.first[lo + 1] ? tb.tail[lo] : kChunk, tb.type[lo]);
  }
}

template <class T>
__device__ __forceinline__ double squares(const T* p, int len) {
  constexpr int L = Pack<T>::kLen;
  double s = 0.0;
  int e = threadIdx.x * L;
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

__global__ __launch_bounds__(kThreads) void squares_kernel(const Table<false> tb, double* slots, int fresh) {
  double s = 0.0;
  each_chunk(tb, [&](int i, int64_t at, int len, int type) {
    if (type == GELIM_T_F32) s += squares((const float*)tb.in[i] + at, len);
    else if (type == GELIM_T_BF16) s += squares((const __bf16*)tb.in[i] + at, len);
    else s += squares((const _Float16*)tb.in[i] + at, len);
  });
  s = block_sum(s);
  if (threadIdx.x == 0) slots[blockIdx.x] = fresh ? s : slots[blockIdx.x] + s;
}

// v f, rounded to fp32: left to itself the compiler may round some of the products straight to fp16, by place
__device__ __forceinline__ float times(float v, float f) {
  float r = v * f;
  asm("" : "+v"(r));
  return r;
}
__device__ __forceinline__ float times(float v, double f) {
  float r = (float)((double)v * f);
  asm("" : "+v"(r));
  return r;
}

template <class T, class F>
__device__ __forceinline__ void scaled(const T* p, T* q, int len, F f) {
  constexpr int L = Pack<T>::kLen;
  int e = threadIdx.x * L;
#pragma unroll 4
  for (; e + L <= len; e += kThreads * L) {
    typename Pack<T>::Mem m = *(const typename Pack<T>::Mem*)(p + e);
#pragma unroll
    for (int i = 0; i < L; ++i) m.v[i] = (T)times((float)m.v[i], f);
    *(typename Pack<T>::Mem*)(q + e) = m;
  }
  for (; e < len; ++e) q[e] = (T)times((float)p[e], f);
}

template <bool APART>
__global__ __launch_bounds__(kThreads) void scale_kernel(const Table<APART> tb, const double* slots, int nslots,
                                                         double max_norm, float* norm_out) {
  double s = 0.0;
  for (int i = threadIdx.x; i < nslots; i += kThreads) s += slots[i];
  const double norm = sqrt(block_sum(s));
  // a NaN norm makes a NaN factor; an infinite max_norm leaves all as it is
  double f = isinf(max_norm) ? 1.0 : max_norm / (norm + 1e-6);
  if (f > 1.0) f = 1.0;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  if (!APART && f == 1.0) return;
  auto scale_by = [&](auto factor) {
    each_chunk(tb, [&](int i, int64_t at, int len, int type) {
      const void* in = tb.in[i];
      void* out = APART ? tb.out[i] : const_cast<void*>(in);
      if (type == GELIM_T_F32) scaled((const float*)in + at, (float*)out + at, len, factor);
      else if (type == GELIM_T_BF16) scaled((const __bf16*)in + at, (__bf16*)out + at, len, factor);
      else scaled((const _Float16*)in + at, (_Float16*)out + at, len, factor);
    });
  };
  if (f > 0.0 && f < 0x1p-100) scale_by(f);
  else scale_by((float)f);
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

// Calls launch(table, whether it is the first) for tables of all tensors.
template <bool APART, class F>
void each_table(const void* const* in, void* const* out, const int64_t* sizes, const int8_t* types, int64_t count,
                F launch) {
  Table<APART> t;
  t.count = t.first[0] = 0;
  bool first = true;
  for (int64_t i = 0; i < count; ++i) {
    if (!sizes[i]) continue;
    const int64_t chunks = (sizes[i] + kChunk - 1) / kChunk;
    if (t.count == t.kMost || t.first[t.count] + chunks > INT32_MAX) {
      launch(t, first);
      first = false;
      t.count = 0;
    }
    t.in[t.count] = in[i];
    if (APART) t.out[t.count] = out[i];
    t.tail[t.count] = (uint16_t)(sizes[i] - (chunks - 1) * kChunk);
    t.type[t.count++] = types[i];
    t.first[t.count] = t.first[t.count - 1] + (int32_t)chunks;
  }
  launch(t, first);  // without any tensor as well: it clears the slots and writes the norm
}

int clip(const void* const* in, void* const* out, const int64_t* sizes, const int8_t* types, int64_t count,
         double max_norm, float* d_norm, double* slots, hipStream_t s) {
  if (!(max_norm >= 0)) return GELIM_FAIL(GELIM_E_ARG, "clip: max_norm must be a number and not negative");
  if (!d_norm || !slots) return GELIM_FAIL(GELIM_E_ARG, "clip: null norm or workspace");
  int64_t chunks = 0;
  bool apart = false;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || (sizes[i] && (!in[i] || !out[i])) || types[i] < GELIM_T_F32 || types[i] > GELIM_T_F16)
      return GELIM_FAIL(GELIM_E_ARG, "clip: bad tensor " + std::to_string(i));
    if (sizes[i] > (int64_t)INT32_MAX * kChunk) return GELIM_FAIL(GELIM_E_ARG, "clip: tensor too large");
    chunks += (sizes[i] + kChunk - 1) / kChunk;
    apart |= sizes[i] && in[i] != out[i];
  }
  GELIM_TRY(check_overlap(in, out, sizes, types, count));
  const int grid = (int)std::clamp<int64_t>(chunks, 1, kSlots);
  each_table<false>(in, out, sizes, types, count, [&](const Table<false>& t, bool first) {
    hipLaunchKernelGGL(squares_kernel, dim3(grid), dim3(kThreads), 0, s, t, slots, first);
  });
  if (apart)
    each_table<true>(in, out, sizes, types, count, [&](const Table<true>& t, bool first) {
      hipLaunchKernelGGL(scale_kernel<true>, dim3(grid), dim3(kThreads), 0, s, t, slots, grid, max_norm,
                         first ? d_norm : nullptr);
    });
  else
    each_table<false>(in, out, sizes, types, count, [&](const Table<false>& t, bool first) {
      hipLaunchKernelGGL(scale_kernel<false>, dim3(grid), dim3(kThreads), 0, s, t, slots, grid, max_norm,
                         first ? d_norm : nullptr);
    });
  HIP_TRY(hipGetLastError());
  return GELIM_OK;
}

}  // namespace
}  // namespace gelim

extern "C" int64_t gelim_clip_workspace(void) { return gelim::kSlots * (int64_t)sizeof(double); }

extern "C" int gelim_clip_norm(const void* const* in, void* const* out, const int64_t* sizes, const int8_t* dtypes,
                               int64_t count, double max_norm, float* d_norm, void* ws, int64_t ws_bytes,
                               void* stream) {
  if (count < 0) return GELIM_FAIL(GELIM_E_ARG, "clip: negative count");
  if (ws_bytes < gelim_clip_workspace()) return GELIM_FAIL(GELIM_E_ARG, "clip: workspace too small");
  try {
    return gelim::clip(in, out, sizes, dtypes, count, max_norm, d_norm, (double*)ws, (hipStream_t)stream);
  } catch (const std::bad_alloc&) {
    return GELIM_FAIL(GELIM_E_NOMEM, "clip: out of host memory");
  }
}
