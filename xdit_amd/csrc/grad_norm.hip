// The norm of a list of gradients, and their clipping:  norm = (sum |g|^p)^(1/p) or max |g|,  g <- g min(1, max_norm / (norm + 1e-6)).
//
// Memory decides both: every element is read once for the norm, read and written once for the clipping.  A workgroup takes a chunk of one
// tensor and finds it by comparing its number with all first chunks at once (they are kernel arguments).  Sums are in 64 bits from the
// first square on (a square of a bf16 or fp32 gradient can leave fp32's range, and 1e9 of them its precision); the conversion to it and the
// multiply-add take about half of the time that a compute unit waits for the element.  Partial sums are added by one workgroup, in a fixed
// order. Measured, a call among others: the norm of 0.89 GB of bf16 143 us (6.2 TB/s; the kernels alone 140), of 2.0 GB of fp32 312 us in
// the kernel (6.3); clipping by it 0.8 GB of bf16 into fp32 475 us, 2.0 GB of fp32 in place 768 us (5.1 either; a copy of 1 GiB: 5.0).
// Small lists are the host's: 84 tensors take 18 us a norm, 6 of them in the kernel.
#include "grad_norm.h"
#include "launchers.h"
#include "row_ops.h"

namespace xdit {
namespace {

// Which tensor a chunk belongs to: the number of first chunks at or below it, less one.
template <int N>
__device__ __forceinline__ int tensor_of(const GradTable<N>& t, unsigned chunk) {
  int n = 0;
#pragma unroll
  for (int i = 0; i < (N + 63) / 64; i++) {
    const int at = i * 64 + (threadIdx.x & 63);
    n += __popcll(__builtin_amdgcn_ballot_w64(at < N && t.first[at < N ? at : N - 1] <= chunk));
  }
  return __builtin_amdgcn_readfirstlane(n - 1);
}

// Element indices count from the 16-byte boundary at or below a tensor's start (`lead` elements before it), so that groups of eight
// are aligned wherever a tensor starts; groups that its ends cut are read element by element.
template <typename T> __device__ __forceinline__ int lead_of(const void* p) { return (int)((uintptr_t)p & 15) / (int)sizeof(T); }

// Eight elements that are not read again before much else has been: past the caches' replacement order (28 blocks' gradients in bf16: 169 -> 152 us).
template <typename T>
__device__ __forceinline__ Raw8<T> stream_raw8(const T* p, int64_t off) {
  Raw8<T> r;
  const auto* v = (const typename Raw8<T>::vec*)(p + off);
#pragma unroll
  for (int i = 0; i < Raw8<T>::N; i++) r.x[i] = __builtin_nontemporal_load(v + i);
  return r;
}
// Groups of eight that a thread asks for at a time: 128 bytes (half of that: 152 us for 0.9 GB of bf16 where this takes 147; twice that: 2
// GB of fp32 and their clipping 1206 us, with this 1090).
template <typename T> constexpr int kGroups = 16 / sizeof(T);

template <int KIND>
__device__ __forceinline__ double norm_join(double a, double b) { return KIND == 0 ? (b > a || b != b ? b : a) : a + b; }
template <int KIND>
__device__ __forceinline__ double norm_add(double acc, float x) {
  const double v = (double)__builtin_fabsf(x);
  return KIND == 2 ? __builtin_fma(v, v, acc) : norm_join<KIND>(acc, v);
}
// Joins the workgroup's values, in a fixed order; the result is thread 0's.
template <int KIND, int WAVES>
__device__ __forceinline__ double workgroup_join(double v) {
  __shared__ double parts[WAVES];
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = norm_join<KIND>(v, __shfl_xor(v, m));
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < WAVES; i++) v = norm_join<KIND>(v, parts[i]);
  return v;
}

// The norm of n partial values, for thread 0 of 256 or (more than kClipPartials of them: four loads of each thread in flight; 7084 took 8.1
// us with 256 threads and a load at a time) 1024; up to that count in the same order either way.
template <int KIND, int THREADS, class Load>
__device__ __forceinline__ float norm_of(Load load, int64_t n) {
  double v = 0.;
  int64_t i = threadIdx.x;
  for (; i + 3 * THREADS < n; i += 4 * THREADS) {
    double x[4];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = load(i + j * THREADS);
#pragma unroll
    for (int j = 0; j < 4; j++) v = norm_join<KIND>(v, x[j]);
  }
  for (; i < n; i += THREADS) v = norm_join<KIND>(v, load(i));
  if constexpr (THREADS > 256) {
    __shared__ double all[THREADS];
    all[threadIdx.x] = v;
    __syncthreads();
    v = 0.;
    if (threadIdx.x < 256)
      for (int j = threadIdx.x; j < THREADS; j += 256) v = norm_join<KIND>(v, all[j]);
  }
  v = workgroup_join<KIND, THREADS / 64>(v);
  return (float)(KIND == 2 ? __builtin_sqrt(v) : v);
}
template <int THREADS>
__device__ __forceinline__ float norm_of(const double* partial, int64_t n, int kind) {
  auto load = [&](int64_t i) { return partial[i]; };
  return kind == 0 ? norm_of<0, THREADS>(load, n) : kind == 1 ? norm_of<1, THREADS>(load, n) : norm_of<2, THREADS>(load, n);
}

template <typename T, int KIND>
__global__ __launch_bounds__(256) void grad_norm_kernel(const NormParams p) {
  const int which = tensor_of(p.t, blockIdx.x);
  const T* src = (const T*)p.t.src[which];
  const int lead = lead_of<T>(src);
  const int64_t begin = (int64_t)(blockIdx.x - p.t.first[which]) * p.chunk;
  const int64_t end = p.t.numel[which] + lead;   // of the tensor
  const T* base = src - lead;
  const int64_t last = begin + p.chunk < end ? begin + p.chunk : end;
  double acc[4] = {0., 0., 0., 0.};
  int64_t i = begin + threadIdx.x * 8;
  constexpr int G = kGroups<T>;
  for (; i + (G - 1) * 2048 + 8 <= last && i >= lead; i += G * 2048) {
    Raw8<T> x[G];
#pragma unroll
    for (int n = 0; n < G; n++) x[n] = stream_raw8<T>(base, i + n * 2048);
#pragma unroll
    for (int n = 0; n < G; n++)
#pragma unroll
      for (int e = 0; e < 8; e++) acc[n & 3] = norm_add<KIND>(acc[n & 3], x[n][e]);
  }
  for (; i < last; i += 2048) {
    if (i >= lead && i + 8 <= last) {
      const Raw8<T> x = load_raw8<T>(base, i);
#pragma unroll
      for (int e = 0; e < 8; e++) acc[0] = norm_add<KIND>(acc[0], x[e]);
    } else {
      for (int64_t j = i; j < i + 8; j++)
        if (j >= lead && j < last) acc[0] = norm_add<KIND>(acc[0], (float)base[j]);
    }
  }
  const double v = workgroup_join<KIND, 4>(norm_join<KIND>(norm_join<KIND>(acc[0], acc[1]), norm_join<KIND>(acc[2], acc[3])));
  if (p.counter == nullptr) {
    if (threadIdx.x == 0) p.partial[blockIdx.x] = v;
    return;
  }
  // The last workgroup to get here adds the sums up, which spares a small list the second launch (84 tensors: 3.3 us a call less, the host's).  Its
  // accesses are device-scope ones, past the XCDs' caches; every workgroup waits for its store before it counts itself.
  __shared__ bool latest;
  if (threadIdx.x == 0) {
    __hip_atomic_store((unsigned long long*)p.partial + blockIdx.x, __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    latest = __hip_atomic_fetch_add(p.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!latest) return;
  const float norm = norm_of<KIND, 256>([&](int64_t i) {
    return __builtin_bit_cast(double, __hip_atomic_load((const unsigned long long*)p.partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  }, gridDim.x);
  if (threadIdx.x == 0) {
    *p.norm = norm;
    __hip_atomic_store(p.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

__global__ __launch_bounds__(1024) void grad_norm_total_kernel(const double* partial, int64_t n, int kind, float* norm) {
  const float v = norm_of<1024>(partial, n, kind);
  if (threadIdx.x == 0) *norm = v;
}

// A list of few chunks saves the launch between the norm and this one: every workgroup adds the partial sums up (84 tensors of a model's
// gains: 6.5 us of host time less a call than with a launch of its own for the sum and a C call of its own for the norm).  Taking the
// chunks from the last to the first, so that what the norm read last might still be in the memory-side cache, changed nothing (1097 us for
// 2 GB).
template <typename S, typename D>
__global__ __launch_bounds__(256) void grad_clip_kernel(const ClipParams p) {
  float norm;
  if (p.norm != nullptr) {
    norm = *p.norm;
  } else {
    __shared__ float total;
    const float v = norm_of<256>(p.partial, p.partials, p.kind);
    if (threadIdx.x == 0) {
      total = v;
      if (p.norm_out != nullptr && blockIdx.x == 0) *p.norm_out = v;
    }
    __syncthreads();
    norm = total;
  }
  // (Ordinary loads and stores: with streaming stores 0.8 GB of bf16 into fp32 took 783 us instead of 600, with streaming loads 604.)
  float factor = p.max_norm / (norm + 1e-6f);
  if (factor > 1.f) factor = 1.f;   // a norm that is not a number stays one
  const int which = tensor_of(p.t, blockIdx.x);
  const S* src = (const S*)p.t.src[which];
  D* dst = (D*)p.dst[which];
  if (factor == 1.f && (const void*)src == (const void*)dst) return;   // nothing to clip
  const int64_t numel = p.t.numel[which];
  const int64_t begin = (int64_t)(blockIdx.x - p.t.first[which]) * p.chunk;
  const int lead = lead_of<S>(src);
  if (lead == lead_of<D>(dst)) {
    const S* sb = src - lead;
    D* db = dst - lead;
    const int64_t end = numel + lead;
    const int64_t last = begin + p.chunk < end ? begin + p.chunk : end;
    int64_t i = begin + threadIdx.x * 8;
    for (; i + 3 * 2048 + 8 <= last && i >= lead; i += 4 * 2048) {
      Raw8<S> x[4];
#pragma unroll
      for (int n = 0; n < 4; n++) x[n] = load_raw8<S>(sb, i + n * 2048);
#pragma unroll
      for (int n = 0; n < 4; n++) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = x[n][e] * factor;
        store8<D>(db, i + n * 2048, v);
      }
    }
    for (; i < last; i += 2048) {
      if (i >= lead && i + 8 <= last) {
        const Raw8<S> x = load_raw8<S>(sb, i);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = x[e] * factor;
        store8<D>(db, i, v);
      } else {
        for (int64_t j = i; j < i + 8; j++)
          if (j >= lead && j < last) db[j] = (D)((float)sb[j] * factor);
      }
    }
  } else {   // source and destination differ in where their 16-byte groups start: element by element
    const int64_t last = begin + p.chunk < numel ? begin + p.chunk : numel;
    for (int64_t i = begin + threadIdx.x; i < last; i += 256) dst[i] = (D)((float)src[i] * factor);
  }
}

template <typename T>
void norm_typed(const NormParams& p, unsigned workgroups, hipStream_t stream) {
  if (p.kind == 0) hipLaunchKernelGGL((grad_norm_kernel<T, 0>), dim3(workgroups), dim3(256), 0, stream, p);
  else if (p.kind == 1) hipLaunchKernelGGL((grad_norm_kernel<T, 1>), dim3(workgroups), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((grad_norm_kernel<T, 2>), dim3(workgroups), dim3(256), 0, stream, p);
}

template <typename S>
void clip_typed(const ClipParams& p, int dst_dtype, unsigned workgroups, hipStream_t stream) {
  if (dst_dtype == 0) hipLaunchKernelGGL((grad_clip_kernel<S, __bf16>), dim3(workgroups), dim3(256), 0, stream, p);
  else if (dst_dtype == 1) hipLaunchKernelGGL((grad_clip_kernel<S, _Float16>), dim3(workgroups), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((grad_clip_kernel<S, float>), dim3(workgroups), dim3(256), 0, stream, p);
}

}  // namespace

hipError_t launch_grad_norm(const NormParams& p, int dtype, unsigned workgroups, hipStream_t stream) {
  if (dtype == 0) norm_typed<__bf16>(p, workgroups, stream);
  else if (dtype == 1) norm_typed<_Float16>(p, workgroups, stream);
  else norm_typed<float>(p, workgroups, stream);
  return hipGetLastError();
}

hipError_t launch_grad_norm_total(const double* partial, int64_t n, int kind, float* norm, hipStream_t stream) {
  hipLaunchKernelGGL(grad_norm_total_kernel, dim3(1), dim3(1024), 0, stream, partial, n, kind, norm);
  return hipGetLastError();
}

hipError_t launch_grad_clip(const ClipParams& p, int src_dtype, int dst_dtype, unsigned workgroups, hipStream_t stream) {
  if (src_dtype == 0) clip_typed<__bf16>(p, dst_dtype, workgroups, stream);
  else if (src_dtype == 1) clip_typed<_Float16>(p, dst_dtype, workgroups, stream);
  else clip_typed<float>(p, dst_dtype, workgroups, stream);
  return hipGetLastError();
}

}  // namespace xdit
