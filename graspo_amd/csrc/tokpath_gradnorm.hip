// tokpath_gradnorm.hip -- the global norm of many gradients, and their
// clipping (gfx950).
//
//   norm = (sum over all elements of |x|^p)^(1/p), p = 1, 2 or infinity
//   x   *= min(1, max_norm / (norm + 1e-6))
//
// over lists of fp32, bf16 and fp16 tensors.  Bound by HBM: the norm reads
// every element once, the clipping reads and writes it once, and reads and
// writes nothing where the factor is 1.
//
// The tensors' addresses and sizes travel in the kernel arguments, up to
// kMost tensors per launch, so that a call neither copies a table to the GPU
// nor keeps one, and can be captured.  A workgroup takes one chunk of one
// tensor; the chunks' sums are 64-bit (no square overflows or underflows) and
// are added in one order by a last kernel, without atomics.  4.13 GB of
// bf16: the norm 0.70 ms (5.9 TB/s), the clipping 1.61 ms (5.1 TB/s both ways).
#include "tokpath_stream.h"

namespace gtp {

int64_t device_cus();  // compute units of the current device

namespace norm {

constexpr int kBlock = 256;
constexpr int kMost = 192;  // 20 bytes each, of 4096 of kernel arguments
enum Power { kOne = 1, kTwo = 2, kMax = 3 };

struct List {
  void* p[kMost];
  int64_t n[kMost];      // elements | dtype << 56
  uint32_t end[kMost];   // chunks of this launch up to and with this tensor
  int count;
  uint32_t first;        // chunk index of the launch's first
  int64_t chunk;         // 16-byte vectors per chunk
};
static_assert(sizeof(List) <= 4000, "kernel arguments");

// The tensor of chunk c of the launch, and the chunk's index in it.
__device__ __forceinline__ int tensor_of(const List& l, uint32_t c, uint32_t& index) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (c < l.end[mid])
      hi = mid;
    else
      lo = mid + 1;
  }
  index = c - (lo ? l.end[lo - 1] : 0u);
  return lo;
}

// A chunk's elements: whole vectors from the tensor's first 16-byte boundary
// on; the first chunk also has the elements before that boundary, the last
// one those behind the last whole vector.
struct Chunk {
  int64_t v0, v1;      // vectors, from `base` on
  int64_t head, tail;  // elements before `base` and behind vector v1
  unsigned char* base;
};
__device__ __forceinline__ Chunk chunk_of(const List& l, int t, uint32_t index, int es) {
  const int64_t n = l.n[t] & 0xFFFFFFFFFFFFFFll;
  unsigned char* p = reinterpret_cast<unsigned char*>(l.p[t]);
  const int64_t off = (int64_t)(-(intptr_t)p & 15) / es, per = 16 / es;
  const int64_t head = min(n, off), vecs = (n - head) / per;
  Chunk c;
  c.base = p + head * es;
  c.v0 = min(vecs, (int64_t)index * l.chunk);
  c.v1 = min(vecs, c.v0 + l.chunk);
  c.head = index == 0 ? head : 0;
  c.tail = c.v1 == vecs && (index == 0 || c.v0 < vecs) ? (n - head) - vecs * per : 0;
  return c;
}

template <typename T>
struct Load {
  static constexpr int kE = Vec<T>::kE;
  typedef typename std::conditional<kE == 4, float, uint16_t>::type S;
  __device__ static __forceinline__ void vec(const uint4& v, float (&x)[kE]) {
    Vec<T>::cvt(u32x4{v.x, v.y, v.z, v.w}, x);
  }
  __device__ static __forceinline__ float one(S v) {
    if constexpr (kE == 4)
      return v;
    else if constexpr (std::is_same<T, uint16_t>::value)
      return u2f((uint32_t)v << 16);
    else
      return f16_to_f32(v);
  }
  __device__ static __forceinline__ S round(float v) {
    if constexpr (kE == 4)
      return v;
    else if constexpr (std::is_same<T, uint16_t>::value)
      return __builtin_bit_cast(uint16_t, (__bf16)v);
    else
      return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};

// Running sum (or, for the maximum, the largest |x| by its bits: NaN is above
// infinity, so that it stays).
template <int kP>
struct Sum {
  double s;
  uint32_t top;
  __device__ __forceinline__ void add(float x) {
    if constexpr (kP == kTwo)
      s = __builtin_fma((double)x, (double)x, s);
    else if constexpr (kP == kOne)
      s += (double)fabsf(x);
    else
      top = max(top, f2u(x) & 0x7FFFFFFFu);
  }
  __device__ __forceinline__ void merge(const Sum& o) {
    if constexpr (kP == kMax)
      top = max(top, o.top);
    else
      s += o.s;
  }
  __device__ __forceinline__ Sum other(int o) const {
    Sum r{};
    if constexpr (kP == kMax)
      r.top = __shfl_xor(top, o, kWave);
    else
      r.s = __shfl_xor(s, o, kWave);
    return r;
  }
  __device__ __forceinline__ double value() const { return kP == kMax ? (double)u2f(top) : s; }
};

template <int kP, int kThreads>
__device__ __forceinline__ double block_sum(Sum<kP> s, Sum<kP>* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s.merge(s.other(o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; ++w) s.merge(red[w]);
  return s.value();
}

constexpr int kAhead = 4;  // vectors in flight per thread

template <int kP, typename T>
__device__ __forceinline__ Sum<kP> sum_chunk(const Chunk& c) {
  typedef Load<T> L;
  Sum<kP> part[kAhead] = {};
  const uint4* v = reinterpret_cast<const uint4*>(c.base);
  int64_t i = c.v0 + threadIdx.x;
  for (; i + (kAhead - 1) * kBlock < c.v1; i += kAhead * kBlock) {
    uint4 w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) w[j] = v[i + j * kBlock];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      float x[L::kE];
      L::vec(w[j], x);
#pragma unroll
      for (int e = 0; e < L::kE; ++e) part[j].add(x[e]);
    }
  }
  for (; i < c.v1; i += kBlock) {
    float x[L::kE];
    L::vec(v[i], x);
#pragma unroll
    for (int e = 0; e < L::kE; ++e) part[0].add(x[e]);
  }
  const typename L::S* s = reinterpret_cast<const typename L::S*>(c.base);
  if (threadIdx.x < c.head) part[1].add(L::one(s[(int64_t)threadIdx.x - c.head]));
  if (threadIdx.x < c.tail) part[2].add(L::one(s[c.v1 * L::kE + threadIdx.x]));
#pragma unroll
  for (int j = 1; j < kAhead; ++j) part[0].merge(part[j]);
  return part[0];
}

template <int kP>
__global__ __launch_bounds__(kBlock) void norm_chunks_kernel(List l, double* __restrict__ out) {
  __shared__ Sum<kP> red[kBlock / kWave];
  uint32_t index;
  const int t = tensor_of(l, blockIdx.x, index);
  const int dtype = (int)(l.n[t] >> 56);
  Sum<kP> s;
  if (dtype == GTP_DTYPE_F32)
    s = sum_chunk<kP, float>(chunk_of(l, t, index, 4));
  else if (dtype == GTP_DTYPE_BF16)
    s = sum_chunk<kP, uint16_t>(chunk_of(l, t, index, 2));
  else
    s = sum_chunk<kP, _Float16>(chunk_of(l, t, index, 2));
  const double v = block_sum<kP, kBlock>(s, red);
  if (threadIdx.x == 0) out[l.first + blockIdx.x] = v;
}

template <int kP>
__global__ __launch_bounds__(1024) void norm_total_kernel(const double* __restrict__ part, int64_t n,
                                                          float* __restrict__ out) {
  __shared__ Sum<kP> red[1024 / kWave];
  Sum<kP> s{};
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    Sum<kP> o{};
    if constexpr (kP == kMax)
      o.top = f2u((float)part[i]);
    else
      o.s = part[i];
    s.merge(o);
  }
  const double v = block_sum<kP, 1024>(s, red);
  if (threadIdx.x == 0) *out = (float)(kP == kTwo ? sqrt(v) : v);
}

// The factor of the clipping; NaN where the norm is NaN.
__device__ __forceinline__ float factor_of(float norm, float max_norm) {
  const float f = max_norm / (norm + 1e-6f);
  return f > 1.0f ? 1.0f : f;
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const Chunk& c, float f) {
  typedef Load<T> L;
  uint4* v = reinterpret_cast<uint4*>(c.base);
  for (int64_t i = c.v0 + threadIdx.x; i < c.v1; i += kBlock) {
    float x[L::kE];
    L::vec(v[i], x);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (L::kE == 4)
        w[k] = f2u(x[k] * f);
      else
        w[k] = (uint32_t)L::round(x[2 * k] * f) | (uint32_t)L::round(x[2 * k + 1] * f) << 16;
    }
    v[i] = uint4{w[0], w[1], w[2], w[3]};
  }
  typename L::S* s = reinterpret_cast<typename L::S*>(c.base);
  if (threadIdx.x < c.head) {
    typename L::S* p = s + ((int64_t)threadIdx.x - c.head);
    *p = L::round(L::one(*p) * f);
  }
  if (threadIdx.x < c.tail) {
    typename L::S* p = s + (c.v1 * L::kE + threadIdx.x);
    *p = L::round(L::one(*p) * f);
  }
}

__global__ __launch_bounds__(kBlock) void clip_chunks_kernel(List l, const float* __restrict__ norm,
                                                             float max_norm) {
  const float f = factor_of(*norm, max_norm);
  if (f == 1.0f) return;
  uint32_t index;
  const int t = tensor_of(l, blockIdx.x, index);
  const int dtype = (int)(l.n[t] >> 56);
  if (dtype == GTP_DTYPE_F32)
    scale_chunk<float>(chunk_of(l, t, index, 4), f);
  else if (dtype == GTP_DTYPE_BF16)
    scale_chunk<uint16_t>(chunk_of(l, t, index, 2), f);
  else
    scale_chunk<_Float16>(chunk_of(l, t, index, 2), f);
}

inline int size_of(int dtype) { return dtype == GTP_DTYPE_F32 ? 4 : 2; }

// Vectors per chunk: 64 KB, and more where a list would have over 8192 such
// chunks for the last kernel to add.
struct Plan {
  int64_t chunk;   // 16-byte vectors
  int64_t chunks;
};
inline int64_t chunks_in(int64_t n, int es, int64_t chunk) {
  return max((int64_t)1, (n * es / 16 + chunk - 1) / chunk);
}
// Calls f(address, elements, dtype) for the tensors that are not empty, those
// that follow one another in memory (the views of a bucket) as one: 504 views
// of 167 MB take 2 launches of chunks instead of 6, and 81 us instead of 97.
constexpr int64_t kLongest = (int64_t)1 << 40;
template <typename F>
void for_spans(const void* const* p, const int64_t* n, const int32_t* dtype, int64_t count, F f) {
  for (int64_t i = 0; i < count;) {
    const int es = size_of(dtype[i]);
    const unsigned char* at = reinterpret_cast<const unsigned char*>(p[i]);
    int64_t all = n[i], k = i + 1;
    for (; k < count && all > 0 && dtype[k] == dtype[i] && at + all * es == p[k] &&
           all + n[k] < kLongest;
         ++k)
      all += n[k];
    if (all > 0) f(const_cast<void*>(p[i]), all, dtype[i]);
    i = k;
  }
}

int plan_of(const void* const* p, const int64_t* n, const int32_t* dtype, int64_t count, Plan& plan) {
  if (count < 0 || (count > 0 && (!p || !n || !dtype))) return GTP_ERR_INVALID_ARGUMENT;
  int64_t bytes = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (dtype[i] < GTP_DTYPE_F32 || dtype[i] > GTP_DTYPE_F16 || n[i] < 0 || (n[i] > 0 && !p[i]) ||
        (reinterpret_cast<uintptr_t>(p[i]) & (size_of(dtype[i]) - 1)))
      return GTP_ERR_INVALID_ARGUMENT;
    bytes += n[i] < kLongest ? n[i] * size_of(dtype[i]) : 0;
    if (n[i] >= kLongest || bytes > (int64_t)1 << 60) return GTP_ERR_UNSUPPORTED;
  }
  plan.chunk = 4096;
  while (bytes / 16 / plan.chunk > 8192) plan.chunk *= 2;
  plan.chunks = 0;
  for_spans(p, n, dtype, count, [&](void*, int64_t m, int dt) {
    plan.chunks += chunks_in(m, size_of(dt), plan.chunk);
  });
  return plan.chunks < (1 << 23) ? GTP_OK : GTP_ERR_UNSUPPORTED;
}

// Calls `launch(list, chunks of it)` over the spans, kMost at a time.
template <typename F>
void for_lists(void* const* p, const int64_t* n, const int32_t* dtype, int64_t count,
               const Plan& plan, F launch) {
  List l;
  l.count = 0;
  l.first = 0;
  l.chunk = plan.chunk;
  uint32_t chunks = 0;
  auto flush = [&] {
    if (l.count == 0) return;
    launch(l, chunks);
    l.first += chunks;
    l.count = 0;
    chunks = 0;
  };
  for_spans(p, n, dtype, count, [&](void* at, int64_t m, int dt) {
    if (l.count == kMost) flush();
    chunks += (uint32_t)chunks_in(m, size_of(dt), plan.chunk);
    l.p[l.count] = at;
    l.n[l.count] = m | (int64_t)dt << 56;
    l.end[l.count] = chunks;
    ++l.count;
  });
  flush();
}

template <int kP>
void norm_launch(void* const* p, const int64_t* n, const int32_t* dtype, int64_t count,
                 const Plan& plan, double* part, float* out, hipStream_t s) {
  for_lists(p, n, dtype, count, plan, [&](const List& l, uint32_t chunks) {
    launch_timed(norm_chunks_kernel<kP>, dim3(chunks), dim3(kBlock), s, l, part);
  });
  hipLaunchKernelGGL(norm_total_kernel<kP>, dim3(1), dim3(1024), 0, s, part, plan.chunks, out);
}

}  // namespace norm
}  // namespace gtp

using namespace gtp;

extern "C" size_t gtp_grad_norm_workspace_bytes(const void* const* tensors, const int64_t* sizes,
                                                const int32_t* dtypes, int64_t count) {
  norm::Plan plan;
  if (norm::plan_of(tensors, sizes, dtypes, count, plan) != GTP_OK) return 0;
  return (size_t)max(plan.chunks, (int64_t)1) * sizeof(double);
}

extern "C" int gtp_grad_norm(const void* const* tensors, const int64_t* sizes,
                             const int32_t* dtypes, int64_t count, int norm_type, float* out_norm,
                             void* workspace, size_t workspace_bytes, void* stream) {
  norm::Plan plan;
  const int rc = norm::plan_of(tensors, sizes, dtypes, count, plan);
  if (rc != GTP_OK) return rc;
  if (!out_norm || !workspace || workspace_bytes < (size_t)plan.chunks * sizeof(double) ||
      (reinterpret_cast<uintptr_t>(workspace) & 7u) ||
      norm_type < norm::kOne || norm_type > norm::kMax)
    return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* part = reinterpret_cast<double*>(workspace);
  void* const* p = const_cast<void* const*>(tensors);
  if (norm_type == norm::kTwo)
    norm::norm_launch<norm::kTwo>(p, sizes, dtypes, count, plan, part, out_norm, s);
  else if (norm_type == norm::kOne)
    norm::norm_launch<norm::kOne>(p, sizes, dtypes, count, plan, part, out_norm, s);
  else
    norm::norm_launch<norm::kMax>(p, sizes, dtypes, count, plan, part, out_norm, s);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

extern "C" int gtp_clip_grads(void* const* tensors, const int64_t* sizes, const int32_t* dtypes,
                              int64_t count, const float* norm, float max_norm, void* stream) {
  norm::Plan plan;
  const int rc = norm::plan_of(tensors, sizes, dtypes, count, plan);
  if (rc != GTP_OK) return rc;
  if (!norm) return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  norm::for_lists(tensors, sizes, dtypes, count, plan, [&](const norm::List& l, uint32_t chunks) {
    hipLaunchKernelGGL(norm::clip_chunks_kernel, dim3(chunks), dim3(norm::kBlock), 0, s, l, norm,
                       max_norm);
  });
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}
