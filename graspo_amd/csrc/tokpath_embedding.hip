// tokpath_embedding.hip -- the embedding lookup with a scale, and the
// gradient of its table by sorted tokens (gfx950).
//
//   out_n = s w_{i_n}        dw_v = s sum over { n : i_n = v } of g_n
//
// over fp32, bf16 or fp16 tables [V, H]: one fp32 product, one rounding.  The
// gradient's sums are fp32, in an order that the ids alone fix (no atomics),
// and are rounded once.
//
// Forward: bound by its reads and writes (or, for a decode step's few rows,
// by one launch).  Backward: V H elements have to be written, most of them
// zeros; the rest is reading g once.
//
// 1. One launch sorts the tokens by id (one workgroup: a stable radix sort
//    of 9-bit digits, each wave ranking its own run of the keys) while all
//    its other workgroups write the table's zeros: the sort's serial steps
//    cost nothing beside them.
// 2. The sorted tokens in chunks: a workgroup walks one chunk in order for a
//    slice of the columns.  A run of equal ids inside the chunk is summed in
//    registers and written; one that crosses a chunk's border leaves its part
//    in fp32.
// 3. Those parts are joined in order, by the chunk that the run begins in.
#include "tokpath_stream.h"

namespace gtp {

int64_t device_cus();  // compute units of the current device

namespace emb {

// fp32 <-> the table's type, one 16-byte vector or one element at a time
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  typedef float store;
  static constexpr int kE = 4;
  __device__ static __forceinline__ float to(float v) { return v; }
  __device__ static __forceinline__ float from(float v) { return v; }
  __device__ static __forceinline__ uint4 pack(const float (&x)[4]) {
    return uint4{f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3])};
  }
};
template <typename Half>
struct Elem16 {
  typedef uint16_t store;
  static constexpr int kE = 8;
  __device__ static __forceinline__ uint16_t from(float v) {
    return __builtin_bit_cast(uint16_t, (Half)v);
  }
  __device__ static __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)from(x[2 * i]) | (uint32_t)from(x[2 * i + 1]) << 16;
    return uint4{w[0], w[1], w[2], w[3]};
  }
};
template <>
struct Elem<uint16_t> : Elem16<__bf16> {  // bf16 bit patterns
  __device__ static __forceinline__ float to(uint16_t v) { return u2f((uint32_t)v << 16); }
};
template <>
struct Elem<_Float16> : Elem16<_Float16> {
  __device__ static __forceinline__ float to(uint16_t v) { return f16_to_f32(v); }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[Elem<T>::kE]) {
  Vec<T>::cvt(u32x4{v.x, v.y, v.z, v.w}, x);
}

__device__ __forceinline__ int64_t id_of(const void* ids, int ids64, int64_t n) {
  return ids64 ? reinterpret_cast<const int64_t*>(ids)[n]
               : (int64_t)reinterpret_cast<const int32_t*>(ids)[n];
}

// ------------------------------------------------------------ forward

// One workgroup per row and kSlice bytes of it; kVec: 16 bytes per thread
// (rows 16-byte aligned and whole), else one element.  An id outside [0, V)
// gives a row of NaN.
constexpr int kRowBlock = 256;
template <typename T, bool kVec>
__global__ __launch_bounds__(kRowBlock) void lookup_kernel(const void* __restrict__ ids, int ids64,
                                                           int64_t ids_stride,
                                                           const void* __restrict__ weight,
                                                           int64_t ld, int64_t V, int64_t H,
                                                           float scale, void* __restrict__ out) {
  typedef typename Elem<T>::store S;
  constexpr int E = Elem<T>::kE;
  const int64_t n = blockIdx.x;
  const int64_t id = id_of(ids, ids64, n * ids_stride);
  const bool ok = id >= 0 && id < V;
  const S* row = reinterpret_cast<const S*>(weight) + (ok ? id : 0) * ld;
  S* to = reinterpret_cast<S*>(out) + n * H;
  const float nan = __builtin_nanf("");
  if constexpr (kVec) {
    for (int64_t c = threadIdx.x; c < H / E; c += blockDim.x) {
      uint4 v = reinterpret_cast<const uint4*>(row)[c];
      if (scale != 1.0f || !ok) {
        float x[E];
        unpack<T>(v, x);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = ok ? x[i] * scale : nan;
        v = Elem<T>::pack(x);
      }
      reinterpret_cast<uint4*>(to)[c] = v;
    }
  } else {
    for (int64_t c = threadIdx.x; c < H; c += blockDim.x) {
      S v = row[c];
      if (scale != 1.0f || !ok) v = Elem<T>::from(ok ? Elem<T>::to(v) * scale : nan);
      to[c] = v;
    }
  }
}

// ------------------------------------------------------------ sorting

constexpr int kSortBlock = 1024, kSortWaves = kSortBlock / kWave;
constexpr int kDigit = 9, kBins = 1 << kDigit;

struct SortArgs {
  const void* ids;
  int ids64;
  int64_t ids_stride, V, padding;
  int N, passes;
  // two buffers each; the sorted tokens end in buffer passes & 1
  uint32_t* key[2];
  int32_t* pos[2];
  uint4* zero;       // the table's gradient
  int64_t zero_vecs;  // whole 16-byte vectors of it
  uint32_t zero_tail;  // and bytes behind them
};

// Key of token n: its id, or V (behind all ids) where it has no gradient.
__device__ __forceinline__ uint32_t key_of(const SortArgs& a, int n) {
  const int64_t id = id_of(a.ids, a.ids64, n * a.ids_stride);
  return id < 0 || id >= a.V || id == a.padding ? (uint32_t)a.V : (uint32_t)id;
}

// One pass, stable: wave w ranks the keys of its run 64 at a time (lanes with
// equal digits find each other by one ballot per bit; the first of them
// advances the wave's counter), the counters are scanned digit by digit over
// the waves, and the keys go to their places.
template <bool kFirst>
__device__ void sort_pass(const SortArgs& a, int pass, uint32_t (*count)[kBins], uint32_t* sums) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t* key = a.key[pass & 1];
  const int32_t* pos = a.pos[pass & 1];
  uint32_t* to_key = a.key[(pass + 1) & 1];
  int32_t* to_pos = a.pos[(pass + 1) & 1];
  const int shift = pass * kDigit;
  for (int i = tid; i < kSortWaves * kBins; i += kSortBlock) count[0][i] = 0;
  __syncthreads();
  const int per = ((a.N + kSortBlock - 1) / kSortBlock) * kWave;
  const int first = min(a.N, wave * per), last = min(a.N, first + per);
  auto load = [&](int n) { return kFirst ? key_of(a, n) : key[n]; };
  for (int n = first + lane; n < last; n += kWave)
    atomicAdd(&count[wave][(load(n) >> shift) & (kBins - 1)], 1u);
  __syncthreads();
  // exclusive scan in the order (digit, wave): thread t takes half a digit
  {
    const int d = tid >> 1, w0 = (tid & 1) * (kSortWaves / 2);
    uint32_t c[kSortWaves / 2], sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves / 2; ++w) {
      c[w] = count[w0 + w][d];
      sum += c[w];
    }
    const uint32_t upto = wave_scan_u32(sum);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t at = upto - sum;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) at += w < wave ? sums[w] : 0;
#pragma unroll
    for (int w = 0; w < kSortWaves / 2; ++w) {
      count[w0 + w][d] = at;
      at += c[w];
    }
  }
  __syncthreads();
  for (int n0 = first; n0 < last; n0 += kWave) {
    const int n = n0 + lane;
    const bool in = n < last;
    const uint32_t k = in ? load(n) : 0u;
    const uint32_t d = (k >> shift) & (kBins - 1);
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < kDigit; ++b) {
      const uint64_t ones = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? ones : ~ones;
    }
    const uint32_t before = __popcll(same & ((1ull << lane) - 1));
    const uint32_t at = count[wave][d] + before;
    wave_lds_sync();
    if (in) {
      to_key[at] = k;
      to_pos[at] = kFirst ? n : pos[n];
      if (before == 0) count[wave][d] = at + (uint32_t)__popcll(same);
    }
    wave_lds_sync();
  }
  __syncthreads();  // (and the global writes are visible to the workgroup)
}

// Workgroup 0 sorts; the others write the zeros.
__global__ __launch_bounds__(kSortBlock) void sort_and_clear_kernel(SortArgs a) {
  if (blockIdx.x > 0) {
    const int64_t workers = (int64_t)(gridDim.x - 1) * kSortBlock;
    const int64_t first = (int64_t)(blockIdx.x - 1) * kSortBlock + threadIdx.x;
    for (int64_t i = first; i < a.zero_vecs; i += workers) a.zero[i] = uint4{0, 0, 0, 0};
    if (first < a.zero_tail / 2)
      reinterpret_cast<uint16_t*>(a.zero + a.zero_vecs)[first] = 0;
    return;
  }
  __shared__ uint32_t count[kSortWaves][kBins];
  __shared__ uint32_t sums[kSortWaves];
  sort_pass<true>(a, 0, count, sums);
  for (int p = 1; p < a.passes; ++p) sort_pass<false>(a, p, count, sums);
}

// ------------------------------------------------------------ sums

struct SumArgs {
  const uint32_t* key;  // sorted
  const int32_t* pos;
  const void* grad;     // [N, H], row stride ld
  int64_t ld, V, H;
  float scale;
  void* out;            // [V, H], row stride H
  float* part;          // [chunks][2][H]: a chunk's first and last run
  int N, chunk, add;    // add: to what the row holds
};

template <typename T, bool kVec>
struct Column {  // a thread's columns: one vector or one element
  typedef typename Elem<T>::store S;
  static constexpr int kE = kVec ? Elem<T>::kE : 1;
  __device__ static __forceinline__ void load(const void* base, int64_t at, float (&x)[kE]) {
    const S* p = reinterpret_cast<const S*>(base) + at;
    if constexpr (kVec)
      unpack<T>(*reinterpret_cast<const uint4*>(p), x);
    else
      x[0] = Elem<T>::to(*p);
  }
  __device__ static __forceinline__ void finish(const SumArgs& a, uint32_t v, int64_t col,
                                                const float (&sum)[kE]) {
    S* p = reinterpret_cast<S*>(a.out) + (int64_t)v * a.H + col;
    float x[kE];
    if (a.add) {
      load(a.out, (int64_t)v * a.H + col, x);
#pragma unroll
      for (int i = 0; i < kE; ++i) x[i] = __builtin_fmaf(sum[i], a.scale, x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) x[i] = sum[i] * a.scale;
    }
    if constexpr (kVec)
      *reinterpret_cast<uint4*>(p) = Elem<T>::pack(x);
    else
      *p = Elem<T>::from(x[0]);
  }
  __device__ static __forceinline__ void put_part(float* p, const float (&x)[kE]) {
#pragma unroll
    for (int i = 0; i < kE; ++i) p[i] = x[i];
  }
};

constexpr int kAhead = 4;  // rows of g in flight per thread

template <typename T, bool kVec>
__global__ __launch_bounds__(kRowBlock) void sum_runs_kernel(SumArgs a) {
  typedef Column<T, kVec> C;
  constexpr int E = C::kE;
  const int64_t col = ((int64_t)blockIdx.y * kRowBlock + threadIdx.x) * E;
  const int first = blockIdx.x * a.chunk, last = min(a.N, first + a.chunk);
  if (a.key[first] >= a.V || col >= a.H) return;
  // whether the first run began before the chunk
  bool from_before = first > 0 && a.key[first - 1] == a.key[first];
  float sum[E];
#pragma unroll
  for (int i = 0; i < E; ++i) sum[i] = 0.0f;
  for (int n0 = first; n0 < last; n0 += kAhead) {
    float x[kAhead][E];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      C::load(a.grad, (int64_t)a.pos[min(n0 + j, last - 1)] * a.ld + col, x[j]);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int n = n0 + j;
      if (n >= last) break;
      const uint32_t v = a.key[n];
      if (v >= a.V) return;
#pragma unroll
      for (int i = 0; i < E; ++i) sum[i] += x[j][i];
      const bool more = n + 1 < a.N && a.key[n + 1] == v;
      if (more && n + 1 < last) continue;
      if (!more && !from_before)
        C::finish(a, v, col, sum);
      else  // the first run's part, or (it began here and goes on) the last one's
        C::put_part(a.part + ((int64_t)blockIdx.x * 2 + (from_before ? 0 : 1)) * a.H + col, sum);
      from_before = false;
#pragma unroll
      for (int i = 0; i < E; ++i) sum[i] = 0.0f;
    }
  }
}

// The runs that cross a border: the chunk that such a run begins in adds its
// parts in order.
template <typename T, bool kVec>
__global__ __launch_bounds__(kRowBlock) void join_runs_kernel(SumArgs a) {
  typedef Column<T, kVec> C;
  constexpr int E = C::kE;
  const int64_t col = ((int64_t)blockIdx.y * kRowBlock + threadIdx.x) * E;
  const int first = blockIdx.x * a.chunk, next = first + a.chunk;
  if (next >= a.N || col >= a.H) return;
  const uint32_t v = a.key[next];
  if (v >= a.V || a.key[next - 1] != v) return;        // nothing crosses this border
  if (a.key[first] == v && first > 0 && a.key[first - 1] == v) return;  // it began earlier
  float sum[E];
  const float* p = a.part + ((int64_t)blockIdx.x * 2 + 1) * a.H + col;
#pragma unroll
  for (int i = 0; i < E; ++i) sum[i] = p[i];
  for (int64_t c = blockIdx.x + 1; c * a.chunk < a.N && a.key[c * a.chunk] == v; ++c) {
    const float* q = a.part + c * 2 * a.H + col;
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] += q[i];
  }
  C::finish(a, v, col, sum);
}

// Tokens per chunk: 32, and fewer while that leaves the chip short of
// workgroups.
inline int chunk_of(int64_t N, int64_t slices) {
  int c = 32;
  while (c > 8 && (N + c - 1) / c * slices < 2 * device_cus()) c /= 2;
  return c;
}

struct Space {
  uint32_t* key[2];
  int32_t* pos[2];
  float* part;
  size_t bytes;
};
inline int size_of(int dtype) { return dtype == GTP_DTYPE_F32 ? 4 : 2; }
// (rows in single elements have more slices, so no more chunks than these)
inline Space space(int dtype, int64_t N, int64_t H, void* ws) {
  const int64_t slices = (H * size_of(dtype) / 16 + kRowBlock - 1) / kRowBlock;
  const int64_t chunk = chunk_of(N, max(slices, (int64_t)1));
  unsigned char* base = reinterpret_cast<unsigned char*>(ws);
  size_t at = 0;
  auto take = [&](size_t n) {
    unsigned char* p = base ? base + at : nullptr;
    at += (n + 255) / 256 * 256;
    return p;
  };
  Space s;
  for (int i = 0; i < 2; ++i) {
    s.key[i] = reinterpret_cast<uint32_t*>(take(N * 4));
    s.pos[i] = reinterpret_cast<int32_t*>(take(N * 4));
  }
  s.part = reinterpret_cast<float*>(take((size_t)((N + chunk - 1) / chunk) * 2 * H * 4));
  s.bytes = at;
  return s;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
void sums_launch(const SumArgs& a, bool vec, dim3 grid, hipStream_t s) {
  if (vec) {
    launch_timed(sum_runs_kernel<T, true>, grid, dim3(kRowBlock), s, a);
    hipLaunchKernelGGL((join_runs_kernel<T, true>), grid, dim3(kRowBlock), 0, s, a);
  } else {
    launch_timed(sum_runs_kernel<T, false>, grid, dim3(kRowBlock), s, a);
    hipLaunchKernelGGL((join_runs_kernel<T, false>), grid, dim3(kRowBlock), 0, s, a);
  }
}

bool bad_sizes(int dtype, int64_t N, int64_t V, int64_t H) {
  return dtype < GTP_DTYPE_F32 || dtype > GTP_DTYPE_F16 || N < 0 || V <= 0 || H <= 0;
}
// what the kernels' 32-bit indices and one launch hold
bool too_large(int64_t N, int64_t V, int64_t H) {
  return N >= (1 << 24) || V >= 0x7FFFFFFFll || H > 65535ll * kRowBlock ||
         H > ((int64_t)1 << 60) / V;
}

}  // namespace emb
}  // namespace gtp

using namespace gtp;

extern "C" int gtp_embedding_rows(const void* ids, int ids_int64, int64_t N, int64_t ids_stride,
                                  const void* weight, int dtype, int64_t V, int64_t H,
                                  int64_t weight_stride, float scale, void* out, void* stream) {
  if (emb::bad_sizes(dtype, N, V, H) || weight_stride < H || ids_stride < 0 ||
      (N > 0 && (!ids || !weight || !out)))
    return GTP_ERR_INVALID_ARGUMENT;
  if (emb::too_large(N, V, H) || weight_stride > ((int64_t)1 << 60) / V)
    return GTP_ERR_UNSUPPORTED;
  if (N == 0) return GTP_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int es = emb::size_of(dtype);
  const bool vec = emb::aligned16(weight) && emb::aligned16(out) && (H * es) % 16 == 0 &&
                   (weight_stride * es) % 16 == 0;
  const int64_t lanes = vec ? H * es / 16 : H;
  const dim3 block((unsigned)min((int64_t)emb::kRowBlock, (lanes + 63) / 64 * 64));
  const dim3 grid((unsigned)N);
  auto launch = [&](auto kernel) {
    launch_timed(kernel, grid, block, s, ids, ids_int64, ids_stride, weight, weight_stride, V, H,
                 scale, out);
  };
  switch (dtype) {
    case GTP_DTYPE_BF16:
      vec ? launch(emb::lookup_kernel<uint16_t, true>) : launch(emb::lookup_kernel<uint16_t, false>);
      break;
    case GTP_DTYPE_F16:
      vec ? launch(emb::lookup_kernel<_Float16, true>) : launch(emb::lookup_kernel<_Float16, false>);
      break;
    default:
      vec ? launch(emb::lookup_kernel<float, true>) : launch(emb::lookup_kernel<float, false>);
  }
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

extern "C" size_t gtp_embedding_backward_workspace_bytes(int dtype, int64_t N, int64_t H) {
  if (emb::bad_sizes(dtype, N, 1, H) || N == 0 || emb::too_large(N, 1, H)) return 0;
  return emb::space(dtype, N, H, nullptr).bytes;
}

extern "C" int gtp_embedding_backward(const void* ids, int ids_int64, int64_t N, int64_t ids_stride,
                                      const void* grad, int dtype, int64_t grad_stride, int64_t V,
                                      int64_t H, float scale, int64_t padding_idx, int accumulate,
                                      void* grad_weight, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (emb::bad_sizes(dtype, N, V, H) || ids_stride < 0 || grad_stride < 0 || !grad_weight ||
      (N > 0 && (!ids || !grad || !workspace)))
    return GTP_ERR_INVALID_ARGUMENT;
  if (emb::too_large(N, V, H) || grad_stride > ((int64_t)1 << 36)) return GTP_ERR_UNSUPPORTED;
  const int es = emb::size_of(dtype);
  if (reinterpret_cast<uintptr_t>(grad_weight) & (es - 1)) return GTP_ERR_INVALID_ARGUMENT;
  const emb::Space sp = emb::space(dtype, N, H, workspace);
  if (N > 0 && workspace_bytes < sp.bytes) return GTP_ERR_INVALID_ARGUMENT;
  if (N == 0 && accumulate) return GTP_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  emb::SortArgs a;
  a.ids = ids;
  a.ids64 = ids_int64;
  a.ids_stride = ids_stride;
  a.V = V;
  a.padding = padding_idx;
  a.N = (int)N;
  a.passes = 1;
  while ((V >> (a.passes * emb::kDigit)) != 0) ++a.passes;
  for (int i = 0; i < 2; ++i) {
    a.key[i] = sp.key[i];
    a.pos[i] = sp.pos[i];
  }
  int64_t clear_groups = 0;
  a.zero = nullptr;
  a.zero_vecs = 0;
  a.zero_tail = 0;
  if (!accumulate) {
    if (!emb::aligned16(grad_weight)) return GTP_ERR_UNSUPPORTED;
    const int64_t bytes = V * H * es;
    a.zero = reinterpret_cast<uint4*>(grad_weight);
    a.zero_vecs = bytes / 16;
    a.zero_tail = (uint32_t)(bytes % 16);
    clear_groups = min((int64_t)2 * device_cus(), (a.zero_vecs + emb::kSortBlock) / emb::kSortBlock);
  }
  launch_timed(emb::sort_and_clear_kernel, dim3((unsigned)(1 + clear_groups)),
               dim3(emb::kSortBlock), s, a);
  if (N > 0) {
    emb::SumArgs q;
    q.key = sp.key[a.passes & 1];
    q.pos = sp.pos[a.passes & 1];
    q.grad = grad;
    q.ld = grad_stride;
    q.V = V;
    q.H = H;
    q.scale = scale;
    q.out = grad_weight;
    q.part = sp.part;
    q.N = (int)N;
    q.add = accumulate ? 1 : 0;
    const bool vec = emb::aligned16(grad) && emb::aligned16(grad_weight) && (H * es) % 16 == 0 &&
                     (grad_stride * es) % 16 == 0;
    const int64_t lanes = vec ? H * es / 16 : H;
    const int64_t slices = (lanes + emb::kRowBlock - 1) / emb::kRowBlock;
    q.chunk = emb::chunk_of(N, slices);
    const dim3 grid((unsigned)((N + q.chunk - 1) / q.chunk), (unsigned)slices);
    switch (dtype) {
      case GTP_DTYPE_BF16:
        emb::sums_launch<uint16_t>(q, vec, grid, s);
        break;
      case GTP_DTYPE_F16:
        emb::sums_launch<_Float16>(q, vec, grid, s);
        break;
      default:
        emb::sums_launch<float>(q, vec, grid, s);
    }
  }
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}
