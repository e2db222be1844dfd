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
// 1. The order: one workgroup sorts the tokens by id (a stable radix sort of
//    9-bit digits, each wave ranking its own run of the keys) and marks the
//    rows that have tokens in V bits.  Where a gradient will be wanted this
//    workgroup runs in the lookup's own launch, beside its rows, and the
//    order is kept for the backward instead of the ids; else it is a launch
//    of its own (6 us for 1000 tokens, 25 us for 8192, 122 us for 32768).
// 2. One launch writes every row of the gradient but those of 3.  Its first
//    workgroups walk the sorted tokens in chunks, in order, for a slice of
//    the columns: a run of equal ids inside the chunk is summed in registers
//    and written; one that crosses a chunk's border leaves its part in fp32.
//    The others write the zeros of the rows without tokens, for which they
//    need only the bits: reading g is hidden behind that.
// 3. The parts are joined in order, by the chunk that the run begins in.
//
// 8192 tokens, bf16 [151936, 4096]: the lookup with the order 43 us (29
// without, 134 MB), the gradient 224 + 7 us, of which writing 1.24 GB of zeros
// alone takes 186.  999 tokens, fp32 [50257, 1027]: 12 and 39 + 4 us (the
// zeros alone 33).  64 tokens of 4096 without a gradient: 2.8 us.
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

struct RowArgs {
  const void* ids;
  int ids64;
  int64_t ids_stride;
  const void* weight;
  int64_t ld, V, H;
  float scale;
  void* out;
  int N, per_row;  // per_row: threads per row, a power of two from 64 on
};

// Row n by threads t = 0..per_row-1; kVec: 16 bytes per thread (rows 16-byte
// aligned and whole), else one element.  An id outside [0, V) gives a row of
// NaN.
template <typename T, bool kVec>
__device__ __forceinline__ void lookup_row(const RowArgs& a, int64_t n, int t) {
  typedef typename Elem<T>::store S;
  constexpr int E = Elem<T>::kE;
  const int64_t id = id_of(a.ids, a.ids64, n * a.ids_stride);
  const bool ok = id >= 0 && id < a.V;
  const S* row = reinterpret_cast<const S*>(a.weight) + (ok ? id : 0) * a.ld;
  S* to = reinterpret_cast<S*>(a.out) + n * a.H;
  const float nan = __builtin_nanf("");
  if constexpr (kVec) {
    for (int64_t c = t; c < a.H / E; c += a.per_row) {
      uint4 v = reinterpret_cast<const uint4*>(row)[c];
      if (a.scale != 1.0f || !ok) {
        float x[E];
        unpack<T>(v, x);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = ok ? x[i] * a.scale : nan;
        v = Elem<T>::pack(x);
      }
      reinterpret_cast<uint4*>(to)[c] = v;
    }
  } else {
    for (int64_t c = t; c < a.H; c += a.per_row) {
      S v = row[c];
      if (a.scale != 1.0f || !ok) v = Elem<T>::from(ok ? Elem<T>::to(v) * a.scale : nan);
      to[c] = v;
    }
  }
}

// Workgroups of one row each.
constexpr int kRowBlock = 256;
template <typename T, bool kVec>
__global__ __launch_bounds__(kRowBlock) void lookup_kernel(RowArgs a) {
  lookup_row<T, kVec>(a, blockIdx.x, threadIdx.x);
}

// ------------------------------------------------------------ sorting

constexpr int kSortBlock = 1024, kSortWaves = kSortBlock / kWave;
constexpr int kDigit = 9, kBins = 1 << kDigit;
constexpr int kRounds = 8;  // keys that a thread has in flight

struct SortArgs {
  const void* ids;
  int ids64;
  int64_t ids_stride, V, padding;
  int N, passes;
  // two buffers each; the sorted tokens end in buffer passes & 1
  uint32_t* key[2];
  int32_t* pos[2];
  uint32_t* rows;  // a bit per row: whether it has a token
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
  for (int n0 = first; n0 < last; n0 += kRounds * kWave) {
    uint32_t k[kRounds];
#pragma unroll
    for (int j = 0; j < kRounds; ++j) k[j] = load(min(n0 + j * kWave + lane, last - 1));
#pragma unroll
    for (int j = 0; j < kRounds; ++j)
      if (n0 + j * kWave + lane < last) {
        atomicAdd(&count[wave][(k[j] >> shift) & (kBins - 1)], 1u);
        if (kFirst && k[j] < a.V)  // (no other workgroup touches the bits)
          __hip_atomic_fetch_or(a.rows + k[j] / 32, 1u << (k[j] & 31), __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_WORKGROUP);
      }
  }
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
  for (int n0 = first; n0 < last; n0 += kRounds * kWave) {
    uint32_t key_at[kRounds];
    int32_t pos_at[kRounds];
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const int n = min(n0 + j * kWave + lane, last - 1);
      key_at[j] = load(n);
      pos_at[j] = kFirst ? n : pos[n];
    }
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      if (n0 + j * kWave >= last) break;
      const bool in = n0 + j * kWave + lane < last;
      const uint32_t d = (key_at[j] >> shift) & (kBins - 1);
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
        to_key[at] = key_at[j];
        to_pos[at] = pos_at[j];
        if (before == 0) count[wave][d] = at + (uint32_t)__popcll(same);
      }
      wave_lds_sync();
    }
  }
  __syncthreads();  // (and the global writes are visible to the workgroup)
}

// The order of a workgroup's tokens.
__device__ __forceinline__ void sort_tokens(const SortArgs& a) {
  __shared__ uint32_t count[kSortWaves][kBins];
  __shared__ uint32_t sums[kSortWaves];
  // (the first pass begins with a barrier)
  for (int64_t i = threadIdx.x; i < (a.V + 31) / 32; i += kSortBlock) a.rows[i] = 0;
  sort_pass<true>(a, 0, count, sums);
  for (int p = 1; p < a.passes; ++p) sort_pass<false>(a, p, count, sums);
}

__global__ __launch_bounds__(kSortBlock) void sort_kernel(SortArgs a) { sort_tokens(a); }

// Workgroup 0 sorts, the others look rows up.
template <typename T, bool kVec>
__global__ __launch_bounds__(kSortBlock) void lookup_and_sort_kernel(RowArgs r, SortArgs a) {
  if (blockIdx.x == 0) {
    sort_tokens(a);
    return;
  }
  const int rows = kSortBlock / r.per_row;
  const int64_t n = (int64_t)(blockIdx.x - 1) * rows + threadIdx.x / r.per_row;
  if (n < r.N) lookup_row<T, kVec>(r, n, threadIdx.x & (r.per_row - 1));
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
  // the zeros, by the workgroups from `sums` on
  const uint32_t* rows;
  int64_t sums, pieces_each;  // pieces per XCD
  int slices;
};

// A thread's columns: one 16-byte vector, or four elements kRowBlock apart (the
// last of them may lie behind the row).
template <typename T, bool kVec>
struct Column {
  typedef typename Elem<T>::store S;
  static constexpr int kE = kVec ? Elem<T>::kE : 4;
  __device__ static __forceinline__ int64_t first(int slice) {
    return (int64_t)slice * kRowBlock * kE + threadIdx.x * (kVec ? kE : 1);
  }
  __device__ static __forceinline__ void load(const SumArgs& a, const void* base, int64_t row,
                                              int64_t col, float (&x)[kE]) {
    const S* p = reinterpret_cast<const S*>(base) + row + col;
    if constexpr (kVec) {
      unpack<T>(*reinterpret_cast<const uint4*>(p), x);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        x[i] = col + i * kRowBlock < a.H ? Elem<T>::to(p[i * kRowBlock]) : 0.0f;
    }
  }
  __device__ static __forceinline__ void finish(const SumArgs& a, uint32_t v, int64_t col,
                                                const float (&sum)[kE]) {
    S* p = reinterpret_cast<S*>(a.out) + (int64_t)v * a.H + col;
    float x[kE];
    if (a.add) {
      load(a, a.out, (int64_t)v * a.H, col, x);
#pragma unroll
      for (int i = 0; i < kE; ++i) x[i] = __builtin_fmaf(sum[i], a.scale, x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) x[i] = sum[i] * a.scale;
    }
    if constexpr (kVec) {
      *reinterpret_cast<uint4*>(p) = Elem<T>::pack(x);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (col + i * kRowBlock < a.H) p[i * kRowBlock] = Elem<T>::from(x[i]);
    }
  }
  // place of the i-th in a part
  __device__ static __forceinline__ int64_t at(int i) { return kVec ? i : i * kRowBlock; }
};

// The first row of [v, last) with (kWith) or without a token, or last.
template <bool kWith>
__device__ __forceinline__ int64_t next_row(const uint32_t* rows, int64_t v, int64_t last) {
  while (v < last) {
    const uint32_t w = (kWith ? rows[v / 32] : ~rows[v / 32]) >> (v & 31);
    if (w) return min(last, v + __builtin_ctz(w));
    v = (v / 32 + 1) * 32;
  }
  return last;
}

// Zeros in piece `n` of kPiece bytes of the table, at addresses that are
// multiples of that, but in rows with a token: run by run of the others, whole
// 16-byte vectors between the elements not aligned to them.  Each XCD takes an
// eighth of the pieces, in order: fills of 206 MB and 1.24 GB take 33 and 186
// us so, 36 and 210 us with the pieces dealt round, and 41 us for 206 MB where
// a piece was three whole rows of 4108 bytes (XCDs sharing lines).
constexpr int64_t kPiece = 1 << 14;
constexpr int kXcds = 8;
template <typename T>
__device__ __forceinline__ void clear_piece(const SumArgs& a, int64_t n) {
  typedef typename Elem<T>::store S;
  constexpr int kPer = 16 / sizeof(S);
  S* base = reinterpret_cast<S*>(a.out);
  const int64_t skew = (int64_t)(reinterpret_cast<uintptr_t>(base) % kPiece / sizeof(S));
  const int64_t from = max((int64_t)0, n * (kPiece / (int64_t)sizeof(S)) - skew);
  const int64_t to = min(a.V * a.H, (n + 1) * (kPiece / (int64_t)sizeof(S)) - skew);
  const int64_t rows_end = (to + a.H - 1) / a.H;
  for (int64_t v = from / a.H; v < rows_end;) {
    int64_t end = rows_end;
    if (a.N > 0) {
      v = next_row<false>(a.rows, v, rows_end);
      end = next_row<true>(a.rows, v, rows_end);
    }
    const int64_t at = max(from, v * a.H), count = min(to, end * a.H) - at;
    S* p = base + at;
    const int64_t head =
        min(count, (int64_t)((-reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(S)));
    const int64_t vecs = (count - head) / kPer, tail = head + vecs * kPer;
    if (threadIdx.x < head) p[threadIdx.x] = S(0);
    uint4* q = reinterpret_cast<uint4*>(p + head);
    for (int64_t c = threadIdx.x; c < vecs; c += kRowBlock) q[c] = uint4{0, 0, 0, 0};
    if (tail + threadIdx.x < count) p[tail + threadIdx.x] = S(0);
    v = end;
  }
}

constexpr int kAhead = 4;  // rows of g in flight per thread

template <typename T, bool kVec>
__global__ __launch_bounds__(kRowBlock) void table_grad_kernel(SumArgs a) {
  typedef Column<T, kVec> C;
  constexpr int E = C::kE;
  if (blockIdx.x >= a.sums) {
    const int64_t b = blockIdx.x - a.sums, n = (b % kXcds) * a.pieces_each + b / kXcds;
    clear_piece<T>(a, n);
    return;
  }
  const int chunk = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int64_t col = C::first(slice);
  const int first = chunk * a.chunk, last = min(a.N, first + a.chunk);
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
      C::load(a, a.grad,
              (int64_t)min((uint32_t)a.pos[min(n0 + j, last - 1)], (uint32_t)a.N - 1) * a.ld, col,
              x[j]);
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
      if (!more && !from_before) {
        C::finish(a, v, col, sum);
      } else {  // the first run's part, or (it began here and goes on) the last one's
        float* p = a.part + ((int64_t)chunk * 2 + (from_before ? 0 : 1)) * a.H + col;
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (kVec || col + C::at(i) < a.H) p[C::at(i)] = sum[i];
      }
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
  const int64_t col = C::first(blockIdx.y);
  const int first = blockIdx.x * a.chunk, next = first + a.chunk;
  if (next >= a.N || col >= a.H) return;
  const uint32_t v = a.key[next];
  if (v >= a.V || a.key[next - 1] != v) return;        // nothing crosses this border
  if (a.key[first] == v && first > 0 && a.key[first - 1] == v) return;  // it began earlier
  float sum[E];
  const float* p = a.part + ((int64_t)blockIdx.x * 2 + 1) * a.H + col;
#pragma unroll
  for (int i = 0; i < E; ++i) sum[i] = kVec || col + C::at(i) < a.H ? p[C::at(i)] : 0.0f;
  for (int64_t c = blockIdx.x + 1; c * a.chunk < a.N && a.key[c * a.chunk] == v; ++c) {
    const float* q = a.part + c * 2 * a.H + col;
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] += kVec || col + C::at(i) < a.H ? q[C::at(i)] : 0.0f;
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

inline int size_of(int dtype) { return dtype == GTP_DTYPE_F32 ? 4 : 2; }

// An order: two buffers of sorted keys and positions, and the rows' bits.
struct Order {
  uint32_t* key[2];
  int32_t* pos[2];
  uint32_t* rows;
  size_t bytes;
};
inline Order order(int64_t N, int64_t V, void* p) {
  uint32_t* w = reinterpret_cast<uint32_t*>(p);
  auto at = [&](int64_t words) { return w ? w + words : nullptr; };
  Order o;
  for (int i = 0; i < 2; ++i) {
    o.key[i] = at(2 * i * N);
    o.pos[i] = reinterpret_cast<int32_t*>(at((2 * i + 1) * N));
  }
  o.rows = at(4 * N);
  o.bytes = N > 0 ? (size_t)(4 * N + (V + 31) / 32) * 4 : 0;
  return o;
}
inline int passes(int64_t V) {
  int n = 1;
  while ((V >> (n * kDigit)) != 0) ++n;
  return n;
}
inline SortArgs sort_args(const void* ids, int ids64, int64_t N, int64_t ids_stride, int64_t V,
                          int64_t padding, const Order& o) {
  SortArgs a;
  a.ids = ids;
  a.ids64 = ids64;
  a.ids_stride = ids_stride;
  a.V = V;
  a.padding = padding;
  a.N = (int)N;
  a.passes = passes(V);
  for (int i = 0; i < 2; ++i) {
    a.key[i] = o.key[i];
    a.pos[i] = o.pos[i];
  }
  a.rows = o.rows;
  return a;
}
// The parts of the runs, fp32.  (Rows in single elements have no fewer slices,
// so no more chunks than these.)
inline size_t part_bytes(int dtype, int64_t N, int64_t H) {
  if (N == 0) return 0;
  const int64_t slices = (H * size_of(dtype) / 16 + kRowBlock - 1) / kRowBlock;
  const int64_t chunk = chunk_of(N, max(slices, (int64_t)1));
  return (size_t)((N + chunk - 1) / chunk) * 2 * H * 4;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
void sums_launch(const SumArgs& a, bool vec, int64_t chunks, hipStream_t s) {
  const dim3 block(kRowBlock);
  const dim3 grid((unsigned)(a.sums + kXcds * a.pieces_each)), joins((unsigned)chunks, (unsigned)a.slices);
  if (grid.x > 0)
    vec ? launch_timed(table_grad_kernel<T, true>, grid, block, s, a)
        : launch_timed(table_grad_kernel<T, false>, grid, block, s, a);
  if (chunks > 1) {
    if (vec)
      hipLaunchKernelGGL((join_runs_kernel<T, true>), joins, block, 0, s, a);
    else
      hipLaunchKernelGGL((join_runs_kernel<T, false>), joins, block, 0, s, a);
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

namespace gtp {
namespace emb {

// With an order: sorted beside the lookup.
int rows_and_order(const void* ids, int ids64, int64_t N, int64_t ids_stride, const void* weight,
                   int dtype, int64_t V, int64_t H, int64_t weight_stride, float scale, void* out,
                   const SortArgs* sort, hipStream_t s) {
  const int es = size_of(dtype);
  const bool vec = aligned16(weight) && aligned16(out) && (H * es) % 16 == 0 &&
                   (weight_stride * es) % 16 == 0;
  const int64_t lanes = vec ? H * es / 16 : H;
  RowArgs r;
  r.ids = ids;
  r.ids64 = ids64;
  r.ids_stride = ids_stride;
  r.weight = weight;
  r.ld = weight_stride;
  r.V = V;
  r.H = H;
  r.scale = scale;
  r.out = out;
  r.N = (int)N;
  r.per_row = kWave;
  while (r.per_row < kRowBlock && r.per_row < lanes) r.per_row *= 2;
  auto launch = [&](auto one, auto both) {
    if (sort) {
      const int rows = kSortBlock / r.per_row;
      launch_timed(both, dim3((unsigned)(1 + (N + rows - 1) / rows)), dim3(kSortBlock), s, r,
                   *sort);
    } else {
      launch_timed(one, dim3((unsigned)N), dim3((unsigned)r.per_row), s, r);
    }
  };
  auto pick = [&](auto t) {
    typedef decltype(t) T;
    vec ? launch(lookup_kernel<T, true>, lookup_and_sort_kernel<T, true>)
        : launch(lookup_kernel<T, false>, lookup_and_sort_kernel<T, false>);
  };
  switch (dtype) {
    case GTP_DTYPE_BF16:
      pick(uint16_t());
      break;
    case GTP_DTYPE_F16:
      pick(_Float16());
      break;
    default:
      pick(float());
  }
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

int check_rows(const void* ids, int64_t N, int64_t ids_stride, const void* weight, int dtype,
               int64_t V, int64_t H, int64_t weight_stride, const void* out) {
  if (bad_sizes(dtype, N, V, H) || weight_stride < H || ids_stride < 0 ||
      (N > 0 && (!ids || !weight || !out)))
    return GTP_ERR_INVALID_ARGUMENT;
  if (too_large(N, V, H) || weight_stride > ((int64_t)1 << 60) / V) return GTP_ERR_UNSUPPORTED;
  return GTP_OK;
}

// The gradient from an order.
int table_grad(const Order& o, int64_t N, const void* grad, int dtype, int64_t grad_stride,
               int64_t V, int64_t H, float scale, int accumulate, void* grad_weight, void* parts,
               hipStream_t s) {
  const int es = size_of(dtype);
  SumArgs q;
  q.key = o.key[passes(V) & 1];
  q.pos = o.pos[passes(V) & 1];
  q.rows = o.rows;
  q.grad = grad;
  q.ld = grad_stride;
  q.V = V;
  q.H = H;
  q.scale = scale;
  q.out = grad_weight;
  q.part = reinterpret_cast<float*>(parts);
  q.N = (int)N;
  q.add = accumulate ? 1 : 0;
  const bool vec = aligned16(grad) && aligned16(grad_weight) && (H * es) % 16 == 0 &&
                   (grad_stride * es) % 16 == 0;
  const int64_t lanes = vec ? H * es / 16 : (H + 3) / 4;
  q.slices = (int)((lanes + kRowBlock - 1) / kRowBlock);
  q.chunk = chunk_of(max(N, (int64_t)1), q.slices);
  const int64_t chunks = (N + q.chunk - 1) / q.chunk;
  q.sums = chunks * q.slices;
  q.pieces_each = 0;
  if (!accumulate) {
    const int64_t bytes = reinterpret_cast<uintptr_t>(grad_weight) % kPiece + V * H * es;
    q.pieces_each = (bytes + kXcds * kPiece - 1) / (kXcds * kPiece);
  }
  // (one launch's workgroups; a gradient that large does not fit the memory)
  if (q.sums + kXcds * q.pieces_each > 0x7FFFFFFFll) return GTP_ERR_UNSUPPORTED;
  switch (dtype) {
    case GTP_DTYPE_BF16:
      sums_launch<uint16_t>(q, vec, chunks, s);
      break;
    case GTP_DTYPE_F16:
      sums_launch<_Float16>(q, vec, chunks, s);
      break;
    default:
      sums_launch<float>(q, vec, chunks, s);
  }
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

int check_grad(int64_t N, const void* grad, int dtype, int64_t grad_stride, int64_t V, int64_t H,
               int accumulate, const void* grad_weight, const void* workspace) {
  if (bad_sizes(dtype, N, V, H) || grad_stride < 0 || !grad_weight ||
      (N > 0 && (!grad || !workspace)))
    return GTP_ERR_INVALID_ARGUMENT;
  if (too_large(N, V, H) || grad_stride > ((int64_t)1 << 36)) return GTP_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(grad_weight) & (size_of(dtype) - 1))
    return GTP_ERR_INVALID_ARGUMENT;
  return GTP_OK;
}

}  // namespace emb
}  // namespace gtp

extern "C" int gtp_embedding_rows(const void* ids, int ids_int64, int64_t N, int64_t ids_stride,
                                  const void* weight, int dtype, int64_t V, int64_t H,
                                  int64_t weight_stride, float scale, void* out, void* stream) {
  const int rc =
      emb::check_rows(ids, N, ids_stride, weight, dtype, V, H, weight_stride, out);
  if (rc != GTP_OK || N == 0) return rc;
  return emb::rows_and_order(ids, ids_int64, N, ids_stride, weight, dtype, V, H, weight_stride,
                             scale, out, nullptr, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t gtp_embedding_order_bytes(int64_t N, int64_t V) {
  if (emb::bad_sizes(0, N, V, 1) || emb::too_large(N, V, 1)) return 0;
  return emb::order(N, V, nullptr).bytes;
}

extern "C" int gtp_embedding_rows_ordered(const void* ids, int ids_int64, int64_t N,
                                          int64_t ids_stride, const void* weight, int dtype,
                                          int64_t V, int64_t H, int64_t weight_stride, float scale,
                                          void* out, int64_t padding_idx, void* order,
                                          size_t order_bytes, void* stream) {
  const int rc =
      emb::check_rows(ids, N, ids_stride, weight, dtype, V, H, weight_stride, out);
  if (rc != GTP_OK || N == 0) return rc;
  const emb::Order o = emb::order(N, V, order);
  if (!order || order_bytes < o.bytes || (reinterpret_cast<uintptr_t>(order) & 3u))
    return GTP_ERR_INVALID_ARGUMENT;
  const emb::SortArgs a =
      emb::sort_args(ids, ids_int64, N, ids_stride, V, padding_idx, o);
  return emb::rows_and_order(ids, ids_int64, N, ids_stride, weight, dtype, V, H, weight_stride,
                             scale, out, &a, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t gtp_embedding_backward_workspace_bytes(int dtype, int64_t N, int64_t V,
                                                         int64_t H) {
  if (emb::bad_sizes(dtype, N, V, H) || N == 0 || emb::too_large(N, V, H)) return 0;
  return emb::part_bytes(dtype, N, H) + emb::order(N, V, nullptr).bytes;
}

extern "C" int gtp_embedding_backward(const void* ids, int ids_int64, int64_t N, int64_t ids_stride,
                                      const void* grad, int dtype, int64_t grad_stride, int64_t V,
                                      int64_t H, float scale, int64_t padding_idx, int accumulate,
                                      void* grad_weight, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  if (ids_stride < 0 || (N > 0 && !ids)) return GTP_ERR_INVALID_ARGUMENT;
  const int rc =
      emb::check_grad(N, grad, dtype, grad_stride, V, H, accumulate, grad_weight, workspace);
  if (rc != GTP_OK) return rc;
  if (N > 0 && (workspace_bytes < gtp_embedding_backward_workspace_bytes(dtype, N, V, H) ||
                (reinterpret_cast<uintptr_t>(workspace) & 3u)))
    return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  unsigned char* at = reinterpret_cast<unsigned char*>(workspace);
  const emb::Order o = emb::order(N, V, at + emb::part_bytes(dtype, N, H));
  if (N > 0) {
    const emb::SortArgs a = emb::sort_args(ids, ids_int64, N, ids_stride, V, padding_idx, o);
    hipLaunchKernelGGL(emb::sort_kernel, dim3(1), dim3(emb::kSortBlock), 0, s, a);
  }
  return emb::table_grad(o, N, grad, dtype, grad_stride, V, H, scale, accumulate, grad_weight,
                         workspace, s);
}

extern "C" size_t gtp_embedding_backward_ordered_workspace_bytes(int dtype, int64_t N, int64_t H) {
  if (emb::bad_sizes(dtype, N, 1, H) || emb::too_large(N, 1, H)) return 0;
  return emb::part_bytes(dtype, N, H);
}

extern "C" int gtp_embedding_backward_ordered(const void* order, size_t order_bytes, int64_t N,
                                              const void* grad, int dtype, int64_t grad_stride,
                                              int64_t V, int64_t H, float scale, int accumulate,
                                              void* grad_weight, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  const int rc =
      emb::check_grad(N, grad, dtype, grad_stride, V, H, accumulate, grad_weight, workspace);
  if (rc != GTP_OK) return rc;
  const emb::Order o = emb::order(N, V, const_cast<void*>(order));
  if (N > 0 && (!order || order_bytes < o.bytes || (reinterpret_cast<uintptr_t>(order) & 3u) ||
                workspace_bytes < emb::part_bytes(dtype, N, H) ||
                (reinterpret_cast<uintptr_t>(workspace) & 3u)))
    return GTP_ERR_INVALID_ARGUMENT;
  return emb::table_grad(o, N, grad, dtype, grad_stride, V, H, scale, accumulate, grad_weight,
                         workspace, reinterpret_cast<hipStream_t>(stream));
}
