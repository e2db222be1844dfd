// tokpath_states.hip -- the models' states follow the beams (gfx950).
//
// A state is a tensor whose first dimension counts the beams' rows (a layer's
// keys or values [R, heads, length, dim], a recurrent state), read and written
// as bytes.
//
// - reorder_kernel, in place: row g K + k becomes row parent[g K + k], of the
//   same group.  A thread holds the same few bytes of all K rows.  Where every
//   source stays, as the parents of a beam step do, it loads and stores those
//   that go elsewhere, four at a time, and rows that stay are neither read nor
//   written.  Any other map of a group onto itself (swaps, cycles) needs no
//   second buffer either: all rows are loaded, moving or not, then the moving
//   ones stored.
// - expand_kernel: row g of a prompt's state to the K rows of its beams, each
//   byte read once.
// Bound by memory: the bytes of the rows that change, read and written.  3 of 8
// beams of 4 groups, 16 tensors of 268 MB filled to 4001 of 4096: 545 us, 5.2
// TB/s; a prompt's 24 tensors to 4 beams, 0.98 GB: 180 us, 5.4 TB/s (the card
// copies at 5.1).  One row of moves at a time and conditional loads took 234
// registers for 8 beams; lists of four moves take 76.  The same 16 tensors with
// all rows of a group in a cycle: 1.73 ms, 4.8 TB/s; two of each 8 swapped: 1.06.
#include "tokpath_common.h"

namespace gtp {
namespace states {

constexpr int kBlock = 256;
constexpr int kMost = 192;   // tensors per launch, addresses in the arguments
constexpr int kMaxBeams = 64;
constexpr int kDims = GTP_STATE_DIMS;

// A row's bytes as units of kBytes: `run` of them in a run without gaps, runs
// in up to kDims dimensions (the innermost first).
struct Shape {
  uint32_t units;          // per row
  uint32_t run;            // units per run
  uint32_t size[kDims];    // runs along each dimension
  int64_t stride[kDims];   // bytes
  int64_t row_stride;      // bytes
};

struct List {
  void* p[kMost];
};
struct Pairs {
  const void* from[kMost];
  void* to[kMost];
};

__device__ __forceinline__ int64_t offset_of(const Shape& s, uint32_t u, int bytes) {
  uint32_t r = u / s.run;
  int64_t at = (int64_t)(u - r * s.run) * bytes;
#pragma unroll
  for (int d = 0; d < kDims; ++d) {
    if (s.size[d] == 1) continue;
    const uint32_t q = r / s.size[d];
    at += (int64_t)(r - q * s.size[d]) * s.stride[d];
    r = q;
  }
  return at;
}

template <int kBytes>
struct Unit;
template <>
struct Unit<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <>
struct Unit<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <>
struct Unit<4> { typedef uint32_t type; };
template <>
struct Unit<2> { typedef uint16_t type; };
template <>
struct Unit<1> { typedef uint8_t type; };

// The workgroup's tile, group and tensor, `tiles` workgroups for each (tensor, group).
struct Place {
  uint32_t tile, group, tensor;
  __device__ __forceinline__ Place(uint32_t tiles, uint32_t groups) {
    const uint32_t at = (uint32_t)flat_workgroup<kBlock>(), rest = at / tiles;
    tile = at - rest * tiles;
    tensor = rest / groups;
    group = rest - tensor * groups;
  }
};

// kMany: more than 16 beams.
template <int kBytes, bool kMany>
__global__ __launch_bounds__(kBlock) void reorder_kernel(List l, Shape s, const int32_t* parents,
                                                         uint32_t groups, int K, uint32_t tiles,
                                                         uint32_t count, int32_t* bad) {
  using U = typename Unit<kBytes>::type;
  const Place place(tiles, groups);
  const uint32_t tile = place.tile, g = place.group, t = place.tensor;
  if (t >= count) return;
  const int64_t base = (int64_t)g * K;
  // lane k: where row k comes from
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t p = lane < K ? (int64_t)parents[base + lane] - base : lane;
  const bool wrong = lane < K && (p < 0 || p >= K);
  const int from = wrong ? lane : (int)p;
  // a parent outside the group leaves its row as it is
  if (bad && __ballot(wrong) && t == 0 && tile == 0 && threadIdx.x == 0) *bad = 1;
  uint64_t moving = __ballot(from != lane);
  // A wave stays whole (lanes past the row's end repeat its last unit: loaded
  // and stored by the same instructions as that one, the same values).
  uint32_t u = tile * kBlock + threadIdx.x;
  if (moving == 0 || __builtin_amdgcn_readfirstlane(u) >= s.units) return;
  if (u >= s.units) u = s.units - 1;
  const bool apart = __ballot(from != lane && ((moving >> from) & 1)) == 0;
  char* at = reinterpret_cast<char*>(l.p[t]) + base * s.row_stride + offset_of(s, u, kBytes);
  auto row = [&](int k) { return at + (int64_t)k * s.row_stride; };
  if (apart) {
    // every source stays, as a beam step's do: four rows at a time
    while (moving) {
      U v[4];
      int to[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        to[i] = moving ? __ffsll((unsigned long long)moving) - 1 : -1;
        moving &= moving - 1;
        if (to[i] >= 0)
          v[i] = *reinterpret_cast<const U*>(row(__builtin_amdgcn_readlane(from, to[i])));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (to[i] >= 0) *reinterpret_cast<U*>(row(to[i])) = v[i];
    }
    return;
  }
  // all loads ahead of all stores
  if constexpr (!kMany) {
    U v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k)
      v[k] = *reinterpret_cast<const U*>(row(__builtin_amdgcn_readlane(from, k < K ? k : K - 1)));
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if ((moving >> k) & 1) *reinterpret_cast<U*>(row(k)) = v[k];
  } else {
    // 4 bytes at a time: 64 rows of them fit the registers
    constexpr int kPart = kBytes < 4 ? kBytes : 4;
    using P = typename Unit<kPart>::type;
#pragma unroll 1
    for (int o = 0; o < kBytes; o += kPart) {
      P v[kMaxBeams];
#pragma unroll
      for (int k = 0; k < kMaxBeams; ++k)
        v[k] = *reinterpret_cast<const P*>(
            row(__builtin_amdgcn_readlane(from, k < K ? k : K - 1)) + o);
#pragma unroll
      for (int k = 0; k < kMaxBeams; ++k)
        if ((moving >> k) & 1) *reinterpret_cast<P*>(row(k) + o) = v[k];
    }
  }
}

// The copies are contiguous: row_units units of kBytes each.
template <int kBytes>
__global__ __launch_bounds__(kBlock) void expand_kernel(Pairs l, Shape s, uint32_t groups, int K,
                                                        uint32_t tiles, uint32_t count) {
  using U = typename Unit<kBytes>::type;
  const Place place(tiles, groups);
  const uint32_t g = place.group, t = place.tensor;
  const uint32_t u = place.tile * kBlock + threadIdx.x;
  if (t >= count || u >= s.units) return;
  const U v = *reinterpret_cast<const U*>(reinterpret_cast<const char*>(l.from[t]) +
                                          (int64_t)g * s.row_stride + offset_of(s, u, kBytes));
  U* to = reinterpret_cast<U*>(l.to[t]) + (int64_t)g * K * s.units + u;
  for (int k = 0; k < K; ++k) to[(int64_t)k * s.units] = v;
}

// ------------------------------------------------------------------- host

// The unit (16 bytes or the largest power of two that divides every address
// and stride) and the row's shape in it.
int shape_of(const gtp_state_shape* q, uintptr_t addresses, Shape& s, int& bytes) {
  uint64_t all = addresses | (uint64_t)q->run_bytes;
  int64_t runs = 1;
  for (int d = 0; d < kDims; ++d) {
    if (q->sizes[d] < 1) return GTP_ERR_INVALID_ARGUMENT;
    if (q->sizes[d] > 0x7FFFFFFF || runs * q->sizes[d] > 0x7FFFFFFF) return GTP_ERR_UNSUPPORTED;
    runs *= q->sizes[d];
    if (q->sizes[d] > 1) all |= (uint64_t)q->strides[d];
    s.size[d] = (uint32_t)q->sizes[d];
    s.stride[d] = q->strides[d];
  }
  all |= (uint64_t)q->row_stride;
  bytes = 16;
  while (bytes > 1 && all % bytes) bytes /= 2;
  if (q->run_bytes / bytes > 0x7FFFFFFF || q->run_bytes / bytes * runs > 0x7FFFFFFF)
    return GTP_ERR_UNSUPPORTED;
  s.run = (uint32_t)(q->run_bytes / bytes);
  s.units = (uint32_t)(s.run * runs);
  s.row_stride = q->row_stride;
  return GTP_OK;
}

int check(const gtp_state_shape* q, int64_t count, int64_t groups, int32_t beams) {
  if (!q || count < 0 || groups < 0 || beams < 1 || q->run_bytes < 0)
    return GTP_ERR_INVALID_ARGUMENT;
  if (beams > kMaxBeams || groups > 0x7FFFFFFF / beams) return GTP_ERR_UNSUPPORTED;
  return GTP_OK;
}

template <int kBytes>
void reorder(const List& l, const Shape& s, const int32_t* parents, int64_t n, int64_t groups,
             int K, int32_t* bad, hipStream_t st) {
  const uint32_t tiles = (s.units + kBlock - 1) / kBlock;
  const dim3 grid = flat_grid<kBlock>(tiles * groups * n);
  if (K <= 16)
    hipLaunchKernelGGL((reorder_kernel<kBytes, false>), grid, dim3(kBlock), 0, st, l, s, parents,
                       (uint32_t)groups, K, tiles, (uint32_t)n, bad);
  else
    hipLaunchKernelGGL((reorder_kernel<kBytes, true>), grid, dim3(kBlock), 0, st, l, s, parents,
                       (uint32_t)groups, K, tiles, (uint32_t)n, bad);
}

// tensors per launch: their workgroups are counted in 31 bits
int64_t per_launch(const Shape& s, int64_t groups, int64_t count) {
  const int64_t each = ((int64_t)s.units + kBlock - 1) / kBlock * groups;
  int64_t n = 0x7FFFFFFFll / (each > 0 ? each : 1);
  if (n > kMost) n = kMost;
  return n < count ? n : count;
}

// What a call launches: `most` tensors at a time (0: nothing to do).  outs: null
// where the tensors are moved in place.
struct Call {
  Shape s;
  int bytes;
  int64_t most;
};
int look(const void* const* tensors, const void* const* outs, bool in_place, int64_t count,
         const gtp_state_shape* shape, int64_t groups, int32_t beams, Call& c) {
  c.most = 0;
  int rc = check(shape, count, groups, beams);
  if (rc != GTP_OK) return rc;
  if (count == 0 || groups == 0 || shape->run_bytes == 0) return GTP_OK;
  if (!tensors || (!in_place && !outs)) return GTP_ERR_INVALID_ARGUMENT;
  uintptr_t all = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (!tensors[i] || (!in_place && !outs[i])) return GTP_ERR_INVALID_ARGUMENT;
    all |= reinterpret_cast<uintptr_t>(tensors[i]);
    if (!in_place) all |= reinterpret_cast<uintptr_t>(outs[i]);
  }
  rc = shape_of(shape, all, c.s, c.bytes);
  if (rc != GTP_OK) return rc;
  c.most = per_launch(c.s, groups, count);
  return c.most < 1 ? GTP_ERR_UNSUPPORTED : GTP_OK;
}

}  // namespace states
}  // namespace gtp

using namespace gtp;

extern "C" int gtp_reorder_states_check(const void* const* tensors, int64_t count,
                                        const gtp_state_shape* shape, int64_t groups,
                                        int32_t beams) {
  states::Call c;
  return states::look(tensors, nullptr, true, count, shape, groups, beams, c);
}

extern "C" int gtp_reorder_states(void* const* tensors, int64_t count,
                                  const gtp_state_shape* shape, const int32_t* parents,
                                  int64_t groups, int32_t beams, int32_t* bad, void* stream) {
  states::Call c;
  const int rc = states::look(tensors, nullptr, true, count, shape, groups, beams, c);
  if (rc != GTP_OK || c.most == 0) return rc;
  if (!parents) return GTP_ERR_INVALID_ARGUMENT;
  const states::Shape& s = c.s;
  const int64_t most = c.most;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int64_t first = 0; first < count; first += most) {
    const int64_t n = count - first < most ? count - first : most;
    states::List l;
    for (int64_t i = 0; i < n; ++i) l.p[i] = tensors[first + i];
    switch (c.bytes) {
      case 16: states::reorder<16>(l, s, parents, n, groups, beams, bad, st); break;
      case 8: states::reorder<8>(l, s, parents, n, groups, beams, bad, st); break;
      case 4: states::reorder<4>(l, s, parents, n, groups, beams, bad, st); break;
      case 2: states::reorder<2>(l, s, parents, n, groups, beams, bad, st); break;
      default: states::reorder<1>(l, s, parents, n, groups, beams, bad, st); break;
    }
  }
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

extern "C" int gtp_expand_states(const void* const* tensors, void* const* outs, int64_t count,
                                 const gtp_state_shape* shape, int64_t groups, int32_t beams,
                                 void* stream) {
  states::Call c;
  const int rc = states::look(tensors, outs, false, count, shape, groups, beams, c);
  if (rc != GTP_OK || c.most == 0) return rc;
  const states::Shape& s = c.s;
  const int64_t most = c.most;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const uint32_t tiles = (s.units + states::kBlock - 1) / states::kBlock;
  for (int64_t first = 0; first < count; first += most) {
    const int64_t n = count - first < most ? count - first : most;
    states::Pairs l;
    for (int64_t i = 0; i < n; ++i) {
      l.from[i] = tensors[first + i];
      l.to[i] = outs[first + i];
    }
    const dim3 grid = flat_grid<states::kBlock>(tiles * groups * n), block(states::kBlock);
    const auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, block, 0, st, l, s, (uint32_t)groups, beams, tiles,
                         (uint32_t)n);
    };
    switch (c.bytes) {
      case 16: run(states::expand_kernel<16>); break;
      case 8: run(states::expand_kernel<8>); break;
      case 4: run(states::expand_kernel<4>); break;
      case 2: run(states::expand_kernel<2>); break;
      default: run(states::expand_kernel<1>); break;
    }
  }
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}
