// tokpath_lora.hip -- low-rank adapters of many requests beside a shared projection (gfx950).
//
// Row n with adapter e = id[n] and scale s_e:
//   u = s_e x A_e^T            [N, r]       out = base + u B_e^T     [N, O]
// and, with g the gradient of out,
//   v = s_e g B_e              [N, r]       dx  = v A_e              [N, K]
//   dA_e = sum_n v_n^T x_n     [r, K]       dB_e = sum_n g_n^T u_n   [O, r]
// (base's gradient is g).  r is small: every product reads or writes one long
// matrix once (a backward's two read g, for v and for dB) and is bound by that, so
// there are three kernels, each on the matrix cores (16x16x32 for 16-bit types,
// 16x16x4 for fp32):
//
// - shrink_kernel: rows x long axis -> [rows, r], the long axis split over
//   waves and workgroups, fp32 partial sums.
// - expand_kernel: [rows, r] -> rows x long axis, added to base.
// - outer_kernel: two tall matrices -> [r, long], rows split over workgroups.
//   Each block of 64 (fp32) or 128 columns loads all of the low-rank operand,
//   which is small beside them at a rank of 16 in 16 bits (a quarter of their
//   bytes) and as much as they are at 64 in fp32.
//
// Rows are sorted by adapter on the device (plan_kernel: a stable counting sort
// of the requests), each adapter's run padded to whole tiles, so a tile has one
// adapter and every sum an order that the ids fix.
//
// u and v are fp32 sums.  As 16-bit operands they are two bf16 parts, hi + lo (16
// bits of them, over fp32's range): rounded once, u alone would cost as much as
// the output's own rounding where base is small, and in fp16 a v below 2^-14,
// as small b or gradients give, would lose its bits.  fp16 values meet them as
// two bf16 parts as well, which is exact.  Both parts have the value's sign and
// are zero only if it is (cut_bf16): with hi to the nearest and lo the rest, one
// bit more is held, but an infinity on either side meets a lo of 0 or of the
// other sign, or becomes inf - inf itself, and the product NaN.
//
// Measured, bf16, 8192 rows of 4096 x 4096 of rank 16 with all gradients: shrink
// 22 and 19 us (64 MB each), expand 35 (128 MB read and written) and 22 (64 MB
// written), outer 31 (128 MB), the rest 10; 138 in all, where 403 MB, and
// g once more, at the card's copying rate are 92.  fp32, 2000 rows of 2048 x 5632, rank 64: 154 us,
// of which the products at fp32's matrix rate are about half.  A few rows: two
// launches of 4-5 us.  Tried without gain: strips' weights loaded ahead (the
// registers cost a wave per SIMD: 35 -> 41 us), 16 rows per wave with more waves
// (48), neighbouring strips in one wave (42), 8 or 16 waves side by side, stores
// past the caches.
#include "tokpath_gemm.h"

namespace gtp {
namespace lora {

using gemm::f32x4;
using gemm::s16x8;

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 256;
constexpr int kRankStep = 64;   // of shrink and outer
constexpr int kWideRank = 32;   // past it both hold four blocks of ranks

// The next bf16 number towards zero, as a float; 0 of 0.  x minus it is exact, of
// x's sign and not 0: an infinity is the largest number and an infinity.
__device__ __forceinline__ float cut_bf16(float x) {
  const uint32_t u = f2u(x);
  return u2f((u - (x != 0.0f ? 1u : 0u)) & 0xFFFF0000u);
}

template <typename T>
struct Mat;
template <>
struct Mat<uint16_t> {
  static constexpr int kE = 8;       // values per 16 bytes
  static constexpr int kParts = 2;   // of a low-rank operand
  __device__ static __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return gemm::Bf16::mul(__builtin_bit_cast(s16x8, a), __builtin_bit_cast(s16x8, b), c);
  }
  // with a low-rank operand
  __device__ static __forceinline__ f32x4 meet(u32x4 a, u32x4 low, f32x4 c) {
    return mma(a, low, c);
  }
  __device__ static __forceinline__ float to(uint16_t v) { return gemm::Bf16::to(v); }
  __device__ static __forceinline__ uint16_t from(float v) { return gemm::Bf16::from(v); }
};
template <>
struct Mat<_Float16> {
  static constexpr int kE = 8;
  static constexpr int kParts = 2;
  __device__ static __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return gemm::F16::mul(__builtin_bit_cast(s16x8, a), __builtin_bit_cast(s16x8, b), c);
  }
  __device__ static __forceinline__ f32x4 meet(u32x4 a, u32x4 low, f32x4 c) {
    u32x4 hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t f[2], d[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = f16_to_f32((uint16_t)(a[k] >> (16 * h)));
        const float top = cut_bf16(x);
        f[h] = f2u(top);
        d[h] = f2u(x - top);
      }
      hi[k] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
      lo[k] = __builtin_amdgcn_perm(d[1], d[0], 0x07060302u);
    }
    c = Mat<uint16_t>::mma(hi, low, c);
    return Mat<uint16_t>::mma(lo, low, c);
  }
  __device__ static __forceinline__ float to(_Float16 v) { return (float)v; }
  __device__ static __forceinline__ _Float16 from(float v) { return (_Float16)v; }
};
template <>
struct Mat<float> {
  static constexpr int kE = 4;
  static constexpr int kParts = 1;
  __device__ static __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a[j]), u2f(b[j]), c, 0, 0, 0);
    return c;
  }
  __device__ static __forceinline__ f32x4 meet(u32x4 a, u32x4 low, f32x4 c) {
    return mma(a, low, c);
  }
  __device__ static __forceinline__ float to(float v) { return v; }
  __device__ static __forceinline__ float from(float v) { return v; }
};

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Any16 {
  u32x4 v;
};

// kE values from p, of which `left` are there; the others are zeros.
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p, int64_t left) {
  constexpr int E = Mat<T>::kE;
  if (left >= E) return reinterpret_cast<const Any16<T>*>(p)->v;
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (j >= left) break;
    if constexpr (E == 4)
      v[j] = __builtin_bit_cast(uint32_t, p[j]);
    else
      v[j / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[j]) << (16 * (j & 1));
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, u32x4 v, int64_t left) {
  constexpr int E = Mat<T>::kE;
  if (left >= E) {
    reinterpret_cast<Any16<T>*>(p)->v = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (j >= left) break;
    if constexpr (E == 4)
      p[j] = u2f(v[j]);
    else
      p[j] = __builtin_bit_cast(T, (uint16_t)(v[j / 2] >> (16 * (j & 1))));
  }
}

// ------------------------------------------------------------------- plan
// Where the rows are in the order of adapters: position p in [0, tiles * T).
// Classes: adapters 0 .. E-1, E: rows without one, E + 1: bad ids.
// In memory (int32): start[E + 3] (a class's first position; the last: the
// end), rows[E + 3], tile[tiles][4] (its class or -1, the class's first request
// in `order` and its rows, the tile's first row among them), order[B].

// Each adapter's scale, or one for all, and where the forward puts them: what
// reads them later, the backward too, has them from there.
struct Scale {
  const float* each;
  float all;
  float* to;
};

struct Tile {
  int e, first, rows, at;
};

__device__ __forceinline__ int class_at(const void* ids, int ids64, int i, int E) {
  const int64_t id = ids64 ? reinterpret_cast<const int64_t*>(ids)[i]
                           : (int64_t)reinterpret_cast<const int32_t*>(ids)[i];
  return id >= 0 && id < E ? (int)id : id == -1 ? E : E + 1;
}

// The plan of at most 64 requests, by every wave that needs it, in registers:
// lane i's request, and lane p's request in their order.
struct Few {
  int c;             // the request's class
  int before, same;  // requests of lower classes, of this one
  int place;         // among those of its class
  int tiles_before, tiles;
  int order;

  __device__ __forceinline__ void make(const void* ids, int ids64, int B, int S, int T, int E,
                                       int lane) {
    c = lane < B ? class_at(ids, ids64, lane, E) : E + 2;
    // by the classes' bits, the highest first: which lanes are alike so far, and
    // how many left them for a lower class
    uint64_t alike = ~0ull;
    before = 0;
    for (int b = 31 - __builtin_clz(E + 2); b >= 0; --b) {
      const bool bit = (c >> b) & 1;
      const uint64_t on = __ballot(bit);
      before += bit ? __popcll(alike & ~on) : 0;
      alike &= bit ? on : ~on;
    }
    same = __popcll(alike);
    place = __popcll(alike & ((1ull << lane) - 1));
    tiles = lane < B ? (same * S + T - 1) / T : 0;
    tiles_before = 0;
    for (uint64_t m = __ballot(lane < B && place == 0); m; m &= m - 1) {
      const int j = __ffsll((unsigned long long)m) - 1;
      tiles_before += __builtin_amdgcn_readlane(c, j) < c ? __builtin_amdgcn_readlane(tiles, j) : 0;
    }
    // (lanes without a request keep out of the requests' places)
    order = __builtin_amdgcn_ds_permute(4 * (lane < B ? before + place : lane), lane);
  }
  // tile t
  __device__ __forceinline__ Tile find(int t, int S, int T, int lane) const {
    const uint64_t m = __ballot(tiles > 0 && place == 0 && t >= tiles_before &&
                                t < tiles_before + tiles);
    if (m == 0) return Tile{-1, 0, 0, 0};
    const int j = __ffsll((unsigned long long)m) - 1;
    return Tile{__builtin_amdgcn_readlane(c, j), __builtin_amdgcn_readlane(before, j),
                __builtin_amdgcn_readlane(same, j) * S,
                (t - __builtin_amdgcn_readlane(tiles_before, j)) * T};
  }
};

struct Plan {
  const int32_t* mem;  // null: all rows in order, adapter 0
  int32_t N, B, S, T, E, tiles;
  const void* ids;     // 64 requests at most, not yet in mem: Few's
  int32_t ids64;

  __host__ __device__ static int64_t head(int64_t E) { return (2 * (E + 3) + 3) / 4 * 4; }
  __host__ __device__ static int64_t words(int64_t B, int64_t E, int64_t tiles) {
    return head(E) + 4 * tiles + B;
  }
  __device__ __forceinline__ int start(int e) const { return mem ? mem[e] : e ? tiles * T : 0; }
  __device__ __forceinline__ int rows(int e) const { return mem ? mem[E + 3 + e] : N; }
  __device__ __forceinline__ Tile tile(int t) const {
    if (!mem) return Tile{0, 0, N, t * T};
    const int4 v = reinterpret_cast<const int4*>(mem + head(E))[t];
    return Tile{v.x, v.y, v.z, v.w};
  }
  // row n of tile t, -1 behind the class's last
  __device__ __forceinline__ int row(const Tile& t, int n) const {
    const int j = t.at + n;
    if (j >= t.rows) return -1;
    if (!mem) return j;
    const int b = j / S;
    return mem[head(E) + 4 * tiles + t.first + b] * S + (j - b * S);
  }
};

// A tile and its rows, for a whole wave.
struct Where {
  Tile tile;
  int order;  // of Few

  __device__ __forceinline__ Where(const Plan& p, int t, int lane) {
    if (p.ids) {
      Few f;
      f.make(p.ids, p.ids64, p.B, p.S, p.T, p.E, lane);
      tile = f.find(t, p.S, p.T, lane);
      order = f.order;
    } else {
      tile = p.tile(t);
      order = 0;
    }
  }
  // row n of the tile, -1 behind the class's last (all lanes call)
  __device__ __forceinline__ int row(const Plan& p, int n) const {
    if (!p.ids) return p.row(tile, n);
    const int j = tile.at + n, b = j / p.S;
    const int request = __shfl(order, (tile.first + b) & (kWave - 1), kWave);
    return j < tile.rows ? request * p.S + (j - b * p.S) : -1;
  }
};

// Few's plan put into memory, by one wave.
__device__ __forceinline__ void keep(const Plan& p, int32_t* mem, int lane) {
  Few f;
  f.make(p.ids, p.ids64, p.B, p.S, p.T, p.E, lane);
  for (int c0 = 0; c0 <= p.E + 2; c0 += kWave) {
    const int c = c0 + lane;
    int start = 0, rows = 0;
    for (uint64_t m = __ballot(lane < p.B && f.place == 0); m; m &= m - 1) {
      const int j = __ffsll((unsigned long long)m) - 1;
      const int o = __builtin_amdgcn_readlane(f.c, j);
      start += o < c ? __builtin_amdgcn_readlane(f.tiles, j) * p.T : 0;
      rows = o == c ? __builtin_amdgcn_readlane(f.same, j) * p.S : rows;
    }
    if (c <= p.E + 2) {
      mem[c] = start;
      mem[p.E + 3 + c] = rows;
    }
  }
  int4* tile = reinterpret_cast<int4*>(mem + Plan::head(p.E));
  for (int t0 = 0; t0 < p.tiles; t0 += kWave) {
    const int t = t0 + lane;
    int4 v = make_int4(-1, 0, 0, 0);
    for (uint64_t m = __ballot(lane < p.B && f.place == 0); m; m &= m - 1) {
      const int j = __ffsll((unsigned long long)m) - 1;
      const int from = __builtin_amdgcn_readlane(f.tiles_before, j);
      if (t >= from && t < from + __builtin_amdgcn_readlane(f.tiles, j))
        v = make_int4(__builtin_amdgcn_readlane(f.c, j), __builtin_amdgcn_readlane(f.before, j),
                      __builtin_amdgcn_readlane(f.same, j) * p.S, (t - from) * p.T);
    }
    if (t < p.tiles) tile[t] = v;
  }
  if (lane < p.B) mem[Plan::head(p.E) + 4 * p.tiles + lane] = f.order;
}

constexpr int kPlanBlock = 1024;
constexpr int kPlanWaves = kPlanBlock / kWave;

// Wave w sorts requests [w B/16, (w + 1) B/16): it counts them by class, the
// counts are summed class by class, and it puts them down in order.
__global__ __launch_bounds__(kPlanBlock) void plan_kernel(const void* ids, int ids64, int B, int S,
                                                          int T, int E, int tiles, int32_t* mem) {
  extern __shared__ int32_t count[];  // [classes][waves]
  __shared__ int32_t first[kMaxAdapters + 2], rows[kMaxAdapters + 2], start[kMaxAdapters + 3];
  const int classes = E + 2, lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  int4* tile = reinterpret_cast<int4*>(mem + Plan::head(E));
  int32_t* order = mem + Plan::head(E) + 4 * tiles;
  for (int i = threadIdx.x; i < classes * kPlanWaves; i += kPlanBlock) count[i] = 0;
  __syncthreads();
  const int share = (B + kPlanWaves - 1) / kPlanWaves;
  const int from = w * share < B ? w * share : B, to = from + share < B ? from + share : B;
  auto class_of = [&](int i) { return class_at(ids, ids64, i, E); };
  // lanes with this lane's class
  auto alike = [&](int c, bool in) {
    uint64_t m = __ballot(in);
    for (int b = 0; (1 << b) < classes; ++b) {
      const uint64_t on = __ballot((c >> b) & 1);
      m &= (c >> b) & 1 ? on : ~on;
    }
    return m;
  };
  const uint64_t below = (1ull << lane) - 1;
  for (int i = from; i < to; i += kWave) {
    const bool in = i + lane < to;
    const int c = in ? class_of(i + lane) : 0;
    const uint64_t m = alike(c, in);
    if (in && (m & below) == 0) count[c * kPlanWaves + w] += __popcll(m);
    wave_lds_sync();
  }
  __syncthreads();
  // exclusive sums: of the requests, and of the positions
  if (threadIdx.x < kWave) {
    int base = 0, pos = 0;
    for (int c0 = 0; c0 < classes; c0 += kWave) {
      const int c = c0 + lane;
      int n = 0;
      if (c < classes) {
#pragma unroll
        for (int k = 0; k < kPlanWaves; ++k) n += count[c * kPlanWaves + k];
      }
      const int padded = (n * S + T - 1) / T * T;
      int a = n, p = padded;
      for (int o = 1; o < kWave; o <<= 1) {
        const int x = __shfl_up(a, o, kWave), y = __shfl_up(p, o, kWave);
        if (lane >= o) {
          a += x;
          p += y;
        }
      }
      if (c < classes) {
        first[c] = base + a - n;
        rows[c] = n * S;
        start[c] = pos + p - padded;
        if (c == classes - 1) start[classes] = pos + p;
      }
      base += __shfl(a, kWave - 1, kWave);
      pos += __shfl(p, kWave - 1, kWave);
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < classes; c += kPlanBlock) {
    int at = first[c];
    mem[c] = start[c];
    mem[E + 3 + c] = rows[c];
    if (c == classes - 1) mem[classes] = start[classes];
    for (int k = 0; k < kPlanWaves; ++k) {
      const int n = count[c * kPlanWaves + k];
      count[c * kPlanWaves + k] = at;
      at += n;
    }
  }
  for (int t = threadIdx.x; t < tiles; t += kPlanBlock) {
    // the last class that begins at or before the tile (empty ones begin where
    // the next one does)
    int lo = 0, hi = classes;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (start[mid] <= t * T) lo = mid;
      else hi = mid;
    }
    tile[t] = t * T < start[classes] ? make_int4(lo, first[lo], rows[lo], t * T - start[lo])
                                     : make_int4(-1, 0, 0, 0);
  }
  __syncthreads();
  for (int i = from; i < to; i += kWave) {
    const bool in = i + lane < to;
    const int c = in ? class_of(i + lane) : 0;
    const uint64_t m = alike(c, in);
    if (in) order[count[c * kPlanWaves + w] + __popcll(m & below)] = i + lane;
    wave_lds_sync();
    if (in && (m & below) == 0) count[c * kPlanWaves + w] += __popcll(m);
    wave_lds_sync();
  }
}

// ----------------------------------------------------------------- shrink

// low[split][position][r] = rows . W_e[r]: x [N, C] against W [E, r, C], both
// along C.  A step is 128 bytes of each row: quad q of the wave takes 32 of
// them, as two 16-byte operands, so that a row's four lanes read a whole line.
template <typename T, int RB, int NB>
__global__ __launch_bounds__(kBlock) void shrink_kernel(Plan plan, const T* x, int64_t ld,
                                                        const T* W, int C, int r, int splits,
                                                        float* low, Scale scale,
                                                        int32_t* kept) {
  constexpr int E = Mat<T>::kE;
  constexpr int kSteps = RB == 1 ? 4 : 1;  // loaded at a time
  constexpr int kRows = RB * 16;
  __shared__ int rows[kRows];
  constexpr int kHalf = NB == 4 && RB == 4 ? 2 : RB;  // blocks of rows summed at a time
  __shared__ float sum[kWaves][kHalf * 16][NB * 16 + 1];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int split = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int r0 = blockIdx.y * kRankStep;
  if (blockIdx.x == plan.tiles * splits) {
    // a workgroup more: what the others' kernels find in memory
    if (blockIdx.y == 0) {
      for (int i = threadIdx.x; i < plan.E; i += kBlock)
        scale.to[i] = scale.each ? scale.each[i] : scale.all;
      if (kept && w == 0) keep(plan, kept, lane);
    }
    return;
  }
  const Where at(plan, tile, lane);
  const int e = at.tile.e;
  if (e < 0 || e >= plan.E) return;
  if (w == 0) {
    const int row = at.row(plan, lane);
    if (lane < kRows) rows[lane] = row;
  }
  __syncthreads();
  const int m = lane & 15, q = lane >> 4;
  const T* px[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    // (a tile's first row is there; rows that are not repeat it)
    const int row = rows[b * 16 + m] < 0 ? rows[0] : rows[b * 16 + m];
    px[b] = x + row * ld + q * 2 * E;
  }
  const T* pw[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int i = r0 + b * 16 + m < r ? r0 + b * 16 + m : r - 1;
    pw[b] = W + ((int64_t)e * r + i) * C + q * 2 * E;
  }
  // the workgroup's steps, its waves by turns
  const int steps = (C + 8 * E - 1) / (8 * E);
  const int turns = (steps + splits * kWaves * kSteps - 1) / (splits * kWaves * kSteps);
  const int share = turns * kWaves * kSteps;
  const int from = split * share;
  const int to = from + share < steps ? from + share : steps;
  f32x4 acc[RB][NB];
#pragma unroll
  for (int a = 0; a < RB; ++a)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // tiles of 32 and 64 rows load a turn ahead; those of 16 mostly have one turn
  constexpr bool kAhead = RB > 1;
  u32x4 nx[kSteps][RB][2], nw[kSteps][NB][2];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int64_t c = (int64_t)(s0 + i) * 8 * E;
      const int64_t left = s0 + i < to ? C - c - q * 2 * E : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < RB; ++b) nx[i][b][h] = load16(px[b] + c + h * E, left - h * E);
#pragma unroll
        for (int b = 0; b < NB; ++b) nw[i][b][h] = load16(pw[b] + c + h * E, left - h * E);
      }
    }
  };
  if (kAhead) load(from + w * kSteps);
  for (int s0 = from + w * kSteps; s0 < to; s0 += kWaves * kSteps) {
    if (!kAhead) load(s0);
    u32x4 vx[kSteps][RB][2], vw[kSteps][NB][2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < RB; ++b) vx[i][b][h] = nx[i][b][h];
#pragma unroll
        for (int b = 0; b < NB; ++b) vw[i][b][h] = nw[i][b][h];
      }
    if (kAhead && s0 + kWaves * kSteps < to) load(s0 + kWaves * kSteps);
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int a = 0; a < RB; ++a)
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[a][b] = Mat<T>::mma(vx[i][a][h], vw[i][b][h], acc[a][b]);
  }
  // acc[a][b][i]: row 16 a + 4 q + i, rank 16 b + m; the waves' sums in order
  const int n = r - r0 < kRankStep ? r - r0 : kRankStep;
  float* to_low = low + ((int64_t)split * plan.tiles + tile) * kRows * r + r0;
#pragma unroll
  for (int a0 = 0; a0 < RB; a0 += kHalf) {
#pragma unroll
    for (int a = 0; a < kHalf; ++a)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[w][a * 16 + 4 * q + i][b * 16 + m] = acc[a0 + a][b][i];
    __syncthreads();
    for (int i = threadIdx.x; i < kHalf * 16 * n; i += kBlock) {
      const int y = i / n, x = i - y * n;
      float v = sum[0][y][x];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) v += sum[k][y][x];
      to_low[(int64_t)(a0 * 16 + y) * r + x] = v;
    }
    if (a0 + kHalf < RB) __syncthreads();
  }
}

// kE low-rank values of a position from k on, the splits' sums; zeros past the
// rank.
template <typename T>
__device__ __forceinline__ void low_sum(const float* low, int64_t split_stride, int splits, int r,
                                        int k, float (&v)[Mat<T>::kE]) {
  constexpr int E = Mat<T>::kE;
#pragma unroll
  for (int j = 0; j < E; ++j) v[j] = 0.0f;
  if (k + E <= r) {
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
      const float* p = low + i * split_stride + k;
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] += p[j];
    }
  } else {
    for (int i = 0; i < splits; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (k + j < r) v[j] += low[i * split_stride + k + j];
  }
}
// Scaled, as the parts' operands.
template <typename T>
__device__ __forceinline__ void low_parts(const float (&v)[Mat<T>::kE], float scale,
                                          u32x4 (&unit)[Mat<T>::kParts]) {
  constexpr int E = Mat<T>::kE, P = Mat<T>::kParts;
#pragma unroll
  for (int h = 0; h < P; ++h) unit[h] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const float x = v[j] * scale;
    if constexpr (E == 4) {
      unit[0][j] = f2u(x);
    } else {
      const float top = cut_bf16(x);
      const uint16_t hi = (uint16_t)(f2u(top) >> 16), lo = gemm::Bf16::from(x - top);
      unit[0][j / 2] |= (uint32_t)hi << (16 * (j & 1));
      unit[1][j / 2] |= (uint32_t)lo << (16 * (j & 1));
    }
  }
}

// The low-rank rows as the products' operands, from the splits' sums, a thread
// for a position's kE values: `units` [positions][parts][chunks] for
// expand_kernel, `turned` [parts][r][positions] for outer_kernel (zeros where
// there is no row of an adapter), either null.
template <typename T>
__device__ __forceinline__ void low_operands(const Plan& plan, const float* low, int splits,
                                             const float* scales, int r, int64_t i, u32x4* units,
                                             T* turned) {
  constexpr int E = Mat<T>::kE, P = Mat<T>::kParts;
  const int64_t n = (int64_t)plan.tiles * plan.T;
  const int chunks = (r + E - 1) / E;
  if (i >= n * chunks) return;
  const int c = (int)(i / n);
  const int64_t p = i - c * n;
  const Tile t = plan.tile((int)(p / plan.T));
  const bool in = t.e >= 0 && t.e < plan.E;
  u32x4 u[P];
  if (in && t.at + (int)(p % plan.T) < t.rows) {
    float v[E];
    low_sum<T>(low + p * r, n * r, splits, r, c * E, v);
    low_parts<T>(v, scales[t.e], u);
  } else {
#pragma unroll
    for (int h = 0; h < P; ++h) u[h] = u32x4{0u, 0u, 0u, 0u};
  }
#pragma unroll
  for (int h = 0; h < P; ++h) {
    if (units && in) units[(p * P + h) * chunks + c] = u[h];
    if (turned) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (c * E + j < r) {
          T x;
          if constexpr (E == 4) x = u2f(u[h][j]);
          else x = __builtin_bit_cast(T, (uint16_t)(u[h][j / 2] >> (16 * (j & 1))));
          turned[((int64_t)h * r + c * E + j) * n + p] = x;
        }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void low_kernel(Plan plan, const float* low, int splits,
                                                     const float* scales, int r, u32x4* units,
                                                     T* turned) {
  low_operands<T>(plan, low, splits, scales, r, (int64_t)blockIdx.x * kBlock + threadIdx.x, units,
                  turned);
}

// ----------------------------------------------------------------- expand

// out[row] = base[row] + low[position] W_e^T: W [E, C, r].  The long axis is
// the product's M: lane (m, q) of a strip of 64 bytes holds 16 consecutive
// bytes of row m.  Contraction units of 16 bytes: the hi part's, then the lo
// part's (which meet the same W).  A strip's base is loaded a strip ahead.
// ready: low_kernel's units; null: summed here, which takes less than a launch
// where a thread has few of them.  turned: as low_kernel's (with ready null).
template <typename T, int RB>
__global__ __launch_bounds__(kBlock, __is_same(T, _Float16) ? 3 : 4) void expand_kernel(
    Plan plan, const float* low, int splits, const float* scales, const T* W, int C, int r,
    const T* base, int64_t ld_base, T* out, int strips, int blocks, const u32x4* ready, T* turned) {
  constexpr int E = Mat<T>::kE, P = Mat<T>::kParts, MB = E / 4;
  constexpr int kRows = RB * 16;
  constexpr int kStrip = 4 * E;  // columns
  extern __shared__ u32x4 frags[];  // [kRows][units + 1]
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int block = blockIdx.x % blocks, tile = blockIdx.x / blocks;
  const int chunks = (r + E - 1) / E, units = P * chunks, ld = units + 1;
  // a thread's low-rank values, ahead of the look at the plan (of a tile without
  // an adapter they are any values, and not used)
  const int n_low = threadIdx.x / chunks, c_low = threadIdx.x - n_low * chunks;
  float v_low[E];
  if (!ready && n_low < kRows)
    low_sum<T>(low + ((int64_t)tile * kRows + n_low) * r, (int64_t)plan.tiles * kRows * r, splits,
               r, c_low * E, v_low);
  const Where at(plan, tile, lane);
  const int e = at.tile.e;
  if (e < 0) return;
  const int m = lane & 15, q = lane >> 4;
  int row[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) row[b] = at.row(plan, b * 16 + m);
  const int first = block * strips * kWaves + w, last = (block + 1) * strips * kWaves;
  u32x4 vb[RB];
  auto load_base = [&](int strip) {
    const int64_t c = (int64_t)strip * kStrip + q * E;
#pragma unroll
    for (int b = 0; b < RB; ++b)
      vb[b] = row[b] >= 0 ? load16(base + row[b] * ld_base + c, C - c) : u32x4{0u, 0u, 0u, 0u};
  };
  if (base) load_base(first);
  // the weights of a strip's units u0 .. u0 + 3: M index m of block b is column
  // E (m / 4) + 4 b + m % 4 of the strip
  auto load_w = [&](int strip, int u0, u32x4 (&to)[MB]) {
    const int u = u0 + q, k = u >= chunks ? u - chunks : u;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      int64_t o = (int64_t)strip * kStrip + E * (m >> 2) + 4 * b + (m & 3);
      if (o >= C) o = C - 1;
      to[b] = load16(W + ((int64_t)e * C + o) * r + k * E, u < units ? r - k * E : 0);
    }
  };
  const bool adapted = e < plan.E;
  if (adapted) {
    if (ready) {
      const u32x4* from = ready + (int64_t)tile * kRows * units;
      for (int i = threadIdx.x; i < kRows * units; i += kBlock)
        frags[i / units * ld + i % units] = from[i];
    } else if (n_low < kRows) {
      u32x4 u[P];
      low_parts<T>(v_low, scales[e], u);
#pragma unroll
      for (int h = 0; h < P; ++h) frags[n_low * ld + h * chunks + c_low] = u[h];
    }
    __syncthreads();
    if (turned && block == 0 && w == 0) {
      // (a lane for a row)
      const int64_t n_all = (int64_t)plan.tiles * kRows;
      const bool in = at.row(plan, lane) >= 0;
      if (lane < kRows)
        for (int k = 0; k < P * r; ++k) {
          const int part = k >= r ? 1 : 0, i = k - part * r;
          const T* f = reinterpret_cast<const T*>(&frags[lane * ld + part * chunks + i / E]);
          turned[k * n_all + tile * kRows + lane] = in ? f[i % E] : T{};
        }
    }
  }
  for (int strip = first; strip < last; strip += kWaves) {
    const int64_t c0 = (int64_t)strip * kStrip;
    if (c0 >= C) break;
    const int64_t c = c0 + q * E, left = C - c;
    u32x4 old[RB];
    if (base) {
#pragma unroll
      for (int b = 0; b < RB; ++b) old[b] = vb[b];
      if (strip + kWaves < last) load_base(strip + kWaves);
    }
    f32x4 acc[RB][MB];
#pragma unroll
    for (int a = 0; a < RB; ++a)
#pragma unroll
      for (int b = 0; b < MB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (adapted) {
      for (int u0 = 0; u0 < units; u0 += 4) {
        const int u = u0 + q;
        u32x4 vw[MB], vl[RB];
        load_w(strip, u0, vw);
#pragma unroll
        for (int a = 0; a < RB; ++a)
          vl[a] = u < units ? frags[(a * 16 + m) * ld + u] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int a = 0; a < RB; ++a)
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[a][b] = Mat<T>::meet(vw[b], vl[a], acc[a][b]);
      }
    }
    const float bad = e > plan.E ? __builtin_nanf("") : 0.0f;
#pragma unroll
    for (int a = 0; a < RB; ++a) {
      if (row[a] < 0 || left <= 0) continue;
      u32x4 v;
#pragma unroll
      for (int j = 0; j < E; j += (E == 4 ? 1 : 2)) {
        if constexpr (E == 4) {
          v[j] = f2u(acc[a][0][j] + (base ? u2f(old[a][j]) : 0.0f) + bad);
        } else {
          float y[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float was = base ? Mat<T>::to(__builtin_bit_cast(
                                         T, (uint16_t)(old[a][j / 2] >> (16 * h))))
                                   : 0.0f;
            y[h] = acc[a][(j + h) / 4][(j + h) % 4] + was + bad;
          }
          v[j / 2] = (uint32_t)__builtin_bit_cast(uint16_t, Mat<T>::from(y[0])) |
                     (uint32_t)__builtin_bit_cast(uint16_t, Mat<T>::from(y[1])) << 16;
        }
      }
      store16(out + (int64_t)row[a] * C + c, v, left);
    }
  }
}

// --------------------------------------------- small pieces of the backward

// A matrix [E][a][b] turned to [E][b][a], in tiles of 32 x 32.
struct Turn {
  const void* in;
  void* out;
  int64_t tiles;  // of all, 0: none
  int a, b;
};

// Ahead of the backward's products, in one launch: a turned, b turned, and
// low_kernel's `turned` of the forward's sums (to null: not).
template <typename T>
__global__ __launch_bounds__(kBlock) void turn_kernel(Turn one, Turn two, Plan plan,
                                                      const float* low, int splits,
                                                      const float* scales, int r, T* to) {
  __shared__ T tile[32][33];
  const int64_t block = flat_workgroup<kBlock>();
  if (block >= one.tiles + two.tiles) {
    if (to)
      low_operands<T>(plan, low, splits, scales, r,
                      (block - one.tiles - two.tiles) * kBlock + threadIdx.x, nullptr, to);
    return;
  }
  const Turn t = block < one.tiles ? one : two;
  const int64_t i = block < one.tiles ? block : block - one.tiles;
  const int across = (t.b + 31) / 32, each = (t.a + 31) / 32 * across;
  const int64_t e = i / each, at = e * t.a * t.b;
  const int k = (int)(i - e * each), x0 = k / across * 32, y0 = k % across * 32;
  const T* in = reinterpret_cast<const T*>(t.in) + at;
  T* out = reinterpret_cast<T*>(t.out) + at;
  const int lane = threadIdx.x & 31, row = threadIdx.x / 32;
#pragma unroll
  for (int j = row; j < 32; j += kBlock / 32)
    if (x0 + j < t.a && y0 + lane < t.b) tile[j][lane] = in[(int64_t)(x0 + j) * t.b + y0 + lane];
  __syncthreads();
#pragma unroll
  for (int j = row; j < 32; j += kBlock / 32)
    if (y0 + j < t.b && x0 + lane < t.a) out[(int64_t)(y0 + j) * t.a + x0 + lane] = tile[lane][j];
}

// ------------------------------------------------------------------ outer

constexpr int kMaxChunk = 1024;  // rows of a chunk, their numbers in LDS

// One of a backward's two: y [N, C] and low [parts][r][positions].
struct Side {
  const void* y;
  const void* low;
  float* part;  // [slots][r][C] (turned: [slots][C][r])
  int64_t ld;
  int32_t C, blocks;  // workgroups along C
  int32_t turned;
};

// part[slot][k][c] = sum over a chunk's rows of one adapter of low[k] y[c].
// Chunk i and adapter e have slot i + e: the next one in the order of positions
// has one of the two raised.  A step is 32 rows: lane (m, q) loads 16 bytes of
// rows 8 q .. 8 q + 7, which turned around are the rows' axis of kE operands.
template <typename T, int NB>
__global__ __launch_bounds__(kBlock) void outer_kernel(Plan plan, Side one, Side two, int r,
                                                       int chunk) {
  constexpr int E = Mat<T>::kE, P = Mat<T>::kParts;
  constexpr int kCols = 16 * E;
  __shared__ float sum[kWaves][16][kCols + 4];
  __shared__ int rows[kMaxChunk];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int i = blockIdx.y, at = blockIdx.x;
  const Side s = at < one.blocks ? one : two;
  const int c0 = (at < one.blocks ? at : at - one.blocks) * kCols;
  const int r0 = blockIdx.z * kRankStep;
  const int64_t n = (int64_t)plan.tiles * plan.T;
  const int m = lane & 15, q = lane >> 4;
  const T* y = reinterpret_cast<const T*>(s.y) + c0 + m * E;
  const T* low = reinterpret_cast<const T*>(s.low);
  const int64_t left = s.C - c0 - m * E;
  const int begin = i * chunk;
  const int end = plan.start(plan.E);  // of the adapters' positions
  const int stop = begin + chunk < end ? begin + chunk : end;
  for (int p = begin + threadIdx.x; p < stop; p += kBlock) {
    const Tile t = plan.tile(p / plan.T);
    rows[p - begin] = plan.row(t, p % plan.T);
  }
  __syncthreads();
  for (int p = begin; p < stop;) {
    const int e = plan.tile(p / plan.T).e;
    const int next = plan.start(e + 1), to = next < stop ? next : stop;
    f32x4 acc[E][NB];
#pragma unroll
    for (int a = 0; a < E; ++a)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int share = ((to - p + kWaves - 1) / kWaves + 31) / 32 * 32;
    const int mine = p + w * share, until = mine + share < to ? mine + share : to;
    u32x4 next_v[8];
    auto load = [&](int s0) {
      // (positions are whole tiles of 16, 32 or 64: 8 of them are there or not)
      const bool in = s0 + q * 8 < until;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int row = in ? rows[s0 + q * 8 + k - begin] : -1;
        next_v[k] = row >= 0 ? load16(y + row * s.ld, left) : u32x4{0u, 0u, 0u, 0u};
      }
    };
    load(mine);
    for (int s0 = mine; s0 < until; s0 += 32) {
      u32x4 v[8], vl[NB][P][2];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = next_v[k];
      load(s0 + 32);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int k = r0 + b * 16 + m;
        const bool in = k < r && s0 + q * 8 < until;
        const T* pl = low + (int64_t)(in ? k : 0) * n + s0 + q * 8;
#pragma unroll
        for (int h = 0; h < P; ++h)
          vl[b][h][0] = load16(pl + h * n * r, in ? E : 0);
        if constexpr (E == 4) vl[b][0][1] = load16(pl + 4, in ? E : 0);
      }
      if constexpr (E == 8) {
        // 8 x 8 values turned: operand j has column 8 m + j of the 8 rows
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u32x4 o;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o[k] = __builtin_amdgcn_perm(v[2 * k + 1][j / 2], v[2 * k][j / 2],
                                         j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < P; ++h) acc[j][b] = Mat<T>::meet(o, vl[b][h][0], acc[j][b]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32x4 o = {v[4 * h][j], v[4 * h + 1][j], v[4 * h + 2][j], v[4 * h + 3][j]};
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[j][b] = Mat<T>::meet(o, vl[b][0][h], acc[j][b]);
          }
      }
    }
    // acc[j][b][k]: rank 16 b + m, column E (4 q + k) + j; the waves' in order
    float* part = s.part + (int64_t)(i + e) * r * s.C;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int j = 0; j < E; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[w][m][E * (4 * q + k) + j] = acc[j][b][k];
      __syncthreads();
      for (int t = threadIdx.x; t < 16 * kCols; t += kBlock) {
        const int x = s.turned ? t % 16 : t / kCols, z = s.turned ? t / 16 : t % kCols;
        const int k = r0 + b * 16 + x, c = c0 + z;
        float v = sum[0][x][z];
#pragma unroll
        for (int wave = 1; wave < kWaves; ++wave) v += sum[wave][x][z];
        if (k < r && c < s.C) part[s.turned ? (int64_t)c * r + k : (int64_t)k * s.C + c] = v;
      }
      __syncthreads();
    }
    p = next;
  }
}

// grad [E][each] from the slots' sums, in order, both sides in one launch
struct Sum {
  const float* part;
  void* grad;
  int64_t each;   // values of an adapter
  int64_t blocks;
};
template <typename T>
__global__ __launch_bounds__(kBlock) void outer_sum_kernel(Plan plan, Sum one, Sum two, int chunk) {
  const int64_t block = flat_workgroup<kBlock>();
  if (block >= one.blocks + two.blocks) return;
  const Sum s = block < one.blocks ? one : two;
  const int64_t t = (block < one.blocks ? block : block - one.blocks) * kBlock + threadIdx.x;
  if (t >= s.each * plan.E) return;
  const int e = (int)(t / s.each);
  const int n = plan.rows(e);
  float v = 0.0f;
  if (n > 0) {
    const int from = plan.start(e) / chunk, to = (plan.start(e) + n - 1) / chunk;
    const float* p = s.part + (int64_t)(from + e) * s.each + (t - e * s.each);
#pragma unroll 8
    for (int i = from; i <= to; ++i, p += s.each) v += *p;
  }
  reinterpret_cast<T*>(s.grad)[t] = Mat<T>::from(v);
}

// ------------------------------------------------------------------- host

// Sizes that the launches and the workspaces go by.
struct Sizes {
  int32_t T, tiles, splits_x, splits_g;
  int64_t plan_bytes, scale_bytes, low_bytes, units_bytes;  // low: the forward's partial sums
};

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Workgroups for the chip, of at least one turn of their waves (shrink_kernel's
// kSteps steps of 128 bytes each).  Every split is a sum more for each low-rank
// value: of tiles of many rows 8 at most, and about 256 workgroups for ranks past
// 32, whose waves have a SIMD to themselves (fp32, 2000 rows, rank 64, all: 154 us,
// with twice or 3/4 of them 162 and 163; bf16, 4096 rows, rank 64: 163 for 174).
int32_t splits_of(int64_t tiles, int64_t C, int64_t size, int T, int r) {
  const int64_t turn = kWaves * (T == 16 ? 4 : 1);
  const int64_t steps = (C * size + 127) / 128;
  int64_t s = (512 + tiles - 1) / tiles, most = (steps + turn - 1) / turn;
  if (T != 16 && r > kWideRank) s = (256 + tiles / 2) / tiles;
  if (T != 16 && most > 8) most = 8;
  if (s > most) s = most;
  return (int32_t)(s < 1 ? 1 : s);
}

Sizes sizes_of(const gtp_lora* q) {
  Sizes z;
  const int64_t N = q->requests * q->rows, size = q->dtype == GTP_DTYPE_F32 ? 4 : 2;
  // 64 rows of fp32 and a rank past 32 take 230 registers in shrink_kernel, 32 rows
  // let three waves run for two (154 us against 163, as above); 16-bit
  // types are level.  (A tile's low-rank rows take 33 KB of LDS at a rank of 128.)
  z.T = N <= 1024 || q->rank > 128 ? 16 : size == 4 && q->rank > kWideRank ? 32 : 64;
  int64_t runs = q->adapters + 2 < q->requests ? q->adapters + 2 : q->requests;
  z.tiles = (int32_t)((N + z.T - 1) / z.T + (q->ids ? runs : 0));
  z.splits_x = splits_of(z.tiles, q->in, size, z.T, q->rank);
  z.splits_g = splits_of(z.tiles, q->out, size, z.T, q->rank);
  z.plan_bytes = q->ids ? round_up(Plan::words(q->requests, q->adapters, z.tiles) * 4, 256) : 0;
  z.scale_bytes = round_up((int64_t)q->adapters * 4, 256);
  z.low_bytes = round_up((int64_t)z.splits_x * z.tiles * z.T * q->rank * 4, 256);
  // low_kernel's operands
  const int64_t E = 16 / size, units = (size == 4 ? 1 : 2) * ((q->rank + E - 1) / E);
  z.units_bytes = (int64_t)z.tiles * z.T * units * 16;
  return z;
}

int check(const gtp_lora* q) {
  if (!q || q->requests < 0 || q->rows < 0 || q->in < 1 || q->out < 1 || q->rank < 1 ||
      q->adapters < 1)
    return GTP_ERR_INVALID_ARGUMENT;
  if (q->dtype != GTP_DTYPE_F32 && q->dtype != GTP_DTYPE_BF16 && q->dtype != GTP_DTYPE_F16)
    return GTP_ERR_INVALID_ARGUMENT;
  if (!q->ids && q->adapters != 1 && q->requests > 0 && q->rows > 0)
    return GTP_ERR_INVALID_ARGUMENT;
  if (q->rank > kMaxRank || q->adapters > kMaxAdapters || q->in > (1 << 24) ||
      q->out > (1 << 24) || q->requests > (1 << 24) || q->rows > (1 << 24) ||
      q->requests * q->rows > (1 << 24) - 131072 ||
      q->rank * (q->in > q->out ? q->in : q->out) > 0x7FFFFFFF ||
      (int64_t)q->adapters * q->rank * (q->in > q->out ? q->in : q->out) > (1ll << 38))
    return GTP_ERR_UNSUPPORTED;
  return GTP_OK;
}

bool aligned(const void* p, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

// few: the plan is not yet in the state, and need not be
Plan plan_of(const gtp_lora* q, const Sizes& z, const void* state, bool few) {
  Plan p;
  p.ids = few ? q->ids : nullptr;
  p.ids64 = q->ids_int64;
  p.mem = q->ids ? reinterpret_cast<const int32_t*>(state) : nullptr;
  p.B = (int32_t)q->requests;
  p.S = (int32_t)q->rows;
  p.N = p.B * p.S;
  p.T = z.T;
  p.E = q->adapters;
  p.tiles = z.tiles;
  return p;
}

template <typename T, int RB, int NB>
void shrink(const Plan& p, const T* x, int64_t ld, const T* W, int64_t C, int r, int splits,
            float* low, Scale scale, int32_t* kept, hipStream_t s) {
  const dim3 grid((uint32_t)((int64_t)p.tiles * splits + (scale.to ? 1 : 0)),
                  (uint32_t)((r + kRankStep - 1) / kRankStep));
  hipLaunchKernelGGL((shrink_kernel<T, RB, NB>), grid, dim3(kBlock), 0, s, p, x, ld, W, (int)C, r,
                     splits, low, scale, kept);
}
template <typename T>
void shrink(const Plan& p, const T* x, int64_t ld, const T* W, int64_t C, int r, int splits,
            float* low, Scale scale, int32_t* kept, hipStream_t s) {
  const auto run = [&](auto kernel) { kernel(p, x, ld, W, C, r, splits, low, scale, kept, s); };
  constexpr int kLarge = sizeof(T) == 4 ? 2 : 4;
  if (p.T == 16)
    run(r <= 16 ? shrink<T, 1, 1> : r <= kWideRank ? shrink<T, 1, 2> : shrink<T, 1, 4>);
  else
    run(r <= 16 ? shrink<T, 4, 1> : r <= kWideRank ? shrink<T, 4, 2> : shrink<T, kLarge, 4>);
}

template <typename T>
void expand(const Plan& p, const float* low, int splits, const float* scales, const T* W, int64_t C,
            int r, const T* base, int64_t ld_base, T* out, const u32x4* ready, T* turned,
            hipStream_t s) {
  constexpr int E = Mat<T>::kE, P = Mat<T>::kParts;
  const int64_t wave_strips = (C + 4 * E * kWaves - 1) / (4 * E * kWaves);
  // strips per wave: fewer where there are few tiles
  int64_t blocks = (1024 + p.tiles - 1) / p.tiles;
  if (blocks > wave_strips) blocks = wave_strips;
  const int strips = (int)((wave_strips + blocks - 1) / blocks);
  blocks = (wave_strips + strips - 1) / strips;
  const size_t lds = (size_t)p.T * (P * ((r + E - 1) / E) + 1) * 16;
  const dim3 grid((uint32_t)(p.tiles * blocks));
  const auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kBlock), lds, s, p, low, splits, scales, W, (int)C, r,
                       base, ld_base, out, strips, (int)blocks, ready, turned);
  };
  if (p.T == 16) {
    run(expand_kernel<T, 1>);
  } else if (p.T == 64) {
    run(expand_kernel<T, 4>);
  } else {
    if constexpr (sizeof(T) == 4) run(expand_kernel<T, 2>);
  }
}

template <typename T>
void low_launch(const Plan& p, const float* low, int splits, const float* scales, int r,
                u32x4* units, T* turned, hipStream_t s) {
  const int64_t n = (int64_t)p.tiles * p.T * ((r + Mat<T>::kE - 1) / Mat<T>::kE);
  hipLaunchKernelGGL(low_kernel<T>, dim3((uint32_t)((n + kBlock - 1) / kBlock)), dim3(kBlock), 0, s,
                     p, low, splits, scales, r, units, turned);
}

// Whether the operands are made in a launch of their own: where expand_kernel
// would have more than 256 of them to sum for a tile (a thread each).
bool low_apart(const gtp_lora* q, const Sizes& z) {
  const int E = q->dtype == GTP_DTYPE_F32 ? 4 : 8;
  return z.T * ((q->rank + E - 1) / E) > kBlock;
}

template <typename T>
void forward(const gtp_lora* q, const Sizes& z, char* state, hipStream_t s) {
  const bool few = q->ids && q->requests <= kWave;
  const Plan p = plan_of(q, z, state, few);
  int32_t* mem = reinterpret_cast<int32_t*>(state);
  if (q->ids && !few)
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanBlock),
                       (size_t)(q->adapters + 2) * kPlanWaves * 4, s, q->ids, (int)q->ids_int64,
                       p.B, p.S, p.T, p.E, p.tiles, mem);
  float* scales = reinterpret_cast<float*>(state + z.plan_bytes);
  float* low = reinterpret_cast<float*>(state + z.plan_bytes + z.scale_bytes);
  shrink<T>(p, reinterpret_cast<const T*>(q->x), q->x_stride, reinterpret_cast<const T*>(q->a),
            q->in, q->rank, z.splits_x, low, Scale{q->scales, q->scale, scales},
            few ? mem : nullptr, s);
  u32x4* units = nullptr;
  if (low_apart(q, z)) {
    units = reinterpret_cast<u32x4*>(state + z.plan_bytes + z.scale_bytes + z.low_bytes);
    low_launch<T>(plan_of(q, z, state, false), low, z.splits_x, scales, q->rank, units,
                  static_cast<T*>(nullptr), s);
  }
  expand<T>(p, low, z.splits_x, scales, reinterpret_cast<const T*>(q->b), q->out, q->rank,
            reinterpret_cast<const T*>(q->base), q->base_stride, reinterpret_cast<T*>(q->y), units,
            static_cast<T*>(nullptr), s);
}

// The backward's workspace.
struct Work {
  int64_t turned_a, turned_b, low_v, units_v, low_tu, low_tv, part_a, part_b, bytes;
  int chunk, chunks;
};

Work work_of(const gtp_lora* q, const Sizes& z) {
  Work k;
  const int64_t size = q->dtype == GTP_DTYPE_F32 ? 4 : 2, parts = size == 4 ? 1 : 2;
  const int64_t n = (int64_t)z.tiles * z.T, r = q->rank, E = q->adapters;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  k.turned_a = take(E * r * q->in * size);
  k.turned_b = take(E * r * q->out * size);
  k.low_v = take((int64_t)z.splits_g * n * r * 4);
  k.units_v = take(z.units_bytes);
  k.low_tu = take(n * r * size * parts);
  k.low_tv = take(n * r * size * parts);
  // chunks of rows: workgroups for the chip, of at least 128 rows; past a rank of
  // 32 outer_kernel runs two to a CU, which 512 fill once, and its four waves have
  // whole steps (fp32, 2000 rows of 2048 x 5632, rank 64: 37 us for 43; at lower
  // ranks 768 are as good, fp32 with a rank of 128 is level)
  const int64_t cols = 16 * (16 / size);
  const int64_t blocks = (q->in + cols - 1) / cols + (q->out + cols - 1) / cols;
  int64_t chunks = r > kWideRank ? 512 / blocks : (768 + blocks - 1) / blocks;
  if (chunks > (n + 127) / 128) chunks = (n + 127) / 128;
  if (chunks < 1) chunks = 1;
  k.chunk = (int)round_up((n + chunks - 1) / chunks, r > kWideRank ? 128 : 64);
  if (k.chunk > kMaxChunk) k.chunk = kMaxChunk;
  k.chunks = (int)((n + k.chunk - 1) / k.chunk);
  k.part_a = take((k.chunks + E) * r * q->in * 4);
  k.part_b = take((k.chunks + E) * r * q->out * 4);
  k.bytes = at;
  return k;
}

template <typename T>
void backward(const gtp_lora* q, const gtp_lora_grads* d, const Sizes& z, const char* state,
              char* ws, hipStream_t s) {
  constexpr int E = Mat<T>::kE;
  const Plan p = plan_of(q, z, state, false);
  const Work k = work_of(q, z);
  const float* scales = reinterpret_cast<const float*>(state + z.plan_bytes);
  const float* low_u = reinterpret_cast<const float*>(state + z.plan_bytes + z.scale_bytes);
  float* low_v = reinterpret_cast<float*>(ws + k.low_v);
  T* turned_a = reinterpret_cast<T*>(ws + k.turned_a);
  T* turned_b = reinterpret_cast<T*>(ws + k.turned_b);
  T* tu = reinterpret_cast<T*>(ws + k.low_tu);
  T* tv = reinterpret_cast<T*>(ws + k.low_tv);
  const int r = q->rank;
  const int64_t na = (int64_t)p.E * r * q->in, nb = (int64_t)p.E * r * q->out;
  const int64_t nl = (int64_t)p.tiles * p.T * ((r + E - 1) / E);
  const bool need_v = d->grad_x || d->grad_a;
  auto blocks_of = [](int64_t n) { return (n + kBlock - 1) / kBlock; };
  auto tiles_of = [](int64_t a, int64_t b) { return (a + 31) / 32 * ((b + 31) / 32); };
  const Turn ta{q->a, turned_a, d->grad_x ? p.E * tiles_of(r, q->in) : 0, r, (int)q->in};
  const Turn tb{q->b, turned_b, need_v ? p.E * tiles_of(q->out, r) : 0, (int)q->out, r};
  const int64_t turns = ta.tiles + tb.tiles + (d->grad_b ? blocks_of(nl) : 0);
  if (turns > 0)
    hipLaunchKernelGGL(turn_kernel<T>, flat_grid<kBlock>(turns), dim3(kBlock), 0, s, ta, tb, p,
                       low_u, z.splits_x, scales, r, d->grad_b ? tu : nullptr);
  if (need_v) {
    u32x4* units = reinterpret_cast<u32x4*>(ws + k.units_v);
    shrink<T>(p, reinterpret_cast<const T*>(d->grad), d->grad_stride, turned_b, q->out, r,
              z.splits_g, low_v, Scale{nullptr, 0.0f, nullptr}, nullptr, s);
    const bool apart = low_apart(q, z) || !d->grad_x;
    T* to = d->grad_a ? tv : nullptr;
    if (apart)
      low_launch<T>(p, low_v, z.splits_g, scales, r, d->grad_x ? units : nullptr, to, s);
    if (d->grad_x)
      expand<T>(p, low_v, z.splits_g, scales, turned_a, q->in, r, static_cast<const T*>(nullptr), 0,
                reinterpret_cast<T*>(d->grad_x), apart ? units : nullptr, apart ? nullptr : to, s);
  }
  if (!d->grad_a && !d->grad_b) return;
  float* part_a = reinterpret_cast<float*>(ws + k.part_a);
  float* part_b = reinterpret_cast<float*>(ws + k.part_b);
  const int64_t cols = 16 * E;
  const Side a{q->x, tv, part_a, q->x_stride, (int32_t)q->in,
               d->grad_a ? (int32_t)((q->in + cols - 1) / cols) : 0, 0};
  const Side b{d->grad, tu, part_b, d->grad_stride, (int32_t)q->out,
               d->grad_b ? (int32_t)((q->out + cols - 1) / cols) : 0, 1};
  const dim3 grid((uint32_t)(a.blocks + b.blocks), (uint32_t)k.chunks,
                  (uint32_t)((r + kRankStep - 1) / kRankStep));
  if (r <= 16)
    hipLaunchKernelGGL((outer_kernel<T, 1>), grid, dim3(kBlock), 0, s, p, a, b, r, k.chunk);
  else if (r <= 32)
    hipLaunchKernelGGL((outer_kernel<T, 2>), grid, dim3(kBlock), 0, s, p, a, b, r, k.chunk);
  else
    hipLaunchKernelGGL((outer_kernel<T, 4>), grid, dim3(kBlock), 0, s, p, a, b, r, k.chunk);
  const Sum sa{part_a, d->grad_a, (int64_t)r * q->in, d->grad_a ? blocks_of(na) : 0};
  const Sum sb{part_b, d->grad_b, (int64_t)r * q->out, d->grad_b ? blocks_of(nb) : 0};
  hipLaunchKernelGGL(outer_sum_kernel<T>, flat_grid<kBlock>(sa.blocks + sb.blocks), dim3(kBlock),
                     0, s, p, sa, sb, k.chunk);
}

}  // namespace lora
}  // namespace gtp

using namespace gtp;

extern "C" size_t gtp_lora_state_bytes(const gtp_lora* q) {
  if (lora::check(q) != GTP_OK) return 0;
  if (q->requests * q->rows == 0) return 256;
  const lora::Sizes z = lora::sizes_of(q);
  return (size_t)(z.plan_bytes + z.scale_bytes + z.low_bytes +
                  (lora::low_apart(q, z) ? z.units_bytes : 0));
}

extern "C" int gtp_lora_add(const gtp_lora* q, void* state, size_t state_bytes, void* stream) {
  const int rc = lora::check(q);
  if (rc != GTP_OK) return rc;
  const int64_t N = q->requests * q->rows;
  if (N == 0) return GTP_OK;
  const uintptr_t size = q->dtype == GTP_DTYPE_F32 ? 4 : 2;
  if (!q->x || !q->a || !q->b || !q->base || !q->y || !state ||
      q->x_stride < 0 || q->base_stride < 0 || state_bytes < gtp_lora_state_bytes(q) ||
      !lora::aligned(state, 16) || !lora::aligned(q->scales, 4) || !lora::aligned(q->x, size) ||
      !lora::aligned(q->a, size) || !lora::aligned(q->b, size) || !lora::aligned(q->base, size) ||
      !lora::aligned(q->y, size) || (q->ids && !lora::aligned(q->ids, q->ids_int64 ? 8 : 4)))
    return GTP_ERR_INVALID_ARGUMENT;
  const lora::Sizes z = lora::sizes_of(q);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  char* mem = reinterpret_cast<char*>(state);
  if (q->dtype == GTP_DTYPE_BF16) lora::forward<uint16_t>(q, z, mem, s);
  else if (q->dtype == GTP_DTYPE_F16) lora::forward<_Float16>(q, z, mem, s);
  else lora::forward<float>(q, z, mem, s);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

extern "C" size_t gtp_lora_backward_workspace_bytes(const gtp_lora* q) {
  if (lora::check(q) != GTP_OK) return 0;
  if (q->requests * q->rows == 0) return 256;
  return (size_t)lora::work_of(q, lora::sizes_of(q)).bytes;
}

extern "C" int gtp_lora_backward(const gtp_lora* q, const gtp_lora_grads* d, const void* state,
                                 size_t state_bytes, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const int rc = lora::check(q);
  if (rc != GTP_OK) return rc;
  if (!d) return GTP_ERR_INVALID_ARGUMENT;
  if (q->requests * q->rows == 0) return GTP_ERR_UNSUPPORTED;
  const uintptr_t size = q->dtype == GTP_DTYPE_F32 ? 4 : 2;
  if (!q->x || !q->a || !q->b || !d->grad || !state || !workspace ||
      q->x_stride < 0 || d->grad_stride < 0 || state_bytes < gtp_lora_state_bytes(q) ||
      workspace_bytes < gtp_lora_backward_workspace_bytes(q) || !lora::aligned(state, 16) ||
      !lora::aligned(workspace, 256) || !lora::aligned(q->x, size) ||
      !lora::aligned(q->a, size) || !lora::aligned(q->b, size) ||
      !lora::aligned(d->grad, size) || (d->grad_x && !lora::aligned(d->grad_x, size)) ||
      (d->grad_a && !lora::aligned(d->grad_a, size)) ||
      (d->grad_b && !lora::aligned(d->grad_b, size)))
    return GTP_ERR_INVALID_ARGUMENT;
  const lora::Sizes z = lora::sizes_of(q);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const char* mem = reinterpret_cast<const char*>(state);
  char* ws = reinterpret_cast<char*>(workspace);
  if (q->dtype == GTP_DTYPE_BF16) lora::backward<uint16_t>(q, d, z, mem, ws, s);
  else if (q->dtype == GTP_DTYPE_F16) lora::backward<_Float16>(q, d, z, mem, ws, s);
  else lora::backward<float>(q, d, z, mem, ws, s);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}
