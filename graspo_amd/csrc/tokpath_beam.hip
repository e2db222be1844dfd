// tokpath_beam.hip -- one step of a beam search over vocabulary-wide logits (gfx950).
//
// For beam k of a group and token v the candidate's score is
//   c[k, v] = score[k] + x[k, v] - log sum_w exp x[k, w],
// and a group's n best (c descending, then beam, then token) go on: finished
// ones into the group's pool, the others into its K slots.
//
// - beam_slices_kernel: each wave streams a slice of one row once.  A chunk of
//   2048 16-bit (1024 fp32) logits is folded into a running sum of exponentials
//   (one reference for the wave, in base 2).  Of what lies above the slice's
//   running threshold only the vector of 8 (4) is noted, by a ballot; 64 of them
//   are read again at a time, a lane each, and their values above the threshold
//   listed; the list is cut to about its n best and the threshold rises to the
//   last of them.  Within a row the order by logit is the order by score, so n
//   per slice do.
// - beam_merge_kernel: a workgroup per group turns the slices' sums into each
//   row's log-sum-exp in 64 bits (scores of different beams are compared; what
//   is left of fp32 in them are the slices' sums and their exponentials), takes
//   the n best of K S n candidates and, in its first wave, one lane per
//   candidate, moves the group on.
// The rows' bytes bound the large calls, two launches and the merge's chain of
// LDS steps the small ones.  bf16 [32 x 8, 248320]: 31 + 9 us (4.1 TB/s; without
// any candidates 28, without exponentials either 27); [1 x 4, 151936]: 7.5 + 6.6
// us, 16 with the host's part.  What brought the slices there, [256, 248320] and
// [64, 151936]: every value above the threshold appended by ballots 63 and 27 us;
// the code a quarter of that size (a wave that runs for 10 us waits for its
// instructions, too) 50 and 27; only vectors noted, the list cut to between n and
// n + n / 2 by halving between the threshold and the largest 31 and 13.  The merge:
// rankings of all against all 37 us; a threshold from groups' maxima, candidates
// held in registers, all loads ahead 7.
#include "tokpath_stream.h"

namespace gtp {
namespace beam {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kU = 4;           // 16-byte vectors per lane and chunk
constexpr int kNoted = 320;     // vectors noted per wave: 63 and a chunk's 256
constexpr int kCap = 640;       // list entries per wave: kMaxSlots and a batch's 512
constexpr int kMaxN = 64;       // candidates: one lane each
constexpr int kMaxK = 32;
constexpr int kMaxSlots = 80;   // keys that a slice gives: n and some more (slots_of)
constexpr int kMaxKeys = 8192;  // K S slots: what the merge holds in registers

struct Rows {
  const void* x;
  const uint8_t* mask;   // bit v of a row: token v is allowed
  const float* score;    // [G, K]
  const uint8_t* done;   // [G] or null
  int64_t V, group_stride, beam_stride, mask_stride;  // mask_stride in bytes
  int32_t G, K, n, S, slots;
  uint32_t row_magic;    // i / (S slots) = i row_magic >> 32, i < kMaxKeys
  int64_t L;             // a slice's logits, a multiple of 512
  uint64_t* keys;        // [G K S slots], 0: none
  float2* sums;          // [G K S]: maximum, sum
};

// A slice's sum is s = sum 2^{(x - m) c + r(m)} with c the fp32 log2(e), where
// the exponents come from one fma, x c - fl(m c), so that r(m) = m c - fl(m c).
// From |m| = 2^16 on r could overflow the exponential: (x - m) c there, r = 0.
__device__ __forceinline__ bool by_fma(float m) { return __builtin_fabsf(m) < 65536.0f; }
__device__ __forceinline__ float residual(float m) {
  return by_fma(m) ? __builtin_fmaf(m, kLog2e, -(m * kLog2e)) : 0.0f;
}

// How many of the mask's lanes lie below this one.
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// A beam that goes on: a finite score in a group that is not done.
__device__ __forceinline__ bool live(const Rows& r, int row) {
  return !(r.done && r.done[row / r.K]) && __builtin_fabsf(r.score[row]) < kPosInf;
}

// A wave's list of what lay above its threshold: cut to the best, in no order,
// when it grows.  count, tau and the list are the same for all lanes.
struct Top {
  uint64_t* list;
  int count;
  float tau;

  // Keeps the best, n to slots of them (count > slots).  most: no value lies
  // above it.  Which of the others stay makes no difference to the n best, and
  // few halvings end between n and slots.
  __device__ __forceinline__ void cut(int n, int slots, float most, int lane) {
    wave_lds_sync();
    // up to 128 entries two per lane; more are read again for each count
    const bool few = count <= 2 * kWave;
    const uint64_t a = lane < count ? list[lane] : 0;
    const uint64_t b = lane + kWave < count ? list[lane + kWave] : 0;
    auto at_least = [&](uint64_t t) {
      int c = __popcll(__ballot(a >= t)) + __popcll(__ballot(b >= t));
      if (!few)
        for (int i = 2 * kWave; i < count; i += kWave)
          c += __popcll(__ballot(i + lane < count && list[i + lane] >= t));
      return __builtin_amdgcn_readfirstlane(c);
    };
    // between the threshold and the largest, by the first 32 bits
    uint32_t lo = __builtin_amdgcn_readfirstlane(ord32(tau));
    uint32_t hi = __builtin_amdgcn_readfirstlane(ord32(most + 0.0f));
    int c = count;
    while (lo < hi && c > slots) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      const int m = at_least((uint64_t)mid << 32);
      if (m >= n) {
        lo = mid;
        c = m;
      } else {
        hi = mid - 1;
      }
    }
    uint64_t T = (uint64_t)lo << 32;
    // many equal ones: the lowest tokens of them
    for (int i = 31; i >= 0 && c > slots; --i) {
      const uint64_t t = T | (1ull << i);
      const int m = at_least(t);
      if (m >= n) {
        T = t;
        c = m;
      }
    }
    int kept = 0;
    for (int i = 0; i < count; i += kWave) {
      const uint64_t x = i + lane < count ? list[i + lane] : 0;
      wave_lds_sync();
      const uint64_t k = __ballot(x >= T);
      if (x >= T) list[kept + lanes_below(k)] = x;
      wave_lds_sync();
      kept += __popcll(k);
    }
    count = kept;
    // (n entries lie at lo or above, and what comes later has a larger token)
    tau = unord32(lo);
  }
};

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned {
  u32x4 v;
};

// The vector at element i of a row, as far as `end`; what lies past it is -inf.
template <typename T>
__device__ __forceinline__ u32x4 load_vec(const T* row, int64_t i, int64_t end) {
  constexpr int E = Vec<T>::kE, kBits = 8 * sizeof(T);
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u
                             : __is_same(T, _Float16) ? 0xFC00FC00u : 0xFF80FF80u;
  u32x4 v = {kNone, kNone, kNone, kNone};
  if (i + E <= end) return reinterpret_cast<const Unaligned<T>*>(row + i)->v;
  if (i >= end) return v;
  // one element on: towards the first, or the last
  auto down = [](u32x4 x, uint32_t in) {
    if constexpr (kBits == 32) return u32x4{x[1], x[2], x[3], in};
    else
      return u32x4{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16, x[2] >> 16 | x[3] << 16,
                   x[3] >> 16 | in << 16};
  };
  if (end >= E) {
    // the row's last E, moved down to begin with element i
    v = reinterpret_cast<const Unaligned<T>*>(row + end - E)->v;
#pragma unroll 1
    for (int64_t k = i + E - end; k > 0; --k) v = down(v, kNone);
  } else {
    // (a row of fewer than E)
#pragma unroll 1
    for (int j = 0; j < E; ++j) {
      uint32_t x = kNone;
      if (j < end) {
        if constexpr (kBits == 32) x = __builtin_bit_cast(uint32_t, row[j]);
        else x = __builtin_bit_cast(uint16_t, row[j]);
      }
      v = down(v, x);
    }
  }
  return v;
}

// The float below t (not below -inf), for "more than that" in "at least t"'s place.
__device__ __forceinline__ float below(float t) {
  const uint32_t u = f2u(t);
  if (t == kNegInf) return t;
  if (t == 0.0f) return u2f(0x80000001u);
  return u2f(u & 0x80000000u ? u + 1 : u - 1);
}

// 64 lanes in `groups` (a power of two) of neighbours: the least of their maxima.
__device__ __forceinline__ float least_maximum(float v, int groups) {
  const int each = kWave / groups;
#define GTP_STEP(J)                                       \
  {                                                       \
    const float o = u2f(lane_xor<J>(f2u(v)));             \
    v = J < each ? fmaxf(v, o) : fminf(v, o);             \
  }
  GTP_STEP(1) GTP_STEP(2) GTP_STEP(4) GTP_STEP(8) GTP_STEP(16) GTP_STEP(32)
#undef GTP_STEP
  return u2f(__builtin_amdgcn_readfirstlane(f2u(v)));
}

// A wave's maximum, in a scalar register.
__device__ __forceinline__ float uniform_max(float v) {
  v = fmaxf(v, u2f(lane_xor<1>(f2u(v))));
  v = fmaxf(v, u2f(lane_xor<2>(f2u(v))));
  v = fmaxf(v, u2f(lane_xor<4>(f2u(v))));
  v = fmaxf(v, u2f(lane_xor<8>(f2u(v))));
  v = fmaxf(v, u2f(lane_xor<16>(f2u(v))));
  v = fmaxf(v, u2f(lane_xor<32>(f2u(v))));
  return u2f(__builtin_amdgcn_readfirstlane(f2u(v)));
}

// A slice's state, carried from chunk to chunk.  The code is kept small: the
// kernel runs a few microseconds, of which fetching it for the first time is a
// part that all waves wait for.
template <typename T, bool kMask>
struct Slice {
  static constexpr int E = Vec<T>::kE;
  static constexpr int64_t kChunk = (int64_t)kU * kWave * E;
  const T* x;
  const uint8_t* mask;
  uint32_t* noted;  // LDS: vectors of the slice
  int64_t begin, end;
  int n, slots, lane, notes;
  Top top;
  float top_x, s;  // the wave's maximum, the lane's sum
  u32x4 v[kU];
  uint32_t bits[kU];

  // the kE bits of the vector at element i
  __device__ __forceinline__ uint32_t bits_at(int64_t i) const {
    return (uint32_t)mask[i >> 3] >> (E == 4 ? i & 7 : 0);
  }
  __device__ __forceinline__ void load(int64_t e) {
    const int64_t i0 = e + (int64_t)lane * E;
    if (e + kChunk <= end) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        v[u] = reinterpret_cast<const Unaligned<T>*>(x + i0 + u * kWave * E)->v;
        if constexpr (kMask) bits[u] = bits_at(i0 + u * kWave * E);
      }
    } else if (e < end) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t i = i0 + u * kWave * E;
        v[u] = load_vec(x, i, end);
        if constexpr (kMask) bits[u] = i < end ? bits_at(i) : 0u;
      }
    }
  }

  // Lists what lies above the threshold in 64 of the noted vectors from `first`
  // on, or the fewer that there are: in the order of their tokens, for of equal
  // logits the first count.
  __device__ __forceinline__ void take(int first) {
    float y[E];
    int64_t i = 0;
    uint32_t hits = 0;
    if (first + lane < notes) {
      i = begin + (int64_t)noted[first + lane] * E;
      Vec<T>::cvt(load_vec(x, i, end), y);
#pragma unroll
      for (int j = 0; j < E; ++j) hits |= y[j] > top.tau ? 1u << j : 0u;
      if constexpr (kMask) hits &= bits_at(i);
    }
    const uint32_t mine = __popc(hits), upto = wave_scan_u32(mine);
    int to = top.count + (int)(upto - mine);
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (hits >> j & 1u) top.list[to++] = rank_key(y[j] + 0.0f, (int32_t)i + j);
    top.count += __builtin_amdgcn_readlane(upto, kWave - 1);
    if (top.count > slots) top.cut(n, slots, top_x, lane);
  }

  // Folds the chunk at e, with the next one's loads on their way (ahead of the
  // first one: only those).
  __device__ __forceinline__ void fold(int64_t e) {
    u32x4 now[kU];
    uint32_t allowed[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      now[u] = v[u];
      if constexpr (kMask) allowed[u] = bits[u];
    }
    load(e + kChunk);
    if (e < begin) return;

    float y[kU][E], m[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      Vec<T>::cvt(now[u], y[u]);
      m[u] = vec_max<E>(y[u]);
    }
    const float most = max3raw(max3raw(m[0], m[1], m[2]), m[3], m[3]);
    static_assert(kU == 4, "");
    if (__ballot(most > top_x)) {
      const float up = uniform_max(fmaxf(most, top_x));
      if (top_x > kNegInf)
        s *= __builtin_amdgcn_exp2f((top_x - up) * kLog2e + (residual(up) - residual(top_x)));
      top_x = up;
    }
    const float from = top_x == kNegInf ? 0.0f : top_x;
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (by_fma(from)) {
      const float base = -(from * kLog2e);
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int j = 0; j < E; ++j)
          part[j & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(y[u][j], kLog2e, base));
    } else {
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int j = 0; j < E; ++j)
          part[j & 3] += __builtin_amdgcn_exp2f((y[u][j] - from) * kLog2e);
    }
    s += (part[0] + part[1]) + (part[2] + part[3]);

    if constexpr (kMask) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        m[u] = kNegInf;
#pragma unroll
        for (int j = 0; j < E; ++j)
          m[u] = max3raw(m[u], (allowed[u] >> j) & 1u ? y[u][j] : kNegInf, m[u]);
      }
    }
    if (e == begin) {
      // as many groups of lanes as candidates: each one's maximum is at least
      // the least of them, a threshold before anything is in the list
      float best = max3raw(max3raw(m[0], m[1], m[2]), m[3], m[3]);
      if (!(best == best)) best = kNegInf;
      const int groups = n <= 1 ? 1 : 1 << (32 - __builtin_clz(n - 1));
      top.tau = below(least_maximum(best, groups));
    }
    const uint32_t id = (uint32_t)((e - begin) / E) + lane;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint64_t k = __ballot(m[u] > top.tau);
      if (k == 0) continue;
      if (m[u] > top.tau) noted[notes + lanes_below(k)] = id + u * kWave;
      notes += __popcll(k);
    }
    const bool last = e + kChunk >= end;
    int taken = 0;
    if (notes >= (last ? 1 : kWave)) {
      wave_lds_sync();
      for (; notes - taken >= (last ? 1 : kWave); taken += kWave) take(taken);
      // fewer than 64 are left
      const int left = notes > taken ? notes - taken : 0;
      const uint32_t id_left = lane < left ? noted[taken + lane] : 0u;
      wave_lds_sync();
      if (lane < left) noted[lane] = id_left;
      notes = left;
    }
  }
};

template <typename T, bool kMask>
__global__ __launch_bounds__(kBlock) void beam_slices_kernel(Rows r) {
  using S = Slice<T, kMask>;
  __shared__ uint64_t lists[kWaves][kCap];
  __shared__ uint32_t noted[kWaves][kNoted];
  const int lane = threadIdx.x & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t at = (int64_t)blockIdx.x * kWaves + wid;
  if (at >= (int64_t)r.G * r.K * r.S) return;
  const int row = (int)(at / r.S), slice = (int)(at % r.S);
  if (!live(r, row)) return;
  S w;
  w.x = reinterpret_cast<const T*>(r.x) + (row / r.K) * r.group_stride +
        (row % r.K) * r.beam_stride;
  w.mask = kMask ? r.mask + row * r.mask_stride : nullptr;
  w.noted = noted[wid];
  w.begin = slice * r.L;
  w.end = w.begin + r.L < r.V ? w.begin + r.L : r.V;
  w.n = r.n;
  w.slots = r.slots;
  w.lane = lane;
  w.notes = 0;
  w.top = Top{lists[wid], 0, kNegInf};
  w.top_x = kNegInf;
  w.s = 0.0f;
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    w.v[u] = u32x4{0u, 0u, 0u, 0u};
    w.bits[u] = 0u;
  }
#pragma unroll 1
  for (int64_t e = w.begin - S::kChunk; e < w.end; e += S::kChunk) w.fold(e);

  wave_lds_sync();
  for (int i = lane; i < r.slots; i += kWave)
    r.keys[at * r.slots + i] = i < w.top.count ? w.top.list[i] : 0ull;
  float s = w.s;
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
  if (lane == 0) r.sums[at] = make_float2(w.top_x, s);
}

// ------------------------------------------------------------------ a step

struct State {
  const float* score;       // [G, K]
  const float* pool_score;  // [G, K], best first, -inf: empty
  const int32_t* pool_row;
  const int32_t* pool_step;
  const uint8_t* done;
  int64_t* token;           // outputs
  int32_t* parent;
  float* new_score;
  float* new_pool_score;
  int32_t* new_pool_row;
  int32_t* new_pool_step;
  uint8_t* new_done;
  int64_t eos, pad;
  double length;            // (step + 1)^penalty
  int32_t step, early;
};

struct Candidates {
  float score[kMaxN];
  int32_t beam[kMaxN];   // -1: none (score -inf)
  int64_t token[kMaxN];
};

// Lane k's beam and pool entry, read ahead of the candidates.
struct Before {
  float score, pool_score;
  int32_t pool_row, pool_step;
  bool done;
};
__device__ __forceinline__ Before before(const State& st, int g, int K, int lane) {
  Before b;
  const int64_t i = (int64_t)g * K + (lane < K ? lane : 0);
  b.score = st.score[i];
  b.pool_score = st.pool_score[i];
  b.pool_row = st.pool_row[i];
  b.pool_step = st.pool_step[i];
  b.done = st.done[g] != 0;
  return b;
}

__device__ __forceinline__ float lane_float(float v, int from) {
  return u2f(__builtin_amdgcn_readlane(f2u(v), from));
}

// Moves group g on, by one wave; c: its n candidates, best first.
__device__ __forceinline__ void advance(const State& st, const Before& old, const Candidates& c,
                                        int g, int K, int n, int lane) {
  const int64_t base = (int64_t)g * K;
  const uint64_t below_lane = (1ull << lane) - 1;
  if (old.done) {
    if (lane < K) {
      st.token[base + lane] = st.pad;
      st.parent[base + lane] = (int32_t)base + lane;
      st.new_score[base + lane] = old.score;
      st.new_pool_score[base + lane] = old.pool_score;
      st.new_pool_row[base + lane] = old.pool_row;
      st.new_pool_step[base + lane] = old.pool_step;
    }
    if (lane == 0) st.new_done[g] = 1;
    return;
  }
  const bool mine = lane < n;
  const int beam = mine ? c.beam[lane] : -1;
  const float score = mine ? c.score[lane] : kNegInf;
  const int64_t token = mine ? c.token[lane] : -1;
  const bool valid = beam >= 0;
  const bool ended = valid && token == st.eos;
  // The pool: what it held (lane k's), then the finished ones among the first K
  // candidates; of equal scores the earlier stays ahead.
  const float held = lane < K ? old.pool_score : kNegInf;
  const float fresh = lane < K && ended ? (float)((double)score / st.length) : kNegInf;
  int rank_held = 0, rank_fresh = 0;
  for (int i = 0; i < K; ++i) {
    const float h = lane_float(held, i), f = lane_float(fresh, i);
    rank_held += (h > held || (h == held && i < lane)) + (f > held);
    rank_fresh += (h >= fresh) + (f > fresh || (f == fresh && i < lane));
  }
  if (lane < K && rank_held < K) {
    st.new_pool_score[base + rank_held] = held;
    st.new_pool_row[base + rank_held] = held == kNegInf ? -1 : old.pool_row;
    st.new_pool_step[base + rank_held] = held == kNegInf ? -1 : old.pool_step;
  }
  if (lane < K && rank_fresh < K) {
    st.new_pool_score[base + rank_fresh] = fresh;
    st.new_pool_row[base + rank_fresh] = fresh == kNegInf ? -1 : (int32_t)base + beam;
    st.new_pool_step[base + rank_fresh] = fresh == kNegInf ? -1 : st.step;
  }
  const uint64_t last_held = __ballot(lane < K && rank_held == K - 1);
  const uint64_t last_fresh = __ballot(lane < K && rank_fresh == K - 1);
  const float last = last_held ? lane_float(held, __ffsll((unsigned long long)last_held) - 1)
                     : last_fresh ? lane_float(fresh, __ffsll((unsigned long long)last_fresh) - 1)
                                  : kNegInf;
  // The first K others go on: a beam's best one stays in its slot, the rest
  // take the free slots in order; slots beyond the candidates' are dead.
  const uint64_t others = __ballot(mine && !ended);
  const int j = __popcll(others & below_lane);
  const bool goes = mine && !ended && j < K;
  const uint64_t going = __ballot(goes && valid);
  uint32_t taken = 0;
  uint64_t staying = 0;
  for (uint64_t left = going; left; left &= left - 1) {
    const int i = __ffsll((unsigned long long)left) - 1;
    const uint32_t slot = 1u << __builtin_amdgcn_readlane(beam, i);
    if (!(taken & slot)) staying |= 1ull << i;
    taken |= slot;
  }
  const bool stays = (staying >> lane) & 1;
  const uint64_t moving = __ballot(goes && !stays);
  uint32_t free = ~taken;
  if (goes) {
    int slot = beam;
    if (!stays) {
      for (int i = __popcll(moving & below_lane); i > 0; --i) free &= free - 1;
      slot = __ffs((int)free) - 1;
    }
    st.token[base + slot] = valid ? token : st.pad;
    st.parent[base + slot] = (int32_t)base + (valid ? beam : slot);
    st.new_score[base + slot] = valid ? score : kNegInf;
  }
  if (__popcll(__ballot(goes)) < K) {
    free = ~taken;
    for (int i = __popcll(moving); i > 0; --i) free &= free - 1;
    if (lane < K && ((free >> lane) & 1u)) {
      st.token[base + lane] = st.pad;
      st.parent[base + lane] = (int32_t)base + lane;
      st.new_score[base + lane] = kNegInf;
    }
  }
  // the best that a live beam's score reaches at this length
  const int first = going ? __ffsll((unsigned long long)going) - 1 : 0;
  const float best = going ? (float)((double)lane_float(score, first) / st.length) : kNegInf;
  if (lane == 0)
    st.new_done[g] = (last > kNegInf && (st.early || last >= best)) || !going ? 1 : 0;
}

__device__ __forceinline__ uint64_t ord64(double d) {
  const uint64_t u = __builtin_bit_cast(uint64_t, d + 0.0);
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unord64(uint64_t o) {
  return __builtin_bit_cast(double, (o >> 63) ? o & 0x7FFFFFFFFFFFFFFFull : ~o);
}

struct Out {
  float* score;    // [G, n], each null or all
  int32_t* beam;
  int64_t* token;
  int32_t* status;  // [G K] or null
};

constexpr int kMergeBlock = 1024;
constexpr int kMergeWaves = kMergeBlock / kWave;
constexpr int kHold = kMaxKeys / kMergeBlock;  // candidates per thread, in registers
constexpr int kList = 1024;                    // candidates that are compared with each other

__device__ __forceinline__ double lane_xor_double(double v, int o) {
  const uint64_t u = shfl_xor_u64(__builtin_bit_cast(uint64_t, v), o);
  return __builtin_bit_cast(double, u);
}

template <bool kStep>
__global__ __launch_bounds__(kMergeBlock) void beam_merge_kernel(Rows r, Out out, State st) {
  __shared__ double offset[kMaxK];  // score - log sum 2^{(x - m) c}; -inf: no candidates
  __shared__ float row_top[kMaxK];  // m
  __shared__ uint32_t best[kMergeWaves][kWave];
  __shared__ uint64_t list_o[kList], list_at[kList];
  __shared__ Candidates c;
  __shared__ int entries;
  __shared__ int row_any[kMaxK], row_status[kMaxK];
  const int g = (int)flat_workgroup<kMergeBlock>();
  if (g >= r.G) return;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int per_row = r.S * r.slots, total = r.K * per_row;
  const int64_t base = (int64_t)g * r.K;
  // All that is read from memory first, whether it will be needed or not: each
  // wait for it is a microsecond.  (What beams that are not live left in the
  // workspace is any bits, and not looked at.)
  uint64_t key[kHold];
#pragma unroll
  for (int j = 0; j < kHold; ++j) {
    key[j] = 0;
    const int i = j * kMergeBlock + tid;
    if (j * kMergeBlock < total && i < total) key[j] = r.keys[base * per_row + i];
  }
  Before old;
  if constexpr (kStep) {
    if (wid == 0) old = before(st, g, r.K, lane);
  }
  const bool done = r.done && r.done[g];
  if (tid == 0) entries = 0;
  if (tid < kMaxK) row_any[tid] = 0;
  if (tid < r.n) {
    c.score[tid] = kNegInf;
    c.beam[tid] = -1;
    c.token[tid] = -1;
  }
  // each row's log-sum-exp (S <= 64: a slice per lane)
  for (int k = wid; k < r.K; k += kMergeWaves) {
    const float score = r.score[base + k];
    float2 v = r.sums[(base + k) * r.S + (lane < r.S ? lane : 0)];
    int status = GTP_ROW_OK;
    double off = -__builtin_huge_val();
    float top = kNegInf;
    if (!done && __builtin_fabsf(score) < kPosInf) {
      if (lane >= r.S) v = make_float2(kNegInf, 0.0f);
      top = uniform_max(v.x);
      // (a NaN stays, also where nothing finite was seen)
      double s = (double)v.y;
      if (v.x > kNegInf && v.x < kPosInf)
        s *= exp2(((double)v.x - (double)top) * (double)kLog2e - (double)residual(v.x));
#pragma unroll
      for (int o = kWave / 2; o > 0; o >>= 1) s += lane_xor_double(s, o);
      // (the exponents are multiples of the fp32 log2(e); without a sum there
      // is no candidate either)
      if (s != s) status = GTP_ROW_NONFINITE;
      else off = (double)score - log2(s) / (double)kLog2e;
    } else if (!done && !(score == kNegInf)) {
      status = GTP_ROW_NONFINITE;
    }
    if (lane == 0) {
      offset[k] = off;
      row_top[k] = top;
      row_status[k] = status;
    }
  }
  __syncthreads();
  if (!done) {
    // a candidate's score in an order of integers (0: none) and its place
    uint64_t o[kHold];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      o[j] = 0;
      if (j * kMergeBlock >= total) continue;
      const int k = (int)__umulhi(j * kMergeBlock + tid, r.row_magic);
      if (key[j] == 0 || offset[k] == -__builtin_huge_val()) continue;
      row_any[k] = 1;
      o[j] = ord64(((double)rank_key_y(key[j]) - (double)row_top[k]) + offset[k]);
      const uint32_t h = (uint32_t)(o[j] >> 32);
      top = h > top ? h : top;
    }
    auto place = [&](int j) {
      return (uint64_t)__umulhi(j * kMergeBlock + tid, r.row_magic) << 32 |
             (uint32_t)rank_key_id(key[j]);
    };
    best[wid][lane] = top;
    __syncthreads();
    // groups of lanes, as many as candidates are wanted or more: the least of
    // their maxima is a threshold that enough of them reach
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w) m = best[w][lane] > m ? best[w][lane] : m;
    const int groups = r.n <= 1 ? 1 : 1 << (32 - __builtin_clz(r.n - 1));
    const int each = kWave / groups;
#define GTP_STEP(J)                                          \
  {                                                          \
    const uint32_t x = lane_xor<J>(m);                       \
    m = J < each ? (x > m ? x : m) : (x < m ? x : m);        \
  }
    GTP_STEP(1) GTP_STEP(2) GTP_STEP(4) GTP_STEP(8) GTP_STEP(16) GTP_STEP(32)
#undef GTP_STEP
    const uint64_t at_least = m > 0 ? (uint64_t)m << 32 : 1ull;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kHold; ++j)
      if (j * kMergeBlock < total) mine += __popcll(__ballot(o[j] >= at_least));
    int to = 0;
    if (mine > 0) {
      if (lane == 0) to = atomicAdd(&entries, mine);
      to = __builtin_amdgcn_readfirstlane(to);
    }
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      if (mine == 0 || j * kMergeBlock >= total) continue;
      const uint64_t k = __ballot(o[j] >= at_least);
      const int e = to + lanes_below(k);
      if (o[j] >= at_least && e < kList) {
        list_o[e] = o[j];
        list_at[e] = place(j);
      }
      to += __popcll(k);
    }
    __syncthreads();
    auto better = [](uint64_t o, uint64_t at, uint64_t than_o, uint64_t than_at) {
      return o > than_o || (o == than_o && at < than_at);
    };
    auto take = [&](int rank, uint64_t o, uint64_t at) {
      c.score[rank] = (float)unord64(o);
      c.beam[rank] = (int32_t)(at >> 32);
      c.token[rank] = (int64_t)(uint32_t)at;
    };
    const int n = entries;
    if (n <= kList) {
      // 16 lanes for an entry
      const int part = tid & 15;
      for (int e0 = 0; e0 < n; e0 += kMergeBlock / 16) {
        const int e = e0 + tid / 16;
        const bool in = e < n;
        const uint64_t mo = in ? list_o[e] : 0, ma = in ? list_at[e] : 0;
        int rank = 0;
        for (int i = part; i < n; i += 16) rank += better(list_o[i], list_at[i], mo, ma) ? 1 : 0;
        rank += (int)lane_xor<1>((uint32_t)rank);
        rank += (int)lane_xor<2>((uint32_t)rank);
        rank += (int)lane_xor<4>((uint32_t)rank);
        rank += (int)lane_xor<8>((uint32_t)rank);
        if (in && part == 0 && rank < r.n) take(rank, mo, ma);
      }
    } else {
      // (many equal scores) one after the other: the best behind the last
      uint64_t last_o = ~0ull, last_at = 0;
      for (int rank = 0; rank < r.n; ++rank) {
        uint64_t mo = 0, ma = ~0ull;
#pragma unroll
        for (int j = 0; j < kHold; ++j) {
          if (o[j] == 0) continue;
          const uint64_t at = place(j);
          if (better(last_o, last_at, o[j], at) && better(o[j], at, mo, ma)) {
            mo = o[j];
            ma = at;
          }
        }
        for (int x = kWave / 2; x > 0; x >>= 1) {
          const uint64_t oo = shfl_xor_u64(mo, x), oa = shfl_xor_u64(ma, x);
          if (better(oo, oa, mo, ma)) {
            mo = oo;
            ma = oa;
          }
        }
        __syncthreads();
        if (lane == 0) {
          list_o[wid] = mo;
          list_at[wid] = ma;
        }
        __syncthreads();
        for (int w = 0; w < kMergeWaves; ++w)
          if (better(list_o[w], list_at[w], mo, ma)) {
            mo = list_o[w];
            ma = list_at[w];
          }
        if (mo == 0) break;
        last_o = mo;
        last_at = ma;
        if (tid == 0) take(rank, mo, ma);
      }
    }
    __syncthreads();
  }
  if (out.status && tid < r.K) {
    // (a live row without a candidate; done groups have none)
    const bool live_row = !done && __builtin_fabsf(r.score[base + tid]) < kPosInf;
    out.status[base + tid] = live_row && row_status[tid] == GTP_ROW_OK && !row_any[tid]
                                 ? GTP_ROW_EMPTY
                                 : row_status[tid];
  }
  if (out.score && tid < r.n) {
    out.score[(int64_t)g * r.n + tid] = c.score[tid];
    out.beam[(int64_t)g * r.n + tid] = c.beam[tid];
    out.token[(int64_t)g * r.n + tid] = c.token[tid];
  }
  if constexpr (kStep) {
    if (wid == 0) advance(st, old, c, g, r.K, r.n, lane);
  }
}

__global__ __launch_bounds__(kWave) void beam_advance_kernel(State st, const float* score,
                                                             const int32_t* beam,
                                                             const int64_t* token, int K, int n) {
  __shared__ Candidates c;
  const int g = blockIdx.x, lane = threadIdx.x;
  const Before old = before(st, g, K, lane);
  if (lane < n) {
    const int64_t i = (int64_t)g * n + lane;
    const int b = beam[i];
    const bool ok = b >= 0 && b < K && score[i] > kNegInf;  // (not NaN)
    c.score[lane] = ok ? score[i] : kNegInf;
    c.beam[lane] = ok ? b : -1;
    c.token[lane] = token[i];
  }
  wave_lds_sync();
  advance(st, old, c, g, K, n, lane);
}

// The best hypotheses of each group behind its last step, and their tokens,
// read backwards from step to step: a lane per hypothesis.
__global__ __launch_bounds__(kWave) void beam_finish_kernel(
    const float* score, const float* pool_score, const int32_t* pool_row, const int32_t* pool_step,
    const uint8_t* done, const int64_t* tokens, const int32_t* parents, int64_t R, int K,
    int steps, double length, int64_t eos, int64_t pad, int give, float* out_score,
    int32_t* out_length, int64_t* out_tokens, int64_t room) {
  __shared__ float s[2 * kMaxK];
  __shared__ int32_t row[2 * kMaxK], step[2 * kMaxK];
  const int g = blockIdx.x, lane = threadIdx.x;
  const int64_t base = (int64_t)g * K;
  if (lane < K) {
    s[lane] = pool_score[base + lane];
    row[lane] = pool_row[base + lane];
    step[lane] = pool_step[base + lane];
    // beams that still go on count at their present length
    const bool open = !done[g] && steps > 0 && score[base + lane] > kNegInf;
    s[K + lane] = open ? (float)((double)score[base + lane] / length) : kNegInf;
    row[K + lane] = (int32_t)base + lane;
    step[K + lane] = steps;
  }
  wave_lds_sync();
  const bool in = lane < 2 * K;
  int rank = 2 * K;
  // (lanes' order for equal scores: the pool, then the beams' own)
  if (in) {
    rank = 0;
    for (int i = 0; i < 2 * K; ++i) rank += s[i] > s[lane] || (s[i] == s[lane] && i < lane) ? 1 : 0;
  }
  if (rank >= give) return;
  const int64_t o = (int64_t)g * give + rank;
  int at = s[lane] == kNegInf ? -1 : row[lane];
  const int t = s[lane] == kNegInf ? -1 : step[lane];
  // (references that are not of these steps and this group give no tokens)
  const bool ok = at >= base && at < base + K && t >= 0 && t <= steps;
  const int n = !ok ? 0 : t < steps ? t + 1 : steps;
  out_score[o] = s[lane];
  out_length[o] = n;
  int64_t* to = out_tokens + o * room;
  for (int i = n; i < steps; ++i) to[i] = pad;
  if (!ok) return;
  if (t < steps) to[t] = eos;
  for (int i = (t < steps ? t : steps) - 1; i >= 0; --i) {
    if (at < base || at >= base + K) {
      to[i] = pad;
      continue;
    }
    to[i] = tokens[(int64_t)i * R + at];
    at = parents[(int64_t)i * R + at];
  }
}

// ------------------------------------------------------------------ launches

// Keys that a slice gives, and slices per row: waves enough for the chip (2048:
// 2 per SIMD) of at least a chunk each, and what the merge can hold.  [4, 151936]
// by chunks of 2048 8.2 us, by two of them 11.4; [256, 248320] with 4096 waves
// 32.3 us for 31.1.
int64_t slots_of(int64_t n) { return n <= 4 ? n + 2 : n <= 16 ? n + n / 2 : n + n / 4; }
void slices_of(int64_t G, int64_t K, int64_t n, int64_t V, int64_t& S, int64_t& L) {
  int64_t want = (2048 + G * K - 1) / (G * K);
  const int64_t most = kMaxKeys / (K * slots_of(n)), full = (V + 2047) / 2048;
  if (want > most) want = most;
  if (want > full) want = full;
  if (want > kWave) want = kWave;
  if (want < 1) want = 1;
  L = ((V + want - 1) / want + 511) / 512 * 512;
  S = (V + L - 1) / L;
}

int check_rows(const gtp_beam_rows* q) {
  if (!q || q->groups < 0 || q->beams < 1 || q->candidates < 1 || q->vocab < 1)
    return GTP_ERR_INVALID_ARGUMENT;
  if (q->dtype != GTP_DTYPE_F32 && q->dtype != GTP_DTYPE_BF16 && q->dtype != GTP_DTYPE_F16)
    return GTP_ERR_INVALID_ARGUMENT;
  if (q->beams > kMaxK || q->candidates > kMaxN || q->vocab > 0x7FFFFFFFll - 4096 ||
      q->groups > (1 << 24) / q->beams)
    return GTP_ERR_UNSUPPORTED;
  return GTP_OK;
}

int check_data(const gtp_beam_rows* q) {
  const int rc = check_rows(q);
  if (rc != GTP_OK || q->groups == 0) return rc;
  if (!q->logits || !q->scores || q->group_stride < 0 || q->beam_stride < 0 ||
      (q->allow_mask && q->mask_stride < (q->vocab + 31) / 32 && q->groups * q->beams > 1))
    return GTP_ERR_INVALID_ARGUMENT;
  const uintptr_t size = q->dtype == GTP_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(q->logits) % size) return GTP_ERR_INVALID_ARGUMENT;
  return GTP_OK;
}

int check_state(const gtp_beam_state* s) {
  if (!s || !s->scores || !s->pool_scores || !s->pool_rows || !s->pool_steps || !s->done ||
      !s->out_tokens || !s->out_parents || !s->out_scores || !s->out_pool_scores ||
      !s->out_pool_rows || !s->out_pool_steps || !s->out_done || s->step < 0 ||
      !(s->length > 0.0) || s->length - s->length != 0.0)
    return GTP_ERR_INVALID_ARGUMENT;
  return GTP_OK;
}

State state_of(const gtp_beam_state* s) {
  return State{s->scores, s->pool_scores, s->pool_rows, s->pool_steps, s->done, s->out_tokens,
               s->out_parents, s->out_scores, s->out_pool_scores, s->out_pool_rows,
               s->out_pool_steps, s->out_done, s->eos_token_id, s->pad_token_id, s->length,
               s->step, s->early_stopping ? 1 : 0};
}

template <typename T>
void launch_slices(const Rows& r, hipStream_t s) {
  const dim3 grid((uint32_t)(((int64_t)r.G * r.K * r.S + kWaves - 1) / kWaves));
  if (r.mask)
    launch_timed(beam_slices_kernel<T, true>, grid, dim3(kBlock), s, r);
  else
    launch_timed(beam_slices_kernel<T, false>, grid, dim3(kBlock), s, r);
}

int run(const gtp_beam_rows* q, const Out& out, const gtp_beam_state* step, void* workspace,
        size_t workspace_bytes, void* stream) {
  const int rc = check_data(q);
  if (rc != GTP_OK || q->groups == 0) return rc;
  if (step) {
    const int rs = check_state(step);
    if (rs != GTP_OK) return rs;
  }
  if (!workspace || workspace_bytes < gtp_beam_workspace_bytes(q) ||
      (reinterpret_cast<uintptr_t>(workspace) & 7u))
    return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Rows r;
  r.x = q->logits;
  r.mask = reinterpret_cast<const uint8_t*>(q->allow_mask);
  r.score = q->scores;
  r.done = q->done;
  r.V = q->vocab;
  r.group_stride = q->group_stride;
  r.beam_stride = q->beam_stride;
  r.mask_stride = q->mask_stride * 4;
  r.G = (int32_t)q->groups;
  r.K = q->beams;
  r.n = q->candidates;
  int64_t S, L;
  slices_of(r.G, r.K, r.n, r.V, S, L);
  r.S = (int32_t)S;
  r.slots = (int32_t)slots_of(r.n);
  r.L = L;
  const uint32_t per_row = (uint32_t)(r.S * r.slots);  // (below 2^13: exact)
  r.row_magic = per_row > 1 ? (uint32_t)(((1ull << 32) + per_row - 1) / per_row) : 0;
  const int64_t slices = (int64_t)r.G * r.K * S;
  r.keys = reinterpret_cast<uint64_t*>(workspace);
  r.sums = reinterpret_cast<float2*>(r.keys + slices * r.slots);
  if (q->dtype == GTP_DTYPE_BF16) launch_slices<uint16_t>(r, s);
  else if (q->dtype == GTP_DTYPE_F16) launch_slices<_Float16>(r, s);
  else launch_slices<float>(r, s);
  const State st = step ? state_of(step) : State{};
  const dim3 grid = flat_grid<kMergeBlock>(r.G);
  if (step)
    hipLaunchKernelGGL(beam_merge_kernel<true>, grid, dim3(kMergeBlock), 0, s, r, out, st);
  else
    hipLaunchKernelGGL(beam_merge_kernel<false>, grid, dim3(kMergeBlock), 0, s, r, out, st);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

}  // namespace beam
}  // namespace gtp

using namespace gtp;

extern "C" size_t gtp_beam_workspace_bytes(const gtp_beam_rows* rows) {
  if (beam::check_rows(rows) != GTP_OK) return 0;
  if (rows->groups == 0) return 8;
  int64_t S, L;
  beam::slices_of(rows->groups, rows->beams, rows->candidates, rows->vocab, S, L);
  const int64_t slots = beam::slots_of(rows->candidates);
  return (size_t)(rows->groups * rows->beams * S) * (size_t)(slots + 1) * 8;
}

extern "C" int gtp_beam_candidates(const gtp_beam_rows* rows, float* out_scores,
                                   int32_t* out_beams, int64_t* out_tokens, int32_t* out_status,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (rows && rows->groups > 0 && (!out_scores || !out_beams || !out_tokens))
    return GTP_ERR_INVALID_ARGUMENT;
  const beam::Out out{out_scores, out_beams, out_tokens, out_status};
  return beam::run(rows, out, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int gtp_beam_step(const gtp_beam_rows* rows, const gtp_beam_state* state,
                             int32_t* out_status, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if (!state) return GTP_ERR_INVALID_ARGUMENT;
  if (rows && (rows->scores != state->scores || rows->done != state->done))
    return GTP_ERR_INVALID_ARGUMENT;
  const beam::Out out{nullptr, nullptr, nullptr, out_status};
  return beam::run(rows, out, state, workspace, workspace_bytes, stream);
}

extern "C" int gtp_beam_advance(const float* scores, const int32_t* beams, const int64_t* tokens,
                                int64_t groups, int32_t num_beams, int32_t candidates,
                                const gtp_beam_state* state, void* stream) {
  if (groups < 0 || num_beams < 1 || candidates < 1) return GTP_ERR_INVALID_ARGUMENT;
  if (num_beams > beam::kMaxK || candidates > beam::kMaxN || groups > (1 << 24) / num_beams)
    return GTP_ERR_UNSUPPORTED;
  if (groups == 0) return GTP_OK;
  const int rc = beam::check_state(state);
  if (rc != GTP_OK) return rc;
  if (!scores || !beams || !tokens) return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(beam::beam_advance_kernel, dim3((uint32_t)groups), dim3(kWave), 0, s,
                     beam::state_of(state), scores, beams, tokens, num_beams, candidates);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

extern "C" int gtp_beam_finish(const float* scores, const float* pool_scores,
                               const int32_t* pool_rows, const int32_t* pool_steps,
                               const uint8_t* done, const int64_t* tokens, const int32_t* parents,
                               int64_t groups, int32_t num_beams, int32_t steps, double length,
                               int64_t eos_token_id, int64_t pad_token_id, int32_t give,
                               float* out_scores, int32_t* out_lengths, int64_t* out_tokens,
                               int64_t out_stride, void* stream) {
  if (groups < 0 || num_beams < 1 || steps < 0 || give < 1 || give > num_beams ||
      out_stride < steps || !(length > 0.0))
    return GTP_ERR_INVALID_ARGUMENT;
  if (num_beams > beam::kMaxK || groups > (1 << 24) / num_beams) return GTP_ERR_UNSUPPORTED;
  if (groups == 0) return GTP_OK;
  if (!scores || !pool_scores || !pool_rows || !pool_steps || !done || !out_scores ||
      !out_lengths || (steps > 0 && (!tokens || !parents || !out_tokens)))
    return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(beam::beam_finish_kernel, dim3((uint32_t)groups), dim3(kWave), 0, s, scores,
                     pool_scores, pool_rows, pool_steps, done, tokens, parents,
                     groups * num_beams, num_beams, steps, length, eos_token_id, pad_token_id, give,
                     out_scores, out_lengths, out_tokens, out_stride);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}
