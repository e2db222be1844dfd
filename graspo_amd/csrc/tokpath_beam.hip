// tokpath_beam.hip -- one step of a beam search over vocabulary-wide logits (gfx950).
//
// For beam k of a group and token v the candidate's score is
//   c[k, v] = score[k] + x[k, v] - log sum_w exp x[k, w],
// and a group's n best (c descending, then beam, then token) go on: finished
// ones into the group's pool, the others into its K slots.
//
// - beam_slices_kernel: each wave streams a slice of one row once.  A chunk of
//   2048 16-bit (1024 fp32) logits is folded into a running sum of exponentials
//   (one reference for the wave, in base 2), and whatever lies above the slice's
//   running threshold is appended to a list in LDS by ballots; past 96 entries
//   the list is cut to its n best and the threshold rises to the last of them.
//   Within a row the order by logit is the order by score, so n per slice do.
// - beam_merge_kernel: a workgroup per group turns the slices' sums into each
//   row's log-sum-exp in 64 bits (scores of different beams are compared, and
//   a sum rounded to 32 bits would decide near-ties), takes the n best of
//   K S n candidates and, in its first wave, one lane per candidate, moves the
//   group on.
// The rows' bytes bound the large calls, two launches and the merge's chain of
// LDS steps the small ones.
#include "tokpath_stream.h"

namespace gtp {
namespace beam {

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;
constexpr int kU = 4;           // 16-byte vectors per lane and chunk
constexpr int kCap = 640;       // list entries per wave: kCut and the 512 of an append
constexpr int kCut = 96;        // entries from which on the list is cut
constexpr int kMaxN = 64;       // candidates: one lane each
constexpr int kMaxK = 32;
constexpr int kMaxKeys = 8192;  // K S n: at most 32 per thread of the merge
constexpr uint32_t kOrdNegInf = 0x007FFFFFu;  // ord32(-inf)

struct Rows {
  const void* x;
  const uint8_t* mask;   // bit v of a row: token v is allowed
  const float* score;    // [G, K]
  const uint8_t* done;   // [G] or null
  int64_t V, group_stride, beam_stride, mask_stride;  // mask_stride in bytes
  int32_t G, K, n, S;
  int64_t L;             // a slice's logits, a multiple of 512
  uint64_t* keys;        // [G K S n]
  float2* sums;          // [G K S]: maximum, sum
};

// A slice's sum is s = sum 2^{(x - m) c + r(m)} with c the fp32 log2(e), where
// the exponents come from one fma, x c - fl(m c), so that r(m) = m c - fl(m c).
// From |m| = 2^16 on r could overflow the exponential: (x - m) c there, r = 0.
__device__ __forceinline__ bool by_fma(float m) { return __builtin_fabsf(m) < 65536.0f; }
__device__ __forceinline__ float residual(float m) {
  return by_fma(m) ? __builtin_fmaf(m, kLog2e, -(m * kLog2e)) : 0.0f;
}

// A beam that goes on: a finite score in a group that is not done.
__device__ __forceinline__ bool live(const Rows& r, int row) {
  return !(r.done && r.done[row / r.K]) && __builtin_fabsf(r.score[row]) < kPosInf;
}

// The n best of a wave's list, in no order, and the threshold that they set.
// count, tau and the list are the same for all lanes.
struct Top {
  uint64_t* list;
  int count;
  float tau;

  // the largest T with at least n keys >= T; n keys exactly stop the search
  template <typename Count>
  __device__ __forceinline__ static uint64_t cut_at(int n, Count count_from) {
    uint64_t T = 0;
    for (int b = 63; b >= 0; --b) {
      const uint64_t t = T | (1ull << b);
      const int c = count_from(t);
      if (c >= n) T = t;
      if (c == n) break;
    }
    return T;
  }

  __device__ __forceinline__ void cut(int n, int lane) {
    if (count <= n) return;
    wave_lds_sync();
    uint64_t T;
    if (count <= 2 * kWave) {
      const uint64_t a = lane < count ? list[lane] : 0;
      const uint64_t b = lane + kWave < count ? list[lane + kWave] : 0;
      T = cut_at(n, [&](uint64_t t) {
        return __popcll(__ballot(a >= t)) + __popcll(__ballot(b >= t));
      });
      wave_lds_sync();
      const uint64_t ka = __ballot(a >= T), kb = __ballot(b >= T);
      const uint64_t below = (1ull << lane) - 1;
      if (a >= T) list[__popcll(ka & below)] = a;
      if (b >= T) list[__popcll(ka) + __popcll(kb & below)] = b;
      count = __popcll(ka) + __popcll(kb);
    } else {
      // rows of many equal logits
      const int m = count;
      T = cut_at(n, [&](uint64_t t) {
        int c = 0;
        for (int i = 0; i < m; i += kWave)
          c += __popcll(__ballot(i + lane < m && list[i + lane] >= t));
        return c;
      });
      int kept = 0;
      for (int i = 0; i < m; i += kWave) {
        const uint64_t a = i + lane < m ? list[i + lane] : 0;
        const uint64_t ka = __ballot(a >= T);
        wave_lds_sync();
        if (a >= T) list[kept + __popcll(ka & ((1ull << lane) - 1))] = a;
        wave_lds_sync();
        kept += __popcll(ka);
      }
      count = kept;
    }
    // what comes later has a larger token id: only more than the last counts
    const uint32_t hi = (uint32_t)(T >> 32);
    tau = hi <= kOrdNegInf ? kNegInf : unord32(hi);
  }

  // Appends y[j] (token id0 + j) where it lies above the threshold.
  template <int E>
  __device__ __forceinline__ void append(const float (&y)[E], int32_t id0, int n, int lane) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const bool in = y[j] > tau;
      const uint64_t at = __ballot(in);
      if (at == 0) continue;
      if (in) list[count + __popcll(at & ((1ull << lane) - 1))] = rank_key(y[j] + 0.0f, id0 + j);
      count += __popcll(at);
    }
    if (count > kCut) cut(n, lane);
  }
};

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Unaligned {
  u32x4 v;
};

// The slice's vector at element e (E elements); what lies past `end` is -inf.
template <typename T>
__device__ __forceinline__ u32x4 load_vec(const T* row, int64_t e, int64_t end) {
  constexpr int E = Vec<T>::kE;
  if (e + E <= end) return reinterpret_cast<const Unaligned<T>*>(row + e)->v;
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u
                             : __is_same(T, _Float16) ? 0xFC00u : 0xFF80u;
  u32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (sizeof(T) == 4) {
      v[w] = e + w < end ? __builtin_bit_cast(uint32_t, row[e + w]) : kNone;
    } else {
      const uint32_t lo = e + 2 * w < end ? __builtin_bit_cast(uint16_t, row[e + 2 * w]) : kNone;
      const uint32_t hi = e + 2 * w + 1 < end ? __builtin_bit_cast(uint16_t, row[e + 2 * w + 1]) : kNone;
      v[w] = lo | hi << 16;
    }
  }
  return v;
}

template <typename T, bool kMask>
__global__ __launch_bounds__(kBlock) void beam_slices_kernel(Rows r) {
  constexpr int E = Vec<T>::kE;
  constexpr int64_t kChunk = (int64_t)kU * kWave * E;
  __shared__ uint64_t lists[kWaves][kCap];
  const int lane = threadIdx.x & (kWave - 1);
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t at = (int64_t)blockIdx.x * kWaves + wid;
  if (at >= (int64_t)r.G * r.K * r.S) return;
  const int row = (int)(at / r.S), slice = (int)(at % r.S);
  if (!live(r, row)) return;
  const T* x = reinterpret_cast<const T*>(r.x) + (row / r.K) * r.group_stride +
               (row % r.K) * r.beam_stride;
  const uint8_t* mask = kMask ? r.mask + row * r.mask_stride : nullptr;
  const int64_t begin = slice * r.L;
  const int64_t end = begin + r.L < r.V ? begin + r.L : r.V;

  Top top{lists[wid], 0, kNegInf};
  float top_x = kNegInf, s = 0.0f;  // the wave's maximum, the lane's sum

  u32x4 next[kU];
  uint32_t bits_next[kU];
  auto load = [&](int64_t e) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t i = e + ((int64_t)u * kWave + lane) * E;
      if (i < end) {
        next[u] = load_vec(x, i, end);
        if constexpr (kMask) bits_next[u] = (uint32_t)mask[i >> 3] >> (i & 7);
      }
    }
  };
  load(begin);
  bool first = true;
  for (int64_t e = begin; e < end; e += kChunk) {
    float y[kU][E];
    uint32_t bits[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t i = e + ((int64_t)u * kWave + lane) * E;
      if (i < end) {
        Vec<T>::cvt(next[u], y[u]);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) y[u][j] = kNegInf;
      }
      if constexpr (kMask) bits[u] = bits_next[u];
    }
    load(e + kChunk);
    const float m = block_max_raw<kU, E>(y);
    if (__ballot(m > top_x)) {
      const float up = wave_max(fmaxf(m, top_x));
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

    auto masked = [&](int u, float (&z)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        z[j] = !kMask || ((bits[u] >> j) & 1u) ? y[u][j] : kNegInf;
    };
    float best = m;
    if (first) {
      // n lanes hold a logit at least as large as the n-th largest of the
      // lanes' maxima: a threshold before anything is in the list
      if constexpr (kMask) {
        best = kNegInf;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          float z[E];
          masked(u, z);
          best = max3raw(best, vec_max<E>(z), best);
        }
      }
      const uint32_t o = best == best ? ord32(best + 0.0f) : kOrdNegInf;
      uint32_t t0 = 0;
      for (int b = 31; b >= 0; --b) {
        const uint32_t t = t0 | (1u << b);
        const int c = __popcll(__ballot(o >= t));
        if (c >= r.n) t0 = t;
        if (c == r.n) break;
      }
      // (the float below it; there is none between the two zeros)
      t0 = t0 == 0x80000000u ? 0x7FFFFFFEu : t0 > 0u ? t0 - 1u : 0u;
      top.tau = t0 <= kOrdNegInf ? kNegInf : unord32(t0);
      first = false;
    }
    if (__ballot(best > top.tau)) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float z[E];
        masked(u, z);
        if (__ballot(vec_max<E>(z) > top.tau))
          top.append<E>(z, (int32_t)(e + ((int64_t)u * kWave + lane) * E), r.n, lane);
      }
    }
  }
  top.cut(r.n, lane);
  wave_lds_sync();
  if (lane < r.n) r.keys[at * r.n + lane] = lane < top.count ? top.list[lane] : 0ull;
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
  if (lane == 0) r.sums[at] = make_float2(top_x, s);
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

struct Scratch {
  float score[2 * kMaxK];
  int32_t row[2 * kMaxK], step[2 * kMaxK];
  int32_t beam[kMaxK];
};

// Moves group g on, by one wave; c: its n candidates, best first.
__device__ __forceinline__ void advance(const State& st, const Candidates& c, Scratch& w, int g,
                                        int K, int n, int lane) {
  const int64_t base = (int64_t)g * K;
  const uint64_t below = (1ull << lane) - 1;
  if (st.done[g]) {
    if (lane < K) {
      st.token[base + lane] = st.pad;
      st.parent[base + lane] = (int32_t)base + lane;
      st.new_score[base + lane] = st.score[base + lane];
      st.new_pool_score[base + lane] = st.pool_score[base + lane];
      st.new_pool_row[base + lane] = st.pool_row[base + lane];
      st.new_pool_step[base + lane] = st.pool_step[base + lane];
    }
    if (lane == 0) st.new_done[g] = 1;
    return;
  }
  const bool mine = lane < n;
  const bool valid = mine && c.beam[lane] >= 0;
  const bool ended = valid && c.token[lane] == st.eos;
  // the pool: what it held, then the finished ones among the first K; of equal
  // scores the earlier stays ahead
  if (lane < K) {
    w.score[lane] = st.pool_score[base + lane];
    w.row[lane] = st.pool_row[base + lane];
    w.step[lane] = st.pool_step[base + lane];
    w.score[K + lane] = ended ? (float)((double)c.score[lane] / st.length) : kNegInf;
    w.row[K + lane] = ended ? (int32_t)base + c.beam[lane] : -1;
    w.step[K + lane] = ended ? st.step : -1;
  }
  wave_lds_sync();
  float last = kNegInf;  // the pool's K-th score
  {
    const bool in = lane < 2 * K;
    const float v = in ? w.score[lane] : 0.0f;
    int rank = 0;
    for (int i = 0; i < 2 * K; ++i) {
      const float o = w.score[i];
      rank += o > v || (o == v && i < lane) ? 1 : 0;
    }
    if (in && rank < K) {
      st.new_pool_score[base + rank] = v;
      st.new_pool_row[base + rank] = v == kNegInf ? -1 : w.row[lane];
      st.new_pool_step[base + rank] = v == kNegInf ? -1 : w.step[lane];
    }
    const uint64_t at = __ballot(in && rank == K - 1);
    if (at) last = __shfl(v, __ffsll((unsigned long long)at) - 1, kWave);
  }
  // the first K others go on
  const uint64_t others = __ballot(mine && !ended);
  const int j = __popcll(others & below);
  const bool goes = mine && !ended && j < K;
  const uint64_t going = __ballot(goes && valid);
  if (lane < K) w.beam[lane] = -1;
  wave_lds_sync();
  if (goes && valid) w.beam[j] = c.beam[lane];
  wave_lds_sync();
  // a beam's best one stays in its slot, the rest take the free slots in order
  uint32_t taken = 0;
  bool again = false;
  for (int i = 0; i < K; ++i) {
    const int p = w.beam[i];
    if (p < 0) continue;
    taken |= 1u << p;
    again |= goes && valid && i < j && p == c.beam[lane];
  }
  const bool moves = goes && (!valid || again);
  const uint64_t moving = __ballot(moves);
  if (goes) {
    int slot;
    if (!moves) {
      slot = c.beam[lane];
    } else {
      uint32_t free = ~taken;
      for (int i = __popcll(moving & below); i > 0; --i) free &= free - 1;
      slot = __ffs((int)free) - 1;
    }
    st.token[base + slot] = valid ? c.token[lane] : st.pad;
    st.parent[base + slot] = (int32_t)base + (valid ? c.beam[lane] : slot);
    st.new_score[base + slot] = valid ? c.score[lane] : kNegInf;
  }
  // Every slot has one of the first n - (ended) >= K candidates when n >= 2 K;
  // a shorter list leaves slots without: dead ones.
  const int given = __popcll(__ballot(goes));
  if (given < K) {
    uint32_t free = ~taken;
    for (int i = __popcll(moving); i > 0; --i) free &= free - 1;
    if (lane < K && (free >> lane) & 1u) {
      st.token[base + lane] = st.pad;
      st.parent[base + lane] = (int32_t)base + lane;
      st.new_score[base + lane] = kNegInf;
    }
  }
  // the best that a live beam's score reaches at this length
  const int best_at = going ? __ffsll((unsigned long long)going) - 1 : 0;
  const float best = going ? (float)((double)c.score[best_at] / st.length) : kNegInf;
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

template <bool kStep>
__global__ __launch_bounds__(kBlock) void beam_merge_kernel(Rows r, Out out, State st) {
  extern __shared__ uint64_t dyn[];  // 2 x entries
  __shared__ double offset[kMaxK];  // score - log sum 2^{(x - m) c}
  __shared__ float row_top[kMaxK];  // m
  __shared__ uint64_t best[kBlock], best_at[kBlock];
  __shared__ Candidates c;
  __shared__ Scratch scratch;
  __shared__ int entries;
  __shared__ uint64_t cut, cut_at;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
  const int per_row = r.S * r.n, total = r.K * per_row;
  const int64_t base = (int64_t)g * r.K;
  const bool done = r.done && r.done[g];
  if (tid == 0) {
    entries = 0;
  }
  if (tid < r.n) {
    c.score[tid] = kNegInf;
    c.beam[tid] = -1;
    c.token[tid] = -1;
  }
  // each row's log-sum-exp
  for (int k = wid; k < r.K; k += kWaves) {
    int status = GTP_ROW_OK;
    double off = -__builtin_huge_val();
    const float score = r.score[base + k];
    float top = kNegInf;
    if (live(r, (int)base + k)) {
      const float2* p = r.sums + (base + k) * r.S;
      for (int i = lane; i < r.S; i += kWave) top = fmaxf(top, p[i].x);
      top = wave_max(top);
      double s = 0.0;
      for (int i = lane; i < r.S; i += kWave) {
        const float2 v = p[i];
        // (a NaN stays, also where nothing finite was seen)
        if (v.y != v.y) s += (double)v.y;
        else if (v.x > kNegInf)
          s += (double)v.y *
               exp2(((double)v.x - (double)top) * (double)kLog2e - (double)residual(v.x));
      }
#pragma unroll
      for (int o = kWave / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
      // (the exponents are multiples of the fp32 log2(e))
      bool any = false;  // (a slice's first key is there where any is)
      for (int i = lane; i < r.S; i += kWave) any |= r.keys[((base + k) * r.S + i) * r.n] != 0;
      const bool some = __ballot(any) != 0;
      if (s != s) status = GTP_ROW_NONFINITE;
      else if (!some) status = GTP_ROW_EMPTY;
      else off = (double)score - log2(s) / (double)kLog2e;
    } else if (!done && !(score == kNegInf)) {
      status = GTP_ROW_NONFINITE;
    }
    if (lane == 0) {
      offset[k] = off;
      row_top[k] = top;
      if (out.status) out.status[base + k] = status;
    }
  }
  __syncthreads();
  // Candidate i: its score in an order of integers (0: none) and its place.
  auto candidate = [&](int i, uint64_t& at) {
    const int k = i / per_row;
    at = ~0ull;
    if (offset[k] == -__builtin_huge_val()) return (uint64_t)0;
    const uint64_t key = r.keys[base * per_row + i];
    if (key == 0) return (uint64_t)0;
    at = (uint64_t)k << 32 | (uint32_t)rank_key_id(key);
    return ord64(((double)rank_key_y(key) - (double)row_top[k]) + offset[k]);
  };
  auto better = [](uint64_t o, uint64_t at, uint64_t than_o, uint64_t than_at) {
    return o > than_o || (o == than_o && at < than_at);
  };
  if (!done) {
    // n threads hold a candidate at least as good as the n-th best of the
    // threads' best ones; what is worse than that is out, so that no more than
    // these threads' candidates are left
    uint64_t mine = 0, mine_at = ~0ull;
    for (int i = tid; i < total; i += kBlock) {
      uint64_t at;
      const uint64_t o = candidate(i, at);
      if (better(o, at, mine, mine_at)) {
        mine = o;
        mine_at = at;
      }
    }
    best[tid] = mine;
    best_at[tid] = mine_at;
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < kBlock; ++i) {
      const uint64_t o = best[i];
      // (threads without any are equal: their number decides)
      if (o >= mine)
        rank += better(o, best_at[i], mine, mine_at) || (mine == 0 && o == 0 && i < tid) ? 1 : 0;
    }
    if (rank == r.n - 1) {
      cut = mine;
      cut_at = mine_at;
    }
    __syncthreads();
    const uint64_t from = cut, from_at = cut_at;
    for (int i = tid; i < total; i += kBlock) {
      uint64_t at;
      const uint64_t o = candidate(i, at);
      if (o == 0 || better(from, from_at, o, at)) continue;
      const int e = atomicAdd(&entries, 1);
      dyn[2 * e] = o;
      dyn[2 * e + 1] = at;
    }
    __syncthreads();
    const int m = entries;
    for (int e = tid; e < m; e += kBlock) {
      const uint64_t o = dyn[2 * e], at = dyn[2 * e + 1];
      int rank = 0;
      for (int i = 0; i < m; ++i) {
        const uint64_t p = dyn[2 * i];
        rank += better(p, dyn[2 * i + 1], o, at) ? 1 : 0;
      }
      if (rank < r.n) {
        c.score[rank] = (float)unord64(o);
        c.beam[rank] = (int32_t)(at >> 32);
        c.token[rank] = (int64_t)(uint32_t)at;
      }
    }
  }
  __syncthreads();
  if (out.score && tid < r.n) {
    out.score[(int64_t)g * r.n + tid] = c.score[tid];
    out.beam[(int64_t)g * r.n + tid] = c.beam[tid];
    out.token[(int64_t)g * r.n + tid] = c.token[tid];
  }
  if (kStep && wid == 0) advance(st, c, scratch, g, r.K, r.n, lane);
}

__global__ __launch_bounds__(kWave) void beam_advance_kernel(State st, const float* score,
                                                             const int32_t* beam,
                                                             const int64_t* token, int K, int n) {
  __shared__ Candidates c;
  __shared__ Scratch scratch;
  const int g = blockIdx.x, lane = threadIdx.x;
  if (lane < n) {
    const int64_t i = (int64_t)g * n + lane;
    const int b = beam[i];
    const bool ok = b >= 0 && b < K && score[i] > kNegInf;  // (not NaN)
    c.score[lane] = ok ? score[i] : kNegInf;
    c.beam[lane] = ok ? b : -1;
    c.token[lane] = token[i];
  }
  wave_lds_sync();
  advance(st, c, scratch, g, K, n, lane);
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

// Slices per row: waves enough for the chip (2048: 2 per SIMD) of at least two
// chunks each, and what the merge can hold.
void slices_of(int64_t G, int64_t K, int64_t n, int64_t V, int64_t& S, int64_t& L) {
  int64_t want = (2048 + G * K - 1) / (G * K);
  const int64_t most = kMaxKeys / (K * n), full = (V + 4095) / 4096;
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
      q->groups * q->beams > (1 << 24))
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
  if (rc != GTP_OK) return rc;
  if (step) {
    const int rs = check_state(step);
    if (rs != GTP_OK) return rs;
  }
  if (q->groups == 0) return GTP_OK;
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
  r.L = L;
  const int64_t slices = (int64_t)r.G * r.K * S;
  r.keys = reinterpret_cast<uint64_t*>(workspace);
  r.sums = reinterpret_cast<float2*>(r.keys + slices * r.n);
  if (q->dtype == GTP_DTYPE_BF16) launch_slices<uint16_t>(r, s);
  else if (q->dtype == GTP_DTYPE_F16) launch_slices<_Float16>(r, s);
  else launch_slices<float>(r, s);
  const int64_t keys = (int64_t)r.K * S * r.n;
  const size_t lds = (size_t)((keys + kBlock - 1) / kBlock * r.n) * 16;
  const State st = step ? state_of(step) : State{};
  if (step)
    hipLaunchKernelGGL(beam_merge_kernel<true>, dim3(r.G), dim3(kBlock), lds, s, r, out, st);
  else
    hipLaunchKernelGGL(beam_merge_kernel<false>, dim3(r.G), dim3(kBlock), lds, s, r, out, st);
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
  return (size_t)(rows->groups * rows->beams * S) * (size_t)(rows->candidates + 1) * 8;
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
  if (num_beams > beam::kMaxK || candidates > beam::kMaxN || groups * num_beams > (1 << 24))
    return GTP_ERR_UNSUPPORTED;
  const int rc = beam::check_state(state);
  if (rc != GTP_OK) return rc;
  if (groups == 0) return GTP_OK;
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
  if (num_beams > beam::kMaxK || groups * num_beams > (1 << 24)) return GTP_ERR_UNSUPPORTED;
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
