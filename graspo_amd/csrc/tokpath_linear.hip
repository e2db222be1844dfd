// tokpath_linear.hip -- token logprobs from hidden states in pieces of the
// vocabulary, without keeping the logits, and their gradients (gfx950).
//
//   x_nv  = h_n . w_v            lse_n = log sum_v exp(x_nv)
//   lp_n  = x_{n,t_n} - lse_n    dx_nv = g_n ([v = t_n] - exp(x_nv - lse_n))
//   dh_n  = sum_v dx_nv w_v      dw_v  = sum_n dx_nv h_n
//
// over bf16 or fp16 hidden states [B, S, K] and weight [V, K].  Four products
// of 2 N K V operations (the logits, the logits again, dh, dw) on the matrix
// cores, every one accumulated in fp32 by the tile loop of tokpath_gemm.h.
//
// - Forward: the logits of a 256 x 256 tile fold into (m, s) per token in
//   registers; one partial state per (128 vocabulary rows, token), merged by
//   a small kernel.
// - Backward, piece by piece of the vocabulary: the piece's logits again,
//   their gradient D rounded once to 16 bits (each element within half a step
//   of its fp32 value; fp16 scaled by a power of two that puts the largest
//   |g| just below 2^15, so that small probabilities keep their bits; the
//   mean's g, one for all rows, left for the end) and
//   written vocabulary-major; then dh += D^T w and dw = D h from it, both
//   accumulated in fp32 and rounded once.  A piece's D takes at most
//   kPieceBytes whatever V is.
//
//   With at most 128 rows the weight's bytes bound the call, the products but
//   dh's run in the kernels of tokpath_few.h, and D is two 16-bit parts.
//
// Rows whose target is ignored, whose target lies outside [0, V) or (backward)
// whose g is 0 are left out of every product: a first kernel lists the others
// in order and a second gathers their hidden states, so the products run over
// the listed rows alone.  Their number stays on the device; grids are sized
// for all rows, and workgroups past the listed ones end at once.
//
// Nothing is summed with atomics: every sum has one order, fixed by the sizes
// and the listed rows.
//
// Replaces the chunked F.linear + logsumexp + logaddexp loop of
// _selected_token_log_probs_from_hidden
// (src/graspo/backends/graspoflow/tensor_utils.py:167-186) under autograd,
// which keeps every chunk's logits.
#include "tokpath_few.h"
#include "tokpath_gemm.h"

namespace gtp {

int64_t device_cus();  // compute units of the current device

namespace lin {

using namespace gemm;

// Bytes of D at a time.  A piece costs dh a pass over its fp32 sums and a
// drain of the chip: at 8192 x 4096 x 131072 dh takes 6.6 ms in one piece of 2
// GiB, 6.7 in two, 7.1 in four, 8.3 in eight; the other products do not care.
constexpr int64_t kPieceBytes = (int64_t)1 << 30;

struct Rows {
  const void* targets;
  int64_t V, S, T, tbstride, trstride, ignore;
  int B, t64, has_ignore;
  __device__ __forceinline__ int64_t target(int64_t b, int64_t s) const {
    const int64_t at = b * tbstride + s * trstride;
    return t64 ? reinterpret_cast<const int64_t*>(targets)[at]
               : (int64_t)reinterpret_cast<const int32_t*>(targets)[at];
  }
};

// What the listing kernel leaves for the others.
struct Meta {
  int32_t n;     // listed rows
  int32_t bad;   // rows whose target lies outside [0, V)
  float inv;     // what D lacks: 1 / a power of two, or the mean's gradient
  int32_t splits;  // shares of dh's products (backward)
};

// What dh's products split their K into.  A share writes sums of its own (one
// row of `width` floats per listed row, `most` rows in all), so that few tiles
// fill the chip: rounds of one tile per CU at 1.5 us a K step, against three
// passes over the sums at 4.5 TB/s.  Picked for the rows that are listed, on
// the device.
struct Shares {
  int32_t column_tiles, cus;
  int32_t low;  // D in two parts: the second one's first row in the sums
  int64_t steps, width, most;
  // rows of the sums
  __host__ __device__ int64_t rows(int64_t listed) const {
    return low > 0 && listed > 0 ? low + listed : listed;
  }
  __host__ __device__ float us(int64_t rows, int64_t k) const {
    const int64_t tiles = (rows + kTile - 1) / kTile * column_tiles;
    return (float)((tiles * k + cus - 1) / cus * ((steps + k - 1) / k)) * 1.5f +
           (float)(k * rows * width) * (12.0f / 4.5e6f);
  }
  __host__ __device__ bool possible(int64_t rows, int64_t k) const {
    return k == 1 || (k <= 32 && steps / k >= 8 && k * rows <= most);
  }
  int64_t best(int64_t rows) const {
    int64_t found = 1;
    for (int64_t k = 2; possible(rows, k); ++k)
      if (us(rows, k) < us(rows, found)) found = k;
    return found;
  }
  // The same by a whole wave.
  __device__ int best_of(int64_t rows) const {
    const int lane = threadIdx.x & 63;
    float least = lane < 32 && possible(rows, lane + 1) ? us(rows, lane + 1) : kPosInf;
    int found = lane + 1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float u = __shfl_xor(least, o, kWave);
      const int k = __shfl_xor(found, o, kWave);
      if (u < least || (u == least && k < found)) {
        least = u;
        found = k;
      }
    }
    return __shfl(found, 0, kWave);
  }
};

// One listed row.
struct Listed {
  int32_t* at;     // its index b * T + s
  int32_t* target;
  float* lse;      // backward only
  float* g;        // backward only: over Meta::inv
};

// ------------------------------------------------------------ listing

constexpr int kListBlock = 1024;

// One workgroup; a thread takes a run of rows, counts those to list, and
// lists them from where the threads before it end: the order stays.  out_lp
// (forward): 0 for ignored rows and NaN for bad ones.  slot (backward): the
// list index of each of the B x S positions, -1 for none.
__global__ __launch_bounds__(kListBlock) void list_rows_kernel(
    Rows a, Listed out, Meta* __restrict__ meta, float* __restrict__ out_lp,
    float* __restrict__ out_lse, uint32_t* __restrict__ verdict, const float* __restrict__ grad,
    const int64_t* __restrict__ mean_count, const float* __restrict__ lse_in,
    int32_t* __restrict__ slot, int scaled, Shares shares) {
  __shared__ uint32_t sums[kListBlock / kWave];
  __shared__ float tops[kListBlock / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t N = (int64_t)a.B * a.T, per = (N + kListBlock - 1) / kListBlock;
  const int64_t first = min(N, tid * per), last = min(N, first + per);
  const bool backward = grad != nullptr;
  const float gm = backward && mean_count ? -grad[0] / (float)mean_count[0] : 0.0f;
  auto g_of = [&](int64_t n) { return mean_count ? gm : grad[n]; };
  uint32_t count = 0;
  float top = 0.0f;
  int bad = 0;
  for (int64_t n = first; n < last; ++n) {
    const int64_t b = n / a.T, s = n - b * a.T, t = a.target(b, s);
    if (a.has_ignore && t == a.ignore) continue;
    if (t < 0 || t >= a.V) {
      bad = 1;
      continue;
    }
    if (backward) {
      const float g = g_of(n);
      if (g == 0.0f) continue;
      top = fmaxf(top, fabsf(g));
    }
    ++count;
  }
  uint32_t upto = wave_scan_u32(count);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  if (lane == 63) sums[wid] = upto;
  if (lane == 0) tops[wid] = top;
  const int any_bad = __syncthreads_or(bad);
  uint32_t before = upto - count, all = 0;
  top = 0.0f;
#pragma unroll
  for (int w = 0; w < kListBlock / kWave; ++w) {
    before += w < wid ? sums[w] : 0;
    all += sums[w];
    top = fmaxf(top, tops[w]);
  }
  // fp16: 2^(15 - e) for 2^(e-1) <= top < 2^e (bounded, so that neither it nor
  // its inverse leaves fp32's normal numbers).  The mean's gradient is one for
  // all rows and left out of D altogether: a target's element g (1 - p) is
  // nearly g in most rows, and one rounding shared by all of them would not
  // average out (4096 tokens of 151936: the error against 64 bits was 0.0027,
  // and is 0.0018 so, of which rounding the results takes 0.0017).
  float scale = 1.0f, inv = 1.0f;
  if (mean_count) {
    scale = scaled ? 16384.0f : 1.0f;
    // (without a row gm is -g / 0, and both gradients are zeros times this)
    inv = all ? gm / scale : 0.0f;
  } else if (scaled && top > 0.0f && top < kPosInf) {
    int e;
    frexpf(top, &e);
    scale = ldexpf(1.0f, min(max(15 - e, -100), 100));
    inv = 1.0f / scale;
  }
  const int splits = backward && wid == 0 ? shares.best_of(shares.rows(all)) : 0;
  if (tid == 0) {
    *meta = Meta{(int32_t)all, any_bad, inv, splits};
    if (verdict)
      __hip_atomic_store(verdict, GTP_VERDICT_GOOD | (any_bad ? GTP_VERDICT_BAD : 0u),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  }
  uint32_t k = before;
  for (int64_t n = first; n < last; ++n) {
    const int64_t b = n / a.T, s = n - b * a.T, t = a.target(b, s);
    const bool skip = a.has_ignore && t == a.ignore, out_of = t < 0 || t >= a.V;
    float g = 0.0f;
    if (backward && !skip && !out_of) g = g_of(n);
    const bool take = !skip && !out_of && !(backward && g == 0.0f);
    if (take) {
      out.at[k] = (int32_t)n;
      out.target[k] = (int32_t)t;
      if (backward) {
        out.lse[k] = lse_in[n];
        out.g[k] = mean_count ? scale : g * scale;
      }
    } else if (out_lp) {
      const float v = skip ? 0.0f : __builtin_nanf("");
      out_lp[n] = v;
      out_lse[n] = v;
    }
    if (slot) slot[b * a.S + s] = take ? (int32_t)k : -1;
    k += take;
  }
  if (slot) {  // positions without a target
    const int64_t rest = a.S - a.T;
    for (int64_t i = tid; i < a.B * rest; i += kListBlock) {
      const int64_t b = i / rest;
      slot[b * a.S + a.T + (i - b * rest)] = -1;
    }
  }
}

// The listed rows' hidden states, one after the other, padded with zeros to
// ld elements (a multiple of 64): one workgroup per row, 16 bytes per thread
// where the rows allow it.
__global__ __launch_bounds__(256) void gather_rows_kernel(const uint16_t* __restrict__ hidden,
                                                          int64_t hb, int64_t hs, int64_t T,
                                                          int64_t K, const Meta* __restrict__ meta,
                                                          const int32_t* __restrict__ at, int vec,
                                                          uint16_t* __restrict__ out, int64_t ld) {
  const int64_t k = blockIdx.x;
  if (k >= meta->n) return;
  const int64_t n = at[k], b = n / T, s = n - b * T;
  const uint16_t* src = hidden + b * hb + s * hs;
  uint16_t* dst = out + k * ld;
  for (int64_t c = threadIdx.x; c < ld / 8; c += 256) {
    uint4 v{0, 0, 0, 0};
    if (vec) {
      if (c * 8 < K) v = reinterpret_cast<const uint4*>(src)[c];
    } else {
      uint32_t e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t lo = c * 8 + 2 * i;
        e[i] = lo < K ? src[lo] : 0u;
        if (lo + 1 < K) e[i] |= (uint32_t)src[lo + 1] << 16;
      }
      v = uint4{e[0], e[1], e[2], e[3]};
    }
    reinterpret_cast<uint4*>(dst)[c] = v;
  }
}

// ------------------------------------------------------------ forward

struct LseArgs {
  Operand w, h;  // [V, K], listed rows [., K]
  int64_t K;
  const Meta* meta;
  const int32_t* target;  // of the listed rows
  float2* partial;        // [2 * tiles of V][ldn]: (m, s)
  float* xt;              // the target's logit of the listed rows
  int64_t ldn;
  int tm, band;           // tiles of V; rows of the tile order's bands
};

// merge of two (m, s) states; an empty one is (-inf, 0)
__device__ __forceinline__ float2 merge_ms(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float fa = a.x == m ? 1.0f : __builtin_amdgcn_exp2f((a.x - m) * kLog2e);
  const float fb = b.x == m ? 1.0f : __builtin_amdgcn_exp2f((b.x - m) * kLog2e);
  return float2{m, a.y * fa + b.y * fb};
}

// The stages and the scratch of a tile loop.
#define GTP_LOOP_LDS                                                                      \
  __shared__ __attribute__((aligned(16))) uint4 sA0[kStage], sA1[kStage], sB0[kStage],    \
      sB1[kStage];                                                                        \
  __shared__ uint32_t s_unread[256]

// Vocabulary x tokens: lane l of a block holds token l & 15 and 4 vocabulary
// rows, so that a token's values fold in registers.
template <typename E>
__global__ __launch_bounds__(kThreads, 1) void lse_kernel(LseArgs a) {
  GTP_LOOP_LDS;
  __shared__ int s_t[2][kTile];  // (twice: a wave may be a tile ahead of another)
  const int n_listed = a.meta->n;
  Tiles at(blockIdx.x, a.tm, (n_listed + kTile - 1) / kTile, 1, a.band);
  if (!at.more()) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wv = wave >> 1, wt = wave & 1;
  Operand h = a.h;
  h.outer = n_listed;
  TileLoop<E, kAlongK, kAlongK> loop(
      Source<kAlongK>(a.w.ld, at.parts_m(), at.part_m(), wave, lane),
      Source<kAlongK>(h.ld, at.parts_n(), at.part_n(), wave, lane), sA0, sA1, sB0, sB1, s_unread,
      wave, lane);
  int vt, tt, share;
  at.place(vt, tt, share);
  loop.start(cursor_of<kAlongK>(a.w, (int64_t)vt * kTile, 0, a.K),
             cursor_of<kAlongK>(h, (int64_t)tt * kTile, 0, a.K));
  int odd = 0;
  for (bool more = true; more; odd ^= 1) {
    at.step();
    more = at.more();
    int vt2 = 0, tt2 = 0;
    Cursor ca{nullptr, 0, 0}, cb = ca;
    if (more) {
      at.place(vt2, tt2, share);
      ca = cursor_of<kAlongK>(a.w, (int64_t)vt2 * kTile, 0, a.K);
      cb = cursor_of<kAlongK>(h, (int64_t)tt2 * kTile, 0, a.K);
    }
    {
      // (the tile's barriers publish them)
      const int64_t k = (int64_t)tt * kTile + threadIdx.x;
      s_t[odd][threadIdx.x] = k < n_listed ? a.target[k] : -1;
    }
    loop.tile(a.K, ca, cb);

    // the lane's vocabulary rows are v0 + 16 x + i
    const int64_t v0 = (int64_t)vt * kTile + wv * 128 + 4 * (lane >> 4);
    const int64_t left = a.w.outer - v0;
    const int lim = (int)min((int64_t)128, max(left, (int64_t)0));  // valid offsets are below
    // (the epilogues are unrolled: a loop over the blocks moves accumulators,
    // and the compiler then also moves some in the products' loop, where it
    // does not see the asm's wait states)
#pragma unroll
    for (int y = 0; y < kB; ++y) {
        const int token = wt * 128 + y * 16 + (lane & 15);
        const int64_t k = (int64_t)tt * kTile + token;
        const int64_t off = (int64_t)s_t[odd][token] - v0;
        const int want = off >= 0 && off < lim ? (int)off : -1;
        float v[4 * kB], xt = 0.0f;
#pragma unroll
        for (int x = 0; x < kB; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float q = acc_read(loop.acc[x][y][i]);
            xt = want == x * 16 + i ? q : xt;
            v[4 * x + i] = x * 16 + i < lim ? q : kNegInf;
          }
        float m = v[0];
#pragma unroll
        for (int i = 1; i < 4 * kB; i += 2) m = max3raw(m, v[i], i + 1 < 4 * kB ? v[i + 1] : v[i]);
        // (the difference first: exact near the maximum, however large that is)
        const float mb = m == kNegInf ? 0.0f : m;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * kB; ++i) s += __builtin_amdgcn_exp2f((v[i] - mb) * kLog2e);
        // (a target's bits 2 and 3 say which of the lane's four groups has it)
        if (want >= 0 && (want & 12) == 0) a.xt[k] = xt;
        float2 st{m, s};
        st = merge_ms(st, float2{__shfl_xor(st.x, 16, kWave), __shfl_xor(st.y, 16, kWave)});
        st = merge_ms(st, float2{__shfl_xor(st.x, 32, kWave), __shfl_xor(st.y, 32, kWave)});
        if (lane < 16 && k < n_listed) a.partial[(int64_t)(vt * 2 + wv) * a.ldn + k] = st;
    }
    vt = vt2;
    tt = tt2;
  }
  wait_vm<0>();  // the loads past the last tile write their zeros
}

// The same partial states for at most 16 kNB rows: a workgroup's 128 vocabulary
// rows in one.
template <typename E, int kNB>
__global__ __launch_bounds__(few::kThreads, 2) void few_lse_kernel(LseArgs a) {
  constexpr int kTok = 16 * kNB;
  __shared__ __attribute__((aligned(16))) uint4 s_h[2][kTok * few::kChunks<kNB>];
  __shared__ float2 s_ms[few::kWaves][kTok];
  const int n = a.meta->n;
  if (n == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = (int64_t)blockIdx.x * few::kRows + wave * few::kWaveRows;
  few::Product<E, kNB, false> x;
  x.run(a.w, first, a.h, n, a.K, s_h);
  const int64_t v0 = first + 4 * (lane >> 4);
  const int lim = (int)min((int64_t)few::kWaveRows, max(a.w.outer - v0, (int64_t)0));
#pragma unroll
  for (int y = 0; y < kNB; ++y) {
    const int k = y * 16 + (lane & 15);
    const int64_t off = (k < n ? (int64_t)a.target[k] : -1) - v0;
    const int want = off >= 0 && off < lim ? (int)off : -1;
    float v[8], xt = 0.0f, m = kNegInf, s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int o = (i / 4) * 16 + (i & 3);
      const float q = x.acc[i / 4][y][i & 3];
      xt = want == o ? q : xt;
      v[i] = o < lim ? q : kNegInf;
      m = max3raw(m, v[i], v[i]);
    }
    const float mb = m == kNegInf ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += __builtin_amdgcn_exp2f((v[i] - mb) * kLog2e);
    if (want >= 0 && (want & 12) == 0) a.xt[k] = xt;
    float2 st{m, s};
    st = merge_ms(st, float2{__shfl_xor(st.x, 16, kWave), __shfl_xor(st.y, 16, kWave)});
    st = merge_ms(st, float2{__shfl_xor(st.x, 32, kWave), __shfl_xor(st.y, 32, kWave)});
    if (lane < 16) s_ms[wave][k] = st;
  }
  __syncthreads();
  const int k = threadIdx.x;
  if (k >= n) return;
  float2 st = s_ms[0][k];
#pragma unroll
  for (int w = 1; w < few::kWaves; ++w) st = merge_ms(st, s_ms[w][k]);
  a.partial[(int64_t)blockIdx.x * a.ldn + k] = st;
}

// The listed rows' logprob and lse from their partial states: kTok rows per
// workgroup, the other threads merging every so many states of them each.
constexpr int kMergeBlock = 1024;
template <int kTok>
__global__ __launch_bounds__(kMergeBlock) void lse_merge_kernel(
    const float2* __restrict__ partial, int64_t ldn, int n_parts, const Meta* __restrict__ meta,
    const int32_t* __restrict__ at, const float* __restrict__ xt, float* __restrict__ out_lp,
    float* __restrict__ out_lse) {
  constexpr int kGroups = kMergeBlock / kTok;
  __shared__ float2 red[kMergeBlock / kWave][kTok];
  const int lt = threadIdx.x % kTok, g = threadIdx.x / kTok;
  const int64_t k = (int64_t)blockIdx.x * kTok + lt;
  const int n = meta->n;
  if ((int64_t)blockIdx.x * kTok >= n) return;
  float2 st{kNegInf, 0.0f};
  if (k < n) {
#pragma unroll 4
    for (int p = g; p < n_parts; p += kGroups) st = merge_ms(st, partial[p * ldn + k]);
  }
#pragma unroll
  for (int o = kTok; o < kWave; o <<= 1)
    st = merge_ms(st, float2{__shfl_xor(st.x, o, kWave), __shfl_xor(st.y, o, kWave)});
  if ((threadIdx.x & 63) < kTok) red[threadIdx.x >> 6][lt] = st;
  __syncthreads();
  if (g != 0 || k >= n) return;
#pragma unroll
  for (int w = 1; w < kMergeBlock / kWave; ++w) st = merge_ms(st, red[w][lt]);
  const float ln_s = __builtin_amdgcn_logf(st.y) * kLn2;
  out_lp[at[k]] = (xt[k] - st.x) - ln_s;
  out_lse[at[k]] = st.x + ln_s;
}

// -sum(logprob) / count over the listed rows and the bad ones (whose NaN is
// the mean then), in 64 bits, one workgroup.
__global__ __launch_bounds__(1024) void mean_kernel(const Meta* __restrict__ meta,
                                                    const int32_t* __restrict__ at,
                                                    const float* __restrict__ lp,
                                                    float* __restrict__ loss,
                                                    int64_t* __restrict__ count) {
  __shared__ double sums[1024 / kWave];
  const int n = meta->n;
  double sum = 0.0;
  for (int k = threadIdx.x; k < n; k += 1024) sum += (double)lp[at[k]];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < 1024 / kWave; ++w) sum += sums[w];
  loss[0] = meta->bad ? __builtin_nanf("") : (float)(-sum / (double)n);
  count[0] = n;
}

// ------------------------------------------------------------ backward

// 16 rows x 128 columns of 16-bit values, held as lane & 15 = row and 4 columns
// in a row per x by `value(x, e)`, written to `out` (row stride ld) in whole
// 256-byte runs: through 4 KB of LDS of the wave's own, whose 16-byte chunks
// are XOR-swizzled by the row.  `rows` and `cols` bound what is written; vec:
// 16-byte stores (else 2-byte ones).  kLive: columns from `live` on get zeros,
// whatever value() made of them.
constexpr int kStoreLds = 256;  // chunks per wave
// the first n of 8 values, zeros behind
__device__ __forceinline__ uint4 first_of(uint4 v, int64_t n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = n >= 2 * i + 2 ? w[i] : n == 2 * i + 1 ? w[i] & 0xFFFFu : 0u;
  return uint4{w[0], w[1], w[2], w[3]};
}
template <bool kLive, typename Value>
__device__ __forceinline__ void store_block(uint4* mine, int lane, uint16_t* out, int64_t ld,
                                            int64_t rows, int64_t cols, int64_t live, bool vec,
                                            Value value) {
  const int row = lane & 15;
  uint2* half = reinterpret_cast<uint2*>(mine);
#pragma unroll
  for (int x = 0; x < kB; ++x) {
    uint16_t e[4];
    value(x, e);
    // columns 16 x + 4 (lane / 16): chunk 2 x + lane / 32, its half lane / 16 & 1
    half[(row * 16 + ((2 * x + (lane >> 5)) ^ row)) * 2 + ((lane >> 4) & 1)] =
        uint2{(uint32_t)e[0] | (uint32_t)e[1] << 16, (uint32_t)e[2] | (uint32_t)e[3] << 16};
  }
  wave_lds_sync();
  const int c = lane & 15, col = c * 8;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = q * 4 + (lane >> 4);
    uint4 v = mine[r * 16 + (c ^ r)];
    if (r < rows && col < cols) {
      uint16_t* to = out + r * ld + col;
      if (kLive && col + 8 > live) v = first_of(v, live - col);
      if (vec) {
        *reinterpret_cast<uint4*>(to) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < cols) to[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
  wave_lds_sync();
}

struct GradArgs {
  Operand h, w;  // listed rows [., K]; the piece's weight rows [., K]
  int64_t K, v_first;
  const Meta* meta;
  Listed rows;
  uint16_t* d;   // [piece rows][ldn]
  int64_t ldn;
  int tm, band;
};

// The piece's D: tokens x vocabulary, lane l of a block holding vocabulary row
// l & 15 and 4 tokens, whose lse, g and targets are in LDS.  Past the last
// listed row D is 0, also where the weight holds an infinity (0 * inf is a NaN
// logit there): dw reads D in chunks of 8 and multiplies what lies past the
// last row by zeros.
template <typename E>
__global__ __launch_bounds__(kThreads, 1) void grad_logits_kernel(GradArgs a) {
  GTP_LOOP_LDS;
  __shared__ __attribute__((aligned(16))) uint4 s_out[kWaves * kStoreLds];
  __shared__ __attribute__((aligned(16))) float s_lse[2][kTile], s_g[2][kTile];
  __shared__ __attribute__((aligned(16))) int s_t[2][kTile];
  const int n_listed = a.meta->n;
  Tiles at(blockIdx.x, a.tm, (n_listed + kTile - 1) / kTile, 1, a.band);
  if (!at.more()) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = wave >> 1, wv = wave & 1;
  Operand h = a.h;
  h.outer = n_listed;
  TileLoop<E, kAlongK, kAlongK> loop(
      Source<kAlongK>(h.ld, at.parts_n(), at.part_n(), wave, lane),
      Source<kAlongK>(a.w.ld, at.parts_m(), at.part_m(), wave, lane), sA0, sA1, sB0, sB1, s_unread,
      wave, lane);
  int vt, tt, share;
  at.place(vt, tt, share);
  loop.start(cursor_of<kAlongK>(h, (int64_t)tt * kTile, 0, a.K),
             cursor_of<kAlongK>(a.w, (int64_t)vt * kTile, 0, a.K));
  int odd = 0;
  for (bool more = true; more; odd ^= 1) {
    at.step();
    more = at.more();
    int vt2 = 0, tt2 = 0;
    Cursor ca{nullptr, 0, 0}, cb = ca;
    if (more) {
      at.place(vt2, tt2, share);
      ca = cursor_of<kAlongK>(h, (int64_t)tt2 * kTile, 0, a.K);
      cb = cursor_of<kAlongK>(a.w, (int64_t)vt2 * kTile, 0, a.K);
    }
    {
      const int64_t k = (int64_t)tt * kTile + threadIdx.x;
      const bool in = k < n_listed;
      // a row past the last: any value (its column is written as zeros)
      s_lse[odd][threadIdx.x] = in ? a.rows.lse[k] : kPosInf;
      s_g[odd][threadIdx.x] = in ? a.rows.g[k] : 0.0f;
      s_t[odd][threadIdx.x] = in ? (int)(a.rows.target[k] - a.v_first) : -1;
    }
    loop.tile(a.K, ca, cb);
#pragma unroll
    for (int y = 0; y < kB; ++y) {
        const int row0 = vt * kTile + wv * 128 + y * 16, v = row0 + (lane & 15);
        const int64_t col0 = (int64_t)tt * kTile + wt * 128;
        store_block<true>(s_out + wave * kStoreLds, lane, a.d + row0 * a.ldn + col0, a.ldn,
                          a.w.outer - row0, a.ldn - col0, n_listed - col0, true,
                    [&](int x, uint16_t (&e)[4]) {
                      const int t0 = wt * 128 + x * 16 + 4 * (lane >> 4);
                      const float4 l = *reinterpret_cast<const float4*>(&s_lse[odd][t0]);
                      const float4 g = *reinterpret_cast<const float4*>(&s_g[odd][t0]);
                      const int4 t = *reinterpret_cast<const int4*>(&s_t[odd][t0]);
                      const float ls[4] = {l.x, l.y, l.z, l.w}, gs[4] = {g.x, g.y, g.z, g.w};
                      const int ts[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
                      for (int i = 0; i < 4; ++i) {
                        const float q = acc_read(loop.acc[x][y][i]);
                        const float p = __builtin_amdgcn_exp2f((q - ls[i]) * kLog2e);
                        e[i] = E::from(gs[i] * ((ts[i] == v ? 1.0f : 0.0f) - p));
                      }
                    });
    }
    vt = vt2;
    tt = tt2;
  }
  wait_vm<0>();
}

// The piece's D for at most 16 kNB rows (past the last: zeros, whatever the
// weight holds), rounded to 16 bits and, 16 kNB elements on, what that left
// out.  With few rows the roundings of D do not average out against the
// results' own (56 rows of 2944: the gradients were off by 0.0026 against 64
// bits, rounding them alone takes 0.0017), the products are not what bounds
// them, and dh's tile has room for as many rows again.
template <typename E, int kNB>
__global__ __launch_bounds__(few::kThreads, 2) void few_grad_logits_kernel(GradArgs a) {
  constexpr int kTok = 16 * kNB;
  __shared__ __attribute__((aligned(16))) uint4 s_h[2][kTok * few::kChunks<kNB>];
  __shared__ __attribute__((aligned(16))) float s_lse[kTok], s_g[kTok];
  __shared__ __attribute__((aligned(16))) int s_t[kTok];
  const int n = a.meta->n, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x < kTok) {  // (the product's barriers publish them)
    const int k = threadIdx.x;
    s_lse[k] = k < n ? a.rows.lse[k] : kPosInf;
    s_g[k] = k < n ? a.rows.g[k] : 0.0f;
    s_t[k] = k < n ? (int)(a.rows.target[k] - a.v_first) : -1;
  }
  const int64_t first = (int64_t)blockIdx.x * few::kRows + wave * few::kWaveRows;
  few::Product<E, kNB, true> x;
  x.run(a.w, first, a.h, n, a.K, s_h);
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int64_t v = first + 16 * b + (lane & 15);
    if (v >= a.w.outer) continue;
#pragma unroll
    for (int y = 0; y < kNB; ++y) {
      const int t0 = 16 * y + 4 * (lane >> 4);
      uint16_t high[4], low[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float g = s_g[t0 + i];
        const float p = __builtin_amdgcn_exp2f((x.acc[b][y][i] - s_lse[t0 + i]) * kLog2e);
        const float d = g == 0.0f ? 0.0f : g * ((s_t[t0 + i] == v ? 1.0f : 0.0f) - p);
        high[i] = E::from(d);
        const float h = E::to(high[i]);
        low[i] = E::from(fabsf(h) < kPosInf ? d - h : 0.0f);
      }
      uint16_t* to = a.d + v * a.ldn + t0;
      *reinterpret_cast<uint2*>(to) = __builtin_bit_cast(uint2, high);
      *reinterpret_cast<uint2*>(to + kTok) = __builtin_bit_cast(uint2, low);
    }
  }
}

struct HiddenArgs {
  Operand d, w;  // D [piece rows][ldn] across K, the piece's weight rows across K
  int64_t K;     // piece rows
  const Meta* meta;
  float* sum;    // [shares][rows of the sums][width]
  Shares shares;
  int64_t width;
  int first, tn, band;
};

// dh in fp32, summed over the pieces in place: a tile's share of the piece's
// rows at a time.
template <typename E>
__global__ __launch_bounds__(kThreads, 1) void grad_hidden_kernel(HiddenArgs a) {
  GTP_LOOP_LDS;
  const int n_rows = (int)a.shares.rows(a.meta->n), splits = a.meta->splits;
  Tiles at(blockIdx.x, (n_rows + kTile - 1) / kTile, a.tn, splits, a.band);
  if (!at.more()) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = wave >> 1, wc = wave & 1;
  const int64_t steps = (a.K + kBK - 1) / kBK, per = (steps + splits - 1) / splits * kBK;
  auto k_of = [&](int split) { return min(a.K, split * per); };
  auto cursor_a = [&](int tt, int split) {
    return cursor_of<kAcrossK>(a.d, (int64_t)tt * kTile, k_of(split), k_of(split + 1) - k_of(split));
  };
  auto cursor_b = [&](int ct, int split) {
    return cursor_of<kAcrossK>(a.w, (int64_t)ct * kTile, k_of(split), k_of(split + 1) - k_of(split));
  };
  TileLoop<E, kAcrossK, kAcrossK> loop(
      Source<kAcrossK>(a.d.ld, at.parts_m(), at.part_m(), wave, lane),
      Source<kAcrossK>(a.w.ld, at.parts_n(), at.part_n(), wave, lane), sA0, sA1, sB0, sB1, s_unread,
      wave, lane);
  int tt, ct, split;
  at.place(tt, ct, split);
  loop.start(cursor_a(tt, split), cursor_b(ct, split));
  for (bool more = true; more;) {
    at.step();
    more = at.more();
    int tt2 = 0, ct2 = 0, split2 = 0;
    Cursor ca{nullptr, 0, 0}, cb = ca;
    if (more) {
      at.place(tt2, ct2, split2);
      ca = cursor_a(tt2, split2);
      cb = cursor_b(ct2, split2);
    }
    loop.tile(k_of(split + 1) - k_of(split), ca, cb);

    float* sum = a.sum + (int64_t)split * n_rows * a.width;
#pragma unroll
    for (int y = 0; y < kB; ++y) {
        const int64_t col = (int64_t)ct * kTile + wc * 128 + y * 16 + (lane & 15);
#pragma unroll
        for (int x = 0; x < kB; ++x) {
          const int k0 = tt * kTile + wt * 128 + x * 16 + 4 * (lane >> 4);
          const int rows = col < a.width ? n_rows - k0 : 0;
          float* to = sum + k0 * a.width + col;
          float q[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = acc_read(loop.acc[x][y][i]);
          if (!a.first) {
            float old[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) old[i] = i < rows ? to[i * a.width] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] += old[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < rows) to[i * a.width] = q[i];
          // (one block's addresses at a time)
          asm volatile("" ::: "memory");
        }
    }
    tt = tt2;
    ct = ct2;
    split = split2;
  }
  wait_vm<0>();
}

// grad_hidden [B x S, width] from the shares' sums; positions that were not
// listed get zeros.  One workgroup per position and 1024 columns.
template <typename E>
__global__ __launch_bounds__(256) void grad_hidden_rows_kernel(const float* __restrict__ sum,
                                                               int64_t width, Shares shares,
                                                               const Meta* __restrict__ meta,
                                                               const int32_t* __restrict__ slot,
                                                               uint16_t* __restrict__ out) {
  const int64_t pos = blockIdx.x, n_rows = shares.rows(meta->n);
  const int k = slot[pos], splits = meta->splits;
  const float inv = meta->inv;
  uint16_t* to = out + pos * width;
  const int64_t c0 = (int64_t)blockIdx.y * 1024 + threadIdx.x;
  float v[4] = {};
  if (k >= 0) {
    int64_t c[4];  // (no branch around a load: columns past the last read the last)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = min(c0 + i * 256, width - 1);
    for (int64_t at = shares.low + k; at >= 0; at -= shares.low) {  // the low part first
      const float* row = sum + at * width;
#pragma unroll 8
      for (int p = 0; p < splits; ++p, row += n_rows * width)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += row[c[i]];
      if (at == k) break;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    // (inv is the mean's gradient, which may be infinite or NaN)
    if (c0 + i * 256 < width) to[c0 + i * 256] = E::from(k >= 0 ? v[i] * inv : 0.0f);
}

struct WeightArgs {
  Operand h, d;  // listed rows across K, D [piece rows][ldn] along K
  const Meta* meta;
  uint16_t* out;  // the piece's first row of grad_weight, row stride ld
  int64_t ld, width;
  int tm, tn, band, vec;
};

// dw of the piece's rows: hidden columns x vocabulary rows, over the listed
// tokens.
template <typename E>
__global__ __launch_bounds__(kThreads, 1) void grad_weight_kernel(WeightArgs a) {
  GTP_LOOP_LDS;
  __shared__ __attribute__((aligned(16))) uint4 s_out[kWaves * kStoreLds];
  Tiles at(blockIdx.x, a.tm, a.tn, 1, a.band);
  if (!at.more()) return;
  const int64_t K = a.meta->n;
  const float inv = a.meta->inv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wc = wave >> 1, wv = wave & 1;
  TileLoop<E, kAcrossK, kAlongK> loop(
      Source<kAcrossK>(a.h.ld, at.parts_n(), at.part_n(), wave, lane),
      Source<kAlongK>(a.d.ld, at.parts_m(), at.part_m(), wave, lane), sA0, sA1, sB0, sB1, s_unread,
      wave, lane);
  int vt, ct, share;
  at.place(vt, ct, share);
  loop.start(cursor_of<kAcrossK>(a.h, (int64_t)ct * kTile, 0, K),
             cursor_of<kAlongK>(a.d, (int64_t)vt * kTile, 0, K));
  for (bool more = true; more;) {
    at.step();
    more = at.more();
    int vt2 = 0, ct2 = 0;
    Cursor ca{nullptr, 0, 0}, cb = ca;
    if (more) {
      at.place(vt2, ct2, share);
      ca = cursor_of<kAcrossK>(a.h, (int64_t)ct2 * kTile, 0, K);
      cb = cursor_of<kAlongK>(a.d, (int64_t)vt2 * kTile, 0, K);
    }
    loop.tile(K, ca, cb);
#pragma unroll
    for (int y = 0; y < kB; ++y) {
        const int64_t row0 = (int64_t)vt * kTile + wv * 128 + y * 16;
        const int64_t col0 = (int64_t)ct * kTile + wc * 128;
        store_block<false>(s_out + wave * kStoreLds, lane, a.out + row0 * a.ld + col0, a.ld,
                           a.d.outer - row0, a.width - col0, 0, a.vec,
                    [&](int x, uint16_t (&e)[4]) {
#pragma unroll
                      for (int i = 0; i < 4; ++i)
                        e[i] = E::from(acc_read(loop.acc[x][y][i]) * inv);
                    });
    }
    vt = vt2;
    ct = ct2;
  }
  wait_vm<0>();
}

// ------------------------------------------------------------ host

inline size_t up(size_t n) { return (n + 255) / 256 * 256; }

// A piece of the workspace, or its size alone where there is none.
struct Carve {
  unsigned char* base;
  size_t at = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + at) : nullptr;
    at += up(count * sizeof(T));
    return p;
  }
};

// Its parts are read in 16-byte chunks.
inline bool usable(const void* workspace) {
  return (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0;
}

// The sizes that a call's kernels share.
struct Shape {
  int64_t N, K8, ldh, ldn;  // rows with a target; K to a multiple of 8; row strides
  int n_vt, n_tt, n_ct;     // tiles of vocabulary, tokens and hidden columns
  int low;                  // few rows: where D's second part begins, else 0
};

inline int tiles(int64_t n) { return (int)((n + kTile - 1) / kTile); }

int shape_of(const gtp_linear_rows* r, Shape& s, Rows& a) {
  if (!r || r->B < 0 || r->S < 0 || r->T < 0 || r->T > r->S || r->K <= 0 || r->V <= 0 ||
      r->hidden_batch_stride < 0 || r->hidden_row_stride < 0 || r->weight_stride < r->K ||
      r->target_batch_stride < 0 || r->target_row_stride < 0)
    return GTP_ERR_INVALID_ARGUMENT;
  if (r->dtype != GTP_DTYPE_BF16 && r->dtype != GTP_DTYPE_F16) return GTP_ERR_UNSUPPORTED;
  if (r->B > kMaxLd || r->S > kMaxLd || r->B * r->S > kMaxLd - kTile || r->K > kMaxLd - 64 ||
      r->V > 0x7FFFFFFFll - kTile)
    return GTP_ERR_UNSUPPORTED;
  s.N = r->B * r->T;
  if (r->B * r->S > 0 && (!r->hidden || !r->weight || (s.N > 0 && !r->targets)))
    return GTP_ERR_INVALID_ARGUMENT;
  // the weight is read in place: whole 16-byte chunks of aligned rows
  s.K8 = (r->K + 7) / 8 * 8;
  if ((r->weight_stride & 7) || r->weight_stride < s.K8 || r->weight_stride > kMaxLd ||
      (reinterpret_cast<uintptr_t>(r->weight) & 15u))
    return GTP_ERR_UNSUPPORTED;
  s.ldh = (r->K + 63) / 64 * 64;
  // (few rows: D's two parts, 64 or 128 of them each)
  s.low = s.N <= few::kMostRows ? (int)(s.N + 63) / 64 * 64 : 0;
  s.ldn = s.low ? 2 * s.low : (s.N + 7) / 8 * 8;
  s.n_vt = tiles(r->V);
  s.n_tt = tiles(s.N);
  s.n_ct = tiles(s.K8);
  // the tiles are numbered in 32 bits
  // (dh's 32 times over)
  if ((int64_t)s.n_vt * s.n_tt >= (int64_t)1 << 24 || (int64_t)s.n_ct * s.n_vt >= (int64_t)1 << 24 ||
      (int64_t)s.n_ct * s.n_tt >= (int64_t)1 << 24)
    return GTP_ERR_UNSUPPORTED;
  a = Rows{r->targets, r->V, r->S, r->T, r->target_batch_stride, r->target_row_stride,
           r->ignore_index, (int)r->B, r->targets_int64 ? 1 : 0, r->has_ignore ? 1 : 0};
  return GTP_OK;
}

struct Forward {
  Meta* meta;
  int32_t *at, *target;
  float* xt;
  uint16_t* h;
  float2* partial;
  size_t bytes;
};
Forward forward_space(const Shape& s, void* ws) {
  Carve c{reinterpret_cast<unsigned char*>(ws)};
  Forward f;
  f.meta = c.take<Meta>(1);
  f.at = c.take<int32_t>(s.N);
  f.target = c.take<int32_t>(s.N);
  f.xt = c.take<float>(s.N);
  f.h = c.take<uint16_t>(s.N * s.ldh);
  f.partial = c.take<float2>((size_t)2 * s.n_vt * s.ldn);
  f.bytes = c.at;
  return f;
}

// Rows of the vocabulary per piece, a multiple of 8 tiles where there are as
// many (which keeps the grids whole), and the room for dh's shares: what all
// rows would take, or three times as many rows in up to 256 MiB.
struct Pieces {
  int64_t rows;
  Shares shares;
};
Pieces pieces_of(const Shape& s, int64_t V, int64_t width) {
  Pieces p;
  const int64_t rows = s.low ? s.low + s.N : s.N;
  const int64_t fit = max(kPieceBytes / (s.ldn * 2), (int64_t)kTile);
  const int64_t unit = fit >= 8 * kTile ? 8 * kTile : kTile;
  const int64_t most = fit / unit * unit, n = (V + most - 1) / most;
  p.rows = min(most, ((V + n - 1) / n + unit - 1) / unit * unit);
  p.shares = Shares{s.n_ct, (int32_t)device_cus(), s.low, (min(p.rows, V) + kBK - 1) / kBK, width,
                    32 * rows};
  p.shares.most = max(p.shares.best(rows) * rows, min(3 * rows, ((int64_t)1 << 26) / width));
  return p;
}

struct Backward {
  Meta* meta;
  Listed rows;
  int32_t* slot;
  uint16_t *h, *d;
  float* sum;
  size_t bytes;
};
Backward backward_space(const gtp_linear_rows* r, const Shape& s, const Pieces& p, void* ws) {
  Carve c{reinterpret_cast<unsigned char*>(ws)};
  Backward b;
  b.meta = c.take<Meta>(1);
  b.rows.at = c.take<int32_t>(s.N);
  b.rows.target = c.take<int32_t>(s.N);
  b.rows.lse = c.take<float>(s.N);
  b.rows.g = c.take<float>(s.N);
  b.slot = c.take<int32_t>(r->B * r->S);
  b.h = c.take<uint16_t>(s.N * s.ldh);
  b.d = c.take<uint16_t>(p.rows * s.ldn);
  b.sum = c.take<float>((size_t)p.shares.most * r->K);
  b.bytes = c.at;
  return b;
}

void gather(const gtp_linear_rows* r, const Shape& s, const Meta* meta, const int32_t* at,
            uint16_t* out, hipStream_t st) {
  const int vec = ((reinterpret_cast<uintptr_t>(r->hidden) & 15u) == 0 &&
                   (r->hidden_batch_stride & 7) == 0 && (r->hidden_row_stride & 7) == 0 &&
                   (r->K & 7) == 0)
                      ? 1
                      : 0;
  hipLaunchKernelGGL(gather_rows_kernel, dim3((unsigned)s.N), dim3(256), 0, st,
                     reinterpret_cast<const uint16_t*>(r->hidden), r->hidden_batch_stride,
                     r->hidden_row_stride, r->T, r->K, meta, at, vec, out, s.ldh);
}

template <typename E>
void forward_launch(const gtp_linear_rows* r, const Shape& s, const Forward& f, hipStream_t st) {
  LseArgs a;
  a.w = Operand{reinterpret_cast<const uint16_t*>(r->weight), r->weight_stride, r->V};
  a.h = Operand{f.h, s.ldh, s.N};
  a.K = s.K8;
  a.meta = f.meta;
  a.target = f.target;
  a.partial = f.partial;
  a.xt = f.xt;
  a.ldn = s.ldn;
  a.tm = s.n_vt;
  a.band = band_rows(s.n_vt, s.n_tt);
  if (s.N <= few::kMostRows) {
    const dim3 grid((unsigned)(2 * s.n_vt)), block(few::kThreads);
    s.N <= 64 ? launch_timed(few_lse_kernel<E, 4>, grid, block, st, a)
              : launch_timed(few_lse_kernel<E, 8>, grid, block, st, a);
    return;
  }
  launch_timed(lse_kernel<E>, dim3(grid_of(s.n_vt, s.n_tt)), dim3(kThreads), st, a);
}

// The three products of a piece of `rows` vocabulary rows from v0 on.
inline Operand piece_of(const gtp_linear_rows* r, int64_t v0, int64_t rows) {
  return Operand{reinterpret_cast<const uint16_t*>(r->weight) + v0 * r->weight_stride,
                 r->weight_stride, rows};
}

template <typename E>
void grad_logits_launch(const gtp_linear_rows* r, const Shape& s, const Backward& b, int64_t v0,
                        int64_t rows, hipStream_t st) {
  GradArgs a;
  a.h = Operand{b.h, s.ldh, s.N};
  a.w = piece_of(r, v0, rows);
  a.K = s.K8;
  a.v_first = v0;
  a.meta = b.meta;
  a.rows = b.rows;
  a.d = b.d;
  a.ldn = s.ldn;
  a.tm = tiles(rows);
  a.band = band_rows(a.tm, s.n_tt);
  if (s.N <= few::kMostRows) {
    const dim3 grid((unsigned)((rows + few::kRows - 1) / few::kRows)), block(few::kThreads);
    s.N <= 64 ? launch_timed(few_grad_logits_kernel<E, 4>, grid, block, st, a)
              : launch_timed(few_grad_logits_kernel<E, 8>, grid, block, st, a);
    return;
  }
  launch_timed(grad_logits_kernel<E>, dim3(grid_of(a.tm, s.n_tt)), dim3(kThreads), st, a);
}

template <typename E>
void grad_hidden_launch(const gtp_linear_rows* r, const Shape& s, const Pieces& p,
                        const Backward& b, int64_t v0,
                        int64_t rows, hipStream_t st) {
  HiddenArgs a;
  a.d = Operand{b.d, s.ldn, s.ldn};
  a.w = piece_of(r, v0, s.K8);
  a.K = rows;
  a.meta = b.meta;
  a.sum = b.sum;
  a.shares = p.shares;
  a.width = r->K;
  a.first = v0 == 0 ? 1 : 0;
  a.tn = s.n_ct;
  a.band = band_rows(s.n_tt, s.n_ct);
  // (the shares are picked on the device: as many workgroups as there can be)
  hipLaunchKernelGGL(grad_hidden_kernel<E>, dim3(kXcds * 32), dim3(kThreads), 0, st, a);
}

template <typename E>
void grad_weight_launch(const gtp_linear_rows* r, const Shape& s, const Backward& b, int64_t v0,
                        int64_t rows, uint16_t* grad_weight, hipStream_t st) {
  const int vec = (r->K & 7) == 0 && (reinterpret_cast<uintptr_t>(grad_weight) & 15u) == 0 ? 1 : 0;
  if (s.N <= few::kMostRows) {
    few::WeightArgs a;
    a.h = Operand{b.h, s.ldh, s.N};
    a.d = Operand{b.d, s.ldn, rows};
    a.n_listed = &b.meta->n;
    a.inv = &b.meta->inv;
    a.out = grad_weight + v0 * r->K;
    a.ld = r->K;
    a.width = r->K;
    const int cols = few::kWaves * (s.N <= 64 ? few::kWaveCols<4> : few::kWaveCols<8>);
    a.slabs = (int)((r->K + cols - 1) / cols);
    // three workgroups per CU (what their registers allow at once), each of 16
    // vocabulary rows at least
    const int64_t ranges = max((int64_t)3 * device_cus() / a.slabs, (int64_t)1);
    a.range = ((rows + ranges - 1) / ranges + 15) / 16 * 16;
    const int64_t each = ((rows + a.range - 1) / a.range + 7) / 8;
    const dim3 grid((unsigned)(8 * each * a.slabs)), block(few::kThreads);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a); };
    if (s.N <= 64)
      vec ? launch(few::few_weight_kernel<E, 4, true>) : launch(few::few_weight_kernel<E, 4, false>);
    else
      vec ? launch(few::few_weight_kernel<E, 8, true>) : launch(few::few_weight_kernel<E, 8, false>);
    return;
  }
  WeightArgs a;
  a.h = Operand{b.h, s.ldh, s.ldh};
  a.d = Operand{b.d, s.ldn, rows};
  a.meta = b.meta;
  a.out = grad_weight + v0 * r->K;
  a.ld = r->K;
  a.width = r->K;
  a.tm = tiles(rows);
  a.tn = s.n_ct;
  a.band = band_rows(a.tm, a.tn);
  a.vec = vec;
  hipLaunchKernelGGL(grad_weight_kernel<E>, dim3(grid_of(a.tm, a.tn)), dim3(kThreads), 0,
                     st, a);
}

template <typename E>
void backward_launch(const gtp_linear_rows* r, const Shape& s, const Pieces& p, const Backward& b,
                     uint16_t* grad_hidden, uint16_t* grad_weight, hipStream_t st) {
  for (int64_t v0 = 0; v0 < r->V; v0 += p.rows) {
    const int64_t rows = min(p.rows, r->V - v0);
    grad_logits_launch<E>(r, s, b, v0, rows, st);
    if (grad_hidden) grad_hidden_launch<E>(r, s, p, b, v0, rows, st);
    if (grad_weight) grad_weight_launch<E>(r, s, b, v0, rows, grad_weight, st);
  }
  if (grad_hidden)
    hipLaunchKernelGGL(grad_hidden_rows_kernel<E>,
                       dim3((unsigned)(r->B * r->S), (unsigned)((r->K + 1023) / 1024)), dim3(256), 0,
                       st, b.sum, r->K, p.shares, b.meta, b.slot, grad_hidden);
}

}  // namespace lin
}  // namespace gtp

using namespace gtp;

extern "C" size_t gtp_linear_logprob_workspace_bytes(const gtp_linear_rows* rows) {
  lin::Shape s;
  lin::Rows a;
  if (lin::shape_of(rows, s, a) != GTP_OK) return 0;
  return lin::forward_space(s, nullptr).bytes;
}

extern "C" int gtp_linear_logprob_rows(const gtp_linear_rows* rows, float* out_logprob,
                                       float* out_lse, float* mean_loss, int64_t* mean_count,
                                       uint32_t* verdict, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  lin::Shape s;
  lin::Rows a;
  const int rc = lin::shape_of(rows, s, a);
  if (rc != GTP_OK) return rc;
  if ((s.N > 0 && (!out_logprob || !out_lse)) || !workspace || (!mean_loss != !mean_count))
    return GTP_ERR_INVALID_ARGUMENT;
  const lin::Forward f = lin::forward_space(s, workspace);
  if (workspace_bytes < f.bytes || !lin::usable(workspace)) return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int i = 1; verdict && i < GTP_VERDICT_WORDS; ++i) verdict[i] = GTP_VERDICT_GOOD;
  hipLaunchKernelGGL(lin::list_rows_kernel, dim3(1), dim3(lin::kListBlock), 0, st, a,
                     lin::Listed{f.at, f.target, nullptr, nullptr}, f.meta, out_logprob, out_lse,
                     verdict, nullptr, nullptr, nullptr, nullptr, 0, lin::Shares{});
  if (s.N > 0) {
    lin::gather(rows, s, f.meta, f.at, f.h, st);
    if (rows->dtype == GTP_DTYPE_BF16)
      lin::forward_launch<gemm::Bf16>(rows, s, f, st);
    else
      lin::forward_launch<gemm::F16>(rows, s, f, st);
    auto merge = [&](auto kernel, int64_t rows_each) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)((s.N + rows_each - 1) / rows_each)),
                         dim3(lin::kMergeBlock), 0, st, f.partial, s.ldn, 2 * s.n_vt, f.meta, f.at,
                         f.xt, out_logprob, out_lse);
    };
    // few rows: more threads for each
    s.N <= few::kMostRows ? merge(lin::lse_merge_kernel<4>, 4) : merge(lin::lse_merge_kernel<16>, 16);
  }
  if (mean_loss)
    hipLaunchKernelGGL(lin::mean_kernel, dim3(1), dim3(1024), 0, st, f.meta, f.at, out_logprob,
                       mean_loss, mean_count);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}

extern "C" size_t gtp_linear_logprob_backward_workspace_bytes(const gtp_linear_rows* rows) {
  lin::Shape s;
  lin::Rows a;
  if (lin::shape_of(rows, s, a) != GTP_OK || s.N == 0) return 0;
  return lin::backward_space(rows, s, lin::pieces_of(s, rows->V, rows->K), nullptr).bytes;
}

extern "C" int gtp_linear_logprob_backward(const gtp_linear_rows* rows, const float* lse,
                                           const float* grad, const int64_t* mean_count,
                                           void* grad_hidden, void* grad_weight, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  lin::Shape s;
  lin::Rows a;
  const int rc = lin::shape_of(rows, s, a);
  if (rc != GTP_OK) return rc;
  // without a row there is nothing to list, and both gradients are zeros that
  // the caller writes
  if (s.N == 0) return GTP_ERR_UNSUPPORTED;
  if (!lse || !grad || !workspace) return GTP_ERR_INVALID_ARGUMENT;
  const lin::Pieces p = lin::pieces_of(s, rows->V, rows->K);
  const lin::Backward b = lin::backward_space(rows, s, p, workspace);
  if (workspace_bytes < b.bytes || !lin::usable(workspace)) return GTP_ERR_INVALID_ARGUMENT;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(lin::list_rows_kernel, dim3(1), dim3(lin::kListBlock), 0, st, a, b.rows,
                     b.meta, nullptr, nullptr, nullptr, grad, mean_count, lse, b.slot,
                     rows->dtype == GTP_DTYPE_F16 ? 1 : 0, p.shares);
  lin::gather(rows, s, b.meta, b.rows.at, b.h, st);
  uint16_t* gh = reinterpret_cast<uint16_t*>(grad_hidden);
  uint16_t* gw = reinterpret_cast<uint16_t*>(grad_weight);
  if (rows->dtype == GTP_DTYPE_BF16)
    lin::backward_launch<gemm::Bf16>(rows, s, p, b, gh, gw, st);
  else
    lin::backward_launch<gemm::F16>(rows, s, p, b, gh, gw, st);
  return hipGetLastError() == hipSuccess ? GTP_OK : GTP_ERR_LAUNCH;
}
