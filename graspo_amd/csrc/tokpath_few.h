// tokpath_few.h -- the vocabulary's products with at most 128 rows (gfx950).
//
// With so few rows the weight's bytes bound them, not the matrix cores: tiles
// of 256 x 256 leave the cores to rows that are not there, and one workgroup
// per CU waits for each step's loads.  So here a wave streams its own rows of
// the weight from memory straight into the operands of the products (each is
// used once, by this wave alone), two stages in flight, and only the few rows
// of the other operand go through LDS, where the workgroup's waves share them.
// Several workgroups per CU hide each other's waits.
//
// 61 rows of 4096, 151936 of the vocabulary, bf16 (1.24 GB; a plain read of it
// in this pattern takes 225 us, a fill 190): the lse 411 us with the tiles and
// 320 so (50 of them the write-back of what ran before), D 381 and 286, dw 385
// and 262; forward and backward 1.39 and 1.12 ms.  At 127 rows 1.37 ms; the
// tiles take 1.50 at 129.  (With D in one part 1.11 and 1.28 ms, and gradients
// off by 0.0024 instead of 0.0017: see few_grad_logits_kernel.)
#pragma once
#include "tokpath_gemm.h"

namespace gtp {
namespace few {

using gemm::f32x4;
using gemm::s16x8;

constexpr int kMostRows = 128;
constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kWaveRows = 32, kRows = kWaves * kWaveRows;  // vocabulary rows
// K per stage, what the registers hold, and the 16-byte chunks of a row in it
template <int kNB>
constexpr int kStep = kNB == 4 ? 128 : 64;
template <int kNB>
constexpr int kChunks = kStep<kNB> / 8;

__device__ __forceinline__ s16x8 as_frag(const uint4& v) { return __builtin_bit_cast(s16x8, v); }

// `count` elements from p on, at most 2 GiB of them; loads past them give 0.
constexpr uint32_t kNowhere = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const uint16_t* p, int64_t count) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), 0,
                                           (int)min(max(2 * count, (int64_t)0), (int64_t)0x7FFFFFF0),
                                           0x00020000);
}
__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t b, uint32_t at) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0));
}

// The workgroups begin at different stages and go round: all at the same one
// read the same part of rows that are a power of two apart, from few memory
// channels (61 rows of 4096, 151936 of the vocabulary: 383 us, and 318 so).
//
// The product of the wave's 32 vocabulary rows with the 16 kNB other rows:
// acc[x][y] over vocabulary block x and row block y.  kRowsFirst: the rows are
// the product's first operand, so that a lane holds vocabulary row lane & 15
// and four rows; else row lane & 15 and four vocabulary rows.
template <typename E, int kNB, bool kRowsFirst>
struct Product {
  static constexpr int kK = kStep<kNB>, kC = kChunks<kNB>, kS = kK / 32;
  static constexpr int kLoads = 16 * kNB * kC / kThreads;  // chunks of h per thread
  f32x4 acc[2][kNB];

  // where chunk c of row t lies: a block's 16 rows on 16 groups of 4 banks
  __device__ static __forceinline__ int place(int t, int c) {
    return t * kC + (c ^ (kC == 16 ? t & 15 : (t >> 1) & 7));
  }

  __device__ __forceinline__ void run(const gemm::Operand& w, int64_t first, const gemm::Operand& h,
                                      int n, int64_t K, uint4 (*s_h)[16 * kNB * kC]) {
    const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15;
    // (loads without branches, or the compiler waits for all of them at each:
    // what lies past the last row or K is out of the buffer's range, and 0)
    const __amdgpu_buffer_rsrc_t w_buf = buffer(w.p + first * w.ld, (w.outer - first) * w.ld);
    const __amdgpu_buffer_rsrc_t h_buf = buffer(h.p, n * h.ld);
    const uint32_t w_at[2] = {(uint32_t)(2 * (r * w.ld + 8 * q)),
                              (uint32_t)(2 * ((16 + r) * w.ld + 8 * q))};
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < kNB; ++y) acc[x][y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    uint4 wa[2][kS], wb[2][kS], hr[kLoads];
    auto load_w = [&](int k0, uint4 (&to)[2][kS]) {
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          to[x][s] = load16(w_buf, k0 + 32 * s + 8 * q < K ? w_at[x] + 2 * (k0 + 32 * s) : kNowhere);
    };
    auto load_h = [&](int k0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = tid + i * kThreads, k = k0 + 8 * (at % kC);
        hr[i] = load16(h_buf, k < h.ld ? 2 * (uint32_t)(at / kC * h.ld + k) : kNowhere);
      }
    };
    auto store_h = [&](uint4* to) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = tid + i * kThreads, row = at / kC, c = at % kC;
        to[place(row, c)] = hr[i];
      }
    };
    auto multiply = [&](const uint4* h_at, const uint4 (&wf)[2][kS]) {
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int y = 0; y < kNB; ++y) {
          const s16x8 b = as_frag(h_at[place(16 * y + r, 4 * s + q)]);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            acc[x][y] = kRowsFirst ? E::mul(b, as_frag(wf[x][s]), acc[x][y])
                                   : E::mul(as_frag(wf[x][s]), b, acc[x][y]);
        }
    };
    // Two stages in flight: what is loaded behind stage i's products is stored
    // (h) and multiplied (the weight) after stage i + 1's.  h's loads come
    // first, so that storing them does not wait for the weight's.
    const int stages = (int)((K + kK - 1) / kK);
    int at = (int)(blockIdx.x % (unsigned)stages);
    auto load = [&](uint4 (&to)[2][kS]) {
      const int k = at * kK;
      at = at + 1 == stages ? 0 : at + 1;
      load_h(k);
      load_w(k, to);
    };
    load(wa);
    store_h(s_h[0]);
    load(wb);
    __syncthreads();
    // (the buffer written in a stage was last read in the one before)
    for (int i = 0; i < stages; i += 2) {
      multiply(s_h[0], wa);
      if (i + 1 >= stages) break;
      store_h(s_h[1]);
      load(wa);
      __syncthreads();
      multiply(s_h[1], wb);
      store_h(s_h[0]);
      load(wb);
      __syncthreads();
    }
  }
};

// dw[v][c] = inv * sum over the rows of D[v][.] h[.][c], D in two parts: a wave holds its 128
// (more than 64 rows: 64) columns of h as first operands and walks the vocabulary 16 rows at a time.
// Bound by the writes.
template <int kNB>
constexpr int kWaveCols = kNB == 4 ? 128 : 64;

struct WeightArgs {
  gemm::Operand h, d;  // listed rows [., ld]; D [piece rows][2][16 kNB], rounded and the rest
  const int32_t* n_listed;
  const float* inv;
  uint16_t* out;  // row stride ld
  int64_t ld, width;
  int slabs;        // of the columns, one per workgroup
  int64_t range;    // vocabulary rows per workgroup, a multiple of 16
};

// D goes through LDS, kStaged rows at a time and a stage ahead: loads wait in
// the memory pipeline behind the stores before them (61 rows of 4096, 151936
// of the vocabulary, D in one part: 353 us with each block's D loaded a block
// ahead, 320 with stages loaded where they are due, 238 so, 216 with one stage
// alone).
// kVec: 16-byte stores.
template <int kNB>
constexpr int kStaged = kNB == 4 ? 96 : 48;

// Two chunks of a stage, and the wait for them.  (In asm: a read that the
// compiler sees waits for the other stage's loads and the stores before them.)
__device__ __forceinline__ void read2(const uint4* p0, const uint4* p1, s16x8& a, s16x8& b) {
  typedef __attribute__((address_space(3))) const uint4 lds_const;
  const uint32_t at0 = (uint32_t)(uintptr_t)(lds_const*)p0, at1 = (uint32_t)(uintptr_t)(lds_const*)p1;
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(a), "=&v"(b)
               : "v"(at0), "v"(at1));
}

template <int kLeft>
__device__ __forceinline__ void wait_all_but() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
}

template <typename E, int kNB, bool kVec>
__global__ __launch_bounds__(kThreads, 2) void few_weight_kernel(WeightArgs a) {
  constexpr int kX = kWaveCols<kNB> / 16, kS = kNB / 2;
  const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the workgroups of one XCD take all columns of a range after one another
  const int xcd = blockIdx.x % 8, in_xcd = blockIdx.x / 8;
  const int64_t first = ((int64_t)(in_xcd / a.slabs) * 8 + xcd) * a.range;
  const int64_t c0 = ((int64_t)(in_xcd % a.slabs) * kWaves + wave) * kWaveCols<kNB>;
  const int64_t last = min(first + a.range, a.d.outer);
  if (first >= last) return;
  constexpr int kC = 4 * kNB;  // 16-byte chunks of a row of D
  constexpr int kLoads = kStaged<kNB> * kC / kThreads;  // per thread and stage
  __shared__ __attribute__((aligned(16))) uint4 s_d0[kStaged<kNB> * kC], s_d1[kStaged<kNB> * kC];
  auto place = [](int t, int c) { return t * kC + (c ^ (t & 15)); };
  const int n = *a.n_listed;
  const float inv = *a.inv;
  // blocks 2 j and 2 j + 1 hold columns 32 j + 8 (m / 4) + m % 4 and 4 more in
  // their row m, so that a lane's results are 8 columns in a row
  s16x8 h[kX][kS];
#pragma unroll
  for (int x = 0; x < kX; ++x)
#pragma unroll
    for (int s = 0; s < kS; ++s) {
      const int64_t c = c0 + 32 * (x / 2) + 8 * (r >> 2) + (r & 3) + 4 * (x & 1);
      s16x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = 32 * s + 8 * q + j;
        v[j] = t < n && c < a.h.ld ? (short)a.h.p[t * a.h.ld + c] : (short)0;
      }
      h[x][s] = v;
    }
  // the lane's 8 columns of block pair x / 2, for the buffers' ranges
  uint32_t col_at[kX / 2];
#pragma unroll
  for (int x = 0; x < kX / 2; ++x) {
    const int64_t c = c0 + 32 * x + 8 * q;
    col_at[x] = c < a.width ? 2 * (uint32_t)(r * a.ld + c) : kNowhere;
  }
  auto block = [&](int64_t v0, int row, const uint4* s_d) {
    f32x4 acc[kX];
#pragma unroll
    for (int x = 0; x < kX; ++x) acc[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int part = kC / 2; part >= 0; part -= kC / 2) {
      s16x8 d[kS];
#pragma unroll
      for (int s = 0; s < kS; s += 2)
        read2(&s_d[place(row + r, part + 4 * s + q)], &s_d[place(row + r, part + 4 * s + 4 + q)],
              d[s], d[s + 1]);
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int x = 0; x < kX; ++x) acc[x] = E::mul(h[x][s], d[s], acc[x]);
    }
    // (rows past the last: none of the buffer)
    const __amdgpu_buffer_rsrc_t out =
        buffer(a.out + v0 * a.ld, min(last - v0, (int64_t)16) * a.ld);
#pragma unroll
    for (int x = 0; x < kX; x += 2) {
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = E::from(acc[x + i / 4][i & 3] * inv);
      if constexpr (kVec) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, e), out, col_at[x / 2], 0,
                                               0);
      } else if (v0 + r < last) {
        const int64_t c = c0 + 16 * x + 8 * q;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < a.width) a.out[(v0 + r) * a.ld + c + i] = e[i];
      }
    }
  };
  // A stage's loads, straight to LDS (its place in the chunks' order is the
  // lane's to read); rows past the last of the piece are 0.
  auto issue = [&](int64_t v0, uint4* stage) {
    const __amdgpu_buffer_rsrc_t rows = buffer(a.d.p + v0 * a.d.ld, (a.d.outer - v0) * a.d.ld);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int slot = (wave * kLoads + j) * kWave, t = (slot + lane) / kC;
      const int c = place(t, (slot + lane) % kC) - t * kC;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (gemm::lds_void*)(stage + slot), 16,
                                               2 * (uint32_t)(t * a.d.ld + 8 * c), 0, 0, 0);
    }
    // (before the stores that the wait below lets be)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  const bool active = c0 < a.width;
  // the stage that is due: its loads are the oldest but a full stage's stores
  auto publish = [&] {
    constexpr int kStores = kVec ? kStaged<kNB> / 16 * (kX / 2) : 0;
    if (active)
      wait_all_but<kStores>();
    else
      wait_all_but<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  int64_t v0 = first;
  // one stage, and whether another follows
  auto stage = [&](const uint4* here, uint4* next) {
    const bool more = v0 + kStaged<kNB> < last;
    if (more) issue(v0 + kStaged<kNB>, next);
    const int rows = (int)min((int64_t)kStaged<kNB>, last - v0);
    if (active)
      for (int row = 0; row < rows; row += 16) block(v0 + row, row, here);
    v0 += kStaged<kNB>;
    if (more) publish();
    return more;
  };
  issue(first, s_d0);
  wait_all_but<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  while (stage(s_d0, s_d1) && stage(s_d1, s_d0)) {
  }
}

}  // namespace few
}  // namespace gtp
