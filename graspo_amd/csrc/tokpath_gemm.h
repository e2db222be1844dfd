// tokpath_gemm.h -- the matrix-core tile loop of the hidden-state losses (gfx950).
//
// One workgroup of 4 waves accumulates a 256 x 256 tile of A B^T in fp32 on
// v_mfma_f32_32x32x16 (bf16 or fp16 operands), each wave 128 x 128 (4 x 4
// blocks, 256 accumulators per lane).  K advances 64 at a time through two
// LDS stages of 32 KB per operand, filled straight from global memory
// (buffer_load_dwordx4 ... lds) while the matrix cores work on the other one.
//
// An operand lies in memory in one of two ways, and neither is copied or
// transposed for the product:
//
// - kAlongK: a row per output index, K contiguous.  A stage holds 256 rows of
//   128 bytes, whose eight 16-byte chunks are XOR-swizzled by bits 1-3 of the
//   row, so that the 16 rows of a fragment read take all 16 bank groups.
// - kAcrossK: a row per K index, output indices contiguous.  A stage holds 64
//   rows of 512 bytes.  ds_read_b64_tr_b16 turns 4 rows x 16 columns around on
//   the way out of LDS: of 16 lanes, lane i receives column i's 4 values.  The
//   16-byte chunks are XOR-swizzled by 4 (row & 3), so that the 4 rows x 64
//   bytes that half a wave reads take all 64 banks.
//
// Nothing past an operand's rows or its K is read: the buffer resource ends
// with the last valid row, a chunk past K gets an offset past that end, and a
// load out of range writes zeros to LDS.
#pragma once

#include "tokpath_stream.h"

namespace gtp {
namespace gemm {

constexpr int kTile = 256;             // rows and columns of a tile
constexpr int kBK = 64;                // K per stage
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kB = 4;                  // 32-wide blocks per wave along each side
constexpr int kQ = 8;                  // 1 KB loads per wave, operand and K step
constexpr int kStage = kTile * kBK / 8;  // 16-byte chunks per operand stage
constexpr int kXcds = 8;
constexpr int kMaxLd = (1 << 22) - 1;  // row strides (elements): 256 rows fit a buffer range
constexpr int kRsrcWord3 = 0x00020000;  // raw buffer: 32-bit data format, no swizzle
constexpr uint32_t kPast = 0x80000000u;  // an offset past every resource

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

enum Layout { kAlongK, kAcrossK };

// 16-bit element types: product and rounding (nearest, ties to even)
struct Bf16 {
  __device__ static __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint16_t from(float v) {
    return __builtin_bit_cast(uint16_t, (__bf16)v);
  }
  __device__ static __forceinline__ float to(uint16_t v) { return u2f((uint32_t)v << 16); }
};
struct F16 {
  __device__ static __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint16_t from(float v) {
    return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
  __device__ static __forceinline__ float to(uint16_t v) { return f16_to_f32(v); }
};

// `outer` rows (kAlongK) or columns (kAcrossK) of 16-bit values; rows 16-byte
// aligned and `ld` elements apart, ld and (kAcrossK) outer multiples of 8.
struct Operand {
  const uint16_t* p;
  int64_t ld, outer;
};

// s_waitcnt vmcnt(0), the other counters untouched
__device__ __forceinline__ void wait_vm0() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// An accumulator read straight from its AGPR (keeps the compiler from
// copying every accumulator to VGPRs at once before an epilogue).
__device__ __forceinline__ float acc_read(float a) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
  return v;
}

// Where an operand's K steps for one tile lie (uniform over the workgroup).
struct Cursor {
  const char* at;  // the next step's first byte
  int64_t left;    // bytes from there to the end of what the tile may read
  int k_left;      // kAlongK: K from there on
};
// Of the tile whose first row (kAlongK) or column (kAcrossK) is `first`, for K
// values of K from k_first (a multiple of 8) on.
template <Layout L>
__device__ __forceinline__ Cursor cursor_of(const Operand& o, int64_t first, int64_t k_first,
                                            int64_t K) {
  const int64_t ld = o.ld * 2, outer = max((int64_t)0, o.outer - first);
  if constexpr (L == kAlongK)
    return Cursor{reinterpret_cast<const char*>(o.p) + first * ld + k_first * 2,
                  min((int64_t)kTile, outer) * ld - k_first * 2, (int)K};
  else
    return Cursor{reinterpret_cast<const char*>(o.p + first) + k_first * ld,
                  outer > 0 && K > 0 ? (K - 1) * ld + outer * 2 : 0, (int)K};
}

// One operand's K steps, in order: wave w's load q of a step fills the 1 KB of
// LDS from chunk (8w + q) * 64 on, 16 bytes per lane.
template <Layout L>
struct Source {
  Cursor c;
  uint32_t v0, v1;  // the lane's byte offset for even and odd q
  int c0, c1;       // kAlongK: its first k within the step
  uint32_t qstep;   // bytes from q to q + 2, halved
  int64_t advance;  // bytes from step to step

  __device__ __forceinline__ Source(int64_t ld_elements, int wave, int lane) : c{nullptr, 0, 0} {
    const int64_t ld = ld_elements * 2;
    if constexpr (L == kAlongK) {
      advance = kBK * 2;
      // LDS row 8 (8w + q) + lane / 8, chunk lane & 7 of it holding chunk
      // (lane & 7) ^ ((row >> 1) & 7) of the row
      const int row = wave * kQ * 8 + (lane >> 3);
      c0 = ((lane & 7) ^ ((lane >> 4) & 7)) * 8;
      c1 = ((lane & 7) ^ ((4 + (lane >> 4)) & 7)) * 8;
      v0 = (uint32_t)(row * ld + c0 * 2);
      v1 = (uint32_t)(row * ld + c1 * 2);
      qstep = (uint32_t)(8 * ld);
    } else {
      advance = kBK * ld;
      // LDS row 2 (8w + q) + lane / 32, chunk lane & 31 of it holding chunk
      // (lane & 31) ^ 4 (row & 3) of the row
      const int row = wave * kQ * 2 + (lane >> 5);
      v0 = (uint32_t)(row * ld + ((lane & 31) ^ ((lane >> 5) << 2)) * 16);
      v1 = (uint32_t)(row * ld + ((lane & 31) ^ ((2 + (lane >> 5)) << 2)) * 16);
      c0 = c1 = 0;
      qstep = (uint32_t)(2 * ld);
    }
  }

  struct Step {
    const char* base;
    int bytes;
    uint32_t v0, v1;
  };
  // The next step; past the last one all its loads are out of range.
  __device__ __forceinline__ Step next() {
    const int n = (int)max((int64_t)0, min(c.left, (int64_t)kPast));
    Step s{c.at, n, v0, v1};
    if constexpr (L == kAlongK) {
      s.v0 = c0 < c.k_left ? v0 : kPast;
      s.v1 = c1 < c.k_left ? v1 : kPast;
      c.k_left -= kBK;
    }
    c.at += advance;
    c.left -= advance;
    return s;
  }
  // the whole offset goes in the VGPR operand: the range check covers it
  __device__ __forceinline__ void issue(const Step& s, int q, uint4* stage, int wave) const {
    const uint32_t v = ((q & 1) ? s.v1 : s.v0) + (uint32_t)q * qstep;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)s.base, (short)0, s.bytes, kRsrcWord3);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(stage + (wave * kQ + q) * 64), 16, v,
                                             0, 0, 0);
  }
};

// Fragment x (32 outer indices from side * 128 + 32 x on) of k16 step kk:
// lane l holds index l & 31 of it and k = 8 (l / 32) .. + 7.
template <Layout L>
__device__ __forceinline__ s16x8 fragment(const uint4* stage, int side, int x, int kk, int lane) {
  if constexpr (L == kAlongK) {
    const int ch = (2 * kk + (lane >> 5)) ^ ((lane >> 1) & 7);
    return __builtin_bit_cast(s16x8, stage[(side * 128 + x * 32 + (lane & 31)) * 8 + ch]);
  } else {
    // row 16 kk + 8 (l / 32) + 4 h + r, columns 32 (4 side + x) + 16 ((l / 16) & 1) + 4 (l & 3)
    const int r = (lane & 15) >> 2;
    const int at = (8 * (lane >> 5) + r) * 512 + side * 256 + ((x ^ r) * 64) +
                   ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    const char* p = reinterpret_cast<const char*>(stage) + at + kk * 16 * 512;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * 512));
    return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

// The tile loop of a workgroup: acc[x][y] = A rows (block x) times B rows
// (block y), lane l of a block holding B index l & 31 and the A indices
// 8 (i / 4) + 4 (l / 32) + (i & 3) for i = 0 .. 15.
//
// The loop runs on from tile to tile: the last two K steps of a tile load the
// first two of the next one, so that its operands come in while the epilogue
// works on the accumulators (a tile started anew cost 12 us of 110 at K =
// 4096).
//
// The four stages are four arrays, so that the compiler sees that the loads in
// flight write to others than it reads (from one array it waits for all loads
// before every transposing read: 877 against 1225 TFLOP/s).
template <typename E, Layout LA, Layout LB>
struct TileLoop {
  typedef typename Source<LA>::Step StepA;
  typedef typename Source<LB>::Step StepB;
  Source<LA> a;
  Source<LB> b;
  uint4 *sA0, *sA1, *sB0, *sB1;
  int wave, lane;
  StepA na;  // the step whose loads are going out
  StepB nb;
  f32x16 acc[kB][kB];
  // fragments of the k16 step at work and of the next one, [0, kB) of A and
  // [kB, 2 kB) of B
  s16x8 f[2][2 * kB];

  __device__ __forceinline__ TileLoop(int64_t lda, int64_t ldb, uint4* sA0_, uint4* sA1_,
                                      uint4* sB0_, uint4* sB1_, int wave_, int lane_)
      : a(lda, wave_, lane_), b(ldb, wave_, lane_), sA0(sA0_), sA1(sA1_), sB0(sB0_), sB1(sB1_),
        wave(wave_), lane(lane_) {}

  __device__ __forceinline__ void issue_one(int j, uint4* sa, uint4* sb) {
    if (j & 1)
      b.issue(nb, j >> 1, sb, wave);
    else
      a.issue(na, j >> 1, sa, wave);
  }
  // read i of a k16 step, in the order in which the MFMAs want them
  __device__ __forceinline__ void read_one(int set, int i, const uint4* sa, const uint4* sb, int kk) {
    if (i == 0)
      f[set][0] = fragment<LA>(sa, wave >> 1, 0, kk, lane);
    else if (i <= kB)
      f[set][kB + i - 1] = fragment<LB>(sb, wave & 1, i - 1, kk, lane);
    else
      f[set][i - kB] = fragment<LA>(sa, wave >> 1, i - kB, kk, lane);
  }
  // 16 MFMAs of one k16 step from fragment set c.  Among them, one after the
  // other so that neither queue holds the matrix cores up: the reads of the
  // next k16 step (kk of stage (ra, rb)) and, with j0 >= 0, the loads j0 ..
  // j0 + 7 into stage (la, lb).
  __device__ __forceinline__ void mfma16(int c, const uint4* ra, const uint4* rb, int kk, int j0,
                                         uint4* la, uint4* lb) {
#pragma unroll
    for (int x = 0; x < kB; ++x)
#pragma unroll
      for (int y = 0; y < kB; ++y) {
        const int i = x * kB + y;
        acc[x][y] = E::mfma(f[c][x], f[c][kB + y], acc[x][y]);
        if (i % 2 == 0) read_one(c ^ 1, i / 2, ra, rb, kk);
        if (i % 2 == 1 && j0 >= 0) issue_one(j0 + i / 2, la, lb);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  // A K step from stage (ca, cb), whose first k16 fragments are already in
  // set 0.  The next step lives in (sa, sb): its loads 0-7 went out during the
  // last k16 of the step before this one, its loads 8-15 go out during the
  // first k16 here.  The barrier that publishes it sits before the last k16:
  // every wave has read all of this step's fragments by then, so the loads 0-7
  // of the step after the next into (ca, cb) go out during that last k16,
  // while the next step's first fragments are read.
  __device__ __forceinline__ void step(uint4* ca, uint4* cb, uint4* sa, uint4* sb) {
    mfma16(0, ca, cb, 1, kQ, sa, sb);
    mfma16(1, ca, cb, 2, -1, sa, sb);
    mfma16(0, ca, cb, 3, -1, sa, sb);
    na = a.next();
    nb = b.next();
    wait_vm0();
    __syncthreads();
    mfma16(1, sa, sb, 0, 0, ca, cb);
  }
  // Ahead of the first tile.
  __device__ __forceinline__ void start(const Cursor& ca, const Cursor& cb) {
    a.c = ca;
    b.c = cb;
    na = a.next();
    nb = b.next();
#pragma unroll
    for (int j = 0; j < 2 * kQ; ++j) issue_one(j, sA0, sB0);
    na = a.next();
    nb = b.next();
#pragma unroll
    for (int j = 0; j < kQ; ++j) issue_one(j, sA1, sB1);
    wait_vm0();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * kB; ++i) read_one(0, i, sA0, sB0, 0);
  }
  // One tile over K (at least its first two steps; past K they are zeros),
  // then on to the tile of the cursors given (empty ones behind the last).
  __device__ __forceinline__ void tile(int64_t K, const Cursor& next_a, const Cursor& next_b) {
#pragma unroll
    for (int x = 0; x < kB; ++x)
#pragma unroll
      for (int y = 0; y < kB; ++y) acc[x][y] = f32x16{};
    // an even number of steps (the stages alternate)
    int pairs = (int)((K + 2 * kBK - 1) / (2 * kBK));
    pairs = pairs < 1 ? 1 : pairs;
    for (int p = 0; p < pairs; ++p) {
      if (p + 1 == pairs) {
        a.c = next_a;
        b.c = next_b;
      }
      step(sA0, sB0, sA1, sB1);
      step(sA1, sB1, sA0, sB0);
    }
    // epilogues read the accumulators by inline asm, which the compiler's
    // hazard checks do not see: no MFMA may be scheduled past this point, and
    // 24 wait states after the last one cover its result latency (11 for an
    // 8-pass MFMA)
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  }
};

// The order of tm x tn tiles (`shares` times over, for products whose K is
// split).  Tiles are numbered through bands of h rows, down each column of a
// band, so that a run of 32 covers a block of h x 32 / h.  Workgroup b runs on
// XCD b mod 8: an XCD takes every eighth run of 32 tiles, one tile per
// workgroup, whose 8 + 4 operand tiles (12 is the fewest for 32 workgroups)
// its L2 serves; up to 256 tiles are cut into eight runs.  h is picked on the
// host for the most tiles that there can be and fits any smaller number.
inline int band_rows(int64_t tm, int64_t tn) {
  int h = 8;
  while (h > 1 && h / 2 >= tm) h /= 2;
  while (h < 32 && 32 / h / 2 >= tn) h *= 2;
  return h;
}
__host__ __device__ __forceinline__ int run_of(int64_t tiles) {
  return tiles >= 32 * kXcds ? 32 : (int)((tiles + kXcds - 1) / kXcds);
}
// Workgroups: one per tile up to one per CU of the whole chip.
inline unsigned grid_of(int64_t tm, int64_t tn, int64_t shares = 1) {
  return (unsigned)(kXcds * run_of(tm * tn * shares));
}
// Walks the tiles of one workgroup.
struct Tiles {
  uint32_t all, each, run, at, tn, h, tm;
  __device__ __forceinline__ Tiles(uint32_t b, int tm_, int tn_, int shares, int h_)
      : each((uint32_t)tm_ * tn_), tn(tn_), h(h_), tm(tm_) {
    all = each * shares;
    run = run_of(all);
    const uint32_t i = b / kXcds;
    at = i < run ? b % kXcds * run + i : all;
  }
  __device__ __forceinline__ bool more() const { return at < all; }
  __device__ __forceinline__ void step() { at += kXcds * run; }
  __device__ __forceinline__ void place(int& m, int& n, int& share) const {
    share = at / each;
    const uint32_t t = at - share * each, band = t / (h * tn), q = t - band * h * tn;
    const uint32_t rows = min(h, tm - band * h);
    m = band * h + q % rows;
    n = q / rows;
  }
};

}  // namespace gemm
}  // namespace gtp
