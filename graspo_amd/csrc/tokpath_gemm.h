// tokpath_gemm.h -- the matrix-core tile loop of the hidden-state losses (gfx950).
//
// One workgroup of 4 waves accumulates a 256 x 256 tile of A B^T in fp32 on
// v_mfma_f32_16x16x32 (bf16 or fp16 operands), each wave 128 x 128 (8 x 8
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
//   16-byte chunks are XOR-swizzled by 4 (row & 3) + 2 (row / 8 & 1), so that
//   the 8 rows x 32 bytes that half a wave reads take all 64 banks.
//
// Nothing past an operand's rows or its K (in whole chunks) is read: the buffer
// resource ends with the last valid row's K, a chunk past K gets an offset past
// that end, and a load out of range writes zeros to LDS.
//
// What bounds it: the part's power (the library's product keeps the matrix
// cores busy 93% of the cycles, at 1.58 GHz).  At 8192 x 4096 x 131072 the four
// products (the lse, D, dh, dw) reach 1434, 1421, 1514 and 1510 TFLOP/s, the
// library's of the same sizes 1538-1630 on that card; cards differ by 7-10%.
// What brought it there from 880-1170, each measured on one box:
// - a stage per array (the compiler waits for all loads in flight before a
//   transposing read of an array that one of them writes): 877 -> 1225 TFLOP/s
//   with both operands across K;
// - the reads and loads one by one among the MFMAs, not ahead of them: +2-6%;
// - tile after tile without a stop (TileLoop): +1-5%, more with a short K;
// - 16 x 16 x 32 in place of 32 x 32 x 16 (half the accumulator traffic per
//   product, so a higher clock), fragments in halves of a side, and the
//   accumulators held in place by inline asm (the compiler moved them between
//   register files): +3-7%;
// - each K step's lines brought into L2 a step ahead of its loads, every line
//   by one of the workgroups that share it: +4-8% (a step's loads alone took
//   1.5 us from behind L2 and 0.7 us from L2, against 1.1 us of products).
#pragma once

#include "tokpath_stream.h"

namespace gtp {
namespace gemm {

constexpr int kTile = 256;             // rows and columns of a tile
constexpr int kBK = 64;                // K per stage
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kB = 8;                  // 16-wide blocks per wave along each side
constexpr int kH = kB / 2;             // half a side
constexpr int kQ = 8;                  // 1 KB loads per wave, operand and K step
constexpr int kStage = kTile * kBK / 8;  // 16-byte chunks per operand stage
constexpr int kXcds = 8;
constexpr int kMaxLd = (1 << 22) - 1;  // row strides (elements): 256 rows fit a buffer range
constexpr int kRsrcWord3 = 0x00020000;  // raw buffer: 32-bit data format, no swizzle
constexpr uint32_t kPast = 0x80000000u;  // an offset past every resource

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

enum Layout { kAlongK, kAcrossK };

// 16-bit element types: product and rounding (nearest, ties to even).  The
// product is inline asm so that an accumulator stays in its registers: from
// the builtins the compiler made 250 moves between register files per 256
// products.  It does not see the asm's wait states: its operands come from LDS
// (which it waits for) and never from a vector instruction, and TileLoop keeps
// what writes or reads an accumulator away from the products.
struct Bf16 {
  __device__ static __forceinline__ void mfma(f32x4& c, s16x8 a, s16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  __device__ static __forceinline__ f32x4 mul(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a),
                                                   __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint16_t from(float v) {
    return __builtin_bit_cast(uint16_t, (__bf16)v);
  }
  __device__ static __forceinline__ float to(uint16_t v) { return u2f((uint32_t)v << 16); }
};
struct F16 {
  __device__ static __forceinline__ void mfma(f32x4& c, s16x8 a, s16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  }
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  __device__ static __forceinline__ f32x4 mul(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a),
                                                  __builtin_bit_cast(x8, b), c, 0, 0, 0);
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

// s_waitcnt vmcnt(n), the other counters untouched
template <int kLeft>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | kLeft);
}

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
__host__ __device__ __forceinline__ Cursor cursor_of(const Operand& o, int64_t first,
                                                     int64_t k_first, int64_t K) {
  // (HIP's min and max are those of int on the host)
  const int64_t ld = o.ld * 2, outer = o.outer > first ? o.outer - first : 0;
  if constexpr (L == kAlongK)
    // (the last row ends with its K's last chunk: a wider row's gap behind it
    // may lie past the end of the memory)
    return Cursor{reinterpret_cast<const char*>(o.p) + first * ld + k_first * 2,
                  outer > 0 && K > 0
                      ? ((outer < kTile ? outer : kTile) - 1) * ld + (K + 7) / 8 * 16
                      : 0,
                  (int)K};
  else
    return Cursor{reinterpret_cast<const char*>(o.p + first) + k_first * ld,
                  outer > 0 && K > 0 ? (K - 1) * ld + outer * 2 : 0, (int)K};
}

// One operand's K steps, in order: wave w's load q of a step fills the 1 KB of
// LDS from chunk (8w + q) * 64 on, 16 bytes per lane.
template <Layout L>
struct Source {
  Cursor c;
  uint32_t v[2][2];  // the lane's byte offset for (q & 1, q / 4)
  int c0, c1;        // kAlongK: its first k within the step, for even and odd q
  uint32_t qstep;    // bytes from q to q + 2, halved
  uint32_t line;     // the line of a step that this lane brings into L2
  int64_t advance;   // bytes from step to step

  // part of parts: this workgroup's share of the lines
  __host__ __device__ __forceinline__ Source(int64_t ld_elements, int parts, int part, int wave, int lane)
      : c{nullptr, 0, 0} {
    const int64_t ld = ld_elements * 2;
    if constexpr (L == kAlongK) {
      advance = kBK * 2;
      // LDS row 8 (8w + q) + lane / 8, chunk lane & 7 of it holding chunk
      // (lane & 7) ^ ((row >> 1) & 7) of the row
      const int row = wave * kQ * 8 + (lane >> 3);
      c0 = ((lane & 7) ^ ((lane >> 4) & 7)) * 8;
      c1 = ((lane & 7) ^ ((4 + (lane >> 4)) & 7)) * 8;
      v[0][0] = v[0][1] = (uint32_t)(row * ld + c0 * 2);
      v[1][0] = v[1][1] = (uint32_t)(row * ld + c1 * 2);
      qstep = (uint32_t)(8 * ld);
      line = (uint32_t)((wave * 64 + lane) * ld);
    } else {
      advance = kBK * ld;
      // LDS row 2 (8w + q) + lane / 32, chunk lane & 31 of it holding chunk
      // (lane & 31) ^ (4 (row & 3) + 2 (row / 8 & 1)) of the row
      const int row = wave * kQ * 2 + (lane >> 5);
#pragma unroll
      for (int odd = 0; odd < 2; ++odd)
#pragma unroll
        for (int high = 0; high < 2; ++high)
          v[odd][high] = (uint32_t)(
              row * ld + ((lane & 31) ^ ((2 * odd + (lane >> 5)) << 2) ^ (high << 1)) * 16);
      c0 = c1 = 0;
      qstep = (uint32_t)(2 * ld);
      line = (uint32_t)((wave * 16 + (lane >> 2)) * ld + (lane & 3) * 128);
    }
    if ((wave * 64 + lane) * parts / 256 != part) line = kPast;
  }

  struct Step {
    const char* base;
    int bytes;
    uint32_t v[2][2];
  };
  __host__ __device__ __forceinline__ int bytes_left() const {
    return (int)(uint32_t)(c.left < 0 ? 0 : c.left < (int64_t)kPast ? c.left : (int64_t)kPast);
  }
  // The next step; past the last one all its loads are out of range.
  __host__ __device__ __forceinline__ Step next() {
    Step s{c.at, bytes_left(), {{v[0][0], v[0][1]}, {v[1][0], v[1][1]}}};
    if constexpr (L == kAlongK) {
      s.v[0][0] = s.v[0][1] = c0 < c.k_left ? v[0][0] : kPast;
      s.v[1][0] = s.v[1][1] = c1 < c.k_left ? v[1][0] : kPast;
      c.k_left -= kBK;
    }
    c.at += advance;
    c.left -= advance;
    return s;
  }
  __host__ __device__ __forceinline__ uint32_t offset(const Step& s, int q) const {
    return s.v[q & 1][q >> 2] + (uint32_t)q * qstep;
  }
  // the whole offset goes in the VGPR operand: the range check covers it
  __device__ __forceinline__ void issue(const Step& s, int q, uint4* stage, int wave) const {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)s.base, (short)0, s.bytes, kRsrcWord3);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(stage + (wave * kQ + q) * 64), 16,
                                             offset(s, q), 0, 0, 0);
  }
  // (a tile's last step may begin past K: the number of steps is even)
  __host__ __device__ __forceinline__ int ahead_bytes() const {
    return L == kAlongK && c.k_left <= 0 ? 0 : bytes_left();
  }
  // The lines of the step that next() will give, into L2 (4 bytes of each go
  // to LDS that nothing reads: a load without a register).
  __device__ __forceinline__ void ahead(uint32_t* unread, int wave) const {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)c.at, (short)0, ahead_bytes(), kRsrcWord3);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(unread + wave * 64), 4, line, 0, 0, 0);
  }
};

// Fragment x (16 outer indices from side * 128 + 16 x on) of k32 step kk:
// lane l holds index l & 15 of it and k = 8 (l / 16) .. + 7.
template <Layout L>
__device__ __forceinline__ s16x8 fragment(const uint4* stage, int side, int x, int kk, int lane) {
  if constexpr (L == kAlongK) {
    const int ch = (4 * kk + (lane >> 4)) ^ ((lane >> 1) & 7);
    return __builtin_bit_cast(s16x8, stage[(side * 128 + x * 16 + (lane & 15)) * 8 + ch]);
  } else {
    // row 32 kk + 8 g + 4 h + r, columns 128 side + 16 x + 4 (l & 3)
    const int r = (lane & 15) >> 2, g = lane >> 4;
    const int chunk = (2 * x + ((lane & 3) >> 1)) ^ (r << 2) ^ ((g & 1) << 1);
    const int at = (8 * g + r) * 512 + side * 256 + chunk * 16 + (lane & 1) * 8;
    const char* p = reinterpret_cast<const char*>(stage) + at + kk * 32 * 512;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * 512));
    return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

// The tile loop of a workgroup: acc[x][y] = A rows (block x) times B rows
// (block y), lane l of a block holding B index l & 15 and the A indices
// 4 (l / 16) + i for i = 0 .. 3.
//
// The loop runs on from tile to tile: the last two K steps of a tile load the
// first two of the next one, so that its operands come in while the epilogue
// works on the accumulators.
//
// A k32 step is four quadrants of 16 products, walked so that each changes one
// side's half, and the fragments of a half are read one quadrant ahead into
// the registers that the other half's quadrant has left: 64 registers of
// fragments in place of 128.
template <typename E, Layout LA, Layout LB>
struct TileLoop {
  typedef typename Source<LA>::Step StepA;
  typedef typename Source<LB>::Step StepB;
  Source<LA> a;
  Source<LB> b;
  uint4 *sA0, *sA1, *sB0, *sB1;
  uint32_t* unread;  // 256 words of LDS
  int wave, lane;
  StepA na;  // the step whose loads are going out
  StepB nb;
  f32x4 acc[kB][kB];
  s16x8 fa[kB], fb[kB];

  __device__ __forceinline__ TileLoop(const Source<LA>& a_, const Source<LB>& b_, uint4* sA0_,
                                      uint4* sA1_, uint4* sB0_, uint4* sB1_, uint32_t* unread_,
                                      int wave_, int lane_)
      : a(a_), b(b_), sA0(sA0_), sA1(sA1_), sB0(sB0_), sB1(sB1_), unread(unread_), wave(wave_),
        lane(lane_) {}

  __device__ __forceinline__ void issue_one(int j, uint4* sa, uint4* sb) {
    if (j & 1)
      b.issue(nb, j >> 1, sb, wave);
    else
      a.issue(na, j >> 1, sa, wave);
  }
  __device__ __forceinline__ void read_a(int x, const uint4* sa, int kk) {
    fa[x] = fragment<LA>(sa, wave >> 1, x, kk, lane);
  }
  __device__ __forceinline__ void read_b(int y, const uint4* sb, int kk) {
    fb[y] = fragment<LB>(sb, wave & 1, y, kk, lane);
  }
  // Quadrant (kX, kY).  Among its products, one after the other so that
  // neither queue holds the matrix cores up: the reads of A's half kReadA (of
  // k32 step ka of sa) and B's half kReadB (kb of sb), -1 for none, and the
  // loads kFirst .. kLast - 1 into (la, lb).
  template <int kX, int kY, int kReadA, int kReadB, int kFirst, int kLast>
  __device__ __forceinline__ void quadrant(const uint4* sa, int ka, const uint4* sb, int kb,
                                           uint4* la, uint4* lb) {
    constexpr int n = kLast - kFirst;
#pragma unroll
    for (int x = 0; x < kH; ++x)
#pragma unroll
      for (int y = 0; y < kH; ++y) {
        const int i = x * kH + y;
        E::mfma(acc[kX * kH + x][kY * kH + y], fa[kX * kH + x], fb[kY * kH + y]);
        if (kReadB >= 0 && i % 4 == 0) read_b(kReadB * kH + i / 4, sb, kb);
        if (kReadA >= 0 && i % 4 == (kReadB >= 0 ? 2 : 0)) read_a(kReadA * kH + i / 4, sa, ka);
        if ((i + 1) * n / 16 != i * n / 16) issue_one(kFirst + i * n / 16, la, lb);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  // A K step from stage (ca, cb), with half 0 of both sides of its first k32
  // step read.  The next step lives in (sa, sb): its loads 0-7 went out in the
  // last two quadrants of the step before this one, its loads 8-15 go out in
  // the first two here.  The barrier that publishes it sits before the last
  // two quadrants: every wave has read all of this step's fragments by then,
  // so the loads 0-7 of the step after the next into (ca, cb) go out during
  // those, while the next step's first fragments are read.  The wait leaves
  // out the two loads of `ahead`, which are behind all of the next step's.
  __device__ __forceinline__ void step(uint4* ca, uint4* cb, uint4* sa, uint4* sb) {
    quadrant<0, 0, -1, 1, 8, 12>(ca, 0, cb, 0, sa, sb);
    quadrant<0, 1, 1, -1, 12, 16>(ca, 0, cb, 0, sa, sb);
    a.ahead(unread, wave);
    b.ahead(unread, wave);
    quadrant<1, 1, 0, -1, 0, 0>(ca, 1, cb, 0, sa, sb);
    quadrant<1, 0, -1, 1, 0, 0>(ca, 0, cb, 1, sa, sb);
    quadrant<0, 1, 1, 0, 0, 0>(ca, 1, cb, 1, sa, sb);
    quadrant<0, 0, -1, -1, 0, 0>(ca, 0, cb, 0, sa, sb);
    na = a.next();
    nb = b.next();
    publish<2>();
    quadrant<1, 0, 0, -1, 0, 4>(sa, 0, sb, 0, ca, cb);
    quadrant<1, 1, -1, 0, 4, 8>(sa, 0, sb, 0, ca, cb);
  }
  // Waits until at most kLeft of the wave's vector-memory accesses are out and
  // its LDS reads are done, then for the other waves.
  template <int kLeft>
  __device__ __forceinline__ void publish() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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
    publish<0>();
#pragma unroll
    for (int i = 0; i < kH; ++i) {
      read_a(i, sA0, 0);
      read_b(i, sB0, 0);
    }
  }
  // One tile over K (at least its first two steps; past K they are zeros),
  // then on to the tile of the cursors given (empty ones behind the last).
  __device__ __forceinline__ void tile(int64_t K, const Cursor& next_a, const Cursor& next_b) {
#pragma unroll
    for (int x = 0; x < kB; ++x)
#pragma unroll
      for (int y = 0; y < kB; ++y) acc[x][y] = f32x4{};
    // the zeros are written here, and 8 wait states before the first product
#pragma unroll
    for (int x = 0; x < kB; ++x)
      asm volatile(""
                   : "+a"(acc[x][0]), "+a"(acc[x][1]), "+a"(acc[x][2]), "+a"(acc[x][3]),
                     "+a"(acc[x][4]), "+a"(acc[x][5]), "+a"(acc[x][6]), "+a"(acc[x][7]));
    asm volatile("s_nop 7" ::: "memory");
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
    // 24 wait states cover the last product's latency before its accumulators
    // are read
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
  // Of the 32 workgroups of a run, those with the same m (or n) share that
  // operand's lines.
  __device__ __forceinline__ int parts_m() const { return max(1u, run / h); }
  __device__ __forceinline__ int part_m() const { return blockIdx.x / kXcds / h % parts_m(); }
  __device__ __forceinline__ int parts_n() const { return min(h, run); }
  __device__ __forceinline__ int part_n() const { return blockIdx.x / kXcds % parts_n(); }
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
