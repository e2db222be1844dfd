// What the tile loop of tokpath_gemm.h reads of its operands, walked on the
// host: every load and prefetch of every lane, as the buffer resource's range
// check lets it through.  An operand is `outer` rows (along K) or columns
// (across K), its rows `ld` elements apart, and its memory ends with its last
// row's last element.  Prints what is read outside and what is not read of it.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../graspo_amd/csrc/tokpath_gemm.h"

using namespace gtp::gemm;

static int64_t failures = 0;

template <Layout L>
struct Walk {
  int64_t outer, K, ld, first, base = (int64_t)1 << 40;
  std::vector<char> seen;  // elements of the tile that a load has read

  int64_t rows() const { return L == kAlongK ? outer : K; }
  // elements of a row that belong to the operand: whole chunks of 8 along K
  int64_t cols() const { return L == kAlongK ? (K + 7) / 8 * 8 : outer; }

  void read(int64_t address, int bytes, bool load, const char* what) {
    for (int64_t at = address; at < address + bytes; at += 2) {
      const int64_t e = (at - base) / 2, row = e / ld, col = e % ld;
      // (across K a row's gap may be read, the memory's end not be passed)
      const bool in = at >= base && row < rows() &&
                      (L == kAlongK ? col < cols() : e < (rows() - 1) * ld + cols());
      if (!in) {
        if (failures++ < 5)
          printf("%s reads row %lld column %lld of outer %lld, K %lld, ld %lld (tile at %lld)\n", what,
                 (long long)row, (long long)col, (long long)outer, (long long)K, (long long)ld,
                 (long long)first);
        return;
      }
      if (load && col < cols()) seen[row * cols() + col] = 1;
    }
  }
  void loads(const std::vector<Source<L>>& lanes, const std::vector<typename Source<L>::Step>& s, int q0,
             int q1) {
    for (int t = 0; t < kThreads; ++t)
      for (int q = q0; q < q1; ++q) {
        const uint32_t off = lanes[t].offset(s[t], q);
        for (uint32_t j = off; j < off + 16; j += 4)
          if ((int64_t)j + 4 <= (int64_t)(uint32_t)s[t].bytes) read((int64_t)s[t].base + j, 4, true, "a load");
      }
  }
  // One tile, then nothing: as TileLoop::start and TileLoop::tile go.
  void run() {
    seen.assign(rows() * cols(), 0);
    Operand o{reinterpret_cast<const uint16_t*>(base), ld, outer};
    std::vector<Source<L>> lanes;
    std::vector<typename Source<L>::Step> s(kThreads);
    for (int t = 0; t < kThreads; ++t) lanes.emplace_back(ld, 1, 0, t / 64, t % 64);
    auto next = [&] {
      for (int t = 0; t < kThreads; ++t) s[t] = lanes[t].next();
    };
    for (auto& l : lanes) l.c = cursor_of<L>(o, first, 0, K);
    next();
    loads(lanes, s, 0, kQ);
    next();
    loads(lanes, s, 0, kQ / 2);
    const int pairs = K > 0 ? (int)((K + 2 * kBK - 1) / (2 * kBK)) : 1;
    for (int p = 0; p < pairs; ++p) {
      if (p + 1 == pairs)
        for (auto& l : lanes) l.c = Cursor{nullptr, 0, 0};
      for (int half = 0; half < 2; ++half) {
        loads(lanes, s, kQ / 2, kQ);
        for (auto& l : lanes)
          if ((int64_t)l.line + 4 <= (int64_t)(uint32_t)l.ahead_bytes())
            read((int64_t)l.c.at + l.line, 4, false, "the prefetch");
        next();
        loads(lanes, s, 0, kQ / 2);
      }
    }
    const int64_t end = std::min(outer, first + kTile);
    for (int64_t i = first; i < end; ++i)
      for (int64_t k = 0; k < K; ++k)
        if (!seen[L == kAlongK ? i * cols() + k : k * cols() + i]) {
          if (failures++ < 5)
            printf("not read: index %lld k %lld of outer %lld, K %lld, ld %lld\n", (long long)i,
                   (long long)k, (long long)outer, (long long)K, (long long)ld);
          return;
        }
  }
};

template <Layout L>
static void all_tiles(int64_t outer, int64_t K, int64_t ld) {
  for (int64_t first = 0; first == 0 || first < outer; first += kTile)
    Walk<L>{outer, K, ld, first}.run();
}

// gemm_ranges along|across outer K ld
int main(int argc, char** argv) {
  if (argc != 5) return 2;
  const int64_t outer = atoll(argv[2]), K = atoll(argv[3]), ld = atoll(argv[4]);
  argv[1][1] == 'l' ? all_tiles<kAlongK>(outer, K, ld) : all_tiles<kAcrossK>(outer, K, ld);
  printf("%lld failures\n", (long long)failures);
  return failures != 0;
}
