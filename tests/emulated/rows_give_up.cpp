// Waits that give up in the bulk-copy kernels of tq4_rows.cu (rows.inc: their source): what has not been read is not overwritten, nothing
// but rows of the caches is ever stored, no copy is in flight when a block ends, and it is reported.
#include "warp.h"

namespace tq4 {
namespace {
#include "rows.inc"
}  // namespace

namespace {
constexpr int kBlock = 16, kRow = 32, kStride = 48, kPages = 24;
int failures = 0;
#define EXPECT(x)                                                             \
  do {                                                                        \
    if (!(x) && failures++ < 10) std::printf("line %d: %s\n", __LINE__, #x);  \
  } while (0)

struct Cache {
  std::vector<unsigned char> now, was;
  explicit Cache(unsigned seed) : now((size_t)kPages * kBlock * kStride) {
    for (auto& b : now) b = (unsigned char)((seed = seed * 1664525u + 1013904223u) >> 24);
    was = now;
  }
  bool row_is(int64_t at, int64_t from) const { return !std::memcmp(now.data() + at, was.data() + from, kRow); }
  bool untouched(int64_t at) const { return row_is(at, at); }
};
Geometry geometry() { return Geometry{kPages, kBlock * kStride, kStride, kBlock, kRow / 16}; }

// lanes whose first wait(s) give up: all of them, or one
struct Who {
  int lane;
  bool is(int l) const { return lane < 0 || l == lane; }
};

void long_lists(int failing, Who who, bool healthy) {
  constexpr int kLayers = 2, kHeld = 5, kOf = 300, kKept = 150, kSeg = 4, kSegments = (kKept + kSeg - 1) / kSeg;
  std::vector<Cache> c{Cache(1), Cache(2)};
  std::vector<int32_t> table(kPages), keep;
  for (int i = 0; i < kPages; ++i) table[i] = (i * 7 + 3) % kPages;
  for (int i = 0; (int)keep.size() < kKept; ++i)
    if (i % 3 != 1 || kOf - i <= kKept - (int)keep.size()) keep.push_back(i);
  int32_t first = kHeld, kept = kKept;
  int ticket = 0, valid = kKept, flag = 0;
  std::vector<int> loaded(kLayers * kSegments, 0);
  CompactArgs a{};
  a.g = geometry();
  a.table = table.data();
  a.table_width = kPages;
  a.first = &first;
  a.keep = keep.data();
  a.keep_width = kKept;
  a.kept = &kept;
  a.seqs = 1;
  a.layers = kLayers;
  a.segments = kSegments;
  a.seg_rows = kSeg;
  a.ticket = &ticket;
  a.valid = &valid;
  a.loaded = loaded.data();
  a.err_flag = &flag;
  Caches at{};
  for (int i = 0; i < kLayers; ++i) at.at[i] = c[i].now.data();
  auto row = [&](int pos) { return (int64_t)table[pos / kBlock] * kBlock * kStride + pos % kBlock * kStride; };
  for (int b = 0; b < kLayers * kSegments; ++b) {
    g_gives_up = [&](int lane, int look) { return !healthy && b == failing && look == 0 && who.is(lane); };
    EXPECT(run_block(b, [&] { compact_long_bulk_kernel(at, a); }));
  }
  if (healthy) {
    EXPECT(flag == 0);
    for (auto& x : c)
      for (int j = 0; j < kKept; ++j) EXPECT(x.row_is(row(kHeld + j), row(kHeld + keep[j])));
    return;
  }
  EXPECT(flag == TQ4_DEV_TIMEOUT);
  const int seg = failing / kLayers, layer = failing % kLayers;  // (tickets: layers fastest)
  for (int l = 0; l < kLayers; ++l)
    for (int j = 0; j < kKept; ++j) {
      const int64_t to = row(kHeld + j), from = row(kHeld + keep[j]);
      if (l != layer) {
        EXPECT(c[l].row_is(to, from));
      } else if (j / kSeg == seg) {
        EXPECT(c[l].untouched(to) && c[l].untouched(from));  // (its rows are where they were)
      } else {
        EXPECT(c[l].untouched(to) || c[l].row_is(to, from));
      }
    }
}

void short_lists(int failing, Who who, bool healthy) {
  constexpr int kLayers = 3, kHeld = 30, kKept = 10;
  std::vector<Cache> c{Cache(1), Cache(2), Cache(3)};
  std::vector<int32_t> table(kPages), keep{0, 2, 3, 7, 8, 9, 12, 20, 21, 30};
  for (int i = 0; i < kPages; ++i) table[i] = (i * 5 + 1) % kPages;
  int32_t first = kHeld, kept = kKept, len = -1;
  int flag = 0;
  CompactArgs a{};
  a.g = geometry();
  a.table = table.data();
  a.table_width = kPages;
  a.first = &first;
  a.keep = keep.data();
  a.keep_width = kKept;
  a.kept = &kept;
  a.lens_out = &len;
  a.seqs = 1;
  a.layers = kLayers;
  a.per_block = 2;
  a.rows = 8;
  a.err_flag = &flag;
  Caches at{};
  for (int i = 0; i < kLayers; ++i) at.at[i] = c[i].now.data();
  auto row = [&](int pos) { return (int64_t)table[pos / kBlock] * kBlock * kStride + pos % kBlock * kStride; };
  for (int b = 0; b < 2; ++b) {
    g_gives_up = [&](int lane, int look) { return !healthy && b == 0 && look == failing && who.is(lane); };
    EXPECT(run_block(b, [&] { compact_short_bulk_kernel(at, a); }));
  }
  EXPECT(len == kHeld + kKept && flag == (healthy ? 0 : TQ4_DEV_TIMEOUT));
  for (int l = 0; l < kLayers; ++l)
    for (int j = 0; j < kKept; ++j) {
      const int64_t to = row(kHeld + j), from = row(kHeld + keep[j]);
      EXPECT(c[l].row_is(to, from) || (!healthy && l < 2 && c[l].untouched(to) && c[l].untouched(from)));
    }
}

void pages(int failing, Who who, bool healthy) {
  constexpr int kLayers = 5;
  std::vector<Cache> c;
  for (int i = 0; i < kLayers; ++i) c.emplace_back(i + 1);
  const int64_t pairs[2][2] = {{3, 8}, {4, 20}};
  int flag = 0;
  CopyArgs a{};
  a.g = geometry();
  a.pairs = pairs;
  a.pairs_64 = 1;
  a.n = 2;
  a.layers = a.per_block = kLayers;
  a.rows = 7;  // (three sets a page: fifteen of them through the four stages)
  a.err_flag = &flag;
  Caches at{};
  for (int i = 0; i < kLayers; ++i) at.at[i] = c[i].now.data();
  for (int b = 0; b < 2; ++b) {
    g_gives_up = [&](int lane, int look) { return !healthy && b == 0 && look == failing && who.is(lane); };
    EXPECT(run_block(b, [&] { copy_blocks_bulk_kernel(at, a); }));
  }
  EXPECT(flag == (healthy ? 0 : TQ4_DEV_TIMEOUT));
  for (int l = 0; l < kLayers; ++l)
    for (int p = 0; p < 2; ++p)
      for (int t = 0; t < kBlock; ++t) {
        const int64_t from = (pairs[p][0] * kBlock + t) * kStride, to = (pairs[p][1] * kBlock + t) * kStride;
        EXPECT(c[l].untouched(from) && (c[l].row_is(to, from) || (!healthy && p == 0 && c[l].untouched(to))));
      }
}
}  // namespace
}  // namespace tq4

int main(int argc, char** argv) {
  using namespace tq4;
  const std::string which = argc > 1 ? argv[1] : "";
  void (*f)(int, Who, bool) = which == "long" ? long_lists : which == "short" ? short_lists : pages;
  f(-1, Who{-1}, true);
  const int n = which == "long" ? 76 : which == "short" ? 3 : 15;
  for (int failing = 0; failing < n; failing += which == "long" ? 15 : 1)
    for (const int lane : {-1, 0, 1}) f(failing, Who{lane}, false);
  std::printf("%d failures\n", failures);
  return failures != 0;
}
