// Checks and plans of the layer operators (csrc/mmf_layer.hpp) on the host: prints a line for every
// expectation that does not hold and exits with their number.
#include <cstdio>
#include <cstring>
#include <set>
#include <vector>

#include "../matmulfreellmcpu_amd/csrc/mmf_layer.hpp"

using namespace mmf;

static int bad = 0;
static void want(const char* what, const char* got, const char* part) {
  const bool ok = part ? got && std::strstr(got, part) : !got;
  if (!ok) {
    std::printf("%s: got '%s', wanted '%s'\n", what, got ? got : "accepted", part ? part : "accepted");
    ++bad;
  }
}
static void is(const char* what, long got, long expect) {
  if (got != expect) {
    std::printf("%s: got %ld, wanted %ld\n", what, got, expect);
    ++bad;
  }
}

// addresses only: nothing here is read
template <class T> static T* at(uintptr_t a) { return reinterpret_cast<T*>(a); }

static NormQArgs norm() {
  return {kF32, at<float>(0x10000), at<float>(0x20000), at<float>(0x900), at<float>(0x30000), nullptr,
          at<int8_t>(0x40000), at<float>(0x50000), 4, 100, 0, 0, 0, 0, 0, 1e-6f};
}
static void norms() {
  auto go = [](const char* what, const char* part, auto&& change) {
    NormQArgs a = norm();
    change(a);
    want(what, check(a), part);
  };
  go("norm", nullptr, [](NormQArgs&) {});
  go("norm type", "dtype", [](NormQArgs& a) { a.dtype = kI8; });
  go("norm type below", "dtype", [](NormQArgs& a) { a.dtype = -1; });
  go("norm stride", "stride", [](NormQArgs& a) { a.ldx = 99; });
  go("norm wide stride", "stride", [](NormQArgs& a) { a.ldcodes = size_t{1} << 32; });
  go("norm null x", "null", [](NormQArgs& a) { a.x = nullptr; });
  go("norm null codes", "null", [](NormQArgs& a) { a.codes = nullptr; });
  go("norm null scales", "null", [](NormQArgs& a) { a.scales = nullptr; });
  go("norm null w", "null", [](NormQArgs& a) { a.w = nullptr; });
  go("norm no rows", nullptr, [](NormQArgs& a) { a.rows = 0, a.x = nullptr; });
  go("norm no columns", nullptr, [](NormQArgs& a) { a.cols = 0; });
  go("norm many rows", "rows", [](NormQArgs& a) { a.rows = kMaxRows + 1; });
  go("norm long rows", "long", [](NormQArgs& a) { a.cols = kMaxCols + 1; });
  go("norm odd address", "aligned", [](NormQArgs& a) { a.x = at<char>(0x10002); });
  go("norm bf16 at 2 bytes", nullptr, [](NormQArgs& a) { a.dtype = kBF16, a.x = at<char>(0x10002); });
  go("norm no residual", nullptr, [](NormQArgs& a) { a.res = nullptr; });
  go("norm h in place of x", nullptr, [](NormQArgs& a) { a.h = const_cast<void*>(a.x); });
  go("norm h in place of res", nullptr, [](NormQArgs& a) { a.h = const_cast<void*>(a.res); });
  go("norm h shifted", "overlaps", [](NormQArgs& a) { a.h = at<float>(0x20004); });
  go("norm h in place, other stride", "overlaps", [](NormQArgs& a) { a.h = const_cast<void*>(a.x), a.ldh = 101; });
  go("norm y on x", "overlaps", [](NormQArgs& a) { a.y = const_cast<void*>(a.x); });
  go("norm y on h", "overlaps", [](NormQArgs& a) { a.y = a.h; });
  go("norm codes on x", "overlaps", [](NormQArgs& a) { a.codes = at<int8_t>(0x10010); });
  go("norm codes on y", "overlaps", [](NormQArgs& a) { a.y = at<float>(0x60000), a.codes = at<int8_t>(0x60001); });
  go("norm neighbours in one buffer", nullptr,
     [](NormQArgs& a) { a.ldx = a.ldh = 200, a.h = at<float>(0x10000 + 400); });
  go("norm touching neighbours", "overlaps",
     [](NormQArgs& a) { a.ldx = a.ldh = 200, a.h = at<float>(0x10000 + 396); });
  // scales [4] and weights [100] beside rows of 400 bytes (codes: 100)
  go("norm scales on x", "overlap", [](NormQArgs& a) { a.scales = at<float>(0x10000 + 1596); });
  go("norm scales behind x", nullptr, [](NormQArgs& a) { a.scales = at<float>(0x10000 + 1600); });
  go("norm scales up to x", nullptr, [](NormQArgs& a) { a.scales = at<float>(0x10000 - 16); });
  go("norm scales into x", "overlap", [](NormQArgs& a) { a.scales = at<float>(0x10000 - 12); });
  go("norm scales on res", "overlap", [](NormQArgs& a) { a.scales = at<float>(0x20000); });
  go("norm scales on h", "overlap", [](NormQArgs& a) { a.scales = at<float>(0x30000 + 4); });
  go("norm scales on y", "overlap", [](NormQArgs& a) { a.y = at<float>(0x60000), a.scales = at<float>(0x60000 + 400); });
  go("norm scales on codes", "overlap", [](NormQArgs& a) { a.scales = at<float>(0x40000 + 396); });
  go("norm scales on w", "overlap", [](NormQArgs& a) { a.scales = at<float>(0x900 + 396); });
  go("norm scales in a gap", nullptr, [](NormQArgs& a) { a.ldx = 200, a.scales = at<float>(0x10000 + 800 - 16); });
  go("norm scales out of a gap", "overlap", [](NormQArgs& a) { a.ldx = 200, a.scales = at<float>(0x10000 + 800 - 12); });
  go("norm h on w", "overlaps", [](NormQArgs& a) { a.w = at<float>(0x30000 - 396); });
  go("norm y on w", "overlaps", [](NormQArgs& a) { a.y = at<float>(0x900); });
  go("norm codes on w", "overlaps", [](NormQArgs& a) { a.codes = at<int8_t>(0x900 + 399); });
  go("norm codes behind w", nullptr, [](NormQArgs& a) { a.codes = at<int8_t>(0x900 + 400); });
}

static void products() {
  want("w4 shape", check_w4(100, 77, 32), nullptr);
  want("w4 whole rows", check_w4(100, 77, 0), nullptr);
  want("w4 no outputs", check_w4(0, 77, 32), "shape");
  want("w4 no inputs", check_w4(7, 0, 32), "shape");
  want("w4 too large", check_w4(kMaxCols + 1, 7, 32), "shape");
  want("w4 group", check_w4(7, 100, 48), "group");
  auto go = [](const char* what, const char* part, auto&& change) {
    W4Args a{kF32, kF32, at<float>(0x10000), nullptr, at<float>(0x20000), 4, 0, 0};
    change(a);
    want(what, check(a, 100, 64), part);
  };
  go("w4", nullptr, [](W4Args&) {});
  go("w4 type", "dtype", [](W4Args& a) { a.dtype = 4; });
  go("w4 out type", "out_dtype", [](W4Args& a) { a.out_dtype = kI8; });
  go("w4 int8 without scales", "scales", [](W4Args& a) { a.dtype = kI8; });
  go("w4 int8", nullptr, [](W4Args& a) { a.dtype = kI8, a.xscales = at<float>(0x900); });
  go("w4 scales without int8", "scales", [](W4Args& a) { a.xscales = at<float>(0x900); });
  go("w4 stride", "stride", [](W4Args& a) { a.ldx = 63; });
  go("w4 out stride", "stride", [](W4Args& a) { a.ldo = 99; });
  go("w4 null", "null", [](W4Args& a) { a.out = nullptr; });
  go("w4 no rows", nullptr, [](W4Args& a) { a.rows = 0, a.x = nullptr; });
  go("w4 alignment", "aligned", [](W4Args& a) { a.out_dtype = kBF16, a.out = at<char>(0x20001); });
  go("w4 overlap", "overlaps", [](W4Args& a) { a.out = at<char>(0x10040); });
  go("w4 out on scales", "overlaps", [](W4Args& a) { a.dtype = kI8, a.xscales = at<float>(0x20000 + 1596); });
  go("w4 scales in a gap of out", nullptr, [](W4Args& a) { a.dtype = kI8, a.ldo = 104, a.xscales = at<float>(0x20000 + 400); });

  // a group of any size at or beyond the row is the row, also past what an int holds
  for (size_t group : {size_t{64}, size_t{1} << 20, (size_t{1} << 31) - 32, size_t{1} << 31, size_t{1} << 32,
                       (size_t{1} << 32) + 32, ~size_t{31}}) {
    want("w4 large group", check_w4(16, 64, group), nullptr);
    const W4Geom g = w4_geom(16, 64, group);
    is("w4 large group's inputs", g.group, 64);
    is("w4 large group's step", g.step, 128);
  }
  is("w4 group", w4_geom(16, 64, 32).group, 32);

  // the packed layout holds every code and scale once, within its bytes
  const size_t shapes[][3] = {{1, 1, 32}, {17, 1031, 32}, {33, 129, 64}, {16, 128, 128}, {100, 96, 96}, {5, 300, 0},
                              {40, 700, 256}, {3, 64, 1024}, {48, 640, 192}};
  for (auto& s : shapes) {
    const W4Geom g = w4_geom(s[0], s[1], s[2]);
    is("w4 step divides the group or the row is one", s[2] == 0 || s[2] >= s[1] || s[2] % g.step == 0, 1);
    std::set<size_t> seen;
    for (int k = 0; k < g.nc * 128; ++k) {
      int found = 0;
      for (int q = 0; q < 4; ++q)
        for (int j = 0; j < 4; ++j)
          for (int e = 0; e < 8; ++e)
            if (k / 128 * 128 + w4_k(g.step, j, q) + e == k) {
              ++found;
              seen.insert(((static_cast<size_t>(k / 128) * 4 + q) * 4 + j) * 8 + w4_nibble(e));
              // all inputs of a word, and of a matrix instruction's lane groups, share a scale
              is("w4 word within a scale", (k % 128) / g.step, w4_k(g.step, j, q) / g.step);
              is("w4 instruction within a scale", w4_k(g.step, j, q) / g.step, w4_k(g.step, j, 0) / g.step);
            }
      is("w4 places of an input", found, 1);
    }
    is("w4 nibbles", static_cast<long>(seen.size()), g.nc * 128);
    is("w4 tiles", g.nt * 16 >= g.N && (g.nt - 1) * 16 < g.N, 1);
    is("w4 scale columns", g.ns * g.step, g.nc * 128);
  }
}

// The few-row kernel's loads of a row stay in its chunk and bring each of its inputs once.
static void product_loads() {
  for (int t : {kBF16, kF16, kI8})
    for (int step : {32, 64, 128}) {
      const int n = w4_load(t, step);
      int got[128] = {};
      for (int q = 0; q < 4; ++q)
        for (int j = 0; j < 4; j += n / 8)
          for (int e = 0; e < n; ++e) {
            const int k = w4_k(step, j, q) + e;
            is("w4 load within its chunk", k < 128, 1);
            if (k < 128) ++got[k];
          }
      for (int k = 0; k < 128; ++k) is("w4 loads of an input", got[k], 1);
    }
}

static void sequences() {
  const size_t lens[] = {3, 0, 5, 9, 0};
  want("lens", check_seqs(lens, 5, 17), nullptr);
  want("lens short", check_seqs(lens, 5, 18), "sum");
  want("lens long", check_seqs(lens, 5, 16), "exceed");
  want("lens one too long", check_seqs(lens, 5, 8), "longer");
  const size_t wraps[] = {~size_t{0}, 2};
  want("lens wrap", check_seqs(wraps, 2, 1), "longer");
  want("equal", check_seqs(nullptr, 4, 12), nullptr);
  want("unequal", check_seqs(nullptr, 5, 12), "divide");
  want("none", check_seqs(nullptr, 0, 0), nullptr);
  want("rows of none", check_seqs(nullptr, 0, 3), "without");

  SeqTab t;
  int tiles = 0;
  is("rows of table", fill_seqs(t, lens, 17, 5, 0, 5, 4, &tiles), 17);
  is("tiles", tiles, 1 + 0 + 2 + 3 + 0);
  is("ragged", t.len, 0);
  is("last row", t.row[5], 17);
  for (int k = 0; k < tiles; ++k) {  // the search of the kernels: sequences whose first tile is at or before k
    int below = 0;
    for (int i = 0; i < t.n; ++i) below += t.tile[i] <= k;
    const int seq = below - 1;
    is("tile in its sequence", t.tile[seq] <= k && k < t.tile[seq + 1], 1);
    is("tile has rows", lens[seq] > static_cast<size_t>(k - t.tile[seq]) * 4, 1);
  }
  is("part of a table", fill_seqs(t, lens, 17, 5, 2, 2, 4, &tiles), 14);
  is("its tiles", tiles, 5);
  is("equal rows", fill_seqs(t, nullptr, 12, 4, 1, 3, 2, &tiles), 9);
  is("equal tiles", tiles, 6);
  const size_t none[] = {0, 0, 0};
  is("no rows", fill_seqs(t, none, 0, 3, 0, 3, 4, &tiles), 0);
  is("no tiles", tiles, 0);
}

static void mixers() {
  const size_t lens[] = {2, 2};
  auto conv = [&](const char* what, const char* part, auto&& change) {
    ConvArgs a{kF32, 1, at<float>(0x20000), at<float>(0x10000), at<float>(0x900), nullptr, at<float>(0x30000),
               lens, 2, 4, 64, 4, 0, 0};
    change(a);
    want(what, check(a), part);
  };
  conv("conv", nullptr, [](ConvArgs&) {});
  conv("conv type", "dtype", [](ConvArgs& a) { a.dtype = kI8; });
  conv("conv width", "width", [](ConvArgs& a) { a.width = 9; });
  conv("conv no width", "width", [](ConvArgs& a) { a.width = 0; });
  conv("conv stride", "stride", [](ConvArgs& a) { a.ldo = 63; });
  conv("conv lens", "sum", [](ConvArgs& a) { a.rows = 5; });
  conv("conv null", "null", [](ConvArgs& a) { a.w = nullptr; });
  conv("conv in place", "overlaps", [](ConvArgs& a) { a.out = const_cast<void*>(a.x); });
  conv("conv state on x", "state", [](ConvArgs& a) { a.state = at<float>(0x10040); });
  conv("conv state on out", "state", [](ConvArgs& a) { a.state = at<float>(0x20000 - 8); });
  conv("conv alignment", "aligned", [](ConvArgs& a) { a.state = at<float>(0x30002); });
  conv("conv no rows", nullptr, [](ConvArgs& a) { a.rows = 0, a.lens = nullptr; });
  conv("conv halves of one buffer", nullptr,
       [](ConvArgs& a) { a.ldx = a.ldo = 128, a.out = at<float>(0x10000 + 256); });

  conv("conv out on w", "overlaps", [](ConvArgs& a) { a.w = at<float>(0x20000 - 1020); });
  conv("conv out behind w", nullptr, [](ConvArgs& a) { a.w = at<float>(0x20000 - 1024); });
  conv("conv out on bias", "overlaps", [](ConvArgs& a) { a.bias = at<float>(0x20000 + 1020); });
  conv("conv state on w", "state", [](ConvArgs& a) { a.state = at<float>(0x900 + 1020); });
  conv("conv state on bias", "state", [](ConvArgs& a) { a.bias = at<float>(0x30000 + 1532); });
  conv("conv bias behind the state", nullptr, [](ConvArgs& a) { a.bias = at<float>(0x30000 + 1536); });
  conv("conv state of width 1 is none", nullptr, [](ConvArgs& a) { a.width = 1, a.state = at<float>(0x900); });
  conv("conv state in a gap", nullptr, [](ConvArgs& a) { a.ldx = 1000, a.state = at<float>(0x10000 + 256); });

  auto scan = [&](const char* what, const char* part, auto&& change) {
    ScanArgs a{};
    a.out = at<float>(0x20000), a.u = at<float>(0x10000), a.dt = at<float>(0x30000), a.B = at<float>(0x40000);
    a.C = at<float>(0x50000), a.A = at<float>(0x900), a.state = at<float>(0x60000);
    a.lens = lens, a.seqs = 2, a.rows = 4, a.D = 64, a.N = 16;
    change(a);
    want(what, check(a), part);
  };
  scan("scan", nullptr, [](ScanArgs&) {});
  scan("scan type", "dtype", [](ScanArgs& a) { a.dtype = 7; });
  scan("scan states", "states", [](ScanArgs& a) { a.N = 129; });
  scan("scan no states", "states", [](ScanArgs& a) { a.N = 0; });
  scan("scan stride", "stride", [](ScanArgs& a) { a.ldb = 15; });
  scan("scan stride of u", "stride", [](ScanArgs& a) { a.ldu = 63; });
  scan("scan lens", "exceed", [](ScanArgs& a) { a.rows = 3; });
  scan("scan null", "null", [](ScanArgs& a) { a.dt = nullptr; });
  scan("scan in place", "overlaps", [](ScanArgs& a) { a.out = const_cast<void*>(a.u); });
  scan("scan on z", "overlaps", [](ScanArgs& a) { a.z = at<float>(0x20004); });
  scan("scan state on B", "state", [](ScanArgs& a) { a.state = at<float>(0x40010); });
  scan("scan state on out", "state", [](ScanArgs& a) { a.state = at<float>(0x20010); });
  scan("scan alignment", "aligned", [](ScanArgs& a) { a.skip = at<float>(0x902); });
  scan("scan B and C in one buffer", nullptr, [](ScanArgs& a) { a.ldb = a.ldc = 32, a.C = at<float>(0x40040); });
  scan("scan out on A", "overlaps", [](ScanArgs& a) { a.A = at<float>(0x20000 + 1020); });
  scan("scan A behind out", nullptr, [](ScanArgs& a) { a.A = at<float>(0x20000 + 1024); });
  scan("scan out on skip", "overlaps", [](ScanArgs& a) { a.skip = at<float>(0x20000 - 4); });
  scan("scan out on dt_bias", "overlaps", [](ScanArgs& a) { a.dt_bias = at<float>(0x20000); });
  scan("scan state on A", "state", [](ScanArgs& a) { a.A = at<float>(0x60000 + 8188); });
  scan("scan state on skip", "state", [](ScanArgs& a) { a.skip = at<float>(0x60000); });
  scan("scan state on dt_bias", "state", [](ScanArgs& a) { a.dt_bias = at<float>(0x60000 - 252); });
  scan("scan dt_bias before the state", nullptr, [](ScanArgs& a) { a.dt_bias = at<float>(0x60000 - 256); });
  scan("scan state in a gap", nullptr, [](ScanArgs& a) { a.ldu = 10000, a.state = at<float>(0x10000 + 256 + 4); });
  scan("scan no rows", nullptr, [](ScanArgs& a) { a.rows = 0, a.lens = nullptr, a.u = nullptr; });
}

// The scan's chunks: all rows in tiles of at least one row each, and their states within the workspace.
static void plans() {
  for (size_t D : {1, 64, 100, 1111, 4096, 100000})
    for (size_t N : {1, 16, 17, 128})
      for (size_t rows : {1, 31, 97, 640, 2048, 100000}) {
        std::vector<size_t> lens = {rows, 0, rows / 2, 1, rows / 3};
        ScanArgs a{};
        a.lens = lens.data(), a.seqs = lens.size(), a.D = D, a.N = N;
        for (size_t l : lens) a.rows += l;
        const ScanPlan p = scan_plan(a, 0, 5);
        is("chunk", p.chunk >= 1, 1);
        SeqTab t;
        int tiles = 0;
        fill_seqs(t, a.lens, a.rows, a.seqs, 0, 5, p.chunk, &tiles);
        if (p.split)
          is("workspace", static_cast<size_t>(tiles) * (N + 1) * D <= kScanWsFloats, 1);
        else
          is("one piece each", tiles, 2 + (rows >= 2) + (rows >= 3));
        is("split asked for", scan_splits(a), p.split);
      }
}

// The many-row product's plan: the laid out rows and the blocks' sums within the workspace, whatever the shape.
static void products_plan() {
  for (size_t N : {1, 16, 1333, 11264, 50000, 1000000})
    for (size_t K : {1, 130, 1031, 6912, 100000, 1000000})
      for (size_t rows : {1, 16, 100, 2048, 70000})
        for (int t : {kF32, kBF16, kF16, kI8})
          for (size_t group : {size_t{32}, size_t{64}, size_t{128}, size_t{0}}) {
            const W4Geom g = w4_geom(N, K, group);
            const size_t most = w4_rows_most(t, g, rows);
            is("rows of a pass", most >= 1, 1);
            if (!w4_lays(t, g, rows)) continue;
            for (size_t r : {most < rows ? most : rows, rows % most ? rows % most : size_t{1}}) {
              const int rt = static_cast<int>((r + 15) / 16);
              const W4Plan p = w4_plan(t, g, rt);
              const size_t sums = p.ks > 1 ? static_cast<size_t>(p.ks) * rt * 16 * g.nt * 16 * 4 : 0;
              is("workspace of a product", w4_lay_bytes(t, g, rt) + sums <= kLayerWsBytes, 1);
              is("waves", p.wn * p.bk == 4 || p.wn * p.bk == 8, 1);
              is("grid", rt <= 65535 && r <= 65535 * 16, 1);
              if (p.ks > 1) is("grid of sums", r <= 65535, 1);
            }
          }
}

// The norm's plan: its threads' vectors hold the row, one fewer each would not, and the form has a kernel.
static void norm_plans() {
  for (int t : {kF32, kBF16, kF16})
    for (size_t rows : {1, 2047, 2048, 100000})
      for (size_t cols = 1; cols <= 40000; ++cols) {
        const NormPlan p = norm_plan(t, rows, cols);
        const size_t vec = 16 / dtype_size(t), held = static_cast<size_t>(p.threads) * p.vecs * vec;
        if (!p.threads) {
          is("norm of rows read twice", cols > 1024 * kNormVecsBlock * vec, 1);
          continue;
        }
        is("norm's threads", p.threads == 64 || p.threads == 256 || (p.threads == 1024 && p.vecs == kNormVecsBlock), 1);
        is("norm's vectors", p.vecs >= 1 && p.vecs <= kNormVecs, 1);
        is("norm holds the row", held >= cols, 1);
        if (p.threads < 1024) is("norm's smallest", held - static_cast<size_t>(p.threads) * vec < cols, 1);
      }
}

int main() {
  norm_plans();
  products_plan();
  plans();
  norms();
  products();
  product_loads();
  sequences();
  mixers();
  std::printf("%d unmet\n", bad);
  return bad ? 1 : 0;
}
