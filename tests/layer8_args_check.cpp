// Checks and plans of the linear attention layer's operators (csrc/mmf_layer8.hpp) on the host: prints a line for every
// expectation that does not hold and exits with their number.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <set>

#include "../matmulfreellmcpu_amd/csrc/mmf_layer8.hpp"

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

static void products() {
  want("w8 shape", check_w8(100, 77), nullptr);
  want("w8 most inputs", check_w8(1, kW8MaxK), nullptr);
  want("w8 too many inputs", check_w8(1, kW8MaxK + 1), "131071");
  is("the largest sum fits", 128l * 128l * static_cast<long>(kW8MaxK) <= 2147483647l, 1);
  want("w8 no outputs", check_w8(0, 77), "shape");
  want("w8 no inputs", check_w8(7, 0), "shape");
  want("w8 too many outputs", check_w8(kMaxCols + 1, 7), "shape");
  want("w8 most weights", check_w8(kMaxCols, 16384), nullptr);
  want("w8 too many weights", check_w8(kMaxCols, 16385), "2^34");
  auto go = [](const char* what, const char* part, auto&& change) {
    W8Args a{kF32, at<int8_t>(0x10001), at<float>(0x900), nullptr, at<float>(0x20000), 4, 0, 0};
    change(a);
    want(what, check(a, 100, 64), part);
  };
  go("w8", nullptr, [](W8Args&) {});
  go("w8 out type", "out_dtype", [](W8Args& a) { a.out_dtype = kI8; });
  go("w8 stride", "stride", [](W8Args& a) { a.ldx = 63; });
  go("w8 out stride", "stride", [](W8Args& a) { a.ldo = 99; });
  go("w8 wide stride", "stride", [](W8Args& a) { a.ldo = kMaxLd + 1; });
  go("w8 null x", "null", [](W8Args& a) { a.x = nullptr; });
  go("w8 null scales", "null", [](W8Args& a) { a.xscales = nullptr; });
  go("w8 null out", "null", [](W8Args& a) { a.out = nullptr; });
  go("w8 no rows", nullptr, [](W8Args& a) { a.rows = 0, a.x = nullptr; });
  go("w8 many rows", "rows", [](W8Args& a) { a.rows = kMaxRows + 1; });
  go("w8 out alignment", "aligned", [](W8Args& a) { a.out_dtype = kBF16, a.out = at<char>(0x20001); });
  go("w8 scale alignment", "aligned", [](W8Args& a) { a.xscales = at<float>(0x902); });
  go("w8 bias alignment", "aligned", [](W8Args& a) { a.bias = at<float>(0x902); });
  go("w8 out on x", "overlaps", [](W8Args& a) { a.out = at<char>(0x10100); });
  go("w8 out behind x", nullptr, [](W8Args& a) { a.out = at<char>(0x10104); });
  go("w8 out on scales", "overlaps", [](W8Args& a) { a.xscales = at<float>(0x20000 + 1596); });
  go("w8 scales behind out", nullptr, [](W8Args& a) { a.xscales = at<float>(0x20000 + 1600); });
  go("w8 out on bias", "overlaps", [](W8Args& a) { a.bias = at<float>(0x20000 - 396); });
  go("w8 bias before out", nullptr, [](W8Args& a) { a.bias = at<float>(0x20000 - 400); });
  // the layout holds every weight once, within its bytes, and pads to whole tiles and chunks
  const size_t shapes[][2] = {{1, 1}, {33, 129}, {64, 128}, {70, 31}};
  for (auto& s : shapes) {
    const W8Geom g = w8_geom(s[0], s[1]);
    is("w8 chunks", g.nk % 4 == 0 && g.nk * 32 >= g.K && g.nk * 32 - 128 < g.K, 1);
    std::set<size_t> seen;
    for (size_t n = 0; n < static_cast<size_t>(g.nt) * 32; ++n)
      for (size_t k = 0; k < static_cast<size_t>(g.nk) * 32; ++k) seen.insert(w8_at(g, n, k));
    is("w8 places", static_cast<long>(seen.size()), static_cast<long>(w8_code_bytes(g)));
    is("w8 last place", static_cast<long>(*seen.rbegin()), static_cast<long>(w8_code_bytes(g)) - 1);
  }
}

// Every kernel is reached, and its grid counts fewer than 2^32 threads at the largest sizes.
static void ways() {
  auto way = [](size_t rows, size_t K, size_t N) { return static_cast<long>(w8_way(w8_geom(N, K), rows)); };
  is("w8 one row", way(1, 2048, 11264), kW8Rows);
  is("w8 16 rows of large weights", way(16, 131071, kMaxCols), kW8Rows);
  is("w8 24 rows", way(24, 6912, 2560), kW8Rows);
  is("w8 40 rows of small weights", way(40, 2048, 2048), kW8Rows);
  is("w8 64 rows", way(64, 2048, 11264), kW8Tile32);
  is("w8 64 rows of many inputs", way(64, 6912, 2560), kW8Tile32x4);
  is("w8 512 rows", way(512, 6912, 2560), kW8Tile64);
  is("w8 2048 rows", way(2048, 2048, 11264), kW8Tile128);
  for (size_t rows : {size_t{65}, size_t{1000}, size_t{65535}})
    for (size_t N : {size_t{1}, size_t{129}, kMaxCols}) {
      const long w = way(rows, 4097, N);
      const size_t r = w == kW8Tile128 ? 128 : w == kW8Tile64 ? 64 : 32, n = w == kW8Tile128 ? 256 : 128;
      is("w8 grid", ((rows + r - 1) / r * ((N + n - 1) / n) + 8) * 1024 < (size_t{1} << 32), 1);
    }
}

static void blocks() {
  auto go = [](const char* what, const char* part, auto&& change) {
    BlockArgs a{kF32, kActSilu, at<float>(0x10000), at<float>(0x20000), at<float>(0x30000), at<float>(0x900), at<float>(0x1900), at<float>(0x2900),
                at<float>(0x40000), at<float>(0x50000), at<int8_t>(0x60000), at<float>(0x70000), 4, 100, 0, 0, 0, 0, 0, 0, 1.0f, 1e-6f};
    change(a);
    want(what, check(a), part);
  };
  go("block", nullptr, [](BlockArgs&) {});
  go("block type", "dtype", [](BlockArgs& a) { a.dtype = kI8; });
  go("block act", "act", [](BlockArgs& a) { a.act = 3; });
  go("block act below", "act", [](BlockArgs& a) { a.act = -1; });
  go("block act without gate", "gate", [](BlockArgs& a) { a.gate = nullptr; });
  go("block gate as it is", nullptr, [](BlockArgs& a) { a.act = kActNone; });
  go("block no gate", nullptr, [](BlockArgs& a) { a.act = kActNone, a.gate = nullptr; });
  for (size_t BlockArgs::*ld : {&BlockArgs::ldb, &BlockArgs::ldx, &BlockArgs::ldgate, &BlockArgs::ldh, &BlockArgs::ldy, &BlockArgs::ldcodes})
    go("block stride", "stride", [&](BlockArgs& a) { a.*ld = 99; });
  go("block null b", "null", [](BlockArgs& a) { a.b = nullptr; });
  go("block no rows", nullptr, [](BlockArgs& a) { a.rows = 0, a.b = a.gate = nullptr; });
  go("block many rows", "rows", [](BlockArgs& a) { a.rows = kMaxRows + 1; });
  go("block long rows", "long", [](BlockArgs& a) { a.cols = kMaxCols + 1; });
  go("block codes alone", "together", [](BlockArgs& a) { a.scales = nullptr; });
  go("block scales alone", "together", [](BlockArgs& a) { a.codes = nullptr; });
  go("block no codes", nullptr, [](BlockArgs& a) { a.codes = nullptr, a.scales = nullptr; });
  go("block nothing", "no output", [](BlockArgs& a) { a.codes = nullptr, a.scales = nullptr, a.h = a.y = nullptr; });
  go("block bare", nullptr, [](BlockArgs& a) { a.x = nullptr, a.w_post = a.w_pre = a.channels = nullptr, a.h = nullptr; });
  go("block odd address", "aligned", [](BlockArgs& a) { a.x = at<char>(0x20002); });
  go("block odd weights", "aligned", [](BlockArgs& a) { a.channels = at<float>(0x2901); });
  go("block h in place of b", nullptr, [](BlockArgs& a) { a.h = const_cast<void*>(a.b); });
  go("block h in place of x", nullptr, [](BlockArgs& a) { a.h = const_cast<void*>(a.x); });
  go("block h in place of the gate", nullptr, [](BlockArgs& a) { a.h = const_cast<void*>(a.gate); });
  go("block h shifted", "overlaps", [](BlockArgs& a) { a.h = at<float>(0x20004); });
  go("block h in place, other stride", "overlaps", [](BlockArgs& a) { a.h = const_cast<void*>(a.x), a.ldh = 101; });
  go("block y on h", "overlaps", [](BlockArgs& a) { a.y = a.h; });
  go("block y on the gate", "overlaps", [](BlockArgs& a) { a.y = at<float>(0x30004); });
  go("block codes on b", "overlaps", [](BlockArgs& a) { a.codes = at<int8_t>(0x10000 + 1599); });
  go("block codes on y", "overlaps", [](BlockArgs& a) { a.codes = at<int8_t>(0x50000); });
  go("block scales on x", "overlap", [](BlockArgs& a) { a.scales = at<float>(0x20000); });
  go("block scales on codes", "overlap", [](BlockArgs& a) { a.scales = at<float>(0x60000 + 396); });
  go("block scales on w_pre", "overlap", [](BlockArgs& a) { a.scales = at<float>(0x1900); });
  go("block h on channels", "overlaps", [](BlockArgs& a) { a.h = at<float>(0x2900); });
  for (int t : {kF32, kBF16})
    for (size_t cols = 1; cols < 70000; cols += cols < 5000 ? 1 : 97) {
      const BlockPlan p = block_plan(t, cols);
      const size_t v = 16 / dtype_size(t);
      is("block plan holds the row", !p.threads ? cols > 2 * 1024 * v : static_cast<size_t>(p.threads) * p.vecs * v >= cols, 1);
      is("block plan's waves", p.threads % 64 == 0 && p.threads <= 1024, 1);
    }
}

static DecayArgs decay() {
  DecayArgs a{};
  a.dtype = kF32;
  a.out = at<float>(0x100000), a.q = at<float>(0x200000), a.k = at<float>(0x300000), a.v = at<float>(0x400000);
  a.decay = at<float>(0x500000), a.gates = at<float>(0x600000), a.state = at<float>(0x700000);
  a.seqs = 2, a.rows = 10, a.heads = 4, a.Dk = 16, a.Dv = 32, a.scale = 0.25f;
  return a;
}
static void attention() {
  auto go = [](const char* what, const char* part, auto&& change) {
    DecayArgs a = decay();
    change(a);
    want(what, check(a), part);
  };
  go("decay", nullptr, [](DecayArgs&) {});
  go("decay type", "dtype", [](DecayArgs& a) { a.dtype = kI8; });
  go("decay no heads", "heads", [](DecayArgs& a) { a.heads = 0; });
  go("decay many heads", "heads", [](DecayArgs& a) { a.heads = kMaxHeads + 1; });
  go("decay shared", nullptr, [](DecayArgs& a) { a.q_heads = 1, a.k_heads = 2, a.v_heads = 4; });
  for (size_t DecayArgs::*h : {&DecayArgs::q_heads, &DecayArgs::k_heads, &DecayArgs::v_heads}) {
    go("decay heads that do not divide", "divide", [&](DecayArgs& a) { a.*h = 3; });
    go("decay more heads than heads", "divide", [&](DecayArgs& a) { a.*h = 8; });
  }
  go("decay Dk", "256", [](DecayArgs& a) { a.Dk = 257; });
  go("decay Dv", "256", [](DecayArgs& a) { a.Dv = 0; });
  go("decay ldq", "stride", [](DecayArgs& a) { a.ldq = 63; });
  go("decay shared ldq", nullptr, [](DecayArgs& a) { a.q_heads = 1, a.ldq = 16; });
  go("decay ldv", "stride", [](DecayArgs& a) { a.ldv = 127; });
  go("decay ldo", "stride", [](DecayArgs& a) { a.ldo = 127; });
  go("decay ldg", "stride", [](DecayArgs& a) { a.ldg = 3; });
  go("decay seqs", "divide", [](DecayArgs& a) { a.seqs = 3; });
  go("decay null", "null", [](DecayArgs& a) { a.v = nullptr; });
  go("decay bare", nullptr, [](DecayArgs& a) { a.decay = a.gates = a.state = nullptr; });
  go("decay no rows", nullptr, [](DecayArgs& a) { a.rows = 0, a.q = nullptr; });
  go("decay alignment", "aligned", [](DecayArgs& a) { a.k = at<char>(0x300002); });
  go("decay gate alignment", "aligned", [](DecayArgs& a) { a.gates = at<float>(0x600002); });
  go("decay state alignment", "aligned", [](DecayArgs& a) { a.state = at<float>(0x700002); });
  go("decay out on v", "overlaps", [](DecayArgs& a) { a.out = const_cast<void*>(a.v); });
  go("decay out on gates", "overlaps", [](DecayArgs& a) { a.gates = at<float>(0x100000); });
  go("decay out on decay", "overlaps", [](DecayArgs& a) { a.decay = at<float>(0x100010); });
  go("decay state on q", "overlaps", [](DecayArgs& a) { a.state = at<float>(0x200000 - 4); });
  go("decay state on gates", "overlaps", [](DecayArgs& a) { a.state = at<float>(0x600000 - 4); });
  go("decay state on decay", "overlaps", [](DecayArgs& a) { a.state = at<float>(0x500000); });
  go("decay state on out", "overlaps", [](DecayArgs& a) { a.state = at<float>(0x100000 + 5116); });
  go("decay one buffer", nullptr, [](DecayArgs& a) {
    a.ldq = a.ldk = a.ldv = 64 + 64 + 128;
    a.k = at<float>(0x200000 + 256), a.v = at<float>(0x200000 + 512);
  });
}

static void steps() {
  DecayArgs a{};
  const size_t ones[] = {1, 1, 1, 1}, other[] = {1, 2, 0, 1};
  a.seqs = 4;
  a.rows = 4;
  is("a row of each without lengths", row_each(a), 1);
  a.lens = ones;
  is("a row of each", row_each(a), 1);
  a.lens = other;
  is("as many rows as sequences", row_each(a), 0);
  a.lens = nullptr;
  a.rows = 8;
  is("two rows of each", row_each(a), 0);
}
static void logps() {
  auto go = [](const char* what, const char* part, auto&& change) {
    LogpArgs a{kF32, at<float>(0x10000), at<int64_t>(0x20000), at<float>(0x30000), at<float>(0x40000), at<int64_t>(0x50000), at<float>(0x60000),
               4, 100, 5, 0, 1.0f};
    change(a);
    want(what, check(a), part);
  };
  go("logp", nullptr, [](LogpArgs&) {});
  go("logp type", "dtype", [](LogpArgs& a) { a.dtype = kI8; });
  go("logp no vocabulary", "vocabulary", [](LogpArgs& a) { a.V = 0; });
  go("logp large vocabulary", "vocabulary", [](LogpArgs& a) { a.V = kMaxCols + 1; });
  go("logp top", "top", [](LogpArgs& a) { a.top = 65; });
  go("logp top of few", "top", [](LogpArgs& a) { a.V = 4; });
  for (float t : {1e-38f, 3e38f}) go("logp temperature", nullptr, [&](LogpArgs& a) { a.temperature = t; });
  for (float t : {0.0f, -1.0f, INFINITY, NAN, 1e-39f, 4e-39f}) go("logp temperature", "temperature", [&](LogpArgs& a) { a.temperature = t; });
  go("logp stride", "stride", [](LogpArgs& a) { a.ld = 99; });
  go("logp null", "null", [](LogpArgs& a) { a.x = nullptr; });
  go("logp ids alone", "together", [](LogpArgs& a) { a.logprobs = nullptr; });
  go("logp logprobs alone", "together", [](LogpArgs& a) { a.ids = nullptr; });
  go("logp top alone", "need", [](LogpArgs& a) { a.top_ids = nullptr; });
  go("logp no top", nullptr, [](LogpArgs& a) { a.top = 0; });
  go("logp nothing", "no output", [](LogpArgs& a) { a.top = 0, a.ids = nullptr, a.logprobs = a.entropy = nullptr; });
  go("logp no rows", nullptr, [](LogpArgs& a) { a.rows = 0, a.x = nullptr; });
  go("logp ids at 4 bytes", "aligned", [](LogpArgs& a) { a.ids = at<int64_t>(0x20004); });
  go("logp bf16 at 2 bytes", nullptr, [](LogpArgs& a) { a.dtype = kBF16, a.x = at<char>(0x10002); });
  go("logp entropy on logits", "overlaps", [](LogpArgs& a) { a.entropy = at<float>(0x10000 + 1596); });
  go("logp entropy behind", nullptr, [](LogpArgs& a) { a.entropy = at<float>(0x10000 + 1600); });
  go("logp entropy on ids", "overlaps", [](LogpArgs& a) { a.entropy = at<float>(0x20000 + 28); });
  go("logp entropy on logprobs", "overlaps", [](LogpArgs& a) { a.entropy = a.logprobs; });
  go("logp top ids on top", "overlaps", [](LogpArgs& a) { a.top_ids = at<int64_t>(0x60000 + 72); });
  go("logp unused top on logits", nullptr, [](LogpArgs& a) { a.top = 0, a.top_logprobs = at<float>(0x10000); });
  for (int t : {kF32, kF16})
    for (size_t rows : {1, 100, 5000})
      for (size_t V : {1, 100, 4096, 4097, 8192, 8193, 16384, 16385, 32000, 32768, 32769, 65536, 200000, 1048576}) {
        const LogpPlan p = logp_plan(t, V, rows);
        const size_t part = static_cast<size_t>(p.threads) * p.vecs * (16 / dtype_size(t));
        is("logp plan holds the row", part && part * p.segs >= V && part * (p.segs - 1) < V, 1);
        is("logp parts joined in one list", p.segs * kMaxTop <= 2048, 1);
        is("logp pass", logp_rows_most(p, kMaxTop) > 0, 1);
        is("logp workspace", logp_rows_most(p, kMaxTop) * logp_row_floats(p, kMaxTop) * 4 <= kLayerWsBytes, 1);
      }
}

int main() {
  products();
  ways();
  blocks();
  attention();
  steps();
  logps();
  return bad;
}
