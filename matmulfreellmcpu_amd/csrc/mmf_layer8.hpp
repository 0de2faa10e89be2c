// mmf_layer8.hpp -- the operators of a linear attention layer with 8-bit weights, and of what its logits say:
// arguments, checks and launch plans.
//
// Plain C++ without HIP, like mmf_layer.hpp. The kernels are in mmf_w8.hip, mmf_decay.hip, mmf_block.hip and
// mmf_logp.hip.
#pragma once

#include "mmf_layer.hpp"

namespace mmf {

inline bool ld_ok(size_t& ld, size_t cols) {
  if (!ld) ld = cols;
  return ld >= cols && ld <= kMaxLd;
}
constexpr const char* kBadLd = "a row stride is smaller than the row, or too large";
constexpr const char* kBadAlign = "a pointer is not aligned to its type";

// ---- products with 8-bit weights ----------------------------------------------------------------
// Weights laid out as matrix operands: [tile of 32 outputs][run of 32 inputs][lane 0..63][16 bytes], lane l the
// 16 inputs from 16 (l / 32) of output l % 32; both padded with zeros, inputs to whole chunks of 128.
struct W8Geom {
  int N, K, nt, nk;  // tiles of 32 outputs, runs of 32 inputs
};
constexpr size_t kW8MaxK = 131071;             // 128 * 128 * K fits 32 bits
constexpr size_t kW8MaxCodes = size_t{1} << 34;  // a thread for 16 of them: a grid has fewer than 2^32
inline const char* check_w8(size_t N, size_t K) {
  if (!N || !K || N > kMaxCols) return "invalid 8-bit weight shape";
  if (K > kW8MaxK) return "more than 131071 inputs: their sums would not fit 32 bits";
  if (N * K > kW8MaxCodes) return "more than 2^34 weights";
  return nullptr;
}
inline W8Geom w8_geom(size_t N, size_t K) {
  return {static_cast<int>(N), static_cast<int>(K), static_cast<int>((N + 31) / 32), static_cast<int>((K + 127) / 128 * 4)};
}
inline size_t w8_code_bytes(const W8Geom& g) { return static_cast<size_t>(g.nt) * g.nk * 1024; }
// Place of weight (n, k) in the layout, in bytes.
MMF_HD inline size_t w8_at(const W8Geom& g, size_t n, size_t k) {
  return ((n / 32 * g.nk + k / 32) * 64 + n % 32 + 32 * (k / 16 % 2)) * 16 + k % 16;
}

// The kernel of a call: few rows by blocks of 16 outputs, or tiles of 32 x 128 (two or four groups of waves share the
// inputs), 64 x 128 and 128 x 256 rows and outputs. Lines by measured times (us):
//   rows       24 x 6912 x 2560 7.8, tiles of 32 12.7; 40 x 2048 x 2048 5.2 and 6.6; 33 x 2048 x 11264 10.7 and 7.1
//   32, four   64 x 6912 x 2560 12.8 (two groups 14.1); 64 x 2048 x 11264 7.4 (7.2)
//   64         512 x 6912 x 2560 22.8, tiles of 32 24.9; 512 x 2048 x 11264 23.0 and 27.1; 256 x 2048 x 11264 15.3 and 15.3
//   128        2048 x 2048 x 11264 58.7, tiles of 64 67; 2048 x 2560 x 6912 48 and 55; 512 x 2048 x 11264 23.5 and 21 to 23
enum W8Way { kW8Rows, kW8Tile32x4, kW8Tile32, kW8Tile64, kW8Tile128 };
inline W8Way w8_way(const W8Geom& g, size_t rows) {
  const size_t weights = static_cast<size_t>(g.N) * g.K;
  auto tiles = [&](size_t r, size_t n) { return (rows + r - 1) / r * ((g.N + n - 1) / n); };
  if (rows <= 16 || (rows <= 32 && weights < (size_t{20} << 20)) || (rows <= 64 && weights <= (size_t{6} << 20))) return kW8Rows;
  if (tiles(128, 256) >= 256) return kW8Tile128;
  if (tiles(32, 128) > 256) return kW8Tile64;
  return g.nk >= 128 && tiles(32, 128) <= 128 ? kW8Tile32x4 : kW8Tile32;
}
constexpr size_t kW8RowsMost = 65535;  // of a launch: tiles count in 32 bits, and so does a grid's threads

struct W8Args {
  int out_dtype;
  const int8_t* x;
  const float *xscales, *bias;  // [rows]; [N] or null
  void* out;
  size_t rows, ldx, ldo;
};
inline const char* check(W8Args& a, size_t N, size_t K) {
  if (!float_type(a.out_dtype)) return "out_dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (!ld_ok(a.ldx, K) || !ld_ok(a.ldo, N)) return kBadLd;
  if (!a.rows) return nullptr;
  if (!a.x || !a.xscales || !a.out) return "null argument";
  const RowsOf x{a.x, a.ldx, K, 1}, o{a.out, a.ldo, N, dtype_size(a.out_dtype)}, s{a.xscales, 1, 1, 4}, b{a.bias, 1, 1, 4};
  for (const RowsOf& t : {o, s, b})
    if (!rows_aligned(t)) return kBadAlign;
  if (rows_overlap(x, o, a.rows) || array_overlaps(a.xscales, a.rows, o, a.rows) || array_overlaps(a.bias, N, o, a.rows))
    return "the output overlaps an input";
  return nullptr;
}

// ---- a block's output onto the residual, and the next block's norm --------------------------------
enum Act : int { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };
struct BlockArgs {
  int dtype, act;                          // of b, x, gate, h, y
  const void *b, *x, *gate;                // x, gate may be null
  const float *w_post, *w_pre, *channels;  // [cols], each may be null
  void *h, *y;                             // may be null
  int8_t* codes;                           // with scales, or both null
  float* scales;                           // [rows]
  size_t rows, cols, ldb, ldx, ldgate, ldh, ldy, ldcodes;
  float scale, eps;
};
inline const char* check(BlockArgs& a) {
  if (!float_type(a.dtype)) return "dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.act < kActNone || a.act > kActSilu) return "act must be MMF_ACT_NONE, MMF_ACT_SIGMOID or MMF_ACT_SILU";
  if (a.act != kActNone && !a.gate && a.rows) return "an activation needs a gate";
  if (a.rows > kMaxRows) return "too many rows";
  if (a.cols > kMaxCols) return "rows are too long";
  for (size_t* ld : {&a.ldb, &a.ldx, &a.ldgate, &a.ldh, &a.ldy, &a.ldcodes})
    if (!ld_ok(*ld, a.cols)) return kBadLd;
  if (!a.rows || !a.cols) return nullptr;
  if (!a.b) return "null argument";
  if (!a.codes != !a.scales) return "codes and scales go together";
  if (!a.h && !a.y && !a.codes) return "no output";
  const size_t es = dtype_size(a.dtype);
  const RowsOf b{a.b, a.ldb, a.cols, es}, x{a.x, a.ldx, a.cols, es}, g{a.gate, a.ldgate, a.cols, es},
      h{a.h, a.ldh, a.cols, es}, y{a.y, a.ldy, a.cols, es}, c{a.codes, a.ldcodes, a.cols, 1};
  for (const RowsOf& t : {b, x, g, h, y})
    if (!rows_aligned(t)) return kBadAlign;
  const float* const params[] = {a.w_post, a.w_pre, a.channels};
  for (const float* p : {a.w_post, a.w_pre, a.channels, static_cast<const float*>(a.scales)})
    if (reinterpret_cast<uintptr_t>(p) % 4) return kBadAlign;
  for (const RowsOf& in : {b, x, g})
    if (a.h && !same_rows(h, in) && rows_overlap(h, in, a.rows)) return "h overlaps an input (it may be b, x or the gate itself)";
  for (const RowsOf& in : {b, x, g, h})
    if (rows_overlap(y, in, a.rows) || rows_overlap(c, in, a.rows)) return "an output overlaps another tensor of the call";
  if (rows_overlap(y, c, a.rows)) return "an output overlaps another tensor of the call";
  for (const RowsOf& t : {b, x, g, h, y, c})
    if (array_overlaps(a.scales, a.rows, t, a.rows)) return "the scales overlap another tensor of the call";
  for (const float* p : params) {
    for (const RowsOf& out : {h, y, c})
      if (array_overlaps(p, a.cols, out, a.rows)) return "an output overlaps the weights";
    if (arrays_overlap(a.scales, a.rows, p, a.cols)) return "the scales overlap another tensor of the call";
  }
  return nullptr;
}
// The kernel of a call: `threads` a row (whole waves), each with `vecs` (1 or 2) vectors of 16 bytes in registers;
// threads 0: rows too long for that, read three times (from a cache).
struct BlockPlan {
  int threads, vecs;
};
inline BlockPlan block_plan(int dtype, size_t cols) {
  const size_t v = 16 / dtype_size(dtype), all = (cols + v - 1) / v;
  for (int vecs : {1, 2}) {
    const size_t t = ((all + vecs - 1) / vecs + 63) / 64 * 64;
    if (t <= 1024) return {static_cast<int>(t), vecs};
  }
  return {0, 0};
}

// ---- linear attention with a decay for each head --------------------------------------------------
constexpr size_t kMaxHead = 256, kMaxHeads = 1024;
struct DecayArgs {
  int dtype;                     // of q, k, v, out
  void* out;                     // [rows, heads * Dv]
  const void *q, *k, *v;         // [rows, q_heads * Dk], [rows, k_heads * Dk], [rows, v_heads * Dv]
  const float *decay, *gates;    // [heads], [rows, heads]; either may be null
  float* state;                  // [seqs, heads, Dk, Dv] or null
  const size_t* lens;
  size_t seqs, rows, heads, q_heads, k_heads, v_heads, Dk, Dv, ldo, ldq, ldk, ldv, ldg;
  float scale;
};
inline const char* check(DecayArgs& a) {
  if (!float_type(a.dtype)) return "dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (!a.heads || a.heads > kMaxHeads) return "the heads must be 1..1024";
  for (size_t* n : {&a.q_heads, &a.k_heads, &a.v_heads}) {
    if (!*n) *n = a.heads;
    if (a.heads % *n) return "the heads of q, k and v must divide the heads";
  }
  if (!a.Dk || !a.Dv || a.Dk > kMaxHead || a.Dv > kMaxHead) return "Dk and Dv must be 1..256";
  if (!ld_ok(a.ldo, a.heads * a.Dv) || !ld_ok(a.ldq, a.q_heads * a.Dk) || !ld_ok(a.ldk, a.k_heads * a.Dk) ||
      !ld_ok(a.ldv, a.v_heads * a.Dv) || !ld_ok(a.ldg, a.heads))
    return kBadLd;
  if (const char* e = check_seqs(a.lens, a.seqs, a.rows)) return e;
  if (!a.rows) return nullptr;
  if (!a.out || !a.q || !a.k || !a.v) return "null argument";
  const size_t es = dtype_size(a.dtype), held = a.seqs * a.heads * a.Dk * a.Dv;
  const RowsOf o{a.out, a.ldo, a.heads * a.Dv, es}, g{a.gates, a.ldg, a.heads, 4},
      ins[] = {{a.q, a.ldq, a.q_heads * a.Dk, es}, {a.k, a.ldk, a.k_heads * a.Dk, es}, {a.v, a.ldv, a.v_heads * a.Dv, es}, g};
  if (!rows_aligned(o)) return kBadAlign;
  for (const float* p : {a.decay, static_cast<const float*>(a.state)})
    if (reinterpret_cast<uintptr_t>(p) % 4) return kBadAlign;
  for (const RowsOf& t : ins) {
    if (!rows_aligned(t)) return kBadAlign;
    if (rows_overlap(o, t, a.rows)) return "the output overlaps an input";
    if (array_overlaps(a.state, held, t, a.rows)) return "the state overlaps another tensor of the call";
  }
  if (array_overlaps(a.state, held, o, a.rows)) return "the state overlaps another tensor of the call";
  if (array_overlaps(a.decay, a.heads, o, a.rows)) return "the output overlaps an input";
  if (arrays_overlap(a.state, held, a.decay, a.heads)) return "the state overlaps another tensor of the call";
  return nullptr;
}

// Sequences of a launch: `len` rows from row `row` on, with the state of sequence `seq`. In tiles of `step` rows (a tile is
// a block's share of a long sequence); those of more than one tile stand first, so that their tiles are numbered from 0
// and only they need slots of the workspace.
constexpr int kDecaySeqs = 192;
struct DecaySeq {
  int row, len, seq, tile;       // tile: its first
};
struct DecayTab {
  int n, step, many;             // sequences, rows of a tile, sequences of more than one tile
  int tiles, cut_tiles;          // of all sequences, and of those of more than one
  DecaySeq of[kDecaySeqs];
};
// Rows that a block multiplies at a time.
constexpr int kDecayChunk = 32;
// The table of n sequences cut into tiles of `step` rows.
inline void fill_decay(DecayTab& t, const DecaySeq* s, int n, int step) {
  t.n = n;
  t.step = step;
  int k = 0, tiles = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = 0; i < n; ++i) {
      if ((s[i].len > step) != (pass == 0)) continue;
      t.of[k] = s[i];
      t.of[k++].tile = tiles;
      tiles += (s[i].len + step - 1) / step;
    }
    if (pass == 0) {
      t.many = k;
      t.cut_tiles = tiles;
    }
  }
  t.tiles = tiles;
}
// Rows of a tile: so many that the tiles of all heads fill the chip twice, and that those of long sequences have room in
// the workspace. At least 128, as each tile writes a state and reads it three times (2048 rows of 16 heads: 39.3 us, and
// 45.2 by tiles of 64), but 64 where such tiles have a compute unit each (one head: 23.1 us, and 28.1 by 128). Nothing is
// cut where the longest sequence would be cut into two: that would be three launches for one.
inline int decay_step(const DecayArgs& a, const DecaySeq* s, int n) {
  constexpr int chunk = kDecayChunk;
  size_t chunks = 0;
  int most = 0;
  for (int i = 0; i < n; ++i) {
    chunks += (s[i].len + chunk - 1) / chunk;
    most = s[i].len > most ? s[i].len : most;
  }
  const size_t blocks = a.heads * ((a.Dv + 127) / 128), per = a.heads * (a.Dk * a.Dv + 2);
  size_t step = (chunks * blocks + 511) / 512 * chunk;
  const size_t least = chunks * blocks <= 512 ? 64 : 128;
  if (step < least) step = least;
  for (;; step *= 2) {
    if (step * 2 >= static_cast<size_t>(most)) return most;
    size_t slots = 0;
    for (int i = 0; i < n; ++i)
      if (static_cast<size_t>(s[i].len) > step) slots += (s[i].len + step - 1) / step;
    if (slots * per <= kLayerWsBytes / 4) return static_cast<int>(step);
  }
}
// Calls ones(tab) for sequences of one row and tiles(tab) for longer ones, up to kDecaySeqs at a time, until one returns a
// value other than `ok`. (Row after row is slower for two already: 32 streams of some two rows, 16 heads of 128 x 128 bf16,
// 24.9 us, and 20.8 by tiles.)
template <class R, class Ones, class Tiles>
R each_decay(const DecayArgs& a, R ok, Ones&& ones, Tiles&& tiles) {
  DecaySeq one[kDecaySeqs], many[kDecaySeqs];
  int n1 = 0, nm = 0, row = 0;
  DecayTab t;
  R r = ok;
  auto flush = [&](bool of_ones) {
    if (of_ones ? n1 : nm) {
      if (of_ones)
        fill_decay(t, one, n1, 1);
      else
        fill_decay(t, many, nm, decay_step(a, many, nm));
      r = of_ones ? ones(t) : tiles(t);
    }
    (of_ones ? n1 : nm) = 0;
  };
  for (size_t i = 0; i < a.seqs && r == ok; ++i) {
    const int len = static_cast<int>(a.lens ? a.lens[i] : a.rows / a.seqs);
    if (!len) continue;
    (len == 1 ? one[n1++] : many[nm++]) = {row, len, static_cast<int>(i), 0};
    row += len;
    if ((len == 1 ? n1 : nm) == kDecaySeqs) flush(len == 1);
  }
  if (r == ok) flush(true);
  if (r == ok) flush(false);
  return r;
}
// Whether all sequences have one row: a step of as many streams, which takes no table.
inline bool row_each(const DecayArgs& a) {
  if (a.rows != a.seqs) return false;
  for (size_t i = 0; a.lens && i < a.seqs; ++i)
    if (a.lens[i] != 1) return false;
  return true;
}
// Whether a call needs the workspace.
inline bool decay_splits(const DecayArgs& a) {
  if (row_each(a)) return false;
  return each_decay(a, 0, [](const DecayTab&) { return 0; }, [](const DecayTab& t) { return t.many ? 1 : 0; }) != 0;
}

// ---- log probabilities of tokens ------------------------------------------------------------------
constexpr size_t kMaxTop = 64;
constexpr float kMinTemperature = 1e-38f;  // 2 log2(e) over it is finite
struct LogpArgs {
  int dtype;
  const void* x;                     // [rows, V]
  const int64_t* ids;                // [rows]; with logprobs, or both null
  float *logprobs, *entropy;         // [rows], may be null
  int64_t* top_ids;                  // [rows, top]
  float* top_logprobs;               // [rows, top]
  size_t rows, V, top, ld;
  float temperature;
};
inline const char* check(LogpArgs& a) {
  if (!float_type(a.dtype)) return "dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (!a.V || a.V > kMaxCols) return "the vocabulary must be 1..1048576";
  if (a.top > kMaxTop || a.top > a.V) return "top must be 0..64 and no more than the vocabulary";
  if (!(a.temperature >= kMinTemperature) || !(a.temperature < 3.4e38f)) return "the temperature must be positive and finite, 1e-38 or more";
  if (!ld_ok(a.ld, a.V)) return kBadLd;
  if (!a.rows) return nullptr;
  if (!a.x) return "null argument";
  if (!a.ids != !a.logprobs) return "ids and logprobs go together";
  if (!a.top) a.top_ids = nullptr, a.top_logprobs = nullptr;
  if (a.top && (!a.top_ids || !a.top_logprobs)) return "top alternatives need top_ids and top_logprobs";
  if (!a.logprobs && !a.entropy && !a.top) return "no output";
  const RowsOf x{a.x, a.ld, a.V, dtype_size(a.dtype)};
  if (!rows_aligned(x)) return kBadAlign;
  const struct {
    const void* p;
    size_t n, esize;
    bool written;
  } arrays[] = {{a.ids, a.rows, 8, false}, {a.logprobs, a.rows, 4, true}, {a.entropy, a.rows, 4, true},
                {a.top_ids, a.rows * a.top, 8, true}, {a.top_logprobs, a.rows * a.top, 4, true}};
  for (const auto& t : arrays) {
    if (reinterpret_cast<uintptr_t>(t.p) % t.esize) return kBadAlign;
    if (t.written && bytes_overlap(t.p, t.n * t.esize, x, a.rows)) return "an output overlaps another tensor of the call";
    for (const auto& u : arrays)
      if (&u != &t && t.written && bytes_overlap(t.p, t.n * t.esize, RowsOf{u.p, u.n, u.n, u.esize}, 1))
        return "an output overlaps another tensor of the call";
  }
  return nullptr;
}
// A row is cut into `segs` parts of at most kLogpPart logits, for blocks of `threads` threads, which hold `vecs` (1, 2, 4
// or 8) vectors of 16 bytes each in registers. Many rows take small blocks, so that several rows are at work on a
// compute unit; few rows large ones, so that each is soon done.
constexpr size_t kLogpPart = 32768;
struct LogpPlan {
  int threads, vecs, segs;
};
inline LogpPlan logp_plan(int dtype, size_t V, size_t rows) {
  const size_t v = 16 / dtype_size(dtype), part = V < kLogpPart ? V : kLogpPart, all = (part + v - 1) / v;
  const int segs = static_cast<int>((V + kLogpPart - 1) / kLogpPart);
  for (size_t threads : {size_t{256}, size_t{512}, size_t{1024}}) {
    if (rows * segs < 256 && threads < 1024) continue;
    for (size_t vecs : {1, 2, 4, 8})
      if (all <= threads * vecs && threads * vecs * v <= kLogpPart && (segs == 1 || threads * vecs * v == kLogpPart))
        return {static_cast<int>(threads), static_cast<int>(vecs), segs};
  }
  return {0, 0, 0};
}
// Workspace of a row in several parts: for each its maximum, sum, weighted sum, and top values with their indices.
inline size_t logp_row_floats(const LogpPlan& p, size_t top) { return p.segs > 1 ? p.segs * (4 + 2 * top) : 0; }
inline size_t logp_rows_most(const LogpPlan& p, size_t top) {  // of a pass
  const size_t n = logp_row_floats(p, top);
  return n ? kLayerWsBytes / 4 / n : kMaxRows;
}

}  // namespace mmf
