// mmf_layer.hpp -- the operators of a recurrent low-bit layer: arguments, checks and launch plans.
//
// Plain C++ without HIP, so that the checks and the plans also compile, and are tested, on a host
// without a device. The kernels are in mmf_normq.hip, mmf_w4.hip, mmf_conv.hip and mmf_scan.hip.
// A row tensor is `rows` rows of `cols` elements, ld elements apart (ld >= cols), at any address
// that its element type is aligned at.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

#ifdef __HIPCC__
#define MMF_HD __host__ __device__
#else
#define MMF_HD
#endif

namespace mmf {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2, kI8 = 3 };

inline size_t dtype_size(int t) { return t == kF32 ? 4 : t == kI8 ? 1 : 2; }
inline bool float_type(int t) { return t == kF32 || t == kBF16 || t == kF16; }

constexpr size_t kMaxRows = size_t{1} << 24;  // of one call, as mmf_bitlinear
constexpr size_t kMaxCols = size_t{1} << 20;  // channels, columns
constexpr size_t kMaxLd = size_t{1} << 31;

// A row tensor's memory.
struct RowsOf {
  const void* p;
  size_t ld, cols, esize;
};

inline bool rows_aligned(const RowsOf& a) { return reinterpret_cast<uintptr_t>(a.p) % a.esize == 0; }

// Whether the bytes from p on share one with a row tensor of `rows` rows: p may stand between two of its rows.
inline bool bytes_overlap(const void* p, size_t bytes, const RowsOf& t, size_t rows) {
  if (!rows || !p || !t.p || !bytes || !t.cols) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(t.p);
  const size_t step = t.ld * t.esize, row = t.cols * t.esize;
  if (a + bytes <= b || a >= b + (rows - 1) * step + row) return false;
  if (a <= b) return true;
  const size_t in = (a - b) % step;  // of the row that starts at or before p; a later one follows if p is past its end
  return in < row || in + bytes > step;
}
inline bool array_overlaps(const void* p, size_t n, const RowsOf& t, size_t rows) { return bytes_overlap(p, n * 4, t, rows); }
// Whether two row tensors of `rows` rows share a byte. Tensors with the same distance from row to row do if their
// columns do; others are compared row by row, where their whole ranges meet.
inline bool rows_overlap(const RowsOf& a, const RowsOf& b, size_t rows) {
  if (!rows || !a.p || !b.p || !a.cols || !b.cols) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  const size_t step = a.ld * a.esize, row = a.cols * a.esize;
  const uintptr_t ea = pa + (rows - 1) * step + row, eb = pb + ((rows - 1) * b.ld + b.cols) * b.esize;
  if (ea <= pb || eb <= pa) return false;
  if (step == b.ld * b.esize) {
    const size_t d = pb >= pa ? (pb - pa) % step : (step - (pa - pb) % step) % step;
    return d < row || d + b.cols * b.esize > step;
  }
  for (size_t r = 0; r < rows; ++r)
    if (bytes_overlap(static_cast<const char*>(a.p) + r * step, row, b, rows)) return true;
  return false;
}
inline bool arrays_overlap(const void* p, size_t n, const void* q, size_t m) {
  return array_overlaps(p, n, RowsOf{q, m, m, 4}, 1);
}
inline bool same_rows(const RowsOf& a, const RowsOf& b) { return a.p == b.p && a.ld == b.ld && a.esize == b.esize; }

// ---- residual addition, RMS norm and int8 codes ------------------------------------------------
struct NormQArgs {
  int dtype;             // of x, res, h, y
  const void *x, *res;   // res may be null
  const float* w;        // [cols]
  void *h, *y;           // may be null
  int8_t* codes;
  float* scales;         // [rows]
  size_t rows, cols, ldx, ldres, ldh, ldy, ldcodes;
  float eps;
};

// The reason why a call is refused, or null. A zero ld means cols.
inline const char* check(NormQArgs& a) {
  if (!float_type(a.dtype)) return "dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (a.cols > kMaxCols) return "rows are too long";
  for (size_t* ld : {&a.ldx, &a.ldres, &a.ldh, &a.ldy, &a.ldcodes}) {
    if (!*ld) *ld = a.cols;
    if (*ld < a.cols || *ld > kMaxLd) return "a row stride is smaller than the row, or too large";
  }
  if (!a.rows || !a.cols) return nullptr;
  if (!a.x || !a.w || !a.codes || !a.scales) return "null argument";
  const size_t es = dtype_size(a.dtype);
  const RowsOf x{a.x, a.ldx, a.cols, es}, r{a.res, a.ldres, a.cols, es}, h{a.h, a.ldh, a.cols, es},
      y{a.y, a.ldy, a.cols, es}, c{a.codes, a.ldcodes, a.cols, 1}, s{a.scales, 1, 1, 4}, w{a.w, a.cols, a.cols, 4};
  for (const RowsOf& t : {x, r, h, y, s, w})
    if (!rows_aligned(t)) return "a pointer is not aligned to its type";
  for (const RowsOf& in : {x, r})
    if (a.h && !same_rows(h, in) && rows_overlap(h, in, a.rows)) return "h overlaps an input (it may be x or res itself)";
  for (const RowsOf& in : {x, r, h})
    if (rows_overlap(y, in, a.rows) || rows_overlap(c, in, a.rows)) return "an output overlaps another tensor of the call";
  if (rows_overlap(y, c, a.rows)) return "an output overlaps another tensor of the call";
  for (const RowsOf& t : {x, r, h, y, c})
    if (array_overlaps(a.scales, a.rows, t, a.rows)) return "the scales overlap another tensor of the call";
  for (const RowsOf& out : {h, y, c})
    if (array_overlaps(a.w, a.cols, out, a.rows)) return "an output overlaps the weights";
  if (arrays_overlap(a.scales, a.rows, a.w, a.cols)) return "the scales overlap another tensor of the call";
  return nullptr;
}

// The kernel of a call: `threads` a row, each with `vecs` vectors of 16 bytes in registers, so that the row is read
// once (threads * vecs vectors hold it), or threads 0: rows too long for that, read twice. A wave a row where
// that fills the chip or a wave's one vector a lane is all it needs; else a block.
struct NormPlan {
  int threads, vecs;
};
constexpr int kNormVecs = 8, kNormVecsBlock = 4;  // the most of a wave or 256 threads, and what 1024 threads have
inline NormPlan norm_plan(int dtype, size_t rows, size_t cols) {
  const size_t v = 16 / dtype_size(dtype), all = (cols + v - 1) / v;
  auto of = [&](size_t threads) {
    return NormPlan{static_cast<int>(threads), static_cast<int>((all + threads - 1) / threads)};
  };
  if (all <= 64 || (all <= 64 * kNormVecs && rows >= 2048)) return of(64);
  if (all <= 256 * kNormVecs) return of(256);
  if (all <= 1024 * kNormVecsBlock) return {1024, kNormVecsBlock};
  return {0, 0};
}

// ---- products with 4-bit weights ----------------------------------------------------------------
// Weights laid out for the kernels. Outputs go in tiles of 16 and inputs in chunks of 128, padded:
//   codes [ntile][chunk][lane 0..63][word 0..3]: lane l holds output 16 ntile + l % 16, and word j
//     the 8 inputs from 128 chunk + w4_k(step, j, l / 16). Element e of a word is its nibble w4_nibble(e).
//   scales [ntile][w4_subs * nchunk][16]: the fp16 scale in the low half, the zero point above it.
// step is the kernel's scale granularity, 32, 64 or 128 inputs: the largest that divides the group
// (of rows that are one group: 128).
struct W4Geom {
  int N, K, group, step, nt, nc, ns;  // inputs of a scale (at most K), tiles of 16 outputs, chunks of 128 inputs, scales a tile row
};
inline W4Geom w4_geom(size_t N, size_t K, size_t group) {
  W4Geom g;
  g.N = static_cast<int>(N);
  g.K = static_cast<int>(K);
  g.group = static_cast<int>(group && group < K ? group : K);
  g.step = !group || group >= K || group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32;
  g.nt = static_cast<int>((N + 15) / 16);
  g.nc = static_cast<int>((K + 127) / 128);
  g.ns = g.nc * (128 / g.step);
  return g;
}
// First input (within its chunk) of word j of a lane of lane group q = lane / 16. With scales every 32
// inputs a matrix instruction's 32 inputs are neighbours; otherwise each lane's 16 of a half chunk are.
MMF_HD inline constexpr int w4_k(int step, int j, int q) {
  return step == 32 ? 32 * j + 8 * q : 64 * (j >> 1) + 16 * q + 8 * (j & 1);
}
// Neighbouring inputs that a lane of the few-row kernel loads of a row at once, from w4_k on: a word's 8, or of
// int8 rows the 16 of two words where these are neighbours. (No load goes past its chunk: a whole last chunk ends
// with the row, and the last row's with the caller's memory.)
MMF_HD inline constexpr int w4_load(int dtype, int step) { return dtype == kI8 && step != 32 ? 16 : 8; }
// Nibble of element e (0..7) of a word: neighbours 2p and 2p + 1 are nibbles p and p + 4, the same bits
// of the word's two halves, so that one mask makes a pair of 16-bit floats of them.
MMF_HD inline constexpr int w4_nibble(int e) { return 4 * (e & 1) + (e >> 1); }
MMF_HD inline size_t w4_code_bytes(const W4Geom& g) { return static_cast<size_t>(g.nt) * g.nc * 1024; }
MMF_HD inline size_t w4_scale_bytes(const W4Geom& g) { return static_cast<size_t>(g.nt) * g.ns * 64; }

inline const char* check_w4(size_t N, size_t K, size_t group) {
  if (!N || !K || N > kMaxCols || K > kMaxCols) return "invalid 4-bit weight shape";
  if (group % 32) return "the group must be a multiple of 32 inputs, or 0 for whole rows";
  return nullptr;
}

// Many rows are laid out as matrix operands first (mmf_w4.hip): bytes of 16 rows' fragments (fp32: two fp16
// parts), and with a number for each row and scale (fp32); rows of a pass, so that these fit the workspace.
constexpr size_t kLayerWsBytes = size_t{128} << 20;
inline size_t w4_frag_bytes(int dtype, const W4Geom& g) {
  return static_cast<size_t>(g.nc) * 128 * 16 * (dtype == kF32 ? 4 : dtype == kI8 ? 1 : 2);
}
MMF_HD inline constexpr bool w4_numbers(int dtype) { return dtype == kF32; }
inline size_t w4_lay_bytes(int dtype, const W4Geom& g, int row_tiles) {  // fragments and numbers
  return row_tiles * (w4_frag_bytes(dtype, g) + (w4_numbers(dtype) ? static_cast<size_t>(g.ns) * 64 : 0));
}
constexpr int kW4TileRows = 64;  // of a wave

// How the many-row kernel's waves stand (wn over 64 outputs each, bk over the inputs; 4 or 8 in all, of
// kW4TileRows rows) and over how many blocks a tile's inputs are split.
struct W4Plan {
  int wn, bk, ks;
};
// The plan of the least time by this count: a chunk of inputs of 64 x 64 outputs takes a SIMD `unit` us (fp32 2.2,
// 16-bit 1.25, int8 0.9 with a scale for 128 inputs; more scalings with more scales), 1.3 times that where a compute unit
// has fewer than 8 waves to overlap, and up to 1.3 times where fewer outputs share the rows' operands; the
// fullest compute unit counts. Split inputs cost a launch and the partial sums, written and read at 4 TB/s.
// Measured (us): fp32 2048 x 6912 x 2560 232 as {4, 1, 1} and 195 as {4, 1, 3}; 512 x 6912 x 2560 149 and 80 as
// {2, 4, 1}; bf16 2048 x 2048 x 2048 44 and 39 as {4, 2, 1}; fp32 2048 x 2048 x 11264 201, as {4, 2, 1} 224.
inline W4Plan w4_pick(int dtype, const W4Geom& g, int row_tiles) {
  const double unit = (dtype == kF32 ? 2.2 : dtype == kI8 ? 0.9 : 1.25) * (g.step == 32 ? 1.8 : g.step == 64 ? 1.2 : 1.0);
  const int rows = (row_tiles + kW4TileRows / 16 - 1) / (kW4TileRows / 16);
  const double sums = row_tiles * 16.0 * g.nt * 16.0 * 4 * 2 / 4e6;  // us of one split's
  const struct {
    int wn, bk;
    double share;
  } forms[] = {{4, 1, 1.0}, {4, 2, 1.0}, {2, 2, 1.15}, {2, 4, 1.3}};
  W4Plan best{4, 1, 1};
  double least = 0;
  for (const auto& f : forms)
    for (int ks = 1; ks <= 8 && (ks == 1 || ks * f.bk <= g.nc); ++ks) {
      const double blocks = static_cast<double>((g.nt + f.wn * 4 - 1) / (f.wn * 4)) * rows * ks;
      const double most = static_cast<double>(static_cast<size_t>((blocks + 255) / 256));  // blocks of a compute unit
      const int chunks = (g.nc + f.bk * ks - 1) / (f.bk * ks), waves = f.wn * f.bk;
      const double t = most * chunks * (waves / 4.0) * unit * f.share * (most * waves < 8 ? 1.3 : 1.0) + (ks > 1 ? 4 + ks * sums : 0);
      if (least == 0 || t < least) {
        least = t;
        best = {f.wn, f.bk, ks};
      }
    }
  return best;
}
// The same, with no more splits than the workspace holds the sums of beside the laid out rows.
inline W4Plan w4_plan(int dtype, const W4Geom& g, int row_tiles) {
  W4Plan p = w4_pick(dtype, g, row_tiles);
  const size_t one = static_cast<size_t>(row_tiles) * g.nt * 1024;  // bytes of one split's sums
  const size_t room = kLayerWsBytes - w4_lay_bytes(dtype, g, row_tiles);
  while (p.ks > 1 && p.ks * one > room) --p.ks;
  return p;
}
// The kernel of a call: of few rows, as they are or (fp32) laid out, or by tiles of many, which are laid out.
// Lines by the products of a call, measured (us): fp32 rows laid out from 0.102 G on (24 x 2048 x 2048 7.3 as they
// are, 8.4 laid out; 16 x 2560 x 2560 8.5 and 7.3; 10 x 6912 x 2560 15.1 and 10.3; 128 x 2048 x 2048 23.8 and 11.1), by
// tiles from 1.6 G on (64 x 6912 x 2560 19.3 laid out, 24.6 by tiles; 128 x 2048 x 11264 38.8 and 29.0). Others by
// tiles from 2.5 G on (bf16 128 x 6912 x 2560 22.6 by few rows' kernel, 24.5 by tiles; 128 x 2048 x 11264 27.4 and
// 21.3).
enum W4Way { kRowsAsIs, kLaidRows, kTiles };
inline W4Way w4_way(int dtype, const W4Geom& g, size_t rows) {
  const double work = static_cast<double>(rows) * g.K * g.N;
  if (rows > 16 && work > (dtype == kF32 ? 1.6e9 : 2.5e9)) return kTiles;
  return dtype == kF32 && rows > 5 && work > 0.102e9 ? kLaidRows : kRowsAsIs;
}
inline bool w4_lays(int dtype, const W4Geom& g, size_t rows) { return w4_way(dtype, g, rows) != kRowsAsIs; }
inline size_t w4_rows_most(int dtype, const W4Geom& g, size_t rows) {
  if (!w4_lays(dtype, g, rows)) return 65535 * 5;  // the grid's second dimension, in tiles of 5 rows or more
  size_t tiles = kLayerWsBytes / w4_lay_bytes(dtype, g, 1);
  if (tiles > 8) tiles = tiles / 8 * 8;
  return 16 * (tiles < 4095 ? tiles : 4095);  // k_w4_sum has a block a row in that dimension
}

struct W4Args {
  int dtype, out_dtype;
  const void* x;
  const float* xscales;  // MMF_I8: a scale per row
  void* out;
  size_t rows, ldx, ldo;
};
inline const char* check(W4Args& a, size_t N, size_t K) {
  if (!float_type(a.dtype) && a.dtype != kI8) return "dtype must be MMF_F32, MMF_BF16, MMF_F16 or MMF_I8";
  if (!float_type(a.out_dtype)) return "out_dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (!a.ldx) a.ldx = K;
  if (!a.ldo) a.ldo = N;
  if (a.ldx < K || a.ldo < N || a.ldx > kMaxLd || a.ldo > kMaxLd)
    return "a row stride is smaller than the row, or too large";
  if (!a.rows) return nullptr;
  if (!a.x || !a.out) return "null argument";
  if ((a.dtype == kI8) != (a.xscales != nullptr)) return "int8 rows need their scales, and other rows have none";
  const RowsOf x{a.x, a.ldx, K, dtype_size(a.dtype)}, o{a.out, a.ldo, N, dtype_size(a.out_dtype)},
      s{a.xscales, 1, 1, 4};
  if (!rows_aligned(x) || !rows_aligned(o) || !rows_aligned(s)) return "a pointer is not aligned to its type";
  if (rows_overlap(x, o, a.rows) || array_overlaps(a.xscales, a.rows, o, a.rows)) return "the output overlaps an input";
  return nullptr;
}

// ---- packed sequences ---------------------------------------------------------------------------
// Rows of several sequences, one after the other. A launch takes up to kSeqs sequences, whose first
// rows and first tiles travel as a kernel argument; sequences of one length need no table.
constexpr int kSeqs = 240;
struct SeqTab {
  int n;                  // sequences of this launch
  int len, tiles;         // of each, where all are alike (len > 0)
  int row[kSeqs + 1];     // else: first row of each, from the launch's first
  int tile[kSeqs + 1];    // first tile of each
};

inline const char* check_seqs(const size_t* lens, size_t seqs, size_t rows) {
  if (seqs > kMaxRows) return "too many sequences";
  if (!seqs) return rows ? "rows without a sequence" : nullptr;
  if (!lens) return rows % seqs ? "the rows do not divide into the sequences" : nullptr;
  size_t sum = 0;
  for (size_t i = 0; i < seqs; ++i) {
    if (lens[i] > rows) return "a sequence is longer than the rows";
    sum += lens[i];
    if (sum > rows) return "the sequences' lengths exceed the rows";
  }
  return sum == rows ? nullptr : "the sequences' lengths do not sum to the rows";
}

// Whether sequences [first, first + n) have one row each: a token of each.
inline bool one_row_each(const size_t* lens, size_t rows, size_t seqs, size_t first, int n) {
  if (!lens) return rows == seqs;
  for (int i = 0; i < n; ++i)
    if (lens[first + i] != 1) return false;
  return true;
}

// The table of sequences [first, first + n) with tiles of `step` rows; returns its rows, and tiles
// in *ntiles.
inline size_t fill_seqs(SeqTab& t, const size_t* lens, size_t rows, size_t seqs, size_t first, int n, int step,
                        int* ntiles) {
  t.n = n;
  const size_t l0 = lens ? lens[first] : rows / seqs;
  bool alike = true;
  for (int i = 1; lens && i < n; ++i) alike = alike && lens[first + i] == l0;
  t.len = alike ? static_cast<int>(l0) : 0;
  t.tiles = static_cast<int>((l0 + step - 1) / step);
  if (alike) {
    *ntiles = n * t.tiles;
    return n * l0;
  }
  int r = 0, k = 0;
  for (int i = 0; i < n; ++i) {
    t.row[i] = r;
    t.tile[i] = k;
    r += static_cast<int>(lens[first + i]);
    k += static_cast<int>((lens[first + i] + step - 1) / step);
  }
  t.row[n] = r;
  t.tile[n] = k;
  *ntiles = k;
  return r;
}

// ---- short causal convolution -------------------------------------------------------------------
constexpr size_t kMaxWidth = 8;
struct ConvArgs {
  int dtype, silu;
  void* out;
  const void* x;
  const float *w, *bias;  // [D, width], [D] or null
  float* state;           // [seqs, width - 1, D] or null
  const size_t* lens;
  size_t seqs, rows, D, width, ldx, ldo;
};
inline const char* check(ConvArgs& a) {
  if (!float_type(a.dtype)) return "dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (a.D > kMaxCols) return "too many channels";
  if (!a.width || a.width > kMaxWidth) return "the width must be 1..8";
  if (!a.ldx) a.ldx = a.D;
  if (!a.ldo) a.ldo = a.D;
  if (a.ldx < a.D || a.ldo < a.D || a.ldx > kMaxLd || a.ldo > kMaxLd)
    return "a row stride is smaller than the row, or too large";
  if (const char* e = check_seqs(a.lens, a.seqs, a.rows)) return e;
  if (!a.rows || !a.D) return nullptr;
  if (!a.out || !a.x || !a.w) return "null argument";
  const size_t es = dtype_size(a.dtype), held = (a.width - 1) * a.D;
  const RowsOf x{a.x, a.ldx, a.D, es}, o{a.out, a.ldo, a.D, es}, w{a.w, 1, 1, 4}, b{a.bias, 1, 1, 4},
      s{a.state, 1, 1, 4};
  for (const RowsOf& t : {x, o, w, b, s})
    if (!rows_aligned(t)) return "a pointer is not aligned to its type";
  if (rows_overlap(x, o, a.rows)) return "the output overlaps the input";
  const size_t all = a.seqs * held;
  for (const RowsOf& t : {x, o})
    if (array_overlaps(a.state, all, t, a.rows)) return "the state overlaps another tensor of the call";
  const struct {
    const float* p;
    size_t n;
  } params[] = {{a.w, a.D * a.width}, {a.bias, a.D}};
  for (const auto& p : params) {
    if (array_overlaps(p.p, p.n, o, a.rows)) return "the output overlaps the weights or the bias";
    if (arrays_overlap(a.state, all, p.p, p.n)) return "the state overlaps another tensor of the call";
  }
  return nullptr;
}

// ---- selective state space scan -----------------------------------------------------------------
constexpr size_t kMaxStates = 128;
struct ScanArgs {
  int dtype, softplus;
  void* out;
  const void *u, *dt, *B, *C, *z;       // z may be null
  const float *A, *skip, *dt_bias;      // [D, N], [D] or null, [D] or null
  float* state;                         // [seqs, N, D] or null
  const size_t* lens;
  size_t seqs, rows, D, N, ldo, ldu, lddt, ldb, ldc, ldz;
};
inline const char* check(ScanArgs& a) {
  if (!float_type(a.dtype)) return "dtype must be MMF_F32, MMF_BF16 or MMF_F16";
  if (a.rows > kMaxRows) return "too many rows";
  if (a.D > kMaxCols) return "too many channels";
  if (!a.N || a.N > kMaxStates) return "the states per channel must be 1..128";
  for (size_t* ld : {&a.ldo, &a.ldu, &a.lddt, &a.ldz}) {
    if (!*ld) *ld = a.D;
    if (*ld < a.D || *ld > kMaxLd) return "a row stride is smaller than the row, or too large";
  }
  for (size_t* ld : {&a.ldb, &a.ldc}) {
    if (!*ld) *ld = a.N;
    if (*ld < a.N || *ld > kMaxLd) return "a row stride is smaller than the row, or too large";
  }
  if (const char* e = check_seqs(a.lens, a.seqs, a.rows)) return e;
  if (!a.rows || !a.D) return nullptr;
  if (!a.out || !a.u || !a.dt || !a.A || !a.B || !a.C) return "null argument";
  const size_t es = dtype_size(a.dtype);
  const RowsOf o{a.out, a.ldo, a.D, es};
  const RowsOf ins[] = {{a.u, a.ldu, a.D, es}, {a.dt, a.lddt, a.D, es}, {a.B, a.ldb, a.N, es}, {a.C, a.ldc, a.N, es},
                        {a.z, a.ldz, a.D, es}};
  const size_t held = a.seqs * a.N * a.D;
  if (!rows_aligned(o)) return "a pointer is not aligned to its type";
  for (const RowsOf& t : ins) {
    if (!rows_aligned(t)) return "a pointer is not aligned to its type";
    if (rows_overlap(o, t, a.rows)) return "the output overlaps an input";
    if (array_overlaps(a.state, held, t, a.rows)) return "the state overlaps another tensor of the call";
  }
  for (const float* p : {a.A, a.skip, a.dt_bias, static_cast<const float*>(a.state)})
    if (reinterpret_cast<uintptr_t>(p) % 4) return "a pointer is not aligned to its type";
  if (array_overlaps(a.state, held, o, a.rows)) return "the state overlaps another tensor of the call";
  const struct {
    const float* p;
    size_t n;
  } params[] = {{a.A, a.D * a.N}, {a.skip, a.D}, {a.dt_bias, a.D}};
  for (const auto& p : params) {
    if (array_overlaps(p.p, p.n, o, a.rows)) return "the output overlaps an input";
    if (arrays_overlap(a.state, held, p.p, p.n)) return "the state overlaps another tensor of the call";
  }
  return nullptr;
}

// How the scan of sequences [first, first + n) is cut: into chunks of `chunk` rows, with two passes
// (split), or in one piece each.
struct ScanPlan {
  bool split;
  int chunk;
};
constexpr size_t kScanWsFloats = size_t{4} << 20;  // of the workspace: the chunks' states and steps: (N + 1) D each
inline ScanPlan scan_plan(const ScanArgs& a, size_t first, int n) {
  size_t most = 0, rows = 0;
  for (int i = 0; i < n; ++i) {
    const size_t l = a.lens ? a.lens[first + i] : a.rows / a.seqs;
    most = l > most ? l : most;
    rows += l;
  }
  const ScanPlan whole{false, static_cast<int>(most ? most : 1)};
  const size_t waves = (a.D + 63) / 64 * ((a.N + 15) / 16);  // of a chunk
  size_t chunk = (rows * waves / 2048 + 31) / 32 * 32;       // fills the chip's 1024 SIMDs twice
  if (chunk < 32) chunk = 32;
  // within the workspace: at most rows / chunk + n chunks
  const size_t per = (a.N + 1) * a.D;
  while (chunk < most && (rows / chunk + n) * per > kScanWsFloats) chunk *= 2;
  if (chunk * 3 > most || (rows / chunk + n) * per > kScanWsFloats) return whole;
  return {true, static_cast<int>(chunk)};
}
// Whether any part of a call needs the workspace.
inline bool scan_splits(const ScanArgs& a) {
  for (size_t q = 0; q < a.seqs; q += kSeqs)
    if (scan_plan(a, q, static_cast<int>(a.seqs - q < kSeqs ? a.seqs - q : kSeqs)).split) return true;
  return false;
}

}  // namespace mmf
