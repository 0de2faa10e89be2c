// mmf_decay.hip -- linear attention with a decay for each head, its state carried between calls.
//
// Per head: S = exp(a) S + k v^T, out = scale q^T S, with a = decay[head] + gates[row, head] the log decay of a row. Over a
// chunk of rows, with G_i the sum of its log decays up to row i and S the state before it,
//   out_i = scale (exp(G_i) q_i^T S + sum_{j <= i} exp(G_i - G_j) (q_i . k_j) v_j)
//   S'    = exp(G) S + sum_j exp(G - G_j) k_j v_j^T
// which are matrix products. G is summed in 64 bits and in powers of two: what counts are differences of long sums.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The log decay of a row in powers of two. 2^-300 times any fp32 number is 0, as 2^-infinity is, and leaves the sums
// that it stands in their digits.
constexpr double kForgets = -300.0;
__device__ __forceinline__ double log2_step(double a) {
  a *= 1.4426950408889634;
  return a < kForgets ? kForgets : a;
}

// The decay over a tile, part * 2^power: it may be outside fp32's range where the states before and after it are not.
struct Keep {
  float part, power;
};
__device__ __forceinline__ Keep keep_of(double log2_total) {
  if (log2_total < kForgets) return {0.0f, 0.0f};
  const double n = __builtin_fmin(__builtin_rint(log2_total), 1e6);
  return {exp2_fast(static_cast<float>(log2_total - n)), static_cast<float>(n)};
}

// ---- a row of each sequence ----------------------------------------------------------------------
// A block takes kCols columns of one head's state of one sequence, in registers: 8 lanes of 4 columns, 32 strips of
// rows, row strip + 32 i each. Bound by the state, read and written once: 64 rows of 20 heads of 128 x 128 (168 MB) 34 us,
// 4.9 TB/s.
constexpr int kCols = 32, kStrips = 32;
struct NoTab {};
template <int DT, int NK, class Tab>
__global__ __launch_bounds__(256) void k_decay_row(DecayArgs a, Tab t, size_t first_seq) {
  using E = Elem<DT>;
  using T = typename E::T;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ float sums[4][kCols];
  const int slices = static_cast<int>((a.Dv + kCols - 1) / kCols);
  const size_t head = blockIdx.x / slices;
  const int c0 = blockIdx.x % slices * kCols + (threadIdx.x & 7) * 4, strip = threadIdx.x >> 3;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int Dk = static_cast<int>(a.Dk), Dv = static_cast<int>(a.Dv);
  size_t row = first_seq + blockIdx.y, seq = row;  // a row of each, where there is no table
  if constexpr (std::is_same_v<Tab, DecayTab>) {
    row = t.of[blockIdx.y].row;
    seq = t.of[blockIdx.y].seq;
  }
  float* state = a.state ? a.state + (seq * a.heads + head) * a.Dk * a.Dv : nullptr;
  const T* q = static_cast<const T*>(a.q) + row * a.ldq + head / (a.heads / a.q_heads) * a.Dk;
  const T* k = static_cast<const T*>(a.k) + row * a.ldk + head / (a.heads / a.k_heads) * a.Dk;
  const T* v = static_cast<const T*>(a.v) + row * a.ldv + head / (a.heads / a.v_heads) * a.Dv;
  const double decay = a.decay ? a.decay[head] : 0.0, gate = a.gates ? a.gates[row * a.ldg + head] : 0.0;
  const bool whole = c0 + 4 <= Dv;

  float S[NK][4] = {};
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int r = strip + kStrips * i;
    if (!state || r >= Dk) continue;
    const float* p = state + static_cast<size_t>(r) * Dv + c0;
    if (whole) {
      const f4u s = *reinterpret_cast<const f4u*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = s[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = c0 + j < Dv ? p[j] : 0.0f;
    }
  }
  const float keep = static_cast<float>(exp(decay + gate));
  float vv[4], y[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) vv[j] = c0 + j < Dv ? E::up(v[c0 + j]) : 0.0f;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int d = strip + kStrips * i;
    if (d >= Dk) continue;
    const float kk = E::up(k[d]), qq = E::up(q[d]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      S[i][j] = __builtin_fmaf(keep, S[i][j], kk * vv[j]);
      y[j] = __builtin_fmaf(qq, S[i][j], y[j]);
    }
  }
#pragma unroll
  for (int n = 8; n < 64; n *= 2)
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] += __shfl_xor(y[j], n);
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[wave][lane * 4 + j] = y[j];
  }
  __syncthreads();
  const int c = blockIdx.x % slices * kCols + threadIdx.x;
  if (threadIdx.x < kCols && c < Dv) {
    const float o = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
    static_cast<T*>(a.out)[row * a.ldo + head * a.Dv + c] = E::down(o * a.scale);
  }
  if (!state) return;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int r = strip + kStrips * i;
    if (r >= Dk) continue;
    float* p = state + static_cast<size_t>(r) * Dv + c0;
    if (whole) {
      *reinterpret_cast<f4u*>(p) = f4u{S[i][0], S[i][1], S[i][2], S[i][3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + j < Dv) p[j] = S[i][j];
    }
  }
}

// The rows of n sequences of one row each: those of a table, or from first_seq on.
template <int DT, class Tab>
hipError_t rows_launch(const DecayArgs& a, const Tab& t, size_t first_seq, int n, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.heads * ((a.Dv + kCols - 1) / kCols)), n);
  if (a.Dk <= 64)
    k_decay_row<DT, 2, Tab><<<grid, 256, 0, s>>>(a, t, first_seq);
  else if (a.Dk <= 128)
    k_decay_row<DT, 4, Tab><<<grid, 256, 0, s>>>(a, t, first_seq);
  else
    k_decay_row<DT, 8, Tab><<<grid, 256, 0, s>>>(a, t, first_seq);
  return hipGetLastError();
}

// ---- chunks of rows ----------------------------------------------------------------------------------
// A block takes 16 columns a wave of one head's state over a tile of a sequence, a chunk of 32 rows at a time; each of its
// waves holds the state of its 16 columns in registers, as the matrix instructions leave it: lane l, column l % 16,
// rows 4 (l / 16) + 0..3 of each 16. A lane's rows of two such tiles are also one operand of the next product over
// these rows, as are the weights of a chunk's rows (k q^T): neither goes through LDS to change its layout. An operand's 32
// inputs then are, for lane group g = l / 16, 4 g + 0..3 and 16 + 4 g + 0..3 of them, in this order, in all products.
//
// Rows stand in LDS as bf16: fp32 in three parts (24 bits), fp16 in two, which is exact. The state, the weights and what is
// added to the state are fp32, in three parts, whatever the rows' type. All pairs of parts are multiplied but the last
// by the last of two numbers of three parts: the parts are cut off, not rounded, so that the second is up to 2^-7 of the number
// and the third up to 2^-14, and what is left out up to 2^-28 of the product, where (second, third) would be 2^-21.
template <int DT>
inline constexpr int kParts = DT == kF32 ? 3 : DT == kF16 ? 2 : 1;
constexpr int kSumParts = 3;  // of the state, the weights and what is added to the state
constexpr int kChunk = kDecayChunk;
enum DecayPass { kEnds = 0, kOutputs = 1 };

// Elements from row to row of a tile of COLS columns: 16 bytes more than a row, so that 16 rows' same elements lie in other
// LDS banks, and every place is one lane's own plus a constant. (Rows turned against each other are free of conflicts in
// every product, but each place is a register then: 195 of them a thread, 2048 x 16 x 128 x 128 bf16 40 us.)
template <int COLS>
inline constexpr int kStride = COLS + 8;

__device__ __forceinline__ float upper(float v) {  // the upper 16 bits, a bf16 number
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u);
}
__device__ __forceinline__ uint16_t upper_bits(float v) { return static_cast<uint16_t>(__builtin_bit_cast(uint32_t, v) >> 16); }

// A uniform address and 32 bits of a lane's own.
template <class T>
__device__ __forceinline__ T& at_bytes(T* base, uint32_t bytes) {
  using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
  return *reinterpret_cast<T*>(reinterpret_cast<Byte*>(base) + bytes);
}

// v in N bf16 parts: the first ones cut off, the last one what is left (of three, and of an fp16 number's two, exactly).
template <int N>
__device__ __forceinline__ void cut(float v, uint16_t* to) {
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    to[i] = upper_bits(v);
    v -= upper(v);
  }
  to[N - 1] = Elem<kBF16>::down(v);
}
template <int N>
__device__ __forceinline__ void cut8(const float* v, bf16x8* to) {
  u16x8 p[N];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint16_t w[N];
    cut<N>(v[j], w);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i][j] = w[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) to[i] = __builtin_bit_cast(bf16x8, p[i]);
}

__device__ __forceinline__ bf16x8 join(u16x4 a, u16x4 b) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
// Inputs of 16 rows of a tile as an operand over columns: lane l, row r0 + l % 16, columns from c0 on. at: by_columns_at().
template <int COLS>
__device__ __forceinline__ int by_columns_at(int lane) {
  return (lane & 15) * kStride<COLS> + (lane >> 4) * 4;
}
template <int COLS>
__device__ __forceinline__ bf16x8 by_columns(const uint16_t* at, int r0, int c0) {
  at += r0 * kStride<COLS> + c0;
  return join(*reinterpret_cast<const u16x4*>(at), *reinterpret_cast<const u16x4*>(at + 16));
}
// 16 columns of a tile as an operand over 32 rows: lane l, column c0 + l % 16. at: by_rows_at(). The LDS hands 16 lanes the
// columns of the 4 rows that they address 4 elements of each.
template <int COLS>
__device__ __forceinline__ int by_rows_at(int lane) {
  return (4 * (lane >> 4) + (lane >> 2 & 3)) * kStride<COLS> + (lane & 3) * 4;
}
template <int COLS>
__device__ __forceinline__ bf16x8 by_rows(const uint16_t* at, int c0) {
  typedef __attribute__((address_space(3))) s16x4* lds;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(at + c0));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(at + 16 * kStride<COLS> + c0));
  return join(__builtin_bit_cast(u16x4, a), __builtin_bit_cast(u16x4, b));
}
// c += a b over all pairs of parts but the third by the third.
template <int NA, int NB>
__device__ __forceinline__ void mma(const bf16x8* a, const bf16x8* b, f32x4& c) {
#pragma unroll
  for (int s = NA + NB - 2 < 3 ? NA + NB - 2 : 3; s >= 0; --s)  // the small products first
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
}

// kChunk rows of COLS columns from global memory, 8 neighbouring columns at a time, in registers and then in LDS. Loads have no
// conditions, so that all are in flight together: rows and columns past the end are read from the last ones and then
// set to 0.
template <int DT, int COLS, int TH, bool EVEN>
struct Tile {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int kVecs = COLS / 8;  // of a row
  static constexpr int kRows = TH >= 32 * kVecs ? 32 : TH >= 16 * kVecs ? 16 : 8, kUsed = kRows * kVecs;  // rows and threads at a time
  static constexpr int kEach = kChunk / kRows, N = kParts<DT>, H = 8 / E::V;
  typename E::Vec v[kEach][H];
  // The thread's first element of a chunk that starts at p, where columns come in groups of 8.
  __device__ __forceinline__ static const T* place(const T* p, size_t ld, int cols) {
    return p + (threadIdx.x % kUsed / kVecs) * ld + max(min(static_cast<int>(threadIdx.x % kVecs) * 8, cols - 8), 0);
  }
  // mine: place() of the chunk at p, of which `rows` are left
  __device__ __forceinline__ void fetch(const T* mine, const T* p, size_t ld, int rows, int cols) {
    if (kUsed < TH && threadIdx.x >= kUsed) return;
    const int r0 = threadIdx.x / kVecs, c = threadIdx.x % kVecs * 8;
    if constexpr (EVEN) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const T* from = mine + i * kRows * ld;
        if (rows < kChunk) from -= max(r0 + i * kRows - rows + 1, 0) * ld;
#pragma unroll
        for (int h = 0; h < H; ++h) v[i][h] = *reinterpret_cast<const typename E::Vec*>(from + h * E::V);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const T* from = p + min(r0 + i * kRows, rows - 1) * ld;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j / E::V][j % E::V] = from[min(c + j, cols - 1)];
      }
    }
    if (rows < kChunk || cols < COLS) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (r0 + i * kRows >= rows || c + j >= cols) v[i][j / E::V][j % E::V] = T{};
    }
  }
  __device__ __forceinline__ void store(uint16_t* tile) const {
    if (kUsed < TH && threadIdx.x >= kUsed) return;
    const int r0 = threadIdx.x / kVecs, c = threadIdx.x % kVecs * 8;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      uint16_t* to = tile + (r0 + i * kRows) * kStride<COLS> + c;
      if constexpr (DT == kBF16) {
        *reinterpret_cast<u16x8*>(to) = v[i][0];
      } else {
        float f[8];
        bf16x8 p[N];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = E::up(v[i][j / E::V][j % E::V]);
        cut8<N>(f, p);
#pragma unroll
        for (int k = 0; k < N; ++k) *reinterpret_cast<bf16x8*>(to + k * kChunk * kStride<COLS>) = p[k];
      }
    }
  }
};

// Running sums over the first 32 lanes.
__device__ __forceinline__ double running_sum(double x) {
  auto moved = [](double v, auto ctrl) {  // of the lane that many places before it in its row of 16, else 0
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    constexpr int k = decltype(ctrl)::value;
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u), k, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u >> 32), k, 0xF, 0xF, true);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
  };
  x += moved(x, std::integral_constant<int, 0x111>{});  // row_shr 1, 2, 4, 8
  x += moved(x, std::integral_constant<int, 0x112>{});
  x += moved(x, std::integral_constant<int, 0x114>{});
  x += moved(x, std::integral_constant<int, 0x118>{});
  const double first = __shfl(x, 15);
  return (threadIdx.x & 63) < 16 ? x : x + first;
}

template <int DT, int DKP, int NW>
struct DecayShape {
  static constexpr int DVP = 16 * NW, N = kParts<DT>, NS = kSumParts;
  static constexpr int kRowPart = kChunk * kStride<DKP>, kColPart = kChunk * kStride<DVP>;
  static constexpr int kRowTile = kRowPart * N, kColTile = kColPart * N, kWeights = 2 * NS * 512;
  static constexpr int kEndsOne = kRowTile + kColTile, kOutOne = 2 * kRowTile + kColTile + kWeights;
  // two buffers where they fit: the next chunk's rows are stored beside the products of this one
  static constexpr int kSumBytes = NW * kChunk * 16, kLds = 160 * 1024 - 512;
  static constexpr int kEndsBuffers = kEndsOne * 4 + kSumBytes <= kLds ? 2 : 1, kOutBuffers = kOutOne * 4 + kSumBytes <= kLds ? 2 : 1;
  static constexpr int kEndsBytes = kEndsOne * 2 * kEndsBuffers, kOutBytes = kOutOne * 2 * kOutBuffers;
  static_assert(kOutBytes + kSumBytes <= kLds && kEndsBytes + kSumBytes <= kLds, "LDS");
};

// A launch's arguments: heads of q, k and v as how many neighbouring heads share one.
struct DecayDev {
  const void *q, *k, *v;
  void* out;
  const float *decay, *gates;
  float *state, *ends;             // ends [slot][head][Dk][Dv]: the states from zeros at the tiles' ends, then those
  Keep* keeps;                     // before the tiles; keeps [slot][head]: the decay over a tile
  size_t ldq, ldk, ldv, ldo, ldg;
  int heads, q_each, k_each, v_each, Dk, Dv;
  float scale;
};

// What bounds it: neither rate. 2048 rows of 16 heads of 128 x 128 bf16 take 11 us (ends) and 20 (outputs), with the matrix cores
// 0.15 and the vector ALUs 0.3 to 0.4 busy: four chunks a tile, each a line of LDS reads, products and two barriers, of eight waves
// a compute unit; more tiles would fill it (8 x 1024 rows: 25 and 66), but each writes and reads a state of 64 KB a head.
template <int DT, int DKP, int NW, int PASS, bool EVEN>
__global__ __launch_bounds__(64 * NW, DT != kF32 && DKP <= 128 && NW == 8 && EVEN ? 4 : 2) void k_decay(DecayDev a, DecayTab t) {
  using Sh = DecayShape<DT, DKP, NW>;
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int C = kChunk, DVP = Sh::DVP, N = Sh::N, NS = Sh::NS, KT = DKP / 16;
  constexpr int kBuffers = PASS == kEnds ? Sh::kEndsBuffers : Sh::kOutBuffers, kOne = PASS == kEnds ? Sh::kEndsOne : Sh::kOutOne;
  extern __shared__ __align__(16) uint16_t lds[];  // a buffer: k, v, and of kOutputs q and the weights [slab][part][lane][8]
  __shared__ double sG[NW][C];
  __shared__ float sFrom[NW][C], sTo[NW][C];       // exp(G_i), exp(G - G_i)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;

  // this block's sequence and rows
  int s = 0;
  DecaySeq seq = t.of[0];
  if (t.n > 1) {
    for (int i = 0; i < t.n; i += 64)
      s += __popcll(__ballot(i + lane < t.n && t.of[min(i + lane, kDecaySeqs - 1)].tile <= static_cast<int>(blockIdx.x)));
    s = __builtin_amdgcn_readfirstlane(s - 1);
    seq = t.of[s];
  }
  const int p0 = (blockIdx.x - seq.tile) * t.step, len = seq.len, p1 = min(p0 + t.step, len);
  if (PASS == kEnds && p1 == len) return;  // nothing comes after the last tile
  const int Dk = a.Dk, Dv = a.Dv, head = blockIdx.z, c0 = blockIdx.y * DVP;
  const size_t first = seq.row + p0;
  const T* qp = static_cast<const T*>(a.q) + first * a.ldq + head / a.q_each * Dk;
  const T* kp = static_cast<const T*>(a.k) + first * a.ldk + head / a.k_each * Dk;
  const T* vp = static_cast<const T*>(a.v) + first * a.ldv + head / a.v_each * Dv + c0;
  T* out = static_cast<T*>(a.out) + first * a.ldo + head * Dv;
  const float* gates = a.gates ? a.gates + first * a.ldg + head : nullptr;
  const double decay = a.decay ? a.decay[head] : 0.0;
  const int rows = p1 - p0;
  const bool cut_up = s < t.many, last = p1 == len;
  const int held = Dk * Dv;
  float* slot = cut_up ? a.ends + (static_cast<size_t>(blockIdx.x) * a.heads + head) * held : nullptr;
  float* state = a.state ? a.state + (static_cast<size_t>(seq.seq) * a.heads + head) * held : nullptr;
  float* put = PASS == kEnds ? slot : last ? state : nullptr;

  Tile<DT, DKP, 64 * NW, EVEN> tk, tq;
  Tile<DT, DVP, 64 * NW, EVEN> tv;
  const int vcols = min(Dv - c0, DVP);
  const T* const kt = tk.place(kp, a.ldk, Dk);
  const T* const vt = tv.place(vp, a.ldv, vcols);
  const T* const qt = tq.place(qp, a.ldq, Dk);
  auto fetch = [&](int p) {
    tk.fetch(kt + p * a.ldk, kp + p * a.ldk, a.ldk, rows - p, Dk);
    tv.fetch(vt + p * a.ldv, vp + p * a.ldv, a.ldv, rows - p, vcols);
    if (PASS == kOutputs) tq.fetch(qt + p * a.ldq, qp + p * a.ldq, a.ldq, rows - p, Dk);
  };
  fetch(0);
  // the decays of the next NW chunks, one by each wave: running sums of its lanes' rows
  double total = 0.0;
  auto gate_of = [&](int p) {
    const int r = p + wave * C + (lane & (C - 1));
    return gates ? gates[min(r, rows - 1) * a.ldg] : 0.0f;
  };
  auto sums = [&](int p, float gate) {
    const bool in = lane < C && p + wave * C + lane < rows;
    const double step = in ? log2_step(decay + gate) : 0.0, x = running_sum(step), end = __shfl(x, C - 1);
    total += __ballot(step == kForgets) ? -__builtin_inf() : end;  // what is forgotten does not grow back by later rows
    if (lane < C) {
      sG[wave][lane] = x;
      sFrom[wave][lane] = exp2_fast(static_cast<float>(x));
      sTo[wave][lane] = exp2_fast(static_cast<float>(end - x));
    }
  };
  float gate = gate_of(0);

  // the state of this wave's columns: lane l, column l % 16, rows 4 (l / 16) + e of each 16
  const int n0 = wave * 16, col = c0 + n0 + c;
  f32x4 S[KT] = {};
  const float* from = PASS == kEnds ? nullptr : cut_up ? slot : state;
  const bool whole = Dk == DKP && c0 + DVP <= Dv;  // no row or column of the state is past its end
  const uint32_t own = (4 * g * Dv + col) * 4;
  if (from && whole) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[k][e] = at_bytes(from + (k * 16 + e) * Dv, own);
  } else if (from) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = k * 16 + 4 * g + e;
        const float f = at_bytes(from, (min(row, Dk - 1) * Dv + min(col, Dv - 1)) * 4);
        S[k][e] = row < Dk && col < Dv ? f : 0.0f;
      }
  }
  bool any = from != nullptr;  // the state may be other than 0
  T* const mine = out + c * a.ldo + c0 + n0 + 4 * g;
  auto store = [&](int b) {
    uint16_t* to = lds + b * kOne;
    tk.store(to);
    tv.store(to + Sh::kRowTile);
    if (PASS == kOutputs) tq.store(to + Sh::kRowTile + Sh::kColTile);
  };
  // two buffers: a chunk's rows are stored while the one before is multiplied
  if (kBuffers == 2) {
    store(0);
    if (C < rows) fetch(C);
  }
  for (int p = 0, ch = 0, buf = 0; p < rows; p += C) {
    if (ch == 0) {
      if (kBuffers == 2 && p) __syncthreads();  // the last chunk's readers of the sums
      if (kBuffers == 1) __syncthreads();
      sums(p, gate);
      if (p + NW * C < rows) gate = gate_of(p + NW * C);
    } else if (kBuffers == 1) {
      __syncthreads();
    }
    if (kBuffers == 1) store(0);
    if (kBuffers == 1 || ch == 0) __syncthreads();
    const int b = ch;
    const bool more = p + C < rows;
    if (kBuffers == 1 && more) fetch(p + C);
    uint16_t* const sK = lds + buf * kOne;
    uint16_t* const sV = sK + Sh::kRowTile;
    uint16_t* const sQ = sV + Sh::kColTile;
    uint16_t* const sP = sQ + Sh::kRowTile;
    const uint16_t* const kc = sK + by_columns_at<DKP>(lane);
    const uint16_t* const qc = sQ + by_columns_at<DKP>(lane);
    const uint16_t* const kr = sK + by_rows_at<DKP>(lane);
    const uint16_t* const vr = sV + by_rows_at<DVP>(lane) + n0;
    f32x4 O[2] = {};
    if constexpr (PASS == kOutputs) {
      // Weights of the chunk's rows (16 slab + i) by rows (16 jt + j): three of the four tiles hold any, a wave each; lane l, row
      // l % 16, inputs 4 g + e. The tile that stands for later rows is 0.
      if (wave < 3) {
        const int slab = wave ? 1 : 0, jt = wave == 2;
        f32x4 W = {};
#pragma unroll
        for (int ks = 0; ks < DKP / 32; ++ks) {
          bf16x8 q[N], k[N];
#pragma unroll
          for (int i = 0; i < N; ++i) {
            q[i] = by_columns<DKP>(qc + i * Sh::kRowPart, slab * 16, ks * 32);
            k[i] = by_columns<DKP>(kc + i * Sh::kRowPart, jt * 16, ks * 32);
          }
          mma<N, N>(k, q, W);
        }
        const int i = slab * 16 + c;
        const double Gi = sG[b][i];
        u16x4 part[NS];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = jt * 16 + 4 * g + e;
          const float d = exp2_fast(static_cast<float>(Gi - sG[b][j]));
          uint16_t w[NS];
          cut<NS>(j <= i ? W[e] * d : 0.0f, w);  // (rows after i may hold anything)
#pragma unroll
          for (int k = 0; k < NS; ++k) part[k][e] = w[k];
        }
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          uint16_t* to = sP + ((slab * NS + k) * 64 + lane) * 8;
          *reinterpret_cast<u16x4*>(to + jt * 4) = part[k];
          if (wave == 0) *reinterpret_cast<u16x4*>(to + 4) = u16x4{};
        }
      }
    }
    if constexpr (PASS == kOutputs) {
      // what the state gives: lane l, row 16 slab + l % 16, columns 4 g + e
      if (any) {
#pragma unroll
        for (int ks = 0; ks < DKP / 32; ++ks) {
          float f[8];
          bf16x8 h[NS];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = S[2 * ks + (e >> 2)][e & 3];
          cut8<NS>(f, h);
#pragma unroll
          for (int sl = 0; sl < 2; ++sl) {
            bf16x8 q[N];
#pragma unroll
            for (int i = 0; i < N; ++i) q[i] = by_columns<DKP>(qc + i * Sh::kRowPart, sl * 16, ks * 32);
            mma<NS, N>(h, q, O[sl]);
          }
        }
#pragma unroll
        for (int sl = 0; sl < 2; ++sl) O[sl] *= sFrom[b][sl * 16 + c];
      }
      __syncthreads();
    }
    if (kBuffers == 2 && more) {
      store(buf ^ 1);
      if (p + 2 * C < rows) fetch(p + 2 * C);
    }
    // this wave's columns of v, as an operand over rows. A weight of 0 would make a NaN of an infinity or NaN in a row that
    // comes later: such numbers are taken out, and the outputs from their row on have none
    bf16x8 v[N];
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = by_rows<DVP>(vr + i * Sh::kColPart, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= (__builtin_bit_cast(u32x4, v[0])[e] & 0x7F807F80u) + 0x00800080u;  // an exponent of all ones carries
    int from_row = C;  // the first row without a number of this lane's column
    const bool some = __ballot(odd & 0x80008000u) != 0;
    if (some) {
      u16x8 h[N];
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] = __builtin_bit_cast(u16x8, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((h[0][e] & 0x7F80) == 0x7F80) {
          from_row = min(from_row, (e >> 2) * 16 + 4 * g + (e & 3));
#pragma unroll
          for (int i = 0; i < N; ++i) h[i][e] = 0;
        }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(bf16x8, h[i]);
      from_row = min(from_row, __shfl_xor(from_row, 16));
      from_row = min(from_row, __shfl_xor(from_row, 32));
    }
    if constexpr (PASS == kOutputs) {
      typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
#pragma unroll
      for (int sl = 0; sl < 2; ++sl) {
        bf16x8 w[NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) w[k] = *reinterpret_cast<const bf16x8*>(sP + ((sl * NS + k) * 64 + lane) * 8);
        mma<N, NS>(v, w, O[sl]);
        if (some) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sl * 16 + c >= __shfl(from_row, 4 * g + e)) O[sl][e] = __builtin_nanf("");
        }
        const int r = p + sl * 16 + c, first_col = c0 + n0 + 4 * g;
        if (r >= rows) continue;
        T* to = mine + (p + sl * 16) * a.ldo;
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = E::down(O[sl][e] * a.scale);
        if (first_col + 4 <= Dv) {
          *reinterpret_cast<T4*>(to) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (first_col + e < Dv) to[e] = o[e];
        }
      }
    }
    if (PASS == kEnds || more || put) {
      if (any) {
        const float keep = sFrom[b][C - 1];
#pragma unroll
        for (int k = 0; k < KT; ++k) S[k] *= keep;
      }
      any = true;
      bf16x8 w[NS];
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = 0.0f;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) f[e] += Elem<kBF16>::up(__builtin_bit_cast(u16x8, v[i])[e]);
        f[e] *= sTo[b][(e >> 2) * 16 + 4 * g + (e & 3)];
      }
      cut8<NS>(f, w);
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        bf16x8 kk[N];
#pragma unroll
        for (int i = 0; i < N; ++i) kk[i] = by_rows<DKP>(kr + i * Sh::kRowPart, k * 16);
        mma<N, NS>(kk, w, S[k]);
      }
      if (some && from_row < C) {
#pragma unroll
        for (int k = 0; k < KT; ++k) S[k] = f32x4{} + __builtin_nanf("");
      }
    }
    if (kBuffers == 2) {
      buf ^= 1;
      if (more && ch != NW - 1) __syncthreads();
    }
    ch = ch == NW - 1 ? 0 : ch + 1;
  }
  if (put && whole) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) at_bytes(put + (k * 16 + e) * Dv, own) = S[k][e];
  } else if (put && col < Dv) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k * 16 + 4 * g + e < Dk) at_bytes(put + (k * 16 + e) * Dv, own) = S[k][e];
  }
  if (PASS == kEnds && blockIdx.y == 0) {  // each wave has the sums of its chunks
    __syncthreads();
    if (lane == 0) sG[wave][0] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
      total = 0.0;
      for (int w = 0; w < NW; ++w) total += sG[w][0];
      a.keeps[static_cast<size_t>(blockIdx.x) * a.heads + head] = keep_of(total);
    }
  }
}

// The states before the tiles in the place of those at their ends, in order: a thread V neighbouring elements, a head and a
// sequence of more than one tile a row of blocks, kBatch tiles' loads in flight.
template <int V>
__global__ __launch_bounds__(256) void k_decay_carry(DecayDev a, DecayTab t) {
  typedef float Vec __attribute__((ext_vector_type(V), aligned(4)));
  constexpr int kBatch = 8;
  const size_t n = a.Dk * a.Dv, i = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) * V;
  if (i >= n) return;
  const DecaySeq seq = t.of[blockIdx.z];
  const int tiles = (seq.len + t.step - 1) / t.step;
  const size_t head = blockIdx.y, step = a.heads * n;
  float* ends = a.ends + (static_cast<size_t>(seq.tile) * a.heads + head) * n + i;
  const Keep* keeps = a.keeps + static_cast<size_t>(seq.tile) * a.heads + head;
  Vec h = {};
  if (a.state) h = *reinterpret_cast<const Vec*>(a.state + (static_cast<size_t>(seq.seq) * a.heads + head) * n + i);
  for (int j = 0; j < tiles; j += kBatch) {
    Vec e[kBatch];
    Keep f[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const size_t q = min(j + k, tiles - 2);  // (the last tile's end is not needed)
      e[k] = *reinterpret_cast<const Vec*>(ends + q * step);
      f[k] = keeps[q * a.heads];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (j + k >= tiles) break;
      *reinterpret_cast<Vec*>(ends + (j + k) * step) = h;
      // a power past what a factor holds is taken of the state first: exactly, as far as the result is a number of fp32
      const int power = static_cast<int>(f[k].power), in = min(max(power, -125), 125);
      const float factor = __builtin_ldexpf(f[k].part, in);
      if (power != in) {
#pragma unroll
        for (int c = 0; c < V; ++c) h[c] = __builtin_ldexpf(h[c], power - in);
      }
#pragma unroll
      for (int c = 0; c < V; ++c) h[c] = __builtin_fmaf(factor, h[c], e[k][c]);
    }
  }
}

template <int DT, int DKP, int NW, bool EVEN>
hipError_t tiles_launch(const DecayDev& a, const DecayTab& t, hipStream_t s) {
  using Sh = DecayShape<DT, DKP, NW>;
  const unsigned heads = a.heads, slices = (a.Dv + Sh::DVP - 1) / Sh::DVP;
  hipError_t e;
  if (t.many) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_decay<DT, DKP, NW, kEnds, EVEN>), hipFuncAttributeMaxDynamicSharedMemorySize,
                            Sh::kEndsBytes);
    if (e != hipSuccess) return e;
    k_decay<DT, DKP, NW, kEnds, EVEN><<<dim3(t.cut_tiles, slices, heads), 64 * NW, Sh::kEndsBytes, s>>>(a, t);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (a.Dk * a.Dv % 4 == 0)
      k_decay_carry<4><<<dim3((a.Dk * a.Dv + 1023) / 1024, heads, t.many), 256, 0, s>>>(a, t);
    else
      k_decay_carry<1><<<dim3((a.Dk * a.Dv + 255) / 256, heads, t.many), 256, 0, s>>>(a, t);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_decay<DT, DKP, NW, kOutputs, EVEN>), hipFuncAttributeMaxDynamicSharedMemorySize,
                          Sh::kOutBytes);
  if (e != hipSuccess) return e;
  k_decay<DT, DKP, NW, kOutputs, EVEN><<<dim3(t.tiles, slices, heads), 64 * NW, Sh::kOutBytes, s>>>(a, t);
  return hipGetLastError();
}

template <int DT>
hipError_t tiles_of(const DecayArgs& a, const DecayTab& t, float* ws, hipStream_t s) {
  DecayDev d{a.q, a.k, a.v, a.out, a.decay, a.gates, a.state, ws, nullptr, a.ldq, a.ldk, a.ldv, a.ldo, a.ldg,
             static_cast<int>(a.heads), static_cast<int>(a.heads / a.q_heads), static_cast<int>(a.heads / a.k_heads),
             static_cast<int>(a.heads / a.v_heads), static_cast<int>(a.Dk), static_cast<int>(a.Dv), a.scale};
  if (t.many) d.keeps = reinterpret_cast<Keep*>(ws + static_cast<size_t>(t.cut_tiles) * a.heads * a.Dk * a.Dv);
  auto sized = [&](auto wide, auto even) {
    constexpr int NW = decltype(wide)::value ? 8 : 4;
    constexpr bool EVEN = decltype(even)::value;
    if (a.Dk <= 64) return tiles_launch<DT, 64, NW, EVEN>(d, t, s);
    if (a.Dk <= 96) return tiles_launch<DT, 96, NW, EVEN>(d, t, s);
    if (a.Dk <= 128) return tiles_launch<DT, 128, NW, EVEN>(d, t, s);
    return tiles_launch<DT, 256, NW, EVEN>(d, t, s);
  };
  const bool even = a.Dk % 8 == 0 && a.Dv % 8 == 0;
  // Blocks of 128 columns read q and k once. (Blocks of 64 are sooner done where each has a compute unit of its own, 1000 x 777
  // fp32 33.7 us and 38.0, but take more of the chip: of three contexts at once 22.0 us a call, and 15.9 by these.)
  if (a.Dv > 64) return even ? sized(std::true_type{}, std::true_type{}) : sized(std::true_type{}, std::false_type{});
  return even ? sized(std::false_type{}, std::true_type{}) : sized(std::false_type{}, std::false_type{});
}

}  // namespace

hipError_t launch_decay(const DecayArgs& a, float* ws, hipStream_t s) {
  if (!a.rows) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (row_each(a)) {
      for (size_t q = 0; q < a.seqs; q += 65535) {
        const hipError_t e = rows_launch<DT>(a, NoTab{}, q, static_cast<int>(a.seqs - q < 65535 ? a.seqs - q : 65535), s);
        if (e != hipSuccess) return e;
      }
      return hipSuccess;
    }
    return each_decay(a, hipSuccess, [&](const DecayTab& t) { return rows_launch<DT>(a, t, 0, t.n, s); },
                      [&](const DecayTab& t) { return tiles_of<DT>(a, t, ws, s); });
  });
}

}  // namespace mmf
