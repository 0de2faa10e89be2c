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
typedef float f32x4 __attribute__((ext_vector_type(4)));

// The log decay of a row in powers of two. 2^-300 times any fp32 number is 0, as 2^-infinity is, and leaves the sums
// that it stands in their digits.
__device__ __forceinline__ double log2_step(double a) {
  a *= 1.4426950408889634;
  return a < -300.0 ? -300.0 : a;
}

// ---- a row of each sequence ----------------------------------------------------------------------
// A block takes kCols columns of one head's state of one sequence, in registers: 8 lanes of 4 columns, 32 strips of
// rows, row strip + 32 i each. Step by step down the sequence.
constexpr int kCols = 32, kStrips = 32;
template <int DT, int NK>
__global__ __launch_bounds__(256) void k_decay_steps(DecayArgs a, DecayTab t, size_t first_seq) {
  using E = Elem<DT>;
  using T = typename E::T;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ float sums[2][4][kCols];
  const int slices = static_cast<int>((a.Dv + kCols - 1) / kCols);
  const size_t head = blockIdx.x / slices;
  const int c0 = blockIdx.x % slices * kCols + (threadIdx.x & 7) * 4, strip = threadIdx.x >> 3;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int Dk = static_cast<int>(a.Dk), Dv = static_cast<int>(a.Dv);
  const bool listed = t.n > 0;  // else a row of each
  const size_t first = listed ? t.row[blockIdx.y] : first_seq + blockIdx.y, seq = listed ? t.seq[blockIdx.y] : first;
  const int len = listed ? t.len[blockIdx.y] : 1;
  float* state = a.state ? a.state + (seq * a.heads + head) * a.Dk * a.Dv : nullptr;
  const T* q = static_cast<const T*>(a.q) + first * a.ldq + head / (a.heads / a.q_heads) * a.Dk;
  const T* k = static_cast<const T*>(a.k) + first * a.ldk + head / (a.heads / a.k_heads) * a.Dk;
  const T* v = static_cast<const T*>(a.v) + first * a.ldv + head / (a.heads / a.v_heads) * a.Dv;
  const float* gates = a.gates ? a.gates + first * a.ldg + head : nullptr;
  T* out = static_cast<T*>(a.out) + first * a.ldo + head * a.Dv;
  const double decay = a.decay ? a.decay[head] : 0.0;
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
  for (int r = 0; r < len; ++r) {
    const float keep = static_cast<float>(exp(decay + (gates ? gates[r * a.ldg] : 0.0)));
    float vv[4], y[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = c0 + j < Dv ? E::up(v[r * a.ldv + c0 + j]) : 0.0f;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int d = strip + kStrips * i;
      if (d >= Dk) continue;
      const float kk = E::up(k[r * a.ldk + d]), qq = E::up(q[r * a.ldq + d]);
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
    float (&s)[4][kCols] = sums[r & 1];
    if (lane < 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[wave][lane * 4 + j] = y[j];
    }
    __syncthreads();
    const int c = blockIdx.x % slices * kCols + threadIdx.x;
    if (threadIdx.x < kCols && c < Dv) {
      const float o = (s[0][threadIdx.x] + s[1][threadIdx.x]) + (s[2][threadIdx.x] + s[3][threadIdx.x]);
      out[r * a.ldo + c] = E::down(o * a.scale);
    }
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

template <int DT>
hipError_t steps_launch(const DecayArgs& a, const DecayTab& t, size_t first_seq, int n, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.heads * ((a.Dv + kCols - 1) / kCols)), n);
  if (a.Dk <= 64)
    k_decay_steps<DT, 2><<<grid, 256, 0, s>>>(a, t, first_seq);
  else if (a.Dk <= 128)
    k_decay_steps<DT, 4><<<grid, 256, 0, s>>>(a, t, first_seq);
  else
    k_decay_steps<DT, 8><<<grid, 256, 0, s>>>(a, t, first_seq);
  return hipGetLastError();
}

// ---- chunks of rows ----------------------------------------------------------------------------------
// A block takes 64 NT columns of one head's state over a tile of a sequence, a chunk of C rows at a time; each of its 4
// waves holds the state of its 16 NT columns in registers, as the matrix instructions leave it: lane l, column l % 16,
// rows 4 (l / 16) + 0..3 of each 16. A lane's rows of two such tiles are also one operand of the next product over
// these rows, as are the weights of a chunk's rows (k q^T): neither goes through LDS to change its layout. An operand's 32
// inputs then are, for lane group g = l / 16, 4 g + 0..3 and 16 + 4 g + 0..3 of them, in this order, in all products.
//
// Rows stand in LDS as bf16: fp32 in three parts (24 bits), fp16 in two, which is exact; parts a and b of two operands
// are multiplied where a + b is less than the more of them, the others are below the last kept digit. The state and
// the weights, which are fp32, enter outputs of 16 bits in two parts (2^-17 of each), of fp32 in three; what is added
// to the state is always cut into three.
template <int DT>
inline constexpr int kParts = DT == kF32 ? 3 : DT == kF16 ? 2 : 1;
template <int DT>
inline constexpr int kSumParts = DT == kF32 ? 3 : 2;  // of the state and the weights
enum DecayPass { kEnds = 0, kOutputs = 1 };

// Place of 4 neighbouring elements (unit u of a row) of a tile of COLS columns, in such units: rows are turned against each
// other so that 16 rows' same unit, 4 rows' 4 neighbouring units and one row's neighbours all lie in other LDS banks.
template <int COLS>
__device__ __forceinline__ int unit_at(int r, int u) {
  if constexpr (COLS == 64) return r * 16 + (u ^ ((r >> 1 & 1) << 2 | (r >> 2 & 1) << 3 | (r >> 3 & 1) << 1));
  return r * (COLS / 4) + (u ^ ((r & 3) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1) << 4));
}

__device__ __forceinline__ float upper(float v) {  // the upper 16 bits, a bf16 number
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xFFFF0000u);
}
__device__ __forceinline__ uint16_t upper_bits(float v) { return static_cast<uint16_t>(__builtin_bit_cast(uint32_t, v) >> 16); }

// v in N bf16 parts: the first ones cut off, the last one rounded (of three: exact).
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
// Inputs of 16 rows of a row tile as an operand over columns: lane l, row r0 + l % 16, columns from c0 on.
template <int COLS>
__device__ __forceinline__ bf16x8 by_columns(const uint16_t* tile, int r0, int c0, int lane) {
  const int r = r0 + (lane & 15), u = c0 / 4 + (lane >> 4);
  return join(*reinterpret_cast<const u16x4*>(tile + unit_at<COLS>(r, u) * 4),
              *reinterpret_cast<const u16x4*>(tile + unit_at<COLS>(r, u + 4) * 4));
}
// 16 columns of a row tile as an operand over rows: lane l, column c0 + l % 16, rows from r0 on. The LDS hands 16 lanes the
// columns of the 4 rows that they address 4 elements of each.
template <int COLS>
__device__ __forceinline__ bf16x8 by_rows(const uint16_t* tile, int r0, int c0, int lane) {
  typedef __attribute__((address_space(3))) s16x4* lds;
  const int r = r0 + 4 * (lane >> 4) + (lane >> 2 & 3), u = c0 / 4 + (lane & 3);
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(tile + unit_at<COLS>(r, u) * 4));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(tile + unit_at<COLS>(r + 16, u) * 4));
  return join(__builtin_bit_cast(u16x4, a), __builtin_bit_cast(u16x4, b));
}
// c += a b over all pairs of parts that count.
template <int NA, int NB>
__device__ __forceinline__ void mma(const bf16x8* a, const bf16x8* b, f32x4& c) {
  constexpr int M = NA > NB ? NA : NB;
#pragma unroll
  for (int s = M - 1; s >= 0; --s)  // the small products first
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
}

// C rows of COLS columns from global memory, 8 neighbouring columns at a time, in registers and then in LDS.
template <int DT, int C, int COLS>
struct Tile {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int kEach = C * COLS / 8 / 256, N = kParts<DT>;
  typename E::Vec v[kEach][8 / E::V];
  __device__ __forceinline__ void fetch(const T* p, size_t ld, int rows, int cols) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = i * 256 + threadIdx.x, r = at / (COLS / 8), c = at % (COLS / 8) * 8;
      const T* from = p + r * ld + c;
#pragma unroll
      for (int h = 0; h < 8 / E::V; ++h) {
        v[i][h] = typename E::Vec{};
        if (r >= rows) continue;
        if (c + (h + 1) * E::V <= cols) {
          v[i][h] = *reinterpret_cast<const typename E::Vec*>(from + h * E::V);
        } else {
#pragma unroll
          for (int j = 0; j < E::V; ++j)
            if (c + h * E::V + j < cols) v[i][h][j] = from[h * E::V + j];
        }
      }
    }
  }
  __device__ __forceinline__ void store(uint16_t* tile) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = i * 256 + threadIdx.x, r = at / (COLS / 8), c = at % (COLS / 8) * 8;
      uint16_t* to = tile + unit_at<COLS>(r, c / 4) * 4;
      if constexpr (DT == kBF16) {
        *reinterpret_cast<u16x8*>(to) = v[i][0];
      } else {
        float f[8];
        bf16x8 p[N];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = E::up(v[i][j / E::V][j % E::V]);
        cut8<N>(f, p);
#pragma unroll
        for (int k = 0; k < N; ++k) *reinterpret_cast<bf16x8*>(to + k * C * COLS) = p[k];
      }
    }
  }
};

template <int DT, int DKP, int NT>
struct DecayShape {
  static constexpr int C = DT == kBF16 ? 64 : 32, DVP = 64 * NT, N = kParts<DT>, NS = kSumParts<DT>;
  static constexpr int kSlabs = C / 16, kSteps = C / 32;
  static constexpr int kRowTile = C * DKP * N, kColTile = C * DVP * N, kWeights = kSlabs * kSteps * NS * 512;
  static constexpr int kEndsBytes = (kRowTile + kColTile) * 2, kOutBytes = (2 * kRowTile + kColTile + kWeights) * 2;
};

struct DecayWs {
  float* ends;   // [slot][head][Dk][Dv]: the states from zeros at the tiles' ends, then those before the tiles
  float* keeps;  // [slot][head]: the decay over a tile
};

template <int DT, int DKP, int NT, int PASS>
__global__ __launch_bounds__(256, DT == kBF16 && DKP <= 128 ? 2 : 1) void k_decay(DecayArgs a, DecayTab t, DecayWs ws) {
  using Sh = DecayShape<DT, DKP, NT>;
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int C = Sh::C, DVP = Sh::DVP, N = Sh::N, NS = Sh::NS, KT = DKP / 16;
  extern __shared__ __align__(16) uint16_t lds[];
  uint16_t* const sK = lds;
  uint16_t* const sV = lds + Sh::kRowTile;
  uint16_t* const sQ = sV + Sh::kColTile;      // of kOutputs alone
  uint16_t* const sP = sQ + Sh::kRowTile;      // [slab][step][part][lane][8]
  __shared__ double sG[2][C];
  __shared__ float sFrom[2][C], sTo[2][C];     // exp(G_i), exp(G - G_i)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;

  // this block's sequence and rows
  int at = 0;
  for (int i = 0; i < t.n; i += 64) at += __popcll(__ballot(i + lane < t.n && t.tile[i + lane] <= static_cast<int>(blockIdx.x)));
  const int s = __builtin_amdgcn_readfirstlane(at - 1);
  const int p0 = (blockIdx.x - t.tile[s]) * t.step, len = t.len[s], p1 = min(p0 + t.step, len);
  if (PASS == kEnds && p1 == len) return;  // nothing comes after the last tile
  const int slices = static_cast<int>((a.Dv + DVP - 1) / DVP);
  const size_t head = blockIdx.y / slices;
  const int Dk = static_cast<int>(a.Dk), Dv = static_cast<int>(a.Dv), c0 = blockIdx.y % slices * DVP;
  const size_t first = t.row[s] + p0;
  const T* qp = static_cast<const T*>(a.q) + first * a.ldq + head / (a.heads / a.q_heads) * a.Dk;
  const T* kp = static_cast<const T*>(a.k) + first * a.ldk + head / (a.heads / a.k_heads) * a.Dk;
  const T* vp = static_cast<const T*>(a.v) + first * a.ldv + head / (a.heads / a.v_heads) * a.Dv + c0;
  T* out = static_cast<T*>(a.out) + first * a.ldo + head * a.Dv;
  const float* gates = a.gates ? a.gates + first * a.ldg + head : nullptr;
  const double decay = a.decay ? a.decay[head] : 0.0;
  const int rows = p1 - p0, vcols = Dv - c0;
  const bool cut_up = s < t.many, last = p1 == len;
  float* slot = cut_up ? ws.ends + (blockIdx.x * a.heads + head) * a.Dk * a.Dv : nullptr;
  float* state = a.state ? a.state + (static_cast<size_t>(t.seq[s]) * a.heads + head) * a.Dk * a.Dv : nullptr;
  float* put = PASS == kEnds ? slot : last ? state : nullptr;

  Tile<DT, C, DKP> tk, tq;
  Tile<DT, C, DVP> tv;
  auto fetch = [&](int p) {
    tk.fetch(kp + p * a.ldk, a.ldk, rows - p, Dk);
    tv.fetch(vp + p * a.ldv, a.ldv, rows - p, vcols);
    if (PASS == kOutputs) tq.fetch(qp + p * a.ldq, a.ldq, rows - p, Dk);
  };
  // the decays of the chunk from row p on, by one wave: running sums of its lanes' rows
  auto gate_of = [&](int p) { return gates && lane < C && p + lane < rows ? gates[static_cast<size_t>(p + lane) * a.ldg] : 0.0f; };
  double total = 0.0;
  auto sums = [&](int p, int b, float gate) {
    double x = lane < C && p + lane < rows ? log2_step(decay + gate) : 0.0;
#pragma unroll
    for (int n = 1; n < C; n *= 2) {
      const double y = __shfl_up(x, n);
      if (lane >= n) x += y;
    }
    const double end = __shfl(x, C - 1);
    total += end;
    if (lane < C) {
      sG[b][lane] = x;
      sFrom[b][lane] = exp2_fast(static_cast<float>(x));
      sTo[b][lane] = exp2_fast(static_cast<float>(end - x));
    }
  };
  fetch(0);
  if (wave == 0) sums(0, 0, gate_of(0));

  // the state of this wave's columns
  const int n0 = wave * NT * 16;  // of the block's
  f32x4 S[KT][NT];
  const float* from = PASS == kEnds ? nullptr : cut_up ? slot : state;
#pragma unroll
  for (int k = 0; k < KT; ++k)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = k * 16 + 4 * g + e, col = c0 + n0 + n * 16 + c;
        S[k][n][e] = from && row < Dk && col < Dv ? from[static_cast<size_t>(row) * Dv + col] : 0.0f;
      }
  bool any = from != nullptr;  // the state may be other than 0

  for (int p = 0, b = 0; p < rows; p += C, b ^= 1) {
    __syncthreads();
    tk.store(sK);
    tv.store(sV);
    if (PASS == kOutputs) tq.store(sQ);
    __syncthreads();
    const bool more = p + C < rows;
    float gate = 0.0f;
    if (more) {
      fetch(p + C);
      if (wave == 0) gate = gate_of(p + C);
    }
    f32x4 O[Sh::kSlabs][NT] = {};
    if constexpr (PASS == kOutputs) {
      // weights of rows 16 wave.. of the chunk: lane l, row i, inputs j = 16 jt + 4 g + e
      if (wave < Sh::kSlabs) {
        f32x4 W[Sh::kSlabs] = {};
#pragma unroll
        for (int ks = 0; ks < DKP / 32; ++ks) {
          bf16x8 q[N], k[N];
#pragma unroll
          for (int i = 0; i < N; ++i) q[i] = by_columns<DKP>(sQ + i * C * DKP, wave * 16, ks * 32, lane);
#pragma unroll
          for (int jt = 0; jt < Sh::kSlabs; ++jt) {
            if (jt > wave) break;
#pragma unroll
            for (int i = 0; i < N; ++i) k[i] = by_columns<DKP>(sK + i * C * DKP, jt * 16, ks * 32, lane);
            mma<N, N>(k, q, W[jt]);
          }
        }
        const int i = wave * 16 + c;
        const double Gi = sG[b][i];
#pragma unroll
        for (int js = 0; js < Sh::kSteps; ++js) {
          if (2 * js > wave) break;
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int j = js * 32 + (e >> 2) * 16 + 4 * g + (e & 3);
            const float d = exp2_fast(static_cast<float>(Gi - sG[b][j]));
            w[e] = j <= i ? W[2 * js + (e >> 2)][e & 3] * d : 0.0f;  // (rows after i may hold anything)
          }
          bf16x8 part[NS];
          cut8<NS>(w, part);
#pragma unroll
          for (int k = 0; k < NS; ++k)
            *reinterpret_cast<bf16x8*>(sP + (((wave * Sh::kSteps + js) * NS + k) * 64 + lane) * 8) = part[k];
        }
      }
      // what the state gives: lane l, row 16 slab + l % 16, columns 4 g + e
      if (any) {
#pragma unroll
        for (int ks = 0; ks < DKP / 32; ++ks) {
          bf16x8 h[NT][NS];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = S[2 * ks + (e >> 2)][n][e & 3];
            cut8<NS>(v, h[n]);
          }
#pragma unroll
          for (int sl = 0; sl < Sh::kSlabs; ++sl) {
            bf16x8 q[N];
#pragma unroll
            for (int i = 0; i < N; ++i) q[i] = by_columns<DKP>(sQ + i * C * DKP, sl * 16, ks * 32, lane);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<NS, N>(h[n], q, O[sl][n]);
          }
        }
#pragma unroll
        for (int sl = 0; sl < Sh::kSlabs; ++sl) {
          const float f = sFrom[b][sl * 16 + c];
#pragma unroll
          for (int n = 0; n < NT; ++n) O[sl][n] *= f;
        }
      }
      __syncthreads();
    }
    // this wave's columns of v, as an operand over rows. A weight of 0 would make a NaN of an infinity or NaN in a row that
    // comes later: such numbers are taken out, and the outputs from their row on have none
    bf16x8 v[Sh::kSteps][NT][N];
    bool odd = false;
#pragma unroll
    for (int js = 0; js < Sh::kSteps; ++js)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[js][n][i] = by_rows<DVP>(sV + i * C * DVP, js * 32, n0 + n * 16, lane);
        const u16x8 h = __builtin_bit_cast(u16x8, v[js][n][0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) odd |= (h[e] & 0x7F80) == 0x7F80;
      }
    int from_row[NT];  // the first row without a number of this lane's column
#pragma unroll
    for (int n = 0; n < NT; ++n) from_row[n] = C;
    odd = __ballot(odd) != 0;
    if (odd) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int js = 0; js < Sh::kSteps; ++js) {
          u16x8 h[N];
#pragma unroll
          for (int i = 0; i < N; ++i) h[i] = __builtin_bit_cast(u16x8, v[js][n][i]);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((h[0][e] & 0x7F80) == 0x7F80) {
              from_row[n] = min(from_row[n], js * 32 + (e >> 2) * 16 + 4 * g + (e & 3));
#pragma unroll
              for (int i = 0; i < N; ++i) h[i][e] = 0;
            }
#pragma unroll
          for (int i = 0; i < N; ++i) v[js][n][i] = __builtin_bit_cast(bf16x8, h[i]);
        }
        from_row[n] = min(from_row[n], __shfl_xor(from_row[n], 16));
        from_row[n] = min(from_row[n], __shfl_xor(from_row[n], 32));
      }
    }
    if constexpr (PASS == kOutputs) {
#pragma unroll
      for (int sl = 0; sl < Sh::kSlabs; ++sl) {
#pragma unroll
        for (int js = 0; js < Sh::kSteps; ++js) {
          if (2 * js > sl) break;
          bf16x8 w[NS];
#pragma unroll
          for (int k = 0; k < NS; ++k)
            w[k] = *reinterpret_cast<const bf16x8*>(sP + (((sl * Sh::kSteps + js) * NS + k) * 64 + lane) * 8);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<N, NS>(v[js][n], w, O[sl][n]);
        }
      }
      if (odd) {
#pragma unroll
        for (int sl = 0; sl < Sh::kSlabs; ++sl)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sl * 16 + c >= __shfl(from_row[n], 4 * g + e)) O[sl][n][e] = __builtin_nanf("");
      }
      typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
#pragma unroll
      for (int sl = 0; sl < Sh::kSlabs; ++sl) {
        const int r = p + sl * 16 + c;
        if (r >= rows) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int col = c0 + n0 + n * 16 + 4 * g;
          T4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = E::down(O[sl][n][e] * a.scale);
          T* to = out + r * a.ldo + col;
          if (col + 4 <= Dv) {
            *reinterpret_cast<T4*>(to) = o;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < Dv) to[e] = o[e];
          }
        }
      }
    }
    if (PASS == kEnds || more || put) {
      const float keep = sFrom[b][C - 1];
      if (any) {
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int n = 0; n < NT; ++n) S[k][n] *= keep;
      }
      any = true;
#pragma unroll
      for (int js = 0; js < Sh::kSteps; ++js) {
        float to[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = sTo[b][js * 32 + (e >> 2) * 16 + 4 * g + (e & 3)];
        bf16x8 w[NT][3];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = 0.0f;
#pragma unroll
            for (int i = N - 1; i >= 0; --i) f[e] += Elem<kBF16>::up(__builtin_bit_cast(u16x8, v[js][n][i])[e]);
            f[e] *= to[e];
          }
          cut8<3>(f, w[n]);
        }
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          bf16x8 kk[N];
#pragma unroll
          for (int i = 0; i < N; ++i) kk[i] = by_rows<DKP>(sK + i * C * DKP, js * 32, k * 16, lane);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<N, 3>(kk, w[n], S[k][n]);
        }
      }
      if (odd) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (from_row[n] < C) {
#pragma unroll
            for (int k = 0; k < KT; ++k) S[k][n] = f32x4{} + __builtin_nanf("");
          }
      }
    }
    if (more && wave == 0) sums(p + C, b ^ 1, gate);
  }
  if (put) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = k * 16 + 4 * g + e, col = c0 + n0 + n * 16 + c;
          if (row < Dk && col < Dv) put[static_cast<size_t>(row) * Dv + col] = S[k][n][e];
        }
  }
  if (PASS == kEnds && threadIdx.x == 0 && c0 == 0) ws.keeps[blockIdx.x * a.heads + head] = exp2_fast(static_cast<float>(total));
}

// The states before the tiles in the place of those at their ends, in order: a thread an element, a head and a sequence of
// more than one tile a row of blocks, kBatch tiles' loads in flight.
__global__ __launch_bounds__(256) void k_decay_carry(DecayArgs a, DecayTab t, DecayWs ws) {
  constexpr int kBatch = 8;
  const size_t n = a.Dk * a.Dv, i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int s = blockIdx.z, tiles = t.tile[s + 1] - t.tile[s];
  const size_t head = blockIdx.y, step = a.heads * n;
  float* ends = ws.ends + (t.tile[s] * a.heads + head) * n + i;
  const float* keeps = ws.keeps + t.tile[s] * a.heads + head;
  float h = a.state ? a.state[(static_cast<size_t>(t.seq[s]) * a.heads + head) * n + i] : 0.0f;
  for (int j = 0; j < tiles; j += kBatch) {
    float e[kBatch], f[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const size_t q = min(j + k, tiles - 2);  // (the last tile's end is not needed)
      e[k] = ends[q * step];
      f[k] = keeps[q * a.heads];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (j + k >= tiles) break;
      ends[(j + k) * step] = h;
      // a state of 0 stays out of the product: a growing head's factor may be infinite over a tile where no row's is
      h = h != 0.0f ? __builtin_fmaf(f[k], h, e[k]) : e[k];
    }
  }
}

template <int DT, int DKP, int NT>
hipError_t tiles_launch(const DecayArgs& a, const DecayTab& t, const DecayWs& ws, hipStream_t s) {
  using Sh = DecayShape<DT, DKP, NT>;
  const unsigned heads = static_cast<unsigned>(a.heads), slices = static_cast<unsigned>((a.Dv + Sh::DVP - 1) / Sh::DVP);
  hipError_t e;
  if (t.many) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_decay<DT, DKP, NT, kEnds>), hipFuncAttributeMaxDynamicSharedMemorySize,
                            Sh::kEndsBytes);
    if (e != hipSuccess) return e;
    k_decay<DT, DKP, NT, kEnds><<<dim3(t.tile[t.many], heads * slices), 256, Sh::kEndsBytes, s>>>(a, t, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    k_decay_carry<<<dim3(static_cast<unsigned>((a.Dk * a.Dv + 255) / 256), heads, t.many), 256, 0, s>>>(a, t, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_decay<DT, DKP, NT, kOutputs>), hipFuncAttributeMaxDynamicSharedMemorySize,
                          Sh::kOutBytes);
  if (e != hipSuccess) return e;
  k_decay<DT, DKP, NT, kOutputs><<<dim3(t.tile[t.n], heads * slices), 256, Sh::kOutBytes, s>>>(a, t, ws);
  return hipGetLastError();
}

template <int DT>
hipError_t tiles_of(const DecayArgs& a, const DecayTab& t, float* ws_mem, hipStream_t s) {
  DecayWs ws{ws_mem, ws_mem ? ws_mem + static_cast<size_t>(t.tile[t.many]) * a.heads * a.Dk * a.Dv : nullptr};
  const bool wide = a.Dv > 64;
  if (a.Dk <= 64) return wide ? tiles_launch<DT, 64, 2>(a, t, ws, s) : tiles_launch<DT, 64, 1>(a, t, ws, s);
  if (a.Dk <= 128) return wide ? tiles_launch<DT, 128, 2>(a, t, ws, s) : tiles_launch<DT, 128, 1>(a, t, ws, s);
  return wide ? tiles_launch<DT, 256, 2>(a, t, ws, s) : tiles_launch<DT, 256, 1>(a, t, ws, s);
}

}  // namespace

hipError_t launch_decay(const DecayArgs& a, float* ws, hipStream_t s) {
  if (!a.rows) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (!a.lens && a.rows == a.seqs) {  // a row of each
      DecayTab none;
      none.n = 0;
      for (size_t q = 0; q < a.seqs; q += 65535) {
        const hipError_t e = steps_launch<DT>(a, none, q, static_cast<int>(a.seqs - q < 65535 ? a.seqs - q : 65535), s);
        if (e != hipSuccess) return e;
      }
      return hipSuccess;
    }
    return each_decay(a, hipSuccess, [&](const DecayTab& t) { return steps_launch<DT>(a, t, 0, t.n, s); },
                      [&](const DecayTab& t) { return tiles_of<DT>(a, t, ws, s); });
  });
}

}  // namespace mmf
