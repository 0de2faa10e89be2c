// mmf_decay.hip -- linear attention with a decay for each head, its state carried between calls.
//
// Per head: S = exp(a) S + k v^T, out = scale q^T S, with a = decay[head] + gates[row, head] the log decay of a row.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

// A block takes kCols columns of one head's state of one sequence, in registers: 8 lanes of 4 columns, 32 strips of
// rows, row strip + 32 i each. Step by step down the sequence.
constexpr int kCols = 32, kStrips = 32;
template <int DT, int NK>
__global__ __launch_bounds__(256) void k_decay_steps(DecayArgs a, SeqTab t, size_t seq0, size_t row0, int single) {
  using E = Elem<DT>;
  using T = typename E::T;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ float sums[2][4][kCols];
  const int slices = static_cast<int>((a.Dv + kCols - 1) / kCols);
  const size_t head = blockIdx.x / slices, seq = blockIdx.y;
  const int c0 = blockIdx.x % slices * kCols + (threadIdx.x & 7) * 4, strip = threadIdx.x >> 3;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int Dk = static_cast<int>(a.Dk), Dv = static_cast<int>(a.Dv);
  const size_t first = row0 + (single ? seq : t.len > 0 ? seq * t.len : t.row[seq]);
  const int len = single ? 1 : t.len > 0 ? t.len : t.row[seq + 1] - t.row[seq];
  if (!len) return;
  float* state = a.state ? a.state + ((seq0 + seq) * a.heads + head) * a.Dk * a.Dv : nullptr;
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
hipError_t steps_launch(const DecayArgs& a, const SeqTab& t, size_t seq0, size_t row0, int n, int single, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.heads * ((a.Dv + kCols - 1) / kCols)), n);
  if (a.Dk <= 64)
    k_decay_steps<DT, 2><<<grid, 256, 0, s>>>(a, t, seq0, row0, single);
  else if (a.Dk <= 128)
    k_decay_steps<DT, 4><<<grid, 256, 0, s>>>(a, t, seq0, row0, single);
  else
    k_decay_steps<DT, 8><<<grid, 256, 0, s>>>(a, t, seq0, row0, single);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_decay(const DecayArgs& a, float*, hipStream_t s) {
  if (!a.rows) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    size_t row0 = 0;
    for (size_t q = 0; q < a.seqs; q += kSeqs) {
      SeqTab t;
      int tiles = 0;
      const int n = static_cast<int>(a.seqs - q < kSeqs ? a.seqs - q : kSeqs);
      const size_t rows = fill_seqs(t, a.lens, a.rows, a.seqs, q, n, 1 << 24, &tiles);
      const hipError_t e = steps_launch<DT>(a, t, q, row0, n, one_row_each(a.lens, a.rows, a.seqs, q, n), s);
      if (e != hipSuccess) return e;
      row0 += rows;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
