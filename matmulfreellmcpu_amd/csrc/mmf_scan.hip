// mmf_scan.hip -- selective state space scan, with its state carried between calls.
//
// Per channel d and state n: h = exp(dt A[d, n]) h + dt u B[n]; y = sum_n C[n] h + skip[d] u, times
// silu(z). dt is softplus(dt + dt_bias[d]) where asked for.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

// log(1 + e) for e in [0, 1] = 2 atanh(s), s = e / (2 + e) <= 1/3, by its series: the terms after
// s^15 / 15 are below 2^-26 of the sum. 1 + e would lose the digits of a small e.
__device__ __forceinline__ float log1p_unit(float e) {
  const float s = e / (2.0f + e), q = s * s;
  float p = 1.0f / 15;
  p = __builtin_fmaf(p, q, 1.0f / 13);
  p = __builtin_fmaf(p, q, 1.0f / 11);
  p = __builtin_fmaf(p, q, 1.0f / 9);
  p = __builtin_fmaf(p, q, 1.0f / 7);
  p = __builtin_fmaf(p, q, 1.0f / 5);
  p = __builtin_fmaf(p, q, 1.0f / 3);
  return 2.0f * __builtin_fmaf(p * q, s, s);
}
__device__ __forceinline__ float softplus(float x) {
  return __builtin_fmaxf(x, 0.0f) + log1p_unit(exp2_fast(-1.44269504f * __builtin_fabsf(x)));
}

// One thread a channel of a sequence, its states one after the other: 16 at a time over all steps.
template <int DT>
__global__ __launch_bounds__(64) void k_scan_seq(ScanArgs a, SeqTab t, size_t seq0, size_t row0) {
  using E = Elem<DT>;
  using T = typename E::T;
  const TileAt at = tile_at(t, blockIdx.x);
  const size_t d = static_cast<size_t>(blockIdx.y) * 64 + threadIdx.x;
  if (d >= a.D) return;
  const int N = static_cast<int>(a.N);
  float* st = a.state ? a.state + (seq0 + at.seq) * a.N * a.D + d : nullptr;
  float h[kMaxStates];
  for (int n = 0; n < N; ++n) h[n] = st ? st[static_cast<size_t>(n) * a.D] : 0.0f;
  const float skip = a.skip ? a.skip[d] : 0.0f, bias = a.dt_bias ? a.dt_bias[d] : 0.0f;
  for (int p = 0; p < at.len; ++p) {
    const size_t r = row0 + at.row + p;
    const float u = E::up(static_cast<const T*>(a.u)[r * a.ldu + d]);
    float dt = E::up(static_cast<const T*>(a.dt)[r * a.lddt + d]) + bias;
    if (a.softplus) dt = softplus(dt);
    const T* B = static_cast<const T*>(a.B) + r * a.ldb;
    const T* C = static_cast<const T*>(a.C) + r * a.ldc;
    float y = skip * u;
    for (int n = 0; n < N; ++n) {
      const float decay = exp2_fast(dt * (a.A[d * a.N + n] * 1.44269504f));
      h[n] = __builtin_fmaf(decay, h[n], dt * u * E::up(B[n]));
      y = __builtin_fmaf(E::up(C[n]), h[n], y);
    }
    if (a.z) y *= silu_fast(E::up(static_cast<const T*>(a.z)[r * a.ldz + d]));
    static_cast<T*>(a.out)[r * a.ldo + d] = E::down(y);
  }
  if (st)
    for (int n = 0; n < N; ++n) st[static_cast<size_t>(n) * a.D] = h[n];
}

}  // namespace

hipError_t launch_sel_scan(const ScanArgs& a, hipStream_t s) {
  if (!a.rows || !a.D) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    size_t row0 = 0;
    for (size_t q = 0; q < a.seqs; q += kSeqs) {
      SeqTab t;
      int tiles = 0;
      const int n = static_cast<int>(a.seqs - q < kSeqs ? a.seqs - q : kSeqs);
      const size_t rows = fill_seqs(t, a.lens, a.rows, a.seqs, q, n, 1 << 24, &tiles);
      if (tiles) {
        k_scan_seq<decltype(dt)::value><<<dim3(tiles, static_cast<unsigned>((a.D + 63) / 64)), 64, 0, s>>>(a, t, q, row0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
      }
      row0 += rows;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
