// mmf_conv.hip -- short causal convolution over each channel, with the inputs carried between calls.
//
// out[t, d] = act(bias[d] + sum_j w[d, j] x[t - W + 1 + j, d]); the inputs before a sequence's first
// row are its state's W - 1 rows, which then become the sequence's last W - 1 inputs.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

constexpr int kConvRows = 8;  // rows of a tile

// One thread a channel and tile. The thread of a sequence's first tile also writes the state, after
// reading it: no other tile reads it.
template <int DT>
__global__ __launch_bounds__(256) void k_conv(ConvArgs a, SeqTab t, size_t seq0, size_t row0) {
  using E = Elem<DT>;
  using T = typename E::T;
  const TileAt at = tile_at(t, blockIdx.x);
  const size_t d = static_cast<size_t>(blockIdx.y) * 256 + threadIdx.x;
  if (d >= a.D) return;
  const int W = static_cast<int>(a.width);
  const T* x = static_cast<const T*>(a.x) + (row0 + at.row) * a.ldx + d;
  float* st = a.state ? a.state + (seq0 + at.seq) * (a.width - 1) * a.D + d : nullptr;
  float w[kMaxWidth];
  for (int j = 0; j < static_cast<int>(kMaxWidth); ++j) w[j] = j < W ? a.w[d * a.width + j] : 0.0f;
  const float bias = a.bias ? a.bias[d] : 0.0f;
  auto input = [&](int p) -> float {  // the sequence's input p, below 0 from the state
    if (p >= 0) return E::up(x[static_cast<size_t>(p) * a.ldx]);
    return st ? st[static_cast<size_t>(p + W - 1) * a.D] : 0.0f;
  };
  const int p0 = at.k * kConvRows;
  for (int p = p0; p < at.len && p < p0 + kConvRows; ++p) {
    float s = bias;
    for (int j = 0; j < W; ++j) s = __builtin_fmaf(w[j], input(p - W + 1 + j), s);
    if (a.silu) s = silu_fast(s);
    static_cast<T*>(a.out)[(row0 + at.row + p) * a.ldo + d] = E::down(s);
  }
  if (st && at.k == 0) {
    // oldest first: entry j is overwritten when only later ones are still to be read
    for (int j = 0; j < W - 1; ++j) st[static_cast<size_t>(j) * a.D] = input(at.len - (W - 1) + j);
  }
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, hipStream_t s) {
  if (!a.rows || !a.D) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    size_t row0 = 0;
    for (size_t q = 0; q < a.seqs; q += kSeqs) {
      SeqTab t;
      int tiles = 0;
      const int n = static_cast<int>(a.seqs - q < kSeqs ? a.seqs - q : kSeqs);
      const size_t rows = fill_seqs(t, a.lens, a.rows, a.seqs, q, n, kConvRows, &tiles);
      if (tiles) {
        k_conv<decltype(dt)::value><<<dim3(tiles, static_cast<unsigned>((a.D + 255) / 256)), 256, 0, s>>>(a, t, q, row0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
      }
      row0 += rows;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
