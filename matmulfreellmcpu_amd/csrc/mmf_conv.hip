// mmf_conv.hip -- short causal convolution over each channel, with the inputs carried between calls.
//
// out[t, d] = act(bias[d] + sum_j w[d, j] x[t - W + 1 + j, d]); the inputs before a sequence's first
// row are its state's W - 1 rows, which then become the sequence's last W - 1 inputs.
//
// Bound by reading x and writing out once. A thread takes 16 bytes of neighbouring channels down a tile of
// rows, the last W - 1 inputs and the weights in registers; a tile reads W - 1 rows of its predecessor again.
// 2500 x 5120 bf16, 51 MB: 16 to 17.7 us alone, 9.2 where other work overlaps a launch's ends; 4096 x 4096 fp32
// 29 us, 4.6 TB/s.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

// The thread of a sequence's first tile also writes the state, after reading it: tiles have at least
// W - 1 rows, so no other tile reads it.
template <int DT, int W>
__global__ __launch_bounds__(64) void k_conv(ConvArgs a, SeqTab t, size_t seq0, size_t row0, int tile_rows) {
  using E = Elem<DT>;
  using T = typename E::T;
  using Vec = typename E::Vec;
  constexpr int V = E::V, kAhead = 4;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  const TileAt at = tile_at(t, blockIdx.x);
  const int D = static_cast<int>(a.D), d = (blockIdx.y * 64 + threadIdx.x) * V;
  if (d >= D) return;
  const bool whole = d + V <= D;
  const T* x = static_cast<const T*>(a.x) + (row0 + at.row) * a.ldx + d;
  T* out = static_cast<T*>(a.out) + (row0 + at.row) * a.ldo + d;
  float* st = W > 1 && a.state ? a.state + (seq0 + at.seq) * (W - 1) * a.D + d : nullptr;

  auto load = [&](size_t p) {  // the channels of the sequence's input p
    Vec v;
    if (whole) {
      v = *reinterpret_cast<const Vec*>(x + p * a.ldx);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = d + i < D ? x[p * a.ldx + i] : T{};
    }
    return v;
  };
  auto floats = [&](const float* p, float* to) {
    if (whole) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const f4u v = *reinterpret_cast<const f4u*>(p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) to[i + k] = v[k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] = d + i < D ? p[i] : 0.0f;
    }
  };
  const int p0 = at.k * tile_rows, p1 = min(p0 + tile_rows, at.len);
  Vec ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) ahead[i] = load(min(p0 + i, p1 - 1));
  float in[W][V], w[V][W], bias[V];  // in[j]: the input that w[., j] takes
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int p = p0 - (W - 1) + j;
    if (p >= 0) {
      const Vec v = load(p);
#pragma unroll
      for (int i = 0; i < V; ++i) in[j + 1][i] = E::up(v[i]);
    } else if (st) {
      floats(st + static_cast<size_t>(p + W - 1) * a.D, in[j + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) in[j + 1][i] = 0.0f;
    }
  }
  if (whole) {  // the channels' weights are neighbours
    float flat[V * W];
#pragma unroll
    for (int i = 0; i < V * W; i += 4) {
      const f4u v = *reinterpret_cast<const f4u*>(a.w + static_cast<size_t>(d) * W + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) flat[i + k] = v[k];
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) w[i][j] = flat[i * W + j];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) w[i][j] = a.w[static_cast<size_t>(min(d + i, D - 1)) * W + j];
  }
  if (a.bias) {
    floats(a.bias + d, bias);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = 0.0f;
  }
  if (st && at.k == 0) {
    // the last W - 1 inputs: entry j is len - (W - 1) + j, or where the sequence is shorter a later entry
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const int p = at.len - (W - 1) + j;
      float v[V];
      if (p >= 0) {
        const Vec u = load(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = E::up(u[i]);
      } else {
        floats(st + static_cast<size_t>(p + W - 1) * a.D, v);
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (d + i < D) st[static_cast<size_t>(j) * a.D + i] = v[i];
    }
  }
  for (int p = p0; p < p1; p += kAhead) {
    Vec now[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) now[i] = ahead[i];
    if (p + kAhead < p1) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ahead[i] = load(min(p + kAhead + i, p1 - 1));
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      if (p + s >= p1) break;
      Vec o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) in[j][i] = in[j + 1][i];
        in[W - 1][i] = E::up(now[s][i]);
        float y = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) y = __builtin_fmaf(w[i][j], in[j][i], y);
        o[i] = E::down(a.silu ? silu_fast(y) : y);
      }
      T* to = out + static_cast<size_t>(p + s) * a.ldo;
      if (whole) {
        *reinterpret_cast<Vec*>(to) = o;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (d + i < D) to[i] = o[i];
      }
    }
  }
}

template <int DT>
hipError_t conv_width(const ConvArgs& a, const SeqTab& t, size_t seq0, size_t row0, int tiles, int tile_rows, hipStream_t s) {
  constexpr int V = Elem<DT>::V;
  const dim3 grid(tiles, static_cast<unsigned>((a.D + 64 * V - 1) / (64 * V)));
  switch (a.width) {
    case 1: k_conv<DT, 1><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 2: k_conv<DT, 2><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 3: k_conv<DT, 3><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 4: k_conv<DT, 4><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 5: k_conv<DT, 5><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 6: k_conv<DT, 6><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 7: k_conv<DT, 7><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    case 8: k_conv<DT, 8><<<grid, 64, 0, s>>>(a, t, seq0, row0, tile_rows); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, hipStream_t s) {
  if (!a.rows || !a.D) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    // Rows of a tile: long tiles read less twice, short ones give more waves (us with 8, 16 and 32 rows: 2048 x
    // 2048 fp32 9.2, 9.9, 13.4; 2500 x 5120 bf16 18.6, 17.2, 18.4; 4096 x 4096 fp32 33.8, 32.0, 29.3).
    const size_t waves = a.rows * ((a.D + 64 * Elem<DT>::V - 1) / (64 * Elem<DT>::V));
    const int step = waves >= 65536 ? 32 : waves >= 20000 ? 16 : 8;
    size_t row0 = 0;
    for (size_t q = 0; q < a.seqs; q += kSeqs) {
      SeqTab t;
      int tiles = 0;
      const int n = static_cast<int>(a.seqs - q < kSeqs ? a.seqs - q : kSeqs);
      const size_t rows = fill_seqs(t, a.lens, a.rows, a.seqs, q, n, step, &tiles);
      if (tiles) {
        const hipError_t e = conv_width<DT>(a, t, q, row0, tiles, step, s);
        if (e != hipSuccess) return e;
      }
      row0 += rows;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
