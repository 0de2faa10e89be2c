// mmf_layer_dev.hpp -- the layer operators' launchers; element types and packed sequences on the device.
#pragma once

#include <hip/hip_runtime.h>

#include "mmf_layer8.hpp"

namespace mmf {

// Launchers of arguments that check() has passed.
hipError_t launch_normq(const NormQArgs& a, hipStream_t s);
hipError_t launch_conv(const ConvArgs& a, hipStream_t s);
// ws: kLayerWsBytes where scan_splits(a)
hipError_t launch_sel_scan(const ScanArgs& a, float* ws, hipStream_t s);
// codes [N, ceil(K / 2)], scales and zeros (or null) [N, ceil(K / group)] on the device -> the packed
// layout in w4_code_bytes(g) and w4_scale_bytes(g) bytes.
hipError_t launch_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, const W4Geom& g,
                          uint32_t* out, uint32_t* out_scales, hipStream_t s);
// ws: kLayerWsBytes where w4_lays(a.dtype, g, a.rows)
hipError_t launch_w4(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, char* ws,
                     hipStream_t s);
hipError_t launch_w8_pack(const int8_t* codes, const W8Geom& g, int8_t* out, hipStream_t s);
hipError_t launch_w8(const W8Args& a, const W8Geom& g, const int8_t* codes, const float* scales, hipStream_t s);
hipError_t launch_block(const BlockArgs& a, hipStream_t s);
// ws: kLayerWsBytes where decay_splits(a)
hipError_t launch_decay(const DecayArgs& a, float* ws, hipStream_t s);
// ws: kLayerWsBytes where logp_plan(a.dtype, a.V, a.rows).segs > 1
hipError_t launch_logp(const LogpArgs& a, float* ws, hipStream_t s);

// Element type DT of a row tensor: V neighbouring elements in one 16-byte access at any address that
// the type is aligned at (gfx950 takes vector accesses at element alignment).
template <int DT> struct Elem;
template <> struct Elem<kF32> {
  static constexpr int V = 4;
  typedef float T;
  typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ float up(T v) { return v; }
  static __device__ __forceinline__ T down(float v) { return v; }
};
template <> struct Elem<kBF16> {
  static constexpr int V = 8;
  typedef uint16_t T;
  typedef uint16_t Vec __attribute__((ext_vector_type(8), aligned(2)));
  static __device__ __forceinline__ float up(T v) { return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16); }
  // to nearest, ties to even (v_cvt_pk_bf16_f32)
  static __device__ __forceinline__ T down(float v) { return __builtin_bit_cast(T, static_cast<__bf16>(v)); }
};
template <> struct Elem<kF16> {
  static constexpr int V = 8;
  typedef uint16_t T;
  typedef uint16_t Vec __attribute__((ext_vector_type(8), aligned(2)));
  static __device__ __forceinline__ float up(T v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  static __device__ __forceinline__ T down(float v) { return __builtin_bit_cast(T, static_cast<_Float16>(v)); }
};

// Calls f(std::integral_constant<int, DT>) for a float type given at run time.
template <class F>
inline hipError_t with_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f(std::integral_constant<int, kF32>{});
    case kBF16: return f(std::integral_constant<int, kBF16>{});
    case kF16: return f(std::integral_constant<int, kF16>{});
  }
  return hipErrorInvalidValue;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// x * sigmoid(x); the exponential of -x overflows to infinity for x below -88, and x / inf is -0.
__device__ __forceinline__ float silu_fast(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + exp2_fast(-1.44269504f * x));
}

// Where a tile stands: its sequence, its number within the sequence, the sequence's first row and length.
struct TileAt {
  int seq, k, row, len;
};
// Tile `tile` of the table (uniform over the block). Ragged tables are searched with all 64 lanes: the
// number of sequences whose first tile is at or before this one.
__device__ __forceinline__ TileAt tile_at(const SeqTab& t, int tile) {
  TileAt r;
  if (t.len > 0) {
    r.seq = tile / t.tiles;
    r.k = tile - r.seq * t.tiles;
    r.row = r.seq * t.len;
    r.len = t.len;
    return r;
  }
  int below = 0;
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < t.n; i += 64) {
    const bool in = i + lane < t.n && t.tile[i + lane] <= tile;
    below += __popcll(__ballot(in));
  }
  // an empty sequence has the first tile of its successor: the last one counted is the one with rows
  r.seq = __builtin_amdgcn_readfirstlane(below - 1);
  r.k = tile - t.tile[r.seq];
  r.row = t.row[r.seq];
  r.len = t.row[r.seq + 1] - r.row;
  return r;
}

}  // namespace mmf
