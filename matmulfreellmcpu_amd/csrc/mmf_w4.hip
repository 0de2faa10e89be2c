// mmf_w4.hip -- products with 4-bit weights that have a scale and a zero point per group of inputs.
//
// out[r, n] = sum_g s[n, g] sum_(k in g) (q[n, k] - z[n, g]) x[r, k], times the row's scale for int8 x.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

// The packed layout (mmf_layer.hpp) from codes [N, ceil(K / 2)], two a byte; one thread a word.
__global__ __launch_bounds__(256) void k_w4_pack(const uint8_t* codes, W4Geom g, uint32_t* out) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= w4_code_bytes(g) / 4) return;
  const int j = i & 3, lane = (i >> 2) & 63;
  const size_t tc = i >> 8;
  const size_t n = tc / g.nc * 16 + (lane & 15);
  const int k0 = static_cast<int>(tc % g.nc) * 128 + w4_k(g.step, j, lane >> 4);
  uint32_t w = 0;
  for (int e = 0; e < 8; ++e) {
    const int k = k0 + e;
    uint32_t q = 0;
    if (n < static_cast<size_t>(g.N) && k < g.K) q = (codes[n * ((g.K + 1) / 2) + k / 2] >> (4 * (k & 1))) & 15;
    w |= q << (4 * w4_nibble(e));
  }
  out[i] = (w << 3) | (w >> 29);
}

__global__ __launch_bounds__(256) void k_w4_pack_scales(const uint16_t* scales, const uint8_t* zeros, W4Geom g,
                                                        uint32_t* out) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= w4_scale_bytes(g) / 4) return;
  const size_t n = i / 16 / g.ns * 16 + (i & 15);
  const int k = static_cast<int>(i / 16 % g.ns) * g.step;
  uint32_t v = 0;
  if (n < static_cast<size_t>(g.N) && k < g.K) {
    const size_t at = n * ((g.K + g.group - 1) / g.group) + k / g.group;
    v = scales[at] | (zeros ? zeros[at] : 8u) << 16;
  }
  out[i] = v;
}

__device__ __forceinline__ uint32_t w4_code(uint32_t w, int e) {
  const uint32_t r = (w >> 3) | (w << 29);
  return (r >> (4 * w4_nibble(e))) & 15;
}

__device__ __forceinline__ void store_as(void* p, int dtype, size_t i, float v) {
  if (dtype == kF32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == kBF16)
    static_cast<uint16_t*>(p)[i] = Elem<kBF16>::down(v);
  else
    static_cast<uint16_t*>(p)[i] = Elem<kF16>::down(v);
}

// One wave a tile of 16 outputs and a row: lane l sums output l % 16 over its part of each chunk.
template <int DT>
__global__ __launch_bounds__(64) void k_w4_dot(W4Args a, W4Geom g, const uint32_t* codes, const uint32_t* scales) {
  const int lane = threadIdx.x, q = lane >> 4;
  const size_t tile = blockIdx.x, row = blockIdx.y;
  float sum = 0.0f;
  for (int c = 0; c < g.nc; ++c)
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = codes[((tile * g.nc + c) * 64 + lane) * 4 + j];
      const int k0 = w4_k(g.step, j, q);
      const uint32_t sz = scales[(tile * g.ns + c * (128 / g.step) + k0 / g.step) * 16 + (lane & 15)];
      const float s = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(sz)));
      float part = 0.0f;
      for (int e = 0; e < 8; ++e) {
        const int k = 128 * c + k0 + e;
        if (k >= g.K) continue;
        float x;
        if constexpr (DT == kI8)
          x = static_cast<const int8_t*>(a.x)[row * a.ldx + k];
        else
          x = Elem<DT>::up(static_cast<const typename Elem<DT>::T*>(a.x)[row * a.ldx + k]);
        part = __builtin_fmaf(static_cast<float>(static_cast<int>(w4_code(w, e)) - static_cast<int>(sz >> 16)), x, part);
      }
      sum = __builtin_fmaf(s, part, sum);
    }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  const size_t n = tile * 16 + (lane & 15);
  if (q == 0 && n < static_cast<size_t>(g.N))
    store_as(a.out, a.out_dtype, row * a.ldo + n, DT == kI8 ? sum * a.xscales[row] : sum);
}

}  // namespace

hipError_t launch_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, const W4Geom& g,
                          uint32_t* out, uint32_t* out_scales, hipStream_t s) {
  const size_t nc = w4_code_bytes(g) / 4, ns = w4_scale_bytes(g) / 4;
  k_w4_pack<<<static_cast<unsigned>((nc + 255) / 256), 256, 0, s>>>(codes, g, out);
  k_w4_pack_scales<<<static_cast<unsigned>((ns + 255) / 256), 256, 0, s>>>(scales, zeros, g, out_scales);
  return hipGetLastError();
}

hipError_t launch_w4(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, hipStream_t s) {
  if (!a.rows) return hipSuccess;
  for (size_t r = 0; r < a.rows; r += 65535) {
    W4Args b = a;
    b.rows = a.rows - r < 65535 ? a.rows - r : 65535;
    b.x = static_cast<const char*>(a.x) + r * a.ldx * dtype_size(a.dtype);
    b.out = static_cast<char*>(a.out) + r * a.ldo * dtype_size(a.out_dtype);
    if (a.xscales) b.xscales = a.xscales + r;
    const dim3 grid(g.nt, static_cast<unsigned>(b.rows));
    if (a.dtype == kI8)
      k_w4_dot<kI8><<<grid, 64, 0, s>>>(b, g, codes, scales);
    else if (a.dtype == kF32)
      k_w4_dot<kF32><<<grid, 64, 0, s>>>(b, g, codes, scales);
    else if (a.dtype == kBF16)
      k_w4_dot<kBF16><<<grid, 64, 0, s>>>(b, g, codes, scales);
    else
      k_w4_dot<kF16><<<grid, 64, 0, s>>>(b, g, codes, scales);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mmf
