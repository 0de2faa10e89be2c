// mmf_w8.hip -- products of int8 rows and int8 weights, with a scale a row and a scale an output.
//
// out[r, n] = xs[r] ws[n] sum_k x[r, k] w[n, k] + bias[n]. The sums are exact in int32, in any order; an output takes
// four fp32 roundings and its type's. Weights stand as matrix operands (mmf_layer8.hpp) and are the matrix
// instruction's first operand, so that a lane's sums are neighbouring outputs of one row.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v4iu __attribute__((ext_vector_type(4), aligned(1)));

// codes [N, K] -> the layout, a thread 16 bytes of it.
__global__ __launch_bounds__(256) void k_w8_pack(const int8_t* codes, W8Geom g, int8_t* out) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<size_t>(g.nt) * g.nk * 64) return;
  const int lane = i & 63;
  const size_t run = i >> 6;
  const int k0 = static_cast<int>(run % g.nk) * 32 + 16 * (lane >> 5);
  const size_t n = run / g.nk * 32 + (lane & 31);
#pragma unroll
  for (int j = 0; j < 16; ++j)
    out[i * 16 + j] = n < static_cast<size_t>(g.N) && k0 + j < g.K ? codes[n * g.K + k0 + j] : static_cast<int8_t>(0);
}

// 16 inputs of a row from k on; what stands past the row's end meets weights of 0 and is not read.
__device__ __forceinline__ v4i load_x(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const v4iu*>(row + k);
  v4i v{};
  for (int j = 0; j < 16 && k + j < K; ++j) v[j / 4] |= static_cast<int>(static_cast<uint8_t>(row[k + j])) << (8 * (j % 4));
  return v;
}

__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
  return __builtin_fmaf(static_cast<float>(sum) * xs, ws, bias);
}
__device__ __forceinline__ void store(void* out, int dtype, size_t at, float v) {
  if (dtype == kF32)
    static_cast<float*>(out)[at] = v;
  else if (dtype == kBF16)
    static_cast<uint16_t*>(out)[at] = Elem<kBF16>::down(v);
  else
    static_cast<uint16_t*>(out)[at] = Elem<kF16>::down(v);
}

// 16 outputs of 16 FM rows a block; its 8 waves share the inputs.
constexpr int kRowWaves = 8;
template <int FM>
__global__ __launch_bounds__(64 * kRowWaves) void k_w8_rows(W8Args a, W8Geom g, const int8_t* codes, const float* scales) {
  __shared__ int sums[kRowWaves][FM][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const size_t r0 = static_cast<size_t>(blockIdx.y) * (16 * FM);
  const int8_t* w = codes + (static_cast<size_t>(blockIdx.x / 2) * g.nk * 64 + (blockIdx.x % 2 * 16 + c) + 32 * (q & 1)) * 16;
  const int8_t* x[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f) x[f] = a.x + min(r0 + 16 * f + c, a.rows - 1) * a.ldx;
  v4i acc[FM] = {};
  for (int ch = wave; ch < g.nk / 2; ch += kRowWaves) {  // 64 inputs each
    const v4i wv = *reinterpret_cast<const v4i*>(w + static_cast<size_t>(2 * ch + (q >> 1)) * 1024);
#pragma unroll
    for (int f = 0; f < FM; ++f)
      acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, load_x(x[f], 64 * ch + 16 * q, g.K), acc[f], 0, 0, 0);
  }
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][f][c * 16 + 4 * q + i] = acc[f][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 256 * FM; i += 64 * kRowWaves) {
    const size_t r = r0 + i / 16;
    const int n = blockIdx.x * 16 + i % 16;
    if (r >= a.rows || n >= g.N) continue;
    int sum = 0;
#pragma unroll
    for (int k = 0; k < kRowWaves; ++k) sum += sums[k][i / 256][i % 256];
    store(a.out, a.out_dtype, r * a.ldo + n, scaled(sum, a.xscales[r], scales[n], a.bias ? a.bias[n] : 0.0f));
  }
}

}  // namespace

hipError_t launch_w8_pack(const int8_t* codes, const W8Geom& g, int8_t* out, hipStream_t s) {
  const size_t n = static_cast<size_t>(g.nt) * g.nk * 64;
  k_w8_pack<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(codes, g, out);
  return hipGetLastError();
}

hipError_t launch_w8(const W8Args& all, const W8Geom& g, const int8_t* codes, const float* scales, char*, hipStream_t s) {
  const size_t most = 65535 * 16;
  for (size_t r = 0; r < all.rows; r += most) {
    W8Args a = all;
    a.rows = all.rows - r < most ? all.rows - r : most;
    a.x += r * all.ldx;
    a.xscales += r;
    a.out = static_cast<char*>(all.out) + r * all.ldo * dtype_size(all.out_dtype);
    const unsigned cols = (g.N + 15) / 16;
    if (a.rows <= 16)
      k_w8_rows<1><<<dim3(cols, 1), 64 * kRowWaves, 0, s>>>(a, g, codes, scales);
    else if (a.rows <= 32)
      k_w8_rows<2><<<dim3(cols, 1), 64 * kRowWaves, 0, s>>>(a, g, codes, scales);
    else
      k_w8_rows<4><<<dim3(cols, static_cast<unsigned>((a.rows + 63) / 64)), 64 * kRowWaves, 0, s>>>(a, g, codes, scales);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mmf
