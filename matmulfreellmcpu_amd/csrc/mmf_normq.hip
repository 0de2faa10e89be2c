// mmf_normq.hip -- residual addition, RMS norm and int8 codes with one scale a row.
//
// h = x + res, y = h * rstd * w with rstd = 1 / sqrt(mean(h^2) + eps), m = max(max|y|, 1e-5):
// scale = m / 127 and code = round(y * 127 / m), ties to even.
// The codes are taken in 64 bits: h * w is exact there, and a value's code hangs on its last bits
// where it lies between two codes.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

template <int DT>
__global__ __launch_bounds__(256) void k_normq(NormQArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  const size_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = a.res ? static_cast<const T*>(a.res) + row * a.ldres : nullptr;
  double sum = 0.0, top = 0.0;
  bool bad = false;
  for (size_t i = threadIdx.x; i < a.cols; i += 256) {
    const float h = res ? E::up(x[i]) + E::up(res[i]) : E::up(x[i]);
    const double hw = static_cast<double>(h) * static_cast<double>(a.w[i]);
    sum = __builtin_fma(static_cast<double>(h), static_cast<double>(h), sum);
    top = __builtin_fmax(top, __builtin_fabs(hw));
    bad |= !(__builtin_fabs(hw) < __builtin_inf());
  }
  __shared__ double s_sum[256], s_top[256];
  s_sum[threadIdx.x] = sum;
  s_top[threadIdx.x] = top;
  bad = __syncthreads_or(bad);
  for (int n = 128; n; n >>= 1) {
    if (threadIdx.x < n) {
      s_sum[threadIdx.x] += s_sum[threadIdx.x + n];
      s_top[threadIdx.x] = __builtin_fmax(s_top[threadIdx.x], s_top[threadIdx.x + n]);
    }
    __syncthreads();
  }
  const double rstd = 1.0 / __builtin_sqrt(s_sum[0] / static_cast<double>(a.cols) + static_cast<double>(a.eps));
  const double m = __builtin_fmax(s_top[0] * rstd, 1e-5);
  const double inv = 127.0 * rstd / m;
  if (threadIdx.x == 0) a.scales[row] = bad ? __builtin_nanf("") : static_cast<float>(m / 127.0);
  for (size_t i = threadIdx.x; i < a.cols; i += 256) {
    const float h = res ? E::up(x[i]) + E::up(res[i]) : E::up(x[i]);
    const double hw = static_cast<double>(h) * static_cast<double>(a.w[i]);
    a.codes[row * a.ldcodes + i] = bad ? 0 : static_cast<int8_t>(__builtin_rint(hw * inv));
    if (a.h) static_cast<T*>(a.h)[row * a.ldh + i] = E::down(h);
    if (a.y) static_cast<T*>(a.y)[row * a.ldy + i] = E::down(static_cast<float>(hw * rstd));
  }
}

}  // namespace

hipError_t launch_normq(const NormQArgs& a, hipStream_t s) {
  if (!a.rows || !a.cols) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    k_normq<decltype(dt)::value><<<static_cast<unsigned>(a.rows), 256, 0, s>>>(a);
    return hipGetLastError();
  });
}

}  // namespace mmf
