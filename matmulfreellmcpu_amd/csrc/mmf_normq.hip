// mmf_normq.hip -- residual addition, RMS norm and int8 codes with one scale a row.
//
// h = x + res, y = h * rstd * w with rstd = 1 / sqrt(mean(h^2) + eps), m = max(max|y|, 1e-5):
// scale = m / 127 and code = round(y * 127 / m), ties to even. rstd cancels in the code, so one pass over
// the row finds all it needs, the sum of squares and the largest |h w|, and the row stays in registers
// until its codes are known: each input is read once and each output written once. Alone, 2048 x 2560 bf16 with h, 37
// MB, takes 11.4 us, 3.2 TB/s, for 7.8 at a copy's rate: all rows start at once, so that loads, arithmetic and stores
// stand one after another; 2048 x 6912 fp32, 184 MB, 30 us; one row 2.6 us, a launch and a load.
//
// The codes are taken in 64 bits: h * w is exact there, and a value's code hangs on its last bits where it
// lies between two codes. fp64 runs at fp32's rate here (about 11 such operations an element, a third of
// the time that its bytes take).
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

// Adds (sum) and maximises (top) over the T threads of a row; all get the result.
template <int T>
__device__ __forceinline__ void row_reduce(double& sum, double& top, bool& bad) {
#pragma unroll
  for (int n = 1; n < 64; n *= 2) {
    sum += __shfl_xor(sum, n);
    top = __builtin_fmax(top, __shfl_xor(top, n));
  }
  bad = __ballot(bad) != 0;
  if constexpr (T > 64) {
    __shared__ double s_sum[T / 64], s_top[T / 64];
    __shared__ int s_bad[T / 64];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      s_sum[wave] = sum;
      s_top[wave] = top;
      s_bad[wave] = bad;
    }
    __syncthreads();
    sum = s_sum[0];
    top = s_top[0];
    int any = s_bad[0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) {
      sum += s_sum[w];
      top = __builtin_fmax(top, s_top[w]);
      any |= s_bad[w];
    }
    bad = any != 0;
  }
}

// T threads a row (one wave, or a block), NV vectors of 16 bytes each.
template <int DT, int T, int NV>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_normq(NormQArgs a) {
  using E = Elem<DT>;
  using ET = typename E::T;
  using Vec = typename E::Vec;
  constexpr int V = E::V;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  typedef int8_t Codes __attribute__((ext_vector_type(V), aligned(1)));
  const size_t row = T < 256 ? static_cast<size_t>(blockIdx.x) * (256 / T) + threadIdx.x / T : blockIdx.x;
  if (row >= a.rows) return;  // whole waves of T = 64; never of a block's row
  const int t = threadIdx.x % T, cols = static_cast<int>(a.cols);
  const ET* x = static_cast<const ET*>(a.x) + row * a.ldx;
  const ET* res = static_cast<const ET*>(a.res) + row * a.ldres;
  constexpr bool kKeep = T < 1024;  // 1024 threads have 128 registers each: the weights are read twice
  float h[NV][V], w[kKeep ? NV : 1][V];
  Vec vx[NV], vr[NV];
  auto weights = [&](int at, float* to) {
    if (at + V <= cols) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const f4u v = *reinterpret_cast<const f4u*>(a.w + at + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) to[j + k] = v[k];
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) to[j] = at + j < cols ? a.w[at + j] : 0.0f;
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * T + t) * V;
    if (at + V <= cols) {
      vx[i] = *reinterpret_cast<const Vec*>(x + at);
      if (a.res) vr[i] = *reinterpret_cast<const Vec*>(res + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool in = at + j < cols;
        vx[i][j] = in ? x[at + j] : ET{};
        vr[i][j] = in && a.res ? res[at + j] : ET{};
      }
    }
    if (kKeep) weights(at, w[i]);
  }
  double sum = 0.0, top = 0.0;
  float fine = 0.0f;  // stays 0 while the weights are finite
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float* wi = w[kKeep ? i : 0];
    if (!kKeep) weights((i * T + t) * V, wi);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[i][j] = a.res ? E::up(vx[i][j]) + E::up(vr[i][j]) : E::up(vx[i][j]);
      const double d = h[i][j];
      sum = __builtin_fma(d, d, sum);
      top = __builtin_fmax(top, __builtin_fabs(d * static_cast<double>(wi[j])));
      fine = __builtin_fmaf(wi[j], 0.0f, fine);
    }
  }
  bool bad = !(fine == 0.0f);
  row_reduce<T>(sum, top, bad);
  bad |= !(sum < __builtin_inf());
  const double rstd = 1.0 / __builtin_sqrt(sum / static_cast<double>(a.cols) + static_cast<double>(a.eps));
  const double m = __builtin_fmax(top * rstd, 1e-5);
  const double inv = 127.0 * rstd / m;
  if (t == 0) a.scales[row] = bad ? __builtin_nanf("") : static_cast<float>(m / 127.0);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * T + t) * V;
    if (at >= cols) break;
    Codes c;
    Vec vh, vy;
    float* wi = w[kKeep ? i : 0];
    if (!kKeep) weights(at, wi);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double hw = static_cast<double>(h[i][j]) * static_cast<double>(wi[j]);
      c[j] = bad ? static_cast<int8_t>(0) : static_cast<int8_t>(static_cast<int>(__builtin_rint(hw * inv)));
      vh[j] = E::down(h[i][j]);
      if (a.y) vy[j] = E::down(static_cast<float>(hw * rstd));
    }
    int8_t* codes = a.codes + row * a.ldcodes + at;
    ET* ho = static_cast<ET*>(a.h) + row * a.ldh + at;
    ET* yo = static_cast<ET*>(a.y) + row * a.ldy + at;
    if (at + V <= cols) {
      *reinterpret_cast<Codes*>(codes) = c;
      if (a.h) *reinterpret_cast<Vec*>(ho) = vh;
      if (a.y) *reinterpret_cast<Vec*>(yo) = vy;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (at + j >= cols) break;
        codes[j] = c[j];
        if (a.h) ho[j] = vh[j];
        if (a.y) yo[j] = vy[j];
      }
    }
  }
}

// Rows that no block holds: the second pass reads them again.
template <int DT>
__global__ __launch_bounds__(256) void k_normq_long(NormQArgs a) {
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

template <int DT, int T, int NV = kNormVecs>
static hipError_t normq_rows(const NormQArgs& a, int vecs, hipStream_t s) {
  if constexpr (NV > 1) {  // the instance of the smallest NV that holds the row
    if (vecs < NV) return normq_rows<DT, T, NV - 1>(a, vecs, s);
  }
  if (vecs != NV) return hipErrorInvalidValue;
  constexpr int B = T < 256 ? 256 : T;
  k_normq<DT, T, NV><<<static_cast<unsigned>((a.rows + B / T - 1) / (B / T)), B, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_normq(const NormQArgs& a, hipStream_t s) {
  if (!a.rows || !a.cols) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const NormPlan p = norm_plan(DT, a.rows, a.cols);
    if (p.threads == 64) return normq_rows<DT, 64>(a, p.vecs, s);
    if (p.threads == 256) return normq_rows<DT, 256>(a, p.vecs, s);
    if (p.threads == 1024)
      k_normq<DT, 1024, kNormVecsBlock><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(a);
    else
      k_normq_long<DT><<<static_cast<unsigned>(a.rows), 256, 0, s>>>(a);
    return hipGetLastError();
  });
}

}  // namespace mmf
