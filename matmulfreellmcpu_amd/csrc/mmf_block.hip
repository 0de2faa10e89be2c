// mmf_block.hip -- a block's output through its norm, gate and residual scale onto the residual, then the next
// block's norm with its int8 codes.
//
// p = b / sqrt(mean(b^2) + eps) * w_post, h = x + scale * channels * act(gate) * p, y = h / sqrt(mean(h^2) + eps) * w_pre,
// codes and scale of y as mmf_normq.hip makes them. h is rounded to fp32 once, from 64 bits, and the second norm is
// taken of that: a code hangs on its last bits where it lies between two, so both norms, the gate's exponential
// and the code are taken in fp64, at fp32's rate on this chip.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

__device__ __forceinline__ double activation(int act, double g) {
  return act == kActNone ? g : (act == kActSilu ? g : 1.0) / (1.0 + exp(-g));
}

// Sum and maximum over a block of whole waves; `bad` joined. Every thread gets the result. `slot` is 0 or 1, in turn:
// a wave that is through the barrier may enter the next reduction while others still read this one.
struct RowSums {
  double sum[2][16], top[2][16];
  int bad[2][16];
};
__device__ __forceinline__ void block_reduce(RowSums& s, int slot, double& sum, double& top, bool& bad) {
#pragma unroll
  for (int n = 1; n < 64; n *= 2) {
    sum += __shfl_xor(sum, n);
    top = __builtin_fmax(top, __shfl_xor(top, n));
  }
  bad = __ballot(bad) != 0;
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
    s.sum[slot][wave] = sum;
    s.top[slot][wave] = top;
    s.bad[slot][wave] = bad;
  }
  __syncthreads();
  sum = s.sum[slot][0];
  top = s.top[slot][0];
  int any = s.bad[slot][0];
  for (int w = 1; w < waves; ++w) {
    sum += s.sum[slot][w];
    top = __builtin_fmax(top, s.top[slot][w]);
    any |= s.bad[slot][w];
  }
  bad = any != 0;
}

// One block a row, NV vectors of 16 bytes a thread.
template <int DT, int NV>
__global__ __launch_bounds__(NV == 8 ? 1024 : 512) void k_block(BlockArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  using Vec = typename E::Vec;
  constexpr int V = E::V;
  typedef int8_t Codes __attribute__((ext_vector_type(V), aligned(1)));
  __shared__ RowSums s;
  const size_t row = blockIdx.x;
  const int cols = static_cast<int>(a.cols), threads = blockDim.x;
  const T* bp = static_cast<const T*>(a.b) + row * a.ldb;
  const T* xp = static_cast<const T*>(a.x) + row * a.ldx;
  const T* gp = static_cast<const T*>(a.gate) + row * a.ldgate;
  Vec vb[NV] = {}, vx[NV] = {}, vg[NV] = {};
  auto load = [&](Vec& v, const T* p, int at) {
    if (at + V <= cols) {
      v = *reinterpret_cast<const Vec*>(p + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = at + j < cols ? p[at + j] : T{};
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * threads + static_cast<int>(threadIdx.x)) * V;
    load(vb[i], bp, at);
    if (a.x) load(vx[i], xp, at);
    if (a.gate) load(vg[i], gp, at);
  }
  double rstd = 1.0;
  if (a.w_post) {
    double sum = 0.0, top = 0.0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double d = E::up(vb[i][j]);
        sum = __builtin_fma(d, d, sum);
      }
    block_reduce(s, 0, sum, top, bad);
    rstd = 1.0 / __builtin_sqrt(sum / static_cast<double>(a.cols) + static_cast<double>(a.eps));
  }
  float h[NV][V];
  double sum = 0.0, top = 0.0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = (i * threads + static_cast<int>(threadIdx.x)) * V + j;
      h[i][j] = 0.0f;
      if (at >= cols) continue;
      double p = E::up(vb[i][j]);
      if (a.w_post) p = p * rstd * static_cast<double>(a.w_post[at]);
      if (a.gate) p *= activation(a.act, E::up(vg[i][j]));
      if (a.channels) p *= static_cast<double>(a.channels[at]);
      p *= static_cast<double>(a.scale);
      if (a.x) p += E::up(vx[i][j]);
      h[i][j] = static_cast<float>(p);
      const double d = h[i][j], hw = a.w_pre ? d * static_cast<double>(a.w_pre[at]) : d;
      sum = __builtin_fma(d, d, sum);
      top = __builtin_fmax(top, __builtin_fabs(hw));
      bad |= !(__builtin_fabs(hw) < __builtin_inf());
    }
  double rstd2 = 1.0, m = 1.0;
  if (a.y || a.codes) {
    block_reduce(s, 1, sum, top, bad);
    bad |= !(sum < __builtin_inf());
    if (a.w_pre) rstd2 = 1.0 / __builtin_sqrt(sum / static_cast<double>(a.cols) + static_cast<double>(a.eps));
    m = __builtin_fmax(top * rstd2, 1e-5);
    if (a.codes && threadIdx.x == 0) a.scales[row] = bad ? __builtin_nanf("") : static_cast<float>(m / 127.0);
  }
  const double inv = 127.0 * rstd2 / m;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * threads + static_cast<int>(threadIdx.x)) * V;
    if (at >= cols) break;
    Codes c = {};
    Vec vh, vy = {};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float w = a.w_pre && at + j < cols ? a.w_pre[at + j] : 1.0f;
      const double hw = static_cast<double>(h[i][j]) * static_cast<double>(w);
      if (a.codes) c[j] = bad ? static_cast<int8_t>(0) : static_cast<int8_t>(static_cast<int>(__builtin_rint(hw * inv)));
      vh[j] = E::down(h[i][j]);
      if (a.y) vy[j] = E::down(static_cast<float>(hw * rstd2));
    }
    int8_t* codes = a.codes + row * a.ldcodes + at;
    T* ho = static_cast<T*>(a.h) + row * a.ldh + at;
    T* yo = static_cast<T*>(a.y) + row * a.ldy + at;
    if (at + V <= cols) {
      if (a.codes) *reinterpret_cast<Codes*>(codes) = c;
      if (a.h) *reinterpret_cast<Vec*>(ho) = vh;
      if (a.y) *reinterpret_cast<Vec*>(yo) = vy;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (at + j >= cols) break;
        if (a.codes) codes[j] = c[j];
        if (a.h) ho[j] = vh[j];
        if (a.y) yo[j] = vy[j];
      }
    }
  }
}

// Rows that no block holds, read three times; a thread makes its elements of h again from b, x and the gate
// before it writes any of them, so that h may stand in their place.
template <int DT>
__global__ __launch_bounds__(512) void k_block_long(BlockArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ RowSums s;
  const size_t row = blockIdx.x;
  const T* bp = static_cast<const T*>(a.b) + row * a.ldb;
  const T* xp = static_cast<const T*>(a.x) + row * a.ldx;
  const T* gp = static_cast<const T*>(a.gate) + row * a.ldgate;
  double rstd = 1.0;
  if (a.w_post) {
    double sum = 0.0, top = 0.0;
    bool bad = false;
    for (size_t i = threadIdx.x; i < a.cols; i += 512) {
      const double d = E::up(bp[i]);
      sum = __builtin_fma(d, d, sum);
    }
    block_reduce(s, 0, sum, top, bad);
    rstd = 1.0 / __builtin_sqrt(sum / static_cast<double>(a.cols) + static_cast<double>(a.eps));
  }
  auto h_at = [&](size_t i) {
    double p = E::up(bp[i]);
    if (a.w_post) p = p * rstd * static_cast<double>(a.w_post[i]);
    if (a.gate) p *= activation(a.act, E::up(gp[i]));
    if (a.channels) p *= static_cast<double>(a.channels[i]);
    p *= static_cast<double>(a.scale);
    if (a.x) p += E::up(xp[i]);
    return static_cast<float>(p);
  };
  double sum = 0.0, top = 0.0;
  bool bad = false;
  for (size_t i = threadIdx.x; (a.y || a.codes) && i < a.cols; i += 512) {
    const double d = h_at(i), hw = a.w_pre ? d * static_cast<double>(a.w_pre[i]) : d;
    sum = __builtin_fma(d, d, sum);
    top = __builtin_fmax(top, __builtin_fabs(hw));
    bad |= !(__builtin_fabs(hw) < __builtin_inf());
  }
  block_reduce(s, 1, sum, top, bad);
  bad |= !(sum < __builtin_inf());
  const double rstd2 = a.w_pre ? 1.0 / __builtin_sqrt(sum / static_cast<double>(a.cols) + static_cast<double>(a.eps)) : 1.0;
  const double m = __builtin_fmax(top * rstd2, 1e-5), inv = 127.0 * rstd2 / m;
  if (a.codes && threadIdx.x == 0) a.scales[row] = bad ? __builtin_nanf("") : static_cast<float>(m / 127.0);
  for (size_t i = threadIdx.x; i < a.cols; i += 512) {
    const float h = h_at(i);
    const double hw = a.w_pre ? static_cast<double>(h) * static_cast<double>(a.w_pre[i]) : static_cast<double>(h);
    if (a.codes) a.codes[row * a.ldcodes + i] = bad ? 0 : static_cast<int8_t>(__builtin_rint(hw * inv));
    if (a.h) static_cast<T*>(a.h)[row * a.ldh + i] = E::down(h);
    if (a.y) static_cast<T*>(a.y)[row * a.ldy + i] = E::down(static_cast<float>(hw * rstd2));
  }
}

}  // namespace

hipError_t launch_block(const BlockArgs& all, hipStream_t s) {
  if (!all.rows || !all.cols) return hipSuccess;
  return with_type(all.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    using T = typename Elem<DT>::T;
    const BlockPlan p = block_plan(DT, all.cols);
    constexpr size_t most = size_t{1} << 20;  // rows of a launch: a grid has fewer than 2^32 threads
    for (size_t r = 0; r < all.rows; r += most) {
      BlockArgs a = all;
      a.rows = all.rows - r < most ? all.rows - r : most;
      a.b = static_cast<const T*>(a.b) + r * a.ldb;
      if (a.x) a.x = static_cast<const T*>(a.x) + r * a.ldx;
      if (a.gate) a.gate = static_cast<const T*>(a.gate) + r * a.ldgate;
      if (a.h) a.h = static_cast<T*>(a.h) + r * a.ldh;
      if (a.y) a.y = static_cast<T*>(a.y) + r * a.ldy;
      if (a.codes) {
        a.codes += r * a.ldcodes;
        a.scales += r;
      }
      const unsigned rows = static_cast<unsigned>(a.rows);
      switch (p.vecs) {
        case 1: k_block<DT, 1><<<rows, p.threads, 0, s>>>(a); break;
        case 2: k_block<DT, 2><<<rows, p.threads, 0, s>>>(a); break;
        case 4: k_block<DT, 4><<<rows, p.threads, 0, s>>>(a); break;
        case 8: k_block<DT, 8><<<rows, p.threads, 0, s>>>(a); break;
        default: k_block_long<DT><<<rows, 512, 0, s>>>(a);
      }
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
