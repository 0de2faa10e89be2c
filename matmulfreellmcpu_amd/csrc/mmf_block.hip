// mmf_block.hip -- a block's output through its norm, gate and residual scale onto the residual, then the next
// block's norm with its int8 codes.
//
// p = b / sqrt(mean(b^2) + eps) * w_post, h = x + scale * channels * act(gate) * p, y = h / sqrt(mean(h^2) + eps) * w_pre,
// codes and scale of y as mmf_normq.hip makes them. h is rounded to fp32 once, from 64 bits, and the second norm is
// taken of that: a code hangs on its last bits where it lies between two, so both norms, the gate's exponential
// and the code are taken in fp64, at fp32's rate on this chip.
//
// What bounds it: of many rows the vector ALUs, 84 instructions an element of bf16 with silu, 30 of them the sigmoid's: 2048 x 2560
// 24.7 us with them 0.57 busy (47 MB: 9.9 at a copy's rate), without a gate 15.2; 2048 x 8192 without 32.7 (117 MB, 3.6 TB/s).
#include <algorithm>

#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

// 1 / (1 + exp(-g)) to some 2^-42: exp of n ln 2 + f by its Taylor series in f (|f| <= 0.35, terms to f^10), n in the
// last places of a sum with 1.5 * 2^52, the reciprocal by one Newton step. That is far below what a code's rounding asks for
// (an error of 2^-34 would change one code in some 10^8), at half the instructions of the library's exponential and division.
__device__ __forceinline__ double sigmoid(float g) {
  constexpr double kBig = 6755399441055744.0;
  const double t = __builtin_fminf(__builtin_fmaxf(g, -700.0f), 700.0f);
  const double z = __builtin_fma(t, -1.4426950408889634, kBig), n = z - kBig;
  double f = __builtin_fma(n, -0.69314718055994529, -t);
  f = __builtin_fma(n, -2.3190468138462996e-17, f);
  double e = 1.0 / 3628800;
  e = __builtin_fma(e, f, 1.0 / 362880);
  e = __builtin_fma(e, f, 1.0 / 40320);
  e = __builtin_fma(e, f, 1.0 / 5040);
  e = __builtin_fma(e, f, 1.0 / 720);
  e = __builtin_fma(e, f, 1.0 / 120);
  e = __builtin_fma(e, f, 1.0 / 24);
  e = __builtin_fma(e, f, 1.0 / 6);
  e = __builtin_fma(e, f, 0.5);
  e = __builtin_fma(e, f, 1.0);
  e = __builtin_fma(e, f, 1.0);
  // (e 2^n: n is at most 1010 in size, so that the exponent stays one)
  const uint64_t bits = __builtin_bit_cast(uint64_t, e) + (__builtin_bit_cast(uint64_t, z) << 52);
  const double d = 1.0 + __builtin_bit_cast(double, bits);
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
  return g != g ? g : r;
}
// v of the lane K places before in its row of 16 lanes, else 0.
template <int K>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u), 0x110 + K, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u >> 32), 0x110 + K, 0xF, 0xF, true);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double of_lane(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// f over a wave of numbers of which 0 is neutral: over rows of 16 lanes, then the four of them.
template <class F>
__device__ __forceinline__ double over_wave(double v, F&& f) {
  v = f(v, moved<1>(v));
  v = f(v, moved<2>(v));
  v = f(v, moved<4>(v));
  v = f(v, moved<8>(v));
  return f(f(of_lane(v, 15), of_lane(v, 31)), f(of_lane(v, 47), of_lane(v, 63)));
}

__device__ __forceinline__ double add(double a, double b) { return a + b; }
// The larger, b of two where a is NaN. (The builtin quiets both first: two more such instructions, of the dearest.)
__device__ __forceinline__ double larger(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// 1 / sqrt(sum / cols + eps), 0 of an infinite sum: two Newton steps.
__device__ __forceinline__ double rsqrt_mean(double sum, double inv_cols, double eps) {
  const double v = __builtin_fma(sum, inv_cols, eps);
  double r = __builtin_amdgcn_rsq(v);
#pragma unroll
  for (int i = 0; i < 2; ++i) r = __builtin_fma(0.5 * r, __builtin_fma(-v * r, r, 1.0), r);
  return v < __builtin_inf() ? r : v != v ? v : 0.0;
}

// Sums and maxima (of numbers not below 0) over a block of whole waves, to all threads. Two slots in turn: a wave that is
// through the barrier may enter the next reduction while others still read this one.
struct RowSums {
  double sum[2][16], top[2][16];
};
template <bool TOP>
__device__ __forceinline__ void block_reduce(RowSums& s, int& slot, double& sum, double& top) {
  sum = over_wave(sum, add);
  if (TOP) top = over_wave(top, larger);
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (waves == 1) return;
  if (lane == 0) {
    s.sum[slot][wave] = sum;
    if (TOP) s.top[slot][wave] = top;
  }
  __syncthreads();
  auto joined = [&](const double (&of)[16], auto&& f) {  // the waves' numbers by lanes, 16 of them at most
    const double v = of[lane & 15];
    double r = (lane & 15) < waves ? v : 0.0;
    r = f(r, moved<1>(r));
    r = f(r, moved<2>(r));
    r = f(r, moved<4>(r));
    r = f(r, moved<8>(r));
    return of_lane(r, 15);
  };
  sum = joined(s.sum[slot], add);
  if (TOP) top = joined(s.top[slot], larger);
  slot ^= 1;
}

// Whether a row whose largest |y| is m has a scale m / 127 in fp32.
__device__ __forceinline__ bool scale_fits(double m) { return m < 127.0 * 0x1.ffffffp127; }
__device__ __forceinline__ float scale_of(double m) { return __builtin_fminf(static_cast<float>(m / 127.0), 0x1.fffffep127f); }

// A block goes through rows, NV vectors of 16 bytes a thread. One vector's weights stay in registers, and the next row's
// vector is on its way meanwhile; two would not fit there. EVEN: rows are whole vectors.
template <int DT, int NV, bool EVEN>
__global__ __launch_bounds__(1024, 4) void k_block(BlockArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  using Vec = typename E::Vec;
  constexpr int V = E::V;
  constexpr bool kKeep = NV == 1;
  typedef int8_t Codes __attribute__((ext_vector_type(V), aligned(1)));
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ RowSums s;
  int slot = 0;
  const int cols = static_cast<int>(a.cols), threads = blockDim.x;
  const double scale = a.scale, inv_cols = 1.0 / static_cast<double>(cols), eps = a.eps;
  const bool norm2 = a.y || a.codes;
  auto place = [&](int i) { return (i * threads + static_cast<int>(threadIdx.x)) * V; };
  // A vector's weights; 0 behind the row, so that what stands there stays 0.
  auto weights = [&](float (&w)[V], const float* p, int at) {
    if (EVEN || at + V <= cols) {
      const int in = EVEN ? min(at, cols - V) : at;
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const f4u v = p ? *reinterpret_cast<const f4u*>(p + in + j) : f4u{1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
        for (int e = 0; e < 4; ++e) w[j + e] = at < cols ? v[e] : 0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = at + j < cols ? (p ? p[at + j] : 1.0f) : 0.0f;
    }
  };
  // what stands before act(gate) / sqrt(mean(b^2) + eps)
  auto factors = [&](double (&f)[V], int at) {
    float post[V], ch[V];
    weights(post, a.w_post, at);
    weights(ch, a.channels, at);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = scale * static_cast<double>(post[j]) * static_cast<double>(ch[j]);
  };
  auto unfit = [&](const float (&w)[V]) {  // 0 while the weights are finite, else NaN
    float r = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) r = __builtin_fmaf(w[j], 0.0f, r);
    return r;
  };
  double kf[V];
  float kw[V], fine = 0.0f;
  if constexpr (kKeep) {
    factors(kf, place(0));
    weights(kw, a.w_pre, place(0));
    fine = unfit(kw);
  }
  struct Row {
    Vec b[NV], x[NV], g[NV];
  };
  auto load = [&](Vec& v, const T* p, int at) {
    if (EVEN) {
      v = *reinterpret_cast<const Vec*>(p + min(at, cols - V));
      if (at >= cols) v = Vec{};
    } else if (at + V <= cols) {
      v = *reinterpret_cast<const Vec*>(p + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = at + j < cols ? p[at + j] : T{};
    }
  };
  auto fetch = [&](Row& r, size_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load(r.b[i], static_cast<const T*>(a.b) + row * a.ldb, place(i));
    if (a.x)
#pragma unroll
      for (int i = 0; i < NV; ++i) load(r.x[i], static_cast<const T*>(a.x) + row * a.ldx, place(i));
    if (a.gate)
#pragma unroll
      for (int i = 0; i < NV; ++i) load(r.g[i], static_cast<const T*>(a.gate) + row * a.ldgate, place(i));
  };
  auto store = [&](auto* to, const auto& v, int at) {  // to: the row's first element
    using Of = std::remove_reference_t<decltype(v)>;
    if (EVEN ? at < cols : at + V <= cols) {
      *reinterpret_cast<std::remove_const_t<Of>*>(to + at) = v;
    } else if (!EVEN) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j < cols) to[at + j] = v[j];
    }
  };
  Row next = {};
  if (kKeep) fetch(next, blockIdx.x);
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (!kKeep) fetch(next, row);
    const Row now = next;
    if (kKeep && row + gridDim.x < a.rows) fetch(next, row + gridDim.x);
    double rstd = 1.0, sum = 0.0, top = 0.0;
    if (a.w_post) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double d = E::up(now.b[i][j]);
          sum = __builtin_fma(d, d, sum);
        }
      block_reduce<false>(s, slot, sum, top);
      rstd = rsqrt_mean(sum, inv_cols, eps);
    }
    float h[NV][V];
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!kKeep) {
        factors(kf, place(i));
        weights(kw, a.w_pre, place(i));
        fine = i ? fine + unfit(kw) : unfit(kw);
      }
      // four at a time: more at once go out of the registers
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        double p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = static_cast<double>(E::up(now.b[i][q + j])) * rstd * kf[q + j];
        if (a.gate) {
          if (a.act == kActNone) {
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] *= E::up(now.g[i][q + j]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] *= sigmoid(E::up(now.g[i][q + j]));
            if (a.act == kActSilu) {
#pragma unroll
              for (int j = 0; j < 4; ++j) p[j] *= E::up(now.g[i][q + j]);
            }
          }
        }
        if (a.x) {
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] += E::up(now.x[i][q + j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[i][q + j] = static_cast<float>(p[j]);
          const double d = h[i][q + j];
          sum = __builtin_fma(d, d, sum);
          top = larger(top, __builtin_fabs(d * static_cast<double>(kw[q + j])));
        }
      }
    }
    double rstd2 = 1.0, inv = 0.0;
    bool bad = false;
    if (norm2) {
      sum += fine;
      block_reduce<true>(s, slot, sum, top);
      if (a.w_pre) rstd2 = rsqrt_mean(sum, inv_cols, eps);
      const double m = larger(top * rstd2, 1e-5);
      bad = !(sum < __builtin_inf()) || !scale_fits(m);
      if (a.codes && threadIdx.x == 0) a.scales[row] = bad ? __builtin_nanf("") : scale_of(m);
      double r = __builtin_amdgcn_rcp(m);
      r = __builtin_fma(r, __builtin_fma(-m, r, 1.0), r);
      r = __builtin_fma(r, __builtin_fma(-m, r, 1.0), r);
      inv = 127.0 * rstd2 * r;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = place(i);
      if (!kKeep) weights(kw, a.w_pre, at);
      if (a.h) {
        Vec v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = E::down(h[i][j]);
        store(static_cast<T*>(a.h) + row * a.ldh, v, at);
      }
      if (!norm2) continue;
      double hw[V];
#pragma unroll
      for (int j = 0; j < V; ++j) hw[j] = static_cast<double>(h[i][j]) * static_cast<double>(kw[j]);
      if (a.y) {
        Vec v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = E::down(static_cast<float>(hw[j] * rstd2));
        store(static_cast<T*>(a.y) + row * a.ldy, v, at);
      }
      if (a.codes) {
        Codes c;
#pragma unroll
        for (int j = 0; j < V; ++j)  // to the nearest, ties to even: the sum's last place is 1
          c[j] = static_cast<int8_t>(__builtin_bit_cast(uint64_t, __builtin_fma(hw[j], inv, 6755399441055744.0)));
        if (bad) c = Codes{};
        store(a.codes + row * a.ldcodes, c, at);
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
  int slot = 0;
  const size_t row = blockIdx.x;
  const T* bp = static_cast<const T*>(a.b) + row * a.ldb;
  const T* xp = static_cast<const T*>(a.x) + row * a.ldx;
  const T* gp = static_cast<const T*>(a.gate) + row * a.ldgate;
  const double inv_cols = 1.0 / static_cast<double>(a.cols);
  double rstd = 1.0, sum = 0.0, top = 0.0;
  if (a.w_post) {
    for (size_t i = threadIdx.x; i < a.cols; i += 512) {
      const double d = E::up(bp[i]);
      sum = __builtin_fma(d, d, sum);
    }
    block_reduce<false>(s, slot, sum, top);
    rstd = rsqrt_mean(sum, inv_cols, a.eps);
  }
  auto h_at = [&](size_t i) {
    double p = static_cast<double>(E::up(bp[i])) * rstd *
               (static_cast<double>(a.scale) * (a.w_post ? static_cast<double>(a.w_post[i]) : 1.0) * (a.channels ? static_cast<double>(a.channels[i]) : 1.0));
    if (a.gate) {
      const float g = E::up(gp[i]);
      if (a.act != kActNone) p *= sigmoid(g);
      if (a.act != kActSigmoid) p *= g;
    }
    if (a.x) p += E::up(xp[i]);
    return static_cast<float>(p);
  };
  sum = 0.0;
  for (size_t i = threadIdx.x; (a.y || a.codes) && i < a.cols; i += 512) {
    const double d = h_at(i), w = a.w_pre ? a.w_pre[i] : 1.0f;
    sum = __builtin_fma(d, d, __builtin_fma(w, 0.0, sum));
    top = larger(top, __builtin_fabs(d * w));
  }
  block_reduce<true>(s, slot, sum, top);
  const double rstd2 = a.w_pre ? rsqrt_mean(sum, inv_cols, a.eps) : 1.0;
  const double m = larger(top * rstd2, 1e-5), inv = 127.0 * rstd2 / m;
  const bool bad = !(sum < __builtin_inf()) || !scale_fits(m);
  if (a.codes && threadIdx.x == 0) a.scales[row] = bad ? __builtin_nanf("") : scale_of(m);
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
      // As many blocks as the chip holds, of as many rows each. A compute unit's four SIMDs hold four waves each: two blocks
      // of five to eight waves (2048 x 2560 bf16 with silu: 24.7 us; by three blocks of five waves, of which a SIMD holds
      // four waves and no more, 27.8).
      const int waves = std::max(p.threads / 64, 1);
      const size_t held = 256 * (waves <= 4 ? 16 / waves : 4 / ((waves + 3) / 4)), each = (a.rows + held - 1) / held;
      const unsigned rows = static_cast<unsigned>(a.rows), blocks = static_cast<unsigned>((a.rows + each - 1) / each);
      const bool even = a.cols % Elem<DT>::V == 0;
      if (p.vecs == 1)
        even ? k_block<DT, 1, true><<<blocks, p.threads, 0, s>>>(a) : k_block<DT, 1, false><<<blocks, p.threads, 0, s>>>(a);
      else if (p.vecs == 2)
        even ? k_block<DT, 2, true><<<blocks, p.threads, 0, s>>>(a) : k_block<DT, 2, false><<<blocks, p.threads, 0, s>>>(a);
      else
        k_block_long<DT><<<rows, 512, 0, s>>>(a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
