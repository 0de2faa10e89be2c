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

// A lane holds a channel's NS states in registers; a wave is 64 channels, and `nw` waves share a
// channel with more states. Every lane needs the same B and C of a step: a block keeps kTile steps of them
// in LDS as fp32 and reads them four at a time, all lanes one address.
//
// What bounds it: the exponentials. A step of 16 states is 16 v_exp_f32 at a quarter of the rate and 64
// other operations, 512 cycles of a SIMD for 64 channels.
//
// Long sequences are cut into chunks so that the chip is full: kSum finds each chunk's end state from
// zeros and the sum of its steps (the decay over a chunk is exp(A * sum dt)), and kApply starts each
// chunk from the states before it, folded in order, and writes the outputs. The first chunk of kSum starts
// from the state itself. A sequence's last chunk needs no sums: its slot of the workspace keeps the
// state at the start, which kApply's last chunk overwrites in `state`.
constexpr int kTile = 32, kGroup4 = 4;
enum ScanPass { kSum = 0, kApply = 1 };

struct ScanWs {
  float* ends;  // [chunk][N][D], or null: sequences in one piece
  float* steps; // [chunk][D]
  int chunk;    // rows of a chunk
};

template <int DT, int NS, int PASS>
__global__ __launch_bounds__(512) void k_scan(ScanArgs a, SeqTab t, ScanWs ws, size_t seq0, size_t row0, int nw) {
  using E = Elem<DT>;
  using T = typename E::T;
  extern __shared__ __align__(16) float lds[];
  const TileAt at = tile_at(t, blockIdx.x);
  const int chunks = (at.len + ws.chunk - 1) / ws.chunk;
  const bool split = ws.ends != nullptr;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % nw, cw = static_cast<int>(blockDim.x >> 6) / nw;
  const int N = static_cast<int>(a.N), n0 = part * NS, np = nw * NS;
  const size_t D = a.D, dd = (static_cast<size_t>(blockIdx.y) * cw + wave / nw) * 64 + lane;
  const bool live = dd < D;
  const size_t d = live ? dd : D - 1;
  float* state = a.state ? a.state + (seq0 + at.seq) * a.N * D + d : nullptr;
  const size_t slot = static_cast<size_t>(blockIdx.x);
  auto end_of = [&](size_t item, int n) -> float& { return ws.ends[(item * a.N + n) * D + d]; };

  if (PASS == kSum && at.k == chunks - 1) {  // no sums of the last chunk: its slot keeps the state
    for (int i = 0; i < NS; ++i)
      if (live && n0 + i < N) end_of(slot, n0 + i) = state ? state[(n0 + i) * D] : 0.0f;
    return;
  }

  float A[NS], h[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) A[i] = n0 + i < N ? a.A[d * a.N + n0 + i] * 1.44269504f : 0.0f;
  if (!split || PASS == kSum) {
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = at.k == 0 && state && n0 + i < N ? state[(n0 + i) * D] : 0.0f;
  } else {
    const size_t first = slot - at.k;
    const size_t from = at.k ? first : first + chunks - 1;
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = n0 + i < N ? end_of(from, n0 + i) : 0.0f;
    for (int j = 1; j < at.k; ++j) {
      const float sum = ws.steps[(first + j) * D + d];
#pragma unroll
      for (int i = 0; i < NS; ++i)
        h[i] = __builtin_fmaf(exp2_fast(sum * A[i]), h[i], n0 + i < N ? end_of(first + j, n0 + i) : 0.0f);
    }
  }
  const float skip = a.skip ? a.skip[d] : 0.0f, bias = a.dt_bias ? a.dt_bias[d] : 0.0f;

  const int p0 = at.k * ws.chunk, p1 = min(p0 + ws.chunk, at.len);
  const size_t r0 = row0 + at.row;
  const T* up = static_cast<const T*>(a.u) + r0 * a.ldu + d;
  const T* dp = static_cast<const T*>(a.dt) + r0 * a.lddt + d;
  const T* zp = PASS == kApply && a.z ? static_cast<const T*>(a.z) + r0 * a.ldz + d : nullptr;
  const T* Bp = static_cast<const T*>(a.B) + r0 * a.ldb;
  const T* Cp = static_cast<const T*>(a.C) + r0 * a.ldc;
  T* out = static_cast<T*>(a.out) + r0 * a.ldo + d;
  float* sB = lds;
  float* sC = lds + kTile * np;
  float* sy = lds + 2 * kTile * np + wave / nw * (2 * nw * kGroup4 * 64);  // [2][nw][steps][lane]
  float total = 0.0f;
  int flip = 0;

  T un[kGroup4], dn[kGroup4], zn[kGroup4] = {};
  auto fetch = [&](int p) {
#pragma unroll
    for (int i = 0; i < kGroup4; ++i) {
      const size_t r = min(p + i, p1 - 1);
      un[i] = up[r * a.ldu];
      dn[i] = dp[r * a.lddt];
      if (zp) zn[i] = zp[r * a.ldz];
    }
  };
  fetch(p0);
  for (int pt = p0; pt < p1; pt += kTile) {
    const int steps = min(kTile, p1 - pt);
    __syncthreads();
    for (int i = threadIdx.x; i < steps * np; i += blockDim.x) {
      const int s = i / np, n = i - s * np;
      const size_t r = pt + s;
      sB[i] = n < N ? E::up(Bp[r * a.ldb + n]) : 0.0f;
      if (PASS == kApply) sC[i] = n < N ? E::up(Cp[r * a.ldc + n]) : 0.0f;
    }
    __syncthreads();
    for (int g = 0; g < steps; g += kGroup4) {
      float u[kGroup4], dt[kGroup4], z[kGroup4];
#pragma unroll
      for (int i = 0; i < kGroup4; ++i) {
        u[i] = E::up(un[i]);
        dt[i] = E::up(dn[i]) + bias;
        z[i] = E::up(zn[i]);
      }
      if (pt + g + kGroup4 < p1) fetch(pt + g + kGroup4);
#pragma unroll
      for (int i = 0; i < kGroup4; ++i) {
        if (g + i >= steps) break;
        const float step = a.softplus ? softplus(dt[i]) : dt[i];
        const float su = step * u[i];
        const float* b = sB + (g + i) * np + n0;
        const float* c = sC + (g + i) * np + n0;
        float y = 0.0f;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          h[n] = __builtin_fmaf(exp2_fast(step * A[n]), h[n], su * b[n]);
          if (PASS == kApply) y = __builtin_fmaf(c[n], h[n], y);
        }
        if (PASS == kSum) {
          total += step;
        } else if (nw == 1) {
          y = __builtin_fmaf(skip, u[i], y);
          if (zp) y *= silu_fast(z[i]);
          if (live) out[static_cast<size_t>(pt + g + i) * a.ldo] = E::down(y);
        } else {
          sy[((flip * nw + part) * kGroup4 + i) * 64 + lane] = y;
        }
      }
      if (PASS == kApply && nw > 1) {  // the parts' sums in their order; part i % nw writes step i
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kGroup4; ++i) {
          if (g + i >= steps || i % nw != part) continue;
          float y = skip * u[i];
          for (int w = 0; w < nw; ++w) y += sy[((flip * nw + w) * kGroup4 + i) * 64 + lane];
          if (zp) y *= silu_fast(z[i]);
          if (live) out[static_cast<size_t>(pt + g + i) * a.ldo] = E::down(y);
        }
        flip ^= 1;
      }
    }
  }
  if (!live) return;
  if (PASS == kSum) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < N) end_of(slot, n0 + i) = h[i];
    if (part == 0) ws.steps[slot * D + d] = total;
  } else if (state && at.k == chunks - 1) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < N) state[(n0 + i) * D] = h[i];
  }
}

template <int DT, int NS>
hipError_t scan_launch(const ScanArgs& a, const SeqTab& t, const ScanWs& ws, size_t seq0, size_t row0, int tiles,
                       hipStream_t s) {
  const int nw = static_cast<int>((a.N + NS - 1) / NS), cw = nw >= 4 ? 1 : 4 / nw;
  const size_t lds = (2 * kTile * static_cast<size_t>(nw) * NS + (nw > 1 ? 2 * nw * kGroup4 * 64 * cw : 0)) * 4;
  const dim3 grid(tiles, static_cast<unsigned>((a.D + cw * 64 - 1) / (cw * 64)));
  if (ws.ends) {
    k_scan<DT, NS, kSum><<<grid, nw * cw * 64, lds, s>>>(a, t, ws, seq0, row0, nw);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  k_scan<DT, NS, kApply><<<grid, nw * cw * 64, lds, s>>>(a, t, ws, seq0, row0, nw);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sel_scan(const ScanArgs& a, float* ws_mem, hipStream_t s) {
  if (!a.rows || !a.D) return hipSuccess;
  return with_type(a.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    size_t row0 = 0;
    for (size_t q = 0; q < a.seqs; q += kSeqs) {
      SeqTab t;
      int tiles = 0;
      const int n = static_cast<int>(a.seqs - q < kSeqs ? a.seqs - q : kSeqs);
      const ScanPlan plan = scan_plan(a, q, n);
      const size_t rows = fill_seqs(t, a.lens, a.rows, a.seqs, q, n, plan.chunk, &tiles);
      if (tiles) {
        ScanWs ws{};
        ws.chunk = plan.chunk;
        if (plan.split) {
          ws.ends = ws_mem;
          ws.steps = ws_mem + static_cast<size_t>(tiles) * a.N * a.D;
        }
        const hipError_t e = a.N <= 4   ? scan_launch<DT, 4>(a, t, ws, q, row0, tiles, s)
                             : a.N <= 8 ? scan_launch<DT, 8>(a, t, ws, q, row0, tiles, s)
                                        : scan_launch<DT, 16>(a, t, ws, q, row0, tiles, s);
        if (e != hipSuccess) return e;
      }
      row0 += rows;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
