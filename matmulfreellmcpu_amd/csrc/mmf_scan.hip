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
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
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

// A in powers of two; infinities as the outermost finite values, so that a step of 0 has the decay 1 with them too
// (the steps that stand behind a sequence's end are such ones).
__device__ __forceinline__ float log2_decay(float A) {
  A *= 1.44269504f;
  return A < -3.4e38f ? -3.4e38f : A > 3.4e38f ? 3.4e38f : A;
}

// A lane holds a channel's NS states in registers; a wave is 64 channels, and NW waves share a channel
// with more states. Every lane needs the same B and C of a step: a block keeps kTile steps of them in LDS as
// fp32 and reads them four at a time, all lanes one address; the next tile's are in flight meanwhile.
//
// What bounds it: the vector ALUs. A step of a state is an exponential (8.6 cycles a wave, measured) and 4
// other operations (4.3 each), 26 cycles for 64 channels, and a step of a channel some 180 more.
//
// Long sequences are cut into chunks so that the chip is full: kSum finds each chunk's end state from
// zeros and the sum of its steps (the decay over a chunk is exp(A * sum dt)), k_carry makes the states
// before each chunk of these, in order, and kApply starts each chunk there and writes the outputs. The first
// chunk of kSum starts from the state itself. A sequence's last chunk needs no sums: its slot of the
// workspace keeps the state at the start, which kApply's last chunk overwrites in `state`. kSum also leaves
// the steps themselves (softplus and all), where the workspace holds them. (kApply folding the chunks before
// its own by itself waits a load's time for each: 2048 x 4096 x 16 fp32 113 us, with k_carry 90.) That case
// takes 34.5 us for kSum, 5.5 for k_carry and 40 for kApply now, their vector ALUs busy 0.86 and 0.69 of the time.
constexpr int kTile = 32, kAhead = 4;
enum ScanPass { kSum = 0, kApply = 1 };

struct ScanWs {
  float* ends;  // [chunk][N][D], or null: sequences in one piece
  float* sums;  // [chunk][D]
  float* dt;    // [row][D], or null
  int chunk;    // rows of a chunk
};

template <int DT, int NS, int NW, int PASS>
__global__ __launch_bounds__(NW == 8 ? 512 : 256) void k_scan(ScanArgs a, SeqTab t, ScanWs ws, size_t seq0, size_t row0) {
  using E = Elem<DT>;
  using T = typename E::T;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int CW = NW >= 4 ? 1 : 4 / NW, NP = NW * NS;        // waves of other channels, padded states
  constexpr int kUnit = NS < 8 ? NS : 8, kUnits = NS / kUnit;
  constexpr int kRows = 64 * CW / NS, kIter = (kTile + kRows - 1) / kRows;  // steps that the block stages at a time
  __shared__ __align__(16) float sB[kTile * NP], sC[PASS == kApply ? kTile * NP : 4];
  __shared__ float sy[PASS == kApply && NW > 1 ? CW : 1][2][NW][kAhead][64];
  const TileAt at = tile_at(t, blockIdx.x);
  const int chunks = (at.len + ws.chunk - 1) / ws.chunk;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave % NW, cwave = wave / NW;
  const int N = static_cast<int>(a.N), n0 = part * NS;
  // A row's address is uniform and a lane adds its channel to it.
  const size_t D = a.D;
  const uint32_t dd = (blockIdx.y * CW + cwave) * 64 + lane, d = min(dd, static_cast<uint32_t>(D) - 1);
  const bool live = dd < D;
  float* state = a.state ? a.state + (seq0 + at.seq) * a.N * D : nullptr;
  float* ends = ws.ends + static_cast<size_t>(blockIdx.x) * a.N * D;  // this chunk's slot

  const int p0 = at.k * ws.chunk, p1 = min(p0 + ws.chunk, at.len);
  const size_t r0 = row0 + at.row;
  const T* up = static_cast<const T*>(a.u) + r0 * a.ldu;
  const T* dp = static_cast<const T*>(a.dt) + r0 * a.lddt;
  const T* zp = PASS == kApply && a.z ? static_cast<const T*>(a.z) + r0 * a.ldz : nullptr;
  T* out = static_cast<T*>(a.out) + r0 * a.ldo;
  float* wdt = ws.dt ? ws.dt + static_cast<size_t>(at.row) * D : nullptr;
  const bool ready = PASS == kApply && wdt;  // the steps are
  const float skip = a.skip ? a.skip[d] : 0.0f, bias = a.dt_bias ? a.dt_bias[d] : 0.0f;

  // the inputs of two groups of steps, each loaded two groups ahead: a load takes longer than a group
  struct Inputs {
    T u[kAhead], dt[kAhead], z[kAhead];
    float step[kAhead];
  };
  Inputs in[2] = {};
  auto fetch = [&](Inputs& g, int p) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const size_t r = min(p + i, p1 - 1);
      g.u[i] = (up + r * a.ldu)[d];
      if (ready)
        g.step[i] = (wdt + r * D)[d];
      else
        g.dt[i] = (dp + r * a.lddt)[d];
      if (zp) g.z[i] = (zp + r * a.ldz)[d];
    }
  };
  auto step_of = [&](const Inputs& g, int i) {
    if (ready) return g.step[i];
    const float v = E::up(g.dt[i]) + bias;
    return a.softplus ? softplus(v) : v;
  };
  fetch(in[0], p0);
  if (p0 + kAhead < p1) fetch(in[1], p0 + kAhead);

  if (PASS == kSum && at.k == chunks - 1) {  // no sums of the last chunk: its slot keeps the state
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (live && n0 + i < N) (ends + (n0 + i) * D)[d] = state ? (state + (n0 + i) * D)[d] : 0.0f;
    for (int p = p0; wdt && part == 0 && p < p1; p += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (live && p + i < p1) (wdt + static_cast<size_t>(p + i) * D)[d] = step_of(in[0], i);
      in[0] = in[1];
      fetch(in[1], p + 2 * kAhead);
    }
    return;
  }

  // a tile's B and C: thread i of the block takes state i % NP of every kRows-th step
  const int sn_ = threadIdx.x % NP, ss = threadIdx.x / NP;
  const T* Bp = static_cast<const T*>(a.B) + r0 * a.ldb + min(sn_, N - 1);
  const T* Cp = static_cast<const T*>(a.C) + r0 * a.ldc + min(sn_, N - 1);
  T bn[kIter], cn[kIter];
  auto fetch_tile = [&](int pt) {
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const size_t r = min(pt + ss + i * kRows, p1 - 1);
      bn[i] = Bp[r * a.ldb];
      if (PASS == kApply) cn[i] = Cp[r * a.ldc];
    }
  };
  fetch_tile(p0);

  // (loads without conditions, so that all are in flight together: what stands past N is not used)
  float A[NS], h[NS];
  const float* Ap = a.A + static_cast<size_t>(d) * a.N;
  if (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NS; i += 4) {
      const f4u v = *reinterpret_cast<const f4u*>(Ap + min(n0 + i, N - 4));
#pragma unroll
      for (int k = 0; k < 4; ++k) A[i + k] = v[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i) A[i] = Ap[min(n0 + i, N - 1)];
  }
  const float* hp = PASS == kApply && ws.ends ? ends : at.k == 0 ? state : nullptr;
  if (hp) {
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = (hp + min(n0 + i, N - 1) * D)[d];
  }
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    A[i] = n0 + i < N ? log2_decay(A[i]) : 0.0f;
    if (!hp || n0 + i >= N) h[i] = 0.0f;
  }
  float total = 0.0f;
  int flip = 0;
  for (int pt = p0; pt < p1; pt += kTile) {
    const int steps = min(kTile, p1 - pt);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int s = ss + i * kRows;
      if (s < kTile) {  // what stands there for no step or state is multiplied by 0 and must be finite
        const bool in = s < steps && sn_ < N;
        sB[s * NP + sn_] = in ? E::up(bn[i]) : 0.0f;
        if (PASS == kApply) sC[s * NP + sn_] = in ? E::up(cn[i]) : 0.0f;
      }
    }
    __syncthreads();
    if (pt + kTile < p1) fetch_tile(pt + kTile);
    float bq[kUnit], cq[kUnit] = {};
    auto read = [&](int row, int n1) {
      const int from = row * NP + n0 + n1;
#pragma unroll
      for (int n = 0; n < kUnit; ++n) {
        bq[n] = sB[from + n];
        if (PASS == kApply) cq[n] = sC[from + n];
      }
    };
    read(0, 0);
    auto group = [&](Inputs& now, int g) {
      // Steps in a line, with no condition between them; the B and C of a unit of kUnit states are read before
      // the unit before it is computed. Steps past the end have dt = 0: the decay is 1 and nothing is added.
      const int left = steps - g;
      float u[kAhead], step[kAhead], z[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        u[i] = E::up(now.u[i]);
        step[i] = step_of(now, i);
        if (PASS == kSum && wdt && part == 0 && live && i < left) (wdt + static_cast<size_t>(pt + g + i) * D)[d] = step[i];
        if (i >= left) step[i] = u[i] = 0.0f;
        if (PASS == kApply) z[i] = E::up(now.z[i]);
      }
      fetch(now, pt + g + 2 * kAhead);
      float y[kAhead] = {};
#pragma unroll
      for (int k = 0; k < kAhead * kUnits; ++k) {
        const int i = k / kUnits, n1 = k % kUnits * kUnit;
        float b[kUnit], c[kUnit];
#pragma unroll
        for (int n = 0; n < kUnit; ++n) b[n] = bq[n], c[n] = cq[n];
        // the next unit's B and C (behind the tile's last step: the last one's, unused)
        if (k + 1 < kAhead * kUnits)
          read(g + (k + 1) / kUnits, (k + 1) % kUnits * kUnit);
        else
          read(min(g + kAhead, kTile - 1), 0);
        const float su = step[i] * u[i];
#pragma unroll
        for (int n = 0; n < kUnit; ++n) {
          h[n1 + n] = __builtin_fmaf(exp2_fast(step[i] * A[n1 + n]), h[n1 + n], su * b[n]);
          if (PASS == kApply) y[i] = __builtin_fmaf(c[n], h[n1 + n], y[i]);
        }
        if (PASS == kSum && n1 == 0) total += step[i];
        __builtin_amdgcn_sched_barrier(0);
      }
      if (PASS == kSum) return;
      if constexpr (NW > 1 && PASS == kApply) {  // the parts' sums in their order; part i % NW writes step i
#pragma unroll
        for (int i = 0; i < kAhead; ++i) sy[cwave][flip][part][i][lane] = y[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (i % NW != part) continue;
          y[i] = 0.0f;
#pragma unroll
          for (int w = 0; w < NW; ++w) y[i] += sy[cwave][flip][w][i][lane];
        }
        flip ^= 1;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (NW > 1 && i % NW != part) continue;
        float o = __builtin_fmaf(skip, u[i], y[i]);
        if (zp) o *= silu_fast(z[i]);
        if (live && i < left) (out + static_cast<size_t>(pt + g + i) * a.ldo)[d] = E::down(o);
      }
    };
    for (int g = 0; g < steps; g += 2 * kAhead) {
      group(in[0], g);
      __builtin_amdgcn_sched_barrier(0);
      if (g + kAhead < steps) {
        group(in[1], g + kAhead);
      } else {
        in[0] = in[1];  // an odd number of groups: only a sequence's end
      }
    }
  }
  if (!live) return;
  if (PASS == kSum) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < N) (ends + (n0 + i) * D)[d] = h[i];
    if (part == 0) (ws.sums + static_cast<size_t>(blockIdx.x) * D)[d] = total;
  } else if (state && at.k == chunks - 1) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < N) (state + (n0 + i) * D)[d] = h[i];
  }
}

// The state before each chunk in the place of each chunk's end state: a thread a state of a channel, one
// sequence a row of blocks, kBatch chunks' loads in flight.
__global__ __launch_bounds__(256) void k_carry(ScanArgs a, SeqTab t, ScanWs ws) {
  constexpr int kBatch = 16;
  const size_t D = a.D, i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const int len = t.len > 0 ? t.len : t.row[blockIdx.y + 1] - t.row[blockIdx.y];
  const int chunks = (len + ws.chunk - 1) / ws.chunk;
  if (i >= D * a.N || chunks < 2) return;
  const size_t first = t.len > 0 ? static_cast<size_t>(blockIdx.y) * t.tiles : t.tile[blockIdx.y];
  const size_t n = i / D, d = i - n * D;
  const float A = log2_decay(a.A[d * a.N + n]);
  float* ends = ws.ends + first * a.N * D + i;
  const float* sums = ws.sums + first * D + d;
  const size_t step = a.N * D;
  float h = ends[(chunks - 1) * step];  // the state at the start
  for (int j = 0; j < chunks; j += kBatch) {
    float e[kBatch], s[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const size_t at = min(j + k, chunks - 1);  // (the last chunk's are not used)
      e[k] = ends[at * step];
      s[k] = sums[min(j + k, chunks - 2) * D];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (j + k >= chunks) break;
      ends[(j + k) * step] = h;
      // The first chunk's end has the state in it. A state of 0 stays out of the product: a growing one's factor
      // (A above 0) may be infinite over a chunk where no step's is.
      h = j + k && h != 0.0f ? __builtin_fmaf(exp2_fast(s[k] * A), h, e[k]) : e[k];
    }
  }
}

template <int DT, int NS, int NW>
hipError_t scan_launch(const ScanArgs& a, const SeqTab& t, const ScanWs& ws, size_t seq0, size_t row0, int tiles,
                       hipStream_t s) {
  constexpr int CW = NW >= 4 ? 1 : 4 / NW;
  const dim3 grid(tiles, static_cast<unsigned>((a.D + CW * 64 - 1) / (CW * 64)));
  if (ws.ends) {
    k_scan<DT, NS, NW, kSum><<<grid, NW * CW * 64, 0, s>>>(a, t, ws, seq0, row0);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_carry<<<dim3(static_cast<unsigned>((a.N * a.D + 255) / 256), t.n), 256, 0, s>>>(a, t, ws);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  k_scan<DT, NS, NW, kApply><<<grid, NW * CW * 64, 0, s>>>(a, t, ws, seq0, row0);
  return hipGetLastError();
}

// One row of each sequence: bound by reading and writing the states. A block is 64 channels, a wave NQ of their
// states; it goes through `per` sequences with the decay rates in registers (their rows of N floats are
// the dearest to read: 64 cache lines a load), the next sequence's state in flight. B and C are one
// load a wave, handed out by v_readlane. The waves' sums meet in LDS. 64 x 5120 x 16 bf16, 45 MB: 11.2 us, 4.0 TB/s
// (by k_scan, whose registers leave half the waves, 19); one sequence of 2048 channels 4.5, a launch.
constexpr int kStepSeqs = 8;  // most sequences of a block
template <int DT, int NQ>
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs a, size_t seq0, size_t row0, int seqs, int per) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float sy[kStepSeqs][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int N = static_cast<int>(a.N), n0 = wave * NQ;
  const size_t D = a.D;
  const uint32_t dd = blockIdx.y * 64 + lane, d = min(dd, static_cast<uint32_t>(D) - 1);
  const bool live = dd < D;
  const int q0 = blockIdx.x * per, q1 = min(q0 + per, seqs);
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f;

  struct Inputs {
    T u, dt, bc;
    float h[NQ];
  };
  auto fetch = [&](Inputs& in, int q) {
    const size_t r = row0 + q;
    in.u = (static_cast<const T*>(a.u) + r * a.ldu)[d];
    in.dt = (static_cast<const T*>(a.dt) + r * a.lddt)[d];
    const int n = min(n0 + (lane & (NQ - 1)), N - 1);
    in.bc = lane & NQ ? (static_cast<const T*>(a.C) + r * a.ldc)[n] : (static_cast<const T*>(a.B) + r * a.ldb)[n];
    if (a.state) {
      const float* h = a.state + (seq0 + q) * N * D;
#pragma unroll
      for (int i = 0; i < NQ; ++i) in.h[i] = (h + min(n0 + i, N - 1) * D)[d];
    }
  };
  Inputs now, next = {};
  fetch(next, q0);
  float A[NQ];
  const float* Ap = a.A + static_cast<size_t>(d) * N;
  if (NQ >= 4 && N % 4 == 0) {
    typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int i = 0; i < NQ; i += 4) {
      const f4u v = *reinterpret_cast<const f4u*>(Ap + min(n0 + i, N - 4));
#pragma unroll
      for (int k = 0; k < 4 && i + k < NQ; ++k) A[i + k] = log2_decay(v[k]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NQ; ++i) A[i] = log2_decay(Ap[min(n0 + i, N - 1)]);
  }
  T uo[kStepSeqs / 4], zo[kStepSeqs / 4] = {};  // of the outputs that this wave writes
#pragma unroll
  for (int k = 0; k < kStepSeqs / 4; ++k) {
    const size_t r = row0 + min(q0 + wave + 4 * k, q1 - 1);
    uo[k] = (static_cast<const T*>(a.u) + r * a.ldu)[d];
    if (a.z) zo[k] = (static_cast<const T*>(a.z) + r * a.ldz)[d];
  }
  for (int q = q0; q < q1; ++q) {
    now = next;
    if (q + 1 < q1) fetch(next, q + 1);
    const float u = E::up(now.u), v = E::up(now.dt) + bias, step = a.softplus ? softplus(v) : v, su = step * u;
    const float bc = E::up(now.bc);
    float y = 0.0f;
    float* h = a.state + (seq0 + q) * N * D;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if (n0 + i >= N) break;
      const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bc), i));
      const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bc), NQ + i));
      const float old = a.state ? now.h[i] : 0.0f;
      const float x = __builtin_fmaf(exp2_fast(step * A[i]), old, su * b);
      y = __builtin_fmaf(c, x, y);
      if (a.state && live) (h + (n0 + i) * D)[d] = x;
    }
    sy[q - q0][wave][lane] = y;
  }
  __syncthreads();
  if (!live) return;
  const float skip = a.skip ? a.skip[d] : 0.0f;
#pragma unroll
  for (int k = 0; k < kStepSeqs / 4; ++k) {
    const int q = q0 + wave + 4 * k;
    if (q >= q1) break;
    float y = (sy[q - q0][0][lane] + sy[q - q0][1][lane]) + (sy[q - q0][2][lane] + sy[q - q0][3][lane]);
    y = __builtin_fmaf(skip, E::up(uo[k]), y);
    if (a.z) y *= silu_fast(E::up(zo[k]));
    (static_cast<T*>(a.out) + (row0 + q) * a.ldo)[d] = E::down(y);
  }
}

template <int DT>
hipError_t step_launch(const ScanArgs& a, size_t seq0, size_t row0, int seqs, hipStream_t s) {
  const unsigned cols = static_cast<unsigned>((a.D + 63) / 64);
  // as many sequences a block as leave two blocks for each compute unit
  int per = kStepSeqs;
  while (per > 1 && static_cast<size_t>(cols) * ((seqs + per - 1) / per) < 512) per /= 2;
  const dim3 grid((seqs + per - 1) / per, cols);
  if (a.N <= 4)
    k_scan_step<DT, 1><<<grid, 256, 0, s>>>(a, seq0, row0, seqs, per);
  else if (a.N <= 8)
    k_scan_step<DT, 2><<<grid, 256, 0, s>>>(a, seq0, row0, seqs, per);
  else if (a.N <= 16)
    k_scan_step<DT, 4><<<grid, 256, 0, s>>>(a, seq0, row0, seqs, per);
  else if (a.N <= 32)
    k_scan_step<DT, 8><<<grid, 256, 0, s>>>(a, seq0, row0, seqs, per);
  else if (a.N <= 64)
    k_scan_step<DT, 16><<<grid, 256, 0, s>>>(a, seq0, row0, seqs, per);
  else
    k_scan_step<DT, 32><<<grid, 256, 0, s>>>(a, seq0, row0, seqs, per);
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
      if (one_row_each(a.lens, a.rows, a.seqs, q, n)) {
        const hipError_t e = step_launch<DT>(a, q, row0, n, s);
        if (e != hipSuccess) return e;
        row0 += n;
        continue;
      }
      const ScanPlan plan = scan_plan(a, q, n);
      const size_t rows = fill_seqs(t, a.lens, a.rows, a.seqs, q, n, plan.chunk, &tiles);
      if (tiles) {
        ScanWs ws{};
        ws.chunk = plan.chunk;
        if (plan.split) {
          ws.ends = ws_mem;
          ws.sums = ws_mem + static_cast<size_t>(tiles) * a.N * a.D;
          if (rows * a.D <= kLayerWsBytes / 4 - kScanWsFloats) ws.dt = ws_mem + kScanWsFloats;
        }
        const hipError_t e = a.N <= 4    ? scan_launch<DT, 4, 1>(a, t, ws, q, row0, tiles, s)
                             : a.N <= 8  ? scan_launch<DT, 8, 1>(a, t, ws, q, row0, tiles, s)
                             : a.N <= 16 ? scan_launch<DT, 16, 1>(a, t, ws, q, row0, tiles, s)
                             : a.N <= 32 ? scan_launch<DT, 16, 2>(a, t, ws, q, row0, tiles, s)
                             : a.N <= 64 ? scan_launch<DT, 16, 4>(a, t, ws, q, row0, tiles, s)
                                         : scan_launch<DT, 16, 8>(a, t, ws, q, row0, tiles, s);
        if (e != hipSuccess) return e;
      }
      row0 += rows;
    }
    return hipSuccess;
  });
}

}  // namespace mmf
