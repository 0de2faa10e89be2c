// mmf_w8.hip -- products of int8 rows and int8 weights, with a scale a row and a scale an output.
//
// out[r, n] = xs[r] ws[n] sum_k x[r, k] w[n, k] + bias[n]. The sums are exact in int32, in any order; an output takes
// three fp32 roundings and its type's. Weights stand as matrix operands (mmf_layer8.hpp) and are the matrix
// instruction's first operand, so that a lane's sums are neighbouring outputs of one row.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v4iu __attribute__((ext_vector_type(4), aligned(1)));
typedef int v16i __attribute__((ext_vector_type(16)));

// codes [N, K] -> the layout, a thread 16 neighbouring inputs of an output, with zeros behind the weights.
__global__ __launch_bounds__(256) void k_w8_pack(const int8_t* codes, W8Geom g, int8_t* out) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<size_t>(g.nt) * g.nk * 64) return;
  const size_t run = i >> 6, n = run / g.nk * 32 + i % 32;
  const int k0 = static_cast<int>(run % g.nk) * 32 + 16 * (i >> 5 & 1);
  int8_t* to = out + w8_at(g, n, k0);
#pragma unroll
  for (int j = 0; j < 16; ++j)
    to[j] = n < static_cast<size_t>(g.N) && k0 + j < g.K ? codes[n * g.K + k0 + j] : static_cast<int8_t>(0);
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

// Few rows: 16 outputs of 16 FM rows a block; its waves share the inputs, U chunks of 64 at a time, all of whose loads are
// in flight together. Bound by the weights' way from memory: 24 x 6912 x 2560 (17.7 MB) 7.9 us, where a copy's rate gives 3.8;
// one row of 2048 x 11264, whose 23 MB a cache holds, 4.0. Blocks of 16 outputs, for as many as there can be.
constexpr int kRowWaves = 8;
template <int FM>
__global__ __launch_bounds__(64 * kRowWaves) void k_w8_rows(W8Args a, W8Geom g, const int8_t* codes, const float* scales) {
  constexpr int U = FM == 4 ? 2 : 4;
  __shared__ int sums[kRowWaves][FM][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const size_t r0 = static_cast<size_t>(blockIdx.y) * (16 * FM);
  const int8_t* w = codes + (static_cast<size_t>(blockIdx.x / 2) * g.nk * 64 + (blockIdx.x % 2 * 16 + c) + 32 * (q & 1)) * 16;
  const int8_t* x[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f) x[f] = a.x + min(r0 + 16 * f + c, a.rows - 1) * a.ldx;
  v4i acc[FM] = {};
  const int chunks = g.nk / 2;
  for (int ch = wave * U; ch < chunks; ch += kRowWaves * U) {
    v4i wv[U], xv[U][FM];
#pragma unroll
    for (int u = 0; u < U; ++u)  // (behind the last chunk its weights again, with inputs of 0)
      wv[u] = *reinterpret_cast<const v4i*>(w + static_cast<size_t>(2 * min(ch + u, chunks - 1) + (q >> 1)) * 1024);
    if (64 * (ch + U) <= g.K) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int f = 0; f < FM; ++f) xv[u][f] = *reinterpret_cast<const v4iu*>(x[f] + 64 * (ch + u) + 16 * q);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int f = 0; f < FM; ++f) xv[u][f] = load_x(x[f], 64 * (ch + u) + 16 * q, g.K);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < FM; ++f) acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u], xv[u][f], acc[f], 0, 0, 0);
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

// Many rows: a block of WN waves takes 32 FM rows and 32 FN outputs a wave. The rows go through LDS, as
// the matrix instruction takes them, a stage of 128 inputs ahead; a wave's weights go straight to its registers, also a
// stage ahead. One barrier a stage. With few tiles, KG such groups of waves share a tile's inputs: a stage takes as long as a
// load, however few rows it has. 2048 x 2048 x 11264: 59 us, 1600 TOP/s, with the matrix cores 0.46 busy: 704 tiles of 16
// stages each, two on a compute unit at a time, are less than one and a half rounds and as many first loads and last stores;
// 8192 x 8192 x 8192 reaches 2200. Tiles of 256 x 256 have the same rate, and no room for the loads ahead.
template <int FM, int FN, int WN, int KG>
struct W8Shape {
  static constexpr int kRows = 32 * FM, kCols = 32 * FN * WN, kWaves = WN, kThreads = 64 * kWaves;
  static constexpr int kStage = kRows * 128, kEach = kStage / 16 / kThreads;
  static constexpr int kOutRow = FN * 32 * 4 + 16, kOutBytes = 32 * kOutRow * kWaves;  // a wave's 32 rows on their way out
  static constexpr int kSums = FM * FN * 4096, kSumBytes = (KG - 1) * kWaves * kSums;  // of the groups but the first
  static constexpr int most(int a, int b) { return a > b ? a : b; }
  static constexpr int kLds = most(2 * kStage * KG, most(kOutBytes, kSumBytes));
};

template <int OT, int FM, int FN, int WN, int KG>
__global__ __launch_bounds__(64 * WN * KG, KG == 4 ? 4 : 2) void k_w8_tile(W8Args a, W8Geom g, const int8_t* codes, const float* scales) {
  using Sh = W8Shape<FM, FN, WN, KG>;
  using E = Elem<OT>;
  using T = typename E::T;
  constexpr int R = Sh::kEach;
  __shared__ __align__(16) char lds_all[Sh::kLds];
  const int lane = threadIdx.x & 63, half = lane >> 5, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = KG > 1 ? wid / Sh::kWaves : 0, wave = KG > 1 ? wid % Sh::kWaves : wid, tid = threadIdx.x - kg * Sh::kThreads;
  char* const lds = lds_all + kg * 2 * Sh::kStage;
  // Blocks go to the 8 XCDs in turn: each takes a run of tiles of its own, down the rows of a column of tiles, which share
  // its weights in that XCD's cache.
  const int nrt = static_cast<int>((a.rows + Sh::kRows - 1) / Sh::kRows), nct = (g.N + Sh::kCols - 1) / Sh::kCols;
  const int tiles = nrt * nct, share = (tiles + 7) / 8, tile = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if (static_cast<int>(blockIdx.x >> 3) >= share || tile >= tiles) return;
  const int r0 = tile % nrt * Sh::kRows, n0 = tile / nrt * Sh::kCols + wave * FN * 32;
  const int s1 = g.nk / 4, per = (s1 + KG - 1) / KG, s0 = kg * per;  // stages, a group's, and its first

  // this thread's share of a stage: 16 inputs (c) of row threadIdx.x / 8 + i kThreads / 8
  const int c = tid & 7, rr = tid >> 3;
  const int8_t* x[R];
  int to[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = rr + i * (Sh::kThreads / 8);
    x[i] = a.x + min(static_cast<size_t>(r0 + r), a.rows - 1) * a.ldx + 16 * c;
    // a fragment is 32 rows of 32 inputs, 1 KB; rows are turned against each other so that 8 neighbouring threads of a row, and
    // 8 rows of a fragment, use other LDS banks
    to[i] = ((c >> 1) * FM + (r >> 5)) * 1024 + (((r & 31) ^ c) + 32 * (c & 1)) * 16;
  }
  v4i xv[R];
  auto fetch_x = [&](int s) {
    if (128 * (s + 1) <= g.K) {
#pragma unroll
      for (int i = 0; i < R; ++i) xv[i] = *reinterpret_cast<const v4iu*>(x[i] + 128 * s);
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) xv[i] = load_x(x[i], 128 * s, g.K - 16 * c);
    }
  };
  auto store_x = [&](int b) {
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<v4i*>(lds + b * Sh::kStage + to[i]) = xv[i];
  };
  const int8_t* w[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) w[j] = codes + static_cast<size_t>(min(n0 / 32 + j, g.nt - 1)) * g.nk * 1024;
  v4i wv[4][FN];  // a stage's; each is loaded again for the next stage once it is used
  auto fetch_w = [&](int s, int k) {
#pragma unroll
    for (int j = 0; j < FN; ++j) wv[k][j] = *reinterpret_cast<const v4i*>(w[j] + static_cast<size_t>(4 * s + k) * 1024 + lane * 16);
  };
  v16i acc[FM][FN] = {};
  v4i xf[2][FM];
  const int from = (((lane & 31) ^ half) + 32 * half) * 16;  // its row is turned by 2 k more
  auto read_x = [&](v4i (&to)[FM], int b, int k) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
      to[i] = *reinterpret_cast<const v4i*>(lds + b * Sh::kStage + (k * FM + i) * 1024 + (from ^ (32 * k)));
  };
  {
    fetch_x(min(s0, s1 - 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) fetch_w(min(s0, s1 - 1), k);
    store_x(0);
    fetch_x(min(s0 + 1, s1 - 1));
    for (int t = 0, b = 0; t < per; ++t, b ^= 1) {
      const int s = s0 + t;
      __syncthreads();
      if (KG > 1 && s >= s1) continue;  // (the last group may have fewer)
      read_x(xf[0], b, 0);
      store_x(b ^ 1);  // (behind the last stage its rows again)
      fetch_x(min(s + 2, s1 - 1));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k < 3) read_x(xf[(k + 1) & 1], b, k + 1);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wv[k][j], xf[k & 1][i], acc[i][j], 0, 0, 0);
        fetch_w(min(s + 1, s1 - 1), k);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if constexpr (KG > 1) {  // the groups' sums, exact in any order, meet in the first
    __syncthreads();
    v4i* const at = reinterpret_cast<v4i*>(lds_all) + (wave * FM * FN * 4) * 64 + lane;
    constexpr int kStep = Sh::kWaves * FM * FN * 4 * 64;
    if (kg) {
#pragma unroll
      for (int i = 0; i < FM * FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          at[(kg - 1) * kStep + (i * 4 + q) * 64] =
              v4i{acc[i / FN][i % FN][4 * q], acc[i / FN][i % FN][4 * q + 1], acc[i / FN][i % FN][4 * q + 2], acc[i / FN][i % FN][4 * q + 3]};
    }
    __syncthreads();
    for (int o = 0; o < KG - 1 && !kg; ++o)
#pragma unroll
      for (int i = 0; i < FM * FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const v4i v = at[o * kStep + (i * 4 + q) * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i / FN][i % FN][4 * q + e] += v[e];
        }
    __syncthreads();  // the sums have been read
    if (kg) return;
  }
  // lane l has row l % 32 of a fragment and outputs 8 q + 4 (l / 32) + 0..3, q = 0..3
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  typedef T T4 __attribute__((ext_vector_type(4)));
  typedef T Tv __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  constexpr int V = 16 / sizeof(T), kLanes = FN * 32 / V;  // lanes of a row on its way out
  f4u sc[FN][4], bi[FN][4];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + j * 32 + 8 * q + 4 * half;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[j][q][e] = scales[min(n + e, g.N - 1)];
        bi[j][q][e] = a.bias ? a.bias[min(n + e, g.N - 1)] : 0.0f;
      }
    }
  if constexpr (KG == 1) __syncthreads();  // the stages have been read
  char* strip = lds_all + wave * 32 * Sh::kOutRow;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const float xs = a.xscales[min(static_cast<size_t>(r0 + i * 32 + (lane & 31)), a.rows - 1)];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = E::down(scaled(acc[i][j][4 * q + e], xs, sc[j][q][e], bi[j][q][e]));
        *reinterpret_cast<T4*>(strip + (lane & 31) * Sh::kOutRow + (j * 32 + 8 * q + 4 * half) * sizeof(T)) = o;
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < 32 * kLanes / 64; ++k) {
      const int r = k * (64 / kLanes) + lane / kLanes, at = lane % kLanes * V;
      const Tv v = *reinterpret_cast<const Tv*>(strip + r * Sh::kOutRow + at * sizeof(T));
      const size_t row = r0 + i * 32 + r;
      const int n = n0 + at;
      if (row >= a.rows) continue;
      T* out = static_cast<T*>(a.out) + row * a.ldo + n;
      if (n + V <= g.N) {
        *reinterpret_cast<Tv*>(out) = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (n + e < g.N) out[e] = v[e];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int FM, int FN, int WN, int KG>
hipError_t tile_launch(const W8Args& a, const W8Geom& g, const int8_t* codes, const float* scales, hipStream_t s) {
  using Sh = W8Shape<FM, FN, WN, KG>;
  const int nrt = static_cast<int>((a.rows + Sh::kRows - 1) / Sh::kRows), nct = (g.N + Sh::kCols - 1) / Sh::kCols;
  const unsigned grid = (nrt * nct + 7) / 8 * 8;
  return with_type(a.out_dtype, [&](auto ot) {
    k_w8_tile<decltype(ot)::value, FM, FN, WN, KG><<<grid, Sh::kThreads * KG, 0, s>>>(a, g, codes, scales);
    return hipGetLastError();
  });
}

template <int FM>
hipError_t rows_launch(const W8Args& a, const W8Geom& g, const int8_t* codes, const float* scales, hipStream_t s) {
  const dim3 grid((g.N + 15) / 16, static_cast<unsigned>((a.rows + 16 * FM - 1) / (16 * FM)));
  k_w8_rows<FM><<<grid, 64 * kRowWaves, 0, s>>>(a, g, codes, scales);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_w8_pack(const int8_t* codes, const W8Geom& g, int8_t* out, hipStream_t s) {
  const size_t n = static_cast<size_t>(g.nt) * g.nk * 64;
  k_w8_pack<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(codes, g, out);
  return hipGetLastError();
}

hipError_t launch_w8(const W8Args& all, const W8Geom& g, const int8_t* codes, const float* scales, hipStream_t s) {
  for (size_t r = 0; r < all.rows; r += kW8RowsMost) {
    W8Args a = all;
    a.rows = all.rows - r < kW8RowsMost ? all.rows - r : kW8RowsMost;
    a.x += r * all.ldx;
    a.xscales += r;
    a.out = static_cast<char*>(all.out) + r * all.ldo * dtype_size(all.out_dtype);
    hipError_t e = hipErrorInvalidValue;
    switch (w8_way(g, a.rows)) {
      case kW8Rows:
        e = a.rows <= 16   ? rows_launch<1>(a, g, codes, scales, s)
            : a.rows <= 32 ? rows_launch<2>(a, g, codes, scales, s)
                           : rows_launch<4>(a, g, codes, scales, s);
        break;
      case kW8Tile32x4: e = tile_launch<1, 1, 4, 4>(a, g, codes, scales, s); break;
      case kW8Tile32: e = tile_launch<1, 1, 4, 2>(a, g, codes, scales, s); break;
      case kW8Tile64: e = tile_launch<2, 1, 4, 2>(a, g, codes, scales, s); break;
      case kW8Tile128: e = tile_launch<4, 2, 4, 1>(a, g, codes, scales, s); break;
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mmf
