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

__device__ __forceinline__ void store_as(void* p, int dtype, size_t i, float v) {
  if (dtype == kF32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == kBF16)
    static_cast<uint16_t*>(p)[i] = Elem<kBF16>::down(v);
  else
    static_cast<uint16_t*>(p)[i] = Elem<kF16>::down(v);
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));

__device__ __forceinline__ uint32_t rotr(uint32_t w, int n) { return __builtin_amdgcn_alignbit(w, w, n); }

// How a type's rows enter the matrix instructions. A code q is made a 16-bit float without a conversion:
// its four bits are set into the mantissa of `base`, which makes it base + q, exact; base + z times the
// sum of the inputs is taken off the group's sum again. int8 rows take the code itself.
template <int DT> struct Mat;
template <> struct Mat<kBF16> {
  static constexpr uint32_t bits = 0x41804180;  // 16: steps of 1/8, so a code sits at bits 3..6
  static constexpr float base = 16.0f;
  using Acc = f32x4;
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t one = 0x3F803F80;
};
template <> struct Mat<kF16> {
  static constexpr uint32_t bits = 0x58005800;  // 128: steps of 1/8
  static constexpr float base = 128.0f;
  using Acc = f32x4;
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t one = 0x3C003C00;
};
template <> struct Mat<kI8> {
  using Acc = i32x4;
  static constexpr uint32_t one = 0x01010101;
};
template <> struct Mat<kF32> : Mat<kBF16> {};  // three bf16 parts

// The matrix operand of a word's 8 codes (16-bit floats), elements in order.
template <int DT>
__device__ __forceinline__ u32x4 w4_operand(uint32_t w) {
  constexpr uint32_t m = 0x00780078, b = Mat<DT>::bits;
  return u32x4{(w & m) | b, ((w >> 4) & m) | b, ((w >> 8) & m) | b, (rotr(w, 12) & m) | b};
}
// ... and as 8 bytes, elements 0 4 1 5 | 2 6 3 7; i8_operand puts the rows' bytes in that order.
__device__ __forceinline__ void w4_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = (w >> 3) & 0x0F0F0F0F;
  hi = rotr(w, 7) & 0x0F0F0F0F;
}
__device__ __forceinline__ void i8_operand(uint32_t x0, uint32_t x1, uint32_t& lo, uint32_t& hi) {
  lo = __builtin_amdgcn_perm(x1, x0, 0x05010400);
  hi = __builtin_amdgcn_perm(x1, x0, 0x07030602);
}

// 16 bytes of a row of 16-bit elements (8) or bytes (16) from element k, zeros behind K.
template <int DT>
__device__ __forceinline__ u32x4 row_16B(const char* row, int k, int K, bool whole) {
  constexpr int ES = DT == kI8 ? 1 : 2, V = 16 / ES;
  if (whole || k + V <= K) return *reinterpret_cast<const u32x4u*>(row + static_cast<size_t>(k) * ES);
  u32x4 v = {0, 0, 0, 0};
  for (int i = 0; i < V; ++i)
    if (k + i < K) {
      const uint32_t e = ES == 1 ? *reinterpret_cast<const uint8_t*>(row + k + i)
                                 : *reinterpret_cast<const uint16_t*>(row + 2 * static_cast<size_t>(k + i));
      v[i * ES / 4] |= e << (8 * (i * ES % 4));
    }
  return v;
}

// Few rows: one pass over the weights, bound by reading them. A block's waves split the chunks of NT
// tiles of 16 outputs; each wave reads its 1 KB of codes per tile and chunk straight into the matrix
// operand's place and multiplies it with CT column tiles. A column is a row, or for fp32 rows one of a row's
// three bf16 parts (hi + mid + lo = x exactly), 5 rows a tile: a wave cuts its chunk's rows into parts
// once, in LDS of its own. The waves' sums meet in LDS in one fixed order.
template <int DT> constexpr int kTileRows = DT == kF32 ? 5 : 16;
constexpr int kPartStride = 272;  // bytes of a column's 128 parts in LDS, 16 apart in banks
template <int DT, int CT> constexpr int kPartBytes = DT == kF32 ? CT * 15 * kPartStride : 0;

template <int DT, int STEP, int NT, int CT>
__global__ __launch_bounds__(CT == 1 ? 1024 : 512) void k_w4_rows(W4Args a, W4Geom g, const uint32_t* codes,
                                                                      const uint32_t* scales) {
  using M = Mat<DT>;
  using Acc = typename M::Acc;
  constexpr int S = 128 / STEP, R = kTileRows<DT>;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int col = lane & 15, q = lane >> 4;
  const int row0 = blockIdx.y * (CT * R), rows = min(static_cast<int>(a.rows) - row0, CT * R);
  const int tile0 = blockIdx.x * NT;
  const size_t es = DT == kF32 ? 4 : DT == kI8 ? 1 : 2;
  const char* x0 = static_cast<const char*>(a.x) + static_cast<size_t>(row0) * a.ldx * es;
  char* part = lds + wave * kPartBytes<DT, CT>;

  const char* xr[CT];  // this lane's row of each column tile (a row past the end repeats the last one)
#pragma unroll
  for (int t = 0; t < CT; ++t) xr[t] = x0 + static_cast<size_t>(min(t * R + (DT == kF32 ? 0 : col), rows - 1)) * a.ldx * es;
  const uint32_t* cw[NT];
  const uint32_t* sw[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const size_t tile = min(tile0 + n, g.nt - 1);
    cw[n] = codes + tile * g.nc * 256 + lane * 4;
    sw[n] = scales + tile * g.ns * 16 + q * 4;
  }

  f32x4 acc[NT][CT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[n][t] = f32x4{0, 0, 0, 0};

  u32x4 w[NT], sz[NT][S];
  auto fetch = [&](int c) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      w[n] = *reinterpret_cast<const u32x4*>(cw[n] + static_cast<size_t>(c) * 256);
#pragma unroll
      for (int s = 0; s < S; ++s) sz[n][s] = *reinterpret_cast<const u32x4*>(sw[n] + (static_cast<size_t>(c) * S + s) * 16);
    }
  };
  int c = wave;
  if (c < g.nc) fetch(c);
  for (; c < g.nc; c += waves) {
    const bool whole = (c + 1) * 128 <= g.K;
    u32x4 cur[NT], csz[NT][S];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      cur[n] = w[n];
#pragma unroll
      for (int s = 0; s < S; ++s) csz[n][s] = sz[n][s];
    }
    // the rows' operands of this chunk
    u32x4 b[CT][4];
    if constexpr (DT == kF32) {
      for (int r = 0; r < rows; ++r) {  // two neighbours a lane, three parts each
        const float* p = reinterpret_cast<const float*>(x0) + r * a.ldx + c * 128 + 2 * lane;
        const int k = c * 128 + 2 * lane;
        float v[2];
        if (whole) {
          const f32x2u u = *reinterpret_cast<const f32x2u*>(p);
          v[0] = u.x;
          v[1] = u.y;
        } else {
          v[0] = k < g.K ? p[0] : 0.0f;
          v[1] = k + 1 < g.K ? p[1] : 0.0f;
        }
        uint32_t h[2], m[2], l[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // cut off, not rounded: each part is exact, and what is left is too
          h[i] = __builtin_bit_cast(uint32_t, v[i]) & 0xFFFF0000u;
          const float r1 = v[i] - __builtin_bit_cast(float, h[i]);
          m[i] = __builtin_bit_cast(uint32_t, r1) & 0xFFFF0000u;
          l[i] = __builtin_bit_cast(uint32_t, r1 - __builtin_bit_cast(float, m[i]));
        }
        char* to = part + (r / 5 * 15 + r % 5 * 3) * kPartStride + 4 * lane;
        *reinterpret_cast<uint32_t*>(to) = (h[0] >> 16) | h[1];
        *reinterpret_cast<uint32_t*>(to + kPartStride) = (m[0] >> 16) | m[1];
        *reinterpret_cast<uint32_t*>(to + 2 * kPartStride) = (l[0] >> 16) | (l[1] & 0xFFFF0000u);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          b[t][j] = *reinterpret_cast<const u32x4*>(part + (t * 15 + min(col, 14)) * kPartStride + 2 * w4_k(STEP, j, q));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else if constexpr (DT == kI8) {
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {  // two words' 16 inputs: neighbours, or with steps of 32 two runs of 8
          u32x4 v;
          if constexpr (STEP == 32) {
            const u32x4 v0 = row_16B<DT>(xr[t], c * 128 + w4_k(STEP, j, q), g.K, whole),
                        v1 = row_16B<DT>(xr[t], c * 128 + w4_k(STEP, j + 1, q), g.K, whole);
            v = u32x4{v0.x, v0.y, v1.x, v1.y};
          } else {
            v = row_16B<DT>(xr[t], c * 128 + w4_k(STEP, j, q), g.K, whole);
          }
          uint32_t lo0, hi0, lo1, hi1;
          i8_operand(v.x, v.y, lo0, hi0);
          i8_operand(v.z, v.w, lo1, hi1);
          b[t][j / 2] = u32x4{lo0, hi0, lo1, hi1};
        }
    } else {
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) b[t][j] = row_16B<DT>(xr[t], c * 128 + w4_k(STEP, j, q), g.K, whole);
    }
    if (c + waves < g.nc) fetch(c + waves);

#pragma unroll
    for (int s = 0; s < S; ++s) {
      // sums of this scale's inputs: the codes' products, and the inputs themselves
      Acc d[NT][CT], sum[CT];
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        sum[t] = Acc{};
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n][t] = Acc{};
      }
      if constexpr (DT == kI8) {
        constexpr uint32_t one = M::one;
        if constexpr (STEP == 32) {  // one word a scale: 32 inputs an instruction
          const int j = s;
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            const long bx = (j & 1) ? (static_cast<long>(b[t][j / 2].w) << 32 | b[t][j / 2].z)
                                    : (static_cast<long>(b[t][j / 2].y) << 32 | b[t][j / 2].x);
            sum[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(static_cast<long>(one) << 32 | one, bx, sum[t], 0, 0, 0);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t lo, hi;
              w4_bytes(cur[n][j], lo, hi);
              d[n][t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(static_cast<long>(hi) << 32 | lo, bx, d[n][t], 0, 0, 0);
            }
          }
        } else {
#pragma unroll
          for (int jj = 0; jj < 2 / S; ++jj) {
            const int j = s * (2 / S) + jj;
            i32x4 aw[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t lo0, hi0, lo1, hi1;
              w4_bytes(cur[n][2 * j], lo0, hi0);
              w4_bytes(cur[n][2 * j + 1], lo1, hi1);
              aw[n] = __builtin_bit_cast(i32x4, u32x4{lo0, hi0, lo1, hi1});
            }
#pragma unroll
            for (int t = 0; t < CT; ++t) {
              const i32x4 bx = __builtin_bit_cast(i32x4, b[t][j]);
              sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, u32x4{one, one, one, one}), bx,
                                                             sum[t], 0, 0, 0);
#pragma unroll
              for (int n = 0; n < NT; ++n) d[n][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(aw[n], bx, d[n][t], 0, 0, 0);
            }
          }
        }
      } else {
        constexpr uint32_t one = M::one;
#pragma unroll
        for (int jj = 0; jj < 4 / S; ++jj) {
          const int j = s * (4 / S) + jj;
          u32x4 aw[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) aw[n] = w4_operand<DT>(cur[n][j]);
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            sum[t] = M::mul(u32x4{one, one, one, one}, b[t][j], sum[t]);
#pragma unroll
            for (int n = 0; n < NT; ++n) d[n][t] = M::mul(aw[n], b[t][j], d[n][t]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // output 4 q + i of the tile
          const uint32_t v = csz[n][s][i];
          const float sc = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v)));
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            if constexpr (DT == kI8) {
              acc[n][t][i] = __builtin_fmaf(sc, static_cast<float>(d[n][t][i] - static_cast<int>(v >> 16) * sum[t][i]),
                                            acc[n][t][i]);
            } else {
              const float z = static_cast<float>(v >> 16) + M::base;
              acc[n][t][i] = __builtin_fmaf(sc, __builtin_fmaf(-z, sum[t][i], d[n][t][i]), acc[n][t][i]);
            }
          }
        }
    }
  }

  // the waves' sums, added in the order of the waves
  __syncthreads();
  f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < CT; ++t) red[((wave * NT + n) * CT + t) * 64 + lane] = acc[n][t];
  __syncthreads();
  const float* sums = reinterpret_cast<const float*>(lds);
  for (int i = threadIdx.x; i < NT * 16 * rows; i += blockDim.x) {
    const int n = i % (NT * 16), r = i / (NT * 16), t = r / R;
    if (tile0 * 16 + n >= g.N) continue;
    const int at = (((n / 16) * CT + t) * 64 + (n % 16 / 4) * 16) * 4 + n % 4;
    float v = 0.0f;
    for (int wv = 0; wv < waves; ++wv) {
      const float* p = sums + wv * (NT * CT * 256) + at;
      if constexpr (DT == kF32) {
        const int c0 = r % 5 * 3;  // the small parts first
        v += (p[(c0 + 2) * 4] + p[(c0 + 1) * 4]) + p[c0 * 4];
      } else {
        v += p[r % 16 * 4];
      }
    }
    if constexpr (DT == kI8) v *= a.xscales[row0 + r];
    store_as(a.out, a.out_dtype, static_cast<size_t>(row0 + r) * a.ldo + tile0 * 16 + n, v);
  }
}

template <int DT, int STEP, int NT, int CT>
hipError_t rows_launch(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, int waves,
                       hipStream_t s) {
  const size_t part = static_cast<size_t>(waves) * kPartBytes<DT, CT>, red = static_cast<size_t>(waves) * NT * CT * 1024;
  const size_t lds = part > red ? part : red;  // at most 64 KB: 16 waves of one column tile, 8 of two
  auto* k = k_w4_rows<DT, STEP, NT, CT>;
  const unsigned per = CT * kTileRows<DT>;
  k<<<dim3((g.nt + NT - 1) / NT, static_cast<unsigned>((a.rows + per - 1) / per)), waves * 64, lds, s>>>(a, g, codes, scales);
  return hipGetLastError();
}

template <int DT, int STEP>
hipError_t rows_pick(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, hipStream_t s) {
  const int R = kTileRows<DT>;
  const int ct = a.rows <= static_cast<size_t>(R) ? 1 : 2;
  const size_t groups = (a.rows + ct * R - 1) / (ct * R);
  const int nt = g.nt * groups >= 512 ? 2 : 1;
  const size_t blocks = (g.nt + nt - 1) / nt * groups;
  int waves = ct == 1 ? 16 : 8;
  while (waves > 1 && (blocks * waves > 8192 || waves > g.nc)) waves /= 2;
  if (ct == 1) return nt == 1 ? rows_launch<DT, STEP, 1, 1>(a, g, codes, scales, waves, s)
                              : rows_launch<DT, STEP, 2, 1>(a, g, codes, scales, waves, s);
  return nt == 1 ? rows_launch<DT, STEP, 1, 2>(a, g, codes, scales, waves, s)
                 : rows_launch<DT, STEP, 2, 2>(a, g, codes, scales, waves, s);
}

template <int DT>
hipError_t rows_step(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, hipStream_t s) {
  return g.step == 32 ? rows_pick<DT, 32>(a, g, codes, scales, s)
         : g.step == 64 ? rows_pick<DT, 64>(a, g, codes, scales, s) : rows_pick<DT, 128>(a, g, codes, scales, s);
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
  constexpr size_t kMost = 65535;  // rows of a launch: the grid's second dimension
  for (size_t r = 0; r < a.rows; r += kMost) {
    W4Args b = a;
    b.rows = a.rows - r < kMost ? a.rows - r : kMost;
    b.x = static_cast<const char*>(a.x) + r * a.ldx * dtype_size(a.dtype);
    b.out = static_cast<char*>(a.out) + r * a.ldo * dtype_size(a.out_dtype);
    if (a.xscales) b.xscales = a.xscales + r;
    const hipError_t e = a.dtype == kF32    ? rows_step<kF32>(b, g, codes, scales, s)
                         : a.dtype == kBF16 ? rows_step<kBF16>(b, g, codes, scales, s)
                         : a.dtype == kF16  ? rows_step<kF16>(b, g, codes, scales, s)
                                            : rows_step<kI8>(b, g, codes, scales, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mmf
