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
  out[i] = w;
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
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));

// The matrix operand of a word's 8 codes is q - z in every type, exact, so that a sum's roundings are those of its own
// terms. (As base + q, with base + z times the sum of the inputs taken off the group's sum, one input 1e4 times the
// others at weights of 0 left 1e-4 of the rest off, with a base of 128 for fp16 rows 1e-3; it is 1e-7 now.)
template <int DT> struct Mat;
template <> struct Mat<kBF16> {
  using Acc = f32x4;
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mat<kF16> {
  using Acc = f32x4;
  static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mat<kI8> {
  using Acc = i32x4;
};
template <> struct Mat<kF32> : Mat<kBF16> {};  // three bf16 parts

// A word's codes as 8 bytes, elements 0 4 1 5 | 2 6 3 7; i8_operand puts the rows' bytes in that order.
__device__ __forceinline__ void w4_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = w & 0x0F0F0F0F;
  hi = (w >> 4) & 0x0F0F0F0F;
}
__device__ __forceinline__ void i8_operand(uint32_t x0, uint32_t x1, uint32_t& lo, uint32_t& hi) {
  lo = __builtin_amdgcn_perm(x1, x0, 0x05010400);
  hi = __builtin_amdgcn_perm(x1, x0, 0x07030602);
}
// Four bytes: a code less its zero point, with b = 0x80 - z in each: their sum is at most 0x8F, so nothing carries.
__device__ __forceinline__ uint32_t less_bytes(uint32_t a, uint32_t b) { return (a + b) ^ 0x80808080u; }

// The zero point of a scale's word (above the scale) in the form that an operand takes it in: 1024 + z twice, or
// 0x80 - z four times.
template <int DT> __device__ __forceinline__ uint32_t zero_of(uint32_t scale) {
  if constexpr (DT == kF16) return 0x64006400u + __builtin_amdgcn_perm(0u, scale, 0x0C020C02);
  return 0x80808080u - __builtin_amdgcn_perm(0u, scale, 0x02020202);
}
// The operand of a word's 8 codes, elements in order.
//   fp16: a code's four bits are set into the mantissa of 1024 (steps of 1: bits 0..3), which makes it 1024 + q
//     without a conversion, and 1024 + z comes off: all exact.
//   bf16: bytes q - z, converted (an integer below 16 has few bits). bf16 has no subtraction of pairs here.
template <int DT>
__device__ __forceinline__ u32x4 operand(uint32_t w, uint32_t zero) {
  u32x4 r;
  if constexpr (DT == kF16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t m = 0x000F000F, b = 0x64006400;
    const u32x4 q = {(w & m) | b, ((w >> 4) & m) | b, ((w >> 8) & m) | b, ((w >> 12) & m) | b};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = q[i];  // (a bit_cast of the element itself takes element 0)
      r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, v) - __builtin_bit_cast(f16x2, zero));
    }
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    uint32_t lo, hi;
    w4_bytes(w, lo, hi);
    lo = less_bytes(lo, zero);
    hi = less_bytes(hi, zero);
    auto at = [](uint32_t v, int i) { return static_cast<float>(static_cast<int8_t>(v >> (8 * i))); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = i & 1 ? hi : lo;
      r[i] = __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(at(v, i >> 1)), static_cast<__bf16>(at(v, 2 + (i >> 1)))});
    }
  }
  return r;
}

// A lane's load of a row of 16-bit elements or bytes: the V elements from k on (16 bytes, or 8), zeros behind K.
template <int DT, int STEP>
__device__ __forceinline__ auto row_load(const char* row, int k, int K, bool whole) {
  constexpr int ES = DT == kI8 ? 1 : 2, V = w4_load(DT, STEP);
  typedef uint32_t Vec __attribute__((ext_vector_type(V * ES / 4)));
  typedef uint32_t VecU __attribute__((ext_vector_type(V * ES / 4), aligned(1)));
  if (whole || k + V <= K) return static_cast<Vec>(*reinterpret_cast<const VecU*>(row + static_cast<size_t>(k) * ES));
  Vec v = {};
  for (int i = 0; i < V; ++i)
    if (k + i < K) {
      const uint32_t e = ES == 1 ? *reinterpret_cast<const uint8_t*>(row + k + i)
                                 : *reinterpret_cast<const uint16_t*>(row + 2 * static_cast<size_t>(k + i));
      v[i * ES / 4] |= e << (8 * (i * ES % 4));
    }
  return v;
}

// ---- rows laid out --------------------------------------------------------------------------------
// Many rows, and fp32 rows from a line on, are first laid out as matrix operands: for each tile of 16 rows, chunk,
// half chunk and part, FR fragments of 1 KB (two of 16-bit elements, one of bytes) in which lane l holds 16 bytes of row
// l % 16; zeros behind the last row and input. Beside fp32 rows' stands a number for each row and
// scale's inputs, [tile][chunk][S][16]: they are two fp16 parts of x 2^k, the sum of which is x 2^k to half a step of
// fp32 (or to 2^-40 of the largest), with 2^k bringing the largest of a scale's inputs below 2^15; the number is 2^-k
// (NaN where an input is none). Other rows are as they are.
template <int DT> constexpr int kParts = DT == kF32 ? 2 : 1;
template <int DT> constexpr int kFrags = DT == kI8 ? 1 : 2;  // of a half chunk and part
template <int DT> constexpr int kOperand = DT == kF32 ? kF16 : DT;

// One block a tile and chunk; 16 lanes a row, 8 inputs a thread.
template <int DT, int STEP>
__global__ __launch_bounds__(256) void k_w4_lay(W4Args a, W4Geom g, char* frags, uint32_t* sums) {
  constexpr int P = kParts<DT>, FR = kFrags<DT>, S = 128 / STEP;
  const int u = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int c = blockIdx.x, k = c * 128 + 8 * u;
  const size_t rt = blockIdx.y, row = rt * 16 + r;
  const bool in = row < a.rows;
  // the unit's place: word j of lane group q
  const int j = STEP == 32 ? u >> 2 : (u >> 3) * 2 + (u & 1), q = STEP == 32 ? u & 3 : (u & 7) >> 1;
  const int h = j >> 1;
  char* to = frags + (rt * g.nc + c) * (2 * P * FR * 1024) + h * (P * FR * 1024) + (16 * q + r) * 16;
  constexpr int U = STEP / 8;  // neighbouring threads that share a scale
  if constexpr (DT == kF32) {
    float v[8];
    uint32_t top = 0;  // the largest magnitude, as bits: infinities and NaN are the largest
    const float* x = static_cast<const float*>(a.x) + row * a.ldx + k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = in && k + i < g.K ? x[i] : 0.0f;
      top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int n = 1; n < U; n *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), n)));
    const uint32_t e = top >> 23, up = min(268u - e, 253u);  // 2^k with k = 14 - exponent, at most 2^126
    const float f = __builtin_bit_cast(float, up << 23);
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h[2], l[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float y = v[2 * i + m] * f;
        const _Float16 p = static_cast<_Float16>(y);
        h[m] = __builtin_bit_cast(uint16_t, p);
        l[m] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(y - static_cast<float>(p)));
      }
      hi[i] = h[0] | h[1] << 16;
      lo[i] = l[0] | l[1] << 16;
    }
    *reinterpret_cast<u32x4*>(to + (j & 1) * 1024) = hi;
    *reinterpret_cast<u32x4*>(to + (FR + (j & 1)) * 1024) = lo;
    if (u % U == 0) sums[((rt * g.nc + c) * S + u / U) * 16 + r] = e == 255 ? 0x7FC00000u : (254 - up) << 23;
  } else if constexpr (DT == kI8) {
    uint32_t x0 = 0, x1 = 0;
    const int8_t* x = static_cast<const int8_t*>(a.x) + row * a.ldx + k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = in && k + i < g.K ? x[i] : 0;
      (i < 4 ? x0 : x1) |= static_cast<uint32_t>(e & 255) << (8 * (i & 3));
    }
    uint32_t lo, hi;
    i8_operand(x0, x1, lo, hi);
    uint32_t* o = reinterpret_cast<uint32_t*>(to + 8 * (j & 1));
    o[0] = lo;
    o[1] = hi;
  } else {
    u32x4 o = {0, 0, 0, 0};
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + row * a.ldx + k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t e = in && k + i < g.K ? x[i] : static_cast<uint16_t>(0);
      o[i / 2] |= static_cast<uint32_t>(e) << (16 * (i & 1));
    }
    *reinterpret_cast<u32x4*>(to + (j & 1) * 1024) = o;
  }
}

// ---- few rows -------------------------------------------------------------------------------------
// Few rows: one pass over the weights, bound by a launch, their loads' way and the operands' making (alone, 1 x 2048 x
// 11264, 12 MB: 6.2 us; 1 x 6912 x 2560 6.4; int8 64 x 2048 x 2048 5.3). A block's waves split the chunks of NT tiles of
// 16 outputs; each wave reads its 1 KB of codes per tile and chunk straight into the matrix operand's place and
// multiplies it with CT tiles of rows. fp32 rows are three bf16 parts each (hi + mid + lo = x exactly), 5 rows a
// tile: a wave cuts its chunk's rows into parts once, in LDS of its own, the next chunk's in flight; or (LAID) they
// were laid out, 16 a tile. The rows are the instruction's first operand, so that a lane's sums are of one output and
// its scale and zero point one word (four words a lane spilled registers with scales for 32 inputs: bf16 108 x 2048 x
// 11264 46 us, 31 now). The waves' sums meet in LDS in one fixed order.
template <int DT, bool LAID> constexpr int kTileRows = DT == kF32 && !LAID ? 5 : 16;
constexpr int kPartStride = 272;  // bytes of a part's 128 inputs in LDS, 16 apart in banks
template <int DT, int CT, bool LAID> constexpr int kPartBytes = DT == kF32 && !LAID ? CT * 15 * kPartStride : 0;

template <int DT, int STEP, int NT, int CT, bool LAID>
__global__ __launch_bounds__(CT == 1 && NT == 1 && !LAID ? 1024 : 512) void k_w4_rows(
    W4Args a, W4Geom g, const uint32_t* codes, const uint32_t* scales, const char* frags, const uint32_t* sums, int row_tiles) {
  static_assert(!LAID || DT == kF32, "other rows are read as they are");
  constexpr int OT = LAID ? kF16 : DT;
  using M = Mat<OT>;
  using Acc = typename M::Acc;
  constexpr int S = 128 / STEP, R = kTileRows<DT, LAID>;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int col = lane & 15, q = lane >> 4;
  const int row0 = blockIdx.y * (CT * R), rows = min(static_cast<int>(a.rows) - row0, CT * R);
  const int tile0 = blockIdx.x * NT;
  const size_t es = DT == kF32 ? 4 : DT == kI8 ? 1 : 2;
  const char* x0 = static_cast<const char*>(a.x) + static_cast<size_t>(row0) * a.ldx * es;
  char* part = lds + wave * kPartBytes<DT, CT, LAID>;

  const char* xr[CT];  // this lane's row of each tile of rows (a row past the end repeats the last one)
#pragma unroll
  for (int t = 0; t < CT; ++t) xr[t] = x0 + static_cast<size_t>(min(t * R + (DT == kF32 ? 0 : col), rows - 1)) * a.ldx * es;
  const uint32_t* cw[NT];
  const uint32_t* sw[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const size_t tile = min(tile0 + n, g.nt - 1);
    cw[n] = codes + tile * g.nc * 256 + lane * 4;
    sw[n] = scales + tile * g.ns * 16 + col;
  }

  // LAID: this lane's place in each tile's fragments and numbers
  const char* fr[CT];
  const uint32_t* num[CT];
  if constexpr (LAID) {
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const size_t rt = min(static_cast<int>(blockIdx.y) * CT + t, row_tiles - 1);
      fr[t] = frags + rt * g.nc * 8192 + lane * 16;
      num[t] = sums + rt * g.ns * 16 + 4 * q;
    }
  }

  f32x4 acc[NT][CT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[n][t] = f32x4{0, 0, 0, 0};

  u32x4 w[NT];
  uint32_t sz[NT][S];
  auto fetch = [&](int c) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      w[n] = *reinterpret_cast<const u32x4*>(cw[n] + static_cast<size_t>(c) * 256);
#pragma unroll
      for (int s = 0; s < S; ++s) sz[n][s] = sw[n][(static_cast<size_t>(c) * S + s) * 16];
    }
  };
  // fp32: two neighbours a lane of each row
  constexpr int kHeld = DT == kF32 && !LAID ? CT * R : 1;
  f32x2u held_x[kHeld];
  auto fetch_rows = [&](int c) {
    if constexpr (DT == kF32 && !LAID) {
      const int k = c * 128 + 2 * lane;
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {
        if (r >= rows) break;
        const float* p = reinterpret_cast<const float*>(x0) + r * a.ldx + k;
        if ((c + 1) * 128 <= g.K) {
          held_x[r] = *reinterpret_cast<const f32x2u*>(p);
        } else {
          held_x[r].x = k < g.K ? p[0] : 0.0f;
          held_x[r].y = k + 1 < g.K ? p[1] : 0.0f;
        }
      }
    }
  };
  int c = wave;
  if (c < g.nc) {
    fetch_rows(c);
    fetch(c);
  }
  for (; c < g.nc; c += waves) {
    const bool whole = (c + 1) * 128 <= g.K;
    u32x4 cur[NT];
    uint32_t csz[NT][S];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      cur[n] = w[n];
#pragma unroll
      for (int s = 0; s < S; ++s) csz[n][s] = sz[n][s];
    }
    // the rows' operands of this chunk
    constexpr int P = LAID ? 2 : 1;
    u32x4 b[CT][4 * P];
    u32x4 x[CT][S];
    if constexpr (LAID) {  // [half][part][word of the half]
#pragma unroll
      for (int t = 0; t < CT; ++t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) b[t][j] = *reinterpret_cast<const u32x4*>(fr[t] + (static_cast<size_t>(c) * 8 + j) * 1024);
#pragma unroll
        for (int s = 0; s < S; ++s) x[t][s] = *reinterpret_cast<const u32x4*>(num[t] + (static_cast<size_t>(c) * S + s) * 16);
      }
    } else if constexpr (DT == kF32) {
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {  // three parts each
        if (r >= rows) break;
        const float v[2] = {held_x[r].x, held_x[r].y};
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
            const auto v0 = row_load<DT, STEP>(xr[t], c * 128 + w4_k(STEP, j, q), g.K, whole);
            const auto v1 = row_load<DT, STEP>(xr[t], c * 128 + w4_k(STEP, j + 1, q), g.K, whole);
            v = u32x4{v0.x, v0.y, v1.x, v1.y};
          } else {
            v = row_load<DT, STEP>(xr[t], c * 128 + w4_k(STEP, j, q), g.K, whole);
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
        for (int j = 0; j < 4; ++j) b[t][j] = row_load<DT, STEP>(xr[t], c * 128 + w4_k(STEP, j, q), g.K, whole);
    }
    if (c + waves < g.nc) {
      fetch_rows(c + waves);
      fetch(c + waves);
    }

#pragma unroll
    for (int s = 0; s < S; ++s) {
      // sums of this scale's inputs: the products, and for int8 (whose zero points come off here) the inputs themselves
      Acc d[NT][CT], sum[CT];
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        sum[t] = Acc{};
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n][t] = Acc{};
      }
      if constexpr (DT == kI8) {
        constexpr uint32_t one = 0x01010101;
        if constexpr (STEP == 32) {  // one word a scale: 32 inputs an instruction
          const int j = s;
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            const long bx = (j & 1) ? (static_cast<long>(b[t][j / 2].w) << 32 | b[t][j / 2].z)
                                    : (static_cast<long>(b[t][j / 2].y) << 32 | b[t][j / 2].x);
            sum[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(bx, static_cast<long>(one) << 32 | one, sum[t], 0, 0, 0);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t lo, hi;
              w4_bytes(cur[n][j], lo, hi);
              d[n][t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(bx, static_cast<long>(hi) << 32 | lo, d[n][t], 0, 0, 0);
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
              sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bx, __builtin_bit_cast(i32x4, u32x4{one, one, one, one}),
                                                             sum[t], 0, 0, 0);
#pragma unroll
              for (int n = 0; n < NT; ++n) d[n][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bx, aw[n], d[n][t], 0, 0, 0);
            }
          }
        }
      } else {
#pragma unroll
        for (int jj = 0; jj < 4 / S; ++jj) {
          const int j = s * (4 / S) + jj;
          u32x4 aw[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) aw[n] = operand<OT>(cur[n][j], zero_of<OT>(csz[n][s]));
#pragma unroll
          for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int n = 0; n < NT; ++n)
                d[n][t] = M::mul(b[t][LAID ? (j >> 1) * 4 + p * 2 + (j & 1) : j], aw[n], d[n][t]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {  // rows 4 q + i of each tile, output `col`
        const uint32_t v = csz[n][s];
        const float sc = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v)));
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (DT == kI8)
              acc[n][t][i] = __builtin_fmaf(sc, static_cast<float>(d[n][t][i] - __mul24(static_cast<int>(v >> 16), sum[t][i])),
                                            acc[n][t][i]);
            else if constexpr (LAID)
              acc[n][t][i] = __builtin_fmaf(sc, d[n][t][i] * __builtin_bit_cast(f32x4, x[t][s])[i], acc[n][t][i]);
            else
              acc[n][t][i] = __builtin_fmaf(sc, d[n][t][i], acc[n][t][i]);
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
  const float* held = reinterpret_cast<const float*>(lds);
  for (int i = threadIdx.x; i < NT * 16 * rows; i += blockDim.x) {
    const int n = i % (NT * 16), r = i / (NT * 16), t = r / R;
    if (tile0 * 16 + n >= g.N) continue;
    const int at = (((n / 16) * CT + t) * 64 + n % 16) * 4;
    auto of = [](int row) { return row / 4 * 64 + row % 4; };  // of a tile
    float v = 0.0f;
    for (int wv = 0; wv < waves; ++wv) {
      const float* p = held + wv * (NT * CT * 256) + at;
      if constexpr (DT == kF32 && !LAID) {
        const int c0 = r % 5 * 3;  // the small parts first
        v += (p[of(c0 + 2)] + p[of(c0 + 1)]) + p[of(c0)];
      } else {
        v += p[of(r % 16)];
      }
    }
    if constexpr (DT == kI8) v *= a.xscales[row0 + r];
    store_as(a.out, a.out_dtype, static_cast<size_t>(row0 + r) * a.ldo + tile0 * 16 + n, v);
  }
}

template <int DT, int STEP, int NT, int CT, bool LAID = false>
hipError_t rows_launch(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, int waves,
                       hipStream_t s, const char* frags = nullptr, const uint32_t* sums = nullptr) {
  const size_t part = static_cast<size_t>(waves) * kPartBytes<DT, CT, LAID>, red = static_cast<size_t>(waves) * NT * CT * 1024;
  const size_t lds = part > red ? part : red;  // at most 64 KB: 16 waves of one tile of rows, 8 of two
  const unsigned per = CT * kTileRows<DT, LAID>;
  k_w4_rows<DT, STEP, NT, CT, LAID>
      <<<dim3((g.nt + NT - 1) / NT, static_cast<unsigned>((a.rows + per - 1) / per)), waves * 64, lds, s>>>(
          a, g, codes, scales, frags, sums, static_cast<int>((a.rows + 15) / 16));
  return hipGetLastError();
}

// Tiles of outputs a wave (nt) and waves a block. `units` is the tiles of outputs times the groups of rows.
// One tile of rows: a wave a tile of outputs; 16 waves where the inputs are long (us: 1 x 6912 x 2560 fp32 6.5 by 8 waves,
// 6.0 by 16; 1 x 2048 x 11264 5.7 and 6.3). Many rows of one tile share the rows' operands over four tiles of
// outputs instead where there are enough of these (bf16 16 x 2048 x 11264 8.7 -> 7.5).
// Two tiles of rows: the rows' operands are most of what is read, so a wave takes as many tiles of outputs as leave
// the chip full, and fewer waves share a block when there are more of them (bf16, one tile -> chosen: 64 x 6912 x
// 2560 27.8 -> 17.3, 128 x 6912 x 2560 44 -> 22, 100 x 2048 x 11264 41 -> 26.5). fp32 rows, whose parts are made
// anew for each of these, take two at most.
template <int DT, int STEP>
hipError_t rows_pick(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, hipStream_t s) {
  constexpr size_t R = kTileRows<DT, false>;
  constexpr bool F = DT == kF32;
  if (a.rows <= R) {
    if constexpr (!F) {
      if (a.rows > 8 && g.nt >= 512) return rows_launch<DT, STEP, 4, 1>(a, g, codes, scales, g.nc < 8 ? g.nc : 8, s);
    }
    const int most = g.nc > 32 ? 16 : 8;
    return rows_launch<DT, STEP, 1, 1>(a, g, codes, scales, g.nc < most ? g.nc : most, s);
  }
  const size_t groups = (a.rows + 2 * R - 1) / (2 * R), units = g.nt * groups;
  const int nt = units <= (F ? 512 : 256) ? 1 : F || units <= 512 ? 2 : 4;
  const size_t blocks = (g.nt + nt - 1) / nt * groups;
  const int most = blocks <= (F ? 1536 : nt == 4 ? 256 : 512) ? 8 : F || blocks <= 512 ? 4 : 2;
  const int waves = g.nc < most ? g.nc : most;
  if (nt == 1) return rows_launch<DT, STEP, 1, 2>(a, g, codes, scales, waves, s);
  if constexpr (!F) {
    if (nt == 4) return rows_launch<DT, STEP, 4, 2>(a, g, codes, scales, waves, s);
  }
  return rows_launch<DT, STEP, 2, 2>(a, g, codes, scales, waves, s);
}

// fp32 rows laid out, by the kernel of few rows.
template <int STEP>
hipError_t laid_rows(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, char* ws, hipStream_t s) {
  const int rt = static_cast<int>((a.rows + 15) / 16);
  uint32_t* sums = reinterpret_cast<uint32_t*>(ws + rt * w4_frag_bytes(kF32, g));
  k_w4_lay<kF32, STEP><<<dim3(g.nc, rt), 256, 0, s>>>(a, g, ws, sums);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const size_t units = static_cast<size_t>(g.nt) * ((rt + 1) / 2);
  const int waves = g.nc < 8 ? g.nc : 8;
  if (rt == 1) return units <= 256 ? rows_launch<kF32, STEP, 1, 1, true>(a, g, codes, scales, waves, s, ws, sums)
                                   : rows_launch<kF32, STEP, 2, 1, true>(a, g, codes, scales, waves, s, ws, sums);
  return units <= 256 ? rows_launch<kF32, STEP, 1, 2, true>(a, g, codes, scales, waves, s, ws, sums)
                      : rows_launch<kF32, STEP, 2, 2, true>(a, g, codes, scales, waves, s, ws, sums);
}

template <int DT>
hipError_t rows_step(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, hipStream_t s) {
  return g.step == 32 ? rows_pick<DT, 32>(a, g, codes, scales, s)
         : g.step == 64 ? rows_pick<DT, 64>(a, g, codes, scales, s) : rows_pick<DT, 128>(a, g, codes, scales, s);
}

// ---- many rows ------------------------------------------------------------------------------------
// A block of up to four groups of WN waves, a wave 64 outputs by TT tiles of rows; the groups, of all blocks of a
// tile, take chunks in turn, and a block's sums meet in LDS in a fixed order. The rows' fragments, their numbers
// and the scales go through LDS, shared by a group's waves, a stage (a chunk, or with two parts half a chunk)
// ahead through registers; codes go straight to their operand's place. The codes' products are summed for a
// scale's inputs alone, and the scale multiplies that sum, so the weights enter unrounded.
//
// 2048 x 2048 x 11264 fp32: 179 us and 13 for laying out, 1.06 PFLOP/s of fp16 products; a large library product
// reaches 1.13 here (bf16 123 and 8, fp16 112 and 8, int8 81 and 5). The matrix cores are busy 0.48 of the time and the vector ALUs (codes to operands, scales)
// 0.40, and overlap little. Measured and slower: blocks' tiles dealt to the L2 caches (213 to 220 us against
// 200 then), a later stage brought into L2 by a word of each line (294 against 216: the registers spill), a
// higher priority for the multiplying wave (215), and for 16-bit rows one tile of outputs after the other, so that
// a tile's scaling stands beside the next one's products (bf16 124 against 117 then).
constexpr int kRowTiles = 4;                                // of a wave: what the registers hold
template <int DT> constexpr int kHalves = DT == kF32 ? 1 : 2;    // half chunks of a stage
template <int DT> constexpr int kStageKB = kHalves<DT>* kParts<DT>* kFrags<DT>;  // of a tile of rows

template <int DT, int STEP, int WN>
__global__ __launch_bounds__(512) void k_w4_gemm(W4Args a, W4Geom g, const uint32_t* codes, const uint32_t* scales,
                                                 const char* frags, const uint32_t* sums, float* partials,
                                                 int row_tiles) {
  constexpr int OT = kOperand<DT>;
  using M = Mat<OT>;
  using Acc = typename M::Acc;
  constexpr int P = kParts<DT>, FR = kFrags<DT>, S = 128 / STEP, TT = kRowTiles, H = kHalves<DT>, KB = kStageKB<DT>;
  constexpr int kPieces = TT * KB / WN;  // KB that a wave moves of a stage
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bk = (blockDim.x >> 6) / WN, group = wave / WN, in = wave % WN;
  const int kw = bk * gridDim.z, kg = blockIdx.z * bk + group;  // the chunks' groups, of all blocks of a tile
  const int gthread = threadIdx.x - group * WN * 64;
  const int q = lane >> 4;
  const int btile = blockIdx.x * (WN * 4), tile0 = btile + in * 4, rt0 = blockIdx.y * TT;
  // LDS of a group: two buffers of the rows' pieces, the scales [WN 4][S][16] and the rows' numbers, if any, [TT][S][16]
  constexpr bool kNumbers = w4_numbers(DT);
  constexpr int pieces = TT * KB, words = (WN * 4 + (kNumbers ? TT : 0)) * S * 16, buf_bytes = pieces * 1024 + words * 4;
  char* mem = lds + group * 2 * buf_bytes;

  const uint32_t* cw[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) cw[n] = codes + static_cast<size_t>(min(tile0 + n, g.nt - 1)) * g.nc * 256 + lane * 4;

  // Loads and LDS writes have no conditions (an index past the end repeats the last one), so that the
  // compiler knows which loads are in flight and waits for no younger ones.
  u32x4 hold[kPieces];
  constexpr int kW = (words + WN * 64 - 1) / (WN * 64);  // words that a thread moves
  uint32_t hold_w[kW];
  const char* from_p[kPieces];
  const uint32_t* from_w[kW];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int p = i * WN + in;
    const size_t rt = min(rt0 + p / KB, row_tiles - 1);
    from_p[i] = frags + rt * g.nc * (2 / H) * (KB * 1024) + (p % KB) * 1024 + lane * 16;
  }
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    const int v = min(i * WN * 64 + gthread, words - 1), unit = v / (S * 16), at = v - unit * (S * 16);
    from_w[i] = (unit < WN * 4 ? scales + static_cast<size_t>(min(btile + unit, g.nt - 1)) * g.ns * 16
                               : sums + static_cast<size_t>(min(rt0 + unit - WN * 4, row_tiles - 1)) * g.ns * 16) + at;
  }
  auto fetch = [&](int c, int half) {
    const size_t st = H == 2 ? c : 2 * c + half;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) hold[i] = *reinterpret_cast<const u32x4*>(from_p[i] + st * (KB * 1024));
#pragma unroll
    for (int i = 0; i < kW; ++i) hold_w[i] = from_w[i][static_cast<size_t>(c) * S * 16];
  };
  auto put = [&](int buf) {
    char* to = mem + buf * buf_bytes;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) *reinterpret_cast<u32x4*>(to + (i * WN + in) * 1024 + lane * 16) = hold[i];
    uint32_t* tw = reinterpret_cast<uint32_t*>(to + pieces * 1024);
#pragma unroll
    for (int i = 0; i < kW; ++i) tw[min(i * WN * 64 + gthread, words - 1)] = hold_w[i];
  };

  f32x4 acc[4][TT];
  Acc d[4][TT];
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[n][t] = f32x4{0, 0, 0, 0};
  u32x4 w[4], next[4];
  const int rounds = (g.nc + kw - 1) / kw;  // the same for all groups: a group without a chunk adds nothing
  auto load_codes = [&](int c) {
#pragma unroll
    for (int n = 0; n < 4; ++n) next[n] = *reinterpret_cast<const u32x4*>(cw[n] + static_cast<size_t>(c) * 256);
  };
  const int last = g.nc - 1;
  load_codes(min(kg, last));
  fetch(min(kg, last), 0);
  put(0);
  __syncthreads();
  for (int r = 0; r < rounds; ++r) {
    const int c = r * kw + kg;
    const bool mine_too = c <= last;
#pragma unroll
    for (int n = 0; n < 4; ++n) w[n] = next[n];
    load_codes(min(c + kw, last));
#pragma unroll
    for (int hs = 0; hs < 2 / H; ++hs) {
      const int cur = H == 2 ? r & 1 : hs;
      if (H == 2 || hs == 1)
        fetch(min(c + kw, last), 0);
      else
        fetch(min(c, last), 1);
      const char* buf = mem + cur * buf_bytes;
      const char* mine = buf + lane * 16;
      const uint32_t* sc_at = reinterpret_cast<const uint32_t*>(buf + pieces * 1024) + in * 4 * S * 16 + 4 * q;
      const uint32_t* x_at = reinterpret_cast<const uint32_t*>(buf + pieces * 1024) + WN * 4 * S * 16 + (lane & 15);

      // the zero points of this lane's outputs of the operand (lane % 16 of each tile)
      uint32_t zero[4];
      auto zeros = [&](int s) {
        const uint32_t* z_at = reinterpret_cast<const uint32_t*>(buf + pieces * 1024) + in * 4 * S * 16 + (lane & 15);
#pragma unroll
        for (int n = 0; n < 4; ++n) zero[n] = zero_of<OT>(z_at[(n * S + s) * 16]);
      };
      auto clear = [&] {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int t = 0; t < TT; ++t) d[n][t] = Acc{};
      };
      auto flush = [&](int s) {
        if (!mine_too) return;
        uint32_t x[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) x[t] = kNumbers ? x_at[(t * S + s) * 16] : 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const u32x4 sz = *reinterpret_cast<const u32x4*>(sc_at + (n * S + s) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float sc = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(sz[i])));
#pragma unroll
            for (int t = 0; t < TT; ++t) {
              if constexpr (kNumbers)
                acc[n][t][i] = __builtin_fmaf(sc, d[n][t][i] * __builtin_bit_cast(float, x[t]), acc[n][t][i]);
              else
                acc[n][t][i] = __builtin_fmaf(sc, static_cast<float>(d[n][t][i]), acc[n][t][i]);
            }
          }
        }
      };
#pragma unroll
      for (int hh = 0; hh < H; ++hh) {
        const int half = H == 2 ? hh : hs;  // of its chunk
        if constexpr (DT == kI8) {
          i32x4 b[TT];
#pragma unroll
          for (int t = 0; t < TT; ++t) b[t] = *reinterpret_cast<const i32x4*>(mine + (t * KB + hh) * 1024);
          if constexpr (STEP == 32) {
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
              clear();
              zeros(2 * half + jj);
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                uint32_t lo, hi;
                w4_bytes(w[n][2 * half + jj], lo, hi);
                const long aw = static_cast<long>(less_bytes(hi, zero[n])) << 32 | less_bytes(lo, zero[n]);
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                  const long bx =
                      static_cast<long>(static_cast<uint32_t>(b[t][2 * jj + 1])) << 32 | static_cast<uint32_t>(b[t][2 * jj]);
                  d[n][t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(aw, bx, d[n][t], 0, 0, 0);
                }
              }
              flush(2 * half + jj);
            }
          } else {
            if (STEP == 64 || half == 0) clear();
            zeros(STEP == 64 ? half : 0);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              uint32_t lo0, hi0, lo1, hi1;
              w4_bytes(w[n][2 * half], lo0, hi0);
              w4_bytes(w[n][2 * half + 1], lo1, hi1);
              const uint32_t z = zero[n];
              const i32x4 aw = __builtin_bit_cast(
                  i32x4, u32x4{less_bytes(lo0, z), less_bytes(hi0, z), less_bytes(lo1, z), less_bytes(hi1, z)});
#pragma unroll
              for (int t = 0; t < TT; ++t) d[n][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(aw, b[t], d[n][t], 0, 0, 0);
            }
          }
        } else {
          if (STEP == 64 || (STEP == 128 && half == 0)) clear();
          if (STEP >= 64) zeros(STEP == 64 ? half : 0);
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            if (STEP == 32) clear(), zeros(2 * half + jj);
            u32x4 aw[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) aw[n] = operand<OT>(w[n][2 * half + jj], zero[n]);
#pragma unroll
            for (int p = 0; p < P; ++p) {
              u32x4 b[TT];
#pragma unroll
              for (int t = 0; t < TT; ++t)
                b[t] = *reinterpret_cast<const u32x4*>(mine + (t * KB + (hh * P + p) * FR + jj) * 1024);
#pragma unroll
              for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int t = 0; t < TT; ++t) d[n][t] = M::mul(aw[n], b[t], d[n][t]);
            }
            if (STEP == 32) flush(2 * half + jj);
          }
        }
        if (STEP == 64) flush(half);
        if (STEP == 128 && half == 1) flush(0);
      }
      put(cur ^ 1);
      __syncthreads();
    }
  }

  if (bk > 1) {  // the groups' sums, in the order of the groups
    f32x4* red = reinterpret_cast<f32x4*>(lds);
    if (group > 0) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int t = 0; t < TT; ++t) red[(((group - 1) * WN + in) * (4 * TT) + n * TT + t) * 64 + lane] = acc[n][t];
    }
    __syncthreads();
    if (group > 0) return;
    for (int k = 0; k < bk - 1; ++k)
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[n][t] += red[((k * WN + in) * (4 * TT) + n * TT + t) * 64 + lane];
  }
  if (partials) {  // one of several blocks of this tile: k_w4_sum adds them
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int rt = rt0 + t;
      if (rt >= row_tiles) continue;
      float* to = partials + ((static_cast<size_t>(blockIdx.z) * row_tiles + rt) * 16 + (lane & 15)) * (g.nt * 16) + 4 * q;
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (tile0 + n < g.nt) *reinterpret_cast<f32x4*>(to + (tile0 + n) * 16) = acc[n][t];
    }
    return;
  }
  auto store = [&](auto ot) {
    using O = Elem<decltype(ot)::value>;
    typedef typename O::T T4 __attribute__((ext_vector_type(4), aligned(sizeof(typename O::T))));
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const size_t row = static_cast<size_t>(rt0 + t) * 16 + (lane & 15);
      if (row >= a.rows) continue;
      const float xsc = DT == kI8 ? a.xscales[row] : 1.0f;
      typename O::T* out = static_cast<typename O::T*>(a.out) + row * a.ldo;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int o = (tile0 + n) * 16 + 4 * q;
        T4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = O::down(DT == kI8 ? acc[n][t][i] * xsc : acc[n][t][i]);
        if (o + 4 <= g.N) {
          *reinterpret_cast<T4*>(out + o) = v;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (o + i < g.N) out[o + i] = v[i];
        }
      }
    }
  };
  if (a.out_dtype == kF32)
    store(std::integral_constant<int, kF32>{});
  else if (a.out_dtype == kBF16)
    store(std::integral_constant<int, kBF16>{});
  else
    store(std::integral_constant<int, kF16>{});
}

// The blocks' partial sums, added in the order of the blocks; four outputs a thread.
template <int DT>
__global__ __launch_bounds__(256) void k_w4_sum(W4Args a, W4Geom g, const float* partials, int row_tiles, int ks) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  const size_t row = blockIdx.y;
  if (n >= g.N) return;
  const float* p = partials + row * (g.nt * 16) + n;
  const size_t step = static_cast<size_t>(row_tiles) * 16 * (g.nt * 16);
  f32x4 v = *reinterpret_cast<const f32x4*>(p);
  for (int k = 1; k < ks; ++k) v += *reinterpret_cast<const f32x4*>(p + k * step);
  if (DT == kI8) v *= a.xscales[row];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < g.N) store_as(a.out, a.out_dtype, row * a.ldo + n + i, v[i]);
}

template <int DT, int STEP>
hipError_t gemm_launch(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, char* ws,
                       hipStream_t s) {
  const int rt = static_cast<int>((a.rows + 15) / 16);
  uint32_t* sums = reinterpret_cast<uint32_t*>(ws + rt * w4_frag_bytes(DT, g));
  k_w4_lay<DT, STEP><<<dim3(g.nc, rt), 256, 0, s>>>(a, g, ws, sums);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  constexpr int TT = kRowTiles, S = 128 / STEP;
  static_assert(TT == kW4TileRows / 16, "the plan's tiles");
  const W4Plan p = w4_plan(DT, g, rt);
  const size_t buf = TT * kStageKB<DT> * 1024 + (p.wn * 4 + (w4_numbers(DT) ? TT : 0)) * S * 64, stages = 2 * p.bk * buf;
  const size_t red = (p.bk - 1) * p.wn * TT * 4096, lds = stages > red ? stages : red;  // up to 152 KB
  const dim3 grid((g.nt + p.wn * 4 - 1) / (p.wn * 4), (rt + TT - 1) / TT, p.ks);
  float* partials = p.ks > 1 ? reinterpret_cast<float*>(ws + w4_lay_bytes(DT, g, rt)) : nullptr;
  const int threads = p.wn * p.bk * 64;
  if (p.wn == 4)
    k_w4_gemm<DT, STEP, 4><<<grid, threads, lds, s>>>(a, g, codes, scales, ws, sums, partials, rt);
  else
    k_w4_gemm<DT, STEP, 2><<<grid, threads, lds, s>>>(a, g, codes, scales, ws, sums, partials, rt);
  e = hipGetLastError();
  if (e != hipSuccess || !partials) return e;
  k_w4_sum<DT><<<dim3((g.N + 1023) / 1024, static_cast<unsigned>(a.rows)), 256, 0, s>>>(a, g, partials, rt, p.ks);
  return hipGetLastError();
}

template <int DT>
hipError_t gemm_step(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, char* ws,
                     hipStream_t s) {
  return g.step == 32 ? gemm_launch<DT, 32>(a, g, codes, scales, ws, s)
         : g.step == 64 ? gemm_launch<DT, 64>(a, g, codes, scales, ws, s) : gemm_launch<DT, 128>(a, g, codes, scales, ws, s);
}

}  // namespace

hipError_t launch_w4_pack(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, const W4Geom& g,
                          uint32_t* out, uint32_t* out_scales, hipStream_t s) {
  const size_t nc = w4_code_bytes(g) / 4, ns = w4_scale_bytes(g) / 4;
  k_w4_pack<<<static_cast<unsigned>((nc + 255) / 256), 256, 0, s>>>(codes, g, out);
  k_w4_pack_scales<<<static_cast<unsigned>((ns + 255) / 256), 256, 0, s>>>(scales, zeros, g, out_scales);
  return hipGetLastError();
}

template <class F>
static hipError_t by_type(int dtype, F&& f) {
  return dtype == kI8 ? f(std::integral_constant<int, kI8>{}) : with_type(dtype, f);
}

hipError_t launch_w4(const W4Args& a, const W4Geom& g, const uint32_t* codes, const uint32_t* scales, char* ws,
                     hipStream_t s) {
  const size_t most = w4_rows_most(a.dtype, g, a.rows);
  for (size_t r = 0; r < a.rows; r += most) {
    W4Args b = a;
    b.rows = a.rows - r < most ? a.rows - r : most;
    b.x = static_cast<const char*>(a.x) + r * a.ldx * dtype_size(a.dtype);
    b.out = static_cast<char*>(a.out) + r * a.ldo * dtype_size(a.out_dtype);
    if (a.xscales) b.xscales = a.xscales + r;
    const hipError_t e = by_type(a.dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      const W4Way way = w4_way(a.dtype, g, a.rows);
      if (way == kTiles) return gemm_step<DT>(b, g, codes, scales, ws, s);
      if constexpr (DT == kF32) {
        if (way == kLaidRows)
          return g.step == 32   ? laid_rows<32>(b, g, codes, scales, ws, s)
                 : g.step == 64 ? laid_rows<64>(b, g, codes, scales, ws, s) : laid_rows<128>(b, g, codes, scales, ws, s);
      }
      return rows_step<DT>(b, g, codes, scales, s);
    });
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mmf
