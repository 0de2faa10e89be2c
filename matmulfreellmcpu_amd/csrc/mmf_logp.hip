// mmf_logp.hip -- log probabilities of given tokens, the distribution's entropy and its most likely tokens.
//
// With m the row's largest logit, z = (x - m) / temperature, s = sum e^z: log p = z - log s, entropy = log s -
// sum(z e^z) / s. The most likely tokens are ordered by logit, ties by the lower index (NaN above all, as sorts
// take it); a logit and its index make one 64-bit number of that order.
//
// What bounds it: reading the logits. A block holds a row, or 32768 elements of a longer one, in registers, so that
// each logit is read once from memory: maximum, sums and candidates are passes over registers.
#include "mmf_layer_dev.hpp"

namespace mmf {
namespace {

constexpr int kWaves = kLogpThreads / 64;
constexpr int kCandidates = 2048;

// A monotone 32-bit image of a logit: larger logits have larger ones, -0 and 0 the same, every NaN the largest.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 + 0 = 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? (k == 0xFFFFFFFFu ? 0x7FC00000u : k & 0x7FFFFFFFu) : ~k);
}
// The order of the top tokens in one number; 0 stands for none.
__device__ __forceinline__ uint64_t pack(uint32_t key, uint32_t index) {
  return static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint32_t index_of(uint64_t p) { return 0xFFFFFFFFu - static_cast<uint32_t>(p); }

struct Sums {
  float top, sum, weighted;  // the maximum, sum e^z, sum z e^z
};

// log p of a token whose logit is v.
__device__ __forceinline__ float logp_of(const Sums& t, float inv_t, float log_sum, float v) {
  return t.sum == 0.0f ? -__builtin_inff() : (v - t.top) * inv_t - log_sum;  // a row of -infinity alone has no tokens
}
__device__ __forceinline__ float entropy_of(const Sums& t, float log_sum) {
  return t.sum == 0.0f ? 0.0f : log_sum - t.weighted / t.sum;
}

// The outputs of a row but its top tokens, by one thread.
template <int DT>
__device__ __forceinline__ void finish(const LogpArgs& a, size_t row, const Sums& t, float inv_t, float log_sum) {
  using E = Elem<DT>;
  if (a.entropy) a.entropy[row] = entropy_of(t, log_sum);
  if (a.logprobs) {
    const int64_t id = a.ids[row];
    const bool in = id >= 0 && id < static_cast<int64_t>(a.V);
    a.logprobs[row] = in ? logp_of(t, inv_t, log_sum, E::up(static_cast<const typename E::T*>(a.x)[row * a.ld + id]))
                         : __builtin_nanf("");
  }
}

template <int DT, int NV>
__global__ __launch_bounds__(kLogpThreads) void k_logp(LogpArgs a, float inv_t, float* ws) {
  using E = Elem<DT>;
  using T = typename E::T;
  using Vec = typename E::Vec;
  constexpr int V = E::V;
  __shared__ float s_top[kWaves], s_sum[kWaves], s_weighted[kWaves];
  __shared__ uint32_t s_key[kWaves];
  __shared__ uint64_t s_best[2][kWaves];
  __shared__ uint64_t list[kCandidates];
  __shared__ int count;
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int from = blockIdx.y * (kLogpThreads * V * NV), len = min(static_cast<int>(a.V) - from, kLogpThreads * V * NV);
  const T* x = static_cast<const T*>(a.x) + row * a.ld + from;
  if (tid == 0) count = 0;

  Vec v[NV];
  const T none = E::down(-__builtin_inff());
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * kLogpThreads + tid) * V;
    if (at + V <= len) {
      v[i] = *reinterpret_cast<const Vec*>(x + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = at + j < len ? x[at + j] : none;
    }
  }
  float top = -__builtin_inff();
  bool nan = false;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float f = E::up(v[i][j]);
      top = __builtin_fmaxf(top, f);
      nan |= f != f;
    }
  const float own = top;
#pragma unroll
  for (int n = 1; n < 64; n *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, n));
  // The wave's top-th largest of its lanes' largest: at least `top` elements are as large. The block's candidates are the
  // elements no smaller than the largest of its waves' bounds.
  uint32_t bound = 0;
  if (a.top) {
    const uint32_t mine = nan ? 0xFFFFFFFFu : tid * V < len ? key_of(own) : 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t next = bound | 1u << bit;
      if (__popcll(__ballot(mine >= next)) >= static_cast<int>(a.top)) bound = next;
    }
  }
  if (lane == 0) {
    s_top[wave] = top;
    s_key[wave] = bound;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    top = __builtin_fmaxf(top, s_top[w]);
    bound = max(bound, s_key[w]);
  }
  // (of -infinity alone the shift is 0, so that the sum is 0, or NaN by a NaN)
  const float shift = top == -__builtin_inff() ? 0.0f : top, scale = inv_t * 1.44269504f;
  float sum = 0.0f, weighted = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float z = E::up(v[i][j]) - shift, e = exp2_fast(z * scale);
      sum += e;
      weighted = __builtin_fmaf(e > 0.0f ? z : 0.0f, e, weighted);
    }
#pragma unroll
  for (int n = 1; n < 64; n *= 2) {
    sum += __shfl_xor(sum, n);
    weighted += __shfl_xor(weighted, n);
  }
  if (lane == 0) {
    s_sum[wave] = sum;
    s_weighted[wave] = weighted;
  }
  if (a.top) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int at = (i * kLogpThreads + tid) * V + j;
        const uint32_t key = key_of(E::up(v[i][j]));
        const bool hit = key >= bound && at < len;
        const uint64_t hits = __ballot(hit);
        if (!hits) continue;
        int place = 0;
        if (lane == 0) place = atomicAdd(&count, __popcll(hits));  // their order in the list does not matter
        place = __builtin_amdgcn_readfirstlane(place) + __popcll(hits & ((1ull << lane) - 1));
        if (hit && place < kCandidates) list[place] = pack(key, from + at);
      }
  }
  __syncthreads();
  sum = weighted = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    sum += s_sum[w];
    weighted += s_weighted[w];
  }
  const Sums t{top, sum, weighted * inv_t};
  const bool whole = gridDim.y == 1;
  const float log_sum = logf(sum);
  float* part = ws + (row * gridDim.y + blockIdx.y) * (4 + 2 * a.top);
  if (tid == 0) {
    if (whole) {
      finish<DT>(a, row, t, inv_t, log_sum);
    } else {
      part[0] = t.top;
      part[1] = t.sum;
      part[2] = t.weighted;
    }
  }
  if (!a.top) return;
  const int k = static_cast<int>(a.top);
  auto put = [&](int rank, uint64_t p) {
    if (!whole) {
      reinterpret_cast<uint64_t*>(part + 4)[rank] = p;
    } else {
      a.top_ids[row * k + rank] = index_of(p);
      a.top_logprobs[row * k + rank] = logp_of(t, inv_t, log_sum, value_of(static_cast<uint32_t>(p >> 32)));
    }
  };
  const int n = count;
  if (n <= kCandidates) {
    for (int c = tid; c < n; c += kLogpThreads) {
      const uint64_t mine = list[c];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += list[o] > mine;
      if (rank < k) put(rank, mine);
    }
    for (int r = n + tid; r < k; r += kLogpThreads) put(r, 0);  // a last part of fewer elements
    return;
  }
  // many equal ones: one at a time, the largest below the last
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int at = (i * kLogpThreads + tid) * V + j;
        const uint64_t p = pack(key_of(E::up(v[i][j])), from + at);
        if (at < len && p < last && p > best) best = p;
      }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint64_t o = __shfl_xor(static_cast<unsigned long long>(best), d);
      best = o > best ? o : best;
    }
    if (lane == 0) s_best[r & 1][wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best = s_best[r & 1][w] > best ? s_best[r & 1][w] : best;
    if (tid == 0) put(r, best);
    last = best;
  }
}

// The parts of a row joined.
template <int DT>
__global__ __launch_bounds__(256) void k_logp_join(LogpArgs a, float inv_t, const float* ws, int segs) {
  __shared__ uint64_t list[2048];
  const size_t row = blockIdx.x;
  const int k = static_cast<int>(a.top), step = 4 + 2 * k;
  const float* part = ws + row * segs * step;
  Sums t{-__builtin_inff(), 0.0f, 0.0f};
  for (int i = 0; i < segs; ++i) t.top = __builtin_fmaxf(t.top, part[i * step]);
  for (int i = 0; i < segs; ++i) {
    const float s = part[i * step + 1], w = part[i * step + 2];
    if (s == 0.0f) continue;
    const float d = (part[i * step] - t.top) * inv_t, f = exp2_fast(d * 1.44269504f);
    t.sum = __builtin_fmaf(f, s, t.sum);
    t.weighted = __builtin_fmaf(f, __builtin_fmaf(f > 0.0f ? d : 0.0f, s, w), t.weighted);
  }
  const float log_sum = logf(t.sum);
  if (threadIdx.x == 0) finish<DT>(a, row, t, inv_t, log_sum);
  if (!k) return;
  const int n = segs * k;
  for (int i = threadIdx.x; i < n; i += 256) list[i] = reinterpret_cast<const uint64_t*>(part + i / k * step + 4)[i % k];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t mine = list[i];
    if (!mine) continue;
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += list[o] > mine;
    if (rank >= k) continue;
    a.top_ids[row * k + rank] = index_of(mine);
    a.top_logprobs[row * k + rank] = logp_of(t, inv_t, log_sum, value_of(static_cast<uint32_t>(mine >> 32)));
  }
}

}  // namespace

hipError_t launch_logp(const LogpArgs& all, float* ws, hipStream_t s) {
  return with_type(all.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const LogpPlan p = logp_plan(DT, all.V);
    const float inv_t = 1.0f / all.temperature;
    size_t most = logp_rows_most(p, all.top);
    if (most > size_t{1} << 20) most = size_t{1} << 20;  // a grid has fewer than 2^32 threads
    for (size_t r = 0; r < all.rows; r += most) {
      LogpArgs a = all;
      a.rows = all.rows - r < most ? all.rows - r : most;
      a.x = static_cast<const char*>(all.x) + r * all.ld * dtype_size(DT);
      if (a.ids) a.ids += r;
      if (a.logprobs) a.logprobs += r;
      if (a.entropy) a.entropy += r;
      if (a.top_ids) a.top_ids += r * all.top;
      if (a.top_logprobs) a.top_logprobs += r * all.top;
      const dim3 grid(static_cast<unsigned>(a.rows), p.segs);
      switch (p.vecs) {
        case 1: k_logp<DT, 1><<<grid, kLogpThreads, 0, s>>>(a, inv_t, ws); break;
        case 2: k_logp<DT, 2><<<grid, kLogpThreads, 0, s>>>(a, inv_t, ws); break;
        case 4: k_logp<DT, 4><<<grid, kLogpThreads, 0, s>>>(a, inv_t, ws); break;
        default:
          if constexpr (DT == kF32) k_logp<DT, 8><<<grid, kLogpThreads, 0, s>>>(a, inv_t, ws);
      }
      hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      if (p.segs > 1) {
        k_logp_join<DT><<<grid.x, 256, 0, s>>>(a, inv_t, ws, p.segs);
        if ((e = hipGetLastError()) != hipSuccess) return e;
      }
    }
    return hipSuccess;
  });
}

}  // namespace mmf
