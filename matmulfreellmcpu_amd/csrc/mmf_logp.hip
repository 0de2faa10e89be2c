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

// (v - m) / 2, for logits whose difference may pass fp32; as exact as the difference. It goes with twice the temperature's
// inverse, two_t, which is finite also times log2(e).
__device__ __forceinline__ float half_less(float v, float half_m) { return __builtin_fmaf(v, 0.5f, -half_m); }

// log p of a token whose logit is v.
__device__ __forceinline__ float logp_of(const Sums& t, float two_t, float log_sum, float v) {
  return t.sum == 0.0f ? -__builtin_inff() : half_less(v, 0.5f * t.top) * two_t - log_sum;  // a row of -infinity alone has no tokens
}
__device__ __forceinline__ float entropy_of(const Sums& t, float log_sum) {
  return t.sum == 0.0f ? 0.0f : log_sum - t.weighted / t.sum;
}

// The logit of a row's given token, if it has one.
template <int DT>
__device__ __forceinline__ float given(const LogpArgs& a, size_t row) {
  using E = Elem<DT>;
  const int64_t id = a.ids[row];
  const bool in = id >= 0 && id < static_cast<int64_t>(a.V);
  return in ? E::up(static_cast<const typename E::T*>(a.x)[row * a.ld + id]) : __builtin_nanf("");
}
// The outputs of a row but its top tokens, by one thread.
__device__ __forceinline__ void finish(const LogpArgs& a, size_t row, const Sums& t, float two_t, float log_sum, float logit) {
  if (a.entropy) a.entropy[row] = entropy_of(t, log_sum);
  if (a.logprobs) a.logprobs[row] = logit != logit ? logit : logp_of(t, two_t, log_sum, logit);
}

// The top tokens of a part with more candidates than the list holds, or with numbers that are none: one at a time, the
// largest below the last, of logits read again.
template <int DT, int TH, class Put>
__device__ __forceinline__ void one_by_one(const typename Elem<DT>::T* x, int from, int len, int k, uint64_t (&s_best)[2][TH / 64], Put put) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int at = tid; at < len; at += TH) {
      const uint64_t p = pack(key_of(Elem<DT>::up(x[at])), from + at);
      if (p < last && p > best) best = p;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint64_t o = __shfl_xor(static_cast<unsigned long long>(best), d);
      best = o > best ? o : best;
    }
    if (lane == 0) s_best[r & 1][wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) best = s_best[r & 1][w] > best ? s_best[r & 1][w] : best;
    if (tid == 0) put(r, best);
    last = best;
  }
}

// A block goes through parts of rows (rows, where one part is a row), the next one's logits on their way meanwhile. 2048 x 32000
// bf16 (131 MB) 45 us, 27.6 at a copy's rate, with the vector ALUs 0.56 busy: two passes over a row's registers and three
// barriers stand between its loads; without top tokens 36.
template <int DT, int TH, int NV, bool WHOLE>
__global__ __launch_bounds__(TH, NV <= 2 ? 8 : 4) void k_logp(LogpArgs a, float two_t, float* ws, uint32_t segs) {
  using E = Elem<DT>;
  using T = typename E::T;
  using Vec = typename E::Vec;
  constexpr int V = E::V, kPart = TH * V * NV, kWaves = TH / 64;
  __shared__ __align__(16) float s_top[64];
  __shared__ float s_sum[kWaves], s_weighted[kWaves], s_bound;
  __shared__ uint64_t s_best[2][kWaves];
  __shared__ uint64_t list[kCandidates];
  __shared__ int s_count[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), k = static_cast<int>(a.top);
  const uint32_t parts = static_cast<uint32_t>(a.rows) * (WHOLE ? 1 : segs);
  auto row_of = [&](uint32_t part) { return WHOLE ? part : part / segs; };
  auto from_of = [&](uint32_t part) { return WHOLE ? 0 : static_cast<int>(part - part / segs * segs) * kPart; };
  auto logits = [&](uint32_t part) { return static_cast<const T*>(a.x) + row_of(part) * a.ld + from_of(part); };
  auto len_of = [&](uint32_t part) { return min(static_cast<int>(a.V) - from_of(part), kPart); };
  const T none = E::down(-__builtin_inff());

  // What keeps registers few: a part's start and length are new in each pass of the loop (places are not kept from one to
  // the next), and logits are widened where they are used, from the bits that were loaded.
  auto fresh = [](int n) {
    n = __builtin_amdgcn_readfirstlane(n);
    asm volatile("" : "+s"(n));
    return n;
  };
  auto narrow = [](Vec (&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(v[i]));
  };
  // Loads without conditions of a lane's own, so that all are in flight together.
  auto fetch = [&](Vec (&v)[NV], uint32_t part) {
    const int len = fresh(len_of(part));
    const T* x = logits(part);
    int t0 = tid;
    asm volatile("" : "+v"(t0));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (i * TH + t0) * V;
      if ((i + 1) * TH * V <= len) {
        v[i] = *reinterpret_cast<const Vec*>(x + at);
      } else if (len % V == 0) {
        v[i] = *reinterpret_cast<const Vec*>(x + min(at, len - V));
        if (at >= len) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[i][j] = none;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = x[min(at + j, len - 1)];
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (at + j >= len) v[i][j] = none;
      }
    }
  };
  Vec v[NV], next[NV];
  if (blockIdx.x < parts) fetch(next, blockIdx.x);
  for (uint32_t part = blockIdx.x; part < parts; part += gridDim.x) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = next[i];
    const size_t row = row_of(part);
    const int from = fresh(from_of(part)), len = fresh(len_of(part));
    float logit = 0.0f;
    if (WHOLE && tid == TH - 1 && a.ids) logit = given<DT>(a, row);
    float own = -__builtin_inff();  // (NaN left out: the sum shows it)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) own = __builtin_fmaxf(own, E::up(v[i][j]));
    narrow(v);
    if (part + gridDim.x < parts) fetch(next, part + gridDim.x);
    float top = own;
#pragma unroll
    for (int n = 1; n < kWaves; n *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, n));
    if (lane % kWaves == 0) s_top[tid / kWaves] = top;
    if (tid < 2) s_count[tid] = 0;
    __syncthreads();
    // every wave has the largest of 64 groups of threads, a lane each
    const float group = s_top[lane];
    top = group;
#pragma unroll
    for (int n = 1; n < 64; n *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, n));
    // The k-th largest of the groups' largest (k at most 64): at least k logits are as large, so that the k largest are
    // among those no smaller than it.
    if (k && wave == 0) {
      typedef float f4 __attribute__((ext_vector_type(4)));
      int above = 0;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const f4 g = reinterpret_cast<const f4*>(s_top)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) above += g[e] > group;
      }
      float least = above < k ? group : __builtin_inff();
#pragma unroll
      for (int n = 1; n < 64; n *= 2) least = __builtin_fminf(least, __shfl_xor(least, n));
      if (lane == 0) s_bound = least;
    }
    // (of -infinity alone the shift is 0, so that the sum is 0, or NaN by a NaN)
    const float half = top == -__builtin_inff() ? 0.0f : 0.5f * top, scale = two_t * 1.44269504f;
    float sum = 0.0f, weighted = 0.0f;  // (sum z log2(e) e^z)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float z = half_less(E::up(v[i][j]), half) * scale, e = exp2_fast(z);
        sum += e;
        weighted = __builtin_fmaf(__builtin_fmaxf(z, -1e30f), e, weighted);  // (below -150 e is 0, and -infinity times it not)
      }
    narrow(v);
#pragma unroll
    for (int n = 1; n < 64; n *= 2) {
      sum += __shfl_xor(sum, n);
      weighted += __shfl_xor(weighted, n);
    }
    if (lane == 0) {
      s_sum[wave] = sum;
      s_weighted[wave] = weighted;
    }
    __syncthreads();
    sum = s_sum[lane & (kWaves - 1)];
    weighted = s_weighted[lane & (kWaves - 1)];
#pragma unroll
    for (int n = 1; n < kWaves; n *= 2) {
      sum += __shfl_xor(sum, n);
      weighted += __shfl_xor(weighted, n);
    }
    const Sums t{top, sum, weighted * 0.693147181f};
    const float log_sum = logf(sum);
    float* out = ws + static_cast<size_t>(part) * (4 + 2 * k);
    if (tid == TH - 1) {
      if (WHOLE) {
        finish(a, row, t, two_t, log_sum, logit);
      } else {
        out[0] = t.top;
        out[1] = t.sum;
        out[2] = t.weighted;
      }
    }
    if (!k) {
      __syncthreads();  // the next row's first writes
      continue;
    }
    auto put = [&](int rank, uint64_t p) {
      if (!WHOLE) {
        reinterpret_cast<uint64_t*>(out + 4)[rank] = p;
      } else {
        a.top_ids[row * k + rank] = index_of(p);
        a.top_logprobs[row * k + rank] = logp_of(t, two_t, log_sum, value_of(static_cast<uint32_t>(p >> 32)));
      }
    };
    // candidates, in an order that does not matter: of the few threads that hold any. A NaN or +infinity (the sum is NaN) has
    // no order in floats and goes the long way.
    const float bound = s_bound;
    const bool odd = sum != sum;
    auto collect = [&](int which, auto&& in) {
      narrow(v);
      int t0 = tid;
      asm volatile("" : "+v"(t0));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float most = E::up(v[i][0]);
#pragma unroll
        for (int j = 1; j < V; ++j) most = __builtin_fmaxf(most, E::up(v[i][j]));
        if (!in(most)) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float f = E::up(v[i][j]);
          const int at = (i * TH + t0) * V + j;
          if (in(f) && at < len) {
            const int place = atomicAdd(&s_count[which], 1);
            if (place < kCandidates) list[place] = pack(key_of(f), from + at);
          }
        }
      }
    };
    if (!odd && own >= bound) collect(0, [&](float f) { return f >= bound; });
    __syncthreads();
    int n = s_count[0], equal = 0;  // listed; ranks left for logits equal to the bound
    if (!odd && n > kCandidates) {  // many equal ones: those above the bound, and the first that equal it
      __syncthreads();
      if (own > bound) collect(1, [&](float f) { return f > bound; });
      __syncthreads();
      n = s_count[1];
      equal = max(k - n, 0);
    }
    if (odd || n > kCandidates) {
      one_by_one<DT, TH>(logits(part), from, len, k, s_best, put);
    } else if (n <= 64) {  // a lane each
      if (wave == 0) {
        const uint64_t mine = lane < n ? list[lane] : 0;
        int rank = 0;
        for (int o = 0; o < n; ++o) {
          const uint64_t other = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), o)) << 32 |
                                 static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), o));
          rank += other > mine;
        }
        if (lane < n && rank < k) put(rank, mine);
        for (int r = n + lane; !equal && r < k; r += 64) put(r, 0);  // a last part of fewer logits
      }
    } else {
      for (int c = tid; c < n; c += TH) {
        const uint64_t mine = list[c];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += list[o] > mine;
        if (rank < k) put(rank, mine);
      }
    }
    if (equal && wave == kWaves - 1) {  // in the order of their ids
      const T* x = logits(part);
      for (int at = lane, done = 0; done < equal; at += 64) {
        const uint64_t hits = __ballot(at < len && E::up(x[min(at, len - 1)]) == bound);
        const int mine = done + __popcll(hits & ((1ull << lane) - 1));
        if ((hits >> lane & 1) && mine < equal) put(n + mine, pack(key_of(bound), from + at));
        done += __popcll(hits);
        if (at - lane >= len) break;  // (never: the bound has that many)
      }
    }
    __syncthreads();  // the next row's first writes
  }
}

// The parts of a row joined.
template <int DT>
__global__ __launch_bounds__(256) void k_logp_join(LogpArgs a, float two_t, const float* ws, int segs) {
  __shared__ uint64_t list[2048];
  const size_t row = blockIdx.x;
  const int k = static_cast<int>(a.top), step = 4 + 2 * k;
  const float* part = ws + row * segs * step;
  Sums t{-__builtin_inff(), 0.0f, 0.0f};
  for (int i = 0; i < segs; ++i) t.top = __builtin_fmaxf(t.top, part[i * step]);
  for (int i = 0; i < segs; ++i) {
    const float s = part[i * step + 1], w = part[i * step + 2];
    if (s == 0.0f) continue;
    const float d = half_less(part[i * step], 0.5f * t.top) * two_t, f = exp2_fast(d * 1.44269504f);
    t.sum = __builtin_fmaf(f, s, t.sum);
    t.weighted = __builtin_fmaf(f, __builtin_fmaf(f > 0.0f ? d : 0.0f, s, w), t.weighted);
  }
  const float log_sum = logf(t.sum);
  if (threadIdx.x == 0) finish(a, row, t, two_t, log_sum, a.ids ? given<DT>(a, row) : 0.0f);
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
    a.top_logprobs[row * k + rank] = logp_of(t, two_t, log_sum, value_of(static_cast<uint32_t>(mine >> 32)));
  }
}

}  // namespace

hipError_t launch_logp(const LogpArgs& all, float* ws, hipStream_t s) {
  return with_type(all.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const LogpPlan p = logp_plan(DT, all.V, all.rows);
    const float two_t = 2.0f / all.temperature;
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
      // as many blocks as the chip holds, all with as many parts, but for the last
      const size_t parts = a.rows * p.segs, held = 256 * (1024 / p.threads) * (p.vecs <= 2 ? 2 : 1), each = (parts + held - 1) / held;
      const unsigned grid = static_cast<unsigned>((parts + each - 1) / each);
      auto go = [&](auto threads, auto vecs) {
        constexpr int TH = decltype(threads)::value, NV = decltype(vecs)::value;
        if constexpr ((TH == 512 && NV < 8) || TH * NV * Elem<DT>::V > kLogpPart) return false;  // no plan's
        if (p.threads != TH || p.vecs != NV) return false;
        if (p.segs == 1)
          k_logp<DT, TH, NV, true><<<grid, TH, 0, s>>>(a, two_t, ws, 1);
        else if constexpr (TH * NV * Elem<DT>::V == kLogpPart)
          k_logp<DT, TH, NV, false><<<grid, TH, 0, s>>>(a, two_t, ws, p.segs);
        return true;
      };
      auto any = [&](auto threads) {
        return go(threads, std::integral_constant<int, 1>{}) || go(threads, std::integral_constant<int, 2>{}) ||
               go(threads, std::integral_constant<int, 4>{}) || go(threads, std::integral_constant<int, 8>{});
      };
      if (!any(std::integral_constant<int, 256>{}) && !any(std::integral_constant<int, 512>{}) && !any(std::integral_constant<int, 1024>{}))
        return hipErrorInvalidValue;
      hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      if (p.segs > 1) {
        k_logp_join<DT><<<static_cast<unsigned>(a.rows), 256, 0, s>>>(a, two_t, ws, p.segs);
        if ((e = hipGetLastError()) != hipSuccess) return e;
      }
    }
    return hipSuccess;
  });
}

}  // namespace mmf
