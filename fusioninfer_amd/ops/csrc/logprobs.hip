// Log-probabilities of rows of logits, the first k tokens of a row, and the
// choice over the beams of a search (gfx950, wave64).
//
// Row l of V tokens: m = max l_j, S = sum exp(l_j - m), log-probability
// (l_j - m) - ln S. A row whose ln S is not finite (a NaN, a +inf, -inf
// throughout) has no distribution.
// Tokens are ordered by logit and then by index, kept in one 64-bit key:
// the logit's order above, the complement of the index below.

#include <hip/hip_runtime.h>

#include "logprobs.h"

namespace fi {

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWaveSize;

FI_DEV float logit_of(const float* p) { return *p; }
FI_DEV float logit_of(const u16* p) { return bf16_to_f32(*p); }

// order of a finite value (or -inf); -0 counts as +0
FI_DEV u32 order_of(float v) {
  const u32 u = __float_as_uint(v + 0.f);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
FI_DEV float value_of(u32 order) {
  return __uint_as_float(order ^ (order >> 31 ? 0x80000000u : 0xffffffffu));
}
FI_DEV u64 key_of(float v, int token) {
  return static_cast<u64>(order_of(v)) << 32 |
         (0xffffffffu - static_cast<u32>(token));
}
FI_DEV int token_of(u64 key) {
  return static_cast<int>(0xffffffffu - static_cast<u32>(key));
}

FI_DEV u64 shuffle_xor(u64 v, int by) {
  const int lo = __shfl_xor(static_cast<int>(v), by);
  const int hi = __shfl_xor(static_cast<int>(v >> 32), by);
  return static_cast<u64>(static_cast<u32>(hi)) << 32 | static_cast<u32>(lo);
}

// maximum over the workgroup, in every thread
FI_DEV u64 block_max(u64 v, u64* scratch) {
  for (int by = 32; by; by >>= 1) {
    const u64 o = shuffle_xor(v, by);
    v = o > v ? o : v;
  }
  __syncthreads();
  if (threadIdx.x % kWaveSize == 0) scratch[threadIdx.x / kWaveSize] = v;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) v = scratch[w] > v ? scratch[w] : v;
  return v;
}

// One workgroup per row: maximum and sum of the exponentials below it, and
// the k first keys, one round of the workgroup each (0: no such token).
template <typename A>
__global__ __launch_bounds__(kThreads) void logit_rows_kernel(
    const A* __restrict__ logits, const int64_t stride, const int V,
    const int k, float2* __restrict__ stats, u64* __restrict__ keys) {
  __shared__ u64 scratch[kWaves];
  __shared__ float fscratch[kWaves];
  const A* row = logits + blockIdx.x * stride;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < V; j += kThreads)
    m = fmaxf(m, logit_of(row + j));
  m = block_reduce_max<kWaves>(wave_reduce_max(m), fscratch);
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f;
  for (int j = threadIdx.x; j < V; j += kThreads)
    s += exp2f((logit_of(row + j) - base) * 1.44269504f);
  __syncthreads();
  s = block_reduce_sum<kWaves>(wave_reduce_sum(s), fscratch);
  if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(m, s);
  u64 last = ~0ull;
  for (int i = 0; i < k; ++i) {
    u64 best = 0;
    if (last) {
      for (int j = threadIdx.x; j < V; j += kThreads) {
        const float v = logit_of(row + j);
        if (v > -INFINITY) {
          const u64 key = key_of(v, j);
          if (key < last && key > best) best = key;
        }
      }
    }
    last = block_max(best, scratch);
    if (threadIdx.x == 0) keys[static_cast<int64_t>(blockIdx.x) * k + i] = last;
  }
}

// A candidate: its score's order, its beam, its key; none has score 0.
struct Choice {
  u64 score, key;
  int beam;
};
FI_DEV bool ahead(const Choice& a, const Choice& b) {
  if (a.score != b.score) return a.score > b.score;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}
FI_DEV u64 score_order(double s) {
  const u64 u = __double_as_longlong(s + 0.0);
  return u ^ (u >> 63 ? ~0ull : 1ull << 63);
}
FI_DEV double score_value(u64 order) {
  return __longlong_as_double(order ^ (order >> 63 ? 1ull << 63 : ~0ull));
}

FI_DEV Choice block_first(Choice c, Choice* scratch) {
  for (int by = 32; by; by >>= 1) {
    const Choice o{shuffle_xor(c.score, by), shuffle_xor(c.key, by),
                   __shfl_xor(c.beam, by)};
    if (ahead(o, c)) c = o;
  }
  __syncthreads();
  if (threadIdx.x % kWaveSize == 0) scratch[threadIdx.x / kWaveSize] = c;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w)
    if (ahead(scratch[w], c)) c = scratch[w];
  return c;
}

FI_DEV bool finite(double v) { return v - v == 0.0; }

// Maximum and ln S of a row. m + ln S is not formed: where m is the type's
// lowest value it would leave nothing of ln S even in 64 bits.
struct RowSum {
  double m, ln;
  FI_DEV explicit RowSum(const float2 s)
      : m(s.x), ln(log(static_cast<double>(s.y))) {}
  FI_DEV bool alive() const { return finite(ln); }
  FI_DEV double of(float v) const { return (v - m) - ln; }
};

// One workgroup per search: the k best of its beams' first tokens.
__global__ __launch_bounds__(kThreads) void beam_join_kernel(
    const float2* __restrict__ stats, const u64* __restrict__ keys,
    const float* __restrict__ scores, const int64_t group_stride,
    const int64_t beam_stride, const int B, const int each, const int k,
    float* __restrict__ out_scores, int* __restrict__ out_parents,
    int* __restrict__ out_tokens) {
  __shared__ Choice scratch[kWaves];
  const int64_t g = blockIdx.x;
  Choice last{~0ull, 0, -1};
  for (int i = 0; i < k; ++i) {
    Choice best{0, 0, 0};
    if (last.score) {
      for (int j = threadIdx.x; j < B * each; j += kThreads) {
        const int b = j / each;
        const u64 key = keys[g * B * each + j];
        const RowSum z(stats[g * B + b]);
        const double c = scores[g * group_stride + b * beam_stride];
        if (!key || !z.alive() || !finite(c)) continue;
        const float v = value_of(static_cast<u32>(key >> 32));
        const Choice o{score_order(c + z.of(v)), key, b};
        if (ahead(last, o) && ahead(o, best)) best = o;
      }
    }
    last = block_first(best, scratch);
    if (threadIdx.x == 0) {
      const bool some = last.score != 0;
      out_scores[g * k + i] =
          some ? static_cast<float>(score_value(last.score)) : -INFINITY;
      out_parents[g * k + i] = some ? last.beam : -1;
      out_tokens[g * k + i] = some ? token_of(last.key) : -1;
    }
  }
}

// One wave per row: log-probabilities of its first k tokens and of a given
// one. Where fewer than k tokens are above -inf, the others follow by index.
template <typename A, typename I>
__global__ __launch_bounds__(kWaveSize) void top_join_kernel(
    const A* __restrict__ logits, const int64_t stride, const int V,
    const float2* __restrict__ stats, const u64* __restrict__ keys,
    const int k, const I* __restrict__ given, float* __restrict__ out_lp,
    int* __restrict__ out_ids, float* __restrict__ out_given) {
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x;
  const RowSum z(stats[r]);
  const bool some = z.alive();
  if (out_given && lane == 0) {
    const int64_t t = given[r];
    float v = -INFINITY;
    if (t >= 0 && t < V) v = z.of(logit_of(logits + r * stride + t));
    out_given[r] = some ? v : NAN;
  }
  int found = 0;
  for (int i0 = 0; i0 < k; i0 += kWaveSize) {
    const int i = i0 + lane;
    const u64 key = i < k && some ? keys[r * k + i] : 0;
    if (key) {
      out_lp[r * k + i] = z.of(value_of(static_cast<u32>(key >> 32)));
      out_ids[r * k + i] = token_of(key);
    }
    found += __popcll(__ballot(key != 0));
  }
  if (!some) {
    for (int i = lane; i < k; i += kWaveSize) {
      out_lp[r * k + i] = NAN;
      out_ids[r * k + i] = i;
    }
    return;
  }
  for (int j0 = 0; found < k && j0 < V; j0 += kWaveSize) {
    const int j = j0 + lane;
    const bool none = j < V && logit_of(logits + r * stride + j) == -INFINITY;
    const u64 mask = __ballot(none);
    const int i = found + __popcll(mask & ((1ull << lane) - 1));
    if (none && i < k) {
      out_lp[r * k + i] = -INFINITY;
      out_ids[r * k + i] = j;
    }
    found += __popcll(mask);
  }
}

}  // namespace

int64_t logit_workspace(int64_t R, int, int k) {
  return R * static_cast<int64_t>(sizeof(float2) + k * sizeof(u64));
}

template <typename A>
static void launch_logit_rows(const A* logits, int64_t stride, int64_t R,
                              int V, int k, void* workspace,
                              hipStream_t stream) {
  float2* stats = static_cast<float2*>(workspace);
  hipLaunchKernelGGL((logit_rows_kernel<A>), dim3(R), dim3(kThreads), 0,
                     stream, logits, stride, V, k, stats,
                     reinterpret_cast<u64*>(stats + R));
}

template <typename A>
void launch_beam_select(const A* logits, int64_t stride, int V,
                        const float* scores, int64_t group_stride,
                        int64_t beam_stride, int64_t G, int B, int k,
                        void* workspace, float* out_scores, int* out_parents,
                        int* out_tokens, hipStream_t stream) {
  const int each = std::min(k, V);
  launch_logit_rows(logits, stride, G * B, V, each, workspace, stream);
  float2* stats = static_cast<float2*>(workspace);
  hipLaunchKernelGGL(beam_join_kernel, dim3(G), dim3(kThreads), 0, stream,
                     stats, reinterpret_cast<u64*>(stats + G * B), scores,
                     group_stride, beam_stride, B, each, k, out_scores,
                     out_parents, out_tokens);
}

template <typename A>
void launch_top_logprobs(const A* logits, int64_t stride, int64_t R, int V,
                         int k, const void* given, bool wide, void* workspace,
                         float* out_lp, int* out_ids, float* out_given,
                         hipStream_t stream) {
  launch_logit_rows(logits, stride, R, V, k, workspace, stream);
  float2* stats = static_cast<float2*>(workspace);
  const u64* keys = reinterpret_cast<u64*>(stats + R);
  if (wide)
    hipLaunchKernelGGL((top_join_kernel<A, int64_t>), dim3(R),
                       dim3(kWaveSize), 0, stream, logits, stride, V, stats,
                       keys, k, static_cast<const int64_t*>(given), out_lp,
                       out_ids, out_given);
  else
    hipLaunchKernelGGL((top_join_kernel<A, int>), dim3(R), dim3(kWaveSize), 0,
                       stream, logits, stride, V, stats, keys, k,
                       static_cast<const int*>(given), out_lp, out_ids,
                       out_given);
}

#define FI_LOGPROBS(A)                                                       \
  template void launch_beam_select<A>(const A*, int64_t, int, const float*,  \
                                      int64_t, int64_t, int64_t, int, int,   \
                                      void*, float*, int*, int*,             \
                                      hipStream_t);                          \
  template void launch_top_logprobs<A>(const A*, int64_t, int64_t, int, int, \
                                       const void*, bool, void*, float*,     \
                                       int*, float*, hipStream_t);
FI_LOGPROBS(float)
FI_LOGPROBS(u16)

}  // namespace fi
