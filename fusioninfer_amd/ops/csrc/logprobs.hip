// Log-probabilities of rows of logits, the first k tokens of a row, and the
// choice over the beams of a search (gfx950, wave64).
//
// Row l of V tokens: m = max l_j, S = sum exp(l_j - m), log-probability
// (l_j - m) - ln S. A row whose ln S is not finite (a NaN, a +inf, -inf
// throughout) has no distribution. Tokens are ordered by logit and then by
// index, kept in one 64-bit key: the logit's order above, the complement of
// the index below.
//
// Two launches. The first reads every logit once: a workgroup holds a chunk of
// a row in registers, and finds its maximum, its sum and its first k keys. The
// second joins the chunks of a row, or of all rows of a search.
//
// First k of what the threads of a workgroup hold: the threads form at least k
// groups; the least of the groups' maxima is a bound that k values or more
// reach, and few more (of random values about k ln k, 54 of 16384 at k = 16).
// Those are written to LDS, and each one's rank among them is its place. Where
// too many values reach the bound (equal ones, or masked ones that leave a
// group without any), the k are found in as many rounds of a maximum instead.

#include <hip/hip_runtime.h>

#include "logprobs.h"

namespace fi {

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWaveSize;
constexpr float kLog2e = 1.44269504f;

FI_DEV float logit_of(const float* p) { return *p; }
FI_DEV float logit_of(const u16* p) { return bf16_to_f32(*p); }

// the logits of 16 bytes
template <typename A>
constexpr int kLanes = 16 / sizeof(A);
FI_DEV void unpack(const u32x4 raw, float (&x)[4], const float*) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(raw[e]);
}
FI_DEV void unpack(const u32x4 raw, float (&x)[8], const u16*) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(raw[e] << 16);
    x[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u);
  }
}

// order of a finite value; -0 counts as +0
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

// The partner's value for a step of a reduction that has made all lanes of
// the step's halves equal: 1, 2, 4, 8, 16 or 32 lanes away.
template <int STEP>
FI_DEV u32 partner(u32 v) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (STEP == 32 || STEP == 16) {
    const auto r = STEP == 32
                       ? __builtin_amdgcn_permlane32_swap(v, v, false, false)
                       : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const int lane = __lane_id();
    return lane & STEP ? r[0] : r[1];
  } else {
    // quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror
    constexpr int ctrl =
        STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;
    return __builtin_amdgcn_update_dpp(0, v, ctrl, 0xF, 0xF, true);
  }
#else
  return v;
#endif
}
template <int STEP>
FI_DEV float partner(float v) {
  return __uint_as_float(partner<STEP>(__float_as_uint(v)));
}
template <int STEP>
FI_DEV u64 partner(u64 v) {
  return static_cast<u64>(partner<STEP>(static_cast<u32>(v >> 32))) << 32 |
         partner<STEP>(static_cast<u32>(v));
}
template <int STEP>
FI_DEV double partner(double v) {
  return __longlong_as_double(
      partner<STEP>(static_cast<u64>(__double_as_longlong(v))));
}

// v of the lane's group of `lanes` lanes (a power of two), and of the wave
template <class T, class Op>
FI_DEV T over_group(T v, int lanes, Op op) {
  if (lanes > 1) v = op(v, partner<1>(v));
  if (lanes > 2) v = op(v, partner<2>(v));
  if (lanes > 4) v = op(v, partner<4>(v));
  if (lanes > 8) v = op(v, partner<8>(v));
  if (lanes > 16) v = op(v, partner<16>(v));
  if (lanes > 32) v = op(v, partner<32>(v));
  return v;
}
template <class T>
FI_DEV T larger(T a, T b) {
  return a > b ? a : b;
}
template <class T>
FI_DEV T smaller(T a, T b) {
  return a < b ? a : b;
}
template <class T>
FI_DEV T wave_max(T v) {
  return over_group(v, kWaveSize, larger<T>);
}

// lanes of a group so that 64 * WAVES threads form at least k of them
template <int WAVES>
FI_DEV int group_lanes(int k) {
  int lanes = kWaveSize;
  while (lanes > 1 && WAVES * kWaveSize / lanes < k) lanes >>= 1;
  return lanes;
}

// Sum of a chunk and its maximum.
struct alignas(16) ChunkSum {
  double s;
  float m;
};

constexpr int kHeld = 320;  // of a wave, in LDS

// A workgroup's chunk: VC groups of the logits that 16 bytes hold, NV of them a
// thread. They are counted from the row's first logit wherever it lies, so that
// equal rows have equal sums; what the last group lacks counts as -inf.
//
// Four instructions per logit and the exponential's four cycles more are about
// what memory leaves time for, so everything else is done per piece or per
// thread: sums go on in 64 bits every piece (a sum that one term dominates
// keeps the others), and the bound is found from the threads' maxima.
template <typename A, int NV>
__global__ __launch_bounds__(kThreads) void logit_chunks_kernel(
    const A* __restrict__ logits, const int64_t stride, const int V,
    const int chunks, const int VC, const int k, ChunkSum* __restrict__ sums,
    u64* __restrict__ keys) {
  constexpr int L = kLanes<A>;
  __shared__ float s_max[kWaves], s_bound[kWaves];
  __shared__ double s_sum[kWaves];
  __shared__ int s_count[kWaves];
  __shared__ u64 s_key[kWaves][kHeld];
  const int tid = threadIdx.x, lane = tid % kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
  const int64_t r = blockIdx.x / chunks;
  const int c = static_cast<int>(blockIdx.x - r * chunks);
  const A* row = logits + r * stride;
  const int end = min((V + L - 1) / L, (c + 1) * VC);
  const int first = c * VC + tid;

  u32x4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = first + i * kThreads;
    const u32 none = sizeof(A) == 4 ? 0xff800000u : 0xff80ff80u;
    raw[i] = u32x4{none, none, none, none};
    if (j < end && (j + 1) * L <= V)
      __builtin_memcpy(&raw[i], row + static_cast<int64_t>(j) * L, 16);
  }
  if (V % L && (c + 1) * VC >= V / L) {  // the last logits
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = first + i * kThreads;
      if (j >= end || j != V / L) continue;
#pragma unroll
      for (int e = 0; e < L; ++e) {
        if (j * L + e >= V) continue;
        const u32 bits = __float_as_uint(logit_of(row + j * L + e));
        if (sizeof(A) == 4)
          raw[i][e % 4] = bits;
        else if (e % 2)
          raw[i][e / 2] = (raw[i][e / 2] & 0xffffu) | bits;
        else
          raw[i][e / 2] = (raw[i][e / 2] & 0xffff0000u) | bits >> 16;
      }
    }
  }

  float x[L], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    unpack(raw[i], x, row);
#pragma unroll
    for (int e = 0; e < L; ++e) m = fmaxf(m, x[e]);
  }
  const int lanes = group_lanes<kWaves>(k);
  const float group = over_group(m, lanes, larger<float>);
  const float least = over_group(group, kWaveSize, smaller<float>);
  m = wave_max(group);
  if (lane == 0) {
    s_max[wave] = m;
    s_bound[wave] = least;
  }
  __syncthreads();
  float bound = s_bound[0];
  m = s_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    m = fmaxf(m, s_max[w]);
    bound = fminf(bound, s_bound[w]);
  }
  if (k == 1) bound = m;
  // -inf is no candidate
  bound = fmaxf(bound, -3.402823466e38f);
  const float from = m == -INFINITY ? 0.f : m;

  double sum = 0.0;
  int held = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    unpack(raw[i], x, row);
    float e2[L];
#pragma unroll
    for (int e = 0; e < L; ++e)
      e2[e] = __builtin_amdgcn_exp2f((x[e] - from) * kLog2e);
#pragma unroll
    for (int n = L / 2; n; n >>= 1)
#pragma unroll
      for (int e = 0; e < n; ++e) e2[e] += e2[e + n];
    sum += static_cast<double>(e2[0]);
    if (k == 0) continue;
#pragma unroll
    for (int e = 0; e < L; ++e) {
      const u64 reach = __ballot(x[e] >= bound);
      if (reach) {
        const int at = held + __popcll(reach & ((1ull << lane) - 1));
        if (x[e] >= bound && at < kHeld)
          s_key[wave][at] =
              key_of(x[e], (first + i * kThreads) * L + e);
        held += __popcll(reach);
      }
    }
  }
  sum = over_group(sum, kWaveSize, [](double a, double b) { return a + b; });
  if (lane == 0) {
    s_sum[wave] = sum;
    s_count[wave] = held;
  }
  __syncthreads();
  if (tid == 0) {
    sum = s_sum[0];
    for (int w = 1; w < kWaves; ++w) sum += s_sum[w];
    sums[blockIdx.x].s = sum;
    sums[blockIdx.x].m = m;
  }
  if (k == 0) return;

  u64* out = keys + static_cast<int64_t>(blockIdx.x) * k;
  int all = 0, most = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    all += s_count[w];
    most = max(most, s_count[w]);
  }
  if (most <= kHeld && k <= kThreads) {
    for (int i = tid; i < all; i += kThreads) {
      int w = 0, at = i;
      while (at >= s_count[w]) at -= s_count[w++];
      const u64 mine = s_key[w][at];
      int rank = 0;
      for (int v = 0; v < kWaves; ++v) {
        const int n = s_count[v];
        for (int j = 0; j < n; ++j) rank += s_key[v][j] > mine;
      }
      if (rank < k) out[rank] = mine;
    }
    for (int i = all + tid; i < k; i += kThreads) out[i] = 0;
    return;
  }
  u64 last = ~0ull;
  for (int n = 0; n < k; ++n) {
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack(raw[i], x, row);
#pragma unroll
      for (int e = 0; e < L; ++e) {
        const u64 key = key_of(x[e], (first + i * kThreads) * L + e);
        if (x[e] > -INFINITY && key < last && key > best) best = key;
      }
    }
    best = wave_max(best);
    __syncthreads();
    if (lane == 0) s_key[wave][0] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = larger(best, s_key[w][0]);
    if (tid == 0) out[n] = best;
    last = best;
    if (!best) {
      for (int i = n + 1 + tid; i < k; i += kThreads) out[i] = 0;
      return;
    }
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
template <int STEP>
FI_DEV Choice partner(const Choice& c) {
  return {partner<STEP>(c.score), partner<STEP>(c.key),
          static_cast<int>(partner<STEP>(static_cast<u32>(c.beam)))};
}

FI_DEV bool finite(double v) { return v - v == 0.0; }

// Maximum and ln S of a row. m + ln S is not formed: where m is the type's
// lowest value it would leave nothing of ln S even in 64 bits.
struct RowSum {
  double ln;
  float m;
  FI_DEV bool alive() const { return finite(ln); }
  FI_DEV double of(float v) const { return (static_cast<double>(v) - m) - ln; }
};

// by one wave, in all of its lanes
FI_DEV RowSum join_sums(const ChunkSum* sums, int chunks, int lane) {
  float m = -INFINITY;
  for (int c = lane; c < chunks; c += kWaveSize) m = fmaxf(m, sums[c].m);
  m = wave_max(m);
  const double from = m == -INFINITY ? 0.0 : m;
  double s = 0.0;
  for (int c = lane; c < chunks; c += kWaveSize)
    s += sums[c].s * exp(sums[c].m - from);
  s = over_group(s, kWaveSize, [](double a, double b) { return a + b; });
  return {log(s), m};
}

constexpr int kJoined = 192;  // of a wave, in LDS

// The first k of N choices, `at(i)` the i-th one, to put(place, choice); places
// that no choice fills get one of score 0.
template <int WAVES, class At, class Put>
FI_DEV void first_choices(const int N, const int k, At at, Put put) {
  __shared__ u64 s_bound[WAVES];
  __shared__ int s_count[WAVES];
  __shared__ Choice s_choice[WAVES][kJoined];
  constexpr int T = WAVES * kWaveSize;
  const int tid = threadIdx.x, lane = tid % kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
  int all = 0, most = kJoined + 1;
  if (k <= T) {
    u64 top = 0;
    for (int i = tid; i < N; i += T) top = larger(top, at(i).score);
    const int lanes = group_lanes<WAVES>(k);
    top = over_group(top, lanes, larger<u64>);
    top = over_group(top, kWaveSize, smaller<u64>);
    if (lane == 0) s_bound[wave] = top;
    __syncthreads();
    u64 bound = s_bound[0];
    for (int w = 1; w < WAVES; ++w) bound = smaller(bound, s_bound[w]);
    bound = larger<u64>(bound, 1);
    int held = 0;
    for (int i0 = wave * kWaveSize; i0 < N; i0 += T) {
      const int i = i0 + lane;
      Choice c{0, 0, 0};
      if (i < N) c = at(i);
      const u64 reach = __ballot(c.score >= bound);
      const int to = held + __popcll(reach & ((1ull << lane) - 1));
      if (c.score >= bound && to < kJoined) s_choice[wave][to] = c;
      held += __popcll(reach);
    }
    if (lane == 0) s_count[wave] = held;
    __syncthreads();
    most = 0;
    for (int w = 0; w < WAVES; ++w) {
      all += s_count[w];
      most = max(most, s_count[w]);
    }
  }
  if (most <= kJoined) {
    for (int i = tid; i < all; i += T) {
      int w = 0, j = i;
      while (j >= s_count[w]) j -= s_count[w++];
      const Choice mine = s_choice[w][j];
      int rank = 0;
      for (int v = 0; v < WAVES; ++v) {
        const int n = s_count[v];
        for (int q = 0; q < n; ++q) rank += ahead(s_choice[v][q], mine);
      }
      if (rank < k) put(rank, mine);
    }
    for (int i = all + tid; i < k; i += T) put(i, Choice{0, 0, 0});
    return;
  }
  Choice last{~0ull, 0, -1};
  for (int n = 0; n < k; ++n) {
    Choice best{0, 0, 0};
    if (last.score)
      for (int i = tid; i < N; i += T) {
        const Choice c = at(i);
        if (c.score && ahead(last, c) && ahead(c, best)) best = c;
      }
    best = over_group(best, kWaveSize, [](const Choice& a, const Choice& b) {
      return ahead(b, a) ? b : a;
    });
    __syncthreads();
    if (lane == 0) s_choice[wave][0] = best;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w)
      if (ahead(s_choice[w][0], best)) best = s_choice[w][0];
    if (tid == 0) put(n, best);
    last = best;
  }
}

// One workgroup per search: the k best of its beams' first tokens.
__global__ __launch_bounds__(kThreads) void beam_join_kernel(
    const ChunkSum* __restrict__ sums, const u64* __restrict__ keys,
    const int chunks, const float* __restrict__ scores,
    const int64_t group_stride, const int64_t beam_stride, const int B,
    const int each, const int k, float* __restrict__ out_scores,
    int* __restrict__ out_parents, int* __restrict__ out_tokens) {
  __shared__ RowSum s_row[kMostBeams];
  __shared__ float s_score[kMostBeams];
  const int64_t g = blockIdx.x;
  const int lane = threadIdx.x % kWaveSize;
  for (int b = threadIdx.x / kWaveSize; b < B; b += kWaves) {
    const RowSum z = join_sums(sums + (g * B + b) * chunks, chunks, lane);
    if (lane == 0) {
      s_row[b] = z;
      const float c = scores[g * group_stride + b * beam_stride];
      s_score[b] = z.alive() ? c : NAN;
    }
  }
  __syncthreads();
  const int of_beam = chunks * each;
  keys += g * B * of_beam;
  first_choices<kWaves>(
      B * of_beam, k,
      [&](int i) -> Choice {
        const u64 key = keys[i];
        const int b = i / of_beam;
        const double c = s_score[b];
        if (!key || !finite(c)) return {0, 0, 0};
        return {score_order(c + s_row[b].of(value_of(key >> 32))), key, b};
      },
      [&](int i, const Choice& c) {
        const bool some = c.score != 0;
        out_scores[g * k + i] =
            some ? static_cast<float>(score_value(c.score)) : -INFINITY;
        out_parents[g * k + i] = some ? c.beam : -1;
        out_tokens[g * k + i] = some ? token_of(c.key) : -1;
      });
}

// One workgroup per row: log-probabilities of its first k tokens and of a
// given one. Where fewer than k tokens are above -inf, the others follow by
// index.
template <typename A, typename I, int WAVES>
__global__ __launch_bounds__(WAVES * kWaveSize) void top_join_kernel(
    const A* __restrict__ logits, const int64_t stride, const int V,
    const ChunkSum* __restrict__ sums, const u64* __restrict__ keys,
    const int chunks, const int k, const I* __restrict__ given,
    float* __restrict__ out_lp, int* __restrict__ out_ids,
    float* __restrict__ out_given) {
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWaveSize;
  const A* row = logits + r * stride;
  const RowSum z = join_sums(sums + r * chunks, chunks, lane);
  const bool some = z.alive();
  if (out_given && tid == 0) {
    const int64_t t = given[r];
    float v = -INFINITY;
    if (t >= 0 && t < V) v = z.of(logit_of(row + t));
    out_given[r] = some ? v : NAN;
  }
  if (k == 0) return;
  out_lp += r * k;
  out_ids += r * k;
  if (!some) {
    for (int i = tid; i < k; i += WAVES * kWaveSize) {
      out_lp[i] = NAN;
      out_ids[i] = i;
    }
    return;
  }
  keys += r * chunks * k;
  __shared__ int s_found;
  if (tid == 0) s_found = k;
  __syncthreads();
  // by the keys alone: two log-probabilities may round to one
  first_choices<WAVES>(
      chunks * k, k,
      [&](int i) -> Choice {
        const u64 key = keys[i];
        return {key, key, 0};
      },
      [&](int i, const Choice& c) {
        if (c.score) {
          out_lp[i] = z.of(value_of(c.key >> 32));
          out_ids[i] = token_of(c.key);
        } else {
          atomicMin(&s_found, i);
        }
      });
  __syncthreads();
  int found = s_found;
  if (tid >= kWaveSize) return;
  for (int j0 = 0; found < k && j0 < V; j0 += kWaveSize) {
    const int j = j0 + lane;
    const bool none = j < V && logit_of(row + j) == -INFINITY;
    const u64 mask = __ballot(none);
    const int i = found + __popcll(mask & ((1ull << lane) - 1));
    if (none && i < k) {
      out_lp[i] = -INFINITY;
      out_ids[i] = j;
    }
    found += __popcll(mask);
  }
}

// How a call is cut: NV pieces of 16 bytes a thread, VC a chunk.
struct Cut {
  int nv, chunks, vc;
};

// Chunks as large as registers hold, 8 pieces a thread, leave the least to
// join; halved until about four workgroups a CU share the call.
Cut cut_of(int64_t R, int V, int size) {
  const int lanes = 16 / size;
  const int pieces = (V + lanes - 1) / lanes;
  Cut cut{8, 0, 0};
  for (;; cut.nv /= 2) {
    cut.chunks = (pieces + cut.nv * kThreads - 1) / (cut.nv * kThreads);
    if (cut.nv == 1 || R * cut.chunks >= 1024) break;
  }
  cut.vc = (pieces + cut.chunks - 1) / cut.chunks;
  return cut;
}

}  // namespace

int64_t logit_workspace(int64_t R, int V, int k, int size) {
  return R * cut_of(R, V, size).chunks *
         static_cast<int64_t>(sizeof(ChunkSum) + k * sizeof(u64));
}

template <typename A>
static Cut launch_logit_chunks(const A* logits, int64_t stride, int64_t R,
                               int V, int k, void* workspace,
                               hipStream_t stream) {
  const Cut cut = cut_of(R, V, sizeof(A));
  ChunkSum* sums = static_cast<ChunkSum*>(workspace);
  u64* keys = reinterpret_cast<u64*>(sums + R * cut.chunks);
  const dim3 grid(R * cut.chunks);
#define FI_CHUNKS(NV)                                                      \
  hipLaunchKernelGGL((logit_chunks_kernel<A, NV>), grid, dim3(kThreads), 0, \
                     stream, logits, stride, V, cut.chunks, cut.vc, k, sums, \
                     keys)
  if (cut.nv == 8)
    FI_CHUNKS(8);
  else if (cut.nv == 4)
    FI_CHUNKS(4);
  else if (cut.nv == 2)
    FI_CHUNKS(2);
  else
    FI_CHUNKS(1);
#undef FI_CHUNKS
  return cut;
}

template <typename A>
void launch_beam_select(const A* logits, int64_t stride, int V,
                        const float* scores, int64_t group_stride,
                        int64_t beam_stride, int64_t G, int B, int k,
                        void* workspace, float* out_scores, int* out_parents,
                        int* out_tokens, hipStream_t stream) {
  const int each = std::min(k, V);
  const Cut cut =
      launch_logit_chunks(logits, stride, G * B, V, each, workspace, stream);
  const ChunkSum* sums = static_cast<const ChunkSum*>(workspace);
  hipLaunchKernelGGL(
      beam_join_kernel, dim3(G), dim3(kThreads), 0, stream, sums,
      reinterpret_cast<const u64*>(sums + G * B * cut.chunks), cut.chunks,
      scores, group_stride, beam_stride, B, each, k, out_scores, out_parents,
      out_tokens);
}

template <typename A, typename I>
static void launch_top_join(const A* logits, int64_t stride, int64_t R, int V,
                            const Cut& cut, int k, const I* given,
                            const ChunkSum* sums, float* out_lp, int* out_ids,
                            float* out_given, hipStream_t stream) {
  const u64* keys = reinterpret_cast<const u64*>(sums + R * cut.chunks);
  // a wave finds up to 64 in one go
  if (k <= kWaveSize && cut.chunks * k <= 512)
    hipLaunchKernelGGL((top_join_kernel<A, I, 1>), dim3(R), dim3(kWaveSize), 0,
                       stream, logits, stride, V, sums, keys, cut.chunks, k,
                       given, out_lp, out_ids, out_given);
  else
    hipLaunchKernelGGL((top_join_kernel<A, I, kWaves>), dim3(R),
                       dim3(kThreads), 0, stream, logits, stride, V, sums,
                       keys, cut.chunks, k, given, out_lp, out_ids, out_given);
}

template <typename A>
void launch_top_logprobs(const A* logits, int64_t stride, int64_t R, int V,
                         int k, const void* given, bool wide, void* workspace,
                         float* out_lp, int* out_ids, float* out_given,
                         hipStream_t stream) {
  const Cut cut =
      launch_logit_chunks(logits, stride, R, V, k, workspace, stream);
  const ChunkSum* sums = static_cast<const ChunkSum*>(workspace);
  if (wide)
    launch_top_join(logits, stride, R, V, cut, k,
                    static_cast<const int64_t*>(given), sums, out_lp, out_ids,
                    out_given, stream);
  else
    launch_top_join(logits, stride, R, V, cut, k,
                    static_cast<const int*>(given), sums, out_lp, out_ids,
                    out_given, stream);
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
