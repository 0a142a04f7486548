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
// First k of what a workgroup holds: of the maxima of separate groups of values
// the k-th largest is a bound that k values or more reach, and few more (18 of
// 16384 random ones at k = 16 and 64 groups). Those are written to LDS, and each
// one's rank among them is its place.

#include <hip/hip_runtime.h>

#include <type_traits>

#include "logprobs.h"

namespace fi {

namespace {

using u64 = unsigned long long;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWaveSize;
// 1.3e-8 too small, relatively: a term exp(-t) comes out by 1.3e-8 t too large,
// and ln S by as much with the terms' mean t, at most ln V (top 1 of 1531 rows is
// off by 5.7e-8 of itself, of which rounding to fp32 is 2.6e-8). The constant's
// rest would cost an instruction a logit.
constexpr float kLog2e = 1.44269504f;

FI_DEV float logit_of(const float* p) { return *p; }
FI_DEV float logit_of(const u16* p) { return bf16_to_f32(*p); }

// 16 bytes of logits from anywhere, past the caches: 2048 rows 95 us a call, 107
// through them, 1531 rows 77 and 86; 80 rows of 32000, which the caches still hold
// from the call before, 13.1 and 11.7
FI_DEV u32x4 read_once(const void* p) {
  typedef u32x4 __attribute__((aligned(2))) Anywhere;
  return __builtin_nontemporal_load(static_cast<const Anywhere*>(p));
}

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

// maximum of three; written out, as the compiler first maxes every operand with
// itself for the sake of signaling NaNs: one makes the maximum NaN, which the next
// fmaxf passes over, and leaves no distribution anyway
FI_DEV float max3(float a, float b, float c) {
  float v = 0.f;
#if defined(__HIP_DEVICE_COMPILE__)
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(v) : "v"(a), "v"(b), "v"(c));
#endif
  return v;
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

// The value of the lane 32, 16, 8, 4, 2 or 1 away, in a reduction that goes
// through these steps in turn: 4 away by a rotation, which takes what repeats
// every 8 lanes. STEP 7: of the lane as far from the other end of 8.
template <int STEP>
FI_DEV u32 partner(u32 v) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (STEP == 32 || STEP == 16) {
    const auto r = STEP == 32
                       ? __builtin_amdgcn_permlane32_swap(v, v, false, false)
                       : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __lane_id() & STEP ? r[0] : r[1];
  } else {
    // row_ror:8, row_half_mirror, row_ror:4, quad_perm [2,3,0,1] and [1,0,3,2]
    constexpr int ctrl = STEP == 8   ? 0x128
                         : STEP == 7 ? 0x141
                         : STEP == 4 ? 0x124
                         : STEP == 2 ? 0x4E
                                     : 0xB1;
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

// over the wave, in every lane
template <class T, class Op>
FI_DEV T over_wave(T v, Op op) {
  v = op(v, partner<32>(v));
  v = op(v, partner<16>(v));
  v = op(v, partner<8>(v));
  v = op(v, partner<4>(v));
  v = op(v, partner<2>(v));
  return op(v, partner<1>(v));
}
template <class T>
FI_DEV T larger(T a, T b) {
  return a > b ? a : b;
}
FI_DEV double wave_sum(double v) {
  return over_wave(v, [](double a, double b) { return a + b; });
}

// Sum of a chunk and its maximum.
struct alignas(16) ChunkSum {
  double s;
  float m;
};

// exp2(v): as exact as the instruction is on half a power of two
FI_DEV double power_of_2(double v) {
  const double whole = rint(v);
  const float part = __builtin_amdgcn_exp2f(static_cast<float>(v - whole));
  return whole < -1000.0
             ? 0.0
             : ldexp(static_cast<double>(part), static_cast<int>(whole));
}
// exp(v), v <= 0
FI_DEV double power(double v) { return power_of_2(v * 1.4426950408889634); }

constexpr int kHeld = 320;  // of a wave, in LDS
constexpr int kAtOnce = 8;   // compared without a question between

// how many of n keys, filled up with 0, are ahead
FI_DEV int ahead_of(const u64* keys, int n, u64 mine) {
  int count = 0;
  for (int j = 0; j < n; j += kAtOnce) {
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) count += keys[j + q] > mine;
  }
  return count;
}

// The k-th largest of the wave's N * 64 orders, from its upper bits down to bit
// LAST; the others are 0.
template <int LAST, int N>
FI_DEV u32 reached_by(const u32 (&order)[N], int k) {
  u32 bound = 0;
#pragma unroll
  for (int bit = 31; bit >= LAST; --bit) {
    const u32 next = bound | 1u << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __popcll(__ballot(order[i] >= next));
    if (count >= k) bound = next;
  }
  return bound;
}

// A workgroup's chunk: NV groups of the logits that 16 bytes hold a thread. They
// are counted from the row's first logit wherever it lies, so that
// equal rows have equal sums; what the last group lacks counts as -inf.
//
// Without choices it takes 7.6 vector instructions a bf16 logit, one of them the
// exponential of four times the cycles, about what memory leaves time for (2048
// rows of 152064: 95 us a call, 6.5 TB/s), so everything else is done per piece
// or per thread: sums go on in 64 bits every piece, after three additions in 32
// bits of bf16 logits and two of fp32 (a sum that one term dominates keeps the
// others), the bound is found from the threads' maxima, and the logits of a piece
// are looked at only where its maximum reaches it. With 16 choices it is 11
// instructions (512 rows of 151936: 31 to 32 us, 27 without).
template <typename A, int NV>
__global__ __launch_bounds__(kThreads) void logit_chunks_kernel(
    const A* __restrict__ logits, const int64_t stride, const int V,
    const int chunks, const int B, const int k, ChunkSum* __restrict__ sums,
    u64* __restrict__ keys) {
  constexpr int L = kLanes<A>, VC = NV * kThreads;
  __shared__ float s_max[kThreads];
  __shared__ double s_sum[kWaves];
  __shared__ int s_count[kWaves], s_votes[2][kWaves];
  __shared__ __attribute__((aligned(16))) u64 s_key[kWaves][kHeld + kAtOnce];
  const int tid = threadIdx.x, lane = tid % kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
  const u64 below = (1ull << lane) - 1;
  const int64_t r = blockIdx.x / chunks;
  const int c = static_cast<int>(blockIdx.x - r * chunks);
  const A* row = logits + r * stride;
  const int end = min((V + L - 1) / L, (c + 1) * VC);
  const int first = c * VC + tid;

  u32x4 raw[NV];
  // a chunk's first logit, for pieces at 32-bit distances from it
  const A* from_first = row + static_cast<int64_t>(c) * VC * L;
  if ((c + 1) * VC * L <= V) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      raw[i] = read_once(from_first + i * kThreads * L + tid * L);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = first + i * kThreads;
      const u32 none = sizeof(A) == 4 ? 0xff800000u : 0xff80ff80u;
      raw[i] = u32x4{none, none, none, none};
      if (j < end && (j + 1) * L <= V)
        raw[i] = read_once(row + static_cast<int64_t>(j) * L);
    }
    if (V % L && c == chunks - 1) {  // the last logits
      u32x4 tail = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < L; ++e) {
        const int t = V / L * L + e;
        const u32 bits =
            t < V ? __float_as_uint(logit_of(row + t)) : 0xff800000u;
        if (sizeof(A) == 4)
          tail[e % 4] = bits;
        else
          tail[e / 2] |= e % 2 ? bits : bits >> 16;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (first + i * kThreads == V / L) raw[i] = tail;
    }
  }

  float x[L], piece[NV], m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    unpack(raw[i], x, row);
    piece[i] = max3(x[0], x[1], x[2]);
#pragma unroll
    for (int e = 3; e < L; e += 2)
      piece[i] = max3(piece[i], x[e], x[min(e + 1, L - 1)]);
    m = fmaxf(m, piece[i]);
  }
  s_max[tid] = m;
  __syncthreads();
  // The groups: four threads each for small k (a sixteenth more values than k
  // reach the bound for 16 of 64 groups, two fifths for 32), a thread each up to
  // half of their number, then a piece each, whose votes the waves exchange.
  float of_thread[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    of_thread[w] = s_max[w * kWaveSize + lane];
    m = fmaxf(m, of_thread[w]);
  }
  const float of_lane = m;
  m = wave_reduce_max(m);
  const auto reached_by_pieces = [&](int last) {
    u32 order[NV], reached = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) order[i] = order_of(piece[i]);
    for (int bit = 31; bit >= last; --bit) {
      const u32 next = reached | 1u << bit;
      int count = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        count += __popcll(__ballot(order[i] >= next));
      if (lane == 0) s_votes[bit % 2][wave] = count;
      __syncthreads();
      count = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) count += s_votes[bit % 2][w];
      if (count >= k) reached = next;
    }
    return reached;
  };
  const auto reached = [&](auto last) {
    constexpr int kLast = decltype(last)::value;
    if (k <= 32) {
      const u32 order[1] = {order_of(of_lane)};
      return reached_by<kLast>(order, k);
    }
    if (k > kThreads / 2) return reached_by_pieces(kLast);
    u32 order[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) order[w] = order_of(of_thread[w]);
    return reached_by<kLast>(order, k);
  };
  // sixteen bits of the order are a bf16 value's, and as near as 2^-7 to others
  float bound = m;
  if (k > 1) {
    u32 order = reached(std::integral_constant<int, 16>());
    if (sizeof(A) == 2 && !(order >> 31)) order |= 0xffffu;
    bound = value_of(order);
  }
  // -inf is no candidate
  bound = fmaxf(bound, -3.402823466e38f);
  const float from = m == -INFINITY ? 0.f : m;

  // exp(l - from) in one multiplication and addition, l log2(e) - c. What c is
  // rounded by is the same for all, and put right below; where it would not be
  // small beside one the difference comes first.
  const float c2 = from * kLog2e;
  const bool near = fabsf(from) <= 32768.f;
  // Logits are taken apart in each pass anew and a piece at a time: kept, or all
  // at once, they would leave a SIMD half as many waves.
  const auto apart = [&](u32x4& of) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_barrier(0);
#endif
    asm volatile("" : "+v"(of));
    unpack(of, x, row);
  };
  double sum = 0.0;
  const auto add_up = [&](auto exponent) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      apart(raw[i]);
#pragma unroll
      for (int e = 0; e < L; ++e)
        x[e] = __builtin_amdgcn_exp2f(exponent(x[e]));
#pragma unroll
      for (int n = L / 2; n; n >>= 1)
#pragma unroll
        for (int e = 0; e < n; ++e) x[e] += x[e + n];
      sum += static_cast<double>(x[0]);
    }
  };
  if (near)
    add_up([&](float v) { return fmaf(v, kLog2e, -c2); });
  else
    add_up([&](float v) { return (v - from) * kLog2e; });
  asm volatile("" : "+v"(sum));
  int held = 0;
  if (k) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (held > kHeld || !__ballot(piece[i] >= bound)) continue;
      apart(raw[i]);
#pragma unroll
      for (int e = 0; e < L; ++e) {
        const u64 reach = __ballot(x[e] >= bound);
        if (reach) {
          const int at = held + __popcll(reach & below);
          if (x[e] >= bound && at < kHeld)
            s_key[wave][at] = key_of(x[e], (first + i * kThreads) * L + e);
          held += __popcll(reach);
        }
      }
    }
  }
  sum = wave_sum(sum);
  if (lane < kAtOnce && held <= kHeld) s_key[wave][held + lane] = 0;
  if (lane == 0) {
    s_sum[wave] = sum;
    s_count[wave] = held;
  }
  __syncthreads();
  if (tid == 0) {
    sum = s_sum[0];
    for (int w = 1; w < kWaves; ++w) sum += s_sum[w];
    if (near)
      sum *= power_of_2(c2 - static_cast<double>(from) * kLog2e);
    sums[blockIdx.x].s = sum;
    sums[blockIdx.x].m = m;
  }
  if (k == 0) return;

  int most = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) most = max(most, s_count[w]);
  if (most > kHeld) {
    // Many equal logits, or large ones in few of the groups. The bound becomes
    // the k-th largest logit, and of those that equal it each wave takes, by
    // index, as many as the larger ones leave of k: k in all at most.
    const auto above = [&](float v) {
      int count = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!__ballot(piece[i] > v)) continue;
        apart(raw[i]);
#pragma unroll
        for (int e = 0; e < L; ++e) count += __popcll(__ballot(x[e] > v));
      }
      __syncthreads();
      if (lane == 0) s_count[wave] = count;
      __syncthreads();
      count = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) count += s_count[w];
      return count;
    };
    if (sizeof(A) == 4 && k > 1)
      bound = fmaxf(bound,
                    value_of(reached(std::integral_constant<int, 0>())));
    int larger_ones = above(bound);
    if (larger_ones >= k) {
      u32 lo = order_of(bound), hi = order_of(m);
      while (hi - lo > 1) {
        const u32 mid = lo + (hi - lo) / 2;
        if (above(value_of(mid)) >= k)
          lo = mid;
        else
          hi = mid;
      }
      bound = value_of(hi);
      larger_ones = above(bound);
    }
    int equal = 0;
    held = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool wanted = equal < k - larger_ones ? piece[i] >= bound
                                                  : piece[i] > bound;
      if (!__ballot(wanted)) continue;
      apart(raw[i]);
      u64 same[L];
      int rank = equal;
#pragma unroll
      for (int e = 0; e < L; ++e) {
        same[e] = __ballot(x[e] == bound);
        equal += __popcll(same[e]);
        rank += __popcll(same[e] & below);
      }
#pragma unroll
      for (int e = 0; e < L; ++e) {
        const bool take =
            x[e] > bound || (x[e] == bound && rank < k - larger_ones);
        rank += x[e] == bound;
        const u64 taken = __ballot(take);
        const int at = held + __popcll(taken & below);
        if (take && at < kHeld)
          s_key[wave][at] = key_of(x[e], (first + i * kThreads) * L + e);
        held += __popcll(taken);
      }
    }
    // more only where a signaling NaN hid its piece's logits from the maximum:
    // the row has no distribution
    held = min(held, kHeld);
    if (lane < kAtOnce) s_key[wave][held + lane] = 0;
    __syncthreads();
    if (lane == 0) s_count[wave] = held;
    __syncthreads();
  }

  // [search, place, beam, chunk]
  const int64_t g = r / B;
  const int lists = B * chunks;
  u64* out = keys + g * k * lists + (blockIdx.x - g * lists);
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += s_count[w];
  for (int i = tid; i < all; i += kThreads) {
    int w = 0, at = i;
    while (at >= s_count[w]) at -= s_count[w++];
    const u64 mine = s_key[w][at];
    int rank = 0;
    for (int v = 0; v < kWaves; ++v)
      rank += ahead_of(s_key[v], s_count[v], mine);
    if (rank < k) out[static_cast<int64_t>(rank) * lists] = mine;
  }
  for (int i = all + tid; i < k; i += kThreads)
    out[static_cast<int64_t>(i) * lists] = 0;
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

// Joined by groups of 8, 16, 32 or 64 lanes, whichever hold the chunks of a row
// (64 go round), in all of the group's lanes. Rows of sums begin at `sums`.
FI_DEV int lanes_for(int chunks) {
  return chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : kWaveSize;
}
template <class T, class Op>
FI_DEV T over_lanes(T v, int lanes, Op op) {
  if (lanes > 32) v = op(v, partner<32>(v));
  if (lanes > 16) v = op(v, partner<16>(v));
  if (lanes > 8) {
    v = op(v, partner<8>(v));
    v = op(v, partner<4>(v));
  } else {
    v = op(v, partner<7>(v));
  }
  v = op(v, partner<2>(v));
  return op(v, partner<1>(v));
}
FI_DEV RowSum join_sums(const ChunkSum* sums, int chunks, int lanes) {
  const int at = threadIdx.x & (lanes - 1);
  ChunkSum own{0.0, -INFINITY};
  if (at < chunks) own = sums[at];
  float m = own.m;
  for (int c = at + kWaveSize; c < chunks; c += kWaveSize)
    m = fmaxf(m, sums[c].m);
  m = over_lanes(m, lanes, larger<float>);
  const double from = m == -INFINITY ? 0.0 : m;
  double s = own.s * power(own.m - from);
  for (int c = at + kWaveSize; c < chunks; c += kWaveSize)
    s += sums[c].s * power(sums[c].m - from);
  s = over_lanes(s, lanes, [](double a, double b) { return a + b; });
  // one term is exp(0), but the instruction rounds it in two factors: below 1
  // it would leave a log-probability above 0
  return {s > 0.0 && s < 1.0 ? 0.0 : log(s), m};
}

// The first k of the choices that `lists` lists hold, `each` of them in order:
// key(i) is that of place i / lists of list i % lists, 0 beyond a list's end,
// and choice(list, key) the choice. To put(place, choice); places that no choice
// fills get one of score 0. near(score, best) orders scores in 32 bits.
//
// A thread reads its first kAhead keys at once, before sums() joins the rows'
// sums: a join is one workgroup's chain of waits. The bound comes from groups of
// those as a chunk's does. Further places are read in turn while the last one read
// of some list reaches it. Where more reach it than LDS holds (equal ones), the
// lists are merged, a choice a round.
constexpr int kAhead = 8;
constexpr int kLastBit = 8;  // of the bound: fifteen bits of mantissa
template <int WAVES, class Key, class Sums, class Of, class Near, class Put>
FI_DEV void first_choices(const int lists, const int each, const int k,
                          Key key, Sums sums, Of choice, Near near, Put put) {
  constexpr int T = WAVES * kWaveSize, kTaken = 2 * T;
  __shared__ u64 s_top[T];
  __shared__ int s_count, s_reached[2], s_full[2], s_votes[2][WAVES];
  __shared__ __attribute__((aligned(16))) u64 s_score[kTaken];
  __shared__ u64 s_key[kTaken];
  __shared__ int s_beam[kTaken];
  __shared__ u16 s_place[WAVES > 1 ? kMostLists : kAhead * T];
  const int tid = threadIdx.x, lane = tid % kWaveSize;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWaveSize);
  const int N = lists * each;
  u64 keys[kAhead];
  const auto read = [&](int from) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int i = from + n * T + tid;
      keys[n] = i < N ? key(i) : 0;
    }
  };
  read(0);
  for (int i = tid; i < kTaken; i += T) s_score[i] = 0;
  if (tid < 2) s_reached[tid] = s_full[tid] = 0;
  if (tid == 0) s_count = 0;
  sums();
  // the lists of keys T apart
  int list = tid % lists;
  const int hop = T % lists;
  Choice got[kAhead];
  const auto weigh = [&](int from) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      got[n] = {0, 0, 0};
      if (from + n * T < N) got[n] = choice(list, keys[n]);
      list += hop;
      if (list >= lists) list -= lists;
    }
  };
  weigh(0);
  u64 top = 0;
#pragma unroll
  for (int n = 0; n < kAhead; ++n) top = larger(top, got[n].score);
  s_top[tid] = top;
  __syncthreads();
  top = 0;
  u64 tops[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    tops[w] = s_top[w * kWaveSize + lane];
    top = larger(top, tops[w]);
  }
  const u64 best = over_wave(top, larger<u64>);
  // where the first keys are all of dead rows there is nothing to be near to:
  // whatever comes later reaches the bound
  const auto order = [&](u64 score) -> u32 {
    return !score ? 0 : best ? near(score, best) : 1;
  };
  u32 of_got[kAhead], bound = 0;
#pragma unroll
  for (int n = 0; n < kAhead; ++n) of_got[n] = order(got[n].score);
  if (k <= 32) {
    const u32 of_lane[1] = {order(top)};
    bound = reached_by<kLastBit>(of_lane, k);
  } else if (k <= T / 2) {
    u32 of_thread[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) of_thread[w] = order(tops[w]);
    bound = reached_by<kLastBit>(of_thread, k);
  } else {
    for (int bit = 31; bit >= kLastBit; --bit) {
      const u32 next = bound | 1u << bit;
      int count = 0;
#pragma unroll
      for (int n = 0; n < kAhead; ++n)
        count += __popcll(__ballot(of_got[n] >= next));
      if constexpr (WAVES > 1) {
        if (lane == 0) s_votes[bit % 2][wave] = count;
        __syncthreads();
        count = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) count += s_votes[bit % 2][w];
      }
      if (count >= k) bound = next;
    }
  }
  bound = larger(bound, 1u);
  // as many rounds as hold a place of all lists make a step
  const int rounds = (lists + kAhead * T - 1) / (kAhead * T);
  const auto take = [&](int round) {
    const int step = round / rounds;
    // a key's next one of its list is another step's from here on
    const int beyond = (step + 1) * rounds * kAhead * T - lists;
    u64 reach[kAhead];
    int count = 0, at = 0;
    bool more = false;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      reach[n] = __ballot(of_got[n] >= bound);
      count += __popcll(reach[n]);
      more |= of_got[n] >= bound && (round * kAhead + n) * T + tid >= beyond;
    }
    if (!count) return;
    more = __ballot(more);
    if (lane == 0) {
      at = atomicAdd(&s_count, count);
      if (more) s_reached[step % 2] = step + 1;
      if (at + count > kTaken) s_full[step % 2] = step + 1;
    }
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int to = at + __popcll(reach[n] & ((1ull << lane) - 1));
      if (of_got[n] >= bound && to < kTaken) {
        s_score[to] = got[n].score;
        s_key[to] = got[n].key;
        s_beam[to] = got[n].beam;
      }
      at += __popcll(reach[n]);
    }
  };
  take(0);
  for (int n = 1; n * kAhead * T < N; ++n) {
    const int step = n / rounds;
    if (n % rounds == 0) {
      // what the others set from here on is the next step's
      __syncthreads();
      const int last = (step - 1) % 2;
      if (s_reached[last] != step || s_full[last] == step) break;
    }
    read(n * kAhead * T);
    weigh(n * kAhead * T);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) of_got[q] = order(got[q].score);
    take(n);
  }
  __syncthreads();
  const int all = s_count;
  if (all <= kTaken) {
    for (int i = tid; i < all; i += T) {
      const Choice mine{s_score[i], s_key[i], s_beam[i]};
      int place = 0, equal = 0;
      for (int j = 0; j < all; j += kAtOnce) {
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          place += s_score[j + q] > mine.score;
          equal += s_score[j + q] == mine.score;
        }
      }
      if (equal > 1)  // equal logits of a beam, often
        for (int j = 0; j < all; j += kAtOnce) {
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) {
            // read without a question, else each read is a branch of its own
            const u64 score = s_score[j + q], key = s_key[j + q];
            const int beam = s_beam[j + q];
            const bool first = (beam < mine.beam) |
                               ((beam == mine.beam) & (key > mine.key));
            place += (score == mine.score) & first;
          }
        }
      if (place < k) put(place, mine);
    }
    for (int i = all + tid; i < k; i += T) put(i, Choice{0, 0, 0});
    return;
  }
  // A thread's lists are T apart; it keeps the best of their heads.
  Choice head{0, 0, 0};
  int of = 0;
  const auto find = [&] {
    head = {0, 0, 0};
    for (int v = tid; v < lists; v += T) {
      const int at = s_place[v];
      if (at == each) continue;
      const Choice c = choice(v, key(at * lists + v));
      if (c.score && ahead(c, head)) {
        head = c;
        of = v;
      }
    }
  };
  __syncthreads();
  for (int v = tid; v < lists; v += T) s_place[v] = 0;
  find();
  for (int n = 0; n < k; ++n) {
    Choice first = over_wave(head, [](const Choice& a, const Choice& b) {
      return ahead(b, a) ? b : a;
    });
    __syncthreads();
    if (lane == 0) {
      s_top[wave] = first.key;
      s_score[wave] = first.score;
      s_beam[wave] = first.beam;
    }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) {
      const Choice c{s_score[w], s_top[w], s_beam[w]};
      if (ahead(c, first)) first = c;
    }
    if (tid == 0) put(n, first);
    if (first.score && first.key == head.key && first.beam == head.beam) {
      ++s_place[of];
      find();
    }
  }
}

// One workgroup per search: the k best of its beams' first tokens. Sixteen waves
// are slower than four even where 32 beams hand on 16384 keys (32 to 33 us a call,
// 24.5 with four), and for one search of 4 beams (12.3 and 10.6).
__global__ __launch_bounds__(kThreads) void beam_join_kernel(
    const ChunkSum* __restrict__ sums, const u64* __restrict__ keys,
    const int chunks, const float* __restrict__ scores,
    const int64_t group_stride, const int64_t beam_stride, const int B,
    const int each, const int k, float* __restrict__ out_scores,
    int* __restrict__ out_parents, int* __restrict__ out_tokens) {
  __shared__ RowSum s_row[kMostBeams];
  __shared__ float s_score[kMostBeams];
  const int64_t g = blockIdx.x;
  const int lists = B * chunks;
  keys += g * lists * each;
  // list / chunks: exact below 2^32 / chunks
  const u32 by_chunks = 0xffffffffu / chunks + 1;
  const bool quick =
      chunks > 1 && static_cast<int64_t>(lists) * chunks < (1ll << 32);
  first_choices<kWaves>(
      lists, each, k, [&](int i) { return keys[i]; },
      [&] {
        const int lanes = lanes_for(chunks);
        for (int b0 = 0; b0 < B; b0 += kThreads / lanes) {
          const int b = b0 + threadIdx.x / lanes;
          const int in = min(b, B - 1);  // all lanes take part
          const float c = scores[g * group_stride + in * beam_stride];
          const RowSum z =
              join_sums(sums + (g * B + in) * chunks, chunks, lanes);
          if (b < B && threadIdx.x % lanes == 0) {
            s_row[b] = z;
            s_score[b] = z.alive() ? c : NAN;
          }
        }
        __syncthreads();
      },
      [&](int list, u64 key) -> Choice {
        const int b = quick ? __umulhi(list, by_chunks) : list / chunks;
        const double c = s_score[b];
        if (!key || !finite(c)) return {0, 0, 0};
        return {score_order(c + s_row[b].of(value_of(key >> 32))), key, b};
      },
      // by how far it is from the best, whatever the scores have come to
      [](u64 score, u64 best) {
        return order_of(
            static_cast<float>(score_value(score) - score_value(best)));
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
  float of = -INFINITY;
  bool inside = false;
  if (out_given) {
    const int64_t t = given[r];
    inside = t >= 0 && t < V;
    if (inside) of = logit_of(row + t);
  }
  RowSum z;
  const auto join = [&] {
    z = join_sums(sums + r * chunks, chunks, kWaveSize);
    if (out_given && tid == 0)
      out_given[r] = !z.alive() ? NAN : inside ? z.of(of) : -INFINITY;
  };
  if (k == 0) {
    join();
    return;
  }
  out_lp += r * k;
  out_ids += r * k;
  keys += r * chunks * k;
  __shared__ int s_found;
  if (tid == 0) s_found = k;
  // by the keys alone: two log-probabilities may round to one
  first_choices<WAVES>(
      chunks, k, k, [&](int i) { return keys[i]; }, join,
      [&](int, u64 key) -> Choice {
        return {z.alive() ? key : 0, key, 0};
      },
      [](u64 key, u64) { return static_cast<u32>(key >> 32); },
      [&](int i, const Choice& c) {
        if (c.score) {
          out_lp[i] = z.of(value_of(c.key >> 32));
          out_ids[i] = token_of(c.key);
        } else if (z.alive()) {
          atomicMin(&s_found, i);
        } else {
          out_lp[i] = NAN;
          out_ids[i] = i;
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

// How a call is cut: pieces of 16 bytes a thread, chunks a row.
struct Cut {
  int nv, chunks;
};

// Chunks as large as registers hold, 8 pieces a thread, leave the least to
// join; halved until 64 workgroups share the call, as long as a chunk has four
// times as many pieces as it gives keys (256 choices of one row 32 us, 142
// without). One search of 4 beams over 151936 tokens takes 10.6 us a call so, 11.4
// to 11.7 by 256 and 2048 workgroups, which read faster but leave more to join, 2
// searches of 32 beams 24.4, by 2048 workgroups 31.7. With 4 and 16 pieces at most
// 64 searches of 8 beams take 45.5 and 42.3 us, 38.2 with 8; top tokens of 1531
// rows 82, 79 and 77. Some small calls would gain by 4: 80 fp32 rows of 32000
// 11.9 us for 13.1, 61 of 151936 14.4 for 15.1.
Cut cut_of(int64_t R, int V, int k, int size) {
  const int lanes = 16 / size;
  const int pieces = (V + lanes - 1) / lanes;
  Cut cut{8, 0};
  for (;; cut.nv /= 2) {
    cut.chunks = (pieces + cut.nv * kThreads - 1) / (cut.nv * kThreads);
    if (cut.nv == 1 || R * cut.chunks >= 64 || cut.nv * kThreads < 8 * k)
      break;
  }
  return cut;
}

}  // namespace

int64_t logit_workspace(int64_t R, int V, int k, int size) {
  return R * cut_of(R, V, k, size).chunks *
         static_cast<int64_t>(sizeof(ChunkSum) + k * sizeof(u64));
}

template <typename A>
static Cut launch_logit_chunks(const A* logits, int64_t stride, int64_t R,
                               int V, int B, int k, void* workspace,
                               hipStream_t stream) {
  const Cut cut = cut_of(R, V, k, sizeof(A));
  ChunkSum* sums = static_cast<ChunkSum*>(workspace);
  u64* keys = reinterpret_cast<u64*>(sums + R * cut.chunks);
  const dim3 grid(R * cut.chunks);
#define FI_CHUNKS(NV)                                                      \
  hipLaunchKernelGGL((logit_chunks_kernel<A, NV>), grid, dim3(kThreads), 0, \
                     stream, logits, stride, V, cut.chunks, B, k, sums, keys)
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
      launch_logit_chunks(logits, stride, G * B, V, B, each, workspace, stream);
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
  // a wave's threads hold up to 512 of them at once
  if (k <= kWaveSize && cut.chunks * k <= kAhead * kWaveSize)
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
      launch_logit_chunks(logits, stride, R, V, 1, k, workspace, stream);
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
