// Operators of a layer of experts: the choice of each token's experts with its
// backward pass, the counting sort that puts (token, choice) pairs in the order
// of their experts, the copy of the rows into that order, the weighted sum back
// with its backward pass, and the update of the balance bias.
//
// No matrix product is involved.  The moves are bound by memory: 65536 slots of 2048
// bfloat16 columns take 50 us to dispatch (93 % of the measured copy rate), 55 to combine with a
// residual (94 %), 98 for the backward pass (90 %), 48 without weights (98 %).  The choice is
// bound by the latency of its dependent maxima: 65536 tokens of 128 float32 logits take 21 us,
// the bytes 5.8; its gradient 18 of 11.0, for the instructions of expf.
#include <math.h>

#include "dgn_kernels.cuh"
#include "dgn_ops.h"

namespace {

using namespace dgn;

constexpr int kMaxExperts = DGN_MAX_EXPERTS, kMaxGroups = DGN_MAX_GROUPS;
constexpr int kMaxChoices = DGN_MAX_CHOICES;  // one lane of a warp for each
constexpr int64_t kMaxRow = 1 << 30;  // so that a column plus a block's width stays a 32-bit number
constexpr float kTiny = 1e-20f;  // keeps the sum that weights are divided by from zero
constexpr unsigned kFull = 0xffffffffu;

template <typename T> __device__ __forceinline__ float widen(T v) { return static_cast<float>(v); }

// ---- choice ------------------------------------------------------------------------------

struct RouteParams {
  const char* logits;
  const float* bias;
  const uint8_t* mask;
  int* indices;
  float* weights;
  long long tokens, stride;
  int experts, k, sigmoid, groups, keep, best, renormalize;
  int bits;        // of an expert's number
  unsigned magic;  // e * magic >> 20 is expert e's group
  int group_lanes; // lanes whose vectors make up a group; 0: not a power of two of them in one team
  float scale;
};

// Keys as whole numbers that sort like the values: 0 is "not to be chosen" (-inf), NaN comes first.
__device__ __forceinline__ u64 order_of(double v) {
  u64 bits = (u64)__double_as_longlong(v);
  if (bits << 1 > 0xffe0000000000000ull) return ~0ull;  // NaN
  if (bits == 0xfff0000000000000ull) return 0;           // -inf
  if (bits == 1ull << 63) bits = 0;                      // -0
  return bits >> 63 ? ~bits : bits | 1ull << 63;
}
__device__ __forceinline__ double value_of(u64 order) {  // of any key but 0
  return __longlong_as_double((long long)(order >> 63 ? order ^ 1ull << 63 : ~order));
}
// The same for float32, -inf and NaN left aside.
__device__ __forceinline__ unsigned order_of(float v) {
  const int bits = __float_as_int(v + 0.f);
  return bits ^ (bits >> 31 | 1 << 31);
}

// Largest key of a warp and the lowest index that has it, the halves of the key one after the other.
__device__ __forceinline__ void first_largest(u64* key, int* index) {
  const unsigned high = *key >> 32, most = __reduce_max_sync(kFull, high);
  const unsigned low = high == most ? (unsigned)*key : 0, rest = __reduce_max_sync(kFull, low);
  *index = __reduce_min_sync(kFull, high == most && low == rest ? (unsigned)*index : ~0u);
  *key = (u64)most << 32 | rest;
}

// Scores of four logits in 64 bits; `over` is the softmax's sum (0: its terms are wanted alone).  One copy for all kernels:
// the few warps that take an exact path wait for its instructions to arrive, and for one value after the other unless
// several are under way.
__device__ __noinline__ void exact_scores(double* v, int sigmoid, double top, double over) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double e = exp(sigmoid ? -v[i] : v[i] - top);
    v[i] = sigmoid ? 1.0 / (1.0 + e) : over != 0.0 ? e / over : e;
  }
}

// One token's choice in 64 bits by a whole warp, its keys' orders in shared memory.  Taken by the
// tokens whose choice hangs on values that float32 does not tell apart, and by those that
// hold a NaN or an infinity: about one in a thousand of random logits, but a small batch waits for
// that one.  Float32 rows with more equal logits at the border than it can put in order go here
// too, though their order is plain: 65536 tokens of 128 equal logits take 188 us, 21 of random ones.
template <typename T>
__device__ __noinline__ void route_exact(const RouteParams& p, long long token, u64* key) {
  const int lane = threadIdx.x & 31, experts = p.experts;
  const T* row = reinterpret_cast<const T*>(p.logits) + token * p.stride;
  // With groups whose values are sums of scores, the scores come first and the logits take their place.
  const bool sums = p.groups > 1 && p.best == 2 && !p.bias;
  float top = -INFINITY;
  for (int e = lane; e < experts; e += 32) top = fmaxf(top, widen(row[e]));
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
  double sum = 0.0;
  if (!p.sigmoid) {
#pragma unroll 1
    for (int base = lane; base < experts; base += 128) {
      double v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = base + i * 32 < experts ? (double)widen(row[base + i * 32]) : -INFINITY;
      exact_scores(v, 0, top, 0.0);  // -inf gives 0
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
  }
  __syncwarp();
#pragma unroll 1
  for (int base = lane; base < experts; base += 128) {
    double v[4];
    bool none[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = base + i * 32 < experts ? (double)widen(row[base + i * 32]) : -INFINITY;
      none[i] = (float)v[i] == -INFINITY;
    }
    if (p.bias || sums) exact_scores(v, p.sigmoid, top, sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = base + i * 32;
      if (e < experts) key[e] = none[i] ? 0 : order_of(p.bias ? v[i] + (double)p.bias[e] : v[i]);
    }
  }
  __syncwarp();
  if (p.groups > 1) {
    const int width = experts / p.groups;
    u64 mine = 0;  // lane g: the value of group g
    if (lane < p.groups) {
      u64 a = 0, b = 0;  // the two largest
      const int turn = lane % width;  // each lane begins at another bank
#pragma unroll 4
      for (int i = 0; i < width; ++i) {
        const int at = i + turn;
        const u64 o = key[lane * width + (at < width ? at : at - width)];
        b = max(b, min(a, o));
        a = max(a, o);
      }
      mine = p.best == 2 && b ? order_of(value_of(a) + value_of(b)) : a;
    }
    unsigned kept = 0;
    for (int n = 0; n < p.keep; ++n) {
      u64 k1 = mine;
      int g = lane;
      first_largest(&k1, &g);
      if (!k1) break;
      kept |= 1u << g;
      if (lane == g) mine = 0;
    }
    __syncwarp();
    for (int e = lane; e < experts; e += 32) {
      if (!(kept >> (e * p.magic >> 20 & 31) & 1)) key[e] = 0;
      else if (sums && key[e]) key[e] = order_of((double)widen(row[e]));
    }
  }
  int index = -1;
  for (int n = 0; n < p.k; ++n) {
    u64 best = 0;
    int at = kMaxExperts;
#pragma unroll 4
    for (int e = lane; e < experts; e += 32) {
      const u64 o = key[e];
      if (o > best) {
        best = o;
        at = e;
      }
    }
    first_largest(&best, &at);
    if (!best) break;
    if (lane == n) index = at;
    if (lane == (at & 31)) key[at] = 0;
  }
  float s = 0.f;
  if (index >= 0) {
    const float l = widen(row[index]);
    s = p.sigmoid ? 1.f / (1.f + expf(-l)) : expf(l - top) / (float)sum;
  }
  float w = s;
  if (p.renormalize) {
    float total = s;
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
    w = s / (total + kTiny);
  }
  if (lane < p.k) {
    p.indices[token * p.k + lane] = index;
    p.weights[token * p.k + lane] = index < 0 ? 0.f : w * p.scale;
  }
}

// The k + 1 largest words of a token, put in the order of their keys in 64 bits: for a
// choice between them that float32 does not decide.  All L lanes of each team of the warp
// call it; `near`: whether this team's words need it.
template <typename T, int L>
__device__ __noinline__ void sort_exact(const RouteParams& p, const T* row, bool near, unsigned* win, u64* key,
                                        unsigned low) {
  const int lane = threadIdx.x % L;
  float top = -INFINITY;
  double sum = 0.0;
  if (p.bias && !p.sigmoid) {
    for (int e = lane; e < p.experts; e += L) top = fmaxf(top, widen(row[e]));
#pragma unroll
    for (int d = L / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
#pragma unroll 1
    for (int base = lane; near && base < p.experts; base += 4 * L) {
      double v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = base + i * L < p.experts ? (double)widen(row[base + i * L]) : -INFINITY;
      exact_scores(v, 0, top, 0.0);  // -inf gives 0
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
#pragma unroll
    for (int d = L / 2; d; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
  }
#pragma unroll 1
  for (int base = lane; near && base <= p.k; base += 4 * L) {
    double v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = base + i * L;
      v[i] = j <= p.k && win[j] ? (double)widen(row[low - (win[j] & low)]) : 0.0;
    }
    if (p.bias) exact_scores(v, p.sigmoid, top, sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = base + i * L;
      if (j <= p.k) key[j] = !win[j] ? 0 : order_of(p.bias ? v[i] + (double)p.bias[low - (win[j] & low)] : v[i]);
    }
  }
  __syncwarp();
  unsigned mine[kMaxChoices / L + 1];
  int rank[kMaxChoices / L + 1];
#pragma unroll
  for (int q = 0; q <= kMaxChoices / L; ++q) {
    const int j = q * L + lane;
    rank[q] = -1;
    if (!near || j > p.k || !win[j]) continue;
    mine[q] = win[j];
    rank[q] = 0;
#pragma unroll 1
    for (int i = 0; i <= p.k; ++i)
      rank[q] += win[i] && (key[i] > key[j] || (key[i] == key[j] && (win[i] & low) > (win[j] & low)));
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q <= kMaxChoices / L; ++q)
    if (rank[q] >= 0) win[rank[q]] = mine[q];
  __syncwarp();
}

// exp(x) to about 2^-22 of its largest value in a row of differences to the maximum.  Weights that are not renormalised
// have it in the softmax's sum alone: off by 0.9 x 2^-24 in the mean of 600 experts, 0.8 with expf throughout.
__device__ __forceinline__ float quick_exp(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

__device__ __forceinline__ float larger(float a, float b) {  // a NaN stays one
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float quick_reciprocal(float x) {  // to one step
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// N values of a row for each of L lanes in float32, -inf behind the last.  VEC: V neighbours
// (16 bytes of the logits) at a time, lane l has the vectors l, l + L, ...; otherwise elements l, l + L, ...
template <typename T, int L, bool VEC>
__device__ __forceinline__ int expert_of(int i, int lane) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  return (i / V * L + lane) * V + i % V;
}
template <typename T, int L, int N, bool VEC, int V = 16 / (int)sizeof(T)>
__device__ __forceinline__ void load_logits(const T* row, bool live, int experts, int lane, float* x) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < N; i += V) {
      const int e = (i / V * L + lane) * V;
#pragma unroll
      for (int j = 0; j < V; j += Elem<T>::E) {
        if (live && e < experts) {
          Elem<T>::unpack(*reinterpret_cast<const uint4*>(row + e + j), x + i + j);
        } else {
#pragma unroll
          for (int n = 0; n < Elem<T>::E; ++n) x[i + j + n] = -INFINITY;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = i * L + lane;
      x[i] = live && e < experts ? widen(row[e]) : -INFINITY;
    }
  }
}

template <int L> __device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int d = L / 2; d; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}
template <int L> __device__ __forceinline__ float team_max(float v) {
#pragma unroll
  for (int d = L / 2; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, d));
  return v;
}
template <int L> __device__ __forceinline__ unsigned team_max(unsigned v) {
#pragma unroll
  for (int d = L / 2; d; d >>= 1) v = max(v, __shfl_xor_sync(kFull, v, d));
  return v;
}

constexpr int kRouteThreads = 128;

// Words of a team: its k + 2 winners, its groups' values, the keys of sort_exact.
constexpr int kWinWords = 36, kTeamWords = kWinWords + kMaxGroups + 2 * (kMaxChoices + 2);
static_assert(kWinWords >= kMaxChoices + 2 && kTeamWords % 4 == 0 && (kWinWords + kMaxGroups) % 2 == 0, "aligned parts");

// Shared memory of one warp: its teams' keys by group, or the keys of route_exact; then the words of its teams.
__host__ __device__ inline int route_values(int experts, int groups, int teams) {
  const int grouped = groups > 1 ? teams * (experts + groups) * 4 : 0;
  return (max(grouped, experts * 8) + 15) / 16 * 16;
}
__host__ __device__ inline int route_shared(int experts, int groups, int teams) {
  return route_values(experts, groups, teams) + teams * kTeamWords * 4;
}

// L lanes for a token, N experts for a lane; experts <= 1 << bits <= L * N.
//
// What bounds it is latency, not the bytes: k + 1 rounds, each a maximum over a lane's words and a chain of
// shuffles that waits for it (0.6 of the issue slots at 43 % of the warps).  65536 tokens of 128 float32
// logits take 21 us, of 256 with a bias 58, four to six times their bytes; blocks are held to 64 registers
// so that eight share an SM.
//
// A key in float32 and its expert's number are one 31-bit word: the key's order without its lowest bits,
// which hold the number, the lowest the largest.  So the words differ, one maximum finds value and place at
// once, and the next largest is the largest of word - last, wrapped around, without anything being marked.
// With a bias the upper bits are not the key's order but its distance from the row's largest
// in even steps, as fine as the scores are exact.  The choice stands if each of the k + 1
// first words is clear of the next: by what its upper bits leave open, and by the rounding of the
// scores where there is a bias.  Otherwise sort_exact orders those k + 1, and where more than
// they are too near the border, or a value is not finite, route_exact makes the whole choice.  16-bit
// logits without a bias lose nothing with the lowest bits and need none of this.
template <typename T, int L, int N, bool VEC>
__global__ void __launch_bounds__(kRouteThreads, N <= 16 ? 8 : 5) route_kernel(const __grid_constant__ RouteParams p) {
  constexpr int TEAMS = 32 / L;
  constexpr unsigned kWrap = 1u << 31;
  extern __shared__ __align__(16) char shared[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x % L, team = (threadIdx.x & 31) / L, experts = p.experts;
  char* mine = shared + warp * route_shared(experts, p.groups, TEAMS);
  unsigned* win = reinterpret_cast<unsigned*>(mine + route_values(experts, p.groups, TEAMS)) +
                  team * kTeamWords;
  float* group_value = reinterpret_cast<float*>(win + kWinWords);
  u64* exact_key = reinterpret_cast<u64*>(group_value + kMaxGroups);
  const long long token = ((long long)blockIdx.x * (kRouteThreads / 32) + warp) * TEAMS + team;
  const bool live = token < p.tokens && !(p.mask && !p.mask[token]);
  const T* row = reinterpret_cast<const T*>(p.logits) + (live ? token : 0) * p.stride;
  const unsigned low = (1u << p.bits) - 1;

  float x[N];
  load_logits<T, L, N, VEC>(row, live, experts, lane, x);
  float peak = x[0];  // a NaN stays one
#pragma unroll
  for (int i = 1; i < N; ++i) peak = larger(peak, x[i]);
  bool odd = !(peak < INFINITY);  // what float32 does not decide
  // Scores of all experts are needed with a bias, and their sum unless it cancels in the weights.
  const bool plain = !p.bias && p.groups == 1;
  float top = 0.f, inv = 1.f, largest_score = 1.f;
  if (!p.sigmoid && !(plain && p.renormalize)) {
    top = team_max<L>(peak);
    if (top == -INFINITY) top = 0.f;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i & 3] += quick_exp(x[i] - top);
    inv = largest_score = 1.f / team_sum<L>((sum[0] + sum[1]) + (sum[2] + sum[3]));
  }
  const auto score_of = [&](float l) { return p.sigmoid ? quick_reciprocal(1.f + quick_exp(-l)) : quick_exp(l - top) * inv; };
  // Twice what a score may be off by.  Softmax: 2^-22 of the largest for its exponential, 15 additions and a quotient at
  // 2^-24.  Sigmoid: its exponential's error weighs s (1 - s), 2^-24 with |l| at its worst; then half a step of the sum
  // and one of the reciprocal.
  const float slack = largest_score * (p.sigmoid ? 0x1p-20f : 0x1p-18f);
  if (p.bias) {  // from here on x is the key
    float b[N];
    load_logits<float, L, N, VEC, 16 / (int)sizeof(T)>(p.bias, live, experts, lane, b);
    peak = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (x[i] > -INFINITY) x[i] = score_of(x[i]) + b[i];
      peak = larger(peak, x[i]);
    }
    odd |= !(peak < INFINITY);
  }

  if (p.groups > 1) {
    // On either side of the border: the least that a kept group may be worth, and the most that another one may be.  A value
    // is off by what its keys are, each by half the slack and its rounding, and by its own rounding.  The keys' magnitudes
    // count, not the sum's: keys of +8 and -8 add up to nothing but their roundings.
    const bool rounded = p.bias || p.best == 2;  // logits alone are compared as they are
    float worst = INFINITY, next = -INFINITY;
    const auto error_of = [&](float a, float b) {
      return rounded ? slack + 0x1p-22f * (fabsf(a) + (p.best == 2 && b > -INFINITY ? fabsf(b) : 0.f)) : 0.f;
    };
    if (VEC && p.group_lanes) {
      // A group is p.group_lanes neighbouring lanes' vectors: its value is made and compared in registers.
      constexpr int V = 16 / (int)sizeof(T), C = VEC ? N / V : 1;
      float value[C], error[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float a = -INFINITY, b = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float l = x[c * V + i], v = p.bias || p.best == 1 || l == -INFINITY ? l : score_of(l);
          b = fmaxf(b, fminf(a, v));
          a = fmaxf(a, v);
        }
        for (int d = p.group_lanes / 2; d; d >>= 1) {
          const float oa = __shfl_xor_sync(kFull, a, d), ob = __shfl_xor_sync(kFull, b, d);
          b = fmaxf(fminf(a, oa), fmaxf(b, ob));
          a = fmaxf(a, oa);
        }
        value[c] = p.best == 2 && b > -INFINITY ? a + b : a;
        error[c] = error_of(a, b);
      }
      int rank[C];
#pragma unroll
      for (int c = 0; c < C; ++c) rank[c] = 0;
#pragma unroll
      for (int o = 0; o < C; ++o)
        for (int from = 0; from < L; from += p.group_lanes) {
          const float other = __shfl_sync(kFull, value[o], team * L + from);
#pragma unroll
          for (int c = 0; c < C; ++c)  // equal ones: the earlier
            rank[c] += other > value[c] || (other == value[c] && (o < c || (o == c && from + p.group_lanes <= lane)));
        }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const bool there = expert_of<T, L, VEC>(c * V, lane) < experts;
        if (rank[c] < p.keep) {
          if (there && value[c] > -INFINITY) worst = fminf(worst, value[c] - error[c]);
        } else {
          if (value[c] > -INFINITY) next = fmaxf(next, value[c] + error[c]);
#pragma unroll
          for (int i = 0; i < V; ++i) x[c * V + i] = -INFINITY;
        }
      }
    } else {
      const int width = experts / p.groups;
      float* values = reinterpret_cast<float*>(mine) + team * (experts + p.groups);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = expert_of<T, L, VEC>(i, lane);
        if (e >= experts) continue;
        const float v = p.bias || p.best == 1 || x[i] == -INFINITY ? x[i] : score_of(x[i]);
        values[e + (e * p.magic >> 20)] = v;  // a word between the groups keeps them in different banks
      }
      __syncwarp();
      float error[kMaxGroups / L];  // of the groups lane, lane + L, ...
#pragma unroll
      for (int n = 0; n < kMaxGroups / L; ++n) {
        const int g = n * L + lane;
        if (g >= p.groups) break;
        float a = -INFINITY, b = -INFINITY;
#pragma unroll 8
        for (int i = 0; i < width; ++i) {
          const float v = values[g * (width + 1) + i];
          b = fmaxf(b, fminf(a, v));
          a = fmaxf(a, v);
        }
        group_value[g] = p.best == 2 && b > -INFINITY ? a + b : a;
        error[n] = error_of(a, b);
      }
      __syncwarp();
      unsigned kept = 0;
#pragma unroll
      for (int n = 0; n < kMaxGroups / L; ++n) {
        const int g = n * L + lane;
        if (g >= p.groups) break;
        const float v = group_value[g];
        int rank = 0;
        for (int o = 0; o < p.groups; ++o) rank += group_value[o] > v || (group_value[o] == v && o < g);
        if (rank < p.keep) {
          kept |= 1u << g;
          if (v > -INFINITY) worst = fminf(worst, v - error[n]);
        } else if (v > -INFINITY) {
          next = fmaxf(next, v + error[n]);
        }
      }
#pragma unroll
      for (int d = L / 2; d; d >>= 1) kept |= __shfl_xor_sync(kFull, kept, d);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!(kept >> (expert_of<T, L, VEC>(i, lane) * p.magic >> 20 & 31) & 1)) x[i] = -INFINITY;
    }
    worst = -team_max<L>(-worst);
    next = team_max<L>(next);
    if (rounded && p.keep < p.groups && next > -INFINITY) odd |= !(worst > next);
  }

  // Words: the upper bits of the key's order, or of its place between the largest and the smallest key.
  // need: how many steps apart two words have to be; least_word: words below it stand for -inf, which comes before the
  // order of the lowest number.
  unsigned word[N], need = 1, least_word = 1u << 22;
  if (!p.bias) {
#pragma unroll
    for (int i = 0; i < N; ++i) word[i] = (order_of(x[i]) >> 1 & ~low) + (low - expert_of<T, L, VEC>(i, lane));
  } else {
    least_word = 1;
    float most = -INFINITY, least = INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      most = fmaxf(most, x[i]);
      least = fminf(least, x[i] > -INFINITY ? x[i] : INFINITY);
    }
    most = team_max<L>(most);
    least = -team_max<L>(-least);
    const float steps = (float)((1 << min(23, 30 - p.bits)) - 1);
    const float range = fminf(most - least, 64.f * largest_score), base = most - range;  // far below: one step holds them all
    const float scale = range > 0.f ? steps / range : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = expert_of<T, L, VEC>(i, lane);
      // 2^23 + step as a float32 has the step in its lowest bits: no conversion.
      const float step = fminf(fmaxf(fmaf(x[i] - base, scale, 0x1p23f), 0x1p23f), 0x1p23f + steps);
      word[i] = x[i] > -INFINITY ? (__float_as_uint(step) - 0x4affffffu) << p.bits | (low - e) : 0;
    }
    // The place's own rounding is below two steps for each of two words; keys are off by half the slack and their rounding.
    // In a row whose keys differ by less than that no two words are far enough apart, at any number of steps.
    need = 5 + (unsigned)fminf((slack + 0x1p-22f * fmaxf(fabsf(most), fabsf(base))) * scale, 0x1p30f);
  }
  unsigned last = kWrap;
  const auto next_word = [&](int j) {
    unsigned best = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) best = __viaddmax_u32(word[i], -last, best);
    best = best >= kWrap ? best + last : 0;
    last = team_max<L>(best);
    if (lane == j % L) win[j] = last < least_word ? 0 : last;
    if (last == 0) last = 1;  // nothing is left: only zeros stay below
  };
  const bool certain = sizeof(T) == 2 && !p.bias;
  const int wanted = p.k + (certain ? 0 : 1);
  for (int j = 0; j < wanted; ++j) next_word(j);
  __syncwarp();
  if (!certain) {
    bool near = false;
    for (int j = lane; j < p.k; j += L) {
      const unsigned a = win[j], b = win[j + 1];
      if (!b || (a >> p.bits) - (b >> p.bits) >= need) continue;
      // Two experts with the same logit and bias are in order; at the border there may be more of them.
      const int e = low - (a & low), f = low - (b & low);
      near |= j + 1 == p.k || widen(row[e]) != widen(row[f]) || (p.bias && p.bias[e] != p.bias[f]);
    }
    const unsigned team_lanes = L == 32 ? ~0u : ((1u << (L & 31)) - 1) << (team * L);
    const unsigned all = __ballot_sync(kFull, near && live);
    if (all) {
      next_word(p.k + 1);  // those that are left over stay below this one
      __syncwarp();
      near = all & team_lanes;
      if (near && win[p.k + 1]) odd |= (win[p.k - 1] >> p.bits) - (win[p.k + 1] >> p.bits) < need;
      sort_exact<T, L>(p, row, near, win, exact_key, low);
    }
  }

  // Choice j belongs to lane j % L.
  float score[kMaxChoices / L];
  int index[kMaxChoices / L];
  const float first = plain && p.renormalize && !p.sigmoid && win[0] ? widen(row[low - (win[0] & low)]) : top;
  float total = 0.f;
#pragma unroll
  for (int q = 0; q < kMaxChoices / L; ++q) {
    const int j = q * L + lane;
    index[q] = -1;
    score[q] = 0.f;
    if (q * L >= p.k) break;
    if (j >= p.k || !win[j]) continue;
    index[q] = low - (win[j] & low);
    const float l = widen(row[index[q]]);
    score[q] = p.sigmoid ? 1.f / (1.f + expf(-l)) : expf(l - first) * inv;
    total += score[q];
  }
  total = p.renormalize ? team_sum<L>(total) + kTiny : 1.f;
  const unsigned again = __ballot_sync(kFull, odd && live);
  const unsigned ours = L == 32 ? ~0u : ((1u << (L & 31)) - 1) << (team * L);
  if (token < p.tokens && !(again & ours)) {
#pragma unroll
    for (int q = 0; q < kMaxChoices / L; ++q) {
      const int j = q * L + lane;
      if (j >= p.k) break;
      p.indices[token * p.k + j] = index[q];
      p.weights[token * p.k + j] = index[q] < 0 ? 0.f : (p.renormalize ? score[q] / total : score[q]) * p.scale;
    }
  }
  __syncwarp();
#pragma unroll 1
  for (int t = 0; t < TEAMS; ++t)
    if (again & (L == 32 ? ~0u : ((1u << (L & 31)) - 1) << (t * L)))
      route_exact<T>(p, token - team + t, reinterpret_cast<u64*>(mine));
}

struct RouteGradParams {
  const float* grad_weights;
  const char* logits;
  const int* indices;
  char* grad;
  long long tokens, stride;
  int experts, k, sigmoid, renormalize;
  float scale;
};

// The gradient of the scores is zero but for the k choices: those are put into a row of
// shared memory, and each lane picks up its own experts'.  The softmax's exponentials are expf's for float32: those of
// the unit alone are off by more the smaller the score is (4e-6 of one 80 below the row's largest), far less than the
// rounding of a 16-bit gradient.  65536 tokens of 128 logits: 17.9 us in float32 (15.1 by the unit), 14.6 in bfloat16.
template <typename T, int L, int N, bool VEC>
__global__ void __launch_bounds__(kRouteThreads) route_grad_kernel(const __grid_constant__ RouteGradParams p) {
  constexpr int Q = kMaxChoices / L, V = VEC ? 16 / (int)sizeof(T) : 1;
  __shared__ __align__(16) float direct[kRouteThreads / L][N * L];
  __shared__ int chosen[kRouteThreads / L][kMaxChoices];
  __shared__ float slope[kRouteThreads / L][kMaxChoices];
  const int lane = threadIdx.x % L, team = threadIdx.x / L, experts = p.experts;
  const long long token = (long long)blockIdx.x * (kRouteThreads / L) + team;
  const bool live = token < p.tokens;
  const T* row = reinterpret_cast<const T*>(p.logits) + (live ? token : 0) * p.stride;
  float x[N];
  load_logits<T, L, N, VEC>(row, live, experts, lane, x);
  int index[Q];
  float ds[Q], logit[Q];
  bool any = false;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int j = q * L + lane;
    index[q] = live && j < p.k ? p.indices[token * p.k + j] : -1;
    if (index[q] < 0 || index[q] >= experts) index[q] = -1;
    any |= index[q] >= 0;
    ds[q] = index[q] < 0 ? 0.f : p.scale * p.grad_weights[token * p.k + j];
    logit[q] = index[q] < 0 ? -INFINITY : widen(row[index[q]]);
  }
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(&direct[team][i * L + lane * 4]) = make_float4(0, 0, 0, 0);
  float top = 0.f, inv = 1.f;
  if (!p.sigmoid) {
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, x[i]);
    top = team_max<L>(top);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float below = x[i] - top;
      x[i] = x[i] == -INFINITY ? 0.f : sizeof(T) == 4 ? expf(below) : quick_exp(below);  // a NaN stays one
      sum[i & 3] += x[i];
    }
    const float all = team_sum<L>((sum[0] + sum[1]) + (sum[2] + sum[3]));
    inv = all == 0.f ? 0.f : 1.f / all;
  }
  // Renormalised weights do not change with a common factor of the scores, so their gradient only sees how the k weights'
  // gradients differ: they are taken from the first one, and what the sum's small addend lets through is added apart.
  // Without this one choice (whose weight is constant) would get the rounding of its own gradient.
  const float common = p.renormalize ? __shfl_sync(kFull, ds[0], (threadIdx.x & 31) / L * L) : 0.f;
  float mine[Q], total = 0.f, dot = 0.f;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    mine[q] = logit[q] == -INFINITY ? 0.f : p.sigmoid ? 1.f / (1.f + expf(-logit[q])) : expf(logit[q] - top) * inv;
    if (index[q] >= 0) ds[q] -= common;
    total += mine[q];
    dot += ds[q] * mine[q];
  }
  if (p.renormalize) {
    total = team_sum<L>(total) + kTiny;
    const float along = team_sum<L>(dot) / total, through = common * (kTiny / total);
    dot = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      ds[q] = index[q] < 0 ? 0.f : (ds[q] - along + through) / total;
      dot += ds[q] * mine[q];
    }
  }
  dot = p.sigmoid ? 0.f : team_sum<L>(dot);
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int j = q * L + lane;
    if (j < p.k) {
      chosen[team][j] = index[q];
      slope[team][j] = ds[q];
    }
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if (index[q] < 0) continue;
    float all = 0.f;  // an expert that stands twice counts twice, in the order of the choices
    for (int j = 0; j < p.k; ++j)
      if (chosen[team][j] == index[q]) all += slope[team][j];
    if (p.sigmoid) {  // s (1 - s) without the cancellation near 1
      const float t = expf(-fabsf(logit[q])), u = 1.f / (1.f + t);
      all *= t * u * u;
    }
    direct[team][index[q]] = all;
  }
  __syncwarp();
  const unsigned ballot = __ballot_sync(kFull, any);
  const bool empty = !(ballot & (L == 32 ? ~0u : ((1u << (L & 31)) - 1) << ((threadIdx.x & 31) / L * L)));
  if (!live) return;
  T* grad = reinterpret_cast<T*>(p.grad) + token * experts;
#pragma unroll
  for (int i = 0; i < N; i += V) {
    const int e = expert_of<T, L, VEC>(i, lane);
    if (e >= experts) break;
    float g[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = direct[team][e + j];
      g[j] = !p.sigmoid ? x[i + j] * inv * (d - dot) : isnan(x[i + j]) ? x[i + j] : d;
      if (empty) g[j] = 0.f;  // a padded token: whatever its logits hold, no gradient
    }
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(grad + e) = Elem<T>::pack(g);
    } else {
      grad[e] = T(g[0]);
    }
  }
}

// ---- plan ----------------------------------------------------------------------------------

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kSMs = 148;
constexpr int kPlanBlocks = kSMs;
// Slots that one block counts before another joins.  65536 slots of 64 experts took 8.5 us with 2048, 9.4 with 1024 and 9.8
// with 4096; 7.1 since the two kernels overlap.
constexpr int kSlotsOfBlock = 2048;

int plan_blocks(int64_t slots) {
  const int64_t n = ceil_div(slots, kSlotsOfBlock);
  return (int)(n < 1 ? 1 : n < kPlanBlocks ? n : kPlanBlocks);
}

struct PlanParams {
  const int* indices;
  int* counts;
  int* offsets;
  int* ends;
  int* positions;
  int* parts;  // [gridDim.x][experts]: how often each block's slots ask for each expert
  long long slots, span;  // span: slots of a block, a multiple of 32
  int experts, align;
};

__global__ void __launch_bounds__(kPlanThreads) plan_count_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int hist[];
  allow_next();
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const long long first = blockIdx.x * p.span, last = min(first + p.span, p.slots);
  for (long long s = first + threadIdx.x; s < last; s += blockDim.x) {
    const int e = p.indices[s];
    if (e >= 0 && e < p.experts) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) p.parts[(long long)blockIdx.x * p.experts + e] = hist[e];
}

// Every block adds up the counts of the blocks before it, then ranks its own slots: warp w takes the w-th run of them.
__global__ void __launch_bounds__(kPlanThreads) plan_place_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int hist[];  // [kPlanWarps][experts], then the place of each warp's next slot of an expert; [2][experts]
  __shared__ int carry[kPlanWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, experts = p.experts;
  for (int i = threadIdx.x; i < (kPlanWarps + 2) * experts; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  const long long first = blockIdx.x * p.span, last = min(first + p.span, p.slots);
  const long long run = (p.span / 32 + kPlanWarps - 1) / kPlanWarps * 32;
  const long long begin = min(first + warp * run, last), end = min(begin + run, last);
  for (long long s = begin + lane; s < end; s += 32) {
    const int e = p.indices[s];
    if (e >= 0 && e < experts) atomicAdd(&hist[warp * experts + e], 1);
  }
  if (gridDim.x > 1) {
    await_previous();  // the slots have been counted meanwhile
    int* sums = hist + kPlanWarps * experts;  // [2][experts]: of all blocks, and of those before this one
    for (int b = warp; b < (int)gridDim.x; b += kPlanWarps)
      for (int e = lane; e < experts; e += 32) {
        const int n = p.parts[(long long)b * experts + e];
        if (!n) continue;
        atomicAdd(&sums[e], n);
        if (b < (int)blockIdx.x) atomicAdd(&sums[experts + e], n);
      }
  }
  __syncthreads();
  // Block starts: a scan of the aligned totals over the experts, two experts for a thread.
  int total[2] = {0, 0}, before[2] = {0, 0}, blocks[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = threadIdx.x * 2 + i;
    if (e < experts) {
      if (gridDim.x == 1) {
        for (int w = 0; w < kPlanWarps; ++w) total[i] += hist[w * experts + e];
      } else {
        total[i] = hist[kPlanWarps * experts + e];
        before[i] = hist[(kPlanWarps + 1) * experts + e];
      }
    }
    blocks[i] = (total[i] + p.align - 1) / p.align * p.align;
  }
  int sum = blocks[0] + blocks[1], scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(kFull, scan, d);
    if (lane >= d) scan += v;
  }
  if (lane == 31) carry[warp] = scan;
  __syncthreads();
  int start = scan - sum;
  for (int w = 0; w < warp; ++w) start += carry[w];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = threadIdx.x * 2 + i;
    if (e < experts) {
      if (blockIdx.x == 0) {
        p.counts[e] = total[i];
        p.offsets[e] = start;
        p.ends[e] = start + total[i];
        if (e == experts - 1) p.offsets[experts] = start + blocks[i];
      }
      int next = start + before[i];
      for (int w = 0; w < kPlanWarps; ++w) {
        const int n = hist[w * experts + e];
        hist[w * experts + e] = next;
        next += n;
      }
      start += blocks[i];
    }
  }
  __syncthreads();
  int* next = hist + warp * experts;
  for (long long s = begin; s < end; s += 32) {
    const int e = s + lane < end ? p.indices[s + lane] : -1;
    const bool there = e >= 0 && e < experts;
    const unsigned same = __match_any_sync(kFull, there ? e : -1);
    const int rank = __popc(same & ((1u << lane) - 1));
    const int base = there ? next[e] : 0;
    __syncwarp();
    if (there && rank == 0) next[e] = base + __popc(same);
    __syncwarp();
    if (s + lane < end) p.positions[s + lane] = there ? base + rank : -1;
  }
}

// ---- moves -----------------------------------------------------------------------------------

constexpr int kMoveThreads = 256;

struct MoveParams {
  const char* x;
  const int* positions;
  const int* offsets;
  const int* ends;
  char* out;
  long long tokens, x_stride, row_bytes, capacity;  // bytes
  int k, experts, share;  // share: blocks for the unused rows of an expert
};

// Zeros in the rows of an expert's block that no slot uses, by `share` blocks of threads.
// They lie in one piece, so they are written by 16 bytes whatever the row.  Such blocks come first in
// the grid: behind the others they would be its tail.
__device__ void clear_rows(char* out, const int* offsets, const int* ends, int block, int share, long long row_bytes,
                           long long capacity) {
  const int e = block / share;
  const long long first = max(0, ends[e]), last = min((long long)offsets[e + 1], capacity);
  if (first >= last) return;
  char* begin = out + first * row_bytes;
  const long long bytes = (last - first) * row_bytes;
  const long long head = min((long long)(-reinterpret_cast<uintptr_t>(begin) & 15), bytes), n = (bytes - head) / 16;
  uint4* body = reinterpret_cast<uint4*>(begin + head);
#pragma unroll 4
  for (long long i = (long long)(block % share) * kMoveThreads + threadIdx.x; i < n; i += (long long)share * kMoveThreads)
    body[i] = make_uint4(0, 0, 0, 0);
  if (block % share) return;
  if (threadIdx.x < head) begin[threadIdx.x] = 0;
  if (threadIdx.x < bytes - head - n * 16) begin[head + n * 16 + threadIdx.x] = 0;
}

// Bytes q .. q + 15 of the 32 bytes {lo, hi}; 0 < q < 16.
__device__ __forceinline__ uint4 shift16(uint4 lo, uint4 hi, unsigned q) {
  unsigned w0 = lo.x, w1 = lo.y, w2 = lo.z, w3 = lo.w, w4 = hi.x, w5 = hi.y, w6 = hi.z;
  if (q & 8) { w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = hi.w; }
  if (q & 4) { w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5; }
  const unsigned bits = (q & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}

// Copies a row between any two addresses by TEAM threads: the aligned vectors of the target are made of the two aligned
// vectors of the source around them (each holds a byte of the row: nothing else is mapped in), its ends byte by byte.
template <int TEAM>
__device__ __forceinline__ void copy_row(char* to, const char* from, int bytes, int me) {
  const int head = min((int)(-reinterpret_cast<uintptr_t>(to) & 15), bytes), n = (bytes - head) / 16;
  for (int i = me; i < head; i += TEAM) to[i] = from[i];
  for (int i = head + n * 16 + me; i < bytes; i += TEAM) to[i] = from[i];
  const unsigned q = (unsigned)(reinterpret_cast<uintptr_t>(from + head) & 15);
  const uint4* source = reinterpret_cast<const uint4*>(from + head - q);
  uint4* target = reinterpret_cast<uint4*>(to + head);
#pragma unroll 2
  for (int i = me; i < n; i += TEAM) target[i] = q ? shift16(source[i], source[i + 1], q) : source[i];
}

// TEAM threads for a token: four words of its row at a time are read once and written to
// each of its k places.  Rows that no word of 4 bytes divides (U a byte) are copied to each place by themselves.
template <typename U, int TEAM>
__global__ void __launch_bounds__(kMoveThreads) dispatch_kernel(const __grid_constant__ MoveParams p) {
  if (blockIdx.x < p.experts * p.share) {
    clear_rows(p.out, p.offsets, p.ends, blockIdx.x, p.share, p.row_bytes, p.capacity);
    return;
  }
  __shared__ int place[kMoveThreads / TEAM][kMaxChoices];
  const int team = threadIdx.x / TEAM, me = threadIdx.x % TEAM;
  const long long t = (long long)(blockIdx.x - p.experts * p.share) * (kMoveThreads / TEAM) + team;
  if (t < p.tokens)
    for (int j = me; j < p.k; j += TEAM) place[team][j] = p.positions[t * p.k + j];
  if (TEAM > 32) __syncthreads();
  else __syncwarp();
  if (t >= p.tokens) return;
  if constexpr (sizeof(U) == 1) {
    for (int j = 0; j < p.k; ++j) {
      const int at = place[team][j];
      if (at >= 0 && at < p.capacity) copy_row<TEAM>(p.out + at * p.row_bytes, p.x + t * p.x_stride, (int)p.row_bytes, me);
    }
    return;
  }
  const U* from = reinterpret_cast<const U*>(p.x + t * p.x_stride);
  const long long n = p.row_bytes / (long long)sizeof(U);
  for (long long base = me; base < n; base += 4 * TEAM) {
    U v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (base + i * TEAM < n) v[i] = from[base + i * TEAM];
    for (int j = 0; j < p.k; ++j) {
      const int at = place[team][j];
      if (at < 0 || at >= p.capacity) continue;
      U* to = reinterpret_cast<U*>(p.out + at * p.row_bytes);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (base + i * TEAM < n) to[base + i * TEAM] = v[i];
    }
  }
}

// Part i (E elements, 16 bytes) of a row for thread `me` of TEAM: words of W neighbouring
// elements, TEAM words apart, so that neighbouring threads read neighbouring words.  W = E: rows
// aligned to 16 bytes; W = 2 (16-bit types) and W = 1: other rows.
template <int BYTES> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<16> { typedef uint4 type; };

template <typename T, int W, int TEAM>
__device__ __forceinline__ uint4 part(const char* row, int i, int me, int cols) {
  constexpr int Q = Elem<T>::E / W;
  typedef typename Word<W * sizeof(T)>::type U;
  uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int c = ((i * Q + q) * TEAM + me) * W;
    if (c < cols) reinterpret_cast<U*>(&v)[q] = *reinterpret_cast<const U*>(row + (size_t)c * sizeof(T));
  }
  return v;
}
template <typename T, int W, int TEAM>
__device__ __forceinline__ void put(char* row, int i, int me, int cols, uint4 v) {
  constexpr int Q = Elem<T>::E / W;
  typedef typename Word<W * sizeof(T)>::type U;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int c = ((i * Q + q) * TEAM + me) * W;
    if (c < cols) *reinterpret_cast<U*>(row + (size_t)c * sizeof(T)) = reinterpret_cast<const U*>(&v)[q];
  }
}

// The same for 16-bit rows that words of two do not divide, whose threads still take E neighbouring elements: the two
// aligned vectors around them, shifted together (each holds an element of the row).
template <typename T, int TEAM>
__device__ __forceinline__ uint4 part_between(const char* row, int i, int me, int cols) {
  constexpr int E = Elem<T>::E;
  const int c = (i * TEAM + me) * E, left = cols - c;
  if (left <= 0) return make_uint4(0, 0, 0, 0);
  const char* p = row + (size_t)c * sizeof(T);
  const unsigned q = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15);
  const uint4* from = reinterpret_cast<const uint4*>(p - q);
  uint4 v = from[0];
  const int here = (16 - (int)q) / (int)sizeof(T);  // elements in the first vector; compared as such, bytes may pass 31 bits
  if (q) v = shift16(v, left > here ? from[1] : make_uint4(0, 0, 0, 0), q);
  return v;  // elements behind the last are the caller's to leave out
}
// Its counterpart, by whole warps: what a lane holds behind an aligned vector of the target goes to the next lane, so that
// aligned vectors are written; only the ends of a warp's piece and of the row go by elements.
template <typename T, int TEAM>
__device__ __forceinline__ void put_between(char* row, int i, int me, int cols, uint4 v) {
  constexpr int E = Elem<T>::E;
  typedef unsigned short U;
  const int c = (i * TEAM + me) * E, left = cols - c, valid = min(left, E), lane = threadIdx.x & 31;
  char* p = row + (size_t)c * sizeof(T);
  const unsigned q = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15);  // the same for all of a row
  const uint4 before = make_uint4(__shfl_up_sync(kFull, v.x, 1), __shfl_up_sync(kFull, v.y, 1),
                                  __shfl_up_sync(kFull, v.z, 1), __shfl_up_sync(kFull, v.w, 1));
  if (left <= 0) return;
  const int mine = (16 - (int)q) / (int)sizeof(T);  // elements in the aligned vector that p lies in
  if (valid >= mine && (lane > 0 || q == 0)) {
    *reinterpret_cast<uint4*>(p - q) = q ? shift16(before, v, 16 - q) : v;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (e >= mine && lane > 0) reinterpret_cast<U*>(p - 16)[e] = reinterpret_cast<const U*>(&before)[e];
      if (e < min(mine, valid)) reinterpret_cast<U*>(p)[e] = reinterpret_cast<const U*>(&v)[e];
    }
  }
  if (lane == 31 || left <= E) {  // nobody takes the rest
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e >= mine && e < valid) reinterpret_cast<U*>(p)[e] = reinterpret_cast<const U*>(&v)[e];
  }
}

struct CombineParams {
  const char* rows;
  const int* positions;
  const float* weights;
  const char* residual;
  char* out;
  long long tokens, capacity, residual_stride;
  int cols, k;
};

// TEAM threads for a token; TWO parts of four of its rows are on their way at a time, and four blocks share an SM:
// 55.5 us for 8192x2048 bfloat16 with 8 choices, 59.9 with the registers that the compiler would take, 56.6 with one part.
template <typename T, int W, int TEAM, int TWO>
__global__ void __launch_bounds__(kMoveThreads, 4) combine_kernel(const __grid_constant__ CombineParams p) {
  constexpr int E = Elem<T>::E, AHEAD = 4;
  __shared__ int place[kMoveThreads / TEAM][kMaxChoices];
  __shared__ float weight[kMoveThreads / TEAM][kMaxChoices];
  const int team = threadIdx.x / TEAM, me = threadIdx.x % TEAM;
  const long long t = (long long)blockIdx.x * (kMoveThreads / TEAM) + team, row_bytes = p.cols * (long long)sizeof(T);
  if (t < p.tokens && me < p.k) {
    const int at = p.positions[t * p.k + me];
    place[team][me] = at < p.capacity ? at : -1;
    weight[team][me] = p.weights ? p.weights[t * p.k + me] : 1.f;
  }
  if (TEAM > 32) __syncthreads();
  else __syncwarp();
  if (t >= p.tokens) return;
  const auto take = [&](const char* row, int i, int thread, int cols) {
    if constexpr (W == 1 && sizeof(T) == 2) return part_between<T, TEAM>(row, i, thread, cols);
    else return part<T, W, TEAM>(row, i, thread, cols);
  };
  const auto give = [&](char* row, int i, int thread, int cols, uint4 v) {
    if constexpr (W == 1 && sizeof(T) == 2) put_between<T, TEAM>(row, i, thread, cols, v);
    else put<T, W, TEAM>(row, i, thread, cols, v);
  };
  const int parts = (p.cols + TEAM * E - 1) / (TEAM * E);
  for (int i = 0; i < parts; i += TWO) {
    float sum[TWO][E], a[E];
    uint4 r[TWO];
#pragma unroll
    for (int u = 0; u < TWO; ++u) {
#pragma unroll
      for (int e = 0; e < E; ++e) sum[u][e] = 0.f;
      if (p.residual) r[u] = take(p.residual + t * p.residual_stride * (long long)sizeof(T), i + u, me, p.cols);
    }
    for (int j = 0; j < p.k; j += AHEAD) {
      uint4 v[AHEAD][TWO];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
        if (j + n < p.k && place[team][j + n] >= 0) {
#pragma unroll
          for (int u = 0; u < TWO; ++u)
            v[n][u] = take(p.rows + place[team][j + n] * row_bytes, i + u, me, p.cols);
        }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n)
        if (j + n < p.k && place[team][j + n] >= 0) {
          const float w = weight[team][j + n];
#pragma unroll
          for (int u = 0; u < TWO; ++u) {
            Elem<T>::unpack(v[n][u], a);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[u][e] = fmaf(w, a[e], sum[u][e]);
          }
        }
    }
#pragma unroll
    for (int u = 0; u < TWO; ++u) {
      if (p.residual) {
        Elem<T>::unpack(r[u], a);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[u][e] += a[e];
      }
      give(p.out + t * row_bytes, i + u, me, p.cols, Elem<T>::pack(sum[u]));
    }
  }
}

struct CombineGradParams {
  const char* grad_out;
  const char* rows;
  const int* positions;
  const float* weights;
  const int* offsets;
  const int* ends;
  char* grad_rows;
  float* grad_weights;
  long long slots, capacity, grad_out_stride;
  int cols, k, experts, share;
};

// A warp for a slot: no warp waits for another.  The slots of a token are neighbours, so its
// row of grad_out comes from memory once and then from the first cache.
template <typename T, int W>
__global__ void __launch_bounds__(kMoveThreads) combine_grad_kernel(const __grid_constant__ CombineGradParams p) {
  constexpr int E = Elem<T>::E, AHEAD = 4;
  const long long row_bytes = p.cols * (long long)sizeof(T);
  if (blockIdx.x < p.experts * p.share) {
    clear_rows(p.grad_rows, p.offsets, p.ends, blockIdx.x, p.share, row_bytes, p.capacity);
    return;
  }
  const long long slot = (long long)(blockIdx.x - p.experts * p.share) * (kMoveThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (slot >= p.slots) return;
  const long long at = p.positions[slot];
  float dot = 0.f;
  if (at >= 0 && at < p.capacity) {
    const float w = p.weights[slot];
    const char* grad = p.grad_out + slot / p.k * p.grad_out_stride * (long long)sizeof(T);
    const char* row = p.rows + at * row_bytes;
    char* to = p.grad_rows + at * row_bytes;
    const int parts = (p.cols + 32 * E - 1) / (32 * E);
    constexpr bool BETWEEN = W == 1 && sizeof(T) == 2;
    for (int i = 0; i < parts; i += AHEAD) {
      uint4 g[AHEAD], y[AHEAD];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {  // parts behind the last hold zeros and are not written
        if constexpr (BETWEEN) {
          y[n] = part_between<T, 32>(row, i + n, lane, p.cols);
          g[n] = part_between<T, 32>(grad, i + n, lane, p.cols);
        } else {
          y[n] = part<T, W, 32>(row, i + n, lane, p.cols);
          g[n] = part<T, W, 32>(grad, i + n, lane, p.cols);
        }
      }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        float a[E], b[E];
        Elem<T>::unpack(g[n], a);
        Elem<T>::unpack(y[n], b);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (!BETWEEN || ((i + n) * 32 + lane) * E + e < p.cols) dot = fmaf(a[e], b[e], dot);
          a[e] *= w;
        }
        if constexpr (BETWEEN) put_between<T, 32>(to, i + n, lane, p.cols, Elem<T>::pack(a));
        else put<T, W, 32>(to, i + n, lane, p.cols, Elem<T>::pack(a));
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(kFull, dot, d);
  if (lane == 0) p.grad_weights[slot] = dot;
}

__global__ void __launch_bounds__(1024) update_bias_kernel(const float* bias, const int* counts, float* out, int experts,
                                                           float rate) {
  __shared__ long long slot[32];
  const int e = threadIdx.x, lane = e & 31;
  const long long mine = e < experts ? counts[e] : 0;
  long long total = mine;
#pragma unroll
  for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
  if (lane == 0) slot[e >> 5] = total;
  __syncthreads();
  total = slot[lane];
#pragma unroll
  for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(kFull, total, d);
  if (e >= experts) return;
  const long long lack = total - (long long)experts * mine;
  out[e] = bias[e] + (lack > 0 ? rate : lack < 0 ? -rate : 0.f);
}

// ---- kernel choice -----------------------------------------------------------------------------

// Lanes for a token: eight where 16 experts a lane suffice, so that a warp works on four tokens at once, and more as
// the experts become more.
int route_lanes(int experts) { return experts <= 128 ? 8 : experts <= 256 ? 16 : 32; }

template <typename T, bool VEC>
const void* route_fn(int experts) {
  if (experts <= 64) return (const void*)route_kernel<T, 8, 8, VEC>;
  if (experts <= 128) return (const void*)route_kernel<T, 8, 16, VEC>;
  if (experts <= 256) return (const void*)route_kernel<T, 16, 16, VEC>;
  if (experts <= 512) return (const void*)route_kernel<T, 32, 16, VEC>;
  return (const void*)route_kernel<T, 32, 32, VEC>;
}
template <typename T, bool VEC>
const void* route_grad_fn(int experts) {
  if (experts <= 64) return (const void*)route_grad_kernel<T, 8, 8, VEC>;
  if (experts <= 128) return (const void*)route_grad_kernel<T, 8, 16, VEC>;
  if (experts <= 256) return (const void*)route_grad_kernel<T, 16, 16, VEC>;
  if (experts <= 512) return (const void*)route_grad_kernel<T, 32, 16, VEC>;
  return (const void*)route_grad_kernel<T, 32, 32, VEC>;
}
// Blocks that clear the unused rows of one expert: one for each 128 KB that the rows beyond the slots may take for it.
int clear_share(int64_t slots, int experts, int64_t capacity, int64_t row_bytes) {
  const int64_t spare = capacity > slots ? (capacity - slots) * row_bytes : 0, each = slots < experts ? slots : experts;
  const int64_t share = ceil_div(spare, each * (128 << 10));
  return (int)(share < 1 ? 1 : share > 16 ? 16 : share);
}

// Threads for a token's row of `words` words, of which each thread takes about four (one where rows are narrow); more
// threads while the tokens do not fill two blocks on each SM.
int move_team(int64_t words, int64_t tokens) {
  const int sizes[] = {8, 32, 128, 256};
  int i = words <= 16 ? 0 : words <= 128 ? 1 : words <= 512 ? 2 : 3;
  while (i < 3 && words > sizes[i] && tokens * sizes[i] < 2 * kMoveThreads * kSMs) ++i;
  return sizes[i];
}

// The same for a sum of rows, of which each thread takes two parts (one where a warp would be half idle).
struct CombineTeam {
  int threads, parts;
};
CombineTeam combine_team(int64_t parts) {
  return {parts <= 64 ? 32 : parts <= 128 ? 64 : parts <= 256 ? 128 : 256, parts <= 32 ? 1 : 2};
}

template <typename U>
const void* dispatch_fn(int team) {
  return team == 8     ? (const void*)dispatch_kernel<U, 8>
         : team == 32  ? (const void*)dispatch_kernel<U, 32>
         : team == 128 ? (const void*)dispatch_kernel<U, 128>
                       : (const void*)dispatch_kernel<U, 256>;
}
template <typename T, int W>
const void* combine_fn(const CombineTeam& c) {
  constexpr int TWO = W == Elem<T>::E ? 2 : 1;
  return c.parts == 1       ? (const void*)combine_kernel<T, W, 32, 1>
         : c.threads == 32  ? (const void*)combine_kernel<T, W, 32, TWO>
         : c.threads == 64  ? (const void*)combine_kernel<T, W, 64, TWO>
         : c.threads == 128 ? (const void*)combine_kernel<T, W, 128, TWO>
                            : (const void*)combine_kernel<T, W, 256, TWO>;
}
template <typename T>
const void* combine_fn(int word, const CombineTeam& team) {
  if (word == Elem<T>::E) return combine_fn<T, Elem<T>::E>(team);
  if constexpr (sizeof(T) == 2)
    if (word == 2) return combine_fn<T, 2>(team);
  return combine_fn<T, 1>(team);
}
template <typename T>
const void* combine_grad_fn(int word) {
  if (word == Elem<T>::E) return (const void*)combine_grad_kernel<T, Elem<T>::E>;
  if constexpr (sizeof(T) == 2)
    if (word == 2) return (const void*)combine_grad_kernel<T, 2>;
  return (const void*)combine_grad_kernel<T, 1>;
}

int check_route(int64_t tokens, int64_t stride, int experts, int k, int score, int dtype) {
  if (!float_dtype(dtype)) return report_error(DGN_ERR_UNSUPPORTED, "logits are float16, bfloat16 or float32");
  if (tokens < 0 || tokens > INT32_MAX) return report_error(DGN_ERR_ARG, "a call takes 0..2^31-1 tokens");
  if (experts < 1 || experts > kMaxExperts) return report_error(DGN_ERR_ARG, "a call takes 1..1024 experts");
  if (k < 1 || k > kMaxChoices || k > experts)
    return report_error(DGN_ERR_ARG, "k must be 1..32 and at most the number of experts");
  if (score != DGN_SCORE_SOFTMAX && score != DGN_SCORE_SIGMOID) return report_error(DGN_ERR_ARG, "unknown score");
  if (stride < experts) return report_error(DGN_ERR_ARG, "a row stride is shorter than the row");
  return DGN_OK;
}

int check_move(int64_t tokens, int k, int64_t capacity, int64_t row) {
  if (tokens < 0 || tokens > INT32_MAX || k < 1 || k > kMaxChoices || tokens * k > INT32_MAX)
    return report_error(DGN_ERR_ARG, "a token has 1..32 choices, a call fewer than 2^31");
  if (capacity < 0 || capacity > INT32_MAX) return report_error(DGN_ERR_ARG, "capacity must be 0..2^31-1 rows");
  if (row < 1 || row > kMaxRow) return report_error(DGN_ERR_ARG, "rows must not be empty or pass 2^30 elements or bytes");
  return DGN_OK;
}

int check_experts(int experts) {
  if (experts < 1 || experts > kMaxExperts) return report_error(DGN_ERR_ARG, "a call takes 1..1024 experts");
  return DGN_OK;
}

int null_pointer(const char* message) { return report_error(DGN_ERR_ARG, message); }
int misaligned() { return report_error(DGN_ERR_ARG, "a pointer is not aligned to its element size"); }

}  // namespace

#define DGN_ON(device) \
  OnDevice on(device); \
  if (on.error() != cudaSuccess) return report_error(DGN_ERR_CUDA, cudaGetErrorString(on.error()))

extern "C" int dgn_route(const void* logits, int64_t stride, const float* bias, const uint8_t* mask, int32_t* indices,
                         float* weights, int64_t tokens, int experts, int k, int score, int groups, int keep, int best,
                         int renormalize, float scale, int dtype, int device, void* stream) {
  int rc = check_route(tokens, stride, experts, k, score, dtype);
  if (rc != DGN_OK) return rc;
  if (groups < 1 || groups > kMaxGroups || experts % groups != 0)
    return report_error(DGN_ERR_ARG, "groups must be 1..32 and divide the number of experts");
  if (keep < 1 || keep > groups) return report_error(DGN_ERR_ARG, "at least one group is kept and at most all");
  if (best != 1 && best != 2) return report_error(DGN_ERR_ARG, "a group is valued by its best 1 or 2 experts");
  if (tokens == 0) return DGN_OK;
  if (!logits || !indices || !weights) return null_pointer("dgn_route: null pointer");
  if (!aligned(logits, dgn_dtype_size(dtype)) || !aligned(bias, 4) || !aligned(indices, 4) || !aligned(weights, 4))
    return misaligned();
  RouteParams p;
  p.logits = static_cast<const char*>(logits);
  p.bias = bias;
  p.mask = mask;
  p.indices = indices;
  p.weights = weights;
  p.tokens = tokens;
  p.stride = stride;
  p.experts = experts;
  p.k = k;
  p.sigmoid = score == DGN_SCORE_SIGMOID;
  p.groups = groups;
  p.keep = keep;
  p.best = best;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  p.bits = 1;
  while (1 << p.bits < experts) ++p.bits;
  p.magic = (unsigned)ceil_div(1 << 20, experts / groups);
  const int elems = 16 / (int)dgn_dtype_size(dtype), teams = 32 / route_lanes(experts);
  const bool vec = experts % elems == 0 && stride % elems == 0 && aligned(logits, 16) && aligned(bias, 16);
  const int width = experts / groups, run = width / elems;
  p.group_lanes = vec && width % elems == 0 && (run & (run - 1)) == 0 && run <= 32 / teams ? run : 0;
  const void* fn = dtype == DGN_F32   ? (vec ? route_fn<float, true>(experts) : route_fn<float, false>(experts))
                   : dtype == DGN_F16 ? (vec ? route_fn<__half, true>(experts) : route_fn<__half, false>(experts))
                   : vec              ? route_fn<__nv_bfloat16, true>(experts)
                                      : route_fn<__nv_bfloat16, false>(experts);
  DGN_ON(device);
  void* args[] = {&p};
  const int warps = kRouteThreads / 32;
  return launch(fn, dim3((unsigned)ceil_div(tokens, warps * teams)), dim3(kRouteThreads),
                (size_t)warps * route_shared(experts, groups, teams), stream, args);
}

extern "C" int dgn_route_grad(const float* grad_weights, const void* logits, int64_t stride, const int32_t* indices,
                              void* grad_logits, int64_t tokens, int experts, int k, int score, int renormalize,
                              float scale, int dtype, int device, void* stream) {
  int rc = check_route(tokens, stride, experts, k, score, dtype);
  if (rc != DGN_OK) return rc;
  if (tokens == 0) return DGN_OK;
  if (!grad_weights || !logits || !indices || !grad_logits) return null_pointer("dgn_route_grad: null pointer");
  const size_t es = dgn_dtype_size(dtype);
  if (!aligned(logits, es) || !aligned(grad_logits, es) || !aligned(indices, 4) || !aligned(grad_weights, 4))
    return misaligned();
  RouteGradParams p;
  p.grad_weights = grad_weights;
  p.logits = static_cast<const char*>(logits);
  p.indices = indices;
  p.grad = static_cast<char*>(grad_logits);
  p.tokens = tokens;
  p.stride = stride;
  p.experts = experts;
  p.k = k;
  p.sigmoid = score == DGN_SCORE_SIGMOID;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  const int elems = 16 / (int)es;
  const bool vec = experts % elems == 0 && stride % elems == 0 && aligned(logits, 16) && aligned(grad_logits, 16);
  const void* fn = dtype == DGN_F32   ? (vec ? route_grad_fn<float, true>(experts) : route_grad_fn<float, false>(experts))
                   : dtype == DGN_F16 ? (vec ? route_grad_fn<__half, true>(experts) : route_grad_fn<__half, false>(experts))
                   : vec              ? route_grad_fn<__nv_bfloat16, true>(experts)
                                      : route_grad_fn<__nv_bfloat16, false>(experts);
  DGN_ON(device);
  void* args[] = {&p};
  return launch(fn, dim3((unsigned)ceil_div(tokens, kRouteThreads / route_lanes(experts))), dim3(kRouteThreads), 0, stream,
                args);
}

extern "C" int64_t dgn_expert_plan_workspace(int64_t slots, int experts) {
  const int blocks = plan_blocks(slots);
  return blocks == 1 || experts < 1 ? 0 : (int64_t)blocks * experts * (int64_t)sizeof(int);
}

extern "C" int dgn_expert_plan(const int32_t* indices, int64_t slots, int experts, int align, int32_t* counts,
                               int32_t* offsets, int32_t* ends, int32_t* positions, void* workspace,
                               int64_t workspace_bytes, int device, void* stream) {
  int rc = check_experts(experts);
  if (rc != DGN_OK) return rc;
  if (slots < 0 || slots > INT32_MAX) return report_error(DGN_ERR_ARG, "a call takes 0..2^31-1 slots");
  if (align < 1 || slots + (slots < experts ? slots : experts) * ((int64_t)align - 1) > INT32_MAX)
    return report_error(DGN_ERR_ARG, "align must be positive and the rows fewer than 2^31");
  if (!counts || !offsets || !ends || (slots && (!indices || !positions))) return null_pointer("dgn_expert_plan: null pointer");
  if (!aligned(indices, 4) || !aligned(counts, 4) || !aligned(offsets, 4) || !aligned(ends, 4) ||
      !aligned(positions, 4) || !aligned(workspace, 4))
    return misaligned();
  const int64_t need = dgn_expert_plan_workspace(slots, experts);
  if (need && (!workspace || workspace_bytes < need))
    return report_error(DGN_ERR_ARG, "dgn_expert_plan: workspace too small");
  PlanParams p;
  p.indices = indices;
  p.counts = counts;
  p.offsets = offsets;
  p.ends = ends;
  p.positions = positions;
  p.parts = static_cast<int*>(workspace);
  p.slots = slots;
  p.experts = experts;
  p.align = align;
  const int blocks = plan_blocks(slots);
  p.span = ceil_div(ceil_div(slots, blocks), 32) * 32;
  DGN_ON(device);
  void* args[] = {&p};
  if (blocks > 1) {
    rc = launch((const void*)plan_count_kernel, dim3(blocks), dim3(kPlanThreads), experts * sizeof(int), stream, args);
    if (rc != DGN_OK) return rc;
  }
  const int smem = (kPlanWarps + 2) * experts * (int)sizeof(int);
  const auto put_in = blocks > 1 ? launch_behind : launch;
  return put_in((const void*)plan_place_kernel, dim3(blocks), dim3(kPlanThreads), smem, stream, args);
}

extern "C" int dgn_expert_dispatch(const void* x, int64_t x_stride, int64_t row_bytes, const int32_t* positions,
                                   const int32_t* offsets, const int32_t* ends, void* out, int64_t tokens, int k,
                                   int experts, int64_t capacity, int device, void* stream) {
  int rc = check_move(tokens, k, capacity, row_bytes);
  if (rc == DGN_OK) rc = check_experts(experts);
  if (rc != DGN_OK) return rc;
  if (x_stride < row_bytes) return report_error(DGN_ERR_ARG, "a row stride is shorter than the row");
  if (tokens == 0 || capacity == 0) return DGN_OK;
  if (!x || !positions || !offsets || !ends || !out) return null_pointer("dgn_expert_dispatch: null pointer");
  if (!aligned(positions, 4) || !aligned(offsets, 4) || !aligned(ends, 4)) return misaligned();
  MoveParams p;
  p.x = static_cast<const char*>(x);
  p.positions = positions;
  p.offsets = offsets;
  p.ends = ends;
  p.out = static_cast<char*>(out);
  p.tokens = tokens;
  p.x_stride = x_stride;
  p.row_bytes = row_bytes;
  p.capacity = capacity;
  p.k = k;
  p.experts = experts;
  // The widest word that divides the addresses, the strides and the row.
  const auto fits = [&](int w) { return aligned(x, w) && aligned(out, w) && x_stride % w == 0 && row_bytes % w == 0; };
  const int word = fits(16) ? 16 : fits(8) ? 8 : fits(4) ? 4 : 1;
  const int team = move_team(word == 1 ? ceil_div(row_bytes, 16) : row_bytes / word, tokens);
  p.share = clear_share(tokens * k, experts, capacity, row_bytes);
  const void* fn = word == 16  ? dispatch_fn<uint4>(team)
                   : word == 8 ? dispatch_fn<uint2>(team)
                   : word == 4 ? dispatch_fn<unsigned>(team)
                               : dispatch_fn<unsigned char>(team);
  DGN_ON(device);
  void* args[] = {&p};
  return launch(fn, dim3((unsigned)(ceil_div(tokens, kMoveThreads / team) + (int64_t)experts * p.share)), dim3(kMoveThreads), 0, stream, args);
}

extern "C" int dgn_expert_combine(const void* rows, const int32_t* positions, const float* weights,
                                  const void* residual, int64_t residual_stride, void* out, int64_t tokens, int k,
                                  int64_t cols, int64_t capacity, int dtype, int device, void* stream) {
  int rc = check_move(tokens, k, capacity, cols);
  if (rc != DGN_OK) return rc;
  if (!float_dtype(dtype)) return report_error(DGN_ERR_UNSUPPORTED, "rows are float16, bfloat16 or float32");
  if (residual && residual_stride < cols) return report_error(DGN_ERR_ARG, "a row stride is shorter than the row");
  if (tokens == 0) return DGN_OK;
  if ((!rows && capacity) || !positions || !out) return null_pointer("dgn_expert_combine: null pointer");
  const int es = (int)dgn_dtype_size(dtype), elems = 16 / es;
  if (!aligned(rows, es) || !aligned(residual, es) || !aligned(out, es) || !aligned(positions, 4) || !aligned(weights, 4))
    return misaligned();
  // Whether words of `w` elements divide the rows and what they lie in.
  const auto fits = [&](int w) {
    return cols % w == 0 && aligned(rows, w * es) && aligned(out, w * es) &&
           (!residual || (aligned(residual, w * es) && residual_stride % w == 0));
  };
  const int word = fits(elems) ? elems : es == 2 && fits(2) ? 2 : 1;
  CombineParams p;
  p.rows = static_cast<const char*>(rows);
  p.positions = positions;
  p.weights = weights;
  p.residual = static_cast<const char*>(residual);
  p.out = static_cast<char*>(out);
  p.tokens = tokens;
  p.cols = (int)cols;
  p.capacity = capacity;
  p.residual_stride = residual_stride;
  p.k = k;
  const CombineTeam team = combine_team(ceil_div(cols, elems));
  const void* fn = dtype == DGN_F32   ? combine_fn<float>(word, team)
                   : dtype == DGN_F16 ? combine_fn<__half>(word, team)
                                      : combine_fn<__nv_bfloat16>(word, team);
  DGN_ON(device);
  void* args[] = {&p};
  return launch(fn, dim3((unsigned)ceil_div(tokens, kMoveThreads / team.threads)), dim3(kMoveThreads), 0, stream, args);
}

extern "C" int dgn_expert_combine_grad(const void* grad_out, int64_t grad_out_stride, const void* rows,
                                       const int32_t* positions, const float* weights, const int32_t* offsets,
                                       const int32_t* ends, void* grad_rows, float* grad_weights, int64_t tokens,
                                       int k, int experts, int64_t cols, int64_t capacity, int dtype, int device,
                                       void* stream) {
  int rc = check_move(tokens, k, capacity, cols);
  if (rc == DGN_OK) rc = check_experts(experts);
  if (rc != DGN_OK) return rc;
  if (!float_dtype(dtype)) return report_error(DGN_ERR_UNSUPPORTED, "rows are float16, bfloat16 or float32");
  if (grad_out_stride < cols) return report_error(DGN_ERR_ARG, "a row stride is shorter than the row");
  if (tokens == 0) return DGN_OK;
  if (!grad_out || !positions || !weights || !offsets || !ends || !grad_weights || (capacity && (!rows || !grad_rows)))
    return null_pointer("dgn_expert_combine_grad: null pointer");
  const int es = (int)dgn_dtype_size(dtype), elems = 16 / es;
  if (!aligned(grad_out, es) || !aligned(rows, es) || !aligned(grad_rows, es) || !aligned(positions, 4) ||
      !aligned(weights, 4) || !aligned(offsets, 4) || !aligned(ends, 4) || !aligned(grad_weights, 4))
    return misaligned();
  const auto fits = [&](int w) {
    return cols % w == 0 && grad_out_stride % w == 0 && aligned(grad_out, w * es) && aligned(rows, w * es) &&
           aligned(grad_rows, w * es);
  };
  const int word = fits(elems) ? elems : es == 2 && fits(2) ? 2 : 1;
  CombineGradParams p;
  p.grad_out = static_cast<const char*>(grad_out);
  p.rows = static_cast<const char*>(rows);
  p.positions = positions;
  p.weights = weights;
  p.offsets = offsets;
  p.ends = ends;
  p.grad_rows = static_cast<char*>(grad_rows);
  p.grad_weights = grad_weights;
  p.slots = tokens * k;
  p.cols = (int)cols;
  p.capacity = capacity;
  p.grad_out_stride = grad_out_stride;
  p.k = k;
  p.experts = experts;
  p.share = clear_share(tokens * k, experts, capacity, cols * es);
  const void* fn = dtype == DGN_F32   ? combine_grad_fn<float>(word)
                   : dtype == DGN_F16 ? combine_grad_fn<__half>(word)
                                      : combine_grad_fn<__nv_bfloat16>(word);
  DGN_ON(device);
  void* args[] = {&p};
  return launch(fn, dim3((unsigned)(ceil_div(tokens * k, kMoveThreads / 32) + (int64_t)experts * p.share)), dim3(kMoveThreads), 0, stream, args);
}

extern "C" int dgn_expert_update_bias(const float* bias, const int32_t* counts, float* out, int experts, float rate,
                                      int device, void* stream) {
  int rc = check_experts(experts);
  if (rc != DGN_OK) return rc;
  if (!bias || !counts || !out) return null_pointer("dgn_expert_update_bias: null pointer");
  if (!aligned(bias, 4) || !aligned(counts, 4) || !aligned(out, 4)) return misaligned();
  DGN_ON(device);
  void* args[] = {&bias, &counts, &out, &experts, &rate};
  return launch((const void*)update_bias_kernel, dim3(1), dim3(1024), 0, stream, args);
}
