// Gated experts: the gate that routes each row to k of E experts, the plan that
// sorts the (row, choice) slots by expert, and the join of the experts' outputs;
// with the backward passes of gate and join.
#include <type_traits>

#include "common.h"

namespace nerfhip {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 32;
constexpr int kMaxGroups = 64;

struct RouteArgs {
  const void* logits;   // [T][E], rows ld apart
  int64_t ld;
  int64_t T;
  int E, k, sigmoid, groups, top_groups, group_top2, renorm;
  const float* bias;    // [E] or null
  float scale;
  float* weights;       // [T][k]
  int* experts;         // [T][k]
};

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// Reductions over the L (16 or 64) lanes of a row: inside 16 lanes by DPP.
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
template <int L, class OP>
__device__ __forceinline__ unsigned reduce32(unsigned v, OP op) {
  v = op(v, dpp<0xB1>(v));    // lane ^ 1
  v = op(v, dpp<0x4E>(v));    // lane ^ 2
  v = op(v, dpp<0x141>(v));   // the other four of 8
  v = op(v, dpp<0x140>(v));   // the other eight of 16
  if constexpr (L == 64) {   // the lanes 16 and 32 away, without LDS: a value swapped with itself
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(b[0], b[1]);
  }
  return v;
}
template <int L>
__device__ __forceinline__ float row_max(float v) {
  return __uint_as_float(reduce32<L>(__float_as_uint(v), [](unsigned a, unsigned b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int L>
__device__ __forceinline__ float row_sum(float v) {
  return __uint_as_float(reduce32<L>(__float_as_uint(v), [](unsigned a, unsigned b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int L>
__device__ __forceinline__ unsigned row_or(unsigned v) {
  return reduce32<L>(v, [](unsigned a, unsigned b) { return a | b; });
}
// LDS written by a row's lanes (all of one wave) may be read by them: a wave's LDS accesses are done in
// their order, so only the compiler has to keep it (a workgroup's fence would wait for stores to memory).
__device__ __forceinline__ void row_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A key and its expert as one positive number: 2^52 + (the key's bits in rising order, 32 bits) * 1024 +
// (1023 - expert). Larger: the higher key, or at equal keys the lower index. One v_max_f64 compares
// both (its rate is FP32's), and a comparison of sorting is two instructions.
__device__ __forceinline__ double pack_key(float key, int e) {
  const unsigned b = __float_as_uint(key + 0.0f);   // (-0 counts as 0)
  const unsigned u = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
  return __hiloint2double((int)(0x43300000u | u >> 22), (int)(u << 10 | (unsigned)(1023 - e)));
}
__device__ __forceinline__ int index_of(double p) { return 1023 - (__double2loint(p) & 1023); }
__device__ __forceinline__ float key_of(double p) {
  const unsigned u = (unsigned)__double2hiint(p) << 22 | (unsigned)__double2loint(p) >> 10;
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  return __hiloint2double((int)dpp<CTRL>((unsigned)__double2hiint(v)), (int)dpp<CTRL>((unsigned)__double2loint(v)));
}
template <int L, class OP>
__device__ __forceinline__ double reduce64(double v, OP op) {
  v = op(v, dpp64<0xB1>(v));
  v = op(v, dpp64<0x4E>(v));
  v = op(v, dpp64<0x141>(v));
  v = op(v, dpp64<0x140>(v));
  if constexpr (L == 64) {
    const unsigned lo = (unsigned)__double2loint(v), hi = (unsigned)__double2hiint(v);
    const auto l16 = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto h16 = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = op(__hiloint2double((int)h16[0], (int)l16[0]), __hiloint2double((int)h16[1], (int)l16[1]));
    const unsigned lo2 = (unsigned)__double2loint(v), hi2 = (unsigned)__double2hiint(v);
    const auto l32 = __builtin_amdgcn_permlane32_swap(lo2, lo2, false, false);
    const auto h32 = __builtin_amdgcn_permlane32_swap(hi2, hi2, false, false);
    v = op(__hiloint2double((int)h32[0], (int)l32[0]), __hiloint2double((int)h32[1], (int)l32[1]));
  }
  return v;
}
template <int L>
__device__ __forceinline__ double row_max(double v) {
  return reduce64<L>(v, [](double a, double b) { return fmax(a, b); });
}
template <int L>
__device__ __forceinline__ double row_sum(double v) {
  return reduce64<L>(v, [](double a, double b) { return a + b; });
}
// A sorting network (merge exchange) for a power of two of values, the largest first.
template <int N>
__device__ __forceinline__ void sort_down(double (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const double hi = fmax(v[i + j], v[i + j + k]), lo = fmin(v[i + j], v[i + j + k]);
            v[i + j] = hi;
            v[i + j + k] = lo;
          }
}

// (key, index) with the higher key, or at equal keys the lower index, over the lanes of a row.
template <int L>
__device__ __forceinline__ void row_best(double& key, int& idx) {
  const double m = row_max<L>(key);
  idx = (int)reduce32<L>(key == m ? (unsigned)idx : ~0u, [](unsigned a, unsigned b) { return a < b ? a : b; });
  key = m;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
// The least key, that of NaN and -inf: below every number that 32 bits hold, -3.4e38 (a mask of the type's
// lowest value) too.
template <class F>
__device__ __forceinline__ F lowest();
template <>
__device__ __forceinline__ float lowest<float>() { return -__builtin_inff(); }
template <>
__device__ __forceinline__ double lowest<double>() { return -1.7976931348623157e+308; }

// An expert's index from a lane's value v: runs of 4 neighbours (one 8- or 16-byte load).
template <int L>
__device__ __forceinline__ int expert_of(int lane, int v) {
  return ((v >> 2) * L + lane) * 4 + (v & 3);
}

// The scores s of a lane's logits, in F.
template <class F, int L, int V>
__device__ __forceinline__ void scores(const RouteArgs& a, const float (&x)[V], float top, int lane, F (&s)[V]) {
  if (a.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = (F)1 / ((F)1 + exp_of(-(F)x[v]));
  } else {
    F sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = expert_of<L>(lane, v) < a.E ? exp_of((F)x[v] - (F)top) : (F)0;
      sum += s[v];
    }
    sum = (F)1 / row_sum<L>(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= sum;
  }
}

template <class F>
__device__ __forceinline__ F ranked(F key) {
  return key > lowest<F>() ? key : lowest<F>();
}

// An expert's group: a shift where groups have a power of two of experts (bits >= 0).
__device__ __forceinline__ int per_bits(int per) { return per & (per - 1) ? -1 : 31 - __builtin_clz(per); }
__device__ __forceinline__ int group_of(int e, int per, int bits) { return bits >= 0 ? e >> bits : e / per; }

// The groups that stay (bits) by the highest or two highest of their keys; `doubt`: whether a dropped one may
// lie above a kept one when each group is off by its scores' errors (`tol` for two groups together) and its keys'
// roundings, which follow the keys' size and not their sum's (keys of a group may cancel): 2^-24 of
// each key and of the sum, taken twice. Any dropped group may be the one, not the next alone.
template <class F, int L, int V>
__device__ __forceinline__ unsigned long long keep_groups(const RouteArgs& a, const F (&key)[V], F* ks, int lane, F tol,
                                                          bool& doubt) {
  const int per = a.E / a.groups, bits = per_bits(per);
  F* gs = ks + a.E + a.groups;
  F* size = gs + a.groups;   // 32 bits: a group's |keys|, 0 for a score of the lowest
  auto score = [&](F b1, F b2) { return a.group_top2 && per > 1 ? (b2 > lowest<F>() ? b1 + b2 : lowest<F>()) : b1; };
  auto put = [&](int j, F b1, F b2) {
    const F s = score(b1, b2);
    gs[j] = s;
    if (sizeof(F) == 4) size[j] = s > lowest<F>() ? fabsf((float)b1) + (a.group_top2 && per > 1 ? fabsf((float)b2) : 0.0f) : 0.0f;
  };
  if (sizeof(F) == 4 && per >= 4 && per <= 64 && bits >= 0) {
    // a group is whole lanes' runs of 4: the two highest by DPP
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      float b1 = -__builtin_inff(), b2 = b1;
      auto add = [&](float o1, float o2) {
        b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
        b1 = fmaxf(b1, o1);
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) add((float)key[v + i], -__builtin_inff());
      if (per > 4) add(dpp_f<0xB1>(b1), dpp_f<0xB1>(b2));
      if (per > 8) add(dpp_f<0x4E>(b1), dpp_f<0x4E>(b2));
      if (per > 16) add(dpp_f<0x141>(b1), dpp_f<0x141>(b2));
      if (per > 32) add(dpp_f<0x140>(b1), dpp_f<0x140>(b2));
      const int e = expert_of<L>(lane, v);
      if (e < a.E && (e & (per - 1)) == 0) put(e >> bits, b1, b2);
    }
  } else {
    // through LDS, lane j takes group j
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = expert_of<L>(lane, v);
      if (e < a.E) ks[e + group_of(e, per, bits)] = key[v];   // (a word between groups: they lie in different banks)
    }
    row_fence();
    for (int j = lane; j < a.groups; j += L) {
      F b1 = -(F)__builtin_inff(), b2 = b1;
#pragma unroll 8
      for (int i = 0; i < per; ++i) {
        const F v = ks[j * (per + 1) + i];
        b2 = v > b1 ? b1 : (v > b2 ? v : b2);
        b1 = v > b1 ? v : b1;
      }
      put(j, b1, b2);
    }
  }
  row_fence();
  // a lane ranks its own groups; all of the row's lanes join their bits
  unsigned lo = 0, hi = 0;
  F last = __builtin_inff(), first = -(F)__builtin_inff();   // lowest kept, highest dropped, by their errors
  for (int j = lane; j < a.groups; j += L) {
    const F mine = gs[j], err = sizeof(F) == 4 ? (F)2.4e-7f * size[j] : (F)0;
    int better = 0;
#pragma unroll 8
    for (int i = 0; i < a.groups; ++i) better += gs[i] > mine || (gs[i] == mine && i < j);
    if (better < a.top_groups) {
      lo |= j < 32 ? 1u << j : 0u;
      hi |= j < 32 ? 0u : 1u << (j - 32);
      last = mine - err < last ? mine - err : last;
    } else {
      first = mine + err > first ? mine + err : first;
    }
  }
  const unsigned long long keep = (unsigned long long)row_or<L>(hi) << 32 | row_or<L>(lo);
  if (sizeof(F) == 4) {
    last = -row_max<L>((float)-last);
    first = row_max<L>((float)first);
    // (not a number: both beyond 32 bits' range, or both the lowest)
    doubt = a.top_groups < a.groups && !(last - first >= tol);
  }
  return keep;
}

// Chooses a row's k experts (into chosen[] in LDS, which its lanes read after a row_fence).
//
// The order is that of 64-bit keys. Without a bias the keys are the logits themselves; with
// one they are computed in 32 bits, and where two neighbours in the order (or the last group kept
// and the first one dropped) are nearer than the keys' error and not made of equal inputs, in
// 64 bits again: then only for the experts that can be among the first k (scores of a softmax: for
// all, its sum takes them all). Nearly every row pays for 32 bits only.
template <int L, int V, class T>
__device__ __forceinline__ void choose(const RouteArgs& a, const T* row, const float (&x)[V], float top, double* lds, int* chosen,
                       int lane) {
  float key[V];
  unsigned out = 0;       // bit v: out of reach (behind the last expert, or in a group that was dropped)
  float tol = 0.0f;   // twice two keys' errors, apart from their last rounding
  const bool scored = a.bias != nullptr || (a.groups > 1 && a.group_top2);
  const int per = a.E / a.groups, bits = per_bits(per);
  if (scored) {
    scores<float, L, V>(a, x, top, lane, key);
    // sigmoid: 3 steps of a score (at most 1). Softmax: 1.2e-6 of one (the sum of 1024 terms: 20 steps),
    // the row's largest at most
    float most = 0.0f;
    if (!a.sigmoid) {
#pragma unroll
      for (int v = 0; v < V; ++v) most = fmaxf(most, key[v]);
      most = row_max<L>(most);
    }
    tol = a.sigmoid ? 8e-7f : 5e-6f * most;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = expert_of<L>(lane, v);
      key[v] = e < a.E ? ranked(a.bias ? key[v] + a.bias[e] : key[v]) : lowest<float>();
      out |= e < a.E ? 0u : 1u << v;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      key[v] = ranked(x[v]);
      out |= expert_of<L>(lane, v) < a.E ? 0u : 1u << v;
    }
  }
  unsigned long long keep = ~0ull;
  if (a.groups > 1) {
    bool doubt = false;
    // (the highest logits without a bias: exact)
    keep = keep_groups<float, L, V>(a, key, (float*)lds, lane, 2.0f * tol, doubt);
    if (doubt && scored) {
      double k64[V];
      scores<double, L, V>(a, x, top, lane, k64);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = expert_of<L>(lane, v);
        k64[v] = e < a.E ? ranked(a.bias ? k64[v] + (double)a.bias[e] : k64[v]) : -(double)__builtin_inff();
      }
      row_fence();
      keep = keep_groups<double, L, V>(a, k64, lds, lane, 0.0, doubt);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = expert_of<L>(lane, v);
      if (e < a.E) {
        if (!a.bias) key[v] = ranked(x[v]);   // the order of the logits
        if (!((keep >> group_of(e, per, bits)) & 1)) out |= 1u << v;
      }
    }
  }
  bool doubt = false;
  float before = __builtin_inff();
  int ib = 0;
  const int rounds = a.bias && a.k < a.E ? a.k + 1 : a.k;   // one more: the first one left out
  double order[V];   // a lane's keys, highest first; 0 (in key_of: NaN) behind them
#pragma unroll
  for (int v = 0; v < V; ++v) order[v] = out >> v & 1 ? 0.0 : pack_key(key[v], expert_of<L>(lane, v));
  sort_down<V>(order);
  auto take = [&](auto depth) {   // (a lane gives at most `rounds` of its keys)
    constexpr int D = decltype(depth)::value;
    for (int j = 0; j < rounds; ++j) {
      const double first = row_max<L>(order[0]);
      const bool mine = order[0] == first;
#pragma unroll
      for (int v = 0; v + 1 < D; ++v) order[v] = mine ? order[v + 1] : order[v];
      order[D - 1] = mine ? 0.0 : order[D - 1];
      const float best = key_of(first);
      const int idx = index_of(first);
      if (a.bias && j > 0 && best > lowest<float>() && before - best < tol + 2.4e-7f * fabsf(before))
        doubt = doubt || !((float)row[ib] == (float)row[idx] && a.bias[ib] == a.bias[idx]);
      if (j < a.k) {
        before = best;
        ib = idx;
        if (lane == 0) chosen[j] = idx;
      }
    }
  };
  if (V > 9 && rounds <= 9) take(std::integral_constant<int, (V > 9 ? 9 : V)>());
  else take(std::integral_constant<int, V>());
  if (!doubt) return;
  // 64 bits, for the experts that may be among the first k: not below the k-th by more than the error
  const float least = fmaxf(before - tol - 2.4e-7f * fabsf(before), lowest<float>());   // (inf - inf: all of them)
  double k64[V];
  if (a.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      k64[v] = -(double)__builtin_inff();
      if (key[v] >= least && !(out >> v & 1)) k64[v] = ranked(1.0 / (1.0 + exp(-(double)x[v])) + (double)a.bias[expert_of<L>(lane, v)]);
    }
  } else {
    scores<double, L, V>(a, x, top, lane, k64);
#pragma unroll
    for (int v = 0; v < V; ++v)
      k64[v] = key[v] >= least && !(out >> v & 1) ? ranked(k64[v] + (double)a.bias[expert_of<L>(lane, v)]) : -(double)__builtin_inff();
  }
  row_fence();
  for (int j = 0; j < a.k; ++j) {
    double best = -(double)__builtin_inff();
    int idx = 0x7fffffff;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (k64[v] > best) {
        best = k64[v];
        idx = expert_of<L>(lane, v);
      }
    row_best<L>(best, idx);
    if (lane == 0) chosen[j] = idx;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (expert_of<L>(lane, v) == idx) k64[v] = -(double)__builtin_inff();
  }
}

// A chosen expert's part in the weights, r_j of the formulas: w_j = scale * r_j.
// Renormalised: s_j / sum of the chosen s, with the chosen logits' largest taken out first
// (m: their maximum; for sigmoid s e^-m = 1 / (e^m + e^(m - l)), m <= 0), so that scores too small
// for 32 bits still have their ratios. In 32 bits, unlike the order: some steps of 2^-24 (5e-8 of a row's norm
// against 64 bits where one rounding is 3e-8), as much as an FP32 sum over experts' rows adds again.
__device__ __forceinline__ float chosen_part(const RouteArgs& a, float l, float m) {
  if (a.renorm) return a.sigmoid ? 1.0f / (expf(m) + expf(m - l)) : expf(l - m);
  return a.sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - m);
}

// A lane's logits, -inf behind the last expert.
template <int L, int V, class T, bool VEC>
__device__ __forceinline__ void load_logits(const T* row, int E, int lane, float (&x)[V]) {
#pragma unroll
  for (int v = 0; v < V; v += 4) {
    const int e = expert_of<L>(lane, v);
    if (VEC) {
      if (e < E) {
        const Vec<T, 4> q = *(const Vec<T, 4>*)(row + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[v + i] = (float)q.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[v + i] = -__builtin_inff();
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[v + i] = e + i < E ? (float)row[e + i] : -__builtin_inff();
    }
  }
}

// Rows of L lanes, 256 / L rows in a workgroup. Reads the logits once, writes k weights and experts.
// Bound by instructions: sorting a lane's keys and the k rounds of the choice (T = 65536: E = 64, k = 2 in
// 11 us, 16.8 MB at 1.5 TB/s; E = 256, k = 8 in 32 us), by one row's latency for few rows (3 us for T = 1).
template <int L, int V, class T, bool VEC>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
  extern __shared__ double route_lds[];
  constexpr int R = 256 / L;
  const int lane = threadIdx.x % L, r = threadIdx.x / L;
  const int64_t t = (int64_t)blockIdx.x * R + r;
  const int per_row = a.groups > 1 ? a.E + 2 * a.groups : 0;
  double* keys = route_lds + (int64_t)r * per_row;
  int* chosen = (int*)(route_lds + (int64_t)R * per_row) + r * kMaxChoices;
  // (a workgroup's last rows may lie behind T: they do the last row again and store nothing, so that
  // a wave's lanes stay together)
  const int64_t tr = t < a.T ? t : a.T - 1;
  const T* row = (const T*)a.logits + tr * a.ld;
  float x[V];
  load_logits<L, V, T, VEC>(row, a.E, lane, x);
  float top = -__builtin_inff();
  unsigned bad = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    top = fmaxf(top, x[v]);
    bad |= x[v] != x[v];
  }
  top = row_max<L>(top);
  bad = row_or<L>(bad) | (!a.sigmoid && top == __builtin_inff());
  choose<L, V>(a, row, x, top, keys, chosen, lane);
  row_fence();
  // lane j holds choice j (and j + L)
  constexpr int C = kMaxChoices / L > 1 ? kMaxChoices / L : 1;
  int e[C];
  float l[C], m = -__builtin_inff(), sum = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int j = lane + c * L;
    e[c] = j < a.k ? chosen[j] : 0;
    l[c] = j < a.k ? (float)row[e[c]] : -__builtin_inff();
    m = fmaxf(m, l[c]);
  }
  if (a.renorm) {
    m = row_max<L>(m);
    if (a.sigmoid) m = fminf(m, 0.0f);
#pragma unroll
    for (int c = 0; c < C; ++c) sum += lane + c * L < a.k ? chosen_part(a, l[c], m) : 0.0f;
    sum = row_sum<L>(sum);
  } else if (!a.sigmoid) {
    m = top;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += expert_of<L>(lane, v) < a.E ? expf(x[v] - top) : 0.0f;
    sum = row_sum<L>(sum);
  } else {
    m = top;
    sum = 1.0f;
  }
  const bool nothing = m == -__builtin_inff();   // every (chosen) logit is -inf
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int j = lane + c * L;
    if (t < a.T && j < a.k) {
      float w = nothing ? 0.0f : chosen_part(a, l[c], m) / sum * a.scale;
      if (bad) w = __builtin_nanf("");
      a.weights[t * a.k + j] = w;
      a.experts[t * a.k + j] = e[c];
    }
  }
}

struct RouteBwdArgs {
  RouteArgs f;          // logits, sizes, score, scale; experts: the forward's choice
  const float* dw;      // [T][k]
  void* dlogits;        // [T][E], contiguous
};

// d logits of a row: renormalised, only the chosen ones have a gradient:
//   softmax: scale r_j (g_j - sum_i r_i g_i);  sigmoid: that times (1 - s_j);
// not renormalised: softmax: p_e (scale g_e - sum_i scale g_i p_i) for every e; sigmoid: scale g s (1 - s).
// The row is put together in LDS and written in one sweep: 33.6 MB in 12 to 13 us (T = 65536, E = 64), 2.7 TB/s.
template <int L, int V, class T, bool VEC>
__global__ __launch_bounds__(256) void route_backward_kernel(const RouteBwdArgs b) {
  extern __shared__ float bwd_lds[];
  const RouteArgs& a = b.f;
  constexpr int R = 256 / L;
  const int lane = threadIdx.x % L, r = threadIdx.x / L;
  const int64_t t = (int64_t)blockIdx.x * R + r, tr = t < a.T ? t : a.T - 1;
  const T* row = (const T*)a.logits + tr * a.ld;
  float* buf = bwd_lds + r * V * L;
  float x[V], top = -__builtin_inff(), sum = 0.0f;
  unsigned bad = 0;
  load_logits<L, V, T, VEC>(row, a.E, lane, x);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    top = fmaxf(top, x[v]);
    bad |= x[v] != x[v];
  }
  top = row_max<L>(top);
  bad = row_or<L>(bad) | (!a.sigmoid && top == __builtin_inff());
#pragma unroll
  for (int v = 0; v < V; ++v) buf[expert_of<L>(lane, v)] = 0.0f;
  const int* ex = a.experts + tr * a.k;
  const float* dw = b.dw + tr * a.k;
  float m = top;
  if (a.renorm) {
    m = -__builtin_inff();
    for (int j = lane; j < a.k; j += L) {
      const int e = ex[j];
      if (e >= 0 && e < a.E) m = fmaxf(m, (float)row[e]);
    }
    m = row_max<L>(m);
    if (a.sigmoid) m = fminf(m, 0.0f);
    for (int j = lane; j < a.k; j += L) {
      const int e = ex[j];
      if (e >= 0 && e < a.E) sum += chosen_part(a, (float)row[e], m);
    }
    sum = row_sum<L>(sum);
  } else if (!a.sigmoid) {
#pragma unroll
    for (int v = 0; v < V; ++v) sum += expert_of<L>(lane, v) < a.E ? expf(x[v] - top) : 0.0f;
    sum = row_sum<L>(sum);
  } else {
    sum = 1.0f;
  }
  const bool nothing = m == -__builtin_inff();
  float dot = 0.0f;
  if (a.renorm || !a.sigmoid) {
    for (int j = lane; j < a.k; j += L) {
      const int e = ex[j];
      if (e >= 0 && e < a.E) dot += chosen_part(a, (float)row[e], m) / sum * dw[j];
    }
    dot = row_sum<L>(dot);
  }
  row_fence();
  for (int j = lane; j < a.k; j += L) {
    const int e = ex[j];
    if (e >= 0 && e < a.E) {
      const float l = (float)row[e], p = chosen_part(a, l, m) / sum;
      float d;
      if (a.renorm) {
        d = p * (dw[j] - dot);
        if (a.sigmoid) d = d / (1.0f + expf(l));          // 1 - s
      } else {
        d = a.sigmoid ? dw[j] * p * (1.0f / (1.0f + expf(l))) : dw[j] * p;
      }
      buf[e] = d * a.scale;
    }
  }
  row_fence();
  if (t < a.T) {
    T* out = (T*)b.dlogits + t * a.E;
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      const int e = expert_of<L>(lane, v);
      Vec<T, 4> o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float d = buf[e + i];
        if (!a.renorm && !a.sigmoid) d -= a.scale * dot * expf(x[v + i] - top) / sum;
        if (nothing) d = 0.0f;
        if (bad) d = __builtin_nanf("");
        o.v[i] = (T)d;
      }
      if (VEC) {
        if (e < a.E) *(Vec<T, 4>*)(out + e) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e + i < a.E) out[e + i] = o.v[i];
      }
    }
  }
}

// ---------------------------------------------------------------- the plan

// A stable counting sort of the n slots by expert. A wave counts, and later places, a run of
// neighbouring slots, 64 at a time in order: lanes with the same expert are found by ballots over
// the bits of its number, so the places follow from counts alone (no atomics that decide an order).
// Bound by the latency of its launches: 131072 slots in 4 + 2 + 5 us. Up to 8192 slots one workgroup does it
// all (8168 slots of 256 experts: 14 us a call, three launches 19; 16384: 25 and 19).
__device__ __forceinline__ unsigned long long same_expert(int e, bool live, int bits) {
  unsigned long long peers = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const bool one = (e >> b) & 1;
    const unsigned long long m = __ballot(one);
    peers &= one ? m : ~m;
  }
  return peers;
}

constexpr int kPlanSegs = 1024;   // runs of slots (one wave each) of a large plan
constexpr int kPlanSmall = 8192;  // up to here one workgroup does everything (LDS: 18 words an expert)
bool plan_is_small(int64_t n, int E) { return n <= kPlanSmall && E <= 512; }

__device__ __forceinline__ void plan_count(const int* experts, int64_t lo, int64_t hi, int E, int* cnt, int lane, int bits) {
  for (int64_t i0 = lo; i0 < hi; i0 += 256) {
    int ex[4];   // (4 times 64 slots on their way at once)
#pragma unroll
    for (int u = 0; u < 4; ++u) ex[u] = i0 + u * 64 + lane < hi ? experts[i0 + u * 64 + lane] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + u * 64 >= hi) break;
      const int e = ex[u];
      const bool live = e >= 0 && e < E;
      const unsigned long long peers = same_expert(e, live, bits);
      if (live && __builtin_ctzll(peers) == lane) cnt[e] += __builtin_popcountll(peers);
      row_fence();
    }
  }
}

__device__ __forceinline__ void plan_place(const int* experts, int64_t lo, int64_t hi, int E, int* at, int lane, int bits,
                                           int* order, int* position) {
  for (int64_t i0 = lo; i0 < hi; i0 += 256) {
    int ex[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) ex[u] = i0 + u * 64 + lane < hi ? experts[i0 + u * 64 + lane] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + u * 64 >= hi) break;
      const int64_t i = i0 + u * 64 + lane;
      const int e = ex[u];
      const bool live = e >= 0 && e < E;
      const unsigned long long peers = same_expert(e, live, bits);
      int p = -1;
      if (live) p = at[e] + __builtin_popcountll(peers & ((1ull << lane) - 1));
      row_fence();
      if (live && __builtin_ctzll(peers) == lane) at[e] += __builtin_popcountll(peers);
      row_fence();
      if (i < hi) position[i] = p;
      if (live) order[p] = (int)i;
    }
  }
}

// Exclusive prefix sums of tot[0..E) into base[0..E], by the whole workgroup (a power of two of
// 256 threads or more; part: one word for each wave).
__device__ __forceinline__ void prefix(const int* tot, int* base, int E, int* part) {
  const int t = threadIdx.x, nt = blockDim.x, lane = t & 63, w = t >> 6;
  const int per = (E + nt - 1) / nt;
  int mine = 0;
  for (int i = 0; i < per; ++i) mine += t * per + i < E ? tot[t * per + i] : 0;
  int sum = mine;
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 63) part[w] = sum;
  __syncthreads();
  int off = sum - mine;
  for (int i = 0; i < w; ++i) off += part[i];
  for (int i = 0; i < per; ++i) {
    const int e = t * per + i;
    if (e < E) {
      base[e] = off;
      off += tot[e];
      if (e == E - 1) base[E] = off;
    }
  }
  __syncthreads();
}

// One workgroup of 16 waves: counts, prefix sums and places in one launch.
__global__ __launch_bounds__(1024) void plan_small_kernel(const int* experts, int n, int E, int bits, int* order,
                                                          int* position, int* offsets) {
  extern __shared__ int plan_lds[];   // counts [16][E], totals [E], bases [E + 1]
  __shared__ int part[16];
  int* cnt = plan_lds;
  int* tot = cnt + 16 * E;
  int* base = tot + E;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  for (int i = t; i < 16 * E; i += 1024) cnt[i] = 0;
  __syncthreads();
  const int seg = ((n + 1023) / 1024) * 64;
  const int lo = w * seg < n ? w * seg : n, hi = lo + seg < n ? lo + seg : n;
  plan_count(experts, lo, hi, E, cnt + w * E, lane, bits);
  __syncthreads();
  for (int e = t; e < E; e += 1024) {
    int s = 0;
    for (int i = 0; i < 16; ++i) {
      const int c = cnt[i * E + e];
      cnt[i * E + e] = s;
      s += c;
    }
    tot[e] = s;
  }
  __syncthreads();
  prefix(tot, base, E, part);
  for (int i = t; i < 16 * E; i += 1024) cnt[i] += base[i % E];
  for (int e = t; e <= E; e += 1024) offsets[e] = base[e];
  for (int i = base[E] + t; i < n; i += 1024) order[i] = -1;
  __syncthreads();
  plan_place(experts, lo, hi, E, cnt + w * E, lane, bits, order, position);
}

// counts [E][kPlanSegs]
__global__ __launch_bounds__(64) void plan_count_kernel(const int* experts, int64_t n, int64_t seg, int E, int bits,
                                                        int* counts) {
  extern __shared__ int plan_lds[];
  const int lane = threadIdx.x;
  for (int e = lane; e < E; e += 64) plan_lds[e] = 0;
  __syncthreads();
  const int64_t lo = blockIdx.x * seg < n ? blockIdx.x * seg : n, hi = lo + seg < n ? lo + seg : n;
  plan_count(experts, lo, hi, E, plan_lds, lane, bits);
  __syncthreads();
  for (int e = lane; e < E; e += 64) counts[(int64_t)e * kPlanSegs + blockIdx.x] = plan_lds[e];
}

// One wave for each expert: its runs' counts become where they begin; totals [E].
__global__ __launch_bounds__(64) void plan_scan_kernel(int* counts, int* totals) {
  constexpr int Q = kPlanSegs / 256;
  int4* row = (int4*)(counts + (int64_t)blockIdx.x * kPlanSegs) + threadIdx.x * Q;
  int4 c[Q];
  int mine = 0;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    c[q] = row[q];
    mine += c[q].x + c[q].y + c[q].z + c[q].w;
  }
  int sum = mine;
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(sum, d);
    if ((int)threadIdx.x >= d) sum += o;
  }
  if (threadIdx.x == 63) totals[blockIdx.x] = sum;
  sum -= mine;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    int4 o;
    o.x = sum;
    o.y = o.x + c[q].x;
    o.z = o.y + c[q].y;
    o.w = o.z + c[q].z;
    sum = o.w + c[q].w;
    row[q] = o;
  }
}

__global__ __launch_bounds__(256) void plan_place_kernel(const int* experts, int64_t n, int64_t seg, int E, int bits,
                                                         const int* counts, const int* totals, int* order, int* position,
                                                         int* offsets) {
  extern __shared__ int plan_lds[];   // bases [E + 1], places [4][E]
  __shared__ int part[4];
  int* base = plan_lds;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  int* at = plan_lds + E + 1 + w * E;
  prefix(totals, base, E, part);
  const int s = (int)blockIdx.x * 4 + w;
  for (int e = lane; e < E; e += 64) at[e] = base[e] + counts[(int64_t)e * kPlanSegs + s];
  if (blockIdx.x == 0)
    for (int e = t; e <= E; e += 256) offsets[e] = base[e];
  for (int64_t i = base[E] + (int64_t)blockIdx.x * 256 + t; i < n; i += (int64_t)gridDim.x * 256) order[i] = -1;
  __syncthreads();
  const int64_t lo = s * seg < n ? s * seg : n, hi = lo + seg < n ? lo + seg : n;
  plan_place(experts, lo, hi, E, at, lane, bits, order, position);
}

// ---------------------------------------------------------------- the join

template <class T, int W>
__device__ __forceinline__ void load_w(float (&f)[W], const T* p, int64_t room, bool vec) {
  if (vec) {
    const Vec<T, W> v = *(const Vec<T, W>*)p;
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = (float)v.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = i < room ? (float)p[i] : 0.0f;
  }
}
template <class T, int W>
__device__ __forceinline__ void store_w(T* p, const float (&f)[W], int64_t room, bool vec) {
  if (vec) {
    Vec<T, W> v;
#pragma unroll
    for (int i = 0; i < W; ++i) v.v[i] = (T)f[i];
    *(Vec<T, W>*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < room) p[i] = (T)f[i];
  }
}

// out[t] = sum_j w[t][j] y[position[t][j]] in the order of j, in 32 bits. A thread takes 16 bytes
// of an output row. Bound by HBM: 131072 rows of 256 in 16 bits (101 MB) in 17.3 us, with their reads
// partly from the last-level cache.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void combine_kernel(const T* __restrict__ y, int64_t rows, int64_t N,
                                                      const float* __restrict__ w, const int* __restrict__ position,
                                                      int64_t Tn, int k, T* __restrict__ out) {
  constexpr int W = 16 / sizeof(T);
  const int64_t cols = cdiv(N, W), total = Tn * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / cols, n = (i - t * cols) * W;
    float acc[W] = {};
#pragma unroll 4
    for (int j = 0; j < k; ++j) {
      const int p = position[t * k + j];
      if (p < 0 || p >= rows) continue;
      const float c = w[t * k + j];
      float v[W];
      load_w<T, W>(v, y + p * N + n, N - n, VEC);
#pragma unroll
      for (int q = 0; q < W; ++q) acc[q] = __builtin_fmaf(c, v[q], acc[q]);
    }
    store_w<T, W>(out + t * N + n, acc, N - n, VEC);
  }
}

// d y[position[t][j]] = w[t][j] d out[t], d w[t][j] = d out[t] . y[position[t][j]]: one wave for
// each t reads d out[t] once. A row is written by the slot that order and position both name for it, else
// with zeros (behind the last expert's rows, or a slot taken out of position): always, and once. Bound by HBM:
// 168 MB in 38 us (131072 rows of 256), 4.4 TB/s.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void combine_backward_kernel(const T* __restrict__ y, int64_t rows, int64_t N,
                                                               const float* __restrict__ w, const int* __restrict__ position,
                                                               const int* __restrict__ order,
                                                               const T* __restrict__ dout, int64_t Tn, int k,
                                                               T* __restrict__ dy, float* __restrict__ dw) {
  constexpr int W = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < Tn; t += waves) {
    for (int j = 0; j < k; ++j) {
      const int p = position[t * k + j];
      const bool live = p >= 0 && p < rows;
      const bool own = live && dy && order[p] == t * k + j;
      const float c = w[t * k + j];
      float dot = 0.0f;
      if (live) {
        for (int64_t n = lane * W; n < N; n += 64 * W) {
          float d[W], v[W];
          load_w<T, W>(d, dout + t * N + n, N - n, VEC);
          if (dw) {
            load_w<T, W>(v, y + p * N + n, N - n, VEC);
#pragma unroll
            for (int q = 0; q < W; ++q) dot = __builtin_fmaf(d[q], v[q], dot);
          }
          if (own) {
#pragma unroll
            for (int q = 0; q < W; ++q) v[q] = c * d[q];
            store_w<T, W>(dy + p * N + n, v, N - n, VEC);
          }
        }
      }
      if (dw) {
        dot = row_sum<64>(dot);
        if (lane == 0) dw[t * k + j] = dot;
      }
    }
  }
  if (dy) {
    // 64 rows at a time are looked at by a wave, a lane each
    for (int64_t p0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 64; p0 < rows; p0 += waves * 64) {
      const int64_t mine = p0 + lane;
      const int s = mine < rows ? order[mine] : -1;
      const bool written = s >= 0 && s < Tn * k && position[s] == mine;
      for (unsigned long long rest = __ballot(mine < rows && !written); rest; rest &= rest - 1) {
        const int64_t p = p0 + __builtin_ctzll(rest);
        const float none[W] = {};
        for (int64_t n = lane * W; n < N; n += 64 * W) store_w<T, W>(dy + p * N + n, none, N - n, VEC);
      }
    }
  }
}

// ---------------------------------------------------------------- launches

int check_route(const NerfRoute* d, const char* who, bool fwd) {
  const char* why = nullptr;
  if (!d || !d->logits || !d->experts || (fwd && !d->weights)) why = "null pointer";
  else if (d->T < 1 || d->T >= (1ll << 31) || d->E < 1 || d->E > kMaxExperts || d->ld < 0)
    why = "bad size (1 to 1024 experts)";
  else if (d->k < 1 || d->k > kMaxChoices || d->k > d->E) why = "k must be 1 to 32, and at most E";
  else if (d->groups < 1 || d->groups > kMaxGroups || d->E % d->groups || d->top_groups < 1 || d->top_groups > d->groups ||
           (int64_t)d->top_groups * (d->E / d->groups) < d->k)
    why = "groups must divide E, and top_groups of them hold k experts";
  else if (d->type < NERF_F32 || d->type > NERF_F16) why = "bad type";
  return why ? fail(NERF_E_ARG, std::string(who) + ": " + why) : 0;
}

RouteArgs route_args(const NerfRoute* d) {
  RouteArgs a;
  a.logits = d->logits;
  a.ld = d->ld;
  a.T = d->T;
  a.E = d->E;
  a.k = d->k;
  a.sigmoid = d->sigmoid;
  a.groups = d->groups;
  a.top_groups = d->top_groups;
  a.group_top2 = d->group_top2;
  a.renorm = d->renorm;
  a.bias = d->bias;
  a.scale = d->scale;
  a.weights = d->weights;
  a.experts = d->experts;
  return a;
}

template <int L, int V, class T, bool VEC>
void go_route(const RouteArgs& a, const float* dw, void* dlogits, hipStream_t st) {
  constexpr int R = 256 / L;
  // (a launch has less than 2^32 threads, a call up to 2^31 rows of 16 or 64 lanes each)
  constexpr int64_t kRows = (int64_t)R << 22;
  for (int64_t t = 0; t < a.T; t += kRows) {
    RouteArgs p = a;
    p.T = a.T - t < kRows ? a.T - t : kRows;
    p.logits = (const T*)a.logits + t * a.ld;
    p.weights = a.weights ? a.weights + t * a.k : nullptr;
    p.experts = a.experts + t * a.k;
    const dim3 grid((unsigned)cdiv(p.T, R));
    if (dlogits) {
      RouteBwdArgs b{p, dw + t * a.k, (T*)dlogits + t * a.E};
      hipLaunchKernelGGL((route_backward_kernel<L, V, T, VEC>), grid, dim3(256), R * V * L * 4, st, b);
    } else {
      const size_t lds = (size_t)R * (a.groups > 1 ? a.E + 2 * a.groups : 0) * 8 + R * kMaxChoices * 4;
      hipLaunchKernelGGL((route_kernel<L, V, T, VEC>), grid, dim3(256), lds, st, p);
    }
  }
}

template <class T, bool VEC>
void go_route_e(const RouteArgs& a, const float* dw, void* dl, hipStream_t st) {
  // 16 lanes for a row waste least (E = 256, k = 8: T = 65536 in 32 us against 59 with 64 lanes, 16384 in 10
  // against 21), but with many experts and few rows the time is one row's, which more lanes shorten (T = 1021:
  // 5.8 against 5.0 us; sigmoid, bias and groups 11.3 against 7.4, at T = 4096 16.1 against 13.1, at 8192 16.9
  // against 19.5; without them 5.9 against 8.0 at 4096)
  if (a.E > 128 && a.E <= 256 && a.T <= (a.bias || a.groups > 1 ? 4096 : 2048)) go_route<64, 4, T, VEC>(a, dw, dl, st);
  else if (a.E <= 64) go_route<16, 4, T, VEC>(a, dw, dl, st);
  else if (a.E <= 128) go_route<16, 8, T, VEC>(a, dw, dl, st);
  else if (a.E <= 256) go_route<16, 16, T, VEC>(a, dw, dl, st);
  else if (a.E <= 512) go_route<64, 8, T, VEC>(a, dw, dl, st);
  else go_route<64, 16, T, VEC>(a, dw, dl, st);
}

template <class T>
void go_route_t(const RouteArgs& a, const float* dw, void* dl, hipStream_t st) {
  const bool vec = a.E % 4 == 0 && a.ld % 4 == 0 && (uintptr_t)a.logits % (4 * sizeof(T)) == 0 &&
                   (uintptr_t)dl % (4 * sizeof(T)) == 0;
  if (vec) go_route_e<T, true>(a, dw, dl, st);
  else go_route_e<T, false>(a, dw, dl, st);
}

int go_route_any(const NerfRoute* d, const float* dw, void* dl, hipStream_t st) {
  const RouteArgs a = route_args(d);
  if (d->type == NERF_F32) go_route_t<float>(a, dw, dl, st);
  else if (d->type == NERF_BF16) go_route_t<bf16>(a, dw, dl, st);
  else go_route_t<f16>(a, dw, dl, st);
  return 0;
}

int bits_of(int E) {
  int b = 0;
  while ((1 << b) < E) ++b;
  return b;
}

}  // namespace
}  // namespace nerfhip

using namespace nerfhip;

extern "C" {

int nerf_route(const NerfRoute* d, nerf_stream_t stream) {
  if (const int rc = check_route(d, "nerf_route", true)) return rc;
  go_route_any(d, nullptr, nullptr, as_stream(stream));
  return check_launch("nerf_route");
}

int nerf_route_backward(const NerfRoute* d, const float* dweights, void* dlogits, nerf_stream_t stream) {
  if (const int rc = check_route(d, "nerf_route_backward", false)) return rc;
  NERF_REQUIRE(dweights && dlogits, "nerf_route_backward: null pointer");
  go_route_any(d, dweights, dlogits, as_stream(stream));
  return check_launch("nerf_route_backward");
}

size_t nerf_expert_plan_workspace(int64_t n, int E) {
  return E < 1 || plan_is_small(n, E) ? 0 : (size_t)E * (kPlanSegs + 1) * 4;
}

int nerf_expert_plan(const int* experts, int64_t n, int E, int* order, int* position, int* offsets, void* workspace,
                     size_t workspace_bytes, nerf_stream_t stream) {
  NERF_REQUIRE(experts && order && position && offsets, "nerf_expert_plan: null pointer");
  NERF_REQUIRE(n >= 1 && n < (1ll << 31) && E >= 1 && E <= kMaxExperts, "nerf_expert_plan: bad size (1 to 1024 experts)");
  const hipStream_t st = as_stream(stream);
  const int bits = bits_of(E);
  if (plan_is_small(n, E)) {
    hipLaunchKernelGGL(plan_small_kernel, dim3(1), dim3(1024), (size_t)(18 * E + 1) * 4, st, experts, (int)n, E, bits,
                       order, position, offsets);
    return check_launch("nerf_expert_plan");
  }
  NERF_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= nerf_expert_plan_workspace(n, E),
               "nerf_expert_plan: workspace too small or unaligned");
  int* counts = (int*)workspace;
  int* totals = counts + (int64_t)E * kPlanSegs;
  const int64_t seg = cdiv(cdiv(n, kPlanSegs), 64) * 64;
  hipLaunchKernelGGL(plan_count_kernel, dim3(kPlanSegs), dim3(64), (size_t)E * 4, st, experts, n, seg, E, bits, counts);
  hipLaunchKernelGGL(plan_scan_kernel, dim3((unsigned)E), dim3(64), 0, st, counts, totals);
  hipLaunchKernelGGL(plan_place_kernel, dim3(kPlanSegs / 4), dim3(256), (size_t)(5 * E + 1) * 4, st, experts, n, seg, E, bits,
                     counts, totals, order, position, offsets);
  return check_launch("nerf_expert_plan");
}

int nerf_expert_combine(const void* y, int type, int64_t rows, int64_t N, const float* weights, const int* position,
                        int64_t T, int k, void* out, nerf_stream_t stream) {
  NERF_REQUIRE(y && weights && position && out, "nerf_expert_combine: null pointer");
  NERF_REQUIRE(rows >= 1 && N >= 1 && T >= 1 && k >= 1 && type >= NERF_F32 && type <= NERF_F16,
               "nerf_expert_combine: bad size or type");
  const hipStream_t st = as_stream(stream);
  const int size = type == NERF_F32 ? 4 : 2, W = 16 / size;
  const int64_t blocks = cdiv(T * cdiv(N, W), 256);
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536)), block(256);
  const bool vec = N % W == 0 && ((uintptr_t)y | (uintptr_t)out) % 16 == 0;
#define NERF_JOIN(TT)                                                                                               \
  do {                                                                                                              \
    auto* kern = vec ? combine_kernel<TT, true> : combine_kernel<TT, false>;                                        \
    hipLaunchKernelGGL(kern, grid, block, 0, st, (const TT*)y, rows, N, weights, position, T, k, (TT*)out);         \
  } while (0)
  if (type == NERF_F32) NERF_JOIN(float);
  else if (type == NERF_BF16) NERF_JOIN(bf16);
  else NERF_JOIN(f16);
#undef NERF_JOIN
  return check_launch("nerf_expert_combine");
}

int nerf_expert_combine_backward(const void* y, int type, int64_t rows, int64_t N, const float* weights,
                                 const int* position, const int* order, const void* dout, int64_t T, int k, void* dy,
                                 float* dweights, nerf_stream_t stream) {
  NERF_REQUIRE(y && weights && position && order && dout && (dy || dweights), "nerf_expert_combine_backward: null pointer");
  NERF_REQUIRE(rows >= 1 && N >= 1 && T >= 1 && k >= 1 && type >= NERF_F32 && type <= NERF_F16,
               "nerf_expert_combine_backward: bad size or type");
  const hipStream_t st = as_stream(stream);
  const int W = type == NERF_F32 ? 4 : 8;
  const int64_t most = T > rows ? T : rows, blocks = cdiv(most, 4);
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536)), block(256);
  const bool vec = N % W == 0 && ((uintptr_t)y | (uintptr_t)dout | (uintptr_t)dy) % 16 == 0;
#define NERF_JOIN(TT)                                                                                              \
  do {                                                                                                             \
    auto* kern = vec ? combine_backward_kernel<TT, true> : combine_backward_kernel<TT, false>;                     \
    hipLaunchKernelGGL(kern, grid, block, 0, st, (const TT*)y, rows, N, weights, position, order, (const TT*)dout, \
                       T, k, (TT*)dy, dweights);                                                                   \
  } while (0)
  if (type == NERF_F32) NERF_JOIN(float);
  else if (type == NERF_BF16) NERF_JOIN(bf16);
  else NERF_JOIN(f16);
#undef NERF_JOIN
  return check_launch("nerf_expert_combine_backward");
}

}  // extern "C"
