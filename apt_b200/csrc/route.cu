// Which experts a row goes to, and with which weights.
//
//   s = softmax(l) or 1 / (1 + exp(-l)) over a row's logits l;   c = l, or s + b with a bias b
//   with groups: of each group the best one or two of s (of s + b), added up; the best `top_groups` groups stay
//   the k largest c, ties to the lowest index;   w_j = scale s_j, or scale s_j / sum_i s_i
//
//   backward, g = scale dL/dw:  s_e (g_e - sum_j g_j s_j) for softmax (g_e = 0 where e is not chosen), g_e s_e (1 - s_e) for the logistic;
//   divided by the sum, p = w / scale:  p_e (g_e - sum_j g_j p_j), times (1 - s_e) for the logistic; 0 where e is not chosen
//
// A team of lanes has a row, NV neighbouring experts a lane, in registers; lanes and slots ascend with the experts. The k-th largest of the
// lanes' own largest (of their two largest each, where lanes are few) is a bound below which nothing is chosen: what is not below it (some ten) goes to
// shared memory, where every candidate finds its place by counting those in front of it. Where there is no room for as many (very many that are equal, or
// more wanted than there are lanes) the bound is raised by halves first. An expert whose logit is -inf is never chosen: where fewer are left than k, the
// others are -1 with weight 0.
//
// Ranks are those of the scores in 64 bits, which are taken for exact. Without a bias logits are compared as they are. In 32 bits two logistic scores differ by less than 2^-20.9 from
// what they should: s (1 - s) (2^-24 |z| + 2^-22) for the rounded argument and the exponential, and three quarters of 2^-22 s for sum and reciprocal, twice. Two
// of a softmax by less than 2^-18.4 of the row's largest: 2^-21.2 each (2^-23 |d| exp(-|d|) for the differences' rounding, 2^-22 and 2^-23 for exponential
// and product), and the sum of up to 1024 exponentials, 2^-18.9, which all scores share. Their sum with the bias is off by 2^-24 of itself. Where
// two that are taken one behind the other, or the last one and the next, are nearer than 2^-20 (2^-18 of the largest) and 2^-22 of their size, the row is
// done again in 64 bits, by a warp for itself (route_again): of rows over 256 experts one in two hundred. Not where both have the same logit and the same bias,
// and so the same score: with a bias of zeros and logits of 16 bits that are two rows in five (67584 over 256: 266 us with them, 72 without). The same goes
// for the last group that stays and the first that does not, by their best with a bias; by their best two the bound is twice that of a score, and that of the
// roundings, which are those of the two and not of what they come to. Where half of the logistics are next to 0 or 1 (logits of deviation 6, biases of zeros)
// most rows are near: 387 us, 485 in groups.
#include <algorithm>

#include "dense.cuh"

namespace apt {

constexpr int kRouteThreads = 128, kRouteFound = APT_ROUTE_MAX_CHOSEN + 2;

struct RouteCall {
  const void* logits;
  const float* bias;
  int64_t rows;
  int experts, k, groups, per, top_groups, best;      // per: experts of a group
  int group_lanes, team_lanes;                        // logarithms
  int sigmoid, renorm;
  int whole_bias;
  int whole;                                          // a lane's experts are there, all or none, and may be read in slices
  int found;                                          // places for candidates
  float scale;
  int64_t* chosen;
  float* weights;
  const float* grad;
  void* grad_logits;
};

// Numbers as unsigned ones of the same order; 0: not to be had. NaN is above all others.
__device__ __forceinline__ uint32_t rank_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);      // -0 is 0
  return v != v ? 0xfffffffeu : v == -INFINITY ? 0u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t r) { return __uint_as_float(r ^ (r >> 31 ? 0x80000000u : 0xffffffffu)); }

template <typename V>
__device__ __forceinline__ V team_sum(V v, int lanes) {
  for (int o = 0; o < lanes; ++o) v += __shfl_xor_sync(0xffffffffu, v, 1 << o);
  return v;
}
__device__ __forceinline__ float team_most(float v, int lanes) {
  for (int o = 0; o < lanes; ++o) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1 << o));
  return v;
}
__device__ __forceinline__ uint32_t team_most(uint32_t v, int lanes) {
  if (lanes == 5) return __reduce_max_sync(0xffffffffu, v);
  for (int o = 0; o < lanes; ++o) v = max(v, __shfl_xor_sync(0xffffffffu, v, 1 << o));
  return v;
}
__device__ __forceinline__ uint32_t team_least(uint32_t v, int lanes) { return ~team_most(~v, lanes); }

struct Team {
  int lane, first, lanes;      // within the team, the team's first in the warp, logarithm of their number
  __device__ __forceinline__ unsigned votes(bool v) const {
    const unsigned all = __ballot_sync(0xffffffffu, v) >> first;
    return lanes == 5 ? all : all & ((1u << (1 << lanes)) - 1);
  }
};

// exp(z), off by two units in the last place and |z| more for its rounded argument; quotients: two units.
__device__ __forceinline__ float exp_short(float z) { return exp2_short(1.4426950408889634f * z); }
// log(1 / (1 + exp(-z)))
__device__ __forceinline__ float log_logistic(float z) { return fminf(z, 0.0f) - log1pf(expf(-fabsf(z))); }
__device__ __forceinline__ bool too_near(float a, float b, float slack) { return !(a - b >= slack + 0x1p-22f * fabsf(a)); }

// Whether the lane's group is one of those that stay: of all groups' values, the same in all lanes of a group. EXACT: values are scores in 32 bits, and
// near: the last that stays and the first that does not are too near one another for those. last: the value of the first of the two.
template <int NV, bool EXACT>
__device__ __forceinline__ bool group_stays(const RouteCall& r, const Team& team, const float (&v)[NV], float slack, bool* near, float* last) {
  const int group = team.lane >> r.group_lanes;
  uint32_t one = 0, two = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t k = rank_of(v[i]);
    two = max(two, min(one, k)), one = max(one, k);
  }
  for (int o = 0; o < r.group_lanes; ++o) {
    const uint32_t a = __shfl_xor_sync(0xffffffffu, one, 1 << o), b = __shfl_xor_sync(0xffffffffu, two, 1 << o);
    two = max(min(one, a), max(two, b)), one = max(one, a);
  }
  const uint32_t key = group >= r.groups ? 0 : r.best == 2 && two ? rank_of(number_of(one) + number_of(two)) : one;
  int above = 0;
  for (int g = 0; g < r.groups; ++g) {
    const uint32_t other = __shfl_sync(0xffffffffu, key, team.first + (g << r.group_lanes));
    above += other > key || (other == key && g < group);
  }
  const bool stays = above < r.top_groups;
  if constexpr (EXACT) {
    const uint32_t a = team_least(stays && group < r.groups ? key : 0xffffffffu, r.team_lanes), b = team_most(stays ? 0u : key, r.team_lanes);
    *last = number_of(a);
    if (r.best == 1) {
      *near = b && too_near(number_of(a), number_of(b), slack);
    } else {
      // Two scores and their sum are rounded by 2^-24 of themselves each, also where biases take the two away from each other: 2^-23 (|one| + |two|) a group,
      // of the largest of all. As bits these numbers have their order, and one that is none is above all, which nothing is far enough from.
      const float size = group < r.groups && key ? fabsf(number_of(one)) + (two ? fabsf(number_of(two)) : 0.0f) : 0.0f;
      const float most = __uint_as_float(team_most(__float_as_uint(size), r.team_lanes));
      *near = b && !(number_of(a) - number_of(b) >= 2.0f * slack + 0x1p-22f * most);
    }
  }
  return stays;
}

// The sum of the numbers of the team's lanes below, and of all, bit by bit; numbers to 2^BITS - 1.
template <int BITS>
__device__ __forceinline__ int lanes_below(const Team& team, int own, int* all) {
  int below = 0, count = 0;
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const unsigned who = team.votes(own >> b & 1);
    below += __popc(who & ((1u << team.lane) - 1)) << b, count += __popc(who) << b;
  }
  *all = count;
  return below;
}

// The bound raised, by halves, until no more keys are not below it than there are places for, and `wanted` still are. Where that many are equal, those
// behind the first ones that are wanted go below it.
template <int NV, int BITS>
__device__ __forceinline__ uint32_t raise_bound(const Team& team, uint32_t (&key)[NV], uint32_t low, bool over, int wanted) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) most = max(most, key[i]);
  uint32_t high = team_most(most, team.lanes) + 1;
  const uint32_t least = team_least(most ? most : high, team.lanes);
  const int have = __popc(team.votes(most != 0));
  if (over && have >= wanted) low = max(low, least);
  int above = 0;      // keys that are not below `high`
  while (__any_sync(0xffffffffu, over && high - low > 1)) {
    const uint32_t middle = low + (high - low) / 2;
    int own = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) own += key[i] >= middle;
    const int count = team_sum(own, team.lanes);
    if (over && high - low > 1) {
      if (count >= wanted) low = middle, over = count > kRouteFound;
      else high = middle, above = count;
    }
  }
  if (__any_sync(0xffffffffu, over)) {
    int own = 0, all;
#pragma unroll
    for (int i = 0; i < NV; ++i) own += key[i] == low;
    int at = above + lanes_below<BITS>(team, own, &all);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (over && key[i] == low && at++ >= wanted) --key[i];
  }
  return low;
}

// The largest keys, largest first and of equal ones the lowest expert's, to best[0 .. wanted): (key, complement of the expert), 0 where there is none.
template <int NV>
__device__ __forceinline__ void take_best(const RouteCall& r, const Team& team, uint32_t (&key)[NV], uint64_t* found, uint64_t* best, int wanted) {
  const int base = (team.lane >> r.group_lanes) * r.per + (team.lane & ((1 << r.group_lanes) - 1)) * NV, lanes = 1 << r.team_lanes;
  const auto entry = [&](int i) { return (uint64_t)key[i] << 32 | (uint32_t)~(base + i); };
  uint32_t one = 0, two = 0, bound = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) two = max(two, min(one, key[i])), one = max(one, key[i]);
  if (r.team_lanes == 5) {      // (equal ones go together: the bound is lower then, and holds as well)
    for (int j = 0; j < wanted && wanted <= lanes; ++j) {
      bound = __reduce_max_sync(0xffffffffu, one);
      if (one == bound) one = 0;
    }
  } else if (r.team_lanes == 4 && wanted <= lanes) {
    int above = 0;
    for (int l = 0; l < lanes; ++l) {
      const uint32_t other = __shfl_sync(0xffffffffu, one, team.first + l);
      above += other > one || (other == one && l < team.lane);
    }
    bound = __shfl_sync(0xffffffffu, one, team.first + __ffs(team.votes(above == wanted - 1)) - 1);
  } else if (wanted <= 2 * lanes) {      // few lanes: by their two largest
    int above_one = 0, above_two = 0;
    for (int l = 0; l < lanes; ++l) {
      const uint32_t a = __shfl_sync(0xffffffffu, one, team.first + l), b = __shfl_sync(0xffffffffu, two, team.first + l);
      const bool before = l < team.lane;
      above_one += (a > one || (a == one && before)) + (b > one || (b == one && before));
      above_two += (a > two || (a == two && l <= team.lane)) + (b > two || (b == two && before));
    }
    const unsigned first = team.votes(above_one == wanted - 1), second = team.votes(above_two == wanted - 1);
    bound = __shfl_sync(0xffffffffu, first ? one : two, team.first + __ffs(first ? first : second) - 1);
  }
  bound = max(bound, 1u);
  // where a lane's candidates go
  constexpr int kBits = NV == 8 ? 4 : NV == 16 ? 5 : NV == 32 ? 6 : 7;
  int own, at, count;
  const auto tally = [&] {
    uint32_t which = 0;
#pragma unroll
    for (int i = 0; i < NV && i < 32; ++i) which |= (uint32_t)(key[i] >= bound) << i;
    own = __popc(which);
    if constexpr (NV > 32) {
#pragma unroll
      for (int i = 32; i < NV; ++i) own += key[i] >= bound;
    }
    at = lanes_below<kBits>(team, own, &count);
  };
  tally();
  if (__any_sync(0xffffffffu, count > kRouteFound)) {
    bound = raise_bound<NV, kBits>(team, key, bound, count > kRouteFound, wanted);
    tally();
  }
  if (own) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (key[i] >= bound) found[at++] = entry(i);
  }
  for (int j = team.lane; j < wanted; j += lanes) best[j] = 0;
  if (team.lane == 0) found[count] = 0;      // two are read at once
  __syncwarp();
  for (int p = team.lane; p < count; p += lanes) {
    const uint64_t me = found[p];
    int place = 0;
    for (int q = 0; q < count; q += 2) {
      const ulonglong2 two = *(const ulonglong2*)(found + q);
      place += (two.x > me) + (two.y > me);
    }
    if (place < wanted) best[place] = me;
  }
  __syncwarp();
}

// The logits of a lane's experts; -inf for those that are not there.
template <typename T, int NV>
__device__ __forceinline__ void load_logits(const T* row, int base, int end, bool whole, float (&z)[NV]) {
  constexpr int VE = 16 / (int)sizeof(T) < NV ? 16 / (int)sizeof(T) : NV;
  if (whole) {
#pragma unroll
    for (int i = 0; i < NV; i += VE) {
      if (base < end) {
        const Raw<T, VE> v = load_raw<T, VE>(row + base + i);
#pragma unroll
        for (int q = 0; q < VE; ++q) z[i + q] = v.get(q);
      } else {
#pragma unroll
        for (int q = 0; q < VE; ++q) z[i + q] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = base + i < end ? Elem<T>::to_f(row[base + i]) : -INFINITY;
  }
}
// The largest of the team's (NaN are passed over) and the sum of exp(z - largest); rows of -inf: 0 and 0.
template <int NV>
__device__ __forceinline__ void row_softmax(const float (&z)[NV], int lanes, float* top, float* sum) {
  float m = z[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) m = fmaxf(m, z[i]);
  for (int o = 0; o < lanes; ++o) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1 << o));
  m = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) s += exp_short(z[i] - m);
  *top = m, *sum = team_sum(s, lanes);
}

// Whether experts whose scores are near `score` are of different logits or biases: of a row whose last pick and the next are the same, say, whether another
// is near them. (A pick near the last one that is not the same has the row done again in any case, so that what lies above is not left out.) Or of a row
// whose groups go by their best, and the last that stays and the first that does not are near: what could make one of them the other lies as near. The
// scores made here need not be those that were ranked, bit by bit: near is wider than both their errors. top, by: of its softmax. A warp's.
template <typename T>
__device__ __noinline__ bool others_near(const RouteCall& r, const T* row, float score, float top, float by, float slack) {
  float z = 0.0f, b = 0.0f;
  bool found = false, other = false;
  for (int e = threadIdx.x % 32; e < r.experts; e += 32) {
    const float v = Elem<T>::to_f(row[e]), s = (r.sigmoid ? logistic(v) : exp_short(v - top) * by) + r.bias[e];
    if (v == -INFINITY || fabsf(s - score) >= slack + 0x1p-22f * fabsf(score)) continue;
    if (!found) found = true, z = v, b = r.bias[e];
    other |= !(v == z && r.bias[e] == b);
  }
  const unsigned who = __ballot_sync(0xffffffffu, found);
  const int first = who ? __ffs(who) - 1 : 0;
  const float one = __shfl_sync(0xffffffffu, z, first), its = __shfl_sync(0xffffffffu, b, first);
  return __any_sync(0xffffffffu, other || (found && !(z == one && b == its)));
}

// A row's picks in 64 bits, by a warp: what experts are ranked by lies in shared memory, 32 neighbours at a time. Few rows come here, and the
// last of them is what a call waits for.
template <typename T>
__device__ __noinline__ void route_again(const RouteCall& r, const T* row, double* c, uint64_t* picks) {
  const int lane = threadIdx.x % 32;
  // padding, say: all logits and biases the same, and the picks are right
  bool equal = true;
  for (int e = lane; e < r.experts; e += 32) equal &= Elem<T>::to_f(row[e]) == Elem<T>::to_f(row[0]) && (!r.bias || r.bias[e] == r.bias[0]);
  if (__all_sync(0xffffffffu, equal)) return;
  double top = 0.0;
  if (!r.sigmoid) {
    float m = -INFINITY;
    for (int e = lane; e < r.experts; e += 32) m = fmaxf(m, Elem<T>::to_f(row[e]));
    m = team_most(m, 5);
    top = m == -INFINITY ? 0.0 : (double)m;
  }
  // four at once: an exponential in 64 bits is a chain of some forty steps
  double total = 0.0;
#pragma unroll 4
  for (int e = lane; e < r.experts; e += 32) {
    const double z = (double)Elem<T>::to_f(row[e]), v = r.sigmoid ? 1.0 / (1.0 + exp(-z)) : exp(z - top);
    c[e] = v, total += v;
  }
  total = r.sigmoid ? 1.0 : team_sum(total, 5);
#pragma unroll 4
  for (int e = lane; e < r.experts; e += 32) c[e] = Elem<T>::to_f(row[e]) == -INFINITY ? -INFINITY : (r.sigmoid ? c[e] : c[e] / total) + (r.bias ? (double)r.bias[e] : 0.0);
  __syncwarp();
  // (a, its place) is in front of (b, its place)
  const auto before = [](double a, int i, double b, int j) { return b != b ? a != a && i < j : a != a || a > b || (a == b && i < j); };
  if (r.groups > 1) {
    double value = -INFINITY;
    if (lane < r.groups) {
      double second = -INFINITY;
      for (int e = lane * r.per; e < (lane + 1) * r.per; ++e) {
        const double v = c[e];
        if (before(v, 0, value, 1)) second = value, value = v;
        else if (before(v, 0, second, 1)) second = v;
      }
      if (r.best == 2 && second != -INFINITY) value += second;
    }
    int above = 0;
    for (int g = 0; g < r.groups; ++g) above += before(__shfl_sync(0xffffffffu, value, g), g, value, lane);
    const unsigned stay = __ballot_sync(0xffffffffu, lane < r.groups && above < r.top_groups);
    for (int e = lane; e < r.experts; e += 32) c[e] = !(stay >> e / r.per & 1) ? -INFINITY : r.bias ? c[e] : (double)Elem<T>::to_f(row[e]);
    __syncwarp();
  }
  for (int j = 0; j < r.k; ++j) {
    double best = -INFINITY;
    int at = r.experts;
#pragma unroll 4
    for (int e = lane; e < r.experts; e += 32)
      if (c[e] != -INFINITY && before(c[e], e, best, at)) best = c[e], at = e;
    for (int o = 16; o; o >>= 1) {
      const double b = __shfl_xor_sync(0xffffffffu, best, o);
      const int i = __shfl_xor_sync(0xffffffffu, at, o);
      if (i < r.experts && (at == r.experts || before(b, i, best, at))) best = b, at = i;
    }
    if (lane == 0) {
      picks[j] = at < r.experts ? (uint64_t)rank_of(Elem<T>::to_f(row[at])) << 32 | (uint32_t)~at : 0;
      if (at < r.experts) c[at] = -INFINITY;
    }
    __syncwarp();
  }
}

// Renormalised weights of a row whose chosen scores are all next to nothing in 32 bits, by their logarithms. One thread.
template <typename T>
__device__ __noinline__ void weights_by_logarithms(const RouteCall& r, const T* row, const uint64_t* best, float* to) {
  const auto value = [&](int j) {
    const float v = Elem<T>::to_f(row[~(uint32_t)best[j]]);
    return r.sigmoid ? log_logistic(v) : v;
  };
  float m = -INFINITY, total = 0.0f;
  for (int j = 0; j < r.k && best[j]; ++j) m = fmaxf(m, value(j));
  for (int j = 0; j < r.k && best[j]; ++j) total += expf(value(j) - m);
  for (int j = 0; j < r.k; ++j) to[j] = best[j] ? r.scale * (expf(value(j) - m) / total) : 0.0f;
}

// 67584 rows over 256 experts in eight groups, logistic with a bias, fp32: by their best 115 us, by their best two 119 (reading 69 MB: 11), without groups and
// bias 45; 151552 over 64, softmax, bf16: 37 (6). Instructions bound it: 1350 of a warp a row in groups and 570 without, 84 and 81 per cent of the issue slots;
// of the last 940 for the four rows of a warp, 88 per cent. 64 of 256: 177; rows whose logits are all the same, eight of 256: 54. EXACT: ranks are those of scores, not of the logits.
template <typename T, int NV, bool GROUPS, bool EXACT>
__global__ void __launch_bounds__(kRouteThreads) k_route(const __grid_constant__ RouteCall r) {
  wait_for_previous();
  extern __shared__ __align__(16) uint64_t room[];
  Team team;
  team.lanes = r.team_lanes, team.lane = threadIdx.x & ((1 << r.team_lanes) - 1), team.first = (threadIdx.x & 31) - team.lane;
  const int number = threadIdx.x >> r.team_lanes, teams = kRouteThreads >> r.team_lanes, lanes = 1 << r.team_lanes;
  const int64_t row = (int64_t)blockIdx.x * teams + number;
  const bool alive = row < r.rows;
  // candidates and the best of them of all teams, and a row in 64 bits a warp
  uint64_t *const found = room + number * r.found, *const best = room + teams * r.found + number * (r.k + 1);
  const T* const from = (const T*)r.logits + (alive ? row : 0) * r.experts;
  const int group = GROUPS ? team.lane >> r.group_lanes : 0, base = GROUPS ? group * r.per + (team.lane & ((1 << r.group_lanes) - 1)) * NV : team.lane * NV;
  const int end = alive && group < r.groups ? (group + 1) * r.per : 0;

  float z[NV], top = 0.0f, sum = 1.0f;
  load_logits<T, NV>(from, base, end, r.whole, z);
  if (!r.sigmoid && (EXACT || !r.renorm)) row_softmax(z, r.team_lanes, &top, &sum);
  uint32_t key[NV];
  bool again = false, equal = false, stays = true;      // equal: the groups at the border are near, or have the same best
  float slack = 0.0f, by = 1.0f, last = 0.0f;           // by: the largest score there can be, last: of the groups that stay
  if constexpr (EXACT) {
    float s[NV], b[NV];
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
      if (!r.bias) {
        b[i] = b[i + 1] = b[i + 2] = b[i + 3] = 0.0f;
      } else if (r.whole_bias) {
        const float4 v = base < end ? *(const float4*)(r.bias + base + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        b[i] = v.x, b[i + 1] = v.y, b[i + 2] = v.z, b[i + 3] = v.w;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) b[i + q] = base + i + q < end ? r.bias[base + i + q] : 0.0f;
      }
    }
    by = r.sigmoid ? 1.0f : 1.0f / sum;
    slack = r.sigmoid ? 0x1p-20f : 0x1p-18f * by;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool there = z[i] != -INFINITY;
      s[i] = there ? (r.sigmoid ? logistic(z[i]) : exp_short(z[i] - top) * by) + b[i] : -INFINITY;
    }
    if constexpr (GROUPS) {
      stays = group_stays<NV, true>(r, team, s, slack, &again, &last);
      // (by their best they may be the same, as picks may)
      if (r.best == 1) equal = again, again = false;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = stays ? rank_of(r.bias ? s[i] : z[i]) : 0;
  } else {
    if constexpr (GROUPS) stays = group_stays<NV, false>(r, team, z, 0.0f, &again, &last);
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = stays ? rank_of(z[i]) : 0;
  }
  // (one more for what the last one is compared with)
  take_best<NV>(r, team, key, found, best, r.k + (EXACT ? 1 : 0));
  if constexpr (EXACT) {
    bool open = false;
    if (r.bias) {
      // what is ranked by the same logit and bias has the same score, and is in its place; if the last one and the next are, what follows may be near both
      const auto same = [&](int e, int f) { return Elem<T>::to_f(from[e]) == Elem<T>::to_f(from[f]) && r.bias[e] == r.bias[f]; };
      for (int j = team.lane; j < r.k; j += lanes) {
        const uint64_t mine = best[j], next = best[j + 1];
        if (next && too_near(number_of((uint32_t)(mine >> 32)), number_of((uint32_t)(next >> 32)), slack)) {
          if (!same(~(uint32_t)mine, ~(uint32_t)next)) again = true;
          else open |= j == r.k - 1;
        }
      }
    }
    const unsigned redo = __ballot_sync(0xffffffffu, again && alive), ask = __ballot_sync(0xffffffffu, open && alive);
    const unsigned ask_groups = GROUPS ? __ballot_sync(0xffffffffu, equal && alive) : 0u;
    if (redo | ask | ask_groups)
      for (int first = 0; first < 32; first += lanes) {
        const unsigned team_of = (lanes == 32 ? ~0u : (1u << lanes) - 1) << first;
        const int n = (threadIdx.x / 32 * 32 + first) >> r.team_lanes;
        const T* const row = (const T*)r.logits + ((int64_t)blockIdx.x * teams + n) * r.experts;
        uint64_t* const picks = room + teams * r.found + n * (r.k + 1);
        const float s = __shfl_sync(0xffffffffu, slack, first), t = __shfl_sync(0xffffffffu, top, first), b = __shfl_sync(0xffffffffu, by, first);
        const float l = GROUPS ? __shfl_sync(0xffffffffu, last, first) : 0.0f;
        if (redo & team_of || (ask & team_of && others_near<T>(r, row, number_of((uint32_t)(picks[r.k - 1] >> 32)), t, b, s)) ||
            (ask_groups & team_of && others_near<T>(r, row, l, t, b, s)))
          route_again<T>(r, row, (double*)(room + teams * (r.found + r.k + 1)) + threadIdx.x / 32 * r.experts, picks);
      }
    __syncwarp();
  }

  // Weights: of the picks' own logits, which without a bias are what they were ranked by, the first the largest of them.
  const auto logit = [&](uint64_t pick) { return r.bias ? Elem<T>::to_f(from[~(uint32_t)pick]) : number_of((uint32_t)(pick >> 32)); };
  const float m = r.bias || !r.renorm ? top : best[0] ? logit(best[0]) : 0.0f;
  const auto score = [&](uint64_t pick) { return !pick ? 0.0f : r.sigmoid ? logistic(logit(pick)) : exp_short(logit(pick) - m); };
  float total = sum;
  if (r.renorm) {
    total = 0.0f;
    for (int j = team.lane; j < r.k; j += lanes) total += score(best[j]);
    total = team_sum(total, r.team_lanes) + (sum - sum);      // a row's scores that are NaN (a bias ranked them then) stay so
  }
  if (!alive) return;
  by = r.renorm || !r.sigmoid ? __fdividef(r.scale, total) : r.scale;
  const bool few = r.renorm && total < 1e-30f;
  for (int j = team.lane; j < r.k; j += lanes) {
    const uint64_t pick = best[j];
    r.chosen[row * r.k + j] = pick ? (int)~(uint32_t)pick : -1;
    if (!few) r.weights[row * r.k + j] = pick ? score(pick) * by : 0.0f;
  }
  if (few && team.lane == 0) weights_by_logarithms<T>(r, from, best, r.weights + row * r.k);
}

// A team of lanes has a row, which lies in shared memory: gradients of the row's picks are found by a lane each, put to their experts, and leave as
// whole rows. With softmax scores that are not renormalised every expert has a gradient, and the logits are there beside them. The same rows as
// above: 24 us (writing 69 MB: 11) and 33 (39 MB: 6).
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) k_route_backward(const __grid_constant__ RouteCall r) {
  wait_for_previous();
  extern __shared__ float rows_of_all[];
  const int lanes = 1 << r.team_lanes, lane = threadIdx.x & (lanes - 1), number = threadIdx.x >> r.team_lanes, teams = kRouteThreads >> r.team_lanes;
  const int64_t row = (int64_t)blockIdx.x * teams + number;
  const bool alive = row < r.rows, dense = !r.sigmoid && !r.renorm;
  const int width = (r.experts + 3) / 4 * 4;
  float* const g = rows_of_all + number * width;
  float* const zs = rows_of_all + (teams + number) * width;                    // dense only
  float* const part = rows_of_all + (dense ? 2 : 1) * teams * width + number * r.k;      // p (or s) of a pick, then its gradient
  int* const pick = (int*)(rows_of_all + (dense ? 2 : 1) * teams * width + teams * r.k) + number * r.k;
  const T* const from = (const T*)r.logits + (alive ? row : 0) * r.experts;
  constexpr int VE = 16 / (int)sizeof(T) < 4 ? 16 / (int)sizeof(T) : 4;

  // what the picks need is asked for in front of all that is waited for
  float m = -INFINITY;
  for (int j = lane; j < r.k; j += lanes) {
    const int64_t given = alive ? r.chosen[row * r.k + j] : -1;
    const int e = given >= 0 && given < r.experts ? (int)given : -1;
    const float v = e >= 0 ? Elem<T>::to_f(from[e]) : -INFINITY;
    pick[j] = e, part[j] = v;
    if (e >= 0) m = fmaxf(m, r.sigmoid ? log_logistic(v) : v);
  }
  float top = 0.0f, sum = 1.0f;
  if (dense) {
    float most = -INFINITY;
    if (r.whole) {
      for (int e = lane * VE; e < r.experts; e += lanes * VE) {
        const Raw<T, VE> v = load_raw<T, VE>(from + e);
#pragma unroll
        for (int q = 0; q < VE; ++q) most = fmaxf(most, v.get(q)), zs[e + q] = v.get(q), g[e + q] = 0.0f;
      }
    } else {
      for (int e = lane; e < r.experts; e += lanes) {
        const float v = Elem<T>::to_f(from[e]);
        most = fmaxf(most, v), zs[e] = v, g[e] = 0.0f;
      }
    }
    most = team_most(most, r.team_lanes);
    top = most == -INFINITY ? 0.0f : most, sum = 0.0f;
    __syncwarp();
    for (int e = lane; e < r.experts; e += lanes) {
      const float s = exp_short(zs[e] - top);
      zs[e] = s, sum += s;
    }
    sum = team_sum(sum, r.team_lanes);
  } else {
    for (int e = lane; e < width; e += lanes) g[e] = 0.0f;
  }
  const auto grad = [&](int j) { return r.scale * r.grad[row * r.k + j]; };
  float dot = 0.0f, total = 0.0f;
  if (r.renorm) {
    m = team_most(m, r.team_lanes);
    for (int j = lane; j < r.k; j += lanes) total += pick[j] >= 0 ? exp_short((r.sigmoid ? log_logistic(part[j]) : part[j]) - m) : 0.0f;
    total = team_sum(total, r.team_lanes);
  }
  const auto share = [&](int j) {
    const float v = part[j];
    return r.renorm ? __fdividef(exp_short((r.sigmoid ? log_logistic(v) : v) - m), total) : r.sigmoid ? logistic(v) : __fdividef(exp_short(v - top), sum);
  };
  if (r.renorm || dense) {
    for (int j = lane; j < r.k; j += lanes)
      if (pick[j] >= 0) dot += share(j) * grad(j);
    dot = team_sum(dot, r.team_lanes);
  }
  for (int j = lane; j < r.k; j += lanes) {
    if (pick[j] < 0) continue;
    // 1 - s without a difference of two near ones
    const float rest = r.sigmoid ? logistic(-part[j]) : 1.0f;
    part[j] = dense ? grad(j) : share(j) * rest * (r.renorm ? grad(j) - dot : grad(j));
  }
  __syncwarp();
  // one lane an expert, in the picks' order: an expert that is named twice has the sum
  for (int j = 0; j < r.k; ++j) {
    const int e = pick[j];
    if (e >= 0 && (e & (lanes - 1)) == lane) g[e] += part[j];
  }
  __syncwarp();
  if (!alive) return;
  T* const to = (T*)r.grad_logits + row * r.experts;
  const float by = dense ? 1.0f / sum : 0.0f;
  const auto out = [&](float s, float g) { return !dense ? g : s == 0.0f ? 0.0f : s * by * (g - dot); };
  if (r.whole) {
    constexpr int W = 16 / (int)sizeof(T);
    for (int e = lane * W; e < r.experts; e += lanes * W) {
      float v[W];
#pragma unroll
      for (int q = 0; q < W; q += 4) {
        const float4 d = *(const float4*)(g + e + q), s = dense ? *(const float4*)(zs + e + q) : d;
        v[q] = out(s.x, d.x), v[q + 1] = out(s.y, d.y), v[q + 2] = out(s.z, d.z), v[q + 3] = out(s.w, d.w);
      }
      store_all<T, W>(to + e, v);
    }
  } else {
    for (int e = lane; e < r.experts; e += lanes) to[e] = Elem<T>::from_f(out(dense ? zs[e] : 0.0f, g[e]));
  }
}

// ---- host side -----------------------------------------------------------------------
// Experts a lane and lanes. What a row costs whatever it holds (bound, places, weights: some 400 instructions) several rows share in a warp that has
// more experts a lane; but a bound that comes of too few of the lanes' largest is too low, and there are too many candidates. So 16 experts a lane where
// that leaves lanes enough, of the groups that stay, else eight; or the fewest with which the groups, each in lanes of its own, a power of two of them,
// fit a warp.
static int route_plan(RouteCall* r) {
  const auto lay_out = [r](int nv) {
    r->group_lanes = 0;
    while ((nv << r->group_lanes) < r->per) ++r->group_lanes;
    r->team_lanes = r->group_lanes;
    while ((1 << (r->team_lanes - r->group_lanes)) < r->groups) ++r->team_lanes;
    return r->team_lanes <= 5;
  };
  if (r->experts > 64 && lay_out(16) && (r->top_groups << r->group_lanes) >= 2 * r->k) return 16;
  int nv = 8;
  while (!lay_out(nv)) nv *= 2;
  return nv;
}

template <typename T, int NV>
static int launch_route(const RouteCall& r, cudaStream_t s) {
  const int teams = kRouteThreads >> r.team_lanes;
  const int64_t blocks = ceil_div(r.rows, teams);
  APT_CHECK_ARG(blocks < 1ll << 31, "route_experts: %lld rows are too many", (long long)r.rows);
  const bool exact = r.bias || (r.groups > 1 && r.best == 2);
  const size_t bytes = ((size_t)teams * (r.found + r.k + 1) + (exact ? kRouteThreads / 32 * r.experts : 0)) * 8;
  if (r.groups > 1) {
    if (exact) APT_FOLLOW((k_route<T, NV, true, true>), blocks, kRouteThreads, bytes, s, r);
    else APT_FOLLOW((k_route<T, NV, true, false>), blocks, kRouteThreads, bytes, s, r);
  } else if constexpr (NV < 64) {
    if (exact) APT_FOLLOW((k_route<T, NV, false, true>), blocks, kRouteThreads, bytes, s, r);
    else APT_FOLLOW((k_route<T, NV, false, false>), blocks, kRouteThreads, bytes, s, r);
  }
  return APT_OK;
}
template <typename T>
static int route(RouteCall r, cudaStream_t s) {
  const int nv = route_plan(&r);
  r.found = (std::min(r.experts, kRouteFound) + 2) / 2 * 2;
  r.whole = r.per % nv == 0 && r.experts * sizeof(T) % 16 == 0 && (uintptr_t)r.logits % 16 == 0;
  r.whole_bias = r.per % nv == 0 && (uintptr_t)r.bias % 16 == 0;
  if (nv == 8) return launch_route<T, 8>(r, s);
  if (nv == 16) return launch_route<T, 16>(r, s);
  if (nv == 32) return launch_route<T, 32>(r, s);
  return launch_route<T, 64>(r, s);
}
// Lanes for a row's picks, and for 64 of its experts each at the most: few, so that many rows are on their way at once.
template <typename T>
static int route_backward(RouteCall r, cudaStream_t s) {
  const bool dense = !r.sigmoid && !r.renorm;
  r.team_lanes = 2;
  while (r.team_lanes < 5 && ((1 << r.team_lanes) < r.k || (1 << r.team_lanes) * (dense ? 8 : 64) < r.experts)) ++r.team_lanes;
  r.whole = r.experts * sizeof(T) % 16 == 0 && ((uintptr_t)r.logits | (uintptr_t)r.grad_logits) % 16 == 0;
  const int teams = kRouteThreads >> r.team_lanes;
  const int64_t blocks = ceil_div(r.rows, teams);
  APT_CHECK_ARG(blocks < 1ll << 31, "route_experts_backward: %lld rows are too many", (long long)r.rows);
  APT_FOLLOW((k_route_backward<T>), blocks, kRouteThreads, (size_t)teams * ((dense ? 2 : 1) * align_up(r.experts, 4) + 2 * r.k) * 4, s, r);
  return APT_OK;
}
static int route_check(const char* who, int dtype, int64_t rows, int64_t experts, int64_t k, int score) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(score == APT_SCORE_SOFTMAX || score == APT_SCORE_SIGMOID, "%s: unknown score %d", who, score);
  APT_CHECK_ARG(rows >= 0 && experts >= 1 && experts <= APT_ROUTE_MAX_EXPERTS, "%s: %lld rows over %lld experts (1 to %d are possible)", who, (long long)rows,
                (long long)experts, APT_ROUTE_MAX_EXPERTS);
  APT_CHECK_ARG(k >= 1 && k <= APT_ROUTE_MAX_CHOSEN && k <= experts, "%s: %lld of %lld experts (1 to %d are possible)", who, (long long)k, (long long)experts,
                APT_ROUTE_MAX_CHOSEN);
  return APT_OK;
}

}  // namespace apt

extern "C" int apt_route_experts(int dtype, const void* logits, int64_t rows, int64_t experts, int64_t k, int score, const float* bias, int64_t groups,
                                 int64_t top_groups, int group_best, int renormalize, float scale, int64_t* chosen, float* weights, void* stream) {
  using namespace apt;
  if (const int e = route_check("apt_route_experts", dtype, rows, experts, k, score)) return e;
  APT_CHECK_ARG(groups >= 1 && groups <= 32 && experts % groups == 0, "apt_route_experts: %lld groups of %lld experts (1 to 32 of the same size are possible)",
                (long long)groups, (long long)experts);
  APT_CHECK_ARG(top_groups >= 1 && top_groups <= groups && k <= experts / groups * top_groups, "apt_route_experts: %lld experts of %lld of %lld groups",
                (long long)k, (long long)top_groups, (long long)groups);
  APT_CHECK_ARG(group_best == 1 || group_best == 2, "apt_route_experts: groups go by their best or their best two, not %d", group_best);
  APT_CHECK_ARG(rows == 0 || (logits && chosen && weights), "apt_route_experts: null buffer");
  if (rows == 0) return APT_OK;
  RouteCall r = {};
  r.logits = logits, r.bias = bias, r.rows = rows, r.experts = (int)experts, r.k = (int)k;
  // groups that all stay are none
  const bool grouped = groups > 1 && top_groups < groups;
  r.groups = grouped ? (int)groups : 1, r.per = grouped ? (int)(experts / groups) : (int)experts, r.top_groups = grouped ? (int)top_groups : 1, r.best = group_best;
  r.sigmoid = score == APT_SCORE_SIGMOID, r.renorm = renormalize != 0, r.scale = scale, r.chosen = chosen, r.weights = weights;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == APT_F32) return route<float>(r, s);
  if (dtype == APT_BF16) return route<__nv_bfloat16>(r, s);
  return route<__half>(r, s);
}

extern "C" int apt_route_experts_backward(int dtype, const void* logits, int64_t rows, int64_t experts, int64_t k, int score, int renormalize, float scale,
                                          const int64_t* chosen, const float* grad_weights, void* grad_logits, void* stream) {
  using namespace apt;
  if (const int e = route_check("apt_route_experts_backward", dtype, rows, experts, k, score)) return e;
  APT_CHECK_ARG(rows == 0 || (logits && chosen && grad_weights && grad_logits), "apt_route_experts_backward: null buffer");
  if (rows == 0) return APT_OK;
  RouteCall r = {};
  r.logits = logits, r.rows = rows, r.experts = r.per = (int)experts, r.k = (int)k, r.groups = r.top_groups = r.best = 1;
  r.sigmoid = score == APT_SCORE_SIGMOID, r.renorm = renormalize != 0, r.scale = scale;
  r.chosen = (int64_t*)chosen, r.grad = grad_weights, r.grad_logits = grad_logits;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == APT_F32) return route_backward<float>(r, s);
  if (dtype == APT_BF16) return route_backward<__nv_bfloat16>(r, s);
  return route_backward<__half>(r, s);
}
