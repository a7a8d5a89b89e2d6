// Which experts a row goes to, and with which weights.
//
//   s = softmax(l) or 1 / (1 + exp(-l)) over a row's logits l;   c = l, or s + b with a bias b
//   with groups: of each group the best one or two of s (of s + b), added up; the best `top_groups` groups stay
//   the k largest c, ties to the lowest index;   w_j = scale s_j, or scale s_j / sum_i s_i
//
//   backward, g = scale dL/dw:  s_e (g_e - sum_j g_j s_j) for softmax (g_e = 0 where e is not chosen), g_e s_e (1 - s_e) for the logistic;
//   divided by the sum, p = w / scale:  p_e (g_e - sum_j g_j p_j), times (1 - s_e) for the logistic; 0 where e is not chosen
//
// A team of lanes has a row, NV neighbouring experts a lane, in registers; lanes and slots ascend with the experts, so that of equal
// values the first lane's first slot is the lowest. k rounds take the largest key each. An expert whose logit is -inf is never chosen:
// where fewer are left than k, the others are -1 with weight 0.
//
// Ranks are those of the exact scores. Without a bias logits are compared as they are. Scores in 32 bits are off by less than 2^-18 of the
// row's largest (the argument's rounding, exp, the sum, the quotient: 1e-6) and their sum with the bias by 2^-23 of itself: where two that were
// taken one behind the other, or the last one and the next, are nearer than twice that, the row is done again in 64 bits.
#include "dense.cuh"

namespace apt {

constexpr int kRouteThreads = 128;

struct RouteCall {
  const void* logits;
  const float* bias;
  int64_t rows;
  int experts, k, groups, per, top_groups, best;      // per: experts of a group
  int group_lanes, team_lanes;                        // logarithms
  int sigmoid, renorm, whole;                         // whole: a lane's experts are there, all or none, and may be read in slices
  float scale;
  int64_t* chosen;
  float* weights;
  const float* grad;
  void* grad_logits;
};

// Numbers as unsigned ones of the same order; 0: not to be had.
__device__ __forceinline__ uint32_t rank_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);      // -0 is 0
  return v != v ? 0xffffffffu : v == -INFINITY ? 0u : u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_of(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return v != v ? ~0ull : v == -INFINITY ? 0ull : u ^ ((int64_t)u < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float number_of(uint32_t r) { return __uint_as_float(r ^ (r >> 31 ? 0x80000000u : 0xffffffffu)); }
template <typename F> struct RankOf { using type = uint32_t; };
template <> struct RankOf<double> { using type = unsigned long long; };

template <typename V>
__device__ __forceinline__ V team_max(V v, int lanes) {
  for (int o = 0; o < lanes; ++o) {
    const V w = __shfl_xor_sync(0xffffffffu, v, 1 << o);
    v = v < w ? w : v;
  }
  return v;
}
template <typename V>
__device__ __forceinline__ V team_sum(V v, int lanes) {
  for (int o = 0; o < lanes; ++o) v += __shfl_xor_sync(0xffffffffu, v, 1 << o);
  return v;
}

struct Team {
  int lane, first, lanes;      // within the team, the team's first in the warp, logarithm of their number
  __device__ __forceinline__ unsigned votes(bool v) const {
    const unsigned all = __ballot_sync(0xffffffffu, v) >> first;
    return lanes == 5 ? all : all & ((1u << (1 << lanes)) - 1);
  }
};

// log(1 / (1 + exp(-z)))
__device__ __forceinline__ float log_logistic(float z) { return fminf(z, 0.0f) - log1pf(expf(-fabsf(z))); }

// The rounds. c: what experts are ranked by, v: what groups are by. Leaves the team's picks; true where two values were too near one another for 32
// bits: `slack`, and a share of the values themselves. (v is looked at closely only where two of them are added up.)
template <typename F, int NV>
__device__ __forceinline__ bool choose(const RouteCall& r, const Team& team, const F (&c)[NV], const F (&v)[NV], F slack, int* picks, bool write) {
  using K = typename RankOf<F>::type;
  constexpr bool kShort = sizeof(F) == 4;
  const int group = team.lane >> r.group_lanes, base = group * r.per + (team.lane & ((1 << r.group_lanes) - 1)) * NV;
  const auto too_near = [](F a, F b, F slack) { return !(a - b >= slack + (F)0x1p-22 * (a < 0 ? -a : a)); };
  bool near = false, kept = true;
  if (r.groups > 1) {
    K one = 0, two = 0;
    F first = 0, second = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const K k = rank_of(v[i]);
      if (k > one) two = one, second = first, one = k, first = v[i];
      else if (k > two) two = k, second = v[i];
    }
    for (int o = 0; o < r.group_lanes; ++o) {
      const K a = __shfl_xor_sync(0xffffffffu, one, 1 << o), b = __shfl_xor_sync(0xffffffffu, two, 1 << o);
      const F x = __shfl_xor_sync(0xffffffffu, first, 1 << o), y = __shfl_xor_sync(0xffffffffu, second, 1 << o);
      if (a > one) {
        const bool mine = one > b;
        two = mine ? one : b, second = mine ? first : y, one = a, first = x;
      } else if (a > two) {
        two = a, second = x;
      }
    }
    const F value = r.best == 2 && two ? first + second : first;
    K key = group < r.groups && one ? rank_of(value) : 0;
    F last = 0;
    kept = false;
    for (int t = 0; t < r.top_groups; ++t) {
      const K top = team_max(key, r.team_lanes);
      const unsigned who = team.votes(key == top && top);
      const int owner = who ? __ffs(who) - 1 : 0;
      last = __shfl_sync(0xffffffffu, value, team.first + owner);
      if (who && owner >> r.group_lanes == group) kept = true, key = 0;
    }
    if (kShort && r.best == 2) {
      const K top = team_max(key, r.team_lanes);
      const unsigned who = team.votes(key == top && top);
      const F next = __shfl_sync(0xffffffffu, value, team.first + (who ? __ffs(who) - 1 : 0));
      near = who && too_near(last, next, 2 * slack);
    }
  }
  K key[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) key[i] = kept ? rank_of(c[i]) : 0;
  F last = 0;
  const int rounds = r.k + (kShort && r.bias ? 1 : 0);      // one more for what the last pick is compared with
  for (int j = 0; j < rounds; ++j) {
    K best = 0;
    int slot = 0;
    F value = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (key[i] > best) best = key[i], slot = i, value = c[i];
    const K top = team_max(best, r.team_lanes);
    const unsigned who = team.votes(best == top && top);
    const int owner = who ? __ffs(who) - 1 : 0;
    const int expert = __shfl_sync(0xffffffffu, base + slot, team.first + owner);
    if (kShort && r.bias) {
      value = __shfl_sync(0xffffffffu, value, team.first + owner);
      if (j && who) near |= too_near(last, value, slack);
      last = value;
    }
    if (j < r.k && write && team.lane == 0) picks[j] = who ? expert : -1;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (who && team.lane == owner && i == slot) key[i] = 0;
  }
  return near;
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
  for (int i = 0; i < NV; ++i) s += expf(z[i] - m);
  *top = m, *sum = team_sum(s, lanes);
}

template <typename T, int NV>
__global__ void __launch_bounds__(kRouteThreads) k_route(const __grid_constant__ RouteCall r) {
  wait_for_previous();
  extern __shared__ int picks_of_all[];
  Team team;
  team.lanes = r.team_lanes, team.lane = threadIdx.x & ((1 << r.team_lanes) - 1), team.first = (threadIdx.x & 31) - team.lane;
  const int number = threadIdx.x >> r.team_lanes;
  const int64_t row = (int64_t)blockIdx.x * (kRouteThreads >> r.team_lanes) + number;
  const bool alive = row < r.rows;
  int* const picks = picks_of_all + number * r.k;
  const T* const from = (const T*)r.logits + (alive ? row : 0) * r.experts;
  const int group = team.lane >> r.group_lanes, base = group * r.per + (team.lane & ((1 << r.group_lanes) - 1)) * NV;
  const int end = alive && group < r.groups ? (group + 1) * r.per : 0;

  float z[NV], top = 0.0f, sum = 1.0f;
  load_logits<T, NV>(from, base, end, r.whole, z);
  if (!r.sigmoid && (r.bias || !r.renorm || (r.groups > 1 && r.best == 2))) row_softmax(z, r.team_lanes, &top, &sum);
  bool near;
  if (r.bias || (r.groups > 1 && r.best == 2)) {
    float s[NV], c[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool there = z[i] != -INFINITY;
      s[i] = there ? (r.sigmoid ? 1.0f / (1.0f + expf(-z[i])) : expf(z[i] - top) / sum) : -INFINITY;
      if (r.bias && there) s[i] += r.bias[base + i];
      c[i] = r.bias ? s[i] : z[i];
    }
    // no score is larger than one, and none of a softmax than that of the largest logit
    near = choose<float, NV>(r, team, c, s, 0x1p-17f * (r.sigmoid ? 1.0f : 1.0f / sum), picks, true);
  } else {
    near = choose<float, NV>(r, team, z, z, 0.0f, picks, true);
  }
  if (__any_sync(0xffffffffu, near)) {
    double s[NV], c[NV], total = 1.0;
    if (!r.sigmoid) {
      total = 0.0;
#pragma unroll
      for (int i = 0; i < NV; ++i) total += exp((double)z[i] - top);
      total = team_sum(total, r.team_lanes);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool there = z[i] != -INFINITY;
      s[i] = there ? (r.sigmoid ? 1.0 / (1.0 + exp(-(double)z[i])) : exp((double)z[i] - top) / total) : -INFINITY;
      if (r.bias && there) s[i] += r.bias[base + i];
      c[i] = r.bias ? s[i] : (double)z[i];
    }
    choose<double, NV>(r, team, c, s, 0.0, picks, near);
  }
  __syncwarp();

  // weights: of the picks' own logits, so that a sum of scores that are all too small for 32 bits is none of zero
  float m = -INFINITY, total = 0.0f;
  const int lanes = 1 << r.team_lanes;
  const auto logit = [&](int e) { return e >= 0 ? Elem<T>::to_f(from[e]) : -INFINITY; };
  if (r.renorm) {
    for (int j = team.lane; j < r.k; j += lanes) {
      const float v = logit(picks[j]);
      m = fmaxf(m, r.sigmoid ? log_logistic(v) : v);
    }
    for (int o = 0; o < r.team_lanes; ++o) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1 << o));
    for (int j = team.lane; j < r.k; j += lanes) {
      const float v = logit(picks[j]);
      if (picks[j] >= 0) total += expf((r.sigmoid ? log_logistic(v) : v) - m);
    }
    total = team_sum(total, r.team_lanes) + (sum - sum);      // a row's scores that are NaN (a bias ranked them then) stay so
  }
  for (int j = team.lane; j < r.k; j += lanes) {
    const int e = picks[j];
    const float v = logit(e);
    float w = 0.0f;
    if (e >= 0) {
      if (r.renorm) w = expf((r.sigmoid ? log_logistic(v) : v) - m) / total;
      else w = r.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top) / sum;
    }
    if (alive) r.chosen[row * r.k + j] = e, r.weights[row * r.k + j] = r.scale * w;
  }
}

template <typename T, int NV>
__global__ void __launch_bounds__(kRouteThreads) k_route_backward(const __grid_constant__ RouteCall r) {
  wait_for_previous();
  extern __shared__ int shared[];
  const int lane = threadIdx.x & ((1 << r.team_lanes) - 1), lanes = 1 << r.team_lanes, number = threadIdx.x >> r.team_lanes, teams = kRouteThreads >> r.team_lanes;
  const int64_t row = (int64_t)blockIdx.x * teams + number;
  const bool alive = row < r.rows;
  int* const pick = shared + number * r.k;
  float* const part = (float*)shared + teams * r.k + number * r.k;            // p (or s) of a pick, then its gradient
  float* const slots = (float*)shared + 2 * teams * r.k + threadIdx.x;        // this lane's experts, kRouteThreads apart
  const T* const from = (const T*)r.logits + (alive ? row : 0) * r.experts;
  const bool dense = !r.sigmoid && !r.renorm;      // gradients for experts that were not chosen too
  float z[NV], top = 0.0f, sum = 1.0f;
  if (dense) {
    load_logits<T, NV>(from, lane * NV, alive ? r.experts : 0, r.whole, z);
    row_softmax(z, r.team_lanes, &top, &sum);
  }
  const auto grad = [&](int j) { return r.scale * r.grad[row * r.k + j]; };
  float m = -INFINITY;
  for (int j = lane; j < r.k; j += lanes) {
    const int64_t given = alive ? r.chosen[row * r.k + j] : -1;
    const int e = given >= 0 && given < r.experts ? (int)given : -1;
    const float v = e >= 0 ? Elem<T>::to_f(from[e]) : -INFINITY, t = r.sigmoid ? log_logistic(v) : v;
    pick[j] = e;
    part[j] = r.renorm ? t : r.sigmoid ? 1.0f / (1.0f + expf(-v)) : expf(v - top) / sum;
    if (e >= 0) m = fmaxf(m, t);
  }
  float dot = 0.0f;
  if (r.renorm) {
    for (int o = 0; o < r.team_lanes; ++o) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1 << o));
    float total = 0.0f;
    for (int j = lane; j < r.k; j += lanes) total += part[j] = pick[j] >= 0 ? expf(part[j] - m) : 0.0f;
    total = team_sum(total, r.team_lanes);
    for (int j = lane; j < r.k; j += lanes)
      if (pick[j] >= 0) part[j] /= total, dot += part[j] * grad(j);
  } else if (dense) {
    for (int j = lane; j < r.k; j += lanes)
      if (pick[j] >= 0) dot += part[j] * grad(j);
  }
  dot = team_sum(dot, r.team_lanes);
  for (int j = lane; j < r.k; j += lanes) {
    if (pick[j] < 0) continue;
    const float g = grad(j);
    if (dense) {
      part[j] = g;
    } else {
      // 1 - s without a difference of two near ones
      const float rest = r.sigmoid ? 1.0f / (1.0f + expf(Elem<T>::to_f(from[pick[j]]))) : 1.0f;
      part[j] = part[j] * rest * (r.renorm ? g - dot : g);
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < NV; ++i) slots[i * kRouteThreads] = 0.0f;
  for (int j = 0; j < r.k; ++j) {
    const int e = pick[j];
    if (e >= 0 && e / NV == lane) slots[e % NV * kRouteThreads] += part[j];
  }
  if (!alive) return;
  T* const to = (T*)r.grad_logits + row * r.experts + lane * NV;
  float out[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    out[i] = slots[i * kRouteThreads];
    if (dense) out[i] = z[i] == -INFINITY ? 0.0f : expf(z[i] - top) / sum * (out[i] - dot);
  }
  if (r.whole) {
    constexpr int VE = 16 / (int)sizeof(T) < NV ? 16 / (int)sizeof(T) : NV;
    if (lane * NV < r.experts) {
#pragma unroll
      for (int i = 0; i < NV; i += VE) {
        float v[VE];
#pragma unroll
        for (int q = 0; q < VE; ++q) v[q] = out[i + q];
        store_all<T, VE>(to + i, v);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane * NV + i < r.experts) to[i] = Elem<T>::from_f(out[i]);
  }
}

// ---- host side -----------------------------------------------------------------------
// Experts a lane and lanes: the fewest experts with which the groups, each in lanes of its own, a power of two of them, fit a warp. Eight
// at least: a round costs the team its exchanges, whatever a lane holds.
static int route_plan(RouteCall* r) {
  int nv = 8;
  for (;; nv *= 2) {
    r->group_lanes = 0;
    while ((nv << r->group_lanes) < r->per) ++r->group_lanes;
    r->team_lanes = r->group_lanes;
    while ((1 << (r->team_lanes - r->group_lanes)) < r->groups) ++r->team_lanes;
    if (r->team_lanes <= 5) return nv;
  }
}

template <typename T, int NV>
static int launch_route(RouteCall r, bool backward, cudaStream_t s) {
  const int teams = kRouteThreads >> r.team_lanes;
  const int64_t blocks = ceil_div(r.rows, teams);
  APT_CHECK_ARG(blocks < 1ll << 31, "route_experts: %lld rows are too many", (long long)r.rows);
  const size_t picks = (size_t)teams * r.k * 4;
  if (backward)
    APT_FOLLOW((k_route_backward<T, NV>), blocks, kRouteThreads, 2 * picks + NV * kRouteThreads * 4, s, r);
  else
    APT_FOLLOW((k_route<T, NV>), blocks, kRouteThreads, picks, s, r);
  return APT_OK;
}
template <typename T>
static int route(RouteCall r, bool backward, cudaStream_t s) {
  const int nv = route_plan(&r);
  r.whole = r.per % nv == 0 && r.experts * sizeof(T) % 16 == 0 && ((uintptr_t)r.logits | (uintptr_t)r.grad_logits) % 16 == 0;
  if (nv == 8) return launch_route<T, 8>(r, backward, s);
  if (nv == 16) return launch_route<T, 16>(r, backward, s);
  if (nv == 32) return launch_route<T, 32>(r, backward, s);
  return launch_route<T, 64>(r, backward, s);
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
  r.groups = grouped ? (int)groups : 1, r.per = grouped ? (int)(experts / groups) : (int)experts, r.top_groups = (int)top_groups, r.best = group_best;
  r.sigmoid = score == APT_SCORE_SIGMOID, r.renorm = renormalize != 0, r.scale = scale, r.chosen = chosen, r.weights = weights;
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == APT_F32) return route<float>(r, false, s);
  if (dtype == APT_BF16) return route<__nv_bfloat16>(r, false, s);
  return route<__half>(r, false, s);
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
  if (dtype == APT_F32) return route<float>(r, true, s);
  if (dtype == APT_BF16) return route<__nv_bfloat16>(r, true, s);
  return route<__half>(r, true, s);
}
