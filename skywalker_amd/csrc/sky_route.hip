// Routing to experts (sky_route_topk) and its gradient.  A wavefront has a row of E logits at a time, lane l the experts PER l, PER l + 1, ...
//   score    s_e = exp(x_e - max) / sum, or 1 / (1 + exp(-x_e))
//   choice   by s_e + b_e, the largest first, equal ones by number.  Both scores ascend with the logit, so without a bias and
//            without pairs of experts the choice goes by the logits themselves, exactly.  Else it is made from scores in fp32, whose error
//            has a bound; where two of those that it hangs on (neighbours among the k + 1 best, the last group that stays and the first
//            that does not) are nearer than that and not alike, the row is chosen again in fp64: one expert more or less is no
//            rounding error.  (32,768 rows of 256, 8 of 4 of 8 groups: all in fp64 96 us.)
//   weights  w_j = scale * s_j, renormalised scale * s_j / sum of the k chosen.  Renormalised, the sum over all experts drops out of
//            softmax scores, and sigmoid scores are taken relative to the largest of the chosen (their logarithms
//            are at hand), so that a row of tiny scores keeps its shares.  In fp64, for as many rows at once as the chosen fill a wavefront.
// Gradient, g_j = scale * dw_j, p_j = share of the chosen j:
//   softmax, renormalised    dx_j = p_j (g_j - sum_i g_i p_i) for the chosen, 0 elsewhere
//   softmax                  dx_e = s_e (g_e [e chosen] - sum_i g_i s_i)
//   sigmoid, renormalised    dx_j = p_j (1 - s_j) (g_j - sum_i g_i p_i)
//   sigmoid                  dx_j = g_j s_j (1 - s_j)
#include "sky_scores.h"

namespace sky {
namespace {

constexpr uint32_t MAX_EXPERTS = 1024, MAX_K = 64, MAX_GROUPS = 64;
constexpr int ROUTE_WAVES = 4;  // of a workgroup

struct RouteArgs {
  const void* logits;
  uint64_t stride;
  uint32_t rows, experts;
  sky_route_rules r;
  uint32_t* ids;
  float* weights;
  const uint32_t* ids_in;
  const float* dweights;
  void* dlogits;
  uint64_t dstride;
};

__device__ __forceinline__ uint64_t double_key(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double key_double(uint64_t v) { return __longlong_as_double((long long)(v ^ ((v >> 63) ? 1ull << 63 : ~0ull))); }
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  v = max(v, dpp0_u64<DPP_QUAD_XOR1, 0xF>(v));
  v = max(v, dpp0_u64<DPP_QUAD_XOR2, 0xF>(v));
  v = max(v, dpp0_u64<DPP_ROW_HALF_MIRROR, 0xF>(v));
  v = max(v, dpp0_u64<DPP_ROW_MIRROR, 0xF>(v));
  v = max(v, shfl_xor_u64(v, 16));
  return max(v, shfl_xor_u64(v, 32));
}
// The largest of the wavefront, in a scalar register.
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
  v = max(v, dpp0<DPP_ROW_SHR1, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_SHR2, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_SHR4, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_SHR8, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_BCAST15, 0xA>(v));
  v = max(v, dpp0<DPP_ROW_BCAST31, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ __forceinline__ bool open_expert(float x) { return x > -__builtin_inff(); }
// log(1 / (1 + exp(-x)))
__device__ __forceinline__ double log_sigmoid(double x) { return fmin(x, 0.0) - log1p(exp(-fabs(x))); }

// The choice of one row in fp64, into lanes first + j.  Keys: 0 is a closed expert, a taken one or none.
template <typename T, int PER>
__device__ __forceinline__ uint32_t choose_exactly(const T* x, const RouteArgs& a, double* staged, uint32_t first, uint32_t id) {
  const uint32_t lane = threadIdx.x & 63, E = a.experts;
  float z[PER], zmax = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    z[i] = lane * PER + i < E ? plain_score((float)x[lane * PER + i]) : -__builtin_inff();
    zmax = fmaxf(zmax, z[i]);
  }
  zmax = wave_max_f32(zmax);
  double sum = 0.0;
  if (!a.r.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += open_expert(z[i]) ? exp((double)z[i] - (double)zmax) : 0.0;
    sum = group_sum_f64<64>(sum);
  }
  uint64_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t e = lane * PER + i;
    key[i] = 0;
    if (open_expert(z[i])) {
      const double score = a.r.sigmoid ? 1.0 / (1.0 + exp(-(double)z[i])) : exp((double)z[i] - (double)zmax) / sum;
      key[i] = double_key(score + (a.r.bias ? (double)a.r.bias[e] : 0.0));
    }
  }
  if (a.r.groups > 1 && a.r.groups_kept < a.r.groups) {
    // a lane has a group: its best choice, or the sum of its two best
    const uint32_t size = E / a.r.groups;
#pragma unroll
    for (int i = 0; i < PER; ++i) staged[lane * PER + i] = __longlong_as_double((long long)key[i]);
    __builtin_amdgcn_wave_barrier();
    uint64_t mine = 0;
    if (lane < a.r.groups) {
      uint64_t best = 0, second = 0;
      for (uint32_t i = 0; i < size; ++i) {
        const uint64_t v = (uint64_t)__double_as_longlong(staged[lane * size + i]);
        second = max(second, min(best, v));
        best = max(best, v);
      }
      // a group without an open expert is worth less than any other; a lone open expert counts by itself
      mine = best;
      if (best && second && a.r.group_top2) mine = double_key(key_double(best) + key_double(second));
    }
    __builtin_amdgcn_wave_barrier();
    uint64_t stay = 0;  // bits of the groups that do
    for (uint32_t j = 0; j < a.r.groups_kept; ++j) {
      const uint64_t best = wave_max_u64(mine);
      if (!best) break;
      const uint32_t g = (uint32_t)__builtin_ctzll(__ballot(mine == best));
      stay |= 1ull << g;
      if (lane == g) mine = 0;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t e = lane * PER + i;
      if (e >= E || !(stay >> (e / size) & 1)) key[i] = 0;
    }
  }
  for (uint32_t j = 0; j < a.r.k; ++j) {
    uint64_t mine = key[0];
    uint32_t at = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > mine) {
        mine = key[i];
        at = i;
      }
    const uint64_t best = wave_max_u64(mine);
    if (!best) break;
    const uint32_t winner = (uint32_t)__builtin_ctzll(__ballot(mine == best));  // of equals the first lane, and its first, has the smallest number
    const uint32_t e = (uint32_t)__shfl((int)(lane * PER + at), (int)winner, 64);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane == winner && at == (uint32_t)i) key[i] = 0;
    if (lane == first + j) id = e;
  }
  return id;
}

// A wavefront takes rows_per_wave rows, which fill it with chosen experts: `slots` lanes (a power of two, at least k) for a row's.
template <typename T, int PER>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_kernel(RouteArgs a, uint32_t rows_per_wave, uint32_t slots) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t row0 = (blockIdx.x * ROUTE_WAVES + wave) * rows_per_wave, E = a.experts, k = a.r.k;
  __shared__ double staged_all[ROUTE_WAVES][64 * PER];
  if (row0 >= a.rows) return;
  double* const staged = staged_all[wave];
  const uint32_t rows = min(rows_per_wave, a.rows - row0);
  const bool grouped = a.r.groups > 1 && a.r.groups_kept < a.r.groups;
  const bool by_logit = !a.r.bias && !(grouped && a.r.group_top2);
  const bool full_sum = !a.r.sigmoid && !a.r.renormalise;  // the sum over all experts goes into the weights
  const uint32_t size = E / a.r.groups, lanes = size / PER;  // of a group
  // groups whose experts are whole lanes, a power of two of them, are reduced across lanes; others through LDS
  const bool whole_lanes = size % PER == 0 && (lanes & (lanes - 1)) == 0;
  float bias[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) bias[i] = a.r.bias && lane * PER + i < E ? a.r.bias[lane * PER + i] : 0.0f;
  uint32_t id = SKY_INVALID;
  double my_sum = 0.0;
  float my_max = 0.0f;
  for (uint32_t n = 0; n < rows; ++n) {
    const T* const x = (const T*)a.logits + (row0 + n) * a.stride;
    float z[PER];
    float zmax = -__builtin_inff();
    if (PER * 64 == E) {
      T v[PER];
      __builtin_memcpy(v, x + lane * PER, sizeof(v));
#pragma unroll
      for (int i = 0; i < PER; ++i) z[i] = plain_score((float)v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) z[i] = lane * PER + i < E ? plain_score((float)x[lane * PER + i]) : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) zmax = fmaxf(zmax, z[i]);
    const uint32_t first = n * slots;  // lane of the row's best
    if (!a.r.sigmoid && !(by_logit && a.r.renormalise)) zmax = key_score(wave_top(score_key(zmax)));
    if (full_sum) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += open_expert(z[i]) ? exp((double)z[i] - (double)zmax) : 0.0;
      sum = group_sum_f64<64>(sum);
      if (lane / slots == n) {
        my_sum = sum;
        my_max = zmax;
      }
    }
    uint32_t key[PER];
    float near = 0.0f;  // choices that are nearer than this may be the other way round
    if (by_logit) {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = open_expert(z[i]) ? score_key(z[i]) : 0;
    } else {
      // Scores: the exponent's product is off by 2^-24 of itself, which its size times the score bounds by 0.53, exponential, sum and
      // quotient by some 2^-22: less than 2^-20 of the largest score in all.  The sum with the bias: 2^-24.
      float s[PER], most;
      if (a.r.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; ++i) s[i] = 1.0f / (1.0f + __builtin_amdgcn_exp2f(fminf(-z[i] * 1.44269504f, 126.0f)));
        most = 1.0f;
      } else {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          s[i] = open_expert(z[i]) ? __builtin_amdgcn_exp2f((z[i] - zmax) * 1.44269504f) : 0.0f;
          sum += s[i];
        }
        most = 1.0f / wave_sum_f32(sum);
#pragma unroll
        for (int i = 0; i < PER; ++i) s[i] *= most;
      }
      float size_of_choice = 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float c = s[i] + bias[i];
        size_of_choice = fmaxf(size_of_choice, fabsf(c));
        key[i] = open_expert(z[i]) ? score_key(c) : 0;
      }
      size_of_choice = key_score(wave_top(score_key(size_of_choice)));
      near = 0x1p-18f * most + 0x1p-22f * size_of_choice;
    }
    bool exact = true;  // the choice so far
    if (grouped) {
      uint32_t best = 0, second = 0;
      uint32_t owner = lane;  // of which group this lane tells the worth, and the first lane of its own group's lanes
      if (whole_lanes) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          second = max(second, min(best, key[i]));
          best = max(best, key[i]);
        }
        for (uint32_t m = 1; m < lanes; m *= 2) {
          const uint32_t b = (uint32_t)__shfl_xor((int)best, (int)m, 64), c = (uint32_t)__shfl_xor((int)second, (int)m, 64);
          second = max(min(best, b), max(second, c));
          best = max(best, b);
        }
        owner = lane * PER < E && lane % lanes == 0 ? lane / lanes : 64;
      } else {
        uint32_t* const words = (uint32_t*)staged;
#pragma unroll
        for (int i = 0; i < PER; ++i) words[lane * PER + i] = key[i];
        __builtin_amdgcn_wave_barrier();
        if (lane < a.r.groups)
          for (uint32_t i = 0; i < size; ++i) {
            const uint32_t v = words[lane * size + i];
            second = max(second, min(best, v));
            best = max(best, v);
          }
        __builtin_amdgcn_wave_barrier();
        owner = lane < a.r.groups ? lane : 64;
      }
      uint32_t mine = best;
      if (best && second && a.r.group_top2) mine = score_key(key_score(best) + key_score(second));
      if (owner == 64) mine = 0;
      uint64_t stay = 0;
      uint32_t last = 0;
      for (uint32_t j = 0; j < a.r.groups_kept; ++j) {
        last = wave_top(mine);
        if (!last) break;
        const uint32_t l = (uint32_t)__builtin_ctzll(__ballot(mine == last)), g = (uint32_t)__builtin_amdgcn_readlane((int)owner, (int)l);
        stay |= 1ull << g;
        if (lane == l) mine = 0;
      }
      const uint32_t next = last ? wave_top(mine) : 0;
      if (!by_logit && next && !(key_score(last) - key_score(next) > 4.0f * near)) exact = false;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t e = lane * PER + i;
        if (e >= E || !(stay >> (e / size) & 1)) key[i] = 0;
      }
    }
    uint32_t before = 0, before_e = 0;
    for (uint32_t j = 0; j < k + (by_logit ? 0u : 1u) && exact; ++j) {
      uint32_t mine = key[0], at = 0;
#pragma unroll
      for (int i = 1; i < PER; ++i)
        if (key[i] > mine) {
          mine = key[i];
          at = i;
        }
      const uint32_t best = wave_top(mine);
      if (!best) break;
      const uint32_t winner = (uint32_t)__builtin_ctzll(__ballot(mine == best));  // of equals the first lane, and its first, has the smallest number
      const uint32_t e = (uint32_t)__builtin_amdgcn_readlane((int)(lane * PER + at), (int)winner);
      if (!by_logit && j && !(key_score(before) - key_score(best) > 2.0f * near))
        // alike: the same logit and bias
        exact = (float)x[e] == (float)x[before_e] && (!a.r.bias || a.r.bias[e] == a.r.bias[before_e]);
      before = best;
      before_e = e;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane == winner && at == (uint32_t)i) key[i] = 0;
      if (lane == first + j && j < k) id = e;
    }
    if (!exact) {
      if (lane / slots == n) id = SKY_INVALID;
      id = choose_exactly<T, PER>(x, a, staged, first, id);
    }
  }
  // the weights of all of the wavefront's rows: lane n * slots + j has the j-th of row n
  const uint32_t n = lane / slots, j = lane % slots;
  const bool mine = n < rows && j < k, in = mine && id != SKY_INVALID;
  const float chosen = in ? plain_score((float)((const T*)a.logits + (row0 + n) * a.stride)[id]) : 0.0f;
  double w = 0.0;
  if (a.r.renormalise) {
    // the first of the order has not got the largest score when a bias or groups decide
    const double l = !in ? 0.0 : a.r.sigmoid ? log_sigmoid(chosen) : (double)chosen;
    double most = in ? l : -__builtin_inf();
    for (uint32_t m = 1; m < slots; m *= 2) most = fmax(most, __shfl_xor(most, (int)m, 64));
    w = in ? exp(l - most) : 0.0;
    double all = w;
    for (uint32_t m = 1; m < slots; m *= 2) all += __shfl_xor(all, (int)m, 64);
    w = all > 0.0 ? w / all : 0.0;
  } else if (in) {
    w = a.r.sigmoid ? 1.0 / (1.0 + exp(-(double)chosen)) : exp((double)chosen - (double)my_max) / my_sum;
  }
  if (mine) {
    a.ids[(uint64_t)(row0 + n) * k + j] = id;
    a.weights[(uint64_t)(row0 + n) * k + j] = in ? (float)((double)a.r.scale * w) : 0.0f;
  }
}

constexpr int COUNT_THREADS = 1024;
__global__ void clear_counts_kernel(uint32_t* counts, uint32_t n) {
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) counts[i] = 0;
}
// How often each expert was chosen: counted in LDS, added to the result once per workgroup and expert.
__global__ __launch_bounds__(COUNT_THREADS) void count_experts_kernel(const uint32_t* __restrict__ ids, uint64_t n, uint32_t E,
                                                                      uint32_t* __restrict__ counts) {
  __shared__ uint32_t c[MAX_EXPERTS];
  for (uint32_t e = threadIdx.x; e < E; e += COUNT_THREADS) c[e] = 0;
  __syncthreads();
  for (uint64_t i = (uint64_t)blockIdx.x * COUNT_THREADS + threadIdx.x; i < n; i += (uint64_t)gridDim.x * COUNT_THREADS) {
    const uint32_t e = ids[i];
    if (e < E) atomicAdd(&c[e], 1u);
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < E; e += COUNT_THREADS)
    if (c[e]) atomicAdd(&counts[e], c[e]);
}

template <typename T, int PER>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_backward_kernel(RouteArgs a) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t row = blockIdx.x * ROUTE_WAVES + wave, E = a.experts, k = a.r.k;
  if (row >= a.rows) return;
  const T* const x = (const T*)a.logits + row * a.stride;
  T* const dx = (T*)a.dlogits + row * a.dstride;
  uint32_t id = SKY_INVALID;
  float g = 0.0f, xj = -__builtin_inff();
  if (lane < k) {
    id = a.ids_in[(uint64_t)row * k + lane];
    if (id < E) {
      g = a.dweights[(uint64_t)row * k + lane] * a.r.scale;
      xj = plain_score((float)x[id]);
    }
    if (!open_expert(xj)) id = SKY_INVALID;
  }
  const bool in = id != SKY_INVALID;
  if (!in) g = 0.0f;
  float zmax = -__builtin_inff(), total = 0.0f;
  float z[PER];
  const bool dense = !a.r.sigmoid && !a.r.renormalise;
  if (dense) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t e = 64 * i + lane;
      z[i] = e < E ? plain_score((float)x[e]) : -__builtin_inff();
      zmax = fmaxf(zmax, z[i]);
    }
    zmax = wave_max_f32(zmax);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      z[i] = open_expert(z[i]) ? expf(z[i] - zmax) : 0.0f;
      total += z[i];
    }
    total = wave_sum_f32(total);
  }
  // the gradient at the chosen entry of this lane (in the dense case: what is added to -s_e * sum g s)
  float d = 0.0f, mean = 0.0f;
  if (a.r.renormalise) {
    const float l = !in ? -__builtin_inff() : a.r.sigmoid ? fminf(xj, 0.0f) - log1pf(expf(-fabsf(xj))) : xj;
    const float most = wave_max_f32(l);
    float p = in ? expf(l - most) : 0.0f;
    const float all = wave_sum_f32(p);
    p = all > 0.0f ? p / all : 0.0f;
    mean = wave_sum_f32(g * p);
    d = p * (g - mean);
    if (a.r.sigmoid) d *= in ? 1.0f / (1.0f + expf(xj)) : 0.0f;
  } else if (a.r.sigmoid) {
    d = in ? g * (1.0f / (1.0f + expf(-xj))) * (1.0f / (1.0f + expf(xj))) : 0.0f;
  } else {
    d = in ? g * expf(xj - zmax) / total : 0.0f;
    mean = wave_sum_f32(d);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t e = 64 * i + lane;
    float v = dense && total > 0.0f ? -(z[i] / total) * mean : 0.0f;
    for (uint32_t j = 0; j < k; ++j) {
      const uint32_t c = (uint32_t)__shfl((int)id, (int)j, 64);
      const float add = __shfl(d, (int)j, 64);
      if (c == e) v += add;
    }
    if (e < E) dx[e] = (T)v;
  }
}

int check_route(const char* who, uint32_t rows, uint32_t experts, const sky_route_rules* r) {
  auto arg = [&](const char* what) { return fail(SKY_ERR_ARG, std::string(who) + ": " + what); };
  if (!r) return arg("rules is null");
  if (!experts) return arg("no experts");
  if (!r->k || r->k > experts) return arg("k must lie in 1 .. experts");
  if (experts > MAX_EXPERTS || r->k > MAX_K || r->groups > MAX_GROUPS)
    return fail(SKY_ERR_LIMIT, std::string(who) + ": more than 1024 experts, 64 chosen or 64 groups");
  if (!r->groups || experts % r->groups) return arg("groups must divide the experts");
  if (!r->groups_kept || r->groups_kept > r->groups) return arg("groups_kept must lie in 1 .. groups");
  if (r->k > r->groups_kept * (experts / r->groups)) return arg("the kept groups have fewer than k experts");
  if (!(r->scale - r->scale == 0.0f)) return arg("scale is not a finite number");
  SKY_TRY(check_aligned(who, "bias", r->bias, 4));
  if (rows > 0x7FFFFFFFu / (uint32_t)ROUTE_WAVES * ROUTE_WAVES) return fail(SKY_ERR_LIMIT, std::string(who) + ": too many rows");
  return SKY_OK;
}

#define SKY_ROUTE_PER(kernel, T)                                                          \
  (experts <= 64 ? launch(kernel<T, 1>)                                                   \
   : experts <= 128 ? launch(kernel<T, 2>)                                                \
   : experts <= 256 ? launch(kernel<T, 4>)                                                \
   : experts <= 512 ? launch(kernel<T, 8>)                                                \
                    : launch(kernel<T, 16>))
#define SKY_ROUTE_LAUNCH(kernel)                       \
  (dtype == SKY_F32 ? SKY_ROUTE_PER(kernel, float)     \
   : dtype == SKY_F16 ? SKY_ROUTE_PER(kernel, _Float16) \
                      : SKY_ROUTE_PER(kernel, __bf16))

}  // namespace
}  // namespace sky

using namespace sky;

extern "C" int sky_route_topk(const void* logits, int dtype, uint32_t rows, uint32_t experts, uint64_t row_stride,
                              const sky_route_rules* rules, uint32_t* ids, float* weights, uint32_t* counts, void* stream) {
  const char* const who = "sky_route_topk";
  SKY_TRY(check_rows(who, "logits", logits, dtype, rows, experts, &row_stride));
  SKY_TRY(check_route(who, rows, experts, rules));
  if (rows && (!ids || !weights)) return fail(SKY_ERR_ARG, "sky_route_topk: ids or weights is null");
  SKY_TRY(check_aligned(who, "ids", ids, 4));
  SKY_TRY(check_aligned(who, "weights", weights, 4));
  SKY_TRY(check_aligned(who, "counts", counts, 4));
  if (!rows && !counts) return SKY_OK;
  SKY_TRY(ensure_device());
  const hipStream_t st = (hipStream_t)stream;
  if (!rows) {
    hipLaunchKernelGGL(clear_counts_kernel, dim3((experts + 255) / 256), dim3(256), 0, st, counts, experts);
    return check_launch();
  }
  RouteArgs a{};
  a.logits = logits;
  a.stride = row_stride;
  a.rows = rows;
  a.experts = experts;
  a.r = *rules;
  a.ids = ids;
  a.weights = weights;
  uint32_t slots = 1;
  while (slots < rules->k) slots *= 2;
  // as many rows a wavefront as fill it with chosen experts, as long as there is a wavefront for every SIMD
  const uint32_t per_wave = std::min(64 / slots, std::max(rows / 2048u, 1u));
  const uint64_t waves = ((uint64_t)rows + per_wave - 1) / per_wave;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)((waves + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(64 * ROUTE_WAVES), 0, st, a, per_wave, slots);
  };
  SKY_ROUTE_LAUNCH(route_kernel);
  if (counts) {
    const uint64_t n = (uint64_t)rows * rules->k;
    hipLaunchKernelGGL(clear_counts_kernel, dim3((experts + 255) / 256), dim3(256), 0, st, counts, experts);
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((n + 4 * COUNT_THREADS - 1) / (4 * COUNT_THREADS), 64);
    hipLaunchKernelGGL(count_experts_kernel, dim3(blocks), dim3(COUNT_THREADS), 0, st, ids, n, experts, counts);
  }
  return check_launch();
}

extern "C" int sky_route_topk_backward(const void* logits, int dtype, uint32_t rows, uint32_t experts, uint64_t row_stride,
                                       const sky_route_rules* rules, const uint32_t* ids, const float* dweights, void* dlogits,
                                       uint64_t dlogits_stride, void* stream) {
  const char* const who = "sky_route_topk_backward";
  SKY_TRY(check_rows(who, "logits", logits, dtype, rows, experts, &row_stride));
  SKY_TRY(check_rows(who, "dlogits", dlogits, dtype, rows, experts, &dlogits_stride));
  SKY_TRY(check_route(who, rows, experts, rules));
  if (rows && (!ids || !dweights)) return fail(SKY_ERR_ARG, "sky_route_topk_backward: ids or dweights is null");
  SKY_TRY(check_aligned(who, "ids", ids, 4));
  SKY_TRY(check_aligned(who, "dweights", dweights, 4));
  if (!rows) return SKY_OK;
  SKY_TRY(ensure_device());
  RouteArgs a{};
  a.logits = logits;
  a.stride = row_stride;
  a.rows = rows;
  a.experts = experts;
  a.r = *rules;
  a.ids_in = ids;
  a.dweights = dweights;
  a.dlogits = dlogits;
  a.dstride = dlogits_stride;
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((rows + ROUTE_WAVES - 1) / ROUTE_WAVES), dim3(64 * ROUTE_WAVES), 0, st, a);
  };
  SKY_ROUTE_LAUNCH(route_backward_kernel);
  return check_launch();
}
