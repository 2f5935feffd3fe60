// Routing to experts (sky_route_topk) and its gradient.  A wavefront has a row of E logits, lane l the experts l, l + 64, ...
//   score    s_e = exp(x_e - max) / sum, or 1 / (1 + exp(-x_e))
//   choice   by s_e + b_e, the largest first, equal ones by number.  Both scores ascend with the logit, so without a bias and
//            without pairs of experts the choice goes by the logits themselves; else it is computed in fp64, because one expert
//            more or less is no rounding error.
//   weights  w_j = scale * s_j, renormalised scale * s_j / sum of the k chosen.  Renormalised, the sum over all experts drops out of
//            softmax scores, and sigmoid scores are taken relative to the largest of the chosen (their logarithms
//            are at hand), so that a row of tiny scores keeps its shares.
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
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
  v = max(v, dpp0_u64<DPP_QUAD_XOR1, 0xF>(v));
  v = max(v, dpp0_u64<DPP_QUAD_XOR2, 0xF>(v));
  v = max(v, dpp0_u64<DPP_ROW_HALF_MIRROR, 0xF>(v));
  v = max(v, dpp0_u64<DPP_ROW_MIRROR, 0xF>(v));
  v = max(v, shfl_xor_u64(v, 16));
  return max(v, shfl_xor_u64(v, 32));
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

// PER experts a lane.  Keys of the choice: 0 is a closed expert, a taken one or none.
template <typename T, int PER>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_kernel(RouteArgs a) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t row = blockIdx.x * ROUTE_WAVES + wave, E = a.experts, k = a.r.k;
  __shared__ double staged[ROUTE_WAVES][64 * PER];
  if (row >= a.rows) return;
  const T* const x = (const T*)a.logits + row * a.stride;
  float z[PER];
  float zmax = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t e = 64 * i + lane;
    z[i] = e < E ? plain_score((float)x[e]) : -__builtin_inff();
    zmax = fmaxf(zmax, z[i]);
  }
  zmax = wave_max_f32(zmax);
  const bool grouped = a.r.groups > 1 && a.r.groups_kept < a.r.groups;
  const bool by_logit = !a.r.bias && !(grouped && a.r.group_top2);
  double sum = 0.0;  // of the softmax, relative to the largest logit
  if (!a.r.sigmoid && (!a.r.renormalise || !by_logit)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += open_expert(z[i]) ? exp((double)z[i] - (double)zmax) : 0.0;
    sum = group_sum_f64<64>(sum);
  }
  auto score = [&](float v) -> double {
    if (a.r.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
    return exp((double)v - (double)zmax) / sum;
  };
  uint64_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t e = 64 * i + lane;
    key[i] = 0;
    if (open_expert(z[i])) {
      const double c = by_logit ? (double)z[i] : score(z[i]) + (a.r.bias ? (double)a.r.bias[e] : 0.0);
      key[i] = double_key(c);
    }
  }
  if (grouped) {
    // a lane has a group: its best choice, or the sum of its two best
    const uint32_t size = E / a.r.groups;
#pragma unroll
    for (int i = 0; i < PER; ++i) staged[wave][64 * i + lane] = __longlong_as_double((long long)key[i]);
    __builtin_amdgcn_wave_barrier();
    uint64_t mine = 0;
    if (lane < a.r.groups) {
      uint64_t first = 0, second = 0;
      for (uint32_t i = 0; i < size; ++i) {
        const uint64_t v = (uint64_t)__double_as_longlong(staged[wave][lane * size + i]);
        second = max(second, min(first, v));
        first = max(first, v);
      }
      auto value = [](uint64_t v) { return __longlong_as_double((long long)(v ^ ((v >> 63) ? 1ull << 63 : ~0ull))); };
      // a group without an open expert is worth less than any other; a lone open expert counts by itself
      mine = first;
      if (first && second && a.r.group_top2) mine = double_key(value(first) + value(second));
    }
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
      const uint32_t e = 64 * i + lane;
      if (e >= E || !(stay >> (e / size) & 1)) key[i] = 0;
    }
  }
  // the k best, the j-th into lane j
  uint32_t id = SKY_INVALID;
  float chosen = -__builtin_inff();
  for (uint32_t j = 0; j < k; ++j) {
    uint64_t mine = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > mine) {
        mine = key[i];
        at = i;
      }
    const uint64_t best = wave_max_u64(mine);
    if (!best) break;
    const uint32_t e = wave_min_u32(mine == best ? 64 * (uint32_t)at + lane : 0xFFFFFFFFu);
    float v = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if ((e >> 6) == (uint32_t)i) {
        v = z[i];
        if (lane == (e & 63)) key[i] = 0;
      }
    }
    v = __shfl(v, (int)(e & 63), 64);
    if (lane == j) {
      id = e;
      chosen = v;
    }
  }
  double w = 0.0;
  if (a.r.renormalise) {
    // the first of the order has not got the largest score when a bias or groups decide
    const bool in = id != SKY_INVALID;
    const double l = !in ? 0.0 : a.r.sigmoid ? log_sigmoid(chosen) : (double)chosen;
    const double top = in ? l : -__builtin_inf();
    double most = top;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) most = fmax(most, __shfl_xor(most, m, 64));
    w = in ? exp(l - most) : 0.0;
    const double all = group_sum_f64<64>(w);
    w = all > 0.0 ? w / all : 0.0;
  } else if (id != SKY_INVALID) {
    w = score(chosen);
  }
  if (lane < k) {
    a.ids[(uint64_t)row * k + lane] = id;
    a.weights[(uint64_t)row * k + lane] = id != SKY_INVALID ? (float)((double)a.r.scale * w) : 0.0f;
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
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((rows + ROUTE_WAVES - 1) / ROUTE_WAVES), dim3(64 * ROUTE_WAVES), 0, st, a);
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
