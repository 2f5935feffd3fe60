// Routing to experts (sky_route_topk) and its gradient.  A wavefront has a row of E logits at a time, lane l the experts PER l, PER l + 1, ...
//   score    s_e = exp(x_e - max) / sum, or 1 / (1 + exp(-x_e))
//   choice   by s_e + b_e, the largest first, equal ones by number.  Both scores ascend with the logit, so without a bias and
//            without pairs of experts the choice goes by the logits themselves, exactly.  Else it is made from scores in fp32, whose error
//            has a bound; where two of those that it hangs on (neighbours among the k + 1 best, what is as near to the last chosen, the
//            last group that stays and the first that does not) are nearer than that and not alike, the row is chosen again in fp64: one
//            expert more or less is no rounding error.  (32,768 rows of 256, 8 of 4 of 8 groups: all in fp64 96 us.)
//   weights  w_j = scale * s_j, renormalised scale * s_j / sum of the k chosen.  Renormalised, the sum over all experts drops out of
//            softmax scores, and sigmoid scores are taken relative to the largest of the chosen (their logarithms
//            are at hand), so that a row of tiny scores keeps its shares.  In fp64, for as many rows at once as the chosen fill a wavefront.
// Bound by the instructions: 32,768 rows of 256 bf16, 8 of them by sigmoid and bias from 4 of 8 groups, 42 us, of which the counts by
// expert take 5, the groups 10 and the rows in doubt 6.
// Gradient, g_j = scale * dw_j, p_j = share of the chosen j:
//   softmax, renormalised    dx_j = p_j (g_j - sum_i g_i p_i) for the chosen, 0 elsewhere
//   softmax                  dx_e = s_e (g_e [e chosen] - sum_i g_i s_i)
//   sigmoid, renormalised    dx_j = p_j (1 - s_j) (g_j - sum_i g_i p_i)
//   sigmoid                  dx_j = g_j s_j (1 - s_j)
#include "sky_scores.h"

namespace sky {
namespace {

constexpr uint32_t MAX_EXPERTS = 1024, MAX_K = 64, MAX_GROUPS = 64;
constexpr uint32_t MAX_ROWS = 1u << 25;  // a launch has fewer than 2^32 threads, 64 for a row at most
constexpr int ROUTE_WAVES = 4;  // of a workgroup

struct RouteArgs {
  const void* logits;
  uint64_t stride;
  uint32_t rows, experts;
  sky_route_rules r;
  uint32_t* ids;
  float* weights;
  uint32_t* counts;  // to be cleared by the first workgroup for the kernel that follows; may be null
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
// Whether a bias of the wavefront's is infinite or NaN: the bound of the fp32 choices does not hold then.
template <int PER>
__device__ __forceinline__ bool some_not_finite(const float (&bias)[PER]) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) odd |= !(fabsf(bias[i]) < __builtin_inff());
  return __ballot(odd) != 0;
}
// e^x of x <= 0, to some 1e-14: the series of e^f on |f| <= ln(2) / 2 through degree 11
__device__ __forceinline__ double exp_negative(double x) {
  const double t = fmax(x * 1.44269504088896340736, -1000.0), n = rint(t), f = (t - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return __longlong_as_double(__double_as_longlong(p) + ((long long)(int)n << 52));
}
// 1 / (1 + exp(-x)) * exp(-m) for m = min(x, 0) or between that and 0: the part of a score that shares hang on
__device__ __forceinline__ double sigmoid_over(double x, double m) { return exp_negative(fmin(x, 0.0) - m) / (1.0 + exp_negative(-fabs(x))); }

__device__ __forceinline__ bool chosen_by_logit(const sky_route_rules& r) { return !r.bias && !(r.groups > 1 && r.groups_kept < r.groups && r.group_top2); }

// Whether two experts of a row have the same logit and bias: the same score then, and they stand by number.
template <typename T>
__device__ __forceinline__ bool alike(const RouteArgs& a, const T* x, uint32_t e, uint32_t f) {
  return (float)x[e] == (float)x[f] && (!a.r.bias || a.r.bias[e] == a.r.bias[f]);
}

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
  const bool by_logit = chosen_by_logit(a.r);
  if (!a.r.sigmoid && !by_logit) {
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
      const double score = by_logit ? (double)z[i] : a.r.sigmoid ? 1.0 / (1.0 + exp(-(double)z[i])) : exp((double)z[i] - (double)zmax) / sum;
      const double choice = score + (a.r.bias ? (double)a.r.bias[e] : 0.0);
      if (choice > -__builtin_inf()) key[i] = double_key(choice);
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

// The weights of the wavefront's rows, a chosen expert a lane: the j-th of `row`, whose lanes lie together, `slots` of them.
template <typename T>
__device__ __forceinline__ void store_weights(const RouteArgs& a, uint32_t row, bool real, uint32_t j, uint32_t slots, uint32_t id, float zmax, double sum) {
  const uint32_t k = a.r.k;
  const bool mine = real && j < k, in = mine && id != SKY_INVALID;
  const float chosen = in ? plain_score((float)((const T*)a.logits + row * a.stride)[id]) : 0.0f;
  double w = 0.0;
  if (a.r.renormalise) {
    // relative to the largest of the chosen, which need not be the first of the order: a bias or groups may have decided
    float top = in ? (a.r.sigmoid ? fminf(chosen, 0.0f) : chosen) : -__builtin_inff();
    for (uint32_t m = 1; m < slots; m *= 2) top = fmaxf(top, __shfl_xor(top, (int)m, 64));
    if (in) w = a.r.sigmoid ? sigmoid_over(chosen, top) : exp_negative((double)chosen - (double)top);
    double all = w;
    for (uint32_t m = 1; m < slots; m *= 2) all += __shfl_xor(all, (int)m, 64);
    w = all > 0.0 ? w / all : 0.0;
  } else if (in) {
    w = a.r.sigmoid ? sigmoid_over(chosen, 0.0) : exp_negative((double)chosen - (double)zmax) / sum;
  }
  if (mine) {
    a.ids[(uint64_t)row * k + j] = id;
    a.weights[(uint64_t)row * k + j] = in ? (float)((double)a.r.scale * w) : 0.0f;
  }
}

// ---------------------------------------------------------------- four rows at a time
// Up to 256 experts, 16 chosen and 16 groups: 16 lanes have a row, lane l of them the experts PER l, PER l + 1, ...  The k best are not
// taken out one after another: the k-th largest of the lanes' largest is no larger than the k-th largest of all, some 11 of 256
// experts reach the 8th, and each of those counts how many come before it.  Everything a row asks of its lanes are rotations within 16
// lanes, which cost an instruction.
constexpr int QUAD_EXPERTS = 256, QUAD_K = 16, QUAD_GROUPS = 16;
constexpr uint32_t QUAD_LISTED = 128;  // candidates of a row; a row with more (many equal ones) is chosen from in fp64, one by one

template <int N>
__device__ __forceinline__ uint32_t turn16(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xF, 0xF, true);  // from lane (l - N) mod 16
}
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, turn16<8>(v));
  v = max(v, turn16<4>(v));
  v = max(v, turn16<2>(v));
  return max(v, turn16<1>(v));
}
__device__ __forceinline__ uint32_t min16(uint32_t v) { return ~max16(~v); }
__device__ __forceinline__ float sum16(float v) {
  v += __uint_as_float(turn16<8>(__float_as_uint(v)));
  v += __uint_as_float(turn16<4>(__float_as_uint(v)));
  v += __uint_as_float(turn16<2>(__float_as_uint(v)));
  return v + __uint_as_float(turn16<1>(__float_as_uint(v)));
}
__device__ __forceinline__ uint32_t prefix16(uint32_t v) { return group_scan_u32<16>(v); }
// How many of the 16 lanes hold more; EQUAL: or as much and are smaller.
template <bool EQUAL, int N = 1>
__device__ __forceinline__ uint32_t larger16(uint32_t v, uint32_t sub) {
  const uint32_t o = turn16<N>(v);
  const uint32_t mine = EQUAL ? o > v || (o == v && sub >= N) : o > v;  // lane (l - N) mod 16 is smaller than l where l >= N
  if constexpr (N < 15)
    return mine + larger16<EQUAL, N + 1>(v, sub);
  else
    return mine;
}
// The same row's lane across: N = 1, 2, 4, 8 (4 and 8: of values that are the same in all of the 4 or 8 lanes that mirror one another)
template <int N>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  return dpp0<N == 1 ? DPP_QUAD_XOR1 : N == 2 ? DPP_QUAD_XOR2 : N == 4 ? DPP_ROW_HALF_MIRROR : DPP_ROW_MIRROR, 0xF>(v);
}

template <typename T, int PER>
__global__ __launch_bounds__(64 * ROUTE_WAVES, 4) void route_quad_kernel(RouteArgs a, uint32_t turns, uint32_t slots) {
  constexpr int WIDE = PER > 4 ? PER / 4 : 1;  // experts a lane where a wavefront has a row
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & 15, quarter = lane >> 4;
  const uint32_t row0 = (blockIdx.x * ROUTE_WAVES + wave) * (4 * turns), E = a.experts, k = a.r.k;
  if (blockIdx.x == 0 && a.counts)
    for (uint32_t e = threadIdx.x; e < E; e += 64 * ROUTE_WAVES) a.counts[e] = 0;
  struct Wave {
    union {
      struct {
        uint32_t key[4][16 * PER];         // of the four rows
        float listed[4][QUAD_LISTED + 4];  // choices (logits where it goes by them), filled up to four with what is none
        uint32_t expert[4][QUAD_LISTED];
        float best[4][QUAD_K + 2];  // the k best and the one after them
        uint32_t place[4][QUAD_K + 2];
      };
      double exact[64 * WIDE];
    };
    uint32_t id[64];  // chosen: row n of the wavefront has slots n * slots ...
    double sum[64];
    float zmax[64];
  };
  __shared__ Wave shared[ROUTE_WAVES];
  if (row0 >= a.rows) return;
  Wave& s = shared[wave];
  const uint32_t rows = min(4 * turns, a.rows - row0);
  const bool grouped = a.r.groups > 1 && a.r.groups_kept < a.r.groups;
  const bool by_logit = chosen_by_logit(a.r);
  const bool full_sum = !a.r.sigmoid && !a.r.renormalise;
  const uint32_t size = E / a.r.groups, lanes = size / PER;  // of a group
  const bool whole_lanes = size % PER == 0 && (lanes & (lanes - 1)) == 0;
  float bias[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) bias[i] = a.r.bias && sub * PER + i < E ? a.r.bias[sub * PER + i] : 0.0f;
  const bool odd = some_not_finite(bias);
  s.id[lane] = SKY_INVALID;
  for (uint32_t t = 0; t < turns; ++t) {
    const uint32_t n = 4 * t + quarter;  // of the wavefront's rows
    if (4 * t >= rows) break;
    const T* const x = (const T*)a.logits + (uint64_t)(row0 + min(n, rows - 1)) * a.stride;
    float z[PER];
    if (PER * 16 == E) {
      T v[PER];
      __builtin_memcpy(v, x + sub * PER, sizeof(v));
#pragma unroll
      for (int i = 0; i < PER; ++i) z[i] = plain_score((float)v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) z[i] = sub * PER + i < E ? plain_score((float)x[sub * PER + i]) : -__builtin_inff();
    }
    float zmax = z[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) zmax = fmaxf(zmax, z[i]);
    zmax = key_score(max16(score_key(zmax)));
    if (full_sum) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const double w = exp_negative((double)z[i] - (double)zmax);
        sum += open_expert(z[i]) ? w : 0.0;
      }
      sum = group_sum_f64<16>(sum);
      if (sub == 0) {
        s.sum[n] = sum;
        s.zmax[n] = zmax;
      }
    }
    uint32_t key[PER];
    float near = 0.0f;  // choices that are nearer than this may be the other way round
    if (by_logit) {
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = open_expert(z[i]) ? score_key(z[i]) : 0;
    } else {
      // What fp32 costs.  Sigmoid: constant and product leave the exponent off by 2^-23.4 of itself, the exponential by 2^-23 more, which
      // moves the score by s (1 - s) of that (0.17 and 0.25 units of 2^-23); sum and reciprocal 1.5 units of s: 2^-22 in all.  Softmax: as much
      // for each, and their sum, 20 additions deep, off by 12 units of 2^-23 for all alike.  The bias: 2^-24 of the choice.  Two
      // choices are the right way round if they differ by twice that; `near` is twice as much again.
      float c[PER], most = 1.0f;
      if (a.r.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z[i] * -1.44269504f));  // of a closed one: 0
      } else {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          c[i] = open_expert(z[i]) ? __builtin_amdgcn_exp2f((z[i] - zmax) * 1.44269504f) : 0.0f;
          sum += c[i];
        }
        most = __builtin_amdgcn_rcpf(sum16(sum));
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] *= most;
      }
      float size_of_choice = 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        c[i] += bias[i];
        size_of_choice = fmaxf(size_of_choice, fabsf(c[i]));
        key[i] = open_expert(z[i]) ? score_key(c[i]) : 0;
      }
      near = (a.r.sigmoid ? 0x1p-20f : 0x1p-18f * most) + 0x1p-22f * key_score(max16(score_key(size_of_choice)));
    }
    bool doubt = odd;  // of this lane
    if (grouped) {
      uint32_t best = 0, second = 0, owner;  // owner: the lane that speaks for this lane's experts
      if (whole_lanes) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          second = max(second, min(best, key[i]));
          best = max(best, key[i]);
        }
        auto join = [&](uint32_t b, uint32_t c) {
          second = max(min(best, b), max(second, c));
          best = max(best, b);
        };
        if (lanes > 1) join(across<1>(best), across<1>(second));
        if (lanes > 2) join(across<2>(best), across<2>(second));
        if (lanes > 4) join(across<4>(best), across<4>(second));
        if (lanes > 8) join(across<8>(best), across<8>(second));
        owner = sub & ~(lanes - 1);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) s.key[quarter][sub * PER + i] = key[i];
        __builtin_amdgcn_wave_barrier();
        if (sub < a.r.groups)
          for (uint32_t i = 0; i < size; ++i) {
            const uint32_t v = s.key[quarter][sub * size + i];
            second = max(second, min(best, v));
            best = max(best, v);
          }
        __builtin_amdgcn_wave_barrier();
        owner = sub;
      }
      uint32_t mine = best;
      if (best && second && a.r.group_top2) mine = score_key(key_score(best) + key_score(second));
      if (owner != sub) mine = 0;
      bool stays = mine && larger16<false>(mine, sub) < a.r.groups_kept;
      if (__ballot((uint32_t)__popc((uint32_t)(__ballot(stays) >> (lane & 48)) & 0xFFFFu) > a.r.groups_kept)) stays = mine && larger16<true>(mine, sub) < a.r.groups_kept;  // equal ones
      const uint32_t last = min16(stays ? mine : 0xFFFFFFFFu), next = max16(stays ? 0 : mine);
      if (!by_logit && next) doubt |= !(key_score(last) - key_score(next) > 3.0f * near);  // (of a NaN among the biases `near` knows nothing)
      const uint32_t stay = (uint32_t)(__ballot(stays) >> (lane & 48)) & 0xFFFFu;
      if (whole_lanes) {
        const bool mine_stays = stay >> owner & 1;
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = mine_stays ? key[i] : 0;
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint32_t e = sub * PER + i;
          if (e >= E || !(stay >> (e / size) & 1)) key[i] = 0;
        }
      }
    }
    // candidates: what reaches the k-th largest of the lanes' largest, or may
    uint32_t top = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) top = max(top, key[i]);
    uint32_t least = min16(larger16<false>(top, sub) < k ? top : 0xFFFFFFFFu);
    if (!by_logit && least) least = score_key(key_score(least) - near);
    least = max(least, 1u);
    uint32_t wanted = 0;  // bits of the lane's candidates
#pragma unroll
    for (int i = 0; i < PER; ++i) wanted |= key[i] >= least ? 1u << i : 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) s.key[quarter][sub * PER + i] = key[i];
    const uint32_t mine = (uint32_t)__popc(wanted), sum = prefix16(mine);
    const uint32_t count = (uint32_t)__shfl((int)sum, (int)(lane | 15), 64), listed = min(count, QUAD_LISTED);
    if (count > QUAD_LISTED) doubt = true;
    __builtin_amdgcn_wave_barrier();
    for (uint32_t at = sum - mine; wanted && at < QUAD_LISTED; ++at) {
      const uint32_t e = sub * PER + (uint32_t)__builtin_ctz(wanted);
      wanted &= wanted - 1;
      s.listed[quarter][at] = key_score(s.key[quarter][e]);
      s.expert[quarter][at] = e;
    }
    if (sub < 4) s.listed[quarter][listed + sub] = -__builtin_inff();
    if (sub == 0 && listed <= k) s.best[quarter][listed] = -__builtin_inff();
    __builtin_amdgcn_wave_barrier();
    for (uint32_t c = sub; c < listed; c += 16) {
      // candidates stand by number: of equal ones the first comes first
      const float v = s.listed[quarter][c];
      const uint32_t e = s.expert[quarter][c];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < listed; j += 4) {
        const float4 o = *(const float4*)&s.listed[quarter][j];
        rank += o.x > v || (o.x == v && j < c);
        rank += o.y > v || (o.y == v && j + 1 < c);
        rank += o.z > v || (o.z == v && j + 2 < c);
        rank += o.w > v || (o.w == v && j + 3 < c);
      }
      if (rank <= k) {
        s.best[quarter][rank] = v;
        s.place[quarter][rank] = e;
        if (rank < k && n < rows) s.id[n * slots + rank] = e;
      }
    }
    __builtin_amdgcn_wave_barrier();
    // (best[listed] is -inf, further than any bound from a finite number: place[listed], which is not set, is then not looked at)
    bool level = false;  // the last that is chosen and the first that is not are alike
    if (!by_logit && !odd && sub < k && sub < listed && !(s.best[quarter][sub] - s.best[quarter][sub + 1] > near)) {
      // alike, the same logit and bias, they stand as they are
      const uint32_t e = s.place[quarter][sub];
      const bool same = alike(a, x, e, s.place[quarter][sub + 1]);
      doubt |= !same;
      level = same && sub == k - 1;
    }
    // then one behind them that is as near may be better than both: all of these have to be alike
    const uint64_t levels = __ballot(level);
    if (levels >> (lane & 48) & 0xFFFFu) {
      const float v = s.best[quarter][k - 1];
      const uint32_t e = s.place[quarter][k - 1];
      for (uint32_t c = sub; c < listed; c += 16)
        if (!(fabsf(v - s.listed[quarter][c]) > near)) doubt |= !alike(a, x, e, s.expert[quarter][c]);
    }
    // rows in doubt, one after another by the whole wavefront
    uint64_t rest = __ballot(doubt);
    while (rest) {
      const uint32_t q = (uint32_t)__builtin_ctzll(rest) >> 4, m = 4 * t + q;
      rest &= ~(0xFFFFull << (16 * q));
      if (m >= rows) continue;
      __builtin_amdgcn_wave_barrier();
      const uint32_t id = choose_exactly<T, WIDE>((const T*)a.logits + (uint64_t)(row0 + m) * a.stride, a, s.exact, 0, SKY_INVALID);
      if (lane < slots) s.id[m * slots + lane] = id;
    }
    __builtin_amdgcn_wave_barrier();
  }
  const uint32_t n = lane / slots;
  store_weights<T>(a, row0 + n, n < rows, lane % slots, slots, s.id[lane], full_sum ? s.zmax[n] : 0.0f, full_sum ? s.sum[n] : 1.0);
}

// ---------------------------------------------------------------- a row at a time
// A wavefront takes rows_per_wave rows, which fill it with chosen experts: `slots` lanes (a power of two, at least k) for a row's.
template <typename T, int PER>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_kernel(RouteArgs a, uint32_t rows_per_wave, uint32_t slots) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t row0 = (blockIdx.x * ROUTE_WAVES + wave) * rows_per_wave, E = a.experts, k = a.r.k;
  if (blockIdx.x == 0 && a.counts)
    for (uint32_t e = threadIdx.x; e < E; e += 64 * ROUTE_WAVES) a.counts[e] = 0;
  __shared__ double staged_all[ROUTE_WAVES][64 * PER];
  if (row0 >= a.rows) return;
  double* const staged = staged_all[wave];
  const uint32_t rows = min(rows_per_wave, a.rows - row0);
  const bool grouped = a.r.groups > 1 && a.r.groups_kept < a.r.groups;
  const bool by_logit = chosen_by_logit(a.r);
  const bool full_sum = !a.r.sigmoid && !a.r.renormalise;  // the sum over all experts goes into the weights
  const uint32_t size = E / a.r.groups, lanes = size / PER;  // of a group
  // groups whose experts are whole lanes, a power of two of them, are reduced across lanes; others through LDS
  const bool whole_lanes = size % PER == 0 && (lanes & (lanes - 1)) == 0;
  float bias[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) bias[i] = a.r.bias && lane * PER + i < E ? a.r.bias[lane * PER + i] : 0.0f;
  const bool odd = some_not_finite(bias);
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
      for (int i = 0; i < PER; ++i) {
        const double w = exp_negative((double)z[i] - (double)zmax);
        sum += open_expert(z[i]) ? w : 0.0;
      }
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
      // What fp32 costs.  Sigmoid: constant and product leave the exponent off by 2^-23.4 of itself, the exponential by 2^-23 more, which
      // moves the score by s (1 - s) of that (0.17 and 0.25 units of 2^-23); sum and reciprocal 1.5 units of s: 2^-22 in all.  Softmax: as much
      // for each, and their sum, 20 additions deep, off by 12 units of 2^-23 for all alike.  The bias: 2^-24 of the choice.  Two
      // choices are the right way round if they differ by twice that; `near` is twice as much again.
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
      near = (a.r.sigmoid ? 0x1p-20f : 0x1p-18f * most) + 0x1p-22f * size_of_choice;
    }
    bool exact = !odd;  // the choice so far
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
      if (!by_logit && next && !(key_score(last) - key_score(next) > 3.0f * near)) exact = false;
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
      if (!by_logit && j && !(key_score(before) - key_score(best) > near)) {
        exact = alike(a, x, e, before_e);
        if (exact && j == k) {  // one behind them that is as near may be better than both: all of these have to be alike
          bool other = false;
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (key[i] && !(key_score(before) - key_score(key[i]) > near)) other |= !alike(a, x, before_e, lane * PER + i);
          exact = __ballot(other) == 0;
        }
      }
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
  const uint32_t n = lane / slots;
  store_weights<T>(a, row0 + n, n < rows, lane % slots, slots, id, my_max, my_sum);
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

// The gradient: G lanes have a row, NP pieces of 16 bytes each, the pieces of a row one after another over the lanes.  The chosen
// entries' own parts meet the row in LDS.  Bound by memory: 32,768 x 256 fp32 13 us, 5.2 TB/s.  (A wavefront a row, the parts by 64
// exchanges between lanes: 34 us.)
template <int G>
__device__ __forceinline__ float group_max_f32(float v) {
  if constexpr (G == 16)
    return key_score(max16(score_key(v)));
  else
    return wave_max_f32(v);
}
template <int G>
__device__ __forceinline__ float group_sum_f32(float v) {
  if constexpr (G == 16)
    return sum16(v);
  else
    return wave_sum_f32(v);
}
template <typename T, int G, int NP>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_backward_kernel(RouteArgs a) {
  constexpr int N = Piece<T>::N, ROWS = 64 / G, KP = (int)MAX_K / G > 1 ? (int)MAX_K / G : 1;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % G;
  const uint32_t want = (blockIdx.x * ROUTE_WAVES + wave) * ROWS + lane / G, E = a.experts, k = a.r.k;
  __shared__ __attribute__((aligned(16))) float parts[ROUTE_WAVES][ROWS][G * NP * N];
  if ((blockIdx.x * ROUTE_WAVES + wave) * ROWS >= a.rows) return;
  const uint32_t row = min(want, a.rows - 1);  // lanes of rows that are not there go along
  const T* const x = (const T*)a.logits + row * a.stride;
  T* const dx = (T*)a.dlogits + row * a.dstride;
  float* const part = parts[wave][lane / G];
  const bool dense = !a.r.sigmoid && !a.r.renormalise;
  uint32_t id[KP];
  float g[KP], xj[KP], d[KP];
#pragma unroll
  for (int i = 0; i < KP; ++i) {
    const uint32_t j = sub + G * i;
    id[i] = j < k ? a.ids_in[(uint64_t)row * k + j] : SKY_INVALID;
    g[i] = id[i] < E ? a.dweights[(uint64_t)row * k + j] * a.r.scale : 0.0f;
    xj[i] = id[i] < E ? plain_score((float)x[id[i]]) : -__builtin_inff();
    if (!open_expert(xj[i])) {
      id[i] = SKY_INVALID;
      g[i] = 0.0f;
    }
  }
  float z[NP][N];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) z[i][e] = 0.0f;
  float zmax = -__builtin_inff(), total = 0.0f;
  if (dense) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t c = (i * G + sub) * N;
      if (c + N <= E) {
        const Piece<T> v = load_piece(x + c);
#pragma unroll
        for (int e = 0; e < N; ++e) z[i][e] = plain_score((float)v.e[e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) z[i][e] = c + e < E ? plain_score((float)x[c + e]) : -__builtin_inff();
      }
#pragma unroll
      for (int e = 0; e < N; ++e) zmax = fmaxf(zmax, z[i][e]);
    }
    zmax = group_max_f32<G>(zmax);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        z[i][e] = open_expert(z[i][e]) ? __builtin_amdgcn_exp2f((z[i][e] - zmax) * 1.44269504f) : 0.0f;
        total += z[i][e];
      }
    total = group_sum_f32<G>(total);
  }
  // the gradient at the chosen entries (in the dense case: what is added to -s_e * sum g s)
  float mean = 0.0f;
  if (a.r.renormalise) {
    // shares relative to the largest of the chosen: e^min(x, 0) / (1 + e^-|x|) is a sigmoid
    float most = -__builtin_inff(), all = 0.0f;
#pragma unroll
    for (int i = 0; i < KP; ++i)
      if (id[i] != SKY_INVALID) most = fmaxf(most, a.r.sigmoid ? fminf(xj[i], 0.0f) : xj[i]);
    most = group_max_f32<G>(most);
    float p[KP];
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      p[i] = id[i] == SKY_INVALID ? 0.0f : a.r.sigmoid ? expf(fminf(xj[i], 0.0f) - most) / (1.0f + expf(-fabsf(xj[i]))) : expf(xj[i] - most);
      all += p[i];
    }
    all = group_sum_f32<G>(all);
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      p[i] = all > 0.0f ? p[i] / all : 0.0f;
      mean += g[i] * p[i];
    }
    mean = group_sum_f32<G>(mean);
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      d[i] = p[i] * (g[i] - mean);
      if (a.r.sigmoid && id[i] != SKY_INVALID) d[i] *= 1.0f / (1.0f + expf(xj[i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      d[i] = 0.0f;
      if (id[i] != SKY_INVALID) d[i] = a.r.sigmoid ? g[i] * (1.0f / (1.0f + expf(-xj[i]))) * (1.0f / (1.0f + expf(xj[i]))) : g[i] * __builtin_amdgcn_exp2f((xj[i] - zmax) * 1.44269504f) / total;
      mean += d[i];
    }
    mean = dense ? group_sum_f32<G>(mean) : 0.0f;
  }
  const float weight = dense && total > 0.0f ? -mean / total : 0.0f;
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int e = 0; e < N; e += 4) *(float4*)&part[(i * G + sub) * N + e] = float4{0.0f, 0.0f, 0.0f, 0.0f};
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < KP; ++i)
    if (id[i] != SKY_INVALID) atomicAdd(&part[id[i]], d[i]);  // ids of a row are distinct as they are chosen
  __builtin_amdgcn_wave_barrier();
  if (want >= a.rows) return;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint32_t c = (i * G + sub) * N;
    Piece<T> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.e[e] = (T)(z[i][e] * weight + part[c + e]);
    if (c + N <= E) {
      store_piece(dx + c, o);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c + e < E) dx[c + e] = o.e[e];
    }
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
  if (rows > MAX_ROWS) return fail(SKY_ERR_LIMIT, std::string(who) + ": more than 2^25 rows");
  return SKY_OK;
}

#define SKY_ROUTE_PER(kernel, T)                                                          \
  (experts <= 64 ? launch(kernel<T, 1>)                                                   \
   : experts <= 128 ? launch(kernel<T, 2>)                                                \
   : experts <= 256 ? launch(kernel<T, 4>)                                                \
   : experts <= 512 ? launch(kernel<T, 8>)                                                \
                    : launch(kernel<T, 16>))
#define SKY_ROUTE_QUAD(kernel, T)                                                         \
  (experts <= 16 ? launch(kernel<T, 1>)                                                   \
   : experts <= 32 ? launch(kernel<T, 2>)                                                 \
   : experts <= 64 ? launch(kernel<T, 4>)                                                 \
   : experts <= 128 ? launch(kernel<T, 8>)                                                \
                    : launch(kernel<T, 16>))
// (16-bit rows have two pieces a lane at most)
#define SKY_ROUTE_PIECES(kernel, T)                                           \
  (lanes == 16 ? (pieces <= 1   ? launch(kernel<T, 16, 1>)                    \
                  : pieces <= 2 ? launch(kernel<T, 16, 2>)                    \
                                : launch(kernel<T, 16, sizeof(T) == 4 ? 4 : 2>)) \
               : (pieces <= 2 ? launch(kernel<T, 64, 2>)                      \
                              : launch(kernel<T, 64, sizeof(T) == 4 ? 4 : 2>)))
#define SKY_ROUTE_LAUNCH(PER, kernel)       \
  (dtype == SKY_F32 ? PER(kernel, float)    \
   : dtype == SKY_F16 ? PER(kernel, _Float16) \
                      : PER(kernel, __bf16))

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
  a.counts = counts;
  uint32_t slots = 1;
  while (slots < rules->k) slots *= 2;
  // Where k lanes of experts are all there are, the least of the lanes' largest lets in many, and where there are fewer, all that may be
  // chosen are candidates, more than are listed, and every row is chosen from one by one.  (us, quads / a row a wavefront: 203 experts
  // by the 14 best, 13 lanes, 7 rows 63 / 8, 20,000 rows 141 / 39, by the 13 best 58 / 50; 256 by the 16 best, 16 lanes, 75 / 56, by
  // the 14 best 39 / 51, by the 9 best 28 / 39.)
  uint32_t per = 1;
  while (16 * per < experts) per *= 2;
  const uint32_t open = experts / rules->groups * rules->groups_kept;
  const bool listed = open <= QUAD_LISTED || rules->k < (open + per - 1) / per;
  if (experts <= QUAD_EXPERTS && rules->k <= QUAD_K && rules->groups <= QUAD_GROUPS && listed) {
    // four rows at a time, as many times as fill the wavefront with chosen experts, as long as there are wavefronts for every SIMD
    slots = std::max(slots, 4u);
    const uint32_t turns = std::min(16 / slots, std::max(rows / 8192u, 1u));
    const uint32_t per_block = 4 * turns * ROUTE_WAVES;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((rows + per_block - 1) / per_block), dim3(64 * ROUTE_WAVES), 0, st, a, turns, slots);
    };
    SKY_ROUTE_LAUNCH(SKY_ROUTE_QUAD, route_quad_kernel);
  } else {
    // as many rows a wavefront as fill it with chosen experts, as long as there is a wavefront for every SIMD
    const uint32_t per_wave = std::min(64 / slots, std::max(rows / 2048u, 1u));
    const uint64_t waves = ((uint64_t)rows + per_wave - 1) / per_wave;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((uint32_t)((waves + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(64 * ROUTE_WAVES), 0, st, a, per_wave, slots);
    };
    SKY_ROUTE_LAUNCH(SKY_ROUTE_PER, route_kernel);
  }
  if (counts) {
    const uint64_t n = (uint64_t)rows * rules->k;
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
  // up to 256 experts four rows a wavefront, more one
  const uint32_t lanes = experts <= QUAD_EXPERTS ? 16 : 64, per_block = 64 / lanes * ROUTE_WAVES;
  const uint32_t pieces = (uint32_t)((experts * dtype_size(dtype) + 16 * lanes - 1) / (16 * lanes));  // a lane: up to 4 of fp32, 2 of 16 bits
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((rows + per_block - 1) / per_block), dim3(64 * ROUTE_WAVES), 0, st, a); };
  SKY_ROUTE_LAUNCH(SKY_ROUTE_PIECES, route_backward_kernel);
  return check_launch();
}
