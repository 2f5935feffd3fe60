// One id of every row of logits by chance (sky_logits_draw).  The entries of a row in the order "largest first, equal ones by column"
// weigh w = exp((z - zmax) / T); what stays of the row is always a beginning of that order (top-k, top-p and min-p each
// cut off an end), and the drawn entry is the first whose weights, summed in the order, pass u times what stays weighs.  So
// everything is one question, asked up to three times: which entry of the order holds rank k, or the unit of mass t?
//
// It is answered without sorting the row.  A workgroup has a row.  A sweep counts the entries (or sums their weights) in
// BINS bins of equal width between the largest and the smallest value; the bin that holds the answer is found by a scan, its
// entries are listed in LDS and sorted, and when they are too many for the list the bin becomes the next interval: it lies
// between the smallest and largest value that were met in it, so that two different values never stay together, and a bin of one
// value is a matter of counting.  Rows of which few entries can be drawn at all (a grammar's, a small top-k, min-p) are
// listed and sorted at once.
//
// Weights are summed in whole numbers (2^-S of the largest weight, S = 62 less the bits of the row's length): sums then do not depend on
// the order of LDS atomics or of lanes.  They are rounded once each, by at most 2^-(S+1) of the largest weight; the
// exponential is taken in fp64, since an id changes with the last bit that its border of the sum is off by.
#include "sky_scores.h"

namespace sky {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t BINS = 2048;  // two per thread
constexpr uint32_t CAP = 2048;   // entries of a list, two per thread
constexpr double NO_MASS = 40.0;  // weights below e^-40 are 0 in units of 2^-S, S <= 50

struct DrawArgs {
  const void* logits;
  uint64_t stride;
  uint32_t columns, rows;
  const float* temperature;
  const uint32_t* top_k;
  const float* top_p;
  const float* min_p;
  const double* uniforms;
  uint64_t seed;
  uint32_t first_walker, step;
  uint32_t* tokens;
  uint64_t tokens_stride;
  float* logprobs;
  uint32_t* kept;
};

struct Shared {
  uint64_t bin[BINS];   // counts or sums; also the list's sums
  uint64_t list[CAP];   // (~key << 32 | column): ascending is the order
  uint64_t wave[WAVES + 1];
  uint32_t n;
  uint32_t lo, hi;  // keys
  uint32_t found, found2;
  uint64_t before;
};

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp0<DPP_QUAD_XOR1, 0xF>(v));
  v = max(v, dpp0<DPP_QUAD_XOR2, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_HALF_MIRROR, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_MIRROR, 0xF>(v));
  v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
}

// The settings and the state of one row.
struct Row {
  double t;
  float zmax;
  int S;  // fraction bits of a weight
};
__device__ __forceinline__ double weight_of(float z, float zmax, double t) { return exp(((double)z - (double)zmax) / t); }
__device__ __forceinline__ uint64_t mass_of(double w, int S) { return (uint64_t)(ldexp(w, S) + 0.5); }

// Exclusive prefix of v over the workgroup, and the total.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, Shared& s, uint64_t* total) {
  const uint64_t inclusive = group_scan_u64<64>(v);
  const uint32_t w = threadIdx.x >> 6, l = threadIdx.x & 63;
  __syncthreads();
  if (l == 63) s.wave[w] = inclusive;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const uint64_t x = s.wave[i];
    before += (uint32_t)i < w ? x : 0;
    all += x;
  }
  *total = all;
  return before + inclusive - v;
}

// The list s.list[0..m) into the order: a bitonic network over the next power of two.
__device__ __forceinline__ void sort_list(Shared& s, uint32_t m) {
  uint32_t size = 64;
  while (size < m) size *= 2;
  for (uint32_t i = threadIdx.x; i < size; i += THREADS)
    if (i >= m) s.list[i] = ~0ull;
  __syncthreads();
  for (uint32_t k = 2; k <= size; k *= 2)
    for (uint32_t j = k / 2; j; j /= 2) {
      const uint32_t i = threadIdx.x;
      if (i < size / 2) {
        const uint32_t a = (i & (j - 1)) | (i & ~(j - 1)) << 1, b = a | j;
        const uint64_t x = s.list[a], y = s.list[b];
        if ((x > y) == ((a & k) == 0)) {
          s.list[a] = y;
          s.list[b] = x;
        }
      }
      __syncthreads();
    }
}
__device__ __forceinline__ float listed_score(uint64_t e) { return key_score(~(uint32_t)(e >> 32)); }

template <typename T>
struct Sweep {
  const T* x;
  uint32_t columns;
  // f(score, column) for every entry that is there
  template <typename F>
  __device__ __forceinline__ void operator()(F f) const {
    constexpr uint32_t N = Piece<T>::N;
    for (uint32_t c = threadIdx.x * N; c < columns; c += THREADS * N) {
      if (c + N <= columns) {
        const Piece<T> v = load_piece(x + c);
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) f(plain_score((float)v.e[e]), c + e);
      } else {
        for (uint32_t e = 0; c + e < columns; ++e) f(plain_score((float)x[c + e]), c + e);
      }
    }
  }
};

// Where an answer lies: the value, how many entries of the same value come before it and its column (NO_COLUMN: not asked for),
// and what all entries before the value amount to (units of mass or entries).
struct Place {
  float z;
  uint32_t tie, column;
  uint64_t before;
};

struct Result {
  uint32_t token, kept;
  double logprob;
};

// Everything about a row whose entries (or as many of them as can matter) are the m entries of the list, unsorted.
__device__ Result draw_listed(Shared& s, uint32_t m, double t, uint32_t top_k, float top_p, float min_p, double u) {
  const int S = 50;  // at most 2^11 weights
  sort_list(s, m);
  const float zmax = listed_score(s.list[0]);
  const uint32_t k = top_k && top_k < m ? top_k : m;
  const uint32_t i0 = 2 * threadIdx.x, i1 = i0 + 1;
  const double w0 = i0 < k ? weight_of(listed_score(s.list[i0]), zmax, t) : -1.0;
  const double w1 = i1 < k ? weight_of(listed_score(s.list[i1]), zmax, t) : -1.0;
  const uint64_t m0 = w0 >= 0 ? mass_of(w0, S) : 0, m1 = w1 >= 0 ? mass_of(w1, S) : 0;
  uint64_t total;
  const uint64_t before = block_scan(m0 + m1, s, &total);
  uint32_t n = k;
  if (top_p < 1.0f || min_p > 0.0f) {
    // entries stay while what comes before them is below p of the total, and their weight at least min_p
    const uint64_t need = top_p < 1.0f ? (uint64_t)ceil(fmax((double)top_p, 0.0) * (double)total) : ~0ull;
    const bool in0 = i0 < k && (i0 == 0 || (before < need && w0 >= (double)min_p));
    const bool in1 = i1 < k && before + m0 < need && w1 >= (double)min_p;
    uint64_t many;
    block_scan((uint64_t)in0 + (uint64_t)in1, s, &many);
    n = (uint32_t)many;
  }
  // what the n entries weigh, by the owner of the last one
  if ((n - 1) >> 1 == threadIdx.x) s.before = before + m0 + ((n - 1) & 1 ? m1 : 0);
  if (threadIdx.x == 0) s.found = n - 1;
  __syncthreads();
  const uint64_t mass = s.before;
  uint64_t unit = (uint64_t)(u * (double)mass);
  if (unit >= mass) unit = mass - 1;
  if (i0 < n && before <= unit && unit < before + m0) s.found = i0;
  if (i1 < n && before + m0 <= unit && unit < before + m0 + m1) s.found = i1;
  __syncthreads();
  const uint64_t e = s.list[s.found];
  Result r;
  r.token = (uint32_t)e;
  r.kept = n;
  r.logprob = ((double)listed_score(e) - (double)zmax) / t - log(ldexp((double)mass, -S));
  return r;
}

// Which bins an interval [lo, hi] of values has.  Monotone in z, the same for equal z, 0 for hi and BINS - 1 for lo.
struct Bins {
  double hi, scale;
  float top, low;
  __device__ __forceinline__ Bins(float h, float l) : hi(h), scale((double)(BINS - 1) / ((double)h - (double)l)), top(h), low(l) {}
  __device__ __forceinline__ bool has(float z) const { return z <= top && z >= low; }
  __device__ __forceinline__ uint32_t of(float z) const { return min((uint32_t)((hi - (double)z) * scale), BINS - 1); }
};

// The entry of the order that holds unit `unit` (RANK: the entry of that rank; else the unit of mass) among the entries between
// `low` and zmax.  `excess` entries of the value `low` are not part of it, its last ones.  Every thread calls it and has the answer.
template <bool RANK, typename T>
__device__ Place locate(const Sweep<T>& sweep, Shared& s, const Row& row, float low, uint32_t excess, uint64_t unit) {
  Place p;
  uint64_t before = 0;
  float hi = row.zmax, lo = low;
  auto value = [&](float z) -> uint64_t { return RANK ? 1ull : mass_of(weight_of(z, row.zmax, row.t), row.S); };
  for (;;) {
    uint32_t n = 0;
    Bins bins(hi, lo < hi ? lo : hi - 1.0f);
    if (lo < hi) {
      __syncthreads();
      s.bin[2 * threadIdx.x] = s.bin[2 * threadIdx.x + 1] = 0;
      if (threadIdx.x == 0) {
        s.n = 0;
        s.lo = 0xFFFFFFFFu;
        s.hi = 0;
      }
      __syncthreads();
      sweep([&](float z, uint32_t) {
        if (bins.has(z)) {
          const uint64_t v = value(z);
          if (v) atomicAdd((unsigned long long*)&s.bin[bins.of(z)], (unsigned long long)v);
        }
      });
      __syncthreads();
      if (excess && bins.has(low) && threadIdx.x == 0) s.bin[bins.of(low)] -= (uint64_t)excess * value(low);
      __syncthreads();
      const uint64_t b0 = s.bin[2 * threadIdx.x], b1 = s.bin[2 * threadIdx.x + 1];
      uint64_t total;
      const uint64_t e = before + block_scan(b0 + b1, s, &total);
      if (e <= unit && unit < e + b0 + b1) {
        const uint32_t second = unit >= e + b0;
        s.found = 2 * threadIdx.x + second;
        s.before = e + (second ? b0 : 0);
      }
      __syncthreads();
      const uint32_t b = s.found;
      before = s.before;
      // the bin's entries: how many, between which values, and the list of them if it holds them
      uint32_t kmin = 0xFFFFFFFFu, kmax = 0;
      sweep([&](float z, uint32_t c) {
        if (bins.has(z) && bins.of(z) == b) {
          const uint32_t key = score_key(z);
          kmin = min(kmin, key);
          kmax = max(kmax, key);
          const uint32_t at = atomicAdd(&s.n, 1u);
          if (at < CAP) s.list[at] = (uint64_t)~key << 32 | c;
        }
      });
      kmin = wave_min_u32(kmin);
      kmax = wave_max_u32(kmax);
      if ((threadIdx.x & 63) == 0 && kmax) {
        atomicMin(&s.lo, kmin);
        atomicMax(&s.hi, kmax);
      }
      __syncthreads();
      n = s.n;
      lo = key_score(s.lo);
      hi = key_score(s.hi);
    }
    if (lo == hi) {  // one value: the place among its equals
      p.z = hi;
      p.tie = (uint32_t)((unit - before) / value(hi));
      p.column = 0xFFFFFFFFu;
      p.before = before;
      return p;
    }
    if (n <= CAP) {
      sort_list(s, n);
      const uint32_t m = lo == low ? n - excess : n;
      const uint32_t i0 = 2 * threadIdx.x, i1 = i0 + 1;
      const uint64_t v0 = i0 < m ? value(listed_score(s.list[i0])) : 0, v1 = i1 < m ? value(listed_score(s.list[i1])) : 0;
      uint64_t total;
      const uint64_t e = before + block_scan(v0 + v1, s, &total);
      if (e <= unit && unit < e + v0) s.found = i0;
      if (e + v0 <= unit && unit < e + v0 + v1) s.found = i1;
      __syncthreads();
      const uint32_t f = s.found;
      p.z = listed_score(s.list[f]);
      p.column = (uint32_t)s.list[f];
      // its equals in the list before it
      uint32_t first = f;
      while (first && listed_score(s.list[first - 1]) == p.z) --first;
      p.tie = f - first;
      if (f >> 1 == threadIdx.x) s.before = e + (f & 1 ? v0 : 0);
      __syncthreads();
      p.before = s.before - (uint64_t)p.tie * value(p.z);
      return p;
    }
  }
}

// How many entries satisfy f(score).
template <typename T, typename F>
__device__ uint32_t count_if(const Sweep<T>& sweep, Shared& s, F f) {
  uint64_t mine = 0, total;
  sweep([&](float z, uint32_t) { mine += f(z) ? 1 : 0; });
  block_scan(mine, s, &total);
  return (uint32_t)total;
}

// The column of entry `tie` among those of value z, by column.
template <typename T>
__device__ uint32_t column_of_tie(const T* x, uint32_t columns, Shared& s, float z, uint32_t tie) {
  uint64_t seen = 0;
  if (threadIdx.x == 0) s.found2 = 0xFFFFFFFFu;
  for (uint32_t base = 0; base < columns; base += THREADS) {
    const uint32_t c = base + threadIdx.x;
    const uint64_t here = c < columns && plain_score((float)x[c]) == z;
    uint64_t total;
    const uint64_t before = seen + block_scan(here, s, &total);
    if (here && before == tie) s.found2 = c;
    seen += total;
    if (seen > tie) break;
  }
  __syncthreads();
  return s.found2;
}

template <typename T>
__device__ Result draw_row(const T* x, uint32_t columns, Shared& s, float temperature, uint32_t top_k, float top_p, float min_p, double u) {
  const Sweep<T> sweep{x, columns};
  // the largest and the smallest value, and how many there are
  uint32_t kmin = 0xFFFFFFFFu, kmax = 0, there = 0;
  sweep([&](float z, uint32_t) {
    const uint32_t key = score_key(z);
    const bool in = z > -__builtin_inff();
    kmin = in ? min(kmin, key) : kmin;
    kmax = in ? max(kmax, key) : kmax;
    there += in;
  });
  if (threadIdx.x == 0) {
    s.lo = 0xFFFFFFFFu;
    s.hi = 0;
    s.n = 0;
  }
  uint64_t many;
  block_scan(there, s, &many);
  kmin = wave_min_u32(kmin);
  kmax = wave_max_u32(kmax);
  if ((threadIdx.x & 63) == 0) {
    atomicMin(&s.lo, kmin);
    atomicMax(&s.hi, kmax);
  }
  __syncthreads();
  const uint32_t n = (uint32_t)many;
  Result r{SKY_INVALID, 0, -__builtin_inf()};
  if (!n) return r;
  Row row;
  row.zmax = key_score(s.hi);
  const float zmin = key_score(s.lo);
  if (!(temperature > 0.0f)) {
    const float zmax = row.zmax;
    r.token = column_of_tie(x, columns, s, zmax, 0);
    r.kept = 1;
    r.logprob = 0.0;
    return r;
  }
  row.t = temperature;
  row.S = 61 - (31 - __clz((int)columns));
  const double t = row.t;
  if (n <= CAP) {
    sweep([&](float z, uint32_t c) {
      if (z > -__builtin_inff()) s.list[atomicAdd(&s.n, 1u)] = (uint64_t)~score_key(z) << 32 | c;
    });
    __syncthreads();
    return draw_listed(s, n, t, top_k, top_p, min_p, u);
  }
  // Entries below `low` weigh nothing.  What stays is the beginning of the order that ends with `count` entries, the last of
  // them of value `low`, of which the last `excess` do not belong to it.
  float low = zmin;
  uint32_t excess = 0, count = n;
  const double cut = (double)row.zmax - NO_MASS * t;
  bool cut_off = false;
  if (top_k && top_k < n) {
    const Place p = locate<true>(sweep, s, row, zmin, 0, top_k - 1);
    low = p.z;
    count = top_k;
    excess = count_if(sweep, s, [&](float z) { return z == low; }) - (p.tie + 1);
    if (top_k <= CAP - 64 && excess <= 64) {  // few: listed and sorted at once
      __syncthreads();
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
      sweep([&](float z, uint32_t c) {
        if (z >= low) s.list[atomicAdd(&s.n, 1u)] = (uint64_t)~score_key(z) << 32 | c;
      });
      __syncthreads();
      return draw_listed(s, top_k + excess, t, top_k, top_p, min_p, u);
    }
  }
  if ((double)low < cut) {
    // the smallest value that has mass: entries below it matter for the count alone
    if (threadIdx.x == 0) s.lo = 0xFFFFFFFFu;
    __syncthreads();
    uint32_t k = 0xFFFFFFFFu;
    sweep([&](float z, uint32_t) {
      if ((double)z >= cut) k = min(k, score_key(z));
    });
    k = wave_min_u32(k);
    if ((threadIdx.x & 63) == 0) atomicMin(&s.lo, k);
    __syncthreads();
    low = key_score(s.lo);
    excess = 0;
    cut_off = true;
    __syncthreads();
  }
  auto mass_from = [&](float z0, uint32_t less) {  // what the entries from z0 on weigh, without `less` of z0's
    uint64_t mine = 0, total;
    sweep([&](float z, uint32_t) {
      if (z >= z0) mine += mass_of(weight_of(z, row.zmax, t), row.S);
    });
    block_scan(mine, s, &total);
    return total - (uint64_t)less * mass_of(weight_of(z0, row.zmax, t), row.S);
  };
  uint64_t mass = mass_from(low, excess);
  float end = low;  // of what stays, for the filters below
  if (top_p < 1.0f) {
    const uint64_t need = max((uint64_t)ceil(fmax((double)top_p, 0.0) * (double)mass), (uint64_t)1);
    const Place p = locate<false>(sweep, s, row, low, excess, min(need, mass) - 1);
    mass = p.before + (uint64_t)(p.tie + 1) * mass_of(weight_of(p.z, row.zmax, t), row.S);
    end = p.z;
    count = count_if(sweep, s, [&](float z) { return z > end; }) + p.tie + 1;
  }
  if (min_p > 0.0f && (weight_of(end, row.zmax, t) < (double)min_p || (cut_off && !(top_p < 1.0f)))) {
    uint64_t mine = 0, in = 0, all, many_in;
    sweep([&](float z, uint32_t) {
      const double w = z > -__builtin_inff() ? weight_of(z, row.zmax, t) : -1.0;
      if (w >= (double)min_p || z == row.zmax) {
        mine += mass_of(w, row.S);
        ++in;
      }
    });
    block_scan(mine, s, &all);
    block_scan(in, s, &many_in);
    if (many_in < count) {
      mass = all;
      count = (uint32_t)many_in;
    }
  }
  uint64_t unit = (uint64_t)(u * (double)mass);
  if (unit >= mass) unit = mass - 1;
  const Place p = locate<false>(sweep, s, row, low, excess, unit);
  r.token = p.column != 0xFFFFFFFFu ? p.column : column_of_tie(x, columns, s, p.z, p.tie);
  r.kept = count;
  r.logprob = ((double)p.z - (double)row.zmax) / t - log(ldexp((double)mass, -row.S));
  return r;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void draw_kernel(DrawArgs a) {
  __shared__ Shared s;
  const uint32_t r = blockIdx.x;
  double u;
  if (a.uniforms) {
    u = fmax(a.uniforms[r], 0.0);
  } else {
    const u32x4 bits = philox(a.seed, a.first_walker + r, a.step, 0, DOM_LOGITS);
    u = ((double)(bits.x >> 5) * 67108864.0 + (double)(bits.y >> 6)) * (1.0 / 9007199254740992.0);
  }
  float top_p = a.top_p ? a.top_p[r] : 1.0f;
  if (!(top_p < 1.0f)) top_p = 1.0f;
  const Result d = draw_row((const T*)a.logits + r * a.stride, a.columns, s, a.temperature ? a.temperature[r] : 1.0f,
                            a.top_k ? a.top_k[r] : 0u, top_p, a.min_p ? a.min_p[r] : 0.0f, u);
  if (threadIdx.x == 0) {
    a.tokens[r * a.tokens_stride] = d.token;
    if (a.logprobs) a.logprobs[r] = (float)d.logprob;
    if (a.kept) a.kept[r] = d.kept;
  }
}

}  // namespace
}  // namespace sky

using namespace sky;

extern "C" int sky_logits_draw_workspace(int dtype, uint32_t rows, uint32_t columns, uint64_t* bytes) {
  uint64_t stride = 0;
  if (!bytes) return fail(SKY_ERR_ARG, "sky_logits_draw_workspace: null output");
  SKY_TRY(check_rows("sky_logits_draw_workspace", "logits", bytes, dtype, rows, columns, &stride));
  *bytes = 0;
  return SKY_OK;
}

extern "C" int sky_logits_draw(const void* logits, int dtype, uint32_t rows, uint32_t columns, uint64_t row_stride,
                               const sky_draw_rules* rules, const double* uniforms, uint64_t philox_seed, uint32_t first_walker,
                               uint32_t step, uint32_t* tokens, uint64_t tokens_stride, float* logprobs, uint32_t* kept,
                               void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* const who = "sky_logits_draw";
  SKY_TRY(check_rows(who, "logits", logits, dtype, rows, columns, &row_stride));
  if (!tokens && rows) return fail(SKY_ERR_ARG, "sky_logits_draw: tokens is null");
  uint64_t want = 0;
  SKY_TRY(sky_logits_draw_workspace(dtype, rows, columns, &want));
  if (workspace && workspace_bytes < want) return fail(SKY_ERR_ARG, "sky_logits_draw: the workspace is too small");
  SKY_TRY(check_aligned(who, "workspace", workspace, 16));
  const sky_draw_rules d = rules ? *rules : sky_draw_rules{};
  const struct {
    const char* name;
    const void* p;
    size_t size;
  } arrays[] = {{"temperature", d.temperature, 4}, {"top_k", d.top_k, 4},   {"top_p", d.top_p, 4},     {"min_p", d.min_p, 4},
                {"uniforms", uniforms, 8},         {"tokens", tokens, 4}, {"logprobs", logprobs, 4}, {"kept", kept, 4}};
  for (const auto& x : arrays) SKY_TRY(check_aligned(who, x.name, x.p, x.size));
  if (!rows) return SKY_OK;
  SKY_TRY(ensure_device());
  const DrawArgs a{logits, row_stride,  columns,      rows, d.temperature, d.top_k,       d.top_p,  d.min_p,
                   uniforms, philox_seed, first_walker, step, tokens,        tokens_stride ? tokens_stride : 1, logprobs, kept};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == SKY_F32)
    hipLaunchKernelGGL(draw_kernel<float>, dim3(rows), dim3(THREADS), 0, st, a);
  else if (dtype == SKY_F16)
    hipLaunchKernelGGL(draw_kernel<_Float16>, dim3(rows), dim3(THREADS), 0, st, a);
  else
    hipLaunchKernelGGL(draw_kernel<__bf16>, dim3(rows), dim3(THREADS), 0, st, a);
  return check_launch();
}
