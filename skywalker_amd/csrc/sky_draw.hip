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
// Two shorter ways take most rows.  Where at most CAP entries can stay (a grammar's rows; top-k of up to SMALL_K: the k-th
// largest of the threads' largest entries is no larger than the k-th largest entry; min-p without top-p) they are listed and sorted
// at once.  And 16-bit logits have no more than 65,536 values: they are counted by value, in 16-bit counters that take
// 128 KB of LDS, and everything else (weights, prefixes, borders) is a matter of the values that occur, a few thousand.
//
// Weights are summed in whole numbers (2^-S of the largest weight, S = 61 less the bits of the row's length, 50 at most): sums then do
// not depend on the order of LDS atomics or of lanes.  They are rounded once each, by at most 2^-(S+1) of the largest weight; the
// exponential is taken in fp64, since an id changes with the last bit that its border of the sum is off by.
#include "sky_scores.h"

namespace sky {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr uint32_t BINS = 2048;  // two per thread
constexpr uint32_t CAP = 2048;   // entries of a list, two per thread
constexpr double NO_MASS = 40.0;  // weights below e^-40 are 0 in units of 2^-S, S <= 50
constexpr uint32_t SMALL_K = 512;  // of the 1024 threads' largest entries: some 710 entries are as large as the 512th of them
constexpr uint32_t VALUES = 65536, CHUNK = 64, CHUNKS = VALUES / CHUNK;  // of 16-bit logits; a wavefront takes a chunk

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

// What a row of 16-bit logits comes to by value.
struct Counters {
  uint32_t value[VALUES / 2];  // places below 32,768 in the low halves, the others in the high ones
  uint32_t chunk_count[CHUNKS];
  uint64_t chunk_mass[CHUNKS];
};
// LDS of a workgroup, which has a CU to itself (its registers see to that as well).
struct Shared {
  union {
    struct {
      uint64_t bin[BINS];   // counts or sums
      uint64_t list[CAP];   // (~key << 32 | column), ascending is the order
    };
    Counters counters;
  };
  uint64_t wave[WAVES + 1];
  uint32_t n;
  uint32_t lo, hi;  // keys
  uint32_t found, found2;
  uint64_t before;
  uint32_t most[THREADS];
  uint32_t wave_most[WAVES], wave_there[WAVES], wave_above[WAVES];
  uint32_t place, chunk;
  uint64_t count_before, mass_before;
};
static_assert(sizeof(Shared) <= 160 * 1024, "LDS of a CU");

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp0<DPP_QUAD_XOR1, 0xF>(v));
  v = max(v, dpp0<DPP_QUAD_XOR2, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_HALF_MIRROR, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_MIRROR, 0xF>(v));
  v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
}

// 2^x of a double x in [-61, 0] times 2^S, rounded to a whole number (S <= 50: below 2^51): the polynomial is the series of
// e^(x ln 2) on [-1/2, 1/2] through degree 11, whose next term is 6e-15.
__device__ __forceinline__ uint64_t power_units(double x, int S) {
  const double n = rint(x), f = (x - n) * 0.69314718055994530942;
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
  // p lies in [0.7, 1.42): its exponent takes n + S >= -31 without leaving the normal numbers; 2^52 leaves the rounded integer in the low bits
  const uint64_t scaled = (uint64_t)__double_as_longlong(p) + ((uint64_t)(int64_t)((int)n + S) << 52);
  return (uint64_t)__double_as_longlong(__longlong_as_double((long long)scaled) + 4503599627370496.0) - 0x4330000000000000ull;
}
// What weights of a row need.
struct Row {
  double t;      // temperature
  double per;    // log2(e) / t
  float zmax;
  int S;         // fraction bits of a weight
  __device__ __forceinline__ Row(double temperature, float z, int s) : t(temperature), per(1.44269504088896340736 / temperature), zmax(z), S(s) {}
  __device__ __forceinline__ double weight(float z) const { return exp(((double)z - (double)zmax) / t); }
  __device__ __forceinline__ uint64_t units(float z) const {
    const double x = ((double)z - (double)zmax) * per;
    return x >= -60.0 ? power_units(x, S) : 0;
  }
  // the logarithm of z's share of `mass` units
  __device__ __forceinline__ double log_share(float z, uint64_t mass) const {
    return ((double)z - (double)zmax) / t - log(ldexp((double)mass, -S));
  }
};

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
#pragma unroll 1
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
  sort_list(s, m);
  const Row row(t, listed_score(s.list[0]), 50);  // at most 2^11 weights
  const uint32_t k = top_k && top_k < m ? top_k : m;
  const uint32_t i0 = 2 * threadIdx.x, i1 = i0 + 1;
  const float z0 = i0 < k ? listed_score(s.list[i0]) : row.zmax, z1 = i1 < k ? listed_score(s.list[i1]) : row.zmax;
  const uint64_t m0 = i0 < k ? row.units(z0) : 0, m1 = i1 < k ? row.units(z1) : 0;
  uint64_t total;
  const uint64_t before = block_scan(m0 + m1, s, &total);
  uint32_t n = k;
  if (top_p < 1.0f || min_p > 0.0f) {
    // entries stay while what comes before them is below p of the total, and their weight at least min_p
    const uint64_t need = top_p < 1.0f ? (uint64_t)ceil(fmax((double)top_p, 0.0) * (double)total) : ~0ull;
    const bool in0 = i0 < k && (i0 == 0 || (before < need && (!(min_p > 0.0f) || row.weight(z0) >= (double)min_p)));
    const bool in1 = i1 < k && before + m0 < need && (!(min_p > 0.0f) || row.weight(z1) >= (double)min_p);
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
  r.logprob = row.log_share(listed_score(e), mass);
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
  auto value = [&](float z) -> uint64_t { return RANK ? 1ull : row.units(z); };
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

__device__ __forceinline__ int fraction_bits(uint32_t columns) { return min(50, 61 - (31 - __clz((int)columns))); }

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
__device__ __forceinline__ Result draw_any_row(const T* x, uint32_t columns, Shared& s, float temperature, uint32_t top_k, float top_p, float min_p, double u) {
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
  const Row row(temperature, key_score(s.hi), fraction_bits(columns));
  const float zmin = key_score(s.lo);
  if (!(temperature > 0.0f)) {
    const float zmax = row.zmax;
    r.token = column_of_tie(x, columns, s, zmax, 0);
    r.kept = 1;
    r.logprob = 0.0;
    return r;
  }
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
    __syncthreads();  // every thread has read the smallest value of all
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
      if (z >= z0) mine += row.units(z);
    });
    block_scan(mine, s, &total);
    return total - (uint64_t)less * row.units(z0);
  };
  uint64_t mass = mass_from(low, excess);
  float end = low;  // of what stays, for the filters below
  if (top_p < 1.0f) {
    const uint64_t need = max((uint64_t)ceil(fmax((double)top_p, 0.0) * (double)mass), (uint64_t)1);
    const Place p = locate<false>(sweep, s, row, low, excess, min(need, mass) - 1);
    mass = p.before + (uint64_t)(p.tie + 1) * row.units(p.z);
    end = p.z;
    count = count_if(sweep, s, [&](float z) { return z > end; }) + p.tie + 1;
  }
  if (min_p > 0.0f && (row.weight(end) < (double)min_p || (cut_off && !(top_p < 1.0f)))) {
    uint64_t mine = 0, in = 0, all, many_in;
    sweep([&](float z, uint32_t) {
      const double w = z > -__builtin_inff() ? row.weight(z) : -1.0;
      if (w >= (double)min_p || z == row.zmax) {
        mine += row.units(z);
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
  r.logprob = row.log_share(p.z, mass);
  return r;
}

// ---------------------------------------------------------------- rows held in registers
// The place of a value: a whole number that ascends with it, turned so that what is not there (NaN, -inf) comes first. +inf is the
// largest finite number and -0 is 0.
template <typename T>
struct Places;
template <>
struct Places<float> {
  static constexpr uint32_t NOTHING = 0xFFFFFEu, TURN = 0x7FFFFFu;  // up to NOTHING: not there
  static __device__ __forceinline__ float value(uint32_t q) { return key_score(q - TURN); }
  static __device__ __forceinline__ uint32_t of(float z) { return score_key(z) + TURN; }  // of a finite z
};
template <>
struct Places<_Float16> {
  static constexpr uint32_t NOTHING = 0x7FEu, LOWEST = 0x7FFu, TURN = 0x3FFu;
  static __device__ __forceinline__ float value(uint32_t q) {
    const uint32_t k = q - TURN;
    const uint16_t bits = (uint16_t)(k ^ (k & 0x8000u ? 0x8000u : 0xFFFFu));
    return (float)__builtin_bit_cast(_Float16, bits);
  }
};
template <>
struct Places<__bf16> {
  static constexpr uint32_t NOTHING = 0xFEu, LOWEST = 0xFFu, TURN = 0x7Fu;
  static __device__ __forceinline__ float value(uint32_t q) {
    const uint32_t k = q - TURN;
    return __uint_as_float(((k ^ (k & 0x8000u ? 0x8000u : 0xFFFFu)) & 0xFFFFu) << 16);
  }
};
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

// NV pieces a thread, and an entry more of those that do not fill a piece: all of a row of at most THREADS * NV * 16 bytes, as places.
template <typename T, int NV>
struct Held {
  static constexpr int N = Piece<T>::N, WORDS = NV * 4 + 1;
  uint32_t q[WORDS];  // a 32-bit place, or two 16-bit places
  uint32_t last;      // column of the last word's entry
  static __device__ __forceinline__ uint32_t column(int i) { return (i * THREADS + threadIdx.x) * N; }

  __device__ __forceinline__ void load(const T* x, uint32_t columns) {
    constexpr uint32_t gone = sizeof(T) == 4 ? 0xFF800000u : __is_same(T, _Float16) ? 0xFC00FC00u : 0xFF80FF80u;  // -inf
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = column(i);
      if (c + N <= columns) {
        __builtin_memcpy(&q[4 * i], x + c, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[4 * i + e] = gone;
      }
    }
    last = columns / N * N + threadIdx.x;
    q[4 * NV] = gone;
    if (last < columns) {
      if constexpr (sizeof(T) == 4)
        q[4 * NV] = __float_as_uint(x[last]);
      else
        q[4 * NV] = (gone & 0xFFFF0000u) | __builtin_bit_cast(uint16_t, x[last]);
    }
  }
  // Bits into places; the largest of the thread, how many are there and how many of them are above the lowest value.
  __device__ __forceinline__ void settle(uint32_t* most, uint32_t* there, uint32_t* above) {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0, n = 0;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // as the pieces arrive; started all at once they would not fit
        const uint32_t b = __float_as_uint(__uint_as_float(q[i]) + 0.0f);
        q[i] = min((b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) + Places<T>::TURN, 0xFFFFFFFEu);
        m = max(m, q[i]);
        n += q[i] > Places<T>::NOTHING;
      }
      *most = m;
      *there = n;
      *above = n;
    } else {
      constexpr uint16_t turn = Places<T>::TURN, nothing = Places<T>::NOTHING, lowest = Places<T>::LOWEST;
      const u16x2 one = {1, 1};
      u16x2 m = {0, 0}, n = {0, 0}, l = {0, 0};
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
        u16x2 v = __builtin_bit_cast(u16x2, q[i]);
        const u16x2 some = __builtin_elementwise_min(v & (uint16_t)0x7FFF, one);
        v &= (u16x2)(-some);  // -0 is 0
        const u16x2 sign = __builtin_bit_cast(u16x2, __builtin_bit_cast(i16x2, v) >> (int16_t)15);
        v = (v ^ (sign | (uint16_t)0x8000)) + turn;
        v = __builtin_elementwise_min(v, u16x2{0xFFFE, 0xFFFE});
        q[i] = __builtin_bit_cast(uint32_t, v);
        m = __builtin_elementwise_max(m, v);
        n += __builtin_elementwise_min(__builtin_elementwise_sub_sat(v, u16x2{nothing, nothing}), one);
        l += __builtin_elementwise_min(__builtin_elementwise_sub_sat(v, u16x2{lowest, lowest}), one);
      }
      *most = max((uint32_t)m.x, (uint32_t)m.y);
      *there = (uint32_t)n.x + n.y;
      *above = (uint32_t)l.x + l.y;
    }
  }
  // f(place) for every entry, and for what is not there
  template <typename F>
  __device__ __forceinline__ void sweep(F f) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if (i % 8 == 0) __builtin_amdgcn_sched_barrier(0);  // the words are taken as they come: mixed, they would not fit beside one another
      if constexpr (sizeof(T) == 4) {
        f(q[i]);
      } else {
        f(q[i] & 0xFFFFu);
        f(q[i] >> 16);
      }
    }
  }
  // f(place, column) for the entries that are wanted, which are few: a piece is taken apart, in a loop that all pieces' code is
  // short for, only if any_of(its four words) says that one of them may be
  template <typename A, typename F>
  __device__ __forceinline__ void pick(A any_of, F f) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t a = q[4 * i], b = q[4 * i + 1], c = q[4 * i + 2], d = q[4 * i + 3];
      if (any_of(a, b, c, d)) {
#pragma unroll 1
        for (int e = 0; e < N; ++e) {
          if constexpr (sizeof(T) == 4) {
            f(a, column(i) + e);
            a = b;
            b = c;
            c = d;
          } else {
            f(a & 0xFFFFu, column(i) + e);
            a = __builtin_amdgcn_alignbit(b, a, 16);
            b = __builtin_amdgcn_alignbit(c, b, 16);
            c = __builtin_amdgcn_alignbit(d, c, 16);
            d >>= 16;
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    f(sizeof(T) == 4 ? q[4 * NV] : q[4 * NV] & 0xFFFFu, last);
  }
  template <typename F>
  __device__ __forceinline__ void from(uint32_t least, F f) const {
    pick([&](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      if constexpr (sizeof(T) == 4) {
        return max(max(a, b), max(c, d)) >= least;
      } else {
        auto v = [](uint32_t x) { return __builtin_bit_cast(u16x2, x); };
        const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(v(a), v(b)), __builtin_elementwise_max(v(c), v(d)));
        return max((uint32_t)m.x, (uint32_t)m.y) >= least;
      }
    }, [&](uint32_t x, uint32_t c) { if (x >= least) f(x, c); });
  }
  template <typename F>
  __device__ __forceinline__ void equal(uint32_t value, F f) const {
    pick([&](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      if constexpr (sizeof(T) == 4) {
        return a == value || b == value || c == value || d == value;
      } else {
        const uint32_t both = value | value << 16;
        auto v = [&](uint32_t x) { return __builtin_bit_cast(u16x2, x ^ both); };
        const u16x2 m = __builtin_elementwise_min(__builtin_elementwise_min(v(a), v(b)), __builtin_elementwise_min(v(c), v(d)));
        return min((uint32_t)m.x, (uint32_t)m.y) == 0;
      }
    }, [&](uint32_t x, uint32_t c) { if (x == value) f(c); });
  }
};

// One chunk of values, the largest first: lane l has its l-th largest.
struct Chunk {
  uint32_t q, count;
  float z;
  uint64_t mass;
};
template <typename T>
__device__ __forceinline__ Chunk chunk_of(const Counters& c, uint32_t chunk, const Row& row) {
  Chunk r;
  r.q = chunk * CHUNK + (CHUNK - 1) - (threadIdx.x & 63);
  const uint32_t both = c.value[r.q & 0x7FFFu];
  r.count = r.q & 0x8000u ? both >> 16 : both & 0xFFFFu;
  r.z = r.count ? Places<T>::value(r.q) : row.zmax;
  r.mass = r.count ? r.count * row.units(r.z) : 0;
  return r;
}
// The value that holds a unit (RANK: of the count; else of mass), from the sums of chunks before each thread's own (thread t has the
// t-th chunk from the top).
struct ValuePlace {
  uint32_t q, tie;
  float z;
  uint64_t count_before, mass_before;  // of the value
};
template <bool RANK, typename T>
__device__ ValuePlace locate_value(Shared& s, const Row& row, uint64_t unit, uint64_t count_before, uint64_t mass_before) {
  const uint32_t mine = CHUNKS - 1 - threadIdx.x;
  const uint64_t before = RANK ? count_before : mass_before;
  const uint64_t here = RANK ? (uint64_t)s.counters.chunk_count[mine] : s.counters.chunk_mass[mine];
  __syncthreads();
  if (before <= unit && unit < before + here) {
    s.chunk = mine;
    s.count_before = count_before;
    s.mass_before = mass_before;
  }
  __syncthreads();
  const Chunk k = chunk_of<T>(s.counters, s.chunk, row);
  const uint64_t counts = s.count_before + group_scan_u64<64>(k.count) - k.count;
  const uint64_t masses = s.mass_before + group_scan_u64<64>(k.mass) - k.mass;
  const uint64_t start = RANK ? counts : masses, size = RANK ? (uint64_t)k.count : k.mass;
  const int lane = (int)__builtin_ctzll(__ballot(start <= unit && unit < start + size) | 1ull << 63);
  ValuePlace p;
  p.q = (uint32_t)__shfl((int)k.q, lane, 64);
  p.z = __shfl(k.z, lane, 64);
  p.count_before = shfl_u64(counts, lane);
  p.mass_before = shfl_u64(masses, lane);
  const uint64_t each = RANK ? 1 : row.units(p.z);
  p.tie = (uint32_t)((unit - (RANK ? p.count_before : p.mass_before)) / each);
  return p;
}

template <typename T, int NV>
__device__ __forceinline__ uint32_t held_column(const Held<T, NV>& held, const T* x, uint32_t columns, Shared& s, uint32_t* room, uint32_t q, uint32_t tie, uint32_t ties) {
  // the columns of the value, listed in CAP words; the one with `tie` of them before it
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  if (ties > CAP) return column_of_tie(x, columns, s, Places<T>::value(q), tie);
  uint32_t* const list = room;
  held.equal(q, [&](uint32_t c) { list[atomicAdd(&s.n, 1u)] = c; });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < ties; i += THREADS) {
    uint32_t below = 0;
    const uint32_t c = list[i];
    for (uint32_t j = 0; j < ties; ++j) below += list[j] < c;
    if (below == tie) s.found2 = c;
  }
  __syncthreads();
  return s.found2;
}

template <typename T, int NV>
__device__ __forceinline__ Result draw_held_row(const T* x, uint32_t columns, Shared& s, float temperature, uint32_t top_k,
                                                float top_p, float min_p, double u) {
  using P = Places<T>;
  Counters* const c = &s.counters;
  constexpr bool BY_VALUE = sizeof(T) == 2;
  Held<T, NV> held;
  held.load(x, columns);
  const bool greedy = !(temperature > 0.0f);
  const bool few = (top_k && top_k <= SMALL_K) || (min_p > 0.0f && !(top_p < 1.0f)) || greedy;  // few entries can stay
  if constexpr (BY_VALUE)
    if (!few)
      for (uint32_t i = threadIdx.x; i < VALUES / 8; i += THREADS) ((uint4*)c->value)[i] = uint4{0, 0, 0, 0};
  uint32_t most, there, above;
  held.settle(&most, &there, &above);
  {
    const uint32_t w = threadIdx.x >> 6;
    const uint32_t m = wave_max_u32(most), n = group_scan_u32<64>(there), l = group_scan_u32<64>(above);
    s.most[threadIdx.x] = most;
    if ((threadIdx.x & 63) == 63) {
      s.wave_most[w] = m;
      s.wave_there[w] = n;
      s.wave_above[w] = l;
    }
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    most = there = above = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      most = max(most, s.wave_most[i]);
      there += s.wave_there[i];
      above += s.wave_above[i];
    }
  }
  Result r{SKY_INVALID, 0, -__builtin_inf()};
  if (!there) return r;
  if (greedy) {
    uint32_t first = 0xFFFFFFFFu;
    held.equal(most, [&](uint32_t col) { first = min(first, col); });
    first = wave_min_u32(first);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave_most[threadIdx.x >> 6] = first;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) first = min(first, s.wave_most[i]);
    r.token = first;
    r.kept = 1;
    r.logprob = 0.0;
    return r;
  }
  const Row row(temperature, P::value(most), fraction_bits(columns));
  uint32_t from = P::NOTHING + 1;  // places from here on are listed
  bool listed = there <= CAP;
  if (!listed && few) {
    if (top_k && top_k <= SMALL_K) {
      // the top_k-th largest of the threads' largest: at least top_k entries are as large
      if (threadIdx.x < 64) {
        uint32_t v[THREADS / 64], lo = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) v[i] = s.most[64 * i + threadIdx.x];
        for (uint32_t bit = sizeof(T) == 4 ? 0x80000000u : 0x8000u; bit; bit >>= 1) {
          uint32_t n = 0;
#pragma unroll
          for (int i = 0; i < THREADS / 64; ++i) n += (uint32_t)__builtin_popcountll(__ballot(v[i] >= (lo | bit)));
          if (n >= top_k) lo |= bit;
        }
        if (threadIdx.x == 0) s.place = lo;
      }
      __syncthreads();
      from = max(from, s.place);
    }
    if (min_p > 0.0f && !(top_p < 1.0f)) {
      // the smallest value that may weigh min_p, with a margin for the logarithm
      const double z = (double)row.zmax + row.t * (log((double)min_p) - 1e-6) - 1e-6 * fabs((double)row.zmax);
      uint32_t lo = 0;
      for (uint32_t bit = sizeof(T) == 4 ? 0x80000000u : 0x8000u; bit; bit >>= 1)
        if ((lo | bit) <= most && ((lo | bit) <= P::NOTHING || (double)P::value(lo | bit) <= z)) lo |= bit;
      from = max(from, lo);
    }
    listed = true;
  }
  if (listed) {
    held.from(from, [&](uint32_t q, uint32_t col) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < CAP) s.list[at] = (uint64_t)~score_key(P::value(q)) << 32 | col;
    });
    __syncthreads();
    const uint32_t n = s.n;
    if (n <= CAP) return draw_listed(s, n, row.t, top_k, top_p, min_p, u);
    __syncthreads();
  }
  if constexpr (BY_VALUE) {
    // values below `cut` weigh nothing; the lowest value of the type, which masks are made of, is not counted by value
    uint32_t cut = 0;
    {
      const double z = (double)row.zmax - NO_MASS * row.t;
      for (uint32_t bit = 0x8000u; bit; bit >>= 1)
        if (((cut | bit) <= P::NOTHING) || ((cut | bit) <= most && (double)P::value((cut | bit)) < z)) cut |= bit;
    }
    if (few) {  // the counters were not cleared above
      for (uint32_t i = threadIdx.x; i < VALUES / 8; i += THREADS) ((uint4*)c->value)[i] = uint4{0, 0, 0, 0};
      __syncthreads();
    }
    if (cut >= P::LOWEST || there == above) {
      held.sweep([&](uint32_t q) {
        if (q > P::LOWEST) atomicAdd(&c->value[q & 0x7FFFu], q & 0x8000u ? 0x10000u : 1u);
      });
      __syncthreads();
      const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
      // a wavefront takes every 16th chunk
      for (uint32_t i = wave; i < CHUNKS; i += WAVES) {
        const uint32_t chunk = CHUNKS - 1 - i;
        uint64_t mass = 0;
        uint32_t count = 0;
        const uint32_t q = chunk * CHUNK + lane, both = c->value[q & 0x7FFFu];
        const uint32_t n = q & 0x8000u ? both >> 16 : both & 0xFFFFu;
        if (__ballot(n != 0)) {
          count = group_scan_u32<64>(n);
          if (chunk * CHUNK + CHUNK > cut) mass = group_scan_u64<64>(n ? n * row.units(P::value(q)) : 0);
        }
        if (lane == 63) {
          c->chunk_count[chunk] = count;
          c->chunk_mass[chunk] = mass;
        }
      }
      __syncthreads();
      uint64_t counted, mass;
      const uint32_t mine = CHUNKS - 1 - threadIdx.x;
      const uint64_t count_before = block_scan(c->chunk_count[mine], s, &counted);
      const uint64_t mass_before = block_scan(c->chunk_mass[mine], s, &mass);
      if (counted == above) {  // no counter has run over
        uint32_t count = there;
        if (top_k && top_k < there) {
          count = top_k;
          if (top_k < above) {
            const ValuePlace p = locate_value<true, T>(s, row, top_k - 1, count_before, mass_before);
            mass = p.mass_before + (uint64_t)(p.tie + 1) * row.units(p.z);
          }
        }
        if (top_p < 1.0f) {
          const uint64_t need = max((uint64_t)ceil(fmax((double)top_p, 0.0) * (double)mass), (uint64_t)1);
          const ValuePlace p = locate_value<false, T>(s, row, min(need, mass) - 1, count_before, mass_before);
          mass = p.mass_before + (uint64_t)(p.tie + 1) * row.units(p.z);
          count = (uint32_t)p.count_before + p.tie + 1;
        }
        if (min_p > 0.0f) {
          // the smallest value that weighs min_p
          uint32_t lo = 0;
          for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
            const uint32_t q = lo | bit;
            if (q <= most && (q <= P::NOTHING || !(row.weight(P::value(q)) >= (double)min_p))) lo = q;
          }
          // `lo` is the last value that does not (or the largest value itself, which always stays)
          const uint32_t least = min(lo + 1, most), chunk = least / CHUNK;
          __syncthreads();
          if (mine == chunk) {
            s.count_before = count_before;
            s.mass_before = mass_before;
          }
          __syncthreads();
          const Chunk k = chunk_of<T>(*c, chunk, row);
          const uint64_t in = s.count_before + shfl_u64(group_scan_u64<64>(k.q >= least ? k.count : 0), 63);
          const uint64_t weighs = s.mass_before + shfl_u64(group_scan_u64<64>(k.q >= least ? k.mass : 0), 63);
          if (least <= P::LOWEST ? there < count : in < count) {
            count = least <= P::LOWEST ? there : (uint32_t)in;
            mass = weighs;
          }
        }
        uint64_t unit = (uint64_t)(u * (double)mass);
        if (unit >= mass) unit = mass - 1;
        const ValuePlace p = locate_value<false, T>(s, row, unit, count_before, mass_before);
        const uint32_t both = c->value[p.q & 0x7FFFu];
        static_assert(sizeof(c->chunk_mass) == CAP * 4, "the sums of chunks, which nobody reads any more, make room for the list");
        r.token = held_column(held, x, columns, s, (uint32_t*)c->chunk_mass, p.q, p.tie, p.q & 0x8000u ? both >> 16 : both & 0xFFFFu);
        r.kept = count;
        r.logprob = row.log_share(p.z, mass);
        return r;
      }
    }
    __syncthreads();
  }
  return draw_any_row(x, columns, s, temperature, top_k, top_p, min_p, u);
}

// NV = 0: a row that registers do not hold
template <typename T, int NV>
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
  const float temperature = a.temperature ? a.temperature[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const uint32_t top_k = a.top_k ? a.top_k[r] : 0u;
  float top_p = a.top_p ? a.top_p[r] : 1.0f;
  if (!(top_p < 1.0f)) top_p = 1.0f;
  const T* const x = (const T*)a.logits + r * a.stride;
  Result d;
  if constexpr (NV == 0)
    d = draw_any_row(x, a.columns, s, temperature, top_k, top_p, min_p, u);
  else
    d = draw_held_row<T, NV>(x, a.columns, s, temperature, top_k, top_p, min_p, u);
  if (threadIdx.x == 0) {
    a.tokens[r * a.tokens_stride] = d.token;
    if (a.logprobs) a.logprobs[r] = (float)d.logprob;
    if (a.kept) a.kept[r] = d.kept;
  }
}

template <typename T>
void launch_draw(const DrawArgs& a, hipStream_t st) {
  constexpr uint32_t N = THREADS * Piece<T>::N;
  const dim3 grid(a.rows), block(THREADS);
  if (a.columns <= 2 * N)
    hipLaunchKernelGGL((draw_kernel<T, 2>), grid, block, 0, st, a);
  else if (a.columns <= 8 * N)
    hipLaunchKernelGGL((draw_kernel<T, 8>), grid, block, 0, st, a);
  else if (a.columns <= 16 * N)
    hipLaunchKernelGGL((draw_kernel<T, 16>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((draw_kernel<T, 0>), grid, block, 0, st, a);
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
    launch_draw<float>(a, st);
  else if (dtype == SKY_F16)
    launch_draw<_Float16>(a, st);
  else
    launch_draw<__bf16>(a, st);
  return check_launch();
}
