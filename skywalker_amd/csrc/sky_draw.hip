// One id of every row of logits by chance (sky_logits_draw).  The entries of a row in the order "largest first, equal ones by column"
// weigh w = exp((z - zmax) / T); what stays of the row is always a beginning of that order (top-k, top-p and min-p each
// cut off an end), and the drawn entry is the first whose weights, summed in the order, pass u times what stays weighs.  So
// everything is one question, asked up to three times: which entry of the order holds rank k, or the unit of mass t?  A row is read
// once to answer it, and in places again; it is never sorted.  What is done depends on how many entries can matter:
//
//   list    at most CAP entries can stay: they are listed in LDS and sorted.  Rows of which a grammar leaves a few, top-k of up to
//           SMALL_K (the k-th largest of the threads' largest entries is no larger than the k-th largest entry) and min-p without top-p.
//           Bound by the reading: 4,096 x 65,536 f16 with a few neighbours each 113 us, 4.7 TB/s.
//   values  16-bit logits have at most 65,536 values: they are counted by value, in 16-bit counters that take 128 KB of
//           LDS, and the rest (weights, prefixes, borders) is a matter of the values that occur, a few thousand.  Bound by the LDS atomics
//           and the second reading, for the columns of equal entries: 256 x 131,072 bf16 by top-p 37 us, 1.8 TB/s.
//   bins    the others (fp32, shorter rows, rows in which a counter runs over): weights are summed in BINS bins of equal width between the largest
//           value and the smallest that weighs anything; the bin that holds the answer is listed and sorted, and
//           when it does not fit the list it becomes the next interval.  That then lies between the smallest and largest value met in it, so
//           that two different values never stay together, and a bin of one value is a matter of counting.  Bound by the fp64 weights
//           and three readings by one CU: 600 x 100,000 fp32 by top-p 244 us.
//   parts   the bins of a few long fp32 rows by several workgroups a row: 40 x 100,003 by top-p 49 us instead of 95.
//
// Weights are summed in whole numbers (2^-S of the largest weight, S = 61 less the bits of the row's length, 50 at most): sums then do
// not depend on the order of LDS atomics or of lanes.  They are rounded once each, by at most 2^-(S+1) of the largest weight; the
// exponential is taken in fp64, since an id changes with the last bit that its border of the sum is off by.
#include "sky_scores.h"

namespace sky {
namespace {

constexpr int THREADS = 1024;        // of a workgroup that has a CU to itself
constexpr int SHORT_THREADS = 256;   // of a workgroup for a shorter row
constexpr uint32_t BINS = 2048;
template <int BT>
constexpr uint32_t CAP = 2 * BT;     // entries of a list: two per thread of the workgroup
constexpr double NO_MASS = 40.0;     // weights below e^-40 are 0 in units of 2^-S, S <= 50
template <int BT>
constexpr uint32_t SMALL_K = BT / 2;  // of 1024 threads' largest entries: some 710 entries are as large as the 512th of them
constexpr uint32_t VALUES = 65536, CHUNK = 256, CHUNKS = VALUES / CHUNK;  // of 16-bit logits; a wavefront takes a chunk, four values a lane
constexpr int PIECES = 16, AHEAD = 4;  // pieces of 16 bytes that a thread tells apart, and of a load that runs while as many are worked on
constexpr uint32_t MAX_COLUMNS = 1u << 26;   // weights keep 35 bits, and what an entry's is divided into 27
constexpr uint32_t SLICE = 1u << 21;         // rows of a launch: fewer than 2^32 threads
constexpr uint32_t NOT_DRAWN = 0xFFFFFFFEu;  // token of a row that draw_short_kernel leaves to draw_kernel

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

// The settings of one row: NaN and what is out of range mean what the header says.
struct Settings {
  float temperature, top_p, min_p;
  uint32_t top_k;
  __device__ __forceinline__ Settings(const DrawArgs& a, uint32_t r) {
    temperature = a.temperature ? a.temperature[r] : 1.0f;
    top_k = a.top_k ? a.top_k[r] : 0u;
    top_p = a.top_p ? a.top_p[r] : 1.0f;
    min_p = a.min_p ? a.min_p[r] : 0.0f;
    if (!(top_p < 1.0f)) top_p = 1.0f;
    if (min_p > 1.0f) top_k = 1;  // not even the equals of the first entry
    if (!(min_p > 0.0f && min_p <= 1.0f)) min_p = 0.0f;
  }
  __device__ __forceinline__ bool greedy() const { return !(temperature > 0.0f); }
  // few entries can stay: top-k of up to `small_k`, and where `by_min_p` min-p without top-p
  __device__ __forceinline__ bool few(uint32_t small_k, bool by_min_p) const {
    return greedy() || (top_k && top_k <= small_k) || (by_min_p && min_p > 0.0f && !(top_p < 1.0f));
  }
};
__device__ __forceinline__ double uniform_of(const DrawArgs& a, uint32_t r) {
  if (a.uniforms) return fmin(fmax(a.uniforms[r], 0.0), 1.0);
  const u32x4 bits = philox(a.seed, a.first_walker + r, a.step, 0, DOM_LOGITS);
  return ((double)(bits.x >> 5) * 67108864.0 + (double)(bits.y >> 6)) * (1.0 / 9007199254740992.0);
}
struct Result {
  uint32_t token, kept;
  double logprob;
};
__device__ __forceinline__ Result nothing_to_draw() { return Result{SKY_INVALID, 0, -__builtin_inf()}; }
__device__ __forceinline__ void store_result(const DrawArgs& a, uint32_t r, const Result& d) {
  a.tokens[r * a.tokens_stride] = d.token;
  if (a.logprobs) a.logprobs[r] = (float)d.logprob;
  if (a.kept) a.kept[r] = d.kept;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp0<DPP_QUAD_XOR1, 0xF>(v));
  v = max(v, dpp0<DPP_QUAD_XOR2, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_HALF_MIRROR, 0xF>(v));
  v = max(v, dpp0<DPP_ROW_MIRROR, 0xF>(v));
  v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
}

// ---------------------------------------------------------------- weights
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
__device__ __forceinline__ int fraction_bits(uint32_t columns) { return min(50, 61 - (31 - __clz((int)columns))); }
// What the weights of a row need.
struct Row {
  double t;    // temperature
  double per;  // log2(e) / t
  float zmax;
  int S;       // fraction bits of a weight
  __device__ __forceinline__ Row(float temperature, float z, int s) : t(temperature), per(1.44269504088896340736 / t), zmax(z), S(s) {}
  __device__ __forceinline__ double weight(float z) const { return exp(((double)z - (double)zmax) / t); }
  __device__ __forceinline__ uint64_t units(float z) const {
    const double x = ((double)z - (double)zmax) * per;
    const uint64_t n = power_units(fmax(x, -60.0), S);
    return x >= -60.0 ? n : 0;
  }
  // rest / each, which is below 2^27
  static __device__ __forceinline__ uint32_t quotient(uint64_t rest, uint64_t each) {
    uint32_t q = (uint32_t)((double)rest / (double)each);  // off by one at most: both are rounded to 53 bits
    if ((uint64_t)q * each > rest) --q;
    if (rest - (uint64_t)q * each >= each) ++q;
    return q;
  }
  // the logarithm of z's share of `mass` units
  __device__ __forceinline__ double log_share(float z, uint64_t mass) const {
    return ((double)z - (double)zmax) / t - log(ldexp((double)mass, -S));
  }
  // units that have to lie before the end of what top-p leaves
  static __device__ __forceinline__ uint64_t needed(float top_p, uint64_t mass) {
    return min(max((uint64_t)ceil(fmax((double)top_p, 0.0) * (double)mass), (uint64_t)1), mass);
  }
  static __device__ __forceinline__ uint64_t drawn(double u, uint64_t mass) { return min((uint64_t)(u * (double)mass), mass - 1); }
};

// ---------------------------------------------------------------- values as places
// The place of a value: the whole number that its bits, those of negative numbers turned over, make: it ascends with the value.  The
// place of what is not there (NaN, -inf) is 0, that of +inf the largest finite number's, that of -0 that of 0.
template <typename T>
struct Places;
template <>
struct Places<float> {
  static constexpr uint32_t ALL = 0xFFFFFFFFu, SIGN = 0x80000000u, INF = 0x7F800000u, LOWEST = 0x00800000u, LARGEST = 0xFF7FFFFFu;
  static __device__ __forceinline__ float value(uint32_t q) { return key_score(q); }
};
template <>
struct Places<_Float16> {
  static constexpr uint32_t ALL = 0xFFFFu, SIGN = 0x8000u, INF = 0x7C00u, LOWEST = 0x0400u, LARGEST = 0xFBFFu;
  static __device__ __forceinline__ float value(uint32_t q) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(q ^ (q & SIGN ? SIGN : ALL))); }
};
template <>
struct Places<__bf16> {
  static constexpr uint32_t ALL = 0xFFFFu, SIGN = 0x8000u, INF = 0x7F80u, LOWEST = 0x0080u, LARGEST = 0xFF7Fu;
  static __device__ __forceinline__ float value(uint32_t q) { return __uint_as_float((q ^ (q & SIGN ? SIGN : ALL)) << 16); }
};
// The place of one element from its bits.
template <typename T>
__device__ __forceinline__ uint32_t place_of_bits(uint32_t b) {
  using P = Places<T>;
  const uint32_t size = b & (P::ALL ^ P::SIGN);
  if (size > P::INF || b == (P::SIGN | P::INF)) return 0;
  if (size == P::INF) return P::LARGEST;
  if (!size) return P::SIGN;
  return b ^ (b & P::SIGN ? P::ALL : P::SIGN);
}
template <typename T>
__device__ __forceinline__ uint32_t place_of(T x) {
  if constexpr (sizeof(T) == 4)
    return place_of_bits<T>(__float_as_uint(x));
  else
    return place_of_bits<T>(__builtin_bit_cast(uint16_t, x));
}
// Words of a row (one 32-bit or two 16-bit elements): bits turned into raw places, which differ from places for what is not finite and
// for -0 (whose raw place is one less than that of 0).  Two instructions a word; what else a row may hold is looked at piece by piece.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ uint32_t raw_places(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return w ^ ((uint32_t)((int32_t)w >> 31) | 0x80000000u);
  } else {
    const uint32_t sign = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, w) >> (int16_t)15);
    return w ^ (sign | 0x80008000u);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4)
    return max(a, b);
  else
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <typename T>
__device__ __forceinline__ uint32_t word_min(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4)
    return min(a, b);
  else
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <typename T>
__device__ __forceinline__ uint32_t piece_max(uint4 w) {
  const uint32_t m = word_max<T>(word_max<T>(w.x, w.y), word_max<T>(w.z, w.w));
  return sizeof(T) == 4 ? m : max(m & 0xFFFFu, m >> 16);
}
template <typename T>
__device__ __forceinline__ uint32_t piece_min(uint4 w) {
  const uint32_t m = word_min<T>(word_min<T>(w.x, w.y), word_min<T>(w.z, w.w));
  return sizeof(T) == 4 ? m : min(m & 0xFFFFu, m >> 16);
}
template <typename T>
__device__ __forceinline__ uint4 raw_places(uint4 w) {
  return uint4{raw_places<T>(w.x), raw_places<T>(w.y), raw_places<T>(w.z), raw_places<T>(w.w)};
}
// f(place, column) for the elements of a piece of bits that begins at column c, in a loop: pieces that are looked at one by one are few.
template <typename T, typename F>
__device__ __forceinline__ void each(uint4 w, uint32_t c, F f) {
#pragma unroll 1
  for (uint32_t e = 0; e < Piece<T>::N; ++e) {
    if constexpr (sizeof(T) == 4) {
      f(place_of_bits<T>(w.x), c + e);
      w = uint4{w.y, w.z, w.w, 0};
    } else {
      f(place_of_bits<T>(w.x & 0xFFFFu), c + e);
      w = uint4{__builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16), __builtin_amdgcn_alignbit(w.w, w.z, 16), w.w >> 16};
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 load_words(const T* p) {
  uint4 w;
  __builtin_memcpy(&w, p, 16);
  return w;
}

// ---------------------------------------------------------------- lists
// An entry of a list: ascending is the order.
__device__ __forceinline__ uint64_t listed(float z, uint32_t column) { return (uint64_t)~score_key(z) << 32 | column; }
__device__ __forceinline__ float listed_score(uint64_t e) { return key_score(~(uint32_t)(e >> 32)); }
constexpr uint64_t LIST_END = ~0ull;

template <int BT>
struct ListShared {
  uint64_t list[CAP<BT>];
  uint64_t wave[BT / 64];
  uint64_t before;
  uint32_t n, found;
};

// Exclusive prefix of v over the workgroup, and the total.
template <int BT>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* waves, uint64_t* total) {
  const uint64_t inclusive = group_scan_u64<64>(v);
  const uint32_t w = threadIdx.x >> 6, l = threadIdx.x & 63;
  __syncthreads();
  if (l == 63) waves[w] = inclusive;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < BT / 64; ++i) {
    const uint64_t x = waves[i];
    before += (uint32_t)i < w ? x : 0;
    all += x;
  }
  *total = all;
  return before + inclusive - v;
}

// list[0..m) into the order.  Up to an entry for two threads: every entry's rank is counted (no barrier between the steps); longer lists
// by a bitonic network over the next power of two.  (us, network alone / so: 2,000 x 8,000 bf16 by top-k of 50 32 / 23, 8 x 131,072 fp32
// by top-k of 120 25 / 22, of 400 34 / 34.)
template <int BT>
__device__ __forceinline__ void sort_list(uint64_t* list, uint32_t m) {
  if (m <= BT / 2) {
    const uint64_t mine = threadIdx.x < m ? list[threadIdx.x] : LIST_END;
    uint32_t rank = 0;
    if (threadIdx.x < m) {
      uint32_t i = 0;
      for (; i + 8 <= m; i += 8)
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) rank += list[i + j] < mine;
      for (; i < m; ++i) rank += list[i] < mine;
    }
    __syncthreads();
    if (threadIdx.x < m) list[rank] = mine;
    __syncthreads();
    return;
  }
  uint32_t size = 64;
  while (size < m) size *= 2;
  for (uint32_t i = m + threadIdx.x; i < size; i += BT) list[i] = LIST_END;
  __syncthreads();
  for (uint32_t k = 2; k <= size; k *= 2)
    for (uint32_t j = k / 2; j; j /= 2) {
      for (uint32_t i = threadIdx.x; i < size / 2; i += BT) {
        const uint32_t a = (i & (j - 1)) | (i & ~(j - 1)) << 1, b = a | j;
        const uint64_t x = list[a], y = list[b];
        if ((x > y) == ((a & k) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
}

// Everything about a row whose entries, or as many of them as can matter, are list[0..n), n <= 64, in any order: by one wavefront.
__device__ __forceinline__ Result draw_wave(uint64_t* list, uint32_t n, const Settings& o, double u) {
  const uint32_t lane = threadIdx.x & 63;
  uint64_t e = lane < n ? list[lane] : LIST_END;
  uint32_t rank = 0;
  for (uint32_t i = 0; i < n; i += 4)
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) rank += i + j < n && list[i + j] < e;
  __builtin_amdgcn_wave_barrier();
  if (lane < n) list[rank] = e;
  __builtin_amdgcn_wave_barrier();
  e = lane < n ? list[lane] : LIST_END;
  const Row row(o.temperature, listed_score(shfl_u64(e, 0)), 50);
  const uint32_t k = o.top_k && o.top_k < n ? o.top_k : n;
  const float z = lane < k ? listed_score(e) : row.zmax;
  const uint64_t mine = lane < k ? row.units(z) : 0, sum = group_scan_u64<64>(mine), before = sum - mine;
  uint32_t stay = k;
  if (o.top_p < 1.0f || o.min_p > 0.0f) {
    const uint64_t need = o.top_p < 1.0f ? Row::needed(o.top_p, shfl_u64(sum, 63)) : ~0ull;
    const bool in = lane < k && before < need && (o.min_p == 0.0f || row.weight(z) >= (double)o.min_p);
    stay = max(1u, (uint32_t)__builtin_popcountll(__ballot(in)));
  }
  const uint64_t mass = shfl_u64(sum, (int)stay - 1), unit = Row::drawn(u, mass);
  const int at = (int)__builtin_ctzll(__ballot(before <= unit && unit < sum));
  return Result{(uint32_t)shfl_u64(e, at), stay, row.log_share(__shfl(z, at, 64), mass)};
}

// The same for m > 64 entries of s.list (or fewer), by the workgroup.
template <int BT>
__device__ __forceinline__ Result draw_listed(ListShared<BT>& s, uint32_t m, const Settings& o, double u) {
  constexpr uint32_t PER = CAP<BT> / BT;
  sort_list<BT>(s.list, m);
  const Row row(o.temperature, listed_score(s.list[0]), 50);  // at most 2^11 weights
  const uint32_t k = o.top_k && o.top_k < m ? o.top_k : m, i0 = PER * threadIdx.x;
  uint64_t mine[PER], sum = 0, total;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    mine[i] = i0 + i < k ? row.units(listed_score(s.list[i0 + i])) : 0;
    sum += mine[i];
  }
  const uint64_t before = block_scan<BT>(sum, s.wave, &total);
  uint32_t n = k;
  if (o.top_p < 1.0f || o.min_p > 0.0f) {
    // entries stay while what comes before them is below p of the total, and their weight at least min_p
    const uint64_t need = o.top_p < 1.0f ? Row::needed(o.top_p, total) : ~0ull;
    uint64_t many = 0, b = before, all;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
      const uint32_t at = i0 + i;
      many += at < k && (at == 0 || (b < need && (o.min_p == 0.0f || row.weight(listed_score(s.list[at])) >= (double)o.min_p)));
      b += mine[i];
    }
    block_scan<BT>(many, s.wave, &all);
    n = (uint32_t)all;
  }
  // what the n entries weigh, by the owner of the last one
  uint64_t b = before;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    b += mine[i];
    if (i0 + i == n - 1) s.before = b;
  }
  __syncthreads();
  const uint64_t mass = s.before, unit = Row::drawn(u, mass);
  b = before;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    if (i0 + i < n && b <= unit && unit < b + mine[i]) s.found = i0 + i;
    b += mine[i];
  }
  __syncthreads();
  const uint64_t e = s.list[s.found];
  return Result{(uint32_t)e, n, row.log_share(listed_score(e), mass)};
}
// The result is thread 0's.
template <int BT>
__device__ __forceinline__ Result draw_list(ListShared<BT>& s, uint32_t n, const Settings& o, double u) {
  if (n > 64) return draw_listed<BT>(s, n, o, u);
  return threadIdx.x < 64 ? draw_wave(s.list, n, o, u) : nothing_to_draw();
}
// Greedy: the first of the order among n listed entries.
template <int BT>
__device__ __forceinline__ Result first_listed(ListShared<BT>& s, uint32_t n) {
  uint64_t best = LIST_END;
  if (threadIdx.x < 64) {
    for (uint32_t i = threadIdx.x; i < n; i += 64) best = min(best, s.list[i]);
#pragma unroll
    for (int m = 1; m < 64; m *= 2) best = min(best, shfl_xor_u64(best, m));
  }
  return Result{(uint32_t)best, 1, 0.0};
}

// A place that at least k of the `counts` values v[i] of the wavefront's lanes reach, and few more (MAX of them are looked at: `counts`
// of a lane; the others are left alone).  `most`: the largest.
template <int MAX>
__device__ __forceinline__ uint32_t place_of_rank(const uint32_t (&v)[MAX], int counts, uint32_t k, uint32_t most) {
  auto reach = [&](uint32_t place) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < MAX; ++i)
      if (i < counts) n += (uint32_t)__builtin_popcountll(__ballot(v[i] >= place));
    return n;
  };
  uint32_t lo = v[0], hi = most;  // k or more reach lo, fewer reach more than hi
#pragma unroll
  for (int i = 1; i < MAX; ++i)
    if (i < counts) lo = min(lo, v[i]);
  lo = wave_min_u32(lo);  // all of them reach it
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2, n = reach(mid);
    if (n >= k) {
      lo = mid;
      if (n <= k + 16) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// ---------------------------------------------------------------- a row a workgroup
struct Counters {
  uint32_t value[VALUES / 2];  // places below 32,768 in the low halves, the others in the high ones
  uint32_t chunk_count[CHUNKS];
  uint64_t chunk_mass[CHUNKS];
};
template <int BT>
struct BinsAndList {
  ListShared<BT> l;
  uint64_t bin[BINS];
};
template <int BT>
union Large {
  BinsAndList<BT> some;
};
template <>
union Large<THREADS> {
  BinsAndList<THREADS> some;
  Counters counters;  // of 16-bit logits
};
// LDS of a workgroup of BT threads: one of 1024 has a CU to itself, of 256 four are on one.
template <int BT>
struct Shared {
  Large<BT> large;
  uint64_t wave[BT / 64];
  uint64_t count_before, mass_before;
  uint32_t most[BT], hit[BT], room[CAP<BT>];
  uint32_t wave_most[BT / 64], wave_least[BT / 64], wave_there[BT / 64], wave_above[BT / 64];
  uint32_t hits, place, chunk, found, lo, hi;
};
static_assert(sizeof(Shared<THREADS>) <= 160 * 1024 && sizeof(Shared<SHORT_THREADS>) <= 40 * 1024, "LDS of a CU");

// A row as the workgroup's threads read it: PIECES each in turns of BT * PIECES, and an entry each of those that do
// not fill a piece.  Kept of it: the largest raw place of each of a thread's pieces (over all turns).
template <typename T, int BT>
struct Reader {
  static constexpr uint32_t N = Piece<T>::N, STEP = BT * N, TURN = STEP * PIECES;
  static constexpr uint32_t HITS = BT;  // pieces that are read a second time an entry a thread
  using P = Places<T>;
  const T* x;
  uint32_t columns, whole;
  uint32_t most[PIECES];
  uint32_t last;  // place of the odd entry, 0: none

  __device__ __forceinline__ Reader(const T* row, uint32_t n) : x(row), columns(n), whole(n / N * N), last(0) {}
  __device__ __forceinline__ uint4 load(uint32_t c) const { return load_words(x + min(c, whole - N)); }  // of a row of a piece and more

  // The first reading.  f(a piece's raw places) for pieces of finite numbers above the lowest; odd(a piece's bits, column) for the others.
  // Returns the largest place of the thread.
  template <typename F, typename G>
  __device__ __forceinline__ uint32_t first(F f, G odd) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) most[i] = 0;
    uint4 w[2][AHEAD];  // those that are worked on, and those that are under way
    if (whole)
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) w[0][i] = load(i * STEP + threadIdx.x * N);
#pragma unroll 1
    for (uint32_t turn = 0; turn < whole; turn += TURN) {
#pragma unroll
      for (int h = 0; h < PIECES / AHEAD; ++h) {
        const uint32_t base = turn + h * AHEAD * STEP;
        if (base >= whole) break;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) w[1 - h % 2][i] = load(base + (AHEAD + i) * STEP + threadIdx.x * N);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          __builtin_amdgcn_sched_barrier(0);  // pieces are worked on as they arrive: all at once they would not fit the registers
          const uint32_t c = base + i * STEP + threadIdx.x * N;
          if (c < whole) {
            const uint4 p = raw_places<T>(w[h % 2][i]);
            uint32_t m = piece_max<T>(p);
            if (m <= P::LARGEST && piece_min<T>(p) > P::LOWEST)
              f(p);
            else
              m = odd(w[h % 2][i], c);
            most[h * AHEAD + i] = max(most[h * AHEAD + i], m);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    uint32_t m = 0;
    if (whole + threadIdx.x < columns) last = place_of(x[whole + threadIdx.x]);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) m = max(m, most[i]);
    return max(m == P::SIGN - 1 ? P::SIGN : m, last);  // -0
  }
  // f(a piece's bits, column) for all pieces: AHEAD of them are under way while as many are worked on
  template <typename F>
  __device__ __forceinline__ void stream(F f) const {
    uint4 w[2][AHEAD];
    if (!whole) return;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) w[0][i] = load(i * STEP + threadIdx.x * N);
#pragma unroll 1
    for (uint32_t base = 0; base < whole; base += 2 * AHEAD * STEP)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) w[1 - h][i] = load(base + ((h + 1) * AHEAD + i) * STEP + threadIdx.x * N);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          const uint32_t c = base + (h * AHEAD + i) * STEP + threadIdx.x * N;
          if (c < whole) f(w[h][i], c);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  // f(place, column) for every entry of the pieces that `wanted` (of a piece's raw places) says yes to, of those whose largest place may
  // reach `least`, and perhaps of others.  Pieces that the maxima name are few, or all are read again and those that are wanted are
  // few; either way an entry of them goes to a thread.  Called by all threads; a barrier is left to the caller.
  template <typename W, typename F>
  __device__ __forceinline__ void again(Shared<BT>& s, uint32_t least, bool many, W wanted, F f) const {
    const uint32_t raw = least == P::SIGN ? P::SIGN - 1 : least;
    uint32_t hits = HITS + 1, step = TURN;
    if (!many) {
      __syncthreads();
      if (threadIdx.x == 0) s.hits = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (most[i] >= raw) {
          const uint32_t at = atomicAdd(&s.hits, 1u);
          if (at < HITS) s.hit[at] = (i * BT + threadIdx.x) * N;
        }
      __syncthreads();
      hits = s.hits;
    }
    if (hits > HITS) {
      __syncthreads();
      if (threadIdx.x == 0) s.hits = 0;
      __syncthreads();
      stream([&](uint4 w, uint32_t c) {
        if (wanted(raw_places<T>(w))) {
          const uint32_t at = atomicAdd(&s.hits, 1u);
          if (at < HITS)
            s.hit[at] = c;
          else
            each<T>(w, c, f);  // not few
        }
      });
      __syncthreads();
      hits = min(s.hits, HITS);
      step = whole;
    }
    for (uint32_t i = threadIdx.x; i < hits * N; i += BT)
      for (uint32_t c = s.hit[i / N] + i % N; c < whole; c += step) f(place_of(x[c]), c);
  }
  // f(place, column) for the entries from `least` on
  template <typename F>
  __device__ __forceinline__ void from(Shared<BT>& s, uint32_t least, F f) const {
    const uint32_t raw = least == P::SIGN ? P::SIGN - 1 : least;
    auto some = [&](uint32_t q, uint32_t c) { if (q >= least) f(q, c); };
    again(s, least, false, [&](uint4 p) { return piece_max<T>(p) >= raw; }, some);
    if (last) some(last, whole + threadIdx.x);
  }
  // f(column) for the entries of a place; `many`: so many entries are larger that the maxima do not tell where they are
  template <typename F>
  __device__ __forceinline__ void equal(Shared<BT>& s, uint32_t place, bool many, F f) const {
    // what is 0 in a word that holds the place's raw bits; two kinds of bits are the place of 0 and that of the largest number
    const uint32_t other = place == P::SIGN ? P::SIGN - 1 : place == P::LARGEST ? P::LARGEST + 1 : place;
    const uint32_t a = sizeof(T) == 4 ? place : place | place << 16, b = sizeof(T) == 4 ? other : other | other << 16;
    auto some = [&](uint32_t q, uint32_t c) { if (q == place) f(c); };
    again(s, place, many, [&](uint4 p) {
      uint32_t m = piece_min<T>(uint4{p.x ^ a, p.y ^ a, p.z ^ a, p.w ^ a});
      if (a != b) m = min(m, piece_min<T>(uint4{p.x ^ b, p.y ^ b, p.z ^ b, p.w ^ b}));
      return m == 0;
    }, some);
    if (last) some(last, whole + threadIdx.x);
  }
  // Entries between two places: f(place, column) for the entries of every piece that holds one, or that holds what is no finite number;
  // returns how many entries of the other pieces are larger.  All of the row is read.
  template <typename F>
  __device__ __forceinline__ uint32_t band(Shared<BT>& s, uint32_t lo, uint32_t hi, F f) const {
    const uint32_t raw = lo == P::SIGN ? P::SIGN - 1 : lo;
    uint32_t larger = 0;
    again(s, 0, true, [&](uint4 p) {
      if (piece_max<T>(p) > P::LARGEST) return true;
      uint32_t in = 0, over = 0;
      auto one = [&](uint32_t q) {
        in |= q - raw <= hi - raw;
        over += q > hi;
      };
      const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          one(w[i]);
        } else {
          one(w[i] & 0xFFFFu);
          one(w[i] >> 16);
        }
      }
      larger += in ? 0 : over;
      return in != 0;
    }, f);
    if (last) f(last, whole + threadIdx.x);
    return larger;
  }
  // f(value) for every entry from `low` on: later readings of the whole row
  template <typename F>
  __device__ __forceinline__ void values(float low, F f) const {
    const uint32_t least = place_of((T)low), raw = least == P::SIGN ? P::SIGN - 1 : least;
    stream([&](uint4 w, uint32_t c) {
      const uint4 p = raw_places<T>(w);
      // (16-bit rows of a workgroup of 1024 come here only if their counters run over: they go without)
      if ((sizeof(T) == 4 || BT != THREADS) && piece_max<T>(p) <= P::LARGEST && piece_min<T>(p) >= raw && least) {
        if constexpr (sizeof(T) == 4) {
          f(__uint_as_float(w.x));
          f(__uint_as_float(w.y));
          f(__uint_as_float(w.z));
          f(__uint_as_float(w.w));
        } else {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            f((float)__builtin_bit_cast(T, (uint16_t)w.x));
            f((float)__builtin_bit_cast(T, (uint16_t)(w.x >> 16)));
            w = uint4{w.y, w.z, w.w, 0};
          }
        }
      } else {
        each<T>(w, c, [&](uint32_t q, uint32_t) { if (q && P::value(q) >= low) f(P::value(q)); });
      }
    });
    if (last && P::value(last) >= low) f(P::value(last));
  }
};

// The column of entry `tie` among those of value z, by column: as few of them as the list holds are listed, more are counted off.
template <typename T, int BT>
__device__ __forceinline__ uint32_t column_of_tie(const Reader<T, BT>& in, Shared<BT>& s, uint32_t q, uint32_t tie, uint32_t ties, uint64_t larger) {
  __syncthreads();
  if (threadIdx.x == 0) s.found = SKY_INVALID;
  if (ties <= CAP<BT>) {
    if (threadIdx.x == 0) s.place = 0;
    in.equal(s, q, larger > 4 * BT, [&](uint32_t c) { s.room[atomicAdd(&s.place, 1u)] = c; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < ties; i += BT) {
      uint32_t below = 0;
      const uint32_t c = s.room[i];
      for (uint32_t j = 0; j < ties; ++j) below += s.room[j] < c;
      if (below == tie) s.found = c;
    }
  } else {
    uint64_t seen = 0;
    for (uint32_t base = 0; base < in.columns && seen <= tie; base += BT) {
      const uint32_t c = base + threadIdx.x;
      const uint64_t here = c < in.columns && place_of(in.x[c]) == q;
      uint64_t total;
      const uint64_t before = seen + block_scan<BT>(here, s.wave, &total);
      if (here && before == tie) s.found = c;
      seen += total;
    }
  }
  __syncthreads();
  return s.found;
}

// ---------------------------------------------------------------- by value
__device__ __forceinline__ uint32_t count_of(const Counters& c, uint32_t q) {
  const uint32_t both = c.value[q & 0x7FFFu];
  return q & 0x8000u ? both >> 16 : both & 0xFFFFu;
}
// A lane's four values of a chunk, the largest first: lane 0 has the four largest.
struct Values {
  uint32_t q;         // place of the largest; the others follow downwards
  uint32_t count[4];
  uint64_t each[4], mass[4];  // units of an entry of the value, and of all of them
  __device__ __forceinline__ uint32_t counts() const { return count[0] + count[1] + count[2] + count[3]; }
  __device__ __forceinline__ uint64_t masses() const { return mass[0] + mass[1] + mass[2] + mass[3]; }
};
__device__ __forceinline__ bool values_of(const Counters& c, uint32_t chunk, Values* v) {
  v->q = chunk * CHUNK + (CHUNK - 1) - 4 * (threadIdx.x & 63);
  uint4 w = *(const uint4*)&c.value[(v->q - 3) & 0x7FFFu];
  const uint32_t shift = v->q & 0x8000u ? 16 : 0;
  v->count[0] = w.w >> shift & 0xFFFFu;
  v->count[1] = w.z >> shift & 0xFFFFu;
  v->count[2] = w.y >> shift & 0xFFFFu;
  v->count[3] = w.x >> shift & 0xFFFFu;
  return __ballot(v->counts() != 0) != 0;
}
template <typename T>
__device__ __forceinline__ void weigh(const Row& row, Values* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v->each[j] = row.units(v->count[j] ? Places<T>::value(v->q - j) : row.zmax);  // without branches: beside one another
#pragma unroll
  for (int j = 0; j < 4; ++j) v->mass[j] = v->count[j] * v->each[j];
}
// The value that holds a unit (RANK: of the count; else of mass), from the sums of chunks before each thread's own (thread t < CHUNKS has
// the t-th chunk from the top).
struct ValuePlace {
  uint32_t q, tie;
  float z;
  uint64_t count_before, mass_before, each;  // before the value; of an entry of it
  __device__ __forceinline__ uint64_t mass_with() const { return mass_before + (uint64_t)(tie + 1) * each; }
};
template <bool RANK, typename T>
__device__ __forceinline__ ValuePlace locate_value(Shared<THREADS>& s, const Row& row, uint64_t unit, uint64_t count_before, uint64_t mass_before) {
  __syncthreads();
  if (threadIdx.x < CHUNKS) {
    const uint32_t mine = CHUNKS - 1 - threadIdx.x;
    const uint64_t before = RANK ? count_before : mass_before;
    const uint64_t here = RANK ? (uint64_t)s.large.counters.chunk_count[mine] : s.large.counters.chunk_mass[mine];
    if (before <= unit && unit < before + here) {
      s.chunk = mine;
      s.count_before = count_before;
      s.mass_before = mass_before;
    }
  }
  __syncthreads();
  Values v;
  values_of(s.large.counters, s.chunk, &v);
  weigh<T>(row, &v);
  uint64_t counts = s.count_before + group_scan_u32<64>(v.counts()) - v.counts(), masses = s.mass_before + group_scan_u64<64>(v.masses()) - v.masses();
  ValuePlace p{0, 0, 0.0f, 0, 0, 0};
  bool here = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t start = RANK ? counts : masses, size = RANK ? (uint64_t)v.count[j] : v.mass[j];
    if (start <= unit && unit < start + size) {
      here = true;
      p.q = v.q - j;
      p.count_before = counts;
      p.mass_before = masses;
      p.each = v.each[j];
    }
    counts += v.count[j];
    masses += v.mass[j];
  }
  const int lane = (int)__builtin_ctzll(__ballot(here) | 1ull << 63);
  p.q = (uint32_t)__shfl((int)p.q, lane, 64);
  p.count_before = shfl_u64(p.count_before, lane);
  p.mass_before = shfl_u64(p.mass_before, lane);
  p.each = shfl_u64(p.each, lane);
  p.z = Places<T>::value(p.q);
  p.tie = RANK ? (uint32_t)(unit - p.count_before) : Row::quotient(unit - p.mass_before, p.each);
  return p;
}
// The largest place up to `most` whose value fails `passes`, which holds from some place on; what is not there fails.
template <typename T, typename F>
__device__ __forceinline__ uint32_t last_failing(uint32_t most, F passes) {
  uint32_t lo = 0;
  for (uint32_t bit = Places<T>::SIGN; bit; bit >>= 1) {
    const uint32_t q = lo | bit;
    if (q <= most && (q < Places<T>::LOWEST || !passes(Places<T>::value(q)))) lo = q;
  }
  return lo;
}
__device__ __forceinline__ void clear_counters(Counters& c) {
  for (uint32_t i = threadIdx.x; i < VALUES / 8; i += THREADS) ((uint4*)c.value)[i] = uint4{0, 0, 0, 0};
}
__device__ __forceinline__ void count_place(Counters& c, uint32_t q) { atomicAdd(&c.value[q & 0x7FFFu], (q >> 15) * 0xFFFFu + 1u); }
__device__ __forceinline__ void count_word(Counters& c, uint32_t w) {
  count_place(c, w & 0xFFFFu);
  count_place(c, w >> 16);
}

// A row that has been counted, all but entries of the lowest value, which masks are made of: `above` of `there`.  false: a counter
// has run over, or the lowest value weighs something.
template <typename T>
__device__ __forceinline__ bool draw_by_value(const Reader<T, THREADS>& in, Shared<THREADS>& s, const Row& row, const Settings& o, double u, uint32_t most, uint32_t there,
                                              uint32_t above, Result* result) {
  using P = Places<T>;
  Counters& c = s.large.counters;
  if (there != above && row.units(P::value(P::LOWEST))) return false;
  if (threadIdx.x == 0) {  // what was counted as -0 is 0
    const uint32_t n = c.value[P::SIGN - 1] & 0xFFFFu;
    c.value[P::SIGN - 1] -= n;
    c.value[0] += n << 16;
  }
  __syncthreads();
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  // a wavefront takes every 16th chunk: those that occur lie together
  for (uint32_t chunk = wave; chunk < CHUNKS; chunk += THREADS / 64) {
    Values v;
    uint64_t mass = 0;
    uint32_t count = 0;
    if (values_of(c, chunk, &v)) {
      weigh<T>(row, &v);
      count = group_scan_u32<64>(v.counts());
      mass = group_scan_u64<64>(v.masses());
    }
    if (lane == 63) {
      c.chunk_count[chunk] = count;
      c.chunk_mass[chunk] = mass;
    }
  }
  __syncthreads();
  uint64_t counted, mass;
  const uint32_t mine = CHUNKS - 1 - threadIdx.x;
  const bool own = threadIdx.x < CHUNKS;
  const uint64_t count_before = block_scan<THREADS>(own ? c.chunk_count[mine] : 0, s.wave, &counted);
  const uint64_t mass_before = block_scan<THREADS>(own ? c.chunk_mass[mine] : 0, s.wave, &mass);
  if (counted != above) return false;
  uint32_t count = there;
  if (o.top_k && o.top_k < there) {
    count = o.top_k;
    if (o.top_k < above) {
      const ValuePlace p = locate_value<true, T>(s, row, o.top_k - 1, count_before, mass_before);
      mass = p.mass_with();
    }
  }
  if (o.top_p < 1.0f) {
    const ValuePlace p = locate_value<false, T>(s, row, Row::needed(o.top_p, mass) - 1, count_before, mass_before);
    mass = p.mass_with();
    count = (uint32_t)p.count_before + p.tie + 1;
  }
  if (o.min_p > 0.0f) {
    const uint32_t least = min(last_failing<T>(most, [&](float z) { return row.weight(z) >= (double)o.min_p; }) + 1, most), chunk = least / CHUNK;
    __syncthreads();
    if (own && mine == chunk) {
      s.count_before = count_before;
      s.mass_before = mass_before;
    }
    __syncthreads();
    Values v;
    values_of(c, chunk, &v);
    weigh<T>(row, &v);
    uint32_t in_count = 0;
    uint64_t in_mass = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v.q - j >= least) {
        in_count += v.count[j];
        in_mass += v.mass[j];
      }
    const uint64_t all_count = s.count_before + (uint32_t)__shfl((int)group_scan_u32<64>(in_count), 63, 64);
    const uint64_t all_mass = s.mass_before + shfl_u64(group_scan_u64<64>(in_mass), 63);
    if (least > P::LOWEST && all_count < count) {
      count = (uint32_t)all_count;
      mass = all_mass;
    }
  }
  const ValuePlace p = locate_value<false, T>(s, row, Row::drawn(u, mass), count_before, mass_before);
  *result = Result{column_of_tie(in, s, p.q, p.tie, count_of(c, p.q), p.count_before), count, row.log_share(p.z, mass)};
  return true;
}

// ---------------------------------------------------------------- by bins
// Which bins an interval [lo, hi] of values has.  Monotone in z, the same for equal z, 0 for hi and BINS - 1 or the one before for lo (0 if
// that is hi).
struct Bins {
  double hi, scale;
  float top, low, narrow;  // narrow: the scale in fp32, 0 where that might not tell lo and hi apart (very wide and very narrow intervals)
  __device__ __forceinline__ Bins(float h, float l) : hi(h), scale(h > l ? (double)(BINS - 1) / ((double)h - (double)l) : 0.0), top(h), low(l) {
    narrow = scale > 1e-30 && scale < 1e30 ? (float)scale : 0.0f;
  }
  __device__ __forceinline__ bool has(float z) const { return z <= top && z >= low; }
  // no value of bins 0 .. b is smaller than the lower edge, none of bins b and on is larger than the upper one
  __device__ __forceinline__ float lower_edge(uint32_t b) const {
    const double z = scale > 0.0 ? hi - ((double)b + 1.0) / scale : (double)low;
    return fmaxf((float)(z - 1e-6 * fabs(z) - 1e-5 * ((double)top - z)), low);
  }
  __device__ __forceinline__ float upper_edge(uint32_t b) const {
    const double z = scale > 0.0 ? hi - (double)b / scale : (double)top;
    return fminf((float)(z + 1e-6 * fabs(z) + 1e-5 * ((double)top - z)), top);
  }
  __device__ __forceinline__ uint32_t of(float z) const {
    return min(narrow != 0.0f ? (uint32_t)((top - z) * narrow) : (uint32_t)((hi - (double)z) * scale), BINS - 1);
  }
};
// Where an answer lies: the value, how many entries of it come before, how many there are, the column (SKY_INVALID: to be looked
// for), and what all entries before the value amount to (units of mass or entries).
struct Place {
  float z;
  uint32_t tie, ties, column;
  uint64_t before, larger;  // `larger`: entries before the value
};
// What a thread knows of the bins it owns, BINS / BT of them.
template <int BT>
struct Filled {
  static constexpr uint32_t PER = BINS / BT;
  uint64_t before, bin[PER], all, total;
};

// The values, RANK: entries; else units of mass, of the entries of [low, zmax], less `excess` entries of the value `low`, in bins.
template <bool RANK, typename T, int BT>
__device__ __forceinline__ Filled<BT> fill_bins(const Reader<T, BT>& in, Shared<BT>& s, const Row& row, const Bins& bins, float low, uint32_t excess) {
  auto value = [&](float z) -> uint64_t { return RANK ? 1ull : row.units(z); };
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < BINS; i += BT) s.large.some.bin[i] = 0;
  __syncthreads();
  in.values(bins.low, [&](float z) {
    if (z <= bins.top) atomicAdd((unsigned long long*)&s.large.some.bin[bins.of(z)], (unsigned long long)value(z));
  });
  __syncthreads();
  if (excess && bins.has(low) && threadIdx.x == 0) s.large.some.bin[bins.of(low)] -= (uint64_t)excess * value(low);
  __syncthreads();
  Filled<BT> f;
  f.all = 0;
#pragma unroll
  for (uint32_t i = 0; i < f.PER; ++i) f.all += f.bin[i] = s.large.some.bin[f.PER * threadIdx.x + i];
  f.before = block_scan<BT>(f.all, s.wave, &f.total);
  return f;
}
// The entry that holds unit `unit`, from the bins of the whole interval.  Every thread calls it and has the answer.
template <bool RANK, typename T, int BT>
__device__ __forceinline__ Place locate(const Reader<T, BT>& in, Shared<BT>& s, const Row& row, Bins bins, Filled<BT> f, float low, uint32_t excess, uint64_t unit) {
  using P = Places<T>;
  auto value = [&](float z) -> uint64_t { return RANK ? 1ull : row.units(z); };
  Place p;
  uint64_t before = 0;
  for (;;) {
    const uint64_t e = before + f.before;
    __syncthreads();
    if (threadIdx.x == 0) {
      s.large.some.l.n = 0;
      s.lo = 0xFFFFFFFFu;
      s.hi = 0;
    }
    if (e <= unit && unit < e + f.all) {
      uint64_t start = e;
#pragma unroll
      for (uint32_t i = 0; i < f.PER; ++i) {
        if (start <= unit && unit < start + f.bin[i]) {
          s.found = f.PER * threadIdx.x + i;
          s.mass_before = start;
        }
        start += f.bin[i];
      }
    }
    __syncthreads();
    const uint32_t b = s.found;
    before = s.mass_before;
    // the bin's entries: how many, between which values, and the list of them if it holds them; and how many entries are larger
    uint32_t kmin = 0xFFFFFFFFu, kmax = 0;
    uint64_t larger = 0;
    uint32_t in_pieces = 0;
    larger = in.band(s, max(place_of((T)bins.lower_edge(b)), P::LOWEST), place_of((T)bins.upper_edge(b)), [&](uint32_t q, uint32_t c) {
      if (!q) return;
      const float z = P::value(q);
      if (z > bins.top) {
        ++in_pieces;
      } else if (z >= bins.low) {
        const uint32_t mine = bins.of(z);
        in_pieces += mine < b;
        if (mine == b) {
          const uint32_t key = score_key(z), at = atomicAdd(&s.large.some.l.n, 1u);
          kmin = min(kmin, key);
          kmax = max(kmax, key);
          if (at < CAP<BT>) s.large.some.l.list[at] = listed(z, c);
        }
      }
    });
    larger += in_pieces;
    kmin = wave_min_u32(kmin);
    kmax = wave_max_u32(kmax);
    if ((threadIdx.x & 63) == 0 && kmax) {
      atomicMin(&s.lo, kmin);
      atomicMax(&s.hi, kmax);
    }
    block_scan<BT>(larger, s.wave, &p.larger);  // its barriers publish the list
    const uint32_t n = s.large.some.l.n;
    const float lo = key_score(s.lo), hi = key_score(s.hi);
    if (lo == hi) {  // one value: the place among its equals
      p = Place{hi, Row::quotient(unit - before, value(hi)), n, SKY_INVALID, before, p.larger};
      if (n == 1) p.column = (uint32_t)s.large.some.l.list[0];
      return p;
    }
    if (n <= CAP<BT>) {
      sort_list<BT>(s.large.some.l.list, n);
      const uint32_t m = lo == low ? n - excess : n, i0 = 2 * threadIdx.x, i1 = i0 + 1;
      const float z0 = i0 < m ? listed_score(s.large.some.l.list[i0]) : 0.0f, z1 = i1 < m ? listed_score(s.large.some.l.list[i1]) : 0.0f;
      const uint64_t v0 = i0 < m ? value(z0) : 0, v1 = i1 < m ? value(z1) : 0;
      uint64_t total;
      const uint64_t at = before + block_scan<BT>(v0 + v1, s.wave, &total);
      if (at <= unit && unit < at + v0) s.found = i0;
      if (at + v0 <= unit && unit < at + v0 + v1) s.found = i1;
      __syncthreads();
      const uint64_t entry = s.large.some.l.list[s.found];
      p.z = listed_score(entry);
      p.column = (uint32_t)entry;
      // its equals in the list: how many come before it, and where the first of them begins
      const bool equal0 = i0 < n && listed_score(s.large.some.l.list[i0]) == p.z, equal1 = i1 < n && listed_score(s.large.some.l.list[i1]) == p.z;
      const bool before0 = i0 ? listed_score(s.large.some.l.list[i0 - 1]) != p.z : true;
      if (equal0 && before0) s.count_before = i0, s.mass_before = at;
      if (equal1 && !equal0) s.count_before = i1, s.mass_before = at + v0;
      uint64_t ties;
      block_scan<BT>((uint64_t)equal0 + (uint64_t)equal1, s.wave, &ties);  // its barriers publish the two above
      p.ties = (uint32_t)ties;
      p.tie = s.found - (uint32_t)s.count_before;
      p.before = s.mass_before;
      p.larger += s.count_before;
      return p;
    }
    bins = Bins(hi, lo);
    f = fill_bins<RANK>(in, s, row, bins, low, excess);
  }
}

template <typename T, int BT>
__device__ __forceinline__ Result draw_by_bins(const Reader<T, BT>& in, Shared<BT>& s, const Row& row, const Settings& o, double u, uint32_t most, float zmin,
                                               uint32_t there) {
  // What stays is the beginning of the order that ends with `count` entries; entries below `low` weigh nothing or do not belong to it, nor
  // do the last `excess` of value `low`.
  float low = zmin;
  uint32_t excess = 0, count = there;
  if (o.top_k && o.top_k < there) {
    const Bins bins(row.zmax, zmin);
    const Filled<BT> f = fill_bins<true>(in, s, row, bins, zmin, 0);
    const Place p = locate<true>(in, s, row, bins, f, zmin, 0, o.top_k - 1);
    low = p.z;
    count = o.top_k;
    excess = p.ties - (p.tie + 1);
  }
  const float cut = (float)fmax((double)row.zmax - NO_MASS * row.t, -3.402823466e38);
  const bool cut_off = low < cut;
  if (cut_off) {
    low = cut;
    excess = 0;
  }
  const Bins bins(row.zmax, low);
  const Filled<BT> f = fill_bins<false>(in, s, row, bins, low, excess);
  uint64_t mass = f.total;
  float end = low;
  if (o.top_p < 1.0f) {
    const Place p = locate<false>(in, s, row, bins, f, low, excess, Row::needed(o.top_p, mass) - 1);
    mass = p.before + (uint64_t)(p.tie + 1) * row.units(p.z);
    end = p.z;
    count = (uint32_t)p.larger + p.tie + 1;
  }
  if (o.min_p > 0.0f && (row.weight(end) < (double)o.min_p || (cut_off && !(o.top_p < 1.0f)))) {
    const uint32_t least = min(last_failing<T>(most, [&](float z) { return row.weight(z) >= (double)o.min_p; }) + 1, most);
    const float z_least = Places<T>::value(max(least, Places<T>::LOWEST));
    uint64_t weighs = 0, many = 0, all, all_many;
    in.values(z_least, [&](float z) {
      weighs += row.units(z);
      ++many;
    });
    block_scan<BT>(weighs, s.wave, &all);
    block_scan<BT>(many, s.wave, &all_many);
    if (all_many < count) {
      mass = all;
      count = (uint32_t)all_many;
    }
  }
  const Place p = locate<false>(in, s, row, bins, f, low, excess, Row::drawn(u, mass));
  Result r{p.column, count, row.log_share(p.z, mass)};
  if (r.token == SKY_INVALID) {
    r.token = column_of_tie(in, s, place_of((T)p.z), p.tie, p.ties, p.larger);
  }
  return r;
}

// The same out of line, for kernels in which it is an exception and would only take the others' registers.
template <typename T, int BT>
__device__ __noinline__ Result draw_by_bins_apart(Reader<T, BT> in, Shared<BT>* s, Row row, Settings o, double u, uint32_t most, float zmin, uint32_t there) {
  return draw_by_bins(in, *s, row, o, u, most, zmin, there);
}

// s.place: a place that at least k of the threads' largest (s.most) reach, and few more, so that at least k entries reach it.  Up to
// BT / 8 the largest of four threads do.  Its barrier publishes it.
template <int BT>
__device__ __forceinline__ void place_for_rank(Shared<BT>& s, uint32_t k, uint32_t most) {
  if (threadIdx.x < 64) {
    uint32_t v[BT / 64];
    const bool quads = k <= BT / 8;
#pragma unroll
    for (int i = 0; i < BT / 64; ++i) v[i] = s.most[64 * i + threadIdx.x];
#pragma unroll
    for (int i = 0; i < BT / 64; i += 4)
      if (quads) v[i / 4] = max(max(v[i], v[i + 1]), max(v[i + 2], v[i + 3]));
    const uint32_t lo = place_of_rank<BT / 64>(v, quads ? BT / 256 : BT / 64, k, most);
    if (threadIdx.x == 0) s.place = lo;
  }
  __syncthreads();
}

// ---------------------------------------------------------------- the kernel
template <typename T, int BT>
__device__ __forceinline__ Result draw_row(const T* x, uint32_t columns, Shared<BT>& s, const Settings& o, double u) {
  using P = Places<T>;
  constexpr bool BY_VALUE = sizeof(T) == 2 && BT == THREADS;
  const bool greedy = o.greedy(), small_k = o.top_k && o.top_k <= SMALL_K<BT>, only_min_p = !BY_VALUE && o.min_p > 0.0f && !(o.top_p < 1.0f);
  const bool few = o.few(SMALL_K<BT>, !BY_VALUE);
  Reader<T, BT> in(x, columns);
  uint32_t most, there = 0, above = 0, least = 0xFFFFFFFFu;  // above: the lowest value
  if constexpr (BY_VALUE) {
    auto odd = [&](uint4 w, uint32_t c) {
      uint32_t m = 0;
      each<T>(w, c, [&](uint32_t q, uint32_t) {
        m = max(m, q);
        there += q != 0;
        above += q > P::LOWEST;
        if (!few && q > P::LOWEST) count_place(s.large.counters, q);
      });
      return m;
    };
    auto regular = [&](uint32_t n) {
      there += n;
      above += n;
    };
    if (few) {
      most = in.first([&](uint4) { regular(Piece<T>::N); }, odd);
    } else {
      clear_counters(s.large.counters);
      __syncthreads();
      most = in.first([&](uint4 p) {
        regular(Piece<T>::N);
        count_word(s.large.counters, p.x);
        count_word(s.large.counters, p.y);
        count_word(s.large.counters, p.z);
        count_word(s.large.counters, p.w);
      }, odd);
      if (in.last > P::LOWEST) count_place(s.large.counters, in.last);
    }
    there += in.last != 0;
    above += in.last > P::LOWEST;
  } else {
    most = in.first([&](uint4 p) {
      there += Piece<T>::N;
      least = min(least, piece_min<T>(p));
    }, [&](uint4 w, uint32_t c) {
      uint32_t m = 0;
      each<T>(w, c, [&](uint32_t q, uint32_t) {
        m = max(m, q);
        there += q != 0;
        least = q ? min(least, q) : least;
      });
      return m;
    });
    there += in.last != 0;
    least = in.last ? min(least, in.last) : least;
  }
  {
    const uint32_t w = threadIdx.x >> 6;
    s.most[threadIdx.x] = most;
    const uint32_t m = wave_max_u32(most), l = wave_min_u32(least), n = group_scan_u32<64>(there), b = group_scan_u32<64>(above);
    if ((threadIdx.x & 63) == 63) {
      s.wave_most[w] = m;
      s.wave_least[w] = l;
      s.wave_there[w] = n;
      s.wave_above[w] = b;
    }
    __syncthreads();
    most = there = above = 0;
#pragma unroll
    for (int i = 0; i < BT / 64; ++i) {
      most = max(most, s.wave_most[i]);
      least = min(least, s.wave_least[i]);
      there += s.wave_there[i];
      above += s.wave_above[i];
    }
  }
  if (!there) return nothing_to_draw();
  if (greedy) {
    if (threadIdx.x == 0) s.place = SKY_INVALID;
    in.equal(s, most, false, [&](uint32_t c) { atomicMin(&s.place, c); });
    __syncthreads();
    return Result{s.place, 1, 0.0};
  }
  const Row row(o.temperature, P::value(most), fraction_bits(columns));
  if (few || there <= CAP<BT>) {
    uint32_t from = 1;  // places from here on are listed
    if (there > CAP<BT> && small_k) {
      place_for_rank<BT>(s, o.top_k, most);
      from = max(from, s.place);
    }
    if (there > CAP<BT> && only_min_p) {
      // the smallest value that may weigh min_p, with a margin for the logarithm
      const double z = (double)row.zmax + row.t * (log((double)o.min_p) - 1e-6) - 1e-6 * fabs((double)row.zmax);
      from = max(from, min(last_failing<T>(most, [&](float v) { return (double)v >= z; }) + 1, most));
    }
    __syncthreads();
    if (threadIdx.x == 0) s.large.some.l.n = 0;
    in.from(s, from, [&](uint32_t q, uint32_t c) {
      const uint32_t at = atomicAdd(&s.large.some.l.n, 1u);
      if (at < CAP<BT>) s.large.some.l.list[at] = listed(P::value(q), c);
    });
    __syncthreads();
    const uint32_t n = s.large.some.l.n;
    if (n <= CAP<BT>) return draw_list(s.large.some.l, n, o, u);
    __syncthreads();  // more than were expected: equal values, or a small min-p
  }
  if constexpr (BY_VALUE) {
    Result r;
    if (!few && draw_by_value(in, s, row, o, u, most, there, above, &r)) return r;
    __syncthreads();
    return draw_by_bins_apart(in, &s, row, o, u, most, P::value(P::LOWEST), there);
  } else {
    return draw_by_bins(in, s, row, o, u, most, P::value(least), there);
  }
}

// ---------------------------------------------------------------- a few long rows, in parts
// A workgroup alone takes a row of fp32 logits at what a CU reads, three or four times, and where there are few rows most CUs have
// nothing to do.  With a workspace `parts` workgroups share a row, in kernels that follow one another:
//   parts_kernel    each part's largest and smallest place and how many entries are there; of rows that are drawn from by top-k of up to
//                   PART_K or greedily the part's k best, in the order
//   fill_kernel     the mass and the number of the entries of every bin, as draw_by_bins has them
//   collect_kernel  the entries of the bin in which top-p or min-p ends the row, and of those bins in which the drawn unit lies for any end in that
//                   bin (next to always one or two)
//   draw_kernel     the draw from these
// All sums are whole numbers in the same units, so that the ids are the same.  What does not fit (top-k above PART_K, min-p without top-p, rows
// with next to nothing in them, lists that run over) is drawn from by draw_kernel alone.
constexpr uint32_t PART_K = SMALL_K<SHORT_THREADS>, MAX_PARTS = 16, MANY_EQUAL = 0xFFFFFFFFu;
struct RowSpace {  // of a row in the workspace
  uint64_t bin[BINS];
  uint64_t list[CAP<THREADS>];              // what collect_kernel found
  uint64_t part_list[MAX_PARTS][PART_K];
  uint32_t count[BINS];
  uint32_t most[MAX_PARTS], least[MAX_PARTS], there[MAX_PARTS], part_count[MAX_PARTS];
  // by collect_kernel: the bins in which top-p, min-p or the first of them end the row, what lies before the latter's, how many entries
  // do, and the mass of all; the bins [first, last] in which the drawn unit may lie, and what lies before each
  uint64_t end_before, total, start[64];
  uint32_t p, m, end, larger, first, last;
  float z_least;
  uint32_t n;  // entries of `list`, more than it holds where they or the bins are too many
};
struct Parts {
  RowSpace* space;
  uint32_t parts, span;
};
// What the parts have found of a row that is neither greedy nor to be drawn from by a small top-k.
struct Whole {
  uint32_t most, least, there;
  __device__ __forceinline__ Whole(const RowSpace& w, uint32_t parts) {
    const uint32_t lane = threadIdx.x & 63;
    const bool in = lane < parts;
    most = wave_max_u32(in ? w.most[lane] : 0);
    least = wave_min_u32(in ? w.least[lane] : 0xFFFFFFFFu);
    there = (uint32_t)__shfl((int)group_scan_u32<64>(in ? w.there[lane] : 0), 63, 64);
  }
};
// What its parts do with a row: list the best, sum up bins (of a row of more than CAP<THREADS> entries), or nothing.
__device__ __forceinline__ bool listed_in_parts(const Settings& o) { return o.few(PART_K, false); }
__device__ __forceinline__ bool summed_in_parts(const Settings& o) { return !o.greedy() && !o.top_k && !(o.min_p > 0.0f && !(o.top_p < 1.0f)); }
__device__ __forceinline__ Bins bins_of(const Row& row, const Whole& w) {
  const float cut = (float)fmax((double)row.zmax - NO_MASS * row.t, -3.402823466e38);
  return Bins(row.zmax, fmaxf(key_score(w.least), cut));
}
// The smallest value that weighs min_p, by a wavefront: six bits of its place at a time.
__device__ __forceinline__ float least_of_min_p(const Row& row, float min_p, uint32_t most) {
  using P = Places<float>;
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = 0;  // the largest place known to weigh less
#pragma unroll 1
  for (int shift = 26; shift > -6; shift -= 6) {
    const int by = max(shift, 0);
    const uint32_t q = lo | lane << by;
    const bool fails = q <= most && (shift >= 0 || lane < 4) && (q < P::LOWEST || !(row.weight(P::value(q)) >= (double)min_p));
    lo |= (63u - (uint32_t)__builtin_clzll(__ballot(fails) | 1ull)) << by;
  }
  return P::value(min(lo + 1, most));
}

__global__ __launch_bounds__(SHORT_THREADS, 4) void parts_kernel(DrawArgs a, Parts p) {
  constexpr int BT = SHORT_THREADS;
  using T = float;
  using P = Places<T>;
  __shared__ Shared<BT> s;
  ListShared<BT>& l = s.large.some.l;
  const uint32_t r = blockIdx.x / p.parts, part = blockIdx.x % p.parts, start = part * p.span, tid = threadIdx.x;
  RowSpace& w = p.space[r];
  const Settings o(a, r);
  const bool few = listed_in_parts(o);
  if (!few && !summed_in_parts(o)) return;
  Reader<T, BT> in((const T*)a.logits + r * a.stride + start, min(p.span, a.columns - start));
  if (!few) {  // what the next kernels add to
    for (uint32_t i = part * BT + tid; i < BINS; i += p.parts * BT) {
      w.bin[i] = 0;
      w.count[i] = 0;
    }
    if (part == 0 && tid == 0) w.n = 0;
  }
  uint32_t there = 0, least = 0xFFFFFFFFu;
  uint32_t most = in.first([&](uint4 q) {
    there += Piece<T>::N;
    least = min(least, piece_min<T>(q));
  }, [&](uint4 v, uint32_t c) {
    uint32_t m = 0;
    each<T>(v, c, [&](uint32_t q, uint32_t) {
      m = max(m, q);
      there += q != 0;
      least = q ? min(least, q) : least;
    });
    return m;
  });
  there += in.last != 0;
  least = in.last ? min(least, in.last) : least;
  s.most[tid] = most;
  most = wave_max_u32(most);
  least = wave_min_u32(least);
  there = group_scan_u32<64>(there);
  if ((tid & 63) == 63) {
    s.wave_most[tid >> 6] = most;
    s.wave_least[tid >> 6] = least;
    s.wave_there[tid >> 6] = there;
  }
  if (tid == 0) l.n = 0;
  __syncthreads();
  most = there = 0;
#pragma unroll
  for (int i = 0; i < BT / 64; ++i) {
    most = max(most, s.wave_most[i]);
    least = min(least, s.wave_least[i]);
    there += s.wave_there[i];
  }
  if (!few) {
    if (tid == 0) {
      w.most[part] = most;
      w.least[part] = least;
      w.there[part] = there;
    }
    return;
  }
  const uint32_t k = o.greedy() ? 1 : o.top_k;
  uint32_t from = 1;
  if (there > CAP<BT>) {
    place_for_rank<BT>(s, k, most);
    from = max(from, s.place);
  }
  if (there)
    in.from(s, from, [&](uint32_t q, uint32_t c) {
      const uint32_t at = atomicAdd(&l.n, 1u);
      if (at < CAP<BT>) l.list[at] = listed(P::value(q), start + c);
    });
  __syncthreads();
  const uint32_t n = l.n;
  if (n > CAP<BT>) {
    if (tid == 0) w.part_count[part] = MANY_EQUAL;
    return;
  }
  sort_list<BT>(l.list, n);
  const uint32_t m = min(n, k);
  if (tid == 0) w.part_count[part] = m;
  if (tid < m) w.part_list[part][tid] = l.list[tid];
}

// f(four values, their first column, bits of those from `low` on) for the pieces of a part, and for the odd entries one by one; values
// that are not meant are `low`.
template <typename F>
__device__ __forceinline__ void each_of_part(const Reader<float, SHORT_THREADS>& in, float low, F f) {
  using P = Places<float>;
  in.stream([&](uint4 v, uint32_t c) {
    const uint32_t word[4] = {v.x, v.y, v.z, v.w};
    float z[4];
    uint32_t wanted = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = place_of_bits<float>(word[i]);
      const bool mine = q && P::value(q) >= low;
      z[i] = mine ? P::value(q) : low;
      wanted |= mine ? 1u << i : 0u;
    }
    f(z, c, wanted);
  });
  const uint32_t c = in.whole + threadIdx.x;
  if (c < in.columns) {
    const uint32_t q = place_of_bits<float>(__float_as_uint(in.x[c]));
    const float z[4] = {q ? P::value(q) : low, low, low, low};
    f(z, c, q && z[0] >= low ? 1u : 0u);
  }
}

__global__ __launch_bounds__(SHORT_THREADS, 4) void fill_kernel(DrawArgs a, Parts p) {
  __shared__ uint64_t bin[BINS];
  __shared__ uint32_t count[BINS];
  const uint32_t r = blockIdx.x / p.parts, start = blockIdx.x % p.parts * p.span;
  RowSpace& w = p.space[r];
  const Settings o(a, r);
  if (!summed_in_parts(o)) return;
  const Whole whole(w, p.parts);
  if (whole.there <= CAP<THREADS>) return;
  const Row row(o.temperature, key_score(whole.most), fraction_bits(a.columns));
  const Bins bins = bins_of(row, whole);
  for (uint32_t i = threadIdx.x; i < BINS; i += SHORT_THREADS) {
    bin[i] = 0;
    count[i] = 0;
  }
  __syncthreads();
  const Reader<float, SHORT_THREADS> in((const float*)a.logits + r * a.stride + start, min(p.span, a.columns - start));
  each_of_part(in, bins.low, [&](const float (&z)[4], uint32_t, uint32_t wanted) {
    uint64_t units[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) units[i] = row.units(z[i]);  // without branches: beside one another
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (wanted >> i & 1) {
        const uint32_t b = bins.of(z[i]);
        atomicAdd((unsigned long long*)&bin[b], (unsigned long long)units[i]);
        atomicAdd(&count[b], 1u);
      }
  });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < BINS; i += SHORT_THREADS)
    if (count[i]) {
      atomicAdd((unsigned long long*)&w.bin[i], (unsigned long long)bin[i]);
      atomicAdd(&w.count[i], count[i]);
    }
}

__global__ __launch_bounds__(SHORT_THREADS, 4) void collect_kernel(DrawArgs a, Parts p) {
  constexpr int BT = SHORT_THREADS;
  constexpr uint32_t PER = BINS / BT;
  __shared__ Shared<BT> s;
  ListShared<BT>& l = s.large.some.l;
  const uint32_t r = blockIdx.x / p.parts, part = blockIdx.x % p.parts, start = part * p.span, tid = threadIdx.x;
  RowSpace& w = p.space[r];
  const Settings o(a, r);
  if (!summed_in_parts(o)) return;
  // what does not depend on one another is asked for at once: the kernel is a chain of waits
  uint64_t mine[PER], sum = 0, total;  // the thread's bins
  uint32_t counts[PER];
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) mine[i] = w.bin[PER * tid + i];
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) counts[i] = w.count[PER * tid + i];
  const double u = uniform_of(a, r);
  const Whole whole(w, p.parts);
  if (whole.there <= CAP<THREADS>) return;
  const Row row(o.temperature, key_score(whole.most), fraction_bits(a.columns));
  const Bins bins = bins_of(row, whole);
  const float z_least = o.min_p > 0.0f ? least_of_min_p(row, o.min_p, whole.most) : 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) sum += mine[i];
  if (tid == 0) l.n = 0;
  const uint64_t before = block_scan<BT>(sum, s.wave, &total);
  auto each_own = [&](auto f) {
    uint64_t at = before;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
      f(PER * tid + i, at, mine[i]);
      at += mine[i];
    }
  };
  auto bin_of = [&](uint64_t unit) {  // the bin that holds a unit of mass
    __syncthreads();
    each_own([&](uint32_t b, uint64_t at, uint64_t size) {
      if (at <= unit && unit < at + size) s.found = b;
    });
    __syncthreads();
    return s.found;
  };
  const uint32_t by_p = o.top_p < 1.0f ? bin_of(Row::needed(o.top_p, total) - 1) : BINS;
  const uint32_t by_m = o.min_p > 0.0f && bins.has(z_least) ? bins.of(z_least) : BINS, end = min(by_p, by_m);
  uint64_t least = total, most = total, end_before = 0;  // of what stays
  if (end < BINS) {
    __syncthreads();
    each_own([&](uint32_t b, uint64_t at, uint64_t size) {
      if (b == end) {
        s.mass_before = at;
        s.count_before = size;
      }
    });
    __syncthreads();
    end_before = s.mass_before;
    least = max(end_before, (uint64_t)1);
    most = end_before + s.count_before;
  }
  const uint32_t first = bin_of(Row::drawn(u, least)), last = bin_of(Row::drawn(u, most));
  constexpr uint32_t STARTS = sizeof(w.start) / sizeof(w.start[0]);
  if (part == 0) {
    each_own([&](uint32_t b, uint64_t at, uint64_t) {
      if (b >= first && b <= last && b - first < STARTS) w.start[b - first] = at;
    });
    uint64_t many = 0, larger;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) many += PER * tid + i < end ? counts[i] : 0;
    block_scan<BT>(many, s.wave, &larger);
    if (tid == 0) {
      w.end_before = end_before;
      w.total = total;
      w.p = by_p;
      w.m = by_m;
      w.end = end;
      w.larger = (uint32_t)larger;
      w.first = first;
      w.last = last;
      w.z_least = z_least;
      if (last - first >= STARTS) atomicAdd(&w.n, CAP<THREADS> + 1);
    }
  }
  const Reader<float, BT> in((const float*)a.logits + r * a.stride + start, min(p.span, a.columns - start));
  each_of_part(in, bins.low, [&](const float (&z)[4], uint32_t c, uint32_t wanted) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = bins.of(z[i]);
      found |= b == end || (b >= first && b <= last) ? 1u << i : 0u;
    }
    found &= wanted;
    if (found)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (found >> i & 1) {
          const uint32_t at = atomicAdd(&l.n, 1u);
          if (at < CAP<BT>) l.list[at] = listed(z[i], start + c + i);
        }
  });
  __syncthreads();
  const uint32_t n = l.n;
  if (tid == 0 && n) s.place = atomicAdd(&w.n, n > CAP<BT> ? CAP<THREADS> + 1 : n);
  __syncthreads();
  const uint32_t at = s.place;
  for (uint32_t i = tid; i < min(n, CAP<BT>); i += BT)
    if (at + i < CAP<THREADS>) w.list[at + i] = l.list[i];
}

// The draw from what the parts have left; false: it is none of theirs.
__device__ __forceinline__ bool draw_collected(Shared<THREADS>& s, const RowSpace& w, uint32_t parts, uint32_t columns, const Settings& o, double u, Result* d) {
  static_assert(CAP<THREADS> == 2 * THREADS, "two entries a thread");
  const uint32_t lane = threadIdx.x & 63, n = w.n, end = w.end, by_p = w.p, by_m = w.m, first = w.first, last = w.last, larger = w.larger;
  const uint64_t total = w.total, end_before = w.end_before, starts = w.start[lane], start = lane <= last - first ? starts : ~0ull;
  const uint64_t listed0 = w.list[threadIdx.x], listed1 = w.list[THREADS + threadIdx.x];  // whatever they are beyond n
  const float z_least = w.z_least;
  const Whole whole(w, parts);
  if (!whole.there) {
    *d = nothing_to_draw();
    return true;
  }
  if (whole.there <= CAP<THREADS> || n > CAP<THREADS>) return false;
  const Row row(o.temperature, key_score(whole.most), fraction_bits(columns));
  const Bins bins = bins_of(row, whole);
  uint64_t* const list = s.large.some.l.list;
  list[threadIdx.x] = listed0;
  list[THREADS + threadIdx.x] = listed1;
  __syncthreads();
  sort_list<THREADS>(list, n);
  uint32_t bin[2], many = 0;
  uint64_t mass[2], weighs = 0, sum;
  bool begins[2];  // a bin's entries
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t at = 2 * threadIdx.x + i;
    const float z = at < n ? listed_score(list[at]) : row.zmax;
    bin[i] = at < n ? bins.of(z) : BINS + 1;
    begins[i] = at < n && (at == 0 || bins.of(listed_score(list[at - 1])) != bin[i]);
    mass[i] = row.units(z);
    if (at >= n) mass[i] = 0;
    if (bin[i] == by_m && z >= z_least) {
      ++many;
      weighs += mass[i];
    }
  }
  const uint64_t before = block_scan<THREADS>(mass[0] + mass[1], s.wave, &sum), own[2] = {before, before + mass[0]};
  // f(entry, the bin's first, what lies before the entry, its mass) for the entries of bin b, before which `at` lies
  auto in_bin = [&](uint32_t b, uint64_t at, auto f) {
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
      if (bin[i] == b && begins[i]) {
        s.place = 2 * threadIdx.x + i;
        s.count_before = own[i];
      }
    __syncthreads();
    const uint32_t from = s.place;
    at -= s.count_before;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
      if (bin[i] == b) f(2 * threadIdx.x + i, from, at + own[i], mass[i]);
    __syncthreads();
  };
  uint64_t all = total, count = whole.there;
  if (by_p == end && end < BINS) {
    const uint64_t unit = Row::needed(o.top_p, total) - 1;
    in_bin(end, end_before, [&](uint32_t at, uint32_t from, uint64_t b, uint64_t size) {
      if (b <= unit && unit < b + size) {
        s.mass_before = b + size;
        s.found = at - from + 1;
      }
    });
    all = s.mass_before;
    count = larger + s.found;
  }
  if (by_m == end && end < BINS) {
    uint64_t n_least, mass_least;
    block_scan<THREADS>(many, s.wave, &n_least);
    block_scan<THREADS>(weighs, s.wave, &mass_least);
    if (larger + n_least < count) {
      count = larger + n_least;
      all = end_before + mass_least;
    }
  }
  // of the bins that may hold it the last that begins before the drawn unit or with it does
  const uint64_t unit = Row::drawn(u, all);
  const int which = 63 - (int)__builtin_clzll(__ballot(start <= unit));
  in_bin(first + (uint32_t)which, shfl_u64(start, which), [&](uint32_t at, uint32_t, uint64_t b, uint64_t size) {
    if (b <= unit && unit < b + size) s.chunk = at;
  });
  const uint64_t e = list[s.chunk];
  *d = Result{(uint32_t)e, (uint32_t)count, row.log_share(listed_score(e), all)};
  return true;
}
// The draw from the lists of a row's parts; false: one of them is none.  The j-th entries of all parts, j = k / parts rounded up, have
// k entries up to the last of them: what comes after that one is not among the k best.
__device__ __forceinline__ bool draw_joined(ListShared<THREADS>& s, const RowSpace& w, uint32_t parts, const Settings& o, double u, Result* d) {
  constexpr int BT = THREADS;
  static_assert(MAX_PARTS * PART_K == 2 * BT && 2 * BT <= CAP<BT> && PART_K % 64 == 0, "two entries a thread, a wavefront in one list at a time");
  const uint32_t lane = threadIdx.x & 63, k = o.greedy() ? 1 : o.top_k, j = (k + parts - 1) / parts;
  // everything is asked for at once; beyond the parts and their counts it is whatever was there
  const uint32_t n = w.part_count[lane % MAX_PARTS], count = lane < parts ? n : 0;
  const uint64_t jth = w.part_list[lane % MAX_PARTS][j - 1];
  uint64_t e[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) e[i] = w.part_list[(i * BT + threadIdx.x) / PART_K][threadIdx.x % PART_K];
  if (threadIdx.x == 0) s.n = 0;
  if (__ballot(count == MANY_EQUAL)) return false;  // every wavefront sees the same counts
  uint64_t last = lane >= parts ? 0 : count >= j ? jth : LIST_END;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) last = max(last, shfl_xor_u64(last, m));
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t entries = (uint32_t)__shfl((int)count, (int)((i * BT + threadIdx.x) / PART_K), 64);
    if (threadIdx.x % PART_K < entries && e[i] <= last) s.list[atomicAdd(&s.n, 1u)] = e[i];
  }
  __syncthreads();
  const uint32_t m = s.n;
  *d = !m ? nothing_to_draw() : o.greedy() ? first_listed(s, m) : draw_list(s, m, o, u);
  return true;
}

// A workgroup of 1024 threads has a row; `left`: only the rows that draw_short_kernel has left.  PARTS: rows that their parts have been
// at (a kernel of its own: the others do without its registers).
template <typename T, bool PARTS>
__global__ __launch_bounds__(THREADS) void draw_kernel(DrawArgs a, bool left, Parts p) {
  __shared__ Shared<THREADS> s;
  const uint32_t r = blockIdx.x;
  if (left && a.tokens[r * a.tokens_stride] != NOT_DRAWN) return;
  const Settings o(a, r);
  const double u = uniform_of(a, r);
  Result d;
  bool done = false;
  if constexpr (PARTS) {
    const RowSpace& w = p.space[r];
    if (listed_in_parts(o))
      done = draw_joined(s.large.some.l, w, p.parts, o, u, &d);
    else if (summed_in_parts(o))
      done = draw_collected(s, w, p.parts, a.columns, o, u, &d);
    __syncthreads();
  }
  if (!done) d = draw_row<T, THREADS>((const T*)a.logits + r * a.stride, a.columns, s, o, u);
  if (threadIdx.x == 0) store_result(a, r, d);
}

// A workgroup of 256 threads has a row, four or more of them a CU: one's loads run beside another's sort.  In longer rows the first
// columns tell whether most entries are not there; such a row is listed as it is read.  `leave`: rows of which many entries can stay are
// left to draw_kernel.
constexpr uint32_t SAMPLE_FROM = 8192;
template <typename T>
__global__ __launch_bounds__(SHORT_THREADS, 4) void draw_short_kernel(DrawArgs a, bool leave) {
  constexpr uint32_t N = Piece<T>::N, STEP = SHORT_THREADS * N, LOADS = 8, LIST = CAP<SHORT_THREADS>;
  using P = Places<T>;
  __shared__ Shared<SHORT_THREADS> s;
  ListShared<SHORT_THREADS>& l = s.large.some.l;
  const uint32_t r = blockIdx.x, tid = threadIdx.x, columns = a.columns, whole = columns / N * N;
  const T* const x = (const T*)a.logits + r * a.stride;
  const Settings o(a, r);
  const bool few = o.few(SMALL_K<SHORT_THREADS>, true);
  if (columns > SAMPLE_FROM && !few) {
    if (tid == 0) l.n = 0;
    __syncthreads();
    auto put = [&](uint32_t q, uint32_t c) {
      if (q) {
        const uint32_t at = atomicAdd(&l.n, 1u);
        if (at < LIST) l.list[at] = listed(P::value(q), c);
      }
    };
    auto piece = [&](uint4 w, uint32_t c) {
      if (piece_max<T>(raw_places<T>(w)) >= P::LOWEST) each<T>(w, c, put);
    };
    piece(load_words(x + tid * N), tid * N);
    __syncthreads();
    const uint32_t seen = l.n;
    __syncthreads();
    if ((uint64_t)seen * columns <= (uint64_t)2 * LIST * STEP) {
      uint32_t c0 = STEP;
      for (; c0 + LOADS * STEP <= whole; c0 += LOADS * STEP) {
        uint4 w[LOADS];
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) w[i] = load_words(x + c0 + i * STEP + tid * N);
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) piece(w[i], c0 + i * STEP + tid * N);
      }
      for (uint32_t c = c0 + tid * N; c < whole; c += STEP) piece(load_words(x + c), c);
      if (whole + tid < columns) put(place_of(x[whole + tid]), whole + tid);
      __syncthreads();
      const uint32_t n = l.n;
      if (n <= LIST) {
        const Result d = n ? draw_list(l, n, o, uniform_of(a, r)) : nothing_to_draw();
        if (tid == 0) store_result(a, r, d);
        return;
      }
      __syncthreads();
    }
  }
  if (leave && !few) {
    if (tid == 0) a.tokens[r * a.tokens_stride] = NOT_DRAWN;
    return;
  }
  const Result d = draw_row<T, SHORT_THREADS>(x, columns, s, o, uniform_of(a, r));
  if (tid == 0) store_result(a, r, d);
}

// Which workgroups draw.  One of 256 threads for a row that is short, and for any where there are more rows than CUs: four of them share a
// CU.  16-bit logits are the exception: a long row of which many entries can stay is drawn from by value, which takes a CU.  (us, 1024 /
// 256 threads: 2,000 x 8,000 bf16 by top-p 146 / 76, top-k of 50 80 / 23; 1,000 x 20,000 by top-p 82 / 74, 400 x 30,000 42 / 63,
// 256 x 131,072 37 / 253; 400 x 100,000 top-k of 50 33 / 25; fp32 100 x 20,000 by top-p 46 / 39, 600 x 100,000 322 / 244,
// 40 x 100,003 top-k of 40 18 / 23.)  The lengths come from 100 rows and more.  With fewer rows than CUs they do not hold for all: 40 x 20,000 bf16
// by top-p 21 / 38, by top-k of 300 and top-p 20 / 55, by top-k of 50 11 / 11, 40 x 5,000 19 / 21, 22 / 30 and 13 / 9, 40 x 1,000 22 / 16, 21 / 23
// and 20 / 9; fp32 40 x 20,000 44 / 40, 23 / 59 and 15 / 12, 40 x 32,768 52 / 52, 23 / 80 and 15 / 14, 40 x 5,000 36 / 21, 23 / 31 and 14 / 9.  One row
// and 200 are as 40 are.  So a few rows of 16 bits above some 5,000, and those by a top-k of 129 to 512, would be drawn from faster by 1024 threads.
constexpr uint32_t SHORT_ROW_16 = 20480, SHORT_ROW_32 = 32768, MANY_ROWS = 256;
// Parts of a row: two workgroups a CU, of at least 4,096 columns each, eight and more.  What rows of few candidates lose is the launches of
// kernels that have nothing to do with them.  (us, a workgroup a row / in parts, fp32: 8 x 131,072 by top-p 114 / 48, top-k of 50
// 19 / 21, of 400 34 / 42; 40 x 100,003 by top-p 95 / 50, top-k of 40 19 / 22; 128 x 100,003, by four, 107 / 95 and 27 / 31.  16-bit rows, whose values are
// counted: 65,536 by top-k of 50 11 / 17.  40 x 100,003, every row its own settings: 21 / 23, and 100-130 / 46 if one row of the 40 has no top-k.)
Parts parts_of(size_t size, uint32_t rows, uint32_t columns, void* workspace) {
  Parts p{};
  if (size != 4 || !rows || columns <= SHORT_ROW_32) return p;
  const uint32_t parts = std::min(std::min(2 * 256 / rows, columns / 4096), MAX_PARTS);
  if (parts < 8) return p;
  p.span = ((columns + parts - 1) / parts + 63) / 64 * 64;
  p.parts = (columns + p.span - 1) / p.span;
  p.space = (RowSpace*)workspace;
  return p;
}

template <typename T>
void launch_draw(const DrawArgs& a, const Parts& p, hipStream_t st) {
  const dim3 grid(a.rows), few(SHORT_THREADS), all(THREADS);
  const bool many = a.rows > MANY_ROWS;
  if constexpr (sizeof(T) == 4) {
    if (many || a.columns <= SHORT_ROW_32) {
      hipLaunchKernelGGL(draw_short_kernel<T>, grid, few, 0, st, a, false);
    } else if (p.parts) {
      const dim3 parts(a.rows * p.parts);
      hipLaunchKernelGGL(parts_kernel, parts, few, 0, st, a, p);
      hipLaunchKernelGGL(fill_kernel, parts, few, 0, st, a, p);
      hipLaunchKernelGGL(collect_kernel, parts, few, 0, st, a, p);
      hipLaunchKernelGGL((draw_kernel<T, true>), grid, all, 0, st, a, false, p);
    } else {
      hipLaunchKernelGGL((draw_kernel<T, false>), grid, all, 0, st, a, false, p);
    }
  } else if (a.columns <= SHORT_ROW_16) {
    hipLaunchKernelGGL(draw_short_kernel<T>, grid, few, 0, st, a, false);
  } else if (many) {
    hipLaunchKernelGGL(draw_short_kernel<T>, grid, few, 0, st, a, true);
    hipLaunchKernelGGL((draw_kernel<T, false>), grid, all, 0, st, a, true, p);
  } else {
    hipLaunchKernelGGL((draw_kernel<T, false>), grid, all, 0, st, a, false, p);
  }
}

}  // namespace
}  // namespace sky

using namespace sky;

extern "C" int sky_logits_draw_workspace(int dtype, uint32_t rows, uint32_t columns, uint64_t* bytes) {
  uint64_t stride = 0;
  if (!bytes) return fail(SKY_ERR_ARG, "sky_logits_draw_workspace: null output");
  SKY_TRY(check_rows("sky_logits_draw_workspace", "logits", bytes, dtype, rows, columns, &stride));
  *bytes = parts_of(dtype_size(dtype), rows, columns, nullptr).parts ? rows * sizeof(RowSpace) : 0;
  return SKY_OK;
}

extern "C" int sky_logits_draw(const void* logits, int dtype, uint32_t rows, uint32_t columns, uint64_t row_stride,
                               const sky_draw_rules* rules, const double* uniforms, uint64_t philox_seed, uint32_t first_walker,
                               uint32_t step, uint32_t* tokens, uint64_t tokens_stride, float* logprobs, uint32_t* kept,
                               void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* const who = "sky_logits_draw";
  SKY_TRY(check_rows(who, "logits", logits, dtype, rows, columns, &row_stride));
  if (columns > MAX_COLUMNS) return fail(SKY_ERR_LIMIT, "sky_logits_draw: more than 2^26 columns");
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
  if (!tokens_stride) tokens_stride = 1;
  const hipStream_t st = (hipStream_t)stream;
  for (uint32_t r = 0; r < rows; r += SLICE) {
    auto from = [&](auto* p) { return p ? p + r : p; };
    const DrawArgs a{(const char*)logits + r * row_stride * dtype_size(dtype), row_stride, columns, std::min(SLICE, rows - r), from(d.temperature),
                     from(d.top_k), from(d.top_p), from(d.min_p), from(uniforms), philox_seed, first_walker + r, step,
                     tokens + r * tokens_stride, tokens_stride, from(logprobs), from(kept)};
    const Parts p = workspace ? parts_of(dtype_size(dtype), rows, columns, workspace) : Parts{};
    if (dtype == SKY_F32)
      launch_draw<float>(a, p, st);
    else if (dtype == SKY_F16)
      launch_draw<_Float16>(a, p, st);
    else
      launch_draw<__bf16>(a, p, st);
    SKY_TRY(check_launch());
  }
  return SKY_OK;
}
