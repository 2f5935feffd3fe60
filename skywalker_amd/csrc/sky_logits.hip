// Logits made ready for a draw (sky_logits_adjust).  For row r and column t, in fp32, rounded to the type once:
//   y = x                                      seen(t): t is in the row's history, n(t): how often from history_first on
//   y = x > 0 ? x / rep : x * rep              if seen(t)
//   y = y - (presence + frequency * n(t))      if n(t) > 0
//   y = y + bias(t)
//   y = -inf                                   if a mask or the graph's row does not allow t
// One pass: every logit is read once at most and written once, before anything overwrites it, so that a call may work in place.
//
// adjust_kernel: a workgroup has a tile of a row, 16 columns a thread, and turns the sparse parts (history, biases, neighbours) into
// arrays over the tile's columns in LDS: counts by integer atomics, whose order does not matter, biases by the thread that
// meets the first of equal ids.  All of a row's tiles read its whole history, from L2.  A chain of waits rather than bytes: 61 rows of
// 100,003 bf16 with histories of up to 2,047 ids, 300 biases and masks 16 us, 1.5 TB/s; one row of 65,536 4.4 us.
//
// adjust_near_kernel: rows that a graph holds to a vertex's neighbours, up to NEAR of them.  A workgroup has a row: the neighbours
// go into a hash table in LDS, where history and biases look themselves up, their logits into registers; the row is filled with
// -inf by a stream of stores, and the neighbours are put in.  Nothing else of the logits is read.  (4,096 rows of 65,536 f16:
// tiles 234 us, most of it the wait for state, row bounds and neighbours, eight times a row; so 109, of which the stores alone are
// 99.)  Rows with more neighbours are done tile by tile by their workgroup.
#include "sky_graph.h"
#include "sky_scores.h"

namespace sky {
namespace {

constexpr uint32_t COLS = 16;                // columns of a thread
constexpr uint32_t MAX_COLUMNS = 1u << 30;   // places of tiles are ints, and a tile may end behind the row
constexpr uint32_t SEEN = 0x80000000u;       // in the history, before history_first
constexpr uint32_t BIAS_SEARCH_MIN = 2048u;  // from so many biases on a tile looks for its own by bisection (two chains of some 12 loads)

struct AdjustArgs {
  const void* logits;
  void* out;
  uint64_t stride, out_stride;
  uint32_t columns, tiles;
  sky_logits_rules r;
  const uint32_t* xadj;
  const uint32_t* adjncy;
  uint32_t V;
};

__device__ __forceinline__ uint32_t lower_bound(const uint32_t* a, uint32_t lo, uint32_t hi, uint32_t key) {
  while (lo < hi) {
    const uint32_t m = lo + (hi - lo) / 2;
    if (a[m] < key)
      lo = m + 1;
    else
      hi = m;
  }
  return lo;
}

// Where a row's history and biases lie: asked for before anything that waits.
struct Sparse {
  uint32_t n, from, begin, end;
  __device__ __forceinline__ Sparse(const AdjustArgs& a, uint32_t row) {
    n = !a.r.history ? 0 : a.r.history_lengths ? min(a.r.history_lengths[row], a.r.history_columns) : a.r.history_columns;
    from = a.r.history_first ? a.r.history_first[row] : 0u;
    begin = a.r.bias_ids ? min(a.r.bias_offsets[row], a.r.bias_count) : 0;
    end = a.r.bias_ids ? min(a.r.bias_offsets[row + 1], a.r.bias_count) : 0;
  }
};
// The history of a row: f(id, counted) for each.  Eight loads at a time.
template <typename F>
__device__ __forceinline__ void each_of_history(const AdjustArgs& a, uint32_t row, const Sparse& p, F f) {
  const uint32_t n = p.n, from = p.from;
  const uint32_t* const h = a.r.history + row * a.r.history_stride;
  for (uint32_t base = threadIdx.x; base < n; base += 8 * blockDim.x) {
    uint32_t id[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) id[i] = base + i * blockDim.x < n ? h[base + i * blockDim.x] : SKY_INVALID;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      if (id[i] < a.columns) f(id[i], base + i * blockDim.x >= from);
  }
}
// The biases of a row between two columns: f(id, sum of its values) for each id.
template <typename F>
__device__ __forceinline__ void each_bias(const AdjustArgs& a, const Sparse& p, uint32_t lowest, uint32_t end_column, F f) {
  const uint32_t begin = p.begin, end = p.end;
  uint32_t lo = begin, hi = end;
  if (hi > lo && hi - lo > BIAS_SEARCH_MIN) {
    lo = lower_bound(a.r.bias_ids, lo, hi, lowest);
    hi = lower_bound(a.r.bias_ids, lo, hi, end_column);
  }
  for (uint32_t i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    const uint32_t id = a.r.bias_ids[i];
    if (id < a.columns && (i == begin || a.r.bias_ids[i - 1] != id)) {
      float sum = a.r.bias_values[i];
      for (uint32_t j = i + 1; j < end && a.r.bias_ids[j] == id; ++j) sum += a.r.bias_values[j];
      f(id, sum);
    }
  }
}
// What becomes of a logit that is allowed.
struct Change {
  float rep, presence, frequency;
  __device__ __forceinline__ Change(const AdjustArgs& a, uint32_t row) {
    const bool history = a.r.history != nullptr;
    rep = history && a.r.repetition ? a.r.repetition[row] : 1.0f;
    presence = history && a.r.presence ? a.r.presence[row] : 0.0f;
    frequency = history && a.r.frequency ? a.r.frequency[row] : 0.0f;
  }
  // n: how often it was counted, and SEEN
  __device__ __forceinline__ float of(float s, uint32_t n) const {
    if (n) {
      s = s > 0.0f ? s / rep : s * rep;
      if (n & ~SEEN) s -= presence + frequency * (float)(n & ~SEEN);
    }
    return s;
  }
};

// Tile t of a row, by the workgroup; `lds`: a word a column for a history, one for biases, a bit for a graph.
template <typename T>
__device__ __forceinline__ void adjust_tile(const AdjustArgs& a, uint32_t row, uint32_t t, uint32_t* lds) {
  constexpr int N = Piece<T>::N, NV = COLS / N;
  const uint32_t threads = blockDim.x, tid = threadIdx.x, tile = COLS * threads;
  const T* const x = (const T*)a.logits + row * a.stride;
  T* const y = (T*)a.out + row * a.out_stride;
  // tiles begin where stores are aligned
  const int phase = (int)((uintptr_t)y / sizeof(T) % N), first = (int)(t * tile) - phase, columns = (int)a.columns;
  if (first >= columns) return;
  const uint32_t c0 = (uint32_t)first;  // may wrap: column - c0 is the place in the tile all the same
  const bool history = a.r.history != nullptr, biased = a.r.bias_ids != nullptr, graph = a.xadj != nullptr;
  uint32_t mask_row = SKY_INVALID;  // of the bit masks
  bool none = false;                // nothing of the row is allowed
  if (a.r.allowed) {
    mask_row = a.r.allowed_row ? a.r.allowed_row[row] : a.r.allowed_rows == 1 ? 0u : row;
    none = mask_row != SKY_INVALID && mask_row >= a.r.allowed_rows;
  }
  const bool masked = mask_row != SKY_INVALID && !none;
  const bool whole_tile = first >= 0 && first + (int)tile <= columns;
  const Sparse sparse(a, row);
  const Change change(a, row);

  Piece<T> v[NV];
  uint32_t stay[NV];  // bits of the elements that masks leave
  auto column = [&](int i) { return first + (int)((i * threads + tid) * N); };
  auto whole = [&](int c) { return whole_tile || (c >= 0 && c + N <= columns); };
  auto load = [&](int i) {  // pieces that are not whole are read element by element
    if (whole(column(i))) v[i] = load_piece(x + column(i));
  };
  const bool early = !graph && !none;  // the row is needed (a mask leaves something of most pieces): its loads run beside the scans below
  if (early) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load(i);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column(i);
    stay[i] = none ? 0u : (1u << N) - 1;
    if (masked) {
      const uint32_t* const m = a.r.allowed + mask_row * a.r.allowed_stride;
      if (whole(c)) {
        const uint64_t lo = m[(uint32_t)c >> 5], hi = m[(uint32_t)(c + N - 1) >> 5];
        stay[i] &= (uint32_t)((lo | hi << 32) >> (c & 31));
      } else {
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (c + e >= 0 && c + e < columns) bits |= (m[(uint32_t)(c + e) >> 5] >> ((c + e) & 31) & 1u) << e;
        stay[i] &= bits;
      }
    }
  }

  uint32_t* const count = lds;
  float* const bias = (float*)(lds + (history ? tile : 0u));
  uint32_t* const can = lds + (history ? tile : 0u) + (biased ? tile : 0u);
  const uint32_t words = (history ? tile : 0u) + (biased ? tile : 0u) + (graph ? tile / 32 : 0u);
  if (words && !none) {
    for (uint32_t i = tid; i < words / 4; i += threads) ((uint4*)lds)[i] = uint4{0, 0, 0, 0};
    __syncthreads();
    if (history)
      each_of_history(a, row, sparse, [&](uint32_t id, bool counted) {
        const uint32_t at = id - c0;
        if (at < tile) {
          if (counted)
            atomicAdd(&count[at], 1u);
          else
            atomicOr(&count[at], SEEN);
        }
      });
    if (biased)
      each_bias(a, sparse, (uint32_t)max(first, 0), (uint32_t)min((int64_t)first + tile, (int64_t)columns), [&](uint32_t id, float sum) {
        if (id - c0 < tile) bias[id - c0] = sum;
      });
    if (graph) {
      const uint32_t s = a.r.states[row * a.r.states_stride];
      if (s < a.V) {
        const uint32_t hi = a.xadj[s + 1];
        for (uint32_t i = a.xadj[s] + tid; i < hi; i += threads) {
          const uint32_t id = a.adjncy[i], at = id - c0;
          if (at < tile && id < a.columns) atomicOr(&can[at >> 5], 1u << (at & 31));
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column(i);
    const uint32_t at = (i * threads + tid) * N;
    if (graph && !none) stay[i] &= can[at >> 5] >> (at & 31);  // N divides 32: the piece's bits lie in one word
    if (!early && stay[i]) load(i);
    auto adjusted = [&](T logit, uint32_t e) {
      float s = (float)logit;
      if (history) s = change.of(s, count[at + e]);
      if (biased) s += bias[at + e];
      return (T)(stay[i] >> e & 1u ? s : -__builtin_inff());
    };
    if (whole(c)) {
      Piece<T> o;
      float s[N];
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = (float)v[i].e[e];
      if (history) {
        uint32_t n[N], any = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) any |= n[e] = count[at + e];
        if (any)  // of most pieces nothing was visited
#pragma unroll
          for (int e = 0; e < N; ++e) s[e] = change.of(s[e], n[e]);
      }
      if (biased)
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += bias[at + e];
      if (__builtin_expect(stay[i] != (1u << N) - 1, 1))
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] = stay[i] >> e & 1u ? s[e] : -__builtin_inff();
#pragma unroll
      for (int e = 0; e < N; ++e) o.e[e] = (T)s[e];
      store_piece(y + c, o);
    } else {
#pragma unroll 1
      for (int e = 0; e < N; ++e)
        if (c + e >= 0 && c + e < columns) y[c + e] = adjusted(x[c + e], e);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(512) void adjust_kernel(AdjustArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  adjust_tile<T>(a, blockIdx.x / a.tiles, blockIdx.x % a.tiles, lds);
}

constexpr uint32_t NEAR_THREADS = 256, NEAR = 1024, SLOTS = 2 * NEAR;  // the table is half full at most
template <typename T>
__global__ __launch_bounds__(NEAR_THREADS) void adjust_near_kernel(AdjustArgs a) {
  constexpr uint32_t N = Piece<T>::N, EACH = NEAR / NEAR_THREADS;
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];  // key, count and bias of a slot, or what a tile takes
  uint32_t* const key = lds;
  uint32_t* const count = lds + SLOTS;
  float* const bias = (float*)(lds + 2 * SLOTS);
  const uint32_t tid = threadIdx.x, row = blockIdx.x;
  const T* const x = (const T*)a.logits + row * a.stride;
  T* const y = (T*)a.out + row * a.out_stride;
  const uint32_t state = a.r.states[row * a.r.states_stride];
  uint32_t lo = 0, hi = 0;
  if (state < a.V) {
    lo = a.xadj[state];
    hi = a.xadj[state + 1];
  }
  if (hi - lo > NEAR) {
    for (uint32_t t = 0; t < a.tiles; ++t) {
      adjust_tile<T>(a, row, t, lds);
      __syncthreads();
    }
    return;
  }
  const uint32_t* mask = nullptr;
  if (a.r.allowed) {
    const uint32_t m = a.r.allowed_row ? a.r.allowed_row[row] : a.r.allowed_rows == 1 ? 0u : row;
    if (m != SKY_INVALID) {
      if (m >= a.r.allowed_rows)
        hi = lo;  // nothing
      else
        mask = a.r.allowed + m * a.r.allowed_stride;
    }
  }
  const bool tables = a.r.history || a.r.bias_ids;
  const Sparse sparse(a, row);
  uint32_t id[EACH], slot[EACH];
  float value[EACH];
  // Every element is written once: of `if (...) id[i] = SKY_INVALID` behind the loads the compiler (ROCm 7.2) kept the first element's
  // write alone, and masks did not reach the others.
#pragma unroll
  for (uint32_t i = 0; i < EACH; ++i) {
    const uint32_t j = lo + tid + i * NEAR_THREADS, v = j < hi ? a.adjncy[j] : SKY_INVALID;
    uint32_t bits = v < a.columns ? 1u : 0u;
    if (mask && bits) bits = mask[v >> 5] >> (v & 31);
    id[i] = bits & 1u ? v : SKY_INVALID;
  }
#pragma unroll
  for (uint32_t i = 0; i < EACH; ++i) value[i] = id[i] != SKY_INVALID ? (float)x[id[i]] : 0.0f;
  if (tables) {
    auto first_slot = [](uint32_t v) { return (v * 0x9E3779B1u) >> 21; };
    static_assert(SLOTS == 1u << 11, "of 11 bits");
    for (uint32_t i = tid; i < SLOTS; i += NEAR_THREADS) {
      key[i] = SKY_INVALID;
      count[i] = 0;
      bias[i] = 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i)
      if (id[i] != SKY_INVALID) {
        uint32_t s = first_slot(id[i]);
        for (;;) {
          const uint32_t was = atomicCAS(&key[s], SKY_INVALID, id[i]);
          if (was == SKY_INVALID || was == id[i]) break;
          s = (s + 1) & (SLOTS - 1);
        }
        slot[i] = s;
      }
    __syncthreads();
    auto find = [&](uint32_t v) {  // its slot; one without its key: it is none of the neighbours
      uint32_t s = first_slot(v);
      while (key[s] != v && key[s] != SKY_INVALID) s = (s + 1) & (SLOTS - 1);
      return s;
    };
    if (a.r.history)
      each_of_history(a, row, sparse, [&](uint32_t v, bool counted) {
        const uint32_t s = find(v);
        if (key[s] == v) {
          if (counted)
            atomicAdd(&count[s], 1u);
          else
            atomicOr(&count[s], SEEN);
        }
      });
    if (a.r.bias_ids)
      each_bias(a, sparse, 0, a.columns, [&](uint32_t v, float sum) {
        const uint32_t s = find(v);
        if (key[s] == v) bias[s] = sum;
      });
  }
  auto settled = [] {  // what this thread has loaded and stored is done, and every thread's is
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
  };
  settled();  // no store before every neighbour's logit is here: the call may work in place
  // the row without its neighbours: whole pieces where stores are aligned, elements before and after
  const T gone = (T)-__builtin_inff();
  Piece<T> none;
#pragma unroll
  for (uint32_t e = 0; e < N; ++e) none.e[e] = gone;
  const uint32_t head = min((uint32_t)((16 - (uintptr_t)y % 16) % 16 / sizeof(T)), a.columns), pieces = (a.columns - head) / N;
  // Every row from a place of its own: rows of a power of two apart would all be at the same channel of memory at a time (4,096 rows
  // of 128 KB 325 us instead of 110).
  const uint32_t shift = (uint32_t)((uint64_t)pieces * (row * 0x9E3779B1u) >> 32) & ~(NEAR_THREADS - 1);
  for (uint32_t i = tid; i < pieces; i += NEAR_THREADS) {
    const uint32_t p = i + shift;
    store_piece(y + head + (p < pieces ? p : p - pieces) * N, none);
  }
  if (tid < head) y[tid] = gone;
  if (head + pieces * N + tid < a.columns) y[head + pieces * N + tid] = gone;
  settled();  // the neighbours' stores come after those; counts and biases are whole
  const Change change(a, row);
#pragma unroll
  for (uint32_t i = 0; i < EACH; ++i)
    if (id[i] != SKY_INVALID) {
      float v = value[i];
      if (a.r.history) v = change.of(v, count[slot[i]]);
      if (a.r.bias_ids) v += bias[slot[i]];
      y[id[i]] = (T)v;
    }
}

int check_rules(const sky_logits_rules* r, uint32_t rows, uint32_t columns, AdjustArgs* a) {
  const char* const who = "sky_logits_adjust";
  auto arg = [&](const char* what) { return fail(SKY_ERR_ARG, std::string(who) + ": " + what); };
  a->xadj = a->adjncy = nullptr;
  a->V = 0;
  if (!r) {
    a->r = sky_logits_rules{};
    return SKY_OK;
  }
  a->r = *r;
  if (r->history) {
    if (!a->r.history_stride) a->r.history_stride = r->history_columns;
    if (a->r.history_stride < r->history_columns) return arg("history_stride is smaller than history_columns");
    if (r->history_columns > 0x7FFFFFFFu) return fail(SKY_ERR_LIMIT, std::string(who) + ": more than 2^31 - 1 ids in a history");
    if (!r->history_columns) a->r.history = nullptr;
  } else if (r->history_columns || r->history_lengths || r->history_first || r->repetition || r->presence || r->frequency) {
    return arg("penalties without a history");
  }
  if (r->bias_offsets || r->bias_ids || r->bias_values || r->bias_count) {
    if (!r->bias_count) {  // every row's list is empty
      a->r.bias_ids = nullptr;
    } else if (!r->bias_offsets || !r->bias_ids || !r->bias_values) {
      return arg("biases need offsets, ids and values");
    }
  }
  if (r->allowed) {
    const uint64_t words = ((uint64_t)columns + 31) / 32;
    if (!a->r.allowed_stride) a->r.allowed_stride = words;
    if (a->r.allowed_stride < words) return arg("allowed_stride is smaller than a row of bits");
    if (!r->allowed_rows) return arg("allowed without rows");
    if (!r->allowed_row && r->allowed_rows != 1 && r->allowed_rows < rows) return arg("fewer mask rows than rows, and no allowed_row");
  } else if (r->allowed_rows || r->allowed_row) {
    return arg("mask rows without masks");
  }
  if (r->graph) {
    if (!r->states) return arg("a graph needs states");
    if (!a->r.states_stride) a->r.states_stride = 1;
  } else if (r->states) {
    return arg("states without a graph");
  }
  const struct {
    const char* name;
    const void* p;
  } words[] = {{"history", r->history},           {"history_lengths", r->history_lengths}, {"history_first", r->history_first},
               {"repetition", r->repetition},     {"presence", r->presence},               {"frequency", r->frequency},
               {"bias_offsets", r->bias_offsets}, {"bias_ids", r->bias_ids},               {"bias_values", r->bias_values},
               {"allowed", r->allowed},           {"allowed_row", r->allowed_row},         {"states", r->states}};
  for (const auto& w : words) SKY_TRY(check_aligned(who, w.name, w.p, 4));
  return SKY_OK;
}

}  // namespace
}  // namespace sky

using namespace sky;

extern "C" int sky_logits_adjust(const void* logits, int dtype, uint32_t rows, uint32_t columns, uint64_t row_stride,
                                 const sky_logits_rules* rules, void* out, uint64_t out_stride, void* stream) {
  AdjustArgs a;
  SKY_TRY(check_rows("sky_logits_adjust", "logits", logits, dtype, rows, columns, &row_stride));
  SKY_TRY(check_rows("sky_logits_adjust", "out", out, dtype, rows, columns, &out_stride));
  if (out == logits && out_stride != row_stride) return fail(SKY_ERR_ARG, "sky_logits_adjust: in place with another stride");
  SKY_TRY(check_rules(rules, rows, columns, &a));
  if (columns > MAX_COLUMNS) return fail(SKY_ERR_LIMIT, "sky_logits_adjust: more than 2^30 columns");
  if (!rows || !columns) return SKY_OK;
  const size_t size = dtype_size(dtype);
  const bool aligned = ((uintptr_t)out | out_stride * size) % 16 == 0, near = a.r.graph != nullptr;
  // counts and biases take 8 bytes of LDS a column: half the tile keeps several workgroups on a CU
  const uint32_t most = near || (a.r.history && a.r.bias_ids) ? 256 : 512;
  uint32_t threads = near ? NEAR_THREADS : 64;
  while (threads < most && threads * COLS < columns) threads *= 2;
  const uint32_t tile = threads * COLS;
  a.tiles = (uint32_t)(((uint64_t)columns + (aligned ? 0 : 16 / size - 1) + tile - 1) / tile);
  const uint64_t grid = near ? rows : (uint64_t)a.tiles * rows;
  if (grid * threads > 0xFFFFFFFFull) return fail(SKY_ERR_LIMIT, "sky_logits_adjust: more than 2^32 - 1 threads, one for 16 columns or 256 for a row by a graph");
  SKY_TRY(ensure_device());
  if (near) {
    int dev = 0;
    SKY_HIP(hipGetDevice(&dev));
    if (dev != a.r.graph->device)
      return fail(SKY_ERR_STATE, "sky_logits_adjust: the graph lives on device " + std::to_string(a.r.graph->device) +
                                     ", the current device is " + std::to_string(dev));
    a.xadj = a.r.graph->xadj;
    a.adjncy = a.r.graph->adjncy;
    a.V = a.r.graph->V;
  }
  a.logits = logits;
  a.out = out;
  a.stride = row_stride;
  a.out_stride = out_stride;
  a.columns = columns;
  const uint32_t arrays = (a.r.history ? tile : 0u) + (a.r.bias_ids ? tile : 0u);
  const uint32_t lds = !near ? arrays : std::max(a.r.history || a.r.bias_ids ? 3 * SLOTS : 0u, arrays + tile / 32);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(threads), lds * 4, (hipStream_t)stream, a); };
  if (dtype == SKY_F32)
    near ? launch(adjust_near_kernel<float>) : launch(adjust_kernel<float>);
  else if (dtype == SKY_F16)
    near ? launch(adjust_near_kernel<_Float16>) : launch(adjust_kernel<_Float16>);
  else
    near ? launch(adjust_near_kernel<__bf16>) : launch(adjust_kernel<__bf16>);
  return check_launch();
}
