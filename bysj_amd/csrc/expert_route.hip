// Routing to experts: scores of a token's experts, the k best of them, their
// weights, the gradient of the logits, and the CSR of the experts' slots (no
// counterpart in the reference; the CSR is the one its segment operators take).
//
//   s = softmax(l)  or  1 / (1 + exp(-l))
//   ranked by key = s + bias (in 64 bits), or by l itself without bias and groups
//   a group's value: the sum of its two best keys; top_groups groups take part
//   w_j = c s_j / S,  S = sum over the chosen + 1e-20  (S = 1 without normalising)
//
//   ds_j = c / S (dw_j - sum_i dw_i s_i / S)
//        = c / S ((dw_j - d) - sum_i (dw_i - d) s_i / S + 1e-20 d / S)  for any d
//   dl = s (ds - sum_i ds_i s_i)  or  ds s (1 - s)
//
// with d = dw_0, so that the gradient of one expert's weight, which is about 1
// whatever its score, is not the rounding error of a difference.
//
// Equal keys go to the lowest index.  A logit or a bias of -inf takes an expert out.
// NaN ranks behind every other one, as does a group with a NaN among its two best
// behind the others, and shows in the weights of a softmax's row, of a sigmoid
// where it is chosen.
//
// A row is held by L lanes, C logits each.  The k best are taken one by one: the
// largest key of a lane's C, of the row's L lanes (DPP steps inside 16 lanes), the
// lowest index that has it.  Rows of up to 256 logits take at most 16 lanes, so
// that four or more rows share the steps between lanes.  Keys without a bias are
// 32-bit integers in the logits' order; with one they are doubles, so that two
// keys next to each other compare as in any other computation of them.
//
// The CSR is a stable counting sort of tokens * k slots into experts + 1 bins, the
// last for slots without an expert: counts per run of kRunSlots slots, a scan, and
// ranks inside a wave from ballots; a single workgroup up to kSmallSlots slots.
//
// Bound by the k dependent steps of a row (a reduction over its lanes each), not by
// the logits' bytes.  Measured: 24,576 rows of 64 in float32, sigmoid, bias, 4 of 8
// groups, k 6: route 19.4 us, backward 6.3, the CSR of 147,456 slots 16; 65,536 rows
// of 256 in bfloat16, softmax, k 8: route 35 us (1 TB/s), backward 26 (2.7 TB/s), the
// CSR of 524,288 slots 24; 192 rows of 8: route 3.1 us, the CSR 2.8 in one launch.
#include <climits>
#include <type_traits>

#include "elements.h"

namespace dpa4k {
namespace {

constexpr int kMaxExperts = DPA4K_EXPERTS_MAX;
constexpr int kMaxGroups = DPA4K_EXPERT_GROUPS_MAX;
constexpr int kBlock = 256;
constexpr float kTiny = 1.0e-20f;

enum { kSoftmax = 0, kSigmoid = 1 };

struct RouteCall {
  const void* logits;
  const float* bias;
  float* weights;      // forward: out; backward: the gradient's input
  int64_t* experts;
  float* statistics;   // [2][tokens]: the softmax's largest logit and sum
  void* dlogits;
  int64_t tokens;
  int n, k, groups, top_groups, scores, normalize;
  float scale;
};

// ---------------------------------------------------------------------------
// across the lanes of a row
// ---------------------------------------------------------------------------

// The largest over L lanes, in every lane.  Inside 16 lanes by DPP (quad
// permutations, then the mirrored half row and row, which meet the other half).
template <int CTRL, typename U>
__device__ __forceinline__ U dpp(U value) {
  if constexpr (sizeof(U) == 4) {
    return __builtin_bit_cast(U, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, value), CTRL, 0xF, 0xF, false));
  } else {
    const int64_t bits = __builtin_bit_cast(int64_t, value);
    const uint32_t lo = dpp<CTRL>(static_cast<uint32_t>(bits));
    const uint32_t hi = dpp<CTRL>(static_cast<uint32_t>(bits >> 32));
    return __builtin_bit_cast(U, static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo));
  }
}

template <int MASK, typename U>
__device__ __forceinline__ U far_lane(U value) {
  if constexpr (sizeof(U) == 4) {
    return __builtin_bit_cast(U, xor_lane<MASK>(__builtin_bit_cast(int, value)));
  } else {
    return __builtin_bit_cast(U, xor_lane<MASK>(__builtin_bit_cast(double, value)));
  }
}

template <int L, typename U, typename F>
__device__ __forceinline__ U over_row(U value, F&& best) {
  if constexpr (L >= 2) value = best(value, dpp<0xB1>(value));
  if constexpr (L >= 4) value = best(value, dpp<0x4E>(value));
  if constexpr (L >= 8) value = best(value, dpp<0x141>(value));
  if constexpr (L >= 16) value = best(value, dpp<0x140>(value));
  if constexpr (L >= 32) value = best(value, far_lane<16>(value));
  if constexpr (L >= 64) value = best(value, far_lane<32>(value));
  return value;
}

template <typename U>
__device__ __forceinline__ U larger(U a, U b) { return a > b ? a : b; }

// ---------------------------------------------------------------------------
// keys
// ---------------------------------------------------------------------------

// A logit as an integer in its order: 0 for -inf (out), 1 for NaN, equal for both zeros.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.0f);
  const uint32_t key = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
  if (x != x) return 1u;
  return x == -INFINITY ? 0u : key;
}

// The key of an expert with a score in 64 bits; -inf is out.  NaN is behind all others,
// which are above -4e38, and two of them together still in front of -inf.
__device__ __forceinline__ double biased(float logit, double score, double bias) {
  const double key = score + bias;
  if (logit == -INFINITY || bias == -INFINITY) return -INFINITY;
  return key != key ? -1.0e300 : key;
}

template <bool WIDE>
using Key = typename std::conditional<WIDE, double, uint32_t>::type;

template <bool WIDE>
__device__ __forceinline__ Key<WIDE> no_key() {
  if constexpr (WIDE) return -INFINITY;
  else return 0u;
}

// Score of a logit: `top` and `sum` are the row's softmax statistics.
__device__ __forceinline__ float score_of(float logit, int scores, float top, float sum) {
  return scores == kSoftmax ? expf(logit - top) / sum : logistic(logit);
}

template <typename T, int L, int C>
struct RouteRow {
  static constexpr int V = 16 / sizeof(T) < C ? 16 / sizeof(T) : C;
  static constexpr int N = C / V;
  static constexpr int kRows = kBlock / L;
  static __device__ __forceinline__ int index(int c, int lane) { return ((c / V) * L + lane) * V + c % V; }
  static __device__ __forceinline__ void load(const T* __restrict__ p, int64_t row, int lane, int n, int64_t total, bool live,
                                              float (&out)[C]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = (i * L + lane) * V;
      const int64_t from = row * n + at;
      const Pack<T, V> raw = load_pack<T, V>(p + from, live ? n - at : 0, total - from);
#pragma unroll
      for (int j = 0; j < V; ++j) out[i * V + j] = live && at + j < n ? static_cast<float>(raw[j]) : -INFINITY;
    }
  }
};

// The best key of a row and the lowest index that has it, among this lane's `key`s.
template <typename T, int L, int C, typename K>
__device__ __forceinline__ K best_of(const K (&key)[C], int lane, int& at) {
  typedef RouteRow<T, L, C> Z;
  K mine = key[0];
#pragma unroll
  for (int c = 1; c < C; ++c) mine = larger(mine, key[c]);
  const K best = over_row<L>(mine, larger<K>);
  int index = INT_MAX;
#pragma unroll
  for (int c = C - 1; c >= 0; --c) index = key[c] == best ? Z::index(c, lane) : index;
  at = over_row<L>(index, [](int a, int b) { return a < b ? a : b; });
  return best;
}

template <typename T, int L, int C, bool WIDE>
__global__ __launch_bounds__(kBlock) void expert_route_kernel(RouteCall call) {
  typedef RouteRow<T, L, C> Z;
  typedef Key<WIDE> K;
  // the chosen of each row; behind them, with groups, each row's group values
  extern __shared__ char lds[];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int n = call.n, k = call.k;
  const int64_t first = block_index() * Z::kRows;
  if (first >= call.tokens) return;
  const int64_t row = first + group;
  const bool live = row < call.tokens;
  const T* logits = static_cast<const T*>(call.logits);
  int* chosen = reinterpret_cast<int*>(lds) + group * k;

  float logit[C];
  Z::load(logits, row, lane, n, call.tokens * n, live, logit);
  float top = 0.0f, sum = 1.0f;
  if (call.scores == kSoftmax) {
    top = logit[0];
#pragma unroll
    for (int c = 1; c < C; ++c) top = fmaxf(top, logit[c]);
    top = over_row<L>(top, [](float a, float b) { return fmaxf(a, b); });
    top = fmaxf(top, -3.4028234663852886e38f);   // a row without experts
    sum = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) sum += expf(logit[c] - top);
    sum = over_row<L>(sum, [](float a, float b) { return a + b; });
  }
  K key[C];
  if constexpr (WIDE) {
    double score[C], inverse = 1.0;
    if (call.scores == kSoftmax) {
      double wide = 0.0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        // of the largest 1, also of an infinite one; a NaN takes its own key alone
        score[c] = exp(logit[c] == top ? 0.0 : static_cast<double>(logit[c]) - static_cast<double>(top));
        wide += score[c] == score[c] ? score[c] : 0.0;
      }
      inverse = over_row<L>(wide, [](double a, double b) { return a + b; });
#pragma unroll
      for (int c = 0; c < C; ++c) score[c] /= inverse;
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) score[c] = 1.0 / (1.0 + exp(-static_cast<double>(logit[c])));
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = Z::index(c, lane);
      key[c] = biased(logit[c], score[c], call.bias != nullptr && e < n ? static_cast<double>(call.bias[e]) : 0.0);
    }
    if (call.groups > 1) {
      double* values = reinterpret_cast<double*>(lds + ((static_cast<size_t>(Z::kRows) * k * sizeof(int) + 7) & ~size_t(7))) +
                       group * call.groups;
      const int members = n / call.groups;
      for (int g = 0; g < call.groups; ++g) {
        double part[C];
        int at;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const int e = Z::index(c, lane);
          part[c] = e >= g * members && e < (g + 1) * members ? key[c] : -INFINITY;
        }
        const double one = best_of<T, L, C>(part, lane, at);
#pragma unroll
        for (int c = 0; c < C; ++c) part[c] = Z::index(c, lane) == at ? -INFINITY : part[c];
        const double two = best_of<T, L, C>(part, lane, at);
        if (lane == 0) values[g] = one + (two == -INFINITY ? 0.0 : two);
      }
      __syncthreads();
      uint64_t allowed = 0;
      for (int g = lane; g < call.groups; g += L) {
        const double mine = values[g];
        int ahead = 0;
        for (int h = 0; h < call.groups; ++h) ahead += values[h] > mine || (values[h] == mine && h < g);
        if (ahead < call.top_groups) allowed |= uint64_t(1) << g;
      }
      allowed = over_row<L>(allowed, [](uint64_t a, uint64_t b) { return a | b; });
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = Z::index(c, lane);
        if (e < n && !((allowed >> (e / members)) & 1)) key[c] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) key[c] = ordered(logit[c]);
  }

  for (int j = 0; j < k; ++j) {
    int at;
    const K best = best_of<T, L, C>(key, lane, at);
#pragma unroll
    for (int c = 0; c < C; ++c) key[c] = Z::index(c, lane) == at ? no_key<WIDE>() : key[c];
    if (lane == 0) chosen[j] = best == no_key<WIDE>() ? -1 : at;
  }
  __syncthreads();
  if (!live) return;
  float total = 0.0f;
  for (int j = lane; j < k; j += L) {
    const int e = chosen[j];
    if (e >= 0) total += score_of(static_cast<float>(logits[row * n + e]), call.scores, top, sum);
  }
  total = over_row<L>(total, [](float a, float b) { return a + b; });
  const float factor = call.normalize ? call.scale / (total + kTiny) : call.scale;
  for (int j = lane; j < k; j += L) {
    const int e = chosen[j];
    call.weights[row * k + j] = e >= 0 ? factor * score_of(static_cast<float>(logits[row * n + e]), call.scores, top, sum) : 0.0f;
    call.experts[row * k + j] = e;
  }
  if (call.statistics != nullptr && call.scores == kSoftmax && lane == 0) {
    call.statistics[row] = top;
    call.statistics[call.tokens + row] = sum;
  }
}

template <typename T, int L, int C>
__global__ __launch_bounds__(kBlock) void expert_route_backward_kernel(RouteCall call) {
  typedef RouteRow<T, L, C> Z;
  __shared__ float ds[Z::kRows][L * C];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int n = call.n, k = call.k;
  const int64_t first = block_index() * Z::kRows;
  if (first >= call.tokens) return;
  const int64_t row = first + group;
  const bool live = row < call.tokens;
  const T* logits = static_cast<const T*>(call.logits);
  float top = 0.0f, sum = 1.0f;
  if (call.scores == kSoftmax && live) {
    top = call.statistics[row];
    sum = call.statistics[call.tokens + row];
  }
  for (int e = lane; e < L * C; e += L) ds[group][e] = 0.0f;
  __syncthreads();
  // sums over the chosen: of s, of (dw - d) s, then of ds s
  float total = 0.0f, dot = 0.0f;
  const float first_dw = live ? call.weights[row * k] : 0.0f;
  for (int j = lane; live && j < k; j += L) {
    const int64_t e = call.experts[row * k + j];
    if (static_cast<uint64_t>(e) >= static_cast<uint64_t>(n)) continue;
    const float s = score_of(static_cast<float>(logits[row * n + e]), call.scores, top, sum);
    total += s;
    dot = fmaf(call.weights[row * k + j] - first_dw, s, dot);
  }
  total = over_row<L>(total, [](float a, float b) { return a + b; }) + kTiny;
  dot = over_row<L>(dot, [](float a, float b) { return a + b; });
  float inner = 0.0f;
  for (int j = lane; live && j < k; j += L) {
    const int64_t e = call.experts[row * k + j];
    if (static_cast<uint64_t>(e) >= static_cast<uint64_t>(n)) continue;
    const float s = score_of(static_cast<float>(logits[row * n + e]), call.scores, top, sum);
    const float dw = call.weights[row * k + j];
    const float d = call.normalize ? call.scale / total * ((dw - first_dw) - dot / total + kTiny / total * first_dw) : call.scale * dw;
    inner = fmaf(d, s, inner);
    ds[group][e] = d;
  }
  inner = over_row<L>(inner, [](float a, float b) { return a + b; });
  __syncthreads();
  if (!live) return;
  T* out = static_cast<T*>(call.dlogits);
  float logit[C];
  Z::load(logits, row, lane, n, call.tokens * n, live, logit);
#pragma unroll
  for (int i = 0; i < Z::N; ++i) {
    const int at = (i * L + lane) * Z::V;
    float part[Z::V];
#pragma unroll
    for (int j = 0; j < Z::V; ++j) {
      const float d = at + j < n ? ds[group][at + j] : 0.0f;
      const float l = logit[i * Z::V + j];
      if (call.scores == kSoftmax) {
        part[j] = l == -INFINITY ? 0.0f : score_of(l, kSoftmax, top, sum) * (d - inner);
      } else {
        float other;
        const float s = logistic(l, other);
        part[j] = d == 0.0f ? 0.0f : d * s * other;
      }
    }
    if (at < n) store_pack<false, T, Z::V>(out + row * n + at, part, n - at);
  }
}

// Calls `use` with the lanes of a row of n logits and the logits a lane holds.
template <typename F>
int with_row(int n, F&& use) {
  using std::integral_constant;
  if (n <= 8) return use(integral_constant<int, 1>{}, integral_constant<int, 8>{});
  if (n <= 16) return use(integral_constant<int, 2>{}, integral_constant<int, 8>{});
  if (n <= 32) return use(integral_constant<int, 4>{}, integral_constant<int, 8>{});
  if (n <= 64) return use(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  if (n <= 128) return use(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  if (n <= 256) return use(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  if (n <= 512) return use(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  return use(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

int check_route(int64_t tokens, int64_t experts, int64_t k, int64_t groups, int64_t top_groups, int scores, int type) {
  if (tokens < 0 || k < 0) return fail(DPA4K_EINVAL, "expert route: negative sizes");
  if (experts < 1 || experts > kMaxExperts) return fail(DPA4K_EINVAL, "expert route takes 1 to %d experts", kMaxExperts);
  if (groups < 1 || groups > kMaxGroups || experts % groups != 0)
    return fail(DPA4K_EINVAL, "expert route: at most %d groups, which divide the experts", kMaxGroups);
  if (top_groups < 1 || top_groups > groups) return fail(DPA4K_EINVAL, "expert route: top_groups must be 1 to groups");
  if (k < 1 || k > top_groups * (experts / groups)) return fail(DPA4K_EINVAL, "expert route: k must be 1 to the experts of top_groups");
  if (scores != kSoftmax && scores != kSigmoid) return fail(DPA4K_EINVAL, "expert route: unknown scores");
  if (!known_type(type)) return fail(DPA4K_EINVAL, "expert route: unknown type");
  if (tokens > INT32_MAX / k) return fail(DPA4K_EINVAL, "expert route takes fewer than 2^31 slots");
  return DPA4K_OK;
}

// ---------------------------------------------------------------------------
// the CSR of the slots
// ---------------------------------------------------------------------------

constexpr int kRunSlots = 2048;
constexpr int kSmallSlots = 8192;

// The bin of a slot: its expert, or `experts` where it has none.
__device__ __forceinline__ int bin_of(const int64_t* __restrict__ chosen, int64_t slot, int experts) {
  const int64_t e = chosen[slot];
  return static_cast<uint64_t>(e) < static_cast<uint64_t>(experts) ? static_cast<int>(e) : experts;
}

// counts[bin][run]
__global__ __launch_bounds__(256) void dispatch_count_kernel(const int64_t* __restrict__ chosen, int64_t slots, int experts,
                                                             int* __restrict__ counts, int runs) {
  __shared__ int bins[kMaxExperts + 1];
  for (int e = threadIdx.x; e <= experts; e += 256) bins[e] = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRunSlots;
#pragma unroll
  for (int i = 0; i < kRunSlots / 256; ++i) {
    const int64_t slot = first + i * 256 + threadIdx.x;
    if (slot < slots) atomicAdd(&bins[bin_of(chosen, slot, experts)], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += 256) counts[static_cast<int64_t>(e) * runs + blockIdx.x] = bins[e];
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int value) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const int other = __shfl_up(value, step, 64);
    if (lane >= step) value += other;
  }
  return value;
}

// A wave per bin: counts become the sums of the runs before, totals[bin] their sum.
__global__ __launch_bounds__(256) void dispatch_scan_kernel(int* __restrict__ counts, int* __restrict__ totals, int bins, int runs) {
  const int bin = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (bin >= bins) return;
  int* at = counts + static_cast<int64_t>(bin) * runs;
  int sum = 0;
  for (int first = 0; first < runs; first += 64) {
    const int run = first + lane;
    const int mine = run < runs ? at[run] : 0;
    const int scanned = wave_scan(mine);
    if (run < runs) at[run] = sum + scanned - mine;
    sum += __shfl(scanned, 63, 64);
  }
  if (lane == 0) totals[bin] = sum;
}

// Places of the slots.  With counts: this workgroup's run of them; without: all, in
// one workgroup.  LDS: [WAVES][bins] counters, [bins] starts.
template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void dispatch_place_kernel(const int64_t* __restrict__ chosen, int64_t slots, int experts,
                                                                    const int* __restrict__ counts, const int* __restrict__ totals,
                                                                    int runs, int per_wave, int64_t* __restrict__ offsets,
                                                                    int64_t* __restrict__ order, int64_t* __restrict__ places) {
  extern __shared__ int bins_of_waves[];
  const int bins = experts + 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  int* mine = bins_of_waves + wave * bins;
  int* starts = bins_of_waves + WAVES * bins;
  for (int e = threadIdx.x; e < WAVES * bins; e += WAVES * 64) bins_of_waves[e] = 0;
  __syncthreads();
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * WAVES + wave) * per_wave;
  const int64_t last = first + per_wave < slots ? first + per_wave : slots;
  for (int64_t slot = first + lane; slot < last; slot += 64) atomicAdd(&mine[bin_of(chosen, slot, experts)], 1);
  __syncthreads();
  if (totals == nullptr) {
    for (int e = threadIdx.x; e < bins; e += WAVES * 64) {
      int sum = 0;
      for (int w = 0; w < WAVES; ++w) sum += bins_of_waves[w * bins + e];
      starts[e] = sum;
    }
    __syncthreads();
  }
  if (wave == 0) {
    int sum = 0;
    for (int from = 0; from < bins; from += 64) {
      const int e = from + lane;
      const int count = e < bins ? (totals != nullptr ? totals[e] : starts[e]) : 0;
      const int scanned = wave_scan(count);
      if (e < bins) {
        starts[e] = sum + scanned - count;
        if (blockIdx.x == 0) offsets[e] = sum + scanned - count;   // offsets[experts] is where the last bin starts
      }
      sum += __shfl(scanned, 63, 64);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += WAVES * 64) {
    int at = starts[e] + (counts != nullptr ? counts[static_cast<int64_t>(e) * runs + blockIdx.x] : 0);
    for (int w = 0; w < WAVES; ++w) {
      const int count = bins_of_waves[w * bins + e];
      bins_of_waves[w * bins + e] = at;
      at += count;
    }
  }
  __syncthreads();
  const int bits = 32 - __clz(experts);
  volatile int* next = mine;
  for (int64_t from = first; from < last; from += 64) {
    const int64_t slot = from + lane;
    const bool live = slot < last;
    const int bin = live ? bin_of(chosen, slot, experts) : 0;
    uint64_t same = __ballot(live);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((bin >> b) & 1);
      same &= (bin >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((uint64_t(1) << lane) - 1));
    if (live) {
      const int place = next[bin] + rank;
      places[slot] = bin < experts ? place : -1;
      order[place] = bin < experts ? slot : -1;
    }
    __builtin_amdgcn_wave_barrier();
    if (live && rank == 0) next[bin] = next[bin] + __popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
}

int64_t dispatch_runs(int64_t slots) { return (slots + kRunSlots - 1) / kRunSlots; }

}  // namespace
}  // namespace dpa4k

using namespace dpa4k;

extern "C" int dpa4k_expert_route_forward(const void* logits, const float* bias, float* weights, int64_t* experts, float* statistics,
                                          int64_t tokens, int64_t n_experts, int64_t k, int64_t groups, int64_t top_groups,
                                          int scores, int normalize, float scale, int type, dpa4k_stream_t stream) {
  clear_error();
  const int status = check_route(tokens, n_experts, k, groups, top_groups, scores, type);
  if (status != DPA4K_OK) return status;
  if (tokens == 0) return DPA4K_OK;
  if (logits == nullptr || weights == nullptr || experts == nullptr) return fail(DPA4K_EINVAL, "expert route: null pointer");
  RouteCall call{};
  call.logits = logits, call.bias = bias, call.weights = weights, call.experts = experts, call.statistics = statistics;
  call.tokens = tokens, call.n = static_cast<int>(n_experts), call.k = static_cast<int>(k);
  call.groups = static_cast<int>(groups), call.top_groups = static_cast<int>(top_groups);
  call.scores = scores, call.normalize = normalize != 0, call.scale = scale;
  const bool wide = bias != nullptr || groups > 1;
  return with_type(type, DPA4K_EINVAL, [&](auto t) {
    return with_row(call.n, [&](auto l, auto c) {
      typedef typename decltype(t)::type T;
      typedef RouteRow<T, l.value, c.value> Z;
      const size_t lds = ((static_cast<size_t>(Z::kRows) * k * sizeof(int) + 7) & ~size_t(7)) +
                         (groups > 1 ? static_cast<size_t>(Z::kRows) * groups * sizeof(double) : 0);
      const dim3 grid = launch_grid((tokens + Z::kRows - 1) / Z::kRows, kBlock);
      if (wide) expert_route_kernel<T, l.value, c.value, true><<<grid, kBlock, lds, as_stream(stream)>>>(call);
      else expert_route_kernel<T, l.value, c.value, false><<<grid, kBlock, lds, as_stream(stream)>>>(call);
      return launched("expert_route_kernel");
    });
  });
}

extern "C" int dpa4k_expert_route_backward(const float* grad_weights, const void* logits, const int64_t* experts,
                                           const float* statistics, void* grad_logits, int64_t tokens, int64_t n_experts, int64_t k,
                                           int scores, int normalize, float scale, int type, dpa4k_stream_t stream) {
  clear_error();
  const int status = check_route(tokens, n_experts, k, 1, 1, scores, type);
  if (status != DPA4K_OK) return status;
  if (tokens == 0) return DPA4K_OK;
  if (grad_weights == nullptr || logits == nullptr || experts == nullptr || grad_logits == nullptr ||
      (scores == kSoftmax && statistics == nullptr))
    return fail(DPA4K_EINVAL, "expert route: null pointer");
  RouteCall call{};
  call.logits = logits, call.weights = const_cast<float*>(grad_weights), call.experts = const_cast<int64_t*>(experts);
  call.statistics = const_cast<float*>(statistics), call.dlogits = grad_logits;
  call.tokens = tokens, call.n = static_cast<int>(n_experts), call.k = static_cast<int>(k);
  call.scores = scores, call.normalize = normalize != 0, call.scale = scale;
  return with_type(type, DPA4K_EINVAL, [&](auto t) {
    return with_row(call.n, [&](auto l, auto c) {
      typedef typename decltype(t)::type T;
      typedef RouteRow<T, l.value, c.value> Z;
      expert_route_backward_kernel<T, l.value, c.value>
          <<<launch_grid((tokens + Z::kRows - 1) / Z::kRows, kBlock), kBlock, 0, as_stream(stream)>>>(call);
      return launched("expert_route_backward_kernel");
    });
  });
}

extern "C" size_t dpa4k_expert_dispatch_workspace_size(int64_t slots, int64_t n_experts) {
  if (slots < 0 || slots > INT32_MAX || n_experts < 1 || n_experts > kMaxExperts || slots <= kSmallSlots) return 0;
  return round_up_256(static_cast<size_t>(n_experts + 1) * dispatch_runs(slots) * sizeof(int)) +
         round_up_256(static_cast<size_t>(n_experts + 1) * sizeof(int));
}

extern "C" int dpa4k_expert_dispatch(const int64_t* experts, int64_t slots, int64_t n_experts, int64_t* offsets, int64_t* order,
                                     int64_t* places, void* workspace, size_t workspace_bytes, dpa4k_stream_t stream) {
  clear_error();
  if (slots < 0) return fail(DPA4K_EINVAL, "expert dispatch: negative sizes");
  if (slots > INT32_MAX) return fail(DPA4K_EINVAL, "expert dispatch takes fewer than 2^31 slots");
  if (n_experts < 1 || n_experts > kMaxExperts) return fail(DPA4K_EINVAL, "expert dispatch takes 1 to %d experts", kMaxExperts);
  if (offsets == nullptr || (slots > 0 && (experts == nullptr || order == nullptr || places == nullptr)))
    return fail(DPA4K_EINVAL, "expert dispatch: null pointer");
  const int n = static_cast<int>(n_experts);
  const hipStream_t on = as_stream(stream);
  if (slots <= kSmallSlots) {
    // a wave takes whole rounds of 64 slots
    const int per_wave = static_cast<int>((slots + 511) / 512) * 64;
    dispatch_place_kernel<8><<<1, 512, static_cast<size_t>(9) * (n + 1) * sizeof(int), on>>>(
        experts, slots, n, nullptr, nullptr, 1, per_wave, offsets, order, places);
    return launched("dispatch_place_kernel");
  }
  if (workspace == nullptr || workspace_bytes < dpa4k_expert_dispatch_workspace_size(slots, n_experts))
    return fail(DPA4K_EWORKSPACE, "expert dispatch: workspace too small");
  Carver carver{static_cast<char*>(workspace), workspace_bytes};
  const int runs = static_cast<int>(dispatch_runs(slots));
  int* counts = carver.take<int>(static_cast<size_t>(n + 1) * runs);
  int* totals = carver.take<int>(n + 1);
  dispatch_count_kernel<<<runs, 256, 0, on>>>(experts, slots, n, counts, runs);
  int status = launched("dispatch_count_kernel");
  if (status != DPA4K_OK) return status;
  dispatch_scan_kernel<<<blocks_for(n + 1, 4), 256, 0, on>>>(counts, totals, n + 1, runs);
  status = launched("dispatch_scan_kernel");
  if (status != DPA4K_OK) return status;
  dispatch_place_kernel<4><<<runs, 256, static_cast<size_t>(5) * (n + 1) * sizeof(int), on>>>(
      experts, slots, n, counts, totals, runs, kRunSlots / 4, offsets, order, places);
  return launched("dispatch_place_kernel");
}
