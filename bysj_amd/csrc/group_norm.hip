// Group norm over samples of rows, channels last, with an optional SiLU,
// forward and backward (no counterpart in the reference: the norm of a batch of
// frames beside its row-wise RMSNorm):
//
//   a sample owns whole rows of C channels, a group D = C / G neighbouring
//   channels of them; n = rows * D
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps)
//   h = (x - mean) rstd,  z = h scale + bias,  y = z  or  z sigmoid(z)
//   dz = dy act'(z),  dbias = sum dz,  dscale = sum dz h,  u = dz scale
//   dx = rstd (u - mean(u) - h mean(u h))
//
// Bound by its streams.  Two schedules:
//
//  - direct: a workgroup of 64 to 1,024 threads per sample holds the sample in
//    registers between its statistics and its output, one launch and one read
//    (16M float32 elements in samples of 8,000, forward: 23 us, 5.8 TB/s;
//    backward 45 us, 4.5 TB/s).  Somewhat longer samples are read twice by it,
//    and any longer ones, if they come in spite of max_rows, piece by piece.
//  - tiles: samples too long for that (or of unknown length) are cut, whatever
//    their lengths, by tiles of equal rows, a workgroup per tile that walks the
//    pieces of samples in it.  A piece leaves its sums in slot (tile + sample),
//    a number no other piece has, since from piece to piece one of the two
//    grows; a sample's slots are consecutive.  A small launch merges them, a
//    third writes the output, with the tiles in reverse order: what was read
//    last is still in the memory-side cache (one sample of 100 MB: forward 22 +
//    7 + 35 us, backward 34 + 5 + 46 + 4 us).
//
// A sample, or a piece, is read as one run of 16-byte vectors.  Vector q of a
// run holds the channels (q V + j) mod C, so with a stride of a multiple of
// lcm(C, V) elements a thread stays on the same V channels at any width C, and
// no access is scalar but in the ragged last vector of a run.  A thread's
// channels make N parts, each of one group: N = 1 where V divides D (runs then
// have no ragged vector), N = 2 where D >= V (a vector crosses one border of
// groups at most, after its first `split` channels), else N = V.
#include <cmath>
#include <type_traits>

#include "common.h"

namespace dpa4k {
namespace {

constexpr int kTileBlock = 256;
constexpr int kMaxChannels = DPA4K_GROUP_NORM_MAX_CHANNELS;
constexpr int64_t kTileBytes = 16384;   // least bytes of a tile
// Most tiles of between kTileBytes and kMostTileBytes: 4 workgroups to a CU, all of
// them resident but in the 16-bit kernels of more than 128 registers (the apply
// kernel where N = 1, 132, and the sums kernel where N = V, 133), which keep 3.
constexpr int64_t kTiles = 1024;
// Most bytes of a tile, 256 vectors a thread, so that sums in 32 bits stay short:
// with 1,024 tiles on 16 GB grad_bias was off by 3.7e-5 of its value under
// gradients of one size.
constexpr int64_t kMostTileBytes = 1 << 20;
constexpr int kLdsGroups = 1024;        // groups of a direct workgroup, whose statistics are kept in LDS
constexpr int64_t kStreamed = 16;       // times what it holds: the longest sample that a direct workgroup is meant for
constexpr float kLog2e = 1.4426950408889634f;

struct Shape {
  int64_t samples, entries, inner;   // a sample owns entries, an entry `inner` rows
  int channels, groups;
  int64_t tile_rows, tiles;
  int64_t long_rows;                 // samples of more rows than this take tiles (or a launch of their own)
  int64_t streamed_rows;             // the most rows that a direct workgroup is meant for
  const int64_t* offsets;            // null: sample s is entry s
};

// ---------------------------------------------------------------------------
// elements
// ---------------------------------------------------------------------------

template <typename T>
constexpr int kVec = 16 / sizeof(T);

template <typename T>
struct vector_of {
  typedef T type __attribute__((ext_vector_type(kVec<T>), aligned(sizeof(T))));
};
template <typename T>
using Raw = typename vector_of<T>::type;

template <typename T>
struct Values {
  float v[kVec<T>];
};

template <typename T>
__device__ __forceinline__ Values<T> to_values(const Raw<T>& raw) {
  Values<T> out;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) out.v[j] = static_cast<float>(raw[j]);
  return out;
}

template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* __restrict__ p) {
  return *reinterpret_cast<const Raw<T>*>(p);
}

template <typename T>
__device__ __forceinline__ Values<T> load_whole(const T* __restrict__ p) {
  return to_values<T>(load_raw(p));
}

// The first `live` elements, zeros behind them.
template <typename T>
__device__ __forceinline__ Values<T> load_part(const T* __restrict__ p, int live) {
  Values<T> out;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) out.v[j] = j < live ? static_cast<float>(p[j]) : 0.0f;
  return out;
}

template <typename T>
__device__ __forceinline__ void store_whole(T* __restrict__ p, const Values<T>& value) {
  Raw<T> raw;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) raw[j] = static_cast<T>(value.v[j]);
  __builtin_nontemporal_store(raw, reinterpret_cast<Raw<T>*>(p));
}

template <typename T>
__device__ __forceinline__ void store_part(T* __restrict__ p, const Values<T>& value, int live) {
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j)
    if (j < live) p[j] = static_cast<T>(value.v[j]);
}

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// `condition`, which is the same everywhere, as a value of each lane.  The compiler
// (of ROCm 7.2) keeps a branch's uniform condition as a mask of the lanes that are
// active in a loop, and may use that mask again behind the loop, where lanes that
// had left it are active: there the branch went the other way.
__device__ __forceinline__ bool per_lane(bool condition) {
  int value = condition ? 1 : 0;
  asm volatile("" : "+v"(value));
  return value != 0;
}

__device__ __forceinline__ float activated(float z, bool silu) { return silu ? z * sigmoid(z) : z; }

// grad act'(z) at z = h weight + shift.
__device__ __forceinline__ float through_activation(float grad, float h, float weight, float shift, bool silu) {
  if (!silu) return grad;
  const float z = fmaf(h, weight, shift);
  const float gate = sigmoid(z);
  return grad * (gate * fmaf(z, 1.0f - gate, 1.0f));
}

// ---------------------------------------------------------------------------
// which thread holds which channels
// ---------------------------------------------------------------------------
//
// A period is lcm(C, V) elements, or period_vectors = C / gcd(C, V) vectors.
// Where a workgroup holds several periods it takes `copies` of them at once;
// where a period is longer than a workgroup it takes it in `passes`.
struct Columns {
  int period_vectors, copies, passes;
  __host__ __device__ int stride_vectors() const { return period_vectors * copies; }
};

int gcd_of(int a, int b) { return b == 0 ? a : gcd_of(b, a % b); }

template <typename T>
Columns columns_for(int channels, int block) {
  Columns c;
  c.period_vectors = channels / gcd_of(channels, kVec<T>);
  c.copies = c.period_vectors < block ? block / c.period_vectors : 1;
  c.passes = (c.period_vectors + block - 1) / block;
  return c;
}

// A thread's share of one pass: the vectors first, first + stride, ... of a
// run, which hold the channels (channel + j) mod C.
struct Share {
  bool live;
  int first, channel;
};

template <typename T, int BLOCK>
__device__ __forceinline__ Share share_of(const Columns& columns, int pass, int channels) {
  Share s;
  s.first = pass * BLOCK + static_cast<int>(threadIdx.x);
  s.live = s.first < columns.stride_vectors();
  s.channel = static_cast<int>(static_cast<uint32_t>(s.first) * kVec<T> % static_cast<uint32_t>(channels));
  return s;
}

// Whether the ragged vector behind the `whole` ones is this thread's.
__device__ __forceinline__ bool owns(const Share& share, int64_t whole, int stride) {
  return share.live && whole >= share.first && (whole - share.first) % stride == 0;
}

// Scale and bias of a thread's channels, and the groups of its parts.
template <typename T, int N>
struct Channels {
  static constexpr int V = kVec<T>;
  float weight[V], shift[V];
  int group[N], split;
  __device__ __forceinline__ Channels(const Share& share, const float* __restrict__ scale,
                                      const float* __restrict__ bias, int channels, int width) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      int c = share.channel + j;
      while (c >= channels) c -= channels;  // at most V / C times
      if (N == V || j == 0) group[N == V ? j : 0] = c / width;
      weight[j] = scale != nullptr ? scale[c] : 1.0f;
      shift[j] = bias != nullptr ? bias[c] : 0.0f;
    }
    split = V;
    if constexpr (N == 2) {
      const int next = (group[0] + 1) * width;
      split = next - share.channel < V ? next - share.channel : V;
      group[1] = next < channels ? group[0] + 1 : 0;
    }
  }
  __device__ __forceinline__ int part_of(int j) const { return N == 1 ? 0 : (N == 2 ? (j < split ? 0 : 1) : j); }
};

// A value per channel of a thread, one where its channels share a group.
template <typename T, int N>
struct PerGroup {
  float v[N == 1 ? 1 : kVec<T>];
  __device__ __forceinline__ float at(int j) const { return v[N == 1 ? 0 : j]; }
};

template <typename T, int N>
__device__ __forceinline__ PerGroup<T, N> per_group(const float* values, const Channels<T, N>& channels) {
  float of_part[N];
#pragma unroll
  for (int i = 0; i < N; ++i) of_part[i] = values[channels.group[i]];
  PerGroup<T, N> out;
#pragma unroll
  for (int j = 0; j < (N == 1 ? 1 : kVec<T>); ++j)
    out.v[j] = N == 2 ? (j < channels.split ? of_part[0] : of_part[N - 1]) : of_part[N == 1 ? 0 : j];
  return out;
}

// ---------------------------------------------------------------------------
// samples
// ---------------------------------------------------------------------------

__device__ __forceinline__ int64_t clamped_offset(const Shape& s, int64_t sample) {
  if (s.offsets == nullptr) return sample;
  const int64_t o = s.offsets[sample];
  return o < 0 ? 0 : (o > s.entries ? s.entries : o);
}

// The last sample that starts at or before `entry`, -1 where none does: 64
// places of the offsets at a time.  Wave-uniform.
__device__ __forceinline__ int64_t sample_at(const Shape& s, int64_t entry) {
  if (s.offsets == nullptr) return entry < s.samples ? entry : s.samples - 1;
  const int lane = threadIdx.x & 63;
  int64_t base = 0, left = s.samples;
  while (left > 0) {
    const int64_t step = (left + 63) >> 6;
    const int64_t at = lane * step;
    const bool before = at < left && s.offsets[base + at] <= entry;
    const int count = __popcll(__ballot(before));
    if (count == 0) break;
    const int64_t skip = (count - 1) * step + 1;
    left = step - 1 < left - skip ? step - 1 : left - skip;
    base += skip;
  }
  return base - 1;
}

// Calls piece(sample, first row, last row) for every long sample with rows in
// the tile, in order; wave-uniform.  Short samples are passed over 64 at a time.
template <typename Piece>
__device__ __forceinline__ void each_piece(const Shape& s, int64_t tile, Piece piece) {
  const int64_t begin = tile * s.tile_rows;
  const int64_t rows = s.entries * s.inner;
  const int64_t end = begin + s.tile_rows < rows ? begin + s.tile_rows : rows;
  const int lane = threadIdx.x & 63;
  int64_t base = s.samples <= 64 ? 0 : sample_at(s, begin / s.inner);
  if (base < 0) base = 0;
  for (;; base += 64) {
    const int64_t sample = base + lane;
    const bool in = sample < s.samples;
    const int64_t first = in ? clamped_offset(s, sample) * s.inner : end;
    const int64_t last = in ? clamped_offset(s, sample + 1) * s.inner : end;
    const bool stop = first >= end;
    const uint64_t stops = __ballot(stop);
    uint64_t hits = __ballot(!stop && last > begin && last - first > s.long_rows);
    if (stops != 0) hits &= (stops & (~stops + 1)) - 1;
    while (hits != 0) {
      const int b = __builtin_ctzll(hits);
      hits &= hits - 1;
      const int64_t f = uniform_lane_i64(first, b), l = uniform_lane_i64(last, b);
      piece(uniform_i64(base + b), f > begin ? f : begin, l < end ? l : end);
    }
    if (stops != 0) return;
  }
}

// Rows [begin, end) that belong to no sample (before the first offset, behind the last).
template <typename T, int BLOCK>
__device__ __forceinline__ void zero_outside(T* __restrict__ out, const Shape& s, int64_t begin, int64_t end) {
  if (s.offsets == nullptr) return;
  const int64_t first = s.samples > 0 ? clamped_offset(s, 0) * s.inner : end;
  const int64_t last = s.samples > 0 ? clamped_offset(s, s.samples) * s.inner : end;
  const int64_t head = (first < end ? first : end) * s.channels;
  int64_t tail = last > begin ? last : begin;
  if (tail < (first < end ? first : end)) tail = first < end ? first : end;
  for (int64_t i = begin * s.channels + threadIdx.x; i < head; i += BLOCK) out[i] = static_cast<T>(0.0f);
  for (int64_t i = tail * s.channels + threadIdx.x; i < end * s.channels; i += BLOCK) out[i] = static_cast<T>(0.0f);
}

// ---------------------------------------------------------------------------
// a workgroup's terms by group of channels
// ---------------------------------------------------------------------------
//
// The threads put their terms into LDS, N each.  In every row of a period group
// g owns D elements, which lie in the vectors of `per_row` threads at most; with
// N = 2 it is the second part of a thread whose vector it starts inside of, and
// the first of the others.  `lanes` lanes (a power of two) add a group's terms.
struct Units {
  int channels, width, pass_first, held;  // held: threads with a vector in this pass
  int first_row, per_row, terms, lanes;
};

template <int BLOCK, int V, int N>
__device__ __forceinline__ Units units_of(const Columns& columns, int pass, int channels, int groups) {
  Units u;
  u.channels = channels;
  u.width = channels / groups;
  u.pass_first = pass * BLOCK;
  const int span = columns.stride_vectors() - u.pass_first;
  u.held = span < BLOCK ? span : BLOCK;
  u.first_row = u.pass_first * V / channels;
  const int rows = ((u.pass_first + u.held) * V - 1) / channels - u.first_row + 1;
  u.per_row = N == 1 ? u.width / V : (N == 2 ? (u.width + V - 2) / V + 1 : u.width);
  u.terms = u.per_row * rows;
  const int share = BLOCK / groups;  // threads per group, if each has some
  u.lanes = 1;
  while (u.lanes < 64 && u.lanes < u.terms && 2 * u.lanes <= share) u.lanes <<= 1;
  return u;
}

// Calls term(place) for the terms lane, lane + lanes, ... of group g.
template <int V, int N, typename Term>
__device__ __forceinline__ void each_term(const Units& u, int g, int lane, Term term) {
  const int rows = u.lanes / u.per_row, columns = u.lanes - rows * u.per_row;  // one step
  int row = lane / u.per_row;
  int column = lane - row * u.per_row;
  for (int i = lane; i < u.terms; i += u.lanes) {
    const int start = (u.first_row + row) * u.channels + g * u.width;  // the group's first element in the period
    if constexpr (N == V && V != 1) {
      const int e = start + column - u.pass_first * V;
      if (e >= 0 && e < u.held * V) term(e);
    } else {
      const int vector = start / V + column;
      const int thread = vector - u.pass_first;
      if (thread >= 0 && thread < u.held && vector * V < start + u.width)
        term(N == 1 ? thread : thread * 2 + (column == 0 && start % V != 0 ? 1 : 0));
    }
    row += rows;
    column += columns;
    if (column >= u.per_row) {
      column -= u.per_row;
      ++row;
    }
  }
}

template <typename F>
__device__ __forceinline__ F lanes_sum(F value, int lanes) {
  for (int mask = 1; mask < lanes; mask <<= 1) value += __shfl_xor(value, mask);
  return value;
}

// ---------------------------------------------------------------------------
// moments
// ---------------------------------------------------------------------------
//
// A thread merges batches into a running mean and sum of squared deviations.  A
// batch is taken relative to the mean so far (the first one to its first value)
// and then to its own mean, so neither a mean far from 0 nor a long sum costs
// digits, and a constant sample has its exact mean.  The threads' pairs meet in
// LDS and are merged pair by pair per group; slots and what follows in 64 bits.
template <typename T>
constexpr int kBatch = 32 / kVec<T>;  // vectors in flight: 32 elements

// Vectors of a thread's share in [q, whole), at most K; where to load the k-th:
// places past the run repeat its last vector, so that no load sits in a branch.
template <int K>
__device__ __forceinline__ int in_reach(int64_t q, int64_t whole, int stride) {
  int n = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) n += q + static_cast<int64_t>(k) * stride < whole ? 1 : 0;
  return n;
}
__device__ __forceinline__ int64_t place_of(int64_t q, int k, int stride, int64_t whole) {
  const int64_t at = q + static_cast<int64_t>(k) * stride;
  return at < whole ? at : whole - 1;
}

template <typename T, int N>
struct Running {
  static constexpr int V = kVec<T>;
  float count[N], mean[N], squares[N];  // of each part
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int i = 0; i < N; ++i) count[i] = mean[i] = squares[i] = 0.0f;
  }
  // n terms of part i with the mean origin + delta, where `origin` is the mean so
  // far (or near the terms where there is none yet).
  __device__ __forceinline__ void merge(int i, float n, float origin, float delta, float spread) {
    const float total = count[i] + n;
    const float weight = n * __builtin_amdgcn_rcpf(total);
    mean[i] = fmaf(delta, weight, origin);
    squares[i] += fmaf(delta * delta, count[i] * weight, spread);
    count[i] = total;
  }
  // The first `n` of the vectors, n > 0.
  template <int K, bool kAll>
  __device__ __forceinline__ void add(const Raw<T> (&batch)[K], int n, int split) {
    const float vectors = static_cast<float>(kAll ? K : n);
    float origin[N], delta[N], spread[N], terms[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      delta[i] = spread[i] = 0.0f;
      terms[i] = vectors * (N == 1 ? V : (N == 2 ? (i == 0 ? split : V - split) : 1));
      origin[i] = count[i] > 0.0f ? mean[i] : static_cast<float>(batch[0][N == 2 && i == 1 ? V - 1 : (N == V ? i : 0)]);
    }
    const auto part = [&](const float(&of)[N], int j) { return N == 2 ? (j < split ? of[0] : of[N - 1]) : of[N == 1 ? 0 : j]; };
    const auto add_to = [&](float(&to)[N], int j, float value) {
      if constexpr (N == 2) {
        to[0] += j < split ? value : 0.0f;
        to[1] += j < split ? 0.0f : value;
      } else {
        to[N == 1 ? 0 : j] += value;
      }
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float column = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float d = static_cast<float>(batch[k][j]) - part(origin, j);
        column += kAll || k < n ? d : 0.0f;
      }
      add_to(delta, j, column);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) delta[i] *= __builtin_amdgcn_rcpf(N == 2 && i == 1 && split == V ? 1.0f : terms[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float column = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float d = (static_cast<float>(batch[k][j]) - part(origin, j)) - part(delta, j);
        const float kept = kAll || k < n ? d : 0.0f;
        column = fmaf(kept, kept, column);
      }
      add_to(spread, j, column);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (N != 2 || i == 0 || split < V) merge(i, terms[i], origin[i], delta[i], spread[i]);
  }
  // The elements behind the last whole vector, one at a time.
  __device__ __forceinline__ void add_part(const Values<T>& part, int live, int split) {
    const auto one = [&](int i, float value) {
      const float origin = count[i] > 0.0f ? mean[i] : value;
      merge(i, 1.0f, origin, value - origin, 0.0f);
    };
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < live) {
        if constexpr (N == 2) {
          if (j < split) one(0, part.v[j]);
          else one(1, part.v[j]);
        } else {
          one(N == 1 ? 0 : j, part.v[j]);
        }
      }
  }
  // The vectors q, q + stride, ... below `whole`.
  __device__ __forceinline__ void add_vectors(const T* __restrict__ run, int64_t q, int64_t whole, int stride, int split) {
    for (; q < whole; q += static_cast<int64_t>(kBatch<T>) * stride) {
      Raw<T> batch[kBatch<T>];
#pragma unroll
      for (int k = 0; k < kBatch<T>; ++k) batch[k] = load_raw(run + place_of(q, k, stride, whole) * V);
      const int n = in_reach<kBatch<T>>(q, whole, stride);
      if (n == kBatch<T>) add<kBatch<T>, true>(batch, n, split);
      else add<kBatch<T>, false>(batch, n, split);
    }
  }
  __device__ __forceinline__ void add_run(const T* __restrict__ run, int64_t elements, const Share& share, int stride, int split) {
    if (!share.live) return;
    const int64_t whole = elements / V;
    add_vectors(run, share.first, whole, stride, split);
    if constexpr (N != 1) {
      const int part = static_cast<int>(elements - whole * V);
      if (part > 0 && owns(share, whole, stride)) add_part(load_part(run + whole * V, part), part, split);
    }
  }
};

// The first `split` of a thread's channels belong to its first group (N = 2).
template <typename T, int N>
__device__ __forceinline__ int split_of(const Share& share, int width) {
  if (N != 2) return kVec<T>;
  const int left = width - share.channel % width;
  return left < kVec<T> ? left : kVec<T>;
}

template <int BLOCK, int N>
struct MomentsLds {
  float count[BLOCK * N], mean[BLOCK * N], squares[BLOCK * N];
};

// A run far longer than its workgroup is meant for, in pieces: the parts of each
// are merged in 64 bits, in LDS that only their thread uses.  In 32 bits alone a
// long run of values of one size lost digits (all roundings go the same way).
// The caller's threads meet before they use the LDS for something else.
template <int BLOCK, int N>
struct MomentsFold {
  double mean[BLOCK * N], squares[BLOCK * N];
};
template <typename T, int N, int BLOCK>
__device__ __forceinline__ void add_pieces(Running<T, N>& running, MomentsFold<BLOCK, N>& fold, const T* __restrict__ run,
                                           const Share& share, int64_t whole, int64_t piece, int stride, int split) {
  double vectors = 0.0;  // merged so far
  for (int64_t begin = 0;; begin += piece) {
    const int64_t end = begin + piece < whole ? begin + piece : whole, q = share.first + begin;
    running.add_vectors(run, q, end, stride, split);
    const double more = q < end ? static_cast<double>((end - q + stride - 1) / stride) : 0.0;
    const double weight = more > 0.0 ? more / (vectors + more) : 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double& mean = fold.mean[threadIdx.x * N + i];
      double& squares = fold.squares[threadIdx.x * N + i];
      if (begin == 0) mean = running.mean[i], squares = running.squares[i];
      else if (running.count[i] > 0.0f) {
        const double delta = running.mean[i] - mean;
        squares += running.squares[i] + delta * delta * (running.count[i] * (1.0 - weight));
        mean += delta * weight;
      }
    }
    vectors += more;
    if (end == whole) break;
    running = Running<T, N>();
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    constexpr int V = kVec<T>;
    running.count[i] = static_cast<float>(vectors * (N == 1 ? V : (N == 2 ? (i == 0 ? split : V - split) : 1)));
    running.mean[i] = static_cast<float>(fold.mean[threadIdx.x * N + i]);
    running.squares[i] = static_cast<float>(fold.squares[threadIdx.x * N + i]);
  }
}

// Calls emit(group, terms, mean, squares) in one lane for every group.
template <int BLOCK, typename T, int N, typename Emit>
__device__ __forceinline__ void merge_moments(const Running<T, N>& mine, bool live, MomentsLds<BLOCK, N>& lds, const Units& u,
                                              int groups, Emit emit) {
  if (live) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lds.count[threadIdx.x * N + i] = mine.count[i];
      lds.mean[threadIdx.x * N + i] = mine.mean[i];
      lds.squares[threadIdx.x * N + i] = mine.squares[i];
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & (u.lanes - 1);
  const int per_round = BLOCK / u.lanes;
  for (int g = static_cast<int>(threadIdx.x) / u.lanes; g < (groups + per_round - 1) / per_round * per_round; g += per_round) {
    float total = 0.0f, mean = 0.0f, squares = 0.0f;
    const auto join = [&](float n, float other, float spread) {
      if (!(n > 0.0f)) return;
      const float origin = total > 0.0f ? mean : other;
      const float delta = other - origin, sum = total + n;
      const float weight = n * __builtin_amdgcn_rcpf(sum);
      mean = fmaf(delta, weight, origin);
      squares += fmaf(delta * delta, total * weight, spread);
      total = sum;
    };
    if (g < groups) each_term<kVec<T>, N>(u, g, lane, [&](int e) { join(lds.count[e], lds.mean[e], lds.squares[e]); });
    for (int mask = 1; mask < u.lanes; mask <<= 1) {
      const float n = __shfl_xor(total, mask), other = __shfl_xor(mean, mask), spread = __shfl_xor(squares, mask);
      join(n, other, spread);
    }
    if (lane == 0 && g < groups) emit(g, total, mean, squares);
  }
}

struct Slot {
  float count, mean, squares;
};

// What two passes over a piece leave of a group.
__device__ __forceinline__ Slot joined(const Slot& a, const Slot& b) {
  if (!(b.count > 0.0f)) return a;
  if (!(a.count > 0.0f)) return b;
  const float total = a.count + b.count, delta = b.mean - a.mean;
  const float weight = b.count * __builtin_amdgcn_rcpf(total);
  return {total, fmaf(delta, weight, a.mean), a.squares + fmaf(delta * delta, a.count * weight, b.squares)};
}

__device__ __forceinline__ float inverse_root(double squares, double count, float eps) {
  return static_cast<float>(1.0 / sqrt(squares / count + static_cast<double>(eps)));
}

// Merges `n` slots, `stride` apart, over `lanes` lanes: (count, mean, squares)
// in every lane.  One sweep: deviations from the first slot's mean, in 64 bits.
struct Merged {
  double count, mean, squares;
};
__device__ __forceinline__ Merged merge_slots(const Slot* __restrict__ slots, int64_t n, int64_t stride, int lane, int lanes) {
  constexpr int U = 8;  // loads in flight
  const double pivot = n > 0 ? slots[0].mean : 0.0;
  double total = 0.0, sum = 0.0, spread = 0.0;
  for (int64_t i = lane; i < n; i += U * lanes) {
    Slot s[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t at = i + k * lanes;
      s[k] = slots[(at < n ? at : i) * stride];
      if (at >= n) s[k].count = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (!(s[k].count > 0.0f)) continue;
      const double delta = s[k].mean - pivot, weighed = s[k].count * delta;
      total += s[k].count;
      sum += weighed;
      spread += fma(weighed, delta, static_cast<double>(s[k].squares));
    }
  }
  total = lanes_sum(total, lanes);
  sum = lanes_sum(sum, lanes);
  spread = lanes_sum(spread, lanes);
  const double centre = total > 0.0 ? sum / total : 0.0;
  const double squares = fma(-sum, centre, spread);
  return {total, pivot + centre, squares < 0.0 ? 0.0 : squares};
}

// ---------------------------------------------------------------------------
// loops over a thread's vectors of a run
// ---------------------------------------------------------------------------

// out = value(x) for the vectors q, q + stride, ... below `whole`, K loads in flight.
template <typename T, int K, typename Value>
__device__ __forceinline__ void map_run(const T* __restrict__ run, T* __restrict__ out, int64_t q, int64_t whole, int stride,
                                        Value value) {
  constexpr int V = kVec<T>;
  for (; q + static_cast<int64_t>(K - 1) * stride < whole; q += static_cast<int64_t>(K) * stride) {
    Raw<T> raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k] = load_raw(run + (q + static_cast<int64_t>(k) * stride) * V);
#pragma unroll
    for (int k = 0; k < K; ++k) store_whole(out + (q + static_cast<int64_t>(k) * stride) * V, value(to_values<T>(raw[k])));
  }
  if (q < whole) {
    Raw<T> raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k] = load_raw(run + place_of(q, k, stride, whole) * V);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (q + static_cast<int64_t>(k) * stride < whole)
        store_whole(out + (q + static_cast<int64_t>(k) * stride) * V, value(to_values<T>(raw[k])));
  }
}

// visit(place, a, b) for the same vectors of two runs.
template <typename T, int K, typename Visit>
__device__ __forceinline__ void each_pair(const T* __restrict__ run_a, const T* __restrict__ run_b, int64_t q, int64_t whole,
                                          int stride, Visit visit) {
  constexpr int V = kVec<T>;
  for (; q < whole; q += static_cast<int64_t>(K) * stride) {
    Raw<T> a[K], b[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t at = place_of(q, k, stride, whole) * V;
      a[k] = load_raw(run_a + at);
      b[k] = load_raw(run_b + at);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (q + static_cast<int64_t>(k) * stride < whole)
        visit((q + static_cast<int64_t>(k) * stride) * V, to_values<T>(a[k]), to_values<T>(b[k]));
  }
}

// ---------------------------------------------------------------------------
// tiles, forward
// ---------------------------------------------------------------------------

template <typename T, int N>
__global__ __launch_bounds__(kTileBlock) void group_norm_moments_kernel(const T* __restrict__ x, Shape s, Columns columns,
                                                                        Slot* __restrict__ slots) {
  __shared__ MomentsLds<kTileBlock, N> lds;
  const int64_t tile = block_index();
  if (tile >= s.tiles) return;
  each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
    Slot* out = slots + (tile + sample) * s.groups;
    for (int pass = 0; pass < columns.passes; ++pass) {
      const Share share = share_of<T, kTileBlock>(columns, pass, s.channels);
      const Units u = units_of<kTileBlock, kVec<T>, N>(columns, pass, s.channels, s.groups);
      Running<T, N> running;
      running.add_run(x + a * s.channels, (b - a) * s.channels, share, columns.stride_vectors(),
                      split_of<T, N>(share, s.channels / s.groups));
      merge_moments<kTileBlock>(running, share.live, lds, u, s.groups, [&](int g, float count, float mean, float squares) {
        const Slot own = {count, mean, squares};
        out[g] = pass == 0 ? own : joined(out[g], own);
      });
      __syncthreads();
    }
  });
}

// The slots of a sample's rows [first, last): where they start and how many.
__device__ __forceinline__ int64_t slots_of(const Shape& s, int64_t sample, int64_t first, int64_t last, int64_t& start) {
  const int64_t tile = first / s.tile_rows;
  start = tile + sample;
  return (last - 1) / s.tile_rows - tile + 1;
}

// A wave per (sample, group) of the long samples.
__global__ __launch_bounds__(256) void group_norm_finish_kernel(const Slot* __restrict__ slots, Shape s, float eps,
                                                                float* __restrict__ mean, float* __restrict__ rstd) {
  const int64_t unit = uniform_i64(block_index() * 4 + (threadIdx.x >> 6));
  if (unit >= s.samples * s.groups) return;
  const int64_t sample = unit / s.groups;
  const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
  const int lane = threadIdx.x & 63;
  if (last - first <= s.long_rows) return;
  int64_t start;
  const int64_t n = slots_of(s, sample, first, last, start);
  const Merged m = merge_slots(slots + start * s.groups + unit % s.groups, n, s.groups, lane, 64);
  if (lane != 0) return;
  mean[unit] = static_cast<float>(m.mean);
  rstd[unit] = inverse_root(m.squares, m.count, eps);
}

// Merging a sample's slots again in every tile instead of in a launch of its
// own was slower: 1,024 tiles on one sample of 100 MB took 60 us against 35 + 5.
template <typename T, int N>
__global__ __launch_bounds__(kTileBlock) void group_norm_apply_kernel(
    const T* __restrict__ x, const float* __restrict__ scale, const float* __restrict__ bias, bool silu,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ y, Shape s, Columns columns) {
  constexpr int V = kVec<T>, K = 4;
  const int64_t block = block_index();
  if (block >= s.tiles) return;
  const int64_t tile = s.tiles - 1 - block;
  const int C = s.channels, G = s.groups;
  const int stride = columns.stride_vectors();
  for (int pass = 0; pass < columns.passes; ++pass) {
    const Share share = share_of<T, kTileBlock>(columns, pass, C);
    const Channels<T, N> channels(share, scale, bias, C, C / G);
    each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
      if (!share.live) return;
      const int64_t elements = (b - a) * C;
      const int64_t whole = elements / V;
      const T* run = x + a * C;
      T* out = y + a * C;
      const PerGroup<T, N> centre = per_group<T, N>(mean + sample * G, channels);
      const PerGroup<T, N> inverse = per_group<T, N>(rstd + sample * G, channels);
      float slope[V];
#pragma unroll
      for (int j = 0; j < V; ++j) slope[j] = inverse.at(j) * channels.weight[j];
      const auto normed = [&](Values<T> value) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          value.v[j] = activated(fmaf(value.v[j] - centre.at(j), slope[j], channels.shift[j]), silu);
        return value;
      };
      map_run<T, K>(run, out, share.first, whole, stride, normed);
      if constexpr (N != 1) {
        const int left = static_cast<int>(elements - whole * V);
        if (left > 0 && owns(share, whole, stride))
          store_part(out + whole * V, normed(load_part(run + whole * V, left)), left);
      }
    });
  }
  const int64_t begin = tile * s.tile_rows, rows = s.entries * s.inner;
  zero_outside<T, kTileBlock>(y, s, begin, begin + s.tile_rows < rows ? begin + s.tile_rows : rows);
}

// ---------------------------------------------------------------------------
// direct, forward
// ---------------------------------------------------------------------------
//
// TS threads hold 32 elements each of a sample (1,024 threads with narrow 16-bit
// groups spill 4 registers).  A longer sample (the workgroup is chosen for the
// mean) is streamed twice, and one that is longer than that
// allows for (max_rows was too small) piece by piece.  Blocks behind the samples
// write the zeros of rows without a sample.
template <typename T>
constexpr int kHeld = 32 / kVec<T>;  // vectors

// Vectors of a piece: no more than the longest sample that should come.
template <typename T>
__device__ __forceinline__ int64_t piece_of(int stride) {
  return kStreamed * kHeld<T> * static_cast<int64_t>(stride);
}

// Statistics of one sample for the threads of a workgroup, by group.  A period of
// at most TS vectors has at most TS groups of V channels or more.
template <int TS, int V, int N>
struct Statistics {
  static constexpr int kGroups = N != V ? TS : (TS * V < kLdsGroups ? TS * V : kLdsGroups);
  float mean[kGroups], rstd[kGroups];
};

template <typename T, int N, int TS>
__global__ __launch_bounds__(TS) void group_norm_direct_kernel(
    const T* __restrict__ x, const float* __restrict__ scale, const float* __restrict__ bias, float eps, bool silu,
    float* __restrict__ mean, float* __restrict__ rstd, T* __restrict__ y, Shape s, Columns columns, int64_t zero_blocks) {
  constexpr int V = kVec<T>;
  __shared__ union {
    MomentsLds<TS, N> lds;
    MomentsFold<TS, N> fold;
  } shared;
  __shared__ Statistics<TS, V, N> statistics;
  const int C = s.channels, G = s.groups;
  const int64_t sample = block_index();
  if (sample >= s.samples) {
    const int64_t part = sample - s.samples, rows = s.entries * s.inner;
    if (part >= zero_blocks) return;
    const int64_t each = (rows + zero_blocks - 1) / zero_blocks;
    const int64_t begin = part * each < rows ? part * each : rows;
    zero_outside<T, TS>(y, s, begin, begin + each < rows ? begin + each : rows);
    return;
  }
  const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
  if (first >= last || last - first > s.long_rows) return;
  const int64_t elements = (last - first) * C;
  const int64_t whole = elements / V;
  const int left = N == 1 ? 0 : static_cast<int>(elements - whole * V);
  const T* run = x + first * C;
  T* out = y + first * C;
  const Share share = share_of<T, TS>(columns, 0, C);
  const int stride = columns.stride_vectors();
  const auto normalise = [&](auto is_long) {
    constexpr bool kLong = decltype(is_long)::value;
    const bool active = kLong ? per_lane(silu) : silu;
    const bool held = !kLong && whole <= static_cast<int64_t>(stride) * kHeld<T>;
    const bool tail = N != 1 && left > 0 && owns(share, whole, stride);
    Running<T, N> running;
    Raw<T> raw[kHeld<T>];
    int mine = 0;  // held vectors of this thread
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k)
        if (static_cast<int64_t>(k) * stride < whole) {  // uniform: no thread has a vector k otherwise
          const int64_t q = share.first + static_cast<int64_t>(k) * stride;
          raw[k] = load_raw(run + (q < whole ? q : whole - 1) * V);
          mine += share.live && q < whole ? 1 : 0;
        }
    }
    if constexpr (kLong) {
      if (share.live) add_pieces(running, shared.fold, run, share, whole, piece_of<T>(stride), stride, split_of<T, N>(share, C / G));
      __syncthreads();
    }
    const Channels<T, N> channels(share, scale, bias, C, C / G);
    if (held) {
      if (mine > 0) running.template add<kHeld<T>, false>(raw, mine, channels.split);
    } else if (!kLong && share.live) {
      running.add_vectors(run, share.first, whole, stride, channels.split);
    }
    if (tail) running.add_part(load_part(run + whole * V, left), left, channels.split);
    const Units u = units_of<TS, V, N>(columns, 0, C, G);
    merge_moments<TS>(running, share.live, shared.lds, u, G, [&](int g, float count, float centre, float squares) {
      statistics.mean[g] = centre;
      statistics.rstd[g] = 1.0f / sqrtf(squares / count + eps);
      mean[sample * G + g] = statistics.mean[g];
      rstd[sample * G + g] = statistics.rstd[g];
    });
    __syncthreads();
    if (!share.live) return;
    const PerGroup<T, N> centre = per_group<T, N>(statistics.mean, channels);
    const PerGroup<T, N> inverse = per_group<T, N>(statistics.rstd, channels);
    float slope[V];
#pragma unroll
    for (int j = 0; j < V; ++j) slope[j] = inverse.at(j) * channels.weight[j];
    const auto normed = [&](Values<T> value) {
#pragma unroll
      for (int j = 0; j < V; ++j) value.v[j] = activated(fmaf(value.v[j] - centre.at(j), slope[j], channels.shift[j]), active);
      return value;
    };
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k)
        if (k < mine) store_whole(out + (share.first + static_cast<int64_t>(k) * stride) * V, normed(to_values<T>(raw[k])));
    } else {
      map_run<T, 4>(run, out, share.first, whole, stride, normed);
    }
    if (tail) store_part(out + whole * V, normed(load_part(run + whole * V, left)), left);
  };
  if (last - first > s.streamed_rows) normalise(std::true_type());
  else normalise(std::false_type());
}

// ---------------------------------------------------------------------------
// backward: sums
// ---------------------------------------------------------------------------

// A thread's sums of dz and dz h per channel.
template <typename T>
struct Sums {
  static constexpr int V = kVec<T>;
  float z[V], zh[V];
  __device__ __forceinline__ Sums() {
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] = zh[j] = 0.0f;
  }
  template <int N>
  __device__ __forceinline__ void add(const Values<T>& grad, const Values<T>& x, const Channels<T, N>& channels,
                                      const PerGroup<T, N>& centre, const PerGroup<T, N>& inverse, bool silu) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float h = (x.v[j] - centre.at(j)) * inverse.at(j);
      const float dz = through_activation(grad.v[j], h, channels.weight[j], channels.shift[j], silu);
      z[j] += dz;
      zh[j] = fmaf(dz, h, zh[j]);
    }
  }
  // The elements behind the last whole vector; the others add nothing.
  template <int N>
  __device__ __forceinline__ void add_part(const Values<T>& grad, const Values<T>& x, int live, const Channels<T, N>& channels,
                                           const PerGroup<T, N>& centre, const PerGroup<T, N>& inverse, bool silu) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < live) {
        const float h = (x.v[j] - centre.at(j)) * inverse.at(j);
        const float dz = through_activation(grad.v[j], h, channels.weight[j], channels.shift[j], silu);
        z[j] += dz;
        zh[j] = fmaf(dz, h, zh[j]);
      }
  }
  __device__ __forceinline__ void add(const Sums& other) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      z[j] += other.z[j];
      zh[j] += other.zh[j];
    }
  }
};

// One term per unit in LDS, for two sums at once.
template <int BLOCK, int V>
struct SumsLds {
  float a[BLOCK * V], b[BLOCK * V];
};

// A thread's sums over the pieces of a long run: see MomentsFold.  Beside SumsLds,
// not in its place: in a union with it the 512-thread kernels reloaded spilled
// registers four times as often (bfloat16).
template <int BLOCK, int V>
struct SumsFold {
  double z[BLOCK * V], zh[BLOCK * V];
  template <typename T>
  __device__ __forceinline__ void add(const Sums<T>& sums, bool first) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      z[threadIdx.x * V + j] = sums.z[j] + (first ? 0.0 : z[threadIdx.x * V + j]);
      zh[threadIdx.x * V + j] = sums.zh[j] + (first ? 0.0 : zh[threadIdx.x * V + j]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void get(Sums<T>& sums) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sums.z[j] = static_cast<float>(z[threadIdx.x * V + j]);
      sums.zh[j] = static_cast<float>(zh[threadIdx.x * V + j]);
    }
  }
};

// Calls emit(group, sum u, sum u h) in one lane for every group.
template <int BLOCK, typename T, int N, typename Emit>
__device__ __forceinline__ void merge_sums(const Sums<T>& mine, const Channels<T, N>& channels, bool live,
                                           SumsLds<BLOCK, kVec<T>>& lds, const Units& u, int groups, Emit emit) {
  constexpr int V = kVec<T>;
  if (live) {
    float sum_u[N], sum_uh[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum_u[i] = sum_uh[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float a = mine.z[j] * channels.weight[j], b = mine.zh[j] * channels.weight[j];
      if constexpr (N == 2) {
        sum_u[0] += j < channels.split ? a : 0.0f;
        sum_uh[0] += j < channels.split ? b : 0.0f;
        sum_u[1] += j < channels.split ? 0.0f : a;
        sum_uh[1] += j < channels.split ? 0.0f : b;
      } else {
        sum_u[N == 1 ? 0 : j] += a;
        sum_uh[N == 1 ? 0 : j] += b;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lds.a[threadIdx.x * N + i] = sum_u[i];
      lds.b[threadIdx.x * N + i] = sum_uh[i];
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & (u.lanes - 1);
  const int per_round = BLOCK / u.lanes;
  for (int g = static_cast<int>(threadIdx.x) / u.lanes; g < (groups + per_round - 1) / per_round * per_round; g += per_round) {
    float sum_u = 0.0f, sum_uh = 0.0f;
    if (g < groups)
      each_term<V, N>(u, g, lane, [&](int e) {
        sum_u += lds.a[e];
        sum_uh += lds.b[e];
      });
    sum_u = lanes_sum(sum_u, u.lanes);
    sum_uh = lanes_sum(sum_uh, u.lanes);
    if (lane == 0 && g < groups) emit(g, sum_u, sum_uh);
  }
}

// A workgroup's sums of dz and dz h per channel, over the threads that share
// it; pass 0 writes `out`, later passes add to it (the same thread each time).
template <int BLOCK, typename T>
__device__ __forceinline__ void write_columns(const Sums<T>& mine, bool live, SumsLds<BLOCK, kVec<T>>& lds,
                                              const Columns& columns, int pass, int channels, float2* __restrict__ out) {
  constexpr int V = kVec<T>;
  if (live)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      lds.a[threadIdx.x * V + j] = mine.z[j];
      lds.b[threadIdx.x * V + j] = mine.zh[j];
    }
  __syncthreads();
  const int origin = pass * BLOCK * V;
  const int span = columns.stride_vectors() * V - origin;
  const int held = span < BLOCK * V ? span : BLOCK * V;
  for (int c = threadIdx.x; c < channels; c += BLOCK) {
    float z = 0.0f, zh = 0.0f;
    int e = c - origin % channels;
    if (e < 0) e += channels;
    for (; e < held; e += channels) {
      z += lds.a[e];
      zh += lds.b[e];
    }
    if (pass == 0) out[c] = {z, zh};
    else out[c] = {out[c].x + z, out[c].y + zh};
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// tiles, backward
// ---------------------------------------------------------------------------

// Per piece: sum u and sum u h of each group.  Per tile: sum dz and sum dz h of
// each channel over all its pieces, kept in registers across them.
template <typename T, int N>
__global__ __launch_bounds__(kTileBlock) void group_norm_sums_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ scale,
    const float* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd, bool silu, Shape s,
    Columns columns, float2* __restrict__ slots, float2* __restrict__ column_sums) {
  constexpr int V = kVec<T>, K = kBatch<T> / 2;
  __shared__ SumsLds<kTileBlock, V> lds;
  const int64_t tile = block_index();
  if (tile >= s.tiles) return;
  const int C = s.channels, G = s.groups;
  for (int pass = 0; pass < columns.passes; ++pass) {
    const Share share = share_of<T, kTileBlock>(columns, pass, C);
    const Units u = units_of<kTileBlock, V, N>(columns, pass, C, G);
    const Channels<T, N> channels(share, scale, bias, C, C / G);
    const int stride = columns.stride_vectors();
    Sums<T> total;
    each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
      const int64_t elements = (b - a) * C;
      const int64_t whole = elements / V;
      const T* run_g = grad + a * C;
      const T* run_x = x + a * C;
      Sums<T> sums;
      if (share.live) {
        const PerGroup<T, N> centre = per_group<T, N>(mean + sample * G, channels);
        const PerGroup<T, N> inverse = per_group<T, N>(rstd + sample * G, channels);
        each_pair<T, K>(run_g, run_x, share.first, whole, stride, [&](int64_t, const Values<T>& gv, const Values<T>& xv) {
          sums.add(gv, xv, channels, centre, inverse, silu);
        });
        if constexpr (N != 1) {
          const int left = static_cast<int>(elements - whole * V);
          if (left > 0 && owns(share, whole, stride))
            sums.add_part(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left), left, channels, centre,
                          inverse, silu);
        }
      }
      float2* out = slots + (tile + sample) * G;
      merge_sums<kTileBlock>(sums, channels, share.live, lds, u, G, [&](int g, float sum_u, float sum_uh) {
        if (pass == 0) out[g] = {sum_u, sum_uh};
        else out[g] = {out[g].x + sum_u, out[g].y + sum_uh};
      });
      total.add(sums);
      __syncthreads();
    });
    if (column_sums != nullptr)
      write_columns<kTileBlock, T>(total, share.live, lds, columns, pass, C, column_sums + tile * C);
  }
}

__device__ __forceinline__ float2 merge_sum_slots(const float2* __restrict__ slots, int64_t n, int64_t stride, int lane,
                                                  int lanes, double count) {
  constexpr int U = 8;  // loads in flight
  double sum_u = 0.0, sum_uh = 0.0;
  for (int64_t i = lane; i < n; i += U * lanes) {
    float2 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t at = i + k * lanes;
      v[k] = slots[(at < n ? at : i) * stride];
      if (at >= n) v[k] = {0.0f, 0.0f};
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      sum_u += v[k].x;
      sum_uh += v[k].y;
    }
  }
  sum_u = lanes_sum(sum_u, lanes);
  sum_uh = lanes_sum(sum_uh, lanes);
  return {static_cast<float>(sum_u / count), static_cast<float>(sum_uh / count)};
}

// A wave per (sample, group): means of u, then of u h, of each sample's groups.
__global__ __launch_bounds__(256) void group_norm_means_kernel(const float2* __restrict__ slots, Shape s,
                                                               float* __restrict__ means) {
  const int64_t unit = uniform_i64(block_index() * 4 + (threadIdx.x >> 6));
  if (unit >= s.samples * s.groups) return;
  const int64_t sample = unit / s.groups;
  const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
  if (last - first <= s.long_rows) return;
  int64_t start;
  const int64_t n = slots_of(s, sample, first, last, start);
  const int lane = threadIdx.x & 63;
  const double count = static_cast<double>(last - first) * (s.channels / s.groups);
  const float2 m = merge_sum_slots(slots + start * s.groups + unit % s.groups, n, s.groups, lane, 64, count);
  if (lane != 0) return;
  means[unit + sample * s.groups] = m.x;
  means[unit + (sample + 1) * s.groups] = m.y;
}

// dbias and dscale: a workgroup per 8 channels, whose 128 threads of each take
// the rows of column sums in turn (8 loads in flight), in 64 bits; a wave's
// rows are added by butterfly, the waves' in order.  64 channels a workgroup
// took 16 us for 2,048 rows of 64 channels.
constexpr int kColumnBlock = 1024;
constexpr int kColumnChannels = 8;

__global__ __launch_bounds__(kColumnBlock) void group_norm_columns_kernel(const float2* __restrict__ column_sums,
                                                                          int64_t rows, int channels,
                                                                          float* __restrict__ grad_scale,
                                                                          float* __restrict__ grad_bias) {
  constexpr int kRows = kColumnBlock / kColumnChannels, kWaves = kColumnBlock / 64, U = 8;
  __shared__ double2 lds[kWaves][kColumnChannels];
  const int of = threadIdx.x % kColumnChannels;
  const int channel = blockIdx.x * kColumnChannels + of;
  double z = 0.0, zh = 0.0;
  if (channel < channels) {
    const float2* at = column_sums + channel;
    int64_t t = threadIdx.x / kColumnChannels;
    for (; t + (U - 1) * kRows < rows; t += U * kRows) {
      float2 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = at[(t + i * kRows) * channels];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        z += v[i].x;
        zh += v[i].y;
      }
    }
    for (; t < rows; t += kRows) {
      z += at[t * channels].x;
      zh += at[t * channels].y;
    }
  }
  z = across_sum<kColumnChannels>(z);
  zh = across_sum<kColumnChannels>(zh);
  if ((threadIdx.x & 63) < kColumnChannels) lds[threadIdx.x >> 6][of] = {z, zh};
  __syncthreads();
  if (threadIdx.x >= kColumnChannels || channel >= channels) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    z += lds[w][of].x;
    zh += lds[w][of].y;
  }
  if (grad_bias != nullptr) grad_bias[channel] = static_cast<float>(z);
  if (grad_scale != nullptr) grad_scale[channel] = static_cast<float>(zh);
}

// grad_x of one vector.
template <typename T, int N>
__device__ __forceinline__ Values<T> gradient_of(const Values<T>& grad, const Values<T>& x, const Channels<T, N>& channels,
                                                 const PerGroup<T, N>& centre, const PerGroup<T, N>& inverse,
                                                 const PerGroup<T, N>& mean_u, const PerGroup<T, N>& mean_uh,
                                                 bool silu) {
  Values<T> out;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) {
    const float h = (x.v[j] - centre.at(j)) * inverse.at(j);
    const float u = through_activation(grad.v[j], h, channels.weight[j], channels.shift[j], silu) * channels.weight[j];
    out.v[j] = inverse.at(j) * ((u - mean_u.at(j)) - h * mean_uh.at(j));
  }
  return out;
}

template <typename T, int N>
__global__ __launch_bounds__(kTileBlock) void group_norm_backward_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ scale,
    const float* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd,
    const float* __restrict__ means, bool silu, T* __restrict__ grad_x, Shape s, Columns columns) {
  constexpr int V = kVec<T>, K = kBatch<T> / 2;
  const int64_t block = block_index();
  if (block >= s.tiles) return;
  const int64_t tile = s.tiles - 1 - block;
  const int C = s.channels, G = s.groups;
  const int stride = columns.stride_vectors();
  for (int pass = 0; pass < columns.passes; ++pass) {
    const Share share = share_of<T, kTileBlock>(columns, pass, C);
    const Channels<T, N> channels(share, scale, bias, C, C / G);
    each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
      if (!share.live) return;
      const int64_t elements = (b - a) * C;
      const int64_t whole = elements / V;
      const T* run_g = grad + a * C;
      const T* run_x = x + a * C;
      T* out = grad_x + a * C;
      const PerGroup<T, N> centre = per_group<T, N>(mean + sample * G, channels);
      const PerGroup<T, N> inverse = per_group<T, N>(rstd + sample * G, channels);
      const PerGroup<T, N> mean_u = per_group<T, N>(means + sample * 2 * G, channels);
      const PerGroup<T, N> mean_uh = per_group<T, N>(means + (sample * 2 + 1) * G, channels);
      const auto gradient = [&](const Values<T>& gv, const Values<T>& xv) {
        return gradient_of<T, N>(gv, xv, channels, centre, inverse, mean_u, mean_uh, silu);
      };
      each_pair<T, K>(run_g, run_x, share.first, whole, stride, [&](int64_t at, const Values<T>& gv, const Values<T>& xv) {
        store_whole(out + at, gradient(gv, xv));
      });
      if constexpr (N != 1) {
        const int left = static_cast<int>(elements - whole * V);
        if (left > 0 && owns(share, whole, stride))
          store_part(out + whole * V, gradient(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left)), left);
      }
    });
  }
  const int64_t begin = tile * s.tile_rows, rows = s.entries * s.inner;
  zero_outside<T, kTileBlock>(grad_x, s, begin, begin + s.tile_rows < rows ? begin + s.tile_rows : rows);
}

// ---------------------------------------------------------------------------
// direct, backward
// ---------------------------------------------------------------------------
//
// TS threads hold 32 elements each of a sample's x and gradient, up to 512
// threads (1,024 would leave 128 registers each, half of them held).  With 16
// elements a thread samples of 60 rows of 64 took 512 threads, of which a CU
// holds two workgroups: 51 us for 3,000 of them (139 MB), 37 us with 32.  512
// threads are held to 128 registers, so that a CU holds two of them (they spill 34
// to 40 registers in float32, 10 to 46 in 16 bits: 16M elements in samples of
// 16,000 took 58 us with one, 50 us with two; 53 and 38 us in bfloat16; with SiLU
// 69 and 37); fewer threads are slower that way (47 and 54 us in samples of 1,024).  A workgroup takes the samples b, b + workgroups, ... and keeps its
// sums per channel across them, one row of column sums in the end.  A longer
// sample is streamed, two vectors of each tensor at once: four would take the
// registers of the third wave of a SIMD from every sample (37 -> 51 us above).
constexpr int kStreamedAtOnce = 2;

// The samples of more than `rows` rows, in pieces: see MomentsFold.  They are left
// for a walk of their own, so that the sums in 64 bits take no registers from the
// others, and what it derives from its arguments it derives again.
template <typename T, int N, int TS>
__device__ __forceinline__ void long_samples(const T* __restrict__ grad, const T* __restrict__ x,
                                             const float* __restrict__ scale, const float* __restrict__ bias,
                                             const float* __restrict__ mean, const float* __restrict__ rstd, bool silu,
                                             T* __restrict__ grad_x, const Shape& s, Columns columns, int64_t workers,
                                             int64_t rows, Sums<T>& total, SumsLds<TS, kVec<T>>& lds,
                                             SumsFold<TS, kVec<T>>& fold, Statistics<TS, kVec<T>, N>& means) {
  constexpr int V = kVec<T>;
  int C = s.channels, G = s.groups;
  asm volatile("" : "+s"(columns.period_vectors), "+s"(columns.copies), "+s"(C), "+s"(G));
  const bool active = per_lane(silu);
  const Share share = share_of<T, TS>(columns, 0, C);
  const Units u = units_of<TS, V, N>(columns, 0, C, G);
  const Channels<T, N> channels(share, scale, bias, C, C / G);
  const int stride = columns.stride_vectors();
  const int64_t piece = piece_of<T>(stride);
  for (int64_t sample = blockIdx.x; sample < s.samples; sample += workers) {
    const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
    if (first >= last || last - first <= rows) continue;
    const int64_t elements = (last - first) * C;
    const int64_t whole = elements / V;
    const int left = N == 1 ? 0 : static_cast<int>(elements - whole * V);
    const T* run_g = grad + first * C;
    const T* run_x = x + first * C;
    const bool tail = N != 1 && left > 0 && owns(share, whole, stride);
    const PerGroup<T, N> centre = per_group<T, N>(mean + sample * G, channels);
    const PerGroup<T, N> inverse = per_group<T, N>(rstd + sample * G, channels);
    Sums<T> sums;
    if (share.live) {
      for (int64_t begin = 0; begin < whole; begin += piece) {
        sums = Sums<T>();
        each_pair<T, 1>(run_g, run_x, share.first + begin, begin + piece < whole ? begin + piece : whole, stride,
                        [&](int64_t, const Values<T>& g, const Values<T>& v) {
                          sums.add(g, v, channels, centre, inverse, active);
                        });
        fold.add(sums, begin == 0);
      }
      fold.get(sums);
    }
    if (tail)
      sums.add_part(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left), left, channels, centre, inverse, active);
    total.add(sums);
    if (grad_x == nullptr) continue;
    const float share_of_one = 1.0f / (static_cast<float>(last - first) * static_cast<float>(C / G));
    merge_sums<TS>(sums, channels, share.live, lds, u, G, [&](int g, float sum_u, float sum_uh) {
      means.mean[g] = sum_u * share_of_one;
      means.rstd[g] = sum_uh * share_of_one;
    });
    __syncthreads();
    if (!share.live) continue;
    T* out = grad_x + first * C;
    const PerGroup<T, N> mean_u = per_group<T, N>(means.mean, channels);
    const PerGroup<T, N> mean_uh = per_group<T, N>(means.rstd, channels);
    const auto gradient = [&](const Values<T>& g, const Values<T>& v) {
      return gradient_of<T, N>(g, v, channels, centre, inverse, mean_u, mean_uh, active);
    };
    each_pair<T, 1>(run_g, run_x, share.first, whole, stride,
                    [&](int64_t at, const Values<T>& g, const Values<T>& v) { store_whole(out + at, gradient(g, v)); });
    if (tail) store_part(out + whole * V, gradient(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left)), left);
  }
}

template <typename T, int N, int TS>
__global__ __launch_bounds__(TS, TS == 512 ? 4 : (N == kVec<T> ? 2 : 3)) void group_norm_direct_backward_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ scale,
    const float* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd, bool silu,
    T* __restrict__ grad_x, Shape s, Columns columns, float2* __restrict__ column_sums, int64_t workers) {
  constexpr int V = kVec<T>;
  __shared__ SumsLds<TS, V> lds;
  __shared__ Statistics<TS, V, N> means;
  const int C = s.channels, G = s.groups;
  const int64_t worker = blockIdx.x;
  if (worker >= workers) {
    const int64_t part = worker - workers, parts = gridDim.x - workers, rows = s.entries * s.inner;
    const int64_t each = (rows + parts - 1) / parts;
    const int64_t begin = part * each < rows ? part * each : rows;
    zero_outside<T, TS>(grad_x, s, begin, begin + each < rows ? begin + each : rows);
    return;
  }
  const Share share = share_of<T, TS>(columns, 0, C);
  const Units u = units_of<TS, V, N>(columns, 0, C, G);
  const Channels<T, N> channels(share, scale, bias, C, C / G);
  const int stride = columns.stride_vectors();
  Sums<T> total;
  bool any_long = false;
  for (int64_t sample = worker; sample < s.samples; sample += workers) {
    const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
    if (first >= last || last - first > s.long_rows) continue;
    if (TS != 512 && last - first > s.streamed_rows) {
      any_long = true;
      continue;
    }
    const int64_t elements = (last - first) * C;
    const int64_t whole = elements / V;
    const int left = N == 1 ? 0 : static_cast<int>(elements - whole * V);
    const T* run_g = grad + first * C;
    const T* run_x = x + first * C;
    const bool held = whole <= static_cast<int64_t>(stride) * kHeld<T>;
    const bool tail = N != 1 && left > 0 && owns(share, whole, stride);
    Raw<T> gv[kHeld<T>], xv[kHeld<T>];
    int mine = 0;
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k)
        if (static_cast<int64_t>(k) * stride < whole) {
          const int64_t q = share.first + static_cast<int64_t>(k) * stride;
          const int64_t at = (q < whole ? q : whole - 1) * V;
          gv[k] = load_raw(run_g + at);
          xv[k] = load_raw(run_x + at);
          mine += share.live && q < whole ? 1 : 0;
        }
    }
    const PerGroup<T, N> centre = per_group<T, N>(mean + sample * G, channels);
    const PerGroup<T, N> inverse = per_group<T, N>(rstd + sample * G, channels);
    Sums<T> sums;
    if (held) {
#pragma unroll
      for (int k = 0; k < kHeld<T>; ++k)
        if (k < mine) sums.add(to_values<T>(gv[k]), to_values<T>(xv[k]), channels, centre, inverse, silu);
    } else if (share.live) {
      each_pair<T, kStreamedAtOnce>(run_g, run_x, share.first, whole, stride,
                                  [&](int64_t, const Values<T>& g, const Values<T>& v) {
                                    sums.add(g, v, channels, centre, inverse, silu);
                                  });
    }
    if constexpr (N != 1)
      if (tail)
        sums.add_part(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left), left, channels, centre, inverse,
                      silu);
    total.add(sums);
    if (grad_x == nullptr) continue;
    const float share_of_one = 1.0f / (static_cast<float>(last - first) * static_cast<float>(C / G));
    merge_sums<TS>(sums, channels, share.live, lds, u, G, [&](int g, float sum_u, float sum_uh) {
      means.mean[g] = sum_u * share_of_one;
      means.rstd[g] = sum_uh * share_of_one;
    });
    __syncthreads();
    if (share.live) {
      T* out = grad_x + first * C;
      const PerGroup<T, N> mean_u = per_group<T, N>(means.mean, channels);
      const PerGroup<T, N> mean_uh = per_group<T, N>(means.rstd, channels);
      const auto gradient = [&](const Values<T>& g, const Values<T>& v) {
        return gradient_of<T, N>(g, v, channels, centre, inverse, mean_u, mean_uh, silu);
      };
      if (held) {
#pragma unroll
        for (int k = 0; k < kHeld<T>; ++k)
          if (k < mine)
            store_whole(out + (share.first + static_cast<int64_t>(k) * stride) * V,
                        gradient(to_values<T>(gv[k]), to_values<T>(xv[k])));
      } else {
        each_pair<T, kStreamedAtOnce>(run_g, run_x, share.first, whole, stride,
                                    [&](int64_t at, const Values<T>& g, const Values<T>& v) { store_whole(out + at, gradient(g, v)); });
      }
      if (tail)
        store_part(out + whole * V, gradient(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left)), left);
    }
    // the next sample's terms go to LDS behind this sample's sync: its means have been written from them by then
  }
  if constexpr (TS != 512) {
    __shared__ SumsFold<TS, V> fold;
    if (any_long)
      long_samples<T, N, TS>(grad, x, scale, bias, mean, rstd, silu, grad_x, s, columns, workers, s.streamed_rows, total, lds,
                             fold, means);
  }
  if (column_sums == nullptr) return;
  __syncthreads();
  write_columns<TS, T>(total, share.live, lds, columns, 0, C, column_sums + worker * C);
}

// The long walk of workgroups of 512 threads, which are short of registers: with
// both walks in one kernel 16M elements in samples of 16,000 took 88 us, with the
// first alone 69.
template <typename T, int N>
__global__ __launch_bounds__(512, 2) void group_norm_long_backward_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ scale,
    const float* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd, bool silu,
    T* __restrict__ grad_x, Shape s, Columns columns, float2* __restrict__ column_sums, int64_t workers) {
  constexpr int V = kVec<T>;
  __shared__ SumsLds<512, V> lds;
  __shared__ SumsFold<512, V> fold;
  __shared__ Statistics<512, V, N> means;
  Sums<T> total;
  long_samples<T, N, 512>(grad, x, scale, bias, mean, rstd, silu, grad_x, s, columns, workers, s.long_rows, total, lds, fold, means);
  if (column_sums == nullptr) return;
  __syncthreads();
  write_columns<512, T>(total, share_of<T, 512>(columns, 0, s.channels).live, lds, columns, 0, s.channels,
                        column_sums + blockIdx.x * static_cast<int64_t>(s.channels));
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int64_t type_bytes(int type) { return type == DPA4K_TYPE_F32 ? 4 : 2; }

// How a call is scheduled, from its sizes alone.
struct Schedule {
  Shape shape;
  int threads;            // of a direct workgroup; 0: tiles alone
  bool tiles;             // whether samples may be longer than a direct workgroup holds
  int64_t workers;        // direct workgroups of the backward
  int64_t zero_blocks;    // direct workgroups for rows without a sample
  bool long_launch;       // whether samples of more than long_rows rows take a direct launch of their own, in the backward
  int64_t column_rows;    // rows of column sums
};

constexpr int kDirectThreads[] = {64, 256, 512, 1024};
// Backward workgroups of a direct launch: as many as are resident on 256 CUs at
// three waves a SIMD, and two of 512 threads to a CU (3,000 samples of 60 rows of
// 64: 39 us with 768 workgroups of 256 threads, 41 with 2,048, 47 with 1,024,
// whose last third finds the CUs full).
constexpr int64_t workers_for(int threads) { return 256 * (threads > 256 ? 2 : 12 / (threads / 64)); }

// No workgroup keeps its sums per channel, in 32 bits, over more samples than this:
// 61M samples of one row, 19,900 to a workgroup, left them off by 1.7e-4 of their
// value under gradients of one size.  More samples take more rounds of as many
// workgroups as are resident (a million of 8 rows of 16: 0.9 ms with 3,072 or 6,144
// workgroups, 1.34 with 3,907, whose second round leaves most CUs idle).
constexpr int64_t kWorkerSamples = 256;

// Checks the sizes, cuts the rows into tiles, and chooses the schedule.  A
// direct workgroup holds 32 elements a thread.  Samples of one length take the
// smallest that holds one.  Ragged samples take the smallest that holds the
// longest where all of them are resident at once, and else one that holds a
// quarter more than the mean: a larger one would idle on most samples (4,096
// samples cut anywhere in 200,000 rows of 64 floats, forward: 99 us with room for
// the longest, 393 rows, 30 with room for 61; 50,000 samples: 176 and 56 us).  A
// sample that is longer is streamed, up to kStreamed times what is held (samples
// of 49 rows of 90 in the mean: 65 us up to 4 times, 43 up to 16).  Longer ones
// take tiles, and all do where no workgroup holds the mean, or in the backward
// one of 512 threads, two to a CU, would (1,000 samples: 86 us, tiles 70).
constexpr int64_t kResidentThreads = 262144;  // 16 waves on each CU

int schedule_of(const char* what, int64_t samples, int64_t entries, int64_t inner, int64_t channels, int64_t groups,
                int type, const int64_t* offsets, int64_t max_entries, bool backward, Schedule& out) {
  if (samples < 0 || entries < 0 || inner < 0) return fail(DPA4K_EINVAL, "%s: negative sizes", what);
  if (channels <= 0 || channels > kMaxChannels)
    return fail(DPA4K_EINVAL, "%s: 1 to %d channels, got %lld", what, kMaxChannels, static_cast<long long>(channels));
  if (groups <= 0 || channels % groups != 0) return fail(DPA4K_EINVAL, "%s: groups must divide the channels", what);
  if (type != DPA4K_TYPE_F32 && type != DPA4K_TYPE_BF16 && type != DPA4K_TYPE_F16)
    return fail(DPA4K_EINVAL, "%s: unknown type", what);
  if (offsets == nullptr && samples != entries) return fail(DPA4K_EINVAL, "%s: without offsets every entry is a sample", what);
  const int64_t most = (int64_t(1) << 60) / channels;
  if ((inner > 0 && entries > most / inner) || samples > most)
    return fail(DPA4K_EINVAL, "%s: the element count overflows 64 bits", what);
  const int64_t rows = entries * inner;
  const int64_t row_bytes = channels * type_bytes(type);
  const int64_t least = kTileBytes / row_bytes;
  int64_t tile_rows = (rows + kTiles - 1) / kTiles;
  if (tile_rows > kMostTileBytes / row_bytes) tile_rows = kMostTileBytes / row_bytes;
  if (tile_rows < least) tile_rows = least;
  if (tile_rows < 1) tile_rows = 1;
  out = {};
  out.shape = {samples, entries, inner, static_cast<int>(channels), static_cast<int>(groups), tile_rows,
               (rows + tile_rows - 1) / tile_rows, 0, 0, offsets};
  if (!grid_fits(samples * groups / 4 + 1, 256) || !grid_fits(samples + 4096, 1024))
    return fail(DPA4K_EINVAL, "%s: the sample count exceeds the launch limit", what);
  const int vec = static_cast<int>(16 / type_bytes(type));
  const int period = static_cast<int>(channels) / gcd_of(static_cast<int>(channels), vec);
  // the smallest direct workgroup that holds `sample_rows`, 0 where none does
  const auto holds = [&](int threads) { return static_cast<int64_t>(threads / period) * period * 32 / channels; };
  const auto threads_for = [&](int64_t sample_rows) {
    if (groups <= kLdsGroups)
      for (int threads : kDirectThreads)
        if (period <= threads && !(backward && threads > 512) && sample_rows <= holds(threads)) return threads;
    return 0;
  };
  if (offsets == nullptr) {
    out.threads = threads_for(inner);
    out.shape.long_rows = out.threads != 0 ? INT64_MAX : 0;
    out.tiles = out.threads == 0;
  } else {
    const int64_t longest = max_entries < 0 ? INT64_MAX : (max_entries < entries ? max_entries : entries) * inner;
    const int for_longest = threads_for(longest);
    out.threads = for_longest;
    if (for_longest == 0 || samples * for_longest > kResidentThreads) {
      out.threads = threads_for(samples > 0 ? rows / samples * 5 / 4 + 1 : 1);
      if (backward && out.threads == 512) out.threads = 0;
    }
    const int64_t limit = kStreamed * holds(out.threads);
    out.tiles = out.threads == 0 || longest > limit;
    out.shape.long_rows = out.threads == 0 ? 0 : (out.tiles ? limit : INT64_MAX);  // with no tiles any sample is streamed
  }
  if (out.threads != 0) {
    const int64_t filled = samples < rows ? samples : rows;  // at most: the others are empty
    const int64_t resident = workers_for(out.threads), rounds = (filled + resident * kWorkerSamples - 1) / (resident * kWorkerSamples);
    const int64_t most = 0xFFFFFFFFLL / out.threads / resident - 1;
    out.workers = resident * (rounds < 1 ? 1 : (rounds < most ? rounds : most));
    if (samples < out.workers) out.workers = samples;
  }
  const int64_t kilobytes64 = rows * row_bytes / 65536 + 1;
  out.zero_blocks = offsets == nullptr || out.tiles ? 0 : (kilobytes64 < 256 ? kilobytes64 : 256);
  out.shape.streamed_rows = kStreamed * holds(out.threads);
  if (backward && out.threads == 512 && offsets != nullptr && !out.tiles && rows > out.shape.streamed_rows) {
    out.long_launch = true;
    out.shape.long_rows = out.shape.streamed_rows;
  }
  out.column_rows = out.workers * (out.long_launch ? 2 : 1) + (out.tiles ? out.shape.tiles : 0);
  return DPA4K_OK;
}

struct Workspace {
  Slot* slots;          // per (piece, group), forward
  float2* sum_slots;    // per (piece, group), backward
  float* means;         // per (sample, sum, group), backward
  float2* column_sums;  // rows of channels, backward
};

template <typename Take>
void each_array(const Schedule& c, bool backward, Take take) {
  const size_t pieces = c.tiles ? static_cast<size_t>(c.shape.tiles + c.shape.samples) * c.shape.groups : 0;
  if (!backward) {
    take(&Workspace::slots, pieces);
    return;
  }
  take(&Workspace::sum_slots, pieces);
  take(&Workspace::means, c.tiles ? static_cast<size_t>(c.shape.samples) * 2 * c.shape.groups : 0);
  take(&Workspace::column_sums, static_cast<size_t>(c.column_rows) * c.shape.channels);
}

size_t workspace_bytes_of(const Schedule& c, bool backward) {
  size_t bytes = 0;
  each_array(c, backward, [&](auto member, size_t count) {
    Workspace w{};
    bytes += round_up_256(count * sizeof(*(w.*member)));
  });
  return bytes;
}

bool carve(const Schedule& c, bool backward, void* workspace, size_t bytes, Workspace& w) {
  if (workspace == nullptr) bytes = 0;
  Carver carver{static_cast<char*>(workspace), bytes};
  bool fits = true;
  each_array(c, backward, [&](auto member, size_t count) {
    using Element = std::remove_reference_t<decltype(*(w.*member))>;
    w.*member = count > 0 ? carver.take<Element>(count) : nullptr;
    fits = fits && (count == 0 || w.*member != nullptr);
  });
  return fits;
}

// Calls LAUNCH(TS) for the schedule's direct workgroup.
#define DPA4K_DIRECT(threads, LAUNCH)   \
  if (threads == 64) LAUNCH(64);        \
  else if (threads == 256) LAUNCH(256); \
  else LAUNCH(512);

template <typename T, int N>
int forward_as(const T* x, const float* scale, const float* bias, T* y, float* mean, float* rstd, const Schedule& c,
               float eps, bool silu, const Workspace& w, hipStream_t stream) {
  const Shape& s = c.shape;
  if (c.threads != 0) {
    const Columns columns = columns_for<T>(s.channels, c.threads);
    const dim3 grid = launch_grid(s.samples + c.zero_blocks > 0 ? s.samples + c.zero_blocks : 1, c.threads);
#define DPA4K_LAUNCH(TS)                                                                                              \
  group_norm_direct_kernel<T, N, TS><<<grid, TS, 0, stream>>>(x, scale, bias, eps, silu, mean, rstd, y, s, columns, \
                                                                     c.zero_blocks)
    if (c.threads == 1024) DPA4K_LAUNCH(1024);
    else DPA4K_DIRECT(c.threads, DPA4K_LAUNCH)
#undef DPA4K_LAUNCH
    if (int e = launched("group_norm_direct_kernel")) return e;
  }
  if (!c.tiles) return DPA4K_OK;
  const Columns columns = columns_for<T>(s.channels, kTileBlock);
  const dim3 grid = launch_grid(s.tiles, kTileBlock);
  group_norm_moments_kernel<T, N><<<grid, kTileBlock, 0, stream>>>(x, s, columns, w.slots);
  if (int e = launched("group_norm_moments_kernel")) return e;
  if (s.samples > 0) {
    group_norm_finish_kernel<<<launch_grid((s.samples * s.groups + 3) / 4, 256), 256, 0, stream>>>(w.slots, s, eps, mean, rstd);
    if (int e = launched("group_norm_finish_kernel")) return e;
  }
  group_norm_apply_kernel<T, N><<<grid, kTileBlock, 0, stream>>>(x, scale, bias, silu, mean, rstd, y, s, columns);
  return launched("group_norm_apply_kernel");
}

template <typename T, int N>
int backward_as(const T* grad, const T* x, const float* scale, const float* bias, const float* mean, const float* rstd,
                T* grad_x, float* grad_scale, float* grad_bias, const Schedule& c, bool silu, const Workspace& w,
                hipStream_t stream) {
  const Shape& s = c.shape;
  const bool parameters = grad_scale != nullptr || grad_bias != nullptr;
  float2* tile_columns = parameters ? w.column_sums : nullptr;
  float2* direct_columns = parameters ? w.column_sums + (c.tiles ? s.tiles * s.channels : 0) : nullptr;
  if (c.threads != 0 && (c.workers > 0 || (grad_x != nullptr && c.zero_blocks > 0))) {
    const Columns columns = columns_for<T>(s.channels, c.threads);
    const unsigned int grid = static_cast<unsigned int>(c.workers + (grad_x != nullptr ? c.zero_blocks : 0));
#define DPA4K_LAUNCH(TS)                                                                                                  \
  group_norm_direct_backward_kernel<T, N, TS><<<grid, TS, 0, stream>>>(grad, x, scale, bias, mean, rstd, silu, grad_x, s, \
                                                                              columns, direct_columns, c.workers)
    DPA4K_DIRECT(c.threads, DPA4K_LAUNCH)
#undef DPA4K_LAUNCH
    if (int e = launched("group_norm_direct_backward_kernel")) return e;
    if (c.long_launch && c.workers > 0) {
      group_norm_long_backward_kernel<T, N><<<static_cast<unsigned int>(c.workers), 512, 0, stream>>>(
          grad, x, scale, bias, mean, rstd, silu, grad_x, s, columns,
          parameters ? direct_columns + c.workers * s.channels : nullptr, c.workers);
      if (int e = launched("group_norm_long_backward_kernel")) return e;
    }
  }
  if (c.tiles) {
    const Columns columns = columns_for<T>(s.channels, kTileBlock);
    const dim3 grid = launch_grid(s.tiles, kTileBlock);
    group_norm_sums_kernel<T, N><<<grid, kTileBlock, 0, stream>>>(grad, x, scale, bias, mean, rstd, silu, s, columns,
                                                                        w.sum_slots, tile_columns);
    if (int e = launched("group_norm_sums_kernel")) return e;
    if (grad_x != nullptr) {
      if (s.samples > 0) {
        group_norm_means_kernel<<<launch_grid((s.samples * s.groups + 3) / 4, 256), 256, 0, stream>>>(w.sum_slots, s, w.means);
        if (int e = launched("group_norm_means_kernel")) return e;
      }
      group_norm_backward_kernel<T, N><<<grid, kTileBlock, 0, stream>>>(grad, x, scale, bias, mean, rstd, w.means, silu,
                                                                              grad_x, s, columns);
      if (int e = launched("group_norm_backward_kernel")) return e;
    }
  }
  if (!parameters) return DPA4K_OK;
  group_norm_columns_kernel<<<blocks_for(s.channels, kColumnChannels), kColumnBlock, 0, stream>>>(w.column_sums, c.column_rows, s.channels,
                                                                                    grad_scale, grad_bias);
  return launched("group_norm_columns_kernel");
}

// The parts of a vector: see the top.
template <typename T>
int parts_of(const Shape& s) {
  const int width = s.channels / s.groups;
  return width % kVec<T> == 0 ? 1 : (width >= kVec<T> ? 2 : kVec<T>);
}

template <typename T>
int forward(const void* x, const float* scale, const float* bias, void* y, float* mean, float* rstd, const Schedule& c,
            float eps, bool silu, const Workspace& w, hipStream_t stream) {
  const int parts = parts_of<T>(c.shape);
  return (parts == 1 ? forward_as<T, 1> : (parts == 2 ? forward_as<T, 2> : forward_as<T, kVec<T>>))(
      static_cast<const T*>(x), scale, bias, static_cast<T*>(y), mean, rstd, c, eps, silu, w, stream);
}

template <typename T>
int backward(const void* grad, const void* x, const float* scale, const float* bias, const float* mean,
             const float* rstd, void* grad_x, float* grad_scale, float* grad_bias, const Schedule& c, bool silu,
             const Workspace& w, hipStream_t stream) {
  const int parts = parts_of<T>(c.shape);
  return (parts == 1 ? backward_as<T, 1> : (parts == 2 ? backward_as<T, 2> : backward_as<T, kVec<T>>))(
      static_cast<const T*>(grad), static_cast<const T*>(x), scale, bias, mean, rstd, static_cast<T*>(grad_x), grad_scale,
      grad_bias, c, silu, w, stream);
}

}  // namespace
}  // namespace dpa4k

using namespace dpa4k;

extern "C" size_t dpa4k_group_norm_workspace_size(int64_t samples, int64_t entries, int64_t inner, int64_t channels,
                                                  int64_t groups, int ragged, int64_t max_entries, int type, int backward) {
  Schedule c;
  static const int64_t some = 0;  // any offsets: the size does not depend on them
  if (schedule_of("group norm", samples, entries, inner, channels, groups, type, ragged != 0 ? &some : nullptr, max_entries,
                  backward != 0, c))
    return 0;
  return workspace_bytes_of(c, backward != 0);
}

extern "C" int dpa4k_group_norm_forward(const void* x, const float* scale, const float* bias, const int64_t* offsets,
                                        void* y, float* mean, float* rstd, int64_t samples, int64_t entries,
                                        int64_t inner, int64_t channels, int64_t groups, int64_t max_entries, float eps,
                                        int silu, int type, void* workspace, size_t workspace_bytes,
                                        dpa4k_stream_t stream_handle) {
  clear_error();
  Schedule c;
  if (int e = schedule_of("group norm", samples, entries, inner, channels, groups, type, offsets, max_entries, false, c)) return e;
  if (!(eps > 0.0f) || !(eps < INFINITY)) return fail(DPA4K_EINVAL, "group norm eps must be a finite positive number");
  if (c.shape.tiles == 0) return DPA4K_OK;
  if (x == nullptr || y == nullptr || (samples > 0 && (mean == nullptr || rstd == nullptr)))
    return fail(DPA4K_EINVAL, "group norm: null pointer");
  Workspace w{};
  if (!carve(c, false, workspace, workspace_bytes, w))
    return fail(DPA4K_EWORKSPACE, "group norm: workspace of %zu bytes is smaller than %zu", workspace_bytes,
                workspace_bytes_of(c, false));
  hipStream_t stream = as_stream(stream_handle);
  if (type == DPA4K_TYPE_F32) return forward<float>(x, scale, bias, y, mean, rstd, c, eps, silu != 0, w, stream);
  if (type == DPA4K_TYPE_BF16) return forward<__bf16>(x, scale, bias, y, mean, rstd, c, eps, silu != 0, w, stream);
  return forward<_Float16>(x, scale, bias, y, mean, rstd, c, eps, silu != 0, w, stream);
}

extern "C" int dpa4k_group_norm_backward(const void* grad, const void* x, const float* scale, const float* bias,
                                         const int64_t* offsets, const float* mean, const float* rstd, void* grad_x,
                                         float* grad_scale, float* grad_bias, int64_t samples, int64_t entries,
                                         int64_t inner, int64_t channels, int64_t groups, int64_t max_entries, int silu,
                                         int type, void* workspace, size_t workspace_bytes, dpa4k_stream_t stream_handle) {
  clear_error();
  Schedule c;
  if (int e = schedule_of("group norm backward", samples, entries, inner, channels, groups, type, offsets, max_entries, true, c))
    return e;
  hipStream_t stream = as_stream(stream_handle);
  if (c.shape.tiles == 0) {
    for (float* out : {grad_scale, grad_bias})
      if (out != nullptr)
        if (int e = zero_fill(out, channels * sizeof(float), stream)) return e;
    return DPA4K_OK;
  }
  if (grad == nullptr || x == nullptr || (samples > 0 && (mean == nullptr || rstd == nullptr)))
    return fail(DPA4K_EINVAL, "group norm backward: null pointer");
  if (grad_x == nullptr && grad_scale == nullptr && grad_bias == nullptr) return DPA4K_OK;
  Workspace w{};
  if (!carve(c, true, workspace, workspace_bytes, w))
    return fail(DPA4K_EWORKSPACE, "group norm backward: workspace of %zu bytes is smaller than %zu", workspace_bytes,
                workspace_bytes_of(c, true));
  if (type == DPA4K_TYPE_F32)
    return backward<float>(grad, x, scale, bias, mean, rstd, grad_x, grad_scale, grad_bias, c, silu != 0, w, stream);
  if (type == DPA4K_TYPE_BF16)
    return backward<__bf16>(grad, x, scale, bias, mean, rstd, grad_x, grad_scale, grad_bias, c, silu != 0, w, stream);
  return backward<_Float16>(grad, x, scale, bias, mean, rstd, grad_x, grad_scale, grad_bias, c, silu != 0, w, stream);
}
