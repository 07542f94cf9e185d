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
// Samples are ragged (CSR offsets) or of equal length, from no row to all of
// them, so the rows are cut into tiles of equal length whatever the samples: a
// workgroup per tile, which walks the pieces of samples in it.  A piece leaves
// its sums in slot (tile + sample), which is different for every piece since
// one of the two grows from piece to piece; a sample's slots are consecutive.
//
// A tile is read as one run of vectors.  Vector q of a run holds the channels
// (q V + j) mod C, so a stride of a multiple of lcm(C, V) elements keeps each
// thread on the same V channels at any width C: no access is scalar but in the
// ragged last vector of a piece.
#include <cmath>

#include "common.h"

namespace dpa4k {
namespace {

constexpr int kBlock = 512;
constexpr int kMaxChannels = DPA4K_GROUP_NORM_MAX_CHANNELS;
constexpr int64_t kTileBytes = 32768;   // least bytes of a tile
constexpr int64_t kTiles = 1024;        // most tiles, where they are larger than that: 4 workgroups per CU
constexpr float kLog2e = 1.4426950408889634f;

struct Shape {
  int64_t samples, entries, inner;   // a sample owns entries, an entry `inner` rows
  int channels, groups;
  int64_t tile_rows, tiles;
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
struct Values {
  float v[kVec<T>];
};

template <typename T>
__device__ __forceinline__ Values<T> load_whole(const T* __restrict__ p) {
  const auto raw = *reinterpret_cast<const typename vector_of<T>::type*>(p);
  Values<T> out;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) out.v[j] = static_cast<float>(raw[j]);
  return out;
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
  typename vector_of<T>::type raw;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) raw[j] = static_cast<T>(value.v[j]);
  *reinterpret_cast<typename vector_of<T>::type*>(p) = raw;
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
Columns columns_for(int channels) {
  Columns c;
  c.period_vectors = channels / gcd_of(channels, kVec<T>);
  c.copies = c.period_vectors < kBlock ? kBlock / c.period_vectors : 1;
  c.passes = (c.period_vectors + kBlock - 1) / kBlock;
  return c;
}

// A thread's share of one pass: the vectors first, first + stride, ... of a
// run, which hold the channels (channel + j) mod C.
struct Share {
  bool live;
  int first, channel;
};

template <typename T>
__device__ __forceinline__ Share share_of(const Columns& columns, int pass, int channels) {
  Share s;
  s.first = pass * kBlock + static_cast<int>(threadIdx.x);
  s.live = s.first < (columns.copies > 1 ? columns.stride_vectors() : columns.period_vectors);
  s.channel = static_cast<int>(static_cast<int64_t>(s.first) * kVec<T> % channels);
  return s;
}

__device__ __forceinline__ int channel_at(const Share& s, int j, int channels) {
  int c = s.channel + j;
  while (c >= channels) c -= channels;  // at most V / C times
  return c;
}

// ---------------------------------------------------------------------------
// samples in a tile
// ---------------------------------------------------------------------------

__device__ __forceinline__ int64_t clamped_offset(const Shape& s, int64_t sample) {
  if (s.offsets == nullptr) return sample;
  const int64_t o = s.offsets[sample];
  return o < 0 ? 0 : (o > s.entries ? s.entries : o);
}

// The last sample that starts at or before `entry`, -1 where none does.
__device__ __forceinline__ int64_t sample_at(const Shape& s, int64_t entry) {
  if (s.offsets == nullptr) return entry < s.samples ? entry : s.samples - 1;
  int64_t low = -1, high = s.samples - 1;
  while (low < high) {
    const int64_t middle = low + ((high - low + 1) >> 1);
    if (s.offsets[middle] <= entry) low = middle;
    else high = middle - 1;
  }
  return low;
}

// Calls piece(sample, first row, last row) for every sample with rows in the
// tile, in order; wave-uniform.
template <typename Piece>
__device__ __forceinline__ void each_piece(const Shape& s, int64_t tile, Piece piece) {
  const int64_t begin = tile * s.tile_rows;
  const int64_t rows = s.entries * s.inner;
  const int64_t end = begin + s.tile_rows < rows ? begin + s.tile_rows : rows;
  int64_t sample = sample_at(s, begin / s.inner);
  if (sample < 0) sample = 0;
  for (; sample < s.samples; ++sample) {
    const int64_t first = clamped_offset(s, sample) * s.inner;
    if (first >= end) break;
    const int64_t last = clamped_offset(s, sample + 1) * s.inner;
    const int64_t a = uniform_i64(first > begin ? first : begin);
    const int64_t b = uniform_i64(last < end ? last : end);
    if (a < b) piece(uniform_i64(sample), a, b);
  }
}

// ---------------------------------------------------------------------------
// sums of a workgroup by group of channels
// ---------------------------------------------------------------------------

// Lanes that add one group's `entries` terms, a power of two.
__device__ __forceinline__ int lanes_for(int entries) {
  int lanes = 1;
  while (lanes < 64 && lanes < entries) lanes <<= 1;
  return lanes;
}

__device__ __forceinline__ double lanes_sum(double value, int lanes) {
  for (int mask = 1; mask < lanes; mask <<= 1) value += __shfl_xor(value, mask);
  return value;
}

// ---------------------------------------------------------------------------
// forward: moments of each piece
// ---------------------------------------------------------------------------
//
// A thread merges batches of kBatch vectors into a running mean and sum of
// squared deviations per channel: the batch's own mean is taken off first, so
// neither a mean far from 0 nor a long sample costs digits.  The threads' pairs
// meet in LDS and are merged per group in 64 bits.
constexpr int kBatch = 4;

struct Moments {
  double count, mean, squares;
};

__device__ __forceinline__ Moments merged(const Moments& a, const Moments& b) {
  const double count = a.count + b.count;
  if (count == 0.0) return a;
  const double delta = b.mean - a.mean;
  const double share = b.count / count;
  return {count, a.mean + delta * share, a.squares + b.squares + delta * delta * a.count * share};
}

template <typename T>
__global__ __launch_bounds__(kBlock) void group_norm_moments_kernel(const T* __restrict__ x, Shape s, Columns columns,
                                                                    Moments* __restrict__ slots) {
  constexpr int V = kVec<T>;
  __shared__ float thread_mean[kBlock * V], thread_squares[kBlock * V];
  __shared__ int thread_count[kBlock];
  const int64_t tile = block_index();
  if (tile >= s.tiles) return;
  const int C = s.channels, D = C / s.groups;
  each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
    const T* run = x + a * C;
    const int64_t elements = (b - a) * C;
    const int64_t whole = elements / V;
    Moments* out = slots + (tile + sample) * s.groups;
    for (int pass = 0; pass < columns.passes; ++pass) {
      const Share share = share_of<T>(columns, pass, C);
      float mean[V], squares[V];
      int count = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) mean[j] = squares[j] = 0.0f;
      const int64_t stride = columns.stride_vectors();
      if (share.live) {
        int64_t q = share.first;
        for (; q + (kBatch - 1) * stride < whole; q += kBatch * stride) {
          Values<T> batch[kBatch];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) batch[k] = load_whole(run + (q + k * stride) * V);
          count += kBatch;
          const float weight = static_cast<float>(kBatch) / static_cast<float>(count);
          const float cross = static_cast<float>(count - kBatch) * weight;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float sum = batch[0].v[j];
#pragma unroll
            for (int k = 1; k < kBatch; ++k) sum += batch[k].v[j];
            const float own = sum * (1.0f / kBatch);
            float spread = 0.0f;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              const float d = batch[k].v[j] - own;
              spread = fmaf(d, d, spread);
            }
            const float delta = own - mean[j];
            mean[j] = fmaf(delta, weight, mean[j]);
            squares[j] = squares[j] + fmaf(delta * delta, cross, spread);
          }
        }
        for (; q < whole; q += stride) {
          const Values<T> value = load_whole(run + q * V);
          ++count;
          const float weight = 1.0f / static_cast<float>(count);
          const float cross = static_cast<float>(count - 1) * weight;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float delta = value.v[j] - mean[j];
            mean[j] = fmaf(delta, weight, mean[j]);
            squares[j] = fmaf(delta * delta, cross, squares[j]);
          }
        }
        // the elements behind the last whole vector: one more for some channels
        const int left = q == whole ? static_cast<int>(elements - whole * V) : 0;
        if (left > 0) {
          const Values<T> value = load_part(run + whole * V, left);
          const float weight = 1.0f / static_cast<float>(count + 1);
          const float cross = static_cast<float>(count) * weight;
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < left) {
              const float delta = value.v[j] - mean[j];
              mean[j] = fmaf(delta, weight, mean[j]);
              squares[j] = fmaf(delta * delta, cross, squares[j]);
            }
        }
        thread_count[threadIdx.x] = count * V + left;  // element j of a thread has count + (j < left) terms
#pragma unroll
        for (int j = 0; j < V; ++j) {
          thread_mean[threadIdx.x * V + j] = mean[j];
          thread_squares[threadIdx.x * V + j] = squares[j];
        }
      }
      __syncthreads();
      // this pass holds the elements [origin, origin + held) of each period
      const int origin = pass * kBlock * V;
      const int span = columns.copies > 1 ? columns.stride_vectors() * V : columns.period_vectors * V;
      const int held = span - origin < kBlock * V ? span - origin : kBlock * V;
      const int first_row = origin / C, last_row = (origin + held - 1) / C;
      const int terms = D * (last_row - first_row + 1);
      const int lanes = lanes_for(terms);
      const int lane = threadIdx.x & (lanes - 1);
      for (int g = static_cast<int>(threadIdx.x) / lanes; g < (s.groups + kBlock / lanes - 1) / (kBlock / lanes) * (kBlock / lanes);
           g += kBlock / lanes) {
        double total = 0.0, sum = 0.0;
        if (g < s.groups)
          for (int i = lane; i < terms; i += lanes) {
            const int e = (first_row + i / D) * C + g * D + i % D - origin;
            if (e < 0 || e >= held) continue;
            const int packed = thread_count[e / V];
            const double n = packed / V + (e % V < packed % V ? 1 : 0);
            total += n;
            sum += n * thread_mean[e];
          }
        total = lanes_sum(total, lanes);
        sum = lanes_sum(sum, lanes);
        const double centre = total > 0.0 ? sum / total : 0.0;
        double spread = 0.0;
        if (g < s.groups)
          for (int i = lane; i < terms; i += lanes) {
            const int e = (first_row + i / D) * C + g * D + i % D - origin;
            if (e < 0 || e >= held) continue;
            const int packed = thread_count[e / V];
            const double n = packed / V + (e % V < packed % V ? 1 : 0);
            const double delta = thread_mean[e] - centre;
            if (n > 0.0) spread += thread_squares[e] + n * delta * delta;
          }
        spread = lanes_sum(spread, lanes);
        if (lane == 0 && g < s.groups) {
          Moments mine = {total, centre, spread};
          if (pass > 0) mine = merged(out[g], mine);
          out[g] = mine;
        }
      }
      __syncthreads();
    }
  });
}

// A wave per (sample, group): its slots in their order, in 64 bits.  A sample
// without rows gets mean 0 and the rstd of variance 0; nothing reads them.
__global__ __launch_bounds__(256) void group_norm_finish_kernel(const Moments* __restrict__ slots, Shape s, float eps,
                                                                float* __restrict__ mean, float* __restrict__ rstd) {
  const int64_t unit = block_index() * 4 + (threadIdx.x >> 6);
  if (unit >= s.samples * s.groups) return;
  const int lane = threadIdx.x & 63;
  const int64_t sample = unit / s.groups;
  const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
  Moments total = {0.0, 0.0, 0.0};
  if (first < last) {
    const int64_t begin = first / s.tile_rows, end = (last - 1) / s.tile_rows;
    for (int64_t t = begin + lane; t <= end; t += 64) total = merged(total, slots[(t + sample) * s.groups + unit % s.groups]);
  }
#pragma unroll
  for (int mask = 1; mask < 64; mask <<= 1) {
    const Moments other = {__shfl_xor(total.count, mask), __shfl_xor(total.mean, mask), __shfl_xor(total.squares, mask)};
    total = (lane & mask) == 0 ? merged(total, other) : merged(other, total);
  }
  if (lane != 0) return;
  mean[unit] = static_cast<float>(total.mean);
  const double variance = total.count > 0.0 ? total.squares / total.count : 0.0;
  rstd[unit] = static_cast<float>(1.0 / sqrt(variance + static_cast<double>(eps)));
}

// ---------------------------------------------------------------------------
// forward: apply
// ---------------------------------------------------------------------------

// Rows of the tile that belong to no sample (before the first offset, behind the last).
template <typename T>
__device__ __forceinline__ void zero_outside(T* __restrict__ out, const Shape& s, int64_t tile) {
  if (s.offsets == nullptr) return;
  const int64_t begin = tile * s.tile_rows, rows = s.entries * s.inner;
  const int64_t end = begin + s.tile_rows < rows ? begin + s.tile_rows : rows;
  const int64_t first = s.samples > 0 ? clamped_offset(s, 0) * s.inner : rows;
  const int64_t last = s.samples > 0 ? clamped_offset(s, s.samples) * s.inner : rows;
  const int64_t head = (first < end ? first : end) * s.channels;
  const int64_t tail = (last > begin ? last : begin) * s.channels;
  for (int64_t i = begin * s.channels + threadIdx.x; i < head; i += kBlock) out[i] = static_cast<T>(0.0f);
  for (int64_t i = tail + threadIdx.x; i < end * s.channels; i += kBlock) out[i] = static_cast<T>(0.0f);
}

template <typename T, bool kSilu>
__global__ __launch_bounds__(kBlock) void group_norm_apply_kernel(const T* __restrict__ x, const float* __restrict__ scale,
                                                                  const float* __restrict__ bias,
                                                                  const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, T* __restrict__ y,
                                                                  Shape s, Columns columns) {
  constexpr int V = kVec<T>;
  const int64_t tile = block_index();
  if (tile >= s.tiles) return;
  const int C = s.channels, D = C / s.groups;
  for (int pass = 0; pass < columns.passes; ++pass) {
    const Share share = share_of<T>(columns, pass, C);
    if (!share.live) continue;
    float weight[V], shift[V];
    int group[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = channel_at(share, j, C);
      group[j] = c / D;
      weight[j] = scale != nullptr ? scale[c] : 1.0f;
      shift[j] = bias != nullptr ? bias[c] : 0.0f;
    }
    each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
      const T* run = x + a * C;
      T* out = y + a * C;
      const int64_t elements = (b - a) * C;
      const int64_t whole = elements / V;
      float centre[V], inverse[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        centre[j] = mean[sample * s.groups + group[j]];
        inverse[j] = rstd[sample * s.groups + group[j]];
      }
      const auto normed = [&](Values<T> value) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float z = fmaf((value.v[j] - centre[j]) * inverse[j], weight[j], shift[j]);
          value.v[j] = kSilu ? z * sigmoid(z) : z;
        }
        return value;
      };
      int64_t q = share.first;
      for (; q < whole; q += columns.stride_vectors()) store_whole(out + q * V, normed(load_whole(run + q * V)));
      const int left = static_cast<int>(elements - whole * V);
      if (q == whole && left > 0) store_part(out + whole * V, normed(load_part(run + whole * V, left)), left);
    });
  }
  zero_outside(y, s, tile);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// dz of one element, and h.
template <bool kSilu>
__device__ __forceinline__ float slope_times(float grad, float h, float weight, float shift) {
  if constexpr (!kSilu) return grad;
  const float z = fmaf(h, weight, shift);
  const float gate = sigmoid(z);
  return grad * (gate * fmaf(z, 1.0f - gate, 1.0f));
}

// Per piece: sum u and sum u h of each group.  Per tile: sum dz and sum dz h of
// each channel, over all its pieces (kept in registers across them; with more
// than one pass, pass by pass).
template <typename T, bool kSilu>
__global__ __launch_bounds__(kBlock) void group_norm_sums_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ scale,
    const float* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd, Shape s,
    Columns columns, double2* __restrict__ slots, float2* __restrict__ tile_sums) {
  constexpr int V = kVec<T>;
  __shared__ float thread_u[kBlock * V], thread_uh[kBlock * V];
  const int64_t tile = block_index();
  if (tile >= s.tiles) return;
  const int C = s.channels, D = C / s.groups;
  for (int pass = 0; pass < columns.passes; ++pass) {
    const Share share = share_of<T>(columns, pass, C);
    const int origin = pass * kBlock * V;
    const int span = columns.copies > 1 ? columns.stride_vectors() * V : columns.period_vectors * V;
    const int held = span - origin < kBlock * V ? span - origin : kBlock * V;
    float weight[V], shift[V], tile_z[V], tile_zh[V];
    int group[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = channel_at(share, j, C);
      group[j] = c / D;
      weight[j] = scale != nullptr ? scale[c] : 1.0f;
      shift[j] = bias != nullptr ? bias[c] : 0.0f;
      tile_z[j] = tile_zh[j] = 0.0f;
    }
    each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
      const int64_t elements = (b - a) * C;
      const int64_t whole = elements / V;
      float sum_z[V], sum_zh[V], centre[V], inverse[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        sum_z[j] = sum_zh[j] = 0.0f;
        centre[j] = mean[sample * s.groups + group[j]];
        inverse[j] = rstd[sample * s.groups + group[j]];
      }
      const auto add = [&](const Values<T>& gv, const Values<T>& xv) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float h = (xv.v[j] - centre[j]) * inverse[j];
          const float dz = slope_times<kSilu>(gv.v[j], h, weight[j], shift[j]);
          sum_z[j] += dz;
          sum_zh[j] = fmaf(dz, h, sum_zh[j]);
        }
      };
      if (share.live) {
        int64_t q = share.first;
        for (; q < whole; q += columns.stride_vectors())
          add(load_whole(grad + a * C + q * V), load_whole(x + a * C + q * V));
        const int left = static_cast<int>(elements - whole * V);
        if (q == whole && left > 0) {
          // a gradient of 0 adds nothing, unless h is not finite
          const Values<T> gv = load_part(grad + a * C + whole * V, left);
          Values<T> xv = load_part(x + a * C + whole * V, left);
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j >= left) xv.v[j] = centre[j];
          add(gv, xv);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          thread_u[threadIdx.x * V + j] = sum_z[j] * weight[j];
          thread_uh[threadIdx.x * V + j] = sum_zh[j] * weight[j];
          tile_z[j] += sum_z[j];
          tile_zh[j] += sum_zh[j];
        }
      }
      __syncthreads();
      const int first_row = origin / C, last_row = (origin + held - 1) / C;
      const int terms = D * (last_row - first_row + 1);
      const int lanes = lanes_for(terms);
      const int lane = threadIdx.x & (lanes - 1);
      double2* out = slots + (tile + sample) * s.groups;
      for (int g = static_cast<int>(threadIdx.x) / lanes; g < (s.groups + kBlock / lanes - 1) / (kBlock / lanes) * (kBlock / lanes);
           g += kBlock / lanes) {
        double u = 0.0, uh = 0.0;
        if (g < s.groups)
          for (int i = lane; i < terms; i += lanes) {
            const int e = (first_row + i / D) * C + g * D + i % D - origin;
            if (e < 0 || e >= held) continue;
            u += thread_u[e];
            uh += thread_uh[e];
          }
        u = lanes_sum(u, lanes);
        uh = lanes_sum(uh, lanes);
        if (lane == 0 && g < s.groups) {
          if (pass > 0) {
            u += out[g].x;
            uh += out[g].y;
          }
          out[g] = {u, uh};
        }
      }
      __syncthreads();
    });
    if (tile_sums == nullptr) continue;
    if (share.live)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        thread_u[threadIdx.x * V + j] = tile_z[j];
        thread_uh[threadIdx.x * V + j] = tile_zh[j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += kBlock) {
      float z = 0.0f, zh = 0.0f;
      bool any = false;
      for (int e = c - origin % C; e < held; e += C)
        if (e >= 0) {
          z += thread_u[e];
          zh += thread_uh[e];
          any = true;
        }
      float2* out = tile_sums + tile * C + c;
      if (pass == 0) *out = {z, zh};
      else if (any) *out = {out->x + z, out->y + zh};
    }
    __syncthreads();
  }
}

// A wave per (sample, group): means of u and u h over its slots.
__global__ __launch_bounds__(256) void group_norm_means_kernel(const double2* __restrict__ slots, Shape s,
                                                               float2* __restrict__ means) {
  const int64_t unit = block_index() * 4 + (threadIdx.x >> 6);
  if (unit >= s.samples * s.groups) return;
  const int lane = threadIdx.x & 63;
  const int64_t sample = unit / s.groups;
  const int64_t first = clamped_offset(s, sample) * s.inner, last = clamped_offset(s, sample + 1) * s.inner;
  double u = 0.0, uh = 0.0;
  if (first < last) {
    const int64_t begin = first / s.tile_rows, end = (last - 1) / s.tile_rows;
    for (int64_t t = begin + lane; t <= end; t += 64) {
      const double2 v = slots[(t + sample) * s.groups + unit % s.groups];
      u += v.x;
      uh += v.y;
    }
  }
  u = group_sum<64>(u);
  uh = group_sum<64>(uh);
  const double count = static_cast<double>((last - first) * (s.channels / s.groups));
  if (lane == 0 && first < last) means[unit] = {static_cast<float>(u / count), static_cast<float>(uh / count)};
}

template <typename T, bool kSilu>
__global__ __launch_bounds__(kBlock) void group_norm_backward_kernel(
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ scale,
    const float* __restrict__ bias, const float* __restrict__ mean, const float* __restrict__ rstd,
    const float2* __restrict__ means, T* __restrict__ grad_x, Shape s, Columns columns) {
  constexpr int V = kVec<T>;
  const int64_t tile = block_index();
  if (tile >= s.tiles) return;
  const int C = s.channels, D = C / s.groups;
  for (int pass = 0; pass < columns.passes; ++pass) {
    const Share share = share_of<T>(columns, pass, C);
    if (!share.live) continue;
    float weight[V], shift[V];
    int group[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = channel_at(share, j, C);
      group[j] = c / D;
      weight[j] = scale != nullptr ? scale[c] : 1.0f;
      shift[j] = bias != nullptr ? bias[c] : 0.0f;
    }
    each_piece(s, tile, [&](int64_t sample, int64_t a, int64_t b) {
      const int64_t elements = (b - a) * C;
      const int64_t whole = elements / V;
      float centre[V], inverse[V], mean_u[V], mean_uh[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int64_t at = sample * s.groups + group[j];
        centre[j] = mean[at];
        inverse[j] = rstd[at];
        mean_u[j] = means[at].x;
        mean_uh[j] = means[at].y;
      }
      const auto gradient = [&](const Values<T>& gv, const Values<T>& xv) {
        Values<T> out;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float h = (xv.v[j] - centre[j]) * inverse[j];
          const float u = slope_times<kSilu>(gv.v[j], h, weight[j], shift[j]) * weight[j];
          out.v[j] = inverse[j] * ((u - mean_u[j]) - h * mean_uh[j]);
        }
        return out;
      };
      const T* run_g = grad + a * C;
      const T* run_x = x + a * C;
      T* out = grad_x + a * C;
      int64_t q = share.first;
      for (; q < whole; q += columns.stride_vectors())
        store_whole(out + q * V, gradient(load_whole(run_g + q * V), load_whole(run_x + q * V)));
      const int left = static_cast<int>(elements - whole * V);
      if (q == whole && left > 0)
        store_part(out + whole * V, gradient(load_part(run_g + whole * V, left), load_part(run_x + whole * V, left)), left);
    });
  }
  zero_outside(grad_x, s, tile);
}

// dbias and dscale: a workgroup per 64 channels, its 16 waves on shares of the
// tiles, in 64 bits, added in order.
constexpr int kColumnWaves = 16;

__global__ __launch_bounds__(kColumnWaves * 64) void group_norm_columns_kernel(const float2* __restrict__ tile_sums,
                                                                               int64_t tiles, int channels,
                                                                               float* __restrict__ grad_scale,
                                                                               float* __restrict__ grad_bias) {
  __shared__ double2 wave_sum[kColumnWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int channel = blockIdx.x * 64 + lane;
  double z = 0.0, zh = 0.0;
  if (channel < channels)
    for (int64_t t = wave; t < tiles; t += kColumnWaves) {
      const float2 v = tile_sums[t * channels + channel];
      z += v.x;
      zh += v.y;
    }
  wave_sum[wave][lane] = {z, zh};
  __syncthreads();
  if (wave != 0 || channel >= channels) return;
#pragma unroll
  for (int w = 1; w < kColumnWaves; ++w) {
    z += wave_sum[w][lane].x;
    zh += wave_sum[w][lane].y;
  }
  if (grad_bias != nullptr) grad_bias[channel] = static_cast<float>(z);
  if (grad_scale != nullptr) grad_scale[channel] = static_cast<float>(zh);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int64_t type_bytes(int type) { return type == DPA4K_TYPE_F32 ? 4 : 2; }

// Checks the sizes and cuts the rows into tiles.
int shape_of(const char* what, int64_t samples, int64_t entries, int64_t inner, int64_t channels, int64_t groups,
             int type, const int64_t* offsets, Shape& s) {
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
  const int64_t least = kTileBytes / (channels * type_bytes(type));
  int64_t tile_rows = (rows + kTiles - 1) / kTiles;
  if (tile_rows < least) tile_rows = least;
  if (tile_rows < 1) tile_rows = 1;
  s = {samples, entries, inner, static_cast<int>(channels), static_cast<int>(groups), tile_rows,
       (rows + tile_rows - 1) / tile_rows, offsets};
  if (!grid_fits(samples * groups / 4 + 1, 256)) return fail(DPA4K_EINVAL, "%s: the sample count exceeds the launch limit", what);
  return DPA4K_OK;
}

struct Workspace {
  void* slots;        // Moments or double2 per (piece, group)
  float2* means;      // per (sample, group), backward
  float2* tile_sums;  // per (tile, channel), backward
};

bool carve(Carver& carver, const Shape& s, bool backward, Workspace& w) {
  const size_t pieces = static_cast<size_t>(s.tiles + s.samples) * s.groups;
  if (!backward) {
    w.slots = carver.take<Moments>(pieces);
    return w.slots != nullptr;
  }
  w.slots = carver.take<double2>(pieces);
  w.means = carver.take<float2>(static_cast<size_t>(s.samples) * s.groups);
  w.tile_sums = carver.take<float2>(static_cast<size_t>(s.tiles) * s.channels);
  return w.slots != nullptr && w.means != nullptr && w.tile_sums != nullptr;
}

size_t workspace_bytes_of(const Shape& s, bool backward) {
  const size_t pieces = static_cast<size_t>(s.tiles + s.samples) * s.groups;
  if (!backward) return round_up_256(pieces * sizeof(Moments));
  return round_up_256(pieces * sizeof(double2)) + round_up_256(static_cast<size_t>(s.samples) * s.groups * sizeof(float2)) +
         round_up_256(static_cast<size_t>(s.tiles) * s.channels * sizeof(float2));
}

template <typename T>
int forward(const void* x, const float* scale, const float* bias, void* y, float* mean, float* rstd, const Shape& s,
            float eps, bool silu, const Workspace& w, hipStream_t stream) {
  const Columns columns = columns_for<T>(s.channels);
  Moments* slots = static_cast<Moments*>(w.slots);
  const dim3 grid = launch_grid(s.tiles, kBlock);
  group_norm_moments_kernel<T><<<grid, kBlock, 0, stream>>>(static_cast<const T*>(x), s, columns, slots);
  if (int e = launched("group_norm_moments_kernel")) return e;
  if (s.samples > 0) {
    group_norm_finish_kernel<<<launch_grid((s.samples * s.groups + 3) / 4, 256), 256, 0, stream>>>(slots, s, eps, mean, rstd);
    if (int e = launched("group_norm_finish_kernel")) return e;
  }
  (silu ? group_norm_apply_kernel<T, true> : group_norm_apply_kernel<T, false>)<<<grid, kBlock, 0, stream>>>(
      static_cast<const T*>(x), scale, bias, mean, rstd, static_cast<T*>(y), s, columns);
  return launched("group_norm_apply_kernel");
}

template <typename T>
int backward(const void* grad, const void* x, const float* scale, const float* bias, const float* mean,
             const float* rstd, void* grad_x, float* grad_scale, float* grad_bias, const Shape& s, bool silu,
             const Workspace& w, hipStream_t stream) {
  const Columns columns = columns_for<T>(s.channels);
  double2* slots = static_cast<double2*>(w.slots);
  const bool parameters = grad_scale != nullptr || grad_bias != nullptr;
  const dim3 grid = launch_grid(s.tiles, kBlock);
  (silu ? group_norm_sums_kernel<T, true> : group_norm_sums_kernel<T, false>)<<<grid, kBlock, 0, stream>>>(
      static_cast<const T*>(grad), static_cast<const T*>(x), scale, bias, mean, rstd, s, columns, slots,
      parameters ? w.tile_sums : nullptr);
  if (int e = launched("group_norm_sums_kernel")) return e;
  if (grad_x != nullptr) {
    if (s.samples > 0) {
      group_norm_means_kernel<<<launch_grid((s.samples * s.groups + 3) / 4, 256), 256, 0, stream>>>(slots, s, w.means);
      if (int e = launched("group_norm_means_kernel")) return e;
    }
    (silu ? group_norm_backward_kernel<T, true> : group_norm_backward_kernel<T, false>)<<<grid, kBlock, 0, stream>>>(
        static_cast<const T*>(grad), static_cast<const T*>(x), scale, bias, mean, rstd, w.means, static_cast<T*>(grad_x), s,
        columns);
    if (int e = launched("group_norm_backward_kernel")) return e;
  }
  if (!parameters) return DPA4K_OK;
  group_norm_columns_kernel<<<blocks_for(s.channels, 64), kColumnWaves * 64, 0, stream>>>(w.tile_sums, s.tiles, s.channels,
                                                                                        grad_scale, grad_bias);
  return launched("group_norm_columns_kernel");
}

}  // namespace
}  // namespace dpa4k

using namespace dpa4k;

extern "C" size_t dpa4k_group_norm_workspace_size(int64_t samples, int64_t entries, int64_t inner, int64_t channels,
                                                  int64_t groups, int type, int backward) {
  Shape s;
  static const int64_t some = 0;  // any offsets: the size does not depend on them
  if (shape_of("group norm", samples, entries, inner, channels, groups, type, &some, s)) return 0;
  return workspace_bytes_of(s, backward != 0);
}

extern "C" int dpa4k_group_norm_forward(const void* x, const float* scale, const float* bias, const int64_t* offsets,
                                        void* y, float* mean, float* rstd, int64_t samples, int64_t entries,
                                        int64_t inner, int64_t channels, int64_t groups, float eps, int silu, int type,
                                        void* workspace, size_t workspace_bytes, dpa4k_stream_t stream_handle) {
  clear_error();
  Shape s;
  if (int e = shape_of("group norm", samples, entries, inner, channels, groups, type, offsets, s)) return e;
  if (!(eps > 0.0f) || !(eps < INFINITY)) return fail(DPA4K_EINVAL, "group norm eps must be a finite positive number");
  if (s.tiles == 0) return DPA4K_OK;
  if (x == nullptr || y == nullptr || (samples > 0 && (mean == nullptr || rstd == nullptr)))
    return fail(DPA4K_EINVAL, "group norm: null pointer");
  Carver carver{static_cast<char*>(workspace), workspace == nullptr ? 0 : workspace_bytes};
  Workspace w{};
  if (!carve(carver, s, false, w))
    return fail(DPA4K_EWORKSPACE, "group norm: workspace of %zu bytes is smaller than %zu", workspace_bytes,
                workspace_bytes_of(s, false));
  hipStream_t stream = as_stream(stream_handle);
  if (type == DPA4K_TYPE_F32) return forward<float>(x, scale, bias, y, mean, rstd, s, eps, silu != 0, w, stream);
  if (type == DPA4K_TYPE_BF16) return forward<__bf16>(x, scale, bias, y, mean, rstd, s, eps, silu != 0, w, stream);
  return forward<_Float16>(x, scale, bias, y, mean, rstd, s, eps, silu != 0, w, stream);
}

extern "C" int dpa4k_group_norm_backward(const void* grad, const void* x, const float* scale, const float* bias,
                                         const int64_t* offsets, const float* mean, const float* rstd, void* grad_x,
                                         float* grad_scale, float* grad_bias, int64_t samples, int64_t entries,
                                         int64_t inner, int64_t channels, int64_t groups, int silu, int type,
                                         void* workspace, size_t workspace_bytes, dpa4k_stream_t stream_handle) {
  clear_error();
  Shape s;
  if (int e = shape_of("group norm backward", samples, entries, inner, channels, groups, type, offsets, s)) return e;
  hipStream_t stream = as_stream(stream_handle);
  if (s.tiles == 0) {
    for (float* out : {grad_scale, grad_bias})
      if (out != nullptr)
        if (int e = zero_fill(out, channels * sizeof(float), stream)) return e;
    return DPA4K_OK;
  }
  if (grad == nullptr || x == nullptr || (samples > 0 && (mean == nullptr || rstd == nullptr)))
    return fail(DPA4K_EINVAL, "group norm backward: null pointer");
  if (grad_x == nullptr && grad_scale == nullptr && grad_bias == nullptr) return DPA4K_OK;
  Carver carver{static_cast<char*>(workspace), workspace == nullptr ? 0 : workspace_bytes};
  Workspace w{};
  if (!carve(carver, s, true, w))
    return fail(DPA4K_EWORKSPACE, "group norm backward: workspace of %zu bytes is smaller than %zu", workspace_bytes,
                workspace_bytes_of(s, true));
  if (type == DPA4K_TYPE_F32)
    return backward<float>(grad, x, scale, bias, mean, rstd, grad_x, grad_scale, grad_bias, s, silu != 0, w, stream);
  if (type == DPA4K_TYPE_BF16)
    return backward<__bf16>(grad, x, scale, bias, mean, rstd, grad_x, grad_scale, grad_bias, s, silu != 0, w, stream);
  return backward<_Float16>(grad, x, scale, bias, mean, rstd, grad_x, grad_scale, grad_bias, s, silu != 0, w, stream);
}
