// The norms around a block with its gate and residual sum, forward and backward
// (no counterpart in the reference, whose RMSNorm stands alone; the residual adds
// and gates around it are passes of their own there):
//
//   r = 1 / sqrt(mean x^2 + eps)        a = x r post      (norm after the block)
//   h = residual + scale act(gate) a                      (residual sum)
//   q = 1 / sqrt(mean h^2 + eps)        y = h q pre       (norm before the next)
//
//   u = dy pre,  g = dh + q (u - h q^2 mean(u h)),  dpre = sum dy h q
//   dresidual = g,  dscale = sum g act a,  dgate = g scale a act'
//   b = g scale act,  dpost = sum b x r,  v = b post,  dx = r (v - x r^2 mean(v x))
//
// Bound by its streams: each input is read once and each output written once,
// because a row stays in the registers of the lanes that share it, L of them with
// E elements each: 8 to 64 lanes of a wave for rows of up to 1,024 (two waves of
// half the elements were as fast forward and slower backward, 126 -> 170 us for
// 30,011 rows of 810, as their sums need a barrier each), a workgroup
// beyond.  h is not kept in 32 bits between the two passes; the backward computes it
// again from the residual, which is as many bytes as reading h, and y and the
// gradients see the unrounded h.
//
// The gradients of post, pre and scale are sums over all rows.  A workgroup walks
// its rows with the columns' sums in LDS, each set of L lanes its own for at most kRunRows
// rows (sums in 32 bits stay short), adds up to 32 of these and leaves one row of
// partial sums; a second launch adds those in 64 bits in a fixed order.
//
// Measured: 24,576 rows of 1,024 in float32 with a gate, forward 92 us (5.5 TB/s of
// its five streams), backward 160 us (5.0 TB/s of eight); 30,011 rows of 810 in
// bfloat16 on a float32 residual, forward 54 us (5.4 TB/s), backward 117 us
// (3.7 TB/s; rows that start anywhere, four tenths of the second chunk's lanes idle).
// Outputs are stored past the caches (through them: 90, 160, 61 and 123 us).  Rows over
// a workgroup with a full gate: 6,144 of 4,096 in float32 91 us (5.6 TB/s) and 225 (3.6), 6,144
// of 8,192 in bfloat16 101 us (5.0) and 243 (3.3).
#include "elements.h"

namespace dpa4k {
namespace {

constexpr int kMaxWidth = DPA4K_RESIDUAL_NORM_MAX_CHANNELS;
constexpr int64_t kRunRows = 256;

enum { kGateNone = 0, kGateFull = 1, kGateRow = 2 };
enum { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };

struct NormCall {
  const void* x;
  const void* residual;
  const void* gate;
  const float* post;
  const float* scale;
  const float* pre;
  void* h;            // forward
  void* y;
  float* r;
  float* q;
  const void* dh;     // backward
  const void* dy;
  void* dx;
  void* dresidual;
  void* dgate;
  float* partial;     // [3][workgroups][width] of dpost, dpre, dscale
  float scale_value, eps;
  int64_t rows;
  int width, gate_kind, act, post_norm, pre_norm, want_sums;
};

// act(gate) and its slope.
__device__ __forceinline__ float gate_value(float gate, int act, float& slope) {
  slope = 1.0f;
  if (act == kActNone) return gate;
  float other;
  const float s = logistic(gate, other);
  if (act == kActSigmoid) {
    slope = s * other;
    return s;
  }
  slope = s * fmaf(gate, other, 1.0f);
  return gate * s;
}

// Sum over the L lanes that share a row, every lane receives it.  With more than
// a wave, `slot` numbers the sums of one row: each has its own words of LDS, so
// that one barrier a sum suffices (the words of sum `slot` are written again only
// behind the barriers of the others, or of `finish`).
template <int L>
__device__ __forceinline__ float row_sum(float value, float (*words)[16], int slot) {
  if constexpr (L <= 64) {
    return group_sum<L>(value);
  } else {
    value = group_sum<64>(value);
    if ((threadIdx.x & 63) == 0) words[slot][threadIdx.x / 64] = value;
    __syncthreads();
    const int first = threadIdx.x / L * (L / 64);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) sum += words[slot][first + w];
    return sum;
  }
}

template <typename T, typename R, int L, int E>
struct Row {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int N = E / V;
  static constexpr int kBlock = L > 256 ? L : 256;
  static constexpr int kGroups = kBlock / L;

  // Elements n V .. of this lane's chunk n: column (n L + lane) V.
  static __device__ __forceinline__ int column(int n, int lane) { return (n * L + lane) * V; }
};

// Whether a chunk of the workgroup's rows from `first` on may reach past the tensor.
template <typename T, typename R, int L, int E>
__device__ __forceinline__ bool near_end(int64_t first, int64_t rows, int width) {
  typedef Row<T, R, L, E> Z;
  return (rows - first - Z::kGroups) * width < Z::V;
}

// One stream at this lane's columns of `row`, as it is in memory.  A ragged chunk is
// read with the start of the next row and masked by `values_of`, or, where the
// workgroup has the last row, behind which nothing may be read, piece by piece.
// All streams of a row are loaded in one block of code and masked behind it: what
// uses a value in between waits for it, and what follows is loaded no sooner.
template <typename T, typename S, int E>
struct Stream {
  static constexpr int V = 16 / sizeof(T);
  Pack<S, V> chunk[E / V];
};

template <bool LAST, typename T, typename R, int L, int E, typename S>
__device__ __forceinline__ void load_stream(const S* __restrict__ p, int64_t row, int lane, int width, int64_t total, bool live,
                                            Stream<T, S, E>& to) {
  typedef Row<T, R, L, E> Z;
#pragma unroll
  for (int n = 0; n < Z::N; ++n) {
    const int c = Z::column(n, lane);
    const int64_t at = row * width + c;
    if constexpr (LAST) to.chunk[n] = load_pack<S, Z::V>(p + at, live ? width - c : 0, total - at);
    else to.chunk[n] = *reinterpret_cast<const Pack<S, Z::V>*>(p + row * width + (c < width ? c : 0));
  }
}

// The values of a stream, zeros behind the row.
template <typename T, typename R, int L, int E, typename S>
__device__ __forceinline__ void values_of(const Stream<T, S, E>& from, int lane, int width, float (&out)[E]) {
  typedef Row<T, R, L, E> Z;
#pragma unroll
  for (int n = 0; n < Z::N; ++n) {
    const int here = width - Z::column(n, lane);
#pragma unroll
    for (int j = 0; j < Z::V; ++j) out[n * Z::V + j] = j < here ? static_cast<float>(from.chunk[n][j]) : 0.0f;
  }
}

template <typename T, typename S, typename R, int L, int E>
__device__ __forceinline__ void store_row(S* __restrict__ p, int64_t row, int lane, int width, bool live, const float (&value)[E]) {
  typedef Row<T, R, L, E> Z;
  if (!live) return;
#pragma unroll
  for (int n = 0; n < Z::N; ++n) {
    const int c = Z::column(n, lane);
    float part[Z::V];
#pragma unroll
    for (int j = 0; j < Z::V; ++j) part[j] = value[n * Z::V + j];
    if (c < width) store_pack<true, S, Z::V>(p + row * width + c, part, width - c);
  }
}

template <typename T, typename R, int L, int E>
__device__ __forceinline__ void load_weight(const float* __restrict__ p, float otherwise, int lane, int width, float (&out)[E]) {
  if (p != nullptr) {
    Stream<T, float, E> raw;
    load_stream<true, T, R, L, E>(p, 0, lane, width, width, true, raw);
    values_of<T, R, L, E>(raw, lane, width, out);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) out[i] = otherwise;
  }
}

// What forward and backward share: h of one row from its inputs.
template <int E>
__device__ __forceinline__ void residual_sum(const float (&x)[E], const float (&residual)[E], const float (&act)[E],
                                             const float (&post)[E], const float (&scale)[E], float r, float (&h)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) h[i] = fmaf(scale[i] * act[i], x[i] * r * post[i], residual[i]);
}

template <typename T, typename R, int L, int E, bool FULL_GATE>
__global__ __launch_bounds__((L > 256 ? L : 256)) void residual_norm_forward_kernel(NormCall call) {
  typedef Row<T, R, L, E> Z;
  __shared__ float words[2][16];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int width = call.width;
  const int64_t total = call.rows * width;
  const T* x_at = static_cast<const T*>(call.x);
  const R* residual_at = static_cast<const R*>(call.residual);
  const T* gate_at = static_cast<const T*>(call.gate);
  const int64_t row = block_index() * Z::kGroups + group;
  if (block_index() * Z::kGroups >= call.rows) return;
  const bool live = row < call.rows;
  const bool last = near_end<T, R, L, E>(block_index() * Z::kGroups, call.rows, width);
  float x[E], residual[E], act[E], post[E], scale[E], h[E];
  Stream<T, T, E> raw_x, raw_gate;
  Stream<T, R, E> raw_residual;
  const auto load = [&](auto at_end) {
    constexpr bool LAST = decltype(at_end)::value;
    load_stream<LAST, T, R, L, E>(x_at, row, lane, width, total, live, raw_x);
    load_stream<LAST, T, R, L, E>(residual_at, row, lane, width, total, live, raw_residual);
    if constexpr (FULL_GATE) load_stream<LAST, T, R, L, E>(gate_at, row, lane, width, total, live, raw_gate);
  };
  if (last) load(std::true_type{});
  else load(std::false_type{});
  values_of<T, R, L, E>(raw_x, lane, width, x);
  values_of<T, R, L, E>(raw_residual, lane, width, residual);
  if constexpr (FULL_GATE) {
    values_of<T, R, L, E>(raw_gate, lane, width, act);
  } else {
    float one = 1.0f, slope;
    if (call.gate_kind == kGateRow) one = gate_value(live ? static_cast<float>(gate_at[row]) : 0.0f, call.act, slope);
#pragma unroll
    for (int i = 0; i < E; ++i) act[i] = one;
  }
  load_weight<T, R, L, E>(call.post, 1.0f, lane, width, post);
  load_weight<T, R, L, E>(call.scale, call.scale_value, lane, width, scale);
  float r = 1.0f;
  if (call.post_norm) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) sum = fmaf(x[i], x[i], sum);
    r = 1.0f / sqrtf(row_sum<L>(sum, words, 0) / static_cast<float>(width) + call.eps);
  }
  if constexpr (FULL_GATE) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float slope;
      act[i] = gate_value(act[i], call.act, slope);
    }
  }
  residual_sum<E>(x, residual, act, post, scale, r, h);
  store_row<T, R, R, L, E>(static_cast<R*>(call.h), row, lane, width, live, h);
  if (call.pre_norm) {
    float pre[E], sum = 0.0f;
    load_weight<T, R, L, E>(call.pre, 1.0f, lane, width, pre);
#pragma unroll
    for (int i = 0; i < E; ++i) sum = fmaf(h[i], h[i], sum);
    const float q = 1.0f / sqrtf(row_sum<L>(sum, words, 1) / static_cast<float>(width) + call.eps);
#pragma unroll
    for (int i = 0; i < E; ++i) pre[i] *= h[i] * q;
    store_row<T, T, R, L, E>(static_cast<T*>(call.y), row, lane, width, live, pre);
    if (call.q != nullptr && live && lane == 0) call.q[row] = q;
  }
  if (call.post_norm && call.r != nullptr && live && lane == 0) call.r[row] = r;
}

// A workgroup's sums of columns lie in LDS, [3][chunks][threads][V], each thread's
// own: registers for them (48 of 250 with 16 elements a lane) would halve the waves
// that are resident, or leave no room to load all streams of a row at once.
template <typename T, typename R, int L, int E>
__device__ __forceinline__ void add_to(float* words, const float (&value)[E]) {
  typedef Row<T, R, L, E> Z;
#pragma unroll
  for (int n = 0; n < Z::N; ++n) {
    float* at = words + (n * Z::kBlock + static_cast<int>(threadIdx.x)) * Z::V;
#pragma unroll
    for (int j = 0; j < Z::V; j += 4) {
      f32x4* four = reinterpret_cast<f32x4*>(at + j);
      f32x4 sum = *four;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += value[n * Z::V + j + i];
      *four = sum;
    }
  }
}

// One sum of columns over the row groups of the workgroup, in order, to its row of
// partial sums.
template <typename T, typename R, int L, int E>
__device__ __forceinline__ void leave_sums(const float* words, float* __restrict__ to, int width) {
  typedef Row<T, R, L, E> Z;
  for (int c = threadIdx.x; c < width; c += Z::kBlock) {
    const int chunk = c / Z::V;
    const float* at = words + (chunk / L * Z::kBlock + chunk % L) * Z::V + c % Z::V;
    float all = 0.0f;
    for (int g = 0; g < Z::kGroups; ++g) all += at[g * L * Z::V];
    to[c] = all;
  }
}

template <typename T, typename R, int L, int E, bool FULL_GATE>
__global__ __launch_bounds__((L > 256 ? L : 256)) void residual_norm_backward_kernel(NormCall call, int64_t blocks) {
  typedef Row<T, R, L, E> Z;
  __shared__ float words[3][16];
  __shared__ __attribute__((aligned(16))) float sums[3][Z::kBlock * E];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int width = call.width;
  const float inverse_width = 1.0f / static_cast<float>(width);
  const int64_t total = call.rows * width;
  const int64_t block = block_index();
  if (block >= blocks) return;
  const T* x_at = static_cast<const T*>(call.x);
  const R* residual_at = static_cast<const R*>(call.residual != nullptr ? call.residual : call.dh);
  const T* gate_at = static_cast<const T*>(call.gate);
  const T* dy_at = call.dy != nullptr ? static_cast<const T*>(call.dy) : x_at;
  const R* dh_at = static_cast<const R*>(call.dh != nullptr ? call.dh : call.residual);
  for (int i = threadIdx.x; i < 3 * Z::kBlock * E; i += Z::kBlock) (&sums[0][0])[i] = 0.0f;
  __syncthreads();

  for (int64_t first = block * Z::kGroups; first < call.rows; first += blocks * Z::kGroups) {
    const int64_t row = first + group;
    const bool live = row < call.rows;
    const bool last = near_end<T, R, L, E>(first, call.rows, width);
    float x[E], act[E], slope[E], post[E], scale[E], g[E];
    // in the place of a stream that is not there another one is read again, which costs no bytes
    Stream<T, T, E> raw_x, raw_gate, raw_dy;
    Stream<T, R, E> raw_residual, raw_dh;
    const auto load = [&](auto at_end) {
      constexpr bool LAST = decltype(at_end)::value;
      load_stream<LAST, T, R, L, E>(x_at, row, lane, width, total, live, raw_x);
      load_stream<LAST, T, R, L, E>(residual_at, row, lane, width, total, live, raw_residual);
      if constexpr (FULL_GATE) load_stream<LAST, T, R, L, E>(gate_at, row, lane, width, total, live, raw_gate);
      load_stream<LAST, T, R, L, E>(dh_at, row, lane, width, total, live, raw_dh);
      load_stream<LAST, T, R, L, E>(dy_at, row, lane, width, total, live, raw_dy);
    };
    if (last) load(std::true_type{});
    else load(std::false_type{});
    values_of<T, R, L, E>(raw_x, lane, width, x);
    if constexpr (FULL_GATE) {
      values_of<T, R, L, E>(raw_gate, lane, width, act);
    } else {
      float one = 1.0f, its_slope = 0.0f;
      if (call.gate_kind == kGateRow) one = gate_value(live ? static_cast<float>(gate_at[row]) : 0.0f, call.act, its_slope);
#pragma unroll
      for (int i = 0; i < E; ++i) act[i] = one, slope[i] = its_slope;
    }
    values_of<T, R, L, E>(raw_dh, lane, width, g);
    if (call.dh == nullptr) {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = 0.0f;
    }
    load_weight<T, R, L, E>(call.post, 1.0f, lane, width, post);
    load_weight<T, R, L, E>(call.scale, call.scale_value, lane, width, scale);
    const float r = call.post_norm && live ? call.r[row] : 1.0f;
    if constexpr (FULL_GATE) {
#pragma unroll
      for (int i = 0; i < E; ++i) act[i] = gate_value(act[i], call.act, slope[i]);
    }
    if (call.dy != nullptr) {
      float residual[E], dy[E], pre[E], h[E];
      values_of<T, R, L, E>(raw_residual, lane, width, residual);
      values_of<T, R, L, E>(raw_dy, lane, width, dy);
      load_weight<T, R, L, E>(call.pre, 1.0f, lane, width, pre);
      const float q = live ? call.q[row] : 0.0f;
      residual_sum<E>(x, residual, act, post, scale, r, h);
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        h[i] *= q;
        pre[i] *= dy[i];
        dy[i] *= h[i];
        dot = fmaf(pre[i], h[i], dot);
      }
      add_to<T, R, L, E>(sums[1], dy);
      dot = row_sum<L>(dot, words, 0) * inverse_width;
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = fmaf(q, fmaf(-h[i], dot, pre[i]), g[i]);
    }
    if (call.dresidual != nullptr) store_row<T, R, R, L, E>(static_cast<R*>(call.dresidual), row, lane, width, live, g);
    // x from here on is x r, the normed row
    float dot = 0.0f, row_gate = 0.0f, of_scale[E], of_post[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x[i] *= r;
      const float a = x[i] * post[i];
      of_scale[i] = g[i] * (act[i] * a);
      const float b = g[i] * scale[i];
      slope[i] *= b * a;   // the gate's gradient
      g[i] = b * act[i];
      of_post[i] = g[i] * x[i];
      g[i] *= post[i];
      dot = fmaf(g[i], x[i], dot);
    }
    add_to<T, R, L, E>(sums[2], of_scale);
    add_to<T, R, L, E>(sums[0], of_post);
    if (call.dgate != nullptr) {
      if (call.gate_kind == kGateFull) {
        store_row<T, T, R, L, E>(static_cast<T*>(call.dgate), row, lane, width, live, slope);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) row_gate += slope[i];
        row_gate = row_sum<L>(row_gate, words, 1);
        if (live && lane == 0) static_cast<T*>(call.dgate)[row] = static_cast<T>(row_gate);
      }
    }
    if (call.post_norm) {
      dot = row_sum<L>(dot, words, 2) * inverse_width;
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = r * fmaf(-x[i], dot, g[i]);
    }
    if (call.dx != nullptr) store_row<T, T, R, L, E>(static_cast<T*>(call.dx), row, lane, width, live, g);
    if constexpr (L > 64) __syncthreads();   // before the words of the next row
  }
  if (!call.want_sums) return;
  __syncthreads();
  for (int sum = 0; sum < 3; ++sum)
    leave_sums<T, R, L, E>(sums[sum], call.partial + (sum * blocks + block) * width, width);
}

// out[c] = sum over the workgroups of partial[.][c], 32 columns a workgroup, eight
// threads a column, in 64 bits.
__global__ __launch_bounds__(256) void column_sums_kernel(const float* __restrict__ partial, int64_t blocks, int width,
                                                          float* __restrict__ dpost, float* __restrict__ dpre,
                                                          float* __restrict__ dscale) {
  __shared__ double words[8][32];
  float* out = blockIdx.y == 0 ? dpost : blockIdx.y == 1 ? dpre : dscale;
  if (out == nullptr) return;
  const int column = blockIdx.x * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  const float* from = partial + blockIdx.y * blocks * width;
  double sum = 0.0;
  if (column < width) {
#pragma unroll 8
    for (int64_t b = part; b < blocks; b += 8) sum += static_cast<double>(from[b * width + column]);
  }
  words[part][threadIdx.x % 32] = sum;
  __syncthreads();
  if (part == 0 && column < width) {
#pragma unroll
    for (int p = 1; p < 8; ++p) sum += words[p][threadIdx.x];
    out[column] = static_cast<float>(sum);
  }
}

// Calls `use` with the lanes and elements a lane of rows of `width`.
template <typename F>
int with_layout(int width, F&& use) {
  if (width <= 64) return use(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
  if (width <= 128) return use(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{});
  if (width <= 256) return use(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
  if (width <= 512) return use(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
  if (width <= 1024) return use(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
  if (width <= 2048) return use(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
  if (width <= 4096) return use(std::integral_constant<int, 256>{}, std::integral_constant<int, 16>{});
  return use(std::integral_constant<int, 512>{}, std::integral_constant<int, 16>{});
}

template <typename F>
int with_types(int type, int residual_type, F&& use) {
  return with_type(type, DPA4K_EINVAL, [&](auto t) -> int {
    typedef typename decltype(t)::type T;
    if (residual_type == DPA4K_TYPE_F32) return use(type_of<T>{}, type_of<float>{});
    if constexpr (!std::is_same<T, float>::value) return use(type_of<T>{}, type_of<T>{});
    return DPA4K_EINVAL;
  });
}

int row_groups(int width) {
  int groups = 0;
  with_layout(width, [&](auto l, auto) {
    groups = (l.value > 256 ? l.value : 256) / l.value;
    return 0;
  });
  return groups;
}

// Workgroups of the backward: as many as are resident, and enough that none walks
// more than kRunRows rows.
int64_t backward_blocks(int64_t rows, int width) {
  const int64_t groups = row_groups(width);
  const int64_t most = (rows + groups - 1) / groups;
  const int64_t resident = width > 4096 ? 256 : 512;
  const int64_t runs = (most + kRunRows - 1) / kRunRows;
  const int64_t blocks = runs > resident ? runs : resident;
  return blocks < most ? blocks : most;
}

int check(int64_t rows, int64_t width, int type, int residual_type, float eps, int gate_kind, int act) {
  if (rows < 0) return fail(DPA4K_EINVAL, "residual norm: negative sizes");
  if (width < 1 || width > kMaxWidth) return fail(DPA4K_EINVAL, "residual norm takes 1 to %d channels", kMaxWidth);
  if (!known_type(type)) return fail(DPA4K_EINVAL, "residual norm: unknown type");
  if (residual_type != type && residual_type != DPA4K_TYPE_F32)
    return fail(DPA4K_EINVAL, "residual norm: the residual's type must be the input's or float32");
  if (!(eps > 0.0f) || eps > 3.0e38f) return fail(DPA4K_EINVAL, "residual norm eps must be finite and positive");
  if (gate_kind < kGateNone || gate_kind > kGateRow) return fail(DPA4K_EINVAL, "residual norm: unknown kind of gate");
  if (act < kActNone || act > kActSilu) return fail(DPA4K_EINVAL, "residual norm: unknown gate activation");
  if (rows > (int64_t(1) << 62) / (width * 4)) return fail(DPA4K_EINVAL, "residual norm: size overflows 64 bits");
  if (!grid_fits(rows, 256)) return fail(DPA4K_EINVAL, "residual norm: row count beyond the launch limit");
  return DPA4K_OK;
}

}  // namespace
}  // namespace dpa4k

using namespace dpa4k;

extern "C" int dpa4k_residual_norm_forward(const void* x, const void* residual, const void* gate, const float* post_scale,
                                           const float* residual_scale, const float* pre_scale, void* h, void* y, float* post_rstd,
                                           float* pre_rstd, int64_t rows, int64_t channels, float residual_factor, float eps,
                                           int post_norm, int pre_norm, int gate_kind, int gate_activation, int type,
                                           int residual_type, dpa4k_stream_t stream) {
  clear_error();
  const int status = check(rows, channels, type, residual_type, eps, gate_kind, gate_activation);
  if (status != DPA4K_OK) return status;
  if (rows == 0) return DPA4K_OK;
  if (x == nullptr || residual == nullptr || h == nullptr || (pre_norm && y == nullptr) || (gate_kind != kGateNone && gate == nullptr))
    return fail(DPA4K_EINVAL, "residual norm: null pointer");
  NormCall call{};
  call.x = x, call.residual = residual, call.gate = gate;
  call.post = post_norm ? post_scale : nullptr, call.scale = residual_scale, call.pre = pre_norm ? pre_scale : nullptr;
  call.h = h, call.y = y, call.r = post_rstd, call.q = pre_rstd;
  call.scale_value = residual_factor, call.eps = eps, call.rows = rows, call.width = static_cast<int>(channels);
  call.gate_kind = gate_kind, call.act = gate_activation, call.post_norm = post_norm != 0, call.pre_norm = pre_norm != 0;
  return with_types(type, residual_type, [&](auto t, auto s) {
    return with_layout(call.width, [&](auto l, auto e) {
      typedef Row<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value> Z;
      const int64_t blocks = (rows + Z::kGroups - 1) / Z::kGroups;
      const dim3 grid = launch_grid(blocks, Z::kBlock);
      if (gate_kind == kGateFull)
        residual_norm_forward_kernel<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value, true>
            <<<grid, Z::kBlock, 0, as_stream(stream)>>>(call);
      else
        residual_norm_forward_kernel<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value, false>
            <<<grid, Z::kBlock, 0, as_stream(stream)>>>(call);
      return launched("residual_norm_forward_kernel");
    });
  });
}

extern "C" size_t dpa4k_residual_norm_workspace_size(int64_t rows, int64_t channels) {
  if (rows < 0 || channels < 1 || channels > kMaxWidth || rows > (int64_t(1) << 62) / (channels * 4)) return 0;
  return round_up_256(static_cast<size_t>(backward_blocks(rows, static_cast<int>(channels)) * channels) * 3 * sizeof(float));
}

extern "C" int dpa4k_residual_norm_backward(const void* grad_h, const void* grad_y, const void* x, const void* residual,
                                            const void* gate, const float* post_scale, const float* residual_scale,
                                            const float* pre_scale, const float* post_rstd, const float* pre_rstd, void* grad_x,
                                            void* grad_residual, void* grad_gate, float* grad_post_scale, float* grad_pre_scale,
                                            float* grad_residual_scale, int64_t rows, int64_t channels, float residual_factor,
                                            int post_norm, int pre_norm, int gate_kind, int gate_activation, int type,
                                            int residual_type, void* workspace, size_t workspace_bytes, dpa4k_stream_t stream) {
  clear_error();
  const int status = check(rows, channels, type, residual_type, 1.0f, gate_kind, gate_activation);
  if (status != DPA4K_OK) return status;
  const int width = static_cast<int>(channels);
  const bool sums = grad_post_scale != nullptr || grad_pre_scale != nullptr || grad_residual_scale != nullptr;
  const hipStream_t on = as_stream(stream);
  if (rows == 0) {
    for (float* p : {grad_post_scale, grad_pre_scale, grad_residual_scale}) {
      if (p == nullptr) continue;
      const int cleared = zero_fill(p, static_cast<size_t>(width) * sizeof(float), on);
      if (cleared != DPA4K_OK) return cleared;
    }
    return DPA4K_OK;
  }
  if ((grad_h == nullptr && grad_y == nullptr) || x == nullptr || (post_norm && post_rstd == nullptr) || (gate_kind != kGateNone && gate == nullptr) ||
      (grad_y != nullptr && (!pre_norm || residual == nullptr || pre_rstd == nullptr)))
    return fail(DPA4K_EINVAL, "residual norm: null pointer");
  const int64_t blocks = backward_blocks(rows, width);
  if (sums && (workspace == nullptr || workspace_bytes < dpa4k_residual_norm_workspace_size(rows, channels)))
    return fail(DPA4K_EWORKSPACE, "residual norm: workspace too small");
  NormCall call{};
  call.x = x, call.residual = residual, call.gate = gate;
  call.post = post_norm ? post_scale : nullptr, call.scale = residual_scale, call.pre = pre_norm ? pre_scale : nullptr;
  call.r = const_cast<float*>(post_rstd), call.q = const_cast<float*>(pre_rstd);
  call.dh = grad_h, call.dy = grad_y, call.dx = grad_x, call.dresidual = grad_residual;
  call.dgate = gate_kind == kGateNone ? nullptr : grad_gate;
  call.partial = static_cast<float*>(workspace);
  call.scale_value = residual_factor, call.rows = rows, call.width = width;
  call.gate_kind = gate_kind, call.act = gate_activation, call.post_norm = post_norm != 0, call.pre_norm = pre_norm != 0;
  call.want_sums = sums;
  const int ran = with_types(type, residual_type, [&](auto t, auto s) {
    return with_layout(width, [&](auto l, auto e) {
      typedef Row<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value> Z;
      const dim3 grid = launch_grid(blocks, Z::kBlock);
      if (gate_kind == kGateFull)
        residual_norm_backward_kernel<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value, true>
            <<<grid, Z::kBlock, 0, on>>>(call, blocks);
      else
        residual_norm_backward_kernel<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value, false>
            <<<grid, Z::kBlock, 0, on>>>(call, blocks);
      return launched("residual_norm_backward_kernel");
    });
  });
  if (ran != DPA4K_OK || !sums) return ran;
  column_sums_kernel<<<dim3(blocks_for(width, 32), 3), 256, 0, on>>>(call.partial, blocks, width, grad_post_scale, grad_pre_scale,
                                                                      grad_residual_scale);
  return launched("column_sums_kernel");
}
