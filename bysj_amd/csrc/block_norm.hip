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
// E elements each: 8 to 64 lanes of a wave for rows of up to 1,024, a workgroup
// beyond.  h is not kept in 32 bits between the two passes; the backward computes
// it again from the residual, which is as many bytes as reading h, and y and the
// gradients see the unrounded h.
//
// The gradients of post, pre and scale are sums over all rows.  A workgroup walks
// its rows with a column's sum in a register, for at most kRunRows rows (sums in
// 32 bits stay short), and leaves one row of partial sums; a second launch adds
// these in 64 bits in a fixed order.
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
  const float s = logistic(gate);
  if (act == kActSigmoid) {
    slope = s * (1.0f - s);
    return s;
  }
  slope = s * fmaf(gate, 1.0f - s, 1.0f);
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
    const int wave = threadIdx.x / 64;
    if ((threadIdx.x & 63) == 0) words[slot][wave] = value;
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) sum += words[slot][w];
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

// Values of one stream at this lane's columns of `row`.
template <typename T, typename S, typename R, int L, int E>
__device__ __forceinline__ void load_row(const S* __restrict__ p, int64_t row, int lane, int width, int64_t total, bool live,
                                         float (&out)[E]) {
  typedef Row<T, R, L, E> Z;
#pragma unroll
  for (int n = 0; n < Z::N; ++n) {
    const int c = Z::column(n, lane);
    const int64_t at = row * width + c;
    const Pack<S, Z::V> raw = load_pack<S, Z::V>(p + at, live ? width - c : 0, total - at);
#pragma unroll
    for (int j = 0; j < Z::V; ++j) out[n * Z::V + j] = static_cast<float>(raw[j]);
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
    if (c < width) store_pack<S, Z::V>(p + row * width + c, part, width - c);
  }
}

template <typename T, typename R, int L, int E>
__device__ __forceinline__ void load_weight(const float* __restrict__ p, float otherwise, int lane, int width, float (&out)[E]) {
  if (p != nullptr) {
    load_row<T, float, R, L, E>(p, 0, lane, width, width, true, out);
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

template <typename T, typename R, int L, int E>
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
  float x[E], residual[E], act[E], post[E], scale[E], h[E];
  load_row<T, T, R, L, E>(x_at, row, lane, width, total, live, x);
  load_row<T, R, R, L, E>(residual_at, row, lane, width, total, live, residual);
  if (call.gate_kind == kGateFull) {
    load_row<T, T, R, L, E>(gate_at, row, lane, width, total, live, act);
  } else {
    const float one = call.gate_kind == kGateRow && live ? static_cast<float>(gate_at[row]) : 1.0f;
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
  if (call.gate_kind != kGateNone) {
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

// One sum of columns: over the row groups of the workgroup, then to its row of
// partial sums.
template <typename T, typename R, int L, int E>
__device__ __forceinline__ void leave_sums(const float (&sum)[E], float* words, float* __restrict__ to, int lane, int group, int width) {
  typedef Row<T, R, L, E> Z;
  if constexpr (Z::kGroups == 1) {
    store_row<T, float, R, L, E>(to, 0, lane, width, true, sum);
  } else {
    // words[group][E][L]; the first L lanes' worth of threads add the groups in order
#pragma unroll
    for (int i = 0; i < E; ++i) words[(group * E + i) * L + lane] = sum[i];
    __syncthreads();
    for (int at = threadIdx.x; at < E * L; at += Z::kBlock) {
      float all = 0.0f;
      for (int g = 0; g < Z::kGroups; ++g) all += words[g * E * L + at];
      const int i = at / L, l = at % L;
      const int c = Z::column(i / Z::V, l) + i % Z::V;
      if (c < width) to[c] = all;
    }
    __syncthreads();
  }
}

template <typename T, typename R, int L, int E>
__global__ __launch_bounds__((L > 256 ? L : 256)) void residual_norm_backward_kernel(NormCall call, int64_t blocks) {
  typedef Row<T, R, L, E> Z;
  __shared__ float words[3][16];
  __shared__ float column_words[Z::kGroups > 1 ? Z::kBlock * E : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  const int width = call.width;
  const float inverse_width = 1.0f / static_cast<float>(width);
  const int64_t total = call.rows * width;
  const int64_t block = block_index();
  if (block >= blocks) return;
  const T* x_at = static_cast<const T*>(call.x);
  const R* residual_at = static_cast<const R*>(call.residual);
  const T* gate_at = static_cast<const T*>(call.gate);
  float sum_post[E], sum_pre[E], sum_scale[E];
#pragma unroll
  for (int i = 0; i < E; ++i) sum_post[i] = sum_pre[i] = sum_scale[i] = 0.0f;

  for (int64_t first = block * Z::kGroups; first < call.rows; first += blocks * Z::kGroups) {
    const int64_t row = first + group;
    const bool live = row < call.rows;
    float x[E], act[E], slope[E], post[E], scale[E], g[E];
    load_row<T, T, R, L, E>(x_at, row, lane, width, total, live, x);
    if (call.gate_kind == kGateFull) {
      load_row<T, T, R, L, E>(gate_at, row, lane, width, total, live, act);
    } else {
      const float one = call.gate_kind == kGateRow && live ? static_cast<float>(gate_at[row]) : 1.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) act[i] = one;
    }
    if (call.dh != nullptr) {
      load_row<T, R, R, L, E>(static_cast<const R*>(call.dh), row, lane, width, total, live, g);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = 0.0f;
    }
    load_weight<T, R, L, E>(call.post, 1.0f, lane, width, post);
    load_weight<T, R, L, E>(call.scale, call.scale_value, lane, width, scale);
    const float r = call.post_norm && live ? call.r[row] : 1.0f;
    if (call.gate_kind != kGateNone) {
#pragma unroll
      for (int i = 0; i < E; ++i) act[i] = gate_value(act[i], call.act, slope[i]);
    }
    if (call.dy != nullptr) {
      float residual[E], dy[E], pre[E], h[E];
      load_row<T, R, R, L, E>(residual_at, row, lane, width, total, live, residual);
      load_row<T, T, R, L, E>(static_cast<const T*>(call.dy), row, lane, width, total, live, dy);
      load_weight<T, R, L, E>(call.pre, 1.0f, lane, width, pre);
      const float q = live ? call.q[row] : 0.0f;
      residual_sum<E>(x, residual, act, post, scale, r, h);
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        h[i] *= q;
        sum_pre[i] = fmaf(dy[i], h[i], sum_pre[i]);
        dy[i] *= pre[i];
        dot = fmaf(dy[i], h[i], dot);
      }
      dot = row_sum<L>(dot, words, 0) * inverse_width;
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = fmaf(q, fmaf(-h[i], dot, dy[i]), g[i]);
    }
    if (call.dresidual != nullptr) store_row<T, R, R, L, E>(static_cast<R*>(call.dresidual), row, lane, width, live, g);
    // x from here on is x r, the normed row
    float dot = 0.0f, row_gate = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x[i] *= r;
      const float a = x[i] * post[i];
      sum_scale[i] = fmaf(g[i], act[i] * a, sum_scale[i]);
      const float b = g[i] * scale[i];
      if (call.gate_kind != kGateNone) slope[i] *= b * a;   // the gate's gradient
      g[i] = b * act[i];
      sum_post[i] = fmaf(g[i], x[i], sum_post[i]);
      g[i] *= post[i];
      dot = fmaf(g[i], x[i], dot);
    }
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
  const int64_t stride = blocks * width;
  float* to = call.partial + block * width;
  leave_sums<T, R, L, E>(sum_post, column_words, to, lane, group, width);
  leave_sums<T, R, L, E>(sum_pre, column_words, to + stride, lane, group, width);
  leave_sums<T, R, L, E>(sum_scale, column_words, to + 2 * stride, lane, group, width);
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
      residual_norm_forward_kernel<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value>
          <<<launch_grid(blocks, Z::kBlock), Z::kBlock, 0, as_stream(stream)>>>(call);
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
  if (x == nullptr || (post_norm && post_rstd == nullptr) || (gate_kind != kGateNone && gate == nullptr) ||
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
      residual_norm_backward_kernel<typename decltype(t)::type, typename decltype(s)::type, l.value, e.value>
          <<<launch_grid(blocks, Z::kBlock), Z::kBlock, 0, on>>>(call, blocks);
      return launched("residual_norm_backward_kernel");
    });
  });
  if (ran != DPA4K_OK || !sums) return ran;
  column_sums_kernel<<<dim3(blocks_for(width, 32), 3), 256, 0, on>>>(call.partial, blocks, width, grad_post_scale, grad_pre_scale,
                                                                      grad_residual_scale);
  return launched("column_sums_kernel");
}
