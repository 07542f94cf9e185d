// The optimiser step over all tensors of a model (no counterpart in the reference, which has no training):
//
//   grad_norm   norm = sqrt(sum g^2) over every gradient, factor = min(1, max_norm / (norm + 1e-6))
//   adamw_step  g' = g * factor
//               m = m * b1 + g' * (1 - b1),   v = v * b2 + (g' * g') * (1 - b2)
//               p = p * (1 - lr wd) - (m / (sqrt(v) * (1 / sqrt(1 - b2^t)) + eps)) * (lr / (1 - b1^t))
//
// A model of this kind is hundreds of tensors, most of them small, so the work
// is cut into chunks of kChunk elements over all tensors, one workgroup each:
// two launches a step whatever the number of tensors.  A plan (built once on
// the host) lists the tensors and the chunks; the gradients, which move from
// step to step, are passed by value to the first launch, which writes them and
// the step's scalars (bias corrections in 64 bits) into the plan.  With moments
// in 32 bits the step is bound by its streams: 28 bytes per float32 element, 72M
// in 379 us, 5.3 TB/s.  With moments in 8 bits (10 bytes per bfloat16 element) it
// is bound by about 100 vector instructions an element: 72M in 181 us.  The norm
// of 72M bfloat16 gradients takes 31 us, 4.7 TB/s.  For 300 tensors of 1.4M
// parameters the two launches take 6 and 9 us.
//
// Every product and sum of the update is rounded to float32 as written above
// (square root and division are the correctly rounded ones), so a step equals
// the same chain of elementwise operations bit for bit.
//
// Moments in 8 bits: 32 consecutive elements share a power of two, 2^(X - 127),
// kept as the byte X.  X is the largest exponent after the magnitude is rounded
// up to three mantissa bits, so no value of the block overflows and scaling is
// exact.  A code is a float with three mantissa bits in the B binades down from
// there: code c > 0 stands for the float32 with the bits (c + ((X - B + 1) << 3)) << 20,
// with B = 16 and a sign bit for the first moment and B = 32 for the second.
// Since the scale is a power of two, a block's grid stays the same when its
// largest value changes, and an average that stands on it moves only by what
// the step adds.  A nonzero second moment never becomes 0: the next step would
// divide a first moment by eps.
//
// Roundings to codes, and to bfloat16 parameters, are stochastic (16 random
// bits): b2 = 0.999 moves v by a thousandth a step, far below half a step of
// any 8-bit code, and a nearest rounding would freeze the average (a bfloat16
// weight likewise).  The mean of the rounded average then follows the exact
// one.  The bits come from an integer mix of (seed, step, position in the plan).
#include <cmath>
#include <cstring>

#include "common.h"

namespace dpa4k {
namespace {

constexpr int kBlock = 256;
constexpr int kChunk = 4096;           // elements of a workgroup
constexpr int kSpan = 32;              // elements that share a scale
constexpr int kPointers = 440;         // gradients passed by value: kernel arguments below 4 KB

// One tensor of a plan.  The first eight fields are set when the plan is built.
struct alignas(128) Record {
  void* param;
  void* exp_avg;
  void* exp_avg_sq;
  uint8_t* exp_avg_scale;
  uint8_t* exp_avg_sq_scale;
  int64_t count;
  uint64_t position;      // of its first element, every tensor padded to kSpan
  int64_t step;           // steps taken
  const void* grad;       // of this step; null where the tensor takes none
  float factor, decay, step_size, inverse_root;
  uint64_t reserved;
  float* values[2];       // float32 moments to read or write
};
static_assert(sizeof(Record) == 128, "records are 128 bytes");
static_assert(offsetof(Record, step) == DPA4K_ADAMW_STEP_OFFSET, "the header's offset of the step count");

struct Chunk {
  int32_t tensor, index;
};

struct PointerList {
  const void* p[kPointers];
};

__host__ __device__ inline uint32_t mix(uint32_t x) {
  // the constants are odd words of the fractions of sqrt(2) and sqrt(3)
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

// ---------------------------------------------------------------------------
// vectors of E elements
// ---------------------------------------------------------------------------

// Up to 16 bytes at any element alignment: one access.
template <typename T>
constexpr int kWide = 16 / sizeof(T) < 8 ? 16 / sizeof(T) : 8;
template <typename T, int N>
struct vector_of {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(uint16_t bf16) { return __uint_as_float(static_cast<uint32_t>(bf16) << 16); }

// Addresses read from a plan are addresses of global memory, which the compiler
// cannot see: it would use flat accesses, which occupy the LDS path as well.
template <typename T>
using Global = __attribute__((address_space(1))) T;
template <typename T>
__device__ __forceinline__ Global<T>* global(T* p) {
  return (Global<T>*)p;
}

template <int E>
struct Floats {
  float v[E];
};

// Elements [at, at + E) of a stream of `count` as float32, zeros past its end.
template <bool kWhole, int E, typename T>
__device__ __forceinline__ Floats<E> load(const T* __restrict__ p, int64_t at, int64_t count) {
  constexpr int N = E < kWide<T> ? E : kWide<T>;
  Floats<E> out;
  if (kWhole) {
#pragma unroll
    for (int part = 0; part < E / N; ++part) {
      const typename vector_of<T, N>::type raw = *(const Global<typename vector_of<T, N>::type>*)(p + at + part * N);
#pragma unroll
      for (int i = 0; i < N; ++i) out.v[part * N + i] = to_float(raw[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) out.v[i] = at + i < count ? to_float(global(p)[at + i]) : 0.0f;
  }
  return out;
}

template <bool kWhole, int E, typename T>
__device__ __forceinline__ void store(T* __restrict__ p, int64_t at, int64_t count, const T (&value)[E]) {
  constexpr int N = E < kWide<T> ? E : kWide<T>;
  if (kWhole) {
#pragma unroll
    for (int part = 0; part < E / N; ++part) {
      typename vector_of<T, N>::type raw;
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = value[part * N + i];
      *(Global<typename vector_of<T, N>::type>*)(p + at + part * N) = raw;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (at + i < count) global(p)[at + i] = value[i];
  }
}

// ---------------------------------------------------------------------------
// codes of 8 bits
// ---------------------------------------------------------------------------
//
// A lane holds E of the 32 values that share a scale: 8 where the parameters are
// bfloat16 (16 bytes), 4 where they are float32 (8 would leave every store half
// a line: the values of 72M codes took 175 us that way, 123 us with 4).

// The largest `value` of the 32 / E lanes of a block.
template <int E>
__device__ __forceinline__ uint32_t block_max(uint32_t value) {
  const auto with = [&](int other) { value = value > static_cast<uint32_t>(other) ? value : static_cast<uint32_t>(other); };
  with(xor_lane<1>(static_cast<int>(value)));
  with(xor_lane<2>(static_cast<int>(value)));
  if constexpr (E == 4) with(xor_lane<4>(static_cast<int>(value)));
  return value;
}

// A lane's E codes, four to a word.
template <int E>
struct Codes {
  uint32_t word[E / 4];
};
template <int E>
__device__ __forceinline__ Codes<E> load_codes(const void* p, int64_t at) {
  Codes<E> out;
  const Global<uint32_t>* words = global(static_cast<uint32_t*>(const_cast<void*>(p))) + at / 4;
#pragma unroll
  for (int i = 0; i < E / 4; ++i) out.word[i] = words[i];
  return out;
}
template <int E>
__device__ __forceinline__ void store_codes(void* p, int64_t at, const Codes<E>& codes) {
  Global<uint32_t>* words = global(static_cast<uint32_t*>(p)) + at / 4;
#pragma unroll
  for (int i = 0; i < E / 4; ++i) words[i] = codes.word[i];
}

// A signed code has a sign bit and 16 binades, an unsigned one 32.
template <bool kSigned>
constexpr uint32_t kBinades = kSigned ? 16u : 32u;

// What a condition of few lanes guards is skipped by the whole wave where no
// lane has it.
__device__ __forceinline__ bool any_lane(bool condition) { return __builtin_expect(__ballot(condition) != 0, 0); }

// The values of a lane's codes, where the scale is not 255 (then the whole block
// stands for NaN: poison_of).
template <bool kSigned, int E>
__device__ __forceinline__ void decode(const Codes<E>& codes, uint32_t top, float (&value)[E]) {
  const uint32_t low = top - kBinades<kSigned> + 1u;
  uint32_t zeros = 0u;  // a bit for each code of 0 (and perhaps for a 1 above one)
#pragma unroll
  for (int w = 0; w < E / 4; ++w) {
    const uint32_t word = kSigned ? codes.word[w] & 0x7F7F7F7Fu : codes.word[w];
    zeros |= (word - 0x01010101u) & ~word & 0x80808080u;
  }
  uint32_t magnitude[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    magnitude[i] = (__builtin_amdgcn_ubfe(codes.word[i / 4], 8 * (i & 3), kSigned ? 7 : 8) + (low << 3)) << 20;
  if (any_lane(zeros != 0u))
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (__builtin_amdgcn_ubfe(codes.word[i / 4], 8 * (i & 3), kSigned ? 7 : 8) == 0u) magnitude[i] = 0u;
#pragma unroll
  for (int i = 0; i < E; ++i)
    value[i] = __uint_as_float(kSigned ? (codes.word[i / 4] << (24 - 8 * (i & 3)) & 0x80000000u) | magnitude[i] : magnitude[i]);
}

__device__ __forceinline__ float poison_of(uint32_t top) { return top == 255u ? NAN : 0.0f; }

// The shared exponent of a block, and this lane's codes.  A block with an
// infinity, a NaN of either sign, a value above 1.875 2^127 (which three mantissa
// bits round up to infinity) or a second moment below 0 takes X = 255 and stands
// for NaN.  A second moment of -0 has to be given as 0.  `random`: 16 bits a
// value (its lower or upper half), compared with the 20 bits cut off.
template <bool kSigned, int E>
__device__ __forceinline__ Codes<E> encode(const float (&value)[E], const uint32_t (&random)[E], uint32_t& top) {
  const auto half_of = [&](int i) { return kSigned ? random[i] & 0xFFFFu : random[i] >> 16; };
  uint32_t word[E], most = 0u;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    word[i] = kSigned ? __float_as_uint(value[i]) & 0x7FFFFFFFu : __float_as_uint(value[i]);
    most = word[i] > most ? word[i] : most;
  }
  most = block_max<E>(most);
  most = ((most < 0x7F800000u ? most : 0x7F800000u) + 0xFFFFFu) >> 23;
  most = most > kBinades<kSigned> ? most : kBinades<kSigned>;
  top = most < 255u ? most : 255u;
  const uint32_t low = (top - kBinades<kSigned> + 1u) << 3;
  int code[E], least_code = 1;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    code[i] = static_cast<int>((word[i] + (half_of(i) << 4)) >> 20) - static_cast<int>(low);
    least_code = code[i] < least_code ? code[i] : least_code;
  }
  // below the least code (few values are): a first moment goes up to it as often
  // as it is its share of it, a second moment unless it is 0
  if (any_lane(least_code < 1)) {
    const float least = __uint_as_float((low + 1u) << 20);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (code[i] < 1) {
        if (kSigned) code[i] = __uint_as_float(word[i]) > least * (static_cast<float>(half_of(i)) * 1.52587890625e-5f) ? 1 : 0;
        else code[i] = word[i] != 0u ? 1 : 0;
      }
  }
  Codes<E> packed;
#pragma unroll
  for (int w = 0; w < E / 4; ++w) {
    packed.word[w] = 0u;
#pragma unroll
    for (int i = 4 * w; i < 4 * w + 4; ++i) {
      uint32_t byte = static_cast<uint32_t>(code[i]);
      if (kSigned) byte = (byte & 0x7Fu) | (__float_as_uint(value[i]) >> 24 & 0x80u);
      else byte &= 0xFFu;
      packed.word[w] |= byte << (8 * (i & 3));
    }
  }
  return packed;
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------

struct StepScalars {
  double lr, beta1, beta2, weight_decay;
  const float* lr_device;
  const float* factor;
};

// One thread per tensor: its gradient's address and this step's scalars.  A
// factor that is NaN (the norm was not finite) takes no step anywhere.
__global__ __launch_bounds__(kBlock) void adamw_begin_kernel(PointerList grads, Record* __restrict__ records,
                                                             int first, int count, StepScalars s) {
  const int i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= count) return;
  Record& r = records[first + i];
  const float factor = s.factor != nullptr ? *s.factor : 1.0f;
  const void* grad = factor == factor ? grads.p[i] : nullptr;
  r.grad = grad;
  if (grad == nullptr) return;
  const int64_t t = r.step + 1;
  r.step = t;
  const double lr = s.lr_device != nullptr ? static_cast<double>(*s.lr_device) : s.lr;
  r.factor = factor;
  r.decay = static_cast<float>(1.0 - lr * s.weight_decay);
  r.step_size = static_cast<float>(lr / (1.0 - pow(s.beta1, static_cast<double>(t))));
  r.inverse_root = static_cast<float>(1.0 / sqrt(1.0 - pow(s.beta2, static_cast<double>(t))));
}

struct UpdateScalars {
  float beta1, rest1, beta2, rest2, eps;  // rest = 1 - beta
  uint32_t seed_low, seed_high;
};

// The random bits of step t at positions whose upper 32 bits are `high`.
__device__ __forceinline__ uint32_t random_key(const UpdateScalars& s, int64_t t, uint32_t high) {
  return mix(s.seed_low ^ mix(s.seed_high + mix(static_cast<uint32_t>(t) + high * 0x9E3779B1u)));
}

// Elements of a lane's vector.
template <typename P, int kBits>
constexpr int kElements = kBits == 8 && sizeof(P) == 2 ? 8 : 4;

template <typename P, typename G, int kBits, bool kWhole>
__device__ __forceinline__ void adamw_update_chunk(const Record& r, int64_t begin, const UpdateScalars& s) {
  constexpr bool kRandom = kBits == 8 || sizeof(P) == 2;
  constexpr int E = kElements<P, kBits>, K = kChunk / (kBlock * E);
  P* const param = static_cast<P*>(r.param);
  const G* const grad = static_cast<const G*>(r.grad);
  const int64_t count = r.count;
  const int64_t padded = (count + kSpan - 1) / kSpan * kSpan;
  const float factor = r.factor, decay = r.decay, step_size = r.step_size, inverse_root = r.inverse_root;
  Floats<E> p[K], g[K], m[K], v[K];
  Codes<E> m_codes[K], v_codes[K];
  uint32_t m_top[K], v_top[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t at = begin + (k * kBlock + static_cast<int>(threadIdx.x)) * E;
    p[k] = load<kWhole, E>(param, at, count);
    g[k] = load<kWhole, E>(grad, at, count);
    if constexpr (kBits == 32) {
      m[k] = load<kWhole, E>(static_cast<const float*>(r.exp_avg), at, count);
      v[k] = load<kWhole, E>(static_cast<const float*>(r.exp_avg_sq), at, count);
    } else {
      const bool live = kWhole || at < padded;
      m_codes[k] = live ? load_codes<E>(r.exp_avg, at) : Codes<E>{};
      v_codes[k] = live ? load_codes<E>(r.exp_avg_sq, at) : Codes<E>{};
      m_top[k] = live ? global(r.exp_avg_scale)[at / kSpan] : kBinades<true>;
      v_top[k] = live ? global(r.exp_avg_sq_scale)[at / kSpan] : kBinades<false>;
    }
  }
  const uint32_t high = static_cast<uint32_t>((r.position + begin) >> 32);
  const uint32_t key = kRandom ? random_key(s, r.step, high) : 0u;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t at = begin + (k * kBlock + static_cast<int>(threadIdx.x)) * E;
    float new_p[E], new_m[E], new_v[E];
    if constexpr (kBits == 8) {
      decode<true, E>(m_codes[k], m_top[k], m[k].v);
      decode<false, E>(v_codes[k], v_top[k], v[k].v);
    }
    const float m_poison = kBits == 8 ? poison_of(m_top[k]) : 0.0f, v_poison = kBits == 8 ? poison_of(v_top[k]) : 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float scaled = g[k].v[i] * factor;
      new_m[i] = m[k].v[i] * (kBits == 8 ? s.beta1 + m_poison : s.beta1) + scaled * s.rest1;
      new_v[i] = v[k].v[i] * (kBits == 8 ? s.beta2 + v_poison : s.beta2) + (scaled * scaled) * s.rest2;
      new_p[i] = p[k].v[i] * decay - (new_m[i] / (sqrtf(new_v[i]) * inverse_root + s.eps)) * step_size;
    }
    uint32_t bits[E];
    if constexpr (kRandom) {
      const uint64_t position = r.position + at;
      const uint32_t own_high = static_cast<uint32_t>(position >> 32);
      const uint32_t own_key = own_high == high ? key : random_key(s, r.step, own_high);
#pragma unroll
      for (int i = 0; i < E; ++i) bits[i] = mix((static_cast<uint32_t>(position) + i) ^ own_key);
    }
    if constexpr (sizeof(P) == 2) {
      uint32_t word[E], most = 0u;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        word[i] = __float_as_uint(new_p[i]) + (mix(bits[i] + 0x9E3779B1u) & 0xFFFFu);
        const uint32_t magnitude = __float_as_uint(new_p[i]) & 0x7FFFFFFFu;
        most = magnitude > most ? magnitude : most;
      }
      if (any_lane(most >= 0x7F800000u))  // infinities stay, NaN stays NaN (quiet)
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (!__builtin_isfinite(new_p[i]))
            word[i] = __builtin_isnan(new_p[i]) ? __float_as_uint(new_p[i]) | 0x00400000u : __float_as_uint(new_p[i]);
      P rounded[E];
#pragma unroll
      for (int i = 0; i < E; ++i) rounded[i] = static_cast<P>(word[i] >> 16);
      store<kWhole, E>(param, at, count, rounded);
    } else {
      store<kWhole, E>(param, at, count, new_p);
    }
    if constexpr (kBits == 32) {
      store<kWhole, E>(static_cast<float*>(r.exp_avg), at, count, new_m);
      store<kWhole, E>(static_cast<float*>(r.exp_avg_sq), at, count, new_v);
    } else {
      if (!kWhole)
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (at + i >= count) new_m[i] = new_v[i] = 0.0f;  // padding stays 0
      uint32_t top_m, top_v;
      const Codes<E> packed_m = encode<true, E>(new_m, bits, top_m);
      const Codes<E> packed_v = encode<false, E>(new_v, bits, top_v);
      if (kWhole || at < padded) {
        store_codes<E>(r.exp_avg, at, packed_m);
        store_codes<E>(r.exp_avg_sq, at, packed_v);
        if ((threadIdx.x & (kSpan / E - 1)) == 0) {
          global(r.exp_avg_scale)[at / kSpan] = static_cast<uint8_t>(top_m);
          global(r.exp_avg_sq_scale)[at / kSpan] = static_cast<uint8_t>(top_v);
        }
      }
    }
  }
}

template <typename P, typename G, int kBits>
__global__ __launch_bounds__(kBlock) void adamw_update_kernel(const Record* __restrict__ records,
                                                              const Chunk* __restrict__ chunks, int64_t n_chunks,
                                                              UpdateScalars s) {
  const int64_t block = block_index();
  if (block >= n_chunks) return;
  const Chunk chunk = chunks[block];
  const Record& r = records[chunk.tensor];
  if (r.grad == nullptr) return;
  const int64_t begin = static_cast<int64_t>(chunk.index) * kChunk;
  if (r.count - begin >= kChunk) adamw_update_chunk<P, G, kBits, true>(r, begin, s);
  else adamw_update_chunk<P, G, kBits, false>(r, begin, s);
}

// ---------------------------------------------------------------------------
// 8-bit moments as float32 values, and back
// ---------------------------------------------------------------------------

__global__ __launch_bounds__(kBlock) void adamw_values_kernel(PointerList list, Record* __restrict__ records,
                                                              int first, int count, int which) {
  const int i = blockIdx.x * kBlock + threadIdx.x;
  if (i < count) records[first + i].values[which] = static_cast<float*>(const_cast<void*>(list.p[i]));
}

template <bool kRead, bool kWhole>
__device__ __forceinline__ void adamw_codes_chunk(const Record& r, int64_t begin) {
  constexpr int E = 4;
  const int64_t count = r.count;
  const int64_t padded = (count + kSpan - 1) / kSpan * kSpan;
#pragma unroll
  for (int k = 0; k < kChunk / (kBlock * E); ++k) {
    const int64_t at = begin + (k * kBlock + static_cast<int>(threadIdx.x)) * E;
    const bool live = kWhole || at < padded;
    if constexpr (kRead) {
      if (!live) continue;
      const Codes<E> m_codes = load_codes<E>(r.exp_avg, at), v_codes = load_codes<E>(r.exp_avg_sq, at);
      const uint32_t m_top = global(r.exp_avg_scale)[at / kSpan], v_top = global(r.exp_avg_sq_scale)[at / kSpan];
      float m[E], v[E];
      decode<true, E>(m_codes, m_top, m);
      decode<false, E>(v_codes, v_top, v);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        m[i] = m_top == 255u ? NAN : m[i];
        v[i] = v_top == 255u ? NAN : v[i];
      }
      store<kWhole, E>(r.values[0], at, count, m);
      store<kWhole, E>(r.values[1], at, count, v);
    } else {
      // every lane takes part in the exponent of its block
      const Floats<E> m = load<kWhole, E>(r.values[0], at, count);
      Floats<E> v = load<kWhole, E>(r.values[1], at, count);
#pragma unroll
      for (int i = 0; i < E; ++i) v.v[i] += 0.0f;  // -0 becomes 0
      uint32_t half[E], top_m, top_v;
#pragma unroll
      for (int i = 0; i < E; ++i) half[i] = 0x80008000u;
      const Codes<E> packed_m = encode<true, E>(m.v, half, top_m);
      const Codes<E> packed_v = encode<false, E>(v.v, half, top_v);
      if (live) {
        store_codes<E>(r.exp_avg, at, packed_m);
        store_codes<E>(r.exp_avg_sq, at, packed_v);
        if ((threadIdx.x & (kSpan / E - 1)) == 0) {
          global(r.exp_avg_scale)[at / kSpan] = static_cast<uint8_t>(top_m);
          global(r.exp_avg_sq_scale)[at / kSpan] = static_cast<uint8_t>(top_v);
        }
      }
    }
  }
}

// kRead: codes to values.  Otherwise values to the nearest codes.
template <bool kRead>
__global__ __launch_bounds__(kBlock) void adamw_codes_kernel(const Record* __restrict__ records,
                                                             const Chunk* __restrict__ chunks, int64_t n_chunks) {
  const int64_t block = block_index();
  if (block >= n_chunks) return;
  const Chunk chunk = chunks[block];
  const Record& r = records[chunk.tensor];
  const int64_t begin = static_cast<int64_t>(chunk.index) * kChunk;
  if (r.count - begin >= kChunk) adamw_codes_chunk<kRead, true>(r, begin);
  else adamw_codes_chunk<kRead, false>(r, begin);
}

// ---------------------------------------------------------------------------
// gradient norm
// ---------------------------------------------------------------------------
//
// Each launch takes up to kNormTensors gradients by value.  Its workgroups take
// equal runs of chunks; a thread sums squares in 64 bits (the card's float64
// rate hides behind the stream), a workgroup leaves one partial, and a last
// small launch adds all partials in their order.

constexpr int kNormTensors = 180;
constexpr int kNormBlocks = 2048;      // workgroups of one launch
constexpr int kNormChunk = 2048;       // elements

struct NormList {
  const void* p[kNormTensors];
  int64_t count[kNormTensors];         // elements * 2, and 1 for bfloat16
  uint32_t first[kNormTensors + 1];    // chunks before each tensor
};

// The squares of elements [begin, end), over the threads of a workgroup.
template <typename T>
__device__ __forceinline__ double run_squares(const T* __restrict__ p, int64_t begin, int64_t end) {
  constexpr int E = kWide<T>, U = 32 / E;  // 32 elements of a thread in flight
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  int64_t at = begin;
  for (; at + U * kBlock * E <= end; at += U * kBlock * E) {
    Floats<E> g[U];
#pragma unroll
    for (int k = 0; k < U; ++k) g[k] = load<true, E>(p, at + (k * kBlock + static_cast<int>(threadIdx.x)) * E, end);
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i)
        sum[i & 3] = __builtin_fma(static_cast<double>(g[k].v[i]), static_cast<double>(g[k].v[i]), sum[i & 3]);
  }
  // what is left, 8 elements of a thread in flight: places past the end repeat
  // the last one and count as 0, so that no load sits in a branch (one element a
  // thread at a time took as long as the whole of a large tensor)
  for (; at < end; at += 8 * kBlock) {
    float g[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t place = at + k * kBlock + static_cast<int>(threadIdx.x);
      g[k] = to_float(global(p)[place < end ? place : end - 1]);
      if (place >= end) g[k] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k & 3] = __builtin_fma(static_cast<double>(g[k]), static_cast<double>(g[k]), sum[k & 3]);
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__device__ __forceinline__ double block_sum(double value) {
  __shared__ double waves[kBlock / 64];
  value = group_sum<64>(value);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = value;
  __syncthreads();
  double total = waves[0];
#pragma unroll
  for (int w = 1; w < kBlock / 64; ++w) total += waves[w];
  return total;
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(NormList list, int tensors, uint32_t chunks,
                                                           double* __restrict__ partial) {
  const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * blockIdx.x / gridDim.x);
  const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(chunks) * (blockIdx.x + 1) / gridDim.x);
  int low = 0, high = tensors - 1;  // the tensor of chunk `begin`: the last that starts at or before it
  while (low < high) {
    const int middle = (low + high + 1) >> 1;
    if (list.first[middle] <= begin) low = middle;
    else high = middle - 1;
  }
  double sum = 0.0;
  for (uint32_t chunk = begin; chunk < end; ++low) {  // the run's part of one tensor at a time
    const uint32_t first = list.first[low], next = list.first[low + 1];
    const uint32_t last = next < end ? next : end;
    const int64_t count = list.count[low] >> 1;
    const int64_t from = static_cast<int64_t>(chunk - first) * kNormChunk, to = static_cast<int64_t>(last - first) * kNormChunk;
    if (list.count[low] & 1) sum += run_squares(static_cast<const uint16_t*>(list.p[low]), from, to < count ? to : count);
    else sum += run_squares(static_cast<const float*>(list.p[low]), from, to < count ? to : count);
    chunk = last > chunk ? last : chunk;
  }
  const double total = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

__global__ __launch_bounds__(kBlock) void grad_norm_total_kernel(const double* __restrict__ partial, int64_t count,
                                                                 double max_norm, float* __restrict__ norm,
                                                                 float* __restrict__ factor) {
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kBlock) sum += partial[i];
  const double total = sqrt(block_sum(sum));
  if (threadIdx.x != 0) return;
  const float rounded = static_cast<float>(total);
  *norm = rounded;
  const double wanted = max_norm > 0.0 ? max_norm / (total + 1.0e-6) : 1.0;
  *factor = fabsf(rounded) < INFINITY ? static_cast<float>(wanted < 1.0 ? wanted : 1.0) : NAN;
}

int64_t norm_chunks(int64_t count) { return (count + kNormChunk - 1) / kNormChunk; }

// Workgroups of the launch over tensors [first, last), or -1 where a size is out of range.
int64_t norm_blocks(const int64_t* counts, int64_t first, int64_t last, uint32_t* starts) {
  int64_t chunks = 0;
  for (int64_t i = first; i < last; ++i) {
    if (starts != nullptr) starts[i - first] = static_cast<uint32_t>(chunks);
    if (counts[i] < 0 || counts[i] > (int64_t(1) << 44)) return -1;
    chunks += norm_chunks(counts[i]);
  }
  if (starts != nullptr) starts[last - first] = static_cast<uint32_t>(chunks);
  if (chunks > 0x7FFFFFFF) return -1;
  return chunks < kNormBlocks ? chunks : kNormBlocks;
}

// Partials of all launches, or -1 where a size is out of range.
int64_t norm_partials(const int64_t* counts, int64_t n_tensors) {
  int64_t partials = 0;
  for (int64_t first = 0; first < n_tensors; first += kNormTensors) {
    const int64_t last = first + kNormTensors < n_tensors ? first + kNormTensors : n_tensors;
    const int64_t blocks = norm_blocks(counts, first, last, nullptr);
    if (blocks < 0) return -1;
    partials += blocks;
  }
  return partials;
}

size_t partial_bytes(int64_t partials) { return round_up_256(static_cast<size_t>(partials) * sizeof(double)); }

int64_t tensor_chunks(int64_t count) { return (count + kChunk - 1) / kChunk; }

size_t chunk_offset(int64_t n_tensors) { return round_up_256(static_cast<size_t>(n_tensors) * sizeof(Record)); }

// Chunks of a plan, or -1 where a size is out of range.
int64_t plan_chunks(const int64_t* counts, int64_t n_tensors, int64_t stride) {
  if (n_tensors < 0 || n_tensors > 0x7FFFFFFF || (n_tensors > 0 && counts == nullptr)) return -1;
  int64_t chunks = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    const int64_t count = counts[i * stride];
    if (count < 0 || tensor_chunks(count) > 0x7FFFFFFF) return -1;
    chunks += tensor_chunks(count);
  }
  return chunks;
}

constexpr int64_t kStructStride = sizeof(dpa4k_adamw_tensor) / sizeof(int64_t);
static_assert(sizeof(dpa4k_adamw_tensor) == 56, "seven 8-byte fields");

int check_plan(const char* what, const void* plan, int64_t n_tensors, int64_t n_chunks) {
  if (n_tensors < 0 || n_chunks < 0) return fail(DPA4K_EINVAL, "%s: negative sizes", what);
  if (n_tensors > 0x7FFFFFFF || !grid_fits(n_chunks, kBlock)) return fail(DPA4K_EINVAL, "%s: plan exceeds the launch limit", what);
  if (n_tensors > 0 && plan == nullptr) return fail(DPA4K_EINVAL, "%s: null pointer", what);
  return DPA4K_OK;
}

template <typename Launch>
void each_list(const void* const* pointers, int64_t n_tensors, Launch launch) {
  for (int64_t first = 0; first < n_tensors; first += kPointers) {
    const int count = static_cast<int>(n_tensors - first < kPointers ? n_tensors - first : kPointers);
    PointerList list;
    std::memset(&list, 0, sizeof(list));
    std::memcpy(list.p, pointers + first, count * sizeof(void*));
    launch(list, static_cast<int>(first), count);
  }
}

template <bool kRead>
int move_states(const char* what, void* plan, int64_t n_tensors, int64_t n_chunks, const void* const* exp_avgs,
                const void* const* exp_avg_sqs, hipStream_t stream) {
  if (int s = check_plan(what, plan, n_tensors, n_chunks)) return s;
  if (n_chunks == 0) return DPA4K_OK;
  if (exp_avgs == nullptr || exp_avg_sqs == nullptr) return fail(DPA4K_EINVAL, "%s: null pointer", what);
  Record* records = static_cast<Record*>(plan);
  const Chunk* chunks = reinterpret_cast<const Chunk*>(static_cast<char*>(plan) + chunk_offset(n_tensors));
  for (int which = 0; which < 2; ++which)
    each_list(which == 0 ? exp_avgs : exp_avg_sqs, n_tensors, [&](const PointerList& list, int first, int count) {
      adamw_values_kernel<<<blocks_for(count, kBlock), kBlock, 0, stream>>>(list, records, first, count, which);
    });
  adamw_codes_kernel<kRead><<<launch_grid(n_chunks, kBlock), kBlock, 0, stream>>>(records, chunks, n_chunks);
  return launched("adamw_codes_kernel");
}

}  // namespace
}  // namespace dpa4k

using namespace dpa4k;

extern "C" size_t dpa4k_grad_norm_workspace_size(const int64_t* counts, int64_t n_tensors) {
  if (counts == nullptr || n_tensors <= 0) return 0;
  const int64_t partials = norm_partials(counts, n_tensors);
  return partials < 0 ? 0 : partial_bytes(partials);
}

extern "C" int dpa4k_grad_norm(const void* const* grads, const int64_t* counts, const int32_t* types,
                               int64_t n_tensors, double max_norm, float* norm, float* factor, void* workspace,
                               size_t workspace_bytes, dpa4k_stream_t stream_handle) {
  clear_error();
  if (n_tensors < 0) return fail(DPA4K_EINVAL, "gradient norm: negative tensor count");
  if (n_tensors > 0 && (grads == nullptr || counts == nullptr || types == nullptr))
    return fail(DPA4K_EINVAL, "gradient norm: null pointer");
  if (norm == nullptr || factor == nullptr) return fail(DPA4K_EINVAL, "gradient norm: null pointer");
  if (!(max_norm < INFINITY)) return fail(DPA4K_EINVAL, "gradient norm: max_norm must be finite");
  for (int64_t i = 0; i < n_tensors; ++i) {
    if (types[i] != DPA4K_TYPE_F32 && types[i] != DPA4K_TYPE_BF16)
      return fail(DPA4K_EINVAL, "gradient norm: gradient %lld has an unknown type", static_cast<long long>(i));
    if (counts[i] < 0 || counts[i] > (int64_t(1) << 44) || (counts[i] > 0 && grads[i] == nullptr))
      return fail(DPA4K_EINVAL, "gradient norm: gradient %lld has a bad size or pointer", static_cast<long long>(i));
  }
  const int64_t all = norm_partials(counts, n_tensors);
  if (all < 0) return fail(DPA4K_EINVAL, "gradient norm: too many elements");
  const size_t needed = partial_bytes(all);
  if (workspace_bytes < needed || (needed > 0 && workspace == nullptr))
    return fail(DPA4K_EWORKSPACE, "gradient norm: workspace of %zu bytes is smaller than %zu", workspace_bytes, needed);
  hipStream_t stream = as_stream(stream_handle);
  double* partial = static_cast<double*>(workspace);
  int64_t partials = 0;
  for (int64_t first = 0; first < n_tensors; first += kNormTensors) {
    const int64_t last = first + kNormTensors < n_tensors ? first + kNormTensors : n_tensors;
    NormList list;
    std::memset(&list, 0, sizeof(list));
    const int64_t blocks = norm_blocks(counts, first, last, list.first);
    for (int64_t i = first; i < last; ++i) {
      list.p[i - first] = grads[i];
      list.count[i - first] = counts[i] * 2 + (types[i] == DPA4K_TYPE_BF16 ? 1 : 0);
    }
    if (blocks == 0) continue;
    const int tensors = static_cast<int>(last - first);
    grad_norm_kernel<<<static_cast<unsigned int>(blocks), kBlock, 0, stream>>>(list, tensors, list.first[tensors],
                                                                               partial + partials);
    if (int s = launched("grad_norm_kernel")) return s;
    partials += blocks;
  }
  grad_norm_total_kernel<<<1, kBlock, 0, stream>>>(partial, partials, max_norm, norm, factor);
  return launched("grad_norm_total_kernel");
}

extern "C" size_t dpa4k_adamw_plan_size(const int64_t* counts, int64_t n_tensors) {
  const int64_t chunks = plan_chunks(counts, n_tensors, 1);
  if (chunks < 0) return 0;
  return chunk_offset(n_tensors) + round_up_256(static_cast<size_t>(chunks) * sizeof(Chunk));
}

extern "C" int dpa4k_adamw_plan(const dpa4k_adamw_tensor* tensors, int64_t n_tensors, int state_bits,
                                void* plan_host, size_t bytes, int64_t* n_chunks) {
  clear_error();
  if (state_bits != 32 && state_bits != 8) return fail(DPA4K_EINVAL, "AdamW plan: state_bits must be 32 or 8");
  if (n_chunks == nullptr || (n_tensors > 0 && (tensors == nullptr || plan_host == nullptr)))
    return fail(DPA4K_EINVAL, "AdamW plan: null pointer");
  const int64_t chunks = plan_chunks(n_tensors > 0 ? &tensors[0].count : nullptr, n_tensors, kStructStride);
  if (chunks < 0) return fail(DPA4K_EINVAL, "AdamW plan: a size is negative or too large");
  const size_t needed = chunk_offset(n_tensors) + round_up_256(static_cast<size_t>(chunks) * sizeof(Chunk));
  if (bytes < needed) return fail(DPA4K_EWORKSPACE, "AdamW plan: %zu bytes are fewer than %zu", bytes, needed);
  *n_chunks = chunks;
  if (n_tensors == 0) return DPA4K_OK;
  std::memset(plan_host, 0, needed);
  Record* records = static_cast<Record*>(plan_host);
  Chunk* table = reinterpret_cast<Chunk*>(static_cast<char*>(plan_host) + chunk_offset(n_tensors));
  uint64_t position = 0;
  int64_t at = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    const dpa4k_adamw_tensor& t = tensors[i];
    if (t.step < 0) return fail(DPA4K_EINVAL, "AdamW plan: tensor %lld has a negative step", static_cast<long long>(i));
    if (t.count > 0 && (t.param == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr ||
                        (state_bits == 8 && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr))))
      return fail(DPA4K_EINVAL, "AdamW plan: tensor %lld has a null pointer", static_cast<long long>(i));
    Record& r = records[i];
    r.param = t.param;
    r.exp_avg = t.exp_avg;
    r.exp_avg_sq = t.exp_avg_sq;
    r.exp_avg_scale = t.exp_avg_scale;
    r.exp_avg_sq_scale = t.exp_avg_sq_scale;
    r.count = t.count;
    r.position = position;
    r.step = t.step;
    position += static_cast<uint64_t>((t.count + kSpan - 1) / kSpan * kSpan);
    for (int64_t c = 0; c < tensor_chunks(t.count); ++c) table[at++] = {static_cast<int32_t>(i), static_cast<int32_t>(c)};
  }
  return DPA4K_OK;
}

extern "C" int dpa4k_adamw_step(void* plan, int64_t n_tensors, int64_t n_chunks, int state_bits, int param_type,
                                int grad_type, const void* const* grads, double lr, const float* lr_device,
                                double beta1, double beta2, double eps, double weight_decay,
                                const float* grad_factor, uint64_t seed, dpa4k_stream_t stream_handle) {
  clear_error();
  if (int s = check_plan("AdamW step", plan, n_tensors, n_chunks)) return s;
  if (state_bits != 32 && state_bits != 8) return fail(DPA4K_EINVAL, "AdamW step: state_bits must be 32 or 8");
  if ((param_type != DPA4K_TYPE_F32 && param_type != DPA4K_TYPE_BF16) ||
      (grad_type != DPA4K_TYPE_F32 && grad_type != DPA4K_TYPE_BF16))
    return fail(DPA4K_EINVAL, "AdamW step: unknown type");
  if (!(lr >= 0.0 && lr < INFINITY) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) ||
      !(static_cast<float>(eps) > 0.0f && eps < INFINITY) || !(weight_decay >= 0.0 && weight_decay < INFINITY))
    return fail(DPA4K_EINVAL, "AdamW step: lr, betas, eps or weight_decay out of range");
  if (n_tensors == 0) return DPA4K_OK;
  if (grads == nullptr) return fail(DPA4K_EINVAL, "AdamW step: null pointer");
  hipStream_t stream = as_stream(stream_handle);
  Record* records = static_cast<Record*>(plan);
  const Chunk* chunks = reinterpret_cast<const Chunk*>(static_cast<char*>(plan) + chunk_offset(n_tensors));
  const StepScalars begin = {lr, beta1, beta2, weight_decay, lr_device, grad_factor};
  each_list(grads, n_tensors, [&](const PointerList& list, int first, int count) {
    adamw_begin_kernel<<<blocks_for(count, kBlock), kBlock, 0, stream>>>(list, records, first, count, begin);
  });
  if (int s = launched("adamw_begin_kernel")) return s;
  if (n_chunks == 0) return DPA4K_OK;
  const UpdateScalars update = {static_cast<float>(beta1), static_cast<float>(1.0 - beta1), static_cast<float>(beta2),
                                static_cast<float>(1.0 - beta2), static_cast<float>(eps),
                                static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32)};
  const dim3 grid = launch_grid(n_chunks, kBlock);
#define DPA4K_ADAMW(P, G)                                                                               \
  (state_bits == 32 ? adamw_update_kernel<P, G, 32> : adamw_update_kernel<P, G, 8>)<<<grid, kBlock, 0, stream>>>( \
      records, chunks, n_chunks, update)
  if (param_type == DPA4K_TYPE_F32) {
    if (grad_type == DPA4K_TYPE_F32) DPA4K_ADAMW(float, float);
    else DPA4K_ADAMW(float, uint16_t);
  } else {
    if (grad_type == DPA4K_TYPE_F32) DPA4K_ADAMW(uint16_t, float);
    else DPA4K_ADAMW(uint16_t, uint16_t);
  }
#undef DPA4K_ADAMW
  return launched("adamw_update_kernel");
}

extern "C" int dpa4k_adamw_read_states(void* plan, int64_t n_tensors, int64_t n_chunks, float* const* exp_avgs,
                                       float* const* exp_avg_sqs, dpa4k_stream_t stream) {
  clear_error();
  return move_states<true>("AdamW read states", plan, n_tensors, n_chunks,
                           reinterpret_cast<const void* const*>(exp_avgs),
                           reinterpret_cast<const void* const*>(exp_avg_sqs), as_stream(stream));
}

extern "C" int dpa4k_adamw_write_states(void* plan, int64_t n_tensors, int64_t n_chunks, const float* const* exp_avgs,
                                        const float* const* exp_avg_sqs, dpa4k_stream_t stream) {
  clear_error();
  return move_states<false>("AdamW write states", plan, n_tensors, n_chunks,
                            reinterpret_cast<const void* const*>(exp_avgs),
                            reinterpret_cast<const void* const*>(exp_avg_sqs), as_stream(stream));
}
