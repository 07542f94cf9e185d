// The experts' products, forward and backward, and the sum of a token's slots (no
// counterpart in the reference; a matrix per segment of its CSR contract):
//
//   place p of expert e, row i of its entry:   z[p, i] = W[e] x[entry(p), i]
//   entry(p) = order[p] / k (x by token) or p (x by place)
//   y = z,  or  silu(z[:F]) z[F:]  with the gated SiLU
//   dx[entry] = sum over its places of W[e]^T dz[p],   dW[e] = sum_p dz[p] x[entry(p)]^T
//   out[t, i] = sum_j w[t, j] y[places[t, j], i]
//
// One tiled product serves all three directions; they differ in which of its two
// operands has the summed index contiguous:
//
//            rows of the result     columns           summed over     x or dz / W
//   forward  a segment's rows       outputs           inputs          both contiguous
//   dx       a segment's rows       inputs            outputs         W across
//   dW       outputs                inputs            rows            both across
//
// A workgroup finds its segment by a scan of the offsets, so that nothing waits for
// the host and the calls can be captured.  Tiles go through LDS in slices of 128
// bytes along the summed index (or of as many rows), double-buffered: the next
// slice is on its way from memory while this one is multiplied.  Results are held
// in 32 bits in the matrix units' registers.  A few rows an expert, which the
// matrices' bytes bound, have a kernel that reads each matrix once.
//
// Measured: 32,768 slots through 32 matrices of 1,024 to 2 x 2,048 in bfloat16 (8,192
// tokens, four slots each), forward with the gate 399 us (690 TFLOP/s), dW 393 (700),
// dx 347 (790), with the gate's dz in two parts 684 and 654 (the operations twice),
// where a library's one product of that size reaches 1,090 to 1,300:
// one workgroup fits a CU with its 256 by 256 tile, so nothing multiplies while it
// starts and stores, and unequal segments leave a last round half filled.  786,432
// rows of 64 by 64 in float32: forward 107 us, dW 104, dx 115 (2 to 4 TB/s over rows
// that are gathered or go to slots).  Eight tokens of four slots, which
// name about 21 of the 32 matrices: 26 us, 6.8 TB/s over 176 MB (some of them cached).
#include <climits>
#include <type_traits>

#include "elements.h"

namespace dpa4k {
namespace {

constexpr int kMaxExperts = DPA4K_EXPERTS_MAX;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { kForward = 0, kGated = 1, kInput = 2, kWeight = 3 };
// how pieces are loaded: each through its own address and registers, or straight to
// LDS with ragged last pieces of rows, or without any
enum { kByPiece = 0, kRagged = 1, kWhole = 2 };
constexpr int kMostRun = 8;

struct ProductCall {
  const void* a;           // x (forward), dz (dx, dW)
  const void* a_low;       // dx, dW: what dz has below `a`, or null (two_parts)
  const void* b;           // W (forward, dx), x (dW)
  void* out;               // y, dx by place or by slot, dW
  float* partial;          // dW: [chunks][n_out][k_in], the sums of the cut segments' chunks
  float* before;           // forward, gated: z, or null
  const int64_t* offsets;
  const int64_t* order;    // null: x by place
  int64_t places;
  int experts, k, inner;   // k: slots of a token, which order is divided by
  int k_in, n_out;         // of W[e], n_out before the gate
  int chunk_rows;          // dW: rows that one workgroup takes; longer segments are cut
  int chunks;              // dW: most chunks of all cut segments; 0 if none can be longer
  int by_slot;             // dx: written at order[p] instead of p
  int run;                 // row tiles that one workgroup takes, up to kMostRun
};

// ---------------------------------------------------------------------------
// segments and tiles
// ---------------------------------------------------------------------------

// Rows [begin, end) of segment e; segment `experts` is what lies behind the last.
struct Span {
  int begin, end;
};

__device__ __forceinline__ Span span_of(const ProductCall& call, int e) {
  const int64_t all = call.places;
  int64_t begin = call.offsets[e], end = e < call.experts ? call.offsets[e + 1] : all;
  begin = begin < 0 ? 0 : (begin > all ? all : begin);
  end = end < begin ? begin : (end > all ? all : end);
  return Span{static_cast<int>(begin * call.inner), static_cast<int>(end * call.inner)};
}

// Workgroups go to the 8 dies in turn.  Each die takes groups of `group` neighbouring
// tiles, which share rows and matrices in its cache; the groups are dealt in turn,
// as tiles of long segments and the unused ones at the end would otherwise all
// fall to one die.
__device__ __forceinline__ int tile_of_block(int block, int tiles, int group) {
  const int round = group * static_cast<int>(kXcds);
  if (block >= tiles / round * round) return block;
  const int die = block % static_cast<int>(kXcds), index = block / static_cast<int>(kXcds);
  return (index / group * static_cast<int>(kXcds) + die) * group + index % group;
}

// Tiles of `rows` rows of a segment; `empty`: an empty one has a tile too.  At most
// kMostTiles, which is more than a launch has, so that the sums over 64 segments fit
// 32 bits whatever the offsets (those of a malformed plan may overlap).
constexpr int kMostTiles = 1 << 24;

__device__ __forceinline__ int tiles_of(const Span& span, int rows, bool empty) {
  const int length = span.end - span.begin;
  const int tiles = length > 0 ? (length - 1) / rows + 1 : (empty ? 1 : 0);
  return tiles < kMostTiles ? tiles : kMostTiles;
}

// The segment that tile `tile` of tiles of `rows` rows belongs to, and the tile's
// number in it; false behind the last.  A wave looks at 64 segments at a time.
__device__ __forceinline__ bool find_tile(const ProductCall& call, int segments, int rows, bool empty, int tile, int& segment,
                                          int& number, Span& span) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int first = 0; first < segments; first += 64) {
    const int e = first + lane;
    int count = 0;
    Span mine{0, 0};
    if (e < segments) {
      mine = span_of(call, e);
      count = tiles_of(mine, rows, empty);
    }
    int upto = count;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int other = __shfl_up(upto, step, 64);
      if (lane >= step) upto += other;
    }
    const uint64_t past = __ballot(before + upto > tile);
    if (past != 0) {
      const int found = __builtin_ctzll(past);
      segment = first + found;
      number = tile - before - __shfl(upto - count, found, 64);
      span.begin = __shfl(mine.begin, found, 64);
      span.end = __shfl(mine.end, found, 64);
      segment = __builtin_amdgcn_readfirstlane(segment);
      number = __builtin_amdgcn_readfirstlane(number);
      span.begin = __builtin_amdgcn_readfirstlane(span.begin);
      span.end = __builtin_amdgcn_readfirstlane(span.end);
      return true;
    }
    before += __shfl(upto, 63, 64);
  }
  return false;
}

// dW: chunks of a segment that is cut, 0 for one that a workgroup takes whole.  At most
// the chunks there are, as segments of a malformed plan may overlap.
__device__ __forceinline__ int chunks_of(const ProductCall& call, const Span& span) {
  const int count = tiles_of(span, call.chunk_rows, true);
  return count < 2 ? 0 : (count < call.chunks ? count : call.chunks);
}

// Chunks of the cut segments in front of `segment`, by a wave.
__device__ __forceinline__ int chunks_before(const ProductCall& call, int segment) {
  int sum = 0;
  for (int e = threadIdx.x & 63; e < segment; e += 64) {
    sum += chunks_of(call, span_of(call, e));
    sum = sum < call.chunks ? sum : call.chunks;
  }
  sum = group_sum<64>(sum);
  return __builtin_amdgcn_readfirstlane(sum < call.chunks ? sum : call.chunks);
}

// The cut segment number `number`, the chunks of those in front of it and its own, by a
// wave; false behind the last.
__device__ __forceinline__ bool cut_segment(const ProductCall& call, int number, int& segment, int& before, int& count) {
  const int lane = threadIdx.x & 63;
  before = 0;
  for (int first = 0; first < call.experts; first += 64) {
    const int mine = first + lane < call.experts ? chunks_of(call, span_of(call, first + lane)) : 0;
    const uint64_t cut = __ballot(mine > 0);
    const uint64_t in_front = cut & ((uint64_t(1) << lane) - 1);
    const uint64_t found = __ballot(mine > 0 && __popcll(in_front) == number);
    const int there = found != 0 ? __builtin_ctzll(found) : 64;
    before += group_sum<64>(lane < there ? mine : 0);
    before = before < call.chunks ? before : call.chunks;
    if (found != 0) {
      segment = first + there;
      count = __shfl(mine, there, 64);
      count = count < call.chunks - before ? count : call.chunks - before;
      return true;
    }
    number -= __popcll(cut);
  }
  return false;
}

// The row of x that row `row` of the places is, in two halves, so that a loop can
// start the load of the slot long before it needs the row.
struct PlaceRow {
  int64_t slot;
  int inside;    // the row of the entry; without an order `slot` is the row itself
};

__device__ __forceinline__ PlaceRow place_row(const ProductCall& call, int row) {
  if (call.order == nullptr) return PlaceRow{row, 0};
  if (call.inner == 1) return PlaceRow{call.order[row], 0};
  const int place = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(call.inner));
  return PlaceRow{call.order[place], row - place * call.inner};
}

__device__ __forceinline__ int64_t row_of_x(const ProductCall& call, const PlaceRow& at) {
  if (call.order == nullptr) return at.slot;
  // an order outside the slots reads token 0
  const uint32_t token = static_cast<uint64_t>(at.slot) < static_cast<uint64_t>(call.places)
                             ? static_cast<uint32_t>(at.slot) / static_cast<uint32_t>(call.k) : 0u;
  return static_cast<int64_t>(token) * call.inner + at.inside;
}

// ---------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------
//
// Along: LDS holds [rows][128 bytes of the summed index], piece c of 16 bytes of row
// r at place c ^ (r / 2 mod 8): 16 rows' pieces of one number cover all 64 banks.
// Across: LDS holds [slice rows][columns], with the 64-byte (float32: 128-byte) parts
// of a row exchanged by the row's number, so that the rows that are read together
// lie in different banks; 16-bit operands are read with the transposing LDS load.
// Thread t of a workgroup fills the 16 bytes t, t + threads, ... of a slice in
// order, as loads that go to LDS without registers do; what is exchanged is which
// piece it loads.

template <typename T>
constexpr int kV = 16 / sizeof(T);           // elements of a piece
template <typename T>
constexpr int kSlice = 128 / sizeof(T);      // summed index of a slice

// dz in 16 bits is held in two parts, unit * high + low, as one of them would round
// every product (and overflow float16 where dx and dW do not).  bfloat16: 2^-18 of the
// value is lost.  float16: 2^-24 of it or 2^-25, up to 1.3e8; a unit of 2048 is the most
// that what the high part leaves, half a step of it, fits the low one for.
template <typename T>
constexpr float kPartUnit = std::is_same<T, _Float16>::value ? 2048.0f : 1.0f;

template <typename T>
__device__ __forceinline__ void two_parts(float value, float& high, float& low) {
  high = static_cast<float>(static_cast<T>(value * (1.0f / kPartUnit<T>)));
  low = __builtin_fabsf(high) < INFINITY ? fmaf(-kPartUnit<T>, high, value) : 0.0f;
}

__device__ __forceinline__ int along_byte(int row, int piece) { return row * 128 + ((piece ^ ((row >> 1) & 7)) << 4); }

template <typename T, int COLS>
__device__ __forceinline__ int across_byte(int row, int byte) {
  constexpr int kRow = COLS * static_cast<int>(sizeof(T));
  if constexpr (sizeof(T) == 4) {
    return row * kRow + (byte ^ (((row >> 2) & 1) << 7));
  } else if constexpr (kRow >= 256) {
    return row * kRow + (byte ^ ((row & 3) << 6));
  } else {
    return row * kRow + (byte ^ (((row >> 1) & 1) << 6));
  }
}

// The piece of its row that lies at 16 bytes number `at` of a slice.
template <typename T, int COLS>
__device__ __forceinline__ int across_piece(int at) {
  constexpr int kPerRow = COLS / kV<T>;
  const int row = at / kPerRow;
  return (across_byte<T, COLS>(row, (at % kPerRow) * 16) - row * kPerRow * 16) / 16;
}

// 16 bytes per lane as operands of the matrix unit: 32 rows (or columns) by 16
// (16-bit) or 8 (float32) of the summed index, lane l holding row l mod 32.
template <typename T>
__device__ __forceinline__ f32x16 multiply(const u32x4& a, const u32x4& b, f32x16 sum) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), sum, 0, 0, 0);
    return sum;
  } else if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), sum, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), sum, 0, 0, 0);
  }
}

// Operand fragment `step` of a slice for the 32 rows from `row` on.
template <typename T>
__device__ __forceinline__ u32x4 along_fragment(const char* lds, int row, int step) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const u32x4*>(lds + along_byte(row + (lane & 31), step * 2 + (lane >> 5)));
}

template <typename T, int COLS>
__device__ __forceinline__ u32x4 across_fragment(const char* lds, int column, int step) {
  const int lane = threadIdx.x & 63;
  u32x4 out;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      out[j] = *reinterpret_cast<const uint32_t*>(lds + across_byte<T, COLS>(step * 8 + (lane >> 5) * 4 + j, (column + (lane & 31)) * 4));
  } else {
    // 16 lanes read four rows by 16 columns; lane c of them receives column c
    const int from = column + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = step * 16 + (lane >> 5) * 8 + half * 4 + ((lane >> 2) & 3);
      const s16x4 part = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(lds + across_byte<T, COLS>(row, from * 2)));
      const uint64_t bits = __builtin_bit_cast(uint64_t, part);
      out[half * 2] = static_cast<uint32_t>(bits);
      out[half * 2 + 1] = static_cast<uint32_t>(bits >> 32);
    }
  }
  return out;
}

// 64 lanes' 16 bytes of a buffer view to 1,024 consecutive bytes of LDS from `to` (the
// same in every lane) on; zeros from offsets past the end of the view.
__device__ __forceinline__ void load_to_lds(BufferView view, uint32_t offset, char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(view, (__attribute__((address_space(3))) void*)to, 16, static_cast<int>(offset), 0, 0, 0);
}

// s_waitcnt vmcnt(0), any number of other operations left.
constexpr int kNoLoadsLeft = 0x0f70;

template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* __restrict__ p, int live, int64_t room) {
  const Pack<T, kV<T>> raw = load_pack<T, kV<T>>(p, live, room);
  u32x4 out;
  __builtin_memcpy(&out, &raw, 16);
  return out;
}

// ---------------------------------------------------------------------------
// the tiled product
// ---------------------------------------------------------------------------

// BM by BN results by WM by WN waves.
template <typename T, int MODE, int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int kThreads = WM * WN * 64;
  static constexpr bool kAcrossA = MODE == kWeight, kAcrossB = MODE == kWeight || MODE == kInput;
  static constexpr int kBytesA = BM * 128, kBytesB = BN * 128;   // of a slice
  static constexpr int kPiecesA = kBytesA / 16 / kThreads, kPiecesB = kBytesB / 16 / kThreads;
  static constexpr int kFragmentsM = BM / WM / 32, kFragmentsN = BN / WN / 32;
  static constexpr int kSteps = 4;                               // of 32 bytes a slice
  static_assert(kBytesA % (16 * kThreads) == 0 && kBytesB % (16 * kThreads) == 0, "whole pieces");
};

template <typename T, int MODE, int BM, int BN, int WM, int WN, int FAST, bool RUN, bool TWO>
__global__ __launch_bounds__((WM * WN * 64)) void expert_product_kernel(ProductCall call, int columns, int tiles, int group) {
  typedef Tile<T, MODE, BM, BN, WM, WN> Z;
  constexpr int V = kV<T>, S = kSlice<T>;
  __shared__ __attribute__((aligned(1024))) char lds_a0[Z::kBytesA];
  __shared__ __attribute__((aligned(1024))) char lds_b0[Z::kBytesB];
  __shared__ __attribute__((aligned(1024))) char lds_a1[Z::kBytesA];
  __shared__ __attribute__((aligned(1024))) char lds_b1[Z::kBytesB];
  // dW: the rows of x of the slices around the present one, found by one thread a row
  __shared__ int rows_of_x[MODE == kWeight ? 4 : 1][MODE == kWeight ? S : 1];
  const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;

  const int block = tile_of_block(blockIdx.x, tiles, group);
  const int column_tile = block % columns, rest = block / columns;
  const int tile_rows = RUN ? call.run * BM : BM;
  int segment, number;
  Span span;
  int row_tile = 0, chunk = -1;                          // dW: the chunk of a cut segment
  if constexpr (MODE == kWeight) {
    const int row_tiles = (call.n_out + BM - 1) / BM;
    row_tile = rest % row_tiles;
    if (!find_tile(call, call.experts, call.chunk_rows, true, rest / row_tiles, segment, number, span)) return;
    if (call.chunks > 0 && chunks_of(call, span) > 0) {
      chunk = chunks_before(call, segment) + number;
      if (chunk >= call.chunks) return;                  // of a malformed plan
    }
    span.begin += number * call.chunk_rows;
    if (span.end - span.begin > call.chunk_rows) span.end = span.begin + call.chunk_rows;
  } else {
    const int segments = MODE == kInput && call.by_slot ? call.experts : call.experts + 1;
    if (!find_tile(call, segments, tile_rows, false, rest, segment, number, span)) return;
  }
  const int half = call.n_out / 2;                       // gated: where the second half starts
  const int first_row = MODE == kWeight ? row_tile * BM : span.begin + number * tile_rows;
  const int rows_left = (MODE == kWeight ? call.n_out : span.end) - first_row;
  const int live_rows = rows_left < tile_rows ? rows_left : tile_rows;
  const int first_column = column_tile * (MODE == kGated ? BN / 2 : BN);
  const int width = MODE == kGated ? half : (MODE == kForward ? call.n_out : call.k_in);   // columns of the result
  const int depth = MODE == kWeight ? span.end - span.begin : (MODE == kInput ? call.n_out : call.k_in);

  if (MODE != kWeight && segment == call.experts) {      // rows of no expert: zeros
    constexpr int kTileColumns = MODE == kGated ? BN / 2 : BN;
    T* y = static_cast<T*>(call.out);
    for (int at = thread; at < live_rows * kTileColumns; at += Z::kThreads) {
      const int c = first_column + at % kTileColumns;
      if (c < width) y[static_cast<int64_t>(first_row + at / kTileColumns) * width + c] = static_cast<T>(0.0f);
    }
    return;
  }

  // dx by slot: where the rows go, -1 for a slot that is none; forward, in runs:
  // the rows of x
  constexpr int kRows = RUN ? kMostRun * BM : BM;
  __shared__ int row_words[MODE == kInput || (RUN && MODE != kWeight) ? kRows : 1];
  if constexpr (MODE == kInput) {
    for (int row = thread; call.by_slot && row < live_rows; row += Z::kThreads) {
      const PlaceRow at = place_row(call, first_row + row);
      row_words[row] = static_cast<uint64_t>(at.slot) < static_cast<uint64_t>(call.places)
                           ? static_cast<int>(at.slot) * call.inner + at.inside : -1;
    }
  } else if constexpr (RUN && MODE != kWeight) {
    for (int row = thread; row < live_rows; row += Z::kThreads)
      row_words[row] = static_cast<int>(row_of_x(call, place_row(call, first_row + row)));
    __syncthreads();
  }

  // This thread's pieces of a slice.  FAST: as 32-bit offsets from bases that are the
  // same for the workgroup, kNoRow where there is none; loads past the end of an
  // operand give zeros.  A ragged last piece of a row is the row's last 16 bytes, so
  // that no load leaves its row: along the summed index, what it repeats is shifted
  // out in LDS; across it, its columns of the result are stored a little further left,
  // where its neighbour stores the same.  Otherwise as elements of which some are there.
  const int64_t skipped_a = (MODE == kInput ? first_row : MODE == kWeight ? span.begin : 0) * static_cast<int64_t>(call.n_out);
  const T* a = static_cast<const T*>(call.a) + skipped_a;
  const T* a_low = TWO ? static_cast<const T*>(call.a_low) + skipped_a : a;
  const T* b = static_cast<const T*>(call.b);
  const int64_t inner = call.inner;
  const int64_t rows_x = (call.order != nullptr ? call.places / call.k : call.places) * inner;
  const int ld_a = MODE == kForward || MODE == kGated ? call.k_in : call.n_out;
  const int64_t matrix = static_cast<int64_t>(call.n_out) * call.k_in;
  int64_t elements_a, elements_b;                        // from the bases to the ends
  if constexpr (MODE == kForward || MODE == kGated) {
    elements_a = rows_x * call.k_in;
  } else if constexpr (MODE == kInput) {
    elements_a = (FAST ? static_cast<int64_t>(live_rows) : call.places * inner - first_row) * call.n_out;
  } else {
    elements_a = (FAST ? static_cast<int64_t>(depth) : call.places * inner - span.begin) * call.n_out;
  }
  if constexpr (MODE == kWeight) {
    elements_b = rows_x * call.k_in;
  } else {
    elements_b = (FAST ? 1 : static_cast<int64_t>(call.experts - segment)) * matrix;
    b += segment * matrix;
  }
  // the piece of its row that lies where this thread's 16 bytes go (rows of this
  // thread's other pieces have the same place in the pattern)
  const int along_piece = (thread & 7) ^ ((thread >> 4) & 7);
  typedef typename std::conditional<(FAST != kByPiece), uint32_t, int64_t>::type Offset;
  Offset from_a[Z::kPiecesA], from_b[Z::kPiecesB];       // FAST: bytes, else elements
  int live_a[Z::kPiecesA], live_b[Z::kPiecesB];          // else; along: whether the row is there, across: elements
  constexpr int kUnit = FAST ? static_cast<int>(sizeof(T)) : 1;
  const auto offset_of = [&](bool there, int64_t element) {
    if constexpr (FAST != kByPiece) return there ? static_cast<uint32_t>(element * kUnit) : kNoRow;
    else return element;
  };
  // what a piece with `live` elements left in its row repeats of the one before
  const auto repeated = [&](int live) { return FAST == kRagged && live > 0 && live < V ? V - live : 0; };
  PlaceRow of_places[Z::kPiecesA];                       // all loads before the first use
  if constexpr (!RUN && (MODE == kForward || MODE == kGated)) {
#pragma unroll
    for (int i = 0; i < Z::kPiecesA; ++i) {
      const int row = (thread + i * Z::kThreads) >> 3;
      of_places[i] = place_row(call, first_row + (row < live_rows ? row : 0));
    }
  }
#pragma unroll
  for (int i = 0; i < Z::kPiecesA; ++i) {
    const int at = thread + i * Z::kThreads;
    if constexpr (Z::kAcrossA) {
      const int column = first_row + across_piece<T, BM>(at) * V;
      live_a[i] = call.n_out - column;
      from_a[i] = offset_of(live_a[i] > 0, static_cast<int64_t>(at / (BM / V)) * call.n_out + column - repeated(live_a[i]));
    } else if constexpr (!RUN) {
      const int row = at >> 3;
      live_a[i] = row < live_rows;
      const int64_t of_row = MODE == kInput ? row : row_of_x(call, of_places[i]);
      from_a[i] = offset_of(row < live_rows, of_row * ld_a + along_piece * V);
    }
  }
#pragma unroll
  for (int i = 0; i < Z::kPiecesB; ++i) {
    const int at = thread + i * Z::kThreads;
    if constexpr (MODE == kWeight) {
      live_b[i] = call.k_in - (first_column + across_piece<T, BN>(at) * V);
      from_b[i] = 0;
    } else if constexpr (MODE == kInput) {
      const int column = first_column + across_piece<T, BN>(at) * V;
      live_b[i] = call.k_in - column;
      from_b[i] = offset_of(live_b[i] > 0, static_cast<int64_t>(at / (BN / V)) * call.k_in + column - repeated(live_b[i]));
    } else {
      const int row = at >> 3;
      int output = first_column + row;
      bool there = output < call.n_out;
      if constexpr (MODE == kGated) {                    // 32 gates, their 32 partners, 32 gates ...
        const int column = first_column + (row >> 6) * 32 + (row & 31);
        output = (row & 32) ? half + column : column;
        there = column < half;
      }
      live_b[i] = there;
      from_b[i] = offset_of(there, there ? static_cast<int64_t>(output) * call.k_in + along_piece * V : 0);
    }
  }

  // Slices of the first part of dz come first, those of what it leaves behind them.
  const int slices_of_part = (depth + S - 1) / S;
  const int slices = TWO ? 2 * slices_of_part : slices_of_part;
  const auto is_low = [&](int slice) { return TWO && slice >= slices_of_part; };
  // summed index where a slice starts; past `depth` for slices behind the last
  const auto start_of = [&](int slice) { return (is_low(slice) ? slice - slices_of_part : slice) * S; };

  // Starts the loads of slice `slice` of row tile `tile` of the run.  FAST: straight to LDS, whose 16 bytes of a
  // wave are consecutive; zeros where there is nothing.  Else to registers.
  u32x4 piece_a[FAST ? 1 : Z::kPiecesA], piece_b[FAST ? 1 : Z::kPiecesB];
  const auto fetch = [&](int tile, int slice, char* to_a, char* to_b) {
    const int done = start_of(slice);
    const T* a_here = is_low(slice) ? a_low : a;
    const int along_left = depth - done - along_piece * V;
    // across, the base moves; along, the offset (to before it, in a ragged last piece)
    const int64_t moved_a = Z::kAcrossA ? static_cast<int64_t>(done) * call.n_out : FAST ? 0 : done;
    const int64_t moved_b = MODE == kWeight ? 0 : Z::kAcrossB ? static_cast<int64_t>(done) * call.k_in : FAST ? 0 : done;
    if constexpr (MODE == kWeight) {
#pragma unroll
      for (int i = 0; i < Z::kPiecesB; ++i) {
        const int at = thread + i * Z::kThreads, row = at / (BN / V);
        from_b[i] = offset_of(done + row < depth && live_b[i] > 0, rows_of_x[slice & 3][row] * static_cast<int64_t>(call.k_in) +
                                                                       call.k_in - live_b[i] - repeated(live_b[i]));
      }
    }
    if constexpr (FAST != kByPiece) {
      const BufferView view_a = buffer_view(a_here + moved_a, (elements_a - moved_a) * static_cast<int64_t>(sizeof(T)));
      const BufferView view_b = buffer_view(b + moved_b, (elements_b - moved_b) * static_cast<int64_t>(sizeof(T)));
      // by arithmetic, as the compiler makes branches around two loads of a choice
      const uint32_t past = static_cast<uint32_t>(along_left - 1) & kNoRow;
      const uint32_t further = static_cast<uint32_t>((done - repeated(along_left)) * kUnit);
      if constexpr (RUN && !Z::kAcrossA) {
#pragma unroll
        for (int i = 0; i < Z::kPiecesA; ++i) {
          const int row = tile * BM + ((thread + i * Z::kThreads) >> 3);
          int of_row = row;
          if constexpr (MODE != kInput) of_row = row_words[row < live_rows ? row : 0];
          from_a[i] = offset_of(row < live_rows, static_cast<int64_t>(of_row) * ld_a + along_piece * V);
        }
      }
#pragma unroll
      for (int i = 0; i < Z::kPiecesA; ++i)
        load_to_lds(view_a, Z::kAcrossA ? from_a[i] : (from_a[i] + further) | past, to_a + (wave * 64 + i * Z::kThreads) * 16);
#pragma unroll
      for (int i = 0; i < Z::kPiecesB; ++i)
        load_to_lds(view_b, Z::kAcrossB ? from_b[i] : (from_b[i] + further) | past, to_b + (wave * 64 + i * Z::kThreads) * 16);
    } else {
#pragma unroll
      for (int i = 0; i < Z::kPiecesA; ++i) {
        const bool there = Z::kAcrossA ? done + (thread + i * Z::kThreads) / (BM / V) < depth : live_a[i] != 0;
        const int left = there ? (Z::kAcrossA ? live_a[i] : along_left) : 0;
        piece_a[i] = load_piece<T>(a_here + from_a[i] + moved_a, left, elements_a - from_a[i] - moved_a);
      }
#pragma unroll
      for (int i = 0; i < Z::kPiecesB; ++i) {
        const bool there = Z::kAcrossB ? done + (thread + i * Z::kThreads) / (BN / V) < depth : live_b[i] != 0;
        const int left = there ? (Z::kAcrossB ? live_b[i] : along_left) : 0;
        piece_b[i] = load_piece<T>(b + from_b[i] + moved_b, left, elements_b - from_b[i] - moved_b);
      }
    }
  };
  // The slice that was fetched is in LDS behind the next barrier.
  const auto land = [&](int slice, char* to_a, char* to_b) {
    if constexpr (FAST != kByPiece) {
      __builtin_amdgcn_s_waitcnt(kNoLoadsLeft);
      const int repeats = repeated(depth - start_of(slice) - along_piece * V);
      if (MODE != kWeight && repeats > 0) {
        const int words = repeats * static_cast<int>(sizeof(T)) / 4;
        const auto align = [&](char* piece) {
          u32x4 w = *reinterpret_cast<u32x4*>(piece);
          if (words & 1) w = u32x4{w[1], w[2], w[3], 0u};
          if (words & 2) w = u32x4{w[2], w[3], 0u, 0u};
          *reinterpret_cast<u32x4*>(piece) = w;
        };
        if constexpr (!Z::kAcrossA) {
#pragma unroll
          for (int i = 0; i < Z::kPiecesA; ++i) align(to_a + (thread + i * Z::kThreads) * 16);
        }
        if constexpr (!Z::kAcrossB) {
#pragma unroll
          for (int i = 0; i < Z::kPiecesB; ++i) align(to_b + (thread + i * Z::kThreads) * 16);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < Z::kPiecesA; ++i) *reinterpret_cast<u32x4*>(to_a + (thread + i * Z::kThreads) * 16) = piece_a[i];
#pragma unroll
      for (int i = 0; i < Z::kPiecesB; ++i) *reinterpret_cast<u32x4*>(to_b + (thread + i * Z::kThreads) * 16) = piece_b[i];
    }
  };

  f32x16 sum[Z::kFragmentsM][Z::kFragmentsN];
  // Float32: sums in two levels, 512 products (256 additions, the matrix unit takes
  // two at a time) and their sums, as additions of one size do not average their
  // roundings out (4,096 inputs: 4.1e-7 off instead of 1.1e-6; 64 more registers, 4%
  // slower at 8,192 slots of 1,024 to 2 x 2,048).  16-bit operands go 16 products an
  // addition and end in 16 bits.
  constexpr bool kFolds = sizeof(T) == 4 && !RUN;   // runs are of short sums
  constexpr int kFoldSlices = 16;
  f32x16 folded[kFolds ? Z::kFragmentsM : 1][kFolds ? Z::kFragmentsN : 1];
  const auto fold = [&] {
#pragma unroll
    for (int m = 0; m < Z::kFragmentsM; ++m)
#pragma unroll
      for (int n = 0; n < Z::kFragmentsN; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          folded[m][n][i] += sum[m][n][i];
          sum[m][n][i] = 0.0f;
        }
  };
  // The first part of dz comes in units of kPartUnit.
  const auto raise = [&](int slice) {
    if (!TWO || kPartUnit<T> == 1.0f || slice != slices_of_part) return;
#pragma unroll
    for (int m = 0; m < Z::kFragmentsM; ++m)
#pragma unroll
      for (int n = 0; n < Z::kFragmentsN; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[m][n][i] *= kPartUnit<T>;
  };
  const auto clear = [&] {
#pragma unroll
    for (int m = 0; m < Z::kFragmentsM; ++m)
#pragma unroll
      for (int n = 0; n < Z::kFragmentsN; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[m][n][i] = 0.0f;
  };

  // Slice s is multiplied from one half of LDS while s + 1 is on its way to the other;
  // inside a slice, the operands of the next step are read while one step's
  // products run.
  const int wave_row = (wave / WN) * (BM / WM), wave_column = (wave % WN) * (BN / WN);
  u32x4 fa[2][Z::kFragmentsM], fb[2][Z::kFragmentsN];
  const auto read = [&](const char* at_a, const char* at_b, int step, u32x4 (&a_to)[Z::kFragmentsM], u32x4 (&b_to)[Z::kFragmentsN]) {
#pragma unroll
    for (int n = 0; n < Z::kFragmentsN; ++n) {
      if constexpr (Z::kAcrossB) b_to[n] = across_fragment<T, BN>(at_b, wave_column + n * 32, step);
      else b_to[n] = along_fragment<T>(at_b, wave_column + n * 32, step);
    }
#pragma unroll
    for (int m = 0; m < Z::kFragmentsM; ++m) {
      if constexpr (Z::kAcrossA) a_to[m] = across_fragment<T, BM>(at_a, wave_row + m * 32, step);
      else a_to[m] = along_fragment<T>(at_a, wave_row + m * 32, step);
    }
  };
  PlaceRow ahead{0, 0};                                  // dW: of the slice behind the next two
  const auto look_ahead = [&](int slice) {
    const int at = start_of(slice) + thread;
    if (MODE == kWeight && thread < S && at < depth) ahead = place_row(call, span.begin + at);
  };
  if constexpr (MODE == kWeight) {
    for (int row = thread; row < 2 * S; row += Z::kThreads) {
      const int at = start_of(row / S) + row % S;
      if (at < depth) rows_of_x[row / S][row % S] = static_cast<int>(row_of_x(call, place_row(call, span.begin + at)));
    }
    look_ahead(2);
    __syncthreads();
  }
  if (slices > 0) {
    fetch(0, 0, lds_a0, lds_b0);
    land(0, lds_a0, lds_b0);
  }
  __syncthreads();
  if (slices > 0) {
    fetch(0, 1, lds_a1, lds_b1);
    read(lds_a0, lds_b0, 0, fa[0], fb[0]);
  }
  // The half at `at` is read for the last time in front of the third step's products;
  // behind them every wave has read it and the next slice has landed, so that the
  // last step's products hide the next slice's first reads.
  // `slice` is multiplied, `landing` lands in the other half, `coming` of `tile` starts.
  const auto turn = [&](int slice, int landing, int tile, int coming, char* at_a, char* at_b, char* next_a, char* next_b) {
#pragma unroll
    for (int step = 0; step < Z::kSteps; ++step) {
      const int to = (step + 1) & 1;
      if (step + 1 < Z::kSteps) read(at_a, at_b, step + 1, fa[to], fb[to]);
      else read(next_a, next_b, 0, fa[to], fb[to]);
      __builtin_amdgcn_sched_barrier(0);   // loads and reads start here, not where their values are used
#pragma unroll
      for (int m = 0; m < Z::kFragmentsM; ++m)
#pragma unroll
        for (int n = 0; n < Z::kFragmentsN; ++n) {
          // gated: rows of the result are the matrix unit's rows, else its columns
          if constexpr (MODE == kGated) sum[m][n] = multiply<T>(fa[step & 1][m], fb[step & 1][n], sum[m][n]);
          else sum[m][n] = multiply<T>(fb[step & 1][n], fa[step & 1][m], sum[m][n]);
        }
      __builtin_amdgcn_sched_barrier(0);
      if (step == Z::kSteps - 2) {
        land(landing, next_a, next_b);
        if (MODE == kWeight && thread < S) rows_of_x[(slice + 2) & 3][thread] = static_cast<int>(row_of_x(call, ahead));
        __syncthreads();
        fetch(tile, coming, at_a, at_b);
        look_ahead(slice + 3);
      }
    }
  };
  // Register i of a lane is row 8 (i / 4) + 4 (lane / 32) + i mod 4 and column lane mod 32
  // of the matrix unit's result.  Its rows are the columns here: four values are
  // stored at once and a lane has few rows to find (dx of 32,768 rows, 2 x 2,048 to
  // 1,024 in bfloat16, 378 -> 354 us).  Gated, its rows are the
  // rows, so that z is stored in whole lines of 128 bytes (516 -> 458 us forward), past
  // the caches, which its 537 MB would empty of rows and matrices (forward alone 391 ->
  // 371 us, the gate's backward behind it 189 -> 164; no change where z fits them).
  const bool partial = MODE == kWeight && chunk >= 0;
  const auto shifted = [&](int index, int size) { return FAST == kRagged && index >= size / V * V ? (V - size % V) % V : 0; };
  const auto store = [&](int tile) {
    const int above = tile * BM;                         // rows of the run above this tile
    if constexpr (MODE == kGated) {
#pragma unroll
      for (int m = 0; m < Z::kFragmentsM; ++m) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = above + wave_row + m * 32 + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
          if (row >= live_rows) continue;
          const int64_t out_row = first_row + row;
#pragma unroll
          for (int n = 0; n < Z::kFragmentsN; n += 2) {
            const int column = first_column + (wave_column >> 1) + (n / 2) * 32 + (lane & 31);
            if (column >= half) continue;
            const float gate = sum[m][n][i], up = sum[m][n + 1][i];
            static_cast<T*>(call.out)[out_row * half + column] = static_cast<T>(gate * logistic(gate) * up);
            if (call.before != nullptr) {
              float* z = call.before + out_row * call.n_out;
              __builtin_nontemporal_store(gate, z + column);
              __builtin_nontemporal_store(up, z + half + column);
            }
          }
        }
      }
      return;
    }
#pragma unroll
    for (int m = 0; m < Z::kFragmentsM; ++m) {
      int row = above + wave_row + m * 32 + (lane & 31);
      if (Z::kAcrossA) row -= shifted(first_row + row, call.n_out);
      if (row >= live_rows) continue;
      int64_t out_row = first_row + row;
      if constexpr (MODE == kInput) {
        if (call.by_slot) out_row = row_words[row];
        if (out_row < 0) continue;
      } else if constexpr (MODE == kWeight) {
        out_row += static_cast<int64_t>(partial ? chunk : segment) * call.n_out;
      }
#pragma unroll
      for (int n = 0; n < Z::kFragmentsN; ++n) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int inside = 8 * g + 4 * (lane >> 5);
          int column = first_column + wave_column + n * 32 + inside;
          if (Z::kAcrossB) column -= shifted(column, call.k_in);
          if (column >= width) continue;
          const int64_t at = out_row * width + column;
          float four[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) four[i] = sum[m][n][4 * g + i];
          if (partial) store_pack<false, float, 4>(call.partial + at, four, width - column);
          else if (MODE == kInput && call.by_slot) store_pack<false, float, 4>(static_cast<float*>(call.out) + at, four, width - column);
          else store_pack<false, T, 4>(static_cast<T*>(call.out) + at, four, width - column);
        }
      }
    }
  };

  // the two halves by name: the compiler then sees that reads of one need not wait
  // for loads to the other
  if constexpr (RUN) {
    // every tile takes an even number of slices, so that the halves do not change
    // places: a last odd one is followed by zeros
    const int padded = slices + (slices & 1);
    for (int tile = 0; tile * BM < live_rows; ++tile) {
      clear();
      for (int slice = 0; slice < padded; slice += 2) {
        const bool wraps = slice + 2 >= padded;
        const int coming = wraps ? 0 : slice + 2;
        raise(slice);
        turn(slice, slice + 1, wraps ? tile + 1 : tile, coming, lds_a0, lds_b0, lds_a1, lds_b1);
        raise(slice + 1);
        turn(slice + 1, coming, wraps ? tile + 1 : tile, coming + 1, lds_a1, lds_b1, lds_a0, lds_b0);
      }
      store(tile);
    }
  } else {
    clear();
    if constexpr (kFolds) {
#pragma unroll
      for (int m = 0; m < Z::kFragmentsM; ++m)
#pragma unroll
        for (int n = 0; n < Z::kFragmentsN; ++n) folded[m][n] = sum[m][n];
    }
    int slice = 0;
    for (; slice + 1 < slices; slice += 2) {
      raise(slice);
      turn(slice, slice + 1, 0, slice + 2, lds_a0, lds_b0, lds_a1, lds_b1);
      raise(slice + 1);
      turn(slice + 1, slice + 2, 0, slice + 3, lds_a1, lds_b1, lds_a0, lds_b0);
      if constexpr (kFolds) {
        if (slice % kFoldSlices == kFoldSlices - 2) fold();
      }
    }
    if (slice < slices) turn(slice, slice + 1, 0, slice + 2, lds_a0, lds_b0, lds_a1, lds_b1);
    if constexpr (kFolds) {
      fold();
#pragma unroll
      for (int m = 0; m < Z::kFragmentsM; ++m)
#pragma unroll
        for (int n = 0; n < Z::kFragmentsN; ++n) sum[m][n] = folded[m][n];
    }
    store(0);
  }
  __builtin_amdgcn_s_waitcnt(kNoLoadsLeft);              // the workgroup's LDS is not given away while loads to it are under way
}

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------

// Forward for a few rows an expert, as when single tokens are served: bound by reading
// the matrices once.  A workgroup takes 16 rows and 64 rows of W (gated: 32 gates
// and their partners); its four waves take every fourth 64 bytes of the summed index,
// each lane 16 of them, straight into the operands of the matrix unit, and add up
// in LDS.  WHOLE: rows of whole 16-byte pieces.
typedef float f32x4m __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ f32x4m multiply16(const u32x4& a, const u32x4& b, f32x4m sum) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), sum, 0, 0, 0);
    return sum;
  } else if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), sum, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), sum, 0, 0, 0);
  }
}

template <typename T, bool GATED, bool WHOLE>
__global__ __launch_bounds__(256) void expert_few_rows_kernel(ProductCall call, int columns) {
  constexpr int V = kV<T>, kRows = 16, kColumns = 64, kGroups = kColumns / 16, kStep = 4 * V, kAhead = 4;
  __shared__ float words[4][kRows][kColumns + 4];
  const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
  const int column_tile = static_cast<int>(blockIdx.x) % columns;
  int segment, number;
  Span span;
  if (!find_tile(call, call.experts + 1, kRows, false, static_cast<int>(blockIdx.x) / columns, segment, number, span)) return;
  const int half = call.n_out / 2;
  const int width = GATED ? half : call.n_out;
  constexpr int kOut = GATED ? kColumns / 2 : kColumns;
  const int first_row = span.begin + number * kRows, first_column = column_tile * kOut;
  const int live_rows = span.end - first_row < kRows ? span.end - first_row : kRows;
  T* y = static_cast<T*>(call.out);
  if (segment == call.experts) {
    for (int at = thread; at < live_rows * kOut; at += 256) {
      const int c = first_column + at % kOut;
      if (c < width) y[static_cast<int64_t>(first_row + at / kOut) * width + c] = static_cast<T>(0.0f);
    }
    return;
  }
  // lane l: row (of x and of W) l mod 16, piece l / 16 of a step
  const int piece = (lane >> 4) * V;
  const T* x = static_cast<const T*>(call.a);
  const T* w = static_cast<const T*>(call.b);
  const int64_t end_x = (call.order != nullptr ? call.places / call.k : call.places) * static_cast<int64_t>(call.inner) * call.k_in;
  const int64_t end_w = static_cast<int64_t>(call.experts) * call.n_out * call.k_in;
  const bool row_there = (lane & 15) < live_rows;
  const int64_t from_x = row_of_x(call, place_row(call, first_row + (row_there ? lane & 15 : 0))) * call.k_in;
  int64_t from_w[kGroups];
  bool there[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    int output = first_column + g * 16 + (lane & 15);
    there[g] = output < width;
    if constexpr (GATED) {
      output = first_column + (g & 1) * 16 + (lane & 15);
      there[g] = output < half;
      if (g >= 2) output += half;
    }
    from_w[g] = (static_cast<int64_t>(segment) * call.n_out + (there[g] ? output : 0)) * call.k_in;
  }
  f32x4m sum[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) sum[g] = f32x4m{0.0f, 0.0f, 0.0f, 0.0f};
  // Register i of a lane: row 4 (lane / 16) + i, column lane mod 16.  float32: sums in two
  // levels, as in tiles, of 512 products of a wave and these in LDS (65,536 inputs of one
  // size: 2e-4 off in one level; 32 rows, 32 experts, 1,024 to 2 x 2,048: 114 -> 118 us, with
  // 16 more registers in place of LDS 128).
  constexpr bool kFolds = sizeof(T) == 4;
  constexpr int kFoldRounds = 512 / (kAhead * kStep);
  const auto word = [&](int g, int i) -> float& { return words[wave][4 * (lane >> 4) + i][g * 16 + (lane & 15)]; };
  if constexpr (kFolds) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) word(g, i) = 0.0f;
  }
  const auto fold = [&] {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        word(g, i) = kFolds ? word(g, i) + sum[g][i] : sum[g][i];
        sum[g][i] = 0.0f;
      }
    }
  };
  const auto load = [&](const T* p, int64_t from, int64_t end, int k, bool is_there) {
    const int left = is_there ? call.k_in - k : 0;
    if constexpr (WHOLE) {
      const Pack<T, V> raw = *reinterpret_cast<const Pack<T, V>*>(p + from + (left > 0 ? k : 0));
      u32x4 out;
      __builtin_memcpy(&out, &raw, 16);
#pragma unroll
      for (int d = 0; d < 4; ++d) out[d] = left > 0 ? out[d] : 0u;
      return out;
    } else {
      return load_piece<T>(p + from + k, left, end - from - k);
    }
  };
  const int steps = (call.k_in + kStep - 1) / kStep;
  const int fold_steps = kFolds ? 4 * kAhead * kFoldRounds : steps;
  for (int from = wave; from < steps; from += fold_steps) {
    const int upto = from + fold_steps < steps ? from + fold_steps : steps;
    for (int first = from; first < upto; first += 4 * kAhead) {
      u32x4 px[kAhead], pw[kAhead][kGroups];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = (first + 4 * i) * kStep + piece;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) pw[i][g] = load(w, from_w[g], end_w, k, there[g]);
        px[i] = load(x, from_x, end_x, k, row_there);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int g = 0; g < kGroups; ++g) sum[g] = multiply16<T>(px[i], pw[i][g], sum[g]);
    }
    if constexpr (kFolds) fold();
  }
  if constexpr (!kFolds) fold();
  __syncthreads();
  for (int at = thread; at < live_rows * kOut; at += 256) {
    const int row = at / kOut, c = at % kOut, column = first_column + c;
    if (column >= width) continue;
    const auto total = [&](int place) {
      return (words[0][row][place] + words[1][row][place]) + (words[2][row][place] + words[3][row][place]);
    };
    const int64_t out_row = first_row + row;
    if constexpr (GATED) {
      const float gate = total(c), up = total(c + 32);
      y[out_row * half + column] = static_cast<T>(gate * logistic(gate) * up);
      if (call.before != nullptr) {
        call.before[out_row * call.n_out + column] = gate;
        call.before[out_row * call.n_out + half + column] = up;
      }
    } else {
      y[out_row * width + column] = static_cast<T>(total(c));
    }
  }
}

template <typename T, bool GATED>
int run_few_rows(const ProductCall& call, hipStream_t stream) {
  const int width = GATED ? call.n_out / 2 : call.n_out;
  const int64_t columns = (width + (GATED ? 31 : 63)) / (GATED ? 32 : 64);
  const int64_t tiles = columns * (call.places * call.inner / 16 + call.experts + 1);
  if (tiles > row_block_limit(256)) return fail(DPA4K_EINVAL, "expert linear: more tiles than a launch takes");
  const unsigned int grid = static_cast<unsigned int>(tiles);
  if (call.k_in % kV<T> == 0)
    expert_few_rows_kernel<T, GATED, true><<<grid, 256, 0, stream>>>(call, static_cast<int>(columns));
  else
    expert_few_rows_kernel<T, GATED, false><<<grid, 256, 0, stream>>>(call, static_cast<int>(columns));
  return launched("expert_few_rows_kernel");
}

// dW[e] of the cut segments: the sum of their chunks' partial sums, in order, in 64 bits.
template <typename T>
__global__ __launch_bounds__(256) void weight_sum_kernel(ProductCall call, int blocks) {
  int e, before, count;
  if (!cut_segment(call, blockIdx.x / blocks, e, before, count)) return;
  const int64_t size = static_cast<int64_t>(call.n_out) * call.k_in;
  const float* from = call.partial + before * size;
  T* out = static_cast<T*>(call.out) + e * size;
  // 32 elements at a time, eight threads each
  __shared__ double words[8][32];
  const int part = threadIdx.x / 32, element = threadIdx.x % 32;
  for (int64_t first = static_cast<int64_t>(blockIdx.x % blocks) * 32; first < size; first += static_cast<int64_t>(blocks) * 32) {
    const int64_t at = first + element;
    double sum = 0.0;
    if (at < size) {
#pragma unroll 8
      for (int c = part; c < count; c += 8) sum += static_cast<double>(from[c * size + at]);
    }
    words[part][element] = sum;
    __syncthreads();
    if (part == 0 && at < size) {
#pragma unroll
      for (int p = 1; p < 8; ++p) sum += words[p][element];
      out[at] = static_cast<T>(sum);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// elementwise parts
// ---------------------------------------------------------------------------

// dz of the gated SiLU; 16 bytes of dy a thread (32,768 rows of 2,048 in bfloat16: 1.2 GB
// in 207 us, 5.8 TB/s).  z comes in 32 bits and dz goes to the products in two parts of
// 16 bits: with one, the gradients were 1.4 times as far from their exact values as
// one rounding puts them, and with z rounded as well 1.8 times.
template <typename T>
__global__ __launch_bounds__(256) void gate_backward_kernel(const T* __restrict__ dy, const float* __restrict__ z, T* __restrict__ dz,
                                                            T* __restrict__ dz_low, int64_t rows, int half) {
  constexpr int V = kV<T>;
  const int pieces = (half + V - 1) / V;
  const bool short_ = rows * pieces <= UINT32_MAX;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < rows * pieces; at += stride) {
    int64_t row, piece;
    split_piece(at, pieces, short_, row, piece);
    const int column = static_cast<int>(piece) * V;
    const int live = half - column;
    const float* gates = z + row * 2 * half + column;
    const int64_t room = (rows - row) * half - column, room_z = (rows - row) * 2 * half - column;
    const Pack<T, V> grad = load_pack<T, V>(dy + row * half + column, live, room);
    const Pack<float, V> gate = load_pack<float, V>(gates, live, room_z);
    const Pack<float, V> up = load_pack<float, V>(gates + half, live, room_z - half);
    float of_gate[V], of_up[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float g = gate[j], d = static_cast<float>(grad[j]);
      float other;
      const float s = logistic(g, other);
      of_gate[j] = d * up[j] * (s * fmaf(g, other, 1.0f));
      of_up[j] = d * (g * s);
    }
    const int64_t to = row * 2 * half + column;
    if constexpr (sizeof(T) == 2) {
      float low_gate[V], low_up[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        two_parts<T>(of_gate[j], of_gate[j], low_gate[j]);
        two_parts<T>(of_up[j], of_up[j], low_up[j]);
      }
      store_pack<false, T, V>(dz_low + to, low_gate, live);
      store_pack<false, T, V>(dz_low + to + half, low_up, live);
    }
    store_pack<false, T, V>(dz + to, of_gate, live);
    store_pack<false, T, V>(dz + to + half, of_up, live);
  }
}

// dx[t] = the sum over the token's slots that have a place, in slot order (8,192
// tokens of 1,024, four slots each, 151 MB: 25 us, 6.0 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void slot_sum_kernel(const float* __restrict__ by_slot, const int64_t* __restrict__ places,
                                                       T* __restrict__ dx, int64_t tokens, int k, int64_t size, int64_t limit) {
  constexpr int V = kV<T>;
  const int64_t pieces = (size + V - 1) / V;
  const bool short_ = tokens * pieces <= UINT32_MAX;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < tokens * pieces; at += stride) {
    int64_t token, piece;
    split_piece(at, pieces, short_, token, piece);
    const int64_t first = piece * V;
    const int live = static_cast<int>(size - first < V ? size - first : V);
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    for (int j = 0; j < k; ++j) {
      const int64_t slot = token * k + j;
      if (static_cast<uint64_t>(places[slot]) >= static_cast<uint64_t>(limit)) continue;
      const Pack<float, V> part = load_pack<float, V>(by_slot + slot * size + first, live, (tokens * k - slot) * size - first);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += part[i];
    }
    store_pack<false, T, V>(dx + token * size + first, sum, live);
  }
}

// ---------------------------------------------------------------------------
// the weighted sum of a token's slots
// ---------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const T* __restrict__ y, const float* __restrict__ weights,
                                                      const int64_t* __restrict__ places, T* __restrict__ out, int64_t tokens, int k,
                                                      int64_t size, int64_t limit) {
  constexpr int V = kV<T>;
  const int64_t pieces = (size + V - 1) / V;
  const bool short_ = tokens * pieces <= UINT32_MAX;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < tokens * pieces; at += stride) {
    int64_t token, piece;
    split_piece(at, pieces, short_, token, piece);
    const int64_t first = piece * V;
    const int live = static_cast<int>(size - first < V ? size - first : V);
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < k; ++j) {
      const int64_t place = places[token * k + j];
      if (static_cast<uint64_t>(place) >= static_cast<uint64_t>(limit)) continue;
      const float w = weights[token * k + j];
      const Pack<T, V> part = load_pack<T, V>(y + place * size + first, live, (limit - place) * size - first);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = fmaf(w, static_cast<float>(part[i]), sum[i]);
    }
    store_pack<true, T, V>(out + token * size + first, sum, live);
  }
}

// dy[place] = w dout[t],  dw = the dot product of dout[t] and y[place].  L lanes a
// token, whose slots they take in turn; behind the tokens, workgroups that clear
// the places of no slot.  Bound by its streams: 16,384 tokens of 1,024 in bfloat16,
// four slots each, 300 MB in 52 us (5.7 TB/s); forward 26 us (6.5 TB/s of 168 MB).
template <typename T, int L>
__global__ __launch_bounds__((L > 256 ? L : 256)) void combine_backward_kernel(
    const T* __restrict__ dout, const T* __restrict__ y, const float* __restrict__ weights, const int64_t* __restrict__ places,
    const int64_t* __restrict__ last, T* __restrict__ dy, float* __restrict__ dw, int64_t tokens, int k, int64_t size, int64_t limit,
    int64_t token_blocks) {
  constexpr int V = kV<T>;
  constexpr int kGroups = 256 / L;
  __shared__ float words[4];
  const int64_t block = block_index();
  const int64_t pieces = (size + V - 1) / V;
  if (block >= token_blocks) {
    if (dy == nullptr) return;
    int64_t from = *last;
    from = from < 0 ? 0 : (from > limit ? limit : from);
    const int64_t clearing = 64, number = block - token_blocks;
    if (number >= clearing) return;
    for (int64_t at = from * size + number * 256 + threadIdx.x; at < limit * size; at += clearing * 256) dy[at] = static_cast<T>(0.0f);
    return;
  }
  const int lane = threadIdx.x % L;
  const int64_t token = block * kGroups + threadIdx.x / L;
  const bool live_token = token < tokens;
  for (int j = 0; j < k; ++j) {
    const int64_t place = live_token ? places[token * k + j] : -1;
    const bool held = static_cast<uint64_t>(place) < static_cast<uint64_t>(limit);
    const float w = held ? weights[token * k + j] : 0.0f;
    double lane_dot = 0.0;   // of pieces' sums in 32 bits; all in 32: 1e-4 off over 4M equal elements
    if (held) {
      for (int64_t piece = lane; piece < pieces; piece += L) {
        const int64_t first = piece * V;
        const int live = static_cast<int>(size - first < V ? size - first : V);
        const Pack<T, V> grad = load_pack<T, V>(dout + token * size + first, live, (tokens - token) * size - first);
        if (dw != nullptr) {
          const Pack<T, V> row = load_pack<T, V>(y + place * size + first, live, (limit - place) * size - first);
          float of_piece = 0.0f;
#pragma unroll
          for (int i = 0; i < V; ++i) of_piece = fmaf(static_cast<float>(grad[i]), static_cast<float>(row[i]), of_piece);
          lane_dot += static_cast<double>(of_piece);
        }
        if (dy != nullptr) {
          float part[V];
#pragma unroll
          for (int i = 0; i < V; ++i) part[i] = w * static_cast<float>(grad[i]);
          store_pack<true, T, V>(dy + place * size + first, part, live);
        }
      }
    }
    if (dw == nullptr) continue;
    float dot = group_sum<(L < 64 ? L : 64)>(static_cast<float>(lane_dot));
    if constexpr (L > 64) {
      if ((threadIdx.x & 63) == 0) words[threadIdx.x / 64] = dot;
      __syncthreads();
      dot = (words[0] + words[1]) + (words[2] + words[3]);
      __syncthreads();
    }
    if (lane == 0 && live_token) dw[token * k + j] = dot;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int check_product(const char* what, int64_t places, int64_t k, int64_t inner, int64_t experts, int64_t k_in, int64_t n_out, int type) {
  if (places < 0 || inner < 0) return fail(DPA4K_EINVAL, "%s: negative sizes", what);
  if (experts < 1 || experts > kMaxExperts) return fail(DPA4K_EINVAL, "%s takes 1 to %d experts", what, kMaxExperts);
  if (k < 1 || places % k != 0) return fail(DPA4K_EINVAL, "%s: the places must be k for each token", what);
  if (k_in < 1 || n_out < 1 || k_in > 65536 || n_out > 65536) return fail(DPA4K_EINVAL, "%s: channels must be 1 to 65536", what);
  if (!known_type(type)) return fail(DPA4K_EINVAL, "%s: unknown type", what);
  // tiles of a row short of 2^31, whatever their number
  if (inner > 0 && places > (INT32_MAX - 1024) / inner) return fail(DPA4K_EINVAL, "%s takes fewer than 2^31 rows", what);
  return DPA4K_OK;
}

template <typename T, int MODE, int BM, int BN, int WM, int WN, int FAST, bool RUN = false, bool TWO = false>
int launch_product(ProductCall call, hipStream_t stream) {
  if constexpr (!TWO && sizeof(T) == 2 && (MODE == kInput || MODE == kWeight)) {
    if (call.a_low != nullptr) return launch_product<T, MODE, BM, BN, WM, WN, FAST, RUN, true>(call, stream);
  }
  typedef Tile<T, MODE, BM, BN, WM, WN> Z;
  const int64_t rows = call.places * call.inner;
  const int64_t width = MODE == kGated ? call.n_out / 2 : (MODE == kForward ? call.n_out : call.k_in);
  const int64_t columns = (width + (MODE == kGated ? BN / 2 : BN) - 1) / (MODE == kGated ? BN / 2 : BN);
  int64_t tiles;
  if (MODE == kWeight) tiles = columns * ((call.n_out + BM - 1) / BM) * (call.experts + (call.chunks > 0 ? rows / call.chunk_rows : 0));
  else tiles = columns * (rows / (RUN ? call.run * BM : BM) + call.experts + 1);
  if (tiles > row_block_limit(Z::kThreads)) return fail(DPA4K_EINVAL, "expert linear: more tiles than a launch takes");
  // two row tiles with all their columns; of dW, one (32,768 rows, 1,024 to 2 x 2,048 in
  // bfloat16: forward 459 -> 420 us against four, dW 439 -> 418 us, as dies then get more equal shares)
  const int64_t group = MODE != kWeight && tiles >= columns * 64 ? columns * 2 : columns;
  expert_product_kernel<T, MODE, BM, BN, WM, WN, FAST, RUN, TWO><<<static_cast<unsigned int>(tiles), Z::kThreads, 0, stream>>>(
      call, static_cast<int>(columns), static_cast<int>(tiles), static_cast<int>(group));
  return launched("expert_product_kernel");
}

template <typename T, int MODE, int FAST>
int run_tiles(const ProductCall& call, hipStream_t stream) {
  const int64_t width = MODE == kForward || MODE == kGated ? call.n_out : call.k_in;
  if constexpr (MODE == kWeight) {
    if (call.n_out <= 64 || call.k_in <= 64) return launch_product<T, MODE, 64, 64, 2, 2, FAST>(call, stream);
  } else {
    // Short sums over many rows: the workgroups' starts (the segment, the rows of x, the
    // first loads) take longer than their products, so each takes a run of tiles
    // and loads the next one while it multiplies and stores (786,432 rows of 64 by
    // 64 in float32: forward 114 -> 104 us, dx 127 -> 116 us; in two rounds 107 and 119).
    if constexpr (FAST == kRagged) {
      const int64_t depth = MODE == kInput ? call.n_out : call.k_in;
      const int64_t rows = call.places * call.inner, columns = width <= 64 ? 1 : (width + 127) / 128;
      const int64_t tiles = rows / 128 * columns, resident = width <= 64 ? 768 : 512;
      constexpr int64_t kRounds = 4;   // of workgroups, so that short runs at the segments' ends even out
      if (depth <= 4 * kSlice<T> && tiles >= 2 * kRounds * resident) {
        ProductCall runs = call;
        runs.run = static_cast<int>(tiles / (kRounds * resident) < kMostRun ? tiles / (kRounds * resident) : kMostRun);
        if (width <= 64) return launch_product<T, MODE, 128, 64, 4, 1, FAST, true>(runs, stream);
        return launch_product<T, MODE, 128, 128, 2, 2, FAST, true>(runs, stream);
      }
    }
    // Float32 is bound by its products: where segments are short, tiles of 32 rows
    // multiply fewer rows that are not there (64 rows an expert, 1,024 to 2 x 2,048:
    // 327 -> 237 us; bfloat16 81 -> 103 us).
    if constexpr (sizeof(T) == 4) {
      if (call.places * call.inner < 96 * call.experts) return launch_product<T, MODE, 32, 128, 1, 2, FAST>(call, stream);
    }
    if (width <= 64) return launch_product<T, MODE, 128, 64, 4, 1, FAST>(call, stream);
  }
  if constexpr (FAST == kRagged && sizeof(T) == 2) {
    if (call.k_in % kV<T> == 0 && call.n_out % kV<T> == 0 && width >= 256 &&
        (MODE == kWeight ? call.n_out : call.places * call.inner / call.experts) >= 256)
      return launch_product<T, MODE, 256, 256, 2, 4, kWhole>(call, stream);
  }
  return launch_product<T, MODE, 128, 128, 2, 2, FAST>(call, stream);
}

template <typename T, int MODE>
int run_product(const ProductCall& call, hipStream_t stream) {
  // Rows are whole 4-byte words and hold a piece of 16 bytes at least, and x, a matrix
  // and a tile of dz lie within 32-bit offsets (with some to spare, which a ragged
  // piece's offset moves back by); other calls load each piece through its own
  // address and registers.
  const int64_t rows_x = (call.order != nullptr ? call.places / call.k : call.places) * call.inner;
  const int64_t limit = (int64_t(kNoRow) - 4096) / static_cast<int64_t>(sizeof(T));
  const auto words = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
  const bool fast = call.k_in * sizeof(T) % 4 == 0 && call.n_out * sizeof(T) % 4 == 0 && call.k_in >= kV<T> && call.n_out >= kV<T> &&
                    words(call.a) && words(call.a_low) && words(call.b) && rows_x * call.k_in < limit &&
                    static_cast<int64_t>(call.n_out) * call.k_in < limit && static_cast<int64_t>(call.n_out) * 256 < limit &&
                    static_cast<int64_t>(call.k_in) * 256 < limit;
  return fast ? run_tiles<T, MODE, kRagged>(call, stream) : run_tiles<T, MODE, kByPiece>(call, stream);
}

// Rows of a segment that one workgroup of dW takes: at most kLongest, 2,048 additions
// of 16-bit operands (6e-5 of equal terms at worst) and 256 and 64 of float32, and where
// the matrices alone do not make tiles enough, so few that about 1,024 workgroups have
// some.  What is longer is cut, by its own length: routing may collapse to one of many
// experts (1,000,000 rows, 32 matrices of 1,024 to 2,048 in bfloat16: 4.4 ms for equal
// segments, 4.8 for a single one, 27.9 uncut).  Shorter cuts would cost partial sums: at
// 4,096 by 4,096 these are an eighth of the operands' bytes, with room for twice as many.
constexpr int64_t kLongest = 32768;

struct Chunks {
  int rows, most;    // most == 0: no segment is longer than that
  int segments;      // that can be longer
};

Chunks weight_chunks(int64_t places, int64_t inner, int64_t experts, int64_t k_in, int64_t n_out) {
  const int64_t rows = places * inner;
  const int64_t edge = n_out <= 64 || k_in <= 64 ? 64 : 128;
  const int64_t tiles = ((n_out + edge - 1) / edge) * ((k_in + edge - 1) / edge);
  int64_t chunk = kLongest;
  if (tiles * experts < 512 && rows > 512 * experts) {
    const int64_t share = ((rows * tiles + 1023) / 1024 + 511) / 512 * 512;
    chunk = share < kLongest ? share : kLongest;
  }
  if (rows <= chunk) return Chunks{static_cast<int>(chunk), 0, 0};
  const int64_t segments = rows / (chunk + 1) < experts ? rows / (chunk + 1) : experts;
  return Chunks{static_cast<int>(chunk), static_cast<int>(rows / chunk + segments), static_cast<int>(segments)};
}

int pieces_grid(int64_t pieces) {
  const int64_t blocks = (pieces + 255) / 256;
  return static_cast<int>(blocks < 8192 ? (blocks > 0 ? blocks : 1) : 8192);
}

}  // namespace
}  // namespace dpa4k

using namespace dpa4k;

extern "C" int dpa4k_expert_linear_forward(const void* x, const void* weight, const int64_t* offsets, const int64_t* order, void* y,
                                           float* before, int64_t places, int64_t k, int64_t inner, int64_t n_experts, int64_t k_in,
                                           int64_t n_out, int gated, int type, dpa4k_stream_t stream) {
  clear_error();
  const int status = check_product("expert linear", places, k, inner, n_experts, k_in, n_out, type);
  if (status != DPA4K_OK) return status;
  if (gated && n_out % 2 != 0) return fail(DPA4K_EINVAL, "expert linear: a gate needs an even number of outputs");
  if (places == 0 || inner == 0) return DPA4K_OK;
  if (x == nullptr || weight == nullptr || offsets == nullptr || y == nullptr) return fail(DPA4K_EINVAL, "expert linear: null pointer");
  ProductCall call{};
  call.a = x, call.b = weight, call.out = y, call.before = before, call.offsets = offsets, call.order = order;
  call.places = places, call.experts = static_cast<int>(n_experts), call.k = static_cast<int>(k), call.inner = static_cast<int>(inner);
  call.k_in = static_cast<int>(k_in), call.n_out = static_cast<int>(n_out);
  return with_type(type, DPA4K_EINVAL, [&](auto t) {
    typedef typename decltype(t)::type T;
    // Rows an expert up to which the matrices' bytes bound it (1,024 to 2 x 2,048, 32
    // experts, us, this way and in tiles: bfloat16 34 and 45 at one row, 56 and 55 at
    // eight, 70 and 58 at 16; float32 143 and 188 at 16 rows, 213 and 178 at 32).
    if (places * inner <= (sizeof(T) == 4 ? 24 : 8) * n_experts)
      return gated ? run_few_rows<T, true>(call, as_stream(stream)) : run_few_rows<T, false>(call, as_stream(stream));
    return gated ? run_product<T, kGated>(call, as_stream(stream)) : run_product<T, kForward>(call, as_stream(stream));
  });
}

extern "C" size_t dpa4k_expert_linear_workspace_size(int64_t places, int64_t k, int64_t inner, int64_t n_experts, int64_t k_in,
                                                     int64_t n_out, int by_token, int want_x, int want_weight) {
  if (places <= 0 || inner <= 0 || n_experts < 1 || k_in < 1 || n_out < 1 || places > INT32_MAX / inner) return 0;
  size_t bytes = 0;
  if (want_x && by_token) bytes = round_up_256(static_cast<size_t>(places * inner) * k_in * sizeof(float));
  if (want_weight) {
    const Chunks chunks = weight_chunks(places, inner, n_experts, k_in, n_out);
    const size_t partial = round_up_256(static_cast<size_t>(chunks.most) * n_out * k_in * sizeof(float));
    bytes = partial > bytes ? partial : bytes;    // one after the other
  }
  return bytes;
}

namespace {

// What both backwards do: dx and dW from dz, whose second part is `grad_low` (or null).
int linear_backward(const void* grad, const void* grad_low, const void* x, const void* weight, const int64_t* offsets,
                    const int64_t* order, const int64_t* slots, void* grad_x, void* grad_weight, int64_t places, int64_t k,
                    int64_t inner, int64_t n_experts, int64_t k_in, int64_t n_out, int type, void* workspace, hipStream_t on) {
  const bool by_token = order != nullptr;
  ProductCall call{};
  call.offsets = offsets, call.order = order;
  call.places = places, call.experts = static_cast<int>(n_experts), call.k = static_cast<int>(k), call.inner = static_cast<int>(inner);
  call.k_in = static_cast<int>(k_in), call.n_out = static_cast<int>(n_out);
  call.a = grad, call.a_low = grad_low;
  return with_type(type, DPA4K_EINVAL, [&](auto t) {
    typedef typename decltype(t)::type T;
    if (grad_x != nullptr) {
      ProductCall of_x = call;
      of_x.b = weight, of_x.out = by_token ? workspace : grad_x, of_x.by_slot = by_token;
      int ran = run_product<T, kInput>(of_x, on);
      if (ran != DPA4K_OK) return ran;
      if (by_token) {
        const int64_t tokens = places / k, size = inner * k_in;
        slot_sum_kernel<T><<<pieces_grid(tokens * ((size + kV<T> - 1) / kV<T>)), 256, 0, on>>>(
            static_cast<const float*>(workspace), slots, static_cast<T*>(grad_x), tokens, static_cast<int>(k), size, places);
        ran = launched("slot_sum_kernel");
        if (ran != DPA4K_OK) return ran;
      }
    }
    if (grad_weight != nullptr) {
      ProductCall of_w = call;
      const Chunks chunks = weight_chunks(places, inner, n_experts, k_in, n_out);
      of_w.b = x, of_w.chunk_rows = chunks.rows, of_w.chunks = chunks.most;
      of_w.out = grad_weight, of_w.partial = static_cast<float*>(workspace);
      int ran = run_product<T, kWeight>(of_w, on);
      if (ran != DPA4K_OK || chunks.most == 0) return ran;
      const int64_t size = k_in * n_out;
      const int64_t blocks = (size + 31) / 32 < 512 ? (size + 31) / 32 : 512;
      weight_sum_kernel<T><<<static_cast<unsigned int>(blocks * chunks.segments), 256, 0, on>>>(of_w, static_cast<int>(blocks));
      return launched("weight_sum_kernel");
    }
    return static_cast<int>(DPA4K_OK);
  });
}

// One part of dz, in bytes; a 16-bit dz has two.
size_t part_bytes(int64_t places, int64_t inner, int64_t n_out, int type) {
  return round_up_256(static_cast<size_t>(places * inner) * n_out * size_of_type(type));
}

}  // namespace

extern "C" int dpa4k_expert_linear_backward(const void* grad, const void* x, const void* weight, const int64_t* offsets,
                                            const int64_t* order, const int64_t* slots, void* grad_x, void* grad_weight,
                                            int64_t places, int64_t k, int64_t inner, int64_t n_experts, int64_t k_in, int64_t n_out,
                                            int type, void* workspace, size_t workspace_bytes, dpa4k_stream_t stream) {
  clear_error();
  const int status = check_product("expert linear", places, k, inner, n_experts, k_in, n_out, type);
  if (status != DPA4K_OK) return status;
  const bool by_token = order != nullptr;
  const bool nothing = places == 0 || inner == 0;
  if (nothing) grad_x = nullptr;
  if (grad_x == nullptr && grad_weight == nullptr) return DPA4K_OK;
  if (offsets == nullptr || (!nothing && grad == nullptr) || (grad_x != nullptr && (weight == nullptr || (by_token && slots == nullptr))) ||
      (grad_weight != nullptr && !nothing && x == nullptr))
    return fail(DPA4K_EINVAL, "expert linear: null pointer");
  const size_t needed = dpa4k_expert_linear_workspace_size(places, k, inner, n_experts, k_in, n_out, by_token, grad_x != nullptr,
                                                           grad_weight != nullptr);
  if (needed > 0 && (workspace == nullptr || workspace_bytes < needed))
    return fail(DPA4K_EWORKSPACE, "expert linear: workspace too small");
  return linear_backward(grad, nullptr, x, weight, offsets, order, slots, grad_x, grad_weight, places, k, inner, n_experts, k_in, n_out,
                         type, workspace, as_stream(stream));
}

extern "C" size_t dpa4k_expert_gated_workspace_size(int64_t places, int64_t k, int64_t inner, int64_t n_experts, int64_t k_in,
                                                    int64_t n_out, int by_token, int want_x, int want_weight, int type) {
  if (places <= 0 || inner <= 0 || n_experts < 1 || k_in < 1 || n_out < 1 || places > INT32_MAX / inner || !known_type(type)) return 0;
  return part_bytes(places, inner, n_out, type) * (size_of_type(type) == 2 ? 2 : 1) +
         dpa4k_expert_linear_workspace_size(places, k, inner, n_experts, k_in, n_out, by_token, want_x, want_weight);
}

extern "C" int dpa4k_expert_gated_backward(const void* grad, const float* before, const void* x, const void* weight,
                                           const int64_t* offsets, const int64_t* order, const int64_t* slots, void* grad_x,
                                           void* grad_weight, int64_t places, int64_t k, int64_t inner, int64_t n_experts, int64_t k_in,
                                           int64_t n_out, int type, void* workspace, size_t workspace_bytes, dpa4k_stream_t stream) {
  clear_error();
  const int status = check_product("expert linear", places, k, inner, n_experts, k_in, n_out, type);
  if (status != DPA4K_OK) return status;
  if (n_out % 2 != 0) return fail(DPA4K_EINVAL, "expert linear: a gate needs an even number of outputs");
  const hipStream_t on = as_stream(stream);
  const bool by_token = order != nullptr;
  const bool nothing = places == 0 || inner == 0;
  if (nothing) grad_x = nullptr;
  if (grad_x == nullptr && grad_weight == nullptr) return DPA4K_OK;
  if (offsets == nullptr || (!nothing && (grad == nullptr || before == nullptr)) ||
      (grad_x != nullptr && (weight == nullptr || (by_token && slots == nullptr))) || (grad_weight != nullptr && !nothing && x == nullptr))
    return fail(DPA4K_EINVAL, "expert linear: null pointer");
  const size_t needed = dpa4k_expert_gated_workspace_size(places, k, inner, n_experts, k_in, n_out, by_token, grad_x != nullptr,
                                                          grad_weight != nullptr, type);
  if (needed > 0 && (workspace == nullptr || workspace_bytes < needed))
    return fail(DPA4K_EWORKSPACE, "expert linear: workspace too small");
  const size_t part = nothing ? 0 : part_bytes(places, inner, n_out, type);
  char* high = static_cast<char*>(workspace);
  char* low = size_of_type(type) == 2 && !nothing ? high + part : nullptr;
  char* rest = low != nullptr ? low + part : high + part;
  if (!nothing) {
    const int ran = with_type(type, DPA4K_EINVAL, [&](auto t) {
      typedef typename decltype(t)::type T;
      const int64_t rows = places * inner, half = n_out / 2;
      gate_backward_kernel<T><<<pieces_grid(rows * ((half + kV<T> - 1) / kV<T>)), 256, 0, on>>>(
          static_cast<const T*>(grad), before, reinterpret_cast<T*>(high), reinterpret_cast<T*>(low), rows, static_cast<int>(half));
      return launched("gate_backward_kernel");
    });
    if (ran != DPA4K_OK) return ran;
  }
  return linear_backward(high, low, x, weight, offsets, order, slots, grad_x, grad_weight, places, k, inner, n_experts, k_in, n_out,
                         type, rest, on);
}

extern "C" int dpa4k_expert_combine_forward(const void* y, const float* weights, const int64_t* slots, void* out, int64_t tokens,
                                            int64_t k, int64_t size, int type, dpa4k_stream_t stream) {
  clear_error();
  if (tokens < 0 || k < 1 || size < 0) return fail(DPA4K_EINVAL, "expert combine: bad sizes");
  if (!known_type(type)) return fail(DPA4K_EINVAL, "expert combine: unknown type");
  if (tokens > INT32_MAX / k) return fail(DPA4K_EINVAL, "expert combine takes fewer than 2^31 slots");
  if (size > INT32_MAX) return fail(DPA4K_EINVAL, "expert combine: an entry has fewer than 2^31 elements");
  if (tokens == 0 || size == 0) return DPA4K_OK;
  if (y == nullptr || weights == nullptr || slots == nullptr || out == nullptr) return fail(DPA4K_EINVAL, "expert combine: null pointer");
  return with_type(type, DPA4K_EINVAL, [&](auto t) {
    typedef typename decltype(t)::type T;
    combine_kernel<T><<<pieces_grid(tokens * ((size + kV<T> - 1) / kV<T>)), 256, 0, as_stream(stream)>>>(
        static_cast<const T*>(y), weights, slots, static_cast<T*>(out), tokens, static_cast<int>(k), size, tokens * k);
    return launched("combine_kernel");
  });
}

extern "C" int dpa4k_expert_combine_backward(const void* grad, const void* y, const float* weights, const int64_t* slots,
                                             const int64_t* last_offset, void* grad_y, float* grad_weights, int64_t tokens, int64_t k,
                                             int64_t size, int type, dpa4k_stream_t stream) {
  clear_error();
  if (tokens < 0 || k < 1 || size < 0) return fail(DPA4K_EINVAL, "expert combine: bad sizes");
  if (!known_type(type)) return fail(DPA4K_EINVAL, "expert combine: unknown type");
  if (tokens > INT32_MAX / k) return fail(DPA4K_EINVAL, "expert combine takes fewer than 2^31 slots");
  if (size > INT32_MAX) return fail(DPA4K_EINVAL, "expert combine: an entry has fewer than 2^31 elements");
  if (tokens == 0) return DPA4K_OK;
  if (slots == nullptr || weights == nullptr || (size > 0 && (grad == nullptr || y == nullptr)) ||
      (grad_y != nullptr && last_offset == nullptr))
    return fail(DPA4K_EINVAL, "expert combine: null pointer");
  return with_type(type, DPA4K_EINVAL, [&](auto t) {
    typedef typename decltype(t)::type T;
    const int64_t pieces = (size + kV<T> - 1) / kV<T>;
    const auto run = [&](auto l) {
      constexpr int L = l.value;
      const int64_t blocks = (tokens + 256 / L - 1) / (256 / L);
      combine_backward_kernel<T, L><<<launch_grid(blocks + 64, 256), 256, 0, as_stream(stream)>>>(
          static_cast<const T*>(grad), static_cast<const T*>(y), weights, slots, last_offset, static_cast<T*>(grad_y), grad_weights,
          tokens, static_cast<int>(k), size, tokens * k, blocks);
      return launched("combine_backward_kernel");
    };
    if (pieces <= 16) return run(std::integral_constant<int, 16>{});
    if (pieces <= 256) return run(std::integral_constant<int, 64>{});
    return run(std::integral_constant<int, 256>{});
  });
}
