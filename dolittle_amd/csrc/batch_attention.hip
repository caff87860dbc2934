// Attention of a batch of sequences over a prefix that they share and caches
// of their own, and the weight that every cached key received.  No reference
// counterpart: the reference decodes one sequence over one contiguous cache.
//
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// over the prefix's keys and, for new row i of a sequence that holds n rows,
// its own keys j < n - rows + i + 1.  A row without a key is zeros.  A key
// that a row does not see has no effect on it, whatever the key's bytes are.
// Outputs are divided by their sum at the end and the maximum lags by at most
// 2^13, so values below 2^114 / keys cannot overflow before that.
//
// Split.  All rows of a KV head (every sequence's, every new row's, the heads
// of the group) are one matrix against the prefix, so the prefix is read once
// for a workgroup's rows and not once per sequence.  A workgroup takes some
// rows and a range of keys of one source (the prefix, or one sequence's cache)
// and leaves their maximum, sum and unnormalised output; k_join joins the
// ranges and adds up the weights of a decode step from the scores that k_ranges
// stored; k_weights computes those of more rows again.
//
// Up to 32 rows, FP32 rows and rows that are not 16-byte pieces run apart: 16
// in every wavefront, the wavefronts taking every fourth step of 32 keys (FP32
// 16) straight from memory into matrix operands.  Scores are K Q^T, so that the
// first operand has a lane per key, and leave a lane with the keys that the
// P^T operand of V^T P^T wants from it; a lane loads C = D / 16 neighbouring
// features of each of its keys, and since any 16 features may form a matrix
// tile, tile j takes feature j of every lane's C: the transposition is a byte
// permute (BF16) or nothing (FP32).  Bound by the key and value stream with one
// step in flight a wavefront: 8 sequences of up to 4607 keys, 101 MB in 26 us,
// of which 4 until the first step has landed (6.15 TB/s is this card's rate for
// a large read).  FP32, 192 rows a KV head over 1001 keys: 19 us, 6 at 154
// TFLOP/s; the matrix unit is busy 34% of the time, and wavefronts, two to a
// SIMD, wait 57% of theirs for an instruction to issue and 29% for loads.
//
// More BF16 rows run together: 16 or 32 in each wavefront, keys and values
// through LDS for all four (64 sequences over 32768 keys 84 us, 114 with every
// wavefront loading its own).  Bound by the chain of one step, products, softmax
// and products again, with fewer than two wavefronts to a SIMD to fill it: 512
// rows of 4 heads over 4096 keys 54 us, 600 TFLOP/s, products 30% of a SIMD's
// cycles and vector instructions 45%; 64 sequences 21% and 31%.  Which form is
// taken goes by rows and storage alone; 128 rows a workgroup instead of 64 where
// those still fill the chip.
//
// BF16 storage rounds P to BF16 (8 bits, off by at most 2^-8 of the value) for the
// product with V, as BF16 matrix operands need: 0.20 to 0.23% off 64-bit results
// where rounding the output alone is 0.17%;
// scores, exponentials, sums, maxima and outputs are FP32 throughout, and so
// are the weights.  FP32 storage runs FP32 matrix instructions.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "batch.h"
#include "dl_device.h"
#include "dl_internal.h"

namespace dl::batch {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kLog2e = 0x1.715476p+0f;
// Scores are in units of ln 2 from the first maximum on: exponentials are the
// hardware's exp2 of one fused multiply-add.  A maximum is raised only when the
// exponentials of a lane's keys of one step sum to more than kMostSum: most
// steps rescale nothing.
constexpr float kMostSum = 8192.0f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// How rows are read: whole 16-byte pieces up to D features; whole pieces up to
// the width; or element by element, for widths or operands that are not
// 16-byte aligned.
enum class Access { kWhole, kPieces, kElements };

// N consecutive elements `offset` bytes past a base that the wavefront shares,
// of which the row's features from `at` on; zeros past the width.
template <class T, int N, Access A>
__device__ __forceinline__ void load_words(const char* base, uint32_t offset, int at, int width, uint32_t* out) {
  constexpr int kWords = N * sizeof(T) / 4;
  const char* p = base + offset;
  if constexpr (A == Access::kElements) {
    const T* e = reinterpret_cast<const T*>(p);
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        out[i] = at + i < width ? __float_as_uint(e[i]) : 0u;
      } else {
        const uint32_t lo = at + 2 * i < width ? e[2 * i] : 0u;
        const uint32_t hi = at + 2 * i + 1 < width ? e[2 * i + 1] : 0u;
        out[i] = lo | (hi << 16);
      }
    }
  } else if constexpr (kWords == 2) {
    const u32x2 v = A == Access::kWhole || at < width ? *reinterpret_cast<const u32x2*>(p) : u32x2{};
    out[0] = v.x;
    out[1] = v.y;
  } else {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const u32x4 v =
          A == Access::kWhole || at + i * kPer < width ? reinterpret_cast<const u32x4*>(p)[i] : u32x4{};
      out[4 * i] = v.x;
      out[4 * i + 1] = v.y;
      out[4 * i + 2] = v.z;
      out[4 * i + 3] = v.w;
    }
  }
}

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
// The value subtracted from scores: 0 while no score is finite, so that
// exp2(-inf - m) is 0 and not NaN.
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.0f : m; }

// Code that few steps run is laid out behind the rest: a workgroup's first pass
// through a step is bound by instruction fetch.
__device__ __forceinline__ bool rare(bool condition) { return __builtin_expect(condition, false); }

__device__ __forceinline__ float group_max(float v) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_sum(float v) {
  v = v + __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// One wavefront's matrix operands for storage type T and heads of up to D
// features.  lane = 16 g + i.
template <class T, int D, Access A>
struct Operands;

template <int D, Access A>
struct Operands<uint16_t, D, A> {
  using T = uint16_t;
  static constexpr int kKeys = 32, kTiles = 2, kSteps = D / 32, C = D / 16;
  static constexpr int kValueRows = 8;
  struct Values {
    uint32_t v[kValueRows][C / 2];
  };
  // A row's features (4 s + g) 8 .. of product step s; `offset` holds the lane's own 16 g bytes.
  static __device__ __forceinline__ void load_row(const char* base, uint32_t offset, int g, int width, u32x4* out) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      load_words<T, 8, A>(base + 64 * s, offset, (4 * s + g) * 8, width, reinterpret_cast<uint32_t*>(&out[s]));
  }
  // The key of value row r in the order in which P holds them.
  static __device__ __forceinline__ constexpr int value_key(int g, int r) { return (r / 4) * 16 + 4 * g + r % 4; }
  // Scores of NQ row tiles against NK key tiles, the chains side by side.
  template <int NQ, int NK>
  static __device__ __forceinline__ void scores(const u32x4 (&k)[NK][kSteps], const u32x4 (&q)[NQ][kSteps], f32x4 (&s)[NQ][NK]) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int t = 0; t < NQ; ++t)
#pragma unroll
        for (int u = 0; u < NK; ++u)
          s[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[u][i]),
                                                            __builtin_bit_cast(bf16x8, q[t][i]),
                                                            i ? s[t][u] : f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
  }
  static constexpr uint32_t kSigns = 0x80008000u;
  // The first operand of feature tile j.
  static __device__ __forceinline__ bf16x8 value_tile(const Values& v, int j) {
    u32x4 w;
    const uint32_t pick = j % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int p = 0; p < 4; ++p) w[p] = __builtin_amdgcn_perm(v.v[2 * p + 1][j / 2], v.v[2 * p][j / 2], pick);
    return __builtin_bit_cast(bf16x8, w);
  }
  template <int QT>
  static __device__ __forceinline__ void rounded(const f32x4 (&p)[QT][kTiles], bf16x8 (&b)[QT]) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) b[t][e] = static_cast<__bf16>(p[t][e / 4][e % 4]);
  }
  template <int QT>
  static __device__ __forceinline__ void products(const Values& v, const f32x4 (&p)[QT][kTiles], f32x4 (&o)[QT][C]) {
    bf16x8 b[QT];
    rounded<QT>(p, b);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const bf16x8 a = value_tile(v, j);
#pragma unroll
      for (int t = 0; t < QT; ++t) o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[t], o[t][j], 0, 0, 0);
    }
  }
  static __device__ __forceinline__ uint32_t without_special(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
  }
};

template <int D, Access A>
struct Operands<float, D, A> {
  using T = float;
  static constexpr int kKeys = 16, kTiles = 1, kSteps = D / 16, C = D / 16;
  static constexpr int kValueRows = 4;
  struct Values {
    uint32_t v[kValueRows][C];
  };
  // `offset` holds the lane's own 16 g bytes.
  static __device__ __forceinline__ void load_row(const char* base, uint32_t offset, int g, int width, u32x4* out) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      load_words<T, 4, A>(base + 64 * s, offset, (4 * s + g) * 4, width, reinterpret_cast<uint32_t*>(&out[s]));
  }
  static __device__ __forceinline__ constexpr int value_key(int g, int r) { return 4 * g + r; }
  template <int NQ, int NK>
  static __device__ __forceinline__ void scores(const u32x4 (&k)[NK][kSteps], const u32x4 (&q)[NQ][kSteps], f32x4 (&s)[NQ][NK]) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < NQ; ++t)
#pragma unroll
          for (int u = 0; u < NK; ++u)
            s[t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[u][i][e]), __uint_as_float(q[t][i][e]),
                                                           i + e ? s[t][u] : f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
  }
  static constexpr uint32_t kSigns = 0x80000000u;
  template <int QT>
  static __device__ __forceinline__ void products(const Values& v, const f32x4 (&p)[QT][kTiles], f32x4 (&o)[QT][C]) {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < QT; ++t)
          o[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v.v[r][j]), p[t][0][r], o[t][j], 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t without_special(uint32_t w) {
    return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
  }
};

// Keys of one range when `keys` are cut into at most `splits`: whole rounds of
// the four wavefronts' steps (kRound keys).
constexpr int kRound = 128;
__host__ __device__ inline uint32_t range_keys(uint32_t keys, uint32_t splits) {
  const uint32_t each = keys / splits + (keys % splits != 0);
  return (each + kRound - 1) / kRound * kRound;
}

struct Args {
  const void *query, *prefix_key, *prefix_value, *key, *value;
  const uint64_t* lengths;
  const float* scale;
  void* out;
  float2* part;  // [ranges][kv head][row]: maximum, sum
  float* sums;   // [ranges][kv head][row][pitch]: unnormalised output
  float2* whole; // [kv head][row]: maximum, 1 / sum, for k_weights, or null
  float* scores; // [batch][kv head][seq row][score_pitch]: own scores before the scale, or null
  const float* weights;
  float* weights_out;
  uint32_t batch, rows, q_heads, kv_heads, group, width, prefix, capacity;
  uint32_t seq_rows, all_rows;          // rows of one sequence and of the batch, per KV head
  uint32_t prefix_splits, own_splits;   // ranges of the prefix, most ranges of an own cache
  uint32_t prefix_each;                 // keys of a range of the prefix
  uint32_t prefix_blocks, prefix_tiles, own_tiles;
  uint32_t pitch, score_pitch;          // row widths of `sums` and `scores`
};

__device__ __forceinline__ uint32_t length_of(const Args& a, uint32_t b) {
  const uint64_t n = a.lengths[b];
  return n < a.capacity ? static_cast<uint32_t>(n) : a.capacity;
}
// Own keys that new row i of a sequence of n rows sees.
__device__ __forceinline__ uint32_t visible(uint32_t n, uint32_t rows, uint32_t i) {
  const uint64_t end = static_cast<uint64_t>(n) + i + 1;
  return end > rows ? min(static_cast<uint32_t>(end - rows), n) : 0u;
}
__device__ __forceinline__ uint64_t query_offset(const Args& a, uint32_t row, uint32_t kvh) {
  return (static_cast<uint64_t>(row / a.group) * a.q_heads + kvh * a.group + row % a.group) * a.width;
}

// Work of one block: XCD x takes the groups x, x + 8, ..., and all row tiles of
// a group, which read the same keys, so that they meet in one L2.
__device__ __forceinline__ bool block_task(uint32_t id, uint32_t groups, uint32_t tiles, uint32_t& group, uint32_t& tile) {
  const uint32_t j = id / 8;
  group = j / tiles * 8 + id % 8;
  tile = j % tiles;
  return group < groups;
}

// The scale in units of ln 2; its sign goes into the query.
__device__ __forceinline__ float factor_of(float scale) { return fabsf(scale) * kLog2e; }
template <class Ops, int N>
__device__ __forceinline__ void take_sign(float scale, u32x4 (&q)[N]) {
  if (scale < 0.0f) {
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = q[i] ^ Ops::kSigns;
  }
}

// What a workgroup does: rows [first, first + count) of the batch's per KV head
// against keys [begin, end) of one source, the result of range `slot`.
struct Range {
  const char *keys, *values;  // the KV head's features of the source's first key
  float* scores;              // of the first row, or null
  uint32_t first, count, kvh, begin, end, slot;
  uint32_t least;             // keys that every row sees
};

// One wavefront's 16 QT rows: running maximum, sum and output.  Lane 16 g + i
// holds row i's scores of the keys 4 g + r of a step's tiles, and in o[t][j][r]
// its feature (4 g + r) C + j, or 16 j + 4 g + r where value operands are read
// across the rows of LDS (Across).
template <class Ops, int QT, bool Across>
struct Rows {
  static constexpr int C = Ops::C, kTiles = Ops::kTiles;
  f32x4 o[QT][C];
  float top[QT], sum[QT];
  float from[QT], most[QT];  // added to scores; the largest step sum that raises nothing
  uint32_t limit[QT];        // keys that the lane's row sees

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      top[t] = -INFINITY;
      from[t] = sum[t] = 0.0f;
      most[t] = -1.0f;
#pragma unroll
      for (int j = 0; j < C; ++j) o[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  static __device__ __forceinline__ int feature(int g, int j, int r) { return Across ? 16 * j + 4 * g + r : (4 * g + r) * C + j; }

  // Scores of the step at key `at` to exponentials against the maximum so far.
  // A row whose exponentials of a step sum to more than 2^13 in some lane (its
  // scores pass that maximum by as much), and that of a first step, raises its
  // maximum and rescales what is summed; other steps need no maximum of their own.
  __device__ __forceinline__ void soften(f32x4 (&p)[QT][kTiles], bool masked, uint32_t at, float factor) {
    const int g = threadIdx.x % 64 / 16;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      auto hide = [&](f32x4 (&v)[kTiles], float value) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (at + 16 * u + 4 * g + r >= limit[t]) v[u][r] = value;
      };
      f32x4 e[kTiles];
      auto weigh = [&] {
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) e[u][r] = exp2_of(fma_rn(p[t][u][r], factor, from[t]));
        if (rare(masked)) hide(e, 0.0f);  // also the NaN of a hidden key under a zero scale
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < kTiles; ++u) s = s + ((e[u][0] + e[u][1]) + (e[u][2] + e[u][3]));
        return s;
      };
      float s = weigh();
      if (rare(__any(!(s <= most[t])))) {
        // Each row by itself: what another row sees changes no bit of this one.
        const bool rises = group_max(s <= most[t] ? 0.0f : 1.0f) > 0.0f;
        if (masked) hide(p[t], -INFINITY);
        float high = -INFINITY;
#pragma unroll
        for (int u = 0; u < kTiles; ++u) high = fmaxf(high, fmaxf(fmaxf(p[t][u][0], p[t][u][1]), fmaxf(p[t][u][2], p[t][u][3])));
        const float highest = group_max(high) * factor, raised = rises ? fmaxf(top[t], highest) : top[t];
        const float less = top[t] == -INFINITY ? 1.0f : exp2_of(top[t] - raised);  // nothing summed yet: zeros
        top[t] = raised;
        from[t] = -reference_of(raised);
        most[t] = raised == -INFINITY ? -1.0f : kMostSum;
        sum[t] = sum[t] * less;
#pragma unroll
        for (int j = 0; j < C; ++j) o[t][j] = o[t][j] * less;
        s = weigh();
      }
      sum[t] = sum[t] + s;
#pragma unroll
      for (int u = 0; u < kTiles; ++u) p[t][u] = e[u];
    }
  }
  // Elements of a step's values that are not finite have left the product: they
  // are added to the rows that see them.  `source` is the step's first row.
  __device__ __forceinline__ void add_special(const f32x4 (&p)[QT][kTiles], uint32_t at, uint32_t end, const char* source,
                                              uint32_t stride, int width, float (*shares)[16]) {
    using T = typename Ops::T;
    const int lane = threadIdx.x % 64, i16 = lane % 16, g = lane / 16;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) shares[16 * u + 4 * g + r][i16] = p[t][u][r];
      __builtin_amdgcn_wave_barrier();
      const uint32_t seen = min(min(limit[t], end), at + Ops::kKeys);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        f32x4 to = o[t][j];
#pragma unroll 1
        for (uint32_t k = 0; at + k < seen; ++k) {
          const T* row = reinterpret_cast<const T*>(source + k * stride);
          const float share = shares[k][i16];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int f = feature(g, j, r);
            const float x = f < width ? load_elem(row, f) : 0.0f;
            to[r] = fabsf(x) < INFINITY ? to[r] : fma_rn(share, x, to[r]);
          }
        }
        o[t][j] = to;
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  // Rows first + 16 t + lane % 16 of the range's result.
  __device__ __forceinline__ void store(const Args& a, const Range& range, uint32_t first, bool whole) const {
    const int lane = threadIdx.x % 64, i16 = lane % 16, g = lane / 16;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      if (first + 16u * t + i16 >= range.count) continue;
      const uint64_t row = (static_cast<uint64_t>(range.slot) * a.kv_heads + range.kvh) * a.all_rows + range.first + first + 16 * t + i16;
      if (g == 0) a.part[row] = make_float2(top[t], sum[t]);
      float* dst = a.sums + row * a.pitch;
#pragma unroll
      for (int m = 0; m < C; ++m) {  // four features in order
        const uint32_t f = Across ? 16 * m + 4 * g : 4 * (g * C + m);
        f32x4 v = o[t][m];
        if constexpr (!Across) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = o[t][(4 * m + e) % C][(4 * m + e) / C];
        }
        if (whole || f < a.pitch) *reinterpret_cast<f32x4*>(dst + f) = v;
      }
    }
  }
};

// The operands of query rows first .. of the range's.
template <class Ops, int QT>
__device__ __forceinline__ void load_queries(const Args& a, const Range& range, uint32_t first, float scale,
                                             u32x4 (&q)[QT][Ops::kSteps]) {
  const int lane = threadIdx.x % 64, i16 = lane % 16, g = lane / 16;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint64_t at = query_offset(a, range.first + min(first + 16u * t + i16, range.count - 1), range.kvh);
    Ops::load_row(reinterpret_cast<const char*>(static_cast<const typename Ops::T*>(a.query) + at), 16 * g, g, a.width, q[t]);
    take_sign<Ops>(scale, q[t]);
  }
}

// Few rows: every wavefront holds all of them and takes every fourth step,
// its keys and values straight from memory, a step ahead.
template <class Ops, int QT>
struct Joined {
  f32x4 o[kWaves / 2 * QT][Ops::C][64];
};

template <class T, int D, int QT, Access A>
__device__ __forceinline__ void run_apart(const Args& a, const Range& range, Rows<Operands<T, D, A>, QT, false>& rows,
                                          Joined<Operands<T, D, A>, QT>& room, float (*shares)[16]) {
  using Ops = Operands<T, D, A>;
  constexpr int C = Ops::C, KT = Ops::kKeys, kTiles = Ops::kTiles;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int i16 = lane % 16, g = lane / 16;
  const int width = a.width;
  const uint32_t stride = a.kv_heads * a.width * sizeof(T), end = range.end;
  const float scale = *a.scale, factor = factor_of(scale);
  u32x4 q[QT][Ops::kSteps];
  load_queries<Ops>(a, range, 0, scale, q);
  rows.clear();

  u32x4 kf[kTiles][Ops::kSteps];
  typename Ops::Values vf;
  // A step's rows by 32-bit offsets from its first key; rows past the last key
  // repeat it: they are masked, and their values cleared.
  const uint32_t key_offset = i16 * stride + 16 * g;
  const uint32_t value_offset = 4 * g * stride + i16 * C * sizeof(T);
  auto load_keys = [&](uint32_t at) {
    const char* base = range.keys + static_cast<uint64_t>(at) * stride;
    const uint32_t most = min(end - at - 1, 63u) * stride + 16 * g;
#pragma unroll
    for (int u = 0; u < kTiles; ++u) Ops::load_row(base, min(key_offset + 16 * u * stride, most), g, width, kf[u]);
  };
  auto load_values = [&](uint32_t at) {
    const char* base = range.values + static_cast<uint64_t>(at) * stride;
    const uint32_t most = min(end - at - 1, 63u) * stride + i16 * C * sizeof(T);
#pragma unroll
    for (int r = 0; r < Ops::kValueRows; ++r)
      load_words<T, C, A>(base, min(value_offset + Ops::value_key(0, r) * stride, most), i16 * C, width, vf.v[r]);
  };
  // Steps past the range repeat its last key: operands are defined on every
  // path.  (With these loads under `next < end`, which leaves no use undefined
  // either, hipcc of ROCm 7.2 assembles value operands in the registers of the
  // first loaded row, whose other words are read later: wrong results from the
  // BF16 kernels of 128 and 256 features.  tests/test_batch_code.py looks for
  // that in the built code.)
  uint32_t at = range.begin + wave * KT;
  if (at < end) {
    load_keys(at);
    load_values(at);
  }
  while (at < end) {
    const uint32_t next = at + kWaves * KT, ahead = min(next, end - 1);
    f32x4 p[QT][kTiles];
    Ops::scores(kf, q, p);
    load_keys(ahead);
    if (range.scores && static_cast<uint32_t>(i16) < range.count) {
      float* row = range.scores + static_cast<uint64_t>(i16) * a.score_pitch + at + 4 * g;
#pragma unroll
      for (int u = 0; u < kTiles; ++u) *reinterpret_cast<f32x4*>(row + 16 * u) = p[0][u];
    }
    const bool masked = at + KT > range.least;
    rows.soften(p, masked, at, factor);
    if (rare(masked)) {
      // Values of keys past the end are cleared.  An infinity or NaN in the
      // values of a key that only some rows see must not reach the others
      // through 0 * inf.
      bool special = false;
#pragma unroll
      for (int r = 0; r < Ops::kValueRows; ++r)
#pragma unroll
        for (uint32_t& w : vf.v[r]) {
          if (at + Ops::value_key(g, r) >= end) w = 0;
          const uint32_t plain = Ops::without_special(w);
          special |= plain != w;
          w = plain;
        }
      if (rare(__any(special)))
        rows.add_special(p, at, end, range.values + static_cast<uint64_t>(at) * stride, stride, width, shares + wave * 32);
    }
    Ops::template products<QT>(vf, p, rows.o);
    load_values(ahead);
    at = next;
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) rows.sum[t] = group_sum(rows.sum[t]);

  // Join the wavefronts: the upper half into the lower, and so on; those without
  // a step have nothing to give.  A giver's maxima and sums lie in its own shares.
  auto stats = [&](int of) { return reinterpret_cast<float2*>(shares + of * 32); };
  const uint32_t steps = end > range.begin ? (end - range.begin + KT - 1) / KT : 0;
#pragma unroll
  for (int half = kWaves / 2; half; half /= 2) {
    if (steps <= static_cast<uint32_t>(half)) continue;
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        if (g == 0) stats(wave)[16 * t + i16] = make_float2(rows.top[t], rows.sum[t]);
#pragma unroll
        for (int j = 0; j < C; ++j) room.o[(wave - half) * QT + t][j][lane] = rows.o[t][j];
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float2 other = stats(wave + half)[16 * t + i16];
        const float raised = fmaxf(rows.top[t], other.x), from = reference_of(raised);
        const float mine = exp2_of(rows.top[t] - from), theirs = exp2_of(other.x - from);
        rows.top[t] = raised;
        rows.sum[t] = fma_rn(rows.sum[t], mine, other.y * theirs);
#pragma unroll
        for (int j = 0; j < C; ++j) rows.o[t][j] = rows.o[t][j] * mine + room.o[wave * QT + t][j][lane] * theirs;
      }
    }
    __syncthreads();
  }
  if (wave == 0) rows.store(a, range, 0, A == Access::kWhole);
}

// Many BF16 rows: a wavefront holds 16 QT rows of its own, and the four share
// the keys and values through LDS, loaded there directly, a tile ahead.  Value
// operands are read across the rows (a lane gives four features of one key and
// gets one feature of four keys), so no register is permuted.  A row of a tile
// keeps its 16-byte pieces at piece ^ swizzle(row): the sixteen rows of a key
// operand, and the eight rows of two pieces that half a wavefront reads of a
// value operand, lie in distinct banks.
template <int D>
struct Stage {
  static constexpr int kKeys = D == 256 ? 32 : 64, kPieces = D / 8, kRowBytes = 2 * D;
  static constexpr int kBytes = kKeys * kRowBytes;  // of keys, and of values
  static __device__ __forceinline__ uint32_t swizzle(uint32_t row) {
    return D == 64 ? 2 * (row / 2 % 4) + row / 8 % 2 : 2 * (row % 8) + row / 8 % 2;
  }
};
// A separate LDS object per stage, so that the compiler adds no waits between
// the loads in flight and the reads.
template <int D, int I>
__device__ __forceinline__ uint8_t* stage_room() {
  __shared__ __align__(1024) uint8_t room[2 * Stage<D>::kBytes];
  return room;
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

template <int D, int QT, Access A>
__device__ __forceinline__ void run_together(const Args& a, const Range& range, Rows<Operands<uint16_t, D, A>, QT, true>& rows,
                                             float (*shares)[16]) {
  using T = uint16_t;
  using Ops = Operands<T, D, A>;
  using S = Stage<D>;
  constexpr int C = Ops::C, KT = Ops::kKeys, kTiles = Ops::kTiles;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i16 = lane % 16, g = lane / 16;
  const uint32_t width = a.width, stride = a.kv_heads * a.width * sizeof(T), end = range.end;
  const float scale = *a.scale, factor = factor_of(scale);
  const uint32_t first = wave * 16 * QT;
  u32x4 q[QT][Ops::kSteps];
  load_queries<Ops>(a, range, first, scale, q);
  rows.clear();

  auto issue = [&](uint8_t* room, uint32_t at) {
    const char* keys = range.keys + static_cast<uint64_t>(at) * stride;
    const char* values = range.values + static_cast<uint64_t>(at) * stride;
#pragma unroll
    for (int i = 0; i < S::kBytes / 1024 / kWaves; ++i) {  // 1024 bytes of each at a time
      const uint32_t slot = (i * kWaves + wave) * 64 + lane, row = slot / S::kPieces;
      uint32_t piece = slot % S::kPieces ^ S::swizzle(row);
      if (A != Access::kWhole && piece * 8 >= width) piece = 0;  // not a piece of the row: cleared or not stored
      const uint32_t offset = min(row, end - at - 1) * stride + piece * 16;
      uint8_t* to = room + (i * kWaves + wave) * 1024;
      __builtin_amdgcn_global_load_lds((const global_ptr*)(keys + offset), (lds_ptr*)to, 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const global_ptr*)(values + offset), (lds_ptr*)(to + S::kBytes), 16, 0, 0);
    }
  };
  const uint32_t value_row = 4 * g + i16 / 4;  // the row of the lane's share of a value read
  auto step = [&](uint8_t* room, uint32_t row0, uint32_t at) {
    u32x4 kf[kTiles][Ops::kSteps];
#pragma unroll
    for (int u = 0; u < kTiles; ++u)
#pragma unroll
      for (int s = 0; s < Ops::kSteps; ++s) {
        kf[u][s] = *reinterpret_cast<const u32x4*>(room + (row0 + 16 * u + i16) * S::kRowBytes + ((4 * s + g) ^ S::swizzle(i16)) * 16);
        if (A != Access::kWhole && (4 * s + g) * 8 >= width) kf[u][s] = u32x4{};
      }
    f32x4 p[QT][kTiles];
    Ops::scores(kf, q, p);
    const bool masked = at + KT > range.least;
    rows.soften(p, masked, at, factor);
    // Feature 16 j + i16 of keys 16 u + 4 g ..: words 2 u, 2 u + 1.
    u32x4 vf[C];
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        uint8_t* from = room + S::kBytes + (row0 + 16 * u + value_row) * S::kRowBytes +
                        ((2 * j + i16 / 2 % 2) ^ S::swizzle(value_row)) * 16 + i16 % 2 * 8;
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)from));
        vf[j][2 * u] = v.x;
        vf[j][2 * u + 1] = v.y;
      }
    if (rare(masked)) {  // as for rows apart
      bool special = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t key = at + 16 * (w / 2) + 4 * g + 2 * (w % 2);
        const uint32_t real = (key < end ? 0xffffu : 0u) | (key + 1 < end ? 0xffff0000u : 0u);
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const uint32_t word = vf[j][w] & real, plain = Ops::without_special(word);
          special |= plain != word;
          vf[j][w] = plain;
        }
      }
      if (rare(__any(special)))
        rows.add_special(p, at, end, range.values + static_cast<uint64_t>(at) * stride, stride, width, shares + wave * 32);
    }
    bf16x8 b[QT];
    Ops::template rounded<QT>(p, b);
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int t = 0; t < QT; ++t)
        rows.o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vf[j]), b[t], rows.o[t][j], 0, 0, 0);
  };
  auto tile = [&](uint8_t* room, uint8_t* other, uint32_t at) {
    __builtin_amdgcn_s_waitcnt(vm_wait(0));  // this tile has landed
    __syncthreads();                         // for everybody, and the other buffer is read
    if (at + S::kKeys < end) issue(other, at + S::kKeys);
    __builtin_amdgcn_sched_barrier(0);
    if (first >= range.count) return;
#pragma unroll 1
    for (uint32_t k = 0; k < S::kKeys && at + k < end; k += KT) step(room, k, at + k);
  };
  if (range.begin < end) issue(stage_room<D, 0>(), range.begin);
  for (uint32_t at = range.begin; at < end; at += 2 * S::kKeys) {
    tile(stage_room<D, 0>(), stage_room<D, 1>(), at);
    if (at + S::kKeys < end) tile(stage_room<D, 1>(), stage_room<D, 0>(), at + S::kKeys);
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) rows.sum[t] = group_sum(rows.sum[t]);
  if (first < range.count) rows.store(a, range, first, A == Access::kWhole);
}

// Rows of a workgroup against one source: kApart holds 16 in every wavefront,
// kTogether1 and kTogether2 16 and 32 in each.
enum class Mode { kApart, kTogether1, kTogether2 };
constexpr bool together(Mode m) { return m != Mode::kApart; }
constexpr int tiles_of(Mode m) { return m == Mode::kTogether2 ? 2 : 1; }
constexpr uint32_t rows_of(Mode m) { return 16 * tiles_of(m) * (together(m) ? kWaves : 1); }

// Wavefronts per SIMD that the registers are held to.
template <int D, Mode M>
constexpr int waves_per_simd() {
  return D == 256 ? 1 : D == 64 && tiles_of(M) == 1 ? 3 : 2;
}

template <class Room>
__device__ __forceinline__ Room* joined_room() {
  __shared__ __align__(16) Room room;
  return &room;
}

template <class T, int D, Mode M, Access A, Mode Kernel, class Limit>
__device__ __forceinline__ void run_range(const Args& a, const Range& range, float (*shares)[16], Limit&& limit) {
  using Ops = Operands<T, D, A>;
  constexpr int QT = tiles_of(M);
  Rows<Ops, QT, together(M)> rows;
  const uint32_t first = together(M) ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 16 * QT : 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) rows.limit[t] = limit(min(first + 16 * t + threadIdx.x % 16, range.count - 1));
  if constexpr (together(M)) {
    run_together<D, QT, A>(a, range, rows, shares);
  } else if constexpr (together(Kernel)) {  // the stages are free: no block runs both
    static_assert(sizeof(Joined<Ops, QT>) <= 2 * Stage<D>::kBytes, "joined outputs outgrow a stage");
    run_apart<T, D, QT, A>(a, range, rows, *reinterpret_cast<Joined<Ops, QT>*>(stage_room<D, 0>()), shares);
  } else {
    run_apart<T, D, QT, A>(a, range, rows, *joined_room<Joined<Ops, QT>>(), shares);
  }
}

// Mode P against the prefix, O against an own cache: a sequence of a decode
// step has few rows where the batch has many.
template <class T, int D, Mode P, Mode O, Access A>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(waves_per_simd<D, P>())))
void k_ranges(const Args a) {
  __shared__ float shares[kWaves * 32][16];
  Range range;
  uint32_t group, tile;
  if (blockIdx.x < a.prefix_blocks) {
    if (!block_task(blockIdx.x, a.kv_heads * a.prefix_splits, a.prefix_tiles, group, tile)) return;
    range.kvh = group / a.prefix_splits;
    range.slot = group % a.prefix_splits;
    range.begin = range.slot * a.prefix_each;
    range.end = range.least = min(range.begin + a.prefix_each, a.prefix);
    range.first = tile * rows_of(P);
    range.count = min(a.all_rows - range.first, rows_of(P));
    range.scores = nullptr;
    const uint64_t at = static_cast<uint64_t>(range.kvh) * a.width * sizeof(T);
    range.keys = static_cast<const char*>(a.prefix_key) + at;
    range.values = static_cast<const char*>(a.prefix_value) + at;
    run_range<T, D, P, A, P>(a, range, shares, [&](uint32_t) { return range.end; });
    return;
  }
  if (!block_task(blockIdx.x - a.prefix_blocks, a.batch * a.kv_heads * a.own_splits, a.own_tiles, group, tile)) return;
  const uint32_t split = group % a.own_splits, b = group / a.own_splits / a.kv_heads;
  range.kvh = group / a.own_splits % a.kv_heads;
  range.slot = a.prefix_splits + split;
  const uint32_t n = length_of(a, b), each = range_keys(n, a.own_splits);
  range.begin = split * each;
  if (range.begin >= n) return;
  const uint32_t first = tile * rows_of(O);
  auto limit = [&](uint32_t row) { return visible(n, a.rows, (first + row) / a.group); };
  range.count = min(a.seq_rows - first, rows_of(O));
  range.end = min(range.begin + each, n);
  range.least = min(range.end, limit(0));
  range.end = min(range.end, max(range.begin, limit(range.count - 1)));  // no row sees further
  range.first = b * a.seq_rows + first;
  range.scores = a.scores ? a.scores + ((static_cast<uint64_t>(b) * a.kv_heads + range.kvh) * a.seq_rows + first) * a.score_pitch : nullptr;
  const uint64_t stride = static_cast<uint64_t>(a.kv_heads) * a.width;
  const uint64_t at = (static_cast<uint64_t>(b) * a.capacity * stride + static_cast<uint64_t>(range.kvh) * a.width) * sizeof(T);
  range.keys = static_cast<const char*>(a.key) + at;
  range.values = static_cast<const char*>(a.value) + at;
  run_range<T, D, O, A, P>(a, range, shares, limit);
}

// The ranges that hold something of one row, in order.
struct RowRanges {
  uint32_t own, seen;
  uint64_t step, base;
  uint32_t before;
  __device__ __forceinline__ RowRanges(const Args& a, uint32_t kvh, uint32_t row, uint32_t n) {
    seen = visible(n, a.rows, row % a.seq_rows / a.group);
    before = a.prefix_splits;
    own = seen ? (seen - 1) / range_keys(n, a.own_splits) + 1 : 0;  // ranges past the last key it sees hold nothing of it
    step = static_cast<uint64_t>(a.kv_heads) * a.all_rows;
    base = static_cast<uint64_t>(kvh) * a.all_rows + row;
  }
  __device__ __forceinline__ uint32_t count() const { return before + own; }
  __device__ __forceinline__ uint64_t place(uint32_t r) const { return r * step + base; }
  // Maximum (as subtracted) and sum over all ranges, by one wavefront.
  __device__ __forceinline__ float2 whole(const float2* part) const {
    const uint32_t lane = threadIdx.x % 64;
    const float2 own_part = lane < count() ? part[place(lane)] : make_float2(-INFINITY, 0.0f);
    float top = own_part.x;
    for (uint32_t r = lane + 64; r < count(); r += 64) top = fmaxf(top, part[place(r)].x);
    const float from = reference_of(wave_max(top));
    float total = exp2_of(own_part.x - from) * own_part.y;
    for (uint32_t r = lane + 64; r < count(); r += 64) {
      const float2 p = part[place(r)];
      total = fma_rn(exp2_of(p.x - from), p.y, total);
    }
#pragma unroll
    for (int off = 32; off; off /= 2) total = total + __shfl_xor(total, off);
    return make_float2(from, total);
  }
};

constexpr int kFewRanges = 8;

// Joins the ranges of one row (4 us where there are few rows, most of it launch
// and the wait for the first loads; 14 us for 16,384 rows of four ranges, 34
// MB).  D / 4 lanes hold a row of a range, four features each, so a wavefront
// reads 256 / D ranges at a time and a workgroup of W = 4 four times as many:
// the loads of a row are a few deep.
template <class T, int D, int W>
__device__ __forceinline__ void join_row(const Args& a, uint32_t task, f32x4 (*room)[64]) {
  constexpr int kLanes = D / 4, kAtOnce = W * 64 / kLanes;
  const int lane = threadIdx.x % 64, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t kvh = task % a.kv_heads, row = task / a.kv_heads;
  const uint32_t f = lane % kLanes * 4, first = wave * (64 / kLanes) + lane / kLanes;
  // What the first ranges left is read before the length says which of them hold
  // something: one wait and not three.
  const uint32_t all = a.prefix_splits + a.own_splits;
  const uint64_t step = static_cast<uint64_t>(a.kv_heads) * a.all_rows, base = static_cast<uint64_t>(kvh) * a.all_rows + row;
  const float* sums = a.sums + (f < a.pitch ? f : 0);
  constexpr int kAhead = W == 1 ? (kFewRanges + kAtOnce - 1) / kAtOnce : 4;
  f32x4 ahead[kAhead];
#pragma unroll
  for (int m = 0; m < kAhead; ++m) {
    ahead[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (static_cast<uint32_t>(m) * kAtOnce < all)
      ahead[m] = *reinterpret_cast<const f32x4*>(sums + (min(m * kAtOnce + first, all - 1) * step + base) * a.pitch);
  }
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float share, const f32x4& v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fma_rn(share, v[e], acc[e]);
  };
  float2 whole;
  uint32_t seen;
  if constexpr (W == 1) {  // at most kFewRanges: every lane has all maxima and sums
    float2 part[kFewRanges];
#pragma unroll
    for (int r = 0; r < kFewRanges; ++r) {
      part[r] = make_float2(-INFINITY, 0.0f);
      if (static_cast<uint32_t>(r) < all) part[r] = a.part[r * step + base];
    }
    const RowRanges ranges(a, kvh, row, length_of(a, row / a.seq_rows));
    seen = ranges.seen;
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < kFewRanges; ++r) {
      if (static_cast<uint32_t>(r) >= ranges.count()) part[r] = make_float2(-INFINITY, 0.0f);
      top = fmaxf(top, part[r].x);
    }
    whole = make_float2(reference_of(top), 0.0f);
#pragma unroll
    for (int r = 0; r < kFewRanges; ++r) {
      const float share = exp2_of(part[r].x - whole.x);
      whole.y = fma_rn(share, part[r].y, whole.y);
      if (r % kAtOnce == static_cast<int>(first) && static_cast<uint32_t>(r) < ranges.count()) add(share, ahead[r / kAtOnce]);
    }
  } else {
    const RowRanges ranges(a, kvh, row, length_of(a, row / a.seq_rows));
    seen = ranges.seen;
    whole = ranges.whole(a.part);
    auto share = [&](uint32_t r) { return exp2_of(a.part[r * step + base].x - whole.x); };
#pragma unroll
    for (int m = 0; m < kAhead; ++m) {
      const uint32_t r = m * kAtOnce + first;
      if (r < ranges.count()) add(share(r), ahead[m]);
    }
#pragma unroll 4
    for (uint32_t r = kAhead * kAtOnce + first; r < ranges.count(); r += kAtOnce)
      add(share(r), *reinterpret_cast<const f32x4*>(sums + (r * step + base) * a.pitch));
  }
#pragma unroll
  for (int off = kLanes; off < 64; off *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] + __shfl_xor(acc[e], off);
  if constexpr (W > 1) {
    __syncthreads();  // the row before is read
    room[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < W; ++w) acc = acc + room[w][lane];
  }
  if (a.whole && lane == 0) a.whole[base] = make_float2(whole.x, 1.0f / whole.y);
  if (lane >= kLanes) return;
  T* out = static_cast<T*>(a.out) + query_offset(a, row, kvh);
  const bool none = a.prefix + seen == 0;
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  } four;
#pragma unroll
  for (int e = 0; e < 4; ++e) store_elem(four.v, e, none ? 0.0f : acc[e] / whole.y);
  if (a.width % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % sizeof four == 0) {
    if (f < a.width) *reinterpret_cast<Four*>(out + f) = four;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (f + e < a.width) out[f + e] = four.v[e];
  }
}

// Weights of up to 16 rows from their stored scores: a thread sums four
// keys' weights over the rows.
constexpr int kWeightKeys = 4 * kThreads;
__device__ __forceinline__ void add_weights(const Args& a, uint32_t block, float2* stats) {
  const uint32_t blocks = a.capacity / kWeightKeys + (a.capacity % kWeightKeys != 0);
  const uint32_t kvh = block % a.kv_heads, b = block / a.kv_heads / blocks;
  const uint32_t key0 = block / a.kv_heads % blocks * kWeightKeys;
  const uint32_t n = length_of(a, b);
  if (key0 >= n) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  for (uint32_t r = wave; r < a.seq_rows; r += kWaves) {
    const float2 whole = RowRanges(a, kvh, b * a.seq_rows + r, n).whole(a.part);
    if (threadIdx.x % 64 == 0) stats[r] = make_float2(whole.x, 1.0f / whole.y);
  }
  __syncthreads();
  const float factor = factor_of(*a.scale);
  const uint32_t key = key0 + 4 * threadIdx.x;
  if (key >= n) return;
  const uint64_t head = static_cast<uint64_t>(b) * a.kv_heads + kvh;
  const float* scores = a.scores + head * a.seq_rows * a.score_pitch + key;
  float sum[4] = {};
#pragma unroll 4
  for (uint32_t r = 0; r < a.seq_rows; ++r) {
    const f32x4 s = *reinterpret_cast<const f32x4*>(scores + static_cast<uint64_t>(r) * a.score_pitch);
    const uint32_t seen = visible(n, a.rows, r / a.group);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (key + e < seen) sum[e] = fma_rn(exp2_of(fma_rn(s[e], factor, -stats[r].x)), stats[r].y, sum[e]);
  }
  const uint64_t at = head * a.capacity + key;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (key + e < n) a.weights_out[at + e] = a.weights[at + e] + sum[e];
}

template <class T, int D, int W>
__global__ __launch_bounds__(kThreads) void k_join(const Args a, uint32_t join_blocks) {
  __shared__ f32x4 room[W == 1 ? 1 : W][64];
  __shared__ float2 stats[16];
  if (blockIdx.x < join_blocks) {
    constexpr uint32_t kTasks = W == 1 ? kWaves : 1;  // of a block at once
    uint32_t task = blockIdx.x * kTasks + (W == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
    for (; task < a.kv_heads * a.all_rows; task += join_blocks * kTasks) join_row<T, D, W>(a, task, room);
  } else {
    add_weights(a, blockIdx.x - join_blocks, stats);
  }
}

// Weights of more rows: the scores again, a workgroup per 16 NT keys, held in
// registers (2048 rows over 4096 keys, 8 KV heads: 42 us, 8 of products; the
// query loads cost 15, the exponentials 2).  The wavefronts walk every fourth
// tile of the rows that see them; a lane sums its keys over its rows, then the
// lanes and the wavefronts add up in a fixed order.  Every key has one owner:
// no atomics.  NT = 8 halves the query loads but leaves one workgroup to a
// compute unit: 35 us at this size, but 34 instead of 24 over 2048 keys.
template <class T, int D, Access A>
__global__ __launch_bounds__(kThreads) void k_weights(const Args a) {
  using Ops = Operands<T, D, A>;
  constexpr int NT = D == 256 ? 2 : 4, kKeys = 16 * NT;
  __shared__ float sums[kWaves][kKeys];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int i16 = lane % 16, g = lane / 16;
  const uint32_t blocks = a.capacity / kKeys + (a.capacity % kKeys != 0);
  const uint32_t kvh = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads / blocks;
  const uint32_t key0 = blockIdx.x / a.kv_heads % blocks * kKeys;
  const uint32_t n = length_of(a, b);
  if (key0 >= n) return;
  const uint32_t stride = a.kv_heads * a.width * sizeof(T);
  const char* keys = static_cast<const char*>(a.key) + (static_cast<uint64_t>(b) * a.capacity + key0) * stride +
                     static_cast<uint64_t>(kvh) * a.width * sizeof(T);
  const float scale = *a.scale, factor = factor_of(scale);
  u32x4 k[NT][Ops::kSteps];
#pragma unroll
  for (int u = 0; u < NT; ++u) Ops::load_row(keys, min(16u * u + i16, n - key0 - 1) * stride + 16 * g, g, a.width, k[u]);
  float sum[NT][4] = {};
  // Row j sees key k from j = (k + rows - n) group on: n - rows + j / group + 1 > k.
  auto first_row = [&](uint32_t key) {
    return static_cast<uint64_t>(key) + a.rows > n ? (key + a.rows - n) * a.group : 0u;
  };
  // The lane's row of a tile, 16 kWaves rows further every time, and its operands;
  // past the last row they repeat it.
  uint32_t r0 = first_row(key0) / 16 * 16 + 16 * wave;
  uint32_t position = (r0 + i16) / a.group, in_group = (r0 + i16) % a.group;
  const uint32_t position_step = 16 * kWaves / a.group, group_step = 16 * kWaves % a.group;
  u32x4 q[1][Ops::kSteps];
  float2 whole;
  auto load_rows = [&] {
    const bool real = position < a.rows;
    const uint32_t at = real ? position : a.rows - 1, of = real ? in_group : a.group - 1;
    const uint64_t row = static_cast<uint64_t>(b) * a.rows + at;
    const T* src = static_cast<const T*>(a.query) + (row * a.q_heads + kvh * a.group + of) * a.width;
    Ops::load_row(reinterpret_cast<const char*>(src), 16 * g, g, a.width, q[0]);
    whole = a.whole[static_cast<uint64_t>(kvh) * a.all_rows + row * a.group + of];
    position += position_step;
    in_group += group_step;
    if (in_group >= a.group) {
      in_group -= a.group;
      ++position;
    }
  };
  f32x4 s[1][NT];
  float from, inverse;
  auto next_scores = [&] {
    take_sign<Ops>(scale, q[0]);
    Ops::scores(k, q, s);
    from = -whole.x;
    inverse = whole.y;
    load_rows();
  };
  if (r0 < a.seq_rows) load_rows();
  // Tiles in which some row does not see some key, or is past the last.
  const uint32_t all_see = first_row(min(key0 + kKeys, n) - 1), step = 16 * kWaves;
  uint32_t need[NT][4];
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t key = key0 + 16 * u + 4 * g + r;
      need[u][r] = key < n ? first_row(key) : 0xffffffffu;
    }
  auto masked = [&] {
    next_scores();
    const uint32_t row = r0 + i16 < a.seq_rows ? r0 + i16 : 0;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r0 + i16 < a.seq_rows && row >= need[u][r])
          sum[u][r] = fma_rn(exp2_of(fma_rn(s[0][u][r], factor, from)), inverse, sum[u][r]);
  };
  for (; r0 < a.seq_rows && (r0 < all_see || key0 + kKeys > n); r0 += step) masked();
  // Whole tiles: the next one's products beside this one's exponentials.
  if (r0 + 16 <= a.seq_rows) {
    next_scores();
    for (; r0 + step + 16 <= a.seq_rows; r0 += step) {
      f32x4 now[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) now[u] = s[0][u];
      const float from_now = from, inverse_now = inverse;
      next_scores();
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[u][r] = fma_rn(exp2_of(fma_rn(now[u][r], factor, from_now)), inverse_now, sum[u][r]);
    }
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[u][r] = fma_rn(exp2_of(fma_rn(s[0][u][r], factor, from)), inverse, sum[u][r]);
    r0 += step;
  }
  if (r0 < a.seq_rows) masked();
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int off = 8; off; off /= 2) sum[u][r] = sum[u][r] + __shfl_xor(sum[u][r], off);
      if (i16 == 0) sums[wave][16 * u + 4 * g + r] = sum[u][r];
    }
  __syncthreads();
  const uint32_t key = key0 + threadIdx.x;
  if (threadIdx.x < kKeys && key < n) {
    const uint64_t at = (static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.capacity + key;
    const float* own = &sums[0][threadIdx.x];
    a.weights_out[at] = a.weights[at] + ((own[0] + own[kKeys]) + (own[2 * kKeys] + own[3 * kKeys]));
  }
}

// ------------------------------------------------------------------- the host
constexpr const char* kTooMany = "too many workgroups";
// A launch's threads are counted in 32 bits; two kinds of blocks share one.
constexpr uint64_t kMostBlocks = (1u << 23) - 8;

uint64_t product(std::initializer_list<uint64_t> factors, uint64_t most, const char* what) {
  uint64_t p = 1;
  for (uint64_t f : factors) {
    require(f == 0 || p <= most / f, what, DL_LENGTH_ERROR);
    p *= f;
  }
  return p;
}

// Row tiles per workgroup, ranges and workspace of one call.
struct Layout {
  Args args{};
  Mode prefix_mode = Mode::kApart, own_mode = Mode::kApart;
  int features = 64;            // D
  bool weighted = false, stored = false;
  uint64_t part_bytes = 0, sums_bytes = 0, whole_bytes = 0, score_bytes = 0;
  uint32_t own_blocks = 0, weight_blocks = 0;

  uint64_t bytes() const { return part_bytes + sums_bytes + whole_bytes + score_bytes; }
  void set_modes(Mode prefix, Mode own) {
    prefix_mode = prefix;
    own_mode = own;
    args.prefix_tiles = static_cast<uint32_t>(ceil_div(args.all_rows, rows_of(prefix)));
    args.own_tiles = static_cast<uint32_t>(ceil_div(args.seq_rows, rows_of(own)));
  }
  void count_blocks() {
    auto blocks = [&](std::initializer_list<uint64_t> groups, uint64_t tiles) {
      const uint64_t rounded = ceil_div(product(groups, kMostBlocks, kTooMany), 8) * 8;
      return static_cast<uint32_t>(product({rounded, tiles}, kMostBlocks, kTooMany));
    };
    args.prefix_blocks = blocks({args.kv_heads, args.prefix_splits}, args.prefix_tiles);
    own_blocks = blocks({args.batch, args.kv_heads, args.own_splits}, args.own_tiles);
    const uint64_t keys = stored ? kWeightKeys : features == 256 ? 32 : 64;  // per block
    weight_blocks = static_cast<uint32_t>(
        weighted ? product({args.batch, args.kv_heads, ceil_div(args.capacity, keys)}, kMostBlocks, kTooMany) : 0);
  }
};

// `pieces`: the rows are 16-byte pieces of BF16, which tiles can share.  Others
// run apart: FP32 is bound by the FP32 matrix rate, not by its loads.
Layout layout_of(const dl_batch_shape* shape, uint64_t prefix, bool weighted, bool pieces) {
  check_shape(shape);
  require(prefix <= kMostKeys, "prefix too long", DL_LENGTH_ERROR);
  require(shape->width <= 256, "head width above 256", DL_LENGTH_ERROR);
  Layout l;
  Args& a = l.args;
  a.batch = static_cast<uint32_t>(shape->batch);
  a.rows = static_cast<uint32_t>(shape->rows);
  a.q_heads = static_cast<uint32_t>(shape->query_heads);
  a.kv_heads = static_cast<uint32_t>(shape->kv_heads);
  a.group = a.q_heads / a.kv_heads;
  a.width = static_cast<uint32_t>(shape->width);
  a.prefix = static_cast<uint32_t>(prefix);
  a.capacity = static_cast<uint32_t>(shape->capacity);
  constexpr const char* kRows = "too many query rows";
  a.seq_rows = static_cast<uint32_t>(product({a.rows, a.group}, 1u << 30, kRows));
  a.all_rows = static_cast<uint32_t>(product({a.seq_rows, a.batch}, 1u << 30, kRows));
  product({a.all_rows, a.kv_heads}, 1u << 30, kRows);
  l.features = a.width <= 64 ? 64 : a.width <= 128 ? 128 : 256;
  l.weighted = weighted;
  l.stored = weighted && a.seq_rows <= 16;
  // Few rows: every wavefront has them all.  More: 64 a workgroup, or 128 where
  // those fill the chip (D = 256 has no registers for two tiles a wavefront).
  auto mode_of = [&](uint32_t rows, uint64_t ranges) {
    if (rows <= 32 || !pieces) return Mode::kApart;
    return l.features < 256 && rows > 64 && ceil_div(rows, 128) * ranges >= 512 ? Mode::kTogether2 : Mode::kTogether1;
  };
  const Mode own = mode_of(a.seq_rows, uint64_t{a.batch} * a.kv_heads * ceil_div(a.capacity, kRound));
  const Mode all = prefix ? mode_of(a.all_rows, a.kv_heads * ceil_div(prefix, kRound)) : own;
  l.set_modes(all, a.seq_rows <= 32 ? Mode::kApart : all);
  // Ranges: as many workgroups as the chip holds at once, each with whole rounds
  // of keys.  Lengths lie on the device, so a cache counts with all its slots: the
  // more of them are free, the fewer ranges are left for the prefix (64 sequences
  // of up to 1000 rows over 32768 keys, caches of 1008 slots 88 us, 2008 106, 8008
  // 224, 32008 814).
  const uint64_t held = 256 * (l.features == 256 ? 1 : l.features == 64 ? 3 : 2);
  const double work = static_cast<double>(a.kv_heads) *
                      (static_cast<double>(a.prefix_tiles) * a.prefix +
                       static_cast<double>(a.batch) * a.own_tiles * a.capacity);
  const uint64_t each = std::max<uint64_t>(kRound, static_cast<uint64_t>(work / held));
  if (prefix) {
    a.prefix_each = range_keys(a.prefix, static_cast<uint32_t>(ceil_div(prefix, each)));
    a.prefix_splits = static_cast<uint32_t>(ceil_div(prefix, a.prefix_each));
  }
  a.own_splits = static_cast<uint32_t>(ceil_div(a.capacity, each));
  l.count_blocks();
  a.pitch = (a.width + 3) / 4 * 4;
  a.score_pitch = (a.capacity + 31) / 32 * 32;
  constexpr const char* kLarge = "workspace too large";
  constexpr uint64_t kMost = UINT64_MAX / 8;
  auto room = [&](std::initializer_list<uint64_t> factors) { return ceil_div(product(factors, kMost, kLarge), 256) * 256; };
  const uint64_t entries = product({uint64_t{a.prefix_splits} + a.own_splits, a.kv_heads, a.all_rows}, kMost, kLarge);
  l.part_bytes = room({entries, 8});
  l.sums_bytes = room({entries, a.pitch, 4});
  l.whole_bytes = weighted && !l.stored ? room({a.kv_heads, a.all_rows, 8}) : 0;
  l.score_bytes = l.stored ? room({a.kv_heads, a.all_rows, a.score_pitch, 4}) : 0;
  return l;
}

// Enough for either storage type and any alignment.
uint64_t workspace_of(const dl_batch_shape* shape, uint64_t prefix, bool weighted) {
  return std::max(layout_of(shape, prefix, weighted, false).bytes(), layout_of(shape, prefix, weighted, true).bytes());
}

template <class T, int D, Access A>
void launch(hipStream_t s, const Layout& l) {
  const Args& a = l.args;
  const unsigned blocks = a.prefix_blocks + l.own_blocks;  // below 2^24: 2^32 threads
  auto run = [&](auto prefix, auto own) {
    k_ranges<T, D, decltype(prefix)::value, decltype(own)::value, A><<<blocks, kThreads, 0, s>>>(a);
  };
  using Apart = std::integral_constant<Mode, Mode::kApart>;
  auto run_own = [&](auto prefix) {
    if (l.own_mode == Mode::kApart)
      run(prefix, Apart{});
    else
      run(prefix, prefix);
  };
  if (l.prefix_mode == Mode::kApart) {
    run(Apart{}, Apart{});
  } else if constexpr (A != Access::kElements && std::is_same_v<T, uint16_t>) {
    if (l.prefix_mode == Mode::kTogether1)
      run_own(std::integral_constant<Mode, Mode::kTogether1>{});
    else if constexpr (D != 256)
      run_own(std::integral_constant<Mode, Mode::kTogether2>{});
  }
  // A workgroup per row where there are many ranges, else a wavefront.
  const uint32_t tasks = a.kv_heads * a.all_rows;
  const uint32_t fused = l.stored ? l.weight_blocks : 0;
  constexpr uint32_t kJoinBlocks = 1u << 22;
  if (a.prefix_splits + a.own_splits > kFewRanges) {
    const uint32_t blocks_of_rows = std::min(tasks, kJoinBlocks);
    k_join<T, D, 4><<<blocks_of_rows + fused, kThreads, 0, s>>>(a, blocks_of_rows);
  } else {
    const uint32_t blocks_of_rows = std::min(static_cast<uint32_t>(ceil_div(tasks, kWaves)), kJoinBlocks);
    k_join<T, D, 1><<<blocks_of_rows + fused, kThreads, 0, s>>>(a, blocks_of_rows);
  }
  if (l.weighted && !l.stored) k_weights<T, D, A><<<l.weight_blocks, kThreads, 0, s>>>(a);
}

template <class T, int D>
void launch_access(hipStream_t s, const Layout& l, Access access) {
  if (access == Access::kWhole)
    launch<T, D, Access::kWhole>(s, l);
  else if (access == Access::kPieces)
    launch<T, D, Access::kPieces>(s, l);
  else
    launch<T, D, Access::kElements>(s, l);
}

template <class T>
void launch_width(hipStream_t s, const Layout& l, Access access) {
  if (l.features == 64)
    launch_access<T, 64>(s, l, access);
  else if (l.features == 128)
    launch_access<T, 128>(s, l, access);
  else
    launch_access<T, 256>(s, l, access);
}

struct Operation {
  const void *query, *prefix_key, *prefix_value, *key, *value, *weights;
  const uint64_t* lengths;
  float* weights_out;
  void* output;
  const float* scale;
  void* workspace;
  uint64_t workspace_bytes;
};

void submit(dl_queue* queue, int dtype, const dl_batch_shape* shape, uint64_t prefix, const Operation& o, bool weighted) {
  require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
  check_shape(shape);
  const bool pieces =
      whole_pieces(shape, dtype == DL_BF16 ? 2 : 4, {o.query, o.prefix_key, o.prefix_value, o.key, o.value});
  Layout l = layout_of(shape, prefix, weighted, pieces && dtype == DL_BF16);
  const Access access = !pieces ? Access::kElements
                        : static_cast<int>(l.args.width) == l.features ? Access::kWhole
                                                                       : Access::kPieces;
  require(o.query && o.key && o.value && o.lengths && o.output && o.scale, "null operand");
  require(prefix == 0 || (o.prefix_key && o.prefix_value), "null prefix operand");
  require(!weighted || (o.weights && o.weights_out), "null weights");
  require(o.workspace != nullptr && reinterpret_cast<uintptr_t>(o.workspace) % 16 == 0, "workspace null or not 16-byte aligned");
  require(o.workspace_bytes >= workspace_of(shape, prefix, weighted), "workspace too small", DL_LENGTH_ERROR);
  enter(queue);
  Args& a = l.args;
  a.query = o.query;
  a.prefix_key = o.prefix_key;
  a.prefix_value = o.prefix_value;
  a.key = o.key;
  a.value = o.value;
  a.lengths = o.lengths;
  a.scale = o.scale;
  a.out = o.output;
  char* room = static_cast<char*>(o.workspace);
  a.part = reinterpret_cast<float2*>(room);
  a.sums = reinterpret_cast<float*>(room + l.part_bytes);
  char* for_weights = room + l.part_bytes + l.sums_bytes;
  if (l.whole_bytes) a.whole = reinterpret_cast<float2*>(for_weights);
  if (l.score_bytes) a.scores = reinterpret_cast<float*>(for_weights);
  a.weights = static_cast<const float*>(o.weights);
  a.weights_out = o.weights_out;
  if (dtype == DL_BF16)
    launch_width<uint16_t>(queue->stream, l, access);
  else
    launch_width<float>(queue->stream, l, access);
  check_launch(queue, weighted ? "attention_weighted" : "attention_shared");
}

}  // namespace
}  // namespace dl::batch

using dl::guard;
using dl::require;

extern "C" {

int dl_attention_shared_bytes(const dl_batch_shape* shape, uint64_t prefix, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::batch::workspace_of(shape, prefix, false);
  });
}

int dl_attention_weighted_bytes(const dl_batch_shape* shape, uint64_t prefix, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::batch::workspace_of(shape, prefix, true);
  });
}

int dl_attention_shared(dl_queue* queue, int dtype, const dl_batch_shape* shape, const void* query,
                        const void* prefix_key, const void* prefix_value, uint64_t prefix, const void* key,
                        const void* value, const uint64_t* lengths, void* output, const float* scale, void* workspace,
                        uint64_t workspace_bytes) {
  return guard([&] {
    dl::batch::submit(queue, dtype, shape, prefix,
                      {query, prefix_key, prefix_value, key, value, nullptr, lengths, nullptr, output, scale, workspace,
                       workspace_bytes},
                      false);
  });
}

int dl_attention_weighted(dl_queue* queue, int dtype, const dl_batch_shape* shape, const void* query,
                          const void* prefix_key, const void* prefix_value, uint64_t prefix, const void* key,
                          const void* value, const uint64_t* lengths, const float* weights, float* weights_out,
                          void* output, const float* scale, void* workspace, uint64_t workspace_bytes) {
  return guard([&] {
    dl::batch::submit(queue, dtype, shape, prefix,
                      {query, prefix_key, prefix_value, key, value, weights, lengths, weights_out, output, scale, workspace,
                       workspace_bytes},
                      true);
  });
}

}  // extern "C"
