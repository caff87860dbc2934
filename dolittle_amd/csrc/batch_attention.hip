// Attention of a batch of sequences over a prefix that they share and caches
// of their own, and the weight that every cached key received.  No reference
// counterpart: the reference decodes one sequence over one contiguous cache.
//
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// over the prefix's keys and, for new row i of a sequence that holds n rows,
// its own keys j < n - rows + i + 1.  A row without a key is zeros.  A key
// that a row does not see has no effect on it, whatever the key's bytes are.
//
// Split.  All rows of a KV head (every sequence's, every new row's, the heads
// of the group) are one matrix against the prefix, so the prefix is read once
// per 16 QT rows and not once per sequence.  A workgroup takes 16 QT rows and a
// range of keys of one source (the prefix, or one sequence's cache); its four
// wavefronts take every fourth step of keys and keep a running maximum, sum
// and output of their own, joined at the end.  k_join joins the ranges.
//
// Matrix operands, without a pass through LDS.  Scores are computed as K Q^T:
// the first operand is K with a lane per key, so K is loaded straight from its
// rows, and the result leaves a lane with scores of one row and the keys that
// the second product's P^T operand wants from it.  That product is V^T P^T:
// a lane loads C = D / 16 neighbouring features of the keys it contracts, and
// since any 16 features may form a matrix tile, tile j takes feature j of each
// lane's C: the transposition is a byte permute of two registers (BF16) or
// nothing (FP32).
//
// BF16 storage rounds P to BF16 (8 bits, relative 2^-9) for the product with V;
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
// A maximum is raised only when a score passes it by this much: exponentials
// stay below e^8, and most steps rescale nothing.
constexpr float kSlack = 8.0f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// How rows are read: whole 16-byte pieces up to D features; whole pieces up to
// the width; or element by element, for widths or operands that are not
// 16-byte aligned.
enum class Access { kWhole, kPieces, kElements };

// N consecutive elements from `at` on as 32-bit words; zeros past the width.
template <class T, int N, Access A>
__device__ __forceinline__ void load_words(const T* row, int at, int width, uint32_t* out) {
  constexpr int kWords = N * sizeof(T) / 4;
  if constexpr (A == Access::kElements) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        out[i] = at + i < width ? __float_as_uint(row[at + i]) : 0u;
      } else {
        const uint32_t lo = at + 2 * i < width ? row[at + 2 * i] : 0u;
        const uint32_t hi = at + 2 * i + 1 < width ? row[at + 2 * i + 1] : 0u;
        out[i] = lo | (hi << 16);
      }
    }
  } else if constexpr (kWords == 2) {
    const u32x2 v = A == Access::kWhole || at < width ? *reinterpret_cast<const u32x2*>(row + at) : u32x2{};
    out[0] = v.x;
    out[1] = v.y;
  } else {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const u32x4 v =
          A == Access::kWhole || at + i * kPer < width ? *reinterpret_cast<const u32x4*>(row + at + i * kPer) : u32x4{};
      out[4 * i] = v.x;
      out[4 * i + 1] = v.y;
      out[4 * i + 2] = v.z;
      out[4 * i + 3] = v.w;
    }
  }
}

// exp(v) by the hardware's exp2; v <= kSlack or NaN.
__device__ __forceinline__ float fast_exp(float v) { return __builtin_amdgcn_exp2f(v * kLog2e); }
// The value subtracted from scores: 0 while no score is finite, so that
// exp(-inf - m) is 0 and not NaN.
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.0f : m; }

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
  struct Keys {
    u32x4 v[kTiles][kSteps];
  };
  struct Values {
    uint32_t v[kValueRows][C / 2];
  };
  // A row's features (4 s + g) 8 .. of product step s.
  static __device__ __forceinline__ void load_row(const T* row, int g, int width, u32x4* out) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) load_words<T, 8, A>(row, (4 * s + g) * 8, width, reinterpret_cast<uint32_t*>(&out[s]));
  }
  // The key of value row r in the order in which P holds them.
  static __device__ __forceinline__ int value_key(int g, int r) { return (r / 4) * 16 + 4 * g + r % 4; }
  static __device__ __forceinline__ void scores(const u32x4* k, const u32x4* q, f32x4& s) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[i]), __builtin_bit_cast(bf16x8, q[i]), s, 0,
                                                  0, 0);
  }
  // The first operand of feature tile j.
  static __device__ __forceinline__ bf16x8 value_tile(const Values& v, int j) {
    u32x4 w;
    const uint32_t pick = j % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int p = 0; p < 4; ++p) w[p] = __builtin_amdgcn_perm(v.v[2 * p + 1][j / 2], v.v[2 * p][j / 2], pick);
    return __builtin_bit_cast(bf16x8, w);
  }
  template <int QT>
  static __device__ __forceinline__ void products(const Values& v, const f32x4 (&p)[QT][kTiles], f32x4 (&o)[QT][C]) {
    bf16x8 b[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) b[t][e] = static_cast<__bf16>(p[t][e / 4][e % 4]);
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
  struct Keys {
    u32x4 v[kTiles][kSteps];
  };
  struct Values {
    uint32_t v[kValueRows][C];
  };
  static __device__ __forceinline__ void load_row(const T* row, int g, int width, u32x4* out) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) load_words<T, 4, A>(row, (4 * s + g) * 4, width, reinterpret_cast<uint32_t*>(&out[s]));
  }
  static __device__ __forceinline__ int value_key(int g, int r) { return 4 * g + r; }
  static __device__ __forceinline__ void scores(const u32x4* k, const u32x4* q, f32x4& s) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i][e]), __uint_as_float(q[i][e]), s, 0, 0, 0);
  }
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
__host__ __device__ inline uint32_t ranges_of(uint32_t keys, uint32_t splits) {
  const uint32_t each = range_keys(keys, splits);
  return keys ? keys / each + (keys % each != 0) : 0;
}

struct Args {
  const void *query, *prefix_key, *prefix_value, *key, *value;
  const uint64_t* lengths;
  const float* scale;
  void* out;
  float2* part;  // [ranges][kv head][row]: maximum, sum
  float* sums;   // [ranges][kv head][row][width]: unnormalised output
  float2* whole; // [kv head][row]: maximum, 1 / sum; null unless the weights are wanted
  const float* weights;
  float* weights_out;
  uint32_t batch, rows, q_heads, kv_heads, group, width, prefix, capacity;
  uint32_t seq_rows, all_rows;          // rows of one sequence and of the batch, per KV head
  uint32_t prefix_splits, own_splits;   // most ranges of a source
  uint32_t prefix_blocks, prefix_tiles, own_tiles;
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

template <class T, int D, int QT, Access A>
__global__ __launch_bounds__(kThreads) void k_ranges(const Args a) {
  using Ops = Operands<T, D, A>;
  constexpr int C = Ops::C, KT = Ops::kKeys, kTiles = Ops::kTiles;
  __shared__ __align__(16) f32x4 joined[QT == 1 ? 4 : 2 * QT][C][64];
  __shared__ float2 stats[2][QT][16];
  __shared__ float masked_p[kWaves][KT][16];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int i16 = lane % 16, g = lane / 16;

  // The rows [first, first + count) of the batch's per KV head, the keys
  // [begin, end) of a source, and where the range's result goes.
  uint32_t first, count, kvh, begin, end, slot, group, tile;
  uint32_t limit[QT], least;
  const T *keys, *values;
  const uint32_t id = blockIdx.x;
  if (id < a.prefix_blocks) {
    if (!block_task(id, a.kv_heads * a.prefix_splits, a.prefix_tiles, group, tile)) return;
    kvh = group % a.kv_heads;
    slot = group / a.kv_heads;
    const uint32_t each = range_keys(a.prefix, a.prefix_splits);
    begin = slot * each;
    if (begin >= a.prefix) return;
    end = min(begin + each, a.prefix);
    first = tile * 16 * QT;
    count = min(a.all_rows - first, 16u * QT);
    keys = static_cast<const T*>(a.prefix_key);
    values = static_cast<const T*>(a.prefix_value);
    least = end;
#pragma unroll
    for (int t = 0; t < QT; ++t) limit[t] = end;
  } else {
    if (!block_task(id - a.prefix_blocks, a.batch * a.kv_heads * a.own_splits, a.own_tiles, group, tile)) return;
    kvh = group % a.kv_heads;
    const uint32_t split = group / a.kv_heads % a.own_splits, b = group / a.kv_heads / a.own_splits;
    slot = a.prefix_splits + split;
    const uint32_t n = length_of(a, b), each = range_keys(n, a.own_splits);
    begin = split * each;
    if (begin >= n) return;
    end = min(begin + each, n);
    first = tile * 16 * QT;
    count = min(a.seq_rows - first, 16u * QT);
    least = min(end, visible(n, a.rows, first / a.group));
    end = min(end, max(begin, visible(n, a.rows, (first + count - 1) / a.group)));  // no row sees further
#pragma unroll
    for (int t = 0; t < QT; ++t) limit[t] = visible(n, a.rows, min(first + 16 * t + i16, first + count - 1) / a.group);
    first += b * a.seq_rows;
    const uint64_t at = static_cast<uint64_t>(b) * a.capacity * a.kv_heads * a.width;
    keys = static_cast<const T*>(a.key) + at;
    values = static_cast<const T*>(a.value) + at;
  }
  const uint32_t stride = a.kv_heads * a.width;
  const int width = a.width;
  keys += static_cast<uint64_t>(kvh) * width;
  values += static_cast<uint64_t>(kvh) * width;
  const float scale = *a.scale;

  u32x4 q[QT][Ops::kSteps];
#pragma unroll
  for (int t = 0; t < QT; ++t)
    Ops::load_row(static_cast<const T*>(a.query) + query_offset(a, first + min(16u * t + i16, count - 1), kvh), g, width, q[t]);

  f32x4 o[QT][C];
  float top[QT], sum[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = -INFINITY;
    sum[t] = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) o[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  typename Ops::Keys kf;
  typename Ops::Values vf;
  // Rows past the last key repeat it: they are masked, and their values cleared.
  auto load_keys = [&](uint32_t at) {
    const T* base = keys + static_cast<uint64_t>(at) * stride;
    const uint32_t last = end - at - 1;
#pragma unroll
    for (int u = 0; u < kTiles; ++u) Ops::load_row(base + min(16u * u + i16, last) * stride, g, width, kf.v[u]);
  };
  auto load_values = [&](uint32_t at) {
    const T* base = values + static_cast<uint64_t>(at) * stride;
    const uint32_t last = end - at - 1;
#pragma unroll
    for (int r = 0; r < Ops::kValueRows; ++r)
      load_words<T, C, A>(base + min(static_cast<uint32_t>(Ops::value_key(g, r)), last) * stride, i16 * C, width, vf.v[r]);
  };

  // The elements of the step's first `seen` keys that are not finite, added to
  // the lane's row of outputs in `joined`.
  auto add_special = [&](const T* row, uint32_t row_stride, uint32_t seen) {
    for (uint32_t k = 0; k < seen; ++k, row += row_stride) {
      const float share = masked_p[wave][k][i16];
#pragma unroll 1
      for (int m = 0; m < 4 * C; ++m) {
        const int f = 4 * g * C + m;
        const float v = f < width ? load_elem(row, f) : 0.0f;
        float& to = reinterpret_cast<float*>(&joined[wave][m % C][lane])[m / C];
        if (!(fabsf(v) < INFINITY)) to = fma_rn(share, v, to);
      }
    }
  };

  // Steps past the range repeat its last key: operands stay defined on every path.
  uint32_t at = begin + wave * KT;
  if (at < end) {
    load_keys(at);
    load_values(at);
  }
  while (at < end) {
    const uint32_t next = at + kWaves * KT;
    f32x4 p[QT][kTiles];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        p[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        Ops::scores(kf.v[u], q[t], p[t][u]);
      }
    load_keys(min(next, end - 1));
    const bool masked = at + KT > least;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float most = -INFINITY;
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float s = p[t][u][r] * scale;
          if (masked && at + 16 * u + 4 * g + r >= limit[t]) s = -INFINITY;
          p[t][u][r] = s;
          most = fmaxf(most, s);
        }
      if (__any(most > top[t] + kSlack)) {
        const float raised = fmaxf(top[t], group_max(most));
        const float factor = top[t] == -INFINITY ? 1.0f : fast_exp(top[t] - raised);  // nothing summed yet: zeros
        top[t] = raised;
        sum[t] = sum[t] * factor;
#pragma unroll
        for (int j = 0; j < C; ++j) o[t][j] = o[t][j] * factor;
      }
      const float from = reference_of(top[t]);
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[t][u][r] = fast_exp(p[t][u][r] - from);
          sum[t] = sum[t] + p[t][u][r];
        }
    }
    if (masked) {
      // Values of keys past the end are cleared.  An infinity or NaN in the
      // values of a key that only some rows see must not reach the others
      // through 0 * inf: such elements leave the product and are added row by
      // row.
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
      if (__any(special)) {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
#pragma unroll
          for (int u = 0; u < kTiles; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) masked_p[wave][16 * u + 4 * g + r][i16] = p[t][u][r];
#pragma unroll
          for (int j = 0; j < C; ++j) joined[wave][j][lane] = o[t][j];
          __builtin_amdgcn_wave_barrier();
          add_special(values + static_cast<uint64_t>(at) * stride, stride, min(min(limit[t], end), at + KT) - at);
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int j = 0; j < C; ++j) o[t][j] = joined[wave][j][lane];
        }
      }
    }
    Ops::template products<QT>(vf, p, o);
    load_values(min(next, end - 1));
    at = next;
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) sum[t] = group_sum(sum[t]);

  // Join the wavefronts: 2 and 3 into 0 and 1, then 1 into 0.
  __syncthreads();
#pragma unroll
  for (int half = 2; half; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        if (g == 0) stats[wave - half][t][i16] = make_float2(top[t], sum[t]);
#pragma unroll
        for (int j = 0; j < C; ++j) joined[(wave - half) * QT + t][j][lane] = o[t][j];
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float2 other = stats[wave][t][i16];
        const float raised = reference_of(fmaxf(top[t], other.x));
        const float mine = fast_exp(top[t] - raised), theirs = fast_exp(other.x - raised);
        top[t] = fmaxf(top[t], other.x);
        sum[t] = fma_rn(sum[t], mine, other.y * theirs);
#pragma unroll
        for (int j = 0; j < C; ++j) o[t][j] = o[t][j] * mine + joined[wave * QT + t][j][lane] * theirs;
      }
    }
    __syncthreads();
  }
  if (wave) return;
  // A lane holds features 4 C g .. of its row, 4 C of them in order.
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (16u * t + i16 >= count) continue;
    const uint64_t row = (static_cast<uint64_t>(slot) * a.kv_heads + kvh) * a.all_rows + first + 16 * t + i16;
    if (g == 0) a.part[row] = make_float2(top[t], sum[t]);
    float* dst = a.sums + row * width;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int f = (4 * g + r) * C + j;
        if (A == Access::kWhole || f < width) dst[f] = o[t][j][r];
      }
  }
}

// Joins the ranges of one row: a wavefront per (KV head, row), the ranges'
// maxima and sums across its lanes, then their outputs one after the other.
template <class T>
__global__ __launch_bounds__(kThreads) void k_join(const Args a) {
  const int lane = threadIdx.x % 64;
  const uint32_t task = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (task >= a.kv_heads * a.all_rows) return;
  const uint32_t kvh = task % a.kv_heads, row = task / a.kv_heads;
  const uint32_t b = row / a.seq_rows, n = length_of(a, b), seen = visible(n, a.rows, row % a.seq_rows / a.group);
  const uint32_t before = ranges_of(a.prefix, a.prefix_splits);
  const uint32_t each = range_keys(n, a.own_splits);
  const uint32_t own = seen ? (seen - 1) / each + 1 : 0;  // ranges past the last key it sees hold nothing of it
  const uint32_t ranges = before + own;
  const uint64_t step = static_cast<uint64_t>(a.kv_heads) * a.all_rows;
  const uint64_t base = static_cast<uint64_t>(kvh) * a.all_rows + row;
  auto place = [&](uint32_t r) { return (r < before ? r : a.prefix_splits + r - before) * step + base; };
  T* out = static_cast<T*>(a.out) + query_offset(a, row, kvh);
  float top = -INFINITY;
  for (uint32_t r = lane; r < ranges; r += 64) top = fmaxf(top, a.part[place(r)].x);
  top = wave_max(top);
  const float from = reference_of(top);
  float total = 0.0f;
  float acc[4] = {};
  for (uint32_t r0 = 0; r0 < ranges; r0 += 64) {
    float factor = 0.0f;
    if (r0 + lane < ranges) {
      const float2 part = a.part[place(r0 + lane)];
      factor = fast_exp(part.x - from);
      total = fma_rn(factor, part.y, total);
    }
    const uint32_t some = min(ranges - r0, 64u);
    for (uint32_t r = 0; r < some; ++r) {
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(factor), r));
      const float* src = a.sums + place(r0 + r) * a.width;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (lane + 64u * k < a.width) acc[k] = fma_rn(f, src[lane + 64 * k], acc[k]);
    }
  }
#pragma unroll
  for (int off = 32; off; off /= 2) total = total + __shfl_xor(total, off);
  const bool none = a.prefix + seen == 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64u * k < a.width) store_elem(out, lane + 64 * k, none ? 0.0f : acc[k] / total);
  if (a.whole && lane == 0) a.whole[base] = make_float2(from, 1.0f / total);
}

// Weights: a wavefront holds 16 keys and walks the rows that see them,
// computing the scores again; a lane sums its 4 keys over its rows, then the
// 16 lanes of a key add up.  Every key has one owner: no atomics.
template <class T, int D, Access A>
__global__ __launch_bounds__(kThreads) void k_weights(const Args a) {
  using Ops = Operands<T, D, A>;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int i16 = lane % 16, g = lane / 16;
  const uint32_t blocks = a.capacity / 64 + (a.capacity % 64 != 0);
  const uint32_t kvh = blockIdx.x % a.kv_heads, b = blockIdx.x / a.kv_heads / blocks;
  const uint32_t key0 = blockIdx.x / a.kv_heads % blocks * 64 + wave * 16;
  const uint32_t n = length_of(a, b);
  if (key0 >= n) return;
  const uint32_t stride = a.kv_heads * a.width;
  const T* keys = static_cast<const T*>(a.key) + (static_cast<uint64_t>(b) * a.capacity + key0) * stride +
                  static_cast<uint64_t>(kvh) * a.width;
  u32x4 k[Ops::kSteps];
  Ops::load_row(keys + min(static_cast<uint32_t>(i16), n - key0 - 1) * stride, g, a.width, k);
  const float scale = *a.scale;
  float sum[4] = {};
  // The first row that sees key0: n - rows + i + 1 > key0.
  const uint64_t from_row = static_cast<uint64_t>(key0) + a.rows > n ? key0 + a.rows - n : 0;
  for (uint32_t r0 = static_cast<uint32_t>(from_row) * a.group / 16 * 16; r0 < a.seq_rows; r0 += 16) {
    const uint32_t in_seq = min(r0 + i16, a.seq_rows - 1), row = b * a.seq_rows + in_seq;
    u32x4 q[Ops::kSteps];
    Ops::load_row(static_cast<const T*>(a.query) + query_offset(a, row, kvh), g, a.width, q);
    const float2 whole = a.whole[static_cast<uint64_t>(kvh) * a.all_rows + row];
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    Ops::scores(k, q, s);
    const uint32_t seen = r0 + i16 < a.seq_rows ? visible(n, a.rows, in_seq / a.group) : 0;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (key0 + 4 * g + r < seen) sum[r] = sum[r] + fast_exp(s[r] * scale - whole.x) * whole.y;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int off = 8; off; off /= 2) sum[r] = sum[r] + __shfl_xor(sum[r], off);
    const uint32_t key = key0 + 4 * g + r;
    if (i16 == 0 && key < n) {
      const uint64_t at = (static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.capacity + key;
      a.weights_out[at] = a.weights[at] + sum[r];
    }
  }
}

// ------------------------------------------------------------------- the host
constexpr const char* kTooMany = "too many workgroups";

// Row tiles per workgroup, ranges and workspace of one call.
struct Layout {
  Args args{};
  int tiles = 1;  // QT
  int features = 64;  // D
  uint64_t part_bytes = 0, sums_bytes = 0, whole_bytes = 0;
  uint32_t own_blocks = 0;
  uint64_t bytes() const { return part_bytes + sums_bytes + whole_bytes; }
  void set_tiles(int count);
  void count_blocks();
};

uint64_t product(std::initializer_list<uint64_t> factors, uint64_t most, const char* what) {
  uint64_t p = 1;
  for (uint64_t f : factors) {
    require(f == 0 || p <= most / f, what, DL_LENGTH_ERROR);
    p *= f;
  }
  return p;
}

void Layout::set_tiles(int count) {
  tiles = count;
  args.prefix_tiles = static_cast<uint32_t>(ceil_div(args.all_rows, 16 * count));
  args.own_tiles = static_cast<uint32_t>(ceil_div(args.seq_rows, 16 * count));
}

void Layout::count_blocks() {
  constexpr uint64_t kMost = 1u << 30;
  auto blocks = [&](std::initializer_list<uint64_t> groups, uint64_t tile_count) {
    return static_cast<uint32_t>(product({ceil_div(product(groups, kMost, kTooMany), 8) * 8, tile_count}, kMost, kTooMany));
  };
  args.prefix_blocks = blocks({args.kv_heads, args.prefix_splits}, args.prefix_tiles);
  own_blocks = blocks({args.batch, args.kv_heads, args.own_splits}, args.own_tiles);
}

Layout layout_of(const dl_batch_shape* shape, uint64_t prefix, bool weighted) {
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
  // Rows per workgroup: few rows leave no tile empty; D = 256 has room for two.
  const uint32_t most_rows = prefix ? a.all_rows : a.seq_rows;
  l.set_tiles(most_rows <= 16 ? 1 : most_rows <= 32 || l.features == 256 ? 2 : 4);
  // Ranges: about kBlocks workgroups in all, each with whole rounds of keys.
  constexpr uint64_t kBlocks = 512;
  const double work = static_cast<double>(a.kv_heads) *
                      (static_cast<double>(a.prefix_tiles) * a.prefix +
                       static_cast<double>(a.batch) * a.own_tiles * a.capacity);
  const uint64_t each = std::max<uint64_t>(kRound, static_cast<uint64_t>(work / kBlocks));
  a.prefix_splits = static_cast<uint32_t>(ceil_div(prefix, each));
  a.own_splits = static_cast<uint32_t>(ceil_div(a.capacity, each));
  l.count_blocks();
  const uint64_t ranges = a.prefix_splits + a.own_splits, most = UINT64_MAX / 8;
  const uint64_t entries = product({ranges, a.kv_heads, a.all_rows}, most, "workspace too large");
  l.part_bytes = ceil_div(product({entries, 8}, most, "workspace too large"), 256) * 256;
  l.sums_bytes = ceil_div(product({entries, a.width, 4}, most, "workspace too large"), 256) * 256;
  l.whole_bytes = weighted ? ceil_div(static_cast<uint64_t>(a.kv_heads) * a.all_rows * 8, 256) * 256 : 0;
  return l;
}

template <class T, int D, Access A>
void launch(hipStream_t s, const Layout& l) {
  const Args& a = l.args;
  const unsigned blocks = a.prefix_blocks + l.own_blocks;  // at most 2^31
  if (l.tiles == 1) {
    k_ranges<T, D, 1, A><<<blocks, kThreads, 0, s>>>(a);
  } else if constexpr (A != Access::kElements) {
    if (l.tiles == 2)
      k_ranges<T, D, 2, A><<<blocks, kThreads, 0, s>>>(a);
    else if constexpr (D != 256)
      k_ranges<T, D, 4, A><<<blocks, kThreads, 0, s>>>(a);
  }
  k_join<T><<<static_cast<unsigned>(ceil_div(static_cast<uint64_t>(a.kv_heads) * a.all_rows, kWaves)), kThreads, 0, s>>>(a);
  if (a.whole) {
    const uint64_t key_blocks = static_cast<uint64_t>(a.batch) * a.kv_heads * ceil_div(a.capacity, 64);
    k_weights<T, D, A><<<static_cast<unsigned>(key_blocks), kThreads, 0, s>>>(a);
  }
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
  Layout l = layout_of(shape, prefix, weighted);
  const bool pieces =
      whole_pieces(shape, dtype == DL_BF16 ? 2 : 4, {o.query, o.prefix_key, o.prefix_value, o.key, o.value});
  const Access access = !pieces ? Access::kElements
                        : static_cast<int>(l.args.width) == l.features ? Access::kWhole
                                                                       : Access::kPieces;
  if (access == Access::kElements) {  // the ranges, and with them the workspace, stay
    l.set_tiles(1);
    l.count_blocks();
  }
  require(o.query && o.key && o.value && o.lengths && o.output && o.scale, "null operand");
  require(prefix == 0 || (o.prefix_key && o.prefix_value), "null prefix operand");
  require(!weighted || (o.weights && o.weights_out), "null weights");
  require(o.workspace != nullptr && reinterpret_cast<uintptr_t>(o.workspace) % 16 == 0, "workspace null or not 16-byte aligned");
  require(o.workspace_bytes >= l.bytes(), "workspace too small", DL_LENGTH_ERROR);
  if (weighted) product({shape->batch, shape->kv_heads, ceil_div(shape->capacity, 64)}, 1u << 30, kTooMany);
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
  if (weighted) a.whole = reinterpret_cast<float2*>(room + l.part_bytes + l.sums_bytes);
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
    *bytes = dl::batch::layout_of(shape, prefix, false).bytes();
  });
}

int dl_attention_weighted_bytes(const dl_batch_shape* shape, uint64_t prefix, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::batch::layout_of(shape, prefix, true).bytes();
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
