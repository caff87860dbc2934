// Attention of new rows over caches held in 4 bits (fp4.h), of all rows in sight or
// of a sliding window and first rows that stay visible.  No reference counterpart.
//
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// New row i of a sequence that holds n rows is at slot p = n - rows + i and sees
// the slots j <= p, under a window only j > p - window or j < sinks.  A row
// without a key is zeros.
//
// Split.  A workgroup takes 16 of a sequence's rows of one KV head (new rows times
// the heads of the group) and a range of the steps of 32 keys that any of them
// sees; its wavefronts take every fourth step, codes straight from memory into
// registers, a step ahead.  Ranges leave their maximum, sum and unnormalised
// output, which k_join joins; a single range writes the output itself.
//
// Operands.  A lane takes D / 4 neighbouring features of a key's codes, one to two
// groups or half of one, and converts them to the first operands of the products K
// Q^T.  Row m of key tile u is the step's key 8 (m / 4) + 4 u + m % 4, which leaves
// lane 16 g + i with row i's scores of the eight neighbouring keys from 8 g on: the
// second operand of V^T P^T as it is.  Its first takes the same eight keys' codes of
// D / 16 neighbouring features, converted and paired by byte permutes; tile j is
// feature j of every lane's.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "batch.h"
#include "dl_device.h"
#include "dl_internal.h"
#include "fp4.h"

namespace dl::fp4 {
namespace {

constexpr int kThreads = 256, kWaves = 4, kKeys = 32;
constexpr float kLog2e = 0x1.715476p+0f;
// A row's maximum is raised only when the exponentials of a lane's keys of one step
// sum to more than this: most steps rescale nothing.
constexpr float kMostSum = 8192.0f;

struct Args {
  const void* query;
  const uint8_t *key_codes, *key_scales, *value_codes, *value_scales;
  const uint64_t* lengths;
  const float* scale;
  void* out;
  float2* part;  // [range][kv head][row]: maximum, sum
  float* sums;   // [range][kv head][row][pitch]: unnormalised output
  uint32_t batch, rows, q_heads, kv_heads, group, width, groups, capacity, window, sinks;
  uint32_t seq_rows, all_rows, splits, tiles, pitch;
};

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ bool rare(bool condition) { return __builtin_expect(condition, false); }
__device__ __forceinline__ float group_max(float v) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float group_sum(float v) {
  v = v + __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ f32x4 product(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t length_of(const Args& a, uint32_t b) {
  const uint64_t n = a.lengths[b];
  return n < a.capacity ? static_cast<uint32_t>(n) : a.capacity;
}

// The slots that one new row sees: [low, end) and those below the sinks.
struct Sight {
  uint32_t low, end;
};
__device__ __forceinline__ Sight sight_of(const Args& a, uint32_t n, uint32_t i) {
  const uint64_t past = static_cast<uint64_t>(n) + i + 1;
  const uint32_t end = past > a.rows ? min(static_cast<uint32_t>(past - a.rows), n) : 0u;
  return {a.window && end > a.window ? end - a.window : 0u, end};
}

// The steps of 32 keys that rows from the one with `first` to the one with `last` in
// sight see: those of the sinks, then those of the windows.
struct Steps {
  uint32_t sinks, begin, end, count;
  __device__ __forceinline__ Steps(const Args& a, const Sight& first, const Sight& last) {
    begin = first.low / kKeys * kKeys;
    sinks = (min(a.sinks, begin) + kKeys - 1) / kKeys;
    if (sinks * kKeys >= begin) sinks = begin = 0;
    end = last.end;
    count = sinks + (end > begin ? (end - begin + kKeys - 1) / kKeys : 0);
  }
  __device__ __forceinline__ uint32_t key(uint32_t step) const {
    return step < sinks ? step * kKeys : begin + (step - sinks) * kKeys;
  }
};
// Steps of one range: whole rounds of the four wavefronts.
__device__ __forceinline__ uint32_t range_steps(uint32_t count, uint32_t splits) {
  return ((count + splits - 1) / splits + kWaves - 1) / kWaves * kWaves;
}

__device__ __forceinline__ uint64_t query_offset(const Args& a, uint32_t row, uint32_t kvh) {
  return (static_cast<uint64_t>(row / a.group) * a.q_heads + kvh * a.group + row % a.group) * a.width;
}

// Eight consecutive query features as product operands; zeros past the width.
template <class T>
__device__ __forceinline__ void query_operands(const T* row, uint32_t at, uint32_t width, bool negative, u32x4* q) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = at + e < width ? load_elem(row, at + e) : 0.0f;
    x[e] = negative ? -v : v;
  }
  if constexpr (sizeof(T) == 4) {
    const Parts p = split(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) q[i] = p.part[i];
  } else {
#pragma unroll
    for (int w = 0; w < 4; ++w)
      q[0][w] = __float_as_uint(x[2 * w]) >> 16 | (__float_as_uint(x[2 * w + 1]) & 0xffff0000u);
  }
}

// Eight exponentials as product operands: rounded to BF16 for BF16 storage (at most
// 2^-8 of the value, as BF16 operands need), exact in three parts for FP32.
template <int kParts>
__device__ __forceinline__ void share_operands(const f32x4 (&p)[2], u32x4 (&b)[kParts]) {
  if constexpr (kParts == 3) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[e / 4][e % 4];
    const Parts s = split(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) b[i] = s.part[i];
  } else {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<__bf16>(p[e / 4][e % 4]);
    b[0] = __builtin_bit_cast(u32x4, v);
  }
}

// N words of codes from a byte offset past a base that the wavefront shares.
template <int N>
__device__ __forceinline__ void load_codes(const uint8_t* base, uint32_t offset, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(base + offset);
  } else {
    typedef uint32_t Words __attribute__((ext_vector_type(N)));
    const Words v = *reinterpret_cast<const Words*>(base + offset);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = v[i];
  }
}

// D features (64, 128 or 256, at least the width) and storage T of query and output.
template <class T, int D>
struct Tile {
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  static constexpr int kSteps = D / 32;                       // products of a key tile
  static constexpr int kKeyWords = D / 32;                    // code words of a lane's D / 4 features
  static constexpr int kKeyScales = D == 256 ? 2 : 1;
  static constexpr int C = D / 16;                            // features of a lane's values
  static constexpr int kValueWords = C < 8 ? 1 : C / 8;       // D = 64: four codes, the lower half of a word
};

template <class T, int D>
__global__ __launch_bounds__(kThreads) void k_attend(const Args a) {
  using S = Tile<T, D>;
  constexpr int C = S::C, kParts = S::kParts;
  __shared__ f32x4 room[kWaves / 2][C][64];
  __shared__ float2 stats[kWaves][16];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i16 = lane % 16, g = lane / 16;
  // XCD x takes the groups x, x + 8, ..., and all row tiles of a group, which read
  // the same keys, so that they meet in one L2.
  const uint32_t in_xcd = blockIdx.x / 8, task = in_xcd / a.tiles * 8 + blockIdx.x % 8, tile = in_xcd % a.tiles;
  if (task >= a.batch * a.kv_heads * a.splits) return;
  const uint32_t range = task % a.splits, kvh = task / a.splits % a.kv_heads, b = task / a.splits / a.kv_heads;
  const uint32_t n = length_of(a, b);
  const uint32_t first = tile * 16, count = min(a.seq_rows - first, 16u);
  const Sight sight = sight_of(a, n, (first + min(i16, count - 1)) / a.group);
  const Sight least = sight_of(a, n, first / a.group), most = sight_of(a, n, (first + count - 1) / a.group);
  const Steps steps(a, least, most);
  const uint32_t each = range_steps(steps.count, a.splits);
  const uint32_t begin = min(range * each, steps.count), end = min(begin + each, steps.count);
  if (begin >= end && range > 0) return;

  const float scale = *a.scale, factor = fabsf(scale) * kLog2e;
  const uint32_t row = b * a.seq_rows + first + min(i16, count - 1);  // the lane's
  u32x4 q[S::kSteps][kParts];
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s)
    query_operands(static_cast<const T*>(a.query) + query_offset(a, row, kvh), g * (D / 4) + 8 * s, a.width, scale < 0.0f, q[s]);

  const uint64_t head = (static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.capacity;
  const uint32_t row_bytes = a.groups * kGroupBytes;
  const uint8_t* key_codes = a.key_codes + head * row_bytes;
  const uint8_t* value_codes = a.value_codes + head * row_bytes;
  const uint8_t* key_scales = a.key_scales + head * a.groups;
  const uint8_t* value_scales = a.value_scales + head * a.groups;

  // A lane's features past the row's last group repeat its last bytes: the query has
  // zeros there, and such features of the output are not stored.
  uint32_t key_words[2][S::kKeyWords], key_bytes[2][S::kKeyScales], value_words[8][S::kValueWords], value_bytes[8];
  constexpr uint32_t kUnit = D < 128 ? 8 : kGroupBytes;  // of a key's codes, within a group
  uint32_t key_at[S::kKeyWords * 4 / kUnit];
#pragma unroll
  for (uint32_t x = 0; x < S::kKeyWords * 4 / kUnit; ++x) key_at[x] = min(g * (D / 8) + x * kUnit, row_bytes - kUnit);
  const uint32_t value_at = min(i16 * (C / 2), row_bytes - C / 2), value_group = min(i16 * C / kGroup, a.groups - 1);
  auto load = [&](uint32_t at) {
    const uint32_t last = n - 1 - at;  // rows past the last repeat it: nobody sees them
    const uint8_t* kc = key_codes + static_cast<uint64_t>(at) * row_bytes;
    const uint8_t* ks = key_scales + static_cast<uint64_t>(at) * a.groups;
    const uint8_t* vc = value_codes + static_cast<uint64_t>(at) * row_bytes;
    const uint8_t* vs = value_scales + static_cast<uint64_t>(at) * a.groups;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t k = min(8 * (i16 / 4) + 4 * u + i16 % 4, last);
#pragma unroll
      for (uint32_t x = 0; x < S::kKeyWords * 4 / kUnit; ++x) load_codes<kUnit / 4>(kc, k * row_bytes + key_at[x], key_words[u] + x * kUnit / 4);
#pragma unroll
      for (int h = 0; h < S::kKeyScales; ++h) key_bytes[u][h] = ks[k * a.groups + min(g * (D / 4) / kGroup + h, a.groups - 1)];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t k = min(8 * g + e, last);
      if constexpr (C == 4)
        value_words[e][0] = *reinterpret_cast<const uint16_t*>(vc + k * row_bytes + value_at);
      else
        load_codes<S::kValueWords>(vc, k * row_bytes + value_at, value_words[e]);
      value_bytes[e] = vs[k * a.groups + value_group];
    }
  };

  f32x4 o[C];
  float top = -INFINITY, from = 0.0f, most_sum = -1.0f, sum = 0.0f;
#pragma unroll
  for (int j = 0; j < C; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  uint32_t step = begin + wave;
  if (step < end) load(steps.key(step));
  for (; step < end; step += kWaves) {
    const uint32_t at = steps.key(step);
    // Scores of the lane's row and the keys at + 8 g + 4 u + r.
    f32x4 p[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      p[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        const u32x4 k = to_bf16(key_words[u][s], scale_of(key_bytes[u][s * S::kKeyScales / S::kSteps]));
#pragma unroll
        for (int i = 0; i < kParts; ++i) p[u] = product(k, q[s][i], p[u]);
      }
    }
    uint32_t words[8][S::kValueWords], bytes[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bytes[e] = value_bytes[e];
#pragma unroll
      for (int w = 0; w < S::kValueWords; ++w) words[e][w] = value_words[e][w];
    }
    load(steps.key(min(step + kWaves, end - 1)));

    const bool masked = at + kKeys > least.end || (a.window && at < most.low && at + kKeys > a.sinks);
    auto hide = [&](f32x4 (&v)[2], float value) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t j = at + 8 * g + 4 * u + r;
          if (j >= sight.end || (j < sight.low && j >= a.sinks)) v[u][r] = value;
        }
    };
    f32x4 e[2];
    auto weigh = [&] {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) e[u][r] = exp2_of(fma_rn(p[u][r], factor, from));
      if (rare(masked)) hide(e, 0.0f);
      return ((e[0][0] + e[0][1]) + (e[0][2] + e[0][3])) + ((e[1][0] + e[1][1]) + (e[1][2] + e[1][3]));
    };
    float s = weigh();
    if (rare(__any(!(s <= most_sum)))) {
      // Each row by itself: what another row sees changes no bit of this one.
      const bool rises = group_max(s <= most_sum ? 0.0f : 1.0f) > 0.0f;
      if (masked) hide(p, -INFINITY);
      float high = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u) high = fmaxf(high, fmaxf(fmaxf(p[u][0], p[u][1]), fmaxf(p[u][2], p[u][3])));
      const float highest = group_max(high) * factor, raised = rises ? fmaxf(top, highest) : top;
      const float less = top == -INFINITY ? 1.0f : exp2_of(top - raised);
      top = raised;
      from = -reference_of(raised);
      most_sum = raised == -INFINITY ? -1.0f : kMostSum;
      sum = sum * less;
#pragma unroll
      for (int j = 0; j < C; ++j) o[j] = o[j] * less;
      s = weigh();
    }
    sum = sum + s;

    if (rare(masked)) {
      // A NaN group of a key that only some rows see must not reach the others
      // through 0 * NaN: it leaves the product and is given to the rows that see it.
      bool special = false;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (bytes[k] == kNanScale) {
          special = true;
          bytes[k] = 127;
        }
      if (rare(__any(special))) {
        const uint8_t* vs = value_scales + static_cast<uint64_t>(at) * a.groups;
#pragma unroll 1
        for (uint32_t k = 0; k < kKeys && at + k < n; ++k) {
          const uint32_t j = at + k;
          if (j >= sight.end || (j < sight.low && j >= a.sinks)) continue;
#pragma unroll
          for (int t = 0; t < C; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (vs[k * a.groups + min(((4 * g + r) * C + t) / kGroup, a.groups - 1)] == kNanScale) o[t][r] = NAN;
        }
      }
    }
    u32x4 shares[kParts];
    share_operands<kParts>(e, shares);
    uint32_t values[8][C / 2];  // pairs of features
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float by = scale_of(bytes[k]);
#pragma unroll
      for (int w = 0; w < S::kValueWords; ++w) {
        const u32x4 v = to_bf16(words[k][w], by);
#pragma unroll
        for (int x = 0; x < (C < 8 ? C / 2 : 4); ++x) values[k][4 * w + x] = v[x];
      }
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      u32x4 v;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        v[w] = __builtin_amdgcn_perm(values[2 * w + 1][j / 2], values[2 * w][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int i = 0; i < kParts; ++i) o[j] = product(v, shares[i], o[j]);
    }
  }
  sum = group_sum(sum);

  // Join the wavefronts: the upper half into the lower, and so on.
#pragma unroll
  for (int half = kWaves / 2; half; half /= 2) {
    if (wave >= half && wave < 2 * half) {
      if (g == 0) stats[wave][i16] = make_float2(top, sum);
#pragma unroll
      for (int j = 0; j < C; ++j) room[wave - half][j][lane] = o[j];
    }
    __syncthreads();
    if (wave < half) {
      const float2 other = stats[wave + half][i16];
      const float raised = fmaxf(top, other.x), base = reference_of(raised);
      const float mine = exp2_of(top - base), theirs = exp2_of(other.x - base);
      top = raised;
      sum = fma_rn(sum, mine, other.y * theirs);
#pragma unroll
      for (int j = 0; j < C; ++j) o[j] = o[j] * mine + room[wave][j][lane] * theirs;
    }
    __syncthreads();
  }
  if (wave || i16 >= count) return;
  // The lane's features (4 g + r) C + j of its row.
  if (a.splits == 1) {
    T* out = static_cast<T*>(a.out) + query_offset(a, row, kvh);
    const float by = sight.end ? 1.0f : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const uint32_t f = (4 * g + r) * C + j;
        if (f < a.width) store_elem(out, f, by == 0.0f ? 0.0f : o[j][r] / sum);
      }
    return;
  }
  const uint64_t place = (static_cast<uint64_t>(range) * a.kv_heads + kvh) * a.all_rows + row;
  if (g == 0) a.part[place] = make_float2(top, sum);
  float* to = a.sums + place * a.pitch;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < C; j += 4) {
      const uint32_t f = (4 * g + r) * C + j;
      if (f < a.pitch) *reinterpret_cast<f32x4*>(to + f) = f32x4{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
    }
}

// Joins the ranges of one row: a wavefront, D / 64 features a lane.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void k_join(const Args a) {
  constexpr int kPer = D / 64;
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint64_t tasks = static_cast<uint64_t>(a.kv_heads) * a.all_rows;
  for (uint64_t task = static_cast<uint64_t>(blockIdx.x) * kWaves + wave; task < tasks; task += static_cast<uint64_t>(gridDim.x) * kWaves) {
    const uint32_t row = static_cast<uint32_t>(task % a.all_rows), kvh = static_cast<uint32_t>(task / a.all_rows);
    const uint32_t in_seq = row % a.seq_rows, tile = in_seq / 16, n = length_of(a, row / a.seq_rows);
    const uint32_t last = min(tile * 16 + 15, a.seq_rows - 1);
    const Sight sight = sight_of(a, n, in_seq / a.group);
    const Steps steps(a, sight_of(a, n, tile * 16 / a.group), sight_of(a, n, last / a.group));
    const uint32_t each = range_steps(steps.count, a.splits);
    const uint32_t ranges = steps.count ? (steps.count + each - 1) / each : 0;
    const uint64_t stride = tasks;
    float top = -INFINITY;
    for (uint32_t r = 0; r < ranges; ++r) top = fmaxf(top, a.part[r * stride + task].x);
    const float from = reference_of(top);
    float sum = 0.0f, acc[kPer] = {};
    for (uint32_t r = 0; r < ranges; ++r) {
      const float2 part = a.part[r * stride + task];
      const float share = exp2_of(part.x - from);
      sum = fma_rn(share, part.y, sum);
      const float* sums = a.sums + (r * stride + task) * a.pitch;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (lane * kPer + e < a.pitch) acc[e] = fma_rn(share, sums[lane * kPer + e], acc[e]);
    }
    T* out = static_cast<T*>(a.out) + query_offset(a, row, kvh);
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (lane * kPer + e < a.width) store_elem(out, lane * kPer + e, sight.end ? acc[e] / sum : 0.0f);
  }
}

// ------------------------------------------------------------------- the host
constexpr uint64_t kMostBlocks = (1u << 23) - 8;

uint64_t times(uint64_t x, uint64_t y, uint64_t most, const char* what) {
  require(y == 0 || x <= most / y, what, DL_LENGTH_ERROR);
  return x * y;
}

struct Layout {
  Args args{};
  uint32_t blocks = 0;
  uint64_t part_bytes = 0, sums_bytes = 0;
  uint64_t bytes() const { return part_bytes + sums_bytes; }
};

Layout layout_of(const dl_batch_shape* shape, uint64_t window, uint64_t sinks) {
  batch::check_shape(shape);
  require(shape->width <= 256, "head width above 256", DL_LENGTH_ERROR);
  Layout l;
  Args& a = l.args;
  a.batch = static_cast<uint32_t>(shape->batch);
  a.rows = static_cast<uint32_t>(shape->rows);
  a.q_heads = static_cast<uint32_t>(shape->query_heads);
  a.kv_heads = static_cast<uint32_t>(shape->kv_heads);
  a.group = a.q_heads / a.kv_heads;
  a.width = static_cast<uint32_t>(shape->width);
  a.groups = static_cast<uint32_t>(groups_of(a.width));
  a.capacity = static_cast<uint32_t>(shape->capacity);
  // A window of the capacity or more hides nothing.
  a.window = window < a.capacity ? static_cast<uint32_t>(window) : 0;
  a.sinks = a.window ? static_cast<uint32_t>(std::min<uint64_t>(sinks, a.capacity)) : 0;
  constexpr const char* kRows = "too many query rows";
  a.seq_rows = static_cast<uint32_t>(times(a.rows, a.group, 1u << 30, kRows));
  a.all_rows = static_cast<uint32_t>(times(a.seq_rows, a.batch, 1u << 30, kRows));
  times(a.all_rows, a.kv_heads, 1u << 30, kRows);
  a.tiles = static_cast<uint32_t>(ceil_div(a.seq_rows, 16));
  a.pitch = (a.width + 3) / 4 * 4;
  // Most steps that a row tile can see, and ranges for two workgroups a compute unit.
  uint64_t keys = a.capacity;
  if (a.window) keys = std::min<uint64_t>(keys, uint64_t{a.window} + a.sinks + 16 + 3 * kKeys);
  const uint64_t rounds = ceil_div(keys, kKeys * kWaves);
  const uint64_t tasks = times(times(a.batch, a.kv_heads, kMostBlocks, "too many workgroups"), a.tiles, kMostBlocks, "too many workgroups");
  a.splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min(ceil_div(rounds, 2), 512 / tasks)));
  const uint64_t groups = times(uint64_t{a.batch} * a.kv_heads, a.splits, kMostBlocks, "too many workgroups");
  l.blocks = static_cast<uint32_t>(times(ceil_div(groups, 8) * 8, a.tiles, kMostBlocks, "too many workgroups"));
  if (a.splits > 1) {
    const uint64_t entries = uint64_t{a.splits} * a.kv_heads * a.all_rows;
    l.part_bytes = ceil_div(entries * 8, 256) * 256;
    l.sums_bytes = ceil_div(entries * a.pitch * 4, 256) * 256;
  }
  return l;
}

template <class T, int D>
void launch(hipStream_t s, const Layout& l) {
  k_attend<T, D><<<l.blocks, kThreads, 0, s>>>(l.args);
  if (l.args.splits > 1) {
    const uint64_t blocks = ceil_div(uint64_t{l.args.kv_heads} * l.args.all_rows, kWaves);
    k_join<T, D><<<static_cast<unsigned>(std::min<uint64_t>(blocks, 1u << 20)), kThreads, 0, s>>>(l.args);
  }
}

template <class T>
void launch_width(hipStream_t s, const Layout& l) {
  if (l.args.width <= 64)
    launch<T, 64>(s, l);
  else if (l.args.width <= 128)
    launch<T, 128>(s, l);
  else
    launch<T, 256>(s, l);
}

}  // namespace
}  // namespace dl::fp4

using dl::guard;
using dl::require;

extern "C" {

int dl_attention_fp4_bytes(const dl_batch_shape* shape, uint64_t window, uint64_t sinks, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::fp4::layout_of(shape, window, sinks).bytes();
  });
}

int dl_attention_fp4(dl_queue* queue, int dtype, const dl_batch_shape* shape, const void* query, const dl_fp4_cache* cache,
                     const uint64_t* lengths, uint64_t window, uint64_t sinks, void* output, const float* scale,
                     void* workspace, uint64_t workspace_bytes) {
  return guard([&] {
    using namespace dl::fp4;
    require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
    Layout l = layout_of(shape, window, sinks);
    require(cache != nullptr, "null cache");
    require(query && cache->key_codes && cache->key_scales && cache->value_codes && cache->value_scales && lengths && output && scale,
            "null operand");
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    require(aligned(cache->key_codes) && aligned(cache->value_codes), "codes not 16-byte aligned");
    require(l.bytes() == 0 || (workspace != nullptr && aligned(workspace)), "workspace null or not 16-byte aligned");
    require(workspace_bytes >= l.bytes(), "workspace too small", DL_LENGTH_ERROR);
    dl::enter(queue);
    Args& a = l.args;
    a.query = query;
    a.key_codes = static_cast<const uint8_t*>(cache->key_codes);
    a.key_scales = static_cast<const uint8_t*>(cache->key_scales);
    a.value_codes = static_cast<const uint8_t*>(cache->value_codes);
    a.value_scales = static_cast<const uint8_t*>(cache->value_scales);
    a.lengths = lengths;
    a.scale = scale;
    a.out = output;
    a.part = static_cast<float2*>(workspace);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.part_bytes);
    if (dtype == DL_BF16)
      launch_width<uint16_t>(queue->stream, l);
    else
      launch_width<float>(queue->stream, l);
    dl::check_launch(queue, "attention_fp4");
  });
}

}  // extern "C"
