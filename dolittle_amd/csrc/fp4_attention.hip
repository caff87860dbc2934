// Attention of new rows over caches held in 4 bits (fp4.h), of all rows in sight or
// of a sliding window and first rows that stay visible.  No reference counterpart.
//
//   s_j = scale * <q, k_j>, out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// New row i of a sequence that holds n rows is at slot p = n - rows + i and sees
// the slots j <= p, under a window only j > p - window or j < sinks.  A row
// without a key is zeros.
//
// Split.  A workgroup takes 16 or 32 of a sequence's rows of one KV head (new rows
// times the heads of the group) and a range of the steps of 32 keys that any of them
// sees; its wavefronts take every fourth step, whose codes come through LDS rooms of
// their own, two steps ahead.  Ranges leave their maximum, sum and unnormalised
// output, which k_join joins; a single range writes the output itself.  Of few rows the
// caches' stream is the bound: 64 sequences of up to 32,768 keys, 8 KV heads of 128
// features, 300 us, 5.0 TB/s; of many the conversions and exponentials beside the
// products: 512 rows of 32 heads over 4096 keys 73 us, 440 TFLOP/s, FP32 126.  There vector
// instructions issue in half of the cycles and products are busy in 27%.
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
  uint32_t seq_rows, all_rows, splits, tiles, tile_rows, pitch;
  bool whole_out;  // output rows in fours of whole alignment
};

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.0f : m; }
// The square root of 2^v, to multiply by twice: what is counted from an old maximum may
// be kMostSum times as large, so a factor below 2^-126, which exp2 gives as zero, can
// leave a value that is not.
__device__ __forceinline__ float root_exp2_of(float v) { return exp2_of(0.5f * v); }
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
// Products' results are there 8 instructions after the last of them.  The compiler counts
// these along straight code and, behind a branch, has read one 3 later: a wrong score.
// So they are waited for here, before any branch.
template <int N>
__device__ __forceinline__ void settle(f32x4 (&p)[N][2]) {
  static_assert(N == 1 || N == 2);
  if constexpr (N == 1)
    asm volatile("s_nop 7" : "+v"(p[0][0]), "+v"(p[0][1]));
  else
    asm volatile("s_nop 7" : "+v"(p[0][0]), "+v"(p[0][1]), "+v"(p[1][0]), "+v"(p[1][1]));
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
template <class T, bool kPieces>
__device__ __forceinline__ void query_operands(const T* row, uint32_t at, uint32_t width, bool negative, u32x4* q) {
  if constexpr (sizeof(T) == 4) {
    float x[8];
    load_eight<T, kPieces>(row, at, width, x);
#pragma unroll
    for (float& v : x) v = negative ? -v : v;
    const Parts p = split(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) q[i] = p.part[i];
  } else {
    const uint32_t signs = negative ? 0x80008000u : 0u;
    if constexpr (kPieces) {
      q[0] = (at < width ? *reinterpret_cast<const u32x4*>(row + at) : u32x4{}) ^ signs;
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t f = at + 2 * w, lo = f < width ? row[f] : 0u, hi = f + 1 < width ? row[f + 1] : 0u;
        q[0][w] = (lo | hi << 16) ^ signs;
      }
    }
  }
}

// Eight exponentials as product operands: exact in three parts for FP32 storage, for
// BF16 in two, what the first leaves rounded again: at most 2^-16 of the value.  One part
// alone, 2^-8, is as far off as the output's own rounding and more where values cancel.
template <int kShares>
__device__ __forceinline__ void share_operands(const f32x4 (&p)[2], u32x4 (&b)[kShares]) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = p[e / 4][e % 4];
  if constexpr (kShares == 3) {
    const Parts s = split(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) b[i] = s.part[i];
  } else {
    bf16x8 high, low;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      high[e] = static_cast<__bf16>(x[e]);
      low[e] = static_cast<__bf16>(x[e] - static_cast<float>(high[e]));
    }
    b[0] = __builtin_bit_cast(u32x4, high);
    b[1] = __builtin_bit_cast(u32x4, low);
  }
}

// D features (64, 128 or 256, at least the width) and storage T of query and output.
template <class T, int D>
struct Tile {
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;       // of a query feature
  static constexpr int kShares = sizeof(T) == 4 ? 3 : 2;      // of a softmax weight
  static constexpr int kSteps = D / 32;                       // products of a key tile
  static constexpr int kKeyWords = D / 32;                    // code words of a lane's D / 4 features
  static constexpr int kKeyScales = D == 256 ? 2 : 1;
  static constexpr int C = D / 16;                            // features of a lane's values
  static constexpr int kValueWords = C < 8 ? 1 : C / 8;       // D = 64: four codes, the lower half of a word
};

// A step's codes of one wavefront: 32 keys, then their values, D / 2 bytes each, and
// with kWords their scales, D / 32 bytes each.  Objects apart, so that the compiler sees
// no use of loads in flight.
constexpr int kRing = 3;
template <int D, int kSlot, bool kWords>
__device__ __forceinline__ uint8_t* step_room() {
  __shared__ __align__(1024) uint8_t room[kWaves * (32 * D + (kWords ? 2 * D : 0))];
  return room;
}

// Of two tiles of rows a wavefront holds twice the queries and outputs: left to itself
// the compiler takes more than 256 registers, one workgroup a unit, 102 us where this
// takes 73.
template <class T, int D, bool kPieces, bool kWords, int QT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(QT))) void k_attend(const Args a) {
  using S = Tile<T, D>;
  constexpr int C = S::C, kParts = S::kParts, kShares = S::kShares;
  __shared__ float2 stats[kWaves][16];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i16 = lane % 16, g = lane / 16;
  // XCD x takes the groups x, x + 8, ..., and all row tiles of a group, which read
  // the same keys, so that they meet in one L2.
  const uint32_t in_xcd = blockIdx.x / 8, task = in_xcd / a.tiles * 8 + blockIdx.x % 8, tile = in_xcd % a.tiles;
  if (task >= a.batch * a.kv_heads * a.splits) return;
  const uint32_t range = task % a.splits, kvh = task / a.splits % a.kv_heads, b = task / a.splits / a.kv_heads;
  const uint32_t n = length_of(a, b);
  const uint32_t first = tile * 16 * QT, count = min(a.seq_rows - first, 16u * QT);
  Sight sight[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) sight[t] = sight_of(a, n, (first + min(16 * t + i16, count - 1)) / a.group);
  const Sight least = sight_of(a, n, first / a.group), most = sight_of(a, n, (first + count - 1) / a.group);
  const Steps steps(a, least, most);
  const uint32_t each = range_steps(steps.count, a.splits);
  const uint32_t begin = min(range * each, steps.count), end = min(begin + each, steps.count);
  if (begin >= end && range > 0) return;

  const float scale = *a.scale, factor = fabsf(scale) * kLog2e;
  auto row_of = [&](int t) { return b * a.seq_rows + first + min(16 * t + i16, count - 1); };  // the lane's
  u32x4 q[QT][S::kSteps][kParts];
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
      query_operands<T, kPieces>(static_cast<const T*>(a.query) + query_offset(a, row_of(t), kvh), g * (D / 4) + 8 * s, a.width,
                                 scale < 0.0f, q[t][s]);

  const uint64_t head = (static_cast<uint64_t>(b) * a.kv_heads + kvh) * a.capacity;
  const uint32_t row_bytes = a.groups * kGroupBytes;
  const uint8_t* key_codes = a.key_codes + head * row_bytes;
  const uint8_t* value_codes = a.value_codes + head * row_bytes;
  const uint8_t* key_scales = a.key_scales + head * a.groups;
  const uint8_t* value_scales = a.value_scales + head * a.groups;

  // Codes go through LDS of the wavefront's own, 1 KiB a load, two steps ahead; scale
  // bytes to registers as far ahead.  Features past the row's last group repeat it: the
  // query has zeros there, and such features of the output are not stored.  Piece p of a
  // key's codes lies at p ^ key / 8, so that the keys of an operand lie in distinct banks.
  // Whole rows of scale words go through LDS too, 1 load (D = 256: 2) for 10 (12): 512 rows
  // over 4096 keys 75 us for 77, 64 sequences of up to 32,768 keys 318 for 330.
  constexpr uint32_t P = D / 32, kRowBytes = D / 2, kHalf = 16 * D;  // pieces of a key; bytes of 32
  constexpr uint32_t kRoom = 2 * kHalf + (kWords ? 2 * D : 0), kWordRow = kWords ? D / 128 : 1;
  const uint32_t value_group = min(i16 * C / kGroup, a.groups - 1);
  struct Scales {
    uint32_t key[2][S::kKeyScales], value[8];
  };
  Scales ring[kRing];
  auto load = [&](uint8_t* room, Scales& to, uint32_t at) __attribute__((always_inline)) {
    const uint32_t last = n - 1 - at;  // rows past the last repeat it: nobody sees them
    const uint8_t* kc = key_codes + static_cast<uint64_t>(at) * row_bytes;
    const uint8_t* vc = value_codes + static_cast<uint64_t>(at) * row_bytes;
    const uint8_t* ks = key_scales + static_cast<uint64_t>(at) * a.groups;
    const uint8_t* vs = value_scales + static_cast<uint64_t>(at) * a.groups;
    uint8_t* mine = room + wave * kRoom;
#pragma unroll
    for (uint32_t x = 0; x < kHalf / 1024; ++x) {
      const uint32_t slot = x * 64 + lane, key = slot / P, piece = min(slot % P ^ key / 8 % P, a.groups - 1);
      const uint32_t from = min(key, last) * row_bytes + piece * kGroupBytes;
      __builtin_amdgcn_global_load_lds((const global_ptr*)(kc + from), (lds_ptr*)(mine + x * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const global_ptr*)(vc + from), (lds_ptr*)(mine + kHalf + x * 1024), 16, 0, 0);
    }
    if constexpr (kWords) {
#pragma unroll
      for (uint32_t x = 0; x < kWordRow; ++x) {
        const uint32_t word = x * 64 + lane, in_half = word % (32 * kWordRow);
        const uint8_t* of = word < 32 * kWordRow ? ks : vs;
        __builtin_amdgcn_global_load_lds((const global_ptr*)(of + min(in_half / kWordRow, last) * P + in_half % kWordRow * 4),
                                         (lds_ptr*)(mine + 2 * kHalf + x * 256), 4, 0, 0);
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t k = min(8 * (i16 / 4) + 4 * u + i16 % 4, last);
#pragma unroll
      for (int h = 0; h < S::kKeyScales; ++h) to.key[u][h] = ks[k * a.groups + min(g * (D / 4) / kGroup + h, a.groups - 1)];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) to.value[e] = vs[min(8 * g + e, last) * a.groups + value_group];
  };
  constexpr int kLoads = 2 * kHalf / 1024 + (kWords ? kWordRow : 2 * S::kKeyScales + 8);

  f32x4 o[QT][C];
  float top[QT], from[QT], most_sum[QT], sum[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    top[t] = -INFINITY;
    from[t] = sum[t] = 0.0f;
    most_sum[t] = -1.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) o[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  auto work = [&](const uint8_t* room, const Scales& by, uint32_t at) __attribute__((always_inline)) {
    const uint8_t* keys = room + wave * kRoom;
    // No branch, which the && and || would be, lies between products and their use.
    const bool masked = (at + kKeys > least.end) | ((a.window != 0) & (at < most.low) & (at + kKeys > a.sinks));
    // Scores of the lane's rows and the keys at + 8 g + 4 u + r.
    f32x4 p[QT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t key = 8 * (i16 / 4) + 4 * u + i16 % 4, swizzle = i16 / 4 % P;
      uint32_t words[S::kKeyWords];
      if constexpr (D == 64) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(keys + key * kRowBytes + (g / 2 ^ swizzle) * 16 + g % 2 * 8);
        words[0] = v.x;
        words[1] = v.y;
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(keys + key * kRowBytes + ((g * (D / 128) + h) ^ swizzle) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) words[4 * h + e] = v[e];
        }
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) p[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        const int h = s * S::kKeyScales / S::kSteps;
        const u32x4 k = to_bf16(words[s], scale_of(kWords ? keys[2 * kHalf + key * P + g * (D / 4) / kGroup + h] : by.key[u][h]));
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
          for (int t = 0; t < QT; ++t) p[t][u] = product(k, q[t][s][i], p[t][u]);
      }
    }
    settle(p);
    uint32_t words[8][S::kValueWords], bytes[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bytes[e] = kWords ? keys[2 * kHalf + D + (8 * g + e) * P + value_group] : by.value[e];
      const uint32_t byte = i16 * (C / 2);  // of the key's codes
      const uint8_t* from = keys + kHalf + (8 * g + e) * kRowBytes + (byte / 16 ^ g % P) * 16 + byte % 16;
      if constexpr (C == 4) {
        words[e][0] = *reinterpret_cast<const uint16_t*>(from);
      } else if constexpr (C == 8) {
        words[e][0] = *reinterpret_cast<const uint32_t*>(from);
      } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(from);
        words[e][0] = v.x;
        words[e][1] = v.y;
      }
    }

    u32x4 shares[QT][kShares];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      auto hide = [&](f32x4 (&v)[2], float value) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t j = at + 8 * g + 4 * u + r;
            if (j >= sight[t].end || (j < sight[t].low && j >= a.sinks)) v[u][r] = value;
          }
      };
      f32x4 e[2];
      auto weigh = [&] {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) e[u][r] = exp2_of(fma_rn(p[t][u][r], factor, from[t]));
        if (rare(masked)) hide(e, 0.0f);
        return ((e[0][0] + e[0][1]) + (e[0][2] + e[0][3])) + ((e[1][0] + e[1][1]) + (e[1][2] + e[1][3]));
      };
      float s = weigh();
      if (rare(__any(!(s <= most_sum[t])))) {
        // Each row by itself: what another row sees changes no bit of this one.
        const bool rises = group_max(s <= most_sum[t] ? 0.0f : 1.0f) > 0.0f;
        if (masked) hide(p[t], -INFINITY);
        float high = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u) high = fmaxf(high, fmaxf(fmaxf(p[t][u][0], p[t][u][1]), fmaxf(p[t][u][2], p[t][u][3])));
        const float highest = group_max(high) * factor, raised = rises ? fmaxf(top[t], highest) : top[t];
        const float less = top[t] == -INFINITY ? 1.0f : root_exp2_of(top[t] - raised);
        top[t] = raised;
        from[t] = -reference_of(raised);
        most_sum[t] = raised == -INFINITY ? -1.0f : kMostSum;
        sum[t] = sum[t] * less * less;
#pragma unroll
        for (int j = 0; j < C; ++j) o[t][j] = o[t][j] * less * less;
        s = weigh();
      }
      sum[t] = sum[t] + s;
      share_operands<kShares>(e, shares[t]);
    }

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
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            if (j >= sight[t].end || (j < sight[t].low && j >= a.sinks)) continue;
#pragma unroll
            for (int x = 0; x < C; ++x)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (vs[k * a.groups + min(((4 * g + r) * C + x) / kGroup, a.groups - 1)] == kNanScale) o[t][x][r] = NAN;
          }
        }
      }
    }
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
      for (int i = 0; i < kShares; ++i)
#pragma unroll
        for (int t = 0; t < QT; ++t) o[t][j] = product(v, shares[t][i], o[t][j]);
    }
  };
  // Loads past the last step repeat it; none lies under a condition, and the loop is left
  // at its end alone: the compiler would wait for all loads in flight.
  auto turn = [&](auto slot, uint32_t step) __attribute__((always_inline)) {
    constexpr int kSlot = decltype(slot)::value, kNext = (kSlot + kRing - 1) % kRing;
    __builtin_amdgcn_s_waitcnt(lds_wait((kRing - 2) * kLoads));  // this step's codes; the room loaded next is read
    asm volatile("" ::: "memory");
    load(step_room<D, kNext, kWords>(), ring[kNext], steps.key(min(step + (kRing - 1) * kWaves, end - 1)));
    __builtin_amdgcn_sched_barrier(0);
    if (step < end) work(step_room<D, kSlot, kWords>(), ring[kSlot], steps.key(step));
  };
  uint32_t step = begin + wave;
  if (step < end) {
    load(step_room<D, 0, kWords>(), ring[0], steps.key(step));
    __builtin_amdgcn_sched_barrier(0);
    load(step_room<D, 1, kWords>(), ring[1], steps.key(min(step + kWaves, end - 1)));
    __builtin_amdgcn_sched_barrier(0);
    for (; step < end; step += kRing * kWaves) {
      turn(std::integral_constant<int, 0>{}, step);
      turn(std::integral_constant<int, 1>{}, step + kWaves);
      turn(std::integral_constant<int, 2>{}, step + 2 * kWaves);
    }
  }
  // The loads past the last step may be under way, to rooms that the join writes.
  __builtin_amdgcn_s_waitcnt(lds_wait(0));
  asm volatile("" ::: "memory");
#pragma unroll
  for (int t = 0; t < QT; ++t) sum[t] = group_sum(sum[t]);

  // Join the wavefronts, a tile of rows at a time: the upper half into the lower, and so on.
  f32x4 (*room)[C][64] = reinterpret_cast<f32x4 (*)[C][64]>(step_room<D, 0, kWords>());
  static_assert(kWaves / 2 * C * 1024 <= kWaves * 32 * D, "joined outputs outgrow a room");
#pragma unroll
  for (int t = 0; t < QT; ++t) {
#pragma unroll
    for (int half = kWaves / 2; half; half /= 2) {
      __syncthreads();  // nothing reads what is written next any more
      if (wave >= half && wave < 2 * half) {
        if (g == 0) stats[wave][i16] = make_float2(top[t], sum[t]);
#pragma unroll
        for (int j = 0; j < C; ++j) room[wave - half][j][lane] = o[t][j];
      }
      __syncthreads();
      if (wave < half) {
        const float2 other = stats[wave + half][i16];
        const float raised = fmaxf(top[t], other.x), base = reference_of(raised);
        const float mine = root_exp2_of(top[t] - base), theirs = root_exp2_of(other.x - base);
        top[t] = raised;
        sum[t] = fma_rn(sum[t] * mine, mine, other.y * theirs * theirs);
#pragma unroll
        for (int j = 0; j < C; ++j) o[t][j] = o[t][j] * mine * mine + room[wave][j][lane] * theirs * theirs;
      }
    }
  }
  if (wave) return;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (16u * t + i16 >= count) continue;
    // The lane's features (4 g + r) C + j of its row.
    if (a.splits == 1) {
      T* out = static_cast<T*>(a.out) + query_offset(a, row_of(t), kvh);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < C; j += 4) {
          const uint32_t f = (4 * g + r) * C + j;
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = sight[t].end ? o[t][j + e][r] / sum[t] : 0.0f;
          if (f < a.width) store_four(out + f, v, a.width - f, a.whole_out);
        }
      continue;
    }
    const uint64_t place = (static_cast<uint64_t>(range) * a.kv_heads + kvh) * a.all_rows + row_of(t);
    if (g == 0) a.part[place] = make_float2(top[t], sum[t]);
    float* to = a.sums + place * a.pitch;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < C; j += 4) {
        const uint32_t f = (4 * g + r) * C + j;
        if (f < a.pitch) *reinterpret_cast<f32x4*>(to + f) = f32x4{o[t][j][r], o[t][j + 1][r], o[t][j + 2][r], o[t][j + 3][r]};
      }
  }
}

// Joins the ranges of one row, W wavefronts a row.  D / 4 lanes hold a row of a range,
// four features each, so a wavefront reads 256 / D ranges at a time.  Sums are read
// before the maxima say how much of them counts: one wait and not two.
template <class T, int D, int W>
__global__ __launch_bounds__(kThreads) void k_join(const Args a) {
  constexpr uint32_t kLanes = D / 4, kAtOnce = W * 64 / kLanes, kAhead = 4, kTasks = kWaves / W;
  __shared__ f32x4 room[kWaves][64];
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t tasks = a.kv_heads * a.all_rows, task = blockIdx.x * kTasks + wave / W;
  if (task >= tasks) return;  // wavefronts of one row end together
  const uint32_t row = task % a.all_rows, kvh = task / a.all_rows;
  const uint32_t in_seq = row % a.seq_rows, tile0 = in_seq / a.tile_rows * a.tile_rows, n = length_of(a, row / a.seq_rows);
  const uint32_t f = lane % kLanes * 4, first = wave % W * (64 / kLanes) + lane / kLanes;
  const float* sums = a.sums + (f < a.pitch ? f : 0);
  f32x4 ahead[kAhead];
#pragma unroll
  for (uint32_t m = 0; m < kAhead; ++m)
    ahead[m] = *reinterpret_cast<const f32x4*>(sums + (static_cast<uint64_t>(min(m * kAtOnce + first, a.splits - 1)) * tasks + task) * a.pitch);
  const Sight sight = sight_of(a, n, in_seq / a.group);
  const Steps steps(a, sight_of(a, n, tile0 / a.group), sight_of(a, n, (min(tile0 + a.tile_rows, a.seq_rows) - 1) / a.group));
  const uint32_t each = range_steps(steps.count, a.splits), ranges = steps.count ? (steps.count + each - 1) / each : 0;
  auto part = [&](uint32_t r) { return a.part[static_cast<uint64_t>(r) * tasks + task]; };
  const float2 mine = lane < ranges ? part(lane) : make_float2(-INFINITY, 0.0f);
  float top = mine.x;
  for (uint32_t r = lane + 64; r < ranges; r += 64) top = fmaxf(top, part(r).x);
  const float from = reference_of(wave_max(top));
  float root = root_exp2_of(mine.x - from), sum = root * mine.y * root;
  for (uint32_t r = lane + 64; r < ranges; r += 64) {
    const float2 p = part(r);
    root = root_exp2_of(p.x - from);
    sum = fma_rn(root, root * p.y, sum);
  }
#pragma unroll
  for (int off = 32; off; off /= 2) sum = sum + __shfl_xor(sum, off);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](uint32_t r, const f32x4& v) {
    const float share = root_exp2_of(part(r).x - from);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fma_rn(share, share * v[e], acc[e]);
  };
#pragma unroll
  for (uint32_t m = 0; m < kAhead; ++m)
    if (m * kAtOnce + first < ranges) add(m * kAtOnce + first, ahead[m]);
  for (uint32_t r = kAhead * kAtOnce + first; r < ranges; r += kAtOnce)
    add(r, *reinterpret_cast<const f32x4*>(sums + (static_cast<uint64_t>(r) * tasks + task) * a.pitch));
#pragma unroll
  for (uint32_t off = kLanes; off < 64; off *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] + __shfl_xor(acc[e], off);
  if constexpr (W > 1) {
    room[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < W; ++w) acc = acc + room[w][lane];
  }
  if (lane >= kLanes) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = sight.end ? acc[e] / sum : 0.0f;
  if (f < a.width) store_four(static_cast<T*>(a.out) + query_offset(a, row, kvh) + f, acc, a.width - f, a.whole_out);
}

// ------------------------------------------------------------------- the host
constexpr uint64_t kMostBlocks = (1u << 23) - 8;
constexpr uint32_t kFewRanges = 8;
constexpr uint64_t kMostRange = 8192;  // keys

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

Layout layout_of(const dl_batch_shape* shape, uint64_t window, uint64_t sinks, bool bf16) {
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
  // Two tiles a wavefront convert the keys and values once for both.  BF16, 512 rows of
  // 32 heads over 4096 keys: 75 us, one tile 100; 1000 rows of them, 511 keys in sight each:
  // 47 and 59; 64 rows a KV head, 4 sequences: 25 and 23.  FP32, with three products for
  // one, gains less: 512 rows 116 and 126, 64 rows of 4 sequences 67 and 61, 100 rows over 2000
  // keys 35 and 32; it stays with one.  Of 256 features two tiles do not fit the registers.
  a.tile_rows = bf16 && a.width <= 128 && a.seq_rows > 64 ? 32 : 16;
  a.tiles = static_cast<uint32_t>(ceil_div(a.seq_rows, a.tile_rows));
  a.pitch = (a.width + 3) / 4 * 4;
  // Most steps that a row tile can see, and ranges for two workgroups a compute unit.
  uint64_t keys = a.capacity;
  if (a.window) keys = std::min<uint64_t>(keys, uint64_t{a.window} + a.sinks + a.tile_rows + 3 * kKeys);
  const uint64_t rounds = ceil_div(keys, kKeys * kWaves);
  constexpr const char* kTiles = "too many row tiles";
  const uint64_t heads = times(a.batch, a.kv_heads, kMostBlocks, kTiles), tasks = times(heads, a.tiles, kMostBlocks, kTiles);
  times(ceil_div(heads, 8) * 8, a.tiles, kMostBlocks, kTiles);
  const uint64_t most = std::max<uint64_t>(1, kMostBlocks / a.tiles / 8 * 8 / heads);  // ranges that a launch has room for
  a.splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min({ceil_div(rounds, 2), std::max(ceil_div(512, tasks), keys / kMostRange), most})));
  // More rows than the join has workgroups for fill the card without ranges.
  if (uint64_t{a.all_rows} * a.kv_heads > kMostBlocks) a.splits = 1;
  l.blocks = static_cast<uint32_t>(ceil_div(heads * a.splits, 8) * 8 * a.tiles);
  if (a.splits > 1) {
    const uint64_t entries = uint64_t{a.splits} * a.kv_heads * a.all_rows;
    l.part_bytes = ceil_div(entries * 8, 256) * 256;
    l.sums_bytes = ceil_div(entries * a.pitch * 4, 256) * 256;
  }
  return l;
}

// One size for either storage type, whose tiles and so ranges differ.
uint64_t bytes_of(const dl_batch_shape* shape, uint64_t window, uint64_t sinks) {
  return std::max(layout_of(shape, window, sinks, true).bytes(), layout_of(shape, window, sinks, false).bytes());
}

template <class T, int D>
void launch(hipStream_t s, const Layout& l, bool pieces, bool words) {
  auto attend = [&](auto tiles) {
    constexpr int QT = decltype(tiles)::value;
    if constexpr (D >= 128) {
      if (pieces && words) return k_attend<T, D, true, true, QT><<<l.blocks, kThreads, 0, s>>>(l.args);
    }
    if (pieces)
      k_attend<T, D, true, false, QT><<<l.blocks, kThreads, 0, s>>>(l.args);
    else
      k_attend<T, D, false, false, QT><<<l.blocks, kThreads, 0, s>>>(l.args);
  };
  bool one = true;
  if constexpr (sizeof(T) == 2 && D < 256) one = l.args.tile_rows == 16;
  if (one)
    attend(std::integral_constant<int, 1>{});
  else if constexpr (sizeof(T) == 2 && D < 256)
    attend(std::integral_constant<int, 2>{});
  // A workgroup per row where there are many ranges, else a wavefront.
  const uint64_t tasks = uint64_t{l.args.kv_heads} * l.args.all_rows;
  if (l.args.splits > kFewRanges)
    k_join<T, D, kWaves><<<static_cast<unsigned>(tasks), kThreads, 0, s>>>(l.args);
  else if (l.args.splits > 1)
    k_join<T, D, 1><<<static_cast<unsigned>(ceil_div(tasks, kWaves)), kThreads, 0, s>>>(l.args);
}

template <class T>
void launch_width(hipStream_t s, const Layout& l, bool pieces) {
  const Args& a = l.args;
  // All groups of the tile's width, in words: whole rows.
  const bool words = a.groups == (a.width <= 128 ? 4 : 8) && reinterpret_cast<uintptr_t>(a.key_scales) % 4 == 0 &&
                     reinterpret_cast<uintptr_t>(a.value_scales) % 4 == 0;
  if (a.width <= 64)
    launch<T, 64>(s, l, pieces, false);
  else if (a.width <= 128)
    launch<T, 128>(s, l, pieces, words);
  else
    launch<T, 256>(s, l, pieces, words);
}

}  // namespace
}  // namespace dl::fp4

using dl::guard;
using dl::require;

extern "C" {

int dl_attention_fp4_bytes(const dl_batch_shape* shape, uint64_t window, uint64_t sinks, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::fp4::bytes_of(shape, window, sinks);
  });
}

int dl_attention_fp4(dl_queue* queue, int dtype, const dl_batch_shape* shape, const void* query, const dl_fp4_cache* cache,
                     const uint64_t* lengths, uint64_t window, uint64_t sinks, void* output, const float* scale,
                     void* workspace, uint64_t workspace_bytes) {
  return guard([&] {
    using namespace dl::fp4;
    require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
    Layout l = layout_of(shape, window, sinks, dtype == DL_BF16);
    const uint64_t bytes = bytes_of(shape, window, sinks);
    require(cache != nullptr, "null cache");
    require(query && cache->key_codes && cache->key_scales && cache->value_codes && cache->value_scales && lengths && output && scale,
            "null operand");
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    require(aligned(cache->key_codes) && aligned(cache->value_codes), "codes not 16-byte aligned");
    require(bytes == 0 || (workspace != nullptr && aligned(workspace)), "workspace null or not 16-byte aligned");
    require(workspace_bytes >= bytes, "workspace too small", DL_LENGTH_ERROR);
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
    a.whole_out = shape->width % 4 == 0 && reinterpret_cast<uintptr_t>(output) % (dtype == DL_BF16 ? 8 : 16) == 0;
    a.part = static_cast<float2*>(workspace);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.part_bytes);
    const bool pieces = (shape->width * (dtype == DL_BF16 ? 2 : 4)) % 16 == 0 && aligned(query);
    if (dtype == DL_BF16)
      launch_width<uint16_t>(queue->stream, l, pieces);
    else
      launch_width<float>(queue->stream, l, pieces);
    dl::check_launch(queue, "attention_fp4");
  });
}

}  // extern "C"
