// Caches that grow and shrink by sequence: the append of new rows at each
// sequence's own length and position, and the eviction of the rows that
// received the least attention.  No reference counterpart: the reference's
// cache is one contiguous sequence whose slots are its positions.
//
// Caches are [batch][capacity][kv_heads][width]; every slot of a KV head has
// its position and its accumulated weight in [batch][kv_heads][capacity].
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "batch.h"
#include "dl_device.h"
#include "dl_internal.h"

namespace dl::batch {
namespace {

// ------------------------------------------------------------------- append
struct AppendArgs {
  const void *query, *key, *value;
  void *query_out, *keys, *values;
  const uint64_t *lengths, *positions;
  uint64_t *lengths_out, *positions_out;
  uint32_t* slots;
  float* weights;
  uint64_t rows, capacity;
  uint32_t q_heads, kv_heads, width;
  double theta;
};

constexpr int kAppendThreads = 256, kAppendPairs = 2048;

__device__ __forceinline__ void advance(const AppendArgs& a, uint64_t b) {
  const uint64_t n = a.lengths[b] < a.capacity ? a.lengths[b] : a.capacity, grown = n + a.rows, first = a.positions[b];
  a.lengths_out[b] = grown < a.capacity ? grown : a.capacity;
  a.positions_out[b] = first + a.rows;
}

// One workgroup per new row.  The rotation's angles depend on the position and
// the feature only, so a row's cosines and sines are computed once, in 64 bits
// from the catalog's FP32 angle, for all its heads.  They and the products stay
// FP32 and a rotated value is rounded once, where the catalog's rotary rounds
// cosine, sine and each product to the storage type (0.26% against 0.17% off in
// BF16; the same bits in FP32).  Bound: the chain of 64-bit operations of one angle.
template <class T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

// N features of a head at a time: 4 where halves of a head are whole packs of
// 4 and the operands lie on their boundaries, else 1.
template <class T, int N>
__global__ __launch_bounds__(kAppendThreads) void k_append(const AppendArgs a, bool advance_here) {
  using Features = Pack<T, N>;
  __shared__ __align__(16) float cosine[kAppendPairs], sine[kAppendPairs];
  const uint64_t b = blockIdx.y;
  const uint32_t half = a.width / 2, packs = half / N;
  const uint64_t n = a.lengths[b], first = a.positions[b];
  for (uint64_t i = blockIdx.x; i < a.rows; i += gridDim.x) {
    const uint64_t position = first + i, slot = n + i, row = b * a.rows + i;
    const bool fits = n < a.capacity && i < a.capacity - n;
    for (uint32_t f = threadIdx.x; f < half; f += kAppendThreads) {
      const float exponent = static_cast<float>(2 * f) / static_cast<float>(a.width);
      const float frequency = static_cast<float>(1.0 / dl_pow_pos(a.theta, static_cast<double>(exponent)));
      const float angle = static_cast<float>(position) * frequency;
      double s, c;
      dl_sincos(static_cast<double>(angle), &s, &c);
      cosine[f] = static_cast<float>(c);
      sine[f] = static_cast<float>(s);
    }
    __syncthreads();
    auto turn = [&](const T* x, T* y, uint32_t heads) {
      for (uint32_t p = threadIdx.x; p < heads * packs; p += kAppendThreads) {
        const uint32_t at = p / packs * a.width, f = p % packs * N;
        const Features lo = *reinterpret_cast<const Features*>(x + at + f), hi = *reinterpret_cast<const Features*>(x + at + half + f);
        Features lo_out, hi_out;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float u = load_elem(lo.v, e), v = load_elem(hi.v, e), c = cosine[f + e], s = sine[f + e];
          store_elem(lo_out.v, e, u * c - v * s);
          store_elem(hi_out.v, e, v * c + u * s);
        }
        *reinterpret_cast<Features*>(y + at + f) = lo_out;
        *reinterpret_cast<Features*>(y + at + half + f) = hi_out;
      }
    };
    const uint64_t query_at = row * a.q_heads * a.width;
    turn(static_cast<const T*>(a.query) + query_at, static_cast<T*>(a.query_out) + query_at, a.q_heads);
    if (fits) {
      const uint32_t key_width = a.kv_heads * a.width;
      const uint64_t from = row * key_width, to = (b * a.capacity + slot) * key_width;
      turn(static_cast<const T*>(a.key) + from, static_cast<T*>(a.keys) + to, a.kv_heads);
      const Features* value = reinterpret_cast<const Features*>(static_cast<const T*>(a.value) + from);
      Features* to_value = reinterpret_cast<Features*>(static_cast<T*>(a.values) + to);
      for (uint32_t f = threadIdx.x; f < key_width / N; f += kAppendThreads) to_value[f] = value[f];
      for (uint32_t h = threadIdx.x; h < a.kv_heads; h += kAppendThreads) {
        const uint64_t at = (b * a.kv_heads + h) * a.capacity + slot;
        a.slots[at] = static_cast<uint32_t>(position);
        a.weights[at] = 0.0f;
      }
    }
    __syncthreads();
  }
  if (advance_here && blockIdx.x == 0 && threadIdx.x == 0) advance(a, b);
}

__global__ __launch_bounds__(64) void k_advance(const AppendArgs a, uint64_t batch) {
  const uint64_t b = static_cast<uint64_t>(blockIdx.x) * 64 + threadIdx.x;
  if (b < batch) advance(a, b);
}

// ------------------------------------------------------------------ eviction
struct EvictArgs {
  void *keys, *values;
  const uint64_t* lengths;
  uint64_t* lengths_out;
  const uint32_t* slots;
  uint32_t* slots_out;
  const float* weights;
  float* weights_out;
  uint2* counts;   // [batch][kv head]: rows that move, rows that stay
  uint64_t* kept;  // [batch][kv head][kept_words]: a bit per slot below the budget
  uint32_t* moves; // [batch][kv head][2][most]: holes, then the rows that fill them
  uint32_t kv_heads, width, capacity, budget, sinks, recent, most, kept_words;
};

constexpr uint32_t kProtected = 0xffffffffu;

// Order of keeping as an unsigned number, never 0: protected rows above all
// weights, NaN as -infinity (the maximum drops it), the two zeros alike (-0 + 0
// is 0).  A row is not protected if its position is one of `open` from the
// sinks on.
__device__ __forceinline__ uint32_t keep_key(float weight, uint32_t position, uint32_t sinks, uint64_t open) {
  if (position - sinks >= open) return kProtected;
  const uint32_t bits = __float_as_uint(fmaxf(weight, -INFINITY) + 0.0f);
  return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}

constexpr int kBins = 2048;

__device__ __forceinline__ uint64_t lane_of(uint64_t v, uint32_t lane) {
  const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane);
  return static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane)) << 32 | low;
}

// One workgroup per sequence and KV head finds the budget-th largest key and
// lists the holes below the budget and the kept rows above it.  Keys are held in
// LDS, or made again from the operands in every pass where a cache is longer
// than kHeldKeys.  The key is found by histograms of kBins bins over the range
// that still holds it, first from the least to the largest key: at most three,
// and the later ones count few keys.  Then a wavefront takes consecutive groups
// of 64 slots, so that its ranks are running sums of population counts, from
// one sum over the wavefronts.  Bound: the chain of barriers and of LDS and
// instruction latency, one compute unit to a head: of 36 us for 32768 rows 12
// are the two reads, 15 the histograms, 8 masks and lists (of 8 us for 2049
// rows 2.7, 5.6 and 3).  Keys in registers by thread, 40 unrolled, read the
// operands at a stride and fetched five times the code: 81 us against 44 for
// the launch.
constexpr uint32_t kHeldKeys = 36 * 1024;

template <int Threads, bool Held>
__global__ __launch_bounds__(Threads) void k_select(const EvictArgs a) {
  constexpr uint32_t kWaves = Threads / 64;
  extern __shared__ uint32_t held[];
  __shared__ uint32_t histogram[kBins];
  __shared__ uint32_t sums[3][kWaves];
  __shared__ uint32_t at_bin, at_left, at_count;
  const uint32_t head = blockIdx.x, tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint64_t length = a.lengths[head / a.kv_heads];
  const uint32_t n = length < a.capacity ? static_cast<uint32_t>(length) : a.capacity;
  if (n <= a.budget) {
    if (tid == 0) a.counts[head] = make_uint2(0, n);
    return;
  }
  const float* weights = a.weights + static_cast<uint64_t>(head) * a.capacity;
  const uint32_t* slots = a.slots + static_cast<uint64_t>(head) * a.capacity;

  // use(slot, load(slot)) for every slot, eight loads of a thread at a time.
  auto each_slot = [&](auto&& load, auto&& use) {
    constexpr int kBatch = 8;
    for (uint32_t base = tid; base < n; base += kBatch * Threads) {
      decltype(load(0u)) v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) v[i] = load(min(base + i * Threads, n - 1));
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (base + i * Threads < n) use(base + i * Threads, v[i]);
    }
  };
  uint32_t newest = 0;
  each_slot([&](uint32_t s) { return slots[s]; },
            [&](uint32_t s, uint32_t position) {
              if constexpr (Held) held[s] = position;
              newest = max(newest, position);
            });
#pragma unroll
  for (int off = 32; off; off /= 2) newest = max(newest, static_cast<uint32_t>(__shfl_xor(newest, off)));
  if (lane == 0) sums[0][wave] = newest;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) newest = max(newest, sums[0][w]);
  __syncthreads();

  // Positions sinks .. newest - recent are open to eviction.
  const uint64_t kept_ends = static_cast<uint64_t>(a.sinks) + a.recent, all_positions = static_cast<uint64_t>(newest) + 1;
  const uint64_t open = all_positions > kept_ends ? all_positions - kept_ends : 0;
  uint32_t low = kProtected, high = 0, safe = 0;
  each_slot([&](uint32_t s) { return weights[s]; },
            [&](uint32_t s, float weight) {
              const uint32_t key = keep_key(weight, Held ? held[s] : slots[s], a.sinks, open);
              if constexpr (Held) held[s] = key;
              const bool is_safe = key == kProtected;
              safe += is_safe;
              low = min(low, key);
              high = max(high, is_safe ? 0u : key);
            });
#pragma unroll
  for (int off = 32; off; off /= 2) {
    low = min(low, static_cast<uint32_t>(__shfl_xor(low, off)));
    high = max(high, static_cast<uint32_t>(__shfl_xor(high, off)));
    safe += __shfl_xor(safe, off);
  }
  if (lane == 0) {
    sums[0][wave] = low;
    sums[1][wave] = high;
    sums[2][wave] = safe;
  }
  __syncthreads();
  safe = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    low = min(low, sums[0][w]);
    high = max(high, sums[1][w]);
    safe += sums[2][w];
  }
  auto key_of = [&](uint32_t s) { return Held ? held[s] : keep_key(weights[s], slots[s], a.sinks, open); };

  // Keys above `found` stay, and of those equal to it the first `left`.
  uint32_t found = kProtected, left = a.budget;
  if (safe < a.budget) {
    left = a.budget - safe;
    while (true) {
      const uint32_t span = high - low;
      const int bits = span ? 32 - __builtin_clz(span) : 0, shift = bits > 11 ? bits - 11 : 0;
      for (uint32_t i = tid; i < kBins; i += Threads) histogram[i] = 0;
      __syncthreads();
      each_slot(key_of, [&](uint32_t, uint32_t key) {
        if (key < low || key > high) return;
        const uint32_t bin = (key - low) >> shift;
        // Rows of one weight, new ones above all, would queue for one word.
        if (__all(bin == static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(bin)))) {
          const uint64_t here = __ballot(1);
          if (lane == static_cast<uint32_t>(__builtin_ctzll(here)))
            atomicAdd(&histogram[bin], static_cast<uint32_t>(__popcll(here)));
        } else {
          atomicAdd(&histogram[bin], 1u);
        }
      });
      __syncthreads();
      // A thread holds the bins below those of the threads before it.
      constexpr int kEach = kBins / Threads;
      uint32_t count[kEach], mine = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) mine += count[i] = histogram[kBins - 1 - (tid * kEach + i)];
      uint32_t before = mine;
#pragma unroll
      for (int off = 1; off < 64; off *= 2) {
        const uint32_t other = __shfl_up(before, off);
        if (lane >= static_cast<uint32_t>(off)) before += other;
      }
      if (lane == 63) sums[0][wave] = before;
      before -= mine;
      __syncthreads();
#pragma unroll
      for (uint32_t w = 0; w < kWaves; ++w) before += w < wave ? sums[0][w] : 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (before < left && before + count[i] >= left) {
          at_bin = kBins - 1 - (tid * kEach + i);
          at_left = left - before;
          at_count = count[i];
        }
        before += count[i];
      }
      __syncthreads();
      low += at_bin << shift;
      high = min(high, low + (1u << shift) - 1);
      left = at_left;
      found = low;
      if (at_count == left) {  // all of them stay
        --found;
        left = 0;
        break;
      }
      if (shift == 0) break;
    }
  }
  __syncthreads();

  // A wavefront takes consecutive groups of 64 slots, 64 groups (a part) at a
  // time, a lane holding one group's masks.  Held keys are one part.
  const uint32_t groups = (n + 63) / 64, each = (groups + kWaves - 1) / kWaves;
  const uint32_t first = min(wave * each, groups), last = min(first + each, groups);
  auto masks = [&](uint32_t part, uint64_t& above, uint64_t& equal) {
    above = equal = 0;
    const uint32_t count = min(last - part, 64u);
    for (uint32_t i = 0; i < count; i += 4) {
      uint32_t keys[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t s = 64 * (part + i + j) + lane;
        keys[j] = s < n ? key_of(s) : 0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t over = __ballot(keys[j] > found), same = __ballot(keys[j] == found);
        if (lane == i + j) {
          above = over;
          equal = same;
        }
      }
    }
    if (lane >= count) above = equal = 0;
  };
  // Sum over the wavefront's lanes, and this lane's sum of those before it.
  auto running = [&](uint32_t value, uint32_t& total) {
    uint32_t run = value;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const uint32_t other = __shfl_up(run, off);
      if (lane >= static_cast<uint32_t>(off)) run += other;
    }
    total = __shfl(run, 63);
    return run - value;
  };
  uint64_t above = 0, equal = 0;
  uint32_t ties = 0, total;
  if (Held) masks(first, above, equal);
  if (left) {
    for (uint32_t part = first; part < last; part += 64) {
      if (!Held) masks(part, above, equal);
      running(__popcll(equal), total);
      ties += total;
    }
    if (lane == 0) sums[0][wave] = ties;
    __syncthreads();
    ties = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) ties += w < wave ? sums[0][w] : 0;
  }
  // Of the group's equal keys the lowest slots stay, as many as are left.
  auto settle = [&](uint32_t& before) {
    uint64_t kept = above;
    if (left) {
      const uint32_t mine = before + running(__popcll(equal), total);
      const uint32_t room = mine < left ? left - mine : 0;
      while (static_cast<uint32_t>(__popcll(equal)) > room) equal &= ~(1ull << (63 - __builtin_clzll(equal)));
      kept |= equal;
      before += total;
    }
    return kept;
  };
  // The slots of a group below the budget.
  auto below_budget = [&](uint32_t part) {
    const uint32_t s = 64 * (part + lane);
    return s >= a.budget ? 0 : a.budget - s >= 64 ? ~0ull : (1ull << (a.budget - s)) - 1;
  };
  uint32_t holes = 0, fillers = 0, before = ties;
  for (uint32_t part = first; part < last; part += 64) {
    if (!Held) masks(part, above, equal);
    const uint64_t kept = settle(before), inside = below_budget(part);
    if (Held) above = kept;
    const bool real = part + lane < last;
    running(real ? __popcll(inside & ~kept) : 0, total);
    holes += total;
    running(real ? __popcll(kept & ~inside) : 0, total);
    fillers += total;
  }
  if (lane == 0) {
    sums[1][wave] = holes;
    sums[2][wave] = fillers;
  }
  __syncthreads();
  uint32_t moving = 0;
  holes = fillers = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    moving += sums[1][w];
    holes += w < wave ? sums[1][w] : 0;
    fillers += w < wave ? sums[2][w] : 0;
  }
  uint32_t* hole = a.moves + static_cast<uint64_t>(head) * 2 * a.most;
  uint32_t* filler = hole + a.most;
  uint64_t* words = a.kept + static_cast<uint64_t>(head) * a.kept_words;
  before = ties;
  for (uint32_t part = first; part < last; part += 64) {
    if (!Held) masks(part, above, equal);
    const uint64_t kept = Held ? above : settle(before), inside = below_budget(part);
    const bool real = part + lane < last;
    const uint64_t empty = real ? inside & ~kept : 0, extra = real ? kept & ~inside : 0;
    if (real && inside) words[part + lane] = kept;
    const uint32_t hole_at = holes + running(__popcll(empty), total);
    holes += total;
    const uint32_t filler_at = fillers + running(__popcll(extra), total);
    fillers += total;
    const uint32_t count = min(last - part, 64u);
    for (uint32_t i = 0; i < count; ++i) {  // one group's slots over the lanes
      const uint64_t here = 1ull << lane, under = here - 1;
      const uint64_t out = lane_of(empty, i), in = lane_of(extra, i);
      const uint32_t to_hole = __builtin_amdgcn_readlane(hole_at, i), to_filler = __builtin_amdgcn_readlane(filler_at, i);
      const uint32_t s = 64 * (part + i) + lane;
      if (out & here) hole[to_hole + __popcll(out & under)] = s;
      if (in & here) filler[to_filler + __popcll(in & under)] = s;
    }
  }
  if (tid == 0) a.counts[head] = make_uint2(moving, a.budget);
}

// Moves the listed rows' pieces of K and V and their weights and positions, and
// copies those of the rows that stay.  Holes lie below the budget and their
// sources at or above it, so no row is both read and written and the outputs
// may be the inputs; no length is read, so neither need lengths_out differ.
// Bound by the copy: 64 heads, 268 MB read and written in 65 us, 4.1 TB/s (a
// large copy reaches 4.9).
template <class Piece>
__global__ __launch_bounds__(256) void k_move(const EvictArgs a, uint32_t row_pieces) {
  const uint32_t head = blockIdx.y, b = head / a.kv_heads, h = head % a.kv_heads;
  const uint32_t moving = a.counts[head].x, left = a.counts[head].y;
  const uint32_t* hole = a.moves + static_cast<uint64_t>(head) * 2 * a.most;
  const uint32_t* filler = hole + a.most;
  const uint32_t first = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  const uint64_t line = static_cast<uint64_t>(head) * a.capacity;
  if (a.weights_out != a.weights || a.slots_out != a.slots) {
    const uint64_t* kept = a.kept + static_cast<uint64_t>(head) * a.kept_words;
    const bool all = left < a.budget || moving == 0;
    for (uint32_t s = first; s < left; s += step)
      if (all || kept[s / 64] >> (s % 64) & 1) {
        a.weights_out[line + s] = a.weights[line + s];
        a.slots_out[line + s] = a.slots[line + s];
      }
  }
  for (uint32_t j = first; j < moving; j += step) {
    a.weights_out[line + hole[j]] = a.weights[line + filler[j]];
    a.slots_out[line + hole[j]] = a.slots[line + filler[j]];
  }
  const uint64_t stride = static_cast<uint64_t>(a.kv_heads) * row_pieces;
  const uint64_t base = static_cast<uint64_t>(b) * a.capacity * stride + static_cast<uint64_t>(h) * row_pieces;
  Piece* keys = static_cast<Piece*>(a.keys) + base;
  Piece* values = static_cast<Piece*>(a.values) + base;
  const uint64_t pieces = static_cast<uint64_t>(moving) * row_pieces;
  auto move = [&](auto count) {  // 32-bit divisions where they do
    using Index = decltype(count);
    for (Index p = first; p < count; p += step) {
      const uint32_t j = static_cast<uint32_t>(p / row_pieces), f = static_cast<uint32_t>(p % row_pieces);
      const uint64_t to = hole[j] * stride + f, from = filler[j] * stride + f;
      const Piece key = keys[from], value = values[from];
      keys[to] = key;
      values[to] = value;
    }
  };
  if (pieces < (1u << 31))
    move(static_cast<uint32_t>(pieces));
  else
    move(pieces);
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.lengths_out[b] = left;
}

// What an eviction keeps in its workspace.
struct EvictLayout {
  uint64_t heads, most, kept_words;
  uint64_t counts() const { return heads * 8; }
  uint64_t kept() const { return heads * kept_words * 8; }
  uint64_t bytes() const { return counts() + kept() + heads * 2 * most * 4; }
};

EvictLayout evict_layout(const dl_batch_shape* shape, uint64_t budget) {
  check_shape(shape);
  require(budget > 0, "empty budget");
  require(shape->batch * shape->kv_heads <= 65535, "too many sequences", DL_LENGTH_ERROR);
  const bool cuts = budget < shape->capacity;
  return {shape->batch * shape->kv_heads, cuts ? std::min(budget, shape->capacity - budget) : 0, cuts ? dl::ceil_div(budget, 64) : 0};
}

}  // namespace
}  // namespace dl::batch

using dl::guard;
using dl::require;

extern "C" {

int dl_cache_append(dl_queue* queue, int dtype, const dl_batch_shape* shape, const void* query, const void* key,
                    const void* value, void* query_out, void* keys, void* values, const uint64_t* lengths,
                    uint64_t* lengths_out, const uint64_t* positions, uint64_t* positions_out, uint32_t* slots,
                    float* weights, double theta) {
  return guard([&] {
    using namespace dl::batch;
    require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
    check_shape(shape);
    require(query && key && value && query_out && keys && values && lengths && lengths_out && positions && positions_out &&
                slots && weights,
            "null operand");
    require(shape->width % 2 == 0, "rotated width must be even");
    require(shape->width / 2 <= kAppendPairs, "head width above 4096", DL_LENGTH_ERROR);
    require(shape->width <= kMostRow / shape->query_heads, "query rows too wide", DL_LENGTH_ERROR);
    require(shape->batch <= 65535, "too many sequences", DL_LENGTH_ERROR);
    require(theta > 0.0 && theta < 1e300, "theta must be positive and finite");
    dl::enter(queue);
    const AppendArgs a{query, key, value, query_out, keys, values, lengths, positions, lengths_out, positions_out, slots, weights,
                       shape->rows, shape->capacity, static_cast<uint32_t>(shape->query_heads),
                       static_cast<uint32_t>(shape->kv_heads), static_cast<uint32_t>(shape->width), theta};
    const dim3 grid(static_cast<unsigned>(std::min<uint64_t>(shape->rows, 1u << 20)), static_cast<unsigned>(shape->batch));
    // A sequence's only workgroup has read its length before it writes the new
    // one, which may be the same word; of several any may still have to.
    const bool apart = lengths != lengths_out && positions != positions_out && lengths != positions_out && positions != lengths_out;
    const bool advance_here = grid.x == 1 || apart;
    uintptr_t low = shape->width / 2 % 4;
    for (const void* p : {query, key, value, static_cast<const void*>(query_out), static_cast<const void*>(keys), static_cast<const void*>(values)})
      low |= reinterpret_cast<uintptr_t>(p) % (dtype == DL_BF16 ? 8 : 16);
    auto run = [&](auto type, auto count) {
      k_append<decltype(type), decltype(count)::value><<<grid, kAppendThreads, 0, queue->stream>>>(a, advance_here);
    };
    using Four = std::integral_constant<int, 4>;
    using One = std::integral_constant<int, 1>;
    if (dtype == DL_BF16)
      low ? run(uint16_t{}, One{}) : run(uint16_t{}, Four{});
    else
      low ? run(float{}, One{}) : run(float{}, Four{});
    if (!advance_here)
      k_advance<<<static_cast<unsigned>(dl::ceil_div(shape->batch, 64)), 64, 0, queue->stream>>>(a, shape->batch);
    dl::check_launch(queue, "cache_append");
  });
}

int dl_cache_evict_bytes(const dl_batch_shape* shape, uint64_t budget, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::batch::evict_layout(shape, budget).bytes();
  });
}

int dl_cache_evict(dl_queue* queue, int dtype, const dl_batch_shape* shape, void* keys, void* values,
                   const uint64_t* lengths, uint64_t* lengths_out, const uint32_t* slots, uint32_t* slots_out,
                   const float* weights, float* weights_out, uint64_t budget, uint64_t sinks, uint64_t recent,
                   void* workspace, uint64_t workspace_bytes) {
  return guard([&] {
    using namespace dl::batch;
    require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
    const EvictLayout l = evict_layout(shape, budget);
    require(keys && values && lengths && lengths_out && slots && slots_out && weights && weights_out, "null operand");
    require(sinks <= budget && recent <= budget - sinks, "sinks and recent rows exceed the budget");
    require(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "workspace null or not 8-byte aligned");
    require(workspace_bytes >= l.bytes(), "workspace too small", DL_LENGTH_ERROR);
    dl::enter(queue);
    char* room = static_cast<char*>(workspace);
    auto word = [](uint64_t v) { return static_cast<uint32_t>(std::min<uint64_t>(v, kMostKeys)); };
    const EvictArgs a{keys, values, lengths, lengths_out, slots, slots_out, weights, weights_out,
                      reinterpret_cast<uint2*>(room), reinterpret_cast<uint64_t*>(room + l.counts()),
                      reinterpret_cast<uint32_t*>(room + l.counts() + l.kept()), static_cast<uint32_t>(shape->kv_heads),
                      static_cast<uint32_t>(shape->width), static_cast<uint32_t>(shape->capacity),
                      word(std::min(budget, shape->capacity)), word(sinks), word(recent), static_cast<uint32_t>(l.most),
                      static_cast<uint32_t>(l.kept_words)};
    const unsigned heads = static_cast<unsigned>(l.heads);
    if (shape->capacity <= 1024)
      k_select<256, true><<<heads, 256, shape->capacity * 4, queue->stream>>>(a);
    else if (shape->capacity <= kHeldKeys)
      k_select<1024, true><<<heads, 1024, shape->capacity * 4, queue->stream>>>(a);
    else
      k_select<1024, false><<<heads, 1024, 0, queue->stream>>>(a);
    const uint64_t size = dtype == DL_BF16 ? 2 : 4, row_bytes = shape->width * size;
    auto move = [&](auto piece) {
      using Piece = decltype(piece);
      const uint32_t row_pieces = static_cast<uint32_t>(row_bytes / sizeof(Piece));
      const uint64_t blocks = dl::ceil_div(std::max(l.most * row_pieces, std::min(budget, shape->capacity)), 256 * 4);
      const dim3 grid(static_cast<unsigned>(std::min<uint64_t>(blocks, 256)), heads);
      k_move<Piece><<<grid, 256, 0, queue->stream>>>(a, row_pieces);
    };
    if (whole_pieces(shape, size, {keys, values}))
      move(dl::u32x4{});
    else if (size == 4)
      move(uint32_t{});
    else
      move(uint16_t{});
    dl::check_launch(queue, "cache_evict");
  });
}

}  // extern "C"
