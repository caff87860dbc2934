// Caches that grow and shrink by sequence: the append of new rows at each
// sequence's own length and position, and the eviction of the rows that
// received the least attention.  No reference counterpart: the reference's
// cache is one contiguous sequence whose slots are its positions.
//
// Caches are [batch][capacity][kv_heads][width]; every slot of a KV head has
// its position and its accumulated weight in [batch][kv_heads][capacity].
#include <algorithm>
#include <cstdint>

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
  const uint64_t n = a.lengths[b] < a.capacity ? a.lengths[b] : a.capacity, grown = n + a.rows;
  a.lengths_out[b] = grown < a.capacity ? grown : a.capacity;
  a.positions_out[b] = a.positions[b] + a.rows;
}

// One workgroup per new row.  The rotation's angles depend on the position and
// the feature only, so a row's cosines and sines are computed once, in 64 bits
// from the catalog's FP32 angle, for all its heads.  They and the products stay
// FP32 and a rotated value is rounded once, where the catalog's rotary rounds
// cosine, sine and each product to the storage type (0.26% against 0.17% off in
// BF16; the same bits in FP32).  Bound: the chain of 64-bit operations of one angle.
template <class T>
__global__ __launch_bounds__(kAppendThreads) void k_append(const AppendArgs a) {
  __shared__ float cosine[kAppendPairs], sine[kAppendPairs];
  const uint64_t b = blockIdx.y;
  const uint32_t half = a.width / 2;
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
    auto turn = [&](const T* x, T* y, uint32_t f) {
      const float lo = load_elem(x, f), hi = load_elem(x, f + half), c = cosine[f], s = sine[f];
      store_elem(y, f, lo * c - hi * s);
      store_elem(y, f + half, hi * c + lo * s);
    };
    const T* query = static_cast<const T*>(a.query) + row * a.q_heads * a.width;
    T* query_out = static_cast<T*>(a.query_out) + row * a.q_heads * a.width;
    for (uint32_t p = threadIdx.x; p < a.q_heads * half; p += kAppendThreads)
      turn(query + p / half * a.width, query_out + p / half * a.width, p % half);
    if (fits) {
      const uint64_t key_width = static_cast<uint64_t>(a.kv_heads) * a.width;
      const T* key = static_cast<const T*>(a.key) + row * key_width;
      const T* value = static_cast<const T*>(a.value) + row * key_width;
      T* to_key = static_cast<T*>(a.keys) + (b * a.capacity + slot) * key_width;
      T* to_value = static_cast<T*>(a.values) + (b * a.capacity + slot) * key_width;
      for (uint32_t p = threadIdx.x; p < a.kv_heads * half; p += kAppendThreads)
        turn(key + p / half * a.width, to_key + p / half * a.width, p % half);
      for (uint32_t f = threadIdx.x; f < key_width; f += kAppendThreads) to_value[f] = value[f];
      for (uint32_t h = threadIdx.x; h < a.kv_heads; h += kAppendThreads) {
        const uint64_t at = (b * a.kv_heads + h) * a.capacity + slot;
        a.slots[at] = static_cast<uint32_t>(position);
        a.weights[at] = 0.0f;
      }
    }
    __syncthreads();
  }
  // A sequence of one workgroup advances here: it has read its length, which
  // lengths_out may be.
  if (gridDim.x == 1 && threadIdx.x == 0) advance(a, b);
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
  uint32_t* moves;  // [batch][kv head][2][most]: holes, then the rows that fill them
  uint32_t* counts; // [batch][kv head]
  uint32_t kv_heads, width, capacity, budget, sinks, recent, most;
};

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

// Order of keeping as an unsigned number: protected rows above all weights, NaN
// as -infinity, the two zeros alike.
__device__ __forceinline__ uint32_t keep_key(float weight, uint32_t position, uint32_t newest, const EvictArgs& a) {
  if (position < a.sinks || static_cast<uint64_t>(position) + a.recent > newest) return 0xffffffffu;
  if (!(weight == weight)) weight = -INFINITY;
  const uint32_t bits = __float_as_uint(weight == 0.0f ? 0.0f : weight);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Sum over the workgroup of each thread's value, and the sum of the threads before.
__device__ __forceinline__ uint32_t scan(uint32_t value, uint32_t* wave_sums, uint32_t& total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint32_t run = value;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const uint32_t other = __shfl_up(run, off);
    if (lane >= off) run += other;
  }
  if (lane == 63) wave_sums[wave] = run;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    const uint32_t s = wave_sums[w];
    before += w < wave ? s : 0;
    total += s;
  }
  __syncthreads();
  return before + run - value;
}

// One workgroup per sequence and KV head: the budget-th largest key by its
// bytes from the top, then one ordered pass that writes what stays and lists
// the holes below the budget and the kept rows above it.
__global__ __launch_bounds__(kSelectThreads) void k_select(const EvictArgs a) {
  __shared__ uint32_t histogram[256];
  __shared__ uint32_t wave_sums[kSelectWaves];
  __shared__ uint32_t shared_prefix, shared_left;
  const uint32_t head = blockIdx.x, b = head / a.kv_heads, tid = threadIdx.x;
  const uint64_t length = a.lengths[b];
  const uint32_t n = length < a.capacity ? static_cast<uint32_t>(length) : a.capacity;
  const float* weights = a.weights + static_cast<uint64_t>(head) * a.capacity;
  const uint32_t* slots = a.slots + static_cast<uint64_t>(head) * a.capacity;
  float* weights_out = a.weights_out + static_cast<uint64_t>(head) * a.capacity;
  uint32_t* slots_out = a.slots_out + static_cast<uint64_t>(head) * a.capacity;
  if (n <= a.budget) {
    for (uint32_t s = tid; s < n; s += kSelectThreads) {
      weights_out[s] = weights[s];
      slots_out[s] = slots[s];
    }
    if (tid == 0) a.counts[head] = 0;
    return;
  }
  uint32_t newest = 0;
  for (uint32_t s = tid; s < n; s += kSelectThreads) newest = max(newest, slots[s]);
#pragma unroll
  for (int off = 32; off; off /= 2) newest = max(newest, static_cast<uint32_t>(__shfl_xor(newest, off)));
  if (tid % 64 == 0) wave_sums[tid / 64] = newest;
  __syncthreads();
  for (int w = 0; w < kSelectWaves; ++w) newest = max(newest, wave_sums[w]);
  __syncthreads();

  // `left`: how many of the keys that share the bytes found so far stay.
  uint32_t found = 0, left = a.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) histogram[tid] = 0;
    __syncthreads();
    const uint32_t above = shift == 24 ? 0 : 0xffffffffu << (shift + 8);
    for (uint32_t s = tid; s < n; s += kSelectThreads) {
      const uint32_t key = keep_key(weights[s], slots[s], newest, a);
      if ((key & above) == found) atomicAdd(&histogram[key >> shift & 255], 1u);
    }
    __syncthreads();
    // Thread t < 256 holds byte 255 - t: the keys at or above it are a running sum.
    uint32_t total;
    const uint32_t mine = tid < 256 ? histogram[255 - tid] : 0;
    const uint32_t before = scan(mine, wave_sums, total);
    if (before < left && before + mine >= left) {
      shared_prefix = found | (255 - tid) << shift;
      shared_left = left - before;
    }
    __syncthreads();
    found = shared_prefix;
    left = shared_left;
    __syncthreads();
  }

  uint32_t equal_before = 0, holes = 0, fillers = 0;
  uint32_t* hole = a.moves + static_cast<uint64_t>(head) * 2 * a.most;
  uint32_t* filler = hole + a.most;
  for (uint32_t base = 0; base < n; base += kSelectThreads) {
    const uint32_t s = base + tid;
    const uint32_t key = s < n ? keep_key(weights[s], slots[s], newest, a) : 0;
    uint32_t total;
    const uint32_t equal = s < n && key == found;
    const uint32_t rank = equal_before + scan(equal, wave_sums, total);
    equal_before += total;
    const bool kept = s < n && (key > found || (equal && rank < left));
    const uint32_t listed = s < n && kept != (s < a.budget);  // a hole below the budget, a kept row above it
    // Rows of one round may lie on both sides of the budget: two sums in one.
    const uint32_t packed = scan(s < a.budget ? listed : listed << 16, wave_sums, total);
    if (listed) {
      if (s < a.budget)
        hole[holes + (packed & 0xffff)] = s;
      else
        filler[fillers + (packed >> 16)] = s;
    }
    holes += total & 0xffff;
    fillers += total >> 16;
    if (kept && s < a.budget) {
      weights_out[s] = weights[s];
      slots_out[s] = slots[s];
    }
  }
  if (tid == 0) a.counts[head] = holes;
  __threadfence_block();
  __syncthreads();
  // Sources lie at or above the budget and are written by nobody, so the
  // outputs may be the inputs.
  for (uint32_t j = tid; j < holes; j += kSelectThreads) {
    weights_out[hole[j]] = weights[filler[j]];
    slots_out[hole[j]] = slots[filler[j]];
  }
}

// Moves the listed rows' pieces of K and V.  Holes lie below the budget and
// their sources at or above it, so the moves are independent of each other.
template <class Piece>
__global__ __launch_bounds__(256) void k_move(const EvictArgs a, uint32_t row_pieces) {
  const uint32_t head = blockIdx.y, b = head / a.kv_heads, h = head % a.kv_heads;
  const uint32_t count = a.counts[head];
  const uint32_t* hole = a.moves + static_cast<uint64_t>(head) * 2 * a.most;
  const uint32_t* filler = hole + a.most;
  const uint64_t stride = static_cast<uint64_t>(a.kv_heads) * row_pieces;
  const uint64_t base = static_cast<uint64_t>(b) * a.capacity * stride + static_cast<uint64_t>(h) * row_pieces;
  Piece* keys = static_cast<Piece*>(a.keys) + base;
  Piece* values = static_cast<Piece*>(a.values) + base;
  const uint64_t pieces = static_cast<uint64_t>(count) * row_pieces;
  for (uint64_t p = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; p < pieces; p += static_cast<uint64_t>(gridDim.x) * 256) {
    const uint64_t j = p / row_pieces, f = p % row_pieces;
    const uint64_t to = hole[j] * stride + f, from = filler[j] * stride + f;
    keys[to] = keys[from];
    values[to] = values[from];
  }
  // This launch reads no length, so lengths_out may be the lengths.
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    const uint64_t n = a.lengths[b];
    a.lengths_out[b] = n < a.budget ? n : a.budget;
  }
}

uint32_t most_moves(const dl_batch_shape* shape, uint64_t budget) {
  return static_cast<uint32_t>(budget < shape->capacity ? std::min(budget, shape->capacity - budget) : 0);
}

uint64_t evict_bytes(const dl_batch_shape* shape, uint64_t budget) {
  check_shape(shape);
  require(budget > 0, "empty budget");
  return shape->batch * shape->kv_heads * (1 + 2ull * most_moves(shape, budget)) * 4;
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
    const dim3 grid(static_cast<unsigned>(shape->rows), static_cast<unsigned>(shape->batch));
    if (dtype == DL_BF16)
      k_append<uint16_t><<<grid, kAppendThreads, 0, queue->stream>>>(a);
    else
      k_append<float><<<grid, kAppendThreads, 0, queue->stream>>>(a);
    if (grid.x > 1)
      k_advance<<<static_cast<unsigned>(dl::ceil_div(shape->batch, 64)), 64, 0, queue->stream>>>(a, shape->batch);
    dl::check_launch(queue, "cache_append");
  });
}

int dl_cache_evict_bytes(const dl_batch_shape* shape, uint64_t budget, uint64_t* bytes) {
  return guard([&] {
    require(bytes != nullptr, "null output");
    *bytes = dl::batch::evict_bytes(shape, budget);
  });
}

int dl_cache_evict(dl_queue* queue, int dtype, const dl_batch_shape* shape, void* keys, void* values,
                   const uint64_t* lengths, uint64_t* lengths_out, const uint32_t* slots, uint32_t* slots_out,
                   const float* weights, float* weights_out, uint64_t budget, uint64_t sinks, uint64_t recent,
                   void* workspace, uint64_t workspace_bytes) {
  return guard([&] {
    using namespace dl::batch;
    require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
    const uint64_t needed = evict_bytes(shape, budget);
    require(keys && values && lengths && lengths_out && slots && slots_out && weights && weights_out, "null operand");
    require(sinks <= budget && recent <= budget - sinks, "sinks and recent rows exceed the budget");
    const uint64_t heads = shape->batch * shape->kv_heads;
    require(heads <= 65535, "too many sequences", DL_LENGTH_ERROR);
    require(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "workspace null or not 4-byte aligned");
    require(workspace_bytes >= needed, "workspace too small", DL_LENGTH_ERROR);
    dl::enter(queue);
    EvictArgs a{keys, values, lengths, lengths_out, slots, slots_out, weights, weights_out, nullptr,
                static_cast<uint32_t*>(workspace), static_cast<uint32_t>(shape->kv_heads),
                static_cast<uint32_t>(shape->width), static_cast<uint32_t>(shape->capacity),
                static_cast<uint32_t>(std::min(budget, shape->capacity)), static_cast<uint32_t>(std::min<uint64_t>(sinks, kMostKeys)),
                static_cast<uint32_t>(std::min<uint64_t>(recent, kMostKeys)), most_moves(shape, budget)};
    a.moves = a.counts + heads;
    k_select<<<static_cast<unsigned>(heads), kSelectThreads, 0, queue->stream>>>(a);
    const uint64_t size = dtype == DL_BF16 ? 2 : 4, row_bytes = shape->width * size;
    auto move = [&](auto piece) {
      using Piece = decltype(piece);
      const uint32_t row_pieces = static_cast<uint32_t>(row_bytes / sizeof(Piece));
      const uint64_t blocks = dl::ceil_div(static_cast<uint64_t>(a.most) * row_pieces, 256 * 4);
      const dim3 grid(static_cast<unsigned>(std::min<uint64_t>(std::max<uint64_t>(blocks, 1), 256)), static_cast<unsigned>(heads));
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
