// Rows held in 4 bits (fp4.h): quantising and reading back, the projection by
// 4-bit weights, and the append of new rows to caches held in 4 bits.  No
// reference counterpart: the reference stores weights and caches in BF16 or FP32.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "batch.h"
#include "dl_device.h"
#include "dl_internal.h"
#include "fp4.h"

namespace dl::fp4 {
namespace {

// Eight consecutive elements of a row that has `width`, from `at` on; zeros past
// the width.  Pieces: the row is whole 16-byte pieces.
template <class T, bool kPieces>
__device__ __forceinline__ void load_eight(const T* row, uint32_t at, uint32_t width, float (&x)[8]) {
  if constexpr (kPieces) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
      const u32x4 v = at + i * kPer < width ? *reinterpret_cast<const u32x4*>(row + at + i * kPer) : u32x4{};
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if constexpr (sizeof(T) == 4)
          x[i * kPer + e] = __uint_as_float(v[e]);
        else
          x[i * kPer + e] = e % 2 ? dl_bf16_hi(v[e / 2]) : dl_bf16_lo(v[e / 2]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = at + e < width ? load_elem(row, at + e) : 0.0f;
  }
}

__device__ __forceinline__ uint32_t largest_of(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (float v : x) m = max(m, magnitude(v));
  return m;
}
// Over the four lanes of a group, eight values each.
__device__ __forceinline__ uint32_t group_largest(uint32_t m) {
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 1)));
  return max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 2)));
}

// ------------------------------------------------------ quantise and read back
// Four lanes take a group, eight values each.
constexpr int kRowThreads = 256;

template <class T, bool kPieces>
__global__ __launch_bounds__(kRowThreads) void k_quantize(const T* __restrict__ x, uint32_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, uint64_t eighths, uint32_t groups,
                                                          uint32_t width) {
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowThreads;
  for (uint64_t p = static_cast<uint64_t>(blockIdx.x) * kRowThreads + threadIdx.x; p < eighths; p += step) {
    const uint64_t row = p / (4 * groups);
    const uint32_t at = static_cast<uint32_t>(p - row * 4 * groups) * 8;
    float v[8];
    load_eight<T, kPieces>(x + row * width, at, width, v);
    const uint32_t byte = scale_byte(group_largest(largest_of(v)));
    codes[p] = to_codes(v, byte);
    if (p % 4 == 0) scales[p / 4] = static_cast<uint8_t>(byte);
  }
}

template <class T, bool kPieces>
__global__ __launch_bounds__(kRowThreads) void k_values(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                        T* __restrict__ x, uint64_t eighths, uint32_t groups, uint32_t width) {
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowThreads;
  for (uint64_t p = static_cast<uint64_t>(blockIdx.x) * kRowThreads + threadIdx.x; p < eighths; p += step) {
    const uint64_t row = p / (4 * groups);
    const uint32_t at = static_cast<uint32_t>(p - row * 4 * groups) * 8;
    const u32x4 v = to_bf16(codes[p], scale_of(scales[p / 4]));
    T* to = x + row * width + at;
    if constexpr (kPieces && sizeof(T) == 2) {
      if (at < width) *reinterpret_cast<u32x4*>(to) = v;
    } else if constexpr (kPieces) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (at + 4 * i < width)
          reinterpret_cast<u32x4*>(to)[i] = u32x4{v[2 * i] << 16, v[2 * i] & 0xffff0000u, v[2 * i + 1] << 16, v[2 * i + 1] & 0xffff0000u};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e < width) store_elem(to, e, e % 2 ? dl_bf16_hi(v[e / 2]) : dl_bf16_lo(v[e / 2]));
    }
  }
}

// ----------------------------------------------------------------- projection
struct ProjectArgs {
  const void* x;
  const uint8_t *codes, *scales;
  void* y;
  const uint64_t* position;
  uint32_t rows, in_w, groups, row_tiles;
  uint64_t out_w;
};

// The product operands of 32 consecutive inputs of a row: four steps of eight.
template <class T, bool kPieces>
struct Inputs;
template <bool kPieces>
struct Inputs<uint16_t, kPieces> {
  static constexpr int kParts = 1;
  u32x4 v[4];
  __device__ __forceinline__ void load(const uint16_t* row, uint32_t at, uint32_t width) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if constexpr (kPieces) {
        v[s] = at + 8 * s < width ? *reinterpret_cast<const u32x4*>(row + at + 8 * s) : u32x4{};
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t f = at + 8 * s + 2 * w;
          const uint32_t lo = f < width ? row[f] : 0u, hi = f + 1 < width ? row[f + 1] : 0u;
          v[s][w] = lo | (hi << 16);
        }
      }
    }
  }
  __device__ __forceinline__ void operands(int s, u32x4 (&b)[1]) const { b[0] = v[s]; }
};
template <bool kPieces>
struct Inputs<float, kPieces> {
  static constexpr int kParts = 3;
  float v[4][8];
  __device__ __forceinline__ void load(const float* row, uint32_t at, uint32_t width) {
#pragma unroll
    for (int s = 0; s < 4; ++s) load_eight<float, kPieces>(row, at + 8 * s, width, v[s]);
  }
  __device__ __forceinline__ void operands(int s, u32x4 (&b)[3]) const {
    const Parts p = split(v[s]);
#pragma unroll
    for (int i = 0; i < 3; ++i) b[i] = p.part[i];
  }
};

__device__ __forceinline__ f32x4 product(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Four consecutive outputs of a row.
template <class T>
__device__ __forceinline__ void store_four(T* to, const f32x4& v, uint64_t left, bool whole) {
  struct alignas(4 * sizeof(T)) Four {
    T v[4];
  } four;
#pragma unroll
  for (int e = 0; e < 4; ++e) store_elem(four.v, e, v[e]);
  if (whole && left >= 4) {
    *reinterpret_cast<Four*>(to) = four;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (static_cast<uint64_t>(e) < left) to[e] = four.v[e];
  }
}

// Up to 16 rows a workgroup, the wavefronts each taking every W-th 256 inputs of
// 16 kTiles outputs.  A lane's 16 bytes of codes are one group of one output and,
// converted, the first operand of four products; the same 32 inputs of a row are
// the second.
template <class T, bool kPieces, int kTiles, int W>
__global__ __launch_bounds__(W * 64) void k_project(const ProjectArgs a) {
  __shared__ f32x4 sums[W][kTiles][64];
  using In = Inputs<T, kPieces>;
  constexpr int kParts = In::kParts;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i16 = lane % 16, g = lane / 16;
  const uint32_t row = blockIdx.x % a.row_tiles * 16 + i16;
  const uint64_t o0 = static_cast<uint64_t>(blockIdx.x / a.row_tiles) * 16 * kTiles;
  const T* x = static_cast<const T*>(a.x) + static_cast<uint64_t>(min(row, a.rows - 1)) * a.in_w;
  const uint32_t width = row < a.rows ? a.in_w : 0;  // rows past the last are zeros
  const u32x4* codes[kTiles];
  const uint8_t* scales[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const uint64_t o = min(o0 + 16 * t + i16, a.out_w - 1);
    codes[t] = reinterpret_cast<const u32x4*>(a.codes) + o * a.groups;
    scales[t] = a.scales + o * a.groups;
  }
  f32x4 acc[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  u32x4 c[2][kTiles];
  uint32_t s[2][kTiles];
  In in[2];
  // Groups past the last repeat it, with codes of zero under a scale of one.
  auto load = [&](uint32_t chunk) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t group = chunk * 8 + 4 * h + g, at = min(group, a.groups - 1);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        c[h][t] = load_stream(codes[t] + at);
        s[h][t] = scales[t][at];
      }
      in[h].load(x, group * kGroup, width);
    }
  };
  const uint32_t chunks = (a.groups + 7) / 8;
  uint32_t chunk = wave;
  if (chunk < chunks) load(chunk);
  for (; chunk < chunks; chunk += W) {
    u32x4 now[2][kTiles];
    float by[2][kTiles];
    In x_now[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool real = chunk * 8 + 4 * h + g < a.groups;
      x_now[h] = in[h];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        now[h][t] = real ? c[h][t] : u32x4{};
        by[h][t] = scale_of(real ? s[h][t] : 127u);
      }
    }
    load(min(chunk + W, chunks - 1));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u32x4 b[kParts];
        x_now[h].operands(e, b);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const u32x4 w = to_bf16(now[h][t][e], by[h][t]);
#pragma unroll
          for (int p = 0; p < kParts; ++p) acc[t] = product(w, b[p], acc[t]);
        }
      }
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= kTiles) return;
  f32x4 sum = sums[0][wave][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) sum = sum + sums[w][wave][lane];
  const uint64_t o = o0 + 16 * wave + 4 * g;
  if (row >= a.rows || o >= a.out_w) return;
  T* y = static_cast<T*>(a.y) + (a.position ? *a.position * a.out_w : 0);
  const bool whole = a.out_w % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0;
  store_four(y + row * a.out_w + o, sum, a.out_w - o, whole);
}

template <class T, bool kPieces>
void launch_project(hipStream_t s, ProjectArgs& a) {
  auto run = [&](auto tiles) {
    constexpr int kTiles = decltype(tiles)::value, kWaves = 8;
    const uint64_t blocks = ceil_div(a.out_w, 16 * kTiles) * a.row_tiles;
    require(blocks <= (1u << 23), "too many workgroups", DL_LENGTH_ERROR);
    k_project<T, kPieces, kTiles, kWaves><<<static_cast<unsigned>(blocks), kWaves * 64, 0, s>>>(a);
  };
  a.row_tiles = static_cast<uint32_t>(ceil_div(a.rows, 16));
  run(std::integral_constant<int, 1>{});
}

// --------------------------------------------------------------------- append
struct AppendArgs {
  const void *query, *key, *value;
  void* query_out;
  dl_fp4_cache cache;
  const uint64_t *lengths, *positions;
  uint64_t *lengths_out, *positions_out;
  uint64_t rows, capacity;
  uint32_t q_heads, kv_heads, width;
  double theta;
};

constexpr int kAppendThreads = 256, kMostWidth = 256;

__device__ __forceinline__ void advance(const AppendArgs& a, uint64_t b) {
  const uint64_t n = a.lengths[b] < a.capacity ? a.lengths[b] : a.capacity, first = a.positions[b];
  a.lengths_out[b] = a.rows < a.capacity - n ? n + a.rows : a.capacity;
  a.positions_out[b] = first + a.rows;
}

// One workgroup per new row.  Cosines and sines of a row are computed once, in 64
// bits from the catalog's FP32 angle; rotated keys go from FP32 to 4 bits in one
// rounding.  32 lanes take a head, eight features each, and four of them a group.
template <class T>
__global__ __launch_bounds__(kAppendThreads) void k_append(const AppendArgs a, bool advance_here) {
  __shared__ float cosine[kMostWidth / 2], sine[kMostWidth / 2];
  const uint64_t b = blockIdx.y;
  const uint32_t half = a.width / 2, groups = (a.width + kGroup - 1) / kGroup;
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
    const T* query = static_cast<const T*>(a.query) + row * a.q_heads * a.width;
    T* query_out = static_cast<T*>(a.query_out) + row * a.q_heads * a.width;
    for (uint32_t p = threadIdx.x; p < a.q_heads * half; p += kAppendThreads) {
      const uint32_t at = p / half * a.width, f = p % half;
      const float u = load_elem(query, at + f), v = load_elem(query, at + half + f), c = cosine[f], s = sine[f];
      store_elem(query_out, at + f, u * c - v * s);
      store_elem(query_out, at + half + f, v * c + u * s);
    }
    if (fits) {
      const uint32_t f0 = threadIdx.x % 32 * 8;
      // Both halves of a wavefront run every pass: shuffles need their lanes.
      for (uint32_t h0 = 0; h0 < a.kv_heads; h0 += kAppendThreads / 32) {
        const uint32_t h = h0 + threadIdx.x / 32;
        const bool real = h < a.kv_heads;
        const uint64_t from = (row * a.kv_heads + (real ? h : 0)) * a.width;
        const uint64_t to = ((b * a.kv_heads + h) * a.capacity + slot) * groups;
        const T* key = static_cast<const T*>(a.key) + from;
        const T* value = static_cast<const T*>(a.value) + from;
        float k[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t f = f0 + e;
          k[e] = v[e] = 0.0f;
          if (f < a.width) {
            const float x = load_elem(key, f);
            k[e] = f < half ? x * cosine[f] - load_elem(key, f + half) * sine[f]
                            : x * cosine[f - half] + load_elem(key, f - half) * sine[f - half];
            v[e] = load_elem(value, f);
          }
        }
        const uint32_t k_byte = scale_byte(group_largest(largest_of(k))), v_byte = scale_byte(group_largest(largest_of(v)));
        if (real && f0 < groups * kGroup) {
          const uint64_t at = to * 4 + f0 / 8;
          static_cast<uint32_t*>(a.cache.key_codes)[at] = to_codes(k, k_byte);
          static_cast<uint32_t*>(a.cache.value_codes)[at] = to_codes(v, v_byte);
          if (f0 % kGroup == 0) {
            static_cast<uint8_t*>(a.cache.key_scales)[at / 4] = static_cast<uint8_t>(k_byte);
            static_cast<uint8_t*>(a.cache.value_scales)[at / 4] = static_cast<uint8_t>(v_byte);
          }
        }
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

// ------------------------------------------------------------------- the host
constexpr uint64_t kMostRows = uint64_t{1} << 40, kMostRowWidth = 1u << 24;

void check_rows(int dtype, uint64_t rows, uint64_t width) {
  require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
  require(rows && width, "empty rows");
  require(rows <= kMostRows && width <= kMostRowWidth, "rows too large", DL_LENGTH_ERROR);
}

bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <class F>
void with_type(int dtype, bool pieces, F&& f) {
  if (dtype == DL_BF16)
    pieces ? f(uint16_t{}, std::true_type{}) : f(uint16_t{}, std::false_type{});
  else
    pieces ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
}

bool whole_rows(int dtype, uint64_t width, const void* base) {
  return (width * (dtype == DL_BF16 ? 2 : 4)) % 16 == 0 && aligned(base, 16);
}

unsigned blocks_of(uint64_t threads) {
  return static_cast<unsigned>(std::min<uint64_t>(ceil_div(threads, kRowThreads), 1u << 16));
}

}  // namespace
}  // namespace dl::fp4

using dl::guard;
using dl::require;

extern "C" {

int dl_fp4_bytes(uint64_t rows, uint64_t width, uint64_t* codes, uint64_t* scales) {
  return guard([&] {
    require(codes && scales, "null output");
    dl::fp4::check_rows(DL_BF16, rows, width);
    *scales = rows * dl::fp4::groups_of(width);
    *codes = *scales * dl::fp4::kGroupBytes;
  });
}

int dl_fp4_quantize(dl_queue* queue, int dtype, const void* input, void* codes, void* scales, uint64_t rows, uint64_t width) {
  return guard([&] {
    using namespace dl::fp4;
    check_rows(dtype, rows, width);
    require(input && codes && scales, "null operand");
    require(aligned(codes, 16), "codes not 16-byte aligned");
    dl::enter(queue);
    const uint64_t groups = groups_of(width), eighths = rows * groups * 4;
    with_type(dtype, whole_rows(dtype, width, input), [&](auto type, auto pieces) {
      using T = decltype(type);
      k_quantize<T, decltype(pieces)::value><<<blocks_of(eighths), kRowThreads, 0, queue->stream>>>(
          static_cast<const T*>(input), static_cast<uint32_t*>(codes), static_cast<uint8_t*>(scales), eighths,
          static_cast<uint32_t>(groups), static_cast<uint32_t>(width));
    });
    dl::check_launch(queue, "fp4_quantize");
  });
}

int dl_fp4_values(dl_queue* queue, int dtype, const void* codes, const void* scales, void* output, uint64_t rows, uint64_t width) {
  return guard([&] {
    using namespace dl::fp4;
    check_rows(dtype, rows, width);
    require(codes && scales && output, "null operand");
    require(aligned(codes, 16), "codes not 16-byte aligned");
    dl::enter(queue);
    const uint64_t groups = groups_of(width), eighths = rows * groups * 4;
    with_type(dtype, whole_rows(dtype, width, output), [&](auto type, auto pieces) {
      using T = decltype(type);
      k_values<T, decltype(pieces)::value><<<blocks_of(eighths), kRowThreads, 0, queue->stream>>>(
          static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<T*>(output), eighths,
          static_cast<uint32_t>(groups), static_cast<uint32_t>(width));
    });
    dl::check_launch(queue, "fp4_values");
  });
}

int dl_projection_fp4(dl_queue* queue, int dtype, const void* input, const void* codes, const void* scales, void* output,
                      uint64_t rows, uint64_t input_width, uint64_t output_width, const uint64_t* output_position) {
  return guard([&] {
    using namespace dl::fp4;
    check_rows(dtype, rows, input_width);
    require(output_width > 0, "empty projection");
    require(rows <= (1u << 30) && output_width <= (1u << 30), "projection too large", DL_LENGTH_ERROR);
    require(input && codes && scales && output, "null operand");
    require(aligned(codes, 16), "codes not 16-byte aligned");
    dl::enter(queue);
    ProjectArgs a{input, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), output, output_position,
                  static_cast<uint32_t>(rows), static_cast<uint32_t>(input_width),
                  static_cast<uint32_t>(groups_of(input_width)), 0, output_width};
    with_type(dtype, whole_rows(dtype, input_width, input), [&](auto type, auto pieces) {
      launch_project<decltype(type), decltype(pieces)::value>(queue->stream, a);
    });
    dl::check_launch(queue, "projection_fp4");
  });
}

int dl_cache_append_fp4(dl_queue* queue, int dtype, const dl_batch_shape* shape, const void* query, const void* key,
                        const void* value, void* query_out, const dl_fp4_cache* cache, const uint64_t* lengths,
                        uint64_t* lengths_out, const uint64_t* positions, uint64_t* positions_out, double theta) {
  return guard([&] {
    using namespace dl::fp4;
    require(dtype == DL_BF16 || dtype == DL_F32, "unsupported storage type");
    dl::batch::check_shape(shape);
    require(cache != nullptr, "null cache");
    require(query && key && value && query_out && cache->key_codes && cache->key_scales && cache->value_codes &&
                cache->value_scales && lengths && lengths_out && positions && positions_out,
            "null operand");
    require(aligned(cache->key_codes, 16) && aligned(cache->value_codes, 16), "codes not 16-byte aligned");
    require(shape->width % 2 == 0, "rotated width must be even");
    require(shape->width <= kMostWidth, "head width above 256", DL_LENGTH_ERROR);
    require(shape->batch <= 65535, "too many sequences", DL_LENGTH_ERROR);
    require(theta > 0.0 && theta < 1e300, "theta must be positive and finite");
    dl::enter(queue);
    const AppendArgs a{query, key, value, query_out, *cache, lengths, positions, lengths_out, positions_out, shape->rows,
                       shape->capacity, static_cast<uint32_t>(shape->query_heads), static_cast<uint32_t>(shape->kv_heads),
                       static_cast<uint32_t>(shape->width), theta};
    const dim3 grid(static_cast<unsigned>(std::min<uint64_t>(shape->rows, 1u << 16)), static_cast<unsigned>(shape->batch));
    // A sequence's only workgroup has read its length before it writes the new
    // one, which may be the same word; of several any may still have to.
    const bool apart = lengths != lengths_out && positions != positions_out && lengths != positions_out && positions != lengths_out;
    const bool advance_here = grid.x == 1 || apart;
    if (dtype == DL_BF16)
      k_append<uint16_t><<<grid, kAppendThreads, 0, queue->stream>>>(a, advance_here);
    else
      k_append<float><<<grid, kAppendThreads, 0, queue->stream>>>(a, advance_here);
    if (!advance_here)
      k_advance<<<static_cast<unsigned>(dl::ceil_div(shape->batch, 64)), 64, 0, queue->stream>>>(a, shape->batch);
    dl::check_launch(queue, "cache_append_fp4");
  });
}

}  // extern "C"
