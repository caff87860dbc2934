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
// Four lanes take a group, eight values each.  Bound by both streams: 12,288 rows of
// 4096 BF16 values to codes and back 48 us, 5.2 TB/s read and written.
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
  uint32_t rows, in_w, groups;
  uint64_t out_w;
};

__device__ __forceinline__ f32x4 product(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Few rows (16 of BF16, 5 of FP32 as three exact parts in columns of their own):
// bound by the weights' stream.  Eight wavefronts cut the inputs, 256 at a time.
// Inputs are the products' second operands; 16 outputs' codes are first operands, a
// lane's 16 bytes being one group of one output, converted in place.
constexpr int kProjectWaves = 8;

template <class T>
constexpr int columns_of = sizeof(T) == 4 ? 5 : 16;  // rows of a workgroup

// The stream goes through LDS, so that every load of a wavefront is 1 KiB of one or two
// rows: a plain read of codes and scales in the operands' order, 16 rows at a time, comes
// at 4.1 TB/s, in their own at 6.7.  8 rows, 4096 to 151,936: 66 us, 5.0 TB/s, launch and
// end included; 1 row, 4096 to 1024: 3.8 us; 3 rows FP32, 12,288 to 4095: 16 us.  A stage is
// 2048 groups: kRow of 2048 / kRow outputs, M tiles of 16, loaded straight to LDS by
// all wavefronts, kStages - 1 ahead.  Of its sixteen units of 16 outputs and 256
// inputs a wavefront takes two.  A barrier a stage says that the stage has landed,
// that the one before it is read and that its sums are there.  Pieces of a row lie at
// piece ^ row, so that the 16 rows of an operand lie in distinct banks.
// A stage's room holds its codes, its scales and the wavefronts' sums.  Objects apart, so
// that the compiler sees no use of loads in flight in a read of another stage and waits
// for none.  That holds for BF16 rows in whole pieces.  Rows that come element by element
// pass through the last room first, after which it waits for all loads before the first
// read of every third stage.  Their kernels of three blocks spill too: 4 or 9 registers
// (FP32), 24 or 26 (BF16), each read back with a wait for all loads.
constexpr int kStageScales = 2048 * kGroupBytes, kStageSums = kStageScales + 2048;
template <int kStage, int kBytes>
__device__ __forceinline__ uint8_t* project_stage() {
  __shared__ __align__(1024) uint8_t room[kBytes];
  return room;
}

// A barrier alone: __syncthreads also waits for all loads to LDS, those of the stages
// ahead among them.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <class T, bool kPieces, bool kWhole, int kRow, int kBlocks>
__global__ __launch_bounds__(kProjectWaves * 64) __attribute__((amdgpu_waves_per_eu(2)))
void k_project_staged(const ProjectArgs a, uint32_t per_group) {
  constexpr int W = kProjectWaves, kRows = columns_of<T>, kOutputs = 2048 / kRow, M = kOutputs / 16;
  constexpr int kStages = 3, kLoads = kWhole ? 5 : 8;  // loads of a wavefront and stage
  constexpr int kChunks = kRow == 128 ? 2 : 1, kSums = kRow == 128 ? 1 : 2;
  constexpr int kRoom = kStageSums + kSums * W * 1024;
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr int kParts = kSplit ? 3 : 1;
  static_assert(!(kSplit && kPieces), "FP32 rows have no form in pieces");
  static_assert(kBlocks == 1 || kRow == 128, "longer rows are cut into blocks");
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i16 = lane % 16, g = lane / 16;
  const uint32_t first_row = blockIdx.y * kRows, rows = min(a.rows - first_row, static_cast<uint32_t>(kRows));
  const T* x = static_cast<const T*>(a.x) + static_cast<uint64_t>(first_row) * a.in_w;
  const uint32_t sets = static_cast<uint32_t>((a.out_w + kOutputs - 1) / kOutputs), first = blockIdx.x * per_group;
  const uint32_t count = min(per_group, sets - first), total = count * kBlocks;

  // The wavefront's chunk of 256 inputs and first tile; its second unit is chunk + 8
  // of the same tile, or the same chunk of a later tile.
  const uint32_t chunk = wave % (kRow / 8 < W ? kRow / 8 : W), tile0 = kRow / 8 < W ? wave / (kRow / 8) : 0;
  constexpr uint32_t kTileStep = kRow == 128 ? 0 : M / 2;

  u32x4 in[kBlocks][kChunks][2][4];
  if constexpr (!kPieces) {
    // Element by element through LDS of the wavefront's own, in the stage loaded last.
    constexpr int kHalf = 128;
    uint16_t* parts = reinterpret_cast<uint16_t*>(project_stage<kStages - 1, kRoom>()) + wave * (kParts * kRows * kHalf);
    static_assert(W * kParts * kRows * kHalf * 2 <= kRoom, "parts outgrow a stage");
    T v[2][2][kRows][2];  // a chunk's elements, loaded a chunk ahead; rows past the last repeat it
    auto load = [&](T (&to)[2][kRows][2], int batch) __attribute__((always_inline)) {
      const uint32_t base = batch / kChunks * kRow * kGroup + (chunk + 8 * (batch % kChunks)) * 256 + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            to[h][r][e] = x[static_cast<uint64_t>(min(static_cast<uint32_t>(r), rows - 1)) * a.in_w + min(base + h * kHalf + 64 * e, a.in_w - 1)];
    };
    const uint32_t column = min(i16, kParts * rows - 1), part = column / rows, in_part = column % rows;
    load(v[0], 0);
#pragma unroll
    for (int batch = 0; batch < kBlocks * kChunks; ++batch) {
      const int b = batch / kChunks, c = batch % kChunks;
      if (batch + 1 < kBlocks * kChunks) load(v[(batch + 1) % 2], batch + 1);
      const uint32_t base = b * kRow * kGroup + (chunk + 8 * c) * 256 + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const T in_row = base + h * kHalf + 64 * e < a.in_w ? v[batch % 2][h][r][e] : T{};
            uint16_t* to = parts + r * kHalf + 64 * e + lane;
            if constexpr (kSplit) {
              uint32_t three[3];
              split(in_row, three);
#pragma unroll
              for (int p = 0; p < 3; ++p) to[p * kRows * kHalf] = static_cast<uint16_t>(three[p] >> 16);
            } else {
              *to = in_row;
            }
          }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < 4; ++s)
          in[b][c][h][s] = *reinterpret_cast<const u32x4*>(parts + (part * kRows + in_part) * kHalf + g * kGroup + 8 * s);
        __builtin_amdgcn_wave_barrier();
      }
    }
  } else {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int s = 0; s < 4; ++s) in[b][c][h][s] = u32x4{};
    if (i16 < rows) {  // other columns are not stored
      const T* row = x + static_cast<uint64_t>(i16) * a.in_w;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t at = b * kRow * kGroup + (chunk + 8 * c) * 256 + (4 * h + g) * kGroup;
#pragma unroll
            for (int s = 0; s < 4; ++s)
              in[b][c][h][s] = at + 8 * s < a.in_w ? *reinterpret_cast<const u32x4*>(row + at + 8 * s) : u32x4{};
          }
    }
  }

  // Groups past the last repeat it, their inputs are zeros; outputs past the last
  // repeat it and are not stored.
  auto code_place = [&](int i, uint32_t block, uint32_t left) {
    const uint32_t at = (i * W + wave) * 64, in_row = at % kRow + lane;  // kRow 128, 64: one row for the wavefront
    const uint32_t row = at / kRow + (kRow < 64 ? in_row / kRow : 0), piece = in_row % kRow ^ row % 16;
    return (min(row, left) * a.groups + min(block * kRow + piece, a.groups - 1)) * kGroupBytes;
  };
  constexpr uint32_t kWords = kRow / 4, kWordSwizzle = kWords < 16 ? kWords : 16;  // words of four scales
  auto scale_place = [&](uint32_t block, uint32_t left) {
    const uint32_t slot = wave * 64 + lane, row = slot / kWords;
    return (min(row, left) * (a.groups / 4) + min(block * kWords + (slot % kWords ^ row % kWordSwizzle), a.groups / 4 - 1)) * 4;
  };
  // Scales of the wavefront's two units, where their rows are not whole words.
  struct Held {
    uint32_t scale[2][2];
  };
  Held ring[kStages];
  auto issue = [&](uint8_t* room, Held& held, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t block = kBlocks == 1 ? 0 : stage % kBlocks;
    const uint64_t o0 = static_cast<uint64_t>(first + stage / kBlocks) * kOutputs;
    const uint8_t* codes = a.codes + o0 * a.groups * kGroupBytes;
    const uint8_t* scales = a.scales + o0 * a.groups;
    const uint32_t left = a.out_w - o0 < kOutputs ? static_cast<uint32_t>(a.out_w - o0) - 1 : kOutputs - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_global_load_lds((const global_ptr*)(codes + code_place(i, block, left)),
                                       (lds_ptr*)(room + (i * W + wave) * 1024), 16, 0, 0);
    if constexpr (kWhole) {
      __builtin_amdgcn_global_load_lds((const global_ptr*)(scales + scale_place(block, left)),
                                       (lds_ptr*)(room + kStageScales + wave * 256), 4, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t row = min((tile0 + u * kTileStep) * 16 + i16, left);
          const uint32_t group = min(block * kRow + (chunk + (kRow == 128 ? 8 * u : 0)) * 8 + 4 * h + g, a.groups - 1);
          held.scale[u][h] = scales[row * a.groups + group];
        }
    }
  };
  f32x4 acc[kSums];
  auto step = [&](const uint8_t* room, const Held& held, auto constant) __attribute__((always_inline)) {
    constexpr int block = decltype(constant)::value;
    if (block == 0)
#pragma unroll
      for (f32x4& v : acc) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = kRow == 128 ? u : 0, to = kRow == 128 ? 0 : u;
      const uint32_t row = (tile0 + u * kTileStep) * 16 + i16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t piece = (chunk + 8 * c) * 8 + 4 * h + g, word = piece / 4;
        const u32x4 code = *reinterpret_cast<const u32x4*>(room + (row * kRow + (piece ^ i16)) * kGroupBytes);
        uint32_t scale = held.scale[u][h];
        if constexpr (kWhole)
          scale = *reinterpret_cast<const uint32_t*>(room + kStageScales + (row * kWords + (word ^ row % kWordSwizzle)) * 4) >> (8 * g) & 255u;
        const float by = scale_of(scale);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc[to] = product(to_bf16(code[s], by), in[block][c][h][s], acc[to]);
      }
    }
  };
  T* y = static_cast<T*>(a.y) + (a.position ? *a.position * a.out_w : 0);
  const bool whole = a.out_w % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0;
  // The sums of set n, whose last stage has this room, by one wavefront a tile.
  auto finish = [&](const uint8_t* room, uint32_t n) __attribute__((always_inline)) {
    const f32x4* sums = reinterpret_cast<const f32x4*>(room + kStageSums) + lane;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if (wave != static_cast<int>((n * M + m) % W)) continue;
      constexpr int kOf = kRow / 8 < W ? kRow / 8 : W;  // wavefronts that have a part of a tile
      const int from = kRow / 8 < W ? m % (W / kOf) * kOf : 0, which = kRow == 128 ? 0 : m / (M / 2);
      f32x4 sum = sums[(which * W + from) * 64];
#pragma unroll
      for (int w = 1; w < kOf; ++w) sum = sum + sums[(which * W + from + w) * 64];
      if constexpr (kSplit) {  // the low parts' columns into the high ones'
        f32x4 all = sum;
#pragma unroll
        for (int p = 1; p < 3; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e) all[e] = all[e] + __shfl(sum[e], lane + p * static_cast<int>(rows));
        sum = all;
      }
      const uint64_t o = (static_cast<uint64_t>(first + n) * M + m) * 16 + 4 * g;
      if (i16 < rows && o < a.out_w) store_four(y + static_cast<uint64_t>(first_row + i16) * a.out_w + o, sum, a.out_w - o, whole);
    }
  };
  auto work = [&](uint8_t* room, const Held& held, uint32_t block) __attribute__((always_inline)) {
    if (block == 0) step(room, held, std::integral_constant<int, 0>{});
    if constexpr (kBlocks > 1)
      if (block == 1) step(room, held, std::integral_constant<int, 1>{});
    if constexpr (kBlocks > 2)
      if (block == 2) step(room, held, std::integral_constant<int, 2>{});
    if (block == kBlocks - 1)
#pragma unroll
      for (int u = 0; u < kSums; ++u) reinterpret_cast<f32x4*>(room + kStageSums)[(u * W + wave) * 64 + lane] = acc[u];
  };
  auto finish_before = [&](const uint8_t* room, uint32_t stage) __attribute__((always_inline)) {
    if (stage && stage % kBlocks == 0) finish(room, stage / kBlocks - 1);
  };
  // A stage with two more behind it: it has landed when only the next one's loads are
  // under way; waits that the compiler adds make this one stricter.  No load here lies
  // under a condition: the compiler would wait for all of them before every read.
  auto turn = [&](auto slot, uint32_t stage) __attribute__((always_inline)) {
    constexpr int kSlot = decltype(slot)::value, kBefore = (kSlot + kStages - 1) % kStages;
    __builtin_amdgcn_s_waitcnt(lds_wait((kStages - 2) * kLoads));
    meet();
    finish_before(project_stage<kBefore, kRoom>(), stage);
    issue(project_stage<kBefore, kRoom>(), ring[kBefore], stage + kStages - 1);
    __builtin_amdgcn_sched_barrier(0);
    work(project_stage<kSlot, kRoom>(), ring[kSlot], kBlocks == kStages ? kSlot : stage % kBlocks);
  };
  auto room_of = [&](uint32_t stage) {
    const uint32_t slot = stage % kStages;
    return slot == 0 ? project_stage<0, kRoom>() : slot == 1 ? project_stage<1, kRoom>() : project_stage<2, kRoom>();
  };
  uint32_t stage = 0;
  if (total < kStages) {
    issue(project_stage<0, kRoom>(), ring[0], 0);
    if (total > 1) issue(project_stage<1, kRoom>(), ring[1], 1);
  } else {
    issue(project_stage<0, kRoom>(), ring[0], 0);
    issue(project_stage<1, kRoom>(), ring[1], 1);
    __builtin_amdgcn_s_waitcnt(vm_wait(2 * kLoads));  // the inputs
    for (;;) {
      turn(std::integral_constant<int, 0>{}, stage++);
      if (stage + kStages - 1 >= total) break;
      turn(std::integral_constant<int, 1>{}, stage++);
      if (stage + kStages - 1 >= total) break;
      turn(std::integral_constant<int, 2>{}, stage++);
      if (stage + kStages - 1 >= total) break;
    }
  }
  for (; stage < total; ++stage) {  // the last stages, which have no loads behind them
    __builtin_amdgcn_s_waitcnt(lds_wait(0));
    meet();
    finish_before(room_of(stage + kStages - 1), stage);
    const uint32_t slot = stage % kStages;
    Held held = {};
    if constexpr (!kWhole)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t of[3] = {ring[0].scale[u / 2][u % 2], ring[1].scale[u / 2][u % 2], ring[2].scale[u / 2][u % 2]};
        held.scale[u / 2][u % 2] = slot == 0 ? of[0] : slot == 1 ? of[1] : of[2];
      }
    work(room_of(stage), held, stage % kBlocks);
  }
  __syncthreads();
  finish(room_of(total - 1), count - 1);
}

// Few rows with more inputs than the staged kernel holds in registers: a workgroup per
// 16 outputs, inputs and codes read as they are needed, a group's all at once.  1 row of
// 12,320 inputs to 4096 outputs takes 16 us, where the staged kernel takes 9.4 for
// 12,288; of 17,408 24 us.  The codes of four groups at once: 19 and 29.
template <class T, bool kPieces>
__global__ __launch_bounds__(kProjectWaves * 64) void k_project_long(const ProjectArgs a) {
  constexpr int W = kProjectWaves, kRows = columns_of<T>, kParts = sizeof(T) == 4 ? 3 : 1;
  __shared__ f32x4 sums[W][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i16 = lane % 16, g = lane / 16;
  const uint32_t first_row = blockIdx.y * kRows, rows = min(a.rows - first_row, static_cast<uint32_t>(kRows));
  const uint32_t column = min(i16, kParts * rows - 1), part = column / rows;
  const T* x = static_cast<const T*>(a.x) + static_cast<uint64_t>(first_row + column % rows) * a.in_w;
  const uint64_t o0 = static_cast<uint64_t>(blockIdx.x) * 16, output = min(o0 + i16, a.out_w - 1) * a.groups;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t group0 = wave * 4; group0 < a.groups; group0 += 4 * W) {
    const uint32_t group = group0 + g, at = min(group, a.groups - 1);  // past the last: its inputs are zeros
    const u32x4 code = load_stream(reinterpret_cast<const u32x4*>(a.codes) + output + at);
    const float by = scale_of(a.scales[output + at]);
    float v[4][8];
#pragma unroll
    for (int s = 0; s < 4; ++s) load_eight<T, kPieces>(x, group * kGroup + 8 * s, a.in_w, v[s]);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const Parts p = split(v[s]);
      acc = product(to_bf16(code[s], by), kParts == 1 || part == 0 ? p.part[0] : part == 1 ? p.part[1] : p.part[2], acc);
    }
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
  f32x4 sum = acc;
#pragma unroll
  for (int w = 1; w < W; ++w) sum = sum + sums[w][lane];
  f32x4 all = sum;
  if constexpr (kParts == 3) {  // the low parts' columns into the high ones'
#pragma unroll
    for (int p = 1; p < 3; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) all[e] = all[e] + __shfl(sum[e], lane + p * static_cast<int>(rows));
  }
  const uint64_t o = o0 + 4 * g;
  if (i16 >= rows || o >= a.out_w) return;
  T* y = static_cast<T*>(a.y) + (a.position ? *a.position * a.out_w : 0);
  const bool whole = a.out_w % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0;
  store_four(y + static_cast<uint64_t>(first_row + i16) * a.out_w + o, all, a.out_w - o, whole);
}

// What loads to LDS take for inputs past the width.
__device__ const u32x4 zero_piece = {0, 0, 0, 0};

// Many rows: four wavefronts share 32 kRowTiles rows, 128 inputs at a time through
// LDS, loaded kStages - 1 steps ahead; each has 32 outputs of its own, whose codes come
// straight from memory as far ahead, so that every code is converted once for all the
// rows.  A 32 x 32 product does twice the operations of a 16 x 16 one for the operands it
// reads; the rates are the same.  512 rows, 4096 to 6144: 39 us, 660 TFLOP/s, 45 with
// weights that no call has read lately.  Products are busy 24% of that, vector instructions
// issue in 19%, and wavefronts wait to issue 47%: the 384 tiles run at once, one or two a
// compute unit, so one or two wavefronts a SIMD cover few of each other's waits and half of
// the units end early.
template <int kStage, int kBytes>
__device__ __forceinline__ uint8_t* many_stage() {
  __shared__ __align__(1024) uint8_t room[kBytes];
  return room;
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kManyOutputs = 128;

template <class T, bool kPieces, bool kWords, int kRowTiles>
__global__ __launch_bounds__(256) void k_project_many(const ProjectArgs a, uint32_t row_tiles) {
  constexpr int W = 4, kRows = 32 * kRowTiles, kParts = sizeof(T) == 4 ? 3 : 1, kRowBytes = 256;
  // A ring of steps where rows go to LDS directly, else two, rows through registers.
  constexpr int kStages = kPieces && sizeof(T) == 2 ? 4 : 2;
  constexpr int kPart = kRows * kRowBytes, kPer = kRows * 16 / 256;  // 16-byte pieces of a thread
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t i32 = lane % 32, half = lane / 32;
  // XCD x takes the output tiles x, x + 8, ..., and all row tiles of one, which read
  // the same codes.
  const uint32_t in_xcd = blockIdx.x / 8, out_tile = in_xcd / row_tiles * 8 + blockIdx.x % 8, row0 = in_xcd % row_tiles * kRows;
  const uint64_t o0 = static_cast<uint64_t>(out_tile) * kManyOutputs + 32 * wave;
  if (static_cast<uint64_t>(out_tile) * kManyOutputs >= a.out_w) return;
  const T* x = static_cast<const T*>(a.x);
  const uint32_t steps = (a.groups + 3) / 4;

  const uint64_t output = min(o0 + i32, a.out_w - 1) * a.groups;
  const u32x4* codes = reinterpret_cast<const u32x4*>(a.codes) + output;
  const uint8_t* scales = a.scales + output;
  // Two of a step's four groups: 2 h + half.
  struct Codes {
    u32x4 code[2];
    uint32_t scale[kWords ? 1 : 2];
  };
  Codes ring[kStages];
  auto load_codes = [&](Codes& to, uint32_t step) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // groups past the last repeat it: their inputs are zeros
      const uint32_t group = min(step * 4 + 2 * h + half, a.groups - 1);
      to.code[h] = codes[group];
      if constexpr (!kWords) to.scale[h] = scales[group];
    }
    if constexpr (kWords) to.scale[0] = *reinterpret_cast<const uint32_t*>(scales + min(step * 4, a.groups - 4));
  };
  auto factor = [&](const Codes& from, int h) __attribute__((always_inline)) {
    if constexpr (kWords) return scale_of(from.scale[0] >> (16 * h + 8 * half) & 255u);
    else return scale_of(from.scale[h]);
  };
  // Piece p (eight inputs) of row r lies at p ^ r.
  constexpr bool kDirect = kPieces && sizeof(T) == 2;
  float held[kDirect ? 1 : kPer][8];
  auto load_rows = [&](uint8_t* room, uint32_t step) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t slot = i * 256 + threadIdx.x, r = slot / 16, piece = slot % 16 ^ r % 16, at = step * 128 + piece * 8;
      const T* row = x + static_cast<uint64_t>(min(row0 + r, a.rows - 1)) * a.in_w;
      if constexpr (kDirect) {
        const void* from = at < a.in_w ? static_cast<const void*>(row + at) : &zero_piece;
        __builtin_amdgcn_global_load_lds((const global_ptr*)from, (lds_ptr*)(room + (i * W + wave) * 1024), 16, 0, 0);
      } else {
        load_eight<T, kPieces>(row, at, a.in_w, held[i]);
      }
    }
  };
  auto store_rows = [&](uint8_t* room) __attribute__((always_inline)) {
    if constexpr (!kDirect) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        uint8_t* to = room + (i * 256 + threadIdx.x) * 16;
        if constexpr (kParts == 3) {
          const Parts p = split(held[i]);
#pragma unroll
          for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x4*>(to + k * kPart) = p.part[k];
        } else {
          u32x4 v;
#pragma unroll
          for (int w = 0; w < 4; ++w) v[w] = __float_as_uint(held[i][2 * w]) >> 16 | (__float_as_uint(held[i][2 * w + 1]) & 0xffff0000u);
          *reinterpret_cast<u32x4*>(to) = v;
        }
      }
    }
  };
  f32x16 acc[kRowTiles];
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r) acc[r] = f32x16{};
  // Rows of a product step (16 inputs) are read two steps before they are multiplied,
  // and codes converted one step before.
  constexpr int kProducts = kRowTiles * kParts;
  u32x4 v[3][kProducts], weight[2];
  auto read = [&](const uint8_t* room, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
      for (int p = 0; p < kParts; ++p)
        v[s % 3][r * kParts + p] = *reinterpret_cast<const u32x4*>(
            room + p * kPart + (32 * r + i32) * kRowBytes + ((8 * (s / 4) + 4 * half + s % 4) ^ i32 % 16) * 16);
  };
  auto convert = [&](const Codes& from, int s) __attribute__((always_inline)) {
    weight[s % 2] = to_bf16(from.code[s / 4][s % 4], factor(from, s / 4));
  };
  auto compute = [&](const uint8_t* room, const Codes& from) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (s < 6) read(room, s + 2);
      if (s < 7) convert(from, s + 1);
#pragma unroll
      for (int i = 0; i < kProducts; ++i)
        acc[i / kParts] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, weight[s % 2]),
                                                                  __builtin_bit_cast(bf16x8, v[s % 3][i]), acc[i / kParts], 0, 0, 0);
      if (s < 7) {
        if (s < 6) __builtin_amdgcn_sched_group_barrier(0x100, kProducts, 0);
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, (6 + kProducts - 1) / kProducts, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr int kBytes = kParts * kPart, kAhead = kStages - 1;
  // Steps past the last have zeros for rows.  No load lies under a condition, and the
  // loop is left at its end alone: the compiler would wait for all loads in flight.
  auto turn = [&](auto slot, uint32_t step) __attribute__((always_inline)) {
    constexpr int kSlot = decltype(slot)::value, kNext = (kSlot + kAhead) % kStages;
    __builtin_amdgcn_s_waitcnt(lds_wait(kDirect ? (kAhead - 1) * (kPer + (kWords ? 3 : 4)) : 63));  // this step's rows
    meet();
    read(many_stage<kSlot, kBytes>(), 0);
    read(many_stage<kSlot, kBytes>(), 1);
    __builtin_amdgcn_sched_barrier(0);
    load_rows(many_stage<kNext, kBytes>(), step + kAhead);
    load_codes(ring[kNext], step + kAhead);
    convert(ring[kSlot], 0);
    __builtin_amdgcn_sched_barrier(0);
    compute(many_stage<kSlot, kBytes>(), ring[kSlot]);
    store_rows(many_stage<kNext, kBytes>());
  };
  auto first = [&](auto slot) __attribute__((always_inline)) {
    constexpr int kSlot = decltype(slot)::value;
    load_rows(many_stage<kSlot, kBytes>(), kSlot);
    load_codes(ring[kSlot], kSlot);
    store_rows(many_stage<kSlot, kBytes>());
    __builtin_amdgcn_sched_barrier(0);
  };
  first(std::integral_constant<int, 0>{});
  if constexpr (kAhead > 1) first(std::integral_constant<int, 1>{});
  if constexpr (kAhead > 2) first(std::integral_constant<int, 2>{});
  for (uint32_t step = 0; step < steps; step += kStages) {
    turn(std::integral_constant<int, 0>{}, step);
    turn(std::integral_constant<int, 1>{}, step + 1);
    if constexpr (kStages > 2) turn(std::integral_constant<int, 2>{}, step + 2);
    if constexpr (kStages > 3) turn(std::integral_constant<int, 3>{}, step + 3);
  }
  T* y = static_cast<T*>(a.y) + (a.position ? *a.position * a.out_w : 0);
  const bool whole = a.out_w % 4 == 0 && reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0;
#pragma unroll
  for (int r = 0; r < kRowTiles; ++r) {
    const uint32_t row = row0 + 32 * r + i32;
    if (row >= a.rows) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint64_t o = o0 + 8 * q + 4 * half;
      const f32x4 four = {acc[r][4 * q], acc[r][4 * q + 1], acc[r][4 * q + 2], acc[r][4 * q + 3]};
      if (o < a.out_w) store_four(y + static_cast<uint64_t>(row) * a.out_w + o, four, a.out_w - o, whole);
    }
  }
}

template <class T, bool kPieces>
void launch_project(hipStream_t s, const ProjectArgs& a) {
  const bool words = a.groups % 4 == 0 && reinterpret_cast<uintptr_t>(a.scales) % 4 == 0;
  // Few rows read the weights once per 16 (FP32 5); many convert them once per 32 or 64
  // and need tiles for most compute units.  4096 x 4096, rows 24, 48 and 128: few 11, 18
  // and 44 us, many by 32 rows 17, 17 and 18, by 64 19, 20 and 21; 4096 x 24576, 48 and
  // 128 rows: few 41 and 97, by 32 42 and 62, by 64 29 and 51.  FP32, 4096 x 4096, rows 20
  // and 24: few 26 and 32, many 37 and 37.
  if (a.rows > (sizeof(T) == 4 ? 20 : 32)) {
    auto many = [&](auto whole_words, auto tiles) {
      constexpr int kRowTiles = decltype(tiles)::value;
      const uint64_t row_tiles = ceil_div(a.rows, 32 * kRowTiles), out_tiles = ceil_div(ceil_div(a.out_w, kManyOutputs), 8) * 8;
      require(row_tiles * out_tiles <= (1u << 23), "too many workgroups", DL_LENGTH_ERROR);
      k_project_many<T, kPieces, decltype(whole_words)::value, kRowTiles>
          <<<static_cast<unsigned>(row_tiles * out_tiles), 256, 0, s>>>(a, static_cast<uint32_t>(row_tiles));
    };
    auto by_rows = [&](auto whole_words) {
      if constexpr (sizeof(T) == 2) {
        if (ceil_div(a.rows, 64) * ceil_div(a.out_w, kManyOutputs) > 128) return many(whole_words, std::integral_constant<int, 2>{});
      }
      many(whole_words, std::integral_constant<int, 1>{});
    };
    words ? by_rows(std::true_type{}) : by_rows(std::false_type{});
    return;
  }
  const uint64_t row_tiles = ceil_div(a.rows, columns_of<T>);
#define I(n) std::integral_constant<int, n>{}
  if (a.groups > 384) {
    require(a.out_w <= (1u << 26), "too many workgroups", DL_LENGTH_ERROR);
    const dim3 grid(static_cast<unsigned>(ceil_div(a.out_w, 16)), static_cast<unsigned>(row_tiles));
    k_project_long<T, kPieces><<<grid, kProjectWaves * 64, 0, s>>>(a);
    return;
  }
  auto run = [&](auto row, auto blocks) {
    constexpr int kRow = decltype(row)::value, kBlocks = decltype(blocks)::value;
    const uint64_t sets = ceil_div(a.out_w, 2048 / kRow), per_group = ceil_div(sets, 256);
    const dim3 grid(static_cast<unsigned>(ceil_div(sets, per_group)), static_cast<unsigned>(row_tiles));
    // FP32 rows go element by element, whole pieces or not.
    constexpr bool kDirect = kPieces && sizeof(T) == 2;
    if (words)
      k_project_staged<T, kDirect, true, kRow, kBlocks><<<grid, kProjectWaves * 64, 0, s>>>(a, static_cast<uint32_t>(per_group));
    else
      k_project_staged<T, kDirect, false, kRow, kBlocks><<<grid, kProjectWaves * 64, 0, s>>>(a, static_cast<uint32_t>(per_group));
  };
  if (a.groups <= 32)
    run(I(32), I(1));
  else if (a.groups <= 64)
    run(I(64), I(1));
  else if (a.groups <= 128)
    run(I(128), I(1));
  else if (a.groups <= 256)
    run(I(128), I(2));
  else
    run(I(128), I(3));
#undef I
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

// Four features of a row at whole alignment.
template <class T>
__device__ __forceinline__ f32x4 load_four(const T* from) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const f32x4*>(from);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    return f32x4{dl_bf16_lo(v.x), dl_bf16_hi(v.x), dl_bf16_lo(v.y), dl_bf16_hi(v.y)};
  }
}

// One workgroup per new row.  Cosines and sines of a row are computed once, in 64
// bits from the catalog's FP32 angle; rotated keys go from FP32 to 4 bits in one
// rounding.  32 lanes take a head, eight features each, and four of them a group.
// What bounds it for few rows is one wait for memory and the 64-bit angles, so the
// rows are asked for before the angles are computed: 8 rows of 32 and 8 heads of 128
// features 5.6 us, 1024 FP32 rows 11.5 (wavefronts wait for memory or a barrier half the
// time), BF16 9.0.  kFours: halves are of whole fours, all rows at their alignment; feature
// by feature these take 7.3, 19 and 15.
template <class T, bool kFours>
__global__ __launch_bounds__(kAppendThreads) void k_append(const AppendArgs a, bool advance_here) {
  __shared__ __align__(16) float cosine[kMostWidth / 2], sine[kMostWidth / 2];
  constexpr uint32_t kEach = kFours ? 4 : 1, kAhead = kFours ? 2 : 1;  // features of a query piece, pieces asked for early
  using Each = std::conditional_t<kFours, f32x4, float>;
  const uint64_t b = blockIdx.y;
  const uint32_t half = a.width / 2, groups = (a.width + kGroup - 1) / kGroup;
  const uint32_t in_half = half / kEach, pieces = a.q_heads * in_half, f0 = threadIdx.x % 32 * 8;
  auto load = [](const T* from) __attribute__((always_inline)) {
    if constexpr (kFours)
      return load_four(from);
    else
      return load_elem(from, 0);
  };
  const uint64_t n = a.lengths[b], first = a.positions[b];
  for (uint64_t i = blockIdx.x; i < a.rows; i += gridDim.x) {
    const uint64_t position = first + i, slot = n + i, row = b * a.rows + i;
    const bool fits = n < a.capacity && i < a.capacity - n;
    const T* query = static_cast<const T*>(a.query) + row * a.q_heads * a.width;
    T* query_out = static_cast<T*>(a.query_out) + row * a.q_heads * a.width;
    Each lower[kAhead], upper[kAhead];
#pragma unroll
    for (uint32_t x = 0; x < kAhead; ++x) {
      const uint32_t p = min(threadIdx.x + x * kAppendThreads, pieces - 1), at = p / in_half * a.width + p % in_half * kEach;
      lower[x] = load(query + at);
      upper[x] = load(query + at + half);
    }
    // Of a head the lane's features, those half a row away, and its values.
    float k[8], other[8], v[8];
    auto ask = [&](uint32_t h) __attribute__((always_inline)) {
      const uint64_t from = (row * a.kv_heads + min(h, a.kv_heads - 1)) * a.width;
      const T* key = static_cast<const T*>(a.key) + from;
      const T* value = static_cast<const T*>(a.value) + from;
#pragma unroll
      for (uint32_t e = 0; e < 8; e += kEach) {
        const uint32_t f = f0 + e < a.width ? f0 + e : 0, o = f < half ? f + half : f - half;
        const Each at = load(key + f), away = load(key + o), val = load(value + f);
        if constexpr (kFours) {
#pragma unroll
          for (int c = 0; c < 4; ++c) k[e + c] = at[c], other[e + c] = away[c], v[e + c] = val[c];
        } else {
          k[e] = at, other[e] = away, v[e] = val;
        }
      }
    };
    ask(threadIdx.x / 32);
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
    auto turn = [&](uint32_t p, const Each& u, const Each& v) __attribute__((always_inline)) {
      const uint32_t f = p % in_half * kEach, at = p / in_half * a.width + f;
      if constexpr (kFours) {
        const f32x4 c = *reinterpret_cast<const f32x4*>(cosine + f), s = *reinterpret_cast<const f32x4*>(sine + f);
        store_four(query_out + at, u * c - v * s, 4, true);
        store_four(query_out + at + half, v * c + u * s, 4, true);
      } else {
        store_elem(query_out, at, u * cosine[f] - v * sine[f]);
        store_elem(query_out, at + half, v * cosine[f] + u * sine[f]);
      }
    };
#pragma unroll
    for (uint32_t x = 0; x < kAhead; ++x)
      if (threadIdx.x + x * kAppendThreads < pieces) turn(threadIdx.x + x * kAppendThreads, lower[x], upper[x]);
    for (uint32_t p = threadIdx.x + kAhead * kAppendThreads; p < pieces; p += kAppendThreads) {
      const uint32_t at = p / in_half * a.width + p % in_half * kEach;
      turn(p, load(query + at), load(query + at + half));
    }
    if (fits) {
      // Both halves of a wavefront run every pass: shuffles need their lanes.
      for (uint32_t h0 = 0; h0 < a.kv_heads; h0 += kAppendThreads / 32) {
        const uint32_t h = h0 + threadIdx.x / 32;
        if (h0) ask(h);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t f = f0 + e;
          if (f >= a.width)
            k[e] = v[e] = 0.0f;
          else
            k[e] = f < half ? k[e] * cosine[f] - other[e] * sine[f] : k[e] * cosine[f - half] + other[e] * sine[f - half];
        }
        const uint32_t k_byte = scale_byte(group_largest(largest_of(k))), v_byte = scale_byte(group_largest(largest_of(v)));
        if (h < a.kv_heads && f0 < groups * kGroup) {
          const uint64_t at = ((b * a.kv_heads + h) * a.capacity + slot) * groups * 4 + f0 / 8;
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
                  static_cast<uint32_t>(groups_of(input_width)), output_width};
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
    const uint64_t four = dtype == DL_BF16 ? 8 : 16;
    const bool fours = shape->width % 8 == 0 && aligned(query, four) && aligned(key, four) && aligned(value, four) && aligned(query_out, four);
    with_type(dtype, fours, [&](auto type, auto whole) {
      k_append<decltype(type), decltype(whole)::value><<<grid, kAppendThreads, 0, queue->stream>>>(a, advance_here);
    });
    if (!advance_here)
      k_advance<<<static_cast<unsigned>(dl::ceil_div(shape->batch, 64)), 64, 0, queue->stream>>>(a, shape->batch);
    dl::check_launch(queue, "cache_append_fp4");
  });
}

}  // extern "C"
