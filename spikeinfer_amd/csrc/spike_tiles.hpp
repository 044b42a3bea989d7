// Pieces of the attention kernels that take packed spikes through the matrix cores in
// 32 x 32 tiles (prefill_attn.hip, tree_attn.hip): operand types, spikes as fp4, the bit
// transpose of a wave's words, the table of softmax weights.
#pragma once

#include <cmath>
#include <cstring>

#include "common.hpp"

namespace spk {
namespace tiles {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

#define SPK_LDS __attribute__((address_space(3)))

constexpr int kTab = 129;  // weights of scores 0..head_dim (<= 128)

// The value of x in the lane whose number differs by J (1, 2, 4 or 8), by data-parallel
// moves: no LDS latency.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  const int v = static_cast<int>(x);
  if constexpr (J == 1) return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
  else if constexpr (J == 2) return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
  else if constexpr (J == 8)  // rotation by 8 within a row of 16
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false));
  else {  // four lanes up for banks 0 and 2 of a row, down for 1 and 3
    const int up = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xF, 0x5, false);
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(up, v, 0x114, 0xF, 0xA, false));
  }
}

// One step of the 32 x 32 bit transpose within each 32-lane half (lane = row,
// bit = column): lanes without bit J trade their J-columns for the partner's
// others.
template <int J>
__device__ __forceinline__ uint32_t transpose_step(uint32_t x, int lane) {
  if constexpr (J == 16) {  // rows of 16 lanes: (even, even) and (odd, odd), a half of each
    const auto sw = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return __builtin_amdgcn_perm(sw[1], sw[0], lane & 16 ? 0x07060302u : 0x05040100u);
  } else {
    constexpr uint32_t m = J == 8 ? 0x00ff00ffu : J == 4 ? 0x0f0f0f0fu : J == 2 ? 0x33333333u : 0x55555555u;
    const uint32_t y = lane_xor<J>(x);
    const bool up = lane & J;
    const uint32_t keep = up ? ~m : m;
    const uint32_t r = __builtin_amdgcn_alignbit(y, y, up ? J : 32 - J);  // rotate right
    return (x & keep) | (r & ~keep);
  }
}

__device__ __forceinline__ uint32_t transpose32(uint32_t x, int lane) {
  x = transpose_step<16>(x, lane);
  x = transpose_step<8>(x, lane);
  x = transpose_step<4>(x, lane);
  x = transpose_step<2>(x, lane);
  return transpose_step<1>(x, lane);
}

// 32 bits as 32 fp4 values of 0.5: nibble n of word i is bit 4n + i.
__device__ __forceinline__ v8i fp4_bits(uint32_t w) {
  v8i r = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = static_cast<int>((w >> i) & 0x11111111u);
  return r;
}

// Rows are divided by the n heads of a kv head with one multiplication, r * inverse >> 32.  Its
// product is off by r * (inverse * n - 2^32) / n: right while that stays below 2^32 / n.
inline uint32_t inverse_of(int n) { return static_cast<uint32_t>(((int64_t(1) << 32) + n - 1) / n); }  // (not of 1)
inline bool divides_to(int64_t most, int n) {
  return n == 1 || most * (static_cast<int64_t>(inverse_of(n)) * n - (int64_t(1) << 32)) < int64_t(1) << 32;
}

// (hi, lo) f16 pairs of exp(s * scale) * 2^15 / exp(D * scale), s = 0..D.
inline void build_table(float scale, int D, uint32_t *tab) {
  static thread_local float last_scale = -1.f;
  static thread_local int last_d = 0;
  static thread_local uint32_t last[kTab];
  if (scale != last_scale || D != last_d) {
    for (int s = 0; s <= D; ++s) {
      const double w = std::ldexp(std::exp((s - D) * static_cast<double>(scale)), 15);
      const _Float16 hi = static_cast<_Float16>(w);
      const _Float16 lo = static_cast<_Float16>(w - static_cast<double>(hi));
      uint16_t a, b;
      std::memcpy(&a, &hi, 2);
      std::memcpy(&b, &lo, 2);
      last[s] = a | (static_cast<uint32_t>(b) << 16);
    }
    last_scale = scale;
    last_d = D;
  }
  std::memcpy(tab, last, sizeof(uint32_t) * (D + 1));
}

}  // namespace tiles
}  // namespace spk
