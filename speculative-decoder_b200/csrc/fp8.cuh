// 8-bit operands with scales: an e4m3 value q stands for q * s, where s is the fp32 scale of its
// group. Activations [M, K] have one scale per row and 128 columns, weights [N, K] one per
// 128 x 128 block; the last groups of a row or column may be short.
//   s = max(max |y| over the group, 2^-100) / 448,   q = e4m3(y / s)
// 448 is e4m3's largest value. The floor keeps 1 / s finite for groups of zeros; a NaN or an
// infinity in a group makes its scale NaN or infinite and so stays visible in every product.
#pragma once
#include "common.cuh"

namespace specb200 {

constexpr int kFp8Group = 128;
constexpr float kE4m3Max = 448.f;
constexpr float kFp8MinAmax = 7.888609052210118e-31f;  // 2^-100

// The larger magnitude, where a NaN wins: fmaxf would drop it, and a group's NaN has to reach its scale.
SPECB200_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
SPECB200_DEVINL float max_mag(float m, float x) { return max_nan(m, fabsf(x)); }
SPECB200_DEVINL float floor_amax(float amax) { return amax < kFp8MinAmax ? kFp8MinAmax : amax; }

inline bool fp8_aligned(const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace specb200
