// Producers of 8-bit operands (fp8.cuh): plain quantization of rows or 128 x 128 blocks, RMSNorm
// with the residual update in front, and SiLU(gate) * up. Everything between the inputs and the
// e4m3 rounding is fp32; the only other rounding is the residual stream's own element type.
//
// All are bound by memory: each input is read once, 16 bytes per lane, and each output written
// once. A group of 128 columns is held by 16 lanes with 8 elements each, so its maximum is four
// shuffles and its scale is written by the group's first lane.
#include <algorithm>

#include "fp8.cuh"
#include "kernels.cuh"

namespace specb200 {
namespace {

// Eight consecutive elements of a row, `valid` of them inside it (the rest read as zero). vec:
// the row starts on a 16-byte boundary.
template <typename T>
SPECB200_DEVINL void load8(const T* p, int valid, bool vec, float (&f)[8]) {
  if (vec && valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    } else {
      const float4 a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < valid ? to_f32<T>(p[i]) : 0.f;
}

template <typename T>
SPECB200_DEVINL void store8(T* p, int valid, bool vec, const float (&f)[8]) {
  if (vec && valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) p[i] = from_f32<T>(f[i]);
}

SPECB200_DEVINL void store_q8(uint8_t* p, int valid, bool vec, const float (&f)[8]) {
  const uint2 v = pack_e4m3(f);
  if (vec && valid >= 8) {
    *reinterpret_cast<uint2*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) p[i] = static_cast<uint8_t>((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
}

SPECB200_DEVINL uint32_t max_mag8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, mag_bits(f[i]));
  return m;
}
// Maximum over the 16 lanes that hold a group.
SPECB200_DEVINL uint32_t half_warp_max(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

struct RowArgs {
  const void* x;       // quantize: [M, K]; SiLU: gate | up
  int64_t ldx;         // elements
  uint8_t* q;
  int64_t ldq;
  float* scales;       // [M, groups] (or [row blocks, groups])
  int M, K, groups;
  int packed;          // SiLU: 1 = 64 gate columns, then their 64 up columns
  int vec_in, vec_out; // rows of x / q start on 16- / 8-byte boundaries
};

constexpr int kRowThreads = 256;

// One group of one row per 16 lanes. kSilu: y = silu(gate) * up, else y = x.
template <typename T, bool kSilu>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(RowArgs a) {
  pdl_launch_dependents();
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> 4;
  const int64_t units = static_cast<int64_t>(a.M) * a.groups;
  pdl_wait();
  const bool live = unit < units;
  const int64_t row = live ? unit / a.groups : 0;
  const int g = live ? static_cast<int>(unit - row * a.groups) : 0;
  const int lane = threadIdx.x & 15;
  const int col = g * kFp8Group + lane * 8;
  const int valid = live ? min(8, max(0, a.K - col)) : 0;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  float y[8];
  if constexpr (kSilu) {
    // packed: feature j is gate column 128 (j / 64) + j % 64, its up column 64 further on
    const int gate_col = a.packed ? ((col >> 6) << 7) + (col & 63) : col;
    float u[8];
    load8<T>(xr + gate_col, valid, a.vec_in, y);
    load8<T>(xr + gate_col + (a.packed ? 64 : a.K), valid, a.vec_in, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = y[i] / (1.f + expf(-y[i])) * u[i];
  } else {
    load8<T>(xr + col, valid, a.vec_in, y);
  }
  const float amax = floor_amax(__uint_as_float(half_warp_max(max_mag8(y))));
  const float inv = kE4m3Max / amax;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] *= inv;
  if (valid > 0) store_q8(a.q + row * a.ldq + col, valid, a.vec_out, y);
  if (live && lane == 0) a.scales[unit] = amax / kE4m3Max;
}

// One 128 x 128 block per CTA, held in registers between the maximum and the rounding: 16 lanes
// per row, 16 rows at a time.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) quantize_blocks_kernel(RowArgs a) {
  constexpr int kPass = kFp8Group / (kRowThreads / 16);
  __shared__ uint32_t sh[kRowThreads / 32];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int g = blockIdx.x % a.groups, rb = blockIdx.x / a.groups;
  const int col = g * kFp8Group + lane * 8;
  const int valid = min(8, max(0, a.K - col));
  pdl_wait();
  float y[kPass][8];
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    const int row = rb * kFp8Group + p * (kRowThreads / 16) + r0;
    const int64_t at = static_cast<int64_t>(min(row, a.M - 1)) * a.ldx + col;
    load8<T>(static_cast<const T*>(a.x) + at, row < a.M ? valid : 0, a.vec_in, y[p]);
  }
#pragma unroll
  for (int p = 0; p < kPass; ++p) m = max(m, max_mag8(y[p]));
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) m = max(m, sh[i]);
  const float amax = floor_amax(__uint_as_float(m));
  const float inv = kE4m3Max / amax;
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    const int row = rb * kFp8Group + p * (kRowThreads / 16) + r0;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[p][i] *= inv;
    if (row < a.M && valid > 0) store_q8(a.q + row * a.ldq + col, valid, a.vec_out, y[p]);
  }
  if (threadIdx.x == 0) a.scales[blockIdx.x] = amax / kE4m3Max;
}

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* delta;   // NULL: no residual update
  int64_t ldd;
  const void* weight;
  void* h;             // NULL without delta; may be x or delta
  int64_t ldh;
  uint8_t* q;
  int64_t ldq;
  float* scales;
  int H, groups;
  float eps;
  int vec_x, vec_d, vec_w, vec_h, vec_q;
};

constexpr int kNormMaxThreads = 1024;
constexpr int kNormMaxChunks = 4;  // 8-element chunks per thread
constexpr int kNormMaxWidth = kNormMaxThreads * kNormMaxChunks * 8;

// h = T(x + delta); y = w h / sqrt(mean(h^2) + eps); (q, scales) = quantize(y). One CTA per row,
// the row in registers.
//
// The quantized values need no norm: with m the group's largest |w h| and r the row's 1 / rms,
// y / s = (w h r) / (m r / 448) = w h (448 / m), so q carries two roundings and only the scale
// waits for the row's sum. Where the floor is in play or a value is not finite, q is formed from
// y itself.
template <typename T, int kChunks>
__global__ void __launch_bounds__(kNormMaxThreads) rmsnorm_fp8_kernel(NormArgs a) {
  __shared__ float sh[kNormMaxThreads / 32];
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, nthr = blockDim.x;
  pdl_wait();
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  float f[kChunks][8];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = (tid + c * nthr) * 8;
    load8<T>(xr + col, a.H - col, a.vec_x, f[c]);
  }
  if (a.delta) {
    const T* dr = static_cast<const T*>(a.delta) + row * a.ldd;
    T* hr = static_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (tid + c * nthr) * 8;
      float d[8];
      load8<T>(dr + col, a.H - col, a.vec_d, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[c][i] = round_to<T>(f[c][i] + d[i]);
      store8<T>(hr + col, a.H - col, a.vec_h, f[c]);
    }
  }
  float ss = 0.f;
  uint32_t m[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = (tid + c * nthr) * 8;
    float w[8];
    load8<T>(static_cast<const T*>(a.weight) + col, a.H - col, a.vec_w, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ss = fmaf(f[c][i], f[c][i], ss);
      f[c][i] *= w[i];
    }
    m[c] = half_warp_max(max_mag8(f[c]));
  }
  ss = warp_sum(ss);
  if ((tid & 31) == 0) sh[tid >> 5] = ss;
  __syncthreads();
  float total = 0.f;
  for (int i = 0; i < nthr / 32; ++i) total += sh[i];
  const float r = 1.f / sqrtf(total / static_cast<float>(a.H) + a.eps);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = (tid + c * nthr) * 8;
    const float top = __uint_as_float(m[c]);
    const float amax = floor_amax(top * r);
    // 2^-100 <= both and finite: 448 / top is finite and the row's factor cancels
    const bool cancels = amax > kFp8MinAmax && amax <= 3.402823466e38f && top >= kFp8MinAmax;
    const float inv = kE4m3Max / (cancels ? top : amax);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[c][i] = (cancels ? f[c][i] : f[c][i] * r) * inv;
    if (col < a.H) store_q8(a.q + row * a.ldq + col, a.H - col, a.vec_q, f[c]);
    if (col < a.H && (tid & 15) == 0) a.scales[row * a.groups + col / kFp8Group] = amax / kE4m3Max;
  }
}

int groups_of(int width) { return (width + kFp8Group - 1) / kFp8Group; }

template <typename T>
bool rows_vec(const void* p, int64_t ld) {
  return fp8_aligned(p, 16) && (ld * sizeof(T)) % 16 == 0;
}

template <typename T>
cudaError_t launch_quantize(RowArgs a, int block_rows, cudaStream_t s) {
  a.vec_in = rows_vec<T>(a.x, a.ldx);
  if (block_rows == 1) {
    const int64_t units = static_cast<int64_t>(a.M) * a.groups;
    const int64_t ctas = (units * 16 + kRowThreads - 1) / kRowThreads;
    return launch_kernel(quantize_rows_kernel<T, false>, dim3(static_cast<unsigned>(ctas)), dim3(kRowThreads), 0, s, true, a);
  }
  const unsigned blocks = static_cast<unsigned>(groups_of(a.M)) * a.groups;
  return launch_kernel(quantize_blocks_kernel<T>, dim3(blocks), dim3(kRowThreads), 0, s, true, a);
}

template <typename T>
cudaError_t launch_silu_mul(RowArgs a, cudaStream_t s) {
  a.vec_in = rows_vec<T>(a.x, a.ldx) && (a.packed || (static_cast<int64_t>(a.K) * sizeof(T)) % 16 == 0);
  const int64_t units = static_cast<int64_t>(a.M) * a.groups;
  const int64_t ctas = (units * 16 + kRowThreads - 1) / kRowThreads;
  return launch_kernel(quantize_rows_kernel<T, true>, dim3(static_cast<unsigned>(ctas)), dim3(kRowThreads), 0, s, true, a);
}

template <typename T>
cudaError_t launch_rmsnorm_fp8(NormArgs a, int M, cudaStream_t s) {
  a.vec_x = rows_vec<T>(a.x, a.ldx);
  a.vec_d = a.delta && rows_vec<T>(a.delta, a.ldd);
  a.vec_w = fp8_aligned(a.weight, 16);
  a.vec_h = a.delta && rows_vec<T>(a.h, a.ldh);
  const int chunks = (a.H + 7) / 8;
  // as many threads as chunks, up to 1024, in whole warps; then 2 or 4 chunks per thread
  const int per = chunks <= kNormMaxThreads ? 1 : chunks <= 2 * kNormMaxThreads ? 2 : 4;
  const int threads = ((chunks + per - 1) / per + 31) / 32 * 32;
  const dim3 grid(static_cast<unsigned>(M)), block(threads);
  if (per == 1) return launch_kernel(rmsnorm_fp8_kernel<T, 1>, grid, block, 0, s, true, a);
  if (per == 2) return launch_kernel(rmsnorm_fp8_kernel<T, 2>, grid, block, 0, s, true, a);
  return launch_kernel(rmsnorm_fp8_kernel<T, 4>, grid, block, 0, s, true, a);
}

}  // namespace
}  // namespace specb200

// ------------------------------------------------------------------------------ C ABI
using namespace specb200;
extern "C" int specb200_set_error(int code, const char* msg);

namespace {
int finish(cudaError_t e) {
  return e == cudaSuccess ? SPECB200_OK : specb200_set_error(SPECB200_ERR_CUDA, cudaGetErrorString(e));
}
// 2^31 - 1 CTAs of 16 groups each, and the pitches in range
bool sizes_ok(int M, int K) { return M >= 0 && K > 0 && K <= (1 << 30) && (static_cast<int64_t>(M) * groups_of(K) + 15) / 16 <= 0x7fffffff; }
}  // namespace

extern "C" int specb200_quantize_fp8(int dtype, const void* x, int64_t ldx, int M, int K, int block_rows, void* q,
                                     int64_t ldq, float* scales, void* stream) {
  if (!sizes_ok(M, K) || ldx < K || ldq < K)
    return specb200_set_error(SPECB200_ERR_ARG, "quantize_fp8: bad M/K or row pitch");
  if (block_rows != 1 && block_rows != kFp8Group)
    return specb200_set_error(SPECB200_ERR_ARG, "quantize_fp8: block_rows must be 1 or 128");
  if (dtype != SPECB200_F32 && dtype != SPECB200_BF16) return specb200_set_error(SPECB200_ERR_UNSUPPORTED, "quantize_fp8: dtype");
  if (M == 0) return SPECB200_OK;
  if (!x || !q || !scales) return specb200_set_error(SPECB200_ERR_ARG, "quantize_fp8: null pointer");
  RowArgs a = {};
  a.x = x;
  a.ldx = ldx;
  a.q = static_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scales = scales;
  a.M = M;
  a.K = K;
  a.groups = groups_of(K);
  a.vec_out = fp8_aligned(q, 8) && ldq % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return finish(dtype == SPECB200_BF16 ? launch_quantize<__nv_bfloat16>(a, block_rows, s) : launch_quantize<float>(a, block_rows, s));
}

extern "C" int specb200_silu_mul_fp8(int dtype, const void* gate_up, int64_t ld, int M, int I, int packed, void* q,
                                     int64_t ldq, float* scales, void* stream) {
  if (!sizes_ok(M, I) || ld < 2 * static_cast<int64_t>(I) || ldq < I)
    return specb200_set_error(SPECB200_ERR_ARG, "silu_mul_fp8: bad M/I or row pitch");
  if (packed && I % 64) return specb200_set_error(SPECB200_ERR_ARG, "silu_mul_fp8: packed rows need I % 64 == 0");
  if (dtype != SPECB200_F32 && dtype != SPECB200_BF16) return specb200_set_error(SPECB200_ERR_UNSUPPORTED, "silu_mul_fp8: dtype");
  if (M == 0) return SPECB200_OK;
  if (!gate_up || !q || !scales) return specb200_set_error(SPECB200_ERR_ARG, "silu_mul_fp8: null pointer");
  RowArgs a = {};
  a.x = gate_up;
  a.ldx = ld;
  a.q = static_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scales = scales;
  a.M = M;
  a.K = I;
  a.groups = groups_of(I);
  a.packed = packed ? 1 : 0;
  a.vec_out = fp8_aligned(q, 8) && ldq % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return finish(dtype == SPECB200_BF16 ? launch_silu_mul<__nv_bfloat16>(a, s) : launch_silu_mul<float>(a, s));
}

extern "C" int specb200_rmsnorm_fp8(int dtype, const void* x, int64_t ldx, const void* delta, int64_t ldd,
                                    const void* weight, int M, int H, float eps, void* h, int64_t ldh, void* q,
                                    int64_t ldq, float* scales, void* stream) {
  if (!sizes_ok(M, H) || ldx < H || ldq < H || (delta && (ldd < H || ldh < H)))
    return specb200_set_error(SPECB200_ERR_ARG, "rmsnorm_fp8: bad M/H or row pitch");
  if (dtype != SPECB200_F32 && dtype != SPECB200_BF16) return specb200_set_error(SPECB200_ERR_UNSUPPORTED, "rmsnorm_fp8: dtype");
  if (H > kNormMaxWidth) return specb200_set_error(SPECB200_ERR_UNSUPPORTED, "rmsnorm_fp8: H is at most 32768");
  if (M == 0) return SPECB200_OK;
  if (!x || !weight || !q || !scales || (delta && !h)) return specb200_set_error(SPECB200_ERR_ARG, "rmsnorm_fp8: null pointer");
  NormArgs a = {};
  a.x = x;
  a.ldx = ldx;
  a.delta = delta;
  a.ldd = ldd;
  a.weight = weight;
  a.h = h;
  a.ldh = ldh;
  a.q = static_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scales = scales;
  a.H = H;
  a.groups = groups_of(H);
  a.eps = eps;
  a.vec_q = fp8_aligned(q, 8) && ldq % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return finish(dtype == SPECB200_BF16 ? launch_rmsnorm_fp8<__nv_bfloat16>(a, M, s) : launch_rmsnorm_fp8<float>(a, M, s));
}
