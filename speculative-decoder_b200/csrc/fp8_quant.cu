// Producers of 8-bit operands (fp8.cuh): plain quantization of rows or 128 x 128 blocks, RMSNorm
// with the residual update in front, and SiLU(gate) * up. Everything between the inputs and the
// e4m3 rounding is fp32; the only other rounding is the residual stream's own element type.
//
// All are bound by memory: each input is read once, in loads of 32 bytes per lane, and each output
// written once, 16 bytes of e4m3 per lane. A group of 128 columns is held by 8 lanes with 16 elements
// each, so its maximum is three shuffles and its scale is written by the group's first lane.
#include <cuda_fp8.h>

#include <algorithm>

#include "fp8.cuh"
#include "kernels.cuh"

namespace specb200 {
namespace {

// Two fp32 values in a register pair, one instruction for both: these kernels run next to the
// power limit, where every instruction saved is clock rate gained.
typedef unsigned long long f32x2;
SPECB200_DEVINL f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
SPECB200_DEVINL float2 unpack2(f32x2 v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
SPECB200_DEVINL f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SPECB200_DEVINL f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SPECB200_DEVINL f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Sixteen consecutive elements of a row, in the form they have in memory.
template <typename T>
struct Raw16 {
  uint32_t v[4 * sizeof(T)];
};
// The same as they are loaded. kAny = false: rows start on 16-byte boundaries; one or two 256-bit
// loads (or 128-bit ones, align 16). kAny = true: rows start anywhere, and what is loaded is the
// 16-byte units that the elements lie in, `shift` bytes of the first one ahead of them (16384 x 2050
// bf16: quantize 22.7 us, RMSNorm 72; with a load per element 38 and 207; with 32-byte units, fewer loads and
// more to shift, 25.6 and 84).
template <typename T, bool kAny>
struct Loaded16 {
  uint32_t v[4 * sizeof(T) + (kAny ? 4 : 0)];
  uint32_t shift;
};
// first, end: the bytes of the whole tensor, beyond which no unit is read.
template <typename T, bool kAny>
SPECB200_DEVINL void load16(Loaded16<T, kAny>& r, const T* p, int valid, int align, const void* first, const void* end) {
  constexpr int kWords = 4 * sizeof(T), kAll = kAny ? kWords + 4 : kWords;
  const char* b = reinterpret_cast<const char*>(p);
  r.shift = 0;
  if constexpr (kAny) {
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15), bytes = min(valid, 16) * static_cast<int>(sizeof(T)) + shift;
    b -= shift;
    if (valid > 0 && b >= first && b + (bytes + 15) / 16 * 16 <= end) {
      r.shift = shift;
#pragma unroll
      for (int i = 0; i < kAll; i += 4) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (4 * i < bytes) q = *reinterpret_cast<const uint4*>(b + 4 * i);
        r.v[i] = q.x; r.v[i + 1] = q.y; r.v[i + 2] = q.z; r.v[i + 3] = q.w;
      }
      if (valid < 16) {  // what follows the row's end
#pragma unroll
        for (int i = 0; i < kAll; ++i) {
          const int left = bytes - 4 * i;
          if (left <= 0) r.v[i] = 0;
          if (left == 2) r.v[i] &= 0xffffu;
        }
      }
      return;
    }
  } else if (align >= 16 && valid >= 16) {
    if (align >= 32) {
#pragma unroll
      for (int i = 0; i < kWords; i += 8)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.v[i]), "=r"(r.v[i + 1]), "=r"(r.v[i + 2]), "=r"(r.v[i + 3]), "=r"(r.v[i + 4]),
                       "=r"(r.v[i + 5]), "=r"(r.v[i + 6]), "=r"(r.v[i + 7])
                     : "l"(b + 4 * i));
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(b + 4 * i);
        r.v[i] = q.x; r.v[i + 1] = q.y; r.v[i + 2] = q.z; r.v[i + 3] = q.w;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kAll; ++i) r.v[i] = 0;
  if (valid <= 0) return;  // lanes behind a row's end: their warp need not go through the single loads
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (sizeof(T) == 2) {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
      const uint32_t lo = 2 * i < valid ? h[2 * i] : 0, hi = 2 * i + 1 < valid ? h[2 * i + 1] : 0;
      r.v[i] = lo | (hi << 16);
    } else {
      r.v[i] = i < valid ? reinterpret_cast<const uint32_t*>(p)[i] : 0;
    }
  }
}
// w[0..kOut) = the words that start `bytes` (0..15, even) into w. kJump: a jump to code for each number of
// words instead of selects, the same one for a whole row. It pays where one or two shifts stand in a
// kernel of few registers (16392 x 2047 bf16: RMSNorm 59 us against 63, rows quantized 20.3 and 21.7) and
// not for blocks (31.7 and 28.7, fp32 56 and 38), SiLU (fp32 58.6 and 56.2) or the fp32 norm (93 and 92).
template <int kOut, bool kHalves, int kSkip>
SPECB200_DEVINL void shift_from(uint32_t (&w)[kOut + 4], uint32_t bits) {
#pragma unroll
  for (int i = 0; i < kOut; ++i) w[i] = kHalves ? __funnelshift_r(w[i + kSkip], w[i + kSkip + (kHalves ? 1 : 0)], bits) : w[i + kSkip];
}
template <int kOut, bool kHalves, bool kJump>
SPECB200_DEVINL void shift_words(uint32_t (&w)[kOut + 4], uint32_t bytes) {
  const uint32_t bits = (bytes & 2) * 8;
  if constexpr (kJump) {
    switch (bytes >> 2) {
      case 0: shift_from<kOut, kHalves, 0>(w, bits); break;
      case 1: shift_from<kOut, kHalves, 1>(w, bits); break;
      case 2: shift_from<kOut, kHalves, 2>(w, bits); break;
      default: shift_from<kOut, kHalves, 3>(w, bits); break;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kOut + 2; ++i) w[i] = bytes & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < kOut + 1; ++i) w[i] = bytes & 4 ? w[i + 1] : w[i];
    if constexpr (kHalves) shift_from<kOut, kHalves, 0>(w, bits);
  }
}
template <bool kJump, typename T, bool kAny>
SPECB200_DEVINL Raw16<T> aligned16(const Loaded16<T, kAny>& l) {
  constexpr int kWords = 4 * sizeof(T);
  Raw16<T> r;
  if constexpr (kAny) {
    uint32_t w[kWords + 4];
#pragma unroll
    for (int i = 0; i < kWords + 4; ++i) w[i] = l.v[i];
    shift_words<kWords, sizeof(T) == 2, kJump>(w, l.shift);
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.v[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.v[i] = l.v[i];
  }
  return r;
}
template <typename T>
SPECB200_DEVINL void unpack16(const Raw16<T>& r, f32x2 (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 2)
      f[i] = pack2(__uint_as_float(r.v[i] << 16), __uint_as_float(r.v[i] & 0xffff0000u));
    else
      f[i] = pack2(__uint_as_float(r.v[2 * i]), __uint_as_float(r.v[2 * i + 1]));
  }
}
// Rounded to T, in memory's form.
template <typename T>
SPECB200_DEVINL Raw16<T> round16(const f32x2 (&f)[8]) {
  Raw16<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = unpack2(f[i]);
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
      r.v[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      r.v[2 * i] = __float_as_uint(v.x);
      r.v[2 * i + 1] = __float_as_uint(v.y);
    }
  }
  return r;
}
// The first `bytes` (0..16) of w to p, which is on a 16-byte boundary.
SPECB200_DEVINL void store_unit(char* p, int bytes, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  if (bytes >= 16) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w0, w1, w2, w3);
    return;
  }
  if (bytes <= 0) return;
  if (bytes & 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w0, w1);
    w0 = w2; w1 = w3;
    p += 8;
  }
  if (bytes & 4) {
    *reinterpret_cast<uint32_t*>(p) = w0;
    w0 = w1;
    p += 4;
  }
  if (bytes & 2) {
    *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w0);
    w0 >>= 16;
    p += 2;
  }
  if (bytes & 1) *p = static_cast<char>(w0);
}
// Sixteen elements of a row per lane, `valid` of them and what follows inside the row; prev, next: the
// lane before, behind holds its neighbours. All lanes of the warp take part. kAny: each lane stores the
// 16-byte units that start among its elements and end with the next lane's first ones; where there is
// no such lane, what lies outside whole units is stored in smaller pieces.
template <typename T, bool kAny>
SPECB200_DEVINL void store16(T* to, int valid, bool prev, bool next, const Raw16<T>& r) {
  constexpr int kWords = 4 * sizeof(T), kBytes = 4 * kWords;
  char* p = reinterpret_cast<char*>(to);
  int bytes = max(valid, 0) * static_cast<int>(sizeof(T));
  if constexpr (kAny) {
    uint32_t w[kWords + 4];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = r.v[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[kWords + i] = __shfl_down_sync(0xffffffffu, r.v[i], 1);
    if (!next) bytes = min(bytes, kBytes);
    const int head = static_cast<int>(-reinterpret_cast<uintptr_t>(p) & 15);
    if (!prev && head) {
      const int n = min(head, bytes);
#pragma unroll
      for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) {
        if (i * static_cast<int>(sizeof(T)) < n) {
          if constexpr (sizeof(T) == 2)
            reinterpret_cast<unsigned short*>(p)[i] = static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)));
          else
            reinterpret_cast<uint32_t*>(p)[i] = w[i];
        }
      }
    }
    shift_words<kWords, sizeof(T) == 2, sizeof(T) == 2>(w, head);
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
      store_unit(p + head + 4 * i, bytes - head - 4 * i, w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else {
    if (valid >= 16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        *reinterpret_cast<uint4*>(p + 4 * i) = make_uint4(r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]);
      return;
    }
    if (valid <= 0) return;
#pragma unroll
    for (int i = 0; i < kWords; i += 4) store_unit(p + 4 * i, bytes - 4 * i, r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]);
  }
}
// e4m3 of 16 values of a row, rounded to nearest even. Finite values beyond 448 (a group's maximum can
// exceed it by an ulp) saturate, NaN stays NaN.
SPECB200_DEVINL void store_e4m3_16(uint8_t* p, int valid, int align, const f32x2 (&f)[8]) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(unpack2(f[2 * i]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(unpack2(f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    v[i] = lo | (hi << 16);
  }
  if (align >= 16 && valid >= 16) {
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
    return;
  }
  if (align >= 16) {
    store_unit(reinterpret_cast<char*>(p), valid, v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < valid) p[i] = static_cast<uint8_t>(v[i / 4] >> (8 * (i & 3)));
}

// e4m3(f * inv).
SPECB200_DEVINL void store_q16(uint8_t* p, int valid, int align, const f32x2 (&f)[8], float inv) {
  const f32x2 inv2 = pack2(inv, inv);
  f32x2 t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = mul2(f[i], inv2);
  store_e4m3_16(p, valid, align, t);
}

// A group's scale, and what divides by it. Where elements lie between two e4m3 numbers the quotient often
// does so too but for the scale's own rounding (bf16 ones most of all), so q = e4m3(x / s) is formed from
// the IEEE quotient by the scale as it is stored: whoever holds x and s can form the same q. Products with
// 448 / amax put 0.03 % of a batch of activations and 0.008 % of a weight matrix on the other side.
//
// The scale: amax (hi + lo) with hi + lo = 1 / 448 to 2^-51 and one rounding of the sum. amax / 7 lies at
// least 1/14 ulp from the middle of two fp32 numbers, so this is the IEEE quotient.
// Elements: 1 / s as hi + lo, hi below it and lo > 0, so that zeros keep their signs. x hi + x lo is off by less
// than 2^-42 of itself before its one rounding (the reciprocal by at most 2^-22, which lo corrects). No
// pair of bf16 mantissas puts x / s within 2^-40 of the middle of two fp32 numbers (the test looks at them
// all), so this is the IEEE quotient; for fp32 one quotient in 2^18 is next to such a middle and may go
// an ulp the other way, which e4m3 sees where it is next to the middle of two of its numbers as well.
// Maxima beyond 2^110 leave lo in the subnormal range and x hi + x lo off by up to 2^-30 before the rounding.
// quantize 32768 x 2048 bf16: 31.5 us (32.0 by products and IEEE divisions for s and 448 / amax, 37.4 with a
// division's correction step instead of lo); weight blocks 16384 x 2048 18.4 (17.6).
struct Divisor {
  float s;       // the scale
  float hi, lo;  // 1 / s
};
SPECB200_DEVINL Divisor divisor_of(float amax) {
  Divisor c;
  const bool finite = amax <= 3.402823466e38f;  // else q = x * (1 / s), which is 0 or NaN
  c.s = finite ? fmaf(amax, 0x1.24924ap-9f, amax * -0x1.b6db6ep-34f) : amax;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(c.s));
  c.hi = r * (1.f - 0x1p-21f);
  c.lo = finite ? fmaf(-c.s, c.hi, 1.f) * r : 0.f;
  return c;
}
// e4m3(f / c.s).
SPECB200_DEVINL void store_quotients16(uint8_t* p, int valid, int align, f32x2 (&f)[8], const Divisor& c) {
  const f32x2 hi = pack2(c.hi, c.hi), lo = pack2(c.lo, c.lo);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fma2(f[i], hi, mul2(f[i], lo));
  store_e4m3_16(p, valid, align, f);
}

SPECB200_DEVINL float max_mag16(const f32x2 (&f)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = unpack2(f[i]);
    m = max_mag(max_mag(m, v.x), v.y);
  }
  return m;
}
// Maximum over the 8 lanes that hold a group.
SPECB200_DEVINL float octet_max(float m) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// silu(g) * u = g u / (1 + 2^(-g log2 e)) for a pair, g >= -87. The exponent is rounded to fp32, which leaves
// |g| 2^-23 in the exponential: nothing next to the 1 for positive gates, and for negative ones a
// relative error that grows as the value itself dies away. An infinite gate gives inf u.
SPECB200_DEVINL f32x2 silu_mul2(f32x2 g, f32x2 u) {
  constexpr float kLog2e = 1.44269504f;
  const float2 t = unpack2(mul2(g, pack2(-kLog2e, -kLog2e)));
  float2 e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  const float2 d = unpack2(add2(pack2(e.x, e.y), pack2(1.f, 1.f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(d.y));
  return mul2(mul2(g, pack2(s.x, s.y)), u);
}

// The same below -87, where the 1 is nothing next to the exponential and the exponential's reciprocal leaves
// fp32's range (the fast reciprocal is zero from -87.34 on): e^g in two halves, one for each factor, which
// reaches as far down as any fp32 `up` can lift the value above what e4m3 holds (-177). -inf gives NaN, as
// the formula does.
SPECB200_DEVINL float silu_mul_far(float g, float u) {
  const float half = expf(0.5f * g);
  return (g * half) * (half * u);
}
// Whether any of 16 gates is below -87 (or a NaN with a sign): as whole numbers, these are the ones above
// that of -87.
template <typename T>
SPECB200_DEVINL bool any_far(const Raw16<T>& g) {
  uint32_t m = g.v[0];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __vmaxu2(m, g.v[i]);
    return max(m >> 16, m & 0xffffu) > 0xc2aeu;
  } else {
#pragma unroll
    for (int i = 1; i < 16; ++i) m = max(m, g.v[i]);
    return m > 0xc2ae0000u;
  }
}

struct RowArgs {
  const void* x;       // quantize: [M, K]; SiLU: gate | up
  int64_t ldx;         // elements
  uint8_t* q;
  int64_t ldq;
  float* scales;       // [M, groups] (or [row blocks, groups])
  int M, K, groups;
  int packed;          // SiLU: 1 = 64 gate columns, then their 64 up columns
  const void* x_end;   // where x's last row ends
  int vec_in, vec_out; // rows of x / q start on boundaries of this many bytes
};

constexpr int kRowThreads = 256;

// One group of the row-major list of all groups per 8 lanes, 16 elements each. kSilu: y =
// silu(gate) * up, else y = x. Bound by memory: what counts is loads in flight, so bf16 keeps to 32
// registers (8 CTAs per SM); two groups per thread at 48 registers took longer at every size. SiLU's two
// inputs off the 16-byte boundaries need more: 16392 x 2047 39.6 us at 6, 43.7 at 8, fp32 56.3 at 4, 60.0 at 5 (now 40.0 and 56.6).
template <typename T, bool kSilu, bool kAny>
__global__ void __launch_bounds__(kRowThreads, (sizeof(T) == 2 ? 8 : 5) - (kSilu && kAny ? (sizeof(T) == 2 ? 2 : 1) : 0))
    quantize_rows_kernel(RowArgs a) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 7;
  const uint32_t groups = a.groups;
  const int64_t start = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 8);  // the same in all threads
  const int64_t row0 = start / groups;
  const uint32_t at = static_cast<uint32_t>(start - row0 * groups) + (threadIdx.x >> 3);
  const uint32_t over = at < groups ? 0u : at / groups;
  const int64_t row = row0 + over;
  const int g = static_cast<int>(at - over * groups), col = g * kFp8Group + lane * 16;
  const int valid = row < a.M ? a.K - col : 0;
  const T* xr = static_cast<const T*>(a.x) + row * a.ldx;
  pdl_wait();
  Loaded16<T, kAny> raw;
  f32x2 y[8];
  if constexpr (kSilu) {
    // packed: feature j is gate column 128 (j / 64) + j % 64, its up column 64 further on
    const int gate = a.packed ? ((col >> 6) << 7) + (col & 63) : col;
    Loaded16<T, kAny> raw_up;
    load16(raw, xr + gate, valid, a.vec_in, a.x, a.x_end);
    load16(raw_up, xr + gate + (a.packed ? 64 : a.K), valid, a.vec_in, a.x, a.x_end);
    f32x2 up[8];
    const Raw16<T> gates = aligned16<false>(raw);
    unpack16<T>(gates, y);
    unpack16<T>(aligned16<false>(raw_up), up);
    const bool far = any_far(gates);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = silu_mul2(y[j], up[j]);
    if (far) {  // rare: the elements are read again, so that the registers of the others need not be kept
      const T* gp = xr + gate;
      const T* upp = gp + (a.packed ? 64 : a.K);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float2 v = unpack2(y[j]);
        const float g0 = 2 * j < valid ? to_f32(gp[2 * j]) : 0.f, g1 = 2 * j + 1 < valid ? to_f32(gp[2 * j + 1]) : 0.f;
        if (g0 < -87.f) v.x = silu_mul_far(g0, to_f32(upp[2 * j]));
        if (g1 < -87.f) v.y = silu_mul_far(g1, to_f32(upp[2 * j + 1]));
        y[j] = pack2(v.x, v.y);
      }
    }
  } else {
    load16(raw, xr + col, valid, a.vec_in, a.x, a.x_end);
    unpack16<T>(aligned16<true>(raw), y);
  }
  const float amax = floor_amax(octet_max(max_mag16(y)));
  const Divisor c = divisor_of(amax);
  if (valid > 0) store_quotients16(a.q + row * a.ldq + col, valid, a.vec_out, y, c);
  if (row < a.M && lane == 0) a.scales[row * groups + g] = c.s;
}

// One 128 x 128 block per CTA, held in registers between the maximum and the rounding: 8 lanes
// per row, 32 rows at a time. Rows off the 16-byte boundaries: a CTA more per SM, although it costs
// spilled registers (16368 x 2050: 29.9 us, fp32 40.8; before the quotients by the stored scale 28.3 and
// 37.2, against 30.2 and 40.9 with a CTA less).
template <typename T, bool kAny>
__global__ void __launch_bounds__(kRowThreads, (sizeof(T) == 2 ? 3 : 2) + kAny) quantize_blocks_kernel(RowArgs a) {
  constexpr int kLanes = kRowThreads / 8, kPass = kFp8Group / kLanes;
  __shared__ float sh[kRowThreads / 32];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  const int g = blockIdx.x % a.groups, rb = blockIdx.x / a.groups;
  const int col = g * kFp8Group + lane * 16;
  const int valid = a.K - col;
  const int rows = min(kFp8Group, a.M - rb * kFp8Group);
  const int64_t first = static_cast<int64_t>(rb) * kFp8Group + r0;
  const T* xp = static_cast<const T*>(a.x) + first * a.ldx + col;
  uint8_t* qp = a.q + first * a.ldq + col;
  pdl_wait();
  Loaded16<T, kAny> x[kPass];
#pragma unroll
  for (int p = 0; p < kPass; ++p)
    load16(x[p], xp + p * kLanes * a.ldx, r0 + p * kLanes < rows ? valid : 0, a.vec_in, a.x, a.x_end);
  float m = 0.f;
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    f32x2 y[8];
    unpack16<T>(aligned16<false>(x[p]), y);
    m = max_nan(m, max_mag16(y));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) m = max_nan(m, sh[i]);
  const Divisor c = divisor_of(floor_amax(m));
#pragma unroll
  for (int p = 0; p < kPass; ++p) {
    f32x2 y[8];
    unpack16<T>(aligned16<false>(x[p]), y);
    if (r0 + p * kLanes < rows && valid > 0) store_quotients16(qp + p * kLanes * a.ldq, valid, a.vec_out, y, c);
  }
  if (threadIdx.x == 0) a.scales[blockIdx.x] = c.s;
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
  int M, H, groups;
  int rows;            // rows that a CTA takes at a time
  float eps;
  const void *x_end, *d_end, *w_end;  // where the last row ends
  int vec_x, vec_d, vec_w, vec_h, vec_q;  // boundaries in bytes
};

constexpr int kNormMaxChunks = 4;                            // groups of a row per 8 lanes
constexpr int kNormMaxWidth = kNormMaxChunks * 64 * kFp8Group;  // 64 octets: 512 threads

// CTAs per SM that the registers are cut for. 32768 x 2048 bf16 with delta, loads ahead: 71.5 us at 3
// CTAs (floor 71.9 at the measured copy bandwidth), 81.8 at 2, and 86.2 at 4, which leaves no room for
// loads ahead; fp32 16384 x 2048: 67.1 at 2, 80.5 at 3. 8192 x 8192 bf16 (two groups per octet): 80.7
// at 3, 84.4 at 2, 87.4 at 4. Rows off the 16-byte boundaries need their registers for the units and
// hide the loads behind other CTAs' work: 16392 x 2047 bf16 59 us, fp32 92 (63 and 92 against 72 and 113 with loads
// ahead, before the last step).
template <typename T, int kChunks, bool kAny>
constexpr int kNormCtas = kChunks == 4 ? 1
                                : kAny       ? (kChunks == 2 && sizeof(T) == 4 ? 2 : 4)
                                             : (kChunks == 2 || sizeof(T) == 2 ? 3 : 2);

// h = T(x + delta); y = w h / sqrt(mean(h^2) + eps); (q, scales) = quantize(y).
//
// Eight lanes hold one group of a row (kChunks groups of a wide one); a CTA takes as many rows at
// a time as it has octets for, and walks over the rows with its weights in registers. With one group per
// octet and rows on 16-byte boundaries the next rows' loads are issued before the current rows' sums are formed. A row's sum of squares is added
// within each octet by shuffles, then over the octets in a fixed order.
//
// The quantized values need no norm: with m the group's largest |w h| and r the row's 1 / rms,
// y / s = (w h r) / (m r / 448) = w h (448 / m), so q carries two roundings and only the scale
// waits for the row's sum. Where the floor is in play or a value is not finite, q is formed from
// y itself.
template <typename T, int kChunks, bool kDelta, bool kAny>
__global__ void __launch_bounds__(kChunks == 4 ? 512 : 256, kNormCtas<T, kChunks, kAny>) rmsnorm_fp8_kernel(NormArgs a) {
  constexpr bool kAhead = kChunks == 1 && !kAny, kJump = sizeof(T) == 2;
  __shared__ float sh[2][64];
  pdl_launch_dependents();
  const int octet = threadIdx.x >> 3, octets = blockDim.x >> 3;
  const int per_row = min(octets, a.groups);  // octets that share a row
  const int team = kChunks == 1 ? octet / per_row : 0;
  const int g0 = octet - team * per_row;
  const int col0 = g0 * kFp8Group + (threadIdx.x & 7) * 16;
  // whether the neighbouring lanes of this warp hold the neighbouring columns
  const bool prev = (threadIdx.x & 31) != 0 && col0 > 0, next = (threadIdx.x & 31) != 31 && col0 + 16 < per_row * kFp8Group;
  const int pitch = octets * kFp8Group;  // from chunk to chunk of a thread
  Raw16<T> w[kChunks];
  Loaded16<T, kAny> x[kChunks], d[kDelta ? kChunks : 1];
  auto valid_of = [&](int64_t row, int c) { return team < a.rows && row < a.M ? a.H - (col0 + c * pitch) : 0; };
  auto load_row = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = col0 + c * pitch, valid = valid_of(row, c);
      load16(x[c], static_cast<const T*>(a.x) + row * a.ldx + col, valid, a.vec_x, a.x, a.x_end);
      if constexpr (kDelta)
        load16(d[c], static_cast<const T*>(a.delta) + row * a.ldd + col, valid, a.vec_d, a.delta, a.d_end);
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.rows;
  int64_t base = static_cast<int64_t>(blockIdx.x) * a.rows;
  pdl_wait();
  if constexpr (kAhead) load_row(base + team);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = col0 + c * pitch;
    Loaded16<T, kAny> l;
    load16(l, static_cast<const T*>(a.weight) + col, a.H - col, a.vec_w, a.weight, a.w_end);
    w[c] = aligned16<false>(l);
  }
  for (int parity = 0; base < a.M; base += step, parity ^= 1) {
    const int64_t row = base + team;
    f32x2 f[kChunks][8];
    float m[kChunks], ss = 0.f;
    if constexpr (!kAhead) load_row(row);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      unpack16<T>(aligned16<kJump>(x[c]), f[c]);
      if constexpr (kDelta) {
        f32x2 g[8];
        unpack16<T>(aligned16<kJump>(d[c]), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[c][i] = add2(f[c][i], g[i]);
        const Raw16<T> h = round16<T>(f[c]);
        store16<T, kAny>(static_cast<T*>(a.h) + row * a.ldh + col0 + c * pitch, valid_of(row, c), prev, next, h);
        unpack16<T>(h, f[c]);
      }
    }
    if constexpr (kAhead) {
      if (base + step < a.M) load_row(row + step);
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      f32x2 g[8], part = pack2(0.f, 0.f);
      unpack16<T>(w[c], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        part = fma2(f[c][i], f[c][i], part);
        f[c][i] = mul2(f[c][i], g[i]);
      }
      const float2 sums = unpack2(part);
      ss += sums.x + sums.y;
      m[c] = octet_max(max_mag16(f[c]));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((threadIdx.x & 7) == 0) sh[parity][octet] = ss;
    __syncthreads();  // one per round: the next round's sums go to the other half
    const float* part = &sh[parity][team * per_row];
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    if (team < a.rows) {
      int i = 0;
      for (; i + 4 <= per_row; i += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[j] += part[i + j];
      }
      for (; i < per_row; ++i) sums[0] += part[i];
    }
    const float total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const float r = 1.f / sqrtf(total / static_cast<float>(a.H) + a.eps);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = col0 + c * pitch, valid = valid_of(row, c);
      const float amax = floor_amax(m[c] * r);
      // 2^-100 <= both and finite: 448 / m is finite and the row's factor cancels
      const bool cancels = amax > kFp8MinAmax && amax <= 3.402823466e38f && m[c] >= kFp8MinAmax;
      if (!cancels) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[c][i] = mul2(f[c][i], pack2(r, r));
      }
      if (valid > 0) {
        store_q16(a.q + row * a.ldq + col, valid, a.vec_q, f[c], kE4m3Max / (cancels ? m[c] : amax));
        if ((threadIdx.x & 7) == 0) a.scales[row * a.groups + col / kFp8Group] = amax / kE4m3Max;
      }
    }
  }
}

int groups_of(int width) { return (width + kFp8Group - 1) / kFp8Group; }

// The largest power of two up to 32 on whose multiples (in bytes) every row starts.
int row_align(const void* p, int64_t pitch_bytes) {
  int n = 32;
  while (n > 1 && (reinterpret_cast<uintptr_t>(p) % n || pitch_bytes % n)) n /= 2;
  return n;
}
template <typename T>
int row_align_of(const void* p, int64_t ld) {
  return row_align(p, ld * static_cast<int64_t>(sizeof(T)));
}

unsigned row_ctas(const RowArgs& a) {
  const int64_t units = static_cast<int64_t>(a.M) * a.groups, per_cta = kRowThreads / 8;
  return static_cast<unsigned>((units + per_cta - 1) / per_cta);
}

// Where the last of M rows of K elements ends.
template <typename T>
const void* end_of(const void* x, int64_t ld, int M, int K) {
  return static_cast<const T*>(x) + (M - 1) * ld + K;
}

template <typename T, bool kSilu>
cudaError_t launch_rows(const RowArgs& a, cudaStream_t s) {
  return a.vec_in >= 16 ? launch_kernel(quantize_rows_kernel<T, kSilu, false>, dim3(row_ctas(a)), dim3(kRowThreads), 0, s, true, a)
                        : launch_kernel(quantize_rows_kernel<T, kSilu, true>, dim3(row_ctas(a)), dim3(kRowThreads), 0, s, true, a);
}

template <typename T>
cudaError_t launch_quantize(RowArgs a, int block_rows, cudaStream_t s) {
  a.vec_in = row_align_of<T>(a.x, a.ldx);
  a.x_end = end_of<T>(a.x, a.ldx, a.M, a.K);
  if (block_rows == 1) return launch_rows<T, false>(a, s);
  const unsigned blocks = static_cast<unsigned>(groups_of(a.M)) * a.groups;
  return a.vec_in >= 16 ? launch_kernel(quantize_blocks_kernel<T, false>, dim3(blocks), dim3(kRowThreads), 0, s, true, a)
                        : launch_kernel(quantize_blocks_kernel<T, true>, dim3(blocks), dim3(kRowThreads), 0, s, true, a);
}

template <typename T>
cudaError_t launch_silu_mul(RowArgs a, cudaStream_t s) {
  a.vec_in = row_align_of<T>(a.x, a.ldx);
  a.x_end = end_of<T>(a.x, a.ldx, a.M, 2 * a.K);
  if (!a.packed) a.vec_in = std::min(a.vec_in, row_align_of<T>(a.x, a.K));  // where the up columns start
  return launch_rows<T, true>(a, s);
}

// As many CTAs as the 148 SMs hold at once, each on every grid-th set of rows. Up to the number that
// the kernel's registers are cut for every row set has its CTA, and the driver need not be asked.
template <int kCtas, typename K>
cudaError_t launch_filled(K kernel, const NormArgs& a, int threads, cudaStream_t s) {
  const int wanted = (a.M - 1) / a.rows + 1;
  int per_sm = kCtas;
  if (wanted > 148 * kCtas) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(kernel, dim3(std::min(wanted, 148 * std::max(1, per_sm))), dim3(threads), 0, s, true, a);
}
template <typename T, int kChunks, bool kAny>
cudaError_t launch_norm_rows(const NormArgs& a, int octets, cudaStream_t s) {
  constexpr int kCtas = kNormCtas<T, kChunks, kAny>;
  const int threads = (octets * 8 + 31) / 32 * 32;
  return a.delta ? launch_filled<kCtas>(rmsnorm_fp8_kernel<T, kChunks, true, kAny>, a, threads, s)
                 : launch_filled<kCtas>(rmsnorm_fp8_kernel<T, kChunks, false, kAny>, a, threads, s);
}
template <typename T, int kChunks>
cudaError_t launch_norm_kernel(const NormArgs& a, int octets, cudaStream_t s) {
  const int align = std::min({a.vec_x, a.vec_d, a.vec_w, a.vec_h});
  return align >= 16 ? launch_norm_rows<T, kChunks, false>(a, octets, s) : launch_norm_rows<T, kChunks, true>(a, octets, s);
}

template <typename T>
cudaError_t launch_rmsnorm_fp8(NormArgs a, cudaStream_t s) {
  a.vec_x = row_align_of<T>(a.x, a.ldx);
  a.vec_d = row_align_of<T>(a.delta, a.ldd);
  a.vec_w = row_align(a.weight, 0);
  a.vec_h = row_align_of<T>(a.h, a.ldh);
  if (!a.delta) a.vec_d = a.vec_h = 32;
  a.x_end = end_of<T>(a.x, a.ldx, a.M, a.H);
  a.d_end = a.delta ? end_of<T>(a.delta, a.ldd, a.M, a.H) : nullptr;
  a.w_end = end_of<T>(a.weight, 0, 1, a.H);
  a.rows = 1;
  if (a.groups > 64) return launch_norm_kernel<T, 4>(a, std::max(32, (a.groups + 3) / 4), s);
  if (a.groups > 32) return launch_norm_kernel<T, 2>(a, (a.groups + 1) / 2, s);
  // few rows: one per CTA, so that they spread over the SMs; many: as many as 32 octets hold
  a.rows = std::max(1, std::min(32 / a.groups, a.M / (2 * 148)));
  return launch_norm_kernel<T, 1>(a, a.rows * a.groups, s);
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
// At most 2^31 - 1 times 16 groups (a CTA takes 32), and columns that fit an int with their up halves
uint64_t bytes_of(int dtype) { return dtype == SPECB200_BF16 ? 2 : 4; }
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
  if (!fp8_aligned(x, bytes_of(dtype)) || !fp8_aligned(scales, 4))
    return specb200_set_error(SPECB200_ERR_ARG, "quantize_fp8: a pointer is not on a boundary of its elements");
  RowArgs a = {};
  a.x = x;
  a.ldx = ldx;
  a.q = static_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scales = scales;
  a.M = M;
  a.K = K;
  a.groups = groups_of(K);
  a.vec_out = row_align(q, ldq);
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
  if (!fp8_aligned(gate_up, bytes_of(dtype)) || !fp8_aligned(scales, 4))
    return specb200_set_error(SPECB200_ERR_ARG, "silu_mul_fp8: a pointer is not on a boundary of its elements");
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
  a.vec_out = row_align(q, ldq);
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
  const uint64_t e = bytes_of(dtype);
  if (!fp8_aligned(x, e) || !fp8_aligned(weight, e) || !fp8_aligned(delta, e) || (delta && !fp8_aligned(h, e)) || !fp8_aligned(scales, 4))
    return specb200_set_error(SPECB200_ERR_ARG, "rmsnorm_fp8: a pointer is not on a boundary of its elements");
  if (delta && M > 1 && ((h == x && ldh != ldx) || (h == delta && ldh != ldd)))
    return specb200_set_error(SPECB200_ERR_ARG, "rmsnorm_fp8: h in the place of x or delta has its row pitch");
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
  a.M = M;
  a.H = H;
  a.groups = groups_of(H);
  a.eps = eps;
  a.vec_q = row_align(q, ldq);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return finish(dtype == SPECB200_BF16 ? launch_rmsnorm_fp8<__nv_bfloat16>(a, s) : launch_rmsnorm_fp8<float>(a, s));
}
