// Linear layers on 8-bit operands (fp8.cuh): with xq, wq e4m3 and b running over the groups of
// 128 along K,
//   y[m, n] = sum_b  sx[m, b] * sw[n / 128, b] * sum_{k in b} xq[m, k] * wq[n, k].
//
// The inner sum runs on the tensor cores (tcgen05.mma kind::f8f6f4, fp32 accumulator in TMEM);
// its 128 products of one group share one pair of scales, so each group's partial tile is read
// back and added to fp32 registers with the factor sx * sw, while the MMAs of the next group run
// into another TMEM buffer. Where tokens lie on the TMEM lanes a thread owns one token and features of
// one weight block, so the factor of a group is one number per thread. Operands come by TMA, K-major
// with the 128-byte swizzle (one atom is one group). Three kernels:
//
// - gemm_fp8_few_kernel: up to 16 tokens x 128 features per CTA, features on the lanes.
// - gemm_fp8_small_kernel: a CTA computes one tile of 128 tokens x 128 features, one or two CTAs per
//   SM. In either, with few tiles K is split over the CTAs of a cluster: each leaves its partial tile in its own
//   shared memory and the cluster adds them through distributed shared memory in split order, so
//   results do not depend on scheduling and no workspace exists that two calls could share.
// - gemm_fp8_pair_kernel: a pair of CTAs (cta_group::2) walks over tiles of 256 tokens x 256
//   features. Each CTA loads half of either operand, so that a group costs an SM 32 KB from L2
//   instead of 48, and holds 128 tokens of the accumulators.
#include <algorithm>
#include <atomic>

#include "fp8.cuh"
#include "gemm.cuh"

namespace specb200 {
namespace {

constexpr int kF8TileM = 128;
constexpr int kF8Block = 128;     // features per weight block
constexpr int kF8MaxSplits = 4;
constexpr int kF8MaxStages = 12;
constexpr int kF8MaxDevices = 64;
constexpr int kF8EpiWarps = 8;
// The small kernel is cut for one or two CTAs per SM: alone a CTA has four TMEM buffers, twice the
// ring, a second producer warp and registers to read ahead (64 x 6144 x 2048: 7.4 us against 9.6; 320 x
// 2048 x 8192 without a split of K: 22.3 against 34.6). Two to an SM hide each other's start and end where there are
// more tiles than SMs.
__host__ __device__ constexpr int f8_small_threads(int per_sm) { return per_sm == 1 ? 352 : 320; }
__host__ __device__ constexpr int f8_small_bufs(int per_sm) { return per_sm == 1 ? 4 : 2; }
// Groups whose weights the small kernels bring to L2 before they wait for the kernel in front. 5 x
// 16384 x 2048 (in a chain of its own kind): 8.0 us, 8.2 without and with 11 groups; the 8 calls of a
// layer of 5 tokens (2048 wide, MLP 8192): 29.8 us, 31.1 without, 29.6 with 11.
constexpr int kF8Ahead = 4;
constexpr int kF8PairThreads = 384;
constexpr int kF8PairStages = 4;
constexpr int kF8OutPiece = 4096; // 32 rows x 128 bytes of output on their way to memory
constexpr uint32_t kF8TileBytes = 128 * kFp8Group;  // 128 rows of one group

struct F8Args {
  int M, N, K;
  int kblocks, m_tiles, n_tiles, splits, stages;
  uint32_t ring_bytes;
  uint32_t x_bytes;     // bytes of a stage's token box (box rows x 128)
  const float* xs;      // [M, kblocks]
  const float* ws;      // [n / 128, kblocks]
  void* y;
  int64_t ldy;
  int out_f32;
  int rows16;           // y's rows are on 16-byte boundaries: tiles are written by TMA, split ones in quads
  int tail16;           // ... and end on one
  int starved;          // no operand is ever loaded: every wait for one runs out
  int32_t* status;
};

// The MMAs of one group (128 of K in four instructions), overwriting the accumulator, and a commit:
// `done` completes once they have run, here and (kPair) in the peer CTA. Every lane of the warp
// executes this, the elected one (leader != 0) issues.
template <bool kPair>
SPECB200_DEVINL void umma_group_e4m3(uint32_t leader, uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                     uint64_t* done) {
  if constexpr (kPair) {
    asm volatile(
        "{\n\t.reg .pred p, first, rest;\n\t"
        "setp.ne.b32 p, %0, 0;\n\t"
        "setp.ne.b32 first, 0, 0;\n\t"
        "setp.eq.b32 rest, 0, 0;\n\t"
        "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%1], %2, %6, %10, first;\n\t"
        "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%1], %3, %7, %10, rest;\n\t"
        "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%1], %4, %8, %10, rest;\n\t"
        "@p tcgen05.mma.cta_group::2.kind::f8f6f4 [%1], %5, %9, %10, rest;\n\t"
        "@p tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%11], %12;\n\t}" ::"r"(leader), "r"(tmem_d), "l"(a), "l"(a + 2),
        "l"(a + 4), "l"(a + 6), "l"(b), "l"(b + 2), "l"(b + 4), "l"(b + 6), "r"(idesc), "r"(smem_u32(done)), "h"(static_cast<unsigned short>(3))
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, first, rest;\n\t"
        "setp.ne.b32 p, %0, 0;\n\t"
        "setp.ne.b32 first, 0, 0;\n\t"
        "setp.eq.b32 rest, 0, 0;\n\t"
        "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %2, %6, %10, first;\n\t"
        "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %3, %7, %10, rest;\n\t"
        "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %4, %8, %10, rest;\n\t"
        "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %5, %9, %10, rest;\n\t"
        "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%11];\n\t}" ::"r"(leader), "r"(tmem_d), "l"(a), "l"(a + 2),
        "l"(a + 4), "l"(a + 6), "l"(b), "l"(b + 2), "l"(b + 4), "l"(b + 6), "r"(idesc), "r"(smem_u32(done))
        : "memory");
  }
}
SPECB200_DEVINL uint32_t elect_leader() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
  return r;
}

// Bounded wait of a whole warp for a phase of one barrier, or of two: every lane polls (no broadcast
// on the fast path) and all take the same way out. Gives up as mbar_wait_bounded does. kFront: the warp may
// stand beside the kernel in front, for any time. No operand is loaded before that one has ended, so the
// limit begins anew at that end (griddepcontrol.wait ahead of the first wait did the same, but 5 x 2048 x
// 2048 took 3.93 us with it and 3.78 without).
template <bool kTwo, bool kFront = false>
SPECB200_DEVINL bool wait_warp(uint64_t* bar, uint32_t parity, uint64_t* bar2, uint32_t parity2, int32_t* status,
                               volatile int* abort) {
  auto ready = [&] {
    const bool a = mbar_try_wait(bar, parity), b = !kTwo || mbar_try_wait(bar2, parity2);
    return __all_sync(0xffffffffu, a && b) != 0;
  };
  if (ready()) return true;
  long long start = clock64();
  bool front = kFront;
  while (true) {
    if (ready()) return true;
    const bool late = clock64() - start > SPECB200_SPIN_LIMIT_CYCLES;
    if (kFront && __any_sync(0xffffffffu, front && late)) {
      pdl_wait();
      front = false;
      start = clock64();
      continue;
    }
    if (late) {
      set_status(status, SPECB200_ERR_TIMEOUT);
      *abort = 1;
    }
    if (__any_sync(0xffffffffu, late || *abort)) return false;
  }
}
SPECB200_DEVINL bool wait_warp(uint64_t* bar, uint32_t parity, int32_t* status, volatile int* abort) {
  return wait_warp<false>(bar, parity, nullptr, 0, status, abort);
}

// Instruction descriptor, kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), e4m3 A and B (bits 7-9
// and 10-12 = 0), both K-major, N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

template <int kN>
SPECB200_DEVINL void tmem_ld(uint32_t taddr, uint32_t (&r)[kN]);
template <>
SPECB200_DEVINL void tmem_ld<32>(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

template <>
SPECB200_DEVINL void tmem_ld<16>(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

SPECB200_DEVINL void cluster_arrive_wait() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
SPECB200_DEVINL uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
SPECB200_DEVINL uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
SPECB200_DEVINL void mbar_arrive_cluster_if(bool cond, uint32_t addr) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(addr),
      "r"(static_cast<int>(cond))
      : "memory");
}
// A load into this CTA's memory that completes on a barrier of the CTA pair's first CTA.
SPECB200_DEVINL void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
template <bool kPair>
SPECB200_DEVINL void f8_tmem_alloc(uint32_t* holder, uint32_t cols) {
  if constexpr (kPair) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(holder, cols);
    tmem_relinquish();
  }
}
template <bool kPair>
SPECB200_DEVINL void f8_tmem_dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (kPair)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
  else
    tmem_dealloc(taddr, cols);
}
SPECB200_DEVINL float4 ld_cluster_f4(uint32_t addr, uint32_t rank) {
  const uint32_t r = cluster_addr(addr, rank);
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(r)
               : "memory");
  return v;
}

// Four consecutive outputs of one token, `valid` of them inside the row.
SPECB200_DEVINL void store_quad(const F8Args& a, int64_t at, int valid, const float (&v)[4]) {
  if (a.out_f32) {
    float* p = static_cast<float*>(a.y) + at;
    if (a.rows16 && valid >= 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = v[i];
    return;
  }
  __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.y) + at;
  if (a.rows16 && valid >= 4) {
    const __nv_bfloat162 b0 = __floats2bfloat162_rn(v[0], v[1]), b1 = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < valid) p[i] = __float2bfloat16_rn(v[i]);
}

// Two fp32 accumulators in a register pair: d += {t0, t1} * f in one instruction.
typedef unsigned long long f32x2;
SPECB200_DEVINL void add2(f32x2& d, uint32_t t0, uint32_t t1, float f) {
  asm("{\n\t.reg .b64 t, g;\n\tmov.b64 t, {%1, %2};\n\tmov.b64 g, {%3, %3};\n\tfma.rn.f32x2 %0, t, g, %0;\n\t}"
      : "+l"(d)
      : "r"(t0), "r"(t1), "f"(f));
}

// Four bytes to shared memory, and an arrival at `bar` once this thread's copies so far are there.
SPECB200_DEVINL void copy_async_4(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
SPECB200_DEVINL void copy_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A weight tile to L2. It stays coherent there, so this may run before the kernel in front has ended,
// even if that kernel is still writing the weights.
SPECB200_DEVINL void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0),
               "r"(c1)
               : "memory");
}
SPECB200_DEVINL void tma_store_2d(const CUtensorMap* map, const void* smem_src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1)
               : "memory");
}

// NaN for 32 tokens of a warp's features that it could not finish because a wait gave up, so that the caller sees
// it without a status word too. (NaN in the sums on the way of the ordinary stores cost every call of the
// small kernel 0.15 us.)
constexpr uint32_t kF8Nan = 0x7fffffffu;
SPECB200_DEVINL void give_up_outputs(const F8Args& a, int m0, int n0, int cols, int lane) {
  const int rows = min(32, a.M - m0), end = min(n0 + cols, a.N);
  for (int r = 0; r < rows; ++r) {
    const int64_t at = static_cast<int64_t>(m0 + r) * a.ldy;
    for (int n = n0 + lane; n < end; n += 32) {
      if (a.out_f32)
        static_cast<uint32_t*>(a.y)[at + n] = kF8Nan;
      else
        static_cast<unsigned short*>(a.y)[at + n] = static_cast<unsigned short>(kF8Nan >> 16);
    }
  }
}

// One warp's 32 tokens x kCols features to memory through kPieces pieces of shared memory, a piece
// being 128 bytes per row (64 bf16 or 32 fp32 features). The 16-byte units of a row are swizzled by
// the row (the 128-byte swizzle TMA reads), so that neither side has bank conflicts. TMA stores
// leave the warp free while the pieces drain; what lies off the 16-byte boundaries is written by the
// warp itself.
template <typename T, int kPieces, int kCols>
SPECB200_DEVINL void store_warp_tile(const F8Args& a, const CUtensorMap& y_map, const float (&acc)[kCols],
                                     uint8_t* bufs, int m0, int n0, int lane) {
  constexpr int kUnit = 16 / sizeof(T), kPiece = 8 * kUnit;
  constexpr int kRound = kPieces * kPiece < kCols ? kPieces * kPiece : kCols;
#pragma unroll
  for (int c0 = 0; c0 < kCols; c0 += kRound) {
    if (a.rows16) {  // what lay in the buffers has been read
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
    }
#pragma unroll
    for (int c = c0; c < c0 + kRound; c += kUnit) {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(acc[c + 2 * j], acc[c + 2 * j + 1]);
          v[j] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          v[j] = __float_as_uint(acc[c + j]);
        }
      }
      const int piece = (c - c0) / kPiece, unit = (c - c0) % kPiece / kUnit;
      *reinterpret_cast<uint4*>(bufs + piece * kF8OutPiece + lane * 128 + ((unit ^ lane) & 7) * 16) =
          make_uint4(v[0], v[1], v[2], v[3]);
    }
    // a piece that the row's end cuts off its 16-byte grid is not TMA's: it would fill the last unit
    auto by_tma = [&](int c) { return a.rows16 && (a.tail16 || n0 + c + kPiece <= a.N); };
    if (a.rows16) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (a.rows16 && lane == 0) {
#pragma unroll
      for (int c = c0; c < c0 + kRound; c += kPiece)
        if (n0 + c < a.N && by_tma(c)) tma_store_2d(&y_map, bufs + (c - c0) / kPiece * kF8OutPiece, n0 + c, m0);
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    for (int c = c0; c < c0 + kRound; c += kPiece) {
      if (by_tma(c)) continue;
      // A row at a time, four bytes per lane: one element, or the pair that starts on a 4-byte boundary.
      // 4096 x 8190 x 64: 39 us (an element per store 123, eight bytes per lane with the rows' ends in
      // smaller pieces 42, fp32 49 and 57).
      const int rows = min(32, a.M - m0), left = a.N - n0 - c;
      const uint8_t* piece = bufs + (c - c0) / kPiece * kF8OutPiece + (lane & 3) * 4;
      T* y = static_cast<T*>(a.y) + static_cast<int64_t>(m0) * a.ldy + n0 + c;
#pragma unroll 16
      for (int r = 0; r < rows; ++r, y += a.ldy) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(piece + r * 128 + (((lane >> 2) ^ r) & 7) * 16);
        if constexpr (sizeof(T) == 4) {
          if (lane < left) y[lane] = __uint_as_float(w);
        } else {
          const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(y) >> 1) & 1, n = 2 * lane + odd;
          const uint32_t next = __shfl_down_sync(0xffffffffu, w, 1);
          unsigned short* o = reinterpret_cast<unsigned short*>(y);
          if (n + 1 < min(left, kPiece))
            *reinterpret_cast<uint32_t*>(o + n) = odd ? (w >> 16) | (next << 16) : w;
          else if (n < left)
            o[n] = static_cast<unsigned short>(odd ? w >> 16 : w);
          if (odd && lane == 0 && left > 0) o[0] = static_cast<unsigned short>(w);
        }
      }
    }
    __syncwarp();
  }
}

// Adds the partial tiles of a cluster's CTAs in split order, each CTA its share of the outputs:
// `rows` rows of 128 features with a pitch of 132 floats, at the same address in every CTA.
SPECB200_DEVINL void add_split_tiles(const F8Args& a, uint32_t tile, int m0, int n0, int rows, int split, int threads) {
  constexpr int kQuads = kF8Block / 4, kPitch = kF8Block + 4;
  for (int i = split * threads + threadIdx.x; i < rows * kQuads; i += a.splits * threads) {
    const int r = i / kQuads, c = (i % kQuads) * 4;
    if (n0 + c >= a.N) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    float4 q[kF8MaxSplits];  // all splits' loads in flight
#pragma unroll
    for (int p = 0; p < kF8MaxSplits; ++p)
      if (p < a.splits) q[p] = ld_cluster_f4(tile + (r * kPitch + c) * 4, p);
#pragma unroll
    for (int p = 0; p < kF8MaxSplits; ++p)
      if (p < a.splits) { v[0] += q[p].x; v[1] += q[p].y; v[2] += q[p].z; v[3] += q[p].w; }
    store_quad(a, static_cast<int64_t>(m0 + r) * a.ldy + n0 + c, a.N - n0 - c, v);
  }
}

// ------------------------------------------------------------------------------ small tiles
// The scales of one group: of a CTA's 128 tokens and of the tile's weight blocks (two for a pair).
struct alignas(16) F8Scales {
  float x[kF8TileM], w[4];
};
struct alignas(16) F8SmallBarriers {
  uint64_t full[kF8MaxStages], done[kF8MaxStages], sfull[kF8MaxStages + 4], tempty[4];
  uint32_t tmem_holder;
  int abort_flag;
};

// One warp's copy of a group's scales to shared memory; `filled` (32 arrivals) completes when they
// are there. sx, sw: this lane's first token's and weight block's scale of the group.
SPECB200_DEVINL void copy_scales(F8Scales& to, uint64_t* filled, const float* sx, const float* sw, int64_t pitch32,
                                 int tokens, bool live_w, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (32 * i + lane < tokens) copy_async_4(&to.x[32 * i + lane], sx + i * pitch32);
  if (live_w) copy_async_4(&to.w[lane], sw);
  copy_async_arrive(filled);
}

// Warps 0-7 read back (w on TMEM lane quarter w % 4, columns 64 (w / 4)..), warp 8 (and 10) loads
// operands and scales, warp 9 issues tcgen05.mma. A stage's `done` barrier frees its operands and completes its
// accumulator. Small calls are bound by latency, so loads start before TMEM is allocated: the
// epilogue learns of the allocation through the first `done`.
template <int kPerSm>
__global__ void __launch_bounds__(f8_small_threads(kPerSm), kPerSm)
    gemm_fp8_small_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                          const __grid_constant__ CUtensorMap y_map, F8Args a) {
  constexpr int kCols = 64;                  // features per epilogue thread
  constexpr int kThreads = f8_small_threads(kPerSm), kBufs = f8_small_bufs(kPerSm);
  constexpr int kProducers = kPerSm == 1 ? 2 : 1;
  constexpr int kLd = kPerSm == 1 ? 32 : 16; // accumulator columns read back at a time (what registers allow)
  constexpr int kPitch = kF8Block + 4;       // partial tile's row pitch (floats)
  // the ring (1024-byte swizzle atoms), which ends up holding the output; barriers; scales
  extern __shared__ __align__(1024) uint8_t smem[];
  F8SmallBarriers& bars = *reinterpret_cast<F8SmallBarriers*>(smem + a.ring_bytes);
  F8Scales* scales = reinterpret_cast<F8Scales*>(&bars + 1);  // stages + kBufs of them
  uint64_t *full = bars.full, *done = bars.done, *sfull = bars.sfull, *tempty = bars.tempty;
  int& abort_flag = bars.abort_flag;
  const uint32_t stage_bytes = kF8TileBytes + a.x_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t stages = a.stages;

  // one barrier per thread: one after another they took half a microsecond
  if (threadIdx.x < stages + kBufs) {
    const uint32_t i = threadIdx.x;
    if (i < stages) {
      mbar_init(&full[i], 1);
      mbar_init(&done[i], 1);
    }
    mbar_init(&sfull[i], 32);
    if (i < kBufs) mbar_init(&tempty[i], kF8EpiWarps);
    if (i == 0) abort_flag = 0;
    fence_mbar_init();
  } else if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
  }
  __syncthreads();

  // a cluster is one tile, its CTAs the splits of K
  const int splits = a.splits, split = static_cast<int>(blockIdx.x) % splits, tile = static_cast<int>(blockIdx.x) / splits;
  const int tile_m = tile % a.m_tiles * kF8TileM, tile_n = tile / a.m_tiles * kF8Block;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.kblocks) * split / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.kblocks) * (split + 1) / splits);

  if (warp == 8 || warp == 10) {
    // One lane loads a group's operands by TMA, all lanes copy its scales; two producers take turns
    // (one takes about 700 cycles per group to issue it all).
    if (lane == 0)
      for (int kb = kb0 + (kProducers > 1 && warp != 8); kb < min(kb1, kb0 + kF8Ahead); kb += kProducers)
        tma_prefetch_2d(&w_map, kb * kFp8Group, tile_n);
    pdl_wait();
    const float* sx = a.xs + static_cast<int64_t>(tile_m + lane) * a.kblocks + kb0;
    const float* sw = a.ws + static_cast<int64_t>(tile_n / kF8Block) * a.kblocks + kb0;
    const int64_t pitch32 = static_cast<int64_t>(32) * a.kblocks;
    const int tokens = a.M - tile_m, groups = a.starved ? 0 : kb1 - kb0, me = warp == 8 ? 0 : 1;
    auto load = [&](int g, uint32_t st) {
      if (lane == 0) {
        uint8_t* s = smem + st * stage_bytes;
        mbar_arrive_expect_tx(&full[st], stage_bytes);
        tma_load_2d(s, &w_map, &full[st], (kb0 + g) * kFp8Group, tile_n);
        tma_load_2d(s + kF8TileBytes, &x_map, &full[st], (kb0 + g) * kFp8Group, tile_m);
      }
      __syncwarp();
    };
    auto fetch = [&](int g, uint32_t slot) {
      copy_scales(scales[slot], &sfull[slot], sx + g, sw + g, pitch32, tokens, lane == 0, lane);
    };
    // The ring's first filling waits for nothing: operands first, then their scales. Scales have
    // kBufs slots more than there are stages: when a stage is done, so are the MMAs that waited for
    // the epilogue to read the slot that comes next. No barrier can run two phases ahead of a wait for
    // it, as there are at least kBufs stages.
    const int first = min(groups, static_cast<int>(stages));
    for (int g = me; g < first; g += kProducers) load(g, g);
    for (int g = me; g < first; g += kProducers) fetch(g, g);
    uint32_t st = 0, phase = 0, slot = stages;
    for (int g = first; g < groups; ++g) {
      if (kProducers == 1 || g % kProducers == me) {
        if (!wait_warp(&done[st], phase, a.status, &abort_flag)) {
          // gave up: this warp's copies in flight get their time to land
          for (int i = max(0, g - static_cast<int>(stages)); i < g; ++i)
            if (lane == 0 && i % kProducers == me)
              mbar_wait_bounded(&full[i % stages], (i / stages) & 1, a.status, nullptr);
          break;
        }
        load(g, st);
        fetch(g, slot);
      }
      if (++st == stages) { st = 0; phase ^= 1; }
      if (++slot == stages + kBufs) slot = 0;
    }
    __syncwarp();
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 9) {
    f8_tmem_alloc<false>(&bars.tmem_holder, kBufs * kF8Block);
    tc_fence_before();
    __syncwarp();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_holder);
    // Only from here on may the next kernel's CTAs start: one that allocated TMEM before this CTA and then
    // waited for it would keep it from ever starting. The first thread that allows it does so for the
    // whole CTA, so no other warp does.
    pdl_launch_dependents();
    constexpr uint32_t idesc = umma_idesc_e4m3(kF8TileM, kF8Block);
    const uint32_t leader = elect_leader();
    const uint64_t dw0 = umma_desc_sw128(smem_u32(smem)), dx0 = umma_desc_sw128(smem_u32(smem + kF8TileBytes));
    uint32_t st = 0, phase = 0, buf = 0, acc_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!wait_warp<true, true>(&tempty[buf], acc_phase ^ 1, &full[st], phase, a.status, &abort_flag)) break;
      tc_fence_after();
      const uint64_t at = static_cast<uint64_t>(st * (stage_bytes >> 4));
      umma_group_e4m3<false>(leader, tmem + buf * kF8Block, dx0 + at, dw0 + at, idesc, &done[st]);
      if (++st == stages) { st = 0; phase ^= 1; }
      if (++buf == kBufs) { buf = 0; acc_phase ^= 1; }
    }
  } else {
    pdl_wait();
    const int quarter = warp & 3, col0 = (warp >> 2) * kCols;
    const int m0 = tile_m + quarter * 32, n0 = tile_n + col0;
    const bool live = m0 < a.M && n0 < a.N;  // warps without outputs only keep step
    float acc[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
    uint32_t st = 0, phase = 0, buf = 0, slot = 0, slot_phase = 0;
    // A poll (`tried`) is issued early, its outcome looked at (`ready`) where it is needed.
    auto try_ready = [&] { return mbar_try_wait(&done[st], phase) && mbar_try_wait(&sfull[slot], slot_phase); };
    auto ready = [&](bool tried) {
      const bool ok = __all_sync(0xffffffffu, tried) ||
                      wait_warp<true>(&done[st], phase, &sfull[slot], slot_phase, a.status, &abort_flag);
      tc_fence_after();
      return ok;
    };
    auto release = [&](uint32_t b) {  // this buffer is read: a later group may overwrite it
      tc_fence_before();
      if (lane == 0) mbar_arrive(&tempty[b]);
    };
    auto advance = [&] {
      if (++st == stages) { st = 0; phase ^= 1; }
      if (++slot == stages + kBufs) { slot = 0; slot_phase ^= 1; }
      if (++buf == kBufs) buf = 0;
    };
    auto factor = [&] { return scales[slot].x[quarter * 32 + lane] * scales[slot].w[0]; };
    bool ok = ready(try_ready());
    const uint32_t tbase = ok ? *reinterpret_cast<volatile uint32_t*>(&bars.tmem_holder) + (static_cast<uint32_t>(quarter * 32) << 16) + col0 : 0;
    int groups = kb1 - kb0;
    if (!live) {
      while (ok) {
        release(buf);
        advance();
        if (--groups == 0) break;
        ok = ready(try_ready());
      }
    } else if constexpr (kPerSm == 1) {
      // 32 columns come back at a time, the next ones and the next group's poll on their way while
      // the last ones are added.
      uint32_t r0[32], r1[32];
      auto add = [&](int c, const uint32_t (&r)[32], float f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(__uint_as_float(r[i]), f, acc[c + i]);
      };
      if (ok) {
        float f = factor();
        tmem_ld<32>(tbase + buf * kF8Block, r0);
        for (;;) {
          tmem_ld_wait();
          tmem_ld<32>(tbase + buf * kF8Block + 32, r1);
          const uint32_t last = buf;
          advance();
          const bool more = --groups > 0, tried = more && try_ready();
          add(0, r0, f);
          tmem_ld_wait();
          release(last);
          if (!more) {
            add(32, r1, f);
            break;
          }
          ok = ready(tried);
          if (!ok) break;
          tmem_ld<32>(tbase + buf * kF8Block, r0);
          const float f1 = factor();
          add(32, r1, f);
          f = f1;
        }
      }
    } else {
      while (ok) {
        const float f = factor();
#pragma unroll
        for (int c = 0; c < kCols; c += kLd) {
          uint32_t r[kLd];
          tmem_ld<kLd>(tbase + buf * kF8Block + c, r);
          tmem_ld_wait();
          if (c + kLd == kCols) release(buf);
#pragma unroll
          for (int i = 0; i < kLd; ++i) acc[c + i] = fmaf(__uint_as_float(r[i]), f, acc[c + i]);
        }
        advance();
        if (--groups == 0) break;
        ok = ready(try_ready());
      }
    }
    // every group is done: the ring is idle and takes the output, or this split's partial tile
    if (ok && live) {
      if (splits > 1) {
        float* p = reinterpret_cast<float*>(smem) + (quarter * 32 + lane) * kPitch + col0;
        if (m0 + lane < a.M) {
#pragma unroll
          for (int i = 0; i < kCols; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        }
      } else if (a.out_f32) {
        store_warp_tile<float, 1>(a, y_map, acc, smem + warp * kF8OutPiece, m0, n0, lane);
      } else {
        store_warp_tile<__nv_bfloat16, 1>(a, y_map, acc, smem + warp * kF8OutPiece, m0, n0, lane);
      }
    } else if (live && splits > 1) {
      for (int i = 0; i < kCols && m0 + lane < a.M; ++i)
        reinterpret_cast<uint32_t*>(smem)[(quarter * 32 + lane) * kPitch + col0 + i] = kF8Nan;
    } else if (live) {
      give_up_outputs(a, m0, n0, kCols, lane);
    }
    if (a.rows16 && splits == 1 && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
  __syncwarp();
  if (splits > 1) {
    cluster_arrive_wait();
    add_split_tiles(a, smem_u32(smem), tile_m, tile_n, min(kF8TileM, a.M - tile_m), split, kThreads);
    cluster_arrive_wait();  // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    f8_tmem_dealloc<false>(*reinterpret_cast<volatile uint32_t*>(&bars.tmem_holder), kBufs * kF8Block);
  }
}

// ------------------------------------------------------------------------------ few tokens
constexpr int kF8FewTokens = 16;  // the least N of an MMA with M = 128
constexpr int kF8FewThreads = 352;
constexpr int kF8FewBufs = 4;
struct alignas(16) F8FewBarriers {
  uint64_t full[kF8MaxStages], done[kF8MaxStages], sfull[kF8MaxStages + kF8FewBufs], tempty[kF8FewBufs];
  uint32_t tmem_holder;
  int abort_flag;
};

// Up to 16 tokens: decode and verify steps, bound by the stream of weights and by latency. Here
// the 128 features lie on the TMEM lanes and the tokens are the MMA's N, so that a group costs half the
// tensor time and every epilogue warp has work: warps 0-3 read the even groups and warps 4-7 the odd
// ones (w on lane quarter w % 4; a thread owns one feature and all tokens), and their sums meet in
// shared memory at the end. Producers, MMA warp and the exchange between splits of K are those of the
// small kernel. 5 x 16384 x 2048 8.0 us (9.2 with the tokens on the lanes), 1 x 6144 x 2048 5.2 (6.3),
// 5 x 2048 x 8192 6.7 (8.0): 2.4-4.2 TB/s of weights, the rest is the way from launch to the first
// operands (about 2 us) and from the last ones to the output.
__global__ void __launch_bounds__(kF8FewThreads, 2)
    gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, F8Args a) {
  constexpr int kTok = kF8FewTokens, kBufs = kF8FewBufs, kProducers = 2;
  constexpr int kPitch = kF8Block + 4;  // row pitch (floats) of the tile where the sums meet
  constexpr uint32_t kStageBytes = kF8TileBytes + kTok * kFp8Group;
  // the ring (1024-byte swizzle atoms), the sums' tile, barriers, scales
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t stages = a.stages;
  float* sums = reinterpret_cast<float*>(smem + stages * kStageBytes);
  F8FewBarriers& bars = *reinterpret_cast<F8FewBarriers*>(sums + kTok * kPitch);
  F8Scales* scales = reinterpret_cast<F8Scales*>(&bars + 1);  // stages + kBufs of them
  uint64_t *full = bars.full, *done = bars.done, *sfull = bars.sfull, *tempty = bars.tempty;
  int& abort_flag = bars.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x < stages + kBufs) {
    const uint32_t i = threadIdx.x;
    if (i < stages) {
      mbar_init(&full[i], 1);
      mbar_init(&done[i], 1);
    }
    mbar_init(&sfull[i], 32);
    if (i < kBufs) mbar_init(&tempty[i], 4);
    if (i == 0) abort_flag = 0;
    fence_mbar_init();
  } else if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&w_map);
    tma_prefetch_desc(&x_map);
  }
  __syncthreads();

  const int splits = a.splits, split = static_cast<int>(blockIdx.x) % splits;
  const int tile_n = static_cast<int>(blockIdx.x) / splits * kF8Block;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.kblocks) * split / splits);
  const int groups = static_cast<int>(static_cast<int64_t>(a.kblocks) * (split + 1) / splits) - kb0;

  if (warp == 8 || warp == 10) {
    if (lane == 0)
      for (int g = warp == 8 ? 0 : 1; g < min(groups, kF8Ahead); g += kProducers) tma_prefetch_2d(&w_map, (kb0 + g) * kFp8Group, tile_n);
    pdl_wait();
    const float* sx = a.xs + static_cast<int64_t>(lane) * a.kblocks + kb0;
    const float* sw = a.ws + static_cast<int64_t>(tile_n / kF8Block) * a.kblocks + kb0;
    const int me = warp == 8 ? 0 : 1;
    auto load = [&](int g, uint32_t st) {
      if (lane == 0) {
        uint8_t* s = smem + st * kStageBytes;
        mbar_arrive_expect_tx(&full[st], kStageBytes);
        tma_load_2d(s, &w_map, &full[st], (kb0 + g) * kFp8Group, tile_n);
        tma_load_2d(s + kF8TileBytes, &x_map, &full[st], (kb0 + g) * kFp8Group, 0);
      }
      __syncwarp();
    };
    auto fetch = [&](int g, uint32_t slot) {
      if (lane < a.M) copy_async_4(&scales[slot].x[lane], sx + g);
      if (lane == 0) copy_async_4(&scales[slot].w[0], sw + g);
      copy_async_arrive(&sfull[slot]);
    };
    // as in the small kernel
    const int loads = a.starved ? 0 : groups, first = min(loads, static_cast<int>(stages));
    for (int g = me; g < first; g += kProducers) load(g, g);
    for (int g = me; g < first; g += kProducers) fetch(g, g);
    uint32_t st = 0, phase = 0, slot = stages;
    for (int g = first; g < loads; ++g) {
      if (g % kProducers == me) {
        if (!wait_warp(&done[st], phase, a.status, &abort_flag)) {
          for (int i = max(0, g - static_cast<int>(stages)); i < g; ++i)
            if (lane == 0 && i % kProducers == me)
              mbar_wait_bounded(&full[i % stages], (i / stages) & 1, a.status, nullptr);
          break;
        }
        load(g, st);
        fetch(g, slot);
      }
      if (++st == stages) { st = 0; phase ^= 1; }
      if (++slot == stages + kBufs) slot = 0;
    }
    __syncwarp();
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 9) {
    f8_tmem_alloc<false>(&bars.tmem_holder, kBufs * kTok);
    tc_fence_before();
    __syncwarp();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_holder);
    pdl_launch_dependents();  // as in the small kernel, after the allocation
    constexpr uint32_t idesc = umma_idesc_e4m3(kF8Block, kTok);
    const uint32_t leader = elect_leader();
    const uint64_t dw0 = umma_desc_sw128(smem_u32(smem)), dx0 = umma_desc_sw128(smem_u32(smem + kF8TileBytes));
    uint32_t st = 0, phase = 0, buf = 0, acc_phase = 0;
    for (int g = 0; g < groups; ++g) {
      if (!wait_warp<true, true>(&tempty[buf], acc_phase ^ 1, &full[st], phase, a.status, &abort_flag)) break;
      tc_fence_after();
      const uint64_t at = static_cast<uint64_t>(st * (kStageBytes >> 4));
      umma_group_e4m3<false>(leader, tmem + buf * kTok, dw0 + at, dx0 + at, idesc, &done[st]);
      if (++st == stages) { st = 0; phase ^= 1; }
      if (++buf == kBufs) { buf = 0; acc_phase ^= 1; }
    }
  } else {
    pdl_wait();
    const int quarter = warp & 3, odd = warp >> 2, feature = quarter * 32 + lane;
    float acc[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) acc[i] = 0.f;
    uint32_t st = odd, phase = 0, slot = odd, slot_phase = 0, buf = odd, tbase = 0;
    bool ok = true;
    for (int g = odd; g < groups; g += 2) {
      ok = wait_warp<true>(&done[st], phase, &sfull[slot], slot_phase, a.status, &abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (g == odd) tbase = *reinterpret_cast<volatile uint32_t*>(&bars.tmem_holder) + (static_cast<uint32_t>(quarter * 32) << 16);
      const F8Scales& sc = scales[slot];
      const float w = sc.w[0];
      uint32_t r[kTok];
      tmem_ld<kTok>(tbase + buf * kTok, r);
      float f[kTok];
#pragma unroll
      for (int i = 0; i < kTok; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(&sc.x[i]);
        f[i] = x.x * w; f[i + 1] = x.y * w; f[i + 2] = x.z * w; f[i + 3] = x.w * w;
      }
      tmem_ld_wait();
      tc_fence_before();  // read: a later group may overwrite it
      if (lane == 0) mbar_arrive(&tempty[buf]);
#pragma unroll
      for (int i = 0; i < kTok; ++i) acc[i] = fmaf(__uint_as_float(r[i]), f[i], acc[i]);
      st += 2;
      if (st >= stages) { st -= stages; phase ^= 1; }
      slot += 2;
      if (slot >= stages + kBufs) { slot -= stages + kBufs; slot_phase ^= 1; }
      buf ^= 2;
    }
    if (!ok) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) acc[i] = __uint_as_float(kF8Nan);
    }
    // the odd groups' sums to shared memory, the even groups' added to them
    if (odd) {
#pragma unroll
      for (int i = 0; i < kTok; ++i)
        if (i < a.M) sums[i * kPitch + feature] = acc[i];
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (!odd) {
      const int n = tile_n + feature;
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        if (i >= a.M) break;
        const float v = acc[i] + sums[i * kPitch + feature];
        if (splits > 1)
          sums[i * kPitch + feature] = v;
        else if (n < a.N && a.out_f32)
          static_cast<float*>(a.y)[static_cast<int64_t>(i) * a.ldy + n] = v;
        else if (n < a.N)
          static_cast<__nv_bfloat16*>(a.y)[static_cast<int64_t>(i) * a.ldy + n] = __float2bfloat16_rn(v);
      }
    }
  }
  __syncwarp();
  if (splits > 1) {
    cluster_arrive_wait();
    add_split_tiles(a, smem_u32(sums), 0, tile_n, a.M, split, kF8FewThreads);
    cluster_arrive_wait();  // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    f8_tmem_dealloc<false>(*reinterpret_cast<volatile uint32_t*>(&bars.tmem_holder), kBufs * kTok);
  }
}

// ------------------------------------------------------------------------------ CTA pairs
constexpr int kF8Slots = kF8PairStages + 2;
struct F8PairBarriers {
  uint64_t full[kF8PairStages], done[2][kF8PairStages], sfull[kF8Slots], tempty[2][2];
  uint32_t tmem_holder;
  int abort_flag;
  F8Scales scales[kF8Slots];
};
constexpr int kF8PairPieces = 2;  // per epilogue warp: its whole bf16 tile
constexpr size_t kF8PairOut = static_cast<size_t>(kF8EpiWarps) * kF8PairPieces * kF8OutPiece;
constexpr size_t kF8PairSmem = kF8PairOut + kF8PairStages * 2 * kF8TileBytes + sizeof(F8PairBarriers);
static_assert(kF8PairSmem <= 227 * 1024, "shared memory of a CTA");

// The tiles of one CTA pair, every (gridDim / 2)-th of the token-major list, without a division per tile.
struct F8TileWalk {
  int m, n, m_tiles, n_tiles, dm, dn;
  SPECB200_DEVINL explicit F8TileWalk(const F8Args& a) : m_tiles(a.m_tiles), n_tiles(a.n_tiles) {
    const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;
    m = first % m_tiles;
    n = first / m_tiles;
    dm = step % m_tiles;
    dn = step / m_tiles;
  }
  SPECB200_DEVINL bool more() const { return n < n_tiles; }
  SPECB200_DEVINL void next() {
    m += dm;
    n += dn;
    if (m >= m_tiles) {
      m -= m_tiles;
      ++n;
    }
  }
  SPECB200_DEVINL int token0(int rank) const { return (2 * m + rank) * kF8TileM; }
  SPECB200_DEVINL int feature0() const { return n * 2 * kF8Block; }
};

// A group's 256 features are multiplied in two halves with a TMEM buffer each (two groups' worth in
// all): half h holds features 64 h..64 h + 63 of either weight block, so that each epilogue thread reads 64
// columns of a half. What a buffer costs besides its MMAs -- the commit's and the release's way
// between warps and CTAs, the read -- then hides behind three other buffers' MMAs; with one buffer per group it
// did not (8192 x 16384 x 2048: 266 us against 286; 245 in the end).
// Warps 0-7 read back (w on TMEM lane quarter w % 4, weight block w / 4), warps 9
// and 10 of the pair's first CTA tcgen05.mma for both; warps 8 and 11 load operands and scales. Either
// kind takes turns: MMAs issue in order and block the warp while the tensor cores are busy, and a
// load of operands and scales takes its warp longer to issue than the MMAs of a group run.
__global__ void __launch_bounds__(kF8PairThreads, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                         const __grid_constant__ CUtensorMap y_map, F8Args a) {
  constexpr int kCols = 128, kLd = 32;  // features per epilogue thread; columns read back at a time
  constexpr uint32_t kStageBytes = 2 * kF8TileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + kF8PairOut;
  F8PairBarriers& bars = *reinterpret_cast<F8PairBarriers*>(ring + kF8PairStages * kStageBytes);
  int& abort_flag = bars.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x < kF8Slots) {
    const int i = threadIdx.x;
    if (i < kF8PairStages) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.done[0][i], 1);
      mbar_init(&bars.done[1][i], 1);
    }
    mbar_init(&bars.sfull[i], 32);
    if (i < 4) mbar_init(&bars.tempty[i >> 1][i & 1], 2 * kF8EpiWarps);
    if (i == 0) abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) f8_tmem_alloc<true>(&bars.tmem_holder, 512);
  tc_fence_before();
  __syncwarp();
  cluster_arrive_wait();  // the peer's barriers are ready, too
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_holder;
  pdl_launch_dependents();  // as in the small kernel, after the allocation

  const int rank = static_cast<int>(cluster_rank());
  const int kblocks = a.kblocks;

  // 384 threads start with 168 registers each, 64,512; the shares below sum to 7,168 + 57,344.
  if (warp >= kF8EpiWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8 || warp == 11) {
      // Every other group each: one lane loads the operands by TMA, all lanes copy the scales, into a
      // ring of two slots more than there are stages. Once the stage of group g is done, the
      // epilogue has read the scales of group g - 2 (the MMAs of g waited for that), whose slot and
      // barrier come next. No barrier can run two phases ahead of a wait for it: the MMAs of a
      // stage's next group wait for loads that follow the wait for its last one.
      if (lane == 0) {
        tma_prefetch_desc(&w_map);
        tma_prefetch_desc(&x_map);
      }
      pdl_wait();
      const bool odd = warp == 11;
      const int64_t pitch = static_cast<int64_t>(32) * kblocks;
      uint32_t st = 0, phase = 0, slot = 0, last = 0, last_phase = 0;
      bool ok = true, mine = !odd, any = false;
      for (F8TileWalk tile(a); tile.more() && ok && !a.starved; tile.next()) {
        const int m0 = tile.token0(rank), n0 = tile.feature0(), block = 2 * tile.n + lane;
        const float* sx = a.xs + static_cast<int64_t>(m0 + lane) * kblocks;
        const float* sw = a.ws + static_cast<int64_t>(block) * kblocks;
        const bool live_w = lane < 2 && block * kF8Block < a.N;
        for (int kb = 0; kb < kblocks; ++kb, mine = !mine) {
          if (mine) {
            ok = wait_warp(&bars.done[1][st], phase ^ 1, a.status, &abort_flag);
            if (!ok) break;
            if (lane == 0) {
              uint8_t* s = ring + st * kStageBytes;
              if (rank == 0) mbar_arrive_expect_tx(&bars.full[st], 2 * kStageBytes);  // both CTAs' loads
              const uint32_t bar = cluster_addr(smem_u32(&bars.full[st]), 0);
              tma_load_2d_pair(s, &w_map, bar, kb * kFp8Group, n0 + rank * kF8Block);
              tma_load_2d_pair(s + kF8TileBytes, &x_map, bar, kb * kFp8Group, m0);
            }
            __syncwarp();
            copy_scales(bars.scales[slot], &bars.sfull[slot], sx + kb, sw + kb, pitch, a.M - m0, live_w, lane);
            any = true;
            last = st;
            last_phase = phase;
          }
          if (++st == kF8PairStages) { st = 0; phase ^= 1; }
          if (++slot == kF8Slots) slot = 0;
        }
      }
      // Tail: this warp's last group is done, and with it all earlier ones (so no commit arrives after
      // the exit), or, where a wait gave up, its copies in flight have had their time to land.
      if (any && ok) ok = wait_warp(&bars.done[1][last], last_phase, a.status, &abort_flag);
      if (any && !ok && lane == 0) mbar_wait_bounded(rank == 0 ? &bars.full[last] : &bars.done[1][last], last_phase, a.status, nullptr);
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (rank == 0) {  // warps 9 and 10: every other group each
      pdl_wait();  // the limit of the waits below is not spent on the kernel in front
      constexpr uint32_t idesc = umma_idesc_e4m3(2 * kF8TileM, kF8Block);
      const uint32_t leader = elect_leader();
      const uint64_t dw0 = umma_desc_sw128(smem_u32(ring)), dx0 = umma_desc_sw128(smem_u32(ring + kF8TileBytes));
      const uint32_t turn = static_cast<uint32_t>(warp - 9);
      uint32_t st = 0, phase = 0, buf = 0, acc_phase = 0;
      bool ok = true;
      for (F8TileWalk tile(a); tile.more() && ok; tile.next()) {
        for (int kb = 0; kb < kblocks; ++kb) {
          if (buf == turn) {
            const uint64_t at = static_cast<uint64_t>(st * (kStageBytes >> 4));
            ok = wait_warp<true>(&bars.tempty[buf][0], acc_phase ^ 1, &bars.full[st], phase, a.status, &abort_flag);
            if (!ok) break;
            tc_fence_after();
            umma_group_e4m3<true>(leader, tmem + buf * 256, dx0 + at, dw0 + at, idesc, &bars.done[0][st]);
            ok = wait_warp(&bars.tempty[buf][1], acc_phase ^ 1, a.status, &abort_flag);
            if (!ok) break;
            tc_fence_after();
            umma_group_e4m3<true>(leader, tmem + buf * 256 + kF8Block, dx0 + at, dw0 + at + (kF8TileBytes >> 5), idesc,
                                  &bars.done[1][st]);
          }
          if (++st == kF8PairStages) { st = 0; phase ^= 1; }
          buf ^= 1;
          acc_phase ^= buf ^ 1;
        }
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    pdl_wait();
    const int quarter = warp & 3, block = warp >> 2;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + block * 64;
    const uint32_t tempty0 = cluster_addr(smem_u32(bars.tempty), 0);  // the issuing CTA's
    uint8_t* out_buf = smem + warp * (kF8PairPieces * kF8OutPiece);
    uint32_t buf = 0, st = 0, phase = 0, slot = 0, slot_phase = 0;
    bool ok = true;
    // this half is read: the next but one group may overwrite it
    auto release = [&](int half) {
      tc_fence_before();
      mbar_arrive_cluster_if(lane == 0, tempty0 + (buf * 2 + half) * sizeof(uint64_t));
    };
    auto next_group = [&] {
      buf ^= 1;
      if (++st == kF8PairStages) { st = 0; phase ^= 1; }
      if (++slot == kF8Slots) { slot = 0; slot_phase ^= 1; }
    };
    // A poll (`try_`) is issued early, its outcome looked at (`ready`) where it is needed.
    auto try_first = [&] { return mbar_try_wait(&bars.done[0][st], phase) && mbar_try_wait(&bars.sfull[slot], slot_phase); };
    auto first_ready = [&](bool tried) {
      return __all_sync(0xffffffffu, tried) ||
             wait_warp<true>(&bars.done[0][st], phase, &bars.sfull[slot], slot_phase, a.status, &abort_flag);
    };
    auto try_second = [&] { return mbar_try_wait(&bars.done[1][st], phase); };
    auto second_ready = [&](bool tried) {
      return __all_sync(0xffffffffu, tried) || wait_warp(&bars.done[1][st], phase, a.status, &abort_flag);
    };
    auto factor = [&] { return bars.scales[slot].x[quarter * 32 + lane] * bars.scales[slot].w[block]; };
    for (F8TileWalk tile(a); tile.more() && ok; tile.next()) {
      const int m0 = tile.token0(rank) + quarter * 32, n0 = tile.feature0() + block * kF8Block;
      if (m0 >= a.M || n0 >= a.N) {  // a warp without outputs only keeps step
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = first_ready(false) && second_ready(false);
          if (!ok) break;
          release(0);
          release(1);
          next_group();
        }
        continue;
      }
      f32x2 acc2[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) acc2[i] = 0;
      // A half's 64 columns come back in two reads and are added once both are there, with the poll for the next
      // half on its way; no read is.
      uint32_t r0[kLd], r1[kLd];
      auto add = [&](int c, const uint32_t (&r)[kLd], float f) {
#pragma unroll
        for (int i = 0; i < kLd; i += 2) add2(acc2[(c + i) / 2], r[i], r[i + 1], f);
      };
      ok = first_ready(try_first());
      if (!ok) break;
      tc_fence_after();
      float f = factor();
      tmem_ld<kLd>(tbase + buf * 256, r0);
      tmem_ld<kLd>(tbase + buf * 256 + 32, r1);
      for (int kb = 0;;) {
        const uint32_t at = tbase + buf * 256;
        tmem_ld_wait();
        release(0);
        const bool second = try_second();
        add(0, r0, f);
        add(32, r1, f);
        ok = second_ready(second);
        if (!ok) break;
        tc_fence_after();
        tmem_ld<kLd>(at + 128, r0);
        tmem_ld<kLd>(at + 160, r1);
        tmem_ld_wait();
        const uint32_t last = buf;
        next_group();
        tc_fence_before();
        mbar_arrive_cluster_if(lane == 0, tempty0 + (last * 2 + 1) * sizeof(uint64_t));
        const bool more = ++kb < kblocks, next = more && try_first();
        add(64, r0, f);
        add(96, r1, f);
        if (!more) break;
        ok = first_ready(next);
        if (!ok) break;
        tc_fence_after();
        tmem_ld<kLd>(tbase + buf * 256, r0);
        tmem_ld<kLd>(tbase + buf * 256 + 32, r1);
        f = factor();
      }
      if (!ok) break;
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[2 * i]), "=f"(acc[2 * i + 1]) : "l"(acc2[i]));
      if (a.out_f32)
        store_warp_tile<float, kF8PairPieces>(a, y_map, acc, out_buf, m0, n0, lane);
      else
        store_warp_tile<__nv_bfloat16, kF8PairPieces>(a, y_map, acc, out_buf, m0, n0, lane);
    }
    if (a.rows16 && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
  }
  tc_fence_before();
  cluster_arrive_wait();  // every arrival at the other's barriers has landed
  __syncthreads();
  // NaN over the tiles of a CTA in which a wait gave up. Here, with nothing kept for it through the loops, whose
  // registers are spent (8192 x 16384 x 2048: 248 us with it where the epilogue's loop ends, 245 without).
  if (__builtin_expect(*reinterpret_cast<volatile int*>(&abort_flag), 0)) {
    int t, r;
    asm volatile("mov.u32 %0, %%tid.x;" : "=r"(t));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    if (t < kF8EpiWarps * 32)
      for (F8TileWalk tile(a); tile.more(); tile.next())
        give_up_outputs(a, tile.token0(r) + (t >> 5 & 3) * 32, tile.feature0() + (t >> 7) * kF8Block, kF8Block, t & 31);
  }
  if (warp == 9) {
    tc_fence_after();
    f8_tmem_dealloc<true>(tmem, 512);
  }
}

// ------------------------------------------------------------------------------ host side
struct F8Plan {
  bool pair, few;
  int per_sm;  // CTAs per SM that the ring (and the small kernel) is cut for
  int splits, stages, box_rows;
  int kblocks, m_tiles, n_tiles;
  size_t ring, smem;
};

F8Plan plan_fp8(int M, int N, int K) {
  F8Plan p = {};
  p.kblocks = (K + kFp8Group - 1) / kFp8Group;
  p.box_rows = std::min(kF8TileM, (M + 7) / 8 * 8);
  p.m_tiles = (M + kF8TileM - 1) / kF8TileM;
  p.n_tiles = (N + kF8Block - 1) / kF8Block;
  p.splits = 1;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  // More than one tile per SM and tokens for pairs: pairs, although their last wave may be partial
  // (512 x 16384 x 2048: 21.0 us against 25.2 on small tiles; 320 x 16384 x 2048: 19.8 and 21.6; 160 x
  // 16384 x 2048: 13.0 and 12.9).
  p.pair = M > kF8TileM && tiles > 148;
  if (p.pair) {
    p.m_tiles = (p.m_tiles + 1) / 2;
    p.n_tiles = (p.n_tiles + 1) / 2;
    p.stages = kF8PairStages;
    p.smem = kF8PairSmem;
    return p;
  }
  // A group takes a CTA alone on its SM about 0.29 us, and the exchange of partial tiles 1.4-2.5 us
  // (more for more tokens): K is split where it is long enough to win that back, at most four
  // ways, and only while all clusters find room at once (four CTAs of an SM each do not fill every
  // GPC; four-CTA clusters find room for 132). 5 x 2048 x 2048: 5.0 us unsplit, 4.2 split in four; 5 x
  // 2048 x 8192: 15.2 and 6.7; 320 x 2048 x 8192: 22.3 and 15.0 in two; but 320 x 2048 x 2048: 7.5 and 8.0.
  p.per_sm = tiles <= 148 ? 1 : 2;
  if (p.kblocks >= (p.box_rows <= 32 ? 16 : 24))
    while (p.splits < kF8MaxSplits && tiles * p.splits * 2 <= (p.splits == 1 ? 148 : 128) && p.kblocks >= 8 * p.splits)
      p.splits *= 2;
  // 32 tokens on the MMA's N were slower than on the lanes (32 x 16384 x 2048: 10.6 against 9.0 us).
  if (M <= kF8FewTokens) {
    p.few = true;
    p.box_rows = kF8FewTokens;
    const size_t stage = kF8TileBytes + kF8FewTokens * kFp8Group;
    const size_t fixed = kF8FewTokens * (kF8Block + 4) * sizeof(float) + sizeof(F8FewBarriers) + kF8FewBufs * sizeof(F8Scales);
    p.stages = static_cast<int>(std::min<size_t>(kF8MaxStages, ((p.per_sm == 1 ? 227 : 113) * 1024 - fixed) / (stage + sizeof(F8Scales))));
    p.smem = fixed + p.stages * (stage + sizeof(F8Scales));
    return p;
  }
  const size_t x_bytes = static_cast<size_t>(p.box_rows) * kFp8Group, stage = kF8TileBytes + x_bytes;
  // An MMA reads 128 token rows: with fewer in a box it runs on into the next stage, whose lanes
  // are never read back; the last stage needs that much room behind it.
  const size_t slack = kF8TileBytes - x_bytes;
  // 228 KB per SM, of which each CTA takes 1 KB for itself: 113 KB each for two CTAs
  const size_t fixed = sizeof(F8SmallBarriers) + f8_small_bufs(p.per_sm) * sizeof(F8Scales);
  p.stages = static_cast<int>(std::min<size_t>(kF8MaxStages, ((p.per_sm == 1 ? 227 : 113) * 1024 - fixed - slack) / (stage + sizeof(F8Scales))));
  p.ring = std::max(p.stages * stage + slack, p.splits > 1 ? static_cast<size_t>(p.box_rows) * (kF8Block + 4) * 4
                                                           : static_cast<size_t>(kF8EpiWarps) * kF8OutPiece);
  p.smem = fixed + p.ring + p.stages * sizeof(F8Scales);
  return p;
}

// The attributes belong to the current device's copy of the kernel.
template <typename K>
cudaError_t prepare_fp8(K kernel, std::atomic<bool> (&ready)[kF8MaxDevices]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < kF8MaxDevices && ready[dev].load(std::memory_order_acquire))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev < kF8MaxDevices) ready[dev].store(true, std::memory_order_release);
  return e;
}

cudaError_t launch_fp8(const F8Plan& p, const CUtensorMap& wm, const CUtensorMap& xm, const CUtensorMap& ym, const F8Args& a,
                       cudaStream_t s) {
  static std::atomic<bool> ready[4][kF8MaxDevices];
  const cudaError_t e = p.few           ? prepare_fp8(gemm_fp8_few_kernel, ready[3])
                        : p.pair          ? prepare_fp8(gemm_fp8_pair_kernel, ready[0])
                        : p.per_sm == 1 ? prepare_fp8(gemm_fp8_small_kernel<1>, ready[1])
                                        : prepare_fp8(gemm_fp8_small_kernel<2>, ready[2]);
  if (e != cudaSuccess) return e;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  const int cluster = p.pair ? 2 : p.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.pair ? std::min<int64_t>(tiles, 74) : tiles) * cluster));
  cfg.blockDim = dim3(p.few ? kF8FewThreads : p.pair ? kF8PairThreads : f8_small_threads(p.per_sm));
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (p.few) return cudaLaunchKernelEx(&cfg, gemm_fp8_few_kernel, wm, xm, a);
  return p.pair ? cudaLaunchKernelEx(&cfg, gemm_fp8_pair_kernel, wm, xm, ym, a)
                : p.per_sm == 1 ? cudaLaunchKernelEx(&cfg, gemm_fp8_small_kernel<1>, wm, xm, ym, a)
                                : cudaLaunchKernelEx(&cfg, gemm_fp8_small_kernel<2>, wm, xm, ym, a);
}

}  // namespace
}  // namespace specb200

// ------------------------------------------------------------------------------ C ABI
using namespace specb200;
extern "C" int specb200_set_error(int code, const char* msg);

namespace {
int run_linear_fp8(const void* x, int64_t ldx, const float* x_scales, const void* w, int64_t ldw, const float* w_scales,
                   int M, int N, int K, int out_f32, void* y, int64_t ldy, bool starved, int32_t* status, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || M > (1 << 30) || N > (1 << 30) || K > (1 << 30))
    return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: bad M/N/K");
  if (ldx < K || ldw < K || ldx % 16 || ldw % 16 || ldy < N)
    return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: row pitch (operands: at least K and a multiple of 16 bytes; y: at least N)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    const cudaError_t e = status ? cudaMemsetAsync(status, 0, sizeof(int32_t), s) : cudaSuccess;
    return e == cudaSuccess ? SPECB200_OK : specb200_set_error(SPECB200_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!x || !x_scales || !w || !w_scales || !y) return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: null pointer");
  if (!fp8_aligned(x, 16) || !fp8_aligned(w, 16))
    return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: operands must start on 16-byte boundaries");
  if (!fp8_aligned(x_scales, 4) || !fp8_aligned(w_scales, 4) || !fp8_aligned(y, out_f32 ? 4 : 2) || !fp8_aligned(status, 4))
    return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: a pointer is not on a boundary of its elements");
  const F8Plan p = plan_fp8(M, N, K);
  if (static_cast<int64_t>(p.m_tiles) * p.n_tiles > (1 << 30)) return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: M x N too large");
  CUtensorMap wm, xm;
  if (!make_tmap_u8_2d(&wm, w, K, N, ldw, kFp8Group, kF8TileM) || !make_tmap_u8_2d(&xm, x, K, M, ldx, kFp8Group, p.box_rows))
    return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: TMA descriptor");
  CUtensorMap ym = {};
  const int esize = out_f32 ? 4 : 2;
  const bool y_rows16 = fp8_aligned(y, 16) && (ldy * esize) % 16 == 0;
  if (!p.few && p.splits == 1 && y_rows16 && !make_tmap_out_2d(&ym, y, out_f32 != 0, N, M, ldy * esize, 128 / esize, 32))
    return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: TMA descriptor");
  F8Args a = {};
  a.M = M;
  a.N = N;
  a.K = K;
  a.kblocks = p.kblocks;
  a.m_tiles = p.m_tiles;
  a.n_tiles = p.n_tiles;
  a.splits = p.splits;
  a.stages = p.stages;
  a.ring_bytes = static_cast<uint32_t>(p.ring);
  a.x_bytes = static_cast<uint32_t>(p.box_rows) * kFp8Group;
  a.xs = x_scales;
  a.ws = w_scales;
  a.y = y;
  a.ldy = ldy;
  a.out_f32 = out_f32 ? 1 : 0;
  a.rows16 = y_rows16;
  a.tail16 = (static_cast<int64_t>(N) * esize) % 16 == 0;
  a.starved = starved;
  a.status = status;
  cudaError_t e = cudaSuccess;
  if (status) e = cudaMemsetAsync(status, 0, sizeof(int32_t), s);
  if (e == cudaSuccess) e = launch_fp8(p, wm, xm, ym, a, s);
  return e == cudaSuccess ? SPECB200_OK : specb200_set_error(SPECB200_ERR_CUDA, cudaGetErrorString(e));
}
}  // namespace

extern "C" int specb200_linear_fp8(const void* x, int64_t ldx, const float* x_scales, const void* w, int64_t ldw,
                                   const float* w_scales, int M, int N, int K, int out_f32, void* y, int64_t ldy,
                                   int32_t* status, void* stream) {
  return run_linear_fp8(x, ldx, x_scales, w, ldw, w_scales, M, N, K, out_f32, y, ldy, false, status, stream);
}

extern "C" int specb200_linear_fp8_wait_probe(const void* x, int64_t ldx, const float* x_scales, const void* w, int64_t ldw,
                                              const float* w_scales, int M, int N, int K, int out_f32, void* y, int64_t ldy,
                                              int32_t* status, void* stream) {
  return run_linear_fp8(x, ldx, x_scales, w, ldw, w_scales, M, N, K, out_f32, y, ldy, true, status, stream);
}
