// Linear layers on 8-bit operands (fp8.cuh): with xq, wq e4m3 and b running over the groups of
// 128 along K,
//   y[m, n] = sum_b  sx[m, b] * sw[n / 128, b] * sum_{k in b} xq[m, k] * wq[n, k].
//
// The inner sum runs on the tensor cores (tcgen05.mma kind::f8f6f4, fp32 accumulator in TMEM);
// its 128 products of one group share one pair of scales, so each group's partial tile is read
// back and added to fp32 registers with the factor sx * sw. Two TMEM buffers alternate: the MMA
// of group b + 1 runs while group b is added.
//
// A CTA computes a tile of 128 tokens x BN features, tokens on the TMEM lanes: a thread then
// owns one token and 64 features of one weight block, and the factor of a group is one number per
// thread. Warp roles: kEpi epilogue warps (warp w reads TMEM lane quarter w % 4, columns
// 64 (w / 4)..), then a warp that issues TMA (both operands K-major with the 128-byte swizzle: one
// atom is one group) and a warp that issues tcgen05.mma.
//
// With few tiles K is split over the CTAs of a cluster. Each leaves its partial tile in its own
// shared memory and the cluster adds them through distributed shared memory in split order, so
// results do not depend on scheduling and no workspace exists that two calls could share.
#include <algorithm>
#include <atomic>

#include "fp8.cuh"
#include "gemm.cuh"

namespace specb200 {
namespace {

constexpr int kF8TileM = 128;
constexpr int kF8Cols = 64;  // features per epilogue thread
constexpr int kF8MaxSplits = 8;
constexpr int kF8MaxStages = 12;
constexpr int kF8MaxDevices = 64;
constexpr int kF8OutBytes = 2048;  // per epilogue warp: 32 rows x 64 bytes of output on their way to memory

// Epilogue warps of a BN-wide tile, and the block around them (with a whole fifth warpgroup
// where registers are redistributed).
__host__ __device__ constexpr int f8_epi_warps(int bn) { return bn / kF8Cols * 4; }
__host__ __device__ constexpr int f8_threads(int bn) { return bn == 256 ? 640 : 320; }

struct F8Barriers {
  uint64_t full[kF8MaxStages], empty[kF8MaxStages], tfull[2], tempty[2];
  uint32_t tmem_holder;
  int abort_flag;
};

struct F8Args {
  int M, N, K;
  int kblocks, m_tiles, n_tiles, splits, stages;
  uint32_t ring_bytes;
  uint32_t x_bytes;     // bytes of a stage's token box (box rows x 128)
  const float* xs;      // [M, kblocks]
  const float* ws;      // [n / 128, kblocks]
  void* y;
  int64_t ldy;
  int out_f32, vec_y;
  int32_t* status;
};

// The MMAs of one group (128 of K in four instructions), overwriting the accumulator, and the two
// commits: the stage is free and the accumulator complete once they have run. Every lane of the
// warp executes this, the elected one (leader != 0) issues.
SPECB200_DEVINL void umma_group_e4m3(uint32_t leader, uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                     uint64_t* stage_free, uint64_t* acc_full) {
  asm volatile(
      "{\n\t.reg .pred p, first, rest;\n\t"
      "setp.ne.b32 p, %0, 0;\n\t"
      "setp.ne.b32 first, 0, 0;\n\t"
      "setp.eq.b32 rest, 0, 0;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %2, %6, %10, first;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %3, %7, %10, rest;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %4, %8, %10, rest;\n\t"
      "@p tcgen05.mma.cta_group::1.kind::f8f6f4 [%1], %5, %9, %10, rest;\n\t"
      "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%11];\n\t"
      "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%12];\n\t}" ::"r"(leader),
      "r"(tmem_d), "l"(a), "l"(a + 2), "l"(a + 4), "l"(a + 6), "l"(b), "l"(b + 2), "l"(b + 4), "l"(b + 6), "r"(idesc),
      "r"(smem_u32(stage_free)), "r"(smem_u32(acc_full))
      : "memory");
}
SPECB200_DEVINL uint32_t elect_leader() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
  return r;
}

// Bounded wait of a whole warp: every lane polls (no broadcast on the fast path) and all take the
// same way out. Gives up as mbar_wait_bounded does.
SPECB200_DEVINL bool wait_warp(uint64_t* bar, uint32_t parity, int32_t* status, volatile int* abort) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long start = clock64();
  while (true) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const bool late = clock64() - start > SPECB200_SPIN_LIMIT_CYCLES;
    if (late) {
      set_status(status, SPECB200_ERR_TIMEOUT);
      *abort = 1;
    }
    if (__any_sync(0xffffffffu, late || *abort)) return false;
  }
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
SPECB200_DEVINL float4 ld_cluster_f4(uint32_t addr, uint32_t rank) {
  uint32_t r;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
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
    if (a.vec_y && valid >= 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = v[i];
    return;
  }
  __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.y) + at;
  if (a.vec_y && valid >= 4) {
    const __nv_bfloat162 b0 = __floats2bfloat162_rn(v[0], v[1]), b1 = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < valid) p[i] = __float2bfloat16_rn(v[i]);
}

// One warp's 32 tokens x 64 features to memory through 2 KB of shared memory, so that rows are
// written in 64-byte pieces: 32 bf16 or 16 fp32 features at a time. The 16-byte units of a row are
// swizzled by the row so that neither side has bank conflicts.
template <typename T>
SPECB200_DEVINL void store_warp_tile(const F8Args& a, const float (&acc)[kF8Cols], uint8_t* buf, int m0, int n0, int lane) {
  constexpr int kUnit = 16 / sizeof(T), kPiece = 4 * kUnit;
  const int row = lane >> 2, unit = lane & 3;
#pragma unroll
  for (int c = 0; c < kF8Cols; c += kPiece) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(acc[c + u * kUnit + 2 * j], acc[c + u * kUnit + 2 * j + 1]);
          v[j] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          v[j] = __float_as_uint(acc[c + u * kUnit + j]);
        }
      }
      *reinterpret_cast<uint4*>(buf + lane * 64 + (u ^ ((lane >> 1) & 3)) * 16) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    __syncwarp();
    const int n = n0 + c + unit * kUnit, left = a.N - n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row + 8 * i, m = m0 + r;
      const uint4 q = *reinterpret_cast<const uint4*>(buf + r * 64 + (unit ^ ((r >> 1) & 3)) * 16);
      if (m < a.M && left > 0) {
        T* p = static_cast<T*>(a.y) + static_cast<int64_t>(m) * a.ldy + n;
        if (a.vec_y && left >= kUnit) {
          *reinterpret_cast<uint4*>(p) = q;
        } else {
          const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
          for (int j = 0; j < kUnit; ++j)
            if (j < left) p[j] = e[j];
        }
      }
    }
    __syncwarp();
  }
}

template <int BN>
__global__ void __launch_bounds__(f8_threads(BN), BN == 128 ? 2 : 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, F8Args a) {
  constexpr int kEpi = f8_epi_warps(BN), kThreads = f8_threads(BN);
  constexpr int kLd = BN == 256 ? 32 : 16;  // accumulator columns read back at a time (what registers allow)
  constexpr int kPitch = BN + 4;            // partial tile's row pitch (floats)
  constexpr uint32_t kWBytes = BN * kFp8Group;
  // output staging, the ring (1024-byte swizzle atoms), then the barriers
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + kEpi * kF8OutBytes;
  F8Barriers& bars = *reinterpret_cast<F8Barriers*>(ring + a.ring_bytes);
  uint64_t *full = bars.full, *empty = bars.empty, *tfull = bars.tfull, *tempty = bars.tempty;
  uint32_t& tmem_holder = bars.tmem_holder;
  int& abort_flag = bars.abort_flag;
  const uint32_t stage_bytes = kWBytes + a.x_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t stages = a.stages;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kEpi);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kEpi + 1) {
    tmem_alloc(&tmem_holder, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  // Only now may the next kernel's CTAs start: one that allocated TMEM before this CTA and then
  // waited for it would keep it from ever starting.
  pdl_launch_dependents();

  const int splits = a.splits;
  const int split = splits > 1 ? static_cast<int>(blockIdx.x) % splits : 0;
  const int first = static_cast<int>(blockIdx.x) / splits, step = static_cast<int>(gridDim.x) / splits;
  const int tiles = a.m_tiles * a.n_tiles;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.kblocks) * split / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.kblocks) * (split + 1) / splits);

  // 640 threads start with 96 registers each, 61,440; the shares below sum to 57,344 + 4,096.
  if (warp >= kEpi) {
    if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == kEpi && lane == 0) {
      tma_prefetch_desc(&w_map);
      tma_prefetch_desc(&x_map);
      pdl_wait();
      uint32_t st = 0, phase = 0, issued = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const int m0 = (t % a.m_tiles) * kF8TileM, n0 = (t / a.m_tiles) * BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_bounded(&empty[st], phase ^ 1, a.status, &abort_flag)) { ok = false; break; }
          uint8_t* s = ring + st * stage_bytes;
          mbar_arrive_expect_tx(&full[st], stage_bytes);
          tma_load_2d(s, &w_map, &full[st], kb * kFp8Group, n0);
          tma_load_2d(s + kWBytes, &x_map, &full[st], kb * kFp8Group, m0);
          if (issued < stages) ++issued;
          if (++st == stages) { st = 0; phase ^= 1; }
        }
      }
      // Tail: the last use of every stage is released (so no commit arrives after the exit), or,
      // where a wait gave up, at least every copy in flight has landed.
      for (uint32_t i = 0; i < issued; ++i) {
        if (st == 0) { st = stages; phase ^= 1; }
        --st;
        if (ok) ok = mbar_wait_bounded(&empty[st], phase, a.status, &abort_flag);
        if (!ok) mbar_wait_bounded(&full[st], phase, a.status, nullptr);
      }
    } else if (warp == kEpi + 1) {
      constexpr uint32_t idesc = umma_idesc_e4m3(kF8TileM, BN);
      const uint32_t leader = elect_leader();
      const uint64_t dw0 = umma_desc_sw128(smem_u32(ring)), dx0 = umma_desc_sw128(smem_u32(ring + kWBytes));
      uint32_t st = 0, phase = 0, buf = 0, acc_phase = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = wait_warp(&tempty[buf], acc_phase ^ 1, a.status, &abort_flag) &&
               wait_warp(&full[st], phase, a.status, &abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t at = static_cast<uint64_t>(st * (stage_bytes >> 4));
          umma_group_e4m3(leader, tmem + buf * BN, dx0 + at, dw0 + at, idesc, &empty[st], &tfull[buf]);
          if (++st == stages) { st = 0; phase ^= 1; }
          buf ^= 1;
          acc_phase ^= buf ^ 1;
        }
      }
    }
    __syncwarp();
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    pdl_wait();
    const int quarter = warp & 3, col0 = (warp >> 2) * kF8Cols;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + col0;
    uint32_t buf = 0, acc_phase = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      const int m0 = (t % a.m_tiles) * kF8TileM + quarter * 32, n0 = (t / a.m_tiles) * BN + col0;
      const bool live = m0 < a.M && n0 < a.N;  // warps without outputs only keep step
      const float* sx = a.xs + static_cast<int64_t>(min(m0 + lane, a.M - 1)) * a.kblocks;
      const float* sw = a.ws + static_cast<int64_t>(min(n0, a.N - 1) / kFp8Group) * a.kblocks;
      float acc[kF8Cols];
#pragma unroll
      for (int i = 0; i < kF8Cols; ++i) acc[i] = 0.f;
      float fx = live ? __ldg(sx + kb0) : 0.f, fw = live ? __ldg(sw + kb0) : 0.f;
      for (int kb = kb0; kb < kb1; ++kb) {
        const float f = fx * fw;
        if (live && kb + 1 < kb1) {
          fx = __ldg(sx + kb + 1);
          fw = __ldg(sw + kb + 1);
        }
        ok = wait_warp(&tfull[buf], acc_phase, a.status, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (live) {
#pragma unroll
          for (int c = 0; c < kF8Cols; c += kLd) {
            uint32_t r[kLd];
            tmem_ld<kLd>(tbase + buf * BN + c, r);
            tmem_ld_wait();
            if (c + kLd == kF8Cols) {  // all read: the next but one group may overwrite it
              tc_fence_before();
              if (lane == 0) mbar_arrive(&tempty[buf]);
            }
#pragma unroll
            for (int i = 0; i < kLd; ++i) acc[c + i] = fmaf(__uint_as_float(r[i]), f, acc[c + i]);
          }
        } else if (lane == 0) {
          mbar_arrive(&tempty[buf]);
        }
        buf ^= 1;
        acc_phase ^= buf ^ 1;
      }
      if (!ok) break;
      if (splits == 1) {
        if (live) {
          if (a.out_f32)
            store_warp_tile<float>(a, acc, smem + warp * kF8OutBytes, m0, n0, lane);
          else
            store_warp_tile<__nv_bfloat16>(a, acc, smem + warp * kF8OutBytes, m0, n0, lane);
        }
      } else if (live) {  // one tile per cluster: every stage has been read, the ring holds the partial tile
        float* p = reinterpret_cast<float*>(ring) + (quarter * 32 + lane) * kPitch + col0;
        if (m0 + lane < a.M) {
#pragma unroll
          for (int i = 0; i < kF8Cols; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        }
      }
    }
  }
  __syncwarp();
  if (splits > 1) {
    cluster_arrive_wait();
    const int m0 = (first % a.m_tiles) * kF8TileM, n0 = (first / a.m_tiles) * BN;
    const int rows = min(kF8TileM, a.M - m0);
    constexpr int kQuads = BN / 4;
    if (!*reinterpret_cast<volatile int*>(&abort_flag)) {
      const uint32_t base = smem_u32(ring);
      for (int i = split * kThreads + threadIdx.x; i < rows * kQuads; i += splits * kThreads) {
        const int r = i / kQuads, c = (i % kQuads) * 4;
        if (n0 + c >= a.N) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int p0 = 0; p0 < splits; p0 += 4) {  // four splits' loads in flight, added in split order
          float4 q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p0 + j < splits) q[j] = ld_cluster_f4(base + (r * kPitch + c) * 4, p0 + j);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (p0 + j < splits) { v[0] += q[j].x; v[1] += q[j].y; v[2] += q[j].z; v[3] += q[j].w; }
        }
        store_quad(a, static_cast<int64_t>(m0 + r) * a.ldy + n0 + c, a.N - n0 - c, v);
      }
    }
    cluster_arrive_wait();  // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kEpi + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * BN);
  }
}

// ------------------------------------------------------------------------------ host side
struct F8Plan {
  int bn, splits, stages, box_rows;
  int kblocks, m_tiles, n_tiles;
  size_t ring, smem;
};

F8Plan plan_fp8(int M, int N, int K) {
  F8Plan p;
  p.kblocks = (K + kFp8Group - 1) / kFp8Group;
  p.m_tiles = (M + kF8TileM - 1) / kF8TileM;
  const int wide = (N + 255) / 256;
  p.bn = static_cast<int64_t>(p.m_tiles) * wide >= 2 * 148 ? 256 : 128;
  p.n_tiles = (N + p.bn - 1) / p.bn;
  p.splits = 1;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  if (p.bn == 128)
    while (p.splits < kF8MaxSplits && tiles * p.splits * 2 <= 2 * 148 && p.kblocks >= 4 * p.splits) p.splits *= 2;
  p.box_rows = std::min(kF8TileM, (M + 7) / 8 * 8);
  const size_t x_bytes = static_cast<size_t>(p.box_rows) * kFp8Group, stage = p.bn * kFp8Group + x_bytes;
  // An MMA reads 128 token rows: with fewer in a box it runs on into the next stage, whose lanes
  // are never read back; the last stage needs that much room behind it.
  const size_t slack = kF8TileM * kFp8Group - x_bytes;
  // 228 KB per SM, of which each CTA takes 1 KB for itself: 113 KB each for two CTAs
  const size_t fixed = static_cast<size_t>(f8_epi_warps(p.bn)) * kF8OutBytes + sizeof(F8Barriers);
  const size_t budget = (p.bn == 128 ? 113 * 1024 : 227 * 1024) - fixed;
  p.stages = static_cast<int>(std::min<size_t>(kF8MaxStages, (budget - slack) / stage));
  p.ring = p.stages * stage + slack;
  if (p.splits > 1) p.ring = std::max(p.ring, static_cast<size_t>(p.box_rows) * (p.bn + 4) * 4);
  p.smem = fixed + p.ring;
  return p;
}

template <int BN>
cudaError_t launch_fp8(const F8Plan& p, const CUtensorMap& wm, const CUtensorMap& xm, const F8Args& a, cudaStream_t s) {
  // the attribute belongs to the current device's copy of the kernel
  static std::atomic<bool> ready[kF8MaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kF8MaxDevices || !ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(gemm_fp8_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(gemm_fp8_kernel<BN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    if (dev < kF8MaxDevices) ready[dev].store(true, std::memory_order_release);
  }
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.splits > 1 ? tiles * p.splits : std::min<int64_t>(tiles, BN == 128 ? 296 : 148)));
  cfg.blockDim = dim3(f8_threads(BN));
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<BN>, wm, xm, a);
}

}  // namespace
}  // namespace specb200

// ------------------------------------------------------------------------------ C ABI
using namespace specb200;
extern "C" int specb200_set_error(int code, const char* msg);

extern "C" int specb200_linear_fp8(const void* x, int64_t ldx, const float* x_scales, const void* w, int64_t ldw,
                                   const float* w_scales, int M, int N, int K, int out_f32, void* y, int64_t ldy,
                                   int32_t* status, void* stream) {
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
  const F8Plan p = plan_fp8(M, N, K);
  if (static_cast<int64_t>(p.m_tiles) * p.n_tiles > (1 << 30)) return specb200_set_error(SPECB200_ERR_ARG, "linear_fp8: M x N too large");
  CUtensorMap wm, xm;
  if (!make_tmap_u8_2d(&wm, w, K, N, ldw, kFp8Group, p.bn) || !make_tmap_u8_2d(&xm, x, K, M, ldx, kFp8Group, p.box_rows))
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
  a.vec_y = fp8_aligned(y, 16) && (ldy * (out_f32 ? 4 : 2)) % 16 == 0;
  a.status = status;
  cudaError_t e = cudaSuccess;
  if (status) e = cudaMemsetAsync(status, 0, sizeof(int32_t), s);
  if (e == cudaSuccess) e = p.bn == 128 ? launch_fp8<128>(p, wm, xm, a, s) : launch_fp8<256>(p, wm, xm, a, s);
  return e == cudaSuccess ? SPECB200_OK : specb200_set_error(SPECB200_ERR_CUDA, cudaGetErrorString(e));
}
