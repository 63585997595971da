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
// owns one token, half of the tile's features lie in one weight block, and the factor of a group
// is one number per thread. Warp 8 issues TMA (both operands K-major with the 128-byte swizzle:
// one atom is one group), warp 9 tcgen05.mma, warps 0-7 read back (w and w + 4 on lane quarter
// w % 4, each half of the columns).
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

constexpr int kF8Threads = 320;
constexpr int kF8EpiWarps = 8;
constexpr int kF8TileM = 128;
constexpr int kF8MaxSplits = 8;
constexpr int kF8MaxDevices = 64;

struct F8Args {
  int M, N, K;
  int kblocks, m_tiles, n_tiles, splits, stages;
  uint32_t x_bytes;     // bytes of a stage's token box (box rows x 128)
  const float* xs;      // [M, kblocks]
  const float* ws;      // [n / 128, kblocks]
  void* y;
  int64_t ldy;
  int out_f32, vec_y;
  int32_t* status;
};

// tcgen05.mma on e4m3 operands, 32 of K per instruction.
SPECB200_DEVINL void umma_e4m3_elect(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor, kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), e4m3 A and B (bits 7-9
// and 10-12 = 0), both K-major, N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

SPECB200_DEVINL void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
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

// n consecutive outputs of one token (n a multiple of 4), `valid` of them inside the row.
template <int kN>
SPECB200_DEVINL void store_row(const F8Args& a, int64_t at, int valid, const float (&v)[kN]) {
  if (a.out_f32) {
    float* p = static_cast<float*>(a.y) + at;
    if (a.vec_y && valid >= kN) {
#pragma unroll
      for (int i = 0; i < kN; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (i < valid) p[i] = v[i];
    return;
  }
  __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.y) + at;
  if (a.vec_y && valid >= kN) {
    if constexpr (kN % 8 == 0) {
#pragma unroll
      for (int i = 0; i < kN; i += 8) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
          u[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(p + i) = make_uint4(u[0], u[1], u[2], u[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; i += 4) {
        const __nv_bfloat162 b0 = __floats2bfloat162_rn(v[i], v[i + 1]), b1 = __floats2bfloat162_rn(v[i + 2], v[i + 3]);
        *reinterpret_cast<uint2*>(p + i) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kN; ++i)
    if (i < valid) p[i] = __float2bfloat16_rn(v[i]);
}

template <int BN>
__global__ void __launch_bounds__(kF8Threads, BN == 128 ? 2 : 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, F8Args a) {
  constexpr int kCols = BN / 2;             // features per epilogue thread
  constexpr int kPitch = BN + 4;            // partial tile's row pitch (floats)
  constexpr uint32_t kWBytes = BN * kFp8Group;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[16], empty[16], tfull[2], tempty[2];
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t stage_bytes = kWBytes + a.x_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = a.stages;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kF8EpiWarps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
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

  if (warp == 8) {
    if (lane == 0) {
      tma_prefetch_desc(&w_map);
      tma_prefetch_desc(&x_map);
      pdl_wait();
      uint32_t it = 0, done = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const int m0 = (t % a.m_tiles) * kF8TileM, n0 = (t / a.m_tiles) * BN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const uint32_t st = it % stages;
          if (!mbar_wait_bounded(&empty[st], ((it / stages) & 1) ^ 1, a.status, &abort_flag)) { ok = false; break; }
          uint8_t* s = smem + st * stage_bytes;
          mbar_arrive_expect_tx(&full[st], stage_bytes);
          tma_load_2d(s, &w_map, &full[st], kb * kFp8Group, n0);
          tma_load_2d(s + kWBytes, &x_map, &full[st], kb * kFp8Group, m0);
        }
      }
      // Tail: the last use of every stage is released (so no commit arrives after the exit), or,
      // where a wait gave up, at least every copy in flight has landed.
      for (done = it > static_cast<uint32_t>(stages) ? it - stages : 0; done < it; ++done) {
        const uint32_t st = done % stages;
        if (ok) ok = mbar_wait_bounded(&empty[st], (done / stages) & 1, a.status, &abort_flag);
        if (!ok) mbar_wait_bounded(&full[st], (done / stages) & 1, a.status, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    constexpr uint32_t idesc = umma_idesc_e4m3(kF8TileM, BN);
    uint32_t it = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t st = it % stages, buf = it & 1;
        ok = mbar_wait_warp(&tempty[buf], ((it >> 1) & 1) ^ 1, a.status, &abort_flag) &&
             mbar_wait_warp(&full[st], (it / stages) & 1, a.status, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dw = umma_desc_sw128(smem_u32(smem + st * stage_bytes));
        const uint64_t dx = umma_desc_sw128(smem_u32(smem + st * stage_bytes + kWBytes));
#pragma unroll
        for (int kk = 0; kk < kFp8Group / 32; ++kk)
          umma_e4m3_elect(tmem + buf * BN, dx + kk * 2, dw + kk * 2, idesc, kk > 0 ? 1u : 0u);
        umma_commit_elect(&empty[st]);
        umma_commit_elect(&tfull[buf]);
      }
    }
    __syncwarp();
  } else {
    pdl_wait();
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * kCols;
    uint32_t it = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      const int m0 = (t % a.m_tiles) * kF8TileM, n0 = (t / a.m_tiles) * BN;
      const int m = m0 + quarter * 32 + lane, n = n0 + half * kCols;
      const bool live = m0 + quarter * 32 < a.M && n < a.N;  // whole warps without outputs only keep step
      const float* sx = a.xs + static_cast<int64_t>(min(m, a.M - 1)) * a.kblocks;
      const float* sw = a.ws + static_cast<int64_t>(min(n, a.N - 1) / kFp8Group) * a.kblocks;
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
      float fx = live ? __ldg(sx + kb0) : 0.f, fw = live ? __ldg(sw + kb0) : 0.f;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t buf = it & 1;
        const float f = fx * fw;
        if (live && kb + 1 < kb1) {
          fx = __ldg(sx + kb + 1);
          fw = __ldg(sw + kb + 1);
        }
        ok = mbar_wait_warp(&tfull[buf], (it >> 1) & 1, a.status, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (live) {
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t r[32];
            tmem_ld32(tbase + buf * BN + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c + i] = fmaf(__uint_as_float(r[i]), f, acc[c + i]);
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[buf]);
      }
      if (!ok) break;
      if (splits == 1) {
        if (m < a.M && n < a.N) store_row<kCols>(a, static_cast<int64_t>(m) * a.ldy + n, a.N - n, acc);
      } else if (live) {  // one tile per cluster: every stage has been read, the ring holds the partial tile
        float* p = reinterpret_cast<float*>(smem) + (quarter * 32 + lane) * kPitch + half * kCols;
#pragma unroll
        for (int i = 0; i < kCols; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
      }
    }
  }
  __syncwarp();
  if (splits > 1) {
    cluster_arrive_wait();
    const int m0 = (first % a.m_tiles) * kF8TileM, n0 = (first / a.m_tiles) * BN;
    const int rows = min(kF8TileM, a.M - m0), quads = BN / 4;
    if (!*reinterpret_cast<volatile int*>(&abort_flag)) {
      const uint32_t base = smem_u32(smem);
      for (int i = split * kF8Threads + threadIdx.x; i < rows * quads; i += splits * kF8Threads) {
        const int r = i / quads, c = (i % quads) * 4;
        if (n0 + c >= a.N) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int p = 0; p < splits; ++p) {
          const float4 q = ld_cluster_f4(base + (r * kPitch + c) * 4, p);
          v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
        }
        store_row<4>(a, static_cast<int64_t>(m0 + r) * a.ldy + n0 + c, a.N - n0 - c, v);
      }
    }
    cluster_arrive_wait();  // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * BN);
  }
}

// ------------------------------------------------------------------------------ host side
struct F8Plan {
  int bn, splits, stages, box_rows;
  int kblocks, m_tiles, n_tiles;
  size_t smem;
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
  const size_t budget = p.bn == 128 ? 110 * 1024 : 222 * 1024;
  p.stages = static_cast<int>(std::min<size_t>(12, (budget - slack) / stage));
  p.smem = 1024 + p.stages * stage + slack;
  if (p.splits > 1) p.smem = std::max<size_t>(p.smem, 1024 + static_cast<size_t>(p.box_rows) * (p.bn + 4) * 4);
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
    e = cudaFuncSetAttribute(gemm_fp8_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(gemm_fp8_kernel<BN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    if (dev < kF8MaxDevices) ready[dev].store(true, std::memory_order_release);
  }
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.splits > 1 ? tiles * p.splits : std::min<int64_t>(tiles, BN == 128 ? 296 : 148)));
  cfg.blockDim = dim3(kF8Threads);
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
