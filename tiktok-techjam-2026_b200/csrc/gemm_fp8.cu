// gemm_fp8.cu -- product of block-scaled e4m3 matrices on tcgen05.
//
//   C[m, n] = act( sum_kb sa[m, kb] sw[n / 128, kb] P_kb[m, n] + bias[n] )
//   P_kb[m, n] = sum over the 128 columns k of block kb of A[m, k] W[n, k]
//
// The scales are arbitrary fp32 numbers, so each block's product P_kb is a
// separate accumulation in tensor memory (four MMAs of K = 32), which warps
// read back, scale and add to fp32 sums in registers while the tensor core
// works on the next block.
//
// Few tokens, in tiles of BT = 16, 32 or 64: the weights are the MMA's 128-row
// operand (TMEM lane = output column n) and the tokens its N operand, so a few
// tokens cost a narrow MMA and not a padded one.  A call of this size is bound
// by its chain launch -> first loads -> MMA -> meeting, then by reading the
// weights (M16 N4096 K4096: 6.7 us, 2.6 by its bytes; M48 N16384 K4096 with
// GELU and an 8-bit output: 17.5 us, 10.4 by its bytes).  The k-blocks of a
// tile are divided over the CTAs of a cluster (so that enough SMs stream the
// weights), whose fp32 sums meet in distributed shared memory: CTA r finishes
// the tokens t = r mod c, adding the CTAs' parts in a fixed order.
//   warp 0      TMA producer: 128 x 128-byte weight and BT x 128-byte token
//               tiles (128-byte swizzle; one k-block) into a stage ring
//   warp 1      owns tensor memory, issues the MMAs
//   warps 2..   scaling: one TMEM lane (one n) per thread, BT tokens (32 of
//               64 in each of two warp groups)
#include <mutex>

#include "fp8.cuh"

namespace tjb {
namespace {

constexpr int kF8Lanes = 128;  // weight rows of a tile = TMEM lanes
constexpr int kF8BK = 128;     // bytes of K per stage: one swizzle row, one scale block
constexpr int kF8ScaleChunk = 8;  // k-blocks whose token scales are staged together

struct GemmF8Args {
  const float* a_scales;  // element (m, kb) at m * as_row + kb * as_blk
  const float* w_scales;  // [ceil(N / 128), K blocks]
  const float* bias;
  void* C;
  float* c_scales;  // [M, ceil(N / 128)] (e4m3 output)
  const int32_t* m_tiles;
  int64_t as_row, as_blk;
  int M, N, K, ldc;
  int out_dtype, act;
  int splits;  // CTAs per cluster (a power of two)
  int first_tile, end_tile;  // wide kernel: the tiles of this launch
};

template <int BT>
struct SkinnyCfg {
  static constexpr int kGroups = BT >= 64 ? 2 : 1;  // scaling warp groups
  static constexpr int kCols = BT / kGroups;        // tokens per scaling thread
  static constexpr int kThreads = 64 + 128 * kGroups;
  static constexpr int kAccs = 4;                   // TMEM accumulators in flight
  static constexpr uint32_t kTmemCols = kAccs * BT;
  // Two CTAs fit an SM.
  static constexpr int kStages = BT == 16 ? 5 : (BT == 32 ? 4 : 3);
  static constexpr uint32_t kWBytes = kF8Lanes * kF8BK;
  static constexpr uint32_t kXBytes = BT * kF8BK;
  static constexpr uint32_t kExBytes = BT * kF8Lanes * 4;  // partial sums from the cluster
  static constexpr uint32_t kScBytes = 2 * kF8ScaleChunk * (BT + 1) * 4;
  static constexpr uint32_t kSmemBytes =
      1024 + kStages * (kWBytes + kXBytes) + kExBytes + kScBytes + 256;
};

// 32 lanes x 16 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld16p(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Four-byte asynchronous copy into shared memory, zero when !valid.
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 4 : 0)
               : "memory");
}

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The four K = 32 MMAs of one 128-byte k-block and two commits, all by one
// elected thread.  The pair's form runs on both CTAs' operands and tensor
// memory and signals the barriers of both.
__device__ __forceinline__ void umma_e4m3_block_w(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                                  uint32_t idesc, uint64_t* bar0, uint64_t* bar1) {
  asm volatile(
      "{\n\t.reg .pred e, z;\n\t.reg .b64 a, b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 z, 0, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, z;\n\t"
      "setp.eq.b32 z, 0, 0;\n\t"
      "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, z;\n\t"
      "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, z;\n\t"
      "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, z;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t}" ::
          "r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(smem_u32(bar0)), "r"(smem_u32(bar1))
      : "memory");
}

__device__ __forceinline__ void umma_e4m3_block_pair_w(uint32_t d_tmem, uint64_t adesc,
                                                       uint64_t bdesc, uint32_t idesc,
                                                       uint64_t* bar0, uint64_t* bar1) {
  asm volatile(
      "{\n\t.reg .pred e, z;\n\t.reg .b64 a, b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 z, 0, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, z;\n\t"
      "setp.eq.b32 z, 0, 0;\n\t"
      "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, z;\n\t"
      "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, z;\n\t"
      "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a, b, %3, z;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%4], %6;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%5], %6;\n\t}" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc),
      "r"(smem_u32(bar0)), "r"(smem_u32(bar1)), "h"(static_cast<uint16_t>(3))
      : "memory");
}

template <int kThreads>
__device__ __forceinline__ void scaling_warps_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
}

// Columns n .. n + 3 of token m (one warp holds 128 columns, this lane four):
// bias, activation, rounding, store.  With an 8-bit output the warp's columns
// are one block.
__device__ __forceinline__ void finish4(const GemmF8Args& args, float4 v, float4 bias, int64_t m,
                                        int n, int lane) {
  v.x += bias.x;
  v.y += bias.y;
  v.z += bias.z;
  v.w += bias.w;
  if (args.act == 1) {
    if (args.out_dtype == TJB_F32) {
      gelu_pair<32>(v.x, v.y);
      gelu_pair<32>(v.z, v.w);
    } else if (args.out_dtype == TJB_E4M3) {
      gelu_pair<8>(v.x, v.y);
      gelu_pair<8>(v.z, v.w);
    } else {
      gelu_pair<16>(v.x, v.y);
      gelu_pair<16>(v.z, v.w);
    }
  }
  if (args.out_dtype == TJB_E4M3) {
    if (n >= args.N) v = make_float4(0.f, 0.f, 0.f, 0.f);
    const float s = block_scale(warp_max_abs(max_abs4(v)));
    if (n < args.N)
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(args.C) + m * args.ldc + n) =
          quantize4(v, divisor(s));
    if (lane == 0) args.c_scales[m * ((args.N + kQBlock - 1) / kQBlock) + n / kQBlock] = s;
  } else if (n < args.N) {
    store4(args.C, args.out_dtype, m * args.ldc + n, v);
  }
}

template <int BT>
__global__ void __launch_bounds__(SkinnyCfg<BT>::kThreads)
    gemm_fp8_skinny_kernel(const __grid_constant__ CUtensorMap tmW,
                           const __grid_constant__ CUtensorMap tmX, const GemmF8Args args) {
  using Cfg = SkinnyCfg<BT>;
  constexpr int kStages = Cfg::kStages, kAccs = Cfg::kAccs, kCols = Cfg::kCols;
  constexpr int kScaleThreads = 128 * Cfg::kGroups;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sW = smem;
  uint8_t* sX = sW + kStages * Cfg::kWBytes;
  float* sEx = reinterpret_cast<float*>(sX + kStages * Cfg::kXBytes);  // [CTA][slot][128]
  float* sSc = sEx + BT * kF8Lanes;                       // [2][kF8ScaleChunk][BT]
  float* sSw = sSc + 2 * kF8ScaleChunk * BT;              // [2][kF8ScaleChunk]
  uint64_t* full = reinterpret_cast<uint64_t*>(sSw + 2 * kF8ScaleChunk);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + kAccs;
  uint64_t* drain = tempty + kAccs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = args.splits;
  const int rank = static_cast<int>(blockIdx.x) & (splits - 1);
  const int tile = static_cast<int>(blockIdx.x) / splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kAccs; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 4 * Cfg::kGroups);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  // Also: every CTA of the cluster has started, so its shared memory may be
  // written from here on.
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // This cluster's tile: 128 output columns, BT tokens from t0.
  constexpr int kPerLive = kLiveTileRows / BT;
  const int t_tiles = args.m_tiles != nullptr
                          ? (args.M + kLiveTileRows - 1) / kLiveTileRows * kPerLive
                          : (args.M + BT - 1) / BT;
  const int n_blk = tile / t_tiles;
  const int tt = tile - n_blk * t_tiles;
  const int kb_count = (args.K + kF8BK - 1) / kF8BK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * kb_count / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * kb_count / splits);
  // The first weight tiles start for L2 while the previous kernel drains (L2
  // holds whatever that kernel may still write to them).
  if (warp == 0 && lane == 0)
    for (int i = kb0; i < kb1 && i < kb0 + kStages; ++i)
      tma_prefetch_2d(&tmW, i * kF8BK, n_blk * kF8Lanes);
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();
  int t0 = tt * BT;
  bool live = true;
  if (args.m_tiles != nullptr) {
    const int li = tt / kPerLive;
    live = li < __ldg(args.m_tiles);
    if (live) t0 = __ldg(args.m_tiles + 1 + li) * kLiveTileRows + (tt % kPerLive) * BT;
  }
  const int tokens = live ? min(BT, args.M - t0) : 0;  // may be <= 0: nothing to do
  const int n_kb = tokens > 0 ? kb1 - kb0 : 0;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ producer
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int i = 0; i < n_kb; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) break;
        mbar_arrive_expect_tx(&full[stage], Cfg::kWBytes + Cfg::kXBytes);
        tma_load_2d(sW + stage * Cfg::kWBytes, &tmW, &full[stage], (kb0 + i) * kF8BK,
                    n_blk * kF8Lanes);
        tma_load_2d(sX + stage * Cfg::kXBytes, &tmX, &full[stage], (kb0 + i) * kF8BK, t0);
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      // Every load has landed before the CTA may release its memory.
      for (int k = issued > kStages ? issued - kStages : 0; k < issued; ++k)
        mbar_wait_drain(&full[k % kStages], (k / kStages) & 1);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = idesc_e4m3(kF8Lanes, BT);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
    };
    for (int i = 0; i < n_kb; ++i) {
      if (!wait(&tempty[acc], acc_phase ^ 1)) break;
      if (!wait(&full[stage], phase)) break;
      tc_fence_after();
      umma_e4m3_block_w(tmem_base + static_cast<uint32_t>(acc * BT),
                        sdesc_sw128(smem_u32(sW + stage * Cfg::kWBytes), 16, 1024),
                        sdesc_sw128(smem_u32(sX + stage * Cfg::kXBytes), 16, 1024), idesc,
                        &tfull[acc], &empty[stage]);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
      if (++acc == kAccs) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    umma_commit_w(drain);
    mbar_wait_drain(drain, 0);
  } else if (n_kb > 0) {
    // ------------------------------------------------------------- scaling
    const int quad = warp & 3;         // TMEM lanes this warp may access
    const int group = (warp - 2) >> 2;  // tokens [group * kCols, + kCols)
    const int tid = threadIdx.x - 64;
    const float* w_scales = args.w_scales + static_cast<int64_t>(n_blk) * kb_count + kb0;
    // Token scales of k-blocks [c * chunk, + chunk) into buffer c & 1, and
    // the weight block's scales beside them.
    auto stage_scales = [&](int c) {
      float* dst = sSc + (c & 1) * kF8ScaleChunk * BT;
      for (int e = tid; e < kF8ScaleChunk * BT; e += kScaleThreads) {
        const int t = e % BT, i = c * kF8ScaleChunk + e / BT;
        const bool valid = t < tokens && i < n_kb;
        const float* src = args.a_scales;
        if (valid) src += (t0 + t) * args.as_row + (kb0 + i) * args.as_blk;
        cp_async4(smem_u32(dst + e), src, valid);
      }
      if (tid < kF8ScaleChunk) {
        const int i = c * kF8ScaleChunk + tid;
        cp_async4(smem_u32(sSw + (c & 1) * kF8ScaleChunk + tid), i < n_kb ? w_scales + i : w_scales,
                  i < n_kb);
      }
    };
    stage_scales(0);
    float sum[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum[j] = 0.f;
    int acc = 0;
    uint32_t acc_phase = 0;
    const uint32_t taddr0 = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + group * kCols;
    for (int i = 0; i < n_kb; ++i) {
      const int c = i / kF8ScaleChunk, ci = i % kF8ScaleChunk;
      if (ci == 0) {
        // Chunk c has arrived for every thread, and every thread is done
        // with chunk c - 1, whose buffer chunk c + 1 takes.
        asm volatile("cp.async.wait_all;" ::: "memory");
        scaling_warps_sync<kScaleThreads>();
        if ((c + 1) * kF8ScaleChunk < n_kb) stage_scales(c + 1);
      }
      // (A wait that ran out has recorded its status; the loop goes on so
      // that every warp still meets the others at the chunk barrier.)
      mbar_wait(&tfull[acc], acc_phase, abort_flag);
      __syncwarp();
      tc_fence_after();
      uint32_t p[kCols];
      if constexpr (kCols == 16) {
        tmem_ld16p(taddr0 + acc * BT, p);
      } else {
#pragma unroll
        for (int j = 0; j < kCols; j += 32) tmem_ld32p(taddr0 + acc * BT + j, p + j);
      }
      tmem_ld_wait_n<kCols>(p);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      const float4* sc = reinterpret_cast<const float4*>(
          sSc + ((c & 1) * kF8ScaleChunk + ci) * BT + group * kCols);
      const float sw = sSw[(c & 1) * kF8ScaleChunk + ci];
#pragma unroll
      for (int j = 0; j < kCols / 4; ++j) {
        const float4 s = sc[j];
        fma2v(sum[4 * j], sum[4 * j + 1], __uint_as_float(p[4 * j]), __uint_as_float(p[4 * j + 1]),
              s.x * sw, s.y * sw, sum[4 * j], sum[4 * j + 1]);
        fma2v(sum[4 * j + 2], sum[4 * j + 3], __uint_as_float(p[4 * j + 2]),
              __uint_as_float(p[4 * j + 3]), s.z * sw, s.w * sw, sum[4 * j + 2], sum[4 * j + 3]);
      }
      if (++acc == kAccs) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    // Token t goes to CTA t mod splits, slot t / splits of this CTA's part.
    const int shift = 31 - __clz(splits);
    const uint32_t mine =
        smem_u32(sEx) +
        static_cast<uint32_t>((rank * (BT >> shift)) * kF8Lanes + quad * 32 + lane) * 4u;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int t = group * kCols + j;
      if (t < tokens)
        st_cluster_f32(map_to_rank(mine + static_cast<uint32_t>((t >> shift) * kF8Lanes) * 4u,
                                   static_cast<uint32_t>(t & (splits - 1))),
                       sum[j]);
    }
  }
  __syncwarp();
  cluster_sync();
  // ------------------------------------------------------------------ output
  // One warp per token of this CTA: lane l holds columns n0 + 4l .. + 3.
  if (warp >= 2) {
    const int shift = 31 - __clz(splits);
    const int n0 = n_blk * kF8Lanes;
    const int n = n0 + lane * 4;
    float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
    if (args.bias != nullptr && n < args.N)
      bias = __ldg(reinterpret_cast<const float4*>(args.bias + n));
    for (int slot = warp - 2; (slot << shift) + rank < tokens; slot += kScaleThreads / 32) {
      const int64_t m = t0 + (slot << shift) + rank;
      const float4* src = reinterpret_cast<const float4*>(sEx + slot * kF8Lanes) + lane;
      float4 v = src[0];
      for (int r = 1; r < splits; ++r) {
        const float4 u = src[r * (BT >> shift) * (kF8Lanes / 4)];
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      finish4(args, v, bias, m, n, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

std::mutex g_f8_mu;
bool g_f8_ready[64][3];

template <int BT>
int launch_skinny(const void* A, const void* W, GemmF8Args args, int lda, int ldw,
                  cudaStream_t stream) {
  using Cfg = SkinnyCfg<BT>;
  constexpr int kSlot = BT == 16 ? 0 : BT == 32 ? 1 : 2;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return TJB_ERR_NO_DEVICE;
  {
    std::lock_guard<std::mutex> lock(g_f8_mu);
    if (!g_f8_ready[dev][kSlot]) {
      if (const int fs = cuda_status(cudaFuncSetAttribute(
              gemm_fp8_skinny_kernel<BT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
              static_cast<int>(Cfg::kSmemBytes))))
        return fs;
      g_f8_ready[dev][kSlot] = true;
    }
  }
  CUtensorMap tmW, tmX;
  int st = make_tmap_2d(&tmW, TJB_E4M3, W, args.K, args.N, ldw, kF8BK, kF8Lanes);
  if (st != TJB_OK) return st;
  st = make_tmap_2d(&tmX, TJB_E4M3, A, args.K, args.M, lda, kF8BK, BT);
  if (st != TJB_OK) return st;
  const int64_t t_tiles = args.m_tiles != nullptr
                              ? static_cast<int64_t>((args.M + kLiveTileRows - 1) / kLiveTileRows) *
                                    (kLiveTileRows / BT)
                              : (args.M + BT - 1) / BT;
  const int64_t tiles = t_tiles * ((args.N + kF8Lanes - 1) / kF8Lanes);
  // As many CTAs per tile as the SMs have room for, at most one per k-block;
  // more than four lose more in their meeting than they gain (M16 N4096 K4096:
  // 6.7 us with four, 7.7 with eight).
  const int64_t slots = static_cast<int64_t>(num_sms()) * 2;
  const int kb_count = (args.K + kF8BK - 1) / kF8BK;
  args.splits = 1;
  while (args.splits < 4 && 2 * args.splits <= kb_count && tiles * 2 * args.splits <= slots)
    args.splits *= 2;
  const int64_t grid = tiles * args.splits;
  if (grid > 2147483647) return TJB_ERR_BAD_SHAPE;
  return launch_kernel_cluster(gemm_fp8_skinny_kernel<BT>, dim3(static_cast<unsigned>(grid)),
                               dim3(Cfg::kThreads), Cfg::kSmemBytes, stream,
                               static_cast<unsigned>(args.splits), tmW, tmX, args);
}

// ------------------------------------------------------------------------
// More tokens: tiles of 256 columns.  Here the tokens are the MMA's rows: a
// thread owns one token and 128 consecutive output columns, which is one weight
// block (one scale product per k-block) and one output block (its 8-bit scale
// needs no exchange).  384 threads:
//   warp 0        TMA producer
//   warp 1        MMA issuer: per k-block four K = 32 MMAs into one of two
//                 256-column TMEM accumulators
//   warps 2, 3    products sa[m, kb] sw[n / 128, kb] of the tile's rows, kChunk
//                 k-blocks at a time, a ring slot ahead of their use, and its
//                 bias
//   warps 4..11   two warp groups, 128 columns each: read P_kb from TMEM in
//                 16-column pieces, the next in flight while one is added to
//                 128 fp32 sums in registers; then GELU, rounding, and TMA
//                 stores from a staging buffer of their own
// Three forms:
//   kPaired  Persistent pairs of SMs (cta_group::2) on tiles of 256 rows, each
//            SM with 128 rows of A and half of the weights: 32 KB of loads a
//            k-block and SM where a single one loads 48 KB.
//   kWhole   Persistent single CTAs on tiles of 128 rows, where the count of
//            tiles divides better by SMs than by pairs.
//   kSplitK  128-row tiles whose k-blocks are divided over the CTAs of a
//            cluster, for too few tiles to fill the SMs.  Each CTA ends with
//            fp32 sums of the whole tile; CTA k finishes rows k * 128 / c ... of
//            it, reading the other CTAs' sums through distributed shared
//            memory and adding them in a fixed order.
// Per k-block and SM the tensor core takes 512 clocks, the multiply-adds 256
// (packed pairs, two clocks a warp).  Measured, a k-block of a pair takes 575
// with MMAs and loads alone, 590 with the reads of tensor memory, 690 with the
// multiply-adds and 740 with scales from the ring; a single CTA 640 and 850.
// The chain MMA -> barrier -> scaling -> barrier -> MMA over two accumulators
// bounds it: every barrier operation and spilled register in the k-loop adds
// to it.  So the k-loop of the scaling warps is unrolled twice, a pair's scales
// are handed over eight k-blocks at a time, and one elected thread issues a
// k-block's MMAs and commits (M8192 N8192 K8192 458 us; four k-blocks a
// hand-over 470, single CTAs 501, those with a loop that is not unrolled 515;
// accumulators of 128 columns, for more slack, 487: their MMAs are bound by
// shared memory).  The scaling threads need the registers that warps 0-3 give
// up (128 x 72 + 256 x 216 = 384 x 168 at launch; kSplitK still spills 24 bytes
// a thread, the other two none).  Under a load that lasts,
// the board's power limit holds the clock near 1.4 GHz.
enum WideForm { kWhole, kSplitK, kPaired };

template <int kForm>
struct WideCfg {
  static constexpr int kStages = kForm == kPaired ? 4 : 3;
  static constexpr int kThreads = 384;
  static constexpr uint32_t kABytes = 128 * kF8BK;
  static constexpr uint32_t kBBytes = (kForm == kPaired ? 128 : 256) * kF8BK;
  static constexpr uint32_t kTmemCols = 512;      // two 256-column accumulators
  // k-blocks of scale products per ring slot
  static constexpr int kChunk = kForm == kPaired ? 8 : 4;
  // Two ring slots of kChunk x 256 scale products, and two tiles' bias.
  static constexpr uint32_t kScaleBytes = 2 * kChunk * 256 * 4 + 2 * 256 * 4;
  static constexpr uint32_t kOutTile = 32 * 128;  // 32 rows x 128 bytes, 128-byte swizzle
  static constexpr uint32_t kOutBytes = 8 * 2 * kOutTile;  // two per scaling warp
  static constexpr uint32_t kSmemBytes =
      1024 + kStages * (kABytes + kBBytes) + kOutBytes + kScaleBytes + 256;
};

// Arrive on the mbarrier at `bar` (shared::cluster address).
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// sum[0..15] += s * p[0..15]
__device__ __forceinline__ void add_scaledN(float* sum, const uint32_t* p, float s) {
#pragma unroll
  for (int j = 0; j < 16; j += 2)
    fma2v(sum[j], sum[j + 1], __uint_as_float(p[j]), __uint_as_float(p[j + 1]), s, s, sum[j],
          sum[j + 1]);
}

// The rows of a split tile that CTA `rank` of C finishes, of which warp `quad`
// of a half takes a quarter: the C parts of each are summed (32 loads in
// flight) and finished.
template <int C>
__device__ __forceinline__ void pull_rows(const GemmF8Args& args, uint32_t half_at, int rank,
                                          int quad, int64_t m0, int n0, int lane) {
  constexpr int kRows = 32 / C;                   // per warp
  constexpr int kGroup = kRows < 8 ? kRows : 8;   // at a time
  const int n = n0 + lane * 4;
  float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
  if (args.bias != nullptr && n < args.N)
    bias = __ldg(reinterpret_cast<const float4*>(args.bias + n));
#pragma unroll 1
  for (int g = 0; g < kRows; g += kGroup) {
    const int row0 = rank * (128 / C) + quad * kRows + g;
    float4 part[kGroup][C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t from = map_to_rank(half_at, static_cast<uint32_t>(c));
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
        part[i][c] = ld_cluster_v4(
            from + static_cast<uint32_t>((row0 + i) * 512 + (lane ^ ((row0 + i) & 31)) * 16));
    }
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      float4 v = part[i][0];
#pragma unroll
      for (int c = 1; c < C; ++c) {
        v.x += part[i][c].x;
        v.y += part[i][c].y;
        v.z += part[i][c].z;
        v.w += part[i][c].w;
      }
      if (m0 + row0 + i < args.M) finish4(args, v, bias, m0 + row0 + i, n, lane);  // warp-uniform
    }
  }
}

template <int kForm>
__global__ void __launch_bounds__(WideCfg<kForm>::kThreads, 1)
    gemm_fp8_wide_kernel(const __grid_constant__ CUtensorMap tmA,
                         const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmC, const GemmF8Args args) {
  using Cfg = WideCfg<kForm>;
  constexpr bool kSplit = kForm == kSplitK, kPair = kForm == kPaired;
  constexpr int kStages = Cfg::kStages, kChunk = Cfg::kChunk;
  constexpr int BN = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kStages * Cfg::kABytes;
  uint8_t* sOut = sB + kStages * Cfg::kBBytes;                        // [warp][2][kOutTile]
  float* sScale = reinterpret_cast<float*>(sOut + Cfg::kOutBytes);  // [slot][k-block][row]
  float* sBias = sScale + 2 * kChunk * 256;                         // [tile & 1][column]
  uint64_t* full = reinterpret_cast<uint64_t*>(sBias + 2 * 256);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* sfull = tempty + 2;
  uint64_t* sempty = sfull + 2;
  uint64_t* drain = sempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = kSplit ? args.splits : 1;
  const int rank = kForm != kWhole ? static_cast<int>(cluster_ctarank()) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], kPair ? 16 : 8);  // the scaling warps (of both CTAs)
      mbar_init(&sfull[b], 2);   // warps 2 and 3
      mbar_init(&sempty[b], 8);  // the scaling warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmC);
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(tmem_slot, Cfg::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, Cfg::kTmemCols);
      tmem_relinquish();
    }
  }
  __syncwarp();
  tc_fence_before();
  // (A pair: both CTAs' barriers and tensor memory, before either signals.)
  if constexpr (kPair)
    cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  const int num_m1 = args.m_tiles != nullptr ? __ldg(args.m_tiles) : (args.M + 127) / 128;
  const int num_m = kPair ? (num_m1 + 1) / 2 : num_m1;
  const int num_n = (args.N + BN - 1) / BN;
  const int num_k = (args.K + kF8BK - 1) / kF8BK;
  // Tiles first, first + step, ... below end; k-blocks [k0, k1) of each.
  const int end = min(num_m * num_n, args.end_tile);
  const int first = args.first_tile + static_cast<int>(blockIdx.x) / (kPair ? 2 : splits);
  const int step =  // (kSplit: one tile)
      kSplit ? end : static_cast<int>(gridDim.x) / (kPair ? 2 : 1);
  const int k0 = kSplit ? rank * num_k / splits : 0;
  const int k1 = kSplit ? (rank + 1) * num_k / splits : num_k;
  // (The order of tile_coords.  Tiles only grow for each role, so the group is
  // counted up, and in a full group the division is a shift: 400 clocks of each
  // tile's start otherwise; M8192 N8192 K1024 82 -> 79 us.)
  int group = kSplit ? first / (kGroupM * num_n) : 0;
  int group_end = (group + 1) * kGroupM * num_n;
  auto coords = [&](int t, int& m_blk, int& n_blk) {
    while (t >= group_end) {
      ++group;
      group_end += kGroupM * num_n;
    }
    const int r = t - (group_end - kGroupM * num_n);
    const int gsize = num_m - group * kGroupM;
    if (gsize >= kGroupM) {
      m_blk = group * kGroupM + r % kGroupM;
      n_blk = r / kGroupM;
    } else {
      m_blk = group * kGroupM + r % gsize;
      n_blk = r / gsize;
    }
    bool has = true;
    if constexpr (kPair) {
      // This CTA's 128 rows of the pair's 256; where the second 128 do not
      // exist its CTA loads the first's again (the MMA needs both) and stores
      // nothing.
      has = 2 * m_blk + rank < num_m1;
      m_blk = 2 * m_blk + (has ? rank : 0);
    }
    if (args.m_tiles != nullptr) m_blk = __ldg(args.m_tiles + 1 + m_blk);
    return has;
  };

  if (warp < 4) {
    regs_dec<72>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ producer
      int stage = 0;
      uint32_t phase = 0, issued = 0, last_parity = 0;
      const uint32_t full_at = kPair ? map_to_rank(smem_u32(full), 0) : 0u;  // (the leader's)
      bool ok = true;
      for (int t = first; ok && t < end; t += step) {
        int m_blk, n_blk;
        coords(t, m_blk, n_blk);
        for (int kb = k0; kb < k1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          if constexpr (kPair) {
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * (Cfg::kABytes + Cfg::kBBytes));
            const uint32_t bar = full_at + static_cast<uint32_t>(stage) * 8u;
            tma_load_2d_pair(sA + stage * Cfg::kABytes, &tmA, bar, kb * kF8BK, m_blk * 128);
            tma_load_2d_pair(sB + stage * Cfg::kBBytes, &tmB, bar, kb * kF8BK,
                             n_blk * BN + rank * 128);
          } else {
            mbar_arrive_expect_tx(&full[stage], Cfg::kABytes + Cfg::kBBytes);
            tma_load_2d(sA + stage * Cfg::kABytes, &tmA, &full[stage], kb * kF8BK, m_blk * 128);
            tma_load_2d(sB + stage * Cfg::kBBytes, &tmB, &full[stage], kb * kF8BK, n_blk * BN);
          }
          issued |= 1u << stage;
          last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // Every load has landed before the CTA may release its memory (a pair's
      // loads count on the leader's barrier: their stage has been read).
      for (int s = 0; s < kStages; ++s)
        if ((issued >> s) & 1u)
          mbar_wait_drain(kPair ? &empty[s] : &full[s], (last_parity >> s) & 1u);
    } else if (warp == 1 && (!kPair || rank == 0)) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc = idesc_e4m3(kPair ? 256 : 128, BN);
      int stage = 0;
      uint32_t phase = 0, it = 0;
      for (int t = first; t < end; t += step) {
        if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const uint32_t acc = it & 1;
          // (A wait that ran out has recorded its status and raised the abort
          // flag, which ends all later ones: the tile runs on to its end.)
          mbar_wait(&tempty[acc], ((it >> 1) & 1) ^ 1, abort_flag);
          mbar_wait(&full[stage], phase, abort_flag);
          __syncwarp();
          tc_fence_after();
          const uint64_t a_desc = sdesc_sw128(smem_u32(sA + stage * Cfg::kABytes), 16, 1024);
          const uint64_t b_desc = sdesc_sw128(smem_u32(sB + stage * Cfg::kBBytes), 16, 1024);
          if constexpr (kPair)
            umma_e4m3_block_pair_w(tmem_base + acc * BN, a_desc, b_desc, idesc, &tfull[acc],
                                   &empty[stage]);
          else
            umma_e4m3_block_w(tmem_base + acc * BN, a_desc, b_desc, idesc, &tfull[acc],
                              &empty[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if constexpr (kPair)
        umma_commit_pair_w(drain, 0x1);
      else
        umma_commit_w(drain);
      mbar_wait_drain(drain, 0);
    } else if (warp >= 2) {
      // ------------------------------------------------------- scales and bias
      // Warps 2 and 3 take 64 rows each, two per lane.
      const int num_nb = (args.N + kQBlock - 1) / kQBlock;
      const int r = (warp - 2) * 64 + lane;
      // Row-major scales whose rows start on 16-byte boundaries: four at a time.
      const bool vec = args.as_blk == 1 && args.as_row % 4 == 0 &&
                       (reinterpret_cast<uintptr_t>(args.a_scales) & 15u) == 0;
      uint32_t c = 0, odd = 0;
      float4 bias;
      bool ok = true;
      for (int t = first; ok && t < end; t += step) {
        int m_blk, n_blk;
        coords(t, m_blk, n_blk);
        const int64_t row = static_cast<int64_t>(m_blk) * 128 + r;
        // Rows past M and columns past N repeat an existing one: their sums
        // are never stored.
        const float* a0 = args.a_scales + min(row, static_cast<int64_t>(args.M - 1)) * args.as_row;
        const float* a1 =
            args.a_scales + min(row + 32, static_cast<int64_t>(args.M - 1)) * args.as_row;
        const float* w0 = args.w_scales + static_cast<int64_t>(2 * n_blk) * num_k;
        const float* w1 = 2 * n_blk + 1 < num_nb ? w0 + num_k : w0;
        if constexpr (!kSplit) {
          // This tile's bias, ready with its first scales (the slot's last
          // readers are two tiles back, before scales that were waited for).
          const int n = n_blk * BN + (warp - 2) * 128 + lane * 4;
          float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
          if (args.bias != nullptr && n < args.N)
            b = __ldg(reinterpret_cast<const float4*>(args.bias + n));
          bias = b;
        }
        for (int kb0 = k0; ok && kb0 < k1; kb0 += kChunk, ++c) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&sempty[c & 1], ((c >> 1) & 1) ^ 1, abort_flag));
#pragma unroll 1
          for (int v = 0; v < kChunk && kb0 + v < k1; v += 4) {
            const int kv = kb0 + v;
            float va[4], vb[4];
            if (vec && kv % 4 == 0 && kv + 4 <= k1) {
              *reinterpret_cast<float4*>(va) = __ldg(reinterpret_cast<const float4*>(a0 + kv));
              *reinterpret_cast<float4*>(vb) = __ldg(reinterpret_cast<const float4*>(a1 + kv));
            } else {
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int kb = min(kv + u, k1 - 1);
                va[u] = __ldg(a0 + kb * args.as_blk);
                vb[u] = __ldg(a1 + kb * args.as_blk);
              }
            }
            float s0[4], s1[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              s0[u] = __ldg(w0 + min(kv + u, k1 - 1));
              s1[u] = __ldg(w1 + min(kv + u, k1 - 1));
            }
            float* dst = sScale + ((c & 1) * kChunk + v) * 256 + r;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              dst[u * 256] = va[u] * s0[u];
              dst[u * 256 + 32] = vb[u] * s0[u];
              dst[u * 256 + 128] = va[u] * s1[u];
              dst[u * 256 + 160] = vb[u] * s1[u];
            }
          }
          if (!kSplit && kb0 == k0) {
            reinterpret_cast<float4*>(sBias + odd * 256)[(warp - 2) * 32 + lane] = bias;
            odd ^= 1;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[c & 1]);
        }
      }
    }
    if constexpr (kSplit) {  // the scaling warps' two meetings below
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {
    regs_inc<216>();
    // ------------------------------------------------- scaling and output
    const int quad = warp & 3;         // TMEM lanes this warp may access
    const int half = (warp - 4) >> 2;  // 128-column half of the tile
    const int r = quad * 32 + lane;    // token row of the tile
    uint8_t* buf = sOut + (warp - 4) * 2 * Cfg::kOutTile;
    const uint32_t taddr0 =
        tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 128);
    const uint32_t tempty_at = kPair ? map_to_rank(smem_u32(tempty), 0) : 0u;  // (the leader's)
    uint32_t it = 0, chunk = 0;  // k-blocks and scale chunks done, over all tiles
    uint32_t odd = 0;            // tiles done, parity
    bool ok = true;
    bool met = !kSplit;  // this warp has been at the cluster's two meetings
    for (int t = first; ok && t < end; t += step) {
      int m_blk, n_blk;
      const bool has = coords(t, m_blk, n_blk);
      const int n0 = n_blk * BN + half * 128;
      // The sums start from the bias, which comes with the first scales;
      // columns past N stay exactly zero (their weight rows load as zeros), as
      // a ragged 8-bit block's scale needs.
      mbar_wait(&sfull[chunk & 1], (chunk >> 1) & 1, abort_flag);
      float sum[128];
#pragma unroll
      for (int j = 0; j < 128; j += 4) {
        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!kSplit) b = reinterpret_cast<const float4*>(sBias + odd * 256 + half * 128)[j / 4];
        sum[j] = b.x;
        sum[j + 1] = b.y;
        sum[j + 2] = b.z;
        sum[j + 3] = b.w;
      }
      odd ^= 1;
#pragma unroll 2
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int u = (kb - k0) & (kChunk - 1);
        if (u == 0 && kb > k0)
          mbar_wait(&sfull[chunk & 1], (chunk >> 1) & 1, abort_flag);
        const float s = sScale[((chunk & 1) * kChunk + u) * 256 + half * 128 + r];
        const uint32_t acc = it & 1;
        mbar_wait(&tfull[acc], (it >> 1) & 1, abort_flag);
        __syncwarp();
        tc_fence_after();
        const uint32_t taddr = taddr0 + acc * BN;
        uint32_t p[2][16];
        tmem_ld16p(taddr, p[0]);
        tmem_ld_wait_n<16>(p[0]);
#pragma unroll
        for (int c = 1; c < 128 / 16; ++c) {
          tmem_ld16p(taddr + c * 16, p[c & 1]);
          add_scaledN(sum + (c - 1) * 16, p[(c - 1) & 1], s);
          tmem_ld_wait_n<16>(p[c & 1]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair)
            mbar_arrive_at(tempty_at + acc * 8u);
          else
            mbar_arrive(&tempty[acc]);
          if (u == kChunk - 1 || kb == k1 - 1) mbar_arrive(&sempty[chunk & 1]);
        }
        if (u == kChunk - 1 || kb == k1 - 1) ++chunk;
        add_scaledN(sum + 128 - 16, p[1], s);
      }
      ok = __all_sync(0xffffffffu, *abort_flag == 0);
      if constexpr (kSplit) {
        // The sums go to this CTA's shared memory as [half][row][32 chunks of
        // 16 bytes, chunk j at j ^ (row & 31)] (the stage ring: this thread
        // has seen the last MMA's barrier, so nothing reads or writes it any
        // more), and CTA k pulls rows k * 128 / c ... of every CTA's.  Neither
        // these stores (a row per lane) nor the loads (a row per warp) meet in
        // a bank, and every remote access is a whole 512-byte row; stored
        // straight into the other CTA, a row per lane, the exchange of eight
        // CTAs took 5.5 us more.
        float4* mine = reinterpret_cast<float4*>(smem) + (half * 128 + r) * 32;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          mine[j ^ lane] =
              make_float4(sum[4 * j], sum[4 * j + 1], sum[4 * j + 2], sum[4 * j + 3]);
        __syncwarp();
        cluster_sync();  // every CTA's sums are in place
        met = true;
        if (n0 < args.N) {
          const int64_t m0 = static_cast<int64_t>(m_blk) * 128;
          const uint32_t half_at = smem_u32(smem) + static_cast<uint32_t>(half * 128 * 512);
          if (splits == 2)
            pull_rows<2>(args, half_at, rank, quad, m0, n0, lane);
          else if (splits == 4)
            pull_rows<4>(args, half_at, rank, quad, m0, n0, lane);
          else
            pull_rows<8>(args, half_at, rank, quad, m0, n0, lane);
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while its sums are being read
        break;
      }
      if (!ok) break;
      if (n0 >= args.N || !has) continue;  // warp-uniform
      if (args.act == 1) {
        if (args.out_dtype == TJB_F32) {
#pragma unroll
          for (int j = 0; j < 128; j += 2) gelu_pair<32>(sum[j], sum[j + 1]);
        } else if (args.out_dtype == TJB_E4M3) {
#pragma unroll
          for (int j = 0; j < 128; j += 2) gelu_pair<8>(sum[j], sum[j + 1]);
        } else {
#pragma unroll
          for (int j = 0; j < 128; j += 2) gelu_pair<16>(sum[j], sum[j + 1]);
        }
      }
      const int row0 = m_blk * 128 + quad * 32;
      // Up to two 32-row x 128-byte pieces of this warp at a time: wait until
      // the stores that last read the buffers are done, write the rows (16-byte
      // chunk k of row l at k ^ (l & 7)), hand them to TMA.  Stored straight
      // from registers, a row per lane, the output went out at 16 bytes a clock
      // (64 KB of fp16: 4100 clocks of a K = 1024 tile's 12000).
      auto out_free = [&]() {
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
      };
      auto out_send = [&](int pieces, int col, int per_piece) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          for (int c = 0; c < pieces; ++c)
            if (col + c * per_piece < args.N)
              tma_store_2d(&tmC, buf + c * Cfg::kOutTile, col + c * per_piece, row0);
          bulk_commit();
        }
      };
      out_free();
      if (args.out_dtype == TJB_E4M3) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 128; j += 2) top = max_abs(top, sum[j], sum[j + 1]);
        const float s = block_scale(top);
        const Divisor div = divisor(s);
        uint32_t w[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) w[j] = quantize4(&sum[4 * j], div);
        stage_row(buf, lane, w);
        out_send(1, n0, 128);
        if (row0 + lane < args.M)
          args.c_scales[static_cast<int64_t>(row0 + lane) * ((args.N + kQBlock - 1) / kQBlock) +
                        n0 / kQBlock] = s;
      } else if (args.out_dtype == TJB_F32) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c == 2) {
            out_send(2, n0, 32);
            out_free();
          }
          uint32_t w[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(sum[c * 32 + j]);
          stage_row(buf + (c & 1) * Cfg::kOutTile, lane, w);
        }
        out_send(2, n0 + 64, 32);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int j = 0; j < 32; ++j)
            w[j] = args.out_dtype == TJB_BF16
                       ? Pack2<__nv_bfloat16>::pack(sum[c * 64 + 2 * j], sum[c * 64 + 2 * j + 1])
                       : Pack2<__half>::pack(sum[c * 64 + 2 * j], sum[c * 64 + 2 * j + 1]);
          stage_row(buf + c * Cfg::kOutTile, lane, w);
        }
        out_send(2, n0, 64);
      }
    }
    // Every bulk store has completed before the CTA exits.
    if (lane == 0) bulk_wait_all();
    if (!met) {  // no tile (a live-tile list with fewer): the same meetings
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  }

  __syncwarp();
  tc_fence_before();
  // (A pair: neither CTA leaves while the other or the MMAs may still touch
  // its barriers, operands or tensor memory.)
  if constexpr (kPair)
    cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (kPair)
      tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    else
      tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// Clusters of 1, 2, 4 and 8 CTAs that run at once, per device.
struct WideLimits {
  int clusters[4];
  int pairs;
  bool known;
};
WideLimits g_f8_wide[64];

int wide_limits(WideLimits& lim) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return TJB_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lock(g_f8_mu);
  WideLimits& l = g_f8_wide[dev];
  if (!l.known) {
    const uint32_t bytes[3] = {WideCfg<kWhole>::kSmemBytes, WideCfg<kSplitK>::kSmemBytes,
                               WideCfg<kPaired>::kSmemBytes};
    const decltype(&gemm_fp8_wide_kernel<kWhole>) kernels[3] = {gemm_fp8_wide_kernel<kWhole>,
                                                       gemm_fp8_wide_kernel<kSplitK>,
                                                       gemm_fp8_wide_kernel<kPaired>};
    for (int i = 0; i < 3; ++i)
      if (const int fs = cuda_status(cudaFuncSetAttribute(
              kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes[i]))))
        return fs;
    l.clusters[0] = num_sms();
    auto resident = [&](WideForm form, int log2, int* clusters) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(num_sms() >> log2 << log2));
      cfg.blockDim = dim3(WideCfg<kWhole>::kThreads);
      cfg.dynamicSmemBytes = bytes[form];
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << log2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      return cuda_status(cudaOccupancyMaxActiveClusters(clusters, kernels[form], &cfg));
    };
    for (int i = 1; i < 4; ++i)
      if (const int qs = resident(kSplitK, i, &l.clusters[i])) return qs;
    if (const int qs = resident(kPaired, 1, &l.pairs)) return qs;
    l.known = true;
  }
  lim = l;
  return TJB_OK;
}

// All tiles in pairs (pairs > 0: that many at once); or the first `whole` tiles
// in rounds of one per SM and the others, if any, with their k-blocks split over
// clusters of 1 << log2 CTAs.
int launch_wide(const void* A, const void* W, GemmF8Args args, int lda, int ldw, int pairs,
                int whole, int log2, cudaStream_t stream) {
  constexpr int kThreads = WideCfg<kWhole>::kThreads;
  CUtensorMap tmA, tmB, tmC;
  int st = make_tmap_2d(&tmA, TJB_E4M3, A, args.K, args.M, lda, kF8BK, 128);
  if (st != TJB_OK) return st;
  st = make_tmap_2d(&tmB, TJB_E4M3, W, args.K, args.N, ldw, kF8BK,
                    pairs > 0 ? 128 : 256);
  if (st != TJB_OK) return st;
  const int esz = args.out_dtype == TJB_F32 ? 4 : args.out_dtype == TJB_E4M3 ? 1 : 2;
  st = make_tmap_2d(&tmC, args.out_dtype, args.C, args.N, args.M,
                    static_cast<uint64_t>(args.ldc) * esz, 128 / esz, 32);
  if (st != TJB_OK) return st;
  const int wide_n = (args.N + 255) / 256;
  args.splits = 1;
  if (pairs > 0) {
    // (64 bits: M comes within 129 of 2^31.)
    const int tiles = static_cast<int>((args.M + INT64_C(255)) / 256) * wide_n;
    args.first_tile = 0;
    args.end_tile = tiles;
    return launch_kernel_cluster(gemm_fp8_wide_kernel<kPaired>,
                                 dim3(2u * static_cast<unsigned>(tiles < pairs ? tiles : pairs)),
                                 dim3(kThreads), WideCfg<kPaired>::kSmemBytes, stream, 2u, tmA, tmB,
                                 tmC, args);
  }
  const int tiles = (args.M + 127) / 128 * wide_n;
  const int sms = num_sms();
  if (whole > 0) {
    args.first_tile = 0;
    args.end_tile = whole;
    st = launch_kernel(gemm_fp8_wide_kernel<kWhole>, dim3(whole < sms ? whole : sms),
                       dim3(kThreads), WideCfg<kWhole>::kSmemBytes, stream, tmA, tmB, tmC, args);
    if (st != TJB_OK) return st;
  }
  if (whole < tiles) {
    args.first_tile = whole;
    args.end_tile = tiles;
    args.splits = 1 << log2;
    st = launch_kernel_cluster(gemm_fp8_wide_kernel<kSplitK>,
                               dim3(static_cast<unsigned>(tiles - whole) << log2), dim3(kThreads),
                               WideCfg<kSplitK>::kSmemBytes, stream,
                               static_cast<unsigned>(args.splits), tmA, tmB, tmC, args);
  }
  return st;
}

}  // namespace
}  // namespace tjb

extern "C" int tjb_gemm_fp8(const void* A, const float* a_scales, int64_t a_scales_row,
                            int64_t a_scales_blk, const void* W, const float* w_scales,
                            const float* bias, void* C, float* c_scales, int M, int N, int K,
                            int lda, int ldw, int ldc, int out_dtype, int act,
                            const int32_t* m_tiles, tjb_stream_t stream) {
  using namespace tjb;
  if (!A || !a_scales || !W || !w_scales || !C || M < 0 || N <= 0 || K <= 0 ||
      a_scales_row < 0 || a_scales_blk < 0)
    return TJB_ERR_INVALID_ARGUMENT;
  if (out_dtype < TJB_F32 || out_dtype > TJB_E4M3) return TJB_ERR_UNSUPPORTED_DTYPE;
  if (act != 0 && act != 1) return TJB_ERR_INVALID_ARGUMENT;
  const bool q = out_dtype == TJB_E4M3;
  if (q && !c_scales) return TJB_ERR_INVALID_ARGUMENT;
  const int unit = q ? 16 : 8;  // output columns
  const int pitch = out_dtype == TJB_F32 ? 4 : unit;  // 16 bytes
  if (K % 16 != 0 || N % unit != 0 || K > kMaxColumns || N > kMaxColumns || lda < K || ldw < K ||
      ldc < N || M > 2147483647 - kLiveTileRows)
    return TJB_ERR_BAD_SHAPE;
  auto misaligned4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; };
  if (lda % 16 != 0 || ldw % 16 != 0 || ldc % pitch != 0 || !aligned16(A) || !aligned16(W) ||
      !aligned16(C) || (bias && !aligned16(bias)) || misaligned4(a_scales) ||
      misaligned4(w_scales) || (q && misaligned4(c_scales)))
    return TJB_ERR_BAD_ALIGNMENT;
  if (!device_ok()) return TJB_ERR_NO_DEVICE;
  if (M == 0) return TJB_OK;
  GemmF8Args args = {};
  args.a_scales = a_scales;
  args.w_scales = w_scales;
  args.bias = bias;
  args.C = C;
  args.c_scales = c_scales;
  args.m_tiles = m_tiles;
  args.as_row = a_scales_row;
  args.as_blk = a_scales_blk;
  args.M = M;
  args.N = N;
  args.K = K;
  args.ldc = ldc;
  args.out_dtype = out_dtype;
  args.act = act;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Up to 64 tokens: the narrowest tile that holds them.
  if (M <= 16) return launch_skinny<16>(A, W, args, lda, ldw, s);
  if (M <= 32) return launch_skinny<32>(A, W, args, lda, ldw, s);
  if (M <= 64) return launch_skinny<64>(A, W, args, lda, ldw, s);
  // More: 64-token tiles (quick to start, their parts quick to meet, but the
  // tensor core a third as busy) or wide ones (pairs, single CTAs, or split over
  // clusters), or wide ones and the rest, by the time that each is expected to
  // take.  The constants, in us, were fitted on a B200 to shapes of M 65-16384,
  // N 128-8192, K 128-16384 with fp16 outputs and no activation (mean error 10 %
  // over 40 other shapes; the choice came within 1 % of the best of the forms on
  // average, 28 % at worst).  They know neither the output's type nor the
  // activation: against them 8-bit outputs are 11 % off on average, with GELU 19 %
  // (always slower), fp32 outputs 15 % and 31 %.
  WideLimits lim;
  if (const int st = wide_limits(lim)) return st;
  const int sms = lim.clusters[0];
  const int num_k = (K + kF8BK - 1) / kF8BK;
  const int64_t num_n = (N + 127) / 128, wide_n = (N + 255) / 256;
  const int64_t tiles = (static_cast<int64_t>(M) + 127) / 128 * wide_n;
  if (tiles > 1073741823) return TJB_ERR_BAD_SHAPE;
  auto skinny_us = [&](int64_t m) {
    const double t = static_cast<double>((m + 63) / 64 * num_n);
    return 4.3 + t * (0.0157 + 0.0024 * num_k);
  };
  auto whole_us = [&](int64_t rounds) { return 2.9 + rounds * (0.52 * num_k + 1.75); };
  // m rows in wide tiles without a split, and the pairs for it (0: single CTAs).
  auto wide_us = [&](int64_t m, int& pairs) {
    const int64_t m1 = (m + 127) / 128, m2 = (m + 255) / 256;
    const double single = whole_us((m1 * wide_n + sms - 1) / sms);
    pairs = 0;
    if (lim.pairs <= 0) return single;
    const int64_t rounds = (m2 * wide_n + lim.pairs - 1) / lim.pairs;
    const double paired = 3.4 + rounds * (0.49 * num_k + 1.7);
    if (paired >= single) return single;
    pairs = lim.pairs;
    return paired;
  };
  double best = skinny_us(M);
  enum { kSkinny, kWide, kRows } form = kSkinny;
  int whole = static_cast<int>(tiles), log2 = 0, pairs = 0;
  const double wide = wide_us(M, pairs);
  if (wide < best) {
    best = wide;
    form = kWide;
  }
  // The last, partial round: split, or its rows in 64-token tiles.
  const int64_t rounds = (tiles + sms - 1) / sms;
  const int64_t full = (rounds - 1) * sms;
  const double full_us = rounds > 1 ? whole_us(rounds - 1) : 0.0;
  for (int i = 1; i < 4 && 1 << i <= num_k && tiles - full <= lim.clusters[i]; ++i) {
    const double us = full_us + 8.9 + 0.66 * num_k / (1 << i);
    if (us < best) {
      best = us;
      form = kWide;
      pairs = 0;
      whole = static_cast<int>(full);
      log2 = i;
    }
  }
  const int64_t rows = full / wide_n * 128;  // (a live-tile list is not cut)
  if (rows > 0 && m_tiles == nullptr) {
    int rows_pairs = 0;
    if (wide_us(rows, rows_pairs) + 1.5 + skinny_us(M - rows) < best) {
      form = kRows;
      pairs = rows_pairs;
    }
  }
  if (form == kSkinny) return launch_skinny<64>(A, W, args, lda, ldw, s);
  if (form == kWide) return launch_wide(A, W, args, lda, ldw, pairs, whole, log2, s);
  const int esz = out_dtype == TJB_F32 ? 4 : q ? 1 : 2;
  args.M = static_cast<int>(rows);
  whole = static_cast<int>(rows / 128 * wide_n);
  if (const int st = launch_wide(A, W, args, lda, ldw, pairs, whole, 0, s)) return st;
  args.M = static_cast<int>(M - rows);
  args.a_scales += rows * a_scales_row;
  args.C = static_cast<uint8_t*>(C) + rows * ldc * esz;
  if (q) args.c_scales += rows * num_n;
  return launch_skinny<64>(static_cast<const uint8_t*>(A) + rows * lda, W, args, lda, ldw, s);
}
