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
// Tokens per tile, BT = 16 .. 128: the weights are the MMA's 128-row operand
// (TMEM lane = output column n) and the tokens its N operand, so a few tokens
// cost a narrow MMA and not a padded one.  The k-blocks of a tile are divided
// over the CTAs of a cluster (so that enough SMs stream the weights), whose
// fp32 sums meet in distributed shared memory: CTA r finishes the tokens
// t = r mod c, adding the CTAs' parts in a fixed order.
//   warp 0      TMA producer: 128 x 128-byte weight and BT x 128-byte token
//               tiles (128-byte swizzle; one k-block) into a stage ring
//   warp 1      owns tensor memory, issues the MMAs
//   warps 2..   scaling: one TMEM lane (one n) per thread, BT tokens (64 of
//               128 in each of two warp groups)
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
};

template <int BT>
struct SkinnyCfg {
  static constexpr int kGroups = BT >= 64 ? 2 : 1;  // scaling warp groups
  static constexpr int kCols = BT / kGroups;        // tokens per scaling thread
  static constexpr int kThreads = 64 + 128 * kGroups;
  static constexpr int kAccs = BT == 128 ? 2 : 4;  // TMEM accumulators in flight
  static constexpr uint32_t kTmemCols = kAccs * BT;
  // Below 128 tokens two CTAs fit an SM (twice the loads in flight).
  static constexpr int kStages = BT == 16 ? 5 : (BT == 64 ? 3 : 4);
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

template <int kThreads>
__device__ __forceinline__ void scaling_warps_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
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
  griddep_wait();
  griddep_launch_dependents();

  // This cluster's tile: 128 output columns, BT tokens from t0.
  constexpr int kPerLive = kLiveTileRows / BT;
  const int t_tiles = args.m_tiles != nullptr
                          ? (args.M + kLiveTileRows - 1) / kLiveTileRows * kPerLive
                          : (args.M + BT - 1) / BT;
  const int n_blk = tile / t_tiles;
  const int tt = tile - n_blk * t_tiles;
  int t0 = tt * BT;
  bool live = true;
  if (args.m_tiles != nullptr) {
    const int li = tt / kPerLive;
    live = li < __ldg(args.m_tiles);
    if (live) t0 = __ldg(args.m_tiles + 1 + li) * kLiveTileRows + (tt % kPerLive) * BT;
  }
  const int tokens = live ? min(BT, args.M - t0) : 0;  // may be <= 0: nothing to do
  const int kb_count = (args.K + kF8BK - 1) / kF8BK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * kb_count / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * kb_count / splits);
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
      const uint32_t w0 = smem_u32(sW + stage * Cfg::kWBytes);
      const uint32_t x0 = smem_u32(sX + stage * Cfg::kXBytes);
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BT);
#pragma unroll
      for (int k = 0; k < kF8BK / 32; ++k)
        umma_e4m3_w(d_tmem, sdesc_sw128(w0 + k * 32, 16, 1024), sdesc_sw128(x0 + k * 32, 16, 1024),
                    idesc, k > 0 ? 1u : 0u);
      umma_commit_w(&empty[stage]);
      umma_commit_w(&tfull[acc]);
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
    const uint32_t mine = smem_u32(sEx) +
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
      v.x += bias.x;
      v.y += bias.y;
      v.z += bias.z;
      v.w += bias.w;
      if (args.act == 1) {
        v.x = gelu_erf(v.x);
        v.y = gelu_erf(v.y);
        v.z = gelu_erf(v.z);
        v.w = gelu_erf(v.w);
      }
      if (args.out_dtype == TJB_E4M3) {
        if (n >= args.N) v = make_float4(0.f, 0.f, 0.f, 0.f);
        const float s = block_scale(__reduce_max_sync(0xffffffffu, abs_bits4(v)));
        if (n < args.N)
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(args.C) + m * args.ldc + n) =
              quantize4(v, s);
        if (lane == 0)
          args.c_scales[m * ((args.N + kQBlock - 1) / kQBlock) + n_blk] = s;
      } else if (n < args.N) {
        store4(args.C, args.out_dtype, m * args.ldc + n, v);
      }
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
bool g_f8_ready[64][4];

template <int BT>
int launch_skinny(const void* A, const void* W, GemmF8Args args, int lda, int ldw,
                  cudaStream_t stream) {
  using Cfg = SkinnyCfg<BT>;
  constexpr int kSlot = BT == 16 ? 0 : BT == 32 ? 1 : BT == 64 ? 2 : 3;
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
  // As many CTAs per tile as the SMs have room for, at most one per k-block.
  const int64_t slots = static_cast<int64_t>(num_sms()) * (BT < 128 ? 2 : 1);
  const int kb_count = (args.K + kF8BK - 1) / kF8BK;
  args.splits = 1;
  while (args.splits < 8 && 2 * args.splits <= kb_count && tiles * 2 * args.splits <= slots)
    args.splits *= 2;
  const int64_t grid = tiles * args.splits;
  if (grid > 2147483647) return TJB_ERR_BAD_SHAPE;
  return launch_kernel_cluster(gemm_fp8_skinny_kernel<BT>, dim3(static_cast<unsigned>(grid)),
                               dim3(Cfg::kThreads), Cfg::kSmemBytes, stream,
                               static_cast<unsigned>(args.splits), tmW, tmX, args);
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
  const int unit = q ? 16 : 8;  // output columns: whole 16-byte pieces
  if (K % 16 != 0 || N % unit != 0 || lda < K || ldw < K || ldc < N ||
      M > 2147483647 - kLiveTileRows)
    return TJB_ERR_BAD_SHAPE;
  auto misaligned4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) != 0; };
  if (lda % 16 != 0 || ldw % 16 != 0 || ldc % unit != 0 || !aligned16(A) || !aligned16(W) ||
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
  // The narrowest tile that holds every token.
  if (M <= 16) return launch_skinny<16>(A, W, args, lda, ldw, s);
  if (M <= 32) return launch_skinny<32>(A, W, args, lda, ldw, s);
  if (M <= 64) return launch_skinny<64>(A, W, args, lda, ldw, s);
  return launch_skinny<128>(A, W, args, lda, ldw, s);
}
