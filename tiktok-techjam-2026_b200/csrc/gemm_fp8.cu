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
  bool wide_stores;  // C and its rows start on 32-byte boundaries
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
        const float s = block_scale(warp_max_abs(max_abs4(v)));
        if (n < args.N)
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(args.C) + m * args.ldc + n) =
              quantize4(v, s, reciprocal(s));
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

// ------------------------------------------------------------------------
// Many tokens: 128 x 256 tiles of C per CTA (with CTAS = 2 a CTA pair shares
// the MMAs of a 256 x 256 tile, CTA r holding token rows 128 r .. of it and
// 128 of its 256 weight rows).  Here the tokens are the MMA's rows: a thread
// owns one token and 128 consecutive output columns, which is one weight
// block (one scale product per k-block) and one output block (its 8-bit scale
// needs no exchange).  Persistent, 384 threads:
//   warp 0        TMA producer
//   warp 1        MMA issuer (leader CTA): per k-block four K = 32 MMAs into
//                 one of two 256-column TMEM accumulators
//   warps 2, 3    products sa[m, kb] sw[n / 128, kb] of the tile's rows, eight
//                 k-blocks at a time, a ring slot ahead of their use
//   warps 4..11   two warp groups, 128 columns each: read P_kb from TMEM in
//                 16-column pieces, the next in flight while one is added to
//                 128 fp32 sums in registers; then GELU, rounding, and 32-byte
//                 stores (a thread holds 128 consecutive values of a row)
// Per k-block and SM the tensor core takes 512 clocks (128 x 256 x 128 at
// 8192 products a clock), the multiply-adds 280 (packed pairs, two clocks a
// warp).  What bounds it is the chain MMA -> barrier -> scaling -> barrier ->
// MMA over the two accumulators: every barrier operation, load and spilled
// register in the k-loop adds to it.  The scaling threads need the registers
// that warps 0-3 give up (128 x 72 + 256 x 216 = 384 x 168 at launch).
template <int CTAS>
struct WideCfg {
  static constexpr int kStages = CTAS == 2 ? 6 : 4;
  static constexpr int kThreads = 384;
  static constexpr int kBRows = 256 / CTAS;       // weight rows a CTA holds per stage
  static constexpr uint32_t kABytes = 128 * kF8BK;
  static constexpr uint32_t kBBytes = kBRows * kF8BK;
  static constexpr uint32_t kTmemCols = 512;      // two 256-column accumulators
  static constexpr int kChunk = 8;                // k-blocks of scale products per ring slot
  static constexpr uint32_t kScaleBytes = 2 * kChunk * 256 * 4;
  static constexpr uint32_t kSmemBytes =
      1024 + kStages * (kABytes + kBBytes) + kScaleBytes + 256;
};

__device__ __forceinline__ void umma_e4m3_pair_w(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                                 uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on an mbarrier of another CTA of the cluster to hand back tensor
// memory that this thread has finished reading.  The reads are complete and
// ordered by tcgen05.fence, and no other memory is handed over, so the arrive
// needs no release at cluster scope (whose fence, once per k-block, made the
// kernel wait 4x the MMA time: 8192 x 4096 x 4096 328 us).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t remote_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}

template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// 32 consecutive bytes of a row of which `cols` elements (per16 to 16 bytes)
// exist; one 32-byte store where the matrix allows it (a thread holds a row,
// so narrower stores would write each 32-byte sector twice).
__device__ __forceinline__ void store32(void* dst, const uint32_t (&w)[8], int cols, int per16,
                                        bool wide) {
  if (wide && cols >= 2 * per16) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
    return;
  }
  uint4* p = static_cast<uint4*>(dst);
  if (cols >= per16) p[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if (cols >= 2 * per16) p[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

template <int CTAS>
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                     uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    umma_e4m3_pair_w(d_tmem, adesc, bdesc, idesc, accumulate);
  else
    umma_e4m3_w(d_tmem, adesc, bdesc, idesc, accumulate);
}

template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CTAS == 2)
    umma_commit_pair_w(bar, 0x3);
  else
    umma_commit_w(bar);
}

// sum[0..15] += s * p[0..15]
__device__ __forceinline__ void add_scaledN(float* sum, const uint32_t* p, float s) {
#pragma unroll
  for (int j = 0; j < 16; j += 2)
    fma2v(sum[j], sum[j + 1], __uint_as_float(p[j]), __uint_as_float(p[j + 1]), s, s, sum[j],
          sum[j + 1]);
}

template <int CTAS>
__global__ void __launch_bounds__(WideCfg<CTAS>::kThreads, 1)
    gemm_fp8_wide_kernel(const __grid_constant__ CUtensorMap tmA,
                         const __grid_constant__ CUtensorMap tmB,
                         const GemmF8Args args) {
  using Cfg = WideCfg<CTAS>;
  constexpr bool kPair = CTAS == 2;
  constexpr int kStages = Cfg::kStages, kChunk = Cfg::kChunk;
  constexpr int BN = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kStages * Cfg::kABytes;
  float* sScale = reinterpret_cast<float*>(sB + kStages * Cfg::kBBytes);  // [slot][k-block][half][row]
  uint64_t* full = reinterpret_cast<uint64_t*>(sScale + 2 * kChunk * 256);  // leader's are used
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;  // leader's are used
  uint64_t* sfull = tempty + 2;
  uint64_t* sempty = sfull + 2;
  uint64_t* drain = sempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_ctarank() : 0u;  // 0: the leader, which issues the MMAs

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);   // the leader's expect-tx arrival + both CTAs' bytes
      mbar_init(&empty[s], 1);  // one commit of the leader's MMAs to both CTAs
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8 * CTAS);  // eight scaling warps of each CTA
      mbar_init(&sfull[b], 2);  // warps 2 and 3
      mbar_init(&sempty[b], 8);  // the scaling warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
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
  // Both CTAs' barriers are initialised and their tensor memory allocated
  // before either signals the other.
  if constexpr (kPair)
    cluster_sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  const int num_m = args.m_tiles != nullptr ? __ldg(args.m_tiles) : (args.M + 127) / 128;
  const int num_mp = (num_m + CTAS - 1) / CTAS;
  const int num_n = (args.N + BN - 1) / BN;
  const int num_k = (args.K + kF8BK - 1) / kF8BK;
  const int num_tiles = num_mp * num_n;
  const int first = static_cast<int>(blockIdx.x) / CTAS;
  const int step = static_cast<int>(gridDim.x) / CTAS;
  // This CTA's 128 token rows of pair tile t.  A pair whose second 128-row
  // tile does not exist loads the first one's rows again (the MMA needs both
  // halves) and its second CTA stores nothing.
  auto coords = [&](int t, int& m_blk, int& n_blk) {
    int mp;
    tile_coords(t, num_mp, num_n, mp, n_blk);
    int mt = CTAS * mp + static_cast<int>(rank);
    const bool has = mt < num_m;
    if (!has) mt = CTAS * mp;
    m_blk = args.m_tiles != nullptr ? __ldg(args.m_tiles + 1 + mt) : mt;
    return has;
  };

  if (warp < 4) {
    regs_dec<72>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ producer
      const uint32_t full_leader = kPair ? map_to_rank(smem_u32(full), 0) : 0u;
      int stage = 0;
      uint32_t phase = 0, issued = 0, last_parity = 0;
      bool ok = true;
      for (int t = first; ok && t < num_tiles; t += step) {
        int m_blk, n_blk;
        coords(t, m_blk, n_blk);
        for (int kb = 0; kb < num_k; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          if (rank == 0)
            mbar_arrive_expect_tx(&full[stage], CTAS * (Cfg::kABytes + Cfg::kBBytes));
          uint8_t* a = sA + stage * Cfg::kABytes;
          uint8_t* b = sB + stage * Cfg::kBBytes;
          const int brow = n_blk * BN + static_cast<int>(rank) * Cfg::kBRows;
          if constexpr (kPair) {
            const uint32_t bar = full_leader + static_cast<uint32_t>(stage) * 8u;
            tma_load_2d_pair(a, &tmA, bar, kb * kF8BK, m_blk * 128);
            tma_load_2d_pair(b, &tmB, bar, kb * kF8BK, brow);
          } else {
            tma_load_2d(a, &tmA, &full[stage], kb * kF8BK, m_blk * 128);
            tma_load_2d(b, &tmB, &full[stage], kb * kF8BK, brow);
          }
          issued |= 1u << stage;
          last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // Every load this CTA issued has landed once the MMAs that read it
      // have released its stage (the loads count on the leader's barrier).
      for (int s = 0; s < kStages; ++s)
        if ((issued >> s) & 1u) mbar_wait_drain(&empty[s], (last_parity >> s) & 1u);
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------- MMA issuer (leader only)
      constexpr uint32_t idesc = idesc_e4m3(128 * CTAS, BN);
      int stage = 0;
      uint32_t phase = 0, it = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
      };
      for (int t = first; ok && t < num_tiles; t += step) {
        for (int kb = 0; kb < num_k; ++kb, ++it) {
          const uint32_t acc = it & 1;
          if (!wait(&full[stage], phase) || !wait(&tempty[acc], ((it >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * Cfg::kABytes);
          const uint32_t b0 = smem_u32(sB + stage * Cfg::kBBytes);
#pragma unroll
          for (int k = 0; k < kF8BK / 32; ++k)
            umma<CTAS>(tmem_base + acc * BN, sdesc_sw128(a0 + k * 32, 16, 1024),
                       sdesc_sw128(b0 + k * 32, 16, 1024), idesc, k > 0 ? 1u : 0u);
          commit<CTAS>(&tfull[acc]);
          commit<CTAS>(&empty[stage]);
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
      // --------------------------------------------------------- scale products
      // Warps 2 and 3 take 64 rows each, two per lane.
      const int num_nb = (args.N + kQBlock - 1) / kQBlock;
      const int r = (warp - 2) * 64 + lane;
      // Row-major scales whose rows start on 16-byte boundaries: four at a time.
      const bool vec = args.as_blk == 1 && args.as_row % 4 == 0 &&
                       (reinterpret_cast<uintptr_t>(args.a_scales) & 15u) == 0;
      uint32_t c = 0;
      bool ok = true;
      for (int t = first; ok && t < num_tiles; t += step) {
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
        for (int kb0 = 0; ok && kb0 < num_k; kb0 += kChunk, ++c) {
          float va[kChunk], vb[kChunk], s0[kChunk], s1[kChunk];
          if (vec && kb0 + kChunk <= num_k) {
#pragma unroll
            for (int u = 0; u < kChunk; u += 4) {
              *reinterpret_cast<float4*>(va + u) = __ldg(reinterpret_cast<const float4*>(a0 + kb0 + u));
              *reinterpret_cast<float4*>(vb + u) = __ldg(reinterpret_cast<const float4*>(a1 + kb0 + u));
            }
#pragma unroll
            for (int u = 0; u < kChunk; ++u) {
              s0[u] = __ldg(w0 + kb0 + u);
              s1[u] = __ldg(w1 + kb0 + u);
            }
          } else {
#pragma unroll
            for (int u = 0; u < kChunk; ++u) {
              const int kb = min(kb0 + u, num_k - 1);
              va[u] = __ldg(a0 + kb * args.as_blk);
              vb[u] = __ldg(a1 + kb * args.as_blk);
              s0[u] = __ldg(w0 + kb);
              s1[u] = __ldg(w1 + kb);
            }
          }
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&sempty[c & 1], ((c >> 1) & 1) ^ 1, abort_flag));
          float* dst = sScale + (c & 1) * kChunk * 256 + r;
#pragma unroll
          for (int u = 0; u < kChunk; ++u) {
            dst[u * 256] = va[u] * s0[u];
            dst[u * 256 + 32] = vb[u] * s0[u];
            dst[u * 256 + 128] = va[u] * s1[u];
            dst[u * 256 + 160] = vb[u] * s1[u];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[c & 1]);
        }
      }
    }
  } else {
    regs_inc<216>();
    // ------------------------------------------------- scaling and output
    const int quad = warp & 3;         // TMEM lanes this warp may access
    const int half = (warp - 4) >> 2;  // 128-column half of the tile
    const int r = quad * 32 + lane;    // token row of the tile
    const uint32_t tempty_leader = kPair ? map_to_rank(smem_u32(tempty), 0) : 0u;
    const uint32_t taddr0 =
        tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 128);
    uint32_t it = 0, chunk = 0;  // k-blocks and scale chunks done, over all tiles
    bool ok = true;
    for (int t = first; ok && t < num_tiles; t += step) {
      int m_blk, n_blk;
      const bool has_rows = coords(t, m_blk, n_blk);
      const int n0 = n_blk * BN + half * 128;
      // The sums start from the bias; columns past N stay exactly zero (their
      // weight rows load as zeros), as a ragged 8-bit block's scale needs.
      float sum[128];
#pragma unroll
      for (int j = 0; j < 128; j += 4) {
        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (args.bias != nullptr && n0 + j < args.N)
          b = __ldg(reinterpret_cast<const float4*>(args.bias + n0 + j));
        sum[j] = b.x;
        sum[j + 1] = b.y;
        sum[j + 2] = b.z;
        sum[j + 3] = b.w;
      }
#pragma unroll 1
      for (int kb = 0; kb < num_k; ++kb, ++it) {
        const int u = kb & (kChunk - 1);
        if (u == 0) ok = mbar_wait(&sfull[chunk & 1], (chunk >> 1) & 1, abort_flag) && ok;
        const float s = sScale[((chunk & 1) * kChunk + u) * 256 + half * 128 + r];
        const uint32_t acc = it & 1;
        ok = mbar_wait(&tfull[acc], (it >> 1) & 1, abort_flag) && ok;
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
            mbar_arrive_remote(tempty_leader + acc * 8u);
          else
            mbar_arrive(&tempty[acc]);
          if (u == kChunk - 1 || kb == num_k - 1) mbar_arrive(&sempty[chunk & 1]);
        }
        if (u == kChunk - 1 || kb == num_k - 1) ++chunk;
        add_scaledN(sum + 128 - 16, p[1], s);
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (!has_rows || n0 >= args.N) continue;  // warp-uniform
      if (args.act == 1) {
#pragma unroll
        for (int j = 0; j < 128; ++j) sum[j] = gelu_erf(sum[j]);
      }
      const int64_t row = static_cast<int64_t>(m_blk) * 128 + r;
      if (row >= args.M) continue;
      const int cols = min(args.N - n0, 128);
      if (args.out_dtype == TJB_E4M3) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 128; ++j) top = max_abs(top, sum[j]);
        const float s = block_scale(top);
        const float inv = reciprocal(s);
        args.c_scales[row * ((args.N + kQBlock - 1) / kQBlock) + n0 / kQBlock] = s;
        uint8_t* dst = static_cast<uint8_t*>(args.C) + row * args.ldc + n0;
#pragma unroll
        for (int j = 0; j < 128; j += 32) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = quantize4(&sum[j + 4 * i], s, inv);
          store32(dst + j, w, cols - j, 16, args.wide_stores);
        }
      } else if (args.out_dtype == TJB_F32) {
        float* dst = static_cast<float*>(args.C) + row * args.ldc + n0;
#pragma unroll
        for (int j = 0; j < 128; j += 8) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(sum[j + i]);
          store32(dst + j, w, cols - j, 4, args.wide_stores);
        }
      } else {
        uint16_t* dst = static_cast<uint16_t*>(args.C) + row * args.ldc + n0;
#pragma unroll
        for (int j = 0; j < 128; j += 16) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = args.out_dtype == TJB_BF16
                       ? Pack2<__nv_bfloat16>::pack(sum[j + 2 * i], sum[j + 2 * i + 1])
                       : Pack2<__half>::pack(sum[j + 2 * i], sum[j + 2 * i + 1]);
          store32(dst + j, w, cols - j, 8, args.wide_stores);
        }
      }
    }
  }

  // Neither CTA releases its tensor memory (or exits) while the leader's
  // MMAs or the peer's scaling warps may still touch the pair's resources.
  __syncwarp();
  tc_fence_before();
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

int g_f8_wide[64][2];  // co-resident clusters per device and form (0: not yet known)

template <int CTAS>
int wide_resident(int& clusters) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return TJB_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lock(g_f8_mu);
  int& known = g_f8_wide[dev][CTAS - 1];
  if (known == 0) {
    if (const int fs = cuda_status(cudaFuncSetAttribute(
            gemm_fp8_wide_kernel<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
            static_cast<int>(WideCfg<CTAS>::kSmemBytes))))
      return fs;
    int n = num_sms();
    if (CTAS == 2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * (num_sms() / 2));
      cfg.blockDim = dim3(WideCfg<CTAS>::kThreads);
      cfg.dynamicSmemBytes = WideCfg<CTAS>::kSmemBytes;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (const int qs = cuda_status(
              cudaOccupancyMaxActiveClusters(&n, gemm_fp8_wide_kernel<CTAS>, &cfg)))
        return qs;
    }
    known = n > 0 ? n : -1;
  }
  clusters = known;
  return clusters > 0 ? TJB_OK : TJB_ERR_LAUNCH;
}

template <int CTAS>
int launch_wide(const void* A, const void* W, GemmF8Args args, int lda, int ldw,
                cudaStream_t stream) {
  using Cfg = WideCfg<CTAS>;
  int clusters = 0;
  if (const int st = wide_resident<CTAS>(clusters)) return st;
  CUtensorMap tmA, tmB;
  int st = make_tmap_2d(&tmA, TJB_E4M3, A, args.K, args.M, lda, kF8BK, 128);
  if (st != TJB_OK) return st;
  st = make_tmap_2d(&tmB, TJB_E4M3, W, args.K, args.N, ldw, kF8BK, Cfg::kBRows);
  if (st != TJB_OK) return st;
  const int64_t esz = args.out_dtype == TJB_F32 ? 4 : args.out_dtype == TJB_E4M3 ? 1 : 2;
  args.wide_stores = ((reinterpret_cast<uintptr_t>(args.C) | (args.ldc * esz)) & 31) == 0;
  const int64_t m_tiles = (static_cast<int64_t>(args.M) + 127) / 128;
  const int64_t tiles = (m_tiles + CTAS - 1) / CTAS * ((args.N + 255) / 256);
  if (tiles > 2147483647) return TJB_ERR_BAD_SHAPE;
  const int n = tiles < clusters ? static_cast<int>(tiles) : clusters;
  return launch_kernel_cluster(gemm_fp8_wide_kernel<CTAS>, dim3(CTAS * n), dim3(Cfg::kThreads),
                               Cfg::kSmemBytes, stream, static_cast<unsigned>(CTAS), tmA, tmB, args);
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
  const int64_t tiles = ((static_cast<int64_t>(M) + 127) / 128) * ((N + 255) / 256);
  if (tiles * 2 >= num_sms()) return launch_wide<1>(A, W, args, lda, ldw, s);
  return launch_skinny<128>(A, W, args, lda, ldw, s);
}
