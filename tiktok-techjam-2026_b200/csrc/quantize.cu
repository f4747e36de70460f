// quantize.cu -- fp32 / fp16 / bf16 matrices to block-scaled e4m3 (HBM-bound:
// each element is read once and one byte written).
#include <mutex>
#include <type_traits>

#include "fp8.cuh"

namespace tjb {
namespace {

constexpr int kQuantThreads = 256;
// Activations: a warp takes kSteps x 512 bytes of a row, all in flight at
// once; 32 (fp32) or 16 (16-bit) neighbouring lanes hold one block, so its
// amax is a few shuffles of values in registers.  Consecutive warps take
// consecutive columns.
// HBM-bound: 16384 x 4096 fp32 52 us, fp16 33 us (51 and 31 at the
// rate of a copy).
template <typename T, int kSteps>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q,
                         float* __restrict__ scales, int rows, int K,
                         const int32_t* __restrict__ m_tiles) {
  constexpr int kElems = Piece16<T>::kElems;       // columns per lane and step
  constexpr int kLanes = kQBlock / kElems;         // lanes per block
  constexpr int kCols = kSteps * 32 * kElems;      // columns per warp
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const unsigned segs = static_cast<unsigned>((K + kCols - 1) / kCols);
  const unsigned item = blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const unsigned row_index = item / segs;
  const int col0 = static_cast<int>(item - row_index * segs) * kCols + lane * kElems;
  int64_t row = row_index;
  if (m_tiles != nullptr) {
    const int64_t li = row / kLiveTileRows;
    if (li >= __ldg(m_tiles)) return;
    row = static_cast<int64_t>(__ldg(m_tiles + 1 + li)) * kLiveTileRows + row % kLiveTileRows;
  }
  if (row >= rows) return;
  const int kb_count = (K + kQBlock - 1) / kQBlock;
  Piece16<T> piece[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int col = col0 + i * 32 * kElems;
    if (col < K) piece[i] = load_piece16(x + row * ldx + col);
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int col = col0 + i * 32 * kElems;
    if (col - lane * kElems >= K) break;  // warp-uniform
    uint32_t top = col < K ? abs_bits(piece[i].max_abs()) : 0u;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (col < K) {
      const float s = block_scale(__uint_as_float(top));
      const Divisor div = divisor(s);
      float f[kElems];
      piece[i].widen(f);
      uint32_t b[kElems / 4];
#pragma unroll
      for (int j = 0; j < kElems / 4; ++j) b[j] = quantize4(f + 4 * j, div);
      uint8_t* dst = q + row * K + col;
      if constexpr (kElems == 8)
        *reinterpret_cast<uint2*>(dst) = make_uint2(b[0], b[1]);
      else
        *reinterpret_cast<uint32_t*>(dst) = b[0];
      if ((lane & (kLanes - 1)) == 0) scales[row * kb_count + col / kQBlock] = s;
    }
  }
}

// Weights: persistent CTAs, one 128 x 128 block at a time in registers
// between the amax and the rounding, while the next two blocks' copies into a
// three-stage shared-memory ring are in flight (a thread reads only what it
// copied itself, so the ring needs no barrier).  A CTA per block without the
// ring left HBM idle while its blocks computed: 16384 x 4096 fp32 78 us, bf16
// 65 us; with it 57 and 33 (51 and 31 at the rate of a copy).
constexpr int kRingStages = 3;

template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_tiles_kernel(const T* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q,
                          float* __restrict__ scales, int N, int K) {
  constexpr int kElems = Piece16<T>::kElems;
  constexpr int kRowPieces = kQBlock / kElems;
  constexpr int kPieces = kQBlock * kRowPieces / kQuantThreads;  // per thread and block
  extern __shared__ uint4 ring[];                                // [stage][piece][thread]
  __shared__ float s_max[2][kQuantThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kb_count = (K + kQBlock - 1) / kQBlock;
  const int tiles = (N + kQBlock - 1) / kQBlock * kb_count;
  // Piece i of this thread: row r0 + i * kRowStep of the block, columns c0 ...
  constexpr int kRowStep = kQuantThreads / kRowPieces;
  const int r0 = threadIdx.x / kRowPieces, c0 = threadIdx.x % kRowPieces * kElems;
  auto fetch = [&](int tile, int stage) {
    if (tile < tiles) {
      const int nb = tile / kb_count;
      const int col = (tile - nb * kb_count) * kQBlock + c0;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int row = nb * kQBlock + r0 + i * kRowStep;
        const bool in = row < N && col < K;
        const uint32_t dst = smem_u32(ring + (stage * kPieces + i) * kQuantThreads + threadIdx.x);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
                     "l"(in ? w + row * ldw + col : w), "r"(in ? 16 : 0)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int step = static_cast<int>(gridDim.x);
  int stage = 0, odd = 0;
  fetch(static_cast<int>(blockIdx.x), 0);
  fetch(static_cast<int>(blockIdx.x) + step, 1);
  for (int tile = static_cast<int>(blockIdx.x); tile < tiles; tile += step) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    Piece16<T> piece[kPieces];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint4 raw = ring[(stage * kPieces + i) * kQuantThreads + threadIdx.x];
      piece[i] = *reinterpret_cast<const Piece16<T>*>(&raw);
    }
    // Stage + 2 (mod 3) held the previous block, which this thread has read.
    fetch(tile + 2 * step, stage == 0 ? 2 : stage - 1);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) top = max_abs(top, piece[i].max_abs());
    top = warp_max_abs(top);
    if (lane == 0) s_max[odd][warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 32; ++i) top = max_abs(top, s_max[odd][i]);
    const float s = block_scale(top);
    const Divisor div = divisor(s);
    const int nb = tile / kb_count;
    const int col = (tile - nb * kb_count) * kQBlock + c0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = nb * kQBlock + r0 + i * kRowStep;
      float f[kElems];
      piece[i].widen(f);
      uint32_t b[kElems / 4];
#pragma unroll
      for (int j = 0; j < kElems / 4; ++j) b[j] = quantize4(f + 4 * j, div);
      if (row < N && col < K) {
        uint8_t* dst = q + static_cast<int64_t>(row) * K + col;
        if constexpr (kElems == 8)
          *reinterpret_cast<uint2*>(dst) = make_uint2(b[0], b[1]);
        else
          *reinterpret_cast<uint32_t*>(dst) = b[0];
      }
    }
    if (threadIdx.x == 0) scales[tile] = s;
    stage = stage == 2 ? 0 : stage + 1;
    odd ^= 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

std::mutex g_quant_mu;
bool g_quant_ready[64][3];

template <typename T>
int launch_quantize_tiles(const void* w, int64_t ldw, void* q, float* scales, int N, int K,
                          cudaStream_t stream) {
  constexpr int smem = kRingStages * kQBlock * kQBlock * static_cast<int>(sizeof(T));
  constexpr int slot = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 1 : 2;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return TJB_ERR_NO_DEVICE;
  {
    std::lock_guard<std::mutex> lock(g_quant_mu);
    if (!g_quant_ready[dev][slot]) {
      if (const int fs = cuda_status(cudaFuncSetAttribute(
              quantize_tiles_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)))
        return fs;
      g_quant_ready[dev][slot] = true;
    }
  }
  const int64_t tiles = static_cast<int64_t>((N + kQBlock - 1) / kQBlock) * ((K + kQBlock - 1) / kQBlock);
  const int64_t most = static_cast<int64_t>(num_sms()) * (sizeof(T) == 4 ? 1 : 2);
  return launch_kernel(quantize_tiles_kernel<T>, dim3(static_cast<unsigned>(tiles < most ? tiles : most)),
                       dim3(kQuantThreads), smem, stream, static_cast<const T*>(w), ldw,
                       static_cast<uint8_t*>(q), scales, N, K);
}

int check_quantize(const void* x, int64_t ldx, int in_dtype, const void* q, const float* scales,
                   int64_t rows, int K) {
  if (!x || !q || !scales || rows < 0 || K <= 0) return TJB_ERR_INVALID_ARGUMENT;
  if (in_dtype < TJB_F32 || in_dtype > TJB_BF16) return TJB_ERR_UNSUPPORTED_DTYPE;
  if (K % 16 != 0 || K > kMaxColumns || ldx < K || rows > 2147483647 - kLiveTileRows)
    return TJB_ERR_BAD_SHAPE;
  // Rows start on 16-byte boundaries.
  if (!aligned16(x) || ldx % (in_dtype == TJB_F32 ? 4 : 8) != 0 || !aligned16(q) ||
      (reinterpret_cast<uintptr_t>(scales) & 3u) != 0)
    return TJB_ERR_BAD_ALIGNMENT;
  return TJB_OK;
}

}  // namespace
}  // namespace tjb

extern "C" int tjb_quantize_blocks(const void* x, int64_t ldx, int in_dtype, void* q,
                                   float* scales, int64_t rows, int K, const int32_t* m_tiles,
                                   tjb_stream_t stream) {
  using namespace tjb;
  if (const int st = check_quantize(x, ldx, in_dtype, q, scales, rows, K)) return st;
  const int kb_count = (K + kQBlock - 1) / kQBlock;
  // With a tile list rows are numbered over whole 128-row tiles.
  const int64_t n =
      m_tiles ? (rows + kLiveTileRows - 1) / kLiveTileRows * kLiveTileRows : rows;
  if (n * kb_count > 2147483647) return TJB_ERR_BAD_SHAPE;
  if (!device_ok()) return TJB_ERR_NO_DEVICE;
  if (rows == 0) return TJB_OK;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    constexpr int kSteps = 4;
    constexpr int cols = kSteps * 32 * Piece16<T>::kElems;
    constexpr int warps = kQuantThreads / 32;
    const int64_t items = n * ((K + cols - 1) / cols);
    return launch_kernel(quantize_rows_kernel<T, kSteps>,
                         dim3(static_cast<unsigned>((items + warps - 1) / warps)),
                         dim3(kQuantThreads), 0, reinterpret_cast<cudaStream_t>(stream),
                         static_cast<const T*>(x), ldx, static_cast<uint8_t*>(q), scales,
                         static_cast<int>(rows), K, m_tiles);
  };
  if (in_dtype == TJB_F32) return go(float{});
  return in_dtype == TJB_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

extern "C" int tjb_quantize_weight_blocks(const void* w, int64_t ldw, int in_dtype, void* q,
                                          float* scales, int64_t N, int K, tjb_stream_t stream) {
  using namespace tjb;
  if (const int st = check_quantize(w, ldw, in_dtype, q, scales, N, K)) return st;
  if (((N + kQBlock - 1) / kQBlock) * ((K + kQBlock - 1) / kQBlock) > 1073741823)
    return TJB_ERR_BAD_SHAPE;
  if (!device_ok()) return TJB_ERR_NO_DEVICE;
  if (N == 0) return TJB_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int n = static_cast<int>(N);
  if (in_dtype == TJB_F32) return launch_quantize_tiles<float>(w, ldw, q, scales, n, K, st);
  if (in_dtype == TJB_F16) return launch_quantize_tiles<__half>(w, ldw, q, scales, n, K, st);
  return launch_quantize_tiles<__nv_bfloat16>(w, ldw, q, scales, n, K, st);
}
