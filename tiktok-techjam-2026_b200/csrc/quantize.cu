// quantize.cu -- fp32 / fp16 / bf16 matrices to block-scaled e4m3 (HBM-bound:
// each element is read once and one byte written).
#include "fp8.cuh"

namespace tjb {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantSeg = 4;  // blocks of 128 columns a warp has in flight

// Activations: one warp per (row, kQuantSeg consecutive blocks); lane l of
// the warp holds columns 4l .. 4l+3 of each block, so a block's amax is one
// warp-wide integer maximum and its bytes leave as one 128-byte line.
template <bool k16>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, bool bf16,
                         uint8_t* __restrict__ q, float* __restrict__ scales, int rows, int K,
                         const int32_t* __restrict__ m_tiles) {
  griddep_wait();
  griddep_launch_dependents();
  const int kb_count = (K + kQBlock - 1) / kQBlock;
  const int segs = (kb_count + kQuantSeg - 1) / kQuantSeg;
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + (threadIdx.x >> 5);
  int64_t row = item / segs;
  const int kb0 = static_cast<int>(item - row * segs) * kQuantSeg;
  if (m_tiles != nullptr) {
    const int64_t li = row / kLiveTileRows;
    if (li >= __ldg(m_tiles)) return;
    row = static_cast<int64_t>(__ldg(m_tiles + 1 + li)) * kLiveTileRows + row % kLiveTileRows;
  }
  if (row >= rows) return;
  Raw4<k16> raw[kQuantSeg];
#pragma unroll
  for (int i = 0; i < kQuantSeg; ++i) {
    const int col = (kb0 + i) * kQBlock + lane * 4;
    if (col < K) raw[i] = load_raw4<k16>(x, row * ldx + col);
  }
#pragma unroll
  for (int i = 0; i < kQuantSeg; ++i) {
    if (kb0 + i >= kb_count) break;  // warp-uniform
    const int col = (kb0 + i) * kQBlock + lane * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < K) v = widen4<k16>(raw[i], bf16);
    const float s = block_scale(__reduce_max_sync(0xffffffffu, abs_bits4(v)));
    if (col < K) *reinterpret_cast<uint32_t*>(q + row * K + col) = quantize4(v, s);
    if (lane == 0) scales[row * kb_count + kb0 + i] = s;
  }
}

// Weights: one CTA per 128 x 128 block, held in registers between the amax
// and the rounding; warp w holds rows w, w + 8, ...
template <bool k16>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_tiles_kernel(const void* __restrict__ w, int64_t ldw, bool bf16,
                          uint8_t* __restrict__ q, float* __restrict__ scales, int N, int K) {
  constexpr int kWarps = kQuantThreads / 32;
  constexpr int kRows = kQBlock / kWarps;
  __shared__ uint32_t s_max[kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kb_count = (K + kQBlock - 1) / kQBlock;
  const int nb = blockIdx.x / kb_count, kb = blockIdx.x - nb * kb_count;
  const int col = kb * kQBlock + lane * 4;
  const int64_t row0 = static_cast<int64_t>(nb) * kQBlock + warp;
  Raw4<k16> raw[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (row0 + i * kWarps < N && col < K)
      raw[i] = load_raw4<k16>(w, (row0 + i * kWarps) * ldw + col);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (row0 + i * kWarps < N && col < K) top = max(top, abs_bits4(widen4<k16>(raw[i], bf16)));
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) top = max(top, s_max[i]);
  const float s = block_scale(top);
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (row0 + i * kWarps < N && col < K)
      *reinterpret_cast<uint32_t*>(q + (row0 + i * kWarps) * K + col) =
          quantize4(widen4<k16>(raw[i], bf16), s);
  if (threadIdx.x == 0) scales[blockIdx.x] = s;
}

int check_quantize(const void* x, int64_t ldx, int in_dtype, const void* q, const float* scales,
                   int64_t rows, int K) {
  if (!x || !q || !scales || rows < 0 || K <= 0) return TJB_ERR_INVALID_ARGUMENT;
  if (in_dtype < TJB_F32 || in_dtype > TJB_BF16) return TJB_ERR_UNSUPPORTED_DTYPE;
  if (K % 16 != 0 || ldx < K || rows > 2147483647 - kLiveTileRows) return TJB_ERR_BAD_SHAPE;
  const uintptr_t vec = in_dtype == TJB_F32 ? 15u : 7u;  // four elements a load
  if ((reinterpret_cast<uintptr_t>(x) & vec) != 0 || ldx % 4 != 0 || !aligned16(q) ||
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
  const int64_t segs = (kb_count + kQuantSeg - 1) / kQuantSeg;
  // With a tile list rows are numbered over whole 128-row tiles.
  const int64_t n =
      m_tiles ? (rows + kLiveTileRows - 1) / kLiveTileRows * kLiveTileRows : rows;
  const int64_t grid = (n * segs + kQuantThreads / 32 - 1) / (kQuantThreads / 32);
  if (grid > 2147483647) return TJB_ERR_BAD_SHAPE;
  if (!device_ok()) return TJB_ERR_NO_DEVICE;
  if (rows == 0) return TJB_OK;
  auto go = [&](auto kern) {
    return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(kQuantThreads), 0,
                         reinterpret_cast<cudaStream_t>(stream), x, ldx, in_dtype == TJB_BF16,
                         static_cast<uint8_t*>(q), scales, static_cast<int>(rows), K, m_tiles);
  };
  return in_dtype == TJB_F32 ? go(quantize_rows_kernel<false>) : go(quantize_rows_kernel<true>);
}

extern "C" int tjb_quantize_weight_blocks(const void* w, int64_t ldw, int in_dtype, void* q,
                                          float* scales, int64_t N, int K, tjb_stream_t stream) {
  using namespace tjb;
  if (const int st = check_quantize(w, ldw, in_dtype, q, scales, N, K)) return st;
  const int64_t grid = ((N + kQBlock - 1) / kQBlock) * ((K + kQBlock - 1) / kQBlock);
  if (grid > 2147483647) return TJB_ERR_BAD_SHAPE;
  if (!device_ok()) return TJB_ERR_NO_DEVICE;
  if (N == 0) return TJB_OK;
  auto go = [&](auto kern) {
    return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(kQuantThreads), 0,
                         reinterpret_cast<cudaStream_t>(stream), w, ldw, in_dtype == TJB_BF16,
                         static_cast<uint8_t*>(q), scales, static_cast<int>(N), K);
  };
  return in_dtype == TJB_F32 ? go(quantize_tiles_kernel<false>) : go(quantize_tiles_kernel<true>);
}
