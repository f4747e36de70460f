// rmsnorm.cu -- residual addition + root-mean-square norm (HBM-bound).
//
//   x = res + delta (fp32),  out = x * rsqrt(mean(x^2) + eps) * w
// The new residual is x rounded once to the residual's type; the norm reads
// the unrounded fp32 sum.  The output is f32 / f16 / bf16, or e4m3 with one
// scale for each row and 128 columns.
//
// One row is owned by TPR threads that hold up to four chunks of it in
// registers, from one read.  Two kernels: 16-byte accesses of eight columns
// where the residual is 16-bit, the delta absent or of its type and all
// pointers are 16-byte aligned, and chunks of four columns for every other
// case.  Consecutive threads take consecutive chunks, so a scale block of 128
// columns is half a warp or a warp, and its amax an integer maximum of values
// already in registers.
#include <type_traits>

#include "fp8.cuh"

namespace tjb {
namespace {

// Row chunks a thread holds (d <= 16 TPR, or 32 TPR with eight columns).  Four
// keep a thread at 40 to 64 registers: what counts is the bytes that all
// threads of an SM have in flight.  Eight chunks of four columns, weights
// fetched ahead of the sum, or a persistent block with the next row in flight
// lost more by the threads they cost (65536 x 4096, fp32 + fp16 to 8 bits:
// 432 us, 436 and 610).
constexpr int kRmsChunks = 4;

// Sum over the TPR threads of a row; every thread of the block calls it.
template <int TPR>
__device__ __forceinline__ float rms_row_sum(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += scratch[warp / kWarps * kWarps + i];
  }
  return v;
}

// kDelta: 0 none, 1 fp32, 2 sixteen bits.
template <int TPR, bool kRes16, int kDelta>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
    add_rmsnorm_kernel(const void* res, const void* delta, void* res_out, void* out,
                       float* __restrict__ out_scales, const float* __restrict__ w, int rows,
                       int d, float eps, int res_dtype, int delta_dtype, int out_dtype,
                       const uint8_t* __restrict__ row_mask,
                       const int32_t* __restrict__ m_tiles) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  constexpr int kRowsPerBlock = BLOCK / TPR;
  __shared__ float scratch[BLOCK / 32];
  const int t = threadIdx.x % TPR;
  griddep_wait();
  griddep_launch_dependents();
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + threadIdx.x / TPR;
  if (m_tiles != nullptr) {
    // Rows are numbered over the listed 128-row tiles (uniform per block).
    const int64_t li = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock / kLiveTileRows;
    if (li >= __ldg(m_tiles)) return;
    row = static_cast<int64_t>(__ldg(m_tiles + 1 + li)) * kLiveTileRows + row % kLiveTileRows;
  }
  const bool active = row < rows;
  const int64_t base = row * d;
  Raw4<kRes16> rr[kRmsChunks];
  Raw4<kDelta == 2> rd[kDelta == 0 ? 1 : kRmsChunks];
#pragma unroll
  for (int i = 0; i < kRmsChunks; ++i) {
    const int col = (i * TPR + t) * 4;
    if (active && col < d) {
      rr[i] = load_raw4<kRes16>(res, base + col);
      if constexpr (kDelta != 0) rd[i] = load_raw4<kDelta == 2>(delta, base + col);
    }
  }
  float4 v[kRmsChunks];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < kRmsChunks; ++i) {
    const int col = (i * TPR + t) * 4;
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (active && col < d) {
      v[i] = widen4<kRes16>(rr[i], res_dtype == TJB_BF16);
      if constexpr (kDelta != 0) {
        const float4 dl = widen4<kDelta == 2>(rd[i], delta_dtype == TJB_BF16);
        v[i].x += dl.x;
        v[i].y += dl.y;
        v[i].z += dl.z;
        v[i].w += dl.w;
      }
      sq += (v[i].x * v[i].x + v[i].y * v[i].y) + (v[i].z * v[i].z + v[i].w * v[i].w);
    }
  }
  const float mean = rms_row_sum<TPR>(sq, scratch) / static_cast<float>(d);
  const float rstd = __frsqrt_rn(mean + eps);
  if (!active) return;  // uniform over each warp
  const bool keep = row_mask == nullptr || __ldg(row_mask + row) != 0;
  const int kb_count = (d + kQBlock - 1) / kQBlock;
#pragma unroll
  for (int i = 0; i < kRmsChunks; ++i) {
    const int col = (i * TPR + t) * 4;
    const int kb = (i * TPR + t) >> 5;  // scale block of this warp's chunk
    if (kb >= kb_count) break;          // warp-uniform
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < d) {
      if (res_out != nullptr) store4(res_out, res_dtype, base + col, v[i]);
      if (keep) {
        const float4 ww = __ldg(reinterpret_cast<const float4*>(w + col));
        y.x = v[i].x * rstd * ww.x;
        y.y = v[i].y * rstd * ww.y;
        y.z = v[i].z * rstd * ww.z;
        y.w = v[i].w * rstd * ww.w;
      }
    }
    if (out_dtype == TJB_E4M3) {
      const float s = block_scale(warp_max_abs(max_abs4(y)));
      if (col < d)
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + base + col) =
            quantize4(y, divisor(s));
      if ((t & 31) == 0) out_scales[row * kb_count + kb] = s;
    } else if (col < d) {
      store4(out, out_dtype, base + col, y);
    }
  }
}

// The same on 16-byte pieces of eight columns, sixteen lanes to a scale block.
// 16384 x 4096, bf16 + bf16 to 8 bits: 75 us (72 at the rate of a copy) against
// 85 in pieces of four, and 79 with two chunks a thread; 8192 x 8192, bf16
// alone: 51 against 69.
template <typename T, bool kDelta, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
    add_rmsnorm16_kernel(const T* res, const T* delta, T* res_out, void* out,
                         float* __restrict__ out_scales, const float* __restrict__ w, int rows,
                         int d, float eps, int out_dtype, const uint8_t* __restrict__ row_mask,
                         const int32_t* __restrict__ m_tiles) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  constexpr int kRowsPerBlock = BLOCK / TPR;
  constexpr int res_dtype = std::is_same<T, __half>::value ? TJB_F16 : TJB_BF16;
  __shared__ float scratch[BLOCK / 32];
  const int t = threadIdx.x % TPR;
  griddep_wait();
  griddep_launch_dependents();
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + threadIdx.x / TPR;
  if (m_tiles != nullptr) {
    const int64_t li = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock / kLiveTileRows;
    if (li >= __ldg(m_tiles)) return;
    row = static_cast<int64_t>(__ldg(m_tiles + 1 + li)) * kLiveTileRows + row % kLiveTileRows;
  }
  const bool active = row < rows;
  const int64_t base = row * d;
  Piece16<T> rr[kRmsChunks], rd[kDelta ? kRmsChunks : 1];
#pragma unroll
  for (int i = 0; i < kRmsChunks; ++i) {
    const int col = (i * TPR + t) * 8;
    if (active && col < d) {
      rr[i] = load_piece16(res + base + col);
      if constexpr (kDelta) rd[i] = load_piece16(delta + base + col);
    }
  }
  float v[kRmsChunks][8];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < kRmsChunks; ++i) {
    const int col = (i * TPR + t) * 8;
    if (active && col < d) {
      rr[i].widen(v[i]);
      if constexpr (kDelta) {
        float dl[8];
        rd[i].widen(dl);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += dl[j];
      }
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j += 2) part += v[i][j] * v[i][j] + v[i][j + 1] * v[i][j + 1];
      sq += part;
    }
  }
  const float mean = rms_row_sum<TPR>(sq, scratch) / static_cast<float>(d);
  const float rstd = __frsqrt_rn(mean + eps);
  if (!active) return;  // uniform over each warp
  const bool keep = row_mask == nullptr || __ldg(row_mask + row) != 0;
  const int kb_count = (d + kQBlock - 1) / kQBlock;
#pragma unroll
  for (int i = 0; i < kRmsChunks; ++i) {
    const int col = (i * TPR + t) * 8;
    if (col - (t & 31) * 8 >= d) break;  // warp-uniform
    float y[8] = {};
    if (col < d) {
      if (kDelta && res_out != nullptr) store8(res_out, res_dtype, base + col, v[i]);
      if (keep) {
        const float4 w0 = __ldg(reinterpret_cast<const float4*>(w + col));
        const float4 w1 = __ldg(reinterpret_cast<const float4*>(w + col) + 1);
        const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = v[i][j] * rstd * ww[j];
      }
    }
    if (out_dtype == TJB_E4M3) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j += 2) top = max_abs(top, y[j], y[j + 1]);
      uint32_t bits = abs_bits(top);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
      const float s = block_scale(__uint_as_float(bits));
      const Divisor div = divisor(s);
      if (col < d) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(out) + base + col) =
            make_uint2(quantize4(y, div), quantize4(y + 4, div));
        if ((t & 15) == 0) out_scales[row * kb_count + col / kQBlock] = s;
      }
    } else if (col < d) {
      store8(out, out_dtype, base + col, y);
    }
  }
}

}  // namespace
}  // namespace tjb

extern "C" int tjb_add_rmsnorm(const void* res, const void* delta, void* res_out, void* out,
                               float* out_scales, const float* w, int64_t rows, int d, float eps,
                               int res_dtype, int delta_dtype, int out_dtype,
                               const uint8_t* row_mask, const int32_t* m_tiles,
                               tjb_stream_t stream) {
  using namespace tjb;
  if (!res || !out || !w || rows < 0 || d <= 0) return TJB_ERR_INVALID_ARGUMENT;
  if (res_dtype < TJB_F32 || res_dtype > TJB_BF16 || delta_dtype < TJB_F32 ||
      delta_dtype > TJB_BF16 || out_dtype < TJB_F32 || out_dtype > TJB_E4M3)
    return TJB_ERR_UNSUPPORTED_DTYPE;
  const bool q = out_dtype == TJB_E4M3;
  if (q && !out_scales) return TJB_ERR_INVALID_ARGUMENT;
  if (d % (q ? 16 : 4) != 0 || d > 16384 || rows > 2147483647 - kLiveTileRows)
    return TJB_ERR_BAD_SHAPE;
  // Vectors of four elements.
  auto misaligned = [](const void* p, int dtype) {
    return (reinterpret_cast<uintptr_t>(p) & (dtype == TJB_F32 ? 15u : 7u)) != 0;
  };
  if (misaligned(res, res_dtype) || (delta && misaligned(delta, delta_dtype)) ||
      (res_out && misaligned(res_out, res_dtype)) || !aligned16(w) || misaligned(out, out_dtype) ||
      (q && (!aligned16(out) || (reinterpret_cast<uintptr_t>(out_scales) & 3u) != 0)))
    return TJB_ERR_BAD_ALIGNMENT;
  if (!device_ok()) return TJB_ERR_NO_DEVICE;
  if (rows == 0) return TJB_OK;
  if (!delta && res_out == res) res_out = nullptr;  // x is there already
  const int64_t n = m_tiles ? (rows + kLiveTileRows - 1) / kLiveTileRows * kLiveTileRows : rows;
  // 16-byte accesses where the types and the alignment allow them.  (Without a
  // delta that kernel writes no residual: a store that hardly any call asks for
  // cost all of them registers; 8192 x 8192 bf16 51.4 -> 53.3 us.)
  const bool vec8 = res_dtype != TJB_F32 && d % 8 == 0 && aligned16(res) && aligned16(out) &&
                    (delta ? delta_dtype == res_dtype && aligned16(delta) &&
                                 (!res_out || aligned16(res_out))
                           : !res_out);
  // Threads per row: enough for the row; with few rows, up to one chunk each,
  // since then the latency of a row counts and not the number of threads.
  const int chunk = vec8 ? 8 : 4;
  int tpr = 32;
  while (chunk * kRmsChunks * tpr < d ||
         (tpr < 1024 && chunk * tpr < d && 2 * n * tpr <= 1024 * num_sms()))
    tpr *= 2;
  auto by_tpr = [&](auto run) {
    switch (tpr) {
      case 32: return run(std::integral_constant<int, 32>{});
      case 64: return run(std::integral_constant<int, 64>{});
      case 128: return run(std::integral_constant<int, 128>{});
      case 256: return run(std::integral_constant<int, 256>{});
      case 512: return run(std::integral_constant<int, 512>{});
      default: return run(std::integral_constant<int, 1024>{});
    }
  };
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto grid = [&](int per_block) {
    return dim3(static_cast<unsigned>((n + per_block - 1) / per_block));
  };
  if (vec8) {
    auto go = [&](auto type, auto kdelta) {
      using T = decltype(type);
      constexpr bool kDelta = decltype(kdelta)::value;
      return by_tpr([&](auto tprc) {
        constexpr int TPR = decltype(tprc)::value;
        constexpr int block = TPR < 256 ? 256 : TPR;
        return launch_kernel(add_rmsnorm16_kernel<T, kDelta, TPR>, grid(block / TPR), dim3(block),
                             0, st, static_cast<const T*>(res), static_cast<const T*>(delta),
                             static_cast<T*>(res_out), out, out_scales, w, static_cast<int>(rows),
                             d, eps, out_dtype, row_mask, m_tiles);
      });
    };
    if (res_dtype == TJB_F16)
      return delta ? go(__half{}, std::true_type{}) : go(__half{}, std::false_type{});
    return delta ? go(__nv_bfloat16{}, std::true_type{}) : go(__nv_bfloat16{}, std::false_type{});
  }
  auto go = [&](auto res16, auto kdelta) {
    return by_tpr([&](auto tprc) {
      constexpr int TPR = decltype(tprc)::value;
      constexpr int block = TPR < 256 ? 256 : TPR;
      return launch_kernel(
          add_rmsnorm_kernel<TPR, decltype(res16)::value, decltype(kdelta)::value>,
          grid(block / TPR), dim3(block), 0, st, res, delta, res_out, out, out_scales, w,
          static_cast<int>(rows), d, eps, res_dtype, delta_dtype, out_dtype, row_mask, m_tiles);
    });
  };
  auto with_delta = [&](auto res16) {
    if (!delta) return go(res16, std::integral_constant<int, 0>{});
    if (delta_dtype == TJB_F32) return go(res16, std::integral_constant<int, 1>{});
    return go(res16, std::integral_constant<int, 2>{});
  };
  return res_dtype == TJB_F32 ? with_delta(std::false_type{}) : with_delta(std::true_type{});
}
