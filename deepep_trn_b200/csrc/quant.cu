// N6: standalone per-token, per-128-channel e4m3 quantisation (the same
// device function the dispatch kernels fuse into their send path).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include "ops.h"

namespace b200ep {

template <typename T16>
__global__ void __launch_bounds__(256) quant_fp8_kernel(const T16* __restrict__ x, uint8_t* __restrict__ q,
                                                        float* __restrict__ scales, int64_t T, int H,
                                                        int round_scale, float amax_floor) {
  const int64_t gw = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t GW = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t t = gw; t < T; t += GW)
    warp_quant_row<T16>(q + t * H, scales + t * (H / 128), x + t * H, H, round_scale, amax_floor);
}

void quant_fp8(const at::Tensor& x, at::Tensor q, at::Tensor scales, bool round_scale, double amax_floor) {
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "x must be bf16 or fp16");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 8 == 0,
              "x must start on a 16-byte boundary, q on one of 8");
  TORCH_CHECK(x.is_contiguous() && q.is_contiguous() && scales.is_contiguous(), "contiguous tensors expected");
  const int H = static_cast<int>(x.size(-1));
  TORCH_CHECK(H % 128 == 0, "hidden must be a multiple of 128");
  const int64_t T = x.numel() / H;
  TORCH_CHECK(q.element_size() == 1 && q.numel() == x.numel(), "q must be a 1-byte tensor shaped like x");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.numel() == T * (H / 128), "scales must be fp32 [.., H/128]");
  // below, the scale would be subnormal or 448 / amax infinite
  TORCH_CHECK(amax_floor >= 0x1p-116 && amax_floor <= 448., "the floor of amax must be between 2^-116 and 448");
  if (T == 0) return;
  const int blocks = static_cast<int>(std::min<int64_t>((T + 7) / 8, 148 * 16));
  auto stream = at::cuda::getCurrentCUDAStream();
  if (x.scalar_type() == at::kHalf)
    quant_fp8_kernel<__half><<<blocks, 256, 0, stream>>>(reinterpret_cast<const __half*>(x.data_ptr()),
                                                        static_cast<uint8_t*>(q.data_ptr()), scales.data_ptr<float>(),
                                                        T, H, round_scale, static_cast<float>(amax_floor));
  else
    quant_fp8_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(
        reinterpret_cast<const __nv_bfloat16*>(x.data_ptr()), static_cast<uint8_t*>(q.data_ptr()),
        scales.data_ptr<float>(), T, H, round_scale, static_cast<float>(amax_floor));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Inverse of the above: e4m3 [T, H] with fp32 scales [T, H/128] -> bf16 (scale * value,
// rounded once). A thread per 16 channels.
__global__ void __launch_bounds__(256) dequant_fp8_kernel(const uint8_t* __restrict__ q, const float* __restrict__ sc,
                                                          __nv_bfloat16* __restrict__ out, int64_t chunks, int H) {
  const int cpr = H / 16;  // chunks per row
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < chunks; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t t = i / cpr;
    const int j = static_cast<int>(i % cpr);
    const int4 v = reinterpret_cast<const int4*>(q)[i];
    const float f = sc[t * (H / 128) + (j >> 3)];
    const __nv_fp8x2_storage_t* b2 = reinterpret_cast<const __nv_fp8x2_storage_t*>(&v);
    alignas(16) __nv_bfloat162 o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 x2 = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(b2[k], __NV_E4M3)));
      o[k] = __floats2bfloat162_rn(x2.x * f, x2.y * f);
    }
    reinterpret_cast<int4*>(out)[2 * i] = reinterpret_cast<const int4*>(o)[0];
    reinterpret_cast<int4*>(out)[2 * i + 1] = reinterpret_cast<const int4*>(o)[1];
  }
}

void dequant_fp8(const at::Tensor& q, const at::Tensor& scales, at::Tensor out) {
  const c10::cuda::CUDAGuard guard(q.device());
  TORCH_CHECK(((reinterpret_cast<uintptr_t>(q.data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) & 15) == 0,
              "q and out must start on 16-byte boundaries");
  TORCH_CHECK(q.is_contiguous() && scales.is_contiguous() && out.is_contiguous(), "contiguous tensors expected");
  const int H = static_cast<int>(q.size(-1));
  TORCH_CHECK(H % 128 == 0 && q.element_size() == 1, "q must be e4m3 [.., H] with H % 128 == 0");
  const int64_t T = q.numel() / H;
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.numel() == T * (H / 128), "scales must be fp32 [.., H/128]");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.numel() == q.numel(), "out must be bf16 shaped like q");
  const int64_t chunks = T * (H / 16);
  if (chunks == 0) return;
  const int blocks = static_cast<int>(std::min<int64_t>((chunks + 255) / 256, 148 * 16));
  dequant_fp8_kernel<<<blocks, 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      static_cast<const uint8_t*>(q.data_ptr()), scales.data_ptr<float>(),
      static_cast<__nv_bfloat16*>(out.data_ptr()), chunks, H);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Weights: e4m3 [.., N, K] with one fp32 scale per 128 x 128 block (edges may be short):
// scale = max(amax, 1e-4) / 448, q = rn(w * (448 / amax)), the constants of the row quantiser.
// A CTA holds one block in registers, as it came (16 or 32 registers a thread, so that several CTAs
// share an SM and some load while others store): each weight is read once and nothing waits but for
// the one reduction. Bound by memory: 32 x 4096 x 7168 bf16 in 451 us, 6.25 TB/s (717 us with 256
// threads that hold 64 fp32 values each, two CTAs an SM). VEC: rows in 8-element chunks on aligned
// addresses, else element by element.
constexpr int kWqThreads = 512;
constexpr int kWqSteps = 128 * 16 / kWqThreads;   // 8-element chunks a thread

// Two 16-bit weights, or one fp32 weight, of a word as it lies in memory.
__device__ __forceinline__ float2 word_values(uint32_t w, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
__device__ __forceinline__ float2 word_values(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 word_values(uint32_t w, float) { return make_float2(__uint_as_float(w), 0.f); }

template <typename T, bool VEC>
__global__ void __launch_bounds__(kWqThreads, sizeof(T) == 2 && VEC ? 3 : 2)
    quant_weight_kernel(const T* __restrict__ w, int64_t row, int64_t group, uint8_t* __restrict__ q,
                        float* __restrict__ scales, int N, int K, int NB, int KB) {
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int kWords = kHalf ? 4 : 8;   // of a chunk
  __shared__ uint32_t s_top[kWqThreads / 32];
  const uint32_t blk = blockIdx.x;
  const int kb = static_cast<int>(blk % KB);
  const uint32_t rest = blk / KB;
  const int nb = static_cast<int>(rest % NB);
  const int64_t g = rest / NB;
  const int col = kb * 128 + (threadIdx.x & 15) * 8, r0 = nb * 128 + (threadIdx.x >> 4);
  const T* src = w + g * group + col;
  uint32_t v[kWqSteps][kWords];
#pragma unroll
  for (int i = 0; i < kWqSteps; ++i) {
    const int r = r0 + kWqThreads / 16 * i;
    if (VEC) {
#pragma unroll
      for (int j = 0; j < kWords / 4; ++j) {
        const int4 x = r < N && col < K ? __ldcs(reinterpret_cast<const int4*>(src + r * row) + j) : make_int4(0, 0, 0, 0);
        v[i][4 * j] = x.x, v[i][4 * j + 1] = x.y, v[i][4 * j + 2] = x.z, v[i][4 * j + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kWords; ++j) {
        alignas(4) T t[kHalf ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (kHalf ? 2 : 1); ++h) {
          const int c = (kHalf ? 2 : 1) * j + h;
          t[h] = r < N && col + c < K ? src[r * row + c] : T(0.f);
        }
        v[i][j] = *reinterpret_cast<const uint32_t*>(t);
      }
    }
  }
  // amax as bits without the sign (16-bit words two by two): in that order a NaN stays the largest
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kWqSteps; ++i)
#pragma unroll
    for (int j = 0; j < kWords; ++j)
      top = kHalf ? __vmaxu2(top, v[i][j] & 0x7fff7fffu) : max(top, v[i][j] & 0x7fffffffu);
  if (kHalf) top = __float_as_uint(word_values(max(top & 0xffffu, top >> 16), T(0.f)).x);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, max(s_top[threadIdx.x & (kWqThreads / 32 - 1)], __float_as_uint(1e-4f)));
  const float amax = __uint_as_float(top);
  const float inv = __fdiv_rn(448.f, amax);
  if (threadIdx.x == 0) scales[blk] = __fdiv_rn(amax, 448.f);
#pragma unroll
  for (int i = 0; i < kWqSteps; ++i) {
    const int r = r0 + kWqThreads / 16 * i;
    if (r >= N || col >= K) continue;
    uint8_t* dst = q + (g * N + r) * K + col;
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float f[4];
      if (kHalf) {
        const float2 x = word_values(v[i][2 * j], T(0.f)), y = word_values(v[i][2 * j + 1], T(0.f));
        f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(v[i][(4 * j + e) % kWords]);
      }
      o[j] = uint32_t(f32x2_to_e4m3x2(f[0] * inv, f[1] * inv)) | (uint32_t(f32x2_to_e4m3x2(f[2] * inv, f[3] * inv)) << 16);
    }
    if (VEC) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < K) dst[j] = static_cast<uint8_t>(o[j >> 2] >> (8 * (j & 3)));
    }
  }
}

std::tuple<at::Tensor, at::Tensor> quant_fp8_weight(const at::Tensor& w, const OptTensor& q_out,
                                                    const OptTensor& scales_out) {
  TORCH_CHECK((w.dim() == 2 || w.dim() == 3) && unit_inner(w), "w must be [N, K] or [G, N, K] with unit inner stride");
  TORCH_CHECK(w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16 || w.scalar_type() == at::kHalf,
              "w must be fp32, bf16 or fp16");
  const int64_t G = w.dim() == 3 ? w.size(0) : 1, N = w.size(-2), K = w.size(-1);
  TORCH_CHECK(N < (1 << 30) && K < (1 << 30), "sizes below 2^30");
  const int64_t NB = (N + 127) / 128, KB = (K + 127) / 128;
  auto shape = w.sizes().vec(), scales_shape = shape;
  scales_shape[shape.size() - 2] = NB;
  scales_shape.back() = KB;
  TORCH_CHECK(q_out.has_value() == scales_out.has_value(), "an output is a pair");
  if (q_out.has_value()) {
    TORCH_CHECK(q_out->device() == w.device() && q_out->scalar_type() == at::kFloat8_e4m3fn && q_out->sizes() == shape &&
                    q_out->is_contiguous(),
                "the output must be contiguous e4m3 of w's sizes on its device");
    TORCH_CHECK(scales_out->device() == w.device() && scales_out->scalar_type() == at::kFloat &&
                    scales_out->sizes() == scales_shape && scales_out->is_contiguous(),
                "the output's scales must be contiguous fp32, one a 128 x 128 block, on w's device");
  }
  if (!w.is_cuda()) return {};  // CPU tensors: the checks alone
  const c10::cuda::CUDAGuard guard(w.device());
  at::Tensor q, sc;
  if (q_out.has_value()) {
    q = *q_out;
    sc = *scales_out;
  } else {
    q = at::detail::empty_cuda(shape, at::kFloat8_e4m3fn, w.device(), c10::nullopt);
    sc = at::detail::empty_cuda(scales_shape, at::kFloat, w.device(), c10::nullopt);
  }
  // 8 values of a row are stored at once: an output of odd offset is written element by element
  const bool aligned = (reinterpret_cast<uintptr_t>(q.data_ptr()) & 7) == 0;
  const int64_t blocks = G * NB * KB;
  if (blocks == 0) return {q, sc};
  TORCH_CHECK(blocks < (1ll << 31), "too many blocks");
  const int64_t es = w.element_size(), row = w.stride(-2), group = w.dim() == 3 ? w.stride(0) : 0;
  const bool vec = aligned && K % 8 == 0 && (reinterpret_cast<uintptr_t>(w.data_ptr()) & 15) == 0 &&
                   row * es % 16 == 0 && group * es % 16 == 0;
  auto s = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto zero) {
    using T = decltype(zero);
    auto k = vec ? quant_weight_kernel<T, true> : quant_weight_kernel<T, false>;
    k<<<static_cast<unsigned>(blocks), kWqThreads, 0, s>>>(static_cast<const T*>(w.data_ptr()), row, group,
                                                          static_cast<uint8_t*>(q.data_ptr()), sc.data_ptr<float>(),
                                                          static_cast<int>(N), static_cast<int>(K),
                                                          static_cast<int>(NB), static_cast<int>(KB));
  };
  if (w.scalar_type() == at::kFloat) go(float{});
  else if (w.scalar_type() == at::kHalf) go(__half{});
  else go(__nv_bfloat16{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {q, sc};
}

}  // namespace b200ep
