// N6: standalone per-token, per-128-channel e4m3 quantisation (the same
// device function the dispatch kernels fuse into their send path).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "ops.h"

namespace b200ep {

template <typename T16>
__global__ void __launch_bounds__(256) quant_fp8_kernel(const T16* __restrict__ x, uint8_t* __restrict__ q,
                                                        float* __restrict__ scales, int64_t T, int H,
                                                        int round_scale) {
  const int64_t gw = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int64_t GW = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  for (int64_t t = gw; t < T; t += GW)
    warp_quant_row<T16>(q + t * H, scales + t * (H / 128), x + t * H, H, round_scale);
}

void quant_fp8(const at::Tensor& x, at::Tensor q, at::Tensor scales, bool round_scale) {
  const c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.is_contiguous() && q.is_contiguous() && scales.is_contiguous(), "contiguous tensors expected");
  const int H = static_cast<int>(x.size(-1));
  TORCH_CHECK(H % 128 == 0, "hidden must be a multiple of 128");
  const int64_t T = x.numel() / H;
  TORCH_CHECK(q.element_size() == 1 && q.numel() == x.numel(), "q must be a 1-byte tensor shaped like x");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.numel() == T * (H / 128), "scales must be fp32 [.., H/128]");
  if (T == 0) return;
  const int blocks = static_cast<int>(std::min<int64_t>((T + 7) / 8, 148 * 16));
  auto stream = at::cuda::getCurrentCUDAStream();
  if (x.scalar_type() == at::kHalf)
    quant_fp8_kernel<__half><<<blocks, 256, 0, stream>>>(reinterpret_cast<const __half*>(x.data_ptr()),
                                                        static_cast<uint8_t*>(q.data_ptr()), scales.data_ptr<float>(),
                                                        T, H, round_scale);
  else
    quant_fp8_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(
        reinterpret_cast<const __nv_bfloat16*>(x.data_ptr()), static_cast<uint8_t*>(q.data_ptr()),
        scales.data_ptr<float>(), T, H, round_scale);
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
// A CTA holds one block in registers: each weight is read once and nothing waits but for the one
// reduction. VEC: rows in 8-element chunks on aligned addresses, else element by element.
constexpr int kWqThreads = 256;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kWqThreads) quant_weight_kernel(const T* __restrict__ w, int64_t row, int64_t group,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scales,
                                                                  int N, int K, int NB, int KB) {
  __shared__ uint32_t s_top[kWqThreads / 32];
  const int64_t blk = blockIdx.x;
  const int kb = static_cast<int>(blk % KB);
  const int nb = static_cast<int>(blk / KB % NB);
  const int64_t g = blk / KB / NB;
  const int col = kb * 128 + (threadIdx.x & 15) * 8, r0 = nb * 128 + (threadIdx.x >> 4);
  const T* src = w + g * group + col;
  float v[8][8];
  uint32_t top = 0;   // amax as bits, so that a NaN stays the largest
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (VEC) {
      if (r < N && col < K) {
        alignas(16) T t[8];
        const int4* p = reinterpret_cast<const int4*>(src + r * row);
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j) reinterpret_cast<int4*>(t)[j] = __ldcs(p + j);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = static_cast<float>(t[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = r < N && col + j < K ? static_cast<float>(src[r * row + j]) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(fabsf(v[i][j])));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __float_as_uint(1e-4f);
#pragma unroll
  for (int i = 0; i < kWqThreads / 32; ++i) top = max(top, s_top[i]);
  const float amax = __uint_as_float(top);
  const float inv = __fdiv_rn(448.f, amax);
  if (threadIdx.x == 0) scales[blk] = __fdiv_rn(amax, 448.f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (r >= N || col >= K) continue;
    uint8_t* dst = q + (g * N + r) * K + col;
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      o[j] = uint32_t(f32x2_to_e4m3x2(v[i][4 * j] * inv, v[i][4 * j + 1] * inv)) |
             (uint32_t(f32x2_to_e4m3x2(v[i][4 * j + 2] * inv, v[i][4 * j + 3] * inv)) << 16);
    if (VEC) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < K) dst[j] = static_cast<uint8_t>(o[j >> 2] >> (8 * (j & 3)));
    }
  }
}

std::tuple<at::Tensor, at::Tensor> quant_fp8_weight(const at::Tensor& w) {
  TORCH_CHECK((w.dim() == 2 || w.dim() == 3) && unit_inner(w), "w must be [N, K] or [G, N, K] with unit inner stride");
  TORCH_CHECK(w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16 || w.scalar_type() == at::kHalf,
              "w must be fp32, bf16 or fp16");
  if (!w.is_cuda()) return {};  // CPU tensors: the checks alone
  const c10::cuda::CUDAGuard guard(w.device());
  const int64_t G = w.dim() == 3 ? w.size(0) : 1, N = w.size(-2), K = w.size(-1);
  TORCH_CHECK(N < (1 << 30) && K < (1 << 30), "sizes below 2^30");
  const int64_t NB = (N + 127) / 128, KB = (K + 127) / 128;
  auto shape = w.sizes().vec();
  auto q = at::empty(shape, w.options().dtype(at::kByte));
  shape[shape.size() - 2] = NB;
  shape.back() = KB;
  auto sc = at::empty(shape, w.options().dtype(at::kFloat));
  const int64_t blocks = G * NB * KB;
  if (blocks == 0) return {q, sc};
  TORCH_CHECK(blocks < (1ll << 31), "too many blocks");
  const int64_t es = w.element_size(), row = w.stride(-2), group = w.dim() == 3 ? w.stride(0) : 0;
  const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(w.data_ptr()) & 15) == 0 && row * es % 16 == 0 &&
                   group * es % 16 == 0;
  auto s = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto zero) {
    using T = decltype(zero);
    auto k = vec ? quant_weight_kernel<T, true> : quant_weight_kernel<T, false>;
    k<<<static_cast<unsigned>(blocks), kWqThreads, 0, s>>>(static_cast<const T*>(w.data_ptr()), row, group,
                                                          q.data_ptr<uint8_t>(), sc.data_ptr<float>(),
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
