// The gate of an expert-parallel layer: scores, selection bias, expert groups, top-k, weights.
//
//   s_e = sigmoid(l_e)  or  softmax(l)_e          c_e = s_e + b_e           (b steers the selection only)
//   groups of E / n consecutive experts are ranked by their largest c, or by the sum of their two
//   largest; the experts of the best g groups compete, and the k largest c are taken in order
//   (ties to the lower id).      w_k = scale * s_k  [ / sum_j s_j ]
//
// An expert whose logit is -inf or NaN (or whose c is) is unavailable. A row with fewer than k
// available experts ends in ids of -1 with weight 0, which dispatch skips.
//
// The order of the selection values does not hang on 32-bit roundings:
//  * without a bias, and with groups ranked by their largest value, the order of c is that of
//    the logits themselves (both scores grow with the logit), which are compared as they are;
//  * otherwise c is formed in fp32 with a bound on its error, and a row in which two values whose
//    order matters lie closer than that bound is selected again in fp64. With 256 experts that
//    is a few rows in a thousand.
//
// Forward and backward read each logit once (T * E) and write T * k * 12 or T * E; a warp takes
// one token, its experts in the lanes' registers.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cfloat>

#include "ops.h"

namespace b200ep {
namespace {

constexpr int kMaxTopk = 32, kMaxGroups = 32, kMaxExperts = 1024;
constexpr uint32_t kAll = 0xffffffffu;
constexpr int kGateWarps = 4;

struct GateArgs {
  const void* logits;
  int64_t stride;        // elements between rows of logits
  const float* bias;     // [E] or nullptr
  int64_t* idx;
  float* w;
  int T, E, K;
  int n, g, gs;          // groups, groups kept, experts per group
  int lanes;             // lanes that scan one group (power of two, lanes * n <= 32)
  int sigmoid, top2, renorm;
  float scale;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// A logit as the gate sees it: NaN is unavailable, +inf is the largest finite value (so that a
// softmax stays defined), -0 is +0.
__device__ __forceinline__ float clean_logit(float v) {
  return v != v ? -INFINITY : fminf(v, FLT_MAX) + 0.f;
}
__device__ __forceinline__ float sigmoid_f32(float x) {
  const float e = expf(-fabsf(x));
  return (x >= 0.f ? 1.f : e) / (1.f + e);
}

template <typename T>
__device__ __forceinline__ T low();
template <>
__device__ __forceinline__ float low<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ double low<double>() { return -static_cast<double>(INFINITY); }

template <typename T>
__device__ __forceinline__ T warp_max(T v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) {
    const T o = __shfl_xor_sync(kAll, v, m);
    v = o > v ? o : v;
  }
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(kAll, v, m);
  return v;
}

// Selection over the warp's values v (lane holds experts lane * EPT + i), destroying them:
// lane j < K gets the j-th largest's id in `mine` (-1 where nothing is left). `slack(a)` bounds
// how far apart two values near `a` must be for their order to be certain; false is returned if
// some order that matters is not. `buf`: E + lanes * n values of shared memory of this warp.
template <typename T, int EPT, typename Slack>
__device__ __forceinline__ bool select(const GateArgs& a, T (&v)[EPT], T* buf, int lane, int& mine, Slack slack) {
  bool sure = true;
  if (a.n > 1) {
    // group values: `lanes` lanes scan each group through shared memory (a group is skewed by
    // `lanes` words from the one before, so that the lanes of different groups hit other banks)
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int e = lane * EPT + i;
      if (e < a.E) buf[e + e / a.gs * a.lanes] = v[i];
    }
    __syncwarp();
    const int grp = lane / a.lanes, sub = lane % a.lanes;
    T t0 = low<T>(), t1 = low<T>();
    if (grp < a.n) {
      const T* p = buf + grp * (a.gs + a.lanes);
      for (int j = sub; j < a.gs; j += a.lanes) {
        const T x = p[j];
        if (x > t0) {
          t1 = t0;
          t0 = x;
        } else if (x > t1) {
          t1 = x;
        }
      }
    }
    for (int m = a.lanes >> 1; m >= 1; m >>= 1) {
      const T o0 = __shfl_xor_sync(kAll, t0, m), o1 = __shfl_xor_sync(kAll, t1, m);
      const T hi = o0 > t0 ? o0 : t0, lo = o0 > t0 ? t0 : o0;
      const T s = o1 > t1 ? o1 : t1;
      t0 = hi;
      t1 = lo > s ? lo : s;
    }
    // the sum counts the second value only where there is one
    const T gv = grp >= a.n ? low<T>() : (a.top2 && t1 > low<T>() ? t0 + t1 : t0);
    int rank = 0;
    for (int j = 0; j < a.n; ++j) {
      const T o = __shfl_sync(kAll, gv, j * a.lanes);
      rank += (o > gv || (o == gv && j < grp)) ? 1 : 0;
    }
    const bool in = grp < a.n && rank < a.g && gv > low<T>();
    const uint32_t kept = __ballot_sync(kAll, in);
    const T worst_in = -warp_max(in ? -gv : low<T>());
    const T best_out = warp_max(in ? low<T>() : gv);
    if (best_out > low<T>() && !(worst_in - best_out > slack(worst_in) + slack(best_out))) sure = false;
    int of = lane * EPT / a.gs, left = a.gs - lane * EPT % a.gs;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      if (of >= a.n || !((kept >> (of * a.lanes & 31)) & 1u)) v[i] = low<T>();
      if (--left == 0) {
        ++of;
        left = a.gs;
      }
    }
    __syncwarp();
  }
  mine = -1;
  T before = low<T>();
  for (int k = 0; k <= a.K; ++k) {
    T best = low<T>();
    int at = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      if (v[i] > best) {
        best = v[i];
        at = i;
      }
    }
    const T top = warp_max(best);
    if (top == low<T>()) break;
    if (k > 0 && !(before - top > slack(before))) sure = false;
    if (k == a.K) break;
    before = top;
    const int from = __ffs(__ballot_sync(kAll, best == top)) - 1;  // ids grow with the lane
    const int id = __shfl_sync(kAll, lane * EPT + at, from);
    if (lane == k) mine = id;
    if (lane == from) {
#pragma unroll
      for (int i = 0; i < EPT; ++i)
        if (i == at) v[i] = low<T>();
    }
  }
  return sure;
}

// The same selection with scores in fp64.
template <int EPT>
__device__ __noinline__ int select_f64(const GateArgs& a, const float* l, double* buf, int lane) {
  double v[EPT];
  double top = 0, sum = 1;
  if (!a.sigmoid) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; ++i) m = fmaxf(m, l[i]);
    top = warp_max(m);
    sum = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) sum += l[i] > -INFINITY ? exp(static_cast<double>(l[i]) - top) : 0.0;
    sum = warp_sum(sum);
  }
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const int e = lane * EPT + i;
    const double x = l[i];
    double s = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum;
    if (a.bias != nullptr && e < a.E) s += static_cast<double>(a.bias[e]);
    v[i] = l[i] > -INFINITY && s == s ? s : low<double>();
  }
  int mine;
  select<double, EPT>(a, v, buf, lane, mine, [](double) { return 0.0; });
  return mine;
}

template <typename T, int EPT>
__global__ void __launch_bounds__(kGateWarps * 32) gate_kernel(GateArgs a) {
  extern __shared__ double gate_smem[];
  const int lane = lane_id(), warp = warp_id();
  const int t = blockIdx.x * kGateWarps + warp;
  if (t >= a.T) return;  // whole warps only: no barrier follows
  double* buf = gate_smem + static_cast<int64_t>(warp) * (a.E + 32);
  const T* row = static_cast<const T*>(a.logits) + static_cast<int64_t>(t) * a.stride;
  float l[EPT], v[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const int e = lane * EPT + i;
    l[i] = e < a.E ? clean_logit(to_f32(row[e])) : -INFINITY;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPT; ++i) m = fmaxf(m, l[i]);
  m = warp_max(m);
  const bool direct = a.bias == nullptr && (a.n == 1 || !a.top2);
  int mine;
  float sum = 1.f;
  if (!a.sigmoid && !(direct && a.renorm)) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) sum += l[i] > -INFINITY ? expf(l[i] - m) : 0.f;
    sum = warp_sum(sum);
  }
  if (direct) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) v[i] = l[i];
    select<float, EPT>(a, v, reinterpret_cast<float*>(buf), lane, mine, [](float) { return 0.f; });
  } else {
    const float inv = 1.f / sum;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int e = lane * EPT + i;
      const float s = a.sigmoid ? sigmoid_f32(l[i]) : expf(l[i] - m) * inv;
      const float c = a.bias != nullptr && e < a.E ? s + a.bias[e] : s;
      v[i] = l[i] > -INFINITY && c == c ? c + 0.f : -INFINITY;
    }
    // Each score is within 2^-21 of its value relative to itself (an exponential and a division
    // within 2 units each, the sums within 1), so within 2^-21 * (largest score); the bias adds
    // one rounding of the sum, and a sum of two such values doubles both and adds another. The
    // bounds below are twice that, for one value of a pair.
    const float most = a.sigmoid ? 1.f : inv;
    const float k0 = most * 0x1p-18f;
    const bool sure = select<float, EPT>(a, v, reinterpret_cast<float*>(buf), lane, mine,
                                         [k0](float x) { return k0 + fabsf(x) * 0x1p-21f; });
    if (!sure) mine = select_f64<EPT>(a, l, buf, lane);
  }
  // weights from the logits of the chosen
  const float x = mine >= 0 ? clean_logit(to_f32(row[mine])) : -INFINITY;
  const bool has = mine >= 0;
  float w = 0.f;
  if (a.renorm) {
    // both scores are proportional to exp(x - r) times a factor between 1/2 and 1 (sigmoid) or 1;
    // r keeps the sum from underflowing
    const float top = warp_max(x);
    if (a.sigmoid) {
      const float r = fminf(top, 0.f);
      w = !has ? 0.f : (x >= 0.f ? 1.f / (1.f + expf(-x)) : expf(x - r) / (1.f + expf(x)));
    } else {
      w = has ? expf(x - top) : 0.f;
    }
    const float total = warp_sum(w);
    w = has ? w / total : 0.f;
  } else {
    w = !has ? 0.f : (a.sigmoid ? sigmoid_f32(x) : expf(x - m) / sum);
  }
  if (lane < a.K) {
    a.idx[static_cast<int64_t>(t) * a.K + lane] = mine;
    a.w[static_cast<int64_t>(t) * a.K + lane] = w * a.scale;
  }
}

struct GateBwdArgs {
  const void* logits;
  int64_t stride;
  const int64_t* idx;
  const float* dw;
  void* d;               // [T, E] contiguous, type of the logits
  int T, E, K;
  int sigmoid, renorm;
  float scale;
};

// With p the normalised (or plain) score of the chosen and dw scaled:
//   sigmoid          d_k = dw_k s_k (1 - s_k)
//   sigmoid, renorm  d_k = p_k (1 - s_k) (dw_k - sum_j p_j dw_j)
//   softmax, renorm  d_k = p_k (dw_k - sum_j p_j dw_j)      (the softmax over the chosen)
//   softmax          d_e = p_e ([e chosen] dw_e - sum_j p_j dw_j)   for every e of the row
// zero elsewhere. An id that occurs twice gets the sum; ids outside [0, E) count for nothing.
template <typename T, int EPT>
__global__ void __launch_bounds__(kGateWarps * 32) gate_bwd_kernel(GateBwdArgs a) {
  const int lane = lane_id(), warp = warp_id();
  const int t = blockIdx.x * kGateWarps + warp;
  if (t >= a.T) return;
  const T* row = static_cast<const T*>(a.logits) + static_cast<int64_t>(t) * a.stride;
  int id = -1;
  float dw = 0.f;
  if (lane < a.K) {
    const int64_t e = a.idx[static_cast<int64_t>(t) * a.K + lane];
    if (e >= 0 && e < a.E) {
      id = static_cast<int>(e);
      dw = a.dw[static_cast<int64_t>(t) * a.K + lane] * a.scale;
    }
  }
  float x = id >= 0 ? clean_logit(to_f32(row[id])) : -INFINITY;
  const bool has = x > -INFINITY;
  if (!has) dw = 0.f;
  float l[EPT];
  float gk = 0.f, dot = 0.f, m = 0.f, inv = 0.f;
  const bool whole = !a.sigmoid && !a.renorm;
  if (whole) {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int e = lane * EPT + i;
      l[i] = e < a.E ? clean_logit(to_f32(row[e])) : -INFINITY;
      m = fmaxf(m, l[i]);
    }
    m = warp_max(m);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      l[i] = l[i] > -INFINITY ? expf(l[i] - m) : 0.f;
      sum += l[i];
    }
    sum = warp_sum(sum);
    inv = sum > 0.f ? 1.f / sum : 0.f;
    dot = warp_sum(has ? expf(x - m) * inv * dw : 0.f);
    gk = dw;
  } else if (!a.renorm) {
    gk = has ? dw * sigmoid_f32(x) * sigmoid_f32(-x) : 0.f;
  } else {
    const float top = warp_max(x);
    float p;
    if (a.sigmoid) {
      const float r = fminf(top, 0.f);
      p = !has ? 0.f : (x >= 0.f ? 1.f / (1.f + expf(-x)) : expf(x - r) / (1.f + expf(x)));
    } else {
      p = has ? expf(x - top) : 0.f;
    }
    const float total = warp_sum(p);
    p = has ? p / total : 0.f;
    dot = warp_sum(p * dw);
    gk = has ? p * (dw - dot) * (a.sigmoid ? sigmoid_f32(-x) : 1.f) : 0.f;
  }
  float out[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) out[i] = 0.f;
  for (int k = 0; k < a.K; ++k) {
    const int e = __shfl_sync(kAll, id, k);
    const float g = __shfl_sync(kAll, gk, k);
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (e == lane * EPT + i) out[i] += g;
  }
  if (whole) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) out[i] = l[i] * inv * (out[i] - dot);
  }
  T* drow = static_cast<T*>(a.d) + static_cast<int64_t>(t) * a.E;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const int e = lane * EPT + i;
    if (e < a.E) drow[e] = from_f32<T>(out[i]);
  }
}

template <typename T>
void launch_gate(const GateArgs& a, cudaStream_t s) {
  const int grid = (a.T + kGateWarps - 1) / kGateWarps;
  const size_t smem = a.n > 1 ? sizeof(double) * kGateWarps * (a.E + 32) : 0;
  if (a.E <= 32) gate_kernel<T, 1><<<grid, kGateWarps * 32, smem, s>>>(a);
  else if (a.E <= 64) gate_kernel<T, 2><<<grid, kGateWarps * 32, smem, s>>>(a);
  else if (a.E <= 128) gate_kernel<T, 4><<<grid, kGateWarps * 32, smem, s>>>(a);
  else if (a.E <= 256) gate_kernel<T, 8><<<grid, kGateWarps * 32, smem, s>>>(a);
  else if (a.E <= 512) gate_kernel<T, 16><<<grid, kGateWarps * 32, smem, s>>>(a);
  else gate_kernel<T, 32><<<grid, kGateWarps * 32, smem, s>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename T>
void launch_gate_bwd(const GateBwdArgs& a, cudaStream_t s) {
  const int grid = (a.T + kGateWarps - 1) / kGateWarps;
  if (a.E <= 32) gate_bwd_kernel<T, 1><<<grid, kGateWarps * 32, 0, s>>>(a);
  else if (a.E <= 64) gate_bwd_kernel<T, 2><<<grid, kGateWarps * 32, 0, s>>>(a);
  else if (a.E <= 128) gate_bwd_kernel<T, 4><<<grid, kGateWarps * 32, 0, s>>>(a);
  else if (a.E <= 256) gate_bwd_kernel<T, 8><<<grid, kGateWarps * 32, 0, s>>>(a);
  else if (a.E <= 512) gate_bwd_kernel<T, 16><<<grid, kGateWarps * 32, 0, s>>>(a);
  else gate_bwd_kernel<T, 32><<<grid, kGateWarps * 32, 0, s>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void check_logits(const at::Tensor& logits) {
  TORCH_CHECK(logits.dim() == 2, "logits must be [T, E]");
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16 ||
                  logits.scalar_type() == at::kHalf,
              "logits must be fp32, bf16 or fp16");
  TORCH_CHECK(unit_inner(logits), "the experts of a row must be contiguous");
  TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) <= kMaxExperts, "need 1 <= E <= 1024");
  TORCH_CHECK(logits.size(0) <= 0x7fffff00, "too many tokens");
}

}  // namespace

// CPU tensors (the torch definition's callers) run the checks alone.
std::tuple<at::Tensor, at::Tensor> router_gate(const at::Tensor& logits, int64_t topk, bool sigmoid,
                                               const OptTensor& bias, int64_t num_groups, int64_t topk_groups,
                                               bool top2, bool renorm, double scale) {
  check_logits(logits);
  GateArgs a{};
  a.T = static_cast<int>(logits.size(0));
  a.E = static_cast<int>(logits.size(1));
  TORCH_CHECK(num_groups >= 1 && num_groups <= kMaxGroups && a.E % num_groups == 0 && topk_groups >= 1 &&
                  topk_groups <= num_groups,
              "need 1 <= topk_groups <= num_groups <= 32 and num_groups dividing E");
  TORCH_CHECK(topk >= 1 && topk <= kMaxTopk && topk <= a.E / num_groups * topk_groups,
              "need 1 <= k <= 32 and k <= the experts of the chosen groups");
  a.K = static_cast<int>(topk);
  a.n = static_cast<int>(num_groups);
  a.g = static_cast<int>(topk_groups);
  a.gs = a.E / a.n;
  a.lanes = 32;
  while (a.lanes * a.n > 32) a.lanes >>= 1;
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == logits.device() && bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                    bias->size(0) == a.E && unit_inner(*bias),
                "bias must be fp32 [E] on the logits' device");
    a.bias = bias->data_ptr<float>();
  }
  if (!logits.is_cuda()) return {};  // the checks alone
  const c10::cuda::CUDAGuard guard(logits.device());
  auto idx = at::empty({a.T, a.K}, logits.options().dtype(at::kLong));
  auto w = at::empty({a.T, a.K}, logits.options().dtype(at::kFloat));
  if (a.T == 0) return {idx, w};
  a.logits = logits.data_ptr();
  a.stride = logits.stride(0);
  a.idx = idx.data_ptr<int64_t>();
  a.w = w.data_ptr<float>();
  a.sigmoid = sigmoid;
  a.top2 = top2;
  a.renorm = renorm;
  a.scale = static_cast<float>(scale);
  auto s = at::cuda::getCurrentCUDAStream();
  if (logits.scalar_type() == at::kFloat) launch_gate<float>(a, s);
  else if (logits.scalar_type() == at::kBFloat16) launch_gate<__nv_bfloat16>(a, s);
  else launch_gate<__half>(a, s);
  return {idx, w};
}

at::Tensor router_gate_bwd(const at::Tensor& logits, const at::Tensor& idx, const at::Tensor& dw, bool sigmoid,
                           bool renorm, double scale) {
  check_logits(logits);
  GateBwdArgs a{};
  a.T = static_cast<int>(logits.size(0));
  a.E = static_cast<int>(logits.size(1));
  TORCH_CHECK(idx.dim() == 2 && idx.size(0) == a.T && idx.size(1) >= 1 && idx.size(1) <= kMaxTopk &&
                  idx.scalar_type() == at::kLong && idx.is_contiguous() && idx.device() == logits.device(),
              "idx must be contiguous int64 [T, k], k <= 32");
  TORCH_CHECK(dw.sizes() == idx.sizes() && dw.scalar_type() == at::kFloat && dw.is_contiguous() &&
                  dw.device() == logits.device(),
              "dw must be contiguous fp32 [T, k]");
  if (!logits.is_cuda()) return {};  // the checks alone
  const c10::cuda::CUDAGuard guard(logits.device());
  auto d = at::empty({a.T, a.E}, logits.options());
  if (a.T == 0) return d;
  a.K = static_cast<int>(idx.size(1));
  a.logits = logits.data_ptr();
  a.stride = logits.stride(0);
  a.idx = idx.data_ptr<int64_t>();
  a.dw = dw.data_ptr<float>();
  a.d = d.data_ptr();
  a.sigmoid = sigmoid;
  a.renorm = renorm;
  a.scale = static_cast<float>(scale);
  auto s = at::cuda::getCurrentCUDAStream();
  if (logits.scalar_type() == at::kFloat) launch_gate_bwd<float>(a, s);
  else if (logits.scalar_type() == at::kBFloat16) launch_gate_bwd<__nv_bfloat16>(a, s);
  else launch_gate_bwd<__half>(a, s);
  return d;
}

}  // namespace b200ep
