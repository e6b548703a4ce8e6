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
//    order matters lie closer than that bound is selected again in fp64. With 256 experts, 8 of
//    them chosen from 4 of 8 groups, that is two rows in a thousand.
//
// Forward and backward read each logit once (T * E) and write T * k * 12 or T * E; a warp takes
// one token, its experts in the lanes' registers (16-byte loads and stores where the rows allow).
// Values are compared as integers of the same order, so that one redux finds the warp's largest.
// 16384 tokens of 256 experts, 8 groups, 8 chosen take 37 us forward and backward in a CUDA graph at 1965 MHz (43
// as calls from the host) where their bytes would take 6; 59 us with values compared as floats by shuffles,
// 4-byte accesses and ids looked for in every lane. One token takes 3.7 us in a graph, of which 2.5 are a launch
// (7.2 before), and 5.8 as a call. What bounds them: forward half by instruction issue (1037 a row, 28.7 of
// 59.6 thousand cycles), half by the chain of a row's dependent steps, which shows in the last wave of CTAs and
// in rows that fp64 decides (an SM has work in 39 of the 59.6); backward by latency (269 a row, issue 40 % busy,
// waiting for loads, exponentials and shared memory).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <cfloat>
#include <climits>

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
  int lanes;             // lanes that scan one group in shared memory (power of two, lanes * n <= 32)
  float inv_gs;          // 1 / gs
  int reg_lanes;         // lanes that hold one group in registers (a power of two), or 0
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
  return fminf(fmaxf(v, -INFINITY), FLT_MAX) + 0.f;   // fmaxf drops a NaN
}
__device__ __forceinline__ float sigmoid_f32(float x) {
  const float e = expf(-fabsf(x));
  return (x >= 0.f ? 1.f : e) / (1.f + e);
}

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

// Integers in the order of the floats (no NaN, no -0).
__device__ __forceinline__ int key_of(float v) {
  const int b = __float_as_int(v);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float of_key(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
constexpr int kNone = static_cast<int>(0x807fffffu);   // key_of(-inf): nothing, or unavailable

// EPT consecutive values of a row from `row`, as fp32 (-inf past E).
template <typename T, int EPT, bool VEC>
__device__ __forceinline__ void load_row(float (&l)[EPT], const T* __restrict__ row, int first, int E) {
  if constexpr (VEC) {
    constexpr int kPer = 16 / sizeof(T) < EPT ? 16 / sizeof(T) : EPT;   // values a load
#pragma unroll
    for (int i = 0; i < EPT; i += kPer) {
      alignas(16) T t[kPer];
      if (first + i < E) {   // E is a multiple of kPer
        if constexpr (kPer * sizeof(T) == 16) *reinterpret_cast<int4*>(t) = *reinterpret_cast<const int4*>(row + first + i);
        else if constexpr (kPer * sizeof(T) == 8) *reinterpret_cast<int2*>(t) = *reinterpret_cast<const int2*>(row + first + i);
        else if constexpr (kPer * sizeof(T) == 4) *reinterpret_cast<int*>(t) = *reinterpret_cast<const int*>(row + first + i);
        else t[0] = row[first + i];
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) l[i + j] = first + i < E ? to_f32(t[j]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPT; ++i) l[i] = first + i < E ? to_f32(row[first + i]) : -INFINITY;
  }
}
template <typename T, int EPT, bool VEC>
__device__ __forceinline__ void store_row(T* __restrict__ row, const float (&l)[EPT], int first, int E) {
  if constexpr (VEC) {
    constexpr int kPer = 16 / sizeof(T) < EPT ? 16 / sizeof(T) : EPT;
#pragma unroll
    for (int i = 0; i < EPT; i += kPer) {
      alignas(16) T t[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) t[j] = from_f32<T>(l[i + j]);
      if (first + i < E) {
        if constexpr (kPer * sizeof(T) == 16) *reinterpret_cast<int4*>(row + first + i) = *reinterpret_cast<const int4*>(t);
        else if constexpr (kPer * sizeof(T) == 8) *reinterpret_cast<int2*>(row + first + i) = *reinterpret_cast<const int2*>(t);
        else if constexpr (kPer * sizeof(T) == 4) *reinterpret_cast<int*>(row + first + i) = *reinterpret_cast<const int*>(t);
        else row[first + i] = t[0];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (first + i < E) row[first + i] = from_f32<T>(l[i]);
  }
}

// e / gs for e <= 1024: a half more than e is never within a rounding of a multiple of gs.
__device__ __forceinline__ int group_of(const GateArgs& a, int e) { return static_cast<int>((e + 0.5f) * a.inv_gs); }

// The groups' part of the selection: of the warp's keys v (lane holds experts lane * EPT + i) those of
// the groups that are not kept become kNone. k0 (if not 0) bounds the error of one score. A group's value is
// certain to 2 k0 and the roundings of score + bias and of the sum, which go with the summands and not with the
// sum, in which they may cancel: below 2^-23 (|t0| + |t1|), of which twice is taken for the bounds' own
// roundings. (The bounds grow with the value, so the two largest are the two largest within them too.) False is
// returned unless the least that a kept group can be is above the most that any other can be.
template <int EPT>
__device__ __forceinline__ bool keep_groups(const GateArgs& a, int (&v)[EPT], int* buf, int lane, float k0) {
  int t0 = kNone, t1 = kNone;   // the two largest of the group that this lane helps to scan
  const int lanes = a.reg_lanes > 0 ? a.reg_lanes : a.lanes, shift = __ffs(lanes) - 1;
  if (a.reg_lanes > 0) {
    // a group is the experts of `reg_lanes` whole lanes
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      t1 = max(t1, min(t0, v[i]));
      t0 = max(t0, v[i]);
    }
  } else {
    // through shared memory, `lanes` lanes a group (a group is skewed by `lanes` words from the one
    // before, so that the lanes of different groups hit other banks)
    int grp = group_of(a, lane * EPT), left = a.gs - (lane * EPT - grp * a.gs);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int e = lane * EPT + i;
      if (e < a.E) buf[e + grp * lanes] = v[i];
      if (--left == 0) {
        ++grp;
        left = a.gs;
      }
    }
    __syncwarp();
    const int g = lane >> shift, sub = lane & (lanes - 1);
    if (g < a.n) {
      const int* p = buf + g * (a.gs + lanes);
      for (int j = sub; j < a.gs; j += lanes) {
        t1 = max(t1, min(t0, p[j]));
        t0 = max(t0, p[j]);
      }
    }
  }
  for (int m = lanes >> 1; m >= 1; m >>= 1) {
    const int o0 = __shfl_xor_sync(kAll, t0, m), o1 = __shfl_xor_sync(kAll, t1, m);
    t1 = max(min(t0, o0), max(t1, o1));
    t0 = max(t0, o0);
  }
  // the sum counts the second value only where there is one
  const int grp = lane >> shift;
  const float x0 = of_key(t0), x1 = a.top2 && t1 > kNone ? of_key(t1) : 0.f;
  const float x = x0 + x1;
  // (two values of the type's lowest make -inf of the sum: the group stays available)
  const float xa = x0 > -INFINITY ? fmaxf(x, -FLT_MAX) : x0;
  int gv = grp >= a.n ? kNone : key_of(xa + 0.f);
  bool in = false;
#pragma unroll 1
  for (int j = 0; j < a.g; ++j) {   // the best group left; its lanes hold the same value, ties go to the first
    const int top = __reduce_max_sync(kAll, gv);
    if (top == kNone) break;
    const int from = (__ffs(__ballot_sync(kAll, gv == top)) - 1) >> shift;
    if (grp == from) {
      in = true;
      gv = kNone;
    }
  }
  bool sure = true;
  if (k0 > 0.f) {
    // (infinities may make a NaN of a bound: fmaxf and fminf put the infinity there that is not certain)
    const float e = 2.f * k0 + fabsf(x0) * 0x1p-22f + fabsf(x1) * 0x1p-22f;
    const int least_in = __reduce_min_sync(kAll, in ? key_of(fmaxf(x - e, -INFINITY)) : INT_MAX);
    const int most_out = __reduce_max_sync(kAll, gv > kNone ? key_of(fminf(xa + e, INFINITY)) : kNone);
    sure = most_out == kNone || least_in > most_out;
  }
  if (a.reg_lanes > 0) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) v[i] = in ? v[i] : kNone;
  } else {
    const uint32_t kept = __ballot_sync(kAll, in);
    int of = group_of(a, lane * EPT), left = a.gs - (lane * EPT - of * a.gs);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      if (of >= a.n || !((kept >> ((of << shift) & 31)) & 1u)) v[i] = kNone;
      if (--left == 0) {
        ++of;
        left = a.gs;
      }
    }
    __syncwarp();
  }
  return sure;
}

// PACKED: the low bits of a key hold EPT - 1 - i, so that a key names its place in the lane and the lower
// id of two equal values comes first. The bits are free where the values are 16-bit logits, and below
// the values' certainty where scores are compared.
template <int EPT>
constexpr int kPackMask = EPT == 1 ? 0 : EPT == 2 ? 1 : EPT == 4 ? 3 : EPT == 8 ? 7 : EPT == 16 ? 15 : 31;

// The K largest keys in order: lane j < K gets the j-th one's id in `mine` (-1 where nothing is left).
template <int EPT, bool PACKED>
__device__ __forceinline__ bool take_largest(const GateArgs& a, int (&v)[EPT], int lane, float k0, int& mine) {
  constexpr int M = kPackMask<EPT>;
  if constexpr (PACKED) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) v[i] = v[i] == kNone ? INT_MIN : (v[i] & ~M) | (M - i);
    if constexpr (EPT <= 8) {   // each lane's keys in descending order, by a sorting network of 1, 5 or 19 exchanges
      auto order = [&](int i, int j) {
        const int hi = max(v[i], v[j]), lo = min(v[i], v[j]);
        v[i] = hi;
        v[j] = lo;
      };
      if constexpr (EPT == 8) {
        order(0, 2), order(1, 3), order(4, 6), order(5, 7), order(0, 4), order(1, 5), order(2, 6), order(3, 7);
        order(0, 1), order(2, 3), order(4, 5), order(6, 7), order(2, 4), order(3, 5), order(1, 4), order(3, 6);
        order(1, 2), order(3, 4), order(5, 6);
      } else if constexpr (EPT == 4) {
        order(0, 2), order(1, 3), order(0, 1), order(2, 3), order(1, 2);
      } else if constexpr (EPT == 2) {
        order(0, 1);
      }
    }
  }
  constexpr int kLow = PACKED ? INT_MIN : kNone;
  int best = kLow, key = kLow, lane_of = 0;   // lane k: the k-th key and its lane
  int top = kLow;
  if constexpr (PACKED && EPT <= 8) {
    best = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < EPT; ++i) best = max(best, v[i]);
  }
  int at = 0;
  const int rounds = k0 > 0.f ? a.K + 1 : a.K;   // one more for the distance of the last from the first left out
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    // without the places, which order equal values within a lane only
    const int value = PACKED ? best & ~M : best;
    top = __reduce_max_sync(kAll, value);
    if (top == kLow) break;
    const int from = __ffs(__ballot_sync(kAll, value == top)) - 1;  // ids grow with the lane
    const int won = PACKED ? __shfl_sync(kAll, best, from) : top;
    if (lane == k) {
      key = won;
      lane_of = from;
    }
    if constexpr (PACKED && EPT <= 8) {
      if (lane == from) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) v[i] = i + 1 < EPT ? v[i + 1] : INT_MIN;
      }
      best = v[0];
    } else if constexpr (PACKED) {
      if (lane == from) {
        best = INT_MIN;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          v[i] = v[i] == won ? INT_MIN : v[i];
          best = max(best, v[i]);
        }
      }
    } else {
      int p = 0;
      if (lane == from) {
        best = kNone;
        bool gone = false;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          if (!gone && v[i] == top) {
            p = i;
            v[i] = kNone;
            gone = true;
          }
          best = max(best, v[i]);
        }
      }
      p = __shfl_sync(kAll, p, from);
      if (lane == k) at = p;
    }
  }
  mine = key == kLow || lane >= a.K ? -1 : lane_of * EPT + (PACKED ? M - (key & M) : at);
  if (k0 > 0.f) {
    // each of the K against the next one (the last against the first left out): the scores' errors, the
    // bias's roundings and the low bits that packing took
    int next = __shfl_down_sync(kAll, key, 1);
    if (lane == a.K - 1) next = top;
    const float x = of_key(PACKED ? key & ~M : key), y = of_key(PACKED ? next & ~M : next);
    const bool near = lane < a.K && key != kLow && next != kLow &&
                      !(x - y > 2.f * k0 + (fabsf(x) + fabsf(y)) * (PACKED ? (M + 2) * 0x1p-23f : 0x1p-23f));
    return !__any_sync(kAll, near);
  }
  return true;
}

// The same selection with scores in fp64, for the rows that need it: one value of shared memory an
// expert, every step in order.
__device__ __noinline__ int select_f64(const GateArgs& a, const float* l, int ept, double* v, int lane) {
  double top = -static_cast<double>(INFINITY), sum = 0;
  if (!a.sigmoid) {
    for (int i = 0; i < ept; ++i) top = fmax(top, static_cast<double>(l[i]));
    top = warp_max(top);
    for (int i = 0; i < ept; ++i) sum += l[i] > -INFINITY ? exp(static_cast<double>(l[i]) - top) : 0.0;
    sum = warp_sum(sum);
  }
  const double none = -static_cast<double>(INFINITY);
  for (int i = 0; i < ept; ++i) {
    const int e = lane * ept + i;
    if (e >= a.E) continue;
    const double x = l[i];
    double s = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum;
    if (a.bias != nullptr) s += static_cast<double>(a.bias[e]);
    v[e] = l[i] > -INFINITY && s == s ? s : none;
  }
  __syncwarp();
  if (a.n > 1) {
    double t0 = none, t1 = none;   // lane j: group j
    for (int j = 0; lane < a.n && j < a.gs; ++j) {
      const double x = v[lane * a.gs + j];
      if (x > t0) {
        t1 = t0;
        t0 = x;
      } else if (x > t1) {
        t1 = x;
      }
    }
    const double gv = a.top2 && t1 > none ? t0 + t1 : t0;
    int rank = 0;
    for (int j = 0; j < a.n; ++j) {
      const double o = __shfl_sync(kAll, gv, j);
      rank += (o > gv || (o == gv && j < lane)) ? 1 : 0;
    }
    const uint32_t kept = __ballot_sync(kAll, lane < a.n && rank < a.g && gv > none);
    for (int e = lane; e < a.E; e += 32)
      if (!((kept >> (e / a.gs)) & 1u)) v[e] = none;
    __syncwarp();
  }
  int mine = -1;
  for (int k = 0; k < a.K; ++k) {
    double best = none;
    int at = INT_MAX;
    for (int e = lane; e < a.E; e += 32)
      if (v[e] > best) {
        best = v[e];
        at = e;
      }
    const double top_v = warp_max(best);
    if (top_v == none) break;
    const int id = __reduce_min_sync(kAll, best == top_v ? at : INT_MAX);
    if (lane == k) mine = id;
    __syncwarp();
    if (lane == 0) v[id] = none;
    __syncwarp();
  }
  return mine;
}

template <typename T, int EPT, bool VEC>
__global__ void __launch_bounds__(kGateWarps * 32, EPT <= 8 ? 12 : 1) gate_kernel(GateArgs a) {
  extern __shared__ double gate_smem[];
  const int lane = lane_id(), warp = warp_id();
  const int t = blockIdx.x * kGateWarps + warp;
  if (t >= a.T) return;  // whole warps only: no barrier follows
  double* buf = gate_smem + static_cast<int64_t>(warp) * (a.E + 32);
  const T* row = static_cast<const T*>(a.logits) + static_cast<int64_t>(t) * a.stride;
  float l[EPT];
  load_row<T, EPT, VEC>(l, row, lane * EPT, a.E);
  const bool direct = a.bias == nullptr && (a.n == 1 || !a.top2);
#pragma unroll
  for (int i = 0; i < EPT; ++i) l[i] = clean_logit(l[i]);
  float m = 0.f, sum = 1.f;
  if (!a.sigmoid && !(direct && a.renorm)) {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; ++i) m = fmaxf(m, l[i]);
    m = of_key(__reduce_max_sync(kAll, key_of(m)));
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) sum += l[i] > -INFINITY ? __expf(l[i] - m) : 0.f;
    sum = warp_sum(sum);
  }
  int v[EPT];
  float k0 = 0.f;
  if (direct) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) v[i] = key_of(l[i]);
  } else {
    const float inv = __fdividef(1.f, sum);
    float bias[EPT];
    if (a.bias != nullptr) load_row<float, EPT, VEC>(bias, a.bias, lane * EPT, a.E);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float x = __expf(a.sigmoid ? -l[i] : l[i] - m);
      float c = a.sigmoid ? __fdividef(1.f, 1.f + x) : x * inv;
      if (a.bias != nullptr) c = fmaxf(c + bias[i], -INFINITY);   // (a NaN is dropped)
      v[i] = l[i] > -INFINITY ? key_of(c + 0.f) : kNone;
    }
    // Bound of one score's error, k0. With the documented errors of __expf (2 + 1.173 |x| units of 2^-23)
    // and __fdividef (2 units):  sigmoid: s (1 - s) (2 + 1.173 |x|) + 1/2 + 2 < 3.3 units, so 2^-20;
    // softmax, relative to the largest score: 3 units each for the exponential and the sum's terms, 18
    // for adding up to 1024 of them, 2 for the quotient: 26 units, so 2^-18.
    k0 = a.sigmoid ? 0x1p-20f : inv * 0x1p-18f;
  }
  bool sure = true;
  if (a.n > 1) sure = keep_groups<EPT>(a, v, reinterpret_cast<int*>(buf), lane, k0);
  int mine;
  // packed keys: 16-bit logits end in 16 zero bits as fp32, and scores are certain to 2^-18 at best
  const bool packed = sizeof(T) == 2 || !direct;
  if (!(packed ? take_largest<EPT, true>(a, v, lane, k0, mine) : take_largest<EPT, false>(a, v, lane, k0, mine))) sure = false;
  if (!sure) mine = select_f64(a, l, EPT, buf, lane);
  // weights from the logits of the chosen
  const float x = mine >= 0 ? clean_logit(to_f32(row[mine])) : -INFINITY;
  const bool has = mine >= 0;
  float w = 0.f;
  if (a.renorm) {
    // both scores are proportional to exp(x - r) times a factor between 1/2 and 1 (sigmoid) or 1;
    // r keeps the sum from underflowing
    const float top = of_key(__reduce_max_sync(kAll, key_of(x)));
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
template <typename T, int EPT, bool VEC>
__global__ void __launch_bounds__(kGateWarps * 32) gate_bwd_kernel(GateBwdArgs a) {
  extern __shared__ float gate_bwd_smem[];
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
    load_row<T, EPT, VEC>(l, row, lane * EPT, a.E);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      l[i] = clean_logit(l[i]);
      m = fmaxf(m, l[i]);
    }
    m = warp_max(m);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      l[i] = l[i] > -INFINITY ? __expf(l[i] - m) : 0.f;
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
  // the chosen experts' values into the row: through shared memory, or one by one where an id occurs twice
  float out[EPT];
  const uint32_t same = __match_any_sync(kAll, id >= 0 ? id : -1 - lane);
  if (__all_sync(kAll, (same & (same - 1)) == 0)) {
    float* buf = gate_bwd_smem + warp * 32 * EPT;
#pragma unroll
    for (int i = 0; i < EPT; ++i) buf[i * 32 + lane] = 0.f;
    __syncwarp();
    // expert e lies at [e % EPT][e / EPT], so that the lanes read their own without bank conflicts
    if (id >= 0) buf[id % EPT * 32 + id / EPT] = gk;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < EPT; ++i) out[i] = buf[i * 32 + lane];
  } else {
#pragma unroll
    for (int i = 0; i < EPT; ++i) out[i] = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int e = __shfl_sync(kAll, id, k);
      const float g = __shfl_sync(kAll, gk, k);
#pragma unroll
      for (int i = 0; i < EPT; ++i)
        if (e == lane * EPT + i) out[i] += g;
    }
  }
  if (whole) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) out[i] = l[i] * inv * (out[i] - dot);
  }
  store_row<T, EPT, VEC>(static_cast<T*>(a.d) + static_cast<int64_t>(t) * a.E, out, lane * EPT, a.E);
}

// Whether rows of `ept` values a lane can be moved in the widest words that hold them.
template <typename T>
bool rows_align(const void* p, int64_t stride, int E, int ept) {
  const int64_t per = std::min<int64_t>(16 / sizeof(T), ept), bytes = per * sizeof(T);
  return E % per == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * static_cast<int64_t>(sizeof(T)) % bytes == 0;
}

template <typename T, int EPT>
void launch_gate_ept(GateArgs a, cudaStream_t s) {
  const int grid = (a.T + kGateWarps - 1) / kGateWarps;
  const size_t smem = sizeof(double) * kGateWarps * (a.E + 32);
  const int lanes = a.gs / EPT;
  a.reg_lanes = a.gs % EPT == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  if (rows_align<T>(a.logits, a.stride, a.E, EPT) && (a.bias == nullptr || rows_align<float>(a.bias, a.E, a.E, EPT)))
    gate_kernel<T, EPT, true><<<grid, kGateWarps * 32, smem, s>>>(a);
  else gate_kernel<T, EPT, false><<<grid, kGateWarps * 32, smem, s>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
template <typename T, int EPT>
void launch_gate_bwd_ept(const GateBwdArgs& a, cudaStream_t s) {
  const int grid = (a.T + kGateWarps - 1) / kGateWarps;
  const size_t smem = sizeof(float) * kGateWarps * 32 * EPT;
  if (rows_align<T>(a.logits, a.stride, a.E, EPT) && rows_align<T>(a.d, a.E, a.E, EPT))
    gate_bwd_kernel<T, EPT, true><<<grid, kGateWarps * 32, smem, s>>>(a);
  else gate_bwd_kernel<T, EPT, false><<<grid, kGateWarps * 32, smem, s>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
template <typename T>
void launch_gate(const GateArgs& a, cudaStream_t s) {
  if (a.E <= 32) launch_gate_ept<T, 1>(a, s);
  else if (a.E <= 64) launch_gate_ept<T, 2>(a, s);
  else if (a.E <= 128) launch_gate_ept<T, 4>(a, s);
  else if (a.E <= 256) launch_gate_ept<T, 8>(a, s);
  else if (a.E <= 512) launch_gate_ept<T, 16>(a, s);
  else launch_gate_ept<T, 32>(a, s);
}
template <typename T>
void launch_gate_bwd(const GateBwdArgs& a, cudaStream_t s) {
  if (a.E <= 32) launch_gate_bwd_ept<T, 1>(a, s);
  else if (a.E <= 64) launch_gate_bwd_ept<T, 2>(a, s);
  else if (a.E <= 128) launch_gate_bwd_ept<T, 4>(a, s);
  else if (a.E <= 256) launch_gate_bwd_ept<T, 8>(a, s);
  else if (a.E <= 512) launch_gate_bwd_ept<T, 16>(a, s);
  else launch_gate_bwd_ept<T, 32>(a, s);
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
  a.inv_gs = 1.f / a.gs;
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
  at::Tensor idx = at::detail::empty_cuda({a.T, a.K}, at::kLong, logits.device(), c10::nullopt);
  at::Tensor w = at::detail::empty_cuda({a.T, a.K}, at::kFloat, logits.device(), c10::nullopt);
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
  at::Tensor d = at::detail::empty_cuda({a.T, a.E}, logits.scalar_type(), logits.device(), c10::nullopt);
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
