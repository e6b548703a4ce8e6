// Grouped fp8 GEMM with one fp32 scale per block of 128, on tcgen05 + TMEM.
//
//   C[rows of g] = (A * sa)[rows of g] @ (B[g] * sb[g])^T
//     A  [rows, K] e4m3, sa one fp32 per (row, 128 channels of K)      (what a dispatch delivers)
//     B  [G, N, K] e4m3 (or [G, K, N], read in place), sb one fp32 per 128 x 128 block
//
// The scales are arbitrary fp32 numbers, so the tensor cores cannot apply them (their block-scaled
// form takes powers of two). A block of 128 products is summed unscaled in tensor memory,
//     T[i, j] = sum_{k in block} a_ik b_jk ,
// and the epilogue warps add sa[i, block] * sb[j / 128, block] * T[i, j] to sums that stay in
// their registers for the whole of K, while the next block is multiplied into the other of two
// TMEM buffers. Per 128 x 256 tile and block that is 32 KFMA on the CUDA cores, as pairs
// (fma.rn.f32x2) 128 issue cycles a scheduler against the 512 cycles of the four MMAs.
//
// Rows come as segments (offsets) or as G slabs of `cap` rows of which counts[g] are in use
// (masked, what a low-latency dispatch delivers); rows outside a group are neither written nor
// used: every row has accumulators of its own.
//
// Epilogues: bf16, fp32, or SwiGLU with quantisation: a 256-wide tile holds 128 gate and 128 up
// columns, so it holds whole 128-blocks of h = silu(gate) * up, which leave as e4m3 with one
// fp32 scale per row and block (scale = max(amax, 1e-4) / 448), the operand of the next product.
//
// 12 warps: TMA producer, TMEM owner + MMA issuer, two idle, 8 epilogue warps (two per TMEM lane quarter,
// 128 columns each). Every wait is bounded; a wait that runs out sets *error, lets the copies in
// flight land, frees the TMEM and returns.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "ops.h"
#include "tcgen05.cuh"

namespace b200ep {
namespace gemm {
namespace {

constexpr int kBM = 128, kBN = 256, kBK = 128;   // tile; kBK one-byte elements fill a swizzle row
constexpr int kStages = 4;
constexpr int kABytes = kBM * kBK, kBBytes = kBN * kBK, kStageBytes = kABytes + kBBytes;
constexpr int kEpiWarps = 8;
constexpr int kFirstEpi = 4;                     // warps 0 and 1 load and multiply, 2 and 3 only lend registers
constexpr int kBlkThreads = 32 * (kFirstEpi + kEpiWarps);
// Registers a thread: 128 sums and their operands need more than an even split of the file
// (168). The first warpgroup gives up what the two epilogue warpgroups take:
// 128 * 64 + 256 * 208 = 61440 of the 384 * 168 = 64512 the block is launched with.
constexpr int kRegsMain = 64, kRegsEpi = 208;
constexpr int kWarpStage = 32 * 64;              // a warp's output staging: 64 bytes of its 32 rows
constexpr int kMaxG = 1024;

enum BlkEpilogue : int { kOutBF16 = 0, kOutF32 = 1, kOutSwiGLU = 2 };

struct BlkArgs {
  const int64_t* offsets;   // [G + 1] or nullptr (masked)
  const int32_t* counts;    // [G] or nullptr
  int G, rows, N, K;        // rows: of A (segments) or of one slab (masked)
  const float* sa;
  int64_t sa_row, sa_group;
  const float* sb;
  int64_t sb_group, sb_n, sb_k;
  uint8_t* C;               // bf16 or fp32; byte strides
  int64_t c_row, c_group;
  uint8_t* H;
  int64_t h_row, h_group;
  float* Hs;
  int64_t hs_row, hs_group;
  uint32_t* error;
  uint64_t timeout_ns;
};

__device__ __forceinline__ void tc_mma_fp8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D fp32, A and B e4m3, M = 128; bit 16 selects an MN-major B
__host__ __device__ constexpr uint32_t idesc_fp8(int n, bool b_mn) {
  return (1u << 4) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ bool wait_blk(uint64_t* bar, uint32_t parity, const BlkArgs& a, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort || global_ns() - t0 > a.timeout_ns) {
      atomicExch(a.error, 1u);
      *abort = 1;
      return false;
    }
  }
  return true;
}

struct Groups {
  int base[kMaxG];       // first row (segments) or 0
  int cnt[kMaxG];        // rows in use
  int pref[kMaxG + 1];   // m tiles of the groups before
};

// Rows and m tiles of every group, from the device's offsets / counts, clamped to the buffer.
__device__ __forceinline__ void load_groups(Groups& s, const BlkArgs& a) {
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
    int64_t b = 0, c = a.rows;
    if (a.offsets != nullptr) {
      const int64_t lo = a.offsets[g], hi = a.offsets[g + 1], top = a.rows;
      b = lo < 0 ? 0 : (lo > top ? top : lo);
      const int64_t e = hi > top ? top : hi;
      c = e > b ? e - b : 0;
    }
    if (a.counts != nullptr) {
      const int64_t n = a.counts[g];
      c = n < 0 ? 0 : (n < c ? n : c);
    }
    s.base[g] = static_cast<int>(b);
    s.cnt[g] = static_cast<int>(c);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int g0 = 0; g0 < a.G; g0 += 32) {
      int v = g0 + lane < a.G ? (s.cnt[g0 + lane] + kBM - 1) / kBM : 0;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, m);
        if (lane >= m) v += o;
      }
      if (g0 + lane < a.G) s.pref[g0 + lane + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) s.pref[0] = 0;
  }
}

struct BlkTile {
  int g, m0, n0;
};
__device__ __forceinline__ bool blk_tile(int t, const BlkArgs& a, const Groups& s, BlkTile& tl) {
  const int ntn = (a.N + kBN - 1) / kBN;
  const int mt = t / ntn;
  if (mt >= s.pref[a.G]) return false;
  int lo = 0, hi = a.G - 1;   // last group with pref[g] <= mt
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.pref[mid] <= mt) lo = mid; else hi = mid - 1;
  }
  tl.g = lo;
  tl.m0 = (mt - s.pref[lo]) * kBM;
  tl.n0 = (t - mt * ntn) * kBN;
  return true;
}

template <int EPI, bool B_MN>
__global__ void __launch_bounds__(kBlkThreads, 1)
    gemm_block_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, BlkArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kStages * kABytes;
  uint8_t* sE = sB + kStages * kBBytes;
  __shared__ Groups s_grp;
  __shared__ uint64_t full[kStages], empty[kStages], tfull[2], tempty[2], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_abort;
  __shared__ uint32_t s_amax[2][2][kBM];   // [tile parity][column half][row]

  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], kEpiWarps);
    }
    mbar_init(&drain, 1);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 2 * kBN);
  load_groups(s_grp, a);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  const int KB = (a.K + kBK - 1) / kBK;

  if (warp < kFirstEpi) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMain));
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      if (lane == 0) {
        uint32_t it = 0;
        BlkTile tl;
        for (int t = blockIdx.x; !s_abort && blk_tile(t, a, s_grp, tl); t += gridDim.x) {
          const int row = a.offsets != nullptr ? s_grp.base[tl.g] + tl.m0 : tl.m0;
          const int slab = a.offsets != nullptr ? 0 : tl.g;
          for (int kb = 0; kb < KB; ++kb, ++it) {
            const int s = it % kStages;
            if (!wait_blk(&empty[s], ((it / kStages) & 1u) ^ 1u, a, &s_abort)) break;
            mbar_arrive_expect_tx(&full[s], kStageBytes);
            tma_load_3d(sA + s * kABytes, &tmA, &full[s], kb * kBK, row, slab);
            uint8_t* db = sB + s * kBBytes;
            if (B_MN) {
#pragma unroll
              for (int j = 0; j < kBN / 128; ++j)
                tma_load_3d(db + j * (128 * kBK), &tmB, &full[s], tl.n0 + 128 * j, kb * kBK, tl.g);
            } else {
              tma_load_3d(db, &tmB, &full[s], kb * kBK, tl.n0, tl.g);
            }
          }
        }
        if (s_abort) {  // copies in flight land before the CTA's shared memory is given up
          for (uint32_t q = it > kStages ? it - kStages : 0; q < it; ++q)
            mbar_wait(&full[q % kStages], (q / kStages) & 1u, 1000000000ull);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_fp8(kBN, B_MN);
        uint32_t it = 0;
        BlkTile tl;
        for (int t = blockIdx.x; !s_abort && blk_tile(t, a, s_grp, tl); t += gridDim.x) {
          for (int kb = 0; kb < KB; ++kb, ++it) {
            const int s = it % kStages, b = it & 1;
            if (!wait_blk(&tempty[b], ((it >> 1) & 1u) ^ 1u, a, &s_abort)) break;
            if (!wait_blk(&full[s], (it / kStages) & 1u, a, &s_abort)) break;
            tc_fence_after();
            const uint64_t ad = smem_desc_k128(sA + s * kABytes);
            const uint64_t bd = B_MN ? smem_desc_mn128(sB + s * kBBytes, 128 * kBK) : smem_desc_k128(sB + s * kBBytes);
            // next 32 channels: 32 bytes along a K-major swizzle row, or 32 rows of 128 bytes
            constexpr uint64_t bstep = B_MN ? (32 * 128) >> 4 : 2;
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k)
              tc_mma_fp8(tmem_base + b * kBN, ad + 2 * k, bd + bstep * k, idesc, k > 0 ? 1u : 0u);
            tc_commit(&empty[s]);
            tc_commit(&tfull[b]);
          }
        }
        tc_commit(&drain);  // every MMA issued is done before TMEM is released
        mbar_wait(&drain, 0, a.timeout_ns);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3;                 // TMEM lane quarter this warp may read
    const int half = (warp - kFirstEpi) >> 2;
    uint8_t* stage = sE + (warp - kFirstEpi) * kWarpStage;
    // this warp's 32-column chunk c of the tile: its 128 columns, or 64 gate and 64 up columns
    auto col_of = [half](int c) {
      return EPI == kOutSwiGLU ? (c < 2 ? half * 64 + 32 * c : 128 + half * 64 + 32 * (c - 2)) : half * 128 + 32 * c;
    };
    const int NB = (a.N + 127) / 128;
    uint32_t it = 0;
    int parity = 0;
    BlkTile tl;
    for (int t = blockIdx.x; !s_abort && blk_tile(t, a, s_grp, tl); t += gridDim.x, parity ^= 1) {
      const int cnt = s_grp.cnt[tl.g];
      const int row = tl.m0 + q * 32 + lane;           // within the group
      const int64_t arow = s_grp.base[tl.g] + min(row, cnt - 1);
      const float* sa = a.sa + tl.g * a.sa_group + arow * a.sa_row;
      const int nb = tl.n0 / 128;
      const int nb0 = EPI == kOutSwiGLU ? nb : min(nb + half, NB - 1);
      const int nb1 = EPI == kOutSwiGLU ? nb + 1 : nb0;
      const float* sb0 = a.sb + tl.g * a.sb_group + nb0 * a.sb_n;
      const float* sb1 = a.sb + tl.g * a.sb_group + nb1 * a.sb_n;
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      float na = sa[0], n0s = sb0[0], n1s = sb1[0];
      bool ok = true;
      for (int kb = 0; kb < KB; ++kb, ++it) {
        const int b = it & 1;
        const float f0 = na * n0s, f1 = EPI == kOutSwiGLU ? na * n1s : f0;
        if (kb + 1 < KB) {
          na = sa[kb + 1];
          n0s = sb0[(kb + 1) * a.sb_k];
          if (EPI == kOutSwiGLU) n1s = sb1[(kb + 1) * a.sb_k];
        }
        if (!wait_blk(&tfull[b], (it >> 1) & 1u, a, &s_abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * kBN;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(taddr + col_of(c), r);
          const uint32_t f = __float_as_uint(c < 2 ? f0 : f1);
          const uint64_t ff = pack2(f, f);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fma2(pack2(r[2 * i], r[2 * i + 1]), ff, acc[c * 16 + i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[b]);
      }
      if (!ok) break;
      // ---- output: 64 bytes of each of the warp's 32 rows at a time, through shared memory (the
      // 16-byte pieces of a row are swapped by row pair, so that 8 lanes hit distinct banks)
      const int first = tl.m0 + q * 32;
      const int64_t grow = s_grp.base[tl.g] + first;
      auto store64 = [&](uint8_t* base, int64_t row_stride, int ncols16, const uint32_t (&v)[16]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<int4*>(stage + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)) =
              make_int4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = j * 8 + (lane >> 2), c = lane & 3;
          const int4 o = *reinterpret_cast<const int4*>(stage + r * 64 + ((c ^ (r >> 1 & 3)) << 4));
          if (first + r < cnt && c < ncols16) *reinterpret_cast<int4*>(base + r * row_stride + 16 * c) = o;
        }
        __syncwarp();
      };
      uint8_t* crow = a.C + tl.g * a.c_group + grow * a.c_row;
      if (EPI == kOutF32) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int col = tl.n0 + half * 128 + 16 * c;
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float x, y;
            unpack2(acc[c * 8 + i], x, y);
            v[2 * i] = __float_as_uint(x);
            v[2 * i + 1] = __float_as_uint(y);
          }
          store64(crow + 4 * static_cast<int64_t>(col), a.c_row, (a.N - col) / 4, v);
        }
      } else if (EPI == kOutBF16 || a.C != nullptr) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = tl.n0 + col_of(c);
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x, y;
            unpack2(acc[c * 16 + i], x, y);
            v[i] = pack_bf16(x, y);
          }
          store64(crow + 2 * static_cast<int64_t>(col), a.c_row, (a.N - col) / 8, v);
        }
      }
      if (EPI == kOutSwiGLU) {
        // h = silu(gate) * up of 64 of the block's 128 columns; the other half's warp has the rest
        float h[64];
        uint32_t top = 0;   // as bits, so that a NaN stays the largest
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float g0, g1, u0, u1;
          unpack2(acc[i], g0, g1);
          unpack2(acc[32 + i], u0, u1);
          h[2 * i] = __fdividef(g0, 1.f + __expf(-g0)) * u0;
          h[2 * i + 1] = __fdividef(g1, 1.f + __expf(-g1)) * u1;
          top = max(top, max(__float_as_uint(fabsf(h[2 * i])), __float_as_uint(fabsf(h[2 * i + 1]))));
        }
        s_amax[parity][half][q * 32 + lane] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");  // this warp and the other half's
        top = max(max(top, s_amax[parity][half ^ 1][q * 32 + lane]), __float_as_uint(1e-4f));
        const float amax = __uint_as_float(top);
        const float inv = __fdiv_rn(448.f, amax);
        uint32_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = uint32_t(f32x2_to_e4m3x2(h[4 * i] * inv, h[4 * i + 1] * inv)) |
                 (uint32_t(f32x2_to_e4m3x2(h[4 * i + 2] * inv, h[4 * i + 3] * inv)) << 16);
        store64(a.H + tl.g * a.h_group + grow * a.h_row + tl.n0 / 2 + half * 64, a.h_row, 4, v);
        if (half == 0 && row < cnt)
          a.Hs[tl.g * a.hs_group + (grow + lane) * a.hs_row + tl.n0 / 256] = __fdiv_rn(amax, 448.f);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * kBN);
  }
}

// ----------------------------------------------------------------------------- host side
// One-byte 3-D map [d2, d1, d0] (strides in bytes), boxes of box1 x 128 bytes, 128B swizzle.
CUtensorMap map_u8_3d(const void* base, int64_t d0, int64_t d1, int64_t d2, int64_t s1, int64_t s2, int box1) {
  TORCH_CHECK((reinterpret_cast<uintptr_t>(base) & 15) == 0, "operands must start on a 16-byte boundary");
  TORCH_CHECK(s1 % 16 == 0 && s2 % 16 == 0, "operand strides must be multiples of 16 bytes");
  CUtensorMap m;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(d0), static_cast<cuuint64_t>(d1), static_cast<cuuint64_t>(d2)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(s1), static_cast<cuuint64_t>(s2)};
  cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box1), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encoder()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (fp8) failed: " + std::to_string(static_cast<int>(r)));
  return m;
}

template <int EPI, bool B_MN>
void launch_block(const CUtensorMap& ma, const CUtensorMap& mb, const BlkArgs& a, int grid, cudaStream_t stream) {
  constexpr int smem = 1024 + kStages * kStageBytes + kEpiWarps * kWarpStage;
  auto kfn = gemm_block_kernel<EPI, B_MN>;
  static std::atomic<uint64_t> seen{0};
  AT_CUDA_CHECK(set_smem_limit_once(seen, kfn, smem));
  kfn<<<grid, kBlkThreads, smem, stream>>>(ma, mb, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

bool on(const at::Tensor& t, const at::Tensor& like) { return t.device() == like.device(); }

// An output with the rows of A: [rows, cols] or [G, cap, cols], unit inner stride, 16-byte rows.
void check_out(const at::Tensor& t, const at::Tensor& A, int64_t cols, int align, const char* what) {
  TORCH_CHECK(on(t, A) && t.dim() == A.dim() && t.size(-1) == cols && unit_inner(t), what,
              " must have A's leading sizes, the product's columns and unit inner stride, on A's device");
  for (int64_t d = 0; d + 1 < A.dim(); ++d) TORCH_CHECK(t.size(d) == A.size(d), what, " must have A's leading sizes");
  const int64_t es = t.element_size();
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) % align) == 0 && t.stride(-2) * es % align == 0 &&
                  (t.dim() == 2 || t.stride(0) * es % align == 0),
              what, " must have rows on 16-byte boundaries");
}

}  // namespace
}  // namespace gemm

void grouped_gemm_fp8_block(const at::Tensor& A, const at::Tensor& sa, const at::Tensor& B, const at::Tensor& sb,
                            const OptTensor& offsets, const OptTensor& counts, const OptTensor& C, const OptTensor& H,
                            const OptTensor& Hs, int64_t epilogue, const at::Tensor& error, int64_t num_sms,
                            double timeout_s, bool b_kn) {
  using namespace gemm;
  auto e4m3 = [](const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte; };
  TORCH_CHECK((A.dim() == 2 || A.dim() == 3) && e4m3(A) && unit_inner(A),
              "A must be e4m3 [rows, K] or [G, cap, K] with unit inner stride");
  TORCH_CHECK(on(B, A) && B.dim() == 3 && e4m3(B) && B.is_contiguous(),
              "B must be contiguous e4m3 [G, N, K] (or [G, K, N] with b_layout 'kn') on A's device");
  const bool masked = A.dim() == 3;
  BlkArgs a{};
  a.G = static_cast<int>(B.size(0));
  const int64_t N = b_kn ? B.size(2) : B.size(1), K = b_kn ? B.size(1) : B.size(2);
  TORCH_CHECK(a.G >= 1 && a.G <= kMaxG, "need 1 <= G <= 1024");
  TORCH_CHECK(K == A.size(-1) && K >= 16 && K % 16 == 0, "K must agree between A and B and be a multiple of 16");
  TORCH_CHECK(N >= 8 && N % (b_kn ? 16 : 8) == 0, "N must be a multiple of 8 (16 for b_layout 'kn')");
  TORCH_CHECK(N < (1 << 30) && K < (1 << 30) && A.size(-2) < (1 << 30), "sizes below 2^30");
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.rows = static_cast<int>(A.size(-2));
  const int64_t KB = (K + 127) / 128, NB = (N + 127) / 128;
  TORCH_CHECK(on(sa, A) && sa.scalar_type() == at::kFloat && sa.dim() == A.dim() && sa.size(-1) == KB && unit_inner(sa),
              "sa must be fp32 with A's leading sizes and ceil(K / 128) columns");
  for (int64_t d = 0; d + 1 < A.dim(); ++d) TORCH_CHECK(sa.size(d) == A.size(d), "sa must have A's leading sizes");
  TORCH_CHECK(on(sb, A) && sb.scalar_type() == at::kFloat && sb.dim() == 3 && sb.is_contiguous() &&
                  sb.size(0) == a.G && sb.size(1) == (b_kn ? KB : NB) && sb.size(2) == (b_kn ? NB : KB),
              "sb must be contiguous fp32 with one scale per 128 x 128 block of B");
  TORCH_CHECK(masked != offsets.has_value(), "2-D A needs offsets [G + 1]; 3-D A takes counts [G] only");
  TORCH_CHECK(!masked || A.size(0) == a.G, "3-D A must have one slab per group");
  if (offsets.has_value()) {
    TORCH_CHECK(on(*offsets, A) && offsets->scalar_type() == at::kLong && offsets->dim() == 1 &&
                    offsets->size(0) == a.G + 1 && offsets->is_contiguous(),
                "offsets must be contiguous int64 [G + 1]");
    a.offsets = offsets->data_ptr<int64_t>();
  }
  if (counts.has_value()) {
    TORCH_CHECK(on(*counts, A) && counts->scalar_type() == at::kInt && counts->dim() == 1 &&
                    counts->size(0) == a.G && counts->is_contiguous(),
                "counts must be contiguous int32 [G]");
    a.counts = counts->data_ptr<int32_t>();
  }
  TORCH_CHECK(epilogue >= 0 && epilogue <= 2 && !(epilogue == kOutSwiGLU && b_kn),
              "unknown epilogue (SwiGLU takes b_layout 'nk')");
  if (epilogue == kOutSwiGLU) {
    TORCH_CHECK(N % 256 == 0, "SwiGLU needs N to be a multiple of 256 (128 gate, 128 up columns)");
    TORCH_CHECK(H.has_value() && Hs.has_value() && e4m3(*H) && Hs->scalar_type() == at::kFloat,
                "SwiGLU needs an e4m3 h and its fp32 scales");
    check_out(*H, A, N / 2, 16, "h");
    check_out(*Hs, A, N / 256, 4, "the scales of h");
    a.H = static_cast<uint8_t*>(H->data_ptr());
    a.h_row = H->stride(-2);
    a.h_group = masked ? H->stride(0) : 0;
    a.Hs = Hs->data_ptr<float>();
    a.hs_row = Hs->stride(-2);
    a.hs_group = masked ? Hs->stride(0) : 0;
  }
  TORCH_CHECK(C.has_value() || epilogue == kOutSwiGLU, "an output is required");
  if (C.has_value()) {
    TORCH_CHECK(C->scalar_type() == (epilogue == kOutF32 ? at::kFloat : at::kBFloat16),
                "the output's type does not match the epilogue");
    check_out(*C, A, N, 16, "the output");
    a.C = static_cast<uint8_t*>(C->data_ptr());
    a.c_row = C->stride(-2) * C->element_size();
    a.c_group = masked ? C->stride(0) * C->element_size() : 0;
  }
  if (!A.is_cuda() || a.rows == 0) return;  // CPU tensors: the checks alone
  const c10::cuda::CUDAGuard guard(A.device());
  TORCH_CHECK(on(error, A) && error.scalar_type() == at::kInt, "error word");
  a.sa = sa.data_ptr<float>();
  a.sa_row = sa.stride(-2);
  a.sa_group = masked ? sa.stride(0) : 0;
  a.sb = sb.data_ptr<float>();
  a.sb_group = NB * KB;
  a.sb_n = b_kn ? 1 : KB;
  a.sb_k = b_kn ? NB : 1;
  a.error = reinterpret_cast<uint32_t*>(error.data_ptr<int32_t>());
  a.timeout_ns = static_cast<uint64_t>(timeout_s * 1e9);
  // a stride over a dimension of one element is arbitrary; the map wants a legal one
  auto stride = [](const at::Tensor& t, int64_t d, int64_t otherwise) { return t.size(d) > 1 ? t.stride(d) : otherwise; };
  const int64_t s1 = stride(A, A.dim() - 2, K);
  const CUtensorMap ma = masked ? map_u8_3d(A.data_ptr(), K, a.rows, a.G, s1, stride(A, 0, s1 * a.rows), kBM)
                                : map_u8_3d(A.data_ptr(), K, a.rows, 1, s1, s1 * a.rows, kBM);
  const CUtensorMap mb = b_kn ? map_u8_3d(B.data_ptr(), N, K, a.G, N, N * K, kBK)
                              : map_u8_3d(B.data_ptr(), K, N, a.G, K, N * K, kBN);
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int grid = num_sms > 0 ? static_cast<int>(std::min<int64_t>(num_sms, sms)) : sms;
  auto stream = at::cuda::getCurrentCUDAStream();
  if (epilogue == kOutSwiGLU) launch_block<kOutSwiGLU, false>(ma, mb, a, grid, stream);
  else if (epilogue == kOutBF16 && b_kn) launch_block<kOutBF16, true>(ma, mb, a, grid, stream);
  else if (epilogue == kOutBF16) launch_block<kOutBF16, false>(ma, mb, a, grid, stream);
  else if (b_kn) launch_block<kOutF32, true>(ma, mb, a, grid, stream);
  else launch_block<kOutF32, false>(ma, mb, a, grid, stream);
}

}  // namespace b200ep
