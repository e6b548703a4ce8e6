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
// TMEM buffers. Per 128 x 256 tile and block that is 32 KFMA on the CUDA cores, 256 cycles of
// their pipes against the 512 cycles of the four MMAs (packed fma.rn.f32x2 has the same rate, and
// cost a move for almost every pair).
//
// Rows come as segments (offsets) or as G slabs of `cap` rows of which counts[g] are in use
// (masked, what a low-latency dispatch delivers); rows outside a group are neither written nor
// used: every row has accumulators of its own.
//
// Epilogues: bf16, fp32, or SwiGLU with quantisation: a 256-wide tile holds 128 gate and 128 up
// columns, so it holds whole 128-blocks of h = silu(gate) * up, which leave as e4m3 with one
// fp32 scale per row and block (scale = max(amax, 1e-4) / 448), the operand of the next product.
//
// 12 warps: TMA producer, two MMA issuers (warp 1 owns the TMEM), a scale warp, 8 epilogue warps (two per TMEM lane quarter,
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
constexpr int kFirstEpi = 4;                     // warps 0 to 3: loads, MMAs, scales
constexpr int kBlkThreads = 32 * (kFirstEpi + kEpiWarps);
// Registers a thread: 128 sums and their operands need more than an even split of the file
// (168). The first warpgroup gives up what the two epilogue warpgroups take:
// 128 * 72 + 256 * 216 = 64512 = 384 * 168, what the block is launched with.
constexpr int kRegsMain = 72, kRegsEpi = 216;
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
// One lane of a converged warp, in the form from which the compiler knows that a single thread issues
// what follows (behind `lane == 0` it guards every tcgen05 and TMA instruction against a diverged warp).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
template <int BYTES>
__device__ __forceinline__ void cp_async(void* smem, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(smem)), "l"(src), "n"(BYTES) : "memory");
}
// Bounded wait (the clock and the abort flag are looked at once in 256 polls). Every hand-over between
// warps through an mbarrier takes about 130 cycles; with a suspend-time hint it took longer still.
__device__ __forceinline__ bool wait_blk(uint64_t* bar, uint32_t parity, const BlkArgs& a, volatile int* abort) {
  uint64_t t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((n & 255u) == 0u) {
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      if (*abort || now - t0 > a.timeout_ns) {
        atomicExch(a.error, 1u);
        *abort = 1;
        return false;
      }
    }
  }
}

struct Groups {
  int cnt[kMaxG];        // rows in use
  int pref[kMaxG + 1];   // m tiles of the groups before
};

// First row of a group (0 for slabs), clamped to the buffer.
__device__ __forceinline__ int64_t group_base(const BlkArgs& a, int g) {
  if (a.offsets == nullptr) return 0;
  const int64_t lo = a.offsets[g], top = a.rows;
  return lo < 0 ? 0 : (lo > top ? top : lo);
}

// Rows and m tiles of every group, from the device's offsets / counts, clamped to the buffer.
__device__ __forceinline__ void load_groups(Groups& s, const BlkArgs& a) {
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
    int64_t c = a.rows;
    if (a.offsets != nullptr) {
      const int64_t hi = a.offsets[g + 1], top = a.rows, b = group_base(a, g);
      const int64_t e = hi > top ? top : hi;
      c = e > b ? e - b : 0;
    }
    if (a.counts != nullptr) {
      const int64_t n = a.counts[g];
      c = n < 0 ? 0 : (n < c ? n : c);
    }
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
  __shared__ uint64_t full[kStages], empty[kStages], tfull[2], tempty[2], drain[2];
  __shared__ __align__(16) float s_sa[2][kBM][4], s_sb[2][2][4];   // scales as they come, four K blocks a unit
  __shared__ float s_scale[2][2][kBM];   // sa * sb of the block in a TMEM buffer: [buffer][128-column half][row]
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
      mbar_init(&tfull[b], 2);   // the MMAs' commit and the scale warp
      mbar_init(&tempty[b], kEpiWarps);
      mbar_init(&drain[b], 1);
    }
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
      uint32_t it = 0;
      BlkTile tl;
      for (int t = blockIdx.x; !s_abort && blk_tile(t, a, s_grp, tl); t += gridDim.x) {
        const int row = static_cast<int>(group_base(a, tl.g)) + tl.m0;
        const int slab = a.offsets != nullptr ? 0 : tl.g;
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % kStages;
          if (!wait_blk(&empty[s], ((it / kStages) & 1u) ^ 1u, a, &s_abort)) break;
          if (elect_one()) {
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
          __syncwarp();
        }
      }
      if (s_abort) {  // copies in flight land before the CTA's shared memory is given up
        for (uint32_t q = it > kStages ? it - kStages : 0; q < it; ++q)
          mbar_wait(&full[q % kStages], (q / kStages) & 1u, 1000000000ull);
      }
    } else if (warp <= 2) {
      // ------------------------------------------------------------------ MMA issuers
      // one warp for each TMEM buffer: the waits and the issue of a K block's MMAs take one warp
      // longer than the MMAs themselves
      const uint32_t b = warp - 1;
      constexpr uint32_t idesc = idesc_fp8(kBN, B_MN);
      uint32_t it = 0;
      BlkTile tl;
      for (int t = blockIdx.x; !s_abort && blk_tile(t, a, s_grp, tl); t += gridDim.x) {
        for (int kb = 0; kb < KB; ++kb, ++it) {
          if ((it & 1u) != b) continue;
          const int s = it % kStages;
          // the buffer comes last: from its release on every cycle delays the next block
          if (!wait_blk(&full[s], (it / kStages) & 1u, a, &s_abort)) break;
          const uint64_t ad = smem_desc_k128(sA + s * kABytes);
          const uint64_t bd = B_MN ? smem_desc_mn128(sB + s * kBBytes, 128 * kBK) : smem_desc_k128(sB + s * kBBytes);
          if (!wait_blk(&tempty[b], ((it >> 1) & 1u) ^ 1u, a, &s_abort)) break;
          tc_fence_after();
          if (elect_one()) {
            // next 32 channels: 32 bytes along a K-major swizzle row, or 32 rows of 128 bytes
            constexpr uint64_t bstep = B_MN ? (32 * 128) >> 4 : 2;
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k)
              tc_mma_fp8(tmem_base + b * kBN, ad + 2 * k, bd + bstep * k, idesc, k > 0 ? 1u : 0u);
            tc_commit(&tfull[b]);
            tc_commit(&empty[s]);
          }
          __syncwarp();
        }
      }
      if (elect_one()) tc_commit(&drain[b]);  // every MMA issued is done before TMEM is released
      __syncwarp();
      mbar_wait(&drain[b], 0, a.timeout_ns);
    } else {
      // ------------------------------------------------------------------ scales (warp 3)
      // The scales of four K blocks (of the tile's 128 rows and two column blocks) are copied
      // asynchronously, a unit ahead of their use and across tiles, 16 bytes a row where the rows
      // of sa allow it; their products go to the epilogue with the block's TMEM buffer.
      const int NB = (a.N + 127) / 128;
      const bool wide = ((reinterpret_cast<uintptr_t>(a.sa) | (a.sa_row * 4) | (a.sa_group * 4)) & 15) == 0;
      int t = blockIdx.x, k0 = 0;      // the unit to be copied next
      BlkTile tl;
      bool left = blk_tile(t, a, s_grp, tl);
      auto copy_unit = [&](int s) {
        if (left) {
          const int cnt = s_grp.cnt[tl.g];
          const float* sa = a.sa + tl.g * a.sa_group + group_base(a, tl.g) * a.sa_row;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* src = sa + min(tl.m0 + 32 * i + lane, cnt - 1) * a.sa_row + k0;
            float* dst = s_sa[s][32 * i + lane];
            if (wide && k0 + 4 <= KB) {
              cp_async<16>(dst, src);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (k0 + j < KB) cp_async<4>(dst + j, src + j);
            }
          }
          // lane h * 4 + j < 8 copies block j of column block h
          const float* sb = a.sb + tl.g * a.sb_group + min(tl.n0 / 128 + (lane >> 2 & 1), NB - 1) * a.sb_n;
          if (lane < 8 && k0 + (lane & 3) < KB)
            cp_async<4>(&s_sb[s][lane >> 2][lane & 3], sb + (k0 + (lane & 3)) * a.sb_k);
          k0 += 4;
          if (k0 >= KB) {
            k0 = 0;
            t += gridDim.x;
            left = blk_tile(t, a, s_grp, tl);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      copy_unit(0);
      copy_unit(1);
      uint32_t it = 0, u = 0;
      bool ok = true;
      BlkTile at;
      for (int tt = blockIdx.x; ok && !s_abort && blk_tile(tt, a, s_grp, at); tt += gridDim.x) {
        for (int kb = 0; kb < KB && ok; ++kb, ++it) {
          const int s = u & 1, j = kb & 3, b = it & 1;
          if (j == 0) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
          }
          float f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = s_sa[s][32 * i + lane][j];
          const float b0 = s_sb[s][0][j], b1 = s_sb[s][1][j];
          ok = wait_blk(&tempty[b], ((it >> 1) & 1u) ^ 1u, a, &s_abort);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s_scale[b][0][32 * i + lane] = f[i] * b0;
            s_scale[b][1][32 * i + lane] = f[i] * b1;
          }
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(&tfull[b]);
          if (j == 3 || kb + 1 == KB) {
            copy_unit(s);
            ++u;
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
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
    const uint32_t tq = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    uint32_t it = 0;
    int parity = 0;
    BlkTile tl;
    for (int t = blockIdx.x; !s_abort && blk_tile(t, a, s_grp, tl); t += gridDim.x, parity ^= 1) {
      const int cnt = s_grp.cnt[tl.g];
      const int row = tl.m0 + q * 32 + lane;           // within the group
      const int64_t base = group_base(a, tl.g);
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // A block's four 32-column chunks go through two register buffers, two loads in flight; the
      // TMEM buffer is handed back once the last is in, with half of the sums still to be added, and
      // the next block's first loads leave before the last chunk is added.
      uint32_t r[2][32];
      bool ok;
      auto add = [&](int c, float f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[c * 32 + i] = fmaf(__uint_as_float(r[c & 1][i]), f, acc[c * 32 + i]);
      };
      float f0 = 0.f, f1 = 0.f;
      auto begin_block = [&]() {   // block `it`: its first chunk and its scales
        ok = wait_blk(&tfull[it & 1], (it >> 1) & 1u, a, &s_abort);
        tc_fence_after();
        if (ok) tmem_ld32_async(tq + (it & 1) * kBN + col_of(0), r[0]);
        f0 = s_scale[it & 1][EPI == kOutSwiGLU ? 0 : half][q * 32 + lane];
        f1 = EPI == kOutSwiGLU ? s_scale[it & 1][1][q * 32 + lane] : f0;
      };
      begin_block();
#pragma unroll 1
      for (int kb = 0; kb < KB && ok; ++kb) {
        const uint32_t taddr = tq + (it & 1) * kBN;
        tmem_ld32_async(taddr + col_of(1), r[1]);
        tmem_wait_ld64(r[0], r[1]);
        add(0, f0);
        tmem_ld32_async(taddr + col_of(2), r[0]);
        add(1, f0);
        tmem_ld32_async(taddr + col_of(3), r[1]);
        tmem_wait_ld64(r[0], r[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[it & 1]);
        ++it;
        const float f = f1;
        add(2, f);
        if (kb + 1 < KB) begin_block();
        add(3, f);
      }
      if (!ok) break;
      // ---- output: 64 bytes of each of the warp's 32 rows at a time, through shared memory (the
      // 16-byte pieces of a row are swapped by row pair, so that 8 lanes hit distinct banks)
      const int first = tl.m0 + q * 32;
      const int64_t grow = base + first;
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
          for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(acc[c * 16 + i]);
          store64(crow + 4 * static_cast<int64_t>(col), a.c_row, (a.N - col) / 4, v);
        }
      } else if (EPI == kOutBF16 || a.C != nullptr) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = tl.n0 + col_of(c);
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = pack_bf16(acc[c * 32 + 2 * i], acc[c * 32 + 2 * i + 1]);
          store64(crow + 2 * static_cast<int64_t>(col), a.c_row, (a.N - col) / 8, v);
        }
      }
      if (EPI == kOutSwiGLU) {
        // h = silu(gate) * up of 64 of the block's 128 columns; the other half's warp has the rest
        float h[64];
        uint32_t top = 0;   // as bits, so that a NaN stays the largest
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          h[i] = __fdividef(acc[i], 1.f + __expf(-acc[i])) * acc[64 + i];
          top = max(top, __float_as_uint(fabsf(h[i])));
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
