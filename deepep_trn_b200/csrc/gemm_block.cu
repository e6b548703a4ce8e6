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
// Two kernels, for groups with many and with few rows:
//  * many: 128 rows x 256 columns, rows of A on the TMEM lanes; a CTA takes whole tiles. 32 groups of
//    1024 rows, N 4096, K 7168, SwiGLU and pre-activation: 1205 us over a timed second, 1600 TFLOP/s, at
//    1297 MHz, to which the 1000 W cap brings the clock: 28 rounds of 56 blocks, 1000 cycles a block. (1028 us
//    in its first moments; 1473 us at about 1565 MHz and 1470 cycles with MMAs behind `lane == 0` and scales
//    loaded by the threads that use them: a third of the cycles was a fifth of the time.) So energy a
//    block bounds it as much as cycles a block, of which the operands' way into shared memory takes 768
//    (48 KB at 64 bytes a cycle).
//  * few (at most kFewTile rows): 256 columns x up to 48 rows, columns of C on the lanes, so that
//    nothing is spent on rows that are not there. Bound by reading B: 32 slabs of 32 rows, the same N
//    and K: 152 us by itself, 6.2 TB/s (prefetching B into L2 ahead of the copies: 232 us). Tiles that do not
//    fill a round of the SMs are taken by clusters that divide K and add their parts through distributed
//    shared memory in a fixed order (4 rows, N 4096, K 4096: 11.5 us, 19.6 in the other form).
// Segments take one of the two, by the rows that there are. For slabs, whose counts only the device
// knows, both are launched where the second is worth it, and each takes its groups.
//
// 12 warps: TMA producer, MMA issuer (one for each TMEM buffer in the kernel for many rows; warp 1 owns
// the TMEM), a scale warp, 8 epilogue warps. Every wait is bounded; a wait that runs out sets *error,
// lets the copies in flight land, frees the TMEM and returns.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <climits>

#include "device_table.h"
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

constexpr int kFewTile = 48;                     // rows of a tile with few rows, and of a group that counts as one
constexpr int kFewStages = 4, kFewBufs = 4;
constexpr int kFewCols = 64;                     // TMEM columns of a buffer's half
constexpr int kFewStageBytes = kBBytes + kFewTile * kBK;
constexpr int kMaxSplit = 8;                     // CTAs of a cluster that divide K
static_assert(kStages % 2 == 0, "two MMA warps take turns: each must see every phase of its stages' barriers");
static_assert(kFewTile <= kFewCols && kFewBufs * 2 * kFewCols <= 2 * kBN, "TMEM columns");

enum Form : int { kBothForms = 0, kAllMany = 1, kAllFew = 2 };
enum BlkEpilogue : int { kOutBF16 = 0, kOutF32 = 1, kOutSwiGLU = 2 };

// Estimated cycles, from measurements. A K block of a tile takes 900, or 1540 where all SMs read a part of
// B of their own from memory. A tile with few rows costs 2300 more, and 6000 where a cluster divides K.
// How well they choose was measured with the form forced, for 1 to 64 groups of 4 to 200 rows, N 1408 to 7168,
// K 512 to 7168:
//  * 72 calls with segments: the form that is chosen takes at most 1.05 of the faster one's time in 66, and
//    1.10 to 1.31 in 6, small calls with few groups (4 rows a group, N 2048, K 4096, 8 groups: 20.0 us as many
//    rows, 16.1 as few);
//  * 114 calls with slabs: at most 1.05 in 92. The second launch takes 5 to 8 us that are not in the estimates,
//    wherever both are launched: 32 slabs of 32 rows, N 4096, K 7168: 162 us as many rows, 152 as few, 168
//    with both; the worst is one slab of 4 rows, N 4096, K 4096: 20.1, 11.7 and 19.4. The groups divided
//    between the two were not the faster way in any call (13 slabs of 2 to 126 rows, N 3584, K 6656: 71 us as
//    many rows, 78 as few, 82 divided).
__host__ __device__ inline int64_t block_cycles(int64_t ctas, int64_t sms, bool own) { return own && ctas * 2 > sms ? 1540 : 900; }
__host__ __device__ inline int64_t many_cycles(int64_t tiles, int64_t KB, int64_t sms, bool own) {
  return (tiles + sms - 1) / sms * KB * block_cycles(tiles, sms, own) + 4000;
}
__host__ __device__ inline int64_t few_cycles(int64_t tiles, int64_t KB, int64_t grid, int64_t split) {
  if (split == 1) return (tiles + grid - 1) / grid * (KB * block_cycles(tiles, grid, true) + 2300) + 4000;
  const int64_t left = tiles % grid, rounds = (left * split + grid - 1) / grid;
  return tiles / grid * (KB * 1540 + 2300) +
         rounds * ((KB + split - 1) / split * block_cycles(left * split, grid, true) + 6000) + 4000;
}

// The groups of a call with slabs: tiles as many rows, as few, and with each group in the form that its rows
// suggest; groups with rows.
struct Tally {
  int many, few, many_part, few_part, busy;
  __host__ __device__ void add(int n) {
    const int m = (n + kBM - 1) / kBM, f = (n + kFewTile - 1) / kFewTile;
    many += m;
    few += f;
    (f > 1 ? many_part : few_part) += f > 1 ? m : f;
    busy += n > 0;
  }
};
// The launches of a call. Both kernels are given the same, and conclude the same from it.
struct Plan {
  int form;                 // Form
  int sms;                  // SMs that the call may use
  int split, few_grid;      // kernel for few rows: CTAs of a cluster that divide K, CTAs
  int many_grid;            // kernel for many rows: CTAs
  bool overlap;             // the second kernel starts while the first still runs
};
// The most rows of a group that counts as one with few, where both kernels are launched: all groups as many,
// all as few, or each by its rows, whichever has the least estimate.
__host__ __device__ inline int few_rows_of(const Tally& t, int64_t N, int64_t K, const Plan& p) {
  const int64_t ntn = (N + kBN - 1) / kBN, KB = (K + kBK - 1) / kBK;
  const int64_t as_many = many_cycles(t.many * ntn, KB, p.sms, t.many == t.busy);
  const int64_t as_few = few_cycles(t.few * ntn, KB, p.few_grid, p.split);
  const int64_t mixed = few_cycles(t.few_part * ntn, KB, p.few_grid, p.split) +
                        many_cycles(t.many_part * ntn, KB, p.sms, t.many_part == t.busy - t.few_part);
  return as_few <= (as_many < mixed ? as_many : mixed) ? INT_MAX : mixed < as_many ? kFewTile : 0;
}

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
  Plan plan;
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
// D fp32, A and B e4m3, M = 128; bits 15 and 16 select an MN-major A and B
__host__ __device__ constexpr uint32_t idesc_fp8(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(kBM >> 4) << 24);
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
__device__ __forceinline__ void give_up(const BlkArgs& a, volatile int* abort) {
  atomicExch(a.error, 1u);
  *abort = 1;
}
// Bounded wait of a whole warp, whose lanes leave it together with one answer: what follows (elect.sync, TMEM
// loads, barriers) needs all of them. The clock and the abort flag are looked at once in 256 polls, of which
// each is suspended for up to 4 us. Every hand-over between warps through an mbarrier takes about 130 cycles;
// with a suspend-time hint it took longer still.
__device__ __forceinline__ bool wait_blk(uint64_t* bar, uint32_t parity, const BlkArgs& a, volatile int* abort) {
  uint64_t t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((n & 255u) == 0u) {
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      if (__any_sync(0xffffffffu, *abort || now - t0 > a.timeout_ns)) {
        give_up(a, abort);
        return false;
      }
    }
  }
}

struct Groups {
  int pref[kMaxG + 1];   // tiles (of rows) of the groups before; none for a group of the other form
};
struct Span {
  int64_t base;          // first row (0 for slabs)
  int cnt;               // rows in use
};

// A group's rows, from the device's offsets / counts, clamped to the buffer.
__device__ __forceinline__ Span group_span(const BlkArgs& a, int g) {
  int64_t b = 0, c = a.rows;
  if (a.offsets != nullptr) {
    const int64_t lo = a.offsets[g], hi = a.offsets[g + 1], top = a.rows;
    b = lo < 0 ? 0 : (lo > top ? top : lo);
    c = (hi > top ? top : hi) - b;
    c = c < 0 ? 0 : c;
  }
  if (a.counts != nullptr) {
    const int64_t n = a.counts[g];
    c = n < 0 ? 0 : (n < c ? n : c);
  }
  return {b, static_cast<int>(c)};
}

// The tiles of the groups that this form takes. All CTAs of both kernels come to the same answer.
template <bool FEW>
__device__ __forceinline__ void load_groups(Groups& s, const BlkArgs& a) {
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) s.pref[g + 1] = group_span(a, g).cnt;
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int few_rows = a.plan.form == kAllFew ? INT_MAX : 0;   // most rows of a group that counts as one with few
    if (a.plan.form == kBothForms) {
      Tally t{};
      for (int g = lane; g < a.G; g += 32) t.add(s.pref[g + 1]);
      t.many = __reduce_add_sync(0xffffffffu, t.many);
      t.few = __reduce_add_sync(0xffffffffu, t.few);
      t.many_part = __reduce_add_sync(0xffffffffu, t.many_part);
      t.few_part = __reduce_add_sync(0xffffffffu, t.few_part);
      t.busy = __reduce_add_sync(0xffffffffu, t.busy);
      few_rows = few_rows_of(t, a.N, a.K, a.plan);
    }
    int total = 0;
    for (int g0 = 0; g0 < a.G; g0 += 32) {
      const int g = g0 + lane, n = g < a.G ? s.pref[g + 1] : 0;
      const bool is_few = n <= few_rows;
      int v = is_few != FEW ? 0 : FEW ? (n + kFewTile - 1) / kFewTile : (n + kBM - 1) / kBM;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, m);
        if (lane >= m) v += o;
      }
      if (g < a.G) s.pref[g + 1] = total + v;
      total += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) s.pref[0] = 0;
  }
}

struct BlkTile {
  int g, m0, n0;
};
// The last group whose share begins at or before t, where a tile of rows counts `per` times.
__device__ __forceinline__ int group_of(int t, int per, const BlkArgs& a, const Groups& s) {
  int lo = 0, hi = a.G - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.pref[mid] * per <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ bool blk_tile(int t, const BlkArgs& a, const Groups& s, BlkTile& tl) {
  const int ntn = (a.N + kBN - 1) / kBN;
  const int mt = t / ntn;
  if (mt >= s.pref[a.G]) return false;
  tl.g = group_of(mt, 1, a, s);
  tl.m0 = (mt - s.pref[tl.g]) * kBM;
  tl.n0 = (t - mt * ntn) * kBN;
  return true;
}
// The work of one CTA on groups with few rows: whole tiles for as many rounds as all CTAs have one,
// then its share of the K blocks of the tiles left over, a cluster to a tile. The row tiles of one
// column tile follow one another, so that B is read once from memory. The next tile is looked up
// while the current one is worked on.
struct FewTiles {
  const BlkArgs& a;
  const Groups& s;
  int whole, tiles;      // tiles [0, whole) go to single CTAs, [whole, tiles) to clusters
  int crank, csize, KB;
  int t;                 // the next tile's number
  BlkTile tl, next;
  Span sp, next_sp;
  int k0, k1, next_k0, next_k1;   // its K blocks
  bool split, next_split, more;
  __device__ __forceinline__ FewTiles(const BlkArgs& a, const Groups& s, int crank, int csize)
      : a(a), s(s), crank(crank), csize(csize), KB((a.K + kBK - 1) / kBK) {
    tiles = s.pref[a.G] * ((a.N + kBN - 1) / kBN);
    whole = csize > 1 ? tiles / static_cast<int>(gridDim.x) * static_cast<int>(gridDim.x) : tiles;
    t = blockIdx.x;
    if (t >= whole) t = whole + blockIdx.x / csize;
    find();
  }
  __device__ __forceinline__ void find() {
    more = t < tiles;
    if (!more) return;
    const int ntn = (a.N + kBN - 1) / kBN;
    const int g = group_of(t, ntn, a, s);
    next_sp = group_span(a, g);
    const int rows = s.pref[g + 1] - s.pref[g], r = t - s.pref[g] * ntn;
    const int col = rows == 1 ? r : r / rows;
    next.g = g;
    next.n0 = col * kBN;
    next.m0 = (r - col * rows) * kFewTile;
    next_split = t >= whole && csize > 1;
    next_k0 = next_split ? static_cast<int>(static_cast<int64_t>(KB) * crank / csize) : 0;
    next_k1 = next_split ? static_cast<int>(static_cast<int64_t>(KB) * (crank + 1) / csize) : KB;
    if (next_split) {
      t += gridDim.x / csize;
    } else {
      t += gridDim.x;
      if (t >= whole && csize > 1) t = whole + blockIdx.x / csize;
    }
  }
  __device__ __forceinline__ bool advance() {
    if (!more) return false;
    tl = next;
    sp = next_sp;
    k0 = next_k0;
    k1 = next_k1;
    split = next_split;
    find();
    return true;
  }
};
// Address of this CTA's shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_peer(const void* bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_addr(bar, rank)) : "memory");
}
__device__ __forceinline__ float4 load_peer(const float* p, uint32_t rank) {
  float4 v;
  // volatile: kept behind the wait and the fence before it
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(peer_addr(p, rank)));
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Barrier of `n` threads that tells each whether all of them are well: warps that share a barrier leave
// together or not at all, so that none is left waiting after a timeout.
__device__ __forceinline__ bool bar_all(int id, int n, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(ok)), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }
// The scales of four K blocks (k0 .. k0 + 3 < k1) of one row of sa.
__device__ __forceinline__ void copy_scales(float* dst, const float* src, int k0, int k1, bool wide) {
  if (wide && k0 + 4 <= k1 && (k0 & 3) == 0) {
    cp_async<16>(dst, src);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k0 + j < k1) cp_async<4>(dst + j, src + j);
  }
}

// ------------------------------------------------------------------------------ groups with many rows
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
  load_groups<false>(s_grp, a);
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
      bool ok = true;
      BlkTile tl;
      for (int t = blockIdx.x; ok && blk_tile(t, a, s_grp, tl); t += gridDim.x) {
        const int row = static_cast<int>(group_span(a, tl.g).base) + tl.m0;
        const int slab = a.offsets != nullptr ? 0 : tl.g;
        for (int kb = 0; kb < KB; ++kb, ++it) {
          const int s = it % kStages;
          ok = wait_blk(&empty[s], ((it / kStages) & 1u) ^ 1u, a, &s_abort);
          if (!ok) break;
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
      land_copies<kStages>(full, it);
    } else if (warp <= 2) {
      // ------------------------------------------------------------------ MMA issuers
      // one warp for each TMEM buffer: the waits and the issue of a K block's MMAs take one warp
      // longer than the MMAs themselves
      const uint32_t b = warp - 1;
      constexpr uint32_t idesc = idesc_fp8(kBN, false, B_MN);
      uint32_t it = 0;
      bool ok = a.timeout_ns != 0;   // without a budget nothing is multiplied, and all that wait for it run out
      if (!ok) give_up(a, &s_abort);
      BlkTile tl;
      for (int t = blockIdx.x; ok && blk_tile(t, a, s_grp, tl); t += gridDim.x) {
        for (int kb = 0; kb < KB; ++kb, ++it) {
          if ((it & 1u) != b) continue;
          const int s = it % kStages;
          // the buffer comes last: from its release on every cycle delays the next block
          ok = wait_blk(&full[s], (it / kStages) & 1u, a, &s_abort);
          if (!ok) break;
          const uint64_t ad = smem_desc_k128(sA + s * kABytes);
          const uint64_t bd = B_MN ? smem_desc_mn128(sB + s * kBBytes, 128 * kBK) : smem_desc_k128(sB + s * kBBytes);
          ok = wait_blk(&tempty[b], ((it >> 1) & 1u) ^ 1u, a, &s_abort);
          if (!ok) break;
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
      Span sp = left ? group_span(a, tl.g) : Span{0, 0};
      auto copy_unit = [&](int s) {
        if (left) {
          const float* sa = a.sa + tl.g * a.sa_group + sp.base * a.sa_row + k0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            copy_scales(s_sa[s][32 * i + lane], sa + min(tl.m0 + 32 * i + lane, sp.cnt - 1) * a.sa_row, k0, KB, wide);
          // lane h * 4 + j < 8 copies block j of column block h
          const float* sb = a.sb + tl.g * a.sb_group + min(tl.n0 / 128 + (lane >> 2 & 1), NB - 1) * a.sb_n;
          if (lane < 8 && k0 + (lane & 3) < KB)
            cp_async<4>(&s_sb[s][lane >> 2][lane & 3], sb + (k0 + (lane & 3)) * a.sb_k);
          k0 += 4;
          if (k0 >= KB) {
            k0 = 0;
            t += gridDim.x;
            left = blk_tile(t, a, s_grp, tl);
            if (left) sp = group_span(a, tl.g);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      copy_unit(0);
      copy_unit(1);
      uint32_t it = 0, u = 0;
      bool ok = true;
      BlkTile at;
      for (int tt = blockIdx.x; ok && blk_tile(tt, a, s_grp, at); tt += gridDim.x) {
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
    bool ok = true;
    BlkTile tl;
    for (int t = blockIdx.x; blk_tile(t, a, s_grp, tl); t += gridDim.x, parity ^= 1) {
      const Span sp = group_span(a, tl.g);
      const int64_t base = sp.base;
      const int cnt = sp.cnt;
      const int row = tl.m0 + q * 32 + lane;           // within the group
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // A block's four 32-column chunks go through two register buffers, two loads in flight; the
      // TMEM buffer is handed back once the last is in, with half of the sums still to be added, and
      // the next block's first loads leave before the last chunk is added.
      uint32_t r[2][32];
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
      if (ok) begin_block();
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
      if (!ok) {
        // the other half's warp of these rows may have got through: meet it at its barrier
        if (EPI == kOutSwiGLU) asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
        continue;
      }
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
          h[i] = silu_mul(acc[i], acc[64 + i]);
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
  // Launched while the kernel for groups with few rows still runs: whoever waits for this one waits for both.
  if (threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * kBN);
  }
}

// ------------------------------------------------------------------------------- groups with few rows
template <int EPI, bool B_MN>
__global__ void __launch_bounds__(kBlkThreads, 1)
    gemm_few_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, BlkArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_part = reinterpret_cast<float*>(smem + kFewStages * kFewStageBytes);   // [kFewTile][kBN] of a finished tile
  __shared__ Groups s_grp;
  __shared__ uint64_t ffull[kFewStages], fempty[kFewStages], ftfull[kFewBufs], ftempty[kFewBufs], pready, pfree, drain;
  __shared__ __align__(16) float s_sa[2][64][4], s_sb[2][2][4];      // scales as they come, four K blocks a unit
  __shared__ __align__(16) float s_scale[kFewBufs * 2 * kFewTile];   // sa * sb: [buffer][column half][row]
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int s_abort;

  // The kernel for the other groups, where there is one, may take the SMs as they fall free.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = warp_id(), lane = lane_id();
  uint32_t crank, csize;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&ffull[s], 1);
      mbar_init(&fempty[s], 1);
    }
    for (int b = 0; b < kFewBufs; ++b) {
      mbar_init(&ftfull[b], 2);   // the MMAs' commit and the scale warp
      mbar_init(&ftempty[b], kEpiWarps);
    }
    mbar_init(&pready, csize);   // every CTA of the cluster has its part in shared memory
    mbar_init(&pfree, csize);    // ... and has read this CTA's
    mbar_init(&drain, 1);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 2 * kBN);
  load_groups<true>(s_grp, a);
  tc_fence_before();
  __syncthreads();
  // The peers' barriers exist once this cluster barrier completes; only the first message to a peer
  // waits for it.
  if (csize > 1) cluster_arrive();
  bool joined = csize == 1;
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  const int NB = (a.N + 127) / 128;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.sa) | (a.sa_row * 4) | (a.sa_group * 4)) & 15) == 0;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    uint32_t it = 0;
    bool ok = true;
    FewTiles f(a, s_grp, crank, csize);
    while (ok && f.advance()) {
      const BlkTile tl = f.tl;
      const int row = static_cast<int>(f.sp.base) + tl.m0;
      const int slab = a.offsets != nullptr ? 0 : tl.g;
      for (int kb = f.k0; kb < f.k1; ++kb, ++it) {
        const int s = it % kFewStages;
        ok = wait_blk(&fempty[s], ((it / kFewStages) & 1u) ^ 1u, a, &s_abort);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&ffull[s], kFewStageBytes);
          uint8_t* db = smem + s * kFewStageBytes;
          if (B_MN) {
#pragma unroll
            for (int j = 0; j < kBN / 128; ++j)
              tma_load_3d(db + j * (128 * kBK), &tmB, &ffull[s], tl.n0 + 128 * j, kb * kBK, tl.g);
          } else {
            tma_load_3d(db, &tmB, &ffull[s], kb * kBK, tl.n0, tl.g);
          }
          tma_load_3d(db + kBBytes, &tmA, &ffull[s], kb * kBK, row, slab);
        }
        __syncwarp();
      }
    }
    land_copies<kFewStages>(ffull, it);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    uint32_t it = 0;
    bool ok = a.timeout_ns != 0;   // as in the other kernel
    if (!ok) give_up(a, &s_abort);
    FewTiles f(a, s_grp, crank, csize);
    while (ok && f.advance()) {
      const int n = (min(f.sp.cnt - f.tl.m0, kFewTile) + 15) / 16 * 16;
      const uint32_t idesc = idesc_fp8(n, B_MN, false);
      for (int kb = f.k0; kb < f.k1; ++kb, ++it) {
        const int s = it % kFewStages, b = it % kFewBufs;
        ok = wait_blk(&ffull[s], (it / kFewStages) & 1u, a, &s_abort);
        if (!ok) break;
        const uint8_t* db = smem + s * kFewStageBytes;
        const uint64_t xd = smem_desc_k128(db + kBBytes);
        ok = wait_blk(&ftempty[b], ((it / kFewBufs) & 1u) ^ 1u, a, &s_abort);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          constexpr uint64_t wstep = B_MN ? (32 * 128) >> 4 : 2;
          // the halves in turn: products into one accumulator wait for one another
          const uint64_t w0 = B_MN ? smem_desc_mn128(db, 128 * kBK) : smem_desc_k128(db);
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              tc_mma_fp8(tmem_base + (b * 2 + h) * kFewCols, w0 + h * ((128 * kBK) >> 4) + wstep * k, xd + 2 * k, idesc,
                         k > 0 ? 1u : 0u);
          }
          tc_commit(&ftfull[b]);
          tc_commit(&fempty[s]);
        }
        __syncwarp();
      }
    }
    if (elect_one()) tc_commit(&drain);  // every MMA issued is done before TMEM is released
    __syncwarp();
    mbar_wait(&drain, 0, a.timeout_ns);
  } else if (warp == 3) {
    // ---------------------------------------------------------------- scales, as in the other kernel
    FewTiles c(a, s_grp, crank, csize);   // the unit to be copied next
    bool left = c.advance();
    int k0 = left ? c.k0 : 0;
    auto copy_unit = [&](int s) {
      if (left) {
        const float* sa = a.sa + c.tl.g * a.sa_group + c.sp.base * a.sa_row + k0;
#pragma unroll
        for (int r0 = 0; r0 < kFewTile; r0 += 32)
          if (r0 + lane < kFewTile)
            copy_scales(s_sa[s][r0 + lane], sa + min(c.tl.m0 + r0 + lane, c.sp.cnt - 1) * a.sa_row, k0, c.k1, wide);
        const float* sb = a.sb + c.tl.g * a.sb_group + min(c.tl.n0 / 128 + (lane >> 2 & 1), NB - 1) * a.sb_n;
        if (lane < 8 && k0 + (lane & 3) < c.k1)
          cp_async<4>(&s_sb[s][lane >> 2][lane & 3], sb + (k0 + (lane & 3)) * a.sb_k);
        k0 += 4;
        if (k0 >= c.k1) {
          left = c.advance();
          k0 = c.k0;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    copy_unit(0);
    copy_unit(1);
    uint32_t it = 0, u = 0;
    bool ok = true;
    FewTiles f(a, s_grp, crank, csize);
    while (ok && f.advance()) {
      for (int kb = f.k0; kb < f.k1 && ok; ++kb, ++it) {
        const int s = u & 1, j = (kb - f.k0) & 3, b = it % kFewBufs;
        if (j == 0) {
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          __syncwarp();
        }
        const float b0 = s_sb[s][0][j], b1 = s_sb[s][1][j];
        const float f0 = s_sa[s][lane][j], f1 = s_sa[s][32 + lane][j];   // (rows past kFewTile: not stored)
        ok = wait_blk(&ftempty[b], ((it / kFewBufs) & 1u) ^ 1u, a, &s_abort);
        float* o = s_scale + b * 2 * kFewTile + lane;
        o[0] = f0 * b0;
        o[kFewTile] = f0 * b1;
        if (lane < kFewTile - 32) {
          o[32] = f1 * b0;
          o[kFewTile + 32] = f1 * b1;
        }
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&ftfull[b]);
        if (j == 3 || kb + 1 == f.k1) {
          copy_unit(s);
          ++u;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= kFirstEpi) {
    // ---------------------------------------------------------------- epilogue
    const int q = warp & 3, half = (warp - kFirstEpi) >> 2, ew = warp - kFirstEpi;
    const uint32_t tq = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + half * kFewCols;
    uint32_t it = 0, round = 0;   // round: tiles shared with the cluster so far
    bool ok = true;
    // (left only where bar_all says so: all eight warps, or none; whole tiles have no barrier, and pass
    // without work once `ok` is false)
    FewTiles ft(a, s_grp, crank, csize);
    while (ft.advance()) {
      const BlkTile tl = ft.tl;
      const Span sp = ft.sp;
      const bool split = ft.split;
      const int n = min(sp.cnt - tl.m0, kFewTile);
      float acc[kFewTile];
#pragma unroll
      for (int i = 0; i < kFewTile; ++i) acc[i] = 0.f;
      for (int kb = ft.k0; kb < ft.k1 && ok; ++kb, ++it) {
        const int b = it % kFewBufs;
        ok = wait_blk(&ftfull[b], (it / kFewBufs) & 1u, a, &s_abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr = tq + b * 2 * kFewCols;
        const float4* f = reinterpret_cast<const float4*>(s_scale + (b * 2 + half) * kFewTile);
        uint32_t r[32];
#pragma unroll
        for (int c = 0; c < (kFewTile + 31) / 32; ++c) {
          if (32 * c < n) {
            tmem_ld32(taddr + 32 * c, r);   // (columns past the rows are read and dropped)
#pragma unroll
            for (int i = 0; i < 8 && 32 * c + 4 * i < kFewTile; ++i) {
              const float4 f4 = f[8 * c + i];
              float* o = acc + 32 * c + 4 * i;
              o[0] = fmaf(__uint_as_float(r[4 * i]), f4.x, o[0]);
              o[1] = fmaf(__uint_as_float(r[4 * i + 1]), f4.y, o[1]);
              o[2] = fmaf(__uint_as_float(r[4 * i + 2]), f4.z, o[2]);
              o[3] = fmaf(__uint_as_float(r[4 * i + 3]), f4.w, o[3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ftempty[b]);
      }
      // this CTA's part, [row][256 columns], once every peer has read the one before
      if (ok && split && round > 0) ok = wait_blk(&pfree, (round - 1) & 1u, a, &s_abort);
      if (ok) {
#pragma unroll
        for (int i = 0; i < kFewTile; ++i)
          if (i < n) s_part[i * kBN + half * 128 + q * 32 + lane] = acc[i];
      }
      __syncwarp();
      if (split && !joined) {
        cluster_wait();
        joined = true;
      }
      ok = bar_all(1, 32 * kEpiWarps, ok);
      if (!ok) break;
      const int parts = split ? csize : 1;
      if (split) {
        if (ew == 0 && lane < static_cast<int>(csize)) arrive_peer(&pready, lane);
        ok = wait_blk(&pready, round & 1u, a, &s_abort);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
      }
      // a warp a row, the rows divided among the CTAs with parts
      for (int i = (split ? crank : 0) + parts * ew; ok && i < n; i += parts * kEpiWarps) {
        const float* p = s_part + i * kBN + 4 * lane;
        float4 x, y;
        if (!split) {
          x = *reinterpret_cast<const float4*>(p);
          y = *reinterpret_cast<const float4*>(p + 128);
        } else {
            x = y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c0 = 0; c0 < kMaxSplit; c0 += 4) {   // in the order of the ranks, four on their way at a time
              if (c0 < static_cast<int>(csize)) {
                float4 v[4], w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const int from = min(c0 + c, static_cast<int>(csize) - 1);
                  v[c] = load_peer(p, from);
                  w[c] = load_peer(p + 128, from);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  if (c0 + c < static_cast<int>(csize)) {
                    x.x += v[c].x, x.y += v[c].y, x.z += v[c].z, x.w += v[c].w;
                    y.x += w[c].x, y.y += w[c].y, y.z += w[c].z, y.w += w[c].w;
                  }
                }
              }
            }
          }
        const int64_t grow = sp.base + tl.m0 + i;
        const int c0 = tl.n0 + 4 * lane, c1 = c0 + 128;
        uint8_t* crow = a.C + tl.g * a.c_group + grow * a.c_row;
        if (EPI == kOutF32) {
          if (c0 < a.N) *reinterpret_cast<float4*>(crow + 4ll * c0) = x;
          if (c1 < a.N) *reinterpret_cast<float4*>(crow + 4ll * c1) = y;
        } else if (EPI == kOutBF16 || a.C != nullptr) {
          if (c0 < a.N) *reinterpret_cast<uint2*>(crow + 2ll * c0) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
          if (c1 < a.N) *reinterpret_cast<uint2*>(crow + 2ll * c1) = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
        }
        if (EPI == kOutSwiGLU) {
          const float h0 = silu_mul(x.x, y.x), h1 = silu_mul(x.y, y.y), h2 = silu_mul(x.z, y.z), h3 = silu_mul(x.w, y.w);
          uint32_t top = max(max(__float_as_uint(fabsf(h0)), __float_as_uint(fabsf(h1))),
                             max(__float_as_uint(fabsf(h2)), __float_as_uint(fabsf(h3))));
          top = max(__reduce_max_sync(0xffffffffu, top), __float_as_uint(1e-4f));
          const float amax = __uint_as_float(top), inv = __fdiv_rn(448.f, amax);
          uint8_t* hrow = a.H + tl.g * a.h_group + grow * a.h_row + tl.n0 / 2;
          reinterpret_cast<uint32_t*>(hrow)[lane] = uint32_t(f32x2_to_e4m3x2(h0 * inv, h1 * inv)) |
                                                    (uint32_t(f32x2_to_e4m3x2(h2 * inv, h3 * inv)) << 16);
          if (lane == 0) a.Hs[tl.g * a.hs_group + grow * a.hs_row + tl.n0 / 256] = __fdiv_rn(amax, 448.f);
        }
      }
      ok = bar_all(1, 32 * kEpiWarps, ok);
      if (!ok) break;
      if (split) {
        if (ew == 0 && lane < static_cast<int>(csize)) arrive_peer(&pfree, lane);
        ++round;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (csize > 1) {   // no CTA leaves while a peer may still read its part
    if (!joined) cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
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

// The kernel for groups with few rows in clusters of `split`.
template <int EPI, bool B_MN>
struct FewLaunch {
  static constexpr int kSmem = 1024 + kFewStages * kFewStageBytes + kFewTile * kBN * 4;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  FewLaunch(int grid, int split, cudaStream_t stream) {
    static std::atomic<uint64_t> seen{0};
    AT_CUDA_CHECK(set_smem_limit_once(seen, gemm_few_kernel<EPI, B_MN>, kSmem));
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kBlkThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
  }
  FewLaunch(const FewLaunch&) = delete;
};
// The clusters of `split` CTAs that are resident together on the current device (a GPC's SMs need not divide
// into clusters, and cards differ), asked for once for each device and size.
template <int EPI, bool B_MN>
int resident_clusters(int split) {
  static DeviceTable<kMaxSplit + 1> resident;
  return resident.get(c10::cuda::current_device(), split, [split] {
    int clusters = 0;
    const FewLaunch<EPI, B_MN> l(split, split, nullptr);
    AT_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&clusters, gemm_few_kernel<EPI, B_MN>, &l.cfg));
    TORCH_CHECK(clusters > 0, "no cluster of the fp8 GEMM fits on this device");
    return clusters;
  });
}

// The forms that a call's rows take, and the launches, for a call that may use `sms` of a device's `all` SMs.
// rows: of all groups together (segments; an upper bound), or of a slab, whose counts only the device knows.
// clusters(split): clusters of that size that are resident together.
template <typename Clusters>
Plan make_plan(int64_t G, int64_t rows, int64_t N, int64_t K, bool masked, int sms, int all, Clusters clusters) {
  Plan p{};
  p.sms = sms;
  const int64_t ntn = (N + kBN - 1) / kBN, KB = (K + kBK - 1) / kBK;
  // tiles of groups with few rows: one a group (slabs), or as many as the rows make
  const int64_t some = std::min(G, rows);
  const int64_t few = (masked ? G : std::max(some, (rows + kFewTile - 1) / kFewTile)) * ntn;
  int64_t least = -1;
  for (int s = 1; s <= kMaxSplit && s * 2 <= std::max<int64_t>(KB, 2) && s <= sms; s *= 2) {
    const int grid = s == 1 ? sms : std::max(1, std::min(clusters(s), sms / s)) * s;
    const int64_t cycles = few_cycles(few, KB, grid, s);
    if (least < 0 || cycles < least) {
      least = cycles;
      p.split = s;
      p.few_grid = grid;
    }
  }
  p.many_grid = sms;
  if (!masked) {
    p.few_grid = static_cast<int>(std::min<int64_t>(p.few_grid, few * p.split));   // no CTA without work
    // half a tile more a group than its rows fill, on average, and at least one
    const int64_t many = std::max<int64_t>(some, (rows + kBM - 1) / kBM + some / 2) * ntn;
    p.form = least < many_cycles(many, KB, sms, many == some * ntn) ? kAllFew : kAllMany;
    p.many_grid = static_cast<int>(std::min<int64_t>(sms, many));
  } else {
    // a decoding step, a tile a group, decides whether the form for few rows is worth its launch
    p.form = least >= many_cycles(few, KB, sms, true) ? kAllMany : rows <= kFewTile ? kAllFew : kBothForms;
  }
  // side by side the two kernels may hold twice `sms` SMs, which a caller that keeps some back must not see
  p.overlap = p.form == kBothForms && sms >= all;
  return p;
}

int granted_sms(int64_t num_sms, int all) { return num_sms > 0 ? static_cast<int>(std::min<int64_t>(num_sms, all)) : all; }

template <int EPI, bool B_MN>
void launch_block(const CUtensorMap& ma, const CUtensorMap& mf, const CUtensorMap& mb, BlkArgs a, bool masked,
                  int64_t num_sms, cudaStream_t stream) {
  const int all = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const Plan& p = a.plan =
      make_plan(a.G, a.rows, a.N, a.K, masked, granted_sms(num_sms, all), all, resident_clusters<EPI, B_MN>);
  if (p.form != kAllMany) {
    const FewLaunch<EPI, B_MN> l(p.few_grid, p.split, stream);
    AT_CUDA_CHECK(cudaLaunchKernelEx(&l.cfg, gemm_few_kernel<EPI, B_MN>, mf, mb, a));
  }
  if (p.form == kAllFew) return;
  constexpr int smem = 1024 + kStages * kStageBytes + kEpiWarps * kWarpStage;
  auto kfn = gemm_block_kernel<EPI, B_MN>;
  static std::atomic<uint64_t> seen{0};
  AT_CUDA_CHECK(set_smem_limit_once(seen, kfn, smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.many_grid);
  cfg.blockDim = dim3(kBlkThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = p.overlap ? 1 : 0;
  AT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kfn, ma, mb, a));
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
  const int64_t most_tiles = ((masked ? int64_t(a.G) * ((a.rows + kFewTile - 1) / kFewTile) : a.rows / kFewTile + a.G)) *
                             ((N + kBN - 1) / kBN);
  TORCH_CHECK(most_tiles < (1ll << 30), "too many tiles");
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
  a.timeout_ns = timeout_ns(timeout_s);
  // a stride over a dimension of one element is arbitrary; the map wants a legal one
  auto stride = [](const at::Tensor& t, int64_t d, int64_t otherwise) { return t.size(d) > 1 ? t.stride(d) : otherwise; };
  const int64_t s1 = stride(A, A.dim() - 2, K);
  const CUtensorMap ma = masked ? map_u8_3d(A.data_ptr(), K, a.rows, a.G, s1, stride(A, 0, s1 * a.rows), kBM)
                                : map_u8_3d(A.data_ptr(), K, a.rows, 1, s1, s1 * a.rows, kBM);
  const CUtensorMap mf = masked ? map_u8_3d(A.data_ptr(), K, a.rows, a.G, s1, stride(A, 0, s1 * a.rows), kFewTile)
                                : map_u8_3d(A.data_ptr(), K, a.rows, 1, s1, s1 * a.rows, kFewTile);
  const CUtensorMap mb = b_kn ? map_u8_3d(B.data_ptr(), N, K, a.G, N, N * K, kBK)
                              : map_u8_3d(B.data_ptr(), K, N, a.G, K, N * K, kBN);
  auto stream = at::cuda::getCurrentCUDAStream();
  if (epilogue == kOutSwiGLU) launch_block<kOutSwiGLU, false>(ma, mf, mb, a, masked, num_sms, stream);
  else if (epilogue == kOutBF16 && b_kn) launch_block<kOutBF16, true>(ma, mf, mb, a, masked, num_sms, stream);
  else if (epilogue == kOutBF16) launch_block<kOutBF16, false>(ma, mf, mb, a, masked, num_sms, stream);
  else if (b_kn) launch_block<kOutF32, true>(ma, mf, mb, a, masked, num_sms, stream);
  else launch_block<kOutF32, false>(ma, mf, mb, a, masked, num_sms, stream);
}

std::tuple<std::string, int64_t, int64_t, int64_t, bool> fp8_block_plan(
    int64_t G, int64_t rows, int64_t N, int64_t K, bool masked, int64_t num_sms,
    const c10::optional<std::vector<int64_t>>& counts, const c10::optional<std::vector<int64_t>>& device) {
  using namespace gemm;
  TORCH_CHECK(G >= 1 && rows >= 1 && N >= 1 && K >= 1, "sizes above zero");
  Plan p;
  if (device.has_value()) {   // SMs, and resident clusters of 2, 4 and 8 CTAs
    TORCH_CHECK(device->size() == 4 && device->at(0) >= 1, "a device is its SMs and its resident clusters of 2, 4 and 8 CTAs");
    const int all = static_cast<int>(device->at(0));
    p = make_plan(G, rows, N, K, masked, granted_sms(num_sms, all), all,
                  [&](int s) { return static_cast<int>(device->at(s == 2 ? 1 : s == 4 ? 2 : 3)); });
  } else {
    const int all = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    p = make_plan(G, rows, N, K, masked, granted_sms(num_sms, all), all, resident_clusters<kOutBF16, false>);
  }
  std::string form = p.form == kAllMany ? "many" : p.form == kAllFew ? "few" : "both";
  if (p.form == kBothForms && counts.has_value()) {
    Tally t{};
    for (const int64_t n : *counts) t.add(static_cast<int>(std::max<int64_t>(0, std::min(n, rows))));
    const int few_rows = few_rows_of(t, N, K, p);
    form = few_rows == INT_MAX ? "both: few" : few_rows == 0 ? "both: many" : "both: mixed";
  }
  return {form, p.split, p.form == kAllMany ? 0 : p.few_grid, p.form == kAllFew ? 0 : p.many_grid, p.overlap};
}

}  // namespace b200ep
