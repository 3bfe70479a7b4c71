// gemm_fp8_many.cu's products where every scale is a power of two, as this package's own conversions make them: the tensor cores
// then apply the scales themselves.
//
//   y[m, n] = sum_b sum_{k in block b} (x[m, k] * sx[b, m]) * (w[n, k] * sw[n / 128, b])
//
// tcgen05.mma kind::mxf8f6f4 takes, for every 32 elements of a row of either operand, a scale of 8 exponent bits; a block of 128
// gives its four the same one.  Nothing is left to do between two blocks of K: sums stay in tensor memory over all of K, and two
// SMs share a tile of 256 x 256 (cta_group::2), each with half of both operands in its shared memory.
//
// The tensor cores cut a sum to float32 after every 32 terms, where the other two kernels take a block's sum out and round: sums of
// 12,288 terms of one sign are 111 * 2^-24 of their value off on average (4,096 terms: 22), all towards zero, against 2 * 2^-24 there
// (1.2); of random signs 0.13 and 0.02 * 2^-24 of the terms' magnitudes.  A bfloat16 result is rounded by up to 65,536 * 2^-24.
//
// Scales lie in tensor memory too.  One warp turns the float32 scales of four k blocks into bytes, a word of them for each row of x
// and for the two blocks of weight rows, as 32 lanes x 16 bytes for 128 rows; tcgen05.cp copies them up in front of the MMAs that use
// them, byte i for the i-th of the four blocks.
//
// What bounds it is the thread that issues the MMAs: a stage's eight run 1,024 cycles, and each load from shared memory takes that
// thread some 200 while they do.  So it waits for one barrier a stage and commits once; scales have a thread of their own, which copies
// them up and arrives for the stage.  (With waits for scales and the copies in the issuing thread: 1,330 cycles a stage, 2,048 x 4,096 x
// 6,144 52 us; as it is 46.)  2,048 x 4,096 to 2 * 12,288 gated 160 us, 2.57 PFLOP/s, of which the power cap takes a part; in tiles of
// 128 x 256 with a multiply-add an output and block 233.
//
// A tile's sums take half of tensor memory, and with scales there is no room for two: the epilogue's eight warps fetch all of it into
// registers and hand it back before they convert or store anything.
//
// Roles: warp 0 copies x and the weights, warp 1 (in the pair's first block) copies scales up, warp 2 allocates tensor memory and (in
// the first block) issues the MMAs, warp 3 prepares scales, warps 4 to 11 are the epilogue.
//
// Every wait is bounded; one that runs out records kStatusWaitTimedOut and every role leaves its loop.  The blocks then tell each other
// how far they came, and both stay until MMAs, copies of scales and both blocks' copies have finished (bounded again; drain.h).
#include "api.h"
#include "drain.h"
#include "fp8_out.cuh"

namespace pe {
namespace fp8pair {
using namespace fp8;

constexpr int BM = 128;          // rows of x of a block: half of a tile
constexpr int BN = 256;          // weight rows of a tile, half of them copied by each block
constexpr int KBS = 2;           // k blocks of a stage
constexpr int STAGES = 3;
constexpr int kBytes = KBS * BM * BK;                       // of one operand's half in a stage
constexpr int kStage = 2 * kBytes;
constexpr int kChunk = 4;        // k blocks whose scales go together
constexpr int SLOTS = 4;         // chunks of scales
constexpr int kSlot = 3 * 512;   // 128 rows of x, 2 x 128 weight rows
constexpr int kTmemCols = 512, kScaleCols = 256, kSlotCols = 16;
constexpr int kRoles = 4, kThreads = 32 * (kRoles + 8);
constexpr size_t kSmem = 1024 + (size_t)STAGES * kStage + SLOTS * kSlot + 8 * kOutWarp;
static_assert(kChunk % KBS == 0, "a stage's scales are of one chunk");

struct Params {
  int M, K, k_blocks;
  bool whole;
  const float* xs; long long xs_ld;
  const float* ws; long long ws_group;  // per group [ceil(w rows / 128)][k_blocks]
  int w_rows;
  const int* offsets; int n_groups;     // null, 0: one group of M rows
  int m_tiles, n_tiles;                 // m_tiles: without groups
  Output out;
  int* status;
};

__device__ __forceinline__ void tmem_alloc2(uint32_t* holder_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(holder_smem)), "r"(cols));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(cols));
}
// copies into this block's shared memory whose bytes count on a barrier that may be the other block's
__device__ __forceinline__ void load_3d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
      ::"r"(tma::smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void load_5d_pair(void* dst, const CUtensorMap* map, int x, int row, int block, int group, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];\n"
      ::"r"(tma::smem_addr(dst)), "l"(map), "r"(x), "r"(row), "r"(0), "r"(block), "r"(group), "r"(bar) : "memory");
}
// arrive on the barrier at this place in both blocks once all that was issued so far has completed
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  const uint16_t mask = 3;
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
               ::"r"(tma::smem_addr(bar)), "h"(mask) : "memory");
}
__device__ __forceinline__ void commit_one(uint64_t* bar) {        // in this block only
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(tma::smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;\n" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// 32 rows of 16 bytes to four columns of tensor memory, the same in all four quarters of its lanes; in both blocks
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ uint64_t scales_desc(uint32_t saddr) {      // no swizzle: 8 rows of 16 bytes, the next 8 behind them
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(128 >> 4) << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  return d;
}
__device__ __forceinline__ void umma_scaled(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// kind::mxf8f6f4: B's scale byte at [4,6), A and B e4m3 (7-9 and 10-12: 0), N >> 3 at [17,23), scales of exponent bits (23), M >> 4 at
// [24,29) (a pair's M counts both blocks), A's scale byte at [29,31)
__device__ __forceinline__ constexpr uint32_t instr_desc_scaled(int m, int n, uint32_t byte) {
  return (byte << 4) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) | (byte << 29);
}

template <int MODE, bool GROUPS>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_pair_kernel(Params p, const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap) {
  constexpr bool GLU = MODE == kGlu || MODE == kGluFp8;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], sf_full[SLOTS], sf_empty[SLOTS], acc_full, acc_empty, drained;
  __shared__ float top_s[2][BM];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int failed;
  __shared__ int started, fed;            // stages whose copies were started, whose scales were handed over
  __shared__ int their_started, their_failed;   // the other block's, when all is over
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  char* scales_s = smem + STAGES * kStage;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const bool leader = rank == 0;
  constexpr int kPerTile = GLU ? BN / 2 : BN;     // outputs of a row in a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tma::mbar_init(&full_bar[s], 2);    // the leader's: its producer, bytes of both blocks, and its scales
      tma::mbar_init(&empty_bar[s], 1);   // a commit, delivered to both blocks
    }
    for (int s = 0; s < SLOTS; ++s) {
      tma::mbar_init(&sf_full[s], 2);     // the leader's: the scale warps of both blocks
      tma::mbar_init(&sf_empty[s], 1);    // a commit, delivered to both blocks
    }
    tma::mbar_init(&acc_full, 1);         // a commit, delivered to both blocks
    tma::mbar_init(&acc_empty, 16);       // the leader's: the epilogue warps of both blocks
    tma::mbar_init(&drained, 2);          // commits behind all that warps 1 and 2 issued, delivered to both blocks
    failed = started = fed = 0;
    tma::fence_barrier_init();
  }
  if (warp == 2) tmem_alloc2(&tmem_holder, kTmemCols);
  fence_before_sync();
  __syncthreads();
  cluster_sync();                         // the other block's barriers exist before anything is sent to them
  fence_after_sync();
  const uint32_t tmem_base = tmem_holder;
  pdl_wait_block();
  pdl_launch_dependents();
  const int m_tiles = GROUPS ? count_tiles(p.offsets, p.n_groups, p.M, 2 * BM) : p.m_tiles;
  const int n_tiles_total = m_tiles * p.n_tiles, first_tile = (int)blockIdx.x >> 1, tile_step = (int)gridDim.x >> 1;
  const int my_tiles = max(0, (n_tiles_total - first_tile + tile_step - 1) / tile_step);
  const int n_st = (p.k_blocks + KBS - 1) / KBS, n_ch = (p.k_blocks + kChunk - 1) / kChunk, chunks = my_tiles * n_ch;
  auto find = [&](int tile, int& group, int& row0, int& rows) {         // this block's rows; all lanes of a warp take part
    const int mt = tile % m_tiles;
    group = 0;
    row0 = mt * 2 * BM;
    rows = min(2 * BM, p.M - row0);
    if (GROUPS) find_group(p.offsets, p.n_groups, p.M, 2 * BM, mt, group, row0, rows);
    row0 += rank * BM;
    rows = min(rows - rank * BM, BM);
  };

  if (warp == 0) {
    int g = 0;                            // stages so far
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles_total && ok; tile += tile_step) {
      int group, m0, rows;
      find(tile, group, m0, rows);
      const int n0 = (tile / m_tiles) * kPerTile, w_row = GLU ? n0 + rank * p.out.N : n0 + rank * BM;
      if (lane == 0) {
        for (int st = 0; st < n_st && ok; ++st, ++g) {
          const int stage = g % STAGES;
          ok = tma::mbar_wait(&empty_bar[stage], ((g / STAGES) & 1) ^ 1);
          if (!ok) break;
          char* to = smem + stage * kStage;
          if (leader) tma::mbar_expect_tx(&full_bar[stage], 2 * kStage);
          const uint32_t bar = map_to_rank(tma::smem_addr(&full_bar[stage]), 0);
          if (p.whole) {                  // blocks beyond K arrive as zeros and still count
            load_3d_pair(to, &amap, 0, m0, st * KBS, bar);
            load_5d_pair(to + kBytes, &bmap, 0, w_row, st * KBS, group, bar);
          } else {
            for (int j = 0; j < KBS; ++j) {
              load_3d_pair(to + j * BM * BK, &amap, (st * KBS + j) * BK, m0, 0, bar);
              load_5d_pair(to + kBytes + j * BM * BK, &bmap, (st * KBS + j) * BK, w_row, 0, group, bar);
            }
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    }
    if (lane == 0) started = g;
    if (!ok) {
      if (lane == 0) report(p.status, kStatusWaitTimedOut, 100, (int)blockIdx.x, g);
      failed = 1;
    }
  } else if (warp == 1) {
    // Copies scales up, a chunk ahead of the MMAs, and arrives for each stage: behind the copies where a chunk begins.  A slot of
    // tensor memory is written again when this thread has seen a stage empty whose predecessor by three, the slot's last user or a later one,
    // is then done (a chunk has a stage at least).
    if (leader && lane == 0) {
      const uint32_t sf_base = tma::smem_addr(scales_s);
      auto copy_up = [&](int c) {
        const int slot = c % SLOTS;
        if (!tma::mbar_wait(&sf_full[slot], (c / SLOTS) & 1)) return false;
        fence_after_sync();
        const uint32_t from = sf_base + slot * kSlot, to = tmem_base + kScaleCols + slot * kSlotCols;
        copy_scales(to, scales_desc(from));
        copy_scales(to + 4, scales_desc(from + 512));
        copy_scales(to + 8, scales_desc(from + 1024));
        commit_both(&sf_empty[slot]);
        return true;
      };
      int g = 0, c = 0;
      bool ok = chunks == 0 || copy_up(0);
      for (int it = 0; it < my_tiles && ok; ++it) {
        for (int st = 0; st < n_st; ++st, ++g) {
          const int stage = g % STAGES;
          ok = tma::mbar_wait(&empty_bar[stage], ((g / STAGES) & 1) ^ 1);
          if (!ok) break;
          if (st * KBS % kChunk == 0) {
            commit_one(&full_bar[stage]);
            fed = g + 1;
            if (++c < chunks) ok = copy_up(c);
            if (!ok) break;
          } else {
            tma::mbar_arrive(&full_bar[stage]);
            fed = g + 1;
          }
        }
      }
      if (!ok) {
        report(p.status, kStatusWaitTimedOut, 105, (int)blockIdx.x, g);
        failed = 1;
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    if (leader && lane == 0) {
      // Little beside the MMAs: they run 1,024 cycles a stage, and every load from shared memory takes this thread 200 beside theirs.
      const uint32_t base = tma::smem_addr(smem);
      int g = 0, c = 0;                   // stages and chunks of scales so far
      bool ok = true;
      for (int it = 0; it < my_tiles && ok; ++it) {
        ok = tma::mbar_wait(&acc_empty, (it & 1) ^ 1);
        for (int st = 0; st < n_st && ok; ++st, ++g) {
          const int stage = g % STAGES, kb0 = st * KBS;
          ok = tma::mbar_wait(&full_bar[stage], (g / STAGES) & 1);
          if (!ok) break;
          fence_after_sync();
          const uint32_t sfa = tmem_base + kScaleCols + c % SLOTS * kSlotCols, sfb = sfa + 4;
          const uint32_t sa = base + stage * kStage, sb = sa + kBytes;
#pragma unroll
          for (int j = 0; j < KBS; ++j) {
            if (kb0 + j >= p.k_blocks) break;
            const uint32_t idesc = instr_desc_scaled(2 * BM, BN, (uint32_t)((kb0 + j) % kChunk));
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma_scaled(tmem_base, smem_desc(sa + j * BM * BK + k * 32), smem_desc(sb + j * BM * BK + k * 32), idesc, sfa, sfb,
                          kb0 > 0 || j > 0 || k > 0 ? 1u : 0u);
          }
          commit_both(&empty_bar[stage]);
          if ((kb0 + KBS) % kChunk == 0 || st == n_st - 1) ++c;
        }
        if (ok) commit_both(&acc_full);
      }
      if (!ok) {
        report(p.status, kStatusWaitTimedOut, 101, (int)blockIdx.x, g);
        failed = 1;
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    int c = 0;
    bool ok = true;
    for (int tile = first_tile; tile < n_tiles_total && ok; tile += tile_step) {
      int group, m0, rows;
      find(tile, group, m0, rows);
      const int n0 = (tile / m_tiles) * kPerTile, last = (p.w_rows - 1) / 128;
      const float* ws = p.ws + (size_t)group * p.ws_group;
      const float* w0 = ws + (size_t)min(n0 / 128, last) * p.k_blocks;
      const float* w1 = ws + (size_t)min(GLU ? (p.out.N + n0) / 128 : n0 / 128 + 1, last) * p.k_blocks;
      float x[4][kChunk], w[2][kChunk];
      auto fetch = [&](int kb0) {         // what is not there counts as 1: its operands are zeros
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          const bool there = kb0 + j < p.k_blocks;
          w[0][j] = there ? w0[kb0 + j] : 1.f;
          w[1][j] = there ? w1[kb0 + j] : 1.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q][j] = there && q * 32 + lane < rows ? p.xs[(size_t)(kb0 + j) * p.xs_ld + m0 + q * 32 + lane] : 1.f;
        }
      };
      auto word = [&](const float (&s)[kChunk]) {
        uint32_t v = 0;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v |= (__float_as_uint(s[j]) >> 23 & 0xffu) << (8 * j);
        return v;
      };
      fetch(0);
      for (int ch = 0; ch < n_ch; ++ch, ++c) {
        const int slot = c % SLOTS;
        ok = __all_sync(0xffffffffu, tma::mbar_wait(&sf_empty[slot], ((c / SLOTS) & 1) ^ 1));
        if (!ok) {
          if (lane == 0) report(p.status, kStatusWaitTimedOut, 103, tile, ch);
          failed = 1;
          break;
        }
        const uint32_t a = word(w[0]), b = word(w[1]);
        uint4* to = reinterpret_cast<uint4*>(scales_s + slot * kSlot) + lane;
        to[0] = make_uint4(word(x[0]), word(x[1]), word(x[2]), word(x[3]));
        to[32] = make_uint4(a, a, a, a);
        to[64] = make_uint4(b, b, b, b);
        tma::fence_proxy_async();
        __syncwarp();
        if (lane == 0) arrive_cluster(map_to_rank(tma::smem_addr(&sf_full[slot]), 0));
        if (ch + 1 < n_ch) fetch((ch + 1) * kChunk);       // behind the fence, which waits for loads too
      }
    }
  } else {
    const int quarter = warp & 3, h = (warp - kRoles) >> 2;
    char* out_buf = scales_s + SLOTS * kSlot + (warp - kRoles) * kOutWarp;
    // first columns of the thread's two runs of 64
    const int c0 = GLU ? h * 64 : h * 128, c1 = GLU ? 128 + h * 64 : h * 128 + 64;
    const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
    int it = 0;
    // the fused conversion has barriers in it: after a wait that ran out the warps go on without waiting
    for (int tile = first_tile; tile < n_tiles_total; tile += tile_step, ++it) {
      int group, m0, rows;
      find(tile, group, m0, rows);
      const int n0 = (tile / m_tiles) * kPerTile;
      if (!failed && !tma::mbar_wait(&acc_full, it & 1)) {
        if (lane == 0) report(p.status, kStatusWaitTimedOut, 104, tile, it);
        failed = 1;
      }
      __syncwarp();
      fence_after_sync();
      float acc[128];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        uint32_t(&v)[16] = reinterpret_cast<uint32_t(&)[16]>(acc[16 * q]);
        tmem_ld16(t_row + (q < 4 ? c0 + q * 16 : c1 + (q - 4) * 16), v);
      }
      tmem_ld_wait();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_cluster(map_to_rank(tma::smem_addr(&acc_empty), 0));
      finish_tile<MODE, GROUPS>(p.out, acc, m0, rows, n0, h, quarter, lane, failed != 0, out_buf, top_s);
    }
  }
  // both blocks meet: neither may leave while the other's copies, commits or arrivals can still reach it
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0) {
    st_cluster(map_to_rank(tma::smem_addr(&their_started), rank ^ 1), started);
    st_cluster(map_to_rank(tma::smem_addr(&their_failed), rank ^ 1), failed);
  }
  __syncwarp();
  cluster_sync();
  if (failed || their_failed) {           // the same answer in both blocks
    // MMAs, which read both blocks' shared memory, copies of scales, and the commits behind them
    if (leader && lane == 0 && (warp == 1 || warp == 2)) commit_both(&drained);
    if (warp == 2 && lane == 0) {
      tma::mbar_wait(&drained, 0);
      if (leader) {                       // both blocks' copies count on this block's barriers
        const int last = max(started, their_started);
        for (int i = max(0, last - STAGES); i < last; ++i) {
          uint64_t* bar = &full_bar[i % STAGES];
          const Owed o = owed_to_stage(i, started, their_started, fed, kStage);
          if (o.expect) tma::mbar_expect_only(bar, o.expect);
          if (o.complete) tma::mbar_complete_only(bar, o.complete);
          for (int k = 0; k < o.arrivals; ++k) tma::mbar_arrive(bar);
          tma::mbar_wait(bar, (i / STAGES) & 1);
        }
      }
    }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 2) {
    fence_after_sync();
    tmem_dealloc2(tmem_base, kTmemCols);
  }
}

template <int MODE, bool GROUPS>
static int launch_mode(const Params& p, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  static bool asked[kDevices] = {};
  const int e = allow_smem_once(gemm_fp8_pair_kernel<MODE, GROUPS>, kSmem, asked);
  if (e != 0) return e;
  // with groups: as many tiles of rows as there can be
  const long long most = GROUPS ? p.M / (2 * BM) + (p.n_groups < p.M ? p.n_groups : p.M) : p.m_tiles, tiles = most * p.n_tiles;
  const int pairs = (int)(tiles < pe::kSMs / 2 ? tiles : pe::kSMs / 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pe::pdl_enabled() ? 2 : 1;
  const cudaError_t ce = cudaLaunchKernelEx(&cfg, gemm_fp8_pair_kernel<MODE, GROUPS>, p, amap, bmap);
  if (ce != cudaSuccess) return (int)ce;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

}  // namespace fp8pair
}  // namespace pe

// The arguments of pe_gemm_fp8_many; all scales are powers of two (of others the exponent is taken).
extern "C" int pe_gemm_fp8_pair(const void* x, long long x_ld, const float* x_scales, long long xs_ld, const void* w, long long w_ld,
                                const float* w_scales, void* y, long long ldy, float* y_scales, long long ys_ld, int M, int N, int K,
                                int out_f32, int kind, float limit, float alpha, const float* bias, const float* row_weight,
                                const int* offsets, int n_groups, int* status, cudaStream_t stream) {
  using namespace pe::fp8pair;
  if (M < 0 || N < 0 || K < 1 || kind < 0 || kind > 3 || n_groups < 0) return PE_ERR_BAD_ARGUMENT;
  if (M == 0 || N == 0) return PE_OK;
  if (M > kMostRows || K > kMostRows) return PE_ERR_UNSUPPORTED_SIZE;
  if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr) return PE_ERR_BAD_ARGUMENT;
  if (x_ld < K || w_ld < K || xs_ld < M || ldy < N || (kind > 0 && out_f32) || (kind == 0 && (bias || y_scales)) || (row_weight && (kind == 0 || n_groups == 0)))
    return PE_ERR_BAD_ARGUMENT;
  if ((n_groups > 0) != (offsets != nullptr)) return PE_ERR_BAD_ARGUMENT;
  if (((uintptr_t)x % 16) || ((uintptr_t)w % 16) || (x_ld % 16) || (w_ld % 16)) return PE_ERR_BAD_ARGUMENT;
  if (y_scales && ((ldy % 16) || ((uintptr_t)y % 16) || ys_ld < M)) return PE_ERR_BAD_ARGUMENT;
  const int groups = n_groups > 0 ? n_groups : 1;
  if ((kind > 0 && N % 128) || N > (1 << 28) || (long long)groups * N > (1 << 29)) return PE_ERR_UNSUPPORTED_SIZE;
  Params p;
  p.M = M; p.K = K; p.k_blocks = (K + BK - 1) / BK; p.whole = K % BK == 0;
  p.xs = x_scales; p.xs_ld = xs_ld; p.ws = w_scales;
  p.w_rows = kind > 0 ? 2 * N : N;
  p.ws_group = (long long)((p.w_rows + 127) / 128) * p.k_blocks;
  p.offsets = offsets; p.n_groups = n_groups;
  p.m_tiles = (M + 2 * BM - 1) / (2 * BM);
  p.n_tiles = kind > 0 ? N / (BN / 2) : (N + BN - 1) / BN;
  p.out = Output{N, y, ldy, y_scales, ys_ld, row_weight, pe::GluEpilogue{kind, limit, alpha, bias}};
  p.status = status;
  if (((long long)p.m_tiles + n_groups) * p.n_tiles * p.k_blocks > 0x7fffffffLL) return PE_ERR_UNSUPPORTED_SIZE;
  CUtensorMap amap, bmap;
  int e = make_map(&amap, x, K, M, x_ld, BM, p.whole, KBS);
  if (e == 0) e = make_weight_map(&bmap, w, K, p.w_rows, w_ld, false, groups, BM, p.whole, KBS);
  if (e != 0) return e;
#define PE_PAIR(MODE) (n_groups > 0 ? launch_mode<MODE, true>(p, amap, bmap, stream) : launch_mode<MODE, false>(p, amap, bmap, stream))
  return kind == 0 ? (out_f32 ? PE_PAIR(kF32) : PE_PAIR(kBf16)) : y_scales ? PE_PAIR(kGluFp8) : PE_PAIR(kGlu);
#undef PE_PAIR
}
