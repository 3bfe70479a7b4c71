// gemm_fp8.cu's products for many rows: y = x . W^T of e4m3 operands with a scale for each block of 128, in tiles of 128 rows of x
// and 256 weight rows.
//
//   y[m, n] = sum_b sx[b, m] * sw[n / 128, b] * sum_{k in block b} x[m, k] * w[n, k]
//
// A k block of 128 is four MMAs (tcgen05.mma kind::f8f6f4) into one of two halves of tensor memory (256 columns), and its sums are
// added up in registers while the next block's MMAs fill the other half.  The rows of x are the MMA's M dimension, so that an
// epilogue thread owns one row: 128 of its columns lie in one block of weight rows, and a block of 128 x 128 outputs takes one
// multiply-add an output with one number a thread, sx * sw.
//
// What bounds it is the way round a half of tensor memory: MMAs, commit, eight warps that read it, their arrival, the next MMAs.
// Two SMs on one tile (cta_group::2) load a third less but have that way lead through the other SM: 1,750 cycles a block and
// half, one SM 1,050.  (Where the scales are powers of two there is no way round: gemm_fp8_pair.cu.)  2,048 x 4,096 x 6,144 64 us,
// 2,048 x 4,096 to 2 * 12,288 gated 233 us, 1.77 PFLOP/s.
//
// GLU: the tile's weight rows are 128 gates and the 128 ups that belong to them, a thread owns 64 of each, and act(gate, up),
// rounded to bfloat16, goes out as it is or quantised again: the tile's 128 outputs of a row are one block, whose largest
// magnitude two threads find together.
//
// Roles: warps 0 and 1 copy x and the weights (TMA; a thread starts a copy only every 150 ns or so), warp 2 allocates tensor memory
// and issues the MMAs, warps 3 to 10 are the epilogue.
//
// Every wait is bounded; one that runs out records kStatusWaitTimedOut, every role leaves its loop, copies still in flight are
// waited for (bounded again) and tensor memory is freed.
#include "api.h"
#include "fp8_out.cuh"

namespace pe {
namespace fp8many {
using namespace fp8;

constexpr int BM = 128;          // rows of x of a tile
constexpr int BN = 256;          // weight rows of a tile
constexpr int STAGES = 4;        // of one k block
constexpr int kBytesA = BM * BK, kBytesB = BN * BK, kStage = kBytesA + kBytesB;
constexpr int kTmemCols = 512;
constexpr int kRoles = 3, kThreads = 32 * (kRoles + 8);
constexpr size_t kSmem = 1024 + (size_t)STAGES * kStage + 8 * kOutWarp;

struct Params {
  int M, N, K, k_blocks;                // N: output columns
  bool whole;
  const float* xs; long long xs_ld;
  const float* ws; long long ws_group;  // per group [ceil(w rows / 128)][k_blocks]
  const int* offsets; int n_groups;     // null, 0: one group of M rows
  int m_tiles, n_tiles;                 // m_tiles: without groups
  Output out;
  int* status;
};

// GROUPS: rows grouped by expert, and weights on rows; the plain products keep kernels of their own, which have registers left.
template <int MODE, bool GROUPS>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_many_kernel(Params p, const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap) {
  constexpr bool GLU = MODE == kGlu || MODE == kGluFp8;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2];
  __shared__ float top_s[2][BM];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int failed;
  __shared__ int started[2], issued;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kPerTile = GLU ? BN / 2 : BN;     // outputs of a row in a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tma::mbar_init(&full_bar[s], 2);    // the two producers
      tma::mbar_init(&empty_bar[s], 1);   // the commit behind a block's MMAs
    }
    for (int b = 0; b < 2; ++b) {
      tma::mbar_init(&acc_full[b], 1);
      tma::mbar_init(&acc_empty[b], 8);   // the epilogue's warps
    }
    failed = issued = 0;
    tma::fence_barrier_init();
  }
  if (warp == 2) tmem_alloc(&tmem_holder, kTmemCols);
  fence_before_sync();
  pdl_wait_block();
  pdl_launch_dependents();
  fence_after_sync();
  const uint32_t tmem_base = tmem_holder;
  // With groups the tiles of rows are those that the offsets give: none is empty.
  const int m_tiles = GROUPS ? count_tiles(p.offsets, p.n_groups, p.M, BM) : p.m_tiles;
  const int n_tiles_total = m_tiles * p.n_tiles;
  auto find = [&](int tile, int& group, int& row0, int& rows) {         // all lanes of a warp take part
    const int mt = tile % m_tiles;
    group = 0;
    row0 = mt * BM;
    rows = min(BM, p.M - row0);
    if (GROUPS) find_group(p.offsets, p.n_groups, p.M, BM, mt, group, row0, rows);
  };

  int loaded = 0;                         // warps 0 and 1: blocks whose copies were started
  if (warp < 2) {
    for (int tile = blockIdx.x; tile < n_tiles_total; tile += gridDim.x) {
      if (__any_sync(0xffffffffu, failed)) break;
      int group, m0, rows;
      find(tile, group, m0, rows);
      const int n0 = (tile / m_tiles) * kPerTile;
      if (lane == 0) {
        for (int kb = 0; kb < p.k_blocks; ++kb, ++loaded) {
          const int stage = loaded % STAGES;
          if (!tma::mbar_wait(&empty_bar[stage], ((loaded / STAGES) & 1) ^ 1)) {
            report(p.status, kStatusWaitTimedOut, 90, tile, kb);
            failed = 1;
            break;
          }
          char* to = smem + stage * kStage;
          const int x = p.whole ? 0 : kb * BK, z = p.whole ? kb : 0;
          if (warp == 0) {
            tma::mbar_expect_tx(&full_bar[stage], kBytesA);
            load_3d(to, &amap, x, m0, z, &full_bar[stage]);
          } else {
            tma::mbar_expect_tx(&full_bar[stage], kBytesB);
            load_5d(to + kBytesA, &bmap, x, n0, z, group, &full_bar[stage]);
          }
        }
      }
      __syncwarp();
    }
  } else if (warp == 2) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(BM, BN);
      const int my_tiles = max(0, (n_tiles_total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x);
      const int total = my_tiles * p.k_blocks;      // k blocks: block `it` goes to half it & 1 of tensor memory
      const uint32_t base = tma::smem_addr(smem);
      for (int it0 = 0; it0 < total && !failed; it0 += STAGES) {
#pragma unroll
        for (int stage = 0; stage < STAGES; ++stage) {
          const int it = it0 + stage, half = stage & 1;
          if (it >= total) break;
          if (!tma::mbar_wait(&full_bar[stage], (it / STAGES) & 1) || !tma::mbar_wait(&acc_empty[half], ((it >> 1) & 1) ^ 1)) {
            report(p.status, kStatusWaitTimedOut, 91, (int)blockIdx.x, it);
            failed = 1;
            break;
          }
          fence_after_sync();
          const uint32_t sa = base + stage * kStage, sb = sa + kBytesA;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma(tmem_base + half * BN, smem_desc(sa + k * 32), smem_desc(sb + k * 32), idesc, k > 0 ? 1u : 0u);
          umma_commit(&acc_full[half]);
          umma_commit(&empty_bar[stage]);
          issued = it + 1;
        }
      }
    }
    __syncwarp();
  } else {
    // ---- epilogue: a warp owns a quarter of the rows (the tensor memory lanes that it may read) and half of the columns: 128
    // neighbouring ones, or with GLU 64 gates and their 64 ups ----
    const int quarter = warp & 3, h = (warp - kRoles) >> 2;
    const int r_tile = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    char* out_buf = smem + STAGES * kStage + (warp - kRoles) * kOutWarp;
    // first columns of the thread's two runs of 64
    const int c0 = GLU ? h * 64 : h * 128, c1 = GLU ? 128 + h * 64 : h * 128 + 64;
    int it = 0;
    // the fused conversion has barriers in it: after a wait that ran out the warps go on without waiting
    for (int tile = blockIdx.x; tile < n_tiles_total; tile += gridDim.x) {
      int group, m0, rows;
      find(tile, group, m0, rows);
      const int n0 = (tile / m_tiles) * kPerTile;
      const int row = m0 + r_tile;
      const bool live = r_tile < rows;
      const float* sx_p = p.xs + (live ? row : 0);
      const int last = ((GLU ? 2 * p.N : p.N) - 1) / 128;
      const float* ws = p.ws + (size_t)group * p.ws_group;
      const float* sw0_p = ws + (size_t)min(GLU ? n0 / 128 : (n0 + c0) / 128, last) * p.k_blocks;
      const float* sw1_p = ws + (size_t)min(GLU ? (p.N + n0) / 128 : (n0 + c0) / 128, last) * p.k_blocks;
      unsigned long long sums[64];        // 128 sums, two neighbouring ones each
#pragma unroll
      for (int j = 0; j < 64; ++j) sums[j] = 0ull;
      float sx = live ? sx_p[0] : 0.f, sw0 = sw0_p[0], sw1 = GLU ? sw1_p[0] : 0.f;
      for (int kb = 0; kb < p.k_blocks; ++kb, ++it) {
        const int half = it & 1;
        const unsigned long long ss0 = pair_of(sx * sw0, sx * sw0), ss1 = GLU ? pair_of(sx * sw1, sx * sw1) : ss0;
        if (kb + 1 < p.k_blocks) {        // the next block's scales are on their way during this one
          sx = live ? sx_p[(size_t)(kb + 1) * p.xs_ld] : 0.f;
          sw0 = sw0_p[kb + 1];
          if (GLU) sw1 = sw1_p[kb + 1];
        }
        if (!failed && !tma::mbar_wait(&acc_full[half], (it >> 1) & 1)) {
          if (lane == 0) report(p.status, kStatusWaitTimedOut, 92, tile, kb);
          failed = 1;
        }
        __syncwarp();
        fence_after_sync();
        const uint32_t t_row = tmem_base + half * BN + lanes;
        uint32_t v[2][16];
        tmem_ld16(t_row + c0, v[0]);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          tmem_ld_wait();
          if (q < 7) tmem_ld16(t_row + (q + 1 < 4 ? c0 + (q + 1) * 16 : c1 + (q - 3) * 16), v[(q + 1) & 1]);
          if (q == 7) {                   // all of the half is read: hand it back
            fence_before_sync();
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&acc_empty[half]);
          }
          const unsigned long long s = q < 4 ? ss0 : ss1;
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(sums[q * 8 + j], v[q & 1][2 * j], v[q & 1][2 * j + 1], s);
        }
      }
      float acc[128];
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        const float2 f = unpair(sums[j]);
        acc[2 * j] = f.x;
        acc[2 * j + 1] = f.y;
      }
      finish_tile<MODE, GROUPS>(p.out, acc, m0, rows, n0, h, quarter, lane, failed != 0, out_buf, top_s);
    }
  }
  if (warp < 2 && lane == 0) started[warp] = loaded;
  fence_before_sync();
  __syncthreads();
  if (warp == 2) {
    if (failed && lane == 0) {            // MMAs that still read this block's shared memory, copies still on their way to it
      for (int i = max(0, issued - STAGES); i < issued; ++i) tma::mbar_wait(&empty_bar[i % STAGES], (i / STAGES) & 1);
      const int last = max(started[0], started[1]);
      for (int i = max(0, last - STAGES); i < last; ++i) {
        if (i >= started[0] || i >= started[1]) tma::mbar_arrive(&full_bar[i % STAGES]);     // for the operand that was not asked for
        tma::mbar_wait(&full_bar[i % STAGES], (i / STAGES) & 1);
      }
    }
    __syncwarp();
    fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int MODE, bool GROUPS>
static int launch_groups(const Params& p, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  static bool asked[kDevices] = {};
  const int e = allow_smem_once(gemm_fp8_many_kernel<MODE, GROUPS>, kSmem, asked);
  if (e != 0) return e;
  // with groups: as many tiles of rows as there can be
  const long long most = p.n_groups > 0 ? p.M / BM + (p.n_groups < p.M ? p.n_groups : p.M) : p.m_tiles, tiles = most * p.n_tiles;
  const cudaError_t ce = pe::launch(gemm_fp8_many_kernel<MODE, GROUPS>, dim3((unsigned)(tiles < pe::kSMs ? tiles : pe::kSMs)), dim3(kThreads), kSmem, stream, p, amap, bmap);
  if (ce != cudaSuccess) return (int)ce;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

template <int MODE>
static int launch_mode(const Params& p, const CUtensorMap& amap, const CUtensorMap& bmap, cudaStream_t stream) {
  return p.n_groups > 0 ? launch_groups<MODE, true>(p, amap, bmap, stream) : launch_groups<MODE, false>(p, amap, bmap, stream);
}

}  // namespace fp8many
}  // namespace pe

// The arguments of pe_gemm_fp8 (gemm_fp8.cu); with an activation N is a multiple of 128.  y_scales (or null): the outputs are
// quantised again, y is e4m3 (ldy bytes between rows, a multiple of 16) and y_scales[b * ys_ld + m] their blocks' scales.
extern "C" int pe_gemm_fp8_many(const void* x, long long x_ld, const float* x_scales, long long xs_ld, const void* w, long long w_ld,
                                const float* w_scales, void* y, long long ldy, float* y_scales, long long ys_ld, int M, int N, int K,
                                int out_f32, int kind, float limit, float alpha, const float* bias, const float* row_weight,
                                const int* offsets, int n_groups, int* status, cudaStream_t stream) {
  using namespace pe::fp8many;
  if (M < 0 || N < 0 || K < 1 || kind < 0 || kind > 3 || n_groups < 0) return PE_ERR_BAD_ARGUMENT;
  if (M == 0 || N == 0) return PE_OK;
  if (M > kMostRows || K > kMostRows) return PE_ERR_UNSUPPORTED_SIZE;
  if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr) return PE_ERR_BAD_ARGUMENT;
  if (x_ld < K || w_ld < K || xs_ld < M || ldy < N || (kind > 0 && out_f32) || (kind == 0 && (bias || y_scales)) || (row_weight && (kind == 0 || n_groups == 0)))
    return PE_ERR_BAD_ARGUMENT;
  if ((n_groups > 0) != (offsets != nullptr)) return PE_ERR_BAD_ARGUMENT;
  if (((uintptr_t)x % 16) || ((uintptr_t)w % 16) || (x_ld % 16) || (w_ld % 16)) return PE_ERR_BAD_ARGUMENT;
  if (y_scales && ((ldy % 16) || ((uintptr_t)y % 16) || ys_ld < M)) return PE_ERR_BAD_ARGUMENT;
  if ((kind > 0 && N % 128) || N > (1 << 28) || (long long)(n_groups > 0 ? n_groups : 1) * N > (1 << 29)) return PE_ERR_UNSUPPORTED_SIZE;
  Params p;
  p.M = M; p.N = N; p.K = K; p.k_blocks = (K + BK - 1) / BK; p.whole = K % BK == 0;
  p.xs = x_scales; p.xs_ld = xs_ld; p.ws = w_scales;
  const int w_rows = kind > 0 ? 2 * N : N;
  p.ws_group = (long long)((w_rows + 127) / 128) * p.k_blocks;
  p.offsets = offsets; p.n_groups = n_groups;
  p.m_tiles = (M + BM - 1) / BM;
  p.n_tiles = kind > 0 ? N / (BN / 2) : (N + BN - 1) / BN;
  p.out = Output{N, y, ldy, y_scales, ys_ld, row_weight, pe::GluEpilogue{kind, limit, alpha, bias}};
  p.status = status;
  if (((long long)p.m_tiles + n_groups) * p.n_tiles * p.k_blocks > 0x7fffffffLL) return PE_ERR_UNSUPPORTED_SIZE;
  CUtensorMap amap, bmap;
  int e = make_map(&amap, x, K, M, x_ld, BM, p.whole, 1);
  if (e == 0) e = make_weight_map(&bmap, w, K, N, w_ld, kind > 0, n_groups > 0 ? n_groups : 1, BN / (kind > 0 ? 2 : 1), p.whole, 1);
  if (e != 0) return e;
  if (kind == 0) return out_f32 ? launch_mode<kF32>(p, amap, bmap, stream) : launch_mode<kBf16>(p, amap, bmap, stream);
  return y_scales ? launch_mode<kGluFp8>(p, amap, bmap, stream) : launch_mode<kGlu>(p, amap, bmap, stream);
}
