// Products of e4m3 operands with a scale for each block of 128, for any number of rows:
//
//   y[m, n] = sum_b sx[b, m] * sw[n / 128, b] * sum_{k in block b} x[m, k] * w[n, k]
//
// The inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4), a k block of 128 into tensor memory columns of its own;
// the outer sum is taken in float32 registers, as the columns of one block after the other are read back.  So the scales cost one
// multiply-add an output and block and no operand is ever widened.
//
// With few rows the product is a stream of the weights through the SMs, and the operands' roles are chosen for that: 128
// weight rows are the MMA's M dimension, NP = 16 to 128 rows of x its N dimension.  Tensor memory then holds 256 / NP blocks' sums
// (16 for NP = 16), and the MMAs never wait for the epilogue while a block's weights are on their way.  K is split over the
// thread blocks of a cluster, which add their sums up through distributed shared memory in the order of their ranks (no
// atomics: the result does not depend on scheduling).
//
// Roles: warp 0 copies (TMA), warp 1 allocates tensor memory and issues the MMAs, the other warps are the epilogue: a thread
// owns a weight row (its tensor memory lane) and NP, for NP = 128 half of them, sums.  The first stages' weights are asked for before
// the kernel waits for its predecessor in the stream.
//
// GLU: a tile is 64 gate rows and the 64 up rows that belong to them, and y = act(gate, up), rounded to bfloat16.
// Groups (routed experts): the rows of x are ordered by group, offsets[g] .. offsets[g + 1] are those of group g, which has a
// matrix of its own; a tile of rows belongs to one group.
//
// Every wait is bounded; one that runs out records kStatusWaitTimedOut, every role leaves its loop, copies still in flight
// are waited for (bounded again) and tensor memory is freed.
#include "api.h"
#include "fp8.cuh"

namespace pe {
namespace fp8 {

struct Params {
  int M, N, K, k_blocks;               // N: output columns
  const float* xs; long long xs_ld;    // [k_blocks][xs_ld]
  const float* ws; long long ws_group; // per group [ceil(rows / 128)][k_blocks]
  int w_rows;                          // weight rows of a group: N, or 2 N with GLU
  void* y; long long ldy; int out_f32;
  int tok_tiles, split;
  const int* offsets; int n_groups;    // null, 0: one group of M rows
  GluEpilogue glu; const float* row_weight;
  int* status;
};

constexpr int kTile = 128;             // weight rows of a tile
constexpr int kTmemCols = 256;

template <int NP> struct Shape {
  static constexpr int kStages = NP == 16 ? 5 : NP == 32 ? 5 : NP == 64 ? 4 : 3;
  static constexpr int kStage = kTile * BK + NP * BK;
  static constexpr int kSlots = kTmemCols / NP;
  static constexpr int kEpiWarps = NP == 128 ? 8 : 4;
  static constexpr int kCols = NP / (kEpiWarps / 4);       // sums of a thread
  static constexpr int kThreads = 64 + 32 * kEpiWarps;
  static constexpr int kChunk = NP == 128 ? 16 : 32;       // k blocks whose scales lie in shared memory
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage;
};

__device__ __forceinline__ void epilogue_sync(int threads) { asm volatile("bar.sync 1, %0;\n" ::"r"(threads) : "memory"); }

// Which group, and which of its tiles of NP rows, token tile `j` is: all lanes of a warp take part.
// Offsets outside 0 .. M count as these.
__device__ __forceinline__ bool find_group(const int* offsets, int n_groups, int M, int np, int j, int& group, int& row0, int& rows) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < n_groups; base += 32) {
    const int g = base + lane;
    int lo = 0, n = 0;
    if (g < n_groups) {
      lo = min(max(offsets[g], 0), M);
      n = max(min(max(offsets[g + 1], 0), M) - lo, 0);
    }
    const int tiles = (n + np - 1) / np;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int first = before + sum - tiles;
    const unsigned hit = __ballot_sync(0xffffffffu, j >= first && j < first + tiles);
    if (hit) {
      const int from = __ffs(hit) - 1;
      group = base + from;
      const int t = j - __shfl_sync(0xffffffffu, first, from);
      row0 = __shfl_sync(0xffffffffu, lo, from) + t * np;
      rows = min(np, __shfl_sync(0xffffffffu, n, from) - t * np);
      return true;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

template <int NP, bool GLU>
__global__ void __launch_bounds__(Shape<NP>::kThreads, 2)
gemm_fp8_kernel(Params p, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
  using S = Shape<NP>;
  constexpr int STAGES = S::kStages, SLOTS = S::kSlots, EPI = S::kEpiWarps, COLS = S::kCols, CH = S::kChunk;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[SLOTS], acc_empty[SLOTS];
  __shared__ __align__(16) float sx_s[CH][NP];
  __shared__ float sw_s[CH][4];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int failed;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? (int)cluster_rank() : 0;
  const int tile = (int)blockIdx.x / p.split;
  const int row_tile = tile / p.tok_tiles, tok_tile = tile - row_tile * p.tok_tiles;
  const int n0 = row_tile * (GLU ? kTile / 2 : kTile);
  const int kb_lo = (int)((long long)p.k_blocks * rank / p.split), kb_hi = (int)((long long)p.k_blocks * (rank + 1) / p.split);
  const int n_kb = kb_hi - kb_lo;

  int group = 0, row0 = tok_tile * NP, rows = min(NP, p.M - row0);
  auto load_w = [&](int i) {           // the weights of this block's k block i
    const int stage = i % STAGES;
    char* sw = smem + stage * S::kStage;
    tma::mbar_expect_tx(&full_bar[stage], S::kStage);
    const int x = (kb_lo + i) * BK, y = group * p.w_rows + n0;
    tma::load_2d(sw, &wmap, x, y, &full_bar[stage]);
    if (GLU) tma::load_2d(sw + kTile / 2 * BK, &wmap, x, y + p.N, &full_bar[stage]);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tma::mbar_init(&full_bar[s], 1);
      tma::mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      tma::mbar_init(&acc_full[s], 1);
      tma::mbar_init(&acc_empty[s], EPI);
    }
    failed = 0;
    tma::fence_barrier_init();
    // without groups the weights' place is known now: they do not come from the kernel before this one
    if (p.n_groups == 0)
      for (int i = 0; i < min(STAGES, n_kb); ++i) load_w(i);
  }
  if (warp == 1) tmem_alloc<1>(&tmem_holder, kTmemCols);
  fence_before_sync();
  pdl_wait_block();
  fence_after_sync();
  const uint32_t tmem_base = tmem_holder;
  bool live = true;
  if (p.n_groups > 0) live = find_group(p.offsets, p.n_groups, p.M, NP, tok_tile, group, row0, rows);   // the same answer in every warp

  int loaded = 0;                      // warp 0: k blocks whose copies were started
  if (!live) {
    // more tiles were launched than the groups' rows fill
  } else if (warp == 0) {
    if (lane == 0) {
      for (; loaded < n_kb && !failed; ++loaded) {
        const int stage = loaded % STAGES;
        if (loaded >= STAGES && !tma::mbar_wait(&empty_bar[stage], ((loaded / STAGES) & 1) ^ 1)) {
          report(p.status, kStatusWaitTimedOut, 70, tile, loaded);
          failed = 1;
          break;
        }
        if (p.n_groups > 0 || loaded >= STAGES) load_w(loaded);
        tma::load_2d(smem + stage * S::kStage + kTile * BK, &xmap, (kb_lo + loaded) * BK, row0, &full_bar[stage]);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(kTile, NP);
      for (int i = 0; i < n_kb && !failed; ++i) {
        const int stage = i % STAGES, slot = i % SLOTS;
        if ((i >= SLOTS && !tma::mbar_wait(&acc_empty[slot], ((i / SLOTS) & 1) ^ 1)) ||
            !tma::mbar_wait(&full_bar[stage], (i / STAGES) & 1)) {
          report(p.status, kStatusWaitTimedOut, 71, tile, i);
          failed = 1;
          break;
        }
        fence_after_sync();
        const uint32_t sw = tma::smem_addr(smem + stage * S::kStage), sx = sw + kTile * BK;
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          umma(tmem_base + slot * NP, smem_desc(sw + k * 32), smem_desc(sx + k * 32), idesc, k > 0 ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        umma_commit(&acc_full[slot]);
      }
    }
    __syncwarp();
    pdl_launch_dependents();
  }
  float acc[COLS];
  const int quarter = warp & 3, row = quarter * 32 + lane;         // of the tile's weight rows
  const int col0 = EPI == 8 && warp >= 6 ? COLS : 0;               // first of this thread's rows of x
  if (live && warp >= 2) {
#pragma unroll
    for (int t = 0; t < COLS; ++t) acc[t] = 0.f;
    // the rows of scales that the tile's weight rows fall into: one, or with GLU the gates' and up to two of the ups'
    const int up0 = p.N + n0;
    const int srow = GLU ? (row < 64 ? 0 : 1 + ((up0 + row - 64) / 128 - up0 / 128)) : 0;
    const float* ws = p.ws + (size_t)group * p.ws_group;
    const int last_srow = (p.w_rows - 1) / 128;
    const int e_tid = threadIdx.x - 64;
    // this loop has barriers in it: after a wait that ran out it goes on without waiting
    for (int i = 0; i < n_kb; ++i) {
      const int slot = i % SLOTS, c = i % CH;
      if (c == 0) {                    // the next chunk of scales
        epilogue_sync(EPI * 32);
        const int n = min(CH, n_kb - i);
        for (int e = e_tid; e < n * NP; e += EPI * 32) {
          const int b = e / NP, t = e - b * NP;
          sx_s[b][t] = t < rows ? p.xs[(size_t)(kb_lo + i + b) * p.xs_ld + row0 + t] : 0.f;
        }
        for (int e = e_tid; e < n * 3; e += EPI * 32) {
          const int b = e / 3, which = e - b * 3;
          const int sr = which == 0 ? n0 / 128 : min(up0 / 128 + which - 1, last_srow);
          if (GLU || which == 0) sw_s[b][which] = ws[(size_t)sr * p.k_blocks + kb_lo + i + b];
        }
        epilogue_sync(EPI * 32);
      }
      if (!failed && !tma::mbar_wait(&acc_full[slot], (i / SLOTS) & 1)) {
        if (lane == 0) report(p.status, kStatusWaitTimedOut, 72, tile, i);
        failed = 1;
      }
      __syncwarp();
      fence_after_sync();
      const float sw = sw_s[c][srow];
      const uint32_t t_row = tmem_base + slot * NP + col0 + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
      for (int t = 0; t < COLS; t += 16) {
        uint32_t v[16];
        tmem_ld16(t_row + t, v);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 sx = *reinterpret_cast<const float4*>(&sx_s[c][col0 + t + 4 * q]);
          acc[t + 4 * q] = fmaf(__uint_as_float(v[4 * q]), sx.x * sw, acc[t + 4 * q]);
          acc[t + 4 * q + 1] = fmaf(__uint_as_float(v[4 * q + 1]), sx.y * sw, acc[t + 4 * q + 1]);
          acc[t + 4 * q + 2] = fmaf(__uint_as_float(v[4 * q + 2]), sx.z * sw, acc[t + 4 * q + 2]);
          acc[t + 4 * q + 3] = fmaf(__uint_as_float(v[4 * q + 3]), sx.w * sw, acc[t + 4 * q + 3]);
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) tma::mbar_arrive(&acc_empty[slot]);
    }
    // the operands' stages are free now: every copy has arrived and every MMA has read them
    if (p.split > 1 || GLU) {
      float* red = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int t = 0; t < COLS; ++t) red[(col0 + t) * kTile + row] = acc[t];
      if (p.split == 1) epilogue_sync(EPI * 32);
    } else if (!failed && n0 + row < p.N) {
#pragma unroll
      for (int t = 0; t < COLS; ++t) {
        if (col0 + t >= rows) break;
        const size_t at = (size_t)(row0 + col0 + t) * p.ldy + n0 + row;
        if (p.out_f32) reinterpret_cast<float*>(p.y)[at] = acc[t];
        else reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(acc[t]);
      }
    }
  }
  if (p.split > 1) cluster_sync();     // all ranks' sums lie in their shared memory
  if (live && warp >= 2 && !failed && (p.split > 1 || GLU)) {
    const uint32_t red = tma::smem_addr(smem);
    uint32_t from[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) from[q] = q < p.split ? (p.split > 1 ? map_to_rank(red, q) : red) : 0;
    auto total = [&](int t, int r) {
      float v[8], s = 0.f;
      const uint32_t off = (uint32_t)(t * kTile + r) * 4;
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = q < p.split ? ld_cluster(from[q] + off) : 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) s += v[q];
      return s;
    };
    constexpr int PER = GLU ? 64 : 128;                // outputs of a row of x
    const int e_tid = threadIdx.x - 64, r = e_tid % PER, sub = e_tid / PER, step = EPI * 32 / PER;
    for (int t = rank + p.split * sub; t < rows; t += p.split * step) {
      float v = total(t, r);
      const size_t at = (size_t)(row0 + t) * p.ldy + n0 + r;
      if (GLU) {
        float u = total(t, r + 64);
        if (n0 + r >= p.N) continue;
        if (p.row_weight) {
          const float w = p.row_weight[row0 + t];
          v *= w;
          u *= w;
        }
        if (p.glu.bias) {
          v += p.glu.bias[n0 + r];
          u += p.glu.bias[p.N + n0 + r];
        }
        reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(glu_fast(p.glu, v, u));
      } else if (n0 + r < p.N) {
        if (p.out_f32) reinterpret_cast<float*>(p.y)[at] = v;
        else reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
      }
    }
  }
  if (warp == 0 && lane == 0 && failed) {              // copies still on their way to this block's shared memory
    for (int i = max(0, loaded - STAGES); i < loaded; ++i) tma::mbar_wait(&full_bar[i % STAGES], (i / STAGES) & 1);
  }
  fence_before_sync();
  __syncthreads();
  if (p.split > 1) cluster_sync();     // nobody reads this block's sums any more
  if (warp == 1) {
    fence_after_sync();
    tmem_dealloc<1>(tmem_base, kTmemCols);
  }
}

template <int NP, bool GLU>
static int launch_np(Params p, const void* x, long long x_ld, long long x_rows, const void* w, long long w_ld, cudaStream_t stream) {
  using S = Shape<NP>;
  const int groups = p.n_groups > 0 ? p.n_groups : 1;
  const int per = GLU ? kTile / 2 : kTile;
  const long long row_tiles = (p.N + per - 1) / per;
  // with groups: every group's last tile may be partly empty, and no more tiles than rows
  p.tok_tiles = p.n_groups > 0 ? p.M / NP + (p.n_groups < p.M ? p.n_groups : p.M) : (p.M + NP - 1) / NP;
  const long long tiles = row_tiles * p.tok_tiles;
  // K is split until a thread block for every SM's two places exists
  int split = 1;
  while (split < 8 && tiles * (split + 1) <= 2 * kSMs && (split + 1) * 4 <= p.k_blocks) ++split;
  p.split = split;
  if (tiles * split > 0x7fffffffLL) return PE_ERR_UNSUPPORTED_SIZE;
  CUtensorMap wmap, xmap;
  int e = make_map(&wmap, w, p.K, (uint64_t)groups * p.w_rows, w_ld, GLU ? kTile / 2 : kTile);
  if (e == 0) e = make_map(&xmap, x, p.K, x_rows, x_ld, NP);
  if (e != 0) return e;
  static bool attr_set = false;
  if (!attr_set) {
    cudaError_t ce = cudaFuncSetAttribute(gemm_fp8_kernel<NP, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem);
    if (ce != cudaSuccess) return (int)ce;
    attr_set = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n_attr = 0;
  if (split > 1) {
    attr[n_attr].id = cudaLaunchAttributeClusterDimension;
    attr[n_attr].val.clusterDim.x = split;
    attr[n_attr].val.clusterDim.y = 1;
    attr[n_attr].val.clusterDim.z = 1;
    ++n_attr;
  }
  if (pe::pdl_enabled()) {
    attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
    ++n_attr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n_attr;
  cudaError_t ce = cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<NP, GLU>, p, wmap, xmap);
  if (ce != cudaSuccess) return (int)ce;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

}  // namespace fp8
}  // namespace pe

// x: M rows of K bytes, x_ld apart; x_scales[b * xs_ld + m]; w: n_groups (0: 1) matrices of N (kind > 0: 2 N, gates then ups) rows,
// w_ld apart; w_scales packed, [group][ceil(rows / 128)][ceil(K / 128)]; kind 0: y = the product, bfloat16 or float32; 1 to 3:
// GluEpilogue's activations, bfloat16.  offsets (n_groups + 1 ints on the device): rows offsets[g] .. offsets[g + 1] belong to
// group g, M is the most rows there can be, and rows from offsets[n_groups] on are left as they are.  row_weight[m] (or null)
// multiplies a row's sums before the activation.
extern "C" int pe_gemm_fp8(const void* x, long long x_ld, const float* x_scales, long long xs_ld, const void* w, long long w_ld,
                           const float* w_scales, void* y, long long ldy, int M, int N, int K, int out_f32, int kind, float limit,
                           float alpha, const float* bias, const float* row_weight, const int* offsets, int n_groups, int* status,
                           cudaStream_t stream) {
  using namespace pe::fp8;
  if (M < 0 || N < 0 || K < 1 || kind < 0 || kind > 3 || n_groups < 0) return PE_ERR_BAD_ARGUMENT;
  if (M == 0 || N == 0) return PE_OK;
  if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr) return PE_ERR_BAD_ARGUMENT;
  if (x_ld < K || w_ld < K || xs_ld < M || ldy < N || (kind > 0 && out_f32) || (kind == 0 && (bias || row_weight))) return PE_ERR_BAD_ARGUMENT;
  if ((n_groups > 0) != (offsets != nullptr)) return PE_ERR_BAD_ARGUMENT;
  if (((uintptr_t)x % 16) || ((uintptr_t)w % 16) || (x_ld % 16) || (w_ld % 16)) return PE_ERR_BAD_ARGUMENT;
  if (N > (1 << 28) || (long long)(n_groups > 0 ? n_groups : 1) * N > (1 << 29)) return PE_ERR_UNSUPPORTED_SIZE;
  Params p;
  p.M = M; p.N = N; p.K = K; p.k_blocks = (K + BK - 1) / BK;
  p.xs = x_scales; p.xs_ld = xs_ld; p.ws = w_scales;
  p.w_rows = kind > 0 ? 2 * N : N;
  p.ws_group = (long long)((p.w_rows + 127) / 128) * p.k_blocks;
  p.y = y; p.ldy = ldy; p.out_f32 = out_f32;
  p.offsets = offsets; p.n_groups = n_groups;
  p.glu = pe::GluEpilogue{kind, limit, alpha, bias};
  p.row_weight = row_weight;
  p.status = status;
  // rows of a tile: the least that hold them all, for groups what an average group has
  const int rows = n_groups > 0 ? (M + n_groups - 1) / n_groups : M;
#define PE_FP8_LAUNCH(NP) \
  return kind > 0 ? launch_np<NP, true>(p, x, x_ld, M, w, w_ld, stream) : launch_np<NP, false>(p, x, x_ld, M, w, w_ld, stream)
  if (rows <= 16) PE_FP8_LAUNCH(16);
  if (rows <= 32) PE_FP8_LAUNCH(32);
  if (rows <= 64) PE_FP8_LAUNCH(64);
  PE_FP8_LAUNCH(128);
#undef PE_FP8_LAUNCH
}
