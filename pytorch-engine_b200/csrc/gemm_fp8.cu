// Products of e4m3 operands with a scale for each block of 128, for any number of rows:
//
//   y[m, n] = sum_b sx[b, m] * sw[n / 128, b] * sum_{k in block b} x[m, k] * w[n, k]
//
// The inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4), a k block of 128 into tensor memory columns of its own;
// the outer sum is taken in float32 registers, as the columns of one block after the other are read back.  So the scales cost one
// multiply-add an output and block and no operand is ever widened.
//
// With few rows the product is a stream of the weights through the SMs, and the operands' roles are chosen for that: up to 128
// weight rows are the MMA's M dimension, NP = 16 to 128 rows of x its N dimension.  K is split over the thread blocks of a cluster;
// each finishes every split-th row of x and reads the others' sums of it through distributed shared memory, in the order of the ranks
// (no atomics: the result does not depend on scheduling).  Sending the sums instead was slower for short products (1,024 x 4,096, 8
// rows: 4.8 against 4.0 us) and 3 % faster for long ones, whose blocks need not wait to be read.
//
// Roles: warp 0 copies the weights and warp 2 the rows (TMA; a thread starts a copy only every 150 ns or so), warp 1 allocates
// tensor memory and issues the MMAs, the other warps are the epilogue: a thread owns a weight row (its tensor memory lane) and NP,
// for NP = 128 half of them, sums.  A stage is KBS k blocks: a commit costs about 0.11 us that the MMAs behind it wait for.
// The first stages' weights are asked for before the kernel waits for its predecessor in the stream, and its own successor may
// start at once: with half an SM's shared memory a block, the next product's weights are on their way while this one still works.
//
// GLU: a tile is up to 64 gate rows and the up rows that belong to them, and y = act(gate, up), rounded to bfloat16.
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
  bool whole;                          // K is whole blocks
  const float* xs; long long xs_ld;    // [k_blocks][xs_ld]
  const __nv_bfloat16* x; long long x_ld;   // RAW
  const float* ws; long long ws_group; // per group [ceil(rows / 128)][k_blocks]
  int w_rows;                          // weight rows of a group: N, or 2 N with GLU
  void* y; long long ldy; int out_f32;
  int tile_rows, tok_tiles, split;     // tile_rows: weight rows of a tile (GLU: gate rows, and as many ups)
  const int* offsets; int n_groups;    // null, 0: one group of M rows
  GluEpilogue glu; const float* row_weight;
  int* status;
};

constexpr int kTile = 128;             // weight rows of a full tile
constexpr int kRoles = 3;              // warps before the epilogue's

template <int NP> struct Shape {
  static constexpr int kKbs = 2;           // k blocks of a stage
  static constexpr int kStages = NP == 16 ? 3 : 2;
  static constexpr int kPerSm = NP == 128 ? 1 : 2;         // thread blocks an SM holds
  static constexpr int kStage = kKbs * (kTile * BK + NP * BK);
  static constexpr int kEpiWarps = NP == 128 ? 8 : 4;
  static constexpr int kCols = NP / (kEpiWarps / 4);       // sums of a thread
  static constexpr int kThreads = 32 * (kRoles + kEpiWarps);
  static constexpr int kChunk = NP == 128 ? 16 : 32;       // k blocks whose scales lie in shared memory
  static constexpr int kTmem = kStages * kKbs * NP <= 128 ? 128 : kStages * kKbs * NP <= 256 ? 256 : 512;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage;
};

__device__ __forceinline__ void epilogue_sync(int threads) { asm volatile("bar.sync 1, %0;\n" ::"r"(threads) : "memory"); }

// The bfloat16 rows of a stage on their way into it (RAW): sixteen lanes a row and block, eight features a lane.
struct RawRows {
  uint4 v[4];
};

template <int NP, bool GLU, bool RAW>
__global__ void __launch_bounds__(Shape<NP>::kThreads, Shape<NP>::kPerSm)
gemm_fp8_kernel(Params p, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
  using S = Shape<NP>;
  constexpr int STAGES = S::kStages, KBS = S::kKbs, EPI = S::kEpiWarps, COLS = S::kCols, CH = S::kChunk, ET = 32 * EPI;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t full_bar[STAGES], done_bar[STAGES], read_bar[STAGES], raw_bar[RAW ? STAGES : 1];
  __shared__ __align__(16) float sx_s[CH][NP];
  __shared__ float sw_s[4][CH];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int failed;
  __shared__ int started[2], issued;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? (int)cluster_rank() : 0;
  const int tile = (int)blockIdx.x / p.split;
  const int row_tile = tile / p.tok_tiles, tok_tile = tile - row_tile * p.tok_tiles;
  const int R = p.tile_rows, n0 = row_tile * R, n_out = min(R, p.N - n0), tile_bytes = (GLU ? 2 : 1) * R * BK;
  const int kb_lo = (int)((long long)p.k_blocks * rank / p.split), kb_hi = (int)((long long)p.k_blocks * (rank + 1) / p.split);
  const int n_kb = kb_hi - kb_lo, n_st = (n_kb + KBS - 1) / KBS;

  int group = 0, row0 = tok_tile * NP, rows = min(NP, p.M - row0);
  auto load_w = [&](int i) {           // the weights of this block's stage i (blocks beyond n_kb are loaded and not used)
    const int stage = i % STAGES;
    char* sw = smem + stage * S::kStage;
    tma::mbar_expect_tx(&full_bar[stage], KBS * tile_bytes);
    const int kb = kb_lo + i * KBS;
    if (p.whole) {
      load_5d(sw, &wmap, 0, n0, kb, group, &full_bar[stage]);
    } else {
      for (int j = 0; j < KBS; ++j) load_5d(sw + j * tile_bytes, &wmap, (kb + j) * BK, n0, 0, group, &full_bar[stage]);
    }
  };
  const int e_tid = (int)threadIdx.x - 32 * kRoles;
  // The rows of scales that the tile's weight rows fall into: up to two, and with GLU two more for the ups.
  const int up0 = p.N + n0;
  auto load_sw = [&](int kb0) {        // of the chunk of blocks from kb0 on
    static_assert(4 * CH <= ET, "a scale a thread");
    const int which = e_tid / CH, b = e_tid % CH;
    if (which < (GLU ? 4 : 2) && kb0 + b < n_kb) {
      const int sr = min((which < 2 ? n0 : up0) / 128 + (which & 1), (p.w_rows - 1) / 128);
      sw_s[which][b] = p.ws[(size_t)group * p.ws_group + (size_t)sr * p.k_blocks + kb_lo + kb0 + b];
    }
  };
  auto load_sx = [&](int kb0) {
    float v[CH * NP / ET];
#pragma unroll
    for (int q = 0; q < CH * NP / ET; ++q) {
      const int e = q * ET + e_tid, b = e / NP, t = e % NP;
      v[q] = kb0 + b < n_kb && t < rows ? p.xs[(size_t)(kb_lo + kb0 + b) * p.xs_ld + row0 + t] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < CH * NP / ET; ++q) (&sx_s[0][0])[q * ET + e_tid] = v[q];
  };
  if (threadIdx.x == 64 && !RAW) prefetch_map(&xmap);
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tma::mbar_init(&full_bar[s], RAW ? 1 : 2);          // the producers: the weights', and the rows'
      // the epilogue's warps, when they have converted a stage's rows: each has then read what the MMAs of the stage before left
      if (RAW) tma::mbar_init(&raw_bar[s], EPI);
      tma::mbar_init(&done_bar[s], 1);    // the commit behind a stage's MMAs
      tma::mbar_init(&read_bar[s], EPI);  // the epilogue's warps
    }
    failed = issued = 0;
    tma::fence_barrier_init();
    // without groups the weights' place is known now: they do not come from the kernel before this one
    if (p.n_groups == 0)
      for (int i = 0; i < min(STAGES, n_st); ++i) load_w(i);
  }
  if (warp == 1) tmem_alloc(&tmem_holder, S::kTmem);
  if (warp >= kRoles && p.n_groups == 0) load_sw(0);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  // The kernel before this one: whoever reads what it wrote, or writes what it may still read, waits for it to have completed.
  // Weights and MMAs need not (with groups they do: the offsets come from it).
  if (warp >= 2 || p.n_groups > 0) pdl_wait();
  if (warp == 2) pdl_launch_dependents();
  const uint32_t tmem_base = tmem_holder;
  bool live = true;
  if (p.n_groups > 0) live = find_group(p.offsets, p.n_groups, p.M, NP, tok_tile, group, row0, rows);   // the same answer in every warp

  int loaded = 0;                      // warps 0 and 2: stages whose copies were started
  if (!live) {
    // more tiles were launched than the groups' rows fill
  } else if (warp == 0 || (warp == 2 && !RAW)) {
    if (lane == 0) {
      for (; loaded < n_st && !failed; ++loaded) {
        const int stage = loaded % STAGES;
        if (loaded >= STAGES && !tma::mbar_wait(&done_bar[stage], ((loaded / STAGES) & 1) ^ 1)) {
          report(p.status, kStatusWaitTimedOut, 70, tile, loaded);
          failed = 1;
          break;
        }
        if (warp == 0) {
          if (p.n_groups > 0 || loaded >= STAGES) load_w(loaded);
        } else {
          tma::mbar_expect_tx(&full_bar[stage], KBS * NP * BK);
          load_blocks(smem + stage * S::kStage + KBS * kTile * BK, &xmap, kb_lo + loaded * KBS, row0, KBS, NP, p.whole, &full_bar[stage]);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(kTile, NP);
      const uint32_t base = tma::smem_addr(smem);
      // Unrolled over the stages: an MMA's descriptors are registers that it reads when it starts, and a loop that writes the same
      // ones again waits for that (a stage of two blocks of 16 rows took 1,290 cycles, of which the MMAs are some 500).
      bool ok = true;
      for (int i0 = 0; i0 < n_st && ok; i0 += STAGES) {
#pragma unroll
        for (int stage = 0; stage < STAGES; ++stage) {
          const int i = i0 + stage, n = n_kb - i * KBS;
          if (n <= 0) break;
          const uint32_t parity = (i / STAGES) & 1;
          ok = tma::mbar_wait_both(RAW ? &raw_bar[RAW ? stage : 0] : &read_bar[stage], RAW ? parity : parity ^ 1, &full_bar[stage], parity);
          if (!ok) {
            report(p.status, kStatusWaitTimedOut, 71, tile, i);
            failed = 1;
            break;
          }
          fence_after_sync();
          const uint32_t sw = base + stage * S::kStage, sx = sw + KBS * kTile * BK;
#pragma unroll
          for (int j = 0; j < KBS; ++j) {
            if (j >= n) break;
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma(tmem_base + (stage * KBS + j) * NP, smem_desc(sw + j * tile_bytes + k * 32), smem_desc(sx + j * NP * BK + k * 32), idesc,
                   k > 0 ? 1u : 0u);
          }
          umma_commit(&done_bar[stage]);
          issued = i + 1;
        }
      }
    }
    __syncwarp();
  }
  // RAW: pass q of this warp is row t of x and block j of the stage; rows that are not there are left out.
  const int raw_lane = 8 * (lane & 15);
  auto raw_at = [&](int q, int& j, int& t) {
    const int item = q * 8 + (warp - kRoles) * 2 + (lane >> 4);
    j = item & (KBS - 1);
    t = item / KBS;
  };
  auto raw_load = [&](int i, RawRows& r) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      int j, t;
      raw_at(q, j, t);
      const int at = (kb_lo + i * KBS + j) * BK + raw_lane;
      r.v[q] = make_uint4(0, 0, 0, 0);
      if (t < rows && i * KBS + j < n_kb && at < p.K) {
        const __nv_bfloat16* x = p.x + (size_t)(row0 + t) * p.x_ld + at;
        if (at + 8 <= p.K) {
          r.v[q] = *reinterpret_cast<const uint4*>(x);
        } else {
          alignas(16) __nv_bfloat16 e[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) e[k] = at + k < p.K ? x[k] : __float2bfloat16_rn(0.f);
          r.v[q] = *reinterpret_cast<const uint4*>(e);
        }
      }
    }
  };
  auto raw_store = [&](int i, const RawRows& r) {
    const int stage = i % STAGES;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      int j, t;
      raw_at(q, j, t);
      if (__all_sync(0xffffffffu, t >= rows)) break;
      float v[8], top = 0.f;
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r.v[q]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 e = __bfloat1622float2(h[k]);
        v[2 * k] = e.x;
        v[2 * k + 1] = e.y;
        top = fmaxf(top, fmaxf(fabsf(e.x), fabsf(e.y)));
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const uint32_t scale = scale_bits(top);
      const float by = inverse_of(scale);
      if (top == INFINITY) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = no_infinity(v[k]);
      }
      char* to = smem + stage * S::kStage + KBS * kTile * BK + (j * NP + t) * BK;
      *reinterpret_cast<uint2*>(to + ((((raw_lane >> 4) ^ (t & 7)) << 4) | (raw_lane & 8))) =
          make_uint2(pack4(v[0] * by, v[1] * by, v[2] * by, v[3] * by), pack4(v[4] * by, v[5] * by, v[6] * by, v[7] * by));
      if ((lane & 15) == 0) sx_s[(i * KBS + j) % CH][t] = __uint_as_float(scale);
    }
    tma::fence_proxy_async();          // the MMAs read what was written here
    __syncwarp();
    if (lane == 0) tma::mbar_arrive(&raw_bar[RAW ? stage : 0]);
  };
  float acc[COLS];
  const int quarter = warp & 3, row = quarter * 32 + lane;         // of the tile's weight rows: with GLU R gates, then R ups
  const int col0 = EPI == 8 && warp >= kRoles + 4 ? COLS : 0;      // first of this thread's rows of x
  // where the operands' stages were, when every copy has arrived and every MMA has read them: [row of x][weight row]
  float* sums = reinterpret_cast<float*>(smem);
  if (live && warp >= kRoles) {
#pragma unroll
    for (int t = 0; t < COLS; ++t) acc[t] = 0.f;
    const bool up = GLU && row >= R;
    const int srow = up ? 2 + ((up0 + row - R) / 128 - up0 / 128) : (n0 + row) / 128 - n0 / 128;
    const bool used = row < (GLU ? 2 : 1) * R;
    RawRows raw[RAW ? STAGES : 1];
    if (RAW) {
#pragma unroll
      for (int i = 0; i < STAGES; ++i) raw_load(i, raw[i]);
#pragma unroll
      for (int i = 0; i < STAGES; ++i)
        if (i < n_st) raw_store(i, raw[i]);
    }
    // this loop has barriers in it: after a wait that ran out it goes on without waiting
    for (int i = 0; i < n_st; ++i) {
      const int stage = i % STAGES, kb0 = i * KBS;
      if (kb0 % CH == 0) {             // the next chunk of scales
        if (i > 0) epilogue_sync(ET);  // everybody is done with the last one
        if (i > 0 || p.n_groups > 0) load_sw(kb0);
        if (!RAW) load_sx(kb0);
        epilogue_sync(ET);
      }
      if (RAW && i + STAGES < n_st) raw_load(i + STAGES, raw[0]);
      if (!failed && !tma::mbar_wait(&done_bar[stage], (i / STAGES) & 1)) {
        if (lane == 0) report(p.status, kStatusWaitTimedOut, 72, tile, i);
        failed = 1;
      }
      if (RAW && !failed) tma::mbar_wait(&raw_bar[RAW ? stage : 0], (i / STAGES) & 1);    // long complete: the other warps' scales are seen
      __syncwarp();
      fence_after_sync();
#pragma unroll
      for (int j = 0; j < KBS; ++j) {
        if (kb0 + j >= n_kb) break;
        const int c = (kb0 + j) % CH;
        const float sw = used ? sw_s[srow][c] : 0.f;
        const uint32_t t_row = tmem_base + (stage * KBS + j) * NP + col0 + ((uint32_t)(quarter * 32) << 16);
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
      }
      fence_before_sync();
      __syncwarp();
      if (!RAW && lane == 0) tma::mbar_arrive(&read_bar[stage]);
      if (RAW && i + STAGES < n_st) raw_store(i + STAGES, raw[0]);
    }
    if (p.split > 1 || GLU) {
#pragma unroll
      for (int t = 0; t < COLS; ++t)
        if (col0 + t < rows) sums[(col0 + t) * kTile + row] = acc[t];
      if (p.split == 1) epilogue_sync(ET);
    } else if (p.split == 1 && !failed && row < n_out) {
#pragma unroll
      for (int t = 0; t < COLS; ++t) {
        if (col0 + t >= rows) break;
        const size_t at = (size_t)(row0 + col0 + t) * p.ldy + n0 + row;
        if (p.out_f32) reinterpret_cast<float*>(p.y)[at] = acc[t];
        else reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(acc[t]);
      }
    }
  }
  __syncwarp();
  if (p.split > 1) cluster_sync();     // all ranks' sums lie in their shared memory
  if (live && warp >= kRoles && !failed && (p.split > 1 || GLU)) {
    // row t of x is finished by rank t % split, four neighbouring outputs a thread and turn
    const int quads = (n_out + 3) / 4, mine = rows > rank ? (rows - rank + p.split - 1) / p.split : 0;
    const int es = p.out_f32 ? 4 : 2;
    const bool vec = n_out % 4 == 0 && ((uintptr_t)p.y % 16) == 0 && (p.ldy * es) % 16 == 0;
    auto finish = [&](auto total) {                    // total(at): the sums of four outputs over the ranks
      for (int e = e_tid; e < mine * quads; e += ET) {
        const int i = e / quads, r = (e - i * quads) * 4, t = rank + p.split * i;
        const float4 g4 = total(t * kTile + r);
        float v[4] = {g4.x, g4.y, g4.z, g4.w};
        if (GLU) {
          const float4 u4 = total(t * kTile + R + r);
          float u[4] = {u4.x, u4.y, u4.z, u4.w};
          const float w = p.row_weight ? p.row_weight[row0 + t] : 1.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] *= w;
            u[k] *= w;
            if (p.glu.bias && r + k < n_out) {
              v[k] += p.glu.bias[n0 + r + k];
              u[k] += p.glu.bias[p.N + n0 + r + k];
            }
            v[k] = glu_fast(p.glu, v[k], u[k]);
          }
        }
        const size_t at = (size_t)(row0 + t) * p.ldy + n0 + r;
        if (p.out_f32) {
          float* y = reinterpret_cast<float*>(p.y) + at;
          if (vec) *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
          else
            for (int k = 0; k < 4 && r + k < n_out; ++k) y[k] = v[k];
        } else {
          __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(p.y) + at;
          const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
          if (vec) {
            *reinterpret_cast<uint2*>(y) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
          } else {
            const __nv_bfloat16 o[4] = {a.x, a.y, b.x, b.y};
            for (int k = 0; k < 4 && r + k < n_out; ++k) y[k] = o[k];
          }
        }
      }
    };
    if (p.split == 1) {
      finish([&](int at) { return *reinterpret_cast<const float4*>(sums + at); });
    } else {
      const uint32_t base = tma::smem_addr(sums);
      uint32_t from[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) from[q] = q < p.split ? map_to_rank(base, q) : base;
      finish([&](int at) {
        float4 o[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < p.split) o[q] = ld_cluster(from[q] + at * 4);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < p.split) {
            v.x += o[q].x; v.y += o[q].y; v.z += o[q].z; v.w += o[q].w;
          }
        return v;
      });
    }
  }
  if (lane == 0 && (warp == 0 || warp == 2)) started[warp >> 1] = max(loaded, warp == 0 && p.n_groups == 0 ? min(STAGES, n_st) : 0);
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    if (failed && lane == 0) {         // MMAs that still read this block's shared memory, copies still on their way to it
      for (int i = max(0, issued - STAGES); i < issued; ++i) tma::mbar_wait(&done_bar[i % STAGES], (i / STAGES) & 1);
      const int last = RAW ? started[0] : max(started[0], started[1]);
      for (int i = max(0, last - STAGES); i < last; ++i) {
        if (!RAW && (i >= started[0] || i >= started[1])) tma::mbar_arrive(&full_bar[i % STAGES]);     // for the operand that was not asked for
        tma::mbar_wait(&full_bar[i % STAGES], (i / STAGES) & 1);
      }
    }
    __syncwarp();
    fence_after_sync();
    tmem_dealloc(tmem_base, S::kTmem);
  }
  __syncwarp();
  if (p.split > 1) cluster_sync();     // nobody reads this block's sums any more
}

// How a product is cut: weight rows of a tile, token tiles, thread blocks that share K.
struct Cut {
  int rows, tok_tiles, split;
  long long blocks;
  int waves_blocks;                    // k blocks one after the other on an SM, over all waves
};
static Cut cut_of(int M, int N, int k_blocks, int n_groups, int np, bool glu) {
  const int places = (np == 128 ? 1 : 2) * kSMs, full = glu ? kTile / 2 : kTile;
  Cut c;
  // with groups: every group's last tile may be partly empty, and no more tiles than rows
  c.tok_tiles = n_groups > 0 ? M / np + (n_groups < M ? n_groups : M) : (M + np - 1) / np;
  auto tiles_of = [&](int rows) { return (long long)((N + rows - 1) / rows) * c.tok_tiles; };
  c.rows = full;
  c.split = 1;
  // Clusters of 2, 4 or 8: those of 3 or 6 do not pack into the chip (6,144 x 4,096, 8 rows: 7.5 us with 4, 9.0 with 3, 12.8 with 6).
  while (c.split < 8 && tiles_of(full) * c.split * 2 <= places && c.split * 2 * 2 <= k_blocks) c.split *= 2;
  // Where the tiles fill the places once and not to the end, smaller ones spread the weights evenly (12,288 gates of 4,096, 8 rows:
  // 19.1 us with 48 rows a tile, 20.8 with 64).
  if (c.split == 1)
    while (c.rows > full / 2 && tiles_of(c.rows - 8) <= places) c.rows -= 8;
  c.blocks = tiles_of(c.rows) * c.split;
  c.waves_blocks = (int)((c.blocks + kSMs - 1) / kSMs) * ((k_blocks + c.split - 1) / c.split);
  return c;
}

template <int NP, bool GLU, bool RAW = false>
static int launch_np(Params p, const void* x, long long x_ld, long long x_rows, const void* w, long long w_ld, cudaStream_t stream) {
  using S = Shape<NP>;
  const int groups = p.n_groups > 0 ? p.n_groups : 1;
  const Cut c = cut_of(p.M, p.N, p.k_blocks, p.n_groups, NP, GLU);
  p.tile_rows = c.rows;
  p.tok_tiles = c.tok_tiles;
  const int split = p.split = c.split;
  if (c.blocks > 0x7fffffffLL) return PE_ERR_UNSUPPORTED_SIZE;
  CUtensorMap wmap, xmap;
  int e = make_weight_map(&wmap, w, p.K, p.N, w_ld, GLU, groups, p.tile_rows, p.whole, S::kKbs);
  if (e == 0 && !RAW) e = make_map(&xmap, x, p.K, x_rows, x_ld, NP, p.whole, S::kKbs);
  if (e != 0) return e;
  if (RAW) xmap = wmap;                // not used
  static bool asked[kDevices] = {};
  e = allow_smem_once(gemm_fp8_kernel<NP, GLU, RAW>, S::kSmem, asked);
  if (e != 0) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c.blocks);
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
  cudaError_t ce = cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<NP, GLU, RAW>, p, wmap, xmap);
  if (ce != cudaSuccess) return (int)ce;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

}  // namespace fp8
}  // namespace pe

// Whether a product runs in tiles of 128 x 256 (gemm_fp8_many.cu): where they take no longer.  A block of K takes an SM 0.60 us there
// and 0.55 us in this file's tiles of 128 x 128, which can share K out (4,096 x 6,144, both files' times in us: 128 rows 24.4 and 15.6,
// 384 rows 24.8 and 21.7, 512 rows 26.2 and 42.9; 12,288 x 4,096: 512 rows 60.1 and 56.0, 700 rows 62.9 and 107.9).  Of groups half are
// taken to fill their last tile and half not to have it.
extern "C" int pe_gemm_fp8_many_takes(int M, int N, int K, int kind, int n_groups) {
  if (N < 1 || K < 1 || (kind > 0 && N % 128)) return 0;
  if ((n_groups > 0 ? (M + n_groups - 1) / n_groups : M) <= 64) return 0;
  const int k_blocks = (K + pe::fp8::BK - 1) / pe::fp8::BK;
  const long long m_tiles = (M + 127LL) / 128 + n_groups / 2, tiles = m_tiles * (kind > 0 ? N / 128 : (N + 255) / 256);
  const pe::fp8::Cut c = pe::fp8::cut_of((int)(m_tiles * 128), N, k_blocks, 0, 128, kind > 0);
  return 11 * ((tiles + pe::kSMs - 1) / pe::kSMs) * k_blocks <= 10LL * c.waves_blocks ? 1 : 0;
}

// Whether a product whose scales are powers of two runs in pairs of SMs (gemm_fp8_pair.cu): where they take less.  A block of K takes a
// pair 0.43 us for 256 x 256, and its launch 1.5 us more than the others' (us, other tiles : pairs; 4,096 x 6,144: 128 rows 15.4 : 17.3,
// 192 rows 21.9 : 17.3, 1,024 rows 43.4 : 31.3; 12,288 x 4,096: 256 rows 33.0 : 43.4, 320 rows 55.6 : 43.0; 4,096 x 2 * 12,288 gated:
// 256 rows 48.6 : 36.9, 320 rows 47.8 : 48.0, 2,048 rows 233 : 160).  Of groups half are taken to fill their last tile and half not to
// have it.
extern "C" int pe_gemm_fp8_pair_takes(int M, int N, int K, int kind, int n_groups) {
  if (N < 1 || K < 1 || M < 1 || M > pe::fp8::kMostRows || K > pe::fp8::kMostRows || (kind > 0 && N % 128)) return 0;
  if ((n_groups > 0 ? (M + n_groups - 1) / n_groups : M) <= 64) return 0;
  const int many = pe_gemm_fp8_many_takes(M, N, K, kind, n_groups);
  const long long k_blocks = (K + pe::fp8::BK - 1) / pe::fp8::BK, n_tiles = kind > 0 ? N / 128 : (N + 255) / 256;
  const long long pairs = (((M + 255LL) / 256 + n_groups / 2) * n_tiles + pe::kSMs / 2 - 1) / (pe::kSMs / 2);
  const long long m_tiles = (M + 127LL) / 128 + n_groups / 2;
  const long long others = many ? 60 * ((m_tiles * n_tiles + pe::kSMs - 1) / pe::kSMs) * k_blocks
                                : 55 * pe::fp8::cut_of((int)(m_tiles * 128), N, (int)k_blocks, 0, 128, kind > 0).waves_blocks;
  return 43 * pairs * k_blocks + 150 <= others ? 1 : 0;
}

// Whether bfloat16 rows are quantised inside the product: up to 16 rows (of an average group).
static bool takes_raw(int M, int n_groups) { return (n_groups > 0 ? (M + n_groups - 1) / n_groups : M) <= 16; }

// raw: x is bfloat16, x_ld in elements, x_scales unused.
static int product(bool raw, const void* x, long long x_ld, const float* x_scales, long long xs_ld, const void* w, long long w_ld,
                   const float* w_scales, void* y, long long ldy, int M, int N, int K, int out_f32, int kind, float limit, float alpha,
                   const float* bias, const float* row_weight, const int* offsets, int n_groups, int* status, cudaStream_t stream) {
  using namespace pe::fp8;
  if (M < 0 || N < 0 || K < 1 || kind < 0 || kind > 3 || n_groups < 0) return PE_ERR_BAD_ARGUMENT;
  if (M == 0 || N == 0) return PE_OK;
  if (M > kMostRows || K > kMostRows) return PE_ERR_UNSUPPORTED_SIZE;
  if (x == nullptr || (!raw && x_scales == nullptr) || w == nullptr || w_scales == nullptr || y == nullptr) return PE_ERR_BAD_ARGUMENT;
  if (x_ld < K || w_ld < K || (!raw && xs_ld < M) || ldy < N || (kind > 0 && out_f32) || (kind == 0 && (bias || row_weight)))
    return PE_ERR_BAD_ARGUMENT;
  if ((n_groups > 0) != (offsets != nullptr)) return PE_ERR_BAD_ARGUMENT;
  if (((uintptr_t)x % 16) || ((uintptr_t)w % 16) || (x_ld * (raw ? 2 : 1)) % 16 || (w_ld % 16)) return PE_ERR_BAD_ARGUMENT;
  if (N > (1 << 28) || (long long)(n_groups > 0 ? n_groups : 1) * N > (1 << 29)) return PE_ERR_UNSUPPORTED_SIZE;
  const int rows = n_groups > 0 ? (M + n_groups - 1) / n_groups : M;     // of an average group
  const int k_blocks = (K + BK - 1) / BK;
  if (!raw && (n_groups > 0 || !row_weight) && pe_gemm_fp8_many_takes(M, N, K, kind, n_groups))
    return pe_gemm_fp8_many(x, x_ld, x_scales, xs_ld, w, w_ld, w_scales, y, ldy, nullptr, 0, M, N, K, out_f32, kind, limit, alpha, bias,
                            row_weight, offsets, n_groups, status, stream);
  Params p;
  p.M = M; p.N = N; p.K = K; p.k_blocks = k_blocks; p.whole = K % BK == 0;
  p.xs = x_scales; p.xs_ld = xs_ld; p.ws = w_scales;
  p.x = (const __nv_bfloat16*)x; p.x_ld = x_ld;
  p.w_rows = kind > 0 ? 2 * N : N;
  p.ws_group = (long long)((p.w_rows + 127) / 128) * p.k_blocks;
  p.y = y; p.ldy = ldy; p.out_f32 = out_f32;
  p.offsets = offsets; p.n_groups = n_groups;
  p.glu = pe::GluEpilogue{kind, limit, alpha, bias};
  p.row_weight = row_weight;
  p.status = status;
  if (raw) {
    if (rows > 16) return PE_ERR_UNSUPPORTED_SIZE;
    return kind > 0 ? launch_np<16, true, true>(p, x, x_ld, M, w, w_ld, stream) : launch_np<16, false, true>(p, x, x_ld, M, w, w_ld, stream);
  }
#define PE_FP8_LAUNCH(NP) \
  return kind > 0 ? launch_np<NP, true>(p, x, x_ld, M, w, w_ld, stream) : launch_np<NP, false>(p, x, x_ld, M, w, w_ld, stream)
  // the least tile of rows that holds them all, for groups what an average group has
  if (rows <= 16) PE_FP8_LAUNCH(16);
  if (rows <= 32) PE_FP8_LAUNCH(32);
  if (rows <= 64) PE_FP8_LAUNCH(64);
  PE_FP8_LAUNCH(128);
#undef PE_FP8_LAUNCH
}

// x: M rows of K bytes, x_ld apart; x_scales[b * xs_ld + m]; w: n_groups (0: 1) matrices of N (kind > 0: 2 N, gates then ups) rows,
// w_ld apart; w_scales packed, [group][ceil(rows / 128)][ceil(K / 128)]; kind 0: y = the product, bfloat16 or float32; 1 to 3:
// GluEpilogue's activations, bfloat16.  offsets (n_groups + 1 ints on the device): rows offsets[g] .. offsets[g + 1] belong to
// group g, M is the most rows there can be, and rows from offsets[n_groups] on are left as they are.  row_weight[m] (or null)
// multiplies a row's sums before the activation.
extern "C" int pe_gemm_fp8(const void* x, long long x_ld, const float* x_scales, long long xs_ld, const void* w, long long w_ld,
                           const float* w_scales, void* y, long long ldy, int M, int N, int K, int out_f32, int kind, float limit,
                           float alpha, const float* bias, const float* row_weight, const int* offsets, int n_groups, int* status,
                           cudaStream_t stream) {
  return product(false, x, x_ld, x_scales, xs_ld, w, w_ld, w_scales, y, ldy, M, N, K, out_f32, kind, limit, alpha, bias, row_weight,
                 offsets, n_groups, status, stream);
}

// pe_gemm_fp8 of rows in bfloat16 or float32, which are quantised first (pe_quantize_rows_fp8's dtype, x, x_ld, row_map, x_rows; with
// groups only the rows below offsets[n_groups]): into `scratch` (16-byte aligned), M rows of ceil(K / 16) * 16 bytes and behind them
// ceil(K / 128) * M floats; or, with scratch null, inside the product: bfloat16 rows on 16-byte boundaries, up to 16 (of an average
// group), no row map.
extern "C" int pe_linear_fp8(int dtype, const void* x, long long x_ld, const int* row_map, int x_rows, void* scratch, const void* w,
                             long long w_ld, const float* w_scales, void* y, long long ldy, int M, int N, int K, int out_f32, int kind,
                             float limit, float alpha, const float* bias, const float* row_weight, const int* offsets, int n_groups,
                             int* status, cudaStream_t stream) {
  if (M < 0 || N < 0 || K < 1 || n_groups < 0) return PE_ERR_BAD_ARGUMENT;
  if (M == 0 || N == 0) return PE_OK;
  if (scratch == nullptr) {
    if (dtype != PE_BF16 || row_map != nullptr || !takes_raw(M, n_groups)) return PE_ERR_BAD_ARGUMENT;
    return product(true, x, x_ld, nullptr, 0, w, w_ld, w_scales, y, ldy, M, N, K, out_f32, kind, limit, alpha, bias, row_weight, offsets,
                   n_groups, status, stream);
  }
  const long long ld = ((long long)K + 15) / 16 * 16;
  float* scales = reinterpret_cast<float*>(reinterpret_cast<char*>(scratch) + ld * M);
  const int e = pe_quantize_rows_fp8(dtype, x, x_ld, row_map, n_groups > 0 ? offsets + n_groups : nullptr, scratch, ld, scales, M, M, K,
                                     x_rows, status, stream);
  if (e != PE_OK) return e;
  return pe_gemm_fp8(scratch, ld, scales, M, w, w_ld, w_scales, y, ldy, M, N, K, out_f32, kind, limit, alpha, bias, row_weight, offsets,
                     n_groups, status, stream);
}
