// What the kernels of 8-bit floating point share: a block's scale and conversion, tensor maps of bytes, the tcgen05 instructions
// of kind::f8f6f4 and of tensor memory, cluster addresses, the tiles of rows grouped by expert.
#pragma once
#include "common.cuh"
#include "tma.cuh"
#include <cuda_fp8.h>

namespace pe {
namespace fp8 {

constexpr int kMostRows = 1 << 30;     // and features: sums of a tile's size and them stay within 32 bits
constexpr int BK = 128;        // bytes of a k block: one 128-byte swizzled row, and the features that share a scale

// ---- a block's scale and values (see quantize_fp8.cu) ------------------------------------------------------------------
// The scale's bits for the largest magnitude `a` of a block: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_bits(float a) {
  const uint32_t b = __float_as_uint(a);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 1) << 23;
}
// 1 / s, a power of two itself
__device__ __forceinline__ float inverse_of(uint32_t scale) { return __uint_as_float((254u << 23) - scale); }

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float no_infinity(float x) { return fabsf(x) == INFINITY ? __uint_as_float(0x7fffffffu) : x; }

// ---- copies and clusters -----------------------------------------------------------------------------------------------
// Rows of bytes, `ld` bytes apart, as [block][row][128]: a copy brings `kbs` blocks of `box_rows` rows as 128-byte swizzled tiles
// one behind the other.  Where the rows are not whole blocks (`whole` false) the view is [1][row][width] and a copy brings one block
// (its first coordinate is the block's first byte).  What lies beyond a row's end or the last row arrives as zeros.
inline int make_map(CUtensorMap* map, const void* base, uint64_t width, uint64_t rows, uint64_t ld, uint32_t box_rows, bool whole, uint32_t kbs) {
  tma::EncodeTiledFn fn = tma::encode_fn();
  if (fn == nullptr) return -5;
  if (((uintptr_t)base % 16) || (ld % 16) || box_rows > 256) return -2;
  cuuint64_t dims[3] = {whole ? (uint64_t)BK : width, rows, whole ? width / BK : 1};
  cuuint64_t strides[2] = {ld, (uint64_t)(whole ? BK : ld)};
  cuuint32_t box[3] = {BK, box_rows, whole ? kbs : 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -2;
}
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
      ::"r"(tma::smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(tma::smem_addr(bar)) : "memory");
}
// `kbs` blocks of `box_rows` rows from block `kb` on, into tiles one behind the other
__device__ __forceinline__ void load_blocks(char* dst, const CUtensorMap* map, int kb, int row, int kbs, int box_rows, bool whole, uint64_t* bar) {
  if (whole) {
    load_3d(dst, map, 0, row, kb, bar);
  } else {
    for (int j = 0; j < kbs; ++j) load_3d(dst + j * box_rows * BK, map, (kb + j) * BK, row, 0, bar);
  }
}

// The weights of `groups` matrices of N rows (glu: 2 N, gates then ups), `ld` bytes apart, as [group][block][half][row][128] (half: gates
// and ups): a copy brings `kbs` blocks of `box_rows` rows, of both halves with glu.  Rows beyond a half's N arrive as zeros.
inline int make_weight_map(CUtensorMap* map, const void* w, uint64_t width, uint64_t N, uint64_t ld, bool glu, uint64_t groups,
                           uint32_t box_rows, bool whole, uint32_t kbs) {
  tma::EncodeTiledFn fn = tma::encode_fn();
  if (fn == nullptr) return -5;
  if (((uintptr_t)w % 16) || (ld % 16) || box_rows > 256) return -2;
  const uint32_t halves = glu ? 2 : 1;
  cuuint64_t dims[5] = {whole ? (uint64_t)BK : width, N, halves, whole ? width / BK : 1, groups};
  cuuint64_t strides[4] = {ld, N * ld, (uint64_t)(whole ? BK : ld), halves * N * ld};
  cuuint32_t box[5] = {BK, box_rows, halves, whole ? kbs : 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(w), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -2;
}
__device__ __forceinline__ void load_5d(void* dst, const CUtensorMap* map, int x, int row, int block, int group, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];\n"
      ::"r"(tma::smem_addr(dst)), "l"(map), "r"(x), "r"(row), "r"(0), "r"(block), "r"(group), "r"(tma::smem_addr(bar)) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
// the address, in the cluster's shared window, of `addr` in the block of rank `rank`
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// the map is on its way before the first copy asks for it
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}

__device__ __forceinline__ void tmem_alloc(uint32_t* holder_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(holder_smem)), "r"(cols));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(cols));
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// arrive on the barrier once every MMA issued so far has completed
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(tma::smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// a and b, times s, added to two neighbouring sums: one instruction for both
__device__ __forceinline__ void fma2(unsigned long long& acc, uint32_t a, uint32_t b, unsigned long long s) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "r"(a), "r"(b));
  asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(acc) : "l"(v), "l"(s));
}
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 unpair(unsigned long long v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
// K-major tile, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f8f6f4: D float32 (bits 4-5: 1), A and B e4m3 (7-9 and 10-12: 0), both K-major, N >> 3 at [17,23), M >> 4 at [24,29)
__host__ __device__ constexpr uint32_t instr_desc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Which group, and which of its tiles of `np` rows, tile `j` is: all lanes of a warp take part.
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

// How many tiles of `np` rows the groups have; all lanes of a warp take part.
__device__ __forceinline__ int count_tiles(const int* offsets, int n_groups, int M, int np) {
  int tiles = 0;
  for (int g = threadIdx.x & 31; g < n_groups; g += 32) {
    const int lo = min(max(offsets[g], 0), M);
    tiles += (max(min(max(offsets[g + 1], 0), M) - lo, 0) + np - 1) / np;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
  return tiles;
}

}  // namespace fp8
}  // namespace pe
