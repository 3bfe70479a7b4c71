// How a tile of 128 rows of x and 256 weight rows of an 8-bit product leaves the registers of its epilogue (gemm_fp8_many.cu,
// gemm_fp8_pair.cu): eight warps, a thread with one row and 128 sums: neighbouring columns, or 64 gates and their 64 ups.
#pragma once
#include "api.h"
#include "fp8.cuh"

namespace pe {
namespace fp8 {

constexpr int kOutRow = 80, kOutWarp = 32 * kOutRow;      // what an epilogue warp has for 64 bytes of each of its rows on their way out

enum Mode { kBf16 = 0, kF32 = 1, kGlu = 2, kGluFp8 = 3 };

struct Output {
  int N;                                // output columns
  void* y; long long ldy;
  float* ys; long long ys_ld;           // kGluFp8: scales of the outputs, [block][row]
  const float* row_weight;
  GluEpilogue glu;
};

// 64 bytes of each of a warp's 32 rows (a row a lane) to rows `row_bytes` apart, of which `n` are there: through shared memory, so that
// four lanes store a row (a lane that stored its own row touched 32 lines with each instruction).  Rows of `buf` are 80 bytes, so that
// the 16-byte accesses of eight lanes to eight rows fall into different banks.
__device__ __forceinline__ void put64(char* buf, int lane, const uint4 (&v)[4], char* to, long long row_bytes, int n) {
  uint4* mine = reinterpret_cast<uint4*>(buf + lane * kOutRow);
#pragma unroll
  for (int j = 0; j < 4; ++j) mine[j] = v[j];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2), part = lane & 3;
    if (r < n) *reinterpret_cast<uint4*>(to + (size_t)r * row_bytes + part * 16) = *reinterpret_cast<const uint4*>(buf + r * kOutRow + part * 16);
  }
  __syncwarp();
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The tile's rows from m0 on, of which `rows` are there (none are written with `failed`), columns n0 on; h: which half of the columns.
// All eight warps take part (a fused conversion has barriers in it).
template <int MODE, bool GROUPS>
__device__ __forceinline__ void finish_tile(const Output& p, float (&acc)[128], int m0, int rows, int n0, int h, int quarter, int lane, bool failed,
                                            char* out_buf, float (&top_s)[2][128]) {
  constexpr bool GLU = MODE == kGlu || MODE == kGluFp8;
  const int r_tile = quarter * 32 + lane, row = m0 + r_tile, c0 = GLU ? h * 64 : h * 128;
  const bool live = r_tile < rows;
  // this warp's first row of y, and how many of its rows are there
  const int es = MODE == kF32 ? 4 : MODE == kGluFp8 ? 1 : 2, n_rows = failed ? 0 : rows - quarter * 32;
  const long long row_bytes = p.ldy * es;
  char* first = reinterpret_cast<char*>(p.y) + (size_t)(m0 + quarter * 32) * row_bytes + (size_t)(n0 + c0) * es;
  const bool vec = ((uintptr_t)p.y % 16) == 0 && row_bytes % 16 == 0;
  if constexpr (!GLU) {
    const int left = p.N - (n0 + c0);
    constexpr int PER = 64 / (MODE == kF32 ? 4 : 2);        // outputs of a row that go together
#pragma unroll
    for (int j = 0; j < 128; j += PER) {
      if (vec && j + PER <= left) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (MODE == kF32)
            v[k] = make_uint4(__float_as_uint(acc[j + 4 * k]), __float_as_uint(acc[j + 4 * k + 1]), __float_as_uint(acc[j + 4 * k + 2]),
                              __float_as_uint(acc[j + 4 * k + 3]));
          else
            v[k] = make_uint4(pack2(acc[(j + 8 * k) & 127], acc[(j + 8 * k + 1) & 127]), pack2(acc[(j + 8 * k + 2) & 127], acc[(j + 8 * k + 3) & 127]),
                              pack2(acc[(j + 8 * k + 4) & 127], acc[(j + 8 * k + 5) & 127]), pack2(acc[(j + 8 * k + 6) & 127], acc[(j + 8 * k + 7) & 127]));
        }
        put64(out_buf, lane, v, first + j * es, row_bytes, n_rows);
      } else if (lane < n_rows) {
        char* y = first + (size_t)lane * row_bytes;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          if (j + k < left) {
            if (MODE == kF32) reinterpret_cast<float*>(y)[j + k] = acc[j + k];
            else reinterpret_cast<__nv_bfloat16*>(y)[j + k] = __float2bfloat16_rn(acc[j + k]);
          }
        }
      }
    }
  } else {
    // N is a multiple of 128 here: the tile's outputs are all there
    if (GROUPS && p.row_weight && live) {
      const float w = p.row_weight[row];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] *= w;
    }
    uint32_t o[32];                   // 64 outputs as bfloat16
    if (p.glu.kind == 1 && p.glu.bias == nullptr) {
#pragma unroll
      for (int j = 0; j < 32; ++j) o[j] = pack2(silu_mul_fast(acc[2 * j], acc[64 + 2 * j]), silu_mul_fast(acc[2 * j + 1], acc[64 + 2 * j + 1]));
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        float g[2] = {acc[2 * j], acc[2 * j + 1]}, u[2] = {acc[64 + 2 * j], acc[64 + 2 * j + 1]};
        if (p.glu.bias) {
          const int col = n0 + c0 + 2 * j;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            g[k] += p.glu.bias[col + k];
            u[k] += p.glu.bias[p.N + col + k];
          }
        }
        o[j] = glu_fast_pair(p.glu, g[0], g[1], u[0], u[1]);
      }
    }
    if (MODE == kGlu) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (vec) {
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = make_uint4(o[16 * c + 4 * k], o[16 * c + 4 * k + 1], o[16 * c + 4 * k + 2], o[16 * c + 4 * k + 3]);
          put64(out_buf, lane, v, first + 64 * c, row_bytes, n_rows);
        } else if (lane < n_rows) {
          __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(first + (size_t)lane * row_bytes) + 32 * c;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            y[2 * j] = reinterpret_cast<const __nv_bfloat162*>(o)[16 * c + j].x;
            y[2 * j + 1] = reinterpret_cast<const __nv_bfloat162*>(o)[16 * c + j].y;
          }
        }
      }
    } else {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(o)[j]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top_s[h][r_tile] = top;         // the other half of the row's 128 outputs is another warp's
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      top = fmaxf(top_s[0][r_tile], top_s[1][r_tile]);
      const uint32_t scale = scale_bits(top);
      const float by = inverse_of(scale);
      const bool inf = top == INFINITY;
      uint32_t q8[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 a = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(o)[2 * j]);
        const float2 b = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(o)[2 * j + 1]);
        q8[j] = inf ? pack4(no_infinity(a.x) * by, no_infinity(a.y) * by, no_infinity(b.x) * by, no_infinity(b.y) * by)
                    : pack4(a.x * by, a.y * by, b.x * by, b.y * by);
      }
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = make_uint4(q8[4 * k], q8[4 * k + 1], q8[4 * k + 2], q8[4 * k + 3]);
      put64(out_buf, lane, v, first, row_bytes, n_rows);
      if (h == 0 && lane < n_rows) p.ys[(size_t)(n0 / 128) * p.ys_ld + row] = __uint_as_float(scale);
      asm volatile("bar.sync 1, 256;\n" ::: "memory");     // the next tile writes top_s again
    }
  }
}

}  // namespace fp8
}  // namespace pe
