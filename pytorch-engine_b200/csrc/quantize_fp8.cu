// Rows and matrices to 8-bit floating point (e4m3: 4 exponent bits, 3 mantissa bits, largest value 448) with one scale for
// each block: 128 neighbouring features of a row, or 128 x 128 elements of a weight matrix.
//
//   a = max |x| over the block ;  s = the smallest 2^e (e >= -126) with a <= 448 * 2^e ;  q = e4m3(x / s)
//
// The scale is a power of two: x / s is then exact, so a block's values do not depend on how a quotient is rounded, and a
// power of two costs e4m3 nothing but its smallest values (its relative precision is the same in every binade).  A NaN stays a
// NaN and does not count for the block's maximum (a block of nothing else has a block of zeros' scale); an infinity becomes a NaN
// (e4m3 has none), and with it the block's scale is 2^120.
//
// Scales of rows are stored by block, [blocks, rows]: the products (gemm_fp8.cu) read one block's scales of many rows at a time.
#include "api.h"
#include "fp8.cuh"

namespace pe {
namespace quant8 {
using namespace fp8;

constexpr int BLOCK = BK;       // features of a block

// Eight neighbouring features of a row as they lie in memory, from column `c`, zeros behind the row's end (or with K = 0).
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ float top() const {
    // the largest magnitudes two at a time; a NaN loses against a number, eight of them against the 0
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
    return fmaxf(fmaxf(__low2float(m), __high2float(m)), 0.f);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
};
template <> struct Raw8<float> {
  float4 v[2];
  __device__ __forceinline__ float top() const {
    return fmaxf(fmaxf(fmaxf(fmaxf(fabsf(v[0].x), fabsf(v[0].y)), fmaxf(fabsf(v[0].z), fabsf(v[0].w))),
                       fmaxf(fmaxf(fabsf(v[1].x), fabsf(v[1].y)), fmaxf(fabsf(v[1].z), fabsf(v[1].w)))), 0.f);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = v[0].x; f[1] = v[0].y; f[2] = v[0].z; f[3] = v[0].w; f[4] = v[1].x; f[5] = v[1].y; f[6] = v[1].z; f[7] = v[1].w;
  }
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* row, int c, int K, bool vec) {
  Raw8<T> r;
  if (vec && c + 8 <= K) {
    r = *reinterpret_cast<const Raw8<T>*>(row + c);
  } else {
    alignas(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c + i < K ? row[c + i] : from_f32<T>(0.f);
    r = *reinterpret_cast<const Raw8<T>*>(e);
  }
  return r;
}
// Rows of values start on 16-byte boundaries, so eight of them at a multiple of eight are one store.
template <typename T>
__device__ __forceinline__ void store8(uint8_t* row, int c, int K, const Raw8<T>& r, uint32_t scale, float a) {
  float v[8];
  r.get(v);
  if (a == INFINITY) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = no_infinity(v[i]);
  }
  const float inv = inverse_of(scale);
  uint2 q;
  q.x = pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  q.y = pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
  if (c + 8 <= K) {
    *reinterpret_cast<uint2*>(row + c) = q;
  } else {
    const uint8_t* b = reinterpret_cast<const uint8_t*>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) row[c + i] = b[i];
  }
}

// Sixteen lanes a block of 128 features, sixteen rows a thread block (so that the scales, which lie by block, leave it 64 bytes at
// a time), U blocks of each row with their loads in flight together.  Blocks that take one turn after the other, the next one's loads
// in flight, were slower (2,048 x 4,096: 9.3 us).  `row_map`: output row r is input row row_map[r]; `n_live` (on the device): only so
// many rows are there.
template <typename T, int U>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, long long x_ld, const int* row_map, const int* n_live,
                                                            uint8_t* values, long long v_ld, float* scales, long long s_ld, int M,
                                                            int K, int x_rows, bool vec, int turns_x, int* status) {
  pdl_wait_block();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 15, blocks = (K + BLOCK - 1) / BLOCK;
  const int ty = blockIdx.x / turns_x, kb0 = (blockIdx.x - ty * turns_x) * U, r = ty * 16 + (threadIdx.x >> 4);
  if (n_live) M = min(M, *n_live);
  // all 32 lanes take part in the shuffles: rows that are not there are not read and not written
  int src = -1;
  if (r < M) {
    src = row_map ? row_map[r] : r;
    if (src < 0 || src >= x_rows) {
      if (lane == 0 && kb0 == 0) report(status, kStatusRowOutOfRange, r, src, x_rows);
      src = -1;
    }
  }
  const T* row = x + (size_t)max(src, 0) * x_ld;
  Raw8<T> v[U];
  float a[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = load8<T>(row, (kb0 + u) * BLOCK + lane * 8, src < 0 ? 0 : K, vec);
#pragma unroll
  for (int u = 0; u < U; ++u) a[u] = v[u].top();
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = fmaxf(a[u], __shfl_xor_sync(0xffffffffu, a[u], o));
  if (src < 0) return;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (kb0 + u >= blocks) break;
    const uint32_t s = scale_bits(a[u]);
    store8<T>(values + (size_t)r * v_ld, (kb0 + u) * BLOCK + lane * 8, K, v[u], s, a[u]);
    if (lane == 0) scales[(size_t)(kb0 + u) * s_ld + r] = __uint_as_float(s);
  }
}

// One thread block for 128 x 128 elements, which it holds in registers between the maximum and the conversion.  Its successor in the
// stream may be a product that asks for these values before it waits for this grid.  So it lets nothing start early, which leaves a
// successor to start when all blocks have ended, and a block ends behind a fence: what it wrote has then reached the memory that all
// SMs and their copies (the async proxy's) read.  (24,576 x 4,096 bfloat16 in a graph: 50.0 us, without the fence 48.6, with every
// thread behind one 53.)
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) quantize_weight_kernel(const T* w, long long w_ld, uint8_t* values, long long v_ld,
                                                                                    float* scales, int N, int K, bool vec) {
  __shared__ float red[32];
  pdl_wait_block();
  const int blocks = (K + BLOCK - 1) / BLOCK;
  const int rb = blockIdx.x / blocks, kb = blockIdx.x - rb * blocks;
  const int c = kb * BLOCK + (threadIdx.x & 15) * 8;
  Raw8<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rb * BLOCK + i * 16 + (threadIdx.x >> 4);
    v[i] = load8<T>(w + (size_t)min(r, N - 1) * w_ld, c, r < N ? K : 0, vec);
  }
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, v[i].top());
  a = block_max(a, red);
  const uint32_t s = scale_bits(a);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rb * BLOCK + i * 16 + (threadIdx.x >> 4);
    if (r < N) store8<T>(values + (size_t)r * v_ld, c, K, v[i], s, a);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    scales[blockIdx.x] = __uint_as_float(s);
    __threadfence();
    asm volatile("fence.proxy.async.global;\n" ::: "memory");
  }
}

// Nothing, behind everything in front of it: see pe_settle_weights.
__global__ void settle_kernel() {}

// rmsnorm.cu's norm (with its residual add) whose result, rounded to bfloat16, is quantised on the way out: what rmsnorm.cu's
// kernel and the one above would give, without the bfloat16 rows between them.  The sum of squares is taken in rmsnorm.cu's order, four
// features a thread; the rest with eight a thread, for which the sixteen lanes of a block need a step less than 32 would (2,011 x 4,096:
// 14.6 us, with four 16.1; asking for several of a thread's features at once made it 19).
__global__ void __launch_bounds__(1024) rmsnorm_residual_fp8_kernel(float* residual, const __nv_bfloat16* delta,
                                                                    const float* __restrict__ weight, uint8_t* values,
                                                                    long long v_ld, float* scales, long long s_ld, int dim,
                                                                    float eps) {
  extern __shared__ float row_buf[];  // dim floats
  __shared__ float red[32];
  const int c0 = threadIdx.x * 4;
  // the weight does not come from the kernel before this one
  float4 w0[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if ((int)threadIdx.x * 8 + 4 * i < dim) w0[i] = *reinterpret_cast<const float4*>(weight + threadIdx.x * 8 + 4 * i);
  pdl_wait_block();
  pdl_launch_dependents();
  const int r = blockIdx.x;
  float* res_row = residual + (size_t)r * dim;
  const __nv_bfloat16* d_row = delta ? delta + (size_t)r * dim : nullptr;
  float ss = 0.f;
  for (int c = c0; c < dim; c += blockDim.x * 4) {
    float4 h = *reinterpret_cast<const float4*>(res_row + c);
    if (d_row) {
      const uint2 u = *reinterpret_cast<const uint2*>(d_row + c);
      const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
      const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
      h.x += a.x; h.y += a.y; h.z += b.x; h.w += b.y;
      *reinterpret_cast<float4*>(res_row + c) = h;
    }
    *reinterpret_cast<float4*>(row_buf + c) = h;
    ss += h.x * h.x + h.y * h.y + h.z * h.z + h.w * h.w;
  }
  const float inv = rsqrtf(block_sum(ss, red) / (float)dim + eps);
  // from here on eight features a thread, sixteen lanes a block; whole warps stay in the loop for the shuffles
  for (int c = threadIdx.x * 8; c - (int)(threadIdx.x & 31) * 8 < dim; c += blockDim.x * 8) {
    uint32_t y[4] = {0, 0, 0, 0};         // bfloat16 pairs
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (c + 4 * i < dim) {
        const float4 h = *reinterpret_cast<const float4*>(row_buf + c + 4 * i);
        const float4 w = c == (int)threadIdx.x * 8 ? w0[i] : *reinterpret_cast<const float4*>(weight + c + 4 * i);
        const __nv_bfloat162 lo = __floats2bfloat162_rn(h.x * inv * w.x, h.y * inv * w.y), hi = __floats2bfloat162_rn(h.z * inv * w.z, h.w * inv * w.w);
        y[2 * i] = *reinterpret_cast<const uint32_t*>(&lo);
        y[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&hi);
      }
    Raw8<__nv_bfloat16> v;
    v.v = make_uint4(y[0], y[1], y[2], y[3]);
    float a = v.top();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (c >= dim) continue;
    const uint32_t s = scale_bits(a);
    store8<__nv_bfloat16>(values + (size_t)r * v_ld, c, dim, v, s, a);
    if ((threadIdx.x & 15) == 0) scales[(size_t)(c / BLOCK) * s_ld + r] = __uint_as_float(s);
  }
}

template <typename T>
static int launch_rows(const T* x, long long x_ld, const int* row_map, const int* n_live, uint8_t* values, long long v_ld, float* scales,
                       long long s_ld, int M, int K, int x_rows, int* status, cudaStream_t stream) {
  const bool vec = ((uintptr_t)x % 16) == 0 && (x_ld * (long long)sizeof(T)) % 16 == 0;
  const int blocks = (K + BLOCK - 1) / BLOCK, row_blocks = (M + 15) / 16;
  // several blocks of a row a thread block where that still leaves every SM four of them
  // (2,048 x 12,288 bfloat16: 15.3 us with four, 17.6 with two, 18.1 with eight)
  constexpr int U = 4;
  const bool many = (long long)row_blocks * blocks >= (long long)U * 4 * kSMs;
  const int per = many ? U : 1, turns_x = (blocks + per - 1) / per;
  if ((long long)turns_x * row_blocks > 0x7fffffffLL) return PE_ERR_UNSUPPORTED_SIZE;
  const dim3 grid((unsigned)(turns_x * row_blocks));
  cudaError_t e = many ? launch(quantize_rows_kernel<T, U>, grid, dim3(256), 0, stream, x, x_ld, row_map, n_live, values, v_ld, scales, s_ld, M, K,
                                x_rows, vec, turns_x, status)
                       : launch(quantize_rows_kernel<T, 1>, grid, dim3(256), 0, stream, x, x_ld, row_map, n_live, values, v_ld, scales, s_ld, M, K,
                                x_rows, vec, turns_x, status);
  if (e != cudaSuccess) return (int)e;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

}  // namespace quant8
}  // namespace pe

// values[r] (M rows, v_ld bytes apart, a multiple of 16, on 16-byte boundaries), scales[b * s_ld + r]; row r is row row_map[r] of x
// (row_map null: r), which has x_rows rows x_ld elements apart.  n_live (or null): only the first *n_live rows are there.
extern "C" int pe_quantize_rows_fp8(int dtype, const void* x, long long x_ld, const int* row_map, const int* n_live, void* values, long long v_ld,
                                    float* scales, long long s_ld, int M, int K, int x_rows, int* status, cudaStream_t stream) {
  using namespace pe::quant8;
  if (M < 0 || K < 0) return PE_ERR_BAD_ARGUMENT;
  if (M == 0 || K == 0) return PE_OK;
  if (x == nullptr || values == nullptr || scales == nullptr || x_ld < K || v_ld < K || s_ld < M || x_rows < 1 || (!row_map && M > x_rows))
    return PE_ERR_BAD_ARGUMENT;
  if (((uintptr_t)values % 16) || (v_ld % 16)) return PE_ERR_BAD_ARGUMENT;
  if (M > kMostRows || K > kMostRows) return PE_ERR_UNSUPPORTED_SIZE;
  if (dtype == PE_BF16) return launch_rows((const __nv_bfloat16*)x, x_ld, row_map, n_live, (uint8_t*)values, v_ld, scales, s_ld, M, K, x_rows, status, stream);
  if (dtype == PE_F32) return launch_rows((const float*)x, x_ld, row_map, n_live, (uint8_t*)values, v_ld, scales, s_ld, M, K, x_rows, status, stream);
  return PE_ERR_UNSUPPORTED_DTYPE;
}

// values as above (N rows), scales[rb * ceil(K / 128) + kb].
extern "C" int pe_quantize_weight_fp8(int dtype, const void* w, long long w_ld, void* values, long long v_ld, float* scales, int N,
                                      int K, cudaStream_t stream) {
  using namespace pe::quant8;
  if (N < 0 || K < 0) return PE_ERR_BAD_ARGUMENT;
  if (N == 0 || K == 0) return PE_OK;
  if (w == nullptr || values == nullptr || scales == nullptr || w_ld < K || v_ld < K) return PE_ERR_BAD_ARGUMENT;
  if (((uintptr_t)values % 16) || (v_ld % 16)) return PE_ERR_BAD_ARGUMENT;
  if (N > kMostRows || K > kMostRows) return PE_ERR_UNSUPPORTED_SIZE;
  const long long cells = (long long)((N + BLOCK - 1) / BLOCK) * ((K + BLOCK - 1) / BLOCK);
  if (cells > 0x7fffffffLL) return PE_ERR_UNSUPPORTED_SIZE;
  cudaError_t e;
  if (dtype == PE_BF16) {
    const bool vec = ((uintptr_t)w % 16) == 0 && (w_ld * 2) % 16 == 0;
    e = pe::launch(quantize_weight_kernel<__nv_bfloat16>, dim3((unsigned)cells), dim3(256), 0, stream, (const __nv_bfloat16*)w, w_ld, (uint8_t*)values, v_ld, scales, N, K, vec);
  } else if (dtype == PE_F32) {
    const bool vec = ((uintptr_t)w % 16) == 0 && (w_ld * 4) % 16 == 0;
    e = pe::launch(quantize_weight_kernel<float>, dim3((unsigned)cells), dim3(256), 0, stream, (const float*)w, w_ld, (uint8_t*)values, v_ld, scales, N, K, vec);
  } else {
    return PE_ERR_UNSUPPORTED_DTYPE;
  }
  if (e != cudaSuccess) return (int)e;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

// What the stream has written up to here may be read as weights by the launches behind: a product asks for its weights while the
// launch in front of it still runs, and this one, which does not start before all in front of it has completed, then stands between.
extern "C" int pe_settle_weights(cudaStream_t stream) {
  const cudaError_t e = pe::launch_after(pe::quant8::settle_kernel, dim3(1), dim3(32), 0, stream);
  if (e != cudaSuccess) return (int)e;
  PE_LAUNCH_CHECK();
  return PE_OK;
}

// Rows of residual (float32) and delta (bfloat16 or null) are packed; dim a multiple of 4, at most 51,200 (a row lies in shared memory).
extern "C" int pe_rmsnorm_residual_fp8(float* residual, const void* delta, const float* weight, void* values, long long v_ld,
                                       float* scales, long long s_ld, int n_rows, int dim, float eps, cudaStream_t stream) {
  using namespace pe::quant8;
  if (n_rows < 0 || dim < 1) return PE_ERR_BAD_ARGUMENT;
  if (n_rows == 0) return PE_OK;
  if (residual == nullptr || weight == nullptr || values == nullptr || scales == nullptr || v_ld < dim || s_ld < n_rows) return PE_ERR_BAD_ARGUMENT;
  const size_t smem = (size_t)dim * sizeof(float);
  if (dim % 4 || smem > 200 * 1024) return PE_ERR_UNSUPPORTED_SIZE;
  if (((uintptr_t)values % 16) || (v_ld % 16) || ((uintptr_t)residual % 16) || ((uintptr_t)weight % 16) || ((uintptr_t)delta % 8)) return PE_ERR_BAD_ARGUMENT;
  // threads as for rmsnorm.cu's kernel, whose sums these are
  int threads = dim >= 2048 ? 512 : (dim >= 512 ? 256 : 128);
  if (n_rows <= 64 && dim > 2048) threads = 1024;
  const int ae = pe::allow_smem(rmsnorm_residual_fp8_kernel, smem);
  if (ae != 0) return ae;
  const cudaError_t e = pe::launch(rmsnorm_residual_fp8_kernel, dim3(n_rows), dim3(threads), smem, stream, residual, (const __nv_bfloat16*)delta, weight, (uint8_t*)values, v_ld, scales, s_ld, dim, eps);
  if (e != cudaSuccess) return (int)e;
  PE_LAUNCH_CHECK();
  return PE_OK;
}
