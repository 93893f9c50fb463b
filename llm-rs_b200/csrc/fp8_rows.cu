// Rows in 8 bits (fp8.cuh) from rows as they are, from a gated unit, and from a residual sum and its norm: what the products of
// gemm_fp8.cu read. All three are bound by memory: a number is read once, its byte written once.
//
// A warp makes 512 numbers of a row, which is one word of scales. Two ways of dealing the numbers to lanes:
//   rows that start on 32-byte boundaries   a lane takes 16 consecutive numbers (loads of 32 bytes, a store of 16); a block's
//                                           maximum is the maximum over 8 neighbouring lanes
//   all others                              a lane takes number lane, lane + 32, .. (loads and stores of one number, coalesced
//                                           over the warp); a block's maximum is the maximum over the warp
#include "fp8.cuh"

constexpr int F8_THREADS = 256;

// Sixteen consecutive numbers from a 32-byte boundary.
__device__ __forceinline__ void f8_load16(const float* p, float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t r[8];
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p + 8 * h));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * h + i] = __uint_as_float(r[i]);
  }
}
__device__ __forceinline__ void f8_load16(const __nv_bfloat16* p, float (&v)[16]) {
  uint32_t r[8];
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(r[i] << 16);
    v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
  }
}

// The warp's 512 numbers, 16 consecutive ones a lane, into `q` (16-byte aligned; null: the lane's numbers are past the row's end)
// and *word.
__device__ __forceinline__ void f8_store_runs(float (&v)[16], uint8_t* q, uint32_t* word) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint32_t byte = f8_scale_byte(top);
  const float inv = f8_inverse(byte);
  if (q) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = f8_pack2(v[4 * i] * inv, v[4 * i + 1] * inv) | f8_pack2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16;
    *reinterpret_cast<uint4*>(q) = make_uint4(p[0], p[1], p[2], p[3]);
  }
  // Lanes 0, 8, 16, 24 hold the four blocks' bytes.
  uint32_t w = byte << (8 * ((threadIdx.x & 31) >> 3));
  w |= __shfl_xor_sync(0xffffffffu, w, 8);
  w |= __shfl_xor_sync(0xffffffffu, w, 16);
  if ((threadIdx.x & 31) == 0) *word = w;
}

// The warp's 512 numbers dealt by 32 (v[i] is number lane + 32 i); `left` numbers of the row are left.
__device__ __forceinline__ void f8_store_dealt(float (&v)[16], uint8_t* q, int left, uint32_t* word) {
  const int lane = threadIdx.x & 31;
  uint32_t w = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    float top = fmaxf(fmaxf(fabsf(v[4 * b]), fabsf(v[4 * b + 1])), fmaxf(fabsf(v[4 * b + 2]), fabsf(v[4 * b + 3])));
    top = warp_max(top);
    const uint32_t byte = f8_scale_byte(top);
    const float inv = f8_inverse(byte);
    w |= byte << (8 * b);
#pragma unroll
    for (int i = 4 * b; i < 4 * b + 4; i += 2) {
      const uint32_t two = f8_pack2(v[i] * inv, v[i + 1] * inv);
      if (lane + 32 * i < left) q[lane + 32 * i] = (uint8_t)two;
      if (lane + 32 * (i + 1) < left) q[lane + 32 * (i + 1)] = (uint8_t)(two >> 8);
    }
  }
  if (lane == 0) *word = w;
}

struct F8Rows {
  uint8_t* q;
  long long pitch;      // bytes between rows, a multiple of 16
  uint32_t* words;      // [word][rows]
  int rows, width, n_words;
};

// ---- rows as they are ---------------------------------------------------------------------------------------------
// Row r from row src[r] (or r) of x; a row whose source is none of x's becomes zeros.
template <typename T, bool RUNS>
__global__ void __launch_bounds__(F8_THREADS)
f8_quantize_kernel(const T* __restrict__ x, long long x_stride, int x_rows, const int* __restrict__ src, const F8Rows o) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * (F8_THREADS / 32) + (threadIdx.x >> 5), word = blockIdx.y;      // a block: one word of eight rows
  if (r >= o.rows) return;
  const int from = src ? src[r] : r, at = word * F8_WORD, left = o.width - at;
  const bool live = from >= 0 && from < x_rows;
  const T* xr = x + (live ? (size_t)from * x_stride : 0) + at;
  uint8_t* q = o.q + (size_t)r * o.pitch + at;
  uint32_t* w = o.words + (size_t)word * o.rows + r;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if (RUNS) {
    if (live && 16 * lane < left) f8_load16(xr + 16 * lane, v);
    f8_store_runs(v, 16 * lane < left ? q + 16 * lane : nullptr, w);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (live && lane + 32 * i < left) v[i] = to_float(xr[lane + 32 * i]);
    f8_store_dealt(v, q, left, w);
  }
}

// ---- the gated unit -------------------------------------------------------------------------------------------------
template <typename T, bool RUNS>
__global__ void __launch_bounds__(F8_THREADS)
f8_unit_kernel(const T* __restrict__ gu, long long gu_stride, int block, const GatedUnit unit, const F8Rows o) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * (F8_THREADS / 32) + (threadIdx.x >> 5), word = blockIdx.y;
  if (r >= o.rows) return;
  const int at = word * F8_WORD, left = o.width - at;
  const T* row = gu + (size_t)r * gu_stride;
  uint8_t* q = o.q + (size_t)r * o.pitch + at;
  uint32_t* w = o.words + (size_t)word * o.rows + r;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if (RUNS) {      // a run of 16 columns lies within a run of `block`
    const int c = at + 16 * lane;
    if (16 * lane < left) {
      float g[16];
      const T* p = row + (size_t)(c / block) * 2 * block + c % block;
      f8_load16(p, g);
      f8_load16(p + block, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = unit(g[i], v[i]);
    }
    f8_store_runs(v, 16 * lane < left ? q + 16 * lane : nullptr, w);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = at + lane + 32 * i;
      if (c < o.width) {
        const T* p = row + (size_t)(c / block) * 2 * block + c % block;
        v[i] = unit(to_float(p[0]), to_float(p[block]));
      }
    }
    f8_store_dealt(v, q, left, w);
  }
}

// ---- the residual sum and the norm ------------------------------------------------------------------------------------
// h += delta, then h / sqrt(mean(h^2) + eps) * weight in 8 bits; with `rows` row i comes from row rows[i] of h and delta, and h is
// left as it is. A block per row; the sum of squares is made in float32 by each thread and in double over the threads.
__device__ __forceinline__ double f8_block_sum(double v, double* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  double t = lane < n ? red[lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// 1 / sqrt(mean + eps), rounded once: CUDA's approximate root and one Newton step in double.
__device__ __forceinline__ float f8_inverse_root(double mean) {
  const double y = rsqrtf((float)mean);
  return (float)(y * (1.5 - 0.5 * mean * y * y));
}

// A thread keeps 16 consecutive numbers of the row in registers (rows of at most 16,384 numbers, 16 at a time).
template <typename T>
__global__ void __launch_bounds__(1024)
f8_norm_runs_kernel(float* __restrict__ h, const T* __restrict__ delta, const float* __restrict__ weight,
                    const int* __restrict__ rows, int h_rows, float eps, double per, const F8Rows o) {
  __shared__ double red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, c = threadIdx.x * 16, from = rows ? rows[r] : r;
  const bool live = c < o.width && from >= 0 && from < h_rows;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  float ss = 0.f;
  if (live) {
    float* hr = h + (size_t)from * o.width + c;
    f8_load16(hr, v);
    if (delta) {
      float d[16];
      f8_load16(delta + (size_t)from * o.width + c, d);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] += d[i];
      if (!rows) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(hr + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
  }
  const double total = f8_block_sum((double)ss, red);
  const float inv = f8_inverse_root(total * per + (double)eps);
  if (live) {
    float wt[16];
    f8_load16(weight + c, wt);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = v[i] * inv * wt[i];
  }
  const int word = threadIdx.x >> 5;
  f8_store_runs(v, c < o.width ? o.q + (size_t)r * o.pitch + c : nullptr, o.words + (size_t)word * o.rows + r);
}

constexpr int F8_NORM_THREADS = 512;
template <typename T>
__global__ void __launch_bounds__(F8_NORM_THREADS)
f8_norm_dealt_kernel(float* __restrict__ h, const T* __restrict__ delta, const float* __restrict__ weight,
                     const int* __restrict__ rows, int h_rows, float eps, double per, const F8Rows o) {
  __shared__ double red[32];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, from = rows ? rows[r] : r, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool live = from >= 0 && from < h_rows;
  float* hr = h + (live ? (size_t)from * o.width : 0);
  const T* dr = delta && live ? delta + (size_t)from * o.width : nullptr;
  float ss = 0.f;
  if (live)
    for (int c = threadIdx.x; c < o.width; c += F8_NORM_THREADS) {
      float v = hr[c];
      if (dr) {
        v += to_float(dr[c]);
        if (!rows) hr[c] = v;
      }
      ss = fmaf(v, v, ss);
    }
  const double total = f8_block_sum((double)ss, red);      // (its barrier also orders the sums above before the loads below)
  const float inv = f8_inverse_root(total * per + (double)eps);
  for (int word = warp; word < o.n_words; word += F8_NORM_THREADS / 32) {
    const int at = word * F8_WORD, left = o.width - at;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = at + lane + 32 * i;
      v[i] = 0.f;
      if (live && c < o.width) {
        v[i] = hr[c];
        if (dr && rows) v[i] += to_float(dr[c]);
        v[i] = v[i] * inv * weight[c];
      }
    }
    f8_store_dealt(v, o.q + (size_t)r * o.pitch + at, left, o.words + (size_t)word * o.rows + r);
  }
}

// ---- entries ------------------------------------------------------------------------------------------------------
static int f8_rows_of(F8Rows* o, const char* what, void* q, long long pitch, void* words, int rows, int width) {
  LLMRS_REQUIRE(rows >= 0 && width > 0, "%s: bad sizes", what);
  LLMRS_REQUIRE(pitch % 16 == 0 && pitch >= width && ((uintptr_t)q & 15) == 0 && ((uintptr_t)words & 3) == 0,
                "%s: rows of q must start at multiples of 16 bytes, scales at multiples of 4", what);
  *o = F8Rows{(uint8_t*)q, pitch, (uint32_t*)words, rows, width, (width + F8_WORD - 1) / F8_WORD};
  LLMRS_REQUIRE(o->n_words <= 65535, "%s: rows of more than %d numbers", what, 65535 * F8_WORD);
  return 0;
}
static bool f8_in_runs(const void* x, long long stride, int size, int width) {
  return width % 16 == 0 && ((uintptr_t)x & 31) == 0 && stride * size % 32 == 0;
}
static dim3 f8_grid(const F8Rows& o) { return dim3((unsigned)((o.rows - 1) / (F8_THREADS / 32) + 1), (unsigned)o.n_words); }

LLMRS_API int llmrs_quantize_fp8(const void* x, int dtype, long long x_stride, int x_rows, const int* src, void* q,
                                 long long pitch, void* words, int rows, int width, cudaStream_t stream) {
  F8Rows o;
  if (const int rc = f8_rows_of(&o, "quantize_fp8", q, pitch, words, rows, width)) return rc;
  if (rows == 0) return 0;
  cudaError_t e;
  if (dtype == LLMRS_F32) {
    auto* k = f8_in_runs(x, x_stride, 4, width) ? f8_quantize_kernel<float, true> : f8_quantize_kernel<float, false>;
    e = llmrs_launch(k, f8_grid(o), dim3(F8_THREADS), 0, stream, true, (const float*)x, x_stride, x_rows, src, o);
  } else if (dtype == LLMRS_BF16) {
    auto* k = f8_in_runs(x, x_stride, 2, width) ? f8_quantize_kernel<__nv_bfloat16, true> : f8_quantize_kernel<__nv_bfloat16, false>;
    e = llmrs_launch(k, f8_grid(o), dim3(F8_THREADS), 0, stream, true, (const __nv_bfloat16*)x, x_stride, x_rows, src, o);
  } else {
    return llmrs_fail("quantize_fp8: unknown dtype %d", dtype);
  }
  if (e != cudaSuccess) return llmrs_fail("quantize_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("quantize_fp8");
}

// gu [rows, 2 * width]: gate and up in alternating runs of `block` columns (which divides the width).
LLMRS_API int llmrs_silu_mul_fp8(const void* gu, int dtype, long long gu_stride, int block, float limit, float alpha, float shift,
                                 void* q, long long pitch, void* words, int rows, int width, cudaStream_t stream) {
  F8Rows o;
  if (const int rc = f8_rows_of(&o, "silu_mul_fp8", q, pitch, words, rows, width)) return rc;
  LLMRS_REQUIRE(block > 0 && width % block == 0, "silu_mul_fp8: runs of %d columns do not divide %d", block, width);
  if (rows == 0) return 0;
  const GatedUnit unit = {limit, alpha, shift};
  const bool runs = block % 16 == 0;
  cudaError_t e;
  if (dtype == LLMRS_F32) {
    auto* k = runs && f8_in_runs(gu, gu_stride, 4, width) ? f8_unit_kernel<float, true> : f8_unit_kernel<float, false>;
    e = llmrs_launch(k, f8_grid(o), dim3(F8_THREADS), 0, stream, true, (const float*)gu, gu_stride, block, unit, o);
  } else if (dtype == LLMRS_BF16) {
    auto* k = runs && f8_in_runs(gu, gu_stride, 2, width) ? f8_unit_kernel<__nv_bfloat16, true> : f8_unit_kernel<__nv_bfloat16, false>;
    e = llmrs_launch(k, f8_grid(o), dim3(F8_THREADS), 0, stream, true, (const __nv_bfloat16*)gu, gu_stride, block, unit, o);
  } else {
    return llmrs_fail("silu_mul_fp8: unknown dtype %d", dtype);
  }
  if (e != cudaSuccess) return llmrs_fail("silu_mul_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("silu_mul_fp8");
}

template <typename T>
static cudaError_t f8_launch_norm(float* h, const T* delta, const float* weight, const int* rows, int h_rows, float eps,
                                  const F8Rows& o, cudaStream_t stream) {
  const bool runs = o.width <= 16384 && f8_in_runs(h, o.width, 4, o.width) && ((uintptr_t)weight & 31) == 0 &&
                    (!delta || f8_in_runs(delta, o.width, (int)sizeof(T), o.width));
  if (runs)
    return llmrs_launch(f8_norm_runs_kernel<T>, dim3(o.rows), dim3(o.n_words * 32), 0, stream, true, h, delta, weight, rows, h_rows,
                        eps, 1.0 / o.width, o);
  return llmrs_launch(f8_norm_dealt_kernel<T>, dim3(o.rows), dim3(F8_NORM_THREADS), 0, stream, true, h, delta, weight, rows, h_rows,
                      eps, 1.0 / o.width, o);
}

// h [h_rows, width] float32 and delta (or null) of `dtype`, contiguous.
LLMRS_API int llmrs_add_rmsnorm_fp8(float* h, const void* delta, int dtype, const float* weight, const int* rows, int h_rows,
                                    float eps, void* q, long long pitch, void* words, int n_rows, int width, cudaStream_t stream) {
  F8Rows o;
  if (const int rc = f8_rows_of(&o, "add_rmsnorm_fp8", q, pitch, words, n_rows, width)) return rc;
  LLMRS_REQUIRE(dtype == LLMRS_F32 || dtype == LLMRS_BF16, "add_rmsnorm_fp8: unknown dtype %d", dtype);
  if (n_rows == 0) return 0;
  const cudaError_t e = dtype == LLMRS_F32
                            ? f8_launch_norm<float>(h, (const float*)delta, weight, rows, h_rows, eps, o, stream)
                            : f8_launch_norm<__nv_bfloat16>(h, (const __nv_bfloat16*)delta, weight, rows, h_rows, eps, o, stream);
  if (e != cudaSuccess) return llmrs_fail("add_rmsnorm_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("add_rmsnorm_fp8");
}
