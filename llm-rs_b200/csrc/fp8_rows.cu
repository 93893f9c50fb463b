// Rows in 8 bits (fp8.cuh) from rows as they are, from a gated unit, and from a residual sum and its norm: what the products of
// gemm_fp8.cu read. All three are bound by memory: a number is read once, its byte written once.
//
// A warp makes 512 numbers of a row, which is one word of scales. Two ways of dealing the numbers to lanes:
//   rows that start on 32-byte boundaries   a lane takes 16 consecutive numbers (loads of 32 bytes, a store of 16); a block's
//                                           maximum is the maximum over 8 neighbouring lanes
//   all others                              a lane takes 4 consecutive numbers of each of the four blocks (loads of what is
//                                           aligned, stores of 4 bytes: q's rows start at multiples of 16); a block's maximum is the
//                                           maximum over the warp
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
    if (isinf(top)) {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        float a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = i == 0 ? v[e] : i == 1 ? v[4 + e] : i == 2 ? v[8 + e] : v[12 + e];
        const uint32_t q4 = f8_pack2_any(a[0] * inv, a[1] * inv) | f8_pack2_any(a[2] * inv, a[3] * inv) << 16;
        if (i == 0) p[0] = q4;
        if (i == 1) p[1] = q4;
        if (i == 2) p[2] = q4;
        if (i == 3) p[3] = q4;
      }
    }
    *reinterpret_cast<uint4*>(q) = make_uint4(p[0], p[1], p[2], p[3]);
  }
  // Lanes 0, 8, 16, 24 hold the four blocks' bytes.
  uint32_t w = byte << (8 * ((threadIdx.x & 31) >> 3));
  w |= __shfl_xor_sync(0xffffffffu, w, 8);
  w |= __shfl_xor_sync(0xffffffffu, w, 16);
  if ((threadIdx.x & 31) == 0) *word = w;
}

// Eight consecutive numbers, from a 32-byte (float32) or a 16-byte boundary.
__device__ __forceinline__ void f8_load8(const float* p, float* v) {
  uint32_t r[8];
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void f8_load8(const __nv_bfloat16* p, float* v) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(r[i] << 16);
    v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void f8_put8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// The warp's 512 numbers by eights (v[8 h + i] is number 256 h + 8 lane + i); `left` numbers of the row are left, a multiple of 16.
// The scale's byte grows with the magnitude, so that the bytes of the lanes' own maxima are what is compared: those of both halves
// in one register.
__device__ __forceinline__ void f8_store_eights(float (&v)[16], uint8_t* q, int left, uint32_t* word) {
  const int lane = threadIdx.x & 31;
  float top[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) top[0] = fmaxf(top[0], fabsf(v[i])), top[1] = fmaxf(top[1], fabsf(v[8 + i]));
  uint32_t both = f8_scale_byte(top[0]) | f8_scale_byte(top[1]) << 16;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (256 * h + 8 * lane >= left) continue;
    const float inv = f8_inverse(h ? both >> 16 : both & 0xffffu);
    float* x = v + 8 * h;
    uint2 p;
    p.x = f8_pack2(x[0] * inv, x[1] * inv) | f8_pack2(x[2] * inv, x[3] * inv) << 16;
    p.y = f8_pack2(x[4] * inv, x[5] * inv) | f8_pack2(x[6] * inv, x[7] * inv) << 16;
    if (isinf(top[h])) {
      p.x = f8_pack2_any(x[0] * inv, x[1] * inv) | f8_pack2_any(x[2] * inv, x[3] * inv) << 16;
      p.y = f8_pack2_any(x[4] * inv, x[5] * inv) | f8_pack2_any(x[6] * inv, x[7] * inv) << 16;
    }
    *reinterpret_cast<uint2*>(q + 256 * h + 8 * lane) = p;
  }
  // Lanes 0-15 hold the bytes of blocks 0 and 2, the others those of 1 and 3.
  uint32_t w = both << (lane < 16 ? 0 : 8);
  w |= __shfl_xor_sync(0xffffffffu, w, 16);
  if (lane == 0) *word = w;
}

// Four consecutive numbers, of which `n` are there (zeros behind them), from any address. bfloat16 numbers come by the words that hold
// them: a word's other half lies in the same aligned four bytes as the number that is asked for.
__device__ __forceinline__ void f8_load4(const float* p, int n, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
}
__device__ __forceinline__ void f8_load4(const __nv_bfloat16* p, int n, float* v) {
  const uint32_t odd = (uint32_t)((uintptr_t)p >> 1) & 1u;      // the first number is a word's upper half
  const uint32_t* w = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
  if (n >= 4) {
    const uint32_t a = w[0], b = w[1], c = odd ? w[2] : 0u;
    const uint32_t lo = __funnelshift_r(a, b, 16 * odd), hi = __funnelshift_r(b, c, 16 * odd);
    v[0] = __uint_as_float(lo << 16), v[1] = __uint_as_float(lo & 0xffff0000u);
    v[2] = __uint_as_float(hi << 16), v[3] = __uint_as_float(hi & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.f;
  }
}

// The warp's 512 numbers by fours (v[4 j + i] is number 128 j + 4 lane + i); `left` numbers of the row are left. The last word of
// a row of q is written whole.
__device__ __forceinline__ void f8_store_fours(float (&v)[16], uint8_t* q, int left, uint32_t* word) {
  const int lane = threadIdx.x & 31;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // The bits of magnitudes are ordered as whole numbers, whose maximum over a warp is one instruction (a NaN counts as 0).
    const float own = fmaxf(fmaxf(fmaxf(fabsf(v[4 * j]), fabsf(v[4 * j + 1])), fmaxf(fabsf(v[4 * j + 2]), fabsf(v[4 * j + 3]))), 0.f);
    const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(own)));
    const uint32_t byte = f8_scale_byte(top);
    const float inv = f8_inverse(byte);
    w |= byte << (8 * j);
    uint32_t p = f8_pack2(v[4 * j] * inv, v[4 * j + 1] * inv) | f8_pack2(v[4 * j + 2] * inv, v[4 * j + 3] * inv) << 16;
    if (isinf(top))
      p = f8_pack2_any(v[4 * j] * inv, v[4 * j + 1] * inv) | f8_pack2_any(v[4 * j + 2] * inv, v[4 * j + 3] * inv) << 16;
    if (128 * j + 4 * lane < left) *reinterpret_cast<uint32_t*>(q + 128 * j + 4 * lane) = p;
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
// Row r from row src[r] (or r) of x; a row whose source is none of x's becomes zeros. A warp makes two words of a row, so that
// the loads of both are in flight (7,211 rows of 4,096 bfloat16 numbers: 16.1 us with one, 15.0 with two; 13.8 at 6.45 TB/s).
template <typename T, bool RUNS>
__global__ void __launch_bounds__(F8_THREADS)
f8_quantize_kernel(const T* __restrict__ x, long long x_stride, int x_rows, const int* __restrict__ src, const F8Rows o) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * (F8_THREADS / 32) + (threadIdx.x >> 5);      // a block: two words of eight rows
  if (r >= o.rows) return;
  const int from = src ? src[r] : r;
  const bool live = from >= 0 && from < x_rows;
  const T* xr = x + (live ? (size_t)from * x_stride : 0);
  float v[2][16];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = (2 * blockIdx.y + h) * F8_WORD, left = live ? o.width - at : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[h][i] = 0.f;
    if (RUNS) {
      if (16 * lane < left) f8_load16(xr + at + 16 * lane, v[h]);
    } else if (left >= F8_WORD) {      // no branch between the loads: they are in flight together
#pragma unroll
      for (int j = 0; j < 4; ++j) f8_load4(xr + at + 128 * j + 4 * lane, 4, v[h] + 4 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (128 * j + 4 * lane < left) f8_load4(xr + at + 128 * j + 4 * lane, left - 128 * j - 4 * lane, v[h] + 4 * j);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int word = 2 * blockIdx.y + h, left = o.width - word * F8_WORD;
    if (left <= 0) break;
    uint8_t* q = o.q + (size_t)r * o.pitch + word * F8_WORD;
    uint32_t* w = o.words + (size_t)word * o.rows + r;
    if (RUNS)
      f8_store_runs(v[h], 16 * lane < left ? q + 16 * lane : nullptr, w);
    else
      f8_store_fours(v[h], q, left, w);
  }
}

// ---- the gated unit -------------------------------------------------------------------------------------------------
// GatedUnit in fewer instructions: the quotient by an approximate reciprocal and one step of the remainder, off by less than an ulp as
// a division is; PLAIN is silu(gate) * up. What bounds the kernel is these instructions beside the memory: 2,048 rows of 12,288
// took 33 us with the division, 24.5 with this (19.5 at 6.45 TB/s).
constexpr float F8_LOG2E = 1.44269504088896f;      // log2(e)
template <bool PLAIN>
__device__ __forceinline__ float f8_unit(const GatedUnit& unit, float gate, float up) {
  const float g = PLAIN ? gate : fminf(gate, unit.limit), u = PLAIN ? up : fminf(fmaxf(up, -unit.limit), unit.limit);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * (PLAIN ? -F8_LOG2E : -F8_LOG2E * unit.alpha)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));      // (0 from 2^126 on: the unit of a gate below -87 is 0)
  return g * r * (PLAIN ? u : u + unit.shift);
}

// `shift`: block = 2^shift, or -1. WAY 0: sixteen columns start on 32-byte boundaries and lie within a run of `block`; 1: four
// columns lie within one (or the layout is plain, block = width); 2: any.
template <typename T, int WAY, bool PLAIN>
__global__ void __launch_bounds__(F8_THREADS)
f8_unit_kernel(const T* __restrict__ gu, long long gu_stride, int block, int shift, const GatedUnit unit, const F8Rows o) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * (F8_THREADS / 32) + (threadIdx.x >> 5), word = blockIdx.y;
  if (r >= o.rows) return;
  const int at = word * F8_WORD, left = o.width - at;
  const T* row = gu + (size_t)r * gu_stride;
  uint8_t* q = o.q + (size_t)r * o.pitch + at;
  uint32_t* w = o.words + (size_t)word * o.rows + r;
  const bool whole = block == o.width;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if (WAY == 0) {
    const int c = at + 16 * lane;
    if (16 * lane < left) {
      float g[16];
      const T* p = row + c + (whole ? 0 : shift >= 0 ? c >> shift << shift : c / block * block);
      f8_load16(p, g);
      f8_load16(p + block, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = f8_unit<PLAIN>(unit, g[i], v[i]);
    }
    f8_store_runs(v, 16 * lane < left ? q + 16 * lane : nullptr, w);
    return;
  }
  float g[16];
  if (WAY == 1 && left >= F8_WORD) {      // no branch between the loads: they are in flight together
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = at + 128 * j + 4 * lane;
      const T* p = row + c + (whole ? 0 : shift >= 0 ? c >> shift << shift : c / block * block);
      f8_load4(p, 4, g + 4 * j);
      f8_load4(p + block, 4, v + 4 * j);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = f8_unit<PLAIN>(unit, g[i], v[i]);
    f8_store_fours(v, q, left, w);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = at + 128 * j + 4 * lane, n = o.width - c;
#pragma unroll
    for (int i = 0; i < 4; ++i) g[4 * j + i] = 0.f;
    if (n <= 0) continue;
    if (WAY == 1) {
      const T* p = row + c + (whole ? 0 : shift >= 0 ? c >> shift << shift : c / block * block);
      f8_load4(p, n, g + 4 * j);
      f8_load4(p + block, n, v + 4 * j);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) {
          const T* p = row + c + i + (size_t)((c + i) / block) * block;
          g[4 * j + i] = to_float(p[0]), v[4 * j + i] = to_float(p[block]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + 128 * j + 4 * lane < o.width) {      // (behind the row's end the unit of zeros need not be zero)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[4 * j + i] = at + 128 * j + 4 * lane + i < o.width ? f8_unit<PLAIN>(unit, g[4 * j + i], v[4 * j + i]) : 0.f;
    }
  f8_store_fours(v, q, left, w);
}

// ---- the residual sum and the norm ------------------------------------------------------------------------------------
// h += delta, then h / sqrt(mean(h^2) + eps) * weight in 8 bits; with `rows` row i comes from row rows[i] of h and delta, and h is
// left as it is. A block per row; sums are float32.
__device__ __forceinline__ float f8_block_sum(float v, float4* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  float* at = reinterpret_cast<float*>(red);
  if (lane == 0) at[warp] = v;
  if (warp == 0 && lane >= n) at[lane] = 0.f;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; 4 * i < n; ++i) {
    const float4 r = red[i];
    t += (r.x + r.y) + (r.z + r.w);
  }
  return t;
}

// 1 / sqrt(mean of the squares + eps). NaN where the squares pass float32.
__device__ __forceinline__ float f8_inverse_root(float squares, int width, float eps) {
  return squares < INFINITY ? 1.0f / sqrtf(squares / (float)width + eps) : NAN;
}

// Rows of at most 16,384 numbers: a warp keeps the 512 numbers of its word in registers between the sum and the result.
template <typename T, bool RUNS, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 512 ? 3 : 1)
f8_norm_kernel(float* __restrict__ h, const T* __restrict__ delta, const float* __restrict__ weight, const int* __restrict__ rows,
               int h_rows, float eps, const F8Rows o) {
  __shared__ float4 red[8];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, lane = threadIdx.x & 31, word = threadIdx.x >> 5, from = rows ? rows[r] : r;
  const bool live = from >= 0 && from < h_rows;
  const int at = word * F8_WORD, left = live ? o.width - at : 0;
  float* hr = h + (live ? (size_t)from * o.width + at : 0);
  const T* dr = delta ? delta + (live ? (size_t)from * o.width + at : 0) : nullptr;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if (RUNS) {
    float d[16];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (256 * h + 8 * lane < left) {
        f8_load8(hr + 256 * h + 8 * lane, v + 8 * h);
        if (dr) f8_load8(dr + 256 * h + 8 * lane, d + 8 * h);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (dr && 256 * h + 8 * lane < left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * h + i] += d[8 * h + i];
        if (!rows) f8_put8(hr + 256 * h + 8 * lane, v + 8 * h);
      }
  } else {
    float d[16];
    if (left >= F8_WORD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f8_load4(hr + 128 * j + 4 * lane, 4, v + 4 * j);
      if (dr) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f8_load4(dr + 128 * j + 4 * lane, 4, d + 4 * j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 128 * j + 4 * lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[4 * j + i] = 0.f;
        if (c < left) f8_load4(hr + c, left - c, v + 4 * j);
        if (dr && c < left) f8_load4(dr + c, left - c, d + 4 * j);
      }
    }
    if (dr) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = 128 * (i / 4) + 4 * lane + i % 4;
        v[i] += d[i];
        if (!rows && c < left) hr[c] = v[i];
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
  const float inv = f8_inverse_root(f8_block_sum(ss, red), o.width, eps);
  float wt[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) wt[i] = 0.f;
  if (RUNS) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (256 * h + 8 * lane < left) f8_load8(weight + at + 256 * h + 8 * lane, wt + 8 * h);
  } else {
    if (left >= F8_WORD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f8_load4(weight + at + 128 * j + 4 * lane, 4, wt + 4 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (128 * j + 4 * lane < left) f8_load4(weight + at + 128 * j + 4 * lane, left - 128 * j - 4 * lane, wt + 4 * j);
    }
  }
  const int there = o.width - at;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = RUNS ? 256 * (i / 8) + 8 * lane : 128 * (i / 4) + 4 * lane + i % 4;
    v[i] = c < left ? v[i] * inv * wt[i] : 0.f;      // (inv may be no number)
  }
  uint8_t* q = o.q + (size_t)r * o.pitch + at;
  uint32_t* w = o.words + (size_t)word * o.rows + r;
  if (RUNS)
    f8_store_eights(v, q, there, w);
  else
    f8_store_fours(v, q, there, w);
}

// Longer rows: read again between the two.
constexpr int F8_NORM_THREADS = 512;
template <typename T>
__global__ void __launch_bounds__(F8_NORM_THREADS)
f8_norm_long_kernel(float* __restrict__ h, const T* __restrict__ delta, const float* __restrict__ weight,
                     const int* __restrict__ rows, int h_rows, float eps, const F8Rows o) {
  __shared__ float4 red[8];
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
  const float total = f8_block_sum(ss, red);      // (its barrier also orders the sums above before the loads below)
  const float inv = f8_inverse_root(total, o.width, eps);
  for (int word = warp; word < o.n_words; word += F8_NORM_THREADS / 32) {
    const int at = word * F8_WORD, left = o.width - at;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = at + 128 * (i / 4) + 4 * lane + i % 4;
      v[i] = 0.f;
      if (live && c < o.width) {
        v[i] = hr[c];
        if (dr && rows) v[i] += to_float(dr[c]);
        v[i] = v[i] * inv * weight[c];
      }
    }
    f8_store_fours(v, o.q + (size_t)r * o.pitch + at, left, o.words + (size_t)word * o.rows + r);
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
// Blocks of eight rows and `words` words.
static dim3 f8_grid(const F8Rows& o, int words) {
  return dim3((unsigned)((o.rows - 1) / (F8_THREADS / 32) + 1), (unsigned)((o.n_words - 1) / words + 1));
}

LLMRS_API int llmrs_quantize_fp8(const void* x, int dtype, long long x_stride, int x_rows, const int* src, void* q,
                                 long long pitch, void* words, int rows, int width, cudaStream_t stream) {
  F8Rows o;
  if (const int rc = f8_rows_of(&o, "quantize_fp8", q, pitch, words, rows, width)) return rc;
  if (rows == 0) return 0;
  cudaError_t e;
  if (dtype == LLMRS_F32) {
    auto* k = f8_in_runs(x, x_stride, 4, width) ? f8_quantize_kernel<float, true> : f8_quantize_kernel<float, false>;
    e = llmrs_launch(k, f8_grid(o, 2), dim3(F8_THREADS), 0, stream, true, (const float*)x, x_stride, x_rows, src, o);
  } else if (dtype == LLMRS_BF16) {
    auto* k = f8_in_runs(x, x_stride, 2, width) ? f8_quantize_kernel<__nv_bfloat16, true> : f8_quantize_kernel<__nv_bfloat16, false>;
    e = llmrs_launch(k, f8_grid(o, 2), dim3(F8_THREADS), 0, stream, true, (const __nv_bfloat16*)x, x_stride, x_rows, src, o);
  } else {
    return llmrs_fail("quantize_fp8: unknown dtype %d", dtype);
  }
  if (e != cudaSuccess) return llmrs_fail("quantize_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("quantize_fp8");
}

template <typename T>
static cudaError_t f8_launch_unit(const T* gu, long long gu_stride, int block, const GatedUnit& unit, const F8Rows& o,
                                  cudaStream_t stream) {
  const bool plain = unit.limit == INFINITY && unit.alpha == 1.0f && unit.shift == 0.0f;
  const int shift = block & (block - 1) ? -1 : __builtin_ctz((unsigned)block);
  const int way = block % 16 == 0 && f8_in_runs(gu, gu_stride, (int)sizeof(T), o.width) ? 0 : block == o.width || block % 4 == 0 ? 1 : 2;
  auto* k = way == 0   ? (plain ? f8_unit_kernel<T, 0, true> : f8_unit_kernel<T, 0, false>)
            : way == 1 ? (plain ? f8_unit_kernel<T, 1, true> : f8_unit_kernel<T, 1, false>)
                       : (plain ? f8_unit_kernel<T, 2, true> : f8_unit_kernel<T, 2, false>);
  return llmrs_launch(k, f8_grid(o, 1), dim3(F8_THREADS), 0, stream, true, gu, gu_stride, block, shift, unit, o);
}

// gu [rows, 2 * width]: gate and up in alternating runs of `block` columns (which divides the width).
LLMRS_API int llmrs_silu_mul_fp8(const void* gu, int dtype, long long gu_stride, int block, float limit, float alpha, float shift,
                                 void* q, long long pitch, void* words, int rows, int width, cudaStream_t stream) {
  F8Rows o;
  if (const int rc = f8_rows_of(&o, "silu_mul_fp8", q, pitch, words, rows, width)) return rc;
  LLMRS_REQUIRE(block > 0 && width % block == 0, "silu_mul_fp8: runs of %d columns do not divide %d", block, width);
  if (rows == 0) return 0;
  const GatedUnit unit = {limit, alpha, shift};
  cudaError_t e;
  if (dtype == LLMRS_F32)
    e = f8_launch_unit((const float*)gu, gu_stride, block, unit, o, stream);
  else if (dtype == LLMRS_BF16)
    e = f8_launch_unit((const __nv_bfloat16*)gu, gu_stride, block, unit, o, stream);
  else
    return llmrs_fail("silu_mul_fp8: unknown dtype %d", dtype);
  if (e != cudaSuccess) return llmrs_fail("silu_mul_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("silu_mul_fp8");
}

template <typename T>
static cudaError_t f8_launch_norm(float* h, const T* delta, const float* weight, const int* rows, int h_rows, float eps,
                                  const F8Rows& o, cudaStream_t stream) {
  if (o.n_words > 32)
    return llmrs_launch(f8_norm_long_kernel<T>, dim3(o.rows), dim3(F8_NORM_THREADS), 0, stream, true, h, delta, weight, rows, h_rows,
                        eps, o);
  const bool runs = f8_in_runs(h, o.width, 4, o.width) && ((uintptr_t)weight & 31) == 0 &&
                    (!delta || f8_in_runs(delta, o.width, (int)sizeof(T), o.width));
  auto* k = o.n_words <= 16 ? (runs ? f8_norm_kernel<T, true, 512> : f8_norm_kernel<T, false, 512>)
                            : (runs ? f8_norm_kernel<T, true, 1024> : f8_norm_kernel<T, false, 1024>);
  return llmrs_launch(k, dim3(o.rows), dim3(o.n_words * 32), 0, stream, true,
                      h, delta, weight, rows, h_rows, eps, o);
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
