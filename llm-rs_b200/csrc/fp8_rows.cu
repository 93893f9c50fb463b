// Rows in 8 bits (fp8.cuh) from rows as they are, from a gated unit, and from a residual sum and its norm: what the products of
// gemm_fp8.cu read. All three are bound by memory: a number is read once, its byte written once.
//
// A warp makes 512 numbers of a row, which is one word of scales. Four ways of dealing the numbers to lanes (F8Way):
//   runs    rows of whole sixteens of bfloat16 that start on 32-byte boundaries: a lane takes 16 consecutive numbers (loads of 32
//           bytes, a store of 16); a block's maximum is the maximum over 8 neighbouring lanes
//   fours   rows of whole fours that start on the boundaries of four numbers: 4 consecutive numbers of each of the four blocks
//           (loads of 16 bytes of float32, of 8 of bfloat16; stores of 4); a block's maximum is the maximum over the warp. float32
//           goes this way: a norm's loads and stores of 32 bytes a lane took 41.1 us where those of 16 took 35.3 (4,001 rows of
//           5,120, sums in float32), a float32 unit 21.7 and 18.3 (3,000 rows of 4,112; 18.9 since its gates may be anything)
//   pairs   all other rows: aligned pairs, 32 neighbours a load, moved over by a number where the row starts inside one. Rows of
//           4,095 bfloat16 numbers (8,000 of them) took 25.9 us by unaligned fours, 36 one by one, 20.9 so (15.3 at 6.45 TB/s)
//   ones    every 32nd number: the norm of such rows, whose sums go back where the numbers came from (2,000 rows of 5,001: 32.3 us by
//           unaligned fours, 25.0 so), and units whose columns alternate by a number that is not a multiple of four
// Words that lie whole within a row go without a comparison a number: on odd rows the instructions are what bounds.
#include "fp8.cuh"

constexpr int F8_THREADS = 256;
enum F8Way : int { F8_RUNS = 0, F8_FOURS = 1, F8_PAIRS = 2, F8_ONES = 3 };

// Sixteen consecutive numbers from a 32-byte boundary.
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

// Four consecutive numbers, from a 16-byte (float32) or an 8-byte boundary.
__device__ __forceinline__ void f8_load4(const float* p, float* v) {
  const float4 q = *reinterpret_cast<const float4*>(p);
  v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
}
__device__ __forceinline__ void f8_load4(const __nv_bfloat16* p, float* v) {
  const uint2 q = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(q.x << 16), v[1] = __uint_as_float(q.x & 0xffff0000u);
  v[2] = __uint_as_float(q.y << 16), v[3] = __uint_as_float(q.y & 0xffff0000u);
}

// This lane's share of a warp's 512 numbers, the first of which is *at(0), by fours or one by one; `left` numbers of the row are left
// (FULL: all of them, which saves a comparison a number).
template <int WAY, bool FULL, typename At>
__device__ __forceinline__ void f8_load(const At& at, int left, float (&v)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 16; i += WAY == F8_FOURS ? 4 : 1) {
    if (WAY == F8_FOURS && (FULL || 32 * i + 4 * lane < left)) f8_load4(at(32 * i + 4 * lane), v + i);
    if (WAY == F8_ONES && (FULL || 32 * i + lane < left)) v[i] = to_float(*at(32 * i + lane));
  }
}
// By pairs, from any address: aligned pairs are loaded; where the row starts in the middle of one, a lane's second number is the first
// of the next lane's.
template <bool FULL>
__device__ __forceinline__ void f8_load_pairs(const __nv_bfloat16* p, int left, float (&v)[16]) {
  const int lane = threadIdx.x & 31, odd = (int)((uintptr_t)p >> 1) & 1;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p - odd);
  uint32_t r[9];
#pragma unroll
  for (int i = 0; i < 9; ++i)
    r[i] = (FULL || max(2 * (32 * i + lane) - odd, 0) < left) && (i < 8 || lane < odd) ? __ldg(w + 32 * i + lane) : 0u;
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __funnelshift_r(r[i], __shfl_sync(0xffffffffu, lane == 0 ? r[i + 1] : r[i], lane + 1), 16);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = 64 * i + 2 * lane;
    v[2 * i] = FULL || n < left ? __uint_as_float(r[i] << 16) : 0.f;
    v[2 * i + 1] = FULL || n + 1 < left ? __uint_as_float(r[i] & 0xffff0000u) : 0.f;
  }
}
template <bool FULL>
__device__ __forceinline__ void f8_load_pairs(const float* p, int left, float (&v)[16]) {
  const int lane = threadIdx.x & 31, odd = (int)((uintptr_t)p >> 2) & 1;
  const float2* w = reinterpret_cast<const float2*>(p - odd);
  float2 r[9];
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    r[i] = make_float2(0.f, 0.f);
    if ((FULL || max(2 * (32 * i + lane) - odd, 0) < left) && (i < 8 || lane < odd)) r[i] = __ldg(w + 32 * i + lane);
  }
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = make_float2(r[i].y, __shfl_sync(0xffffffffu, lane == 0 ? r[i + 1].x : r[i].x, lane + 1));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = 64 * i + 2 * lane;
    v[2 * i] = FULL || n < left ? r[i].x : 0.f;
    v[2 * i + 1] = FULL || n + 1 < left ? r[i].y : 0.f;
  }
}

// The warp's 512 numbers, of which `left` are there: v[4 j + i] is number 128 j + 4 lane + i (fours), 128 j + 64 (i / 2) + 2 lane + i % 2
// (pairs), 128 j + 32 i + lane (ones). Room behind a row's end, which reaches to the next multiple of 16, may be written.
template <int WAY, bool FULL>
__device__ __forceinline__ void f8_store(float (&v)[16], uint8_t* q, int left, uint32_t* word) {
  const int lane = threadIdx.x & 31;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float* x = v + 4 * j;
    // The bits of magnitudes are ordered as whole numbers, whose maximum over a warp is one instruction (a NaN counts as 0).
    const float own = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))), 0.f);
    const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(own)));
    const uint32_t byte = f8_scale_byte(top);
    const float inv = f8_inverse(byte);
    w |= byte << (8 * j);
    uint32_t p = f8_pack2(x[0] * inv, x[1] * inv) | f8_pack2(x[2] * inv, x[3] * inv) << 16;
    if (isinf(top)) p = f8_pack2_any(x[0] * inv, x[1] * inv) | f8_pack2_any(x[2] * inv, x[3] * inv) << 16;
    if (WAY == F8_FOURS) {
      if (FULL || 128 * j + 4 * lane < left) *reinterpret_cast<uint32_t*>(q + 128 * j + 4 * lane) = p;
    } else if (WAY == F8_PAIRS) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = 128 * j + 64 * h + 2 * lane;
        if (FULL || n < left) *reinterpret_cast<uint16_t*>(q + n) = (uint16_t)(p >> (16 * h));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (FULL || 128 * j + 32 * i + lane < left) q[128 * j + 32 * i + lane] = (uint8_t)(p >> (8 * i));
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
// Row r from row src[r] (or r) of x; a row whose source is none of x's becomes zeros. By runs a warp makes two words of a row, so that
// the loads of both are in flight (7,211 rows of 4,096 bfloat16 numbers: 16.1 us with one, 15.0 with two; 13.8 at 6.45 TB/s). The other
// ways are bound by their instructions.
template <typename T, int WAY, bool FULL>
__device__ __forceinline__ void f8_quantize_word(const T* x, int left, uint8_t* q, int q_left, uint32_t* word) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if constexpr (WAY == F8_PAIRS)
    f8_load_pairs<FULL>(x, left, v);
  else
    f8_load<WAY, FULL>([&](int c) { return x + c; }, left, v);
  f8_store<WAY, FULL>(v, q, q_left, word);
}

template <typename T, int WAY>
__global__ void __launch_bounds__(F8_THREADS)
f8_quantize_kernel(const T* __restrict__ x, long long x_stride, int x_rows, const int* __restrict__ src, const F8Rows o) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * (F8_THREADS / 32) + (threadIdx.x >> 5);      // a block: a word, or two, of eight rows
  if (r >= o.rows) return;
  const int from = src ? src[r] : r;
  const bool live = from >= 0 && from < x_rows;
  const T* xr = x + (live ? (size_t)from * x_stride : 0);
  if constexpr (WAY != F8_RUNS) {
    const int at = blockIdx.y * F8_WORD, q_left = o.width - at;
    uint8_t* q = o.q + (size_t)r * o.pitch + at;
    uint32_t* w = o.words + (size_t)blockIdx.y * o.rows + r;
    if (live && q_left >= F8_WORD)
      f8_quantize_word<T, WAY, true>(xr + at, q_left, q, q_left, w);
    else
      f8_quantize_word<T, WAY, false>(xr + at, live ? q_left : 0, q, q_left, w);
  } else {
    float v[2][16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = (2 * blockIdx.y + h) * F8_WORD, left = live ? o.width - at : 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[h][i] = 0.f;
      if (16 * lane < left) f8_load16(xr + at + 16 * lane, v[h]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int word = 2 * blockIdx.y + h, left = o.width - word * F8_WORD;
      if (left <= 0) break;
      uint8_t* q = o.q + (size_t)r * o.pitch + word * F8_WORD + 16 * lane;
      f8_store_runs(v[h], 16 * lane < left ? q : nullptr, o.words + (size_t)word * o.rows + r);
    }
  }
}

// ---- the gated unit -------------------------------------------------------------------------------------------------
// GatedUnit in fewer instructions: with t = alpha gate and e = e^(-|t| / 2) the sigmoid of t is 1 / (1 + e^2), times e^2 where t < 0: there
// gate and up are multiplied by e each, so that no product on the way leaves float32 where the result does not (a single
// e^2, or 1 + e^-t, ends at t = -87). The power and the reciprocal are approximate: off by some 2^-21 of itself, and by |t| 2^-23 more
// for t < 0 (the exponent's own rounding), before a rounding of 2^-4; 0 for t < -174, where e^t is below 2^-251. PLAIN is silu(gate) * up.
// What bounded the kernel were these instructions beside the memory: 2,048 rows of 12,288 took 33 us with expf and a division,
// 20.1 as gate / (1 + e^-t), 20.8 with this (19.5 at 6.45 TB/s). A look for gates below -87 in place of it took 20.6 and, where one word in a
// hundred holds one, 21.7 (those numbers again) or 27 (their word again).
constexpr float F8_LOG2E = 1.44269504088896f;      // log2(e)
// The smaller (larger) of two; a NaN where either is one, so that a limit hides none.
__device__ __forceinline__ float f8_min(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float f8_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// SELECT: e or 1 for every number, which float32 rows and numbers one by one hold in fewer registers (float32, 3,000 rows of 4,112: 18.9
// us; 20.7 by branches, which take bfloat16 runs 20.8 where selecting takes 21.0).
template <bool PLAIN, bool SELECT>
__device__ __forceinline__ float f8_unit(const GatedUnit& unit, float gate, float up) {
  float g = PLAIN ? gate : f8_min(gate, unit.limit), u = PLAIN ? up : f8_min(f8_max(up, -unit.limit), unit.limit) + unit.shift;
  const float y = g * (PLAIN ? 0.5f * F8_LOG2E : 0.5f * F8_LOG2E * unit.alpha);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-fabsf(y)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, e, 1.0f)));
  if constexpr (SELECT) {
    e = y < 0.0f ? e : 1.0f;
    g *= e, u *= e;
  } else if (y < 0.0f) {
    g *= e, u *= e;
  }
  return g * r * u;
}

// gate(c): where column c's gate is; its up is `block` further. A lane's sixteen (runs) or four (fours) columns lie within a run of
// `block`; pairs: the layout is plain.
template <typename T, int WAY, bool PLAIN, bool FULL, typename Gate>
__device__ __forceinline__ void f8_unit_word(const Gate& gate, int block, int at, int left, const GatedUnit& unit, uint8_t* q,
                                             uint32_t* word) {
  const int lane = threadIdx.x & 31;
  float g[16], v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = v[i] = 0.f;
  if constexpr (WAY == F8_PAIRS) {
    f8_load_pairs<FULL>(gate(at), left, g);
    f8_load_pairs<FULL>(gate(at) + block, left, v);
  } else {
    f8_load<WAY, FULL>([&](int c) { return gate(at + c); }, left, g);
    f8_load<WAY, FULL>([&](int c) { return gate(at + c) + block; }, left, v);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = WAY == F8_FOURS ? 128 * (i / 4) + 4 * lane : WAY == F8_PAIRS ? 64 * (i / 2) + 2 * lane + i % 2 : 32 * i + lane;
    v[i] = FULL || c < left ? f8_unit<PLAIN, sizeof(T) == 4 || WAY == F8_ONES>(unit, g[i], v[i]) : 0.f;      // (the unit of zeros need not be zero)
  }
  f8_store<WAY, FULL>(v, q, left, word);
}

// `shift`: block = 2^shift, or -1. Blocks an SM at the least (one B200): with eight in place of six, runs of 2,048 x 12,288 take
// 20.4 us in place of 20.8 in a burst, but 23.4 in place of 22.5 where calls follow one another for seconds under the power limit;
// pairs, 4,000 rows of 1,001, 6.5 and 5.8; numbers one by one, 3,000 rows of 4,095, 43.5 with six, 41.4 with five.
template <typename T, int WAY, bool PLAIN>
__global__ void __launch_bounds__(F8_THREADS, sizeof(T) == 4 ? 4 : WAY == F8_ONES ? 5 : 6)
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
  auto gate = [&](int c) { return row + c + (whole ? 0 : shift >= 0 ? c >> shift << shift : c / block * block); };
  if constexpr (WAY == F8_RUNS) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
    if (16 * lane < left) {
      float g[16];
      const T* p = gate(at + 16 * lane);
      f8_load16(p, g);
      f8_load16(p + block, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = f8_unit<PLAIN, false>(unit, g[i], v[i]);
    }
    f8_store_runs(v, 16 * lane < left ? q + 16 * lane : nullptr, w);
  } else if (left >= F8_WORD) {
    f8_unit_word<T, WAY, PLAIN, true>(gate, block, at, left, unit, q, w);
  } else {
    f8_unit_word<T, WAY, PLAIN, false>(gate, block, at, left, unit, q, w);
  }
}

// ---- the residual sum and the norm ------------------------------------------------------------------------------------
// h += delta, then h / sqrt(mean(h^2) + eps) * weight in 8 bits; with `rows` row i comes from row rows[i] of h and delta, and h is
// left as it is. A block per row. The sum of squares is made in double (in float32 a thread's share of a long row errs by many ulps, all
// to one side where its numbers are alike, and passes the type's range long before the mean does), and the result
// is carried in two float32 numbers until it is rounded to float32 once: a number next to a border of e4m3 falls on the formula's side
// of it but for half an ulp of float32 (4,001 rows of 5,120: 37.4 us; 36.9
// with a thread's squares in float32, 34.9 at 6.45 TB/s).
__device__ __forceinline__ double f8_square(float v, double sum) { return fma((double)v, (double)v, sum); }
__device__ __forceinline__ double f8_block_sum(double v, double2* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  double* at = reinterpret_cast<double*>(red);
  if (lane == 0) at[warp] = v;
  if (warp == 0 && lane >= n) at[lane] = 0.0;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; 2 * i < n; ++i) t += red[i].x + red[i].y;
  return t;
}

// 1 / sqrt(mean) as the sum of two float32 numbers: CUDA's approximate root and one Newton step in double (its root in double took 38.5
// us). NaN where the mean of the squares, with the eps, passes float32. Without an eps a small row's mean may lie below float32: the
// row is then normed 2^100 times as large (a branch that a row takes as a whole; always multiplying took 38.1 us).
constexpr float F8_SMALL = 0x1p-100f, F8_UP = 0x1p100f;
struct F8Root { float hi, lo; };
__device__ __forceinline__ F8Root f8_inverse_root(double mean) {
  const double y = rsqrtf((float)mean), root = y > 0.0 ? y * (1.5 - 0.5 * mean * y * y) : (double)NAN;
  F8Root r;
  r.hi = (float)root, r.lo = (float)(root - (double)r.hi);
  return r;
}
// v * root * w, rounded once.
__device__ __forceinline__ float f8_scaled(float v, F8Root root, float w) {
  const float p = v * root.hi, e = fmaf(v, root.lo, fmaf(v, root.hi, -p)), r = p * w;
  return r + fmaf(e, w, fmaf(p, w, -r));
}

// Rows of at most 16,384 numbers: a warp keeps the 512 numbers of its word in registers between the sum and the result.
template <typename T, int WAY, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 512 ? 2 : 1)
f8_norm_kernel(float* __restrict__ h, const T* __restrict__ delta, const float* __restrict__ weight, const int* __restrict__ rows,
               int h_rows, float eps, double per, const F8Rows o) {
  __shared__ double2 red[16];
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
  float d[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) d[i] = 0.f;
  f8_load<WAY, false>([&](int c) { return hr + c; }, left, v);
  if (dr) f8_load<WAY, false>([&](int c) { return dr + c; }, left, d);
  if (dr) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += d[i];
    if (!rows) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (WAY == F8_ONES && 32 * i + lane < left) hr[32 * i + lane] = v[i];
        if (WAY == F8_FOURS && i % 4 == 0 && 32 * i + 4 * lane < left)
          *reinterpret_cast<float4*>(hr + 32 * i + 4 * lane) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
  }
  float wt[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) wt[i] = 0.f;
  f8_load<WAY, false>([&](int c) { return weight + at + c; }, left, wt);
  double ss[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < 16; ++i) ss[i % 4] = f8_square(v[i], ss[i % 4]);      // (one chain of sixteen: 37.6 us)
  double mean = f8_block_sum(ss[0] + ss[1] + (ss[2] + ss[3]), red) * per + (double)eps;
  if ((float)mean < F8_SMALL) {
    mean *= (double)F8_UP * (double)F8_UP;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= F8_UP;
  }
  const F8Root inv = f8_inverse_root(mean);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = WAY == F8_FOURS ? 128 * (i / 4) + 4 * lane : 32 * i + lane;
    v[i] = c < left ? f8_scaled(v[i], inv, wt[i]) : 0.f;      // (inv may be no number)
  }
  f8_store<WAY, false>(v, o.q + (size_t)r * o.pitch + at, o.width - at, o.words + (size_t)word * o.rows + r);
}

// Longer rows: read again between the two.
constexpr int F8_NORM_THREADS = 512;
template <typename T>
__global__ void __launch_bounds__(F8_NORM_THREADS)
f8_norm_long_kernel(float* __restrict__ h, const T* __restrict__ delta, const float* __restrict__ weight,
                     const int* __restrict__ rows, int h_rows, float eps, double per, const F8Rows o) {
  __shared__ double2 red[16];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, from = rows ? rows[r] : r, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool live = from >= 0 && from < h_rows;
  float* hr = h + (live ? (size_t)from * o.width : 0);
  const T* dr = delta && live ? delta + (size_t)from * o.width : nullptr;
  double ss = 0.0;
  if (live)
    for (int c = threadIdx.x; c < o.width; c += F8_NORM_THREADS) {
      float v = hr[c];
      if (dr) {
        v += to_float(dr[c]);
        if (!rows) hr[c] = v;
      }
      ss = f8_square(v, ss);
    }
  double mean = f8_block_sum(ss, red) * per + (double)eps;      // (its barrier also orders the sums above before the loads below)
  const float up = (float)mean < F8_SMALL ? F8_UP : 1.0f;
  mean *= (double)up * (double)up;
  const F8Root inv = f8_inverse_root(mean);
  for (int word = warp; word < o.n_words; word += F8_NORM_THREADS / 32) {
    const int at = word * F8_WORD, left = o.width - at;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int c = at + 32 * i + lane;
      v[i] = 0.f;
      if (live && c < o.width) {
        v[i] = hr[c];
        if (dr && rows) v[i] += to_float(dr[c]);
        v[i] = f8_scaled(v[i] * up, inv, weight[c]);
      }
    }
    f8_store<F8_ONES, false>(v, o.q + (size_t)r * o.pitch + at, left, o.words + (size_t)word * o.rows + r);
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
// How rows that are `stride` numbers of `size` bytes apart may be dealt.
static F8Way f8_way(const void* x, long long stride, int size, int width) {
  const long long at = (long long)(uintptr_t)x | stride * size;
  return size == 2 && width % 16 == 0 && at % 32 == 0 ? F8_RUNS : width % 4 == 0 && at % (4 * size) == 0 ? F8_FOURS : F8_PAIRS;
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
    auto* k = f8_way(x, x_stride, 4, width) == F8_FOURS ? f8_quantize_kernel<float, F8_FOURS> : f8_quantize_kernel<float, F8_PAIRS>;
    e = llmrs_launch(k, f8_grid(o, 1), dim3(F8_THREADS), 0, stream, true, (const float*)x, x_stride, x_rows, src, o);
  } else if (dtype == LLMRS_BF16) {
    const F8Way way = f8_way(x, x_stride, 2, width);
    auto* k = way == F8_RUNS    ? f8_quantize_kernel<__nv_bfloat16, F8_RUNS>
              : way == F8_FOURS ? f8_quantize_kernel<__nv_bfloat16, F8_FOURS>
                                : f8_quantize_kernel<__nv_bfloat16, F8_PAIRS>;
    e = llmrs_launch(k, f8_grid(o, way == F8_RUNS ? 2 : 1), dim3(F8_THREADS), 0, stream, true, (const __nv_bfloat16*)x, x_stride, x_rows, src, o);
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
  F8Way way = f8_way(gu, gu_stride, (int)sizeof(T), o.width);
  if (way == F8_RUNS && block % 16) way = F8_FOURS;
  if ((way == F8_FOURS && block % 4) || (way == F8_PAIRS && block != o.width)) way = F8_ONES;
  auto* k = way == F8_FOURS   ? (plain ? f8_unit_kernel<T, F8_FOURS, true> : f8_unit_kernel<T, F8_FOURS, false>)
            : way == F8_PAIRS ? (plain ? f8_unit_kernel<T, F8_PAIRS, true> : f8_unit_kernel<T, F8_PAIRS, false>)
                              : (plain ? f8_unit_kernel<T, F8_ONES, true> : f8_unit_kernel<T, F8_ONES, false>);
  if constexpr (sizeof(T) == 2)
    if (way == F8_RUNS) k = plain ? f8_unit_kernel<T, F8_RUNS, true> : f8_unit_kernel<T, F8_RUNS, false>;
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
  const double per = 1.0 / o.width;
  if (o.n_words > 32)
    return llmrs_launch(f8_norm_long_kernel<T>, dim3(o.rows), dim3(F8_NORM_THREADS), 0, stream, true, h, delta, weight, rows, h_rows,
                        eps, per, o);
  const bool fours = f8_way(h, o.width, 4, o.width) != F8_PAIRS && ((uintptr_t)weight & 15) == 0 &&
                     (!delta || f8_way(delta, o.width, (int)sizeof(T), o.width) != F8_PAIRS);
  auto* k = o.n_words <= 16 ? (fours ? f8_norm_kernel<T, F8_FOURS, 512> : f8_norm_kernel<T, F8_ONES, 512>)
                            : (fours ? f8_norm_kernel<T, F8_FOURS, 1024> : f8_norm_kernel<T, F8_ONES, 1024>);
  return llmrs_launch(k, dim3(o.rows), dim3(o.n_words * 32), 0, stream, true,
                      h, delta, weight, rows, h_rows, eps, per, o);
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
