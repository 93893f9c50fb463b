// Products of rows in 8 bits (fp8.cuh) on tcgen05: y[t, n] = sum_b 2^(Ex[t, b] + Ew[n, b]) * sum_{k in block b} x[t, k] * w[n, k],
// dense or grouped by expert (rows sorted by group, a list of tiles of rows, each group's own weights).
//
// The scales are powers of two, which tcgen05.mma.kind::mxf8f6f4.block_scale applies itself: the sums stay in tensor memory in
// float32 over the whole of k and nothing is promoted on the CUDA cores. A block of 128 numbers is four MMAs of k = 32 that name
// the same byte of a row's word of scales; a word serves four blocks.
//
// The weights are the M side whatever the number of tokens is, the tokens the N side: an MMA is as wide as the tile's rows, in
// steps of 16, so that few tokens and a group's ragged end cost what they have. One thread copies by TMA, one issues the MMAs;
// four warps move the words of scales from memory to tensor memory (a warp can write the 32 lanes that its index modulo 4 names,
// and the MMA wants every word in all four quarters). In the epilogue a lane holds a feature, a column a token. Two kernels:
//   few tokens   tiles of 128 features by up to NT tokens, a block each, two blocks an SM; with few tiles the range of k is split
//                over a cluster of blocks that send their sums to the block that adds them up, in the order of the ranks. Bound by
//                the stream of the weights.
//   many tokens  tiles of 256 features by 256 tokens on pairs of SMs (cta_group::2), walked by a pair per two SMs; a tile's stores
//                run under the next one's MMAs. Bound by the tensor cores.
//
// Every wait is bounded (see gemm_tcgen05.cu): a block that gives up drains its copies and MMAs, records a code in *error_flag,
// frees its tensor memory and returns.
#include <atomic>

#include "fp8.cuh"
#include "tcgen05_util.cuh"

uint32_t llmrs_tc_wait_limit();
int llmrs_tc_skipped_copy();

constexpr int G8_BM = 128, G8_BK = 128;              // features a block's tile, bytes of k a stage
constexpr uint32_t G8_A_BYTES = G8_BM * G8_BK;
constexpr int G8_SLOTS = 4;                          // words of scales (of 512 numbers each) under way in tensor memory

enum G8Epilogue : int { G8_STORE = 0, G8_ADD = 1 };

struct G8Params {
  void* out;
  long long ldo;
  int out_f32, epilogue, vec, vec4;      // rows of out start at multiples of 16 bytes, of four numbers
  const uint32_t* xs;      // word g of row r: xs[g * xs_stride + r]
  const uint32_t* ws;
  long long xs_stride, ws_stride;
  int x_rows, w_rows;      // rows of x; rows of all groups' weights
  int N, n_f, n_t, nkb;    // features a group, tiles of features, tiles of tokens (dense), blocks of k
  int nt, x_box, stages;   // tokens a tile, rows of x that a copy brings; few tokens: stages of the ring
  const int* tiles;        // grouped: [tile][3] = group, first row, rows; null: dense
  const int* n_tiles;
  int max_tiles, groups;
  int* error_flag;
  uint32_t wait_limit;
  int test_skip_kb;
};

// Instruction descriptor: e4m3 x e4m3 with E8M0 scales, both K-major, M = 128 (or 256 over a pair); `byte` of the words of scales.
__device__ __forceinline__ uint32_t g8_idesc(int m, int n, int byte) {
  return (1u << 23) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)byte << 4) | ((uint32_t)byte << 29);
}
__device__ __forceinline__ void g8_mma(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa, uint32_t sb,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void g8_st4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
// 16 consecutive float32 columns of this thread's lane.
__device__ __forceinline__ void g8_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void g8_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t g8_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t g8_map_rank(uint32_t local_addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
  return remote;
}
// Whether `ok` holds in all of 128 threads (four warps; barrier 1).
__device__ __forceinline__ bool g8_all_of_four(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}
__device__ __forceinline__ void g8_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void g8_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// (In line throughout: a call would make a role's registers spill.)
__device__ __forceinline__ bool g8_wait(uint32_t bar, uint32_t parity, uint32_t limit, volatile int* abort_flag) {
  return mbar_try_wait(bar, parity) || mbar_wait(bar, parity, limit, abort_flag);
}
__device__ __forceinline__ void g8_prefetch(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void g8_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// A stage of the ring of copies, or a slot of the ring of scales, and the parity of its barriers' phase.
struct G8Ring {
  int size, at;
  uint32_t phase;
  __device__ __forceinline__ explicit G8Ring(int n) : size(n), at(0), phase(0) {}
  __device__ __forceinline__ void next() {
    const bool wrap = ++at == size;
    at = wrap ? 0 : at;
    phase ^= wrap ? 1u : 0u;
  }
};

// The tile of work item t: group, first row of x, rows, first feature (tiles of `bm` features).
struct G8Tile { int group, m0, rows, f0; };
__device__ __forceinline__ G8Tile g8_tile(const G8Params& p, int t, int n_row_tiles, int bm) {
  const int f = t / n_row_tiles, i = t - f * n_row_tiles;
  G8Tile w;
  w.f0 = f * bm;
  if (p.tiles) {
    w.group = p.tiles[3 * i], w.m0 = p.tiles[3 * i + 1], w.rows = min(p.tiles[3 * i + 2], p.nt);
    if (w.group < 0 || w.group >= p.groups || w.m0 < 0 || w.m0 >= p.x_rows || w.rows < 0)
      w.group = w.m0 = w.rows = 0;      // names what is not there: nothing is computed for it
    w.rows = min(w.rows, p.x_rows - w.m0);
  } else {
    w.group = 0, w.m0 = i * p.nt, w.rows = min(p.nt, p.x_rows - w.m0);
  }
  return w;
}

// A lane's words of scales of some steps of 512 numbers: of the features w_row + lane + 32 j and of the tokens m0 + lane + 32 j.
template <int NT> struct G8Words {
  static constexpr int STEPS = NT > 128 ? 2 : 4;
  uint32_t w[STEPS][4], x[STEPS][NT > 128 ? 8 : 4];
};
template <int NT>
__device__ __forceinline__ void g8_load_words(const G8Params& p, int w_row, int m0, int base, int g1, int lane, G8Words<NT>& o) {
#pragma unroll
  for (int u = 0; u < G8Words<NT>::STEPS; ++u) {
    const int g = min(base + u, g1 - 1);
    const uint32_t* wg = p.ws + (size_t)g * p.ws_stride;
    const uint32_t* xg = p.xs + (size_t)g * p.xs_stride;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.w[u][j] = __ldg(wg + min(w_row + lane + 32 * j, p.w_rows - 1));
#pragma unroll
    for (int j = 0; j < (NT > 128 ? 8 : 4); ++j) o.x[u][j] = 32 * j < NT ? __ldg(xg + min(m0 + lane + 32 * j, p.x_rows - 1)) : 0u;
  }
}
// Words u of them into the slot at `taddr` (this warp's lanes): the features' in columns 0-3, the tokens' from 4 on.
template <int NT>
__device__ __forceinline__ void g8_put_words(const G8Words<NT>& o, int u, uint32_t taddr) {
  g8_st4(taddr, o.w[u]);
#pragma unroll
  for (int h = 0; h < (NT > 128 ? 2 : 1); ++h) {
    const uint32_t x[4] = {o.x[u][4 * h], o.x[u][4 * h + 1], o.x[u][4 * h + 2], o.x[u][4 * h + 3]};
    g8_st4(taddr + 4 + 4 * h, x);
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  tc_fence_before();
  __syncwarp();
}

// Column c of `v` is token row + c of feature n; `count` columns are there.
template <int COLS>
__device__ __forceinline__ void g8_store(const G8Params& p, int row, int n, int count, const float (&v)[COLS]) {
  const size_t at = (size_t)row * p.ldo + n;
  if (p.epilogue == G8_ADD) {
    float* o = (float*)p.out + at;
    constexpr int STEP = COLS < 8 ? COLS : 8;      // loads in flight together
#pragma unroll
    for (int c = 0; c < COLS; c += STEP) {
      float h[STEP];
      const float* i = o;
#pragma unroll
      for (int e = 0; e < STEP; ++e, i += p.ldo) h[e] = c + e < count ? *i : 0.f;
#pragma unroll
      for (int e = 0; e < STEP; ++e, o += p.ldo)
        if (c + e < count) *o = h[e] + v[c + e];
    }
  } else if (p.out_f32) {
    float* o = (float*)p.out + at;
#pragma unroll
    for (int e = 0; e < COLS; ++e, o += p.ldo)
      if (e < count) *o = v[e];
  } else {
    __nv_bfloat16* o = (__nv_bfloat16*)p.out + at;
#pragma unroll
    for (int e = 0; e < COLS; ++e, o += p.ldo)
      if (e < count) *o = __float2bfloat16_rn(v[e]);
  }
}

// Features n .. n + 3 of a token.
__device__ __forceinline__ void g8_store4(const G8Params& p, int row, int n, float4 v) {
  const size_t at = (size_t)row * p.ldo + n;
  const float x[4] = {v.x, v.y, v.z, v.w};
  const int left = p.N - n;
  if (p.out_f32) {
    float* o = (float*)p.out + at;
    if (p.vec4 && left >= 4) {
      if (p.epilogue == G8_ADD) {
        const float4 h = *reinterpret_cast<const float4*>(o);
        v.x += h.x, v.y += h.y, v.z += h.z, v.w += h.w;
      }
      *reinterpret_cast<float4*>(o) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) o[e] = p.epilogue == G8_ADD ? o[e] + x[e] : x[e];
    }
  } else {
    __nv_bfloat16* o = (__nv_bfloat16*)p.out + at;
    if (p.vec4 && left >= 4) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) o[e] = __float2bfloat16_rn(x[e]);
    }
  }
}

// The bfloat16 results of a warp's 32 features (from f0) for 64 tokens (from `row`, of which `count` are there), through 4 KB of
// shared memory: a lane holds a feature (two tokens a register), a store takes 16 bytes of a token's row. Stores of a number a lane,
// 64 bytes a warp, took longer than a short tile's products.
constexpr int G8_STAGE_TOKENS = 64;
constexpr uint32_t G8_STAGED_BYTES = G8_STAGE_TOKENS * 64;
template <int PAIRS>
__device__ __forceinline__ void g8_store_staged(const G8Params& p, unsigned char* buf, int lane, int row, int f0, int count,
                                                const __nv_bfloat162 (&v)[PAIRS], int first) {
#pragma unroll
  for (int e = 0; e < G8_STAGE_TOKENS / 2; ++e) {
    *reinterpret_cast<__nv_bfloat16*>(buf + (2 * e) * 64 + 2 * lane) = v[first + e].x;
    *reinterpret_cast<__nv_bfloat16*>(buf + (2 * e + 1) * 64 + 2 * lane) = v[first + e].y;
  }
  __syncwarp();
  const int n = f0 + lane % 4 * 8, left = p.N - n;
  __nv_bfloat16* o = (__nv_bfloat16*)p.out + (size_t)(row + lane / 4) * p.ldo + n;
#pragma unroll
  for (int i = 0; i < G8_STAGE_TOKENS / 8; ++i, o += 8 * p.ldo) {
    if (8 * i + lane / 4 >= count) continue;
    const uint4 q = *reinterpret_cast<const uint4*>(buf + 512 * i + 16 * lane);
    if (left >= 8) {
      *reinterpret_cast<uint4*>(o) = q;
    } else {
      const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&q);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) o[e] = h[e];
    }
  }
  __syncwarp();
}

// ---- few tokens -------------------------------------------------------------------------------------------------------
constexpr int G8F_THREADS = 192, G8_MAX_SPLITS = 8;

template <int NT> struct G8Few {
  static constexpr uint32_t STAGE_BYTES = G8_A_BYTES + NT * G8_BK;
  static constexpr int MAX_STAGES = 12;
  // Split: NT tokens' sums, rounded up to whole shares.
  static constexpr uint32_t SUM_BYTES = (NT + G8_MAX_SPLITS - 1) * G8_BM * 4;
  static constexpr int ACC_COLS = NT < 32 ? 32 : NT, SLOT_COLS = 8, COLS = ACC_COLS + G8_SLOTS * SLOT_COLS <= 64    ? 64
                                                                          : ACC_COLS + G8_SLOTS * SLOT_COLS <= 128 ? 128
                                                                                                                   : 256;
  // full[S], empty[S], scales_full[4], scales_empty[4], acc_full, received, drain
  static constexpr int BARS = 2 * MAX_STAGES + 2 * G8_SLOTS + 3;
  static constexpr size_t FIXED = 1024 + BARS * 8 + 16;
  static size_t smem(int stages, int splits) { return FIXED + (size_t)stages * STAGE_BYTES + (splits > 1 ? SUM_BYTES : 0); }
};

template <int NT>
__global__ void __launch_bounds__(G8F_THREADS, 2)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const G8Params p) {
  using C = G8Few<NT>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* stages = reinterpret_cast<unsigned char*>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);
  const int splits = (int)gridDim.z, split = (int)blockIdx.z;      // the blocks of a cluster share a tile's range of k
  // Split: this block's sums (once the stages are free) and, [rank][token of its share][feature], what the others send.
  float* own = reinterpret_cast<float*>(stages);
  float* sums = reinterpret_cast<float*>(stages + (size_t)p.stages * C::STAGE_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<unsigned char*>(sums) + (splits > 1 ? C::SUM_BYTES : 0));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* sent = abort_flag + 1;      // split: this block's sums have been sent
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t full0 = tc_smem(bars), empty0 = full0 + 8 * C::MAX_STAGES, sc_full0 = empty0 + 8 * C::MAX_STAGES,
                 sc_empty0 = sc_full0 + 8 * G8_SLOTS, acc_full = sc_empty0 + 8 * G8_SLOTS, received = acc_full + 8,
                 drain_bar = received + 8;
  const int kb0 = (int)((long long)split * p.nkb / splits), kb1 = (int)((long long)(split + 1) * p.nkb / splits);

  pdl_launch_dependents();
  if (warp == 0) {      // a barrier or two a lane (one lane for all of them took 700 cycles)
    for (int s = lane; s < C::BARS; s += 32) {
      const uint32_t bar = full0 + 8 * s;
      mbar_init(bar, bar >= sc_full0 && bar < sc_empty0 ? 4 : bar == received ? 2 : 1);
    }
    if (lane == 0) {
      g8_prefetch_map(&map_w);
      g8_prefetch_map(&map_x);
      *abort_flag = *sent = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  } else if (tid == 64 && !p.tiles) {
    // The first weights on their way into the L2 while the kernel before this one ends (a hint: they are copied only after it).
    for (int kb = kb0; kb < kb1 && kb < kb0 + 2 * p.stages; ++kb) g8_prefetch(&map_w, kb * G8_BK, (int)blockIdx.x / p.n_t * G8_BM);
  }
  __syncthreads();
  if (splits > 1) g8_cluster_arrive();
  pdl_wait();      // everything below reads or writes what earlier kernels may have touched
  const int n_row_tiles = p.tiles ? min(*p.n_tiles, p.max_tiles) : p.n_t;
  if (blockIdx.x >= (long long)n_row_tiles * p.n_f) {      // a list's tiles may be fewer than the grid has room for; the whole cluster
    if (splits > 1) g8_cluster_wait();
    return;
  }
  // Tensor memory is asked for after the wait: a block that held some while it waits for an earlier kernel could keep that kernel's
  // blocks from theirs. The copies start meanwhile.
  uint32_t tmem_base = 0;
  if (warp >= 1) {
    if (warp == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_slot)), "r"(C::COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    asm volatile("bar.sync 2, %0;" ::"n"(G8F_THREADS - 32) : "memory");
    tc_fence_after();
    tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  }
  const uint32_t tmem_scales = tmem_base + C::ACC_COLS;
  const G8Tile w = g8_tile(p, blockIdx.x, n_row_tiles, G8_BM);
  const int w_row = w.group * p.N + w.f0;
  int copies = 0;      // warp 0: stages whose copies it has requested
  // Split: the split-th share of the tile's tokens is this block's to add up.
  const int share = (w.rows + splits - 1) / splits, mine = max(min(share, w.rows - split * share), 0);
  bool met = false;
  if (splits > 1 && tid == 0) mbar_expect_tx(received, (uint32_t)((splits - 1) * mine) * G8_BM * 4);      // from the other blocks

  if (w.rows == 0) {
    // nothing to compute
  } else if (warp == 0) {
    if (tc_elect_one()) {
      const int boxes = (w.rows + p.x_box - 1) / p.x_box;
      const uint32_t bytes = G8_A_BYTES + (uint32_t)(boxes * p.x_box) * G8_BK;
      G8Ring r(p.stages);
      for (int kb = kb0; kb < kb1; ++kb, ++copies, r.next()) {
        if (!g8_wait(empty0 + 8 * r.at, r.phase ^ 1, p.wait_limit, abort_flag)) break;
        if (kb == p.test_skip_kb) continue;
        const uint32_t bar = full0 + 8 * r.at, dst = tc_smem(stages) + (uint32_t)r.at * C::STAGE_BYTES;
        mbar_expect_tx(bar, bytes);
        tma_load_2d(dst, &map_w, bar, kb * G8_BK, w_row);
        tma_load_2d(dst + G8_A_BYTES, &map_x, bar, kb * G8_BK, w.m0);
        for (int b = 1; b < boxes; ++b)      // (ragged tiles)
          tma_load_2d(dst + G8_A_BYTES + (uint32_t)(b * p.x_box) * G8_BK, &map_x, bar, kb * G8_BK, w.m0 + b * p.x_box);
      }
    }
    __syncwarp();
    copies = __reduce_max_sync(0xffffffffu, copies);
  } else if (warp == 1) {
    if (tc_elect_one()) {
      const uint32_t idesc0 = g8_idesc(G8_BM, (w.rows + 15) & ~15, 0);
      G8Ring r(p.stages);
      G8Ring sc(G8_SLOTS);
      bool ok = true;
      uint32_t acc = 0;
      for (int g = kb0 / 4; 4 * g < kb1 && ok; ++g, sc.next()) {      // a word of scales
        ok = g8_wait(sc_full0 + 8 * sc.at, sc.phase, p.wait_limit, abort_flag);
        const uint32_t sa = tmem_scales + (uint32_t)(sc.at * C::SLOT_COLS);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (4 * g + j < kb0 || 4 * g + j >= kb1 || !ok) continue;
          ok = g8_wait(full0 + 8 * r.at, r.phase, p.wait_limit, abort_flag);
          if (!ok) continue;
          tc_fence_after();
          const uint32_t a_addr = tc_smem(stages) + (uint32_t)r.at * C::STAGE_BYTES, idesc = idesc0 | g8_idesc(0, 0, j);
          const uint64_t a_desc = tc_smem_desc(a_addr), b_desc = tc_smem_desc(a_addr + G8_A_BYTES);
#pragma unroll
          for (int k = 0; k < G8_BK / 32; ++k) {
            g8_mma(tmem_base, a_desc + (uint64_t)(k * 2), b_desc + (uint64_t)(k * 2), idesc, sa, sa + 4, acc);
            acc = 1;
          }
          tc_commit(empty0 + 8 * r.at);
          r.next();
        }
        tc_commit(sc_empty0 + 8 * sc.at);
      }
      if (ok) tc_commit(acc_full);
    }
    __syncwarp();
  } else {
    // Words of scales. Four words a row are asked for at a time, and the next four before these are stored: a word at a time
    // waited for the memory's latency every 512 numbers.
    const int quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int g1 = (kb1 + 3) / 4;
    G8Words<NT> now, next;
    int base = kb0 / 4;
    g8_load_words<NT>(p, w_row, w.m0, base, g1, lane, now);
    G8Ring sc(G8_SLOTS);
    bool ok = true;
    while (base < g1 && ok) {
      if (base + 4 < g1) g8_load_words<NT>(p, w_row, w.m0, base + 4, g1, lane, next);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (base + u >= g1 || !ok) continue;
        ok = __all_sync(0xffffffffu, g8_wait(sc_empty0 + 8 * sc.at, sc.phase ^ 1, p.wait_limit, abort_flag));
        if (!ok) continue;
        tc_fence_after();
        g8_put_words<NT>(now, u, tmem_scales + (uint32_t)(sc.at * C::SLOT_COLS) + lanes);
        if (lane == 0) g8_arrive(sc_full0 + 8 * sc.at);
        sc.next();
      }
      now = next, base += 4;
    }
    // The epilogue.
    constexpr int CH = NT < 32 ? NT : 32;
    const int f = quarter * 32 + lane, n = w.f0 + f;
    ok = ok && __all_sync(0xffffffffu, g8_wait(acc_full, 0, p.wait_limit, abort_flag));
    if (ok) tc_fence_after();
    if (splits == 1) {
      if (p.vec && !p.out_f32 && NT >= 64) {
        for (int c = 0; c < w.rows && ok; c += G8_STAGE_TOKENS) {      // the stages are free: every MMA of the block has been done
          __nv_bfloat162 keep[G8_STAGE_TOKENS / 2];
#pragma unroll
          for (int h = 0; h < G8_STAGE_TOKENS; h += 32) {
            float v[32];
            tc_ld32(tmem_base + lanes + c + h, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) keep[h / 2 + e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
          }
          g8_store_staged(p, stages + quarter * G8_STAGED_BYTES, lane, w.m0 + c, n - lane, w.rows - c, keep, 0);
        }
      } else {
        for (int c = 0; c < w.rows && ok; c += CH) {      // all lanes: the reads are warp-wide
          float v[32];
          tc_ld32(tmem_base + lanes + c, v);
          if (n < p.N) g8_store<CH>(p, w.m0 + c, n, w.rows - c, reinterpret_cast<float (&)[CH]>(v));
          __syncwarp();
        }
      }
    } else {
      // This block's sums into its own (free) stages, [token][feature].
      for (int c = 0; c < w.rows && ok; c += CH) {
        float v[32];
        tc_ld32(tmem_base + lanes + c, v);
        float* to = own + (size_t)c * G8_BM + f;
#pragma unroll
        for (int e = 0; e < CH; ++e) to[e * G8_BM] = v[e];
        __syncwarp();
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      ok = g8_all_of_four(ok);
      g8_cluster_wait();      // every block of the cluster runs: what it is sent has a place
      met = true;
      if (ok && warp == 2 && tc_elect_one()) {
        *sent = 1;
        g8_arrive(received);      // this block's own share is there
        for (int r = 0; r < splits; ++r) {
          const int theirs = min(share, w.rows - r * share);
          if (r == split || theirs <= 0) continue;
          asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(g8_map_rank(tc_smem(sums + (size_t)split * share * G8_BM), (uint32_t)r)),
                       "r"(tc_smem(own + (size_t)r * share * G8_BM)), "r"((uint32_t)theirs * G8_BM * 4),
                       "r"(g8_map_rank(received, (uint32_t)r))
                       : "memory");
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  if (splits > 1) {
    if (!met) g8_cluster_wait();
    if (mine > 0) {
      // The other blocks' sums of this block's tokens: a warp adds up a token's 128 features, four a lane.
      const bool all = __all_sync(0xffffffffu, g8_wait(received, 0, p.wait_limit, abort_flag));
      const int n = w.f0 + 4 * lane;
      for (int j = warp; j < mine && all; j += G8F_THREADS / 32) {
        const float4* from = reinterpret_cast<const float4*>(sums + (size_t)j * G8_BM) + lane;
        const float4 kept = reinterpret_cast<const float4*>(own + (size_t)(split * share + j) * G8_BM)[lane];
        float4 part[G8_MAX_SPLITS];
#pragma unroll
        for (int r = 0; r < G8_MAX_SPLITS; ++r)
          if (r < splits) part[r] = r == split ? kept : from[(size_t)r * share * (G8_BM / 4)];
        float4 v = part[0];
#pragma unroll
        for (int r = 1; r < G8_MAX_SPLITS; ++r)
          if (r < splits) v.x += part[r].x, v.y += part[r].y, v.z += part[r].z, v.w += part[r].w;
        g8_store4(p, w.m0 + split * share + j, n, v);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {
    // The block gave up: the MMAs that were issued must be done, and no copy may still be on its way here.
    if (warp == 1) {
      if (tc_elect_one()) tc_commit(drain_bar);
      __syncwarp();
      mbar_drain(drain_bar, 0, p.wait_limit);
    } else if (tid == 0) {
      for (int i = copies > p.stages ? copies - p.stages : 0; i < copies; ++i)
        if (kb0 + i != p.test_skip_kb) mbar_drain(full0 + 8 * (i % p.stages), (uint32_t)(i / p.stages) & 1, p.wait_limit);
      if (mine > 0 && splits > 1) {
        if (!*sent) g8_arrive(received);
        mbar_drain(received, 0, p.wait_limit);
      }
      if (p.error_flag) atomicExch(p.error_flag, 1);
    }
    __syncthreads();
  }
  if (splits > 1) g8_cluster_arrive();      // what was sent here has come
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::COLS) : "memory");
  }
  if (splits > 1) g8_cluster_wait();      // what this block sent has been received: its shared memory may go
}

// ---- many tokens ------------------------------------------------------------------------------------------------------
// A pair of blocks makes a tile of 256 features by up to 256 tokens: block r holds features 128 r .. 128 r + 127 (its rows of the
// accumulator) and brings their weights and half of the tokens' rows; both hold the words of all tokens. The leader's thread
// issues the MMAs of both.
//   full[s], scales_full[s]    (leader's) both blocks' copies, or words, of a stage or slot are there
//   empty[s], scales_empty[s]  (each block's) the MMAs that read it are done
//   acc_full[2]                (each block's) the tile's sums are complete;  acc_empty[2] (leader's): both epilogues have read them
// Warps 2-5 write the words of scales, warps 6-13 run the epilogue: a quarter of the rows and half of the columns each. The words of
// scales leave 464 columns of tensor memory for the sums: every other tile has its at the lower end, the others at the upper, so
// that a tile's epilogue runs under the next one's MMAs wherever two neighbours have 464 tokens or fewer; else the next tile
// waits until this one's sums are read (an epilogue warp keeps its bfloat16 results in registers and gives tensor memory back
// before it stores).
constexpr int G8P_THREADS = 448, G8P_EPI_WARP = 6, G8P_STAGES = 6, G8P_NT = 256;
constexpr uint32_t G8P_STAGE_BYTES = G8_A_BYTES + G8P_NT / 2 * G8_BK;
constexpr int G8P_SLOT_COLS = 12, G8P_SUM_COLS = 512 - G8_SLOTS * G8P_SLOT_COLS, G8P_BARS = 2 * G8P_STAGES + 2 * G8_SLOTS + 5;
constexpr size_t G8P_SMEM = 1024 + (size_t)G8P_STAGES * G8P_STAGE_BYTES + G8P_BARS * 8 + 16;      // (four words behind the barriers)

// A copy into this block's shared memory whose bytes are counted by a barrier that may lie in the pair's other block.
__device__ __forceinline__ void g8_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void g8_mma_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                                            uint32_t sb, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
      : "memory");
}
// An arrival, in both blocks, on the barrier at this offset when every MMA issued so far by this thread is done.
__device__ __forceinline__ void g8_commit_pair(uint32_t bar) {
  const uint16_t both = 3;
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(both) : "memory");
}
__device__ __forceinline__ void g8_commit_pair_local(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void g8_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// Bounded wait on a barrier that threads of the other block arrive on (acquire at cluster scope).
__device__ __forceinline__ bool g8_try_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool g8_wait_cluster_slow(uint32_t bar, uint32_t parity, uint32_t limit, volatile int* abort_flag) {
  for (uint32_t it = 0; it < limit; ++it) {
    if (g8_try_cluster(bar, parity)) return true;
    if (it > 128) {
      __nanosleep(64);
      if (*abort_flag) return false;
    }
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ bool g8_wait_cluster(uint32_t bar, uint32_t parity, uint32_t limit, volatile int* abort_flag) {
  return g8_try_cluster(bar, parity) || g8_wait_cluster_slow(bar, parity, limit, abort_flag);
}
// The tokens of a pair's MMA: whole steps of 16, half of them in each block.
__device__ __forceinline__ int g8_pair_n(int rows) { return max((rows + 15) & ~15, 16); }

__global__ void __launch_bounds__(G8P_THREADS, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const G8Params p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* stages = reinterpret_cast<unsigned char*>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(stages + (size_t)G8P_STAGES * G8P_STAGE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + G8P_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* theirs = abort_flag + 1;      // copies that the other block had requested when it gave up; -1: it did not
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t full0 = tc_smem(bars), empty0 = full0 + 8 * G8P_STAGES, sc_full0 = empty0 + 8 * G8P_STAGES,
                 sc_empty0 = sc_full0 + 8 * G8_SLOTS, acc_full = sc_empty0 + 8 * G8_SLOTS, acc_empty = acc_full + 16,
                 drain_bar = acc_empty + 16;
  const uint32_t rank = g8_rank();      // 0: the leader
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, nkb = p.nkb;

  pdl_launch_dependents();
  if (warp == 0) {
    for (int s = lane; s < G8P_BARS; s += 32) {      // four, or eight, warps of both blocks arrive on two of the kinds
      const uint32_t bar = full0 + 8 * s;
      mbar_init(bar, bar >= sc_full0 && bar < sc_empty0 ? 8 : bar >= acc_empty && bar < drain_bar ? 16 : 1);
    }
    if (lane == 0) {
      g8_prefetch_map(&map_w);
      g8_prefetch_map(&map_x);
      *abort_flag = 0;
      *theirs = -1;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  g8_cluster_arrive();      // the peer's barriers exist before anything is sent to them
  g8_cluster_wait();
  pdl_wait();
  uint32_t tmem_base = 0;      // (asked for after the wait, see above; the same columns in both blocks)
  if (warp >= 1) {
    if (warp == 1) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    asm volatile("bar.sync 2, %0;" ::"n"(G8P_THREADS - 32) : "memory");
    tc_fence_after();
    tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  }
  const uint32_t tmem_scales = tmem_base + G8P_SUM_COLS;
  const int n_row_tiles = p.tiles ? min(*p.n_tiles, p.max_tiles) : p.n_t, n_work = n_row_tiles * p.n_f;
  int copies = 0;      // stages whose copies this block has requested

  if (warp == 0) {
    if (tc_elect_one()) {
      G8Ring r(G8P_STAGES);
      bool ok = true;
      for (int t = pair; t < n_work && ok; t += n_pairs) {
        const G8Tile w = g8_tile(p, t, n_row_tiles, 2 * G8_BM);
        const int half = g8_pair_n(w.rows) / 2, boxes = (half + p.x_box - 1) / p.x_box;
        const int w_row = w.group * p.N + w.f0 + (int)rank * G8_BM, m0 = w.m0 + (int)rank * half;
        const uint32_t bytes = G8_A_BYTES + (uint32_t)(boxes * p.x_box) * G8_BK;
        for (int kb = 0; kb < nkb; ++kb, ++copies, r.next()) {
          ok = g8_wait(empty0 + 8 * r.at, r.phase ^ 1, p.wait_limit, abort_flag);
          if (!ok) break;
          if (copies == p.test_skip_kb) continue;
          if (rank == 0) mbar_expect_tx(full0 + 8 * r.at, 2 * bytes);      // of both blocks
          const uint32_t dst = tc_smem(stages) + (uint32_t)r.at * G8P_STAGE_BYTES, bar = g8_map_rank(full0 + 8 * r.at, 0u);
          g8_load_pair(dst, &map_w, bar, kb * G8_BK, w_row);
          g8_load_pair(dst + G8_A_BYTES, &map_x, bar, kb * G8_BK, m0);
          for (int b = 1; b < boxes; ++b)      // (ragged tiles)
            g8_load_pair(dst + G8_A_BYTES + (uint32_t)(b * p.x_box) * G8_BK, &map_x, bar, kb * G8_BK, m0 + b * p.x_box);
        }
      }
    }
    __syncwarp();
    copies = __reduce_max_sync(0xffffffffu, copies);
  } else if (warp == 1) {
    if (rank == 0 && tc_elect_one()) {
      G8Ring r(G8P_STAGES);
      G8Ring sc(G8_SLOTS);
      bool ok = true;
      int lt = 0, before = 0;      // tiles so far, tokens of the last one's MMAs
      for (int t = pair; t < n_work && ok; t += n_pairs, ++lt) {
        const int n = g8_pair_n(g8_tile(p, t, n_row_tiles, 2 * G8_BM).rows), end = lt & 1;
        const uint32_t idesc0 = g8_idesc(2 * G8_BM, n, 0), d_addr = tmem_base + (end ? G8P_SUM_COLS - n : 0);
        // Both epilogues have read the tile that lay at this end, and the one at the other where this one reaches into it.
        ok = g8_wait_cluster(acc_empty + 8 * end, (uint32_t)((lt >> 1) & 1) ^ 1, p.wait_limit, abort_flag);
        if (ok && before + n > G8P_SUM_COLS)
          ok = g8_wait_cluster(acc_empty + 8 * (1 - end), (uint32_t)((lt - 1) >> 1) & 1, p.wait_limit, abort_flag);
        if (!ok) break;
        before = n;
        tc_fence_after();
        uint32_t acc = 0;
        for (int kb = 0; kb < nkb && ok; kb += 4, sc.next()) {      // a word of scales
          ok = g8_wait_cluster(sc_full0 + 8 * sc.at, sc.phase, p.wait_limit, abort_flag);
          const uint32_t sa = tmem_scales + (uint32_t)(sc.at * G8P_SLOT_COLS);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (kb + j >= nkb || !ok) continue;
            ok = g8_wait_cluster(full0 + 8 * r.at, r.phase, p.wait_limit, abort_flag);
            if (!ok) continue;
            tc_fence_after();
            const uint32_t a_addr = tc_smem(stages) + (uint32_t)r.at * G8P_STAGE_BYTES, idesc = idesc0 | g8_idesc(0, 0, j);
            const uint64_t a_desc = tc_smem_desc(a_addr), b_desc = tc_smem_desc(a_addr + G8_A_BYTES);
#pragma unroll
            for (int k = 0; k < G8_BK / 32; ++k) {
              g8_mma_pair(d_addr, a_desc + (uint64_t)(k * 2), b_desc + (uint64_t)(k * 2), idesc, sa, sa + 4, acc);
              acc = 1;
            }
            g8_commit_pair(empty0 + 8 * r.at);
            r.next();
          }
          g8_commit_pair(sc_empty0 + 8 * sc.at);
        }
        if (ok) g8_commit_pair(acc_full + 8 * end);
      }
    }
    __syncwarp();
  } else if (warp < G8P_EPI_WARP) {
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int g1 = (nkb + 3) / 4;
    G8Words<G8P_NT> now, next;
    int t = pair, base = 0;
    auto load = [&](int t, int base, G8Words<G8P_NT>& o) {
      const G8Tile w = g8_tile(p, t, n_row_tiles, 2 * G8_BM);
      g8_load_words<G8P_NT>(p, w.group * p.N + w.f0 + (int)rank * G8_BM, w.m0, base, g1, lane, o);
    };
    if (t < n_work) load(t, base, now);
    G8Ring sc(G8_SLOTS);
    bool ok = true;
    while (t < n_work && ok) {
      int t2 = t, base2 = base + G8Words<G8P_NT>::STEPS;
      if (base2 >= g1) t2 += n_pairs, base2 = 0;
      if (t2 < n_work) load(t2, base2, next);
#pragma unroll
      for (int u = 0; u < G8Words<G8P_NT>::STEPS; ++u) {
        if (base + u >= g1 || !ok) continue;
        ok = __all_sync(0xffffffffu, g8_wait(sc_empty0 + 8 * sc.at, sc.phase ^ 1, p.wait_limit, abort_flag));
        if (!ok) continue;
        tc_fence_after();
        g8_put_words<G8P_NT>(now, u, tmem_scales + (uint32_t)(sc.at * G8P_SLOT_COLS) + lanes);
        if (lane == 0) g8_arrive_cluster(g8_map_rank(sc_full0 + 8 * sc.at, 0u));
        sc.next();
      }
      now = next, t = t2, base = base2;
    }
  } else {
    const int quarter = warp & 3, c0 = (warp - G8P_EPI_WARP) / 4 * (G8P_NT / 2);
    bool ok = true;
    int lt = 0;
    for (int t = pair; t < n_work && ok; t += n_pairs, ++lt) {
      const G8Tile w = g8_tile(p, t, n_row_tiles, 2 * G8_BM);
      const int n = w.f0 + (int)rank * G8_BM + quarter * 32 + lane, left = min(w.rows - c0, G8P_NT / 2);      // columns of this warp's half
      const int end = lt & 1;
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(c0 + (end ? G8P_SUM_COLS - g8_pair_n(w.rows) : 0));
      ok = __all_sync(0xffffffffu, g8_wait(acc_full + 8 * end, (uint32_t)(lt >> 1) & 1, p.wait_limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      if (p.out_f32) {
        for (int c = 0; c < left; c += 16) {      // all lanes: the reads are warp-wide
          float v[16];
          g8_ld16(taddr + c, v);
          if (n < p.N) g8_store<16>(p, w.m0 + c0 + c, n, left - c, v);
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) g8_arrive_cluster(g8_map_rank(acc_empty + 8 * end, 0u));
      } else {
        __nv_bfloat162 keep[G8P_NT / 4];
#pragma unroll
        for (int c = 0; c < G8P_NT / 2; c += 16) {
          if (c >= left) continue;
          float v[16];
          g8_ld16(taddr + c, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) keep[c / 2 + e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) g8_arrive_cluster(g8_map_rank(acc_empty + 8 * end, 0u));
        if (n < p.N) {
          __nv_bfloat16* o = (__nv_bfloat16*)p.out + (size_t)(w.m0 + c0) * p.ldo + n;
#pragma unroll
          for (int e = 0; e < G8P_NT / 4; ++e, o += 2 * p.ldo) {
            if (2 * e < left) o[0] = keep[e].x;
            if (2 * e + 1 < left) o[p.ldo] = keep[e].y;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // The block gave up. The MMAs that were issued must be done before tensor memory is freed.
    if (rank == 0 && warp == 1) {
      if (tc_elect_one()) g8_commit_pair_local(drain_bar);
      __syncwarp();
      mbar_drain(drain_bar, 0, p.wait_limit);
    } else if (tid == 0) {
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(g8_map_rank(tc_smem(const_cast<int*>(theirs)), rank ^ 1)), "r"(copies) : "memory");
      if (p.error_flag) atomicExch(p.error_flag, 1);
    }
    __syncthreads();
  }
  // Neither block may free tensor memory or leave while the other still computes into it or signals its barriers.
  tc_fence_before();
  g8_cluster_arrive();
  g8_cluster_wait();
  if (*abort_flag || *theirs >= 0) {      // (the same in both blocks)
    // The copies that were requested must have landed in both. The leader's barriers count them: of a stage that only the other
    // block came to (it gave up later) the leader has still to say how many bytes are on their way.
    if (rank == 0 && tid == 0) {
      for (int i = copies > G8P_STAGES ? copies - G8P_STAGES : 0; i < max(copies, *theirs); ++i) {
        const uint32_t bar = full0 + 8 * (i % G8P_STAGES);
        if (i == p.test_skip_kb) continue;
        if (i >= copies) {
          const int half = g8_pair_n(g8_tile(p, pair + i / nkb * n_pairs, n_row_tiles, 2 * G8_BM).rows) / 2;
          mbar_expect_tx(bar, G8_A_BYTES + (uint32_t)((half + p.x_box - 1) / p.x_box * p.x_box) * G8_BK);
        }
        mbar_drain(bar, (uint32_t)(i / G8P_STAGES) & 1, p.wait_limit);
      }
    }
    __syncthreads();
    g8_cluster_arrive();
    g8_cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
static int g8_map(CUtensorMap* map, const void* base, long long rows, long long K, long long pitch, int box_rows) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return llmrs_fail("gemm_fp8: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(cuuint32_t)G8_BK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return llmrs_fail("gemm_fp8: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return 0;
}

// The current device, its multiprocessors (asked for once: every call of the runtime costs part of a microsecond).
constexpr int G8_DEVICES = 64;
static int g8_device(int* sms) {
  static std::atomic<int> known[G8_DEVICES];
  int dev = 0;
  cudaGetDevice(&dev);
  const bool in = dev >= 0 && dev < G8_DEVICES;
  int n = in ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (in) known[dev].store(n, std::memory_order_relaxed);
  }
  *sms = n > 0 ? n : 1;
  return dev;
}

typedef void (*G8Kernel)(CUtensorMap, CUtensorMap, G8Params);
// `allowed`: devices on which the kernel may already use the most shared memory that it takes.
static int g8_launch(G8Kernel kernel, std::atomic<unsigned long long>* allowed, size_t most, size_t smem, int dev, int threads,
                     dim3 grid, dim3 cluster, const CUtensorMap& mw, const CUtensorMap& mx, const G8Params& p,
                     cudaStream_t stream) {
  const unsigned long long bit = 1ull << (dev % G8_DEVICES);
  cudaError_t e = cudaSuccess;
  if (dev >= G8_DEVICES || !(allowed->load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return llmrs_fail("gemm_fp8: shared memory %zu: %s", most, cudaGetErrorString(e));
    allowed->fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster.x;
  attr[0].val.clusterDim.y = cluster.y;
  attr[0].val.clusterDim.z = cluster.z;
  cfg.numAttrs = 1;
  if (g_llmrs_pdl) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  e = cudaLaunchKernelEx(&cfg, kernel, mw, mx, p);
  if (e != cudaSuccess) return llmrs_fail("gemm_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("gemm_fp8");
}
// A block's shared memory: what an SM has for one or for two blocks (1 KB of each is the system's).
constexpr size_t G8_SMEM_ONE = 227 * 1024, G8_SMEM_TWO = 113 * 1024;
template <int NT>
static int g8_stages(int nkb, int splits, int per_sm) {
  using C = G8Few<NT>;
  int stages = (int)(((per_sm == 1 ? G8_SMEM_ONE : G8_SMEM_TWO) - C::smem(0, splits)) / C::STAGE_BYTES);
  const int k_blocks = (nkb + splits - 1) / splits;
  if (stages > C::MAX_STAGES) stages = C::MAX_STAGES;
  if (stages > k_blocks) stages = k_blocks;
  // Split, the stages hold what a block sends.
  const int least = splits > 1 ? (int)((C::SUM_BYTES - 1) / C::STAGE_BYTES + 1) : 1;
  if (stages < least) stages = least;
  return C::smem(stages, splits) <= (per_sm == 1 ? G8_SMEM_ONE : G8_SMEM_TWO) ? stages : 0;
}
template <int NT>
static int g8_launch_few(const CUtensorMap& mw, const CUtensorMap& mx, G8Params& p, int dev, int tiles, int splits, int per_sm,
                         cudaStream_t stream) {
  static std::atomic<unsigned long long> allowed;
  p.stages = g8_stages<NT>(p.nkb, splits, per_sm);
  if (p.stages == 0) p.stages = g8_stages<NT>(p.nkb, splits, 1);
  return g8_launch(gemm_fp8_few_kernel<NT>, &allowed, G8_SMEM_ONE, G8Few<NT>::smem(p.stages, splits), dev, G8F_THREADS,
                   dim3((unsigned)tiles, 1, (unsigned)splits), dim3(1, 1, (unsigned)splits), mw, mx, p, stream);
}

// Blocks of the few-token kernel an SM: two where one each would not hold them all (clusters leave SMs over).
static int g8_per_sm(long long blocks, int splits, int sms) { return blocks > (splits > 2 ? sms * 4 / 5 : sms) ? 2 : 1; }

// The way of a product: tokens a tile (256: on pairs), blocks that share a tile's k, blocks an SM, tiles of tokens (pairs, dense).
struct G8Choice { int nt, splits, per_sm, n_t; };

// The microseconds that each way is expected to take, and the way that takes least. What the parts stand for, fitted to some 5,900
// products of 1 to 16,384 rows, dense and of 4 to 64 groups, each timed every way on a B200 (over 2,700 others the way taken is on
// average 2 % behind the best one, in one of a hundred more than 30 %; 16 x 128 x 128 takes 2.9 us):
//   a block copies, and its MMAs take, a block of k in .10 us + .6 ns a token; the blocks of an SM together get some 120 GB/s, all
//   together 10 TB/s (the memory and the L2); a wave of blocks after another starts 2.7 us late, or .5 where the memory is what
//   bounds; a split costs .56 us + 27 ns a token for the exchange of the sums; a wave of a list's blocks that have no tile .13 us;
//   a pair of the other kernel takes .257 us + .45 ns a token for a block of k of its 256 features (the copies; the MMAs of 256
//   tokens are .27), .8 us a tile more, or 1 where two neighbours do not fit tensor memory together.
// Measured, us (tokens x features x K; NT / splits): 1 x 6,144 x 4,096 16/1 9.4, 16/2 8.1, 16/5 7.7, 16/8 10.7; 32 x 4,096 x 4,096
// 32/1 8.8, 32/3 7.2, 16/4 7.7; 128 x 6,144 x 4,096 64/1 10.3, 64/2 12.4, 128/1 11.8, pair 17.5; 512 x 4,096 x 4,096 128/1 11.8, 64/1
// 14.1, pair 17.4; 2,048 x 4,096 x 4,096 pair 31.0, 128/1 37.2; 128 rows of 32 groups of 2,048 x 2,048 32/1 22.4, pair 28.6.
// tile_rows 0: dense; else the most rows of a list's tiles, of which there are at most `max_tiles`, and no more than rows as a rule.
static G8Choice g8_choose(int rows, int tile_rows, int max_tiles, int groups, int N, int K, int sms) {
  const int nkb = (K - 1) / G8_BK + 1, live = max_tiles < rows ? max_tiles : rows;
  const int fill = tile_rows ? (rows - 1) / live + 1 : 0;      // rows a tile has on average
  const double memory = ((double)(groups < rows ? groups : rows) * N + rows) * K / 10e6;
  G8Choice best = {256, 1, 1, 0};
  const int pairs = sms / 2 > 0 ? sms / 2 : 1, pair_f = (N - 1) / 256 + 1;
  double least = 1e30;
  const int from = tile_rows ? live : (rows - 1) / 256 + 1, to = tile_rows ? live : (rows - 1) / 128 + 1;
  for (int tiles = from; tiles <= to; ++tiles) {      // (more than a few are not tried: the first ones differ most)
    if (tiles > from + 8) break;
    int n = ((rows - 1) / tiles + 16) & ~15;
    if (tile_rows) n = fill < 16 ? (tile_rows < 16 ? tile_rows : 16) : fill < tile_rows ? fill : tile_rows;
    const double waves = (double)(((long long)tiles * pair_f + pairs - 1) / pairs);
    const double walk = waves * (nkb * (.257 + .00045 * n) + (2 * n > G8P_SUM_COLS ? 1.0 : .8));
    const double t = 5.2 + (walk > memory ? walk : memory);
    if (t < least) least = t, best.n_t = tiles;
  }
  for (int nt = 16; nt <= 128; nt *= 2) {
    if (tile_rows ? nt < tile_rows : nt >= 2 * rows && nt > 16) continue;
    const long long n_f = (N - 1) / G8_BM + 1, tiles = (tile_rows ? live : (rows - 1) / nt + 1) * n_f;
    const int n = tile_rows && fill < nt ? (fill < 16 ? 16 : fill) : nt;
    for (int splits = 1; splits <= G8_MAX_SPLITS && splits <= nkb && (splits == 1 || tiles * splits <= 2 * sms); ++splits) {
      const long long blocks = tiles * splits, grid = tile_rows ? max_tiles * n_f * splits : blocks;
      int per_sm = g8_per_sm(grid, splits, sms);
      const auto stages = nt == 16 ? g8_stages<16> : nt == 32 ? g8_stages<32> : nt == 64 ? g8_stages<64> : g8_stages<128>;
      if (stages(nkb, splits, per_sm) == 0) per_sm = 1;
      // Clusters leave SMs over: 132 of 148 are held by blocks in fours, one an SM, 120 in eights.
      const double held = (double)per_sm * sms * (splits <= 2 ? 1.0 : splits <= 4 ? .89 : .81);
      const double waves = (double)(long long)((blocks + held - 1) / held);
      const int together = per_sm == 2 && blocks > sms ? 2 : 1;
      const double shared = together * (16.4 + .128 * n) / 120, alone = .10 + .0006 * n;
      const double walk = waves * ((nkb + splits - 1) / splits) * (shared > alone ? shared : alone) + 2.7 * (waves - 1);
      const double stream = memory + .5 * (waves - 1);
      const double t = 2.1 + .002 * nt + (splits > 1 ? .56 + .027 * n : 0.0) + (walk > stream ? walk : stream) +
                       .13 * (double)(grid - blocks) / held;
      if (t < least) least = t, best = {nt, splits, per_sm, 0};
    }
  }
  return best;
}

// The same, remembered by the sizes (the estimates of the 30 ways cost part of a microsecond).
static G8Choice g8_chosen(int rows, int tile_rows, int max_tiles, int groups, int N, int K, int sms) {
  struct Known { int rows, tile_rows, max_tiles, groups, N, K, sms; G8Choice way; };
  static thread_local Known known[64];      // rows 0: empty
  const unsigned h = (unsigned)rows * 0x9E3779B1u ^ (unsigned)N * 0x85EBCA77u ^ (unsigned)K * 0xC2B2AE3Du ^ (unsigned)max_tiles * 0x27D4EB2Fu;
  Known& k = known[(h ^ h >> 15) % 64];
  if (k.rows != rows || k.tile_rows != tile_rows || k.max_tiles != max_tiles || k.groups != groups || k.N != N || k.K != K || k.sms != sms)
    k = {rows, tile_rows, max_tiles, groups, N, K, sms, g8_choose(rows, tile_rows, max_tiles, groups, N, K, sms)};
  return k.way;
}

// x: x_rows rows of K e4m3 numbers x_pitch bytes apart, xs their words of scales (word g of row r at
// g * xs_stride + r); w: groups * N rows, ws the same of them. tile_rows: the most rows of a tile of the list, or 0: dense
// (one group, no list). nt: tokens a tile (256: the kernel on pairs), splits: blocks that share a tile's k; 0: chosen here.
LLMRS_API int llmrs_gemm_fp8(const void* x, long long x_pitch, const void* xs, long long xs_stride, int x_rows, const void* w,
                             long long w_pitch, const void* ws, long long ws_stride, void* out, long long ldo, int out_dtype,
                             int epilogue, int N, int K, int groups, const int* tiles, const int* n_tiles, int max_tiles,
                             int tile_rows, int nt, int splits, int* error_flag, cudaStream_t stream) {
  const bool grouped = tile_rows != 0;
  const char* what = grouped ? "gemm_fp8_grouped" : "gemm_fp8";
  LLMRS_REQUIRE(x_rows >= 0 && N > 0 && K > 0 && groups > 0, "%s: bad sizes", what);
  LLMRS_REQUIRE(x_pitch % 16 == 0 && w_pitch % 16 == 0 && x_pitch >= K && w_pitch >= K && (((uintptr_t)x | (uintptr_t)w) & 15) == 0,
                "%s: rows must start at multiples of 16 bytes", what);
  LLMRS_REQUIRE((((uintptr_t)xs | (uintptr_t)ws) & 3) == 0, "%s: scales must start at a multiple of 4 bytes", what);
  LLMRS_REQUIRE((long long)groups * N <= 0x7ffffe00LL && K <= 0x7ffffe00 && x_rows <= 0x7ffffe00, "%s: too many rows", what);
  LLMRS_REQUIRE(epilogue == G8_STORE || (epilogue == G8_ADD && out_dtype == LLMRS_F32), "%s: unknown epilogue %d", what, epilogue);
  if (x_rows == 0 || (grouped && max_tiles == 0)) return 0;
  LLMRS_REQUIRE(!grouped || (tiles && n_tiles && tile_rows > 0 && tile_rows <= 256), "%s: a list of tiles of 1 to 256 rows, got %d",
                what, tile_rows);
  int sms;
  const int dev = g8_device(&sms), nkb = (K - 1) / G8_BK + 1;
  int per_sm = 0, n_t = 0;
  if (nt == 0) {
    const G8Choice way = g8_chosen(x_rows, tile_rows, max_tiles, groups, N, K, sms);
    nt = way.nt, splits = way.splits, per_sm = way.per_sm, n_t = way.n_t;
  } else if (splits == 0) {
    splits = 1;
  }
  const bool pair = nt == 256;
  LLMRS_REQUIRE(!grouped || nt >= tile_rows, "%s: tiles of %d tokens for a list of tiles of %d", what, nt, tile_rows);
  G8Params p = {};
  p.out = out, p.ldo = ldo, p.out_f32 = out_dtype == LLMRS_F32, p.epilogue = epilogue;
  p.xs = (const uint32_t*)xs, p.ws = (const uint32_t*)ws, p.xs_stride = xs_stride, p.ws_stride = ws_stride, p.x_rows = x_rows;
  p.w_rows = groups * N, p.N = N, p.nkb = nkb, p.n_f = (N - 1) / (pair ? 2 * G8_BM : G8_BM) + 1;
  p.n_t = n_t > 0 && pair && !grouped ? n_t : (x_rows - 1) / nt + 1;
  // Dense: tiles of one size, and one copy of their rows a stage; a list's tiles are ragged, their rows come 32 at a time.
  p.nt = grouped ? nt : ((x_rows - 1) / p.n_t + 16) & ~15;
  if (!grouped) p.n_t = (x_rows - 1) / p.nt + 1;      // (rounded up, they may be fewer)
  p.x_box = grouped ? (nt < 32 ? nt : 32) : (pair ? p.nt / 2 : p.nt);
  p.vec = ((uintptr_t)out & 15) == 0 && ldo % 8 == 0;
  p.vec4 = ((uintptr_t)out & (p.out_f32 ? 15 : 7)) == 0 && ldo % 4 == 0;
  p.tiles = grouped ? tiles : nullptr, p.n_tiles = n_tiles, p.max_tiles = max_tiles, p.groups = groups;
  p.error_flag = error_flag, p.wait_limit = llmrs_tc_wait_limit(), p.test_skip_kb = llmrs_tc_skipped_copy();
  const long long work = (long long)(grouped ? max_tiles : p.n_t) * p.n_f;
  LLMRS_REQUIRE(work <= 0x7fffffffLL, "%s: too many tiles", what);
  LLMRS_REQUIRE(splits >= 1 && splits <= G8_MAX_SPLITS && splits <= nkb, "%s: 1 to %d parts of k, got %d", what, G8_MAX_SPLITS, splits);
  if (per_sm == 0) per_sm = g8_per_sm(work * splits, splits, sms);
  CUtensorMap mw, mx;
  if (const int rc = g8_map(&mw, w, (long long)groups * N, K, w_pitch, G8_BM)) return rc;
  if (const int rc = g8_map(&mx, x, x_rows, K, x_pitch, p.x_box)) return rc;
  switch (pair ? 256 : nt) {
    case 16: return g8_launch_few<16>(mw, mx, p, dev, (int)work, splits, per_sm, stream);
    case 32: return g8_launch_few<32>(mw, mx, p, dev, (int)work, splits, per_sm, stream);
    case 64: return g8_launch_few<64>(mw, mx, p, dev, (int)work, splits, per_sm, stream);
    case 128: return g8_launch_few<128>(mw, mx, p, dev, (int)work, splits, per_sm, stream);
    case 256: {
      static std::atomic<unsigned long long> allowed;
      const int pairs = sms / 2 > 0 ? sms / 2 : 1;
      return g8_launch(gemm_fp8_pair_kernel, &allowed, G8P_SMEM, G8P_SMEM, dev, G8P_THREADS,
                       dim3(2u * (unsigned)(work < pairs ? work : pairs)), dim3(2, 1, 1), mw, mx, p, stream);
    }
    default: return llmrs_fail("%s: tiles of 16, 32, 64, 128 or 256 tokens, got %d", what, nt);
  }
}
