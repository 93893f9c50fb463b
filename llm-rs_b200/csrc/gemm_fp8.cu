// Products of rows in 8 bits (fp8.cuh) on tcgen05: y[t, n] = sum_b 2^(Ex[t, b] + Ew[n, b]) * sum_{k in block b} x[t, k] * w[n, k],
// dense or grouped by expert (rows sorted by group, a list of tiles of rows, each group's own weights).
//
// The scales are powers of two, which tcgen05.mma.kind::mxf8f6f4.block_scale applies itself: the sums stay in tensor memory in
// float32 over the whole of k and nothing is promoted on the CUDA cores. A block of 128 numbers is four MMAs of k = 32 that name
// the same byte of a row's word of scales; a word serves four blocks.
//
// A tile is 128 features (the M side, whatever the number of tokens is) by up to NT tokens (the N side; an MMA is as wide as the
// tile's rows, in steps of 16, so that a group's ragged end costs what it has). Warp 0 copies by TMA, warp 1 issues the MMAs, warps
// 2-5 move the words of scales from memory to tensor memory (a warp can write the 32 lanes that its index modulo 4 names, and the
// MMA wants every word in all four quarters), warps 6-9 run the epilogue: a lane holds a feature, a column a token.
//
// With few tiles the range of k is split over a cluster of blocks, whose sums are added through distributed shared memory in
// the order of the ranks; else a block per SM walks the tiles, a tile's epilogue under the next one's MMAs where tensor memory holds
// two accumulators.
//
// Every wait is bounded (see gemm_tcgen05.cu): a block that gives up drains its copies and MMAs, records a code in *error_flag,
// frees its tensor memory and returns.
#include "fp8.cuh"
#include "tcgen05_util.cuh"

uint32_t llmrs_tc_wait_limit();
int llmrs_tc_skipped_copy();

constexpr int G8_THREADS = 320, G8_EPI_WARP = 6;
constexpr int G8_BM = 128, G8_BK = 128;              // features a tile, bytes of k a stage
constexpr uint32_t G8_A_BYTES = G8_BM * G8_BK;
constexpr int G8_SCALE_SLOTS = 4;                    // words of scales of 512 numbers each under way in tensor memory

enum G8Epilogue : int { G8_STORE = 0, G8_ADD = 1 };

struct G8Params {
  void* out;
  long long ldo;
  int out_f32, epilogue;
  const uint32_t* xs;      // word g of row r: xs[g * xs_stride + r]
  const uint32_t* ws;
  long long xs_stride, ws_stride;
  int x_rows, w_rows;      // rows of x; rows of all groups' weights
  int N, n_f, n_t, nkb;    // features a group, tiles of features, tiles of tokens (dense), blocks of k
  int x_box;               // rows of x that a copy brings
  const int* tiles;        // grouped: [tile][3] = group, first row, rows; null: dense
  const int* n_tiles;
  int max_tiles, groups;
  int* error_flag;
  uint32_t wait_limit;
  int test_skip_kb;
};

template <int NT> struct G8Config {
  static constexpr uint32_t B_BYTES = NT * G8_BK, STAGE_BYTES = G8_A_BYTES + B_BYTES;
  static constexpr int STAGES = NT == 16 ? 11 : NT == 32 ? 10 : NT == 64 ? 8 : NT == 128 ? 6 : 4;
  static constexpr int ACC_COLS = NT < 32 ? 32 : NT, ACC_BUFS = NT == 256 ? 1 : 2;
  static constexpr int SB_COLS = NT <= 128 ? 4 : 8, SLOT_COLS = 4 + SB_COLS;      // words of the features, words of the tokens
  static constexpr int USED = ACC_COLS * ACC_BUFS + G8_SCALE_SLOTS * SLOT_COLS;
  static constexpr int COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  // full[S], empty[S], acc_full[2], acc_empty[2], scales_full[4], scales_empty[4], drain
  static constexpr int BARS = 2 * STAGES + 4 + 2 * G8_SCALE_SLOTS + 1;
  static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + BARS * 8 + 16;
};

// Instruction descriptor: e4m3 x e4m3 with E8M0 scales, both K-major, M = 128; N and the scales' byte are added.
__device__ __forceinline__ uint32_t g8_idesc(int n, int byte) {
  return (1u << 23) | (1u << 27) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)byte << 4) | ((uint32_t)byte << 29);
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
__device__ __forceinline__ void g8_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t g8_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void g8_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float g8_ld_cluster(uint32_t local_addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// The tile of work item t: group, first row of x, rows, first feature.
struct G8Tile { int group, m0, rows, f0; };
template <int NT>
__device__ __forceinline__ G8Tile g8_tile(const G8Params& p, int t, int n_row_tiles) {
  const int i = t % n_row_tiles, f = t / n_row_tiles;
  G8Tile w;
  w.f0 = f * G8_BM;
  if (p.tiles) {
    w.group = p.tiles[3 * i], w.m0 = p.tiles[3 * i + 1], w.rows = min(p.tiles[3 * i + 2], NT);
    if (w.group < 0 || w.group >= p.groups || w.m0 < 0 || w.m0 >= p.x_rows || w.rows < 0)
      w.group = w.m0 = w.rows = 0;      // names what is not there: nothing is computed for it
    w.rows = min(w.rows, p.x_rows - w.m0);
  } else {
    w.group = 0, w.m0 = i * NT, w.rows = min(NT, p.x_rows - w.m0);
  }
  return w;
}

__device__ __forceinline__ void g8_store(const G8Params& p, int row, int n, float v) {
  const size_t at = (size_t)row * p.ldo + n;
  if (p.epilogue == G8_ADD)
    ((float*)p.out)[at] += v;
  else if (p.out_f32)
    ((float*)p.out)[at] = v;
  else
    ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(v);
}

template <int NT>
__global__ void __launch_bounds__(G8_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const G8Params p) {
  using C = G8Config<NT>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* stages = reinterpret_cast<unsigned char*>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(stages + (size_t)C::STAGES * C::STAGE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t full0 = tc_smem(bars), empty0 = full0 + 8 * C::STAGES, acc_full0 = empty0 + 8 * C::STAGES,
                 acc_empty0 = acc_full0 + 16, sc_full0 = acc_empty0 + 16, sc_empty0 = sc_full0 + 8 * G8_SCALE_SLOTS,
                 drain_bar = sc_empty0 + 8 * G8_SCALE_SLOTS;
  const int splits = (int)gridDim.z, split = (int)blockIdx.z;      // the blocks of a cluster share a tile's range of k
  const int kb0 = (int)((long long)split * p.nkb / splits), kb1 = (int)((long long)(split + 1) * p.nkb / splits);

  pdl_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < 2 * C::STAGES + 2; ++s) mbar_init(full0 + 8 * s, 1);
    mbar_init(acc_empty0, 128);
    mbar_init(acc_empty0 + 8, 128);
    for (int s = 0; s < G8_SCALE_SLOTS; ++s) {
      mbar_init(sc_full0 + 8 * s, 4);
      mbar_init(sc_empty0 + 8 * s, 1);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_slot)), "r"(C::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot, tmem_scales = tmem_base + C::ACC_COLS * C::ACC_BUFS;
  pdl_wait();      // everything below reads or writes what earlier kernels may have touched
  const int n_row_tiles = p.tiles ? min(*p.n_tiles, p.max_tiles) : p.n_t, n_work = n_row_tiles * p.n_f;
  long long copies = 0;      // warp 0: stages whose copies it has requested

  if (warp == 0) {
    const bool leader = tc_elect_one();
    long long it = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < n_work && ok; t += gridDim.x) {
      const G8Tile w = g8_tile<NT>(p, t, n_row_tiles);
      const int w_row = w.group * p.N + w.f0, boxes = max((w.rows + p.x_box - 1) / p.x_box, 1);
      const uint32_t bytes = G8_A_BYTES + (uint32_t)(boxes * p.x_box) * G8_BK;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = (int)(it % C::STAGES);
        if (it >= C::STAGES) {
          ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, (uint32_t)((it / C::STAGES) - 1) & 1, p.wait_limit, abort_flag));
          if (!ok) break;
        }
        if (leader && it != p.test_skip_kb) {
          const uint32_t bar = full0 + 8 * s, dst = tc_smem(stages + (size_t)s * C::STAGE_BYTES);
          mbar_expect_tx(bar, bytes);
          tma_load_2d(dst, &map_w, bar, kb * G8_BK, w_row);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(dst + G8_A_BYTES + (uint32_t)(b * p.x_box) * G8_BK, &map_x, bar, kb * G8_BK, w.m0 + b * p.x_box);
        }
        __syncwarp();
      }
    }
    copies = it;
  } else if (warp == 1) {
    const bool leader = tc_elect_one();
    long long it = 0, sc = 0;      // stages and words of scales taken so far
    int lt = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < n_work && ok; t += gridDim.x, ++lt) {
      const G8Tile w = g8_tile<NT>(p, t, n_row_tiles);
      const int n = max((w.rows + 15) & ~15, 16), buf = lt % C::ACC_BUFS;
      if (lt >= C::ACC_BUFS) {      // the epilogue has read the tile that lay in this buffer
        ok = __all_sync(0xffffffffu, mbar_wait(acc_empty0 + 8 * buf, (uint32_t)((lt / C::ACC_BUFS) - 1) & 1, p.wait_limit, abort_flag));
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t d_addr = tmem_base + (uint32_t)(buf * C::ACC_COLS);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = (int)(it % C::STAGES), slot = (int)(sc % G8_SCALE_SLOTS);
        if (kb == kb0 || (kb & 3) == 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(sc_full0 + 8 * slot, (uint32_t)(sc / G8_SCALE_SLOTS) & 1, p.wait_limit, abort_flag));
          if (!ok) break;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, (uint32_t)(it / C::STAGES) & 1, p.wait_limit, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t a_addr = tc_smem(stages + (size_t)s * C::STAGE_BYTES), sa = tmem_scales + (uint32_t)(slot * C::SLOT_COLS),
                         idesc = g8_idesc(n, kb & 3);
          const uint64_t a_desc = tc_smem_desc(a_addr), b_desc = tc_smem_desc(a_addr + G8_A_BYTES);
#pragma unroll
          for (int k = 0; k < G8_BK / 32; ++k)
            g8_mma(d_addr, a_desc + (uint64_t)(k * 2), b_desc + (uint64_t)(k * 2), idesc, sa, sa + 4, (kb > kb0 || k > 0) ? 1u : 0u);
          tc_commit(empty0 + 8 * s);
          if ((kb & 3) == 3 || kb + 1 == kb1) tc_commit(sc_empty0 + 8 * slot);
        }
        if ((kb & 3) == 3 || kb + 1 == kb1) ++sc;
        __syncwarp();
      }
      if (leader && ok) tc_commit(acc_full0 + 8 * buf);
      __syncwarp();
    }
  } else if (warp < G8_EPI_WARP) {
    // Words of scales: lane l of the quarter holds the words of rows l, l + 32, l + 64, .. in neighbouring columns.
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    long long sc = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < n_work && ok; t += gridDim.x) {
      const G8Tile w = g8_tile<NT>(p, t, n_row_tiles);
      const int w_row = w.group * p.N + w.f0;
      for (int g = kb0 / 4; g < (kb1 + 3) / 4; ++g, ++sc) {
        const int slot = (int)(sc % G8_SCALE_SLOTS);
        uint32_t a[4], b[4], c[4];
        const uint32_t* wg = p.ws + (size_t)g * p.ws_stride;
        const uint32_t* xg = p.xs + (size_t)g * p.xs_stride;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = __ldg(wg + min(w_row + lane + 32 * j, p.w_rows - 1));
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = 32 * j < NT ? __ldg(xg + min(w.m0 + lane + 32 * j, p.x_rows - 1)) : 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = NT > 128 ? __ldg(xg + min(w.m0 + lane + 128 + 32 * j, p.x_rows - 1)) : 0u;
        if (sc >= G8_SCALE_SLOTS) {
          ok = __all_sync(0xffffffffu, mbar_wait(sc_empty0 + 8 * slot, (uint32_t)((sc / G8_SCALE_SLOTS) - 1) & 1, p.wait_limit, abort_flag));
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t at = tmem_scales + (uint32_t)(slot * C::SLOT_COLS) + quarter;
        g8_st4(at, a);
        g8_st4(at + 4, b);
        if (NT > 128) g8_st4(at + 8, c);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) g8_arrive(sc_full0 + 8 * slot);
      }
    }
  } else {
    const int quarter = warp & 3;
    int lt = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < n_work && ok; t += gridDim.x, ++lt) {
      const G8Tile w = g8_tile<NT>(p, t, n_row_tiles);
      const int buf = lt % C::ACC_BUFS, n = w.f0 + quarter * 32 + lane;
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * buf, (uint32_t)(lt / C::ACC_BUFS) & 1, p.wait_limit, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * C::ACC_COLS);
      for (int c = 0; c < w.rows; c += 32) {      // all lanes: the reads are warp-wide
        float v[32];
        tc_ld32(taddr + c, v);
        if (splits > 1) {
          // The stages are free: every MMA of the block has been done.
          float* part = reinterpret_cast<float*>(stages);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e < NT) part[(size_t)(c + e) * G8_BM + quarter * 32 + lane] = v[e];
        } else if (n < p.N) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c + e < w.rows) g8_store(p, w.m0 + c + e, n, v[e]);
        }
        __syncwarp();
      }
      tc_fence_before();
      g8_arrive(acc_empty0 + 8 * buf);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // The block gave up: the MMAs that were issued must be done, and no copy may still be on its way here.
    if (warp == 1) {
      if (tc_elect_one()) tc_commit(drain_bar);
      __syncwarp();
      mbar_drain(drain_bar, 0, p.wait_limit);
    } else if (tid == 0) {
      for (long long i = copies > C::STAGES ? copies - C::STAGES : 0; i < copies; ++i)
        if (i != p.test_skip_kb) mbar_drain(full0 + 8 * (int)(i % C::STAGES), (uint32_t)(i / C::STAGES) & 1, p.wait_limit);
      if (p.error_flag) atomicExch(p.error_flag, 1);
    }
    __syncthreads();
    if (splits > 1) {      // nothing of this block enters the sums
      float* part = reinterpret_cast<float*>(stages);
      for (int i = tid; i < NT * G8_BM; i += G8_THREADS) part[i] = 0.f;
      __syncthreads();
    }
  }
  if (warp == 0) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::COLS) : "memory");
  }
  if (splits > 1) {
    // One tile a cluster (the grid covers them all). Block r adds up the tokens r, r + splits, ..
    g8_cluster_sync();
    if ((int)blockIdx.x < n_work) {
      const G8Tile w = g8_tile<NT>(p, blockIdx.x, n_row_tiles);
      const uint32_t part = tc_smem(stages);
      const int rank = (int)g8_rank(), f = tid % G8_BM, n = w.f0 + f;
      for (int c = rank + tid / G8_BM * splits; c < w.rows && tid < 2 * G8_BM; c += 2 * splits) {
        float v = 0.f;
        for (int r = 0; r < splits; ++r) v += g8_ld_cluster(part + (uint32_t)(c * G8_BM + f) * 4, (uint32_t)r);
        if (n < p.N) g8_store(p, w.m0 + c, n, v);
      }
    }
    g8_cluster_sync();      // no block leaves while its sums may be read
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

static int g8_sms() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 1;
}

template <int NT>
static int g8_launch(const CUtensorMap& mw, const CUtensorMap& mx, const G8Params& p, int blocks, int splits, cudaStream_t stream) {
  using C = G8Config<NT>;
  cudaError_t e = cudaFuncSetAttribute(gemm_fp8_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
  if (e != cudaSuccess) return llmrs_fail("gemm_fp8: shared memory %zu: %s", C::SMEM, cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, (unsigned)splits);
  cfg.blockDim = dim3(G8_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = (unsigned)splits;
  cfg.numAttrs = 1;
  if (g_llmrs_pdl) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  e = cudaLaunchKernelEx(&cfg, gemm_fp8_kernel<NT>, mw, mx, p);
  if (e != cudaSuccess) return llmrs_fail("gemm_fp8 launch: %s", cudaGetErrorString(e));
  return llmrs_launch_status("gemm_fp8");
}

// x: x_rows rows of K e4m3 numbers x_pitch bytes apart, xs their words of scales (word g of row r at
// g * xs_stride + r); w: groups * N rows, ws the same of them. tile_rows: the most rows of a tile of the list, or 0: dense
// (one group, no list).
LLMRS_API int llmrs_gemm_fp8(const void* x, long long x_pitch, const void* xs, long long xs_stride, int x_rows, const void* w,
                             long long w_pitch, const void* ws, long long ws_stride, void* out, long long ldo, int out_dtype, int epilogue, int N, int K, int groups,
                             const int* tiles, const int* n_tiles, int max_tiles, int tile_rows, int* error_flag,
                             cudaStream_t stream) {
  const bool grouped = tile_rows != 0;
  const char* what = grouped ? "gemm_fp8_grouped" : "gemm_fp8";
  LLMRS_REQUIRE(x_rows >= 0 && N > 0 && K > 0 && groups > 0, "%s: bad sizes", what);
  LLMRS_REQUIRE(x_pitch % 16 == 0 && w_pitch % 16 == 0 && x_pitch >= K && w_pitch >= K && (((uintptr_t)x | (uintptr_t)w) & 15) == 0,
                "%s: rows must start at multiples of 16 bytes", what);
  LLMRS_REQUIRE((((uintptr_t)xs | (uintptr_t)ws) & 3) == 0, "%s: scales must start at a multiple of 4 bytes", what);
  LLMRS_REQUIRE((long long)groups * N <= 0x7fffff00LL && K <= 0x7fffff00 && x_rows <= 0x7fffff00, "%s: too many rows", what);
  LLMRS_REQUIRE(epilogue == G8_STORE || (epilogue == G8_ADD && out_dtype == LLMRS_F32), "%s: unknown epilogue %d", what, epilogue);
  if (x_rows == 0 || (grouped && max_tiles == 0)) return 0;
  const int rows = grouped ? tile_rows : x_rows;
  const int nt = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  LLMRS_REQUIRE(!grouped || (tiles && n_tiles && tile_rows > 0 && tile_rows <= 256), "%s: a list of tiles of 1 to 256 rows, got %d", what, tile_rows);
  G8Params p = {};
  p.out = out, p.ldo = ldo, p.out_f32 = out_dtype == LLMRS_F32, p.epilogue = epilogue;
  p.xs = (const uint32_t*)xs, p.ws = (const uint32_t*)ws, p.xs_stride = xs_stride, p.ws_stride = ws_stride, p.x_rows = x_rows, p.w_rows = groups * N;
  p.N = N, p.n_f = (N - 1) / G8_BM + 1, p.n_t = (x_rows - 1) / nt + 1, p.nkb = (K - 1) / G8_BK + 1;
  p.x_box = nt < 32 ? nt : 32;
  p.tiles = grouped ? tiles : nullptr, p.n_tiles = n_tiles, p.max_tiles = max_tiles, p.groups = groups;
  p.error_flag = error_flag, p.wait_limit = llmrs_tc_wait_limit(), p.test_skip_kb = llmrs_tc_skipped_copy();
  const long long work = (long long)(grouped ? max_tiles : p.n_t) * p.n_f;
  LLMRS_REQUIRE(work <= 0x7fffffffLL, "%s: too many tiles", what);
  CUtensorMap mw, mx;
  if (const int rc = g8_map(&mw, w, (long long)groups * N, K, w_pitch, G8_BM)) return rc;
  if (const int rc = g8_map(&mx, x, x_rows, K, x_pitch, p.x_box)) return rc;
  const int sms = g8_sms();
  int splits = 1;
  if (nt <= 64)
    for (int s = 2; s <= 8; s *= 2)
      if (work * s <= sms && p.nkb / s >= 2) splits = s;
  const int blocks = splits > 1 ? (int)work : (int)(work < sms ? work : sms);
  switch (nt) {
    case 16: return g8_launch<16>(mw, mx, p, blocks, splits, stream);
    case 32: return g8_launch<32>(mw, mx, p, blocks, splits, stream);
    case 64: return g8_launch<64>(mw, mx, p, blocks, splits, stream);
    case 128: return g8_launch<128>(mw, mx, p, blocks, splits, stream);
    default: return g8_launch<256>(mw, mx, p, blocks, splits, stream);
  }
}
