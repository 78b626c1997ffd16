// Products of two microscaled 4-bit matrices on the 5th-generation tensor cores:
//
//   C[t, n] = sum_g 2^(xs[t, g] + ws[n, g] - 254) * sum_{k in group g} xc[t, k] wc[n, k] (+ bias[n]) (+ residual[t, n])
//
// The instruction (kind::mxf4, K = 64) takes codes as they are stored, from shared memory, and the powers of its two groups of 32
// from tensor memory, where row r of an operand has its powers in lane r % 32 of every quarter of the lanes, column r / 32: four
// groups per 32-bit column. Weight rows take the 128-row operand and rows of x the other, as in gemm_mx4.cu.
//
// Warps of a CTA: 0 loads codes by TMA, 1 issues, 2-5 bring the powers to shared memory, 6-9 write results. A row's powers for a
// step of 256 columns are eight bytes at any address; the thread that owns the row puts them where the copy to tensor memory (32
// lanes x 16 bytes, repeated for the four quarters) takes them: four groups of row r at (r % 32) * 16 + (r / 32) * 4. Where rows
// start on four bytes they come by cp.async, else through registers, a step ahead.
//
// 48 x 4096 x 12288 takes 13 us, by the latency of launch, loads and exchange (25 MB of weights); 8111 x 12288 x 4096 212 us under the power
// cap, powers laid out and all, 3.9 PFLOP/s, by the results: a tile has 16 steps of K.
#include "mx4_tile.cuh"

namespace {
using namespace pxl;

constexpr int kThreads = 320;
constexpr int kStep = 256;                       // columns of a stage
constexpr int kCodes = kTileRows * kStep / 2;    // bytes of the weights' codes in a stage
constexpr int kMaxStages = 8, kScaleBufs = 4;
constexpr int kAtom = 512;                       // bytes of four groups' powers of 128 rows

struct ScaleArgs {
  const uint8_t* xs;
  const uint8_t* ws;
  int row_bytes;  // K / 32
  int words;      // every row's powers start on four bytes
  // LAID: powers in the order of the stages, of a block of weight rows and of a tile of rows of x [step of K][128 rows]
  const uint8_t* laid_w;
  const uint8_t* laid_x;
};

__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}\n"
      :
      : "r"(d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(leader)
      : "memory");
}
// e2m1 x e2m1 with e8m0 powers, both K-major; `group` (0 or 2): the first of the two powers within a column
__device__ __forceinline__ uint32_t mx4_idesc(int n, uint32_t group) {
  return (group << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(kTileRows >> 7) << 27) | (group << 29);
}
// 512 bytes of powers -> four columns of every quarter of the lanes, in the order of the instructions around it
__device__ __forceinline__ void copy_powers(uint32_t tmem, uint32_t smem_at, uint32_t leader) {
  // rows of 16 bytes, eight rows 128 bytes apart, no swizzle
  const uint64_t desc = static_cast<uint64_t>((smem_at & 0x3ffffu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t"
      "}\n"
      :
      : "r"(tmem), "l"(desc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void copy_word(uint32_t dst, const uint8_t* src, int bytes) {  // of four; the rest become zeros
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <bool SPLIT, bool LAID>
__global__ void __launch_bounds__(kThreads, LAID ? 1 : 2) gemm_mx4_rows_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                                                    const __grid_constant__ CUtensorMap tmap_w, const ScaleArgs sc,
                                                                    int* status, const TileArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stage_bytes = kCodes + g.bt * (kStep / 2);
  const int halves = g.bt > 128 ? 2 : 1, power_bytes = 2 * (1 + halves) * kAtom;  // of a stage: [weights, rows of x][128 rows][word]
  uint8_t* powers = smem + g.stages * stage_bytes;
  float* staging = reinterpret_cast<float*>(powers + g.stages * power_bytes);
  __shared__ __align__(8) uint64_t bars[3 * kMaxStages + 2 * 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, sfull0 = empty0 + 8 * kMaxStages,
                 dfull0 = sfull0 + 8 * kMaxStages, dempty0 = dfull0 + 16;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int x_cols = 4 * halves, scale_cols = 8 + 2 * x_cols;  // columns of powers: per four groups of x's rows; per step
  const int tmem_cols = g.d_bufs * g.d_cols + kScaleBufs * scale_cols > 256 ? 512 : 256;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < g.stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1), mbar_init(sfull0 + 8 * s, 128);
    for (int b = 0; b < g.d_bufs; ++b) mbar_init(dfull0 + 8 * b, 1), mbar_init(dempty0 + 8 * b, LAID ? 8 : 4);
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot, tmem_s = tmem + g.d_bufs * g.d_cols;

  const int items = g.n_blocks * g.t_tiles;
  const int i0 = SPLIT ? blockIdx.x / g.splits : blockIdx.x, i_step = SPLIT ? items : gridDim.x;
  const int kb0 = SPLIT ? static_cast<int>(cluster_cta_rank()) * g.kb_per : 0;
  const int kb1 = SPLIT ? min(kb0 + g.kb_per, g.k_blocks) : g.k_blocks;

  const uint32_t stage_tx = stage_bytes + (LAID ? power_bytes : 0);
  pdl_wait();  // (either operand may be of rows that the kernel before quantises)
  pdl_launch_dependents();

  if (warp == 0) {
    const uint32_t leader = elect_leader(), s0 = smem_u32(smem);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, nullptr);
      for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t fb = full0 + 8 * stage, at = s0 + stage * stage_bytes;
        ok = wait_parked(empty0 + 8 * stage, phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_EMPTY);
        if (!ok) break;
        expect_tx(fb, stage_tx, leader);
        tma_box(at, &tmap_w, fb, kb * (kStep / 2), it.n_blk * kTileRows, leader);
        tma_box(at + kCodes, &tmap_x, fb, kb * (kStep / 2), it.row0, leader);
        if (LAID && leader) {
          const uint32_t to = smem_u32(powers) + stage * power_bytes;
          bulk_load_g2s(to, sc.laid_w + (static_cast<int64_t>(it.n_blk) * g.k_blocks + kb) * (2 * kAtom), 2 * kAtom, fb);
          bulk_load_g2s(to + 2 * kAtom, sc.laid_x + (static_cast<int64_t>(it.row0 / g.bt) * g.k_blocks + kb) * (2 * halves * kAtom),
                        2 * halves * kAtom, fb);
        }
        if (++stage == g.stages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    int stage = 0, sb = 0, db = 0;
    uint32_t phase = 0, d_phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, nullptr);
      const int cols = ceil_div(it.rows, 16) * 16;
      const uint32_t idesc0 = mx4_idesc(cols, 0), idesc2 = mx4_idesc(cols, 2);
      ok = wait_parked(dempty0 + 8 * db, d_phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
      for (int kb = kb0; ok && kb < kb1; ++kb) {
        ok = wait_parked(full0 + 8 * stage, phase, abort_flag, status, PXL_DEV_TIMEOUT_FULL) &&
             (LAID || wait_parked(sfull0 + 8 * stage, phase, abort_flag, status, PXL_DEV_TIMEOUT_FULL));
        if (!ok) break;
        if (!LAID) fence_proxy_async_smem();
        tc_fence_after_sync();
        const uint64_t da = umma_desc_k_sw128(smem_u32(smem) + stage * stage_bytes);
        const uint64_t dx = umma_desc_k_sw128(smem_u32(smem) + stage * stage_bytes + kCodes);
        const uint32_t sfa = tmem_s + sb * scale_cols, sfx = sfa + 8, from = smem_u32(powers) + stage * power_bytes;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          copy_powers(sfa + 4 * j, from + j * kAtom, leader);
          copy_powers(sfx + x_cols * j, from + (2 + j) * kAtom, leader);
          if (halves == 2) copy_powers(sfx + x_cols * j + 4, from + (4 + j) * kAtom, leader);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_mx4(tmem + db * g.d_cols, da + 2 * k, dx + 2 * k, k & 1 ? idesc2 : idesc0, sfa + (k >> 1) * 4, sfx + (k >> 1) * x_cols,
                  kb > kb0 || k > 0 ? 1u : 0u, leader);
        commit(empty0 + 8 * stage, leader);
        if (++stage == g.stages) stage = 0, phase ^= 1;
        if (++sb == kScaleBufs) sb = 0;
      }
      if (!ok) break;
      commit(dfull0 + 8 * db, leader);
      if (++db == g.d_bufs) db = 0, d_phase ^= 1;
    }
  } else if (!LAID && warp < 6) {
    // ---- powers: of weight row tid, and of rows tid and 128 + tid of x
    const int tid = static_cast<int>(threadIdx.x) - 64, parts = 1 + halves;
    const uint32_t at = smem_u32(powers) + (tid & 31) * 16 + (tid >> 5) * 4;
    auto row_of = [&](const Item& it, int p, const uint8_t*& src) {
      const int row = p == 0 ? it.n_blk * kTileRows + tid : (p - 1) * 128 + tid;
      src = p == 0 ? sc.ws + static_cast<int64_t>(row) * sc.row_bytes : sc.xs + static_cast<int64_t>(it.row0 + row) * sc.row_bytes;
      return p == 0 ? row < g.N : row < it.rows;
    };
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, nullptr);
      const uint8_t* src[3];
      bool in[3];
#pragma unroll
      for (int p = 0; p < 3; ++p)
        if (p < parts) in[p] = row_of(it, p, src[p]);
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = wait_parked(empty0 + 8 * stage, phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_EMPTY);
        if (!ok) break;
        const int bytes = min(8, sc.row_bytes - kb * 8);  // behind the last group: zeros, a finite power for codes of 0
        const uint32_t dst = at + stage * power_bytes;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          if (p >= parts) break;
          const uint8_t* from = src[p] + kb * 8;
          const int n = in[p] ? bytes : 0;
          if (sc.words) {
            copy_word(dst + 2 * p * kAtom, n > 0 ? from : sc.ws, min(n, 4));
            copy_word(dst + (2 * p + 1) * kAtom, n > 4 ? from + 4 : sc.ws, max(n - 4, 0));
          } else {  // the words that hold them, no further than the last byte's
            const int off = static_cast<int>(reinterpret_cast<uintptr_t>(from) & 3);
            const uint32_t* words = reinterpret_cast<const uint32_t*>(from - off);
            const uint32_t w0 = n > 0 ? __ldg(words) : 0, w1 = n + off > 4 ? __ldg(words + 1) : 0, w2 = n + off > 8 ? __ldg(words + 2) : 0;
            uint32_t lo = __funnelshift_r(w0, w1, off * 8), hi = __funnelshift_r(w1, w2, off * 8);
            if (n < 8) hi = n <= 4 ? 0u : hi & ((1u << (8 * (n - 4))) - 1u);
            if (n < 4) lo &= (1u << (8 * n)) - 1u;
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + 2 * p * kAtom), "r"(lo) : "memory");
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + (2 * p + 1) * kAtom), "r"(hi) : "memory");
          }
        }
        // (every thread arrives once its own are there; the warp that issues orders them before the tensor core's reads)
        if (sc.words) asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sfull0 + 8 * stage) : "memory");
        else mbar_arrive(sfull0 + 8 * stage);
        if (++stage == g.stages) stage = 0, phase ^= 1;
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
  } else {
    // (with the powers laid out ahead, both fours of warps write results)
    const int group = LAID ? (warp - 2) >> 2 : 0;
    write_results<SPLIT, true>(g, nullptr, i0, i_step, items, kb0 == 0, tmem, dfull0, dempty0, reinterpret_cast<float*>(smem),
                               staging + group * (kStaging / 4), group, LAID ? 2 : 1, warp & 3, lane, abort_flag, status);
  }

  if constexpr (SPLIT) {
    // Every thread of every CTA passes both barriers, also after a failed wait (all other waits are bounded).
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2) add_ranges(g, i0, smem_u32(smem), static_cast<int>(threadIdx.x) - 64, kThreads - 64, abort_flag);
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are being read
  }
  __syncwarp();
  if (*abort_flag) __nanosleep(200000);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, tmem_cols);
}

constexpr int kLaySteps = 4;
// Scales [R, row_bytes] -> the stages' order: for every tile of `per` rows and step of K, 1 or 2 times 128 rows' eight bytes as they
// go to tensor memory; zeros (a finite power, for codes of 0) where there are no rows or groups. A block: 128 rows, four steps.
__global__ void __launch_bounds__(256) mx4_lay_powers_kernel(const uint8_t* __restrict__ ws, int w_rows, const uint8_t* __restrict__ xs,
                                                             int x_rows, int x_per, int x_halves, int row_bytes, int steps, int w_tiles,
                                                             uint8_t* __restrict__ laid_w, uint8_t* __restrict__ laid_x) {
  __shared__ __align__(16) uint32_t out[kLaySteps * 256];
  pdl_wait();
  pdl_launch_dependents();
  const bool is_x = static_cast<int>(blockIdx.x) >= w_tiles;
  const int t = is_x ? blockIdx.x - w_tiles : blockIdx.x, halves = is_x ? x_halves : 1, half = t % halves, tile = t / halves;
  const int per = is_x ? x_per : kTileRows, step0 = blockIdx.y * kLaySteps;
  const uint8_t* s = is_x ? xs : ws;
#pragma unroll
  for (int i = threadIdx.x; i < 128 * 2 * kLaySteps; i += 256) {
    const int r = i / (2 * kLaySteps), w = i % (2 * kLaySteps), row = tile * per + half * 128 + r, at = step0 * 8 + w * 4;
    uint32_t v = 0;
    if (half * 128 + r < per && row < (is_x ? x_rows : w_rows) && at < row_bytes) {
      const uint8_t* p = s + static_cast<int64_t>(row) * row_bytes + at;
      const int n = min(4, row_bytes - at), off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
      const uint32_t* words = reinterpret_cast<const uint32_t*>(p - off);  // (no further than the last byte's)
      v = __funnelshift_r(__ldg(words), off + n > 4 ? __ldg(words + 1) : 0u, off * 8);
      if (n < 4) v &= (1u << (8 * n)) - 1u;
    }
    out[(w >> 1) * 256 + (w & 1) * 128 + (r & 31) * 4 + (r >> 5)] = v;
  }
  __syncthreads();
  const int count = min(kLaySteps, steps - step0);
  uint8_t* dst = (is_x ? laid_x : laid_w) + ((static_cast<int64_t>(tile) * steps + step0) * halves + half) * (2 * kAtom);
  for (int i = threadIdx.x; i < count * 64; i += 256)
    *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(i >> 6) * halves * (2 * kAtom) + (i & 63) * 16) = reinterpret_cast<const uint4*>(out)[i];
}

// Width of the token tiles for more than 256 tokens. A tile's time is that of 92 tokens more than it has (128, 160, 192: 0.77, 0.88, 1);
// beyond 192 there is one accumulator, and no products hide its results (224, 256: 1.35, 1.54 for 16 steps of K, 1.25, 1.44 for 48). A
// last round that is not full takes about the mean of a round and of its part of one. 8192 x 12288 x 4096 in tiles of 160 tokens 230 us,
// 192 211, 256 246; 1000 x 8192 x 12288 66, 62, 60; 1500 x 5120 x 25600 114, 115, 111, and 98 in tiles of 224.
int tile_tokens(int M, int n_blocks, int steps) {
  const int sms = pxl_host::num_sms();
  int best = 192;
  int64_t least = INT64_MAX;
  for (int bt = 96; bt <= 256; bt += 16) {
    const int64_t tiles = static_cast<int64_t>(pxl::ceil_div(M, bt)) * n_blocks, rounds = (tiles + sms - 1) / sms;
    const int64_t time = bt <= 192 ? 20 * (bt + 92) : 31 * bt + 13200 / steps;
    const int64_t cost = (rounds * sms + tiles) * time;
    if (cost <= least) least = cost, best = bt;
  }
  return best;
}

struct RowsPlan {
  TileArgs g;
  int64_t items;
  int slots, laid;
};
// Tiles of tokens and how their powers are brought in; the same for the workspace's size and the launch. Rows of x that share their
// powers' copies with few others take them from where they are (one launch less); with more than 128 the copies, of four bytes here
// and there, would be what bounds the kernel (8111 x 12288 x 4096: 336 us, 212 with the powers laid out ahead; 3484 x 28286 x 768 126, 87).
bool plan_rows(RowsPlan& p, int M, int N, int K) {
  static bool configured[64] = {};
  if (!pxl_host::allow_smem(configured, gemm_mx4_rows_kernel<false, false>, gemm_mx4_rows_kernel<true, false>, gemm_mx4_rows_kernel<false, true>))
    return false;
  TileArgs& g = p.g;
  g.M = M, g.N = N;
  g.n_blocks = pxl::ceil_div(N, kTileRows), g.k_blocks = pxl::ceil_div(K, kStep);
  // One tile for up to 256 tokens (us, one and two): 96 x 5120 x 25600 26 and 32, 203 29 and 50, 256 39 and 53; 128 x 25600 x 5120 27 and 25,
  // 256 34 and 31; 128 x 12288 x 4096 15 and 19, 256 18 and 19; 203 x 4096 x 4096 15.7 and 13.3.
  g.t_tiles = M <= 256 ? 1 : pxl::ceil_div(M, tile_tokens(M, g.n_blocks, g.k_blocks));
  g.bt = pxl::ceil_div(pxl::ceil_div(M, g.t_tiles), 16) * 16;
  g.t_group = g.t_tiles;
  p.items = static_cast<int64_t>(g.n_blocks) * g.t_tiles;
  const int sms = pxl_host::num_sms();
  const bool two = g.bt <= 64;  // CTAs per SM, as in gemm_mx4.cu
  p.slots = two ? 2 * sms : sms;
  g.d_cols = pxl::ceil_div(g.bt, 32) * 32;
  g.d_bufs = !two && g.d_cols <= 192 ? 2 : 1;
  pxl_host::split_k(g, p.items, p.slots, 6, gemm_mx4_rows_kernel<true, false>, kThreads);
  p.laid = g.splits == 1 && M > 128;
  return true;
}

}  // namespace

// bytes of scratch that pxl_gemm_mx4_rows needs
PXL_EXPORT int64_t pxl_gemm_mx4_rows_workspace(int M, int N, int K) {
  RowsPlan p{};
  if (M <= 0 || N <= 0 || K <= 0 || !plan_rows(p, M, N, K) || !p.laid) return 0;
  return (static_cast<int64_t>(p.g.n_blocks) + static_cast<int64_t>(p.g.t_tiles) * (p.g.bt > 128 ? 2 : 1)) * p.g.k_blocks * (2 * kAtom);
}

PXL_EXPORT int pxl_gemm_mx4_rows(const void* xc, const void* xs, const void* wc, const void* ws, void* C, int64_t ldc,
                                 const void* bias, const void* residual, int64_t ldr, int M, int N, int K, void* workspace,
                                 int64_t workspace_bytes, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 32 || !pxl_host::on16(xc, 0) || !pxl_host::on16(wc, 0)) return PXL_ERR_INVALID_ARG;
  RowsPlan p{};
  if (!plan_rows(p, M, N, K)) return PXL_ERR_CUDA;
  TileArgs& g = p.g;
  if (p.items > 0x7fffffff) return PXL_ERR_TOO_LARGE;
  if (p.laid && (!pxl_host::on16(workspace, 0) || workspace == nullptr || workspace_bytes < pxl_gemm_mx4_rows_workspace(M, N, K)))
    return PXL_ERR_INVALID_ARG;
  g.C = C, g.ldc = ldc, g.bias = static_cast<const bf16*>(bias), g.residual = static_cast<const bf16*>(residual), g.ldr = ldr;
  g.vec = pxl_host::on16(C, 2 * ldc) && (!residual || pxl_host::on16(residual, 2 * ldr));
  ScaleArgs sc{static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(ws), K / 32, 0};
  sc.words = !((reinterpret_cast<uintptr_t>(xs) | reinterpret_cast<uintptr_t>(ws) | static_cast<uintptr_t>(K / 32)) & 3);
  const int halves = g.bt > 128 ? 2 : 1;
  const int stage_bytes = kCodes + g.bt * (kStep / 2) + 2 * (1 + halves) * kAtom;
  const int rest = 1024 + (g.splits > 1 ? 0 : p.laid ? 2 * kStaging : kStaging);
  g.stages = ((p.slots > pxl_host::num_sms() ? 113 * 1024 : pxl_host::kTileSmem) - 512 - rest) / stage_bytes;
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  if (g.stages < 1) return PXL_ERR_TOO_LARGE;
  int smem = rest + g.stages * stage_bytes;
  if (g.splits > 1 && smem < 1024 + g.bt * kPitch * 4) smem = 1024 + g.bt * kPitch * 4;
  CUtensorMap tx, tw;
  if (!pxl_host::make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xc, M, K / 2, K / 2, g.bt, kStep / 2) ||
      !pxl_host::make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wc, N, K / 2, K / 2, kTileRows, kStep / 2))
    return PXL_ERR_TENSORMAP;
  if (p.laid) {
    uint8_t* const laid_w = static_cast<uint8_t*>(workspace);
    uint8_t* const laid_x = laid_w + static_cast<int64_t>(g.n_blocks) * g.k_blocks * (2 * kAtom);
    sc.laid_w = laid_w, sc.laid_x = laid_x;
    pxl_host::launch(mx4_lay_powers_kernel, dim3(g.n_blocks + g.t_tiles * halves, pxl::ceil_div(g.k_blocks, kLaySteps)), 256, 0, stream, sc.ws, N,
                     sc.xs, M, g.bt, halves, sc.row_bytes, g.k_blocks, g.n_blocks, laid_w, laid_x);
    return pxl_host::launch_tiles(gemm_mx4_rows_kernel<false, true>, gemm_mx4_rows_kernel<true, false>, g, static_cast<int>(p.items), p.slots,
                                  kThreads, smem, stream, tx, tw, sc, status);
  }
  return pxl_host::launch_tiles(gemm_mx4_rows_kernel<false, false>, gemm_mx4_rows_kernel<true, false>, g, static_cast<int>(p.items), p.slots,
                                kThreads, smem, stream, tx, tw, sc, status);
}
