// Products of two microscaled 4-bit matrices on the 5th-generation tensor cores:
//
//   C[t, n] = sum_g 2^(xs[t, g] + ws[n, g] - 254) * sum_{k in group g} xc[t, k] wc[n, k] (+ bias[n]) (+ residual[t, n])
//
// The instruction (kind::mxf4, K = 64) takes codes as they are stored, from shared memory, and the powers of its two groups of 32
// from tensor memory, where row r of an operand has its powers in lane r % 32 of every quarter of the lanes, column r / 32: four
// groups per 32-bit column. Weight rows take the 128-row operand and rows of x the other, as in gemm_mx4.cu.
//
// Warps of a CTA: 0 loads codes by TMA, 1 issues, 2-5 bring the powers into tensor memory, 6-9 write results. A row's powers for
// a step of 256 columns are eight bytes at any address: a thread copies them (cp.async, three steps ahead) from the rows that it
// owns, and takes those that its lane needs from shared memory.
#include "mx4_tile.cuh"

namespace {
using namespace pxl;

constexpr int kThreads = 320;
constexpr int kStep = 256;                       // columns of a stage
constexpr int kCodes = kTileRows * kStep / 2;    // bytes of the weights' codes in a stage
constexpr int kMaxStages = 8, kRing = 4, kScaleBufs = 4;

struct ScaleArgs {
  const uint8_t* xs;
  const uint8_t* ws;
  int row_bytes;  // K / 32
  int whole;      // every row's eight bytes start on eight bytes
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
__device__ __forceinline__ void tmem_st_x4(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void copy_async(uint32_t dst, const uint8_t* src, int bytes, bool eight) {  // the rest becomes zeros
  if (eight) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2) gemm_mx4_rows_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                                                    const __grid_constant__ CUtensorMap tmap_w, const ScaleArgs sc,
                                                                    int* status, const TileArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stage_bytes = kCodes + g.bt * (kStep / 2);
  float* staging = reinterpret_cast<float*>(smem + g.stages * stage_bytes);
  uint8_t* ring = reinterpret_cast<uint8_t*>(staging) + (SPLIT ? 0 : kStaging);
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 2 * kScaleBufs + 2 * 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, sfull0 = empty0 + 8 * kMaxStages,
                 sempty0 = sfull0 + 8 * kScaleBufs, dfull0 = sempty0 + 8 * kScaleBufs, dempty0 = dfull0 + 16;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int x_cols = g.bt > 128 ? 8 : 4, scale_cols = 8 + 2 * x_cols;  // columns of powers: per four groups of x's rows; per step
  const int tmem_cols = g.d_bufs * g.d_cols + kScaleBufs * scale_cols > 256 ? 512 : 256;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < g.stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    for (int b = 0; b < kScaleBufs; ++b) mbar_init(sfull0 + 8 * b, 4), mbar_init(sempty0 + 8 * b, 1);
    for (int b = 0; b < g.d_bufs; ++b) mbar_init(dfull0 + 8 * b, 1), mbar_init(dempty0 + 8 * b, 4);
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

  if (warp == 0 && lane == 0 && g.early) {
    const Item it = item_of(i0, g, nullptr);
    for (int s = 0; s < g.stages && kb0 + s < kb1; ++s) {
      mbar_arrive_expect_tx(full0 + 8 * s, stage_bytes);
      tma_load_2d(smem_u32(smem) + s * stage_bytes, &tmap_w, full0 + 8 * s, (kb0 + s) * (kStep / 2), it.n_blk * kTileRows);
    }
  }
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    const uint32_t leader = elect_leader(), s0 = smem_u32(smem);
    int stage = 0, done = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, nullptr);
      for (int kb = kb0; kb < kb1; ++kb, ++done) {
        const uint32_t fb = full0 + 8 * stage, at = s0 + stage * stage_bytes;
        if (!g.early || done >= g.stages) {
          ok = wait_warp(empty0 + 8 * stage, phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_EMPTY);
          if (!ok) break;
          expect_tx(fb, stage_bytes, leader);
          tma_box(at, &tmap_w, fb, kb * (kStep / 2), it.n_blk * kTileRows, leader);
        }
        tma_box(at + kCodes, &tmap_x, fb, kb * (kStep / 2), it.row0, leader);
        if (++stage == g.stages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_leader();
    int stage = 0, sb = 0, db = 0;
    uint32_t phase = 0, s_phase = 0, d_phase = 0;
    bool ok = true;
    for (int i = i0; ok && i < items; i += i_step) {
      const Item it = item_of(i, g, nullptr);
      const int cols = ceil_div(it.rows, 16) * 16;
      const uint32_t idesc0 = mx4_idesc(cols, 0), idesc2 = mx4_idesc(cols, 2);
      ok = wait_warp(dempty0 + 8 * db, d_phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
      for (int kb = kb0; ok && kb < kb1; ++kb) {
        ok = wait_warp(full0 + 8 * stage, phase, abort_flag, status, PXL_DEV_TIMEOUT_FULL) &&
             wait_warp(sfull0 + 8 * sb, s_phase, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t da = umma_desc_k_sw128(smem_u32(smem) + stage * stage_bytes);
        const uint64_t dx = umma_desc_k_sw128(smem_u32(smem) + stage * stage_bytes + kCodes);
        const uint32_t sfa = tmem_s + sb * scale_cols, sfx = sfa + 8;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_mx4(tmem + db * g.d_cols, da + 2 * k, dx + 2 * k, k & 1 ? idesc2 : idesc0, sfa + (k >> 1) * 4, sfx + (k >> 1) * x_cols,
                  kb > kb0 || k > 0 ? 1u : 0u, leader);
        commit(empty0 + 8 * stage, leader);
        commit(sempty0 + 8 * sb, leader);
        if (++stage == g.stages) stage = 0, phase ^= 1;
        if (++sb == kScaleBufs) sb = 0, s_phase ^= 1;
      }
      if (!ok) break;
      commit(dfull0 + 8 * db, leader);
      if (++db == g.d_bufs) db = 0, d_phase ^= 1;
    }
  } else if (warp < 6) {
    // ---- powers. After a wait that ran out the loop goes on: the warps meet at the barrier of every step.
    const int q = warp & 3, tid = static_cast<int>(threadIdx.x) - 64;
    const int pitch = sc.whole ? 8 : 12, parts = g.bt > 128 ? 3 : 2, slot_bytes = (128 * parts) * pitch;
    const uint32_t ring0 = smem_u32(ring);
    auto fetch = [&](const Item& it, int kb, int slot) {  // rows tid (of 128) of the weights, of x's first and second 128
      const int bytes = min(8, sc.row_bytes - kb * 8);
      for (int p = 0; p < parts; ++p) {
        const int row = p == 0 ? it.n_blk * kTileRows + tid : (p - 1) * 128 + tid;
        const bool in = p == 0 ? row < g.N : row < it.rows;
        const uint8_t* src = p == 0 ? sc.ws + static_cast<int64_t>(row) * sc.row_bytes : sc.xs + static_cast<int64_t>(it.row0 + row) * sc.row_bytes;
        src += kb * 8;
        const uint32_t dst = ring0 + slot * slot_bytes + (p * 128 + tid) * pitch;
        if (sc.whole) {
          copy_async(dst, in ? src : sc.ws, in ? bytes : 0, true);
        } else {  // the words that hold them: no further than the last byte's
          const int off = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 3);
          for (int w = 0; w < 3; ++w) {
            const bool need = in && 4 * w < off + bytes;
            copy_async(dst + 4 * w, need ? src - off + 4 * w : sc.ws - (reinterpret_cast<uintptr_t>(sc.ws) & 3), need ? 4 : 0, false);
          }
        }
      }
    };
    auto take = [&](const Item& it, int kb, int slot, int p, int row, uint32_t& lo, uint32_t& hi) {
      const uint32_t at = ring0 + slot * slot_bytes + (p * 128 + row) * pitch;
      uint32_t w0, w1, w2 = 0;
      if (sc.whole) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(lo), "=r"(hi) : "r"(at));
        return;
      }
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w0) : "r"(at));
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w1) : "r"(at + 4));
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w2) : "r"(at + 8));
      const uintptr_t src = p == 0 ? reinterpret_cast<uintptr_t>(sc.ws) + static_cast<int64_t>(it.n_blk * kTileRows + row) * sc.row_bytes
                                   : reinterpret_cast<uintptr_t>(sc.xs) + static_cast<int64_t>(it.row0 + (p - 1) * 128 + row) * sc.row_bytes;
      const uint32_t off = static_cast<uint32_t>(src + kb * 8) & 3u;
      lo = __funnelshift_r(w0, w1, off * 8), hi = __funnelshift_r(w1, w2, off * 8);
      const int bytes = min(8, sc.row_bytes - kb * 8);  // what follows is another row's, or nothing: any finite power for codes of 0
      if (bytes < 8) hi = bytes <= 4 ? 0u : hi & ((1u << (8 * (bytes - 4))) - 1u);
      if (bytes < 4) lo &= (1u << (8 * bytes)) - 1u;
    };
    int ni = i0, nkb = kb0, n_slot = 0;
    Item next = item_of(min(i0, items - 1), g, nullptr);
    auto ahead = [&]() {
      if (ni < items) {
        fetch(next, nkb, n_slot);
        if (++nkb == kb1) {
          nkb = kb0, ni += i_step;
          if (ni < items) next = item_of(ni, g, nullptr);
        }
      }
      cp_async_commit();
      n_slot = (n_slot + 1) % kRing;
    };
    for (int s = 0; s < kRing - 1; ++s) ahead();
    int sb = 0, slot = 0;
    uint32_t s_phase = 0;
    bool ok = true;
    for (int i = i0; i < items; i += i_step) {
      const Item it = item_of(i, g, nullptr);
      for (int kb = kb0; kb < kb1; ++kb) {
        cp_async_wait<kRing - 2>();
        named_bar_sync(2, 128);
        ahead();  // into the slot of the step before, which every warp has left
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) take(it, kb, slot, 0, 32 * c + lane, lo[c], hi[c]);
        ok = ok && wait_warp(sempty0 + 8 * sb, s_phase ^ 1, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_EMPTY);
        tc_fence_after_sync();
        const uint32_t dst = tmem_s + sb * scale_cols + (static_cast<uint32_t>(q * 32) << 16);
        tmem_st_x4(dst, lo);
        tmem_st_x4(dst + 4, hi);
        for (int p = 1; p < parts; ++p) {
#pragma unroll
          for (int c = 0; c < 4; ++c) take(it, kb, slot, p, 32 * c + lane, lo[c], hi[c]);
          tmem_st_x4(dst + 8 + (p - 1) * 4, lo);
          tmem_st_x4(dst + 8 + x_cols + (p - 1) * 4, hi);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(sfull0 + 8 * sb);
        if (++sb == kScaleBufs) sb = 0, s_phase ^= 1;
        slot = (slot + 1) % kRing;
      }
    }
    cp_async_wait<0>();
  } else {
    write_results<SPLIT>(g, nullptr, i0, i_step, items, kb0 == 0, tmem, dfull0, dempty0, reinterpret_cast<float*>(smem), staging, warp & 3, lane,
                         static_cast<int>(threadIdx.x) - 192, abort_flag, status);
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

}  // namespace

PXL_EXPORT int pxl_gemm_mx4_rows(const void* xc, const void* xs, const void* wc, const void* ws, void* C, int64_t ldc,
                                 const void* bias, const void* residual, int64_t ldr, int M, int N, int K, int* status,
                                 cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 32 || !pxl_host::on16(xc, 0) || !pxl_host::on16(wc, 0)) return PXL_ERR_INVALID_ARG;
  TileArgs g{};
  g.C = C, g.ldc = ldc, g.bias = static_cast<const bf16*>(bias), g.residual = static_cast<const bf16*>(residual), g.ldr = ldr;
  g.M = M, g.N = N;
  g.n_blocks = pxl::ceil_div(N, kTileRows), g.k_blocks = pxl::ceil_div(K, kStep);
  g.t_tiles = pxl::ceil_div(M, 256);
  g.bt = pxl::ceil_div(pxl::ceil_div(M, g.t_tiles), 16) * 16;
  g.vec = pxl_host::on16(C, 2 * ldc) && (!residual || pxl_host::on16(residual, 2 * ldr));
  const int64_t items = static_cast<int64_t>(g.n_blocks) * g.t_tiles;
  if (items > 0x7fffffff) return PXL_ERR_TOO_LARGE;
  const int sms = pxl_host::num_sms();
  const bool two = g.bt <= 128;  // CTAs per SM, as in gemm_mx4.cu
  const int slots = two ? 2 * sms : sms;
  g.d_bufs = 1;
  g.d_cols = pxl::ceil_div(g.bt, 32) * 32;
  pxl_host::split_k(g, static_cast<int>(items), slots, 2);
  ScaleArgs sc{static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(ws), K / 32, 0};
  sc.whole = !((reinterpret_cast<uintptr_t>(xs) | reinterpret_cast<uintptr_t>(ws) | static_cast<uintptr_t>(K / 32)) & 7);
  const int stage_bytes = kCodes + g.bt * (kStep / 2);
  const int rest = 1024 + kRing * 128 * (g.bt > 128 ? 3 : 2) * (sc.whole ? 8 : 12) + (g.splits > 1 ? 0 : kStaging);
  g.stages = ((two ? 113 : 226) * 1024 - 512 - rest) / stage_bytes;
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  if (g.stages < 1) return PXL_ERR_TOO_LARGE;
  int smem = rest + g.stages * stage_bytes;
  if (g.splits > 1 && smem < 1024 + g.bt * kPitch * 4) smem = 1024 + g.bt * kPitch * 4;
  CUtensorMap tx, tw;
  if (!pxl_host::make_tmap_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xc, M, K / 2, K / 2, g.bt, kStep / 2) ||
      !pxl_host::make_tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, wc, N, K / 2, K / 2, kTileRows, kStep / 2))
    return PXL_ERR_TENSORMAP;
  static bool configured[64] = {false};
  return pxl_host::launch_tiles(gemm_mx4_rows_kernel<false>, gemm_mx4_rows_kernel<true>, configured, g, static_cast<int>(items), slots,
                                kThreads, smem, stream, 226 * 1024, tx, tw, sc, status);
}
