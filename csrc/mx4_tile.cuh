// Output tiles of the products with microscaled weights: 128 weight rows (lanes of the accumulator) by up to 256 rows of x, called
// tokens here (its columns). What a launch's work items are, and how their results leave tensor memory.
#pragma once

#include "mx4.cuh"
#include "tc_issue.cuh"

namespace pxl {

constexpr int kPitch = kTileRows + 4;  // floats of a token's results in shared memory
constexpr int kChunk = 32;             // tokens whose results are written at a time
constexpr int kStaging = kChunk * kPitch * 4;  // of the four warps that write (also: two chunks' halves of 64 rows)

template <bool B>
struct Bool {
  static constexpr bool value = B;
};

// Warp-collective wait, the same result in every lane. The hardware parks the warp for up to the hint's time, so that a wait costs
// three instructions: expanding 4-bit weights is bound by the instructions that a SM issues.
__device__ __forceinline__ uint32_t wait_hinted(uint32_t bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(ns)
      : "memory");
  return ok;
}
static __device__ __noinline__ bool wait_again(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  const uint64_t t0 = global_timer_ns();
  while (true) {
    if (wait_hinted(bar, parity, 100000u)) return true;
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      if (status) atomicCAS(status, 0, code);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait_parked(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, wait_hinted(bar, parity, 100000u))) return true;
  return __all_sync(0xffffffffu, wait_again(bar, parity, abort_flag, status, code)) != 0;
}

struct TileArgs {
  void* C;
  const float* row_scale;  // [experts, N rounded up to 128], or none
  const bf16* bias;
  const bf16* residual;
  int64_t ldc, ldr;
  int M, N, epi, out_f32;
  float limit;
  int n_blocks, k_blocks, t_tiles;
  int t_group;             // tiles of tokens that go through all weights together
  int bt;                  // tokens of a tile, a multiple of 16
  int stages, d_bufs, d_cols;
  int splits, kb_per;      // SPLIT: CTAs of a cluster, one per range of K blocks
  const int* offsets;      // grouped: first row of every expert, and the end
  int experts;
  int vec;                 // SPLIT, STAGED: results and residual may be taken in whole 16-byte vectors
  int early;               // in a launch chain: weights of the first tile may be read ahead of the wait
};

struct Item {
  int n_blk, row0, rows, expert;
};

// Item i of the launch: a block of weight rows, and a tile of tokens. Tiles of tokens of a group follow one another for a block of
// weights, unless there are experts: then the blocks of an expert's weights follow for a tile.
__device__ __forceinline__ Item item_of(int i, const TileArgs& g, const int* first_tile) {
  Item it;
  if (g.offsets == nullptr) {
    const int per = g.t_group * g.n_blocks, first = i / per * g.t_group, wide = min(g.t_group, g.t_tiles - first), at = i % per;
    it.n_blk = at / wide;
    it.row0 = (first + at % wide) * g.bt;
    it.rows = min(g.bt, g.M - it.row0);
    it.expert = 0;
    return it;
  }
  const int tile = i / g.n_blocks;
  it.n_blk = i % g.n_blocks;
  int lo = 0, hi = g.experts;  // the last expert whose first tile is not behind `tile`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile[mid] <= tile) lo = mid;
    else hi = mid;
  }
  it.expert = lo;
  it.row0 = g.offsets[lo] + (tile - first_tile[lo]) * g.bt;
  it.rows = min(g.bt, g.offsets[lo + 1] - it.row0);
  return it;
}

// SPLIT, STAGED: the residual of eight results in one vector, where there is one; asked for ahead of the results, because its way from
// memory takes as long as a chunk of them.
__device__ __forceinline__ bf16x8 residual8(const TileArgs& g, bool glu, int n_blk, int t, int c) {
  const int n0 = n_blk * (glu ? 64 : 128) + c;
  bf16x8 v = {};
  if (g.residual && g.vec && n0 + 8 <= (glu ? g.N / 2 : g.N)) v = ld_bf16x8(g.residual + t * g.ldr + n0);
  return v;
}
// Eight results of a token, columns c .. c + 7 of the block (of its 64 outputs, where it is gated), in bf16.
__device__ __forceinline__ void finish8(const TileArgs& g, float (&f)[16], bool glu, int n_blk, int t, int c, const bf16x8& v) {
  const int n0 = n_blk * (glu ? 64 : 128) + c, n_out = glu ? g.N / 2 : g.N;
  if (n0 >= n_out) return;
  if (glu) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = mx4_gate(f[j], f[8 + j], g.epi, g.limit);
  }
  const bool whole = g.vec && n0 + 8 <= n_out;
  if (g.residual) {
    const bf16* r = g.residual + t * g.ldr + n0;
    if (whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 p = unpack_bf16x2(v.u[j]);
        f[2 * j] += p.x, f[2 * j + 1] += p.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n0 + j < n_out) f[j] += __bfloat162float(r[j]);
    }
  }
  bf16* dst = static_cast<bf16*>(g.C) + t * g.ldc + n0;
  if (whole) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.u[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
    st_bf16x8(dst, o);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n0 + j < n_out) dst[j] = __float2bfloat16(f[j]);
  }
}

// Groups of four warps, one per quarter of the lanes, that take an accumulator's chunks of tokens in turn. A lane has a weight row.
// A warp writes 32 neighbours of a token at a time; or (STAGED, with a residual) a chunk goes through shared memory to be read and written
// in vectors of eight: which pays for products of two 4-bit matrices with a residual (100 x 16384 x 512 7.6 us, 8.2 without; 8192 x 4096 x
// 12288 234 and 241; 4718 x 6656 x 8544 204 and 205), and costs without one (4096 x 12288 x 1024 55.1 us, 50.6 without; 4096 x 4096 x 4096
// 41.6 and 39.6; 8111 x 12288 x 4096 216 and 213), with bf16 rows (8192 x 24576 x 4096 1 %; 24008 experts' rows in fp32 7 %) and where rows
// start on no 16 bytes (3484 x 28286 x 768 305 us, 86 without). A chunk's residual is asked for as a whole: one value after the other,
// 4718 x 6656 x 8544 with bf16 rows takes 863 us, 465 so. Gate and up rows are 64 lanes apart: their warps
// hand each other half of a chunk's tokens. SPLIT: results stay in shared memory as [token][weight row], for add_ranges. `parts`: room
// for a tile's results (SPLIT), `staging`: kStaging bytes (STAGED, gated).
template <bool SPLIT, bool STAGED>
__device__ __forceinline__ void write_results(const TileArgs& g, const int* first_tile, int i0, int i_step, int items, bool with_bias,
                                              uint32_t tmem, uint32_t dfull0, uint32_t dempty0, float* parts, float* staging, int group,
                                              int groups, int q, int lane, volatile int* abort_flag, int* status) {
  const int r = q * 32 + lane;
  const bool glu = g.epi != PXL_EPI_NONE;
  int db = 0, buf = 0;
  uint32_t d_phase = 0;
  bool ok = true;
  for (int i = i0; i < items; i += i_step) {
    const Item it = item_of(i, g, first_tile);
    const int n = it.n_blk * kTileRows + r;
    const float factor = g.row_scale ? g.row_scale[static_cast<int64_t>(it.expert) * g.n_blocks * kTileRows + n] : 1.f;
    const float add = g.bias && n < g.N && with_bias ? __bfloat162float(g.bias[static_cast<int64_t>(it.expert) * g.N + n]) : 0.f;
    // after a wait that ran out the loop goes on without results: the warps meet at every barrier below
    ok = ok && wait_parked(dfull0 + 8 * db, d_phase, abort_flag, status, PXL_DEV_TIMEOUT_TMEM_FULL);
    tc_fence_after_sync();
    for (int c0 = group * kChunk; c0 < it.rows; c0 += groups * kChunk) {
      bf16x8 res[4];
      if constexpr (STAGED && !SPLIT) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int e = r + 128 * u, t = min(c0 + e / 16, it.rows - 1);
          res[u] = residual8(g, false, it.n_blk, it.row0 + t, e % 16 * 8);
        }
      }
      uint32_t v[32];
      tmem_ld_32x32b_x32(tmem + db * g.d_cols + c0 + (static_cast<uint32_t>(q * 32) << 16), v);
      tmem_ld_wait();
      const int m = min(kChunk, it.rows - c0);
      const int64_t t0 = it.row0 + c0;
      if constexpr (SPLIT) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < m) parts[(c0 + j) * kPitch + r] = __uint_as_float(v[j]) * factor + add;
      } else if (STAGED && g.vec && g.residual) {
        named_bar_sync(1 + group, 128);  // (the last chunk has been read)
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j < m) staging[j * kPitch + r] = __uint_as_float(v[j]) * factor + add;
        named_bar_sync(1 + group, 128);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int e = r + 128 * u, t = e / 16, c = e % 16 * 8;
          if (!ok || t >= m) break;
          float f[16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 x = *reinterpret_cast<const float4*>(staging + t * kPitch + c + h * 4);
            f[4 * h] = x.x, f[4 * h + 1] = x.y, f[4 * h + 2] = x.z, f[4 * h + 3] = x.w;
          }
          finish8(g, f, false, it.n_blk, it.row0 + c0 + t, c, res[u]);
        }
      } else if (STAGED || !glu) {
        if (!ok || n >= g.N) continue;
        // (one kind of loop each: a choice per result, or its address from scratch, doubles the whole kernel's time)
        float y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(v[j]) * factor + add;
        if (g.residual) {
          // (all asked for at once: behind the last token, the last one's again)
          const bf16* from = g.residual + t0 * g.ldr + n;
          bf16 z[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = from[min(j, m - 1) * g.ldr];
#pragma unroll
          for (int j = 0; j < 32; ++j) y[j] += __bfloat162float(z[j]);
        }
        if (g.out_f32) {
          float* dst = static_cast<float*>(g.C) + t0 * g.ldc + n;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (j >= m) break;
            dst[j * g.ldc] = y[j];
          }
        } else {
          bf16* dst = static_cast<bf16*>(g.C) + t0 * g.ldc + n;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (j >= m) break;
            dst[j * g.ldc] = __float2bfloat16(y[j]);
          }
        }
      } else {
        float* const mine = staging + buf * (kChunk * 64) + (r & 63);
        const int col = it.n_blk * 64 + (r & 63);
        auto half = [&](auto up) {  // gate rows give away tokens 16 .. 31 of the chunk, up rows 0 .. 15
          constexpr bool kUp = decltype(up)::value;
          constexpr int kGive = kUp ? 0 : 16, kKeep = kUp ? 16 : 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) mine[(kGive + j) * 64] = __uint_as_float(v[kGive + j]) * factor + add;
          named_bar_sync(1 + group, 128);  // (the buffer's readers of two chunks ago have met at the one before)
          if (!ok) return;
          float y[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float own = __uint_as_float(v[kKeep + j]) * factor + add, other = mine[(kKeep + j) * 64];
            y[j] = kUp ? mx4_gate(other, own, g.epi, g.limit) : mx4_gate(own, other, g.epi, g.limit);
          }
          bf16* dst = static_cast<bf16*>(g.C) + (t0 + kKeep) * g.ldc + col;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (kKeep + j >= m) break;
            dst[j * g.ldc] = __float2bfloat16(y[j]);
          }
        };
        if (q >= 2) half(Bool<true>());
        else half(Bool<false>());
        buf ^= 1;
      }
    }
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(dempty0 + 8 * db);
    if (++db == g.d_bufs) db = 0, d_phase ^= 1;
  }
}

// CTA r of a cluster adds its share of the tile's tokens over the cluster, in K order, and writes it (between two cluster barriers).
__device__ __forceinline__ void add_ranges(const TileArgs& g, int i, uint32_t parts, int tid, int threads, volatile int* abort_flag) {
  const Item it = item_of(i, g, nullptr);
  const int share = ceil_div(it.rows, g.splits), r0 = static_cast<int>(cluster_cta_rank()) * share, r1 = min(r0 + share, it.rows);
  const bool glu = g.epi != PXL_EPI_NONE;
  const int per = glu ? 8 : 16;
  for (int e = tid; e < (r1 - r0) * per; e += threads) {
    const int t = r0 + e / per, c = e % per * 8;
    const bf16x8 res = residual8(g, glu, it.n_blk, it.row0 + t, c);
    float f[16] = {};
    for (int s = 0; s < g.splits; ++s) {
      const uint32_t src = cluster_map_shared(parts + (t * kPitch + c) * 4, s);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (h >= 2 && !glu) break;
        const float4 x = ld_shared_cluster_f32x4(src + (h & 1) * 16 + (h >> 1) * 256);
        f[4 * h] += x.x, f[4 * h + 1] += x.y, f[4 * h + 2] += x.z, f[4 * h + 3] += x.w;
      }
    }
    if (!*abort_flag) finish8(g, f, glu, it.n_blk, it.row0 + t, c, res);
  }
}

}  // namespace pxl

namespace pxl_host {

// Clusters of `size` CTAs that run at a time, counted as if there were room for one CTA per SM, also where tiles of up to 64 rows leave
// room for two. (A GPU processing cluster's SMs that are no multiple of the size stay empty.)
template <typename Kernel>
inline int max_clusters(Kernel kernel, int size, int threads, int smem) {
  static int cached[64][9] = {};
  int& n = cached[current_device_slot()][size];
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size * 64);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = num_sms() / size;
    }
  }
  return n;
}

// Ranges of K blocks for a launch of `items` tiles, none of them empty and all but the last of two blocks at least: the number of rounds
// times a range's blocks and what a round costs besides, in blocks. `slots`: CTAs at a time without clusters.
template <typename Kernel>
inline void split_k(pxl::TileArgs& g, int64_t items, int slots, int besides, Kernel split, int threads) {
  g.splits = 1, g.kb_per = g.k_blocks;
  if (g.offsets || items >= slots) return;
  int64_t least = g.k_blocks + besides;
  for (int s = 2; s <= 8 && g.k_blocks >= 2 * s; ++s) {
    const int per = pxl::ceil_div(g.k_blocks, s), used = pxl::ceil_div(g.k_blocks, per);
    const int n = max_clusters(split, used, threads, 200 * 1024);
    const int64_t cost = (items + n - 1) / n * (per + besides + 2);
    if (cost < least) least = cost, g.splits = used, g.kb_per = per;
  }
}

inline bool on16(const void* p, int64_t row_bytes) { return !((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row_bytes)) & 15); }

constexpr int kTileSmem = 226 * 1024;
template <typename... Kernels>
inline bool allow_smem(bool (&configured)[64], Kernels... kernels) {
  bool& done = configured[current_device_slot()];
  if (!done) done = ((cudaFuncSetAttribute(kernels, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmem) == cudaSuccess) && ...);
  return done;
}

// one / split: the kernel without and with a cluster
template <typename Kernel, typename... Args>
inline int launch_tiles(Kernel one, Kernel split, pxl::TileArgs& g, int items, int slots, int threads, int smem, cudaStream_t stream,
                        Args... args) {
  const bool is_split = g.splits > 1;
  const int64_t grid = is_split ? static_cast<int64_t>(items) * g.splits : items < slots ? items : slots;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (is_split) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(g.splits);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  const bool in_chain = chained();
  g.early = in_chain && !g.offsets;
  if (in_chain) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, is_split ? split : one, args..., g) == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
}

}  // namespace pxl_host
