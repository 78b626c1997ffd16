// Products of up to four rows with microscaled 4-bit weights, and a few tokens' routed experts, straight from global memory.
//
// Bound by the bytes of the weights and, with few of them, by latency: no tensor memory, no stages, no barriers on the way. A warp
// takes 16 weight rows and every so many blocks of 128 columns; lane (g, t) = (lane / 4, lane % 4) reads the 32 codes of column
// group t for two of the rows (16 bytes each, four blocks ahead), makes them bf16 and feeds mma.sync, whose K order is free: the
// lane's own 32 columns take the places of its quarter of K, and it reads x there (32 values of row g) in the same order. The
// warps that share rows add their sums in shared memory, and over a cluster where an expert's K is split further.
//
// The two rows of a lane are 8 apart, or a gate row and its up row (64 apart), so that a lane has both.
#include "mx4.cuh"

namespace {
using namespace pxl;

constexpr int kThreads = 256, kAhead = 4;
constexpr int kMaxTop = 64;
constexpr int kMaxX = 96 * 1024;  // bytes of x in a CTA's shared memory
enum Mode { kDense = 0, kExpertsIn = 1, kExpertsOut = 2 };

struct FewArgs {
  const bf16* x;
  const uint8_t* w;
  const float* row_scale;
  void* C;
  const bf16* bias;
  const bf16* residual;  // kExpertsOut: base
  int64_t ldx, ldc, ldr;
  int T, N, K, epi;
  float limit;
  int n_blocks, k_blocks;
  int share;             // warps of a CTA that share rows (a power of two)
  int splits;            // CTAs of a cluster, each with a part of K; 1 for kDense
  // experts: item = a pair of a token and one of its experts (kExpertsIn), or a token (kExpertsOut)
  const int* ids;
  const float* weights;
  int top, experts;
  Mx4Shift shift;
};

struct Codes {
  uint4 lo, hi;
  uint32_t p_lo, p_hi;
};

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int MODE, bool GLU>
__global__ void __launch_bounds__(kThreads, MODE == kDense ? 3 : 2) gemv_mx4_kernel(const FewArgs g) {
  extern __shared__ __align__(16) uint8_t x_smem[];  // [row of x][block][column group][16 bytes, in another order per group]
  __shared__ float4 red[kThreads];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, row = lane >> 2, t4 = lane & 3;
  const int splits = MODE == kDense ? 1 : g.splits;
  const int rank = splits > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int cta = splits > 1 ? blockIdx.x / splits : blockIdx.x;
  const int n_blk = cta / g.share, group = cta % g.share * (8 / g.share) + warp / g.share;  // 16 rows: group of the block
  const int r_lo = GLU ? 8 * group + row : 16 * group + row;
  constexpr int kApart = GLU ? 64 : 8;
  const int r_hi = r_lo + kApart;
  const int item = blockIdx.y;
  const int64_t expert_bytes = static_cast<int64_t>(g.n_blocks) * g.k_blocks * kBlockBytes;

  // ---- experts of the item (kExpertsIn: one)
  __shared__ int s_expert[kMaxTop];
  __shared__ float s_weight[kMaxTop];
  const int slots = MODE == kExpertsOut ? g.top : 1;
  if constexpr (MODE != kDense) {
    pdl_wait();  // (ids come from the kernels before)
    if (threadIdx.x < slots) {
      const int at = MODE == kExpertsOut ? item * g.top + threadIdx.x : item, e = g.ids[at];
      s_expert[threadIdx.x] = e >= 0 && e < g.experts ? e : -1;
      s_weight[threadIdx.x] = MODE == kExpertsOut ? g.weights[at] : 1.f;
    }
    __syncthreads();
  }
  auto expert_of = [&](int slot) { return MODE == kDense ? 0 : s_expert[slot]; };

  // ---- blocks of columns (kExpertsOut: those of a token's experts one behind the other): the CTA's [b0, b1), every share-th a warp's
  const int total = g.k_blocks * slots, per = ceil_div(total, splits);
  const int b0 = rank * per, b1 = min(b0 + per, total), first = b0 + warp % g.share;
  const int count = first < b1 ? (b1 - first + g.share - 1) / g.share : 0;
  const uint8_t* const row_of_blocks = g.w + static_cast<int64_t>(n_blk) * g.k_blocks * kBlockBytes;
  const int code_at = (t4 * kTileRows + r_lo) * 16, power_at = kCodeBytes + r_lo * 4 + t4;
  // the block that is loaded next
  int l_slot = MODE == kExpertsOut ? first / g.k_blocks : 0, l_kb = first - l_slot * g.k_blocks;
  int l_left = count;
  const uint8_t* l_at = nullptr;
  auto seek = [&]() {
    const int e = l_left > 0 ? expert_of(l_slot) : -1;
    l_at = e < 0 ? nullptr : row_of_blocks + e * expert_bytes + static_cast<int64_t>(l_kb) * kBlockBytes;
  };
  seek();
  auto load = [&](Codes& c) {
    if (l_left <= 0) return;
    if (MODE == kDense || l_at != nullptr) {
      c.lo = ld_stream(l_at + code_at);
      c.hi = ld_stream(l_at + code_at + kApart * 16);
      c.p_lo = __ldg(l_at + power_at);
      c.p_hi = __ldg(l_at + power_at + kApart * 4);
      l_at += g.share * kBlockBytes;
    }
    --l_left;
    if constexpr (MODE == kExpertsOut) {
      l_kb += g.share;
      if (l_kb >= g.k_blocks) {
        do l_kb -= g.k_blocks, ++l_slot;
        while (l_kb >= g.k_blocks);
        seek();
      }
    }
  };
  Codes c[kAhead] = {};
#pragma unroll
  for (int s = 0; s < kAhead; ++s) load(c[s]);
  pdl_wait();
  pdl_launch_dependents();

  // ---- the CTA's columns of x, zeros behind the last one
  const int T = MODE == kDense ? g.T : 1, pitch = (b1 - b0) * 256 + 32;
  for (int t = 0; t < T; ++t) {
    for (int i = threadIdx.x; i < (b1 - b0) * 16; i += kThreads) {
      const int b = b0 + (i >> 4), slot = MODE == kExpertsOut ? b / g.k_blocks : 0, kg = i >> 2 & 3, j = i & 3;
      const int k = (b - slot * g.k_blocks) * kTileCols + kg * 32 + j * 8;
      const int xr = MODE == kDense ? t : MODE == kExpertsIn ? item / g.top : item * g.top + slot;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k < g.K && expert_of(slot) >= 0) v = *reinterpret_cast<const uint4*>(g.x + xr * g.ldx + k);
      *reinterpret_cast<uint4*>(x_smem + t * pitch + (i >> 2) * 64 + (j ^ (kg >> 1)) * 16) = v;
    }
  }
  __syncthreads();

  float acc[4] = {}, sum[4] = {};  // of an expert; of a token's experts (kExpertsOut)
  int cur = MODE == kExpertsOut ? first / g.k_blocks : 0, kb = first - cur * g.k_blocks;
  auto fold = [&]() {              // an expert's sums go into the token's
    const int e = expert_of(cur);
    if (e >= 0) {
      const float* s = g.row_scale + (static_cast<int64_t>(e) * g.n_blocks + n_blk) * kTileRows;
      const float f_lo = s_weight[cur] * s[r_lo], f_hi = s_weight[cur] * s[r_hi];
      sum[0] += f_lo * acc[0], sum[1] += f_lo * acc[1], sum[2] += f_hi * acc[2], sum[3] += f_hi * acc[3];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.f;
  };
  uint4 xv[4] = {};  // rows of x that do not exist stay zeros
  const bool has_row = row < T;
  const uint32_t x_swap = (t4 >> 1) * 16;
  uint32_t x_at = smem_u32(x_smem) + row * pitch + t4 * 64 + (first - b0) * 256;
  auto step = [&](const Codes& c) {
    if (has_row) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(xv[j].x), "=r"(xv[j].y), "=r"(xv[j].z), "=r"(xv[j].w)
                     : "r"(x_at + ((j * 16) ^ x_swap)));
    }
    x_at += g.share * 256;
    const uint32_t p_lo = c.p_lo << 7 | c.p_lo << 23, p_hi = c.p_hi << 7 | c.p_hi << 23;
    const uint32_t lo[4] = {c.lo.x, c.lo.y, c.lo.z, c.lo.w}, hi[4] = {c.hi.x, c.hi.y, c.hi.z, c.hi.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[4], h[4];
      mx4_word(lo[j], p_lo, g.shift, a);
      mx4_word(hi[j], p_hi, g.shift, h);
      const uint32_t a0[4] = {a[0], h[0], a[1], h[1]}, a1[4] = {a[2], h[2], a[3], h[3]};
      const uint32_t v0[2] = {xv[j].x, xv[j].y}, v1[2] = {xv[j].z, xv[j].w};
      mma_m16n8k16_bf16(acc, a0, v0);
      mma_m16n8k16_bf16(acc, a1, v1);
    }
  };
  for (int n = 0; n < count; n += kAhead) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      if (n + s < count) {
        if constexpr (MODE == kExpertsOut) {
          if (kb >= g.k_blocks) {
            fold();
            do kb -= g.k_blocks, ++cur;
            while (kb >= g.k_blocks);
          }
          kb += g.share;
        }
        step(c[s]);  // (of an expert that does not exist: what the registers hold, not folded)
        load(c[s]);
      }
    }
  }
  if constexpr (MODE == kExpertsOut) {
    if (count > 0) fold();
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = sum[i];
  }

  // ---- sums of the warps that share rows, then of the cluster's CTAs
  red[threadIdx.x] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (warp % g.share == 0) {
    float4 v = red[threadIdx.x];
    for (int s = 1; s < g.share; ++s) {
      const float4 o = red[threadIdx.x + 32 * s];
      v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    acc[0] = v.x, acc[1] = v.y, acc[2] = v.z, acc[3] = v.w;
    if (splits > 1) red[threadIdx.x] = v;
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync_all();
    if (rank == 0 && warp % g.share == 0) {
      for (int s = 1; s < splits; ++s) {
        const float4 o = ld_shared_cluster_f32x4(cluster_map_shared(smem_u32(&red[threadIdx.x]), s));
        acc[0] += o.x, acc[1] += o.y, acc[2] += o.z, acc[3] += o.w;
      }
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (rank != 0 || warp % g.share != 0) return;

  // ---- rows r_lo (acc[0], acc[1]) and r_hi (acc[2], acc[3]) for rows 2 t4 and 2 t4 + 1 of x
  const int n_lo = n_blk * kTileRows + r_lo, n_hi = n_blk * kTileRows + r_hi;
  bf16* const C = static_cast<bf16*>(g.C);
  if constexpr (MODE == kExpertsOut) {
    if (t4 != 0) return;
    float y[2] = {acc[0], acc[2]};
    for (int s = 0; s < g.top && g.bias; ++s) {
      const int e = expert_of(s);
      if (e < 0) continue;
      const float f = s_weight[s];
      const bf16* b = g.bias + static_cast<int64_t>(e) * g.N;
      if (n_lo < g.N) y[0] += f * __bfloat162float(b[n_lo]);
      if (n_hi < g.N) y[1] += f * __bfloat162float(b[n_hi]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = i ? n_hi : n_lo;
      if (n >= g.N) continue;
      if (g.residual) y[i] += __bfloat162float(g.residual[item * g.ldr + n]);
      C[item * g.ldc + n] = __float2bfloat16(y[i]);
    }
  } else {
    const int e = expert_of(0);
    if (e < 0) return;
    const float* s = g.row_scale + static_cast<int64_t>(e) * g.n_blocks * kTileRows;
    const bf16* bias = g.bias ? g.bias + static_cast<int64_t>(e) * g.N : nullptr;
    const float f_lo = s[n_lo], f_hi = s[n_hi];
    const float b_lo = bias && n_lo < g.N ? __bfloat162float(bias[n_lo]) : 0.f, b_hi = bias && n_hi < g.N ? __bfloat162float(bias[n_hi]) : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 2 * t4 + i;
      if (MODE == kDense ? t >= g.T : t > 0) continue;
      const int64_t out_row = MODE == kDense ? t : item;
      const float lo = acc[i] * f_lo + b_lo, hi = acc[2 + i] * f_hi + b_hi;
      if (GLU) {
        C[out_row * g.ldc + n_blk * 64 + r_lo] = __float2bfloat16(mx4_gate(lo, hi, g.epi, g.limit));
        continue;
      }
      const bf16* res = g.residual ? g.residual + out_row * g.ldr : nullptr;
      if (n_lo < g.N) C[out_row * g.ldc + n_lo] = __float2bfloat16(res ? lo + __bfloat162float(res[n_lo]) : lo);
      if (n_hi < g.N) C[out_row * g.ldc + n_hi] = __float2bfloat16(res ? hi + __bfloat162float(res[n_hi]) : hi);
    }
  }
}

// Warps that share rows and CTAs per cluster (enough for their columns of x to fit) for `groups` groups of 16 rows and `total` blocks
// of columns; 0: more of x than fits.
int few_splits(int groups, int total, int T, int* share) {
  // 20 to 40 warps per SM, of two blocks each at least: 25600 x 5120 25.2, 26.2 and 27.7 us with 2, 4 and 8 that share rows, 12288 x
  // 4096 15.3, 12.8 and 13.5, 6144 x 4096 13.4, 10.6 and 8.8. (Resident at a time are 24 per SM of a dense product and 16 of experts.)
  *share = 1;
  while (*share < 8 && groups * *share * 2 <= pxl_host::num_sms() * 40 && total / (*share * 2) >= 2) *share *= 2;
  int splits = 1;
  while (splits <= 8 && T * (pxl::ceil_div(total, splits) * 256 + 32) > kMaxX) ++splits;
  return splits <= 8 ? splits : 0;
}

template <int MODE, bool GLU>
int launch_few(FewArgs g, int items, cudaStream_t stream) {
  g.n_blocks = pxl::ceil_div(g.N, kTileRows), g.k_blocks = pxl::ceil_div(g.K, kTileCols);
  g.shift = kMx4Shift;
  const int total = g.k_blocks * (MODE == kExpertsOut ? g.top : 1), T = MODE == kDense ? g.T : 1;
  g.splits = few_splits(8 * g.n_blocks * items, total, T, &g.share);
  if (g.splits == 0 || (MODE == kDense && g.splits > 1)) return PXL_ERR_TOO_LARGE;
  static bool configured[64] = {false};
  const int dev = pxl_host::current_device_slot();
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(gemv_mx4_kernel<MODE, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxX) != cudaSuccess)
      return PXL_ERR_CUDA;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(g.n_blocks * g.share * g.splits), items);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = T * (pxl::ceil_div(total, g.splits) * 256 + 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (g.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(g.splits);
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pxl_host::chained()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, gemv_mx4_kernel<MODE, GLU>, g) == cudaSuccess ? PXL_OK : PXL_ERR_CUDA;
}

}  // namespace

namespace pxl_host {

// Up to four rows where two warps at least share rows, else the tensor-memory kernel is as fast (4 rows: 12288 x 4096 15.0 us here
// and 17.2 there, 51200 x 5120 46 and 40; 8 rows of 4096 x 4096 11.0 and 9.9).
bool gemv_mx4_takes(int M, int N, int K) {
  int share;
  const int groups = 8 * pxl::ceil_div(N, kTileRows), total = pxl::ceil_div(K, kTileCols);
  return M <= 4 && groups * 2 <= num_sms() * 40 && few_splits(groups, total, M, &share) == 1;
}

int gemv_mx4(const void* x, int64_t ldx, const void* w, const float* row_scale, void* C, int64_t ldc, const void* bias,
             const void* residual, int64_t ldr, int M, int N, int K, int epi, float limit, cudaStream_t stream) {
  FewArgs g{};
  g.x = static_cast<const bf16*>(x), g.ldx = ldx, g.w = static_cast<const uint8_t*>(w), g.row_scale = row_scale, g.C = C, g.ldc = ldc;
  g.bias = static_cast<const bf16*>(bias), g.residual = static_cast<const bf16*>(residual), g.ldr = ldr;
  g.T = M, g.N = N, g.K = K, g.epi = epi, g.limit = limit;
  return epi == PXL_EPI_NONE ? launch_few<kDense, false>(g, 1, stream) : launch_few<kDense, true>(g, 1, stream);
}

}  // namespace pxl_host

// The rows between the two products, h, are bf16: they are the second product's operand on the tensor cores, as the bf16 experts' are. One
// rounding of each, which leaves the results within 0.0024 of their size where the sums in fp32 alone leave 0.0017 (half a step of bf16).
// Up to sixteen pairs whose experts' matrices (read for every pair) are 64 MB together, and whose columns of x fit shared memory. Device
// time here and by way of sorted rows and grouped products: one token through 4 of 32 experts of 2880 x 2880 37 and 45 us, two tokens
// (105 MB) 74 and 55; two tokens through 4 of 128 of 2048 x 768 18 and 31, eight through one of 2880 x 2880 (105 MB) 60 and 53.
PXL_EXPORT int pxl_moe_mx4_few_takes(int T, int top, int K, int I) {
  if (T <= 0 || top <= 0 || top > kMaxTop || K <= 0 || I <= 0) return 0;
  const int64_t pairs = T * static_cast<int64_t>(top);
  if (pairs > 16 || pairs * 3 * I * K / 2 > (64 << 20)) return 0;
  int share;
  const int k_in = pxl::ceil_div(K, kTileCols), k_out = pxl::ceil_div(I, kTileCols) * top;
  return few_splits(8 * pxl::ceil_div(2 * I, kTileRows) * T * top, k_in, 1, &share) > 0 &&
         few_splits(8 * pxl::ceil_div(K, kTileRows) * T, k_out, 1, &share) > 0;
}

PXL_EXPORT int pxl_moe_mx4_few(const void* x, int64_t ldx, const int* ids, const float* weights, const void* w1, const float* row_scale1,
                               const void* b1, const void* w2, const float* row_scale2, const void* b2, const void* base, void* h,
                               void* out, int T, int top, int E, int K, int I, int epi, float limit, cudaStream_t stream) {
  if (T <= 0 || top <= 0 || top > kMaxTop || E <= 0 || K <= 0 || K % 32 || I <= 0 || I % 64 || T * static_cast<int64_t>(top) > 65535) return PXL_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(h) | static_cast<uintptr_t>(ldx * 2)) & 15) return PXL_ERR_INVALID_ARG;
  if (epi != PXL_EPI_SILU_MUL && epi != PXL_EPI_CLIP_GLU) return PXL_ERR_INVALID_ARG;
  FewArgs g{};
  g.ids = ids, g.weights = weights, g.top = top, g.experts = E;
  g.x = static_cast<const bf16*>(x), g.ldx = ldx, g.w = static_cast<const uint8_t*>(w1), g.row_scale = row_scale1;
  g.bias = static_cast<const bf16*>(b1), g.C = h, g.ldc = I, g.N = 2 * I, g.K = K, g.epi = epi, g.limit = limit;
  const int r = launch_few<kExpertsIn, true>(g, T * top, stream);
  if (r != PXL_OK) return r;
  g.x = static_cast<const bf16*>(h), g.ldx = I, g.w = static_cast<const uint8_t*>(w2), g.row_scale = row_scale2;
  g.bias = static_cast<const bf16*>(b2), g.residual = static_cast<const bf16*>(base), g.ldr = K, g.C = out, g.ldc = K, g.N = K, g.K = I;
  g.epi = PXL_EPI_NONE;
  return launch_few<kExpertsOut, false>(g, T, stream);
}
