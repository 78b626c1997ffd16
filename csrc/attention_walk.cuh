// How the decode attention kernels go through paged keys: tiles of 64 of them, the blocks of a tile's pages, and the way of a CTA along
// the tiles of all (sequence, key head) pairs when they are dealt out evenly.
#pragma once

#include "common.cuh"
#include "pxl_api.h"

namespace pxl {

constexpr int kKeyTile = 64;

// Tiles of the keys [0, keep) and [lo, hi), first to last: those of the kept keys that lie before the window's first tile,
// then the window's (keep <= 0: none kept).
struct KeyTiles {
  int front, first, total;
  __device__ KeyTiles(int lo, int hi, int keep) {
    first = lo / kKeyTile;
    const int kept = keep > 0 ? ceil_div(keep, kKeyTile) : 0;
    front = kept < first ? kept : first;
    total = hi > lo ? front + ceil_div(hi, kKeyTile) - first : 0;
  }
  __device__ int operator[](int i) const { return i < front ? i : first + i - front; }
};

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
  return v;
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v;
}

// Producer warp: the blocks of the pages of 32 / (pages per tile) tiles at a time, one per lane, the next ones read while these are
// used. Read tile by tile, the latency of a table read was the time of a tile: 1.2 us (e4m3 0.7) with one CTA per SM, whatever the
// consumers did.
struct TileBlocks {
  const int* bt;
  KeyTiles tiles;
  int t_begin, n_tiles, page_size, shift, hi, max_blocks;  // shift: log2(pages per tile)
  int64_t num_blocks;
  int* status;
  int now = 0, ahead = 0;

  __device__ __forceinline__ int look(int it) const {
    const int lane = threadIdx.x & 31;
    it += lane >> shift;
    if (it >= n_tiles) return 0;
    int bi = (tiles[t_begin + it] << shift) + (lane & ((1 << shift) - 1));
    if (bi * page_size >= hi) bi = (hi - 1) / page_size;  // beyond the context: re-read the last page (masked)
    return bi < max_blocks ? bt[bi] : -1;
  }
  __device__ __forceinline__ void begin() { ahead = look(0); }
  // block of page lane % ppt of tile `it`; called by the whole warp, tile after tile
  __device__ __forceinline__ int operator()(int it) {
    const int per = 32 >> shift, i = it & (per - 1);
    if (i == 0) {
      now = ahead;
      ahead = look(it + per);  // not looked at before it is needed
      if (now < 0 || now >= num_blocks) {
        if (status) atomicCAS(status, 0, PXL_DEV_BAD_BLOCK_DECODE);
        now = 0;
      }
    }
    return __shfl_sync(0xffffffffu, now, (i << shift) + (threadIdx.x & ((1 << shift) - 1)));
  }
};

struct DecodeWork {
  const int* ctx_lens;
  int B, Hkv, window, keep;

  __device__ __forceinline__ KeyTiles tiles(int b, int& lo, int& hi) const {
    hi = __ldg(ctx_lens + b);
    lo = (window > 0 && hi > window) ? hi - window : 0;
    return KeyTiles(lo, hi, keep);
  }
  __device__ __forceinline__ int weight(int b) const {  // a pair without keys has a result too
    int lo, hi;
    const int n = tiles(b, lo, hi).total;
    return n > 0 ? n : 1;
  }
  __device__ __forceinline__ int64_t total() const {  // whole warp
    int sum = 0;
    for (int b = threadIdx.x & 31; b < B; b += 32) sum += weight(b);
    return static_cast<int64_t>(__reduce_add_sync(0xffffffffu, sum)) * Hkv;
  }
  // The pair that tile `pos` of the row belongs to, and which of its tiles it is; whole warp.
  __device__ __forceinline__ void find(int64_t pos, int& b, int& kvh, int& t) const {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;  // of the chunk of 32 sequences
    for (int b0 = 0; b0 < B; b0 += 32) {
      const int w = b0 + lane < B ? weight(b0 + lane) : 0;
      int incl = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + static_cast<int64_t>(incl) * Hkv > pos);
      if (past) {
        const int at = __ffs(past) - 1;
        const int rest = static_cast<int>(pos - before - static_cast<int64_t>(__shfl_sync(0xffffffffu, incl - w, at)) * Hkv);
        const int wa = __shfl_sync(0xffffffffu, w, at);
        b = b0 + at;
        kvh = rest / wa;
        t = rest % wa;
        return;
      }
      before += static_cast<int64_t>(__shfl_sync(0xffffffffu, incl, 31)) * Hkv;
    }
    b = B, kvh = 0, t = 0;
  }
};

// Where the CTAs' shares begin: the first total % ctas of them are one tile longer.
struct DecodeShares {
  int64_t each;
  int longer;
  __device__ __forceinline__ DecodeShares(int64_t total, int ctas) : each(total / ctas), longer(static_cast<int>(total % ctas)) {}
  __device__ __forceinline__ int64_t operator[](int cta) const { return each * cta + min(cta, longer); }
};

// The share of CTA `rank` of the 2^log that have a pair to themselves.
struct PairShare {
  int pair, rank, log;
};

// One CTA's way along the row, a pair (or the part of one that is its share) at a time. Uncut: the pairs that begin in its share, whole.
struct DecodeWalk {
  DecodeWork work;
  int left, b, kvh, t, weight, take, lo, hi;  // tiles left; of the pair, tiles t .. t + take of `weight`
  KeyTiles tiles;
  bool uncut;

  __device__ __forceinline__ DecodeWalk(const DecodeWork& w, int cta, int ctas, bool uncut = false) : work(w), tiles(0, 0, 0), uncut(uncut) {
    const DecodeShares at(work.total(), ctas);
    left = static_cast<int>(at[cta + 1] - at[cta]);
    b = kvh = t = weight = take = lo = hi = 0;
    if (left > 0) {
      work.find(at[cta], b, kvh, t);
      enter();
      if (uncut && t > 0) {
        take = weight - t;
        next();
      }
    }
  }
  __device__ __forceinline__ DecodeWalk(const DecodeWork& w, const PairShare& of)
      : work(w), b(of.pair / w.Hkv), kvh(of.pair % w.Hkv), tiles(0, 0, 0), uncut(false) {
    tiles = work.tiles(b, lo, hi);
    weight = tiles.total > 0 ? tiles.total : 1;
    t = weight * of.rank >> of.log;
    left = take = (weight * (of.rank + 1) >> of.log) - t;
  }
  __device__ __forceinline__ void enter() {
    tiles = work.tiles(b, lo, hi);
    weight = tiles.total > 0 ? tiles.total : 1;
    take = uncut ? weight : min(left, weight - t);
  }
  __device__ __forceinline__ int count() const { return tiles.total > 0 ? take : 0; }
  __device__ __forceinline__ bool whole() const { return take == weight; }
  __device__ __forceinline__ void next() {
    left -= take;
    t += take;
    if (t == weight) {
      t = 0;
      if (++kvh == work.Hkv) kvh = 0, ++b;
    }
    if (left > 0) enter();
  }
};

}  // namespace pxl
