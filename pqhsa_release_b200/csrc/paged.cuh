// Shared parts of the dense paged-cache kernels (paged_attend.cu, paged_evict.cu): the argument block, which keys of
// a request are visible, and how the key tiles of all requests are shared out over a persistent grid.
#pragma once

#include <atomic>
#include <utility>

#include "common.cuh"

namespace pqhsa {

constexpr int kPagedGroupRows = 32;    // query rows of one KV head that go through the cache together
constexpr int kPagedMaxRows = 64;      // query_len * group at most: two passes of kPagedGroupRows
constexpr int kPagedMaxQuery = 8;
constexpr int kPagedMassCtas = 4;      // CTAs of the weights' kernel on an SM (the attention has one)
constexpr int kPagedMaxCtas = 1024;    // counters in the workspace, one per CTA of a kernel, of which there are fewer than this

struct PagedArgs {
  const void* k_base;
  const void* v_base;
  const int32_t* block_table;  // null: contiguous, request r is page r of block_size rows
  int32_t max_blocks, block_size, num_blocks;
  int64_t stride_block, stride_head, stride_row;
  int32_t B, H, G, T, R;       // requests, KV heads, query heads per KV head, query tokens, R = G * T rows
  int32_t groups;              // passes over a KV head's keys: ceil(R / kPagedGroupRows)
  int32_t cap;                 // row stride of key_pos / mass / scores
  int32_t limit;               // slots a request can have: min(cap, what its block-table row addresses)
  float scale_log2, softcap, cap_log2, cap_in;  // cap_log2 = softcap log2(e), cap_in = 2 log2(e) scale / softcap
  const float* slopes;
  int32_t window, sinks;
  const int32_t* seq_lens;
  const int32_t* first_key;
  const int32_t* query_pos;
  const int32_t* key_pos;
  float* mass;
  const void* q;
  int64_t q_sr, q_st, q_sh;
  void* out;
  int64_t o_sr, o_st, o_sh;
  float* lse;
  int32_t* tickets;            // [kPagedMaxCtas], zero between launches
  float2* part_ml;             // [2 * CTAs][kPagedGroupRows] (max, sum) of a stream's part
  float* part_acc;             // [2 * CTAs][rows of a pass][128]
  float* row_lse2;             // [B * H][R] log2 sum 2^s of every query row
  float* scores;               // [B * H][R][score_stride] scores in log2 units, only with mass
  int64_t score_stride;        // cap, rounded up to whole tiles
  int32_t g_inv;               // 65536 / G + 1: row / G of the few rows there are without a division
  int32_t tile_log2;           // keys per tile of the attention kernel that runs (fixes the shares)

  // token, query head in the group and place of query row `row` (token * G + head) of a KV head
  __host__ __device__ int token_of(int row) const { return row * g_inv >> 16; }
  __host__ __device__ int head_of(int row) const { return row - token_of(row) * G; }
  __host__ __device__ int64_t q_row(int row) const { return token_of(row) * q_st + head_of(row) * q_sh; }
};

int launch_paged_attend(const PagedArgs& a, int dtype, cudaStream_t st);
int launch_paged_mass(const PagedArgs& a, cudaStream_t st);

struct PagedEvict {
  int32_t budget, recent;
  int32_t* new_lens;   // may be the lengths read
  float* new_mass;     // [B, H, cap], may be the mass read
  int32_t* new_pos;    // [B, H, cap], may be the positions read
  int32_t* source;     // [B, H, budget]
  int32_t* scratch;    // [B, H, 2 budget + 8]: moves, then (from 8) the slots to fill and (from 8 + budget) those that fill them
};
int launch_paged_evict(const PagedArgs& a, const PagedEvict& e, int dtype, cudaStream_t st);
int launch_paged_append(const PagedArgs& a, const void* k, const void* v, int32_t* new_lens, int dtype, cudaStream_t st);

#ifdef __CUDACC__

// Lets a kernel have `smem` bytes of dynamic shared memory on the current device (asked of the runtime once a device).
static inline cudaError_t paged_allow_smem(const void* kern, size_t smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Launch with the attributes of the paged kernels; cluster > 0: as clusters of that many CTAs in x.
template <typename... P, typename... A>
static inline cudaError_t paged_launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, A&&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}

// Every kernel here is launched with programmatic stream serialization: it may be placed on the GPU while the one
// before it in the stream ends.  wait_for_grid comes before its first access to global memory: from there on it sees
// all that came before.  (Inputs are read with ordinary loads: the read-only path is for data that does not change
// while a kernel runs, and this one may have begun before they were written.)  next_grid lets the kernel behind be
// placed from now on instead of at this one's end.
__device__ __forceinline__ void wait_for_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_grid() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Element offset of slot t of request r, KV head h; negative when the slot's page is not in the cache (a block-table
// entry outside 0 .. num_blocks - 1: such a key is invisible, nothing of it is read or written).
__device__ __forceinline__ int64_t paged_offset(const PagedArgs& a, int r, int h, int t) {
  int64_t blk = r;
  int row = t;
  if (a.block_table != nullptr) {
    const int b = t / a.block_size;
    row = t - b * a.block_size;
    const int32_t e = a.block_table[(int64_t)r * a.max_blocks + b];
    if (e < 0 || e >= a.num_blocks) return -1;
    blk = e;
  }
  return blk * a.stride_block + (int64_t)h * a.stride_head + (int64_t)row * a.stride_row;
}

// Whether the page of slot t of request r is in the cache.
__device__ __forceinline__ bool paged_there(const PagedArgs& a, int r, int t) {
  return a.block_table == nullptr || (unsigned)a.block_table[(int64_t)r * a.max_blocks + t / a.block_size] < (unsigned)a.num_blocks;
}

// What a request's query tokens can see.  Query token t sits at position p_first + t; a key at position x is visible
// to position p when first <= x <= p and (no window, or p - x < window, or x - first < sinks).  Slots are positions
// unless key_pos says otherwise; then every slot has to be looked at, else only the tiles of [first, first + sinks)
// and of the window.
struct PagedGeom {
  int n, first, p_first, p_last;
  int a0, na, b0, tiles;  // tiles a0 .. a0 + na, then b0 ..; tiles >= 1, so that every row gets its output
};
__device__ __forceinline__ PagedGeom paged_geom(const PagedArgs& a, int r) {
  PagedGeom g;
  g.n = min(max(a.seq_lens[r], 0), a.limit);
  g.first = a.first_key != nullptr ? max(a.first_key[r], 0) : 0;
  g.p_last = a.query_pos != nullptr ? max(a.query_pos[r], -1) : g.n - 1;
  g.p_first = g.p_last - (a.T - 1);
  const int tl = a.tile_log2, up = (1 << tl) - 1;
  const int end = (g.n + up) >> tl;
  g.a0 = g.na = g.b0 = 0;
  if (a.key_pos == nullptr) {
    const int lo = min(g.first, g.n);
    g.b0 = lo >> tl;
    if (a.window > 0) {
      const int w = (int)min(max((long long)lo, (long long)g.p_first - a.window + 1), (long long)g.n);  // first slot of the window
      const int s = min(a.sinks, w - lo);                              // sink slots in front of it
      g.a0 = lo >> tl;
      g.na = s > 0 ? ((lo + s + up) >> tl) - g.a0 : 0;
      g.b0 = max(w >> tl, g.a0 + g.na);
    }
  }
  g.tiles = max(g.na + max(end - g.b0, 0), 1);
  return g;
}
__device__ __forceinline__ int paged_tile(const PagedGeom& g, int j) { return j < g.na ? g.a0 + j : g.b0 + j - g.na; }
__device__ __forceinline__ bool paged_sees(const PagedGeom& g, const PagedArgs& a, int x, int p) {
  return x >= g.first && x <= p && (a.window == 0 || p - x < a.window || x - g.first < a.sinks);
}

// Of a key at position x: whether some query token sees it, and whether all do (if some do).
struct PagedSight {
  bool any, all;
};
__device__ __forceinline__ PagedSight paged_sight(const PagedGeom& g, const PagedArgs& a, bool there, int x) {
  PagedSight s;
  s.any = there && x >= g.first && x <= g.p_last;
  s.all = x <= g.p_first;
  if (a.window > 0) {
    const bool sink = x - g.first < a.sinks;
    s.any = s.any && (g.p_first - x < a.window || sink);
    s.all = s.all && (g.p_last - x < a.window || sink);
  }
  return s;
}

// How the key tiles of all streams - stream (r, h, pass) in that order, `total` tiles (the host refuses shapes that
// could pass 31 bits) - are shared out over the CTAs, whatever the lengths; every warp works it out by itself.
//
// Equal shares: the tiles form one sequence of which each of C CTAs takes a contiguous share, total / C tiles, one more
// for the first total % C of them.  No CTA has more to do than another, but one whose share runs over the end of a
// stream pays for the merge and the start twice.
//
// Aligned shares, with no more streams than CTAs: every stream gets CTAs of its own, in proportion to its tiles and no
// more than give each warp a tile.  Taken where the largest share is at most half as large again as an equal one and
// kPagedSlack tiles more: a second stream costs a CTA about 2 us, the time of some 12 tiles of 8 KB at an SM's part of
// the memory rate, and an SM that has more to read than others can draw more than its part of it.  us, aligned against
// equal, with the largest share over the equal one (8 KV heads): one request of 1K 9.3 / 13.9 (2.3, slack); 16 of 4096
// 48.1 / 50.1 (1.2); a 4-token step of 8 requests in windows of 4096 34.3 / 37.4 (1.5); 9 of 2K-12K 60.0 / 49.5 (1.95).
constexpr int kPagedSlack = 12;
struct PagedShares {
  int total, C, q, rem;
  int c0, parts;    // aligned: first CTA of this CTA's stream, and how many it has; else parts = 0
  int x, x_end;     // tiles of this CTA, counted along the sequence (equal shares) or in its stream (aligned)
  __device__ __forceinline__ int first(int c) const { return c * q + min(c, rem); }
  __device__ __forceinline__ int owner(int x) const {  // equal shares: CTA that has tile x
    const int wide = rem * (q + 1);
    return x < wide ? x / (q + 1) : rem + (x - wide) / q;
  }
};

struct PagedCursor {
  int r, h, pass;   // request, KV head, pass over its keys
  int tile;         // next tile of that stream
  PagedGeom g;
};

// Shares of this launch and the cursor at the first tile of CTA `cta`; false if it has none.  All lanes of a warp call;
// lane l looks after requests l, l + 32, ...; `warps`: tiles a CTA works on at a time.
__device__ __forceinline__ bool paged_locate(const PagedArgs& a, int ctas, int cta, int warps, PagedShares& sh, PagedCursor& c) {
  const int lane = threadIdx.x & 31, per = a.H * a.groups, streams = a.B * per;
  int mine = lane < a.B ? paged_geom(a, lane).tiles : 0;
  int sum = mine;
  for (int r = lane + 32; r < a.B; r += 32) sum += paged_geom(a, r).tiles;
  sh.total = __reduce_add_sync(0xffffffffu, sum) * per;
  sh.C = min(ctas, sh.total);  // CTAs with a share: none of them is empty
  sh.q = sh.total / sh.C;
  sh.rem = sh.total - sh.q * sh.C;
  sh.parts = 0;
  // aligned: CTAs of a stream of that many tiles, one and its share of those left over (rounded down: all together at
  // most `ctas`; the factor covers the rounding of the quotient)
  const float left = (float)(ctas - streams) / (float)sh.total * (1.f - 0x1p-20f);
  auto ctas_of = [&](int tiles) { return min(1 + (int)((float)tiles * left), (tiles + warps - 1) / warps); };
  bool aligned = streams <= ctas;
  if (aligned) {
    int most = mine > 0 ? (mine + ctas_of(mine) - 1) / ctas_of(mine) : 0;
    for (int r = lane + 32; r < a.B; r += 32) {
      const int t = paged_geom(a, r).tiles, n = ctas_of(t);
      most = max(most, (t + n - 1) / n);
    }
    aligned = __reduce_max_sync(0xffffffffu, most) <= sh.q + (sh.q >> 1) + kPagedSlack;
  }
  // each request has `per` streams of `unit` places (CTAs or tiles): find the one of place x
  const int x = aligned ? cta : sh.first(cta);
  if (!aligned && cta >= sh.C) return false;
  int before = 0;
  for (int base = 0;; base += 32) {
    if (base > 0) mine = base + lane < a.B ? paged_geom(a, base + lane).tiles : 0;
    const int unit = mine > 0 ? per * (aligned ? ctas_of(mine) : mine) : 0;
    int incl = unit;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + incl > x);
    if (past != 0u) {
      const int at = __ffs(past) - 1;
      c.r = base + at;
      before += __shfl_sync(0xffffffffu, incl - unit, at);
      break;
    }
    if (base + 32 >= a.B) return false;  // aligned: a CTA that no stream needs
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  c.g = paged_geom(a, c.r);
  const int unit = aligned ? ctas_of(c.g.tiles) : c.g.tiles;
  const int sub = (x - before) / unit, i = x - before - sub * unit;
  c.h = sub / a.groups;
  c.pass = sub - c.h * a.groups;
  if (aligned) {
    sh.c0 = cta - i;
    sh.parts = unit;
    sh.x = c.tile = c.g.tiles * i / unit;  // fits 31 bits: at most 2^21 tiles and 2^10 - 1 CTAs (the host sees to both)
    sh.x_end = c.g.tiles * (i + 1) / unit;
  } else {
    c.tile = i;
    sh.x = x;
    sh.x_end = sh.first(cta + 1);
  }
  return true;
}

__device__ __forceinline__ void paged_next_stream(const PagedArgs& a, PagedCursor& c) {
  c.tile = 0;
  if (++c.pass < a.groups) return;
  c.pass = 0;
  if (++c.h < a.H) return;
  c.h = 0;
  ++c.r;
  if (c.r < a.B) c.g = paged_geom(a, c.r);
}

#endif  // __CUDACC__

}  // namespace pqhsa
