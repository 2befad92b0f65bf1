// Eviction from a paged cache by accumulated attention weight, and the append of a step's rows.
//
// Eviction keeps, per (request, KV head), the `budget` slots of the largest key
//   key_i = +inf   if the slot holds one of the first `sinks` positions or of the last `recent` ones
//           mass_i otherwise (NaN counts as -inf), ties going to the lower slot
// and packs them into slots 0 .. budget - 1 by moving as little as can be: a kept slot below the budget stays where it
// is, and the i-th slot below it that is not kept (ascending) takes over the i-th kept slot behind it.  All sources
// lie behind the budget and all targets below it, so the moves need no order among themselves; a key's position moves
// with it (key_pos), which is what the attention goes by.
//
// A slot whose page is not in the cache holds nothing that could be moved, and nothing can be moved to it: below the
// budget it ranks before all keys (it stays what it is, and the budget has a slot less for others), behind it after all.
// At least `budget` slots rank before the latter (those below the budget alone are as many), so none of them is kept.
//
// Two launches.  The selection is one thread block cluster per stream: the CTAs keep the keys of their share of the
// slots in shared memory (read once), find the budget-th largest in three passes of 11, 11 and 10 bits over a histogram
// that is summed through distributed shared memory, then number the holes and the kept slots behind the budget in slot order
// and write both lists.  The moves go over the whole GPU, four to a warp, all their loads in flight before the stores:
// they are the bytes of the operator (4 rows a move against 8 bytes a slot for the selection).  One B200, 32 streams from
// 131072 slots down to 16384: selection 29 us (34 MB read; three passes with a cluster barrier each), moves 90 us
// (470 MB, 5.2 TB/s with rows of 256 bytes in random order; eight to a warp and four CTAs to an SM 4 us more).
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace pqhsa {

constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvShare = 49152;   // most keys a CTA keeps in shared memory (192 KB)
constexpr int kEvAhead = 4;
constexpr int kEvMoves = 4;       // moves of a warp at a time
template <typename E> constexpr int kEvMoveCtas = sizeof(E) == 2 ? 5 : 4;  // CTAs of them on an SM: as many as hold their rows in registers

// Order-preserving key, +0 and -0 alike, NaN as -inf (the other operand of fmaxf).  Positions outside sinks ..
// sinks + free - 1 are kept before all others: one unsigned comparison, true for all with free = 0.
__device__ __forceinline__ uint32_t evict_key(int sinks, unsigned free, float mass, int pos) {
  const int u = __float_as_int(fmaxf(mass, kNegInf) + 0.f);
  const uint32_t k = (uint32_t)(u ^ ((u >> 31) | (int)0x80000000));  // float_key without a branch
  return (unsigned)pos - (unsigned)sinks >= free ? 0xff800000u : k;  // the key of +inf
}

constexpr uint32_t kEvStays = 0xff800001u, kEvGone = 1u;  // keys of slots on missing pages: above that of +inf, below that of -inf

constexpr int kEvBins = 2048;
struct EvictShared {
  uint32_t hist[2][kEvBins];
  uint32_t prefix;
  int remaining;
  int wtot[32];
  int4 warp[kEvWarps], cta;        // slots above T and at T, below the budget and behind it: (gt, eq, gt, eq)
};

// Lane j holds the counts of the j-th of some consecutive ranges of slots [lo, hi) (j < parts), `ties` slots at T lie
// before them and `take` of all those at T stay, lowest slots first: sums of (slots at T, holes, kept slots behind the
// budget) over the ranges, on every lane.
__device__ __forceinline__ int3 evict_sums(int4 c, bool part, int lo, int hi, int ties, int take, int K) {
  if (!part) c = make_int4(0, 0, 0, 0);
  int incl = c.y + c.w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if ((threadIdx.x & 31) >= o) incl += v;
  }
  const int before = ties + incl - (c.y + c.w);
  const int taken = min(max(take - before, 0), c.y + c.w), taken_lo = min(taken, c.y);
  const int holes = part ? min(max(K - lo, 0), hi - lo) - c.x - taken_lo : 0;
  const int lates = c.z + taken - taken_lo;
  return make_int3(__shfl_sync(0xffffffffu, incl, 31), __reduce_add_sync(0xffffffffu, holes), __reduce_add_sync(0xffffffffu, lates));
}

// RESIDENT: the keys stay in shared memory; else (a share of more than kEvShare slots) every sweep makes them again.
template <bool RESIDENT>
__global__ void __launch_bounds__(kEvThreads, 1) evict_select_kernel(const PagedArgs a, const PagedEvict e) {
  extern __shared__ __align__(16) uint32_t keys_s[];
  __shared__ EvictShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x, ranks = gridDim.x;
  auto sync_all = [&]() {  // a cluster barrier of one CTA would cost as much as one of eight
    if (ranks > 1) cluster.sync();
    else __syncthreads();
  };
  const int64_t stream = blockIdx.y;
  const int r = blockIdx.y / a.H;
  wait_for_grid();
  const int n = min(max(a.seq_lens[r], 0), a.limit), K = e.budget;
  const float* mass = a.mass + stream * a.cap;
  const int32_t* pos = a.key_pos + stream * a.cap;
  float* new_mass = e.new_mass + stream * a.cap;
  int32_t* new_pos = e.new_pos + stream * a.cap;
  int32_t* source = e.source + stream * K;
  int32_t* count = e.scratch + stream * (2 * (int64_t)K + 8);
  int32_t* holes = count + 8;
  int32_t* lates = holes + K;
  const bool apart = e.new_mass != a.mass, apart_pos = e.new_pos != a.key_pos;
  if (n <= K) {  // everything stays (the same for all CTAs of the cluster)
    for (int i = rank * kEvThreads + tid; i < K; i += ranks * kEvThreads) {
      source[i] = i < n ? i : -1;
      if (i < n && apart) new_mass[i] = mass[i];
      if (i < n && apart_pos) new_pos[i] = pos[i];
    }
    if (rank == 0 && tid == 0) *count = 0;
    return;
  }
  // positions that are neither sinks nor above query_pos - recent
  const unsigned open = (unsigned)max((long long)a.query_pos[r] - e.recent - a.sinks + 1, 0LL);
  const int share = ((n + ranks - 1) / ranks + 127) / 128 * 128;
  const int lo = min(rank * share, n), hi = min(lo + share, n);
  // Keys of slots i .. i + 3 (i a multiple of 4 from lo on); 0, which no slot has, past the share.  Sweeps ask for
  // kEvAhead of them at a time: their latency is what a sweep costs.
  const bool wide = ((a.cap & 3) | (((uintptr_t)a.mass | (uintptr_t)a.key_pos) & 15)) == 0;
  auto fetch = [&](int i, float4& m, int4& p) {
    m = make_float4(0.f, 0.f, 0.f, 0.f);
    p = make_int4(0, 0, 0, 0);
    if (wide && i + 4 <= hi) {
      m = *reinterpret_cast<const float4*>(mass + i);
      p = *reinterpret_cast<const int4*>(pos + i);
    } else {
      if (i < hi) m.x = mass[i], p.x = pos[i];
      if (i + 1 < hi) m.y = mass[i + 1], p.y = pos[i + 1];
      if (i + 2 < hi) m.z = mass[i + 2], p.z = pos[i + 2];
      if (i + 3 < hi) m.w = mass[i + 3], p.w = pos[i + 3];
    }
  };
  auto make = [&](int i, const float4& m, const int4& p) {
    return make_uint4(i < hi ? evict_key(a.sinks, open, m.x, p.x) : 0u, i + 1 < hi ? evict_key(a.sinks, open, m.y, p.y) : 0u,
                      i + 2 < hi ? evict_key(a.sinks, open, m.z, p.z) : 0u, i + 3 < hi ? evict_key(a.sinks, open, m.w, p.w) : 0u);
  };
  // What slots below the budget hold if they stay; the moves write over the others.
  const bool wide_source = ((K & 3) | ((uintptr_t)e.source & 15)) == 0;
  const bool wide_new = wide && (((uintptr_t)e.new_mass | (uintptr_t)e.new_pos) & 15) == 0;
  auto stay = [&](int i, const float4& m, const int4& p) {
    const int to = min(hi, K);
    if (i >= to) return;
    if (i + 4 <= to && wide_source) {
      *reinterpret_cast<int4*>(source + i) = make_int4(i, i + 1, i + 2, i + 3);
    } else {
      for (int q = i; q < min(i + 4, to); ++q) source[q] = q;
    }
    if (i + 4 <= to && wide_new) {
      if (apart) *reinterpret_cast<float4*>(new_mass + i) = m;
      if (apart_pos) *reinterpret_cast<int4*>(new_pos + i) = p;
    } else {
      for (int q = i; q < min(i + 4, to); ++q) {
        if (apart) new_mass[q] = mass[q];
        if (apart_pos) new_pos[q] = pos[q];
      }
    }
  };
  // Pages of the share that are not in the cache: rare, so slots are asked for theirs one by one only where there is one.
  bool gap = false;
  if (a.block_table != nullptr && lo < hi)
    for (int b = lo / a.block_size + tid; b <= (hi - 1) / a.block_size; b += kEvThreads)
      gap |= (unsigned)a.block_table[(int64_t)r * a.max_blocks + b] >= (unsigned)a.num_blocks;
  for (int i = tid; i < 2 * kEvBins; i += kEvThreads) sh.hist[i / kEvBins][i % kEvBins] = 0u;
  if (tid == 0) {
    sh.prefix = 0u;
    sh.remaining = K;
  }
  const bool gaps = __syncthreads_or(gap) != 0;
  auto placed = [&](int i, uint32_t k) { return i >= hi || paged_there(a, r, i) ? k : i < K ? kEvStays : kEvGone; };
  auto placed4 = [&](int i, const uint4& k) {
    return gaps ? make_uint4(placed(i, k.x), placed(i + 1, k.y), placed(i + 2, k.z), placed(i + 3, k.w)) : k;
  };
  auto key4 = [&](int i) {
    if constexpr (RESIDENT) return i < hi ? *reinterpret_cast<const uint4*>(keys_s + (i - lo)) : make_uint4(0u, 0u, 0u, 0u);
    float4 m;
    int4 p;
    fetch(i, m, p);
    return placed4(i, make(i, m, p));
  };
  auto key1 = [&](int i) {
    if (i >= hi) return 0u;
    if constexpr (RESIDENT) return keys_s[i - lo];
    const uint32_t k = evict_key(a.sinks, open, mass[i], pos[i]);
    return gaps ? placed(i, k) : k;
  };

  // The K-th largest key T, and how many of the slots with that key stay.  Keys that many slots share (no weight, and
  // the protected ones) are counted in registers: atomics of a warp to one address would queue up.
  const uint32_t key_zero = float_key(0.f), key_inf = float_key(-kNegInf);
  uint32_t mask = 0u;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit_mask = pass == 2 ? 1023u : 2047u;
    uint32_t* hist = sh.hist[pass & 1];
    const uint32_t prefix = sh.prefix;
    int zeros = 0, infs = 0;
    auto tally = [&](uint32_t k) {
      if (pass > 0 && (k & mask) != prefix) return;
      zeros += k == key_zero;
      infs += k == key_inf;
      if (k != key_zero && k != key_inf) atomicAdd(&hist[(k >> shift) & digit_mask], 1u);
    };
    constexpr int kStep = 4 * kEvThreads;
    for (int b = lo + 4 * tid; b < hi; b += kStep * kEvAhead) {
      if (pass == 0) {
        float4 m[kEvAhead];
        int4 p[kEvAhead];
#pragma unroll
        for (int u = 0; u < kEvAhead; ++u) fetch(b + kStep * u, m[u], p[u]);
#pragma unroll
        for (int u = 0; u < kEvAhead; ++u) {
          const int i = b + kStep * u;
          if (i >= hi) break;
          const uint4 k = placed4(i, i + 4 <= hi ? make_uint4(evict_key(a.sinks, open, m[u].x, p[u].x), evict_key(a.sinks, open, m[u].y, p[u].y),
                                                              evict_key(a.sinks, open, m[u].z, p[u].z), evict_key(a.sinks, open, m[u].w, p[u].w))
                                                 : make(i, m[u], p[u]));
          if constexpr (RESIDENT) *reinterpret_cast<uint4*>(keys_s + (i - lo)) = k;
          if (i < K) stay(i, m[u], p[u]);
          tally(k.x); tally(k.y); tally(k.z); tally(k.w);  // slots past the end count below all that are there
        }
      } else {
        uint4 k[kEvAhead];
#pragma unroll
        for (int u = 0; u < kEvAhead; ++u) k[u] = key4(b + kStep * u);
#pragma unroll
        for (int u = 0; u < kEvAhead; ++u) {
          if (b + kStep * u >= hi) break;
          if ((k[u].x & mask) != prefix && (k[u].y & mask) != prefix && (k[u].z & mask) != prefix && (k[u].w & mask) != prefix) continue;
          tally(k[u].x); tally(k[u].y); tally(k[u].z); tally(k[u].w);
        }
      }
    }
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    infs = __reduce_add_sync(0xffffffffu, infs);
    if (lane == 0) {
      if (zeros != 0) atomicAdd(&hist[(key_zero >> shift) & digit_mask], (uint32_t)zeros);
      if (infs != 0) atomicAdd(&hist[(key_inf >> shift) & digit_mask], (uint32_t)infs);
    }
    sync_all();
    // thread t owns digits d + 1 and d: the counts from the top are a prefix sum over the threads
    const int d = kEvBins - 2 - 2 * tid;
    uint2 own = make_uint2(0u, 0u);
    if (ranks == 1) {
      own = *reinterpret_cast<const uint2*>(&hist[d]);
    } else {
#pragma unroll 8
      for (int c = 0; c < ranks; ++c) {
        const uint2 x = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&hist[d], c));
        own.x += x.x;
        own.y += x.y;
      }
    }
    *reinterpret_cast<uint2*>(&sh.hist[(pass & 1) ^ 1][d]) = make_uint2(0u, 0u);  // read by all in the pass before
    const int need = sh.remaining;
    int total;
    const int above = block_exscan((int)(own.x + own.y), sh.wtot, &total);  // its barriers order `remaining` too
    if (above < need && need <= above + (int)own.y) {
      sh.prefix = prefix | ((uint32_t)(d + 1) << shift);
      sh.remaining = need - above;
    } else if (above + (int)own.y < need && need <= above + (int)(own.x + own.y)) {
      sh.prefix = prefix | ((uint32_t)d << shift);
      sh.remaining = need - above - (int)own.y;
    }
    mask |= digit_mask << shift;
    __syncthreads();
  }
  const uint32_t T = sh.prefix;
  const int take = sh.remaining;

  // Slots in order: a warp owns a range of the share, four slots a lane at a time.  One sweep counts, and from the counts
  // of the ranges before it a warp knows how many of its ties stay and where its holes and late slots go in the lists.
  const int span = (share / kEvWarps + 127) / 128 * 128;
  auto w_lo = [&](int w) { return min(lo + w * span, hi); };
  const int begin = w_lo(warp), end = w_lo(warp + 1);
  int4 mine = make_int4(0, 0, 0, 0);
#pragma unroll 4
  for (int g = begin; g < end; g += 128) {
    const int i = g + 4 * lane;
    const uint4 k4 = key4(i);  // a range ends with the share or where the next begins: `end` needs no check of its own
    const int gt = (k4.x > T) + (k4.y > T) + (k4.z > T) + (k4.w > T);
    const int eq = (k4.x == T) + (k4.y == T) + (k4.z == T) + (k4.w == T);
    if (g + 128 <= K) {
      mine.x += gt;
      mine.y += eq;
    } else if (g >= K) {
      mine.z += gt;
      mine.w += eq;
    } else {
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool low = i + q < K;
        mine.x += low && k[q] > T;
        mine.y += low && k[q] == T;
        mine.z += !low && k[q] > T;
        mine.w += !low && k[q] == T;
      }
    }
  }
  mine = make_int4(__reduce_add_sync(0xffffffffu, mine.x), __reduce_add_sync(0xffffffffu, mine.y),
                   __reduce_add_sync(0xffffffffu, mine.z), __reduce_add_sync(0xffffffffu, mine.w));
  if (lane == 0) sh.warp[warp] = mine;
  __syncthreads();
  const int4 of_warp = lane < kEvWarps ? sh.warp[lane] : make_int4(0, 0, 0, 0);
  if (warp == 0) {
    const int4 c = make_int4(__reduce_add_sync(0xffffffffu, of_warp.x), __reduce_add_sync(0xffffffffu, of_warp.y),
                             __reduce_add_sync(0xffffffffu, of_warp.z), __reduce_add_sync(0xffffffffu, of_warp.w));
    if (lane == 0) sh.cta = c;
  }
  sync_all();
  int4 of_cta = make_int4(0, 0, 0, 0);
  if (lane < rank) of_cta = *cluster.map_shared_rank(&sh.cta, lane);
  const int3 ctas = evict_sums(of_cta, lane < rank, min(lane * share, n), min(lane * share + share, n), 0, take, K);
  if (ranks > 1) cluster.barrier_arrive();  // this CTA reads no other's shared memory from here on
  const int3 warps = evict_sums(of_warp, lane < warp, w_lo(lane), w_lo(lane + 1), ctas.x, take, K);
  int tied = ctas.x + warps.x, at_hole = ctas.y + warps.y, at_late = ctas.z + warps.z;
  const int ties = mine.y + mine.w;
  const bool some = tied < take && take < tied + ties;  // in one warp of the cluster at most the ties are told apart
  const uint32_t least = tied >= take ? T + 1u : T;     // smallest key that stays (T is below the largest 32-bit number)
  const unsigned below = (1u << lane) - 1u;
  // 32 slots at a time, so that what a warp adds to a list is one run of words
#pragma unroll 4
  for (int g = begin; g < end; g += 32) {
    const int i = g + lane;
    const uint32_t k = key1(i);
    bool keep = k >= least;
    if (some) {
      const unsigned same = __ballot_sync(0xffffffffu, k == T);
      if (k == T) keep = tied + __popc(same & below) < take;
      tied += __popc(same);
    }
    if (g < K) {
      const unsigned hole = __ballot_sync(0xffffffffu, i < min(K, end) && !keep);
      if ((hole >> lane) & 1u) holes[at_hole + __popc(hole & below)] = i;
      at_hole += __popc(hole);
    }
    if (g + 32 > K) {
      const unsigned late = __ballot_sync(0xffffffffu, i >= K && keep);
      if ((late >> lane) & 1u) lates[at_late + __popc(late & below)] = i;
      at_late += __popc(late);
    }
  }
  if (rank == ranks - 1 && tid == kEvThreads - 1) *count = at_late;  // the last range ends with all of them
  if (ranks > 1) cluster.barrier_wait();  // no CTA ends while another may read its shared memory
}

// The moves of an item (kEvMoves of a stream): where lane j moves a row from and to, asked for one item ahead.
template <typename E>
__global__ void __launch_bounds__(256, kEvMoveCtas<E>) evict_move_kernel(const PagedArgs a, const PagedEvict e, int per) {
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5), items = a.B * a.H * per;  // 31 bits: the host bounds requests x heads x slots
  E* kb = static_cast<E*>(const_cast<void*>(a.k_base));
  E* vb = static_cast<E*>(const_cast<void*>(a.v_base));
  constexpr int half = sizeof(E) / 2;  // 16-byte pieces of a row for each of 16 lanes
  int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  wait_for_grid();
  int dst = -1, src = -1;
  auto fetch = [&](int item) {
    dst = -1;
    if (item >= items || lane >= kEvMoves) return;
    const int st = item / per, first = (item - st * per) * kEvMoves;
    const int64_t stream = st;
    const int32_t* count = e.scratch + stream * (2 * (int64_t)e.budget + 8);
    if (first + lane < *count) {
      dst = count[8 + first + lane];
      src = count[8 + e.budget + first + lane];
    }
  };
  fetch(w);
  for (; w < items; w += warps) {
    const int st = w / per, r = st / a.H, h = st - r * a.H;
    const int64_t stream = st;
    int64_t from = 0, to = -1;
    float mass = 0.f;
    int pos = 0;
    const int d0 = dst, s0 = src;
    if (d0 >= 0) {
      from = paged_offset(a, r, h, s0);
      to = paged_offset(a, r, h, d0);
      mass = a.mass[stream * a.cap + s0];
      pos = a.key_pos[stream * a.cap + s0];
      if (from < 0) from = 0, to = -1;  // the selection moves only between pages that are there: bounds, should the table change
    }
    fetch(w + warps);
    const E* base = lane < 16 ? kb : vb;
    uint4 row[kEvMoves][half];
#pragma unroll
    for (int j = 0; j < kEvMoves; ++j) {
      // a row that does not move is read from the cache's first place, so that no load waits behind a branch
      const int64_t f = __shfl_sync(0xffffffffu, from, j);
#pragma unroll
      for (int p = 0; p < half; ++p) row[j][p] = __ldcs(reinterpret_cast<const uint4*>(base + f) + (lane & 15) + 16 * p);
    }
    if (d0 >= 0) {
      e.source[stream * e.budget + d0] = s0;
      e.new_mass[stream * a.cap + d0] = mass;
      e.new_pos[stream * a.cap + d0] = pos;
    }
#pragma unroll
    for (int j = 0; j < kEvMoves; ++j) {
      const int64_t t = __shfl_sync(0xffffffffu, to, j);
      if (t >= 0) {
#pragma unroll
        for (int p = 0; p < half; ++p) *(reinterpret_cast<uint4*>(const_cast<E*>(base) + t) + (lane & 15) + 16 * p) = row[j][p];
      }
    }
  }
  for (long long r = (long long)blockIdx.x * blockDim.x + threadIdx.x; r < a.B; r += (long long)gridDim.x * blockDim.x)
    e.new_lens[r] = min(a.seq_lens[r], min(e.budget, a.limit));
}

int launch_paged_evict(const PagedArgs& a, const PagedEvict& e, int dtype, cudaStream_t st) {
  // CTAs per stream: enough that a share fits shared memory twice over, and with few streams enough to use the GPU.
  // The histograms of a cluster cross its network: on 32 streams of 128K slots 8 CTAs of 512 threads took 47 us where
  // 4 of 1024 took 33, now 29 (2 CTAs of an SM ask for 128 KB a pass); on 8 streams of 4352 slots one CTA takes 13 us, two 15.
  int ranks = 1;
  while (ranks < 8 && (a.limit > ranks * 32768 || (a.limit > ranks * 8192 && a.B * a.H * ranks * 2 <= sm_count()))) ranks *= 2;
  const int share = ((a.limit + ranks - 1) / ranks + 127) / 128 * 128;
  const bool resident = share <= kEvShare;
  const size_t smem = resident ? sizeof(uint32_t) * (size_t)share : 0;
  auto kern = resident ? evict_select_kernel<true> : evict_select_kernel<false>;
  static std::atomic<uint64_t> allowed{0};
  if (resident && paged_allow_smem((const void*)kern, sizeof(uint32_t) * kEvShare, allowed) != cudaSuccess)
    return check_launch("evict_select shared memory");
  if (paged_launch(kern, dim3(ranks, a.B * a.H), kEvThreads, smem, st, ranks, a, e) != cudaSuccess) return check_launch("evict_select");
  const int most = e.budget < a.limit ? (e.budget < a.limit - e.budget ? e.budget : a.limit - e.budget) : 0;
  const int per = (most + kEvMoves - 1) / kEvMoves;
  const long long want = ((long long)a.B * a.H * per + 7) / 8 + 1, cap = (long long)sm_count() * (dtype == PQHSA_F32 ? kEvMoveCtas<float> : kEvMoveCtas<__half>);
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  PQHSA_DISPATCH_E(dtype, {
    if (paged_launch(evict_move_kernel<E>, dim3(grid), 256, 0, st, 0, a, e, per > 0 ? per : 1) != cudaSuccess) return check_launch("evict_move");
  });
  return check_launch("evict_move");
}

// One CTA per request: T rows of every KV head go to slots n .. n + T - 1 with their positions and no weight yet.  A
// negative length marks an idle request; rows that do not fit the request's slots, or whose page is missing, are
// dropped.
template <typename E>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedArgs a, const E* k, const E* v,
                                                           int32_t* new_lens) {
  const int r = blockIdx.x, lane = threadIdx.x & 31;
  wait_for_grid();
  const int n = a.seq_lens[r];
  E* kb = static_cast<E*>(const_cast<void*>(a.k_base));
  E* vb = static_cast<E*>(const_cast<void*>(a.v_base));
  constexpr int pieces = kD * sizeof(E) / 16;
  for (int i = threadIdx.x >> 5; n >= 0 && i < a.T * a.H; i += blockDim.x >> 5) {
    const int t = i / a.H, h = i % a.H;
    if (n >= a.limit - t) break;
    const int slot = n + t;
    const int64_t stream = (int64_t)r * a.H + h, off = paged_offset(a, r, h, slot);
    if (lane == 0 && a.key_pos != nullptr)
      const_cast<int32_t*>(a.key_pos)[stream * a.cap + slot] = a.query_pos != nullptr ? a.query_pos[r] - (a.T - 1) + t : slot;
    if (lane == 0 && a.mass != nullptr) a.mass[stream * a.cap + slot] = 0.f;
    if (off < 0) continue;
    const int64_t src = (int64_t)r * a.q_sr + (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
    for (int p = lane; p < 2 * pieces; p += 32) {
      const int x = (p % pieces) * (16 / (int)sizeof(E));
      *reinterpret_cast<uint4*>((p < pieces ? kb : vb) + off + x) = *reinterpret_cast<const uint4*>((p < pieces ? k : v) + src + x);
    }
  }
  __syncthreads();  // new_lens may be the lengths read
  if (threadIdx.x == 0) new_lens[r] = n < 0 ? n : (int)min((long long)n + a.T, (long long)max(a.limit, n));
}

int launch_paged_append(const PagedArgs& a, const void* k, const void* v, int32_t* new_lens, int dtype, cudaStream_t st) {
  PQHSA_DISPATCH_E(dtype, {
    if (paged_launch(paged_append_kernel<E>, dim3(a.B), 256, 0, st, 0, a, static_cast<const E*>(k), static_cast<const E*>(v), new_lens) != cudaSuccess)
      return check_launch("paged_append");
  });
  return check_launch("paged_append");
}

}  // namespace pqhsa
