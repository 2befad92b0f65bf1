// Attention of a request's newest tokens over its whole paged cache, read in place: the dense form of the decode
// step (the reference leaves it to the serving engine's own kernel, pq_hsa_decode_runtime.py:790-822).
//
//   s(t, i) = scale <q_t, k_i>;  s = cap tanh(s / cap);  s -= slope (p_t - x_i)      x_i: position of key i
//   out_t = sum_i e^s v_i / sum_i e^s over the visible keys;  lse_t = ln sum_i e^s
//
// Bound by the bytes of K and V, each read once for the G * T query rows that share a KV head (two passes over the
// keys for more than 32 rows).  One pass with a running maximum and sum per row, in the base-2 domain and in fp32.
//
// Split: the key tiles of all (request, KV head, pass) streams form one sequence; a persistent grid of one CTA per SM
// takes shares of it, equal ones or whole numbers of CTAs to a stream (paged.cuh).  Inside a CTA the tiles of a stream go to the warps in turn, each
// with a ring of tiles in shared memory filled by 16-byte asynchronous copies; the warps' states are merged in shared
// memory where a stream (or the share) ends.  A stream that lies in one share is finished there; of one that several
// CTAs share (at most two of a CTA's streams: its first and its last), each writes (max, sum, acc) as it gets there
// and takes a ticket when all its tiles are done; the CTA whose ticket is the last folds the parts: no second launch,
// no CTA waits for another, and one fence a CTA.
//
// Keys that no row may see are not read at all: their rows in shared memory are filled with zeros, so whatever a page
// holds there (NaN included) stays out.  A key that only some rows of the step see takes part with p = 0 for the
// others, and its value row is multiplied only where p is not 0.
#include <type_traits>

#include "paged.cuh"

namespace pqhsa {

constexpr int kPWarps = 8;
constexpr int kPThreads = kPWarps * 32;
constexpr float kLazy = 8.f;  // a running maximum is raised once a score passes it by 2^8: sums stay far from overflow
constexpr float kFloor = -1.7e38f;  // the maximum before any key: finite, so that a score of -inf is p = 0 and not 2^NaN

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t smem, const void* gmem, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(take ? 16 : 0) : "memory");
}

// cap tanh(x / cap), x = scale dot, in log2 units, of z = 2 log2(e) x / cap.
//
// |x| >= cap / 16: cap - 2 cap / (1 + 2^z), two approximations of 2^-22 on a value of 1: off by 2^-18 of the score at
// most, where the sum behind it is off by more (130 roundings of its terms).  Below, where the difference would cancel
// (all scores, with a cap that is large against them): x (1 - u^2 / 3 + 2 u^4 / 15), u = x / cap, whose next term is
// 17 u^6 / 315 < 2^-28.  Eleven instructions against some twenty-five of tanhf; infinities end at the cap, NaN stays.
__device__ __forceinline__ float capped(const PagedArgs& a, float dot) {
  constexpr float kZ2 = 1.f / (4.f * kLog2e * kLog2e);  // u^2 of z^2
  const float z = dot * a.cap_in, z2 = z * z;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(z)));
  const float x = dot * a.scale_log2, small = fmaf(x * z2, fmaf(z2, kZ2 * kZ2 * 2.f / 15.f, -kZ2 / 3.f), x);
  return z2 < 1.f / (256.f * kZ2) ? small : fmaf(-2.f * a.cap_log2, r, a.cap_log2);
}
// score in log2 units of a dot product; p - x is the distance of the key
__device__ __forceinline__ float paged_score(const PagedArgs& a, float dot, float slope_log2, int distance) {
  float s = a.softcap > 0.f ? capped(a, dot) : dot * a.scale_log2;
  if (a.slopes != nullptr) s = fmaf(-slope_log2, (float)distance, s);
  return s;
}

// An element of a merge buffer [warps][rows][128]: the rows of a warp's accumulator layout in different banks.
__device__ __forceinline__ int merge_at(int entry, int row, int rows, int dim) {
  return (entry * rows + row) * kD + (dim ^ (((row >> 1) & 3) << 3));
}

template <typename E>
__device__ __forceinline__ void paged_store_row(const PagedArgs& a, int r, int h, int pass, int row, int lane, float M, float L, float4 o) {
  const int full = pass * kPagedGroupRows + row;
  const int t = a.token_of(full), hq = h * a.G + full - t * a.G;
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;  // an empty row is zero, a NaN stays one
  E* dst = static_cast<E*>(a.out) + (int64_t)r * a.o_sr + (int64_t)t * a.o_st + (int64_t)hq * a.o_sh + lane * 4;
  const E v[4] = {from_f<E>(o.x * inv), from_f<E>(o.y * inv), from_f<E>(o.z * inv), from_f<E>(o.w * inv)};
  if constexpr (sizeof(E) == 4) {
    *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(v);
  } else {
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
  }
  if (lane == 0) {
    const float l2 = L == 0.f ? kNegInf : M + log2f(L);
    if (a.lse != nullptr) a.lse[((int64_t)r * a.T + t) * (a.H * a.G) + hq] = l2 * 0.69314718055994531f;
    a.row_lse2[((int64_t)r * a.H + h) * a.R + full] = l2;
  }
}

// Running state of a row: o and L are relative to 2^M.  A part that has seen no key has M = kFloor, L = 0, o = 0.
struct RowSum {
  float M = kFloor, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void raise(float m) {
    const float to = fmaxf(M, m), f = ex2(M - to);
    M = to;
    L *= f;
    o.x *= f; o.y *= f; o.z *= f; o.w *= f;
  }
  __device__ __forceinline__ void add(float2 ml, const float4& v) {  // ml.x <= M
    const float f = ex2(ml.x - M);
    L = fmaf(ml.y, f, L);
    o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
  }
};

// Streams this CTA has a part of, to be folded by the CTA that finishes the last of their parts.
struct PagedPending {
  int r, h, pass, c0, parts, last;
};

// Ends a stream in this share (all threads): the states of `entries` warps in ml [entries][ROWS] and acc are merged and
// written as output rows (the share holds the whole stream) or as a part of it.
template <typename E, int ROWS, int WARPS>
__device__ __forceinline__ void paged_finish(const PagedArgs& a, const PagedShares& sh, const PagedCursor& c, int x, int count,
                                             int rows, int entries, const float2* ml, const float* acc, PagedPending* pend) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool starts = c.tile == 0, whole = starts && count == c.g.tiles;
  const size_t part = (size_t)2 * blockIdx.x + (starts ? 1 : 0);
  for (int row = warp; row < rows; row += WARPS) {
    RowSum s;
    for (int w = 0; w < entries; ++w) s.M = fmaxf(s.M, ml[w * ROWS + row].x);
    for (int w = 0; w < entries; ++w)
      s.add(ml[w * ROWS + row], *reinterpret_cast<const float4*>(acc + merge_at(w, row, ROWS, lane * 4)));
    if (whole) {
      paged_store_row<E>(a, c.r, c.h, c.pass, row, lane, s.M, s.L, s.o);
    } else {
      if (lane == 0) a.part_ml[part * kPagedGroupRows + row] = make_float2(s.M, s.L);
      *reinterpret_cast<float4*>(a.part_acc + (part * ROWS + row) * kD + lane * 4) = s.o;
    }
  }
  if (!whole && threadIdx.x == 0) {
    PagedPending& p = pend[starts ? 1 : 0];
    p.r = c.r;
    p.h = c.h;
    p.pass = c.pass;
    p.c0 = sh.parts > 0 ? sh.c0 : sh.owner(x - c.tile);
    p.parts = sh.parts > 0 ? sh.parts : sh.owner(x - c.tile + c.g.tiles - 1) - p.c0 + 1;
  }
}

// Folds every `by`-th part, from part `at` on, of N rows of stream p (a warp; the loads of kAhead parts in flight).
template <int ROWS, int N>
__device__ __forceinline__ void paged_fold_rows(const PagedArgs& a, const PagedPending& p, const int (&row)[N], int at, int by, RowSum (&s)[N]) {
  constexpr int kAhead = 16 / N;
  const int lane = threadIdx.x & 31;
  for (int p0 = at; p0 < p.parts; p0 += kAhead * by) {
    float2 x[N][kAhead];
    float4 v[N][kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int q = p0 + u * by;
      const size_t place = (size_t)2 * (p.c0 + q) + (q == 0 ? 1 : 0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[i][u] = make_float2(kFloor, 0.f);
        v[i][u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (q < p.parts) {
          x[i][u] = __ldcg(&a.part_ml[place * kPagedGroupRows + row[i]]);
          v[i][u] = __ldcg(reinterpret_cast<const float4*>(a.part_acc + (place * ROWS + row[i]) * kD + lane * 4));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float top = x[i][0].x;
#pragma unroll
      for (int u = 1; u < kAhead; ++u) top = fmaxf(top, x[i][u].x);
      s[i].raise(top);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) s[i].add(x[i][u], v[i][u]);
    }
  }
}

// After the last tile of the CTA (all threads): tickets for its parts, and the fold of the streams it ends.
template <typename E, int ROWS, int WARPS>
__device__ __forceinline__ void paged_fold(const PagedArgs& a, PagedPending* pend, float2* ml, float* acc) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  next_grid();
  __syncthreads();  // the parts are written (by all threads) and pend is set
  if (threadIdx.x < 2 && pend[threadIdx.x].parts != 0) {
    PagedPending& p = pend[threadIdx.x];
    __threadfence();
    p.last = atomicAdd(a.tickets + p.c0, 1) == p.parts - 1;
    if (p.last != 0) {
      a.tickets[p.c0] = 0;
      __threadfence();
    }
  }
  __syncthreads();
  // while the parts of a row are few: the rows of both streams shared out over the warps, one row or two at a time
  constexpr int kFew = 16;
  const auto rows_of = [&](int i) { return pend[i].last != 0 ? min(a.R - pend[i].pass * kPagedGroupRows, kPagedGroupRows) : 0; };
  const int rows0 = pend[0].parts <= kFew ? rows_of(0) : 0, rows1 = pend[1].parts <= kFew ? rows_of(1) : 0;
  if (rows0 + rows1 <= WARPS) {
    if (warp < rows0 + rows1) {
      const int i = warp < rows0 ? 0 : 1, row = warp - (i != 0 ? rows0 : 0);
      const PagedPending& p = pend[i];
      RowSum s[1];
      paged_fold_rows<ROWS, 1>(a, p, {row}, 0, 1, s);
      paged_store_row<E>(a, p.r, p.h, p.pass, row, lane, s[0].M, s[0].L, s[0].o);
    }
  } else {
    const int items0 = (rows0 + 1) / 2, items1 = (rows1 + 1) / 2;
    for (int item = warp; item < items0 + items1; item += WARPS) {
      const int i = item < items0 ? 0 : 1, first = (item - (i != 0 ? items0 : 0)) * 2, rows = rows_of(i);
      const PagedPending& p = pend[i];
      const int row[2] = {first, min(first + 1, rows - 1)};
      RowSum s[2];
      paged_fold_rows<ROWS, 2>(a, p, row, 0, 1, s);
      paged_store_row<E>(a, p.r, p.h, p.pass, first, lane, s[0].M, s[0].L, s[0].o);
      if (first + 1 < rows) paged_store_row<E>(a, p.r, p.h, p.pass, first + 1, lane, s[1].M, s[1].L, s[1].o);
    }
  }
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const PagedPending& p = pend[i];
    const int rows = p.parts > kFew ? rows_of(i) : 0;
    // a long stream: several warps to a row (all of them for one row, one for eight), each folds every per-th part
    const int per = rows <= 1 ? WARPS : rows <= 2 ? WARPS / 2 : rows <= 4 ? WARPS / 4 : 1;
    const int at = warp % per;
    for (int base = 0; base < rows; base += WARPS / per) {
      const int row = base + warp / per;
      RowSum one[1];
      RowSum& s = one[0];
      if (row < rows) paged_fold_rows<ROWS, 1>(a, p, {row}, at, per, one);
      if (per > 1) {
        __syncthreads();  // the buffer of the round before has been read
        if (lane == 0) ml[warp] = make_float2(s.M, s.L);
        *reinterpret_cast<float4*>(acc + warp * kD + lane * 4) = s.o;
        __syncthreads();
        if (at != 0) continue;
        for (int w = warp + 1; w < warp + per; ++w) {
          s.raise(ml[w].x);
          s.add(ml[w], *reinterpret_cast<const float4*>(acc + w * kD + lane * 4));
        }
      }
      if (row < rows) paged_store_row<E>(a, p.r, p.h, p.pass, row, lane, s.M, s.L, s.o);
    }
  }
}

// ---- fp32 caches: CUDA cores, tiles of 8 keys ---------------------------------------------------------------
// Scores: lane = (key, quarter of the dimensions); a quarter's lanes look after every fourth row for the softmax.
// Values: lane = 4 dimensions of all rows.  Row of a tile in shared memory: 16-byte pieces, piece j at j ^ (key & 7).
constexpr int kKeys = 8;

__device__ __forceinline__ float4 tile_piece(const float* tile, int key, int elem) {  // elem: a multiple of 4
  return *reinterpret_cast<const float4*>(tile + key * kD + (((elem >> 2) ^ (key & 7)) << 2));
}

__device__ __forceinline__ ulonglong2 tile_pairs(const float* tile, int key, int elem) {
  return *reinterpret_cast<const ulonglong2*>(tile + key * kD + (((elem >> 2) ^ (key & 7)) << 2));
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {  // of two floats each
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <int ROWS, int STAGES, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) paged_attend_kernel(const PagedArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int kStage = 2 * kKeys * kD;  // elements of a stage: 8 key rows, then 8 value rows
  constexpr int OWN = ROWS / 4;
  float* ring = reinterpret_cast<float*>(smem_raw) + (threadIdx.x >> 5) * (STAGES * kStage);
  float* acc_s = reinterpret_cast<float*>(smem_raw);  // merge buffer over the rings, used between streams
  static_assert(ROWS <= 2 * STAGES * kKeys, "the merge buffer fits the rings");
  float* q_s = reinterpret_cast<float*>(smem_raw) + WARPS * STAGES * kStage;         // [ROWS][128]
  float* p_s = q_s + ROWS * kD + (threadIdx.x >> 5) * (ROWS * kKeys);                  // per warp [ROWS][8]
  float2* ml_s = reinterpret_cast<float2*>(q_s + ROWS * kD + WARPS * ROWS * kKeys);  // [warps][ROWS]
  __shared__ int pos_s[WARPS][STAGES][kKeys];
  __shared__ int seen_s[WARPS][STAGES];  // keys some row of the step sees; << 16: keys not all of them see
  __shared__ PagedPending pend_s[2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int key = lane & 7, quarter = lane >> 3;
  const float* kb = static_cast<const float*>(a.k_base);
  const float* vb = static_cast<const float*>(a.v_base);

  if (tid < 2) pend_s[tid].parts = pend_s[tid].last = 0;
  wait_for_grid();
  PagedCursor c;
  PagedShares sh;
  if (!paged_locate(a, gridDim.x, blockIdx.x, WARPS, sh, c)) return;
  int x = sh.x;
  const int x_end = sh.x_end;

  while (true) {
    const int count = min(c.g.tiles - c.tile, x_end - x);  // tiles of this stream in the share
    const int h = c.h, row0 = c.pass * kPagedGroupRows, rows = min(a.R - row0, kPagedGroupRows);
    const int mine = count > warp ? (count - warp + WARPS - 1) / WARPS : 0;
    const int32_t* kpos = a.key_pos != nullptr ? a.key_pos + ((int64_t)c.r * a.H + h) * a.cap : nullptr;
    // fills ring slot `st` with tile number `it` of this warp
    auto load = [&](int it, int st) {
      if (it < mine) {
        const int slot = paged_tile(c.g, c.tile + warp + it * WARPS) * kKeys + key;
        int64_t off = -1;
        int pos = -1;
        if (slot < c.g.n) {
          off = paged_offset(a, c.r, h, slot);
          pos = kpos != nullptr ? max(kpos[slot], -1) : slot;
        }
        const PagedSight v = paged_sight(c.g, a, off >= 0, pos);
        const unsigned seen = __ballot_sync(0xffffffffu, v.any) & 0xffu, mixed = __ballot_sync(0xffffffffu, v.any && !v.all) & 0xffu;
        if (lane < kKeys) pos_s[warp][st][lane] = pos;
        if (lane == 0) seen_s[warp][st] = (int)(seen | mixed << 16);
        float* dst = ring + st * kStage;
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {  // a row is 32 pieces of 16 bytes: one a lane
          const int64_t o = __shfl_sync(0xffffffffu, off, k);
          const bool take = (seen >> k) & 1u;
          const int64_t e = (take ? o : 0) + lane * 4;
          const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + k * kD + ((lane ^ k) << 2));
          cp_async16_zfill(to, kb + e, take);
          cp_async16_zfill(to + kKeys * kD * 4, vb + e, take);
        }
      }
      cp_async_commit();
    };
    __syncthreads();  // the merge buffer and q_s are free again
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) load(st, st);
    for (int i = tid; i < ROWS * (kD / 4); i += WARPS * 32) {
      const int row = i / (kD / 4), d = i % (kD / 4) * 4, full = row0 + row;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows)
        v = *(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + (int64_t)c.r * a.q_sr + (int64_t)h * a.G * a.q_sh + a.q_row(full) + d));
      *reinterpret_cast<float4*>(q_s + row * kD + d) = v;
    }
    float slope[OWN], m[OWN], l[OWN], acc[ROWS][4];
    int p_at[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int full = row0 + 4 * i + quarter;
      const bool live = 4 * i + quarter < rows;
      p_at[i] = live ? c.g.p_first + a.token_of(full) : -1;
      slope[i] = live && a.slopes != nullptr ? kLog2e * a.slopes[h * a.G + a.head_of(full)] : 0.f;
      m[i] = kFloor;
      l[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    __syncthreads();

    for (int it = 0; it < mine; ++it) {
      const int st = it % STAGES;
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      load(it + STAGES - 1, (it + STAGES - 1) % STAGES);
      const float* kt = ring + st * kStage;
      const float* vt = kt + kKeys * kD;
      float s[ROWS];
      uint64_t s2[ROWS];  // sums of even and of odd dimensions: two multiply-adds an instruction
#pragma unroll
      for (int i = 0; i < ROWS; ++i) s2[i] = 0ull;
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // 32 dimensions of a quarter, 4 at a time, each quarter in its own order (banks)
        const int d = quarter * 32 + ((j ^ (2 * quarter)) & 7) * 4;
        const ulonglong2 kv = tile_pairs(kt, key, d);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const ulonglong2 qv = *reinterpret_cast<const ulonglong2*>(q_s + i * kD + d);
          s2[i] = fma_pair(kv.y, qv.y, fma_pair(kv.x, qv.x, s2[i]));
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        s[i] = __uint_as_float((uint32_t)s2[i]) + __uint_as_float((uint32_t)(s2[i] >> 32));
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 8);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 16);
      }
      const int pos = pos_s[warp][st][key];
      const unsigned flags = (unsigned)seen_s[warp][st];
      float own[OWN];
      bool raise = false;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const float dot = quarter == 0 ? s[4 * i] : quarter == 1 ? s[4 * i + 1] : quarter == 2 ? s[4 * i + 2] : s[4 * i + 3];
        own[i] = paged_score(a, dot, slope[i], p_at[i] - pos);
        if (flags != 0xffu && !(((flags >> key) & 1u) != 0u && paged_sees(c.g, a, pos, p_at[i]))) own[i] = kNegInf;
        raise |= own[i] > m[i] + kLazy;
      }
      if (a.scores != nullptr) {
        const int slot = paged_tile(c.g, c.tile + warp + it * WARPS) * kKeys + key;
        float* dst = a.scores + (((int64_t)c.r * a.H + h) * a.R + row0) * a.score_stride + slot;
        if (slot < c.g.n) {
#pragma unroll
          for (int i = 0; i < OWN; ++i)
            if (4 * i + quarter < rows) dst[(int64_t)(4 * i + quarter) * a.score_stride] = own[i];
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          float top = own[i];
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float to = fmaxf(m[i], top);
          const float f = ex2(m[i] - to);
          m[i] = to;
          l[i] *= f;
#pragma unroll
          for (int qd = 0; qd < 4; ++qd) {
            const float g = __shfl_sync(0xffffffffu, f, qd * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[4 * i + qd][j] *= g;
          }
        }
      }
      __syncwarp();  // p_s of the tile before has been read
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const float p = ex2(own[i] - m[i]);
        l[i] += p;
        p_s[(4 * i + quarter) * kKeys + key] = p;
      }
      __syncwarp();
      auto values = [&](auto guard) {  // guard: a key that only some rows see is multiplied only where p is not 0
#pragma unroll
        for (int k4 = 0; k4 < kKeys; k4 += 4) {
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = tile_piece(vt, k4 + k, lane * 4);
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const float4 p = *reinterpret_cast<const float4*>(p_s + i * kKeys + k4);
            const float pk[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (guard.value && pk[k] == 0.f) continue;
              acc[i][0] = fmaf(pk[k], v[k].x, acc[i][0]);
              acc[i][1] = fmaf(pk[k], v[k].y, acc[i][1]);
              acc[i][2] = fmaf(pk[k], v[k].z, acc[i][2]);
              acc[i][3] = fmaf(pk[k], v[k].w, acc[i][3]);
            }
          }
        }
      };
      if ((flags >> 16) != 0u) values(std::true_type{});
      else values(std::false_type{});
      __syncwarp();  // the slot may be filled again
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with its ring: the merge buffer lies over it
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
      if (key == 0) ml_s[warp * ROWS + 4 * i + quarter] = make_float2(m[i], l[i]);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      *reinterpret_cast<float4*>(acc_s + merge_at(warp, i, ROWS, lane * 4)) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    __syncthreads();
    paged_finish<float, ROWS, WARPS>(a, sh, c, x, count, rows, WARPS, ml_s, acc_s, pend_s);
    x += count;
    if (x >= x_end) break;
    paged_next_stream(a, c);
  }
  paged_fold<float, ROWS, WARPS>(a, pend_s, ml_s, acc_s);
}

template <int ROWS, int STAGES, int WARPS>
static int launch_fp32(const PagedArgs& a, cudaStream_t st) {
  constexpr size_t smem = sizeof(float) * (WARPS * STAGES * 2 * kKeys * kD + ROWS * kD + WARPS * ROWS * kKeys) +
                          sizeof(float2) * WARPS * ROWS;
  static_assert(smem <= 225 * 1024, "shared memory of a CTA");
  auto kern = paged_attend_kernel<ROWS, STAGES, WARPS>;
  static std::atomic<uint64_t> allowed{0};
  if (paged_allow_smem((const void*)kern, smem, allowed) != cudaSuccess)
    return check_launch("paged_attend shared memory");
  if (paged_launch(kern, dim3(sm_count()), WARPS * 32, smem, st, 0, a) != cudaSuccess) return check_launch("paged_attend");
  return PQHSA_OK;
}

// ---- tensor-core kernel for 16-bit caches: tiles of 16 keys ----------------------------------------------
// Both products run transposed, so that the many keys (and dimensions) are the 16 rows of an m16n8k16 and the few query
// rows its 8 columns: S^T[16 keys, 8 rows] = K q^T and O^T[16 dims, 8 rows] += V^T P^T.  K rows are the A operand as they
// lie (ldmatrix), V the A operand transposed (ldmatrix.trans); P^T gets from the accumulator layout of S^T into the B
// layout with one 8x8 transpose in registers per 8 keys.  A thread holds the same two query rows of every 8 in S^T and
// in O^T, so maxima, sums and rescaling need no exchange.  p is rounded to the 16-bit type for the product with V (half
// a step; the sum it is divided by adds them unrounded in 32 bits).  Against one row per m16 (P V with 16 rows
// of which 4 or 8 are real) this halves the instructions and the accumulators.  A second product with what the rounding
// took off p brings the error against 64 bits from 2.4e-3 to the output's own 1.7e-3 (bf16), but costs 1-2 % up to 8
// rows, 8 % for 16 and 20-30 % for more, and makes a NaN of an infinite value whose p is rounded to itself: not taken.
//
// fp16 has no numbers between 0 and 2^-24, and few bits below 2^-14: with p = 2^(s - m) at most 2^8, thousands of keys some
// 17 nats below one loud key (a sink) would vanish from the product while the sum counts them.  Its p are therefore
// 2^(s - m) with m = kBelow under the row's maximum when it is raised, and raised again after 2 more: at most 2^15, a
// whole half down to 2^-27 of the row's largest weight, off by at most 2^-38 of it further below.  bf16 has the exponents
// of fp32.
constexpr int kMKeys = 16;
template <typename E> constexpr float kBelow = 0.f;
template <> constexpr float kBelow<__half> = 13.f;
template <typename E> constexpr float kRaise = kLazy;
template <> constexpr float kRaise<__half> = 15.f;

template <typename E> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename E> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The copies run ahead of the products across the ends of streams: a warp's tiles of all its CTA's streams form one
// sequence, which `ahead` walks STAGES - 1 tiles in front of `c`; the merge of a stream's warps has its own buffer, so
// the ring stays full meanwhile.  What a tile's addresses depend on (page table, stored positions) is asked for one tile
// before the tile itself.  SHAPED: scores have a cap or a distance bias.
template <typename E, int NB, int STAGES, bool SHAPED>
__global__ void __launch_bounds__(kPThreads, 1) paged_attend_mma_kernel(const PagedArgs a) {
  constexpr int ROWS = 8 * NB;
  constexpr bool QREG = NB <= 2;  // query rows as B fragments in registers; from shared memory when they would fill them
  constexpr int kStageB = 2 * kMKeys * kD * 2;  // bytes of a stage: 16 key rows, then 16 value rows, 256 bytes each
  constexpr int kHalf = kPWarps / 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  float* acc_s = reinterpret_cast<float*>(smem_raw + (size_t)kPWarps * STAGES * kStageB);  // merge buffer [warps / 2][ROWS][128]
  float2* ml_s = reinterpret_cast<float2*>(acc_s + kHalf * ROWS * kD);                     // [warps][ROWS]
  uint8_t* q_s = reinterpret_cast<uint8_t*>(ml_s + kPWarps * ROWS);                        // [ROWS][128] E, swizzled, only without QREG
  __shared__ int pos_s[kPWarps][STAGES][kMKeys];
  __shared__ int seen_s[kPWarps][STAGES];   // keys some row of the step sees; << 16: keys not all of them see
  __shared__ PagedPending pend_s[2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t4 = lane & 3, l4 = lane >> 2;
  const E* kb = static_cast<const E*>(a.k_base);
  const E* vb = static_cast<const E*>(a.v_base);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem_raw) + warp * (STAGES * kStageB);
  // Lane's addresses inside a tile.  Piece j of row k lies at j ^ (k & 7): an even piece 2 i further on is the address
  // with i << 5 exclusive-ored in, as tiles start on 256-byte boundaries.
  const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, v_row = (lane & 7) + (lane >> 4) * 8;  // K: rows 0-7 | 8-15, then the
  const uint32_t k_lane = ring + k_row * 256 + ((((uint32_t)lane >> 4) ^ (k_row & 7)) << 4);    // upper 8 dims; V: the upper 8
  const uint32_t v_lane = ring + (kMKeys + v_row) * 256 + (((((uint32_t)lane >> 3) & 1) ^ (v_row & 7)) << 4);  // dims, then rows 8-15
  const int g_row = lane >> 3, g_piece = lane & 7;                                              // copies: 4 rows x 128 bytes at a time
  const uint32_t g_lane = ring + g_row * 256 + ((g_piece ^ g_row) << 4);

  if (tid < 2) pend_s[tid].parts = pend_s[tid].last = 0;
  wait_for_grid();
  PagedCursor c;
  PagedShares sh;
  if (!paged_locate(a, gridDim.x, blockIdx.x, kPWarps, sh, c)) return;
  int x = sh.x;
  const int x_end = sh.x_end;

  // the copies' cursor: tile number `at` of the `at_end` of this warp in stream `ahead`
  PagedCursor ahead = c;
  int ahead_x = x;
  auto tiles_of = [&](int count) { return count > warp ? (count - warp + kPWarps - 1) / kPWarps : 0; };
  int at = 0, at_end = tiles_of(min(ahead.g.tiles - ahead.tile, x_end - ahead_x));
  bool more = true;
  // a tile of whole pages or of a contiguous cache lies in one piece: its rows are stride_row apart
  const bool even = a.block_table == nullptr || a.block_size % kMKeys == 0;
  // next tile, and for each lane the page of key (lane & 15), its row there and its position (one no token sees: -1)
  int n_slot0 = 0, n_entry = -1, n_row = 0, n_pos = -1;
  auto fetch = [&]() {
    while (at == at_end) {  // on to the next stream in which this warp has a tile
      ahead_x += min(ahead.g.tiles - ahead.tile, x_end - ahead_x);
      if (ahead_x >= x_end) {
        more = false;
        return;
      }
      paged_next_stream(a, ahead);
      at = 0;
      at_end = tiles_of(min(ahead.g.tiles, x_end - ahead_x));
    }
    n_slot0 = paged_tile(ahead.g, ahead.tile + warp + at * kPWarps) * kMKeys;
    ++at;
    const int slot = n_slot0 + (lane & (kMKeys - 1));
    n_entry = ahead.r;
    n_row = slot;
    n_pos = slot;
    const bool there = slot < ahead.g.n;
    if (!there) n_pos = n_entry = -1;
    if (a.key_pos != nullptr && there) n_pos = a.key_pos[((int64_t)ahead.r * a.H + ahead.h) * a.cap + slot];
    if (a.block_table != nullptr) {
      const int b = (unsigned)slot / (unsigned)a.block_size;
      n_row = slot - b * a.block_size;
      if (there) n_entry = a.block_table[(int64_t)ahead.r * a.max_blocks + b];
    }
  };
  auto load = [&](int st) {  // `ahead` is still in the tile's stream
    if (more) {
      const PagedGeom& g = ahead.g;
      n_pos = max(n_pos, -1);  // not in fetch, which must not wait for what it asks for
      const bool page = n_entry >= 0 && n_entry < a.num_blocks;
      const PagedSight v = paged_sight(g, a, page, n_pos);
      const unsigned seen = __ballot_sync(0xffffffffu, v.any) & 0xffffu, mixed = __ballot_sync(0xffffffffu, v.any && !v.all) << 16;
      if (lane < kMKeys) pos_s[warp][st][lane] = n_pos;
      if (lane == 0) seen_s[warp][st] = (int)(seen | mixed);
      const int64_t off = (page ? n_entry : 0) * a.stride_block + ahead.h * a.stride_head + (int64_t)n_row * a.stride_row;
      const uint32_t to = g_lane + st * kStageB;
      if (even && seen == 0xffffu) {
        const int64_t step = 4 * a.stride_row;
        int64_t o = __shfl_sync(0xffffffffu, off, g_row) + g_piece * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i, o += step) {
          const E* kr = kb + o;
          const E* vr = vb + o;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            cp_async16((to ^ ((i & 1) << 6)) + i * 1024 + j * 128, kr + j * 64);
            cp_async16((to ^ ((i & 1) << 6)) + i * 1024 + j * 128 + kMKeys * 256, vr + j * 64);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t o = __shfl_sync(0xffffffffu, off, 4 * i + g_row) + g_piece * 8;
          const bool take = (seen >> (4 * i + g_row)) & 1u;
          const E* kr = kb + (take ? o : 0);
          const E* vr = vb + (take ? o : 0);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            cp_async16_zfill((to ^ ((i & 1) << 6)) + i * 1024 + j * 128, kr + j * 64, take);
            cp_async16_zfill((to ^ ((i & 1) << 6)) + i * 1024 + j * 128 + kMKeys * 256, vr + j * 64, take);
          }
        }
      }
    }
    cp_async_commit();
  };

  uint32_t qf[QREG ? NB : 1][8][2];
  auto load_q = [&](const PagedCursor& s) {
    const int row0 = s.pass * kPagedGroupRows, rows = min(a.R - row0, kPagedGroupRows);
    const E* base = static_cast<const E*>(a.q) + (int64_t)s.r * a.q_sr + (int64_t)s.h * a.G * a.q_sh;
    if constexpr (QREG) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int row = 8 * nb + l4, full = row0 + row;
        const E* src = base + a.q_row(full) + 2 * t4;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qf[nb][kk][0] = row < rows ? *(reinterpret_cast<const uint32_t*>(src + kk * 16)) : 0u;
          qf[nb][kk][1] = row < rows ? *(reinterpret_cast<const uint32_t*>(src + kk * 16 + 8)) : 0u;
        }
      }
    } else {
      for (int i = tid; i < ROWS * 16; i += kPThreads) {
        const int row = i >> 4, piece = i & 15, full = row0 + row;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows)
          v = *(reinterpret_cast<const uint4*>(base + a.q_row(full)) + piece);
        *reinterpret_cast<uint4*>(q_s + row * 256 + ((piece ^ (row & 7)) << 4)) = v;
      }
      __syncthreads();
    }
  };

  fetch();
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) {
    load(st);
    fetch();
  }
  load_q(c);
  int st = 0;  // ring slot of the next tile

  while (true) {
    const int count = min(c.g.tiles - c.tile, x_end - x);  // tiles of this stream in the share
    const int mine = tiles_of(count);
    const int h = c.h, row0 = c.pass * kPagedGroupRows, rows = min(a.R - row0, kPagedGroupRows);
    float m[NB][2], l[NB][2], slope[NB][2], o[NB][8][4];
    int p_at[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = 8 * nb + 2 * t4 + j, full = row0 + row;
        m[nb][j] = kFloor;
        l[nb][j] = 0.f;
        p_at[nb][j] = row < rows ? c.g.p_first + a.token_of(full) : -1;
        slope[nb][j] = SHAPED && row < rows && a.slopes != nullptr ? kLog2e * a.slopes[h * a.G + a.head_of(full)] : 0.f;
      }
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nb][db][j] = 0.f;
    }

    for (int it = 0; it < mine; ++it) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();  // the tile has landed, and the slot before it may be filled again
      load(st == 0 ? STAGES - 1 : st - 1);
      fetch();
      const uint32_t kt = k_lane + st * kStageB, vt = v_lane + st * kStageB;
      float s[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[nb][j] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; kk += 2) {
        uint32_t a0[4], a1[4];
        ldmatrix4(a0, kt ^ (kk << 5));
        ldmatrix4(a1, kt ^ ((kk + 1) << 5));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if constexpr (QREG) {
            mma16816<E>(s[nb], a0, qf[nb][kk][0], qf[nb][kk][1]);
            mma16816<E>(s[nb], a1, qf[nb][kk + 1][0], qf[nb][kk + 1][1]);
          } else {
            uint32_t b[4];
            const int row = 8 * nb + (lane & 7), piece = 2 * kk + (lane >> 3);
            ldmatrix4(b, (uint32_t)__cvta_generic_to_shared(q_s) + row * 256 + ((piece ^ (row & 7)) << 4));
            mma16816<E>(s[nb], a0, b[0], b[1]);
            mma16816<E>(s[nb], a1, b[2], b[3]);
          }
        }
      }
      // s[nb][0], [1]: key l4, rows 2 t4 and 2 t4 + 1 of block nb; [2], [3]: key l4 + 8.  Rows past the step's are not
      // masked: their query is 0 and nothing of them is written.
      const unsigned flags = (unsigned)seen_s[warp][st];
      const unsigned mixed = flags >> 16;
      if constexpr (SHAPED) {
        const int pos0 = pos_s[warp][st][l4], pos1 = pos_s[warp][st][l4 + 8];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[nb][j] = paged_score(a, s[nb][j], slope[nb][j & 1], p_at[nb][j & 1] - (j < 2 ? pos0 : pos1));
      } else {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[nb][j] *= a.scale_log2;
      }
      if (flags != 0xffffu) {
        const int pos0 = pos_s[warp][st][l4], pos1 = pos_s[warp][st][l4 + 8];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (((flags >> (j < 2 ? l4 : l4 + 8)) & 1u) == 0u || !paged_sees(c.g, a, j < 2 ? pos0 : pos1, p_at[nb][j & 1])) s[nb][j] = kNegInf;
      }
      bool raise = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) raise |= s[nb][j] > m[nb][j & 1] + kRaise<E>;
      if (a.scores != nullptr) {
        const int slot = paged_tile(c.g, c.tile + warp + it * kPWarps) * kMKeys + l4;
        float* dst = a.scores + (((int64_t)c.r * a.H + h) * a.R + row0 + 2 * t4) * a.score_stride + slot;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (8 * nb + 2 * t4 + (j & 1) < rows && slot + (j >> 1) * 8 < c.g.n)
              dst[(int64_t)(8 * nb + (j & 1)) * a.score_stride + (j >> 1) * 8] = s[nb][j];
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = fmaxf(s[nb][j], s[nb][j + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float to = fmaxf(m[nb][j], top - kBelow<E>);
            const float f = ex2(m[nb][j] - to);
            m[nb][j] = to;
            l[nb][j] *= f;
#pragma unroll
            for (int db = 0; db < 8; ++db) {
              o[nb][db][j] *= f;
              o[nb][db][j + 2] *= f;
            }
          }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[nb][j] = ex2(s[nb][j] - m[nb][j & 1]);
          l[nb][j & 1] += s[nb][j];
        }
      if (mixed != 0u) {
        // Keys that only some rows see (at most the last query_len - 1 and as many at the window's edge): a product with
        // p = 0 would let an infinite or NaN value through, so these are added one by one and then taken out.
        uint8_t* vrow = smem_raw + ((size_t)(warp * STAGES + st) * 2 + 1) * (kMKeys * 256);
        unsigned left = mixed;
        while (left != 0u) {
          const int k = __ffs(left) - 1;
          left &= left - 1;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const float pa = __shfl_sync(0xffffffffu, k < 8 ? s[nb][0] : s[nb][2], (k & 7) * 4 + t4);
            const float pb = __shfl_sync(0xffffffffu, k < 8 ? s[nb][1] : s[nb][3], (k & 7) * 4 + t4);
#pragma unroll
            for (int d = 0; d < 16; ++d) {
              const float v = to_f(*reinterpret_cast<const E*>(vrow + k * 256 + ((d ^ (k & 7)) << 4) + l4 * 2));
              float& oa = o[nb][d >> 1][(d & 1) * 2];
              float& ob = o[nb][d >> 1][(d & 1) * 2 + 1];
              oa = pa != 0.f ? fmaf(pa, v, oa) : oa;
              ob = pb != 0.f ? fmaf(pb, v, ob) : ob;
            }
          }
          __syncwarp();
          *reinterpret_cast<uint2*>(vrow + k * 256 + lane * 8) = make_uint2(0u, 0u);
        }
        __syncwarp();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if ((mixed >> l4) & 1u) s[nb][0] = s[nb][1] = 0.f;
          if ((mixed >> (l4 + 8)) & 1u) s[nb][2] = s[nb][3] = 0.f;
        }
      }
      uint32_t pf[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        pf[nb][0] = transpose8x8(pack2<E>(s[nb][0], s[nb][1]));
        pf[nb][1] = transpose8x8(pack2<E>(s[nb][2], s[nb][3]));
      }
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        uint32_t av[4];
        ldmatrix4_trans(av, vt ^ (db << 5));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16816<E>(o[nb][db], av, pf[nb][0], pf[nb][1]);
      }
      st = st + 1 == STAGES ? 0 : st + 1;
    }

    // the stream's end in this share: the upper warps hand their state to the lower ones, these are merged by rows
    PagedCursor following = c;
    const bool done = x + count >= x_end;
    if (!done) {
      paged_next_stream(a, following);
      if constexpr (QREG) load_q(following);  // arrives during the merge
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], d);
    auto put = [&](int entry) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (l4 == 0) ml_s[entry * ROWS + 8 * nb + 2 * t4 + j] = make_float2(m[nb][j], l[nb][j]);
#pragma unroll
        for (int db = 0; db < 8; ++db)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc_s[merge_at(entry, 8 * nb + 2 * t4 + (j & 1), ROWS, db * 16 + l4 + (j >> 1) * 8)] = o[nb][db][j];
      }
    };
    __syncthreads();  // the merge buffer (and q_s) of the stream before has been read
    if (warp >= kHalf) put(warp - kHalf);
    __syncthreads();
    if (warp < kHalf) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float f[2], g[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 other = ml_s[warp * ROWS + 8 * nb + 2 * t4 + j];
          const float to = fmaxf(m[nb][j], other.x);
          f[j] = ex2(m[nb][j] - to);
          g[j] = ex2(other.x - to);
          m[nb][j] = to;
          l[nb][j] = fmaf(l[nb][j], f[j], other.y * g[j]);
        }
#pragma unroll
        for (int db = 0; db < 8; ++db)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[nb][db][j] = fmaf(o[nb][db][j], f[j & 1], g[j & 1] * acc_s[merge_at(warp, 8 * nb + 2 * t4 + (j & 1), ROWS, db * 16 + l4 + (j >> 1) * 8)]);
      }
      __syncwarp();
      put(warp);
    }
    __syncthreads();
    paged_finish<E, ROWS, kPWarps>(a, sh, c, x, count, rows, kHalf, ml_s, acc_s, pend_s);
    if (done) break;
    if constexpr (!QREG) load_q(following);  // q_s was last read before the merge
    x += count;
    c = following;
  }
  cp_async_wait<0>();
  paged_fold<E, ROWS, kPWarps>(a, pend_s, ml_s, acc_s);
}

template <typename E, int NB, int STAGES, bool SHAPED>
static int launch_mma(const PagedArgs& a, cudaStream_t st) {
  constexpr int ROWS = 8 * NB;
  constexpr size_t smem = (size_t)kPWarps * STAGES * 2 * kMKeys * kD * 2 + sizeof(float) * (kPWarps / 2) * ROWS * kD +
                          sizeof(float2) * kPWarps * ROWS + (NB > 2 ? ROWS * 256 : 0);
  static_assert(smem <= 225 * 1024 + 512, "shared memory of a CTA");
  auto kern = paged_attend_mma_kernel<E, NB, STAGES, SHAPED>;
  static std::atomic<uint64_t> allowed{0};
  if (paged_allow_smem((const void*)kern, smem, allowed) != cudaSuccess)
    return check_launch("paged_attend shared memory");
  if (paged_launch(kern, dim3(sm_count()), kPThreads, smem, st, 0, a) != cudaSuccess) return check_launch("paged_attend");
  return PQHSA_OK;
}

// ---- accumulated weights -----------------------------------------------------------------------------
// mass[r, h, i] += sum over the rows of 2^(s - lse): one pass over the scores the attention kernel left (4 bytes per
// row and key, much of it gone to DRAM where the cache rows have passed through L2 since), the same tiles in equal
// shares, four keys to a thread: 8 us at 1M keys of 4 rows, and 7 for writing the scores.  The rows of a key are added in row order by one thread: no atomics, the same bits every run.
constexpr int kMassThreads = 256;
__global__ void __launch_bounds__(kMassThreads) paged_mass_kernel(const PagedArgs a) {
  // a.groups is 1 here: one stream per KV head.  The shares need only what was there before the attention kernel, which
  // let this one be placed after it had waited for it.
  PagedCursor c;
  PagedShares sh;
  if (!paged_locate(a, gridDim.x, blockIdx.x, kMassThreads / 32, sh, c)) return;
  int x = sh.x;
  const int x_end = sh.x_end;
  const int quads = a.tile_log2 - 2;  // log2 of the quads of keys in a tile
  __shared__ float z_s[kPagedMaxRows];
  const bool wide = (a.cap & 3) == 0 && ((uintptr_t)a.mass & 15) == 0;
  wait_for_grid();  // scores and row sums are there
  while (true) {
    const int count = min(c.g.tiles - c.tile, x_end - x);
    const int64_t stream = (int64_t)c.r * a.H + c.h;
    const float* scores = a.scores + stream * a.R * a.score_stride;
    float* mass = a.mass + stream * a.cap;
    __syncthreads();  // z_s of the stream before has been read
    for (int row = threadIdx.x; row < a.R; row += kMassThreads) {
      const float z = __ldcg(a.row_lse2 + stream * a.R + row);
      z_s[row] = z == kNegInf ? -kNegInf : z;  // a row that sees no key adds 2^(-inf - inf) = 0
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count << quads; i += kMassThreads) {
      const int slot = (paged_tile(c.g, c.tile + (i >> quads)) << a.tile_log2) + ((i & ((1 << quads) - 1)) << 2);
      if (slot >= c.g.n) continue;
      const bool four = slot + 4 <= c.g.n;
      float4 old = make_float4(0.f, 0.f, 0.f, 0.f), w = old;
      if (four && wide) {
        old = *reinterpret_cast<const float4*>(mass + slot);
      } else {
        old.x = mass[slot];
        if (slot + 1 < c.g.n) old.y = mass[slot + 1];
        if (slot + 2 < c.g.n) old.z = mass[slot + 2];
        if (four) old.w = mass[slot + 3];
      }
      const float* from = scores + slot;
      // a key that the row does not see has no weight of it, not even of a row whose sum is NaN
      auto weight = [](float s, float z) { return s == kNegInf ? 0.f : ex2(s - z); };
      auto add = [&](const float4& s, float z) {
        w.x += weight(s.x, z);
        w.y += weight(s.y, z);
        w.z += weight(s.z, z);
        w.w += weight(s.w, z);
      };
      int row = 0;
      for (; row + 4 <= a.R; row += 4) {
        float4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j, from += a.score_stride) s[j] = __ldcg(reinterpret_cast<const float4*>(from));
#pragma unroll
        for (int j = 0; j < 4; ++j) add(s[j], z_s[row + j]);
      }
      for (; row < a.R; ++row, from += a.score_stride) add(__ldcg(reinterpret_cast<const float4*>(from)), z_s[row]);
      // keys that no row saw, whose weight is 0, are left as they were
      if (four && wide && w.x != 0.f && w.y != 0.f && w.z != 0.f && w.w != 0.f) {
        *reinterpret_cast<float4*>(mass + slot) = make_float4(old.x + w.x, old.y + w.y, old.z + w.z, old.w + w.w);
      } else {
        if (w.x != 0.f) mass[slot] = old.x + w.x;
        if (w.y != 0.f && slot + 1 < c.g.n) mass[slot + 1] = old.y + w.y;
        if (w.z != 0.f && slot + 2 < c.g.n) mass[slot + 2] = old.z + w.z;
        if (w.w != 0.f && four) mass[slot + 3] = old.w + w.w;
      }
    }
    x += count;
    if (x >= x_end) return;
    paged_next_stream(a, c);
  }
}

int launch_paged_mass(const PagedArgs& a, cudaStream_t st) {
  PagedArgs b = a;
  b.groups = 1;
  if (paged_launch(paged_mass_kernel, dim3(sm_count() * kPagedMassCtas), kMassThreads, 0, st, 0, b) != cudaSuccess) return check_launch("paged_mass");
  return PQHSA_OK;
}

// Accumulators of the 8, 16 or 32 rows nearest above those there are (of more than 32, 32 to a pass).  With 32 rows the merge
// buffer leaves room for a ring of two tiles a warp instead of three, and 10 registers a thread are spilled (29 with a cap or bias).  us over
// 4 x 128K keys of 8 KV heads in bf16, 328 at the copy rate: 8 rows 312, 16 rows 330, 24 rows 370, 32 rows 386 (capped
// 480); 40 to 64 rows, whose two passes both read the keys, 693.
template <typename E, bool SHAPED> static int launch_16bit(const PagedArgs& a, int rows, cudaStream_t st) {
  return rows <= 8 ? launch_mma<E, 1, 3, SHAPED>(a, st) : rows <= 16 ? launch_mma<E, 2, 3, SHAPED>(a, st) : launch_mma<E, 4, 2, SHAPED>(a, st);
}

// fp32: few rows wait for memory, and twelve warps with two tiles each ask for more of it than eight with three; from 16
// rows on the products are what takes the time, and the accumulators leave registers for eight warps.  us over 4 x 32K keys
// (164 at the copy rate), 12 x 2 | 8 x 3 | 8 x 2: 4 rows 161 | 209 | 195, 8 rows 235 | 286 | 285, 16 rows 454 | 443 | 440,
// 32 rows - | 1042 | 1038, 64 rows (two passes) 2058.  One request of 1K: 4 rows 9.1 | 8.6 | 8.4.
int launch_paged_attend(const PagedArgs& a, int dtype, cudaStream_t st) {
  PagedArgs b = a;
  const int rows = a.R < kPagedGroupRows ? a.R : kPagedGroupRows;
  int rc = PQHSA_OK;
  if (dtype == PQHSA_F32) {
    b.tile_log2 = 3;
    rc = rows <= 4 ? launch_fp32<4, 2, 12>(b, st) : rows <= 8 ? launch_fp32<8, 2, 12>(b, st) : rows <= 16 ? launch_fp32<16, 3, 8>(b, st) : launch_fp32<32, 3, 8>(b, st);
  } else {
    b.tile_log2 = 4;
    const bool shaped = a.softcap > 0.f || a.slopes != nullptr;
    if (dtype == PQHSA_BF16)
      rc = shaped ? launch_16bit<__nv_bfloat16, true>(b, rows, st) : launch_16bit<__nv_bfloat16, false>(b, rows, st);
    else
      rc = shaped ? launch_16bit<__half, true>(b, rows, st) : launch_16bit<__half, false>(b, rows, st);
  }
  if (rc != PQHSA_OK || a.mass == nullptr) return rc;
  return launch_paged_mass(b, st);
}

}  // namespace pqhsa
