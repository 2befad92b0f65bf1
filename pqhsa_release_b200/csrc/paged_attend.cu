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
// takes equal contiguous shares of it (paged.cuh).  Inside a CTA the tiles of a stream go to the warps in turn, each
// with a ring of tiles in shared memory filled by 16-byte asynchronous copies; the warps' states are merged in shared
// memory where a stream (or the share) ends.  A stream that lies in one share is finished there; of one that several
// CTAs share, each writes (max, sum, acc), and the CTA whose ticket is the last folds them: no second launch, and no
// CTA waits for another.
//
// Keys that no row may see are not read at all: their rows in shared memory are filled with zeros, so whatever a page
// holds there (NaN included) stays out.  A key that only some rows of the step see takes part with p = 0 for the
// others, and its value row is multiplied only where p is not 0.
#include "paged.cuh"

namespace pqhsa {

constexpr int kPWarps = 8;
constexpr int kPThreads = kPWarps * 32;
constexpr float kLazy = 8.f;  // a running maximum is raised once a score passes it by 2^8: sums stay far from overflow

__device__ __forceinline__ void cp_async16_zfill(uint32_t smem, const void* gmem, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(take ? 16 : 0) : "memory");
}

// score in log2 units of a dot product; p - x is the distance of the key
__device__ __forceinline__ float paged_score(const PagedArgs& a, float dot, float slope_log2, int distance) {
  float s = a.softcap > 0.f ? a.cap_log2 * tanhf(dot * a.cap_in) : dot * a.scale_log2;
  if (a.slopes != nullptr) s = fmaf(-slope_log2, (float)distance, s);
  return s;
}

// Ends a stream's part: the warps' (max, sum) in ml and accumulators in acc (rows of kAccStride floats) are merged and
// written as output rows (the CTA had the whole stream) or as a partial.  All threads call; rows = rows of the pass.
constexpr int kAccStride = kD + 4;
template <typename E>
__device__ __forceinline__ void paged_store_row(const PagedArgs& a, const PagedCursor& c, int row, int lane, float M, float L,
                                                float4 o) {
  const int pass = c.sub % a.groups, h = c.sub / a.groups, full = pass * kPagedGroupRows + row;
  const int t = full / a.G, hq = h * a.G + full % a.G;
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;  // an empty row is zero, a NaN stays one
  E* dst = static_cast<E*>(a.out) + (int64_t)c.r * a.o_sr + (int64_t)t * a.o_st + (int64_t)hq * a.o_sh + lane * 4;
  const E v[4] = {from_f<E>(o.x * inv), from_f<E>(o.y * inv), from_f<E>(o.z * inv), from_f<E>(o.w * inv)};
  if constexpr (sizeof(E) == 4) {
    *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(v);
  } else {
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
  }
  if (lane == 0) {
    const float l2 = L == 0.f ? kNegInf : M + log2f(L);
    if (a.lse != nullptr) a.lse[((int64_t)c.r * a.T + t) * (a.H * a.G) + hq] = l2 * 0.69314718055994531f;
    a.row_lse2[((int64_t)c.r * a.H + h) * a.R + full] = l2;
  }
}

template <typename E>
__device__ void paged_finish(const PagedArgs& a, const PagedCursor& c, long long x0, int tile0, int tiles, long long total,
                             int C, int rows, int pass_rows, const float2* ml, const float* acc, int* last_s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool whole = tile0 == 0 && tiles == c.g.tiles;
  const size_t part = (size_t)2 * blockIdx.x + (tile0 == 0 ? 1 : 0);  // at most one part of a CTA starts a stream it does not end
  for (int row = warp; row < rows; row += kPWarps) {
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < kPWarps; ++w) M = fmaxf(M, ml[w * pass_rows + row].x);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kPWarps; ++w) {
      const float2 x = ml[w * pass_rows + row];
      if (x.x == kNegInf && x.y == 0.f) continue;  // this warp saw no key of the row
      const float f = ex2(x.x - M);
      const float4 v = *reinterpret_cast<const float4*>(acc + ((size_t)w * pass_rows + row) * kAccStride + lane * 4);
      L = fmaf(x.y, f, L);
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    if (whole) {
      paged_store_row<E>(a, c, row, lane, M, L, o);
    } else {
      if (lane == 0) a.part_ml[part * kPagedGroupRows + row] = make_float2(M, L);
      *reinterpret_cast<float4*>(a.part_acc + (part * pass_rows + row) * kD + lane * 4) = o;
    }
  }
  if (whole) return;
  // the parts of a stream lie in CTAs c0 .. c1; the one whose ticket is the last folds them
  const int c0 = (int)(((x0 + 1) * C - 1) / total), c1 = (int)(((x0 + c.g.tiles) * C - 1) / total);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int seen = atomicAdd(a.tickets + c0, 1);
    *last_s = seen == c1 - c0;
    if (seen == c1 - c0) a.tickets[c0] = 0;
  }
  __syncthreads();
  if (*last_s == 0) return;
  __threadfence();
  const int parts = c1 - c0 + 1;
  for (int row = warp; row < rows; row += kPWarps) {
    float M = kNegInf;
    for (int s = lane; s < parts; s += 32) M = fmaxf(M, __ldcg(&a.part_ml[((size_t)2 * (c0 + s) + (s == 0)) * kPagedGroupRows + row].x));
    M = warp_max(M);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < parts; ++s) {
      const size_t p = (size_t)2 * (c0 + s) + (s == 0);
      const float2 x = __ldcg(&a.part_ml[p * kPagedGroupRows + row]);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_acc + (p * pass_rows + row) * kD + lane * 4));
      const float f = x.x == kNegInf && x.y == 0.f ? 0.f : ex2(x.x - M);
      L = fmaf(x.y, f, L);
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    paged_store_row<E>(a, c, row, lane, M, L, o);
  }
}

// ---- CUDA-core kernel: tiles of 8 keys -----------------------------------------------------------------
// Scores: lane = (key, quarter of the dimensions); a quarter's lanes share the rows of the step for the softmax.
// Values: lane = 4 dimensions of all rows.  Row of a tile in shared memory: 16-byte pieces, piece j at j ^ (key & 7).
constexpr int kKeys = 8;

template <typename E> __device__ __forceinline__ const E* tile_piece(const E* tile, int key, int elem) {
  constexpr int n = 16 / sizeof(E);  // elements of a piece; elem is a multiple of 4
  const int piece = elem / n;
  return tile + key * kD + ((piece ^ (key & 7)) * n) + elem % n;
}
__device__ __forceinline__ void tile4(const float* p, float (&v)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
template <typename E> __device__ __forceinline__ void tile4(const E* p, float (&v)[4]) {
  unpack4(*reinterpret_cast<const uint2*>(p), static_cast<const E*>(nullptr), v);
}

template <typename E, int ROWS, int STAGES>
__global__ void __launch_bounds__(kPThreads, 1) paged_attend_kernel(const PagedArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr int kStage = 2 * kKeys * kD;  // elements of a stage: 8 key rows, then 8 value rows
  E* ring = reinterpret_cast<E*>(smem_raw) + (threadIdx.x >> 5) * (STAGES * kStage);
  float* acc_s = reinterpret_cast<float*>(smem_raw);  // merge buffer over the rings, used between streams
  constexpr size_t kRing = sizeof(E) * kPWarps * STAGES * kStage;
  constexpr size_t kMerge = sizeof(float) * kPWarps * ROWS * kAccStride;
  uint8_t* tail = smem_raw + (kRing > kMerge ? kRing : kMerge);
  float* q_s = reinterpret_cast<float*>(tail);                                   // [ROWS][128]
  float* p_s = q_s + ROWS * kD + (threadIdx.x >> 5) * (ROWS * kKeys);             // per warp [ROWS][8]
  float2* ml_s = reinterpret_cast<float2*>(q_s + ROWS * kD + kPWarps * ROWS * kKeys);  // [warps][ROWS]
  __shared__ int pos_s[kPWarps][STAGES][kKeys];
  __shared__ int seen_s[kPWarps][STAGES];
  __shared__ int last_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int key = lane & 7, quarter = lane >> 3;
  constexpr int OWN = ROWS / 4;
  const E* kb = static_cast<const E*>(a.k_base);
  const E* vb = static_cast<const E*>(a.v_base);

  const long long total = paged_total(a);
  const int C = (int)min((long long)gridDim.x, total);  // CTAs with a share: none of them is empty
  if (blockIdx.x >= C) return;
  long long x = paged_share(total, blockIdx.x, C);
  const long long x_end = paged_share(total, blockIdx.x + 1, C);
  PagedCursor c = paged_locate(a, x);

  while (true) {
    const int count = (int)min((long long)(c.g.tiles - c.tile), x_end - x);  // tiles of this stream in the share
    const int pass = c.sub % a.groups, h = c.sub / a.groups;
    const int row0 = pass * kPagedGroupRows, rows = min(a.R - row0, kPagedGroupRows);
    __syncthreads();  // the merge buffer and q_s are free again
    for (int i = tid; i < ROWS * (kD / 4); i += kPThreads) {
      const int row = i / (kD / 4), d = i % (kD / 4) * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (row < rows) {
        const int full = row0 + row;
        load4(static_cast<const E*>(a.q) + (int64_t)c.r * a.q_sr + (int64_t)(full / a.G) * a.q_st +
                  (int64_t)(h * a.G + full % a.G) * a.q_sh + d, v);
      }
      *reinterpret_cast<float4*>(q_s + row * kD + d) = make_float4(v[0], v[1], v[2], v[3]);
    }
    float slope[OWN], m[OWN], l[OWN], acc[ROWS][4];
    int p_at[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int full = row0 + 4 * i + quarter;
      const bool live = 4 * i + quarter < rows;
      p_at[i] = live ? c.g.p_first + full / a.G : -1;
      slope[i] = live && a.slopes != nullptr ? kLog2e * __ldg(a.slopes + h * a.G + full % a.G) : 0.f;
      m[i] = kNegInf;
      l[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    __syncthreads();

    const int mine = count > warp ? (count - warp + kPWarps - 1) / kPWarps : 0;
    const int32_t* kpos = a.key_pos != nullptr ? a.key_pos + ((int64_t)c.r * a.H + h) * a.cap : nullptr;
    // fills ring slot `st` with tile number `it` of this warp
    auto load = [&](int it, int st) {
      if (it < mine) {
        const int slot = paged_tile(c.g, c.tile + warp + it * kPWarps) * kKeys + key;
        int64_t off = -1;
        int pos = -1;
        if (slot < c.g.n) {
          off = paged_offset(a, c.r, h, slot);
          pos = kpos != nullptr ? __ldg(kpos + slot) : slot;
        }
        bool any = off >= 0 && pos >= c.g.first && pos <= c.g.p_last;
        if (any && a.window > 0) any = c.g.p_first - pos < a.window || pos - c.g.first < a.sinks;
        const unsigned seen = __ballot_sync(0xffffffffu, any) & 0xffu;
        if (lane < kKeys) pos_s[warp][st][lane] = pos;
        if (lane == 0) seen_s[warp][st] = (int)seen;
        // a row is kD * sizeof(E) / 16 pieces: 32 lanes cover 1 (fp32) or 2 (16-bit) rows at a time
        constexpr int pieces = kD * (int)sizeof(E) / 16, at_once = 32 / pieces;
        E* dst = ring + st * kStage;
#pragma unroll
        for (int r = 0; r < kKeys; r += at_once) {
          const int k = r + lane / pieces, piece = lane % pieces;
          const int64_t o = __shfl_sync(0xffffffffu, off, k);
          const bool take = (seen >> k) & 1u;
          const int64_t e = (take ? o : 0) + piece * (16 / (int)sizeof(E));
          const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + k * kD + (piece ^ (k & 7)) * (16 / (int)sizeof(E)));
          cp_async16_zfill(to, kb + e, take);
          cp_async16_zfill(to + kKeys * kD * sizeof(E), vb + e, take);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) load(st, st);
    for (int it = 0; it < mine; ++it) {
      const int st = it % STAGES;
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      load(it + STAGES - 1, (it + STAGES - 1) % STAGES);
      const E* kt = ring + st * kStage;
      const E* vt = kt + kKeys * kD;
      float s[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) s[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // 32 dimensions of a quarter, 4 at a time, each quarter in its own order (banks)
        const int d = quarter * 32 + ((j ^ (2 * quarter)) & 7) * 4;
        float kv[4];
        tile4(tile_piece(kt, key, d), kv);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const float4 qv = *reinterpret_cast<const float4*>(q_s + i * kD + d);
          s[i] = fmaf(kv[0], qv.x, fmaf(kv[1], qv.y, fmaf(kv[2], qv.z, fmaf(kv[3], qv.w, s[i]))));
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 8);
        s[i] += __shfl_xor_sync(0xffffffffu, s[i], 16);
      }
      const int pos = pos_s[warp][st][key];
      const bool here = (seen_s[warp][st] >> key) & 1;
      float own[OWN];
      bool raise = false;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const float dot = quarter == 0 ? s[4 * i] : quarter == 1 ? s[4 * i + 1] : quarter == 2 ? s[4 * i + 2] : s[4 * i + 3];
        own[i] = here && paged_sees(c.g, a, pos, p_at[i]) ? paged_score(a, dot, slope[i], p_at[i] - pos) : kNegInf;
        raise |= own[i] > m[i] + kLazy;
      }
      if (a.scores != nullptr) {
        const int slot = paged_tile(c.g, c.tile + warp + it * kPWarps) * kKeys + key;
        float* dst = a.scores + (((int64_t)c.r * a.H + h) * a.R + row0) * a.cap + slot;
        if (slot < c.g.n) {
#pragma unroll
          for (int i = 0; i < OWN; ++i)
            if (4 * i + quarter < rows) dst[(int64_t)(4 * i + quarter) * a.cap] = own[i];
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          float top = own[i];
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float to = fmaxf(m[i], top);
          const float f = m[i] == kNegInf ? (to == kNegInf ? 1.f : 0.f) : ex2(m[i] - to);
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
        const float p = own[i] == kNegInf ? 0.f : ex2(own[i] - m[i]);
        l[i] += p;
        p_s[(4 * i + quarter) * kKeys + key] = p;
      }
      __syncwarp();
#pragma unroll
      for (int k4 = 0; k4 < kKeys; k4 += 4) {
        float v[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) tile4(tile_piece(vt, k4 + k, lane * 4), v[k]);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const float4 p = *reinterpret_cast<const float4*>(p_s + i * kKeys + k4);
          const float pk[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = pk[k] != 0.f ? fmaf(pk[k], v[k][j], acc[i][j]) : acc[i][j];
        }
      }
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
      *reinterpret_cast<float4*>(acc_s + ((size_t)warp * ROWS + i) * kAccStride + lane * 4) =
          make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    __syncthreads();
    paged_finish<E>(a, c, x - c.tile, c.tile, count, total, C, rows, ROWS, ml_s, acc_s, &last_s);
    x += count;
    if (x >= x_end) return;
    paged_next_stream(a, c);
  }
}

template <typename E, int ROWS, int STAGES>
static int launch_simple(const PagedArgs& a, cudaStream_t st) {
  constexpr size_t ring = sizeof(E) * kPWarps * STAGES * 2 * kKeys * kD;
  constexpr size_t merge = sizeof(float) * kPWarps * ROWS * kAccStride;
  constexpr size_t smem = (ring > merge ? ring : merge) + sizeof(float) * (ROWS * kD + kPWarps * ROWS * kKeys) +
                          sizeof(float2) * kPWarps * ROWS;
  static_assert(smem <= 220 * 1024, "shared memory of a CTA");
  auto kern = paged_attend_kernel<E, ROWS, STAGES>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return check_launch("paged_attend shared memory");
  kern<<<sm_count(), kPThreads, smem, st>>>(a);
  return check_launch("paged_attend");
}

// ---- accumulated weights -----------------------------------------------------------------------------
// mass[r, h, i] += sum over the rows of 2^(s - lse): one pass over the scores the attention kernel left (4 bytes per
// row and key, which come from L2 while the cache rows went past it), the same shares of the same tiles.  The rows of
// a key are added in row order by one thread: no atomics, the same bits every run.
__global__ void __launch_bounds__(256) paged_mass_kernel(const PagedArgs a) {
  const long long total = paged_total(a);  // a.groups is 1 here: one stream per KV head
  long long x = paged_share(total, blockIdx.x, gridDim.x);
  const long long x_end = paged_share(total, blockIdx.x + 1, gridDim.x);
  if (x >= x_end) return;
  PagedCursor c = paged_locate(a, x);
  const int keys = 1 << a.tile_log2;
  while (true) {
    const int count = (int)min((long long)(c.g.tiles - c.tile), x_end - x);
    const int64_t stream = (int64_t)c.r * a.H + c.sub;
    for (int i = threadIdx.x; i < count * keys; i += blockDim.x) {
      const int slot = paged_tile(c.g, c.tile + (i >> a.tile_log2)) * keys + (i & (keys - 1));
      if (slot >= c.g.n) continue;
      float w = 0.f;
      for (int row = 0; row < a.R; ++row) {
        const float s = __ldcg(a.scores + (stream * a.R + row) * a.cap + slot);
        const float z = __ldcg(a.row_lse2 + stream * a.R + row);
        w += s == kNegInf ? 0.f : ex2(s - z);
      }
      if (w != 0.f) a.mass[stream * a.cap + slot] += w;  // keys no row saw are left as they were
    }
    x += count;
    if (x >= x_end) return;
    paged_next_stream(a, c);
  }
}

int launch_paged_mass(const PagedArgs& a, cudaStream_t st) {
  PagedArgs b = a;
  b.groups = 1;
  paged_mass_kernel<<<sm_count() * 8, 256, 0, st>>>(b);
  return check_launch("paged_mass");
}

int launch_paged_attend(const PagedArgs& a, int dtype, cudaStream_t st) {
  PagedArgs b = a;
  b.tile_log2 = 3;
  int rc = PQHSA_OK;
  const int rows = a.R < kPagedGroupRows ? a.R : kPagedGroupRows;
  PQHSA_DISPATCH_E(dtype, {
    rc = rows <= 8 ? launch_simple<E, 8, 2>(b, st) : rows <= 16 ? launch_simple<E, 16, 2>(b, st) : launch_simple<E, 32, 2>(b, st);
  });
  if (rc != PQHSA_OK || a.mass == nullptr) return rc;
  return launch_paged_mass(b, st);
}

}  // namespace pqhsa
