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

// ---- tensor-core kernel for 16-bit caches: tiles of 16 keys ----------------------------------------------
// Both products run transposed, so that the many keys (and dimensions) are the 16 rows of an m16n8k16 and the few query
// rows its 8 columns: S^T[16 keys, 8 rows] = K q^T and O^T[16 dims, 8 rows] += V^T P^T.  K rows are the A operand as they
// lie (ldmatrix), V the A operand transposed (ldmatrix.trans); P^T gets from the accumulator layout of S^T into the B
// layout with one 8x8 transpose in registers per 8 keys.  A thread holds the same two query rows of every 8 in S^T and
// in O^T, so maxima, sums and rescaling need no exchange.  p is rounded to the 16-bit type for the product with V (half
// a step of a value in 0 .. 2^8; the sum it is divided by keeps 32 bits).  Against one row per m16 (P V with 16 rows
// of which 4 or 8 are real) this halves the instructions and the accumulators.
constexpr int kMKeys = 16;

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

// A warp's view of the tiles it has still to fetch: lane i < 16 looks after key i.  What the addresses depend on (page
// table, stored positions) is requested one tile before it is needed.
struct TileFetch {
  int32_t entry;  // page
  int32_t row;    // row in the page
  int32_t pos;    // position, or a value no token sees
};

template <typename E, int NB, int STAGES>
__global__ void __launch_bounds__(kPThreads, 1) paged_attend_mma_kernel(const PagedArgs a) {
  constexpr int ROWS = 8 * NB;
  constexpr bool QREG = NB <= 2;  // query rows as B fragments in registers; from shared memory when they would fill them
  constexpr int kStageB = 2 * kMKeys * kD * 2;  // bytes of a stage: 16 key rows, then 16 value rows, 256 bytes each
  extern __shared__ __align__(128) uint8_t smem_raw[];
  constexpr size_t kRing = (size_t)kPWarps * STAGES * kStageB;
  constexpr size_t kMerge = sizeof(float) * kPWarps * ROWS * kAccStride;
  float* acc_s = reinterpret_cast<float*>(smem_raw);  // merge buffer over the rings, used between streams
  uint8_t* tail = smem_raw + (kRing > kMerge ? kRing : kMerge);
  float2* ml_s = reinterpret_cast<float2*>(tail);                 // [warps][ROWS]
  uint8_t* q_s = tail + sizeof(float2) * kPWarps * ROWS;          // [ROWS][128] E, pieces swizzled, only without QREG
  __shared__ int pos_s[kPWarps][STAGES][kMKeys];
  __shared__ int seen_s[kPWarps][STAGES];   // keys some row of the step sees; << 16: keys not all of them see
  __shared__ int last_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t4 = lane & 3, l4 = lane >> 2;
  const E* kb = static_cast<const E*>(a.k_base);
  const E* vb = static_cast<const E*>(a.v_base);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem_raw) + warp * (STAGES * kStageB);
  // shared-memory addresses inside a tile, before the 16-byte piece is added: piece j of row k lies at j ^ (k & 7)
  const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_hi = lane >> 4;          // K: rows 0-7 | 8-15, then the upper 8 dims
  const int v_row = (lane & 7) + (lane >> 4) * 8, v_hi = (lane >> 3) & 1;          // V: upper 8 dims, then rows 8-15
  const int g_row = lane >> 3, g_piece = lane & 7;                                 // copies: 4 rows x 128 bytes at a time

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
    const int mine = count > warp ? (count - warp + kPWarps - 1) / kPWarps : 0;
    const int32_t* kpos = a.key_pos != nullptr ? a.key_pos + ((int64_t)c.r * a.H + h) * a.cap : nullptr;
    const int32_t* table = a.block_table != nullptr ? a.block_table + (int64_t)c.r * a.max_blocks : nullptr;

    auto fetch = [&](int it) {
      TileFetch f = {-1, 0, -1};
      if (it < mine && lane < kMKeys) {
        const int slot = paged_tile(c.g, c.tile + warp + it * kPWarps) * kMKeys + lane;
        if (slot < c.g.n) {
          f.pos = kpos != nullptr ? __ldg(kpos + slot) : slot;
          f.entry = c.r;
          f.row = slot;
          if (table != nullptr) {
            const int b = slot / a.block_size;
            f.row = slot - b * a.block_size;
            f.entry = __ldg(table + b);
          }
        }
      }
      return f;
    };
    auto load = [&](int it, int st, const TileFetch& f) {
      if (it < mine) {
        bool any = f.entry >= 0 && f.entry < a.num_blocks && f.pos >= c.g.first && f.pos <= c.g.p_last;
        bool all = f.pos <= c.g.p_first;
        if (a.window > 0) {
          const bool sink = f.pos - c.g.first < a.sinks;
          any = any && (c.g.p_first - f.pos < a.window || sink);
          all = all && (c.g.p_last - f.pos < a.window || sink);
        }
        const unsigned seen = __ballot_sync(0xffffffffu, any), mixed = __ballot_sync(0xffffffffu, any && !all);
        if (lane < kMKeys) pos_s[warp][st][lane] = f.pos;
        if (lane == 0) seen_s[warp][st] = (int)((seen & 0xffffu) | (mixed << 16));
        const int64_t off = any ? f.entry * a.stride_block + h * a.stride_head + f.row * a.stride_row : 0;
        const uint32_t dst = ring + st * kStageB;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 4 * i + g_row;
          const int64_t o = __shfl_sync(0xffffffffu, off, k) + g_piece * 8;
          const bool take = (seen >> k) & 1u;
          const uint32_t to = dst + k * 256 + ((g_piece ^ (k & 7)) << 4);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            cp_async16_zfill(to + j * 128, kb + o + j * 64, take);
            cp_async16_zfill(to + j * 128 + kMKeys * 256, vb + o + j * 64, take);
          }
        }
      }
      cp_async_commit();
    };

    uint32_t qf[QREG ? NB : 1][8][2];
    if constexpr (!QREG) __syncthreads();  // q_s of the stream before has been read
    if constexpr (QREG) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int row = 8 * nb + l4, full = row0 + row;
        const E* src = static_cast<const E*>(a.q) + (int64_t)c.r * a.q_sr + (int64_t)(full / a.G) * a.q_st +
                       (int64_t)(h * a.G + full % a.G) * a.q_sh + 2 * t4;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qf[nb][kk][0] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16)) : 0u;
          qf[nb][kk][1] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16 + 8)) : 0u;
        }
      }
    } else {
      for (int i = tid; i < ROWS * 16; i += kPThreads) {
        const int row = i >> 4, piece = i & 15, full = row0 + row;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows)
          v = __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(a.q) + (int64_t)c.r * a.q_sr +
                                                   (int64_t)(full / a.G) * a.q_st + (int64_t)(h * a.G + full % a.G) * a.q_sh) + piece);
        *reinterpret_cast<uint4*>(q_s + row * 256 + ((piece ^ (row & 7)) << 4)) = v;
      }
      __syncthreads();
    }
    TileFetch next = fetch(0);
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) {
      const TileFetch f = next;
      next = fetch(st + 1);
      load(st, st, f);
    }
    float m[NB][2], l[NB][2], slope[NB][2], o[NB][8][4];
    int p_at[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = 8 * nb + 2 * t4 + j, full = row0 + row;
        m[nb][j] = kNegInf;
        l[nb][j] = 0.f;
        p_at[nb][j] = row < rows ? c.g.p_first + full / a.G : -1;
        slope[nb][j] = row < rows && a.slopes != nullptr ? kLog2e * __ldg(a.slopes + h * a.G + full % a.G) : 0.f;
      }
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nb][db][j] = 0.f;
    }

    for (int it = 0; it < mine; ++it) {
      const int st = it % STAGES;
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      {
        const TileFetch f = next;
        next = fetch(it + STAGES);
        load(it + STAGES - 1, (it + STAGES - 1) % STAGES, f);
      }
      const uint32_t kt = ring + st * kStageB, vt = kt + kMKeys * 256;
      float s[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[nb][j] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; kk += 2) {
        uint32_t a0[4], a1[4];
        ldmatrix4(a0, kt + k_row * 256 + (((2 * kk + k_hi) ^ (k_row & 7)) << 4));
        ldmatrix4(a1, kt + k_row * 256 + (((2 * kk + 2 + k_hi) ^ (k_row & 7)) << 4));
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
      // s[nb][0], [1]: key l4, rows 2 t4 and 2 t4 + 1 of block nb; [2], [3]: key l4 + 8
      const unsigned flags = (unsigned)seen_s[warp][st];
      const int pos0 = pos_s[warp][st][l4], pos1 = pos_s[warp][st][l4 + 8];
      const bool seen0 = (flags >> l4) & 1u, seen1 = (flags >> (l4 + 8)) & 1u;
      const unsigned mixed = flags >> 16;
      bool raise = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int pos = j < 2 ? pos0 : pos1, p = p_at[nb][j & 1];
          bool vis = (j < 2 ? seen0 : seen1) && p >= 0;
          if (mixed != 0u) vis = vis && paged_sees(c.g, a, pos, p);
          s[nb][j] = vis ? paged_score(a, s[nb][j], slope[nb][j & 1], p - pos) : kNegInf;
          raise |= s[nb][j] > m[nb][j & 1] + kLazy;
        }
      }
      if (a.scores != nullptr) {
        const int slot = paged_tile(c.g, c.tile + warp + it * kPWarps) * kMKeys + l4;
        float* dst = a.scores + (((int64_t)c.r * a.H + h) * a.R + row0 + 2 * t4) * a.cap + slot;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (8 * nb + 2 * t4 + (j & 1) < rows && slot + (j >> 1) * 8 < c.g.n)
              dst[(int64_t)(8 * nb + (j & 1)) * a.cap + (j >> 1) * 8] = s[nb][j];
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = fmaxf(s[nb][j], s[nb][j + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float to = fmaxf(m[nb][j], top);
            const float f = m[nb][j] == kNegInf ? (to == kNegInf ? 1.f : 0.f) : ex2(m[nb][j] - to);
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
          s[nb][j] = s[nb][j] == kNegInf ? 0.f : ex2(s[nb][j] - m[nb][j & 1]);
          l[nb][j & 1] += s[nb][j];
        }
      if (mixed != 0u) {
        // Keys that only some rows see (at most the last query_len - 1 and as many at the window's edge): a product with
        // p = 0 would let an infinite or NaN value through, so these are added one by one and then taken out.
        uint8_t* vrow = smem_raw + (vt - (uint32_t)__cvta_generic_to_shared(smem_raw));
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
        ldmatrix4_trans(av, vt + v_row * 256 + (((2 * db + v_hi) ^ (v_row & 7)) << 4));
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16816<E>(o[nb][db], av, pf[nb][0], pf[nb][1]);
      }
      __syncwarp();  // the slot may be filled again
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with its ring: the merge buffer lies over it
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nb][j] += __shfl_xor_sync(0xffffffffu, l[nb][j], d);
        if (l4 == 0) ml_s[warp * ROWS + 8 * nb + 2 * t4 + j] = make_float2(m[nb][j], l[nb][j]);
      }
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc_s[((size_t)warp * ROWS + 8 * nb + 2 * t4 + (j & 1)) * kAccStride + db * 16 + l4 + (j >> 1) * 8] = o[nb][db][j];
    }
    __syncthreads();
    paged_finish<E>(a, c, x - c.tile, c.tile, count, total, C, rows, ROWS, ml_s, acc_s, &last_s);
    x += count;
    if (x >= x_end) return;
    __syncthreads();  // the rings are free again
    paged_next_stream(a, c);
  }
}

template <typename E, int NB, int STAGES>
static int launch_mma(const PagedArgs& a, cudaStream_t st) {
  constexpr int ROWS = 8 * NB;
  constexpr size_t ring = (size_t)kPWarps * STAGES * 2 * kMKeys * kD * 2;
  constexpr size_t merge = sizeof(float) * kPWarps * ROWS * kAccStride;
  constexpr size_t smem = (ring > merge ? ring : merge) + sizeof(float2) * kPWarps * ROWS + (NB > 2 ? ROWS * 256 : 0);
  static_assert(smem <= 220 * 1024, "shared memory of a CTA");
  auto kern = paged_attend_mma_kernel<E, NB, STAGES>;
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
  const int rows = a.R < kPagedGroupRows ? a.R : kPagedGroupRows;
  int rc = PQHSA_OK;
  if (dtype == PQHSA_F32) {
    b.tile_log2 = 3;
    rc = rows <= 8 ? launch_simple<float, 8, 2>(b, st) : rows <= 16 ? launch_simple<float, 16, 2>(b, st) : launch_simple<float, 32, 2>(b, st);
  } else {
    b.tile_log2 = 4;
    if (dtype == PQHSA_BF16) {
      using E = __nv_bfloat16;
      rc = rows <= 8 ? launch_mma<E, 1, 3>(b, st) : rows <= 16 ? launch_mma<E, 2, 3>(b, st) : launch_mma<E, 4, 3>(b, st);
    } else {
      using E = __half;
      rc = rows <= 8 ? launch_mma<E, 1, 3>(b, st) : rows <= 16 ? launch_mma<E, 2, 3>(b, st) : launch_mma<E, 4, 3>(b, st);
    }
  }
  if (rc != PQHSA_OK || a.mass == nullptr) return rc;
  return launch_paged_mass(b, st);
}

}  // namespace pqhsa
