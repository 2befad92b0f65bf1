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
// Two launches: the selection (one CTA per stream: radix select over the keys, then the slots in order), which leaves
// source[i] = the slot whose key slot i takes over, and the moves over the whole GPU.
#include "paged.cuh"
#include "radix_select.cuh"

namespace pqhsa {

constexpr int kEvThreads = 1024;

// order-preserving key, +0 and -0 alike, NaN as -inf
__device__ __forceinline__ uint32_t evict_key(const PagedArgs& a, int recent, int last, float mass, int pos) {
  if (pos < a.sinks || (long long)pos > (long long)last - recent) return float_key(-kNegInf);
  return float_key(mass != mass ? kNegInf : mass + 0.f);
}

__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const PagedArgs a, const PagedEvict e) {
  __shared__ RadixShared sh;
  __shared__ int wtot[32];
  const int tid = threadIdx.x, r = blockIdx.x / a.H;
  const int64_t stream = blockIdx.x;
  const int n = min(max(__ldg(a.seq_lens + r), 0), a.limit), K = e.budget;
  int32_t* source = e.source + stream * K;
  for (int i = tid; i < K; i += kEvThreads) source[i] = i < n ? i : -1;
  if (n <= K) return;
  const int last = __ldg(a.query_pos + r);
  const float* mass = a.mass + stream * a.cap;
  const int32_t* pos = a.key_pos + stream * a.cap;
  int32_t* holes = e.holes + stream * K;
  auto key = [&](int i) { return evict_key(a, e.recent, last, mass[i], pos[i]); };
  uint32_t T;
  int ties;
  block_radix_threshold<kEvThreads>(key, n, K, sh, T, ties);
  int tied = 0, hole = 0, late = 0;  // slots so far
  for (int base = 0; base < n; base += kEvThreads) {
    const int i = base + tid;
    const uint32_t k = i < n ? key(i) : 0u;
    int total;
    const int rank = tied + block_exscan(i < n && k == T ? 1 : 0, wtot, &total);
    tied += total;
    const bool keep = i < n && (k > T || (k == T && rank < ties));
    const int at = hole + block_exscan(i < K && !keep ? 1 : 0, wtot, &total);
    hole += total;
    if (i < K && !keep) holes[at] = i;
    const int from = late + block_exscan(i >= K && keep ? 1 : 0, wtot, &total);
    late += total;
    __syncthreads();  // holes of this round are written; those a late slot needs lie in this round or before
    if (i >= K && keep) source[holes[from]] = i;
  }
}

// One warp per 32 kept slots: positions and weights by lane, then the moved rows one after the other.
template <typename E>
__global__ void __launch_bounds__(256) evict_move_kernel(const PagedArgs a, const PagedEvict e) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  const long long first = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int per = (e.budget + 31) / 32;
  E* kb = static_cast<E*>(const_cast<void*>(a.k_base));
  E* vb = static_cast<E*>(const_cast<void*>(a.v_base));
  constexpr int pieces = kD * sizeof(E) / 16;
  for (long long w = first; w < (long long)a.B * a.H * per; w += warps) {
    const int64_t stream = w / per;
    const int r = (int)(stream / a.H), h = (int)(stream % a.H), i = (int)(w % per) * 32 + lane;
    const int src = i < e.budget ? e.source[stream * e.budget + i] : -1;
    int64_t from = -1, to = -1;
    if (src >= 0) {
      e.new_mass[stream * a.cap + i] = a.mass[stream * a.cap + src];
      e.new_pos[stream * a.cap + i] = a.key_pos[stream * a.cap + src];
      if (src != i) {
        from = paged_offset(a, r, h, src);
        to = paged_offset(a, r, h, i);
      }
    }
    unsigned moves = __ballot_sync(0xffffffffu, from >= 0 && to >= 0);
    while (moves != 0u) {
      const int j = __ffs(moves) - 1;
      moves &= moves - 1;
      const int64_t f = __shfl_sync(0xffffffffu, from, j), t = __shfl_sync(0xffffffffu, to, j);
#pragma unroll
      for (int p = lane; p < 2 * pieces; p += 32) {
        const int x = (p % pieces) * (16 / (int)sizeof(E));
        const E* s = (p < pieces ? kb : vb) + f + x;
        E* d = (p < pieces ? kb : vb) + t + x;
        *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(s);
      }
    }
  }
  for (long long r = (long long)blockIdx.x * blockDim.x + threadIdx.x; r < a.B; r += (long long)gridDim.x * blockDim.x)
    e.new_lens[r] = min(a.seq_lens[r], min(e.budget, a.limit));
}

int launch_paged_evict(const PagedArgs& a, const PagedEvict& e, int dtype, cudaStream_t st) {
  evict_select_kernel<<<a.B * a.H, kEvThreads, 0, st>>>(a, e);
  if (int rc = check_launch("evict_select")) return rc;
  const long long warps = (long long)a.B * a.H * ((e.budget + 31) / 32);
  const long long want = (warps + 7) / 8, most = (long long)sm_count() * 8;
  const unsigned grid = (unsigned)(want < most ? want : most);
  PQHSA_DISPATCH_E(dtype, (evict_move_kernel<E><<<grid, 256, 0, st>>>(a, e)));
  return check_launch("evict_move");
}

// One CTA per request: T rows of every KV head go to slots n .. n + T - 1 with their positions and no weight yet.  A
// negative length marks an idle request; rows that do not fit the request's slots, or whose page is missing, are
// dropped.
template <typename E>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedArgs a, const E* __restrict__ k, const E* __restrict__ v,
                                                           int32_t* new_lens) {
  const int r = blockIdx.x, lane = threadIdx.x & 31;
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
  PQHSA_DISPATCH_E(dtype, (paged_append_kernel<E><<<a.B, 256, 0, st>>>(a, static_cast<const E*>(k), static_cast<const E*>(v),
                                                                      new_lens)));
  return check_launch("paged_append");
}

}  // namespace pqhsa
