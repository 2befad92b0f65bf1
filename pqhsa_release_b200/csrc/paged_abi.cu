// extern "C" entry points of the dense paged-cache operators: validation, workspace layout, launches.
#include <math.h>

#include "paged.cuh"

namespace pqhsa {

static inline size_t align256(size_t v) { return (v + 255) / 256 * 256; }

static inline size_t paged_score_stride(int cap) { return ((size_t)cap + 15) / 16 * 16; }

struct PagedWs {
  size_t part_ml, part_acc, row_lse2, scores, total;
};
static PagedWs paged_ws(const pqhsa_paged_params* p) {
  PagedWs w;
  const size_t parts = (size_t)2 * sm_count(), R = (size_t)p->group * p->query_len;
  const size_t rows = R < kPagedGroupRows ? (R + 7) / 8 * 8 : kPagedGroupRows;
  const size_t streams = (size_t)p->requests * p->kv_heads;
  size_t off = sizeof(int32_t) * kPagedMaxCtas;  // counters first: they stay where they are whatever the call's size
  w.part_ml = off;
  off = align256(off + parts * kPagedGroupRows * sizeof(float2));
  w.part_acc = off;
  off = align256(off + parts * (rows <= 8 ? 8 : rows <= 16 ? 16 : 32) * kD * sizeof(float));
  w.row_lse2 = off;
  off = align256(off + streams * R * sizeof(float));
  w.scores = off;
  if (p->mass != nullptr) off = align256(off + streams * R * paged_score_stride(p->slot_capacity) * sizeof(float));
  w.total = off;
  return w;
}

static int check_paged(const pqhsa_paged_params* p) {
  if (p == nullptr) return set_error(PQHSA_E_NULL, "params is null");
  if (p->abi_version != PQHSA_ABI_VERSION)
    return set_error(PQHSA_E_SHAPE, "abi_version %d, library speaks %d", p->abi_version, PQHSA_ABI_VERSION);
  if (p->dtype < PQHSA_F32 || p->dtype > PQHSA_F16) return set_error(PQHSA_E_DTYPE, "unknown dtype %d", p->dtype);
  if (p->head_dim != kD) return set_error(PQHSA_E_SHAPE, "head_dim must be %d, got %d", kD, p->head_dim);
  if (p->requests < 0 || p->requests > (1 << 16)) return set_error(PQHSA_E_SHAPE, "requests must be in 0..65536");
  if (p->kv_heads < 1 || p->kv_heads > 1024) return set_error(PQHSA_E_SHAPE, "kv_heads must be in 1..1024");
  if (p->group < 1 || p->group > 16) return set_error(PQHSA_E_SHAPE, "group must be in 1..16, got %d", p->group);
  if (p->query_len < 1 || p->query_len > kPagedMaxQuery)
    return set_error(PQHSA_E_SHAPE, "query_len must be in 1..%d, got %d", kPagedMaxQuery, p->query_len);
  if (p->group * p->query_len > kPagedMaxRows)
    return set_error(PQHSA_E_SHAPE, "group * query_len must be at most %d, got %d", kPagedMaxRows, p->group * p->query_len);
  if (p->slot_capacity < 1 || p->slot_capacity > (1 << 24))
    return set_error(PQHSA_E_SHAPE, "slot_capacity must be in 1..2^24, got %d", p->slot_capacity);
  if ((long long)p->requests * p->kv_heads * 2 * (p->slot_capacity / 8 + 2) > 0x7fffffffLL)
    return set_error(PQHSA_E_SHAPE, "requests * kv_heads * slot_capacity must stay below 2^33");
  return PQHSA_OK;
}

static int check_cache(const pqhsa_paged_params* p) {
  if (!p->k_base || !p->v_base) return set_error(PQHSA_E_NULL, "k_base / v_base is null");
  if (!p->seq_lens) return set_error(PQHSA_E_NULL, "seq_lens is null");
  if (p->block_size <= 0 || p->num_blocks <= 0 || (p->block_table != nullptr && p->max_blocks <= 0))
    return set_error(PQHSA_E_SHAPE, "block_size, num_blocks and max_blocks must be positive");
  if (p->block_table == nullptr && p->num_blocks < p->requests)
    return set_error(PQHSA_E_SHAPE, "a contiguous cache needs a block per request (%d for %d)", p->num_blocks, p->requests);
  const int64_t row_align = p->dtype == PQHSA_F32 ? 4 : 8;
  if (p->stride_block % row_align || p->stride_head % row_align || p->stride_row % row_align)
    return set_error(PQHSA_E_SHAPE, "KV strides must keep rows 16-byte aligned");
  if (((uintptr_t)p->k_base | (uintptr_t)p->v_base) & 15) return set_error(PQHSA_E_SHAPE, "k_base / v_base must be 16-byte aligned");
  if (p->sink_tokens < 0 || p->window < 0) return set_error(PQHSA_E_SHAPE, "window and sink_tokens must be non-negative");
  return PQHSA_OK;
}

static int check_rows(const pqhsa_paged_params* p, const void* base, int64_t sr, int64_t st, int64_t sh, const char* what) {
  if (base == nullptr) return set_error(PQHSA_E_NULL, "%s is null", what);
  const int64_t row_align = p->dtype == PQHSA_F32 ? 4 : 8;
  if (((uintptr_t)base & 15) || sr % row_align || st % row_align || sh % row_align)
    return set_error(PQHSA_E_SHAPE, "rows of %s must be 16-byte aligned", what);
  return PQHSA_OK;
}

static PagedArgs paged_args(const pqhsa_paged_params* p) {
  PagedArgs a = {};
  a.k_base = p->k_base; a.v_base = p->v_base;
  a.block_table = p->block_table;
  a.max_blocks = p->max_blocks; a.block_size = p->block_size; a.num_blocks = p->num_blocks;
  a.stride_block = p->stride_block; a.stride_head = p->stride_head; a.stride_row = p->stride_row;
  a.B = p->requests; a.H = p->kv_heads; a.G = p->group; a.T = p->query_len; a.R = p->group * p->query_len;
  a.groups = (a.R + kPagedGroupRows - 1) / kPagedGroupRows;
  a.g_inv = 65536 / p->group + 1;
  a.cap = p->slot_capacity;
  const long long room = p->block_table != nullptr ? (long long)p->max_blocks * p->block_size : p->block_size;
  a.limit = room < a.cap ? (int)room : a.cap;
  a.scale_log2 = p->scale * kLog2e;
  a.softcap = p->softcap;
  a.cap_log2 = p->softcap * kLog2e;
  a.cap_in = p->softcap > 0.f ? 2.f * kLog2e * p->scale / p->softcap : 0.f;
  a.slopes = p->alibi_slopes;
  a.window = p->window; a.sinks = p->sink_tokens;
  a.seq_lens = p->seq_lens; a.first_key = p->first_key; a.query_pos = p->query_pos;
  a.key_pos = p->key_pos; a.mass = p->mass;
  a.q = p->q; a.q_sr = p->q_stride_request; a.q_st = p->q_stride_token; a.q_sh = p->q_stride_head;
  a.out = p->out; a.o_sr = p->out_stride_request; a.o_st = p->out_stride_token; a.o_sh = p->out_stride_head;
  a.lse = p->lse;
  return a;
}

}  // namespace pqhsa

using namespace pqhsa;

extern "C" {

size_t pqhsa_paged_workspace_bytes(const pqhsa_paged_params* p) {
  return check_paged(p) == PQHSA_OK ? paged_ws(p).total : 0;
}

int pqhsa_paged_attention(const pqhsa_paged_params* p, void* stream) {
  if (int rc = check_paged(p)) return rc;
  if (p->requests == 0) return PQHSA_OK;
  if (int rc = check_cache(p)) return rc;
  if (int rc = check_rows(p, p->q, p->q_stride_request, p->q_stride_token, p->q_stride_head, "q")) return rc;
  if (int rc = check_rows(p, p->out, p->out_stride_request, p->out_stride_token, p->out_stride_head, "out")) return rc;
  if (p->key_pos != nullptr && p->query_pos == nullptr) return set_error(PQHSA_E_NULL, "key_pos needs query_pos");
  if (!isfinite(p->scale) || !isfinite(p->softcap) || p->softcap < 0.f || !isfinite(paged_args(p).cap_in))
    return set_error(PQHSA_E_SHAPE, "scale must be finite, softcap finite, non-negative and not vanishing against scale");
  if (!p->workspace || ((uintptr_t)p->workspace & 255))
    return set_error(PQHSA_E_WORKSPACE, "workspace missing or not 256-byte aligned");
  if (sm_count() * kPagedMassCtas >= kPagedMaxCtas)
    return set_error(PQHSA_E_CAPACITY, "more than %d SMs", (kPagedMaxCtas - 1) / kPagedMassCtas);
  const PagedWs w = paged_ws(p);
  if (p->workspace_bytes < w.total)
    return set_error(PQHSA_E_WORKSPACE, "workspace has %zu bytes, %zu needed", p->workspace_bytes, w.total);
  PagedArgs a = paged_args(p);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.tickets = reinterpret_cast<int32_t*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  a.part_acc = reinterpret_cast<float*>(ws + w.part_acc);
  a.row_lse2 = reinterpret_cast<float*>(ws + w.row_lse2);
  a.scores = p->mass != nullptr ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  a.score_stride = (int64_t)paged_score_stride(p->slot_capacity);
  return launch_paged_attend(a, p->dtype, (cudaStream_t)stream);
}

int pqhsa_paged_append(const pqhsa_paged_params* p, const void* k, const void* v, int32_t* new_lens, void* stream) {
  if (int rc = check_paged(p)) return rc;
  if (p->requests == 0) return PQHSA_OK;
  if (int rc = check_cache(p)) return rc;
  if (int rc = check_rows(p, k, p->q_stride_request, p->q_stride_token, p->q_stride_head, "k")) return rc;
  if (int rc = check_rows(p, v, p->q_stride_request, p->q_stride_token, p->q_stride_head, "v")) return rc;
  if (!new_lens) return set_error(PQHSA_E_NULL, "new_lens is null");
  return launch_paged_append(paged_args(p), k, v, new_lens, p->dtype, (cudaStream_t)stream);
}

int pqhsa_paged_evict(const pqhsa_paged_params* p, int32_t budget, int32_t recent, int32_t* new_lens, float* new_mass,
                      int32_t* new_pos, int32_t* source, int32_t* scratch, void* stream) {
  if (int rc = check_paged(p)) return rc;
  if (p->requests == 0) return PQHSA_OK;
  if (int rc = check_cache(p)) return rc;
  if (!p->mass || !p->key_pos || !p->query_pos) return set_error(PQHSA_E_NULL, "an eviction needs mass, key_pos and query_pos");
  if (!new_lens || !new_mass || !new_pos || !source || !scratch) return set_error(PQHSA_E_NULL, "an output of the eviction is null");
  if (budget < 1 || budget > (1 << 24)) return set_error(PQHSA_E_SHAPE, "budget must be in 1..2^24, got %d", budget);
  if (recent < 0 || (long long)recent + p->sink_tokens > budget)
    return set_error(PQHSA_E_SHAPE, "sink_tokens %d + recent %d must fit the budget %d", p->sink_tokens, recent, budget);
  if ((long long)p->requests * p->kv_heads > 65535) return set_error(PQHSA_E_SHAPE, "requests * kv_heads must be at most 65535");
  const PagedEvict e = {budget, recent, new_lens, new_mass, new_pos, source, scratch};
  return launch_paged_evict(paged_args(p), e, p->dtype, (cudaStream_t)stream);
}

unsigned long long pqhsa_stream_capture_id(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

}  // extern "C"
