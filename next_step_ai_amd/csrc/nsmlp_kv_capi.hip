// C ABI of the paged 8-bit K/V cache and its attention: argument validation
// and launches.  Declarations are in include/nsmlp.h.
#include <math.h>
#include <string.h>

#include "nsmlp_kv.h"

namespace nsmlp {

namespace {

int check_device() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return set_error(NSMLP_ENODEV, "no HIP device");
  return NSMLP_OK;
}

int block_shift(int tokens) { return tokens == 16 ? 4 : tokens == 32 ? 5 : tokens == 64 ? 6 : -1; }

int cache_view(const nsmlp_kv_cache* c, KvView& v) {
  if (c == nullptr) return set_error(NSMLP_EINVAL, "cache must be non-NULL");
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(NSMLP_EINVAL, "head_dim %d must be 64 or 128", c->head_dim);
  if (block_shift(c->block_tokens) < 0)
    return set_error(NSMLP_EINVAL, "block_tokens %d must be 16, 32 or 64", c->block_tokens);
  if (c->format != NSMLP_KV_INT8 && c->format != NSMLP_KV_E4M3)
    return set_error(NSMLP_EINVAL, "unknown cache format %d", c->format);
  if (c->kv_heads < 1 || c->kv_heads > 1024) return set_error(NSMLP_EINVAL, "kv_heads %d out of range [1, 1024]", c->kv_heads);
  if (c->num_blocks < 1 || c->num_blocks > (1 << 26))
    return set_error(NSMLP_EINVAL, "num_blocks %d out of range [1, 2^26]", c->num_blocks);
  if (c->data == nullptr || c->scale == nullptr) return set_error(NSMLP_EINVAL, "cache data and scale must be non-NULL");
  if (!aligned16(c->data) || !aligned16(c->scale)) return set_error(NSMLP_EINVAL, "cache data and scale must be 16-byte aligned");
  v.data = c->data;
  v.scale = c->scale;
  v.num_blocks = c->num_blocks;
  v.heads = c->kv_heads;
  v.D = c->head_dim;
  v.B = c->block_tokens;
  v.b_shift = block_shift(c->block_tokens);
  v.fmt = c->format;
  return NSMLP_OK;
}

int check_dtype(int dtype) {
  if (dtype != NSMLP_DTYPE_F16 && dtype != NSMLP_DTYPE_BF16) return set_error(NSMLP_EINVAL, "unknown dtype %d", dtype);
  return NSMLP_OK;
}

// rows of [heads][D] elements that 16-byte loads may read
int check_rows(const char* what, const void* p, long long row, long long head) {
  if (p == nullptr) return set_error(NSMLP_EINVAL, "%s must be non-NULL", what);
  if (!aligned16(p) || row % 8 != 0 || head % 8 != 0)
    return set_error(NSMLP_EINVAL, "%s must be 16-byte aligned with row and head strides that are multiples of 8 elements", what);
  return NSMLP_OK;
}

int check_batch(const nsmlp_kv_batch* b) {
  if (b == nullptr) return set_error(NSMLP_EINVAL, "batch must be non-NULL");
  if (b->requests < 1 || b->requests > kKvMaxRequests)
    return set_error(NSMLP_EINVAL, "requests %d out of range [1, %d]", b->requests, kKvMaxRequests);
  if (b->max_blocks < 1 || b->max_blocks > (1 << 24))
    return set_error(NSMLP_EINVAL, "max_blocks %d out of range [1, 2^24]", b->max_blocks);
  if (b->num_blocks < 1 || b->num_blocks > (1 << 26))
    return set_error(NSMLP_EINVAL, "num_blocks %d out of range [1, 2^26]", b->num_blocks);
  if (block_shift(b->block_tokens) < 0)
    return set_error(NSMLP_EINVAL, "block_tokens %d must be 16, 32 or 64", b->block_tokens);
  if (b->kv_heads < 1 || b->kv_heads > 1024 || b->q_heads < 1 || b->q_heads > 1024 * b->kv_heads)
    return set_error(NSMLP_EINVAL, "q_heads %d and kv_heads %d out of range", b->q_heads, b->kv_heads);
  if (b->cached == nullptr || b->table == nullptr || b->ring == nullptr || b->state == nullptr)
    return set_error(NSMLP_EINVAL, "cached, table, ring and state must be non-NULL");
  return NSMLP_OK;
}

constexpr int kMaxTokens = 1 << 24;

// query rows per token and K/V head (the attention itself wants a whole number)
int group_of(const nsmlp_kv_batch* b) { return (b->q_heads + b->kv_heads - 1) / b->kv_heads; }

int batch_schedule(const nsmlp_kv_batch* b, int total, int max_new, KvSchedule& s) {
  int rc = check_batch(b);
  if (rc) return rc;
  if (total < 0 || total > kMaxTokens) return set_error(NSMLP_EINVAL, "total %d out of range [0, 2^24]", total);
  if (max_new < 0) return set_error(NSMLP_EINVAL, "max_new %d must not be negative", max_new);
  const int group = group_of(b);
  if ((long long)total * group > (1LL << 28)) return set_error(NSMLP_EINVAL, "%d tokens of %d heads: too many rows", total, group);
  if ((long long)b->requests * b->max_blocks > (1LL << 30))
    return set_error(NSMLP_EINVAL, "%d requests of %d blocks: at most 2^30 table entries", b->requests, b->max_blocks);
  s = kv_schedule(b->requests, total, max_new == 0 ? total : max_new, group, b->kv_heads);
  return NSMLP_OK;
}

int check_step(const nsmlp_kv_batch* b, const nsmlp_kv_step* st, KvSchedule& s) {
  if (st == nullptr) return set_error(NSMLP_EINVAL, "step must be non-NULL");
  int rc = batch_schedule(b, st->total, st->max_new, s);
  if (rc) return rc;
  if ((st->total > 0 && st->slots == nullptr) || st->q_start == nullptr || st->kv_len == nullptr || st->next == nullptr ||
      st->info == nullptr || st->schedule == nullptr)
    return set_error(NSMLP_EINVAL, "the step's arrays must be non-NULL");
  if (!aligned16(st->schedule)) return set_error(NSMLP_EINVAL, "the schedule must be 16-byte aligned");
  if (st->schedule_bytes < (size_t)s.ints * 4)
    return set_error(NSMLP_ENOSPC, "the schedule needs %zu bytes, got %zu", (size_t)s.ints * 4, st->schedule_bytes);
  return NSMLP_OK;
}

}  // namespace

}  // namespace nsmlp

using namespace nsmlp;

extern "C" {

int nsmlp_kv_append(const nsmlp_kv_cache* cache, const void* k, long long k_row_stride, long long k_head_stride,
                    const void* v, long long v_row_stride, long long v_head_stride, int dtype, const int64_t* slots, int n,
                    void* stream) {
  NSMLP_FAULT_POINT("kv_append");
  KvAppendArgs a;
  int rc = cache_view(cache, a.c);
  if (rc || (rc = check_dtype(dtype))) return rc;
  if (n < 0 || n > kMaxTokens || (long long)n * a.c.heads > (1 << 28))
    return set_error(NSMLP_EINVAL, "n = %d rows of %d heads: at most 2^24 rows and 2^28 heads' rows", n, a.c.heads);
  if (n == 0) return NSMLP_OK;
  if (slots == nullptr) return set_error(NSMLP_EINVAL, "slots must be non-NULL");
  if ((rc = check_rows("k", k, k_row_stride, k_head_stride)) || (rc = check_rows("v", v, v_row_stride, v_head_stride))) return rc;
  if ((rc = check_device())) return rc;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_row = k_row_stride, a.k_head = k_head_stride, a.v_row = v_row_stride, a.v_head = v_head_stride;
  a.slots = slots;
  a.n = n;
  launch_kv_append(a, dtype == NSMLP_DTYPE_BF16, (hipStream_t)stream);
  return check_launch("nsmlp_kv_append");
}

int nsmlp_kv_read(const nsmlp_kv_cache* cache, const int64_t* slots, int n, void* k_out, void* v_out, int dtype,
                  void* stream) {
  NSMLP_FAULT_POINT("kv_read");
  KvReadArgs a;
  int rc = cache_view(cache, a.c);
  if (rc || (rc = check_dtype(dtype))) return rc;
  if (n < 0 || n > kMaxTokens || (long long)n * a.c.heads > (1 << 28))
    return set_error(NSMLP_EINVAL, "n = %d rows of %d heads: at most 2^24 rows and 2^28 heads' rows", n, a.c.heads);
  if (n == 0) return NSMLP_OK;
  if (slots == nullptr) return set_error(NSMLP_EINVAL, "slots must be non-NULL");
  if ((rc = check_rows("k_out", k_out, 0, 0)) || (rc = check_rows("v_out", v_out, 0, 0))) return rc;
  if ((rc = check_device())) return rc;
  a.slots = slots;
  a.n = n;
  a.k = (uint16_t*)k_out;
  a.v = (uint16_t*)v_out;
  launch_kv_read(a, dtype == NSMLP_DTYPE_BF16, (hipStream_t)stream);
  return check_launch("nsmlp_kv_read");
}

size_t nsmlp_kv_schedule_bytes(const nsmlp_kv_batch* batch, int total, int max_new) {
  KvSchedule s;
  return batch_schedule(batch, total, max_new, s) ? 0 : (size_t)s.ints * 4;
}

int nsmlp_kv_plan(const nsmlp_kv_batch* batch, const int32_t* new_tokens, const nsmlp_kv_step* step, void* stream) {
  NSMLP_FAULT_POINT("kv_plan");
  KvPlanArgs a;
  int rc = check_step(batch, step, a.s);
  if (rc) return rc;
  if (new_tokens == nullptr) return set_error(NSMLP_EINVAL, "new_tokens must be non-NULL");
  if ((rc = check_device())) return rc;
  a.R = batch->requests;
  a.total = step->total;
  a.max_blocks = batch->max_blocks;
  a.num_blocks = batch->num_blocks;
  a.B = batch->block_tokens;
  a.b_shift = block_shift(a.B);
  a.group = group_of(batch);
  a.cached = batch->cached;
  a.fresh = new_tokens;
  a.table = batch->table;
  a.ring = batch->ring;
  a.state = batch->state;
  a.slots = step->slots;
  a.q_start = step->q_start;
  a.kv_len = step->kv_len;
  a.next = step->next;
  a.info = step->info;
  a.sched = step->schedule;
  a.max_new = step->max_new == 0 ? 1 << 30 : step->max_new;
  a.row_limit = (1 << 28) / a.group;  // rows of a request fit 32 bits
  launch_kv_plan(a, (hipStream_t)stream);
  return check_launch("nsmlp_kv_plan");
}

int nsmlp_kv_commit(const nsmlp_kv_batch* batch, const nsmlp_kv_step* step, const int32_t* finished, void* stream) {
  NSMLP_FAULT_POINT("kv_commit");
  int rc = check_batch(batch);
  if (rc) return rc;
  if (step != nullptr && (step->next == nullptr || step->info == nullptr))
    return set_error(NSMLP_EINVAL, "the step's arrays must be non-NULL");
  if ((rc = check_device())) return rc;
  KvCommitArgs a;
  a.R = batch->requests;
  a.max_blocks = batch->max_blocks;
  a.num_blocks = batch->num_blocks;
  a.B = batch->block_tokens;
  a.b_shift = block_shift(a.B);
  a.cached = batch->cached;
  a.table = batch->table;
  a.ring = batch->ring;
  a.state = batch->state;
  a.next = step != nullptr ? step->next : nullptr;
  a.info = step != nullptr ? step->info : nullptr;
  a.finished = finished;
  launch_kv_commit(a, (hipStream_t)stream);
  return check_launch("nsmlp_kv_commit");
}

size_t nsmlp_paged_attention_workspace_bytes(const nsmlp_kv_batch* batch, int total, int max_new, int head_dim) {
  KvSchedule s;
  size_t off[4];
  if (batch_schedule(batch, total, max_new, s) || (head_dim != 64 && head_dim != 128)) return 0;
  return align_up(kCounterBytes) + kv_attn_partial_floats(s, batch->kv_heads, head_dim, off) * sizeof(float);
}

int nsmlp_paged_attention(const nsmlp_kv_cache* cache, const nsmlp_kv_batch* batch, const nsmlp_kv_step* step, const void* q,
                          long long q_row_stride, long long q_head_stride, int dtype, float scale, void* out, float* lse,
                          void* ws, size_t ws_bytes, void* stream) {
  NSMLP_FAULT_POINT("paged_attention");
  KvAttnArgs a;
  int rc = cache_view(cache, a.c);
  if (rc || (rc = check_step(batch, step, a.s)) || (rc = check_dtype(dtype))) return rc;
  if (cache->kv_heads != batch->kv_heads || cache->num_blocks != batch->num_blocks || cache->block_tokens != batch->block_tokens)
    return set_error(NSMLP_EINVAL, "the cache has %d heads and %d blocks of %d tokens, the batch %d, %d and %d", cache->kv_heads,
                     cache->num_blocks, cache->block_tokens, batch->kv_heads, batch->num_blocks, batch->block_tokens);
  if (batch->q_heads % batch->kv_heads != 0)
    return set_error(NSMLP_EINVAL, "q_heads %d must be a multiple of kv_heads %d", batch->q_heads, batch->kv_heads);
  if (!(scale > 0.0f) || !isfinite(scale)) return set_error(NSMLP_EINVAL, "scale %g must be positive and finite", (double)scale);
  if (step->total == 0) return NSMLP_OK;
  if ((rc = check_rows("q", q, q_row_stride, q_head_stride)) || (rc = check_rows("out", out, 0, 0))) return rc;
  size_t off[4];
  const size_t need = align_up(kCounterBytes) + kv_attn_partial_floats(a.s, batch->kv_heads, cache->head_dim, off) * sizeof(float);
  if (ws == nullptr || ws_bytes < need) return set_error(NSMLP_ENOSPC, "attention workspace needs %zu bytes, got %zu", need, ws_bytes);
  if (((uintptr_t)ws & (kAlign - 1)) != 0) return set_error(NSMLP_EINVAL, "workspace must be 256-byte aligned");
  if ((rc = check_device())) return rc;
  float* part = (float*)((char*)ws + align_up(kCounterBytes));
  a.acc_a = part + off[0], a.ml_a = part + off[1], a.acc_b = part + off[2], a.ml_b = part + off[3];
  a.status = (int*)((char*)ws + kStatusOff);
  a.count = (int*)((char*)ws + kBlkCountOff);
  a.q = (const uint16_t*)q;
  a.q_row = q_row_stride, a.q_head = q_head_stride;
  a.out = (uint16_t*)out;
  a.lse = lse;
  a.table = batch->table;
  a.q_start = step->q_start;
  a.kv_len = step->kv_len;
  a.sched = step->schedule;
  a.max_blocks = batch->max_blocks;
  a.R = batch->requests;
  a.total = step->total;
  a.group = group_of(batch);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  launch_kv_attention(a, dtype == NSMLP_DTYPE_BF16, (hipStream_t)stream);
  return check_launch("nsmlp_paged_attention");
}

}  // extern "C"
