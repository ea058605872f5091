// swa_paged_api.cu -- the extern "C" entry points of the rotary and paged-cache operators:
// argument checks and parameter blocks.
#include <limits.h>

#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
cudaError_t launch_rotary(const RotaryParams& r, const SwaRotaryArgs& a, cudaStream_t st);
cudaError_t launch_paged_append(const PagedParams& c, const RotaryParams& r, const SwaPagedAppendArgs& a,
                                cudaStream_t st);
cudaError_t launch_paged_decode(const PagedParams& c, const SwaPagedDecodeArgs& a, cudaStream_t st);
cudaError_t launch_paged_evict(const PagedParams& c, const SwaPagedEvictArgs& a, cudaStream_t st);
size_t paged_decode_workspace(const SwaPagedDecodeArgs& a);
size_t paged_evict_workspace(const SwaPagedEvictArgs& a);
}  // namespace swa

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A device workspace of at least `need` bytes, 256-byte aligned.
int check_workspace(const void* ws, size_t bytes, size_t need) {
  if (need && (!ws || bytes < need)) return SWA_ERR_WORKSPACE;
  return (reinterpret_cast<uintptr_t>(ws) & 255u) ? SWA_ERR_WORKSPACE : SWA_OK;
}

int build_rotary(const SwaRotary& r, int head_dim, bool need_ptrs, swa::RotaryParams* o) {
  if (r.n_axes < 1 || r.n_freq < 0 || r.n_freq > SWA_ROTARY_MAX_FREQS || 2 * r.n_freq > head_dim)
    return SWA_ERR_INVALID_ARG;
  if (r.pos_stride_axis < 0 || r.pos_stride_b < 0 || r.pos_stride_l < 0) return SWA_ERR_UNSUPPORTED;
  for (int i = 0; i < r.n_freq; ++i)
    if (r.axis[i] >= r.n_axes) return SWA_ERR_INVALID_ARG;
  if (need_ptrs && r.n_freq > 0 && (!r.inv_freq || !r.positions)) return SWA_ERR_INVALID_ARG;
  o->inv_freq = r.inv_freq;
  o->positions = r.positions;
  o->ps_axis = r.pos_stride_axis; o->ps_b = r.pos_stride_b; o->ps_l = r.pos_stride_l;
  o->pos_is_64 = r.pos_is_64; o->n_freq = r.n_freq; o->interleaved = r.interleaved;
  o->scale = r.scale;
  for (int i = 0; i < SWA_ROTARY_MAX_FREQS; ++i) o->axis[i] = i < r.n_freq ? r.axis[i] : 0;
  return SWA_OK;
}

// Heads share the blocks of one grid dimension.
bool heads_ok(int64_t q, int64_t kv) { return q + 2 * kv <= 65535; }

bool strides_ok(const SwaTensor& t) { return t.stride_b >= 0 && t.stride_h >= 0 && t.stride_l >= 0; }
bool packed_ok(const SwaPackedTensor& t) { return t.ptr && t.stride_t >= 0 && t.stride_h >= 0; }

int build_cache(const SwaPagedKV& c, swa::PagedParams* o) {
  if (c.batch < 0 || c.n_kv_heads <= 0 || c.n_pages < 0 || c.max_pages < 0 || c.page_size <= 0)
    return SWA_ERR_INVALID_ARG;
  if (c.head_dim <= 0 || c.head_dim > 128) return SWA_ERR_INVALID_ARG;
  if (c.dtype != SWA_F16 && c.dtype != SWA_BF16) return SWA_ERR_UNSUPPORTED;
  if (c.head_dim != 16 && c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) return SWA_ERR_UNSUPPORTED;
  if (c.page_size % 16) return SWA_ERR_UNSUPPORTED;
  if ((int64_t)c.max_pages * c.page_size > INT32_MAX - 1024) return SWA_ERR_UNSUPPORTED;  // slots are 32-bit
  if ((int64_t)c.batch * c.n_kv_heads > INT32_MAX / 1024) return SWA_ERR_UNSUPPORTED;
  const int64_t s[] = {c.k_stride_page, c.k_stride_head, c.k_stride_row, c.v_stride_page, c.v_stride_head,
                       c.v_stride_row};
  for (int64_t x : s)
    if (x < 0 || x % 8) return SWA_ERR_UNSUPPORTED;
  if (c.table_stride < 0 || c.w_stride_b < 0 || c.w_stride_h < 0 || c.p_stride_b < 0 || c.p_stride_h < 0)
    return SWA_ERR_UNSUPPORTED;
  // books are written: no two of their rows may be one
  const auto apart = [&](int64_t b, int64_t h) { return (b > 0 || c.batch <= 1) && (h > 0 || c.n_kv_heads <= 1); };
  if ((c.weights && !apart(c.w_stride_b, c.w_stride_h)) || (c.positions && !apart(c.p_stride_b, c.p_stride_h)))
    return SWA_ERR_INVALID_ARG;
  if (c.batch > 0) {
    // (a pool of no page and a table of no column need no address)
    if ((c.n_pages > 0 && (!c.k || !c.v)) || (c.max_pages > 0 && !c.page_table) || !c.seq_lens)
      return SWA_ERR_INVALID_ARG;
    if (!aligned16(c.k) || !aligned16(c.v)) return SWA_ERR_UNSUPPORTED;
  }
  o->k = c.k; o->v = c.v;
  o->kp = c.k_stride_page; o->kh = c.k_stride_head; o->kr = c.k_stride_row;
  o->vp = c.v_stride_page; o->vh = c.v_stride_head; o->vr = c.v_stride_row;
  o->table = c.page_table; o->table_stride = c.table_stride;
  o->seq_lens = c.seq_lens; o->seen = c.seen ? c.seen : c.seq_lens;
  o->weights = c.weights; o->positions = c.positions;
  o->wb = c.w_stride_b; o->wh = c.w_stride_h; o->pb = c.p_stride_b; o->ph = c.p_stride_h;
  o->n_pages = c.n_pages; o->page_size = c.page_size; o->max_pages = c.max_pages;
  o->batch = c.batch; o->n_kv_heads = c.n_kv_heads;
  o->page_error = nullptr;
  return SWA_OK;
}

int bind_flag(swa::PagedParams* c) {
  c->page_error = swa::page_error_ptr();
  return c->page_error ? SWA_OK : SWA_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int swa_rotary(const SwaRotaryArgs* a, void* stream) {
  if (!a) return SWA_ERR_INVALID_ARG;
  if (a->batch < 0 || a->seq_len < 0 || a->n_q_heads <= 0 || a->n_kv_heads < 0) return SWA_ERR_INVALID_ARG;
  if (a->head_dim <= 0 || a->head_dim > 128 || a->head_dim % 2) return SWA_ERR_INVALID_ARG;
  if (a->dtype != SWA_F16 && a->dtype != SWA_BF16) return SWA_ERR_UNSUPPORTED;
  if ((int64_t)a->batch * a->seq_len > INT32_MAX / 2 || !heads_ok(a->n_q_heads, a->n_kv_heads))
    return SWA_ERR_UNSUPPORTED;
  const bool empty = (int64_t)a->batch * a->seq_len == 0;
  swa::RotaryParams r;
  if (int st = build_rotary(a->r, a->head_dim, !empty, &r)) return st;
  if (empty) return SWA_OK;
  const bool has_k = a->k.ptr && a->n_kv_heads > 0;
  if (!a->q.ptr || !a->q_out.ptr || (has_k && !a->k_out.ptr)) return SWA_ERR_INVALID_ARG;
  if (!strides_ok(a->q) || !strides_ok(a->q_out)) return SWA_ERR_UNSUPPORTED;
  if (has_k && (!strides_ok(a->k) || !strides_ok(a->k_out))) return SWA_ERR_UNSUPPORTED;
  return swa::host_record(swa::launch_rotary(r, *a, static_cast<cudaStream_t>(stream)));
}

int swa_paged_append(const SwaPagedAppendArgs* a, void* stream) {
  if (!a) return SWA_ERR_INVALID_ARG;
  swa::PagedParams c;
  if (int st = build_cache(a->cache, &c)) return st;
  if (a->n_tokens < 0 || a->n_q_heads < 0) return SWA_ERR_INVALID_ARG;
  if (!heads_ok(a->n_q_heads, c.n_kv_heads) || a->n_tokens > INT32_MAX / 2) return SWA_ERR_UNSUPPORTED;
  const bool empty = a->n_tokens == 0 || c.batch == 0;
  swa::RotaryParams r = {};
  if (a->use_rotary)
    if (int st = build_rotary(a->r, a->cache.head_dim, !empty, &r)) return st;
  if (!a->use_rotary && a->n_q_heads) return SWA_ERR_INVALID_ARG;
  if (a->n_tokens > 0 && c.batch == 0) return SWA_ERR_INVALID_ARG;
  if (empty) return SWA_OK;
  if (!a->cu_new && a->n_tokens % c.batch) return SWA_ERR_INVALID_ARG;
  if (!packed_ok(a->k) || !packed_ok(a->v)) return SWA_ERR_INVALID_ARG;
  if (a->n_q_heads && (!packed_ok(a->q) || !packed_ok(a->q_out))) return SWA_ERR_INVALID_ARG;
  if (int st = bind_flag(&c)) return st;
  return swa::host_record(swa::launch_paged_append(c, r, *a, static_cast<cudaStream_t>(stream)));
}

size_t swa_paged_decode_workspace_size(const SwaPagedDecodeArgs* a) {
  swa::PagedParams c;
  if (!a || a->n_q_heads <= 0 || build_cache(a->cache, &c) != SWA_OK || c.batch == 0) return 0;
  if (a->n_q_heads % c.n_kv_heads) return 0;
  return swa::paged_decode_workspace(*a);
}

int swa_paged_decode(const SwaPagedDecodeArgs* a, void* stream) {
  if (!a) return SWA_ERR_INVALID_ARG;
  swa::PagedParams c;
  if (int st = build_cache(a->cache, &c)) return st;
  if (a->n_q_heads <= 0 || a->n_q_heads % c.n_kv_heads || a->sink_size < 0) return SWA_ERR_INVALID_ARG;
  if ((int64_t)c.batch * (a->n_q_heads + 16 * (int64_t)c.n_kv_heads) > INT32_MAX / 64) return SWA_ERR_UNSUPPORTED;
  if (!(a->softmax_scale == a->softmax_scale) || !(a->decay == a->decay)) return SWA_ERR_INVALID_ARG;
  if (c.batch == 0) return SWA_OK;
  if (!packed_ok(a->q) || !packed_ok(a->o)) return SWA_ERR_INVALID_ARG;
  if (!aligned16(a->q.ptr) || a->q.stride_t % 8 || a->q.stride_h % 8) return SWA_ERR_UNSUPPORTED;
  if (!aligned16(a->o.ptr) || a->o.stride_t % 8 || a->o.stride_h % 8) return SWA_ERR_UNSUPPORTED;
  if (a->weights_out) {
    if (a->wo_stride_b < 0 || a->wo_stride_h < 0) return SWA_ERR_UNSUPPORTED;
    if ((a->wo_stride_b == 0 && c.batch > 1) || (a->wo_stride_h == 0 && c.n_kv_heads > 1)) return SWA_ERR_INVALID_ARG;
    // a block per 256 slots of a KV head, in one grid
    if (((int64_t)c.max_pages * c.page_size / 256 + 1) * c.n_kv_heads * c.batch > INT32_MAX / 2) return SWA_ERR_UNSUPPORTED;
  }
  if (int st = check_workspace(a->workspace, a->workspace_bytes, swa_paged_decode_workspace_size(a))) return st;
  if (int st = bind_flag(&c)) return st;
  return swa::host_record(swa::launch_paged_decode(c, *a, static_cast<cudaStream_t>(stream)));
}

size_t swa_paged_evict_workspace_size(const SwaPagedEvictArgs* a) {
  swa::PagedParams c;
  if (!a || a->keep <= 0 || build_cache(a->cache, &c) != SWA_OK || c.batch == 0) return 0;
  return swa::paged_evict_workspace(*a);
}

int swa_paged_evict(const SwaPagedEvictArgs* a, void* stream) {
  if (!a) return SWA_ERR_INVALID_ARG;
  swa::PagedParams c;
  if (int st = build_cache(a->cache, &c)) return st;
  if (a->keep <= 0 || a->trigger < 0 || a->sink_size < 0 || a->recent < 0) return SWA_ERR_INVALID_ARG;
  if ((int64_t)a->sink_size + a->recent > a->keep) return SWA_ERR_INVALID_ARG;
  if (c.batch == 0) return SWA_OK;
  if (!c.weights || !c.positions) return SWA_ERR_INVALID_ARG;
  // nothing can be longer than the budget
  if (a->keep >= (int64_t)c.max_pages * c.page_size) return SWA_OK;
  if (int st = check_workspace(a->workspace, a->workspace_bytes, swa_paged_evict_workspace_size(a))) return st;
  // token numbers go by a count that evictions do not shorten
  if (!a->cache.seen || a->cache.seen == a->cache.seq_lens) return SWA_ERR_INVALID_ARG;
  if (int st = bind_flag(&c)) return st;
  return swa::host_record(swa::launch_paged_evict(c, *a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
