// swa_paged_evict.cu -- cuts the sequences of a paged cache down to a budget by the weight that
// attention has laid on each slot.
//
// One block per (KV head, sequence).  Each slot has a 32-bit key: held tokens the largest, then
// the weights in order.  The budget-th largest key is found bit by bit; slots above it are kept,
// of those equal to it the lowest.  Slots that come free below the budget and kept slots behind
// it are numbered in order, and the i-th of the one takes the i-th of the other.
#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
namespace {

constexpr int kThreads = 1024;

struct EvictParams {
  PagedParams c;
  int keep, trigger, sink, recent, row_bytes;
  int32_t* lists;  // [batch, Hkv, 2, keep]: free slots, then the slots that fill them
};

// Order-preserving map of a weight to [0x007fffff, 0xff800000]: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.f) w = 0.f;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t slot_key(const EvictParams& p, int b, int h, int slot) {
  const int pos = p.c.positions[b * p.c.pb + h * p.c.ph + slot];
  if (pos < p.sink || pos >= (int64_t)p.c.seen[b] - p.recent) return 0xffffffffu;
  return weight_key(p.c.weights[b * p.c.wb + h * p.c.wh + slot]);
}

// Exclusive rank of this thread among the threads whose flag is set, and their number.
__device__ __forceinline__ int block_rank(bool flag, int* total) {
  __shared__ int warp_count[kThreads / 32];
  const unsigned vote = __ballot_sync(~0u, flag);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  __syncthreads();
  if (lane == 0) warp_count[warp] = __popc(vote);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_count[w];
    all += warp_count[w];
  }
  *total = all;
  return before + __popc(vote & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictParams p) {
  const int h = blockIdx.x, b = blockIdx.y;
  bool bad = false;
  const int n = paged_len(p.c, b, &bad);
  if (bad && threadIdx.x == 0) *p.c.page_error = 1;
  if (bad || n <= p.keep || n <= p.trigger) return;
  // the largest key that at least `keep` slots reach
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t probe = t | (1u << bit);
    int count = 0;
    for (int s = threadIdx.x; s < n; s += kThreads) count += slot_key(p, b, h, s) >= probe;
    for (int x = 16; x; x >>= 1) count += __shfl_xor_sync(~0u, count, x);
    __shared__ int sum[kThreads / 32];
    __syncthreads();
    if (threadIdx.x % 32 == 0) sum[threadIdx.x / 32] = count;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kThreads / 32; ++w) all += sum[w];
    if (all >= p.keep) t = probe;
  }
  int above = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int s = base + threadIdx.x;
    int all;
    block_rank(s < n && slot_key(p, b, h, s) > t, &all);
    above += all;
  }
  const int room = p.keep - above;
  int32_t* free_list = p.lists + (int64_t)(b * p.c.n_kv_heads + h) * 2 * p.keep;
  int32_t* move_list = free_list + p.keep;
  int equal = 0, n_free = 0, n_move = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int s = base + threadIdx.x;
    const uint32_t key = s < n ? slot_key(p, b, h, s) : 0u;
    int all;
    const int nth = equal + block_rank(s < n && key == t, &all);
    equal += all;
    const bool kept = s < n && (key > t || (key == t && nth < room));
    const bool is_free = s < p.keep && !kept, is_move = kept && s >= p.keep;
    int at = n_free + block_rank(is_free, &all);
    n_free += all;
    if (is_free) free_list[at] = s;
    at = n_move + block_rank(is_move, &all);
    n_move += all;
    if (is_move) move_list[at] = s;
  }
  __syncthreads();
  // 16 bytes a thread, K and V
  const int per_row = p.row_bytes / 16;
  for (int64_t e = threadIdx.x; e < (int64_t)n_move * per_row; e += kThreads) {
    const int i = (int)(e / per_row), part = (int)(e % per_row);
    const int to = free_list[i], from = move_list[i];
    const int pt = paged_page(p.c, b, to / p.c.page_size, &bad), pf = paged_page(p.c, b, from / p.c.page_size, &bad);
    if (pt >= 0 && pf >= 0) {
      char* k = static_cast<char*>(p.c.k) + 2 * h * p.c.kh + 16 * part;
      char* v = static_cast<char*>(p.c.v) + 2 * h * p.c.vh + 16 * part;
      const int rt = to % p.c.page_size, rf = from % p.c.page_size;
      *reinterpret_cast<uint4*>(k + 2 * (pt * p.c.kp + rt * p.c.kr)) =
          *reinterpret_cast<const uint4*>(k + 2 * (pf * p.c.kp + rf * p.c.kr));
      *reinterpret_cast<uint4*>(v + 2 * (pt * p.c.vp + rt * p.c.vr)) =
          *reinterpret_cast<const uint4*>(v + 2 * (pf * p.c.vp + rf * p.c.vr));
    }
    if (part == 0) {
      float* w = p.c.weights + b * p.c.wb + h * p.c.wh;
      int32_t* x = p.c.positions + b * p.c.pb + h * p.c.ph;
      w[to] = w[from];
      x[to] = x[from];
    }
  }
  if (bad) *p.c.page_error = 1;
}

__global__ void evict_lens_kernel(EvictParams p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.c.batch) return;
  bool bad = false;
  const int n = paged_len(p.c, b, &bad);
  if (!bad && n > p.keep && n > p.trigger) p.c.seq_lens[b] = p.keep;
}

}  // namespace

size_t paged_evict_workspace(const SwaPagedEvictArgs& a) {
  return ((size_t)a.cache.batch * a.cache.n_kv_heads * 2 * a.keep * sizeof(int32_t) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_evict(const PagedParams& c, const SwaPagedEvictArgs& a, cudaStream_t st) {
  EvictParams p;
  p.c = c;
  p.keep = a.keep; p.trigger = a.trigger; p.sink = a.sink_size; p.recent = a.recent;
  p.row_bytes = 2 * a.cache.head_dim;
  p.lists = static_cast<int32_t*>(a.workspace);
  evict_kernel<<<dim3(c.n_kv_heads, c.batch), kThreads, 0, st>>>(p);
  evict_lens_kernel<<<(c.batch + 127) / 128, 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace swa
