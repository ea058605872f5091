// swa_paged_decode.cu -- attention of one new token per sequence over its paged cache.
//
// o[b, h] = softmax([scale q k_j (visible j), sink_h]) v.  One block per (query head, sequence):
// each warp walks every fourth visible slot with a running maximum and sum, the four are joined
// at the end.
#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
namespace {

constexpr int kThreads = 128;

struct DecodeParams {
  PagedParams c;
  int Hq, W, S, D;
  float scale_log2;
  const void* q; void* o;
  int64_t qb, qh, ob, oh;
  float* lse;
  const float* sinks;
  float* wout;
  int64_t wob, woh;
  float decay;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) decode_kernel(DecodeParams p) {
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int hk = h / (p.Hq / p.c.n_kv_heads), D = p.D;
  const T* q = static_cast<const T*>(p.q) + b * p.qb + h * p.qh;
  bool bad = false;
  const int n = paged_len(p.c, b, &bad);
  const VisibleSlots vis = visible_slots(n, p.W, p.S);
  const int total = vis.sinks + n - vis.first;
  float m = -INFINITY, l = 0.f, acc[4] = {};
  for (int u = warp; u < total; u += kThreads / 32) {
    const int slot = u < vis.sinks ? u : u - vis.sinks + vis.first;
    const int page = paged_page(p.c, b, slot / p.c.page_size, &bad);
    if (page < 0) continue;
    const int row = slot % p.c.page_size;
    const T* k = static_cast<const T*>(p.c.k) + page * p.c.kp + hk * p.c.kh + row * p.c.kr;
    const T* v = static_cast<const T*>(p.c.v) + page * p.c.vp + hk * p.c.vh + row * p.c.vr;
    float s = 0.f;
    for (int d = lane; d < D; d += 32) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s), f = m == mn ? 1.f : exp2f(m - mn), e = mn == -INFINITY ? 0.f : exp2f(s - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < D) acc[i] = acc[i] * f + e * to_f32(v[lane + 32 * i]);
  }
  __shared__ float sm[4], sl[4], sa[4][128];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int i = 0; i < 4; ++i) sa[warp][lane + 32 * i] = acc[i];
  bad = __syncthreads_or(bad);
  const float sink = p.sinks ? p.sinks[h] * kLog2e : -INFINITY;
  float mm = sink;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w]);
  const float base = mm == -INFINITY ? 0.f : mm;
  float ll = exp2f(sink - base), oo = 0.f;
  const int d = threadIdx.x;
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(sm[w] - base);
    ll += sl[w] * f;
    oo += sa[w][d] * f;
  }
  if (bad) {
    ll = NAN;
    if (d == 0) *p.c.page_error = 1;
  }
  if (d < D) static_cast<T*>(p.o)[b * p.ob + h * p.oh + d] = from_f32<T>(ll == 0.f ? 0.f : oo / ll);
  if (d == 0) p.lse[(int64_t)b * p.Hq + h] = ll == 0.f ? -INFINITY : mm + log2f(ll);
}

// weights_out = decay * weights + the group's softmax weights, from the finished lse.
template <typename T>
__global__ void __launch_bounds__(kThreads) weights_kernel(DecodeParams p) {
  const int hk = blockIdx.y, b = blockIdx.z, G = p.Hq / p.c.n_kv_heads;
  bool bad = false;
  const int n = paged_len(p.c, b, &bad);
  const VisibleSlots vis = visible_slots(n, p.W, p.S);
  const int slot = blockIdx.x * kThreads + threadIdx.x;
  if (slot >= n) return;
  float w = p.c.weights ? p.decay * p.c.weights[b * p.c.wb + hk * p.c.wh + slot] : 0.f;
  if (slot < vis.sinks || slot >= vis.first) {
    const int page = paged_page(p.c, b, slot / p.c.page_size, &bad);
    if (page >= 0) {
      const T* k = static_cast<const T*>(p.c.k) + page * p.c.kp + hk * p.c.kh + slot % p.c.page_size * p.c.kr;
      for (int g = 0; g < G; ++g) {
        const int h = hk * G + g;
        const T* q = static_cast<const T*>(p.q) + b * p.qb + h * p.qh;
        float s = 0.f;
        for (int d = 0; d < p.D; ++d) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
        w += exp2f(s * p.scale_log2 - p.lse[(int64_t)b * p.Hq + h]);
      }
    }
  }
  p.wout[b * p.wob + hk * p.woh + slot] = w;
}

}  // namespace

size_t paged_decode_workspace(const SwaPagedDecodeArgs& a) {
  return ((size_t)a.cache.batch * a.n_q_heads * sizeof(float) + 255) & ~(size_t)255;
}

template <typename T>
static cudaError_t launch(const DecodeParams& p, cudaStream_t st) {
  decode_kernel<T><<<dim3(p.Hq, p.c.batch), kThreads, 0, st>>>(p);
  if (p.wout) {
    const int cap = p.c.max_pages * p.c.page_size;
    weights_kernel<T><<<dim3((cap + kThreads - 1) / kThreads, p.c.n_kv_heads, p.c.batch), kThreads, 0, st>>>(p);
  }
  return cudaGetLastError();
}

cudaError_t launch_paged_decode(const PagedParams& c, const SwaPagedDecodeArgs& a, cudaStream_t st) {
  DecodeParams p;
  p.c = c;
  p.Hq = a.n_q_heads; p.W = a.window_size; p.S = a.sink_size; p.D = a.cache.head_dim;
  p.scale_log2 = a.softmax_scale * kLog2e;
  p.q = a.q.ptr; p.o = a.o.ptr;
  p.qb = a.q.stride_t; p.qh = a.q.stride_h; p.ob = a.o.stride_t; p.oh = a.o.stride_h;
  p.lse = a.lse ? a.lse : static_cast<float*>(a.workspace);
  p.sinks = a.sink_logits;
  p.wout = a.weights_out; p.wob = a.wo_stride_b; p.woh = a.wo_stride_h;
  p.decay = a.decay;
  return a.cache.dtype == SWA_F16 ? launch<__half>(p, st) : launch<__nv_bfloat16>(p, st);
}

}  // namespace swa
