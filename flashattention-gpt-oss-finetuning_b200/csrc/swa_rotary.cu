// swa_rotary.cu -- rotary positions with several axes, and the append of rotated keys (and of
// values) to a paged cache.
//
// Frequency i of n turns one pair of values of each head by theta_i = position[axis_i] *
// inv_freq_i: (x, y) -> scale (x cos - y sin, y cos + x sin), the pair being (i, n + i) or, when
// interleaved, (2 i, 2 i + 1).  The map is linear, so its gradient is the same with -theta.
#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
namespace {

constexpr int kThreads = 256;

// One value of a rotated row: d < 2 n_freq from its pair, the others copied.
template <typename T>
__device__ __forceinline__ T rotated(const RotaryParams& r, const T* row, int d, int64_t b, int64_t l, float sign) {
  const int n = r.n_freq;
  if (d >= 2 * n) return row[d];
  int i, x, y;
  bool second;
  if (r.interleaved) {
    i = d >> 1; second = d & 1; x = 2 * i; y = x + 1;
  } else {
    second = d >= n; i = second ? d - n : d; x = i; y = i + n;
  }
  float c, s;
  rotary_cos_sin(r, b, l, i, &c, &s);
  s *= sign;
  const float fx = to_f32(row[x]), fy = to_f32(row[y]);
  return from_f32<T>(second ? fmaf(fy, c, fx * s) : fmaf(fx, c, -fy * s));
}

struct RotaryTensors {
  const void* in;
  void* out;
  Strides si, so;
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(RotaryParams r, RotaryTensors q, RotaryTensors k, int B, int Hq, int Hkv, int L, int D, float sign) {
  // a pair per thread, so that outputs may lie over their inputs; copied values count in pairs too
  const int64_t n = (int64_t)B * L * (Hq + Hkv) * (D / 2);
  for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < n; at += (int64_t)gridDim.x * kThreads) {
    const int p = (int)(at % (D / 2));
    int64_t rest = at / (D / 2);
    const int l = (int)(rest % L);
    rest /= L;
    int h = (int)(rest % (Hq + Hkv));
    const int b = (int)(rest / (Hq + Hkv));
    const bool is_q = h < Hq;
    if (!is_q) h -= Hq;
    const RotaryTensors& t = is_q ? q : k;
    const T* in = static_cast<const T*>(t.in) + b * t.si.b + h * t.si.h + l * t.si.l;
    T* out = static_cast<T*>(t.out) + b * t.so.b + h * t.so.h + l * t.so.l;
    int x = 2 * p, y = x + 1;
    if (!r.interleaved && p < r.n_freq) {
      x = p;
      y = p + r.n_freq;
    }
    const T a = rotated(r, in, x, b, l, sign), c = rotated(r, in, y, b, l, sign);
    out[x] = a;
    out[y] = c;
  }
}

struct AppendParams {
  PagedParams c;
  RotaryParams r;
  const int32_t* cu;
  int n_tokens, Hq, D, use_rotary;
  const void* k; const void* v; const void* q; void* qo;
  int64_t kt, kh, vt, vh, qt, qh, ot, oh;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendParams p) {
  const int t = blockIdx.x;
  int b, start, end;
  if (p.cu) {
    int lo = 0, hi = p.c.batch - 1;  // the last sequence that starts at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    b = lo; start = p.cu[b]; end = p.cu[b + 1];
  } else {
    const int m = p.n_tokens / p.c.batch;
    b = t / m; start = b * m; end = start + m;
  }
  const int D = p.D, Hkv = p.c.n_kv_heads;
  for (int e = threadIdx.x; e < p.Hq * D; e += kThreads) {
    const int h = e / D, d = e % D;
    const T* row = static_cast<const T*>(p.q) + t * p.qt + h * p.qh;
    static_cast<T*>(p.qo)[t * p.ot + h * p.oh + d] = rotated(p.r, row, d, 0, t, 1.f);
  }
  bool bad = false;
  paged_len(p.c, b, &bad);
  const int slot = p.c.seq_lens[b] - (end - t);
  int page = -1;
  if (t < start || t >= end || slot < 0 || bad) bad = true;
  else page = paged_page(p.c, b, slot / p.c.page_size, &bad);
  if (bad) {
    if (threadIdx.x == 0) *p.c.page_error = 1;
    return;
  }
  const int row = slot % p.c.page_size;
  for (int e = threadIdx.x; e < Hkv * D; e += kThreads) {
    const int h = e / D, d = e % D;
    const T* kin = static_cast<const T*>(p.k) + t * p.kt + h * p.kh;
    const T* vin = static_cast<const T*>(p.v) + t * p.vt + h * p.vh;
    T* ko = static_cast<T*>(p.c.k) + page * p.c.kp + h * p.c.kh + row * p.c.kr;
    T* vo = static_cast<T*>(p.c.v) + page * p.c.vp + h * p.c.vh + row * p.c.vr;
    ko[d] = p.use_rotary ? rotated(p.r, kin, d, 0, t, 1.f) : kin[d];
    vo[d] = vin[d];
  }
  for (int h = threadIdx.x; h < Hkv; h += kThreads) {
    if (p.c.weights) p.c.weights[b * p.c.wb + h * p.c.wh + slot] = 0.f;
    if (p.c.positions) p.c.positions[b * p.c.pb + h * p.c.ph + slot] = p.c.seen[b] - (end - t);
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& r, const SwaRotaryArgs& a, cudaStream_t st) {
  const RotaryTensors q = {a.q.ptr, a.q_out.ptr, {a.q.stride_b, a.q.stride_h, a.q.stride_l},
                           {a.q_out.stride_b, a.q_out.stride_h, a.q_out.stride_l}};
  const RotaryTensors k = {a.k.ptr, a.k_out.ptr, {a.k.stride_b, a.k.stride_h, a.k.stride_l},
                           {a.k_out.stride_b, a.k_out.stride_h, a.k_out.stride_l}};
  const int hkv = a.k.ptr ? a.n_kv_heads : 0;
  const int64_t n = (int64_t)a.batch * a.seq_len * (a.n_q_heads + hkv) * (a.head_dim / 2);
  const int64_t blocks = (n + kThreads - 1) / kThreads;
  const int grid = (int)(blocks < 148 * 64 ? blocks : 148 * 64);
  const float sign = a.inverse ? -1.f : 1.f;
  if (a.dtype == SWA_F16)
    rotary_kernel<__half><<<grid, kThreads, 0, st>>>(r, q, k, a.batch, a.n_q_heads, hkv, a.seq_len, a.head_dim, sign);
  else
    rotary_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(r, q, k, a.batch, a.n_q_heads, hkv, a.seq_len, a.head_dim,
                                                           sign);
  return cudaGetLastError();
}

cudaError_t launch_paged_append(const PagedParams& c, const RotaryParams& r, const SwaPagedAppendArgs& a,
                                cudaStream_t st) {
  AppendParams p;
  p.c = c;
  p.r = r;
  p.cu = a.cu_new;
  p.n_tokens = a.n_tokens; p.Hq = a.n_q_heads; p.D = a.cache.head_dim; p.use_rotary = a.use_rotary;
  p.k = a.k.ptr; p.v = a.v.ptr; p.q = a.q.ptr; p.qo = a.q_out.ptr;
  p.kt = a.k.stride_t; p.kh = a.k.stride_h; p.vt = a.v.stride_t; p.vh = a.v.stride_h;
  p.qt = a.q.stride_t; p.qh = a.q.stride_h; p.ot = a.q_out.stride_t; p.oh = a.q_out.stride_h;
  if (a.cache.dtype == SWA_F16) append_kernel<__half><<<a.n_tokens, kThreads, 0, st>>>(p);
  else append_kernel<__nv_bfloat16><<<a.n_tokens, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace swa
