// swa_rotary.cu -- rotary positions with several axes, and the append of rotated keys (and of
// values) to a paged cache.
//
// Frequency i of n turns one pair of values of each head by theta_i = position[axis_i] *
// inv_freq_i: (x, y) -> scale (x cos - y sin, y cos + x sin), the pair being (i, n + i) or, when
// interleaved, (2 i, 2 i + 1).  The map is linear, so its gradient is the same with -theta.
//
// Bound by the bytes of q, k (and v): read once, written once.  A block takes a few tokens and a
// range of heads.  It first forms the tokens' cos and sin, once for all of its heads, in shared
// memory; then a thread stays with one token and two pieces of a head (those that hold both ends
// of its pairs), keeps their cos and sin in registers, and walks over heads.  A piece is 16 bytes
// where sizes, strides and addresses allow it, else 4 or 2.  A thread has read all of a row that it
// writes, so outputs may lie on their inputs.
//
// Measured on a B200 (6.56 TB/s copy): q and k of the GPT-OSS layer (4 x 72 heads x 4096 x 64, 302
// MB moved) 50 us, 6.0 TB/s; 8 x 36 heads x 3000 x 128 (443 MB) 73 us, 6.1 TB/s; 14004 packed
// prompt tokens into pages (288 MB) 54 us, 5.3 TB/s; 64 single tokens 4 us.
#include "sm100.cuh"
#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
namespace {

constexpr int kThreads = 256;
// 8 tokens share a block and its angles: at the GPT-OSS layer 4 took 61 us, 8 54, 16 55, 32 57, and a
// prompt of 512 tokens 7.3 us with 4, 6.4 with 8 (5.4 with fewer blocks)
constexpr int kMaxTokens = 8;
// heads whose loads a thread has under way, and blocks an SM (64 registers a thread): 1 and 6 take
// 63 us, 2 and 4 54, 3 and 3 56, 4 and 3 54 (50 with the first rows called for before the angles)
constexpr int kHeadsAhead = 2;
constexpr int kBlocksPerSm = 4;
constexpr int kSmemSeqs = 1024;  // sequences whose offsets are searched in shared memory

struct Rows {
  const void* in;
  void* out;
  Strides si, so;
};

struct RowsParams {
  RotaryParams r;
  Rows q, k, v;  // v: append alone
  int tokens, L, Hq, Hk, D, copy_v;
  int tok, lanes, heads_par, heads_block;  // tokens, threads per row, rows at a time, heads of a block
  float sign;
  // append
  PagedParams c;
  const int32_t* cu;
};

template <int V> struct PieceOf;
template <> struct PieceOf<8> { using type = uint4; };
template <> struct PieceOf<2> { using type = uint32_t; };
template <> struct PieceOf<1> { using type = uint16_t; };

// Two neighbouring values as a 32-bit word.
__device__ __forceinline__ float2 unpack(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 unpack(uint32_t w, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// Rotates a thread's two pieces: across them, or, with `self`, pairs inside each of them (the
// second only where `both`: it may lie behind the values that turn).
template <typename T, int V>
__device__ __forceinline__ void turn(typename PieceOf<V>::type* a, typename PieceOf<V>::type* b, const float* c,
                                     const float* s, bool self, bool both) {
  if constexpr (V == 1) {
    T* x = reinterpret_cast<T*>(a);
    T* y = reinterpret_cast<T*>(b);
    const float u = Pack<T>::to(*x), w = Pack<T>::to(*y);
    *x = Pack<T>::from(fmaf(u, c[0], -w * s[0]));
    *y = Pack<T>::from(fmaf(w, c[0], u * s[0]));
  } else {
    uint32_t* x = reinterpret_cast<uint32_t*>(a);
    uint32_t* y = reinterpret_cast<uint32_t*>(b);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 u = unpack(x[j], T()), w = unpack(y[j], T());
      if (self) {
        x[j] = Pack<T>::pack(fmaf(u.x, c[j], -u.y * s[j]), fmaf(u.y, c[j], u.x * s[j]));
        if (both) {
          const float e = c[V / 2 + j], f = s[V / 2 + j];
          y[j] = Pack<T>::pack(fmaf(w.x, e, -w.y * f), fmaf(w.y, e, w.x * f));
        }
      } else {
        x[j] = Pack<T>::pack(fmaf(u.x, c[2 * j], -w.x * s[2 * j]), fmaf(u.y, c[2 * j + 1], -w.y * s[2 * j + 1]));
        y[j] = Pack<T>::pack(fmaf(w.x, c[2 * j], u.x * s[2 * j]), fmaf(w.y, c[2 * j + 1], u.y * s[2 * j + 1]));
      }
    }
  }
}

template <typename T, int V, bool APPEND>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) rows_kernel(const __grid_constant__ RowsParams p) {
  using Piece = typename PieceOf<V>::type;
  __shared__ float2 turns[kMaxTokens][SWA_ROTARY_MAX_FREQS];
  __shared__ int seq[kMaxTokens], slot[kMaxTokens], page[kMaxTokens], number[kMaxTokens];
  __shared__ int32_t cu_copy[APPEND ? kSmemSeqs + 1 : 1];
  const int n = p.r.n_freq, t0 = blockIdx.x * p.tok;
  const int count = p.tokens - t0 < p.tok ? p.tokens - t0 : p.tok;
  const int heads0 = blockIdx.y * p.heads_block;
  const int lane = threadIdx.x % p.lanes, tt = threadIdx.x / p.lanes % p.tok;
  const int first = threadIdx.x / (p.lanes * p.tok), t = t0 + tt;
  const int64_t b = APPEND ? 0 : t / p.L, l = APPEND ? t : t % p.L;
  const bool works = first < p.heads_par && tt < count;
  // this thread's two pieces (element offsets) and whether they turn
  const bool self = V > 1 && p.r.interleaved, turned = lane * V < (self ? 2 * n : n);
  int x, y;
  if (self) {
    x = lane * V;
    y = x + p.lanes * V;
  } else {
    x = turned ? (V == 1 && p.r.interleaved ? 2 * lane : lane * V) : 2 * lane * V;
    y = turned ? (V == 1 && p.r.interleaved ? x + 1 : x + n) : x + V;
  }
  sm100::pdl_wait();
  // the first rows come while the angles are formed: 50 us for the layer, 52.5 without
  if (works) {
    const int to = heads0 + p.heads_block < p.Hq ? heads0 + p.heads_block : p.Hq;
#pragma unroll
    for (int i = 0; i < kHeadsAhead; ++i) {
      const int h = heads0 + first + i * p.heads_par;
      if (h < to) {
        const T* in = static_cast<const T*>(p.q.in) + b * p.q.si.b + l * p.q.si.l + h * p.q.si.h;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(in + x));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(in + y));
      }
    }
  }

  if constexpr (APPEND) {
    const int32_t* cu = p.cu;
    if (cu && p.c.batch <= kSmemSeqs) {
      for (int i = threadIdx.x; i <= p.c.batch; i += kThreads) cu_copy[i] = cu[i];
      __syncthreads();
      cu = cu_copy;
    }
    if ((int)threadIdx.x < count) {
      const int t = t0 + threadIdx.x;
      int b, start, end;
      if (cu) {
        int lo = 0, hi = p.c.batch - 1;  // the last sequence that starts at or before t
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (cu[mid] <= t) lo = mid; else hi = mid - 1;
        }
        b = lo; start = cu[b]; end = cu[b + 1];
      } else {
        const int m = p.tokens / p.c.batch;
        b = t / m; start = b * m; end = start + m;
      }
      bool bad = t < start || t >= end;
      const int s = paged_len(p.c, b, &bad) - (end - t);
      bad |= s < 0;
      const int g = bad ? -1 : paged_page(p.c, b, s / p.c.page_size, &bad);
      if (bad) *p.c.page_error = 1;
      seq[threadIdx.x] = b;
      slot[threadIdx.x] = s;
      page[threadIdx.x] = g;
      number[threadIdx.x] = p.c.seen[b] - (end - t);
    }
  }
  for (int e = threadIdx.x; e < count * n; e += kThreads) {
    const int t = e / n, i = e % n, at = t0 + t;
    float c, s;
    rotary_cos_sin(p.r, APPEND ? 0 : at / p.L, APPEND ? at : at % p.L, i, &c, &s);
    turns[t][i] = make_float2(c, s * p.sign);
  }
  __syncthreads();

  if (!works) return;
  float c[V], s[V];
  if (self) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 u = x < 2 * n ? turns[tt][x / 2 + j] : make_float2(0.f, 0.f);
      const float2 w = y < 2 * n ? turns[tt][y / 2 + j] : make_float2(0.f, 0.f);
      c[j] = u.x; s[j] = u.y; c[V / 2 + j] = w.x; s[V / 2 + j] = w.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 u = turned ? turns[tt][lane * V + j] : make_float2(0.f, 0.f);
      c[j] = u.x; s[j] = u.y;
    }
  }
  const int heads = p.Hq + p.Hk + (APPEND ? p.Hk : 0);
  const int end = heads0 + p.heads_block < heads ? heads0 + p.heads_block : heads;

  // heads [from, to) of the block's range that belong to one tensor, whose head 0 is `base`
  auto walk = [&](const void* in0, void* out0, int64_t in_row, int64_t out_row, int64_t in_head, int64_t out_head, int base,
                  int count_heads, bool turns_here) {
    const int from = heads0 > base ? heads0 : base, to = end < base + count_heads ? end : base + count_heads;
    int h = from + first;
    const T* in = static_cast<const T*>(in0) + in_row + (int64_t)(h - base) * in_head;
    T* out = static_cast<T*>(out0) + out_row + (int64_t)(h - base) * out_head;
    const int64_t in_step = in_head * p.heads_par, out_step = out_head * p.heads_par;
    while (h < to) {
      Piece a[kHeadsAhead], z[kHeadsAhead];
#pragma unroll
      for (int i = 0; i < kHeadsAhead; ++i)
        if (h + i * p.heads_par < to) {
          a[i] = *reinterpret_cast<const Piece*>(in + x);
          z[i] = *reinterpret_cast<const Piece*>(in + y);
          in += in_step;
        }
#pragma unroll
      for (int i = 0; i < kHeadsAhead; ++i)
        if (h + i * p.heads_par < to) {
          if (turns_here) turn<T, V>(&a[i], &z[i], c, s, self, y < 2 * n);
          *reinterpret_cast<Piece*>(out + x) = a[i];
          *reinterpret_cast<Piece*>(out + y) = z[i];
          out += out_step;
        }
      h += kHeadsAhead * p.heads_par;
    }
  };
  walk(p.q.in, p.q.out, b * p.q.si.b + l * p.q.si.l, b * p.q.so.b + l * p.q.so.l, p.q.si.h, p.q.so.h, 0, p.Hq, turned);
  if constexpr (!APPEND) {
    walk(p.k.in, p.k.out, b * p.k.si.b + l * p.k.si.l, b * p.k.so.b + l * p.k.so.l, p.k.si.h, p.k.so.h, p.Hq, p.Hk, turned);
  } else if (page[tt] >= 0) {
    const int64_t g = page[tt], row = slot[tt] % p.c.page_size;
    walk(p.k.in, p.c.k, l * p.k.si.l, g * p.c.kp + row * p.c.kr, p.k.si.h, p.c.kh, p.Hq, p.Hk, turned);
    walk(p.v.in, p.c.v, l * p.v.si.l, g * p.c.vp + row * p.c.vr, p.v.si.h, p.c.vh, p.Hq + p.Hk, p.Hk, false);
    // weights and token numbers, by the threads with the rows of k
    if (lane == 0 && (p.c.weights || p.c.positions))
      for (int h = (heads0 > p.Hq ? heads0 : p.Hq) + first; h < end && h < p.Hq + p.Hk; h += p.heads_par) {
        const int hk = h - p.Hq;
        if (p.c.weights) p.c.weights[seq[tt] * p.c.wb + hk * p.c.wh + slot[tt]] = 0.f;
        if (p.c.positions) p.c.positions[seq[tt] * p.c.pb + hk * p.c.ph + slot[tt]] = number[tt];
      }
  }
}

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int v) {
  return reinterpret_cast<uintptr_t>(p) % (2 * v) == 0 && a % v == 0 && b % v == 0 && c % v == 0;
}
bool aligned(const Rows& r, int v) {
  return aligned(r.in, r.si.b, r.si.h, r.si.l, v) && aligned(r.out, r.so.b, r.so.h, r.so.l, v);
}

// The widest piece that sizes, strides and addresses allow: 8, 2 or 1 values.
int piece(const RowsParams& p) {
  const int widths[] = {8, 2};
  for (int v : widths) {
    const bool fits = p.D % (2 * v) == 0 && (p.r.interleaved ? 2 * p.r.n_freq : p.r.n_freq) % v == 0;
    if (fits && aligned(p.q, v) && (!p.Hk || aligned(p.k, v)) && (!p.copy_v || aligned(p.v, v))) return v;
  }
  return 1;
}

template <typename T, int V, bool APPEND> cudaError_t launch(RowsParams p, cudaStream_t st) {
  p.lanes = p.D / (2 * V);
  const int heads = p.Hq + p.Hk + (APPEND ? p.Hk : 0);
  p.tok = kMaxTokens;
  while (p.tok > 1 && (p.tok * p.lanes > kThreads || p.tok / 2 >= p.tokens)) p.tok /= 2;
  p.heads_par = kThreads / (p.tok * p.lanes);
  const int64_t x = (p.tokens + p.tok - 1) / p.tok;
  // heads are divided among blocks until every SM has one, no further: each block forms its tokens'
  // angles anew (a prompt of 1024 tokens: 6.1 us so, 9.9 with eight blocks an SM)
  int64_t groups = (148 + x - 1) / x;
  const int64_t most = (heads + p.heads_par - 1) / p.heads_par;
  if (groups > most) groups = most;
  if (groups < 1) groups = 1;
  p.heads_block = (int)((heads + groups - 1) / groups);
  const int y = (heads + p.heads_block - 1) / p.heads_block;
  return launch_pdl(rows_kernel<T, V, APPEND>, dim3((unsigned)x, (unsigned)y), kThreads, 0, st, p);
}

template <bool APPEND> cudaError_t launch(const RowsParams& p, int dtype, cudaStream_t st) {
  const int v = piece(p);
  if (dtype == SWA_F16)
    return v == 8 ? launch<__half, 8, APPEND>(p, st) : v == 2 ? launch<__half, 2, APPEND>(p, st) : launch<__half, 1, APPEND>(p, st);
  return v == 8   ? launch<__nv_bfloat16, 8, APPEND>(p, st)
         : v == 2 ? launch<__nv_bfloat16, 2, APPEND>(p, st)
                  : launch<__nv_bfloat16, 1, APPEND>(p, st);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& r, const SwaRotaryArgs& a, cudaStream_t st) {
  RowsParams p = {};
  p.r = r;
  p.q = {a.q.ptr, a.q_out.ptr, {a.q.stride_b, a.q.stride_h, a.q.stride_l},
         {a.q_out.stride_b, a.q_out.stride_h, a.q_out.stride_l}};
  p.Hk = a.k.ptr ? a.n_kv_heads : 0;
  if (p.Hk)
    p.k = {a.k.ptr, a.k_out.ptr, {a.k.stride_b, a.k.stride_h, a.k.stride_l},
           {a.k_out.stride_b, a.k_out.stride_h, a.k_out.stride_l}};
  p.tokens = a.batch * a.seq_len; p.L = a.seq_len; p.Hq = a.n_q_heads; p.D = a.head_dim;
  p.sign = a.inverse ? -1.f : 1.f;
  return launch<false>(p, a.dtype, st);
}

cudaError_t launch_paged_append(const PagedParams& c, const RotaryParams& r, const SwaPagedAppendArgs& a,
                                cudaStream_t st) {
  RowsParams p = {};
  p.r = r;
  if (!a.use_rotary) p.r.n_freq = 0;
  p.q = {a.q.ptr, a.q_out.ptr, {0, a.q.stride_h, a.q.stride_t}, {0, a.q_out.stride_h, a.q_out.stride_t}};
  // the pages' rows are 16-byte aligned
  p.k = {a.k.ptr, c.k, {0, a.k.stride_h, a.k.stride_t}, {}};
  p.v = {a.v.ptr, c.v, {0, a.v.stride_h, a.v.stride_t}, {}};
  p.copy_v = 1;
  p.tokens = a.n_tokens; p.L = a.n_tokens; p.Hq = a.n_q_heads; p.Hk = c.n_kv_heads; p.D = a.cache.head_dim;
  p.sign = 1.f;
  p.c = c;
  p.cu = a.cu_new;
  return launch<true>(p, a.cache.dtype, st);
}

}  // namespace swa
