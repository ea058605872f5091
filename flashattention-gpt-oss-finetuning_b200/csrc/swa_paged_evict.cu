// swa_paged_evict.cu -- cuts the sequences of a paged cache down to a budget by the weight that
// attention has laid on each slot.
//
// Each slot has a 32-bit key: held tokens the largest, then the weights in order.  The budget-th
// largest key t is found digit by digit (11, 11 and 10 bits) from histograms; slots above t are
// kept, and of those equal to t the lowest.  Slots that come free below the budget and kept slots
// behind it are numbered in order, and the i-th of the one takes the i-th of the other: no row is
// both read and written, so all of them move at once, and only as many as have to.
//
// A (sequence, KV head) belongs to a cluster of 1 to 8 blocks, each with a stretch of the slots,
// whose keys it keeps in shared memory: the weights and token numbers are read once (8 bytes a slot).
// Histograms and counts of the other blocks are read through distributed shared memory, one
// cluster barrier a digit.  What bounds it: the dependent steps (load, three digits, two counts)
// for small caches, the moved rows (2 x 4 D bytes each) for large ones.
#include <cooperative_groups.h>

#include <type_traits>

#include "sm100.cuh"
#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kMaxKeys = 40960;  // keys a block keeps (160 KB); more are read again from memory
constexpr int kMoves = 4;        // 16-byte pieces of K and V that a thread has under way

struct EvictParams {
  PagedParams c;
  int keep, trigger, sink, recent;
  int pieces, piece_bits;  // 16-byte pieces of a row, a power of two
  int32_t* lists;  // [batch, Hkv, 2, keep]: free slots, then the slots that fill them
};

// Order-preserving map of a weight to [0x007fffff, 0xff800000]: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.f) w = 0.f;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sum of x over the lanes before this one.
__device__ __forceinline__ int warp_before(int x, int lane) {
  int y = x;
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(~0u, y, o);
    if (lane >= o) y += z;
  }
  return y - x;
}

struct Shared {
  uint32_t hist[3][kBins];
  int warp[kWarps][2];   // counts of each warp
  int block[3][2];       // this block's counts, by round
  int found[3][3];       // digit, slots above it, slots in it
  int sums[kWarps];
  int last_equal;
};

template <bool KEEP_KEYS>
__global__ void __launch_bounds__(kThreads) evict_kernel(const __grid_constant__ EvictParams p, int cluster) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = blockIdx.x % cluster, at = blockIdx.x / cluster;
  const int h = at % p.c.n_kv_heads, b = at / p.c.n_kv_heads;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  bool bad = false;
  const int n = paged_len(p.c, b, &bad);
  if (bad && tid == 0) *p.c.page_error = 1;
  if (bad || n <= p.keep || n <= p.trigger) return;  // alike for the cluster
  // this block's slots [lo, hi), a warp's [wlo, whi)
  const int per = (n + cluster * kThreads - 1) / (cluster * kThreads) * kThreads;
  const int lo = rank * per;
  const int wlo = lo + warp * (per / kWarps), whi = min(n, wlo + per / kWarps);

  const float* w = p.c.weights + b * p.c.wb + h * p.c.wh;
  const int32_t* pos = p.c.positions + b * p.c.pb + h * p.c.ph;
  const int64_t late = (int64_t)p.c.seen[b] - p.recent;
  auto read_key = [&](int s) -> uint32_t {
    const int x = pos[s];
    return x < p.sink || x >= late ? 0xffffffffu : weight_key(w[s]);
  };
  auto key_of = [&](int s) -> uint32_t { return KEEP_KEYS ? keys[s - lo] : read_key(s); };

  for (int i = tid; i < 3 * kBins; i += kThreads) (&sh.hist[0][0])[i] = 0;
  __syncthreads();
  // digits from the top; `prefix` holds those found
  uint32_t prefix = 0;
  int need = p.keep, equal = 0;
#pragma unroll
  for (int round = 0; round < 3; ++round) {
    constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
    const int shift = kShift[round], bins = 1 << kBits[round];
    uint32_t* hist = sh.hist[round];
#pragma unroll 4
    for (int base = wlo; base < whi; base += 32) {
      const int s = base + lane;
      const bool in = s < whi;
      uint32_t key = 0;
      if (in) {
        if (round == 0) {
          key = read_key(s);
          if (KEEP_KEYS) keys[s - lo] = key;
        } else {
          key = key_of(s);
        }
      }
      const bool counts = in && (round == 0 || (key >> (shift + kBits[round])) == prefix);
      const uint32_t digit = (key >> shift) & (bins - 1);
      // runs of one digit (held tokens, weights of 0) as one addition
      int alike;
      __match_all_sync(~0u, counts ? digit : 0xffffffffu, &alike);
      if (alike) {
        if (counts && lane == 0) atomicAdd(&hist[digit], 32u);
      } else if (counts) {
        atomicAdd(&hist[digit], 1u);
      }
    }
    if (cluster > 1) cl.sync(); else __syncthreads();
    // each thread four bins, from the top: bins - 4 tid - 4 ...
    const int own = bins - 4 * tid - 4;
    uint4 sum = make_uint4(0, 0, 0, 0);
    if (own >= 0)
      for (int r = 0; r < cluster; ++r) {
        const uint32_t* other = cluster > 1 ? cl.map_shared_rank(hist, r) : hist;
        const uint4 x = *reinterpret_cast<const uint4*>(other + own);
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
    const int mine = (int)(sum.x + sum.y + sum.z + sum.w);
    int above = warp_before(mine, lane);
    if (lane == 31) sh.sums[warp] = above + mine;
    __syncthreads();
    for (int i = 0; i < warp; ++i) above += sh.sums[i];
    if (above < need && above + mine >= need) {
      const int c[4] = {(int)sum.w, (int)sum.z, (int)sum.y, (int)sum.x};
      int i = 0;
      while (above + c[i] < need) above += c[i++];
      sh.found[round][0] = own + 3 - i;
      sh.found[round][1] = above;
      sh.found[round][2] = c[i];
    }
    __syncthreads();
    prefix = prefix << kBits[round] | (uint32_t)sh.found[round][0];
    need -= sh.found[round][1];
    equal = sh.found[round][2];
  }
  const uint32_t t = prefix;

  // the blocks' and warps' counts before this warp, of two numbers at once
  auto offsets = [&](int round, int x, int y, int* bx, int* by) {
    if (lane == 0) sh.warp[warp][0] = x, sh.warp[warp][1] = y;
    __syncthreads();
    int ax = 0, ay = 0, tx = 0, ty = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i == warp) ax = tx, ay = ty;
      tx += sh.warp[i][0];
      ty += sh.warp[i][1];
    }
    if (cluster > 1) {
      if (tid == 0) sh.block[round][0] = tx, sh.block[round][1] = ty;
      cl.sync();
      for (int r = 0; r < rank; ++r) {
        const int* o = cl.map_shared_rank(&sh.block[round][0], r);
        ax += o[0];
        ay += o[1];
      }
    }
    *bx = ax;
    *by = ay;
  };

  // `need` of the `equal` slots with key t are kept, the lowest: those up to slot last_equal
  int last_equal = n;
  if (need < equal) {
    int x = 0, before, unused;
    for (int base = wlo; base < whi; base += 32) {
      const int s = base + lane;
      x += __popc(__ballot_sync(~0u, s < whi && key_of(s) == t));
    }
    if (tid == 0) sh.last_equal = -1;
    offsets(0, x, 0, &before, &unused);
    if (before < need && before + x >= need) {
      for (int base = wlo; base < whi; base += 32) {
        const int s = base + lane;
        const unsigned votes = __ballot_sync(~0u, s < whi && key_of(s) == t);
        if (before + __popc(votes) >= need) {
          if (votes >> lane & 1 && before + __popc(votes & ((1u << lane) - 1)) + 1 == need) sh.last_equal = s;
          break;
        }
        before += __popc(votes);
      }
    }
    if (cluster > 1) cl.sync(); else __syncthreads();
    for (int r = 0; r < cluster; ++r) {
      const int x = *(cluster > 1 ? cl.map_shared_rank(&sh.last_equal, r) : &sh.last_equal);
      if (x >= 0) last_equal = x;
    }
    __syncthreads();
  }
  auto kept = [&](int s) -> bool {
    const uint32_t key = key_of(s);
    return key > t || (key == t && s <= last_equal);
  };
  int n_free = 0, n_move = 0, free0, move0;
  for (int base = wlo; base < whi; base += 32) {
    const int s = base + lane;
    const unsigned votes = __ballot_sync(~0u, s < whi && kept(s) != (s < p.keep));
    const unsigned below = __ballot_sync(~0u, s < p.keep);
    n_free += __popc(votes & below);
    n_move += __popc(votes & ~below);
  }
  offsets(1, n_free, n_move, &free0, &move0);
  int32_t* free_list = p.lists + (int64_t)at * 2 * p.keep;
  int32_t* move_list = free_list + p.keep;
  for (int base = wlo; base < whi; base += 32) {
    const int s = base + lane;
    const bool one = s < whi && kept(s) != (s < p.keep);
    const unsigned votes = __ballot_sync(~0u, one), below = __ballot_sync(~0u, s < p.keep), lower = (1u << lane) - 1;
    if (one) {
      if (s < p.keep) free_list[free0 + __popc(votes & below & lower)] = s;
      else move_list[move0 + __popc(votes & ~below & lower)] = s;
    }
    free0 += __popc(votes & below);
    move0 += __popc(votes & ~below);
  }
  // all moves: the last block's last warp ends at their number
  if (warp == kWarps - 1 && lane == 0) sh.block[2][0] = move0;
  __threadfence();
  if (cluster > 1) cl.sync(); else __syncthreads();
  const int moves = *(cluster > 1 ? cl.map_shared_rank(&sh.block[2][0], cluster - 1) : &sh.block[2][0]);

  // 16 bytes of K and of V a thread, neighbouring pieces by neighbouring threads
  const int64_t all = (int64_t)moves * p.pieces;
  const int stride = cluster * kThreads;
  for (int64_t e0 = rank * kThreads + tid; e0 < all; e0 += stride * kMoves) {
    uint4 kx[kMoves], vx[kMoves];
    char *kd[kMoves], *vd[kMoves];
    bool ok[kMoves];
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int64_t e = e0 + i * stride;
      ok[i] = e < all;
      if (ok[i]) {
        const int m = (int)(e >> p.piece_bits), part = (int)e & (p.pieces - 1);
        const int to = free_list[m], from = move_list[m];
        const int pt = paged_page(p.c, b, to / p.c.page_size, &bad), pf = paged_page(p.c, b, from / p.c.page_size, &bad);
        ok[i] = pt >= 0 && pf >= 0;
        if (part == 0) {
          float* wr = p.c.weights + b * p.c.wb + h * p.c.wh;
          int32_t* pr = p.c.positions + b * p.c.pb + h * p.c.ph;
          wr[to] = wr[from];
          pr[to] = pr[from];
        }
        if (ok[i]) {
          char* k = static_cast<char*>(p.c.k) + 2 * h * p.c.kh + 16 * part;
          char* v = static_cast<char*>(p.c.v) + 2 * h * p.c.vh + 16 * part;
          const int rt = to % p.c.page_size, rf = from % p.c.page_size;
          kd[i] = k + 2 * (pt * p.c.kp + rt * p.c.kr);
          vd[i] = v + 2 * (pt * p.c.vp + rt * p.c.vr);
          kx[i] = *reinterpret_cast<const uint4*>(k + 2 * (pf * p.c.kp + rf * p.c.kr));
          vx[i] = *reinterpret_cast<const uint4*>(v + 2 * (pf * p.c.vp + rf * p.c.vr));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      if (ok[i]) {
        *reinterpret_cast<uint4*>(kd[i]) = kx[i];
        *reinterpret_cast<uint4*>(vd[i]) = vx[i];
      }
  }
  if (bad) *p.c.page_error = 1;
  if (cluster > 1) cl.sync();  // nobody leaves while its count is read
}

// The lengths, once every head has read the old ones.
__global__ void evict_lens_kernel(PagedParams c, int keep, int trigger) {
  sm100::pdl_wait();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= c.batch) return;
  bool bad = false;
  const int n = paged_len(c, b, &bad);
  if (!bad && n > keep && n > trigger) c.seq_lens[b] = keep;
}

// Blocks per (sequence, KV head): as few as give every SM two, or each block no more than 2048 slots.
int cluster_size(const PagedParams& c) {
  const int64_t heads = (int64_t)c.batch * c.n_kv_heads, slots = (int64_t)c.max_pages * c.page_size;
  int size = 1;
  while (size < kMaxCluster && (heads * size < 2 * 148 || slots / size > kMaxKeys) && slots / size > 2048) size *= 2;
  return size;
}

template <bool KEEP_KEYS>
cudaError_t launch(const EvictParams& p, int cluster, int smem, cudaStream_t st) {
  auto kern = evict_kernel<KEEP_KEYS>;
  cudaError_t e = allow_smem<std::integral_constant<bool, KEEP_KEYS>>(kern, kMaxKeys * 4);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cluster * p.c.n_kv_heads * p.c.batch));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, cluster);
}

}  // namespace

size_t paged_evict_workspace(const SwaPagedEvictArgs& a) {
  return ((size_t)a.cache.batch * a.cache.n_kv_heads * 2 * a.keep * sizeof(int32_t) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_evict(const PagedParams& c, const SwaPagedEvictArgs& a, cudaStream_t st) {
  EvictParams p;
  p.c = c;
  p.keep = a.keep; p.trigger = a.trigger; p.sink = a.sink_size; p.recent = a.recent;
  p.pieces = a.cache.head_dim / 8;
  p.piece_bits = p.pieces == 2 ? 1 : p.pieces == 4 ? 2 : p.pieces == 8 ? 3 : 4;
  p.lists = static_cast<int32_t*>(a.workspace);
  const int cluster = cluster_size(c);
  const int64_t slots = (int64_t)c.max_pages * c.page_size;
  const int64_t per = (slots + cluster * kThreads - 1) / (cluster * kThreads) * kThreads;
  cudaError_t e = per <= kMaxKeys ? launch<true>(p, cluster, (int)per * 4, st) : launch<false>(p, cluster, 0, st);
  if (e != cudaSuccess) return e;
  return launch_pdl(evict_lens_kernel, (c.batch + 127) / 128, 128, 0, st, c, p.keep, p.trigger);
}

}  // namespace swa
