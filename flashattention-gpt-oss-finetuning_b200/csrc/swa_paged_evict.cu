// swa_paged_evict.cu -- cuts the sequences of a paged cache down to a budget by the weight that
// attention has laid on each slot.
//
// Each slot has a 32-bit key: held tokens the largest, then the weights in order.  The budget-th
// largest key t is found digit by digit, 8 bits at a time, from histograms; slots above t are
// kept, and of those equal to t the lowest.  Slots that come free below the budget and kept slots
// behind it are numbered in order, and the i-th of the one takes the i-th of the other: no row is
// both read and written, so all of them move at once, and only as many as have to.
//
// select_kernel: a (sequence, KV head) belongs to a cluster of 1 to 8 blocks, each with a stretch of
// the slots, whose keys it keeps in shared memory: the weights and token numbers are read once (8
// bytes a slot).  Blocks send one another their histograms and counts through distributed shared
// memory, one cluster barrier a digit.  move_kernel: a thread per 16 bytes of K and of V of a row
// that moves, and the lengths.  What bounds the first are its dependent steps (load, four digits, two
// counts), the second the rows, 128 or 256 scattered bytes each.
//
// A sequence with a page out of range among those in use is not cut: no row, weight or number of it
// moves and its length stays, like one whose length is out of range.  Every block looks through the
// sequence's whole table, so that all its heads decide alike without a word between them.
//
// Measured on a B200, from a CUDA graph: 4 x 8 heads of 16384 to 32768 slots cut to 4096 (57 MB of rows
// move) 34 us (with cold caches select 20, move 17); 64 x 4 heads of dim 128 with some 1080 slots cut to
// 1024, in one kernel, 13 us (cold 17).
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
constexpr int kBins = 256;
constexpr int kDigits = 4;
constexpr int kMaxCluster = 8;
// keys a block keeps, 96 KB (two blocks an SM up to 23552 keys, one beyond); more are read again from memory
constexpr int kMaxKeys = 24576;
constexpr int kAhead = 8;        // slots whose loads a thread has under way
constexpr int kMoveThreads = 256;

struct EvictParams {
  PagedParams c;
  int keep, trigger, sink, recent;
  int pieces, piece_bits;  // 16-byte pieces of a row, a power of two
  int32_t* counts;  // [batch, Hkv]: moves, -1 where the sequence is not cut
  int32_t* lists;   // [batch, Hkv, 2, most]: free slots, then the slots that fill them
  int most;         // moves that a (sequence, KV head) can have
  int all_here;     // 1: a cluster is a sequence, a block a head, and select_kernel moves the rows itself
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

// A 16-byte piece of K and of V of slot `from` to slot `to`, with the first also weight and position.
// (select_kernel has found both pages in range; one that is not, in a table written meanwhile, is not followed.)
__device__ __forceinline__ void move_piece(const EvictParams& p, int b, int h, int to, int from, int part) {
  bool bad = false;
  const int pt = paged_page(p.c, b, to / p.c.page_size, &bad), pf = paged_page(p.c, b, from / p.c.page_size, &bad);
  if (bad) return;
  char* k = static_cast<char*>(p.c.k) + 2 * h * p.c.kh + 16 * part;
  char* v = static_cast<char*>(p.c.v) + 2 * h * p.c.vh + 16 * part;
  const int rt = to % p.c.page_size, rf = from % p.c.page_size;
  const uint4 x = *reinterpret_cast<const uint4*>(k + 2 * (pf * p.c.kp + rf * p.c.kr));
  const uint4 y = *reinterpret_cast<const uint4*>(v + 2 * (pf * p.c.vp + rf * p.c.vr));
  *reinterpret_cast<uint4*>(k + 2 * (pt * p.c.kp + rt * p.c.kr)) = x;
  *reinterpret_cast<uint4*>(v + 2 * (pt * p.c.vp + rt * p.c.vr)) = y;
  if (part == 0) {
    float* w = p.c.weights + b * p.c.wb + h * p.c.wh;
    int32_t* x = p.c.positions + b * p.c.pb + h * p.c.ph;
    w[to] = w[from];
    x[to] = x[from];
  }
}

struct Shared {
  uint32_t hist[kDigits][kBins];
  uint32_t sent[2][kMaxCluster][kBins];  // the blocks' histograms, of even and odd digits
  int warp[kWarps][2];                   // counts of each warp
  int block[2][kMaxCluster][2];          // the blocks' counts, by round
  int found[kDigits][3];                 // digit, slots above it, slots in it
  int sums[kBins / 32];                  // counts of 32 bins each
  int last_equal;                        // the last slot with key t that is kept
};

template <bool KEEP_KEYS>
__global__ void __launch_bounds__(kThreads, 2) select_kernel(const __grid_constant__ EvictParams p, int cluster) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = blockIdx.x % cluster, at = blockIdx.x / cluster;
  const int h = at % p.c.n_kv_heads, b = at / p.c.n_kv_heads;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  sm100::pdl_wait();
  sm100::pdl_trigger();
  bool bad = false;
  const int n = paged_len(p.c, b, &bad);
  if (bad || n <= p.keep || n <= p.trigger) {  // alike for the cluster
    if (tid == 0 && rank == 0) {
      if (!p.all_here) p.counts[at] = -1;
      if (bad) *p.c.page_error = 1;
    }
    return;
  }
  // this block's slots [lo, hi), a warp's [wlo, whi); sums that can pass 2^31 without a sign (n may reach
  // 2^31 - 1025, and 8 blocks' stretches then end at 2^31)
  const unsigned all_threads = (unsigned)(cluster * kThreads);
  const int per = (int)(((unsigned)n + all_threads - 1) / all_threads) * kThreads;
  const int lo = rank * per;
  const int wlo = lo + warp * (per / kWarps), whi = (int)min((unsigned)n, (unsigned)wlo + (unsigned)(per / kWarps));

  const float* w = p.c.weights + b * p.c.wb + h * p.c.wh;
  const int32_t* pos = p.c.positions + b * p.c.pb + h * p.c.ph;
  const int64_t late = (int64_t)p.c.seen[b] - p.recent;
  auto make_key = [&](float weight, int x) -> uint32_t { return x < p.sink || x >= late ? 0xffffffffu : weight_key(weight); };
  auto key_of = [&](int s) -> uint32_t { return KEEP_KEYS ? keys[s - lo] : make_key(w[s], pos[s]); };


  for (int i = tid; i < kDigits * kBins; i += kThreads) (&sh.hist[0][0])[i] = 0;
  // waited for before the first write to another block, or before the sequence's new length is written
  if (cluster > 1 || p.all_here) cl.barrier_arrive();
  __syncthreads();
  // digits from the top; `prefix` holds those found
  uint32_t prefix = 0;
  int need = p.keep, equal = 0;
#pragma unroll
  for (int round = 0; round < kDigits; ++round) {
    const int shift = 24 - 8 * round;
    uint32_t* hist = sh.hist[round];
    // one addition for the lanes with the same digit: weights lie in few octaves, held tokens and
    // weights of 0 in one place
    auto count = [&](bool counts, uint32_t key) {
      const uint32_t digit = counts ? (key >> shift) & (kBins - 1) : kBins;
      const unsigned alike = __match_any_sync(~0u, digit);
      if (counts && lane == __ffs(alike) - 1) atomicAdd(&hist[digit], (uint32_t)__popc(alike));
    };
    if (round == 0) {
      for (int base = wlo; base < whi; base += 32 * kAhead) {
        float weight[kAhead];
        int x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int s = base + 32 * i + lane;
          weight[i] = s < whi ? w[s] : 0.f;
          x[i] = s < whi ? pos[s] : 0;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int s = base + 32 * i + lane;
          const uint32_t key = make_key(weight[i], x[i]);
          if (KEEP_KEYS && s < whi) keys[s - lo] = key;
          if (base + 32 * i < whi) count(s < whi, key);
        }
      }
      // the pages in use, all of them, by the last warps first, which have the fewest slots (by the first ones 0.2 us
      // more for 64 x 4 heads of some 1080 slots)
      for (int i = kThreads - 1 - tid; i < (n - 1) / p.c.page_size + 1; i += kThreads) paged_page(p.c, b, i, &bad);
      bad = __syncthreads_or(bad);
    } else {
      for (int base = wlo; base < whi; base += 32) {
        const int s = base + lane;
        const uint32_t key = s < whi ? key_of(s) : 0u;
        const bool counts = s < whi && key >> (shift + 8) == prefix;
        if (__any_sync(~0u, counts)) count(counts, key);
      }
      __syncthreads();
    }
    if (cluster > 1) {
      // 16 bytes of the histogram to a block by each thread
      const int to = tid / (kBins / 4), part = tid % (kBins / 4);
      if (round == 0) cl.barrier_wait();
      if (to < cluster)
        *cl.map_shared_rank(reinterpret_cast<uint4*>(sh.sent[round & 1][rank]) + part, to) =
            reinterpret_cast<const uint4*>(hist)[part];
      cl.sync();
    }
    // a bin a thread, from the top
    int here = 0, above = 0;
    if (tid < kBins) {
      const int bin = kBins - 1 - tid;
      if (cluster > 1) {
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < cluster) here += sh.sent[round & 1][r][bin];
      } else {
        here = hist[bin];
      }
      above = warp_before(here, lane);
      if (lane == 31) sh.sums[warp] = above + here;
    }
    __syncthreads();
    if (tid < kBins) {
#pragma unroll
      for (int i = 0; i < kBins / 32; ++i)
        if (i < warp) above += sh.sums[i];
      if (above < need && above + here >= need) {  // one thread
        sh.found[round][0] = kBins - 1 - tid;
        sh.found[round][1] = above;
        sh.found[round][2] = here;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)sh.found[round][0];
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
      if (tid < cluster) {
        int* o = cl.map_shared_rank(&sh.block[round][rank][0], tid);
        o[0] = tx;
        o[1] = ty;
      }
      cl.sync();
      for (int r = 0; r < rank; ++r) {
        ax += sh.block[round][r][0];
        ay += sh.block[round][r][1];
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
    offsets(0, x, 0, &before, &unused);
    if (before < need && before + x >= need) {  // one warp of the cluster
      for (int base = wlo; base < whi; base += 32) {
        const int s = base + lane;
        const unsigned votes = __ballot_sync(~0u, s < whi && key_of(s) == t);
        if (before + __popc(votes) >= need) {
          if (votes >> lane & 1 && before + __popc(votes & ((1u << lane) - 1)) + 1 == need)
            for (int r = 0; r < cluster; ++r) *(cluster > 1 ? cl.map_shared_rank(&sh.last_equal, r) : &sh.last_equal) = s;
          break;
        }
        before += __popc(votes);
      }
    }
    if (cluster > 1) cl.sync(); else __syncthreads();
    last_equal = sh.last_equal;
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
  int32_t* free_list = p.lists + (int64_t)at * 2 * p.most;
  int32_t* move_list = free_list + p.most;
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
  // the last block's last warp ends at their number
  if (rank == cluster - 1 && warp == kWarps - 1 && lane == 0) {
    if (bad) *p.c.page_error = 1;
    if (!p.all_here) p.counts[at] = bad ? -1 : move0;
    else sh.block[0][0][0] = bad ? 0 : move0;
  }
  if (p.all_here) {
    __syncthreads();
    const int pieces = sh.block[0][0][0] << p.piece_bits;
    for (int e = tid; e < pieces; e += kThreads) {
      const int m = e >> p.piece_bits;
      move_piece(p, b, h, free_list[m], move_list[m], e & (p.pieces - 1));
    }
    cl.barrier_wait();  // every head has read the old length
    if (h == 0 && tid == 0 && !bad) p.c.seq_lens[b] = p.keep;
  }
}

// blockIdx.y strides over (sequence, KV head), blockIdx.x over the pieces of its moves; then the
// lengths.  One piece a thread and full occupancy: two a thread at half of it are 3 us slower where
// 57 MB move (17 us with cold caches, 3.4 TB/s in scattered rows of 128 bytes).
__global__ void __launch_bounds__(kMoveThreads, 8) move_kernel(const __grid_constant__ EvictParams p) {
  sm100::pdl_wait();
  const int heads = p.c.batch * p.c.n_kv_heads;
  const int64_t e = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x;
  const int m = (int)(e >> p.piece_bits), part = (int)e & (p.pieces - 1);
  for (int at = blockIdx.y; at < heads; at += gridDim.y) {
    const int h = at % p.c.n_kv_heads, b = at / p.c.n_kv_heads, moves = p.counts[at];
    if (moves >= 0 && h == 0 && e == 0) p.c.seq_lens[b] = p.keep;
    if (m >= moves) continue;
    const int32_t* free_list = p.lists + (int64_t)at * 2 * p.most;
    move_piece(p, b, h, free_list[m], free_list[p.most + m], part);
  }
}

// Blocks per (sequence, KV head): as many as fit beside one another (two an SM), of no less than
// 2048 slots each; more where a block could not keep its keys.  (4 x 8 heads of 32768 slots, calls with
// the copy that restores the weights, when this was chosen: 8 blocks a head 43 us, 4 46.)
int cluster_size(const PagedParams& c) {
  const int64_t heads = (int64_t)c.batch * c.n_kv_heads, slots = (int64_t)c.max_pages * c.page_size;
  int size = 1;
  while (size < kMaxCluster && slots / size > 2048 && (heads * size * 2 <= 2 * 148 || slots / size > kMaxKeys)) size *= 2;
  return size;
}

template <bool KEEP_KEYS>
cudaError_t launch(const EvictParams& p, int cluster, int smem, cudaStream_t st) {
  auto kern = select_kernel<KEEP_KEYS>;
  cudaError_t e = allow_smem<std::integral_constant<bool, KEEP_KEYS>>(kern, kMaxKeys * 4);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cluster * p.c.n_kv_heads * p.c.batch));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)(p.all_here ? p.c.n_kv_heads : cluster);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p, cluster);
}

}  // namespace

// The moves that one (sequence, KV head) can have: a free slot below keep, a slot from keep on.
static int64_t most_moves(const SwaPagedEvictArgs& a) {
  const int64_t behind = (int64_t)a.cache.max_pages * a.cache.page_size - a.keep;
  return behind < 0 ? 0 : behind < a.keep ? behind : a.keep;
}
static size_t count_ints(const SwaPagedEvictArgs& a) {
  return ((size_t)a.cache.batch * a.cache.n_kv_heads + 63) & ~(size_t)63;
}

size_t paged_evict_workspace(const SwaPagedEvictArgs& a) {
  const size_t lists = (size_t)a.cache.batch * a.cache.n_kv_heads * 2 * most_moves(a);
  return ((count_ints(a) + lists) * sizeof(int32_t) + 255) & ~(size_t)255;
}

cudaError_t launch_paged_evict(const PagedParams& c, const SwaPagedEvictArgs& a, cudaStream_t st) {
  EvictParams p;
  p.c = c;
  p.keep = a.keep; p.trigger = a.trigger; p.sink = a.sink_size; p.recent = a.recent;
  p.pieces = a.cache.head_dim / 8;
  p.piece_bits = p.pieces == 2 ? 1 : p.pieces == 4 ? 2 : p.pieces == 8 ? 3 : 4;
  p.counts = static_cast<int32_t*>(a.workspace);
  p.lists = p.counts + count_ints(a);
  p.most = (int)most_moves(a);
  const int cluster = cluster_size(c);
  const int64_t slots = (int64_t)c.max_pages * c.page_size;
  // Few moves, at most four pieces a thread, of heads that fit in a cluster: one kernel does it all
  // (calls one after the other, when this was chosen: 8 heads of one sequence 12.8 us, 14.0 with two kernels;
  // with the copy that restores the weights, 2 us on the GPU and a launch, 64 x 4 heads of dim 128
  // 22.1 and 22.6).
  p.all_here = cluster == 1 && c.n_kv_heads <= kMaxCluster && (int64_t)p.most * p.pieces <= 4 * kThreads;
  const int64_t per = (slots + cluster * kThreads - 1) / (cluster * kThreads) * kThreads;
  cudaError_t e = per <= kMaxKeys ? launch<true>(p, cluster, (int)per * 4, st) : launch<false>(p, cluster, 0, st);
  if (e != cudaSuccess || p.all_here) return e;
  const int64_t x = ((int64_t)p.most * p.pieces + kMoveThreads - 1) / kMoveThreads;
  const int heads = c.batch * c.n_kv_heads;
  return launch_pdl(move_kernel, dim3((unsigned)x, (unsigned)(heads < 65535 ? heads : 65535)), kMoveThreads, 0, st, p);
}

}  // namespace swa
