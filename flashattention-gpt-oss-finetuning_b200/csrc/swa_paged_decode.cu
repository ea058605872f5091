// swa_paged_decode.cu -- attention of one new token per sequence over its paged cache, split over
// the cache's length and joined.
//
// o[b, h] = sum_j p_j v_j / l, p_j = exp2(s_j - m), s_j = scale log2(e) q k_j over the visible
// slots j, with the running maximum m and sum l of an online softmax.  Partial (m, l, o) of
// disjoint sets of slots are joined exactly: (m, l, o) -> (max m, sum l 2^(m - max), ...).
//
// Work is cut into units of 16 slots, all of one page.  Where no sequence can have many visible
// slots, a (sequence, KV head) belongs to one block or even one warp, which finishes it.  Else the
// units of all sequences and KV heads, in a row, are dealt out evenly to the warps of the grid,
// whatever the lengths: a warp walks its range, a block joins its warps' pieces, and a sequence that
// spans blocks leaves a partial per block for finish_kernel.  The device alone knows the lengths, so
// the host needs none.  (More than 16 query heads a KV head are tiles of 16, each a block's, which walk
// the same range at the same time: every tile copies K and V to its SM, from DRAM they come once.)
//
// A warp keeps a ring of three units of K and V in shared memory, filled by 16-byte cp.async.  It
// multiplies with mma.sync m16n8k16: up to 8 (or 16) query heads of the KV head are the 16 rows, so
// K and V are read once per group.  The operator is bound by the bytes of the cache: 8 heads of dim 64
// need 8 flops a byte.  (tcgen05 takes 64 or 128 rows and shared-memory operands, and a TMEM round trip
// for the softmax of 8 rows; there is no rate to gain here.)  The weights p are multiplied as two
// 16-bit pieces, hi + lo, so that rounding them adds 2^-18 (bf16) to a result that is rounded at
// 2^-9: with 8 heads the lo pieces are the tile's other 8 rows and cost nothing.
//
// Measured on a B200 (6.56 TB/s copy), from a CUDA graph, 8 KV heads of dim 64 with 8 query heads each: 32 sequences of
// 129 to 16384 slots (542 MB) 96 us, 5.7 TB/s; 256 windows of 128 (72 MB) 16 us, 4.5 TB/s, bound by the
// dependent steps of one short walk a warp; one window 4.5 us, all of it latency; one sequence of
// 131072 slots with its weights (277 MB) 69 us, of which 54 the attention (268 MB, and 34 MB of scores
// written) and 15 the weights.
#include "sm100.cuh"
#include "swa_host.cuh"
#include "swa_paged.cuh"

namespace swa {
namespace {

using sm100::saddr;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnit = 16;     // slots per unit
constexpr int kSms = 148;

template <int D> struct Shape {
  static constexpr int kUnitBytes = 2 * kUnit * D * 2;  // K and V
  // Three stages and four blocks an SM (128 registers a thread): 97 us where four and three take 101
  // (32 sequences of up to 16384 slots, D 64), and 256 windows fit in one wave (17 us, not 23).
  static constexpr int kStages = 3;
  static constexpr int kRing = kStages * kUnitBytes;    // per warp
  static constexpr int kBlocksPerSm = D == 128 ? 2 : 4;
  static constexpr int kMaxBlocks = kSms * kBlocksPerSm;
};

struct DecodeParams {
  PagedParams c;
  int Hq, G, tiles, W, S;  // tiles: row tiles per KV head
  int units_per_page;
  int max_units;           // bound on the units of a sequence
  int warps;               // warps per (sequence, KV head, tile), 1 or kWarps; 0: dealt out
  float scale_log2;
  const void* q; void* o;
  int64_t qb, qh, ob, oh;
  float* lse;              // [B, Hq] or null
  const float* sinks;
  float* wout;
  int64_t wob, woh;
  float decay;
  int weigh_here;          // 1: decode_kernel itself writes wout
  float* partials;         // [blocks][2] Partial
  float* heads;            // [blocks][warps] Partial: the first piece of a warp that has two
  int2* spans;             // [B * Hkv * tiles]: first and last group of blocks, where dealt out
  float* scores;           // [B * Hkv * tiles][max_units][16][ROWS]
};

// m[ROWS], l[ROWS], o[ROWS][D]
template <int D, int ROWS> struct Partial {
  static constexpr int kFloats = ROWS * (D + 2);
  static __device__ __forceinline__ float* m(float* p) { return p; }
  static __device__ __forceinline__ float* l(float* p) { return p + ROWS; }
  static __device__ __forceinline__ float* o(float* p) { return p + 2 * ROWS; }
};

// The units of a sequence: those of its sinks that lie before the window's first, then the window's.
struct Sequence {
  int n, first, sinks, c0, a, units;
  bool bad;
};
__device__ __forceinline__ Sequence sequence(const DecodeParams& p, int b) {
  Sequence s;
  s.bad = false;
  s.n = paged_len(p.c, b, &s.bad);
  const VisibleSlots v = visible_slots(s.n, p.W, p.S);
  s.first = v.first;
  s.sinks = v.sinks;
  s.c0 = v.first / kUnit;
  const int sink_units = (v.sinks + kUnit - 1) / kUnit;
  s.a = sink_units < s.c0 ? sink_units : s.c0;
  const int u = s.a + (s.n + kUnit - 1) / kUnit - s.c0;
  s.units = u > 0 ? u : 1;  // an empty sequence has one, all masked, that writes its output
  return s;
}
__device__ __forceinline__ int unit_chunk(const Sequence& s, int u) { return u < s.a ? u : u - s.a + s.c0; }

// Units, per KV head, of this lane's sequences: `per_lane` neighbouring ones.
__device__ __forceinline__ int64_t lane_units(const DecodeParams& p, int lane, int* per_lane) {
  const int per = (p.c.batch + 31) / 32;
  *per_lane = per;
  int64_t u = 0;
  for (int i = 0; i < per; ++i) {
    const int b = lane * per + i;
    if (b < p.c.batch) u += sequence(p, b).units;
  }
  return u;
}
__device__ __forceinline__ int64_t warp_sum(int64_t x) {
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}
__device__ __forceinline__ int64_t warp_prefix(int64_t x, int lane) {  // exclusive
  int64_t y = x;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t z = __shfl_up_sync(~0u, y, o);
    if (lane >= o) y += z;
  }
  return y - x;
}

// Blocks that share `total` units, two for each warp: a warp is without any only where there are fewer
// than kWarps of them in all.
__device__ __forceinline__ int active_blocks(int64_t total, int blocks) {
  const int64_t n = (total + 2 * kWarps - 1) / (2 * kWarps);
  return n < blocks ? (int)n : blocks;
}

// ---------------------------------------------------------------------------------------
// tensor-core and copy primitives
// ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// 16 bytes to shared memory
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the same, zeros where !ok (then nothing is read)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte piece `piece` of row `row` in a unit of 16 rows: pieces are swizzled so
// that eight rows' equal pieces, an ldmatrix, lie in different banks.
template <int D> __device__ __forceinline__ uint32_t swizzled(int row, int piece) {
  constexpr int kPieces = D / 8;
  const int x = D >= 64 ? (row & 7) : D == 32 ? ((row >> 1) & 3) : ((row >> 2) & 1);
  return (uint32_t)(row * kPieces + (piece ^ x)) * 16;
}

// A sequence with a page or a length out of range: its partials' maximum is NaN (a score's NaN never gets into
// a maximum, only into sums), and its log-sum-exp this one, which no arithmetic yields; whoever writes
// weights leaves those of such a sequence alone.
__device__ __forceinline__ float bad_lse() { return __uint_as_float(0xffc0bad0u); }
__device__ __forceinline__ bool is_bad(float lse) { return __float_as_uint(lse) == 0xffc0bad0u; }
// The larger one; NaN where one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A finished row's output and log-sum-exp from its joined maximum, sum and value.
struct Row {
  float inv, lse;
};
__device__ __forceinline__ Row finish(float m, float l, float sink) {
  const float top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
  const float f = fast_exp2(m - base), total = l * f + fast_exp2(sink - base);
  Row r;
  r.inv = total == 0.f ? 0.f : f / total;
  r.lse = m != m ? bad_lse() : total == 0.f ? -INFINITY : top + log2f(total);
  return r;
}

// ---------------------------------------------------------------------------------------
// A warp's walk over units [u0, u1) of one (sequence, KV head, tile)
// ---------------------------------------------------------------------------------------
template <typename T, int D, int ROWS, bool WEIGH> struct Walk {
  static constexpr int kHalves = ROWS == 16 ? 2 : 1;  // rows of a thread: lane / 4 (+ 8)
  static constexpr int kNt = D / 8, kKs = D / 16, kStages = Shape<D>::kStages;

  float o[kNt][4];
  float m[kHalves], l[kHalves];
  bool bad;

  __device__ __forceinline__ void run(const DecodeParams& p, uint32_t ring, int lane, int b, int hv, const Sequence& s,
                                      int u0, int u1) {
    const int h = hv / p.tiles, tile = hv % p.tiles;
    const int g = lane / 4, t = lane % 4;
    bad = s.bad;
#pragma unroll
    for (int i = 0; i < kNt; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < kHalves; ++i) m[i] = -INFINITY, l[i] = 0.f;

    // A lane copies kCopies pieces of K and of V of every unit, kRows rows apart.
    constexpr int kPieces = D / 8, kCopies = kUnit * kPieces / 32, kRows = 32 / kPieces;
    const int row0 = lane / kPieces, piece = lane % kPieces;
    const T* kbase = static_cast<const T*>(p.c.k) + h * p.c.kh + row0 * p.c.kr + piece * 8;
    const T* vbase = static_cast<const T*>(p.c.v) + h * p.c.vh + row0 * p.c.vr + piece * 8;
    const int64_t kstep = kRows * p.c.kr, vstep = kRows * p.c.vr;
    uint32_t to[kCopies];
#pragma unroll
    for (int e = 0; e < kCopies; ++e) to[e] = swizzled<D>(row0 + e * kRows, piece);

    // page of unit u0 + 32 i + lane, looked up 32 units at a time
    const int upp = p.units_per_page;
    auto pages = [&](int u) -> int {
      if (u >= u1) return -1;
      const int chunk = unit_chunk(s, u);
      if (chunk * kUnit >= s.n) return -1;
      return paged_page(p.c, b, chunk / upp, &bad);
    };
    int ids = pages(u0 + lane);
    // the loads' place: unit, its chunk, the chunk's place in its page, the ring's stage
    int lu = u0, lchunk = unit_chunk(s, u0), lin = lchunk % upp, lstage = 0;

    auto issue = [&]() {
      if (lu < u1) {
        const int i = (lu - u0) & 31;
        if (i == 0 && lu != u0) ids = pages(lu + lane);
        const int page = __shfl_sync(~0u, ids, i), slot0 = lchunk * kUnit;
        const T* kp = kbase + (page < 0 ? 0 : page) * p.c.kp + lin * (kUnit * p.c.kr);
        const T* vp = vbase + (page < 0 ? 0 : page) * p.c.vp + lin * (kUnit * p.c.vr);
        const uint32_t kd = ring + (uint32_t)lstage * Shape<D>::kUnitBytes, vd = kd + kUnit * D * 2;
        if (page >= 0 && slot0 + kUnit <= s.n && (slot0 >= s.first || slot0 + kUnit <= s.sinks)) {
#pragma unroll
          for (int e = 0; e < kCopies; ++e) {
            copy16(kd + to[e], kp);
            copy16(vd + to[e], vp);
            kp += kstep;
            vp += vstep;
          }
        } else {
#pragma unroll
          for (int e = 0; e < kCopies; ++e) {
            const int slot = slot0 + row0 + e * kRows;
            const bool ok = page >= 0 && slot < s.n && (slot >= s.first || slot < s.sinks);
            copy16(kd + to[e], kp, ok);
            copy16(vd + to[e], vp, ok);
            kp += kstep;
            vp += vstep;
          }
        }
        ++lchunk;
        if (++lin == upp) lin = 0;
        if (++lu == s.a) {
          lchunk = s.c0;
          lin = lchunk % upp;
        }
        if (++lstage == kStages) lstage = 0;
      }
      copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();

    // Q as the A operand, rows past the group's heads as zeros
    uint32_t qa[kKs][4];
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = g + (r & 1) * 8, col = ks * 16 + (r >> 1) * 8 + 2 * t;
        const int head = tile * ROWS + row;
        qa[ks][r] = row < ROWS && head < p.G
                        ? *reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + b * p.qb +
                                                             (int64_t)(h * p.G + head) * p.qh + col)
                        : 0u;
      }

    // Addresses of the matrices in a unit: pieces differ in address bits that the swizzle's are
    // exclusive-ored into, so a piece further on is an exclusive or away.
    const uint32_t kfrag = ring + swizzled<D>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
    const uint32_t vfrag = ring + kUnit * D * 2 + swizzled<D>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
    int chunk = unit_chunk(s, u0);
    uint32_t stage = 0;
    for (int u = u0; u < u1; ++u) {
      issue();
      copy_wait<kStages - 1>();
      __syncwarp();
      float sc[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) {
        uint32_t kb[4];
        ldsm4(kb, (kfrag + stage) ^ (ks * 32));
        mma16816<T>(sc[0], qa[ks], kb[0], kb[1]);
        mma16816<T>(sc[1], qa[ks], kb[2], kb[3]);
      }
      const int slot0 = chunk * kUnit;
      const bool full = slot0 + kUnit <= s.n && (slot0 >= s.first || slot0 + kUnit <= s.sinks);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2 * kHalves; ++e) sc[j][e] *= p.scale_log2;
      if (!full) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int slot = slot0 + 8 * j + 2 * t + e;
            if (slot >= s.n || (slot < s.first && slot >= s.sinks))
#pragma unroll
              for (int r = 0; r < kHalves; ++r) sc[j][2 * r + e] = -INFINITY;
          }
      }
      if constexpr (WEIGH) {
        float* out = p.scores + (((int64_t)b * p.c.n_kv_heads * p.tiles + hv) * p.max_units + u) * (ROWS * kUnit);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < kHalves; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              out[(8 * j + 2 * t + e) * ROWS + g + 8 * r] = tile * ROWS + g + 8 * r < p.G ? sc[j][2 * r + e] : -INFINITY;
      }
      float up[kHalves];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < kHalves; ++r) {
        float x = fmaxf(max3f(sc[0][2 * r], sc[0][2 * r + 1], sc[1][2 * r]), sc[1][2 * r + 1]);
        x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
        x = fmaxf(x, __shfl_xor_sync(~0u, x, 2));
        up[r] = fmaxf(m[r], x);
        grew |= up[r] > m[r];
      }
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int r = 0; r < kHalves; ++r) {
          const float f = up[r] > m[r] ? fast_exp2(m[r] - up[r]) : 1.f;
          m[r] = up[r];
          l[r] *= f;
          if (kHalves == 1) {  // both halves of the tile are this row: its hi and its lo sums
#pragma unroll
            for (int i = 0; i < kNt; ++i) o[i][0] *= f, o[i][1] *= f, o[i][2] *= f, o[i][3] *= f;
          } else {
#pragma unroll
            for (int i = 0; i < kNt; ++i) o[i][2 * r] *= f, o[i][2 * r + 1] *= f;
          }
        }
      }
      uint32_t hi[kHalves][2], lo[kHalves][2];
#pragma unroll
      for (int r = 0; r < kHalves; ++r) {
        const float base = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x = fast_exp2(sc[j][2 * r] - base), y = fast_exp2(sc[j][2 * r + 1] - base);
          l[r] += x + y;
          hi[r][j] = Pack<T>::pack(x, y);
          const T* q = reinterpret_cast<const T*>(&hi[r][j]);
          lo[r][j] = Pack<T>::pack(x - Pack<T>::to(q[0]), y - Pack<T>::to(q[1]));
        }
      }
#pragma unroll
      for (int i = 0; i < kNt; i += 2) {
        uint32_t vb[4];
        ldsm4t(vb, (vfrag + stage) ^ (i * 16));
        if (kHalves == 1) {
          const uint32_t a[4] = {hi[0][0], lo[0][0], hi[0][1], lo[0][1]};
          mma16816<T>(o[i], a, vb[0], vb[1]);
          mma16816<T>(o[i + 1], a, vb[2], vb[3]);
        } else {
          const uint32_t a[4] = {hi[0][0], hi[kHalves - 1][0], hi[0][1], hi[kHalves - 1][1]};
          const uint32_t c[4] = {lo[0][0], lo[kHalves - 1][0], lo[0][1], lo[kHalves - 1][1]};
          mma16816<T>(o[i], a, vb[0], vb[1]);
          mma16816<T>(o[i + 1], a, vb[2], vb[3]);
          mma16816<T>(o[i], c, vb[0], vb[1]);
          mma16816<T>(o[i + 1], c, vb[2], vb[3]);
        }
      }
      __syncwarp();
      chunk = u + 1 == s.a ? s.c0 : chunk + 1;
      stage += Shape<D>::kUnitBytes;
      if (stage == Shape<D>::kRing) stage = 0;
    }
    copy_wait<0>();
    __syncwarp();
    bad = __any_sync(~0u, bad);
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      l[r] += __shfl_xor_sync(~0u, l[r], 1);
      l[r] += __shfl_xor_sync(~0u, l[r], 2);
      if (bad) m[r] = l[r] = NAN;
    }
    if (kHalves == 1)
#pragma unroll
      for (int i = 0; i < kNt; ++i) o[i][0] += o[i][2], o[i][1] += o[i][3];
    if (bad && lane == 0) *p.c.page_error = 1;
  }

  __device__ __forceinline__ void store(float* part, int lane) const {
    using P = Partial<D, ROWS>;
    const int g = lane / 4, t = lane % 4;
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      if (t == 0) {
        P::m(part)[g + 8 * r] = m[r];
        P::l(part)[g + 8 * r] = l[r];
      }
#pragma unroll
      for (int i = 0; i < kNt; ++i)
        *reinterpret_cast<float2*>(P::o(part) + (g + 8 * r) * D + 8 * i + 2 * t) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    }
  }

  // The output of a (sequence, KV head, tile) that this warp has walked whole.
  __device__ __forceinline__ void write(const DecodeParams& p, int lane, int b, int hv) const {
    const int h = hv / p.tiles, tile = hv % p.tiles, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      const int row = tile * ROWS + g + 8 * r, head = h * p.G + row;
      if (row < p.G) {
        const Row f = finish(m[r], l[r], p.sinks ? p.sinks[head] * kLog2e : -INFINITY);
        T* out = static_cast<T*>(p.o) + b * p.ob + head * p.oh + 2 * t;
#pragma unroll
        for (int i = 0; i < kNt; ++i)
          *reinterpret_cast<uint32_t*>(out + 8 * i) = Pack<T>::pack(o[i][2 * r] * f.inv, o[i][2 * r + 1] * f.inv);
        if (p.lse && t == 0) p.lse[(int64_t)b * p.Hq + head] = f.lse;
      }
    }
  }
};

// Joins up to kMost partials, at part[0 .. count), of one (sequence, KV head, tile) by all threads of
// the block: into the output, or into `into` where it is given.
template <typename T, int D, int ROWS, int kMost>
__device__ __forceinline__ void join(const DecodeParams& p, int b, int hv, int count, float* const (&part)[kMost],
                                     float* into) {
  using P = Partial<D, ROWS>;
  const int h = hv / p.tiles, tile = hv % p.tiles;
  const int rows = p.G - tile * ROWS < ROWS ? p.G - tile * ROWS : ROWS;
  for (int e = threadIdx.x; e < rows * (D / 2); e += kThreads) {
    const int r = e / (D / 2), d = e % (D / 2) * 2;
    float m[kMost], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      m[i] = i < count ? P::m(part[i])[r] : -INFINITY;
      top = max_nan(top, m[i]);
    }
    const float base = top == -INFINITY ? 0.f : top;
    float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < count) {
        const float f = fast_exp2(m[i] - base);
        const float2 v = *reinterpret_cast<const float2*>(P::o(part[i]) + r * D + d);
        l = fmaf(P::l(part[i])[r], f, l);
        x = fmaf(v.x, f, x);
        y = fmaf(v.y, f, y);
      }
    if (into) {
      if (d == 0) {
        P::m(into)[r] = top;
        P::l(into)[r] = l;
      }
      *reinterpret_cast<float2*>(P::o(into) + r * D + d) = make_float2(x, y);
    } else {
      const int head = h * p.G + tile * ROWS + r;
      const Row w = finish(top, l, p.sinks ? p.sinks[head] * kLog2e : -INFINITY);
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.ob + head * p.oh + d) = Pack<T>::pack(x * w.inv, y * w.inv);
      if (p.lse && d == 0) p.lse[(int64_t)b * p.Hq + head] = w.lse;
    }
  }
}

// What a row's scores are taken from for its weights: the log-sum-exp; 0 for one whose scores are all -inf,
// so that it adds 0 and not NaN, as its output is 0.
__device__ __forceinline__ float weight_base(float lse) { return lse == -INFINITY ? 0.f : lse; }

// The softmax weights on a visible slot, summed over the heads of a tile: exp2 of the stored scores
// less the finished log-sum-exp.  Rows without a head add 0: their scores are -inf.
template <int ROWS>
__device__ __forceinline__ float slot_weight(const DecodeParams& p, const Sequence& s, int bh, int slot,
                                             const float (&lse)[ROWS]) {
  const int place = slot < s.a * kUnit ? slot : slot - (s.c0 - s.a) * kUnit;
  const float4* sc = reinterpret_cast<const float4*>(p.scores + ((int64_t)bh * p.max_units * kUnit + place) * ROWS);
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < ROWS; r += 4) {
    const float4 x = sc[r / 4];
    sum += (fast_exp2(x.x - lse[r]) + fast_exp2(x.y - lse[r + 1])) +
           (fast_exp2(x.z - lse[r + 2]) + fast_exp2(x.w - lse[r + 3]));
  }
  return sum;
}
__device__ __forceinline__ float old_weight(const DecodeParams& p, int b, int h, int slot) {
  return p.c.weights ? p.decay * p.c.weights[b * p.c.wb + h * p.c.wh + slot] : 0.f;
}

// wout of one (sequence, KV head) of one tile, by `step` threads that have its scores and its lse.
template <int ROWS>
__device__ __forceinline__ void weigh(const DecodeParams& p, const Sequence& s, int b, int h, int first, int step) {
  float lse[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) lse[r] = r < p.G ? weight_base(p.lse[(int64_t)b * p.Hq + h * p.G + r]) : 0.f;
  if (is_bad(lse[0])) return;
#pragma unroll 4
  for (int slot = first; slot < s.n; slot += step) {
    float w = old_weight(p, b, h, slot);
    if (slot < s.sinks || slot >= s.first) w += slot_weight<ROWS>(p, s, b * p.c.n_kv_heads + h, slot, lse);
    p.wout[b * p.wob + h * p.woh + slot] = w;
  }
}

struct Piece {
  int bh, u0, u1, units;
};

// A warp's place among all units, in shared memory: it is wanted between sequences alone.
struct Deal {
  int64_t at, total;
  int blocks;
};

template <typename T, int D, int ROWS, bool WEIGH>
__global__ void __launch_bounds__(kThreads, Shape<D>::kBlocksPerSm) decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ Piece pieces[kWarps][2];
  __shared__ Deal deals[kWarps];
  using P = Partial<D, ROWS>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int vh = p.c.n_kv_heads * p.tiles;
  unsigned char* ring = smem + warp * Shape<D>::kRing;
  // All earlier launches are over past the wait, and only then may finish_kernel start: it reads lengths
  // and weights before its own wait.
  sm100::pdl_wait();
  sm100::pdl_trigger();

  // this warp's range: units [u, ...) of (b, hv), `todo` of them
  int b, hv, u;
  int64_t todo;
  Sequence s;
  if (p.warps) {
    const int bh = blockIdx.x * (kWarps / p.warps) + warp / p.warps;
    if (bh >= p.c.batch * vh) return;  // (warps of the last block, where p.warps is 1)
    b = bh / vh;
    hv = bh % vh;
    s = sequence(p, b);
    const int part = warp % p.warps, share = (s.units + p.warps - 1) / p.warps;
    u = min(part * share, s.units);
    todo = min(u + share, s.units) - u;
  } else {
    int per;
    const int64_t mine = lane_units(p, lane, &per);
    const int heads = p.c.n_kv_heads, group = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
    const int64_t total = warp_sum(mine) * heads, before = warp_prefix(mine, lane) * heads;
    const int blocks = active_blocks(total, gridDim.x / p.tiles);
    if (group >= blocks) return;
    const int64_t b0 = total * group / blocks, b1 = total * (group + 1) / blocks;
    const int64_t at = b0 + (b1 - b0) * warp / kWarps;
    todo = b0 + (b1 - b0) * (warp + 1) / kWarps - at;
    // the lane whose sequences hold `at`, then the sequence
    const unsigned has = __ballot_sync(~0u, at >= before && at < before + mine * heads);
    const int src = has ? __ffs(has) - 1 : 0;
    int64_t rest = at - __shfl_sync(~0u, before, src);
    b = src * per;
    s = sequence(p, b);
    while (todo > 0 && rest >= (int64_t)s.units * heads) {
      rest -= (int64_t)s.units * heads;
      s = sequence(p, ++b);
    }
    hv = (int)(rest / s.units) * p.tiles + tile;
    u = (int)(rest % s.units);
    if (lane == 0) deals[warp] = {at, total, blocks};
  }
  if (lane < 2) pieces[warp][lane].bh = -1;
  __syncwarp();
  Walk<T, D, ROWS, WEIGH> w;
  while (todo > 0) {
    const int u1 = (int)(todo < s.units - u ? u + todo : s.units);
    if (!p.warps && lane == 0) {
      Deal& d = deals[warp];
      // block c holds units [total c / blocks, total (c + 1) / blocks)
      if (u == 0)
        p.spans[b * vh + hv] = make_int2(blockIdx.x / p.tiles, (int)(((d.at + s.units) * d.blocks - 1) / d.total));
      d.at += u1 - u;
    }
    w.run(p, saddr(ring), lane, b, hv, s, u, u1);
    todo -= u1 - u;
    if (u == 0 && u1 == s.units) {
      w.write(p, lane, b, hv);
    } else if (todo > 0) {  // the end of a sequence; the ring is needed again
      w.store(p.heads + ((int64_t)blockIdx.x * kWarps + warp) * P::kFloats, lane);
      if (lane == 0) pieces[warp][0] = {b * vh + hv, u, u1, s.units};
    } else {
      w.store(reinterpret_cast<float*>(ring), lane);
      if (lane == 0) pieces[warp][1] = {b * vh + hv, u, u1, s.units};
    }
    u = 0;
    if (todo > 0 && (hv += p.tiles) >= vh) {  // (b and hv stay at the last one)
      hv %= p.tiles;
      s = sequence(p, ++b);
    }
  }
  if (p.warps == 1) {
    if constexpr (WEIGH) {
      __syncwarp();
      if (p.weigh_here) weigh<ROWS>(p, s, b, hv, lane, 32);
    }
    return;
  }
  __syncthreads();

  if (p.warps) {  // one (sequence, KV head, tile), its pieces in the first warps' rings
    float* part[kWarps];
    int count = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      part[i] = reinterpret_cast<float*>(smem + i * Shape<D>::kRing);
      count += pieces[i][1].bh >= 0;
    }
    if (count) join<T, D, ROWS>(p, b, hv, count, part, nullptr);  // (none: a warp walked it whole)
    if constexpr (WEIGH) {
      __syncthreads();
      if (p.weigh_here) weigh<ROWS>(p, s, b, hv, threadIdx.x, kThreads);
    }
    return;
  }
  // join neighbouring pieces of the same (sequence, KV head, tile)
  for (int i = 0; i < 2 * kWarps;) {
    const Piece a = pieces[i / 2][i % 2];
    if (a.bh < 0) {
      ++i;
      continue;
    }
    float* part[kWarps];  // at most one of every warp
    int count = 0, end = a.u1;
#pragma unroll
    for (int j = 0; j < 2 * kWarps; ++j) {
      if (j < i || pieces[j / 2][j % 2].bh != a.bh) continue;
      float* at = j % 2 ? reinterpret_cast<float*>(smem + j / 2 * Shape<D>::kRing)
                        : p.heads + ((int64_t)blockIdx.x * kWarps + j / 2) * P::kFloats;
#pragma unroll
      for (int k = 0; k < kWarps; ++k)  // (a place known at compile time: registers)
        if (k == count) part[k] = at;
      ++count;
      end = pieces[j / 2][j % 2].u1;
    }
    int last = i;  // a sequence's pieces are neighbours, but for warps without that piece
    for (int j = i; j < 2 * kWarps; ++j)
      if (pieces[j / 2][j % 2].bh == a.bh) last = j;
    i = last + 1;
    const bool done = a.u0 == 0 && end == a.units;
    float* into = done ? nullptr : p.partials + ((int64_t)blockIdx.x * 2 + (a.u0 > 0 ? 0 : 1)) * P::kFloats;
    join<T, D, ROWS>(p, a.bh / vh, a.bh % vh, count, part, into);
  }
}

// The groups of blocks, a block for each tile, that hold units of one (sequence, KV head), and the
// partials of one tile.
template <int D, int ROWS> struct Span {
  int c0, c1, tile, tiles;
  float* partials;
  __device__ __forceinline__ Span(const DecodeParams& p, int bh) : tile(bh % p.tiles), tiles(p.tiles), partials(p.partials) {
    const int2 s = p.warps ? make_int2(0, 0) : p.spans[bh];
    c0 = s.x;
    c1 = s.y;
  }
  __device__ __forceinline__ bool split() const { return c1 > c0; }
  // The first block's last run of units, the others' first.
  __device__ __forceinline__ float* part(int c) const {
    return partials + (((int64_t)c * tiles + tile) * 2 + (c > c0 ? 0 : 1)) * Partial<D, ROWS>::kFloats;
  }
};

// Maximum and sum of row r over a span's partials, by one warp.
template <int D, int ROWS>
__device__ __forceinline__ void span_stats(const Span<D, ROWS>& s, int r, int lane, float* m, float* l) {
  using P = Partial<D, ROWS>;
  float mm = -INFINITY, ll = 0.f;
  for (int c = s.c0 + lane; c <= s.c1; c += 32) {
    const float x = P::m(s.part(c))[r], y = P::l(s.part(c))[r], up = max_nan(mm, x), base = up == -INFINITY ? 0.f : up;
    ll = ll * fast_exp2(mm - base) + y * fast_exp2(x - base);
    mm = up;
  }
  float top = mm;
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
  ll *= fast_exp2(mm - (top == -INFINITY ? 0.f : top));
  for (int o = 16; o; o >>= 1) ll += __shfl_xor_sync(~0u, ll, o);
  *m = top;
  *l = ll;
}

// Adds partial (mi, li, oi) of a row to (m, l, acc).
template <int V>
__device__ __forceinline__ void join_row(float* m, float* l, float* acc, float mi, float li, const float* oi) {
  const float up = max_nan(*m, mi), base = up == -INFINITY ? 0.f : up;
  const float f = fast_exp2(*m - base), g = fast_exp2(mi - base);
  *m = up;
  *l = *l * f + li * g;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = acc[i] * f + oi[i] * g;
}

// After decode_kernel.  Blocks [0, joins) join the rows of sequences that span blocks, `share` warps a
// row.  Behind them, with weights_out, blocks of SLOTS slots of a (sequence, KV head):
//   weights_out = decay * weights + sum over the heads of exp2(stored score - log-sum-exp),
// with the log-sum-exp joined once more where it spans blocks, so that nothing waits for the joins.
template <typename T, int D, int ROWS, int SLOTS>
__global__ void __launch_bounds__(kThreads, 8)
finish_kernel(const __grid_constant__ DecodeParams p, int joins, int share, int weight_tiles) {
  using P = Partial<D, ROWS>;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, vh = p.c.n_kv_heads * p.tiles;
  if ((int)blockIdx.x < joins) {
    constexpr int V = D >= 32 ? D / 32 : 1;  // values of a lane
    __shared__ float sums[kWarps][D], stats[kWarps][2];
    const int at = blockIdx.x * (kWarps / share) + warp / share, bh = at / ROWS, r = at % ROWS, sub = warp % share;
    const int b = bh / vh, hv = bh % vh, row = hv % p.tiles * ROWS + r, head = hv / p.tiles * p.G + row;
    bool go = b < p.c.batch && row < p.G;
    const float sink = go && p.sinks ? p.sinks[head] * kLog2e : -INFINITY;
    sm100::pdl_wait();
    const Span<D, ROWS> s(p, go ? bh : 0);
    go = go && s.split();
    float m = -INFINITY, l = 0.f, acc[V] = {};
    const bool live = lane * V < D;
    constexpr int kAhead = 4;
    if (go)
      for (int c = s.c0 + sub; c <= s.c1; c += share * kAhead) {
        float mi[kAhead], li[kAhead], oi[kAhead][V];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const bool in = c + j * share <= s.c1;
          float* q = s.part(in ? c + j * share : c);
          mi[j] = in ? P::m(q)[r] : -INFINITY;
          li[j] = in ? P::l(q)[r] : 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) oi[j][i] = in && live ? P::o(q)[r * D + lane * V + i] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) join_row<V>(&m, &l, acc, mi[j], li[j], oi[j]);
      }
    if (share > 1) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (live) sums[warp][lane * V + i] = acc[i];
      if (lane == 0) stats[warp][0] = m, stats[warp][1] = l;
      __syncthreads();
    }
    if (!go || sub) return;
    for (int j = 1; j < share; ++j) {
      float other[V];
#pragma unroll
      for (int i = 0; i < V; ++i) other[i] = live ? sums[warp + j][lane * V + i] : 0.f;
      join_row<V>(&m, &l, acc, stats[warp + j][0], stats[warp + j][1], other);
    }
    const Row w = finish(m, l, sink);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (live) static_cast<T*>(p.o)[b * p.ob + head * p.oh + lane * V + i] = Pack<T>::from(acc[i] * w.inv);
    if (p.lse && lane == 0) p.lse[(int64_t)b * p.Hq + head] = w.lse;
    return;
  }
  const int at = blockIdx.x - joins, hk = at / weight_tiles % p.c.n_kv_heads, b = at / weight_tiles / p.c.n_kv_heads;
  const Sequence s = sequence(p, b);
  const int slot0 = at % weight_tiles * SLOTS;
  if (slot0 >= s.n) {
    sm100::pdl_wait();  // (every block waits: the grid is not over before the one that it follows)
    return;
  }
  constexpr int kPer = SLOTS / kThreads;
  __shared__ float shared_lse[ROWS];
  float w[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int slot = slot0 + i * kThreads + threadIdx.x;
    w[i] = slot < s.n ? old_weight(p, b, hk, slot) : 0.f;
  }
  sm100::pdl_wait();
  for (int tile = 0; tile < p.tiles; ++tile) {
    const int rows = p.G - tile * ROWS < ROWS ? p.G - tile * ROWS : ROWS, head0 = hk * p.G + tile * ROWS;
    const float* finished = p.lse + (int64_t)b * p.Hq + head0;
    if (tile) __syncthreads();
    const Span<D, ROWS> span(p, b * vh + hk * p.tiles + tile);
    if (!span.split()) {
      if ((int)threadIdx.x < ROWS) shared_lse[threadIdx.x] = (int)threadIdx.x < rows ? weight_base(finished[threadIdx.x]) : 0.f;
    } else {
      for (int r = warp; r < ROWS; r += kWarps) {
        float m = -INFINITY, l = 0.f;
        if (r < rows) span_stats(span, r, lane, &m, &l);
        if (lane == 0)
          shared_lse[r] = r < rows ? weight_base(finish(m, l, p.sinks ? p.sinks[head0 + r] * kLog2e : -INFINITY).lse) : 0.f;
      }
    }
    __syncthreads();
    float lse[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) lse[r] = shared_lse[r];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int slot = slot0 + i * kThreads + threadIdx.x;
      if (slot < s.n && (slot < s.sinks || slot >= s.first))
        w[i] += slot_weight<ROWS>(p, s, b * vh + hk * p.tiles + tile, slot, lse);
    }
  }
  if (is_bad(shared_lse[0])) return;  // (all tiles are, or none)
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int slot = slot0 + i * kThreads + threadIdx.x;
    if (slot < s.n) p.wout[b * p.wob + hk * p.woh + slot] = w[i];
  }
}

// What a call needs of the workspace, in floats each, every part a multiple of 64.
struct Plan {
  int rows, tiles, max_units, warps, blocks, weigh_here, weigh_slots;
  size_t lse, partials, heads, spans, scores;
};
size_t round64(size_t n) { return (n + 63) & ~(size_t)63; }

// Visible units up to which a (sequence, KV head) is one warp's or one block's, so that nothing is
// left to join, where there are enough of them to fill the GPU.  Measured with 8 KV heads of dim 64:
// 1 x 500 slots 7.6 us by block, 7.8 dealt out; 16 x 2100 20.7 and 24; 16 x 4200 35.6 and 33.7; 24 x 4200
// 42 and 44; 48 x 4200 66 and 76.  Longer ones are dealt out: their lengths may differ more.
constexpr int kUnitsWarp = 32, kUnitsBlock = 136, kSeqsBlock = 96, kUnitsMany = 264, kSeqsMany = 192;
// Slots of a table up to which whoever finishes a sequence writes its weights as well, instead of a
// second kernel with a thread a slot: 8 KV heads, 4 x 250 slots 7.2 us and 8.6, 48 x 250 10.6 and 11.0,
// 48 x 500 19.1 and 17.1; 100 x 60 by warps 7.5 and 9.0, 100 x 250 24 and 18.5.
constexpr int kWeighBlock = 256, kWeighWarp = 64;
// Slots of a block of finish_kernel's weights: few; but many where sequences span blocks, whose
// partials every block joins once more, and there are more than a wave of blocks or very long spans.
// 8 KV heads: one sequence of 4200 slots 13.0 us with 256 and 15.3 with 1024, 4 of 8400 27.1 and 27.4, 4 of
// 16000 43.1 and 41.3, one of 131072 89 and 70; 2 KV heads, 32000 slots 26.6 and 19.0.
constexpr int kFewSlots = 256, kManySlots = 1024;

Plan plan(const SwaPagedDecodeArgs& a) {
  const SwaPagedKV& c = a.cache;
  const int G = a.n_q_heads / c.n_kv_heads, D = c.head_dim;
  Plan r = {};
  r.rows = G <= 8 ? 8 : 16;
  r.tiles = (G + r.rows - 1) / r.rows;
  const int64_t cap = (int64_t)c.max_pages * c.page_size;
  int64_t units = (cap + kUnit - 1) / kUnit;
  const int64_t w = a.window_size > 0 ? a.window_size : 0;
  // the sinks' units, the window's, and one more where it begins inside a unit
  const int64_t bound = ((int64_t)a.sink_size + kUnit - 1) / kUnit + (w + kUnit - 1) / kUnit + 1;
  if (bound < units) units = bound;
  r.max_units = units > 0 ? (int)units : 1;
  const int64_t seqs = (int64_t)c.batch * c.n_kv_heads * r.tiles;
  const int most = D == 128 ? Shape<128>::kMaxBlocks : Shape<64>::kMaxBlocks;
  if (r.max_units <= kUnitsWarp) r.warps = seqs >= most ? 1 : kWarps;
  else if (r.max_units <= kUnitsBlock && seqs >= kSeqsBlock) r.warps = kWarps;
  else if (r.max_units <= kUnitsMany && seqs >= kSeqsMany) r.warps = kWarps;
  if (r.warps) {
    r.blocks = (int)((seqs * r.warps + kWarps - 1) / kWarps);
  } else {
    const int64_t want = ((int64_t)c.batch * c.n_kv_heads * r.max_units + 2 * kWarps - 1) / (2 * kWarps);
    const int64_t groups = most > r.tiles ? most / r.tiles : 1;
    r.blocks = (int)(want < groups ? want : groups) * r.tiles;
  }
  // whoever finishes a short sequence writes its weights too: no second kernel
  r.weigh_here = a.weights_out && r.tiles == 1 && cap <= (r.warps == 1 ? kWeighWarp : r.warps ? kWeighBlock : 0);
  const int64_t weigh_blocks = (cap + kFewSlots - 1) / kFewSlots * c.batch * c.n_kv_heads;
  r.weigh_slots = r.warps || (weigh_blocks <= 8 * kSms && r.blocks <= 128 * seqs) ? kFewSlots : kManySlots;
  const size_t part = (size_t)r.rows * (D + 2);
  r.lse = a.weights_out && !a.lse ? round64((size_t)c.batch * a.n_q_heads) : 0;
  r.partials = r.warps ? 0 : round64(2 * part * r.blocks);
  r.heads = r.warps ? 0 : round64(kWarps * part * r.blocks);
  r.spans = r.warps ? 0 : round64(2 * (size_t)seqs);
  r.scores = a.weights_out ? round64((size_t)seqs * r.max_units * r.rows * kUnit) : 0;
  return r;
}

template <typename T, int D, int ROWS, bool WEIGH>
cudaError_t launch_decode(const DecodeParams& p, int blocks, cudaStream_t st) {
  constexpr int smem = kWarps * Shape<D>::kRing;
  auto kern = decode_kernel<T, D, ROWS, WEIGH>;
  cudaError_t e = allow_smem<Walk<T, D, ROWS, WEIGH>>(kern, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, (unsigned)blocks, kThreads, smem, st, p);
}

template <typename T, int D, int ROWS>
cudaError_t launch(const DecodeParams& p, const Plan& pl, cudaStream_t st) {
  cudaError_t e = p.wout ? launch_decode<T, D, ROWS, true>(p, pl.blocks, st) : launch_decode<T, D, ROWS, false>(p, pl.blocks, st);
  if (e != cudaSuccess) return e;
  // four warps a row where the rows alone do not fill the GPU and their spans are long: one sequence of
  // 2100 slots 8.8 us so, 9.8 with one warp a row; a ragged batch of 32 97 and 95
  const int64_t rows = (int64_t)p.c.batch * p.c.n_kv_heads * p.tiles * ROWS;
  const int share = rows <= kSms * 8 ? kWarps : 1;
  const int64_t joins = p.warps ? 0 : (rows * share + kWarps - 1) / kWarps;
  const int64_t slots = (int64_t)p.c.max_pages * p.c.page_size;
  const int64_t tiles = p.wout && !p.weigh_here ? (slots + pl.weigh_slots - 1) / pl.weigh_slots : 0;
  const int64_t blocks = joins + tiles * p.c.n_kv_heads * p.c.batch;
  if (blocks == 0) return cudaSuccess;
  return launch_pdl(pl.weigh_slots == kFewSlots ? finish_kernel<T, D, ROWS, kFewSlots> : finish_kernel<T, D, ROWS, kManySlots>,
                    (unsigned)blocks, kThreads, 0, st, p, (int)joins, share, (int)tiles);
}

template <typename T, int ROWS>
cudaError_t launch_dim(int D, const DecodeParams& p, const Plan& pl, cudaStream_t st) {
  switch (D) {
    case 16: return launch<T, 16, ROWS>(p, pl, st);
    case 32: return launch<T, 32, ROWS>(p, pl, st);
    case 64: return launch<T, 64, ROWS>(p, pl, st);
    default: return launch<T, 128, ROWS>(p, pl, st);
  }
}

}  // namespace

size_t paged_decode_workspace(const SwaPagedDecodeArgs& a) {
  const Plan r = plan(a);
  return (r.lse + r.partials + r.heads + r.spans + r.scores) * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedParams& c, const SwaPagedDecodeArgs& a, cudaStream_t st) {
  const Plan pl = plan(a);
  DecodeParams p;
  p.c = c;
  p.Hq = a.n_q_heads; p.G = a.n_q_heads / c.n_kv_heads; p.tiles = pl.tiles;
  p.W = a.window_size; p.S = a.sink_size;
  p.units_per_page = c.page_size / kUnit;
  p.max_units = pl.max_units; p.warps = pl.warps;
  p.scale_log2 = a.softmax_scale * kLog2e;
  p.q = a.q.ptr; p.o = a.o.ptr;
  p.qb = a.q.stride_t; p.qh = a.q.stride_h; p.ob = a.o.stride_t; p.oh = a.o.stride_h;
  float* ws = static_cast<float*>(a.workspace);
  p.lse = a.lse ? a.lse : pl.lse ? ws : nullptr;
  p.partials = ws + pl.lse;
  p.heads = p.partials + pl.partials;
  p.spans = reinterpret_cast<int2*>(p.heads + pl.heads);
  p.scores = pl.scores ? p.heads + pl.heads + pl.spans : nullptr;
  p.sinks = a.sink_logits;
  p.wout = a.weights_out; p.wob = a.wo_stride_b; p.woh = a.wo_stride_h;
  p.decay = a.decay;
  p.weigh_here = pl.weigh_here;
  if (a.cache.dtype == SWA_F16)
    return pl.rows == 8 ? launch_dim<__half, 8>(a.cache.head_dim, p, pl, st) : launch_dim<__half, 16>(a.cache.head_dim, p, pl, st);
  return pl.rows == 8 ? launch_dim<__nv_bfloat16, 8>(a.cache.head_dim, p, pl, st)
                      : launch_dim<__nv_bfloat16, 16>(a.cache.head_dim, p, pl, st);
}

}  // namespace swa
