// swa_paged.cuh -- parameter blocks and device helpers of the rotary and paged-cache kernels.
#pragma once

#include "swa_common.cuh"
#include "swa_params.cuh"

namespace swa {

struct RotaryParams {
  const float* inv_freq;
  const void* positions;
  int64_t ps_axis, ps_b, ps_l;
  int pos_is_64, n_freq, interleaved;
  float scale;
  uint8_t axis[SWA_ROTARY_MAX_FREQS];
};

struct PagedParams {
  void* k;
  void* v;
  int64_t kp, kh, kr, vp, vh, vr;  // element strides of page, head, row
  const int32_t* table;
  int64_t table_stride;
  int32_t* seq_lens;
  const int32_t* seen;  // never null: seq_lens where the caller gave none
  float* weights;
  int32_t* positions;
  int64_t wb, wh, pb, ph;
  int n_pages, page_size, max_pages, batch, n_kv_heads;
  int* page_error;
};

// Slots of sequence b in use, cut to what its table can hold; *bad is set where it held more.
__device__ __forceinline__ int paged_len(const PagedParams& c, int b, bool* bad) {
  const int n = c.seq_lens[b], cap = c.max_pages * c.page_size;
  if (n > cap) {
    *bad = true;
    return cap;
  }
  return n < 0 ? 0 : n;
}

// The page of a slot, or -1 (and *bad) where the table's entry is out of range.
__device__ __forceinline__ int paged_page(const PagedParams& c, int b, int table_col, bool* bad) {
  const int p = c.table[(int64_t)b * c.table_stride + table_col];
  if (static_cast<unsigned>(p) >= static_cast<unsigned>(c.n_pages)) {
    *bad = true;
    return -1;
  }
  return p;
}

// The slots that the newest of n tokens sees: the sinks [0, sinks) that lie before its window,
// then the window [first, n).
struct VisibleSlots {
  int sinks, first;
};
__host__ __device__ __forceinline__ VisibleSlots visible_slots(int n, int W, int S) {
  VisibleSlots r;
  r.first = W >= n ? 0 : (W > 0 ? n - W : n);
  r.sinks = S < r.first ? S : r.first;
  return r;
}

// cos and sin (times scale) of position * inv_freq.  The product in 64 bits: at position 2^17 a
// 32-bit product would be off by up to 2^-8 rad; in 64 bits the angle, in turns, is exact to
// about 2^-53 of itself, and what is left of whole turns is small enough for 32 bits.
__device__ __forceinline__ void rotary_cos_sin(const RotaryParams& r, int64_t b, int64_t l, int i, float* c,
                                               float* s) {
  const int64_t at = r.axis[i] * r.ps_axis + b * r.ps_b + l * r.ps_l;
  const double pos = r.pos_is_64 ? (double)static_cast<const int64_t*>(r.positions)[at]
                                 : (double)static_cast<const int32_t*>(r.positions)[at];
  const double half_turns = pos * (double)r.inv_freq[i] * 0.31830988618379067154;  // 1 / pi
  const double rest = half_turns - 2.0 * rint(0.5 * half_turns);
  float sn, cs;
  sincospif((float)rest, &sn, &cs);
  *c = cs * r.scale;
  *s = sn * r.scale;
}

}  // namespace swa
