// What the jagged attention kernels share: their parameters, and where a CTA's rows lie.
#pragma once

#include "common.cuh"

namespace b200tbe {

struct AttnDev {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;              // [heads][total_q], or null in a forward pass that keeps nothing
  const void* q_offsets;   // [batch + 1]
  const void* k_offsets;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;   // strides in elements
  int64_t total_q, total_k;
  int32_t batch, heads, kv_heads, group, D;
  int32_t offset_bytes;
  int32_t causal;
  int32_t fours;   // of the 32-bit kernels: operands may be read in fours of elements
  float scale;
  // backward
  const void* grad;
  void* dq;
  void* dk;
  void* dv;
  float* delta;            // [heads][total_q]
  int64_t g_row, g_head, dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
};

// Tiles of 128 rows, of queries and of keys, listed in the caller's scratch as (stretch, tile inside it) by the delta
// kernel (all of them) or by the short sequences' kernels (what they leave). The tickets say how many of them (times
// heads) are taken.
struct TileList {
  int32_t* tickets;   // [2]
  int32_t* counts;    // [2]
  int2* q_tiles;
  int2* k_tiles;
  int32_t q_room, k_room;
  // of an fp16 backward pass, zero before: the largest |dO|^2 of a stretch's rows [batch + 2][heads], the largest |v|^2
  // [batch + 2][kv_heads], as the bits of floats (which compare as they do)
  uint32_t* grad_norms;
  uint32_t* v_norms;
};

int attention_forward_simt(const AttnDev& p, int dtype, cudaStream_t stream);
int attention_backward_simt(const AttnDev& p, int dtype, cudaStream_t stream);
// Tensor-core kernels: whether they take these arguments, and the launches. B200TBE_ERR_UNSUPPORTED from a
// launch (nothing was enqueued): the driver made no tensor map of them, the 32-bit kernels take over.
bool attention_forward_fits(const AttnDev& p, int dtype);
int attention_forward_tc(const AttnDev& p, const TileList* list, int dtype, int32_t* status, cudaStream_t stream);
// Sequences of at most 128 queries and keys; the others' tiles go on the list (whose words are zero before).
int attention_short_forward(const AttnDev& p, const TileList& list, int dtype, int32_t* status, cudaStream_t stream);
int attention_short_backward(const AttnDev& p, const TileList& list, int dtype, int32_t* status, cudaStream_t stream);
// All tiles, the long sequences' first, as attention_delta() lists them. With k_room 0, of the queries alone.
int attention_list(const AttnDev& p, const TileList& list, cudaStream_t stream);
// delta of the listed tiles; in fp16 their norms too.
int attention_delta_listed(const AttnDev& p, const TileList& list, int dtype, cudaStream_t stream);
bool attention_backward_fits(const AttnDev& p, int dtype);
int attention_backward_tc(const AttnDev& p, const TileList& plan, int dtype, int32_t* status, cudaStream_t stream);
int attention_delta(const AttnDev& p, const TileList& plan, int dtype, cudaStream_t stream);

// One sequence's rows on both sides, or a stretch of rows that no sequence owns (klen 0).
struct SeqRange {
  int64_t q0, k0;
  int32_t qlen, klen;
};

__device__ __forceinline__ int64_t clamped_offset(const void* offsets, int32_t offset_bytes, int64_t i, int64_t total) {
  const int64_t o = offset_bytes == 8 ? load_index<int64_t>(offsets, i) : load_index<int32_t>(offsets, i);
  return o < 0 ? 0 : (o > total ? total : o);
}

// The rows [0, total) in batch + 2 stretches: what lies before the first sequence, the sequences, and
// what lies behind the last. Stretch i begins at bound(i).
__device__ __forceinline__ int64_t stretch_bound(const void* offsets, int32_t offset_bytes, int32_t batch, int64_t total,
                                                 int32_t i) {
  if (i <= 0) return 0;
  if (i > batch + 1) return total;
  return clamped_offset(offsets, offset_bytes, i - 1, total);
}

// Tiles without a plan: stretch i's tiles of kRows rows take the slots from bound(i) / kRows + i on. That
// base grows by at least as many slots as the stretch has tiles, whatever the lengths, so the grid (total /
// kRows + batch + 2) is known on the host, at most one slot per stretch stays empty, and a CTA finds its
// stretch with one search over the offsets. Called by a whole warp; false: the slot is empty.
// *first is the tile's first row inside its stretch, *stretch its number (0 and batch + 1: no sequence).
template <int kRows>
__device__ __forceinline__ bool find_tile(const void* offsets, int32_t offset_bytes, int32_t batch, int64_t total,
                                          int64_t slot, int32_t* stretch, int64_t* begin, int64_t* first, int64_t* end) {
  int32_t lo = 0, n = batch + 2;   // the last stretch whose base is at most slot lies in [lo, lo + n)
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int32_t step = (n + 31) / 32;
    const int32_t i = lo + lane * step;
    const bool ok = lane * step < n &&
                    stretch_bound(offsets, offset_bytes, batch, total, i) / kRows + i <= slot;
    const unsigned votes = __ballot_sync(kFullMask, ok);
    const int32_t at = 31 - __clz(votes | 1u);
    lo += at * step;
    n = min(step, n - at * step);
  }
  *stretch = lo;
  *begin = stretch_bound(offsets, offset_bytes, batch, total, lo);
  *end = stretch_bound(offsets, offset_bytes, batch, total, lo + 1);
  *first = (slot - (*begin / kRows + lo)) * kRows;
  return *first >= 0 && *begin + *first < *end;
}

template <int kRows>
inline int64_t tile_slots(int64_t total, int64_t batch) { return total / kRows + batch + 2; }

// The rows of the other side that go with stretch i.
__device__ __forceinline__ void other_rows(const void* offsets, int32_t offset_bytes, int32_t batch, int64_t total,
                                           int32_t stretch, int64_t* begin, int32_t* len) {
  if (stretch < 1 || stretch > batch) {
    *begin = 0;
    *len = 0;
    return;
  }
  *begin = clamped_offset(offsets, offset_bytes, stretch - 1, total);
  const int64_t e = clamped_offset(offsets, offset_bytes, stretch, total);
  *len = e > *begin ? static_cast<int32_t>(e - *begin) : 0;
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace b200tbe
