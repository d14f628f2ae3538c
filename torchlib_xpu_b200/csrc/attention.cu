// C entry points of the jagged attention: argument checks and the choice of kernels.
#include "attention.cuh"

namespace b200tbe {
namespace {

constexpr int kMaxHeadDim = 256;

int check_forward(const b200tbe_attention_params* p) {
  if (p == nullptr) return B200TBE_ERR_BAD_ARG;
  if (p->dtype != B200TBE_FP32 && p->dtype != B200TBE_FP16 && p->dtype != B200TBE_BF16) return B200TBE_ERR_UNSUPPORTED;
  if (p->head_dim < 1 || p->head_dim > kMaxHeadDim) return B200TBE_ERR_UNSUPPORTED;
  if (p->offset_bytes != 4 && p->offset_bytes != 8) return B200TBE_ERR_UNSUPPORTED;
  if (p->batch < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0 || p->total_q < 0 || p->total_k < 0)
    return B200TBE_ERR_BAD_ARG;
  // places inside a sequence are 32-bit, and so are grids
  if (p->total_q > 0x7fffff00ll || p->total_k > 0x7fffff00ll || p->batch > 0x7fffff00) return B200TBE_ERR_TOO_LARGE;
  if ((p->total_q > 0 || p->total_k > 0) && (p->q_offsets == nullptr || p->k_offsets == nullptr)) return B200TBE_ERR_BAD_ARG;
  if (p->total_q > 0 && (p->q == nullptr || p->out == nullptr)) return B200TBE_ERR_BAD_ARG;
  if (p->total_k > 0 && (p->k == nullptr || p->v == nullptr)) return B200TBE_ERR_BAD_ARG;
  return B200TBE_OK;
}

AttnDev device_params(const b200tbe_attention_params* p) {
  AttnDev d{};
  d.q = p->q, d.k = p->k, d.v = p->v, d.out = p->out, d.lse = p->lse;
  d.q_offsets = p->q_offsets, d.k_offsets = p->k_offsets;
  d.q_row = p->q_stride, d.q_head = p->q_head_stride, d.k_row = p->k_stride, d.k_head = p->k_head_stride;
  d.v_row = p->v_stride, d.v_head = p->v_head_stride, d.o_row = p->out_stride, d.o_head = p->out_head_stride;
  d.total_q = p->total_q, d.total_k = p->total_k;
  d.batch = p->batch, d.heads = p->heads, d.kv_heads = p->kv_heads, d.group = p->heads / p->kv_heads, d.D = p->head_dim;
  d.offset_bytes = p->offset_bytes, d.causal = p->causal, d.scale = p->scale;
  return d;
}

size_t rounded(size_t n) { return (n + 15) / 16 * 16; }

// delta, then the list's tickets and counts, the norms (of gradients and of values), then the two lists
struct Scratch {
  size_t delta, words, norms, q_tiles, k_tiles;
  size_t total() const { return delta + words + 2 * norms + q_tiles + k_tiles; }
};

Scratch backward_scratch(int64_t total_q, int64_t total_k, int64_t batch, int64_t heads) {
  Scratch s;
  s.delta = rounded(static_cast<size_t>(total_q) * heads * sizeof(float));
  s.words = 16;
  s.norms = rounded((static_cast<size_t>(batch) + 2) * heads * sizeof(uint32_t));
  s.q_tiles = rounded(static_cast<size_t>(tile_slots<128>(total_q, batch)) * sizeof(int2));
  s.k_tiles = rounded(static_cast<size_t>(tile_slots<128>(total_k, batch)) * sizeof(int2));
  return s;
}

TileList list_at(char* at, const Scratch& s, int64_t total_q, int64_t total_k, int64_t batch) {
  TileList list;
  list.tickets = reinterpret_cast<int32_t*>(at);
  list.counts = list.tickets + 2;
  list.grad_norms = reinterpret_cast<uint32_t*>(at + s.words);
  list.v_norms = reinterpret_cast<uint32_t*>(at + s.words + s.norms);
  list.q_tiles = reinterpret_cast<int2*>(at + s.words + 2 * s.norms);
  list.k_tiles = reinterpret_cast<int2*>(at + s.words + 2 * s.norms + s.q_tiles);
  list.q_room = static_cast<int32_t>(tile_slots<128>(total_q, batch));
  list.k_room = static_cast<int32_t>(tile_slots<128>(total_k, batch));
  return list;
}

// Batches whose sequences are at most 128 long on average go through the short sequences' kernels first. There
// the general kernels' CTAs, one or two an SM, would each spend most of a sequence's time waiting: 4096 sequences
// of 0 to 128 positions, 4 heads of 64, bf16, causal, take 141 us forward and 418 backward with, 255 and 1351 without. The two
// meet later the fewer query heads a key head has, and never far below 128 on average (forward + backward, with against without):
//   sequences    positions   4 heads of 64           4 heads of 128          8 heads of 128 over 1 key head
//   1024 (512)   0 to 256    136 + 544, 227 + 596    170 + 746, 249 + 845    167 + 571, 164 + 562 (half as many sequences)
//   512          0 to 512    160 + 601, 206 + 585    175 + 802, 245 + 801    175 + 639, 165 + 553 (256)
//   1024 (512)   128         60 + 141, 82 + 386      96 + 241, 103 + 608     85 + 194, 109 + 413
//   2048 (1024)  0 to 128    79 + 223, 135 + 680     129 + 339, 166 + 951    126 + 295, 181 + 626
bool mostly_short(const AttnDev& d) {
  return d.batch > 0 && d.total_q <= static_cast<int64_t>(d.batch) * 128 && d.total_k <= static_cast<int64_t>(d.batch) * 128;
}
// Several waves of tiles of sequences of different lengths: sorted first (5 to 8 us), so that the longest are not the
// last. 96 batches of up to 200 queries and 1500 keys, 6 heads of 80: 77 us unsorted, 60 with the sorting.
bool listed_first(const AttnDev& d) {
  const bool by_rows = d.group % 2 != 0 && d.total_q > static_cast<int64_t>(d.batch) * 128;   // tiles of 256, which no list has
  return d.batch > 1 && !by_rows && (d.total_q / 128 + d.batch) * d.heads > 2 * kNumSMs;
}
// ... and here nothing can be longer.
bool all_short(const AttnDev& d) { return d.total_q <= 128 && d.total_k <= 128; }

}  // namespace
}  // namespace b200tbe

using namespace b200tbe;

extern "C" size_t b200tbe_jagged_attention_scratch_bytes(int64_t total_q, int32_t batch) {
  if (total_q < 0 || batch < 0) return 0;
  const Scratch s = backward_scratch(total_q, 0, batch, 0);
  return s.words + s.q_tiles;
}

extern "C" int b200tbe_jagged_attention(const b200tbe_attention_params* p, b200tbe_stream_t stream_) {
  const int st = check_forward(p);
  if (st != B200TBE_OK) return st;
  if (p->scratch != nullptr && (!aligned_to(p->scratch, 16) ||
                                p->scratch_bytes < b200tbe_jagged_attention_scratch_bytes(p->total_q, p->batch)))
    return B200TBE_ERR_SCRATCH;
  if (p->total_q == 0) return B200TBE_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const AttnDev d = device_params(p);
  if (attention_forward_fits(d, p->dtype)) {
    const TileList* rest = nullptr;
    TileList list;
    int tc = B200TBE_ERR_UNSUPPORTED;
    if ((p->scratch != nullptr || all_short(d)) && mostly_short(d)) {
      if (p->scratch != nullptr)
        list = list_at(static_cast<char*>(p->scratch), backward_scratch(d.total_q, 0, d.batch, 0), d.total_q, 0, d.batch);
      else
        list = TileList{};   // nothing goes on it
      if (!all_short(d) && cudaMemsetAsync(p->scratch, 0, 16, stream) != cudaSuccess) return B200TBE_ERR_LAUNCH;
      tc = attention_short_forward(d, list, p->dtype, p->status, stream);
      if (tc == B200TBE_OK && all_short(d)) return tc;
      if (tc == B200TBE_OK) rest = &list;
      if (tc != B200TBE_OK && tc != B200TBE_ERR_UNSUPPORTED) return tc;
    } else if (p->scratch != nullptr && listed_first(d)) {
      list = list_at(static_cast<char*>(p->scratch), backward_scratch(d.total_q, 0, d.batch, 0), d.total_q, 0, d.batch);
      list.k_room = 0;
      tc = attention_list(d, list, stream);
      if (tc != B200TBE_OK) return tc;
      rest = &list;
    }
    tc = attention_forward_tc(d, rest, p->dtype, p->status, stream);
    if (tc != B200TBE_ERR_UNSUPPORTED) return tc;
  }
  return attention_forward_simt(d, p->dtype, stream);
}

extern "C" size_t b200tbe_jagged_attention_backward_scratch_bytes(int64_t total_q, int64_t total_k, int32_t batch,
                                                                  int32_t heads) {
  if (total_q < 0 || total_k < 0 || batch < 0 || heads <= 0) return 0;
  return backward_scratch(total_q, total_k, batch, heads).total();
}

extern "C" int b200tbe_jagged_attention_backward(const b200tbe_attention_backward_params* p, b200tbe_stream_t stream_) {
  if (p == nullptr) return B200TBE_ERR_BAD_ARG;
  const b200tbe_attention_params* f = &p->forward;
  int st = check_forward(f);
  if (st != B200TBE_OK) return st;
  if (f->total_q > 0 && (p->grad_out == nullptr || f->lse == nullptr || p->grad_q == nullptr)) return B200TBE_ERR_BAD_ARG;
  if (f->total_k > 0 && (p->grad_k == nullptr || p->grad_v == nullptr)) return B200TBE_ERR_BAD_ARG;
  const Scratch s = backward_scratch(f->total_q, f->total_k, f->batch, f->heads);
  if (p->scratch == nullptr || p->scratch_bytes < s.total() || !aligned_to(p->scratch, 16)) return B200TBE_ERR_SCRATCH;
  if (f->total_q == 0 && f->total_k == 0) return B200TBE_OK;
  AttnDev d = device_params(f);
  d.grad = p->grad_out, d.dq = p->grad_q, d.dk = p->grad_k, d.dv = p->grad_v, d.delta = static_cast<float*>(p->scratch);
  d.g_row = p->grad_out_stride, d.g_head = p->grad_out_head_stride, d.dq_row = p->grad_q_stride, d.dq_head = p->grad_q_head_stride;
  d.dk_row = p->grad_k_stride, d.dk_head = p->grad_k_head_stride, d.dv_row = p->grad_v_stride, d.dv_head = p->grad_v_head_stride;
  const TileList list = list_at(static_cast<char*>(p->scratch) + s.delta, s, f->total_q, f->total_k, f->batch);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  bool fits = attention_backward_fits(d, f->dtype);
  const bool ranged = fits && f->dtype == B200TBE_FP16;   // the general kernels need the norms
  const size_t cleared = s.words + (ranged ? 2 * s.norms : 0);
  if (fits && !all_short(d) && (ranged || mostly_short(d)) && cudaMemsetAsync(list.tickets, 0, cleared, stream) != cudaSuccess)
    return B200TBE_ERR_LAUNCH;
  bool listed = false;
  if (fits && mostly_short(d)) {
    st = attention_short_backward(d, list, f->dtype, f->status, stream);
    if (st == B200TBE_OK && all_short(d)) return st;
    if (st != B200TBE_OK && st != B200TBE_ERR_UNSUPPORTED) return st;
    listed = st == B200TBE_OK;
    fits = listed;   // the general kernels make the same tensor maps
  }
  if (ranged && fits && !listed) {
    st = attention_list(d, list, stream);
    if (st != B200TBE_OK) return st;
    listed = true;
  }
  st = listed ? attention_delta_listed(d, list, f->dtype, stream) : attention_delta(d, list, f->dtype, stream);
  if (st != B200TBE_OK) return st;
  if (fits) {
    st = attention_backward_tc(d, list, f->dtype, f->status, stream);
    if (st != B200TBE_ERR_UNSUPPORTED) return st;
    if (listed) {   // the 32-bit kernels take every row
      st = attention_delta(d, list, f->dtype, stream);
      if (st != B200TBE_OK) return st;
    }
  }
  return attention_backward_simt(d, f->dtype, stream);
}
