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

}  // namespace
}  // namespace b200tbe

using namespace b200tbe;

extern "C" int b200tbe_jagged_attention(const b200tbe_attention_params* p, b200tbe_stream_t stream_) {
  const int st = check_forward(p);
  if (st != B200TBE_OK) return st;
  if (p->total_q == 0) return B200TBE_OK;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const AttnDev d = device_params(p);
  if (attention_forward_fits(d, p->dtype)) {
    const int tc = attention_forward_tc(d, p->dtype, p->status, stream);
    if (tc != B200TBE_ERR_UNSUPPORTED) return tc;
  }
  return attention_forward_simt(d, p->dtype, stream);
}

namespace {

size_t rounded(size_t n) { return (n + 15) / 16 * 16; }

// delta, then the tickets and counts, then the two lists
struct BackwardScratch {
  size_t delta, words, q_tiles, k_tiles;
  size_t total() const { return delta + words + q_tiles + k_tiles; }
};

BackwardScratch scratch_of(int64_t total_q, int64_t total_k, int64_t batch, int64_t heads) {
  BackwardScratch s;
  s.delta = rounded(static_cast<size_t>(total_q) * heads * sizeof(float));
  s.words = 16;
  s.q_tiles = rounded(static_cast<size_t>(tile_slots<128>(total_q, batch)) * sizeof(int2));
  s.k_tiles = rounded(static_cast<size_t>(tile_slots<128>(total_k, batch)) * sizeof(int2));
  return s;
}

}  // namespace

extern "C" size_t b200tbe_jagged_attention_backward_scratch_bytes(int64_t total_q, int64_t total_k, int32_t batch,
                                                                  int32_t heads) {
  if (total_q < 0 || total_k < 0 || batch < 0 || heads <= 0) return 0;
  return scratch_of(total_q, total_k, batch, heads).total();
}

extern "C" int b200tbe_jagged_attention_backward(const b200tbe_attention_backward_params* p, b200tbe_stream_t stream_) {
  if (p == nullptr) return B200TBE_ERR_BAD_ARG;
  const b200tbe_attention_params* f = &p->forward;
  int st = check_forward(f);
  if (st != B200TBE_OK) return st;
  if (f->total_q > 0 && (p->grad_out == nullptr || f->lse == nullptr || p->grad_q == nullptr)) return B200TBE_ERR_BAD_ARG;
  if (f->total_k > 0 && (p->grad_k == nullptr || p->grad_v == nullptr)) return B200TBE_ERR_BAD_ARG;
  const BackwardScratch s = scratch_of(f->total_q, f->total_k, f->batch, f->heads);
  if (p->scratch == nullptr || p->scratch_bytes < s.total() || !aligned_to(p->scratch, 16)) return B200TBE_ERR_SCRATCH;
  if (f->total_q == 0 && f->total_k == 0) return B200TBE_OK;
  AttnDev d = device_params(f);
  d.grad = p->grad_out, d.dq = p->grad_q, d.dk = p->grad_k, d.dv = p->grad_v, d.delta = static_cast<float*>(p->scratch);
  d.g_row = p->grad_out_stride, d.g_head = p->grad_out_head_stride, d.dq_row = p->grad_q_stride, d.dq_head = p->grad_q_head_stride;
  d.dk_row = p->grad_k_stride, d.dk_head = p->grad_k_head_stride, d.dv_row = p->grad_v_stride, d.dv_head = p->grad_v_head_stride;
  char* at = static_cast<char*>(p->scratch) + s.delta;
  BackwardPlan plan;
  plan.tickets = reinterpret_cast<int32_t*>(at);
  plan.counts = plan.tickets + 2;
  plan.q_tiles = reinterpret_cast<int2*>(at + s.words);
  plan.k_tiles = reinterpret_cast<int2*>(at + s.words + s.q_tiles);
  plan.q_room = static_cast<int32_t>(tile_slots<128>(f->total_q, f->batch));
  plan.k_room = static_cast<int32_t>(tile_slots<128>(f->total_k, f->batch));
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  st = attention_delta(d, plan, f->dtype, stream);
  if (st != B200TBE_OK) return st;
  if (attention_backward_fits(d, f->dtype)) {
    const int tc = attention_backward_tc(d, plan, f->dtype, f->status, stream);
    if (tc != B200TBE_ERR_UNSUPPORTED) return tc;
  }
  return attention_backward_simt(d, f->dtype, stream);
}
