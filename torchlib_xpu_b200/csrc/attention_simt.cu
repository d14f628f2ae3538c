// Jagged attention in 32-bit arithmetic: every type, head dimension up to 256, any strides.
//
//   S = scale q k^T over the keys a query sees, P = exp(S - m) / l, O = P v
//   dV = P^T dO,  dP = dO v^T,  dS = P (dP - rowsum(dO O)),  dQ = scale dS k,  dK = scale dS^T q
//
// A CTA of 256 threads takes a tile of kT rows of one head (queries in the forward pass and for dQ, keys for
// dK and dV) and walks the other side in tiles of kT. Operands lie in shared memory as fp32, transposed
// ([d][row]), so that a step over d is two 16-byte reads for kR x kR products of a thread; the running maximum
// and sum of a row stay in the registers of the sixteen threads that share it. Bound by the shared-memory reads that
// feed the fp32 pipe (77 % of their rate; 48 sequences of 1 to 257 positions, 4 heads of 32, fp32: forward 46 us, dQ 56, dK
// and dV 78). Nothing is added across CTAs: the results do not depend on scheduling.
// A query that sees no key has output 0, log-sum -infinity and no part in any gradient.
#include "attention.cuh"

namespace b200tbe {
namespace {

constexpr int kThreads = 256;

// Tile rows, products of a thread a side, and the padded row of a transposed operand.
template <int kDP>
struct Shape {
  static constexpr int kT = kDP <= 128 ? 64 : 32;
  static constexpr int kR = kT / 16;
  static constexpr int kPad = kT + 4;
  static constexpr int kC = kDP / 16;   // output columns of a thread
  static constexpr int kOperand = kDP * kPad;   // floats of a transposed operand, of a tile of weights
  static constexpr int kWeights = kT * kPad;
};

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&x);
    return make_float4(to_float<T>(e[0]), to_float<T>(e[1]), to_float<T>(e[2]), to_float<T>(e[3]));
  }
}

// rows [first, first + kT) of one head into dst[d][row]; rows at or past `rows` and columns past D are zero. Lanes
// take consecutive rows: the stores meet no bank twice, and what a row's other lanes want next is in L1.
template <typename T, int kDP>
__device__ __forceinline__ void load_transposed(float* dst, const T* src, int64_t row_stride, int first, int rows, int D, bool fours) {
  using S = Shape<kDP>;
  if (fours) {   // D, strides and addresses are whole fours of elements
    constexpr int kEach = S::kT * kDP / 4 / kThreads;
    float4 x[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int i = u * kThreads + threadIdx.x, r = i % S::kT, d = i / S::kT * 4;
      x[u] = d < D && first + r < rows ? load4(src + static_cast<int64_t>(first + r) * row_stride + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int i = u * kThreads + threadIdx.x, r = i % S::kT, d = i / S::kT * 4;
      float* to = dst + d * S::kPad + r;
      to[0] = x[u].x, to[S::kPad] = x[u].y, to[2 * S::kPad] = x[u].z, to[3 * S::kPad] = x[u].w;
    }
    return;
  }
  for (int i = threadIdx.x; i < S::kT * kDP; i += kThreads) {
    const int r = i % S::kT, d = i / S::kT;
    dst[d * S::kPad + r] = d < D && first + r < rows ? to_float<T>(src[static_cast<int64_t>(first + r) * row_stride + d]) : 0.f;
  }
}

// acc[a][b] += sum over d of x[d][ty*kR + a] * y[d][tx*kR + b]
template <int kDP>
__device__ __forceinline__ void products(float (&acc)[Shape<kDP>::kR][Shape<kDP>::kR], const float* x, const float* y,
                                         int tx, int ty) {
  using S = Shape<kDP>;
#pragma unroll 4
  for (int d = 0; d < kDP; ++d) {
    float a[S::kR], b[S::kR];
    if constexpr (S::kR == 4) {
      *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(x + d * S::kPad + ty * 4);
      *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(y + d * S::kPad + tx * 4);
    } else {
      *reinterpret_cast<float2*>(a) = *reinterpret_cast<const float2*>(x + d * S::kPad + ty * 2);
      *reinterpret_cast<float2*>(b) = *reinterpret_cast<const float2*>(y + d * S::kPad + tx * 2);
    }
#pragma unroll
    for (int i = 0; i < S::kR; ++i)
#pragma unroll
      for (int j = 0; j < S::kR; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
  }
}

// acc[a][c] += sum over t of w[t][ty*kR + a] * y[c*16 + tx][t]   (w: weights of the tile, t along the other side)
template <int kDP>
__device__ __forceinline__ void accumulate(float (&acc)[Shape<kDP>::kR][Shape<kDP>::kC], const float* w, const float* y,
                                           int tx, int ty) {
  using S = Shape<kDP>;
#pragma unroll 2
  for (int t = 0; t < S::kT; t += 4) {
    float a[4][S::kR];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* from = w + (t + u) * S::kPad + ty * S::kR;
      if constexpr (S::kR == 4)
        *reinterpret_cast<float4*>(a[u]) = *reinterpret_cast<const float4*>(from);
      else
        *reinterpret_cast<float2*>(a[u]) = *reinterpret_cast<const float2*>(from);
    }
#pragma unroll
    for (int c = 0; c < S::kC; ++c) {
      const float4 b = *reinterpret_cast<const float4*>(y + (c * 16 + tx) * S::kPad + t);
#pragma unroll
      for (int i = 0; i < S::kR; ++i) {
        acc[i][c] = fmaf(a[0][i], b.x, acc[i][c]);
        acc[i][c] = fmaf(a[1][i], b.y, acc[i][c]);
        acc[i][c] = fmaf(a[2][i], b.z, acc[i][c]);
        acc[i][c] = fmaf(a[3][i], b.w, acc[i][c]);
      }
    }
  }
}

// A thread's products to shared memory, its rows (or columns) side by side.
template <int kDP>
__device__ __forceinline__ void store_columns_of(float* to, const float (&x)[Shape<kDP>::kR][Shape<kDP>::kR], int tx, int ty) {
  using S = Shape<kDP>;
#pragma unroll
  for (int j = 0; j < S::kR; ++j) {
    float* at = to + (tx * S::kR + j) * S::kPad + ty * S::kR;
    if constexpr (S::kR == 4)
      *reinterpret_cast<float4*>(at) = make_float4(x[0][j], x[1][j], x[2][j], x[3][j]);
    else
      *reinterpret_cast<float2*>(at) = make_float2(x[0][j], x[1][j]);
  }
}
template <int kDP>
__device__ __forceinline__ void store_rows_of(float* to, const float (&x)[Shape<kDP>::kR][Shape<kDP>::kR], int tx, int ty) {
  using S = Shape<kDP>;
#pragma unroll
  for (int i = 0; i < S::kR; ++i) {
    float* at = to + (ty * S::kR + i) * S::kPad + tx * S::kR;
    if constexpr (S::kR == 4)
      *reinterpret_cast<float4*>(at) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
    else
      *reinterpret_cast<float2*>(at) = make_float2(x[i][0], x[i][1]);
  }
}

struct Tile {
  int64_t begin;    // the stretch's first row
  int64_t other;    // first row of the other side
  int32_t first, len, other_len, stretch;
  int32_t ok;
};

template <int kT>
__device__ __forceinline__ Tile find(const void* mine, const void* other, const AttnDev& p, int64_t total,
                                     int64_t other_total, int64_t slot) {
  Tile t{};
  int64_t first, end;
  t.ok = find_tile<kT>(mine, p.offset_bytes, p.batch, total, slot, &t.stretch, &t.begin, &first, &end);
  t.first = static_cast<int32_t>(first);
  t.len = static_cast<int32_t>(end - t.begin);
  other_rows(other, p.offset_bytes, p.batch, other_total, t.stretch, &t.other, &t.other_len);
  return t;
}

template <typename T, int kDP>
__global__ void __launch_bounds__(kThreads) forward_kernel(const AttnDev p) {
  using S = Shape<kDP>;
  extern __shared__ float smem[];
  float* qs = smem;
  float* ks = qs + S::kOperand;
  float* vs = ks + S::kOperand;
  float* ps = vs + S::kOperand;
  const int head = blockIdx.x % p.heads, kv = head / p.group;
  const Tile t = find<S::kT>(p.q_offsets, p.k_offsets, p, p.total_q, p.total_k, blockIdx.x / p.heads);
  if (!t.ok) return;
  const T* q = static_cast<const T*>(p.q) + t.begin * p.q_row + head * p.q_head;
  const T* k = static_cast<const T*>(p.k) + t.other * p.k_row + kv * p.k_head;
  const T* v = static_cast<const T*>(p.v) + t.other * p.v_row + kv * p.v_head;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int shift = t.other_len - t.len;   // query i sees the keys up to i + shift
  load_transposed<T, kDP>(qs, q, p.q_row, t.first, t.len, p.D, p.fours);

  float o[S::kR][S::kC] = {};
  float top[S::kR], sum[S::kR];
#pragma unroll
  for (int i = 0; i < S::kR; ++i) top[i] = -INFINITY, sum[i] = 0.f;
  const int last = p.causal ? min(t.other_len, min(t.len, t.first + S::kT) + shift) : t.other_len;
  for (int j0 = 0; j0 < last; j0 += S::kT) {
    __syncthreads();
    load_transposed<T, kDP>(ks, k, p.k_row, j0, t.other_len, p.D, p.fours);
    load_transposed<T, kDP>(vs, v, p.v_row, j0, t.other_len, p.D, p.fours);
    __syncthreads();
    float s[S::kR][S::kR] = {};
    products<kDP>(s, qs, ks, tx, ty);
#pragma unroll
    for (int i = 0; i < S::kR; ++i) {
      const int row = t.first + ty * S::kR + i;
      const int sees = p.causal ? min(t.other_len, row + shift + 1) : t.other_len;
      float m = top[i];
#pragma unroll
      for (int j = 0; j < S::kR; ++j) {
        s[i][j] = j0 + tx * S::kR + j < sees ? s[i][j] * p.scale : -INFINITY;
        m = fmaxf(m, s[i][j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, w));
      const float base = m == -INFINITY ? 0.f : m;   // a row that has seen nothing yet
      const float keep = expf(top[i] - base);
      top[i] = m;
      float add = 0.f;
#pragma unroll
      for (int j = 0; j < S::kR; ++j) {
        s[i][j] = expf(s[i][j] - base);
        add += s[i][j];
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) add += __shfl_xor_sync(kFullMask, add, w);
      sum[i] = sum[i] * keep + add;
#pragma unroll
      for (int c = 0; c < S::kC; ++c) o[i][c] *= keep;
    }
    store_columns_of<kDP>(ps, s, tx, ty);
    __syncthreads();
    accumulate<kDP>(o, ps, vs, tx, ty);
  }
  T* out = static_cast<T*>(p.out) + t.begin * p.o_row + head * p.o_head;
#pragma unroll
  for (int i = 0; i < S::kR; ++i) {
    const int row = t.first + ty * S::kR + i;
    if (row >= t.len) continue;
    const float inv = sum[i] > 0.f ? 1.f / sum[i] : (sum[i] == 0.f ? 0.f : sum[i]);
#pragma unroll
    for (int c = 0; c < S::kC; ++c)
      if (c * 16 + tx < p.D) out[row * p.o_row + c * 16 + tx] = from_float<T>(o[i][c] * inv);
    if (p.lse != nullptr && tx == 0)
      p.lse[head * p.total_q + t.begin + row] = sum[i] == 0.f ? -INFINITY : top[i] + logf(sum[i]);
  }
}

// P and dS of a tile (rows: ty, keys: tx) from its scores and dP. What lies past the lengths or behind the
// mask is zero, whatever the rows there hold.
template <int kDP>
__device__ __forceinline__ void weights_of(float (&s)[Shape<kDP>::kR][Shape<kDP>::kR],
                                           float (&dp)[Shape<kDP>::kR][Shape<kDP>::kR], const float* lse,
                                           const float* delta, int i0, int j0, int qlen, int klen, int shift, bool causal,
                                           float scale, int tx, int ty) {
  using S = Shape<kDP>;
#pragma unroll
  for (int i = 0; i < S::kR; ++i) {
    const int row = i0 + ty * S::kR + i;
    const int sees = row >= qlen ? 0 : (causal ? min(klen, row + shift + 1) : klen);
    const float m = row < qlen ? lse[row] : 0.f, dl = row < qlen ? delta[row] : 0.f;
#pragma unroll
    for (int j = 0; j < S::kR; ++j) {
      const bool in = j0 + tx * S::kR + j < sees;
      const float w = in ? expf(s[i][j] * scale - m) : 0.f;
      dp[i][j] = in ? w * (dp[i][j] - dl) : 0.f;
      s[i][j] = w;
    }
  }
}

template <typename T, int kDP>
__global__ void __launch_bounds__(kThreads) dq_kernel(const AttnDev p) {
  using S = Shape<kDP>;
  extern __shared__ float smem[];
  float* qs = smem;
  float* gs = qs + S::kOperand;
  float* ks = gs + S::kOperand;
  float* vs = ks + S::kOperand;
  float* ws = vs + S::kOperand;
  const int head = blockIdx.x % p.heads, kv = head / p.group;
  const Tile t = find<S::kT>(p.q_offsets, p.k_offsets, p, p.total_q, p.total_k, blockIdx.x / p.heads);
  if (!t.ok) return;
  const T* k = static_cast<const T*>(p.k) + t.other * p.k_row + kv * p.k_head;
  const T* v = static_cast<const T*>(p.v) + t.other * p.v_row + kv * p.v_head;
  const float* lse = p.lse + head * p.total_q + t.begin;
  const float* delta = p.delta + head * p.total_q + t.begin;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int shift = t.other_len - t.len;
  load_transposed<T, kDP>(qs, static_cast<const T*>(p.q) + t.begin * p.q_row + head * p.q_head, p.q_row, t.first, t.len, p.D, p.fours);
  load_transposed<T, kDP>(gs, static_cast<const T*>(p.grad) + t.begin * p.g_row + head * p.g_head, p.g_row, t.first, t.len,
                          p.D, p.fours);
  float acc[S::kR][S::kC] = {};
  const int last = p.causal ? min(t.other_len, min(t.len, t.first + S::kT) + shift) : t.other_len;
  for (int j0 = 0; j0 < last; j0 += S::kT) {
    __syncthreads();
    load_transposed<T, kDP>(ks, k, p.k_row, j0, t.other_len, p.D, p.fours);
    load_transposed<T, kDP>(vs, v, p.v_row, j0, t.other_len, p.D, p.fours);
    __syncthreads();
    float s[S::kR][S::kR] = {}, dp[S::kR][S::kR] = {};
    products<kDP>(s, qs, ks, tx, ty);
    products<kDP>(dp, gs, vs, tx, ty);
    weights_of<kDP>(s, dp, lse, delta, t.first, j0, t.len, t.other_len, shift, p.causal, p.scale, tx, ty);
    store_columns_of<kDP>(ws, dp, tx, ty);
    __syncthreads();
    accumulate<kDP>(acc, ws, ks, tx, ty);
  }
  T* out = static_cast<T*>(p.dq) + t.begin * p.dq_row + head * p.dq_head;
#pragma unroll
  for (int i = 0; i < S::kR; ++i) {
    const int row = t.first + ty * S::kR + i;
    if (row >= t.len) continue;
#pragma unroll
    for (int c = 0; c < S::kC; ++c)
      if (c * 16 + tx < p.D) out[row * p.dq_row + c * 16 + tx] = from_float<T>(acc[i][c] * p.scale);
  }
}

// A key head's gradient is the sum over its query heads: one CTA walks them all, in order.
template <typename T, int kDP>
__global__ void __launch_bounds__(kThreads) dkv_kernel(const AttnDev p) {
  using S = Shape<kDP>;
  extern __shared__ float smem[];
  float* qs = smem;
  float* gs = qs + S::kOperand;
  float* ks = gs + S::kOperand;
  float* vs = ks + S::kOperand;
  float* ws = vs + S::kOperand;   // [query][key]
  const int kv = blockIdx.x % p.kv_heads;
  const Tile t = find<S::kT>(p.k_offsets, p.q_offsets, p, p.total_k, p.total_q, blockIdx.x / p.kv_heads);
  if (!t.ok) return;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int shift = t.len - t.other_len;
  load_transposed<T, kDP>(ks, static_cast<const T*>(p.k) + t.begin * p.k_row + kv * p.k_head, p.k_row, t.first, t.len, p.D, p.fours);
  load_transposed<T, kDP>(vs, static_cast<const T*>(p.v) + t.begin * p.v_row + kv * p.v_head, p.v_row, t.first, t.len, p.D, p.fours);
  float dk[S::kR][S::kC] = {}, dv[S::kR][S::kC] = {};
  const int from = p.causal ? max(0, t.first - shift) / S::kT * S::kT : 0;   // the first query that sees a key of this tile
  for (int head = kv * p.group; head < (kv + 1) * p.group; ++head) {
    const T* q = static_cast<const T*>(p.q) + t.other * p.q_row + head * p.q_head;
    const T* g = static_cast<const T*>(p.grad) + t.other * p.g_row + head * p.g_head;
    const float* lse = p.lse + head * p.total_q + t.other;
    const float* delta = p.delta + head * p.total_q + t.other;
    for (int i0 = from; i0 < t.other_len; i0 += S::kT) {
      __syncthreads();
      load_transposed<T, kDP>(qs, q, p.q_row, i0, t.other_len, p.D, p.fours);
      load_transposed<T, kDP>(gs, g, p.g_row, i0, t.other_len, p.D, p.fours);
      __syncthreads();
      float s[S::kR][S::kR] = {}, dp[S::kR][S::kR] = {};
      products<kDP>(s, qs, ks, tx, ty);
      products<kDP>(dp, gs, vs, tx, ty);
      weights_of<kDP>(s, dp, lse, delta, i0, t.first, t.other_len, t.len, shift, p.causal, p.scale, tx, ty);
      store_rows_of<kDP>(ws, s, tx, ty);
      __syncthreads();
      accumulate<kDP>(dv, ws, gs, tx, ty);
      __syncthreads();
      store_rows_of<kDP>(ws, dp, tx, ty);
      __syncthreads();
      accumulate<kDP>(dk, ws, qs, tx, ty);
    }
  }
  T* dko = static_cast<T*>(p.dk) + t.begin * p.dk_row + kv * p.dk_head;
  T* dvo = static_cast<T*>(p.dv) + t.begin * p.dv_row + kv * p.dv_head;
#pragma unroll
  for (int i = 0; i < S::kR; ++i) {
    const int row = t.first + ty * S::kR + i;
    if (row >= t.len) continue;
#pragma unroll
    for (int c = 0; c < S::kC; ++c)
      if (c * 16 + tx < p.D) {
        dko[row * p.dk_row + c * 16 + tx] = from_float<T>(dk[i][c] * p.scale);
        dvo[row * p.dv_row + c * 16 + tx] = from_float<T>(dv[i][c]);
      }
  }
}

template <auto kKernel>
int launch(int64_t blocks, int floats, const AttnDev& p, cudaStream_t stream) {
  if (blocks > 0x7fffffff) return B200TBE_ERR_TOO_LARGE;
  const int bytes = floats * 4;
  if (!allow_shared_memory<kKernel>(bytes)) return B200TBE_ERR_LAUNCH;
  kKernel<<<static_cast<unsigned>(blocks), kThreads, bytes, stream>>>(p);
  return launch_status();
}

template <typename T, int kDP>
int forward_as(const AttnDev& p, cudaStream_t stream) {
  return launch<forward_kernel<T, kDP>>(tile_slots<Shape<kDP>::kT>(p.total_q, p.batch) * p.heads,
                3 * Shape<kDP>::kOperand + Shape<kDP>::kWeights, p, stream);
}

template <typename T, int kDP>
int backward_as(const AttnDev& p, cudaStream_t stream) {
  constexpr int kFloats = 4 * Shape<kDP>::kOperand + Shape<kDP>::kWeights;
  int st = B200TBE_OK;
  if (p.total_q > 0)
    st = launch<dq_kernel<T, kDP>>(tile_slots<Shape<kDP>::kT>(p.total_q, p.batch) * p.heads, kFloats, p, stream);
  if (st == B200TBE_OK && p.total_k > 0)
    st = launch<dkv_kernel<T, kDP>>(tile_slots<Shape<kDP>::kT>(p.total_k, p.batch) * p.kv_heads, kFloats, p, stream);
  return st;
}

// Whether every operand can be read in fours of elements.
AttnDev in_fours(AttnDev p, int elem_bytes, bool backward) {
  const uint64_t size = 4 * elem_bytes;
  uint64_t off = (reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) % size;
  if (backward) off |= reinterpret_cast<uintptr_t>(p.grad) % size;
  for (int64_t x : {static_cast<int64_t>(p.D), p.q_row, p.q_head, p.k_row, p.k_head, p.v_row, p.v_head, backward ? p.g_row : 0,
                    backward ? p.g_head : 0})
    off |= x % 4 != 0;
  p.fours = off == 0;
  return p;
}

template <typename T>
int forward_of(const AttnDev& p, cudaStream_t stream) {
  if (p.D <= 32) return forward_as<T, 32>(p, stream);
  if (p.D <= 64) return forward_as<T, 64>(p, stream);
  if (p.D <= 128) return forward_as<T, 128>(p, stream);
  return forward_as<T, 256>(p, stream);
}

template <typename T>
int backward_of(const AttnDev& p, cudaStream_t stream) {
  if (p.D <= 32) return backward_as<T, 32>(p, stream);
  if (p.D <= 64) return backward_as<T, 64>(p, stream);
  if (p.D <= 128) return backward_as<T, 128>(p, stream);
  return backward_as<T, 256>(p, stream);
}

}  // namespace

int attention_forward_simt(const AttnDev& p, int dtype, cudaStream_t stream) {
  const AttnDev d = in_fours(p, dtype == B200TBE_FP32 ? 4 : 2, false);
  if (dtype == B200TBE_FP32) return forward_of<float>(d, stream);
  if (dtype == B200TBE_FP16) return forward_of<__half>(d, stream);
  return forward_of<__nv_bfloat16>(d, stream);
}

int attention_backward_simt(const AttnDev& p, int dtype, cudaStream_t stream) {
  const AttnDev d = in_fours(p, dtype == B200TBE_FP32 ? 4 : 2, true);
  if (dtype == B200TBE_FP32) return backward_of<float>(d, stream);
  if (dtype == B200TBE_FP16) return backward_of<__half>(d, stream);
  return backward_of<__nv_bfloat16>(d, stream);
}

}  // namespace b200tbe
