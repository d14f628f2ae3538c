// Jagged attention of sequences with at most 128 queries and 128 keys, forward and backward, on the tensor cores:
// fp16 and bf16, head dimensions that are multiples of 8 up to 128.
//
// A batch of short sequences is bound by the chain of each of them (copy, product, softmax, product, store: some
// microseconds) and by HBM, not by the tensor cores. So a CTA takes one sequence and head from beginning to end
// without roles or pipelines, and small enough that several share an SM and hide one another's chain: the forward
// pass takes 128 columns of tensor memory (P and O lie where the scores were), the backward pass 256. With all of a
// row's keys in one tile the backward pass is one kernel of five products, not two of seven, and needs neither the
// forward pass's output nor a kernel for delta: delta = rowsum(P dP), which equals rowsum(dO O).
// What is longer is put on the list of tiles that the general kernels take afterwards.
#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200tbe {
namespace {

constexpr int kRows = 128;   // queries and keys at most
constexpr int kBox = 32;     // rows a tensor copy brings
constexpr float kLog2e = 1.4426950408889634f;

struct ShortDev {
  AttnDev a;
  TileList plan;
  int32_t* status;
};

struct Sequence {
  int64_t q0, k0;
  int q, k;
  bool gap;   // rows of no sequence: they see nothing, and nothing sees them
};

// The sequence of this CTA. false: it is not a short one; its tiles are on the list (by the first head's CTA), or
// there is nothing to do.
__device__ __forceinline__ bool sequence_of(const ShortDev& p, int stretch, bool first_head, bool list_keys, Sequence* s) {
  const AttnDev& a = p.a;
  s->q0 = stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, stretch);
  s->k0 = stretch_bound(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch);
  const int64_t q = max(static_cast<int64_t>(0), stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, stretch + 1) - s->q0);
  const int64_t k = max(static_cast<int64_t>(0), stretch_bound(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch + 1) - s->k0);
  s->q = static_cast<int>(q);
  s->k = static_cast<int>(k);
  s->gap = stretch < 1 || stretch > a.batch;
  if (q <= kRows && k <= kRows) return q > 0 || k > 0;
  if (!first_head) return false;
  __shared__ int at;
  for (int side = 0; side < (list_keys ? 2 : 1); ++side) {
    const int n = static_cast<int>(((side == 0 ? q : k) + kRows - 1) / kRows);
    if (n == 0) continue;
    if (threadIdx.x == 0) at = atomicAdd(p.plan.counts + side, n);
    __syncthreads();
    const int room = side == 0 ? p.plan.q_room : p.plan.k_room;
    int2* list = side == 0 ? p.plan.q_tiles : p.plan.k_tiles;
    for (int t = threadIdx.x; t < n; t += blockDim.x)
      if (at + t < room) list[at + t] = make_int2(stretch, side == 0 ? n - 1 - t : t);
    __syncthreads();
  }
  return false;
}

// rows [0, rows) of a head in boxes of kBox rows; returns the bytes that will arrive
template <int kDP>
__device__ __forceinline__ uint32_t load_rows(uint8_t* tile, const CUtensorMap* map, int head, int64_t row, int rows, uint64_t* bar) {
  uint32_t bytes = 0;
  for (int r = 0; r < rows; r += kBox)
    for (int x = 0; x < kDP / 64; ++x) {
      tma_load_3d(tile + x * kRows * 128 + r * 128, map, x * 64, head, static_cast<int>(row) + r, bar);
      bytes += kBox * 128;
    }
  return bytes;
}

// Rows [rows, next multiple of 16) become zero: other sequences' rows, whose zero weights would not cancel NaN.
template <int kDP>
__device__ __forceinline__ void zero_tail(uint8_t* tile, int rows) {
  const int count = (16 - rows % 16) % 16;
  for (int i = threadIdx.x; i < count * (kDP / 64) * 8; i += blockDim.x) {
    const int x = i / (count * 8), rest = i % (count * 8);
    *reinterpret_cast<uint4*>(tile + x * kRows * 128 + rows * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ uint32_t up16(int n) { return static_cast<uint32_t>(n + 15) & ~15u; }

// 32 columns of an accumulator row, times f, to memory (those below D)
template <bool kBf16>
__device__ __forceinline__ void store_columns(uint16_t* out, const uint32_t (&o)[32], int from, int D, float f) {
#pragma unroll
  for (int e = 0; e < 32; e += 8)
    if (from + e < D) {
      uint4 v;
      v.x = pack2<kBf16>(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f);
      v.y = pack2<kBf16>(__uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
      v.z = pack2<kBf16>(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f);
      v.w = pack2<kBf16>(__uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f);
      *reinterpret_cast<uint4*>(out + from + e) = v;
    }
}

__device__ __forceinline__ void store_zeros(uint16_t* out, int from, int to, int D) {
  for (int e = from; e < to && e < D; e += 8) *reinterpret_cast<uint4*>(out + e) = make_uint4(0, 0, 0, 0);
}

// A wait gave up: report it, and let what is in flight land before its memory is given back.
__device__ __forceinline__ void report(const int* dead, int32_t* status) {
  if (*dead) {
    if (threadIdx.x == 0 && status != nullptr) atomicOr(status, B200TBE_DEV_WAIT_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
}

template <int kDP>
struct Forward {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kSmem = 3 * kTileBytes + 1024;
  static constexpr int kColumns = kDP == 64 ? 128 : 256;
  static constexpr int kCtas = kDP == 64 ? 4 : 2;
};

// A CTA's items are blockIdx.x, blockIdx.x + gridDim.x, ...: the next one's copies are under way while this one's
// softmax and products run.
template <bool kBf16, int kDP>
__global__ void __launch_bounds__(128, Forward<kDP>::kCtas)
    attention_short_fwd_kernel(const ShortDev p, const __grid_constant__ CUtensorMap q_map,
                               const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using L = Forward<kDP>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t qk_full, v_full, s_full, o_full;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  const AttnDev& a = p.a;
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ks = qs + L::kTileBytes;
  uint8_t* vs = ks + L::kTileBytes;
  const int warp = threadIdx.x / 32, row = threadIdx.x, items = (a.batch + 2) * a.heads;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&qk_full, 1);
    mbar_init(&v_full, 1);
    mbar_init(&s_full, 1);
    mbar_init(&o_full, 1);
    dead_word = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(&tmem_base, L::kColumns);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base, lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t s_at = tmem + lanes, o_at = tmem + lanes + 64;
  const float c = a.scale * kLog2e;

  // the first item from `i` on with products to compute; those without any get their zeros on the way
  auto next_work = [&](int i, Sequence* s) {
    for (; i < items; i += gridDim.x) {
      const int stretch = i / a.heads, head = i - stretch * a.heads;
      if (!sequence_of(p, stretch, head == 0, false, s) || s->q == 0) continue;
      if (!s->gap && s->k > 0) break;
      if (row < s->q) {
        store_zeros(static_cast<uint16_t*>(a.out) + (s->q0 + row) * a.o_row + head * a.o_head, 0, kDP, a.D);
        if (a.lse != nullptr) a.lse[head * a.total_q + s->q0 + row] = -INFINITY;
      }
    }
    return i;
  };
  auto copy_qk = [&](int i, const Sequence& s) {
    const int head = i % a.heads;
    mbar_expect(&qk_full, ((s.q + kBox - 1) / kBox + (s.k + kBox - 1) / kBox) * kBox * kDP * 2);
    load_rows<kDP>(qs, &q_map, head, s.q0, s.q, &qk_full);
    load_rows<kDP>(ks, &k_map, head / a.group, s.k0, s.k, &qk_full);
  };
  auto copy_v = [&](int i, const Sequence& s) {
    mbar_expect(&v_full, (s.k + kBox - 1) / kBox * kBox * kDP * 2);
    load_rows<kDP>(vs, &v_map, i % a.heads / a.group, s.k0, s.k, &v_full);
  };
  Sequence s, n;
  int item = next_work(blockIdx.x, &s);
  if (item < items && threadIdx.x == 0) {
    copy_qk(item, s);
    copy_v(item, s);
  }
  for (uint32_t phase = 0; item < items; phase ^= 1) {
    const int next = next_work(item + gridDim.x, &n), head = item % a.heads;
    // Only this warp: the next copies may complete before another one has looked, and a barrier two phases on looks
    // as it did before. (The other barriers' next phases come after a __syncthreads() behind every warp's wait.)
    if (warp == 0) warp_wait(&qk_full, phase, dead);
    if (warp == 0 && elect_one()) {
      mma_along_k<kDP / 16, kRows>(tmem, smem_addr(qs), smem_addr(ks), mma_desc(kBf16, kRows, up16(s.k), false, false),
                                   (a.D + 15) / 16);
      mma_commit(&s_full);
    }
    __syncwarp();
    const int shift = s.k - s.q;
    const int limit = row >= s.q ? 0 : (a.causal ? min(s.k, row + shift + 1) : s.k);
    const int chunks = warp * 32 < s.q ? (s.k + 31) / 32 : 0;   // a warp whose rows are all behind the last computes nothing
    float sum = 0.f;
    warp_wait(&s_full, phase, dead);
    tc_fence_after();
    if (next < items && threadIdx.x == 0) copy_qk(next, n);
    float m = -INFINITY;
    for (int i = 0; i < chunks; ++i) {
      uint32_t x[32];
      tmem_ld32(x, s_at + i * 32);
      tmem_wait_ld();
      const int left = limit - i * 32;
      if (__all_sync(kFullMask, left >= 32)) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) m = max3(m, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) m = e < left ? fmaxf(m, __uint_as_float(x[e])) : m;
      }
    }
    const float base = m == -INFINITY ? 0.f : m * c;
    // a chunk's weights go to columns that its own scores or earlier ones had
    for (int i = 0; i < chunks; ++i) {
      uint32_t x[32], w[16];
      tmem_ld32(x, s_at + i * 32);
      tmem_wait_ld();
      const int left = limit - i * 32;
      uint64_t add = 0;
      if (__any_sync(kFullMask, left < 32)) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e >= left) x[e] = 0xff800000u;
      }
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 y = unpair(fma2(as_pair(&x[e]), pair(c, c), pair(-base, -base)));
        const float p0 = fast_exp2(y.x), p1 = fast_exp2(y.y);
        add = add2(add, pair(p0, p1));
        w[e / 2] = pack2<kBf16>(p0, p1);
      }
      sum += unpair(add).x + unpair(add).y;
      tmem_st16(s_at + i * 16, w);
    }
    tmem_wait_st();
    warp_wait(&v_full, phase, dead);
    if (s.k % 16 != 0) {
      zero_tail<kDP>(vs, s.k);
      fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0 && elect_one()) {
      mma_over_rows<0>(tmem + 64, tmem, smem_addr(vs), mma_desc(kBf16, kRows, up16(a.D), false, true), (s.k + 15) / 16, false);
      mma_commit(&o_full);
    }
    __syncwarp();
    warp_wait(&o_full, phase, dead);
    tc_fence_after();
    if (next < items && threadIdx.x == 0) copy_v(next, n);
    uint32_t o[kDP / 32][32];
    if (warp * 32 < s.q) {
#pragma unroll
      for (int i = 0; i < kDP / 32; ++i) tmem_ld32(o[i], o_at + i * 32);
    }
    tmem_wait_ld();
    tc_fence_before();
    const int failed = __syncthreads_or(*dead);   // also: the next scores may come
    tc_fence_after();
    if (row < s.q) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint16_t* out = static_cast<uint16_t*>(a.out) + (s.q0 + row) * a.o_row + head * a.o_head;
#pragma unroll
      for (int i = 0; i < kDP / 32; ++i) {
        if (sum == 0.f)
          store_zeros(out, i * 32, i * 32 + 32, a.D);
        else
          store_columns<kBf16>(out, o[i], i * 32, a.D, inv);
      }
      if (a.lse != nullptr)
        a.lse[head * a.total_q + s.q0 + row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
    }
    if (failed) break;
    item = next;
    s = n;
  }
  __syncthreads();
  report(&dead_word, p.status);
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_free(tmem, L::kColumns);
}

// Backward. Shared memory: q, dO, k, v, and over v (not read after dP) first P, then dS, as [query][key] in two
// halves of 64 keys, which the matrix instructions read either way: rows of keys for dQ = dS k, columns of queries for
// dV = P^T dO and dK = dS^T q. dV is computed under the arithmetic on dP.
// Tensor memory: scores, dP, and the gradients: in their place when the key head has one query head (kAlone), in
// columns of their own when several heads' are summed.
template <int kDP, bool kAlone>
struct Backward {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kWeightBytes = kRows * kRows * 2;
  static constexpr int kSmem = 3 * kTileBytes + kWeightBytes + 1024;
  static constexpr int kColumns = kDP == 64 && kAlone ? 256 : 512;
  static constexpr int kCtas = kDP == 64 && kAlone ? 2 : 1;
};

// d[key][.] (+)= sum over queries of w[query][key] x[query][.], 16 queries a step
__device__ __forceinline__ void transposed(uint32_t d, uint32_t w, uint32_t x, uint32_t desc, int steps, bool add) {
  const uint64_t w0 = smem_desc(w, kRows * 128), x0 = smem_desc(x, kRows * 128);
#pragma unroll
  for (int t = 0; t < 8; ++t)
    if (t < steps) mma_ss(d, w0 + t * (2048 >> 4), x0 + t * (2048 >> 4), desc, t > 0 || add);
}

template <bool kBf16, int kDP, bool kAlone>
__global__ void __launch_bounds__(256, Backward<kDP, kAlone>::kCtas)
    attention_short_bwd_kernel(const ShortDev p, const __grid_constant__ CUtensorMap q_map,
                               const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                               const __grid_constant__ CUtensorMap g_map) {
  using L = Backward<kDP, kAlone>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t kv_full, q_full, s_full, v_done, d_full;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  __shared__ float halves[2][kRows];
  const AttnDev& a = p.a;
  const int items = (a.batch + 2) * a.kv_heads;
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* gs = qs + L::kTileBytes;
  uint8_t* ks = gs + L::kTileBytes;
  uint8_t* vs = ks + L::kTileBytes;
  uint8_t* ps = vs;
  const int warp = threadIdx.x / 32, half = warp / 4, row = threadIdx.x % 128;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&kv_full, 1);
    mbar_init(&q_full, 1);
    mbar_init(&s_full, 1);
    mbar_init(&v_done, 1);
    mbar_init(&d_full, 1);
    dead_word = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(&tmem_base, L::kColumns);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base, lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
  const uint32_t dp = tmem + kRows, dv = kAlone && kDP == 64 ? tmem : tmem + 2 * kRows, dk = dv + kDP;
  const uint32_t dq = kAlone && kDP == 64 ? tmem + 2 * kDP : tmem;
  const uint32_t s_at = tmem + lanes + half * 64, dp_at = dp + lanes + half * 64;
  const int d_steps = (a.D + 15) / 16;
  const uint64_t c2 = pair(a.scale * kLog2e, a.scale * kLog2e);
  const uint32_t desc = mma_desc(kBf16, kRows, up16(a.D), true, true);

  auto dq_row = [&](const Sequence& s, int head) {
    return static_cast<uint16_t*>(a.dq) + (s.q0 + row) * a.dq_row + head * a.dq_head;
  };
  auto dkv_row = [&](const Sequence& s, int kv) {
    return half == 0 ? static_cast<uint16_t*>(a.dv) + (s.k0 + row) * a.dv_row + kv * a.dv_head
                     : static_cast<uint16_t*>(a.dk) + (s.k0 + row) * a.dk_row + kv * a.dk_head;
  };
  // the first item from `i` on with products to compute; those without any get their zeros on the way
  auto next_work = [&](int i, Sequence* s) {
    for (; i < items; i += gridDim.x) {
      const int stretch = i / a.kv_heads, kv = i - stretch * a.kv_heads;
      if (!sequence_of(p, stretch, kv == 0, true, s)) continue;
      if (!s->gap && s->q > 0 && s->k > 0) break;
      if (row < s->q && half == 0)
        for (int g = 0; g < a.group; ++g) store_zeros(dq_row(*s, kv * a.group + g), 0, kDP, a.D);
      if (row < s->k) store_zeros(dkv_row(*s, kv), 0, kDP, a.D);
    }
    return i;
  };
  // the tiles of head g of an item
  auto copy = [&](int i, const Sequence& s, int g) {
    const int kv = i % a.kv_heads, head = kv * a.group + g, q_rows = (s.q + kBox - 1) / kBox * kBox;
    mbar_expect(&kv_full, (g == 0 ? 2 : 1) * ((s.k + kBox - 1) / kBox * kBox) * kDP * 2);
    if (g == 0) load_rows<kDP>(ks, &k_map, kv, s.k0, s.k, &kv_full);
    load_rows<kDP>(vs, &v_map, kv, s.k0, s.k, &kv_full);   // again for each head: weights took its place
    mbar_expect(&q_full, 2 * q_rows * kDP * 2);
    load_rows<kDP>(qs, &q_map, head, s.q0, s.q, &q_full);
    load_rows<kDP>(gs, &g_map, head, s.q0, s.q, &q_full);
  };
  Sequence s, n;
  int item = next_work(blockIdx.x, &s);
  if (item < items && threadIdx.x == 0) copy(item, s, 0);
  uint32_t phase = 0;
  int failed = 0;
  while (item < items && !failed) {
    const int next = next_work(item + gridDim.x, &n), kv = item % a.kv_heads;
    const int shift = s.k - s.q, q_steps = (s.q + 15) / 16;
    const int limit = row >= s.q ? 0 : (a.causal ? min(s.k, row + shift + 1) : s.k);
    const int left = limit - half * 64;
    // a warp whose rows are all behind the last computes nothing
    const int chunks = warp % 4 * 32 < s.q ? max(0, min(2, (s.k - half * 64 + 31) / 32)) : 0;
    for (int g = 0; g < a.group; ++g, phase ^= 1) {
      const int head = kv * a.group + g;
      float lse2 = 0.f;
      if (row < s.q) {
        lse2 = a.lse[head * a.total_q + s.q0 + row] * kLog2e;
        if (lse2 == -INFINITY) lse2 = INFINITY;
      }
      warp_wait(&kv_full, phase, dead);
      warp_wait(&q_full, phase, dead);
      if (s.k % 16 != 0 || s.q % 16 != 0) {
        zero_tail<kDP>(ks, s.k);
        zero_tail<kDP>(qs, s.q);
        zero_tail<kDP>(gs, s.q);
        fence_async_smem();
        __syncthreads();
      }
      if (warp == 0 && elect_one()) {
        const uint32_t s_desc = mma_desc(kBf16, kRows, up16(s.k), false, false);
        mma_along_k<kDP / 16, kRows>(tmem, smem_addr(qs), smem_addr(ks), s_desc, d_steps);
        mma_along_k<kDP / 16, kRows>(dp, smem_addr(gs), smem_addr(vs), s_desc, d_steps);
        mma_commit(&s_full);
      }
      __syncwarp();
      warp_wait(&s_full, phase, dead);
      tc_fence_after();
      // ---- P, and the row's part of delta ----
      uint32_t w[2][32];
      uint64_t part = 0;
      // a row of 64 keys is 128 bytes, its 16-byte pieces exchanged by the row's number, as the copies do it
      uint8_t* p_row = ps + half * kRows * 128 + row * 128;
      auto put = [&](int i) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) y[u] = pack2<kBf16>(__uint_as_float(w[i][e + 2 * u]), __uint_as_float(w[i][e + 2 * u + 1]));
          *reinterpret_cast<uint4*>(p_row + (((i * 32 + e) / 8) ^ (row % 8)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      };
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < chunks) {
          uint32_t x[32];
          tmem_ld32(w[i], s_at + i * 32);
          tmem_ld32(x, dp_at + i * 32);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = unpair(fma2(as_pair(&w[i][e]), c2, pair(-lse2, -lse2)));
            w[i][e] = __float_as_uint(fast_exp2(y.x));
            w[i][e + 1] = __float_as_uint(fast_exp2(y.y));
          }
          if (__any_sync(kFullMask, left < i * 32 + 32)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (i * 32 + e >= left) w[i][e] = 0u, x[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) part = fma2(as_pair(&w[i][e]), as_pair(&x[e]), part);
        }
      halves[half][row] = unpair(part).x + unpair(part).y;
      tc_fence_before();
      __syncthreads();   // also: all of dP is computed, so v may be written over
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < chunks) put(i);
      fence_async_smem();
      __syncthreads();
      if (warp == 0 && elect_one()) {
        transposed(dv, smem_addr(ps), smem_addr(gs), desc, q_steps, g > 0);
        mma_commit(&v_done);
      }
      __syncwarp();
      // ---- dS ----
      const float delta = halves[0][row] + halves[1][row];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < chunks) {
          uint32_t x[32];
          tmem_ld32(x, dp_at + i * 32);
          tmem_wait_ld();
          if (__any_sync(kFullMask, left < i * 32 + 32)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (i * 32 + e >= left) x[e] = 0u;   // with a weight of zero: whatever the rows there hold
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = unpair(mul2(as_pair(&w[i][e]), add2(as_pair(&x[e]), pair(-delta, -delta))));
            w[i][e] = __float_as_uint(y.x);
            w[i][e + 1] = __float_as_uint(y.y);
          }
        }
      warp_wait(&v_done, phase, dead);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < chunks) put(i);
      fence_async_smem();
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
      if (warp == 0 && elect_one()) {
        transposed(dk, smem_addr(ps), smem_addr(qs), desc, q_steps, g > 0);
        const uint32_t dq_desc = mma_desc(kBf16, kRows, up16(a.D), false, true);
        const uint64_t w0 = smem_desc(smem_addr(ps), 16), x0 = smem_desc(smem_addr(ks), kRows * 128);
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (t < (s.k + 15) / 16)
            mma_ss(dq, w0 + (((t / 4) * kRows * 128 + (t % 4) * 32) >> 4), x0 + t * (2048 >> 4), dq_desc, t > 0);
        mma_commit(&d_full);
      }
      __syncwarp();
      warp_wait(&d_full, phase, dead);
      tc_fence_after();
      // the tiles have been read: the next ones' copies go under this one's stores
      if (threadIdx.x == 0) {
        if (g + 1 < a.group)
          copy(item, s, g + 1);
        else if (next < items)
          copy(next, n, 0);
      }
      __syncwarp();
#pragma unroll 1
      for (int i = half * kDP / 2; i < (half + 1) * kDP / 2 && warp % 4 * 32 < s.q; i += 32) {
        uint32_t o[32];
        tmem_ld32(o, dq + lanes + i);
        tmem_wait_ld();
        if (row < s.q) store_columns<kBf16>(dq_row(s, head), o, i, a.D, a.scale);
      }
      if (g + 1 == a.group) {
#pragma unroll 1
        for (int i = 0; i < kDP && warp % 4 * 32 < s.k; i += 32) {
          uint32_t o[32];
          tmem_ld32(o, (half == 0 ? dv : dk) + lanes + i);
          tmem_wait_ld();
          if (row < s.k) store_columns<kBf16>(dkv_row(s, kv), o, i, a.D, half == 0 ? 1.f : a.scale);
        }
      }
      tc_fence_before();
      failed = __syncthreads_or(*dead);   // before the next head's products
      tc_fence_after();
      if (failed) break;
    }
    item = next;
    s = n;
  }
  __syncthreads();
  report(&dead_word, p.status);
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_free(tmem, L::kColumns);
}

template <bool kBf16, int kDP>
int launch_forward(const ShortDev& p, cudaStream_t stream) {
  using L = Forward<kDP>;
  const AttnDev& a = p.a;
  CUtensorMap q, k, v;
  if (!rows_map(&q, kBf16, a.q, a.total_q, a.heads, a.D, a.q_row, a.q_head, kBox) ||
      !rows_map(&k, kBf16, a.k, a.total_k, a.kv_heads, a.D, a.k_row, a.k_head, kBox) ||
      !rows_map(&v, kBf16, a.v, a.total_k, a.kv_heads, a.D, a.v_row, a.v_head, kBox))
    return B200TBE_ERR_UNSUPPORTED;
  const int64_t blocks = (static_cast<int64_t>(a.batch) + 2) * a.heads;
  if (blocks > 0x7fff0000) return B200TBE_ERR_UNSUPPORTED;   // items are counted in 32 bits
  const auto kernel = attention_short_fwd_kernel<kBf16, kDP>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess) return B200TBE_ERR_LAUNCH;
  // all of the SM's shared memory, or fewer CTAs fit than the launch bounds promise
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess) return B200TBE_ERR_LAUNCH;
  const int64_t ctas = kNumSMs * L::kCtas;
  kernel<<<static_cast<unsigned>(blocks < ctas ? blocks : ctas), 128, L::kSmem, stream>>>(p, q, k, v);
  return launch_status();
}

template <bool kBf16, int kDP, bool kAlone>
int launch_backward(const ShortDev& p, cudaStream_t stream) {
  using L = Backward<kDP, kAlone>;
  const AttnDev& a = p.a;
  CUtensorMap q, k, v, g;
  if (!rows_map(&q, kBf16, a.q, a.total_q, a.heads, a.D, a.q_row, a.q_head, kBox) ||
      !rows_map(&k, kBf16, a.k, a.total_k, a.kv_heads, a.D, a.k_row, a.k_head, kBox) ||
      !rows_map(&v, kBf16, a.v, a.total_k, a.kv_heads, a.D, a.v_row, a.v_head, kBox) ||
      !rows_map(&g, kBf16, a.grad, a.total_q, a.heads, a.D, a.g_row, a.g_head, kBox))
    return B200TBE_ERR_UNSUPPORTED;
  const int64_t blocks = (static_cast<int64_t>(a.batch) + 2) * a.kv_heads;
  if (blocks > 0x7fff0000) return B200TBE_ERR_UNSUPPORTED;   // items are counted in 32 bits
  const auto kernel = attention_short_bwd_kernel<kBf16, kDP, kAlone>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess) return B200TBE_ERR_LAUNCH;
  // all of the SM's shared memory, or fewer CTAs fit than the launch bounds promise
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess) return B200TBE_ERR_LAUNCH;
  const int64_t ctas = kNumSMs * L::kCtas;
  kernel<<<static_cast<unsigned>(blocks < ctas ? blocks : ctas), 256, L::kSmem, stream>>>(p, q, k, v, g);
  return launch_status();
}

template <bool kBf16>
int backward_of(const ShortDev& p, cudaStream_t stream) {
  if (p.a.D <= 64)
    return p.a.group == 1 ? launch_backward<kBf16, 64, true>(p, stream) : launch_backward<kBf16, 64, false>(p, stream);
  return launch_backward<kBf16, 128, false>(p, stream);
}

}  // namespace

int attention_short_forward(const AttnDev& a, const TileList& plan, int dtype, int32_t* status, cudaStream_t stream) {
  const ShortDev p{a, plan, status};
  if (dtype == B200TBE_BF16) return a.D <= 64 ? launch_forward<true, 64>(p, stream) : launch_forward<true, 128>(p, stream);
  return a.D <= 64 ? launch_forward<false, 64>(p, stream) : launch_forward<false, 128>(p, stream);
}

int attention_short_backward(const AttnDev& a, const TileList& plan, int dtype, int32_t* status, cudaStream_t stream) {
  const ShortDev p{a, plan, status};
  return dtype == B200TBE_BF16 ? backward_of<true>(p, stream) : backward_of<false>(p, stream);
}

}  // namespace b200tbe
