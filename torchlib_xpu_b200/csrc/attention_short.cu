// Jagged attention of sequences with at most 128 queries and 128 keys, forward and backward, on the tensor cores:
// fp16 and bf16, head dimensions that are multiples of 8 up to 128.
//
// A batch of short sequences is bound by the chain of each of them (copy, product, softmax, product, store: some
// microseconds) and by HBM, not by the tensor cores. So a CTA takes one sequence and head from beginning to end
// without roles or pipelines, and as small as it goes, so that several share an SM and hide one another's chain. The forward
// pass takes 128 columns of tensor memory for heads of up to 64 (P and O lie where the scores were; four CTAs an SM), 256 beyond
// (two). The backward pass takes a key head with all its query heads, one after the other: 256 columns for one query head of up to 64
// (two CTAs an SM), else 512 (one, with nothing beside it: still at least twice as fast as the general kernels up to 64 positions on average; figures in attention.cu). With all of a
// row's keys in one tile the backward pass is one kernel of five products, not two of seven, and needs neither the
// forward pass's output nor a kernel for delta: delta = rowsum(P dP), which equals rowsum(dO O).
// What is longer is put on the list of tiles that the general kernels take afterwards.
// 4096 sequences of 0 to 128 positions, 4 heads of 64, causal: forward 137 us (its bytes take 82 at the copy rate), backward
// 397 us (143); the general kernels take 255 and 1351.
#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200tbe {
namespace {

constexpr int kRows = 128;   // queries and keys at most
constexpr int kBox = 64;     // rows a tensor copy brings: fewer copies to issue than with 32, fewer rows than with 128
constexpr float kLog2e = 1.4426950408889634f;

struct ShortDev {
  AttnDev a;
  TileList plan;
  int32_t* status;
};

// A sequence and head: its rows, or q < 0 when there are no more.
struct Job {
  int q0, k0, q, k, head;
};

// The jobs of a CTA, found by one of its warps (which has the fewest rows to compute): sequence after sequence, with
// the offsets of the next one read ahead. What is not a short sequence's goes on the list of tiles on the way (by
// its first head's finder), and rows that nothing reaches get their zeros.
template <bool kBackward>
struct Finder {
  const ShortDev& p;
  int stretch, head, step, head_step, heads;
  int qa, qb, ka, kb;

  __device__ __forceinline__ Finder(const ShortDev& p_) : p(p_) {
    heads = kBackward ? p.a.kv_heads : p.a.heads;
    stretch = blockIdx.x / heads;
    head = blockIdx.x - stretch * heads;
    step = gridDim.x / heads;
    head_step = gridDim.x - step * heads;
    read();
  }
  __device__ __forceinline__ void read() {
    const AttnDev& a = p.a;
    qa = static_cast<int>(stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, stretch));
    qb = static_cast<int>(stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, stretch + 1));
    ka = static_cast<int>(stretch_bound(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch));
    kb = static_cast<int>(stretch_bound(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch + 1));
  }
  __device__ __forceinline__ void list(int of, int side, int n) {
    const int lane = threadIdx.x % 32, room = side == 0 ? p.plan.q_room : p.plan.k_room;
    int2* tiles = side == 0 ? p.plan.q_tiles : p.plan.k_tiles;
    int at = 0;
    if (lane == 0) at = atomicAdd(p.plan.counts + side, n);
    at = __shfl_sync(kFullMask, at, 0);
    // offsets that decrease give more tiles than there is room for, or than an int counts
    for (int t = lane; t < n; t += 32)
      if (static_cast<unsigned>(at + t) < static_cast<unsigned>(room)) tiles[at + t] = make_int2(of, side == 0 ? n - 1 - t : t);
  }
  __device__ __forceinline__ void zeros(void* base, int64_t row, int64_t stride, int rows) {
    const int vecs = p.a.D / 8;
    for (int i = threadIdx.x % 32; i < rows * vecs; i += 32)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + row + i / vecs * stride + i % vecs * 8) = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ Job next() {
    const AttnDev& a = p.a;
    for (;;) {
      if (stretch > a.batch + 1) return Job{0, 0, -1, 0, 0};
      const Job job{qa, ka, max(0, qb - qa), max(0, kb - ka), head};
      const int of = stretch;
      head += head_step;
      stretch += step + (head >= heads ? 1 : 0);
      if (head >= heads) head -= heads;
      if (stretch <= a.batch + 1) read();
      const bool gap = of < 1 || of > a.batch;   // rows of no sequence: they see nothing, and nothing sees them
      if (job.q > kRows || job.k > kRows) {
        if (job.head == 0) {
          list(of, 0, (job.q + kRows - 1) / kRows);
          if (kBackward) list(of, 1, (job.k + kRows - 1) / kRows);
        }
        continue;
      }
      if (!gap && job.q > 0 && job.k > 0) return job;
      if constexpr (kBackward) {
        for (int g = 0; g < a.group; ++g)
          zeros(a.dq, job.q0 * a.dq_row + (job.head * a.group + g) * a.dq_head, a.dq_row, job.q);
        zeros(a.dk, job.k0 * a.dk_row + job.head * a.dk_head, a.dk_row, job.k);
        zeros(a.dv, job.k0 * a.dv_row + job.head * a.dv_head, a.dv_row, job.k);
      } else {
        zeros(a.out, job.q0 * a.o_row + job.head * a.o_head, a.o_row, job.q);
        if (a.lse != nullptr)
          for (int i = threadIdx.x % 32; i < job.q; i += 32) a.lse[job.head * a.total_q + job.q0 + i] = -INFINITY;
      }
    }
  }
};

// rows [0, rows) of a head in boxes of kBox rows
template <int kDP>
__device__ __forceinline__ void load_rows(uint32_t tile, const CUtensorMap* map, int head, int row, int rows, uint64_t* bar) {
#pragma unroll
  for (int r = 0; r < kRows; r += kBox)
    if (r < rows) {
#pragma unroll
      for (int x = 0; x < kDP / 64; ++x) tma_load_3d(tile + x * kRows * 128 + r * 128, map, x * 64, head, row + r, bar);
    }
}
__device__ __forceinline__ int boxed(int rows) { return (rows + kBox - 1) / kBox * kBox; }

// Rows [rows, next multiple of 16) become zero: other sequences' rows, whose zero weights would not cancel NaN.
// By a whole warp.
template <int kDP>
__device__ __forceinline__ void zero_tail(uint8_t* tile, int rows) {
  const int count = (16 - rows % 16) % 16;
  for (int i = threadIdx.x % 32; i < count * 8; i += 32)
#pragma unroll
    for (int x = 0; x < kDP / 64; ++x)
      *reinterpret_cast<uint4*>(tile + x * kRows * 128 + rows * 128 + i * 16) = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ uint32_t up16(int n) { return static_cast<uint32_t>(n + 15) & ~15u; }

template <int kDP>
struct Forward {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kSmem = 3 * kTileBytes + 1024;
  static constexpr int kColumns = kDP == 64 ? 128 : 256;
  static constexpr int kCtas = kDP == 64 ? 4 : 2;
};

// A CTA takes jobs as long as there are some; the next one's copies are under way while this one's softmax and products
// run. Warp 0 issues the products, warp 3 finds the jobs and issues the copies.
template <bool kBf16, int kDP>
__global__ void __launch_bounds__(128, Forward<kDP>::kCtas)
    attention_short_fwd_kernel(const ShortDev p, const __grid_constant__ CUtensorMap q_map,
                               const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using L = Forward<kDP>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t qk_full, v_full, s_full, o_full;
  __shared__ Job jobs[2];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  const AttnDev& a = p.a;
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* vs = qs + 2 * L::kTileBytes;
  const uint32_t q_at = smem_addr(qs), k_at = q_at + L::kTileBytes, v_at = k_at + L::kTileBytes;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / 32, 0), row = threadIdx.x;
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
  const uint64_t c2 = pair(c, c);

  auto copy_qk = [&](const Job& s) {
    mbar_expect(&qk_full, (boxed(s.q) + boxed(s.k)) * kDP * 2);
    load_rows<kDP>(q_at, &q_map, s.head, s.q0, s.q, &qk_full);
    load_rows<kDP>(k_at, &k_map, s.head / a.group, s.k0, s.k, &qk_full);
  };
  auto copy_v = [&](const Job& s) {
    mbar_expect(&v_full, boxed(s.k) * kDP * 2);
    load_rows<kDP>(v_at, &v_map, s.head / a.group, s.k0, s.k, &v_full);
  };
  Finder<false> finder(p);
  Job n{0, 0, -1, 0, 0};
  if (warp == 3) {
    n = finder.next();
    if (n.q > 0 && elect_one()) {
      copy_qk(n);
      copy_v(n);
    }
    __syncwarp();
    if (row == 96) jobs[0] = n;
  }
  __syncthreads();
  for (int turn = 0, failed = 0; !failed; ++turn) {
    const Job s = jobs[turn & 1];
    if (s.q < 0) break;
    const uint32_t phase = turn & 1;
    if (warp == 0) {
      // Only this warp waits for these copies: the next ones may complete before another warp has looked, and a
      // barrier two phases on looks as it did before. (The other barriers' next phases come after a __syncthreads()
      // behind every warp's wait.)
      warp_wait(&qk_full, phase, dead);
      if (elect_one()) {
        mma_along_k<kDP / 16, kRows>(tmem, q_at, k_at, mma_desc(kBf16, kRows, up16(s.k), false, false), (a.D + 15) / 16);
        mma_commit(&s_full);
      }
      __syncwarp();
    } else if (warp == 3) {
      n = finder.next();
      if (row == 96) jobs[(turn + 1) & 1] = n;
    }
    warp_wait(&s_full, phase, dead);
    tc_fence_after();
    if (warp == 3) {
      if (n.q > 0 && elect_one()) copy_qk(n);
      __syncwarp();
    }
    float sum = 0.f, base = 0.f;
    if (warp * 32 < s.q) {   // a warp whose rows are all behind the last computes nothing
      const int chunks = (s.k + 31) / 32;
      const int limit = row >= s.q ? 0 : (a.causal ? min(s.k, row + s.k - s.q + 1) : s.k);
      auto largest = [&](uint32_t (&x)[32], int i, float m) {   // of chunk i, whose masked scores become -infinity
        if (__any_sync(kFullMask, limit < i * 32 + 32)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (i * 32 + e >= limit) x[e] = 0xff800000u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) m = max3(m, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
        return m;
      };
      // a chunk's weights go to columns that its own scores or earlier ones had
      auto weigh = [&](const uint32_t (&x)[32], int i) {
        uint32_t w[16];
        uint64_t add = 0;
        const uint64_t minus = pair(-base, -base);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 y = unpair(fma2(as_pair(&x[e]), c2, minus));
          const float p0 = fast_exp2(y.x), p1 = fast_exp2(y.y);
          add = add2(add, pair(p0, p1));
          w[e / 2] = pack2<kBf16>(p0, p1);
        }
        sum += unpair(add).x + unpair(add).y;
        tmem_st16(s_at + i * 16, w);
      };
      uint32_t x[2][32];
      float m = -INFINITY;
      if (chunks > 2) {   // the second half's maximum first; its scores are read again when the first half is done
        tmem_ld32(x[0], s_at + 64);
        if (chunks > 3) tmem_ld32(x[1], s_at + 96);
        tmem_wait_ld();
        m = largest(x[0], 2, m);
        if (chunks > 3) m = largest(x[1], 3, m);
      }
      tmem_ld32(x[0], s_at);
      if (chunks > 1) tmem_ld32(x[1], s_at + 32);
      tmem_wait_ld();
      m = largest(x[0], 0, m);
      if (chunks > 1) m = largest(x[1], 1, m);
      base = m == -INFINITY ? 0.f : m * c - kLift<kBf16>;
      weigh(x[0], 0);
      if (chunks > 1) weigh(x[1], 1);
      if (chunks > 2) {
        tmem_ld32(x[0], s_at + 64);
        if (chunks > 3) tmem_ld32(x[1], s_at + 96);
        tmem_wait_ld();
        largest(x[0], 2, m);
        weigh(x[0], 2);
        if (chunks > 3) {
          largest(x[1], 3, m);
          weigh(x[1], 3);
        }
      }
      tmem_wait_st();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      warp_wait(&v_full, phase, dead);
      if (s.k % 16 != 0) {
        zero_tail<kDP>(vs, s.k);
        fence_async_smem();
        __syncwarp();
      }
      tc_fence_after();
      if (elect_one()) {
        mma_over_rows<0>(tmem + 64, tmem, v_at, mma_desc(kBf16, kRows, up16(a.D), false, true), (s.k + 15) / 16, false);
        mma_commit(&o_full);
      }
      __syncwarp();
    }
    warp_wait(&o_full, phase, dead);
    tc_fence_after();
    if (warp * 32 < s.q) {   // through v's place, which has been read
      uint32_t o[kDP / 32][32];
#pragma unroll
      for (int i = 0; i < kDP / 32; ++i) tmem_ld32(o[i], o_at + i * 32);
      tmem_wait_ld();
      uint16_t* out = static_cast<uint16_t*>(a.out) + (s.q0 + warp * 32) * a.o_row + s.head * a.o_head;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int i = 0; i < kDP / 32; ++i)
        store_columns<kBf16>(vs + warp * 2048, o[i], inv, sum == 0.f, out, a.o_row, s.q - warp * 32, i * 32, a.D);
      if (a.lse != nullptr && row < s.q)
        a.lse[s.head * a.total_q + s.q0 + row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
    }
    fence_async_smem();
    tc_fence_before();
    failed = __syncthreads_or(*dead);
    tc_fence_after();
    if (warp == 3) {
      if (n.q > 0 && !failed && elect_one()) copy_v(n);
      __syncwarp();
    }
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
  // the results' way out, 2 KB a warp: with 64 columns the half of the weights' place that v does not share
  static constexpr int kStage = kDP == 64 ? kRows * 128 : kWeightBytes;
  static constexpr int kSmem = 3 * kTileBytes + kWeightBytes + (kDP == 64 ? 0 : 8 * 2048) + 1024;
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
  __shared__ uint64_t full, s_full, v_done, d_full;
  __shared__ Job jobs[2];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  __shared__ float halves[2][kRows];
  __shared__ uint32_t tops[8];   // of the warps, the largest |dP|
  const AttnDev& a = p.a;
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* gs = qs + L::kTileBytes;
  uint8_t* ks = gs + L::kTileBytes;
  uint8_t* ps = ks + L::kTileBytes;   // and v
  const uint32_t q_at = smem_addr(qs), g_at = smem_addr(gs), k_at = smem_addr(ks), v_at = smem_addr(ps), p_at = v_at;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / 32, 0), half = warp / 4, row = threadIdx.x % 128;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&full, 1);
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
  uint8_t* stage = ps + L::kStage + warp * 2048;
  constexpr float kDown = kBf16 ? 1.f : 0x1p-14f;   // 2^-kLift

  auto copy = [&](const Job& s, int g) {
    const int head = s.head * a.group + g;
    mbar_expect(&full, ((g == 0 ? 2 : 1) * boxed(s.k) + 2 * boxed(s.q)) * kDP * 2);
    load_rows<kDP>(q_at, &q_map, head, s.q0, s.q, &full);
    if (g == 0) load_rows<kDP>(k_at, &k_map, s.head, s.k0, s.k, &full);
    load_rows<kDP>(g_at, &g_map, head, s.q0, s.q, &full);
    load_rows<kDP>(v_at, &v_map, s.head, s.k0, s.k, &full);   // again for each head: weights took its place
  };
  Finder<true> finder(p);
  Job n{0, 0, -1, 0, 0};
  if (warp == 7) {
    n = finder.next();
    if (n.q > 0 && elect_one()) copy(n, 0);
    __syncwarp();
    if (row == 127) jobs[0] = n;
  }
  __syncthreads();
  uint32_t phase = 0;
  for (int turn = 0, failed = 0; !failed; ++turn) {
    const Job s = jobs[turn & 1];
    if (s.q < 0) break;
    const int q_steps = (s.q + 15) / 16;
    const int limit = row >= s.q ? 0 : (a.causal ? min(s.k, row + s.k - s.q + 1) : s.k);
    const int left = limit - half * 64;
    // a warp whose rows are all behind the last computes nothing
    const bool rows_here = warp % 4 * 32 < s.q, keys_here = warp % 4 * 32 < s.k;
    const int chunks = rows_here ? max(0, min(2, (s.k - half * 64 + 31) / 32)) : 0;
    float unit = 1.f;
    for (int g = 0; g < a.group; ++g, phase ^= 1) {
      const int head = s.head * a.group + g;
      if (warp == 0) {
        warp_wait(&full, phase, dead);
        if (s.k % 16 != 0 || s.q % 16 != 0) {
          zero_tail<kDP>(ks, s.k);
          zero_tail<kDP>(qs, s.q);
          zero_tail<kDP>(gs, s.q);
          fence_async_smem();
          __syncwarp();
        }
        if (elect_one()) {
          const uint32_t s_desc = mma_desc(kBf16, kRows, up16(s.k), false, false);
          mma_along_k<kDP / 16, kRows>(tmem, q_at, k_at, s_desc, d_steps);
          mma_along_k<kDP / 16, kRows>(dp, g_at, v_at, s_desc, d_steps);
          mma_commit(&s_full);
        }
        __syncwarp();
      } else if (warp == 7 && g == 0) {
        n = finder.next();
        if (row == 127) jobs[(turn + 1) & 1] = n;
      }
      float lse2 = 0.f;   // under the products
      if (row < s.q) {
        lse2 = a.lse[head * a.total_q + s.q0 + row] * kLog2e;
        if (lse2 == -INFINITY) lse2 = INFINITY;
      }
      warp_wait(&s_full, phase, dead);
      tc_fence_after();
      // ---- P, and the row's part of delta ----
      uint32_t w[2][32], x[32];
      uint64_t part = 0;
      float top = 0.f;
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
      const uint64_t minus = pair(kLift<kBf16> - lse2, kLift<kBf16> - lse2);   // w is P lifted
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < chunks) {
          tmem_ld32(w[i], s_at + i * 32);
          tmem_ld32(x, dp_at + i * 32);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = unpair(fma2(as_pair(&w[i][e]), c2, minus));
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
          if constexpr (!kBf16) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) top = max3(top, fabsf(__uint_as_float(x[e])), fabsf(__uint_as_float(x[e + 1])));
          }
          put(i);   // v, whose place it is, has been read
        }
      halves[half][row] = unpair(part).x + unpair(part).y;
      if constexpr (!kBf16) {
        const uint32_t bits = __reduce_max_sync(kFullMask, __float_as_uint(top));
        if (threadIdx.x % 32 == 0) tops[warp] = bits;
      }
      fence_async_smem();
      tc_fence_before();
      __syncthreads();
      if (warp == 0) {
        tc_fence_after();
        if (elect_one()) {
          transposed(dv, p_at, g_at, mma_desc(kBf16, kRows, up16(a.D), true, true), q_steps, g > 0);
          mma_commit(&v_done);
        }
        __syncwarp();
      }
      // ---- dS ----
      // In fp16 dS, at most twice the largest |dP|, is multiplied by a power of two that keeps it under 2^15 (why: unit_of() of the
      // general kernels). Heads that are summed share theirs: where a later one needs a smaller, the sums so far follow it.
      if constexpr (!kBf16) {
        uint32_t bits = tops[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) bits = max(bits, tops[i]);
        const int x_of = static_cast<int>(bits >> 23);   // biased; 0 and 255: nothing there, or nothing finite
        const float needs = x_of > 0 && x_of < 255 ? __int_as_float(min(127 + 60, 2 * 127 + 13 - x_of) << 23) : (x_of == 0 ? 0x1p60f : 1.f);
        if (kAlone || g == 0) {
          unit = needs;
        } else if (needs < unit) {
          const float follow = needs / unit;
          unit = needs;
          if (half == 1) {
#pragma unroll 1
            for (int i = 0; i < kDP; i += 32) {
              tmem_ld32(x, dk + lanes + i);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * follow);
              tmem_st32(dk + lanes + i, x);
            }
            tmem_wait_st();
          }
        }
      }
      const float here = unit * kDown;   // dS from the lifted P, and delta, which was summed with it
      const float delta = (halves[0][row] + halves[1][row]) * kDown * here;
      const uint64_t unit2 = pair(here, here), minus_delta = pair(-delta, -delta);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < chunks) {
          tmem_ld32(x, dp_at + i * 32);
          tmem_wait_ld();
          if (__any_sync(kFullMask, left < i * 32 + 32)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (i * 32 + e >= left) x[e] = 0u;   // with a weight of zero: whatever the rows there hold
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = unpair(mul2(as_pair(&w[i][e]), less_delta<kBf16>(as_pair(&x[e]), unit2, minus_delta)));
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
      if (warp == 0) {
        tc_fence_after();
        if (elect_one()) {
          transposed(dk, p_at, q_at, mma_desc(kBf16, kRows, up16(a.D), true, true), q_steps, g > 0);
          const uint32_t dq_desc = mma_desc(kBf16, kRows, up16(a.D), false, true);
          const uint64_t w0 = smem_desc(p_at, 16), x0 = smem_desc(k_at, kRows * 128);
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (t < (s.k + 15) / 16)
              mma_ss(dq, w0 + (((t / 4) * kRows * 128 + (t % 4) * 32) >> 4), x0 + t * (2048 >> 4), dq_desc, t > 0);
          mma_commit(&d_full);
        }
        __syncwarp();
      }
      warp_wait(&d_full, phase, dead);
      tc_fence_after();
      // the tiles have been read: the next ones' copies go under this one's stores
      if (warp == 7) {
        if (g + 1 < a.group) {
          if (elect_one()) copy(s, g + 1);
        } else if (n.q > 0) {
          if (elect_one()) copy(n, 0);
        }
        __syncwarp();
      }
      const bool last = g + 1 == a.group;
      const int64_t stride = half == 0 ? a.dv_row : a.dk_row;
      const float f = half == 0 ? kDown : a.scale / unit;
      uint16_t* dq_out = static_cast<uint16_t*>(a.dq) + (s.q0 + warp % 4 * 32) * a.dq_row + head * a.dq_head;
      uint16_t* dkv_out = static_cast<uint16_t*>(half == 0 ? a.dv : a.dk) + (s.k0 + warp % 4 * 32) * stride +
                          s.head * (half == 0 ? a.dv_head : a.dk_head);
      const uint32_t dkv_at = (half == 0 ? dv : dk) + lanes;
#pragma unroll 1
      for (int i = half * kDP / 2; i < (half + 1) * kDP / 2 && rows_here; i += 32) {
        tmem_ld32(x, dq + lanes + i);
        tmem_wait_ld();
        store_columns<kBf16>(stage, x, a.scale / unit, false, dq_out, a.dq_row, s.q - warp % 4 * 32, i, a.D);
      }
#pragma unroll 1
      for (int i = 0; i < kDP && last && keys_here; i += 32) {
        tmem_ld32(x, dkv_at + i);
        tmem_wait_ld();
        store_columns<kBf16>(stage, x, f, false, dkv_out, stride, s.k - warp % 4 * 32, i, a.D);
      }
      fence_async_smem();
      tc_fence_before();
      failed = __syncthreads_or(*dead);   // before the next head's products
      tc_fence_after();
      if (failed) break;
    }
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
  if (!allow_shared_memory<attention_short_fwd_kernel<kBf16, kDP>>(L::kSmem)) return B200TBE_ERR_LAUNCH;
  const int64_t ctas = kNumSMs * L::kCtas;
  attention_short_fwd_kernel<kBf16, kDP><<<static_cast<unsigned>(blocks < ctas ? blocks : ctas), 128, L::kSmem, stream>>>(p, q, k, v);
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
  if (!allow_shared_memory<attention_short_bwd_kernel<kBf16, kDP, kAlone>>(L::kSmem)) return B200TBE_ERR_LAUNCH;
  const int64_t ctas = kNumSMs * L::kCtas;
  attention_short_bwd_kernel<kBf16, kDP, kAlone><<<static_cast<unsigned>(blocks < ctas ? blocks : ctas), 256, L::kSmem, stream>>>(p, q, k, v, g);
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
