// Gradients of the jagged attention on the tensor cores: fp16 and bf16, head dimensions that are multiples of 8
// up to 128.
//
//   P = exp2(c S - lse log2 e),  dP = dO v^T,  dS = P (dP - delta),  c = scale log2 e
//   dQ = scale dS k                     (a CTA walks the keys of 128 queries)
//   dV = P^T dO,  dK = scale dS^T q     (a CTA walks the queries of 128 keys, of all heads that share them)
//
// Two kernels, so that no sum crosses a CTA and the results do not depend on scheduling: S and dP are computed
// twice (7 products instead of 5), and nothing is added in memory. Scores and dP come into tensor memory with a row for
// each four threads; four warpgroups take a quarter of the columns each (two with half of them: dK and dV 455 instead of
// 430 us). P and dS go back into tensor memory, each in its own columns' place, as the left operand of the next
// product: rounded to the operands' type, since the tensor cores multiply 16-bit operands, and summed in fp32. In fp16, dS is
// taken in a unit of the sequence's own (unit_of(), below).
// The CTAs take the tiles of a list, which an earlier kernel of the pass leaves, one after the other.
//
// What bounds them: of a tile's 128 x 128 the products take 2048 (dK, dV) and 1536 cycles (dQ) at 128 columns, those
// from shared memory longer, since its bandwidth feeds just one operand pair at that rate; the exponentials take 1024
// more under some of them, and the handing over between the warps that multiply and those that weigh does the rest. 7
// sequences of 301 to 4099 positions, 16 heads of 128 over 4 key heads, causal, fp16: dK and dV 415 us, dQ 309 us, the tensor
// cores 48 and 50 % busy.
#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200tbe {
namespace {

constexpr int kRows = 128;   // queries of a tile, keys of a tile
constexpr int kParts = 4;                       // warpgroups that share a tile's columns, 32 each
constexpr int kThreads = kParts * 128 + 128;
constexpr int kIssue = kParts * 4, kCopy = kIssue + 1, kStats = kIssue + 2;   // warps
// registers: 96 x 640 threads are launched as 112 four times and 32 a warpgroup
constexpr int kWeightRegs = 112, kOtherRegs = 32;
constexpr float kLog2e = 1.4426950408889634f;

struct BwdDev {
  AttnDev a;
  TileList plan;
  int32_t* status;
};

template <int kDP>
struct Layout {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kStage = 2048;   // a warp's way out for results
  static constexpr int kDqSmem = 6 * kTileBytes + kParts * 4 * kStage + 1024;
  static constexpr int kDkvSmem = 6 * kTileBytes + 8 * kStage + 1024;
};

struct DqBarriers {
  uint64_t q_full, q_empty, a_full, k_full[3], k_empty[3], v_full, v_empty, s_full, dp_full, s_loaded, ds_full, done;
};
struct DkvBarriers {
  uint64_t kv_full, kv_empty, q_full[2], q_empty[2], g_full[2], g_empty[2], s_full, dp_full, p_full, ds_full, stat_full[2],
      stat_empty[2], done;
};

// What a tile's CTA knows.
struct Item {
  int begin, other, first, len, other_len, head, stretch;
};

// Tile and head `index` of the list of tiles of queries (kOf 0) or of keys (1).
template <int kOf>
__device__ __forceinline__ Item item_at(const BwdDev& p, int64_t index) {
  const AttnDev& a = p.a;
  const int heads = kOf == 0 ? a.heads : a.kv_heads;
  const int2 at = (kOf == 0 ? p.plan.q_tiles : p.plan.k_tiles)[index / heads];
  const void* mine = kOf == 0 ? a.q_offsets : a.k_offsets;
  const int64_t total = kOf == 0 ? a.total_q : a.total_k;
  Item it;
  int64_t other;
  const int64_t begin = stretch_bound(mine, a.offset_bytes, a.batch, total, at.x);
  other_rows(kOf == 0 ? a.k_offsets : a.q_offsets, a.offset_bytes, a.batch, kOf == 0 ? a.total_k : a.total_q, at.x, &other,
             &it.other_len);
  it.begin = static_cast<int>(begin);
  it.other = static_cast<int>(other);
  it.len = static_cast<int>(stretch_bound(mine, a.offset_bytes, a.batch, total, at.x + 1) - begin);
  it.first = at.y * kRows;
  it.head = static_cast<int>(index % heads);
  it.stretch = at.x;
  return it;
}

// The squares of the two norms that bound the dS of an item, multiplied. What a key head's query heads add up to
// needs one unit (here by a whole warp); a query head's dQ has its own.
template <bool kBf16, int kOf>
__device__ __forceinline__ float norms_of(const BwdDev& p, const Item& it) {
  if constexpr (kBf16) return 0.f;
  const AttnDev& a = p.a;
  const int kv = kOf == 0 ? it.head / a.group : it.head;
  const uint32_t* norms = p.plan.grad_norms + static_cast<int64_t>(it.stretch) * a.heads;
  uint32_t largest = 0;
  if constexpr (kOf == 0) {
    largest = norms[it.head];
  } else {
    for (int h = threadIdx.x % 32; h < a.group; h += 32) largest = max(largest, norms[kv * a.group + h]);
    largest = __reduce_max_sync(kFullMask, largest);
  }
  return __uint_as_float(largest) * __uint_as_float(p.plan.v_norms[static_cast<int64_t>(it.stretch) * a.kv_heads + kv]);
}
// A power of two by which dS is multiplied before it is rounded, and its products divided afterwards. |dS| is at most
// 2 max|dO| max|v| of the sequence (Cauchy and Schwarz for each dP; delta is a mean of them): output gradients of 10^4, which
// loss scaling makes, take it past 65504 where dQ and dK fit fp16, and gradients of 10^-4 take most of it below fp16's normal range. In
// this unit it stays at or under 2^15, and 2^-38 max|dO| max|v| is the most that its last bits are worth. A sequence's unit does not depend on
// the rest of the batch, and results do not depend on the unit but for those last bits. bf16 has fp32's range and no unit.
template <bool kBf16>
__device__ __forceinline__ float unit_of(float squares) {
  if constexpr (kBf16) return 1.f;
  const int x = static_cast<int>(__float_as_uint(squares) >> 23) - 127;   // below 2^(x + 1), the root at most 2^((x + 2) >> 1)
  const float unit = __int_as_float((127 + 14 - ((x + 2) >> 1)) << 23);
  return squares > 0.f && squares < INFINITY ? unit : 1.f;
}

// The next item nobody has taken, or -1; by a whole warp.
template <int kOf>
__device__ __forceinline__ int64_t ticket_of(const BwdDev& p) {
  int ticket = 0;
  if (threadIdx.x % 32 == 0) ticket = atomicAdd(p.plan.tickets + kOf, 1);
  ticket = __shfl_sync(kFullMask, ticket, 0);
  const int64_t all = static_cast<int64_t>(min(p.plan.counts[kOf], kOf == 0 ? p.plan.q_room : p.plan.k_room)) *
                      (kOf == 0 ? p.a.heads : p.a.kv_heads);
  return ticket < all ? ticket : -1;
}

// Zero rows [rows, next multiple of 16) of a tile in shared memory: rows of other sequences, which a zero weight
// would not cancel if they held NaN. By a whole warp.
template <int kDP>
__device__ __forceinline__ void zero_tail(uint8_t* tile, int rows) {
  const int count = (16 - rows % 16) % 16;
  for (int i = threadIdx.x % 32; i < count * (kDP / 64) * 8; i += 32) {
    const int x = i / (count * 8), rest = i % (count * 8);
    *reinterpret_cast<uint4*>(tile + x * kRows * 128 + rows * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncwarp();
}

template <int kDP>
__device__ __forceinline__ void load_tile(uint8_t* tile, const CUtensorMap* map, int head, int row, uint64_t* bar) {
  for (int x = 0; x < kDP / 64; ++x) tma_load_3d(smem_addr(tile) + x * kRows * 128, map, x * 64, head, row, bar);
}

// 64 elements of row `row` of a tile in shared memory (as the tensor copies leave it) to this thread's lane of tensor
// memory, two a column: a left operand.
__device__ __forceinline__ void copy_row(uint32_t to, const uint8_t* tile, int row) {
  uint32_t r[32];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint4 v = *reinterpret_cast<const uint4*>(tile + row * 128 + (c ^ (row % 8)) * 16);
    r[4 * c] = v.x, r[4 * c + 1] = v.y, r[4 * c + 2] = v.z, r[4 * c + 3] = v.w;
  }
  tmem_st32(to, r);
  tmem_wait_st();
}

// 32 columns from `col` on of a warp's accumulator rows in tensor memory, times f, to memory: `rows` of them.
template <bool kBf16>
__device__ __forceinline__ void store_rows(uint8_t* stage, uint16_t* out, int64_t stride, uint32_t at, int col, int D, float f,
                                           bool computed, int rows) {
  if (rows <= 0) return;
  uint32_t o[32];
  if (computed) {
    tmem_ld32(o, at + col);
    tmem_wait_ld();
  }
  store_columns<kBf16>(stage, o, f, !computed, out, stride, rows, col, D);
}

// x = exp2(x c + m) in place, two and two
__device__ __forceinline__ void exponentials4(uint32_t (&x)[32], int e, uint64_t c, uint64_t m0, uint64_t m1) {
  const float2 a = unpair(fma2(as_pair(&x[e]), c, m0)), b = unpair(fma2(as_pair(&x[e + 2]), c, m1));
  x[e] = __float_as_uint(fast_exp2(a.x));
  x[e + 1] = __float_as_uint(fast_exp2(a.y));
  x[e + 2] = __float_as_uint(fast_exp2(b.x));
  x[e + 3] = __float_as_uint(fast_exp2(b.y));
}
__device__ __forceinline__ void exponentials(uint32_t (&x)[32], uint64_t c, uint64_t m) {
#pragma unroll
  for (int e = 0; e < 32; e += 4) exponentials4(x, e, c, m, m);
}

// Where the queries see few keys, dS goes into the products in two parts: rounded, and what the rounding left. Such a row
// of dS also bears the error of its delta (from an O that was rounded), which dQ multiplies by the mean of its keys: large
// for few keys, falling with their number. With the rounding of dS beside it, dQ of sequences of some hundred positions
// was off by half as much again as its own last rounding (0.0025 against 0.0017 in bf16), and dK under a causal mask by
// nearly as much (0.00031 against 0.00021 in fp16; now 0.00026), as its early queries see few keys. Long sequences' kernels (fp16,
// causal, heads of 128): dQ 300 to 303 us, dK and dV 413 to 421; in two parts for all tiles dQ alone took 377.
constexpr int kFewTiles = 2;
__device__ __forceinline__ bool in_two_parts(int tiles) { return tiles <= kFewTiles; }

// Tensor memory: scores, dP (dS takes its place), dQ, and the queries and dO, copied there once: as left operands from
// shared memory they would be read again for every tile of keys, and its bandwidth, not the tensor cores', would bound
// the products. The scores of the next keys are computed as soon as these are in registers, under the arithmetic on dP;
// dQ and the next dP under the exponentials. Keys are held until dQ and come three tiles ahead, values one.
//
// In both kernels the items go through the CTA's roles without a common stop (while one is finished, the next one's copies
// and first products are under way), so the barriers' phases run on over the items and every role counts for itself.
template <bool kBf16, int kDP>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dq_kernel(const BwdDev p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap g_map) {
  using L = Layout<kDP>;
  extern __shared__ uint8_t raw[];
  __shared__ DqBarriers bars;
  __shared__ Queue queue;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  const AttnDev& a = p.a;
  if (p.plan.counts[0] <= 0) return;
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* gs = qs + L::kTileBytes;
  uint8_t* ks = gs + L::kTileBytes;
  uint8_t* vs = ks + 3 * L::kTileBytes;
  uint8_t* stage = vs + L::kTileBytes;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, kParts * 128);
    mbar_init(&bars.a_full, kParts * 128);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
    }
    mbar_init(&bars.v_full, 1);
    mbar_init(&bars.v_empty, 1);
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.s_loaded, kParts * 128);
    mbar_init(&bars.ds_full, kParts * 128);
    mbar_init(&bars.done, 1);
    queue_init(&queue, kParts * 4 + 1);
    dead_word = 0;
    fence_barrier_init();
  }
  if (warp == kIssue) tmem_alloc(&tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base, dp_at = tmem + kRows, dq_at = tmem + 2 * kRows, q_at = dq_at + kDP, g_at = q_at + kDP / 2;
  // tiles of keys that an item's queries see
  auto tiles_of = [&](const Item& it) {
    const int sees = a.causal ? min(it.other_len, min(it.len, it.first + kRows) + it.other_len - it.len) : it.other_len;
    return sees > 0 ? (sees + kRows - 1) / kRows : 0;
  };

  if (warp >= kIssue) {
    give_registers<kOtherRegs>();
    if (warp == kCopy) {
      // ---- copies ----
      bool alive = true;
      int items = 0, tile = 0;   // with products, and their tiles
      for (int turn = 0; alive; ++turn) {
        const int64_t index = ticket_of<0>(p);
        alive = put_item(&queue, turn, index, dead);
        if (index < 0 || !alive) break;
        const Item it = item_at<0>(p, index);
        const int n = tiles_of(it), kv = it.head / a.group;
        if (n == 0) continue;
        alive = items == 0 || warp_wait(&bars.q_empty, (items - 1) & 1, dead);
        if (alive && elect_one()) {
          mbar_expect(&bars.q_full, 2 * L::kTileBytes);
          load_tile<kDP>(qs, &q_map, it.head, it.begin + it.first, &bars.q_full);
          load_tile<kDP>(gs, &g_map, it.head, it.begin + it.first, &bars.q_full);
        }
        __syncwarp();
        for (int j = 0; alive && j < n; ++j, ++tile) {
          const int st = tile % 3, row = it.other + j * kRows;
          alive = tile < 3 || warp_wait(&bars.k_empty[st], (tile / 3 - 1) & 1, dead);
          if (alive && elect_one()) {
            mbar_expect(&bars.k_full[st], L::kTileBytes);
            load_tile<kDP>(ks + st * L::kTileBytes, &k_map, kv, row, &bars.k_full[st]);
          }
          __syncwarp();
          alive = alive && (tile < 1 || warp_wait(&bars.v_empty, (tile - 1) & 1, dead));
          if (alive && elect_one()) {
            mbar_expect(&bars.v_full, L::kTileBytes);
            load_tile<kDP>(vs, &v_map, kv, row, &bars.v_full);
          }
          __syncwarp();
        }
        ++items;
      }
    } else if (warp == kIssue) {
      // ---- matrix instructions ----
      const int d_steps = (a.D + 15) / 16;
      const uint32_t dq_desc = mma_desc(kBf16, kRows, (a.D + 15) & ~15, false, true);
      bool alive = true;
      int items = 0, tile = 0;   // tile: the item's first
      for (int turn = 0; alive; ++turn) {
        const int64_t index = take_item(&queue, turn, dead);
        if (index < 0) break;
        const Item it = item_at<0>(p, index);
        const int n = tiles_of(it);
        if (n == 0) continue;
        auto keys_of = [&](int j) { return min(kRows, it.other_len - j * kRows); };
        auto scores = [&](int j) {   // whole warp
          const int of = tile + j, keys = keys_of(j);
          uint8_t* at = ks + of % 3 * L::kTileBytes;
          if (!warp_wait(&bars.k_full[of % 3], (of / 3) & 1, dead)) return false;
          if (keys % 16 != 0) zero_tail<kDP>(at, keys);
          if (of > 0 && !warp_wait(&bars.s_loaded, (of - 1) & 1, dead)) return false;
          tc_fence_after();
          if (elect_one()) {
            mma_along_k_ts<kDP / 16, kRows>(tmem, q_at, smem_addr(at), mma_desc(kBf16, kRows, (keys + 15) & ~15, false, false), d_steps);
            mma_commit(&bars.s_full);
          }
          __syncwarp();
          return true;
        };
        auto d_weights = [&](int j) {
          if (!warp_wait(&bars.v_full, (tile + j) & 1, dead)) return false;
          if (elect_one()) {
            mma_along_k_ts<kDP / 16, kRows>(dp_at, g_at, smem_addr(vs), mma_desc(kBf16, kRows, (keys_of(j) + 15) & ~15, false, false),
                                            d_steps);
            mma_commit(&bars.dp_full);
            mma_commit(&bars.v_empty);
          }
          __syncwarp();
          return true;
        };
        alive = warp_wait(&bars.a_full, items & 1, dead);
        tc_fence_after();
        alive = alive && scores(0) && d_weights(0);
        for (int j = 0; alive && j < n; ++j) {
          if (j + 1 < n) alive = scores(j + 1);
          alive = alive && warp_wait(&bars.ds_full, (tile + j) & 1, dead);
          tc_fence_after();
          if (alive && elect_one()) {
            const uint32_t k_at = smem_addr(ks) + (tile + j) % 3 * L::kTileBytes;
            const int steps = (keys_of(j) + 15) / 16;
            mma_over_rows<16, 2>(dq_at, dp_at + 16, k_at, dq_desc, steps, j > 0);
            if (in_two_parts(n)) mma_over_rows<16, 2>(dq_at, dp_at, k_at, dq_desc, steps, true);
            mma_commit(&bars.k_empty[(tile + j) % 3]);
            if (j + 1 == n) mma_commit(&bars.done);
          }
          __syncwarp();
          if (j + 1 < n) alive = alive && d_weights(j + 1);
        }
        tile += n;
        ++items;
      }
      // arrivals that nobody else waits for any more have to come before the barriers' memory goes
      if (alive && tile > 0) {
        warp_wait(&bars.v_empty, (tile - 1) & 1, dead);
        for (int st = 0; st < 3 && st < tile; ++st) warp_wait(&bars.k_empty[st], ((tile - st + 2) / 3 - 1) & 1, dead);
      }
    }
  } else {
    take_registers<kWeightRegs>();
    // ---- weights: a row and 32 columns a thread ----
    const int part = warp / 4, local = (warp % 4) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t s_at = tmem + lanes + part * 32, ds_at = dp_at + lanes + part * 32;
    const float c = a.scale * kLog2e;
    const uint64_t c2 = pair(c, c);
    bool alive = true;
    int items = 0, tile = 0;
    // The queries' rows by two warpgroups, dO's by the others, once the last item's products with theirs are done.
    auto bring = [&]() {
      if (!warp_wait(&bars.q_full, items & 1, dead)) return false;
      if (part % 2 < kDP / 64) copy_row((part < 2 ? q_at : g_at) + lanes + part % 2 * 32, (part < 2 ? qs : gs) + part % 2 * kRows * 128, local);
      tc_fence_before();
      mbar_arrive(&bars.a_full);
      mbar_arrive(&bars.q_empty);
      return true;
    };
    int64_t index = take_item(&queue, 0, dead);
    bool brought = false;
    for (int turn = 1; index >= 0; ++turn) {
      const Item it = item_at<0>(p, index);
      const int n = tiles_of(it), row = it.first + local, klen = it.other_len;
      const int limit = row >= it.len ? 0 : (a.causal ? min(klen, row + klen - it.len + 1) : klen);
      const float squares = norms_of<kBf16, 0>(p, it);
      float lse2 = 0.f, delta = 0.f;
      if (row < it.len) {
        lse2 = a.lse[it.head * a.total_q + it.begin + row] * kLog2e;
        delta = a.delta[it.head * a.total_q + it.begin + row];
        if (lse2 == -INFINITY) lse2 = INFINITY;
      }
      const float unit = unit_of<kBf16>(squares);
      const uint64_t unit2 = pair(unit, unit), minus_delta = pair(-delta * unit, -delta * unit);
      if (n > 0 && !brought) alive = bring();
      for (int j = 0; alive && j < n; ++j, ++tile) {
        alive = warp_wait(&bars.s_full, tile & 1, dead);
        if (!alive) break;
        tc_fence_after();
        const bool any = row - lane < it.len && klen - j * kRows - part * 32 > 0;   // rows and columns of the sequence here
        const int left = limit - j * kRows - part * 32;
        uint32_t s[32];
        if (any) tmem_ld32(s, s_at);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(&bars.s_loaded);
        if (any) exponentials(s, c2, pair(-lse2, -lse2));
        alive = warp_wait(&bars.dp_full, tile & 1, dead);
        if (!alive) break;
        tc_fence_after();
        if (any) {
          uint32_t dp[32], w[16];
          tmem_ld32(dp, ds_at);
          tmem_wait_ld();
          const bool cut = __any_sync(kFullMask, left < 32);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 d = unpair(mul2(as_pair(&s[e]), less_delta<kBf16>(as_pair(&dp[e]), unit2, minus_delta)));
            if (cut) {
              d.x = e < left ? d.x : 0.f;
              d.y = e + 1 < left ? d.y : 0.f;
            }
            s[e] = __float_as_uint(d.x);
            s[e + 1] = __float_as_uint(d.y);
            w[e / 2] = pack2<kBf16>(d.x, d.y);
          }
          tmem_st16(ds_at + 16, w);
          if (in_two_parts(n)) {   // and what the rounding left
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 r = unpack2<kBf16>(w[e / 2]);
              w[e / 2] = pack2<kBf16>(__uint_as_float(s[e]) - r.x, __uint_as_float(s[e + 1]) - r.y);
            }
            tmem_st16(ds_at, w);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars.ds_full);
      }
      if (alive && n > 0) alive = warp_wait(&bars.done, items++ & 1, dead);
      if (!alive) break;
      tc_fence_after();
      // the next item's operands before this one's results, so that its first products run under the stores; dQ is
      // written again only after the next dS, which this warp is then still to bring
      index = take_item(&queue, turn, dead);
      brought = index >= 0 && tiles_of(item_at<0>(p, index)) > 0;
      if (brought) alive = bring();
      if (!alive) break;
      if (part < kDP / 32)
        store_rows<kBf16>(stage + warp * L::kStage, static_cast<uint16_t*>(a.dq) + (it.begin + static_cast<int64_t>(row - lane)) * a.dq_row + it.head * a.dq_head,
                          a.dq_row, dq_at + lanes, part * 32, a.D, a.scale / unit, n > 0, it.len - row + lane);
    }
    tc_fence_before();
  }
  __syncthreads();
  report(&dead_word, p.status);
  __syncthreads();
  tc_fence_after();
  if (warp == kIssue) tmem_free(tmem, 512);
}

// Tensor memory: scores (transposed: a key a row; P, lifted, takes their place), dP (dS takes its place), dV, dK. dV and
// the next scores are computed under the arithmetic on dP, dK and the next dP under the exponentials.
template <bool kBf16, int kDP>
__global__ void __launch_bounds__(kThreads, 1)
    attention_dkv_kernel(const BwdDev p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap g_map) {
  using L = Layout<kDP>;
  extern __shared__ uint8_t raw[];
  __shared__ DkvBarriers bars;
  __shared__ Queue queue;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  // [stage][lse log2 e less the lift of P, delta in the item's unit without the lift][query], and that unit
  __shared__ __align__(16) float stats[2][2][kRows];
  __shared__ float units[2];
  constexpr float kDown = kBf16 ? 1.f : 0x1p-14f;      // 2^-kLift
  const AttnDev& a = p.a;
  if (p.plan.counts[1] <= 0) return;
  uint8_t* ks = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* vs = ks + L::kTileBytes;
  uint8_t* qs = vs + L::kTileBytes;
  uint8_t* gs = qs + 2 * L::kTileBytes;
  uint8_t* stage = gs + 2 * L::kTileBytes;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&bars.kv_full, 1);
    mbar_init(&bars.kv_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.q_empty[i], 1);
      mbar_init(&bars.g_full[i], 1);
      mbar_init(&bars.g_empty[i], 1);
      mbar_init(&bars.stat_full[i], 32);
      mbar_init(&bars.stat_empty[i], kParts * 128);
    }
    mbar_init(&bars.s_full, 1);
    mbar_init(&bars.dp_full, 1);
    mbar_init(&bars.p_full, kParts * 128);
    mbar_init(&bars.ds_full, kParts * 128);
    mbar_init(&bars.done, 1);
    queue_init(&queue, kParts * 4 + 2);
    dead_word = 0;
    fence_barrier_init();
  }
  if (warp == kIssue) tmem_alloc(&tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base, dp_at = tmem + kRows, dv_at = dp_at + kRows, dk_at = dv_at + kDP;
  // the first tile of queries with one that sees a key of the item, and how many there are from it on, of one head
  auto from_of = [&](const Item& it) { return a.causal ? max(0, it.first - (it.len - it.other_len)) / kRows : 0; };
  // whether the queries of an item's tile j see few keys
  auto few_keys = [&](const Item& it, int from, int j, int per_head) {
    const int sees = a.causal ? min(it.len, (from + j % per_head + 1) * kRows + it.len - it.other_len) : it.len;
    return in_two_parts((sees + kRows - 1) / kRows);
  };
  auto per_head_of = [&](const Item& it) { return max(0, (it.other_len + kRows - 1) / kRows - from_of(it)); };

  if (warp >= kIssue) {
    give_registers<kOtherRegs>();
    if (warp == kCopy) {
      // ---- copies ----
      bool alive = true;
      int items = 0, tile = 0;   // with products, and their tiles of queries
      for (int turn = 0; alive; ++turn) {
        const int64_t index = ticket_of<1>(p);
        alive = put_item(&queue, turn, index, dead);
        if (index < 0 || !alive) break;
        const Item it = item_at<1>(p, index);
        const int from = from_of(it), per_head = per_head_of(it), n = per_head * a.group;
        if (n == 0) continue;
        alive = items == 0 || warp_wait(&bars.kv_empty, (items - 1) & 1, dead);
        if (alive && elect_one()) {
          mbar_expect(&bars.kv_full, 2 * L::kTileBytes);
          load_tile<kDP>(ks, &k_map, it.head, it.begin + it.first, &bars.kv_full);
          load_tile<kDP>(vs, &v_map, it.head, it.begin + it.first, &bars.kv_full);
        }
        __syncwarp();
        for (int j = 0; alive && j < n; ++j, ++tile) {
          const int st = tile & 1, row = it.other + (from + j % per_head) * kRows, head = it.head * a.group + j / per_head;
          const uint32_t before = (tile / 2 - 1) & 1;
          // q, wanted first, apart from dO: both take longer than the arithmetic that hides them
          alive = tile < 2 || warp_wait(&bars.q_empty[st], before, dead);
          if (alive && elect_one()) {
            mbar_expect(&bars.q_full[st], L::kTileBytes);
            load_tile<kDP>(qs + st * L::kTileBytes, &q_map, head, row, &bars.q_full[st]);
          }
          __syncwarp();
          alive = alive && (tile < 2 || warp_wait(&bars.g_empty[st], before, dead));
          if (alive && elect_one()) {
            mbar_expect(&bars.g_full[st], L::kTileBytes);
            load_tile<kDP>(gs + st * L::kTileBytes, &g_map, head, row, &bars.g_full[st]);
          }
          __syncwarp();
        }
        ++items;
      }
    } else if (warp == kStats) {
      // ---- the queries' log-sums and deltas ----
      bool alive = true;
      int tile = 0;
      for (int turn = 0; alive; ++turn) {
        const int64_t index = take_item(&queue, turn, dead);
        if (index < 0) break;
        const Item it = item_at<1>(p, index);
        const int from = from_of(it), per_head = per_head_of(it), n = per_head * a.group;
        const float unit = unit_of<kBf16>(norms_of<kBf16, 1>(p, it)) * kDown;
        for (int j = 0; j < n; ++j, ++tile) {
          const int st = tile & 1, i0 = (from + j % per_head) * kRows, head = it.head * a.group + j / per_head;
          alive = tile < 2 || warp_wait(&bars.stat_empty[st], (tile / 2 - 1) & 1, dead);
          if (!alive) break;
          for (int e = lane; e < kRows; e += 32) {
            const bool in = i0 + e < it.other_len;
            const int64_t at = head * a.total_q + it.other + i0 + e;
            const float lse2 = in ? a.lse[at] * kLog2e : INFINITY;
            stats[st][0][e] = lse2 == -INFINITY ? INFINITY : lse2 - kLift<kBf16>;
            stats[st][1][e] = in ? a.delta[at] * unit : 0.f;
          }
          if (lane == 0) units[st] = unit;
          mbar_arrive(&bars.stat_full[st]);
        }
      }
    } else if (warp == kIssue) {
      // ---- matrix instructions ----
      const int d_steps = (a.D + 15) / 16;
      const uint32_t k_at = smem_addr(ks), v_at = smem_addr(vs);
      const uint32_t out_desc = mma_desc(kBf16, kRows, (a.D + 15) & ~15, false, true);
      bool alive = true;
      int items = 0, tile = 0;   // tile: the item's first
      for (int turn = 0; alive; ++turn) {
        const int64_t index = take_item(&queue, turn, dead);
        if (index < 0) break;
        const Item it = item_at<1>(p, index);
        const int from = from_of(it), per_head = per_head_of(it), n = per_head * a.group;
        if (n == 0) continue;
        auto rows_of = [&](int j) { return min(kRows, it.other_len - (from + j % per_head) * kRows); };
        auto stage_of = [&](int j) { return ((tile + j) & 1) * L::kTileBytes; };
        auto arrived = [&](uint64_t* bar, uint8_t* tiles, int j) {
          const bool ok = warp_wait(bar + ((tile + j) & 1), ((tile + j) / 2) & 1, dead);
          if (ok && rows_of(j) % 16 != 0) zero_tail<kDP>(tiles + stage_of(j), rows_of(j));
          return ok;
        };
        auto scores = [&](int j) {
          if (elect_one()) {
            mma_along_k<kDP / 16, kRows>(tmem, k_at, smem_addr(qs) + stage_of(j), mma_desc(kBf16, kRows, (rows_of(j) + 15) & ~15, false, false),
                                         d_steps);
            mma_commit(&bars.s_full);
          }
          __syncwarp();
        };
        auto d_weights = [&](int j) {
          if (elect_one()) {
            mma_along_k<kDP / 16, kRows>(dp_at, v_at, smem_addr(gs) + stage_of(j), mma_desc(kBf16, kRows, (rows_of(j) + 15) & ~15, false, false),
                                         d_steps);
            mma_commit(&bars.dp_full);
            if (j + 1 == n) mma_commit(&bars.kv_empty);
          }
          __syncwarp();
        };
        alive = warp_wait(&bars.kv_full, items & 1, dead) && arrived(bars.q_full, qs, 0);
        if (alive) scores(0);
        alive = alive && arrived(bars.g_full, gs, 0);
        if (alive) d_weights(0);
        for (int j = 0; alive && j < n; ++j) {
          const bool more = j + 1 < n;
          const int steps = (rows_of(j) + 15) / 16, of = tile + j;
          alive = warp_wait(&bars.p_full, of & 1, dead);
          if (!alive) break;
          tc_fence_after();
          if (elect_one()) {
            mma_over_rows<16, 2>(dv_at, tmem, smem_addr(gs) + stage_of(j), out_desc, steps, j > 0);
            mma_commit(&bars.g_empty[of & 1]);
          }
          __syncwarp();
          if (more) {
            alive = arrived(bars.q_full, qs, j + 1);
            if (!alive) break;
            scores(j + 1);
          }
          alive = (!more || arrived(bars.g_full, gs, j + 1)) && warp_wait(&bars.ds_full, of & 1, dead);
          if (!alive) break;
          tc_fence_after();
          if (elect_one()) {
            mma_over_rows<16, 2>(dk_at, dp_at + 16, smem_addr(qs) + stage_of(j), out_desc, steps, j > 0);
            if (few_keys(it, from, j, per_head)) mma_over_rows<16, 2>(dk_at, dp_at, smem_addr(qs) + stage_of(j), out_desc, steps, true);
            mma_commit(&bars.q_empty[of & 1]);
            if (!more) mma_commit(&bars.done);
          }
          __syncwarp();
          if (more) d_weights(j + 1);
        }
        tile += n;
        ++items;
      }
      // arrivals that nobody else waits for any more have to come before the barriers' memory goes
      if (alive && items > 0) {
        warp_wait(&bars.kv_empty, (items - 1) & 1, dead);
        for (int st = 0; st < 2 && st < tile; ++st) {
          const uint32_t last = ((tile - st + 1) / 2 - 1) & 1;
          warp_wait(&bars.q_empty[st], last, dead);
          warp_wait(&bars.g_empty[st], last, dead);
        }
      }
    }
  } else {
    take_registers<kWeightRegs>();
    // ---- weights: a key and 32 queries a thread ----
    const int part = warp / 4, local = (warp % 4) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t s_at = tmem + lanes + part * 32, ds_at = dp_at + lanes + part * 32;
    const uint64_t c2 = pair(a.scale * kLog2e, a.scale * kLog2e);
    bool alive = true;
    int items = 0, tile = 0;
    for (int turn = 0; alive; ++turn) {
      const int64_t index = take_item(&queue, turn, dead);
      if (index < 0) break;
      const Item it = item_at<1>(p, index);
      const int from = from_of(it), per_head = per_head_of(it), n = per_head * a.group;
      const int key = it.first + local, shift = it.len - it.other_len;
      float unit = kDown;
      for (int j = 0; j < n; ++j, ++tile) {
        const int st = tile & 1, i0 = (from + j % per_head) * kRows + part * 32;
        alive = warp_wait(&bars.stat_full[st], (tile / 2) & 1, dead) && warp_wait(&bars.s_full, tile & 1, dead);
        if (!alive) break;
        tc_fence_after();
        const bool any = key - lane < it.len && it.other_len - i0 > 0;   // rows and columns of the sequence here
        // columns [low, high) are queries of the sequence that see the key
        const int low = a.causal ? key - shift - i0 : 0, high = it.other_len - i0;
        const bool cut = __any_sync(kFullMask, low > 0 || high < 32);
        uint32_t s[32], w[16];
        if (any) {
          tmem_ld32(s, s_at);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(&stats[st][0][part * 32 + e]);
            exponentials4(s, e, c2, pair(-x.x, -x.y), pair(-x.z, -x.w));
          }
          if (cut) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < low || e >= high) s[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) w[e / 2] = pack2<kBf16>(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
          tmem_st16(s_at, w);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars.p_full);
        alive = warp_wait(&bars.dp_full, tile & 1, dead);
        if (!alive) break;
        tc_fence_after();
        if (any) {
          uint32_t dp[32];
          tmem_ld32(dp, ds_at);
          tmem_wait_ld();
          const uint64_t unit2 = pair(units[st], units[st]);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 d = *reinterpret_cast<const float4*>(&stats[st][1][part * 32 + e]);
            float2 x = unpair(mul2(as_pair(&s[e]), less_delta<kBf16>(as_pair(&dp[e]), unit2, pair(-d.x, -d.y))));
            float2 y = unpair(mul2(as_pair(&s[e + 2]), less_delta<kBf16>(as_pair(&dp[e + 2]), unit2, pair(-d.z, -d.w))));
            if (cut) {
              x.x = e < low || e >= high ? 0.f : x.x;
              x.y = e + 1 < low || e + 1 >= high ? 0.f : x.y;
              y.x = e + 2 < low || e + 2 >= high ? 0.f : y.x;
              y.y = e + 3 < low || e + 3 >= high ? 0.f : y.y;
            }
            s[e] = __float_as_uint(x.x), s[e + 1] = __float_as_uint(x.y);
            s[e + 2] = __float_as_uint(y.x), s[e + 3] = __float_as_uint(y.y);
            w[e / 2] = pack2<kBf16>(x.x, x.y);
            w[e / 2 + 1] = pack2<kBf16>(y.x, y.y);
          }
          tmem_st16(ds_at + 16, w);
          if (few_keys(it, from, j, per_head)) {   // and what the rounding left
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 r = unpack2<kBf16>(w[e / 2]);
              w[e / 2] = pack2<kBf16>(__uint_as_float(s[e]) - r.x, __uint_as_float(s[e + 1]) - r.y);
            }
            tmem_st16(ds_at, w);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars.ds_full);
        if constexpr (!kBf16) unit = units[st];
        mbar_arrive(&bars.stat_empty[st]);
      }
      if (alive && n > 0) alive = warp_wait(&bars.done, items++ & 1, dead);
      if (!alive) break;
      tc_fence_after();
      // dV and dK are written again only after the next P and dS, which this warp is then still to bring
      if (part % 2 == 0) {   // dV by one warpgroup, dK by another: shared memory has no room for four ways out
        const bool first = part == 0;
        const int64_t stride = first ? a.dv_row : a.dk_row;
        uint16_t* out = static_cast<uint16_t*>(first ? a.dv : a.dk) + (it.begin + static_cast<int64_t>(key - lane)) * stride +
                        it.head * (first ? a.dv_head : a.dk_head);
#pragma unroll 1
        for (int i = 0; i < kDP; i += 32)
          store_rows<kBf16>(stage + (part / 2 * 4 + warp % 4) * L::kStage, out, stride, (first ? dv_at : dk_at) + lanes, i, a.D,
                            first ? kDown : a.scale * kDown / unit, n > 0, it.len - key + lane);
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  report(&dead_word, p.status);
  __syncthreads();
  tc_fence_after();
  if (warp == kIssue) tmem_free(tmem, 512);
}

template <bool kBf16, int kDP>
int launch(const BwdDev& p, cudaStream_t stream) {
  using L = Layout<kDP>;
  const AttnDev& a = p.a;
  CUtensorMap q, k, v, g;
  if (!rows_map(&q, kBf16, a.q, a.total_q, a.heads, a.D, a.q_row, a.q_head, kRows) ||
      !rows_map(&k, kBf16, a.k, a.total_k, a.kv_heads, a.D, a.k_row, a.k_head, kRows) ||
      !rows_map(&v, kBf16, a.v, a.total_k, a.kv_heads, a.D, a.v_row, a.v_head, kRows) ||
      !rows_map(&g, kBf16, a.grad, a.total_q, a.heads, a.D, a.g_row, a.g_head, kRows))
    return B200TBE_ERR_UNSUPPORTED;
  const int64_t q_tiles = tile_slots<kRows>(a.total_q, a.batch) * a.heads;
  const int64_t k_tiles = tile_slots<kRows>(a.total_k, a.batch) * a.kv_heads;
  if (q_tiles > 0x7fffff00 || k_tiles > 0x7fffff00) return B200TBE_ERR_UNSUPPORTED;   // tickets are 32-bit
  if (!allow_shared_memory<attention_dq_kernel<kBf16, kDP>>(L::kDqSmem) ||
      !allow_shared_memory<attention_dkv_kernel<kBf16, kDP>>(L::kDkvSmem))
    return B200TBE_ERR_LAUNCH;
  attention_dkv_kernel<kBf16, kDP><<<static_cast<unsigned>(k_tiles < kNumSMs ? k_tiles : kNumSMs), kThreads, L::kDkvSmem, stream>>>(p, q, k, v, g);
  const int st = launch_status();
  if (st != B200TBE_OK) return st;
  attention_dq_kernel<kBf16, kDP><<<static_cast<unsigned>(q_tiles < kNumSMs ? q_tiles : kNumSMs), kThreads, L::kDqSmem, stream>>>(p, q, k, v, g);
  return launch_status();
}

}  // namespace

bool attention_backward_fits(const AttnDev& a, int dtype) {
  return attention_forward_fits(a, dtype) && a.total_q > 0 && mappable(a.grad, a.total_q, a.heads, a.g_row, a.g_head) &&
         aligned_to(a.dq, 16) && aligned_to(a.dk, 16) && aligned_to(a.dv, 16) && a.dq_row % 8 == 0 && a.dq_head % 8 == 0 &&
         a.dk_row % 8 == 0 && a.dk_head % 8 == 0 && a.dv_row % 8 == 0 && a.dv_head % 8 == 0;
}

int attention_backward_tc(const AttnDev& a, const TileList& plan, int dtype, int32_t* status, cudaStream_t stream) {
  const BwdDev p{a, plan, status};
  if (dtype == B200TBE_BF16) return a.D <= 64 ? launch<true, 64>(p, stream) : launch<true, 128>(p, stream);
  return a.D <= 64 ? launch<false, 64>(p, stream) : launch<false, 128>(p, stream);
}

}  // namespace b200tbe
