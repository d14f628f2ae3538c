// Jagged attention forward on the tensor cores: fp16 and bf16, head dimensions that are multiples of 8 up to 128.
//
//   S = q k^T,  P = exp2(c S - c m),  O = P v / rowsum(P),   c = scale log2 e,  m >= row maximum - 8 / c
//
// A CTA holds one or two tiles of 128 queries (kNQ). Their scores and their sums O lie in tensor memory (128
// columns each; the weights P take the place of the scores they come from), queries, keys and values in shared
// memory, brought by tensor copies. One warp copies, one issues the matrix instructions, and four warps for
// each query tile do the softmax, a thread for each row: no shuffles, the row's maximum and sum are its registers.
// While one tile's softmax runs, the tensor cores work on the other's products.
//
// A row's maximum is not followed exactly: as long as it has not grown by more than 2^8 in P, the old one stays,
// O needs no rescaling, and P, at most 256, keeps the same relative precision. (fp16 P is lifted by another 2^6, which the
// difference from the maximum takes along: kLift.) Normalising with the same sum makes the result independent of that choice. P is rounded to the operands' type, since the tensor cores multiply
// 16-bit operands; it is summed, like everything, in fp32.
//
// What bounds it: for 128 queries and 128 keys of 128 columns the products take 1024 cycles, the exponentials 1024 at 16
// a clock and SM, and the two operands of the scores, from shared memory, its whole bandwidth. A query tile's chain
// is 2540 cycles of softmax and 1520 of waiting for its own two products; the two tiles' chains overlap. Five prompts
// of 611 to 8192 positions, 32 heads of 128 over 8 key heads, causal: 1165 us a pass in a loop, which the power cap slows
// down (935 TFLOP/s; 1020 us in a short run), the tensor cores 45 to 50 % busy. Not better, as measured before the CTAs stayed (1138 us
// then): weights handed over in two halves (1176 us), a quarter of the exponentials by a polynomial on the FMA pipe (1426).
#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200tbe {
namespace {

constexpr int kRows = 128;   // queries of a tile, keys of a tile

struct FwdDev {
  AttnDev a;
  int32_t pair_heads;   // the two query tiles: 1: two heads' (one key head, same rows), 0: consecutive rows of a head
  int32_t* status;
  // The CTAs' items: the tiles of 128 queries of a list, or without one those of the slots, times heads (or pairs).
  int32_t listed;
  int64_t slots;
  TileList list;
};

template <int kDP, int kNQ>
struct Layout {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kStages = kNQ == 1 && kDP == 128 ? 1 : 2;
  static constexpr int kStage = 2048;   // a warp's way out for results
  static constexpr int kSmem = (kNQ + 2 * kStages) * kTileBytes + kNQ * 4 * kStage + 1024;
  static constexpr int kThreads = kNQ * 128 + 128;
  // registers: 168 x 384 threads are launched as 208 + 208 + 80 a warpgroup, 128 x 256 as 152 + 104
  static constexpr int kSoftmaxRegs = kNQ == 1 ? 152 : 208;
  static constexpr int kOtherRegs = kNQ == 1 ? 104 : 80;
  static constexpr int kColumns = kNQ == 1 ? 256 : 512;
  static constexpr int kCtas = kNQ == 1 ? 2 : 1;   // per SM
};

struct Barriers {
  uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2];
};

// A CTA's queries: rows row0 .. of a stretch of qlen rows that begins at row `begin`, of one head (or two), with the
// stretch's keys; n[s]: tiles of keys that the rows of query tile s see.
template <int kNQ>
struct Item {
  int begin, k0, row0, qlen, klen, head;
  int n[kNQ], most;
};

// All items of the launch (of the list, as many as it has).
template <int kNQ>
__device__ __forceinline__ int64_t all_items(const FwdDev& p) {
  const int per_slot = kNQ == 2 && p.pair_heads ? p.a.heads / 2 : p.a.heads;
  return (p.listed ? min(p.list.counts[0], p.list.q_room) : p.slots) * static_cast<int64_t>(per_slot);
}

// Item `index`, found by a whole warp for itself. false: its slot is empty.
template <int kNQ>
__device__ __forceinline__ bool find_item(const FwdDev& p, int64_t index, Item<kNQ>* item) {
  const AttnDev& a = p.a;
  const bool pair_heads = kNQ == 2 && p.pair_heads;
  const int per_slot = pair_heads ? a.heads / 2 : a.heads;
  int64_t slot = index / per_slot, begin, first, end, k0;
  int32_t stretch;
  if (p.listed) {
    const int2 at = p.list.q_tiles[slot];
    stretch = at.x;
    first = static_cast<int64_t>(at.y) * kRows;
    begin = stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, stretch);
    end = stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, stretch + 1);
  } else {
    if (a.causal) slot = p.slots - 1 - slot;   // later tiles of a sequence see more keys: they go first
    const bool ok = kNQ == 2 && !pair_heads
                        ? find_tile<2 * kRows>(a.q_offsets, a.offset_bytes, a.batch, a.total_q, slot, &stretch, &begin, &first, &end)
                        : find_tile<kRows>(a.q_offsets, a.offset_bytes, a.batch, a.total_q, slot, &stretch, &begin, &first, &end);
    if (!ok) return false;
  }
  other_rows(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch, &k0, &item->klen);
  item->begin = static_cast<int>(begin);
  item->k0 = static_cast<int>(k0);
  item->row0 = static_cast<int>(first);
  item->qlen = static_cast<int>(end - begin);
  item->head = static_cast<int>(index % per_slot) * (pair_heads ? 2 : 1);
  item->most = 0;
#pragma unroll
  for (int s = 0; s < kNQ; ++s) {
    const int from = item->row0 + (pair_heads ? 0 : s * kRows);
    const int sees = a.causal ? min(item->klen, min(item->qlen, from + kRows) + item->klen - item->qlen) : item->klen;
    item->n[s] = from < item->qlen && sees > 0 ? (sees + kRows - 1) / kRows : 0;
    item->most = max(item->most, item->n[s]);
  }
  return true;
}

// The CTA's items go through its roles one after the other without a common stop: while the softmax warps finish one, the
// next one's copies and first scores are under way. So the barriers' phases run on over the items; every role counts
// for itself what it has waited for.
template <bool kBf16, int kDP, int kNQ>
__global__ void __launch_bounds__(Layout<kDP, kNQ>::kThreads, Layout<kDP, kNQ>::kCtas)
    attention_fwd_kernel(const FwdDev p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map) {
  using L = Layout<kDP, kNQ>;
  constexpr int kSt = L::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ Barriers bars;
  __shared__ Queue queue;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  const AttnDev& a = p.a;
  if (p.listed && p.list.counts[0] <= 0) return;
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ks = qs + kNQ * L::kTileBytes;
  uint8_t* vs = ks + kSt * L::kTileBytes;
  uint8_t* stage = vs + kSt * L::kTileBytes;
  const int warp = __shfl_sync(kFullMask, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const bool pair_heads = kNQ == 2 && p.pair_heads;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.o_empty[i], 128);
    }
    queue_init(&queue, kNQ * 4 + 1);
    dead_word = 0;
    fence_barrier_init();
  }
  if (warp == kNQ * 4) tmem_alloc(&tmem_base, L::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  Item<kNQ> it;

  if (warp >= kNQ * 4) {
    give_registers<L::kOtherRegs>();
    if (warp == kNQ * 4 + 1) {
      // ---- copies ----
      bool alive = true;
      int items = 0, tile = 0;   // with products, and their tiles of keys
      const int64_t all = all_items<kNQ>(p);
      for (int turn = 0; alive; ++turn) {
        // off a list whoever is ready takes the next, so that the CTAs end together
        int64_t index = blockIdx.x + static_cast<int64_t>(turn) * gridDim.x;
        if (p.listed) {
          int ticket = 0;
          if (lane == 0) ticket = atomicAdd(p.list.tickets, 1);
          index = __shfl_sync(kFullMask, ticket, 0);
        }
        if (index >= all) index = -1;
        alive = put_item(&queue, turn, index, dead);
        if (index < 0 || !alive) break;
        if (!find_item(p, index, &it) || it.most == 0) continue;
        const int kv = it.head / a.group;
        alive = items == 0 || warp_wait(&bars.q_empty, (items - 1) & 1, dead);
        if (alive && elect_one()) {
          mbar_expect(&bars.q_full, kNQ * L::kTileBytes);
#pragma unroll
          for (int s = 0; s < kNQ; ++s)
#pragma unroll
            for (int x = 0; x < kDP / 64; ++x)
              tma_load_3d(smem_addr(qs) + s * L::kTileBytes + x * kRows * 128, &q_map, x * 64, it.head + (pair_heads ? s : 0),
                          it.begin + it.row0 + (pair_heads ? 0 : s * kRows), &bars.q_full);
        }
        __syncwarp();
        for (int j = 0; alive && j < it.most; ++j, ++tile) {
          const int st = tile % kSt;
          const uint32_t before = (tile / kSt - 1) & 1;
          alive = tile < kSt || warp_wait(&bars.k_empty[st], before, dead);
          if (alive && elect_one()) {
            mbar_expect(&bars.k_full[st], L::kTileBytes);
#pragma unroll
            for (int x = 0; x < kDP / 64; ++x)
              tma_load_3d(smem_addr(ks) + st * L::kTileBytes + x * kRows * 128, &k_map, x * 64, kv, it.k0 + j * kRows, &bars.k_full[st]);
          }
          __syncwarp();
          alive = alive && (tile < kSt || warp_wait(&bars.v_empty[st], before, dead));
          if (alive && elect_one()) {
            mbar_expect(&bars.v_full[st], L::kTileBytes);
#pragma unroll
            for (int x = 0; x < kDP / 64; ++x)
              tma_load_3d(smem_addr(vs) + st * L::kTileBytes + x * kRows * 128, &v_map, x * 64, kv, it.k0 + j * kRows, &bars.v_full[st]);
          }
          __syncwarp();
        }
        ++items;
      }
    } else if (warp == kNQ * 4) {
      // ---- matrix instructions ----
      const int d_steps = (a.D + 15) / 16;
      const uint32_t pv_desc = mma_desc(kBf16, kRows, (a.D + 15) & ~15, false, true);
      bool alive = true;
      int items = 0, tile = 0;                // as the copies count them; tile: the item's first
      int weighed[kNQ] = {}, summed[kNQ] = {};   // tiles of a stream whose weights have come, its items
      for (int turn = 0; alive; ++turn) {
        const int64_t index = take_item(&queue, turn, dead);
        if (index < 0) break;
        if (!find_item(p, index, &it) || it.most == 0) continue;
        // scores of stream s with key tile j; keys past the sequence's end are not multiplied
        auto scores = [&](int s, int j) {
          const int keys = min(kRows, (it.klen - j * kRows + 15) & ~15);
          mma_along_k<kDP / 16, kRows>(tmem + s * kRows, smem_addr(qs) + s * L::kTileBytes,
                                       smem_addr(ks) + (tile + j) % kSt * L::kTileBytes, mma_desc(kBf16, kRows, keys, false, false),
                                       d_steps);
          mma_commit(&bars.s_full[s]);
        };
        alive = warp_wait(&bars.q_full, items & 1, dead) && warp_wait(&bars.k_full[tile % kSt], (tile / kSt) & 1, dead);
        if (alive && elect_one()) {
#pragma unroll
          for (int s = 0; s < kNQ; ++s)
            if (it.n[s] > 0) scores(s, 0);
          mma_commit(&bars.k_empty[tile % kSt]);
          if (it.most == 1) mma_commit(&bars.q_empty);
        }
        __syncwarp();
        for (int j = 0; alive && j < it.most; ++j) {
          const int st = (tile + j) % kSt, next = (tile + j + 1) % kSt;
          alive = warp_wait(&bars.v_full[st], ((tile + j) / kSt) & 1, dead);
          if (!alive) break;
          const int keys = min(kRows, it.klen - j * kRows), steps = (keys + 15) / 16;
          if (keys % 16 != 0) {
            // rows of other sequences up to the next 16: their weights are zero, which would not cancel NaN
            const int count = 16 - keys % 16;
            for (int i = lane; i < count * 8; i += 32)
#pragma unroll
              for (int x = 0; x < kDP / 64; ++x)
                *reinterpret_cast<uint4*>(vs + st * L::kTileBytes + x * kRows * 128 + keys * 128 + i * 16) = make_uint4(0, 0, 0, 0);
            fence_async_smem();
            __syncwarp();
          }
#pragma unroll
          for (int s = 0; s < kNQ; ++s) {
            if (j < it.n[s]) {
              alive = alive && warp_wait(&bars.p_full[s], weighed[s]++ & 1, dead);
              // the stream's last sums have been read
              if (j == 0 && summed[s] > 0) alive = alive && warp_wait(&bars.o_empty[s], (summed[s] - 1) & 1, dead);
              tc_fence_after();
              if (alive && elect_one()) {
                mma_over_rows(tmem + kNQ * kRows + s * kDP, tmem + s * kRows + 64, smem_addr(vs) + st * L::kTileBytes, pv_desc, steps,
                              j > 0);
                if (j + 1 == it.n[s]) mma_commit(&bars.o_full[s]);
              }
              __syncwarp();
              if (j + 1 == it.n[s]) ++summed[s];
            }
            if (j + 1 < it.n[s]) {
              alive = alive && warp_wait(&bars.k_full[next], ((tile + j + 1) / kSt) & 1, dead);
              if (alive && elect_one()) scores(s, j + 1);
              __syncwarp();
            }
          }
          if (alive && elect_one()) {
            mma_commit(&bars.v_empty[st]);
            if (j + 1 < it.most) mma_commit(&bars.k_empty[next]);
            if (j + 2 == it.most) mma_commit(&bars.q_empty);
          }
          __syncwarp();
        }
        tile += it.most;
        ++items;
      }
      // arrivals that nobody else waits for any more have to come before the barriers' memory goes
      if (alive && items > 0) {
        warp_wait(&bars.q_empty, (items - 1) & 1, dead);
        for (int st = 0; st < kSt && st < tile; ++st) {
          const int uses = (tile - st + kSt - 1) / kSt;
          warp_wait(&bars.k_empty[st], (uses - 1) & 1, dead);
          warp_wait(&bars.v_empty[st], (uses - 1) & 1, dead);
        }
      }
    }
  } else {
    take_registers<L::kSoftmaxRegs>();
    // ---- softmax: thread = row ----
    const int s = warp / 4;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t s_at = tmem + lanes + s * kRows, o_at = tmem + lanes + kNQ * kRows + s * kDP;
    const float c = a.scale * 1.4426950408889634f;
    constexpr float kLag = 8.f, kHere = kBf16 ? 0.f : kLift<kBf16> - kLag;   // the lift that the lag leaves
    bool alive = true;
    int scored = 0, summed = 0;   // tiles of the stream, and its items
    for (int turn = 0; alive; ++turn) {
      const int64_t index = take_item(&queue, turn, dead);
      if (index < 0) break;
      if (!find_item(p, index, &it)) continue;
      const int row = it.row0 + (pair_heads ? 0 : s * kRows) + (warp % 4) * 32 + lane;
      const int tiles = it.n[kNQ == 2 ? s : 0];
      const int limit = row >= it.qlen ? 0 : (a.causal ? min(it.klen, row + it.klen - it.qlen + 1) : it.klen);   // keys that the row sees
      float top = -INFINITY, base = 0.f;   // the maximum in use; times c, less the lift
      float sum = 0.f;
      for (int j = 0; j < tiles; ++j, ++scored) {
        alive = warp_wait(&bars.s_full[s], scored & 1, dead);
        if (!alive) break;
        tc_fence_after();
        const int left = limit - j * kRows;                        // of this tile, for this row
        // 32 columns each, of the tile; a warp whose rows are all behind the last computes nothing
        const int chunks = row - lane < it.qlen ? min(4, (it.klen - j * kRows + 31) / 32) : 0;
        const bool cut = __any_sync(kFullMask, left < kRows);
        // The scores of the columns [32 from, 32 (from + kN)) into registers, masked; returns their maximum.
        auto fetch = [&](auto& x, int from) {
          constexpr int kN = sizeof(x) / sizeof(x[0]);
#pragma unroll
          for (int i = 0; i < kN; ++i)
            if (from + i < chunks) tmem_ld32(x[i], s_at + (from + i) * 32);
          tmem_wait_ld();
          float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kN; ++i)
            if (from + i < chunks) {
              if (cut) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if ((from + i) * 32 + e >= left) x[i][e] = 0xff800000u;
              }
#pragma unroll
              for (int e = 0; e < 32; e += 2)
                m[e / 2 % 4] = max3(m[e / 2 % 4], __uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1]));
            }
          return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        };
        // A maximum of the row's scores: nothing follows it until it has grown by 2^8 in P.
        auto follow = [&](float now) {
          if (j == 0) {
            top = now;
            base = now == -INFINITY ? 0.f : now * c - kHere;
          } else if (__any_sync(kFullMask, now * c > base + (kLag + kHere))) {
            top = fmaxf(top, now);
            const float next = top == -INFINITY ? 0.f : top * c - kHere, keep = fast_exp2(base - next);
            base = next;
            sum *= keep;
            // the products up to the last tile are in O: they came before these scores
#pragma unroll 1
            for (int i = 0; i < kDP; i += 16) {
              uint32_t o[16];
              tmem_ld16(o, o_at + i);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st16(o_at + i, o);
            }
          }
        };
        uint64_t add[2] = {0, 0};
        // Their weights, 16 bits each, to the second half of the tile's columns.
        auto weigh = [&](auto& x, int from) {
          constexpr int kN = sizeof(x) / sizeof(x[0]);
          const uint64_t c2 = pair(c, c), minus = pair(-base, -base);
#pragma unroll
          for (int i = 0; i < kN; ++i)
            if (from + i < chunks) {
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 y = unpair(fma2(as_pair(&x[i][e]), c2, minus));
                const float p0 = fast_exp2(y.x), p1 = fast_exp2(y.y);
                add[e / 2 % 2] = add2(add[e / 2 % 2], pair(p0, p1));
                w[e / 2] = pack2<kBf16>(p0, p1);
              }
              tmem_st16(s_at + 64 + (from + i) * 16, w);
            }
        };
        if constexpr (kNQ == 2) {
          uint32_t x[4][32];
          follow(fetch(x, 0));
          weigh(x, 0);
        } else {
          // two CTAs a SM leave room for half a row: the first half is read again once the second's weights are
          // in its place
          uint32_t x[2][32];
          const float low = fetch(x, 0);
          follow(fmaxf(low, fetch(x, 2)));
          weigh(x, 2);
          fetch(x, 0);
          weigh(x, 0);
        }
        const float2 all = unpair(add2(add[0], add[1]));
        sum += all.x + all.y;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars.p_full[s]);
      }
      if (!alive) break;
      // ---- result ----
      if (tiles > 0) {
        alive = warp_wait(&bars.o_full[s], summed++ & 1, dead);
        if (!alive) break;
        tc_fence_after();
      }
      const int h = it.head + (pair_heads ? s : 0);
      const bool here = row - lane < it.qlen;
      uint16_t* out = static_cast<uint16_t*>(a.out) + (it.begin + static_cast<int64_t>(row - lane)) * a.o_row + h * a.o_head;
#pragma unroll 1
      for (int i = 0; i < kDP; i += 32) {
        uint32_t o[32];
        if (here && tiles > 0) {
          tmem_ld32(o, o_at + i);
          tmem_wait_ld();
        }
        if (tiles > 0 && i + 32 == kDP) {   // the next item's sums may come
          tc_fence_before();
          mbar_arrive(&bars.o_empty[s]);
        }
        if (here)
          store_columns<kBf16>(stage + warp * L::kStage, o, 1.f / sum, sum == 0.f || tiles == 0, out, a.o_row, it.qlen - row + lane, i,
                               a.D);
      }
      if (a.lse != nullptr && row < it.qlen)
        a.lse[h * a.total_q + it.begin + row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
    }
    tc_fence_before();
  }
  __syncthreads();
  report(&dead_word, p.status);
  __syncthreads();
  tc_fence_after();
  if (warp == kNQ * 4) tmem_free(tmem, L::kColumns);
}

template <bool kBf16, int kDP, int kNQ>
int launch(FwdDev p, cudaStream_t stream) {
  using L = Layout<kDP, kNQ>;
  const AttnDev& a = p.a;
  CUtensorMap q, k, v;
  if (!rows_map(&q, kBf16, a.q, a.total_q, a.heads, a.D, a.q_row, a.q_head, kRows) ||
      !rows_map(&k, kBf16, a.k, a.total_k, a.kv_heads, a.D, a.k_row, a.k_head, kRows) ||
      !rows_map(&v, kBf16, a.v, a.total_k, a.kv_heads, a.D, a.v_row, a.v_head, kRows))
    return B200TBE_ERR_UNSUPPORTED;
  p.slots = kNQ == 2 && !p.pair_heads ? tile_slots<2 * kRows>(a.total_q, a.batch) : tile_slots<kRows>(a.total_q, a.batch);
  const int64_t items = p.slots * (p.pair_heads && kNQ == 2 ? a.heads / 2 : a.heads), ctas = kNumSMs * L::kCtas;
  if (items > 0x7fff0000) return B200TBE_ERR_UNSUPPORTED;   // tickets are 32-bit
  if (!allow_shared_memory<attention_fwd_kernel<kBf16, kDP, kNQ>>(L::kSmem)) return B200TBE_ERR_LAUNCH;
  attention_fwd_kernel<kBf16, kDP, kNQ><<<static_cast<unsigned>(items < ctas ? items : ctas), L::kThreads, L::kSmem, stream>>>(p, q, k, v);
  return launch_status();
}

template <bool kBf16>
int forward_of(const FwdDev& p, bool two, cudaStream_t stream) {
  if (p.a.D <= 64) return two ? launch<kBf16, 64, 2>(p, stream) : launch<kBf16, 64, 1>(p, stream);
  return two ? launch<kBf16, 128, 2>(p, stream) : launch<kBf16, 128, 1>(p, stream);
}

}  // namespace

// A masked score times the scale has to stay -infinity, and the largest score has to stay the largest: scales
// that are zero, negative or out of all proportion go to the 32-bit kernels.
bool attention_forward_fits(const AttnDev& a, int dtype) {
  return (dtype == B200TBE_FP16 || dtype == B200TBE_BF16) && a.D <= 128 && a.D % 8 == 0 && a.total_k > 0 && a.scale >= 1e-30f &&
         a.scale <= 1e30f && mappable(a.q, a.total_q, a.heads, a.q_row, a.q_head) &&
         mappable(a.k, a.total_k, a.kv_heads, a.k_row, a.k_head) && mappable(a.v, a.total_k, a.kv_heads, a.v_row, a.v_head) &&
         aligned_to(a.out, 16) && a.o_row % 8 == 0 && a.o_head % 8 == 0;
}

int attention_forward_tc(const AttnDev& a, const TileList* list, int dtype, int32_t* status, cudaStream_t stream) {
  FwdDev p{a, a.group % 2 == 0, status, list != nullptr, 0, list != nullptr ? *list : TileList{}};
  // Two query tiles a CTA read keys and values once for both and keep the tensor cores busy under the softmax.
  // Sequences so short that the second tile would mostly be empty, and tiles off a list, take one tile, and two
  // CTAs a SM.
  const bool two = p.pair_heads || (list == nullptr && a.total_q > static_cast<int64_t>(a.batch) * kRows);
  return dtype == B200TBE_BF16 ? forward_of<true>(p, two, stream) : forward_of<false>(p, two, stream);
}

bool mappable(const void* base, int64_t rows, int heads, int64_t row_stride, int64_t head_stride) {
  return aligned_to(base, 16) && (rows <= 1 || (row_stride > 0 && row_stride % 8 == 0 && row_stride < (1ll << 38))) &&
         (heads <= 1 || (head_stride > 0 && head_stride % 8 == 0 && head_stride < (1ll << 38)));
}

bool rows_map(CUtensorMap* map, bool bf16, const void* base, int64_t rows, int heads, int D, int64_t row_stride,
              int64_t head_stride, int box_rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess) return Encode(nullptr);
    return found == cudaDriverEntryPointSuccess ? reinterpret_cast<Encode>(f) : Encode(nullptr);
  }();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  // a dimension of one has no stride of its own
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? head_stride * 2 : 512),
                                 static_cast<cuuint64_t>(rows > 1 ? row_stride * 2 : 512)};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(box_rows)}, ones[3] = {1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims,
                strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace b200tbe
