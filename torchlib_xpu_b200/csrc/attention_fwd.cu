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
// O needs no rescaling, and P, at most 256, keeps the same relative precision. Normalising with the same sum
// makes the result independent of that choice.
#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200tbe {
namespace {

constexpr int kRows = 128;   // queries of a tile, keys of a tile

struct FwdDev {
  AttnDev a;
  int32_t pair_heads;   // the two query tiles: 1: two heads' (one key head, same rows), 0: consecutive rows of a head
  int32_t* status;
  // With a list of tiles of 128 queries (what the short sequences' kernel left over) the CTAs take them one after
  // the other; without one, a CTA takes its slot's tile.
  int32_t listed;
  TileList plan;
};

template <int kDP, int kNQ>
struct Layout {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kStages = kNQ == 1 && kDP == 128 ? 1 : 2;
  static constexpr int kSmem = (kNQ + 2 * kStages) * kTileBytes + 1024;
  static constexpr int kThreads = kNQ * 128 + 128;
  // registers: 168 x 384 threads are launched as 208 + 208 + 80 a warpgroup, 128 x 256 as 152 + 104
  static constexpr int kSoftmaxRegs = kNQ == 1 ? 152 : 208;
  static constexpr int kOtherRegs = kNQ == 1 ? 104 : 80;
  static constexpr int kColumns = kNQ == 1 ? 256 : 512;
  static constexpr int kCtas = kNQ == 1 ? 2 : 1;   // per SM
};

struct Barriers {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
};
struct Shared {
  Barriers b;
  uint32_t tmem;
  int dead;
};

// A CTA's queries: rows row0 .. of a stretch of qlen rows that begins at row `begin`, of one head (or two), with the
// stretch's keys.
struct Item {
  int64_t begin, k0;
  int row0, qlen, klen, head;
};

// The item of this CTA's slot; false: it has none.
template <bool kTwo>
__device__ __forceinline__ bool slot_item(const FwdDev& p, bool pair_heads, int per_slot, Item* item) {
  const AttnDev& a = p.a;
  const int64_t slots = gridDim.x / per_slot;
  // later tiles of a sequence see more keys: they go first
  const int64_t slot = a.causal ? slots - 1 - blockIdx.x / per_slot : blockIdx.x / per_slot;
  int32_t stretch;
  int64_t first, end;
  const bool ok = kTwo && !pair_heads ? find_tile<2 * kRows>(a.q_offsets, a.offset_bytes, a.batch, a.total_q, slot, &stretch,
                                                             &item->begin, &first, &end)
                                      : find_tile<kRows>(a.q_offsets, a.offset_bytes, a.batch, a.total_q, slot, &stretch,
                                                         &item->begin, &first, &end);
  if (!ok) return false;
  other_rows(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch, &item->k0, &item->klen);
  item->row0 = static_cast<int>(first);
  item->qlen = static_cast<int>(end - item->begin);
  item->head = static_cast<int>(blockIdx.x % per_slot) * (pair_heads ? 2 : 1);
  return true;
}

// The next item of the list: one thread takes a ticket for the CTA. false: none are left.
__device__ __forceinline__ bool list_item(const FwdDev& p, int per_slot, bool pair_heads, int* ticket, Item* item) {
  const AttnDev& a = p.a;
  if (threadIdx.x == 0) *ticket = atomicAdd(p.plan.tickets, 1);
  __syncthreads();
  const int t = *ticket;
  if (t / per_slot >= min(p.plan.counts[0], p.plan.q_room)) return false;
  const int2 at = p.plan.q_tiles[t / per_slot];
  item->begin = stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, at.x);
  item->qlen = static_cast<int>(stretch_bound(a.q_offsets, a.offset_bytes, a.batch, a.total_q, at.x + 1) - item->begin);
  other_rows(a.k_offsets, a.offset_bytes, a.batch, a.total_k, at.x, &item->k0, &item->klen);
  item->row0 = at.y * kRows;
  item->head = t % per_slot * (pair_heads ? 2 : 1);
  return true;
}

template <bool kBf16, int kDP, int kNQ>
__global__ void __launch_bounds__(Layout<kDP, kNQ>::kThreads, Layout<kDP, kNQ>::kCtas)
    attention_fwd_kernel(const FwdDev p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map) {
  using L = Layout<kDP, kNQ>;
  extern __shared__ uint8_t raw[];
  __shared__ Shared bars;
  __shared__ int ticket;
  const AttnDev& a = p.a;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* qs = smem;
  uint8_t* ks = qs + kNQ * L::kTileBytes;
  uint8_t* vs = ks + L::kStages * L::kTileBytes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  const bool pair_heads = kNQ == 2 && p.pair_heads;
  const int per_slot = pair_heads ? a.heads / 2 : a.heads;
  Item item;
  if (!p.listed && !slot_item<kNQ == 2>(p, pair_heads, per_slot, &item)) return;
  if (threadIdx.x == 0) bars.dead = 0;
  if (warp == kNQ * 4) tmem_alloc(&bars.tmem, L::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  volatile int* dead = &bars.dead;

  if (warp >= kNQ * 4) {
    give_registers<L::kOtherRegs>();
    for (bool fresh = true; !*dead && (p.listed ? list_item(p, per_slot, pair_heads, &ticket, &item) : fresh); fresh = false) {
      const int64_t begin = item.begin;
      const int head = item.head, kv = head / a.group, klen = item.klen, qlen = item.qlen, row0 = item.row0, shift = klen - qlen;
      const int64_t k0 = item.k0;
      // key tiles that the streams' rows see
      int n[kNQ];
#pragma unroll
      for (int s = 0; s < kNQ; ++s) {
        const int from = row0 + (pair_heads ? 0 : s * kRows);
        const int sees = a.causal ? min(klen, min(qlen, from + kRows) + shift) : klen;
        n[s] = from < qlen && sees > 0 ? (sees + kRows - 1) / kRows : 0;
      }
      const int most = kNQ == 2 ? max(n[0], n[kNQ - 1]) : n[0];
      __syncthreads();   // the barriers are set up
      if (warp == kNQ * 4 + 1) {
        // ---- copies ----
        if (lane == 0 && most > 0) {
          mbar_expect(&bars.b.q_full, kNQ * L::kTileBytes);
          for (int s = 0; s < kNQ; ++s)
            for (int x = 0; x < kDP / 64; ++x)
              tma_load_3d(smem_addr(qs) + s * L::kTileBytes + x * kRows * 128, &q_map, x * 64, head + (pair_heads ? s : 0),
                          static_cast<int>(begin) + row0 + (pair_heads ? 0 : s * kRows), &bars.b.q_full);
          for (int j = 0; j < most; ++j) {
            const int st = j % L::kStages;
            const uint32_t before = (j / L::kStages - 1) & 1;
            if (j >= L::kStages && !mbar_wait(&bars.b.k_empty[st], before, dead)) break;
            mbar_expect(&bars.b.k_full[st], L::kTileBytes);
            for (int x = 0; x < kDP / 64; ++x)
              tma_load_3d(smem_addr(ks) + st * L::kTileBytes + x * kRows * 128, &k_map, x * 64, kv, static_cast<int>(k0) + j * kRows,
                          &bars.b.k_full[st]);
            if (j >= L::kStages && !mbar_wait(&bars.b.v_empty[st], before, dead)) break;
            mbar_expect(&bars.b.v_full[st], L::kTileBytes);
            for (int x = 0; x < kDP / 64; ++x)
              tma_load_3d(smem_addr(vs) + st * L::kTileBytes + x * kRows * 128, &v_map, x * 64, kv, static_cast<int>(k0) + j * kRows,
                          &bars.b.v_full[st]);
          }
        }
      } else if (warp == kNQ * 4) {
        // ---- matrix instructions ----
        const int d_steps = (a.D + 15) / 16;
        bool alive = most == 0 || warp_wait(&bars.b.q_full, 0, dead);
        // scores of stream s with key tile j; keys past the sequence's end are not multiplied
        auto scores = [&](int s, int j) {
          const int keys = min(kRows, (klen - j * kRows + 15) & ~15);
          const uint32_t desc = mma_desc(kBf16, kRows, keys, false, false);
          const uint32_t q_at = smem_addr(qs + s * L::kTileBytes), k_at = smem_addr(ks + (j % L::kStages) * L::kTileBytes);
          mma_along_k<kDP / 16, kRows>(tmem + s * kRows, q_at, k_at, desc, d_steps);
          mma_commit(&bars.b.s_full[s]);
        };
        if (alive && most > 0) {
          alive = warp_wait(&bars.b.k_full[0], 0, dead);
          if (alive && elect_one()) {
#pragma unroll
            for (int s = 0; s < kNQ; ++s)
              if (n[s] > 0) scores(s, 0);
            if (L::kStages < most) mma_commit(&bars.b.k_empty[0]);
          }
        }
        const uint32_t pv_desc = mma_desc(kBf16, kRows, (a.D + 15) & ~15, false, true);
        for (int j = 0; alive && j < most; ++j) {
          const int st = j % L::kStages, next = (j + 1) % L::kStages;
          alive = warp_wait(&bars.b.v_full[st], (j / L::kStages) & 1, dead);
          if (!alive) break;
          const int keys = min(kRows, klen - j * kRows);
          if (keys % 16 != 0) {
            // rows of other sequences up to the next 16: their weights are zero, which would not cancel NaN
            for (int i = lane; i < (16 - keys % 16) * (kDP / 64) * 8; i += 32) {
              const int x = i / ((16 - keys % 16) * 8), rest = i % ((16 - keys % 16) * 8);
              *reinterpret_cast<uint4*>(vs + st * L::kTileBytes + x * kRows * 128 + keys * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
            __syncwarp();
          }
          const int steps = (keys + 15) / 16;
          const uint32_t v_at = smem_addr(vs + st * L::kTileBytes);
#pragma unroll
          for (int s = 0; s < kNQ; ++s) {
            if (j < n[s]) {
              alive = alive && warp_wait(&bars.b.p_full[s], j & 1, dead);
              tc_fence_after();
              if (alive && elect_one()) {
                mma_over_rows<0>(tmem + kNQ * kRows + s * kDP, tmem + s * kRows + 64, v_at, pv_desc, steps, j > 0);
                if (j + 1 == n[s]) mma_commit(&bars.b.o_full[s]);
              }
            }
            if (j + 1 < n[s]) {
              alive = alive && warp_wait(&bars.b.k_full[next], ((j + 1) / L::kStages) & 1, dead);
              if (alive && elect_one()) scores(s, j + 1);
            }
          }
          if (alive && elect_one()) {
            if (j + L::kStages < most) mma_commit(&bars.b.v_empty[st]);
            if (j + 1 + L::kStages < most) mma_commit(&bars.b.k_empty[next]);
          }
          __syncwarp();
        }
      }
      __syncthreads();
      tc_fence_after();
    }
  } else {
    take_registers<L::kSoftmaxRegs>();
    for (bool fresh = true; !*dead && (p.listed ? list_item(p, per_slot, pair_heads, &ticket, &item) : fresh); fresh = false) {
      const int64_t begin = item.begin;
      const int head = item.head, klen = item.klen, qlen = item.qlen, row0 = item.row0, shift = klen - qlen;
      // key tiles that the streams' rows see
      int n[kNQ];
#pragma unroll
      for (int s = 0; s < kNQ; ++s) {
        const int from = row0 + (pair_heads ? 0 : s * kRows);
        const int sees = a.causal ? min(klen, min(qlen, from + kRows) + shift) : klen;
        n[s] = from < qlen && sees > 0 ? (sees + kRows - 1) / kRows : 0;
      }
      const int most = kNQ == 2 ? max(n[0], n[kNQ - 1]) : n[0];
      if (threadIdx.x == 0) {
        if (!fresh) mbar_forget(&bars.b);
        mbar_init(&bars.b.q_full, 1);
        for (int i = 0; i < 2; ++i) {
          mbar_init(&bars.b.k_full[i], 1);
          mbar_init(&bars.b.k_empty[i], 1);
          mbar_init(&bars.b.v_full[i], 1);
          mbar_init(&bars.b.v_empty[i], 1);
          mbar_init(&bars.b.s_full[i], 1);
          mbar_init(&bars.b.p_full[i], 128);
          mbar_init(&bars.b.o_full[i], 1);
        }
        fence_barrier_init();
      }
      __syncthreads();
      // ---- softmax: thread = row ----
      const int s = warp / 4;
      const int local = (warp % 4) * 32 + lane;
      const int row = row0 + (pair_heads ? 0 : s * kRows) + local;
      const int tiles = n[kNQ == 2 ? s : 0];
      const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
      const uint32_t s_at = tmem + lanes + s * kRows, o_at = tmem + lanes + kNQ * kRows + s * kDP;
      const int limit = row >= qlen ? 0 : (a.causal ? min(klen, row + shift + 1) : klen);   // keys that the row sees
      const float c = a.scale * 1.4426950408889634f;
      float top = -INFINITY, base = 0.f;   // the maximum in use, times c
      float sum = 0.f;
      bool alive = true;
      for (int j = 0; j < tiles; ++j) {
        alive = warp_wait(&bars.b.s_full[s], j & 1, dead);
        if (!alive) break;
        tc_fence_after();
        const int left = limit - j * kRows;                        // of this tile, for this row
        // 32 columns each, of the tile; a warp whose rows are all behind the last computes nothing
        const int chunks = row - lane < qlen ? min(4, (klen - j * kRows + 31) / 32) : 0;
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
            base = now == -INFINITY ? 0.f : now * c;
          } else if (__any_sync(kFullMask, now * c > base + 8.f)) {
            top = fmaxf(top, now);
            const float next = top == -INFINITY ? 0.f : top * c, keep = fast_exp2(base - next);
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
        mbar_arrive(&bars.b.p_full[s]);
      }
      // ---- result ----
      if (alive && tiles > 0) alive = warp_wait(&bars.b.o_full[s], 0, dead);
      tc_fence_after();
      const int h = head + (pair_heads ? s : 0);
      if (tiles == 0 && most > 0) warp_wait(&bars.b.q_full, 0, dead);
      if (row - lane < qlen) {   // through the queries' place: they have come, and all products with them are done
        uint16_t* out = static_cast<uint16_t*>(a.out) + (begin + row - lane) * a.o_row + h * a.o_head;
#pragma unroll 1
        for (int i = 0; i < kDP; i += 32) {
          uint32_t o[32];
          if (tiles > 0) {
            tmem_ld32(o, o_at + i);
            tmem_wait_ld();
          }
          store_columns<kBf16>(qs + s * L::kTileBytes + warp % 4 * 2048, o, 1.f / sum, sum == 0.f || tiles == 0, out, a.o_row,
                               qlen - row + lane, i, a.D);
        }
      }
      fence_async_smem();
      if (a.lse != nullptr && row < qlen)
        a.lse[h * a.total_q + begin + row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
    }
  }
  if (bars.dead) {
    // a wait gave up: report it, and let what is in flight land before the memory is given back
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, B200TBE_DEV_WAIT_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  tc_fence_after();
  if (warp == kNQ * 4) tmem_free(tmem, L::kColumns);
}

template <bool kBf16, int kDP, int kNQ>
int launch(const FwdDev& p, int64_t slots, cudaStream_t stream) {
  using L = Layout<kDP, kNQ>;
  const AttnDev& a = p.a;
  CUtensorMap q, k, v;
  if (!rows_map(&q, kBf16, a.q, a.total_q, a.heads, a.D, a.q_row, a.q_head, kRows) ||
      !rows_map(&k, kBf16, a.k, a.total_k, a.kv_heads, a.D, a.k_row, a.k_head, kRows) ||
      !rows_map(&v, kBf16, a.v, a.total_k, a.kv_heads, a.D, a.v_row, a.v_head, kRows))
    return B200TBE_ERR_UNSUPPORTED;
  int64_t blocks = slots * (p.pair_heads && kNQ == 2 ? a.heads / 2 : a.heads);
  if (blocks > 0x7fffff00) return p.listed ? B200TBE_ERR_UNSUPPORTED : B200TBE_ERR_TOO_LARGE;
  if (p.listed && blocks > kNumSMs * L::kCtas) blocks = kNumSMs * L::kCtas;
  const auto kernel = attention_fwd_kernel<kBf16, kDP, kNQ>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess)
    return B200TBE_ERR_LAUNCH;
  kernel<<<static_cast<unsigned>(blocks), L::kThreads, L::kSmem, stream>>>(p, q, k, v);
  return launch_status();
}

template <bool kBf16>
int forward_of(const FwdDev& p, bool two, cudaStream_t stream) {
  const AttnDev& a = p.a;
  const int64_t slots = two && !p.pair_heads ? tile_slots<2 * kRows>(a.total_q, a.batch) : tile_slots<kRows>(a.total_q, a.batch);
  if (a.D <= 64) return two ? launch<kBf16, 64, 2>(p, slots, stream) : launch<kBf16, 64, 1>(p, slots, stream);
  return two ? launch<kBf16, 128, 2>(p, slots, stream) : launch<kBf16, 128, 1>(p, slots, stream);
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
  FwdDev p{a, a.group % 2 == 0, status, list != nullptr, list != nullptr ? *list : TileList{}};
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
