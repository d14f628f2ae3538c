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
};

template <int kDP, int kNQ>
struct Layout {
  static constexpr int kTileBytes = kRows * kDP * 2;
  static constexpr int kStages = kNQ == 1 && kDP == 128 ? 1 : 2;
  static constexpr int kSmem = (kNQ + 2 * kStages) * kTileBytes + 1024;
  static constexpr int kThreads = kNQ * 128 + 128;
  // registers: 168 x 384 threads are launched as 208 + 208 + 80 a warpgroup, 128 x 256 as 176 + 80
  static constexpr int kSoftmaxRegs = kNQ == 1 ? 176 : 208;
  static constexpr int kColumns = kNQ == 1 ? 256 : 512;
  static constexpr int kCtas = kNQ == 1 ? 2 : 1;   // per SM
};

struct Barriers {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
  int dead;
};

template <bool kBf16, int kDP, int kNQ>
__global__ void __launch_bounds__(Layout<kDP, kNQ>::kThreads, Layout<kDP, kNQ>::kCtas)
    attention_fwd_kernel(const FwdDev p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map) {
  using L = Layout<kDP, kNQ>;
  extern __shared__ uint8_t raw[];
  __shared__ Barriers bars;
  const AttnDev& a = p.a;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* qs = smem;
  uint8_t* ks = qs + kNQ * L::kTileBytes;
  uint8_t* vs = ks + L::kStages * L::kTileBytes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  const bool pair_heads = kNQ == 2 && p.pair_heads;
  const int per_slot = pair_heads ? a.heads / 2 : a.heads;
  const int64_t slots = gridDim.x / per_slot;
  // later tiles of a sequence see more keys: they go first
  const int64_t slot = a.causal ? slots - 1 - blockIdx.x / per_slot : blockIdx.x / per_slot;
  const int head = static_cast<int>(blockIdx.x % per_slot) * (pair_heads ? 2 : 1), kv = head / a.group;
  int32_t stretch;
  int64_t begin, first, end;
  const bool ok = kNQ == 2 && !pair_heads
                      ? find_tile<2 * kRows>(a.q_offsets, a.offset_bytes, a.batch, a.total_q, slot, &stretch, &begin, &first, &end)
                      : find_tile<kRows>(a.q_offsets, a.offset_bytes, a.batch, a.total_q, slot, &stretch, &begin, &first, &end);
  if (!ok) return;
  int64_t k0;
  int32_t klen;
  other_rows(a.k_offsets, a.offset_bytes, a.batch, a.total_k, stretch, &k0, &klen);
  const int qlen = static_cast<int>(end - begin), row0 = static_cast<int>(first), shift = klen - qlen;
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
    mbar_init(&bars.q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_full[i], 1);
    }
    bars.dead = 0;
    fence_barrier_init();
  }
  if (warp == kNQ * 4) tmem_alloc(&bars.tmem, L::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  volatile int* dead = &bars.dead;

  if (warp >= kNQ * 4) {
  give_registers<80>();
  if (warp == kNQ * 4 + 1) {
    // ---- copies ----
    if (lane == 0 && most > 0) {
      mbar_expect(&bars.q_full, kNQ * L::kTileBytes);
      for (int s = 0; s < kNQ; ++s)
        for (int x = 0; x < kDP / 64; ++x)
          tma_load_3d(qs + s * L::kTileBytes + x * kRows * 128, &q_map, x * 64, head + (pair_heads ? s : 0),
                      static_cast<int>(begin) + row0 + (pair_heads ? 0 : s * kRows), &bars.q_full);
      for (int j = 0; j < most; ++j) {
        const int st = j % L::kStages;
        const uint32_t before = (j / L::kStages - 1) & 1;
        if (j >= L::kStages && !mbar_wait(&bars.k_empty[st], before, dead)) break;
        mbar_expect(&bars.k_full[st], L::kTileBytes);
        for (int x = 0; x < kDP / 64; ++x)
          tma_load_3d(ks + st * L::kTileBytes + x * kRows * 128, &k_map, x * 64, kv, static_cast<int>(k0) + j * kRows,
                      &bars.k_full[st]);
        if (j >= L::kStages && !mbar_wait(&bars.v_empty[st], before, dead)) break;
        mbar_expect(&bars.v_full[st], L::kTileBytes);
        for (int x = 0; x < kDP / 64; ++x)
          tma_load_3d(vs + st * L::kTileBytes + x * kRows * 128, &v_map, x * 64, kv, static_cast<int>(k0) + j * kRows,
                      &bars.v_full[st]);
      }
    }
  } else if (warp == kNQ * 4) {
    // ---- matrix instructions ----
    const int d_steps = (a.D + 15) / 16;
    bool alive = most == 0 || warp_wait(&bars.q_full, 0, dead);
    // scores of stream s with key tile j; keys past the sequence's end are not multiplied
    auto scores = [&](int s, int j) {
      const int keys = min(kRows, (klen - j * kRows + 15) & ~15);
      const uint32_t desc = mma_desc(kBf16, kRows, keys, false, false);
      const uint32_t q_at = smem_addr(qs + s * L::kTileBytes), k_at = smem_addr(ks + (j % L::kStages) * L::kTileBytes);
      for (int d = 0; d < d_steps; ++d) {
        const uint32_t off = (d / 4) * kRows * 128 + (d % 4) * 32;
        mma_ss(tmem + s * kRows, smem_desc(q_at + off, 16), smem_desc(k_at + off, 16), desc, d > 0);
      }
      mma_commit(&bars.s_full[s]);
    };
    if (alive && most > 0) {
      alive = warp_wait(&bars.k_full[0], 0, dead);
      if (alive && lane == 0) {
#pragma unroll
        for (int s = 0; s < kNQ; ++s)
          if (n[s] > 0) scores(s, 0);
        if (L::kStages < most) mma_commit(&bars.k_empty[0]);
      }
    }
    const uint32_t pv_desc = mma_desc(kBf16, kRows, (a.D + 15) & ~15, false, true);
    for (int j = 0; alive && j < most; ++j) {
      const int st = j % L::kStages, next = (j + 1) % L::kStages;
      alive = warp_wait(&bars.v_full[st], (j / L::kStages) & 1, dead);
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
          alive = alive && warp_wait(&bars.p_full[s], j & 1, dead);
          tc_fence_after();
          if (alive && lane == 0) {
            for (int t = 0; t < steps; ++t)
              mma_ts(tmem + kNQ * kRows + s * kDP, tmem + s * kRows + t * 8, smem_desc(v_at + t * 2048, kRows * 128), pv_desc,
                     j > 0 || t > 0);
            if (j + 1 == n[s]) mma_commit(&bars.o_full[s]);
          }
        }
        if (j + 1 < n[s]) {
          alive = alive && warp_wait(&bars.k_full[next], ((j + 1) / L::kStages) & 1, dead);
          if (alive && lane == 0) scores(s, j + 1);
        }
      }
      if (alive && lane == 0) {
        if (j + L::kStages < most) mma_commit(&bars.v_empty[st]);
        if (j + 1 + L::kStages < most) mma_commit(&bars.k_empty[next]);
      }
      __syncwarp();
    }
  }
  } else {
    // ---- softmax: thread = row ----
    take_registers<L::kSoftmaxRegs>();
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
      alive = warp_wait(&bars.s_full[s], j & 1, dead);
      if (!alive) break;
      tc_fence_after();
      const int left = limit - j * kRows;                        // of this tile, for this row
      const int chunks = min(4, (klen - j * kRows + 31) / 32);   // 32 columns each, of the tile
      uint32_t x[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < chunks) tmem_ld32(x[i], s_at + i * 32);
      tmem_wait_ld();
      if (__any_sync(kFullMask, left < kRows)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (i * 32 + e >= left) x[i][e] = 0xff800000u;
      }
      float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 32; ++e) m[e % 4] = fmaxf(m[e % 4], __uint_as_float(x[i][e]));
      const float now = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      if (j == 0) {
        top = now;
        base = now == -INFINITY ? 0.f : now * c;
      } else if (__any_sync(kFullMask, now * c > base + 8.f)) {
        const float fresh = fmaxf(top, now);
        const float fresh_base = fresh == -INFINITY ? 0.f : fresh * c;
        const float keep = fast_exp2(base - fresh_base);
        top = fresh;
        base = fresh_base;
        sum *= keep;
        // the products up to the last tile are in O: they came before these scores
        for (int i = 0; i < kDP / 32; ++i) {
          uint32_t o[32];
          tmem_ld32(o, o_at + i * 32);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
          tmem_st32(o_at + i * 32, o);
        }
      }
      float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < chunks) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float p0 = fast_exp2(fmaf(__uint_as_float(x[i][e]), c, -base));
            const float p1 = fast_exp2(fmaf(__uint_as_float(x[i][e + 1]), c, -base));
            add[e % 4] += p0;
            add[e % 4 + 1] += p1;
            w[e / 2] = pack2<kBf16>(p0, p1);
          }
          tmem_st16(s_at + i * 16, w);
        }
      }
      sum += (add[0] + add[1]) + (add[2] + add[3]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars.p_full[s]);
    }
    // ---- result ----
    if (alive && tiles > 0) alive = warp_wait(&bars.o_full[s], 0, dead);
    tc_fence_after();
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int h = head + (pair_heads ? s : 0);
    uint16_t* out = static_cast<uint16_t*>(a.out) + (begin + row) * a.o_row + h * a.o_head;
#pragma unroll 1
    for (int i = 0; i < kDP / 32; ++i) {
      uint32_t o[32];
      if (alive && tiles > 0) {
        tmem_ld32(o, o_at + i * 32);
        tmem_wait_ld();
      }
      if (row < qlen) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (i * 32 + e < a.D) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (sum != 0.f) {
              v.x = pack2<kBf16>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
              v.y = pack2<kBf16>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
              v.z = pack2<kBf16>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
              v.w = pack2<kBf16>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            }
            *reinterpret_cast<uint4*>(out + i * 32 + e) = v;
          }
        }
      }
    }
    if (a.lse != nullptr && row < qlen)
      a.lse[h * a.total_q + begin + row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
    tc_fence_before();
  }
  __syncthreads();
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
  const int64_t blocks = slots * (p.pair_heads && kNQ == 2 ? a.heads / 2 : a.heads);
  if (blocks > 0x7fffffff) return B200TBE_ERR_TOO_LARGE;
  const auto kernel = attention_fwd_kernel<kBf16, kDP, kNQ>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess) return B200TBE_ERR_LAUNCH;
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

int attention_forward_tc(const AttnDev& a, int dtype, int32_t* status, cudaStream_t stream) {
  FwdDev p{a, a.group % 2 == 0, status};
  // Two query tiles a CTA read keys and values once for both and keep the tensor cores busy under the softmax.
  // Sequences so short that the second tile would mostly be empty take one tile, and two CTAs a SM.
  const bool two = p.pair_heads || a.total_q > static_cast<int64_t>(a.batch) * kRows;
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
