// The first launch of a backward pass: delta[head][row] = sum over d of dO * O, and the list of tiles that the
// tensor-core kernels take.
#include "attention.cuh"

namespace b200tbe {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;   // of a tile

// How much work a tile of the stretch is, coarsely.
__device__ __forceinline__ int weight_class(int64_t rows) { return rows >= 2048 ? 2 : rows >= 512 ? 1 : 0; }

// Both lists by one CTA: the stretches' tiles are counted, summed up to each stretch, and written by its warp.
// The tiles are taken in the list's order, so the long sequences' come first; within a sequence later queries see
// more keys, and earlier keys are seen by more queries: those come first.
__device__ __forceinline__ void list_tiles(const AttnDev& p, const TileList& plan) {
  __shared__ int64_t warp_sums[kThreads / 32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  __shared__ int present;
  if (threadIdx.x == 0) present = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.batch + 2; i += kThreads) {
    const int c = weight_class(stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, i + 1) -
                               stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, i));
    if (c > 0) atomicOr(&present, 1 << c);
  }
  __syncthreads();
  int64_t base = 0;   // tiles of queries in the low half, of keys in the high half
  const int rounds = (p.batch + 2 + kThreads - 1) / kThreads;
  for (int turn = 0; turn < 3 * rounds; ++turn) {
    const int c = 2 - turn / rounds, s0 = turn % rounds * kThreads, i = s0 + threadIdx.x;
    if (c > 0 && (present >> c & 1) == 0) continue;
    int64_t mine = 0;
    if (i < p.batch + 2) {
      const int64_t q = stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, i + 1) -
                        stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, i);
      const int64_t k = stretch_bound(p.k_offsets, p.offset_bytes, p.batch, p.total_k, i + 1) -
                        stretch_bound(p.k_offsets, p.offset_bytes, p.batch, p.total_k, i);
      if (weight_class(q) == c)
        mine = max(static_cast<int64_t>(0), (q + kRows - 1) / kRows) + (max(static_cast<int64_t>(0), (k + kRows - 1) / kRows) << 32);
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(kFullMask, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) upto += warp_sums[w];
      all += warp_sums[w];
    }
    const int64_t at = base + upto - mine;
    auto write = [&](int stretch, int64_t n, int64_t to, int t0, int step) {
      const int nq = static_cast<int>(n & 0xffffffff), nk = static_cast<int>(n >> 32);
      const int tq = static_cast<int>(to & 0xffffffff), tk = static_cast<int>(to >> 32);
      // offsets that decrease give more tiles than there is room for
      for (int t = t0; t < nq; t += step)
        if (tq + t < plan.q_room) plan.q_tiles[tq + t] = make_int2(stretch, nq - 1 - t);
      for (int t = t0; t < nk; t += step)
        if (tk + t < plan.k_room) plan.k_tiles[tk + t] = make_int2(stretch, t);
    };
    // few tiles by the stretch's thread, many by its warp
    const bool many = (mine & 0xffffffff) > 4 || (mine >> 32) > 4;
    if (!many) write(i, mine, at, 0, 1);
    for (unsigned left = __ballot_sync(kFullMask, many); left != 0; left &= left - 1) {
      const int l = __ffs(left) - 1;
      write(s0 + warp * 32 + l, __shfl_sync(kFullMask, mine, l), __shfl_sync(kFullMask, at, l), lane, 32);
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    plan.tickets[0] = plan.tickets[1] = 0;
    plan.counts[0] = min(static_cast<int>(base & 0xffffffff), plan.q_room);
    plan.counts[1] = min(static_cast<int>(base >> 32), plan.k_room);
  }
}

// Group of kLanes lanes for a row of one head, a vector of kElems elements each; block 0 lists the tiles.
template <typename T, int kElems, int kLanes>
__global__ void __launch_bounds__(kThreads) delta_kernel(const AttnDev p, const TileList plan) {
  if (blockIdx.x == 0) {
    list_tiles(p, plan);
    return;
  }
  struct __align__(sizeof(T) * kElems) Vec {
    T x[kElems];
  };
  const int64_t at = static_cast<int64_t>(blockIdx.x - 1) * (kThreads / kLanes) + threadIdx.x / kLanes;
  const bool in = at < p.total_q * p.heads;
  // 64-bit divisions would cost more than the rest
  const int64_t row = !in ? 0 : at >> 32 == 0 ? static_cast<uint32_t>(at) / static_cast<uint32_t>(p.heads) : at / p.heads;
  const int head = in ? static_cast<int>(at - row * p.heads) : 0;
  const T* g = static_cast<const T*>(p.grad) + row * p.g_row + head * p.g_head;
  const T* o = static_cast<const T*>(p.out) + row * p.o_row + head * p.o_head;
  float s = 0.f;
  for (int d = threadIdx.x % kLanes * kElems; in && d < p.D; d += kLanes * kElems) {
    const Vec x = *reinterpret_cast<const Vec*>(g + d), y = *reinterpret_cast<const Vec*>(o + d);
#pragma unroll
    for (int e = 0; e < kElems; ++e) s = fmaf(to_float<T>(x.x[e]), to_float<T>(y.x[e]), s);
  }
#pragma unroll
  for (int w = kLanes / 2; w > 0; w >>= 1) s += __shfl_xor_sync(kFullMask, s, w);
  if (in && threadIdx.x % kLanes == 0) p.delta[head * p.total_q + row] = s;
}

// The same for the rows of the listed tiles alone.
template <typename T, int kElems, int kLanes>
__global__ void __launch_bounds__(kThreads) delta_listed_kernel(const AttnDev p, const TileList list) {
  struct __align__(sizeof(T) * kElems) Vec {
    T x[kElems];
  };
  const int64_t all = static_cast<int64_t>(min(list.counts[0], list.q_room)) * p.heads;
  for (int64_t item = blockIdx.x; item < all; item += gridDim.x) {
    const int2 tile = list.q_tiles[item / p.heads];
    const int head = static_cast<int>(item % p.heads);
    const int64_t first = stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, tile.x) + tile.y * kRows;
    const int64_t end = stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, tile.x + 1);
    for (int r = threadIdx.x / kLanes; r < kRows; r += kThreads / kLanes) {
      const int64_t row = first + r;
      float s = 0.f;
      if (row < end) {
        const T* g = static_cast<const T*>(p.grad) + row * p.g_row + head * p.g_head;
        const T* o = static_cast<const T*>(p.out) + row * p.o_row + head * p.o_head;
        for (int d = threadIdx.x % kLanes * kElems; d < p.D; d += kLanes * kElems) {
          const Vec x = *reinterpret_cast<const Vec*>(g + d), y = *reinterpret_cast<const Vec*>(o + d);
#pragma unroll
          for (int e = 0; e < kElems; ++e) s = fmaf(to_float<T>(x.x[e]), to_float<T>(y.x[e]), s);
        }
      }
#pragma unroll
      for (int w = kLanes / 2; w > 0; w >>= 1) s += __shfl_xor_sync(kFullMask, s, w);
      if (row < end && threadIdx.x % kLanes == 0) p.delta[head * p.total_q + row] = s;
    }
  }
}

template <typename T, int kElems, int kLanes>
int launch(const AttnDev& p, const TileList& plan, cudaStream_t stream) {
  constexpr int kPerBlock = kThreads / kLanes;
  const int64_t blocks = (p.total_q * p.heads + kPerBlock - 1) / kPerBlock + 1;
  if (blocks > 0x7fffffff) return B200TBE_ERR_TOO_LARGE;
  delta_kernel<T, kElems, kLanes><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p, plan);
  return launch_status();
}

template <typename T>
int delta_of(const AttnDev& p, const TileList& plan, cudaStream_t stream) {
  constexpr int kElems = 16 / sizeof(T);
  const bool vectors = aligned_to(p.grad, 16) && aligned_to(p.out, 16) && p.D % kElems == 0 && p.g_row % kElems == 0 &&
                       p.g_head % kElems == 0 && p.o_row % kElems == 0 && p.o_head % kElems == 0;
  if (!vectors) return launch<T, 1, 32>(p, plan, stream);
  if (p.D <= 4 * kElems) return launch<T, kElems, 4>(p, plan, stream);
  if (p.D <= 8 * kElems) return launch<T, kElems, 8>(p, plan, stream);
  return launch<T, kElems, 16>(p, plan, stream);
}

}  // namespace

int attention_delta_listed(const AttnDev& p, const TileList& list, int dtype, cudaStream_t stream) {
  // 16-byte vectors: the tensor-core kernels that use the list have checked the strides
  const int64_t most = static_cast<int64_t>(list.q_room) * p.heads;
  const unsigned blocks = static_cast<unsigned>(most < kNumSMs * 8 ? most : kNumSMs * 8);
  if (dtype == B200TBE_FP16)
    delta_listed_kernel<__half, 8, 8><<<blocks, kThreads, 0, stream>>>(p, list);
  else
    delta_listed_kernel<__nv_bfloat16, 8, 8><<<blocks, kThreads, 0, stream>>>(p, list);
  return launch_status();
}

int attention_delta(const AttnDev& p, const TileList& plan, int dtype, cudaStream_t stream) {
  if (dtype == B200TBE_FP32) return delta_of<float>(p, plan, stream);
  if (dtype == B200TBE_FP16) return delta_of<__half>(p, plan, stream);
  return delta_of<__nv_bfloat16>(p, plan, stream);
}

}  // namespace b200tbe
