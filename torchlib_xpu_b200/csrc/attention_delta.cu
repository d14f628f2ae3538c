// The first launch of a backward pass: delta[head][row] = sum over d of dO * O, and the list of tiles that the
// tensor-core kernels take.
#include "attention.cuh"

namespace b200tbe {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;   // of a tile

// How much work a tile of a stretch is, to a factor of two: by the rows of the other side.
constexpr int kClasses = 8;
__device__ __forceinline__ int weight_class(int64_t rows) {
  const int64_t tiles = rows / kRows;
  return tiles <= 0 ? 0 : min(kClasses - 1, 64 - __clzll(tiles));
}

// Both lists by one CTA: the classes' tiles are counted, then every stretch takes room in its class. The tiles are taken
// in the list's order, so the long sequences' come first (which of two in a class does not matter: no result depends on
// it); within a sequence later queries see more keys, and earlier keys are seen by more queries: those come first.
__device__ __forceinline__ void list_tiles(const AttnDev& p, const TileList& list) {
  __shared__ int next[2][kClasses];   // of queries, of keys
  const int lane = threadIdx.x % 32;
  auto rows_of = [&](const void* offsets, int64_t total, int i) {
    return i >= p.batch + 2 ? static_cast<int64_t>(0)
                            : max(static_cast<int64_t>(0), stretch_bound(offsets, p.offset_bytes, p.batch, total, i + 1) -
                                                               stretch_bound(offsets, p.offset_bytes, p.batch, total, i));
  };
  if (threadIdx.x < 2 * kClasses) next[threadIdx.x / kClasses][threadIdx.x % kClasses] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < p.batch + 2; i += kThreads) {
    const int64_t q = rows_of(p.q_offsets, p.total_q, i), k = rows_of(p.k_offsets, p.total_k, i);
    const int c = weight_class(max(q, k));
    if (q > 0) atomicAdd(&next[0][c], static_cast<int>((q + kRows - 1) / kRows));
    if (k > 0) atomicAdd(&next[1][c], static_cast<int>((k + kRows - 1) / kRows));
  }
  __syncthreads();
  if (threadIdx.x < 2) {   // where the classes begin, the heaviest first
    int at = 0;
    for (int c = kClasses - 1; c >= 0; --c) {
      const int n = next[threadIdx.x][c];
      next[threadIdx.x][c] = at;
      at += n;
    }
    list.tickets[threadIdx.x] = 0;
    // offsets that decrease give more tiles than there is room for
    list.counts[threadIdx.x] = min(at, threadIdx.x == 0 ? list.q_room : list.k_room);
  }
  __syncthreads();
  auto write = [&](int stretch, int nq, int nk, int tq, int tk, int first, int step) {
    for (int t = first; t < nq; t += step)
      if (static_cast<unsigned>(tq + t) < static_cast<unsigned>(list.q_room)) list.q_tiles[tq + t] = make_int2(stretch, nq - 1 - t);
    for (int t = first; t < nk; t += step)
      if (static_cast<unsigned>(tk + t) < static_cast<unsigned>(list.k_room)) list.k_tiles[tk + t] = make_int2(stretch, t);
  };
  for (int i0 = 0; i0 < p.batch + 2; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const int64_t q = rows_of(p.q_offsets, p.total_q, i), k = rows_of(p.k_offsets, p.total_k, i);
    const int c = weight_class(max(q, k)), nq = static_cast<int>((q + kRows - 1) / kRows), nk = static_cast<int>((k + kRows - 1) / kRows);
    const int tq = nq > 0 ? atomicAdd(&next[0][c], nq) : 0, tk = nk > 0 ? atomicAdd(&next[1][c], nk) : 0;
    // few tiles by the stretch's thread, many by its warp
    const bool many = nq > 4 || nk > 4;
    if (!many) write(i, nq, nk, tq, tk, 0, 1);
    for (unsigned left = __ballot_sync(kFullMask, many); left != 0; left &= left - 1) {
      const int l = __ffs(left) - 1;
      write(i - lane + l, __shfl_sync(kFullMask, nq, l), __shfl_sync(kFullMask, nk, l), __shfl_sync(kFullMask, tq, l),
            __shfl_sync(kFullMask, tk, l), lane, 32);
    }
  }
}

__global__ void __launch_bounds__(kThreads) list_kernel(const AttnDev p, const TileList plan) { list_tiles(p, plan); }

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

// Into the word goes the largest of the warp's numbers, none of which is below zero. Which of them comes last does not matter.
__device__ __forceinline__ void keep_largest(uint32_t* word, float x) {
  const uint32_t bits = __reduce_max_sync(kFullMask, __float_as_uint(x));
  if (threadIdx.x % 32 == 0 && bits > __ldcg(word)) atomicMax(word, bits);
}

// The same for the rows of the listed tiles alone, kLanes x kElems columns or fewer; with kNorms also the norms of their dO
// and of their values.
template <typename T, int kElems, int kLanes, bool kNorms>
__global__ void __launch_bounds__(kThreads) delta_listed_kernel(const AttnDev p, const TileList list) {
  struct __align__(sizeof(T) * kElems) Vec {
    T x[kElems];
  };
  constexpr int kEach = kThreads / kLanes, kAtOnce = 4;   // rows at once, a group of lanes' rows on their way
  const int d = threadIdx.x % kLanes * kElems, r0 = threadIdx.x / kLanes;
  const bool in = d < p.D;
  const int64_t all = static_cast<int64_t>(min(list.counts[0], list.q_room)) * p.heads;
  for (int64_t item = blockIdx.x; item < all; item += gridDim.x) {
    const int2 tile = list.q_tiles[item / p.heads];
    const int head = static_cast<int>(item % p.heads);
    const int64_t first = stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, tile.x) + tile.y * kRows;
    const int64_t end = stretch_bound(p.q_offsets, p.offset_bytes, p.batch, p.total_q, tile.x + 1);
    float most = 0.f;
#pragma unroll 1
    for (int r = r0; r < kRows; r += kAtOnce * kEach) {
      Vec x[kAtOnce], y[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int64_t row = first + r + u * kEach;
        x[u] = y[u] = Vec{};
        if (row < end && in) {
          x[u] = *reinterpret_cast<const Vec*>(static_cast<const T*>(p.grad) + row * p.g_row + head * p.g_head + d);
          y[u] = *reinterpret_cast<const Vec*>(static_cast<const T*>(p.out) + row * p.o_row + head * p.o_head + d);
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int64_t row = first + r + u * kEach;
        float s = 0.f, norm = 0.f;
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
          s = fmaf(to_float<T>(x[u].x[e]), to_float<T>(y[u].x[e]), s);
          if constexpr (kNorms) norm = fmaf(to_float<T>(x[u].x[e]), to_float<T>(x[u].x[e]), norm);
        }
#pragma unroll
        for (int w = kLanes / 2; w > 0; w >>= 1) {
          s += __shfl_xor_sync(kFullMask, s, w);
          if constexpr (kNorms) norm += __shfl_xor_sync(kFullMask, norm, w);
        }
        if (row < end && threadIdx.x % kLanes == 0) p.delta[head * p.total_q + row] = s;
        most = fmaxf(most, norm);
      }
    }
    if constexpr (kNorms) keep_largest(list.grad_norms + static_cast<int64_t>(tile.x) * p.heads + head, most);
  }
  if constexpr (kNorms) {
    const int64_t values = static_cast<int64_t>(min(list.counts[1], list.k_room)) * p.kv_heads;
    for (int64_t item = blockIdx.x; item < values; item += gridDim.x) {
      const int2 tile = list.k_tiles[item / p.kv_heads];
      const int head = static_cast<int>(item % p.kv_heads);
      const int64_t first = stretch_bound(p.k_offsets, p.offset_bytes, p.batch, p.total_k, tile.x) + tile.y * kRows;
      const int64_t end = stretch_bound(p.k_offsets, p.offset_bytes, p.batch, p.total_k, tile.x + 1);
      float most = 0.f;
#pragma unroll 1
      for (int r = r0; r < kRows; r += kAtOnce * kEach) {
        Vec x[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int64_t row = first + r + u * kEach;
          x[u] = Vec{};
          if (row < end && in) x[u] = *reinterpret_cast<const Vec*>(static_cast<const T*>(p.v) + row * p.v_row + head * p.v_head + d);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          float norm = 0.f;
#pragma unroll
          for (int e = 0; e < kElems; ++e) norm = fmaf(to_float<T>(x[u].x[e]), to_float<T>(x[u].x[e]), norm);
#pragma unroll
          for (int w = kLanes / 2; w > 0; w >>= 1) norm += __shfl_xor_sync(kFullMask, norm, w);
          most = fmaxf(most, norm);
        }
      }
      keep_largest(list.v_norms + static_cast<int64_t>(tile.x) * p.kv_heads + head, most);
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

int attention_list(const AttnDev& p, const TileList& list, cudaStream_t stream) {
  list_kernel<<<1, kThreads, 0, stream>>>(p, list);
  return launch_status();
}

int attention_delta_listed(const AttnDev& p, const TileList& list, int dtype, cudaStream_t stream) {
  // 16-byte vectors: the tensor-core kernels that use the list have checked the strides
  const int64_t most = static_cast<int64_t>(list.q_room) * p.heads;
  const unsigned blocks = static_cast<unsigned>(most < kNumSMs * 8 ? most : kNumSMs * 8);
  if (dtype == B200TBE_FP16 && p.D <= 64)
    delta_listed_kernel<__half, 8, 8, true><<<blocks, kThreads, 0, stream>>>(p, list);
  else if (dtype == B200TBE_FP16)
    delta_listed_kernel<__half, 8, 16, true><<<blocks, kThreads, 0, stream>>>(p, list);
  else if (p.D <= 64)
    delta_listed_kernel<__nv_bfloat16, 8, 8, false><<<blocks, kThreads, 0, stream>>>(p, list);
  else
    delta_listed_kernel<__nv_bfloat16, 8, 16, false><<<blocks, kThreads, 0, stream>>>(p, list);
  return launch_status();
}

int attention_delta(const AttnDev& p, const TileList& plan, int dtype, cudaStream_t stream) {
  if (dtype == B200TBE_FP32) return delta_of<float>(p, plan, stream);
  if (dtype == B200TBE_FP16) return delta_of<__half>(p, plan, stream);
  return delta_of<__nv_bfloat16>(p, plan, stream);
}

}  // namespace b200tbe
