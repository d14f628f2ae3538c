// The paged key-value cache: jagged rows appended to it, and the attention of one new token over it.
#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200tbe {
namespace {

struct CacheDev {
  char* k;
  char* v;
  const int32_t* page_table;
  const void* lengths;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;   // elements
  int64_t table_stride, num_pages;
  int32_t max_pages, page_size, batch, kv_heads, D, length_bytes;
  int32_t page_shift;   // log2 of page_size, or -1
  int32_t* status;
};

__device__ __forceinline__ void raise(const CacheDev& c) {
  if (c.status != nullptr) atomicOr(c.status, B200TBE_DEV_INDEX_OUT_OF_RANGE);
}

__device__ __forceinline__ int64_t raw_length(const CacheDev& c, int b) {
  return c.length_bytes == 8 ? load_index<int64_t>(c.lengths, b) : load_index<int32_t>(c.lengths, b);
}

// Positions of sequence b that its row of the page table can hold.
__device__ __forceinline__ int length_of(const CacheDev& c, int b) {
  const int64_t n = raw_length(c, b);
  const int64_t most = min(static_cast<int64_t>(c.max_pages) * c.page_size, static_cast<int64_t>(0x7fffff00));
  return n < 0 ? 0 : static_cast<int>(n > most ? most : n);
}

__device__ __forceinline__ int page_of(const CacheDev& c, int x) { return c.page_shift >= 0 ? x >> c.page_shift : x / c.page_size; }

// ---- append ----------------------------------------------------------------------------------
// A warp takes up to eight consecutive rows: lane l finds where row l goes (a search over the offsets), then the warp
// moves the rows' heads as one stream, 16 bytes a lane where everything is aligned, keys and values together. Bound by
// HBM: every row is read once and written once (27 450 rows of 8 heads of 128, bf16: 41 us, 5.5 TB/s).
struct AppendDev {
  CacheDev c;
  const char* k;
  const char* v;
  int64_t k_row, k_head, v_row, v_head;   // elements
  const void* offsets;
  int64_t total;
  int32_t offset_bytes, elem_bytes, rows_per_warp;
};

template <typename VecT>
__global__ void __launch_bounds__(256) append_kernel(const AppendDev p) {
  const int lane = threadIdx.x & 31;
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32) * p.rows_per_warp;
  if (row0 >= p.total) return;
  const int rows = static_cast<int>(min(static_cast<int64_t>(p.rows_per_warp), p.total - row0));
  int64_t page = -1;
  int32_t slot = 0;
  if (lane < rows) {
    const int64_t row = row0 + lane;
    // the last sequence that begins at or before the row
    int lo = 0, hi = p.c.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (clamped_offset(p.offsets, p.offset_bytes, mid, p.total) <= row) lo = mid; else hi = mid;
    }
    const int64_t begin = clamped_offset(p.offsets, p.offset_bytes, lo, p.total);
    const int64_t end = clamped_offset(p.offsets, p.offset_bytes, lo + 1, p.total);
    if (row >= begin && row < end) {
      const int64_t at = raw_length(p.c, lo) - (end - row);
      if (at >= 0 && at / p.c.page_size < p.c.max_pages) {
        page = __ldg(p.c.page_table + lo * p.c.table_stride + at / p.c.page_size);
        slot = static_cast<int32_t>(at % p.c.page_size);
      }
      if (page < 0 || page >= p.c.num_pages) {
        page = -1;
        raise(p.c);
      }
    }
  }
  const int per_head = p.c.D * p.elem_bytes / static_cast<int>(sizeof(VecT));
  const int vecs = per_head * p.c.kv_heads;
  const int all = vecs * rows;   // the rows of this warp as one stream of vectors
  constexpr int kUnroll = 4;
  for (int i0 = 0; i0 < all; i0 += 32 * kUnroll) {
    VecT kx[kUnroll], vx[kUnroll];
    VecT* kd[kUnroll];
    VecT* vd[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * 32 + lane;
      const int r = min(i / vecs, rows - 1);
      const int64_t pg = __shfl_sync(kFullMask, page, r);
      const int sl = __shfl_sync(kFullMask, slot, r);
      kd[u] = nullptr;
      if (i < all && pg >= 0) {
        const int w = i - r * vecs, h = w / per_head, e = w - h * per_head;
        const int64_t row = row0 + r;
        kx[u] = __ldcs(reinterpret_cast<const VecT*>(p.k + (row * p.k_row + h * p.k_head) * p.elem_bytes) + e);
        vx[u] = __ldcs(reinterpret_cast<const VecT*>(p.v + (row * p.v_row + h * p.v_head) * p.elem_bytes) + e);
        kd[u] = reinterpret_cast<VecT*>(p.c.k + (pg * p.c.k_page + sl * p.c.k_slot + h * p.c.k_head) * p.elem_bytes) + e;
        vd[u] = reinterpret_cast<VecT*>(p.c.v + (pg * p.c.v_page + sl * p.c.v_slot + h * p.c.v_head) * p.elem_bytes) + e;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (kd[u] != nullptr) {
        *kd[u] = kx[u];
        *vd[u] = vx[u];
      }
  }
}

// ---- one new token ---------------------------------------------------------------------------
//   out[h] = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),   s_t = scale q[h] . k[t]
//
// Work is counted in tiles of kTile positions of one unit: a sequence, a key head and up to kHeads of its
// query heads. All units in one line, each as long as its tiles and kUnitCost more (what beginning and ending one
// takes), are cut into equal pieces, one for each CTA, so that the GPU is evenly loaded whatever the lengths.
// (Without the unit's own cost the CTAs that got the short sequences of a mixed batch were the last by a third.) A unit inside one CTA is finished there. One that a cut divides leaves
// a piece (m, l, unnormalised sum) in each CTA's slot; a second kernel joins the pieces in their order:
//   m = max m_i,  l = sum l_i exp(m_i - m),  out = sum o_i exp(m_i - m) / l
constexpr int kTile = 64;
constexpr int kHeads = 8;
constexpr int kUnitCost = 2;
constexpr int kAnswerThreads = 128;
constexpr int kAnswerCtas = kNumSMs * 8;

// Where a CTA's piece of the line begins.
struct Start {
  int32_t unit, tile, tiles, ctas;   // unit, tile inside it, the unit's tiles, CTAs with work
  int64_t first, all;                // the unit's first place in the line, the line's length
};

struct AnswerDev {
  CacheDev c;
  const void* q;
  void* out;
  int64_t q_row, q_head, o_row, o_head;
  int32_t heads, group, per, chunks, units;   // chunks of `per` query heads a key head; units a sequence
  float scale_log2;   // scale log2 e: scores, maxima and log-sums are in powers of two
  Start* starts;     // [gridDim.x]
  float* stats;      // [2 * gridDim.x][kHeads][2]: m, l
  float* sums;       // [2 * gridDim.x][kHeads][D]
};

__device__ __forceinline__ int tiles_of(const CacheDev& c, int b) { return max(1, (length_of(c, b) + kTile - 1) / kTile); }

// Where the CTA's piece of the line begins, and its end. All threads.
__device__ __forceinline__ Start find_start(const AnswerDev& p, int64_t* end) {
  __shared__ int64_t sums[kAnswerThreads / 32];
  __shared__ Start found;
  const int n = p.c.batch, per = (n + kAnswerThreads - 1) / kAnswerThreads;
  const int b0 = min(n, static_cast<int>(threadIdx.x) * per), b1 = min(n, b0 + per);
  int64_t mine = 0;   // of these sequences' units of one kind
  for (int b = b0; b < b1; ++b) mine += tiles_of(p.c, b) + kUnitCost;
  int64_t upto = mine;   // inclusive sum over the threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(kFullMask, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kAnswerThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  all *= p.units;
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), all);
  const int64_t at = blockIdx.x < ctas ? all * blockIdx.x / ctas : all;
  *end = blockIdx.x < ctas ? all * (blockIdx.x + 1) / ctas : all;
  int64_t first = (before + upto - mine) * p.units;
  if (at >= first && at < first + mine * p.units) {
    int b = b0;
    int64_t tiles = tiles_of(p.c, b);
    while (at >= first + (tiles + kUnitCost) * p.units) {
      first += (tiles + kUnitCost) * p.units;
      tiles = tiles_of(p.c, ++b);
    }
    const int64_t u = (at - first) / (tiles + kUnitCost);
    first += u * (tiles + kUnitCost);
    found = Start{static_cast<int32_t>(b * p.units + u), static_cast<int32_t>(max(static_cast<int64_t>(0), at - first - kUnitCost)),
                  static_cast<int32_t>(tiles), static_cast<int32_t>(ctas), first, all};
  }
  __syncthreads();
  // the joining kernel may be set up meanwhile: it waits for this one's end (without a limit; nothing here waits for it)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Start s = found;
  if (at >= *end) s = Start{-1, 0, 0, static_cast<int32_t>(ctas), at, all};   // no piece
  if (threadIdx.x == 0) p.starts[blockIdx.x] = s;
  return s;
}

// Any type, head dimension and stride, in 32-bit arithmetic: scores by a thread for each position, sums by a
// thread for each column.
template <typename T, int kCols>   // columns of a thread: D <= kCols * kAnswerThreads
__global__ void __launch_bounds__(kAnswerThreads) answer_simt_kernel(const AnswerDev p) {
  extern __shared__ float smem[];
  float* qs = smem;                              // [kHeads][D]
  float* ks = qs + kHeads * p.c.D;               // [kTile][D + 1]
  __shared__ float ps[kHeads][kTile];
  __shared__ float top[kHeads], sum[kHeads], keep[kHeads];
  __shared__ int64_t k_at[kTile], v_at[kTile];   // the tile's positions in the cache, -1: none
  const int D = p.c.D, tid = threadIdx.x;
  int64_t end;
  Start s = find_start(p, &end);
  for (; s.first < end; s.first += s.tiles + kUnitCost, ++s.unit, s.tile = 0) {
    if (s.unit >= p.units * p.c.batch) break;
    s.tiles = tiles_of(p.c, s.unit / p.units);
    const int stop = static_cast<int>(min(static_cast<int64_t>(s.tiles), end - s.first - kUnitCost));
    if (stop <= s.tile) continue;
    const int b = s.unit / p.units, u = s.unit % p.units, kv = u / p.chunks;
    const int head0 = kv * p.group + (u % p.chunks) * p.per;
    const int heads = min(p.per, (kv + 1) * p.group - head0);
    const int len = length_of(p.c, b);
    __syncthreads();
    for (int i = tid; i < heads * D; i += kAnswerThreads) {
      const int h = i / D, d = i % D;
      qs[i] = to_float<T>(static_cast<const T*>(p.q)[b * p.q_row + (head0 + h) * p.q_head + d]);
    }
    if (tid < kHeads) top[tid] = -INFINITY, sum[tid] = 0.f;
    if (tid == 0 && s.tile == 0 && raw_length(p.c, b) != len) raise(p.c);
    float o[kHeads][kCols] = {};
    for (int tile = s.tile; tile < stop; ++tile) {
      __syncthreads();
      if (tid < kTile) {
        const int t = tile * kTile + tid;
        k_at[tid] = v_at[tid] = -1;
        if (t < len) {
          const int64_t page = __ldg(p.c.page_table + b * p.c.table_stride + t / p.c.page_size);
          if (page >= 0 && page < p.c.num_pages) {
            const int64_t slot = t % p.c.page_size;
            k_at[tid] = page * p.c.k_page + slot * p.c.k_slot + kv * p.c.k_head;
            v_at[tid] = page * p.c.v_page + slot * p.c.v_slot + kv * p.c.v_head;
          } else {
            raise(p.c);
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < kTile * D; i += kAnswerThreads) {
        const int t = i / D, d = i % D;
        ks[t * (D + 1) + d] = k_at[t] >= 0 ? to_float<T>(reinterpret_cast<const T*>(p.c.k)[k_at[t] + d]) : 0.f;
      }
      __syncthreads();
      for (int i = tid; i < kTile * heads; i += kAnswerThreads) {
        const int t = i % kTile, h = i / kTile;
        float x = 0.f;
        for (int d = 0; d < D; ++d) x = fmaf(qs[h * D + d], ks[t * (D + 1) + d], x);
        ps[h][t] = k_at[t] >= 0 ? x * p.scale_log2 : -INFINITY;
      }
      __syncthreads();
      for (int h = tid / 32; h < heads; h += kAnswerThreads / 32) {
        const int lane = tid & 31;
        const float a = ps[h][lane], c = ps[h][lane + 32], was = top[h];
        float m = fmaxf(was, fmaxf(a, c));
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, w));
        const float base = m == -INFINITY ? 0.f : m;
        const float ea = exp2f(a - base), ec = exp2f(c - base);
        ps[h][lane] = ea;
        ps[h][lane + 32] = ec;
        const float add = warp_sum(ea + ec);
        if (lane == 0) {
          keep[h] = exp2f(was - base);
          top[h] = m;
          sum[h] = sum[h] * keep[h] + add;
        }
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int d = c * kAnswerThreads + tid;
        if (d < D) {
#pragma unroll
          for (int h = 0; h < kHeads; ++h)
            if (h < heads) o[h][c] *= keep[h];
#pragma unroll 8
          for (int t = 0; t < kTile; ++t) {
            const float x = v_at[t] >= 0 ? to_float<T>(reinterpret_cast<const T*>(p.c.v)[v_at[t] + d]) : 0.f;
#pragma unroll
            for (int h = 0; h < kHeads; ++h)
              if (h < heads) o[h][c] = fmaf(ps[h][t], x, o[h][c]);
          }
        }
      }
    }
    __syncthreads();
    const bool whole = s.tile == 0 && stop == s.tiles;
    const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (s.tile == 0 ? 1 : 0);
    if (!whole && tid < heads) {
      p.stats[(part * kHeads + tid) * 2] = top[tid];
      p.stats[(part * kHeads + tid) * 2 + 1] = sum[tid];
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int d = c * kAnswerThreads + tid;
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        if (h < heads && d < D) {
          if (whole)
            static_cast<T*>(p.out)[b * p.o_row + (head0 + h) * p.o_head + d] = from_float<T>(sum[h] == 0.f ? 0.f : o[h][c] / sum[h]);
          else
            p.sums[(part * kHeads + h) * D + d] = o[h][c];
        }
    }
  }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// d[16][8] += a[16][16] b[16][8], fp32 sums
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Copies 16 bytes to shared memory without waiting for them; zeros where `on` is false.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

template <int kDP>
struct Ring {
  static constexpr int kKC = kDP / 32, kVC = kDP / 64;      // 16-byte pieces of a lane's fragments of a key, of a value
  static constexpr int kLanes = kDP / 8, kRows = 32 / kLanes;   // lanes that copy a row, rows of a copy
  static constexpr int kTiles = kDP == 64 ? 2 : 1;          // of a step: independent products hide one another's latency
  static constexpr int kRegion = 16 * kLanes;               // pieces of 16 keys, or values
  static constexpr int kStep = kTiles * 2 * kRegion;        // 8 KB a warp
  static constexpr int kStages = 2, kCtas = 3;              // per SM
  static constexpr int kBytes = kAnswerThreads / 32 * kStages * kStep * 16;
  static constexpr int kSumRow = kDP + 4;
  static_assert(kBytes >= kAnswerThreads / 32 * kHeads * kSumRow * 4, "the warps' sums take the ring's place");
};

// 16-bit types, head dimensions that are multiples of 8 up to kDP. A warp takes 16 positions of a tile:
//   S^T [16 positions][8 heads] = k q^T,   O^T [D][8 heads] += v^T P^T
// by warp-level matrix instructions. The order of an inner dimension is free as long as both operands share it, so
// a lane's fragments are whole 16-byte pieces of rows: for S^T, lane (g, t) of a row of four takes elements
// 8 (t + 4c) .. + 7 of position g's key, and of head g's query; for O^T it takes elements 8 (g + 8c) .. + 7 of the
// values of positions 2t, 2t + 1, 2t + 8, 2t + 9, whose pairs two byte permutes put side by side.
//
// A warp copies whole rows (16 or 8 lanes side by side) into its own part of a ring in shared memory, a step ahead.
// Bound by HBM, and sensitive to how it is asked: 64 sequences of 1 to 8191 positions, 32 heads of 128 over 8 key
// heads, take 219 us for the copies alone when each lane copies the pieces that it will use itself (64 bytes of a
// row side by side), 166 us in whole rows, where the copy rate would give 164. A piece's place in its row is
// exchanged by the row's number, differently for keys and values, so that no eight lanes meet in a bank. Warps meet
// only at the end of a unit. That case takes 173 us in this kernel, 182 with the joining of the pieces (5.9 TB/s). As in the forward pass over whole sequences the maximum in use only follows when it has
// grown by 2^8.
template <bool kBf16, int kDP>
__global__ void __launch_bounds__(kAnswerThreads, Ring<kDP>::kCtas) answer_mma_kernel(const AnswerDev p) {
  using R = Ring<kDP>;
  constexpr int kKC = R::kKC, kVC = R::kVC, kStages = R::kStages, kTiles = R::kTiles, kL = R::kLanes;
  constexpr float kLag = 8.f, kHere = kBf16 ? 0.f : kLift<kBf16> - kLag;   // all sums of a call are lifted alike, until they are divided
  extern __shared__ uint4 ring[];
  __shared__ float stats[kAnswerThreads / 32][kHeads][2];
  __shared__ longlong2 places[kAnswerThreads / 32][32];   // where the positions' keys and values begin
  float* sums = reinterpret_cast<float*>(ring);   // [warp][head][kSumRow]
  const int D = p.c.D, tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane % 4;
  const uint4* mine = ring + warp * kStages * R::kStep;
  const uint32_t mine_at = smem_addr(mine);
  int64_t end;
  Start s = find_start(p, &end);
  for (; s.first < end; s.first += s.tiles + kUnitCost, ++s.unit, s.tile = 0) {
    if (s.unit >= p.units * p.c.batch) break;
    s.tiles = tiles_of(p.c, s.unit / p.units);
    const int stop = static_cast<int>(min(static_cast<int64_t>(s.tiles), end - s.first - kUnitCost));
    if (stop <= s.tile) continue;
    const int b = s.unit / p.units, u = s.unit % p.units, kv = u / p.chunks;
    const int head0 = kv * p.group + (u % p.chunks) * p.per;
    const int heads = min(p.per, (kv + 1) * p.group - head0);
    const int len = length_of(p.c, b);
    if (tid == 0 && s.tile == 0 && raw_length(p.c, b) != len) raise(p.c);
    const uint16_t* kc = reinterpret_cast<const uint16_t*>(p.c.k) + kv * p.c.k_head;
    const uint16_t* vc = reinterpret_cast<const uint16_t*>(p.c.v) + kv * p.c.v_head;
    uint4 q[kKC];
#pragma unroll
    for (int c = 0; c < kKC; ++c) {
      const int d = 8 * (t + 4 * c);
      q[c] = make_uint4(0, 0, 0, 0);
      if (g < heads && d < D)
        q[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + b * p.q_row + (head0 + g) * p.q_head + d);
    }
    // the page and the place in it of a position of this warp's share of a step's tiles: lane % 16 of tile lane / 16;
    // place -1: behind the last
    int page, slot;
    auto locate = [&](int tile) {
      const int of = tile + (kTiles == 2 ? lane / 16 : 0), x = of * kTile + warp * 16 + (lane & 15);
      page = -1;
      slot = -1;
      if (of < stop && x < len) {
        const int n = page_of(p.c, x);
        slot = x - n * p.c.page_size;
        page = __ldg(p.c.page_table + b * p.c.table_stride + n);
      }
    };
    uint32_t part[kStages] = {};   // the lanes whose positions take part, of the steps on their way, the newest first
    auto shift_part = [&](uint32_t newest) {
#pragma unroll
      for (int i = kStages - 1; i > 0; --i) part[i] = part[i - 1];
      part[0] = newest;
    };
    auto copy = [&](int stage) {   // the step that was located last
      if (slot >= 0 && (page < 0 || page >= p.c.num_pages)) {
        page = -1;
        raise(p.c);
      }
      shift_part(__ballot_sync(kFullMask, page >= 0));
      __syncwarp();   // the places, and the stage, have been read
      places[warp][lane] = make_longlong2(page < 0 ? -1 : page * p.c.k_page + slot * p.c.k_slot,
                                          page < 0 ? -1 : page * p.c.v_page + slot * p.c.v_slot);
      __syncwarp();
      const int piece = lane % kL;
      const bool column = piece * 8 < D;
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 16 / R::kRows; ++i) {
          const int row = i * R::kRows + lane / kL;
          const longlong2 from = places[warp][j * 16 + row];
          const bool on = from.x >= 0 && column;
          const uint32_t to = mine_at + (stage * R::kStep + j * 2 * R::kRegion + row * kL) * 16;
          copy16(to + (piece ^ (4 * (row & 1))) * 16, on ? kc + from.x + piece * 8 : kc, on);
          copy16(to + (R::kRegion + (piece ^ (2 * (row / 2 % 4)))) * 16, on ? vc + from.y + piece * 8 : vc, on);
        }
    };
    float o[kVC * 4][4] = {};
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};   // of heads 2t and 2t + 1
    __syncthreads();   // the last unit's sums, which lie in the ring, have been read
    locate(s.tile);
    for (int i = 0; i < kStages - 1; ++i) {
      if (s.tile + i * kTiles < stop) copy(i); else shift_part(0);
      copies_commit();
      locate(s.tile + (i + 1) * kTiles);
    }
    int stage = 0;
    for (int tile = s.tile; tile < stop; tile += kTiles) {
      {
        const int next = stage == 0 ? kStages - 1 : stage - 1;   // (stage + kStages - 1) % kStages, read a step ago
        if (tile + (kStages - 1) * kTiles < stop) copy(next); else shift_part(0);
        copies_commit();
        locate(tile + kStages * kTiles);
      }
      copies_wait<kStages - 1>();
      __syncwarp();   // the other lanes' copies too
      const uint4* from = mine + stage * R::kStep;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const uint32_t in = part[kStages - 1];
      float x[kTiles][4] = {};
#pragma unroll
      for (int c = 0; c < kKC; ++c)
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const uint4* k = from + j * 2 * R::kRegion + g * kL + ((t + 4 * c) ^ (4 * (g & 1)));
          const uint4 k0 = k[0], k1 = k[8 * kL];
          mma16816<kBf16>(x[j], k0.x, k1.x, k0.y, k1.y, q[c].x, q[c].y);
          mma16816<kBf16>(x[j], k0.z, k1.z, k0.w, k1.w, q[c].z, q[c].w);
        }
      float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[j][i] = (in >> (j * 16 + g + i / 2 * 8) & 1) != 0 ? x[j][i] * p.scale_log2 : -INFINITY;
          most[i & 1] = fmaxf(most[i & 1], x[j][i]);
        }
      if (__any_sync(kFullMask, most[0] > top[0] + kLag || most[1] > top[1] + kLag)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = fmaxf(top[i], most[i]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, w));
          const float keep = m == -INFINITY ? 1.f : fast_exp2(top[i] - m);
          top[i] = m;
          sum[i] *= keep;
#pragma unroll
          for (int r = 0; r < kVC * 4; ++r) {
            o[r][i] *= keep;
            o[r][2 + i] *= keep;
          }
        }
      }
      uint32_t w[kTiles][2];
      const float base[2] = {top[0] == -INFINITY ? 0.f : top[0] - kHere, top[1] == -INFINITY ? 0.f : top[1] - kHere};
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[j][i] = fast_exp2(x[j][i] - base[i & 1]);
          sum[i & 1] += x[j][i];
        }
        w[j][0] = transpose8x8(pack2<kBf16>(x[j][0], x[j][1]));
        w[j][1] = transpose8x8(pack2<kBf16>(x[j][2], x[j][3]));
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int c = 0; c < kVC; ++c) {
          uint32_t a[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = from[j * 2 * R::kRegion + R::kRegion + (2 * t + (i & 1) + 8 * (i / 2)) * kL + ((g + 8 * c) ^ (2 * t))];
            a[i][0] = v.x, a[i][1] = v.y, a[i][2] = v.z, a[i][3] = v.w;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            mma16816<kBf16>(o[c * 4 + r], __byte_perm(a[0][r], a[1][r], 0x5410), __byte_perm(a[0][r], a[1][r], 0x7632),
                            __byte_perm(a[2][r], a[3][r], 0x5410), __byte_perm(a[2][r], a[3][r], 0x7632), w[j][0], w[j][1]);
        }
    }
    copies_wait<0>();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) sum[i] += __shfl_xor_sync(kFullMask, sum[i], w);
    __syncthreads();   // every warp is done with its part of the ring
    if (g < 2) {
      stats[warp][2 * t + g][0] = g == 0 ? top[0] : top[1];
      stats[warp][2 * t + g][1] = g == 0 ? sum[0] : sum[1];
    }
#pragma unroll
    for (int c = 0; c < kVC; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float2*>(&sums[(warp * kHeads + 2 * t + i) * R::kSumRow + 8 * (g + 8 * c) + 2 * r]) =
              make_float2(o[c * 4 + r][i], o[c * 4 + r][2 + i]);
    __syncthreads();
    const bool whole = s.tile == 0 && stop == s.tiles;
    const int64_t slot_of = 2 * static_cast<int64_t>(blockIdx.x) + (s.tile == 0 ? 1 : 0);
    for (int i = tid; i < heads * D; i += kAnswerThreads) {
      const int h = i / D, d = i - h * D;
      float m = stats[0][h][0];
#pragma unroll
      for (int w = 1; w < kAnswerThreads / 32; ++w) m = fmaxf(m, stats[w][h][0]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kAnswerThreads / 32; ++w) {
        const float f = fast_exp2(stats[w][h][0] - base);
        l = fmaf(f, stats[w][h][1], l);
        x = fmaf(f, sums[(w * kHeads + h) * R::kSumRow + d], x);
      }
      if (whole) {
        const uint32_t y = pack2<kBf16>(l == 0.f ? 0.f : x / l, 0.f);
        static_cast<uint16_t*>(p.out)[b * p.o_row + (head0 + h) * p.o_head + d] = static_cast<uint16_t>(y);
      } else {
        p.sums[(slot_of * kHeads + h) * D + d] = x;
        if (d == 0) {
          p.stats[(slot_of * kHeads + h) * 2] = m;
          p.stats[(slot_of * kHeads + h) * 2 + 1] = l;
        }
      }
    }
  }
}

// fp32, head dimensions that are multiples of 4 up to kDP, up to kH query heads of a key head. Eight lanes share a
// position, a warp takes four positions at once and 4 kPos a step; a lane has elements 4 (t + 8c) .. + 3 of its
// positions' keys and values, of the heads' queries (in shared memory) and of their sums. Scores are summed over the
// eight lanes by shuffles, the warp's four groups of lanes are summed at the end of a unit. Every lane copies its own
// pieces into its own places of the ring: eight lanes side by side are 128 bytes of a row.
// Bound by HBM as long as a key head has few query heads (2 D FMAs a head and position against 8 D bytes), and for short
// sequences by the chain of each unit: 300 of 0 to 400 positions, 8 heads of 48 over 4 key heads, take 36 us, of which
// the bytes are 14.
template <int kDP, int kH>
struct RingF {
  static constexpr int kC = kDP / 32;                 // 16-byte pieces of a lane for a key or a value
  static constexpr int kPos = kDP == 64 && kH > 2 ? 4 : 2;   // positions of a lane in a step
  static constexpr int kPieces = 2 * kPos * kC;
  static constexpr int kStep = kPieces * 512;         // 4 or 8 KB
  static constexpr int kStages = 3;
  static constexpr int kCtas = kH > 2 || kDP == 128 ? 2 : 4;   // per SM: few heads leave registers for more warps
  static constexpr int kSteps = 4 / kPos;             // of a tile
  static constexpr int kBytes = kAnswerThreads / 32 * kStages * kStep;
  static_assert(kBytes >= kAnswerThreads / 32 * kH * kDP * 4, "the warps' sums take the ring's place");
};

template <int kDP, int kH>
__global__ void __launch_bounds__(kAnswerThreads, RingF<kDP, kH>::kCtas) answer_fma_kernel(const AnswerDev p) {
  using R = RingF<kDP, kH>;
  constexpr int kC = R::kC, kPos = R::kPos, kStages = R::kStages;
  extern __shared__ uint4 ring[];
  __shared__ float stats[kAnswerThreads / 32][kH][2];
  __shared__ __align__(16) float qs[kH][kDP];
  float* sums = reinterpret_cast<float*>(ring);   // [warp][head][kDP]
  const int D = p.c.D, tid = threadIdx.x, lane = tid & 31, warp = tid / 32, group = lane / 8, t = lane % 8;
  const uint4* mine = ring + warp * kStages * R::kPieces * 32 + lane;
  const uint32_t mine_at = smem_addr(mine);
  int64_t end;
  Start s = find_start(p, &end);
  for (; s.first < end; s.first += s.tiles + kUnitCost, ++s.unit, s.tile = 0) {
    if (s.unit >= p.units * p.c.batch) break;
    s.tiles = tiles_of(p.c, s.unit / p.units);
    const int stop = static_cast<int>(min(static_cast<int64_t>(s.tiles), end - s.first - kUnitCost));
    if (stop <= s.tile) continue;
    const int b = s.unit / p.units, u = s.unit % p.units, kv = u / p.chunks;
    const int head0 = kv * p.group + (u % p.chunks) * p.per;
    const int heads = min(p.per, (kv + 1) * p.group - head0);
    const int len = length_of(p.c, b);
    if (tid == 0 && s.tile == 0 && raw_length(p.c, b) != len) raise(p.c);
    const float* kc = reinterpret_cast<const float*>(p.c.k) + kv * p.c.k_head;
    const float* vc = reinterpret_cast<const float*>(p.c.v) + kv * p.c.v_head;
    __syncthreads();   // the last unit's queries, and its sums, which lie in the ring, have been read
    for (int i = tid; i < kH * kDP; i += kAnswerThreads) {
      const int h = i / kDP, d = i % kDP;
      qs[h][d] = h < heads && d < D ? static_cast<const float*>(p.q)[b * p.q_row + (head0 + h) * p.q_head + d] : 0.f;
    }
    __syncthreads();
    const int first_step = s.tile * R::kSteps, last_step = stop * R::kSteps;
    // the page and the place in it of position lane % (4 kPos) of this warp's share of a step; place -1: behind the last
    int page, slot;
    auto locate = [&](int step) {
      const int x = step / R::kSteps * kTile + warp * 16 + step % R::kSteps * 4 * kPos + lane % (4 * kPos);
      page = -1;
      slot = -1;
      if (step < last_step && x < len) {
        const int n = page_of(p.c, x);
        slot = x - n * p.c.page_size;
        page = __ldg(p.c.page_table + b * p.c.table_stride + n);
      }
    };
    uint32_t part = 0;   // which of the lane's positions take part, kPos bits a step, the newest lowest
    auto copy = [&](int stage) {   // the step that was located last
      if (slot >= 0 && (page < 0 || page >= p.c.num_pages)) {
        page = -1;
        raise(p.c);
      }
      // where the position's key and value begin, in elements; -1: takes no part
      const int64_t k_at = page < 0 ? -1 : page * p.c.k_page + slot * p.c.k_slot;
      const int64_t v_at = page < 0 ? -1 : page * p.c.v_page + slot * p.c.v_slot;
      const uint32_t to = mine_at + stage * R::kStep;
#pragma unroll
      for (int i = 0; i < kPos; ++i) {
        const int64_t k_from = __shfl_sync(kFullMask, k_at, i * 4 + group), v_from = __shfl_sync(kFullMask, v_at, i * 4 + group);
        const bool in = k_from >= 0;
        part = part << 1 | (in ? 1u : 0u);
        const float* kr = kc + k_from + 4 * t;
        const float* vr = vc + v_from + 4 * t;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const bool on = in && 4 * (t + 8 * c) < D;
          copy16(to + (i * kC + c) * 512, on ? kr + 32 * c : kc, on);
          copy16(to + ((kPos + i) * kC + c) * 512, on ? vr + 32 * c : vc, on);
        }
      }
    };
    float o[kH][kC][4] = {};
    float top[kH], sum[kH];
#pragma unroll
    for (int h = 0; h < kH; ++h) top[h] = -INFINITY, sum[h] = 0.f;
    locate(first_step);
    for (int i = 0; i < kStages - 1; ++i) {
      if (first_step + i < last_step) copy(i); else part <<= kPos;
      copies_commit();
      locate(first_step + i + 1);
    }
    int stage = 0;
    for (int step = first_step; step < last_step; ++step) {
      {
        const int next = stage == 0 ? kStages - 1 : stage - 1;   // (stage + kStages - 1) % kStages, read a step ago
        if (step + kStages - 1 < last_step) copy(next); else part <<= kPos;
        copies_commit();
        locate(step + kStages);
      }
      copies_wait<kStages - 1>();
      const uint4* from = mine + stage * (R::kStep / 16);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const uint32_t in = part >> (kPos * (kStages - 1));
      float x[kH][kPos];
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        if (h < heads) {
#pragma unroll
          for (int i = 0; i < kPos; ++i) x[h][i] = 0.f;
#pragma unroll
          for (int c = 0; c < kC; ++c) {
            const float4 q = *reinterpret_cast<const float4*>(&qs[h][4 * (t + 8 * c)]);
#pragma unroll
            for (int i = 0; i < kPos; ++i) {
              const uint4 k = from[(i * kC + c) * 32];
              x[h][i] = fmaf(__uint_as_float(k.x), q.x, x[h][i]);
              x[h][i] = fmaf(__uint_as_float(k.y), q.y, x[h][i]);
              x[h][i] = fmaf(__uint_as_float(k.z), q.z, x[h][i]);
              x[h][i] = fmaf(__uint_as_float(k.w), q.w, x[h][i]);
            }
          }
          float most = -INFINITY;
#pragma unroll
          for (int i = 0; i < kPos; ++i) {
#pragma unroll
            for (int w = 1; w < 8; w <<= 1) x[h][i] += __shfl_xor_sync(kFullMask, x[h][i], w);
            x[h][i] = (in >> (kPos - 1 - i) & 1) != 0 ? x[h][i] * p.scale_log2 : -INFINITY;
            most = fmaxf(most, x[h][i]);
          }
          if (__any_sync(kFullMask, most > top[h] + 8.f)) {
            float m = fmaxf(top[h], most);
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 8));
            m = fmaxf(m, __shfl_xor_sync(kFullMask, m, 16));
            const float keep = m == -INFINITY ? 1.f : exp2f(top[h] - m);
            top[h] = m;
            sum[h] *= keep;
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[h][c][e] *= keep;
          }
          const float base = top[h] == -INFINITY ? 0.f : top[h];
#pragma unroll
          for (int i = 0; i < kPos; ++i) {
            x[h][i] = exp2f(x[h][i] - base);
            sum[h] += x[h][i];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kPos; ++i)
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const uint4 v = from[((kPos + i) * kC + c) * 32];
#pragma unroll
          for (int h = 0; h < kH; ++h)
            if (h < heads) {
              o[h][c][0] = fmaf(x[h][i], __uint_as_float(v.x), o[h][c][0]);
              o[h][c][1] = fmaf(x[h][i], __uint_as_float(v.y), o[h][c][1]);
              o[h][c][2] = fmaf(x[h][i], __uint_as_float(v.z), o[h][c][2]);
              o[h][c][3] = fmaf(x[h][i], __uint_as_float(v.w), o[h][c][3]);
            }
        }
    }
    copies_wait<0>();
    __syncthreads();   // every warp is done with its part of the ring
#pragma unroll
    for (int h = 0; h < kH; ++h)
      if (h < heads) {
#pragma unroll
        for (int w = 8; w < 32; w <<= 1) {
          sum[h] += __shfl_xor_sync(kFullMask, sum[h], w);
#pragma unroll
          for (int c = 0; c < kC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[h][c][e] += __shfl_xor_sync(kFullMask, o[h][c][e], w);
        }
        if (lane == 0) {
          stats[warp][h][0] = top[h];
          stats[warp][h][1] = sum[h];
        }
        if (group == 0) {
#pragma unroll
          for (int c = 0; c < kC; ++c)
            *reinterpret_cast<float4*>(&sums[(warp * kH + h) * kDP + 4 * (t + 8 * c)]) =
                make_float4(o[h][c][0], o[h][c][1], o[h][c][2], o[h][c][3]);
        }
      }
    __syncthreads();
    const bool whole = s.tile == 0 && stop == s.tiles;
    const int64_t slot_of = 2 * static_cast<int64_t>(blockIdx.x) + (s.tile == 0 ? 1 : 0);
    for (int i = tid; i < heads * D; i += kAnswerThreads) {
      const int h = i / D, d = i - h * D;
      float m = stats[0][h][0];
#pragma unroll
      for (int w = 1; w < kAnswerThreads / 32; ++w) m = fmaxf(m, stats[w][h][0]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kAnswerThreads / 32; ++w) {
        const float f = exp2f(stats[w][h][0] - base);
        l = fmaf(f, stats[w][h][1], l);
        x = fmaf(f, sums[(w * kH + h) * kDP + d], x);
      }
      if (whole) {
        static_cast<float*>(p.out)[b * p.o_row + (head0 + h) * p.o_head + d] = l == 0.f ? 0.f : x / l;
      } else {
        p.sums[(slot_of * kHeads + h) * D + d] = x;
        if (d == 0) {
          p.stats[(slot_of * kHeads + h) * 2] = m;
          p.stats[(slot_of * kHeads + h) * 2 + 1] = l;
        }
      }
    }
  }
}

// Block (c, h): when the cut before CTA c is the first inside a unit, the unit's head h. The pieces' weights by a thread
// each, then their sums by as many threads a column as there are.
template <typename T>
__global__ void __launch_bounds__(kAnswerThreads) join_kernel(const AnswerDev p) {
  __shared__ float weights[kAnswerCtas];
  __shared__ float shared[kAnswerThreads / 32], sums[kAnswerThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the answers' kernel is done
  const int c = blockIdx.x + 1, h = blockIdx.y, tid = threadIdx.x;
  const Start s = p.starts[c];
  if (s.unit < 0 || s.tile == 0) return;
  const Start before = p.starts[c - 1];
  if (before.unit == s.unit && before.tile > 0) return;
  const int u = s.unit % p.units, kv = u / p.chunks, b = s.unit / p.units;
  const int head = kv * p.group + (u % p.chunks) * p.per + h;
  if (h >= p.per || head >= (kv + 1) * p.group) return;
  // pieces from CTA c - 1 (in its second slot) to the one that holds the unit's last tile (in their first slots)
  const int last = static_cast<int>(((s.first + kUnitCost + s.tiles) * s.ctas - 1) / s.all);
  const int pieces = last - c + 2;
  auto piece = [&](int i) { return (2 * static_cast<int64_t>(c - 1 + i) + (i == 0 ? 1 : 0)) * kHeads + h; };
  auto over_block = [&](float x, bool largest) {
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
      const float y = __shfl_xor_sync(kFullMask, x, w);
      x = largest ? fmaxf(x, y) : x + y;
    }
    __syncthreads();
    if (tid % 32 == 0) shared[tid / 32] = x;
    __syncthreads();
    x = shared[0];
#pragma unroll
    for (int w = 1; w < kAnswerThreads / 32; ++w) x = largest ? fmaxf(x, shared[w]) : x + shared[w];
    return x;
  };
  float m = -INFINITY;
  for (int i = tid; i < pieces; i += kAnswerThreads) m = fmaxf(m, weights[i] = p.stats[piece(i) * 2]);
  m = over_block(m, true);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int i = tid; i < pieces; i += kAnswerThreads) {
    weights[i] = exp2f(weights[i] - base);
    l = fmaf(weights[i], p.stats[piece(i) * 2 + 1], l);
  }
  l = over_block(l, false);   // also: the weights are there
  const int columns = p.c.D <= 32 ? 32 : p.c.D <= 64 ? 64 : 128, shares = kAnswerThreads / columns, share = tid / columns;
  for (int d0 = 0; d0 < p.c.D; d0 += columns) {
    const int d = d0 + tid % columns;
    float o = 0.f;
    if (d < p.c.D) {
#pragma unroll 4
      for (int i = share; i < pieces; i += shares) o = fmaf(weights[i], p.sums[piece(i) * p.c.D + d], o);
    }
    __syncthreads();
    sums[tid] = o;
    __syncthreads();
    if (share == 0 && d < p.c.D) {
      for (int w = 1; w < shares; ++w) o += sums[w * columns + tid];
      static_cast<T*>(p.out)[b * p.o_row + head * p.o_head + d] = from_float<T>(l == 0.f ? 0.f : o / l);
    }
  }
}

int elem_bytes_of(int dtype) { return dtype == B200TBE_FP32 ? 4 : 2; }

int check_cache(const b200tbe_paged_cache* c) {
  if (c == nullptr) return B200TBE_ERR_BAD_ARG;
  if (c->dtype != B200TBE_FP32 && c->dtype != B200TBE_FP16 && c->dtype != B200TBE_BF16) return B200TBE_ERR_UNSUPPORTED;
  if (c->head_dim < 1 || c->head_dim > 256) return B200TBE_ERR_UNSUPPORTED;
  if (c->length_bytes != 4 && c->length_bytes != 8) return B200TBE_ERR_UNSUPPORTED;
  if (c->batch < 0 || c->kv_heads < 1 || c->page_size < 1 || c->max_pages < 0 || c->num_pages < 0) return B200TBE_ERR_BAD_ARG;
  if (c->batch > 0 && c->lengths == nullptr) return B200TBE_ERR_BAD_ARG;
  if (c->batch > 0 && c->max_pages > 0 && c->page_table == nullptr) return B200TBE_ERR_BAD_ARG;
  if (c->num_pages > 0 && (c->k_cache == nullptr || c->v_cache == nullptr)) return B200TBE_ERR_BAD_ARG;
  return B200TBE_OK;
}

CacheDev cache_dev(const b200tbe_paged_cache* c) {
  CacheDev d{};
  d.k = static_cast<char*>(c->k_cache), d.v = static_cast<char*>(c->v_cache);
  d.page_table = c->page_table, d.lengths = c->lengths;
  d.k_page = c->k_page_stride, d.k_slot = c->k_slot_stride, d.k_head = c->k_head_stride;
  d.v_page = c->v_page_stride, d.v_slot = c->v_slot_stride, d.v_head = c->v_head_stride;
  d.table_stride = c->page_table_stride, d.num_pages = c->num_pages, d.max_pages = c->max_pages;
  d.page_size = c->page_size, d.batch = c->batch, d.kv_heads = c->kv_heads, d.D = c->head_dim;
  d.length_bytes = c->length_bytes, d.status = c->status;
  d.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (d.page_size == 1 << i) d.page_shift = i;
  return d;
}

template <typename VecT>
int launch_append(const AppendDev& p, cudaStream_t stream) {
  const int64_t warps = (p.total + p.rows_per_warp - 1) / p.rows_per_warp, blocks = (warps + 7) / 8;
  if (blocks > 0x7fffffff) return B200TBE_ERR_TOO_LARGE;
  append_kernel<VecT><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  return launch_status();
}

// Launched while the answers' kernel still runs, whose results it waits for: its launch costs no time of its own.
template <typename T>
int join(const AnswerDev& p, int ctas, cudaStream_t stream) {
  if (ctas < 2) return B200TBE_OK;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas - 1, p.per < p.group ? p.per : p.group);
  config.blockDim = dim3(kAnswerThreads);
  config.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, join_kernel<T>, p) == cudaSuccess ? B200TBE_OK : B200TBE_ERR_LAUNCH;
}

// 16-byte reads of everything, and a head dimension that the registers hold
bool answer_in_pieces(const AnswerDev& p, int elem_bytes) {
  uint64_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.c.k) | reinterpret_cast<uintptr_t>(p.c.v);
  for (int64_t x : {static_cast<int64_t>(p.c.D), p.q_row, p.q_head, p.c.k_page, p.c.k_slot, p.c.k_head, p.c.v_page, p.c.v_slot,
                    p.c.v_head})
    bits |= static_cast<uint64_t>(x * elem_bytes);
  return bits % 16 == 0 && p.c.D <= 128;
}

template <int kDP, int kH>
int launch_answer_fma(AnswerDev p, int64_t most, cudaStream_t stream) {
  using R = RingF<kDP, kH>;
  if (!allow_shared_memory<answer_fma_kernel<kDP, kH>>(R::kBytes)) return B200TBE_ERR_LAUNCH;
  p.per = kH;
  p.chunks = (p.group + p.per - 1) / p.per;
  p.units = p.c.kv_heads * p.chunks;
  if (static_cast<int64_t>(p.units) * p.c.batch > 0x7fffffff) return B200TBE_ERR_TOO_LARGE;
  const int64_t tiles = static_cast<int64_t>(p.units) * p.c.batch * (most + kUnitCost);
  const int ctas = static_cast<int>(tiles < kNumSMs * R::kCtas ? tiles : kNumSMs * R::kCtas);
  answer_fma_kernel<kDP, kH><<<ctas, kAnswerThreads, R::kBytes, stream>>>(p);
  const int st = launch_status();
  return st != B200TBE_OK ? st : join<float>(p, ctas, stream);
}

template <typename T, bool kBf16, int kDP>
int launch_answer_mma(const AnswerDev& p, int64_t tiles, cudaStream_t stream) {
  using R = Ring<kDP>;
  if (!allow_shared_memory<answer_mma_kernel<kBf16, kDP>>(R::kBytes)) return B200TBE_ERR_LAUNCH;
  const int ctas = static_cast<int>(tiles < kNumSMs * R::kCtas ? tiles : kNumSMs * R::kCtas);
  answer_mma_kernel<kBf16, kDP><<<ctas, kAnswerThreads, R::kBytes, stream>>>(p);
  const int st = launch_status();
  return st != B200TBE_OK ? st : join<T>(p, ctas, stream);
}

template <typename T>
int launch_answer(const AnswerDev& p, int ctas, cudaStream_t stream) {
  const int bytes = (kHeads * p.c.D + kTile * (p.c.D + 1)) * 4;
  constexpr int kMost = (kHeads * 256 + kTile * 257) * 4;   // at the largest head dimension
  if (p.c.D <= kAnswerThreads) {
    if (!allow_shared_memory<answer_simt_kernel<T, 1>>(kMost)) return B200TBE_ERR_LAUNCH;
    answer_simt_kernel<T, 1><<<ctas, kAnswerThreads, bytes, stream>>>(p);
  } else {
    if (!allow_shared_memory<answer_simt_kernel<T, 2>>(kMost)) return B200TBE_ERR_LAUNCH;
    answer_simt_kernel<T, 2><<<ctas, kAnswerThreads, bytes, stream>>>(p);
  }
  const int st = launch_status();
  return st != B200TBE_OK ? st : join<T>(p, ctas, stream);
}

}  // namespace
}  // namespace b200tbe

using namespace b200tbe;

extern "C" int b200tbe_paged_cache_append(const b200tbe_paged_cache* cache, const void* k, const void* v, int64_t k_stride,
                                          int64_t k_head_stride, int64_t v_stride, int64_t v_head_stride,
                                          const void* offsets, int32_t offset_bytes, int64_t total,
                                          b200tbe_stream_t stream_) {
  const int st = check_cache(cache);
  if (st != B200TBE_OK) return st;
  if (offset_bytes != 4 && offset_bytes != 8) return B200TBE_ERR_UNSUPPORTED;
  if (total < 0) return B200TBE_ERR_BAD_ARG;
  if (total == 0 || cache->batch == 0) return B200TBE_OK;
  if (k == nullptr || v == nullptr || offsets == nullptr) return B200TBE_ERR_BAD_ARG;
  AppendDev p{};
  p.c = cache_dev(cache);
  p.k = static_cast<const char*>(k), p.v = static_cast<const char*>(v);
  p.k_row = k_stride, p.k_head = k_head_stride, p.v_row = v_stride, p.v_head = v_head_stride;
  p.offsets = offsets, p.offset_bytes = offset_bytes, p.total = total;
  p.elem_bytes = elem_bytes_of(cache->dtype);
  if (static_cast<int64_t>(cache->head_dim) * cache->kv_heads * p.elem_bytes > (1 << 24)) return B200TBE_ERR_TOO_LARGE;
  // rows are shared out so that a small batch still uses every SM
  p.rows_per_warp = static_cast<int32_t>(total / (kNumSMs * 64) < 1 ? 1 : (total / (kNumSMs * 64) > 8 ? 8 : total / (kNumSMs * 64)));
  uint64_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(p.c.k) |
                  reinterpret_cast<uintptr_t>(p.c.v);
  for (int64_t s : {static_cast<int64_t>(p.c.D), p.k_row, p.k_head, p.v_row, p.v_head, p.c.k_page, p.c.k_slot, p.c.k_head,
                    p.c.v_page, p.c.v_slot, p.c.v_head})
    bits |= static_cast<uint64_t>(s * p.elem_bytes);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (bits % 16 == 0) return launch_append<uint4>(p, stream);
  if (bits % 4 == 0) return launch_append<uint32_t>(p, stream);
  return launch_append<uint16_t>(p, stream);
}

extern "C" size_t b200tbe_paged_attention_scratch_bytes(int32_t head_dim) {
  if (head_dim < 1) return 0;
  return kAnswerCtas * (sizeof(Start) + 2 * kHeads * (2 + static_cast<size_t>(head_dim)) * sizeof(float));
}

extern "C" int b200tbe_paged_attention(const b200tbe_paged_cache* cache, const void* q, void* out, int64_t q_stride,
                                       int64_t q_head_stride, int64_t out_stride, int64_t out_head_stride, int32_t heads,
                                       float scale, void* scratch, size_t scratch_bytes, b200tbe_stream_t stream_) {
  const int st = check_cache(cache);
  if (st != B200TBE_OK) return st;
  if (heads < 1 || heads % cache->kv_heads != 0) return B200TBE_ERR_BAD_ARG;
  if (cache->batch == 0) return B200TBE_OK;
  if (q == nullptr || out == nullptr) return B200TBE_ERR_BAD_ARG;
  if (scratch == nullptr || scratch_bytes < b200tbe_paged_attention_scratch_bytes(cache->head_dim) || !aligned_to(scratch, 16))
    return B200TBE_ERR_SCRATCH;
  AnswerDev p{};
  p.c = cache_dev(cache);
  // copies of nothing still name an address
  if (cache->num_pages == 0) p.c.k = p.c.v = static_cast<char*>(const_cast<void*>(q));
  p.q = q, p.out = out;
  p.q_row = q_stride, p.q_head = q_head_stride, p.o_row = out_stride, p.o_head = out_head_stride;
  p.heads = heads, p.group = heads / cache->kv_heads, p.per = kHeads, p.chunks = (p.group + kHeads - 1) / kHeads;
  p.units = cache->kv_heads * p.chunks;
  if (static_cast<int64_t>(p.units) * cache->batch > 0x7fffffff) return B200TBE_ERR_TOO_LARGE;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.starts = static_cast<Start*>(scratch);
  p.stats = reinterpret_cast<float*>(p.starts + kAnswerCtas);
  p.sums = p.stats + 2 * kAnswerCtas * kHeads * 2;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  // as many CTAs as the cache could give tiles to
  int64_t most = (static_cast<int64_t>(cache->max_pages) * cache->page_size + kTile - 1) / kTile;
  if (most < 1) most = 1;
  const int64_t tiles = static_cast<int64_t>(p.units) * cache->batch * (most + kUnitCost);
  if (cache->dtype == B200TBE_FP32 && answer_in_pieces(p, 4))
    return p.c.D <= 64 ? (p.group <= 2 ? launch_answer_fma<64, 2>(p, most, stream) : launch_answer_fma<64, 8>(p, most, stream))
                       : (p.group <= 2 ? launch_answer_fma<128, 2>(p, most, stream) : launch_answer_fma<128, 4>(p, most, stream));
  if (cache->dtype != B200TBE_FP32 && answer_in_pieces(p, 2)) {
    if (cache->dtype == B200TBE_FP16)
      return p.c.D <= 64 ? launch_answer_mma<__half, false, 64>(p, tiles, stream) : launch_answer_mma<__half, false, 128>(p, tiles, stream);
    return p.c.D <= 64 ? launch_answer_mma<__nv_bfloat16, true, 64>(p, tiles, stream)
                       : launch_answer_mma<__nv_bfloat16, true, 128>(p, tiles, stream);
  }
  const int ctas = static_cast<int>(tiles < kAnswerCtas ? tiles : kAnswerCtas);
  if (cache->dtype == B200TBE_FP32) return launch_answer<float>(p, ctas, stream);
  if (cache->dtype == B200TBE_FP16) return launch_answer<__half>(p, ctas, stream);
  return launch_answer<__nv_bfloat16>(p, ctas, stream);
}
