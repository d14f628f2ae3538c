// The sm_100a instructions that the tensor-core attention kernels are made of: barriers, tensor copies, tensor
// memory and its matrix instruction. Every wait for a barrier is bounded. tmem_alloc() is not: it waits until CTAs on its SM,
// of any kernel, have freed columns. It ends because a CTA allocates once, before it has anything that another could wait for,
// and comes to tmem_free() whether its waits succeed or give up.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace b200tbe {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Clock cycles after which a wait gives up (about two seconds): nothing here waits on another CTA, so only a
// fault in the kernel itself could take that long.
constexpr long long kWaitCycles = 4ll << 30;

// Waits for the phase of this parity. false: this wait, or another one of the CTA, gave up.
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try(bar, parity)) return true;
  const long long begin = clock64();
  while (!mbar_try(bar, parity)) {
    if (*dead) return false;
    if (clock64() - begin > kWaitCycles && !mbar_try(bar, parity)) {   // looked at once more: the clock ran on while
      *dead = 1;                                                         // another process had the GPU
      return false;
    }
  }
  return true;
}

// The same for a whole warp, which goes on together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  return __all_sync(kFullMask, mbar_wait(bar, parity, dead));
}

// At a kernel's end, by the whole CTA, between two barriers: if a wait gave up, report it, and let what is in flight land before
// its memory is given back.
__device__ __forceinline__ void report(const int* dead, int32_t* status) {
  if (*dead) {
    if (threadIdx.x == 0 && status != nullptr) atomicOr(status, B200TBE_DEV_WAIT_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
}

// Registers of a warpgroup from here on; the block's shares must not exceed what it was launched with.
template <int kRegs>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

__device__ __forceinline__ void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// shared-memory writes of this thread, before asynchronous units read them
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}


// Tensor memory: 128 lanes x 512 columns of 32 bits a SM. A whole warp allocates and frees.
__device__ __forceinline__ void tmem_alloc(uint32_t* where, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}

__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}

__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// A shared-memory operand in rows of 128 bytes, swizzled in groups of eight rows (1024 bytes, 1024-aligned):
// what a tensor copy with a 128-byte swizzle writes.
//   along k ("K-major"): a row is 64 elements of k; 32 bytes further in start address are the next 16.
//   along m or n ("MN-major"): a row is 64 elements of m or n for one k; `lead` bytes to the next 64 of them,
//   2048 bytes further are the next 16 of k.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// One thread of a warp that is together here; the same one each time. (The compiler keeps what follows in uniform
// registers, where the matrix instruction wants its operands: with a lane number instead, moving them there took
// longer than the instructions themselves.)
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}

// fp32 accumulators, both operands bf16 or both fp16
__device__ __forceinline__ constexpr uint32_t mma_desc(bool bf16, int m, int n, bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn_major ? 1u : 0u) << 15) |
         ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// d (+)= a b^T for 16 elements of k; issued by one thread. a in shared memory or in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
      "l"(b), "r"(desc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
      "l"(b), "r"(desc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
// d[128][n] (+)= a b^T over up to kMost x 16 elements of k, both operands along k: rows of 64 elements in tiles of
// `rows` x 128 bytes. Unrolled, so that a step costs two additions beside the instruction.
template <int kMost, int kRowsOfTile>
__device__ __forceinline__ void mma_along_k(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, int steps) {
  const uint64_t a0 = smem_desc(a, 16), b0 = smem_desc(b, 16);
#pragma unroll
  for (int t = 0; t < kMost; ++t) {
    const uint64_t off = ((t / 4) * kRowsOfTile * 128 + (t % 4) * 32) >> 4;
    if (t < steps) mma_ss(d, a0 + off, b0 + off, desc, t > 0);
  }
}

// The same with a in tensor memory, two elements a column.
template <int kMost, int kRowsOfTile>
__device__ __forceinline__ void mma_along_k_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, int steps) {
  const uint64_t b0 = smem_desc(b, 16);
#pragma unroll
  for (int t = 0; t < kMost; ++t)
    if (t < steps) mma_ts(d, a + t * 8, b0 + (((t / 4) * kRowsOfTile * 128 + (t % 4) * 32) >> 4), desc, t > 0);
}

// d[128][n] (+)= w x over up to 128 rows of x, 16 a step: w in tensor memory, two 16-bit elements a column, kSkip columns
// left out after every kRun steps' worth; x in tiles of 128 rows, n along the row.
template <int kSkip = 0, int kRun = 8>
__device__ __forceinline__ void mma_over_rows(uint32_t d, uint32_t w, uint32_t x, uint32_t desc, int steps, bool add) {
  const uint64_t x0 = smem_desc(x, 128 * 128);
#pragma unroll
  for (int t = 0; t < 8; ++t)
    if (t < steps) mma_ts(d, w + t * 8 + t / kRun * kSkip, x0 + t * (2048 >> 4), desc, t > 0 || add);
}

// Arrives once all matrix instructions that this thread has issued are done. Some thread has to wait for it: an
// arrival nobody waits for could come after the barrier's memory has been given to something else.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t as_pair(const uint32_t* x) {
  return pair(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Binary places by which weights of at most 1 are lifted before they are rounded to 16 bits. fp16 holds what is below 2^-14
// with ever fewer bits, and many small weights may be what a result is made of; its upper half, unused otherwise, takes them down to
// 2^-28 (and leaves a factor of four for a score's rounding). bf16 has fp32's range.
template <bool kBf16>
constexpr float kLift = kBf16 ? 0.f : 14.f;

// Of a backward pass: dP - delta, in fp16 in a unit, which minus_delta has already.
template <bool kBf16>
__device__ __forceinline__ uint64_t less_delta(uint64_t dp, uint64_t unit, uint64_t minus_delta) {
  if constexpr (kBf16)
    return add2(dp, minus_delta);
  else
    return fma2(dp, unit, minus_delta);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The numbers of the CTA's items, handed from the warp that copies to the others, a few ahead; -1 ends them.
struct Queue {
  static constexpr int kRoom = 4;
  uint64_t full[kRoom], empty[kRoom];
  int64_t index[kRoom];
};
__device__ __forceinline__ void queue_init(Queue* queue, int takers) {
  for (int i = 0; i < Queue::kRoom; ++i) {
    mbar_init(&queue->full[i], 1);
    mbar_init(&queue->empty[i], takers);
  }
}
__device__ __forceinline__ bool put_item(Queue* queue, int turn, int64_t index, volatile int* dead) {
  const int at = turn % Queue::kRoom;
  if (turn >= Queue::kRoom && !warp_wait(&queue->empty[at], (turn / Queue::kRoom - 1) & 1, dead)) return false;
  if (threadIdx.x % 32 == 0) {
    queue->index[at] = index;
    mbar_arrive(&queue->full[at]);
  }
  __syncwarp();
  return true;
}
// the turn's item, -1 after the last or when a wait gave up
__device__ __forceinline__ int64_t take_item(Queue* queue, int turn, volatile int* dead) {
  const int at = turn % Queue::kRoom;
  if (!warp_wait(&queue->full[at], (turn / Queue::kRoom) & 1, dead)) return -1;
  const int64_t index = queue->index[at];
  __syncwarp();
  if (threadIdx.x % 32 == 0) mbar_arrive(&queue->empty[at]);
  return index;
}

// 32 columns of a warp's 32 accumulator rows (a row a lane), times f, rounded, to memory: columns [col, col + 32) of the
// rows out, out + stride, ...; `rows` of them, columns below D. Through 2 KB of shared memory of the warp's own, so
// that an instruction writes eight rows' 64 bytes; 16 bytes a lane in 32 rows took most of a short sequence's time.
template <bool kBf16>
__device__ __forceinline__ void store_columns(uint8_t* stage, const uint32_t (&o)[32], float f, bool zero, uint16_t* out,
                                              int64_t stride, int rows, int col, int D) {
  const int lane = threadIdx.x % 32;
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    uint32_t y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      y[u] = zero ? 0u : pack2<kBf16>(__uint_as_float(o[e + 2 * u]) * f, __uint_as_float(o[e + 2 * u + 1]) * f);
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((e / 8) ^ (lane / 2 % 4)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
  }
  __syncwarp();
  const int first = lane / 4, c = lane % 4;
  out += first * stride + col + c * 8;
  rows = col + c * 8 < D ? rows - first : 0;
  const uint8_t* from = stage + first * 64 + (c ^ (first / 2 % 4)) * 16;   // the same piece in every eighth row
#pragma unroll
  for (int i = 0; i < 4; ++i, out += 8 * stride)
    if (i * 8 < rows) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(from + i * 512);
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (kBf16)
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  else
    return half2_bits_to_float2(x);
}

// A tensor map over [rows][heads][D] of 16-bit elements, in boxes of 64 columns of one head x `box_rows` rows.
// Columns past D and rows past the end read as zero. false: the driver refuses it.
bool rows_map(CUtensorMap* map, bool bf16, const void* base, int64_t rows, int heads, int D, int64_t row_stride,
              int64_t head_stride, int box_rows);
// Strides and addresses that a tensor map can take.
bool mappable(const void* base, int64_t rows, int heads, int64_t row_stride, int64_t head_stride);

}  // namespace b200tbe
