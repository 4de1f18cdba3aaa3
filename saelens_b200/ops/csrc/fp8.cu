// Matrix product with a frozen weight in 8-bit floating point (e4m3), one scale per block of 128:
//     y[m, f] = sum over blocks b of  xs[m, b] ws[f / 128, b]  sum over r in b of  xq[m, r] wq[f, r]   (+ bias[f])
// x is quantised on the way in, one scale for a row's 128 consecutive values:
//     xs = max(|x|) / 448,   xq = e4m3(448 x / max(|x|))
// (448 is the largest e4m3 value; the quotient is formed as (7/16 x) / max * 1024, whose numerator
// is exact for 16-bit x and cannot overflow, so it is rounded once and values on the border of two
// e4m3 neighbours fall the same way in any arithmetic; the maximum is at least 448 * 2^-126, so that
// a scale is a normal number; a block with an infinity or NaN makes its whole row NaN).
// The weight has a scale for each 128 x 128 block.  The gradient of x is the same product with the
// roles of the weight's sides changed, dx = Q(dy) W: the weight is then read as an MN-major operand,
// in place.
//
// The tensor cores sum one block of 128 exactly scaled alike, in fp32; the scales differ from block
// to block, so each block's accumulator is read out of tensor memory, scaled and added to fp32 sums
// in registers while the next block is multiplied into a second accumulator.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>
#include <torch/types.h>

#include <algorithm>
#include <atomic>
#include <tuple>
#include <type_traits>

#include "block_ops.h"
#include "check.h"
#include "common.cuh"
#include "tmap.h"
#include "vec.cuh"

namespace sb {
namespace fp8 {

constexpr int BLK = 128;               // values a scale covers, along the reduction and (weights) the features
constexpr float MAXV = 448.f;
constexpr uint32_t LEAST_BITS = 0x04e00000u;  // 448 * 2^-126

// ---------------------------------------------------------------------------------------------
// quantisation
// ---------------------------------------------------------------------------------------------
// Bit patterns of absolute values order like the values, with NaN above infinity: a NaN stays.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// e4m3 of 448 v / most, the quotient rounded once.  t is the product with a rounded reciprocal; its
// exact residual, which one fused multiply-add gives, times that reciprocal makes it the correctly
// rounded quotient (Markstein 1990).  A division for every value made the quantisation issue-bound (41
// us for 8192 x 4096 values, whose bytes take 15), and one only for values near a border of e4m3 little
// less: of 16-bit values many lie on one.  Scaled by 1024 so that the reciprocal stays a normal
// number; an infinite maximum gives NaN.
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float most, float by) {  // by = 1024 / most
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float num = v[j] * 0.4375f, q = num * by;
    t[j] = __fmaf_rn(__fmaf_rn(q * -0.0009765625f, most, num), by, q);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(t[4 * h], t[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(t[4 * h + 2], t[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// 8 values from column c of a row; columns from K on are 0.  ALIGNED: rows start on 16 bytes and K is
// a multiple of 8.
template <class T, bool ALIGNED>
__device__ __forceinline__ vec::Pack<T, 8> load_pack(const T* row, int64_t c, int64_t K) {
  vec::Pack<T, 8> p;
  p.zero();
  if (ALIGNED) {
    if (c < K) p.load(row + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < K) reinterpret_cast<T*>(p.r)[j] = row[c + j];
  }
  return p;
}
template <class T, bool ALIGNED>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t K, float (&v)[8]) {
  load_pack<T, ALIGNED>(row, c, K).unpack(v);
}

// A key of the largest absolute value of 8: its bits in T, in which two 16-bit values compare at once.
template <class T>
__device__ __forceinline__ uint32_t most_key(const vec::Pack<T, 8>& p) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p.r);
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int j = 1; j < 4; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
    return max(m & 0xffffu, m >> 16);
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(p.get(j)));
    return m;
  }
}
// The value of a key, LEAST at least.
template <class T>
__device__ __forceinline__ float key_value(uint32_t key) {
  uint32_t bits = key;
  if constexpr (std::is_same_v<T, __half>) bits = __float_as_uint(__half2float(__ushort_as_half(uint16_t(key))));
  else if constexpr (sizeof(T) == 2) bits = key << 16;
  return __uint_as_float(max(bits, LEAST_BITS));
}

// The largest absolute value (as bits, at least LEAST_BITS) of the 16 lanes of a half-warp.
__device__ __forceinline__ float half_warp_most(const float (&v)[8]) {
  uint32_t m = LEAST_BITS;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return __uint_as_float(m);
}

// Rows: a half-warp quantises a row's 128 values, 8 a lane; 16 rows a block, PER blocks of 128 a
// half-warp (all loads issued before the first maximum).  2 bytes are read and 1 written a value, but issue
// slots bind before memory does: 8192 x 4096 values in 26 us at 66% of the issue slots (15 us of bytes at
// the copy rate), 2048 x 14336 in 23 (13).
template <class T, bool ALIGNED, int PER>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t M, int64_t K,
                                                            uint8_t* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale, int64_t lds) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 15;
  const int64_t row = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int64_t kb0 = int64_t(blockIdx.y) * PER, KB = (K + BLK - 1) / BLK;
  const T* from = x + (row < M ? row : 0) * ldx;
  vec::Pack<T, 8> p[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) p[i] = load_pack<T, ALIGNED>(from, (kb0 + i) * BLK + lane * 8, row < M ? K : 0);
  uint32_t key[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    key[i] = most_key<T>(p[i]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) key[i] = max(key[i], __shfl_xor_sync(0xffffffffu, key[i], o));
    if ((lane & (PER - 1)) == i) mine = key[i];
  }
  // lane i divides for block i (lanes from PER on again), and the others take the reciprocal from it
  const float most = key_value<T>(mine), by = 1024.f / most;
  if (lane < PER && row < M && kb0 + lane < KB) scale[(kb0 + lane) * lds + row] = most / MAXV;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t c = (kb0 + i) * BLK + lane * 8;
    const float r = __shfl_sync(0xffffffffu, by, (threadIdx.x & 16) + i);
    float v[8];
    p[i].unpack(v);
    if (row < M && c < ldq) *reinterpret_cast<uint2*>(q + row * ldq + c) = quantize8(v, key_value<T>(key[i]), r);
  }
}

// Weights: a block of 256 threads quantises one 128 x 128 block, 64 values a thread in registers.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T* __restrict__ x, int64_t ldx, int64_t N, int64_t K,
                                                              uint8_t* __restrict__ q, int64_t ldq,
                                                              float* __restrict__ scale) {
  __shared__ uint32_t red[8];
  const int64_t kb = blockIdx.x, nb = blockIdx.y;
  const int64_t c = kb * BLK + (threadIdx.x & 15) * 8;
  float v[8][8];
  uint32_t m = LEAST_BITS;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = nb * BLK + i * 16 + (threadIdx.x >> 4);
    if (row < N) {
      load8<T, ALIGNED>(x + row * ldx, c, K, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const float most = __uint_as_float(m), by = 1024.f / most;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = nb * BLK + i * 16 + (threadIdx.x >> 4);
    if (row < N && c < ldq) *reinterpret_cast<uint2*>(q + row * ldq + c) = quantize8(v[i], most, by);
  }
  if (threadIdx.x == 0) scale[nb * gridDim.x + kb] = most / MAXV;
}

// ---------------------------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------------------------
// Instruction descriptor of kind::f8f6f4: e4m3 operands, fp32 accumulator; the bits mark MN-major ones.
__host__ __device__ constexpr uint32_t make_idesc(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t(N >> 3) << 17) |
         (uint32_t(M >> 4) << 24);
}
__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Over a pair of blocks, issued by its first one.
__device__ __forceinline__ void umma_e4m3_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Arrival on a barrier of either block of a pair, ordered within this block.  Across the pair it hands over
// the accumulator, which has been read by then (tcgen05.wait::ld), and nothing else: row scales have a
// barrier of their block's own.  A cluster-wide release waits for every access under way and took twice
// the time of the products.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// mbar_wait_bounded that reads the clock only after 64 tries: a wait is on the way of every block of
// 128 here, and most end within the first.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, int code) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_bounded(bar, parity, abort, status, code);
}

__device__ __forceinline__ void st_release_cta(int* p, int v) {
  asm volatile("st.release.cta.shared.b32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
// Wait until the count at p reaches `least`; limits as for a barrier.
__device__ __forceinline__ bool wait_count(int* p, int least, volatile int* abort, int* status, int code) {
  unsigned long long t0 = 0;
  for (int i = 0;; ++i) {
    int v;
    asm volatile("ld.acquire.cta.shared.b32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
    if (v >= least) return true;
    if ((i & 63) == 63) {
      if (*abort) return false;
      const unsigned long long now = globaltimer_ns();
      if (!t0) t0 = now;
      if (now - t0 > kWaitTimeoutNs) {
        *abort = 1;
        if (status) atomicCAS(status, 0, code);
        return false;
      }
    }
  }
}

struct Prod {
  const void* x;        // fused quantisation: the rows themselves
  int64_t ldx;
  const float* ws;      // scale of (feature block, reduction block) at fb * ws_f + rb * ws_r
  int64_t ws_f, ws_r;
  const float* bias;    // [features] or nullptr
  void* out;            // [M, ldo]
  int64_t ldo;
  int M, F, R;          // rows, features, length of the reduction
  int splits;           // parts of the reduction (the cluster's blocks)
  int* status;
};

// ---- few rows -------------------------------------------------------------------------------
// Up to NT rows.  The weight is the tensor cores' 128-row operand and the rows of x the narrow one, so
// that no part of the tile is idle weight; the time is the weight's bytes.  A block owns 128
// features and a part of the reduction; the blocks of a cluster hold the parts of the same features.
// Column c of the sums belongs to block c % splits: every block writes its part of it there, over
// distributed shared memory, and after one cluster barrier the owner adds the parts in block order.
// (Reading the parts instead took two barriers and a remote round trip, 3.3 us of 13.)  With launches
// queued one row 4096 -> 6144 takes 10.4 us and 24 rows 14336 -> 4096 18.6 (25 and 59 MB of weight: 3.9 and
// 9.0 us at the copy rate).  The 24 rows' quantisation hides beside the product, which takes 18.2 by itself,
// 3.2 TB/s with 1.7 of its blocks an SM side by side.
//   warp 0      weight tiles by TMA (and x tiles and scales, unless they are quantised here)
//   warp 1      tcgen05.mma, 4 a block of 128
//   warps 2..5  scaled sums in registers: a feature a thread, NT columns
//   warps 6..9  FUSED: quantise x into the stage's tile, a half-warp for a row's 128 values
template <int NT>
struct Few {
  static constexpr int W_BYTES = BLK * BLK, X_BYTES = NT * BLK, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = NT <= 16 ? 5 : NT <= 32 ? 4 : 3;
  // accumulators: the products run so many blocks ahead of the sums
  static constexpr int ACC = NT <= 16 ? 8 : 4;
  static constexpr int RING = STAGES + ACC;  // scales outlive their tile by the accumulators
  static constexpr int SLOT = NT < 32 ? 32 : NT;  // floats of a slot: a TMA copy starts on 128 bytes of shared memory
  static constexpr int TMEM = ACC * NT;
  // parts of the columns that a block owns: [columns][splits][128 features], NT + splits - 1 of 512 bytes at most
  static constexpr int SMEM = STAGES * STAGE + RING * SLOT * 4 + (NT + 8) * 512 + 1024 + 512;
};

template <int NT, bool FUSED, bool ALIGNED, bool W_MN, class TX, class TO>
__global__ void __launch_bounds__(FUSED ? 320 : 192, 2)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                    const __grid_constant__ CUtensorMap tmS, const __grid_constant__ Prod a) {
  using C = Few<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + C::STAGES * C::W_BYTES;
  float* sS = reinterpret_cast<float*>(sX + C::STAGES * C::X_BYTES);  // [RING][SLOT]
  float* parts = sS + C::RING * C::SLOT;
  uint64_t* full = reinterpret_cast<uint64_t*>(parts + (NT + 8) * 128);
  uint64_t* empty = full + C::STAGES;
  uint64_t* sfull = empty + C::STAGES;
  uint64_t* tfull = sfull + C::RING;
  uint64_t* tempty = tfull + C::ACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + C::ACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* released = reinterpret_cast<int*>(tmem_slot + 2);  // FUSED: blocks below this have a free stage

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % a.splits, fb = blockIdx.x / a.splits;
  const int RB = (a.R + BLK - 1) / BLK;
  const int rb0 = int(int64_t(split) * RB / a.splits), n = int(int64_t(split + 1) * RB / a.splits) - rb0;

  auto load_w = [&](int j) {
    const int s = j % C::STAGES, r = (rb0 + j) * BLK;
    mbar_arrive_expect_tx(&full[s], FUSED ? C::W_BYTES : C::STAGE + NT * 4);
    if (W_MN) tma_load_2d(sW + s * C::W_BYTES, &tmW, &full[s], fb * BLK, r);
    else tma_load_2d(sW + s * C::W_BYTES, &tmW, &full[s], r, fb * BLK);
  };
  // the weight depends on no kernel before: its first tiles are on their way before anything else
  const int first = min(n, C::STAGES);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], FUSED ? 1 + a.M : 1);
      mbar_init(&empty[s], 1);
    }
    if (FUSED)
      for (int s = 0; s < C::RING; ++s) mbar_init(&sfull[s], a.M);
    for (int s = 0; s < C::ACC; ++s) {
      mbar_init(&tfull[s], 1);
      mbar_init(&tempty[s], 4);
    }
    *abort_flag = 0;
    *released = first;
    fence_mbar_init();
    for (int j = 0; j < first; ++j) load_w(j);
    if (!FUSED) tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM);
    tmem_relinquish();
  }
  // items of the quantising half-warps: item i is 128 values of row i % M of reduction block i / M
  const int hw = (threadIdx.x - 192) >> 4, l = threadIdx.x & 15;
  float v[8];
  auto load_item = [&](int i) {
    const int j = i < n * a.M ? i / a.M : 0, m = i < n * a.M ? i - j * a.M : 0;
    load8<TX, ALIGNED>(static_cast<const TX*>(a.x) + m * a.ldx, int64_t(rb0 + j) * BLK + l * 8, i < n * a.M ? a.R : 0, v);
  };
  if (FUSED && warp >= 6) load_item(hw);
  // the cluster's blocks have all started once this barrier is through, which is asked for only at the end
  __syncwarp();
  if (a.splits > 1) cluster_arrive_relaxed();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float acc[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) acc[c] = 0.f;
  const int q = warp & 3;
  const int f = fb * BLK + q * 32 + lane;  // this thread's feature (warps 2..5)

  if (warp == 0) {
    if (elect_one()) {
      auto load_x = [&](int j) {
        const int s = j % C::STAGES;
        tma_load_2d(sX + s * C::X_BYTES, &tmX, &full[s], (rb0 + j) * BLK, 0);
        tma_load_2d(sS + (j % C::RING) * C::SLOT, &tmS, &full[s], 0, rb0 + j);
      };
      bool ok = true;
      if (!FUSED) {
        grid_dependency_wait();
        for (int i = 0; i < first; ++i) load_x(i);
      }
      int j = first;
      for (; j < n; ++j) {
        const int s = j % C::STAGES;
        if (!wait_bar(&empty[s], ((j / C::STAGES) & 1) ^ 1, abort_flag, a.status, kTimeoutTmaProducer)) {
          ok = false;
          break;
        }
        if (FUSED) st_release_cta(released, j + 1);
        load_w(j);
        if (!FUSED) load_x(j);
      }
      if (!ok) {  // the copies in flight land before the block leaves
        for (int i = max(0, j - C::STAGES); i < j; ++i) {
          volatile int dummy = 0;
          mbar_wait_bounded(&full[i % C::STAGES], (i / C::STAGES) & 1, &dummy, nullptr, 0);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc(128, NT, W_MN, false);
      for (int j = 0; j < n; ++j) {
        const int s = j % C::STAGES, t = j % C::ACC;
        if (!wait_bar(&tempty[t], ((j / C::ACC) & 1) ^ 1, abort_flag, a.status, kTimeoutMmaTmemEmpty)) break;
        if (!wait_bar(&full[s], (j / C::STAGES) & 1, abort_flag, a.status, kTimeoutMmaFull)) break;
        tc_fence_after();
        const uint32_t w = smem_u32(sW + s * C::W_BYTES), x = smem_u32(sX + s * C::X_BYTES);
#pragma unroll
        for (int k = 0; k < BLK / 32; ++k)
          umma_e4m3(tmem + t * NT, W_MN ? make_sdesc_sw128_mnmajor(w + k * 4096, 16384) : make_sdesc_sw128_kmajor(w + k * 32),
                    make_sdesc_sw128_kmajor(x + k * 32), idesc, k > 0);
        umma_commit(&empty[s]);
        umma_commit(&tfull[t]);
      }
    }
    __syncwarp();
  } else if (warp < 6) {
    float wv = 0.f;  // lane l: the weight's scale of block (j & ~31) + l
    for (int j = 0; j < n; ++j) {
      if ((j & 31) == 0 && j + lane < n) wv = a.ws[fb * a.ws_f + (rb0 + j + lane) * a.ws_r];
      const float ws = __shfl_sync(0xffffffffu, wv, j & 31);
      const int t = j % C::ACC, g = j % C::RING;
      bool ok = true;
      // the products waited for the scales that came with their tile; those written here have their own barrier
      if (FUSED) ok = wait_bar(&sfull[g], (j / C::RING) & 1, abort_flag, a.status, kTimeoutEpilogue);
      ok = ok && wait_bar(&tfull[t], (j / C::ACC) & 1, abort_flag, a.status, kTimeoutEpilogue);
      if (!__all_sync(0xffffffffu, ok)) break;  // the warp leaves as one
      tc_fence_after();
      uint32_t r[NT];
#pragma unroll
      for (int c = 0; c < NT; c += 16) tmem_ld_x16(tmem + (uint32_t(q * 32) << 16) + t * NT + c, r + c);
      tmem_ld_wait();
      const float4* xs = reinterpret_cast<const float4*>(sS + g * C::SLOT);
#pragma unroll
      for (int c = 0; c < NT; c += 4) {
        const float4 v = xs[c / 4];
        acc[c] += __uint_as_float(r[c]) * (v.x * ws);
        acc[c + 1] += __uint_as_float(r[c + 1]) * (v.y * ws);
        acc[c + 2] += __uint_as_float(r[c + 2]) * (v.z * ws);
        acc[c + 3] += __uint_as_float(r[c + 3]) * (v.w * ws);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[t]);
    }
    __syncwarp();
  } else if (FUSED) {
    const uint32_t mask = 0xffffu << (lane & 16);
    const int items = n * a.M;
    // every half-warp takes part in the warp's shuffles, with or without an item of its own
    for (int i0 = hw & ~1; i0 < items; i0 += 8) {
      const int i = i0 + (hw & 1);
      const bool have = i < items;
      const int j = have ? i / a.M : 0, m = have ? i - j * a.M : 0;
      const float most = half_warp_most(v);
      const uint2 w = quantize8(v, most, 1024.f / most);
      load_item(i + 8);  // the next one's values arrive meanwhile
      const int s = j % C::STAGES, g = j % C::RING;
      bool ok = true;
      // A half-warp skips blocks, so a stage's barrier may be several phases from the one it would wait
      // for and its parity says nothing; the loading thread has waited for each phase and counts them.
      if (have) ok = wait_count(released, j + 1, abort_flag, a.status, kTimeoutTmaProducer);
      if (have && ok) {
        // row m of the stage's tile in the 128-byte swizzle: 16-byte granule l / 2 at (l / 2) ^ (m % 8)
        *reinterpret_cast<uint2*>(sX + s * C::X_BYTES + m * BLK + (((l >> 1) ^ (m & 7)) << 4) + (l & 1) * 8) = w;
        if (l == 0) sS[g * C::SLOT + m] = most / MAXV;
        fence_proxy_async_smem();
        __syncwarp(mask);
        if (l == 0) {
          mbar_arrive(&full[s]);
          mbar_arrive(&sfull[g]);
        }
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, !ok)) break;
    }
    __syncwarp();
  }

  auto store = [&](int m, float v) {
    if (f < a.F) static_cast<TO*>(a.out)[m * a.ldo + f] = vec::from_f<TO>(v + (a.bias ? a.bias[f] : 0.f));
  };
  const bool sums = warp >= 2 && warp < 6;
  if (a.splits == 1) {
    if (sums)
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (c < a.M) store(c, acc[c]);
  } else {
    cluster_wait();
    if (sums) {
      const uint32_t mine = smem_u32(parts) + uint32_t(split * BLK + q * 32 + lane) * 4;
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (c < a.M) st_cluster_f32(mapa_shared(mine + uint32_t(c / a.splits * a.splits) * BLK * 4, uint32_t(c % a.splits)), acc[c]);
    }
    cluster_sync_all();
    if (sums)
      for (int c = split; c < a.M; c += a.splits) {
        const float* p = parts + (c / a.splits * a.splits) * BLK + q * 32 + lane;
        float v = 0.f;
        for (int k = 0; k < a.splits; ++k) v += p[k * BLK];
        store(c, v);
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// ---- many rows ------------------------------------------------------------------------------
// Persistent; PAIR: two SMs (a cluster of 2) share a 256 x 256 tile by one cta_group::2 product, each
// staging half of either operand, else one SM has a 128 x 128 or 128 x 256 tile.  A stage's bytes pass
// shared memory twice, written by TMA and read by the tensor core: 64 KB for 512 cycles of products in a
// pair, 96 KB on one SM with a 128 x 256 tile, which that bounds.  Every block of 128 of the
// reduction goes to one of two TMEM accumulators, and the hand-over between products and sums is what
// a block costs: 840 cycles a pair's, of which the products are 541 (without any scaling 690).  Under
// sustained load the 1 kW limit binds: 77% of the same kernel's rate without scales.  8192 x 4096 ->
// 28672 takes 0.91 ms by itself (2.1 PFLOP/s) and 1.05 under a long load (1.54 GHz at that limit), 2048 x
// 4096 -> 14336 0.131 and 0.145, with row scales and weight scales applied, rows quantised before.
//   warps 0..7   scaled sums in registers: a row a thread, half of the tile's features (warps 0-3 the first)
//   warp 8       TMA;  warp 9  tcgen05.mma (in the pair's first block);  warps 10, 11 only give up registers
template <bool PAIR, int BN_>
struct Many {
  static constexpr int BM = PAIR ? 256 : 128, BN = BN_, W_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int X_BYTES = 128 * BLK, W_BYTES = W_ROWS * BLK, STAGE = X_BYTES + W_BYTES;  // of one block
  static constexpr int STAGES = W_ROWS == 256 ? 3 : 5;
  static constexpr int RING = STAGES + 2;  // row scales outlive their tile by the two accumulators
  static constexpr int OUT = 32 * 128;     // one warp's staging tile: 32 rows of 128 bytes
  static constexpr int SMEM = STAGES * STAGE + 8 * OUT + RING * 512 + 1024 + 256;
  static constexpr int GROUP = 4096 / BN;  // feature tiles walked together (L2 reuse)
  static constexpr int COLS = BN / 2;      // features of a thread
  // registers of a thread: the launch gives 168, the summing warps take what the others give up
  static constexpr int REGS_SUM = 224, REGS_REST = 56;
};
constexpr int MANY_THREADS = 384;

__device__ __forceinline__ void walk(int t, int num_m, int num_f, int group, int& mt, int& ft) {
  const int g = t / (num_m * group), first = g * group;
  const int size = min(group, num_f - first);
  const int r = t - g * num_m * group;
  mt = r / size;
  ft = first + r % size;
}

// A warp stores 128 bytes of each of its 32 rows (lane: row `lane`, values v, from column c0 of the
// tile's feature range) through its staging tile, so that a store instruction covers 4 rows x 128
// contiguous bytes.  `wide`: rows of out start on 16 bytes.
template <class TO>
__device__ __forceinline__ void store_rows(uint8_t* stage, const float* v, TO* out, int64_t ldo, int row0, int M, int c0,
                                           int F, int lane, bool wide) {
  constexpr int PER = 16 / int(sizeof(TO));
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    vec::Pack<TO, PER> p;
#pragma unroll
    for (int j = 0; j < PER; ++j) p.set(j, v[g * PER + j]);
    p.store(reinterpret_cast<TO*>(stage + lane * 128 + ((g ^ (lane & 7)) << 4)));
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3), g = lane & 7;
    const int row = row0 + r, col = c0 + g * PER;
    vec::Pack<TO, PER> p;
    p.load(reinterpret_cast<const TO*>(stage + r * 128 + ((g ^ (r & 7)) << 4)));
    if (row < M && col < F) {
      TO* o = out + int64_t(row) * ldo + col;
      if (wide && col + PER <= F) {
        p.store(o);
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (col + j < F) o[j] = vec::from_f<TO>(p.get(j));
      }
    }
  }
  __syncwarp();
}

template <bool PAIR, int BN, bool W_MN, class TO>
__global__ void __launch_bounds__(MANY_THREADS, 1)
    many_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                     const __grid_constant__ CUtensorMap tmS, const __grid_constant__ Prod a) {
  using C = Many<PAIR, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sW = smem + C::STAGES * C::X_BYTES;
  uint8_t* sOut = smem + C::STAGES * C::STAGE;
  float* sS = reinterpret_cast<float*>(sOut + 8 * C::OUT);       // [RING][128] scales of the block's rows
  uint64_t* full = reinterpret_cast<uint64_t*>(sS + C::RING * 128);  // in the first block: both blocks' loads
  uint64_t* empty = full + C::STAGES;                            // in each block
  uint64_t* tfull = empty + C::STAGES;                           // in each block
  uint64_t* tempty = tfull + 2;                                  // in the first block: both blocks' warps
  // PAIR, in each block: its own warps have read a slot of row scales.  On one SM tempty says as much.
  uint64_t* sfree = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sfree + C::RING);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = PAIR ? int(cluster_ctarank()) : 0;
  const int first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x, tile_step = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int num_m = (a.M + C::BM - 1) / C::BM, num_f = (a.F + C::BN - 1) / C::BN, tiles = num_m * num_f;
  const int RB = (a.R + BLK - 1) / BLK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&tfull[s], 1);
      mbar_init(&tempty[s], PAIR ? 16 : 8);
    }
    if (PAIR)
      for (int s = 0; s < C::RING; ++s) mbar_init(&sfree[s], 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, 2 * C::BN);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 2 * C::BN);
      tmem_relinquish();
    }
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // both blocks' barriers stand before any remote arrival
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_REST));
    if (warp == 8) {
      if (elect_one()) {
        uint32_t it = 0;
        bool ok = true;
        for (int t = first_tile; t < tiles && ok; t += tile_step) {
          int mt, ft;
          walk(t, num_m, num_f, C::GROUP, mt, ft);
          const int row = mt * C::BM + cta * 128, col = ft * C::BN + cta * C::W_ROWS;
          for (int rb = 0; rb < RB; ++rb, ++it) {
            const int s = it % C::STAGES;
            if (!wait_bar(&empty[s], ((it / C::STAGES) & 1) ^ 1, abort_flag, a.status, kTimeoutTmaProducer)) {
              ok = false;
              break;
            }
            float* ss = sS + (it % C::RING) * 128;
            if (PAIR && !wait_bar(&sfree[it % C::RING], ((it / C::RING) & 1) ^ 1, abort_flag, a.status, kTimeoutTmaProducer)) {
              ok = false;
              break;
            }
            if (PAIR) {
              const uint32_t fb = mapa_shared(smem_u32(&full[s]), 0);
              if (cta == 0) mbar_arrive_expect_tx(&full[s], 2 * (C::STAGE + 512));
              tma_load_2d_pair(sX + s * C::X_BYTES, &tmX, fb, rb * BLK, row);
              tma_load_2d_pair(ss, &tmS, fb, row, rb);
              if (W_MN) tma_load_2d_pair(sW + s * C::W_BYTES, &tmW, fb, col, rb * BLK);
              else tma_load_2d_pair(sW + s * C::W_BYTES, &tmW, fb, rb * BLK, col);
            } else {
              mbar_arrive_expect_tx(&full[s], C::STAGE + 512);
              tma_load_2d(sX + s * C::X_BYTES, &tmX, &full[s], rb * BLK, row);
              tma_load_2d(ss, &tmS, &full[s], row, rb);
              if (W_MN) {
#pragma unroll
                for (int c = 0; c < C::W_ROWS / 128; ++c)
                  tma_load_2d(sW + s * C::W_BYTES + c * 16384, &tmW, &full[s], col + c * 128, rb * BLK);
              } else tma_load_2d(sW + s * C::W_BYTES, &tmW, &full[s], rb * BLK, col);
            }
          }
        }
        if (!ok && cta == 0) {  // the copies in flight land before the block leaves
          const uint32_t first = it > C::STAGES ? it - C::STAGES : 0;
          for (uint32_t j = first; j < it; ++j) {
            volatile int dummy = 0;
            mbar_wait_bounded(&full[j % C::STAGES], (j / C::STAGES) & 1, &dummy, nullptr, 0);
          }
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      if (cta == 0 && elect_one()) {
        constexpr uint32_t idesc = make_idesc(C::BM, C::BN, false, W_MN);
        uint32_t it = 0;
        bool ok = true;
        for (int t = first_tile; t < tiles && ok; t += tile_step) {
          for (int rb = 0; rb < RB; ++rb, ++it) {
            const int s = it % C::STAGES, c = it & 1;
            // the stage is there long before; the accumulator is what the products wait for
            if (!wait_bar(&full[s], (it / C::STAGES) & 1, abort_flag, a.status, kTimeoutMmaFull) ||
                !wait_bar(&tempty[c], ((it >> 1) & 1) ^ 1, abort_flag, a.status, kTimeoutMmaTmemEmpty)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t x = smem_u32(sX + s * C::X_BYTES), w = smem_u32(sW + s * C::W_BYTES);
#pragma unroll
            for (int k = 0; k < BLK / 32; ++k) {
              const uint64_t xd = make_sdesc_sw128_kmajor(x + k * 32);
              const uint64_t wd = W_MN ? make_sdesc_sw128_mnmajor(w + k * 4096, 16384) : make_sdesc_sw128_kmajor(w + k * 32);
              if (PAIR) umma_e4m3_pair(tmem + c * C::BN, xd, wd, idesc, k > 0);
              else umma_e4m3(tmem + c * C::BN, xd, wd, idesc, k > 0);
            }
            if (PAIR) {
              const uint32_t e = smem_u32(&empty[s]), f = smem_u32(&tfull[c]);
              umma_commit_pair(f);
              umma_commit_pair(mapa_shared(f, 1));
              umma_commit_pair(e);
              umma_commit_pair(mapa_shared(e, 1));
            } else {
              umma_commit(&tfull[c]);
              umma_commit(&empty[s]);
            }
          }
        }
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SUM));
    const int q = warp & 3, half = warp >> 2;
    constexpr int COLS = C::COLS, CHUNKS = COLS / 32;
    uint8_t* stage = sOut + warp * C::OUT;
    const bool wide = (a.ldo * int64_t(sizeof(TO))) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
    const uint32_t lead_empty = PAIR ? mapa_shared(smem_u32(tempty), 0) : 0u;
    const uint32_t lanes = tmem + (uint32_t(q * 32) << 16) + half * COLS;
    const float* my_scale = sS + q * 32 + lane;
    uint32_t it = 0;
    int g = 0;
    bool ok = true;
    for (int t = first_tile; t < tiles && ok; t += tile_step) {
      int mt, ft;
      walk(t, num_m, num_f, C::GROUP, mt, ft);
      const int row0 = mt * C::BM + cta * 128 + q * 32;
      const int col0 = ft * C::BN + half * COLS;
      const float* ws = a.ws + (col0 / BLK) * a.ws_f;
      float wv = 0.f;  // lane l: the weight's scale of block (rb & ~31) + l
      float acc[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
      // A block's turn is bounded by what this warp does in a row, so nothing in it waits: a chunk of 32
      // columns is read while the one before it is added, and the next block's first chunk while
      // this block's last one is, where that block's products are done by then (`ahead`).
      uint32_t r[2][32];
      bool ahead = false;
      for (int rb = 0; rb < RB; ++rb, ++it) {
        if ((rb & 31) == 0) wv = rb + lane < RB && col0 < a.F ? ws[(rb + lane) * a.ws_r] : 0.f;
        const int c = it & 1;
        const uint32_t at = lanes + c * C::BN;
        if (!ahead) {
          ok = __all_sync(0xffffffffu, wait_bar(&tfull[c], (it >> 1) & 1, abort_flag, a.status, kTimeoutEpilogue));
          if (!ok) break;  // the warp leaves as one
          tc_fence_after();
          tmem_ld_32x32b_x32(at, r[0]);
        }
        const float sc = my_scale[g * 128] * __shfl_sync(0xffffffffu, wv, rb & 31);
        const uint32_t scale_read = smem_u32(&sfree[g]);
        g = g + 1 == C::RING ? 0 : g + 1;
#pragma unroll
        for (int h = 0; h < CHUNKS; ++h) {
          tmem_ld_wait();
          if (h + 1 < CHUNKS) {
            tmem_ld_32x32b_x32(at + (h + 1) * 32, r[(h + 1) & 1]);
          } else {  // read out: the accumulator is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_pair(lead_empty + c * 8);
              else mbar_arrive(&tempty[c]);
            }
            ahead = rb + 1 < RB && __all_sync(0xffffffffu, mbar_test(&tfull[c ^ 1], ((it + 1) >> 1) & 1));
            if (ahead) {
              tc_fence_after();
              tmem_ld_32x32b_x32(lanes + (c ^ 1) * C::BN, r[0]);
            }
            if (PAIR && lane == 0) mbar_arrive_pair(scale_read);  // behind what the next block waits for
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[h * 32 + i] += __uint_as_float(r[h & 1][i]) * sc;
        }
      }
      if (!ok) break;
      constexpr int CH = 128 / int(sizeof(TO));  // columns of a staged store
#pragma unroll
      for (int c = 0; c < COLS / CH; ++c) {
        if (a.bias) {
#pragma unroll
          for (int i = 0; i < CH; ++i)
            if (col0 + c * CH + i < a.F) acc[c * CH + i] += __ldg(a.bias + col0 + c * CH + i);
        }
        store_rows<TO>(stage, acc + c * CH, static_cast<TO*>(a.out), a.ldo, row0, a.M, col0 + c * CH, a.F, lane, wide);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // no block leaves while its pair may still touch its memory
  if (warp == 9) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem, 2 * C::BN);
    else tmem_dealloc(tmem, 2 * C::BN);
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

static bool rows_aligned(const torch::Tensor& x) {
  return x.size(1) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 &&
         (x.size(0) <= 1 || (x.stride(0) * x.element_size()) % 16 == 0);
}

static bool float_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

static void check_rows(const torch::Tensor& x, const char* what) {
  SB_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) <= 1 || x.stride(1) == 1) && float_type(x.scalar_type()), what,
           ": CUDA bf16, fp16 or fp32 [rows, columns], columns contiguous");
  SB_CHECK(x.size(1) >= 1 && x.size(0) < (1ll << 31) - 256 && x.size(1) < (1ll << 31) - 256, what, ": size");
}

// Kernel attributes are set once for each kernel (K is its address) and device.
template <auto K>
static void set_once(cudaFuncAttribute what, int value) {
  static std::atomic<uint64_t> done{0};
  const int device = c10::cuda::current_device();
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (done.load() & bit) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(K, what, value));
  done.fetch_or(bit);
}

template <class T>
static void quantize_rows_t(const torch::Tensor& x, uint8_t* q, int64_t ldq, float* s, int64_t lds, cudaStream_t st) {
  const int64_t M = x.size(0), K = x.size(1), KB = (K + BLK - 1) / BLK;
  const int64_t rb = (M + 15) / 16;
  // several blocks of 128 a half-warp once there are blocks for every SM without
  const int per = rb * KB >= 148 * 8 * 2 ? 4 : 1;
  const int64_t ny = (KB + per - 1) / per;
  SB_CHECK(ny <= 65535, "quantize_fp8: rows of more than 8 million values");
  const dim3 grid{unsigned(rb), unsigned(ny)};
  const T* p = static_cast<const T*>(x.data_ptr());
  auto go = [&](auto aligned, auto n) {
    constexpr auto kern = quantize_rows_kernel<T, decltype(aligned)::value, decltype(n)::value>;
    // The SM's memory is divided as the product's blocks want it, or none of them starts beside this kernel.
    set_once<kern>(cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    kern<<<grid, 256, 0, st>>>(p, x.stride(0), M, K, q, ldq, s, lds);
  };
  using One = std::integral_constant<int, 1>;
  using Four = std::integral_constant<int, 4>;
  if (rows_aligned(x)) per == 1 ? go(std::true_type{}, One{}) : go(std::true_type{}, Four{});
  else per == 1 ? go(std::false_type{}, One{}) : go(std::false_type{}, Four{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

static void quantize_rows(const torch::Tensor& x, uint8_t* q, int64_t ldq, float* s, int64_t lds, cudaStream_t st) {
  if (x.scalar_type() == at::kBFloat16) quantize_rows_t<__nv_bfloat16>(x, q, ldq, s, lds, st);
  else if (x.scalar_type() == at::kHalf) quantize_rows_t<__half>(x, q, ldq, s, lds, st);
  else quantize_rows_t<float>(x, q, ldq, s, lds, st);
}

template <class T>
static void quantize_blocks_t(const torch::Tensor& x, uint8_t* q, int64_t ldq, float* s, cudaStream_t st) {
  const int64_t N = x.size(0), K = x.size(1);
  const int64_t nb = (N + BLK - 1) / BLK;
  SB_CHECK(nb <= 65535, "quantize_fp8: more than 8 million rows");
  const dim3 grid{unsigned((K + BLK - 1) / BLK), unsigned(nb)};
  const T* p = static_cast<const T*>(x.data_ptr());
  if (rows_aligned(x)) quantize_blocks_kernel<T, true><<<grid, 256, 0, st>>>(p, x.stride(0), N, K, q, ldq, s);
  else quantize_blocks_kernel<T, false><<<grid, 256, 0, st>>>(p, x.stride(0), N, K, q, ldq, s);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// The weight as the product reads it: features F, reduction R, and where its scales lie.
struct Weight {
  const void* q;
  int64_t ld, F, R;
  bool mn;  // stored [R, F]: the gradient's product
  const float* ws;
  int64_t ws_f, ws_r;
};

static Weight weight_of(const torch::Tensor& w, const torch::Tensor& s, bool transposed) {
  SB_CHECK(w.is_cuda() && w.dim() == 2 && w.scalar_type() == at::kFloat8_e4m3fn && (w.size(1) <= 1 || w.stride(1) == 1),
           "fp8 product: the weight must be CUDA e4m3 [features, width], width contiguous");
  const int64_t N = w.size(0), K = w.size(1);
  SB_CHECK(N >= 1 && K >= 1 && N < (1ll << 31) - 256 && K < (1ll << 31) - 256, "fp8 product: size of the weight");
  const int64_t ld = N > 1 ? w.stride(0) : up(K, 16);
  SB_CHECK(ld % 16 == 0 && ld >= K && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
           "fp8 product: rows of the weight must start on 16 bytes (quantize_fp8 lays them out so)");
  const int64_t NB = (N + BLK - 1) / BLK, KB = (K + BLK - 1) / BLK;
  SB_CHECK(s.device() == w.device() && s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == NB && s.size(1) == KB,
           "fp8 product: the weight's scales must be fp32 [", NB, ", ", KB, "]");
  Weight r{};
  r.q = w.data_ptr();
  r.ld = ld;
  r.mn = transposed;
  r.F = transposed ? K : N;
  r.R = transposed ? N : K;
  r.ws = s.data_ptr<float>();
  r.ws_f = transposed ? s.stride(1) : s.stride(0);
  r.ws_r = transposed ? s.stride(0) : s.stride(1);
  return r;
}

// Tensor maps are made by the driver, which wants a current context: a thread that has called nothing
// of the runtime yet (autograd's, for one) has none.
static void bind_context(const torch::Tensor& t) { C10_CUDA_CHECK(cudaSetDevice(t.device().index())); }

static CUtensorMap weight_map(const Weight& w, int box_features) {
  // box: 128 along the stored row by 128 (or the tile's features) rows
  const int64_t rows = w.mn ? w.R : w.F, cols = w.mn ? w.F : w.R;
  return make_tmap_2d(w.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, cols, w.ld, w.mn ? BLK : box_features, BLK,
                      CU_TENSOR_MAP_SWIZZLE_128B);
}

template <auto kern>
static void launch(dim3 grid, int threads, int smem, int cluster, bool dependent, cudaStream_t st,
                   const CUtensorMap& tW, const CUtensorMap& tX, const CUtensorMap& tS, const Prod& a) {
  set_once<kern>(cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (dependent) {  // may start while the kernel before it (the quantisation) still runs
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tW, tX, tS, a));
}

constexpr int FEW = 64;         // rows up to which the few-rows kernel runs
constexpr int FUSED_ROWS = 2;  // rows up to which it quantises them itself (of 4096 -> 6144: 2 rows 12 us, apart 14.6; 4 rows 17 against 14)

// Parts of the reduction: up to 8, and 256 blocks in all.  Blocks of half an SM's shared memory follow
// one another on it without a gap, so more parts than SMs pay until the clusters no longer fit side by
// side: 48 feature tiles of 32 blocks take 14.8, 11.2, 10.9, 10.6, 10.6, 12.9 us in 1 to 6 parts, 32
// tiles of 112 blocks 43, 29, 25, 22, 22, 21 and in 8 21; 224 tiles 25 us in one part, 29 in two.
static int splits_for(int64_t feature_tiles, int64_t reduction_blocks) {
  return int(std::max<int64_t>(1, std::min<int64_t>({256 / feature_tiles, 8, reduction_blocks})));
}

template <int NT, bool FUSED, class TX, class TO>
static void few_rows(const Weight& w, const CUtensorMap& tX, const CUtensorMap& tS, Prod a, bool x_aligned, bool dependent, cudaStream_t st) {
  const int64_t tiles = (w.F + BLK - 1) / BLK;
  SB_CHECK(tiles < (1ll << 27), "fp8 product: size of the weight");
  const CUtensorMap tW = weight_map(w, BLK);
  const int threads = FUSED ? 320 : 192, smem = Few<NT>::SMEM;
  a.splits = splits_for(tiles, (w.R + BLK - 1) / BLK);
  auto go = [&](auto aligned, auto mn) {
    launch<few_rows_kernel<NT, FUSED, decltype(aligned)::value, decltype(mn)::value, TX, TO>>(
        dim3(unsigned(tiles * a.splits)), threads, smem, a.splits, dependent, st, tW, tX, tS, a);
  };
  if constexpr (FUSED) {
    if (!x_aligned) {
      w.mn ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
      return;
    }
  }
  w.mn ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
}

template <bool PAIR, int BN, class TO>
static void many_rows(const Weight& w, const CUtensorMap& tX, const CUtensorMap& tS, const Prod& a, bool dependent, cudaStream_t st) {
  using C = Many<PAIR, BN>;
  const int64_t tiles = ((a.M + C::BM - 1) / C::BM) * ((w.F + C::BN - 1) / C::BN);
  SB_CHECK(tiles < (1ll << 30), "fp8 product: too many tiles");
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const dim3 grid{unsigned(PAIR ? 2 * std::min<int64_t>(tiles, sms / 2) : std::min<int64_t>(tiles, sms))};
  const CUtensorMap tW = weight_map(w, C::W_ROWS);
  const int cluster = PAIR ? 2 : 1;
  if (w.mn) launch<many_rows_kernel<PAIR, BN, true, TO>>(grid, MANY_THREADS, C::SMEM, cluster, dependent, st, tW, tX, tS, a);
  else launch<many_rows_kernel<PAIR, BN, false, TO>>(grid, MANY_THREADS, C::SMEM, cluster, dependent, st, tW, tX, tS, a);
}

// Quantised rows (uint8 [M, R] with row stride ldq) and their scales ([blocks][lds]) times the weight.
// `dependent`: launched right behind the kernel that quantises them, which may still run.
template <class TO>
static void product(const uint8_t* q, int64_t ldq, const float* scales, int64_t lds, const Weight& w, const Prod& a, bool dependent, cudaStream_t st) {
  const int box = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= FEW ? 64 : 128;
  const CUtensorMap tX = make_tmap_2d(q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.M, w.R, ldq, box, BLK, CU_TENSOR_MAP_SWIZZLE_128B);
  const CUtensorMap tS = make_tmap_2d(scales, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, (w.R + BLK - 1) / BLK, a.M, lds * 4, 1, box,
                                      CU_TENSOR_MAP_SWIZZLE_NONE);
  if (a.M <= 16) few_rows<16, false, float, TO>(w, tX, tS, a, true, dependent, st);
  else if (a.M <= 32) few_rows<32, false, float, TO>(w, tX, tS, a, true, dependent, st);
  else if (a.M <= FEW) few_rows<64, false, float, TO>(w, tX, tS, a, true, dependent, st);
  else {
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    // While one wave of SMs holds all tiles, the time is that of one tile: 0.37 us a block of 128 for 128
    // features, 0.49 for 256, 0.54 for a pair's (333 x 5120 -> 7168: 44, 29 and 31 us).  Beyond, a pair's
    // tile costs least for its size (2048 x 4096 -> 14336: 176, 146 and 137 us).
    const int64_t m = (a.M + 127) / 128;
    if (m * ((w.F + 127) / 128) <= sms) many_rows<false, 128, TO>(w, tX, tS, a, dependent, st);
    else if (m * ((w.F + 255) / 256) <= sms) many_rows<false, 256, TO>(w, tX, tS, a, dependent, st);
    else many_rows<true, 256, TO>(w, tX, tS, a, dependent, st);
  }
}

static Prod prod_of(const Weight& w, int64_t M, const c10::optional<torch::Tensor>& bias, const torch::Tensor& out,
                    const torch::Tensor& status, const torch::Tensor& weight) {
  SB_CHECK(out.device() == weight.device() && out.dim() == 2 && out.size(0) == M && out.size(1) == w.F &&
               (w.F <= 1 || out.stride(1) == 1) && (M <= 1 || out.stride(0) >= w.F) && float_type(out.scalar_type()),
           "fp8 product: out must be bf16, fp16 or fp32 [rows, features] on the weight's device, rows apart");
  if (bias)
    SB_CHECK(bias->device() == weight.device() && bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                 bias->size(0) == w.F && bias->is_contiguous(),
             "fp8 product: bias must be contiguous fp32 [features]");
  SB_CHECK(status.device() == weight.device() && status.scalar_type() == at::kInt && status.numel() >= 1, "fp8 product: status word");
  Prod a{};
  a.ws = w.ws;
  a.ws_f = w.ws_f;
  a.ws_r = w.ws_r;
  a.bias = bias ? bias->data_ptr<float>() : nullptr;
  a.out = out.data_ptr();
  a.ldo = M > 1 ? out.stride(0) : w.F;
  a.M = int(M);
  a.F = int(w.F);
  a.R = int(w.R);
  a.status = status.data_ptr<int>();
  return a;
}

template <class T>
static void linear_t(const torch::Tensor& x, const Weight& w, Prod a, cudaStream_t st) {
  if (a.M <= FUSED_ROWS) {
    a.x = x.data_ptr();
    a.ldx = x.stride(0);
    few_rows<16, true, T, T>(w, CUtensorMap{}, CUtensorMap{}, a, rows_aligned(x), false, st);
    return;
  }
  const int64_t ldq = up(w.R, 16), lds = up(a.M, 4), RB = (w.R + BLK - 1) / BLK;
  // one allocation: the values, then the scales
  const int64_t values = up(a.M * ldq, 256);
  torch::Tensor held = torch::empty({values + RB * lds * 4}, x.options().dtype(at::kByte));
  uint8_t* q = held.data_ptr<uint8_t>();
  float* s = reinterpret_cast<float*>(q + values);
  quantize_rows(x, q, ldq, s, lds, st);
  // dependent: the quantisation itself began after everything before it had ended
  product<T>(q, ldq, s, lds, w, a, true, st);
}

}  // namespace fp8

// e4m3 values and scales of x [rows, columns]: `block_rows` 1 gives a scale for each row's 128
// columns, 128 one for each 128 x 128 block.  The values' rows start on 16 bytes; row scales come
// back as a [rows, blocks] view of column-major storage.
std::tuple<torch::Tensor, torch::Tensor> quantize_fp8(const torch::Tensor& x, int64_t block_rows) {
  fp8::check_rows(x, "quantize_fp8");
  SB_CHECK(block_rows == 1 || block_rows == fp8::BLK, "quantize_fp8: block_rows must be 1 or 128, got ", block_rows);
  const at::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int64_t M = x.size(0), K = x.size(1), KB = (K + fp8::BLK - 1) / fp8::BLK, ldq = fp8::up(K, 16);
  torch::Tensor q = torch::empty({M, ldq}, x.options().dtype(at::kByte));
  uint8_t* qp = q.data_ptr<uint8_t>();
  torch::Tensor s;
  if (block_rows == 1) {
    const int64_t lds = fp8::up(M, 4);
    torch::Tensor store = torch::empty({KB, lds}, x.options().dtype(at::kFloat));
    if (M) fp8::quantize_rows(x, qp, ldq, store.data_ptr<float>(), lds, st);
    s = store.t().narrow(0, 0, M);
  } else {
    s = torch::empty({(M + fp8::BLK - 1) / fp8::BLK, KB}, x.options().dtype(at::kFloat));
    float* sp = s.data_ptr<float>();
    if (M == 0) {
    } else if (x.scalar_type() == at::kBFloat16) fp8::quantize_blocks_t<__nv_bfloat16>(x, qp, ldq, sp, st);
    else if (x.scalar_type() == at::kHalf) fp8::quantize_blocks_t<__half>(x, qp, ldq, sp, st);
    else fp8::quantize_blocks_t<float>(x, qp, ldq, sp, st);
  }
  return {q.narrow(1, 0, K).view(at::kFloat8_e4m3fn), s};
}

// out = quantised x times the weight (transposed: the product over the weight's rows, the gradient
// of x), plus bias.  x [rows, R] bf16, fp16 or fp32; weight e4m3 [N, K], scales [N / 128, K / 128].
void fp8_product(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& scale,
                 const c10::optional<torch::Tensor>& bias, bool transposed, const torch::Tensor& out,
                 const torch::Tensor& status) {
  fp8::check_rows(x, "linear_fp8");
  const fp8::Weight w = fp8::weight_of(weight, scale, transposed);
  SB_CHECK(x.device() == weight.device() && x.size(1) == w.R, "linear_fp8: x must be [rows, ", w.R, "] on the weight's device");
  SB_CHECK(out.scalar_type() == x.scalar_type(), "linear_fp8: out must have x's type");
  const fp8::Prod a = fp8::prod_of(w, x.size(0), bias, out, status, weight);
  if (a.M == 0) return;
  const at::cuda::CUDAGuard guard(x.device());
  fp8::bind_context(x);
  auto st = at::cuda::getCurrentCUDAStream();
  if (x.scalar_type() == at::kBFloat16) fp8::linear_t<__nv_bfloat16>(x, w, a, st);
  else if (x.scalar_type() == at::kHalf) fp8::linear_t<__half>(x, w, a, st);
  else fp8::linear_t<float>(x, w, a, st);
}

// The same for rows that are quantised already: a e4m3 [rows, K], its scales [rows, K / 128] with
// stride 1 between rows (quantize_fp8's).
void gemm_fp8(const torch::Tensor& a, const torch::Tensor& a_scale, const torch::Tensor& weight,
              const torch::Tensor& scale, const c10::optional<torch::Tensor>& bias, const torch::Tensor& out,
              const torch::Tensor& status) {
  const fp8::Weight w = fp8::weight_of(weight, scale, false);
  const int64_t M = a.dim() == 2 ? a.size(0) : 0, RB = (w.R + fp8::BLK - 1) / fp8::BLK;
  SB_CHECK(a.device() == weight.device() && a.dim() == 2 && a.scalar_type() == at::kFloat8_e4m3fn && a.size(1) == w.R &&
               (w.R <= 1 || a.stride(1) == 1) && M < (1ll << 31) - 256,
           "gemm_fp8: a must be e4m3 [rows, ", w.R, "] on the weight's device, columns contiguous");
  const int64_t ldq = M > 1 ? a.stride(0) : fp8::up(w.R, 16);
  SB_CHECK(ldq % 16 == 0 && ldq >= w.R && reinterpret_cast<uintptr_t>(a.data_ptr()) % 16 == 0,
           "gemm_fp8: rows of a must start on 16 bytes (quantize_fp8 lays them out so)");
  SB_CHECK(a_scale.device() == a.device() && a_scale.scalar_type() == at::kFloat && a_scale.dim() == 2 &&
               a_scale.size(0) == M && a_scale.size(1) == RB && (M <= 1 || a_scale.stride(0) == 1),
           "gemm_fp8: a's scales must be fp32 [", M, ", ", RB, "] with stride 1 between rows");
  const fp8::Prod p = fp8::prod_of(w, M, bias, out, status, weight);
  if (M == 0) return;
  const int64_t lds = RB > 1 ? a_scale.stride(1) : fp8::up(M, 4);
  SB_CHECK(lds % 4 == 0 && lds >= M && reinterpret_cast<uintptr_t>(a_scale.data_ptr()) % 16 == 0,
           "gemm_fp8: a's scales must be laid out as quantize_fp8 does (blocks 16-byte aligned)");
  const float* sp = a_scale.data_ptr<float>();
  const at::cuda::CUDAGuard guard(a.device());
  fp8::bind_context(a);
  auto st = at::cuda::getCurrentCUDAStream();
  const uint8_t* q = static_cast<const uint8_t*>(a.data_ptr());
  if (out.scalar_type() == at::kBFloat16) fp8::product<__nv_bfloat16>(q, ldq, sp, lds, w, p, false, st);
  else if (out.scalar_type() == at::kHalf) fp8::product<__half>(q, ldq, sp, lds, w, p, false, st);
  else fp8::product<float>(q, ldq, sp, lds, w, p, false, st);
}

}  // namespace sb
