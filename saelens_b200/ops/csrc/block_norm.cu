// The end of one sub-block of a decoder and the start of the next, in one pass over the rows:
//     u = post(branch)            (post-norm, optional)
//     r = x + scale * gate * u    (gate optional; r is rounded to the rows' type: the stream)
//     y = pre(r)                  (the norm that the next sub-block reads; it reads the stored r)
// with post and pre both RMS norms, t s w with s = rsqrt(mean(t^2) + eps), or both layer norms,
// (t - mean) s w + b with s = rsqrt(mean((t - mean)^2) + eps); `one_plus` weighs with 1 + w.
// `round_branch` also rounds u, and scale * gate * u where there is one, to the rows' type: what a
// program that stores the branch before it adds it computes.
//
// Backward, with t^ = (t - mean) s and h = g w for an incoming gradient g of a norm's output:
//     dt = s (h - [mean(h)] - t^ mean(h t^)),  dw = sum over rows of g t^,  db = sum of g
//     dx = dr + dpre,  du = scale gate dx,  dgate = sum of scale dx u,  dbranch = dpost(du).
//
// Memory bounds both directions: forward reads x and branch and writes r and y, backward reads
// dr, dy, r and the branch where it is needed, and writes dx and dbranch.  8192 bf16 rows of 4096 go
// forward in 42 us (6.3 TB/s), with a post-norm in 48; backward, which also waits for its rows and
// adds column sums, in 79 (3.4 TB/s) and 137.  A row is held in the
// registers of one block between the sums, so every value moves once.  Sums are 32-bit and
// deterministic: thread t holds the vectors t, t + threads, ..., lanes are joined by a butterfly
// and warps in order, and a layer norm's weight and bias enter as one fused multiply-add, as in the
// single norms of the producer, so that the results are theirs bit for bit.
// Column sums of the backward pass are kept by the thread that owns the column, over consecutive
// rows; a second kernel adds the blocks' sums in block order.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include <algorithm>
#include <type_traits>

#include "block_ops.h"
#include "check.h"
#include "vec.cuh"

namespace sb {
namespace bnorm {

constexpr int THREADS = 256;          // of a row in vectors of 8
constexpr int THREADS_NARROW = 512;   // of a wide row in single values
template <int VEC>
constexpr int MAX_THREADS = VEC == 1 ? THREADS_NARROW : THREADS;
template <int VEC>
constexpr int WARPS = MAX_THREADS<VEC> / 32;

// Sum over the block; `red` is one of the caller's buffers of MOST floats, each used once a row.
template <int MOST>
__device__ __forceinline__ float block_sum(float v, float* red, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (i < warps) t += red[i];
  return t;
}
struct Fwd {
  const void *x, *branch, *w, *b, *post_w, *post_b, *gate;
  int64_t ldx, ldb;    // row strides of x and branch
  int64_t gate_div;    // gate row of a row: row / gate_div
  void *stream, *normed;
  float *rstd, *mean, *post_rstd, *post_mean;  // per row, or nullptr
  int D;
  float eps, post_eps, scale;
  int one_plus, round_branch;
};

// NV vectors of VEC elements a thread; POST: there is a post-norm; LAYER: layer norms.
// What hides the latencies of a row (loads, one to four sums, vectors from the L2 cache) is other rows
// on the SM, so registers are held to what FWD_BLOCKS blocks leave.
template <class T, int VEC, int NV>
constexpr int FWD_BLOCKS = VEC == 1                     ? (NV <= 4 ? 3 : NV <= 8 ? 2 : 1)
                           : NV * int(sizeof(T)) <= 2 ? 7
                           : NV * int(sizeof(T)) <= 4 ? 6
                           : NV * int(sizeof(T)) <= 8 ? 3
                                                      : 1;
template <class T, int VEC, int NV, bool LAYER, bool POST>
__global__ void __launch_bounds__(MAX_THREADS<VEC>, FWD_BLOCKS<T, VEC, NV>) fwd_kernel(const __grid_constant__ Fwd a) {
  __shared__ float red[4][WARPS<VEC>];
  using P = vec::Pack<T, VEC>;
  const int warps = blockDim.x >> 5;
  const int nvec = a.D / VEC;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* br = static_cast<const T*>(a.branch) + row * a.ldb;
  const T* gate = a.gate ? static_cast<const T*>(a.gate) + (row / a.gate_div) * a.D : nullptr;
  const float add = a.one_plus ? 1.f : 0.f;
  P px[NV], pb[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      pb[i].load(br + VEC * v);
      px[i].load(x + VEC * v);
    }
  }
  float mean = 0.f, inv = 1.f;
  if (POST) {
    float s = 0.f;
    if (LAYER) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (threadIdx.x + i * blockDim.x < nvec) {
          float f[VEC];
          pb[i].unpack(f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) s += f[j];
        }
      mean = block_sum<WARPS<VEC>>(s, red[0], warps) / float(a.D);
      s = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (threadIdx.x + i * blockDim.x < nvec) {
        float f[VEC];
        pb[i].unpack(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float c = LAYER ? f[j] - mean : f[j];
          s += c * c;
        }
      }
    inv = rsqrtf(block_sum<WARPS<VEC>>(s, red[1], warps) / float(a.D) + a.post_eps);
    if (a.post_rstd && threadIdx.x == 0) {
      a.post_rstd[row] = inv;
      if (LAYER) a.post_mean[row] = mean;
    }
  }
  float s = 0.f;
  // u: the branch's vector, through its norm where there is one -> the stream's vector
  auto finish = [&](int i, int v, float (&u)[VEC]) {
    float f[VEC];
    px[i].unpack(f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = __fadd_rn(f[j], u[j]);  // u is a value of its own, as a stored branch is
    px[i].pack(f);
    px[i].store(static_cast<T*>(a.stream) + row * a.D + VEC * v);
    px[i].unpack(f);  // as stored
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += LAYER ? f[j] : f[j] * f[j];
  };
  const bool plain = !gate && a.scale == 1.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      float u[VEC];
      pb[i].unpack(u);
      if (POST) {
        P w, b;
        float fw[VEC], fb[VEC];
        w.load(static_cast<const T*>(a.post_w) + VEC * v);
        w.unpack(fw);
        if (LAYER && a.post_b) b.load(static_cast<const T*>(a.post_b) + VEC * v);
        else b.zero();
        b.unpack(fb);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (LAYER) u[j] = __fmaf_rn((u[j] - mean) * inv, fw[j] + add, fb[j]);
          else u[j] = u[j] * inv * (fw[j] + add);
        }
        if (a.round_branch) {
          b.pack(u);
          b.unpack(u);
        }
      }
      if (!plain) {
        P g;
        float fg[VEC];
        if (gate) {
          g.load(gate + VEC * v);
          g.unpack(fg);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[j] = (gate ? u[j] * fg[j] : u[j]) * a.scale;
        if (a.round_branch) {
          g.pack(u);
          g.unpack(u);
        }
      }
      finish(i, v, u);
    }
  }
  float total = block_sum<WARPS<VEC>>(s, red[2], warps);
  if (LAYER) {
    mean = total / float(a.D);
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (threadIdx.x + i * blockDim.x < nvec) {
        float f[VEC];
        px[i].unpack(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += (f[j] - mean) * (f[j] - mean);
      }
    total = block_sum<WARPS<VEC>>(s, red[3], warps);
  }
  inv = rsqrtf(total / float(a.D) + a.eps);
  if (a.rstd && threadIdx.x == 0) {
    a.rstd[row] = inv;
    if (LAYER) a.mean[row] = mean;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      P w, b;
      float f[VEC], fw[VEC], fb[VEC];
      w.load(static_cast<const T*>(a.w) + VEC * v);
      w.unpack(fw);
      if (LAYER && a.b) b.load(static_cast<const T*>(a.b) + VEC * v);
      else b.zero();
      if (LAYER) b.unpack(fb);
      px[i].unpack(f);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        f[j] = LAYER ? __fmaf_rn((f[j] - mean) * inv, fw[j] + add, fb[j]) : f[j] * inv * (fw[j] + add);
      px[i].pack(f);
      px[i].store(static_cast<T*>(a.normed) + row * a.D + VEC * v);
    }
  }
}

// Column sums of the backward pass, in this order in shared memory and in the partial sums.
enum Sum { kW = 0, kB, kPostW, kPostB, kGate, kSums };

struct Bwd {
  const void *d_stream, *d_normed;  // either may be nullptr: no gradient came in
  int64_t ld_ds, ld_dn;
  const void *stream, *branch, *w, *post_w, *post_b, *gate;
  int64_t ldb, gate_div;
  const float *rstd, *mean, *post_rstd, *post_mean;
  void *dx, *dbranch;  // dbranch may be nullptr
  void* dgate;         // token gates: [rows, D]; sequence gates: [sequences, D]; else nullptr
  float* partial;      // [blocks][slots][D]
  float* edge;         // sequence gates: [units][2][D], sequences that reach over a unit's rows
  int slot[kSums];     // place of each sum among the `slots` that are wanted, or -1
  int slots;
  int64_t rows, rows_per_unit;  // a unit: the rows of one group
  int groups, group_threads;
  int D;
  float scale;
  int one_plus;
  int gate_mode;  // 0 none, 1 channel, 2 sequence, 3 token
};

// Sum over a group of `threads` threads of the block that meet at barrier `id`.
template <int MOST>
__device__ __forceinline__ float2 group_sum2(float2 v, float2* red, int tid, int threads, int id) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if ((tid & 31) == 0) red[tid >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
  float2 t = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < MOST; ++i)
    if (i < threads / 32) t.x += red[i].x, t.y += red[i].y;
  return t;
}

// A block is `groups` groups of threads, each with rows of its own.  Where a thread has one vector
// (rows of up to 2048 values) its column sums stay in registers and a block has several groups, so
// that rows wait for their sums side by side and there are few blocks' sums to join; wider rows keep
// theirs in shared memory, one group a block.  4104 fp32 rows of 768 with five sums: 39 -> 30 us, and
// the sums' join 10 -> 6.
constexpr int GROUP_THREADS = 512;
template <class T, int VEC, int NV, bool LAYER, bool POST>
__global__ void __launch_bounds__(VEC == 8 && NV == 1 ? GROUP_THREADS : MAX_THREADS<VEC>) bwd_kernel(const __grid_constant__ Bwd a) {
  constexpr bool REG = VEC == 8 && NV == 1;
  // [slots][VEC][vectors]: value j of vector v at (slot * VEC + j) * nvec + v, so that neighbouring
  // threads are in neighbouring banks
  extern __shared__ float sums[];
  constexpr int GROUPS = REG ? GROUP_THREADS / 32 : 1;
  __shared__ float2 red_all[GROUPS][2][2][WARPS<VEC>];
  using P = vec::Pack<T, VEC>;
  const int threads = a.group_threads;
  const int group = threadIdx.x / threads, tid = threadIdx.x - group * threads, bar = 1 + group;
  auto red = red_all[group];
  const int nvec = a.D / VEC;
  const int64_t unit = int64_t(blockIdx.x) * a.groups + group;
  const int64_t r0 = min(unit * a.rows_per_unit, a.rows), r1 = min(r0 + a.rows_per_unit, a.rows);
  auto sum_at = [&](int slot, int v, int j) -> float& { return sums[(slot * VEC + j) * nvec + v]; };
  float acc[REG ? kSums : 1][VEC];
  if (REG) {
#pragma unroll
    for (int k = 0; k < (REG ? kSums : 1); ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[k][j] = 0.f;
  } else {
    for (int v = tid; v < nvec; v += threads)
      for (int k = 0; k < a.slots; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum_at(k, v, j) = 0.f;
    // no barrier: a thread's columns are its own
  }
  auto add = [&](int kind, int v, int j, float value) {
    if (a.slot[kind] >= 0) {
      if constexpr (REG) acc[kind][j] += value;
      else sum_at(a.slot[kind], v, j) += value;
    }
  };
  const float one = a.one_plus ? 1.f : 0.f;
  const bool need_gate = a.gate_mode && (a.gate_mode == 3 ? a.dgate != nullptr : a.slot[kGate] >= 0);
  const bool need_branch = POST || need_gate;
  for (int64_t row = r0; row < r1; ++row) {
    const int par = int(row - r0) & 1;  // buffers of the block sums alternate between rows
    const T* st = static_cast<const T*>(a.stream) + row * a.D;
    const T* gate = a.gate_mode ? static_cast<const T*>(a.gate) + (row / a.gate_div) * a.D : nullptr;
    P pr[NV], pn[NV], ps[NV], pb[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tid + i * threads;
      if (v < nvec) {
        if (a.d_normed) {
          pn[i].load(static_cast<const T*>(a.d_normed) + row * a.ld_dn + VEC * v);
          pr[i].load(st + VEC * v);
        }
        if (a.d_stream) ps[i].load(static_cast<const T*>(a.d_stream) + row * a.ld_ds + VEC * v);
        else ps[i].zero();
        if (need_branch) pb[i].load(static_cast<const T*>(a.branch) + row * a.ldb + VEC * v);
      }
    }
    const float inv = a.rstd[row], mean = LAYER ? a.mean[row] : 0.f;
    const float pinv = POST ? a.post_rstd[row] : 1.f, pmean = POST && LAYER ? a.post_mean[row] : 0.f;
    float g[NV][VEC];  // the stream's gradient
    float2 c = make_float2(0.f, 0.f);
    if (a.d_normed) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = tid + i * threads;
        if (v < nvec) {
          P w;
          w.load(static_cast<const T*>(a.w) + VEC * v);
          float fw[VEC], fn[VEC], fr[VEC];
          w.unpack(fw);
          pn[i].unpack(fn);
          pr[i].unpack(fr);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float t = (LAYER ? fr[j] - mean : fr[j]) * inv, h = fn[j] * (fw[j] + one);
            g[i][j] = h;
            c.x += h * t;
            if (LAYER) c.y += h;
            add(kW, v, j, fn[j] * t);
            if (LAYER) add(kB, v, j, fn[j]);
          }
        }
      }
      c = group_sum2<WARPS<VEC>>(c, red[par][0], tid, threads, bar);
      c.x /= float(a.D);
      c.y /= float(a.D);
    }
    float2 e = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = tid + i * threads;
      if (v < nvec) {
        P pk;
        float dr[VEC], fw[VEC], u[VEC], bh[VEC], fg[VEC];
        ps[i].unpack(dr);
        if (a.d_normed) {
          float fr[VEC];
          pr[i].unpack(fr);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float t = (LAYER ? fr[j] - mean : fr[j]) * inv;
            dr[j] += inv * (g[i][j] - (LAYER ? c.y : 0.f) - t * c.x);
          }
        }
        pk.pack(dr);
        pk.store(static_cast<T*>(a.dx) + row * a.D + VEC * v);
        if (POST) {
          pk.load(static_cast<const T*>(a.post_w) + VEC * v);
          pk.unpack(fw);
        }
        if (need_branch) {
          pb[i].unpack(bh);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (POST) bh[j] = (LAYER ? bh[j] - pmean : bh[j]) * pinv;
        }
        if (a.gate_mode) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) u[j] = POST ? bh[j] * (fw[j] + one) : bh[j];
          if (POST && LAYER && a.post_b) {
            pk.load(static_cast<const T*>(a.post_b) + VEC * v);
            pk.unpack(fg);
#pragma unroll
            for (int j = 0; j < VEC; ++j) u[j] += fg[j];
          }
          if (need_gate) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              u[j] *= a.scale * dr[j];
              if (a.gate_mode != 3) add(kGate, v, j, u[j]);
            }
            if (a.gate_mode == 3) {
              pk.pack(u);
              pk.store(static_cast<T*>(a.dgate) + row * a.D + VEC * v);
            }
          }
          pk.load(gate + VEC * v);
          pk.unpack(fg);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float du = dr[j] * a.scale;
          if (a.gate_mode) du *= fg[j];
          if (POST) {
            add(kPostW, v, j, du * bh[j]);
            if (LAYER) add(kPostB, v, j, du);
            du *= fw[j] + one;
            e.x += du * bh[j];
            if (LAYER) e.y += du;
          }
          g[i][j] = du;
        }
      }
    }
    if (POST) {
      e = group_sum2<WARPS<VEC>>(e, red[par][1], tid, threads, bar);
      e.x /= float(a.D);
      e.y /= float(a.D);
    }
    if (a.dbranch) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = tid + i * threads;
        if (v < nvec) {
          P o;
          if (POST) {
            float fb[VEC];
            pb[i].unpack(fb);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const float bh = (LAYER ? fb[j] - pmean : fb[j]) * pinv;
              g[i][j] = pinv * (g[i][j] - (LAYER ? e.y : 0.f) - bh * e.x);
            }
          }
          o.pack(g[i]);
          o.store(static_cast<T*>(a.dbranch) + row * a.D + VEC * v);
        }
      }
    }
    // a sequence ends here or the unit's rows do: its gate's sum leaves the unit
    if (a.gate_mode == 2 && a.slot[kGate] >= 0) {
      const int64_t q = row / a.gate_div;
      const bool ends = (row + 1) % a.gate_div == 0;
      if (ends || row + 1 == r1) {
        const bool inside = q * a.gate_div >= r0;
        for (int v = tid; v < nvec; v += threads) {
          vec::Pack<float, VEC> f;
          P o;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float& s = REG ? acc[REG ? kGate : 0][j] : sum_at(a.slot[kGate], v, j);
            f.set(j, s);
            o.set(j, s);
            s = 0.f;
          }
          if (inside && ends) o.store(static_cast<T*>(a.dgate) + q * a.D + VEC * v);
          else f.store(a.edge + (unit * 2 + (inside ? 1 : 0)) * a.D + VEC * v);
        }
      }
    }
  }
  const int out_slots = a.gate_mode == 2 && a.slot[kGate] >= 0 ? a.slots - 1 : a.slots;  // the gate's slot is the last
  if (REG) {
    // the groups' sums in order of the groups, through one vector of shared memory a thread and kind
    for (int k = 0; k < kSums; ++k) {
      if (a.slot[k] < 0 || a.slot[k] >= out_slots) continue;  // uniform
      __syncthreads();
      if (tid < nvec)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float value = 0.f;
#pragma unroll
          for (int m = 0; m < (REG ? kSums : 1); ++m) value = m == k ? acc[m][j] : value;
          sums[(group * VEC + j) * threads + tid] = value;
        }
      __syncthreads();
      for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
        vec::Pack<float, VEC> f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float t = 0.f;
          for (int m = 0; m < a.groups; ++m) t += sums[(m * VEC + j) * threads + v];
          f.set(j, t);
        }
        f.store(a.partial + (int64_t(blockIdx.x) * out_slots + a.slot[k]) * a.D + VEC * v);
      }
    }
  } else {
    for (int v = tid; v < nvec; v += threads)
      for (int k = 0; k < out_slots; ++k) {
        vec::Pack<float, VEC> f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) f.set(j, sum_at(k, v, j));
        f.store(a.partial + (int64_t(blockIdx.x) * out_slots + k) * a.D + VEC * v);
      }
  }
}

struct Join {
  const float* partial;
  void* out[kSums];
  int blocks, slots, D;
};

// out[k][col] = sum of partial[block][k][col] over the blocks: 32 columns a block, JOIN_ROWS groups
// of blocks added in order, then the groups in order.
constexpr int JOIN_ROWS = 16;
template <class T>
__global__ void __launch_bounds__(32 * JOIN_ROWS) join_kernel(const __grid_constant__ Join a) {
  __shared__ float part[JOIN_ROWS][32];
  const int col = blockIdx.x * 32 + threadIdx.x, k = blockIdx.y;
  float s = 0.f;
  if (col < a.D) {
    const int64_t step = int64_t(a.slots) * a.D;
    const float* p = a.partial + int64_t(k) * a.D + col;
    const int per = (a.blocks + JOIN_ROWS - 1) / JOIN_ROWS;
    const int b0 = threadIdx.y * per, b1 = min(b0 + per, a.blocks);
#pragma unroll 8
    for (int b = b0; b < b1; ++b) s += p[b * step];
  }
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < a.D) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < JOIN_ROWS; ++i) t += part[i][threadIdx.x];
    static_cast<T*>(a.out[k])[col] = vec::from_f<T>(t);
  }
}

// Gates of sequences that lie in several units' rows: the units' parts in order.
template <class T>
__global__ void __launch_bounds__(256) edge_kernel(const float* edge, T* dgate, int64_t rows_per_unit, int64_t S, int D) {
  const int64_t q = blockIdx.x;
  const int64_t first = q * S / rows_per_unit, last = ((q + 1) * S - 1) / rows_per_unit;
  if (first == last) return;  // written by its unit
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= D) return;
  float s = 0.f;
  for (int64_t b = first; b <= last; ++b)
    s += edge[(b * 2 + (q * S >= b * rows_per_unit ? 1 : 0)) * D + col];
  dgate[q * D + col] = vec::from_f<T>(s);
}

// Threads of a row: one for each vector of 8 values (wide) or each value, up to a limit.  4096 bf16
// rows of single values with both norms take 18 us at width 1001 with 256 threads and 25 with 512, at
// 3585 83 and 61.
static int threads_for(int64_t D, bool wide) {
  const int64_t most = wide || D <= 4 * THREADS ? THREADS : THREADS_NARROW;
  return int(std::min<int64_t>(most, ((wide ? D / 8 : D) + 31) / 32 * 32));
}

// Calls f with (VEC, NV) as constants: the fewest vectors a thread that hold the row.
template <class F>
static void with_shape(int64_t D, bool wide, F f) {
  if (wide) {
    const int64_t nv = (D / 8 + THREADS - 1) / THREADS;
    if (nv <= 1) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    else if (nv <= 2) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    else if (nv <= 4) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
  } else {
    if (D <= 4 * THREADS) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    else if (D <= 8 * THREADS_NARROW) f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  }
}

template <class T>
static void run_fwd(const Fwd& a, int64_t rows, bool wide, bool layer, cudaStream_t stream) {
  const dim3 grid{unsigned(rows)}, block{unsigned(threads_for(a.D, wide))};
  with_shape(a.D, wide, [&](auto V, auto N) {
    constexpr int VEC = decltype(V)::value, NV = decltype(N)::value;
    if (layer && a.post_w) fwd_kernel<T, VEC, NV, true, true><<<grid, block, 0, stream>>>(a);
    else if (layer) fwd_kernel<T, VEC, NV, true, false><<<grid, block, 0, stream>>>(a);
    else if (a.post_w) fwd_kernel<T, VEC, NV, false, true><<<grid, block, 0, stream>>>(a);
    else fwd_kernel<T, VEC, NV, false, false><<<grid, block, 0, stream>>>(a);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <class T, int VEC, int NV, bool LAYER, bool POST>
static void launch_bwd(const Bwd& a, unsigned blocks, size_t smem, cudaStream_t stream) {
  auto kern = bwd_kernel<T, VEC, NV, LAYER, POST>;
  if (smem > 40 * 1024)
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  kern<<<dim3(blocks), dim3(a.groups * a.group_threads), smem, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <class T>
static void run_bwd(const Bwd& a, unsigned blocks, bool wide, bool layer, size_t smem, cudaStream_t stream) {
  with_shape(a.D, wide, [&](auto V, auto N) {
    constexpr int VEC = decltype(V)::value, NV = decltype(N)::value;
    if (layer && a.post_w) launch_bwd<T, VEC, NV, true, true>(a, blocks, smem, stream);
    else if (layer) launch_bwd<T, VEC, NV, true, false>(a, blocks, smem, stream);
    else if (a.post_w) launch_bwd<T, VEC, NV, false, true>(a, blocks, smem, stream);
    else launch_bwd<T, VEC, NV, false, false>(a, blocks, smem, stream);
  });
}

static bool aligned(const torch::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Widths are held in registers: 8 vectors of 8 a thread, or 16 single values where D is no multiple
// of 8 or a row does not start on 16 bytes.
constexpr int64_t MAX_D = 8 * 8 * THREADS, MAX_D_NARROW = 16 * THREADS_NARROW;
constexpr size_t MAX_SUMS = 224 * 1024;  // bytes of shared memory for column sums

}  // namespace bnorm

// See the head of this file.  x, branch: [rows, D] of one type (bf16, fp16, fp32), contiguous
// rows; vectors [D] and gate [gate_rows, D] contiguous, of the same type; row r reads gate row
// r / gate_div.  Writes stream and normed ([rows, D] contiguous) and, if given, the statistics
// stats [4, rows] fp32: rstd and mean of the pre-norm, rstd and mean of the post-norm.
void residual_norm_fwd(const torch::Tensor& x, const torch::Tensor& branch, const torch::Tensor& w,
                       const c10::optional<torch::Tensor>& b, const c10::optional<torch::Tensor>& post_w,
                       const c10::optional<torch::Tensor>& post_b, const c10::optional<torch::Tensor>& gate,
                       int64_t gate_div, double eps, double post_eps, double scale, bool layer, bool one_plus,
                       bool round_branch, const torch::Tensor& stream, const torch::Tensor& normed,
                       const c10::optional<torch::Tensor>& stats) {
  const auto type = x.scalar_type();
  SB_CHECK(x.is_cuda() && x.dim() == 2 && branch.sizes() == x.sizes(), "residual_norm: x and branch must be CUDA [rows, D]");
  SB_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "residual_norm: bf16, fp16 or fp32");
  const int64_t rows = x.size(0), D = x.size(1);
  SB_CHECK(D >= 1 && rows < (1ll << 31), "residual_norm: size");
  auto same = [&](const torch::Tensor& t) { return t.device() == x.device() && t.scalar_type() == type; };
  SB_CHECK(same(branch) && (D == 1 || (x.stride(1) == 1 && branch.stride(1) == 1)), "residual_norm: rows must be contiguous, of one type, on one device");
  auto vector = [&](const torch::Tensor& t) { return same(t) && t.dim() == 1 && t.size(0) == D && t.is_contiguous(); };
  SB_CHECK(vector(w) && (!b || vector(*b)) && (!post_w || vector(*post_w)) && (!post_b || vector(*post_b)),
           "residual_norm: weights and biases must be contiguous [D] of x's type");
  SB_CHECK((layer || (!b && !post_b)) && (post_w || !post_b), "residual_norm: biases belong to layer norms");
  SB_CHECK(same(stream) && same(normed) && stream.sizes() == x.sizes() && normed.sizes() == x.sizes() &&
               stream.is_contiguous() && normed.is_contiguous(),
           "residual_norm: outputs must be contiguous, like x");
  if (gate)
    SB_CHECK(same(*gate) && gate->dim() == 2 && gate->size(1) == D && gate->is_contiguous() && gate_div >= 1 &&
                 (rows == 0 || (rows - 1) / gate_div < gate->size(0)),
             "residual_norm: gate must be contiguous [gate rows, D] of x's type");
  if (stats)
    SB_CHECK(stats->device() == x.device() && stats->scalar_type() == at::kFloat && stats->dim() == 2 &&
                 stats->size(0) == 4 && stats->size(1) == rows && stats->is_contiguous(),
             "residual_norm: stats must be fp32 [4, rows]");
  const int64_t e = x.element_size();
  bool wide = D % 8 == 0 && (rows <= 1 || ((x.stride(0) * e) % 16 == 0 && (branch.stride(0) * e) % 16 == 0));
  for (const torch::Tensor* t : {&x, &branch, &w, &stream, &normed}) wide = wide && bnorm::aligned(*t);
  for (const auto* t : {&b, &post_w, &post_b, &gate}) wide = wide && (!*t || bnorm::aligned(**t));
  SB_CHECK(D <= (wide ? bnorm::MAX_D : bnorm::MAX_D_NARROW), "residual_norm: width ", D, " is above ",
           wide ? bnorm::MAX_D : bnorm::MAX_D_NARROW);
  if (rows == 0) return;
  auto ptr = [](const c10::optional<torch::Tensor>& t) -> const void* { return t ? t->data_ptr() : nullptr; };
  bnorm::Fwd a{};
  a.x = x.data_ptr(); a.branch = branch.data_ptr(); a.w = w.data_ptr();
  a.b = ptr(b); a.post_w = ptr(post_w); a.post_b = ptr(post_b); a.gate = ptr(gate);
  a.ldx = x.stride(0); a.ldb = branch.stride(0); a.gate_div = gate_div;
  a.stream = stream.data_ptr(); a.normed = normed.data_ptr();
  if (stats) {
    float* s = stats->data_ptr<float>();
    a.rstd = s; a.mean = s + rows; a.post_rstd = s + 2 * rows; a.post_mean = s + 3 * rows;
  }
  a.D = int(D);
  a.eps = float(eps); a.post_eps = float(post_eps); a.scale = float(scale);
  a.one_plus = one_plus; a.round_branch = round_branch;
  const at::cuda::CUDAGuard guard(x.device());
  auto st = at::cuda::getCurrentCUDAStream();
  if (type == at::kBFloat16) bnorm::run_fwd<__nv_bfloat16>(a, rows, wide, layer, st);
  else if (type == at::kHalf) bnorm::run_fwd<__half>(a, rows, wide, layer, st);
  else bnorm::run_fwd<float>(a, rows, wide, layer, st);
}

// Whether the backward pass can hold `sums` column sums of width D.
bool residual_norm_bwd_fits(int64_t D, int64_t sums) { return size_t(D) * sums * 4 <= bnorm::MAX_SUMS; }

// Whether rows of width D are held by 16-byte vectors alone, and whether those of t can be read so.
bool residual_norm_needs_vectors(int64_t D) { return D > bnorm::MAX_D_NARROW; }
bool residual_norm_vectors(const torch::Tensor& t) {
  return bnorm::aligned(t) && (t.size(0) <= 1 || (t.stride(0) * t.element_size()) % 16 == 0);
}

// Gradients of residual_norm_fwd.  d_stream / d_normed may be absent (no gradient).  Writes dx, and
// where given dbranch, dw, db, dpost_w, dpost_b ([D] of x's type) and dgate (like gate).  gate_mode:
// 0 none, 1 one gate row, 2 a gate row for gate_div consecutive rows, 3 a gate row for each row.
void residual_norm_bwd(const c10::optional<torch::Tensor>& d_stream, const c10::optional<torch::Tensor>& d_normed,
                       const torch::Tensor& stream, const torch::Tensor& branch, const torch::Tensor& w,
                       const c10::optional<torch::Tensor>& post_w, const c10::optional<torch::Tensor>& post_b,
                       const c10::optional<torch::Tensor>& gate, int64_t gate_div, int64_t gate_mode, double scale,
                       bool layer, bool one_plus, const torch::Tensor& stats, const torch::Tensor& dx,
                       const c10::optional<torch::Tensor>& dbranch, const c10::optional<torch::Tensor>& dw,
                       const c10::optional<torch::Tensor>& db, const c10::optional<torch::Tensor>& dpost_w,
                       const c10::optional<torch::Tensor>& dpost_b, const c10::optional<torch::Tensor>& dgate) {
  const auto type = stream.scalar_type();
  SB_CHECK(stream.is_cuda() && stream.dim() == 2 && stream.is_contiguous(), "residual_norm: stream must be CUDA [rows, D]");
  SB_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "residual_norm: bf16, fp16 or fp32");
  const int64_t rows = stream.size(0), D = stream.size(1);
  auto same = [&](const torch::Tensor& t) { return t.device() == stream.device() && t.scalar_type() == type; };
  auto rowwise = [&](const torch::Tensor& t) { return same(t) && t.sizes() == stream.sizes() && (D == 1 || t.stride(1) == 1); };
  auto vector = [&](const c10::optional<torch::Tensor>& t) { return !t || (same(*t) && t->dim() == 1 && t->size(0) == D && t->is_contiguous()); };
  SB_CHECK((!d_stream || rowwise(*d_stream)) && (!d_normed || rowwise(*d_normed)) && rowwise(branch) && rowwise(dx) &&
               dx.is_contiguous() && (!dbranch || (rowwise(*dbranch) && dbranch->is_contiguous())),
           "residual_norm: gradients must be [rows, D] of the stream's type");
  SB_CHECK(vector(w) && vector(post_w) && vector(post_b) && vector(dw) && vector(db) && vector(dpost_w) && vector(dpost_b),
           "residual_norm: vectors must be contiguous [D]");
  SB_CHECK(stats.device() == stream.device() && stats.scalar_type() == at::kFloat && stats.numel() == 4 * rows && stats.is_contiguous(),
           "residual_norm: stats must be fp32 [4, rows]");
  SB_CHECK((gate_mode == 0) == !gate.has_value() && gate_mode >= 0 && gate_mode <= 3 && gate_div >= 1, "residual_norm: gate mode");
  if (gate)
    SB_CHECK(same(*gate) && gate->dim() == 2 && gate->size(1) == D && gate->is_contiguous() &&
                 (rows == 0 || (rows - 1) / gate_div < gate->size(0)) && (gate_mode != 1 || gate->size(0) == 1) &&
                 (gate_mode != 2 || rows == 0 || gate->size(0) * gate_div == rows) &&
                 (gate_mode != 3 || (gate_div == 1 && gate->size(0) == rows)) &&
                 (!dgate || (same(*dgate) && dgate->sizes() == gate->sizes() && dgate->is_contiguous())),
             "residual_norm: gate");
  SB_CHECK(gate || !dgate, "residual_norm: dgate without a gate");
  SB_CHECK((layer || (!db && !dpost_b)) && (post_w || (!dpost_w && !dpost_b)), "residual_norm: gradient of an absent vector");
  bool wide = D % 8 == 0 && bnorm::aligned(stream) && bnorm::aligned(w) && bnorm::aligned(dx);
  wide = wide && residual_norm_vectors(branch) && (!d_stream || residual_norm_vectors(*d_stream)) &&
         (!d_normed || residual_norm_vectors(*d_normed));
  for (const auto* t : {&post_w, &post_b, &gate, &dbranch, &dgate}) wide = wide && (!*t || bnorm::aligned(**t));
  SB_CHECK(D <= (wide ? bnorm::MAX_D : bnorm::MAX_D_NARROW), "residual_norm: width ", D, " is above ",
           wide ? bnorm::MAX_D : bnorm::MAX_D_NARROW);
  const at::cuda::CUDAGuard guard(stream.device());
  auto st = at::cuda::getCurrentCUDAStream();
  bnorm::Bwd a{};
  void* outs[bnorm::kSums];
  int slots = 0;
  for (int k = 0; k < bnorm::kSums; ++k) a.slot[k] = -1;
  auto want = [&](int k, const c10::optional<torch::Tensor>& t) {
    if (t) {
      a.slot[k] = slots;
      outs[slots++] = t->data_ptr();
    }
  };
  want(bnorm::kW, dw);
  want(bnorm::kB, db);
  want(bnorm::kPostW, dpost_w);
  want(bnorm::kPostB, dpost_b);
  if (gate_mode == 1 || gate_mode == 2) want(bnorm::kGate, dgate);  // last: sequence gates leave earlier
  a.slots = slots;
  const bool seq = gate_mode == 2 && dgate.has_value();
  const int joined = seq ? slots - 1 : slots;
  if (rows == 0) {
    for (const auto* t : {&dw, &db, &dpost_w, &dpost_b, &dgate})
      if (*t) (*t)->zero_();
    return;
  }
  const size_t held = size_t(D) * slots * 4;
  SB_CHECK(held <= bnorm::MAX_SUMS, "residual_norm: ", slots, " column sums of width ", D, " do not fit shared memory");
  // units: as many as run at once, fewer when rows are few (a block's sums are written and read again)
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const bool reg = wide && D / 8 <= bnorm::THREADS;  // the kernel's NV == 1
  a.group_threads = bnorm::threads_for(D, wide);
  // a group's barrier is one of the block's 16, the first of which is the whole block's
  a.groups = reg ? std::min(15, bnorm::GROUP_THREADS / a.group_threads) : 1;
  const size_t smem = reg ? size_t(a.groups) * a.group_threads * 8 * 4 : held;
  const int64_t resident = reg ? 1 : std::max<int64_t>(1, std::min<int64_t>(1024 / a.group_threads, (220 * 1024) / int64_t(smem + 2048)));
  const int64_t least = slots && !reg ? 8 : 1;
  a.rows_per_unit = std::max<int64_t>((rows + sms * resident * a.groups - 1) / (sms * resident * a.groups), std::min<int64_t>(least, (rows + sms - 1) / sms));
  const int64_t units = (rows + a.rows_per_unit - 1) / a.rows_per_unit, blocks = (units + a.groups - 1) / a.groups;
  torch::Tensor partial, edge;
  const auto f32 = stream.options().dtype(at::kFloat);
  if (joined) {
    partial = torch::empty({blocks * joined * D}, f32);
    a.partial = partial.data_ptr<float>();
  }
  if (seq) {
    edge = torch::empty({units * 2 * D}, f32);
    a.edge = edge.data_ptr<float>();
  }
  auto ptr = [](const c10::optional<torch::Tensor>& t) -> void* { return t ? t->data_ptr() : nullptr; };
  a.d_stream = ptr(d_stream); a.d_normed = ptr(d_normed);
  a.ld_ds = d_stream ? d_stream->stride(0) : 0; a.ld_dn = d_normed ? d_normed->stride(0) : 0;
  a.stream = stream.data_ptr(); a.branch = branch.data_ptr(); a.w = w.data_ptr();
  a.post_w = ptr(post_w); a.post_b = ptr(post_b); a.gate = ptr(gate);
  a.ldb = branch.stride(0); a.gate_div = gate_div;
  const float* s = stats.data_ptr<float>();
  a.rstd = s; a.mean = s + rows; a.post_rstd = s + 2 * rows; a.post_mean = s + 3 * rows;
  a.dx = dx.data_ptr(); a.dbranch = ptr(dbranch);
  a.dgate = gate_mode >= 2 ? ptr(dgate) : nullptr;
  a.rows = rows; a.D = int(D);
  a.scale = float(scale); a.one_plus = one_plus; a.gate_mode = int(gate_mode);
  auto finish = [&](auto zero) {
    using T = decltype(zero);
    bnorm::run_bwd<T>(a, unsigned(blocks), wide, layer, smem, st);
    if (joined) {
      bnorm::Join j{};
      j.partial = a.partial;
      for (int k = 0; k < joined; ++k) j.out[k] = outs[k];
      j.blocks = int(blocks); j.slots = joined; j.D = int(D);
      bnorm::join_kernel<T><<<dim3(unsigned((D + 31) / 32), unsigned(joined)), dim3(32, bnorm::JOIN_ROWS), 0, st>>>(j);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
    if (seq) {
      bnorm::edge_kernel<T><<<dim3(unsigned(rows / gate_div), unsigned((D + 255) / 256)), dim3(256), 0, st>>>(
          a.edge, static_cast<T*>(dgate->data_ptr()), a.rows_per_unit, gate_div, int(D));
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
  };
  if (type == at::kBFloat16) finish(__nv_bfloat16{});
  else if (type == at::kHalf) finish(__half{});
  else finish(float{});
}

}  // namespace sb
