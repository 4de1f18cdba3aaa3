// Rotary positions of q and k in one launch.
//
// Pair i of a head (i < rot / 2) at position p is turned by the angle p * freq[i]:
//     a' = f (a cos - b sin),   b' = f (b cos + a sin)
// with f the factor that a stretched context puts on cos and sin.  (a, b) are channels
// (i, rot/2 + i) in the half layout and (2i, 2i + 1) in the interleaved one; channels from `rot`
// on pass through.  The gradient is the transposed rotation (sin negated).
//
// Angles are formed in 64 bits: p * freq / 2 pi, of which only the fraction of a turn goes on to
// the 32-bit sine and cosine, so that a position of 10^6 is as exact as a small one (in 32 bits it
// would be off by up to 0.06 rad).  There is no table and no largest position.
//
// Every value is read and written once, so memory bounds it.  A thread has one place in the heads of
// a token, a chunk of VEC pairs (the two vectors of VEC elements that hold them in either layout, 16
// bytes each where sizes and alignment allow it), and turns it in several heads: it forms its
// angles once, in registers, behind the loads of its first heads.  Angles shared by a block through
// shared memory are formed once for all heads, but every load waits at a barrier for them: 8192
// tokens of 40 heads of 128 took 37 us so, 43 with the first loads before the barrier, and take 29.5
// this way (5.7 TB/s).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include <algorithm>

#include "block_ops.h"
#include "check.h"
#include "vec.cuh"

namespace sb {
namespace rotary {

constexpr int THREADS = 128;
constexpr int HEADS = 4;  // heads of a thread at most, whose loads are under way at once

struct Side {  // q or k
  const void* in;
  void* out;
  int64_t in_b, in_s, in_h;  // strides in elements; the last dimension is contiguous
  int64_t out_b, out_s, out_h;
  int heads;
};

struct Args {
  Side q, k;
  const void* pos;  // int64 or int32 [B, S] with strides, or nullptr: pos0 + s
  int64_t pos_b, pos_s, pos0;
  int pos32;
  const double* freq;  // [rot / 2]
  float factor;
  int inverse;
  int64_t tokens, threads;  // threads: tokens * lanes * chunks of a head
  int S, d, rot;
  int chunks;  // of a head: those that turn, then those that pass through (two vectors each)
  int lanes;   // threads that share a chunk's heads: lane l has heads l, l + lanes, ..., HEADS at most
};

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, 6) kernel(const __grid_constant__ Args a) {
  const int64_t at = int64_t(blockIdx.x) * THREADS + threadIdx.x;
  if (at >= a.threads) return;
  int64_t tok, b, s;
  int j, lane;
  if (a.threads < (int64_t(1) << 31)) {  // 32-bit divisions are a third of the others
    const uint32_t r = uint32_t(at) / uint32_t(a.chunks);
    j = int(uint32_t(at) - r * uint32_t(a.chunks));
    const uint32_t t = r / uint32_t(a.lanes);
    lane = int(r - t * uint32_t(a.lanes));
    const uint32_t bb = t / uint32_t(a.S);
    tok = t, b = bb, s = t - bb * uint32_t(a.S);
  } else {
    const int64_t r = at / a.chunks;
    j = int(at - r * a.chunks);
    tok = r / a.lanes;
    lane = int(r - tok * a.lanes);
    b = tok / a.S, s = tok - b * a.S;
  }
  const int half = a.rot / 2, turned = half / VEC;
  const int heads = a.q.heads + a.k.heads;
  // the chunk's two vectors within a head; a chunk that passes through may have but one
  const bool turns = j < turned;
  const int g = 2 * (j - turned);
  const int i0 = !turns ? a.rot + VEC * g : INTERLEAVED ? 2 * VEC * j : VEC * j;
  const int i1 = !turns || INTERLEAVED ? i0 + VEC : half + VEC * j;
  const bool two = turns || i1 < a.d;
  const T* qi = static_cast<const T*>(a.q.in) + b * a.q.in_b + s * a.q.in_s;
  const T* ki = static_cast<const T*>(a.k.in) + b * a.k.in_b + s * a.k.in_s;
  T* qo = static_cast<T*>(a.q.out) + b * a.q.out_b + s * a.q.out_s;
  T* ko = static_cast<T*>(a.k.out) + b * a.k.out_b + s * a.k.out_s;
  vec::Pack<T, VEC> u[HEADS], v[HEADS];
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const int h = lane + n * a.lanes;
    if (h < heads) {
      const T* p = h < a.q.heads ? qi + h * a.q.in_h : ki + (h - a.q.heads) * a.k.in_h;
      u[n].load(p + i0);
      if (two) v[n].load(p + i1);
    }
  }
  float c[VEC], sn[VEC];
  if (turns) {
    int64_t p = a.pos0 + s;
    if (a.pos) {
      const int64_t e = b * a.pos_b + s * a.pos_s;
      p = a.pos32 ? int64_t(static_cast<const int*>(a.pos)[e]) : static_cast<const int64_t*>(a.pos)[e];
    }
#pragma unroll
    for (int m = 0; m < VEC; ++m) {
      const double turn = double(p) * a.freq[VEC * j + m] * 0.15915494309189533577;  // 1 / (2 pi)
      sincospif(2.f * float(turn - rint(turn)), &sn[m], &c[m]);
      c[m] *= a.factor;
      sn[m] *= a.inverse ? -a.factor : a.factor;
    }
  }
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const int h = lane + n * a.lanes;
    if (h >= heads) break;
    if (turns) {
      float x[VEC], y[VEC];
      u[n].unpack(x);
      v[n].unpack(y);
      if (INTERLEAVED) {
        // the 2 VEC channels of (u, v) are VEC neighbouring pairs
        auto at2 = [&](int m) -> float& { return m < VEC ? x[m < VEC ? m : 0] : y[m < VEC ? 0 : m - VEC]; };
#pragma unroll
        for (int m = 0; m < VEC; ++m) {
          float &A = at2(2 * m), &B = at2(2 * m + 1);
          const float na = A * c[m] - B * sn[m];
          B = B * c[m] + A * sn[m];
          A = na;
        }
      } else {
#pragma unroll
        for (int m = 0; m < VEC; ++m) {
          const float na = x[m] * c[m] - y[m] * sn[m];
          y[m] = y[m] * c[m] + x[m] * sn[m];
          x[m] = na;
        }
      }
      u[n].pack(x);
      v[n].pack(y);
    }
    T* o = h < a.q.heads ? qo + h * a.q.out_h : ko + (h - a.q.heads) * a.k.out_h;
    u[n].store(o + i0);
    if (two) v[n].store(o + i1);
  }
}

// Whether every access of VEC elements of t is aligned to itself (16 bytes at most).
static bool fits(const torch::Tensor& t, int64_t vec) {
  const int64_t bytes = std::min<int64_t>(16, vec * t.element_size());
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) * t.element_size()) % bytes) return false;
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0;
}

template <class T, int VEC>
static void launch(const Args& a, bool interleaved, cudaStream_t stream) {
  const int64_t blocks = (a.threads + THREADS - 1) / THREADS;
  SB_CHECK(blocks < (1ll << 31), "rotary: too many tokens");
  if (interleaved) kernel<T, VEC, true><<<dim3(unsigned(blocks)), THREADS, 0, stream>>>(a);
  else kernel<T, VEC, false><<<dim3(unsigned(blocks)), THREADS, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <class T>
static void launch_vec(const Args& a, int vec, bool interleaved, cudaStream_t stream) {
  constexpr int kMost = 16 / int(sizeof(T));
  if (vec >= kMost) launch<T, kMost>(a, interleaved, stream);
  else if (vec >= 4) launch<T, (kMost < 4 ? kMost : 4)>(a, interleaved, stream);
  else if (vec >= 2) launch<T, 2>(a, interleaved, stream);
  else launch<T, 1>(a, interleaved, stream);
}

static Side side(const torch::Tensor& in, const torch::Tensor& out) {
  Side s{};
  s.in = in.data_ptr();
  s.out = out.data_ptr();
  s.in_b = in.stride(0); s.in_s = in.stride(1); s.in_h = in.stride(2);
  s.out_b = out.stride(0); s.out_s = out.stride(1); s.out_h = out.stride(2);
  s.heads = int(in.size(2));
  return s;
}

}  // namespace rotary

// Turns q [B, S, H, d] and, if given, k [B, S, KV, d] (bf16, fp16 or fp32, last dim contiguous) into
// q_out / k_out of the same sizes, which may be the inputs themselves.  freq: fp64 [rot / 2].
// positions: int64 or int32 [B, S] (strides may be 0), or none: pos0, pos0 + 1, ...
void rotary_fwd(const torch::Tensor& q, const c10::optional<torch::Tensor>& k, const torch::Tensor& freq,
                const c10::optional<torch::Tensor>& positions, int64_t pos0, bool interleaved, bool inverse,
                double factor, const torch::Tensor& q_out, const c10::optional<torch::Tensor>& k_out) {
  SB_CHECK(q.is_cuda() && q.dim() == 4 && (q.size(3) <= 1 || q.stride(3) == 1), "rotary: q must be CUDA [B, S, H, d], last dim contiguous");
  const auto type = q.scalar_type();
  SB_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "rotary: bf16, fp16 or fp32");
  const int64_t B = q.size(0), S = q.size(1), d = q.size(3), rot = 2 * freq.numel();
  SB_CHECK(freq.device() == q.device() && freq.scalar_type() == at::kDouble && freq.dim() == 1 && freq.is_contiguous(),
           "rotary: freq must be contiguous fp64 [rot / 2] on q's device");
  SB_CHECK(rot >= 2 && rot <= d, "rotary: 2 * freq.numel() = ", rot, " channels turn, a head has ", d);
  SB_CHECK(S < (1ll << 31) && d <= 8192 && q.size(2) <= 65536, "rotary: size");
  auto check = [&](const torch::Tensor& t, int64_t heads, const char* name) {
    SB_CHECK(t.device() == q.device() && t.scalar_type() == type && t.dim() == 4 && t.size(0) == B && t.size(1) == S &&
                 t.size(2) == heads && t.size(3) == d && (d <= 1 || t.stride(3) == 1),
             "rotary: ", name, " must match q in device, type, B, S and d, last dim contiguous");
  };
  check(q_out, q.size(2), "q_out");
  rotary::Args a{};
  a.q = rotary::side(q, q_out);
  if (k) {
    SB_CHECK(k_out.has_value() && k->dim() == 4 && k->size(2) <= 65536, "rotary: k needs k_out");
    check(*k, k->size(2), "k");
    check(*k_out, k->size(2), "k_out");
    a.k = rotary::side(*k, *k_out);
  }
  if (positions) {
    const auto pt = positions->scalar_type();
    SB_CHECK(positions->device() == q.device() && (pt == at::kLong || pt == at::kInt) && positions->dim() == 2 &&
                 positions->size(0) == B && positions->size(1) == S,
             "rotary: positions must be int64 or int32 [B, S] on q's device");
    a.pos = positions->data_ptr();
    a.pos_b = positions->stride(0);
    a.pos_s = positions->stride(1);
    a.pos32 = pt == at::kInt;
  }
  a.pos0 = pos0;
  a.freq = freq.data_ptr<double>();
  a.factor = float(factor);
  a.inverse = inverse ? 1 : 0;
  a.tokens = B * S;
  a.S = int(S);
  a.d = int(d);
  a.rot = int(rot);
  // out of place the channels from rot on are written too
  const bool copy = q.data_ptr() != q_out.data_ptr() || (k && k->data_ptr() != k_out->data_ptr());
  const int heads = a.q.heads + a.k.heads;
  if (a.tokens == 0 || heads == 0) return;
  // the widest vector that every part of a head and every stride is a multiple of
  int vec = 16 / int(q.element_size());
  while (vec > 1 && ((rot / 2) % vec || d % vec || !rotary::fits(q, vec) || !rotary::fits(q_out, vec) ||
                     (k && (!rotary::fits(*k, vec) || !rotary::fits(*k_out, vec)))))
    vec /= 2;
  a.chunks = int((rot / 2) / vec + (copy ? ((d - rot) / vec + 1) / 2 : 0));
  // a thread turns its chunk in HEADS heads, in fewer where that leaves SMs short of threads
  const int64_t wave = 148 * 1024;
  int64_t lanes = (heads + rotary::HEADS - 1) / rotary::HEADS;
  while (lanes < heads && a.tokens * a.chunks * lanes < wave) lanes = std::min<int64_t>(heads, 2 * lanes);
  a.lanes = int(lanes);
  a.threads = a.tokens * a.chunks * lanes;
  const at::cuda::CUDAGuard guard(q.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  if (type == at::kBFloat16) rotary::launch_vec<__nv_bfloat16>(a, vec, interleaved, stream);
  else if (type == at::kHalf) rotary::launch_vec<__half>(a, vec, interleaved, stream);
  else rotary::launch_vec<float>(a, vec, interleaved, stream);
}

}  // namespace sb
