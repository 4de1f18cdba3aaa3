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
// would be off by up to 0.06 rad).  They cost rot / 2 products a token for all its heads, kept in
// shared memory; there is no table and no largest position.
//
// Every value is read and written once, so memory bounds it.  A block turns `tokens` tokens (one,
// unless heads are few or narrow); a thread handles chunks of VEC pairs: the two vectors of VEC
// elements that hold them in either layout, 16 bytes each where sizes and alignment allow it.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include <algorithm>

#include "block_ops.h"
#include "check.h"
#include "vec.cuh"

namespace sb {
namespace rotary {

constexpr int MAX_THREADS = 512;

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
  int64_t tokens;
  int S, d, rot;
  int per_block;  // tokens of a block
  int copy;       // 1: the channels from rot on are written too (out of place)
};

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(MAX_THREADS) kernel(const __grid_constant__ Args a) {
  extern __shared__ float2 cs[];  // [per_block][rot / 2]: cos and sin of each pair
  const int half = a.rot / 2;
  const int64_t t0 = int64_t(blockIdx.x) * a.per_block;
  const int nt = int(min(int64_t(a.per_block), a.tokens - t0));
  for (int e = threadIdx.x; e < nt * half; e += blockDim.x) {
    const int t = e / half, i = e - t * half;
    const int64_t tok = t0 + t;
    const int64_t b = tok / a.S, s = tok - b * a.S;
    int64_t p = a.pos0 + s;
    if (a.pos) {
      const int64_t at = b * a.pos_b + s * a.pos_s;
      p = a.pos32 ? int64_t(static_cast<const int*>(a.pos)[at]) : static_cast<const int64_t*>(a.pos)[at];
    }
    const double turns = double(p) * a.freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
    float sn, c;
    sincospif(2.f * float(turns - rint(turns)), &sn, &c);
    cs[e] = make_float2(c * a.factor, a.inverse ? -sn * a.factor : sn * a.factor);
  }
  __syncthreads();

  const int turned = half / VEC;                                // chunks of a head that turn
  const int rest = a.copy ? (a.d - a.rot) / VEC : 0;            // vectors of a head that pass through
  const int per_head = turned + (rest + 1) / 2;
  const int heads = a.q.heads + a.k.heads;
  const int per_token = heads * per_head;
  for (int e = threadIdx.x; e < nt * per_token; e += blockDim.x) {
    const int t = e / per_token;
    int r = e - t * per_token;
    int h = r / per_head;
    const int j = r - h * per_head;
    const int64_t tok = t0 + t;
    const int64_t b = tok / a.S, s = tok - b * a.S;
    const bool isq = h < a.q.heads;
    const Side& w = isq ? a.q : a.k;
    if (!isq) h -= a.q.heads;
    const T* in = static_cast<const T*>(w.in) + b * w.in_b + s * w.in_s + h * w.in_h;
    T* out = static_cast<T*>(w.out) + b * w.out_b + s * w.out_s + h * w.out_h;
    vec::Pack<T, VEC> u, v;
    if (j < turned) {
      const int iu = INTERLEAVED ? 2 * VEC * j : VEC * j;
      const int iv = INTERLEAVED ? iu + VEC : half + VEC * j;
      u.load(in + iu);
      v.load(in + iv);
      const float2* c = cs + t * half + VEC * j;
      if (INTERLEAVED) {
        // the 2 VEC channels of (u, v) are VEC neighbouring pairs
        vec::Pack<T, VEC> x, y;
#pragma unroll
        for (int m = 0; m < VEC; ++m) {
          const float A = 2 * m < VEC ? u.get(2 * m < VEC ? 2 * m : 0) : v.get(2 * m < VEC ? 0 : 2 * m - VEC);
          const float B = 2 * m + 1 < VEC ? u.get(2 * m + 1 < VEC ? 2 * m + 1 : 0)
                                          : v.get(2 * m + 1 < VEC ? 0 : 2 * m + 1 - VEC);
          const float na = A * c[m].x - B * c[m].y, nb = B * c[m].x + A * c[m].y;
          if (2 * m < VEC) x.set(2 * m < VEC ? 2 * m : 0, na);
          else y.set(2 * m < VEC ? 0 : 2 * m - VEC, na);
          if (2 * m + 1 < VEC) x.set(2 * m + 1 < VEC ? 2 * m + 1 : 0, nb);
          else y.set(2 * m + 1 < VEC ? 0 : 2 * m + 1 - VEC, nb);
        }
        x.store(out + iu);
        y.store(out + iv);
      } else {
#pragma unroll
        for (int m = 0; m < VEC; ++m) {
          const float A = u.get(m), B = v.get(m);
          u.set(m, A * c[m].x - B * c[m].y);
          v.set(m, B * c[m].x + A * c[m].y);
        }
        u.store(out + iu);
        v.store(out + iv);
      }
    } else {
      const int g = 2 * (j - turned);
      const int at = a.rot + VEC * g;
      u.load(in + at);
      if (g + 1 < rest) v.load(in + at + VEC);
      u.store(out + at);
      if (g + 1 < rest) v.store(out + at + VEC);
    }
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
  const int half = a.rot / 2;
  const int64_t items = int64_t(a.q.heads + a.k.heads) * (half / VEC + ((a.copy ? (a.d - a.rot) / VEC : 0) + 1) / 2);
  const int threads = int(std::min<int64_t>(MAX_THREADS, std::max<int64_t>(64, (std::max<int64_t>(items * a.per_block, half) + 31) / 32 * 32)));
  const int64_t blocks = (a.tokens + a.per_block - 1) / a.per_block;
  SB_CHECK(blocks < (1ll << 31), "rotary: too many tokens");
  const size_t smem = size_t(a.per_block) * half * sizeof(float2);
  if (interleaved)
    kernel<T, VEC, true><<<dim3(unsigned(blocks)), dim3(threads), smem, stream>>>(a);
  else
    kernel<T, VEC, false><<<dim3(unsigned(blocks)), dim3(threads), smem, stream>>>(a);
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
  a.copy = (q.data_ptr() != q_out.data_ptr() || (k && k->data_ptr() != k_out->data_ptr())) ? 1 : 0;
  const int heads = a.q.heads + a.k.heads;
  if (a.tokens == 0 || heads == 0) return;
  // the widest vector that every part of a head and every stride is a multiple of
  int vec = 16 / int(q.element_size());
  while (vec > 1 && ((rot / 2) % vec || d % vec || !rotary::fits(q, vec) || !rotary::fits(q_out, vec) ||
                     (k && (!rotary::fits(*k, vec) || !rotary::fits(*k_out, vec)))))
    vec /= 2;
  // tokens of a block: one while a token fills it, more when its chunks are fewer than 256, as long
  // as every SM still has several blocks and the angles fit 32 KB
  const int64_t items = int64_t(heads) * ((rot / 2) / vec + ((d - rot) / vec + 1) / 2);
  int64_t per = std::max<int64_t>(1, 256 / items);
  per = std::min<int64_t>(per, std::max<int64_t>(1, a.tokens / (148 * 4)));
  per = std::min<int64_t>(per, std::max<int64_t>(1, 32768 / (rot / 2 * int64_t(sizeof(float2)))));
  a.per_block = int(per);
  const at::cuda::CUDAGuard guard(q.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  if (type == at::kBFloat16) rotary::launch_vec<__nv_bfloat16>(a, vec, interleaved, stream);
  else if (type == at::kHalf) rotary::launch_vec<__half>(a, vec, interleaved, stream);
  else rotary::launch_vec<float>(a, vec, interleaved, stream);
}

}  // namespace sb
