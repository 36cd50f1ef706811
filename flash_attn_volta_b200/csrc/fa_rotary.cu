// Rotary positions: y1 = M (x1 cos a - x2 sin a), y2 = M (x2 cos a + x1 sin a)
// for each pair (x1, x2) of the first R dims of a head, a = pos * inv_freq[i];
// the dims behind R are copied.  Pairs are (i, i + R/2) ("half") or
// (2i, 2i + 1) ("interleaved").  The map is M times a rotation, so its
// transpose, the gradient, is the same kernel with -a (`inverse`).
//
// Bound by HBM: each element is read once and written once, 6 flops a pair.
// The angles depend on the token alone, so a CTA takes whole tokens (all heads
// of q and of k in one launch), makes the R/2 cosines and sines of each once in
// shared memory and uses them for every head: with 20 heads the 64-bit angle
// costs one pair in 20.  A thread loads its vectors before it computes angles,
// so the loads' latency covers them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "fa_kernels.h"
#include "fa_rotary.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 2;          // vectors (pairs of vectors) in flight per thread
constexpr int kMaxAngles = 4096;   // cosines and sines of a CTA: 32 KB

struct RotaryPart {
  const void* in;
  void* out;
  long long sb, ss, sh;  // input strides in elements
  int heads;
};

struct RotaryParams {
  RotaryPart q, k;
  const double* inv_freq;
  const void* positions;  // int32 or int64 (pos64), or null
  long long pos_sb;       // its batch stride
  long long first;        // position of token 0 without `positions`
  long long tokens;       // batch * seqlen
  int S, D, half, per_cta, pos64;
  float magnitude, sign;
};

// One thread's share of a head: a vector of VEC first halves and the VEC
// second halves of the same pairs (half), or VEC elements = VEC/2 pairs
// (interleaved), or VEC elements behind R.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) fa_rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 cs[];
  griddep_wait();
  griddep_launch_dependents();
  using V = Pack16<VEC>;
  const unsigned half = p.half, D = p.D;
  const unsigned turning = INTER ? 2 * half / VEC : half / VEC;  // items of a head that rotate
  const unsigned per_head = turning + (D - 2 * half) / VEC;
  const unsigned heads = p.q.heads + p.k.heads, per_token = heads * per_head;
  const long long tok0 = (long long)blockIdx.x * p.per_cta;
  const int ntok = (int)min((long long)p.per_cta, p.tokens - tok0);
  const unsigned total = ntok * per_token;

  for (unsigned base = 0; base < total || base == 0; base += kThreads * kItems) {
    V a[kItems], b[kItems];
    T* dst[kItems];
    unsigned where[kItems];  // angle index; ~0u: copied
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const unsigned it = base + u * kThreads + threadIdx.x;
      dst[u] = nullptr;
      if (it >= total) continue;
      const unsigned tok = it / per_token, rem = it % per_token;
      unsigned h = rem / per_head;
      const unsigned j = rem % per_head;
      const bool is_k = h >= (unsigned)p.q.heads;
      const RotaryPart& part = is_k ? p.k : p.q;
      if (is_k) h -= p.q.heads;
      const long long t = tok0 + tok, bt = t / p.S, s = t % p.S;
      const T* src = static_cast<const T*>(part.in) + bt * part.sb + s * part.ss + h * part.sh;
      T* out = static_cast<T*>(part.out) + (t * part.heads + h) * (long long)D;
      const bool turns = j < turning;
      const unsigned e = turns ? j * VEC : 2 * half + (j - turning) * VEC;
      a[u] = *reinterpret_cast<const V*>(src + e);
      if (!INTER && turns) b[u] = *reinterpret_cast<const V*>(src + e + half);
      dst[u] = out + e;
      where[u] = turns ? tok * half + (INTER ? e / 2 : e) : ~0u;
    }
    if (base == 0) {
      for (unsigned i = threadIdx.x; i < ntok * half; i += kThreads) {
        const long long t = tok0 + i / half, bt = t / p.S, s = t % p.S;
        const long long at = bt * p.pos_sb + s;
        const long long pos = p.positions == nullptr ? p.first + s
                              : p.pos64 ? static_cast<const long long*>(p.positions)[at]
                                        : static_cast<const int*>(p.positions)[at];
        float2 c = rotary_cos_sin((double)pos, p.inv_freq[i % half], p.magnitude);
        c.y *= p.sign;
        cs[i] = c;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      if (dst[u] == nullptr) continue;
      if (where[u] != ~0u) {
        const float2* w = cs + where[u];
        if (INTER) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float x = Elem<T>::value(a[u].v[2 * i]), y = Elem<T>::value(a[u].v[2 * i + 1]);
            a[u].v[2 * i] = Elem<T>::bits(x * w[i].x - y * w[i].y);
            a[u].v[2 * i + 1] = Elem<T>::bits(y * w[i].x + x * w[i].y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float x = Elem<T>::value(a[u].v[i]), y = Elem<T>::value(b[u].v[i]);
            a[u].v[i] = Elem<T>::bits(x * w[i].x - y * w[i].y);
            b[u].v[i] = Elem<T>::bits(y * w[i].x + x * w[i].y);
          }
          *reinterpret_cast<V*>(dst[u] + half) = b[u];
        }
      }
      *reinterpret_cast<V*>(dst[u]) = a[u];
    }
  }
}

template <typename T, int VEC>
int launch(const RotaryParams& p, bool interleaved, unsigned grid, size_t smem, cudaStream_t st) {
  const cudaError_t e =
      interleaved
          ? launch_pdl(fa_rotary_kernel<T, (VEC > 1 ? VEC : 2), true>, dim3(grid), dim3(kThreads),
                       smem, st, p)
          : launch_pdl(fa_rotary_kernel<T, VEC, false>, dim3(grid), dim3(kThreads), smem, st, p);
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

template <typename T>
int launch_vec(const RotaryParams& p, int vec, bool interleaved, unsigned grid, size_t smem,
               cudaStream_t st) {
  switch (vec) {
    case 8: return launch<T, 8>(p, interleaved, grid, smem, st);
    case 4: return launch<T, 4>(p, interleaved, grid, smem, st);
    case 2: return launch<T, 2>(p, interleaved, grid, smem, st);
    default: return launch<T, 1>(p, interleaved, grid, smem, st);
  }
}

// The widest vector (in elements) that every address of a part is a multiple of.
int part_vec(const fa_sm100_heads& x) {
  const unsigned long long m = (reinterpret_cast<uintptr_t>(x.in) / 2) |
                               (reinterpret_cast<uintptr_t>(x.out) / 2) |
                               (unsigned long long)x.stride_batch |
                               (unsigned long long)x.stride_seq | (unsigned long long)x.stride_head;
  return (m & 1) ? 1 : (m & 2) ? 2 : (m & 4) ? 4 : 8;
}

bool bad_part(const fa_sm100_heads& x) {
  return !x.in || !x.out || x.heads < 1 ||
         ((reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) & 1u);
}

}  // namespace
}  // namespace fa_sm100

extern "C" int fa_sm100_rotary(const fa_sm100_heads* q, const fa_sm100_heads* k,
                               const double* inv_freq, int rotary_dim, int interleaved,
                               float magnitude, int inverse, const void* positions,
                               int positions_64, long long positions_stride, long long first,
                               int batch, int seqlen, int head_dim, int dtype, void* stream) {
  using namespace fa_sm100;
  if (!q || !inv_freq || batch < 1 || seqlen < 1) return FA_ERR_ARG;
  if (head_dim < 2 || head_dim % 2 || head_dim > 65536) return FA_ERR_ARG;
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim || rotary_dim > 2 * kMaxAngles)
    return FA_ERR_ARG;
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return FA_ERR_ARG;
  if (bad_part(*q) || (k && bad_part(*k))) return FA_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(inv_freq) & 7u) return FA_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(positions) & (positions_64 ? 7u : 3u)) return FA_ERR_ARG;
  if (((long long)q->heads + (k ? k->heads : 0)) * head_dim > (1 << 26)) return FA_ERR_ARG;
  RotaryParams p = {};
  p.q = {q->in, q->out, q->stride_batch, q->stride_seq, q->stride_head, q->heads};
  if (k) p.k = {k->in, k->out, k->stride_batch, k->stride_seq, k->stride_head, k->heads};
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.pos_sb = positions_stride;
  p.pos64 = positions_64;
  p.first = first;
  p.tokens = (long long)batch * seqlen;
  p.S = seqlen;
  p.D = head_dim;
  p.half = rotary_dim / 2;
  p.magnitude = magnitude;
  p.sign = inverse ? -1.f : 1.f;
  int vec = part_vec(*q);
  if (k && part_vec(*k) < vec) vec = part_vec(*k);
  // a vector may not cross from the rotated dims into the others
  const int unit = interleaved ? rotary_dim : rotary_dim / 2;
  while (vec > 1 && (unit % vec || head_dim % vec || rotary_dim % vec)) vec /= 2;
  if (interleaved && vec == 1) return FA_ERR_ARG;  // a pair has to be 4-byte aligned
  const int per_head = (interleaved ? head_dim : head_dim - p.half) / vec;
  const long long per_token = (long long)(p.q.heads + p.k.heads) * per_head;
  // whole tokens until each thread has kItems vectors: 2 measured against 1 and 4 at
  // 8 x 2048 tokens of 16 + 16 heads of 128 (see the timing below)
  long long per_cta = (long long)kThreads * kItems / per_token;
  if (per_cta > kMaxAngles / p.half) per_cta = kMaxAngles / p.half;
  if (per_cta < 1) per_cta = 1;
  p.per_cta = (int)per_cta;
  const long long grid = (p.tokens + per_cta - 1) / per_cta;
  if (grid > 2147483647LL) return FA_ERR_ARG;
  const size_t smem = (size_t)per_cta * p.half * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FA_DTYPE_BF16
             ? launch_vec<__nv_bfloat16>(p, vec, interleaved != 0, (unsigned)grid, smem, st)
             : launch_vec<__half>(p, vec, interleaved != 0, (unsigned)grid, smem, st);
}
