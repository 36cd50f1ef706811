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
  int S, D, half, per_cta, pos64;  // per_cta: tokens of a CTA, all of one sequence
  int per_seq, per_head, width;    // CTAs of a sequence, items of a head, items of a row of threads
  float magnitude, sign;
};

// One thread's share of a head (an item): a vector of VEC first halves and the
// VEC second halves of the same pairs (half), or VEC elements = VEC/2 pairs
// (interleaved), or VEC elements behind R.  The threads stand as `rows` rows of
// `width` items; a row is one head of one token, and each thread steps down the
// rows with additions alone.  A vector's i-th cosine and sine are `turning`
// apart in shared memory, so the lanes of a row read neighbouring words.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads, 4) fa_rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 cs[];
  griddep_wait();
  griddep_launch_dependents();
  using V = Pack16<VEC>;
  constexpr int PAIRS = INTER ? VEC / 2 : VEC;
  const int half = p.half, turning = half / PAIRS;  // items of a head that rotate
  const int heads = p.q.heads + p.k.heads;
  const int b = blockIdx.x / p.per_seq, s0 = (blockIdx.x - b * p.per_seq) * p.per_cta;
  const int ntok = min(p.per_cta, p.S - s0);
  const int row = threadIdx.x / p.width, col = threadIdx.x - row * p.width;
  const int step = kThreads / p.width, step_tok = step / heads, step_h = step - step_tok * heads;
  int tok = row < step ? row / heads : ntok, h = row - row / heads * heads;

  auto fill = [&]() {
    for (int i = threadIdx.x; i < ntok * half; i += kThreads) {
      const int at = i / half, f = i - at * half;
      const long long s = s0 + at, where = b * p.pos_sb + s;
      const long long pos = p.positions == nullptr ? p.first + s
                            : p.pos64 ? static_cast<const long long*>(p.positions)[where]
                                      : static_cast<const int*>(p.positions)[where];
      float2 c = rotary_cos_sin((double)pos, p.inv_freq[f], p.magnitude);
      c.y *= p.sign;
      cs[at * half + f % PAIRS * turning + f / PAIRS] = c;
    }
    __syncthreads();
  };
  bool filled = false;
  while (tok < ntok || !filled) {
    for (int j = col; j < p.per_head || !filled; j += p.width) {
      V a[kItems], o[kItems];
      T* dst[kItems];
      const float2* w[kItems];  // null: copied
      const bool turns = j < turning;
      const int e = turns ? j * VEC : 2 * half + (j - turning) * VEC;
      int t = tok, hh = h;
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        dst[u] = nullptr;
        if (t < ntok && j < p.per_head) {
          const bool is_k = hh >= p.q.heads;
          const RotaryPart& part = is_k ? p.k : p.q;
          const int hp = is_k ? hh - p.q.heads : hh;
          const T* src = static_cast<const T*>(part.in) + b * part.sb + (s0 + t) * part.ss + hp * part.sh + e;
          dst[u] = static_cast<T*>(part.out) + (((long long)b * p.S + s0 + t) * part.heads + hp) * p.D + e;
          w[u] = turns ? cs + t * half + j : nullptr;
          a[u] = *reinterpret_cast<const V*>(src);
          if (!INTER && turns) o[u] = *reinterpret_cast<const V*>(src + half);
        }
        t += step_tok;
        hh += step_h;
        if (hh >= heads) {
          hh -= heads;
          ++t;
        }
      }
      if (!filled) {
        filled = true;
        fill();
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        if (dst[u] == nullptr) continue;
        if (w[u] != nullptr) {
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            const float2 c = w[u][i * turning];
            uint16_t& lo = INTER ? a[u].v[2 * i] : a[u].v[i];
            uint16_t& hi = INTER ? a[u].v[2 * i + (VEC > 1)] : o[u].v[i];
            const float x = Elem<T>::value(lo), y = Elem<T>::value(hi);
            lo = Elem<T>::bits(x * c.x - y * c.y);
            hi = Elem<T>::bits(y * c.x + x * c.y);
          }
          if (!INTER) *reinterpret_cast<V*>(dst[u] + half) = o[u];
        }
        *reinterpret_cast<V*>(dst[u]) = a[u];
      }
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      tok += step_tok;
      h += step_h;
      if (h >= heads) {
        h -= heads;
        ++tok;
      }
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
  p.per_head = (interleaved ? head_dim : head_dim - p.half) / vec;
  p.width = p.per_head < kThreads ? p.per_head : kThreads;
  const long long per_token = (long long)(p.q.heads + p.k.heads) * p.per_head;
  // whole tokens until each thread has two rounds of kItems vectors
  long long per_cta = 2LL * kThreads * kItems / per_token;
  if (per_cta > kMaxAngles / p.half) per_cta = kMaxAngles / p.half;
  if (per_cta > seqlen) per_cta = seqlen;
  if (per_cta < 1) per_cta = 1;
  p.per_cta = (int)per_cta;
  p.per_seq = (int)((seqlen + per_cta - 1) / per_cta);
  const long long grid = (long long)p.per_seq * batch;
  if (grid > 2147483647LL) return FA_ERR_ARG;
  const size_t smem = (size_t)per_cta * p.half * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FA_DTYPE_BF16
             ? launch_vec<__nv_bfloat16>(p, vec, interleaved != 0, (unsigned)grid, smem, st)
             : launch_vec<__half>(p, vec, interleaved != 0, (unsigned)grid, smem, st);
}
