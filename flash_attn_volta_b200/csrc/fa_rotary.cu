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
// so the loads' latency covers them.  Measured on one B200, per launch: 8 x 2048
// tokens of 32 heads of 128 42 us (6.4 TB/s), 40009 tokens of 32 heads of 64, half of
// each in interleaved pairs, 55 us (6.0 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "fa_kernels.h"
#include "fa_rotary.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kThreads = 256;
// Vectors (half: pairs of vectors) in flight per thread: 64 bytes of loads.
__host__ __device__ constexpr int items_of(bool interleaved) { return interleaved ? 4 : 2; }
constexpr int kStreamRounds = 2;   // rounds of the plain kernel from which the streaming one takes over
constexpr int kMaxAngles = 4096;   // cosines and sines of a CTA: 32 KB

// The streaming kernel's ring: stages, and bytes of a CTA.
__host__ __device__ constexpr int stages_of(bool interleaved) { return interleaved ? 6 : 4; }
constexpr size_t ring_bytes(bool interleaved, int vec) {
  return (size_t)stages_of(interleaved) * (interleaved ? 1 : 2) * kThreads * 2 * vec;
}

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
  FastDiv per_seq, per_head, heads;  // CTAs of a sequence, items of a head, heads of q and k
  float magnitude, sign;
};

// One thread's share of a head (an item): a vector of VEC first halves and the
// VEC second halves of the same pairs (half), or VEC elements = VEC/2 pairs
// (interleaved), or VEC elements behind R.  A vector's i-th cosine and sine are
// `turning` apart in shared memory, so neighbouring lanes read neighbouring
// words.  Addresses inside a CTA's tokens are 32-bit offsets from 64-bit bases
// where the strides allow it (SMALL).
template <typename T, int VEC, bool INTER, bool SMALL>
__global__ void __launch_bounds__(kThreads, 4) fa_rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 cs[];
  griddep_wait();
  griddep_launch_dependents();
  using V = Pack16<VEC>;
  using Off = typename std::conditional<SMALL, int, long long>::type;
  constexpr int PAIRS = INTER ? VEC / 2 : VEC, ITEMS = items_of(INTER);
  const int half = p.half, turning = half / PAIRS;  // items of a head that rotate
  const int b = p.per_seq.div(blockIdx.x), s0 = (blockIdx.x - b * p.per_seq.d) * p.per_cta;
  const int ntok = min(p.per_cta, p.S - s0);
  const int total = ntok * (int)(p.heads.d * p.per_head.d);
  const T* in_q = static_cast<const T*>(p.q.in) + b * p.q.sb + s0 * p.q.ss;
  const T* in_k = static_cast<const T*>(p.k.in) + b * p.k.sb + s0 * p.k.ss;
  T* out_q = static_cast<T*>(p.q.out) + ((long long)b * p.S + s0) * p.q.heads * p.D;
  T* out_k = static_cast<T*>(p.k.out) + ((long long)b * p.S + s0) * p.k.heads * p.D;

  for (int base = 0; base < total; base += kThreads * ITEMS) {
    V a[ITEMS], o[ITEMS];
    T* dst[ITEMS];
    int w[ITEMS];  // first angle; -1: copied
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const int it = base + u * kThreads + threadIdx.x;
      dst[u] = nullptr;
      if (it >= total) continue;
      const int row = p.per_head.div(it), j = it - row * p.per_head.d;
      const int tok = p.heads.div(row), h = row - tok * p.heads.d;
      const bool turns = j < turning, is_k = h >= p.q.heads;
      const int e = turns ? j * VEC : 2 * half + (j - turning) * VEC;
      const T* src;
      if (is_k) {
        const int hp = h - p.q.heads;
        src = in_k + ((Off)tok * (Off)p.k.ss + (Off)hp * (Off)p.k.sh + e);
        dst[u] = out_k + ((Off)(tok * p.k.heads + hp) * p.D + e);
      } else {
        src = in_q + ((Off)tok * (Off)p.q.ss + (Off)h * (Off)p.q.sh + e);
        dst[u] = out_q + ((Off)(tok * p.q.heads + h) * p.D + e);
      }
      w[u] = turns ? tok * half + j : -1;
      a[u] = *reinterpret_cast<const V*>(src);
      if (!INTER && turns) o[u] = *reinterpret_cast<const V*>(src + half);
    }
    if (base == 0) {
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
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      if (dst[u] == nullptr) continue;
      if (w[u] >= 0) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const float2 c = cs[w[u] + i * turning];
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
}

// The same for many tokens: a CTA takes so many that the grid is one wave, and
// each thread streams its vectors through a ring of its own in shared memory
// (no other thread reads them, so the waits are the thread's own): the loads in
// flight then need no registers and do not stop while a round is computed.  A
// thread keeps its column (its dims of a head) and steps down the rows (heads of
// tokens).  Against the kernel above: 42 / 55 us and 55 / 86 us at the sizes there.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads, 4) fa_rotary_stream_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  griddep_wait();
  griddep_launch_dependents();
  using V = Pack16<VEC>;
  constexpr int PAIRS = INTER ? VEC / 2 : VEC, LOADS = INTER ? 1 : 2, NS = stages_of(INTER);
  V* ring = reinterpret_cast<V*>(smem) + threadIdx.x;  // (stage, load) at * kThreads
  float2* cs = reinterpret_cast<float2*>(smem + (size_t)NS * LOADS * kThreads * sizeof(V));
  const int half = p.half, turning = half / PAIRS;
  const int b = p.per_seq.div(blockIdx.x), s0 = (blockIdx.x - b * p.per_seq.d) * p.per_cta;
  const int ntok = min(p.per_cta, p.S - s0), rows = ntok * (int)p.heads.d;
  const T* in_q = static_cast<const T*>(p.q.in) + b * p.q.sb + s0 * p.q.ss;
  const T* in_k = static_cast<const T*>(p.k.in) + b * p.k.sb + s0 * p.k.ss;
  T* out_q = static_cast<T*>(p.q.out) + ((long long)b * p.S + s0) * p.q.heads * p.D;
  T* out_k = static_cast<T*>(p.k.out) + ((long long)b * p.S + s0) * p.k.heads * p.D;
  const int first = p.per_head.div(threadIdx.x), col = threadIdx.x - first * p.per_head.d;
  const int step = kThreads / p.per_head.d;
  const bool turns = col < turning;
  const int e = turns ? col * VEC : 2 * half + (col - turning) * VEC;
  const int start = first < step ? first : rows;  // threads without a whole row idle

  auto load = [&](int row, int stage) {
    if (row < rows) {
      const int tok = p.heads.div(row), h = row - tok * p.heads.d;
      const T* src = h < p.q.heads
                         ? in_q + (tok * (int)p.q.ss + h * (int)p.q.sh + e)
                         : in_k + (tok * (int)p.k.ss + (h - p.q.heads) * (int)p.k.sh + e);
      const uint32_t dst = smem_u32(ring + stage * LOADS * kThreads);
      cp_async<sizeof(V)>(dst, src);
      if (!INTER && turns) cp_async<sizeof(V)>(dst + kThreads * sizeof(V), src + half);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load(start + i * step, i);
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
  int stage = 0;
  for (int row = start; row < rows; row += step) {
    load(row + (NS - 1) * step, stage == 0 ? NS - 1 : stage - 1);
    cp_async_wait<NS - 1>();
    V a = ring[stage * LOADS * kThreads], o;
    const int tok = p.heads.div(row), h = row - tok * p.heads.d;
    T* dst = h < p.q.heads ? out_q + ((tok * p.q.heads + h) * p.D + e)
                           : out_k + ((tok * p.k.heads + h - p.q.heads) * p.D + e);
    if (turns) {
      if (!INTER) o = ring[(stage * LOADS + 1) * kThreads];
      const float2* w = cs + tok * half + col;
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 c = w[i * turning];
        uint16_t& lo = INTER ? a.v[2 * i] : a.v[i];
        uint16_t& hi = INTER ? a.v[2 * i + 1] : o.v[i];
        const float x = Elem<T>::value(lo), y = Elem<T>::value(hi);
        lo = Elem<T>::bits(x * c.x - y * c.y);
        hi = Elem<T>::bits(y * c.x + x * c.y);
      }
      if (!INTER) *reinterpret_cast<V*>(dst + half) = o;
    }
    *reinterpret_cast<V*>(dst) = a;
    if (++stage == NS) stage = 0;
  }
  cp_async_wait<0>();
}

template <typename T, int VEC>
int launch_stream(const RotaryParams& p, bool interleaved, unsigned grid, size_t angles, cudaStream_t st) {
  if constexpr (VEC > 1) {
    auto kernel = interleaved ? fa_rotary_stream_kernel<T, VEC, true> : fa_rotary_stream_kernel<T, VEC, false>;
    const size_t smem = ring_bytes(interleaved, VEC) + angles;  // below 48 KB
    return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, p) == cudaSuccess ? FA_OK
                                                                                      : FA_ERR_LAUNCH;
  }
  return FA_ERR_ARG;
}

template <typename T, int VEC>
int launch(const RotaryParams& p, bool interleaved, bool small, unsigned grid, size_t smem,
           cudaStream_t st) {
  constexpr int IV = VEC > 1 ? VEC : 2;
  auto kernel = interleaved ? (small ? fa_rotary_kernel<T, IV, true, true>
                                     : fa_rotary_kernel<T, IV, true, false>)
                            : (small ? fa_rotary_kernel<T, VEC, false, true>
                                     : fa_rotary_kernel<T, VEC, false, false>);
  return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, p) == cudaSuccess ? FA_OK
                                                                                    : FA_ERR_LAUNCH;
}

template <typename T>
int launch_vec(const RotaryParams& p, int vec, bool interleaved, bool small, bool stream,
               unsigned grid, size_t smem, cudaStream_t st) {
  if (stream) {
    switch (vec) {
      case 8: return launch_stream<T, 8>(p, interleaved, grid, smem, st);
      case 4: return launch_stream<T, 4>(p, interleaved, grid, smem, st);
      default: return launch_stream<T, 2>(p, interleaved, grid, smem, st);
    }
  }
  switch (vec) {
    case 8: return launch<T, 8>(p, interleaved, small, grid, smem, st);
    case 4: return launch<T, 4>(p, interleaved, small, grid, smem, st);
    case 2: return launch<T, 2>(p, interleaved, small, grid, smem, st);
    default: return launch<T, 1>(p, interleaved, small, grid, smem, st);
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

// Every element of a CTA's tokens is within 2^31 of the first one.
bool small_offsets(const fa_sm100_heads& x, long long tokens, int D) {
  const double reach = (double)tokens * (x.stride_seq < 0 ? -x.stride_seq : x.stride_seq) +
                       (double)x.heads * (x.stride_head < 0 ? -x.stride_head : x.stride_head) +
                       (double)tokens * x.heads * D + D;
  return reach < 2147483647.0;
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
  if (interleaved && (part_vec(*q) == 1 || (k && part_vec(*k) == 1))) return FA_ERR_ARG;  // 4-byte pairs
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
  const int rc = bind_device();
  if (rc != FA_OK) return rc;
  int vec = part_vec(*q);
  if (k && part_vec(*k) < vec) vec = part_vec(*k);
  // a vector may not cross from the rotated dims into the others
  const int unit = interleaved ? rotary_dim : rotary_dim / 2;
  while (vec > 1 && (unit % vec || head_dim % vec || rotary_dim % vec)) vec /= 2;
  const int per_head = (interleaved ? head_dim : head_dim - p.half) / vec;
  const int heads = q->heads + (k ? k->heads : 0);
  // whole tokens until the threads have their vectors: one round, so that CTAs
  // in different phases overlap.  One against two rounds, us: 1000 tokens of 40 heads
  // of 128 6.4 / 7.0, 1500 of them 8.5 / 7.4, 4000 of 32 heads of 64 7.6 / 8.2, and
  // 9.2 / 9.8 with half of each in interleaved pairs
  const long long per_token = (long long)heads * per_head;
  const long long per_round = (long long)kThreads * items_of(interleaved != 0);
  long long per_cta = per_round / per_token;
  // many tokens: one wave of four CTAs per SM that stream, where that gives each
  // thread enough rounds
  const long long slots = 4LL * sm_count() / batch, per_seq = slots < 1 ? 1 : slots;
  const long long room = (long long)(48 * 1024 - ring_bytes(interleaved != 0, vec)) / (8LL * p.half);
  long long many = (seqlen + per_seq - 1) / per_seq;
  if (room >= 1 && many > room) many = (many + (many + room - 1) / room - 1) / ((many + room - 1) / room);
  const bool fits = small_offsets(*q, many, head_dim) && (!k || small_offsets(*k, many, head_dim));
  const bool stream_rounds =
      vec > 1 && per_head <= kThreads && many <= room && fits && many * per_token >= kStreamRounds * per_round;
  if (stream_rounds) per_cta = many;
  if (per_cta > kMaxAngles / p.half) per_cta = kMaxAngles / p.half;
  if (per_cta > seqlen) per_cta = seqlen;
  if (per_cta < 1) per_cta = 1;
  p.per_cta = (int)per_cta;
  p.per_head = FastDiv(per_head);
  p.heads = FastDiv(heads);
  p.per_seq = FastDiv((unsigned)((seqlen + per_cta - 1) / per_cta));
  const long long grid = (long long)p.per_seq.d * batch;
  if (grid > 2147483647LL) return FA_ERR_ARG;
  const bool small = small_offsets(*q, per_cta, head_dim) && (!k || small_offsets(*k, per_cta, head_dim));
  const size_t smem = (size_t)per_cta * p.half * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FA_DTYPE_BF16
             ? launch_vec<__nv_bfloat16>(p, vec, interleaved != 0, small, stream_rounds, (unsigned)grid,
                                         smem, st)
             : launch_vec<__half>(p, vec, interleaved != 0, small, stream_rounds, (unsigned)grid,
                                         smem, st);
}
