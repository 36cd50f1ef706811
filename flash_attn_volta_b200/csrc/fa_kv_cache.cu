// The paged key/value cache: appending new tokens (with the rotary rotation of
// q and k on the way, and rounding to 4 bits) and reading the cache back into
// contiguous keys and values.  Layout: fa_kv_cache.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "fa_kernels.h"
#include "fa_kv_cache.cuh"
#include "fa_rotary.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {

int check_kv_cache(const fa_sm100_kv_cache* c) {
  if (!c || !c->k_pages || c->num_pages < 1 || c->nheads_kv < 1) return FA_ERR_ARG;
  if (c->dtype != FA_DTYPE_F16 && c->dtype != FA_DTYPE_BF16) return FA_ERR_ARG;
  const int D = c->head_dim, page = c->page_size;
  if (page < kBlockTokens || page > 1024 || (page & (page - 1))) return FA_ERR_ARG;
  if (c->bits == 16) {
    if (D != 16 && D != 32 && D != 64 && D != 128) return FA_ERR_ARG;
    if (!c->v_pages || (reinterpret_cast<uintptr_t>(c->v_pages) & 15u)) return FA_ERR_ARG;
  } else if (c->bits == 4) {
    if (D != 32 && D != 64 && D != 128) return FA_ERR_ARG;
  } else {
    return FA_ERR_ARG;
  }
  if (reinterpret_cast<uintptr_t>(c->k_pages) & 15u) return FA_ERR_ARG;
  // a row of the cache is a coordinate of a tensor map
  if ((long long)c->num_pages * c->nheads_kv * page > 2147483647LL) return FA_ERR_ARG;
  return FA_OK;
}

KvView kv_view(const fa_sm100_kv_cache* c, const int* table, int table_width, int* status) {
  KvView v;
  v.k = static_cast<uint8_t*>(c->k_pages);
  v.v = static_cast<uint8_t*>(c->v_pages);
  v.table = table;
  v.table_width = table_width;
  v.num_pages = c->num_pages;
  v.page = c->page_size;
  v.heads = c->nheads_kv;
  v.D = c->head_dim;
  v.bits = c->bits;
  v.status = status;
  return v;
}

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 4096;

struct AppendPart {
  const void* in;
  long long sb, ss, sh;
  int heads;
};

struct AppendParams {
  KvView kv;
  AppendPart part[3];  // q, k, v
  void* q_out;
  const int* starts;
  const int* counts;       // null: every token is new
  const double* inv_freq;  // null: no rotation
  FastDiv per_seq, q_heads, k_heads;  // CTAs of a sequence, heads of q (0 without q), of k and v
  int S, half, per_cta, page_shift, chunk_shift;
  float magnitude;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Rounds the 32 values of a group, 8 in each of 4 neighbouring lanes, to codes.
// Returns (s, m); a group with a NaN reads back as NaN, infinities as the
// largest fp16 (its rounding to codes apart).  The quotient (x - m) / s is the correctly rounded one
// (Markstein: with r = 1/s rounded, q = d r, then q + r (d - q s) in fused
// steps), so a code is the definition's also where it is half a step; adding
// 1.5 2^23 rounds it to a whole number, ties to even, in the sum's low bits.
__device__ __forceinline__ uint32_t quantise(float (&x)[8], uint32_t (&code)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = max_nan(-65504.f, min_nan(x[i], 65504.f));
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  const __half m = __float2half_rd(lo);
  const float mf = __half2float(m);
  const __half s = __float2half_ru(__fdiv_rn(hi - mf, 15.f));
  const float sf = __half2float(s), r = __frcp_rn(sf);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - mf, q = d * r;
    const float c = fmaf(fmaf(-q, sf, d), r, q);  // 0 / 0 and NaN become 0 below
    code[i] = __float_as_uint(fminf(fmaxf(c, 0.f), 15.f) + 12582912.f) & 15u;
  }
  return (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(m) << 16);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8], uint32_t signs = 0u) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack2(v[i] ^ signs);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]),
                    Elem<T>::pack2(x[4], x[5]), Elem<T>::pack2(x[6], x[7]));
}

// a c - b s and a c + b s of one rotated dim.  For 4 bits each product and the
// sum are rounded to fp32 apart, as the formula reads, so that the value that
// is rounded to a code does not depend on what is fused.
template <int BITS>
__device__ __forceinline__ float turn(float a, float c, float b, float s) {
  return BITS == 4 ? __fadd_rn(__fmul_rn(a, c), __fmul_rn(b, s)) : a * c + b * s;
}
template <int BITS>
__device__ __forceinline__ float2 angle(double pos, double inv_freq, float magnitude) {
  return BITS == 4 ? rotary_cos_sin_exact(pos, inv_freq, magnitude) : rotary_cos_sin(pos, inv_freq, magnitude);
}

// Rotates the 8 dims e.. of a row whose own values are x.  WIDE: the thread's
// angles stand `stride` apart from `w` on (neighbouring lanes read neighbouring
// words) and the partner dims' values are y, negated in the first halves.
// Otherwise `w` holds the angles in order and partner dims are read from `row`.
template <bool INTER, int BITS>
__device__ __forceinline__ void rotate_wide(const float2* w, int stride, float (&x)[8],
                                            const float (&y)[8]) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 c = w[i / 2 * stride];
      const float a = x[i], b = x[i + 1];
      x[i] = turn<BITS>(a, c.x, -b, c.y);
      x[i + 1] = turn<BITS>(b, c.x, a, c.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 c = w[i * stride];
      x[i] = turn<BITS>(x[i], c.x, y[i], c.y);
    }
  }
}
template <typename T, bool INTER, int BITS>
__device__ __forceinline__ void rotate_any(const uint16_t* row, int e, int half, const float2* w,
                                           float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = e + i;
    if (d >= 2 * half) break;
    if constexpr (INTER) {
      if (i % 2) continue;
      const float2 c = w[d / 2];
      const float a = x[i], b = x[i + 1];
      x[i] = turn<BITS>(a, c.x, -b, c.y);
      x[i + 1] = turn<BITS>(b, c.x, a, c.y);
    } else {
      const bool first = d < half;
      const float2 c = w[first ? d : d - half];
      const float y = Elem<T>::value(row[first ? d + half : d - half]);
      x[i] = turn<BITS>(x[i], c.x, first ? -y : y, c.y);
    }
  }
}

// 8 dims (chunk c) of head h of K (part 1) or V (part 2) to the cache row
// `place` (of head 0; -1: not stored).  4 bits: all lanes of the warp take part.
template <typename T, int BITS>
__device__ __forceinline__ void store_item(const AppendParams& p, int part, int c, int h, int place,
                                           float (&x)[8]) {
  const KvView& kv = p.kv;
  const int to = place + (h << p.page_shift);  // row of the cache
  if constexpr (BITS == 16) {
    if (place >= 0)
      *reinterpret_cast<uint4*>((part == 1 ? kv.k : kv.v) + ((long long)to * kv.D + c * 8) * 2) = pack8<T>(x);
  } else {
    uint32_t code[8];
    const uint32_t sm = quantise(x, code);
    if (place < 0) return;
    const Kv4 lay(kv.D);
    const int NG = lay.groups(), grp = c / 4, t4 = c % 4, r = to % kBlockTokens;
    uint8_t* blk = kv.k + (long long)(to / kBlockTokens) * lay.bytes();
    if (part == 1) {
      const uint32_t w = code[0] | code[2] << 4 | code[4] << 8 | code[6] << 12 | code[1] << 16 |
                         code[3] << 20 | code[5] << 24 | code[7] << 28;
      reinterpret_cast<uint32_t*>(blk)[(r * 4 + t4) * NG + grp] = w;
      if (t4 == 0) reinterpret_cast<uint32_t*>(blk + lay.k_params())[r * NG + grp] = sm;
    } else {
      const int tp = r / 8, tt = r % 8 / 2, hi = r % 2;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int g = 2 * t4 + n;
        const uint32_t w =
            code[4 * n] | code[4 * n + 1] << 4 | code[4 * n + 2] << 8 | code[4 * n + 3] << 12;
        reinterpret_cast<uint16_t*>(blk + lay.v_codes())[(((tp * 8 + g) * 4 + tt) * NG + grp) * 2 + hi] =
            (uint16_t)w;
      }
      if (t4 == 0) {
        uint16_t* vp = reinterpret_cast<uint16_t*>(blk + lay.v_params());
        const int k = (grp * 4 + tt) * 4 + tp * 2 + hi;
        vp[k] = (uint16_t)sm;
        vp[k + 16 * NG] = (uint16_t)(sm >> 16);
      }
    }
  }
}

// New tokens into the cache.  Bound by HBM for prompts (every input is read
// once, every output written once) and by latency for single tokens: one
// launch does the rotation of q and k, the page lookup and both writes.
// A CTA takes whole tokens of one sequence; it makes their cosines and sines
// and finds their places in the cache once for all heads.  An item is 8
// consecutive dims of a head of q, k or v (the half layout reads the partner
// dims a second time, from L1).  The items of q, k and v start at multiples of
// 32, so a warp works on one of them, and the 4 lanes that hold a group of 32
// dims reduce its minimum and maximum by shuffles.
// WIDE: 16-byte loads at 32-bit offsets, and rotated dims that end at an item's
// border.  One token of each of 64 sequences takes the host longer (7 us) than
// the device.
template <typename T, bool INTER, int BITS, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) fa_kv_append_kernel(const AppendParams p) {
  extern __shared__ float2 cs[];
  griddep_wait();
  griddep_launch_dependents();
  const KvView& kv = p.kv;
  const int b = p.per_seq.div(blockIdx.x), s0 = (blockIdx.x - b * p.per_seq.d) * p.per_cta;
  const int ntok = min(p.per_cta, p.S - s0);
  int* places = reinterpret_cast<int*>(cs + p.per_cta * p.half);  // row of head 0, or -1
  const int hk = kv.heads;
  const long long first = (long long)p.starts[b] + s0;
  const int fresh = p.counts == nullptr ? ntok : max(0, min(ntok, max(p.counts[b], 0) - s0));  // tokens to store
  const int nq = (ntok * (int)p.q_heads.d) << p.chunk_shift, nk = (fresh * hk) << p.chunk_shift;
  const int k0 = (nq + 31) & ~31, v0 = k0 + ((nk + 31) & ~31), end = v0 + ((nk + 31) & ~31);
  for (int i = threadIdx.x; i < fresh; i += kThreads) {
    const long long pos = first + i;
    const int id = kv.page_of(b, pos, p.page_shift);
    if (id < 0) kv.report(kStatusPage);
    places[i] = id < 0 ? -1 : ((id * hk) << p.page_shift) | ((int)pos & (kv.page - 1));
  }
  const int mask = (1 << p.chunk_shift) - 1;
  T* q_out = static_cast<T*>(p.q_out) + ((((long long)b * p.S + s0) * p.q_heads.d) << (p.chunk_shift + 3));

  for (int base = threadIdx.x; base < end || base < kThreads; base += 2 * kThreads) {
    uint4 own[2], other[2];
    const T* at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int it = base + u * kThreads;
      const int part = it < k0 ? 0 : it < v0 ? 1 : 2;  // the same in all lanes of a warp
      const int i = it - (part == 0 ? 0 : part == 1 ? k0 : v0);
      const AppendPart& src = p.part[part];
      const int row = i >> p.chunk_shift, e = (i & mask) * 8;
      const FastDiv& heads = part == 0 ? p.q_heads : p.k_heads;
      const int tok = heads.div(row), h = row - tok * heads.d;
      const T* from = static_cast<const T*>(src.in) + b * src.sb + s0 * src.ss;
      if (WIDE) {
        at[u] = from + (tok * (int)src.ss + h * (int)src.sh);
        if (i < (part == 0 ? nq : nk) && it < end) {
          own[u] = *reinterpret_cast<const uint4*>(at[u] + e);
          if (!INTER && part < 2 && e < 2 * p.half)
            other[u] = *reinterpret_cast<const uint4*>(at[u] + (e < p.half ? e + p.half : e - p.half));
        }
      } else {
        at[u] = from + (tok * src.ss + h * src.sh);
      }
    }
    if (base < kThreads) {
      constexpr int N = INTER ? 4 : 8;  // pairs of an item
      for (int i = threadIdx.x; i < ntok * p.half; i += kThreads) {
        const int tok = i / p.half, f = i - tok * p.half;
        cs[tok * p.half + (WIDE ? f % N * (p.half / N) + f / N : f)] =
            angle<BITS>((double)(first + tok), p.inv_freq[f], p.magnitude);
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int it = base + u * kThreads;
      if (it >= end) break;  // whole warps
      const int part = it < k0 ? 0 : it < v0 ? 1 : 2;
      const int i = it - (part == 0 ? 0 : part == 1 ? k0 : v0);
      const bool there = i < (part == 0 ? nq : nk);
      const int row = i >> p.chunk_shift, c = i & mask, e = c * 8;
      const FastDiv& heads = part == 0 ? p.q_heads : p.k_heads;
      const int tok = there ? heads.div(row) : 0, h = row - tok * heads.d;
      float x[8] = {};
      if (there) {
        const bool turns = part < 2 && e < 2 * p.half;
        const float2* w = cs + tok * p.half;
        if (WIDE) {
          unpack8<T>(own[u], x);
          if (turns) {
            float y[8];
            const bool lower = e < p.half;
            if (!INTER) unpack8<T>(other[u], y, lower ? 0x80008000u : 0u);
            rotate_wide<INTER, BITS>(w + (INTER || lower ? c : c - p.half / 8), p.half / (INTER ? 4 : 8), x, y);
          }
        } else {
          const uint16_t* raw = reinterpret_cast<const uint16_t*>(at[u]);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = Elem<T>::value(raw[e + k]);
          if (turns) rotate_any<T, INTER, BITS>(raw, e, p.half, w, x);
        }
        if (part == 0) *reinterpret_cast<uint4*>(q_out + (long long)i * 8) = pack8<T>(x);
      }
      if (part == 0) continue;
      store_item<T, BITS>(p, part, c, h, there ? places[tok] : -1, x);
    }
  }
}

// The same for prompts: a CTA takes so many tokens that the grid is few waves, and
// each thread streams its vectors through a ring of its own in shared memory.
// The rows are the heads of q, then of k, then of v of the CTA's tokens; a thread
// keeps its dims of a row.  Measured on one B200: 6 prompts of up to 4096 tokens, 3 x 16
// heads of 64, fp16 44 us, against 89 with the kernel above (its issue slots were 78 %
// busy with each token's set-up) and 35 that its reads and writes (q of the padding
// rows among them) take at the copy rate; 4 x 1024 tokens of 32 + 2 x 8 heads of 128 into
// 4 bits 28 us, issue-bound (rounding to codes).
constexpr int kStreamStages = 4;

template <typename T, bool INTER, int BITS>
__global__ void __launch_bounds__(kThreads, 4) fa_kv_append_stream_kernel(const AppendParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  griddep_wait();
  griddep_launch_dependents();
  constexpr int LOADS = INTER ? 1 : 2, NS = kStreamStages, N = INTER ? 4 : 8;
  const KvView& kv = p.kv;
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;
  float2* cs = reinterpret_cast<float2*>(smem + NS * LOADS * kThreads * 16);
  int* places = reinterpret_cast<int*>(cs + p.per_cta * p.half);
  const int b = p.per_seq.div(blockIdx.x), s0 = (blockIdx.x - b * p.per_seq.d) * p.per_cta;
  const int ntok = min(p.per_cta, p.S - s0), hk = kv.heads;
  const long long first = (long long)p.starts[b] + s0;
  const int fresh = p.counts == nullptr ? ntok : max(0, min(ntok, max(p.counts[b], 0) - s0));
  const int c = threadIdx.x & ((1 << p.chunk_shift) - 1), e = c * 8;
  const int step = kThreads >> p.chunk_shift, whole = (32 >> p.chunk_shift) - 1;  // rows of a warp - 1
  const int nq = ntok * (int)p.q_heads.d, nk = fresh * hk;
  const bool turning = e < 2 * p.half, lower = e < p.half;
  const uint32_t signs = lower ? 0x80008000u : 0u;
  const int partner = lower ? p.half : -p.half;
  T* q_out = static_cast<T*>(p.q_out) + ((((long long)b * p.S + s0) * p.q_heads.d) << (p.chunk_shift + 3)) + e;
  const int start = threadIdx.x >> p.chunk_shift;
  const float2* angles = cs + (INTER || lower ? c : c - p.half / 8);

  // The rows of one of q (0), k (1) and v (2); `ready` runs behind the first loads.
  auto run = [&](auto part_tag, int rows, const FastDiv heads, auto&& ready) {
    constexpr int PART = decltype(part_tag)::value;
    const AppendPart& src = p.part[PART];
    const T* from = static_cast<const T*>(src.in) + b * src.sb + s0 * src.ss + e;
    const int ss = (int)src.ss, sh = (int)src.sh;
    auto load = [&](int row, int stage) {
      if (row < rows) {
        const int tok = heads.div(row), h = row - tok * heads.d;
        const T* at = from + (tok * ss + h * sh);
        const uint32_t dst = smem_u32(ring + stage * LOADS * kThreads);
        cp_async<16>(dst, at);
        if (!INTER && PART < 2 && turning) cp_async<16>(dst + kThreads * 16, at + partner);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) load(start + i * step, i);
    ready();
    int stage = 0;
    // the same number of rounds for all lanes of a warp
    const int end = PART == 0 ? rows : (rows + whole) & ~whole;
    for (int row = start; row < end; row += step) {
      load(row + (NS - 1) * step, stage == 0 ? NS - 1 : stage - 1);
      cp_async_wait<NS - 1>();
      const bool there = PART == 0 || row < rows;
      const int tok = there ? heads.div(row) : 0, h = row - tok * heads.d;
      float x[8] = {};
      if (there) {
        unpack8<T>(ring[stage * LOADS * kThreads], x);
        if (PART < 2 && turning) {
          float y[8];
          if (!INTER) unpack8<T>(ring[(stage * LOADS + 1) * kThreads], y, signs);
          rotate_wide<INTER, BITS>(angles + tok * p.half, p.half / N, x, y);
        }
      }
      if (PART == 0)
        *reinterpret_cast<uint4*>(q_out + ((long long)row << (p.chunk_shift + 3))) = pack8<T>(x);
      else
        store_item<T, BITS>(p, PART, c, h, there ? places[tok] : -1, x);
      if (++stage == NS) stage = 0;
    }
    cp_async_wait<0>();
  };
  run(std::integral_constant<int, 0>{}, nq, p.q_heads, [&]() {
    for (int i = threadIdx.x; i < fresh; i += kThreads) {
      const long long pos = first + i;
      const int id = kv.page_of(b, pos, p.page_shift);
      if (id < 0) kv.report(kStatusPage);
      places[i] = id < 0 ? -1 : ((id * hk) << p.page_shift) | ((int)pos & (kv.page - 1));
    }
    for (int i = threadIdx.x; i < ntok * p.half; i += kThreads) {
      const int tok = i / p.half, f = i - tok * p.half;
      cs[tok * p.half + f % N * (p.half / N) + f / N] =
          angle<BITS>((double)(first + tok), p.inv_freq[f], p.magnitude);
    }
    __syncthreads();
  });
  run(std::integral_constant<int, 1>{}, nk, p.k_heads, [] {});
  run(std::integral_constant<int, 2>{}, nk, p.k_heads, [] {});
}

template <typename T, int BITS>
int launch_append_stream(const AppendParams& p, bool interleaved, unsigned grid, size_t smem,
                         cudaStream_t st) {
  auto kernel = interleaved ? fa_kv_append_stream_kernel<T, true, BITS>
                            : fa_kv_append_stream_kernel<T, false, BITS>;
  return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, p) == cudaSuccess ? FA_OK
                                                                                    : FA_ERR_LAUNCH;
}

template <typename T, int BITS, bool WIDE>
int launch_append(const AppendParams& p, bool interleaved, unsigned grid, size_t smem,
                  cudaStream_t st) {
  const cudaError_t e =
      interleaved ? launch_pdl(fa_kv_append_kernel<T, true, BITS, WIDE>, dim3(grid), dim3(kThreads),
                               smem, st, p)
                  : launch_pdl(fa_kv_append_kernel<T, false, BITS, WIDE>, dim3(grid), dim3(kThreads),
                               smem, st, p);
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

template <typename T>
int launch_append_t(const AppendParams& p, bool is_wide, bool stream, bool interleaved, unsigned grid,
                    size_t smem, cudaStream_t st) {
  if (stream)
    return p.kv.bits == 16 ? launch_append_stream<T, 16>(p, interleaved, grid, smem, st)
                           : launch_append_stream<T, 4>(p, interleaved, grid, smem, st);
  if (p.kv.bits == 16)
    return is_wide ? launch_append<T, 16, true>(p, interleaved, grid, smem, st)
                   : launch_append<T, 16, false>(p, interleaved, grid, smem, st);
  return is_wide ? launch_append<T, 4, true>(p, interleaved, grid, smem, st)
                 : launch_append<T, 4, false>(p, interleaved, grid, smem, st);
}

// ---------------------------------------------------------------- read
struct ReadParams {
  KvView kv;
  const int* lengths;
  void* k_out;  // (batch, max_len, heads, D)
  void* v_out;
  int max_len, page_shift;
};

// 4-bit codes to values: a nibble pair masked out of its word is two fp16
// subnormals (c 2^-24 from bits 0..3, c 2^-20 from bits 4..7), which convert
// exactly.
__device__ __forceinline__ float2 pair_of(uint32_t masked) {
  return __half22float2(*reinterpret_cast<const __half2*>(&masked));
}
// Two values of the cache in the result's type.
template <typename T>
__device__ __forceinline__ uint32_t read2(float a, float b) {
  const uint32_t w = Elem<T>::pack2(a, b);
  return std::is_same<T, __half>::value ? most_half2(w) : w;
}
template <int N>
__device__ __forceinline__ void load_words(const uint32_t* at, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = *at;
  }
}

// The cached tokens as contiguous K and V, rows behind a sequence's length
// zero.  Bound by HBM: the cache is read once, K and V written once.  A warp
// takes one 16-token block of one head and has all its loads in flight at
// once.  4-bit: lane (g, t) = (lane / 4, lane % 4) reads the words that it
// would read in the attention kernel, each once: 8 dims of each group of tokens
// g and g + 8 (K), 4 dims of each group of tokens 2 t, 2 t + 1 and the two 8
// further (V); a store instruction writes whole 32-byte sectors.  Measured on one
// B200: 12 sequences of 33 to 6001 tokens, 8 heads of 64, 4-bit 27 us (6.3 TB/s).
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(kThreads) fa_kv_read_kernel(const ReadParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const KvView& kv = p.kv;
  const int b = blockIdx.y, first = blockIdx.x * kBlockTokens, lane = threadIdx.x % 32;
  const int h = blockIdx.z * (kThreads / 32) + threadIdx.x / 32;
  const int given = p.lengths[b], len = min(kv.clamp_length(given), p.max_len);
  const bool speaks = lane == 0 && h == 0;
  if (kv.bad_length(given) && blockIdx.x == 0 && speaks) kv.report(kStatusPage);
  if (h >= kv.heads) return;
  const int rows = min(p.max_len - first, kBlockTokens);  // tokens of the block to write
  int copied = max(0, min(len - first, kBlockTokens));    // and to copy
  int id = -1;
  if (copied > 0) {
    id = kv.page_of(b, first, p.page_shift);
    if (id < 0 && speaks) kv.report(kStatusPage);
  }
  if (id < 0) copied = 0;
  constexpr int CHUNKS = D / 8;
  // of token 0 of the block, in 16-byte vectors; a token is `pitch` further
  const int pitch = kv.heads * CHUNKS;
  const long long out = (((long long)b * p.max_len + first) * kv.heads + h) * CHUNKS;
  uint4* k_out = static_cast<uint4*>(p.k_out) + out;
  uint4* v_out = static_cast<uint4*>(p.v_out) + out;
  const int at = id < 0 ? 0 : (((id * kv.heads + h) << p.page_shift) | (first & (kv.page - 1)));
  if (copied < rows) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i = copied * CHUNKS + lane; i < rows * CHUNKS; i += 32) {
      const int o = i / CHUNKS * pitch + i % CHUNKS;
      k_out[o] = zero;
      v_out[o] = zero;
    }
    if (copied == 0) return;
  }
  if constexpr (BITS == 16) {
    constexpr int N = (16 * CHUNKS + 31) / 32;  // vectors of a lane
    const uint4* ks = reinterpret_cast<const uint4*>(kv.k) + (long long)at * CHUNKS;
    const uint4* vs = reinterpret_cast<const uint4*>(kv.v) + (long long)at * CHUNKS;
    uint4 x[N], y[N];
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (u * 32 + lane < copied * CHUNKS) {
        x[u] = ks[u * 32 + lane];
        y[u] = vs[u * 32 + lane];
      }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int i = u * 32 + lane;
      if (i < copied * CHUNKS) {
        k_out[i / CHUNKS * pitch + i % CHUNKS] = x[u];
        v_out[i / CHUNKS * pitch + i % CHUNKS] = y[u];
      }
    }
  } else {
    constexpr Kv4 lay(D);
    constexpr int NG = lay.groups();
    const int g = lane / 4, t = lane % 4;
    const uint8_t* blk = kv.k + (long long)(at / kBlockTokens) * lay.bytes();
    const uint32_t* kc = reinterpret_cast<const uint32_t*>(blk);
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(blk + lay.k_params());
    const uint32_t* vc = reinterpret_cast<const uint32_t*>(blk + lay.v_codes());
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + lay.v_params());
    uint32_t k[2][NG], kq[2][NG], v[2][NG], vs[2 * NG], vm[2 * NG];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      load_words<NG>(kc + (n * 32 + lane) * NG, k[n]);
      load_words<NG>(kp + (n * 8 + g) * NG, kq[n]);
      load_words<NG>(vc + (n * 32 + lane) * NG, v[n]);
    }
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {  // the four tokens' scales and minima
      const uint2 s = *reinterpret_cast<const uint2*>(vp + (grp * 4 + t) * 2);
      const uint2 m = *reinterpret_cast<const uint2*>(vp + 8 * NG + (grp * 4 + t) * 2);
      vs[2 * grp] = s.x;
      vs[2 * grp + 1] = s.y;
      vm[2 * grp] = m.x;
      vm[2 * grp + 1] = m.y;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = n * 8 + g;
      if (r < copied) {
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          const float2 sm = pair_of(kq[n][grp]);
          const float s24 = sm.x * 0x1p24f, s20 = sm.x * 0x1p20f;
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 c = pair_of((i < 2 ? k[n][grp] : k[n][grp] >> 8) & (i % 2 ? 0x00F000F0u : 0x000F000Fu));
            x[2 * i] = fmaf(i % 2 ? s20 : s24, c.x, sm.y);
            x[2 * i + 1] = fmaf(i % 2 ? s20 : s24, c.y, sm.y);
          }
          k_out[r * pitch + grp * 4 + t] =
              make_uint4(read2<T>(x[0], x[1]), read2<T>(x[2], x[3]), read2<T>(x[4], x[5]), read2<T>(x[6], x[7]));
        }
      }
      const int r0 = n * 8 + 2 * t;
      if (r0 < copied) {
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          const float2 s = pair_of(vs[2 * grp + n]), m = pair_of(vm[2 * grp + n]);  // of both tokens
          float2 c[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            c[i] = pair_of((i < 2 ? v[n][grp] : v[n][grp] >> 8) & (i % 2 ? 0x00F000F0u : 0x000F000Fu));
          float x[4], y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = fmaf(s.x * (i % 2 ? 0x1p20f : 0x1p24f), c[i].x, m.x);
            y[i] = fmaf(s.y * (i % 2 ? 0x1p20f : 0x1p24f), c[i].y, m.y);
          }
          uint2* to = reinterpret_cast<uint2*>(v_out + r0 * pitch) + grp * 8 + g;
          to[0] = make_uint2(read2<T>(x[0], x[1]), read2<T>(x[2], x[3]));
          if (r0 + 1 < copied)
            to[2 * pitch] = make_uint2(read2<T>(y[0], y[1]), read2<T>(y[2], y[3]));
        }
      }
    }
  }
}

template <typename T, int D>
cudaError_t launch_read(const ReadParams& p, dim3 grid, cudaStream_t st) {
  if (p.kv.bits == 16) return launch_pdl(fa_kv_read_kernel<T, D, 16>, grid, dim3(kThreads), 0, st, p);
  if constexpr (D >= 32) return launch_pdl(fa_kv_read_kernel<T, D, 4>, grid, dim3(kThreads), 0, st, p);
  return cudaErrorInvalidValue;
}
template <typename T>
cudaError_t launch_read_d(const ReadParams& p, dim3 grid, cudaStream_t st) {
  switch (p.kv.D) {
    case 16: return launch_read<T, 16>(p, grid, st);
    case 32: return launch_read<T, 32>(p, grid, st);
    case 64: return launch_read<T, 64>(p, grid, st);
    default: return launch_read<T, 128>(p, grid, st);
  }
}

int log2_of(int x) {
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

bool bad_append_part(const fa_sm100_heads& x) {
  return !x.in || x.heads < 1 || (reinterpret_cast<uintptr_t>(x.in) & 1u);
}
// 16-byte vectors, and a CTA's tokens within 2^31 elements.
bool wide(const fa_sm100_heads& x, long long tokens) {
  const double reach = (double)tokens * (x.stride_seq < 0 ? -x.stride_seq : x.stride_seq) +
                       (double)x.heads * (x.stride_head < 0 ? -x.stride_head : x.stride_head);
  return !(reinterpret_cast<uintptr_t>(x.in) & 15u) &&
         !((x.stride_batch | x.stride_seq | x.stride_head) & 7) && reach < 2147480000.0;
}

}  // namespace
}  // namespace fa_sm100

extern "C" int fa_sm100_kv_append(const fa_sm100_kv_cache* cache, const fa_sm100_heads* k,
                                  const fa_sm100_heads* v, const fa_sm100_heads* q,
                                  const int* page_table, int table_width, const int* starts,
                                  const int* counts, const double* inv_freq, int rotary_dim,
                                  int interleaved, float magnitude, int batch, int seqlen,
                                  int* status, void* stream) {
  using namespace fa_sm100;
  int rc = check_kv_cache(cache);
  if (rc != FA_OK) return rc;
  if (batch < 1 || seqlen < 1 || table_width < 1 || !page_table || !starts) return FA_ERR_ARG;
  if (!k || !v || bad_append_part(*k) || bad_append_part(*v)) return FA_ERR_ARG;
  if (k->heads != cache->nheads_kv || v->heads != cache->nheads_kv) return FA_ERR_ARG;
  if (q && (bad_append_part(*q) || !q->out || (reinterpret_cast<uintptr_t>(q->out) & 15u)))
    return FA_ERR_ARG;
  if (q && (long long)q->heads * cache->head_dim > (1 << 20)) return FA_ERR_ARG;
  if ((long long)k->heads * cache->head_dim > (1 << 20)) return FA_ERR_ARG;
  const uintptr_t ints = reinterpret_cast<uintptr_t>(page_table) | reinterpret_cast<uintptr_t>(starts) |
                         reinterpret_cast<uintptr_t>(counts);
  if ((ints & 3u) || (reinterpret_cast<uintptr_t>(inv_freq) & 7u)) return FA_ERR_ARG;
  if (inv_freq && (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > cache->head_dim)) return FA_ERR_ARG;
  if ((rc = bind_device()) != FA_OK) return rc;
  AppendParams p = {};
  p.kv = kv_view(cache, page_table, table_width, status);
  if (q) p.part[0] = {q->in, q->stride_batch, q->stride_seq, q->stride_head, q->heads};
  p.part[1] = {k->in, k->stride_batch, k->stride_seq, k->stride_head, k->heads};
  p.part[2] = {v->in, v->stride_batch, v->stride_seq, v->stride_head, v->heads};
  p.q_out = q ? q->out : nullptr;
  p.starts = starts;
  p.counts = counts;
  p.inv_freq = inv_freq;
  p.half = inv_freq ? rotary_dim / 2 : 0;
  p.S = seqlen;
  p.magnitude = magnitude;
  p.page_shift = log2_of(cache->page_size);
  p.chunk_shift = log2_of(cache->head_dim / 8);
  // whole tokens until every thread has two items: one round
  const long long per_token = (long long)((q ? q->heads : 0) + 2 * k->heads) * (cache->head_dim / 8);
  long long per_cta = 2 * kThreads / per_token;
  // prompts: CTAs that stream, two waves of four per SM (ragged counts leave some
  // CTAs with less to do), where that gives each thread enough rounds
  const size_t ring = (size_t)kStreamStages * (interleaved ? 1 : 2) * kThreads * 16;
  const size_t each = p.half * sizeof(float2) + sizeof(int);  // of a token
  const long long slots = 8LL * sm_count() / batch, per_seq = slots < 1 ? 1 : slots;
  const long long room = (long long)((48 * 1024 - ring) / each);
  long long many = (seqlen + per_seq - 1) / per_seq;
  if (many > room) many = (many + (many + room - 1) / room - 1) / ((many + room - 1) / room);
  const auto fits = [&](long long tokens) {
    return wide(*k, tokens) && wide(*v, tokens) && (!q || wide(*q, tokens)) &&
           (interleaved ? p.half % 4 : p.half % 8) == 0;
  };
  const bool streams = fits(many) && many * per_token >= 2 * 2 * kThreads;
  if (streams) per_cta = many;
  if (p.half > 0 && per_cta > kMaxAngles / p.half) per_cta = kMaxAngles / p.half;
  if (per_cta > seqlen) per_cta = seqlen;
  if (per_cta < 1) per_cta = 1;
  p.per_cta = (int)per_cta;
  const bool is_wide = fits(per_cta);
  p.per_seq = FastDiv((unsigned)((seqlen + per_cta - 1) / per_cta));
  p.k_heads = FastDiv((unsigned)k->heads);
  if (q) p.q_heads = FastDiv((unsigned)q->heads);
  const long long grid = (long long)p.per_seq.d * batch;
  if (grid > 2147483647LL) return FA_ERR_ARG;
  const size_t smem = (streams ? ring : 0) + (size_t)per_cta * each;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == FA_DTYPE_BF16
             ? launch_append_t<__nv_bfloat16>(p, is_wide, streams, interleaved != 0, (unsigned)grid,
                                              smem, st)
             : launch_append_t<__half>(p, is_wide, streams, interleaved != 0, (unsigned)grid,
                                              smem, st);
}

extern "C" int fa_sm100_kv_read(const fa_sm100_kv_cache* cache, const int* page_table,
                                int table_width, const int* lengths, void* k_out, void* v_out,
                                int batch, int max_len, int* status, void* stream) {
  using namespace fa_sm100;
  int rc = check_kv_cache(cache);
  if (rc != FA_OK) return rc;
  if (batch < 1 || batch > 65535 || max_len < 1 || table_width < 1) return FA_ERR_ARG;
  if (!page_table || !lengths || !k_out || !v_out) return FA_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(page_table) | reinterpret_cast<uintptr_t>(lengths)) & 3u)
    return FA_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u)
    return FA_ERR_ARG;
  if ((long long)cache->nheads_kv * cache->head_dim > (1 << 20)) return FA_ERR_ARG;
  if ((rc = bind_device()) != FA_OK) return rc;
  ReadParams p;
  p.kv = kv_view(cache, page_table, table_width, status);
  p.lengths = lengths;
  p.k_out = k_out;
  p.v_out = v_out;
  p.max_len = max_len;
  p.page_shift = log2_of(cache->page_size);
  constexpr int kWarps = kThreads / 32;
  const dim3 grid((unsigned)(((long long)max_len + kBlockTokens - 1) / kBlockTokens), (unsigned)batch,
                  (unsigned)((cache->nheads_kv + kWarps - 1) / kWarps));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache->dtype == FA_DTYPE_BF16 ? launch_read_d<__nv_bfloat16>(p, grid, st)
                                                      : launch_read_d<__half>(p, grid, st);
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}
