// The paged key/value cache: appending new tokens (with the rotary rotation of
// q and k on the way, and rounding to 4 bits) and reading the cache back into
// contiguous keys and values.  Layout: fa_kv_cache.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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
  AppendPart q, k, v;
  void* q_out;
  const int* starts;
  const int* counts;  // null: every token is new
  const double* inv_freq;  // null: no rotation
  long long tokens;
  int S, half, per_cta;
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
// largest fp16.  The division is correctly rounded, so a code is the definition's
// also where (x - m) / s is half a step.
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
  const float sf = __half2float(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = rintf(__fdiv_rn(x[i] - mf, sf));  // 0 / 0 and NaN become 0
    code[i] = (uint32_t)fminf(fmaxf(c, 0.f), 15.f);
  }
  return (uint32_t)__half_as_ushort(s) | ((uint32_t)__half_as_ushort(m) << 16);
}

// 8 consecutive dims of a row as fp32; VEC elements per load.
template <typename T, int VEC>
__device__ __forceinline__ void load8(const T* src, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += VEC) {
    const Pack16<VEC> p = *reinterpret_cast<const Pack16<VEC>*>(src + i);
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[i + j] = Elem<T>::value(p.v[j]);
  }
}

// Rotates the 8 dims e.. of a row (the thread's own values in x).
template <typename T, int VEC, bool INTER>
__device__ __forceinline__ void rotate8(const T* row, int e, int half, const float2* cs,
                                        float (&x)[8]) {
  if (e >= 2 * half) return;
  if (INTER) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (e + i < 2 * half) {
        const float2 w = cs[(e + i) / 2];
        const float a = x[i], b = x[i + 1];
        x[i] = a * w.x - b * w.y;
        x[i + 1] = b * w.x + a * w.y;
      }
    }
    return;
  }
  float y[8];
  if (VEC == 8 && half % 8 == 0) {
    load8<T, VEC>(row + (e < half ? e + half : e - half), y);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = e + i;
      y[i] = d < 2 * half
                 ? Elem<T>::value(reinterpret_cast<const uint16_t*>(row)[d < half ? d + half : d - half])
                 : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = e + i;
    if (d < half) {
      const float2 w = cs[d];
      x[i] = x[i] * w.x - y[i] * w.y;
    } else if (d < 2 * half) {
      const float2 w = cs[d - half];
      x[i] = x[i] * w.x + y[i] * w.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ Pack16<8> pack8(const float (&x)[8]) {
  Pack16<8> p;
#pragma unroll
  for (int i = 0; i < 8; ++i) p.v[i] = Elem<T>::bits(x[i]);
  return p;
}

// New tokens into the cache.  Bound by HBM for prompts (every input is read
// once, every output written once) and by latency for single tokens: one
// launch does the rotation of q and k, the page lookup and both writes.
// A CTA takes whole tokens, whose cosines and sines it makes once for all
// heads; an item is 8 consecutive dims of a head of q, k or v (the half layout
// reads the partner dims a second time, from L1).  The item ranges of q, k and
// v start at multiples of 32, so a warp works on one of them, and the 4 lanes
// that hold a group of 32 dims reduce its minimum and maximum by shuffles.
template <typename T, int VEC, bool INTER, int BITS>
__global__ void __launch_bounds__(kThreads) fa_kv_append_kernel(const AppendParams p) {
  extern __shared__ float2 cs[];
  griddep_wait();
  griddep_launch_dependents();
  const KvView& kv = p.kv;
  const int D = kv.D, chunks = D / 8;
  const long long tok0 = (long long)blockIdx.x * p.per_cta;
  const int ntok = (int)min((long long)p.per_cta, p.tokens - tok0);
  const int nq = ntok * p.q.heads * chunks, nk = ntok * kv.heads * chunks;
  const int k0 = (nq + 31) & ~31, v0 = k0 + ((nk + 31) & ~31), end = v0 + ((nk + 31) & ~31);
  if (p.half > 0) {
    for (int i = threadIdx.x; i < ntok * p.half; i += kThreads) {
      const long long t = tok0 + i / p.half;
      const long long pos = p.starts[t / p.S] + t % p.S;
      cs[i] = rotary_cos_sin((double)pos, p.inv_freq[i % p.half], p.magnitude);
    }
    __syncthreads();
  }
  for (int it = threadIdx.x; it < end; it += kThreads) {
    const int part = it < k0 ? 0 : it < v0 ? 1 : 2;  // the same in all lanes of a warp
    const int i = it - (part == 0 ? 0 : part == 1 ? k0 : v0);
    const bool there = i < (part == 0 ? nq : nk);
    const int heads = part == 0 ? p.q.heads : kv.heads;
    const int c = i % chunks, th = i / chunks, h = th % heads;
    const int tok = there ? th / heads : 0;
    const long long t = tok0 + tok;
    const int b = (int)(t / p.S), s = (int)(t % p.S);
    const AppendPart& src = part == 0 ? p.q : part == 1 ? p.k : p.v;
    float x[8] = {};
    const T* row = static_cast<const T*>(src.in) + b * src.sb + s * src.ss + (there ? h : 0) * src.sh;
    if (there) {
      load8<T, VEC>(row + c * 8, x);
      if (part < 2 && p.half > 0) rotate8<T, VEC, INTER>(row, c * 8, p.half, cs + tok * p.half, x);
    }
    if (part == 0) {
      if (there)
        *reinterpret_cast<Pack16<8>*>(static_cast<T*>(p.q_out) + (t * heads + h) * D + c * 8) = pack8<T>(x);
      continue;
    }
    const bool is_new = there && (p.counts == nullptr || s < p.counts[b]);
    const long long pos = (long long)p.starts[b] + s;
    const int id = is_new ? kv.page_of(b, pos) : -1;
    if (is_new && id < 0) kv.report(kStatusPage);
    const int token = (int)(pos & (kv.page - 1));
    if (BITS == 16) {
      if (id >= 0)
        *reinterpret_cast<Pack16<8>*>((part == 1 ? kv.k : kv.v) + kv.row16(id, h, token) + c * 16) =
            pack8<T>(x);
      continue;
    }
    uint32_t code[8];
    const uint32_t sm = quantise(x, code);
    if (id < 0) continue;
    const Kv4 lay(D);
    const int NG = lay.groups(), grp = c / 4, t4 = c % 4, r = token % kBlockTokens;
    uint8_t* blk = kv.k + kv.block4(id, h, token);
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
        const uint32_t w = code[4 * n] | code[4 * n + 1] << 4 | code[4 * n + 2] << 8 | code[4 * n + 3] << 12;
        reinterpret_cast<uint16_t*>(blk + lay.v_codes())[(((tp * 8 + g) * 4 + tt) * NG + grp) * 2 + hi] =
            (uint16_t)w;
      }
      if (t4 == 0) {
        uint16_t* vp = reinterpret_cast<uint16_t*>(blk + lay.v_params());
        const int at = (grp * 4 + tt) * 4 + tp * 2 + hi;
        vp[at] = (uint16_t)sm;
        vp[at + 16 * NG] = (uint16_t)(sm >> 16);
      }
    }
  }
}

template <typename T, int VEC, int BITS>
int launch_append(const AppendParams& p, bool interleaved, unsigned grid, size_t smem,
                  cudaStream_t st) {
  const cudaError_t e =
      interleaved ? launch_pdl(fa_kv_append_kernel<T, VEC, true, BITS>, dim3(grid), dim3(kThreads),
                               smem, st, p)
                  : launch_pdl(fa_kv_append_kernel<T, VEC, false, BITS>, dim3(grid), dim3(kThreads),
                               smem, st, p);
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

template <typename T>
int launch_append_t(const AppendParams& p, int vec, bool interleaved, unsigned grid, size_t smem,
                    cudaStream_t st) {
  if (p.kv.bits == 16)
    return vec == 8 ? launch_append<T, 8, 16>(p, interleaved, grid, smem, st)
                    : launch_append<T, 1, 16>(p, interleaved, grid, smem, st);
  return vec == 8 ? launch_append<T, 8, 4>(p, interleaved, grid, smem, st)
                  : launch_append<T, 1, 4>(p, interleaved, grid, smem, st);
}

// ---------------------------------------------------------------- read
struct ReadParams {
  KvView kv;
  const int* lengths;
  void* k_out;  // (batch, max_len, heads, D)
  void* v_out;
  int max_len;
};

__device__ __forceinline__ float2 params_of(uint32_t sm) {
  return make_float2(__half2float(__ushort_as_half((uint16_t)sm)),
                     __half2float(__ushort_as_half((uint16_t)(sm >> 16))));
}

// The cached tokens as contiguous K and V, rows behind a sequence's length
// zero.  Bound by HBM: the cache is read once, K and V written once.  A CTA
// takes one 16-token block of a sequence, all heads; an item is 8 dims of one
// token (of two neighbouring tokens for 4-bit V, whose words hold both), so
// stores are 16 bytes wide and contiguous over a token's heads.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) fa_kv_read_kernel(const ReadParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const KvView& kv = p.kv;
  const int D = kv.D, chunks = D / 8, b = blockIdx.y, first = blockIdx.x * kBlockTokens;
  const int given = p.lengths[b], len = min(kv.clamp_length(given), p.max_len);
  if (kv.bad_length(given) && blockIdx.x == 0 && threadIdx.x == 0) kv.report(kStatusPage);
  const int there = max(0, min(len - first, kBlockTokens));  // tokens of the block to copy
  const int rows = min(p.max_len - first, kBlockTokens);     // tokens of the block to write
  int id = -1;
  if (there > 0) {
    id = kv.page_of(b, first);
    if (id < 0 && threadIdx.x == 0) kv.report(kStatusPage);
  }
  const int token0 = first & (kv.page - 1);
  const int copied = id < 0 ? 0 : there;
  T* k_out = static_cast<T*>(p.k_out) + ((long long)b * p.max_len + first) * kv.heads * D;
  T* v_out = static_cast<T*>(p.v_out) + ((long long)b * p.max_len + first) * kv.heads * D;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const int per_token = kv.heads * chunks;
  if (copied < rows) {  // zero the rest
    for (int i = copied * per_token + threadIdx.x; i < rows * per_token; i += kThreads) {
      reinterpret_cast<uint4*>(k_out)[i] = zero;
      reinterpret_cast<uint4*>(v_out)[i] = zero;
    }
  }
  if (BITS == 16) {
#pragma unroll 4
    for (int i = threadIdx.x; i < copied * per_token; i += kThreads) {
      const int c = i % chunks, h = i / chunks % kv.heads, r = i / per_token;
      const long long at = kv.row16(id, h, token0 + r) + c * 16;
      reinterpret_cast<uint4*>(k_out)[i] = *reinterpret_cast<const uint4*>(kv.k + at);
      reinterpret_cast<uint4*>(v_out)[i] = *reinterpret_cast<const uint4*>(kv.v + at);
    }
    return;
  }
  const Kv4 lay(D);
  const int NG = lay.groups();
  for (int i = threadIdx.x; i < copied * per_token; i += kThreads) {
    const int c = i % chunks, h = i / chunks % kv.heads, r = i / per_token;
    const int grp = c / 4, t4 = c % 4;
    const uint8_t* blk = kv.k + kv.block4(id, h, token0);
    const uint32_t w = reinterpret_cast<const uint32_t*>(blk)[(r * 4 + t4) * NG + grp];
    const float2 sm = params_of(reinterpret_cast<const uint32_t*>(blk + lay.k_params())[r * NG + grp]);
    float x[8];
#pragma unroll
    for (int d = 0; d < 8; ++d)
      x[d] = fmaf(sm.x, (float)(w >> (d / 2 * 4 + d % 2 * 16) & 15u), sm.y);
    *reinterpret_cast<Pack16<8>*>(k_out + (long long)i * 8) = pack8<T>(x);
  }
  const int pairs = (copied + 1) / 2;
  for (int i = threadIdx.x; i < pairs * per_token; i += kThreads) {
    const int c = i % chunks, h = i / chunks % kv.heads, rp = i / per_token;
    const int grp = c / 4, g = c % 4 * 2, tp = rp / 4, tt = rp % 4;
    const uint8_t* blk = kv.k + kv.block4(id, h, token0);
    const uint32_t* vc = reinterpret_cast<const uint32_t*>(blk + lay.v_codes());
    const uint32_t w0 = vc[((tp * 8 + g) * 4 + tt) * NG + grp];
    const uint32_t w1 = vc[((tp * 8 + g + 1) * 4 + tt) * NG + grp];
    const uint16_t* vp = reinterpret_cast<const uint16_t*>(blk + lay.v_params());
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      if (2 * rp + hi >= copied) break;
      const int at = (grp * 4 + tt) * 4 + tp * 2 + hi;
      const float s = __half2float(__ushort_as_half(vp[at]));
      const float m = __half2float(__ushort_as_half(vp[at + 16 * NG]));
      float x[8];
#pragma unroll
      for (int d = 0; d < 8; ++d)
        x[d] = fmaf(s, (float)((d < 4 ? w0 : w1) >> (hi * 16 + d % 4 * 4) & 15u), m);
      *reinterpret_cast<Pack16<8>*>(v_out + ((long long)(2 * rp + hi) * per_token + h * chunks + c) * 8) =
          pack8<T>(x);
    }
  }
}

bool bad_append_part(const fa_sm100_heads& x) {
  return !x.in || x.heads < 1 || (reinterpret_cast<uintptr_t>(x.in) & 1u);
}
bool wide(const fa_sm100_heads& x) {
  return !(reinterpret_cast<uintptr_t>(x.in) & 15u) &&
         !((x.stride_batch | x.stride_seq | x.stride_head) & 7);
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
  AppendParams p = {};
  p.kv = kv_view(cache, page_table, table_width, status);
  if (q) p.q = {q->in, q->stride_batch, q->stride_seq, q->stride_head, q->heads};
  p.k = {k->in, k->stride_batch, k->stride_seq, k->stride_head, k->heads};
  p.v = {v->in, v->stride_batch, v->stride_seq, v->stride_head, v->heads};
  p.q_out = q ? q->out : nullptr;
  p.starts = starts;
  p.counts = counts;
  p.inv_freq = inv_freq;
  p.half = inv_freq ? rotary_dim / 2 : 0;
  p.tokens = (long long)batch * seqlen;
  p.S = seqlen;
  p.magnitude = magnitude;
  const int vec = wide(*k) && wide(*v) && (!q || wide(*q)) ? 8 : 1;
  // whole tokens until every thread has two items
  const long long per_token = (long long)(p.q.heads + 2 * p.k.heads) * (cache->head_dim / 8);
  long long per_cta = 2 * kThreads / per_token;
  if (p.half > 0 && per_cta > kMaxAngles / p.half) per_cta = kMaxAngles / p.half;
  if (per_cta < 1) per_cta = 1;
  p.per_cta = (int)per_cta;
  const long long grid = (p.tokens + per_cta - 1) / per_cta;
  if (grid > 2147483647LL) return FA_ERR_ARG;
  const size_t smem = (size_t)per_cta * p.half * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == FA_DTYPE_BF16
             ? launch_append_t<__nv_bfloat16>(p, vec, interleaved != 0, (unsigned)grid, smem, st)
             : launch_append_t<__half>(p, vec, interleaved != 0, (unsigned)grid, smem, st);
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
  ReadParams p;
  p.kv = kv_view(cache, page_table, table_width, status);
  p.lengths = lengths;
  p.k_out = k_out;
  p.v_out = v_out;
  p.max_len = max_len;
  const dim3 grid((unsigned)(((long long)max_len + kBlockTokens - 1) / kBlockTokens), (unsigned)batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (cache->dtype == FA_DTYPE_BF16)
    e = cache->bits == 16
            ? launch_pdl(fa_kv_read_kernel<__nv_bfloat16, 16>, grid, dim3(kThreads), 0, st, p)
            : launch_pdl(fa_kv_read_kernel<__nv_bfloat16, 4>, grid, dim3(kThreads), 0, st, p);
  else
    e = cache->bits == 16 ? launch_pdl(fa_kv_read_kernel<__half, 16>, grid, dim3(kThreads), 0, st, p)
                          : launch_pdl(fa_kv_read_kernel<__half, 4>, grid, dim3(kThreads), 0, st, p);
  return e == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}
