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
  AppendPart part[3];  // q, k, v
  void* q_out;
  const int* starts;
  const int* counts;       // null: every token is new
  const double* inv_freq;  // null: no rotation
  int S, half, per_cta, per_seq, page_shift, chunk_shift;
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
// largest fp16.  The quotient (x - m) / s is the correctly rounded one
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
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack2(v[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]),
                    Elem<T>::pack2(x[4], x[5]), Elem<T>::pack2(x[6], x[7]));
}

// Where the angle of pair i stands: the 8 angles of a thread's dims are `half / 8`
// apart, so that neighbouring threads read neighbouring words (WIDE: half % 8
// == 0); interleaved pairs, of which a thread has 4, likewise.
template <bool INTER, bool WIDE>
__device__ __forceinline__ int angle_at(int i, int half) {
  constexpr int N = INTER ? 4 : 8;
  return WIDE ? i % N * (half / N) + i / N : i;
}

// Rotates the 8 dims e.. of a row (the thread's own values in x, WIDE: those of
// the partner dims in y).
template <typename T, bool INTER, bool WIDE>
__device__ __forceinline__ void rotate8(const T* row, int e, int half, const float2* cs,
                                        float (&x)[8], float (&y)[8]) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (WIDE || e + i < 2 * half) {
        const float2 w = cs[angle_at<INTER, WIDE>((e + i) / 2, half)];
        const float a = x[i], b = x[i + 1];
        x[i] = a * w.x - b * w.y;
        x[i + 1] = b * w.x + a * w.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = e + i;
      if (!WIDE) {
        if (d >= 2 * half) break;
        y[i] = Elem<T>::value(reinterpret_cast<const uint16_t*>(row)[d < half ? d + half : d - half]);
      }
      const bool first = d < half;
      const float2 w = cs[angle_at<INTER, WIDE>(first ? d : d - half, half)];
      x[i] = x[i] * w.x + (first ? -y[i] : y[i]) * w.y;
    }
  }
}

// New tokens into the cache.  Bound by HBM for prompts (every input is read
// once, every output written once) and by latency for single tokens: one
// launch does the rotation of q and k, the page lookup and both writes.
// A CTA takes whole tokens of one sequence; it makes their cosines and sines
// and finds their places in the cache once for all heads.  The rows are the
// heads of q, k and v of each token, D/8 threads to a row; a thread holds 8
// consecutive dims (the half layout reads the partner dims a second time, from
// L1) and steps down the rows with additions alone.  The 4 lanes that hold a
// group of 32 dims reduce its minimum and maximum by shuffles.
// WIDE: 16-byte loads, and rotated dims that end at a thread's border.
template <typename T, bool INTER, int BITS, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) fa_kv_append_kernel(const AppendParams p) {
  extern __shared__ float2 cs[];
  griddep_wait();
  griddep_launch_dependents();
  const KvView& kv = p.kv;
  const int b = blockIdx.x / p.per_seq, s0 = (blockIdx.x - b * p.per_seq) * p.per_cta;
  const int ntok = min(p.per_cta, p.S - s0);
  int* places = reinterpret_cast<int*>(cs + p.per_cta * p.half);  // row of head 0, or -1
  const int hq = p.part[0].heads, hk = kv.heads, heads = hq + 2 * hk;
  const int c = threadIdx.x & ((1 << p.chunk_shift) - 1), e = c * 8;
  const int row = threadIdx.x >> p.chunk_shift, step = kThreads >> p.chunk_shift;
  const int step_tok = step / heads, step_h = step - step_tok * heads;
  int tok = row / heads, h = row - tok * heads;
  const bool turning = e < 2 * p.half;

  const long long first = (long long)p.starts[b] + s0;
  for (int i = threadIdx.x; i < ntok; i += kThreads) {
    int at = -1;
    if (p.counts == nullptr || s0 + i < p.counts[b]) {
      const long long pos = first + i;
      const int id = kv.page_of(b, pos, p.page_shift);
      if (id < 0)
        kv.report(kStatusPage);
      else
        at = ((id * hk) << p.page_shift) | ((int)pos & (kv.page - 1));
    }
    places[i] = at;
  }

  bool filled = false;
  // the same number of rounds for all lanes of a warp: the warp's first row leads
  int lead_tok = (int)((threadIdx.x & ~31u) >> p.chunk_shift) / heads;
  int lead_h = (int)((threadIdx.x & ~31u) >> p.chunk_shift) - lead_tok * heads;
  while (lead_tok < ntok || !filled) {
    uint4 own[2], other[2];
    int rt[2], rh[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      rt[u] = tok;
      rh[u] = h;
      if (WIDE && tok < ntok) {
        const int part = h < hq ? 0 : h < hq + hk ? 1 : 2;
        const AppendPart& src = p.part[part];
        const T* at = static_cast<const T*>(src.in) + b * src.sb + (s0 + tok) * src.ss +
                      (h - (part == 0 ? 0 : part == 1 ? hq : hq + hk)) * src.sh;
        own[u] = *reinterpret_cast<const uint4*>(at + e);
        if (!INTER && turning && part < 2)
          other[u] = *reinterpret_cast<const uint4*>(at + (e < p.half ? e + p.half : e - p.half));
      }
      tok += step_tok;
      h += step_h;
      if (h >= heads) {
        h -= heads;
        ++tok;
      }
      lead_tok += step_tok;
      lead_h += step_h;
      if (lead_h >= heads) {
        lead_h -= heads;
        ++lead_tok;
      }
    }
    if (!filled) {
      for (int i = threadIdx.x; i < ntok * p.half; i += kThreads) {
        const int at = i / p.half, f = i - at * p.half;
        cs[at * p.half + angle_at<INTER, WIDE>(f, p.half)] =
            rotary_cos_sin((double)(first + at), p.inv_freq[f], p.magnitude);
      }
      __syncthreads();
      filled = true;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool there = rt[u] < ntok;
      const int part = rh[u] < hq ? 0 : rh[u] < hq + hk ? 1 : 2;
      const int hp = rh[u] - (part == 0 ? 0 : part == 1 ? hq : hq + hk);
      float x[8] = {}, y[8];
      if (there) {
        const AppendPart& src = p.part[part];
        const T* at = static_cast<const T*>(src.in) + b * src.sb + (s0 + rt[u]) * src.ss + hp * src.sh;
        if (WIDE) {
          unpack8<T>(own[u], x);
          if (!INTER && turning) unpack8<T>(other[u], y);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = Elem<T>::value(reinterpret_cast<const uint16_t*>(at)[e + i]);
        }
        if (part < 2 && turning) rotate8<T, INTER, WIDE>(at, e, p.half, cs + rt[u] * p.half, x, y);
        if (part == 0)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) +
                                    (((long long)b * p.S + s0 + rt[u]) * hq + hp) * kv.D + e) = pack8<T>(x);
      }
      const int place = there && part > 0 ? places[rt[u]] : -1;
      const int at = place + (hp << p.page_shift);  // row of the cache
      if (BITS == 16) {
        if (place >= 0)
          *reinterpret_cast<uint4*>((part == 1 ? kv.k : kv.v) + ((long long)at * kv.D + e) * 2) = pack8<T>(x);
        continue;
      }
      if (!__any_sync(0xffffffffu, place >= 0)) continue;
      uint32_t code[8];
      const uint32_t sm = quantise(x, code);
      if (place < 0) continue;
      const Kv4 lay(kv.D);
      const int NG = lay.groups(), grp = c / 4, t4 = c % 4, r = at % kBlockTokens;
      uint8_t* blk = kv.k + (long long)(at / kBlockTokens) * lay.bytes();
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
          const int i = (grp * 4 + tt) * 4 + tp * 2 + hi;
          vp[i] = (uint16_t)sm;
          vp[i + 16 * NG] = (uint16_t)(sm >> 16);
        }
      }
    }
  }
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
int launch_append_t(const AppendParams& p, bool is_wide, bool interleaved, unsigned grid, size_t smem,
                    cudaStream_t st) {
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
  int max_len, page_shift, chunk_shift;
};

// 4-bit codes to values: a nibble pair masked out of its word is two fp16
// subnormals (c 2^-24 from bits 0..3, c 2^-20 from bits 4..7), which convert
// exactly; `s24` and `s20` are the scale times 2^24 and 2^20.
__device__ __forceinline__ float2 pair_of(uint32_t masked) {
  return __half22float2(*reinterpret_cast<const __half2*>(&masked));
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
  const int D = kv.D, b = blockIdx.y, first = blockIdx.x * kBlockTokens;
  const int given = p.lengths[b], len = min(kv.clamp_length(given), p.max_len);
  if (kv.bad_length(given) && blockIdx.x == 0 && threadIdx.x == 0) kv.report(kStatusPage);
  const int there = max(0, min(len - first, kBlockTokens));  // tokens of the block to copy
  const int rows = min(p.max_len - first, kBlockTokens);     // tokens of the block to write
  int id = -1;
  if (there > 0) {
    id = kv.page_of(b, first, p.page_shift);
    if (id < 0 && threadIdx.x == 0) kv.report(kStatusPage);
  }
  const int copied = id < 0 ? 0 : there;
  uint4* k_out = reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + ((long long)b * p.max_len + first) * kv.heads * D);
  uint4* v_out = reinterpret_cast<uint4*>(static_cast<T*>(p.v_out) + ((long long)b * p.max_len + first) * kv.heads * D);
  const int per_token = kv.heads << p.chunk_shift;
  if (copied < rows) {  // zero the rest
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i = copied * per_token + threadIdx.x; i < rows * per_token; i += kThreads) {
      k_out[i] = zero;
      v_out[i] = zero;
    }
  }
  // row of the cache: head 0, the block's first token
  const int at0 = id < 0 ? 0 : ((id * kv.heads) << p.page_shift) | (first & (kv.page - 1));
  const int c = threadIdx.x & ((1 << p.chunk_shift) - 1), row = threadIdx.x >> p.chunk_shift;
  const int step = kThreads >> p.chunk_shift;
  const int step_tok = step / kv.heads, step_h = step - step_tok * kv.heads;
  const int tok0 = row / kv.heads, h0 = row - tok0 * kv.heads;
  auto next = [&](int& tok, int& h) {
    tok += step_tok;
    h += step_h;
    if (h >= kv.heads) {
      h -= kv.heads;
      ++tok;
    }
  };
  auto out_at = [&](int tok, int h) { return tok * per_token + (h << p.chunk_shift) + c; };
  if (BITS == 16) {
    const uint4* ks = reinterpret_cast<const uint4*>(kv.k);
    const uint4* vs = reinterpret_cast<const uint4*>(kv.v);
    int tok = tok0, h = h0;
    while (tok < copied) {
      uint4 x[4], y[4];
      int o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        o[u] = -1;
        if (tok < copied) {
          const long long at = ((long long)(at0 + (h << p.page_shift) + tok) << p.chunk_shift) + c;
          x[u] = ks[at];
          y[u] = vs[at];
          o[u] = out_at(tok, h);
        }
        next(tok, h);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (o[u] >= 0) {
          k_out[o[u]] = x[u];
          v_out[o[u]] = y[u];
        }
    }
    return;
  }
  const Kv4 lay(D);
  const int NG = lay.groups(), grp = c / 4, t4 = c % 4;
  auto block = [&](int h) {
    return kv.k + (long long)((at0 + (h << p.page_shift)) / kBlockTokens) * lay.bytes();
  };
  {
    int r = tok0, h = h0;
    while (r < copied) {
      uint32_t w[2], sm[2];
      int o[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        o[u] = -1;
        if (r < copied) {
          const uint8_t* blk = block(h);
          w[u] = reinterpret_cast<const uint32_t*>(blk)[(r * 4 + t4) * NG + grp];
          sm[u] = reinterpret_cast<const uint32_t*>(blk + lay.k_params())[r * NG + grp];
          o[u] = out_at(r, h);
        }
        next(r, h);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (o[u] < 0) continue;
        const float2 par = pair_of(sm[u]);
        const float s24 = par.x * 0x1p24f, s20 = par.x * 0x1p20f;
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = pair_of((i < 2 ? w[u] : w[u] >> 8) & (i % 2 ? 0x00F000F0u : 0x000F000Fu));
          x[2 * i] = fmaf(i % 2 ? s20 : s24, f.x, par.y);
          x[2 * i + 1] = fmaf(i % 2 ? s20 : s24, f.y, par.y);
        }
        k_out[o[u]] = pack8<T>(x);
      }
    }
  }
  const int pairs = (copied + 1) / 2, g = t4 * 2;
  int rp = tok0, h = h0;
  while (rp < pairs) {
    const uint8_t* blk = block(h);
    const int tp = rp / 4, tt = rp % 4;
    const uint32_t* vc = reinterpret_cast<const uint32_t*>(blk + lay.v_codes());
    const uint32_t w0 = vc[((tp * 8 + g) * 4 + tt) * NG + grp];
    const uint32_t w1 = vc[((tp * 8 + g + 1) * 4 + tt) * NG + grp];
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + lay.v_params()) + (grp * 4 + tt) * 2 + tp;
    const float2 s = pair_of(vp[0]), m = pair_of(vp[8 * NG]);  // of both tokens
    const int o = out_at(2 * rp, h);
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = i < 4 ? w0 : w1;
      const float2 f = pair_of((i % 4 < 2 ? w : w >> 8) & (i % 2 ? 0x00F000F0u : 0x000F000Fu));
      x[0][i] = fmaf(s.x * (i % 2 ? 0x1p20f : 0x1p24f), f.x, m.x);
      x[1][i] = fmaf(s.y * (i % 2 ? 0x1p20f : 0x1p24f), f.y, m.y);
    }
    v_out[o] = pack8<T>(x[0]);
    if (2 * rp + 1 < copied) v_out[o + per_token] = pack8<T>(x[1]);
    next(rp, h);
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
  const bool is_wide = wide(*k) && wide(*v) && (!q || wide(*q)) &&
                       (interleaved ? p.half % 4 : p.half % 8) == 0;
  // whole tokens until every thread has four items
  const long long per_token = (long long)(p.part[0].heads + 2 * k->heads) * (cache->head_dim / 8);
  long long per_cta = 4 * kThreads / per_token;
  if (p.half > 0 && per_cta > kMaxAngles / p.half) per_cta = kMaxAngles / p.half;
  if (per_cta > seqlen) per_cta = seqlen;
  if (per_cta < 1) per_cta = 1;
  p.per_cta = (int)per_cta;
  p.per_seq = (int)((seqlen + per_cta - 1) / per_cta);
  const long long grid = (long long)p.per_seq * batch;
  if (grid > 2147483647LL) return FA_ERR_ARG;
  const size_t smem = (size_t)per_cta * (p.half * sizeof(float2) + sizeof(int));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == FA_DTYPE_BF16
             ? launch_append_t<__nv_bfloat16>(p, is_wide, interleaved != 0, (unsigned)grid, smem, st)
             : launch_append_t<__half>(p, is_wide, interleaved != 0, (unsigned)grid, smem, st);
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
  p.page_shift = log2_of(cache->page_size);
  p.chunk_shift = log2_of(cache->head_dim / 8);
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
