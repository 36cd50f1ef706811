// Attention of a few query tokens per sequence over the paged key/value cache
// (fa_kv_cache.cuh): o_i = sum_j softmax_j(scale q_i . k_j) v_j over the cached
// tokens j below row i's limit.
//
// Bound by HBM: the cache is read once, 4 rows D flops a token and K/V head
// (rows: the query heads that share it times the query tokens), so at 8 rows
// 16 flops a 16-bit byte.  That needs no 128-row tensor-core tiles; what it
// needs is loads in flight and few instructions per cached byte:
//
// * Work split.  The tiles (4 warps x U blocks of 16 tokens) of all (sequence,
//   K/V head, row block) segments form one list, cut into equal contiguous
//   shares, one per CTA, whatever the lengths are.  The lengths stay on the
//   device: each CTA sums them itself.  A segment inside one share is finished
//   there; one that crosses shares leaves fp32 partial results (maximum, sum,
//   O) that fa_decode_merge_kernel joins in a fixed order.
// * Each warp streams its own blocks through a private ring of bulk copies (TMA
//   tiles for 16-bit pages, plain bulk copies for 4-bit blocks) with its own
//   mbarriers, running maximum, sum and O, across segment borders; the warps
//   meet only at the end of a segment.
// * The products run transposed, S^T = K Q^T and O^T += V^T P^T (mma.sync
//   m16n8k16): 16 tokens, or dims, are the rows and 8 query rows the columns, so
//   nothing is wasted at 8 rows; the running maximum of a query row is per
//   lane column in S^T and in O^T alike, and P^T becomes the second product's
//   operand by one 8x8 transpose (movmatrix) each.
// * 4-bit codes are used as they are: a nibble masked out of its word is the
//   fp16 subnormal c 2^-24 (bits 0..3) or c 2^-20 (bits 4..7), exact in the
//   matrix instruction, so 8 codes cost one shift and four ANDs (the integer pipe
//   is the busiest: 45 % at 2 x 131072 tokens).  The power of two goes into q (K) or
//   the final factor (V).  Summing V's even dims as whole bytes 16 c1 + c0 and parting
//   them at the end saves an AND in five and 5 % of the time, but the matrix
//   instruction's sums are truncated, and 16 c1 is 17 times the sum that is wanted:
//   the error against 64 bits grew from 2.1e-4 to 2.6e-4 there.  Scales and minima enter
//   outside: S = sum_g s_g (c_g . q_g) + m_g sum(q_g), with the second sum as
//   one more matrix instruction on the parameter words themselves (q's group
//   sums as an fp16 head and tail), and O = sum_t (p_t s_t) c_t + p_t m_t.
//
// Rounded to fewer than 32 bits: p to the operand type (fp16 times 2^12, see kLift;
// bf16 as it is, with fp32's range), at 4 bits its product with the token's scale to fp16
// (the scale relative to a power of two near the largest one, see `se`), and q to fp16 at
// 4 bits after a power of two per row (exact but for elements below 2^-24 of the
// largest).
//
// Measured on one B200 (replayed): 64 sequences of 5 to 8192 tokens, 32 / 8 heads of
// 128, 16-bit 175 us (6.1 TB/s of the cache), 96 such at 4 bits 108 us (4.7 TB/s);
// two of 100003 and 131072 tokens at 4 bits 61 us, of which 48 stream at 6.2 TB/s (two
// of 131072 67 us, of 262144 121) and 13 are fixed: lengths, pages and the first copy
// follow one another, and the last tile, the join of the warps and the second launch.
// A CTA holds 4 warps, an SM two CTAs: 12 or 16 warps an SM with 2 blocks a tile were
// slower (69 and 76 against 64 us for the two long ones), as a tile's fixed steps
// then count twice.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "fa_kernels.h"
#include "fa_kv_cache.cuh"
#include "fast_div.cuh"
#include "sm100_ptx.cuh"

namespace fa_sm100 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// A maximum is left as it is while no score is more than kSlack (in log2) above it: the
// probabilities then reach 4.
constexpr float kSlack = 2.f;
// Probabilities are taken times 2^kLift where they become 16-bit fp16 operands: they
// reach 2^14 and are normal numbers down to 2^-26 of the largest (unlifted, 2^-14: of
// 70000 tokens 18 below one in score a fifth of their part of the output was lost).
constexpr float kLift = 12.f;
// From 2^kFar on (in log2) a maximum is off the product that it was rounded from, and that
// the fused subtraction uses, by up to 1 and more, and the probabilities would leave fp16:
// the row's scores are then divided by the power of two that brings the maximum below
// 2^kFar.  (Gaps shrink with them, those below 20 2^-23 of the maximum to where they
// count: less than the sums of products are off, (D + 8) 2^-22.)
constexpr int kFar = 24;
constexpr float kLn2 = 0.69314718055994531f;

// Per-instantiation constants.
// Column blocks of 8 query rows that a CTA's registers hold.
constexpr int max_nt(int D) { return D <= 64 ? 4 : 2; }

// Blocks of a warp per tile, stages of its ring, CTAs per SM.
constexpr int blocks_of(int D, int bits, int nt) {
  return bits == 16 ? (D == 128 ? 1 : 2) : nt == 1 ? 4 : 2;
}
constexpr int stages_of(int D, int bits, int nt) {
  return bits == 16 ? 3 : D == 128 ? (nt == 1 ? 2 : 4) : 4;
}
constexpr int kCtas = 2;
// The start and end of a segment (its q, the join of the warps) take a CTA about
// as long as so many tiles, so the list has that many empty places behind each
// segment's tiles and shares with many short segments hold fewer tiles.  96
// sequences of 5 to 8192 tokens at 4 bits (tiles of 256): 137, 114, 108, 111 us
// with 0, 1, 2, 4 places; 24 sequences of 5 query tokens (tiles of 128): 46, 41,
// 37, 36 us; 64 sequences at 16 bits (tiles of 64): 174.4, 173.6, 173.1, 173.9 us.
constexpr int cost_of(int D, int bits, int nt) {
  return bits == 4 ? 512 / (kWarps * blocks_of(D, bits, nt) * 16) : 2;
}

template <int D, int BITS, int NT>
struct Cfg {
  static constexpr int kU = blocks_of(D, BITS, NT);
  static constexpr int kBlockBytes = BITS == 16 ? 64 * D : 20 * D;
  static constexpr int kStageBytes = kU * kBlockBytes;
  static constexpr int kStages = stages_of(D, BITS, NT);
  static constexpr int kTile = kWarps * kU * kBlockTokens;  // tokens
  static constexpr int kCost = cost_of(D, BITS, NT);
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMiscBytes = NT <= 2 ? 512 : 640;  // barriers and small shared variables
  static constexpr int kJoinStride = D + 4;  // floats of a row in the join buffer
  // The warps join all 8 rows of a column block at once, or 4 where there is no room.
  static constexpr int kJoinRows =
      kCtas * (kRingBytes + kWarps * 8 * kJoinStride * 4 + kMiscBytes + 1024) <= 228 * 1024 ? 8 : 4;
  static constexpr int kJoinBytes = kWarps * kJoinRows * kJoinStride * 4;
  static constexpr int kSmem = kRingBytes + kJoinBytes + kMiscBytes;
  static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
  static constexpr int kGroups = D / 32;
};

struct DecodeParams {
  KvView kv;
  const void* q;       // (B, Sq, H, D)
  void* out;           // (B, Sq, H, D)
  float* lse;          // (B, H, Sq) or null
  const int* lengths;  // (B)
  const int* starts;   // (B) or null: length - Sq
  FastDiv grid_div, group_div, rb_div, segs_div;
  float* part_o;       // (2 * grid, ROWS, D)
  float2* part_ml;     // (2 * grid, ROWS): maximum (log2 domain), sum
  int B, Sq, H, group, row_blocks, causal, page_shift, bf16;
  int negate;
  int whole;   // a share is whole segments: those that begin in it
  int direct;  // and CTA i's is segment i
  int skip_copy;  // test hook: the first CTA's first block is not brought
  float scale_log2;  // |scale| log2 e, above 0; `negate`: the scale is negative (q's sign changes)
  unsigned long long timeout_ns;
};

// N words of shared memory as one load.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* at, uint32_t (&w)[N]) {
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
    w[0] = *reinterpret_cast<const uint32_t*>(at);
  }
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && Elem<T>::kIdescAB == 0) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// The same with zero to add to.
template <typename T>
__device__ __forceinline__ void mma16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  static_assert(Elem<T>::kIdescAB == 0, "fp16 operands");
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float low_half(uint32_t w) {
  return __half2float(__ushort_as_half((uint16_t)w));
}

// Position in the tile list.
struct Cursor {
  int b, h, rb, tt, nt, len;  // sequence, K/V head, row block, tile of nt (nt: behind them), length
};

template <int TILE>
__device__ __forceinline__ int tiles_of(int len) {
  const int n = (len + TILE - 1) / TILE;
  return n < 1 ? 1 : n;  // a sequence without tokens has one tile, which writes its zeros
}

// The list's places cut into shares: the first `more` hold each + 1, the others
// `each`.
struct Shares {
  unsigned total, each, more;
  __device__ __forceinline__ unsigned begin(unsigned c) const { return c * each + min(c, more); }
  __device__ __forceinline__ unsigned of(unsigned place) const {
    const unsigned cut = more * (each + 1);
    return place < cut ? place / (each + 1) : more + (place - cut) / each;
  }
};

// Where a share begins: the sequence that holds its first place, the places
// before that sequence, its tiles and length.
struct Spot {
  unsigned before;
  int b, len;
};

// Sums the places of all sequences and finds the first place of a share.  All
// threads of the CTA take part; each looks at the sequences of its own.
template <int TILE, int COST>
__device__ __forceinline__ Shares locate(const DecodeParams& p, int segs, unsigned share, Spot& spot,
                                         unsigned* warp_sum) {
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int chunk = (p.B + kThreads - 1) / kThreads;
  const int b0 = min(tid * chunk, p.B), b1 = min(b0 + chunk, p.B);
  auto places = [&](int len) { return (unsigned)(tiles_of<TILE>(len) + COST) * segs; };
  unsigned mine = 0;
  int len = 0;
  for (int b = b0; b < b1; ++b) {
    len = p.kv.clamp_length(p.lengths[b]);
    mine += places(len);
  }
  unsigned before = mine;  // inclusive scan
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const unsigned o = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += o;
  }
  if (lane == 31) warp_sum[w] = before;
  if (tid == 0) spot = {0, 0, 0};  // a share behind the list's end has no first place
  __syncthreads();
  Shares sh = {};
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) before += warp_sum[i];
    sh.total += warp_sum[i];
  }
  sh.each = p.grid_div.div(sh.total);
  sh.more = sh.total - sh.each * p.grid_div.d;
  const unsigned want = sh.begin(share);
  unsigned at = before - mine;
  if (want >= at && want < before) {
    for (int b = b0; b < b1; ++b) {
      if (chunk > 1) len = p.kv.clamp_length(p.lengths[b]);
      const unsigned n = places(len);
      if (want < at + n) {
        spot = {at, b, len};
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  return sh;
}

// 8 dims of a finished row: out = x / sum, and the row's log-sum-exp.
template <int D>
__device__ __forceinline__ void write_row(const DecodeParams& p, int b, int h, int rr, int d,
                                          float top, float sum, const float (&x)[8]) {
  const int qpos = (int)p.group_div.div(rr), hq = h * p.group + (rr - qpos * p.group);
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = p.bf16 ? Elem<__nv_bfloat16>::pack2(x[2 * j] * inv, x[2 * j + 1] * inv)
                  : Elem<__half>::pack2(x[2 * j] * inv, x[2 * j + 1] * inv);
    if (p.kv.bits == 4 && !p.bf16) w[j] = most_half2(w[j]);
  }
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) +
                            (((long long)b * p.Sq + qpos) * p.H + hq) * D + d) =
      make_uint4(w[0], w[1], w[2], w[3]);
  if (p.lse && d == 0)
    p.lse[((long long)b * p.H + hq) * p.Sq + qpos] =
        sum == 0.f ? INFINITY : (top + log2f(sum)) * kLn2;
}

// T: the element type of 16-bit pages; 4-bit codes are multiplied as fp16
// whatever q's type is.
template <typename T, int D, int BITS, int NT>
__global__ void __launch_bounds__(kThreads, kCtas)
    fa_decode_kernel(const DecodeParams p, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v) {
  using C = Cfg<D, BITS, NT>;
  using M = T;  // operand type
  constexpr int U = C::kU, NS = C::kStages, ROWS = 8 * NT, NG = BITS == 4 ? C::kGroups : 1;
  constexpr int KSTEPS = D / 16;
  constexpr float LIFT = Elem<M>::kIdescAB == 0 ? kLift : 0.f;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  struct Misc {
    uint64_t bars[kWarps * NS];
    Spot spot;
    unsigned warp_sum[kWarps];
    float2 join_ml[kWarps][8];
    uint8_t cut[kWarps][ROWS];  // powers of two that the rows' scores were divided by
    int abort_flag;
  };
  static_assert(sizeof(Misc) <= C::kMiscBytes, "small shared variables");
  float* join = reinterpret_cast<float*>(smem_raw + C::kRingBytes);
  Misc& sh = *reinterpret_cast<Misc*>(smem_raw + C::kRingBytes + C::kJoinBytes);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t my_ring = smem_u32(smem_raw) + warp * NS * C::kStageBytes;
  const uint32_t my_bars = smem_u32(sh.bars + warp * NS);

  if (tid == 0) sh.abort_flag = 0;
  if (lane < NS) mbar_init(my_bars + lane * 8, U);
  fence_barrier_init();
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();

  const int segs = p.kv.heads * p.row_blocks;  // segments of a sequence
  const WaitCtx wait{&sh.abort_flag, p.kv.status, p.timeout_ns};
  int left;  // places of the share
  // To the next tile; returns the places of the list that this takes.
  auto advance = [&](Cursor& c) {
    if (++c.tt < c.nt) return 1;
    const int places = 1 + C::kCost + c.nt - c.tt;
    c.tt = 0;
    if (++c.rb < p.row_blocks) return places;
    c.rb = 0;
    if (++c.h < p.kv.heads) return places;
    c.h = 0;
    if (++c.b >= p.B) return places;
    c.len = p.kv.clamp_length(p.lengths[c.b]);
    c.nt = tiles_of<C::kTile>(c.len);
    return places;
  };
  Cursor cur;
  if (p.direct) {
    cur.b = (int)p.segs_div.div(blockIdx.x);
    const unsigned hr = blockIdx.x - cur.b * p.segs_div.d;
    cur.len = p.kv.clamp_length(p.lengths[cur.b]);
    cur.nt = tiles_of<C::kTile>(cur.len);
    cur.h = (int)p.rb_div.div(hr);
    cur.rb = (int)hr - cur.h * p.row_blocks;
    cur.tt = 0;
    left = cur.nt;
    __syncthreads();
  } else {
    const Shares shares = locate<C::kTile, C::kCost>(p, segs, blockIdx.x, sh.spot, sh.warp_sum);  // synchronises
    left = (int)(shares.begin(blockIdx.x + 1) - shares.begin(blockIdx.x));
    if (left == 0) return;
    cur.b = sh.spot.b;
    cur.len = sh.spot.len;
    cur.nt = tiles_of<C::kTile>(cur.len);
    const unsigned in = shares.begin(blockIdx.x) - sh.spot.before, places = cur.nt + C::kCost;
    const unsigned hr = in / places;
    cur.tt = (int)(in - hr * places);
    cur.h = (int)p.rb_div.div(hr);
    cur.rb = (int)hr - cur.h * p.row_blocks;
    if (cur.tt >= cur.nt || (p.whole && cur.tt > 0)) {  // on to the next segment
      const int over = (int)places - cur.tt;
      cur.tt = cur.nt - 1;
      advance(cur);
      left -= over;
      if (left <= 0) return;
    }
  }

  // ---- producer: lane u < U brings block u of the warp's share of a tile
  // (a whole segment that begins in the share is brought to its end)
  Cursor pc = cur;
  int to_issue = left;
  auto more_to_issue = [&]() { return to_issue > 0 || (p.whole && pc.tt > 0); };
  constexpr uint32_t ALL = (1u << U) - 1u;
  uint32_t ok_bits = 0;    // U bits for each stage: blocks that hold tokens
  uint32_t in_flight = 0;  // stages whose copies have not been waited for
  uint32_t odd = ~0u;      // stages whose last copies complete an odd phase
  auto block_token = [&](const Cursor& c, int u) {
    return c.tt * C::kTile + (u * kWarps + warp) * kBlockTokens;  // a short tile's blocks go to all warps
  };
  auto look_up = [&](const Cursor& c, bool wanted) {  // page of the lane's block, if it has one
    const int tok = block_token(c, lane);
    return wanted && lane < U && tok < c.len
               ? p.kv.table[(long long)c.b * p.kv.table_width + (tok >> p.page_shift)]
               : 0;
  };
  auto issue = [&](int stage, int next_id) {
    const bool tokens = lane < U && block_token(pc, lane) < pc.len, ok = tokens && !p.kv.bad_page(next_id);
    if (lane < U) {
      const uint32_t bar = my_bars + stage * 8;
      if (tokens && !ok) p.kv.report(kStatusPage);
      if (ok) {
        // block (16-bit: row) of the cache, below 2^31
        const int at = (((next_id * p.kv.heads + pc.h) << p.page_shift) |
                        (block_token(pc, lane) & (p.kv.page - 1)));
        const uint32_t dst = my_ring + stage * C::kStageBytes + lane * C::kBlockBytes;
        mbar_arrive_expect_tx(bar, C::kBlockBytes);
        if (p.skip_copy && blockIdx.x == 0 && tid == 0 && to_issue == left) {
          // the barrier waits for bytes that do not come
        } else if constexpr (BITS == 4) {
          bulk_load(dst, p.kv.k + (long long)(at / kBlockTokens) * C::kBlockBytes, C::kBlockBytes, bar);
        } else {
#pragma unroll
          for (int x = 0; x < D; x += 64) {
            tma_load_2d(dst + x * 32, &tm_k, bar, x, at);
            tma_load_2d(dst + 32 * D + x * 32, &tm_v, bar, x, at);
          }
        }
      } else {
        mbar_arrive(bar);
      }
    }
    ok_bits = (ok_bits & ~(ALL << stage * U)) | (__ballot_sync(0xffffffffu, ok) & ALL) << stage * U;
    in_flight |= 1u << stage;
    odd ^= 1u << stage;
    to_issue -= advance(pc);
  };

  // ---- consumer state
  uint32_t raw[NT][KSTEPS][2];  // q as it is loaded
  uint32_t qf[NT][KSTEPS][2];   // q as the second operand of S^T
  uint32_t qsum[NT][2];         // 4-bit: (0, head), (0, tail) of group t's sum
  float f[NT][2];               // factor of a score to the log2 domain, per column (above 0)
  int lim[NT][2];               // tokens that a column's query row sees
  int col_q[NT][2];             // query token of a column's row; -1: none
  float o[KSTEPS][NT][4], om[NT][4], l[NT][2];
  // 4-bit: exponent field of the largest scale of V so far; scales enter the products
  // times 2^(15 - se), below 2, and O is kept in that unit.  (As they were, products of
  // small values or of a long tail were subnormal or 0 in fp16, up to a fifth of the
  // output.  96 sequences of 5 to 8192 tokens 110 -> 114 us.)
  uint32_t se = 0;
  bool cuts = false;            // some row's scores were divided
  float mf[NT][2];              // running maximum in the log2 domain
  int min_lim = 0, max_lim = 0, qp_first = 0, qp_last = 0, start = 0;

  auto limit_of = [&](int qpos) {
    if (!p.causal) return cur.len;
    const long long n = (long long)start + qpos + 1;
    return n < 0 ? 0 : n < cur.len ? (int)n : cur.len;
  };

  auto load_q = [&](const Cursor& c) {
    const int rows = p.Sq * p.group;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int rr = c.rb * ROWS + n * 8 + g;
      const bool there = rr < rows;
      const int qpos = there ? (int)p.group_div.div(rr) : 0, hq = c.h * p.group + (there ? rr - qpos * p.group : 0);
      const uint16_t* src = static_cast<const uint16_t*>(p.q) + (((long long)c.b * p.Sq + qpos) * p.H + hq) * D;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            raw[n][k][i] = there ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 * i + 2 * t) : 0u;
      } else {
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (there) w = *reinterpret_cast<const uint4*>(src + 32 * grp + 8 * t);
          raw[n][2 * grp][0] = w.x;
          raw[n][2 * grp][1] = w.y;
          raw[n][2 * grp + 1][0] = w.z;
          raw[n][2 * grp + 1][1] = w.w;
        }
      }
    }
  };

  // Limits, sums and q of the segment at `cur`, whose q load_q has read.
  auto begin_segment = [&]() {
    const int rb = cur.rb, rows = p.Sq * p.group;
    start = p.starts ? p.starts[cur.b] : cur.len - p.Sq;
    qp_first = (int)p.group_div.div(rb * ROWS);
    qp_last = (int)p.group_div.div(min(rows, (rb + 1) * ROWS) - 1);
    min_lim = limit_of(qp_first);
    max_lim = limit_of(qp_last);
    se = 0;
    cuts = false;
    if (lane < ROWS) sh.cut[warp][lane] = 0;
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = rb * ROWS + n * 8 + 2 * t + i;
        col_q[n][i] = rr < rows ? (int)p.group_div.div(rr) : -1;
        lim[n][i] = rr < rows ? limit_of(col_q[n][i]) : 0;
        mf[n][i] = -INFINITY;
        l[n][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) om[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[k][n][i] = 0.f;

      if constexpr (BITS == 16) {
        const uint32_t signs = p.negate ? 0x80008000u : 0u;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          qf[n][k][0] = raw[n][k][0] ^ signs;
          qf[n][k][1] = raw[n][k][1] ^ signs;
        }
        f[n][0] = f[n][1] = p.scale_log2;
      } else {
        // q scaled by a power of two, largest element in [2^10, 2^11), as fp16;
        // its elements are exact down to 2^-24 of the largest
        auto pair = [&](int grp, int i) {
          const uint32_t w = raw[n][2 * grp + i / 2][i % 2];
          return p.bf16 ? Elem<__nv_bfloat16>::unpack2(w) : Elem<__half>::unpack2(w);
        };
        uint32_t most = 0;  // largest magnitudes of the even and odd dims, as 16-bit patterns
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) most = __vmaxu2(most, raw[n][k][i] & 0x7FFF7FFFu);
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const uint32_t one = max(most & 0xFFFFu, most >> 16);
        const float top = p.bf16 ? Elem<__nv_bfloat16>::value((uint16_t)one) : Elem<__half>::value((uint16_t)one);
        int e = (int)(__float_as_uint(top) >> 23) - 127;  // 2^e <= top < 2^(e + 1)
        e = max(-116, min(e, 127));
        const float up = __uint_as_float((uint32_t)(127 + 10 - e) << 23);
        const float turn = p.negate ? -up : up;
        float down = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2 * 1024.f;  // 2^20 / up
        down = fmaxf(fminf(down, FLT_MAX), FLT_MIN);  // finite, and above 0
        float mine = 0.f;  // sum of group t
#pragma unroll
        for (int grp = 0; grp < NG; ++grp) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = pair(grp, i);
            const float x = v.x * turn, y = v.y * turn;
            sum += x + y;
            // codes of the first two dims of four stand 4 bits lower: their q is 2^4 larger
            const uint32_t h2 = Elem<__half>::pack2(x, y);
            qf[n][2 * grp + i / 2][i % 2] = i % 2 ? h2 : hmul2(h2, 0x4C004C00u);  // x 16
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (t == grp) mine = sum * 0.015625f;  // 2^-6: below 2^11
        }
        const __half head = __float2half_rn(mine);
        const __half tail = __float2half_rn(mine - __half2float(head));
        qsum[n][0] = (uint32_t)__half_as_ushort(head) << 16;
        qsum[n][1] = (uint32_t)__half_as_ushort(tail) << 16;
        f[n][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        f[n][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
    }
  };

  // One tile.  `edge`: some block has no tokens, or tokens that some row does
  // not see; without it every score counts.
  auto step = [&](int stage, uint32_t ok_mask, auto edge_tag) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    const uint32_t base = my_ring + stage * C::kStageBytes;
    const uint8_t* bytes = smem_raw + (warp * NS + stage) * C::kStageBytes;
    auto skipped = [&](int u) {
      return EDGE && !((ok_mask >> u & 1u) && block_token(cur, u) < max_lim);
    };
    float s[U][NT][4], top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
    // ---- S^T = K Q^T
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (skipped(u)) continue;
      [[maybe_unused]] const uint32_t blk = base + u * C::kBlockBytes;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][n][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          uint32_t a[4];
          constexpr int WB = D * 2 >= 128 ? 128 : D * 2;  // bytes of a swizzled row
          const int r = (lane & 7) + (lane & 8);
          const int ch = 2 * k + (lane >> 4);  // 16-byte chunk of the row
          const int sw = WB == 128 ? (r & 7) : WB == 64 ? (r >> 1 & 3) : (r >> 2 & 1);
          ldsm4(blk + (ch / (WB / 16)) * (16 * WB) + r * WB + ((ch % (WB / 16)) ^ sw) * 16, a);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma16816<M>(s[u][n], a[0], a[1], a[2], a[3], qf[n][k][0], qf[n][k][1]);
        }
      } else {
        constexpr Kv4 lay(D);
        const uint8_t* at = bytes + u * C::kBlockBytes;
        uint32_t w0[NG], w1[NG], q0[NG], q1[NG];  // codes and parameters of tokens g, g + 8
        load_words<NG>(at + lane * (NG * 4), w0);
        load_words<NG>(at + (32 + lane) * (NG * 4), w1);
        load_words<NG>(at + lay.k_params() + g * (NG * 4), q0);
        load_words<NG>(at + lay.k_params() + (g + 8) * (NG * 4), q1);
        uint32_t p0[1] = {0}, p1[1] = {0};  // parameters of group t
        if (t < NG) {
          load_words<1>(at + lay.k_params() + (g * NG + t) * 4, p0);
          load_words<1>(at + lay.k_params() + ((g + 8) * NG + t) * 4, p1);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // the groups' first halves, then their second ones: no product waits
          // for the one before it
          float c[NG][4], cm[4];
#pragma unroll
          for (int grp = 0; grp < NG; ++grp)
            mma16816_zero<M>(c[grp], w0[grp] & 0x000F000Fu, w1[grp] & 0x000F000Fu,
                             w0[grp] & 0x00F000F0u, w1[grp] & 0x00F000F0u, qf[n][2 * grp][0],
                             qf[n][2 * grp][1]);
          mma16816_zero<M>(cm, p0[0], p1[0], p0[0], p1[0], qsum[n][0], qsum[n][1]);
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) {
            const uint32_t x0 = w0[grp] >> 8, x1 = w1[grp] >> 8;
            mma16816<M>(c[grp], x0 & 0x000F000Fu, x1 & 0x000F000Fu, x0 & 0x00F000F0u,
                        x1 & 0x00F000F0u, qf[n][2 * grp + 1][0], qf[n][2 * grp + 1][1]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][n][i] = cm[i] * 0x1p-14f;
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) {
            const float s0 = low_half(q0[grp]), s1 = low_half(q1[grp]);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][n][i] = fmaf(i < 2 ? s0 : s1, c[grp][i], s[u][n][i]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (EDGE) {
          const int tok0 = block_token(cur, u);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tok0 + g + (i >> 1) * 8 >= lim[n][i & 1]) s[u][n][i] = -INFINITY;
        }
        top[n][0] = fmaxf(top[n][0], fmaxf(s[u][n][0], s[u][n][2]));
        top[n][1] = fmaxf(top[n][1], fmaxf(s[u][n][1], s[u][n][3]));
      }
    }
    // ---- running maximum and largest scale; O and the sum follow them
    bool above = false;
    // The lane's two scales of block u (tokens that no row sees: 0).
    auto scales = [&](int u) {
      uint32_t w[1] = {0};
      if (lane < 8 * NG) {
        load_words<1>(bytes + u * C::kBlockBytes + Kv4(D).v_params() + lane * 4, w);
        if constexpr (EDGE) {
          const int to = max_lim - block_token(cur, u), tok = (lane >> 1 & 3) * 2 + (lane & 1) * 8;
          w[0] &= (tok < to ? 0xFFFFu : 0u) | (tok + 1 < to ? 0xFFFF0000u : 0u);
        }
      }
      return w[0];
    };
    if constexpr (BITS == 4) {
      uint32_t most = (se << 10 | 0x3FFu) * 0x10001u;  // the largest scales that `se` is right for
      const uint32_t had = most;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!skipped(u)) most = __vmaxu2(most, scales(u));
      above = most != had;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) above |= top[n][i] * f[n][i] > mf[n][i] + kSlack;
    if (__any_sync(0xffffffffu, above)) {
      bool far = false;
      float shrink = 1.f;  // of O's codes
      if constexpr (BITS == 4) {
        uint32_t now = se;
#pragma unroll 1
        for (int u = 0; u < U; ++u) {
          if (skipped(u)) continue;
          const uint32_t w = scales(u), a = w >> 10 & 31u, b = w >> 26 & 31u;
          if (a < 31u) now = max(now, a);  // a group with a NaN has none
          if (b < 31u) now = max(now, b);
        }
        now = __reduce_max_sync(0xffffffffu, now);
        shrink = __uint_as_float((127u + se - now) << 23);
        se = now;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 4; d < 32; d *= 2)
            top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], d));
          const float now = fmaxf(mf[n][i], top[n][i] * f[n][i]);
          far |= fabsf(now) >= 0x1p24f && fabsf(now) < INFINITY;
          const float keep = now == -INFINITY ? 1.f : ex2(mf[n][i] - now);
          mf[n][i] = now;
          l[n][i] *= keep;
          om[n][i] *= keep;
          om[n][i + 2] *= keep;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            o[k][n][i] *= keep * shrink;
            o[k][n][i + 2] *= keep * shrink;
          }
        }
      static_assert(kFar == 24, "the bound above");
      if (cuts |= __any_sync(0xffffffffu, far)) {
        // the power of two of each row, from its true maximum: it shrinks again where the
        // maximum was far below 0 and is not any more
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int had = sh.cut[warp][n * 8 + 2 * t + i];
            const int e = (int)(__float_as_uint(mf[n][i]) >> 23 & 255u) - 127;
            const int by = e == 128 ? 0 : max(e + had - (kFar - 1), 0) - had;
            const float less = __uint_as_float((uint32_t)(127 - by) << 23);
            f[n][i] *= less;
            mf[n][i] *= less;
            __syncwarp();
            if (g == 0) sh.cut[warp][n * 8 + 2 * t + i] = had + by;
          }
        __syncwarp();
      }
    }
    float from[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)  // no score above -inf yet: every probability is 0
        from[n][i] = fmaxf(mf[n][i], -3.4e38f) - LIFT;
    // 2^(15 - se), twice
    const uint32_t unit = (se < 30 ? (30u - se) << 10 : 0x200u) * 0x10001u;
    // ---- P^T, O^T += V^T P^T
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (skipped(u)) continue;
      [[maybe_unused]] const uint32_t blk = base + u * C::kBlockBytes;
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = ex2(fmaf(s[u][n][i], f[n][i & 1], -from[n][i & 1]));
        l[n][0] += e[0] + e[2];
        l[n][1] += e[1] + e[3];
        pf[n][0] = transpose8x8(Elem<M>::pack2(e[0], e[1]));
        pf[n][1] = transpose8x8(Elem<M>::pack2(e[2], e[3]));
      }
      // Values that a row does not see must not reach its sum even as 0 x NaN.
      // Those that no row of the block sees are set to zero; where the rows'
      // limits differ and some value is not finite, each query token's rows are
      // multiplied apart and the other columns kept.
      const int tok0 = block_token(cur, u);
      bool apart = false;
      if constexpr (EDGE) {
        if (p.causal && qp_last > qp_first && tok0 + kBlockTokens > min_lim) {
          constexpr uint32_t EXP = Elem<M>::kIdescAB == 0 ? 0x7C00u : 0x7F80u;
          // the block's values (4-bit: V's parameters), two to a word
          constexpr int WORDS = BITS == 16 ? 8 * D : 16 * NG;
          const uint32_t* at = reinterpret_cast<const uint32_t*>(
              bytes + u * C::kBlockBytes + (BITS == 16 ? 32 * D : Kv4(D).v_params()));
          for (int i = lane; i < WORDS; i += 32) {
            const uint32_t w = at[i];
            apart |= (w & EXP) == EXP || (w >> 16 & EXP) == EXP;
          }
          apart = __any_sync(0xffffffffu, apart);
        }
      }
      const int passes = apart ? qp_last - qp_first + 1 : 1;
#pragma unroll 1
      for (int pass = 0; pass < passes; ++pass) {
        uint32_t keep0 = ~0u, keep1 = ~0u;  // token pairs (2t, 2t + 1), (2t + 8, 2t + 9)
        bool mine[NT][2];
        auto add = [&](float (&acc)[4], int n, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                       uint32_t b0, uint32_t b1) {
          if (!EDGE || !apart) {
            mma16816<M>(acc, a0, a1, a2, a3, b0, b1);
          } else {
            float c[4] = {acc[0], acc[1], acc[2], acc[3]};
            mma16816<M>(c, a0, a1, a2, a3, b0, b1);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = mine[n][i & 1] ? c[i] : acc[i];
          }
        };
        if constexpr (EDGE) {
          const int to = (apart ? limit_of(qp_first + pass) : max_lim) - tok0;
          if (apart && to <= 0) continue;
          keep0 = (2 * t < to ? 0xFFFFu : 0u) | (2 * t + 1 < to ? 0xFFFF0000u : 0u);
          keep1 = (2 * t + 8 < to ? 0xFFFFu : 0u) | (2 * t + 9 < to ? 0xFFFF0000u : 0u);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) mine[n][i] = !apart || col_q[n][i] == qp_first + pass;
        }
        if constexpr (BITS == 16) {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            uint32_t a[4];
            constexpr int WB = D * 2 >= 128 ? 128 : D * 2;
            const int r = (lane & 7) + ((lane >> 4) << 3);
            const int ch = 2 * k + ((lane >> 3) & 1);
            const int sw = WB == 128 ? (r & 7) : WB == 64 ? (r >> 1 & 3) : (r >> 2 & 1);
            ldsm4_trans(blk + 32 * D + (ch / (WB / 16)) * (16 * WB) + r * WB +
                            ((ch % (WB / 16)) ^ sw) * 16, a);
            if constexpr (EDGE) {
              a[0] &= keep0;
              a[1] &= keep0;
              a[2] &= keep1;
              a[3] &= keep1;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) add(o[k][n], n, a[0], a[1], a[2], a[3], pf[n][0], pf[n][1]);
          }
        } else {
          constexpr Kv4 lay(D);
          const uint8_t* at = bytes + u * C::kBlockBytes;
          uint32_t w0[NG], w1[NG], mm[2] = {0, 0};
          load_words<NG>(at + lay.v_codes() + lane * (NG * 4), w0);
          load_words<NG>(at + lay.v_codes() + (32 + lane) * (NG * 4), w1);
          if (g < NG) load_words<2>(at + lay.v_params() + 32 * NG + lane * 8, mm);
          if constexpr (EDGE) {
            mm[0] &= keep0;
            mm[1] &= keep1;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) add(om[n], n, mm[0], 0u, mm[1], 0u, pf[n][0], pf[n][1]);
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) {
            uint32_t sc[2];
            load_words<2>(at + lay.v_params() + (grp * 4 + t) * 8, sc);
            if constexpr (EDGE) {
              sc[0] &= keep0;
              sc[1] &= keep1;
            }
            sc[0] = hmul2(sc[0], unit);
            sc[1] = hmul2(sc[1], unit);
            const uint32_t x0 = w0[grp] >> 8, x1 = w1[grp] >> 8;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t b0 = hmul2(pf[n][0], sc[0]), b1 = hmul2(pf[n][1], sc[1]);
              add(o[2 * grp][n], n, w0[grp] & 0x000F000Fu, w0[grp] & 0x00F000F0u,
                  w1[grp] & 0x000F000Fu, w1[grp] & 0x00F000F0u, b0, b1);
              add(o[2 * grp + 1][n], n, x0 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x000F000Fu,
                  x1 & 0x00F000F0u, b0, b1);
            }
          }
        }
      }
    }
  };

  // The warps' results of a segment, joined; `first`: this share holds the
  // segment's first tile, `last`: its last.
  auto end_segment = [&](bool first, bool last) {
    const int h = cur.h, rb = cur.rb, rows = p.Sq * p.group;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // the column block's even rows, then its odd ones
        constexpr int JR = C::kJoinRows, EACH = JR / 4;
#pragma unroll
        for (int d = 4; d < 32; d *= 2) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
        const int place = t * EACH + (EACH == 2 ? i : 0);
        constexpr float DOWN = LIFT > 0.f ? 0x1p-12f : 1.f;
        static_assert(kLift == 12.f, "2^-kLift");
        if (g == 0) {
          const uint32_t cut = sh.cut[warp][n * 8 + 2 * t + i];
          sh.join_ml[warp][place] = make_float2(mf[n][i] * __uint_as_float((127u + cut) << 23), l[n][i] * DOWN);
        }
        float* dst = join + (warp * JR + place) * C::kJoinStride;
        if constexpr (BITS == 16) {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            dst[16 * k + g] = o[k][n][i] * DOWN;
            dst[16 * k + 8 + g] = o[k][n][i + 2] * DOWN;
          }
        } else {
#pragma unroll
          for (int grp = 0; grp < NG; ++grp) {
            const float mm = __shfl_sync(0xffffffffu, om[n][i], grp * 4 + t) * DOWN;
            // 2^24 and 2^20 (codes), 2^(se - 15) (scales), 2^-kLift
            const float x24 = __uint_as_float((124u + se) << 23), x20 = __uint_as_float((120u + se) << 23);
            *reinterpret_cast<float4*>(dst + 32 * grp + 4 * g) =
                make_float4(fmaf(o[2 * grp][n][i], x24, mm), fmaf(o[2 * grp][n][i + 2], x20, mm),
                            fmaf(o[2 * grp + 1][n][i], x24, mm), fmaf(o[2 * grp + 1][n][i + 2], x20, mm));
          }
        }
        if (EACH == 2 && i == 0) continue;
        __syncthreads();
        constexpr int PER_ROW = D / 8;
        for (int j = tid; j < JR * PER_ROW; j += kThreads) {
          const int tr = j / PER_ROW, d = j % PER_ROW * 8, r = n * 8 + (EACH == 2 ? tr : 2 * tr + i);
          const int rr = rb * ROWS + r;
          float top = -INFINITY, sum = 0.f, x[8] = {};
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh.join_ml[w][tr].x);
          const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float2 ml = sh.join_ml[w][tr];
            const float e = ex2(ml.x - safe);
            sum = fmaf(e, ml.y, sum);
            const float* src = join + (w * JR + tr) * C::kJoinStride + d;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = fmaf(e, src[k], x[k]);
          }
          if (rr >= rows) continue;
          if (first && last) {
            write_row<D>(p, cur.b, h, rr, d, top, sum, x);
          } else {
            const long long slot = (2LL * blockIdx.x + (first ? 1 : 0)) * ROWS + r;
            float4* to = reinterpret_cast<float4*>(p.part_o + slot * D + d);
            to[0] = make_float4(x[0], x[1], x[2], x[3]);
            to[1] = make_float4(x[4], x[5], x[6], x[7]);
            if (d == 0) p.part_ml[slot] = make_float2(top, sum);
          }
        }
        __syncthreads();
      }
    }
  };

  // ---- the share, tile by tile
  // The first pages, q and copies are asked for before anything waits.
  constexpr bool AHEAD = NT == 1;  // q is read ahead where there are registers for it
  if (AHEAD) load_q(cur);
  {
    int ids[NS];
    Cursor c = pc;
    int rest = to_issue;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const bool wanted = rest > 0 || (p.whole && c.tt > 0);
      ids[s] = look_up(c, wanted);
      if (wanted) rest -= advance(c);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s)
      if (more_to_issue()) issue(s, ids[s]);
  }
  int next_id = look_up(pc, more_to_issue());  // read ahead of its use
  int stage = 0;
  bool fresh = true, first = false, stopped = false;
#pragma unroll 1
  while (left > 0 || (p.whole && !fresh)) {
    if (fresh) {
      first = cur.tt == 0;
      if (!AHEAD) load_q(cur);
      begin_segment();
      if (first && tid == 0 && cur.h == 0 && cur.rb == 0 && p.kv.bad_length(p.lengths[cur.b])) p.kv.report(kStatusPage);
    }
    const bool last = cur.tt + 1 == cur.nt;
    Cursor next = cur;
    const int places = advance(next);
    const bool goes_on = left > places || (p.whole && !last);
    if (AHEAD && last && goes_on) load_q(next);
    // a wait may run out for some lanes and end for others: the warp goes one way
    const bool here = __all_sync(0xffffffffu, mbar_wait(my_bars + stage * 8, odd >> stage & 1u, wait));
    if (here) {
      in_flight &= ~(1u << stage);
      const uint32_t ok = ok_bits >> stage * U & ALL;
      if (ok == ALL && block_token(cur, U - 1) + kBlockTokens <= min_lim)
        step(stage, ok, std::false_type{});
      else if (ok != 0)
        step(stage, ok, std::true_type{});
    }
    __syncwarp();
    stopped |= !here;  // a copy did not arrive: bring no more
    if (!stopped && more_to_issue()) {
      issue(stage, next_id);
      next_id = look_up(pc, more_to_issue());
    }
    if (last || !goes_on) end_segment(first, last);
    fresh = last;
    left -= places;
    cur = next;
    if (++stage == NS) stage = 0;
  }
  // After a wait that ran out, copies may still be under way into this CTA's memory.
  for (int s = 0; s < NS; ++s)
    if (in_flight >> s & 1u) mbar_wait_drain(my_bars + s * 8, odd >> s & 1u, max(p.timeout_ns, 1000000000ull));
}

// Running join of partial results: 8 dims of a row.
struct RowSum {
  float top = -INFINITY, sum = 0.f, x[8] = {};
  __device__ __forceinline__ void add(float2 ml, float4 u, float4 v) {
    const float now = fmaxf(top, ml.x);
    const float safe = now == -INFINITY ? 0.f : now;
    const float old = ex2(top - safe), e = ex2(ml.x - safe);
    const float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    top = now;
    sum = fmaf(e, ml.y, sum * old);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(e, y[j], x[j] * old);
  }
  __device__ __forceinline__ void take(const DecodeParams& p, long long slot, int D, int d) {
    const float4* src = reinterpret_cast<const float4*>(p.part_o + slot * D + d);
    add(p.part_ml[slot], src[0], src[1]);
  }
};

// Joins the partial results of the segments that cross shares, in the order of
// the shares.  blockIdx.x is a border between two shares; the border that a
// segment crosses first does its work.  With many shares to a segment a CTA takes
// two rows (blockIdx.y) and a thread, which holds 8 dims, every P-th share, so
// that all loads are in flight at once.
template <int D, int BITS, int NT>
__global__ void __launch_bounds__(kThreads) fa_decode_merge_kernel(const DecodeParams p) {
  using C = Cfg<D, BITS, NT>;
  constexpr int ROWS = 8 * NT, PER_ROW = D / 8, P = kThreads / 2 / PER_ROW;
  __shared__ Spot spot;
  __shared__ unsigned warp_sum[kWarps];
  __shared__ float4 part_x[2][P][D / 4];
  __shared__ float2 part_ml[2][P];
  const int segs = p.kv.heads * p.row_blocks;
  const unsigned border = blockIdx.x + 1;
  const Shares shares = locate<C::kTile, C::kCost>(p, segs, border, spot, warp_sum);
  const unsigned at = shares.begin(border);
  const int b = spot.b, nt = tiles_of<C::kTile>(spot.len);
  const unsigned places = nt + C::kCost, hr = (at - spot.before) / places;
  const unsigned t0 = spot.before + hr * places, t1 = t0 + nt - 1;
  const bool crossed = at < shares.total && at > t0 && at <= t1 && shares.begin(border - 1) <= t0;
  const int c0 = (int)border - 1, c1 = crossed ? (int)shares.of(t1) : 0;
  griddep_wait();  // also where nothing is to do: the grid after this one may rely on it
  griddep_launch_dependents();
  if (!crossed) return;
  const int h = (int)p.rb_div.div(hr), rb = (int)hr - h * p.row_blocks, rows = p.Sq * p.group;
  if (gridDim.y == 1) {
    // few shares to a segment: a thread takes all of them for its 8 dims
    for (int i = threadIdx.x; i < min(rows - rb * ROWS, ROWS) * PER_ROW; i += kThreads) {
      const int r = i / PER_ROW, d = i % PER_ROW * 8;
      RowSum sum;
#pragma unroll 4
      for (int c = c0; c <= c1; ++c)
        sum.take(p, (2LL * c + (c == c0 ? 1 : 0)) * ROWS + r, D, d);
      write_row<D>(p, b, h, rb * ROWS + r, d, sum.top, sum.sum, sum.x);
    }
    return;
  }
  const int half = threadIdx.x / (kThreads / 2), i = threadIdx.x % (kThreads / 2);
  const int pg = i / PER_ROW, d = i % PER_ROW * 8;
  const int r = blockIdx.y * 2 + half, rr = rb * ROWS + r;
  RowSum sum;
#pragma unroll 4
  for (int c = c0 + pg; c <= c1; c += P) sum.take(p, (2LL * c + (c == c0 ? 1 : 0)) * ROWS + r, D, d);
  part_x[half][pg][d / 4] = make_float4(sum.x[0], sum.x[1], sum.x[2], sum.x[3]);
  part_x[half][pg][d / 4 + 1] = make_float4(sum.x[4], sum.x[5], sum.x[6], sum.x[7]);
  if (d == 0) part_ml[half][pg] = make_float2(sum.top, sum.sum);
  __syncthreads();
  if (pg != 0 || rr >= rows) return;
#pragma unroll
  for (int k = 1; k < P; ++k) sum.add(part_ml[half][k], part_x[half][k][d / 4], part_x[half][k][d / 4 + 1]);
  write_row<D>(p, b, h, rr, d, sum.top, sum.sum, sum.x);
}

template <typename T, int D, int BITS, int NT>
int launch_decode(DecodeParams& p, const CUtensorMap& tk, const CUtensorMap& tv, bool split,
                  cudaStream_t st) {
  using C = Cfg<D, BITS, NT>;
  auto kernel = fa_decode_kernel<T, D, BITS, NT>;
  constexpr int kTag = 1000 + ((sizeof(T) == 2 && Elem<T>::kIdescAB == 0) ? 0 : 1) + 2 * NT +
                       8 * (BITS == 4) + 16 * D;
  if (!smem_attr_set<kTag>(reinterpret_cast<const void*>(kernel), C::kSmem)) return FA_ERR_LAUNCH;
  if (launch_pdl(kernel, dim3(p.grid_div.d), dim3(kThreads), C::kSmem, st, p, tk, tv) != cudaSuccess)
    return FA_ERR_LAUNCH;
  if (!split) return FA_OK;
  // Many shares to a segment (few segments): its rows are spread over CTAs, too
  // (with two or three shares that takes 3.5 us of dependent steps, this way 1.5).
  const long long segs = (long long)p.B * p.kv.heads * p.row_blocks;
  const unsigned y = p.grid_div.d > 4 * segs ? 4 * NT : 1;
  return launch_pdl(fa_decode_merge_kernel<D, BITS, NT>, dim3(p.grid_div.d - 1, y), dim3(kThreads), 0, st,
                    p) == cudaSuccess
             ? FA_OK
             : FA_ERR_LAUNCH;
}

template <typename T, int D, int BITS>
int launch_decode_nt(DecodeParams& p, int nt, const CUtensorMap& tk, const CUtensorMap& tv,
                     bool split, cudaStream_t st) {
  switch (nt) {
    case 1: return launch_decode<T, D, BITS, 1>(p, tk, tv, split, st);
    case 2: return launch_decode<T, D, BITS, 2>(p, tk, tv, split, st);
  }
  if constexpr (max_nt(D) > 2) {
    if (nt == 3) return launch_decode<T, D, BITS, 3>(p, tk, tv, split, st);
    return launch_decode<T, D, BITS, 4>(p, tk, tv, split, st);
  }
  return FA_ERR_ARG;
}

template <int D>
int launch_decode_d(DecodeParams& p, int nt, const CUtensorMap& tk, const CUtensorMap& tv,
                    bool split, cudaStream_t st) {
  if (p.kv.bits == 4) {
    if constexpr (D >= 32) return launch_decode_nt<__half, D, 4>(p, nt, tk, tv, split, st);
    return FA_ERR_ARG;
  }
  return p.bf16 ? launch_decode_nt<__nv_bfloat16, D, 16>(p, nt, tk, tv, split, st)
                : launch_decode_nt<__half, D, 16>(p, nt, tk, tv, split, st);
}

int launch_decode_any(DecodeParams& p, int nt, const CUtensorMap& tk, const CUtensorMap& tv,
                      bool split, cudaStream_t st) {
  switch (p.kv.D) {
    case 16: return launch_decode_d<16>(p, nt, tk, tv, split, st);
    case 32: return launch_decode_d<32>(p, nt, tk, tv, split, st);
    case 64: return launch_decode_d<64>(p, nt, tk, tv, split, st);
    default: return launch_decode_d<128>(p, nt, tk, tv, split, st);
  }
}

// Tiles (of the table's room) up to which segments are not split, so that no second
// launch joins them.  Replayed, whole against split, us: 16-bit, 16 heads of 64,
// 300 tokens (3 tiles) 5.8 / 7.2, 777 (7) 9.5 / 7.6, where the second launch costs
// the host 2.5 us more, 2000 (16) 17.9 / 8.4; 4-bit, 8 heads of 128, 1000 tokens (4)
// 12.3 / 11.6, of 16 sequences 13.3 / 16.1, 2000 (8) 17.5 / 10.7.
constexpr int whole_tiles(int bits) { return bits == 4 ? 4 : 7; }
// Places are counted in 31 bits.
constexpr long long kMaxPlaces = 1LL << 31;

struct Plan {
  int nt, row_blocks, grid;
  long long places;  // of the list, at most
  bool split;  // segments may cross shares: a second launch joins them
};

// Query rows in as few row blocks as the registers allow; as many CTAs as
// the SMs hold, fewer when the tables have room for fewer tiles.
Plan plan_of(const fa_sm100_kv_cache* c, int table_width, int batch, int seqlen, int nheads) {
  Plan pl;
  const long long rows = (long long)seqlen * (nheads / c->nheads_kv);
  const int most_rows = 8 * max_nt(c->head_dim);
  pl.row_blocks = (int)((rows + most_rows - 1) / most_rows);
  pl.nt = (int)((rows + 8LL * pl.row_blocks - 1) / (8LL * pl.row_blocks));
  const int tile = kWarps * kBlockTokens * blocks_of(c->head_dim, c->bits, pl.nt);
  const long long per_seg = ((long long)table_width * c->page_size + tile - 1) / tile;
  const long long segs = (long long)batch * c->nheads_kv * pl.row_blocks, tiles = segs * per_seg;
  const long long most = (long long)sm_count() * kCtas;
  pl.places = segs * (per_seg + cost_of(c->head_dim, c->bits, pl.nt));
  pl.split = per_seg > whole_tiles(c->bits);
  const long long grid = pl.split ? tiles : segs;
  pl.grid = (int)(grid < most ? grid : most);
  if (pl.grid == 1) pl.split = false;
  return pl;
}

size_t partial_bytes(const Plan& pl, int D) {
  return pl.split ? (size_t)2 * pl.grid * 8 * pl.nt * (D * sizeof(float) + sizeof(float2)) : 0;
}

bool decode_shape_ok(const fa_sm100_kv_cache* c, int table_width, int batch, int seqlen, int nheads) {
  return check_kv_cache(c) == FA_OK && table_width >= 1 && batch >= 1 && seqlen >= 1 && nheads >= 1 &&
         nheads % c->nheads_kv == 0 && (long long)seqlen * nheads <= (1LL << 24) &&
         (long long)table_width * c->page_size <= 2147483647LL - 65536 &&
         (long long)batch * seqlen * nheads <= 2147483647LL;
}

}  // namespace
}  // namespace fa_sm100

extern "C" size_t fa_sm100_decode_workspace_bytes(const fa_sm100_kv_cache* cache, int table_width,
                                                  int batch, int seqlen, int nheads) {
  using namespace fa_sm100;
  if (!decode_shape_ok(cache, table_width, batch, seqlen, nheads)) return 0;
  const Plan pl = plan_of(cache, table_width, batch, seqlen, nheads);
  return pl.places < kMaxPlaces ? partial_bytes(pl, cache->head_dim) + 256 : 0;
}

extern "C" int fa_sm100_decode(const fa_sm100_kv_cache* cache, const void* q, void* out, float* lse,
                               const int* page_table, int table_width, const int* lengths,
                               const int* starts, void* workspace, size_t workspace_bytes, int batch,
                               int seqlen, int nheads, float sm_scale, int causal, int* status,
                               void* stream) {
  using namespace fa_sm100;
  if (!cache || !decode_shape_ok(cache, table_width, batch, seqlen, nheads)) return FA_ERR_ARG;
  if (!q || !out || !page_table || !lengths || !std::isfinite(sm_scale)) return FA_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) return FA_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(page_table) |
       reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(starts)) & 3u)
    return FA_ERR_ARG;
  int rc = bind_device();
  if (rc != FA_OK) return rc;
  const Plan pl = plan_of(cache, table_width, batch, seqlen, nheads);
  if (pl.places >= kMaxPlaces) return FA_ERR_ARG;
  const size_t need = partial_bytes(pl, cache->head_dim);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return FA_ERR_WORKSPACE;
  if (pl.grid < 1) return FA_ERR_DEVICE;
  CUtensorMap tk = {}, tv = {};
  if (cache->bits == 16) {
    const long long rows = (long long)cache->num_pages * cache->nheads_kv * cache->page_size;
    if ((rc = make_rows_map(&tk, cache->k_pages, rows, cache->head_dim, kBlockTokens, cache->dtype)) != FA_OK)
      return rc;
    if ((rc = make_rows_map(&tv, cache->v_pages, rows, cache->head_dim, kBlockTokens, cache->dtype)) != FA_OK)
      return rc;
  }
  DecodeParams p = {};
  p.kv = kv_view(cache, page_table, table_width, status);
  p.q = q;
  p.out = out;
  p.lse = lse;
  p.lengths = lengths;
  p.starts = starts;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) +
                                        (size_t)2 * pl.grid * 8 * pl.nt * cache->head_dim * sizeof(float));
  p.B = batch;
  p.Sq = seqlen;
  p.H = nheads;
  p.group = nheads / cache->nheads_kv;
  p.row_blocks = pl.row_blocks;
  p.causal = causal ? 1 : 0;
  while ((1 << p.page_shift) < cache->page_size) ++p.page_shift;
  p.grid_div = FastDiv(pl.grid);
  p.group_div = FastDiv(p.group);
  p.rb_div = FastDiv(pl.row_blocks);
  p.segs_div = FastDiv(cache->nheads_kv * pl.row_blocks);
  p.whole = !pl.split;
  p.direct = p.whole && pl.grid == (long long)batch * cache->nheads_kv * pl.row_blocks;
  p.negate = sm_scale < 0.f;
  p.bf16 = cache->dtype == FA_DTYPE_BF16;
  p.scale_log2 = fmaxf(fabsf(sm_scale) * 1.44269504088896341f, FLT_MIN);
  p.skip_copy = debug_flags() & 2;
  p.timeout_ns = wait_timeout_ns();
  return launch_decode_any(p, pl.nt, tk, tv, pl.split, static_cast<cudaStream_t>(stream));
}
