// Layout of the paged key/value cache (include/fa_sm100.h, fa_sm100_kv_cache).
//
// 4-bit pages are (pages, kv heads, page/16) blocks of 16 tokens of one head.
// A group is 32 consecutive dims of one token: minimum m (fp16, rounded down),
// scale s (fp16, (max - m) / 15 rounded up), codes c = rint((x - m) / s) in
// 0..15, value m + s c.  Rounding m down and s up keeps every value inside
// [m, m + 15 s], so no code is clipped; m + 15 s may reach 65536, which fp16
// results hold to 65504 (most_half2).  A block is, in this order,
//   K codes   one word of 8 codes per (token, t, group); it holds dims
//             32 group + 8 t + 0..7, codes of even dims in the low half
//             (dims 0, 2, 4, 6 from bit 0 up), of odd dims in the high half
//   K params  (s, m) as one word per (token, group)
//   V codes   one word of 8 codes per (tp, g, t, group): dims
//             32 group + 4 g + 0..3 of token 8 tp + 2 t (low half) and of the
//             next token (high half)
//   V params  s as (group, t, tp, token parity) fp16, then m likewise
// The orders are those in which a lane (g, t) = (lane / 4, lane % 4) of the
// decode kernel's matrix instructions reads them: every warp read of a block
// is contiguous, and a masked word is an operand register (fa_decode.cu).
// Each byte belongs to one token, so tokens can be appended one at a time.
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace fa_sm100 {

constexpr int kBlockTokens = 16;

struct Kv4 {  // offsets of a block's parts in bytes; D is 32, 64 or 128
  int D;
  __host__ __device__ constexpr explicit Kv4(int d) : D(d) {}
  __host__ __device__ constexpr int groups() const { return D / 32; }
  __host__ __device__ constexpr int k_params() const { return 8 * D; }
  __host__ __device__ constexpr int v_codes() const { return 10 * D; }
  __host__ __device__ constexpr int v_params() const { return 18 * D; }
  __host__ __device__ constexpr int bytes() const { return 20 * D; }
};

// Two fp16 values, at most 65504 each; NaN stays.
__device__ __forceinline__ uint32_t most_half2(uint32_t w) {
  const __half2 r = __hmin2_nan(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x7BFF)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

struct KvView {  // a cache as the kernels take it
  uint8_t* k;    // 16-bit: keys (pages, heads, page, D); 4-bit: blocks
  uint8_t* v;    // 16-bit: values; 4-bit: null
  const int* table;
  int table_width, num_pages, page, heads, D, bits;
  int* status;

  __device__ __forceinline__ bool bad_page(int id) const { return (unsigned)id >= (unsigned)num_pages; }
  __device__ __forceinline__ void report(int bit) const {
    if (status) atomicOr(status, bit);
  }
  // Page id of token `pos` of sequence b, or -1.
  __device__ __forceinline__ int page_of(int b, long long pos, int page_shift) const {
    const long long i = pos >> page_shift;
    if (pos < 0 || i >= table_width) return -1;
    const int id = table[(long long)b * table_width + i];
    return bad_page(id) ? -1 : id;
  }
  // Tokens of a sequence that the table has room for.
  __device__ __forceinline__ int clamp_length(int n) const {
    const long long room = (long long)table_width * page;
    return n < 0 ? 0 : n > room ? (int)room : n;
  }
  __device__ __forceinline__ bool bad_length(int n) const {
    return n < 0 || n > (long long)table_width * page;
  }
};

// Host-side checks of a cache description (0: fine).
int check_kv_cache(const fa_sm100_kv_cache* c);
KvView kv_view(const fa_sm100_kv_cache* c, const int* table, int table_width, int* status);

}  // namespace fa_sm100
