// The paged K/V cache held in 4 bits: its layout in memory, the quantiser's
// tables as the kernels take them, and the codes' decoding to fp16 pairs.
//
// Pool: page-major.  A page holds, for each head, page_size / 16 blocks of 16
// tokens, and a block is 1088 consecutive bytes
//     [16 x 32 bytes K codes | 16 x 32 bytes V codes | 16 x (K norm, V norm)]
// so that everything attention needs of 16 tokens of a head is one aligned
// run of memory, and of a page one longer run: one bulk copy brings it.
//
// A vector's 64 codes are 8 words; nibble p of word w is coordinate 8w + p: the
// magnitude's index in its low three bits, the sign in its top bit.  A byte is
// two codes, of neighbouring coordinates of a token or, once two tokens' words
// are zipped, of one coordinate of both: one of 256 fp16 pairs either way.  A
// key norm's sign bit marks a masked token.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace cc2 {
namespace kv4 {

constexpr int kBlockTokens = 16;
constexpr int kBlockBytes = 1088;
constexpr int kVCodes = 512, kNorms = 1024;  // offsets in a block

// Where a page and a head's blocks of it start.
struct Pool {
  uint8_t* pages;
  long long page_bytes;
  int head_bytes;
  int num_pages;
  int page_shift;  // log2 page_size
  int heads;
  int norm_bf16;   // norms are bf16 (else fp16)
};

// One rotation for the kernels that quantise and restore (by value: its entries
// are operands in constant memory).  Coordinate i of the rotated vector comes
// from element place[i] / 4, times sign[i].
struct Turn {
  uint32_t place[64];
  float sign[64];
};

// The magnitude of a coordinate by one comparison: r = round(511 |y| / 8n) is in 0..511 (|y| <= 8n), and of the
// bounds at most one, `bound`, can lie among the |y| of r / 8's cell; `below` bounds lie under it.
struct Cells {
  struct Cell {
    float bound;  // +inf: none
    uint32_t below;
  } of[64];
};

// The levels as the fp16 decoders take them: f c_i split into its fp16 value
// and, for fp32 calls, what that leaves over.  The factor f (64 .. 127) keeps the
// rest of the split out of fp16's subnormal range, and the values close to fp16's;
// it is taken out again from the queries and at the end.  `lo` and `hi` are the low and the high bytes of the eight fp16
// values, for byte permutes.
struct Levels {
  float scale;  // f
  uint16_t value[8], rest[8];
  uint32_t lo[2], hi[2];
};

// Bit of a word of codes that holds the sign of coordinate p (0..7) of it.
__host__ __device__ constexpr int sign_bit(int p) { return 4 * p + 3; }

__device__ __forceinline__ float norm_value(uint16_t bits, int norm_bf16) {
  const uint16_t b = bits & 0x7fffu;
  return norm_bf16 ? __uint_as_float((uint32_t)b << 16) : __half2float(__ushort_as_half(b));
}

// Norm as it is held: 16 bits, a finite norm above fp16's range capped at its
// largest value (the vector keeps its direction), a norm that is not finite as
// NaN (the codes could not say which coordinate was not).
__device__ __forceinline__ uint16_t norm_bits(float n, int norm_bf16) {
  if (!(n <= 3.402823466e38f)) return 0x7fffu;
  n = fminf(n, 65504.0f);
  return norm_bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(n)) : __half_as_ushort(__float2half_rn(n));
}

// Slot of a token: byte offset of its block and its place in it.
__device__ __forceinline__ long long block_offset(const Pool& p, int page, int head, int off) {
  return (long long)page * p.page_bytes + (long long)head * p.head_bytes + (long long)(off >> 4) * kBlockBytes;
}

// --- decoding to fp16 -------------------------------------------------------
// A byte permute looks four 3-bit indices up in a table of 8 bytes at once.
// The 8 coordinates of a word as four fp16 pairs (0 1) (2 3) (4 5) (6 7).
__device__ __forceinline__ void decode_pairs(uint32_t w, const uint32_t lo[2], const uint32_t hi[2], uint32_t out[4]) {
  const uint32_t s = w & 0x77777777u, s2 = s >> 16, x = w << 4;
  // the signs of four coordinates as the top bits of four bytes
  const uint32_t n0 = __byte_perm(x, w, 0x5140), n1 = __byte_perm(x, w, 0x7362);
  const uint32_t l0 = __byte_perm(lo[0], lo[1], s), l1 = __byte_perm(lo[0], lo[1], s2);
  const uint32_t h0 = __byte_perm(hi[0], hi[1], s) ^ (n0 & 0x80808080u);
  const uint32_t h1 = __byte_perm(hi[0], hi[1], s2) ^ (n1 & 0x80808080u);
  out[0] = __byte_perm(l0, h0, 0x5140);
  out[1] = __byte_perm(l0, h0, 0x7362);
  out[2] = __byte_perm(l1, h1, 0x5140);
  out[3] = __byte_perm(l1, h1, 0x7362);
}
// Codes of tokens a and b zipped: byte i of u is coordinate 2i of both, of v 2i + 1.
__device__ __forceinline__ void zip(uint32_t a, uint32_t b, uint32_t& u, uint32_t& v) {
  constexpr uint32_t m = 0x0f0f0f0fu;
  u = (a & m) | ((b << 4) & ~m);
  v = ((a >> 4) & m) | (b & ~m);
}

// --- host side --------------------------------------------------------------
// Whether rows and heads start on 16 bytes.
inline bool rows_ok(int dtype, const void* p, int64_t ld, int64_t hs) {
  const int64_t e = dtype == CC2_BF16 ? 8 : 4;  // elements of 16 bytes
  return ((uintptr_t)p & 15u) == 0 && ld % e == 0 && hs % e == 0;
}
int check_cache(const cc2_kv4_cache* c, const char* what, Pool& pool);
int make_turn(const cc2_kv4_quant& q, const char* what, Turn& t);
Levels make_levels(const cc2_kv4_cache& c);
// Device error words of the cache's kernels: DEV_ERR_CACHE_RANGE, and one for waits that ran out.
int error_words(int** p);

}  // namespace kv4
}  // namespace cc2
