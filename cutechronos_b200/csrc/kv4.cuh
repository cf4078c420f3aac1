// The paged K/V cache held in 4 bits: its layout in memory, the quantiser's
// tables as the kernels take them, and the codes' decoding to fp16 pairs.
//
// Pool: page-major.  A page holds, for each head, page_size / 16 blocks of 16
// tokens, and a block is 1088 consecutive bytes
//     [16 x 32 bytes K codes | 16 x 32 bytes V codes | 16 x (K norm, V norm)]
// so that everything attention needs of 16 tokens of a head is one aligned
// run of memory, and of a page one longer run: one bulk copy brings it.
//
// A vector's 64 codes are 8 words; nibble p of word w holds the 3-bit magnitude
// index of coordinate 8w + p in its low bits.  The nibbles' top bits hold the
// signs, but not each its own nibble's: bits 7, 15, 23, 31 are coordinates
// 0..3's and bits 3, 11, 19, 27 coordinates 4..7's, so that a decoder merges
// four signs with four looked-up bytes in one operation, whether it makes
// pairs of neighbouring coordinates of one token (decode_pairs) or of one
// coordinate of two tokens (decode_zip).  A key norm's sign bit marks a
// masked token.
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

// One quantiser for the kernels that quantise and restore (by value).
struct Quant {
  float levels[8];
  // Element e of a vector is rotated coordinate go[e] & 63, negated if bit 7 is set.
  uint8_t go[64];
  // The magnitude by one comparison: r = round(512 |y| / 8n) is in 0..512 (|y| <= 8n), and of the bounds at most one,
  // `bound`, can lie among the |y| of r / 8's cell; `below` bounds lie under it.
  struct Cell {
    float bound;  // +inf: none
    uint32_t below;
  } cells[65];
};

// Level tables of the fp16 decoder: 64 c_i split into its fp16 value and, for
// fp32 calls, what that leaves over, each as four words: bytes 0 and 1 of the
// eight values (8 low bytes, 8 high bytes).  The factor 64 keeps the rest of
// the split out of fp16's subnormal range; it is exact and taken out again at
// the end.
struct Levels {
  uint32_t lo[2], hi[2];    // fp16(64 c)
  uint32_t rlo[2], rhi[2];  // fp16(64 c - fp16(64 c))
};

// Bit of a word of codes that holds the sign of coordinate p (0..7) of it.
__host__ __device__ constexpr int sign_bit(int p) { return p < 4 ? 8 * p + 7 : 8 * (p - 4) + 3; }

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
__device__ __forceinline__ uint32_t look(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// The 8 coordinates of a word as four fp16 pairs (0 1) (2 3) (4 5) (6 7).
__device__ __forceinline__ void decode_pairs(uint32_t w, const uint32_t lo[2], const uint32_t hi[2], uint32_t out[4]) {
  const uint32_t s = w & 0x77777777u, s2 = s >> 16;
  const uint32_t l0 = look(lo[0], lo[1], s), l1 = look(lo[0], lo[1], s2);
  const uint32_t h0 = look(hi[0], hi[1], s) ^ (w & 0x80808080u);
  const uint32_t h1 = look(hi[0], hi[1], s2) ^ ((w << 4) & 0x80808080u);
  out[0] = __byte_perm(l0, h0, 0x5140);
  out[1] = __byte_perm(l0, h0, 0x7362);
  out[2] = __byte_perm(l1, h1, 0x5140);
  out[3] = __byte_perm(l1, h1, 0x7362);
}

// Coordinate p of tokens a and b as the fp16 pair out[p], p = 0..7.
struct Zip {
  uint32_t u, v, su, sv, tu, tv;  // selectors of even / odd coordinates; their signs (low, high half)
};
__device__ __forceinline__ Zip zip(uint32_t a, uint32_t b) {
  constexpr uint32_t m = 0x0f0f0f0fu;
  Zip z;
  z.u = ((a & m) | ((b << 4) & ~m)) & 0x77777777u;
  z.v = (((a >> 4) & m) | (b & ~m)) & 0x77777777u;
  const uint32_t s0 = __byte_perm(a, b, 0x6240), s1 = __byte_perm(a, b, 0x7351);
  z.su = s0 & 0x80808080u;
  z.tu = (s0 << 4) & 0x80808080u;
  z.sv = s1 & 0x80808080u;
  z.tv = (s1 << 4) & 0x80808080u;
  return z;
}
__device__ __forceinline__ void decode_zip(const Zip& z, const uint32_t lo[2], const uint32_t hi[2], uint32_t out[8]) {
  uint32_t l, h;
  l = look(lo[0], lo[1], z.u);
  h = look(hi[0], hi[1], z.u) ^ z.su;
  out[0] = __byte_perm(l, h, 0x5140);
  out[2] = __byte_perm(l, h, 0x7362);
  l = look(lo[0], lo[1], z.u >> 16);
  h = look(hi[0], hi[1], z.u >> 16) ^ z.tu;
  out[4] = __byte_perm(l, h, 0x5140);
  out[6] = __byte_perm(l, h, 0x7362);
  l = look(lo[0], lo[1], z.v);
  h = look(hi[0], hi[1], z.v) ^ z.sv;
  out[1] = __byte_perm(l, h, 0x5140);
  out[3] = __byte_perm(l, h, 0x7362);
  l = look(lo[0], lo[1], z.v >> 16);
  h = look(hi[0], hi[1], z.v >> 16) ^ z.tv;
  out[5] = __byte_perm(l, h, 0x5140);
  out[7] = __byte_perm(l, h, 0x7362);
}

// --- host side --------------------------------------------------------------
int check_cache(const cc2_kv4_cache* c, const char* what, Pool& pool);
int make_quant(const cc2_kv4_quant& q, const char* what, Quant& r);
Levels make_levels(const cc2_kv4_quant& q);
// Device error word of the cache's kernels (DEV_ERR_CACHE_RANGE).
int error_word(int** p);

}  // namespace kv4
}  // namespace cc2
