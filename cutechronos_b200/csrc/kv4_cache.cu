// Appending to and reading from the paged 4-bit K/V cache (layout: kv4.cuh,
// definition: cc2.h).
//
// Append: y = H (s * x[perm]) of every K (rotated to its position first) and V
// vector, each coordinate to a sign and one of 8 magnitudes, the norm to 16
// bits.  Read: the other way.  The memory's share is small (324 bytes a token
// and head in bf16), so both are bound by the instructions a vector takes, and
// everything here is laid out to save them:
//  - four threads bring a vector in (or out), one thread then owns it whole: its
//    butterflies are register adds, two at a time, with no shuffles;
//  - sign and permutation are applied by the owner, for whom they are constants
//    of the launch: an element is one load at a constant place, times +-1 on
//    the multiply pipe, and rows of 64 floats at a pitch of 65 keep these loads
//    and the four threads' stores free of bank conflicts;
//  - a magnitude takes one lookup and one comparison (Cells): three comparisons
//    of a binary search and their selects ran on the half-rate integer pipe and
//    were its limit;
//  - a block has 16 tokens of 4 heads, so that its owners' codes are 512 bytes
//    in one piece, and rows come in and go out as whole lines: with the 64 units
//    in (token, head) order each owner's 32 bytes were a line of their own;
//  - places in the cache, pointers and positions are worked out once a vector.
// Measured, 131072 tokens of 8 heads, bf16: append 165 us (340 MB, 2.1 TB/s),
// read 96 us (3.5 TB/s); read of 55760 entries of 24 sequences as fp32 53 us
// (4.9 TB/s).  Append uses 77% of the shared-memory pipe's cycles (an owner's 64
// loads, the 64 stores before them, 64 table lookups of which some meet in a
// bank) and 67% of the issue slots; read 68% and 69%; registers (80) and rows
// leave room for 24 warps an SM.  At an earlier state (171 us) tables of single
// words (fewer bank conflicts, one load more) took 174 us; 16 copies of the table
// took 206 and three comparisons in place of the table 260.
#include <algorithm>
#include <cmath>

#include "kv4.cuh"
#include "tc_attn.cuh"

namespace cc2 {
namespace kv4 {

__device__ int g_kv4_error[2] = {0, 0};  // DEV_ERR_CACHE_RANGE; not 0: a wait ran out

int error_words(int** p) {
  static int* at[64] = {};  // per device: the words' address does not change
  int dev = 0;
  CC2_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && at[dev] != nullptr) {
    *p = at[dev];
    return CC2_OK;
  }
  CC2_CUDA(cudaGetSymbolAddress((void**)p, g_kv4_error));
  if (dev < 64) at[dev] = *p;
  return CC2_OK;
}

int check_cache(const cc2_kv4_cache* c, const char* what, Pool& pool) {
  CC2_REQUIRE(c != nullptr && c->pages != nullptr, "%s: null cache", what);
  CC2_REQUIRE(((uintptr_t)c->pages & 15u) == 0, "%s: pages must be 16-byte aligned", what);
  CC2_REQUIRE(c->num_pages > 0 && c->heads > 0, "%s: the cache has no pages or no heads", what);
  size_t bytes = 0;
  CC2_TRY(cc2_kv4_page_bytes(c->page_size, c->heads, &bytes));
  CC2_REQUIRE(c->norm_dtype == 0 || c->norm_dtype == 1, "%s: norm_dtype must be 0 (float16) or 1 (bfloat16)", what);
  CC2_REQUIRE(c->rope_cs == nullptr || c->rope_len > 0, "%s: rope_len must be positive", what);
  CC2_REQUIRE(((uintptr_t)c->rope_cs & 15u) == 0, "%s: rope_cs must be 16-byte aligned", what);
  pool.pages = (uint8_t*)c->pages;
  pool.page_bytes = (long long)bytes;
  pool.head_bytes = c->page_size / kBlockTokens * kBlockBytes;
  pool.num_pages = c->num_pages;
  pool.page_shift = 0;
  while ((1 << pool.page_shift) < c->page_size) ++pool.page_shift;
  pool.heads = c->heads;
  pool.norm_bf16 = c->norm_dtype;
  return CC2_OK;
}

int make_turn(const cc2_kv4_quant& q, const char* what, Turn& t) {
  uint64_t met = 0;
  for (int i = 0; i < 64; ++i) {
    const uint32_t e = q.perm[i] & 63u;
    met |= 1ull << e;
    t.place[i] = 4 * e;
    t.sign[i] = (q.signs >> i) & 1 ? -1.0f : 1.0f;
  }
  CC2_REQUIRE(met == ~0ull, "%s: a quantiser's perm is no permutation", what);
  return CC2_OK;
}

namespace {

int make_cells(const cc2_kv4_cache& cache, const char* what, Cells& r) {
  for (int j = 0; j < 7; ++j)
    CC2_REQUIRE(cache.bounds[j] > (j ? cache.bounds[j - 1] : 0.0f) && cache.bounds[j] < 1.0f,
                "%s: the bounds must ascend between 0 and 1", what);
  int j = 0;  // bounds below the cell
  for (int c = 0; c < 64; ++c) {
    // |y| / 8n of r = 8c .. 8c + 7, with room for the rounding of r itself
    const float lo = (8 * c - 0.52f) / 511.0f, hi = (8 * c + 7.52f) / 511.0f;
    while (j < 7 && cache.bounds[j] <= lo) ++j;
    const bool in = j < 7 && cache.bounds[j] <= hi;
    CC2_REQUIRE(!in || j == 6 || cache.bounds[j + 1] > hi, "%s: the bounds must be more than 1/60 apart", what);
    r.of[c].bound = in ? cache.bounds[j] : INFINITY;
    r.of[c].below = (uint32_t)j;
  }
  return CC2_OK;
}

}  // namespace

namespace {

constexpr int kThreads = 128;
constexpr int kUnits = 64;   // (token, head) pairs a block handles: a thread for each K and each V
constexpr int kInPitch = 65, kOutPitch = 69;  // words of a row: append, read (its halves 4 words apart)

struct Places {
  const int32_t* seq;
  const int32_t* pos;
  const int32_t* table;
  int table_ld, table_cols, num_seqs;  // elements from row to row, entries of a row
};

// Byte offset of the block of token t's head, -1 for a token to skip.
__device__ __forceinline__ long long place(const Pool& pool, const Places& at, int t, int head, int pos_limit, int* off,
                                           int* err) {
  const int s = at.seq[t], pos = at.pos[t];
  if (s < 0 || pos < 0) return -1;
  const int pg = pos >> pool.page_shift;
  if (s >= at.num_seqs || pg >= at.table_cols || pos >= pos_limit) {
    atomicOr(err, (int)DEV_ERR_CACHE_RANGE);
    return -1;
  }
  const int page = at.table[(long long)s * at.table_ld + pg];
  if ((unsigned)page >= (unsigned)pool.num_pages) {
    atomicOr(err, (int)DEV_ERR_CACHE_RANGE);
    return -1;
  }
  *off = pos & ((1 << pool.page_shift) - 1);
  return block_offset(pool, page, head, *off);
}

// Eight neighbouring values as they lie in memory, and as floats.
template <typename T> struct Raw;
template <> struct Raw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <> struct Raw<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float* x) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
// Thread c of 8: its eighth of a row (halves 4 words apart) to memory.
__device__ __forceinline__ void store_part(float* p, const float* row, int c) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float* x = row + 36 * half + 4 * c;
    reinterpret_cast<float4*>(p)[8 * half + c] = make_float4(x[0], x[1], x[2], x[3]);
  }
}
__device__ __forceinline__ void store_part(__nv_bfloat16* p, const float* row, int c) {
  const float* x = row + 8 * c + (c & 4);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&h);
  }
  reinterpret_cast<uint4*>(p)[c] = make_uint4(w[0], w[1], w[2], w[3]);
}

// Butterflies of width 1, 2, ..., 32 over 64 registers, each sum and difference rounded once: width 1 within pairs of
// neighbours, the others two at a time (a - b as a + b * -1, the product exact).
__device__ __forceinline__ void walsh(float (&y)[64]) {
  using namespace tcx;
  uint64_t p[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) p[i] = f2_pack(__fadd_rn(y[2 * i], y[2 * i + 1]), __fsub_rn(y[2 * i], y[2 * i + 1]));
  const uint64_t minus = f2_pack(-1.0f, -1.0f);
#pragma unroll
  for (int w = 1; w < 32; w <<= 1)
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (!(i & w)) {
        const uint64_t a = p[i], b = p[i + w];
        p[i] = f2_add(a, b);
        p[i + w] = f2_fma(b, minus, a);
      }
#pragma unroll
  for (int i = 0; i < 32; ++i) f2_unpack(p[i], y[2 * i], y[2 * i + 1]);
}

// What a block knows of its units.
struct Unit {
  long long block;   // byte offset of the unit's block of 16 tokens, -1: skip
  int pos;           // to rotate to
  int slot;          // place in the block of 16; bit 8: masked
};

// A block's 64 units: 16 neighbouring tokens of each of 4 heads (the next 16
// tokens' where the heads run out).  Their rows in shared memory are 4 t + h: a
// warp that brings 8 rows in or out has one or two tokens' (one line of RoPE
// factors for 4 of them); the owners, lane = token, have 16 neighbours of a head,
// whose codes are 512 bytes in one piece.
struct Units {
  int tokens, heads;
  // of row r; false past the end (then the last token's)
  __device__ __forceinline__ bool find(int r, int& t, int& h) const {
    const unsigned q = blockIdx.x * 4u + ((unsigned)r & 3u), run = q / (unsigned)heads;
    h = (int)(q - run * (unsigned)heads);
    t = (int)run * 16 + (r >> 2);
    const bool is = t < tokens;
    t = min(t, tokens - 1);
    return is;
  }
  static __device__ __forceinline__ int row_of(int tid) { return 4 * (tid & 15) + ((tid >> 4) & 3); }
};
// Place of a row of floats: the second 32 rows two words on, which keeps the
// owners' accesses (rows 4 apart and two heads) free of bank conflicts at a pitch
// that is odd.
template <int kPitch> __device__ __forceinline__ int row_at(int row) { return row * kPitch + 2 * (row >> 5); }
template <int kPitch> constexpr int kRowsWords = 2 * kUnits * kPitch + 8;

// An owner's row: at constant places, times constant signs.
__device__ __forceinline__ void take_row(const float* row, const Turn& turn, float (&y)[64]) {
#pragma unroll
  for (int i = 0; i < 64; ++i)
    y[i] = __fmul_rn(*reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(row) + turn.place[i]), turn.sign[i]);
}

template <typename T, bool kRope>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 6 : 5)
append_kernel(const __grid_constant__ Pool pool, const __grid_constant__ Turn turn_k, const __grid_constant__ Turn turn_v,
              const __grid_constant__ Cells table, const T* __restrict__ k, long long k_ld, long long k_hs,
              const T* __restrict__ v, long long v_ld, long long v_hs, int tokens, Places at,
              const uint8_t* __restrict__ mask, const float2* __restrict__ rope, int rope_len, int* __restrict__ err) {
  pdl_launch_dependents();
  __shared__ __align__(16) float rows[kRowsWords<kInPitch>];
  __shared__ float norm[2 * kUnits];
  __shared__ Cells::Cell cells[64];
  __shared__ Unit units[kUnits];
  constexpr int kIts = kUnits * 4 / kThreads;
  const int tid = threadIdx.x;
  if (tid < 64) cells[tid] = table.of[tid];
  pdl_wait();
  const Units my{tokens, pool.heads};

  // four threads bring a vector in: thread c its values 8c .. 8c+7 and 32 + 8c ..
  const int c = tid & 3;
  Raw<T> raw[2][kIts][2];
#pragma unroll
  for (int it = 0; it < kIts; ++it) {
    int t, h;
    my.find(it * (kThreads / 4) + (tid >> 2), t, h);
    const T* from = k + (long long)t * k_ld + (long long)h * k_hs + 8 * c;
    raw[0][it][0].load(from);
    raw[0][it][1].load(from + 32);
    from = v + (long long)t * v_ld + (long long)h * v_hs + 8 * c;
    raw[1][it][0].load(from);
    raw[1][it][1].load(from + 32);
  }
  if (tid < kUnits) {
    Unit u;
    u.block = -1;
    u.pos = 0;
    u.slot = 0;
    int t, h;
    if (my.find(tid, t, h)) {
      int off = 0;
      u.block = place(pool, at, t, h, kRope ? rope_len : 0x7fffffff, &off, err);
      u.slot = (off & (kBlockTokens - 1)) | (mask != nullptr && mask[t] == 0 ? 256 : 0);
      if (kRope && u.block >= 0) u.pos = at.pos[t];
    }
    units[tid] = u;
  }
  __syncthreads();

#pragma unroll
  for (int is_v = 1; is_v >= 0; --is_v) {
#pragma unroll
    for (int it = 0; it < kIts; ++it) {
      const int r = it * (kThreads / 4) + (tid >> 2);
      float a[8], b[8];
      raw[is_v][it][0].get(a);
      raw[is_v][it][1].get(b);
      if (kRope && !is_v) {
        const float4* cs = reinterpret_cast<const float4*>(rope + (long long)units[r].pos * 32 + 8 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 f = cs[j];
          const float a0 = a[2 * j], b0 = b[2 * j], a1 = a[2 * j + 1], b1 = b[2 * j + 1];
          a[2 * j] = __fsub_rn(__fmul_rn(a0, f.x), __fmul_rn(b0, f.y));
          b[2 * j] = __fadd_rn(__fmul_rn(b0, f.x), __fmul_rn(a0, f.y));
          a[2 * j + 1] = __fsub_rn(__fmul_rn(a1, f.z), __fmul_rn(b1, f.w));
          b[2 * j + 1] = __fadd_rn(__fmul_rn(b1, f.z), __fmul_rn(a1, f.w));
        }
      }
      // squares added in halves: i and i + 32, then 16 and 8 apart (the threads of
      // a vector), then 4, 2, 1 apart
      float s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = __fadd_rn(__fmul_rn(a[j], a[j]), __fmul_rn(b[j], b[j]));
      // each thread keeps half of the sums at either step, j and j + 4 together
      const bool up = (c & 2) != 0, odd = (c & 1) != 0;
      float h[4];  // j = 0, 1, 4, 5 or 2, 3, 6, 7
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = (i & 1) + 2 * (i & 2);
        h[i] = __fadd_rn(up ? s[j + 2] : s[j], __shfl_xor_sync(0xffffffffu, up ? s[j] : s[j + 2], 2));
      }
      float n2 = __fadd_rn(__fadd_rn(odd ? h[1] : h[0], __shfl_xor_sync(0xffffffffu, odd ? h[0] : h[1], 1)),
                           __fadd_rn(odd ? h[3] : h[2], __shfl_xor_sync(0xffffffffu, odd ? h[2] : h[3], 1)));
      n2 = __fadd_rn(n2, __shfl_xor_sync(0xffffffffu, n2, 2));
      n2 = __fadd_rn(n2, __shfl_xor_sync(0xffffffffu, n2, 1));
      float* row = rows + row_at<kInPitch>(is_v * kUnits + r) + 8 * c;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        row[j] = a[j];
        row[32 + j] = b[j];
      }
      if (c == 0) norm[is_v * kUnits + r] = __fsqrt_rn(n2);
    }
  }
  __syncthreads();

  const int is_v = tid >= kUnits;  // whole warps
  const int mine = is_v * kUnits + Units::row_of(tid);
  const Unit& u = units[mine & (kUnits - 1)];
  if (u.block < 0) return;
  float y[64];
  if (is_v) take_row(rows + row_at<kInPitch>(mine), turn_v, y);  // two copies, each with its own constants
  else take_row(rows + row_at<kInPitch>(mine), turn_k, y);
  walsh(y);
  const float n = norm[mine];
  const float n8 = __fmul_rn(n, 8.0f);
  if (n8 > 0.0f && n8 < 0x1p-50f) {  // squares may have lost bits below fp32's range: a |y| above 8n would leave the cells
#pragma unroll
    for (int i = 0; i < 64; ++i) y[i] = fminf(fmaxf(y[i], -n8), n8);
  }
  const float fine = n8 > 0.0f ? __fdividef(511.0f, n8) : 0.0f;  // its error is within the cells' room
  const uint8_t* entries = reinterpret_cast<const uint8_t*>(cells);
  uint32_t word[8];
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    uint32_t code = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const float x = y[8 * w + p], a = fabsf(x);
      // r in the low bits of 2^23 + r: its cell's entry (a NaN points at one of them too)
      const uint32_t r = __float_as_uint(fmaf(a, fine, 8388608.0f)) & 0x1f8u;
      const Cells::Cell cell = *reinterpret_cast<const Cells::Cell*>(entries + r);
      code += cell.below * (1u << (4 * p));
      if (a > __fmul_rn(cell.bound, n8)) code += 1u << (4 * p);
      if (x < 0.0f) code |= 1u << sign_bit(p);
    }
    word[w] = code;
  }
  uint8_t* block = pool.pages + u.block;
  const int slot = u.slot & 255;
  uint4* codes = reinterpret_cast<uint4*>(block + (is_v ? kVCodes : 0) + slot * 32);
  codes[0] = make_uint4(word[0], word[1], word[2], word[3]);
  codes[1] = make_uint4(word[4], word[5], word[6], word[7]);
  uint16_t nb = norm_bits(n, pool.norm_bf16);
  if (!is_v && (u.slot & 256)) nb |= 0x8000u;
  reinterpret_cast<uint16_t*>(block + kNorms)[2 * slot + is_v] = nb;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 6)
read_kernel(const __grid_constant__ Pool pool, const __grid_constant__ Turn turn_k, const __grid_constant__ Turn turn_v,
            const float4 levels_lo, const float4 levels_hi, T* __restrict__ k_out, T* __restrict__ v_out, int tokens,
            Places at, int* __restrict__ err) {
  pdl_launch_dependents();
  __shared__ __align__(16) float rows[kRowsWords<kOutPitch>];
  __shared__ __align__(16) float level[16];  // of a code, sign and magnitude
  const int tid = threadIdx.x;
  if (tid == 0) {
    float4* to = reinterpret_cast<float4*>(level);
    to[0] = levels_lo;
    to[1] = levels_hi;
    to[2] = make_float4(-levels_lo.x, -levels_lo.y, -levels_lo.z, -levels_lo.w);
    to[3] = make_float4(-levels_hi.x, -levels_hi.y, -levels_hi.z, -levels_hi.w);
  }
  pdl_wait();
  __syncthreads();
  const Units my{tokens, pool.heads};
  {
    const bool is_v = tid >= kUnits;
    int off = 0, t, h;
    long long at_block = -1;
    if (my.find(Units::row_of(tid), t, h) && (is_v ? v_out : k_out) != nullptr)
      at_block = place(pool, at, t, h, 0x7fffffff, &off, err);
    float f = 0.0f;
    float y[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) y[i] = 0.0f;
    if (at_block >= 0) {
      const uint8_t* block = pool.pages + at_block;
      const int slot = off & (kBlockTokens - 1);
      const uint4* codes = reinterpret_cast<const uint4*>(block + (is_v ? kVCodes : 0) + slot * 32);
      const uint4 w0 = codes[0], w1 = codes[1];
      const uint32_t word[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
      f = 0.125f * norm_value(reinterpret_cast<const uint16_t*>(block + kNorms)[2 * slot + is_v], pool.norm_bf16);
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const uint32_t w = word[i >> 3];
        const int p = i & 7;
        const uint32_t sel = (p ? w >> (4 * p - 2) : w << 2) & 60u;  // a level's byte offset
        y[i] = *reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(level) + sel);
      }
      walsh(y);
    }
    uint8_t* row = reinterpret_cast<uint8_t*>(rows + row_at<kOutPitch>(is_v * kUnits + Units::row_of(tid)));
    if (is_v) {
#pragma unroll
      for (int i = 0; i < 64; ++i)
        *reinterpret_cast<float*>(row + turn_v.place[i]) = __fmul_rn(__fmul_rn(y[i], f), turn_v.sign[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 64; ++i)
        *reinterpret_cast<float*>(row + turn_k.place[i]) = __fmul_rn(__fmul_rn(y[i], f), turn_k.sign[i]);
    }
  }
  __syncthreads();
  // eight threads a row: whole lines
  const int c = tid & 7;
#pragma unroll
  for (int is_v = 0; is_v < 2; ++is_v) {
    T* out = is_v ? v_out : k_out;
    if (out == nullptr) continue;
#pragma unroll
    for (int it = 0; it < kUnits * 8 / kThreads; ++it) {
      const int r = it * (kThreads / 8) + (tid >> 3);
      int t, h;
      if (!my.find(r, t, h)) continue;
      const float* row = rows + row_at<kOutPitch>(is_v * kUnits + r);
      store_part(out + ((long long)t * pool.heads + h) * 64, row, c);
    }
  }
}

// 64-bit indexes to 32 bits, what does not fit to the nearest that does.
__global__ void __launch_bounds__(256)
index32_kernel(const int64_t* __restrict__ in, long long ld, long long inc, unsigned cols, unsigned n, int32_t* __restrict__ out) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= n) return;
  const int64_t v = in[(long long)(i / cols) * ld + (long long)(i % cols) * inc];
  out[i] = (int32_t)max(min((long long)v, 0x7fffffffLL), -0x80000000LL);
}

int check_places(const char* what, int T, const int32_t* seq, const int32_t* pos, const int32_t* table, int table_ld,
                 int table_cols, int num_seqs) {
  CC2_REQUIRE(T >= 0 && seq && pos && table, "%s: null sequences, positions or block table", what);
  CC2_REQUIRE(table_cols > 0 && num_seqs > 0, "%s: empty block table", what);
  CC2_REQUIRE(table_cols <= table_ld, "%s: block table of %d columns with rows %d apart", what, table_cols, table_ld);
  return CC2_OK;
}

int grid_of(int T, int heads, int* grid) {
  const long long blocks = (((long long)T + 15) / 16 * heads + 3) / 4;
  CC2_REQUIRE(blocks <= 0x1fffffffLL, "kv4: too many tokens for one call");
  *grid = (int)blocks;
  return CC2_OK;
}

}  // namespace
}  // namespace kv4

int read_kv4_error(int clear, int* value) {
  int words[2];
  CC2_CUDA(cudaMemcpyFromSymbol(words, kv4::g_kv4_error, sizeof words));
  *value = words[0] | (words[1] ? DEV_ERR_CACHE_TIMEOUT : 0);
  if (clear) {
    const int z[2] = {0, 0};
    CC2_CUDA(cudaMemcpyToSymbol(kv4::g_kv4_error, z, sizeof z));
  }
  return CC2_OK;
}

int launch_kv4_index32(const int64_t* in, int64_t ld, int64_t inc, int rows, int cols, int32_t* out, cudaStream_t st) {
  CC2_REQUIRE(rows >= 0 && cols >= 0 && (long long)rows * cols <= 0x7fffffffLL, "kv4_index32: bad size %d x %d", rows, cols);
  const unsigned n = (unsigned)rows * (unsigned)cols;
  if (n == 0) return CC2_OK;
  CC2_REQUIRE(in && out, "kv4_index32: null operand");
  CC2_CUDA(launch_k(kv4::index32_kernel, (n + 255u) / 256u, 256, 0, st, in, (long long)ld, (long long)inc, (unsigned)cols, n, out));
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

int launch_kv4_append(const cc2_kv4_cache* cache, int dtype, const void* k, int64_t k_ld, int64_t k_hs, const void* v,
                      int64_t v_ld, int64_t v_hs, int T, const int32_t* seq, const int32_t* pos, const uint8_t* mask,
                      const int32_t* table, int table_ld, int table_cols, int num_seqs, cudaStream_t st) {
  using namespace kv4;
  Pool pool;
  CC2_TRY(check_cache(cache, "kv4_append", pool));
  CC2_REQUIRE(dtype == CC2_BF16 || dtype == CC2_F32, "kv4_append: unsupported dtype %d", dtype);
  if (T == 0) return CC2_OK;
  CC2_TRY(check_places("kv4_append", T, seq, pos, table, table_ld, table_cols, num_seqs));
  CC2_REQUIRE(k && v, "kv4_append: null keys or values");
  CC2_REQUIRE(rows_ok(dtype, k, k_ld, k_hs) && rows_ok(dtype, v, v_ld, v_hs),
              "kv4_append: keys and values must start on 16 bytes, as must their strides");
  int grid = 0, *err = nullptr;
  CC2_TRY(grid_of(T, pool.heads, &grid));
  CC2_TRY(error_words(&err));
  Turn turn_k, turn_v;
  Cells cells;
  CC2_TRY(make_turn(cache->key, "kv4_append", turn_k));
  CC2_TRY(make_turn(cache->value, "kv4_append", turn_v));
  CC2_TRY(make_cells(*cache, "kv4_append", cells));
  const Places at{seq, pos, table, table_ld, table_cols, num_seqs};
  const float2* rope = (const float2*)cache->rope_cs;
#define CC2_APPEND(TT, ROPE)                                                                                        \
  CC2_CUDA(launch_k(append_kernel<TT, ROPE>, grid, kThreads, 0, st, pool, turn_k, turn_v, cells, (const TT*)k, (long long)k_ld,    \
                    (long long)k_hs, (const TT*)v, (long long)v_ld, (long long)v_hs, T, at, mask, rope,             \
                    cache->rope_len, err))
  if (dtype == CC2_BF16) {
    if (rope != nullptr) CC2_APPEND(__nv_bfloat16, true); else CC2_APPEND(__nv_bfloat16, false);
  } else {
    if (rope != nullptr) CC2_APPEND(float, true); else CC2_APPEND(float, false);
  }
#undef CC2_APPEND
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

int launch_kv4_read(const cc2_kv4_cache* cache, int dtype, void* k_out, void* v_out, int T, const int32_t* seq,
                    const int32_t* pos, const int32_t* table, int table_ld, int table_cols, int num_seqs,
                    cudaStream_t st) {
  using namespace kv4;
  Pool pool;
  CC2_TRY(check_cache(cache, "kv4_read", pool));
  CC2_REQUIRE(dtype == CC2_BF16 || dtype == CC2_F32, "kv4_read: unsupported dtype %d", dtype);
  if (T == 0 || (!k_out && !v_out)) return CC2_OK;
  CC2_TRY(check_places("kv4_read", T, seq, pos, table, table_ld, table_cols, num_seqs));
  CC2_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15u) == 0, "kv4_read: outputs must be 16-byte aligned");
  int grid = 0, *err = nullptr;
  CC2_TRY(grid_of(T, pool.heads, &grid));
  CC2_TRY(error_words(&err));
  Turn turn_k, turn_v;
  CC2_TRY(make_turn(cache->key, "kv4_read", turn_k));
  CC2_TRY(make_turn(cache->value, "kv4_read", turn_v));
  for (int i = 0; i < 64; ++i) {  // the second half of a row is 4 words on
    turn_k.place[i] += turn_k.place[i] >= 128 ? 16u : 0u;
    turn_v.place[i] += turn_v.place[i] >= 128 ? 16u : 0u;
  }
  const float* lv = cache->levels;
  const float4 lo = make_float4(lv[0], lv[1], lv[2], lv[3]), hi = make_float4(lv[4], lv[5], lv[6], lv[7]);
  const Places at{seq, pos, table, table_ld, table_cols, num_seqs};
  if (dtype == CC2_BF16) {
    CC2_CUDA(launch_k(read_kernel<__nv_bfloat16>, grid, kThreads, 0, st, pool, turn_k, turn_v, lo, hi,
                      (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, T, at, err));
  } else {
    CC2_CUDA(launch_k(read_kernel<float>, grid, kThreads, 0, st, pool, turn_k, turn_v, lo, hi, (float*)k_out,
                      (float*)v_out, T, at, err));
  }
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

}  // namespace cc2

extern "C" int cc2_kv4_page_bytes(int page_size, int heads, size_t* bytes) {
  using namespace cc2;
  CC2_REQUIRE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
              "kv4: page_size must be 16, 32, 64, 128 or 256, got %d", page_size);
  CC2_REQUIRE(heads > 0 && heads <= 65536, "kv4: bad number of heads %d", heads);
  CC2_REQUIRE(bytes != nullptr, "kv4: bytes is null");
  *bytes = (size_t)heads * (page_size / kv4::kBlockTokens) * kv4::kBlockBytes;
  return CC2_OK;
}
