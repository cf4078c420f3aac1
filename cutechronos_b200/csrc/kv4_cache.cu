// Appending to and reading from the paged 4-bit K/V cache (layout: kv4.cuh,
// definition: cc2.h).
//
// Append: y = H (s * x[perm]) / (8 n) of every K (rotated to its position
// first) and V vector, each coordinate to a sign and one of 8 magnitudes, the
// norm to 16 bits.  Bound by the arithmetic next to the memory: a token's head
// moves 324 bytes (bf16), about 5e-11 s of the card's copy rate, and takes some
// 2,300 operations, about 6e-11 s of its fp32 lanes.
// So one thread owns a whole vector: the butterflies are 64 register adds a
// width with no shuffles, sign and permutation are the same for all threads of
// a warp, and the permutation costs nothing beyond the shared-memory read that
// brings the vector in.  Rows of 64 floats at a pitch of 65 make that read and
// the write before it free of bank conflicts.  Codes leave as two 16-byte
// stores a thread.
#include <algorithm>

#include "kv4.cuh"

namespace cc2 {
namespace kv4 {

__device__ int g_kv4_error = 0;

int error_word(int** p) {
  static int* at[64] = {};  // per device: the word's address does not change
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

Quant make_quant(const cc2_kv4_quant& q) {
  Quant r;
  for (int i = 0; i < 8; ++i) r.levels[i] = q.levels[i];
  for (int i = 0; i < 7; ++i) r.bounds[i] = q.bounds[i];
  r.signs[0] = (uint32_t)q.signs;
  r.signs[1] = (uint32_t)(q.signs >> 32);
  for (int i = 0; i < 64; ++i) r.perm[i] = q.perm[i] & 63;
  return r;
}

namespace {

constexpr int kThreads = 128;
constexpr int kUnits = 64;   // (token, head) pairs a block handles: a thread for each K and each V
constexpr int kPitch = 65;

struct Places {
  const int32_t* seq;
  const int32_t* pos;
  const int32_t* table;
  int table_ld, num_seqs;
};

// Byte offset of the block of token t's head, -1 for a token to skip.
__device__ __forceinline__ long long place(const Pool& pool, const Places& at, int t, int head, int pos_limit, int* off,
                                           int* err) {
  const int s = at.seq[t], pos = at.pos[t];
  if (s < 0 || pos < 0) return -1;
  const int pg = pos >> pool.page_shift;
  if (s >= at.num_seqs || pg >= at.table_ld || pos >= pos_limit) {
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

template <typename T> __device__ __forceinline__ void load8(const T* p, float* x);
template <> __device__ __forceinline__ void load8<float>(const float* p, float* x) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* x) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* x);
template <> __device__ __forceinline__ void store8<float>(float* p, const float* x) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Butterflies of width 1, 2, ..., 32 over 64 registers.
__device__ __forceinline__ void walsh(float (&y)[64]) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      if (i & w) continue;
      const float a = y[i], b = y[i + w];
      y[i] = __fadd_rn(a, b);
      y[i + w] = __fsub_rn(a, b);
    }
  }
}

__device__ __forceinline__ void encode(const float (&y)[64], float n8, const Quant& q, uint32_t (&word)[8]) {
  float t[7];
#pragma unroll
  for (int j = 0; j < 7; ++j) t[j] = __fmul_rn(q.bounds[j], n8);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    uint32_t c = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) {  // three comparisons find the magnitude: 4, 2, 1
      const float v = y[8 * w + p], a = fabsf(v);
      const bool h = a > t[3];
      const bool m = a > (h ? t[5] : t[1]);
      const bool l = a > (m ? (h ? t[6] : t[2]) : (h ? t[4] : t[0]));
      c |= (h ? 4u << (4 * p) : 0u) | (m ? 2u << (4 * p) : 0u) | (l ? 1u << (4 * p) : 0u);
      c |= v < 0.0f ? 1u << sign_bit(p) : 0u;
    }
    word[w] = c;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
append_kernel(const __grid_constant__ Pool pool, const __grid_constant__ Quant qk, const __grid_constant__ Quant qv,
              const T* __restrict__ k, long long k_ld, long long k_hs, const T* __restrict__ v, long long v_ld,
              long long v_hs, int tokens, Places at, const uint8_t* __restrict__ mask,
              const float2* __restrict__ rope, int rope_len, int* __restrict__ err) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float rows[2 * kUnits * kPitch];
  __shared__ float norm[2 * kUnits];
  const int tid = threadIdx.x;
  const long long units = (long long)tokens * pool.heads;
  const long long u0 = (long long)blockIdx.x * kUnits;
  const int pos_limit = rope != nullptr ? rope_len : 0x7fffffff;

  // four threads bring a vector in: thread c its values 8c .. 8c+7 and 32 + 8c ..
#pragma unroll
  for (int it = 0; it < 2 * kUnits * 4 / kThreads; ++it) {
    const int task = it * kThreads + tid, r = task >> 2, c = task & 3;
    const bool is_v = r >= kUnits;
    const long long u = u0 + (r & (kUnits - 1));
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.0f;
    if (u < units) {
      const int t = (int)(u / pool.heads), h = (int)(u % pool.heads);
      const T* x = is_v ? v + (long long)t * v_ld + (long long)h * v_hs : k + (long long)t * k_ld + (long long)h * k_hs;
      load8(x + 8 * c, a);
      load8(x + 32 + 8 * c, b);
      if (!is_v && rope != nullptr) {
        const int pos = at.pos[t];
        if (pos >= 0 && pos < rope_len) {
          const float4* cs = reinterpret_cast<const float4*>(rope + (long long)pos * 32 + 8 * c);
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
      }
    }
    // squares added in halves: i and i + 32, then 16 and 8 apart (the threads of
    // a vector), then 4, 2, 1 apart
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __fadd_rn(__fmul_rn(a[j], a[j]), __fmul_rn(b[j], b[j]));
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = __fadd_rn(s[j], __shfl_xor_sync(0xffffffffu, s[j], o));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
      for (int j = 0; j < o; ++j) s[j] = __fadd_rn(s[j], s[j + o]);
    }
    float* row = rows + r * kPitch;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      row[8 * c + j] = a[j];
      row[32 + 8 * c + j] = b[j];
    }
    if (c == 0) norm[r] = __fsqrt_rn(s[0]);
  }
  __syncthreads();

  const bool is_v = tid >= kUnits;  // whole warps
  const long long u = u0 + (tid & (kUnits - 1));
  if (u >= units) return;
  const int t = (int)(u / pool.heads), h = (int)(u % pool.heads);
  int off = 0;
  const long long at_block = place(pool, at, t, h, pos_limit, &off, err);
  if (at_block < 0) return;
  const float* row = rows + tid * kPitch;
  const float n = norm[tid];
  const float n8 = __fmul_rn(n, 8.0f);
  const Quant& q = is_v ? qv : qk;
  float y[64];
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const float x = row[q.perm[i]];
    y[i] = (q.signs[i >> 5] >> (i & 31)) & 1u ? -x : x;
  }
  walsh(y);
  uint32_t word[8];
  encode(y, n8, q, word);
  uint8_t* block = pool.pages + at_block;
  const int slot = off & (kBlockTokens - 1);
  uint4* codes = reinterpret_cast<uint4*>(block + (is_v ? kVCodes : 0) + slot * 32);
  codes[0] = make_uint4(word[0], word[1], word[2], word[3]);
  codes[1] = make_uint4(word[4], word[5], word[6], word[7]);
  uint16_t nb = norm_bits(n, pool.norm_bf16);
  if (!is_v && mask != nullptr && mask[t] == 0) nb |= 0x8000u;
  reinterpret_cast<uint16_t*>(block + (is_v ? kVNorms : kKNorms))[slot] = nb;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
read_kernel(const __grid_constant__ Pool pool, const __grid_constant__ Quant qk, const __grid_constant__ Quant qv,
            T* __restrict__ k_out, T* __restrict__ v_out, int tokens, Places at, int* __restrict__ err) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float rows[2 * kUnits * kPitch];
  __shared__ float level[2][8];
  const int tid = threadIdx.x;
  const long long units = (long long)tokens * pool.heads;
  const long long u0 = (long long)blockIdx.x * kUnits;
  if (tid < 16) level[tid >> 3][tid & 7] = (tid >> 3 ? qv : qk).levels[tid & 7];
  __syncthreads();
  {
    const bool is_v = tid >= kUnits;
    const long long u = u0 + (tid & (kUnits - 1));
    int off = 0;
    long long at_block = -1;
    if (u < units && (is_v ? v_out : k_out) != nullptr)
      at_block = place(pool, at, (int)(u / pool.heads), (int)(u % pool.heads), 0x7fffffff, &off, err);
    const Quant& q = is_v ? qv : qk;
    float* row = rows + tid * kPitch;
    if (at_block >= 0) {
      const uint8_t* block = pool.pages + at_block;
      const int slot = off & (kBlockTokens - 1);
      const uint4* codes = reinterpret_cast<const uint4*>(block + (is_v ? kVCodes : 0) + slot * 32);
      const uint4 w0 = codes[0], w1 = codes[1];
      const uint32_t word[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
      const float f = 0.125f * norm_value(reinterpret_cast<const uint16_t*>(block + (is_v ? kVNorms : kKNorms))[slot],
                                          pool.norm_bf16);
      const float* lv = level[is_v];
      float y[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const uint32_t w = word[i >> 3];
        const float c = lv[(w >> (4 * (i & 7))) & 7u];
        y[i] = __uint_as_float(__float_as_uint(c) ^ ((w << (31 - sign_bit(i & 7))) & 0x80000000u));
      }
      walsh(y);
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const float x = __fmul_rn(y[i], f);
        row[q.perm[i]] = (q.signs[i >> 5] >> (i & 31)) & 1u ? -x : x;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 64; ++i) row[i] = 0.0f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 2 * kUnits * 4 / kThreads; ++it) {
    const int task = it * kThreads + tid, r = task >> 2, c = task & 3;
    const bool is_v = r >= kUnits;
    const long long u = u0 + (r & (kUnits - 1));
    T* out = is_v ? v_out : k_out;
    if (u >= units || out == nullptr) continue;
    const float* row = rows + r * kPitch;
    float a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] = row[8 * c + j];
      b[j] = row[32 + 8 * c + j];
    }
    store8(out + u * 64 + 8 * c, a);
    store8(out + u * 64 + 32 + 8 * c, b);
  }
}

int check_places(const char* what, int T, const int32_t* seq, const int32_t* pos, const int32_t* table, int table_ld,
                 int num_seqs) {
  CC2_REQUIRE(T >= 0 && seq && pos && table, "%s: null sequences, positions or block table", what);
  CC2_REQUIRE(table_ld > 0 && num_seqs > 0, "%s: empty block table", what);
  return CC2_OK;
}

bool rows_ok(int dtype, const void* p, int64_t ld, int64_t hs) {
  const int64_t e = dtype == CC2_BF16 ? 8 : 4;  // elements of 16 bytes
  return ((uintptr_t)p & 15u) == 0 && ld % e == 0 && hs % e == 0;
}

int grid_of(int T, int heads, int* grid) {
  const long long blocks = ((long long)T * heads + kUnits - 1) / kUnits;
  CC2_REQUIRE(blocks <= 0x7fffffffLL, "kv4: too many tokens for one call");
  *grid = (int)blocks;
  return CC2_OK;
}

}  // namespace
}  // namespace kv4

int read_kv4_error(int clear, int* value) {
  CC2_CUDA(cudaMemcpyFromSymbol(value, kv4::g_kv4_error, sizeof(int)));
  if (clear) {
    int z = 0;
    CC2_CUDA(cudaMemcpyToSymbol(kv4::g_kv4_error, &z, sizeof(int)));
  }
  return CC2_OK;
}

int launch_kv4_append(const cc2_kv4_cache* cache, int dtype, const void* k, int64_t k_ld, int64_t k_hs, const void* v,
                      int64_t v_ld, int64_t v_hs, int T, const int32_t* seq, const int32_t* pos, const uint8_t* mask,
                      const int32_t* table, int table_ld, int num_seqs, cudaStream_t st) {
  using namespace kv4;
  Pool pool;
  CC2_TRY(check_cache(cache, "kv4_append", pool));
  CC2_REQUIRE(dtype == CC2_BF16 || dtype == CC2_F32, "kv4_append: unsupported dtype %d", dtype);
  if (T == 0) return CC2_OK;
  CC2_TRY(check_places("kv4_append", T, seq, pos, table, table_ld, num_seqs));
  CC2_REQUIRE(k && v, "kv4_append: null keys or values");
  CC2_REQUIRE(rows_ok(dtype, k, k_ld, k_hs) && rows_ok(dtype, v, v_ld, v_hs),
              "kv4_append: keys and values must start on 16 bytes, as must their strides");
  int grid = 0, *err = nullptr;
  CC2_TRY(grid_of(T, pool.heads, &grid));
  CC2_TRY(error_word(&err));
  const Quant qk = make_quant(cache->key), qv = make_quant(cache->value);
  const Places at{seq, pos, table, table_ld, num_seqs};
  const float2* rope = (const float2*)cache->rope_cs;
  if (dtype == CC2_BF16) {
    CC2_CUDA(launch_k(append_kernel<__nv_bfloat16>, grid, kThreads, 0, st, pool, qk, qv, (const __nv_bfloat16*)k,
                      (long long)k_ld, (long long)k_hs, (const __nv_bfloat16*)v, (long long)v_ld, (long long)v_hs, T, at,
                      mask, rope, cache->rope_len, err));
  } else {
    CC2_CUDA(launch_k(append_kernel<float>, grid, kThreads, 0, st, pool, qk, qv, (const float*)k, (long long)k_ld,
                      (long long)k_hs, (const float*)v, (long long)v_ld, (long long)v_hs, T, at, mask, rope,
                      cache->rope_len, err));
  }
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

int launch_kv4_read(const cc2_kv4_cache* cache, int dtype, void* k_out, void* v_out, int T, const int32_t* seq,
                    const int32_t* pos, const int32_t* table, int table_ld, int num_seqs, cudaStream_t st) {
  using namespace kv4;
  Pool pool;
  CC2_TRY(check_cache(cache, "kv4_read", pool));
  CC2_REQUIRE(dtype == CC2_BF16 || dtype == CC2_F32, "kv4_read: unsupported dtype %d", dtype);
  if (T == 0 || (!k_out && !v_out)) return CC2_OK;
  CC2_TRY(check_places("kv4_read", T, seq, pos, table, table_ld, num_seqs));
  CC2_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15u) == 0, "kv4_read: outputs must be 16-byte aligned");
  int grid = 0, *err = nullptr;
  CC2_TRY(grid_of(T, pool.heads, &grid));
  CC2_TRY(error_word(&err));
  const Quant qk = make_quant(cache->key), qv = make_quant(cache->value);
  const Places at{seq, pos, table, table_ld, num_seqs};
  if (dtype == CC2_BF16) {
    CC2_CUDA(launch_k(read_kernel<__nv_bfloat16>, grid, kThreads, 0, st, pool, qk, qv, (__nv_bfloat16*)k_out,
                      (__nv_bfloat16*)v_out, T, at, err));
  } else {
    CC2_CUDA(launch_k(read_kernel<float>, grid, kThreads, 0, st, pool, qk, qv, (float*)k_out, (float*)v_out, T, at, err));
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
