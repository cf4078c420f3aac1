// Attention over the 4-bit cache for many rows (prompt chunks, an encoder's
// whole series) on tcgen05, bf16 calls.  Mathematics and arguments as in
// attn_kv4.cu; here the codes of 128 keys are decoded once to shared memory and
// serve 256 rows.
//
// A first kernel rotates the queries into the codes' frame and leaves them in
// the workspace as fp16 tiles in the tensor core's shared-memory order, each
// row scaled to below 2^8.  Then persistent blocks, one an SM, walk items
// (sequence, head, 256 rows, chunk of keys):
//   warp 0        loader: finds the items, brings raw key blocks by bulk copies
//   warp 3        the same for the items' query tiles
//   warps 20-23   decoders, a key a thread: K^ and V^ tiles as fp16, norms
//                 multiplied in after scaling them by a power of two a block
//   warps 1, 2    MMA issuers of the two tiles of 128 rows
//   warps 4-19    softmax, a row a thread: four chains, each a tile and every
//                 other step of 64 keys
//   warps 24-31   output, four a tile: join its two chains, turn the sums out of
//                 the codes' frame (butterflies in shared memory), write rows
// A chain is S_j = Q K_j^T -> running maximum (moved only past 2^8), P_j =
// 2^(S_j - m) as fp16 over S_j's place in TMEM -> O += P_j V_j -> S_{j+2}, with a
// maximum, sum and O of its own.  One warp alone leaves its scheduler idle most
// of the time (each of the steps waits for the one before it); four warps a
// scheduler, none of which waits for another, fill it.
// Exponents: K^ of a block is scaled by 2^(8 - eK) with eK from its largest norm
// (norms below 2^8, products with the levels below 2^15), which goes into the
// scores' factor; V^ by 2^(8 - eV), which goes into P's exponent.  A row's
// running maximum is that of score + eV of the score's block, so what P and V^
// have as fp16 is measured against the largest P V of the blocks so far and not
// against the largest V: P = 2^(x + eV - m + 7), up to 2^15.  Neither costs an
// operation a score.  fp16 keeps its 11 bits down to 2^-22 of a block's largest
// norm and of a row's largest P 2^eV.
// A masked key's column is -inf and its V^ zero.  A K that is not finite makes
// its column of scores NaN, which is hidden like others.  A V that is not finite
// is zero, so that it cannot reach through 0 * NaN the rows that do not see it;
// those that do are marked, by the sign of their sum of weights, for the output.
// Every wait is bounded (about 2 s): on expiry all roles leave their loops,
// copies and MMAs in flight are waited for, TMEM is freed, the kernel returns.
// Measured: 2048, 1450 and 853 tokens against 16384, 11603 and 6822 keys, 4
// heads on each of 8, causal, 724 us, 596 TFLOP/s of the scores' and values'
// products; 256 series of 133 tokens, 12 heads, 168 us (40 of them the first
// kernel).  What bounds it: issue slots are 65% used, the exponentials' unit 60%,
// and a step's chain of waits does not fill the rest; a third of the instructions
// are the decoders', two thirds the softmax'.  Computing part of the exponentials
// as polynomials made it slower (812 -> 833 us and more at an earlier state), two
// chains in place of four too (1196 against 979).  The roles' code has to stay
// small: they run at the same time, and instructions that miss their cache were
// what bound the series (245 us with 77 KB of code and rolled-out masks, 178 with
// 64 KB).  A second buffer for Q in place of the third stage of K and V: series
// 165 us, prompt chunks 779.
#include "kv4_attn.cuh"

namespace cc2 {
namespace kv4 {
namespace {

using namespace tcx;

constexpr int kThreads = 1024;
constexpr int kSoftmaxWarp = 4, kDecodeWarp = 20, kOutWarp = 24;
constexpr int kTile = 128;                      // rows of a pipeline, keys of a block
constexpr uint32_t kTileBytes = 128 * 128;      // 128 rows of 64 fp16
constexpr uint32_t kRawBytes = 8 * kBlockBytes;
constexpr int kKvStages = 3, kRawStages = 2, kItems = 4;
constexpr int kSumPitch = 68 * 4;  // bytes of a row's staged sums
constexpr uint32_t kQAt = 0, kKvAt = 2 * kTileBytes, kRawAt = kKvAt + kKvStages * 2 * kTileBytes,
                   kSumAt = kRawAt + kRawStages * kRawBytes,
                   kSmem = kSumAt + 256 * kSumPitch;
constexpr uint32_t kTmemCols = 512;
constexpr int kStep = 64;                       // keys of a step of the softmax
// TMEM columns of tile g, chain c: S (and P over it) at 128 g + 64 c, O at 256 + 128 g + 64 c
constexpr uint32_t kSCol = 0, kOCol = 256;
constexpr float kRescaleLog2 = 8.0f, kLiftLog2 = 7.0f;  // P up to 2^(8 + 7)

__device__ __forceinline__ uint32_t idesc_f16(int M, int N, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? (1u << 16) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What a pipeline needs of an item.
struct Item {
  int seq;       // -1: no more items
  int head, row0, rows, q_start, n, len, split, chunks;
  int c0, c1;    // keys of the chunk that some row of the item sees
  int blocks[2], key_end[2];
  int lane0[2];  // TMEM lane of a tile's first row
  long long q_tile;
};

struct Note {  // on half a block of keys: bit k of the words is key k
  uint32_t seen[2];    // the key counts
  uint32_t poison[2];  // its V is not finite
};

struct Control {
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t raw_full[kRawStages], raw_empty[kRawStages];
  uint64_t kv_full[kKvStages], kv_empty[kKvStages];
  uint64_t q_full[2], q_empty[2], o_full[2], o_free[2], mma_done[2];
  uint64_t s_full[2][2], p_full[2][2];  // [tile][chain]
  Item items[kItems];
  alignas(16) Note notes[kKvStages][2];
  alignas(16) float4 exps[kKvStages];   // 2^(eK - 134), eV - 126, 2^(119 - eV)
  float m[2][2][2][128], l[2][2][2][128];  // [turn][tile][chain][row]
  uint32_t top[2][4];
  uint32_t tmem;
  int abort_flag;
};

// Rounds of a ring of n stages.
template <int N>
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) i = 0, phase ^= 1u;
  }
};

// A warp's bounded wait: its lanes go on together or leave together.  The try
// suspends the warp for up to `kSuspendNs`, so that a role that waits does not
// take issue slots from the softmax and decoder warps of its scheduler.
constexpr uint32_t kSuspendNs = 4000;
__device__ __forceinline__ bool try_suspended(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(kSuspendNs)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int* flag, int* err) {
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
    if (__all_sync(0xffffffffu, try_suspended(bar, parity))) return true;
    const bool late = globaltimer_ns() - t0 > kWaitLimitNs;
    if (late && *flag == 0) {
      *flag = 1;
      atomicOr(err, 1);
    }
    if (__any_sync(0xffffffffu, late || *flag)) return false;
  }
}
__device__ __forceinline__ bool wait(uint64_t& bar_, uint32_t parity, Control& c, int* err) {
  const uint32_t bar = smem_u32(&bar_);
  return __all_sync(0xffffffffu, try_suspended(bar, parity)) || wait_long(bar, parity, &c.abort_flag, err);
}

// Of 32 keys that count, those below the row's limit.
__device__ __forceinline__ uint32_t visible(uint32_t seen, int limit) {
  return limit >= 32 ? seen : limit <= 0 ? 0u : seen & ((1u << limit) - 1u);
}
// Scores of keys that the row does not see.
__device__ __forceinline__ void hide(uint32_t (&v)[16], uint32_t vis) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!((vis >> i) & 1u)) v[i] = 0xff800000u;
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// ------------------------------------------------------------------ queries --
// A block rotates 128 rows of the call for some heads, whatever sequences the
// rows belong to.  The rotation is a product with a 64 x 64 matrix of +-1, which
// mma.sync takes from a row's elements as they come from memory: a lane has four
// neighbours of each 16, RoPE turns them in registers (its pairs, 32 apart, are
// one lane's), and the matrix' rows are in the order that this gives.  In bf16,
// as the elements and the next 8 bits of what RoPE leaves of them (2^-17 of an
// element where the fp16 result keeps 2^-11); sums in fp32.  Finished rows leave
// through shared memory as whole 128-byte lines.
constexpr int kQThreads = 128;

// The last sequence that starts at or before the token; -1: none does.
__device__ __forceinline__ int find_seq(const Args& a, int tok, int lane) {
  if (a.cu == nullptr) return tok / a.max_q;
  int seq = -1;
  for (int i = lane; i - lane < a.num_seqs; i += 32)
    seq += __popc(__ballot_sync(0xffffffffu, i < a.num_seqs && a.cu[i] <= tok));
  return seq;
}

__device__ __forceinline__ void mma_pm1(float (&d)[4], const uint32_t (&x)[4], uint2 b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b.x), "r"(b.y));
}

// A row of no sequence, of some heads.  Not inlined: the kernel's registers are full, and such rows are few.
__device__ __noinline__ void fill_row(const Args& a, int row, int head0, int head1) {
  const int heads = a.pool.heads * a.group, tok = row / a.group;
  for (int head = head0; head < head1; ++head) {
    const int qh = head * a.group + row % a.group;
    uint4* const out = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (long long)tok * a.o_ld + (long long)qh * a.o_hs);
    if (a.fill & 1)
      for (int i = 0; i < 8; ++i) out[i] = make_uint4(0, 0, 0, 0);
    if (a.fill & 2) a.lse[(long long)tok * heads + qh] = -INFINITY;
  }
}

__global__ void __launch_bounds__(kQThreads, 4)
rotate_queries_kernel(const __grid_constant__ Args a, const long long q_tiles, const int per) {
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.counter = 0;  // for the kernel after this one
  __shared__ __align__(16) uint8_t stage[128 * 128];
  __shared__ uint2 matrix[4 * 8 * 32];  // [16 elements][8 coordinates][lane]
  __shared__ const __nv_bfloat16* row_at[128];
  __shared__ long long row_to[128];  // row among the tiles of head 0; -1: none
  __shared__ int row_pos[128];
  __shared__ uint8_t coord[64];  // of an element, its sign in bit 7
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = blockIdx.x * 128, all = a.total_q * a.group;
  if (tid < 64) {
    const uint32_t i = a.rk.inv[tid];
    coord[tid] = (uint8_t)(i | ((a.rk.signs[i >> 5] >> (i & 31)) & 1u) << 7);
  }
  {
    // this thread's row: a block's rows mostly belong to one sequence, the others follow it
    const int near = find_seq(a, base / a.group, lane);
    const int row = base + tid;
    const __nv_bfloat16* from = nullptr;
    int pos = -1;
    long long to = -1;
    if (row < all) {
      const int tok = row / a.group;
      int seq = near;
      if (a.cu == nullptr) seq = tok / a.max_q;
      else
        while (seq + 1 < a.num_seqs && a.cu[seq + 1] <= tok) ++seq;
      if (seq >= 0) {
        const Span s = span_of(a, seq, 0, false);
        const int in_seq = row - s.q_start * a.group;
        if (in_seq >= 0 && in_seq < s.rows) {  // a cu_q that falls may find a sequence that starts after the token
          from = (const __nv_bfloat16*)a.q + (long long)tok * a.q_ld + (long long)(row % a.group) * a.q_hs;
          to = first_query_tile(a, seq, s.q_start) * 128 + in_seq;
          if (a.rotate) pos = s.len - s.n + (tok - s.q_start);
          if (pos >= a.rope_len) {
            if (a.rotate) atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
            pos = -1;
          }
        }
      }
    }
    if (a.fill && row < all && from == nullptr) fill_row(a, row, blockIdx.y * per, min((int)(blockIdx.y + 1) * per, a.pool.heads));
    row_at[tid] = from;
    row_to[tid] = to;
    row_pos[tid] = pos;
  }
  __syncthreads();
#pragma unroll 2
  for (int k = tid; k < 4 * 8 * 32; k += kQThreads) {
    const int n = 8 * ((k >> 5) & 7) + ((k & 31) >> 2), t = k >> 8, col = 32 * (t >> 1) + 8 * (k & 3) + 4 * (t & 1);
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t i = coord[col + j];
      v[j] = 0x3f80u | ((__popc(n & i & 63u) ^ (i >> 7)) & 1u) << 15;  // +-1
    }
    matrix[k] = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
  }
  __syncthreads();
  const int c = lane & 3;
  const float by = a.qscale;
  const int head0 = blockIdx.y * per, head1 = min(head0 + per, a.pool.heads);
#pragma unroll 1
  for (int mt = 0; mt < 2; ++mt) {
    const int first = 32 * warp + 16 * mt + (lane >> 2);  // the lane's rows: this one and the eighth after it
    float4 cs[2][4];  // [half][elements 8c + 2j, 8c + 2j + 1]: cosine, sine; of all heads
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int p = row_pos[first + 8 * half];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        cs[half][j] = p >= 0 ? *reinterpret_cast<const float4*>(a.rope + (long long)p * 32 + 8 * c + 2 * j)
                             : make_float4(1.0f, 0.0f, 1.0f, 0.0f);
    }
    uint4 next[2][2];  // the next head's elements
    auto fetch = [&](int head) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const __nv_bfloat16* q = row_at[first + 8 * half];
        next[half][0] = next[half][1] = make_uint4(0, 0, 0, 0);
        if (q != nullptr && head < head1) {
          q += (long long)(head * a.group) * a.q_hs + 8 * c;
          next[half][0] = *reinterpret_cast<const uint4*>(q);
          next[half][1] = *reinterpret_cast<const uint4*>(q + 32);
        }
      }
    };
    fetch(head0);
#pragma unroll 1
    for (int head = head0; head < head1; ++head) {
      uint32_t hi[4][4], lo[4][4];  // [elements][row + 8 * half, elements 0, 1 / 2, 3]
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint4 u = next[half][0], v = next[half][1];
        hi[0][half] = u.x, hi[0][half + 2] = u.y, hi[1][half] = u.z, hi[1][half + 2] = u.w;
        hi[2][half] = v.x, hi[2][half + 2] = v.y, hi[3][half] = v.z, hi[3][half + 2] = v.w;
        if (a.rotate) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = j >> 1, i = half + 2 * (j & 1);
            const float4 f = cs[half][j];
            const uint32_t pw = hi[t][i], qw = hi[t + 2][i];
            const float p0 = __uint_as_float(pw << 16), p1 = __uint_as_float(pw & 0xffff0000u);
            const float q0 = __uint_as_float(qw << 16), q1 = __uint_as_float(qw & 0xffff0000u);
            const float x0 = p0 * f.x - q0 * f.y, y0 = q0 * f.x + p0 * f.y;
            const float x1 = p1 * f.z - q1 * f.w, y1 = q1 * f.z + p1 * f.w;
            const uint32_t x = pack_bf16(x0, x1), y = pack_bf16(y0, y1);
            hi[t][i] = x;
            hi[t + 2][i] = y;
            lo[t][i] = pack_bf16(x0 - __uint_as_float(x << 16), x1 - __uint_as_float(x & 0xffff0000u));
            lo[t + 2][i] = pack_bf16(y0 - __uint_as_float(y << 16), y1 - __uint_as_float(y & 0xffff0000u));
          }
        }
      }
      fetch(head + 1);
      float y[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.0f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const uint2 b = matrix[(8 * t + n) * 32 + lane];
          if (a.rotate) mma_pm1(y[n], lo[t], b);
          mma_pm1(y[n], hi[t], b);
        }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float top = 0.0f;
#pragma unroll
        for (int n = 0; n < 8; ++n) top = max3(top, fabsf(y[n][2 * half]), fabsf(y[n][2 * half + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(__float_as_uint(top * fabsf(by)) >> 23), 30), 254);
        const float up = by * __int_as_float((261 - e) << 23);  // 2^(134 - e): the row below 2^8
        const long long to = row_to[first + 8 * half];
        // the 16-byte pieces exchanged within 8 rows of a tile as the tensor core reads them
        uint8_t* out = stage + (first + 8 * half) * 128 + 4 * c;
        const int r7 = (int)to & 7;
#pragma unroll
        for (int n = 0; n < 8; ++n)
          *reinterpret_cast<uint32_t*>(out + ((n ^ r7) << 4)) = pack_half(y[n][2 * half] * up, y[n][2 * half + 1] * up);
        if (to >= 0 && c == 0)  // 2^(e - 134) / 64
          const_cast<float*>(a.q_scale)[head * q_tiles * 128 + to] = __int_as_float((e - 13) << 23);
      }
      __syncwarp();
      uint8_t* const tiles = const_cast<uint8_t*>(a.qt) + head * q_tiles * kTileBytes + 16 * (lane & 7);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 32 * warp + 16 * mt + 4 * i + (lane >> 3);
        const long long to = row_to[k];
        if (to >= 0) *reinterpret_cast<uint4*>(tiles + to * 128) = *reinterpret_cast<const uint4*>(stage + k * 128 + 16 * (lane & 7));
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------- attention --
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const __grid_constant__ Args a, const long long q_tiles, const int total_items) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ Control ctl;
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  const uint32_t smem = smem_u32(smem_raw) + pad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* const err = a.wait_err;
  pdl_launch_dependents();

  if (tid == 0) {
    for (int i = 0; i < kItems; ++i) mbar_init(smem_u32(&ctl.item_full[i]), 1), mbar_init(smem_u32(&ctl.item_empty[i]), 31);
    for (int i = 0; i < kRawStages; ++i) mbar_init(smem_u32(&ctl.raw_full[i]), 1), mbar_init(smem_u32(&ctl.raw_empty[i]), 4);
    for (int i = 0; i < kKvStages; ++i) mbar_init(smem_u32(&ctl.kv_full[i]), 4), mbar_init(smem_u32(&ctl.kv_empty[i]), 2 + 16);
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&ctl.q_full[g]), 1);
      mbar_init(smem_u32(&ctl.q_empty[g]), 1);
      mbar_init(smem_u32(&ctl.o_full[g]), 2);
      mbar_init(smem_u32(&ctl.o_free[g]), 4);
      mbar_init(smem_u32(&ctl.mma_done[g]), 1);
      for (int c = 0; c < 2; ++c) {
        mbar_init(smem_u32(&ctl.s_full[g][c]), 1);
        mbar_init(smem_u32(&ctl.p_full[g][c]), 4);
      }
    }
    ctl.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = ctl.tmem;

  if (warp < kSoftmaxWarp) {
    if (warp == 0) {
      // ---------------- loader ----------------
      Ring<kItems> it;
      Ring<kRawStages> raw;
      long long n_items = 0, n_raw = 0;
      const int mask = (1 << a.pool.page_shift) - 1;
      const int run = min((mask + 1) / kBlockTokens, 8);  // blocks of 16 keys a copy brings
      bool ok = true;
      // Items are taken as blocks get to them (their costs differ by the rows' and
      // sequences' lengths): a few at a time where there are many, since many of
      // them may turn out to have no rows or no keys.
      const int batch = min(max(total_items / (8 * (int)gridDim.x), 1), 32);
      while (ok) {
        int base = 0;
        if (lane == 0) base = atomicAdd(a.counter, batch);
        base = __shfl_sync(0xffffffffu, base, 0);
        const bool any_left = base < total_items;
        const int mine = lane < batch ? base + lane : total_items;  // each lane looks at one item
        Item d;
        d.seq = -1;
        if (mine < total_items) {
          unsigned idx = (unsigned)mine;
          const int tile = a.row_tiles - 1 - (int)(idx % a.row_tiles);  // causal rows with the most keys first
          idx /= a.row_tiles;
          d.split = (int)(idx % a.splits);
          idx /= a.splits;
          d.head = (int)(idx % a.pool.heads);
          const int seq = (int)(idx / a.pool.heads);
          const Span s = span_of(a, seq, tile, d.split == 0 && d.head == 0 && tile == 0);
          d.chunks = chunks_of(a, s);
          if (s.row0 < s.rows && d.split < max(d.chunks, 1)) {
            d.seq = seq;
            d.row0 = s.row0;
            d.rows = s.rows;
            d.q_start = s.q_start;
            d.n = s.n;
            d.len = s.len;
            d.c0 = d.split * a.chunk;
            d.c1 = min(s.keys, d.c0 + a.chunk);
            for (int g = 0; g < 2; ++g) {
              const int first = s.row0 + kTile * g, last = min(first + kTile, s.rows) - 1;
              int end = first < s.rows ? (a.causal ? min(s.len - s.n + last / a.group + 1, s.len) : s.len) : 0;
              end = min(end, d.c1);
              d.key_end[g] = end;
              d.blocks[g] = end > d.c0 ? (end - d.c0 + kTile - 1) / kTile : 0;
            }
            d.q_tile = (long long)d.head * q_tiles + first_query_tile(a, seq, s.q_start) + s.row0 / kTile;
          }
        }
        unsigned live = __ballot_sync(0xffffffffu, d.seq >= 0);
        while (ok && (live != 0 || !any_left)) {
          const int src = live != 0 ? __ffs(live) - 1 : 0;
          live &= live - 1;
          if (n_items >= kItems && !wait(ctl.item_empty[it.i], it.phase ^ 1u, ctl, err)) {
            ok = false;
            break;
          }
          if (lane == src) {
            // A scheduler has one quarter of the lanes of both tiles: a tile that leaves quarters unused starts in
            // another one each time, so that short tiles do not all fall to the first.
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int used = (min(d.rows - d.row0 - kTile * g, kTile) + 31) / 32, n = (int)n_items;
              d.lane0[g] = used > 3 ? 0 : used == 3 ? 32 * (n & 1) : used == 2 ? 64 * (n & 1) : 32 * (n & 3);
            }
            ctl.items[it.i] = d;
            if (!any_left) ctl.items[it.i].seq = -1;
          }
          __syncwarp();
          const Item& e = ctl.items[it.i];
          const int seq = e.seq, c0 = e.c0, c1 = e.c1, head = e.head, nb = max(e.blocks[0], e.blocks[1]);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctl.item_full[it.i]));
          it.next();
          ++n_items;
          if (seq < 0) {
            ok = false;
            break;
          }
          const int* table = a.table + (long long)seq * a.table_ld;
          const int first = lane * run;  // this lane's first block of 16 keys
          int page = -1;
          if (nb > 0 && lane < 8 && c0 + first * kBlockTokens < c1 && first < 8)
            page = table[(c0 + first * kBlockTokens) >> a.pool.page_shift];
          for (int j = 0; j < nb && ok; ++j) {
            const int key0 = c0 + j * kTile;
            const int n = min((c1 - key0 + kBlockTokens - 1) / kBlockTokens, 8);
            if (n_raw >= kRawStages && !wait(ctl.raw_empty[raw.i], raw.phase ^ 1u, ctl, err)) {
              ok = false;
              break;
            }
            const uint32_t bar = smem_u32(&ctl.raw_full[raw.i]);
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)n * kBlockBytes);
            __syncwarp();
            if (lane < 8 && first < n) {
              if ((unsigned)page >= (unsigned)a.pool.num_pages) {
                atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
                page = 0;
              }
              bulk_load(smem + kRawAt + raw.i * kRawBytes + first * kBlockBytes,
                        a.pool.pages + block_offset(a.pool, page, head, (key0 + first * kBlockTokens) & mask),
                        (uint32_t)min(run, n - first) * kBlockBytes, bar);
            }
            const int next = key0 + kTile + first * kBlockTokens;  // the next block's page, ahead of its copy
            if (j + 1 < nb && lane < 8 && first < 8 && next < c1) page = table[next >> a.pool.page_shift];
            raw.next();
            ++n_raw;
          }
        }
        if (!any_left) break;
      }
      // no copy may still be landing in shared memory when the block exits
      if (lane == 0) {
        const unsigned long long t0 = globaltimer_ns();
        for (int k = 0; k < kRawStages && k < n_raw; ++k) {
          const long long at = n_raw - 1 - k;
          while (!mbar_try(smem_u32(&ctl.raw_full[at % kRawStages]), (uint32_t)(at / kRawStages) & 1u) &&
                 globaltimer_ns() - t0 < kWaitLimitNs) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 3) {
      // ---------------- query loader ----------------
      Ring<kItems> it;
      uint32_t nq[2] = {0, 0};
      bool ok = true;
      while (ok) {
        if (!wait(ctl.item_full[it.i], it.phase, ctl, err)) break;
        const Item& e = ctl.items[it.i];
        const int seq = e.seq, rows = e.rows - e.row0, blocks[2] = {e.blocks[0], e.blocks[1]},
                  lane0[2] = {e.lane0[0], e.lane0[1]};
        const long long q_tile = e.q_tile;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
        it.next();
        if (seq < 0) break;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (blocks[g] == 0 || !ok) continue;
          if (nq[g] > 0) ok = wait(ctl.q_empty[g], (nq[g] - 1) & 1u, ctl, err);
          if (!ok) break;
          if (lane == 0) {  // the tile's rows, in groups of 8
            const uint32_t bytes = (uint32_t)min((rows - kTile * g + 7) / 8, kTile / 8) * 1024u;
            mbar_arrive_expect_tx(smem_u32(&ctl.q_full[g]), bytes);
            bulk_load(smem + kQAt + g * kTileBytes + lane0[g] * 128, a.qt + (q_tile + g) * kTileBytes, bytes, smem_u32(&ctl.q_full[g]));
          }
          __syncwarp();
          ++nq[g];
        }
      }
      if (lane == 0) {  // as above
        const unsigned long long t0 = globaltimer_ns();
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (nq[g] > 0)
            while (!mbar_try(smem_u32(&ctl.q_full[g]), (nq[g] - 1) & 1u) && globaltimer_ns() - t0 < kWaitLimitNs) {
            }
      }
      __syncwarp();
    } else if (warp < 3) {
      // ---------------- MMA issuer of tile g ----------------
      // The warp stays converged and what it branches on is broadcast, so that
      // descriptors stay in uniform registers; one elected lane issues.  The tensor
      // core runs its products in order: S_{j+2} may follow P_j V_j, whose P it
      // overwrites, at once, and its completion says that P_j V_j is done too.
      const int g = warp - 1;
      Ring<kItems> it;
      Ring<kKvStages> kv_s, kv_p;  // stage of the next S, of the next P V
      uint32_t nt = 0, np0 = 0, np1 = 0;  // items with keys, steps of the two chains
      const uint32_t t_s = tmem + kSCol + 128u * g, t_o = tmem + kOCol + 128u * g;
      const uint64_t dq = sw128_desc(smem + kQAt + g * kTileBytes), dk0 = sw128_desc(smem + kKvAt),
                     dv0 = sw128_desc(smem + kKvAt + kTileBytes);
      const uint32_t id_o = idesc_f16(128, 64, true);
      constexpr uint64_t kStage = 2 * kTileBytes >> 4, kHalf = kTileBytes / 2 >> 4;  // descriptor steps
      bool ok = true;
      while (ok) {
        if (!wait(ctl.item_full[it.i], it.phase, ctl, err)) break;
        const Item& e = ctl.items[it.i];
        const int seq = __shfl_sync(0xffffffffu, e.seq, 0), blocks = __shfl_sync(0xffffffffu, e.blocks[g], 0),
                  keys = __shfl_sync(0xffffffffu, e.key_end[g] - e.c0, 0),
                  all = __shfl_sync(0xffffffffu, max(e.blocks[0], e.blocks[1]), 0);
        if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
        __syncwarp();
        it.next();
        if (seq < 0) break;
        const int steps = blocks > 0 ? (keys + kStep - 1) / kStep : 0;
        if (steps > 0) ok = wait(ctl.q_full[g], nt & 1u, ctl, err);
        for (int j = -2; j < steps && ok; ++j) {  // P_j V_j, then S_{j+2}
          if (j >= 0) {
            const int n = min((keys - j * kStep + 15) >> 4, kStep / 16);
            const uint32_t c = j & 1, parity = (c ? np1++ : np0++) & 1u;
            const uint64_t dv = dv0 + kv_p.i * kStage + c * kHalf;
            const bool last = j == steps - 1, done = c == 1 || last;
            // the first product of an item waits until the item before has been read out
            ok = (j > 0 || nt == 0 || wait(ctl.o_free[g], (nt - 1) & 1u, ctl, err)) &&
                 wait(ctl.p_full[g][c], parity, ctl, err);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t tp = t_s + 64u * c, to = t_o + 64u * c, acc = j > 1 ? 1u : 0u;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < n) mma_bf16_ts(to, tp + 8u * k, dv + 128u * k, id_o, k > 0 ? 1u : acc);
              if (done) mma_commit(smem_u32(&ctl.kv_empty[kv_p.i]));
              if (last) {
                mma_commit(smem_u32(&ctl.o_full[g]));
                mbar_arrive(smem_u32(&ctl.o_full[g]));  // hands on the maxima and sums that came with P
              }
            }
            __syncwarp();
            if (done) kv_p.next();
          }
          const int i = j + 2;
          if (i < steps) {
            const uint32_t id = idesc_f16(128, min((keys - i * kStep + 15) & ~15, kStep), false), c = i & 1;
            if (c == 0) ok = wait(ctl.kv_full[kv_s.i], kv_s.phase, ctl, err);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dk = dk0 + kv_s.i * kStage + c * kHalf;
            const bool last = i == steps - 1;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_bf16(t_s + 64u * c, dq + 2u * k, dk + 2u * k, id, k > 0);
              mma_commit(smem_u32(&ctl.s_full[g][c]));
              if (last) mma_commit(smem_u32(&ctl.q_empty[g]));
            }
            __syncwarp();
            if (c == 1 || last) kv_s.next();
          }
        }
        if (steps > 0) ++nt;
        for (int j = blocks; j < all && ok; ++j) {  // blocks that only the other tile's rows see
          ok = wait(ctl.kv_full[kv_p.i], kv_p.phase, ctl, err);
          if (ok && lane == 0) mbar_arrive(smem_u32(&ctl.kv_empty[kv_p.i]));
          __syncwarp();
          kv_p.next();
          kv_s.next();
        }
      }
      if (nt > 0 && elect_one()) {  // every MMA has completed before TMEM is released
        mma_commit(smem_u32(&ctl.mma_done[g]));
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try(smem_u32(&ctl.mma_done[g]), 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
        }
      }
      __syncwarp();
    }
  } else if (warp >= kDecodeWarp && warp < kOutWarp) {
    // ---------------- decoders ----------------
    Ring<kItems> it;
    Ring<kRawStages> raw;
    Ring<kKvStages> kv;
    long long n_kv = 0;
    const int k = tid - kDecodeWarp * 32, w = warp - kDecodeWarp;  // key of the block, warp
    uint32_t flip = 0;
    bool ok = true;
    while (ok) {
      // the four warps meet at named barriers: they leave together
      if (!barrier_and(1, 128, wait(ctl.item_full[it.i], it.phase, ctl, err))) break;
      const Item& e = ctl.items[it.i];
      const int seq = e.seq, c0 = e.c0, c1 = e.c1, nb = max(e.blocks[0], e.blocks[1]);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
      it.next();
      if (seq < 0) break;
      for (int j = 0; j < nb; ++j) {
        ok = wait(ctl.raw_full[raw.i], raw.phase, ctl, err);
        if (ok && n_kv >= kKvStages) ok = wait(ctl.kv_empty[kv.i], kv.phase ^ 1u, ctl, err);
        const uint32_t src = smem + kRawAt + raw.i * kRawBytes + (k >> 4) * kBlockBytes;
        uint32_t nbits = 0;
        if (ok) {
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(nbits) : "r"(src + kNorms + (k & 15) * 4));
        }
        const bool seen = !(nbits & 0x8000u) && c0 + j * kTile + k < c1;
        const float nk = seen ? norm_value((uint16_t)nbits, a.pool.norm_bf16) : 0.0f;
        float nv = seen ? norm_value((uint16_t)(nbits >> 16), a.pool.norm_bf16) : 0.0f;
        const bool bad = !(nv <= 3.402823466e38f);
        if (bad) nv = 0.0f;
        const uint32_t sb = __ballot_sync(0xffffffffu, seen), pb = __ballot_sync(0xffffffffu, bad);
        const uint32_t tk = __reduce_max_sync(0xffffffffu, nk <= 3.402823466e38f ? __float_as_uint(nk) : 0u) >> 23;
        const uint32_t tv = __reduce_max_sync(0xffffffffu, __float_as_uint(nv)) >> 23;
        if (lane == 0) ctl.top[flip][w] = tk | tv << 16;
        ok = barrier_and(1, 128, ok);
        if (!ok) break;
        uint32_t ek = 20, ev = 40;  // 2^-86: a row's sum, in units of 2^-eV, stays far inside fp32
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t t = ctl.top[flip][i];
          ek = max(ek, t & 0xffffu);
          ev = max(ev, t >> 16);
        }
        flip ^= 1u;
        if (lane == 0) {
          ctl.notes[kv.i][w >> 1].seen[w & 1] = sb;
          ctl.notes[kv.i][w >> 1].poison[w & 1] = pb;
          if (w == 0)
            ctl.exps[kv.i] = make_float4(__int_as_float(((int)ek - 7) << 23), (float)((int)ev - 126),
                                         __int_as_float((246 - (int)ev) << 23), 0.0f);
        }
        // norms below 2^8: 2^(134 - e)
        const __half2 hk = __float2half2_rn(nk * __int_as_float((261 - (int)ek) << 23));
        const __half2 hv = __float2half2_rn(nv * __int_as_float((261 - (int)ev) << 23));
        const uint32_t dst = smem + kKvAt + kv.i * 2 * kTileBytes + k * 128;
        // warps past the last key's group of 16 have nothing that an MMA reads
        const bool used = 32 * w < c1 - (c0 + j * kTile);
#pragma unroll 1
        for (int m = 0; m < 2 && used; ++m) {
          const __half2 n = m ? hv : hk;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t c[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
                         : "r"(src + m * kVCodes + (k & 15) * 32 + h * 16));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t o[4];
              decode_pairs(c[i], a.levels.lo, a.levels.hi, o);
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&o[p]), n);
                o[p] = *reinterpret_cast<const uint32_t*>(&x);
              }
              sts128(dst + m * kTileBytes + (((4 * h + i) ^ (k & 7)) << 4), o[0], o[1], o[2], o[3]);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&ctl.raw_empty[raw.i]));
          mbar_arrive(smem_u32(&ctl.kv_full[kv.i]));
        }
        raw.next();
        kv.next();
        ++n_kv;
      }
    }
  } else if (warp < kDecodeWarp) {
    // ---------------- softmax: chain c of tile g ----------------
    const int g = (warp - kSoftmaxWarp) >> 3, c = ((warp - kSoftmaxWarp) >> 2) & 1, quarter = warp & 3,
              r = 32 * quarter + lane;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16);
    const uint32_t t_s = t_lane + kSCol + 128u * g + 64u * c, t_o = t_lane + kOCol + 128u * g;
    Ring<kItems> it;
    Ring<kKvStages> kv;
    uint32_t n = 0, nt = 0;  // steps of this chain, items with keys
    bool ok = true;
    while (ok) {
      if (!wait(ctl.item_full[it.i], it.phase, ctl, err)) break;
      const Item& in = ctl.items[it.i];
      const int seq = in.seq, c0 = in.c0, blocks = in.blocks[g], all = max(in.blocks[0], in.blocks[1]);
      const int lane0 = in.lane0[g], at = r - lane0, row = in.row0 + kTile * g + at;
      const bool warp_rows = 32 * quarter >= lane0 && row - lane < in.rows;
      const int limit = a.causal ? min(in.len - in.n + row / a.group + 1, in.len) : in.len;  // keys the row sees
      const int clear = a.causal ? in.len - in.n + (in.row0 + kTile * g) / a.group + 1 : in.len;
      const int keys = in.key_end[g] - c0, steps = blocks > 0 ? (keys + kStep - 1) / kStep : 0;
      const float* q_scale = a.q_scale + (in.q_tile + g) * 128 + at;
      const bool valid = at >= 0 && row < in.rows && blocks > 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
      it.next();
      if (seq < 0) break;
      const float rs = valid ? *q_scale : 0.0f;
      float m = -INFINITY, l = 0.0f;  // largest score + eV, sum of 2^(score - m)
      bool lost = false;              // the row sees a V that is not finite
      for (int t = 0; t < all; ++t) {
        // the decoders' notes on the block, then the scores
        if (!wait(ctl.kv_full[kv.i], kv.phase, ctl, err)) {
          ok = false;
          break;
        }
        const int j = 2 * t + c;
        const Note note = ctl.notes[kv.i][c];
        const float4 ex = ctl.exps[kv.i];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.kv_empty[kv.i]));
        kv.next();
        if (j >= steps) continue;
        const int key0 = c0 + j * kStep;
        // rs 2^(eK - 134).  Both are least where there is nothing to scale, a row of zeros over keys of zero norm or all
        // masked; their product would be 0 then and 0 * -inf, a hidden score, NaN.  At 2^-100 scores are 0 all the same.
        const float sc = fmaxf(rs * ex.x, 0x1p-100f);
        const bool clean = key0 + kStep <= clear && (note.seen[0] & note.seen[1]) == 0xffffffffu &&
                           (note.poison[0] | note.poison[1]) == 0;
        const int cols = min(keys - j * kStep, kStep);
        if (!wait(ctl.s_full[g][c], n & 1u, ctl, err)) {
          ok = false;
          break;
        }
        ++n;
        tc_fence_after();
        float scale = 1.0f;
        bool rescale = false;
        if (warp_rows) {
          // two passes over S, 32 scores in registers at a time: 64 would spill
          const bool two = cols > 32;
          if (!clean) {  // first the scores of keys that the row does not see, in place
            uint32_t vis[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              vis[h] = visible(note.seen[h], limit - key0 - 32 * h);
              lost = lost || (note.poison[h] & vis[h]) != 0;
            }
#pragma unroll 1
            for (int i = 0; i < (two ? 4 : 2); ++i) {
              uint32_t v[16];
              tmem_ld16(t_s + 16u * i, v);
              tmem_ld_wait();
              hide(v, (i < 2 ? vis[0] : vis[1]) >> (16 * (i & 1)));
              tmem_st16(t_s + 16u * i, v);
            }
            tmem_st_wait();
          }
          float b0 = -INFINITY, b1 = -INFINITY, b2 = -INFINITY, b3 = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !two) break;
            uint32_t v[32];
            tmem_ld32(t_s + 32u * h, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              b0 = max3(b0, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
              b1 = max3(b1, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
              b2 = max3(b2, __uint_as_float(v[i + 4]), __uint_as_float(v[i + 5]));
              b3 = max3(b3, __uint_as_float(v[i + 6]), __uint_as_float(v[i + 7]));
            }
          }
          const float bm = fmaf(fmaxf(max3(b0, b1, b2), b3), sc, ex.y);
          if (bm > m + kRescaleLog2 || (m == -INFINITY && bm > m)) {
            scale = m == -INFINITY ? 0.0f : ex2(m - bm);
            l *= scale;
            m = bm;
            rescale = true;
          }
          // P = 2^(x + eV - m + 7), of which the row's sum takes 2^(eV + 7) back out
          const float off = ex.y + kLiftLog2 - (m == -INFINITY ? 0.0f : m);
          const uint64_t sc2 = f2_pack(sc, sc), off2 = f2_pack(off, off);
          uint64_t la = f2_pack(0.0f, 0.0f), lb = la;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !two) break;
            uint32_t v[32];
            tmem_ld32(t_s + 32u * h, v);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const uint64_t x2 = f2_fma(f2_pack(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), sc2, off2);
              float x0, x1;
              f2_unpack(x2, x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              if (k & 1) lb = f2_add(lb, f2_pack(x0, x1)); else la = f2_add(la, f2_pack(x0, x1));
              v[k] = pack_half(x0, x1);
            }
            tmem_st16(t_s + 16u * h, v);  // over scores that both passes have read
          }
          float l0, l1;
          f2_unpack(f2_add(la, lb), l0, l1);
          l += (l0 + l1) * ex.z;
        }
        if (t > 0 && __any_sync(0xffffffffu, rescale)) {  // S_j's completion said that O stands still
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            uint32_t o[16];
            tmem_ld16(t_o + 64u * c + 16u * i, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * scale);
            tmem_st16(t_o + 64u * c + 16u * i, o);
          }
        }
        if (j + 2 >= steps) {  // the chain's last step: its maximum and sum, once the item before has been read out
          if (nt > 0 && !wait(ctl.o_free[g], (nt - 1) & 1u, ctl, err)) {
            ok = false;
            break;
          }
          const int turn = (int)(nt & 1u);
          ctl.m[turn][g][c][r] = m;
          ctl.l[turn][g][c][r] = lost ? -l : l;
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.p_full[g][c]));
      }
      if (!ok) break;

      if (steps > 0) ++nt;
    }
  } else {
    // ---------------- output ----------------
    const int g = (warp - kOutWarp) >> 2, quarter = warp & 3, r = 32 * quarter + lane;
    const uint32_t t_o = tmem + ((uint32_t)(32 * quarter) << 16) + kOCol + 128u * g;
    uint8_t* const stage = smem_raw + pad + kSumAt + (128 * g + 32 * quarter) * kSumPitch;  // this warp's
    Ring<kItems> it;
    uint32_t nt = 0;  // the tile's items with keys
    // the places in a staged row of this lane's eight coordinates of an output row, and their signs
    uint32_t from[4] = {0, 0, 0, 0}, flip[4] = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint32_t i = a.rv.inv[8 * (lane & 7) + t];
      from[t >> 1] |= (4u * (i & ~3u) + 2u * (i & 3u)) << (16 * (t & 1));
      flip[t >> 1] |= ((a.rv.signs[i >> 5] >> (i & 31)) & 1u) << (16 * (t & 1) + 15);
    }
    bool ok = true;
    while (ok) {
      if (!wait(ctl.item_full[it.i], it.phase, ctl, err)) break;
      const Item& in = ctl.items[it.i];
      struct {
        int seq, head, row0, rows, q_start, split, chunks, keys, lane0;
      } e = {in.seq,   in.head,   in.row0,                   in.rows,    in.q_start,
             in.split, in.chunks, in.key_end[g] - in.c0, in.lane0[g]};
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
      it.next();
      if (e.seq < 0) break;
      const int row = e.row0 + kTile * g + r - e.lane0;
      const bool warp_rows = 32 * quarter >= e.lane0 && row - lane < e.rows, valid = warp_rows && row < e.rows;
      const bool some = e.keys > 0, two = e.keys > kStep;
      const uint32_t turn = nt & 1u;
      float m = -INFINITY, l = 0.0f, fa = 0.0f, fb = 0.0f;
      if (some) {
        if (!wait(ctl.o_full[g], turn, ctl, err)) {
          ok = false;
          break;
        }
        ++nt;
        tc_fence_after();
        const float ma = ctl.m[turn][g][0][r], mb = two ? ctl.m[turn][g][1][r] : -INFINITY;
        m = fmaxf(ma, mb);
        const float wa = ma == -INFINITY ? 0.0f : ex2(ma - m), wb = mb == -INFINITY ? 0.0f : ex2(mb - m);
        const float la = ctl.l[turn][g][0][r], lb = two ? ctl.l[turn][g][1][r] : 0.0f;
        l = fabsf(la) * wa + fabsf(lb) * wb;
        // 2^-7, 2^-8 and 1 / 64 take the scales of P, V and the levels back out; a sum below 0 says that O is lost
        fa = la < 0.0f || lb < 0.0f ? __int_as_float(0x7fffffff) : wa * 0x1p-21f;
        fb = wb * 0x1p-21f;
      }
      const bool part = e.chunks > 1;
      if (!part) {
        const float inv = l == 0.0f ? 0.0f : __fdividef(a.back, l);
        fa *= inv;
        fb *= inv;
      }
      // 16 coordinates at a time: the chains joined, and butterflies of width 1..8
      float* sums = reinterpret_cast<float*>(stage + lane * kSumPitch);
      long long at = 0;
      if (part) {
        Span s;
        s.q_start = e.q_start;
        at = part_at(a, s, e.head, e.split, row);
      }
      float* const to = part ? a.part + at * 64 : sums;
      if (warp_rows) {
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t x[16], y[16];
          tmem_ld16(t_o + 16u * h, x);
          tmem_ld16(t_o + 64u + 16u * h, y);
          tmem_ld_wait();
          float o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)  // a chain without a step has no O
            o[i] = fmaf(__uint_as_float(two ? y[i] : 0u), fb, __uint_as_float(some ? x[i] : 0u) * fa);
          if (!part) {
#pragma unroll
            for (int w = 1; w < 16; w <<= 1)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (!(i & w)) {
                  const float u = o[i], v = o[i + w];
                  o[i] = u + v;
                  o[i + w] = u - v;
                }
          }
          float4* dst = reinterpret_cast<float4*>(to + 16 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!part || valid) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      if (some) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.o_free[g]));
      }
      if (part && valid) a.part_ml[at] = make_float2(m, l);
      if (part || !warp_rows) continue;
      // widths 16 and 32, in place: four coordinates from each of the four 16s become bf16 over the first two of them
#pragma unroll 1
      for (int i = 0; i < 16; i += 4) {
        float z[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 f = *reinterpret_cast<const float4*>(sums + i + 16 * k);
          z[0][k] = f.x, z[1][k] = f.y, z[2][k] = f.z, z[3][k] = f.w;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float p = z[w][0] + z[w][1], q = z[w][0] - z[w][1], u = z[w][2] + z[w][3], v = z[w][2] - z[w][3];
          z[w][0] = p + u, z[w][1] = q + v, z[w][2] = p - u, z[w][3] = q - v;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint2*>(sums + i + 16 * k) = make_uint2(pack_bf16(z[0][k], z[1][k]), pack_bf16(z[2][k], z[3][k]));
      }
      __syncwarp();
      // signs and permutation on the way out: eight lanes a row, which each have the same eight places in all rows
      const int tok = row / a.group, qh = e.head * a.group + row % a.group;
      const unsigned long long mine =
          (unsigned long long)((__nv_bfloat16*)a.out + (long long)(e.q_start + tok) * a.o_ld + (long long)qh * a.o_hs);
      const int n_rows = min(32, e.rows - (row - lane));
#pragma unroll 2
      for (int i = 0; i < n_rows; i += 4) {
        const int k = i + (lane >> 3);
        uint8_t* dst = (uint8_t*)__shfl_sync(0xffffffffu, mine, k);
        const uint8_t* src = stage + k * kSumPitch;
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t x = *reinterpret_cast<const uint16_t*>(src + (from[t] & 0xffffu)),
                         y = *reinterpret_cast<const uint16_t*>(src + (from[t] >> 16));
          w[t] = (x | y << 16) ^ flip[t];
        }
        if (k < n_rows) *reinterpret_cast<uint4*>(dst + 16 * (lane & 7)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncwarp();
      if (a.lse != nullptr && valid)
        a.lse[(long long)(e.q_start + tok) * (a.pool.heads * a.group) + qh] =
            l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

}  // namespace

int launch_attend_tc(const Args& a, cudaStream_t st) {
  const long long q_tiles = query_tiles((long long)a.total_q * a.group, a.num_seqs);
  const long long items = (long long)a.num_seqs * a.pool.heads * a.splits * a.row_tiles;
  CC2_REQUIRE(q_tiles <= 0x7fffffffLL && a.pool.heads <= 65535, "kv4_attention: too many rows for one call");
  static unsigned long long attr_done = 0;  // one bit per device
  int dev = 0;
  CC2_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !((attr_done >> dev) & 1ull)) {
    CC2_CUDA(cudaFuncSetAttribute(attend_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem + 1024));
    if (dev < 64) attr_done |= 1ull << dev;
  }
  const unsigned q_blocks = (unsigned)(((long long)a.total_q * a.group + 127) / 128);
  // Heads a block: as many as leave one round of blocks.  1 / 2 / 3 / 6 / 12 of 12 heads with 408576 rows (6 leave one
  // round): 182 / 170 / 170 / 167 / 174 us for the whole call.
  const int per = (int)std::min<long long>(a.pool.heads, ((long long)q_blocks * a.pool.heads + 4 * num_sms() - 1) / (4 * num_sms()));
  CC2_CUDA(launch_k(rotate_queries_kernel, dim3(q_blocks, (unsigned)((a.pool.heads + per - 1) / per)), kQThreads, 0, st, a,
                    q_tiles, per));
  const unsigned grid = (unsigned)std::min<long long>(items, num_sms());
  CC2_CUDA(launch_k(attend_tc_kernel, grid, kThreads, kSmem + 1024, st, a, q_tiles, (int)items));
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

}  // namespace kv4
}  // namespace cc2
