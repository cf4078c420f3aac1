// Attention over the 4-bit cache for many rows (prompt chunks, an encoder's
// whole series) on tcgen05, bf16 calls.  Mathematics and arguments as in
// attn_kv4.cu; here the codes of 128 keys are decoded once to shared memory and
// serve 256 rows.
//
// A first kernel rotates the queries into the codes' frame and leaves them in
// the workspace as fp16 tiles in the tensor core's shared-memory order, each
// row scaled to below 2^8.  Then persistent blocks, one an SM, walk items
// (sequence, head, 256 rows, chunk of keys):
//   warp 0        loader: finds the items, brings raw key blocks and query
//                 tiles by bulk copies
//   warps 12-15   decoders, a key a thread: K^ and V^ tiles as fp16, norms
//                 multiplied in after scaling them by a power of two a block
//   warps 1, 2    MMA issuers of the two pipelines (128 rows each):
//                 S_j = Q K_j^T, O += P_j V_j, P in TMEM
//   warps 4-11    softmax, a row a thread: running maximum (moved only past
//                 2^8), exponentials partly as a polynomial on the FMA pipe,
//                 P as fp16; at the end O back out of the codes' frame (64
//                 registers of butterflies) and to memory
// Exponents: K^ of a block is scaled by 2^-eK with eK from its largest norm,
// which goes into the scores' factor; V^ by 2^-eV, which goes into P's exponent
// against the largest eV so far.  Neither costs an operation a score.
// A masked key's column is -inf and its V^ zero.  A K or V that is not finite
// is zero too and instead marks the rows that see it (their sum becomes NaN), so
// that it cannot reach the others through 0 * NaN.
// Every wait is bounded (about 2 s): on expiry all roles leave their loops,
// copies and MMAs in flight are waited for, TMEM is freed, the kernel returns.
#include "kv4_attn.cuh"

namespace cc2 {
namespace kv4 {
namespace {

using namespace tcx;

constexpr int kThreads = 512;
// 128 x (40 + 72) + 256 x 200 = 65536 registers, what the block is launched with (512 x 128)
constexpr int kRegsControl = 40, kRegsDecode = 72, kRegsSoftmax = 200;
constexpr int kTile = 128;                      // rows of a pipeline, keys of a block
constexpr uint32_t kTileBytes = 128 * 128;      // 128 rows of 64 fp16
constexpr uint32_t kRawBytes = 8 * kBlockBytes;
constexpr int kKvStages = 3, kRawStages = 3, kItems = 4;
constexpr int kOutPitch = 132;                  // bytes a staged output row
constexpr uint32_t kQAt = 0, kKvAt = 2 * kTileBytes, kRawAt = kKvAt + kKvStages * 2 * kTileBytes,
                   kOutAt = kRawAt + kRawStages * kRawBytes, kSmem = kOutAt + 2 * 128 * kOutPitch;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSCol = 0, kPCol = 256, kOCol = 384;  // + 128 G, 64 G, 64 G for pipeline G
constexpr float kRescaleLog2 = 8.0f;
constexpr uint32_t kPolyPairs = (1u << 2) | (1u << 5) | (1u << 7) | (1u << 10) | (1u << 13) | (1u << 15);

__device__ __forceinline__ uint32_t idesc_f16(int M, int N, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? (1u << 16) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
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
  long long q_tile;
};

struct Control {
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t raw_full[kRawStages], raw_empty[kRawStages];
  uint64_t kv_full[kKvStages], kv_empty[kKvStages];
  uint64_t q_full[2], q_empty[2], s_full[2], s_free[2], p_full[2], p_free[2], o_full[2], mma_done[2];
  Item items[kItems];
  uint32_t seen[kKvStages][4];    // bit k: key k of the block counts
  uint32_t poison[kKvStages][4];  // bit k: its K or V is not finite
  int e_k[kKvStages], e_v[kKvStages];
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

// A warp's bounded wait: its lanes go on together or leave together.
__device__ __forceinline__ bool wait(uint64_t& bar, uint32_t parity, Control& c, int* err) {
  return __all_sync(0xffffffffu, mbar_wait_inl(smem_u32(&bar), parity, &c.abort_flag, err));
}

// Butterflies of a row of 64 in registers.
__device__ __forceinline__ void walsh(float* y) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1)
#pragma unroll
    for (int i = 0; i < 64; ++i)
      if (!(i & w)) {
        const float a = y[i], b = y[i + w];
        y[i] = a + b;
        y[i + w] = a - b;
      }
}

// ------------------------------------------------------------------ queries --
// A block rotates a tile of 128 rows of one head: a thread a row, as in
// kv4_cache.cu.
constexpr int kQThreads = 128, kQPitch = 65;

__global__ void __launch_bounds__(kQThreads)
rotate_queries_kernel(const __grid_constant__ Args a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float rows[128 * kQPitch];
  const int tid = threadIdx.x, lane = tid & 31;
  const int head = blockIdx.y;
  const long long tile = blockIdx.x;
  // the last sequence whose tiles start at or before this one
  int seq = -1;
  for (int i = lane; i - lane < a.num_seqs; i += 32) {
    const bool in = i < a.num_seqs &&
                    first_query_tile(a, i, a.cu != nullptr ? min(max(a.cu[i], 0), a.total_q) : i * a.max_q) <= tile;
    seq += __popc(__ballot_sync(0xffffffffu, in));
  }
  if (seq < 0) return;
  Span s = span_of(a, seq, 0, tile == 0 && head == 0 && tid == 0);
  const int row0 = (int)(tile - first_query_tile(a, seq, s.q_start)) * 128;
  if (row0 >= s.rows) return;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int r = it * 32 + (tid >> 2), c = tid & 3, row = row0 + r;
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.0f;
    if (row < s.rows) {
      const int i = row / a.group;
      const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (long long)(s.q_start + i) * a.q_ld +
                               (long long)(head * a.group + row % a.group) * a.q_hs + 8 * c;
      const uint4 u = *reinterpret_cast<const uint4*>(q), v = *reinterpret_cast<const uint4*>(q + 32);
      const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
      const int pos = s.len - s.n + i;
      if (a.rotate && pos >= 0) {
        if (pos >= a.rope_len) {
          atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
        } else {
          const float2* cs = a.rope + (long long)pos * 32 + 8 * c;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 f = cs[j];
            const float p = x[j], q1 = x[8 + j];
            x[j] = p * f.x - q1 * f.y;
            x[8 + j] = q1 * f.x + p * f.y;
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      rows[r * kQPitch + 8 * c + j] = x[j];
      rows[r * kQPitch + 32 + 8 * c + j] = x[8 + j];
    }
  }
  __syncthreads();
  float y[64];
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const float x = rows[tid * kQPitch + a.rk.perm[i]];
    y[i] = (a.rk.signs[i >> 5] >> (i & 31)) & 1u ? -x : x;
  }
  walsh(y);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    y[i] *= 0.125f * a.qscale;
    top = fmaxf(top, fabsf(y[i]));
  }
  const int e = min(max((int)(__float_as_uint(top) >> 23), 30), 254);
  const float up = __int_as_float((261 - e) << 23);  // 2^(134 - e): the row below 2^8
  const long long at = (long long)head * gridDim.x + tile;
  uint8_t* dst = const_cast<uint8_t*>(a.qt) + at * kTileBytes + tid * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c) {  // 16-byte pieces, exchanged within 8 rows as the tensor core reads them
    uint4 w;
    w.x = pack_half(y[8 * c] * up, y[8 * c + 1] * up);
    w.y = pack_half(y[8 * c + 2] * up, y[8 * c + 3] * up);
    w.z = pack_half(y[8 * c + 4] * up, y[8 * c + 5] * up);
    w.w = pack_half(y[8 * c + 6] * up, y[8 * c + 7] * up);
    *reinterpret_cast<uint4*>(dst + ((c ^ (tid & 7)) << 4)) = w;
  }
  const_cast<float*>(a.q_scale)[at * 128 + tid] = __int_as_float((e - 13) << 23);  // 2^(e - 134) / 64
}

// ---------------------------------------------------------------- attention --
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const __grid_constant__ Args a, const long long q_tiles, const int total_items) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ Control ctl;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* const err = a.wait_err;
  pdl_launch_dependents();

  if (tid == 0) {
    for (int i = 0; i < kItems; ++i) mbar_init(smem_u32(&ctl.item_full[i]), 1), mbar_init(smem_u32(&ctl.item_empty[i]), 14);
    for (int i = 0; i < kRawStages; ++i) mbar_init(smem_u32(&ctl.raw_full[i]), 1), mbar_init(smem_u32(&ctl.raw_empty[i]), 4);
    for (int i = 0; i < kKvStages; ++i) mbar_init(smem_u32(&ctl.kv_full[i]), 4), mbar_init(smem_u32(&ctl.kv_empty[i]), 2 + 8);
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&ctl.q_full[g]), 1);
      mbar_init(smem_u32(&ctl.q_empty[g]), 1);
      mbar_init(smem_u32(&ctl.s_full[g]), 1);
      mbar_init(smem_u32(&ctl.s_free[g]), 4);
      mbar_init(smem_u32(&ctl.p_full[g]), 4);
      mbar_init(smem_u32(&ctl.p_free[g]), 1);
      mbar_init(smem_u32(&ctl.o_full[g]), 1);
      mbar_init(smem_u32(&ctl.mma_done[g]), 1);
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

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
  else if (warp >= 12) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsDecode));
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));

  if (warp == 0) {
    // ---------------- loader ----------------
    Ring<kItems> it;
    Ring<kRawStages> raw;
    long long n_items = 0, n_raw = 0;
    uint32_t nq[2] = {0, 0};
    const int mask = (1 << a.pool.page_shift) - 1;
    const int run = min((mask + 1) / kBlockTokens, 8);  // blocks of 16 keys a copy brings
    bool ok = true;
    for (long long base = blockIdx.x; ok; base += 32LL * gridDim.x) {
      // each lane looks at one item
      const long long mine = base + (long long)lane * gridDim.x;
      const bool any_left = base < total_items;
      Item d;
      d.seq = -1;
      if (mine < total_items) {
        unsigned idx = (unsigned)mine;
        const int tile = (int)(idx % a.row_tiles);
        idx /= a.row_tiles;
        d.split = (int)(idx % a.splits);
        idx /= a.splits;
        d.head = (int)(idx % a.pool.heads);
        const int seq = (int)(idx / a.pool.heads);
        const Span s = span_of(a, seq, tile, false);
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
          ctl.items[it.i] = d;
          if (!any_left) ctl.items[it.i].seq = -1;
        }
        __syncwarp();
        const Item& e = ctl.items[it.i];
        const int seq = e.seq, c0 = e.c0, c1 = e.c1, head = e.head, rows = e.rows - e.row0;
        const int blocks[2] = {e.blocks[0], e.blocks[1]};
        const long long q_tile = e.q_tile;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.item_full[it.i]));
        it.next();
        ++n_items;
        if (seq < 0) {
          ok = false;
          break;
        }
        for (int g = 0; g < 2 && ok; ++g) {
          if (blocks[g] == 0) continue;
          if (nq[g] > 0 && !wait(ctl.q_empty[g], (nq[g] - 1) & 1u, ctl, err)) {
            ok = false;
            break;
          }
          if (lane == 0) {  // the tile's rows, in groups of 8
            const uint32_t bytes = (uint32_t)min((rows - kTile * g + 7) / 8, kTile / 8) * 1024u;
            mbar_arrive_expect_tx(smem_u32(&ctl.q_full[g]), bytes);
            bulk_load(smem + kQAt + g * kTileBytes, a.qt + (q_tile + g) * kTileBytes, bytes, smem_u32(&ctl.q_full[g]));
          }
          ++nq[g];
        }
        const int* table = a.table + (long long)seq * a.table_ld;
        const int nb = max(blocks[0], blocks[1]);
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
      for (int g = 0; g < 2; ++g)
        if (nq[g] > 0)
          while (!mbar_try(smem_u32(&ctl.q_full[g]), (nq[g] - 1) & 1u) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
    }
    __syncwarp();
  } else if (warp < 3) {
    // ---------------- MMA issuer of pipeline g ----------------
    const int g = warp - 1;
    Ring<kItems> it;
    Ring<kKvStages> kv_s, kv_p;  // stage of the next S, of the next P V
    uint32_t ns = 0, np = 0, nt = 0;
    const uint32_t t_s = tmem + kSCol + 128u * g, t_p = tmem + kPCol + 64u * g, t_o = tmem + kOCol + 64u * g;
    const uint64_t dq = sw128_desc(smem + kQAt + g * kTileBytes);
    bool ok = true, any = false;
    while (ok) {
      if (!wait(ctl.item_full[it.i], it.phase, ctl, err)) break;
      const Item& e = ctl.items[it.i];
      const int seq = e.seq, c0 = e.c0, blocks = e.blocks[g], key_end = e.key_end[g];
      const int all = max(e.blocks[0], e.blocks[1]);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
      it.next();
      if (seq < 0) break;
      auto issue_s = [&](int j) -> bool {
        if (!wait(ctl.kv_full[kv_s.i], kv_s.phase, ctl, err)) return false;
        if (ns > 0 && !wait(ctl.s_free[g], (ns - 1) & 1u, ctl, err)) return false;
        tc_fence_after();
        if (lane == 0) {
          const int cols = min((key_end - c0 - j * kTile + 15) / 16 * 16, kTile);
          const uint32_t id = idesc_f16(128, cols, false);
          const uint64_t dk = sw128_desc(smem + kKvAt + kv_s.i * 2 * kTileBytes);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_bf16(t_s, dq + 2u * k, dk + 2u * k, id, k > 0);
          mma_commit(smem_u32(&ctl.s_full[g]));
          if (j == blocks - 1) mma_commit(smem_u32(&ctl.q_empty[g]));
        }
        __syncwarp();
        any = true;
        kv_s.next();
        ++ns;
        return true;
      };
      if (blocks > 0) {
        if (!wait(ctl.q_full[g], nt & 1u, ctl, err)) break;
        ++nt;
        ok = issue_s(0);
        for (int j = 0; j < blocks && ok; ++j) {
          if (j + 1 < blocks) ok = issue_s(j + 1);
          if (!ok || !wait(ctl.p_full[g], np & 1u, ctl, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (lane == 0) {
            const int steps = min((key_end - c0 - j * kTile + 15) / 16, kTile / 16);
            const uint32_t id = idesc_f16(128, 64, true);
            const uint64_t dv = sw128_desc(smem + kKvAt + kv_p.i * 2 * kTileBytes + kTileBytes);
            for (int k = 0; k < steps; ++k) mma_bf16_ts(t_o, t_p + 8u * k, dv + 128u * k, id, (j > 0 || k > 0) ? 1u : 0u);
            mma_commit(smem_u32(&ctl.p_free[g]));
            mma_commit(smem_u32(&ctl.kv_empty[kv_p.i]));
            if (j == blocks - 1) mma_commit(smem_u32(&ctl.o_full[g]));
          }
          __syncwarp();
          kv_p.next();
          ++np;
        }
      }
      for (int j = blocks; j < all && ok; ++j) {  // blocks that only the other pipeline's rows see
        if (!wait(ctl.kv_full[kv_p.i], kv_p.phase, ctl, err)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive(smem_u32(&ctl.kv_empty[kv_p.i]));
        __syncwarp();
        kv_p.next();
        kv_s.next();
      }
    }
    if (any && lane == 0) {  // every MMA has completed before TMEM is released
      mma_commit(smem_u32(&ctl.mma_done[g]));
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try(smem_u32(&ctl.mma_done[g]), 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
    __syncwarp();
  } else if (warp >= 12) {
    // ---------------- decoders ----------------
    Ring<kItems> it;
    Ring<kRawStages> raw;
    Ring<kKvStages> kv;
    long long n_kv = 0;
    const int k = tid - 12 * 32, w = warp - 12;  // key of the block, warp
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
          uint16_t kb, vb;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(kb) : "r"(src + kKNorms + (k & 15) * 2));
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(vb) : "r"(src + kVNorms + (k & 15) * 2));
          nbits = kb | (uint32_t)vb << 16;
        }
        const bool seen = !(nbits & 0x8000u) && c0 + j * kTile + k < c1;
        float nk = seen ? norm_value((uint16_t)nbits, a.pool.norm_bf16) : 0.0f;
        float nv = seen ? norm_value((uint16_t)(nbits >> 16), a.pool.norm_bf16) : 0.0f;
        const bool bad = !(nv <= 3.402823466e38f && nk <= 3.402823466e38f);
        if (bad) nk = nv = 0.0f;
        const uint32_t sb = __ballot_sync(0xffffffffu, seen), pb = __ballot_sync(0xffffffffu, bad);
        const uint32_t tk = __reduce_max_sync(0xffffffffu, __float_as_uint(nk)) >> 23;
        const uint32_t tv = __reduce_max_sync(0xffffffffu, __float_as_uint(nv)) >> 23;
        if (lane == 0) ctl.top[flip][w] = tk | tv << 16;
        ok = barrier_and(1, 128, ok);
        if (!ok) break;
        uint32_t ek = 20, ev = 20;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t t = ctl.top[flip][i];
          ek = max(ek, t & 0xffffu);
          ev = max(ev, t >> 16);
        }
        flip ^= 1u;
        if (lane == 0) {
          ctl.seen[kv.i][w] = sb;
          ctl.poison[kv.i][w] = pb;
          if (w == 0) ctl.e_k[kv.i] = (int)ek, ctl.e_v[kv.i] = (int)ev;
        }
        // norms below 1: 2^(126 - e)
        const __half2 hk = __float2half2_rn(nk * __int_as_float((253 - (int)ek) << 23));
        const __half2 hv = __float2half2_rn(nv * __int_as_float((253 - (int)ev) << 23));
        const uint32_t dst = smem + kKvAt + kv.i * 2 * kTileBytes + k * 128;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const Levels& lv = m ? a.lv : a.lk;
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
              decode_pairs(c[i], lv.lo, lv.hi, o);
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
  } else if (warp >= 4) {
    // ---------------- softmax and output of pipeline g ----------------
    const int g = warp >= 8 ? 1 : 0, quarter = warp & 3, r = 32 * quarter + lane;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16);
    const uint32_t t_s = t_lane + kSCol + 128u * g, t_p = t_lane + kPCol + 64u * g, t_o = t_lane + kOCol + 64u * g;
    Ring<kItems> it;
    Ring<kKvStages> kv;
    uint32_t ns = 0, np = 0, nt = 0;
    bool ok = true;
    while (ok) {
      if (!wait(ctl.item_full[it.i], it.phase, ctl, err)) break;
      const Item& in = ctl.items[it.i];
      struct {
        int seq, head, row0, rows, q_start, split, chunks, c0, key_end;
      } e = {in.seq, in.head, in.row0, in.rows, in.q_start, in.split, in.chunks, in.c0, in.key_end[g]};
      const int blocks = in.blocks[g], all = max(in.blocks[0], in.blocks[1]);
      const int row = e.row0 + kTile * g + r;
      const bool valid = row < e.rows;
      const bool warp_rows = e.row0 + kTile * g + 32 * quarter < e.rows;
      const int tok = row / a.group;
      const int limit = a.causal ? min(in.len - in.n + tok + 1, in.len) : in.len;  // keys the row sees
      const int clear = a.causal ? in.len - in.n + (e.row0 + kTile * g) / a.group + 1 : in.len;
      const long long q_tile = in.q_tile;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[it.i]));
      it.next();
      if (e.seq < 0) break;
      const float rs = valid && blocks > 0 ? a.q_scale[(q_tile + g) * 128 + r] : 0.0f;
      float m = -INFINITY, l = 0.0f;
      int ve = 0;
      for (int j = 0; j < blocks; ++j) {
        // the decoders' notes on the block, then the scores
        if (!wait(ctl.kv_full[kv.i], kv.phase, ctl, err) || !wait(ctl.s_full[g], ns & 1u, ctl, err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int key0 = e.c0 + j * kTile;
        uint32_t sw[4], pw = 0;
        bool clean = key0 + kTile <= clear;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sw[i] = ctl.seen[kv.i][i];
          pw |= ctl.poison[kv.i][i];
          clean = clean && sw[i] == 0xffffffffu;
        }
        clean = clean && pw == 0;
        const float sc = rs * __int_as_float((ctl.e_k[kv.i] + 1) << 23);  // rs 2^(eK - 126)
        const int ev = ctl.e_v[kv.i];
        const int cols = min(e.key_end - key0, kTile);
        uint32_t v[128];
        if (warp_rows) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (32 * c < cols) tmem_ld32(t_s + 32u * c, v + 32 * c);
          tmem_ld_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.s_free[g]));
        ++ns;
        float scale = 1.0f;
        bool rescale = false;
        if (warp_rows) {
          if (!clean) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (32 * c < cols) {
                const int rel = limit - key0 - 32 * c;
                const uint32_t vis = rel >= 32 ? sw[c] : rel <= 0 ? 0u : sw[c] & ((1u << rel) - 1u);
                if (ctl.poison[kv.i][c] & vis) l = __int_as_float(0x7fffffff);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!((vis >> i) & 1u)) v[32 * c + i] = 0xff800000u;
              }
            }
          }
          float b0 = -INFINITY, b1 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (32 * c < cols) {
#pragma unroll
              for (int i = 32 * c; i < 32 * c + 32; i += 4) {
                b0 = max3(b0, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                b1 = max3(b1, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
              }
            }
          const float bm = fmaxf(b0, b1) * sc;
          if (j == 0) {
            m = bm;
            ve = ev;
          } else {
            if (bm > m + kRescaleLog2 || (m == -INFINITY && bm > m)) {
              scale = m == -INFINITY ? 0.0f : ex2(m - bm);
              l *= scale;
              m = bm;
              rescale = true;
            }
            if (ev > ve) {
              scale *= __int_as_float((127 - min(ev - ve, 126)) << 23);
              ve = ev;
              rescale = true;
            }
          }
        }
        if (np > 0 && !wait(ctl.p_free[g], (np - 1) & 1u, ctl, err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_rows) {
          // P = 2^(x - m) times 2^(eV - largest eV), the latter taken back out of the row's sum
          const float dv = (float)max(ev - ve, -60);
          const float off = (m == -INFINITY ? 0.0f : -m) + dv;
          const uint64_t sc2 = f2_pack(sc, sc), off2 = f2_pack(off, off);
          uint64_t l2 = f2_pack(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (32 * c < cols) {
              uint32_t pk[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const uint64_t x2 =
                    f2_fma(f2_pack(__uint_as_float(v[32 * c + 2 * k]), __uint_as_float(v[32 * c + 2 * k + 1])), sc2, off2);
                uint64_t p2;
                if ((kPolyPairs >> k) & 1u) {
                  p2 = f2_exp2_poly(x2);
                } else {
                  float x0, x1;
                  f2_unpack(x2, x0, x1);
                  p2 = f2_pack(ex2(x0), ex2(x1));
                }
                l2 = f2_add(l2, p2);
                float p0, p1;
                f2_unpack(p2, p0, p1);
                pk[k] = pack_half(p0, p1);
              }
              tmem_st16(t_p + 16u * c, pk);
            }
          }
          float l0, l1;
          f2_unpack(l2, l0, l1);
          l += (l0 + l1) * __int_as_float((127 - (int)dv) << 23);
        }
        if (j > 0 && __any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + 32u * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * scale);
            tmem_st32(t_o + 32u * c, o);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&ctl.p_full[g]));
          mbar_arrive(smem_u32(&ctl.kv_empty[kv.i]));
        }
        ++np;
        kv.next();
      }
      if (!ok) break;
      for (int j = blocks; j < all; ++j) {
        if (!wait(ctl.kv_full[kv.i], kv.phase, ctl, err)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive(smem_u32(&ctl.kv_empty[kv.i]));
        kv.next();
      }
      if (!ok) break;
      float o[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) o[i] = 0.0f;
      if (blocks > 0) {
        if (!wait(ctl.o_full[g], nt & 1u, ctl, err)) {
          ok = false;
          break;
        }
        ++nt;
        tc_fence_after();
        if (warp_rows) {
#pragma unroll
          for (int c = 0; c < 2; ++c) tmem_ld32(t_o + 32u * c, reinterpret_cast<uint32_t*>(o) + 32 * c);
          tmem_ld_wait();
        }
        tc_fence_before();
      }
      if (!warp_rows) continue;
      if (m == -INFINITY && l == l) l = 0.0f;
      const float down = blocks > 0 ? __int_as_float((ve - 5) << 23) : 0.0f;  // 2^(eV - 126) / 64
      if (e.chunks > 1) {
        if (valid) {
          Span s;
          s.q_start = e.q_start;
          const long long at = part_at(a, s, e.head, e.split, row);
          float4* dst = reinterpret_cast<float4*>(a.part + at * 64);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            dst[i] = make_float4(o[4 * i] * down, o[4 * i + 1] * down, o[4 * i + 2] * down, o[4 * i + 3] * down);
          a.part_ml[at] = make_float2(m, l);
        }
        continue;
      }
      const float inv = l == 0.0f ? 0.0f : down * 0.125f / l;
#pragma unroll
      for (int i = 0; i < 64; ++i) o[i] *= inv;
      walsh(o);
      // out through shared memory: the permutation, then whole rows
      const uint32_t stage = smem + kOutAt + g * 128 * kOutPitch + 32 * quarter * kOutPitch;
      const uint32_t my = stage + lane * kOutPitch;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const uint16_t b = __bfloat16_as_ushort(__float2bfloat16_rn((a.rv.signs[i >> 5] >> (i & 31)) & 1u ? -o[i] : o[i]));
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(my + 2u * a.rv.perm[i]), "h"(b) : "memory");
      }
      __syncwarp();
      const int qh = e.head * a.group + row % a.group;
      const unsigned long long mine =
          (unsigned long long)((__nv_bfloat16*)a.out + (long long)(e.q_start + tok) * a.o_ld + (long long)qh * a.o_hs);
      const int n_rows = min(32, e.rows - (e.row0 + kTile * g + 32 * quarter));
      for (int i = 0; i < n_rows; ++i) {
        uint32_t* dst = (uint32_t*)__shfl_sync(0xffffffffu, mine, i);
        uint32_t x;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(stage + i * kOutPitch + 4 * lane));
        dst[lane] = x;
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
  CC2_CUDA(launch_k(rotate_queries_kernel, dim3((unsigned)q_tiles, (unsigned)a.pool.heads), kQThreads, 0, st, a));
  const unsigned grid = (unsigned)std::min<long long>(items, num_sms());
  CC2_CUDA(launch_k(attend_tc_kernel, grid, kThreads, kSmem + 1024, st, a, q_tiles, (int)items));
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

}  // namespace kv4
}  // namespace cc2
