// Attention over the paged 4-bit K/V cache (layout: kv4.cuh, definition: cc2.h).
//
// With K^ = n_k R^T c_k and V^ = n_v R'^T c_v (R the quantiser's rotation, c the
// codes' levels) the cache is never rotated back:
//   q . K^ = n_k (R q) . c_k,     sum p V^ = R'^T sum (p n_v) c_v,
// so a row is rotated once going in and once coming out, and the products run
// on the levels themselves, as fp16 on the tensor cores with fp32 sums.
//
// Rows are the queries of one sequence that share a head of keys: row r is
// query token r / group, head r % group.  A unit of work is one head of keys of
// one sequence, up to 4, 8, 16 or 32 rows and a chunk of the keys; persistent blocks walk
// the units, one for each of their teams of warps; a team's warps take 64-key
// stages of its unit in turn, each with a ring of its own that bulk copies fill,
// and an online softmax of its own, joined at the end of the unit while the next
// one's first stage is on its way.
//   S^T (16 keys x 8 rows) = K (the A operand, decoded in registers) . Q^T
//   O^T (16 coordinates x 8 rows) += V^T (A, decoded) . P^T
// Keys and coordinates as the long axis of the product: one token's query
// fills 2 of 8 columns (its two fp16 parts) and not 2 of 16 rows.  P^T comes from S^T by one matrix
// move a register pair.
// Decoding: a byte of codes is an fp16 pair (K: neighbouring coordinates; V: one
// coordinate of two tokens, their words zipped first), looked up in a table of
// 256 pairs in shared memory that every lane has its own bank's copy of, so no
// lookup waits for another: one byte permute makes the address of two values
// (the code byte above the lane's place, hence 256 bytes an entry) and one load
// brings them.  One block an SM, for one table.  Byte permutes of the levels' bytes
// took 1.6 (K) and 2.1 (V) operations a value on the half-rate integer pipe, which
// was 73% busy and bound the kernel.
// Measured, one token for each of 64 sequences of up to 16384 tokens, 12 heads
// (484 MB of cache): 145 us, 3.3 TB/s; 207 us with the byte permutes; 192 us with
// a fixed chunk of keys a block instead of the call's work cut evenly over teams
// that stay.  A stage of 64 keys takes a warp some 815 instructions; issue slots
// are 63% used, the load/store pipe 58% and the integer pipe 51%, with 16 warps
// an SM: at 128 registers they fill the register file.  Of the table's 64 KB
// bf16 calls use every other 128 bytes, fp32 calls all.
// What must not leave the type's range is scaled by powers of two, which are
// exact: a row of Q to below 2^8, P n_v to below 2^14 against the largest norm
// met so far; in fp32 calls against the row's largest P n_v itself, so that two
// fp16 parts keep 2^-22 of it whatever the norms beside it (against the largest
// norm a row was off by 6e-5 where that was 2^16 above those that counted; the
// row's own costs 3 to 4%: 64 sequences of 4096 tokens, 8 heads, 2 rows a head
// 94 us for 91).
// Rounding: P n_v to fp16 (2^-12 of each, next to the output's bf16 with 2^-9;
// from 2^-20 of the largest norm met on, below it a bit less for each power of
// two),
// the levels to fp16 after a common factor that moves all of them close to its
// values, Q to one or two fp16 parts (split_q).  fp32 calls split all three into
// two parts and sum three products, which leaves about 2^-22.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "kv4_attn.cuh"

namespace cc2 {
namespace kv4 {

// fp16 keeps the levels to 2^-12 of each at best, the same error in every key.
// One factor for all of them, taken out again exactly where it does not matter,
// moves them: of 32 in an octave the one that leaves the least, weighted by how
// much of a vector's length a level holds (coordinates are nearly normal with
// variance 1 / 64).  Lloyd-Max levels: 2.4e-4 of a level without, 0.9e-4 with it.
float level_scale(const float (&c)[8]) {
  float weight[8], best = INFINITY, scale = 64.0f;
  for (int i = 0; i < 8; ++i) {
    const float width = i < 7 ? c[i + 1] - c[i] : c[i] - c[i - 1];
    weight[i] = width * std::exp(-32.0f * c[i] * c[i]);
  }
  for (int k = 0; k < 64; k += 2) {
    const float f = 64.0f + (float)k;
    float sum = 0.0f;
    for (int i = 0; i < 8; ++i) {
      const float x = f * c[i];
      uint32_t u;
      memcpy(&u, &x, sizeof u);
      u = (u + 0xfffu + ((u >> 13) & 1u)) & ~0x1fffu;  // 11 bits
      float h;
      memcpy(&h, &u, sizeof h);
      sum += weight[i] * (h - x) * (h - x);
    }
    sum /= f * f;
    if (sum < best) best = sum, scale = f;
  }
  return scale;
}

Levels make_levels(const cc2_kv4_cache& cache) {
  Levels r{};
  r.scale = level_scale(cache.levels);
  for (int i = 0; i < 8; ++i) {
    const float c = r.scale * cache.levels[i];
    const __half h = __float2half_rn(c);
    r.value[i] = __half_as_ushort(h);
    r.rest[i] = __half_as_ushort(__float2half_rn(c - __half2float(h)));
    r.lo[i >> 2] |= (uint32_t)(r.value[i] & 255) << 8 * (i & 3);
    r.hi[i >> 2] |= (uint32_t)(r.value[i] >> 8) << 8 * (i & 3);
  }
  return r;
}

namespace {

using namespace tcx;

constexpr int kStageKeys = 64;
constexpr int kStageBytes = kStageKeys / kBlockTokens * kBlockBytes;  // 4352
// Whether a bf16 call is the tcgen05 kernel's.  It costs the same for 17 rows of a
// sequence and head as for 128; this one costs a pass over the keys for each 32
// rows, but less for a key and more for a sequence.  This one / tcgen05, us, 8 heads:
//   20 to 24 rows, 256 sequences of 1024 tokens 237 / 203, of 1500 271 / 274,
//   64 sequences of 512 62 / 47, of 2048 102 / 117, 16 of 8192 72 / 123;
//   32 rows, 256 sequences of 256 tokens 129 / 90, 64 of 1024 90 / 70, 32 of 4096 79 / 117;
//   40 rows, 64 sequences of 2048 tokens 165 / 127, 32 of 4096 121 / 121, 16 of 8192 106 / 128;
//   64 rows, 64 sequences of 2048 tokens 183 / 138, 32 of 4096 136 / 127, 1 of 32768 52 / 43;
//   16 rows, 256 sequences of 512 tokens 130 / 129, 64 of 1024 55 / 67.
bool for_tcgen05(int dtype, int rows, int max_len) {
  return dtype == CC2_BF16 && (rows > 32 || (rows > 16 && max_len <= 1024));
}
constexpr int kQPitch = 72;  // halves
constexpr int kOPitch = 66;  // floats

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float2 unpack_half(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
// Teams of a block and their warps: what registers and shared memory leave room for.
template <int R, bool F32> constexpr int teams_of() { return R == 16 && !F32 ? 3 : 2; }
// Whether Q is held as two fp16 parts.  One part's rounding, the same for every key, is most of what a long context
// costs in precision (131072 keys, scores of deviation 2: 0.9e-3 of the output next to its own rounding's 1.7e-3, 0.4e-3
// with both).  Up to 4 rows the second part takes columns that would be empty; as products of their own they cost 5%
// with 8 rows and 10% with 16, and would 17% with 32, which keeps one like the tcgen05 kernel.
template <int R, bool F32> constexpr bool split_q() { return R <= 16 || F32; }
template <int R, bool F32> constexpr int warps_of() { return R <= 8 && !F32 ? 8 : 4; }

template <int R, bool F32>
struct Shared {
  static constexpr int kTeams = teams_of<R, F32>(), kWarps = warps_of<R, F32>(), kRows = R;
  struct Team {
    alignas(128) uint8_t ring[kWarps][2][kStageBytes];
    alignas(16) __half q[split_q<R, F32>() ? 2 : 1][kRows][kQPitch];  // and what its rounding leaves
    float rs[kRows];
    float m[kWarps][kRows], l[kWarps][kRows];
    uint64_t full[kWarps][2];
    const float* sums[kWarps];  // a warp's joined sums: in its ring, beside the slot that the next unit's first stage takes
  };
  alignas(256) uint8_t pairs[256][256];  // every lane's copy of the pair of codes (low nibble, high nibble); fp32: and its rest
  Team team[kTeams];
  Turns turns;
  int abort_flag;
  static_assert(kRows * kOPitch * 4 <= 2 * kStageBytes, "a warp's sums fit its ring");
};
// Whether a warp's sums leave one slot of its ring free.
template <int R> constexpr bool sums_in_a_slot() { return R * kOPitch * 4 <= kStageBytes; }

template <bool kBf16> __device__ __forceinline__ float norm_of(uint32_t bits) { return norm_value((uint16_t)bits, kBf16); }

// Walks a team's rounds unit by unit; every warp of the team does so for itself,
// its lanes holding 32 sequences' places on the line.
struct Walk {
  long long at, end;         // the team's rounds
  int window;                // first of the 32 sequences
  SeqCost mine;              // of sequence window + lane
  long long cost_at, unit_at;  // where that sequence starts
  long long window_end, window_units;
  // what next() found
  int seq, head, tile, r0, r1;
  long long unit;
  bool whole;

  __device__ __forceinline__ void load(const Args& a, int lane, long long cost0, long long units0, bool report = false) {
    mine = SeqCost{0, 0, 0, 0};
    if (window + lane < a.num_seqs) mine = cost_of(a, window + lane, report);
    long long c = mine.cost, u = mine.units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long pc = __shfl_up_sync(0xffffffffu, c, o), pu = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) c += pc, u += pu;
    }
    window_end = cost0 + __shfl_sync(0xffffffffu, c, 31);
    window_units = units0 + __shfl_sync(0xffffffffu, u, 31);
    cost_at = cost0 + c - mine.cost;
    unit_at = units0 + u - mine.units;
  }
  __device__ __forceinline__ void start(const Args& a, int team, int lane) {
    long long total = 0;
    if (a.num_seqs <= 32) {
      window = 0;
      load(a, lane, 0, 0, team == 0);  // what is out of range shows here: a sequence may have no unit
      total = window_end;
    } else {
      for (int i = lane; i < a.num_seqs; i += 32) total += cost_of(a, i, team == 0).cost;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      window = 0;
      load(a, lane, 0, 0);
    }
    at = team_start(total, team, a.teams);
    end = team_start(total, team + 1, a.teams);
  }
  __device__ __forceinline__ bool next(const Args& a, int lane) {
    while (at < end) {
      while (at >= window_end) {
        window += 32;
        load(a, lane, window_end, window_units);
      }
      const unsigned before = __ballot_sync(0xffffffffu, mine.cost > 0 && cost_at <= at);
      const int src = 31 - __clz(before);
      seq = window + src;
      const int tiles = __shfl_sync(0xffffffffu, mine.tiles, src), rounds = __shfl_sync(0xffffffffu, mine.rounds, src);
      const long long rest = at - __shfl_sync(0xffffffffu, cost_at, src);
      const long long k = rest / (rounds + 1);
      r0 = (int)(rest - k * (rounds + 1));
      unit = __shfl_sync(0xffffffffu, unit_at, src) + k;
      head = (int)(k / tiles);
      tile = (int)(k % tiles);
      r1 = (int)min((long long)rounds, r0 + (end - at));
      whole = r0 == 0 && r1 == rounds;
      at += rounds + 1 - r0;
      if (r0 < r1) return true;
    }
    return false;
  }
};

// R rows a tile: 4 (each in two columns of the products), or 8, 16, 32 in as many columns.
template <int R, bool F32, bool NormBf16>
__global__ void __launch_bounds__(32 * warps_of<R, F32>() * teams_of<R, F32>(), 1)
attend_kernel(const __grid_constant__ Args a) {
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  using S = Shared<R, F32>;
  constexpr bool kPaired = R == 4;
  constexpr int NB = kPaired ? 1 : R / 8, kPer = kPaired ? 1 : 2;  // blocks of 8 columns, rows of a lane in one
  constexpr bool kSplit = !kPaired && split_q<R, F32>();           // Q's second part by products of its own
  constexpr int kRows = S::kRows, kWarps = S::kWarps;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  S& all = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, team = (tid >> 5) / kWarps, warp = (tid >> 5) % kWarps;
  typename S::Team& sm = all.team[team];
  const int g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sm.full[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) all.abort_flag = 0;
  load_turns(all.turns, a, tid);
  for (int e = tid >> 5; e < 256; e += kWarps * S::kTeams) {  // the table; an entry's 32 copies by one store
    const uint32_t i = e & 7, j = (e >> 4) & 7, sign = (uint32_t)(e & 8) << 12 | (uint32_t)(e & 128) << 24;
    const uint32_t v = ((uint32_t)a.levels.value[i] | (uint32_t)a.levels.value[j] << 16) ^ sign;
    if (F32) {
      const uint32_t r = ((uint32_t)a.levels.rest[i] | (uint32_t)a.levels.rest[j] << 16) ^ sign;
      reinterpret_cast<uint2*>(all.pairs[e])[lane] = make_uint2(v, r);
    } else {
      reinterpret_cast<uint32_t*>(all.pairs[e])[lane] = v;
    }
  }
  pdl_wait();
  __syncthreads();
  // every lane of the team's warps, and whether all say yes
  auto meet = [&](bool yes) { return barrier_and(1u + (uint32_t)team, 32u * kWarps, yes); };

  // the pairs of a word's four bytes
  const uint32_t mine_at = (uint32_t)lane * (F32 ? 8u : 4u);
  auto look = [&](uint32_t w, uint32_t (&v)[4], uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = __byte_perm(w, mine_at, 0x6604 | i << 4);  // byte 0 the lane's place, byte 1 the codes
      if (F32) {
        const uint2 x = *reinterpret_cast<const uint2*>(smem_raw + at);
        v[i] = x.x, r[i] = x.y;
      } else {
        v[i] = *reinterpret_cast<const uint32_t*>(smem_raw + at);
      }
    }
  };

  // a stage's blocks of 16 keys, page by page (a page of 64 tokens or more holds
  // a whole stage), into the slot of the warp's stage number n
  const int run = min((1 << a.pool.page_shift) / kBlockTokens, 4);  // blocks of a copy
  struct Unit {
    Span s;
    int seq, head, c0, c1, stages;  // its keys, this warp's stages of them
    long long piece;
    bool whole;
  };
  auto issue = [&](const Unit& u, int i, uint32_t n) {
    const int c1 = u.c1, key0 = u.c0 + (warp + kWarps * i) * kStageKeys;
    const int blocks = min((c1 - key0 + kBlockTokens - 1) / kBlockTokens, 4);
    const uint32_t bar = smem_u32(&sm.full[warp][n & 1u]);
    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)blocks * kBlockBytes);
    __syncwarp();
    const int first = lane * run;
    if (first < blocks) {
      const int key = key0 + first * kBlockTokens;
      int page = a.table[(long long)u.seq * a.table_ld + (key >> a.pool.page_shift)];
      if ((unsigned)page >= (unsigned)a.pool.num_pages) {
        atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
        page = 0;  // in bounds; the rows are unspecified
      }
      const uint8_t* src = a.pool.pages + block_offset(a.pool, page, u.head, key & ((1 << a.pool.page_shift) - 1));
      bulk_load(smem_u32(sm.ring[warp][n & 1u]) + (uint32_t)first * kBlockBytes, src,
                (uint32_t)min(run, blocks - first) * kBlockBytes, bar);
    }
  };
  Walk walk;
  const int team_at = (int)blockIdx.x * S::kTeams + team;
  walk.start(a, team_at, lane);
  if (a.fill) fill_rows<T>(a, blockIdx.x * blockDim.x + tid, gridDim.x * blockDim.x);
  auto next = [&](Unit& u) {
    if (!walk.next(a, lane)) return false;
    u.s = span_of(a, walk.seq, walk.tile, false);
    u.seq = walk.seq;
    u.head = walk.head;
    u.c0 = walk.r0 * (kWarps * kStageKeys);
    u.c1 = min(u.s.keys, walk.r1 * (kWarps * kStageKeys));
    const int stages = u.c1 > u.c0 ? (u.c1 - u.c0 + kStageKeys - 1) / kStageKeys : 0;
    u.stages = stages > warp ? (stages - 1 - warp) / kWarps + 1 : 0;
    u.piece = walk.unit + team_at;
    u.whole = walk.whole;
    return true;
  };
  Unit coming;
  bool more = next(coming);
  uint32_t n = 0;      // stages that this warp has taken
  int ahead = 0;       // of the unit's stages, those under way
  bool broken = false;
  while (more) {
    const Unit u = coming;
    const Span& s = u.s;
    const int c0 = u.c0, c1 = u.c1, mine = u.stages;
    for (; ahead < min(mine, 2); ++ahead) issue(u, ahead, n + (uint32_t)ahead);

    // the rows: rotated to their positions, then as the keys' codes are, scaled
    for (int r = warp; r < kRows; r += kWarps) {
      const int row = s.row0 + r;
      if (row >= s.rows) {  // a column of zeros
#pragma unroll
        for (int p = 0; p < (split_q<R, F32>() ? 2 : 1); ++p) sm.q[p][r][lane] = sm.q[p][r][lane + 32] = __float2half_rn(0.0f);
        if (lane == 0) sm.rs[r] = 1.0f;
        continue;
      }
      const int i = row / a.group;
      const T* q = (const T*)a.q + (long long)(s.q_start + i) * a.q_ld +
                   (long long)(u.head * a.group + row % a.group) * a.q_hs;
      float x0 = tof<T>(q[lane]), x1 = tof<T>(q[lane + 32]);
      const int pos = s.len - s.n + i;
      if (a.rotate && pos >= 0) {
        if (pos >= a.rope_len) {
          if (lane == 0) atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
        } else {
          const float2 cs = a.rope[(long long)pos * 32 + lane];
          const float x = x0;
          x0 = x * cs.x - x1 * cs.y;
          x1 = x1 * cs.x + x * cs.y;
        }
      }
      float y0 = flip(spread_get(x0, x1, all.turns.k_perm[lane]), a.rk.signs, 0, lane);
      float y1 = flip(spread_get(x0, x1, all.turns.k_perm[lane + 32]), a.rk.signs, 1, lane);
      spread_walsh(y0, y1, lane);
      y0 *= a.qscale;
      y1 *= a.qscale;
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(y0), fabsf(y1))));
      const int e = min(max((int)(top >> 23), 30), 254);
      const float up = __int_as_float((261 - e) << 23);  // 2^(134 - e)
      y0 *= up;
      y1 *= up;
      const __half g0 = __float2half_rn(y0), g1 = __float2half_rn(y1);
      sm.q[0][r][lane] = g0;
      sm.q[0][r][lane + 32] = g1;
      if (split_q<R, F32>()) {
        sm.q[split_q<R, F32>() ? 1 : 0][r][lane] = __float2half_rn(y0 - __half2float(g0));
        sm.q[split_q<R, F32>() ? 1 : 0][r][lane + 32] = __float2half_rn(y1 - __half2float(g1));
      }
      if (lane == 0) sm.rs[r] = __int_as_float((e - 13) << 23);  // 2^(e - 134) / 64: undoes both scalings
    }
    meet(true);

    uint32_t qf[NB][kSplit ? 16 : 8];
    float rs[NB][2];
    int limit[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int p = 0; p < (kSplit ? 2 : 1); ++p) {  // a paired row's parts are neighbouring columns
        const __half* column = kPaired ? sm.q[kPaired ? g & 1 : 0][g >> 1] : sm.q[p][8 * b + g];
        const uint4* src = reinterpret_cast<const uint4*>(column + 16 * t);
        const uint4 x = src[0], y = src[1];
        uint32_t* d = &qf[b][8 * p];
        d[0] = x.x, d[1] = x.y, d[2] = x.z, d[3] = x.w, d[4] = y.x, d[5] = y.y, d[6] = y.z, d[7] = y.w;
      }
#pragma unroll
      for (int c = 0; c < kPer; ++c) {
        const int r = 8 * b + kPer * t + c;
        rs[b][c] = sm.rs[r];
        limit[b][c] = a.causal ? min(s.len - s.n + (s.row0 + r) / a.group + 1, s.len) : s.len;
      }
    }
    // every row sees all keys below `clear`
    const int clear = a.causal ? s.len - s.n + s.row0 / a.group + 1 : s.len;

    float m[NB][2], lift[NB][2], neg[NB][2], l[NB][2], acc[4][NB][4];
    int pe[NB][2];  // fp32: exponent of the row's largest P n_v
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b][0] = m[b][1] = lift[b][0] = lift[b][1] = -INFINITY;
      neg[b][0] = neg[b][1] = 0.0f;
      pe[b][0] = pe[b][1] = 20;
      l[b][0] = l[b][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][b][0] = acc[i][b][1] = acc[i][b][2] = acc[i][b][3] = 0.0f;
    }
    int ve = 20;  // exponent of the largest V norm met
    const int krow = (g >> 1) + 4 * (g & 1);  // key of S^T rows g and (+ 8) g + 8 in a block of 16

    // One stage of 64 keys.  kEdge: some key is past the end or not for every row.
    auto attend_stage = [&](auto edge_, uint32_t stage, int key0, const uint32_t (&nb)[4][2]) {
      constexpr bool kEdge = decltype(edge_)::value;
      float x[4][NB][4];
      float nv[4][2];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t blk = stage + j * kBlockBytes;
#pragma unroll
        for (int b = 0; b < NB; ++b) x[j][b][0] = x[j][b][1] = x[j][b][2] = x[j][b][3] = 0.0f;
        const uint2 w0 = lds64(blk + krow * 32 + t * 8), w1 = lds64(blk + (krow + 8) * 32 + t * 8);
        const uint32_t wa[2] = {w0.x, w0.y}, wb[2] = {w1.x, w1.y};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t da[4], db[4], ra[4], rb[4];
          look(wa[h], da, ra);
          look(wb[h], db, rb);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t f[4] = {da[2 * p], db[2 * p], da[2 * p + 1], db[2 * p + 1]};
            const int k = 2 * (2 * h + p);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              if (F32) {
                const uint32_t e[4] = {ra[2 * p], rb[2 * p], ra[2 * p + 1], rb[2 * p + 1]};
                mma(x[j][b], e, qf[b][k], qf[b][k + 1]);
              }
              if (kSplit) mma(x[j][b], f, qf[b][kSplit ? 8 + k : k], qf[b][kSplit ? 9 + k : k]);
              mma(x[j][b], f, qf[b][k], qf[b][k + 1]);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float nk = norm_of<NormBf16>(nb[j][c]);
          nv[j][c] = norm_of<NormBf16>(nb[j][c] >> 16);
          const bool seen = !(nb[j][c] & 0x8000u) && (!kEdge || key0 + 16 * j + krow + 8 * c < c1);
          if (!seen) nk = nv[j][c] = 0.0f;
          // where not every row sees a V that is not finite, it must not set the scale for the others
          if (!kEdge || nv[j][c] <= 3.402823466e38f) top = max(top, __float_as_uint(nv[j][c]));
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              float& v = x[j][b][2 * c + i];
              if (kPaired) v += x[j][b][2 * c + 1];
              v *= nk;
              if (!seen || (kEdge && key0 + 16 * j + krow + 8 * c >= limit[b][i])) v = -INFINITY;
            }
        }
      }

      // The running maximum moves only when a score is more than 2^8 above it, the
      // largest norm when a larger one comes; then the sums so far follow.
      const int ve_new = F32 ? ve : max(ve, (int)(__reduce_max_sync(0xffffffffu, top) >> 23));
      float mx[NB][2];
      float drop[NB][2];  // fp32: log2 of what the maximum's move takes the sums down by
      bool moved = ve_new != ve;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
          drop[b][c] = 0.0f;
          float v = -INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j) v = max3(v, x[j][b][c], x[j][b][c + 2]);
          mx[b][c] = v;
          moved = moved || v > lift[b][c];
        }
      if (__any_sync(0xffffffffu, moved)) {
        const float fv = __int_as_float((127 + max(ve - ve_new, -126)) << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < kPer; ++c) {
            float v = mx[b][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            v = fmaxf(m[b][c], v);
            drop[b][c] = m[b][c] == -INFINITY ? -INFINITY : (m[b][c] - v) * rs[b][c];
            const float f = ex2(drop[b][c]);
            m[b][c] = v;
            neg[b][c] = v == -INFINITY ? 0.0f : -v * rs[b][c];
            lift[b][c] = v + 8.0f / rs[b][c];  // -inf until a key is seen
            l[b][c] *= f;
            if (F32) continue;  // its sums follow below
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              acc[k][b][c] *= f * fv;
              acc[k][b][c + 2] *= f * fv;
            }
          }
        ve = ve_new;
      }
      float up[NB][2];  // fp32: 2^(140 - pe)
      if (F32) {
        // Scores become P n_v.  The exponent that a row's have moves when one passes 2^15 by it or its maximum moved; then
        // the sums so far follow.
        bool other = moved;
        float most[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          most[b][0] = most[b][1] = 0.0f;
          const uint64_t r2 = f2_pack(rs[b][0], rs[b][1]), g2 = f2_pack(neg[b][0], neg[b][1]);
          uint64_t l2 = f2_pack(l[b][0], l[b][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& v0 = x[j][b][2 * i];
              float& v1 = x[j][b][2 * i + 1];
              float p0, p1;
              f2_unpack(f2_fma(f2_pack(v0, v1), r2, g2), p0, p1);
              const uint64_t p2 = f2_pack(ex2(p0), ex2(p1));
              l2 = f2_add(l2, p2);
              f2_unpack(f2_mul(p2, f2_pack(nv[j][i], nv[j][i])), p0, p1);
              v0 = kEdge && v0 == -INFINITY ? 0.0f : p0;  // a key that a row does not see adds nothing
              v1 = kEdge && v1 == -INFINITY ? 0.0f : p1;
              most[b][0] = fmaxf(most[b][0], v0);
              most[b][1] = fmaxf(most[b][1], v1);
            }
          f2_unpack(l2, l[b][0], l[b][1]);
          other = other || (int)(__float_as_uint(most[b][0]) >> 23) > pe[b][0] + 1 ||
                  (int)(__float_as_uint(most[b][1]) >> 23) > pe[b][1] + 1;
        }
        if (__any_sync(0xffffffffu, other)) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int c = 0; c < kPer; ++c) {
              float v = most[b][c];
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
              const bool none = drop[b][c] == -INFINITY;
              const int e = max(none ? 20 : max(20, pe[b][c] + (int)ceilf(fmaxf(drop[b][c], -300.0f))),
                                (int)(__float_as_uint(v) >> 23));
              const float fit = none ? 0.0f : ex2(drop[b][c] + (float)(pe[b][c] - e));
              pe[b][c] = e;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                acc[k][b][c] *= fit;
                acc[k][b][c + 2] *= fit;
              }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < kPer; ++c) up[b][c] = __int_as_float((267 - pe[b][c]) << 23);
      }
      const float vs = __int_as_float((259 - ve) << 23);  // 2^(132 - ve): norms below 2^6, P n_v below 2^14

#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t blk = stage + j * kBlockBytes + kVCodes + g * 4;
        uint32_t pf[NB][F32 ? 4 : 2];
        const uint64_t n0 = f2_pack(nv[j][0] * vs, nv[j][0] * vs), n1 = f2_pack(nv[j][1] * vs, nv[j][1] * vs);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float p[4];
          if (F32) {
            const uint64_t u2 = f2_pack(up[b][0], up[b][1]);
            f2_unpack(f2_mul(f2_pack(x[j][b][0], x[j][b][1]), u2), p[0], p[1]);
            f2_unpack(f2_mul(f2_pack(x[j][b][2], x[j][b][3]), u2), p[2], p[3]);
          } else if (kPaired) {  // the odd columns' stay zero
            p[1] = p[3] = 0.0f;
            f2_unpack(f2_fma(f2_pack(x[j][b][0], x[j][b][2]), f2_pack(rs[b][0], rs[b][0]), f2_pack(neg[b][0], neg[b][0])), p[0], p[2]);
            p[0] = ex2(p[0]);
            p[2] = ex2(p[2]);
            l[b][0] += p[0] + p[2];
          } else {
            const uint64_t r2 = f2_pack(rs[b][0], rs[b][1]), g2 = f2_pack(neg[b][0], neg[b][1]);
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              f2_unpack(f2_fma(f2_pack(x[j][b][c], x[j][b][c + 1]), r2, g2), p[c], p[c + 1]);
              p[c] = ex2(p[c]);
              p[c + 1] = ex2(p[c + 1]);
            }
            f2_unpack(f2_add(f2_add(f2_pack(l[b][0], l[b][1]), f2_pack(p[0], p[1])), f2_pack(p[2], p[3])), l[b][0], l[b][1]);
          }
          if (F32) {
          } else if (kEdge) {  // a key that a row does not see adds nothing, whatever its norm
#pragma unroll
            for (int c = 0; c < 4; c += 3 - kPer) p[c] = x[j][b][c] == -INFINITY ? 0.0f : p[c] * (c < 2 ? nv[j][0] : nv[j][1]) * vs;
          } else if (kPaired) {
            p[0] *= nv[j][0] * vs;
            p[2] *= nv[j][1] * vs;
          } else {
            f2_unpack(f2_mul(f2_pack(p[0], p[1]), n0), p[0], p[1]);
            f2_unpack(f2_mul(f2_pack(p[2], p[3]), n1), p[2], p[3]);
          }
          const uint32_t h0 = pack_half(p[0], p[1]), h1 = pack_half(p[2], p[3]);
          pf[b][0] = transpose8(h0);
          pf[b][1] = transpose8(h1);
          if (F32) {
            const float2 f0 = unpack_half(h0), f1 = unpack_half(h1);
            pf[b][F32 ? 2 : 0] = transpose8(pack_half(p[0] - f0.x, p[1] - f0.y));
            pf[b][F32 ? 3 : 1] = transpose8(pack_half(p[2] - f1.x, p[3] - f1.y));
          }
        }
        uint32_t u0, v0, u1, v1;  // even and odd coordinates of tokens t, t + 4 and t + 8, t + 12
        zip(lds32(blk + t * 32), lds32(blk + (t + 4) * 32), u0, v0);
        zip(lds32(blk + (t + 8) * 32), lds32(blk + (t + 12) * 32), u1, v1);
        uint32_t d[4][4], r[4][4];
        look(u0, d[0], r[0]);
        look(v0, d[1], r[1]);
        look(u1, d[2], r[2]);
        look(v1, d[3], r[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t f[4] = {d[0][k], d[1][k], d[2][k], d[3][k]};
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            if (F32) {
              const uint32_t e[4] = {r[0][k], r[1][k], r[2][k], r[3][k]};
              mma(acc[k][b], e, pf[b][0], pf[b][1]);
              mma(acc[k][b], f, pf[b][F32 ? 2 : 0], pf[b][F32 ? 3 : 1]);
            }
            mma(acc[k][b], f, pf[b][0], pf[b][1]);
          }
        }
      }
    };

    for (int i = 0; i < mine; ++i, ++n) {
      const int key0 = c0 + (warp + kWarps * i) * kStageKeys;
      const uint32_t stage = smem_u32(sm.ring[warp][n & 1u]);
      // the lanes leave together: one may see the block's abort flag where another saw its stage
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.full[warp][n & 1u]), (n >> 1) & 1u, &all.abort_flag, a.wait_err))) {
        broken = true;
        break;
      }
      uint32_t nb[4][2];  // norms of this lane's keys: K low, V high
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) nb[j][c] = lds32(stage + j * kBlockBytes + kNorms + (krow + 8 * c) * 4);
      if (key0 + kStageKeys > min(clear, c1)) attend_stage(std::true_type{}, stage, key0, nb);
      else attend_stage(std::false_type{}, stage, key0, nb);
      __syncwarp();  // the stage is in registers
      if (ahead < mine) issue(u, ahead, n + 2u), ++ahead;
    }

    // the next unit's first stage sets out before this one is joined
    ahead = 0;
    more = next(coming);
    if (sums_in_a_slot<R>() && more && !broken && coming.stages > 0) issue(coming, 0, n), ahead = 1;
    float* mine_sums = reinterpret_cast<float*>(sm.ring[warp][sums_in_a_slot<R>() ? (n + 1u) & 1u : 0]);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < kPer; ++c) {
        const float down = __int_as_float((F32 ? pe[b][c] - 19 : ve - 11) << 23);  // 2^(ve - 132) / 64, 2^(pe - 140) / 64
        float v = l[b][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        const int r = 8 * b + kPer * t + c;
        if (g == 0) {
          sm.m[warp][r] = m[b][c] * rs[b][c];
          sm.l[warp][r] = v;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<float2*>(mine_sums + r * kOPitch + 8 * g + 2 * k) =
              make_float2(acc[k][b][c] * down, acc[k][b][c + 2] * down);
      }
    if (lane == 0) sm.sums[warp] = mine_sums;
    if (!meet(!broken)) break;
    for (int r = warp; r < kRows && s.row0 + r < s.rows; r += kWarps) {
      float top = sm.m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][r]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sm.m[w][r] - base);
        sum += sm.l[w][r] * f;
        o0 += sm.sums[w][r * kOPitch + lane] * f;
        o1 += sm.sums[w][r * kOPitch + lane + 32] * f;
      }
      if (u.whole) {
        finish_row<T>(a, all.turns, s, u.head, s.row0 + r, o0, o1, top, sum, lane);
      } else {
        const long long at = u.piece * kRows + r;
        if (at >= a.parts) {  // sequences that overlap have more units than rows make
          if (lane == 0) atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
          continue;
        }
        a.part[at * 64 + lane] = o0;
        a.part[at * 64 + lane + 32] = o1;
        if (lane == 0) a.part_ml[at] = make_float2(top, sum);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the sums' places go back to the copies
    meet(true);
  }
  if (broken || all.abort_flag) {  // a wait ran out: nothing may still be landing when the block ends
    const unsigned long long t0 = globaltimer_ns();
    for (uint32_t i = n; i < n + 2u; ++i)
      while (!mbar_try(smem_u32(&sm.full[warp][i & 1u]), (i >> 1) & 1u) && globaltimer_ns() - t0 < kWaitLimitNs) {
      }
  }
}

// Joins the chunks (tcgen05) or pieces of the rows that have more than one:
// kRowWarps warps a row, each a share of them.
template <typename T, int kRowWarps, bool kPieces>
__global__ void __launch_bounds__(128)
join_kernel(const __grid_constant__ Args a) {
  __shared__ Turns turns;
  __shared__ float share[4][66];
  pdl_launch_dependents();
  load_turns(turns, a, threadIdx.x);
  __syncthreads();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kRowWarps;
  const long long w = (long long)blockIdx.x * (4 / kRowWarps) + warp / kRowWarps;
  const int rows = a.total_q * a.group;
  const int head = (int)(w / rows), call_row = (int)(w % rows), tok = call_row / a.group;
  if (head >= a.pool.heads) return;
  int seq = 0;  // the last sequence that starts at or before the row's token
  if (a.cu == nullptr) {
    seq = tok / a.max_q;
  } else {
    for (int i = lane; i - lane < a.num_seqs; i += 32)
      seq += __popc(__ballot_sync(0xffffffffu, i < a.num_seqs && a.cu[i] <= tok));
    --seq;
  }
  if (seq < 0) return;
  const int q0 = a.cu == nullptr ? seq * a.max_q : a.cu[seq];
  const int row = (tok - q0) * a.group + call_row % a.group;
  const Span s = span_of(a, seq, row / a.tile_rows, false);
  if (row < 0 || row >= s.rows) return;
  int chunks = chunks_of(a, s);
  long long first = part_at(a, s, head, 0, row), step = (long long)a.pool.heads * rows;
  if (kPieces) {
    long long cost = 0, units = 0, total = 0;  // up to the sequence; of all
    for (int i = lane; i < a.num_seqs; i += 32) {
      const SeqCost c = cost_of(a, i);
      total += c.cost;
      if (i < seq) cost += c.cost, units += c.units;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      cost += __shfl_xor_sync(0xffffffffu, cost, o);
      units += __shfl_xor_sync(0xffffffffu, units, o);
    }
    const SeqCost c = cost_of(a, seq);
    const long long k = (long long)head * c.tiles + row / a.tile_rows, at = cost + k * (c.rounds + 1);
    const int t0 = team_of(total, at, a.teams);
    chunks = team_of(total, at + c.rounds - 1, a.teams) - t0 + 1;
    first = (units + k + t0) * a.tile_rows + row % a.tile_rows;
    step = a.tile_rows;
    if (first + (chunks - 1) * step >= a.parts) return;  // as where they are written
  }
  if (chunks <= 1) return;
  float top = -INFINITY;
  for (int c = lane; c < chunks; c += 32) top = fmaxf(top, a.part_ml[first + c * step].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
#pragma unroll 8
  for (int c = part; c < chunks; c += kRowWarps) {
    const float2 ml = a.part_ml[first + c * step];
    const float2 o = *reinterpret_cast<const float2*>(a.part + (first + c * step) * 64 + 2 * lane);
    const float f = ex2(ml.x - base);
    sum += ml.y * f;
    o0 += o.x * f;
    o1 += o.y * f;
  }
  // through shared memory: coordinates 2 lane, 2 lane + 1 to lane, lane + 32
  share[warp][2 * lane] = o0;
  share[warp][2 * lane + 1] = o1;
  if (lane == 0) share[warp][64] = sum;
  if (kRowWarps > 1) __syncthreads();  // a block has one row then
  else __syncwarp();
  if (part != 0) return;
  o0 = o1 = sum = 0.0f;
#pragma unroll
  for (int p = 0; p < kRowWarps; ++p) {
    o0 += share[warp + p][lane];
    o1 += share[warp + p][lane + 32];
    sum += share[warp + p][64];
  }
  finish_row<T>(a, turns, s, head, row, o0, o1, top, sum, lane);
}

struct Plan {
  bool tc;  // attn_kv4_tc.cu's kernel
  bool joined;
  int row_tiles, tile_rows;
  int chunk, splits;               // tcgen05
  int round_keys, blocks, teams;   // else
  long long tiles;
  size_t part_bytes, ml_bytes, q_bytes, scale_bytes;
  size_t bytes() const { return part_bytes + ml_bytes + q_bytes + scale_bytes; }
};

int plan(const Pool& pool, int dtype, int q_heads, int num_seqs, int total_q, int max_q, int max_len, Plan& p) {
  CC2_REQUIRE(dtype == CC2_BF16 || dtype == CC2_F32, "kv4_attention: unsupported dtype %d", dtype);
  CC2_REQUIRE(q_heads > 0 && q_heads % pool.heads == 0,
              "kv4_attention: %d query heads are no multiple of the cache's %d", q_heads, pool.heads);
  CC2_REQUIRE(num_seqs > 0 && total_q >= 0 && max_q >= 0 && max_len >= 0, "kv4_attention: negative sizes or no sequence");
  CC2_REQUIRE(max_len <= 1 << 30, "kv4_attention: max_len %d is above 2^30", max_len);
  CC2_REQUIRE(std::max(max_q, total_q) <= 0x7fffffff / 64 / q_heads, "kv4_attention: %d query rows are too many",
              std::max(max_q, total_q));
  const int rows = std::max(1, max_q * (q_heads / pool.heads));
  p = Plan{};
  p.tc = for_tcgen05(dtype, rows, max_len);
  // As few columns as hold the rows: with 16 sequences of 8192 tokens and 8 heads, one / two / four blocks of 8 take
  // 35 / 43 / 61 us for 4 rows, 56 / 47 / 66 for 12, 92 / 72 / 73 for 32 (there four spare half the passes over the
  // keys' bytes); a block with 4 rows in column pairs and one with 8 35 / 39.  fp32 splits need the registers of four.
  p.tile_rows = p.tc ? kTcRows : dtype == CC2_F32 ? (rows <= 8 ? 8 : 16) : rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const long long tiles = (long long)num_seqs * pool.heads * p.row_tiles;
  if (p.tc) {
    // Blocks take items as they get to them: about four an SM even them out; a chunk's own cost is some 1000 keys.
    // One / two / four / eight an SM: 168 / 123 / 113 / 119 us for 64 tokens of 2 sequences of 65536, 8 heads;
    // 229 / 185 / 172 / 186 us for 256 tokens of 4 of 32768; 299 / 305 / 310 / 311 us where there are items enough.
    const long long want = (4LL * num_sms() + tiles - 1) / tiles;
    const int splits = (int)std::min<long long>(std::max(1, (max_len + 1023) / 1024), std::max<long long>(1, want));
    p.chunk = ((std::max(1, max_len) + splits - 1) / splits + 255) / 256 * 256;
    p.splits = std::max(1, (max_len + p.chunk - 1) / p.chunk);
    CC2_REQUIRE(tiles * p.splits <= 0x7f000000LL, "kv4_attention: too many rows and keys for one call");
    const size_t n = p.splits > 1 ? (size_t)p.splits * total_q * q_heads : 0;
    p.part_bytes = n * 64 * sizeof(float);
    p.ml_bytes = align_up(n * sizeof(float2), 128);
    p.tiles = query_tiles((long long)total_q * (q_heads / pool.heads), num_seqs) * pool.heads;
    p.q_bytes = (size_t)p.tiles * 128 * 128;
    p.scale_bytes = (size_t)p.tiles * 128 * sizeof(float) + 128;  // and the items' counter
  } else {
    const bool f32 = dtype == CC2_F32;
    const int warps = p.tile_rows <= 8 && !f32 ? warps_of<4, false>() : 4, a_block = p.tile_rows == 16 && !f32 ? teams_of<16, false>() : 2;
    static_assert(warps_of<8, false>() == warps_of<4, false>() && warps_of<16, false>() == 4 && warps_of<32, false>() == 4 &&
                      warps_of<8, true>() == 4 && warps_of<16, true>() == 4 && teams_of<4, false>() == 2 &&
                      teams_of<8, false>() == 2 && teams_of<32, false>() == 2 && teams_of<8, true>() == 2 &&
                      teams_of<16, true>() == 2,
                  "as assumed above");
    p.round_keys = warps * kStageKeys;
    // no more blocks than there are rounds
    const long long rounds = (long long)num_seqs * pool.heads * p.row_tiles * std::max(1, (max_len + p.round_keys - 1) / p.round_keys);
    p.blocks = (int)std::min<long long>((rounds + a_block - 1) / a_block, num_sms());
    p.teams = p.blocks * a_block;
    p.joined = max_len > p.round_keys;
    if (p.joined) {
      const long long units = ((long long)total_q * (q_heads / pool.heads) / p.tile_rows + num_seqs) * pool.heads;
      const size_t n = (size_t)(units + p.teams) * p.tile_rows;
      p.part_bytes = n * 64 * sizeof(float);
      p.ml_bytes = align_up(n * sizeof(float2), 128);
    }
  }
  p.joined = p.tc ? p.splits > 1 : p.joined;
  return CC2_OK;
}

template <int R, bool F32, bool NormBf16>
int launch(const Args& a, const Plan& p, cudaStream_t st) {
  const size_t smem = sizeof(Shared<R, F32>);
  static unsigned long long attr_done = 0;  // one bit per device
  int dev = 0;
  CC2_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !((attr_done >> dev) & 1ull)) {
    CC2_CUDA(cudaFuncSetAttribute(attend_kernel<R, F32, NormBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev < 64) attr_done |= 1ull << dev;
  }
  CC2_CUDA(launch_k(attend_kernel<R, F32, NormBf16>, (unsigned)p.blocks, 32 * teams_of<R, F32>() * warps_of<R, F32>(),
                    smem, st, a));
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}
template <int R, bool F32>
int launch(const Args& a, const Plan& p, cudaStream_t st) {
  return a.pool.norm_bf16 ? launch<R, F32, true>(a, p, st) : launch<R, F32, false>(a, p, st);
}

template <typename T>
int join(const Args& a, const Plan& p, cudaStream_t st) {
  if (!p.joined) return CC2_OK;
  const long long rows = (long long)a.total_q * a.group * a.pool.heads;
  // Where there are fewer rows than warps on the card, four share one: a row then has many parts.  Whole calls with
  // four / one a row: 35.0 / 37.1 us with 128 rows, 113 / 121 us with 1024 in 8 chunks, 51 / 49 us with 2048,
  // 51 / 43 us with 4096, 178 / 145 us with 16384.
  const bool four = rows <= 16LL * num_sms();
  const unsigned grid = (unsigned)(four ? rows : (rows + 3) / 4);
  if (p.tc) {
    if (four) CC2_CUDA(launch_k(join_kernel<T, 4, false>, grid, 128, 0, st, a));
    else CC2_CUDA(launch_k(join_kernel<T, 1, false>, grid, 128, 0, st, a));
  } else {
    if (four) CC2_CUDA(launch_k(join_kernel<T, 4, true>, grid, 128, 0, st, a));
    else CC2_CUDA(launch_k(join_kernel<T, 1, true>, grid, 128, 0, st, a));
  }
  CC2_CHECK_LAUNCH();
  return CC2_OK;
}

}  // namespace
}  // namespace kv4

int kv4_attention_workspace(const cc2_kv4_cache* cache, int dtype, int q_heads, int num_seqs, int total_q, int max_q,
                            int max_len, size_t* bytes) {
  kv4::Pool pool;
  CC2_TRY(kv4::check_cache(cache, "kv4_attention", pool));
  CC2_REQUIRE(bytes != nullptr, "kv4_attention: bytes is null");
  kv4::Plan p;
  CC2_TRY(kv4::plan(pool, dtype, q_heads, num_seqs, total_q, max_q, max_len, p));
  *bytes = p.bytes();
  return CC2_OK;
}

int launch_kv4_attention(const cc2_kv4_cache* cache, int dtype, const void* q, int64_t q_ld, int64_t q_hs, void* out,
                         int64_t o_ld, int64_t o_hs, int q_heads, int num_seqs, int total_q, const int32_t* cu_q,
                         int max_q, const int32_t* seq_lens, int max_len, const int32_t* table, int table_ld,
                         int causal, float scale, int rotate_q, int fill, float* lse, void* ws, size_t ws_bytes,
                         cudaStream_t st) {
  using namespace kv4;
  Args a{};
  CC2_TRY(check_cache(cache, "kv4_attention", a.pool));
  Plan p;
  CC2_TRY(plan(a.pool, dtype, q_heads, num_seqs, total_q, max_q, max_len, p));
  CC2_REQUIRE((fill & ~3) == 0, "kv4_attention: bad fill %d", fill);
  if (cu_q == nullptr) fill = 0;  // every row has a sequence
  if (lse == nullptr) fill &= 1;
  if (total_q == 0 || (max_q == 0 && fill == 0)) return CC2_OK;
  CC2_REQUIRE(q && out && seq_lens && table && table_ld > 0, "kv4_attention: null operand");
  CC2_REQUIRE(cu_q != nullptr || (long long)num_seqs * max_q == total_q,
              "kv4_attention: without cu_q the rows must be num_seqs * max_q, got %d", total_q);
  CC2_REQUIRE(rows_ok(dtype, q, q_ld, q_hs) && rows_ok(dtype, out, o_ld, o_hs),
              "kv4_attention: rows must start on 16 bytes, as must their strides");
  CC2_REQUIRE(!rotate_q || cache->rope_cs, "kv4_attention: the cache has no table to rotate queries with");
  CC2_REQUIRE(std::isfinite(scale), "kv4_attention: scale must be finite");
  if (ws_bytes < p.bytes() || (p.bytes() > 0 && (ws == nullptr || ((uintptr_t)ws & 15u) != 0))) {
    set_error("kv4_attention: workspace of %zu bytes (16-byte aligned) needed, got %zu", p.bytes(), ws_bytes);
    return CC2_E_WORKSPACE;
  }
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.q_ld = q_ld;
  a.q_hs = q_hs;
  a.o_ld = o_ld;
  a.o_hs = o_hs;
  a.cu = cu_q;
  a.lens = seq_lens;
  a.table = table;
  a.rope = (const float2*)cache->rope_cs;
  a.qt = (uint8_t*)ws;
  a.part = (float*)(a.qt + p.q_bytes);
  a.part_ml = (float2*)((char*)a.part + p.part_bytes);
  a.counter = (int*)((char*)a.part_ml + p.ml_bytes);
  a.q_scale = (float*)((char*)a.counter + 128);
  CC2_TRY(error_words(&a.range_err));
  a.wait_err = a.range_err + 1;
  a.table_ld = table_ld;
  a.rope_len = cache->rope_len;
  a.max_len = max_len;
  a.num_seqs = num_seqs;
  a.total_q = total_q;
  a.max_q = max_q;
  a.group = q_heads / a.pool.heads;
  a.chunk = p.chunk;
  a.splits = p.splits;
  a.row_tiles = p.row_tiles;
  a.tile_rows = p.tile_rows;
  a.teams = p.teams;
  a.parts = (long long)(p.part_bytes / (64 * sizeof(float)));
  a.round_keys = p.round_keys;
  a.causal = causal != 0;
  a.rotate = rotate_q != 0;
  a.fill = fill;
  const cc2_kv4_quant* quant[2] = {&cache->key, &cache->value};
  Rotation* rotation[2] = {&a.rk, &a.rv};
  for (int k = 0; k < 2; ++k) {
    Rotation& r = *rotation[k];
    r.signs[0] = (uint32_t)quant[k]->signs;
    r.signs[1] = (uint32_t)(quant[k]->signs >> 32);
    for (int i = 0; i < 64; ++i) r.inv[r.perm[i] = quant[k]->perm[i] & 63] = (uint8_t)i;
  }
  a.levels = make_levels(*cache);
  a.back = 8.0f / a.levels.scale;
  a.qscale = scale * 1.4426950408889634f * a.back;
  if (p.tc) CC2_TRY(launch_attend_tc(a, st));
  else if (dtype == CC2_F32) CC2_TRY(p.tile_rows == 8 ? (launch<8, true>(a, p, st)) : (launch<16, true>(a, p, st)));
  else if (p.tile_rows <= 8) CC2_TRY(p.tile_rows == 4 ? (launch<4, false>(a, p, st)) : (launch<8, false>(a, p, st)));
  else CC2_TRY(p.tile_rows == 16 ? (launch<16, false>(a, p, st)) : (launch<32, false>(a, p, st)));
  return dtype == CC2_F32 ? join<float>(a, p, st) : join<__nv_bfloat16>(a, p, st);
}

}  // namespace cc2
