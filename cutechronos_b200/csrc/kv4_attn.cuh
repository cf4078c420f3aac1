// Shared by the kernels of attention over the 4-bit cache: their arguments,
// what rows and keys a block has, the rotation of a row spread over a warp.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kv4.cuh"
#include "tc_attn.cuh"

namespace cc2 {
namespace kv4 {

using tcx::ex2;

struct Rotation {
  uint32_t signs[2];
  alignas(4) uint8_t perm[64];  // coordinate perm[i] of a vector is i of the rotated one
  alignas(4) uint8_t inv[64];
};

// Keys' permutation going in and values' coming out, in shared memory: lanes
// that index the kernel's arguments apart are served one by one.
struct Turns {
  alignas(4) uint8_t k_perm[64];
  alignas(4) uint8_t v_inv[64];
};
template <typename A>
__device__ __forceinline__ void load_turns(Turns& t, const A& a, int tid) {
  if (tid < 16) reinterpret_cast<uint32_t*>(t.k_perm)[tid] = reinterpret_cast<const uint32_t*>(a.rk.perm)[tid];
  else if (tid < 32) reinterpret_cast<uint32_t*>(t.v_inv)[tid - 16] = reinterpret_cast<const uint32_t*>(a.rv.inv)[tid - 16];
}

struct Args {
  Pool pool;
  const void* q;
  void* out;
  float* lse;
  long long q_ld, q_hs, o_ld, o_hs;
  const int* cu;
  const int* lens;
  const int* table;
  const float2* rope;
  float* part;       // tcgen05: [split][head][row of the call][64], else [piece][row][64]: a part's sums, rotated
  float2* part_ml;   // the same places: maximum (log2) and sum of exponentials
  long long parts;   // else: the places there are
  const uint8_t* qt;  // rotated queries as fp16 tiles (attn_kv4_tc.cu) and their rows' scales
  const float* q_scale;
  int* counter;       // items that the tcgen05 kernel's blocks have taken
  int* wait_err;
  int* range_err;
  int table_ld, rope_len, max_len;
  int num_seqs, total_q, max_q, group;
  int chunk, splits, row_tiles, tile_rows;
  int teams, round_keys;  // else: teams of warps on the card, keys that one takes in a round of its warps
  int causal, rotate;
  int fill;      // rows of no sequence: 1 in out, 2 in lse
  float qscale;  // scale * log2(e) / 8 * 64 / f: of a rotated query (f: the levels' factor)
  float back;    // 64 / f / 8: of a rotated sum
  Rotation rk, rv;
  Levels levels;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"((uint64_t)__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// A vector spread over a warp, coordinates lane and lane + 32.
__device__ __forceinline__ float spread_get(float lo, float hi, int i) {
  const float a = __shfl_sync(0xffffffffu, lo, i & 31), b = __shfl_sync(0xffffffffu, hi, i & 31);
  return i < 32 ? a : b;
}
__device__ __forceinline__ void spread_walsh(float& lo, float& hi, int lane) {
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, lo, w), b = __shfl_xor_sync(0xffffffffu, hi, w);
    lo = (lane & w) ? a - lo : lo + a;
    hi = (lane & w) ? b - hi : hi + b;
  }
  const float a = lo;
  lo = a + hi;
  hi = a - hi;
}
__device__ __forceinline__ float flip(float x, const uint32_t signs[2], int half, int lane) {
  return (signs[half] >> lane) & 1u ? -x : x;
}

// What a block or a row tile works on.
struct Span {
  int row0, rows;      // first row of the tile, rows of the sequence
  int q_start, n;      // first query token, query tokens
  int len;             // cached tokens
  int keys;            // the tile's rows see none from here on
};

__device__ __forceinline__ Span span_of(const Args& a, int seq, int row_tile, bool report) {
  Span s;
  int q0 = seq * a.max_q, q1 = q0 + a.max_q;
  if (a.cu != nullptr) {
    q0 = a.cu[seq];
    q1 = a.cu[seq + 1];
  }
  const int len = a.lens[seq];
  const long long room = (long long)a.table_ld << a.pool.page_shift;
  const int most = (int)min((long long)a.max_len, room);
  const bool bad = q0 < 0 || q1 < q0 || q1 > a.total_q || q1 - q0 > a.max_q || len < 0 || len > most;
  if (bad && report) atomicOr(a.range_err, (int)DEV_ERR_CACHE_RANGE);
  s.q_start = min(max(q0, 0), a.total_q);
  s.n = min(min(max(q1, s.q_start), a.total_q) - s.q_start, a.max_q);
  s.len = min(max(len, 0), most);
  s.row0 = row_tile * a.tile_rows;
  s.rows = s.n * a.group;
  const int last = (min(s.row0 + a.tile_rows, s.rows) - 1) / a.group;  // the tile's last query token
  s.keys = a.causal ? min(max(s.len - s.n + last + 1, 0), s.len) : s.len;
  return s;
}

// Rows that no sequence has, before the first one's and from the end of the
// last one's on: 0, and -inf as log-sum-exp.  Thread `id` of `threads`; a call's
// rows times heads times 64 fit 31 bits.
template <typename T>
__device__ __forceinline__ void fill_rows(const Args& a, unsigned id, unsigned threads) {
  constexpr unsigned kParts = 64 * sizeof(T) / 16;
  const unsigned head = min(max(a.cu[0], 0), a.total_q), tail = min(max(a.cu[a.num_seqs], (int)head), a.total_q);
  const unsigned heads = a.pool.heads * a.group, parts = (head + a.total_q - tail) * heads * kParts;
  for (unsigned i = id; i < parts; i += threads) {
    const unsigned row = i / kParts, at = row / heads, tok = at < head ? at : at - head + tail, h = row - at * heads;
    if (a.fill & 1)
      reinterpret_cast<uint4*>((T*)a.out + (long long)tok * a.o_ld + (long long)h * a.o_hs)[i % kParts] = make_uint4(0, 0, 0, 0);
    if ((a.fill & 2) && i % kParts == 0) a.lse[(long long)tok * heads + h] = -INFINITY;
  }
}

// The work of a call without tcgen05, as one line of rounds: sequence after
// sequence, head after head, row tile after row tile, each of as many rounds of
// a team's warps as its keys take (one at least) and one more for what a unit
// costs by itself.  Team t of N gets the rounds from floor(t W / N) on, so all
// take the same time whatever the sequences' lengths; a unit that crosses a
// border is joined from its pieces.  Pieces are numbered unit + team, which
// grows along the line.
struct SeqCost {
  int tiles;       // of a head's rows
  int rounds;      // of a unit's keys
  long long units, cost;
};
__device__ __forceinline__ SeqCost cost_of(const Args& a, int seq, bool report = false) {
  const Span s = span_of(a, seq, 0, report);
  SeqCost c;
  c.tiles = (s.rows + a.tile_rows - 1) / a.tile_rows;
  c.rounds = max((s.len + a.round_keys - 1) / a.round_keys, 1);
  c.units = (long long)c.tiles * a.pool.heads;
  c.cost = c.units * (c.rounds + 1);
  return c;
}
// No more teams than rounds take part: none of them is without one.
__device__ __forceinline__ long long team_start(long long total, int team, int teams) {
  teams = (int)min((long long)teams, max(total, 1LL));
  return total * min(team, teams) / teams;
}
__device__ __forceinline__ int team_of(long long total, long long round, int teams) {
  return (int)(((round + 1) * min((long long)teams, total) - 1) / total);
}

// Place of a row's sums among the parts.
__device__ __forceinline__ long long part_at(const Args& a, const Span& s, int head, int split, int row) {
  return ((long long)split * a.pool.heads + head) * ((long long)a.total_q * a.group) +
         (long long)s.q_start * a.group + row;
}

// Number of chunks that hold keys of the tile.
__device__ __forceinline__ int chunks_of(const Args& a, const Span& s) { return (s.keys + a.chunk - 1) / a.chunk; }

// One row's sums -> output and log-sum-exp: lane holds coordinates lane and lane + 32 of the rotated sum.
template <typename T>
__device__ __forceinline__ void finish_row(const Args& a, const Turns& turns, const Span& s, int head, int row, float o0, float o1, float m,
                                           float l, int lane) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  spread_walsh(o0, o1, lane);
  o0 = flip(o0 * (a.back * inv), a.rv.signs, 0, lane);
  o1 = flip(o1 * (a.back * inv), a.rv.signs, 1, lane);
  const float x0 = spread_get(o0, o1, turns.v_inv[lane]);
  const float x1 = spread_get(o0, o1, turns.v_inv[lane + 32]);
  const int tok = s.q_start + row / a.group, qh = head * a.group + row % a.group;
  T* out = (T*)a.out + (long long)tok * a.o_ld + (long long)qh * a.o_hs;
  out[lane] = fromf<T>(x0);
  out[lane + 32] = fromf<T>(x1);
  if (a.lse != nullptr && lane == 0)
    a.lse[(long long)tok * (a.pool.heads * a.group) + qh] =
        l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}


// attn_kv4_tc.cu: tiles of 256 rows on tcgen05 (bf16 calls).  Rotated queries in the workspace: tiles of 128 rows for
// each head, sequence s from tile floor(q_start * group / 128) + s on.
constexpr int kTcRows = 256;
__host__ __device__ inline long long query_tiles(long long total_rows, int num_seqs) {
  return total_rows / 128 + num_seqs;
}
__device__ __forceinline__ long long first_query_tile(const Args& a, int seq, int q_start) {
  return (long long)q_start * a.group / 128 + seq;
}
int launch_attend_tc(const Args& a, cudaStream_t st);

}  // namespace kv4
}  // namespace cc2
