// Causal attention of a step's new tokens over a paged bf16 / fp16 layer, and of whole prompts
// over their own packed K and V rows, gfx950.
//
// For row i of request r (n new tokens, context c): o = sum_t p_t v_t / sum_t p_t over the tokens
// t = 0 .. c - n + i, p_t = 2^(s_t - m), s_t = scale * log2(e) * q.k_t, m a running reference
// that never exceeds the running maximum of s and is at most kSlack below it, so that the sums
// stay in range and the accumulators are rescaled only when the maximum has moved by more.
// Scores, weights' sums and outputs accumulate in f32; the weights are rounded to the inputs'
// type for the second matrix product (2^-9 or 2^-12 of each, like the output's own rounding).
//
// The query heads of a group read the same K and V, so a request's rows are (token, head of the
// group) pairs, row m = token * group + head, and a tile of rows serves them together: a single
// token is `group` rows, and every K and V byte is read once per tile.
//
// Two kernels share the rows of a launch by one rule, on the GPU, where the lengths are:
//   * attention_few: requests of at most 16 rows (a decode step, a few drafted tokens). Bound by
//     reading K and V: a wave streams 32 tokens at a time, K straight into the matrix operand's
//     registers, V into LDS for the transposing reads.
//   * attention_tiles: 128 rows by 64 tokens a step. Bound by the matrix and vector units.
// Both give S^T = K Q^T, so that a row's scores lie in one lane (and its partners 32 or 16 lanes
// away): the maximum and the sum need one or two lane swaps a step, rescaling is a lane's own
// product, and the weights are the second product's operand O^T = V^T P^T as they are, with V's
// tokens taken in the order in which the lanes hold them.
//
// Work split: a request's context is cut into splits of equal length where there are too few
// tiles for the chip; the length comes from the sums over all requests, which every workgroup
// forms for itself from the lengths (a wave scan), so that nothing is read back to the host and
// a captured call follows new lengths. attention_merge joins the splits.
//
// Values in masked places: scores there are replaced before use. A weight of zero times an
// infinite or NaN V value would still reach the sums of rows that do not see it, so a row whose
// sums are not finite is formed again, token by token and over its own tokens alone (slow_row).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "splitzip_common.h"

namespace unchainkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kT = 256;           // threads of the split kernels
constexpr int kWaves = kT / kWave;
constexpr int kFewRows = 16;      // rows of a request that attention_few takes
constexpr int kFewStep = 32;      // tokens of a wave's step in attention_few
constexpr int kFewRound = kWaves * kFewStep;  // tokens of a workgroup's round: unit of its splits
constexpr int kTileRows = 128;
constexpr int kTileTokens = 64;   // tokens of a step of attention_tiles: unit of its splits
constexpr unsigned int kLeastTileSteps = 4;  // of a split
// A maximum before any token: the lowest float, not -inf, so that rows whose scores are all -inf
// have weights of zero and a sum of zero (whose quotient is NaN, as the formula's).
constexpr float kNoMax = -3.402823466e38f;
constexpr float kSlack = 8.f;     // log2: weights stay below 2^8
constexpr float kLn2 = 0.6931471805599453f;

template <typename E>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<_Float16> {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Two values rounded to E (nearest even), in one dword.
template <typename E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, typename Elem<E>::x2));
}

template <typename E>
__device__ __forceinline__ typename Elem<E>::x8 pack8(const float* p) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack2<E>(p[2 * i], p[2 * i + 1]);
  return __builtin_bit_cast(typename Elem<E>::x8, v);
}

// What attention_merge has to know of a slot that holds the first split of some rows: rows first ..
// first + rows of the request whose rows start at `start`, row m's last token at shift + m / group,
// in the slots slot, slot + kv_heads, ... (`splits` of them). splits == 0: nothing to join.
struct Job {
  unsigned int start, first;
  int shift;
  unsigned short rows, splits;
};
static_assert(sizeof(Job) == 16, "one load");

struct AttendArgs {
  const unsigned char* q;
  unsigned char* out;        // [tokens][q_heads][D]
  float* lse;                // [tokens][q_heads] or null
  const unsigned char* k;    // paged: K plane; else the packed K rows
  const unsigned char* v;
  const int* starts;         // [requests + 1]
  const int* contexts;       // [requests]; null: a request's own rows (prompts)
  const int* tables;         // [requests][table_stride]; null for prompts
  float* partial;            // slots of the tiles, then of the few
  struct Job* jobs;          // one for each slot
  unsigned long long q_row, q_head;  // bytes from token to token, from head to head
  unsigned long long k_row, k_head, v_row, v_head;
  unsigned long long table_stride;
  unsigned int table_width, blocks, block_tokens;
  Divider by_block;
  unsigned int tokens, requests, q_heads, kv_heads, group;
  unsigned int few_rows;      // most rows of a request that goes to the streaming path; 0: none
  unsigned int tiles_too;     // whether tiles are taken (else longer requests are left out)
  unsigned int tile_groups, few_groups;  // workgroups of the two paths
  unsigned int few_target, tile_target;   // workgroups to split for
  unsigned int max_query;     // requests with more new tokens are left out
  unsigned int tile_slots, few_slots;  // partial slots: of the tiles, then of the few
  float scale_log2;
};

// One request as its lengths in device memory say, with lengths that cannot be cut down to
// nothing: rows outside the tensor are nobody's.
struct Request {
  unsigned int start, n, ctx;
  bool bad;  // a context longer than the block table
};

__device__ __forceinline__ Request load_request(const AttendArgs& a, unsigned int r) {
  Request q{0, 0, 0, false};
  if (r >= a.requests) return q;
  const int s0 = a.starts[r], s1 = a.starts[r + 1];
  if (s0 < 0 || s1 < s0 || (unsigned int)s1 > a.tokens) return q;
  q.start = (unsigned int)s0;
  q.n = (unsigned int)(s1 - s0);
  q.ctx = q.n;
  if (a.contexts != nullptr) {
    const unsigned long long most = (unsigned long long)a.table_width * a.block_tokens;
    const int c = a.contexts[r];
    q.ctx = c < 0 ? 0u : (unsigned int)c;
    if (q.ctx > most) {
      q.bad = true;
      q.ctx = (unsigned int)most;
    }
  }
  return q;
}

// Which kernel takes a request: 0 none, 1 attention_few, 2 attention_tiles.
__device__ __forceinline__ int kind_of(const AttendArgs& a, const Request& q) {
  if (q.n == 0 || q.n > a.max_query) return 0;
  const unsigned long long rows = (unsigned long long)q.n * a.group;
  if (rows <= a.few_rows) return 1;
  return a.tiles_too ? 2 : 0;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d, kWave);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v = fmaxf(v, __shfl_xor(v, d, kWave));
  return v;
}

// Inclusive sum over the wave's lanes, on the VALU: shifts by 1, 2, 4, 8 within each row of 16
// lanes, then the rows' ends into the rows behind them.
__device__ __forceinline__ unsigned int wave_scan(unsigned int v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
  return v;
}
__device__ __forceinline__ unsigned int lane_value(unsigned int v, int lane) {
  return (unsigned int)__builtin_amdgcn_readlane((int)v, lane);
}

__device__ __forceinline__ unsigned int steps_of(unsigned int tokens, unsigned int step) {
  return tokens / step + (tokens % step != 0 ? 1u : 0u);
}

__device__ __forceinline__ unsigned int tiles_of(const AttendArgs& a, unsigned int n) {
  return (n * a.group + kTileRows - 1) / kTileRows;
}

// Steps of a split on the streaming path and of a tile's, from the sums over all requests (each
// lane a request, 64 at a time; `head` holds the first 64, which most launches end with). Few:
// the even share of all rounds over few_target workgroups. Tiles: no split (0) once there are
// tile_target tiles, else the even share of all tiles' steps, a tile of a request counted with
// the request's mean context (a request's sum beyond kMostSteps, which the 32-bit sums do not
// take, is not split either).
struct SplitSteps {
  unsigned int few, tiles;
};
constexpr unsigned int kMostSteps = 1u << 25;

// ceil(sum / parts), by a 32-bit division where it serves.
__device__ __forceinline__ unsigned int share_of(unsigned long long sum, unsigned int parts) {
  sum += parts - 1;
  return (sum >> 32) == 0 ? (unsigned int)sum / parts : (unsigned int)(sum / parts);
}

__device__ __forceinline__ SplitSteps split_steps(const AttendArgs& a, const Request& head) {
  unsigned long long few = 0, tiles = 0, tile_steps = 0;
  bool large = false;
  for (unsigned int r0 = 0; r0 < a.requests; r0 += kWave) {
    const Request q = r0 == 0 ? head : load_request(a, r0 + __lane_id());
    const int kind = kind_of(a, q);
    if (a.few_rows != 0)
      few += lane_value(wave_scan(kind == 1 ? steps_of(q.ctx, kFewRound) : 0u), 63);
    if (a.tiles_too != 0) {
      const unsigned int t = kind == 2 ? tiles_of(a, q.n) : 0u;
      const unsigned long long all =
          (unsigned long long)t * steps_of(q.ctx - min(q.ctx, q.n) / 2, kTileTokens);
      large |= __ballot(all > kMostSteps) != 0;
      tiles += lane_value(wave_scan(t), 63);
      tile_steps += lane_value(wave_scan((unsigned int)min(all, (unsigned long long)kMostSteps)), 63);
    }
  }
  few *= a.kv_heads;
  tiles *= a.kv_heads;
  tile_steps *= a.kv_heads;
  SplitSteps s;
  s.few = max(1u, share_of(few, a.few_target));
  s.tiles = tiles >= a.tile_target || large ? 0u
                                            : max(kLeastTileSteps, share_of(tile_steps, a.tile_target));
  return s;
}

__device__ __forceinline__ unsigned int few_splits(unsigned int ctx, unsigned int steps) {
  return max(1u, steps_of(steps_of(ctx, kFewRound), steps));
}
__device__ __forceinline__ unsigned int tile_splits(unsigned int ctx, unsigned int steps) {
  return steps == 0 ? 1u : max(1u, steps_of(steps_of(ctx, kTileTokens), steps));
}

// The request that item `item` belongs to, request r having count(r) of them; false past the
// last one. All wave-uniform.
struct Place {
  Request q;
  unsigned int r, index;  // index within the request
};

template <typename Count>
__device__ __forceinline__ bool find_item(const AttendArgs& a, const Request& head,
                                          unsigned int item, Count count, Place& p) {
  unsigned long long before = 0;
  for (unsigned int r0 = 0; r0 < a.requests; r0 += kWave) {
    const Request q = r0 == 0 ? head : load_request(a, r0 + __lane_id());
    const unsigned int own = count(q), sum = wave_scan(own), all = lane_value(sum, 63);
    if (item < before + all) {
      const unsigned int in = item - (unsigned int)before;
      const int at = __ffsll((long long)__ballot(sum > in)) - 1;
      p.r = r0 + (unsigned int)at;
      p.index = in - lane_value(sum - own, at);
      p.q.start = lane_value(q.start, at);
      p.q.n = lane_value(q.n, at);
      p.q.ctx = lane_value(q.ctx, at);
      p.q.bad = lane_value(q.bad ? 1u : 0u, at) != 0;
      return true;
    }
    before += all;
  }
  return false;
}

// Row of K and V that token t of a request has: its place in the layer through the block table
// (bad: the table names no block of the layer there; block 0 is read instead), or its packed row.
template <bool kPaged>
__device__ __forceinline__ unsigned int kv_row(const AttendArgs& a, const int* table,
                                               unsigned int start, unsigned int t, int id,
                                               bool& bad) {
  if constexpr (kPaged) {
    const unsigned int blk = div_u32(t, a.by_block.m, a.by_block.d);
    const bool ok = (unsigned int)id < a.blocks;
    bad |= !ok;
    return (ok ? (unsigned int)id : 0u) * a.block_tokens + (t - blk * a.block_tokens);
  } else {
    return start + t;
  }
}
template <bool kPaged>
__device__ __forceinline__ int block_id(const AttendArgs& a, const int* table, unsigned int t) {
  if constexpr (kPaged)
    return table[div_u32(t, a.by_block.m, a.by_block.d)];
  else
    return 0;
}

// 16 bytes a lane from global memory straight into LDS: lane l's land at dst + 16 l.
__device__ __forceinline__ void load_to_lds(const unsigned char* src, unsigned char* dst) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) unsigned char*)src,
      (__attribute__((address_space(3))) unsigned char*)dst, 16, 0, 0);
}

// The same from a buffer: lanes whose 16 bytes end past it get zeros.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const unsigned char* base, unsigned int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(base), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void load_to_lds(Buffer b, unsigned int offset, unsigned char* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) unsigned char*)dst, 16,
                                           (int)offset, 0, 0, 0);
}

// Waits until at most N of the wave's loads are in flight.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 0xF70 | (N >> 4) << 14);
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ u32x2 read_transposed(const unsigned char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) i16x4*)p));
}

// One row over tokens [t0, t1), all of which it sees, in f32 and without the matrix units; a
// wave's lanes take a token each for the scores and D / 64 dims each for the output.
template <typename E, int D, bool kPaged>
__device__ __forceinline__ void slow_row(const AttendArgs& a, const int* table, unsigned int start,
                                      const unsigned char* q, unsigned int kv_head, unsigned int t0,
                                      unsigned int t1, float& m, float& l, float (&acc)[D / 64]) {
  typedef typename Elem<E>::x8 x8;
  const unsigned int lane = __lane_id();
  const unsigned char* kb = a.k + kv_head * a.k_head;
  const unsigned char* vb = a.v + kv_head * a.v_head;
  m = kNoMax;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) acc[i] = 0.f;
  for (unsigned int t = t0; t < t1; t += kWave) {
    const unsigned int own = min(t + lane, t1 - 1);
    bool bad = false;
    const unsigned int row = kv_row<kPaged>(a, table, start, own, block_id<kPaged>(a, table, own), bad);
    const unsigned char* k = kb + row * a.k_row;
    float s = 0.f;
    for (int c = 0; c < D / 8; ++c) {
      const x8 x = *reinterpret_cast<const x8*>(q + 16 * c), y = *reinterpret_cast<const x8*>(k + 16 * c);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf((float)x[j], (float)y[j], s);
    }
    s = t + lane < t1 ? s * a.scale_log2 : -INFINITY;
    const float top = fmaxf(m, wave_max(s)), alpha = exp2f(m - top);
    const float p = t + lane < t1 ? exp2f(s - top) : 0.f;
    m = top;
    l = l * alpha + wave_sum(p);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] *= alpha;
    const unsigned int count = min(t1 - t, (unsigned int)kWave);
    for (unsigned int j = 0; j < count; ++j) {
      const float w = __shfl(p, (int)j, kWave);
      const unsigned char* v = vb + uniform(__shfl(row, (int)j, kWave)) * a.v_row;
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
        acc[i] = fmaf(w, (float)reinterpret_cast<const E*>(v)[lane * (D / 64) + i], acc[i]);
    }
  }
}

// Where a row's result goes: the output (of one split), or its place among the partials, a
// slot's rows as (m, l) pairs and then their D sums.
template <int D>
__device__ __forceinline__ float* slot_ml(const AttendArgs& a, bool few, unsigned int slot) {
  constexpr unsigned int kFew = kFewRows * (D + 2), kTile = kTileRows * (D + 2);
  return few ? a.partial + (unsigned long long)a.tile_slots * kTile + (unsigned long long)slot * kFew
             : a.partial + (unsigned long long)slot * kTile;
}
template <int D>
__device__ __forceinline__ float* slot_acc(const AttendArgs& a, bool few, unsigned int slot) {
  return slot_ml<D>(a, few, slot) + 2 * (few ? kFewRows : kTileRows);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// A row (m, l, sums) by a wave whose lanes hold D / 64 sums each, from slow_row.
template <typename E, int D>
__device__ __forceinline__ void store_slow(const AttendArgs& a, bool split, bool few,
                                           unsigned int slot, unsigned int slot_row,
                                           unsigned long long out_row, bool none, float m, float l,
                                           const float (&acc)[D / 64]) {
  const unsigned int lane = __lane_id();
  if (split) {
    float* ml = slot_ml<D>(a, few, slot) + 2 * slot_row;
    float* dst = slot_acc<D>(a, few, slot) + slot_row * D;
    if (lane == 0) {
      ml[0] = m;
      ml[1] = l;
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) dst[lane * (D / 64) + i] = acc[i];
  } else {
    E* dst = reinterpret_cast<E*>(a.out) + out_row * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) dst[lane * (D / 64) + i] = (E)(none ? 0.f : acc[i] / l);
    if (a.lse != nullptr && lane == 0)
      a.lse[out_row] = none ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

// A slot's job, by one thread of its workgroup. (Row ranges that overlap each other can ask for
// more slots than there are: their rows stay as they were.)
__device__ __forceinline__ void store_job(const AttendArgs& a, bool few, unsigned int slot, Job j) {
  const unsigned int slots = few ? a.few_slots : a.tile_slots;
  if (threadIdx.x != 0 || slot >= slots) return;
  if (j.splits != 0 && slot + (unsigned long long)(j.splits - 1) * a.kv_heads >= slots) j.splits = 0;
  a.jobs[(few ? a.tile_slots : 0u) + slot] = j;
}

// ---------------------------------------------------------------------------
// 128 rows by 64 tokens a step

// Lane l of a wave has row l % 32 of the wave's 32 and, of every 16 tokens, those with
// (token / 4) % 2 == l / 32 (the 32x32 matrix instruction's output rows). K lies in LDS as rows
// of D values, V too, both with their 16-byte pieces exchanged within a row so that the lanes of
// one read spread over the banks: K's piece c of row t at c ^ (t % 16), read 16 bytes a lane by 32
// rows; V's 64-byte quarters q at q ^ (t % 4), read transposed 8 bytes a lane, 4 tokens by 32 dims
// per half wave.
template <typename E, int D, bool kPaged, bool kRuns>
__device__ __forceinline__ void tile_path(const AttendArgs& a, const Request& first_requests,
                                          const SplitSteps& steps, unsigned int block,
                                          unsigned char* s0, unsigned char* s1) {
  typedef typename Elem<E>::x8 x8;
  constexpr int kRowBytes = 2 * D, kPieces = kRowBytes / 16;  // pieces of a row
  constexpr int kRowsPerLoad = kWave / kPieces, kLoads = 16 / kRowsPerLoad;
  constexpr int kTileBytes = kTileTokens * kRowBytes;
  constexpr int kSlabs = D / 16, kDimTiles = D / 32;

  const unsigned int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const unsigned int half = lane / 32, col = lane % 32;
  const unsigned int head = block % a.kv_heads, item = block / a.kv_heads, slot = block;
  Place p;
  if (!find_item(a, first_requests, item, [&](const Request& q) -> unsigned int {
        return kind_of(a, q) == 2 ? tiles_of(a, q.n) * tile_splits(q.ctx, steps.tiles) : 0u;
      }, p)) {
    store_job(a, false, slot, Job{});
    return;
  }
  const unsigned int all = tile_splits(p.q.ctx, steps.tiles);
  // the tiles with the longest contexts first
  const unsigned int tile = tiles_of(a, p.q.n) - 1 - p.index / all, split = p.index % all;
  const unsigned int rows = p.q.n * a.group;
  const unsigned int m0 = tile * kTileRows;
  // last visible token of a row (negative: none)
  const int shift = (int)p.q.ctx - (int)p.q.n;
  const int last_of_tile = shift + (int)((min(rows, m0 + kTileRows) - 1) / a.group);
  const unsigned int seen = last_of_tile < 0 ? 0u : (unsigned int)last_of_tile + 1;
  const unsigned int splits = tile_splits(seen, steps.tiles);  // of this tile
  store_job(a, false, slot,
            Job{p.q.start, m0, shift, (unsigned short)min(rows - m0, (unsigned int)kTileRows),
                (unsigned short)(split == 0 && splits > 1 ? splits : 0u)});
  if (split >= splits) return;
  const unsigned int t_begin = split * steps.tiles * kTileTokens;
  const unsigned int t_end =
      splits == 1 ? seen : min(seen, t_begin + steps.tiles * kTileTokens);
  const unsigned int mw = m0 + wave * 32, m = mw + col;
  const bool valid = m < rows;
  const unsigned int token = valid ? m / a.group : 0u;
  const unsigned int q_head = head * a.group + (valid ? m - token * a.group : 0u);
  const int limit = valid ? shift + (int)token : -1;
  // of the wave's rows: the last visible token of the first and of the last
  const int first_limit = shift + (int)(mw / a.group);
  const int last_limit = mw < rows ? shift + (int)((min(rows, mw + 32) - 1) / a.group) : -1;

  const int* table = kPaged ? a.tables + p.r * a.table_stride : nullptr;
  const unsigned char* kb = a.k + head * a.k_head;
  const unsigned char* vb = a.v + head * a.v_head;
  bool bad = p.q.bad;

  // the row's query as the second operand: dims 16 s + 8 half .. + 7 of slab s (a lane without a
  // row has the request's first: a column of the products that nobody reads)
  x8 q[kSlabs];
  const unsigned char* q_row = a.q + (unsigned long long)(p.q.start + token) * a.q_row +
                               (unsigned long long)q_head * a.q_head;
#pragma unroll
  for (int s = 0; s < kSlabs; ++s) {
    q[s] = *reinterpret_cast<const x8*>(q_row + 32 * s + 16 * half);
  }

  // this wave's share of a tile: 16 tokens of K and V. Where they follow each other in memory
  // (prompts; layers whose blocks are whole groups of 16 tokens) the wave forms their address once,
  // on the scalar unit, and a lane's offsets from it never change.
  const unsigned int piece = lane % kPieces, sub = lane / kPieces;
  unsigned int k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const unsigned int in = i * kRowsPerLoad + sub;  // the token's place among the wave's 16
    const unsigned int k_piece = piece ^ (D == 128 ? in : (in >> 1) & 7);
    const unsigned int v_piece = piece ^ (D == 128 ? (in & 3) << 2 : ((in >> 1) & 1) << 2);
    k_off[i] = (kRuns ? in * (unsigned int)a.k_row : 0u) + 16 * k_piece;
    v_off[i] = (kRuns ? in * (unsigned int)a.v_row : 0u) + 16 * v_piece;
  }
  constexpr int kIds = kRuns ? 1 : kLoads;
  int ids[kIds];
  auto token_of = [&](unsigned int base, int i) {
    return min(base + wave * 16 + (kRuns ? 0 : i * kRowsPerLoad + sub), t_end - 1);
  };
  auto fetch_ids = [&](unsigned int base) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) ids[i] = block_id<kPaged>(a, table, token_of(base, i));
  };
  auto issue = [&](unsigned int base, unsigned char* bk, unsigned char* bv) {
    const unsigned int at = wave * 16 * kRowBytes;
    if constexpr (kRuns) {
      // tokens past the end are outside the buffers
      const unsigned int first = base + wave * 16, count = min(t_end - min(first, t_end), 16u);
      const unsigned int row = uniform(kv_row<kPaged>(a, table, p.q.start, token_of(base, 0), ids[0], bad));
      // (sizes moved to scalars: with one in a vector register each load became a loop over lanes)
      const Buffer kr = buffer_of(
          kb + row * a.k_row,
          uniform(count == 0 ? 0u : (count - 1) * (unsigned int)a.k_row + kRowBytes));
      const Buffer vr = buffer_of(
          vb + row * a.v_row,
          uniform(count == 0 ? 0u : (count - 1) * (unsigned int)a.v_row + kRowBytes));
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        load_to_lds(kr, k_off[i], bk + at + i * kRowsPerLoad * kRowBytes);
        load_to_lds(vr, v_off[i], bv + at + i * kRowsPerLoad * kRowBytes);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const unsigned int row = kv_row<kPaged>(a, table, p.q.start, token_of(base, i), ids[i], bad);
        load_to_lds(kb + row * a.k_row + k_off[i], bk + at + i * kRowsPerLoad * kRowBytes);
        load_to_lds(vb + row * a.v_row + v_off[i], bv + at + i * kRowsPerLoad * kRowBytes);
      }
    }
  };

  f32x16 o[kDimTiles];
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m_ref = kNoMax, l_run = 0.f;

  // K operand: row col (+ 32), piece 2 s + half; V operand: tokens 4 half + i / 4 (i = lane % 16) of
  // 16, dims 16 (lane / 16 % 2) + 4 (i % 4) of 32
  const unsigned int k_at = col * kRowBytes, k_x = D == 128 ? col & 15 : (col >> 1) & 7;
  const unsigned int v_tok = 4 * half + (lane % 16) / 4;
  const unsigned int v_x = D == 128 ? v_tok & 3 : (v_tok >> 1) & 1;
  const unsigned int v_at = v_tok * kRowBytes + 32 * ((lane / 16) % 2) + 8 * (lane % 4);

  auto step = [&](unsigned int base, const unsigned char* bk, const unsigned char* bv) {
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
#pragma unroll
      for (int c = 0; c < kSlabs; ++c) {
        const x8 kf = *reinterpret_cast<const x8*>(bk + k_at + 32 * t * kRowBytes +
                                                   16 * ((2 * c + half) ^ k_x));
        s[t] = Elem<E>::mma32(kf, q[c], s[t]);
      }
    }
    if ((int)base + kTileTokens - 1 > first_limit) {
      const int left = limit - (int)base - 4 * (int)half;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[t][i] = 32 * t + 8 * (i / 4) + i % 4 <= left ? s[t][i] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    {
      const unsigned int u = __builtin_bit_cast(unsigned int, top);
      const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      top = fmaxf(__builtin_bit_cast(float, (unsigned int)w[0]),
                  __builtin_bit_cast(float, (unsigned int)w[1]));
    }
    top *= a.scale_log2;
    if (__ballot(top > m_ref + kSlack) != 0) {
      const float now = fmaxf(m_ref, top), alpha = __builtin_amdgcn_exp2f(m_ref - now);
      m_ref = now;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
    }
    float sum = 0.f;
    x8 w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[c / 2][8 * (c % 2) + i], a.scale_log2, -m_ref));
        sum += e[i];
      }
      w[c] = pack8<E>(e);
    }
    l_run += sum;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d) {
        const unsigned char* src = bv + v_at + 16 * c * kRowBytes + 64 * (d ^ v_x);
        const u32x2 lo = read_transposed(src), hi = read_transposed(src + 8 * kRowBytes);
        o[d] = Elem<E>::mma32(__builtin_bit_cast(x8, u32x4{lo.x, lo.y, hi.x, hi.y}), w[c], o[d]);
      }
  };

  if (t_begin < t_end) {
    fetch_ids(t_begin);
    issue(t_begin, s0, s0 + kTileBytes);
    if (t_begin + kTileTokens < t_end) fetch_ids(t_begin + kTileTokens);
    unsigned int base = t_begin;
    auto turn = [&](unsigned char* now, unsigned char* next) {
      // this tile's loads have landed, and every wave is done with the other buffer
      wait_loads<0>();
      __syncthreads();
      if (base + kTileTokens < t_end) {
        issue(base + kTileTokens, next, next + kTileBytes);
        if (base + 2 * kTileTokens < t_end) fetch_ids(base + 2 * kTileTokens);
      }
      if ((int)base <= last_limit) step(base, now, now + kTileBytes);
      base += kTileTokens;
    };
    while (base < t_end) {
      turn(s0, s1);
      if (base >= t_end) break;
      turn(s1, s0);
    }
  }

  bad = __syncthreads_or(bad) != 0;
  l_run += __shfl_xor(l_run, 32, 64);
  float check = l_run * 0.f;
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) check = fmaf(o[d][i], 0.f, check);
  check += __shfl_xor(check, 32, 64);
  const bool again = valid && !bad && !(check == 0.f);
  const unsigned long long out_row = (unsigned long long)(p.q.start + token) * a.q_heads + q_head;
  if (bad) m_ref = l_run = NAN;
  if (valid && !again) {
    if (splits > 1) {
      float* ml = slot_ml<D>(a, false, slot) + 2 * (m - m0);
      float* dst = slot_acc<D>(a, false, slot) + (m - m0) * D;
      if (half == 0) {
        ml[0] = m_ref;
        ml[1] = l_run;
      }
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * i + 4 * half) =
              f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    } else {
      // a row that sees no token is zero
      const bool none = limit < 0 && !bad;
      const float inv = none ? 0.f : 1.f / l_run;
      unsigned char* dst = a.out + out_row * kRowBytes;
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x2*>(dst + 2 * (32 * d + 8 * i + 4 * half)) =
              u32x2{pack2<E>(o[d][4 * i] * inv, o[d][4 * i + 1] * inv),
                    pack2<E>(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv)};
      if (a.lse != nullptr && half == 0)
        a.lse[out_row] = none ? -INFINITY : (m_ref + log2f(l_run)) * kLn2;
    }
  }
  unsigned int redo = (unsigned int)__ballot(again);
  while (redo != 0) {
    const unsigned int at = uniform((unsigned int)__ffs((int)redo) - 1);
    redo &= redo - 1;
    const unsigned int row_m = mw + at, tok = row_m / a.group, qh = head * a.group + row_m % a.group;
    const unsigned int own = (unsigned int)max(shift + (int)tok + 1, 0);  // tokens it sees
    float rm, rl, acc[D / 64];
    slow_row<E, D, kPaged>(a, table, p.q.start,
                           a.q + (unsigned long long)(p.q.start + tok) * a.q_row +
                               (unsigned long long)qh * a.q_head,
                           head, t_begin, min(t_end, own), rm, rl, acc);
    store_slow<E, D>(a, splits > 1, false, slot, row_m - m0,
                     (unsigned long long)(p.q.start + tok) * a.q_heads + qh, own == 0, rm, rl, acc);
  }
}

// ---------------------------------------------------------------------------
// at most 16 rows, streaming

// Lane l has row l % 16 and, of every 16 tokens, the four from 4 (l / 16) on. A wave's step is 32
// tokens: K as the first operand of S^T = K Q^T straight from memory (lane l: token l % 16, 16
// bytes at 16 (l / 16) of every 64), V through the wave's own LDS, without a barrier, with 32-byte
// pieces of row t at piece ^ (t % 8), so that the 16 tokens of a transposed read spread over the
// banks. The waves of a workgroup take turns at 32 tokens of a split and join their sums in LDS.
template <typename E, int D>
__device__ __forceinline__ void few_path(const AttendArgs& a, const Request& first_requests,
                                         const SplitSteps& steps, unsigned int block,
                                         unsigned char* s0, unsigned char* s1) {
  typedef typename Elem<E>::x8 x8;
  constexpr int kRowBytes = 2 * D, kPieces = kRowBytes / 16;
  constexpr int kRowsPerLoad = kWave / kPieces, kLoads = kFewStep / kRowsPerLoad;
  constexpr int kStageBytes = kFewStep * kRowBytes;
  constexpr int kSlabs = D / 32, kDimTiles = D / 16;
  // the waves' sums, then their (m, l), once the stages are read
  float* const s_acc = reinterpret_cast<float*>(s0);
  float* const s_ml = reinterpret_cast<float*>(s1);
  static_assert(kStageBytes >= kFewRows * D * 4, "a wave's sums fit its stage");

  const unsigned int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const unsigned int col = lane % 16, grp = lane / 16;
  const unsigned int head = block % a.kv_heads, item = block / a.kv_heads, slot = block;
  Place p;
  if (!find_item(a, first_requests, item, [&](const Request& q) -> unsigned int {
        return kind_of(a, q) == 1 ? few_splits(q.ctx, steps.few) : 0u;
      }, p)) {
    store_job(a, true, slot, Job{});
    return;
  }
  const unsigned int splits = few_splits(p.q.ctx, steps.few), split = p.index;
  store_job(a, true, slot,
            Job{p.q.start, 0, (int)p.q.ctx - (int)p.q.n, (unsigned short)(p.q.n * a.group),
                (unsigned short)(split == 0 && splits > 1 ? splits : 0u)});
  const unsigned int rows = p.q.n * a.group;
  const unsigned int t_begin = split * steps.few * kFewRound;
  const unsigned int t_end = min(p.q.ctx, t_begin + steps.few * kFewRound);
  const int shift = (int)p.q.ctx - (int)p.q.n;
  const bool valid = col < rows;
  const unsigned int token = valid ? col / a.group : 0u;
  const unsigned int q_head = head * a.group + (valid ? col - token * a.group : 0u);
  const int limit = valid ? shift + (int)token : -1;

  const int* table = a.tables + p.r * a.table_stride;
  const unsigned char* kb = a.k + head * a.k_head;
  const unsigned char* vb = a.v + head * a.v_head;
  bool bad = p.q.bad;

  x8 q[kSlabs];
  const unsigned char* q_row = a.q + (unsigned long long)(p.q.start + token) * a.q_row +
                               (unsigned long long)q_head * a.q_head;
#pragma unroll
  for (int s = 0; s < kSlabs; ++s) {
    q[s] = *reinterpret_cast<const x8*>(q_row + 64 * s + 16 * grp);
  }

  struct Keys {
    u32x4 v[2][kSlabs];
  };
  unsigned char* const stage0 = s0 + wave * kStageBytes;
  unsigned char* const stage1 = s1 + wave * kStageBytes;
  const unsigned int piece = lane % kPieces, sub = lane / kPieces;
  // lane l looks up token l % 32 of a step
  auto token_of = [&](unsigned int base) { return min(base + lane % 32, t_end - 1); };
  auto issue = [&](unsigned int base, int id, Keys& k, unsigned char* stage) {
    const unsigned int row = kv_row<true>(a, table, 0u, token_of(base), id, bad);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned char* src = kb + (unsigned int)__shfl(row, 16 * u + (int)col, kWave) * a.k_row;
#pragma unroll
      for (int s = 0; s < kSlabs; ++s)
        k.v[u][s] = *reinterpret_cast<const u32x4*>(src + 64 * s + 16 * grp);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const unsigned int in = i * kRowsPerLoad + sub;
      const unsigned int x = D == 128 ? in & 7 : (in >> 1) & 3;
      load_to_lds(vb + (unsigned int)__shfl(row, (int)in, kWave) * a.v_row + 16 * (piece ^ (x << 1)),
                  stage + i * kRowsPerLoad * kRowBytes);
    }
  };

  f32x4 o[kDimTiles];
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d) o[d] = f32x4{0, 0, 0, 0};
  float m_ref = kNoMax, l_run = 0.f;
  const unsigned int v_tok = 4 * grp + col / 4;
  const unsigned int v_x = D == 128 ? v_tok & 7 : (v_tok >> 1) & 3;
  const unsigned int v_at = v_tok * kRowBytes + 8 * (col % 4);

  auto step = [&](unsigned int base, const Keys& k, const unsigned char* stage) {
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4 st = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kSlabs; ++c)
        st = Elem<E>::mma16(__builtin_bit_cast(x8, k.v[u][c]), q[c], st);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * u + j] = st[j];
    }
    if ((int)base + kFewStep - 1 > shift) {
      const int left = limit - (int)base - 4 * (int)grp;
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = 16 * (j / 4) + j % 4 <= left ? s[j] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    top *= a.scale_log2;
    if (__ballot(top > m_ref + kSlack) != 0) {
      const float now = fmaxf(m_ref, top), alpha = __builtin_amdgcn_exp2f(m_ref - now);
      m_ref = now;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][j] *= alpha;
    }
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(fmaf(s[j], a.scale_log2, -m_ref));
      l_run += e[j];
    }
    const x8 w = pack8<E>(e);
    const unsigned char* bv = stage + v_at;
#pragma unroll
    for (int d = 0; d < kDimTiles; ++d) {
      const unsigned char* src = bv + 32 * (d ^ v_x);
      const u32x2 lo = read_transposed(src), hi = read_transposed(src + 16 * kRowBytes);
      o[d] = Elem<E>::mma16(__builtin_bit_cast(x8, u32x4{lo.x, lo.y, hi.x, hi.y}), w, o[d]);
    }
  };

  unsigned int base = t_begin + wave * kFewStep;
  if (base < t_end) {
    Keys k0, k1;
    issue(base, block_id<true>(a, table, token_of(base)), k0, stage0);
    int id = block_id<true>(a, table, token_of(base + kFewRound));
    for (;;) {
      // the next step's loads go out (past the end: the last token again), then this step's
      // are waited for
      issue(base + kFewRound, id, k1, stage1);
      id = block_id<true>(a, table, token_of(base + 2 * kFewRound));
      wait_loads<2 * kSlabs + kLoads + 1>();
      step(base, k0, stage0);
      base += kFewRound;
      if (base >= t_end) break;
      issue(base + kFewRound, id, k0, stage0);
      id = block_id<true>(a, table, token_of(base + 2 * kFewRound));
      wait_loads<2 * kSlabs + kLoads + 1>();
      step(base, k1, stage1);
      base += kFewRound;
      if (base >= t_end) break;
    }
  }
  wait_loads<0>();

  // ---- the waves' sums meet in LDS, thread t takes row t / 16 and D / 16 dims of it ----
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  bad = __syncthreads_or(bad) != 0;
  if (grp == 0) {
    s_ml[2 * (wave * kFewRows + col)] = m_ref;
    s_ml[2 * (wave * kFewRows + col) + 1] = l_run;
  }
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d)
    *reinterpret_cast<f32x4*>(s_acc + (wave * kFewRows + col) * D + 16 * d + 4 * grp) = o[d];
  __syncthreads();
  constexpr int kVals = D / 16;
  const unsigned int row_m = tid / 16, d0 = (tid % 16) * kVals;
  float big = kNoMax, l = 0.f, acc[kVals];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) big = fmaxf(big, s_ml[2 * (w * kFewRows + row_m)]);
#pragma unroll
  for (int i = 0; i < kVals; ++i) acc[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float f = exp2f(s_ml[2 * (w * kFewRows + row_m)] - big);
    l += s_ml[2 * (w * kFewRows + row_m) + 1] * f;
#pragma unroll
    for (int i = 0; i < kVals; ++i) acc[i] += s_acc[(w * kFewRows + row_m) * D + d0 + i] * f;
  }
  float check = l * 0.f;
#pragma unroll
  for (int i = 0; i < kVals; ++i) check = fmaf(acc[i], 0.f, check);
#pragma unroll
  for (int d = 1; d < 16; d *= 2) check += __shfl_xor(check, d, 64);
  const bool in = row_m < rows;
  const bool again = in && !bad && !(check == 0.f);
  const unsigned int tok = in ? row_m / a.group : 0u;
  const unsigned int qh = head * a.group + (in ? row_m - tok * a.group : 0u);
  const unsigned long long out_row = (unsigned long long)(p.q.start + tok) * a.q_heads + qh;
  if (bad) big = l = NAN;
  if (in && !again) {
    if (splits > 1) {
      float* ml = slot_ml<D>(a, true, slot) + 2 * row_m;
      float* dst = slot_acc<D>(a, true, slot) + row_m * D + d0;
      if (d0 == 0) {
        ml[0] = big;
        ml[1] = l;
      }
#pragma unroll
      for (int i = 0; i < kVals; i += 4)
        *reinterpret_cast<f32x4*>(dst + i) = f32x4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
    } else {
      const bool none = shift + (int)tok < 0 && !bad;
      const float inv = none ? 0.f : 1.f / l;
      uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + out_row * kRowBytes + 2 * d0);
#pragma unroll
      for (int i = 0; i < kVals; i += 2) dst[i / 2] = pack2<E>(acc[i] * inv, acc[i + 1] * inv);
      if (a.lse != nullptr && d0 == 0)
        a.lse[out_row] = none ? -INFINITY : (big + log2f(l)) * kLn2;
    }
  }
  const unsigned long long flags = __ballot(again);
#pragma unroll 1
  for (unsigned int i = 0; i < 4; ++i) {
    if (((flags >> (16 * i)) & 1) == 0) continue;
    const unsigned int mm = 4 * wave + i, t = mm / a.group, h = head * a.group + mm % a.group;
    const unsigned int seen = (unsigned int)max(shift + (int)t + 1, 0);
    float rm, rl, ra[D / 64];
    slow_row<E, D, true>(a, table, p.q.start,
                         a.q + (unsigned long long)(p.q.start + t) * a.q_row +
                             (unsigned long long)h * a.q_head,
                         head, t_begin, min(t_end, seen), rm, rl, ra);
    store_slow<E, D>(a, splits > 1, true, slot, mm,
                     (unsigned long long)(p.q.start + t) * a.q_heads + h, seen == 0, rm, rl, ra);
  }
}

// ---------------------------------------------------------------------------
// both paths in one launch

// Workgroups take the two paths in turns of 8 (one on each XCD, so that a KV head of eight stays
// on its XCD's L2), so that streaming and matrix work run beside each other, then what is left of
// the longer list.
template <typename E, int D, bool kPaged, bool kTiles, bool kFew, bool kRuns>
__global__ __launch_bounds__(kT, 2) void attention_step(AttendArgs a) {
  // (a variable for each buffer: the compiler orders a read of one behind the loads into it, and
  // not behind those into the other)
  constexpr int kBuffer = 2 * kTileTokens * 2 * D;
  static_assert(kBuffer == kWaves * kFewStep * 2 * D, "both paths' stages");
  __shared__ __align__(1024) unsigned char s0[kBuffer];
  __shared__ __align__(1024) unsigned char s1[kBuffer];
  const Request first_requests = load_request(a, __lane_id());
  const SplitSteps steps = split_steps(a, first_requests);
  unsigned int block = blockIdx.x;
  bool few = kFew;
  if constexpr (kTiles && kFew) {
    const unsigned int turns = min(a.tile_groups, a.few_groups) / 8;
    if (block < 16 * turns) {
      few = (block / 8) % 2 != 0;
      block = block / 16 * 8 + block % 8;
    } else {
      block -= 8 * turns;
      few = block >= a.tile_groups;
      if (few) block -= a.tile_groups - 8 * turns;
    }
  }
  if (kFew && few) {
    if constexpr (kFew) few_path<E, D>(a, first_requests, steps, block, s0, s1);
  } else {
    if constexpr (kTiles) tile_path<E, D, kPaged, kRuns>(a, first_requests, steps, block, s0, s1);
  }
}

// ---------------------------------------------------------------------------
// the splits of a row joined

// A workgroup looks at its share of the slots' jobs with one load and takes those that have
// something to join: 16 rows of a tile with a thread for 8 (D = 64: 4) sums of a row, or 4 rows of
// the streaming path, which has more splits, with four threads that share a row's splits.
constexpr int kTileParts = kTileRows / 16, kFewParts = kFewRows / 4;

template <typename E, int D>
__global__ __launch_bounds__(kT) void attention_merge(AttendArgs a) {
  constexpr int kVals = D / 16;
  constexpr int kBatch = 8;
  __shared__ float s_part[kT][kVals + 2];
  const unsigned int tid = threadIdx.x, lane = tid & 63;
  const unsigned int tile_jobs = a.tile_slots * kTileParts;
  const unsigned int jobs = tile_jobs + a.few_slots * kFewParts;
  auto slot_of = [&](unsigned int j) {
    return j < tile_jobs ? j / kTileParts : a.tile_slots + (j - tile_jobs) / kFewParts;
  };
  for (unsigned int j0 = blockIdx.x; j0 < jobs; j0 += kWave * gridDim.x) {
    const unsigned int mine = j0 + lane * gridDim.x;
    unsigned long long todo = __ballot(mine < jobs && a.jobs[slot_of(min(mine, jobs - 1))].splits != 0);
    while (todo != 0) {
      const unsigned int j = j0 + ((unsigned int)__ffsll((long long)todo) - 1) * gridDim.x;
      todo &= todo - 1;
      const bool few = j >= tile_jobs;
      const unsigned int job_slot = slot_of(j);
      const Job job = a.jobs[job_slot];
      const unsigned int slot = few ? job_slot - a.tile_slots : job_slot;
      const unsigned int head = slot % a.kv_heads;
      const unsigned int shares = few ? 4 : 1;  // threads that share a row's splits
      const unsigned int share = (tid / 16) % shares, dims = (tid % 16) * kVals;
      const unsigned int row = few ? (j - tile_jobs) % kFewParts * 4 + tid / 64
                                   : j % kTileParts * 16 + tid / 16;
      const bool in = row < job.rows;
      const unsigned int use = in ? row : 0u;
      float big = kNoMax, l = 0.f, acc[kVals];
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kVals; ++i) acc[i] = 0.f;
      for (unsigned int b = share; b < job.splits; b += shares * kBatch) {
        f32x2 ml[kBatch];
        f32x4 v[kBatch][kVals / 4];
        // (past the last split the last one again, without weight: loads behind branches would
        // wait for each other)
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const unsigned int at = slot + min(b + k * shares, job.splits - 1u) * a.kv_heads;
          ml[k] = *reinterpret_cast<const f32x2*>(slot_ml<D>(a, few, at) + 2 * use);
          const float* src = slot_acc<D>(a, few, at) + use * D + dims;
#pragma unroll
          for (int i = 0; i < kVals / 4; ++i) v[k][i] = *reinterpret_cast<const f32x4*>(src + 4 * i);
        }
        float top = big;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (b + k * shares >= job.splits) ml[k] = f32x2{kNoMax, 0.f};
          bad |= ml[k].x != ml[k].x;
          top = fmaxf(top, ml[k].x);
        }
        const float alpha = exp2f(big - top);
        big = top;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < kVals; ++i) acc[i] *= alpha;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const float f = b + k * shares < job.splits ? exp2f(ml[k].x - big) : 0.f;
          l += ml[k].y * f;
#pragma unroll
          for (int i = 0; i < kVals; ++i) acc[i] = f != 0.f ? fmaf(v[k][i / 4][i % 4], f, acc[i]) : acc[i];
        }
      }
      if (few) {
        __syncthreads();  // the job before this one is done with the LDS
        float* own = s_part[tid];
        own[0] = bad ? NAN : big;
        own[1] = l;
#pragma unroll
        for (int i = 0; i < kVals; ++i) own[2 + i] = acc[i];
        __syncthreads();
        big = kNoMax;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float m = s_part[tid / 64 * 64 + 16 * k + tid % 16][0];
          bad |= m != m;
          big = fmaxf(big, m);
        }
        l = 0.f;
#pragma unroll
        for (int i = 0; i < kVals; ++i) acc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* src = s_part[tid / 64 * 64 + 16 * k + tid % 16];
          const float f = exp2f(src[0] - big);
          l += src[1] * f;
#pragma unroll
          for (int i = 0; i < kVals; ++i) acc[i] += src[2 + i] * f;
        }
        if (share != 0) continue;
      }
      if (!in) continue;
      const unsigned int m = job.first + row, tok = m / a.group;
      const unsigned long long out_row =
          (unsigned long long)(job.start + tok) * a.q_heads + head * a.group + (m - tok * a.group);
      const bool none = job.shift + (int)tok < 0 && !bad;
      const float inv = bad ? NAN : none ? 0.f : 1.f / l;
      uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (out_row * D + dims) * 2);
#pragma unroll
      for (int i = 0; i < kVals; i += 2) dst[i / 2] = pack2<E>(acc[i] * inv, acc[i + 1] * inv);
      if (a.lse != nullptr && dims == 0)
        a.lse[out_row] = bad ? NAN : none ? -INFINITY : (big + log2f(l)) * kLn2;
    }
  }
}

}  // namespace
}  // namespace unchainkv

using namespace unchainkv;

namespace {

unsigned long long compute_units() {
  static std::mutex mu;
  static unsigned long long cached[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  std::lock_guard<std::mutex> lock(mu);
  if (cached[dev] == 0) {
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        cus <= 0)
      cus = 256;
    cached[dev] = (unsigned long long)cus;
  }
  return cached[dev];
}

// Bounds of a call's grids and partial slots, from what the host knows: tokens (rows of q),
// requests, the longest context that the tables (or the rows) can hold, and the longest request.
struct Bounds {
  unsigned long long few_target, tile_target;
  unsigned long long few_items, tile_items;  // times KV heads: workgroups, and partial slots
  bool few, tiles;
};

Bounds bounds_of(unsigned long long tokens, unsigned long long requests, unsigned long long kv_heads,
                 unsigned long long group, unsigned long long max_context,
                 unsigned long long max_query, bool paged) {
  Bounds b{};
  b.few_target = b.tile_target = 2 * compute_units();  // workgroups resident at once
  const unsigned long long active = std::min(tokens, requests);
  const unsigned long long rows = max_query * group;
  b.few = paged && active != 0;
  b.tiles = !paged || rows > kFewRows;
  if (b.few) {
    // sum over requests of ceil(rounds / steps) <= all rounds / steps + requests
    const unsigned long long most = std::max(1ull, (max_context + kFewRound - 1) / kFewRound);
    b.few_items = std::min(active * most, b.few_target / kv_heads + active + 1);
  }
  if (b.tiles) {
    const unsigned long long tiles = tokens * group / kTileRows + active;
    const unsigned long long most =
        std::max(1ull, (max_context + kTileTokens * kLeastTileSteps - 1) / (kTileTokens * kLeastTileSteps));
    // split, there are fewer than tile_target tiles, and of tiles * context / steps <= 2 *
    // tile_target more; not split, one item a tile
    b.tile_items = std::max(tiles, std::min(tiles * most, (3 * b.tile_target) / kv_heads + 1));
  }
  return b;
}

unsigned long long tile_slots_of(const Bounds& b, unsigned long long kv_heads) {
  // (only split launches write partials)
  return b.tiles ? std::min(b.tile_items * kv_heads, 3 * b.tile_target + kv_heads) : 0;
}

// The slots' partials, then their jobs.
unsigned long long partial_bytes(const Bounds& b, unsigned long long kv_heads,
                                 unsigned long long head_dim) {
  return (b.few_items * kv_heads * kFewRows + tile_slots_of(b, kv_heads) * kTileRows) *
         (head_dim + 2) * sizeof(float);
}
unsigned long long workspace_of(const Bounds& b, unsigned long long kv_heads,
                                unsigned long long head_dim) {
  return partial_bytes(b, kv_heads, head_dim) +
         (b.few_items * kv_heads + tile_slots_of(b, kv_heads)) * sizeof(Job);
}

template <typename E, int D, bool kPaged>
long long launch(const AttendArgs& a, hipStream_t stream) {
  const dim3 grid(a.tile_groups + a.few_groups), threads(kT);
  if constexpr (!kPaged)
    hipLaunchKernelGGL((attention_step<E, D, false, true, false, true>), grid, threads, 0, stream, a);
  else if (a.tile_groups == 0)
    hipLaunchKernelGGL((attention_step<E, D, true, false, true, false>), grid, threads, 0, stream, a);
  else if (a.block_tokens % 16 == 0)
    hipLaunchKernelGGL((attention_step<E, D, true, true, true, true>), grid, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((attention_step<E, D, true, true, true, false>), grid, threads, 0, stream, a);
  hipError_t st = hipGetLastError();
  if (st != hipSuccess) return fail("attention_step", st);
  const unsigned int jobs = a.tile_slots * kTileParts + a.few_slots * kFewParts;
  hipLaunchKernelGGL((attention_merge<E, D>), dim3(std::min(jobs, 1024u)), threads, 0, stream, a);
  st = hipGetLastError();
  if (st != hipSuccess) return fail("attention_merge", st);
  return (long long)((unsigned long long)a.tokens * a.q_heads * D * 2);
}

template <bool kPaged>
long long launch_typed(const AttendArgs& a, unsigned long long head_dim, unsigned long long dtype,
                       hipStream_t stream) {
  if (head_dim == 128)
    return dtype ? launch<_Float16, 128, kPaged>(a, stream) : launch<__bf16, 128, kPaged>(a, stream);
  return dtype ? launch<_Float16, 64, kPaged>(a, stream) : launch<__bf16, 64, kPaged>(a, stream);
}

constexpr unsigned long long kMostRows = 0x7FFFFFFFull;
constexpr unsigned long long kMostStride = 1ull << 27;  // 16 rows' offsets fit 32 bits

// Bytes from the first to the last of rows x heads pieces of head_bytes.
unsigned long long extent(unsigned long long rows, unsigned long long row_bytes,
                          unsigned long long heads, unsigned long long head_step,
                          unsigned long long head_bytes) {
  return (rows - 1) * row_bytes + (heads - 1) * head_step + head_bytes;
}

bool sizes_ok(unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
              unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_query) {
  return tokens != 0 && tokens <= kMostRows && requests != 0 && requests <= kMostRows &&
         kv_heads != 0 && kv_heads <= 4096 && q_heads != 0 && q_heads <= 65536 &&
         q_heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128) && max_query != 0 &&
         max_query <= tokens && tokens * q_heads <= kMostRows;
}

}  // namespace

extern "C" unsigned long long kvq_splitzip_chunk_attention_workspace_bytes(
    unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_context,
    unsigned long long max_query) {
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_of(bounds_of(tokens, requests, kv_heads, q_heads / kv_heads, max_context,
                                 max_query, true), kv_heads, head_dim);
}

extern "C" unsigned long long kvq_splitzip_prompt_attention_workspace_bytes(
    unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_query) {
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_of(bounds_of(tokens, requests, kv_heads, q_heads / kv_heads, max_query,
                                 max_query, false), kv_heads, head_dim);
}

extern "C" long long kvq_splitzip_chunk_attention_paged(
    unsigned long long q_ptr, unsigned long long q_row_bytes, unsigned long long q_head_bytes,
    unsigned long long tokens, unsigned long long q_heads, unsigned long long kv_heads,
    unsigned long long head_dim, unsigned long long dtype, unsigned long long kv_ptr,
    unsigned long long blocks, unsigned long long block_tokens, unsigned long long tables_ptr,
    unsigned long long table_stride, unsigned long long table_width,
    unsigned long long query_starts_ptr, unsigned long long context_tokens_ptr,
    unsigned long long requests, unsigned long long max_query, unsigned long long out_ptr,
    unsigned long long lse_ptr, unsigned long long workspace_ptr,
    unsigned long long workspace_bytes, float scale, unsigned long long stream_ptr) {
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query) || dtype > 1 ||
      q_ptr == 0 || q_ptr % 16 != 0 || q_row_bytes % 16 != 0 || q_head_bytes % 16 != 0 ||
      kv_ptr == 0 || kv_ptr % 16 != 0 || blocks == 0 || block_tokens == 0 || blocks > kMostRows ||
      block_tokens > kMostRows || blocks * block_tokens > kMostRows || tables_ptr == 0 ||
      table_width == 0 || table_width > kMostRows || table_stride < table_width ||
      query_starts_ptr == 0 || context_tokens_ptr == 0 || out_ptr == 0 || out_ptr % 16 != 0 ||
      !(scale > 0.f) || !std::isfinite(scale))
    return 0;
  const unsigned long long max_context = std::min(table_width * block_tokens, kMostRows);
  const Bounds b = bounds_of(tokens, requests, kv_heads, q_heads / kv_heads, max_context, max_query, true);
  const unsigned long long need = workspace_of(b, kv_heads, head_dim);
  if (workspace_ptr == 0 || workspace_ptr % 16 != 0 || workspace_bytes < need) return 0;
  if ((b.tile_items + b.few_items) * kv_heads > kMostRows) return 0;
  const unsigned long long out_bytes = tokens * q_heads * head_dim * 2;
  if (overlap(out_ptr, out_bytes, q_ptr, extent(tokens, q_row_bytes, q_heads, q_head_bytes, 2 * head_dim)) ||
      overlap(out_ptr, out_bytes, kv_ptr, 4 * blocks * block_tokens * kv_heads * head_dim))
    return 0;
  AttendArgs a{};
  a.q = reinterpret_cast<const unsigned char*>(q_ptr);
  a.out = reinterpret_cast<unsigned char*>(out_ptr);
  a.lse = reinterpret_cast<float*>(lse_ptr);
  a.k = reinterpret_cast<const unsigned char*>(kv_ptr);
  a.k_head = a.v_head = 2 * head_dim;
  a.k_row = a.v_row = kv_heads * a.k_head;
  a.v = a.k + blocks * block_tokens * a.k_row;
  a.starts = reinterpret_cast<const int*>(query_starts_ptr);
  a.contexts = reinterpret_cast<const int*>(context_tokens_ptr);
  a.tables = reinterpret_cast<const int*>(tables_ptr);
  a.partial = reinterpret_cast<float*>(workspace_ptr);
  a.jobs = reinterpret_cast<Job*>(workspace_ptr + partial_bytes(b, kv_heads, head_dim));
  a.q_row = q_row_bytes;
  a.q_head = q_head_bytes;
  a.table_stride = table_stride;
  a.table_width = (unsigned int)std::min(table_width, max_context / block_tokens + 1);
  a.blocks = (unsigned int)blocks;
  a.block_tokens = (unsigned int)block_tokens;
  a.by_block = make_divider((unsigned int)block_tokens);
  a.tokens = (unsigned int)tokens;
  a.requests = (unsigned int)requests;
  a.q_heads = (unsigned int)q_heads;
  a.kv_heads = (unsigned int)kv_heads;
  a.group = (unsigned int)(q_heads / kv_heads);
  a.few_rows = kFewRows;
  a.tiles_too = b.tiles ? 1u : 0u;
  a.few_target = (unsigned int)b.few_target;
  a.tile_target = (unsigned int)b.tile_target;
  a.max_query = (unsigned int)max_query;
  a.tile_slots = (unsigned int)tile_slots_of(b, kv_heads);
  a.few_slots = a.few_groups = (unsigned int)(b.few_items * kv_heads);
  a.tile_groups = (unsigned int)(b.tile_items * kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  return launch_typed<true>(a, head_dim, dtype, reinterpret_cast<hipStream_t>(stream_ptr));
}

extern "C" long long kvq_splitzip_prompt_attention(
    unsigned long long q_ptr, unsigned long long q_row_bytes, unsigned long long q_head_bytes,
    unsigned long long k_ptr, unsigned long long k_row_bytes, unsigned long long k_head_bytes,
    unsigned long long v_ptr, unsigned long long v_row_bytes, unsigned long long v_head_bytes,
    unsigned long long tokens, unsigned long long q_heads, unsigned long long kv_heads,
    unsigned long long head_dim, unsigned long long dtype, unsigned long long query_starts_ptr,
    unsigned long long requests, unsigned long long max_query, unsigned long long out_ptr,
    unsigned long long lse_ptr, unsigned long long workspace_ptr,
    unsigned long long workspace_bytes, float scale, unsigned long long stream_ptr) {
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query) || dtype > 1 ||
      q_ptr == 0 || k_ptr == 0 || v_ptr == 0 ||
      (q_ptr | q_row_bytes | q_head_bytes | k_ptr | k_row_bytes | k_head_bytes | v_ptr |
       v_row_bytes | v_head_bytes) % 16 != 0 ||
      k_row_bytes > kMostStride || v_row_bytes > kMostStride || query_starts_ptr == 0 ||
      out_ptr == 0 || out_ptr % 16 != 0 || !(scale > 0.f) || !std::isfinite(scale))
    return 0;
  const Bounds b = bounds_of(tokens, requests, kv_heads, q_heads / kv_heads, max_query, max_query, false);
  const unsigned long long need = workspace_of(b, kv_heads, head_dim);
  if (workspace_ptr == 0 || workspace_ptr % 16 != 0 || workspace_bytes < need) return 0;
  if (b.tile_items * kv_heads > kMostRows) return 0;
  const unsigned long long out_bytes = tokens * q_heads * head_dim * 2;
  if (overlap(out_ptr, out_bytes, q_ptr, extent(tokens, q_row_bytes, q_heads, q_head_bytes, 2 * head_dim)) ||
      overlap(out_ptr, out_bytes, k_ptr, extent(tokens, k_row_bytes, kv_heads, k_head_bytes, 2 * head_dim)) ||
      overlap(out_ptr, out_bytes, v_ptr, extent(tokens, v_row_bytes, kv_heads, v_head_bytes, 2 * head_dim)))
    return 0;
  AttendArgs a{};
  a.q = reinterpret_cast<const unsigned char*>(q_ptr);
  a.out = reinterpret_cast<unsigned char*>(out_ptr);
  a.lse = reinterpret_cast<float*>(lse_ptr);
  a.k = reinterpret_cast<const unsigned char*>(k_ptr);
  a.v = reinterpret_cast<const unsigned char*>(v_ptr);
  a.k_row = k_row_bytes;
  a.k_head = k_head_bytes;
  a.v_row = v_row_bytes;
  a.v_head = v_head_bytes;
  a.starts = reinterpret_cast<const int*>(query_starts_ptr);
  a.partial = reinterpret_cast<float*>(workspace_ptr);
  a.jobs = reinterpret_cast<Job*>(workspace_ptr + partial_bytes(b, kv_heads, head_dim));
  a.q_row = q_row_bytes;
  a.q_head = q_head_bytes;
  a.tokens = (unsigned int)tokens;
  a.requests = (unsigned int)requests;
  a.q_heads = (unsigned int)q_heads;
  a.kv_heads = (unsigned int)kv_heads;
  a.group = (unsigned int)(q_heads / kv_heads);
  a.few_rows = 0;
  a.tiles_too = 1;
  a.few_target = (unsigned int)b.few_target;
  a.tile_target = (unsigned int)b.tile_target;
  a.max_query = (unsigned int)max_query;
  a.tile_slots = (unsigned int)tile_slots_of(b, kv_heads);
  a.few_slots = a.few_groups = (unsigned int)(b.few_items * kv_heads);
  a.tile_groups = (unsigned int)(b.tile_items * kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  return launch_typed<false>(a, head_dim, dtype, reinterpret_cast<hipStream_t>(stream_ptr));
}
