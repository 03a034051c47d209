// Causal attention of a step's new tokens over a paged bf16 / fp16 layer, and of whole prompts
// over their own packed K and V rows, gfx950; and attention of rows over all tokens of a source of another
// length (causal 0), in a layer or in packed rows.
//
// For row i of request r (n new tokens, context c): o = sum_t p_t v_t / sum_t p_t over the tokens
// t = 0 .. c - n + i, p_t = 2^(s_t - m), s_t = scale * log2(e) * q.k_t, m a running reference
// kLift to kLift + kSlack below the running maximum of s, so that the sums stay in range and the
// accumulators are rescaled only when the maximum has moved by kSlack.
// Scores, weights' sums and outputs accumulate in f32; the weights are rounded to the inputs'
// type for the second matrix product, as the matrix unit takes it (by at most 2^-8 or 2^-11 of each,
// like the output's own rounding). fp16 has no more than that for values of 2^-14 and above, and steps
// of 2^-24 below, so its weights are kept 2^7 larger (kLift; the largest are then 2^15): those below
// 2^-21 of the largest are off by up to 2^-32 of it, a context of n tokens by n * 2^-32 of its
// largest V value (n * 2^-25 without, which 32768 tokens of weight 2^-26 beside one of 1 lost whole).
// Over sources streamed rows (attention_few, and short requests beside tiles in a layer) lose none of it: what the
// rounding leaves has a product of its own, on matrix units that wait for memory. Tiles do lose it: bf16 prompts over
// sources are off by 0.0021 to 0.0024 of their size, and with weights in f32 by 0.0017, the output's own rounding. The
// second product takes 616 us there in place of 455 (4 prompts over 4386 .. 14280 tokens), 53.8 in place of 46.6 (16
// packed prompts over up to 1912), 14.7 in place of 13.0 (64 rows over 1500), as tiles have neither matrix units that
// wait nor registers to spare.
//
// The query heads of a group read the same K and V, so a request's rows are (token, head of the
// group) pairs, row m = token * group + head, and a tile of rows serves them together: a single
// token is `group` rows, and every K and V byte is read once per tile.
//
// Two kernels, by the rows that a request of the call can have:
//   * attention_few: at most 16 (decode steps). Bound by reading K and V: a wave streams 32 tokens
//     at a time, K straight into the matrix operand's registers, V into LDS for the transposing
//     reads. 32 requests of 8192 tokens, 32 / 8 heads of 128: 191 us for 1.07 GB, 5.6 TB/s.
//   * attention_tiles: more; 256 rows (64-dim heads: 128) by 64 tokens a step, requests of at most 16
//     rows streamed like the others. Bound by the matrix and vector units, and by the clock that the
//     power limit leaves them: a prompt of 16384 tokens, 8 / 1 heads of 128: 475 us, 1.16 PFLOP/s, the
//     matrix units busy 63 % of the cycles at 1.7 GHz (the library's product of 8192^3: 1.29, 69 %);
//     8 of 4096, 32 / 8 heads: 1063 us, 1.03 PFLOP/s; heads of 64 reach 0.86, as they have twice the
//     softmax for each product (VALU active 0.74 of the cycles, matrix units 0.44).
// Over sources the same two: a request's rows, the beams of one token among them, read its source once. 32
// requests of 5 rows, 1500 tokens, 20 heads of 64 in fp16: 53 us for 247 MB; 4 of 659 .. 862 rows over 4386 ..
// 14280 tokens, 32 / 8 heads of 128: 455 to 462 us, 1.01 to 1.03 PFLOP/s, on other cards up to 5 % more (384 tiles of
// 69 to 224 steps on 256 CUs: the longest CU has 259 steps of 227 on average; cut finer, the partials cost more than
// the balance gives).
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
#include <initializer_list>
#include <mutex>
#include <type_traits>

#include "splitzip_common.h"

namespace unchainkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;         // waves of a workgroup of attention_few, two of them on a CU
// Of one of attention_tiles: 8 of 128-dim heads, whose registers and LDS leave room for one workgroup
// on a CU, and 4 of 64-dim heads, of which a CU has three that fill each other's starts and ends (24
// prompts of up to 1247 tokens: 38.9 us, with 8 waves 49.9; 8 x 4096 640 and 709).
constexpr int tile_waves(int D) { return D == 128 ? 8 : 4; }
constexpr int tile_rows(int D) { return 32 * tile_waves(D); }
constexpr int kMergeThreads = 256;
// An odd count, so that the slots of the first splits, which have the work and lie at even distances,
// fall to all of them (32 requests of 8192 tokens: 6.2 us, 11.6 with 1024 workgroups).
constexpr unsigned int kMergeGroups = 1021;
// Rows of a request that is streamed: by attention_few, and by attention_tiles where longer requests
// are beside it (as tiles a chunk of 2048 behind 8192 and 64 single tokens, 32 / 8 heads of 64, take
// 366 us, so 274; 3 chunks and 29 single tokens of 128-dim heads 310 and 298; 64 single tokens and 4
// times 8, heads of 64, 202 and 218). 32 rows, as two sets of 16, gained nothing over tiles.
constexpr int kFewRows = 16;
constexpr int kFewStep = 32;      // tokens of a wave's step in attention_few,
constexpr int kFewUnit = kWaves * kFewStep;  // of a round of its workgroup's: unit of its splits
constexpr int kTileTokens = 64;   // tokens of a step of attention_tiles: unit of its splits
// Steps of a split, at least: its start and its share of the joining take as long as some of them (4
// requests of 64 tokens behind 4000: 39.1 us at 12, 44.8 at 16).
constexpr unsigned int kLeastTileSteps = 12;
// Over sources a tile has no steps that its first rows spare, and shorter splits gain where there are few tiles (one
// request of 64 rows, 1500 tokens, 16 heads of 64: 14.3 us at 4, 20.7 at 12; 4 of 3 rows, 5000 tokens, 7 / 1 heads of
// 128 17.7 and 22.5; 4 of 300, 1500, 32 / 8 heads the same). Of tiles for at most half the CUs sources
// of fewer than kLeastTileSteps are cut too (one of 64 rows, 600 tokens 13.1 and 15.4, 400 tokens 12.8 and 12.4).
constexpr unsigned int kLeastSourceTileSteps = 4, kWholeSourceTileSteps = 8;
// Of a streamed split, in rounds of kFewUnit tokens (4 requests of 4096 tokens, 32 / 8 heads of 128:
// 22.5 us at 4, 24.6 at 1). A call whose block tables hold no more than kWholeFewSteps is not cut at
// all and joins nothing: one launch (one request, 32 / 8 heads of 64, 1024 tokens: 12.6 us, cut 16.8,
// for the host's second submission: captured 10.8 and 11.2; of 128 dims, uncut and cut, 768 tokens 13.7
// and 16.0, 1024 the same, 1536 21.1 and 16.0).
constexpr unsigned int kLeastFewSteps = 4, kWholeFewSteps = 8;
// Sources are mostly of about one length, so that cutting them gains no balance: up to twice that they are taken
// whole where they fill three quarters of the CUs (12 requests of 5 rows, 1500 tokens, 20 heads of 64: 19.3 us and
// 25.0; 30 of one row, 2000 tokens, 32 / 8 heads of 128: 41.9 and 47.1). Of those that leave most CUs idle, at most
// an eighth of them taken, shorter ones are cut, and into more splits, up to 16 of one round (one request, captured:
// 16 heads of 64, 1000 tokens 9.1 us and 11.2, 768 tokens 9.0 and 9.6, 640 tokens 9.0 and 8.8; 32 / 8 heads of 128,
// 1000 tokens 11.4 and 16.4, 512 tokens 11.3 both; 8 requests of the latter, a quarter of the CUs, 2000 tokens 22.1
// and 21.2).
constexpr unsigned int kWholeSourceSteps = 16, kFineSplits = 16;
constexpr unsigned int whole_fine_steps(unsigned long long head_dim) { return head_dim == 64 ? 6 : 4; }
// A maximum before any token: the lowest float, not -inf, so that rows whose scores are all -inf
// have weights of zero and a sum of zero (whose quotient is NaN, as the formula's).
constexpr float kNoMax = -3.402823466e38f;
constexpr float kSlack = 8.f;     // log2: weights stay below 2^(kLift + 8)
constexpr float kLn2 = 0.6931471805599453f;

template <typename E>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static constexpr float kLift = 0.f;  // log2 that the largest weights are raised by
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
  static constexpr float kLift = 7.f;
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
  const int* tables;         // [requests][table_stride]; null: packed rows
  const int* sources;        // [requests], the first packed row of K and V; null: the request's own
  float* partial;            // of each slot
  struct Job* jobs;          // one for each slot
  unsigned long long q_row, q_head;  // bytes from token to token, from head to head
  unsigned long long k_row, k_head, v_row, v_head;
  unsigned long long table_stride;
  unsigned int table_width, blocks, block_tokens;
  Divider by_block;
  unsigned int tokens, requests, q_heads, kv_heads, group;
  unsigned int few_target, tile_target;   // workgroups to split for, of the two paths
  unsigned int tile_least;    // steps of a tile's split, at least
  unsigned int fine;          // 1: streamed splits may be shorter than kLeastFewSteps, up to kFineSplits of a request
  unsigned int max_query;     // requests with more new tokens are left out
  unsigned int max_source;    // and, of packed sources, those with more tokens
  unsigned int kv_rows;       // rows of packed sources
  unsigned int causal;        // 1: row i of n sees the context without its last n - i - 1 tokens; 0: all
  unsigned int slots;         // partial slots
  unsigned int items;         // of the tiles' grid, beside one that clears what slots they leave
  float scale_log2;
};

// One request as its lengths in device memory say, with lengths that cannot be cut down to
// nothing: rows outside the tensor are nobody's, and neither are those of a request that is longer
// than the call allows.
struct Request {
  unsigned int r, start, n, ctx;
  bool bad;  // a context longer than the block table, or rows outside the source
};

__device__ __forceinline__ Request load_request(const AttendArgs& a, unsigned int r) {
  Request q{r, 0, 0, 0, false};
  if (r >= a.requests) return q;
  const int s0 = a.starts[r], s1 = a.starts[r + 1];
  if (s0 < 0 || s1 < s0 || (unsigned int)s1 > a.tokens || (unsigned int)(s1 - s0) > a.max_query)
    return q;
  q.start = (unsigned int)s0;
  q.n = (unsigned int)(s1 - s0);
  q.ctx = q.n;
  if (a.contexts != nullptr) {
    const int c = a.contexts[r];
    q.ctx = c < 0 ? 0u : (unsigned int)c;
    if (a.tables != nullptr) {
      const unsigned long long most = (unsigned long long)a.table_width * a.block_tokens;
      if (q.ctx > most) {
        q.bad = true;
        q.ctx = (unsigned int)most;
      }
    } else if (q.ctx > a.max_source) {
      q.n = q.ctx = 0;
    } else if (q.ctx != 0) {
      const int s = a.sources[r];
      if (s < 0 || (unsigned int)s + q.ctx > a.kv_rows) {
        q.bad = true;
        q.ctx = 0;
      }
    }
  }
  return q;
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

template <int kRows>
__device__ __forceinline__ unsigned int tiles_of(const AttendArgs& a, unsigned int n) {
  return (n * a.group + kRows - 1) / kRows;
}

constexpr unsigned int kNoSlot = ~0u;

// Sums of 64 lanes' values stay below 2^32.
constexpr unsigned int kMostSteps = 1u << 25;

// ceil(sum * heads / parts), or a little more past 2^32 / parts (one 32-bit division serves: every
// workgroup waits for it), but at most kMostSteps: no request that is cut has more. The sum of 2^31
// requests times their heads may pass 64 bits.
__host__ __device__ __forceinline__ constexpr unsigned int share_of(unsigned long long sum,
                                                                    unsigned int heads, unsigned int parts) {
  const unsigned long long all = (sum >> 50) != 0 ? ~0ull : sum * heads + parts - 1;
  if (all >= (unsigned long long)kMostSteps * parts) return kMostSteps;
  const bool wide = (all >> 32) != 0;
  const unsigned int share = (wide ? (unsigned int)(all >> 16) + parts : (unsigned int)all) / parts;
  return wide ? share << 16 : share;
}
static_assert(share_of(0, 8, 192) == 0 && share_of(1, 1, 192) == 1 && share_of(384, 1, 192) == 2 &&
              share_of(385, 1, 192) == 3 && share_of(192u << 20, 8, 192) == 8u << 20, "rounded up");
static_assert(share_of(1ull << 32, 1, 192) * 192ull >= 1ull << 32 &&
              share_of(1ull << 32, 1, 192) < 22500000u &&  // (of 22369622)
              share_of(1ull << 37, 8, 192) == kMostSteps && share_of(1ull << 56, 4096, 512) == kMostSteps &&
              share_of((1ull << 50) - 1, 4096, 512) == kMostSteps, "the share, or what cuts nothing");

// The launch's work, which every workgroup finds its own item of by itself. Requests lie one in a
// lane, 64 at a time (`first`: the first 64, which most launches end with), each with its tiles
// (streaming: one) of `steps` steps of kStep tokens. A request of more than `cap` steps, the even
// share of all tiles' steps over the workgroups to split for, is cut into the fewest splits of at
// most that, all of about one length. A cut tile has at least two, so that all cut tiles together
// have at most twice (all steps / cap) splits, in as many slots, and at most (all steps / cap) more
// than there are tiles.
template <bool kTiles, int kRows, bool kStream>
struct Work {
  static constexpr unsigned int kStep = kTiles ? kTileTokens : kFewUnit;
  const AttendArgs& a;
  Request first;
  unsigned int cap;  // steps of a split, at most; 0: nothing is cut

  // whether a request of n tokens is streamed
  __device__ __forceinline__ bool few(unsigned int n) const {
    return !kTiles || (kStream && n * a.group <= kFewRows);
  }
  __device__ __forceinline__ unsigned int tiles(const Request& q) const {
    return few(q.n) ? (q.n != 0 ? 1u : 0u) : tiles_of<kRows>(a, q.n);
  }
  __device__ __forceinline__ unsigned int steps(const Request& q) const {
    return steps_of(q.ctx, kStep);
  }
  __device__ __forceinline__ unsigned int splits(const Request& q) const {
    return cap == 0 ? 1u : max(1u, steps_of(steps(q), cap));
  }
  // tokens of a split of a request in `splits`
  __device__ __forceinline__ unsigned int split_tokens(const Request& q, unsigned int splits) const {
    return steps_of(steps(q), splits) * kStep;
  }
  __device__ __forceinline__ Request requests(unsigned int r0) const {
    return r0 == 0 ? first : load_request(a, r0 + __lane_id());
  }

  __device__ __forceinline__ explicit Work(const AttendArgs& args)
      : a(args), first(load_request(args, __lane_id())), cap(0) {
    if (kTiles && a.requests > 1 && a.requests <= kWave) sort();
    unsigned long long sum = 0;
    bool large = false;
    for (unsigned int r0 = 0; r0 < a.requests; r0 += kWave) {
      const Request q = requests(r0);
      const unsigned int t = tiles(q);
      const unsigned long long own = (unsigned long long)t * steps(q);
      large |= __ballot(own > kMostSteps) != 0;
      sum += lane_value(wave_scan((unsigned int)min(own, (unsigned long long)kMostSteps)), 63);
    }
    const unsigned int parts = kTiles ? a.tile_target : a.few_target;
    unsigned int least = kTiles ? a.tile_least : kLeastFewSteps;
    if (!kTiles && a.fine != 0)
      least = (unsigned int)min((unsigned long long)least, sum / (kFineSplits * a.requests) + 1);
    if (!large && a.slots != 0) cap = max(least, share_of(sum, a.kv_heads, parts));
  }

  // The lanes' requests with the longest contexts first.
  __device__ __forceinline__ void sort() {
    const unsigned int lane = __lane_id();
    const unsigned int key = min(first.n != 0 ? steps(first) + 1 : 0u, kMostSteps) << 6 | (63 - lane);
    unsigned int rank = 0;
    for (unsigned int j = 0; j < a.requests; ++j) rank += lane_value(key, (int)j) > key ? 1u : 0u;
    const int to = 4 * (int)(lane < a.requests ? rank : lane);
    first.r = (unsigned int)__builtin_amdgcn_ds_permute(to, (int)first.r);
    first.start = (unsigned int)__builtin_amdgcn_ds_permute(to, (int)first.start);
    first.n = (unsigned int)__builtin_amdgcn_ds_permute(to, (int)first.n);
    first.ctx = (unsigned int)__builtin_amdgcn_ds_permute(to, (int)first.ctx);
    first.bad = __builtin_amdgcn_ds_permute(to, first.bad ? 1 : 0) != 0;
  }

  // Item `item`: its request, its index among the request's items (splits of one tile beside each
  // other), whether it has a slot (where the request is cut; streaming: always), and the slots that
  // the items before it have, whose number is its own. False past the last one. All wave-uniform.
  __device__ __forceinline__ bool find(unsigned int item, Request& q, unsigned int& index,
                                       bool& has_slot, unsigned int& slot) const {
    unsigned long long before = 0, slots = 0;
    for (unsigned int r0 = 0; r0 < a.requests; r0 += kWave) {
      const Request l = requests(r0);
      const unsigned int parts = splits(l), own = tiles(l) * parts, sum = wave_scan(own);
      const unsigned int slot_own = !kTiles || parts > 1 ? own : 0u, slot_sum = wave_scan(slot_own);
      const unsigned int all = lane_value(sum, 63);
      if (item < before + all) {
        const unsigned int in = item - (unsigned int)before;
        const int at = __ffsll((long long)__ballot(sum > in)) - 1;
        index = in - lane_value(sum - own, at);
        q.r = lane_value(l.r, at);
        q.start = lane_value(l.start, at);
        q.n = lane_value(l.n, at);
        q.ctx = lane_value(l.ctx, at);
        q.bad = lane_value(l.bad ? 1u : 0u, at) != 0;
        has_slot = lane_value(slot_own, at) != 0;
        slot = (unsigned int)slots + lane_value(slot_sum - slot_own, at) + (has_slot ? index : 0u);
        return true;
      }
      before += all;
      slots += lane_value(slot_sum, 63);
    }
    slot = (unsigned int)min(slots, (unsigned long long)kNoSlot);
    return false;
  }
};

// What a kernel's rows see: their own request's context up to themselves, or all tokens of a source. (Kernels of
// their own: one for both, told by an argument, took 18 registers more for streamed rows of 64 dims; 3 chunks beside
// 29 single tokens 293 us and now 288, 4 prompts over 4386 .. 14280 tokens of sources 471 and 463, 16 requests of
// up to 6 rows 34.4 and 33.9.)
enum Sight { kOwnContext, kWholeSource };

// The last token of a request that its first row sees (negative: none).
template <Sight kSight>
__device__ __forceinline__ int first_seen(const Request& q) {
  return (int)q.ctx - (int)(kSight == kOwnContext ? q.n : 1u);
}

// The first row of K and V of a request of packed rows.
template <bool kPaged, Sight kSight>
__device__ __forceinline__ unsigned int kv_start(const AttendArgs& a, const Request& q) {
  if constexpr (kPaged) return 0;
  if constexpr (kSight == kOwnContext) return q.start;
  return q.ctx == 0 ? 0u : (unsigned int)a.sources[q.r];
}

// Row of K and V that token t of a request has: its place in the layer through the block table
// (bad: the table names no block of the layer there; block 0 is read instead), or its packed row.
template <bool kPaged>
__device__ __forceinline__ unsigned int kv_row(const AttendArgs& a, unsigned int start,
                                               unsigned int t, int id, unsigned int& bad) {
  if constexpr (kPaged) {
    const unsigned int blk = div_u32(t, a.by_block.m, a.by_block.d);
    const bool ok = (unsigned int)id < a.blocks;
    bad |= ok ? 0u : 1u;
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
    unsigned int bad = 0;
    const unsigned int row = kv_row<kPaged>(a, start, own, block_id<kPaged>(a, table, own), bad);
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

// Whether any lane of the workgroup has it, through `space` in LDS.
__device__ __forceinline__ bool any_lane(unsigned int has, unsigned char* space) {
  unsigned int* const flag = reinterpret_cast<unsigned int*>(space);
  __syncthreads();
  if (threadIdx.x == 0) *flag = 0;
  __syncthreads();
  if (has) *flag = 1;
  __syncthreads();
  return *flag != 0;
}

// Where a row's result goes: the output (of one split), or its place among the partials, a
// slot's rows as (m, l) pairs and then their D sums.
template <int D, int kRows>
__device__ __forceinline__ float* slot_ml(const AttendArgs& a, unsigned int slot) {
  return a.partial + (unsigned long long)slot * (kRows * (D + 2));
}
template <int D, int kRows>
__device__ __forceinline__ float* slot_acc(const AttendArgs& a, unsigned int slot) {
  return slot_ml<D, kRows>(a, slot) + 2 * kRows;
}

// A row (m, l, sums) by a wave whose lanes hold D / 64 sums each, from slow_row.
template <typename E, int D, int kRows>
__device__ __forceinline__ void store_slow(const AttendArgs& a, bool split,
                                           unsigned int slot, unsigned int slot_row,
                                           unsigned long long out_row, bool none, float m, float l,
                                           const float (&acc)[D / 64]) {
  const unsigned int lane = __lane_id();
  if (split) {
    float* ml = slot_ml<D, kRows>(a, slot) + 2 * slot_row;
    float* dst = slot_acc<D, kRows>(a, slot) + slot_row * D;
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

// A slot's job, by one thread of its workgroup; `slot` counts for one KV head. (Row ranges that
// overlap each other can ask for more slots than there are: rows without theirs stay as they were.)
__device__ __forceinline__ void store_job(const AttendArgs& a, unsigned int slot, unsigned int head,
                                          Job j) {
  const unsigned int slots = a.slots / a.kv_heads;
  if (threadIdx.x != 0 || slot >= slots) return;
  if (slot + (unsigned long long)j.splits > slots) j.splits = 0;
  a.jobs[slot * a.kv_heads + head] = j;
}
// Nothing to join in the slots from `slot` on, by the workgroup.
__device__ __forceinline__ void clear_jobs(const AttendArgs& a, unsigned int slot, unsigned int head) {
  for (unsigned long long s = (unsigned long long)slot + threadIdx.x; s < a.slots / a.kv_heads; s += blockDim.x)
    a.jobs[s * a.kv_heads + head] = Job{};
}

// ---------------------------------------------------------------------------
// 32 rows a wave by 64 tokens a step

// Lane l of a wave has row l % 32 of the wave's 32 and, of every 16 tokens, those with
// (token / 4) % 2 == l / 32 (the 32x32 matrix instruction's output rows). K lies in LDS as rows
// of D values, V too, both with their 16-byte pieces exchanged within a row so that the lanes of
// one read spread over the banks: K's piece c of row t at c ^ (t % 16), read 16 bytes a lane by 32
// rows; V's 64-byte quarters q at q ^ (t % 4), read transposed 8 bytes a lane, 4 tokens by 32 dims
// per half wave.
template <typename E, int D, bool kPaged, bool kRuns, Sight kSight>
__device__ __forceinline__ void tile_path(const AttendArgs& a, const Request& request,
                                          unsigned int order, unsigned int split, unsigned int most,
                                          unsigned int split_tokens, bool whole, unsigned int slot,
                                          unsigned int head, unsigned char* s0, unsigned char* s1,
                                          unsigned char* s2) {
  typedef typename Elem<E>::x8 x8;
  constexpr int kRowBytes = 2 * D, kPieces = kRowBytes / 16;  // pieces of a row
  constexpr int kRowsPerLoad = kWave / kPieces, kLoads = 8 / kRowsPerLoad;
  constexpr int kTileBytes = kTileTokens * kRowBytes;
  constexpr int kSlabs = D / 16, kDimTiles = D / 32;
  constexpr int kN = tile_waves(D), kTileRows = tile_rows(D);
  constexpr int kOwn = kTileTokens / kN, kOwnRuns = kOwn / 8;  // a wave's tokens of a tile's loads

  const unsigned int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const unsigned int half = lane / 32, col = lane % 32;
  // the tiles with the longest contexts first
  const unsigned int tile = tiles_of<kTileRows>(a, request.n) - 1 - order;
  const unsigned int rows = request.n * a.group;
  const unsigned int m0 = tile * kTileRows;
  constexpr unsigned int kMore = kSight == kOwnContext ? 1 : 0;  // tokens that each row sees beside the one before it
  // last visible token of a row (negative: none)
  const int shift = first_seen<kSight>(request);
  const int last_of_tile = shift + (int)(kMore * ((min(rows, m0 + kTileRows) - 1) / a.group));
  const unsigned int seen = last_of_tile < 0 ? 0u : (unsigned int)last_of_tile + 1;
  const unsigned int splits = most == 1 ? 1u : max(1u, steps_of(seen, split_tokens));  // of this tile
  if (most > 1)
    store_job(a, slot, head,
              Job{request.start, m0, shift, (unsigned short)min(rows - m0, (unsigned int)kTileRows),
                  (unsigned short)(split == 0 && splits > 1 && whole ? splits : 0u)});
  if (split >= splits) return;
  slot = slot * a.kv_heads + head;
  const unsigned int t_begin = split * split_tokens;
  const unsigned int t_end = splits == 1 ? seen : min(seen, t_begin + split_tokens);
  const unsigned int mw = m0 + wave * 32, m = mw + col;
  const bool valid = m < rows;
  const unsigned int token = valid ? m / a.group : 0u;
  const unsigned int q_head = head * a.group + (valid ? m - token * a.group : 0u);
  const int limit = valid ? shift + (int)(kMore * token) : -1;
  // the last visible token of the wave's first row
  const int first_limit = shift + (int)(kMore * (mw / a.group));
  const unsigned int source = kv_start<kPaged, kSight>(a, request);

  const int* table = kPaged ? a.tables + request.r * a.table_stride : nullptr;
  const unsigned char* kb = a.k + head * a.k_head;
  const unsigned char* vb = a.v + head * a.v_head;
  unsigned int bad = request.bad ? 1u : 0u;

  // the row's query as the second operand: dims 16 s + 8 half .. + 7 of slab s (a lane without a
  // row has the request's first: a column of the products that nobody reads)
  x8 q[kSlabs];
  const unsigned char* q_row = a.q + (unsigned long long)(request.start + token) * a.q_row +
                               (unsigned long long)q_head * a.q_head;
#pragma unroll
  for (int s = 0; s < kSlabs; ++s) {
    q[s] = *reinterpret_cast<const x8*>(q_row + 32 * s + 16 * half);
  }

  // This wave's share of a tile's loads: kOwn tokens of K and V, in runs of 8. Where a run's follow
  // each other in memory (prompts; layers whose blocks are whole groups of 8 tokens) the wave forms
  // their address once, on the scalar unit, and a lane's offsets from it never change.
  const unsigned int piece = lane % kPieces, sub = lane / kPieces;
  unsigned int k_off[kOwnRuns][kLoads], v_off[kOwnRuns][kLoads];
#pragma unroll
  for (int u = 0; u < kOwnRuns; ++u)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const unsigned int in = i * kRowsPerLoad + sub;                // the token's place in its run
      const unsigned int at = (kOwn * wave + 8 * u) % 16 + in;       // and among 16
      const unsigned int k_piece = piece ^ (D == 128 ? at : (at >> 1) & 7);
      const unsigned int v_piece = piece ^ (D == 128 ? (at & 3) << 2 : ((at >> 1) & 1) << 2);
      k_off[u][i] = (kRuns ? in * (unsigned int)a.k_row : 0u) + 16 * k_piece;
      v_off[u][i] = (kRuns ? in * (unsigned int)a.v_row : 0u) + 16 * v_piece;
    }
  constexpr int kIds = kRuns ? kOwnRuns : kOwnRuns * kLoads;
  const unsigned int first_at = wave * kOwn * kRowBytes;
  auto token_of = [&](unsigned int base, int i) {
    return min(base + wave * kOwn + (kRuns ? 8 * i : i * kRowsPerLoad + sub), t_end - 1);
  };
  int ids[kIds];               // of the tile whose K is loaded next
  unsigned int next_row[kIds], row_of[kIds];  // of that tile, and of the one whose V is
  // (by a lane's index of zero, which the compiler cannot see through: a scalar load would not be
  // among the vector loads that the waits below count)
  unsigned int zero = 0;
  if constexpr (kPaged) asm("v_mov_b32 %0, 0" : "=v"(zero));
  auto fetch_ids = [&](unsigned int base) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) ids[i] = block_id<kPaged>(a, table + zero, token_of(base, i));
  };
  auto find_rows = [&](unsigned int base) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      next_row[i] = kv_row<kPaged>(a, source, token_of(base, i), ids[i], bad);
      if (kRuns) next_row[i] = uniform(next_row[i]);
    }
  };
  // Sizes of the buffers of a run's rows (kRuns): whole tiles lie inside the tensor, the last one
  // ends with the tokens, and one behind it has none.
  const unsigned int last_base = t_end == 0 ? 0u : (t_end - 1 - t_begin) / kTileTokens * kTileTokens + t_begin;
  unsigned int k_last[kOwnRuns], v_last[kOwnRuns];
#pragma unroll
  for (int u = 0; u < kOwnRuns; ++u) {
    const int left = (int)t_end - (int)(last_base + wave * kOwn + 8 * u);
    const unsigned int last_rows = uniform((unsigned int)max(min(left, 8), 0));
    k_last[u] = last_rows == 0 ? 0u : (last_rows - 1) * (unsigned int)a.k_row + kRowBytes;
    v_last[u] = last_rows == 0 ? 0u : (last_rows - 1) * (unsigned int)a.v_row + kRowBytes;
  }
  auto load_plane = [&](unsigned int base, const unsigned char* src, unsigned long long stride,
                        const unsigned int (&last_bytes)[kOwnRuns], const unsigned int (&row)[kIds],
                        const unsigned int (&off)[kOwnRuns][kLoads], unsigned char* dst) {
    const unsigned int inside = base < last_base ? 0x7FFFFFFFu : 0u;
    const unsigned int at_last = base == last_base ? 0x7FFFFFFFu : 0u;
#pragma unroll
    for (int u = 0; u < kOwnRuns; ++u)
      if constexpr (kRuns) {
        const unsigned int bytes = inside | (at_last & last_bytes[u]);
        const Buffer buffer = buffer_of(src + row[u] * stride, bytes);
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          load_to_lds(buffer, off[u][i], dst + first_at + (8 * u + i * kRowsPerLoad) * kRowBytes);
      } else {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          load_to_lds(src + row[u * kLoads + i] * stride + off[u][i],
                      dst + first_at + (8 * u + i * kRowsPerLoad) * kRowBytes);
      }
  };
  // The loads of a round in three steps: K of the tile behind `base`, V of the tile there. (Tokens
  // past the end are outside the buffers, or the last one again.)
  constexpr int kInFlight = 2 * kOwnRuns * kLoads + (kPaged ? kIds : 0);  // a round's
  auto load_step = [&](int j, unsigned int base, unsigned char* to) {
    if (j == 0) {
      find_rows(base + kTileTokens);
      fetch_ids(base + 2 * kTileTokens);  // (before the loads, which the next round then does not wait for)
    } else if (j == 1) {
      load_plane(base + kTileTokens, kb, a.k_row, k_last, next_row, k_off, to);
    } else if (j == 2) {
      load_plane(base, vb, a.v_row, v_last, row_of, v_off, to + kTileBytes);
#pragma unroll
      for (int i = 0; i < kIds; ++i) row_of[i] = next_row[i];
    }
  };

  f32x16 o[kDimTiles];
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m_ref = kNoMax, l_run = 0.f;
  f32x16 s[2];  // scores of a tile
  x8 w[4];      // its weights,
  f32x16 late;  // and the exponents of those that its products of O begin with computing

  // K operand: row col (+ 32), piece 2 s + half; V operand: tokens 4 half + i / 4 (i = lane % 16) of
  // 16, dims 16 (lane / 16 % 2) + 4 (i % 4) of 32
  const unsigned int k_at = col * kRowBytes, k_x = D == 128 ? col & 15 : (col >> 1) & 7;
  const unsigned int v_tok = 4 * half + (lane % 16) / 4;
  const unsigned int v_x = D == 128 ? v_tok & 3 : (v_tok >> 1) & 1;
  const unsigned int v_at = v_tok * kRowBytes + 32 * ((lane / 16) % 2) + 8 * (lane % 4);

  // The weights of the second half of a tile's tokens: value j of 16.
  float late_sum = 0.f, pair = 0.f;
  auto late_weight = [&](int j) {
    const float e = __builtin_amdgcn_exp2f(late[j]);
    late_sum += e;
    if (j % 2 == 0) {
      pair = e;
    } else {
      u32x4 x = __builtin_bit_cast(u32x4, w[2 + j / 8]);
      x[j % 8 / 2] = pack2<E>(pair, e);
      w[2 + j / 8] = __builtin_bit_cast(x8, x);
    }
  };
  // Products of a phase, each with its operand read from LDS: first those of S (16 dims, 32 tokens,
  // the halves in turns), with the late weights of the tile before between them, then those of its
  // O (16 tokens, 32 dims); each operand is read kAhead products before its own, in this order (left
  // to itself the compiler waits for each read just issued).
  constexpr int kOuts = 4 * kDimTiles, kScores = 2 * kSlabs, kAhead = D == 128 ? 4 : 2;
  auto operand = [&](int i, const unsigned char* bv, const unsigned char* bk) {
    if (i < kScores)
      return *reinterpret_cast<const x8*>(bk + k_at + 32 * (i % 2) * kRowBytes +
                                          16 * ((2 * (i / 2) + half) ^ k_x));
    i -= kScores;
    const unsigned char* src =
        bv + v_at + 16 * (i / kDimTiles) * kRowBytes + 64 * ((i % kDimTiles) ^ v_x);
    const u32x2 lo = read_transposed(src), hi = read_transposed(src + 8 * kRowBytes);
    return __builtin_bit_cast(x8, u32x4{lo.x, lo.y, hi.x, hi.y});
  };
  auto product = [&](int i, x8 f) {
    if (i < kScores) {
      f32x16 zero;
#pragma unroll
      for (int j = 0; j < 16; ++j) zero[j] = 0.f;
      s[i % 2] = Elem<E>::mma32(f, q[i / 2], i < 2 ? zero : s[i % 2]);
    } else {
      i -= kScores;
      o[i % kDimTiles] = Elem<E>::mma32(f, w[i / kDimTiles], o[i % kDimTiles]);
    }
  };
  auto products = [&](auto first, auto count, const unsigned char* from, auto between) {
    constexpr int kFirst = decltype(first)::value, kCount = decltype(count)::value;
    x8 f[kCount];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = operand(kFirst + i, from + kTileBytes, from);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < kCount) f[i + kAhead] = operand(kFirst + i + kAhead, from + kTileBytes, from);
      product(kFirst + i, f[i]);
      between(i);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto scores = [&](const unsigned char* from) {
    products(std::integral_constant<int, 0>(), std::integral_constant<int, kScores>(), from, [](int) {});
  };
  auto both = [&](const unsigned char* from) {
    products(std::integral_constant<int, 0>(), std::integral_constant<int, kScores + kOuts>(), from,
             [&](int i) {
               if (i >= kScores) return;
#pragma unroll
               for (int j = 0; j < 16 / kScores; ++j) late_weight(16 / kScores * i + j);
             });
    l_run += late_sum;
    late_sum = 0.f;
  };
  auto outputs = [&](const unsigned char* from) {
#pragma unroll
    for (int j = 0; j < 16; ++j) late_weight(j);
    products(std::integral_constant<int, kScores>(), std::integral_constant<int, kOuts>(), from,
             [](int) {});
    l_run += late_sum;
    late_sum = 0.f;
  };
  // (the loads are spread over it: each takes its time to be issued)
  auto softmax = [&](unsigned int base, auto between) {
    if ((int)base + kTileTokens - 1 > first_limit) {
      const int left = limit - (int)base - 4 * (int)half;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[t][i] = 32 * t + 8 * (i / 4) + i % 4 <= left ? s[t][i] : -INFINITY;
    }
    between(0);
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    {
      const unsigned int u = __builtin_bit_cast(unsigned int, top);
      const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      top = fmaxf(__builtin_bit_cast(float, (unsigned int)x[0]),
                  __builtin_bit_cast(float, (unsigned int)x[1]));
    }
    top *= a.scale_log2;
    if (__ballot(top > m_ref + (Elem<E>::kLift + kSlack)) != 0) {
      const float now = fmaxf(m_ref, top - Elem<E>::kLift), alpha = __builtin_amdgcn_exp2f(m_ref - now);
      m_ref = now;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) late[i] = fmaf(s[1][i], a.scale_log2, -m_ref);
    __builtin_amdgcn_sched_barrier(0);
    between(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float e[8], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[0][8 * c + i], a.scale_log2, -m_ref));
        sum += e[i];
      }
      l_run += sum;
      w[c] = pack8<E>(e);
      if (c == 0) {
        __builtin_amdgcn_sched_barrier(0);
        between(2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  const unsigned int count = (t_end - min(t_begin, t_end) + kTileTokens - 1) / kTileTokens;
  if (count != 0) {
    const unsigned int base_end = t_begin + count * kTileTokens;
    // Round i in two phases, a barrier behind each; waves 0-3 (one on each SIMD) do their products
    // in the first, O of tile i - 1 and S of tile i, and the softmax of tile i in the second; waves
    // 4-7 are a phase behind, so that the matrix unit of every SIMD has one wave's products while
    // the vector unit has the other's softmax. Tile i's K lies in buffer i % 3 and its V in buffer
    // (i + 1) % 3, so that a round reads one buffer; K of tile i + 2 and V of tile i + 1 are loaded in
    // round i (with the softmax) into the one that round i - 1 read, and have landed at the end of
    // the next round.
    auto load = [&](unsigned int base, unsigned char* to) {
#pragma unroll
      for (int j = 0; j < 3; ++j) load_step(j, base, to);
    };
    // (4 waves: each SIMD's other wave is of the workgroup beside it, and a round has one barrier)
    auto phase_end = [&](bool always) {
      if (!always && kN == 4) return;
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    // rounds 1 .. count - 1: the round's tile, the buffer it reads and the one it loads
    auto rounds = [&](auto one) {
      for (unsigned int base = t_begin + kTileTokens; base < base_end;) {
        one(base, s1, s0);
        base += kTileTokens;
        if (base >= base_end) break;
        one(base, s2, s1);
        base += kTileTokens;
        if (base >= base_end) break;
        one(base, s0, s2);
        base += kTileTokens;
      }
    };
    const unsigned char* const last = count % 3 == 0 ? s0 : count % 3 == 1 ? s1 : s2;
    auto with_loads = [&](unsigned int base, unsigned char* to) {
      return [&, base, to](int j) { load_step(j, base, to); };
    };
    fetch_ids(t_begin);
    find_rows(t_begin);
    load_plane(t_begin, kb, a.k_row, k_last, next_row, k_off, s0);
#pragma unroll
    for (int i = 0; i < kIds; ++i) row_of[i] = next_row[i];
    fetch_ids(t_begin + kTileTokens);
    load(t_begin, s1);
    wait_loads<kInFlight>();
    phase_end(true);
    if (mw >= rows) {
      // a wave without rows
      auto idle = [&](unsigned int base, const unsigned char*, unsigned char* to) {
        load(base + kTileTokens, to);
        phase_end(false);
        wait_loads<kInFlight>();
        phase_end(true);
      };
      idle(t_begin, s0, s2);
      rounds(idle);
      phase_end(false);
      phase_end(true);
    } else if (kN == 4 || wave < 4) {
      scores(s0);
      phase_end(false);
      softmax(t_begin, with_loads(t_begin + kTileTokens, s2));
      wait_loads<kInFlight>();
      phase_end(true);
      rounds([&](unsigned int base, const unsigned char* from, unsigned char* to) {
        both(from);
        phase_end(false);
        softmax(base, with_loads(base + kTileTokens, to));
        wait_loads<kInFlight>();
        phase_end(true);
      });
      outputs(last);
      phase_end(false);
      phase_end(true);
    } else {
      load(t_begin + kTileTokens, s2);
      phase_end(true);
      scores(s0);
      wait_loads<kInFlight>();
      phase_end(true);
      rounds([&](unsigned int base, const unsigned char* from, unsigned char* to) {
        softmax(base - kTileTokens, with_loads(base + kTileTokens, to));
        phase_end(true);
        both(from);
        wait_loads<kInFlight>();
        phase_end(true);
      });
      softmax(base_end - kTileTokens, [](int) {});
      phase_end(true);
      outputs(last);
      phase_end(true);
    }
    wait_loads<0>();
  }

  bad = any_lane(bad, s2);
  l_run += __shfl_xor(l_run, 32, 64);
  float check = l_run * 0.f;
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) check = fmaf(o[d][i], 0.f, check);
  check += __shfl_xor(check, 32, 64);
  const bool again = valid && !bad && !(check == 0.f);
  const unsigned long long out_row = (unsigned long long)(request.start + token) * a.q_heads + q_head;
  if (bad) m_ref = l_run = NAN;
  if (valid && !again) {
    if (splits > 1) {
      float* ml = slot_ml<D, kTileRows>(a, slot) + 2 * (m - m0);
      float* dst = slot_acc<D, kTileRows>(a, slot) + (m - m0) * D;
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
    const unsigned int own = (unsigned int)max(shift + (int)(kMore * tok) + 1, 0);  // tokens it sees
    float rm, rl, acc[D / 64];
    slow_row<E, D, kPaged>(a, table, source,
                           a.q + (unsigned long long)(request.start + tok) * a.q_row +
                               (unsigned long long)qh * a.q_head,
                           head, t_begin, min(t_end, own), rm, rl, acc);
    store_slow<E, D, kTileRows>(a, splits > 1, slot, row_m - m0,
                     (unsigned long long)(request.start + tok) * a.q_heads + qh, own == 0, rm, rl, acc);
  }
}

// ---------------------------------------------------------------------------
// at most 16 rows, streaming

// Lane l has row l % 16 and, of every 16 tokens, the four from 4 (l / 16) on. A wave's step is 32
// tokens: K as the first operand of S^T = K Q^T straight from memory, V through the wave's own LDS,
// without a barrier, with 32-byte pieces of row t at piece ^ (t % 8), so that the 16 tokens of a
// transposed read spread over the banks. The kN waves of a workgroup take turns at 32 tokens of a
// split and join their sums in LDS (s0, s1: the waves' stages, and then s0 their sums; s2: their
// (m, l)). kRows: of a slot.
//
// K's rows of 256 bytes (128 dims) are loaded whole, four of them by one load: lane l has piece l % 4
// of the 64 bytes at 64 (l / 16), of token 4 (l % 16 / 4) + j for load j. The operand's "rows" are
// then pieces of four tokens, of which only those that meet their own piece of Q count: four
// products of a load, with Q's pieces c = 0 .. 3, give token 4 (l / 16) + j's score as the sum of their
// elements c. Three of four results are thrown away, on matrix units that have nothing else to do, and
// no load takes apart 16 rows: 32 requests of 8192 tokens 200 -> 196.6 us, 16 of 1024 19.2 -> 17.6, 64
// single tokens of 500 .. 16000 and four times 8 354 -> 332. (64 dims: lane l has token l % 16, 16
// bytes at 16 (l / 16) of every 64, each counting.)
// Of 64-dim sources (kWholeSource) a load takes eight whole rows: lane l has piece 4 (l
// % 2) + l / 16 of token 16 u + 4 (l % 16 / 4) + 2 s + l / 2 % 2 for load (u, s); its product with the pieces
// 0 .. 3 of Q counts in even rows of the result and that with 4 .. 7 in odd ones: 32 requests of 5 rows, 1500
// tokens, 20 heads 55.5 -> 53.9 us, 64 of one row, 100 .. 16000 tokens, 32 / 8 heads 118 -> 113.
template <typename E, int D, int kN, int kRows, bool kPaged, Sight kSight>
__device__ __forceinline__ void few_path(const AttendArgs& a, const Request& request, unsigned int split,
                                         unsigned int splits, unsigned int split_tokens, bool whole,
                                         unsigned int slot, unsigned int head, unsigned char* __restrict__ s0,
                                         unsigned char* __restrict__ s1,
                                         unsigned char* __restrict__ s2) {
  typedef typename Elem<E>::x8 x8;
  constexpr int kRowBytes = 2 * D, kPieces = kRowBytes / 16;
  constexpr int kRowsPerLoad = kWave / kPieces, kLoads = kFewStep / kRowsPerLoad;
  constexpr int kStageBytes = kFewStep * kRowBytes;
  constexpr int kSlabs = D / 32, kDimTiles = D / 16;
  constexpr unsigned int kRound = kN * kFewStep;
  constexpr bool kWhole = D == 128, kHalves = D == 64 && kSight == kWholeSource;  // rows of K are loaded whole
  static_assert(kStageBytes >= kFewRows * D * 4, "a wave's sums fit its stage");

  const unsigned int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const unsigned int col = lane % 16, grp = lane / 16;
  constexpr unsigned int kMore = kSight == kOwnContext ? 1 : 0;  // tokens that each row sees beside the one before it
  store_job(a, slot, head,
            Job{request.start, 0, first_seen<kSight>(request),
                (unsigned short)(request.n * a.group),
                (unsigned short)(split == 0 && splits > 1 && whole ? splits : 0u)});
  slot = slot * a.kv_heads + head;
  const unsigned int rows = request.n * a.group;
  const unsigned int t_begin = split * split_tokens;
  const unsigned int t_end = splits == 1 ? request.ctx : min(request.ctx, t_begin + split_tokens);
  const int shift = first_seen<kSight>(request);
  const unsigned int source = kv_start<kPaged, kSight>(a, request);

  const int* table = kPaged ? a.tables + request.r * a.table_stride : nullptr;
  const unsigned char* kb = a.k + head * a.k_head;
  const unsigned char* vb = a.v + head * a.v_head;
  unsigned int bad = request.bad ? 1u : 0u;

  const bool valid = col < rows;
  const unsigned int token = valid ? col / a.group : 0u;
  const unsigned int q_head = head * a.group + (valid ? col - token * a.group : 0u);
  const int limit = valid ? shift + (int)(kMore * token) : -1;
  x8 q[kSlabs];
  const unsigned char* q_row = a.q + (unsigned long long)(request.start + token) * a.q_row +
                               (unsigned long long)q_head * a.q_head;
#pragma unroll
  for (int s = 0; s < kSlabs; ++s)
    q[s] = *reinterpret_cast<const x8*>(q_row + (kWhole ? 64 * grp + 16 * s : 64 * s + 16 * grp));

  struct Keys {
    u32x4 v[2][kSlabs];
  };
  unsigned char* const stage0 = s0 + wave * kStageBytes;
  unsigned char* const stage1 = s1 + wave * kStageBytes;
  const unsigned int piece = lane % kPieces, sub = lane / kPieces;
  // lane l looks up token l % 32 of a step
  auto token_of = [&](unsigned int base) { return min(base + lane % 32, t_end - 1); };
  auto issue = [&](unsigned int base, int id, Keys& k, unsigned char* stage) {
    const unsigned int row = kv_row<kPaged>(a, source, token_of(base), id, bad);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (kWhole) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          k.v[u][j] = *reinterpret_cast<const u32x4*>(
              kb + (unsigned int)__shfl(row, 16 * u + 4 * (int)(col / 4) + j, kWave) * a.k_row + 64 * grp +
              16 * (col % 4));
      } else if constexpr (kHalves) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
          k.v[u][s] = *reinterpret_cast<const u32x4*>(
              kb + (unsigned int)__shfl(row, 16 * u + 4 * (int)(col / 4) + 2 * s + (int)(col / 2 % 2), kWave) *
                       a.k_row + 64 * (col % 2) + 16 * grp);
      } else {
        const unsigned char* src = kb + (unsigned int)__shfl(row, 16 * u + (int)col, kWave) * a.k_row;
#pragma unroll
        for (int s = 0; s < kSlabs; ++s)
          k.v[u][s] = *reinterpret_cast<const u32x4*>(src + 64 * s + 16 * grp);
      }
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
      if constexpr (kWhole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4 part[4];
#pragma unroll
          for (int c = 0; c < 4; ++c)
            part[c] = Elem<E>::mma16(__builtin_bit_cast(x8, k.v[u][j]), q[c], f32x4{0, 0, 0, 0});
          s[4 * u + j] = (part[0][0] + part[1][1]) + (part[2][2] + part[3][3]);
        }
      } else if constexpr (kHalves) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const x8 rows8 = __builtin_bit_cast(x8, k.v[u][c]);
          const f32x4 even = Elem<E>::mma16(rows8, q[0], f32x4{0, 0, 0, 0});
          const f32x4 odd = Elem<E>::mma16(rows8, q[1], f32x4{0, 0, 0, 0});
          s[4 * u + 2 * c] = even[0] + odd[1];
          s[4 * u + 2 * c + 1] = even[2] + odd[3];
        }
      } else {
        f32x4 st = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kSlabs; ++c)
          st = Elem<E>::mma16(__builtin_bit_cast(x8, k.v[u][c]), q[c], st);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * u + j] = st[j];
      }
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
    if (__ballot(top > m_ref + (Elem<E>::kLift + kSlack)) != 0) {
      const float now = fmaxf(m_ref, top - Elem<E>::kLift), alpha = __builtin_amdgcn_exp2f(m_ref - now);
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
    if constexpr (kSight == kOwnContext) {
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d) {
        const unsigned char* src = bv + 32 * (d ^ v_x);
        const u32x2 lo = read_transposed(src), hi = read_transposed(src + 16 * kRowBytes);
        o[d] = Elem<E>::mma16(__builtin_bit_cast(x8, u32x4{lo.x, lo.y, hi.x, hi.y}), w, o[d]);
      }
    } else {
      // (sources: what the rounding of the weights leaves, so that the output's rounding is the only one of its size)
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] -= (float)w[j];
      const x8 rest = pack8<E>(e);
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d) {
        const unsigned char* src = bv + 32 * (d ^ v_x);
        const u32x2 lo = read_transposed(src), hi = read_transposed(src + 16 * kRowBytes);
        const x8 v = __builtin_bit_cast(x8, u32x4{lo.x, lo.y, hi.x, hi.y});
        o[d] = Elem<E>::mma16(v, w, o[d]);
        o[d] = Elem<E>::mma16(v, rest, o[d]);
      }
    }
  };

  unsigned int base = t_begin + wave * kFewStep;
  if (base < t_end) {
    Keys k0, k1;
    issue(base, block_id<kPaged>(a, table, token_of(base)), k0, stage0);
    int id = block_id<kPaged>(a, table, token_of(base + kRound));
    for (;;) {
      // the next step's loads go out (past the end: the last token again), then this step's
      // are waited for
      issue(base + kRound, id, k1, stage1);
      id = block_id<kPaged>(a, table, token_of(base + 2 * kRound));
      wait_loads<2 * kSlabs + kLoads + (kPaged ? 1 : 0)>();
      step(base, k0, stage0);
      base += kRound;
      if (base >= t_end) break;
      issue(base + kRound, id, k0, stage0);
      id = block_id<kPaged>(a, table, token_of(base + 2 * kRound));
      wait_loads<2 * kSlabs + kLoads + (kPaged ? 1 : 0)>();
      step(base, k1, stage1);
      base += kRound;
      if (base >= t_end) break;
    }
  }
  wait_loads<0>();

  // ---- the waves' sums meet in LDS, a thread takes kVals dims of a row ----
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  bad = any_lane(bad, s2);
  __syncthreads();
  float* const s_acc = reinterpret_cast<float*>(s0);
  float* const s_ml = reinterpret_cast<float*>(s2);
  if (grp == 0) {
    s_ml[2 * (wave * kFewRows + col)] = m_ref;
    s_ml[2 * (wave * kFewRows + col) + 1] = l_run;
  }
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d)
    *reinterpret_cast<f32x4*>(s_acc + (wave * kFewRows + col) * D + 16 * d + 4 * grp) = o[d];
  __syncthreads();
  constexpr unsigned int kShare = 4 * kN;  // threads of a row
  constexpr int kVals = D / kShare;
  static_assert(kVals == 4 || kVals == 8, "stored by 16 bytes");
  const unsigned int row_m = tid / kShare, d0 = (tid % kShare) * kVals;
  float big = kNoMax, l = 0.f, acc[kVals];
#pragma unroll
  for (int w = 0; w < kN; ++w) big = fmaxf(big, s_ml[2 * (w * kFewRows + row_m)]);
#pragma unroll
  for (int i = 0; i < kVals; ++i) acc[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kN; ++w) {
    const float f = exp2f(s_ml[2 * (w * kFewRows + row_m)] - big);
    l += s_ml[2 * (w * kFewRows + row_m) + 1] * f;
#pragma unroll
    for (int i = 0; i < kVals; ++i) acc[i] += s_acc[(w * kFewRows + row_m) * D + d0 + i] * f;
  }
  float check = l * 0.f;
#pragma unroll
  for (int i = 0; i < kVals; ++i) check = fmaf(acc[i], 0.f, check);
#pragma unroll
  for (unsigned int d = 1; d < kShare; d *= 2) check += __shfl_xor(check, d, 64);
  const bool in = row_m < rows;
  const bool again = in && !bad && !(check == 0.f);
  const unsigned int tok = in ? row_m / a.group : 0u;
  const unsigned int qh = head * a.group + (in ? row_m - tok * a.group : 0u);
  const unsigned long long out_row = (unsigned long long)(request.start + tok) * a.q_heads + qh;
  if (bad) big = l = NAN;
  if (in && !again) {
    if (splits > 1) {
      float* ml = slot_ml<D, kRows>(a, slot) + 2 * row_m;
      float* dst = slot_acc<D, kRows>(a, slot) + row_m * D + d0;
      if (d0 == 0) {
        ml[0] = big;
        ml[1] = l;
      }
#pragma unroll
      for (int i = 0; i < kVals; i += 4)
        *reinterpret_cast<f32x4*>(dst + i) = f32x4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
    } else {
      const bool none = shift + (int)(kMore * tok) < 0 && !bad;
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
  for (unsigned int i = 0; i < kWave / kShare; ++i) {
    if (((flags >> (kShare * i)) & 1) == 0) continue;
    const unsigned int mm = kWave / kShare * wave + i, t = mm / a.group, h = head * a.group + mm % a.group;
    const unsigned int seen = (unsigned int)max(shift + (int)(kMore * t) + 1, 0);
    float rm, rl, ra[D / 64];
    slow_row<E, D, kPaged>(a, table, source,
                         a.q + (unsigned long long)(request.start + t) * a.q_row +
                             (unsigned long long)h * a.q_head,
                         head, t_begin, min(t_end, seen), rm, rl, ra);
    store_slow<E, D, kRows>(a, splits > 1, slot, mm,
                            (unsigned long long)(request.start + t) * a.q_heads + h, seen == 0, rm, rl, ra);
  }
}

// ---------------------------------------------------------------------------
// the launches

// (a variable for each buffer: the compiler orders a read of one behind the loads into it, and not
// behind those into the others)
template <typename E, int D, bool kPaged, bool kRuns, Sight kSight>
__global__ __launch_bounds__(kWave * tile_waves(D), D == 128 ? 2 : 3) void attention_tiles(AttendArgs a) {
  constexpr int kN = tile_waves(D), kRows = tile_rows(D);
  constexpr int kBuffer = 2 * kTileTokens * 2 * D;
  constexpr int kStages = kPaged ? kN * kFewStep * 2 * D : kBuffer;  // of the streaming waves
  __shared__ __align__(1024) unsigned char s0[kStages];
  __shared__ __align__(1024) unsigned char s1[kStages];
  __shared__ __align__(1024) unsigned char s2[kBuffer];
  const unsigned int head = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
  const Work<true, kRows, kPaged> work(a);
  Request request;
  unsigned int index, slot;
  bool has_slot;
  const bool found = work.find(item, request, index, has_slot, slot);
  if (item == a.items) {  // the last one, for the slots that the others do not use
    clear_jobs(a, slot, head);
    return;
  }
  if (!found) return;
  const unsigned int most = work.splits(request), split_tokens = work.split_tokens(request, most);
  const unsigned int order = index / most, split = index - order * most;
  // (row ranges that overlap each other can ask for more items than there are: a tile without all its
  // splits is left)
  const bool whole = item - split + most <= a.items;
  if constexpr (kPaged) {
    if (work.few(request.n)) {
      if (!has_slot) slot = kNoSlot;
      few_path<E, D, kN, kRows, kPaged, kSight>(a, request, split, most, split_tokens, whole, slot, head, s0, s1, s2);
      return;
    }
  }
  tile_path<E, D, kPaged, kRuns, kSight>(a, request, order, split, most, split_tokens, whole, slot, head, s0, s1, s2);
}

template <typename E, int D, bool kPaged, Sight kSight>
__global__ __launch_bounds__(kWave * kWaves, 2) void attention_few(AttendArgs a) {
  constexpr int kBuffer = kWaves * kFewStep * 2 * D;
  __shared__ __align__(1024) unsigned char s0[kBuffer];
  __shared__ __align__(1024) unsigned char s1[kBuffer];
  __shared__ __align__(16) unsigned char s2[kWaves * 16 * 2 * sizeof(float)];
  const unsigned int head = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
  const Work<false, kFewRows, kPaged> work(a);
  Request request;
  unsigned int split, slot;
  bool has_slot;
  if (!work.find(item, request, split, has_slot, slot)) {
    store_job(a, item, head, Job{});
    return;
  }
  const unsigned int splits = work.splits(request);
  few_path<E, D, kWaves, kFewRows, kPaged, kSight>(a, request, split, splits, work.split_tokens(request, splits),
                                                   true, slot, head, s0, s1, s2);
}

// ---------------------------------------------------------------------------
// the splits of a row joined

// A workgroup looks at its share of the slots' jobs with one load and takes those that have
// something to join: 16 rows of a tile with a thread for 8 (D = 64: 4) sums of a row, or 4 rows of
// the streaming path, which has more splits, with four threads that share a row's splits.
template <typename E, int D, bool kTiles>
__global__ __launch_bounds__(kMergeThreads) void attention_merge(AttendArgs a) {
  constexpr int kRows = kTiles ? tile_rows(D) : kFewRows;
  constexpr int kVals = D / 16, kBatch = 4;
  constexpr unsigned int kShares = kTiles ? 1 : 4;  // threads that share a row's splits
  constexpr unsigned int kJobRows = 16 / kShares, kParts = kRows / kJobRows;
  __shared__ float s_part[kTiles ? 1 : kMergeThreads][kVals + 2];
  const unsigned int tid = threadIdx.x, lane = tid & 63;
  const unsigned int jobs = a.slots * kParts;
  for (unsigned int j0 = blockIdx.x; j0 < jobs; j0 += kWave * gridDim.x) {
    const unsigned int mine = j0 + lane * gridDim.x;
    const Job own = a.jobs[min(mine, jobs - 1) / kParts];
    unsigned long long todo =
        __ballot(mine < jobs && own.splits != 0 && mine % kParts * kJobRows < own.rows);
    while (todo != 0) {
      const int at = __ffsll((long long)todo) - 1;
      const unsigned int j = j0 + (unsigned int)at * gridDim.x;
      todo &= todo - 1;
      const unsigned int slot = j / kParts, head = slot % a.kv_heads;
      const unsigned int counts = lane_value((unsigned int)own.splits << 16 | own.rows, at);
      const Job job{lane_value(own.start, at), lane_value(own.first, at), (int)lane_value((unsigned int)own.shift, at),
                    (unsigned short)counts, (unsigned short)(counts >> 16)};
      const unsigned int share = tid / 16 % kShares, dims = tid % 16 * kVals;
      const unsigned int row = j % kParts * kJobRows + tid / (16 * kShares);
      const bool in = row < job.rows;
      const unsigned int use = in ? row : 0u;
      float big = kNoMax, l = 0.f, acc[kVals];
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kVals; ++i) acc[i] = 0.f;
      for (unsigned int b = share; b < job.splits; b += kShares * kBatch) {
        f32x2 ml[kBatch];
        f32x4 v[kBatch][kVals / 4];
        // (past the last split the last one again, without weight: loads behind branches would
        // wait for each other)
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const unsigned int at = slot + min(b + k * kShares, job.splits - 1u) * a.kv_heads;
          ml[k] = *reinterpret_cast<const f32x2*>(slot_ml<D, kRows>(a, at) + 2 * use);
          const float* src = slot_acc<D, kRows>(a, at) + use * D + dims;
#pragma unroll
          for (int i = 0; i < kVals / 4; ++i) v[k][i] = *reinterpret_cast<const f32x4*>(src + 4 * i);
        }
        float top = big;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (b + k * kShares >= job.splits) ml[k] = f32x2{kNoMax, 0.f};
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
          // (a weight of zero joins too: a row's NaN and infinite values stay; what a row does not
          // see is zero in its sums)
          const bool split = b + k * kShares < job.splits;
          const float f = split ? exp2f(ml[k].x - big) : 0.f;
          l += ml[k].y * f;
#pragma unroll
          for (int i = 0; i < kVals; ++i) acc[i] = split ? fmaf(v[k][i / 4][i % 4], f, acc[i]) : acc[i];
        }
      }
      if constexpr (!kTiles) {
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
      const bool none = job.shift + (int)(a.causal * tok) < 0 && !bad;
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

// A call's grid and partial slots, from what the host knows: tokens (rows of q), requests, the
// longest context that the tables (or the rows) can hold, and the longest request. Which kernel it
// is goes by the longest request's rows alone.
struct Plan {
  bool tiles, fine;
  unsigned int tile_least;  // steps of a tile's split, at least
  unsigned long long few_target, tile_target;  // workgroups that splits are made for
  unsigned long long groups, slots;            // workgroups, partial slots
  unsigned long long items;                    // of the tiles
};

// Splits of `active` requests at most, that are made for `target` workgroups, with one that has none.
unsigned long long few_slots(unsigned long long target, unsigned long long kv_heads, unsigned long long active) {
  return (target / kv_heads + active + 1) * kv_heads;
}

Plan plan_of(unsigned long long tokens, unsigned long long requests, unsigned long long kv_heads,
             unsigned long long group, unsigned long long head_dim, unsigned long long max_context,
             unsigned long long max_query, bool paged, bool causal = true) {
  Plan p{};
  p.tiles = !paged || max_query * group > kFewRows;
  p.tile_least = causal ? kLeastTileSteps : kLeastSourceTileSteps;
  // (streaming: as many as run at once; 64 requests of 128 .. 32000 tokens, 8 / 1 heads of 128: 39.8 us,
  // with three quarters of it 41.3, with half more 44.9)
  // (of 64-dim sources four run on a CU: 64 requests of 128 .. 16000 tokens, 32 / 8 heads 113 us with two, 105
  // with four; 32 of 200 .. 16000, 8 heads 73 and 66; 8 of 8000 the same)
  p.few_target = (head_dim == 64 && !causal ? 4 : 2) * compute_units();
  // (tiles: three quarters of the CUs, twice that with workgroups of four waves. Longer splits, so
  // fewer of them, than an even share: 16 requests of 6 tokens behind 300 .. 8000 38.0 us and 45.8, a prompt of 1443 39.3 and 52.9;
  // with a share of a fourth to a half of it 3 chunks beside 29 decodes took 402 and not 311)
  p.tile_target = std::max(1ull, compute_units() * (head_dim == 128 ? 3 : 6) / 4);
  const unsigned long long active = std::min(tokens, requests);
  if (p.tiles) {
    const unsigned long long rows = (unsigned long long)tile_rows((int)head_dim);
    const unsigned long long tiles = tokens * group / rows + active;
    const bool half = !causal && 2 * tiles * kv_heads <= compute_units();
    const double whole = kTileTokens * (half ? kWholeSourceTileSteps : kLeastTileSteps);
    bool cut = (double)max_context > whole;
    if (cut && !paged) {
      // A prompt of L of the n rows of q, of r prompts that fill them, is cut where its L / 64 steps are
      // more than a workgroup's share of all, which is at least that of L * group / rows tiles of L
      // tokens and of the r - 1 others at equal lengths: L > share * (L^2 + (n - L)^2 / (r - 1)).
      // Where that holds for no length, nothing is cut, which spares the joining (7 us). Prompts that
      // do not fill the rows are not cut then either.
      const double n = (double)tokens, others = (double)active - 1;
      const double share = (double)(group * kv_heads) / (double)(rows * p.tile_target);
      double l = n;
      if (others > 0)  // where the right side is least above the left
        l = std::min(std::max((0.5 / share + n / others) / (1 + 1 / others), whole + 1), (double)max_context);
      cut = l > share * (l * l + (others > 0 ? (n - l) * (n - l) / others : 0.));
    }
    // (see Work; the share of one KV head)
    const unsigned long long more = cut ? p.tile_target / kv_heads + 1 : 0;
    p.slots = 2 * more * kv_heads;
    p.items = tiles + more;
    p.groups = (p.items + (cut ? 1 : 0)) * kv_heads;
  } else {
    const unsigned long long whole = active * kv_heads, cus = compute_units();
    p.fine = !causal && 8 * whole <= cus;
    const unsigned int steps = causal ? kWholeFewSteps : p.fine ? whole_fine_steps(head_dim) :
                               4 * whole >= 3 * cus ? kWholeSourceSteps : kWholeFewSteps;
    const bool cut = max_context > kFewUnit * steps;
    p.groups = whole;
    if (cut) p.groups = p.slots = few_slots(p.few_target, kv_heads, active);
  }
  return p;
}

// The slots' partials, then their jobs.
unsigned long long partial_bytes(const Plan& p, unsigned long long head_dim) {
  return p.slots * (p.tiles ? tile_rows((int)head_dim) : kFewRows) * (head_dim + 2) * sizeof(float);
}
unsigned long long workspace_of(const Plan& p, unsigned long long head_dim) {
  return partial_bytes(p, head_dim) + p.slots * sizeof(Job);
}

// Enough for every call of at most these sizes. (It does not grow with all of them: rows that many
// prompts share are cut less than those of one, and streamed requests have a slot each, tiles have not.)
unsigned long long workspace_bound(unsigned long long tokens, unsigned long long requests,
                                   unsigned long long kv_heads, unsigned long long group,
                                   unsigned long long head_dim, unsigned long long max_context,
                                   unsigned long long max_query, bool paged, bool causal = true) {
  Plan plan = plan_of(tokens, requests, kv_heads, group, head_dim, max_context, max_query, paged, causal);
  // (of fewer tiles sources are cut that more of them leave whole)
  if (!causal && plan.tiles && max_context > kTileTokens * kWholeSourceTileSteps)
    plan.slots = 2 * (plan.tile_target / kv_heads + 1) * kv_heads;
  const unsigned long long own = workspace_of(plan, head_dim);
  if (!paged) {
    // (of one prompt the shortest that can be cut at all is cut the soonest; all that are cut need the same)
    const unsigned long long n = std::min<unsigned long long>(max_query, kTileTokens * kLeastTileSteps + 1);
    return std::max(own, workspace_of(plan_of(n, 1, kv_heads, group, head_dim, n, n, false), head_dim));
  }
  const unsigned long long few = std::min<unsigned long long>(max_query, kFewRows / group);
  if (few == 0) return own;
  Plan most = plan_of(tokens, requests, kv_heads, group, head_dim, max_context, few, true, causal);
  // (and of fewer requests)
  if (!causal && max_context > kFewUnit * whole_fine_steps(head_dim))
    most.slots = few_slots(most.few_target, kv_heads, std::min(tokens, requests));
  return std::max(own, workspace_of(most, head_dim));
}

template <typename E, int D, bool kTiles>
hipError_t launch_merge(const AttendArgs& a, hipStream_t stream) {
  const unsigned int jobs = a.slots * (kTiles ? tile_rows(D) / 16 : kFewRows / 4);
  if (jobs == 0) return hipSuccess;  // (no context that is long enough to be split)
  hipLaunchKernelGGL((attention_merge<E, D, kTiles>), dim3(std::min(jobs, kMergeGroups)),
                     dim3(kMergeThreads), 0, stream, a);
  return hipGetLastError();
}

template <typename E, int D, bool kPaged, Sight kSight>
long long launch(const AttendArgs& a, const Plan& p, hipStream_t stream) {
  const dim3 grid((unsigned int)p.groups);
  hipError_t st = hipSuccess;
  if (p.tiles) {
    const dim3 threads(kWave * tile_waves(D));
    if constexpr (!kPaged)
      hipLaunchKernelGGL((attention_tiles<E, D, false, true, kSight>), grid, threads, 0, stream, a);
    else if (a.block_tokens % 8 == 0)
      hipLaunchKernelGGL((attention_tiles<E, D, true, true, kSight>), grid, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((attention_tiles<E, D, true, false, kSight>), grid, threads, 0, stream, a);
    st = hipGetLastError();
    if (st != hipSuccess) return fail("attention_tiles", st);
    st = launch_merge<E, D, true>(a, stream);
  } else {
    // (prompts always go to attention_tiles)
    if constexpr (kPaged || kSight == kWholeSource)
      hipLaunchKernelGGL((attention_few<E, D, kPaged, kSight>), grid, dim3(kWave * kWaves), 0, stream, a);
    st = hipGetLastError();
    if (st != hipSuccess) return fail("attention_few", st);
    st = launch_merge<E, D, false>(a, stream);
  }
  if (st != hipSuccess) return fail("attention_merge", st);
  return (long long)((unsigned long long)a.tokens * a.q_heads * D * 2);
}

template <bool kPaged, Sight kSight>
long long launch_typed(const AttendArgs& a, const Plan& p, unsigned long long head_dim,
                       unsigned long long dtype, hipStream_t stream) {
  if (head_dim == 128)
    return dtype ? launch<_Float16, 128, kPaged, kSight>(a, p, stream)
                 : launch<__bf16, 128, kPaged, kSight>(a, p, stream);
  return dtype ? launch<_Float16, 64, kPaged, kSight>(a, p, stream)
               : launch<__bf16, 64, kPaged, kSight>(a, p, stream);
}
template <bool kPaged>
long long launch_typed(const AttendArgs& a, const Plan& p, unsigned long long head_dim,
                       unsigned long long dtype, hipStream_t stream) {
  return a.causal ? launch_typed<kPaged, kOwnContext>(a, p, head_dim, dtype, stream)
                  : launch_typed<kPaged, kWholeSource>(a, p, head_dim, dtype, stream);
}

constexpr unsigned long long kMostRows = 0x7FFFFFFFull;
constexpr unsigned long long kMostGroups = 0xFFFFFFFFull / (kWave * 8);  // a grid's threads fit 32 bits
constexpr float kLog2E = 1.4426950408889634f;
constexpr unsigned long long kMostStride = 1ull << 27;  // 8 rows' offsets fit 31 bits

// Bytes from the first to the last of rows x heads pieces of head_bytes.
unsigned long long extent(unsigned long long rows, unsigned long long row_bytes,
                          unsigned long long heads, unsigned long long head_step,
                          unsigned long long head_bytes) {
  return (rows - 1) * row_bytes + (heads - 1) * head_step + head_bytes;
}

struct Bytes {
  unsigned long long at, count;
};
// Whether what a call writes lies over nothing that it reads, and over nothing else that it writes
// (some workgroups still read when others write).
bool results_apart(std::initializer_list<Bytes> written, std::initializer_list<Bytes> read) {
  for (const Bytes* w = written.begin(); w != written.end(); ++w) {
    for (const Bytes& r : read)
      if (overlap(w->at, w->count, r.at, r.count)) return false;
    for (const Bytes* o = written.begin(); o != w; ++o)
      if (overlap(w->at, w->count, o->at, o->count)) return false;
  }
  return true;
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
  max_query = std::min(max_query, tokens);
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_bound(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_context, max_query, true);
}

extern "C" unsigned long long kvq_splitzip_prompt_attention_workspace_bytes(
    unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_query) {
  max_query = std::min(max_query, tokens);
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_bound(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_query, max_query, false);
}

extern "C" unsigned long long kvq_splitzip_prompt_attention_least_workspace_bytes(
    unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_query) {
  max_query = std::min(max_query, tokens);
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_of(plan_of(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_query, max_query,
                              false), head_dim);
}

extern "C" unsigned long long kvq_splitzip_cross_attention_workspace_bytes(
    unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_source,
    unsigned long long max_query) {
  max_query = std::min(max_query, tokens);
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_bound(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_source, max_query, true,
                         false);
}

extern "C" unsigned long long kvq_splitzip_cross_attention_least_workspace_bytes(
    unsigned long long tokens, unsigned long long requests, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long max_source,
    unsigned long long max_query) {
  max_query = std::min(max_query, tokens);
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query)) return 0;
  return workspace_of(plan_of(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_source, max_query, true,
                              false), head_dim);
}

namespace {

// Over a paged layer: a step's own context (causal), or a source.
long long attend_paged(
    unsigned long long q_ptr, unsigned long long q_row_bytes, unsigned long long q_head_bytes,
    unsigned long long tokens, unsigned long long q_heads, unsigned long long kv_heads,
    unsigned long long head_dim, unsigned long long dtype, unsigned long long kv_ptr,
    unsigned long long blocks, unsigned long long block_tokens, unsigned long long tables_ptr,
    unsigned long long table_stride, unsigned long long table_width,
    unsigned long long query_starts_ptr, unsigned long long context_tokens_ptr,
    unsigned long long requests, unsigned long long max_query, unsigned long long out_ptr,
    unsigned long long lse_ptr, unsigned long long workspace_ptr,
    unsigned long long workspace_bytes, float scale, unsigned long long stream_ptr, bool causal) {
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query) || dtype > 1 ||
      q_ptr == 0 || q_ptr % 16 != 0 || q_row_bytes % 16 != 0 || q_head_bytes % 16 != 0 ||
      kv_ptr == 0 || kv_ptr % 16 != 0 || blocks == 0 || block_tokens == 0 || blocks > kMostRows ||
      block_tokens > kMostRows || blocks * block_tokens > kMostRows || tables_ptr == 0 ||
      table_width == 0 || table_width > kMostRows || table_stride < table_width ||
      query_starts_ptr == 0 || context_tokens_ptr == 0 || out_ptr == 0 || out_ptr % 16 != 0 ||
      !(scale > 0.f) || !std::isfinite(scale * kLog2E))
    return 0;
  const unsigned long long max_context = std::min(table_width * block_tokens, kMostRows);
  const Plan plan = plan_of(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_context, max_query, true,
                            causal);
  const unsigned long long need = workspace_of(plan, head_dim);
  if (need != 0 && (workspace_ptr == 0 || workspace_ptr % 16 != 0 || workspace_bytes < need)) return 0;
  if (plan.groups > kMostGroups) return 0;
  const unsigned long long out_bytes = tokens * q_heads * head_dim * 2;
  if (!results_apart(
          {{out_ptr, out_bytes}, {lse_ptr, lse_ptr ? 4 * tokens * q_heads : 0}, {workspace_ptr, need}},
          {{q_ptr, extent(tokens, q_row_bytes, q_heads, q_head_bytes, 2 * head_dim)},
           {kv_ptr, 4 * blocks * block_tokens * kv_heads * head_dim},
           {tables_ptr, 4 * ((requests - 1) * table_stride + table_width)},
           {query_starts_ptr, 4 * (requests + 1)}, {context_tokens_ptr, 4 * requests}}))
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
  a.jobs = reinterpret_cast<Job*>(workspace_ptr + partial_bytes(plan, head_dim));
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
  a.few_target = (unsigned int)plan.few_target;
  a.fine = plan.fine ? 1 : 0;
  a.tile_target = (unsigned int)plan.tile_target;
  a.tile_least = plan.tile_least;
  a.max_query = (unsigned int)max_query;
  a.causal = causal ? 1 : 0;
  a.slots = (unsigned int)plan.slots;
  a.items = (unsigned int)plan.items;
  a.scale_log2 = scale * kLog2E;
  return launch_typed<true>(a, plan, head_dim, dtype, reinterpret_cast<hipStream_t>(stream_ptr));
}

}  // namespace

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
  return attend_paged(q_ptr, q_row_bytes, q_head_bytes, tokens, q_heads, kv_heads, head_dim, dtype, kv_ptr,
                      blocks, block_tokens, tables_ptr, table_stride, table_width, query_starts_ptr,
                      context_tokens_ptr, requests, max_query, out_ptr, lse_ptr, workspace_ptr,
                      workspace_bytes, scale, stream_ptr, true);
}

extern "C" long long kvq_splitzip_cross_attention_paged(
    unsigned long long q_ptr, unsigned long long q_row_bytes, unsigned long long q_head_bytes,
    unsigned long long tokens, unsigned long long q_heads, unsigned long long kv_heads,
    unsigned long long head_dim, unsigned long long dtype, unsigned long long kv_ptr,
    unsigned long long blocks, unsigned long long block_tokens, unsigned long long tables_ptr,
    unsigned long long table_stride, unsigned long long table_width,
    unsigned long long query_starts_ptr, unsigned long long context_tokens_ptr,
    unsigned long long requests, unsigned long long max_query, unsigned long long out_ptr,
    unsigned long long lse_ptr, unsigned long long workspace_ptr,
    unsigned long long workspace_bytes, float scale, unsigned long long stream_ptr) {
  return attend_paged(q_ptr, q_row_bytes, q_head_bytes, tokens, q_heads, kv_heads, head_dim, dtype, kv_ptr,
                      blocks, block_tokens, tables_ptr, table_stride, table_width, query_starts_ptr,
                      context_tokens_ptr, requests, max_query, out_ptr, lse_ptr, workspace_ptr,
                      workspace_bytes, scale, stream_ptr, false);
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
      out_ptr == 0 || out_ptr % 16 != 0 || !(scale > 0.f) || !std::isfinite(scale * kLog2E))
    return 0;
  const Plan plan = plan_of(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_query, max_query, false);
  const unsigned long long need = workspace_of(plan, head_dim);
  if (need != 0 && (workspace_ptr == 0 || workspace_ptr % 16 != 0 || workspace_bytes < need)) return 0;
  if (plan.groups > kMostGroups) return 0;
  const unsigned long long out_bytes = tokens * q_heads * head_dim * 2;
  if (!results_apart(
          {{out_ptr, out_bytes}, {lse_ptr, lse_ptr ? 4 * tokens * q_heads : 0}, {workspace_ptr, need}},
          {{q_ptr, extent(tokens, q_row_bytes, q_heads, q_head_bytes, 2 * head_dim)},
           {k_ptr, extent(tokens, k_row_bytes, kv_heads, k_head_bytes, 2 * head_dim)},
           {v_ptr, extent(tokens, v_row_bytes, kv_heads, v_head_bytes, 2 * head_dim)},
           {query_starts_ptr, 4 * (requests + 1)}}))
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
  a.jobs = reinterpret_cast<Job*>(workspace_ptr + partial_bytes(plan, head_dim));
  a.q_row = q_row_bytes;
  a.q_head = q_head_bytes;
  a.tokens = (unsigned int)tokens;
  a.requests = (unsigned int)requests;
  a.q_heads = (unsigned int)q_heads;
  a.kv_heads = (unsigned int)kv_heads;
  a.group = (unsigned int)(q_heads / kv_heads);
  a.few_target = (unsigned int)plan.few_target;
  a.tile_target = (unsigned int)plan.tile_target;
  a.tile_least = plan.tile_least;
  a.max_query = (unsigned int)max_query;
  a.causal = 1;
  a.slots = (unsigned int)plan.slots;
  a.items = (unsigned int)plan.items;
  a.scale_log2 = scale * kLog2E;
  return launch_typed<false>(a, plan, head_dim, dtype, reinterpret_cast<hipStream_t>(stream_ptr));
}

extern "C" long long kvq_splitzip_cross_attention(
    unsigned long long q_ptr, unsigned long long q_row_bytes, unsigned long long q_head_bytes,
    unsigned long long k_ptr, unsigned long long k_row_bytes, unsigned long long k_head_bytes,
    unsigned long long v_ptr, unsigned long long v_row_bytes, unsigned long long v_head_bytes,
    unsigned long long source_rows, unsigned long long tokens, unsigned long long q_heads,
    unsigned long long kv_heads, unsigned long long head_dim, unsigned long long dtype,
    unsigned long long query_starts_ptr, unsigned long long source_starts_ptr,
    unsigned long long source_tokens_ptr, unsigned long long requests, unsigned long long max_query,
    unsigned long long max_source, unsigned long long out_ptr, unsigned long long lse_ptr,
    unsigned long long workspace_ptr, unsigned long long workspace_bytes, float scale,
    unsigned long long stream_ptr) {
  if (!sizes_ok(tokens, requests, q_heads, kv_heads, head_dim, max_query) || dtype > 1 ||
      q_ptr == 0 || k_ptr == 0 || v_ptr == 0 || source_rows == 0 || source_rows > kMostRows ||
      max_source > source_rows ||
      (q_ptr | q_row_bytes | q_head_bytes | k_ptr | k_row_bytes | k_head_bytes | v_ptr |
       v_row_bytes | v_head_bytes) % 16 != 0 ||
      k_row_bytes > kMostStride || v_row_bytes > kMostStride || query_starts_ptr == 0 ||
      source_starts_ptr == 0 || source_tokens_ptr == 0 || out_ptr == 0 || out_ptr % 16 != 0 ||
      !(scale > 0.f) || !std::isfinite(scale * kLog2E))
    return 0;
  // (as over a layer: sources' lengths do not follow from the rows of q)
  const Plan plan = plan_of(tokens, requests, kv_heads, q_heads / kv_heads, head_dim, max_source, max_query, true,
                            false);
  const unsigned long long need = workspace_of(plan, head_dim);
  if (need != 0 && (workspace_ptr == 0 || workspace_ptr % 16 != 0 || workspace_bytes < need)) return 0;
  if (plan.groups > kMostGroups) return 0;
  const unsigned long long out_bytes = tokens * q_heads * head_dim * 2;
  if (!results_apart(
          {{out_ptr, out_bytes}, {lse_ptr, lse_ptr ? 4 * tokens * q_heads : 0}, {workspace_ptr, need}},
          {{q_ptr, extent(tokens, q_row_bytes, q_heads, q_head_bytes, 2 * head_dim)},
           {k_ptr, extent(source_rows, k_row_bytes, kv_heads, k_head_bytes, 2 * head_dim)},
           {v_ptr, extent(source_rows, v_row_bytes, kv_heads, v_head_bytes, 2 * head_dim)},
           {query_starts_ptr, 4 * (requests + 1)}, {source_starts_ptr, 4 * requests},
           {source_tokens_ptr, 4 * requests}}))
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
  a.contexts = reinterpret_cast<const int*>(source_tokens_ptr);
  a.sources = reinterpret_cast<const int*>(source_starts_ptr);
  a.partial = reinterpret_cast<float*>(workspace_ptr);
  a.jobs = reinterpret_cast<Job*>(workspace_ptr + partial_bytes(plan, head_dim));
  a.q_row = q_row_bytes;
  a.q_head = q_head_bytes;
  a.tokens = (unsigned int)tokens;
  a.requests = (unsigned int)requests;
  a.q_heads = (unsigned int)q_heads;
  a.kv_heads = (unsigned int)kv_heads;
  a.group = (unsigned int)(q_heads / kv_heads);
  a.few_target = (unsigned int)plan.few_target;
  a.fine = plan.fine ? 1 : 0;
  a.tile_target = (unsigned int)plan.tile_target;
  a.tile_least = plan.tile_least;
  a.max_query = (unsigned int)max_query;
  a.max_source = (unsigned int)max_source;
  a.kv_rows = (unsigned int)source_rows;
  a.slots = (unsigned int)plan.slots;
  a.items = (unsigned int)plan.items;
  a.scale_log2 = scale * kLog2E;
  return launch_typed<false>(a, plan, head_dim, dtype, reinterpret_cast<hipStream_t>(stream_ptr));
}
