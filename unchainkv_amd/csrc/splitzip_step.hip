// A serving step's tables and the cache write, gfx950: block tables, row ranges, slots and
// positions from the requests' lengths, and the new tokens' K and V rows into a paged layer, as they
// are or with K and Q rotated by position.
//
// Plan. With b tokens to a block, request r holds ceil(cached_r / b) blocks and needs
// ceil((cached_r + new_r) / b). Fresh blocks come off the free list in request order, so an
// exclusive sum over the requests gives each its place in the list, and another one its rows
// among the step's packed tokens. Token i of request r has position p = cached_r + i and slot
// table[r][p / b] * b + p % b. What bounds it is latency (a 64-request decode step reads and
// writes 2 KB): one launch, in which every workgroup forms the sums of all requests for itself
// (kChunk at a time, in LDS) instead of waiting for another one's; a fresh block's id is taken
// from the free list by the workgroups that need it for a slot, so none reads a table entry
// that another one writes. Measured: 5.0 us for a decode step of 64 requests, 5.9 for 256 of which
// 16 have 1024 .. 2048 new tokens.
//
// Write. A copy with the destination row chosen by slot: each lane moves units of 16 bytes (or
// the largest the tensors' strides and addresses allow), its K and V units of two tokens in
// flight at once. Bound by HBM: 32768 tokens of 8 x 128, 268 MB read and written, 42.8 us (6.3 TB/s,
// partly from the caches; 52.4 us, 5.1 TB/s, where its inputs are cold).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "splitzip_common.h"

namespace unchainkv {
namespace {

constexpr int kStepThreads = 256;
constexpr int kPerThread = 4;                       // requests a thread sums
constexpr int kChunk = kStepThreads * kPerThread;   // requests a workgroup holds at a time

struct PlanArgs {
  const int* new_tokens;     // [requests]
  const int* cached_tokens;  // [requests]
  int* tables;               // [requests][table_stride], width entries used
  const int* free_blocks;    // [free_count]
  const int* free_start;     // [1]
  int* query_starts;         // [requests + 1]
  int* context_tokens;       // [requests]
  long long* slots;          // [max_tokens]
  long long* positions;      // [max_tokens]
  int* free_next;            // [1]
  int* lacking;              // [1]
  unsigned long long table_stride;
  unsigned int requests, width, block_tokens, free_count, max_tokens;
};

__device__ __forceinline__ unsigned int blocks_of(unsigned int tokens, unsigned int b) {
  return tokens / b + (tokens % b != 0 ? 1u : 0u);
}

// Inclusive sum over the wave's lanes.
template <typename T>
__device__ __forceinline__ T wave_sum_scan(T v) {
  const unsigned int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const T o = __shfl_up(v, d, kWave);
    if (lane >= (unsigned int)d) v += o;
  }
  return v;
}

// Last index i in [0, count) with first[i] <= x (first ascending, first[0] <= x).
__device__ __forceinline__ unsigned int owner_of(const unsigned long long* first, unsigned int count,
                                                 unsigned long long x) {
  unsigned int lo = 0, hi = count;
  while (hi - lo > 1) {
    const unsigned int mid = (lo + hi) / 2;
    if (first[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kStepThreads) void plan_step(PlanArgs a) {
  __shared__ unsigned long long s_row[kChunk];    // first packed row of each request
  __shared__ unsigned long long s_fresh[kChunk];  // fresh blocks of the requests before it
  __shared__ unsigned int s_cached[kChunk];
  __shared__ unsigned long long s_wave[2][kStepThreads / kWave];
  const unsigned int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned int threads = gridDim.x * kStepThreads, first = blockIdx.x * kStepThreads + tid;
  const unsigned int b = a.block_tokens;
  const unsigned long long free_start = (unsigned long long)max(a.free_start[0], 0);
  unsigned long long rows_before = 0, fresh_before = 0, too_wide = 0;
  for (unsigned int r0 = 0; r0 < a.requests; r0 += kChunk) {
    const unsigned int count = min(a.requests - r0, (unsigned int)kChunk);
    // negative lengths count as none
    unsigned int cached[kPerThread], tokens[kPerThread], fresh[kPerThread];
    unsigned long long rows = 0, blocks = 0, wide = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const unsigned int i = tid * kPerThread + k;
      const bool in = i < count;
      cached[k] = in ? (unsigned int)max(a.cached_tokens[r0 + i], 0) : 0u;
      tokens[k] = in ? (unsigned int)max(a.new_tokens[r0 + i], 0) : 0u;
      const unsigned int held = blocks_of(cached[k], b), need = blocks_of(cached[k] + tokens[k], b);
      fresh[k] = min(need, a.width) - min(held, a.width);
      wide += need - held - fresh[k];
      rows += tokens[k];
      blocks += fresh[k];
    }
    const unsigned long long rows_scan = wave_sum_scan(rows), blocks_scan = wave_sum_scan(blocks);
    __syncthreads();  // the chunk before this one is done with the LDS
    if (lane == 63) {
      s_wave[0][wave] = rows_scan;
      s_wave[1][wave] = blocks_scan;
    }
    __syncthreads();
    unsigned long long row = rows_before + rows_scan - rows;
    unsigned long long at = fresh_before + blocks_scan - blocks;
    unsigned long long rows_all = 0, blocks_all = 0;
#pragma unroll
    for (unsigned int w = 0; w < kStepThreads / kWave; ++w) {
      if (w < wave) {
        row += s_wave[0][w];
        at += s_wave[1][w];
      }
      rows_all += s_wave[0][w];
      blocks_all += s_wave[1][w];
    }
    too_wide += wide;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const unsigned int i = tid * kPerThread + k;
      if (i < count) {
        s_row[i] = row;
        s_fresh[i] = at;
        s_cached[i] = cached[k];
        if (blockIdx.x == 0) {
          a.query_starts[r0 + i] = (int)min(row, 0x7FFFFFFFull);
          a.context_tokens[r0 + i] = (int)min(cached[k] + tokens[k], 0x7FFFFFFFu);
        }
      }
      row += tokens[k];
      at += fresh[k];
    }
    __syncthreads();
    const unsigned long long rows_end = rows_before + rows_all;
    // slots and positions of the chunk's tokens
    for (unsigned long long t = first; t < a.max_tokens && t < rows_end; t += threads) {
      if (t < rows_before) continue;
      const unsigned int i = owner_of(s_row, count, t);
      const unsigned int p = s_cached[i] + (unsigned int)(t - s_row[i]);
      const unsigned int blk = p / b, held = blocks_of(s_cached[i], b);
      int id = -1;
      if (blk < a.width) {
        if (blk < held) {
          id = a.tables[(r0 + i) * a.table_stride + blk];
        } else {
          const unsigned long long f = free_start + s_fresh[i] + (blk - held);
          if (f < a.free_count) id = a.free_blocks[f];
        }
      }
      a.slots[t] = id >= 0 ? (long long)id * b + p % b : -1;
      a.positions[t] = p;
    }
    // fresh entries of the chunk's block tables
    for (unsigned long long j = first; j < blocks_all; j += threads) {
      const unsigned int i = owner_of(s_fresh, count, fresh_before + j);
      const unsigned long long f = fresh_before + j, listed = free_start + f;
      const unsigned int blk = blocks_of(s_cached[i], b) + (unsigned int)(f - s_fresh[i]);
      a.tables[(r0 + i) * a.table_stride + blk] =
          listed < a.free_count ? a.free_blocks[listed] : -1;
    }
    rows_before = rows_end;
    fresh_before += blocks_all;
  }
  // rows behind the last request's
  for (unsigned long long t = first; t < a.max_tokens; t += threads) {
    if (t < rows_before) continue;
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
  if (blockIdx.x == 0) {
    const unsigned long long scan = wave_sum_scan(too_wide);
    __syncthreads();
    if (lane == 63) s_wave[0][wave] = scan;
    __syncthreads();
    if (tid == 0) {
      unsigned long long lacking = 0;
#pragma unroll
      for (int w = 0; w < kStepThreads / kWave; ++w) lacking += s_wave[0][w];
      const unsigned long long taken = free_start + fresh_before;
      if (taken > a.free_count) lacking += taken - max(free_start, (unsigned long long)a.free_count);
      a.query_starts[a.requests] = (int)min(rows_before, 0x7FFFFFFFull);
      a.free_next[0] = (int)min(taken, max(free_start, (unsigned long long)a.free_count));
      a.lacking[0] = (int)min(lacking, 0x7FFFFFFFull);
    }
  }
}

struct WriteArgs {
  const unsigned char* k;   // rows of a plane's source
  const unsigned char* v;
  unsigned char* layer;     // K plane; the V plane follows plane_bytes later
  const long long* slots;
  unsigned long long plane_bytes, row_bytes, slot_count;
  unsigned long long k_row, v_row;    // bytes from token to token
  unsigned long long k_head, v_head;  // bytes from head to head
  unsigned int tokens, units;         // units of a row
  unsigned int head_units;            // units of a head within a row
  Divider by_units, by_head;
};

template <typename U>
__global__ __launch_bounds__(kStepThreads) void write_rows(WriteArgs a) {
  constexpr int kTokens = 2;
  const unsigned int total = a.tokens * a.units;  // below 2^30
  const unsigned int stride = gridDim.x * kStepThreads;
  unsigned int i = blockIdx.x * kStepThreads + threadIdx.x;
  for (; i < total; i += kTokens * stride) {
    U k[kTokens], v[kTokens];
    unsigned long long to[kTokens];
    bool in[kTokens];
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
      const unsigned int at = i + n * stride;
      in[n] = at < total;
      const unsigned int use = in[n] ? at : i;
      const unsigned int token = div_u32(use, a.by_units.m, a.by_units.d);
      const unsigned int unit = use - token * a.units;
      const unsigned int head = div_u32(unit, a.by_head.m, a.by_head.d);
      const unsigned int within = unit - head * a.head_units;
      const long long slot = a.slots[token];
      in[n] = in[n] && slot >= 0 && (unsigned long long)slot < a.slot_count;
      to[n] = (unsigned long long)slot * a.row_bytes + (unsigned long long)unit * sizeof(U);
      const unsigned int inner = within * (unsigned int)sizeof(U);
      k[n] = load_stream<U>(a.k + token * a.k_row + head * a.k_head + inner);
      v[n] = load_stream<U>(a.v + token * a.v_row + head * a.v_head + inner);
    }
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
      if (!in[n]) continue;
      *reinterpret_cast<U*>(a.layer + to[n]) = k[n];
      *reinterpret_cast<U*>(a.layer + a.plane_bytes + to[n]) = v[n];
    }
  }
}

// Rotate and write: pairs (x, y) of a head's first `rotary` values become (x cos - y sin, y cos + x sin), with
// the cosines and sines of the token's position from a table, in f32 and rounded once; K goes to its slot with V,
// Q to a tensor of its own. Bound by HBM: 32768 tokens of 32 + 2 x 8 heads of 128, 808 MB read and written, 145
// us, 5.6 TB/s (a large copy: 5.1; one wave a token with a head at a time: 156). A decode step of 64 tokens by
// latency, 3.6 us (rotate_small): the position's load, then the table's row.
struct RotateArgs {
  const unsigned char *q, *k, *v;
  unsigned char* out;          // [tokens][q_heads][dim]
  unsigned char* layer;        // K plane; the V plane follows plane_bytes later
  const float* table;          // [positions][rotary]: cosines, then sines
  const long long* slots;
  const long long* positions;
  unsigned long long q_row, q_head, k_row, k_head, v_row, v_head;  // bytes
  unsigned long long plane_bytes, slot_count, table_rows;
  unsigned int tokens, q_heads, kv_heads, dim, rotary;
  unsigned int first;          // token of this launch
  unsigned int units;          // of the pairs of a head
  unsigned int lanes_heads;    // heads that a wave's lanes take at once
  unsigned int rotating, waves_log;  // waves of a token that rotate, and the logarithm of all
  Divider by_rest, by_head;    // units of a head that are not rotated, and all
};
struct SmallArgs : RotateArgs {
  unsigned int together;       // tokens of a workgroup
  Divider by_units, by_turned, by_copied;  // rotated units of a head, of a token, and others of a token
};

// Of a lane, before another wave of the token takes its share: 8192 tokens of 64 + 2 x 20 heads of 128, all rotated
// 82.6 us (one wave for each sort 86.8; one batch a lane 112), 20 of 128 values rotated 142 (307); 125 tokens of the
// latter's kind 4.5 (39).
constexpr unsigned int kRotatedBatches = 2, kCopiedUnits = 4;
constexpr unsigned int kFewTokens = 256;
constexpr unsigned int kMostSmall = 1u << 22;    // workgroups of a launch,
constexpr unsigned int kMostRotated = 1u << 25;  // waves of a launch, whose threads fit 32 bits

template <typename E, int N>
struct Values {
  typedef E type __attribute__((ext_vector_type(N)));
};

// N pairs turned by their cosines and sines: N values of a head's first half and N of its second, or (kAdjacent) 2 N
// values side by side.
template <typename E, int N, bool kAdjacent>
__device__ __forceinline__ void turn(typename Values<E, N>::type x, typename Values<E, N>::type y,
                                     const float (&c)[N], const float (&s)[N], unsigned char* dst,
                                     unsigned char* dst2) {
  typename Values<E, N>::type x2, y2;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // places of the pair's values among the 2 N
    const int first = kAdjacent ? 2 * i : i, second = kAdjacent ? 2 * i + 1 : N + i;
    const float p = (float)(first < N ? x[first % N] : y[first % N]);
    const float r = (float)(second < N ? x[second % N] : y[second % N]);
    const E p2 = (E)(p * c[i] - r * s[i]), r2 = (E)(r * c[i] + p * s[i]);
    if (first < N) x2[first % N] = p2; else y2[first % N] = p2;
    if (second < N) x2[second % N] = r2; else y2[second % N] = r2;
  }
  *reinterpret_cast<typename Values<E, N>::type*>(dst) = x2;
  *reinterpret_cast<typename Values<E, N>::type*>(dst2) = y2;
}

// Two sorts of waves for each token. In the first a lane keeps the cosines and sines of N pairs and takes them to
// one head after another. The second copies what is not rotated, the heads' other values and V, kUnit at a time,
// and waits for no position or table. kBatch: heads of a lane whose loads go out together.
template <typename E, int N, int kUnit, bool kAdjacent, int kBatch>
__global__ __launch_bounds__(kStepThreads) void rotate_rows(RotateArgs a) {
  typedef typename Values<E, N>::type Unit;
  typedef typename Values<uint16_t, kUnit>::type Copy;
  const unsigned int lane = threadIdx.x & 63;
  const unsigned int job = uniform(blockIdx.x * (kStepThreads / kWave) + (threadIdx.x >> 6));
  const unsigned int waves = 1u << a.waves_log, wave = job & (waves - 1), token = a.first + (job >> a.waves_log);
  if (token >= a.tokens) return;
  const long long slot = a.slots[token];
  const bool write = slot >= 0 && (unsigned long long)slot < a.slot_count;
  const unsigned char* const q = a.q + token * a.q_row;
  const unsigned char* const k = a.k + token * a.k_row;
  const unsigned int head_bytes = a.dim * sizeof(E), pairs = a.rotary / 2;
  unsigned char* const out = a.out + (unsigned long long)token * a.q_heads * head_bytes;
  unsigned char* const layer = a.layer + (write ? (unsigned long long)slot : 0ull) * a.kv_heads * head_bytes;
  // heads of Q, and then of K where the token has a place
  const unsigned int heads = a.q_heads + (write ? a.kv_heads : 0u);
  auto source = [&](unsigned int h) {
    return h < a.q_heads ? q + h * a.q_head : k + (h - a.q_heads) * a.k_head;
  };
  auto target = [&](unsigned int h) {
    return h < a.q_heads ? out + h * head_bytes : layer + (h - a.q_heads) * head_bytes;
  };
  if (wave < a.rotating) {
    const long long position = a.positions[token];
    const bool known = position >= 0 && (unsigned long long)position < a.table_rows;
    const float* const table = a.table + (known ? (unsigned long long)position * a.rotary : 0ull);
    const unsigned int width = min(a.units, (unsigned int)kWave), sub = lane / width;
    if (sub >= a.lanes_heads) return;
    for (unsigned int u = lane - sub * width; u < a.units; u += kWave) {
      const unsigned int at = (kAdjacent ? 2 * N : N) * sizeof(E) * u;
      const unsigned int at2 = at + (kAdjacent ? N : pairs) * sizeof(E);
      float c[N], s[N];
      const unsigned int start = wave * kBatch * a.lanes_heads + sub, step = a.rotating * kBatch * a.lanes_heads;
      for (unsigned int h0 = start; h0 < heads; h0 += step) {
        // (the rows' loads go out before the table's, which wait for the position)
        Unit x[kBatch], y[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const unsigned int h = h0 + b * a.lanes_heads;
          const unsigned char* src = source(h < heads ? h : h0);
          x[b] = *reinterpret_cast<const Unit*>(src + at);
          y[b] = *reinterpret_cast<const Unit*>(src + at2);
        }
        if (h0 == start) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            c[i] = known ? table[u * N + i] : NAN;
            s[i] = known ? table[pairs + u * N + i] : NAN;
          }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const unsigned int h = h0 + b * a.lanes_heads;
          if (h >= heads) continue;
          unsigned char* dst = target(h);
          turn<E, N, kAdjacent>(x[b], y[b], c, s, dst + at, dst + at2);
        }
      }
    }
    return;
  }
  const unsigned char* const v = a.v + token * a.v_row;
  const unsigned int rest = (a.dim - a.rotary) / kUnit, head_units = a.dim / kUnit;
  const unsigned int others = rest * heads, all = others + (write ? head_units * a.kv_heads : 0u);
  constexpr int kCopies = kUnit == 8 ? 2 : 4;
  const unsigned int copying = waves - a.rotating;
  for (unsigned int i0 = (wave - a.rotating) * kCopies * kWave + lane; i0 < all; i0 += copying * kCopies * kWave) {
    Copy x[kCopies];
    unsigned char* dst[kCopies];
#pragma unroll
    for (int n = 0; n < kCopies; ++n) {
      const unsigned int i = i0 + n * kWave, use = i < all ? i : i0;
      const bool value = use >= others;
      const unsigned int in = value ? use - others : use;
      const unsigned int h = div_u32(in, value ? a.by_head.m : a.by_rest.m, value ? a.by_head.d : a.by_rest.d);
      const unsigned int at = ((value ? 0u : a.rotary) + (in - h * (value ? head_units : rest)) * kUnit) * sizeof(E);
      x[n] = *reinterpret_cast<const Copy*>((value ? v + h * a.v_head : source(h)) + at);
      dst[n] = (value ? layer + a.plane_bytes + h * head_bytes : target(h)) + at;
    }
#pragma unroll
    for (int n = 0; n < kCopies; ++n)
      if (i0 + n * kWave < all) *reinterpret_cast<Copy*>(dst[n]) = x[n];
  }
}

// A thread for each unit of a token, first those that are rotated, and several tokens to a workgroup: where a
// token has no more units than a workgroup threads (32768 tokens of 2 + 2 x 1 heads of 64 11.1 us, by rotate_rows
// 24.4; 4 + 2 x 1 of 128 31.6 and 34.9; 16 + 2 x 2 of 128, half of them rotated, 75.0 and 82.3), and twice that
// where there are a few hundred tokens (64 of 32 + 2 x 8 heads of 128 3.6 us and 3.9, 256 of them 4.0 and 4.3, 512
// 5.7 and 4.7, 32768 209 and 148, as each unit loads its own cosines).
template <typename E, int N, int kUnit, bool kAdjacent>
__global__ __launch_bounds__(2 * kStepThreads) void rotate_small(SmallArgs a) {
  typedef typename Values<E, N>::type Unit;
  typedef typename Values<uint16_t, kUnit>::type Copy;
  const unsigned int head_bytes = a.dim * sizeof(E), pairs = a.rotary / 2, turned = a.together * a.by_turned.d;
  const bool turns = threadIdx.x < turned;
  const Divider by = turns ? a.by_turned : a.by_copied;
  const unsigned int i = turns ? threadIdx.x : threadIdx.x - turned, among = div_u32(i, by.m, by.d);
  const unsigned int unit = i - among * by.d, token = a.first + blockIdx.x * a.together + among;
  if (among >= a.together || token >= a.tokens) return;
  const long long slot = a.slots[token];
  const bool write = slot >= 0 && (unsigned long long)slot < a.slot_count;
  unsigned char* const out = a.out + (unsigned long long)token * a.q_heads * head_bytes;
  unsigned char* const layer = a.layer + (write ? (unsigned long long)slot : 0ull) * a.kv_heads * head_bytes;
  const unsigned int others = (a.dim - a.rotary) / kUnit * (a.q_heads + a.kv_heads);
  const bool value = !turns && unit >= others;
  const unsigned int in = value ? unit - others : unit;
  const Divider by_head = turns ? a.by_units : value ? a.by_head : a.by_rest;
  const unsigned int h = div_u32(in, by_head.m, by_head.d), u = in - h * by_head.d;
  const bool query = !value && h < a.q_heads;
  if (!query && !write) return;
  const unsigned int own = query || value ? h : h - a.q_heads;  // its head of Q, K or V
  const unsigned char* const src = query   ? a.q + token * a.q_row + own * a.q_head
                                   : value ? a.v + token * a.v_row + own * a.v_head
                                           : a.k + token * a.k_row + own * a.k_head;
  unsigned char* const dst = (query ? out : layer + (value ? a.plane_bytes : 0ull)) + own * head_bytes;
  if (turns) {
    const unsigned int at = (kAdjacent ? 2 * N : N) * sizeof(E) * u;
    const unsigned int at2 = at + (kAdjacent ? N : pairs) * sizeof(E);
    const Unit x = *reinterpret_cast<const Unit*>(src + at), y = *reinterpret_cast<const Unit*>(src + at2);
    const long long position = a.positions[token];
    const bool known = position >= 0 && (unsigned long long)position < a.table_rows;
    const float* const table = a.table + (known ? (unsigned long long)position * a.rotary : 0ull) + u * N;
    float c[N], s[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      c[n] = known ? table[n] : NAN;
      s[n] = known ? table[pairs + n] : NAN;
    }
    turn<E, N, kAdjacent>(x, y, c, s, dst + at, dst + at2);
  } else {
    const unsigned int at = ((value ? 0u : a.rotary) + u * kUnit) * sizeof(E);
    *reinterpret_cast<Copy*>(dst + at) = *reinterpret_cast<const Copy*>(src + at);
  }
}

// As many heads at once as a lane has, up to 5: 32768 tokens of 32 + 8 heads of 128, five of them for a lane,
// 146 us at 5, 149 at 3, 153 at 1; of 24 + 3 heads of 128, 32 of them rotated, one for a lane, 100.7 us at 1, 107 at
// 3, 141 at 5, as places past the last head load it again.
template <typename E, int N, int kUnit, bool kAdjacent>
void launch_batch(RotateArgs a, hipStream_t stream) {
  const unsigned int own = (a.q_heads + a.kv_heads + a.lanes_heads - 1) / a.lanes_heads;
  const unsigned int batch = own == 1 ? 1 : own <= 3 ? 3 : 5;
  const unsigned int copies = ((a.dim - a.rotary) * (a.q_heads + a.kv_heads) + a.dim * a.kv_heads) / kUnit;
  a.by_rest = make_divider((a.dim - a.rotary) / kUnit);
  a.by_head = make_divider(a.dim / kUnit);
  const unsigned int turned = a.units * (a.q_heads + a.kv_heads);
  const unsigned int units = turned + copies;
  if (units <= kStepThreads || (units <= 2 * kStepThreads && a.tokens <= kFewTokens)) {
    SmallArgs m{a};
    const dim3 threads(units <= kStepThreads ? kStepThreads : 2 * kStepThreads);
    m.together = threads.x / units;
    m.by_units = make_divider(a.units);
    m.by_turned = make_divider(turned);
    m.by_copied = make_divider(copies);
    const unsigned int most = kMostSmall * m.together;
    for (m.first = 0; m.first < a.tokens; m.first += std::min(most, a.tokens - m.first))
      hipLaunchKernelGGL((rotate_small<E, N, kUnit, kAdjacent>),
                         dim3((std::min(most, a.tokens - m.first) + m.together - 1) / m.together), threads, 0, stream,
                         m);
    return;
  }
  // (one of each sort, or up to 8 in all, at most half of them rotating)
  auto waves = [](unsigned int work, unsigned int each) { return std::max((work + each - 1) / each, 1u); };
  a.rotating = std::min(waves(own, kRotatedBatches * batch), 4u);
  a.waves_log = 1;
  while (a.waves_log < 3 && 1u << a.waves_log < a.rotating + waves(copies, kCopiedUnits * kWave)) ++a.waves_log;
  constexpr unsigned int kWaves = kStepThreads / kWave;
  const unsigned int most = kMostRotated >> a.waves_log;
  for (unsigned int left = a.tokens; left != 0;) {
    const unsigned int now = std::min(left, most);
    a.first = a.tokens - left;
    const dim3 grid(((now << a.waves_log) + kWaves - 1) / kWaves), threads(kStepThreads);
    if (batch == 1)
      hipLaunchKernelGGL((rotate_rows<E, N, kUnit, kAdjacent, 1>), grid, threads, 0, stream, a);
    else if (batch == 3)
      hipLaunchKernelGGL((rotate_rows<E, N, kUnit, kAdjacent, 3>), grid, threads, 0, stream, a);
    else
      hipLaunchKernelGGL((rotate_rows<E, N, kUnit, kAdjacent, 5>), grid, threads, 0, stream, a);
    left -= now;
  }
}

// unit: values of a copy
template <typename E, bool kAdjacent>
void launch_rotate(const RotateArgs& a, unsigned int unit, hipStream_t stream) {
  if (unit == 8)
    launch_batch<E, 8, 8, kAdjacent>(a, stream);
  else if (unit == 4)
    launch_batch<E, 2, 4, kAdjacent>(a, stream);
  else
    launch_batch<E, 1, 1, kAdjacent>(a, stream);
}

}  // namespace
}  // namespace unchainkv

using namespace unchainkv;

extern "C" long long kvq_splitzip_plan_step_paged(
    unsigned long long new_tokens_ptr, unsigned long long cached_tokens_ptr,
    unsigned long long requests, unsigned long long tables_ptr, unsigned long long table_stride,
    unsigned long long table_width, unsigned long long free_blocks_ptr,
    unsigned long long free_count, unsigned long long free_start_ptr,
    unsigned long long block_tokens, unsigned long long max_tokens,
    unsigned long long query_starts_ptr, unsigned long long context_tokens_ptr,
    unsigned long long slots_ptr, unsigned long long positions_ptr,
    unsigned long long free_next_ptr, unsigned long long lacking_ptr,
    unsigned long long stream_ptr) {
  constexpr unsigned long long kMost = 0x7FFFFFFFull;
  if (new_tokens_ptr == 0 || cached_tokens_ptr == 0 || requests == 0 || requests > kMost ||
      tables_ptr == 0 || table_width == 0 || table_width > kMost || table_stride < table_width ||
      (free_blocks_ptr == 0 && free_count != 0) || free_count > kMost || free_start_ptr == 0 ||
      block_tokens == 0 || block_tokens > kMost || max_tokens > kMost || query_starts_ptr == 0 ||
      context_tokens_ptr == 0 || (max_tokens != 0 && (slots_ptr == 0 || positions_ptr == 0)) ||
      free_next_ptr == 0 || lacking_ptr == 0)
    return 0;
  // every workgroup reads the inputs while others write results
  const unsigned long long in[][2] = {
      {new_tokens_ptr, 4 * requests}, {cached_tokens_ptr, 4 * requests},
      {free_blocks_ptr, 4 * free_count}, {free_start_ptr, 4}};
  const unsigned long long out[][2] = {
      {tables_ptr, 4 * ((requests - 1) * table_stride + table_width)},
      {query_starts_ptr, 4 * (requests + 1)}, {context_tokens_ptr, 4 * requests},
      {slots_ptr, 8 * max_tokens}, {positions_ptr, 8 * max_tokens}, {free_next_ptr, 4},
      {lacking_ptr, 4}};
  for (const auto& o : out) {
    for (const auto& i : in)
      if (overlap(o[0], o[1], i[0], i[1])) return 0;
    for (const auto& p : out)
      if (&o != &p && overlap(o[0], o[1], p[0], p[1])) return 0;
  }
  PlanArgs a{};
  a.new_tokens = reinterpret_cast<const int*>(new_tokens_ptr);
  a.cached_tokens = reinterpret_cast<const int*>(cached_tokens_ptr);
  a.tables = reinterpret_cast<int*>(tables_ptr);
  a.free_blocks = reinterpret_cast<const int*>(free_blocks_ptr);
  a.free_start = reinterpret_cast<const int*>(free_start_ptr);
  a.query_starts = reinterpret_cast<int*>(query_starts_ptr);
  a.context_tokens = reinterpret_cast<int*>(context_tokens_ptr);
  a.slots = reinterpret_cast<long long*>(slots_ptr);
  a.positions = reinterpret_cast<long long*>(positions_ptr);
  a.free_next = reinterpret_cast<int*>(free_next_ptr);
  a.lacking = reinterpret_cast<int*>(lacking_ptr);
  a.table_stride = table_stride;
  a.requests = (unsigned int)requests;
  a.width = (unsigned int)table_width;
  a.block_tokens = (unsigned int)block_tokens;
  a.free_count = (unsigned int)free_count;
  a.max_tokens = (unsigned int)max_tokens;
  const unsigned long long grid = std::min<unsigned long long>(
      std::max<unsigned long long>(1, (max_tokens + kStepThreads - 1) / kStepThreads), 512);
  hipLaunchKernelGGL(plan_step, dim3((unsigned int)grid), dim3(kStepThreads), 0,
                     reinterpret_cast<hipStream_t>(stream_ptr), a);
  const hipError_t st = hipGetLastError();
  if (st != hipSuccess) return fail("plan_step", st);
  return (long long)requests;
}

extern "C" long long kvq_splitzip_write_kv_paged(
    unsigned long long k_ptr, unsigned long long v_ptr, unsigned long long tokens,
    unsigned long long heads, unsigned long long head_bytes, unsigned long long k_row_bytes,
    unsigned long long k_head_bytes, unsigned long long v_row_bytes,
    unsigned long long v_head_bytes, unsigned long long kv_ptr, unsigned long long plane_bytes,
    unsigned long long slot_count, unsigned long long slots_ptr, unsigned long long stream_ptr) {
  constexpr unsigned long long kMost = 0x7FFFFFFFull;
  if (k_ptr == 0 || v_ptr == 0 || tokens == 0 || tokens > kMost || heads == 0 || head_bytes == 0 ||
      heads > kMost || head_bytes > kMost || heads * head_bytes > kMost || kv_ptr == 0 ||
      slots_ptr == 0 || slot_count > kMost ||
      slot_count * heads * head_bytes > plane_bytes)
    return 0;
  const unsigned long long layer_bytes = plane_bytes + slot_count * heads * head_bytes;
  if (overlap(kv_ptr, layer_bytes, k_ptr,
              (tokens - 1) * k_row_bytes + (heads - 1) * k_head_bytes + head_bytes) ||
      overlap(kv_ptr, layer_bytes, v_ptr,
              (tokens - 1) * v_row_bytes + (heads - 1) * v_head_bytes + head_bytes) ||
      overlap(kv_ptr, layer_bytes, slots_ptr, 8 * tokens))
    return 0;
  WriteArgs a{};
  a.layer = reinterpret_cast<unsigned char*>(kv_ptr);
  a.plane_bytes = plane_bytes;
  a.row_bytes = heads * head_bytes;
  a.slot_count = slot_count;
  a.k_row = k_row_bytes;
  a.v_row = v_row_bytes;
  a.k_head = k_head_bytes;
  a.v_head = v_head_bytes;
  // the largest unit that every row, head and address is a multiple of
  const unsigned long long all = k_ptr | v_ptr | kv_ptr | head_bytes | k_row_bytes | v_row_bytes |
                                 plane_bytes | (heads > 1 ? k_head_bytes | v_head_bytes : 0);
  const unsigned int unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4
                            : all % 2 == 0 ? 2 : 1;
  a.units = (unsigned int)(a.row_bytes / unit);
  a.head_units = (unsigned int)(head_bytes / unit);
  a.by_units = make_divider(a.units);
  a.by_head = make_divider(a.head_units);
  if (a.units > 1u << 20) return 0;  // (a row of that size has no use)
  // units of a launch: few enough for 32-bit indexes with the last iteration's overhang
  const unsigned long long most = (1u << 30) / a.units;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  for (unsigned long long first = 0; first < tokens; first += most) {
    a.tokens = (unsigned int)std::min(most, tokens - first);
    a.k = reinterpret_cast<const unsigned char*>(k_ptr + first * k_row_bytes);
    a.v = reinterpret_cast<const unsigned char*>(v_ptr + first * v_row_bytes);
    a.slots = reinterpret_cast<const long long*>(slots_ptr) + first;
    const unsigned int total = a.tokens * a.units;
    const dim3 g(std::min<unsigned int>((total + kStepThreads - 1) / kStepThreads, 4096));
    const dim3 t(kStepThreads);
    if (unit == 16)
      hipLaunchKernelGGL(write_rows<u32x4>, g, t, 0, stream, a);
    else if (unit == 8)
      hipLaunchKernelGGL(write_rows<u32x2>, g, t, 0, stream, a);
    else if (unit == 4)
      hipLaunchKernelGGL(write_rows<uint32_t>, g, t, 0, stream, a);
    else if (unit == 2)
      hipLaunchKernelGGL(write_rows<uint16_t>, g, t, 0, stream, a);
    else
      hipLaunchKernelGGL(write_rows<unsigned char>, g, t, 0, stream, a);
    const hipError_t st = hipGetLastError();
    if (st != hipSuccess) return fail("write_rows", st);
  }
  return (long long)(2 * tokens * a.row_bytes);
}

extern "C" long long kvq_splitzip_rotate_write_kv_paged(
    unsigned long long q_ptr, unsigned long long q_row_bytes, unsigned long long q_head_bytes,
    unsigned long long q_heads, unsigned long long k_ptr, unsigned long long k_row_bytes,
    unsigned long long k_head_bytes, unsigned long long v_ptr, unsigned long long v_row_bytes,
    unsigned long long v_head_bytes, unsigned long long tokens, unsigned long long kv_heads,
    unsigned long long head_dim, unsigned long long dtype, unsigned long long kv_ptr,
    unsigned long long plane_bytes, unsigned long long slot_count, unsigned long long slots_ptr,
    unsigned long long positions_ptr, unsigned long long rotation_ptr, unsigned long long rotation_rows,
    unsigned long long rotary_dim, unsigned long long adjacent, unsigned long long out_ptr,
    unsigned long long stream_ptr) {
  constexpr unsigned long long kMost = 0x7FFFFFFFull, kMostHeads = 65536, kMostDim = 4096;
  if (q_ptr == 0 || k_ptr == 0 || v_ptr == 0 || kv_ptr == 0 || slots_ptr == 0 || positions_ptr == 0 ||
      rotation_ptr == 0 || out_ptr == 0 || tokens == 0 || tokens > kMost || q_heads == 0 ||
      q_heads > kMostHeads || kv_heads == 0 || kv_heads > kMostHeads || head_dim == 0 ||
      head_dim > kMostDim || rotary_dim == 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim ||
      rotation_rows == 0 || rotation_rows > kMost || dtype > 1 || slot_count > kMost || rotation_ptr % 4 != 0 ||
      (q_ptr | q_row_bytes | q_head_bytes | k_ptr | k_row_bytes | k_head_bytes | v_ptr | v_row_bytes |
       v_head_bytes | kv_ptr | plane_bytes | out_ptr) % 2 != 0)
    return 0;
  const unsigned long long head_bytes = 2 * head_dim, row_bytes = kv_heads * head_bytes;
  if (slot_count * row_bytes > plane_bytes) return 0;
  const unsigned long long in[][2] = {
      {q_ptr, (tokens - 1) * q_row_bytes + (q_heads - 1) * q_head_bytes + head_bytes},
      {k_ptr, (tokens - 1) * k_row_bytes + (kv_heads - 1) * k_head_bytes + head_bytes},
      {v_ptr, (tokens - 1) * v_row_bytes + (kv_heads - 1) * v_head_bytes + head_bytes},
      {slots_ptr, 8 * tokens}, {positions_ptr, 8 * tokens}, {rotation_ptr, 4 * rotation_rows * rotary_dim}};
  const unsigned long long out[][2] = {{kv_ptr, plane_bytes + slot_count * row_bytes},
                                       {out_ptr, tokens * q_heads * head_bytes}};
  for (const auto& o : out)
    for (const auto& i : in)
      if (overlap(o[0], o[1], i[0], i[1])) return 0;
  if (overlap(out[0][0], out[0][1], out[1][0], out[1][1])) return 0;
  // 8 values at a time where every row, head and address allows it, and both parts of a head are such runs;
  // else two pairs and copies of 4 values, or one by one
  const unsigned long long all = q_ptr | q_row_bytes | k_ptr | k_row_bytes | v_ptr | v_row_bytes | kv_ptr |
                                 plane_bytes | out_ptr | (q_heads > 1 ? q_head_bytes : 0) |
                                 (kv_heads > 1 ? k_head_bytes | v_head_bytes : 0) | head_bytes;
  const unsigned int unit = (all | rotary_dim) % 16 == 0 ? 8 : (all | 2 * rotary_dim) % 8 == 0 ? 4 : 1;
  RotateArgs a{};
  a.q = reinterpret_cast<const unsigned char*>(q_ptr);
  a.k = reinterpret_cast<const unsigned char*>(k_ptr);
  a.v = reinterpret_cast<const unsigned char*>(v_ptr);
  a.out = reinterpret_cast<unsigned char*>(out_ptr);
  a.layer = reinterpret_cast<unsigned char*>(kv_ptr);
  a.table = reinterpret_cast<const float*>(rotation_ptr);
  a.slots = reinterpret_cast<const long long*>(slots_ptr);
  a.positions = reinterpret_cast<const long long*>(positions_ptr);
  a.q_row = q_row_bytes;
  a.q_head = q_head_bytes;
  a.k_row = k_row_bytes;
  a.k_head = k_head_bytes;
  a.v_row = v_row_bytes;
  a.v_head = v_head_bytes;
  a.plane_bytes = plane_bytes;
  a.slot_count = slot_count;
  a.table_rows = rotation_rows;
  a.tokens = (unsigned int)tokens;
  a.q_heads = (unsigned int)q_heads;
  a.kv_heads = (unsigned int)kv_heads;
  a.dim = (unsigned int)head_dim;
  a.rotary = (unsigned int)rotary_dim;
  a.units = (unsigned int)(rotary_dim / 2 / (unit == 8 ? 8 : unit == 4 ? 2 : 1));
  a.lanes_heads = std::max(1u, kWave / a.units);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  if (dtype == 0)
    adjacent ? launch_rotate<__bf16, true>(a, unit, stream) : launch_rotate<__bf16, false>(a, unit, stream);
  else
    adjacent ? launch_rotate<_Float16, true>(a, unit, stream) : launch_rotate<_Float16, false>(a, unit, stream);
  const hipError_t st = hipGetLastError();
  if (st != hipSuccess) return fail("rotate_rows", st);
  return (long long)(2 * tokens * (q_heads * head_bytes + 2 * row_bytes));
}
