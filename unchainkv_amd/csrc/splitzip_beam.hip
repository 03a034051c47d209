// A beam search's step over paged layers, gfx950: the best continuations of a request's beams, and the block
// tables and layers in the order of the chosen parents.
//
// Select. Beam b offers token t at x[b][t] - m - log sum_t exp(x[b][t] - m) + score[b], m = max_t x[b][t]; of all
// beams and tokens the best n are given, equal ones by their places.
//   * beam_scan reads every logit once, a wave 4 KB of a row at a time, and keeps the maximum of each 256 of them
//     and, of each wave's share, (m, sum exp(x - m)): one pass, sums in f32 of at most 32 terms a lane. Bound by
//     HBM: 64 requests of 8 beams (one of them finished), 131072 logits in bf16, 117 MB: 24.0 us, 4.9 TB/s (a
//     large copy: 5.1). A lane takes 64 bytes that follow each other: with 16 a lane, interleaved, a maximum of
//     256 took five exchanges for each 8 logits and the call 28.5 us.
//   * beam_pick, a workgroup for each request, joins the sums in 64 bits and searches. The best n values lie in
//     the n segments with the largest maxima (equal ones: the first), as each of n segments that come before a
//     value's own holds one that comes before it. So: a bound that n of some wave's lanes reach; the segments above
//     it, ranked; the logits of the best n of them, read again, that are no less than the n-th maximum; ranked.
//     Nothing here grows with the vocabulary but the maxima's loads. Bound by latency: 12.0 us for the call above,
//     6.8 for one request of 4 beams, 32000 logits (loads 1.5 us, twice; log, bound and lists; 49 us when every
//     list was formed by taking one maximum after another).
// Values are formed and compared in 64 bits from a row's sum, whose terms and joins within a wave are in 32: a
// beam's own offers come in their exact order, and those of two beams wherever they differ by more than the
// roundings of the two sums, at most 2^-16.7 of each. (32 bits of a sum of log probabilities would not even hold
// differences that exact sums leave.) Scores of 131072 bf16 logits are off by 2.6e-8 of their size, with sums in 64
// bits by 2.5e-8, the last rounding's.
//
// Reorder. Row r * beams + j follows parent p[j]. One thread reads all beams' entries of a column and then
// writes them, so that a table can be reordered in place: entries of full blocks are shared. The last, partly
// filled block goes on with its first child; the others take, in order, blocks that no parent's row has, and copy
// its tokens. Blocks of the context that no row of the request lists any more go below the free list's first
// entry, in an order that does not depend on the launch (request, column, beam). Two launches, order_tables and
// copy_tails, as the list needs all tables' counts and the copies the tables' last blocks. Bound by latency: 3.5 +
// 3.5 us for one request of 4 beams and 16 layers, 6.2 + 7.4 for 48 of 4 and 8 layers (33 MB read and written).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "splitzip_common.h"

namespace unchainkv {
namespace {

constexpr int kScanThreads = 256;
constexpr int kLaneBytes = 64;                                // of a row that a lane takes at a time
constexpr int kSegment = 256;                                 // logits whose maximum is kept
constexpr unsigned int kGridRows = 32768;                     // of a grid's second dimension
constexpr int kPickThreads = 1024;
constexpr int kMostBeams = 32, kMostCandidates = 64;
constexpr int kMostItems = 8;                                 // segments that a lane of beam_pick holds
constexpr int kOwnTokens = kSegment / kWave;                  // tokens of one
// Chunks of a request's rows, 4 KB each, up to which beam_pick scans them by itself, a wave each: one launch (4 beams,
// 8000 logits in bf16, captured: 9.7 us and 9.9, 300 logits 9.5 and 10.8, and 3.5 us less of the host's time; twice as
// many chunks 12.2 and 10.0, as a CU reads no faster).
constexpr unsigned int kWholeChunks = 16;
constexpr unsigned int kChunkSegments = kWave * kLaneBytes / 2 / kSegment;  // of one, at most
constexpr unsigned int kMostVocab = 1u << 20;
static_assert(kMostVocab <= 8 * kMostItems * kWave * kSegment, "the largest groups hold a row");
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2E = 1.4426950408889634f;

struct SelectArgs {
  const unsigned char* logits;     // [requests][beams][vocab], strides in elements
  const float* scores;             // [requests][beams]
  const unsigned char* ended;      // [requests][beams] or null
  float* maxima;                   // [requests * beams][segments]
  float2* sums;                    // [requests * beams][chunks]: (max, sum)
  float* out_scores;               // [requests][candidates]
  int* out_parents;
  long long* out_tokens;
  unsigned long long request_stride, beam_stride;
  unsigned int requests, beams, vocab, candidates, end_token;
  unsigned int segments, chunks;  // of a row
  unsigned int parts;         // waves that search a beam
  unsigned int group, items;  // segments of an item, items of a row
};

// Logits by their type, 16 bytes of them from any address.
struct Bf16 {
  typedef struct __attribute__((packed, aligned(2))) { u32x4 v; } Raw;
  static constexpr int kBytes = 2, kLoad = 8;
  static __device__ __forceinline__ float one(const unsigned char* p, unsigned int i) {
    return __uint_as_float((unsigned int)reinterpret_cast<const uint16_t*>(p)[i] << 16);
  }
  static __device__ __forceinline__ float of(const Raw& r, int i) {
    return __uint_as_float(i % 2 == 0 ? r.v[i / 2] << 16 : r.v[i / 2] & 0xFFFF0000u);
  }
};
struct Fp16 {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef struct __attribute__((packed, aligned(2))) { x8 v; } Raw;
  static constexpr int kBytes = 2, kLoad = 8;
  static __device__ __forceinline__ float one(const unsigned char* p, unsigned int i) {
    return (float)reinterpret_cast<const _Float16*>(p)[i];
  }
  static __device__ __forceinline__ float of(const Raw& r, int i) { return (float)r.v[i]; }
};
struct Fp32 {
  typedef float x4 __attribute__((ext_vector_type(4)));
  typedef struct __attribute__((packed, aligned(4))) { x4 v; } Raw;
  static constexpr int kBytes = 4, kLoad = 4;
  static __device__ __forceinline__ float one(const unsigned char* p, unsigned int i) {
    return reinterpret_cast<const float*>(p)[i];
  }
  static __device__ __forceinline__ float of(const Raw& r, int i) { return r.v[i]; }
};
template <typename T>
constexpr int kLaneLogits = kLaneBytes / T::kBytes;

// A beam that offers no token of its own: finished, or without a hypothesis yet.
__device__ __forceinline__ bool is_ended(const SelectArgs& a, unsigned int row) {
  return a.ended != nullptr && a.ended[row] != 0;
}
__device__ __forceinline__ bool is_open(const SelectArgs& a, unsigned int row) {
  return !is_ended(a, row) && a.scores[row] != -INFINITY;
}

template <typename T>
__device__ __forceinline__ const unsigned char* row_of(const SelectArgs& a, unsigned int row) {
  const unsigned int request = row / a.beams;
  return a.logits + (request * a.request_stride + (row - request * a.beams) * a.beam_stride) * T::kBytes;
}

template <int kControl, int kRowMask>
__device__ __forceinline__ float shifted(float v) {
  const int u = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, kControl, kRowMask, 0xF, false));
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, shifted<0x111, 0xF>(v));
  v = fmaxf(v, shifted<0x112, 0xF>(v));
  v = fmaxf(v, shifted<0x114, 0xF>(v));
  v = fmaxf(v, shifted<0x118, 0xF>(v));
  v = fmaxf(v, shifted<0x142, 0xA>(v));
  v = fmaxf(v, shifted<0x143, 0xC>(v));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// A row's chunk by a wave: 64 lanes' 64 bytes; a lane's logits follow each other, so that a segment's maximum
// takes three or four exchanges between lanes for 32 or 16 logits of each. maxima, sums: the row's.
template <typename T>
__device__ __forceinline__ void scan_chunk(const SelectArgs& a, unsigned int row, unsigned int chunk, float* maxima,
                                           float2* sums) {
  constexpr int kOwn = kLaneLogits<T>, kLoads = kOwn / T::kLoad, kLanes = kSegment / kOwn;
  const unsigned int lane = __lane_id();
  const unsigned char* src = row_of<T>(a, row);
  const unsigned int base = chunk * (kWave * kOwn);
  const unsigned int at = base + lane * kOwn;
  float x[kOwn];
  if (base + kWave * kOwn <= a.vocab) {
    typename T::Raw raw[kLoads];
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      raw[n] = *reinterpret_cast<const typename T::Raw*>(src + (at + n * T::kLoad) * T::kBytes);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) x[i] = T::of(raw[i / T::kLoad], i % T::kLoad);
  } else if (a.vocab >= T::kLoad) {
    // The row's end: loads that would pass it are of its last logits, of which those count that no load before
    // has (all go out together; behind a branch for each the call took 1.5 us more).
    typename T::Raw raw[kLoads];
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      raw[n] = *reinterpret_cast<const typename T::Raw*>(
          src + min(at + n * T::kLoad, a.vocab - T::kLoad) * T::kBytes);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const unsigned int from = at + i / T::kLoad * T::kLoad;
      x[i] = from + T::kLoad <= a.vocab + i % T::kLoad ? T::of(raw[i / T::kLoad], i % T::kLoad) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) x[i] = at + i < a.vocab ? T::one(src, at + i) : -INFINITY;
  }
  float own = x[0];
#pragma unroll
  for (int i = 1; i < kOwn; ++i) own = fmaxf(own, x[i]);
  const float top = fmaxf(own, kLowest);
  float sum = 0.f;
  if (__all(fabsf(top) < 1e6f)) {
    // 2^(x log2 e - r) with one rounding, r = top log2 e rounded, and that rounding put right in the sum
    const float r = top * kLog2E;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum += __builtin_amdgcn_exp2f(fmaf(x[i], kLog2E, -r));
    sum *= __builtin_amdgcn_exp2f(-fmaf(top, kLog2E, -r));
  } else {
    // (no logit but -inf, or values whose products with log2 e leave the range or its small steps)
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum += __builtin_amdgcn_exp2f((x[i] - top) * kLog2E);
  }
  // (a NaN, or infinity, which makes the row's sum NaN: every value that is not -inf is then NaN)
  own = sum != sum ? INFINITY : own;
  own = fmaxf(own, shifted<0x111, 0xF>(own));
  own = fmaxf(own, shifted<0x112, 0xF>(own));
  own = fmaxf(own, shifted<0x114, 0xF>(own));
  if constexpr (kLanes == 16) own = fmaxf(own, shifted<0x118, 0xF>(own));
  const unsigned int segment = at / kSegment;
  if (lane % kLanes == kLanes - 1 && segment < a.segments)
    maxima[segment] = own;
  const float big = wave_max(top);
  sum *= __builtin_amdgcn_exp2f((top - big) * kLog2E);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d, kWave);
  if (lane == 0) sums[chunk] = make_float2(big, sum);
}

template <typename T>
__global__ __launch_bounds__(kScanThreads) void beam_scan(SelectArgs a) {
  const unsigned int row = blockIdx.z * kGridRows + blockIdx.y;
  const unsigned int chunk = uniform(blockIdx.x * (kScanThreads / kWave) + (threadIdx.x >> 6));
  if (chunk >= a.chunks || row >= a.requests * a.beams || !is_open(a, row)) return;
  scan_chunk<T>(a, row, chunk, a.maxima + (unsigned long long)row * a.segments,
                a.sums + (unsigned long long)row * a.chunks);
}

// Values as numbers that compare alike: NaN above all, -0 as 0, nothing as 0.
__device__ __forceinline__ unsigned long long key_of(double v) {
  if (v != v) return ~0ull;
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v + 0.0);
  return (u >> 63) != 0 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double value_of(unsigned long long key) {
  if (key == ~0ull) return NAN;
  return __builtin_bit_cast(double, (key >> 63) != 0 ? key & ~(1ull << 63) : ~key);
}

// The wave's largest.
template <int kControl, int kRowMask>
__device__ __forceinline__ unsigned long long larger(unsigned long long v) {
  const int lo = (int)v, hi = (int)(v >> 32);
  const unsigned int olo = (unsigned int)__builtin_amdgcn_update_dpp(lo, lo, kControl, kRowMask, 0xF, false);
  const unsigned int ohi = (unsigned int)__builtin_amdgcn_update_dpp(hi, hi, kControl, kRowMask, 0xF, false);
  const unsigned long long o = (unsigned long long)ohi << 32 | olo;
  return o > v ? o : v;
}
__device__ __forceinline__ unsigned long long wave_largest(unsigned long long v) {
  v = larger<0x111, 0xF>(v);
  v = larger<0x112, 0xF>(v);
  v = larger<0x114, 0xF>(v);
  v = larger<0x118, 0xF>(v);
  v = larger<0x142, 0xA>(v);
  v = larger<0x143, 0xC>(v);
  const unsigned int lo = (unsigned int)__builtin_amdgcn_readlane((int)(unsigned int)v, 63);
  const unsigned int hi = (unsigned int)__builtin_amdgcn_readlane((int)(v >> 32), 63);
  return (unsigned long long)hi << 32 | lo;
}

struct Beam {
  double top, rest, score;  // the largest logit, and log sum exp(x - top)
  bool open, ended;
  // what a token of some logit is worth (of a beam that is not open, none); the largest logit first, beside
  // which the logarithm would be lost where all are masked by their type's lowest value
  __device__ __forceinline__ unsigned long long key(float logit) const {
    return logit == -INFINITY ? key_of(-INFINITY) : key_of(((double)logit - top) - rest + score);
  }
};

// The best of a wave's keys (key t of lane l has number t * 64 + l, 0: none), best first, equal ones by
// their numbers, and at most `most`; take(key, number, n) for each, by all lanes.
template <int kCount, typename Take>
__device__ __forceinline__ void best_of(unsigned long long (&keys)[kCount], unsigned int most, Take take) {
  const unsigned int lane = __lane_id();
  for (unsigned int n = 0; n < most; ++n) {
    unsigned long long own = keys[0];
#pragma unroll
    for (int t = 1; t < kCount; ++t) own = keys[t] > own ? keys[t] : own;
    const unsigned long long best = wave_largest(own);
    if (best == 0) break;
    unsigned int number = ~0u;
#pragma unroll
    for (int t = kCount - 1; t >= 0; --t) {
      const unsigned long long equal = __ballot(keys[t] == best);
      if (equal != 0) number = t * kWave + (unsigned int)__ffsll((long long)equal) - 1;
    }
#pragma unroll
    for (int t = 0; t < kCount; ++t)
      if (t * kWave + lane == number) keys[t] = 0;
    take(best, number, n);
  }
}

// A bound that at least `most` of the lanes' keys reach, nearly the largest one; 0 where there are not that
// many: bits from the top, each kept while enough lanes have no less. (18 of them, with steps of 2^-6 of a
// value: the others would take as long and spare few of the keys.)
__device__ __forceinline__ unsigned long long reached(unsigned long long key, unsigned int most) {
  const unsigned int high = (unsigned int)(key >> 32);
  unsigned int bound = 0;
  for (unsigned int bit = 1u << 31; bit >= 1u << 14; bit >>= 1) {
    const unsigned int count = (unsigned int)__popcll(__ballot(high >= (bound | bit)));
    if (count < most) continue;
    bound |= bit;
    if (count == most) break;
  }
  return (unsigned long long)bound << 32;
}

// How many of a list come before (key, id).
__device__ __forceinline__ unsigned int rank_of(const unsigned long long* keys, const unsigned int* ids,
                                                unsigned int count, unsigned long long key, unsigned int id) {
  unsigned int rank = 0;
#pragma unroll 8
  for (unsigned int j = 0; j < count; ++j) {
    const unsigned long long k = keys[j];
    const unsigned int i = ids[j];
    rank += (unsigned int)(k > key) | ((unsigned int)(k == key) & (unsigned int)(i < id));
  }
  return rank;
}

// kItems: segments, or groups of them, that a lane holds of a row; kTokens: tokens of a group that it does. kWhole: it
// scans the rows itself before.
template <typename T, int kItems, int kTokens, bool kWhole>
__global__ __launch_bounds__(kPickThreads) void beam_pick(SelectArgs a) {
  constexpr int kWaves = kPickThreads / kWave;
  __shared__ Beam s_beam[kMostBeams];
  // segments that may be among the best, and then values: at most 64 of each wave, and of each segment
  __shared__ unsigned long long s_key[kMostCandidates * kMostCandidates];
  __shared__ unsigned int s_id[kMostCandidates * kMostCandidates];
  __shared__ unsigned long long s_bound[kWaves];
  __shared__ unsigned int s_chosen[kMostCandidates], s_segments, s_count;
  __shared__ unsigned long long s_least;
  __shared__ float s_maxima[kWhole ? kWholeChunks * kChunkSegments : 1];
  __shared__ float2 s_sums[kWhole ? kWholeChunks : 1];
  const unsigned int request = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const unsigned int row0 = request * a.beams, most = a.candidates;
  const unsigned int group = kTokens == kOwnTokens ? 1 : a.group, items = a.items;
  const unsigned int units = a.beams * a.parts;  // a wave's work each
  if (tid == 0) {
    s_segments = s_count = 0;
    s_least = 0;
  }
  if (tid < kMostCandidates) s_chosen[tid] = ~0u;
  if constexpr (kWhole) {
    static_assert(kWholeChunks <= kWaves);
    const unsigned int b = wave / a.chunks;
    if (b < a.beams && is_open(a, row0 + b))
      scan_chunk<T>(a, row0 + b, wave - b * a.chunks, s_maxima + b * a.segments, s_sums + b * a.chunks);
    __syncthreads();
  }

  // A part of a beam's items as keys by their maxima.
  auto load = [&](unsigned int unit, unsigned long long (&keys)[kItems]) {
    const unsigned int b = unit / a.parts, row = row0 + b;
    const unsigned int from = (unit - b * a.parts) * (kItems * kWave) + lane;
    // (all loads go out together; what a beam that is not open has there counts for nothing)
    const float* maxima = kWhole ? s_maxima + b * a.segments : a.maxima + (unsigned long long)row * a.segments;
    const float2* sums = kWhole ? s_sums + b * a.chunks : a.sums + (unsigned long long)row * a.chunks;
    float largest[kItems];
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
      const unsigned int item = min(from + t * kWave, items - 1);
      largest[t] = maxima[item * group];
      for (unsigned int s = item * group + 1; s < min(a.segments, (item + 1) * group); ++s)
        largest[t] = fmaxf(largest[t], maxima[s]);
    }
    const float2 none = make_float2(kLowest, 0.f);
    const float2 own = lane < a.chunks ? sums[lane] : none;
    Beam beam{0., 0., a.scores[row], is_open(a, row), is_ended(a, row)};
    float top = own.x;
    for (unsigned int c = lane + kWave; c < a.chunks; c += kWave) top = fmaxf(top, sums[c].x);
    top = wave_max(top);
    double sum = own.y * __builtin_amdgcn_exp2f((own.x - top) * kLog2E);
    for (unsigned int c = lane + kWave; c < a.chunks; c += kWave)
      sum += sums[c].y * __builtin_amdgcn_exp2f((sums[c].x - top) * kLog2E);
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d, kWave);
    beam.top = top;
    beam.rest = log(sum);
#pragma unroll
    for (int t = 0; t < kItems; ++t) largest[t] = beam.open ? largest[t] : -INFINITY;
    if (lane == 0) s_beam[b] = beam;
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
      const unsigned int item = from + t * kWave;
      keys[t] = beam.key(largest[t]);
      if (beam.ended && a.end_token / (kSegment * group) == item) keys[t] = key_of(beam.score);
      if (item >= items) keys[t] = 0;
    }
  };
  // The items that may be among the best: those that no part has `most` above. Where one has too many, its
  // best `most`.
  auto offer = [&](unsigned int unit, unsigned long long (&keys)[kItems], unsigned long long least) {
    const unsigned int b = unit / a.parts, id0 = b * items + (unit - b * a.parts) * (kItems * kWave);
    unsigned int count = 0;
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
      if (keys[t] < least) keys[t] = 0;
      count += (unsigned int)__popcll(__ballot(keys[t] != 0));
    }
    if (count == 0) return;
    unsigned int at = 0;
    if (lane == 0) at = atomicAdd(&s_segments, count > kMostCandidates ? min(count, most) : count);
    at = uniform(at);
    if (count <= kMostCandidates) {
#pragma unroll
      for (int t = 0; t < kItems; ++t) {
        const unsigned long long mask = __ballot(keys[t] != 0);
        if (keys[t] != 0) {
          const unsigned int to = at + (unsigned int)__popcll(mask & ((1ull << lane) - 1));
          s_key[to] = keys[t];
          s_id[to] = id0 + t * kWave + lane;
        }
        at += (unsigned int)__popcll(mask);
      }
    } else {
      best_of(keys, most, [&](unsigned long long key, unsigned int number, unsigned int n) {
        if (lane == 0) {
          s_key[at + n] = key;
          s_id[at + n] = id0 + number;
        }
      });
    }
  };
  auto largest_of = [&](const unsigned long long (&keys)[kItems]) {
    unsigned long long own = keys[0];
#pragma unroll
    for (int t = 1; t < kItems; ++t) own = keys[t] > own ? keys[t] : own;
    return own;
  };
  // (a wave's first stays in its registers, any others are loaded again: more than 16 beams are rare)
  unsigned long long keys0[kItems], bound = 0;
  for (unsigned int u = wave; u < units; u += kWaves) {
    unsigned long long keys[kItems];
    load(u, keys);
    bound = max(bound, reached(largest_of(keys), most));
    if (u == wave) {
#pragma unroll
      for (int t = 0; t < kItems; ++t) keys0[t] = keys[t];
    }
  }
  if (lane == 0) s_bound[wave] = bound;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) bound = max(bound, s_bound[w]);
  for (unsigned int u = wave; u < units; u += kWaves) {
    if (u == wave) {
      offer(u, keys0, bound);
    } else {
      unsigned long long keys[kItems];
      load(u, keys);
      offer(u, keys, bound);
    }
  }
  __syncthreads();
  // the best `most` of those
  const unsigned int all = s_segments;
  for (unsigned int i = tid; i < all; i += kPickThreads) {
    const unsigned long long key = s_key[i];
    const unsigned int id = s_id[i], rank = rank_of(s_key, s_id, all, key, id);
    if (rank >= most) continue;
    s_chosen[rank] = id;
    if (rank == most - 1) s_least = key;
  }
  __syncthreads();
  // their values that are no less than the last one's, into a list
  const unsigned long long least = s_least;
  for (unsigned int c = wave; c < most; c += kWaves) {
    const unsigned int id = s_chosen[c];
    if (id == ~0u) continue;
    const unsigned int b = id / items, first = (id - b * items) * group * kSegment;
    const Beam beam = s_beam[b];
    const unsigned char* src = row_of<T>(a, row0 + b);
    unsigned long long keys[kTokens], masks[kTokens];
    auto keep = [&](unsigned long long bound) {
      unsigned int count = 0;
#pragma unroll
      for (int t = 0; t < kTokens; ++t) {
        if (keys[t] < bound) keys[t] = 0;
        masks[t] = __ballot(keys[t] != 0);
        count += (unsigned int)__popcll(masks[t]);
      }
      return count;
    };
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const unsigned int in = t * kWave + lane, token = first + in;
      const bool there = in < group * kSegment && token < a.vocab;
      keys[t] = beam.key(beam.open && there ? T::one(src, token) : -INFINITY);
      if (beam.ended && token == a.end_token) keys[t] = key_of(beam.score);
      if (!there) keys[t] = 0;
    }
    unsigned int count = keep(least);
    if (count > most) {
      // (few segments, whose maxima bound too little)
      unsigned long long own = keys[0];
#pragma unroll
      for (int t = 1; t < kTokens; ++t) own = keys[t] > own ? keys[t] : own;
      count = keep(max(1ull, reached(own, most)));
      if (count > kMostCandidates) {
        // Equal ones, as of a beam that is not in use: the first of them, where the largest are enough.
        const unsigned long long top = wave_largest(own);
        unsigned int equal = 0;
#pragma unroll
        for (int t = 0; t < kTokens; ++t) equal += (unsigned int)__popcll(__ballot(keys[t] == top));
        if (equal >= most) {
          unsigned int before = 0;
#pragma unroll
          for (int t = 0; t < kTokens; ++t) {
            const unsigned long long mask = __ballot(keys[t] == top);
            if (keys[t] != top || before + (unsigned int)__popcll(mask & ((1ull << lane) - 1)) >= most) keys[t] = 0;
            before += (unsigned int)__popcll(mask);
          }
          count = keep(1);
        }
      }
    }
    unsigned int at = 0;
    if (lane == 0) at = atomicAdd(&s_count, count > kMostCandidates ? most : count);
    at = uniform(at);
    if (count <= kMostCandidates) {
#pragma unroll
      for (int t = 0; t < kTokens; ++t) {
        if (keys[t] != 0) {
          const unsigned int to = at + (unsigned int)__popcll(masks[t] & ((1ull << lane) - 1));
          s_key[to] = keys[t];
          s_id[to] = b * a.vocab + first + t * kWave + lane;
        }
        at += (unsigned int)__popcll(masks[t]);
      }
    } else {
      best_of(keys, most, [&](unsigned long long key, unsigned int number, unsigned int n) {
        if (lane == 0) {
          s_key[at + n] = key;
          s_id[at + n] = b * a.vocab + first + number;
        }
      });
    }
  }
  __syncthreads();
  const unsigned int count = s_count;
  for (unsigned int i = tid; i < count; i += kPickThreads) {
    const unsigned long long key = s_key[i];
    const unsigned int id = s_id[i];
    const unsigned int rank = rank_of(s_key, s_id, count, key, id);
    if (rank >= most) continue;
    const unsigned long long to = (unsigned long long)request * most + rank;
    const unsigned int b = id / a.vocab;
    a.out_scores[to] = (float)value_of(key);
    a.out_parents[to] = (int)b;
    a.out_tokens[to] = id - b * a.vocab;
  }
}

// ---------------------------------------------------------------------------

constexpr int kOrderThreads = 256;  // columns of a workgroup
constexpr int kOrderWaves = kOrderThreads / kWave;
constexpr unsigned int kAtOnce = 8;  // of a column's entries
constexpr int kMostLayers = 64;     // of a launch

struct OrderArgs {
  const int* tables;               // [requests * beams][table_stride]
  int* out;                        // [requests * beams][out_stride]; may be tables
  const int* parents;              // [requests][beams]
  const int* contexts;             // [requests * beams]
  int* copied_from;                // [requests * beams]
  int* free_blocks;
  const int* free_start;
  int* free_next;
  int* lacking;
  int* unlisted;
  int4* copies;                    // [requests * beams]: block, its copy, tokens; none: -1
  int2* counts;                    // [requests][chunks]: (released, lacking) of a workgroup's columns
  int* released;                   // [requests][chunks][beams * (kOrderThreads + 1)]
  unsigned long long table_stride, out_stride;
  unsigned int requests, beams, width, chunks, block_tokens, free_count;
  Divider by_block;
};

// Exclusive sum over the workgroup, and the whole.
__device__ __forceinline__ unsigned int group_scan(unsigned int v, unsigned int* space, unsigned int& all) {
  const unsigned int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned int scan = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const unsigned int o = (unsigned int)__shfl_up((int)scan, d, kWave);
    if (lane >= (unsigned int)d) scan += o;
  }
  if (lane == 63) space[wave] = scan;
  __syncthreads();
  unsigned int at = scan - v;
  all = 0;
#pragma unroll
  for (unsigned int w = 0; w < kOrderWaves; ++w) {
    if (w < wave) at += space[w];
    all += space[w];
  }
  return at;
}

__global__ __launch_bounds__(kOrderThreads) void order_tables(OrderArgs a) {
  extern __shared__ int s_entry[];  // [beams][kOrderThreads]: a thread's column
  __shared__ int s_parent[kMostBeams], s_spare[kMostBeams];
  __shared__ unsigned int s_wave[kOrderWaves], s_lacking, s_left;
  const unsigned int tid = threadIdx.x, lane = tid & 63;
  const unsigned int request = blockIdx.y, beams = a.beams, row0 = request * beams;
  const unsigned int column = blockIdx.x * kOrderThreads + tid;
  const unsigned int context = (unsigned int)max(a.contexts[row0], 0);
  const unsigned int full = div_u32(context, a.by_block.m, a.by_block.d);
  const unsigned int rest = context - full * a.block_tokens;
  // whether this workgroup has the last, partly filled block's column
  const bool tail = rest != 0 && full < a.width && full / kOrderThreads == blockIdx.x;
  if (tid < beams) s_parent[tid] = a.parents[row0 + tid];
  if (tid == 0) s_lacking = s_left = 0;
  // the last blocks of a lane's beam (read with the rest: nobody else has that column)
  const int last = tail && tid < beams ? a.tables[(row0 + tid) * a.table_stride + full] : -1;
  int* const own = s_entry + tid;
  const bool there = column < a.width && (column < full || a.out != a.tables) && !(tail && column == full);
  bool same = true;
  if (there) {
    int first = 0;
    for (unsigned int b0 = 0; b0 < beams; b0 += kAtOnce) {
      int id[kAtOnce];  // (past the last beam its entry again: the loads wait for none before)
#pragma unroll
      for (unsigned int n = 0; n < kAtOnce; ++n)
        id[n] = a.tables[(row0 + min(b0 + n, beams - 1)) * a.table_stride + column];
      first = b0 == 0 ? id[0] : first;
#pragma unroll
      for (unsigned int n = 0; n < kAtOnce; ++n) {
        if (b0 + n < beams) own[(b0 + n) * kOrderThreads] = id[n];
        same &= id[n] == first;
      }
    }
  }
  __syncthreads();
  const bool known = lane < beams && (unsigned int)s_parent[lane] < beams;
  unsigned int with_child = 0;  // beams that have one
  for (unsigned int j = 0; j < beams; ++j) {
    const unsigned int p = (unsigned int)s_parent[j];
    if (p < beams) with_child |= 1u << p;
  }
  const unsigned int orphans = beams - (unsigned int)__popcll(__ballot(known));

  unsigned int released = 0;  // the beams whose entry of this column is
  if (there) {
    const bool held = column < full;
#pragma unroll 4
    for (unsigned int j = 0; j < beams; ++j) {
      const unsigned int p = held ? (unsigned int)s_parent[j] : j;
      const int id = own[min(p, beams - 1) * kOrderThreads];
      a.out[(row0 + j) * a.out_stride + column] = p < beams ? id : -1;
    }
    if (held && (!same || with_child == 0)) {
      // entries of beams without children that no other beam with one has, once each
      for (unsigned int b = 0; b < beams; ++b) {
        const int id = own[b * kOrderThreads];
        if ((with_child >> b & 1) != 0 || id < 0) continue;
        unsigned int equal = 0;  // the beams that list it
#pragma unroll 8
        for (unsigned int c = 0; c < beams; ++c) equal |= own[c * kOrderThreads] == id ? 1u << c : 0u;
        if ((equal & (with_child | ((1u << b) - 1))) == 0) released |= 1u << b;
      }
    }
  }
  const unsigned int group = request * a.chunks + blockIdx.x;
  int* const list = a.released + (unsigned long long)group * (beams * (kOrderThreads + 1));
  unsigned int all;
  unsigned int at = group_scan((unsigned int)__popc(released), s_wave, all);
  for (; released != 0; released &= released - 1) list[at++] = own[(__ffs((int)released) - 1) * kOrderThreads];

  // The last blocks, by one wave, a lane for each beam: the first child of a block keeps it, the others take
  // those that no child has, in order.
  if (tid < kWave && tail) {
    const int id = last, parent = known ? s_parent[lane] : 0;
    const int source = __shfl(id, parent, kWave);
    bool taken = false, used = false, again = false;
    const unsigned long long children = __ballot(known);
    for (unsigned int j = 0; j < beams; ++j) {
      const bool child = (children >> j & 1) != 0;
      const int its = __builtin_amdgcn_readlane(source, (int)j), other = __builtin_amdgcn_readlane(id, (int)j);
      taken |= child && j < lane && its == source;
      used |= child && its == id;
      again |= j < lane && other == id;
    }
    const bool moves = known && source >= 0 && taken, spare = lane < beams && id >= 0 && !used && !again;
    const unsigned long long below = (1ull << lane) - 1, movers = __ballot(moves), spares = __ballot(spare);
    if (spare) s_spare[__popcll(spares & below)] = id;
    asm volatile("" ::: "memory");  // (one wave: its LDS accesses are in order)
    const unsigned int turn = (unsigned int)__popcll(movers & below), count = (unsigned int)__popcll(spares);
    int to = known ? source : -1;
    if (moves) to = turn < count ? s_spare[turn] : -1;
    const bool copied = moves && to >= 0;
    const unsigned int without = (unsigned int)__popcll(__ballot(known && to < 0));
    if (lane < beams) {
      a.out[(row0 + lane) * a.out_stride + full] = to;
      a.copied_from[row0 + lane] = copied ? source : -1;
      a.copies[row0 + lane] = make_int4(copied ? source : -1, to, (int)rest, 0);
    }
    const unsigned int taking = min((unsigned int)__popcll(movers), count);
    const unsigned int rank = (unsigned int)__popcll(spares & below);
    if (spare && rank >= taking) list[all + rank - taking] = id;
    if (lane == 0) {
      s_lacking = without;
      s_left = count - taking;
    }
  } else if (blockIdx.x == 0 && tid < beams && (rest == 0 || full >= a.width)) {
    // no block to be copied: whole blocks only, or a table that ends before the last one
    a.copied_from[row0 + tid] = -1;
    a.copies[row0 + tid] = make_int4(-1, -1, 0, 0);
  }
  __syncthreads();
  if (tid == 0)
    a.counts[group] = make_int2((int)(all + s_left), (int)(s_lacking + (blockIdx.x == 0 ? orphans : 0u)));
}

struct CopyArgs {
  OrderArgs o;
  unsigned long long block_bytes, row_bytes;  // of a plane's block, of a token
  unsigned int blocks, layers;
  bool list;  // this launch's last workgroup writes the free list
  unsigned char* layer[kMostLayers];
};

// The released blocks of all workgroups of order_tables, in order, below the list's first free entry.
__device__ __forceinline__ void list_released(const OrderArgs& a) {
  __shared__ unsigned int s_wave[2][kOrderWaves];
  const unsigned int tid = threadIdx.x;
  const unsigned int groups = a.requests * a.chunks;
  const unsigned int share = (groups + kOrderThreads - 1) / kOrderThreads;
  const unsigned int g0 = min(groups, tid * share), g1 = min(groups, g0 + share);
  const long long start = min(max(a.free_start[0], 0), (int)a.free_count);
  unsigned int own = 0, lacking = 0;
  for (unsigned int g = g0; g < g1; ++g) {
    const int2 c = a.counts[g];
    own += (unsigned int)c.x;
    lacking += (unsigned int)c.y;
  }
  unsigned int all, all_lacking;
  const unsigned int before = group_scan(own, s_wave[0], all);
  group_scan(lacking, s_wave[1], all_lacking);
  long long at = start - (long long)(all - before);
  for (unsigned int g = g0; own != 0 && g < g1; ++g) {
    const unsigned int count = (unsigned int)a.counts[g].x;
    const int* src = a.released + (unsigned long long)g * (a.beams * (kOrderThreads + 1));
    for (unsigned int i = 0; i < count; ++i, ++at)
      if (at >= 0) a.free_blocks[at] = src[i];
  }
  if (tid == 0) {
    a.free_next[0] = (int)max(start - (long long)all, 0ll);
    a.unlisted[0] = (int)max((long long)all - start, 0ll);
    a.lacking[0] = (int)all_lacking;
  }
}

// A workgroup copies the tokens of one row's last block, one plane of one layer.
template <typename U>
__global__ __launch_bounds__(kOrderThreads) void copy_tails(CopyArgs a) {
  if (a.list && blockIdx.x + 1 == gridDim.x) {
    list_released(a.o);
    return;
  }
  const unsigned int planes = 2 * a.layers;
  const unsigned int row = blockIdx.x / planes, plane = blockIdx.x - row * planes;
  const int4 copy = a.o.copies[row];
  if ((unsigned int)copy.x >= a.blocks || (unsigned int)copy.y >= a.blocks) return;
  unsigned char* base = a.layer[plane / 2] + (plane % 2) * (a.blocks * a.block_bytes);
  const U* src = reinterpret_cast<const U*>(base + (unsigned int)copy.x * a.block_bytes);
  U* dst = reinterpret_cast<U*>(base + (unsigned int)copy.y * a.block_bytes);
  const unsigned int units = (unsigned int)((unsigned int)copy.z * a.row_bytes / sizeof(U));
  constexpr unsigned int kAtOnce = 4;
  for (unsigned int i = threadIdx.x; i < units; i += kAtOnce * kOrderThreads) {
    U v[kAtOnce];
#pragma unroll
    for (unsigned int n = 0; n < kAtOnce; ++n) v[n] = src[min(i + n * kOrderThreads, units - 1)];
#pragma unroll
    for (unsigned int n = 0; n < kAtOnce; ++n)
      if (i + n * kOrderThreads < units) dst[i + n * kOrderThreads] = v[n];
  }
}

}  // namespace
}  // namespace unchainkv

using namespace unchainkv;

namespace {

// Chunks of a row, a wave's each: 4 KB. (Twice that for a wave: 64 requests of 8 beams, 131072 logits in bf16 37.8 us
// and 36.5, 256 of 4 beams, 50257 logits in fp16 44.1 and 32.7, 1024 of 8, 2500 in bf16 48.3 and 44.2; 2000 of 8, 5000
// 96.7 and 98.3.) A row of more segments than a wave's lanes hold is searched by several, as far as there are waves.
void shape(unsigned long long dtype, SelectArgs& a) {
  const unsigned int chunk = kWave * kLaneBytes / (dtype == 2 ? 4 : 2);
  a.chunks = (a.vocab + chunk - 1) / chunk;
  a.segments = (a.vocab + kSegment - 1) / kSegment;
  a.parts = 1;
  while (2 * a.parts * a.beams <= kPickThreads / kWave && a.segments > kMostItems * kWave * a.parts) a.parts *= 2;
  const unsigned int lanes = a.parts * kWave;
  a.group = (a.segments + kMostItems * lanes - 1) / (kMostItems * lanes);
  a.items = (a.segments + a.group - 1) / a.group;
}

bool select_ok(unsigned long long requests, unsigned long long beams, unsigned long long vocab,
               unsigned long long candidates) {
  return requests != 0 && beams != 0 && beams <= kMostBeams && vocab != 0 && vocab <= kMostVocab &&
         candidates != 0 && candidates <= kMostCandidates && candidates <= beams * vocab &&
         requests <= 1u << 20;
}

// Every row's maxima, then sums of as many chunks as it can have (those of f32): more for more rows or
// tokens, whatever their type.
unsigned long long maxima_bytes(unsigned long long rows, unsigned long long vocab) {
  return (4 * rows * ((vocab + kSegment - 1) / kSegment) + 15) / 16 * 16;
}
unsigned long long select_bytes(unsigned long long rows, unsigned long long vocab) {
  constexpr unsigned long long kLeast = kWave * kLaneLogits<Fp32>;
  return maxima_bytes(rows, vocab) + sizeof(float2) * rows * ((vocab + kLeast - 1) / kLeast);
}

bool is_whole(const SelectArgs& a) { return a.beams * a.chunks <= kWholeChunks; }

// As few registers as hold a row's items.
template <typename T>
void launch_pick(const SelectArgs& a, hipStream_t stream) {
  const dim3 grid(a.requests), threads(kPickThreads);
  const unsigned int held = (a.items + a.parts * kWave - 1) / (a.parts * kWave);
  if (is_whole(a))
    hipLaunchKernelGGL((beam_pick<T, 2, kOwnTokens, true>), grid, threads, 0, stream, a);
  else if (held <= 2)
    hipLaunchKernelGGL((beam_pick<T, 2, kOwnTokens, false>), grid, threads, 0, stream, a);
  else if (held <= 4)
    hipLaunchKernelGGL((beam_pick<T, 4, kOwnTokens, false>), grid, threads, 0, stream, a);
  else if (a.group == 1)
    hipLaunchKernelGGL((beam_pick<T, kMostItems, kOwnTokens, false>), grid, threads, 0, stream, a);
  else if (a.group == 2)
    hipLaunchKernelGGL((beam_pick<T, kMostItems, 2 * kOwnTokens, false>), grid, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((beam_pick<T, kMostItems, 8 * kOwnTokens, false>), grid, threads, 0, stream, a);
}
static_assert(kWholeChunks * kChunkSegments <= 2 * kWave, "a wave's lanes hold two of a whole row's segments each");

unsigned int chunks_of(unsigned long long width) {
  return (unsigned int)((width + kOrderThreads - 1) / kOrderThreads);
}
bool order_ok(unsigned long long requests, unsigned long long beams, unsigned long long width) {
  return requests != 0 && requests <= 65535 && beams != 0 && beams <= kMostBeams && width != 0 &&
         width <= 1u << 24;
}

}  // namespace

extern "C" unsigned long long kvq_splitzip_beam_select_workspace_bytes(unsigned long long requests,
                                                                       unsigned long long beams,
                                                                       unsigned long long vocab) {
  if (!select_ok(requests, beams, vocab, 1)) return 0;
  return select_bytes(requests * beams, vocab);
}

extern "C" long long kvq_splitzip_beam_select(
    unsigned long long logits_ptr, unsigned long long dtype, unsigned long long request_stride,
    unsigned long long beam_stride, unsigned long long scores_ptr, unsigned long long ended_ptr,
    unsigned long long requests, unsigned long long beams, unsigned long long vocab,
    unsigned long long candidates, unsigned long long end_token, unsigned long long out_scores_ptr,
    unsigned long long out_parents_ptr, unsigned long long out_tokens_ptr,
    unsigned long long workspace_ptr, unsigned long long workspace_bytes,
    unsigned long long stream_ptr) {
  if (!select_ok(requests, beams, vocab, candidates) || dtype > 2 || logits_ptr == 0 ||
      logits_ptr % (dtype == 2 ? 4 : 2) != 0 || scores_ptr == 0 || (ended_ptr != 0 && end_token >= vocab) ||
      out_scores_ptr == 0 || out_parents_ptr == 0 || out_tokens_ptr == 0 || workspace_ptr == 0 ||
      workspace_ptr % 16 != 0)
    return 0;
  const unsigned long long rows = requests * beams, need = select_bytes(rows, vocab);
  if (workspace_bytes < need) return 0;
  const unsigned long long picked = requests * candidates;
  const unsigned long long in[][2] = {
      {logits_ptr, ((requests - 1) * request_stride + (beams - 1) * beam_stride + vocab) * (dtype == 2 ? 4 : 2)},
      {scores_ptr, 4 * rows}, {ended_ptr, ended_ptr ? rows : 0}};
  const unsigned long long out[][2] = {{out_scores_ptr, 4 * picked}, {out_parents_ptr, 4 * picked},
                                       {out_tokens_ptr, 8 * picked}, {workspace_ptr, need}};
  for (const auto& o : out) {
    for (const auto& i : in)
      if (overlap(o[0], o[1], i[0], i[1])) return 0;
    for (const auto& p : out)
      if (&o != &p && overlap(o[0], o[1], p[0], p[1])) return 0;
  }
  SelectArgs a{};
  a.vocab = (unsigned int)vocab;
  a.beams = (unsigned int)beams;
  shape(dtype, a);
  a.logits = reinterpret_cast<const unsigned char*>(logits_ptr);
  a.scores = reinterpret_cast<const float*>(scores_ptr);
  a.ended = reinterpret_cast<const unsigned char*>(ended_ptr);
  a.maxima = reinterpret_cast<float*>(workspace_ptr);
  a.sums = reinterpret_cast<float2*>(workspace_ptr + maxima_bytes(rows, vocab));
  a.out_scores = reinterpret_cast<float*>(out_scores_ptr);
  a.out_parents = reinterpret_cast<int*>(out_parents_ptr);
  a.out_tokens = reinterpret_cast<long long*>(out_tokens_ptr);
  a.request_stride = request_stride;
  a.beam_stride = beam_stride;
  a.requests = (unsigned int)requests;
  a.candidates = (unsigned int)candidates;
  a.end_token = (unsigned int)end_token;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  constexpr unsigned int kChunks = kScanThreads / kWave;  // of a workgroup
  const dim3 grid((a.chunks + kChunks - 1) / kChunks, (unsigned int)std::min<unsigned long long>(rows, kGridRows),
                  (unsigned int)((rows + kGridRows - 1) / kGridRows));
  hipError_t st = hipSuccess;
  if (!is_whole(a)) {
    if (dtype == 0)
      hipLaunchKernelGGL(beam_scan<Bf16>, grid, dim3(kScanThreads), 0, stream, a);
    else if (dtype == 1)
      hipLaunchKernelGGL(beam_scan<Fp16>, grid, dim3(kScanThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(beam_scan<Fp32>, grid, dim3(kScanThreads), 0, stream, a);
    st = hipGetLastError();
    if (st != hipSuccess) return fail("beam_scan", st);
  }
  if (dtype == 0)
    launch_pick<Bf16>(a, stream);
  else if (dtype == 1)
    launch_pick<Fp16>(a, stream);
  else
    launch_pick<Fp32>(a, stream);
  st = hipGetLastError();
  if (st != hipSuccess) return fail("beam_pick", st);
  return (long long)picked;
}

extern "C" unsigned long long kvq_splitzip_reorder_beams_workspace_bytes(unsigned long long requests,
                                                                         unsigned long long beams,
                                                                         unsigned long long width) {
  if (!order_ok(requests, beams, width)) return 0;
  return 16 * requests * beams + requests * chunks_of(width) * (8 + 4 * beams * (kOrderThreads + 1));
}

extern "C" long long kvq_splitzip_reorder_beams_paged(
    const unsigned long long* layers, unsigned long long layer_count, unsigned long long blocks,
    unsigned long long block_tokens, unsigned long long row_bytes, unsigned long long tables_ptr,
    unsigned long long table_stride, unsigned long long table_width, unsigned long long out_ptr,
    unsigned long long out_stride, unsigned long long parents_ptr, unsigned long long context_tokens_ptr,
    unsigned long long requests, unsigned long long beams, unsigned long long free_blocks_ptr,
    unsigned long long free_count, unsigned long long free_start_ptr, unsigned long long copied_from_ptr,
    unsigned long long free_next_ptr, unsigned long long lacking_ptr, unsigned long long unlisted_ptr,
    unsigned long long workspace_ptr, unsigned long long workspace_bytes, unsigned long long stream_ptr) {
  constexpr unsigned long long kMost = 0x7FFFFFFFull;
  if (!order_ok(requests, beams, table_width) || (layer_count != 0 && layers == nullptr) ||
      layer_count > kMost || blocks == 0 || blocks > kMost || block_tokens == 0 || block_tokens > kMost ||
      row_bytes == 0 || row_bytes % 2 != 0 || row_bytes > kMost || blocks * block_tokens > kMost ||
      block_tokens * row_bytes > kMost || requests * beams * table_width > kMost ||
      tables_ptr == 0 || table_stride < table_width || out_ptr == 0 || out_stride < table_width ||
      parents_ptr == 0 || context_tokens_ptr == 0 || (free_blocks_ptr == 0 && free_count != 0) ||
      free_count > kMost || free_start_ptr == 0 || copied_from_ptr == 0 || free_next_ptr == 0 ||
      lacking_ptr == 0 || unlisted_ptr == 0 || workspace_ptr == 0 || workspace_ptr % 16 != 0)
    return 0;
  const unsigned long long need = kvq_splitzip_reorder_beams_workspace_bytes(requests, beams, table_width);
  if (workspace_bytes < need) return 0;
  const unsigned long long rows = requests * beams;
  const unsigned long long table_bytes = 4 * ((rows - 1) * table_stride + table_width);
  const unsigned long long out_bytes = 4 * ((rows - 1) * out_stride + table_width);
  const bool in_place = out_ptr == tables_ptr && out_stride == table_stride;
  const unsigned long long in[][2] = {{parents_ptr, 4 * rows}, {context_tokens_ptr, 4 * rows},
                                      {free_start_ptr, 4}, {tables_ptr, in_place ? 0 : table_bytes}};
  const unsigned long long out[][2] = {{out_ptr, out_bytes}, {free_blocks_ptr, 4 * free_count},
                                       {copied_from_ptr, 4 * rows}, {free_next_ptr, 4},
                                       {lacking_ptr, 4}, {unlisted_ptr, 4}, {workspace_ptr, need}};
  const unsigned long long layer_bytes = 2 * blocks * block_tokens * row_bytes;
  for (const auto& o : out) {
    for (const auto& i : in)
      if (overlap(o[0], o[1], i[0], i[1])) return 0;
    for (const auto& p : out)
      if (&o != &p && overlap(o[0], o[1], p[0], p[1])) return 0;
    for (unsigned long long l = 0; l < layer_count; ++l)
      if (overlap(o[0], o[1], layers[l], layer_bytes)) return 0;
  }
  bool wide = row_bytes % 16 == 0;
  for (unsigned long long l = 0; l < layer_count; ++l) {
    if (layers[l] == 0 || layers[l] % 2 != 0) return 0;
    wide = wide && layers[l] % 16 == 0;
    for (const auto& i : in)
      if (overlap(layers[l], layer_bytes, i[0], i[1])) return 0;
    if (overlap(layers[l], layer_bytes, tables_ptr, table_bytes)) return 0;
  }
  if (rows * 2 * std::min<unsigned long long>(layer_count, kMostLayers) > 0xFFFFFF) return 0;
  CopyArgs c{};
  OrderArgs& a = c.o;
  a.tables = reinterpret_cast<const int*>(tables_ptr);
  a.out = reinterpret_cast<int*>(out_ptr);
  a.parents = reinterpret_cast<const int*>(parents_ptr);
  a.contexts = reinterpret_cast<const int*>(context_tokens_ptr);
  a.copied_from = reinterpret_cast<int*>(copied_from_ptr);
  a.free_blocks = reinterpret_cast<int*>(free_blocks_ptr);
  a.free_start = reinterpret_cast<const int*>(free_start_ptr);
  a.free_next = reinterpret_cast<int*>(free_next_ptr);
  a.lacking = reinterpret_cast<int*>(lacking_ptr);
  a.unlisted = reinterpret_cast<int*>(unlisted_ptr);
  a.table_stride = table_stride;
  a.out_stride = out_stride;
  a.requests = (unsigned int)requests;
  a.beams = (unsigned int)beams;
  a.width = (unsigned int)table_width;
  a.chunks = chunks_of(table_width);
  a.block_tokens = (unsigned int)block_tokens;
  a.free_count = (unsigned int)free_count;
  a.by_block = make_divider(a.block_tokens);
  a.copies = reinterpret_cast<int4*>(workspace_ptr);
  a.counts = reinterpret_cast<int2*>(workspace_ptr + 16 * rows);
  a.released = reinterpret_cast<int*>(a.counts + requests * a.chunks);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  hipLaunchKernelGGL(order_tables, dim3(a.chunks, a.requests), dim3(kOrderThreads),
                     beams * kOrderThreads * sizeof(int), stream, a);
  hipError_t st = hipGetLastError();
  if (st != hipSuccess) return fail("order_tables", st);
  c.block_bytes = block_tokens * row_bytes;
  c.row_bytes = row_bytes;
  c.blocks = (unsigned int)blocks;
  for (unsigned long long l = 0;;) {
    c.layers = (unsigned int)std::min<unsigned long long>(layer_count - l, kMostLayers);
    for (unsigned int i = 0; i < c.layers; ++i) c.layer[i] = reinterpret_cast<unsigned char*>(layers[l + i]);
    l += c.layers;
    c.list = l == layer_count;
    const unsigned long long groups = rows * 2 * c.layers + (c.list ? 1 : 0);
    if (wide)
      hipLaunchKernelGGL(copy_tails<u32x4>, dim3((unsigned int)groups), dim3(kOrderThreads), 0, stream, c);
    else
      hipLaunchKernelGGL(copy_tails<uint16_t>, dim3((unsigned int)groups), dim3(kOrderThreads), 0, stream, c);
    st = hipGetLastError();
    if (st != hipSuccess) return fail("copy_tails", st);
    if (c.list) break;
  }
  return (long long)rows;
}
