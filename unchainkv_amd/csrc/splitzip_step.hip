// A serving step's tables and the cache write, gfx950: block tables, row ranges, slots and
// positions from the requests' lengths, and the new tokens' K and V rows into a paged layer.
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
