// Block tables and slot maps from request lengths, on the GPU.
//
// Sequence b holds ceil(ctx_b / bs) blocks and takes new_b more tokens: it grows to
// ceil((ctx_b + new_b) / bs) blocks, taken off the head of the free list in row order, as the
// block manager on the host pops them (engine/kv_cache.py:40-74).  Token i of it lies at position
// ctx_b + i, slot table[b][position / bs] * bs + position % bs.
//
// One launch: every CTA scans the batch's lengths by itself (a few KB, out of L2 after the first
// CTA), then maps its share of the tokens; a token finds its sequence by bisecting the scanned
// starts in shared memory.  A token at the first position of a new block writes that block into
// the table.  No CTA reads what another writes: entries below ceil(ctx_b / bs) are only read, the
// ones above only written.  Bound by latency: a scan, a bisection and two dependent loads.
#include <climits>

#include "common.cuh"
#include "host.h"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxBatch = 8192;  // starts and block offsets of the whole batch in shared memory

struct SlotArgs {
  int64_t* slots;
  int32_t* positions;
  int32_t* seq_start;
  int32_t* granted;
  int32_t* head_out;
  int32_t* tables;
  int64_t table_stride;
  int64_t max_blocks;
  const int32_t* ctx;
  const int32_t* add;
  const int32_t* free_blocks;
  const int32_t* head_in;
  int64_t num_free;
  int64_t tokens;
  int batch;
  int bs;
  unsigned* err;
};

__device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Inclusive scan over the block of two 64-bit values per thread.
__device__ __forceinline__ void block_scan2(int64_t& x, int64_t& y, int64_t (*warps)[2]) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t px = __shfl_up_sync(0xffffffffu, x, o), py = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += px;
      y += py;
    }
  }
  __syncthreads();
  if (lane == 31) {
    warps[wid][0] = x;
    warps[wid][1] = y;
  }
  __syncthreads();
  for (int w = 0; w < wid; ++w) {
    x += warps[w][0];
    y += warps[w][1];
  }
}

__global__ void __launch_bounds__(kThreads) assign_slots_kernel(SlotArgs a) {
  extern __shared__ int32_t sm[];
  __shared__ int64_t warps[kThreads / 32][2];
  __shared__ int64_t carry[2];
  int32_t* start = sm;                // [batch + 1]
  int32_t* first = sm + a.batch + 1;  // [batch] offset of the sequence's first new block; -1: not granted
  // dependents start at this kernel's end only: they read its outputs as step metadata before they wait
  pdl_wait();
  const int tid = threadIdx.x;
  const int64_t head = a.head_in != nullptr ? max(static_cast<int64_t>(*a.head_in), int64_t(0)) : 0;
  const int64_t avail = max(a.num_free - head, int64_t(0));
  if (tid == 0) {
    carry[0] = carry[1] = 0;
    start[0] = 0;
  }
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + tid;
    int64_t add = 0, need = 0, total, blocks;
    bool ok = false;
    if (b < a.batch) {
      const int64_t ctx = a.ctx[b];
      add = a.add[b];
      ok = ctx >= 0 && add >= 0;
      if (!ok && blockIdx.x == 0) report(a.err, kDevBadPosition);
      add = max(add, int64_t(0));
      ok = ok && ctx + add <= a.max_blocks * a.bs;
      need = ok ? ceil_div(ctx + add, a.bs) - ceil_div(ctx, a.bs) : 0;
    }
    total = add;
    block_scan2(total, need, warps);  // need becomes inclusive; what the sequence asks for is in `blocks`
    const int64_t t0 = carry[0], n0 = carry[1];
    blocks = need;
    total += t0;
    if (b < a.batch) {
      start[b + 1] = static_cast<int32_t>(min(total, int64_t(INT_MAX)));
      ok = ok && total <= a.tokens;
      first[b] = ok ? 0 : -1;
    }
    __syncthreads();
    if (tid == kThreads - 1) {
      carry[0] = total;
      carry[1] = n0 + blocks;
    }
    __syncthreads();
  }
  // Offsets into the free list.  A sequence that is refused for its length or its tokens takes no
  // blocks, and where the pool runs short the ones behind a refused sequence may still fit: the
  // common case (everything fits) is a scan, the short one is walked in row order.
  const bool enough = carry[1] <= avail;
  __syncthreads();
  if (enough) {
    if (tid == 0) carry[1] = 0;
    __syncthreads();
    for (int base = 0; base < a.batch; base += kThreads) {
      const int b = base + tid;
      int64_t need = 0, zero = 0;
      if (b < a.batch && first[b] >= 0) {
        const int64_t ctx = a.ctx[b];
        need = ceil_div(ctx + a.add[b], a.bs) - ceil_div(ctx, a.bs);
      }
      const int64_t own = need;
      block_scan2(zero, need, warps);
      const int64_t n0 = carry[1];
      if (b < a.batch && first[b] >= 0) first[b] = static_cast<int32_t>(n0 + need - own);
      __syncthreads();
      if (tid == kThreads - 1) carry[1] = n0 + need;
      __syncthreads();
    }
  } else {
    if (tid == 0) {
      int64_t taken = 0;
      for (int b = 0; b < a.batch; ++b) {
        if (first[b] < 0) continue;
        const int64_t ctx = a.ctx[b];
        const int64_t need = ceil_div(ctx + a.add[b], a.bs) - ceil_div(ctx, a.bs);
        if (taken + need <= avail) {
          first[b] = static_cast<int32_t>(taken);
          taken += need;
        } else {
          first[b] = -1;
        }
      }
      carry[1] = taken;
    }
    __syncthreads();
  }

  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.batch; b += kThreads) a.seq_start[b] = start[b];
    for (int b = tid; b < a.batch; b += kThreads) a.granted[b] = first[b] >= 0 ? 1 : 0;
    if (tid == 0) *a.head_out = static_cast<int32_t>(head + carry[1]);
  }

  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  const int32_t last = start[a.batch];
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + tid; t < a.tokens; t += step) {
    int64_t slot = -1;
    int64_t pos = 0;
    if (t < last) {
      int lo = 0, hi = a.batch;  // start[lo] <= t < start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
      }
      const int64_t ctx = max(a.ctx[lo], 0);
      pos = ctx + (t - start[lo]);
      if (first[lo] >= 0) {
        const int64_t bi = pos / a.bs, held = ceil_div(ctx, a.bs);
        int32_t* row = a.tables + lo * a.table_stride;
        int32_t id;
        if (bi < held) {
          id = row[bi];
        } else {
          id = a.free_blocks[head + first[lo] + (bi - held)];
          if (pos == bi * a.bs) row[bi] = id;
        }
        slot = id < 0 ? -1 : static_cast<int64_t>(id) * a.bs + (pos - bi * a.bs);
      }
    }
    a.slots[t] = slot;
    a.positions[t] = static_cast<int32_t>(min(pos, int64_t(INT_MAX)));
  }
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_assign_slots(int64_t* slots, int32_t* positions, int32_t* seq_start, int32_t* granted,
                                int32_t* free_head_out, int32_t* block_tables, int64_t table_stride,
                                int64_t max_blocks, const int32_t* ctx_lens, const int32_t* new_lens,
                                const int32_t* free_blocks, int64_t num_free, const int32_t* free_head,
                                int64_t batch, int64_t block_size, int64_t num_tokens, mvb_stream_t stream) {
  MVB_REQUIRE(seq_start && free_head_out, "mvb_assign_slots: null pointer");
  MVB_REQUIRE(batch >= 0 && batch <= kMaxBatch, "mvb_assign_slots: batch %lld (at most %d)", (long long)batch,
              kMaxBatch);
  MVB_REQUIRE(batch == 0 || (granted && ctx_lens && new_lens), "mvb_assign_slots: null pointer");
  MVB_REQUIRE(max_blocks >= 0 && (batch == 0 || max_blocks == 0 || block_tables), "mvb_assign_slots: block_tables");
  MVB_REQUIRE(batch <= 1 || table_stride >= max_blocks, "mvb_assign_slots: table_stride %lld < max_blocks %lld",
              (long long)table_stride, (long long)max_blocks);
  MVB_REQUIRE(num_free >= 0 && num_free <= INT_MAX && (num_free == 0 || free_blocks), "mvb_assign_slots: free list");
  MVB_REQUIRE(block_size > 0 && block_size <= (1 << 20), "mvb_assign_slots: block_size %lld", (long long)block_size);
  MVB_REQUIRE(max_blocks <= INT_MAX / block_size, "mvb_assign_slots: %lld blocks a sequence", (long long)max_blocks);
  MVB_REQUIRE(num_tokens >= 0 && num_tokens <= INT_MAX && (num_tokens == 0 || (slots && positions)),
              "mvb_assign_slots: num_tokens %lld", (long long)num_tokens);
  MVB_REQUIRE(free_head_out != free_head, "mvb_assign_slots: free_head_out may not be free_head");
  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "mvb_assign_slots: no device");
  SlotArgs a = {slots,    positions, seq_start,   granted,   free_head_out, block_tables, table_stride,
                max_blocks, ctx_lens,  new_lens,    free_blocks, free_head,  num_free,     num_tokens,
                static_cast<int>(batch), static_cast<int>(block_size), device_status_ptr()};
  const size_t smem = (2 * batch + 1) * sizeof(int32_t);
  if (smem > 48 * 1024) MVB_TRY(set_smem(assign_slots_kernel, smem, "assign_slots"));
  int64_t grid = (num_tokens + 2 * kThreads - 1) / (2 * kThreads);
  grid = grid < 1 ? 1 : grid > sms ? sms : grid;
  return launch("assign_slots", assign_slots_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem,
                reinterpret_cast<cudaStream_t>(stream), a);
}
