// Block tables and slot maps from request lengths, on the GPU.
//
// Sequence b holds ceil(ctx_b / bs) blocks and takes new_b more tokens: it grows to
// ceil((ctx_b + new_b) / bs) blocks, taken off the head of the free list in row order, as the
// block manager on the host pops them (engine/kv_cache.py:40-74).  Token i of it lies at position
// ctx_b + i, slot table[b][position / bs] * bs + position % bs.
//
// Where lengths go back (rejected drafts) ceil(ctx_b / bs) is less than what the sequence was given, so the caller
// keeps the count of blocks, held_b: the sequence grows by what ceil((ctx_b + new_b) / bs) exceeds it, entries below
// held_b are used again, and held_b becomes the larger of the two.
//
// One launch: every CTA scans the batch's lengths by itself (a few KB, out of L2 after the first
// CTA), then maps its share of the tokens; a token finds its sequence by bisecting the scanned
// starts in shared memory.  A token at the first position of a new block writes that block into
// the table.  No CTA reads what another writes: entries below held_b are only read, the ones above only written,
// and held_b is updated when all have read it, by the one CTA or by a launch of its own.  Bound by latency: a scan, a
// bisection and two dependent loads (4.4 us for 64 sequences of one token, 5.7 for 200 of 500 to 1000).
//
// A batch whose starts do not fit into shared memory is cut into pieces of 4,096 sequences, a block each: sums of
// the pieces, then starts and sums of the blocks needed, then offsets into the free list, then the tokens, a
// launch each.
#include <climits>

#include "common.cuh"
#include "host.h"

namespace mvb {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxShared = 8192;          // sequences whose starts and offsets one block holds in shared memory
constexpr int kMaxBatch = 1 << 20;
constexpr int kPer = 8;                   // sequences of a thread in the launches over pieces
constexpr int kPiece = kPer * kThreads;

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
  int32_t* held;  // blocks that a sequence holds, updated; nullptr: ceil(ctx / bs)
  const int32_t* free_blocks;
  const int32_t* head_in;
  int64_t num_free;
  int64_t tokens;
  int batch;
  int bs;
  unsigned* err;
};

__device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

__device__ __forceinline__ int64_t held_blocks(const SlotArgs& a, int64_t b, int64_t ctx) {
  return a.held != nullptr ? a.held[b] : ceil_div(ctx, a.bs);
}
// Blocks that sequence b lacks for its new tokens, its lengths being good.
__device__ __forceinline__ int64_t blocks_lacking(const SlotArgs& a, int64_t b, int64_t ctx, int64_t add) {
  return max(ceil_div(ctx + add, a.bs) - held_blocks(a, b, ctx), int64_t(0));
}
// Lengths of a sequence that can be: none negative, and the blocks it holds enough for what it has, and in its row.
__device__ __forceinline__ bool lengths_good(const SlotArgs& a, int64_t b, int64_t ctx, int64_t add) {
  if (ctx < 0 || add < 0) return false;
  if (a.held == nullptr) return true;
  const int64_t held = a.held[b];
  return held >= ceil_div(ctx, a.bs) && held <= a.max_blocks;
}
__device__ __forceinline__ void update_held(const SlotArgs& a, int64_t b, bool granted) {
  if (granted) a.held[b] = static_cast<int32_t>(max(int64_t(a.held[b]), ceil_div(int64_t(a.ctx[b]) + a.add[b], a.bs)));
}

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

// Slots and positions of this block's tokens.
__device__ __forceinline__ void map_tokens(const SlotArgs& a, int64_t head, const int32_t* start, const int32_t* first) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  const int32_t last = start[a.batch];
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; t < a.tokens; t += step) {
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
        const int64_t bi = pos / a.bs, held = held_blocks(a, lo, ctx);
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

__global__ void __launch_bounds__(kThreads) assign_slots_kernel(const SlotArgs a) {
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
  __syncthreads();  // the scans hold others, but there are none for an empty batch
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + tid;
    int64_t add = 0, need = 0, total, blocks;
    bool ok = false;
    if (b < a.batch) {
      const int64_t ctx = a.ctx[b];
      add = a.add[b];
      ok = lengths_good(a, b, ctx, add);
      if (!ok && blockIdx.x == 0) report(a.err, kDevBadPosition);
      add = max(add, int64_t(0));
      ok = ok && ctx + add <= a.max_blocks * a.bs;
      need = ok ? blocks_lacking(a, b, ctx, add) : 0;
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
        need = blocks_lacking(a, b, a.ctx[b], a.add[b]);
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
        const int64_t need = blocks_lacking(a, b, a.ctx[b], a.add[b]);
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
  map_tokens(a, head, start, first);
  if (a.held != nullptr && gridDim.x == 1) {
    __syncthreads();  // all have read
    for (int b = tid; b < a.batch; b += kThreads) update_held(a, b, first[b] >= 0);
  }
}

// The held blocks of a call of several CTAs.
__global__ void __launch_bounds__(kThreads) slot_held_kernel(const SlotArgs a) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (b < a.batch) update_held(a, b, a.granted[b] != 0);
}

// ---- batches of more than kMaxShared sequences
struct BigArgs {
  int64_t* piece_add;   // [pieces] tokens of a piece
  int64_t* piece_need;  // [pieces] blocks it needs
  int32_t* first;       // [batch] blocks needed (-1: refused), then the offset of the first one
};

// Sum over the block, in every thread.
__device__ __forceinline__ int64_t block_sum(int64_t x, int64_t (*warps)[2]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5][0] = x;
  __syncthreads();
  int64_t all = 0;
  for (int w = 0; w < kThreads / 32; ++w) all += warps[w][0];
  return all;
}
// Sum of v[0 .. n), in every thread.
__device__ __forceinline__ int64_t sum_before(const int64_t* v, int n, int64_t (*warps)[2]) {
  int64_t x = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) x += v[i];
  return block_sum(x, warps);
}

__global__ void __launch_bounds__(kThreads) slot_sums_kernel(const SlotArgs a, const BigArgs g) {
  __shared__ int64_t warps[kThreads / 32][2];
  pdl_wait();
  const int64_t b0 = static_cast<int64_t>(blockIdx.x) * kPiece + threadIdx.x * kPer;
  int64_t add = 0;
  for (int i = 0; i < kPer; ++i)
    if (b0 + i < a.batch) add += max(a.add[b0 + i], 0);
  add = block_sum(add, warps);
  if (threadIdx.x == 0) g.piece_add[blockIdx.x] = add;
}

__global__ void __launch_bounds__(kThreads) slot_starts_kernel(const SlotArgs a, const BigArgs g) {
  __shared__ int64_t warps[kThreads / 32][2];
  const int64_t b0 = static_cast<int64_t>(blockIdx.x) * kPiece + threadIdx.x * kPer;
  int64_t own = 0, zero = 0;
  for (int i = 0; i < kPer; ++i)
    if (b0 + i < a.batch) own += max(a.add[b0 + i], 0);
  int64_t at = own;
  const int64_t before = sum_before(g.piece_add, blockIdx.x, warps);
  block_scan2(at, zero, warps);
  at += before - own;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.seq_start[0] = 0;
  int64_t needs = 0;
  for (int i = 0; i < kPer; ++i) {
    const int64_t b = b0 + i;
    if (b >= a.batch) break;
    const int64_t ctx = a.ctx[b], add = a.add[b];
    bool ok = lengths_good(a, b, ctx, add);
    if (!ok) report(a.err, kDevBadPosition);
    at += max(add, int64_t(0));
    a.seq_start[b + 1] = static_cast<int32_t>(min(at, int64_t(INT_MAX)));
    ok = ok && ctx + add <= a.max_blocks * a.bs && at <= a.tokens;
    const int64_t need = ok ? blocks_lacking(a, b, ctx, add) : 0;
    needs += need;
    g.first[b] = ok ? static_cast<int32_t>(need) : -1;
  }
  needs = block_sum(needs, warps);
  if (threadIdx.x == 0) g.piece_need[blockIdx.x] = needs;
}

__global__ void __launch_bounds__(kThreads) slot_offsets_kernel(const SlotArgs a, const BigArgs g) {
  __shared__ int64_t warps[kThreads / 32][2];
  const int64_t head = a.head_in != nullptr ? max(static_cast<int64_t>(*a.head_in), int64_t(0)) : 0;
  const int64_t avail = max(a.num_free - head, int64_t(0));
  const int64_t all = sum_before(g.piece_need, gridDim.x, warps);
  if (all > avail) {  // short: in row order, 32 sequences at a time, one by one where they do not all fit
    if (blockIdx.x != 0 || threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    int64_t taken = 0;
    for (int64_t b = lane; b - lane < a.batch; b += 32) {
      const int need = b < a.batch ? g.first[b] : -1;
      int64_t sum = max(need, 0);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const int64_t last = __shfl_sync(0xffffffffu, sum, 31);
      int64_t at = need < 0 ? -1 : taken + sum - need;
      if (taken + last <= avail) {
        taken += last;
      } else {
        for (int j = 0; j < 32; ++j) {
          const int want = __shfl_sync(0xffffffffu, need, j);
          const bool fits = want >= 0 && taken + want <= avail;
          if (j == lane) at = fits ? taken : -1;
          if (fits) taken += want;
        }
      }
      if (b < a.batch) {
        g.first[b] = static_cast<int32_t>(at);
        a.granted[b] = at >= 0 ? 1 : 0;
      }
    }
    if (lane == 0) *a.head_out = static_cast<int32_t>(head + taken);
    return;
  }
  const int64_t b0 = static_cast<int64_t>(blockIdx.x) * kPiece + threadIdx.x * kPer;
  int32_t need[kPer];
  int64_t own = 0, zero = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    need[i] = b0 + i < a.batch ? g.first[b0 + i] : -1;
    own += max(need[i], 0);
  }
  int64_t at = own;
  const int64_t before = sum_before(g.piece_need, blockIdx.x, warps);
  block_scan2(at, zero, warps);
  at += before - own;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (b0 + i >= a.batch) break;
    g.first[b0 + i] = need[i] < 0 ? -1 : static_cast<int32_t>(at);
    a.granted[b0 + i] = need[i] < 0 ? 0 : 1;
    at += max(need[i], 0);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.head_out = static_cast<int32_t>(head + all);
}

__global__ void __launch_bounds__(kThreads) slot_tokens_kernel(const SlotArgs a, const BigArgs g) {
  const int64_t head = a.head_in != nullptr ? max(static_cast<int64_t>(*a.head_in), int64_t(0)) : 0;
  map_tokens(a, head, a.seq_start, g.first);
}

int64_t slot_pieces(int64_t batch) { return (batch + kPiece - 1) / kPiece; }

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int64_t mvb_assign_slots_workspace_bytes(int64_t batch) {
  return batch <= kMaxShared ? 0 : slot_pieces(batch) * 16 + batch * 4;
}

extern "C" int mvb_assign_slots(int64_t* slots, int32_t* positions, int32_t* seq_start, int32_t* granted,
                                int32_t* free_head_out, int32_t* block_tables, int64_t table_stride,
                                int64_t max_blocks, const int32_t* ctx_lens, const int32_t* new_lens,
                                const int32_t* free_blocks, int64_t num_free, const int32_t* free_head,
                                int64_t batch, int64_t block_size, int64_t num_tokens, void* workspace,
                                int64_t workspace_bytes, mvb_stream_t stream) {
  return mvb_assign_slots_ex(slots, positions, seq_start, granted, free_head_out, block_tables, table_stride, max_blocks,
                             ctx_lens, new_lens, nullptr, free_blocks, num_free, free_head, batch, block_size, num_tokens,
                             workspace, workspace_bytes, stream);
}

extern "C" int mvb_assign_slots_ex(int64_t* slots, int32_t* positions, int32_t* seq_start, int32_t* granted,
                                   int32_t* free_head_out, int32_t* block_tables, int64_t table_stride,
                                   int64_t max_blocks, const int32_t* ctx_lens, const int32_t* new_lens,
                                   int32_t* held_blocks, const int32_t* free_blocks, int64_t num_free,
                                   const int32_t* free_head, int64_t batch, int64_t block_size, int64_t num_tokens,
                                   void* workspace, int64_t workspace_bytes, mvb_stream_t stream) {
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
  MVB_REQUIRE(held_blocks == nullptr || batch == 0 || (held_blocks != ctx_lens && held_blocks != new_lens),
              "mvb_assign_slots: held_blocks may not be a length");
  const int sms = current_sm_count();
  MVB_REQUIRE(sms > 0, "mvb_assign_slots: no device");
  SlotArgs a = {slots,    positions, seq_start,   granted,   free_head_out, block_tables, table_stride,
                max_blocks, ctx_lens,  new_lens,    held_blocks, free_blocks,   free_head,    num_free,
                num_tokens, static_cast<int>(batch), static_cast<int>(block_size), device_status_ptr()};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t grid = (num_tokens + 2 * kThreads - 1) / (2 * kThreads);
  grid = grid < 1 ? 1 : grid > sms ? sms : grid;
  const dim3 blocks(static_cast<unsigned>(grid)), threads(kThreads);
  const dim3 per_sequence(static_cast<unsigned>((batch + kThreads - 1) / kThreads));
  if (batch <= kMaxShared) {
    const size_t smem = (2 * batch + 1) * sizeof(int32_t);
    // past 48 KB together with the kernel's static arrays a launch has to be allowed for: once, for the largest batch
    static std::atomic<uint64_t> done{0};
    if (smem > 40 * 1024)
      MVB_TRY(set_smem_once(done, assign_slots_kernel, (2 * kMaxShared + 1) * sizeof(int32_t), "assign_slots"));
    MVB_TRY(launch("assign_slots", assign_slots_kernel, blocks, threads, smem, st, a));
    if (held_blocks == nullptr || grid == 1) return MVB_OK;
    slot_held_kernel<<<per_sequence, threads, 0, st>>>(a);  // a plain launch: the one before has ended
    return cuda_status(cudaGetLastError(), "assign_slots");
  }
  MVB_REQUIRE(workspace && aligned(workspace, 8) && workspace_bytes >= mvb_assign_slots_workspace_bytes(batch),
              "mvb_assign_slots: a workspace of %lld bytes, 8-byte aligned (got %lld)",
              (long long)mvb_assign_slots_workspace_bytes(batch), (long long)workspace_bytes);
  const int64_t n = slot_pieces(batch);
  BigArgs g;
  g.piece_add = static_cast<int64_t*>(workspace);
  g.piece_need = g.piece_add + n;
  g.first = reinterpret_cast<int32_t*>(g.piece_need + n);
  const dim3 pieces(static_cast<unsigned>(n));
  // the launches after the first one are plain: each reads what the one before it wrote
  MVB_TRY(launch("assign_slots", slot_sums_kernel, pieces, threads, 0, st, a, g));
  slot_starts_kernel<<<pieces, threads, 0, st>>>(a, g);
  slot_offsets_kernel<<<pieces, threads, 0, st>>>(a, g);
  slot_tokens_kernel<<<blocks, threads, 0, st>>>(a, g);
  if (held_blocks != nullptr) slot_held_kernel<<<per_sequence, threads, 0, st>>>(a);
  return cuda_status(cudaGetLastError(), "assign_slots");
}
