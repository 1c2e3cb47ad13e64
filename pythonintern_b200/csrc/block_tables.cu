// Block tables and slot maps built on the GPU from request lengths.
//
// The host bookkeeping these replace for a step that stays on the device:
// engine/model/kv_cache.py:172-227 (FIFO free list, one table per sequence) and the
// per-token slot walk of engine/model/attention.py:166-184 (slot = table[p / bs] * bs + p % bs).
//
// State: tables [n_seqs, table_stride] (-1 where no block is held), lens [n_seqs] tokens per
// sequence (a sequence holds ceil(len / bs) blocks), a ring of free block ids and
// free_state = {head, count, 0, 0}.  extend() takes blocks from the ring's head in sequence
// order and writes the maps of the new tokens; truncate() gives the blocks behind the kept
// tokens back to the ring's tail, in sequence and then table order, as the host list would.
//
// Every CTA scans all n_seqs lengths by itself (two prefix sums kept in shared memory), which
// costs less than a second launch or a grid barrier would; the items (groups of tokens, or
// blocks to give back) are then spread over the grid, each finding its sequence by bisection
// of the prefix.  Nothing that a CTA reads is written before every CTA has read it: the last
// CTA to finish (a ticket in free_state[2], put back to 0) updates lens and the ring's state.
// A call that cannot be served whole (a bad length, a row past the table, too few free blocks,
// more tokens than the maps hold) raises its bit in *status and changes nothing.
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxSeqs = 16384;  // two int32 prefix sums of this length fill 128 KB of shared memory
constexpr int kPerThread = 4;    // tokens (or blocks) per item: 16- and 32-byte stores of the maps

struct TablesParams {
  int32_t* tables;
  int n_seqs, stride, bs;
  int32_t* lens;
  const int32_t* arg;  // extend: new tokens; truncate: tokens to keep
  int32_t* ring;
  int num_blocks;
  int32_t* state;
  int64_t max_tokens;
  int32_t* seq_start;
  int64_t* positions;
  int32_t* table_index;
  int64_t* slots;
  int32_t* ctx_lens;
  int64_t* last_rows;
  int32_t* status;
};

struct Span {
  int items;   // extend: new tokens; truncate: blocks given back
  int blocks;  // extend: blocks taken
  bool bad;
};

template <bool EXTEND>
__device__ __forceinline__ Span span_of(const TablesParams& p, int s) {
  const int len = p.lens[s], a = p.arg[s];
  Span r{0, 0, len < 0 || a < 0};
  if (r.bad) return r;
  const int64_t held = ((int64_t)len + p.bs - 1) / p.bs;
  if (EXTEND) {
    const int64_t after = (int64_t)len + a;
    const int64_t want = (after + p.bs - 1) / p.bs;
    r.bad = want > p.stride || after > 0x7fffffff;
    r.items = a;
    r.blocks = r.bad ? 0 : (int)(want - held);
  } else {
    r.bad = held > p.stride;
    const int64_t kept = ((int64_t)min(a, len) + p.bs - 1) / p.bs;
    r.items = r.bad ? 0 : (int)(held - kept);
  }
  return r;
}

// Largest s with prefix[s] <= x, for prefix[0] = 0 and x below the total: sequences without
// items share their successor's prefix and are passed over.
__device__ __forceinline__ int find_seq(const int* prefix, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Ring slot `x` places behind `head`, both below num_blocks (x may equal it).
__device__ __forceinline__ int64_t ring_slot(const TablesParams& p, int64_t head, int64_t x) {
  const int64_t at = head + x;
  return at >= p.num_blocks ? at - p.num_blocks : at;
}

template <bool EXTEND>
__global__ void __launch_bounds__(kThreads) block_tables_kernel(TablesParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int sm[];
  int* item0 = sm;                // [n_seqs] items before sequence s
  int* block0 = sm + p.n_seqs;    // [n_seqs] blocks taken before sequence s (extend)
  __shared__ int64_t w_items[kThreads / 32], w_blocks[kThreads / 32];
  __shared__ int last_cta;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // Prefix sums over the sequences: each thread sums a run of consecutive ones.
  const int per = (p.n_seqs + kThreads - 1) / kThreads;
  const int s0 = min(p.n_seqs, tid * per), s1 = min(p.n_seqs, s0 + per);
  int64_t items = 0, blocks = 0;
  bool bad = false;
  for (int s = s0; s < s1; ++s) {
    const Span x = span_of<EXTEND>(p, s);
    bad |= x.bad;
    items += x.items;
    blocks += x.blocks;
  }
  int64_t inc_i = items, inc_b = blocks;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, inc_i, o), b = __shfl_up_sync(0xffffffffu, inc_b, o);
    if (lane >= o) {
      inc_i += a;
      inc_b += b;
    }
  }
  if (lane == 31) {
    w_items[warp] = inc_i;
    w_blocks[warp] = inc_b;
  }
  bad = __syncthreads_or(bad);
  int64_t base_i = inc_i - items, base_b = inc_b - blocks, total = 0, taken = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) {
      base_i += w_items[w];
      base_b += w_blocks[w];
    }
    total += w_items[w];
    taken += w_blocks[w];
  }
  const bool alloc = p.ring != nullptr;
  int head = 0, count = 0, error = bad ? B2_DEV_RANGE : 0;
  if (alloc) {
    head = p.state[0];
    count = p.state[1];
    if (head < 0 || head >= p.num_blocks || count < 0 || count > p.num_blocks) error = B2_DEV_RANGE;
  }
  if (EXTEND) {
    if (total > p.max_tokens) error = B2_DEV_RANGE;
    if (!error && alloc && taken > count) error = B2_DEV_NO_BLOCKS;
  } else if (!error && count + total > p.num_blocks) {
    error = B2_DEV_RANGE;  // more blocks would come back than the pool has
  }
  if (error) {  // every CTA finds the same: nothing is changed
    if (blockIdx.x == 0 && tid == 0) raise_status(p.status, error);
    return;
  }
  for (int s = s0; s < s1; ++s) {
    const Span x = span_of<EXTEND>(p, s);
    item0[s] = (int)base_i;
    if (EXTEND) {
      block0[s] = (int)base_b;
      if (blockIdx.x == 0) {
        p.seq_start[s] = (int)base_i;
        p.last_rows[s] = x.items > 0 ? base_i + x.items - 1 : -1;
      }
    }
    base_i += x.items;
    base_b += x.blocks;
  }
  if (EXTEND && blockIdx.x == 0 && tid == 0) p.seq_start[p.n_seqs] = (int)total;
  __syncthreads();

  const int64_t step = (int64_t)gridDim.x * kThreads * kPerThread;
  for (int64_t i0 = ((int64_t)blockIdx.x * kThreads + tid) * kPerThread; i0 < total; i0 += step) {
    int s = find_seq(item0, p.n_seqs, (int)i0);
    int s_end = s + 1 < p.n_seqs ? item0[s + 1] : (int)total;
    const int n = (int)min((int64_t)kPerThread, total - i0);
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
      if (e >= n) break;
      const int i = (int)i0 + e;
      while (i >= s_end) {
        ++s;
        s_end = s + 1 < p.n_seqs ? item0[s + 1] : (int)total;
      }
      const int len = p.lens[s];
      const int held = (int)(((int64_t)len + p.bs - 1) / p.bs);
      if (EXTEND) {
        const int pos = len + (i - item0[s]);
        const int j = pos / p.bs, off = pos - j * p.bs;
        int blk;
        if (alloc && j >= held) {
          blk = p.ring[ring_slot(p, head, (int64_t)block0[s] + (j - held))];
          if (off == 0) p.tables[(int64_t)s * p.stride + j] = blk;  // a taken block's first token is new
        } else {
          blk = p.tables[(int64_t)s * p.stride + j];
        }
        const bool ok = blk >= 0 && blk < p.num_blocks;
        if (!ok) raise_status(p.status, B2_DEV_RANGE);
        p.positions[i] = pos;
        p.table_index[i] = s;
        p.slots[i] = ok ? (int64_t)blk * p.bs + off : -1;
        p.ctx_lens[i] = pos + 1;
      } else {
        const int kept = (int)(((int64_t)min(p.arg[s], len) + p.bs - 1) / p.bs);
        int32_t* entry = p.tables + (int64_t)s * p.stride + kept + (i - item0[s]);
        p.ring[ring_slot(p, head, (int64_t)count + i)] = *entry;
        *entry = -1;
      }
    }
  }
  if (!alloc) return;  // maps alone: no state to move on

  __threadfence();
  __syncthreads();
  if (tid == 0) last_cta = atomicAdd(&p.state[2], 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last_cta) return;
  for (int s = tid; s < p.n_seqs; s += kThreads) {
    const int len = p.lens[s], a = p.arg[s];
    p.lens[s] = EXTEND ? len + a : min(len, a);
  }
  if (tid == 0) {
    if (EXTEND) {
      p.state[0] = (int)ring_slot(p, head, taken);
      p.state[1] = count - (int)taken;
    } else {
      p.state[1] = count + (int)total;
    }
    p.state[2] = 0;
  }
}

// Opts the kernel into its largest shared memory once per device.
template <bool EXTEND>
int allow_smem() {
  static std::mutex mu;
  static std::set<int> done;
  int dev = 0;
  B2_TRY_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(dev)) return B2_OK;
  B2_TRY_CUDA(cudaFuncSetAttribute(block_tables_kernel<EXTEND>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   2 * kMaxSeqs * (int)sizeof(int)));
  done.insert(dev);
  return B2_OK;
}

template <bool EXTEND>
int launch(const TablesParams& p, int64_t items_bound, cudaStream_t stream) {
  const int rc = allow_smem<EXTEND>();
  if (rc) return rc;
  const int64_t want = (items_bound + kThreads * kPerThread - 1) / (kThreads * kPerThread);
  const int grid = (int)(want < 1 ? 1 : want > 2 * sm_count() ? 2 * sm_count() : want);
  B2_TRY_CUDA(launch_pdl(block_tables_kernel<EXTEND>, dim3(grid), dim3(kThreads),
                         (EXTEND ? 2 : 1) * (size_t)p.n_seqs * sizeof(int), stream, p));
  return B2_OK;
}

}  // namespace
}  // namespace b2

extern "C" {

int b2_block_tables_extend(int32_t* block_tables, int n_seqs, int table_stride, int32_t* lens,
                           const int32_t* new_lens, int block_size, int32_t* free_ring, int num_blocks,
                           int32_t* free_state, int max_tokens, int32_t* seq_start, int64_t* positions,
                           int32_t* table_index, int64_t* slots, int32_t* ctx_lens, int64_t* last_rows,
                           int32_t* status, b2_stream_t stream) {
  B2_CHECK_ARG(n_seqs > 0 && table_stride > 0 && block_size > 0 && num_blocks > 0 && max_tokens >= 0,
               "b2_block_tables_extend: bad sizes");
  if (n_seqs > b2::kMaxSeqs)
    return b2::fail(B2_ENOTSUP, "b2_block_tables_extend: %d sequences (at most %d)", n_seqs, b2::kMaxSeqs);
  B2_CHECK_ARG(block_tables && lens && new_lens && seq_start && last_rows,
               "b2_block_tables_extend: null pointer");
  B2_CHECK_ARG(max_tokens == 0 || (positions && table_index && slots && ctx_lens),
               "b2_block_tables_extend: null map");
  B2_CHECK_ARG((free_ring == nullptr) == (free_state == nullptr),
               "b2_block_tables_extend: the free ring and its state come together");
  b2::TablesParams p{};
  p.tables = block_tables;
  p.n_seqs = n_seqs;
  p.stride = table_stride;
  p.bs = block_size;
  p.lens = lens;
  p.arg = new_lens;
  p.ring = free_ring;
  p.num_blocks = num_blocks;
  p.state = free_state;
  p.max_tokens = max_tokens;
  p.seq_start = seq_start;
  p.positions = positions;
  p.table_index = table_index;
  p.slots = slots;
  p.ctx_lens = ctx_lens;
  p.last_rows = last_rows;
  p.status = status;
  return b2::launch<true>(p, max_tokens, stream);
}

int b2_block_tables_truncate(int32_t* block_tables, int n_seqs, int table_stride, int32_t* lens,
                             const int32_t* keep_lens, int block_size, int32_t* free_ring, int num_blocks,
                             int32_t* free_state, int32_t* status, b2_stream_t stream) {
  B2_CHECK_ARG(n_seqs > 0 && table_stride > 0 && block_size > 0 && num_blocks > 0,
               "b2_block_tables_truncate: bad sizes");
  if (n_seqs > b2::kMaxSeqs)
    return b2::fail(B2_ENOTSUP, "b2_block_tables_truncate: %d sequences (at most %d)", n_seqs, b2::kMaxSeqs);
  B2_CHECK_ARG(block_tables && lens && keep_lens && free_ring && free_state,
               "b2_block_tables_truncate: null pointer");
  b2::TablesParams p{};
  p.tables = block_tables;
  p.n_seqs = n_seqs;
  p.stride = table_stride;
  p.bs = block_size;
  p.lens = lens;
  p.arg = keep_lens;
  p.ring = free_ring;
  p.num_blocks = num_blocks;
  p.state = free_state;
  p.status = status;
  // At most the whole pool comes back.
  return b2::launch<false>(p, num_blocks, stream);
}

}  // extern "C"
