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
// Every CTA scans all n_seqs lengths by itself (lengths and two prefix sums kept in shared memory),
// which costs less than a second launch or a grid barrier would; the items (groups of tokens, or
// blocks to give back) are then spread over the grid, each finding its sequence by bisection
// of the prefix.  Nothing that a CTA reads is written before every CTA has read it: the last
// CTA to finish (a ticket in free_state[2], put back to 0) updates lens and the ring's state.
// A call that cannot be served whole (a bad length, a row past the table, too few free blocks,
// more tokens than the maps hold) raises its bit in *status and changes nothing.  A block id outside the pool, in
// the ring or in a table, is found only when its block is moved: it is moved as -1, and reported.
//
// Bound by latency: one extend and one truncate of 128 sequences with 5 new tokens each take 12.2 us in a graph, 16 new
// prompts of 1 024 tokens 9.5, 2 048 ragged sequences 20.0 (5.2 MB: 0.8 us of reading and writing); a chain of
// loads, scan, bisection, dependent loads and stores, and the ticket, twice.
#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"

namespace b2 {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxSeqs = 16384;  // three int32 arrays of this length fill 192 KB of shared memory
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
  bool fill;  // extend: entries of no token are written too
  int32_t* status;
};

struct Span {
  int items;   // extend: new tokens; truncate: blocks given back
  int blocks;  // extend: blocks taken
  bool bad;
};

// Blocks that hold n >= 0 tokens: the sum stays below 2^32.
__device__ __forceinline__ int blocks_of(const TablesParams& p, int n) {
  return (int)(((uint32_t)n + (uint32_t)p.bs - 1) / (uint32_t)p.bs);
}

template <bool EXTEND>
__device__ __forceinline__ Span span_of(const TablesParams& p, int len, int a) {
  Span r{0, 0, len < 0 || a < 0};
  if (r.bad) return r;
  const int held = blocks_of(p, len);
  if (EXTEND) {
    r.bad = (uint32_t)len + (uint32_t)a > 0x7fffffffu || blocks_of(p, len + a) > p.stride;
    r.items = a;
    r.blocks = r.bad ? 0 : blocks_of(p, len + a) - held;
  } else {
    r.bad = held > p.stride;
    r.items = r.bad ? 0 : held - blocks_of(p, min(a, len));
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

// Map entries i and on, as those of no token.
__device__ __forceinline__ void fill_from(const TablesParams& p, int64_t i) {
  for (i += (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < p.max_tokens; i += (int64_t)gridDim.x * blockDim.x) {
    p.positions[i] = -1;
    p.table_index[i] = 0;
    p.slots[i] = -1;
    p.ctx_lens[i] = 0;
  }
}

template <bool EXTEND>
__global__ void __launch_bounds__(kMaxThreads) block_tables_kernel(TablesParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ int sm[];
  int* lens = sm;                     // [n_seqs]
  int* item0 = sm + p.n_seqs;         // [n_seqs] items before sequence s
  int* third = sm + 2 * p.n_seqs;     // [n_seqs] extend: blocks taken before sequence s; truncate: tokens to keep
  __shared__ int64_t w_items[kMaxThreads / 32], w_blocks[kMaxThreads / 32];
  __shared__ int last_cta;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;

  // The lengths come in once, together; what they ask for stays in shared memory, since every later
  // step would wait for it again.
  bool bad = false;
  for (int s = tid; s < p.n_seqs; s += threads) {
    const int len = p.lens[s], a = p.arg[s];
    const Span x = span_of<EXTEND>(p, len, a);
    bad |= x.bad;
    lens[s] = len;
    item0[s] = x.items;
    third[s] = EXTEND ? x.blocks : min(a, len);
  }
  const bool alloc = p.ring != nullptr;
  const int head = alloc ? p.state[0] : 0, count = alloc ? p.state[1] : 0;
  bad = __syncthreads_or(bad);

  // Prefix sums over the sequences: each thread sums a run of consecutive ones.
  const int per = (p.n_seqs + threads - 1) / threads;
  const int s0 = min(p.n_seqs, tid * per), s1 = min(p.n_seqs, s0 + per);
  int64_t items = 0, blocks = 0;
  for (int s = s0; s < s1; ++s) {
    items += item0[s];
    if (EXTEND) blocks += third[s];
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
  __syncthreads();
  int64_t base_i = inc_i - items, base_b = inc_b - blocks, total = 0, taken = 0;
  for (int w = 0; w < threads / 32; ++w) {
    if (w < warp) {
      base_i += w_items[w];
      base_b += w_blocks[w];
    }
    total += w_items[w];
    taken += w_blocks[w];
  }
  int error = bad ? B2_DEV_RANGE : 0;
  if (alloc && (head < 0 || head >= p.num_blocks || count < 0 || count > p.num_blocks)) error = B2_DEV_RANGE;
  if (EXTEND) {
    if (total > p.max_tokens) error = B2_DEV_RANGE;
    if (!error && alloc && taken > count) error = B2_DEV_NO_BLOCKS;
  } else if (!error && count + total > p.num_blocks) {
    error = B2_DEV_RANGE;  // more blocks would come back than the pool has
  }
  if (error) {  // every CTA finds the same: nothing is changed
    if (blockIdx.x == 0 && tid == 0) raise_status(p.status, error);
    if (EXTEND && p.fill) {  // the maps of a step without tokens
      if (blockIdx.x == 0)
        for (int s = tid; s <= p.n_seqs; s += threads) {
          p.seq_start[s] = 0;
          if (s < p.n_seqs) p.last_rows[s] = -1;
        }
      fill_from(p, 0);
    }
    return;
  }
  for (int s = s0; s < s1; ++s) {
    const int n = item0[s];
    item0[s] = (int)base_i;
    if (EXTEND) {
      const int taken_here = third[s];
      third[s] = (int)base_b;
      base_b += taken_here;
      if (blockIdx.x == 0) {
        p.seq_start[s] = (int)base_i;
        p.last_rows[s] = n > 0 ? base_i + n - 1 : -1;
      }
    }
    base_i += n;
  }
  if (EXTEND && blockIdx.x == 0 && tid == 0) p.seq_start[p.n_seqs] = (int)total;
  if (EXTEND && p.fill) fill_from(p, total);
  __syncthreads();

  const int64_t step = (int64_t)gridDim.x * threads * kPerThread;
  for (int64_t i0 = ((int64_t)blockIdx.x * threads + tid) * kPerThread; i0 < total; i0 += step) {
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
      const int len = lens[s];
      if (EXTEND) {
        const int held = blocks_of(p, len);
        const int pos = len + (i - item0[s]);
        const int j = pos / p.bs, off = pos - j * p.bs;
        const bool take = alloc && j >= held;
        int blk = take ? p.ring[ring_slot(p, head, (int64_t)third[s] + (j - held))] : p.tables[(int64_t)s * p.stride + j];
        if (blk < 0 || blk >= p.num_blocks) {
          blk = -1;
          raise_status(p.status, B2_DEV_RANGE);
        }
        if (take && off == 0) p.tables[(int64_t)s * p.stride + j] = blk;  // a taken block's first token is new
        p.positions[i] = pos;
        p.table_index[i] = s;
        p.slots[i] = blk >= 0 ? (int64_t)blk * p.bs + off : -1;
        p.ctx_lens[i] = pos + 1;
      } else {
        int32_t* entry = p.tables + (int64_t)s * p.stride + blocks_of(p, third[s]) + (i - item0[s]);
        int blk = *entry;
        if (blk < 0 || blk >= p.num_blocks) {  // a hole in what the sequence should hold: it stays one
          blk = -1;
          raise_status(p.status, B2_DEV_RANGE);
        }
        p.ring[ring_slot(p, head, (int64_t)count + i)] = blk;
        *entry = -1;
      }
    }
  }
  if (!alloc) return;  // maps alone: no state to move on

  if (gridDim.x > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) last_cta = atomicAdd(&p.state[2], 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last_cta) return;
  }
  for (int s = tid; s < p.n_seqs; s += threads)
    p.lens[s] = EXTEND ? lens[s] + ((s + 1 < p.n_seqs ? item0[s + 1] : (int)total) - item0[s]) : third[s];
  if (tid == 0) {
    if (EXTEND) {
      p.state[0] = (int)ring_slot(p, head, taken);
      p.state[1] = count - (int)taken;
    } else {
      p.state[1] = count + (int)total;
    }
    if (gridDim.x > 1) p.state[2] = 0;
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
                                   3 * kMaxSeqs * (int)sizeof(int)));
  done.insert(dev);
  return B2_OK;
}

template <bool EXTEND>
int launch(const TablesParams& p, int64_t items_bound, cudaStream_t stream) {
  const int rc = allow_smem<EXTEND>();
  if (rc) return rc;
  // Every CTA reads all lengths: 2 048 sequences (one extend and one truncate) take 18.6 us with 512 threads and
  // 24.0 with 256, 128 sequences 12.0 and 11.2.  1024 threads are slower for both.
  const int threads = p.n_seqs > 1024 ? kMaxThreads : 256;
  const int64_t want = (items_bound + threads * kPerThread - 1) / (threads * kPerThread);
  const int grid = (int)(want < 1 ? 1 : want > 2 * sm_count() ? 2 * sm_count() : want);
  B2_TRY_CUDA(launch_pdl(block_tables_kernel<EXTEND>, dim3(grid), dim3(threads),
                         3 * (size_t)p.n_seqs * sizeof(int), stream, p));
  return B2_OK;
}

int extend(const char* name, bool fill, int32_t* block_tables, int n_seqs, int table_stride, int32_t* lens,
           const int32_t* new_lens, int block_size, int32_t* free_ring, int num_blocks, int32_t* free_state,
           int max_tokens, int32_t* seq_start, int64_t* positions, int32_t* table_index, int64_t* slots,
           int32_t* ctx_lens, int64_t* last_rows, int32_t* status, cudaStream_t stream) {
  B2_CHECK_ARG(n_seqs > 0 && table_stride > 0 && block_size > 0 && num_blocks > 0 && max_tokens >= 0,
               "%s: bad sizes", name);
  if (n_seqs > kMaxSeqs)
    return fail(B2_ENOTSUP, "%s: %d sequences (at most %d)", name, n_seqs, kMaxSeqs);
  B2_CHECK_ARG(block_tables && lens && new_lens && seq_start && last_rows, "%s: null pointer", name);
  B2_CHECK_ARG(max_tokens == 0 || (positions && table_index && slots && ctx_lens), "%s: null map", name);
  B2_CHECK_ARG((free_ring == nullptr) == (free_state == nullptr),
               "%s: the free ring and its state come together", name);
  TablesParams p{};
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
  p.fill = fill;
  p.status = status;
  return launch<true>(p, max_tokens, stream);
}

}  // namespace
}  // namespace b2

extern "C" {

int b2_block_tables_extend(int32_t* block_tables, int n_seqs, int table_stride, int32_t* lens,
                           const int32_t* new_lens, int block_size, int32_t* free_ring, int num_blocks,
                           int32_t* free_state, int max_tokens, int32_t* seq_start, int64_t* positions,
                           int32_t* table_index, int64_t* slots, int32_t* ctx_lens, int64_t* last_rows,
                           int32_t* status, b2_stream_t stream) {
  return b2::extend("b2_block_tables_extend", false, block_tables, n_seqs, table_stride, lens, new_lens, block_size,
                    free_ring, num_blocks, free_state, max_tokens, seq_start, positions, table_index, slots, ctx_lens,
                    last_rows, status, stream);
}

int b2_block_tables_extend_filled(int32_t* block_tables, int n_seqs, int table_stride, int32_t* lens,
                                  const int32_t* new_lens, int block_size, int32_t* free_ring, int num_blocks,
                                  int32_t* free_state, int max_tokens, int32_t* seq_start, int64_t* positions,
                                  int32_t* table_index, int64_t* slots, int32_t* ctx_lens, int64_t* last_rows,
                                  int32_t* status, b2_stream_t stream) {
  return b2::extend("b2_block_tables_extend_filled", true, block_tables, n_seqs, table_stride, lens, new_lens,
                    block_size, free_ring, num_blocks, free_state, max_tokens, seq_start, positions, table_index,
                    slots, ctx_lens, last_rows, status, stream);
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
  // What comes back is known on the device alone: at most the whole pool, most often a block or two per
  // sequence.  The grid has room for 32 blocks of each at once and walks what there is.
  return b2::launch<false>(p, std::min<int64_t>(num_blocks, 32 * (int64_t)n_seqs), stream);
}

}  // extern "C"
