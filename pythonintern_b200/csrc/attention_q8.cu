// Paged GQA attention over the 8-bit KV cache: one query token per row, or many per sequence.
//
// For a query at position p of a sequence, with the tile scales ks, vs of each block:
//   s_t = scale * ks[block(t)] * (q . kc_t),   out = sum_t softmax(s)_t * vs[block(t)] * vc_t,
// over the keys t the query may see; a query that sees none gives zeros.
#include "q8.cuh"

namespace b2 {
namespace {

struct Q8AttnParams {
  const void* q;
  int64_t ld_q;
  int n_rows, nq, nkv;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  int num_blocks;
  const int32_t* tables;
  int table_rows, table_stride;
  // one token per row: keys 0 .. ctx_lens[row] - 1 of table row table_index[row] (null: row)
  const int32_t* table_index;
  const int32_t* ctx_lens;
  int compat_pad;
  // many tokens per sequence (seq_start not null): row r of sequence s sees keys
  // 0 .. seq_ctx0[s] + r - seq_start[s]
  const int32_t* seq_start;
  const int32_t* seq_ctx0;
  int n_seqs;
  float scale_log2;
  void* out;
  int64_t ld_out;
  int32_t* status;
};

constexpr int kRowThreads = 128;

// The simplest form: one CTA per (query row, q head), 128 keys at a time.
template <typename T, int HD, int CODE>
__global__ void __launch_bounds__(kRowThreads) q8_attn_row_kernel(Q8AttnParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sq[HD], sp[kRowThreads], red[32];
  __shared__ int64_t sblk[kRowThreads];
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int g = h / (p.nq / p.nkv);
  int trow, ctx;
  if (p.seq_start) {
    int s = -1;
    for (int i = 0; i < p.n_seqs; ++i)
      if (row >= p.seq_start[i] && row < p.seq_start[i + 1]) s = i;
    if (s < 0) return;  // behind the last sequence: left as it was
    trow = s;
    ctx = (p.seq_ctx0 ? p.seq_ctx0[s] : 0) + row - p.seq_start[s] + 1;
  } else {
    trow = p.table_index ? p.table_index[row] : row;
    ctx = max(0, p.ctx_lens[row]);
  }
  if (trow < 0 || trow >= p.table_rows || (int64_t)p.table_stride * kQ8Block < ctx) {
    if (tid == 0) raise_status(p.status, B2_DEV_RANGE);
    ctx = trow < 0 || trow >= p.table_rows ? 0 : p.table_stride * kQ8Block;
  }
  int npad = 0;
  if (p.compat_pad) {
    int mx = 0;
    for (int i = 0; i < p.n_rows; ++i) mx = max(mx, p.ctx_lens[i]);
    npad = max(0, mx - ctx);
  }
  const int32_t* table = p.tables + (int64_t)trow * p.table_stride;
  const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)row * p.ld_q + (int64_t)h * HD;
  for (int d = tid; d < HD; d += kRowThreads) sq[d] = to_f32(q[d]);
  float m = npad > 0 ? 0.f : -INFINITY, l = (float)npad, acc = 0.f;
  for (int t0 = 0; t0 < ctx; t0 += kRowThreads) {
    __syncthreads();
    const int t = t0 + tid;
    float s = -INFINITY;
    int64_t blk = -1;
    if (t < ctx) {
      blk = table[t / kQ8Block];
      if (blk < 0 || blk >= p.num_blocks) {
        raise_status(p.status, B2_DEV_RANGE);
        blk = -1;
      } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(p.k_cache + q8_tile(blk, p.nkv, g, HD) + t % kQ8Block * HD);
        float dot = 0.f;
        for (int i = 0; i < HD / 4; ++i) {
          float v[4];
          Q8<CODE>::decode4(w[i], v);
          for (int e = 0; e < 4; ++e) dot = fmaf(v[e], sq[i * 4 + e], dot);
        }
        s = dot * p.k_scale[q8_scale(blk, p.nkv, g)] * p.scale_log2;
      }
    }
    sblk[tid] = blk;
    float mx = warp_max(s);
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    mx = m;
    for (int w = 0; w < kRowThreads / 32; ++w) mx = fmaxf(mx, red[w]);
    const float corr = mx == -INFINITY ? 1.f : exp2f(m - mx);
    sp[tid] = blk < 0 ? 0.f : exp2f(s - mx);
    __syncthreads();
    m = mx;
    l *= corr;
    acc *= corr;
    const int n = min(kRowThreads, ctx - t0);
    for (int i = 0; i < n; ++i) {
      l += sp[i];
      if (tid < HD && sblk[i] >= 0) {
        float v[4];
        Q8<CODE>::decode4(p.v_cache[q8_tile(sblk[i], p.nkv, g, HD) + (t0 + i) % kQ8Block * HD + tid], v);
        acc = fmaf(sp[i] * p.v_scale[q8_scale(sblk[i], p.nkv, g)], v[0], acc);
      }
    }
  }
  if (tid < HD) {
    T* out = reinterpret_cast<T*>(p.out) + (int64_t)row * p.ld_out + (int64_t)h * HD;
    out[tid] = from_f32<T>(l == 0.f ? 0.f : acc / l);
  }
}

int check_q8_attention(const char* name, const Q8AttnParams& p, int hd, int cache_dtype, int layer, int bs, int dtype) {
  B2_CHECK_ARG(p.n_rows >= 0 && p.nq > 0 && p.nkv > 0 && p.nq % p.nkv == 0, "%s: bad head counts", name);
  B2_CHECK_ARG(valid_dtype(dtype), "%s: bad dtype", name);
  B2_CHECK_ARG(valid_q8_dtype(cache_dtype), "%s: bad cache dtype", name);
  B2_CHECK_ARG(p.num_blocks > 0 && p.table_stride > 0 && p.table_rows > 0 && layer >= 0, "%s: bad cache geometry", name);
  B2_CHECK_ARG(p.table_stride <= 0x7fffffff / kQ8Block, "%s: table_stride %d too large", name, p.table_stride);
  if (bs != kQ8Block) return fail(B2_ENOTSUP, "%s: block_size %d (16 only)", name, bs);
  if (hd != 32 && hd != 64 && hd != 128) return fail(B2_ENOTSUP, "%s: head_dim %d not supported (32, 64, 128)", name, hd);
  if (p.nq / p.nkv > 16) return fail(B2_ENOTSUP, "%s: nq/nkv = %d not supported (1..16)", name, p.nq / p.nkv);
  B2_CHECK_ARG(p.ld_q >= (int64_t)p.nq * hd && p.ld_out >= (int64_t)p.nq * hd, "%s: row strides too small", name);
  return B2_OK;
}

int check_q8_pointers(const char* name, const Q8AttnParams& p, int dtype) {
  B2_CHECK_ARG(p.q && p.k_cache && p.v_cache && p.k_scale && p.v_scale && p.tables && p.out, "%s: null pointer", name);
  const size_t esz = dtype_bytes(dtype);
  B2_CHECK_ARG(((uintptr_t)p.q % 16) == 0 && ((p.ld_q * esz) % 16) == 0 && ((uintptr_t)p.out % 16) == 0 &&
                   ((p.ld_out * esz) % 16) == 0 && ((uintptr_t)p.k_cache % 16) == 0 && ((uintptr_t)p.v_cache % 16) == 0,
               "%s: q, out and the cache must be 16-byte aligned", name);
  return B2_OK;
}

template <typename T, int HD>
int launch_rows(const Q8AttnParams& p, int cache_dtype, cudaStream_t s) {
  const dim3 grid(p.n_rows, p.nq);
  if (cache_dtype == B2_I8)
    B2_TRY_CUDA(launch_pdl((q8_attn_row_kernel<T, HD, B2_I8>), grid, dim3(kRowThreads), 0, s, p));
  else
    B2_TRY_CUDA(launch_pdl((q8_attn_row_kernel<T, HD, B2_E4M3>), grid, dim3(kRowThreads), 0, s, p));
  return B2_OK;
}

int launch(const Q8AttnParams& p, int hd, int cache_dtype, int dtype, cudaStream_t s) {
  if (dtype == B2_BF16) {
    if (hd == 32) return launch_rows<__nv_bfloat16, 32>(p, cache_dtype, s);
    if (hd == 64) return launch_rows<__nv_bfloat16, 64>(p, cache_dtype, s);
    return launch_rows<__nv_bfloat16, 128>(p, cache_dtype, s);
  }
  if (hd == 32) return launch_rows<float, 32>(p, cache_dtype, s);
  if (hd == 64) return launch_rows<float, 64>(p, cache_dtype, s);
  return launch_rows<float, 128>(p, cache_dtype, s);
}

void set_cache(Q8AttnParams& p, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
               int layer, int hd) {
  const size_t tiles = (size_t)layer * p.num_blocks * p.nkv;
  p.k_cache = static_cast<const uint8_t*>(k_cache) + tiles * kQ8Block * hd;
  p.v_cache = static_cast<const uint8_t*>(v_cache) + tiles * kQ8Block * hd;
  p.k_scale = k_scale + tiles;
  p.v_scale = v_scale + tiles;
}

}  // namespace
}  // namespace b2

extern "C" {

size_t b2_paged_attention_q8_workspace_bytes(int n_rows, int nq, int nkv, int head_dim) { return 0; }

int b2_paged_attention_q8(const void* q, int64_t ld_q, int n_rows, int nq, int nkv, int head_dim, const void* k_cache,
                          const void* v_cache, const float* k_scale, const float* v_scale, int cache_dtype, int layer,
                          int num_blocks, int block_size, const int32_t* block_tables, int table_rows,
                          int table_stride, const int32_t* table_index, const int32_t* ctx_lens, int compat_pad,
                          float scale, void* out, int64_t ld_out, int dtype, void* workspace, size_t workspace_bytes,
                          int32_t* status, b2_stream_t stream) {
  using namespace b2;
  const char* name = "b2_paged_attention_q8";
  Q8AttnParams p{q, ld_q, n_rows, nq, nkv, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale,
                 num_blocks, block_tables, table_rows, table_stride, table_index, ctx_lens, compat_pad, nullptr,
                 nullptr, 0, scale * 1.4426950408889634f, out, ld_out, status};
  int rc = check_q8_attention(name, p, head_dim, cache_dtype, layer, block_size, dtype);
  if (rc || n_rows == 0) return rc;
  rc = check_q8_pointers(name, p, dtype);
  if (rc) return rc;
  B2_CHECK_ARG(ctx_lens, "%s: null pointer", name);
  B2_CHECK_ARG(table_index || n_rows <= table_rows, "%s: %d rows for %d table rows", name, n_rows, table_rows);
  set_cache(p, k_cache, v_cache, k_scale, v_scale, layer, head_dim);
  return launch(p, head_dim, cache_dtype, dtype, stream);
}

size_t b2_prefill_attention_q8_workspace_bytes(int n_rows, int nq, int nkv, int head_dim, int n_seqs) { return 0; }

int b2_prefill_attention_q8(const void* q, int64_t ld_q, int n_rows, int nq, int nkv, int head_dim,
                            const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                            int cache_dtype, int layer, int num_blocks, int block_size, const int32_t* block_tables,
                            int table_rows, int table_stride, const int32_t* seq_start, const int32_t* seq_ctx0,
                            int n_seqs, float scale, void* out, int64_t ld_out, int dtype, void* workspace,
                            size_t workspace_bytes, int32_t* status, b2_stream_t stream) {
  using namespace b2;
  const char* name = "b2_prefill_attention_q8";
  Q8AttnParams p{q, ld_q, n_rows, nq, nkv, (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale,
                 num_blocks, block_tables, table_rows, table_stride, nullptr, nullptr, 0, seq_start, seq_ctx0, n_seqs,
                 scale * 1.4426950408889634f, out, ld_out, status};
  int rc = check_q8_attention(name, p, head_dim, cache_dtype, layer, block_size, dtype);
  if (rc) return rc;
  B2_CHECK_ARG(n_seqs >= 0, "%s: bad sizes", name);
  if (n_rows == 0 || n_seqs == 0) return B2_OK;
  rc = check_q8_pointers(name, p, dtype);
  if (rc) return rc;
  B2_CHECK_ARG(seq_start, "%s: null pointer", name);
  B2_CHECK_ARG(n_seqs <= table_rows, "%s: %d sequences for %d table rows", name, n_seqs, table_rows);
  set_cache(p, k_cache, v_cache, k_scale, v_scale, layer, head_dim);
  return launch(p, head_dim, cache_dtype, dtype, stream);
}

}  // extern "C"
