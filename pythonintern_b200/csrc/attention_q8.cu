// Paged GQA attention over the 8-bit KV cache: one query token per row, or many per sequence.
//
// For a query at position p of a sequence, with the tile scales ks, vs of each block:
//   s_t = scale * ks[block(t)] * (q . kc_t),   out = sum_t softmax(s)_t * vs[block(t)] * vc_t,
// over the keys t the query may see; a query that sees none gives zeros.
//
// Work.  A tile is up to 8 * NT (query token, q head) columns that share a kv head: the heads
// of one decode row, or those of consecutive tokens of one sequence.  It reads ceil(keys / 16)
// blocks; the blocks of all tiles and heads in a row form one line of steps, cut into equal
// chunks, one per resident warp, so ragged contexts cost no more than even ones.  A warp works
// alone (no barrier in the loop).  A tile that lies in one chunk is finished there; the pieces of
// others go to the workspace as softmax states.  Those of one CTA are joined by its own warps after its
// loop; only a tile that reaches over CTAs, at most one begins in each, is left to a second kernel.
// Every CTA finds the cut by itself from the lengths, so nothing waits on the host.
//
// What bounds it (heads 32/8 of 128, measured in a graph): int8 decode of 128 rows over 2 048 keys reads 540 MB in
// 100-107 us, 5.0-5.4 TB/s of 6.55 measured (its loop runs at the copy's rate; 4.5 us go to finding the cut and
// the first tiles, some 8 to filling and draining and the join); one row over 8 192 keys 17 us, of which
// 2.6 are reading; drafts of 5 tokens for 48 sequences 96 us, bound by the work on a step (expanding
// codes, products, softmax), not by its bytes.
//
// One step.  S^T[16 keys x 8 NT] = K Q^T and O^T[head_dim x 8 NT] += V^T P^T on
// mma.sync.m16n8k16 with float16 operands and float32 sums.  A code of 8 bits is exact in
// float16, so nothing is rounded on the way in.
//  * The tiles of K and V (one block and kv head: 16 * head_dim bytes in one run) come by cp.async
//    into a three-stage ring of the warp's own, two steps ahead and across the ends of tiles.
//  * K: lane (r, t) = (lane / 4, lane % 4) reads head_dim / 4 contiguous codes of keys r and
//    r + 8.  The order of the head_dim axis inside the product is free, so its codes are taken
//    as the k indexes of that lane and q is laid out to match.
//  * V: the lane reads head_dim / 8 codes of the keys 2t, 2t+1, 2t+8, 2t+9; a byte shuffle pairs
//    two keys' codes of one dimension, which is the transposed operand.
//  * P^T leaves the S^T fragments for the B fragments by an 8x8 transpose in registers.
//  * q is scaled by a power of two per column, so that its largest magnitude is near 2^14, and
//    split: one float16 term holds bf16 (values 2^-38 below the largest are cut), two hold
//    float32 up to 2^-22 of an element.
// Softmax statistics are float32: l = sum 2^(s - m), and P = 2^(s - m) vs 2^(m - m2) is rounded to
// float16 (to two terms for float32 queries).  The second reference m2 follows the largest
// s + log2(vs), so a scale that differs by orders of magnitude between blocks costs no precision; it stays
// within 2^100 of m, however loud the keys of V tiles of zeros are.
// References move only when a value would pass 2^15 and then to where it is 2^8, so the common
// step needs no maximum across lanes, only one vote.
#include "q8.cuh"

#include <algorithm>
#include <mutex>
#include <set>
#include <type_traits>
#include <utility>

namespace b2 {

bool prefill_q8_tc_serves(int rep);
int prefill_attention_q8_tc(const void* q, int64_t ld_q, int n_rows, int nq, int nkv, const uint8_t* k_cache,
                            const uint8_t* v_cache, const float* k_scale, const float* v_scale, int cache_dtype,
                            int num_blocks, const int32_t* tables, int table_stride, const int32_t* seq_start,
                            const int32_t* seq_ctx0, int n_seqs, float scale, void* out, int64_t ld_out,
                            int32_t* status, cudaStream_t stream);

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
  // workspace
  int4* ws_open;    // [CTAs]: the (tile, kv head) that begins in a CTA and ends in a later one: that
                    // CTA (-1: there is none), unit, tile in it, kv head
  int2* ws_piece;   // [CTAs]: slots of the CTA's piece of one that began before it, and of that one
  float4* ws_stat;  // [slots][columns]: m, l, m2
  float* ws_o;      // [slots][columns][head_dim]
};


// ------------------------------------------------------------------ the cut of the work
constexpr int kGroups = 256;   // prefix sums kept in shared memory
constexpr int kMinChunk = 2;   // steps a warp takes at least

struct Unit {  // a decode row, or a sequence of a prefill
  int start, len, ctx0;  // first row of q, tokens, keys before the first token
};

__device__ __forceinline__ int table_row(const Q8AttnParams& p, int u) {
  return !p.seq_start && p.table_index ? p.table_index[u] : u;
}

__device__ __forceinline__ Unit unit_of(const Q8AttnParams& p, int u, bool& bad) {
  Unit r{u, 0, 0};
  const int64_t most = (int64_t)p.table_stride * kQ8Block;
  if (!p.seq_start) {
    const int row = table_row(p, u), ctx = p.ctx_lens[u];
    const bool there = row >= 0 && row < p.table_rows;
    bad = !there || ctx > most;
    const int keys = there ? (int)min((int64_t)ctx, most) : 0;  // a context past its table row: the row's keys
    r.len = keys > 0 ? 1 : 0;
    r.ctx0 = keys - 1;
  } else {
    const int a = p.seq_start[u], b = p.seq_start[u + 1];
    const int ctx0 = p.seq_ctx0 ? p.seq_ctx0[u] : 0;
    bad = a < 0 || b > p.n_rows || b < a || ctx0 < 0 || (b > a && (int64_t)ctx0 + b - a > most);
    if (!bad) {
      r.start = a;
      r.len = b - a;
      r.ctx0 = ctx0;
    }
  }
  return r;
}

__device__ __forceinline__ Unit unit_of(const Q8AttnParams& p, int u) {
  bool bad;
  return unit_of(p, u, bad);
}

__device__ __forceinline__ int blocks_of(int64_t keys) {
  return (int)((uint64_t)(keys + kQ8Block - 1) / kQ8Block);
}

// Blocks of the first x tiles of a unit: sum over j = 1..x of ceil((ctx0 + min(j qt, len)) / 16).
// Over the full tiles the remainders repeat with period 16 / gcd(qt, 16), and every further
// period adds the same number to each of its terms.
__device__ __forceinline__ int64_t blocks_before(const Unit& u, int qt, int x) {
  if (x <= 1) return x == 0 ? 0 : blocks_of((int64_t)u.ctx0 + min(qt, u.len));  // a decode row, say
  const int full = min(x, u.len / qt);
  int per = kQ8Block;
  while (per > 1 && (qt * (per / 2)) % kQ8Block == 0) per /= 2;
  const int64_t rounds = full / per, add = (int64_t)qt * per / kQ8Block;
  int64_t one = 0;
  for (int j = 1; j <= min(per, full); ++j) one += blocks_of((int64_t)u.ctx0 + j * qt);
  int64_t sum = rounds * one + per * add * (rounds * (rounds - 1) / 2);
  if (rounds == 0) sum = one;
  else
    for (int j = (int)rounds * per + 1; j <= full; ++j) sum += blocks_of((int64_t)u.ctx0 + (int64_t)j * qt);
  if (x > full) sum += blocks_of((int64_t)u.ctx0 + u.len);
  return sum;
}

__device__ __forceinline__ int tiles_of(const Unit& u, int qt) { return u.len <= 1 ? u.len : (u.len + qt - 1) / qt; }

struct Cut {
  int64_t total;  // steps of the call, all kv heads
  int64_t chunk;  // steps per warp
  int tiles;
  int max_ctx;    // longest context (compat_pad)
};

// What every CTA keeps in shared memory of the line of steps.
struct Line {
  int64_t steps[kGroups];  // blocks (of one kv head) before a group of units
  int tiles[kGroups];      // tiles before it
  Unit unit[kGroups];      // its first unit
};

// Prefix sums over groups of units.  Called by the whole CTA.
template <int WARPS>
__device__ __forceinline__ Cut make_cut(const Q8AttnParams& p, int qt, int n_units, int per_group, Line& line,
                                        int warps, bool report) {
  __shared__ int64_t w_steps[WARPS];
  __shared__ int w_tiles[WARPS], w_ctx[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int threads = 32 * WARPS;
  const int groups = (n_units + per_group - 1) / per_group;
  const int per_thread = (groups + threads - 1) / threads;
  int64_t steps = 0;
  int tiles = 0, max_ctx = 0;
  bool bad = false;
  const int g0 = min(groups, tid * per_thread), g1 = min(groups, g0 + per_thread);
  for (int g = g0; g < g1; ++g) {
    line.steps[g] = steps;
    line.tiles[g] = tiles;
    for (int u = g * per_group; u < min(n_units, (g + 1) * per_group); ++u) {
      bool odd;
      const Unit x = unit_of(p, u, odd);
      if (u == g * per_group) line.unit[g] = x;
      bad |= odd;
      const int n = tiles_of(x, qt);
      steps += blocks_before(x, qt, n);
      tiles += n;
      if (p.compat_pad) max_ctx = max(max_ctx, p.ctx_lens[u]);
    }
  }
  if (report && bad) raise_status(p.status, B2_DEV_RANGE);
  int64_t inc_s = steps;
  int inc_t = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, inc_s, o);
    const int b = __shfl_up_sync(0xffffffffu, inc_t, o);
    max_ctx = max(max_ctx, __shfl_xor_sync(0xffffffffu, max_ctx, o));
    if (lane >= o) {
      inc_s += a;
      inc_t += b;
    }
  }
  if (lane == 31) {
    w_steps[warp] = inc_s;
    w_tiles[warp] = inc_t;
    w_ctx[warp] = max_ctx;
  }
  __syncthreads();
  Cut c{0, 0, 0, 0};
  int64_t base_s = inc_s - steps;
  int base_t = inc_t - tiles;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) {
      base_s += w_steps[w];
      base_t += w_tiles[w];
    }
    c.total += w_steps[w];
    c.tiles += w_tiles[w];
    c.max_ctx = max(c.max_ctx, w_ctx[w]);
  }
  for (int g = g0; g < g1; ++g) {
    line.steps[g] += base_s;
    line.tiles[g] += base_t;
  }
  __syncthreads();
  c.total *= p.nkv;
  const int64_t even =
      c.total >> 32 ? (c.total + warps - 1) / warps : ((uint32_t)c.total + warps - 1) / (uint32_t)warps;
  c.chunk = max((int64_t)kMinChunk, even);
  return c;
}

struct Place {  // where a step lies
  Unit unit;
  int u, j;       // unit and tile in it
  int tile;       // number of the tile in the call
  int g;          // kv head
  int block;      // block in the tile
  int blocks;     // blocks of the tile
  int begin;      // first step of (tile, kv head), counted from the warp's first
};

// Finds step x of the line; the same for all lanes of a warp.
__device__ __forceinline__ Place find_step(const Q8AttnParams& p, int64_t x, int qt, int n_units, int per_group,
                                           const Line& line) {
  const int groups = (n_units + per_group - 1) / per_group;
  // the last group that begins at or before x (empty ones share their successor's begin): every lane looks at
  // some, which waits for shared memory once where a bisection would eight times
  int lo = 0;
#pragma unroll
  for (int g = 0; g < kGroups; g += 32)
    if (g + (int)(threadIdx.x & 31) < groups && line.steps[g + (threadIdx.x & 31)] * p.nkv <= x) ++lo;
  lo = __reduce_add_sync(0xffffffffu, lo) - 1;
  Place r;
  r.u = lo * per_group;
  r.tile = line.tiles[lo];
  int64_t before = line.steps[lo];
  for (r.unit = line.unit[lo];; r.unit = unit_of(p, ++r.u)) {
    const int n = tiles_of(r.unit, qt);
    const int64_t all = blocks_before(r.unit, qt, n);
    if (x < (before + all) * p.nkv || r.u == n_units - 1) break;
    before += all;
    r.tile += n;
  }
  int a = 0, b = tiles_of(r.unit, qt) - 1;
  while (a < b) {
    const int mid = (a + b + 1) >> 1;
    if ((before + blocks_before(r.unit, qt, mid)) * p.nkv <= x) a = mid; else b = mid - 1;
  }
  r.j = a;
  r.tile += a;
  before += blocks_before(r.unit, qt, a);
  r.blocks = blocks_of((int64_t)r.unit.ctx0 + min((a + 1) * qt, r.unit.len));
  const int64_t in = x - before * p.nkv;
  r.g = in >> 32 ? (int)(in / r.blocks) : (int)((uint32_t)in / (uint32_t)r.blocks);
  r.block = (int)(in - (int64_t)r.g * r.blocks);
  r.begin = -r.block;
  return r;
}

// Moves to the first step of the next (tile, kv head).
__device__ __forceinline__ void next_pair(const Q8AttnParams& p, Place& r, int qt, int per_group, const Line& line) {
  r.begin += r.blocks;
  r.block = 0;
  if (++r.g < p.nkv) return;
  r.g = 0;
  ++r.tile;
  ++r.j;
  while (r.j >= tiles_of(r.unit, qt)) {  // the caller has checked that there is another step
    ++r.u;
    r.unit = per_group == 1 ? line.unit[r.u] : unit_of(p, r.u);
    r.j = 0;
  }
  r.blocks = blocks_of((int64_t)r.unit.ctx0 + min((r.j + 1) * qt, r.unit.len));
}

// ------------------------------------------------------------------ fragments
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Two pairs of codes (the bytes 0, 1 and 2, 3 of x) as float16 pairs.  BIASED: as the float16
// numbers (code + 128) * 2^-24, whose bits are the byte itself.
template <int CODE, bool BIASED = false>
__device__ __forceinline__ void expand(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if constexpr (BIASED) {
    const uint32_t u = x ^ 0x80808080u;
    lo = prmt(u, 0u, 0x4140);
    hi = prmt(u, 0u, 0x4342);
  } else if constexpr (CODE == B2_I8) {
    // 0x6400 | u is the float16 1024 + u for a byte u; u = code + 128
    const uint32_t u = x ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t a = prmt(u, 0x64646464u, 0x4140), b = prmt(u, 0x64646464u, 0x4342);
    const __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    const __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  }
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Four elements of q, as they are in memory.
template <typename T>
struct Raw4 {
  using Type = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;
};
__device__ __forceinline__ void widen4(const float4& a, float (&v)[4]) {
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void widen4(const uint2& a, float (&v)[4]) {
  v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
  v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
}

constexpr float kRoom = 15.f;       // log2 of the largest P
constexpr float kLift = 8.f;        // log2 of the largest P when a reference has just moved
constexpr float kNoRef = -1e30f;    // reference of a column that has seen no key
// m2 is held within 2^kGap of m, which runs ahead of it where V tiles of scale 0 hold the loudest keys: 2^(m - m2)
// stays finite, and what float16 cuts off P (2^-25) is 2^-133 of a code, since l is 2^8 or more.
constexpr float kGap = 100.f;

// One CTA per SM, of as many warps as its registers allow (decode of 128 rows over 2 048 keys, 8 heads of 128: 100 us
// with 12 warps; 16 of them spill), each with a ring of three tiles of K and V: a fourth is no faster, nor
// are two blocks at a time.
constexpr int warps_of(int hd, int nt, int terms) {
  return nt * terms > 2 ? 8 : nt * terms == 2 || hd == 128 ? 12 : 16;
}

template <typename T, int HD, int CODE, int NT>
struct AttnCfg {
  static constexpr int N = 8 * NT;                       // columns of a tile
  static constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;   // float16 terms of q and P
  // S from K codes + 128 taken as float16 subnormals: q . (c + 128) - 128 sum(q), half the work of
  // making signed numbers of them.  It costs S a rounding of 128 |sum q| in float32, nothing
  // next to the float16 of P; float32 queries do without.
  static constexpr bool BIASED = CODE == B2_I8 && TERMS == 1;
  static constexpr int KW = HD / 16;                     // words of codes a lane holds of a key; MMAs of S
  static constexpr int VW = HD / 32;                     // and of a key's values
  static constexpr int TILE = kQ8Block * HD;             // bytes of codes of one block and head
  static constexpr int Q_BYTES = KW * NT * TERMS * 32 * 8;
  static constexpr int WARPS = warps_of(HD, NT, TERMS);
  static constexpr int STAGES = 3;                       // tiles of K and V a warp holds or has in flight
  static constexpr int WARP_BYTES = STAGES * 2 * TILE;
  // rings, then the q fragments
  static constexpr int SMEM = WARPS * (WARP_BYTES + Q_BYTES);
  static_assert(SMEM + (int)sizeof(Line) + 512 <= 232448, "shared memory above the 227 KB a CTA may use");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

// Byte offset of 16-byte chunk `chunk` of key row `row` in a tile in shared memory: chunks are
// swapped by the row's place in 128 bytes, so that eight lanes reading a column of chunks, or a
// row of them, touch different banks.
template <int HD>
__device__ __forceinline__ int tile_at(int row, int chunk) {
  constexpr int CHUNKS = HD / 16;
  return row * HD + ((chunk ^ (row * HD / 128 & (CHUNKS - 1))) << 4);
}

// A softmax in part: l = sum 2^(s - m), o = sum 2^(s - m2) vs v; a lane's HD / 32 dims.
template <int HD>
struct Piece {
  float m, l, m2, o[HD / 32];
};

// Column c of n pieces in the workspace as one.  The warp's share of o: pieces part_of, part_of +
// share, ...
template <int HD, typename SlotOf>
__device__ __forceinline__ Piece<HD> join_pieces(const Q8AttnParams& p, const SlotOf& slot_of, int n, int columns,
                                                 int c, int part_of, int share, int lane) {
  constexpr int E = HD / 32, BATCH = 4;  // pieces in flight
  Piece<HD> r;
  float v[BATCH][E], z[BATCH];
  auto fetch = [&](int k) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int64_t at = (int64_t)slot_of(min(k + b * share, n - 1)) * columns + c;
      z[b] = p.ws_stat[at].z;
#pragma unroll
      for (int e = 0; e < E; ++e) v[b][e] = p.ws_o[at * HD + lane * E + e];
    }
  };
  fetch(part_of);
  float m = kNoRef, l = 0.f, m2 = kNoRef;
  for (int k = lane; k < n; k += 32) {
    const float4 st = p.ws_stat[(int64_t)slot_of(k) * columns + c];
    const float mn = fmaxf(m, st.x);
    l = l * exp2f(m - mn) + st.y * exp2f(st.x - mn);
    m = mn;
    m2 = fmaxf(m2, st.z);
  }
  r.m = warp_max(m);
  r.m2 = warp_max(m2);
  r.l = warp_sum(l * exp2f(m - r.m));
#pragma unroll
  for (int e = 0; e < E; ++e) r.o[e] = 0.f;
  for (int k = part_of; k < n; k += BATCH * share) {
    if (k != part_of) fetch(k);
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const float f = k + b * share < n ? exp2f(z[b] - r.m2) : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) r.o[e] = k + b * share < n ? fmaf(v[b][e], f, r.o[e]) : r.o[e];
    }
  }
  return r;
}

// The result of one row and q head; npad keys of score 0 and value 0 join its denominator.
template <typename T, int HD>
__device__ __forceinline__ void write_head(const Q8AttnParams& p, int row, int head, int lane, const Piece<HD>& r,
                                           int npad) {
  constexpr int E = HD / 32;
  const float l = npad > 0 ? r.l + (float)npad * exp2f(-r.m) : r.l;
  const float f = r.m2 == kNoRef ? (l == l ? 0.f : l) : exp2f(r.m2 - r.m) / l;
  T* dst = reinterpret_cast<T*>(p.out) + (int64_t)row * p.ld_out + (int64_t)head * HD + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = from_f32<T>(r.o[e] * f);
}

struct Join {
  int warp, slot, pieces, whole, row, g, ncol, npad;
};

// Up to 32 consecutive steps of one (tile, kv head); lane i holds what step i needs.
struct Window {
  int cnt;       // steps; 0: behind the warp's chunk
  int g;         // kv head
  int id;        // block id, -1 outside the pool
  float ks, vs;  // scales
};

template <typename T, int HD, int CODE, int NT>
__global__ void __launch_bounds__(AttnCfg<T, HD, CODE, NT>::WARPS * 32, 1)
q8_attn_kernel(const Q8AttnParams p, int qt, int n_units, int per_group) {
  pdl_wait();
  pdl_trigger();
  using C = AttnCfg<T, HD, CODE, NT>;
  constexpr int KW = C::KW, VW = C::VW, TERMS = C::TERMS, N = C::N, STAGES = C::STAGES, WARPS = C::WARPS;
  __shared__ Line line;
  __shared__ Join joins[WARPS];
  __shared__ int n_joins;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r8 = lane >> 2, t4 = lane & 3;
  const int warps = gridDim.x * WARPS, w = blockIdx.x * WARPS + warp;
  const int rep = p.nq / p.nkv;
  const uint32_t ring_at = smem_u32(smem) + warp * C::WARP_BYTES;
  uint2* sq = reinterpret_cast<uint2*>(smem + WARPS * C::WARP_BYTES + warp * C::Q_BYTES) + lane;
  const uint32_t sq_at = smem_u32(sq);
  // what the lane reads of a tile: its codes of keys r8 (and, 8 rows on, r8 + 8), of keys 2 t4 and
  // 2 t4 + 1 (and 8 rows on)
  uint32_t k_off[KW == 8 ? 2 : 1], v_off[2];
#pragma unroll
  for (int c = 0; c < (KW == 8 ? 2 : 1); ++c)
    k_off[c] = KW == 2 ? tile_at<HD>(r8, t4 >> 1) + (t4 & 1) * 8 : tile_at<HD>(r8, t4 * (KW / 4) + c);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    v_off[h] = C::TILE + (VW == 4   ? tile_at<HD>(2 * t4 + h, r8)
                          : VW == 2 ? tile_at<HD>(2 * t4 + h, r8 >> 1) + (r8 & 1) * 8
                                    : tile_at<HD>(2 * t4 + h, r8 >> 2) + (r8 & 3) * 4);

  const Cut cut = make_cut<WARPS>(p, qt, n_units, per_group, line, warps, blockIdx.x == 0);
  // a seq_start that goes back may name more tokens than there are rows: nothing is computed
  const bool sane = !p.seq_start || (int64_t)cut.tiles <= (int64_t)(p.n_rows / qt) + n_units;
  if (threadIdx.x == 0) {
    p.ws_open[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (!sane && blockIdx.x == 0) raise_status(p.status, B2_DEV_RANGE);
  }
  if (!sane) return;
  const int64_t x_begin = w * cut.chunk, x_end = min(cut.total, x_begin + cut.chunk);
  if (!p.seq_start) {  // decode rows without keys: from the last warps, which have the least to do
    for (int u = warps - 1 - w; u < n_units; u += warps) {
      if ((per_group == 1 ? line.unit[u] : unit_of(p, u)).len > 0) continue;
      T* dst = reinterpret_cast<T*>(p.out) + (int64_t)u * p.ld_out;
      for (int i = lane; i < p.nq * HD; i += 32) dst[i] = from_f32<T>(0.f);
    }
  }

  int left = (int)max((int64_t)0, x_end - x_begin);  // steps behind the windows taken so far
  // The window that begins at `from` (cnt 0 at the end of the chunk): starts the loads of its ids.
  auto take = [&](const Place& from) -> Window {
    Window win;
    win.cnt = min(min(32, from.blocks - from.block), left);
    left -= win.cnt;
    win.g = from.g;
    win.id = -1;
    if (lane < win.cnt)
      win.id = p.tables[(int64_t)table_row(p, from.u) * p.table_stride + from.block + lane];
    return win;
  };
  auto advance = [&](Place& pl, int cnt) {
    pl.block += cnt;
    if (pl.block == pl.blocks) next_pair(p, pl, qt, per_group, line);
  };
  auto scales_of = [&](Window& win) {
    const bool in_pool = win.id >= 0 && win.id < p.num_blocks;
    if (lane < win.cnt && !in_pool) raise_status(p.status, B2_DEV_RANGE);
    if (!in_pool) win.id = -1;
    const int64_t at = in_pool ? q8_scale(win.id, p.nkv, win.g) : 0;
    win.ks = p.k_scale[at];
    win.vs = p.v_scale[at];
  };

  // The copies of a step's tiles: every lane 16-byte pieces of K and of V, 512 bytes of the run
  // with each; one commit group per step.  (TMA tile loads cost the warp 500 cycles a step to issue.)
  int n_open = 0;                // tiles in the ring or on their way
  int at_slot = 0, to_slot = 0;  // next to consume, next to ask for
  constexpr int PIECES = HD / 32;
  uint32_t to_off[PIECES];
#pragma unroll
  for (int c = 0; c < PIECES; ++c) to_off[c] = tile_at<HD>((lane + 32 * c) / (HD / 16), lane % (HD / 16));
  auto issue = [&](const Window& win, int i) {
    const uint32_t dst = ring_at + to_slot * (2 * C::TILE);
    to_slot = to_slot == STAGES - 1 ? 0 : to_slot + 1;
    const int id = __shfl_sync(0xffffffffu, win.id, i);
    ++n_open;
    if (id >= 0 && id < p.num_blocks) {  // else the step is left out
      const int64_t at = ((int64_t)id * p.nkv + win.g) * C::TILE + lane * 16;
      const uint8_t *ks = p.k_cache + at, *vs = p.v_cache + at;
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        cp_async16(dst + to_off[c], ks + c * 512);
        cp_async16(dst + C::TILE + to_off[c], vs + c * 512);
      }
    }
    cp_async_commit();
  };

  // q of a tile's columns.  Where they are few, the raw loads are made ahead, so that their latency
  // hides behind the ids'; more would not fit the registers.
  using Raw = typename Raw4<T>::Type;
  constexpr bool EARLY = NT * TERMS == 1;
  const uint32_t inv_rep = (65536u + rep - 1) / rep;  // c / rep = c * inv_rep >> 16 for c < 32, rep <= 16
  Raw raw[KW];
  auto load_q = [&](const Place& at, int nt) {
    const int tok0 = at.j * qt, ncol = min(qt, at.unit.len - tok0) * rep;
    const int col = nt * 8 + r8, tok = (int)(col * inv_rep >> 16);
    const bool live = col < ncol;
    const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(at.unit.start + tok0 + (live ? tok : 0)) * p.ld_q +
                   (int64_t)(at.g * rep + (live ? col - tok * rep : 0)) * HD + t4 * (HD / 4);
#pragma unroll
    for (int k = 0; k < KW; ++k) raw[k] = reinterpret_cast<const Raw*>(src)[k];
  };

  Place at{};
  if (left > 0) at = find_step(p, x_begin, qt, n_units, per_group, line);
  Window cur = take(at), nxt = cur;
  if (EARLY && cur.cnt > 0) load_q(at, 0);
  nxt.cnt = 0;
  if (left > 0) {
    Place to = at;
    advance(to, cur.cnt);
    nxt = take(to);
  }
  int sent = 0, sent_nxt = 0;  // steps of either window whose tiles were asked for
  auto top_up = [&]() {
    while (n_open < STAGES) {
      if (sent < cur.cnt) issue(cur, sent++);
      else if (sent_nxt < nxt.cnt) issue(nxt, sent_nxt++);
      else break;
    }
  };
  top_up();
  if (cur.cnt > 0) scales_of(cur);

  float colscale[NT][2], bias[NT][2];
  int lim[NT][2];  // last key of the lane's columns
  float o[2 * VW][NT][4];
  float m[NT][2], m2[NT][2], lift[NT][2], l[NT][2];  // references, 2^(m - m2), sums
  int i0 = 0;          // first block of the current (tile, kv head) that this warp sees
  bool start = true;   // a (tile, kv head) begins with this window
  bool first = true;   // nothing has been written out yet
  bool open = false;   // the last tile went to the workspace in part
  bool single = false;  // ... and it was the first

  while (cur.cnt > 0) {
    const int tok0 = at.j * qt, ntok = min(qt, at.unit.len - tok0);
    const int ncol = ntok * rep;
    const int pos0 = at.unit.ctx0 + tok0;  // position of the tile's first token
    const int pos_last = pos0 + ntok - 1;
    if (start) {
      start = false;
      i0 = at.block;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (!EARLY) load_q(at, nt);
        const bool live = nt * 8 + r8 < ncol;
        float big = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          float v[4];
          widen4(raw[k], v);
#pragma unroll
          for (int e = 0; e < 4; ++e) big = fmaxf(big, fabsf(v[e]));
        }
        if (!live) big = 0.f;
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^ex brings `big` to [2^14, 2^15) (below it, if `big` is not a normal number); in two factors,
        // so that neither overflows.  Infinite and NaN heads are left as they are.
        const int field = (int)(__float_as_uint(big) >> 23);
        const int ex = field == 0 || field == 255 ? (field ? 0 : 140) : 141 - field, ex2nd = ex / 2;
        const float up = __uint_as_float((uint32_t)(127 + ex2nd) << 23);
        const float up2 = __uint_as_float((uint32_t)(127 + ex - ex2nd) << 23);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          float v[4];
          widen4(raw[k], v);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = live ? v[e] * up * up2 : 0.f;
#pragma unroll
          for (int term = 0; term < TERMS; ++term) {
            uint2 f;
            f.x = pack_f16(v[0], v[1]);
            f.y = pack_f16(v[2], v[3]);
            if (C::BIASED) {  // of what the products will see
              const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f.x));
              const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&f.y));
              sum += (a.x + a.y) + (b.x + b.y);
            }
            sq[((k * NT + nt) * TERMS + term) * 32] = f;
            if (TERMS == 2) {
              const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f.x));
              const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&f.y));
              v[0] -= a.x; v[1] -= a.y; v[2] -= b.x; v[3] -= b.y;
            }
          }
        }
        const float back = live ? p.scale_log2 * __uint_as_float((uint32_t)(127 - ex2nd) << 23) *
                                      __uint_as_float((uint32_t)(127 - ex + ex2nd) << 23) *
                                      (C::BIASED ? 0x1p24f : 1.f)
                                : 0.f;
        if (C::BIASED) {
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = nt * 8 + 2 * t4 + e;
          colscale[nt][e] = __shfl_sync(0xffffffffu, back, (2 * t4 + e) * 4);
          if (C::BIASED) bias[nt][e] = __shfl_sync(0xffffffffu, sum, (2 * t4 + e) * 4) * (-128.f * 0x1p-24f);
          lim[nt][e] = c < ncol ? pos0 + (int)(c * inv_rep >> 16) : -1;
          m[nt][e] = m2[nt][e] = kNoRef;
          lift[nt][e] = l[nt][e] = 0.f;
        }
#pragma unroll
        for (int d = 0; d < 2 * VW; ++d) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
      }
      asm volatile("" ::: "memory");  // the fragments are read back by lds8
    }
    const int tail_from = (pos0 + 1) / kQ8Block - at.block;  // steps whose keys some column does not see

    for (int i = 0; i < cur.cnt; ++i) {
      if (i == 0 && nxt.cnt > 0) scales_of(nxt);  // its ids were asked for a window ago
      const uint32_t tile = ring_at + at_slot * (2 * C::TILE);
      const bool live = __shfl_sync(0xffffffffu, cur.id, i) >= 0;  // a block outside the pool is passed over
      const float ks = __shfl_sync(0xffffffffu, cur.ks, i), vs = __shfl_sync(0xffffffffu, cur.vs, i);
      const int key0 = (at.block + i) * kQ8Block;
      const bool tail = i >= tail_from;
      at_slot = at_slot == STAGES - 1 ? 0 : at_slot + 1;
      --n_open;  // as many groups were committed behind this step's
      static_assert(STAGES == 3, "the waits below");
      if (n_open >= 2) cp_async_wait<2>();
      else if (n_open == 1) cp_async_wait<1>();
      else cp_async_wait<0>();
      __syncwarp();
      if (!live) {
        top_up();
        continue;
      }
      float s[NT][4], s_odd[NT][4];  // two chains of products where columns are few
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = s_odd[nt][e] = 0.f;
      uint32_t kw[2][KW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows eight apart have the same swizzle
        if constexpr (KW == 2) {
          const uint2 v = lds8(tile + k_off[0] + h * 8 * HD);
          kw[h][0] = v.x; kw[h][1] = v.y;
        } else {
#pragma unroll
          for (int k = 0; k < KW; k += 4) {
            const uint4 v = lds16(tile + k_off[k / 4] + h * 8 * HD);
            kw[h][k] = v.x; kw[h][k + 1] = v.y; kw[h][k + 2] = v.z; kw[h][k + 3] = v.w;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        uint2 qf[NT][TERMS];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int term = 0; term < TERMS; ++term) qf[nt][term] = lds8(sq_at + ((k * NT + nt) * TERMS + term) * 32 * 8);
        uint32_t a[4];
        expand<CODE, C::BIASED>(kw[0][k], a[0], a[2]);
        expand<CODE, C::BIASED>(kw[1][k], a[1], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int term = 0; term < TERMS; ++term)
            mma_f16(NT == 1 && (k & 1) ? s_odd[nt] : s[nt], a, qf[nt][term].x, qf[nt][term].y);
      }
      if constexpr (NT == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] += s_odd[0][e];
      }
      const float lv = vs == 0.f ? -INFINITY : __log2f(vs);  // only places a reference: approximate
      // scores; the tail of the tile's keys is masked per column, after the scaling: a factor that is 0
      // (a tile of zeros, a head next to zeros), negative or NaN would not leave a masked score at -inf
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float cs = colscale[nt][e] * ks, c0 = C::BIASED ? bias[nt][e] * cs : 0.f;
          s[nt][e] = fmaf(s[nt][e], cs, c0);
          s[nt][2 + e] = fmaf(s[nt][2 + e], cs, c0);
        }
      if (tail) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (key0 + r8 > lim[nt][e]) s[nt][e] = -INFINITY;
            if (key0 + r8 + 8 > lim[nt][e]) s[nt][2 + e] = -INFINITY;
          }
      }
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          move |= fmaxf(s[nt][e], s[nt][2 + e]) > fminf(m[nt][e], m2[nt][e] - lv) + kRoom;
      if (__any_sync(0xffffffffu, move)) {  // references move, to 2^8 below their columns' largest
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
            const float mn = fmaxf(m[nt][e], mx - kLift);
            float m2n = fmaxf(m2[nt][e], mx - kLift + lv);
            if (m2n != kNoRef) m2n = fmaxf(m2n, mn - kGap);
            l[nt][e] *= ex2(m[nt][e] - mn);
            const float c = ex2(m2[nt][e] - m2n);
            m[nt][e] = mn;
            m2[nt][e] = m2n;
            lift[nt][e] = m2n == kNoRef ? 0.f : ex2(mn - m2n);
#pragma unroll
            for (int d = 0; d < 2 * VW; ++d) {
              o[d][nt][e] *= c;
              o[d][nt][2 + e] *= c;
            }
          }
      }
      uint32_t pb[NT][TERMS][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float pa[2], pc[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          pa[e] = ex2(s[nt][e] - m[nt][e]);  // -inf gives 0
          pc[e] = ex2(s[nt][2 + e] - m[nt][e]);
          l[nt][e] += pa[e] + pc[e];
          // a column that sees none of the block's keys takes nothing from its scale.  Where the product would
          // overflow, the exponentials it meets are 2^-112 or less: keys of less than 2^-120 of the softmax.
          const float f = vs == 0.f || (tail && key0 > lim[nt][e]) ? 0.f : q8_finite(vs * lift[nt][e]);
          pa[e] *= f;
          pc[e] *= f;
        }
#pragma unroll
        for (int term = 0; term < TERMS; ++term) {
          const uint32_t lo = pack_f16(pa[0], pa[1]), hi = pack_f16(pc[0], pc[1]);
          pb[nt][term][0] = transpose8x8(lo);
          pb[nt][term][1] = transpose8x8(hi);
          if (TERMS == 2) {
            const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&lo));
            const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            pa[0] -= fa.x; pa[1] -= fa.y; pc[0] -= fb.x; pc[1] -= fb.y;
          }
        }
      }
      {
        uint32_t vw[4][VW];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t a = tile + v_off[h & 1] + (h >> 1) * 8 * HD;
          if constexpr (VW == 4) {
            const uint4 v = lds16(a);
            vw[h][0] = v.x; vw[h][1] = v.y; vw[h][2] = v.z; vw[h][3] = v.w;
          } else if constexpr (VW == 2) {
            const uint2 v = lds8(a);
            vw[h][0] = v.x; vw[h][1] = v.y;
          } else {
            vw[h][0] = lds4(a);
          }
        }
        // V of keys no column sees counts as 0, whatever its codes (an e4m3 NaN among them)
        if (tail && key0 + kQ8Block - 1 > pos_last) {
          const int k0 = key0 + 2 * t4;
#pragma unroll
          for (int h = 0; h < 4; ++h)
            if (k0 + (h & 1) + (h >> 1) * 8 > pos_last) {
#pragma unroll
              for (int v = 0; v < VW; ++v) vw[h][v] = 0u;
            }
        }
#pragma unroll
        for (int v = 0; v < VW; ++v) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            uint32_t a[4];
            expand<CODE>(prmt(vw[0][v], vw[1][v], sel), a[0], a[1]);
            expand<CODE>(prmt(vw[2][v], vw[3][v], sel), a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int term = 0; term < TERMS; ++term)
                mma_f16(o[2 * v + half][nt], a, pb[nt][term][0], pb[nt][term][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the tiles: their slots may be asked for again
      top_up();
    }
    const bool done = at.block + cur.cnt == at.blocks;
    Place to = at;  // where the next window begins
    if (nxt.cnt > 0) advance(to, cur.cnt);
    if (done || nxt.cnt == 0) {
      // The lane holds, of columns 2 t4 and 2 t4 + 1 of every n-tile, dims r8 * HD/8 .. + HD/8 - 1.
      if (EARLY && nxt.cnt > 0) load_q(to, 0);  // (done: the next window begins another tile or head)
      const bool whole = i0 == 0 && done;
      const int64_t slot = 2 * (int64_t)w + (first ? 0 : 1);
      if (first && i0 > 0 && warp == 0 && lane == 0) p.ws_piece[blockIdx.x].x = (int)slot;
      open = !whole && nxt.cnt == 0;
      single = first;
      const int npad = p.compat_pad ? max(0, cut.max_ctx - (pos0 + 1)) : 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float lt = l[nt][e];
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, sh);
          const int c = nt * 8 + 2 * t4 + e;
          if (c >= ncol) continue;
          float f = 1.f;
          if (whole) {
            if (npad > 0) lt += (float)npad * exp2f(-m[nt][e]);  // keys of score 0 and value 0
            f = m2[nt][e] == kNoRef ? (lt == lt ? 0.f : lt) : exp2f(m2[nt][e] - m[nt][e]) / lt;
          }
          float v[4 * VW];
#pragma unroll
          for (int d = 0; d < 2 * VW; ++d) {
            v[2 * d] = o[d][nt][e] * f;
            v[2 * d + 1] = o[d][nt][2 + e] * f;
          }
          if (whole) {
            const int tok = (int)(c * inv_rep >> 16);
            T* dst = reinterpret_cast<T*>(p.out) + (int64_t)(at.unit.start + tok0 + tok) * p.ld_out +
                     (int64_t)(at.g * rep + c - tok * rep) * HD + r8 * (4 * VW);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
              for (int d = 0; d < VW; ++d)
                reinterpret_cast<float4*>(dst)[d] = make_float4(v[4 * d], v[4 * d + 1], v[4 * d + 2], v[4 * d + 3]);
            } else {
#pragma unroll
              for (int d = 0; d < VW; ++d) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(v[4 * d], v[4 * d + 1]);
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[4 * d + 2], v[4 * d + 3]);
                reinterpret_cast<uint2*>(dst)[d] =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
              }
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(p.ws_o + (slot * N + c) * HD + r8 * (4 * VW));
#pragma unroll
            for (int d = 0; d < VW; ++d) dst[d] = make_float4(v[4 * d], v[4 * d + 1], v[4 * d + 2], v[4 * d + 3]);
            if (r8 == 0) p.ws_stat[slot * N + c] = make_float4(m[nt][e], lt, m2[nt][e], 0.f);
          }
        }
      first = false;
      start = true;
    }
    if (nxt.cnt == 0) break;  // `at` stays the last tile's
    at = to;
    cur = nxt;
    sent = sent_nxt;
    sent_nxt = 0;
    nxt.cnt = 0;
    if (left > 0) {
      advance(to, cur.cnt);
      nxt = take(to);
    }
    top_up();
  }

  // Pieces of one (tile, kv head) within the CTA are joined here: into the output, or, where other
  // CTAs have some too, into the slot of the first.  Every warp whose last tile stays open and
  // that is the first of the CTA to have a piece of it says so; then the warps share the columns.
  if (threadIdx.x == 0) n_joins = 0;
  __syncthreads();
  if (open && (i0 == 0 || warp == 0)) {
    const int slot = 2 * w + (single ? 0 : 1);
    const int last_w = w + (at.begin + at.blocks - 1) / (int)cut.chunk, cta_last = blockIdx.x * WARPS + WARPS - 1;
    const bool whole = i0 == 0 && last_w <= cta_last;
    if (lane == 0) {
      if (!whole && i0 == 0) {
        p.ws_open[blockIdx.x] = make_int4(last_w / WARPS, at.u, at.j, at.g);
        p.ws_piece[blockIdx.x].y = slot;
      } else if (!whole) {
        p.ws_piece[blockIdx.x].x = slot;
      }
      const int pieces = min(last_w, cta_last) - w + 1, tok0 = at.j * qt;
      if (pieces > 1)
        joins[atomicAdd(&n_joins, 1)] =
            Join{w, slot, pieces, whole, at.unit.start + tok0, at.g, min(qt, at.unit.len - tok0) * rep,
                 p.compat_pad ? max(0, cut.max_ctx - (at.unit.ctx0 + tok0 + 1)) : 0};
    }
  }
  __syncthreads();
  int before = 0;
  for (int k = 0; k < n_joins; ++k) {
    const Join jn = joins[k];
    // columns are dealt to the warps in turn
    for (int c = (warp + WARPS - before % WARPS) % WARPS; c < jn.ncol; c += WARPS) {
      const auto slot_of = [&](int q) { return q == 0 ? jn.slot : 2 * (jn.warp + q); };
      const Piece<HD> r = join_pieces<HD>(p, slot_of, jn.pieces, N, c, 0, 1, lane);
      if (jn.whole) {
        const int tok = (int)(c * inv_rep >> 16);
        write_head<T, HD>(p, jn.row + tok, jn.g * rep + c - tok * rep, lane, r, jn.npad);
      } else {  // every lane has read what it replaces
        const int64_t to = (int64_t)jn.slot * N + c;
        if (lane == 0) p.ws_stat[to] = make_float4(r.m, r.l, r.m2, 0.f);
        float* dst = p.ws_o + to * HD + lane * (HD / 32);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) dst[e] = r.o[e];
      }
    }
    before += jn.ncol;
  }
}

// Joins the pieces of the tiles that reach over several CTAs: block x takes the one that begins in
// CTA x of the kernel above, its columns z, z + gridDim.z, ...; the warps share columns and pieces.
constexpr int kJoinWarps = 8;

template <typename T, int HD>
__global__ void __launch_bounds__(kJoinWarps * 32) q8_join_kernel(Q8AttnParams p, int qt, int columns) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = HD / 32;
  __shared__ float part[kJoinWarps][HD];
  __shared__ int most[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = blockIdx.x;
  const int4 open = p.ws_open[cta];
  if (open.x < 0) return;
  const int rep = p.nq / p.nkv, n = open.x - cta + 1;
  const Unit u = unit_of(p, open.y);
  const int tok0 = open.z * qt, ncol = min(qt, u.len - tok0) * rep;
  int npad = 0;
  if (p.compat_pad) {
    int mx = 0;
    for (int i = threadIdx.x; i < p.n_rows; i += kJoinWarps * 32) mx = max(mx, p.ctx_lens[i]);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) most[warp] = mx;
    __syncthreads();
    for (int i = 0; i < kJoinWarps; ++i) mx = max(mx, most[i]);
    npad = max(0, mx - (u.ctx0 + 1));
  }
  const int here = (ncol - (int)blockIdx.z + (int)gridDim.z - 1) / (int)gridDim.z;  // columns of this block
  int share = 1;                                                                    // warps per column
  while (share * 2 * here <= kJoinWarps && share < n) share *= 2;
  const auto slot_of = [&](int q) { return q == 0 ? p.ws_piece[cta].y : p.ws_piece[cta + q].x; };
  for (int i0 = 0; i0 < here; i0 += kJoinWarps / share) {
    const int i = i0 + warp / share, c = blockIdx.z + i * gridDim.z, part_of = warp % share;
    const bool live = i < here;
    Piece<HD> r;
    if (live) r = join_pieces<HD>(p, slot_of, n, columns, c, part_of, share, lane);
    if (share > 1) {
      __syncthreads();
      if (live)
#pragma unroll
        for (int e = 0; e < E; ++e) part[warp][lane * E + e] = r.o[e];
      __syncthreads();
      if (live && part_of == 0)
        for (int w = 1; w < share; ++w)
#pragma unroll
          for (int e = 0; e < E; ++e) r.o[e] += part[warp + w][lane * E + e];
    }
    if (live && part_of == 0) write_head<T, HD>(p, u.start + tok0 + c / rep, open.w * rep + c % rep, lane, r, npad);
  }
}

int check_q8_attention(const char* name, const Q8AttnParams& p, int hd, int cache_dtype, int layer, int bs, int dtype) {
  B2_CHECK_ARG(p.n_rows >= 0 && p.nq > 0 && p.nkv > 0 && p.nq % p.nkv == 0, "%s: bad head counts", name);
  B2_CHECK_ARG(valid_dtype(dtype), "%s: bad dtype", name);
  B2_CHECK_ARG(valid_q8_dtype(cache_dtype), "%s: bad cache dtype", name);
  B2_CHECK_ARG(p.num_blocks > 0 && p.table_stride > 0 && p.table_rows > 0 && layer >= 0, "%s: bad cache geometry",
               name);
  B2_CHECK_ARG(p.table_stride <= 0x7fffffff / kQ8Block, "%s: table_stride %d too large", name, p.table_stride);
  if (bs != kQ8Block) return fail(B2_ENOTSUP, "%s: block_size %d (16 only)", name, bs);
  if (hd != 32 && hd != 64 && hd != 128)
    return fail(B2_ENOTSUP, "%s: head_dim %d not supported (32, 64, 128)", name, hd);
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


// ------------------------------------------------------------------ host side
// Which prefills run on tcgen05 (prefill_q8_tc.cu).  Its items are two tiles of 128 columns of a sequence and
// head, one per SM at a time, 22 ns per key; this file's kernel cuts all tiles of 32 columns evenly over
// the SMs, 13 ns per key and tile of an SM.  Both are proportional to the context, which only the
// device knows, so the rule compares tiles with rounds of items.  Both sides measured (us, here / tcgen05):
//   heads 32/8, 1 sequence, 32 000 keys:    64 tokens  210 / 722,  128  375 / 723,  256  746 / 726
//   heads 32/8, 8 sequences, 4 000 keys:    16 tokens   86 /  94,   32  137 /  76,  256  796 / 203
//   heads  8/8, 64 sequences, 1 000 keys:   16 tokens   58 / 107,   64  165 / 110,  256  507 / 139
//   heads  8/1, 64 sequences, 1 000 keys:    8 tokens   45 /  29,   16   65 /  26,   64  153 /  35
bool tensor_prefill(int n_rows, int n_seqs, int nq, int nkv, int hd, float scale, int dtype) {
  const int rep = nq / nkv;
  if (dtype != B2_BF16 || hd != 128 || !prefill_q8_tc_serves(rep) || !(scale > 0.f)) return false;
  const int64_t tokens = ((int64_t)n_rows + n_seqs - 1) / n_seqs, narrow = 32 / rep, wide = 2 * (128 / rep);
  const int64_t tiles = (tokens + narrow - 1) / narrow * n_seqs * nkv;
  const int64_t items = (tokens + wide - 1) / wide * n_seqs * nkv;
  const int64_t sms = sm_count(), rounds = (items + sms - 1) / sms;
  return 3 * tiles >= 4 * sms * rounds;
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct AttnPlan {
  int nt, qt, units, per_group, ctas, slots;
  size_t piece, stat, o, total;  // workspace offsets
};

// Columns of a tile.  A decode row has rep columns.  A sequence of a prefill has tokens * rep;
// wide tiles read the cache once for more of them, narrow ones keep more warps resident and
// waste fewer columns of the products, so the width follows the mean length (48 drafts of 5 tokens, 4 heads
// to a kv head: 96 us in 24 columns, 129 in 32).
AttnPlan plan_of(int n_rows, int nq, int nkv, int hd, int n_seqs, bool prefill, int dtype) {
  AttnPlan a{};
  const int rep = nq / nkv, terms = dtype == B2_F32 ? 2 : 1;
  const int64_t columns = prefill ? (int64_t)((n_rows + n_seqs - 1) / n_seqs) * rep : rep;
  a.nt = columns <= 8 && rep <= 8 ? 1 : columns <= 16 || terms == 2 ? 2 : columns <= 24 ? 3 : 4;
  a.qt = prefill ? 8 * a.nt / rep : 1;
  a.units = prefill ? n_seqs : n_rows;
  a.per_group = (a.units + kGroups - 1) / kGroups;
  a.ctas = sm_count();
  a.slots = 2 * a.ctas * warps_of(hd, a.nt, terms);
  a.piece = align256((size_t)a.ctas * sizeof(int4));
  a.stat = a.piece + align256((size_t)a.ctas * sizeof(int2));
  a.o = a.stat + align256((size_t)a.slots * 8 * a.nt * sizeof(float4));
  a.total = a.o + (size_t)a.slots * 8 * a.nt * hd * sizeof(float);
  return a;
}

// Opts a kernel into `bytes` of dynamic shared memory once per (kernel, device).
int allow_smem(const void* fn, size_t bytes) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int dev = 0;
  B2_TRY_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({fn, dev})) return B2_OK;
  B2_TRY_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  done.insert({fn, dev});
  return B2_OK;
}

template <typename T, int HD, int CODE, int NT>
int launch_tiles(const Q8AttnParams& p, const AttnPlan& a, cudaStream_t s) {
  using C = AttnCfg<T, HD, CODE, NT>;
  const int rc = allow_smem((const void*)q8_attn_kernel<T, HD, CODE, NT>, C::SMEM);
  if (rc) return rc;
  B2_TRY_CUDA(launch_pdl((q8_attn_kernel<T, HD, CODE, NT>), dim3(a.ctas), dim3(C::WARPS * 32), C::SMEM, s, p, a.qt,
                         a.units, a.per_group));
  B2_TRY_CUDA(launch_pdl((q8_join_kernel<T, HD>), dim3(a.ctas, 1, std::min(4, a.qt * (p.nq / p.nkv))),
                         dim3(kJoinWarps * 32), 0, s, p, a.qt, 8 * a.nt));
  return B2_OK;
}

template <typename T, int HD, int CODE>
int launch_nt(const Q8AttnParams& p, const AttnPlan& a, cudaStream_t s) {
  if (a.nt == 1) return launch_tiles<T, HD, CODE, 1>(p, a, s);
  if (a.nt == 2) return launch_tiles<T, HD, CODE, 2>(p, a, s);
  if constexpr (sizeof(T) == 2)
    return a.nt == 3 ? launch_tiles<T, HD, CODE, 3>(p, a, s) : launch_tiles<T, HD, CODE, 4>(p, a, s);
  return fail(B2_ENOTSUP, "attention over the 8-bit cache: no tile of %d columns", 8 * a.nt);
}

template <typename T>
int launch_hd(const Q8AttnParams& p, int hd, int code, const AttnPlan& a, cudaStream_t s) {
  if (code == B2_I8) {
    if (hd == 32) return launch_nt<T, 32, B2_I8>(p, a, s);
    if (hd == 64) return launch_nt<T, 64, B2_I8>(p, a, s);
    return launch_nt<T, 128, B2_I8>(p, a, s);
  }
  if (hd == 32) return launch_nt<T, 32, B2_E4M3>(p, a, s);
  if (hd == 64) return launch_nt<T, 64, B2_E4M3>(p, a, s);
  return launch_nt<T, 128, B2_E4M3>(p, a, s);
}

int launch(const char* name, Q8AttnParams& p, int hd, int cache_dtype, int dtype, void* workspace, size_t bytes,
           cudaStream_t s) {
  const AttnPlan a = plan_of(p.n_rows, p.nq, p.nkv, hd, p.n_seqs, p.seq_start != nullptr, dtype);
  B2_CHECK_ARG(workspace && bytes >= a.total, "%s: workspace of %zu bytes needed, %zu given", name, a.total, bytes);
  B2_CHECK_ARG(((uintptr_t)workspace % 16) == 0, "%s: the workspace must be 16-byte aligned", name);
  char* ws = static_cast<char*>(workspace);
  p.ws_open = reinterpret_cast<int4*>(ws);
  p.ws_piece = reinterpret_cast<int2*>(ws + a.piece);
  p.ws_stat = reinterpret_cast<float4*>(ws + a.stat);
  p.ws_o = reinterpret_cast<float*>(ws + a.o);
  return dtype == B2_BF16 ? launch_hd<__nv_bfloat16>(p, hd, cache_dtype, a, s)
                          : launch_hd<float>(p, hd, cache_dtype, a, s);
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

size_t b2_paged_attention_q8_workspace_bytes(int n_rows, int nq, int nkv, int head_dim, int dtype) {
  if (n_rows <= 0 || nkv <= 0 || nq < nkv || nq / nkv > 16 || head_dim <= 0) return 0;
  return b2::plan_of(n_rows, nq, nkv, head_dim, 0, false, dtype).total;
}

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
                 nullptr, 0, scale * 1.4426950408889634f, out, ld_out, status, nullptr, nullptr, nullptr, nullptr};
  int rc = check_q8_attention(name, p, head_dim, cache_dtype, layer, block_size, dtype);
  if (rc || n_rows == 0) return rc;
  rc = check_q8_pointers(name, p, dtype);
  if (rc) return rc;
  B2_CHECK_ARG(ctx_lens, "%s: null pointer", name);
  B2_CHECK_ARG(table_index || n_rows <= table_rows, "%s: %d rows for %d table rows", name, n_rows, table_rows);
  set_cache(p, k_cache, v_cache, k_scale, v_scale, layer, head_dim);
  return launch(name, p, head_dim, cache_dtype, dtype, workspace, workspace_bytes, stream);
}

size_t b2_prefill_attention_q8_workspace_bytes(int n_rows, int nq, int nkv, int head_dim, int n_seqs, int dtype) {
  if (n_rows <= 0 || n_seqs <= 0 || nkv <= 0 || nq < nkv || nq / nkv > 16 || head_dim <= 0) return 0;
  return b2::plan_of(n_rows, nq, nkv, head_dim, n_seqs, true, dtype).total;
}

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
                 scale * 1.4426950408889634f, out, ld_out, status, nullptr, nullptr, nullptr, nullptr};
  int rc = check_q8_attention(name, p, head_dim, cache_dtype, layer, block_size, dtype);
  if (rc) return rc;
  B2_CHECK_ARG(n_seqs >= 0, "%s: bad sizes", name);
  if (n_rows == 0 || n_seqs == 0) return B2_OK;
  rc = check_q8_pointers(name, p, dtype);
  if (rc) return rc;
  B2_CHECK_ARG(seq_start, "%s: null pointer", name);
  B2_CHECK_ARG(n_seqs <= table_rows, "%s: %d sequences for %d table rows", name, n_seqs, table_rows);
  set_cache(p, k_cache, v_cache, k_scale, v_scale, layer, head_dim);
  if (tensor_prefill(n_rows, n_seqs, nq, nkv, head_dim, scale, dtype))
    return prefill_attention_q8_tc(q, ld_q, n_rows, nq, nkv, p.k_cache, p.v_cache, p.k_scale, p.v_scale, cache_dtype,
                                   num_blocks, block_tables, table_stride, seq_start, seq_ctx0, n_seqs, scale, out,
                                   ld_out, status, stream);
  return launch(name, p, head_dim, cache_dtype, dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
