// Per-head RMS norm of q and k, rotary embedding and the paged KV write in one pass, into a
// cache of the model's type or of 8 bits; and the read-back of 8-bit tiles.
//
// The rotation and the slots are those of engine/model/attention.py:46-63 and :166-184; the
// reference has neither the norms nor an 8-bit cache.  For each token and q or k head x
//   y = x * rsqrt(mean(x^2) + eps) * weight   (no norm where the weight pointer is null)
//   out[d] = y[d] cos[d] - y[d + h] sin[d],  out[d + h] = y[d + h] cos[d + h] + y[d] sin[d + h],
// h = head_dim / 2, all in float32 and rounded once when it is stored.  Values are stored as
// they are.
//
// Layout of the work: a group of head_dim / 16 lanes holds one token's head at a time, each lane 8
// elements of the lower half and the 8 they rotate with in the upper one, so a head is read
// and written in 16-byte pieces, the rotation stays within a lane and the mean takes
// log2(head_dim / 16) shuffles.
//
// Measured (heads 32/8 of 128, in a graph): bf16 cache, 16 384 tokens: 95 us, 404 MB at 4.3 TB/s (bound by
// the issue of instructions, 0.65 of the copy's rate); 8 tokens: 2.5 us.  int8 cache and the read-back of 128 blocks:
// 128 tokens 10.9 us, two launches and their chains of loads.  e4m3 cache, 7 947 ragged tokens of heads 32/4
// of 64, with the read-back: 32 us.
//
// 8-bit tiles.  The tokens of a call that fall into one block form a run; one warp per (run,
// head) holds the run's values in registers, takes their largest magnitude and writes codes
// and scale.  Where the run begins inside a block, the slots before it are history: the tile
// keeps its old scale if that is larger, else the old codes are rounded again under the new
// one (code * old / new, to nearest), which a tile's growing maximum makes ever rarer.
#include "q8.cuh"

#include <algorithm>

namespace b2 {
namespace {

struct NormRopeParams {
  const void* qkv;
  int64_t ld_qkv;
  int n_tokens, nq, nkv;
  const float* q_weight;
  const float* k_weight;
  float eps;
  const int64_t* rope_pos;
  const int64_t* store_pos;
  const int32_t* table_index;
  const int32_t* tables;
  int table_rows, table_stride, num_blocks, bs;
  const float* cos;
  const float* sin;
  int max_seq_len;
  void* q_out;
  void* k_cache;
  void* v_cache;
  float* k_scale;
  float* v_scale;
  int heads;        // heads a lane group takes of its token
  int chunk;        // tokens whose runs a tile block looks for, at most 16
  int tile_blocks;  // blocks that write tiles, before those of the q heads
  int32_t* status;
};

// 8 elements as float32.
__device__ __forceinline__ void ld8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void ld8(const __nv_bfloat16* p, float (&v)[8]) { load16_f32<__nv_bfloat16>(p, v); }
__device__ __forceinline__ void st8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void st8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 o;
  uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = o;
}

// Two products, sums or fused products at once.  (Not for the rotation: the assembler fuses a packed
// product with a packed sum in spite of their .rn.)
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ void ld8(const float* p, float2 (&v)[4]) { ld8(p, reinterpret_cast<float(&)[8]>(v)); }

// What a lane needs of the tables for one token: cos and sin of its 8 elements of either half, the
// low half's sin negated.
struct Angles {
  float2 cl[4], sl[4], ch[4], sh[4];
};
template <int HD>
__device__ __forceinline__ void load_angles(const NormRopeParams& p, int64_t rope, int li, Angles& a) {
  const float *c = p.cos + rope * HD + li * 8, *s = p.sin + rope * HD + li * 8;
  ld8(c, a.cl);
  ld8(s, a.sl);
  ld8(c + HD / 2, a.ch);
  ld8(s + HD / 2, a.sh);
#pragma unroll
  for (int e = 0; e < 4; ++e) a.sl[e] = make_float2(-a.sl[e].x, -a.sl[e].y);
}

// Norm (if `norm`) and rotation of a head that LANES lanes hold, LANES-wise in every group of the
// warp: all 32 lanes come here.
template <int LANES>
__device__ __forceinline__ void norm_rotate(float2 (&lo)[4], float2 (&hi)[4], bool norm, const float2 (&wl)[4],
                                            const float2 (&wh)[4], float eps, const Angles& a) {
  if (norm) {
    float2 s2 = mul2(lo[0], lo[0]), t2 = mul2(hi[0], hi[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) {
      s2 = fma2(lo[e], lo[e], s2);
      t2 = fma2(hi[e], hi[e], t2);
    }
    s2 = add2(s2, t2);
    float ss = s2.x + s2.y;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.f / (16 * LANES)) + eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = mul2(mul2(lo[e], make_float2(r, r)), wl[e]);
      hi[e] = mul2(mul2(hi[e], make_float2(r, r)), wh[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // two roundings a product, as the separate rotation kernel: without norms and in the
    // model's type the two give the same bits
    const float2 x = make_float2(__fadd_rn(__fmul_rn(lo[e].x, a.cl[e].x), __fmul_rn(hi[e].x, a.sl[e].x)),
                                 __fadd_rn(__fmul_rn(lo[e].y, a.cl[e].y), __fmul_rn(hi[e].y, a.sl[e].y)));
    const float2 y = make_float2(__fadd_rn(__fmul_rn(hi[e].x, a.ch[e].x), __fmul_rn(lo[e].x, a.sh[e].x)),
                                 __fadd_rn(__fmul_rn(hi[e].y, a.ch[e].y), __fmul_rn(lo[e].y, a.sh[e].y)));
    lo[e] = x;
    hi[e] = y;
  }
}

struct Place {
  bool rope_ok, slot_ok;
  int64_t rope;  // position in the tables
  int64_t block;
  int64_t pos;  // position in the cache
  int off;      // its slot within the block
};

__device__ __forceinline__ Place place_of(const NormRopeParams& p, int tok) {
  Place r;
  r.rope = p.rope_pos[tok];
  r.pos = p.store_pos ? p.store_pos[tok] : r.rope;
  const int row = p.table_index ? p.table_index[tok] : tok;
  r.rope_ok = r.rope >= 0 && r.rope < p.max_seq_len;
  r.block = -1;
  r.off = 0;
  if (r.pos >= 0 && r.pos < (int64_t)p.table_stride * p.bs && row >= 0 && row < p.table_rows) {
    const int64_t at = r.pos / p.bs;
    r.off = (int)(r.pos - at * p.bs);
    r.block = p.tables[(int64_t)row * p.table_stride + at];
  }
  r.slot_ok = r.block >= 0 && r.block < p.num_blocks;
  return r;
}

// Heads h0 .. h0 + p.heads - 1 of one token per lane group: q heads, and with KV the k and v heads of a
// cache of the model's type.  The groups of a warp take the same heads of successive tokens, so that
// a warp does not part at the q, k and v heads' borders.  The token's angles are read once for
// all its heads, and two heads are on their way while one is worked on.
template <typename T, int HD, bool KV>
__device__ __forceinline__ void rope_block(const NormRopeParams& p, int64_t block) {
  constexpr int LANES = HD / 16, GROUPS = 32 / LANES, HALF = HD / 2;
  const int li = threadIdx.x % LANES, grp = threadIdx.x % 32 / LANES;
  const int heads = KV ? p.nq + 2 * p.nkv : p.nq, chunks = (heads + p.heads - 1) / p.heads;
  const int64_t item = block * 4 + (threadIdx.x >> 5);
  const int64_t mine = item / chunks * GROUPS + grp;
  const bool live = mine < p.n_tokens;
  const int tok = live ? (int)mine : p.n_tokens - 1;
  const int h0 = (int)(item % chunks) * p.heads, h1 = min(heads, h0 + p.heads);
  const T* src = reinterpret_cast<const T*>(p.qkv) + (int64_t)tok * p.ld_qkv + li * 8;
  auto fetch = [&](int h, T (&r)[16]) {
    const T* at = src + (int64_t)min(h, h1 - 1) * HD;
#pragma unroll
    for (int i = 0; i < 8 * (int)sizeof(T) / 16; ++i) {
      reinterpret_cast<uint4*>(r)[i] = reinterpret_cast<const uint4*>(at)[i];
      reinterpret_cast<uint4*>(r + 8)[i] = reinterpret_cast<const uint4*>(at + HALF)[i];
    }
  };
  alignas(16) T first[16], second[16];  // the next two heads
  fetch(h0, first);
  fetch(h0 + 1, second);
  const Place at = place_of(p, tok);
  if (live && h0 == 0 && li == 0 && !(at.rope_ok && at.slot_ok)) raise_status(p.status, B2_DEV_RANGE);
  Angles a;
  load_angles<HD>(p, at.rope_ok ? at.rope : 0, li, a);
  T* q_out = reinterpret_cast<T*>(p.q_out) + (int64_t)tok * p.nq * HD + li * 8;
  const int64_t slot = ((at.block * p.bs + at.off) * p.nkv) * HD + li * 8;
  const bool keep_q = live && at.rope_ok, keep_kv = keep_q && at.slot_ok;
  const float* weight = nullptr;
  float2 wl[4], wh[4];
  auto work = [&](int h, T (&r)[16]) {
    if (KV && h >= p.nq + p.nkv) {
      if (keep_kv) {
        T* dst = reinterpret_cast<T*>(p.v_cache) + slot + (int64_t)(h - p.nq - p.nkv) * HD;
#pragma unroll
        for (int i = 0; i < 8 * (int)sizeof(T) / 16; ++i) {
          reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(r)[i];
          reinterpret_cast<uint4*>(dst + HALF)[i] = reinterpret_cast<const uint4*>(r + 8)[i];
        }
      }
      fetch(h + 2, r);
      return;
    }
    float2 lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = make_float2(to_f32(r[2 * e]), to_f32(r[2 * e + 1]));
      hi[e] = make_float2(to_f32(r[8 + 2 * e]), to_f32(r[9 + 2 * e]));
    }
    fetch(h + 2, r);
    const float* w = h < p.nq ? p.q_weight : p.k_weight;
    if (w && w != weight) {
      ld8(w + li * 8, wl);
      ld8(w + HALF + li * 8, wh);
      weight = w;
    }
    norm_rotate<LANES>(lo, hi, w != nullptr, wl, wh, p.eps, a);
    if (h < p.nq ? keep_q : keep_kv) {
      T* dst = h < p.nq ? q_out + (int64_t)h * HD : reinterpret_cast<T*>(p.k_cache) + slot + (int64_t)(h - p.nq) * HD;
      st8(dst, reinterpret_cast<float(&)[8]>(lo));
      st8(dst + HALF, reinterpret_cast<float(&)[8]>(hi));
    }
  };
  for (int h = h0; h < h1; h += 2) {
    work(h, first);
    if (h + 1 < h1) work(h + 1, second);
  }
}

// Five CTAs per SM for bf16 (bf16 16 384 tokens x 48 heads of 128: 95 us, 4.3 TB/s; as the compiler
// would have it 106), which float32 has no registers for.  Half as many elements per lane fill the SM
// with twice the warps and are slower (105): what bounds it is the issue of instructions, not the
// bytes under way.
template <typename T, int HD>
__global__ void __launch_bounds__(128, sizeof(T) == 2 ? 5 : 3) qk_norm_rope_kernel(NormRopeParams p) {
  pdl_wait();
  pdl_trigger();
  rope_block<T, HD, true>(p, blockIdx.x);
}

// Runs and tiles of the 8-bit cache: one warp per (k or v, head), for the runs that begin among
// p.chunk tokens.
template <typename T, int HD, int CODE>
__device__ __forceinline__ void tile_block(const NormRopeParams& p, int64_t block) {
  constexpr int LANES = HD / 16, G = 32 / LANES, ITERS = kQ8Block / G, HALF = HD / 2;
  const int lane = threadIdx.x & 31, li = lane % LANES, grp = lane / LANES;
  const int head_blocks = (2 * p.nkv + 3) / 4;
  const int head = (int)(block % head_blocks) * 4 + (threadIdx.x >> 5);  // k heads, then v heads
  if (head >= 2 * p.nkv) return;
  const bool is_k = head < p.nkv;
  const int g = is_k ? head : head - p.nkv;
  uint8_t* cache = reinterpret_cast<uint8_t*>(is_k ? p.k_cache : p.v_cache);
  float* scales = is_k ? p.k_scale : p.v_scale;
  // Lane i looks at token t0 + i: where it goes, and whether it goes on with the run of the token
  // before.  Sixteen tokens behind the chunk's belong to runs that begin in it.
  const int t0 = (int)(block / head_blocks) * p.chunk, mine = t0 + lane;
  const bool there = mine < p.n_tokens;
  const Place at = place_of(p, there ? mine : t0);
  const int row = p.table_index ? p.table_index[there ? mine : t0] : mine;
  const int off = (int)(at.pos & (kQ8Block - 1));
  int64_t pos_before = __shfl_up_sync(0xffffffffu, at.pos, 1);
  int row_before = __shfl_up_sync(0xffffffffu, row, 1);
  if (lane == 0 && t0 > 0) {
    pos_before = p.store_pos ? p.store_pos[t0 - 1] : p.rope_pos[t0 - 1];
    row_before = p.table_index ? p.table_index[t0 - 1] : t0 - 1;
  }
  const bool goes_on = mine > 0 && off > 0 && row_before == row && pos_before + 1 == at.pos;
  const unsigned on = __ballot_sync(0xffffffffu, there && goes_on);
  unsigned begins = __ballot_sync(0xffffffffu, there && lane < p.chunk && at.slot_ok && !goes_on);
  const unsigned good = __ballot_sync(0xffffffffu, there && at.rope_ok);
  const bool norm = is_k && p.k_weight != nullptr;
  float2 wl[4], wh[4];
  if (norm) {
    ld8(p.k_weight + li * 8, wl);
    ld8(p.k_weight + HALF + li * 8, wh);
  }
  for (; begins; begins &= begins - 1) {
    const int b = __ffs(begins) - 1, t = t0 + b;
    const int len = b == 31 ? 1 : __ffs(~(on >> (b + 1)));  // the run's tokens: 1 and those that go on
    if (!(good >> b & ((1u << len) - 1))) continue;  // none to be stored: the tile stays as it is
    const int first = __shfl_sync(0xffffffffu, off, b);
    const int64_t blk = __shfl_sync(0xffffffffu, at.block, b);
    float2 lo[ITERS][4], hi[ITERS][4];
    bool have[ITERS];
    int64_t rope[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      const int i = it * G + grp;
      have[it] = i < len;
      const T* src = reinterpret_cast<const T*>(p.qkv) + (int64_t)(t + (have[it] ? i : 0)) * p.ld_qkv +
                     (int64_t)(p.nq + head) * HD + li * 8;
      ld8(src, reinterpret_cast<float(&)[8]>(lo[it]));
      ld8(src + HALF, reinterpret_cast<float(&)[8]>(hi[it]));
      const int from = have[it] ? b + i : b;  // below 32: len ends with the lanes
      rope[it] = __shfl_sync(0xffffffffu, at.rope, from);
      // a token with a bad position is not stored (it is reported with its q heads)
      const bool rope_ok = __shfl_sync(0xffffffffu, (int)at.rope_ok, from);  // by every lane
      have[it] = have[it] && rope_ok;
      if (!have[it]) rope[it] = 0;
    }
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      if (is_k) {
        Angles a;
        load_angles<HD>(p, rope[it], li, a);
        norm_rotate<LANES>(lo[it], hi[it], norm, wl, wh, p.eps, a);
      }
      if (have[it]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = reinterpret_cast<const float(&)[8]>(lo[it])[e];
          const float y = reinterpret_cast<const float(&)[8]>(hi[it])[e];
          amax = fmaxf(amax, fmaxf(fabsf(x), fabsf(y)));
          bad |= !(fabsf(x) <= 3.402823466e38f) || !(fabsf(y) <= 3.402823466e38f);
        }
      }
    }
    amax = warp_max(amax);
    bad = __any_sync(0xffffffffu, bad);
    float scale = amax / Q8<CODE>::kTop;
    if (!(scale >= kQ8Tiny)) scale = 0.f;
    if (bad) scale = __int_as_float(0x7fffffff);
    const int64_t si = q8_scale(blk, p.nkv, g);
    uint8_t* tile = cache + q8_tile(blk, p.nkv, g, HD);
    if (first > 0) {
      const float old = scales[si];
      if (old >= scale || old != old) {
        scale = old;
      } else if (scale == scale) {  // the tile's maximum grew: round the history again
        const float ratio = old / scale;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
          const int slot = it * G + grp;
          if (slot < first) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint2* w = reinterpret_cast<uint2*>(tile + slot * HD + half * HALF + li * 8);
              uint2 c = *w;
              float v[4];
              Q8<CODE>::decode4(c.x, v);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] *= ratio;
              c.x = Q8<CODE>::encode4(v);
              Q8<CODE>::decode4(c.y, v);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] *= ratio;
              c.y = Q8<CODE>::encode4(v);
              *w = c;
            }
          }
        }
      }
      __syncwarp();  // every lane has read the old scale
    }
    const float inv = scale > 0.f ? 1.f / scale : 0.f;  // 0 for a tile of zeros and for NaN
    // A poisoned run's codes are 0: no NaN code is stored, since a product with it would also reach
    // rows that do not see its tile.
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      if (!have[it]) continue;
      const int slot = first + it * G + grp;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float(&y)[8] = reinterpret_cast<const float(&)[8]>(half ? hi[it] : lo[it]);
        float v[4];
        uint2 c;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = bad ? 0.f : y[e] * inv;
        c.x = Q8<CODE>::encode4(v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = bad ? 0.f : y[4 + e] * inv;
        c.y = Q8<CODE>::encode4(v);
        *reinterpret_cast<uint2*>(tile + slot * HD + half * HALF + li * 8) = c;
      }
    }
    if (lane == 0) scales[si] = scale;
    __syncwarp();  // a token given twice finds the tile as this run left it
  }
}

// Tiles and q heads in one launch: they have nothing to do with each other, and the tiles' chains of
// loads hide behind the q heads' traffic (bf16 ragged prefill of 7 947 tokens, heads 32/4 of 64: 32 us,
// in two launches 52; 3 CTAs per SM 38, 5 spill and take 36).
template <typename T, int HD, int CODE>
__global__ void __launch_bounds__(128, 4) qk_norm_rope_q8_kernel(NormRopeParams p) {
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x < p.tile_blocks) tile_block<T, HD, CODE>(p, blockIdx.x);
  else rope_block<T, HD, false>(p, blockIdx.x - p.tile_blocks);
}

// out[i, token, head, :] = code * scale of block ids[i], [n, 16, nkv, head_dim].
template <typename T, int CODE>
__global__ void __launch_bounds__(128) kv_read_q8_kernel(const uint8_t* k_cache, const uint8_t* v_cache,
                                                         const float* k_scale, const float* v_scale, int num_blocks,
                                                         int nkv, int hd, const int32_t* ids, int n, T* k_out,
                                                         T* v_out, int32_t* status) {
  pdl_wait();
  pdl_trigger();
  const int per = kQ8Block * nkv * hd / 8;  // 8-element pieces of one block
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)n * per) return;
  const int b = (int)(i / per), w = (int)(i % per);
  const int d = w % (hd / 8) * 8, slot = w / (hd / 8) % kQ8Block, g = w / (hd / 8) / kQ8Block;
  const int64_t blk = ids[b];
  const bool ok = blk >= 0 && blk < num_blocks;
  if (!ok && w == 0) raise_status(status, B2_DEV_RANGE);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (ok) {
      const uint8_t* tile = (kv ? v_cache : k_cache) + q8_tile(blk, nkv, g, hd);
      const uint2 c = *reinterpret_cast<const uint2*>(tile + slot * hd + d);
      const float s = (kv ? v_scale : k_scale)[q8_scale(blk, nkv, g)];
      float a[4];
      Q8<CODE>::decode4(c.x, a);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e] * s;
      Q8<CODE>::decode4(c.y, a);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 + e] = a[e] * s;
    }
    st8((kv ? v_out : k_out) + (((int64_t)b * kQ8Block + slot) * nkv + g) * hd + d, v);
  }
}

int check_norm_rope(const char* name, const NormRopeParams& p, int hd, int layer, int dtype) {
  B2_CHECK_ARG(p.n_tokens >= 0 && p.nq > 0 && p.nkv > 0, "%s: bad head counts", name);
  B2_CHECK_ARG(valid_dtype(dtype), "%s: bad dtype", name);
  if (hd != 32 && hd != 64 && hd != 128)
    return fail(B2_ENOTSUP, "%s: head_dim %d not supported (32, 64, 128)", name, hd);
  B2_CHECK_ARG(p.ld_qkv >= ((int64_t)p.nq + 2 * (int64_t)p.nkv) * hd, "%s: ld_qkv too small", name);
  B2_CHECK_ARG(p.num_blocks > 0 && p.bs > 0 && p.table_stride > 0 && p.table_rows > 0 && layer >= 0 &&
                   p.max_seq_len > 0, "%s: bad cache geometry", name);
  if (p.n_tokens == 0) return B2_OK;
  B2_CHECK_ARG(p.qkv && p.rope_pos && p.tables && p.cos && p.sin && p.q_out && p.k_cache && p.v_cache,
               "%s: null pointer", name);
  B2_CHECK_ARG(p.table_index || p.n_tokens <= p.table_rows, "%s: %d tokens for %d table rows", name, p.n_tokens,
               p.table_rows);
  const size_t esz = dtype_bytes(dtype);
  B2_CHECK_ARG(((uintptr_t)p.qkv % 16) == 0 && ((p.ld_qkv * esz) % 16) == 0 && ((uintptr_t)p.q_out % 16) == 0 &&
                   ((uintptr_t)p.k_cache % 16) == 0 && ((uintptr_t)p.v_cache % 16) == 0 &&
                   ((uintptr_t)p.cos % 16) == 0 && ((uintptr_t)p.sin % 16) == 0 &&
                   ((uintptr_t)p.q_weight % 16) == 0 && ((uintptr_t)p.k_weight % 16) == 0,
               "%s: buffers must be 16-byte aligned", name);
  return B2_OK;
}

// Heads per lane group.  More of them share one reading of the token's angles (16 384 tokens of 48
// heads, 4 CTAs per SM: 123 us with 2, 109 with 4, 106 with 8, 107 with 16); fewer keep 64 or more lane
// groups per SM when tokens are few.
int heads_per_group(int n_tokens, int heads) {
  int h = 1;
  while (h < 8 && (int64_t)n_tokens * heads / (2 * h) >= 64 * (int64_t)sm_count()) h *= 2;
  return h;
}

template <int HD>
int64_t rope_blocks(const NormRopeParams& p, int heads) {
  constexpr int GROUPS = 32 / (HD / 16);
  const int64_t warps = (int64_t)((p.n_tokens + GROUPS - 1) / GROUPS) * ((heads + p.heads - 1) / p.heads);
  return (warps + 3) / 4;
}

template <typename T, int HD>
int launch_rope(NormRopeParams& p, cudaStream_t s) {
  const int heads = p.nq + 2 * p.nkv;
  p.heads = heads_per_group(p.n_tokens, heads);
  const int64_t grid = rope_blocks<HD>(p, heads);
  B2_CHECK_ARG(grid <= 0x7fffffff, "qk_norm_rope: %d tokens are too many for one call", p.n_tokens);
  B2_TRY_CUDA(launch_pdl((qk_norm_rope_kernel<T, HD>), dim3((unsigned)grid), dim3(128), 0, s, p));
  return B2_OK;
}

template <typename T, int HD>
int launch_q8(NormRopeParams& p, int cache_dtype, cudaStream_t s) {
  p.heads = heads_per_group(p.n_tokens, p.nq);
  // A warp looks for the runs of `chunk` tokens with one load and works them off in turn, so a chunk should hold
  // about one run: the mean length of a table row's tokens, and more where there are chunks enough.  In us, heads
  // 32/8 of 128, in chunks of 1 / 4 / 16: 4 prompts of 64 tokens 7.2 / 6.3 / 7.1, of 512 28 / 16 / 13, of 2 048
  // 131 / 73 / 57; one token each for 256 rows 11 / 20 / 51, 1 024 rows 34 / 32 / 66, 4 096 rows 133 / 107 / 114
  // (8: 101).
  p.chunk = std::min(16, std::max({1, p.n_tokens / p.table_rows, std::min(8, p.n_tokens / 512)}));
  const int64_t tiles = (int64_t)((p.n_tokens + p.chunk - 1) / p.chunk) * ((2 * p.nkv + 3) / 4);
  const int64_t grid = tiles + rope_blocks<HD>(p, p.nq);
  B2_CHECK_ARG(grid <= 0x7fffffff, "qk_norm_rope: %d tokens are too many for one call", p.n_tokens);
  p.tile_blocks = (int)tiles;
  if (cache_dtype == B2_I8)
    B2_TRY_CUDA(launch_pdl((qk_norm_rope_q8_kernel<T, HD, B2_I8>), dim3((unsigned)grid), dim3(128), 0, s, p));
  else
    B2_TRY_CUDA(launch_pdl((qk_norm_rope_q8_kernel<T, HD, B2_E4M3>), dim3((unsigned)grid), dim3(128), 0, s, p));
  return B2_OK;
}

}  // namespace
}  // namespace b2

extern "C" {

int b2_qk_norm_rope_kv_write(const void* qkv, int64_t ld_qkv, int n_tokens, int nq, int nkv, int head_dim,
                             const float* q_weight, const float* k_weight, float eps, const int64_t* rope_pos,
                             const int64_t* store_pos, const int32_t* table_index, const int32_t* block_tables,
                             int table_rows, int table_stride, int num_blocks, int block_size, const float* cos,
                             const float* sin, int max_seq_len, void* q_out, void* k_cache, void* v_cache, int layer,
                             int dtype, int32_t* status, b2_stream_t stream) {
  using namespace b2;
  NormRopeParams p{qkv, ld_qkv, n_tokens, nq, nkv, q_weight, k_weight, eps, rope_pos, store_pos, table_index,
                   block_tables, table_rows, table_stride, num_blocks, block_size, cos, sin, max_seq_len, q_out,
                   k_cache, v_cache, nullptr, nullptr, 0, 0, 0, status};
  const int rc = check_norm_rope("b2_qk_norm_rope_kv_write", p, head_dim, layer, dtype);
  if (rc || n_tokens == 0) return rc;
  const size_t off = (size_t)layer * num_blocks * block_size * nkv * head_dim * dtype_bytes(dtype);
  p.k_cache = static_cast<char*>(k_cache) + off;
  p.v_cache = static_cast<char*>(v_cache) + off;
#define B2_ROPE_CASE(T, HD) return launch_rope<T, HD>(p, stream)
  if (dtype == B2_BF16) {
    if (head_dim == 32) B2_ROPE_CASE(__nv_bfloat16, 32);
    if (head_dim == 64) B2_ROPE_CASE(__nv_bfloat16, 64);
    B2_ROPE_CASE(__nv_bfloat16, 128);
  }
  if (head_dim == 32) B2_ROPE_CASE(float, 32);
  if (head_dim == 64) B2_ROPE_CASE(float, 64);
  B2_ROPE_CASE(float, 128);
#undef B2_ROPE_CASE
}

int b2_qk_norm_rope_kv_write_q8(const void* qkv, int64_t ld_qkv, int n_tokens, int nq, int nkv, int head_dim,
                                const float* q_weight, const float* k_weight, float eps, const int64_t* rope_pos,
                                const int64_t* store_pos, const int32_t* table_index, const int32_t* block_tables,
                                int table_rows, int table_stride, int num_blocks, int block_size, const float* cos,
                                const float* sin, int max_seq_len, void* q_out, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, int cache_dtype, int layer, int dtype,
                                int32_t* status, b2_stream_t stream) {
  using namespace b2;
  NormRopeParams p{qkv, ld_qkv, n_tokens, nq, nkv, q_weight, k_weight, eps, rope_pos, store_pos, table_index,
                   block_tables, table_rows, table_stride, num_blocks, block_size, cos, sin, max_seq_len, q_out,
                   k_cache, v_cache, k_scale, v_scale, 0, 0, 0, status};
  B2_CHECK_ARG(valid_q8_dtype(cache_dtype), "b2_qk_norm_rope_kv_write_q8: bad cache dtype");
  if (block_size != kQ8Block)
    return fail(B2_ENOTSUP, "b2_qk_norm_rope_kv_write_q8: block_size %d (16 only)", block_size);
  const int rc = check_norm_rope("b2_qk_norm_rope_kv_write_q8", p, head_dim, layer, dtype);
  if (rc || n_tokens == 0) return rc;
  B2_CHECK_ARG(k_scale && v_scale, "b2_qk_norm_rope_kv_write_q8: null scales");
  const size_t tiles = (size_t)layer * num_blocks * nkv;
  p.k_cache = static_cast<char*>(k_cache) + tiles * kQ8Block * head_dim;
  p.v_cache = static_cast<char*>(v_cache) + tiles * kQ8Block * head_dim;
  p.k_scale = k_scale + tiles;
  p.v_scale = v_scale + tiles;
#define B2_Q8_CASE(T, HD) return launch_q8<T, HD>(p, cache_dtype, stream)
  if (dtype == B2_BF16) {
    if (head_dim == 32) B2_Q8_CASE(__nv_bfloat16, 32);
    if (head_dim == 64) B2_Q8_CASE(__nv_bfloat16, 64);
    B2_Q8_CASE(__nv_bfloat16, 128);
  }
  if (head_dim == 32) B2_Q8_CASE(float, 32);
  if (head_dim == 64) B2_Q8_CASE(float, 64);
  B2_Q8_CASE(float, 128);
#undef B2_Q8_CASE
}

int b2_kv_read_q8(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                  int cache_dtype, int layer, int num_blocks, int block_size, int nkv, int head_dim,
                  const int32_t* block_ids, int n_blocks, void* k_out, void* v_out, int out_dtype, int32_t* status,
                  b2_stream_t stream) {
  using namespace b2;
  B2_CHECK_ARG(valid_q8_dtype(cache_dtype), "b2_kv_read_q8: bad cache dtype");
  B2_CHECK_ARG(valid_dtype(out_dtype), "b2_kv_read_q8: bad dtype");
  B2_CHECK_ARG(num_blocks > 0 && nkv > 0 && head_dim > 0 && layer >= 0 && n_blocks >= 0,
               "b2_kv_read_q8: bad cache geometry");
  if (block_size != kQ8Block) return fail(B2_ENOTSUP, "b2_kv_read_q8: block_size %d (16 only)", block_size);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(B2_ENOTSUP, "b2_kv_read_q8: head_dim %d not supported (32, 64, 128)", head_dim);
  if (n_blocks == 0) return B2_OK;
  B2_CHECK_ARG(k_cache && v_cache && k_scale && v_scale && block_ids && k_out && v_out, "b2_kv_read_q8: null pointer");
  B2_CHECK_ARG(((uintptr_t)k_cache % 16) == 0 && ((uintptr_t)v_cache % 16) == 0 && ((uintptr_t)k_out % 16) == 0 &&
                   ((uintptr_t)v_out % 16) == 0, "b2_kv_read_q8: buffers must be 16-byte aligned");
  const size_t tiles = (size_t)layer * num_blocks * nkv;
  const uint8_t* kc = static_cast<const uint8_t*>(k_cache) + tiles * kQ8Block * head_dim;
  const uint8_t* vc = static_cast<const uint8_t*>(v_cache) + tiles * kQ8Block * head_dim;
  const int64_t pieces = (int64_t)n_blocks * kQ8Block * nkv * head_dim / 8;
  const int64_t grid = (pieces + 127) / 128;
  B2_CHECK_ARG(grid <= 0x7fffffff && (int64_t)kQ8Block * nkv * head_dim <= 0x7fffffff,
               "b2_kv_read_q8: %d blocks are too many for one call", n_blocks);
  auto go = [&](auto kernel, auto* ko, auto* vo) -> int {
    B2_TRY_CUDA(launch_pdl(kernel, dim3((unsigned)grid), dim3(128), 0, stream, kc, vc, k_scale + tiles,
                           v_scale + tiles, num_blocks, nkv, head_dim, block_ids, n_blocks, ko, vo, status));
    return B2_OK;
  };
  if (out_dtype == B2_BF16) {
    auto* ko = static_cast<__nv_bfloat16*>(k_out);
    auto* vo = static_cast<__nv_bfloat16*>(v_out);
    return cache_dtype == B2_I8 ? go(kv_read_q8_kernel<__nv_bfloat16, B2_I8>, ko, vo)
                                : go(kv_read_q8_kernel<__nv_bfloat16, B2_E4M3>, ko, vo);
  }
  auto* ko = static_cast<float*>(k_out);
  auto* vo = static_cast<float*>(v_out);
  return cache_dtype == B2_I8 ? go(kv_read_q8_kernel<float, B2_I8>, ko, vo)
                              : go(kv_read_q8_kernel<float, B2_E4M3>, ko, vo);
}

}  // extern "C"
