// Shared pieces of the two tcgen05 prefill attention kernels (prefill_tc.cu over the pool in the
// model's type, prefill_q8_tc.cu over the 8-bit cache): tile sizes, TMEM layout, the
// enumeration of the work items and the operand descriptors.
#pragma once
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace b2 {
namespace pftc {

using namespace b2::tc;

constexpr int HD = 128;
constexpr int ROWS = 128;                              // MMA M: (token, head) rows per Q tile
constexpr int KT = 64;                                 // keys per KV tile (4 pool blocks)
constexpr int NG = 2;                                  // Q tiles (softmax groups) per item
constexpr int kGroupWarps = 4;                         // one per TMEM lane quarter
constexpr uint32_t HALF = KT * 64 * 2;                 // 8 KB: 64 keys x 64 dims
constexpr uint32_t STAGE = 4 * HALF;                   // K lo | K hi | V lo | V hi
constexpr uint32_t Q_HALF = ROWS * 64 * 2;             // 16 KB
constexpr uint32_t Q_BYTES = 2 * Q_HALF;               // one Q tile, lo | hi
// TMEM per group (256 columns): S[2] (64 each) then O (128); 512 in all.  P(j) in 16 bits
// overwrites the first 32 columns of S(j)'s buffer once the softmax has read S(j).
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t GROUP_COLS = 256, COL_S = 0, COL_O = 128;

struct Params {
  int n_rows, nq, nkv;
  int num_blocks;
  const int32_t* tables;
  int table_stride;
  const int32_t* seq_start;
  const int32_t* seq_ctx0;
  int n_seqs;
  float scale_log2;
  void* out;
  int64_t ld_out;
  int32_t* status;
};

// Shared-memory descriptor of an MN-major operand with 128-byte swizzle: 64-element rows
// along N (128 bytes), 8-row groups along K `sbo` bytes apart, the next 64 N-elements
// `lbo` bytes on (sm_100 descriptor version 1).
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 32 lanes x 32 consecutive 32-bit columns stored to TMEM (the caller waits with
// tmem_wait_st() before the tensor cores may read them).
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One work item: kv head g and up to two Q tiles of one sequence (tile 1 may be empty).
struct Item {
  int rs, ctx0, g;
  int t0[NG], nt[NG], n_kv[NG];
  const int32_t* table;
  bool valid;
};

// Q-tile pairs of QT tokens over all sequences (every lane of the calling warp gets the total).
__device__ __forceinline__ int count_pairs(const Params& p, int qt, int lane) {
  int total = 0;
  for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
    const int s = s0 + lane;
    int np = 0;
    if (s < p.n_seqs) {
      const int len = p.seq_start[s + 1] - p.seq_start[s];
      np = len > 0 ? ((len + qt - 1) / qt + 1) / 2 : 0;
    }
    total += __reduce_add_sync(0xffffffffu, np);
  }
  return total;
}

// Item w: kv head w % nkv of pair w / nkv, pairs numbered sequence by sequence with each
// sequence's last (longest) tiles first: pair u holds tiles 2u and 2u + 1 counted from the
// end of the sequence.  Every warp computes the same answer (warp prefix sums over the
// sequences); all lanes of the calling warp take part.
template <int QT>
__device__ Item find_item(const Params& p, int w, int lane) {
  Item it{};
  it.valid = false;
  const int bx = w / p.nkv;
  it.g = w % p.nkv;
  int seq = -1, pair = 0, base = 0;
  for (int s0 = 0; s0 < p.n_seqs && seq < 0; s0 += 32) {
    const int s = s0 + lane;
    int np = 0;
    if (s < p.n_seqs) {
      const int len = p.seq_start[s + 1] - p.seq_start[s];
      np = len > 0 ? ((len + QT - 1) / QT + 1) / 2 : 0;
    }
    int inc = np;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const int total = __shfl_sync(0xffffffffu, inc, 31);
    const int b = bx - base;
    if (b < total) {
      const unsigned hit = __ballot_sync(0xffffffffu, b < inc);
      const int l = __ffs(hit) - 1;
      const int inc_l = __shfl_sync(0xffffffffu, inc, l);
      const int np_l = __shfl_sync(0xffffffffu, np, l);
      seq = s0 + l;
      pair = b - (inc_l - np_l);
    }
    base += total;
  }
  if (seq < 0) return it;
  const int rs = p.seq_start[seq], re = p.seq_start[seq + 1];
  const int ctx0 = p.seq_ctx0 ? p.seq_ctx0[seq] : 0;
  if (rs < 0 || re > p.n_rows || ctx0 < 0) {
    if (lane == 0) raise_status(p.status, B2_DEV_RANGE);
    return it;
  }
  const int len = re - rs;
  const int ntile = (len + QT - 1) / QT;
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    const int tile = 2 * pair + q;  // counted from the end of the sequence
    if (tile < ntile) {
      it.t0[q] = (ntile - 1 - tile) * QT;          // first token of the tile within its sequence
      it.nt[q] = min(QT, len - it.t0[q]);          // tokens in the tile (>= 1)
      it.n_kv[q] = (ctx0 + it.t0[q] + it.nt[q] - 1) / KT + 1;  // KV tiles up to its last position
    } else {
      it.t0[q] = 0;
      it.nt[q] = 0;
      it.n_kv[q] = 0;
    }
  }
  it.rs = rs;
  it.ctx0 = ctx0;
  it.table = p.tables + (int64_t)seq * p.table_stride;
  it.valid = true;
  return it;
}

static int allow_smem_once(const void* fn, size_t bytes) {
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

static int encode(CUtensorMap* m, const void* ptr, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
  auto fn = encode_fn();
  if (!fn) return fail(B2_ECUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint32_t es[3] = {1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(ptr), dims, strides, box, es,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B2_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return B2_OK;
}

}  // namespace pftc
}  // namespace b2
