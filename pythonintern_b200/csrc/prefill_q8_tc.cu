// Causal varlen prefill attention over the 8-bit KV cache on the 5th-generation tensor cores
// (tcgen05 + TMEM), head_dim 128.
//
// The schedule of prefill_tc.cu (pairs of 128-row Q tiles sharing 64-key K/V tiles, S, P and O in
// TMEM, one persistent CTA per SM), with converters in the producer's place for K and V: four warps
// read the codes of a K/V tile a tile ahead into registers (per block and kv head one run of
// 2 KB), widen them and store them as the swizzled operands of a three-stage ring.  K codes are exact in bf16
// (q stays as it is) and V codes in f16 (P is rounded to f16, 2^-11), so the only rounding that
// prefill over the model's type does not have is the cache's own.  The scales stay out of the
// operands: a K scale multiplies its 16 columns of S in the softmax, a V scale its 16 columns of
// P.  l is summed against a reference m that follows the scores, P against a second one, m2, that
// follows the largest s + log2(vs), so f16 keeps its precision however the scales of blocks differ.
//
// 16 prompts of 1 024 tokens, heads 32/8, int8: 266 us, 517 TFLOP/s (prefill_tc.cu on a bf16 cache: 262).  As there, the
// issue of the MMAs and the hand-offs between the roles bound it: four converter warps and the register split
// 368 -> 334 us, scales fetched a tile ahead 307, one election per batch of MMAs instead of per MMA 269.
#include "prefill_tc.cuh"
#include "q8.cuh"

namespace b2 {
namespace pftc {
namespace {

constexpr int ST = 3;             // operand ring stages
constexpr int kConvertWarps = 4;
// Warpgroups: control (producer, MMA, two idle warps), two of softmax, converters.  The block is
// launched with 128 registers a thread and hands them out again: 88 + 2 * 168 + 88 = 4 * 128.
constexpr int kSoftmaxWarp = 4, kConvertWarp = kSoftmaxWarp + NG * kGroupWarps;
constexpr int kThreads = 32 * (kConvertWarp + kConvertWarps);
constexpr int kFewRegs = 88, kManyRegs = 168;
static_assert(2 * kFewRegs + 2 * kManyRegs <= 4 * 128, "more registers than the block is launched with");
// Layout (1024-byte aligned): operand ring, Q[NG][2]: 224 KB.
constexpr uint32_t OFF_Q = ST * STAGE;
constexpr int kSeqCache = 192;  // sequences whose lengths are kept in shared memory
constexpr size_t SMEM = OFF_Q + NG * 2 * Q_BYTES + 1024;
static_assert(SMEM + 8 * kSeqCache + 512 <= 232448, "shared memory above the 227 KB a CTA may use");
constexpr float kRoom = 15.f;  // log2 of the largest P
constexpr float kLift = 8.f;   // log2 of P's largest value when a reference has just moved
// m2 is held within 2^kGap of m, which runs ahead of it where V tiles of scale 0 hold the loudest keys: 2^(m - m2)
// stays finite, and what f16 cuts off P (2^-25) is 2^-133 of a code, since l is 2^8 or more.
constexpr float kGap = 100.f;

// Stands for a factor of the scores that is 0 (a K scale of 0, or one whose product with the call's scale rounds to
// 0): -inf * 0 is not -inf.  The smallest number, so that no sum of codes it multiplies becomes a score to speak of.
constexpr float kTiny = 0x1p-149f;

struct ParamsQ8 : Params {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
};

// Instruction descriptor, kind::f16: f16 A and B, f32 accumulator, both K-major.
__host__ __device__ constexpr uint32_t instr_desc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// A sequence whose tokens do not fit its table row is left out (every role finds the same).
__device__ __forceinline__ bool usable(const ParamsQ8& p, const Item& it, int lane) {
  if (!it.valid) return false;
  const int64_t keys = (int64_t)it.ctx0 + it.t0[0] + it.nt[0];
  if (keys <= (int64_t)p.table_stride * kQ8Block) return true;
  if (lane == 0) raise_status(p.status, B2_DEV_RANGE);
  return false;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of float32 for the packed instructions.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Four codes as two 16-bit pairs: bf16 or f16, exact.
template <int CODE, bool BF16>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == B2_I8 && BF16) {
    // 0x4300 | u is the bf16 128 + u for u < 128, and 0x4380 is 256: a code is its low seven
    // bits less 128 where its sign is set, (128 + low) - (128 or 256)
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
    uint32_t al = a & 0xff7fff7fu, as = a & 0xff80ff80u, bl = b & 0xff7fff7fu, bs = b & 0xff80ff80u;
    const __nv_bfloat162 ha = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&al), *reinterpret_cast<__nv_bfloat162*>(&as));
    const __nv_bfloat162 hb = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&bl), *reinterpret_cast<__nv_bfloat162*>(&bs));
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else if constexpr (CODE == B2_I8) {
    // 0x6400 | u is the f16 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    const __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
    if constexpr (BF16) {
      const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
      const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
      const __nv_bfloat162 ha = __floats2bfloat162_rn(fa.x, fa.y), hb = __floats2bfloat162_rn(fb.x, fb.y);
      lo = *reinterpret_cast<const uint32_t*>(&ha);
      hi = *reinterpret_cast<const uint32_t*>(&hb);
    }
  }
}

template <int REP, int CODE>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_q8_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const ParamsQ8 params) {
  constexpr int QT = ROWS / REP;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[NG][2];
  __shared__ __align__(8) uint64_t q_empty[NG][2];
  __shared__ __align__(8) uint64_t kv_full[ST];
  __shared__ __align__(8) uint64_t kv_empty[ST];
  __shared__ __align__(8) uint64_t s_full[NG][2];
  __shared__ __align__(8) uint64_t p_full[NG][2];
  __shared__ __align__(8) uint64_t pv_done[NG][2];
  __shared__ __align__(8) uint64_t o_empty[NG];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int32_t seq_start[kSeqCache + 1], seq_ctx0[kSeqCache];

  pdl_wait();  // the metadata, q and the pool may come from the preceding kernels
  pdl_trigger();
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // every role looks its items up by itself: from shared memory, where the lengths fit
  ParamsQ8 p = params;
  if (p.n_seqs <= kSeqCache) {
    for (int i = threadIdx.x; i <= p.n_seqs; i += kThreads) {
      seq_start[i] = params.seq_start[i];
      if (i < p.n_seqs && params.seq_ctx0) seq_ctx0[i] = params.seq_ctx0[i];
    }
    __syncthreads();
    p.seq_start = seq_start;
    if (params.seq_ctx0) p.seq_ctx0 = seq_ctx0;
  }
  if (blockIdx.x == 0) {  // a seq_start that goes back or leaves the rows is reported, whatever it names
    bool bad = false;
    for (int i = threadIdx.x; i < p.n_seqs; i += kThreads)
      bad |= p.seq_start[i] < 0 || p.seq_start[i + 1] > p.n_rows || p.seq_start[i + 1] < p.seq_start[i];
    if (bad) raise_status(p.status, B2_DEV_RANGE);
  }
  const int pairs = count_pairs(p, QT, lane);
  // sequences that fit the rows have at most (len / QT + 2) / 2 pairs each; more: nothing is computed
  if (pairs < 0 || pairs > p.n_rows / QT / 2 + p.n_seqs + 1) return;
  const int n_items = pairs * p.nkv;
  if ((int)blockIdx.x >= n_items) return;  // nothing allocated yet

  if (threadIdx.x == 0) {
    for (int g = 0; g < NG; ++g) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&q_full[g][b], 1);
        mbar_init(&q_empty[g][b], kGroupWarps);
      }
      for (int b = 0; b < 2; ++b) mbar_init(&s_full[g][b], 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&p_full[g][b], kGroupWarps);
        mbar_init(&pv_done[g][b], 1);
      }
      mbar_init(&o_empty[g], kGroupWarps);
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(&kv_full[s], kConvertWarps);
      mbar_init(&kv_empty[s], 1);
    }
    mbar_init(&drain_bar, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // The first usable item after w (w becomes its number; n_items or more: none).
  auto next_item = [&](int& w) -> Item {
    Item it{};
    for (w += gridDim.x; w < n_items; w += gridDim.x) {
      it = find_item<QT>(p, w, lane);
      if (usable(p, it, lane)) break;
    }
    return it;
  };

  if (warp < kSoftmaxWarp) {
   regs_dec<kFewRegs>();
   if (warp == 0) {
    // ---------------- TMA producer
    const uint64_t pol_q = policy_evict_first();
    int iq[NG] = {0, 0};  // Q loads into each group's buffer
    bool ok = true;
    int w = (int)blockIdx.x - (int)gridDim.x;
    for (Item it = next_item(w); w < n_items && ok; it = next_item(w)) {
      if (lane == 0) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if (it.nt[g] == 0 || !ok) continue;
          const int qb = iq[g] & 1;
          if (!mbar_wait(&q_empty[g][qb], ((uint32_t)(iq[g] >> 1) & 1u) ^ 1u)) {
            raise_status(p.status, B2_DEV_PIPE_TIMEOUT);
            ok = false;
            continue;
          }
          uint8_t* qs = smem + OFF_Q + (g * 2 + qb) * Q_BYTES;
          // rows behind QT * REP hold what they held: they belong to no token, and a row of Q reaches
          // only its own row of S and O
          mbar_arrive_expect_tx(&q_full[g][qb], QT * REP * HD * 2);
          tma_load_3d(qs, &tmQ, &q_full[g][qb], 0, it.g * REP, it.rs + it.t0[g], pol_q);
          tma_load_3d(qs + Q_HALF, &tmQ, &q_full[g][qb], 64, it.g * REP, it.rs + it.t0[g], pol_q);
          ++iq[g];
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
    if (lane == 0) {
      // Copies still in flight (only after an aborted pipeline) land before the CTA exits.
      for (int g = 0; g < NG; ++g)
        for (int qb = 0; qb < 2; ++qb) {
          const int loads = (iq[g] + 1 - qb) / 2;  // copies made into buffer qb of group g
          if (loads > 0) mbar_wait(&q_full[g][qb], (uint32_t)(loads - 1) & 1u, 100000000ull);
        }
    }
    __syncwarp();
   } else if (warp == 1) {
    // ---------------- MMA issuer
    // The whole warp runs this control code; one elected lane issues a batch of tcgen05.mma with
    // its commit.  (An election for every MMA, as in the bf16 kernel, takes its issue slots from
    // sixteen warps here: 307 against 269 us at 16 x 1024 tokens.)  The tensor
    // cores queue only about one MMA ahead, so a wait on a barrier that has already completed
    // (a few hundred cycles for the answer) would leave them idle: the barrier of the next
    // step is tested before the current step's MMAs are issued (peek) and only waited for
    // when that answer was no.  S(n) into S buffer n & 1 needs no barrier of its own: the
    // softmax hands over P(n - 2) only after it has read S(n - 2), and PV(n - 2) is issued
    // (after that hand-over) before S(n).
    constexpr uint32_t idesc_s = instr_desc_bf16(ROWS, KT);
    constexpr uint32_t idesc_pv = instr_desc_f16(ROWS, HD) | (1u << 16);  // B (V) MN-major
    int iq[NG] = {0, 0};  // Q tiles consumed per group
    int js[NG] = {0, 0};  // S tiles issued per group
    int jp[NG] = {0, 0};  // PV tiles issued per group
    int io[NG] = {0, 0};  // items started per group (O hand-offs)
    int qb[NG] = {0, 0};  // the Q buffer of the current item, per group
    int J = 0;
    bool ok = true;
    Peek pk_kv{0u, 0u, false}, pk_pf[NG] = {{0u, 0u, false}, {0u, 0u, false}};
    auto peek_pf = [&](int g) { peek(pk_pf[g], &p_full[g][jp[g] & 1], (uint32_t)(jp[g] >> 1) & 1u); };
    auto peek_kv = [&](int Jn) { peek(pk_kv, &kv_full[Jn % ST], (uint32_t)(Jn / ST) & 1u); };
    // O_g (+)= P_g V of the K/V tile in ring stage `st`; `first` starts the item's O; `ahead`
    // looks at the barrier of the step after this one, before this step's MMAs are issued.
    auto issue_pv = [&](int g, int st, bool first, auto&& ahead) -> bool {
      const int pb = jp[g] & 1;
      if (!__all_sync(0xffffffffu, wait_peeked(pk_pf[g], &p_full[g][pb], (uint32_t)(jp[g] >> 1) & 1u))) return false;
      if (first) {  // the previous item's O has been read out of TMEM
        if (!__all_sync(0xffffffffu, mbar_wait(&o_empty[g], ((uint32_t)io[g] & 1u) ^ 1u))) return false;
        ++io[g];
      }
      tc_fence_after();
      ahead();
      const uint32_t p_tmem = tmem + g * GROUP_COLS + COL_S + pb * KT;  // P(jp) in S buffer jp & 1
      const uint32_t v_addr = smem_u32(smem + (size_t)st * STAGE + 2 * HALF);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)  // 16 keys per MMA: +8 TMEM columns of P, +2 KB of V rows
          umma_bf16_ts(tmem + g * GROUP_COLS + COL_O, p_tmem + kk * 8,
                       smem_desc_sw128_mn(v_addr + kk * 2048, HALF, 1024), idesc_pv, (first && kk == 0) ? 0u : 1u);
        umma_commit(&pv_done[g][pb]);
      }
      ++jp[g];
      return true;
    };
    int w = (int)blockIdx.x - (int)gridDim.x;
    Item it = next_item(w);
    while (w < n_items && ok) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        if (it.nt[g] == 0 || !ok) continue;
        qb[g] = iq[g] & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&q_full[g][qb[g]], (uint32_t)(iq[g] >> 1) & 1u))) ok = false;
        ++iq[g];
      }
      for (int j = 0; j < it.n_kv[0] && ok; ++j, ++J) {
        const int st = J % ST;
        if (!__all_sync(0xffffffffu, wait_peeked(pk_kv, &kv_full[st], (uint32_t)(J / ST) & 1u))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t k_addr = smem_u32(smem + (size_t)st * STAGE);
        const int g_last = j < it.n_kv[1] ? 1 : 0;  // the last S batch of this tile
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if (j >= it.n_kv[g]) continue;
          if (g == g_last) {  // next: PV_0 of tile j - 1, or the next K/V tile
            if (j >= 1) peek_pf(0);
            else peek_kv(J + 1);
          }
          const int b = js[g] & 1;
          const uint32_t q_addr = smem_u32(smem + OFF_Q + (g * 2 + qb[g]) * Q_BYTES);
          if (elect_one()) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_bf16(tmem + g * GROUP_COLS + COL_S + b * KT, smem_desc_sw128(q_addr + half * Q_HALF) + 2 * kk,
                          smem_desc_sw128(k_addr + half * HALF) + 2 * kk, idesc_s, (half | kk) ? 1u : 0u);
            umma_commit(&s_full[g][b]);
          }
          ++js[g];
        }
        if (j >= 1) {
          const int pst = (J - 1) % ST;
          const bool two = j - 1 < it.n_kv[1];  // group 1 also has a PV of tile j - 1
          if (ok) ok = issue_pv(0, pst, j == 1, [&] {
              if (two) peek_pf(1);
              else peek_kv(J + 1);
            });
          if (ok && two) ok = issue_pv(1, pst, j == 1, [&] { peek_kv(J + 1); });
          if (elect_one()) umma_commit(&kv_empty[pst]);  // both groups' S and PV of tile j - 1 are issued
        }
      }
      const Item item = it;
      it = next_item(w);  // looked up while the softmax of the last tile runs
      if (ok) {  // the item's last tile (J is already the next tile's index)
        const int pst = (J - 1) % ST;
        const bool two = item.n_kv[1] == item.n_kv[0];
        const bool first = item.n_kv[0] == 1;
        ok = issue_pv(0, pst, first, [&] {
          if (two) peek_pf(1);
          else peek_kv(J);
        });
        if (ok && two) ok = issue_pv(1, pst, first, [&] { peek_kv(J); });
        if (elect_one()) umma_commit(&kv_empty[pst]);
      }
      if (!ok && lane == 0) raise_status(p.status, B2_DEV_PIPE_TIMEOUT);
    }
    // every MMA issued by the elected lane has completed once drain_bar fires
    if (elect_one()) umma_commit(&drain_bar);
    mbar_wait(&drain_bar, 0, 100000000ull);
    __syncwarp();
   }
  } else if (warp < kConvertWarp) {
    regs_inc<kManyRegs>();
    // ---------------- softmax: one thread per MMA row of its group's Q tile
    const int sw = warp - kSoftmaxWarp;      // 0..7
    const int grp = sw / kGroupWarps;        // 0: the later Q tile, 1: the one before
    const int quarter = warp & 3;            // TMEM lane quarter this warp may access
    const int m = quarter * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16) + grp * GROUP_COLS;
    const int tk = m / REP;
    int js = 0;  // S tiles consumed by this group (the PV of tile js - 1 is the latest issued)
    bool ok = true;
    Peek pk_s{0u, 0u, false};  // the next S tile, tested while this tile's P is written
    int w = (int)blockIdx.x - (int)gridDim.x;
    Item next = next_item(w);
    int items = 0;  // this group's Q tiles
    while (w < n_items && ok) {
      const Item it = next;
      // this group's tile (selected without indexing, so the item stays in registers)
      const int nt = grp ? it.nt[1] : it.nt[0];
      const int t0 = grp ? it.t0[1] : it.t0[0];
      const int n_kv = grp ? it.n_kv[1] : it.n_kv[0];
      if (nt == 0) {
        next = next_item(w);
        continue;
      }
      const bool row_ok = tk < nt;
      const int pos = it.ctx0 + t0 + tk;  // this row's token position (the last key it attends to)
      // l = sum e, e = 2^(s - m); P = e vs 2^(m - m2) in f16, so that m2 follows s + log2(vs)
      float m_ref = -INFINITY, m2_ref = -INFINITY, lift = 0.f, l_run = 0.f;
      // Lane b < 4 sees to block b of a tile: its id is read two tiles ahead, its scales one.  Every
      // row needs the factor kc of its raw scores (-1: a block outside the pool) and the V scale.
      auto id_of = [&](int j) -> int {
        const int bi = j * (KT / 16) + lane;
        if (lane >= KT / 16 || j >= n_kv || bi >= p.table_stride) return -1;
        const int blk = it.table[bi];
        return blk < p.num_blocks ? blk : -1;
      };
      float ks_raw, vs_raw;
      int id_raw;
      auto fetch = [&](int id) {
        id_raw = id;
        ks_raw = id >= 0 ? p.k_scale[(int64_t)id * p.nkv + it.g] : 0.f;
        vs_raw = id >= 0 ? p.v_scale[(int64_t)id * p.nkv + it.g] : 1.f;
      };
      int id_next = id_of(0);
      fetch(id_next);
      id_next = id_of(1);
      for (int j = 0; j < n_kv; ++j, ++js) {
        const int b = js & 1;
        const int k0 = j * KT;
        // the scales were fetched a tile ago: their latency is behind the last tile's work
        const float factor = ks_raw * p.scale_log2;
        const float kc_own = id_raw < 0 ? -1.f : factor == 0.f ? kTiny : factor;
        float kc[KT / 16], vs[KT / 16];
        bool gap = false;  // a block of the tile is outside the pool
#pragma unroll
        for (int u = 0; u < KT / 16; ++u) {
          kc[u] = __shfl_sync(0xffffffffu, kc_own, u);
          vs[u] = __shfl_sync(0xffffffffu, vs_raw, u);
          gap |= kc[u] < 0.f;
        }
        fetch(id_next);
        id_next = id_of(j + 2);
        // warp-uniform verdicts: the TMEM loads and stores below are .sync.aligned
        if (!__all_sync(0xffffffffu, wait_peeked(pk_s, &s_full[grp][b], (uint32_t)(js >> 1) & 1u))) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[64];
        tmem_ld32_nowait(trow + COL_S + b * KT, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
        tmem_ld32_nowait(trow + COL_S + b * KT + 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
        tmem_wait_ld();
        // raw sums q . codes; masked keys are -inf (every factor below is positive)
        float sv[64];
        if (row_ok && k0 + KT - 1 <= pos && !gap) {  // every key of the tile is visible (the common case)
#pragma unroll
          for (int e = 0; e < 64; ++e) sv[e] = __uint_as_float(sr[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 64; ++e)
            sv[e] = (row_ok && k0 + e <= pos && !(kc[e / 16] < 0.f)) ? __uint_as_float(sr[e]) : -INFINITY;
          // a block none of whose keys the row sees adds nothing, whatever its scales
#pragma unroll
          for (int u = 0; u < KT / 16; ++u)
            if (!row_ok || k0 + u * 16 > pos || kc[u] < 0.f) {
              kc[u] = kTiny;
              vs[u] = 0.f;
            }
        }
        float mx = -INFINITY, mx2 = -INFINITY;
#pragma unroll
        for (int u = 0; u < KT / 16; ++u) {
          const float* t = sv + u * 16;
          const float a = max3(t[0], t[1], t[2]), c = max3(t[3], t[4], t[5]), d = max3(t[6], t[7], t[8]);
          const float f = max3(t[9], t[10], t[11]), g = max3(t[12], t[13], t[14]);
          const float top = fmaxf(max3(a, c, d), max3(f, g, t[15])) * kc[u];
          mx = fmaxf(mx, top);
          mx2 = fmaxf(mx2, vs[u] == 0.f ? -INFINITY : top + __log2f(vs[u]));  // only places a reference
        }
        // the references move when a value would pass 2^15, to where it is 2^8
        bool need = false;
        float corr = 1.f;
        if (mx > m_ref + kRoom || mx2 > m2_ref + kRoom) {
          const float mn = fmaxf(m_ref, mx - kLift);
          float m2n = fmaxf(m2_ref, mx2 - kLift);
          if (m2n != -INFINITY) m2n = fmaxf(m2n, mn - kGap);
          l_run *= exp2f(m_ref - mn);  // from -inf: times 0, and l_run is 0
          if (m2_ref != -INFINITY) {   // else the row's O is empty
            need = m2n != m2_ref;
            corr = exp2f(m2_ref - m2n);
          }
          m_ref = mn;
          m2_ref = m2n;
          lift = m2n == -INFINITY ? 0.f : exp2f(mn - m2n);
        }
        if (__any_sync(0xffffffffu, need)) {
          // O must hold PV(js - 1) before it is rescaled (need implies j >= 1)
          if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[grp][(js - 1) & 1], (uint32_t)((js - 1) >> 1) & 1u))) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32_nowait(trow + COL_O + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st32(trow + COL_O + c, o);
          }
          tmem_wait_st();
        }
        // e = exp2(raw * kc - m), P = e * vs * 2^(m - m2) in f16; a row with nothing visible keeps
        // P = 0 (m = -inf is replaced by 0).  Pairs of keys share the packed float32 instructions.
        const float m_sub = m_ref == -INFINITY ? 0.f : m_ref;
        const uint64_t c2 = pack2(-m_sub, -m_sub);
        uint32_t pw[32];  // the row's P in f16 pairs: word w holds keys 2w (low half) and 2w + 1
#pragma unroll
        for (int u = 0; u < KT / 16; ++u) {
          // the next S tile this group consumes (in this item or the next): ask now, so that the
          // answer has arrived when this tile is done
          if (u == 1) peek(pk_s, &s_full[grp][(js + 1) & 1], (uint32_t)((js + 1) >> 1) & 1u);
          // where the product would overflow, the exponentials it meets are 2^-112 or less (2^-120 of the softmax)
          const float f = vs[u] == 0.f ? 0.f : q8_finite(vs[u] * lift);
          const uint64_t k2 = pack2(kc[u], kc[u]), f2 = pack2(f, f);
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int e2 = 0; e2 < 8; ++e2) {
            const int e = u * 16 + e2 * 2;
            float x0, x1;
            unpack2(fma2(pack2(sv[e], sv[e + 1]), k2, c2), x0, x1);
            const uint64_t e12 = pack2(ex2_approx(x0), ex2_approx(x1));  // -inf gives 0
            sum[e2 & 1] = add2(sum[e2 & 1], e12);
            unpack2(mul2(e12, f2), x0, x1);
            const __half2 h2 = __floats2half2_rn(x0, x1);
            pw[u * 8 + e2] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          float s0, s1;
          unpack2(add2(sum[0], sum[1]), s0, s1);
          l_run += s0 + s1;
        }
        // P over the first 32 columns of this S buffer (read above): the A operand of PV(js),
        // which the tensor cores run before S(js + 2) rewrites the buffer
        tmem_st32(trow + COL_S + b * KT, pw);
        tmem_wait_st();
        tc_fence_before();  // P and the rescaled O columns are read by the tensor cores
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[grp][b]);
      }
      if (!ok) break;
      // O / l to global memory once the item's last PV has completed (the next item is looked up
      // meanwhile); then O may be reused.  The rows go through this group's Q buffer, which no MMA
      // reads any more, so that they are written whole: a thread's own row in 16-byte pieces would
      // touch 32 rows with every store.
      next = next_item(w);
      if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[grp][(js - 1) & 1], (uint32_t)((js - 1) >> 1) & 1u))) {
        ok = false;
        break;
      }
      tc_fence_after();
      // O and l have references of their own; a row without weight gives 0 (NaN if a tile it saw is)
      const float inv = m2_ref == -INFINITY ? (l_run == l_run ? 0.f : l_run) : exp2f(m2_ref - m_ref) / l_run;
      const int qb = items++ & 1;
      uint8_t* stage = smem + OFF_Q + (grp * 2 + qb) * Q_BYTES + quarter * 32 * (HD * 2);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        tmem_ld32_nowait(trow + COL_O + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int u = 0; u < 32; u += 8) {
          uint32_t wv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            __nv_bfloat162 h2 = __floats2bfloat162_rn(__uint_as_float(o[u + 2 * e]) * inv,
                                                      __uint_as_float(o[u + 2 * e + 1]) * inv);
            wv[e] = *reinterpret_cast<uint32_t*>(&h2);
          }
          const int piece = (c + u) / 8;  // of the row's sixteen, spread over the banks
          *reinterpret_cast<uint4*>(stage + lane * (HD * 2) + (piece ^ (lane & 7)) * 16) =
              make_uint4(wv[0], wv[1], wv[2], wv[3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[grp]);
      __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)(it.rs + t0) * p.ld_out +
                           (int64_t)it.g * REP * HD + (lane & 15) * 8;
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {  // two rows at a time
        const int r = 2 * i + (lane >> 4), row = quarter * 32 + r;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + r * (HD * 2) + ((lane & 15) ^ (r & 7)) * 16);
        if (row / REP < nt) *reinterpret_cast<uint4*>(out + (int64_t)(row / REP) * p.ld_out + (row % REP) * HD) = v;
      }
      fence_proxy_async_smem();  // the buffer goes back to TMA
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[grp][qb]);
    }
    if (!ok && lane == 0) raise_status(p.status, B2_DEV_PIPE_TIMEOUT);
  } else {
    regs_dec<kFewRegs>();
    // ---------------- converters: codes to the operands, K exact in bf16, V exact in f16
    // 16-byte pieces of codes (16 dims of one key).  The eight threads of a store phase write two
    // keys' rows of one 64-dim half, whose swizzled chunks fall into different banks.
    const int c = threadIdx.x - 32 * kConvertWarp;
    const int half = (c >> 3) & 1, key0 = (c >> 4) * 2 + ((c >> 2) & 1), ch = c & 3;
    constexpr int PIECES = KT * HD / 16 / (32 * kConvertWarps), KEYS = KT / PIECES;  // keys key0 + KEYS i
    int J = 0;
    bool ok = true;
    int w = (int)blockIdx.x - (int)gridDim.x;
    for (Item it = next_item(w); w < n_items && ok; it = next_item(w)) {
      const int last_pos = it.ctx0 + it.t0[0] + it.nt[0] - 1;  // tile 0 is the later one
      // Lane b < 4 holds the id of block b of a tile, read a tile ahead of its codes.  A block
      // outside the pool is reported (where a row attends to its keys) and block 0 read instead.
      auto id_of = [&](int j) -> int {
        const int bi = j * (KT / 16) + lane;
        if (lane >= KT / 16 || j >= it.n_kv[0]) return -1;
        const int blk = bi < p.table_stride ? it.table[bi] : -1;
        if (blk >= 0 && blk < p.num_blocks) return blk;
        if (bi * 16 <= last_pos) raise_status(p.status, B2_DEV_RANGE);
        return -1;
      };
      uint4 kcode[PIECES], vcode[PIECES];
      const int64_t at = ((int64_t)it.g * 16 + key0) * HD + half * 64 + ch * 16;
      auto load = [&](const uint8_t* cache, int ids, uint4 (&code)[PIECES]) {
#pragma unroll
        for (int u = 0; u < KT / 16; ++u) {
          const int64_t tile = (int64_t)max(0, __shfl_sync(0xffffffffu, ids, u)) * p.nkv * (16 * HD) + at;
#pragma unroll
          for (int i = 0; i < 16 / KEYS; ++i)
            code[u * (16 / KEYS) + i] = *reinterpret_cast<const uint4*>(cache + tile + i * KEYS * HD);
        }
      };
      int ids = id_of(0), ids_next = id_of(1);
      load(p.k_cache, ids, kcode);
      load(p.v_cache, ids, vcode);
      for (int j = 0; j < it.n_kv[0]; ++j, ++J) {
        const int st = J % ST;
        const unsigned in_pool = __ballot_sync(0xffffffffu, ids >= 0);
        ids = ids_next;
        ids_next = id_of(j + 2);
        if (!__all_sync(0xffffffffu, mbar_wait(&kv_empty[st], ((uint32_t)(J / ST) & 1u) ^ 1u))) {
          ok = false;
          break;
        }
        uint8_t* dst = smem + (size_t)st * STAGE + half * HALF + key0 * 128;
        const int x0 = ((2 * ch) ^ (key0 & 7)) * 16, x1 = ((2 * ch + 1) ^ (key0 & 7)) * 16;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          uint4 a, b;
          widen<CODE, true>(kcode[i].x, a.x, a.y);
          widen<CODE, true>(kcode[i].y, a.z, a.w);
          widen<CODE, true>(kcode[i].z, b.x, b.y);
          widen<CODE, true>(kcode[i].w, b.z, b.w);
          *reinterpret_cast<uint4*>(dst + i * KEYS * 128 + x0) = a;
          *reinterpret_cast<uint4*>(dst + i * KEYS * 128 + x1) = b;
        }
        load(p.k_cache, ids, kcode);  // the next tile's codes arrive while this one's are used
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          // keys that no row sees: whatever their codes (an e4m3 NaN among them), V is 0
          const int key = key0 + KEYS * i;
          if (j * KT + key > last_pos || !(in_pool >> (key / 16) & 1)) vcode[i] = make_uint4(0, 0, 0, 0);
          uint4 a, b;
          widen<CODE, false>(vcode[i].x, a.x, a.y);
          widen<CODE, false>(vcode[i].y, a.z, a.w);
          widen<CODE, false>(vcode[i].z, b.x, b.y);
          widen<CODE, false>(vcode[i].w, b.z, b.w);
          *reinterpret_cast<uint4*>(dst + 2 * HALF + i * KEYS * 128 + x0) = a;
          *reinterpret_cast<uint4*>(dst + 2 * HALF + i * KEYS * 128 + x1) = b;
        }
        load(p.v_cache, ids, vcode);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[st]);
      }
    }
    if (!ok && lane == 0) raise_status(p.status, B2_DEV_PIPE_TIMEOUT);
  }

  // ---------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}


}  // namespace
}  // namespace pftc

// Heads to a kv head that the kernel is compiled for.
bool prefill_q8_tc_serves(int rep) { return (rep >= 1 && rep <= 8) || rep == 12 || rep == 16; }

// Launches the tensor-core prefill attention over the 8-bit cache (bf16 q, head_dim 128).
// k_cache ... v_scale are those of the layer.  Returns B2_ENOTSUP, launching nothing, for shapes
// it does not serve.
int prefill_attention_q8_tc(const void* q, int64_t ld_q, int n_rows, int nq, int nkv, const uint8_t* k_cache,
                            const uint8_t* v_cache, const float* k_scale, const float* v_scale, int cache_dtype,
                            int num_blocks, const int32_t* tables, int table_stride, const int32_t* seq_start,
                            const int32_t* seq_ctx0, int n_seqs, float scale, void* out, int64_t ld_out,
                            int32_t* status, cudaStream_t stream) {
  using namespace pftc;
  const int rep = nq / nkv;
  if (!prefill_q8_tc_serves(rep)) return fail(B2_ENOTSUP, "prefill q8 tc: nq/nkv = %d", rep);
  if (!(scale > 0.f)) return fail(B2_ENOTSUP, "prefill q8 tc: scale %g", (double)scale);
  ParamsQ8 p{};
  p.n_rows = n_rows;
  p.nq = nq;
  p.nkv = nkv;
  p.num_blocks = num_blocks;
  p.tables = tables;
  p.table_stride = table_stride;
  p.seq_start = seq_start;
  p.seq_ctx0 = seq_ctx0;
  p.n_seqs = n_seqs;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = out;
  p.ld_out = ld_out;
  p.status = status;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  const int qt = ROWS / rep;
  CUtensorMap mq;
  const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)nq, (cuuint64_t)n_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)ld_q * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)rep, (cuuint32_t)qt};
  const int rc = encode(&mq, q, 3, dims, strides, box);
  if (rc) return rc;
  const long items = (long)((n_rows / qt + n_seqs) / 2 + n_seqs) * nkv;  // an upper bound; the kernel counts exactly
  const dim3 grid((unsigned)(items < sm_count() ? items : sm_count()));
  auto go = [&](void (*k)(const CUtensorMap, const ParamsQ8)) -> int {
    const int rc = allow_smem_once((const void*)k, SMEM);
    if (rc) return rc;
    B2_TRY_CUDA(launch_pdl(k, grid, dim3(kThreads), SMEM, stream, mq, p));
    return B2_OK;
  };
  const bool i8 = cache_dtype == B2_I8;
#define B2_CASE(REP) \
  case REP: return go(i8 ? prefill_q8_tc_kernel<REP, B2_I8> : prefill_q8_tc_kernel<REP, B2_E4M3>)
  switch (rep) {
    B2_CASE(1);
    B2_CASE(2);
    B2_CASE(3);
    B2_CASE(4);
    B2_CASE(5);
    B2_CASE(6);
    B2_CASE(7);
    B2_CASE(8);
    B2_CASE(12);
    default: return go(i8 ? prefill_q8_tc_kernel<16, B2_I8> : prefill_q8_tc_kernel<16, B2_E4M3>);
  }
#undef B2_CASE
}

}  // namespace b2
