// Attention of prompt portions over pages in 8 bits on the 5th-generation tensor cores, bfloat16 queries, heads of up to 128.
//
// A CTA takes 128 queries of NT query heads that read the same key/value head (NT 2 where heads come in pairs, and CTAs are many) and
// walks the request's keys in blocks of 64 positions:
//   converters  4 or 8 warps: codes (bulk copies of 16 positions each, two blocks ahead) to fp16 operands of K and V in 128-byte-swizzled
//               shared memory, once for all NT heads; the scales of the block's four groups of 16 positions beside them
//   issuers     2 warps a head: S_t = Q_t K^T (M 128 x N 64) into tensor memory, and O_t += P_t V with P_t read from tensor memory
//   softmax     4 warps for each head, a thread a query: S from tensor memory, masks, running maximum and sum in float32, P as fp16 beside S
// The softmax threads take a row of S into registers and let go of it: S of the next block is formed while they work on this one, and
// P V of the block before as well (two buffers of P), so that the chain of a tile's blocks is its softmax alone.  (With P over S in
// blocks of 128 keys P V and S stood in that chain: 398 us for the 2048 queries below, against 357 at that time.)
// Two heads of a CTA have chains of their own, and a converted block serves both.
//
// Bound by the softmax warps' chain.  2048 queries of 32/8 heads of 128 at position 6144: 263 us, 915 TFLOP/s of products (64 keys and two
// heads: products 1344 clocks, a block 2120, of which 1670 are a thread's 64 exponentials beside another head's on the same scheduler,
// 120 the scores' way into registers, 330 barriers), and 256 CTAs on 148 SMs.  Steps on the way: a look at every weight for one that is too
// large 359 us, at the sums of a group of them 342; then bulk copies of the codes (converters that loaded them had taken more time for
// addresses than for codes) and a pass that is done again as code of its own (no register is copied for it): 284.  The tiles start in the
// order of their list, the most keys first as the engine lists them: 263; from its end it was 281 (2048 queries at 0: 56 and 73, 8192 at 0:
// 581 and 645, 4096 of 16 heads of 64 at 0: 75 and 104).  A polynomial for a part of the exponentials (a quarter: 282, a half: 296, when
// the kernel took 284) moves them from one busy unit to another and was left out; so were two threads a query, 32 keys of a block
// each: 304, the pair has to agree on its maximum in every block.
//
// Codes: u = code + 128 in the low byte of an fp16 is the subnormal number u * 2^-24, exact; K enters that way (two codes a bit
// operation), and 128 * 2^-24 sum(q), a number of the query, comes off S in the multiply-add that scales it.  V enters as the exact
// codes (1024 + u less 1152).  Both give the bytes 0, 2, 1, 3 of every four in that order: Q's columns are stored in the same order, and
// O's are put back when a row is written.  Queries are scaled by a power of two to [2^14, 2^15) at most, as fp16 exact to 2^-28 of their
// largest number.
// Scales: s = scale * sk * (q . codes) with sk the block's key scale; the weight that meets V's codes is w = exp(s) * sv, so the exponent
// gets log2(sv), the base follows the largest s + log2(sv) (w is what enters O: a weight that is small beside it may round away, whatever
// its sv), and the sum below takes exp(s) = w / sv a group at a time.  A group of values of nothing (sv 0) adds to the sum alone, which
// it does beside the others, with a maximum of its own (as codes of 0 with some sv it would raise the base, and the weights of groups
// of small values would round away).  The base is set 2^7 below the largest, and again once the weights of a group sum to more than the
// largest fp16, so O is scaled again, by the softmax threads in tensor memory, a few times a row at most.  A weight loses
// 2^-12 of itself down to 2^-14, below that 2^-25 at most: 2^-32 of the largest, of 131072 keys together 3e-5 of it (with the base at
// the largest and room for 2^12 beyond it, 2^-25 of it for each: a flat tail that holds a 250th of the weight could vanish).
//
// Every wait is bounded; a wait that gives up sets an abort flag that all roles see, the CTA frees its tensor memory and reports
// MLXB_ST_WAIT_TIMEOUT.  The order in which a query's keys are added depends on its position and window alone; when its base is set again
// is a vote of the 32 queries of a warp, so its last bits depend on the queries beside it too, that is on how a prompt was cut.
#include <cuda_fp16.h>

#include "tcgen05.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int BLK = 16;              // positions that share a scale
constexpr int TQ = 128;              // queries of a tile
constexpr int TK = 64;               // keys of a block
constexpr int GR = TK / BLK;         // groups of a block
constexpr int SMS = 148;
constexpr int XR = 8;                // blocks whose scales are kept
constexpr float LOG2E = 1.4426950408889634f;
constexpr float UNIT = 5.9604644775390625e-8f;          // 2^-24
constexpr float UP = 7.f;            // log2 of the largest weight after the base of the exponentials has been set
constexpr float HIGH = 65504.f;      // the largest sum of a group's weights that a pass leaves be: the largest fp16

struct PortionArgs {
  const __nv_bfloat16* q;
  int ldq;
  const int4* tiles;
  const int* block_table;
  int n_tokens, n_req, max_pages, n_pages, page, Hq, Hkv, dim, window;
  float scale;
  const int8_t *k8, *v8;
  const float *ks, *vs, *sinks;
  __nv_bfloat16* out;
  int ldo, vec;
  int* status;
};

template <int DP, int NT>
struct Shape {
  static constexpr int CTAS = NT == 1 && DP == 64 ? 2 : 1;        // on an SM
  static constexpr int SOFT = 4 * NT, CONV = DP == 128 ? 8 : 4;   // warps
  // converters work in NG groups, a block each, that have RD blocks of codes each under way; KST buffers of K and of V: what fits
  static constexpr int NG = 2, RD = 2, GW = CONV / NG, KST = (NT == 2) == (DP == 64) ? 4 : 3;
  static constexpr int THREADS = 32 * (SOFT + CONV + 4);          // (the last four issue products)
  // registers a thread, at launch (what the launch bounds leave: 640 x 96, 512 x 128, 384 x 80 twice) and then by role, no more in all
  static constexpr int R_LAUNCH = CTAS == 2 ? 80 : NT == 2 && DP == 128 ? 96 : 128;
  static constexpr int R_SOFT = CTAS == 2 ? 128 : 144, R_CONV = 72, R_ISSUE = NT == 1 ? 24 : 40;
  static_assert(32 * (SOFT * R_SOFT + CONV * R_CONV + 4 * R_ISSUE) <= THREADS * R_LAUNCH, "registers");
  static constexpr uint32_t COLS = NT == 1 ? 256 : 512;           // of tensor memory: S_t at 128 t, two buffers of P_t behind it; then O_t
  static constexpr int QSPAN = TQ * 128, SPAN = TK * 128;         // bytes of a tile's rows of 64 columns
  static constexpr int QTILE = QSPAN * (DP / 64), TILE = SPAN * (DP / 64), RAW = TK * DP;
};

template <int DP, int NT>
struct Smem {
  using H = Shape<DP, NT>;
  alignas(1024) uint8_t q[NT][H::QTILE];
  alignas(1024) uint8_t k[H::KST][H::TILE];
  alignas(1024) uint8_t v[H::KST][H::TILE];
  alignas(1024) uint8_t raw_k[H::NG][H::RD][H::RAW], raw_v[H::NG][H::RD][H::RAW];      // codes as they come
  float sk[XR][GR], lsv[XR][GR], rsv[XR][GR];           // of the last blocks: key scale, log2 and reciprocal of the value scale
  uint32_t marks[XR];                                   // bit g: group g has no page; bit 8 + g: its values are 0
  uint32_t nothing[H::NG];                              // groups whose values are 0 whatever their codes
  alignas(8) uint64_t q_full[NT], k_full[H::KST], k_free[H::KST], v_full[H::KST], v_free[H::KST];
  uint64_t s_full[NT], s_read[NT], p_full[NT][2], pv_done[NT][2], drained[2 * NT];
  uint64_t rk_full[H::NG][H::RD], rv_full[H::NG][H::RD];
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ uint64_t desc_of(uint32_t saddr, uint32_t lbo_bytes) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor for kind::f16: float32 accumulator, A and B fp16, A K-major, B K-major or MN-major (bit 16), N/8 in bits
// 17-22, M/16 in bits 24-28.
__host__ __device__ constexpr uint32_t idesc_of(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TQ >> 4) << 24);
}
// A from tensor memory
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// Waits for the loads from tensor memory so far.  The registers they fill go through the statement: what is done with them stays behind it.
__device__ __forceinline__ void ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}
__device__ __forceinline__ void ld_wait(uint32_t (&r)[2][32]) {
  ld_wait(r[0]);
  ld_wait(r[1]);
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
// Registers a thread from here on.  More are asked for with `inc`, fewer with `dec`: the other way round is an illegal instruction.
template <int N, int AT_LAUNCH>
__device__ __forceinline__ void registers() {
  if constexpr (N > AT_LAUNCH) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else if constexpr (N < AT_LAUNCH) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// two float32 at a time
__device__ __forceinline__ void fma2(float& x0, float& x1, float a0, float a1, float b, float c) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}" : "=f"(x0), "=f"(x1) : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float& x0, float& x1, float a0, float a1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(x0), "+f"(x1) : "f"(a0), "f"(a1));
}
// mbar_wait_warp with one look at the barrier in front of its loop.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, done != 0) || mbar_wait_warp(bar, parity, abort_flag);
}
// `bytes` (a multiple of 16, as both addresses) from global to shared memory; the barrier counts them.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// A barrier of some of the CTA's warps.
__device__ __forceinline__ void group_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
__device__ __forceinline__ uint32_t masked_xor(uint32_t w, uint32_t x) {      // (w & 0x00ff00ff) ^ x
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(y) : "r"(w), "r"(0x00ff00ffu), "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t less1152(uint32_t x) {
  uint32_t y;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
  return y;
}

// tiles: int32 [n_tiles][4] = (row of the tile's first token, queries (0: skipped) up to 128, block-table row of the request, position of
// the first query).
template <int DP, int NT>
__global__ void __launch_bounds__(Shape<DP, NT>::THREADS, Shape<DP, NT>::CTAS)
portions_kernel(const PortionArgs a) {
  using H = Shape<DP, NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<DP, NT>& sm = *reinterpret_cast<Smem<DP, NT>*>(smem_raw);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int heads = a.Hq / NT, by_tile = blockIdx.x / heads;
  const int4 tile = a.tiles[by_tile];                   // in the list's order: its first tiles start first
  // (a list without one tile to do must not end before its predecessor has: what comes next waits for this grid only)
  if (tile.y <= 0) {
    if (blockIdx.x == 0) pdl_wait();
    return;
  }
  const int row0 = tile.x, n_rows = min(tile.y, TQ), req = tile.z, pos0 = tile.w;
  if (row0 < 0 || row0 > a.n_tokens - n_rows || req < 0 || req >= a.n_req || pos0 < 0 || pos0 > INT_MAX - TQ) {
    if (blockIdx.x == 0) pdl_wait();
    if (threadIdx.x == 0) atomicOr(a.status, MLXB_ST_POSITION_RANGE);
    return;
  }
  const int h0 = (blockIdx.x - by_tile * heads) * NT, hk = h0 / (a.Hq / a.Hkv);
  const int last_pos = pos0 + n_rows - 1;
  const int first_key = a.window > 0 && pos0 - a.window + 1 > 0 ? pos0 - a.window + 1 : 0;
  const int kb_lo = first_key / TK, n_blocks = last_pos / TK - kb_lo + 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NT; ++i) {
      mbar_init(&sm.q_full[i], 4);
      mbar_init(&sm.s_full[i], 2);
      mbar_init(&sm.s_read[i], 4);
      for (int b = 0; b < 2; ++b) { mbar_init(&sm.p_full[i][b], 4); mbar_init(&sm.pv_done[i][b], 1); }
    }
    for (int i = 0; i < H::KST; ++i) {
      mbar_init(&sm.k_full[i], H::GW);
      mbar_init(&sm.v_full[i], H::GW);
      mbar_init(&sm.k_free[i], NT);
      mbar_init(&sm.v_free[i], NT);
    }
    for (int i = 0; i < 2 * NT; ++i) mbar_init(&sm.drained[i], 1);
    for (int i = 0; i < H::NG * H::RD; ++i) { mbar_init(&sm.rk_full[0][0] + i, 1); mbar_init(&sm.rv_full[0][0] + i, 1); }
    sm.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == H::SOFT + H::CONV) {   // an issuer owns the tensor memory
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(H::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = sm.tmem_base;
  const uint32_t tmem_o = tmem + NT * 2 * TK;           // O_t at tmem_o + DP t
  volatile int* abort_flag = &sm.abort_flag;
  pdl_trigger();

  if (warp >= H::SOFT + H::CONV) {
    registers<H::R_ISSUE, H::R_LAUNCH>();
    // Warp t of these issues S_t, warp NT + t the products P_t V.  (One warp for all of them was the bound: a product took it about 145
    // clocks whatever its size.)  One value for the warp, and known as that to the compiler: what the products take stays in uniform
    // registers.
    const int w = warp - H::SOFT - H::CONV, t = w % NT;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0) + (uint32_t)(2 * t * TK);      // this head's S, P 64 columns on
    const int n = __shfl_sync(0xffffffffu, n_blocks, 0);
    bool ok = true;
    if (w < NT) {
      constexpr uint32_t idesc = idesc_of(TK, false);
      const uint64_t dq = desc_of(smem_u32(sm.q[0]), 16) + (uint32_t)(t * (H::QTILE / 16)), dk0 = desc_of(smem_u32(sm.k[0]), 16);
      ok = wait_warp(&sm.q_full[t], 0, abort_flag);
      for (int i = 0; i < n && ok; ++i) {
        if (!(ok = wait_warp(&sm.k_full[i % H::KST], (uint32_t)((i / H::KST) & 1), abort_flag))) break;
        // P V of the block before last has read the buffer that this block's P goes to
        if (i >= 2 && !(ok = wait_warp(&sm.pv_done[t][i & 1], (uint32_t)(((i - 2) >> 1) & 1), abort_flag))) break;
        if (i > 0 && !(ok = wait_warp(&sm.s_read[t], (uint32_t)((i - 1) & 1), abort_flag))) break;     // S is in registers
        after_sync();
        // with the scales, which came with the keys, and that buffer the softmax has all it needs once S is there
        if (lane == 0) mbar_arrive(&sm.s_full[t]);
        if (elect_one()) {
          const uint64_t dk = dk0 + (uint32_t)((i % H::KST) * (H::TILE / 16));
#pragma unroll
          for (int j = 0; j < DP / 16; ++j)             // 16 columns: 32 bytes inside a span of 64, then the next span
            umma_bf16(tm, dq + (uint32_t)((j >> 2) * (H::QSPAN / 16) + 2 * (j & 3)),
                      dk + (uint32_t)((j >> 2) * (H::SPAN / 16) + 2 * (j & 3)), idesc, j > 0 ? 1u : 0u);
#ifdef MLXB_TEST_WAIT_TIMEOUT
          if (!g_test_withhold_arrival || i > 0)       // the test's missing arrival
#endif
          umma_commit(&sm.s_full[t]);
          umma_commit(&sm.k_free[i % H::KST]);
        }
        __syncwarp();
      }
    } else if (w < 2 * NT) {
      constexpr uint32_t idesc = idesc_of(DP, true);
      const uint64_t dv0 = desc_of(smem_u32(sm.v[0]), H::SPAN);
      const uint32_t to = __shfl_sync(0xffffffffu, tmem_o, 0) + (uint32_t)(t * DP);
      for (int i = 0; i < n && ok; ++i) {
        if (!(ok = wait_warp(&sm.v_full[i % H::KST], (uint32_t)((i / H::KST) & 1), abort_flag))) break;
        if (!(ok = wait_warp(&sm.p_full[t][i & 1], (uint32_t)((i >> 1) & 1), abort_flag))) break;      // P_t is written
        after_sync();
        if (elect_one()) {
          const uint64_t dv = dv0 + (uint32_t)((i % H::KST) * (H::TILE / 16));
#pragma unroll
          for (int j = 0; j < TK / 16; ++j)             // 16 keys: 8 columns of P, 16 rows of V
            umma_ts(to, tm + (uint32_t)(TK + (i & 1) * (TK / 2) + 8 * j), dv + (uint32_t)(j * (16 * 128 / 16)), idesc, i > 0 || j > 0 ? 1u : 0u);
          umma_commit(&sm.pv_done[t][i & 1]);
          umma_commit(&sm.v_free[i % H::KST]);
        }
        __syncwarp();
      }
    }
    if (w < 2 * NT) {
      // whatever ended the loop: no product is under way when the tensor memory is freed
      if (elect_one()) umma_commit(&sm.drained[w]);
      __syncwarp();
      int never = 0;
      mbar_wait_warp(&sm.drained[w], 0, &never);
    }
  } else if (warp >= H::SOFT) {
    registers<H::R_CONV, H::R_LAUNCH>();
    // converters: a thread takes 16 codes (a piece of a row) at a time.  The codes are copied 16 positions at a time.
    // Where a CTA has one head, one warp of a group sees to the codes of K, another to those of V, a third to the scales: with one for all of
    // it that warp was what the blocks waited for (128 queries of 32/8 heads of 128 at 8000: 117 us, 108 so).  Where it has two, the softmax is,
    // and every warp that looks pages up takes issue slots from it (2048 queries at 6144: 290 us so, 284 with one).
    const int group = (warp - H::SOFT) / H::GW, c = threadIdx.x - 32 * (H::SOFT + group * H::GW);
    const int cw = (warp - H::SOFT) % H::GW;
    constexpr int V_BY = NT == 1 ? 1 : 0, SCALES_BY = NT == 1 && H::GW > 2 ? 2 : 0;
    const bool brings_k = cw == 0, brings_v = cw == V_BY, brings_scales = cw == SCALES_BY, leads = brings_k || brings_v || brings_scales;
    const int pieces = a.dim / 16, per = a.page / BLK, copy = BLK * a.dim;
    const int* bt = a.block_table + (size_t)req * a.max_pages;
    // pad columns: zeros, once
    for (int e = c; e < (DP / 16 - pieces) * TK; e += 32 * H::GW) {
      const int r = e % TK, p16 = pieces + e / TK;
      for (int b = group; b < H::KST; b += H::NG)
        for (int s = 0; s < 2; ++s) {
          const int p = (p16 & 3) * 2 + s, at = (p16 >> 2) * H::SPAN + r * 128 + ((p ^ (r & 7)) << 4);
          *reinterpret_cast<uint4*>(sm.k[b] + at) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(sm.v[b] + at) = make_uint4(0, 0, 0, 0);
        }
    }
    // Lane i of a warp (i < GR, and the lanes behind them again) knows in which page group i of a block is, and then which tile of the
    // pool that is (-1: none).  The two are apart because a load that is used at once holds the warp up for its whole latency.
    const int shift = __ffs(a.page) - 1;
    auto first_of = [&](int i) { return (kb_lo + i) * TK + (lane & (GR - 1)) * BLK; };
    auto wanted = [&](int i) { return i < n_blocks && first_of(i) <= last_pos && first_of(i) + BLK > first_key; };
    auto look_up = [&](int i) {
      const int lp = first_of(i) >> shift;
      return wanted(i) && lp < a.max_pages ? bt[lp] : -1;
    };
    auto tile_of = [&](int i, int pg) {
      if (!wanted(i)) return -1;
      if (pg < 0 || pg >= a.n_pages) {
        if (c < GR) atomicOr(a.status, pg < 0 ? MLXB_ST_POSITION_RANGE : MLXB_ST_PAGE_RANGE);
        return -1;
      }
      return (pg * a.Hkv + hk) * per + ((first_of(i) & (a.page - 1)) / BLK);
    };
    // the codes of a block: what has no page is left as it is (any byte is a code, and its weight will be 0)
    auto fetch = [&](const int8_t* pool, uint8_t* dst, uint64_t* bar, int id) {
      const uint32_t have = __ballot_sync(0xffffffffu, lane < GR && id >= 0);
      if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(have) * copy));
      __syncwarp();
      if (have >> lane & 1)
        bulk_load(dst + lane * copy, pool + (size_t)(uint32_t)id * copy, (uint32_t)copy, bar);
    };
    constexpr int PIECES = DP / 16;                     // of a row at most: 8 or 4
    constexpr int N = TK * PIECES / (32 * H::GW);       // of a thread
    static_assert(N == GR, "a thread has a row of each group");
    // eight neighbouring threads take four pieces of a row and four of the next: neither their loads nor their stores meet in a bank
    const int odd = c >> 2 & 1;
    const int piece = PIECES == 8 ? (c & 3) + 4 * (odd ^ (c >> 3 & 1)) : c & 3, r_first = PIECES == 8 ? odd + 2 * (c >> 4) : c >> 2;
    const bool mine = piece < pieces;
    const int from0 = r_first * a.dim + piece * 16;
    const int place0 = (piece >> 2) * H::SPAN + r_first * 128 + ((((piece & 3) * 2) ^ (r_first & 7)) << 4);
    constexpr int AHEAD = H::NG * H::RD;
    auto bar_of = [&](uint64_t (&bars)[H::NG][H::RD], int i) { return &bars[group][i / H::NG % H::RD]; };
    auto turn_of = [&](int i) { return (uint32_t)(i / AHEAD & 1); };
    int page_next = leads ? look_up(group + AHEAD) : -1;
    int ids[H::RD];                                     // of the blocks under way
#pragma unroll
    for (int d = 0; d < H::RD; ++d) ids[d] = -1;
    float sk = 0.f, sv = 0.f;
    const int8_t *k8 = a.k8, *v8 = a.v8;
    const float *ks = a.ks, *vs = a.vs;
    int last_k = -1, last_v = -1;                       // blocks whose codes were asked for last
    if (leads) {
      int pages[H::RD];
#pragma unroll
      for (int d = 0; d < H::RD; ++d) pages[d] = look_up(group + d * H::NG);
#pragma unroll
      for (int d = 0; d < H::RD; ++d) ids[d] = tile_of(group + d * H::NG, pages[d]);
      pdl_wait();
      k8 = after_wait(a.k8), v8 = after_wait(a.v8);
      ks = after_wait(a.ks), vs = after_wait(a.vs);
#pragma unroll
      for (int d = 0; d < H::RD; ++d) {
        const int i = group + d * H::NG;
        if (i >= n_blocks) break;
        if (brings_k) {
          fetch(k8, sm.raw_k[group][d], &sm.rk_full[group][d], ids[d]);
          last_k = i;
        }
        if (d == 0 && brings_scales && lane < GR && ids[0] >= 0) { sk = __ldcg(ks + ids[0]); sv = __ldcg(vs + ids[0]); }
        if (brings_v) {
          fetch(v8, sm.raw_v[group][d], &sm.rv_full[group][d], ids[d]);
          last_v = i;
        }
      }
    }
    // A warp that gives up goes on to meet the others of its group at their barrier.
    bool ok = true;
    for (int i = group; i < n_blocks; i += H::NG) {
      const int b = i % H::KST, stage = i / H::NG % H::RD;
      const uint32_t turn = (uint32_t)((i / H::KST) & 1);
      int id = -1;
      if (leads) {
        id = tile_of(i + AHEAD, page_next);
        page_next = look_up(i + AHEAD + H::NG);
      }
      ok = ok && wait_warp(bar_of(sm.rk_full, i), turn_of(i), abort_flag);
      ok = ok && (i < H::KST || wait_warp(&sm.k_free[b], turn ^ 1u, abort_flag));
      if (ok) {
        const uint8_t* src = sm.raw_k[group][stage] + from0;
        uint8_t *dst = sm.k[b] + place0, *dst2 = sm.k[b] + (place0 ^ 16);
        if (mine) {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + n * copy);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) { y[2 * e] = masked_xor(w[e], 0x00800080u); y[2 * e + 1] = masked_xor(w[e] >> 8, 0x00800080u); }
            *reinterpret_cast<uint4*>(dst + n * BLK * 128) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(dst2 + n * BLK * 128) = make_uint4(y[4], y[5], y[6], y[7]);
          }
        }
        if (brings_scales) {
          const uint32_t gone = __ballot_sync(0xffffffffu, ids[0] < 0) & ((1u << GR) - 1);
          const uint32_t nothing = __ballot_sync(0xffffffffu, sv == 0.f) & ((1u << GR) - 1);
          if (lane < GR) {
            sm.sk[i % XR][lane] = sk;
            sm.lsv[i % XR][lane] = sv > 0.f ? log2f(sv) : 0.f;
            sm.rsv[i % XR][lane] = sv > 0.f ? 1.f / sv : 1.f;
            if (lane == 0) { sm.marks[i % XR] = gone | (nothing & ~gone) << 8; sm.nothing[group] = nothing; }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.k_full[b]);
      }
      group_sync(1 + group, 32 * H::GW);                // these codes of K were read by all
      if (brings_k && ok && i + AHEAD < n_blocks) {
        fetch(k8, sm.raw_k[group][stage], &sm.rk_full[group][stage], id);
        last_k = i + AHEAD;
      }
      if (brings_scales) {                              // of the group's next block
        sk = sv = 0.f;
        const int next = H::RD == 1 ? id : ids[H::RD - 1];
        if (lane < GR && next >= 0) { sk = __ldcg(ks + next); sv = __ldcg(vs + next); }
      }
      ok = ok && wait_warp(bar_of(sm.rv_full, i), turn_of(i), abort_flag);
      ok = ok && (i < H::KST || wait_warp(&sm.v_free[b], turn ^ 1u, abort_flag));
      if (ok) {
        const uint32_t nothing = sm.nothing[group];
        const uint8_t* src = sm.raw_v[group][stage] + from0;
        uint8_t *dst = sm.v[b] + place0, *dst2 = sm.v[b] + (place0 ^ 16);
        if (mine) {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            uint4 x = *reinterpret_cast<const uint4*>(src + n * copy);
            if (nothing >> n & 1) x = make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[2 * e] = less1152(masked_xor(w[e], 0x64806480u));
              y[2 * e + 1] = less1152(masked_xor(w[e] >> 8, 0x64806480u));
            }
            *reinterpret_cast<uint4*>(dst + n * BLK * 128) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(dst2 + n * BLK * 128) = make_uint4(y[4], y[5], y[6], y[7]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.v_full[b]);
      }
      group_sync(1 + group, 32 * H::GW);
      if (brings_v && ok && i + AHEAD < n_blocks) {
        fetch(v8, sm.raw_v[group][stage], &sm.rv_full[group][stage], id);
        last_v = i + AHEAD;
      }
#pragma unroll
      for (int d = 0; d + 1 < H::RD; ++d) ids[d] = ids[d + 1];
      ids[H::RD - 1] = id;
    }
    if (!ok) {                                 // no copy is under way when the shared memory is given up
      int never = 0;
#pragma unroll
      for (int d = 0; d < H::RD; ++d) {
        if (last_k - d * H::NG >= 0) mbar_wait_warp(bar_of(sm.rk_full, last_k - d * H::NG), turn_of(last_k - d * H::NG), &never);
        if (last_v - d * H::NG >= 0) mbar_wait_warp(bar_of(sm.rv_full, last_v - d * H::NG), turn_of(last_v - d * H::NG), &never);
      }
    }
  } else {
    registers<H::R_SOFT, H::R_LAUNCH>();
    // softmax: thread r of a head's 128 owns query row r, which is lane r of tensor memory
    const int t = warp >> 2, r = threadIdx.x & 127, h = h0 + t;
    const int pos = pos0 + r;
    const int lo = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + 2 * t * TK + lanes, t_o = tmem_o + t * DP + lanes;
    float fac, off;
    pdl_wait();
    {
      const __nv_bfloat16* qr = after_wait(a.q) + (size_t)(row0 + r) * a.ldq + (size_t)h * a.dim;
      uint32_t x[DP / 2];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < DP / 8; ++e) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < n_rows && 8 * e < a.dim) {
          if (a.vec & 1) {
            u = *reinterpret_cast<const uint4*>(qr + 8 * e);
          } else {
            const unsigned short* p = reinterpret_cast<const unsigned short*>(qr) + 8 * e;
            u = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
          }
        }
        x[4 * e] = u.x; x[4 * e + 1] = u.y; x[4 * e + 2] = u.z; x[4 * e + 3] = u.w;
      }
#pragma unroll
      for (int e = 0; e < DP / 2; ++e) top = max(top, max(x[e] << 16 & 0x7fffffffu, x[e] & 0x7fff0000u));
      const int e2 = max((int)(top >> 23) - 127, -100);
      const float up = __uint_as_float((uint32_t)(127 + 14 - e2) << 23);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < DP / 8; ++e) {
        uint32_t y[4];
#pragma unroll
        for (int w = 0; w < 2; ++w) {                   // columns 0, 2 and 1, 3 of four
          const uint32_t x0 = x[4 * e + 2 * w], x1 = x[4 * e + 2 * w + 1];
          y[2 * w] = half2_of(__uint_as_float(x0 << 16) * up, __uint_as_float(x1 << 16) * up);
          y[2 * w + 1] = half2_of(__uint_as_float(x0 & 0xffff0000u) * up, __uint_as_float(x1 & 0xffff0000u) * up);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y[w]));
          sum += f.x + f.y;
        }
        const int p = e & 7;
        *reinterpret_cast<uint4*>(sm.q[t] + (e >> 3) * H::QSPAN + r * 128 + ((p ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
      }
      off = sum * (128.f * UNIT);
      fac = __uint_as_float((uint32_t)(127 - 14 + e2) << 23) * (a.scale * LOG2E / UNIT);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[t]);
    }
    float m = -INFINITY, l = 0.f;      // the base of the exponentials, which follows the largest s + log2(sv); the sum
    float m0 = -INFINITY, l0 = 0.f;    // the maximum of s, and the sum, of groups whose values are 0
    bool ok = true;
    for (int i = 0; i < n_blocks && ok; ++i) {
      const int key0 = (kb_lo + i) * TK, x4 = i % XR;
      if (!(ok = wait_warp(&sm.s_full[t], (uint32_t)(i & 1), abort_flag))) break;
      after_sync();
      const uint32_t marks = sm.marks[x4];
      uint32_t s[TK / 32][32];
#pragma unroll
      for (int c = 0; c < TK / 32; ++c) tmem_ld32(t_s + 32 * c, s[c]);
      ld_wait(s);
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.s_read[t]);        // the next S may be formed over it
      // blocks that every row of the tile sees whole, with values in every group, need none of this
      if (marks != 0 || key0 + TK - 1 > pos0 || (a.window > 0 && key0 < last_pos - a.window + 1)) {
        const int first = lo - key0, last = pos - key0;
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) {
          const int f = first - 32 * c, e1 = last - 32 * c;
          uint32_t bits = f <= 0 ? 0xffffffffu : f > 31 ? 0u : 0xffffffffu << f;
          bits &= e1 >= 31 ? 0xffffffffu : e1 < 0 ? 0u : (2u << e1) - 1u;
          if (marks >> (2 * c) & 1) bits &= 0xffff0000u;
          if (marks >> (2 * c + 1) & 1) bits &= 0x0000ffffu;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(bits >> e & 1)) s[c][e] = 0xff800000u;          // -inf: its exponential below is 0
        }
        if (marks >> 8) {
          // groups whose values are 0: into their own sum, and out of what follows
#pragma unroll
          for (int g = 0; g < GR; ++g) {
            if (!(marks >> (8 + g) & 1)) continue;
            uint32_t* x = &s[g >> 1][16 * (g & 1)];
            const float f = fmaxf(fac * sm.sk[x4][g], 1e-30f);
            float top = __uint_as_float(x[0]);
#pragma unroll
            for (int e = 1; e < BLK; ++e) top = fmaxf(top, __uint_as_float(x[e]));
            top = fmaxf((top - off) * f, m0);
            const float base = top == -INFINITY ? 0.f : top, k = fmaf(-off, f, -base);
            l0 *= ex2(m0 - base);
            m0 = top;
#pragma unroll
            for (int e = 0; e < BLK; ++e) {
              l0 += ex2(fmaf(__uint_as_float(x[e]), f, k));
              x[e] = 0xff800000u;
            }
          }
        }
      }
      // A pass with the maximum as it is; the sums of its groups show whether it was too low (the search for the largest score would take
      // as long as a third of the exponentials).  Then, and in blocks before which a row has seen nothing, the maximum first.
      const uint32_t t_p = t_s + TK + (uint32_t)((i & 1) * (TK / 2));
      auto raise_max = [&]() {
        // UP below the largest of s + log2(sv).  In a group the scale is one number above 0 (a key scale of 0 counts as one that leaves scores of
        // next to nothing, so that -inf stays -inf), so its largest score is the largest raw score's.
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const uint32_t* x = &s[g >> 1][16 * (g & 1)];
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[e] = fmaxf(fmaxf(__uint_as_float(x[e]), __uint_as_float(x[e + 4])), fmaxf(__uint_as_float(x[e + 8]), __uint_as_float(x[e + 12])));
          const float top = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
          mx = fmaxf(mx, fmaf(top - off, fmaxf(fac * sm.sk[x4][g], 1e-30f), sm.lsv[x4][g]));
        }
        mx -= UP;
        const bool grow = mx > m;
        const float corr = grow ? ex2(m - mx) : 1.f;  // 2^-inf = 0
        if (grow) m = mx;
        l *= corr;
        if (i > 0 && __any_sync(0xffffffffu, grow)) { // O as P V of the block before leaves it
          if (!wait_warp(&sm.pv_done[t][(i - 1) & 1], (uint32_t)(((i - 1) >> 1) & 1), abort_flag)) return false;
          after_sync();
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t y[32];
            tmem_ld32(t_o + 32 * c, y);
            ld_wait(y);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t z[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) z[e] = __float_as_uint(__uint_as_float(y[16 * half + e]) * corr);
              st16(t_o + 32 * c + 16 * half, z);
            }
          }
          st_wait();
        }
        return true;
      };
      float add;
      auto weigh = [&]() {
        const float base = m == -INFINITY ? 0.f : m;
        add = 0.f;
        float top = -INFINITY;                          // the largest sum of a group's weights
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) {
          uint32_t packed[16];
#pragma unroll
          for (int gg = 0; gg < 2; ++gg) {
            const int g = 2 * c + gg;
            const float f = fmaxf(fac * sm.sk[x4][g], 1e-30f), k = fmaf(-off, f, sm.lsv[x4][g] - base);
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int e = 0; e < BLK; e += 2) {
              float p0, p1;
              fma2(p0, p1, __uint_as_float(s[c][16 * gg + e]), __uint_as_float(s[c][16 * gg + e + 1]), f, k);
              p0 = ex2(p0);
              p1 = ex2(p1);
              add2(sum0, sum1, p0, p1);
              packed[8 * gg + (e >> 1)] = half2_of(p0, p1);
            }
            sum0 += sum1;
            top = fmaxf(top, sum0);
            add = fmaf(sum0, sm.rsv[x4][g], add);
          }
          st16(t_p + 16 * c, packed);
        }
        return __any_sync(0xffffffffu, top > HIGH);
      };
      if (__any_sync(0xffffffffu, m == -INFINITY)) ok = raise_max();
      if (ok && weigh()) ok = raise_max() && (weigh(), true);
      l += add;
      if (!ok) break;
      st_wait();
      before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[t][i & 1]);
    }
    // (the products of a head are formed in order: with the last one all are there)
    if (ok) ok = wait_warp(&sm.pv_done[t][(n_blocks - 1) & 1], (uint32_t)(((n_blocks - 1) >> 1) & 1), abort_flag);
    if (ok) {
      after_sync();
      l += l0 * (m != -INFINITY ? ex2(m0 - m) : 0.f);
      if (a.sinks && m != -INFINITY) l += ex2(a.sinks[h] * LOG2E - m);
      const float inv = l != 0.f ? 1.f / l : 0.f;
      __nv_bfloat16* dst = a.out + (size_t)(row0 + r) * a.ldo + (size_t)h * a.dim;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(t_o + 32 * c, o);
        ld_wait(o);
        if (r < n_rows) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (32 * c + e >= a.dim) break;
          float y[8];
#pragma unroll
          for (int w = 0; w < 8; w += 4) {              // stored as columns 0, 2, 1, 3
            y[w] = __uint_as_float(o[e + w]) * inv;
            y[w + 2] = __uint_as_float(o[e + w + 1]) * inv;
            y[w + 1] = __uint_as_float(o[e + w + 2]) * inv;
            y[w + 3] = __uint_as_float(o[e + w + 3]) * inv;
          }
          if (a.vec & 2) {
            *reinterpret_cast<uint4*>(dst + 32 * c + e) = pack8(y);
          } else {
#pragma unroll
            for (int w = 0; w < 8; ++w) dst[32 * c + e + w] = __float2bfloat16_rn(y[w]);
          }
        }
        }
        __syncwarp();
      }
    }
  }

  before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && sm.abort_flag) atomicOr(a.status, MLXB_ST_WAIT_TIMEOUT);
  if (warp == H::SOFT + H::CONV) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(H::COLS) : "memory");
  }
}

template <int DP, int NT>
static int launch(const PortionArgs& a, int n_tiles, cudaStream_t stream) {
  constexpr size_t smem = sizeof(Smem<DP, NT>);
  static_assert((smem + 1024) * Shape<DP, NT>::CTAS <= 228 * 1024, "shared memory");
  static SharedLimit limit;
  if (cudaError_t e = limit.raise(portions_kernel<DP, NT>, smem))
    return mlxb_fail((int)e, "kv8_portions: %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
  const long long blocks = (long long)n_tiles * (a.Hq / NT);
  if (blocks > INT_MAX) return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: %d tiles of %d heads", n_tiles, a.Hq);
  launch_pdl(portions_kernel<DP, NT>, dim3((unsigned)blocks), dim3(Shape<DP, NT>::THREADS), smem, stream, a);
  return mlxb_check_launch("kv8_portions");
}

// Arguments as one record of 8-byte fields: the caller fills it in a tenth of the time that as many arguments of a call take it.
struct PortionRecord {
  const void* q;
  const int *tiles, *block_table;
  const int8_t *k8, *v8;
  const float *ks, *vs, *sinks;
  void* out;
  int* status;
  long long ldq, n_tokens, n_tiles, n_req, max_pages, n_pages, page, Hq, Hkv, dim, window, ldo;
  double scale;
};

// q, out: [n_tokens, Hq * dim] at row strides ldq, ldo; dim a multiple of 16 up to 128; scale > 0.
MLXB_EXPORT int mlxb_kv8_portions(const PortionRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(PortionRecord)) return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: a record of %lld bytes", bytes);
  const PortionRecord& x = *rec;
  const int n_tiles = (int)x.n_tiles, Hq = (int)x.Hq, Hkv = (int)x.Hkv, dim = (int)x.dim, page = (int)x.page;
  if (n_tiles <= 0) return 0;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq > 65535) return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: %d query heads over %d key/value heads", Hq, Hkv);
  if (dim % 16 || dim < 16 || dim > 128) return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: head size %d (a multiple of 16 up to 128)", dim);
  if (page < BLK || (page & (page - 1))) return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: page size %d (a power of two of at least %d)", page, BLK);
  if (!(x.scale > 0.)) return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: scale %g", x.scale);
  if (((uintptr_t)x.k8 | (uintptr_t)x.v8 | (uintptr_t)x.tiles) & 15)
    return mlxb_fail(MLXB_BAD_ARG, "kv8_portions: pools and tiles must be 16-byte aligned");
  const int vec = (x.ldq % 8 == 0 && !((uintptr_t)x.q & 15) ? 1 : 0) | (x.ldo % 8 == 0 && !((uintptr_t)x.out & 15) ? 2 : 0);
  const PortionArgs a{(const __nv_bfloat16*)x.q, (int)x.ldq, (const int4*)x.tiles, x.block_table, (int)x.n_tokens, (int)x.n_req, (int)x.max_pages, (int)x.n_pages, page, Hq,
                      Hkv, dim, (int)x.window, (float)x.scale, x.k8, x.v8, x.ks, x.vs, x.sinks, (__nv_bfloat16*)x.out, (int)x.ldo, vec,
                      x.status};
  // Two heads a CTA halve the conversions, one head a CTA fills more SMs and has an SM's arithmetic for itself: pairs where single heads
  // would be more CTAs than run at once.  256 queries of 32/8 heads of 128 at position 1000 22.8 us by single heads, 33.4 by pairs; 512 of
  // 16/4 heads of 64 at 2000 40.4 and 44.1; but 1024 of 32/8 heads of 128 at 0 (256 CTAs or 128) 32.1 and 29.5.  A row's bits are the same.
  const bool pairs = (Hq / Hkv) % 2 == 0 && (long long)n_tiles * Hq > SMS * (dim <= 64 ? Shape<64, 1>::CTAS : Shape<128, 1>::CTAS);
  if (dim <= 64) return pairs ? launch<64, 2>(a, n_tiles, stream) : launch<64, 1>(a, n_tiles, stream);
  return pairs ? launch<128, 2>(a, n_tiles, stream) : launch<128, 1>(a, n_tiles, stream);
}
