// Attention of single queries over pages in 8 bits for bfloat16 queries: the products on the tensor cores, codes turned into their
// operands in registers.  Built once for each head size (MLXB_HEAD_DIM).
//
// A block takes an item after the other, its warps a quarter of the item's keys each: asynchronous copies bring a warp's tiles into a
// ring of its own in shared memory, several ahead, the first of the next item while the warps' sums of this one come together.  Rows
// of several chunks leave sums that a second kernel adds up.
// A warp takes 16 keys at a time (a block with one scale; never more than one page) for up to eight query heads that read the same
// key/value head:
//   S^T [16 keys x 8 heads] = K [16 x dim] Q^T      m16n8k32 in whole numbers: K's codes are A as they lie in memory
//   O^T [dim x 8 heads]    += V^T [dim x 16] P^T    m16n8k16 in fp16: V's codes are A, transposed
// Which columns of K a thread's registers stand for is free as long as Q's do too, and which rows of O^T likewise, so a thread loads
// 16 neighbouring bytes of a key where it needs four times four of them.  P leaves the first product as [keys x heads] and enters the
// second as [heads x keys]: movmatrix turns it in two instructions.
// A query enters as whole numbers of 16 bits, its largest at 32512, in two products (high and low byte): a number is off by 2^-16 of the
// largest at most, the scores by 3e-5 of their spread for normal numbers, a tenth of what rounding P costs; the sums are exact.
// A code of V enters as fp16 bits 00uu, u = code + 128: the subnormal number u * 2^-24, exact, for one bit operation on two codes (two for
// the odd bytes).  The 128 comes off where the product starts: at -128 sum(p), which a product with ones gives and which is the softmax's
// sum below as well (of the weights as they were rounded).  The scale sk of a key block multiplies the scores in float32; that of a value
// block, sv, is in the exponent: P is exp(s) sv, rounded to fp16 relative to a base m that follows the largest s + log2(sv), so that what
// rounds away is small in O and not merely in weight (a first token that takes most of the weight often has values of next to nothing).
// The sum below takes P / sv, a tile at a time.  The base is set 7 below the largest (P up to 2^7) and set again once a P would pass 2^15,
// which fp16 just takes: most tiles need neither shuffles nor another scaling of O.  A P loses 2^-12 of itself down to 2^-14, below that
// 2^-25 at most: 2^-32 of the largest.  A tile of values of nothing (sv 0) adds to the sum alone, and moves the base only where
// the sum would pass 2^100.
//
// Bound by the bytes of the cache, and for few or short rows by the latencies of a part: rows, pages, tiles, sums, the join.  64 rows of up to
// 8192 positions, 32/8 heads of 128: 112 us, 5.0 TB/s (the same copies without any arithmetic: 109 to 124); one row at 131072: 56 us, 4.8 TB/s;
// 8 rows of up to 4000: 19.4; one row of 16 heads of 64 at 520: 7.0.  A chunk of at least 1024 keys leaves one row of 8192 positions with 64
// blocks (14.8 us); its four quarters as blocks of their own, joined in the same order, would give the same bits, and are not built.  What decided
// it, for the 64 rows: neighbouring heads of a page read at
// about the same time (items are numbered with the heads innermost); a chunk shared by a block's four warps instead of a warp's own (157 us:
// four times the partial sums); the next item's first tiles under way while sums are merged; the join in a kernel of its own (a block that
// finds itself the last of a row by a counter waits for a fence, an atomic and the sums in turn).  Blocks of 8 warps, two an SM, have
// longer waits at each merge: 129 us, but 13.0 instead of 14.6 for one row of 8192.  Three blocks an SM with rings of four tiles: 110, one
// row at 131072 51 us, but 31.8 instead of 26.6 for 64 rows of up to 1000, 16 heads of 64 (1024 items in rounds of 444, not 592).
#include <float.h>

#include "kv8_rows.cuh"

MLXB_DEFINE_LAST_ERROR()

#ifndef MLXB_HEAD_DIM
#define MLXB_HEAD_DIM 64
#endif
constexpr int DH = MLXB_HEAD_DIM;
static_assert(DH % 16 == 0 && DH >= 16 && DH <= 256, "head size");
constexpr int WARPS = 4;
constexpr int HT = 8;                                   // query heads of an item
constexpr int TILE = 2 * 16 * DH;                       // bytes of a tile: 16 keys, 16 values
constexpr int STAGES = 12288 / TILE < 2 ? 2 : 12288 / TILE;      // of a warp's ring
constexpr int CTAS = DH > 128 ? 3 : 4;                  // of an SM
constexpr size_t RING = (size_t)WARPS * STAGES * TILE;
constexpr int KT = DH / 16;                             // words of a key a thread holds, m tiles of O
constexpr int KS = (KT + 1) / 2;                        // k steps of S
constexpr int KW = DH % 64 == 0 ? 16 : DH % 32 == 0 ? 8 : 4;      // bytes of a key a thread loads at once
constexpr int NK = DH / 4 / KW;
constexpr int VW = DH % 128 == 0 ? 16 : DH % 64 == 0 ? 8 : DH % 32 == 0 ? 4 : 2;      // ... of a value
constexpr int NV = DH / 8 / VW;
constexpr int VR = VW >= 4 ? DH / 32 : DH / 16;         // registers of a value
constexpr float LOG2E = 1.4426950408889634f;
// log2 of the largest P: where the base of the exponentials is set anew, and at most; of the largest weight where values are nothing
constexpr float UP = 7.f, MOST = 15.f, ABOVE = 100.f;
constexpr float UNIT = 5.9604644775390625e-8f;          // 2^-24: what a code's operand counts in
constexpr uint32_t ONES = 0x3c003c00u;

// Where 16-byte piece c of row r of a tile's keys (values) lies in shared memory: so that the eight lanes of a wide load meet in no
// bank.  A key load's lanes stand on rows r, r + 1 (four neighbouring pieces each), a value load's on rows 0, 2, 4, 6 of the same one or
// two pieces.
__device__ __forceinline__ int key_at(int r, int c) {
  if constexpr (DH % 128 == 0) return r * DH + ((c ^ ((r & 1) << 2)) << 4);
  return r * DH + (c << 4);
}
__device__ __forceinline__ int value_at(int r, int c) {
  if constexpr (DH % 128 == 0) return r * DH + ((c ^ (((r >> 1) & 3) << 1)) << 4);
  if constexpr (DH == 64) {
    const int s = (r >> 1) | ((r & 1) << 3);
    return s * DH + ((c ^ (s & 2)) << 4);
  }
  return r * DH + (c << 4);
}
template <int W>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* r) {
  if constexpr (W == 16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
  } else if constexpr (W == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r[0] = u.x; r[1] = u.y;
  } else if constexpr (W == 4) {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    r[0] = *reinterpret_cast<const unsigned short*>(p);
  }
}
__device__ __forceinline__ void copy16(uint32_t dst, const int8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Bytes 0 and 2 (1 and 3) of w, each + 128, as the low bits of two fp16: (code + 128) * 2^-24, exact (a subnormal number).
__device__ __forceinline__ uint32_t even(uint32_t w) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(y) : "r"(w), "r"(0x00ff00ffu), "r"(0x00800080u));      // (a & b) ^ c
  return y;
}
__device__ __forceinline__ uint32_t odd(uint32_t w) { return even(w >> 8); }
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                    float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// whole numbers: 16 x 32 codes by 32 x 8
__device__ __forceinline__ void imma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

constexpr int PART = 8 * (DH + 2);                      // floats of an item's sums: m[8], l[8], then O as the lanes hold it

// A sum for those that multiply it by weights, some of them 0: of values around 2^-100 it may pass the range of float32.
__device__ __forceinline__ float in_range(float x) { return x == INFINITY ? FLT_MAX : x; }

__device__ __forceinline__ int column_of(int c, int g) { return (c / VW * 8 + g) * VW + c % VW; }      // column c of lane group g's

// An item and a warp's share of it.
struct Job {
  Item x;
  int hk, h0, nh, first, mine;                          // key/value head, first query head, how many; first key and number of tiles
  uint32_t tile_id, missing;
  float sk, sv;
};

__global__ void __launch_bounds__(WARPS * 32, CTAS)
rows_tc_kernel(const RowsArgs a, int tiles, int group_tiles, int q_vec) {
  extern __shared__ __align__(128) uint8_t ring[];      // the warps' tiles, then what is kept of the rows
  __shared__ int warp_sums[WARPS], sm_spare[WARPS];
  __shared__ float sm_m[WARPS][HT], sm_l[WARPS][HT];
  const Rows rows(reinterpret_cast<int*>(ring + RING), a.n_rows);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int total = schedule(a, rows, warp_sums) * tiles;
  const int G = a.Hq / a.Hkv, per = a.page / BLK;
  uint8_t* my_ring = ring + warp * (STAGES * TILE);
  const uint32_t my_ring_u32 = (uint32_t)__cvta_generic_to_shared(my_ring);
  pdl_wait();
  pdl_trigger();
  // where this lane's pieces of a tile lie, the same for every tile
  const int key_base = key_at(g, (t * KW) >> 4) + ((t * KW) & 15), key_other = DH % 128 == 0 ? key_base ^ 64 : key_base + 4 * KW;
  const int value_base = value_at(2 * t, (g * VW) >> 4) + ((g * VW) & 15);
  const int8_t *k8 = after_wait(a.k8), *v8 = after_wait(a.v8);
  const float *ks = after_wait(a.ks), *vs = after_wait(a.vs);
  Job job;
  // lane i learns of the i-th of the warp's next 32 tiles which tile of the pool it is, and its scales; missing: tiles without a page
  auto look_up = [&](Job& b, int i0) {
    const int i = i0 + lane, key = b.first + i * BLK;
    bool none = false;
    if (i < b.mine) {
      const int pg = page_of(a, a.block_table + (size_t)b.x.row.req * a.max_pages, key);
      none = pg < 0;
      if (!none) {
        b.tile_id = (uint32_t)(pg * a.Hkv + b.hk) * per + (key & (a.page - 1)) / BLK;
        b.sk = __ldcg(ks + b.tile_id);
        b.sv = __ldcg(vs + b.tile_id);
      }
    }
    b.missing = __ballot_sync(0xffffffffu, none);
  };
  // tile i of the n looked up, on its way into stage st; a group of copies for every tile, an empty one where there is none
  auto fetch = [&](const Job& b, int i, int n, int st) {
    if (i < n && !(b.missing >> i & 1)) {
      const size_t at = (size_t)__shfl_sync(0xffffffffu, b.tile_id, i) * (16 * DH) + lane * 16;
      const uint32_t dst = my_ring_u32 + st * TILE;
#pragma unroll
      for (int e0 = 0; e0 < DH; e0 += 32) {
        const int e = e0 + lane, row = e / (DH / 16), c = e % (DH / 16);
        if (DH % 32 == 0 || e < DH) {
          copy16(dst + key_at(row, c), k8 + at + e0 * 16);
          copy16(dst + 16 * DH + value_at(row, c), v8 + at + e0 * 16);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int st = 0;                                           // the stage of the warp's next tile
  // the first tiles of an item: all stages but the one before st
  auto begin = [&](Job& b, int it) {
    b.x = item_of(a, rows, it, tiles);
    b.hk = b.x.tile / group_tiles;
    const int j0 = (b.x.tile - b.hk * group_tiles) * HT;
    b.nh = min(HT, G - j0);
    b.h0 = b.hk * G + j0;
    // a quarter of the item's tiles each
    const int n = (b.x.end - b.x.begin + BLK - 1) / BLK, each = (n + WARPS - 1) / WARPS;
    b.first = b.x.begin + warp * each * BLK;
    b.mine = max(0, min(each, n - warp * each));
    look_up(b, 0);
    for (int i = 0, s = st; i < STAGES - 1; ++i, s = s + 1 == STAGES ? 0 : s + 1) fetch(b, i, min(32, b.mine), s);
  };
  int it = blockIdx.x;
  if (it < total) begin(job, it);
  while (it < total) {
    const int h0 = job.h0, nh = job.nh, n_tiles = job.mine;
    const Item& x = job.x;
    const int lo = a.window > 0 ? x.row.pos - a.window + 1 : 0;

    // The queries of head g, columns (i * 4 + t) * KW .., as 256 * high + low with the largest at 32512.
    uint32_t qh[KS][2], ql[KS][2];
    float fac;
    {
      const __nv_bfloat16* qr = after_wait((const __nv_bfloat16*)a.q) + (size_t)x.row.tok * a.ldq + (size_t)(h0 + g) * DH;
      float v[KT][4];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const int c = (j / (KW / 4) * 4 + t) * KW + j % (KW / 4) * 4;
        if (g < nh) {
          if (q_vec) {
            const uint2 u = *reinterpret_cast<const uint2*>(qr + c);
            v[j][0] = __uint_as_float(u.x << 16);
            v[j][1] = __uint_as_float(u.x & 0xffff0000u);
            v[j][2] = __uint_as_float(u.y << 16);
            v[j][3] = __uint_as_float(u.y & 0xffff0000u);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = to_f(qr[c + e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[j][e]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // a query that is not finite: scores of NaN; one of next to nothing: scores of 0
      const float largest = __uint_as_float(top);
      const bool fine = top < 0x7f800000u && top >= 0x0d800000u;        // 2^-100
      const float up = fine ? 32512.f / largest : 0.f;
      fac = top >= 0x7f800000u ? NAN : fine ? largest / 32512.f * (a.scale * LOG2E) : 0.f;
#pragma unroll
      for (int j = 0; j < KS * 2; ++j) {
        uint32_t high = 0, low = 0;
        if (j < KT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // 1.5 * 2^23 + n: n's two's complement in the low bits
            const int n = (int)(__float_as_uint(fmaf(v[j < KT ? j : 0][e], up, 12582912.f)) << 16) >> 16;
            const int h = (n + 128) >> 8;
            high |= (uint32_t)(h & 0xff) << (8 * e);
            low |= (uint32_t)(n & 0xff) << (8 * e);
          }
        }
        qh[j >> 1][j & 1] = high;
        ql[j >> 1][j & 1] = low;
      }
    }
    const float fac0 = __shfl_sync(0xffffffffu, fac, 8 * t), fac1 = __shfl_sync(0xffffffffu, fac, 8 * t + 4);      // of heads 2t, 2t + 1

    float o[KT][4];
#pragma unroll
    for (int j = 0; j < KT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float lsv_of = 0.f, rsv_of = 0.f;                   // of the tiles looked up: log2 and reciprocal of the value scale (0, 0: values of nothing)

    auto work = [&](int i, int i32, int st) {           // tile i, the i32-th of those looked up
      if (job.missing >> i32 & 1) return;
      const float sk = __shfl_sync(0xffffffffu, job.sk, i32), lsv = __shfl_sync(0xffffffffu, lsv_of, i32);
      const float rsv = __shfl_sync(0xffffffffu, rsv_of, i32);
      const uint8_t* kp = my_ring + st * TILE;
      const uint8_t* vp = kp + 16 * DH + value_base;
      uint32_t fk[2][KT];
#pragma unroll
      for (int i2 = 0; i2 < NK; ++i2) {
        const uint8_t* p = DH % 128 == 0 ? kp + (i2 & 1 ? key_other : key_base) + (i2 >> 1) * 128 : kp + key_base + i2 * 4 * KW;
        load_bytes<KW>(p, &fk[0][i2 * (KW / 4)]);
        load_bytes<KW>(p + 8 * DH, &fk[1][i2 * (KW / 4)]);
      }
      int c[4] = {0, 0, 0, 0}, c2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const bool pair = 2 * j + 1 < KT;
        const uint32_t a2 = pair ? fk[0][pair ? 2 * j + 1 : 0] : 0u, a3 = pair ? fk[1][pair ? 2 * j + 1 : 0] : 0u;
        imma(c, fk[0][2 * j], fk[1][2 * j], a2, a3, qh[j][0], qh[j][1]);
        imma(c2, fk[0][2 * j], fk[1][2 * j], a2, a3, ql[j][0], ql[j][1]);
      }
      // s + log2(sv) of keys g and g + 8, heads 2t and 2t + 1, in units of log2 (the sums stay below 2^31 for heads of up to 256)
      const float a0 = sk * fac0, a1 = sk * fac1;
      float s0 = fmaf((float)(c[0] * 256 + c2[0]), a0, lsv), s1 = fmaf((float)(c[1] * 256 + c2[1]), a1, lsv);
      float s2 = fmaf((float)(c[2] * 256 + c2[2]), a0, lsv), s3 = fmaf((float)(c[3] * 256 + c2[3]), a1, lsv);
      if (i == 0 || i == n_tiles - 1) {                 // (a window begins in a row's first tile)
        const int key = job.first + i * BLK;
        const bool in = key + g >= lo && key + g < x.end, in8 = key + g + 8 >= lo && key + g + 8 < x.end;
        if (!in) s0 = s1 = -INFINITY;
        if (!in8) s2 = s3 = -INFINITY;
      }
      if (__any_sync(0xffffffffu, rsv == 0.f || s0 > m0 + MOST || s2 > m0 + MOST || s1 > m1 + MOST || s3 > m1 + MOST)) {
        float t0 = fmaxf(s0, s2), t1 = fmaxf(s1, s3);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        const float above = rsv == 0.f ? ABOVE : UP;
        t0 = fmaxf(t0 - above, m0);
        t1 = fmaxf(t1 - above, m1);
        const float r0 = ex2(m0 - (t0 == -INFINITY ? 0.f : t0)), r1 = ex2(m1 - (t1 == -INFINITY ? 0.f : t1));
        m0 = t0;
        m1 = t1;
        l0 *= r0;
        l1 *= r1;
#pragma unroll
        for (int j = 0; j < KT; ++j) { o[j][0] *= r0; o[j][1] *= r1; o[j][2] *= r0; o[j][3] *= r1; }
        if (rsv == 0.f) {
          const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
          float y0 = ex2(s0 - b0) + ex2(s2 - b0), y1 = ex2(s1 - b1) + ex2(s3 - b1);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            y0 += __shfl_xor_sync(0xffffffffu, y0, d);
            y1 += __shfl_xor_sync(0xffffffffu, y1, d);
          }
          l0 += y0;
          l1 += y1;
          return;
        }
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      const float p0 = ex2(s0 - b0), p1 = ex2(s1 - b1), p2 = ex2(s2 - b0), p3 = ex2(s3 - b1);
      const uint32_t pb0 = turned(pack_half2(p0, p1)), pb1 = turned(pack_half2(p2, p3));
      float sum[4];                                     // of the weights as they were rounded, in every row
      mma(sum, ONES, ONES, ONES, ONES, pb0, pb1, 0.f, 0.f, 0.f, 0.f);
      l0 = fmaf(sum[0], rsv, l0);
      l1 = fmaf(sum[1], rsv, l1);
      const float n0 = sum[0] * (-128.f * UNIT), n1 = sum[1] * (-128.f * UNIT);
      uint32_t fv[4][VR];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i2 = 0; i2 < NV; ++i2) {
          // row 2t + (j & 1) + 8 (j >> 1): the same pieces of it as of row 2t
          const int at = DH == 64 ? (4 * (j >> 1) + 8 * (j & 1)) * DH : ((j & 1) + (j >> 1) * 8) * DH;
          load_bytes<VW>(vp + at + i2 * 8 * VW, &fv[j][VW >= 4 ? i2 * (VW / 4) : i2]);
        }
      }
#pragma unroll
      for (int w = 0; w < VR; ++w) {
        constexpr int PER = VW >= 4 ? 2 : 1;            // m tiles of a register: columns (0, 1) of two keys, then (2, 3)
#pragma unroll
        for (int r = 0; r < PER; ++r) {
          const uint32_t x01 = __byte_perm(fv[0][w], fv[1][w], r ? 0x7632 : 0x5410);
          const uint32_t x23 = __byte_perm(fv[2][w], fv[3][w], r ? 0x7632 : 0x5410);
          float d[4];
          mma(d, even(x01), odd(x01), even(x23), odd(x23), pb0, pb1, n0, n1, n0, n1);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[PER * w + r][e] += d[e];
        }
      }
    };
    for (int i0 = 0; i0 < n_tiles; i0 += 32) {
      const int n = min(32, n_tiles - i0);
      if (i0 > 0) {
        look_up(job, i0);
        for (int i = 0, s = st; i < STAGES - 1; ++i, s = s + 1 == STAGES ? 0 : s + 1) fetch(job, i, n, s);
      }
      // (here, behind the first copies: the scales are on their way as long as the tiles)
      lsv_of = job.sv > 0.f ? __log2f(job.sv) : 0.f;
      rsv_of = job.sv > 0.f ? __fdividef(1.f, job.sv) : 0.f;
      for (int i = 0; i < n; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                                   // every lane's copies of tile i are there, and tile i - 1 has been read
        fetch(job, i + STAGES - 1, n, st == 0 ? STAGES - 1 : st - 1);
        work(i0 + i, i, st);
        st = st + 1 == STAGES ? 0 : st + 1;
      }
    }
    __syncwarp();
    // the next item's first tiles are on their way while the warps' sums come together in the stage that they leave free
    const Item done = job.x;
    it += gridDim.x;
    if (it < total) begin(job, it);
    const int spare = st == 0 ? STAGES - 1 : st - 1;
    float4* mine4 = reinterpret_cast<float4*>(my_ring + spare * TILE);
#pragma unroll
    for (int j = 0; j < KT; ++j) mine4[j * 32 + lane] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
    if (g == 0) {
      sm_m[warp][2 * t] = m0; sm_m[warp][2 * t + 1] = m1;
      sm_l[warp][2 * t] = in_range(l0); sm_l[warp][2 * t + 1] = in_range(l1);
    }
    if (lane == 0) sm_spare[warp] = warp * (STAGES * TILE) + spare * TILE;
    __syncthreads();
    {
      float w0[WARPS], w1[WARPS], tot0 = 0.f, tot1 = 0.f;      // of heads 2t, 2t + 1
      float top0 = sm_m[0][2 * t], top1 = sm_m[0][2 * t + 1];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) { top0 = fmaxf(top0, sm_m[w][2 * t]); top1 = fmaxf(top1, sm_m[w][2 * t + 1]); }
      const float b0 = top0 == -INFINITY ? 0.f : top0, b1 = top1 == -INFINITY ? 0.f : top1;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        w0[w] = ex2(sm_m[w][2 * t] - b0);
        w1[w] = ex2(sm_m[w][2 * t + 1] - b1);
        tot0 = fmaf(w0[w], sm_l[w][2 * t], tot0);
        tot1 = fmaf(w1[w], sm_l[w][2 * t + 1], tot1);
      }
      const bool one = 2 * t < nh, two = 2 * t + 1 < nh;
      float* part = a.partial + (((size_t)done.index * tiles + done.tile) * a.most_chunks + done.chunk) * PART;
      if (done.n_chunks > 1 && threadIdx.x < 4) {
        reinterpret_cast<float2*>(part)[t] = make_float2(top0, top1);
        reinterpret_cast<float2*>(part + 8)[t] = make_float2(in_range(tot0), in_range(tot1));
      }
      if (done.n_chunks == 1) {
        if (a.sinks) {
          if (one) tot0 += ex2(a.sinks[h0 + 2 * t] * LOG2E - b0);
          if (two) tot1 += ex2(a.sinks[h0 + 2 * t + 1] * LOG2E - b1);
        }
        tot0 = tot0 != 0.f ? 1.f / (tot0 * UNIT) : 0.f;
        tot1 = tot1 != 0.f ? 1.f / (tot1 * UNIT) : 0.f;
      }
      __nv_bfloat16* out = (__nv_bfloat16*)a.out + (size_t)done.row.tok * a.ldo + (size_t)(h0 + 2 * t) * DH;
      for (int j = warp; j < KT; j += WARPS) {
        if (!one) continue;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 v = reinterpret_cast<const float4*>(ring + sm_spare[w])[j * 32 + lane];
          y.x = fmaf(w0[w], v.x, y.x); y.y = fmaf(w1[w], v.y, y.y); y.z = fmaf(w0[w], v.z, y.z); y.w = fmaf(w1[w], v.w, y.w);
        }
        if (done.n_chunks > 1) {
          __stcg(reinterpret_cast<float4*>(part + 16) + j * 32 + lane, y);
        } else {
          const int d0 = column_of(2 * j, g), d1 = column_of(2 * j + 1, g);
          out[d0] = __float2bfloat16_rn(y.x * tot0);
          out[d1] = __float2bfloat16_rn(y.z * tot0);
          if (two) {
            out[DH + d0] = __float2bfloat16_rn(y.y * tot1);
            out[DH + d1] = __float2bfloat16_rn(y.w * tot1);
          }
        }
      }
    }
    __syncthreads();
  }
}

constexpr int JOIN = 8;                                 // warps of a block that joins

// The sums of a row's chunks, added in the order of `runs` runs of chunks (1, 2, 4 or 8: few chunks make few blocks, many are read in
// parallel).  A block has JOIN / runs pairs of eight columns of a (row, tile of heads), a warp one pair of them and one run.  The first O
// of a run are on their way with the maxima and sums: one latency, not three, where a run is short.
__global__ void __launch_bounds__(32 * JOIN)
rows_tc_join_kernel(const RowsArgs a, int tiles, int group_tiles, int runs) {
  extern __shared__ float weights[];                    // [chunk][8]
  __shared__ float red[JOIN][8], red2[JOIN][8];
  __shared__ float4 sums[JOIN][32];
  constexpr int EARLY = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & 3, pairs = JOIN / runs;
  const int i = blockIdx.x / tiles, tile = blockIdx.x - i * tiles, run = warp / pairs, j = blockIdx.y * pairs + warp - run * pairs;
  const RowSpan row = row_span(a, i);
  const int n = chunks_of(a, row.n);
  pdl_wait();
  pdl_trigger();
  if (n <= 1) return;
  const int hk = tile / group_tiles, G = a.Hq / a.Hkv, j0 = (tile - hk * group_tiles) * HT, nh = min(HT, G - j0), h0 = hk * G + j0;
  const float* all = after_wait(a.partial) + (size_t)blockIdx.x * a.most_chunks * PART;
  const bool mine = 2 * t < nh && j < KT;
  const int each = (n + runs - 1) / runs, c0 = run * each, c1 = min(n, c0 + each);
  auto o_of = [&](int c) { return __ldcg(reinterpret_cast<const float4*>(all + (size_t)c * PART + 16) + j * 32 + lane); };
  float4 early[EARLY];
#pragma unroll
  for (int e = 0; e < EARLY; ++e) early[e] = mine && c0 + e < c1 ? o_of(c0 + e) : make_float4(0.f, 0.f, 0.f, 0.f);
  const int h = threadIdx.x & 7, first = threadIdx.x >> 3;
  const float l_first = first < n ? __ldcg(all + (size_t)first * PART + 8 + h) : 0.f;
  float top = -INFINITY;
  bool odd = false;                                     // fmaxf leaves NaN out
  for (int c = first; c < n; c += 4 * JOIN) {
    const float m = __ldcg(all + (size_t)c * PART + h);
    weights[c * 8 + h] = m;
    odd |= m != m;
    top = fmaxf(top, m);
  }
  if (odd) top = INFINITY;                              // inf - inf below: NaN for the whole head
#pragma unroll
  for (int d = 8; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane < 8) red[warp][lane] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JOIN; ++w) top = fmaxf(top, red[w][h]);
  if (top == -INFINITY) top = 0.f;                      // no key at all has a page: zeros
  float total = 0.f;
  for (int c = first; c < n; c += 4 * JOIN) {
    const float w = ex2(weights[c * 8 + h] - top);
    weights[c * 8 + h] = w;
    total = fmaf(w, c == first ? l_first : __ldcg(all + (size_t)c * PART + 8 + h), total);
  }
  // the sink's term by lanes that all of a head share: into the first warp's sum
  if (a.sinks && threadIdx.x < 8 && h < nh) total += ex2(a.sinks[h0 + h] * LOG2E - top);
#pragma unroll
  for (int d = 8; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  if (lane < 8) red2[warp][lane] = total;
  __syncthreads();
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine) {
    auto add = [&](int c, const float4& v) {
      const float2 w = *reinterpret_cast<const float2*>(weights + c * 8 + 2 * t);
      s.x = fmaf(w.x, v.x, s.x); s.y = fmaf(w.y, v.y, s.y); s.z = fmaf(w.x, v.z, s.z); s.w = fmaf(w.y, v.w, s.w);
    };
#pragma unroll
    for (int e = 0; e < EARLY; ++e)
      if (c0 + e < c1) add(c0 + e, early[e]);
#pragma unroll 4
    for (int c = c0 + EARLY; c < c1; ++c) add(c, o_of(c));
  }
  if (runs > 1) {
    sums[warp][lane] = s;
    __syncthreads();
    if (run) return;
    for (int w = warp + pairs; w < JOIN; w += pairs) {
      const float4 v = sums[w][lane];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  if (!mine) return;
  float l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int w = 0; w < JOIN; ++w) { l0 += red2[w][2 * t]; l1 += red2[w][2 * t + 1]; }
  l0 = l0 != 0.f ? 1.f / (l0 * UNIT) : 0.f;
  l1 = l1 != 0.f ? 1.f / (l1 * UNIT) : 0.f;
  __nv_bfloat16* out = (__nv_bfloat16*)a.out + (size_t)row.tok * a.ldo + (size_t)(h0 + 2 * t) * DH;
  const int lo = column_of(2 * j, lane >> 2), hi = column_of(2 * j + 1, lane >> 2);
  out[lo] = __float2bfloat16_rn(s.x * l0);
  out[hi] = __float2bfloat16_rn(s.z * l0);
  if (2 * t + 1 < nh) {
    out[DH + lo] = __float2bfloat16_rn(s.y * l1);
    out[DH + hi] = __float2bfloat16_rn(s.w * l1);
  }
}

// As mlxb_kv8_rows for bfloat16 and heads of MLXB_HEAD_DIM; tiles of eight query heads: partial n_rows * tiles * most_chunks * 8 *
// (dim + 2) floats, counters n_rows * tiles (tiles: Hkv * ceil(Hq / Hkv / 8)).
MLXB_EXPORT int mlxb_kv8_rows_tc(const RowsRecord* rec, long long bytes, cudaStream_t stream) {
  RowsArgs a;
  if (int e = rows_args(rec, bytes, "kv8_rows_tc", a)) return e;
  if (a.n_rows <= 0) return 0;
  if (a.dim != DH) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: head size %d, this library is for %d", a.dim, DH);
  const int Hq = a.Hq, Hkv = a.Hkv, n_rows = a.n_rows, most_chunks = a.most_chunks;
  const int group_tiles = (Hq / Hkv + HT - 1) / HT, tiles = Hkv * group_tiles;
  const size_t smem = RING + rows_bytes(n_rows);
  const long long most = (long long)n_rows * most_chunks * tiles, fill = (long long)CTAS * mlxb_sm_count();
  static SharedLimit limit;
  if (cudaError_t e = limit.raise(rows_tc_kernel, RING + rows_bytes(ROWS_MOST)))
    return mlxb_fail((int)e, "kv8_rows_tc: shared memory: %s", cudaGetErrorString(e));
  launch_pdl(rows_tc_kernel, dim3((unsigned)(most < fill ? most : fill)), dim3(WARPS * 32), smem, stream, a, tiles, group_tiles,
             (a.ldq % 4 == 0 && !((uintptr_t)a.q & 7)) ? 1 : 0);
  if (int e = mlxb_check_launch("kv8_rows_tc")) return e;
  if (most_chunks == 1) return 0;
  int runs = 1;                                         // eight chunks at once, then more warps
  while (runs < JOIN && runs * 8 < most_chunks) runs *= 2;
  launch_pdl(rows_tc_join_kernel, dim3((unsigned)n_rows * tiles, (KT * runs + JOIN - 1) / JOIN), dim3(32 * JOIN), (size_t)most_chunks * 32, stream,
             a, tiles, group_tiles, runs);
  return mlxb_check_launch("kv8_rows_tc (join)");
}
