// Attention of single queries over pages in 8 bits for bfloat16 queries: the products on the tensor cores, the keys and values of a
// tile straight from memory into the registers that the products take.  Built once for each head size (MLXB_HEAD_DIM).
//
// A warp takes 16 keys at a time (a block with one scale; never more than one page) for up to eight query heads that read the same
// key/value head, as m16n8k16 products:
//   S^T [16 keys x 8 heads] = K [16 x dim] Q^T      the codes are A, row by row
//   O^T [dim x 8 heads]    += V^T [dim x 16] P^T    the codes are A again, transposed
// Which columns of K a thread's registers stand for is free as long as Q's do too, and which rows of O^T likewise, so a thread loads
// 16 neighbouring bytes of a key where it needs four times four of them, and nothing goes through shared memory.  P leaves the first
// product as [keys x heads] and enters the second as [heads x keys]: movmatrix turns it in two instructions.
// Codes become fp16: the code + 128 in the low byte of 1024 (one byte permutation for two), less 1152, both exact.  A query is scaled by
// a power of two so that its largest number lies in [2^14, 2^15): its 8 bits stay exact in fp16 down to 2^-28 of the largest.  The
// scale of a key block multiplies the scores, the scale of a value block the block's O, both in float32; P is rounded to fp16 (11
// bits, 2^-12 of a weight).  The maximum that the exponentials are relative to follows a score only once that is more than 8 (a factor
// 256) beyond it: all scores of a row stay below 2^8 in P, and most tiles need neither shuffles nor another scaling of O.
#include "kv8_rows.cuh"

MLXB_DEFINE_LAST_ERROR()

#ifndef MLXB_HEAD_DIM
#define MLXB_HEAD_DIM 64
#endif
constexpr int DH = MLXB_HEAD_DIM;
static_assert(DH % 16 == 0 && DH >= 16 && DH <= 256, "head size");
constexpr int WARPS = 4;
constexpr int HT = 8;                                   // query heads of an item
constexpr int CTAS = DH > 128 ? 2 : 3;                  // of an SM
constexpr int KT = DH / 16;                             // k steps of S, m tiles of O
constexpr int KW = DH % 64 == 0 ? 16 : DH % 32 == 0 ? 8 : 4;      // bytes of a key a thread loads at once
constexpr int NK = DH / 4 / KW;
constexpr int VW = DH % 128 == 0 ? 16 : DH % 64 == 0 ? 8 : DH % 32 == 0 ? 4 : 2;      // ... of a value
constexpr int NV = DH / 8 / VW;
constexpr int VR = VW >= 4 ? DH / 32 : DH / 16;         // registers of a value
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 8.f;

struct Tile { uint32_t k[2][KT], v[4][VR]; };

template <int W>
__device__ __forceinline__ void load_bytes(const int8_t* p, uint32_t* r) {
  if constexpr (W == 16) {
    const uint4 u = __ldcg(reinterpret_cast<const uint4*>(p));
    r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
  } else if constexpr (W == 8) {
    const uint2 u = __ldcg(reinterpret_cast<const uint2*>(p));
    r[0] = u.x; r[1] = u.y;
  } else if constexpr (W == 4) {
    r[0] = __ldcg(reinterpret_cast<const uint32_t*>(p));
  } else {
    r[0] = __ldcg(reinterpret_cast<const unsigned short*>(p));
  }
}
// two codes + 128 (bytes a and b of w) as fp16
template <int SEL>
__device__ __forceinline__ uint32_t half2_of(uint32_t w) {
  const uint32_t x = __byte_perm(w, 0x64646464u, SEL);
  uint32_t y;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
  return y;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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

__global__ void __launch_bounds__(WARPS * 32, CTAS)
rows_tc_kernel(const RowsArgs a, int tiles, int group_tiles, int q_vec) {
  extern __shared__ int dyn[];                          // prefix sums, then the weights of the last step
  __shared__ int warp_sums[WARPS], last;
  __shared__ float sm_m[WARPS][HT], sm_l[WARPS][HT], fin_m[HT], fin_l[HT];
  __shared__ float sm_o[WARPS][HT * DH];
  int* prefix = dyn;
  float* weights = reinterpret_cast<float*>(dyn + a.n_rows + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int total = schedule(a, prefix, warp_sums) * tiles;
  const int G = a.Hq / a.Hkv, per = a.page / BLK;
  pdl_wait();
  pdl_trigger();
  const int8_t *k8 = after_wait(a.k8), *v8 = after_wait(a.v8);
  const float *ks = after_wait(a.ks), *vs = after_wait(a.vs);
  for (int it = blockIdx.x; it < total; it += gridDim.x) {
    const Item x = item_of(a, prefix, it, tiles);
    const int hk = x.tile / group_tiles, j0 = (x.tile - hk * group_tiles) * HT, nh = min(HT, G - j0), h0 = hk * G + j0;
    const int* bt = a.block_table + (size_t)x.row.req * a.max_pages;
    const int lo = a.window > 0 ? x.row.pos - a.window + 1 : 0;
    const int n_tiles = (x.end - x.begin + BLK - 1) / BLK;        // of the item; this warp's: warp, warp + 4, ...

    // lane i knows the page, row and scales of the warp's i-th tile of the next 32
    int pg_row = -1;                                    // page * page rows + row of the tile in its page, head 0; -1: no page
    float skl = 0.f, svl = 0.f;
    int pg_id = 0;
    auto look_up = [&](int i0) {
      const int i = warp + WARPS * (i0 + lane), key = x.begin + i * BLK;
      pg_row = -1;
      if (i < n_tiles) {
        pg_id = page_of(a, bt, key);
        if (pg_id >= 0) {
          const int r = key & (a.page - 1);
          pg_row = r;
          const size_t at = ((size_t)pg_id * a.Hkv + hk) * per + r / BLK;
          skl = __ldcg(ks + at);
          svl = __ldcg(vs + at);
        }
      }
    };
    look_up(0);
    auto fetch = [&](int i, Tile& f) {                  // tile i of the 32 looked up
      const int r = __shfl_sync(0xffffffffu, pg_row, i), id = __shfl_sync(0xffffffffu, pg_id, i);
      if (r < 0) return;
      const size_t at = (((size_t)id * a.Hkv + hk) * a.page + r) * DH;
      const int8_t* kp = k8 + at + (size_t)g * DH + t * KW;
#pragma unroll
      for (int i2 = 0; i2 < NK; ++i2) {
        load_bytes<KW>(kp + i2 * 4 * KW, &f.k[0][i2 * (KW / 4)]);
        load_bytes<KW>(kp + 8 * DH + i2 * 4 * KW, &f.k[1][i2 * (KW / 4)]);
      }
      const int8_t* vp = v8 + at + (size_t)(2 * t) * DH + g * VW;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i2 = 0; i2 < NV; ++i2)
          load_bytes<VW>(vp + ((j & 1) + (j >> 1) * 8) * DH + i2 * 8 * VW, &f.v[j][VW >= 4 ? i2 * (VW / 4) : i2]);
      }
    };
    Tile buf[2];
    const int mine = n_tiles > warp ? (n_tiles - warp + WARPS - 1) / WARPS : 0;
    if (mine > 0) fetch(0, buf[0]);

    // the queries of head g: columns (i * 4 + t) * KW ..
    uint32_t qf[KT][2];
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
      const int e2 = max((int)(top >> 23) - 127, -100);           // the exponent of the largest
      const float up = __uint_as_float((uint32_t)(127 + 14 - e2) << 23);
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        qf[j][0] = pack_half2(v[j][0] * up, v[j][1] * up);
        qf[j][1] = pack_half2(v[j][2] * up, v[j][3] * up);
      }
      fac = __uint_as_float((uint32_t)(127 - 14 + e2) << 23) * (a.scale * LOG2E);
    }
    const float fac0 = __shfl_sync(0xffffffffu, fac, 8 * t), fac1 = __shfl_sync(0xffffffffu, fac, 8 * t + 4);      // of heads 2t, 2t + 1

    float o[KT][4];
#pragma unroll
    for (int j = 0; j < KT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    auto work = [&](int i, int i32, const Tile& f) {    // the warp's tile i, the i32-th of those looked up
      if (__shfl_sync(0xffffffffu, pg_row, i32) < 0) return;
      const float sk = __shfl_sync(0xffffffffu, skl, i32), sv = __shfl_sync(0xffffffffu, svl, i32);
      const int key = x.begin + (warp + WARPS * i) * BLK;
      float c[4] = {0.f, 0.f, 0.f, 0.f}, c2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const uint32_t u = f.k[0][j] ^ 0x80808080u, w = f.k[1][j] ^ 0x80808080u;
        mma(j & 1 ? c2 : c, half2_of<0x5140>(u), half2_of<0x5140>(w), half2_of<0x5342>(u), half2_of<0x5342>(w), qf[j][0], qf[j][1]);
      }
      // scores of keys g and g + 8, heads 2t and 2t + 1, in units of log2
      const float a0 = sk * fac0, a1 = sk * fac1;
      float s0 = (c[0] + c2[0]) * a0, s1 = (c[1] + c2[1]) * a1, s2 = (c[2] + c2[2]) * a0, s3 = (c[3] + c2[3]) * a1;
      if (key < lo || key + BLK > x.end) {
        const bool in = key + g >= lo && key + g < x.end, in8 = key + g + 8 >= lo && key + g + 8 < x.end;
        if (!in) s0 = s1 = -INFINITY;
        if (!in8) s2 = s3 = -INFINITY;
      }
      if (__any_sync(0xffffffffu, s0 > m0 + SLACK || s2 > m0 + SLACK || s1 > m1 + SLACK || s3 > m1 + SLACK)) {
        float t0 = fmaxf(s0, s2), t1 = fmaxf(s1, s3);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        t0 = fmaxf(t0, m0);
        t1 = fmaxf(t1, m1);
        const float r0 = ex2(m0 - (t0 == -INFINITY ? 0.f : t0)), r1 = ex2(m1 - (t1 == -INFINITY ? 0.f : t1));
        m0 = t0;
        m1 = t1;
        l0 *= r0;
        l1 *= r1;
#pragma unroll
        for (int j = 0; j < KT; ++j) { o[j][0] *= r0; o[j][1] *= r1; o[j][2] *= r0; o[j][3] *= r1; }
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      const float p0 = ex2(s0 - b0), p1 = ex2(s1 - b1), p2 = ex2(s2 - b0), p3 = ex2(s3 - b1);
      l0 += p0 + p2;
      l1 += p1 + p3;
      const uint32_t pb0 = turned(pack_half2(p0, p1)), pb1 = turned(pack_half2(p2, p3));
#pragma unroll
      for (int w = 0; w < VR; ++w) {
        const uint32_t v0 = f.v[0][w] ^ 0x80808080u, v1 = f.v[1][w] ^ 0x80808080u, v2 = f.v[2][w] ^ 0x80808080u, v3 = f.v[3][w] ^ 0x80808080u;
        const uint32_t lo01 = __byte_perm(v0, v1, 0x5140), lo23 = __byte_perm(v2, v3, 0x5140);
        constexpr int PER = VW >= 4 ? 2 : 1;            // m tiles of a register
        {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma(d, half2_of<0x5140>(lo01), half2_of<0x5342>(lo01), half2_of<0x5140>(lo23), half2_of<0x5342>(lo23), pb0, pb1);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[PER * w][e] = fmaf(sv, d[e], o[PER * w][e]);
        }
        if constexpr (PER == 2) {
          const uint32_t hi01 = __byte_perm(v0, v1, 0x7362), hi23 = __byte_perm(v2, v3, 0x7362);
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma(d, half2_of<0x5140>(hi01), half2_of<0x5342>(hi01), half2_of<0x5140>(hi23), half2_of<0x5342>(hi23), pb0, pb1);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[PER * w + 1][e] = fmaf(sv, d[e], o[PER * w + 1][e]);
        }
      }
    };
    for (int i0 = 0; i0 < mine; i0 += 32) {
      if (i0 > 0) {
        look_up(i0);
        fetch(0, buf[0]);
      }
      const int n = min(32, mine - i0);
      for (int i = 0; i < n; i += 2) {
        if (i + 1 < n) fetch(i + 1, buf[1]);
        work(i0 + i, i, buf[0]);
        if (i + 2 < n) fetch(i + 2, buf[0]);
        if (i + 1 < n) work(i0 + i + 1, i + 1, buf[1]);
      }
    }
    // the warps' sums
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, d);
      l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    if (g == 0) {
      sm_m[warp][2 * t] = m0; sm_m[warp][2 * t + 1] = m1;
      sm_l[warp][2 * t] = l0; sm_l[warp][2 * t + 1] = l1;
    }
#pragma unroll
    for (int j = 0; j < KT; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {                     // column 2 j + e of this thread's
        const int c = 2 * j + e, d = (c / VW * 8 + g) * VW + c % VW;
        if (2 * t < nh) sm_o[warp][2 * t * DH + d] = o[j][2 * e];
        if (2 * t + 1 < nh) sm_o[warp][(2 * t + 1) * DH + d] = o[j][2 * e + 1];
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nh * DH; e += WARPS * 32) {
      const int h = e / DH;
      float top = sm_m[0][h];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm_m[w][h]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, tot = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float c = ex2(sm_m[w][h] - base);
        sum = fmaf(sm_o[w][e], c, sum);
        tot = fmaf(sm_l[w][h], c, tot);
      }
      sm_o[0][e] = sum;
      if (e == h * DH) { fin_m[h] = top; fin_l[h] = tot; }
    }
    __syncthreads();
    finish_item<__nv_bfloat16>(a, x, tiles, HT, h0, nh, fin_m, fin_l, sm_o[0], weights, &last, LOG2E, [](float v) { return ex2(v); });
    __syncthreads();
  }
}

// As mlxb_kv8_rows for bfloat16 and heads of MLXB_HEAD_DIM; tiles of eight query heads: partial n_rows * tiles * most_chunks * 8 *
// (dim + 2) floats, counters n_rows * tiles (tiles: Hkv * ceil(Hq / Hkv / 8)).
MLXB_EXPORT int mlxb_kv8_rows_tc(const void* q, int ldq, const int* rows, const int* positions, const int* token_req,
                                 const int* block_table, int max_pages, int n_pages, int page, int Hq, int Hkv, int dim, int window,
                                 float scale, const int8_t* k8, const int8_t* v8, const float* ks, const float* vs, float* partial,
                                 int* counters, int most_chunks, void* out, int ldo, int n_rows, int* status, const float* sinks,
                                 cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (n_rows > ROWS_MOST) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: %d rows, a launch takes %d", n_rows, ROWS_MOST);
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: %d query heads over %d key/value heads", Hq, Hkv);
  if (dim != DH) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: head size %d, this library is for %d", dim, DH);
  if (page < BLK || (page & (page - 1))) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: page size %d (a power of two of at least %d)", page, BLK);
  if (most_chunks <= 0) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: %d chunks of a row", most_chunks);
  if (((uintptr_t)k8 | (uintptr_t)v8 | (uintptr_t)partial) & 15)
    return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: pools and scratch memory must be 16-byte aligned");
  const RowsArgs a{q, ldq, rows, positions, token_req, block_table, max_pages, n_pages, page, Hq, Hkv, dim, window, scale, k8, v8, ks,
                   vs, sinks, partial, counters, most_chunks, out, ldo, n_rows, status};
  const int group_tiles = (Hq / Hkv + HT - 1) / HT, tiles = Hkv * group_tiles;
  const size_t smem = (size_t)(n_rows + 1 + (most_chunks + 1) * HT) * 4;
  const long long most = (long long)n_rows * most_chunks * tiles, fill = (long long)CTAS * mlxb_sm_count();
  static SharedLimit limit;
  const size_t all = (ROWS_MOST + 1 + 4096) * 4;
  if (smem > all) return mlxb_fail(MLXB_BAD_ARG, "kv8_rows_tc: %d rows, %d chunks", n_rows, most_chunks);
  if (cudaError_t e = limit.raise(rows_tc_kernel, all)) return mlxb_fail((int)e, "kv8_rows_tc: shared memory: %s", cudaGetErrorString(e));
  launch_pdl(rows_tc_kernel, dim3((unsigned)(most < fill ? most : fill)), dim3(WARPS * 32), smem, stream, a, tiles, group_tiles,
             (ldq % 4 == 0 && !((uintptr_t)q & 7)) ? 1 : 0);
  return mlxb_check_launch("kv8_rows_tc");
}
