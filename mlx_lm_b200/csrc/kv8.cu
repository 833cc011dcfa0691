// Keys and values of a step into pages that hold them in 8 bits, and back.
//
// Pages of one layer: codes int8 [n_pages][heads][page][head_dim], scales float32 [n_pages][heads][page / 16]: one scale for
// each block of 16 positions and head; a code stands for code * scale.
//
// append  For a block of a request and a head: A = the largest |x| among the finite numbers that the step brings, S = A / 127 (0
//         below 2^-100).  A step that brings the block's first position sets the scale to S; a later one to the larger of S and
//         the scale as it was, and if that grows, the older codes become rint(code * (old / new)).  New codes are
//         clamp(rint(x * (1 / scale)), -127, 127).  So a scale never falls while a block fills, a code is rounded again only when
//         a larger number arrives, and what a block holds depends on how the step cut the request only through that second
//         rounding.  A number that is not finite cannot be held: NaN becomes 0, an infinity the largest code of its sign, and the
//         status word says so, and where the caller gives flags for its requests, that of the request.
//         Keys (and the step's queries beside them) are turned by their position on the way: the pair (u, v) of dimensions
//         (i, i + half), or (2i, 2i + 1), becomes (u c - v s, v c + u s), c and s the cosine and sine of the float32 angle
//         position * freq[i] times `mscale`.  Products, sums, the quotient and the reciprocal are rounded one by one (no fused
//         multiply-add): x decides a code by its rounding, and another order of roundings would be another code now and then.
// read    The values at given positions, rounded to the output's type.
//
// Both are bound by their latencies: where rows are few, by that of the look-ups, the loads and the stores in turn; where they are many, of a
// warp's loads, which nothing but the other four warps of its scheduler hides.  8192 rows of 32/8 heads of 128 at position 0, turned, append
// and the read behind it 57 us: 234 MB, 4.1 TB/s; the append alone 46, DRAM 37 % and issue slots 54 % used (a warp waits 2.2 issues for
// a load, 1.5 for arithmetic, 1.2 for instructions, 0.9 for shared memory, 0.8 at barriers, for each that it makes).
// (232 us with divisions in the loops and sines for each row of each head: sines are a CTA's now, and every number is formed twice, for its
// block's largest and for its code, since registers for a block's numbers would cost a third of the warps.)  One row of a request 5.5 us,
// 64 requests' 6.5.  A lane of the read takes 16 codes: 8, so that a warp's stores are whole runs of 512 bytes, took 1 us longer for one row
// (twice the steps) and no less for 8192.
//
// Rows of a request stand together in order of position without gaps (the order in which a step lists them): the row whose predecessor
// is of another request or block leads its block's rows.  A leader's block and head are one warp's, so nothing is written by two warps.
// A row that goes back, or leaves positions out inside its block, would lead a block that has a leader already: it and the rows that
// follow on from it are left out and reported.
#include <float.h>

#include <type_traits>

#include "common.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int BLK = 16;              // positions that share a scale
constexpr int MAX_WARPS = 8;
constexpr uint32_t INF_BITS = 0x7f800000u;

template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, float (&v)[4]) {      // the first n of four columns
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f(p[i]) : 0.f;
}
// Four neighbouring elements as they lie in memory, and as numbers.
template <typename T> struct Four;
template <> struct Four<float> { float4 v; };
template <> struct Four<__nv_bfloat16> { uint2 v; };
__device__ __forceinline__ void unpack4(const Four<float>& r, float (&v)[4]) { v[0] = r.v.x; v[1] = r.v.y; v[2] = r.v.z; v[3] = r.v.w; }
__device__ __forceinline__ void unpack4(const Four<__nv_bfloat16>& r, float (&v)[4]) {
  v[0] = __uint_as_float(r.v.x << 16);
  v[1] = __uint_as_float(r.v.x & 0xffff0000u);
  v[2] = __uint_as_float(r.v.y << 16);
  v[3] = __uint_as_float(r.v.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, bool vec, const float (&v)[4]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = v[i];
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, bool vec, const float (&v)[4]) {
  if (vec) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __float2bfloat16_rn(v[i]);
  }
}
// rint(x * inv) in the low byte, for |x * inv| < 127.5.  1.5 * 2^23 + n has n's two's complement in its low bits, and adding it rounds
// to the nearest whole number, ties to even.
__device__ __forceinline__ uint32_t code_of(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); }
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float inv) {
  const uint32_t lo = __byte_perm(code_of(x[0], inv), code_of(x[1], inv), 0x0040);
  const uint32_t hi = __byte_perm(code_of(x[2], inv), code_of(x[3], inv), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// The larger magnitudes of two pairs (signs are of no meaning); NaN if one is.
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

struct AppendArgs {
  const void *k, *v, *q;         // [T, heads * dk], [T, heads * dv], [T, q heads * dk], or null
  void* q_out;                   // [T, q heads * dim]
  int ldk, ldv, ldq, ldo;
  int T, Hkv, G;                 // G: query heads to a key/value head (0: no queries)
  int dk, dv, dim;
  const float* freq;
  int half, interleaved;
  float mscale;
  const int *positions, *token_req, *block_table;
  int n_req, max_pages, n_pages, page;
  int8_t *k8, *v8;
  float *ks, *vs;
  int* status;
  const int* slots;              // [n_req]: a request's place among the flags
  int* not_finite;               // [n_flags], or null
  int n_flags;
  int chunk, heads_per_cta;
};

struct Leader {
  int row, n, pos, page_id, req;      // page_id < 0: nothing is stored
};

// A CTA takes the leaders among `chunk` rows and a group of heads: it lists the leaders, forms the sines and cosines of all their rows
// once in shared memory, and its warps take the pairs (leader, head; keys, values or one query head).  A warp holds all the numbers of
// a pair (16 rows of up to 128 columns: 64 a lane) in registers between the search for the largest and the codes, so a number is
// read once.  LPR lanes stand on a row, 8 columns each in two groups of 4: the groups of a lane are a rotation's two halves where
// these are whole groups, so that a pair's numbers meet in one lane.
// WIDE: four columns an access, and where something turns, both halves of a pair in one lane; else column by column.
template <typename T, int LPR, bool WIDE>
__global__ void __launch_bounds__(MAX_WARPS * 32, WIDE && sizeof(T) == 2 && LPR <= 16 ? 3 : 1)
append_kernel(const AppendArgs a) {
  constexpr int RP = 32 / LPR;                 // rows at a time
  constexpr int PASSES = BLK / RP;
  extern __shared__ __align__(16) float2 turn[];      // [rows][half]: cosine and sine
  __shared__ Leader lead[BLK];
  __shared__ int n_lead, last_row, pos_of[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
  const int row0 = blockIdx.x * a.chunk;
  if (warp == 0) {
    // Lane i looks at row row0 + i (a leader of this CTA is among the first `chunk`, its rows among the 15 behind it): where a row
    // begins something new shows how far the rows before it reach.
    const int t = row0 + lane;
    const int r = t < a.T ? a.token_req[t] : -1, p = t < a.T ? a.positions[t] : 0;
    int rb = __shfl_up_sync(0xffffffffu, r, 1), pb = __shfl_up_sync(0xffffffffu, p, 1);
    if (lane == 0) { rb = row0 > 0 ? a.token_req[row0 - 1] : -1; pb = row0 > 0 ? a.positions[row0 - 1] : 0; }
    const bool fresh = r < 0 || rb != r || pb != p - 1 || (p & (BLK - 1)) == 0;
    const bool astray = rb == r && pb != p - 1 && (p <= pb || p / BLK == pb / BLK);
    const uint32_t starts = __ballot_sync(0xffffffffu, fresh);
    pos_of[lane] = p;
    const bool leads = fresh && r >= 0 && lane < a.chunk;
    const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
    int end = row0;
    if (leads) {
      const uint32_t behind = lane < 31 ? starts >> (lane + 1) : 0u;
      const int n = behind ? __ffs(behind) : BLK;           // (a block ends after 16 rows at most: with a chunk of 16 within the 32)
      const int lp = p / a.page;
      int pg = -1;
      if (r >= a.n_req || p < 0 || lp >= a.max_pages || (astray && a.k)) {
        if (a.k && blockIdx.y == 0) atomicOr(a.status, MLXB_ST_POSITION_RANGE);
      } else {
        pg = a.block_table[(size_t)r * a.max_pages + lp];
        if (pg >= a.n_pages) {
          if (a.k && blockIdx.y == 0) atomicOr(a.status, MLXB_ST_PAGE_RANGE);
          pg = -1;
        }
      }
      lead[__popc(leaders & ((1u << lane) - 1u))] = Leader{t, n, p, pg, r};
      end = t + n;
    }
    end = __reduce_max_sync(0xffffffffu, end);
    if (lane == 0) { n_lead = __popc(leaders); last_row = end; }
  }
  __syncthreads();
  const int nl = n_lead;
  if (nl == 0) {
    // a step of rows of no request alone must not end before its predecessor has: what comes next waits for this grid only
    if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
    return;
  }
  // (rows between two leaders that are of no request get an angle nobody uses)
  if (a.half > 0) {
    const int di = blockDim.x / a.half, dj = blockDim.x - di * a.half, n = (last_row - row0) * a.half;
    int i = threadIdx.x / a.half, j = threadIdx.x - i * a.half;
    for (int e = threadIdx.x; e < n; e += blockDim.x) {
      float sn, cs;
      sincosf(__fmul_rn((float)pos_of[i], a.freq[j]), &sn, &cs);
      turn[e] = make_float2(__fmul_rn(cs, a.mscale), __fmul_rn(sn, a.mscale));
      i += di;
      j += dj;
      if (j >= a.half) { j -= a.half; ++i; }
    }
  }
  pdl_wait();
  pdl_trigger();
  __syncthreads();

  const int per = a.page / BLK;
  const int kinds = (a.k ? 2 : 0) + a.G;
  const int h0 = blockIdx.y * a.heads_per_cta, nh = min(a.heads_per_cta, a.Hkv - h0);
  const int sub = lane / LPR, l = lane & (LPR - 1);
  const int hg = a.half >> 2;
  // the pairs (leader, w), w = head * kinds + kind, one after the other without a division a pair
  const int nk = nh * kinds;
  const uint32_t by_kinds = (65536u + kinds - 1) / kinds;       // w / kinds = w * by_kinds >> 16 for w * kinds < 65536
  int li = 0, w = warp;
  for (;; w += n_warps) {
    while (w >= nk && li < nl) { w -= nk; ++li; }
    if (li >= nl) break;
    const Leader ld = lead[li];
    const int hw = (int)(w * by_kinds >> 16), h = h0 + hw;
    int kind = w - hw * kinds;                 // 0 keys, 1 values, 2 + i query head i of the group
    if (!a.k) kind += 2;
    const bool turned = kind != 1 && a.half > 0;
    const T* src;
    int ld_src, width;
    if (kind == 0) { src = (const T*)a.k + (size_t)h * a.dk; ld_src = a.ldk; width = a.dk; }
    else if (kind == 1) { src = (const T*)a.v + (size_t)h * a.dv; ld_src = a.ldv; width = a.dv; }
    else { src = (const T*)a.q + ((size_t)h * a.G + kind - 2) * a.dk; ld_src = a.ldq; width = a.dk; }
    src = after_wait(src);
    // the two groups of four columns of this lane
    int c0, c1;
    if (WIDE && turned) {
      c0 = l < hg ? 4 * l : 2 * a.half + 8 * (l - hg);
      c1 = l < hg ? c0 + a.half : c0 + 4;
    } else {
      c0 = 8 * l;
      c1 = c0 + 4;
    }
    const bool mine = 8 * l < a.dim;
    auto value = [&](const T* row, const float2* cs, int i) {      // column i, turned, wherever its partner is
      const float x = i < width ? to_f(row[i]) : 0.f;
      if (i >= 2 * a.half) return x;
      const bool lower = a.interleaved ? !(i & 1) : i < a.half;
      const int j = a.interleaved ? (i ^ 1) : lower ? i + a.half : i - a.half;
      const float y = to_f(row[j]);
      const float2 t = cs[a.interleaved ? i >> 1 : lower ? i : j];
      return lower ? __fsub_rn(__fmul_rn(x, t.x), __fmul_rn(y, t.y)) : __fadd_rn(__fmul_rn(x, t.x), __fmul_rn(y, t.y));
    };
    const float2* cs0 = turn + (ld.row - row0) * a.half;
    // All loads of a pair go out before the first number is used: one latency a pair, not one a row.  What is loaded stays as it is; the
    // numbers are formed from it twice (for the largest, then for the codes), which takes fewer registers than keeping them.
    Four<T> raw[WIDE ? PASSES : 1][2];
    if constexpr (WIDE) {
      const T* row = src + (size_t)(ld.row + sub) * ld_src + c0;
      const size_t step = (size_t)RP * ld_src;
      const int apart = c1 - c0, left = ld.n - sub;
      const bool lower = mine && c0 < width, upper = mine && c1 < width;
#pragma unroll
      for (int s = 0; s < PASSES; ++s, row += step) {
        raw[s][0] = Four<T>{};
        raw[s][1] = Four<T>{};
        if (lower && s * RP < left) raw[s][0] = *reinterpret_cast<const Four<T>*>(row);
        if (upper && s * RP < left) raw[s][1] = *reinterpret_cast<const Four<T>*>(row + apart);
      }
    }
    auto numbers = [&](int s, float (&x)[4], float (&y)[4]) {      // both groups of row s * RP + sub, turned
      const float2* cs = cs0 + (s * RP + sub) * a.half;
      if constexpr (WIDE) {
        unpack4(raw[s][0], x);
        unpack4(raw[s][1], y);
        if (turned && l < hg) {
          const float4 t01 = *reinterpret_cast<const float4*>(cs + c0), t23 = *reinterpret_cast<const float4*>(cs + c0 + 2);
          const float2 t[4] = {make_float2(t01.x, t01.y), make_float2(t01.z, t01.w), make_float2(t23.x, t23.y), make_float2(t23.z, t23.w)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = x[e], q = y[e];
            x[e] = __fsub_rn(__fmul_rn(p, t[e].x), __fmul_rn(q, t[e].y));
            y[e] = __fadd_rn(__fmul_rn(q, t[e].x), __fmul_rn(p, t[e].y));
          }
        }
      } else {
        const T* row = src + (size_t)(ld.row + s * RP + sub) * ld_src;
        if (turned) {
#pragma unroll
          for (int e = 0; e < 4; ++e) { x[e] = value(row, cs, c0 + e); y[e] = value(row, cs, c1 + e); }
        } else {
          load4(row + c0, width - c0, x);
          load4(row + c1, width - c1, y);
        }
      }
    };
    if (kind >= 2) {
      T* dst = (T*)a.q_out + ((size_t)h * a.G + kind - 2) * a.dim + (size_t)(ld.row + sub) * a.ldo + c0;
      const size_t step = (size_t)RP * a.ldo;
      const int apart = c1 - c0, left = mine ? ld.n - sub : 0;
#pragma unroll
      for (int s = 0; s < PASSES; ++s, dst += step) {
        if (s * RP >= left) break;
        float x[4], y[4];
        numbers(s, x, y);
        store4(dst, WIDE, x);
        store4(dst + apart, WIDE, y);
      }
      continue;
    }
    if (ld.page_id < 0) continue;
    // the largest magnitude, as bits; NaN and infinities come out on top
    uint32_t top = 0;
    if constexpr (WIDE && sizeof(T) == 2) {
      // as the numbers came, two at a time: all there is to it for values, and whether a key is not finite
      uint32_t pairs = 0;
#pragma unroll
      for (int s = 0; s < PASSES; ++s)
        pairs = max_abs2(max_abs2(max_abs2(max_abs2(pairs, raw[s][0].v.x), raw[s][0].v.y), raw[s][1].v.x), raw[s][1].v.y);
      top = max(pairs << 16 & 0x7fffffffu, pairs & 0x7fff0000u);
    }
    if (!(WIDE && sizeof(T) == 2) || (turned && top < INF_BITS)) {
      top = 0;
      float large = 0.f;                       // (no NaN comes from finite numbers, and fmaxf finds infinities)
#pragma unroll
      for (int s = 0; s < PASSES; ++s) {
        if (s * RP >= ld.n) break;
        if (mine && s * RP + sub < ld.n) {
          float x[4], y[4];
          numbers(s, x, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (WIDE && sizeof(T) == 2) large = fmaxf(large, fmaxf(fabsf(x[e]), fabsf(y[e])));
            else top = max(top, max(__float_as_uint(x[e]) & 0x7fffffffu, __float_as_uint(y[e]) & 0x7fffffffu));
          }
        }
      }
      top = max(top, __float_as_uint(large));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const bool odd = top >= INF_BITS;          // something is not finite: the largest of the others, and NaN becomes 0
    if (odd) {
      if (lane == 0) {
        atomicOr(a.status, MLXB_ST_NOT_FINITE);
        if (a.not_finite) {
          const int i = a.slots[ld.req];
          if ((unsigned)i < (unsigned)a.n_flags) a.not_finite[i] = 1;
        }
      }
      top = 0;
#pragma unroll
      for (int s = 0; s < PASSES; ++s) {
        if (s * RP >= ld.n) break;
        if (mine && s * RP + sub < ld.n) {
          float x[4], y[4];
          numbers(s, x, y);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bx = __float_as_uint(x[e]) & 0x7fffffffu, by = __float_as_uint(y[e]) & 0x7fffffffu;
            if (bx < INF_BITS) top = max(top, bx);
            if (by < INF_BITS) top = max(top, by);
          }
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
    }
    const float largest = __uint_as_float(top);
    float scale = largest < 7.888609052210118e-31f ? 0.f : __fdiv_rn(largest, 127.f);
    const int off = ld.pos & (BLK - 1), in_page = ld.pos & (a.page - 1);
    int8_t* codes = (kind ? a.v8 : a.k8) + (((size_t)ld.page_id * a.Hkv + h) * a.page + (in_page - off)) * a.dim;
    float* sp = (kind ? a.vs : a.ks) + ((size_t)ld.page_id * a.Hkv + h) * per + in_page / BLK;
    if (off > 0) {
      const float old = *sp;
      if (scale > old) {                       // older codes of the block to the larger scale
        const float ratio = __fdiv_rn(old, scale);
        for (int e = lane * 16; e < off * a.dim; e += 512) {
          uint4 c = *reinterpret_cast<const uint4*>(codes + e);
          uint32_t* cw = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const char4 b = *reinterpret_cast<const char4*>(&cw[j]);
            const float f[4] = {(float)b.x, (float)b.y, (float)b.z, (float)b.w};
            cw[j] = codes4(f, ratio);
          }
          *reinterpret_cast<uint4*>(codes + e) = c;
        }
      } else {
        scale = old;
      }
    }
    __syncwarp();
    if (lane == 0) *sp = scale;
    const float inv = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
      if (s * RP >= ld.n) break;
      const int i = s * RP + sub;
      if (mine && i < ld.n) {
        int8_t* dst = codes + (off + i) * a.dim;
        float x[4], y[4];
        numbers(s, x, y);
        if (odd) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float most = fminf(127.f * scale, FLT_MAX);      // (of an infinity the largest code; 127 * (FLT_MAX / 127) rounds up)
            x[e] = x[e] != x[e] ? 0.f : fminf(fmaxf(x[e], -most), most);
            y[e] = y[e] != y[e] ? 0.f : fminf(fmaxf(y[e], -most), most);
          }
        }
        *reinterpret_cast<uint32_t*>(dst + c0) = scale > 0.f ? codes4(x, inv) : 0u;
        *reinterpret_cast<uint32_t*>(dst + c1) = scale > 0.f ? codes4(y, inv) : 0u;
      }
    }
  }
}

// Arguments as one record of 8-byte fields: the caller fills it in a tenth of the time that as many arguments of a call take it.
struct AppendRecord {
  const void *k, *v, *q;
  void* q_out;
  const float* freq;
  const int *positions, *token_req, *block_table;
  int8_t *k8, *v8;
  float *ks, *vs;
  int* status;
  const int* slots;
  int* not_finite;
  long long dtype, ldk, ldv, ldq, ldo, T, Hkv, G, dk, dv, dim, half, interleaved, n_req, max_pages, n_pages, page, n_flags;
  double mscale;
};

// Keys [T, Hkv * dk] and values [T, Hkv * dv] (dtype; rows at strides ldk, ldv) into the pages; queries [T, Hkv * G * dk] turned into
// q_out [T, Hkv * G * dim] (G 0: none; k and v null: queries only).  Columns of a head from dk (dv) to dim are zeros.  page a power of
// two of at least 16, dim a multiple of 16 up to 256, freq [half] with 2 * half <= dk.
MLXB_EXPORT int mlxb_kv8_append(const AppendRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(AppendRecord)) return mlxb_fail(MLXB_BAD_ARG, "kv8_append: a record of %lld bytes", bytes);
  const AppendRecord& x = *rec;
  const int dtype = (int)x.dtype, ldk = (int)x.ldk, ldv = (int)x.ldv, ldq = (int)x.ldq, ldo = (int)x.ldo, T = (int)x.T, Hkv = (int)x.Hkv;
  const int G = (int)x.G, dk = (int)x.dk, dv = (int)x.dv, dim = (int)x.dim, half = (int)x.half, page = (int)x.page;
  const void *k = x.k, *v = x.v, *q = x.q;
  void* q_out = x.q_out;
  const float* freq = x.freq;
  int8_t *k8 = x.k8, *v8 = x.v8;
  if (dtype != MLXB_F32 && dtype != MLXB_BF16) return mlxb_fail(MLXB_BAD_DTYPE, "kv8_append: dtype code %d", dtype);
  if (T <= 0) return 0;
  if (Hkv <= 0 || G < 0 || G > 250 || dim % 16 || dim < 16 || dim > 256 || dk <= 0 || dk > dim || dv <= 0 || dv > dim)
    return mlxb_fail(MLXB_BAD_ARG, "kv8_append: %d heads of %d and %d columns in rows of %d (a multiple of 16 up to 256)", Hkv, dk, dv, dim);
  if (page < BLK || (page & (page - 1))) return mlxb_fail(MLXB_BAD_ARG, "kv8_append: page size %d (a power of two of at least %d)", page, BLK);
  if (half < 0 || 2 * half > dk || (half && !freq)) return mlxb_fail(MLXB_BAD_ARG, "kv8_append: %d pairs of %d columns", half, dk);
  if ((k == nullptr) != (v == nullptr) || (!k && !G) || (G && (!q || !q_out)))
    return mlxb_fail(MLXB_BAD_ARG, "kv8_append: keys and values go together, and queries with an output");
  if (((uintptr_t)k8 | (uintptr_t)v8) & 15) return mlxb_fail(MLXB_BAD_ARG, "kv8_append: pools must be 16-byte aligned");
  const size_t item = dtype == MLXB_F32 ? 4 : 2;
  auto fits = [&](const void* p, int ld, int d) { return (((uintptr_t)p) % (4 * item)) == 0 && ld % 4 == 0 && d % 4 == 0; };
  AppendArgs a{k, v, q, q_out, ldk, ldv, ldq, ldo, T, Hkv, G, dk, dv, dim, freq, half, (int)x.interleaved, (float)x.mscale,
               x.positions, x.token_req, x.block_table, (int)x.n_req, (int)x.max_pages, (int)x.n_pages, page, k8, v8, x.ks, x.vs, x.status,
               x.slots, x.not_finite, (int)x.n_flags, 1, 1};
  // four columns an access: whole groups of four, aligned, and pairs that are whole groups apart
  const bool wide = (!k || (fits(k, ldk, dk) && fits(v, ldv, dv))) && (!G || (fits(q, ldq, dk) && fits(q_out, ldo, dim))) &&
                    (half == 0 || (!x.interleaved && half % 4 == 0));
  // Few rows: a CTA a row, so that single tokens of different requests spread over the device; many: 16 rows, mostly a block's, share a
  // CTA, its sines and its look-ups.  Microseconds with the read behind it, 32/8 heads of 128, a row a CTA and 16: 64 single tokens
  // 6.6 and 22.6, 256 19.1 and 31.2, a portion of 256 11.0 and 10.5, of 512 14.4 and 10.7, of 8192 74 and 56.
  a.chunk = T <= 256 ? 1 : BLK;
  const int kinds = (k ? 2 : 0) + G;
  // Heads of a CTA: as many as keep its warps busy, and more (they share the sines) while there are still four CTAs for every SM: a portion
  // of 8192 56 us, 71 without the second half of the rule.
  a.heads_per_cta = kinds >= MAX_WARPS ? 1 : MAX_WARPS / kinds;
  const long long chunks = (T + a.chunk - 1) / a.chunk;
  while (2 * a.heads_per_cta <= Hkv && 2 * a.heads_per_cta * kinds * kinds < 65536 &&
         chunks * ((Hkv + 2 * a.heads_per_cta - 1) / (2 * a.heads_per_cta)) >= 4ll * mlxb_sm_count())
    a.heads_per_cta *= 2;
  if (a.heads_per_cta > Hkv) a.heads_per_cta = Hkv;
  const int warps = kinds * a.heads_per_cta < MAX_WARPS ? kinds * a.heads_per_cta : MAX_WARPS;
  const dim3 grid((T + a.chunk - 1) / a.chunk, (Hkv + a.heads_per_cta - 1) / a.heads_per_cta);
  if (grid.y > 65535) return mlxb_fail(MLXB_BAD_ARG, "kv8_append: %d heads", Hkv);
  const size_t smem = (size_t)(a.chunk + BLK - 1) * half * sizeof(float2);      // at most 31 rows of 128 pairs: 31 KB
  auto go = [&](auto kernel) { launch_pdl(kernel, grid, dim3(32 * warps), smem, stream, a); };
  const int lanes = dim / 8;
  auto sized = [&](auto type, auto w) {
    using T = decltype(type);
    constexpr bool W = decltype(w)::value;
    if (lanes <= 4) go(append_kernel<T, 4, W>);
    else if (lanes <= 8) go(append_kernel<T, 8, W>);
    else if (lanes <= 16) go(append_kernel<T, 16, W>);
    else go(append_kernel<T, 32, W>);
  };
  if (dtype == MLXB_F32) {
    if (wide) sized(float{}, std::true_type{}); else sized(float{}, std::false_type{});
  } else {
    if (wide) sized(__nv_bfloat16{}, std::true_type{}); else sized(__nv_bfloat16{}, std::false_type{});
  }
  return mlxb_check_launch("kv8_append");
}

// ---- what the pages hold

// A warp takes a row (its page looked up once), a lane 16 codes at a time, keys and values: 16 bytes in, 32 or 64 out.
template <typename T>
__global__ void __launch_bounds__(256)
read_kernel(const int* __restrict__ positions, const int* __restrict__ token_req, const int* __restrict__ block_table, int n_req,
            int max_pages, int n_pages, int page, int Hkv, int dim, const int8_t* k8, const int8_t* v8, const float* ks, const float* vs, T* k_out,
            int ldk, T* v_out, int ldv, int n_rows, int vec, int* status) {
  const int lane = threadIdx.x & 31, t = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int r = t < n_rows ? token_req[t] : -1;
  int p = 0, pg = -1;
  if (r >= 0) {
    p = positions[t];
    const int lp = p / page;
    if (r < n_req && p >= 0 && lp < max_pages) pg = block_table[(size_t)r * max_pages + lp];
    if (pg < 0 || pg >= n_pages) {
      if (lane == 0) atomicOr(status, pg < 0 ? MLXB_ST_POSITION_RANGE : MLXB_ST_PAGE_RANGE);
      pg = -1;
    }
  }
  pdl_wait();
  pdl_trigger();
  if (r < 0) return;
  k8 = after_wait(k8); v8 = after_wait(v8);
  ks = after_wait(ks); vs = after_wait(vs);
  const int per_head = dim / 16, per = page / BLK, in = p & (page - 1);
  const uint32_t by_head = (65536u + per_head - 1) / per_head;       // e / per_head = e * by_head >> 16 for e * per_head < 65536
#pragma unroll 4
  for (int w = lane; w < 2 * Hkv * per_head; w += 32) {
    const bool is_v = w >= Hkv * per_head;
    const int e = is_v ? w - Hkv * per_head : w, h = (int)(e * by_head >> 16), d = (e - h * per_head) * 16;
    float o[16];
    if (pg >= 0) {
      const size_t head = (size_t)pg * Hkv + h;
      const uint4 c4 = *reinterpret_cast<const uint4*>((is_v ? v8 : k8) + (head * page + in) * dim + d);
      const float s = (is_v ? vs : ks)[head * per + in / BLK];
      // code + 128 in the low byte of 2^23, less 2^23 + 128
      const uint32_t cw[4] = {c4.x ^ 0x80808080u, c4.y ^ 0x80808080u, c4.z ^ 0x80808080u, c4.w ^ 0x80808080u};
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j] = (__uint_as_float(__byte_perm(cw[j >> 2], 0x4b000000u, 0x7540 + (j & 3))) - 8388736.f) * s;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j] = 0.f;
    }
    T* dst = is_v ? v_out + (size_t)t * ldv + e * 16 : k_out + (size_t)t * ldk + e * 16;
    if (vec) {
      if constexpr (sizeof(T) == 2) {
        float lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { lo[j] = o[j]; hi[j] = o[8 + j]; }
        reinterpret_cast<uint4*>(dst)[0] = pack8(lo);
        reinterpret_cast<uint4*>(dst)[1] = pack8(hi);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(dst)[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) dst[j] = from_f<T>(o[j]);
    }
  }
}

struct ReadRecord {
  const int *positions, *token_req, *block_table;
  const int8_t *k8, *v8;
  const float *ks, *vs;
  void *k_out, *v_out;
  int* status;
  long long dtype, n_req, max_pages, n_pages, page, Hkv, dim, ldk, ldv, n_rows;
};

// k_out, v_out [n_rows, Hkv * dim]: what the pages stand for at position positions[t] of request token_req[t] (< 0: row left as it is;
// a position without a page: zeros and a status bit).
MLXB_EXPORT int mlxb_kv8_read(const ReadRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(ReadRecord)) return mlxb_fail(MLXB_BAD_ARG, "kv8_read: a record of %lld bytes", bytes);
  const ReadRecord& x = *rec;
  const int dtype = (int)x.dtype, n_req = (int)x.n_req, max_pages = (int)x.max_pages, n_pages = (int)x.n_pages, page = (int)x.page, Hkv = (int)x.Hkv;
  const int dim = (int)x.dim, ldk = (int)x.ldk, ldv = (int)x.ldv, n_rows = (int)x.n_rows;
  const int *positions = x.positions, *token_req = x.token_req, *block_table = x.block_table;
  const int8_t *k8 = x.k8, *v8 = x.v8;
  const float *ks = x.ks, *vs = x.vs;
  void *k_out = x.k_out, *v_out = x.v_out;
  int* status = x.status;
  if (dtype != MLXB_F32 && dtype != MLXB_BF16) return mlxb_fail(MLXB_BAD_DTYPE, "kv8_read: dtype code %d", dtype);
  if (n_rows <= 0) return 0;
  if (Hkv <= 0 || Hkv > 255 || dim % 16 || dim < 16 || dim > 256)
    return mlxb_fail(MLXB_BAD_ARG, "kv8_read: %d heads of %d (255 at most, a multiple of 16 up to 256)", Hkv, dim);
  if (page < BLK || (page & (page - 1))) return mlxb_fail(MLXB_BAD_ARG, "kv8_read: page size %d (a power of two of at least %d)", page, BLK);
  if (((uintptr_t)k8 | (uintptr_t)v8) & 15) return mlxb_fail(MLXB_BAD_ARG, "kv8_read: pools must be 16-byte aligned");
  const size_t item = dtype == MLXB_F32 ? 4 : 2;
  const int vec = !(((uintptr_t)k_out | (uintptr_t)v_out) & 15) && (ldk * item) % 16 == 0 && (ldv * item) % 16 == 0;
  const dim3 grid((unsigned)((n_rows + 7) / 8));
  if (dtype == MLXB_F32)
    launch_pdl(read_kernel<float>, grid, dim3(256), 0, stream, positions, token_req, block_table, n_req, max_pages, n_pages, page, Hkv, dim,
               k8, v8, ks, vs, (float*)k_out, ldk, (float*)v_out, ldv, n_rows, vec, status);
  else
    launch_pdl(read_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, positions, token_req, block_table, n_req, max_pages, n_pages, page,
               Hkv, dim, k8, v8, ks, vs, (__nv_bfloat16*)k_out, ldk, (__nv_bfloat16*)v_out, ldv, n_rows, vec, status);
  return mlxb_check_launch("kv8_read");
}
