// Attention of single float32 queries over pages in 8 bits on the CUDA cores, all arithmetic in float32.
//
// y = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M), s_j = scale * (q . k_j), over the keys j that the row sees, k_j and v_j codes
// times the scale of their block of 16 positions and head; a sink adds exp(sink - M) to the sum below.  One pass over the keys: LPK
// lanes stand on a key, 16 columns each (16 bytes of codes a load), every group of lanes keeps its own maximum, sum and weighted
// values of up to four query heads, and what the codes of a key were turned into serves all of them.  The scale of a key's block
// multiplies its score, that of a value's block the score's exponential.
#include "kv8_rows.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int WARPS = 4;
constexpr int HT = 4;                // query heads of an item

// 16 codes as float32: the code + 128 in the low byte of 2^23, less 2^23 + 128
__device__ __forceinline__ void codes16(const uint4& c, float (&f)[16]) {
  const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(__byte_perm(w[i >> 2], 0x4b000000u, 0x7540 + (i & 3))) - 8388736.f;
}

template <int LPK>
__global__ void __launch_bounds__(WARPS * 32)
rows_kernel(const RowsArgs a, int tiles, int group_tiles) {
  constexpr int KPW = 32 / LPK, NG = WARPS * KPW;     // keys at a time: of a warp, of the CTA
  extern __shared__ int dyn[];                        // what is kept of the rows, then the weights of the last step
  __shared__ int warp_sums[WARPS], last;
  __shared__ float sm_m[WARPS][HT], sm_l[WARPS][HT], sm_o[WARPS][HT][256];
  __shared__ float fin_m[HT], fin_l[HT], fin_o[HT * 256];
  const Rows rows(dyn, a.n_rows);
  float* weights = reinterpret_cast<float*>(dyn + 4 * a.n_rows + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int total = schedule(a, rows, warp_sums) * tiles;
  const int G = a.Hq / a.Hkv, D = a.dim, per = a.page / BLK;
  const int grp = warp * KPW + lane / LPK, part = lane & (LPK - 1);
  const bool mine = part * 16 < D;
  pdl_wait();
  pdl_trigger();
  const int8_t *k8 = after_wait(a.k8), *v8 = after_wait(a.v8);
  const float *ks = after_wait(a.ks), *vs = after_wait(a.vs);
  for (int it = blockIdx.x; it < total; it += gridDim.x) {
    const Item x = item_of(a, rows, it, tiles);
    const int hk = x.tile / group_tiles, j0 = (x.tile - hk * group_tiles) * HT, nh = min(HT, G - j0), h0 = hk * G + j0;
    const int* bt = a.block_table + (size_t)x.row.req * a.max_pages;
    const int lo = a.window > 0 ? x.row.pos - a.window + 1 : 0;
    float q[HT][16], o[HT][16], m[HT], l[HT];
    const float* qr = after_wait((const float*)a.q) + (size_t)x.row.tok * a.ldq + (size_t)h0 * D + part * 16;
#pragma unroll
    for (int h = 0; h < HT; ++h) {
      m[h] = -INFINITY; l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        q[h][i] = mine && h < nh ? qr[h * D + i] : 0.f;
        o[h][i] = 0.f;
      }
    }
    for (int key = x.begin + grp; key - grp < x.end; key += NG) {     // (all lanes of a warp stay together)
      const bool in = key < x.end && key >= lo;
      int pg = -1;
      if (in) pg = page_of(a, bt, key);
      const bool seen = pg >= 0;
      uint4 ck = make_uint4(0, 0, 0, 0), cv = ck;
      float sk = 0.f, sv = 0.f;
      if (seen) {
        const int r = key & (a.page - 1);
        const size_t at = ((size_t)pg * a.Hkv + hk) * a.page + r, as = ((size_t)pg * a.Hkv + hk) * per + r / BLK;
        if (mine) {
          ck = *reinterpret_cast<const uint4*>(k8 + at * D + part * 16);
          cv = *reinterpret_cast<const uint4*>(v8 + at * D + part * 16);
        }
        sk = ks[as];
        sv = vs[as];
      }
      float f[16], s[HT];
      codes16(ck, f);
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        s[h] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h] = fmaf(q[h][i], f[i], s[h]);
#pragma unroll
        for (int d = 1; d < LPK; d <<= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], d);
      }
      if (!seen) continue;                            // (the shuffles are behind every lane)
      codes16(cv, f);
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        const float t = s[h] * (sk * a.scale);
        if (t > m[h]) {
          const float c = expf(m[h] - t);
          m[h] = t;
          l[h] *= c;
#pragma unroll
          for (int i = 0; i < 16; ++i) o[h][i] *= c;
        }
        const float p = expf(t - m[h]), w = p * sv;
        l[h] += p;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[h][i] = fmaf(w, f[i], o[h][i]);
      }
    }
    // the groups of a warp, then the warps
#pragma unroll
    for (int h = 0; h < HT; ++h) {
#pragma unroll
      for (int d = LPK; d < 32; d <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m[h], d), lo_ = __shfl_xor_sync(0xffffffffu, l[h], d);
        const float top = fmaxf(m[h], mo), base = top == -INFINITY ? 0.f : top;
        const float c0 = expf(m[h] - base), c1 = expf(mo - base);
        l[h] = l[h] * c0 + lo_ * c1;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[h][i] = o[h][i] * c0 + __shfl_xor_sync(0xffffffffu, o[h][i], d) * c1;
        m[h] = top;
      }
      if (lane < LPK && mine) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sm_o[warp][h][part * 16 + i] = o[h][i];
        if (lane == 0) { sm_m[warp][h] = m[h]; sm_l[warp][h] = l[h]; }
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nh * D; e += blockDim.x) {
      const int h = e / D, d = e - h * D;
      float top = sm_m[0][h];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm_m[w][h]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, tot = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float c = expf(sm_m[w][h] - base);
        sum += sm_o[w][h][d] * c;
        tot += sm_l[w][h] * c;
      }
      fin_o[e] = sum;
      if (d == 0) { fin_m[h] = top; fin_l[h] = tot; }
    }
    __syncthreads();
    finish_item<float>(a, x, tiles, HT, h0, nh, fin_m, fin_l, fin_o, weights, &last, 1.f, [](float v) { return expf(v); });
    __syncthreads();
  }
}

// out [row, Hq * dim] for the rows `rows` (int32 indices into positions, token_req, q and out; null: rows 0 .. n_rows - 1): one query
// of each head at the row's position.  partial: n_rows * tiles * most_chunks * 4 * (dim + 2) floats; counters: n_rows * tiles, zero
// before the first call and left zero (tiles: Hkv * ceil(Hq / Hkv / 4)).
MLXB_EXPORT int mlxb_kv8_rows(const RowsRecord* rec, long long bytes, cudaStream_t stream) {
  RowsArgs a;
  if (int e = rows_args(rec, bytes, "kv8_rows", a)) return e;
  if (a.n_rows <= 0) return 0;
  const int Hq = a.Hq, Hkv = a.Hkv, dim = a.dim, n_rows = a.n_rows, most_chunks = a.most_chunks;
  const int group_tiles = (Hq / Hkv + HT - 1) / HT, tiles = Hkv * group_tiles;
  const size_t smem = rows_bytes(n_rows) + (size_t)(most_chunks + 1) * HT * 4;
  const long long most = (long long)n_rows * most_chunks * tiles, fill = 4ll * mlxb_sm_count();
  const dim3 grid((unsigned)(most < fill ? most : fill));
  auto go = [&](auto kernel) { launch_pdl(kernel, grid, dim3(WARPS * 32), smem, stream, a, tiles, group_tiles); };
  if (dim <= 16) go(rows_kernel<1>);
  else if (dim <= 32) go(rows_kernel<2>);
  else if (dim <= 64) go(rows_kernel<4>);
  else if (dim <= 128) go(rows_kernel<8>);
  else go(rows_kernel<16>);
  return mlxb_check_launch("kv8_rows");
}
