// Attention of single float32 queries over pages in 8 bits on the CUDA cores, all arithmetic in float32.
//
// y = sum_j exp(s_j - M) v_j / sum_j exp(s_j - M), s_j = scale * (q . k_j), over the keys j that the row sees, k_j and v_j codes
// times the scale of their block of 16 positions and head; a sink adds exp(sink - M) to the sum below.  One pass over the keys, a block
// of 16 at a time (one page, one scale), up to four query heads together: what the codes of a key were turned into serves all of them.
//   scores   two lanes a key, 16 of its columns each in turn, the queries from shared memory
//   weights  two of the heads each of the two lanes, to shared memory (times the value block's scale)
//   values   a lane four columns, all 16 keys; fewer lanes a key, and more keys at a time, where heads are small
// The maximum follows a score only once that is more than 8 beyond it.  The next block's codes are loaded before a block's are used.
// Bound by latencies: long rows by that of a block's codes and of the chain from its scores to its weights, with 166 registers a thread and so less
// than three warps a scheduler to hide them (issue slots 55 %, FMA pipe 31 %, DRAM 19 % used; of the 4 issues that a warp waits for each
// that it makes 1.2 are for loads, 0.6 for arithmetic, 0.4 for shared memory); short rows by those of a part: its query, its pages, its codes, the
// sums.  8 rows of 8192 positions, 32/8 heads of 128: 82 us, 13 TFLOP/s, 1.6 TB/s of codes; 4 rows under a window of 1000, 16/4
// heads of 64: 10.8 us.  (With eight lanes a key, each with 16 columns of it and of the output, the sums of a score
// went through shuffles and all eight lanes formed the same exponential: 250 and 13.2 us, at two warps a scheduler for the registers.)
#include <type_traits>

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

__device__ __forceinline__ void codes4(uint32_t c, float (&f)[4]) {
  c ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(c, 0x4b000000u, 0x7540 + i)) - 8388736.f;
}

// A CTA's sums for the heads h0 .. h0 + nh - 1 of an item, in shared memory: m[h], l[h], o[h * dim + d].  A row of one chunk goes
// to the output; else the sums go to scratch memory and the CTA that comes last for the (row, tile) adds them up in the order of the
// chunks.  Every thread of the CTA calls it; weights: [most_chunks + 1][HT].
__device__ __forceinline__ void finish_item(const RowsArgs& a, const Item& x, int tiles, int h0, int nh, const float* m, const float* l,
                                            const float* o, float* weights, int* last) {
  const int D = a.dim;
  float* out = (float*)a.out + (size_t)x.row.tok * a.ldo + (size_t)h0 * D;
  if (x.n_chunks == 1) {
    for (int e = threadIdx.x; e < nh * D; e += blockDim.x) {
      const int h = e / D;
      const float total = a.sinks ? l[h] + expf(a.sinks[h0 + h] - m[h]) : l[h];
      out[e] = total != 0.f ? o[e] / total : 0.f;
    }
    return;
  }
  const size_t per = (size_t)HT * (D + 2);
  const size_t slot = ((size_t)x.index * tiles + x.tile) * a.most_chunks;
  float* mine = a.partial + (slot + x.chunk) * per;
  for (int e = threadIdx.x; e < nh * D; e += blockDim.x) __stcg(mine + 2 * HT + e, o[e]);
  if (threadIdx.x < nh) {
    __stcg(mine + threadIdx.x, m[threadIdx.x]);
    __stcg(mine + HT + threadIdx.x, l[threadIdx.x]);
  }
  __threadfence();
  __syncthreads();
  int* counter = a.counters + (size_t)x.index * tiles + x.tile;
  if (threadIdx.x == 0) *last = atomicAdd(counter, 1) == x.n_chunks - 1;
  __syncthreads();
  if (!*last) return;
  __threadfence();
  if (threadIdx.x == 0) *counter = 0;
  const float* all = a.partial + slot * per;
  // weights of the chunks: exp(m_c - M) / total, a warp a head, a lane a chunk
  const int lane = threadIdx.x & 31;
  for (int h = threadIdx.x >> 5; h < nh; h += blockDim.x >> 5) {
    float top = -INFINITY, total = 0.f;
    bool odd = false;                                  // fmaxf leaves NaN out
    for (int c = lane; c < x.n_chunks; c += 32) {
      const float mc = __ldcg(all + c * per + h);
      odd |= mc != mc;
      top = fmaxf(top, mc);
    }
    top = __any_sync(0xffffffffu, odd) ? NAN : warp_max(top);
    if (top == -INFINITY) top = 0.f;                  // no key at all has a page: zeros
    for (int c = lane; c < x.n_chunks; c += 32) {
      const float w = expf(__ldcg(all + c * per + h) - top);
      weights[c * HT + h] = w;
      total = fmaf(w, __ldcg(all + c * per + HT + h), total);
    }
    total = warp_sum(total);
    if (a.sinks) total += expf(a.sinks[h0 + h] - top);
    if (lane == 0) weights[a.most_chunks * HT + h] = total != 0.f ? 1.f / total : 0.f;
  }
  __syncthreads();
  for (int e = 4 * threadIdx.x; e < nh * D; e += 4 * blockDim.x) {
    const int h = e / D;
    const float* w = weights + h;
    const float* p = all + 2 * HT + e;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
    for (int c = 0; c < x.n_chunks; ++c) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p + c * per));
      const float wc = w[c * HT];
      sum.x = fmaf(wc, v.x, sum.x); sum.y = fmaf(wc, v.y, sum.y); sum.z = fmaf(wc, v.z, sum.z); sum.w = fmaf(wc, v.w, sum.w);
    }
    const float r = w[a.most_chunks * HT];
    out[e] = sum.x * r; out[e + 1] = sum.y * r; out[e + 2] = sum.z * r; out[e + 3] = sum.w * r;
  }
}

// DP: the head size or the power of two above it; HN: query heads of an item at most (1 or 4).
template <int DP, int HN>
__global__ void __launch_bounds__(WARPS * 32)
rows_kernel(const RowsArgs a, int tiles, int group_tiles) {
  constexpr int KC = DP < 32 ? 1 : DP / 32;           // 16-byte pieces of a key that a lane takes
  constexpr int LV = DP < 128 ? DP / 4 : 32, PC = DP / 4 / LV;      // lanes of a value, its pieces of 4 columns that a lane has
  constexpr int KP = 32 / LV, ST = BLK / KP;          // values at a time, times
  constexpr float SLACK = 8.f;
  extern __shared__ int dyn[];                        // what is kept of the rows, then the weights of the last step
  __shared__ int warp_sums[WARPS], last;
  __shared__ __align__(16) float sm_q[HN][DP < 32 ? 32 : DP], sm_p[WARPS][BLK][HN], sm_o[WARPS][HN][DP];
  __shared__ float sm_m[WARPS][HN], sm_l[WARPS][HN];
  __shared__ float fin_m[HT], fin_l[HT], fin_o[HN * DP];
  const Rows rows(dyn, a.n_rows);
  float* weights = reinterpret_cast<float*>(dyn + 4 * a.n_rows + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int total = schedule(a, rows, warp_sums) * tiles;
  const int G = a.Hq / a.Hkv, D = a.dim, per = a.page / BLK;
  const int key = lane >> 1, half = lane & 1, vk = lane / LV, col = (lane % LV) * 4;
  pdl_wait();
  pdl_trigger();
  const int8_t *k8 = after_wait(a.k8), *v8 = after_wait(a.v8);
  const float *ks = after_wait(a.ks), *vs = after_wait(a.vs);
  for (int it = blockIdx.x; it < total; it += gridDim.x) {
    const Item x = item_of(a, rows, it, tiles);
    const int hk = x.tile / group_tiles, j0 = (x.tile - hk * group_tiles) * HT, nh = min(HN, G - j0), h0 = hk * G + j0;
    const int* bt = a.block_table + (size_t)x.row.req * a.max_pages;
    const int lo = a.window > 0 ? x.row.pos - a.window + 1 : 0;
    // a quarter of the item's blocks each
    const int n_all = (x.end - x.begin + BLK - 1) / BLK, each = (n_all + WARPS - 1) / WARPS;
    const int first = x.begin + warp * each * BLK, n = max(0, min(each, n_all - warp * each));
    const float* qr = after_wait((const float*)a.q) + (size_t)x.row.tok * a.ldq + (size_t)h0 * D;
    constexpr int QW = DP < 32 ? 32 : DP;
    for (int e = threadIdx.x; e < HN * QW; e += WARPS * 32) {
      const int h = e / QW, d = e - h * QW;
      sm_q[h][d] = h < nh && d < D ? qr[h * D + d] : 0.f;
    }
    float o[HN][PC][4], m[HN], l[HN > 1 ? 2 : 1];     // (l: of heads half and 2 + half)
#pragma unroll
    for (int h = 0; h < HN; ++h) {
      m[h] = -INFINITY;
#pragma unroll
      for (int c = 0; c < PC; ++c) o[h][c][0] = o[h][c][1] = o[h][c][2] = o[h][c][3] = 0.f;
    }
    l[0] = l[HN > 1 ? 1 : 0] = 0.f;
    uint32_t tile_id = 0, missing = 0;
    float sk_of = 0.f, sv_of = 0.f;
    // lane i learns of the i-th of the warp's next 32 blocks which tile of the pool it is, and its scales
    auto look_up = [&](int i0) {
      const int i = i0 + lane, at = first + i * BLK;
      bool none = false;
      if (i < n) {
        const int pg = page_of(a, bt, at);
        none = pg < 0;
        if (!none) {
          tile_id = (uint32_t)(pg * a.Hkv + hk) * per + (at & (a.page - 1)) / BLK;
          sk_of = __ldcg(ks + tile_id);
          sv_of = __ldcg(vs + tile_id);
        }
      }
      missing = __ballot_sync(0xffffffffu, none);
    };
    auto load = [&](int i, int have, uint4 (&kx)[KC], uint32_t (&vx)[ST][PC]) {
      if (i >= have || (missing >> i & 1)) return;
      const size_t at = (size_t)__shfl_sync(0xffffffffu, tile_id, i) * (BLK * D);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int d = (2 * c + half) * 16;
        kx[c] = d < D ? __ldcg(reinterpret_cast<const uint4*>(k8 + at + key * D + d)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int c = 0; c < PC; ++c)
          vx[s][c] = col + 128 * c < D ? __ldcg(reinterpret_cast<const uint32_t*>(v8 + at + (s * KP + vk) * D + col + 128 * c)) : 0u;
    };
    auto work = [&](int i, int i32, const uint4 (&kx)[KC], const uint32_t (&vx)[ST][PC]) {
      if (missing >> i32 & 1) return;
      const float sk = __shfl_sync(0xffffffffu, sk_of, i32) * a.scale, sv = __shfl_sync(0xffffffffu, sv_of, i32);
      float t[HN], u[HN];
#pragma unroll
      for (int h = 0; h < HN; ++h) t[h] = u[h] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        float f[16];
        codes16(kx[c], f);
#pragma unroll
        for (int h = 0; h < HN; ++h) {
          const float4* qq = reinterpret_cast<const float4*>(&sm_q[h][(2 * c + half) * 16]);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 y = qq[w];
            t[h] = fmaf(y.x, f[4 * w], t[h]);
            u[h] = fmaf(y.y, f[4 * w + 1], u[h]);
            t[h] = fmaf(y.z, f[4 * w + 2], t[h]);
            u[h] = fmaf(y.w, f[4 * w + 3], u[h]);
          }
        }
      }
      bool high = false;
#pragma unroll
      for (int h = 0; h < HN; ++h) {
        t[h] += u[h];
        t[h] += __shfl_xor_sync(0xffffffffu, t[h], 1);
        t[h] *= sk;
        if (i == 0 || i == n - 1) {                   // (a window begins in a row's first block)
          const int p = first + i * BLK + key;
          if (p < lo || p >= x.end) t[h] = -INFINITY;
        }
        high |= t[h] > m[h] + SLACK;
      }
      if (__any_sync(0xffffffffu, high)) {
#pragma unroll
        for (int h = 0; h < HN; ++h) {
          float top = t[h];
#pragma unroll
          for (int d = 2; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(top, m[h]);
          const float r = expf(m[h] - (top == -INFINITY ? 0.f : top));
          m[h] = top;
          if ((h & 1) == half || HN == 1) l[h >> 1] *= r;
#pragma unroll
          for (int c = 0; c < PC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[h][c][e] *= r;
        }
      }
#pragma unroll
      for (int y = 0; y < (HN > 1 ? 2 : 1); ++y) {
        const float tt = HN > 1 && half ? t[HN > 1 ? 2 * y + 1 : 0] : t[2 * y], mm = HN > 1 && half ? m[HN > 1 ? 2 * y + 1 : 0] : m[2 * y];
        const float p = expf(tt - (mm == -INFINITY ? 0.f : mm));
        l[y] += p;
        if (HN > 1 || half == 0) sm_p[warp][key][HN > 1 ? 2 * y + half : 0] = p * sv;
      }
      __syncwarp();
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        float p[HN];
        if constexpr (HN == 4) {
          const float4 w = *reinterpret_cast<const float4*>(sm_p[warp][s * KP + vk]);
          p[0] = w.x; p[HN > 1 ? 1 : 0] = w.y; p[HN > 2 ? 2 : 0] = w.z; p[HN > 3 ? 3 : 0] = w.w;
        } else {
          p[0] = sm_p[warp][s * KP + vk][0];
        }
#pragma unroll
        for (int c = 0; c < PC; ++c) {
          float f[4];
          codes4(vx[s][c], f);
#pragma unroll
          for (int h = 0; h < HN; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[h][c][e] = fmaf(p[h], f[e], o[h][c][e]);
        }
      }
      __syncwarp();                                   // the weights have been read
    };
    __syncthreads();                                  // the queries are there
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int have = min(32, n - i0);
      look_up(i0);
      uint4 kx[2][KC];
      uint32_t vx[2][ST][PC];
      load(0, have, kx[0], vx[0]);
      for (int i = 0; i < have; i += 2) {
        load(i + 1, have, kx[1], vx[1]);
        work(i0 + i, i, kx[0], vx[0]);
        if (i + 1 >= have) break;
        load(i + 2, have, kx[0], vx[0]);
        work(i0 + i + 1, i + 1, kx[1], vx[1]);
      }
    }
    // the lanes of a warp, then the warps
#pragma unroll
    for (int y = 0; y < (HN > 1 ? 2 : 1); ++y) {
#pragma unroll
      for (int d = 2; d < 32; d <<= 1) l[y] += __shfl_xor_sync(0xffffffffu, l[y], d);
      if (lane == half && (HN > 1 || half == 0)) sm_l[warp][HN > 1 ? 2 * y + half : 0] = l[y];
    }
#pragma unroll
    for (int h = 0; h < HN; ++h) {
      if (lane == 0) sm_m[warp][h] = m[h];
#pragma unroll
      for (int c = 0; c < PC; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int d = LV; d < 32; d <<= 1) o[h][c][e] += __shfl_xor_sync(0xffffffffu, o[h][c][e], d);
        if (vk == 0) *reinterpret_cast<float4*>(&sm_o[warp][h][col + 128 * c]) = make_float4(o[h][c][0], o[h][c][1], o[h][c][2], o[h][c][3]);
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
    finish_item(a, x, tiles, h0, nh, fin_m, fin_l, fin_o, weights, &last);
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
  auto sized = [&](auto heads) {
    constexpr int HN = decltype(heads)::value;
    if (dim <= 16) go(rows_kernel<16, HN>);
    else if (dim <= 32) go(rows_kernel<32, HN>);
    else if (dim <= 64) go(rows_kernel<64, HN>);
    else if (dim <= 128) go(rows_kernel<128, HN>);
    else go(rows_kernel<256, HN>);
  };
  if (Hq == Hkv) sized(std::integral_constant<int, 1>{});
  else sized(std::integral_constant<int, HT>{});
  return mlxb_check_launch("kv8_rows");
}
