// What the kernels for single queries over pages in 8 bits share: how the rows' keys are cut into items, and how an item's result
// becomes a row of the output.
//
// A row (one query of each head, at position p of its request) sees keys max(0, p - window + 1) .. p.  They are cut into chunks that
// begin at multiples of 16 positions; how many there are goes by the row's own number of keys and by the numbers of heads, never by
// what else is in the batch, so that a row's bits do not depend on its neighbours.  An item is a chunk of a row for one tile of query
// heads that read the same key/value head.  The grid is as large as the device (or the most items there can be) and every CTA walks
// items blockIdx.x, blockIdx.x + gridDim.x, ...: lengths are known on the device only, and a grid for the longest row would be mostly
// empty blocks.  The items of all rows are numbered by a prefix sum that each CTA forms for itself.
#pragma once

#include "common.cuh"

constexpr int BLK = 16;              // positions that share a scale
constexpr int ROWS_MOST = 1024;      // rows a launch takes: what a CTA knows of them is in shared memory

struct RowsArgs {
  const void* q;
  int ldq;
  const int *rows, *positions, *token_req, *block_table;
  int n_tokens, n_req, max_pages, n_pages, page, Hq, Hkv, dim, window;
  float scale;
  const int8_t *k8, *v8;
  const float *ks, *vs, *sinks;
  float* partial;
  int* counters;
  int most_chunks, least_chunk;      // how many chunks of a row at most, of how many keys at least
  void* out;
  int ldo, n_rows;
  int* status;
};

// Keys of a chunk for a row of n keys: `least` (a multiple of 64) or more, in at most `most` chunks.
__device__ __forceinline__ int chunk_keys(int n, int most, int least) {
  const int c = ((n + most - 1) / most + 63) & ~63;
  return c > least ? c : least;
}

struct RowSpan { int tok, req, pos, first, n; };      // first: a multiple of 16; n: keys from there to the query (0: no such row)

__device__ __forceinline__ RowSpan span_of(const RowsArgs& a, int tok, int req, int pos) {
  RowSpan s{tok, req, pos, 0, 0};
  if (req < 0 || req >= a.n_req || pos < 0 || pos / a.page >= a.max_pages) return s;      // a row that pads the step, or one out of range
  const int lo = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
  s.first = lo & ~(BLK - 1);
  s.n = pos + 1 - s.first;
  return s;
}
__device__ __forceinline__ RowSpan row_span(const RowsArgs& a, int i) {
  const int tok = a.rows ? a.rows[i] : i;
  if ((unsigned)tok >= (unsigned)a.n_tokens) return RowSpan{0, a.n_req, 0, 0, 0};
  return span_of(a, tok, a.token_req[tok], a.positions[tok]);
}
__device__ __forceinline__ int chunks_of(const RowsArgs& a, int n) {
  if (n == 0) return 0;
  const int keys = chunk_keys(n, a.most_chunks, a.least_chunk);
  return (n + keys - 1) / keys;
}

// What a CTA keeps of the rows: 4 n_rows + 1 integers.
struct Rows {
  int *prefix, *tok, *req, *pos;     // prefix[i]: chunks of the rows before row i
  __device__ __forceinline__ Rows(int* mem, int n) : prefix(mem), tok(mem + n + 1), req(tok + n), pos(req + n) {}
};
static inline size_t rows_bytes(int n_rows) { return (size_t)(4 * n_rows + 1) * 4; }

// Fills `rows` in; returns the number of all chunks.  Every thread of the CTA calls it.
__device__ __forceinline__ int schedule(const RowsArgs& a, const Rows& rows, int* warp_sums) {
  const int n = a.n_rows, seg = (n + blockDim.x - 1) / blockDim.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
  const int b = min(n, (int)threadIdx.x * seg), e = min(n, b + seg);
  int sum = 0;
  for (int i = b; i < e; ++i) {
    const RowSpan s = row_span(a, i);
    if (s.n == 0 && s.req >= 0 && blockIdx.x == 0) atomicOr(a.status, MLXB_ST_POSITION_RANGE);
    const int c = chunks_of(a, s.n);
    rows.tok[i] = s.tok;
    rows.req[i] = s.req;
    rows.pos[i] = s.pos;
    rows.prefix[i + 1] = c;
    sum += c;
  }
  int run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  int before = run - sum;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
  int total = 0;
  for (int w = 0; w < n_warps; ++w) total += warp_sums[w];
  for (int i = b; i < e; ++i) { before += rows.prefix[i + 1]; rows.prefix[i + 1] = before; }
  if (threadIdx.x == 0) rows.prefix[0] = 0;
  __syncthreads();
  return total;
}

struct Item {
  RowSpan row;
  int index, chunk, n_chunks, begin, end, tile;       // keys begin .. end - 1 (begin a multiple of 16)
};

// Item `it` of `tiles` tiles of heads: neighbouring items are the tiles of one chunk, whose pages lie together.
__device__ __forceinline__ Item item_of(const RowsArgs& a, const Rows& rows, int it, int tiles) {
  Item x;
  const int g = it / tiles;
  x.tile = it - g * tiles;
  int lo = 0, hi = a.n_rows - 1;                      // the last row whose prefix is <= g
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (rows.prefix[mid] <= g) lo = mid; else hi = mid - 1;
  }
  x.index = lo;
  x.chunk = g - rows.prefix[lo];
  x.n_chunks = rows.prefix[lo + 1] - rows.prefix[lo];
  x.row = span_of(a, rows.tok[lo], rows.req[lo], rows.pos[lo]);
  const int c = chunk_keys(x.row.n, a.most_chunks, a.least_chunk);
  x.begin = x.row.first + x.chunk * c;
  x.end = min(x.begin + c, x.row.pos + 1);
  return x;
}

// The page of a key, or -1 where the request has none (reported).
__device__ __forceinline__ int page_of(const RowsArgs& a, const int* bt, int key) {
  const int pg = bt[key / a.page];
  if (pg >= 0 && pg < a.n_pages) return pg;
  atomicOr(a.status, pg < 0 ? MLXB_ST_POSITION_RANGE : MLXB_ST_PAGE_RANGE);
  return -1;
}

// A CTA's sums for the heads h0 .. h0 + nh - 1 of an item, in shared memory: m[h], l[h], o[h * dim + d].  A row of one chunk goes
// to the output; else the sums go to scratch memory and the CTA that comes last for the (row, tile) adds them up in the order of the
// chunks.  Exp(x): the exponential in the unit of m.  Every thread of the CTA calls it; weights: [most_chunks][nh].
template <typename T, typename Exp>
__device__ __forceinline__ void finish_item(const RowsArgs& a, const Item& x, int tiles, int tile_heads, int h0, int nh, const float* m,
                                            const float* l, const float* o, float* weights, int* last, float sink_unit, Exp exp_) {
  const int D = a.dim;
  T* out = (T*)a.out + (size_t)x.row.tok * a.ldo + (size_t)h0 * D;
  if (x.n_chunks == 1) {
    for (int e = threadIdx.x; e < nh * D; e += blockDim.x) {
      const int h = e / D;
      const float total = a.sinks ? l[h] + exp_(a.sinks[h0 + h] * sink_unit - m[h]) : l[h];
      out[e] = from_f<T>(total != 0.f ? o[e] / total : 0.f);
    }
    return;
  }
  const size_t per = (size_t)tile_heads * (D + 2);
  const size_t slot = ((size_t)x.index * tiles + x.tile) * a.most_chunks;
  float* mine = a.partial + (slot + x.chunk) * per;
  for (int e = threadIdx.x; e < nh * D; e += blockDim.x) __stcg(mine + 2 * tile_heads + e, o[e]);
  if (threadIdx.x < nh) {
    __stcg(mine + threadIdx.x, m[threadIdx.x]);
    __stcg(mine + tile_heads + threadIdx.x, l[threadIdx.x]);
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
      const float w = exp_(__ldcg(all + c * per + h) - top);
      weights[c * tile_heads + h] = w;
      total = fmaf(w, __ldcg(all + c * per + tile_heads + h), total);
    }
    total = warp_sum(total);
    if (a.sinks) total += exp_(a.sinks[h0 + h] * sink_unit - top);
    if (lane == 0) weights[a.most_chunks * tile_heads + h] = total != 0.f ? 1.f / total : 0.f;
  }
  __syncthreads();
  for (int e = 4 * threadIdx.x; e < nh * D; e += 4 * blockDim.x) {
    const int h = e / D;
    const float* w = weights + h;
    const float* p = all + 2 * tile_heads + e;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
    for (int c = 0; c < x.n_chunks; ++c) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p + c * per));
      const float wc = w[c * tile_heads];
      sum.x = fmaf(wc, v.x, sum.x); sum.y = fmaf(wc, v.y, sum.y); sum.z = fmaf(wc, v.z, sum.z); sum.w = fmaf(wc, v.w, sum.w);
    }
    const float r = w[a.most_chunks * tile_heads];
    out[e] = from_f<T>(sum.x * r); out[e + 1] = from_f<T>(sum.y * r);
    out[e + 2] = from_f<T>(sum.z * r); out[e + 3] = from_f<T>(sum.w * r);
  }
}

// Arguments of the entry points as one record of 8-byte fields: the caller fills it in a tenth of the time that as many arguments of a
// call take it.
struct RowsRecord {
  const void* q;
  const int *rows, *positions, *token_req, *block_table;
  const int8_t *k8, *v8;
  const float *ks, *vs, *sinks;
  float* partial;
  int* counters;
  void* out;
  int* status;
  long long ldq, n_tokens, n_req, max_pages, n_pages, page, Hq, Hkv, dim, window, most_chunks, least_chunk, ldo, n_rows;
  double scale;
};

static inline int rows_args(const RowsRecord* rec, long long bytes, const char* what, RowsArgs& a) {
  if (!rec || bytes != sizeof(RowsRecord)) return mlxb_fail(MLXB_BAD_ARG, "%s: a record of %lld bytes", what, bytes);
  const RowsRecord& x = *rec;
  a = RowsArgs{x.q, (int)x.ldq, x.rows, x.positions, x.token_req, x.block_table, (int)x.n_tokens, (int)x.n_req, (int)x.max_pages, (int)x.n_pages,
               (int)x.page, (int)x.Hq, (int)x.Hkv, (int)x.dim, (int)x.window, (float)x.scale, x.k8, x.v8, x.ks, x.vs, x.sinks, x.partial, x.counters,
               (int)x.most_chunks, (int)x.least_chunk, x.out, (int)x.ldo, (int)x.n_rows, x.status};
  if (a.n_rows > ROWS_MOST) return mlxb_fail(MLXB_BAD_ARG, "%s: %d rows, a launch takes %d", what, a.n_rows, ROWS_MOST);
  if (a.Hkv <= 0 || a.Hq <= 0 || a.Hq % a.Hkv) return mlxb_fail(MLXB_BAD_ARG, "%s: %d query heads over %d key/value heads", what, a.Hq, a.Hkv);
  if (a.dim % 16 || a.dim < 16 || a.dim > 256) return mlxb_fail(MLXB_BAD_ARG, "%s: head size %d (a multiple of 16 up to 256)", what, a.dim);
  if (a.page < BLK || (a.page & (a.page - 1)))
    return mlxb_fail(MLXB_BAD_ARG, "%s: page size %d (a power of two of at least %d)", what, a.page, BLK);
  if (a.most_chunks <= 0 || a.most_chunks > 1024 || a.least_chunk < 64 || a.least_chunk % 64)
    return mlxb_fail(MLXB_BAD_ARG, "%s: %d chunks of a row, of %d keys at least", what, a.most_chunks, a.least_chunk);
  if (((uintptr_t)a.k8 | (uintptr_t)a.v8 | (uintptr_t)a.partial) & 15)
    return mlxb_fail(MLXB_BAD_ARG, "%s: pools and scratch memory must be 16-byte aligned", what);
  return 0;
}
