// What the kernels for single queries over pages in 8 bits share: their arguments, and how the rows' keys are cut into items.
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
