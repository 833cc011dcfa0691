// Rows into 8-bit floating point (the format and layout are in fp8.cuh).
//
// fp8_quantize   rows of a matrix, or of a stack of them (groups): weights once, a layer's input every step.
// fp8_gather     the rows of a plan's slots (moe_plan, moe_route_plan): tile t of the plan gets rows tile_rows * t .. and a tile of scales of its
//                own, so that the products' tiles begin where their scales do, wherever an expert's slots begin.
//
// A warp takes 512 columns of a row, a lane 16 neighbours: the eight lanes of a run of 128 find its largest magnitude in three
// exchanges, a lane's codes are one store of 16 bytes and the four scales one word.  Every number is read once.  Large matrices are bound by their bytes (8192 x
// 8192 bfloat16: 34 us, 5.9 TB/s), small ones are a chain of latencies (1.5 us behind another kernel).  Gathering rounds a row once for each of its slots:
// 32768 slots of 2048 columns, 8 a row, take 33 us, bound by instructions (71 % of the issue slots; 201 MB through the L2, 29 MB of them from memory).
#include "fp8.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int FQ_WARPS = 8;

// 16 neighbours of a row of T, as they lie in memory; zeros behind column K.  VEC: K, the row's stride and its address are such that they
// lie in whole 16-byte pieces.
template <typename T>
struct Sixteen {
  uint32_t w[4 * sizeof(T)];
  template <bool VEC>
  __device__ __forceinline__ void load(const T* row, int c, int K) {
    if (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) {
        const uint4 u = c + i * (16 / (int)sizeof(T)) < K ? reinterpret_cast<const uint4*>(row + c)[i] : make_uint4(0u, 0u, 0u, 0u);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else if (sizeof(T) == 2) {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t lo = c + 2 * i < K ? p[c + 2 * i] : 0u, hi = c + 2 * i + 1 < K ? p[c + 2 * i + 1] : 0u;
        w[i] = lo | hi << 16;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = c + i < K ? reinterpret_cast<const uint32_t*>(row)[c + i] : 0u;
    }
  }
  __device__ __forceinline__ float number(int i) const {
    if (sizeof(T) == 2) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    return __uint_as_float(w[i]);
  }
  // the bits (of a float32) of the largest magnitude, not finite ones too: NaN beats all others
  __device__ __forceinline__ uint32_t largest() const {
    if constexpr (sizeof(T) == 2) {
      uint32_t top = w[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(w[i]));
      top &= 0x7fff7fffu;
      return max(top << 16, top & 0xffff0000u);
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, w[i] & 0x7fffffffu);
      return top;
    }
  }
};

__device__ __forceinline__ uint32_t run_max(uint32_t v) {        // over the eight lanes of a run
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 512 columns of one row, by a warp: codes to `out` (this lane's 16; `in`: they exist), the four scales to `scale` (the row's word in its tile)
template <typename T>
__device__ __forceinline__ void quantize512(const Sixteen<T>& x, bool in, uint8_t* out, uint8_t* scale, int lane) {
  uint32_t top = run_max(x.largest());
  int e;
  uint32_t w[4];
  if (__all_sync(0xffffffffu, top < 0x7f800000u)) {
    e = fp8_exponent(top);
    const float f = fp8_power(-e);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = fp8_quad(x.number(4 * i) * f, x.number(4 * i + 1) * f, x.number(4 * i + 2) * f, x.number(4 * i + 3) * f);
  } else {                                                        // rare: something is not finite
    top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, fp8_magnitude(x.number(i)));
    e = fp8_exponent(run_max(top));
    const float f = fp8_power(-e);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = fp8_quad(fp8_or_nan(x.number(4 * i)) * f, fp8_or_nan(x.number(4 * i + 1)) * f, fp8_or_nan(x.number(4 * i + 2)) * f, fp8_or_nan(x.number(4 * i + 3)) * f);
  }
  if (in) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  uint32_t s = (uint32_t)(e + 127) << (8 * (lane >> 3));
  s |= __shfl_xor_sync(0xffffffffu, s, 8);
  s |= __shfl_xor_sync(0xffffffffu, s, 16);
  if (lane == 0) *reinterpret_cast<uint32_t*>(scale) = s;
}

// AT items of a warp have their loads out together: one where a call is a chain of latencies (4096 x 4096 bfloat16: 10.4 us beside 11.0 with four), four where it is
// bytes (8192 x 8192: 34.2 us, 5.9 TB/s, beside 37.2).  float32 has twice the bytes out with one and gains nothing (57.1 beside 57.6).
template <typename T, bool VEC, int AT>
__global__ void __launch_bounds__(32 * FQ_WARPS, AT == 1 ? 8 : 4)
fp8_quantize_kernel(const T* x, long long ldx, int rows, int K, int group_rows, uint8_t* __restrict__ codes, int ld, uint8_t* __restrict__ scales) {
  pdl_wait();
  // The next kernel starts early behind few rows only: behind many its CTAs would take the registers this one runs in (8192 x 8192: 75 us instead of 40).
  if (AT == 1 && rows <= 128) pdl_trigger();
  x = after_wait(x);
  const int lane = threadIdx.x & 31, kgs = (K + 511) >> 9, tiles = (group_rows + 127) >> 7;
  const long long items = (long long)rows * kgs, first = ((long long)blockIdx.x * FQ_WARPS + (threadIdx.x >> 5)) * AT;
  if (first >= items) return;
  Sixteen<T> v[AT];
  long long r = first / kgs;
  int kg = (int)(first - r * kgs);
  const long long r0 = r;
  const int kg0 = kg;
#pragma unroll
  for (int j = 0; j < AT; ++j) {
    if (r < rows) v[j].template load<VEC>(x + r * ldx, 512 * kg + 16 * lane, K);
    if (++kg == kgs) { kg = 0; ++r; }
  }
  r = r0;
  kg = kg0;
  int group = (int)(r / group_rows), in = (int)(r - (long long)group * group_rows);
#pragma unroll
  for (int j = 0; j < AT; ++j) {
    if (r >= rows) return;
    quantize512<T>(v[j], 512 * kg + 16 * lane < ld, codes + r * ld + 512 * kg + 16 * lane, scales + (((long long)group * tiles + (in >> 7)) * kgs + kg) * FP8_TILE + fp8_scale_row(in), lane);
    if (++kg == kgs) {
      kg = 0;
      ++r;
      if (++in == group_rows) { in = 0; ++group; }
    }
  }
}

// A warp takes a row of a tile (where there are few, a part of its columns).  Blocks are short so that the last ones to run are few: with four
// rows a warp 32768 rows of 2048 took 37 us, 1.1 rounds of blocks over the SMs being two.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * FQ_WARPS, VEC && sizeof(T) == 2 ? 6 : 4)
fp8_gather_kernel(const T* x, long long ldx, int K, int a_div, const int* sorted, const int* tile_info, const int* n_tiles, int tile_rows,
                  uint8_t* __restrict__ codes, int ld, uint8_t* __restrict__ scales, int S, bool few) {
  pdl_wait();
  if (few) pdl_trigger();           // many rows: the next kernel's CTAs would take the registers this one runs in
  x = after_wait(x);
  sorted = after_wait(sorted);
  tile_info = after_wait(tile_info);
  const int t = blockIdx.x, have = after_wait(n_tiles)[0], first = tile_info[3 * t + 1], rows = min(tile_rows, tile_info[3 * t + 2]);
  if (t >= have || rows <= 0) return;
  const int lane = threadIdx.x & 31, kgs = (K + 511) >> 9, warps = gridDim.y * FQ_WARPS, warp = blockIdx.y * FQ_WARPS + (threadIdx.x >> 5);
  const int parts = max(1, min(kgs, warps / rows)), row_warps = warps / parts, part = warp / row_warps;
  if (part >= parts) return;
  for (int r = warp - part * row_warps; r < rows; r += row_warps) {
    const int place = first + r, slot = place >= 0 && place < S ? sorted[place] : -1;
    if (slot < 0 || slot >= S) continue;             // no plan says so
    const T* px = x + (long long)(slot / a_div) * ldx;
    uint8_t* pc = codes + ((long long)t * tile_rows + r) * ld;
    uint8_t* ps = scales + (long long)t * kgs * FP8_TILE + fp8_scale_row(r);
    for (int kg = part; kg < kgs; kg += parts) {
      const int c = 512 * kg + 16 * lane;
      Sixteen<T> v;
      v.template load<VEC>(px, c, K);
      quantize512<T>(v, c < ld, pc + c, ps + kg * FP8_TILE, lane);
    }
  }
}

template <typename T>
static bool whole_pieces(const void* x, long long ldx, int K) {
  return !(K & (16 / (int)sizeof(T) - 1)) && !(((uintptr_t)x | (uintptr_t)(ldx * (long long)sizeof(T))) & 15);
}

static int check(const char* what, const void* x, int K, long long ldx, const void* codes, int ld, const void* scales) {
  if (!x || !codes || !scales || K <= 0 || ldx < K || ld < K || (ld & 15) || (((uintptr_t)codes | (uintptr_t)scales) & 15))
    return mlxb_fail(MLXB_BAD_ARG, "%s: rows of %d at stride %lld, codes at stride %d", what, K, ldx, ld);
  return 0;
}

// Arguments as records of 8-byte fields: a caller fills one in a tenth of the time of as many arguments.
struct QuantizeRecord {
  const void* x;
  void *codes, *scales;
  long long dtype, ldx, rows, K, group_rows, ld;
};
struct GatherRecord {
  const void* x;
  const int *sorted, *tile_info, *n_tiles;
  void *codes, *scales;
  long long dtype, ldx, K, a_div, S, max_tiles, tile_rows, ld;
};

// x: `dtype` [rows, K] at row stride ldx; codes [rows, ld] with ld = K rounded up to 16; scales as in fp8.cuh for groups of group_rows rows.
MLXB_EXPORT int mlxb_fp8_quantize(const QuantizeRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(QuantizeRecord)) return mlxb_fail(MLXB_BAD_ARG, "fp8_quantize: a record of %lld bytes", bytes);
  if (rec->rows > 0x7fffffffLL || rec->K > 0x7fffff00LL) return mlxb_fail(MLXB_BAD_ARG, "fp8_quantize: %lld rows of %lld", rec->rows, rec->K);
  const void* x = rec->x;
  void *codes = rec->codes, *scales = rec->scales;
  const int dtype = (int)rec->dtype, rows = (int)rec->rows, K = (int)rec->K, group_rows = (int)rec->group_rows, ld = (int)rec->ld;
  const long long ldx = rec->ldx;
  if (rows <= 0) return 0;
  if (int e = check("fp8_quantize", x, K, ldx, codes, ld, scales)) return e;
  if (group_rows <= 0 || rows % group_rows) return mlxb_fail(MLXB_BAD_ARG, "fp8_quantize: %d rows in groups of %d", rows, group_rows);
  const long long items = (long long)rows * ((K + 511) / 512);
  const bool many = dtype == MLXB_BF16 && whole_pieces<__nv_bfloat16>(x, ldx, K) && items >= 32LL * FQ_WARPS * mlxb_sm_count();
  const long long blocks = many ? (items + 4 * FQ_WARPS - 1) / (4 * FQ_WARPS) : (items + FQ_WARPS - 1) / FQ_WARPS;
  if (blocks > 0x7fffffffLL) return mlxb_fail(MLXB_BAD_ARG, "fp8_quantize: %d rows of %d", rows, K);
#define LAUNCH(T, V, AT)                                                                                                                        \
  launch_pdl(fp8_quantize_kernel<T, V, AT>, dim3((unsigned)blocks), dim3(32 * FQ_WARPS), 0, stream, (const T*)x, ldx, rows, K, group_rows, \
             (uint8_t*)codes, ld, (uint8_t*)scales)
  if (dtype == MLXB_BF16) {
    if (many) LAUNCH(__nv_bfloat16, true, 4);
    else if (whole_pieces<__nv_bfloat16>(x, ldx, K)) LAUNCH(__nv_bfloat16, true, 1);
    else LAUNCH(__nv_bfloat16, false, 1);
  } else if (dtype == MLXB_F32) {
    if (whole_pieces<float>(x, ldx, K)) LAUNCH(float, true, 1);
    else LAUNCH(float, false, 1);
  } else {
    return mlxb_fail(MLXB_BAD_DTYPE, "fp8_quantize: dtype code %d", dtype);
  }
#undef LAUNCH
  return mlxb_check_launch("fp8_quantize");
}

// The rows of a plan with tiles of tile_rows slots: row first + i of tile t is row sorted[first + i] / a_div of x and row tile_rows * t + i of
// codes; scales are a group a tile.  Rows of a tile behind its last slot are left as they were.
MLXB_EXPORT int mlxb_fp8_gather(const GatherRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(GatherRecord)) return mlxb_fail(MLXB_BAD_ARG, "moe_gather_fp8: a record of %lld bytes", bytes);
  if (rec->K > 0x7fffff00LL || rec->max_tiles > 0x7fffffffLL || rec->S > 0x7fffffffLL) return mlxb_fail(MLXB_BAD_ARG, "moe_gather_fp8: rows of %lld, %lld tiles", rec->K, rec->max_tiles);
  const void* x = rec->x;
  const int *sorted = rec->sorted, *tile_info = rec->tile_info, *n_tiles = rec->n_tiles;
  void *codes = rec->codes, *scales = rec->scales;
  const int dtype = (int)rec->dtype, K = (int)rec->K, a_div = (int)rec->a_div, S = (int)rec->S, max_tiles = (int)rec->max_tiles, tile_rows = (int)rec->tile_rows, ld = (int)rec->ld;
  const long long ldx = rec->ldx;
  if (max_tiles <= 0) return 0;
  if (int e = check("moe_gather_fp8", x, K, ldx, codes, ld, scales)) return e;
  if (a_div <= 0 || (tile_rows != 16 && tile_rows != 128)) return mlxb_fail(MLXB_BAD_ARG, "moe_gather_fp8: tiles of %d rows", tile_rows);
  const dim3 grid(max_tiles, tile_rows / FQ_WARPS);
  const bool few = (long long)grid.x * grid.y <= 4LL * mlxb_sm_count();
#define GO(T, V)                                                                                                                             \
  launch_pdl(fp8_gather_kernel<T, V>, grid, dim3(32 * FQ_WARPS), 0, stream, (const T*)x, ldx, K, a_div, sorted, tile_info, n_tiles, tile_rows, \
             (uint8_t*)codes, ld, (uint8_t*)scales, S, few)
  if (dtype == MLXB_BF16) {
    if (whole_pieces<__nv_bfloat16>(x, ldx, K)) GO(__nv_bfloat16, true);
    else GO(__nv_bfloat16, false);
  } else if (dtype == MLXB_F32) {
    if (whole_pieces<float>(x, ldx, K)) GO(float, true);
    else GO(float, false);
  } else {
    return mlxb_fail(MLXB_BAD_DTYPE, "moe_gather_fp8: dtype code %d", dtype);
  }
#undef GO
  return mlxb_check_launch("moe_gather_fp8");
}
