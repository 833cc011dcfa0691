// Rows into 8-bit floating point (the format and layout are in fp8.cuh).
//
// fp8_quantize   rows of a matrix, or of a stack of them (groups): weights once, a layer's input every step.
// fp8_gather     the rows of a plan's slots (moe_plan, moe_route_plan): tile t of the plan gets rows tile_rows * t .. and a tile of scales of its
//                own, so that the products' tiles begin where their scales do, wherever an expert's slots begin.
//
// A warp takes 512 columns of a row, a lane 16 neighbours: the eight lanes of a run of 128 find its largest magnitude in three
// exchanges, a lane's codes are one store of 16 bytes and the four scales one word.  Every number is read once; the kernel is bound by
// its bytes.
#include "fp8.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int FQ_WARPS = 8;

// 16 numbers from column c on; zeros behind column K.  VEC: K, the row's stride and its address are such that 16 of them are whole 16-byte pieces.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* row, int c, int K, float (&v)[16]) {
  if (VEC) {
    if (c < K) {
      const uint4* p = reinterpret_cast<const uint4*>(row + c);
      if (sizeof(T) == 2) {
        const uint4 a = p[0], b = p[1];
        float lo[8], hi[8];
        unpack8(a, lo);
        unpack8(b, hi);
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i] = lo[i]; v[8 + i] = hi[i]; }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 a = p[i];
          v[4 * i] = __uint_as_float(a.x); v[4 * i + 1] = __uint_as_float(a.y);
          v[4 * i + 2] = __uint_as_float(a.z); v[4 * i + 3] = __uint_as_float(a.w);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < K ? to_f(row[c + i]) : 0.f;
  }
}

// 512 columns from 512 * kg on of one row, by a warp: codes to `out` (the row), the four scales to `scale` (the row's word in its tile)
template <typename T, bool VEC>
__device__ __forceinline__ void quantize512(const T* row, int kg, int K, int ld, uint8_t* out, uint8_t* scale, int lane) {
  const int c = 512 * kg + 16 * lane;
  float v[16];
  load16<T, VEC>(row, c, K, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, fp8_magnitude(v[i]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = fp8_exponent(top);
  const float f = fp8_power(-e);
  uint4 u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = fp8_quad(v[4 * i] * f, v[4 * i + 1] * f, v[4 * i + 2] * f, v[4 * i + 3] * f);
  if (c < ld) *reinterpret_cast<uint4*>(out + c) = u;
  uint32_t s = (uint32_t)(e + 127) << (8 * (lane >> 3));
  s |= __shfl_xor_sync(0xffffffffu, s, 8);
  s |= __shfl_xor_sync(0xffffffffu, s, 16);
  if (lane == 0) *reinterpret_cast<uint32_t*>(scale) = s;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * FQ_WARPS)
fp8_quantize_kernel(const T* x, long long ldx, int rows, int K, int group_rows, uint8_t* __restrict__ codes, int ld, uint8_t* __restrict__ scales) {
  pdl_wait();
  pdl_trigger();
  x = after_wait(x);
  const int lane = threadIdx.x & 31, kgs = (K + 511) >> 9;
  const long long w = (long long)blockIdx.x * FQ_WARPS + (threadIdx.x >> 5);
  const long long r = w / kgs;
  if (r >= rows) return;
  const int kg = (int)(w - r * kgs);
  const int group = (int)(r / group_rows), in = (int)(r - (long long)group * group_rows);
  const int tiles = (group_rows + 127) >> 7;
  quantize512<T, VEC>(x + r * ldx, kg, K, ld, codes + r * ld, scales + (((long long)group * tiles + (in >> 7)) * kgs + kg) * FP8_TILE + fp8_scale_row(in), lane);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * FQ_WARPS)
fp8_gather_kernel(const T* x, long long ldx, int K, int a_div, const int* sorted, const int* tile_info, const int* n_tiles, int tile_rows,
                  uint8_t* __restrict__ codes, int ld, uint8_t* __restrict__ scales) {
  pdl_wait();
  pdl_trigger();
  x = after_wait(x);
  sorted = after_wait(sorted);
  tile_info = after_wait(tile_info);
  const int t = blockIdx.x;
  if (t >= after_wait(n_tiles)[0]) return;
  const int first = tile_info[3 * t + 1], items = tile_info[3 * t + 2];
  const int lane = threadIdx.x & 31, kgs = (K + 511) >> 9;
  for (int w = blockIdx.y * FQ_WARPS + (threadIdx.x >> 5); w < items * kgs; w += gridDim.y * FQ_WARPS) {
    const int r = w / kgs, kg = w - r * kgs;
    const long long src = sorted[first + r] / a_div;
    quantize512<T, VEC>(x + src * ldx, kg, K, ld, codes + ((long long)t * tile_rows + r) * ld, scales + ((long long)t * kgs + kg) * FP8_TILE + fp8_scale_row(r), lane);
  }
}

template <typename T>
static bool whole_pieces(const void* x, long long ldx, int K) {
  return !(K & 15) && !(((uintptr_t)x | (uintptr_t)(ldx * (long long)sizeof(T))) & 15);
}

static int check(const char* what, const void* x, int K, long long ldx, const void* codes, int ld, const void* scales) {
  if (!x || !codes || !scales || K <= 0 || ldx < K || ld < K || (ld & 15) || (((uintptr_t)codes | (uintptr_t)scales) & 15))
    return mlxb_fail(MLXB_BAD_ARG, "%s: rows of %d at stride %lld, codes at stride %d", what, K, ldx, ld);
  return 0;
}

// x: `dtype` [rows, K] at row stride ldx; codes [rows, ld] with ld = K rounded up to 16; scales as in fp8.cuh for groups of group_rows rows.
MLXB_EXPORT int mlxb_fp8_quantize(int dtype, const void* x, long long ldx, int rows, int K, int group_rows, void* codes, int ld, void* scales,
                                  cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (int e = check("fp8_quantize", x, K, ldx, codes, ld, scales)) return e;
  if (group_rows <= 0 || rows % group_rows) return mlxb_fail(MLXB_BAD_ARG, "fp8_quantize: %d rows in groups of %d", rows, group_rows);
  const long long blocks = ((long long)rows * ((K + 511) / 512) + FQ_WARPS - 1) / FQ_WARPS;
  if (blocks > 0x7fffffffLL) return mlxb_fail(MLXB_BAD_ARG, "fp8_quantize: %d rows of %d", rows, K);
#define GO(T, V)                                                                                                                             \
  launch_pdl(fp8_quantize_kernel<T, V>, dim3((unsigned)blocks), dim3(32 * FQ_WARPS), 0, stream, (const T*)x, ldx, rows, K, group_rows, \
             (uint8_t*)codes, ld, (uint8_t*)scales)
  if (dtype == MLXB_BF16) {
    if (whole_pieces<__nv_bfloat16>(x, ldx, K)) GO(__nv_bfloat16, true);
    else GO(__nv_bfloat16, false);
  } else if (dtype == MLXB_F32) {
    if (whole_pieces<float>(x, ldx, K)) GO(float, true);
    else GO(float, false);
  } else {
    return mlxb_fail(MLXB_BAD_DTYPE, "fp8_quantize: dtype code %d", dtype);
  }
#undef GO
  return mlxb_check_launch("fp8_quantize");
}

// The rows of a plan with tiles of tile_rows slots: row first + i of tile t is row sorted[first + i] / a_div of x and row tile_rows * t + i of
// codes; scales are a group a tile.  Rows of a tile behind its last slot are left as they were.
MLXB_EXPORT int mlxb_fp8_gather(int dtype, const void* x, long long ldx, int K, int a_div, const int* sorted, const int* tile_info,
                                const int* n_tiles, int max_tiles, int tile_rows, void* codes, int ld, void* scales, cudaStream_t stream) {
  if (max_tiles <= 0) return 0;
  if (int e = check("moe_gather_fp8", x, K, ldx, codes, ld, scales)) return e;
  if (a_div <= 0 || tile_rows <= 0 || tile_rows > 128) return mlxb_fail(MLXB_BAD_ARG, "moe_gather_fp8: tiles of %d rows", tile_rows);
  const int most = tile_rows * ((K + 511) / 512);
  const dim3 grid(max_tiles, max(1, min(16, most / FQ_WARPS / 4)));
#define GO(T, V)                                                                                                                             \
  launch_pdl(fp8_gather_kernel<T, V>, grid, dim3(32 * FQ_WARPS), 0, stream, (const T*)x, ldx, K, a_div, sorted, tile_info, n_tiles, tile_rows, \
             (uint8_t*)codes, ld, (uint8_t*)scales)
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
