// Rows of numbers in 8-bit floating point, and what the products of such rows share.
//
// Format.  A row of K numbers is K codes (e4m3) and one scale 2^e for each run of 128 columns.  e is the least whole number with
// (largest finite magnitude of the run) <= 448 * 2^e, within -127 .. 127; a code is x * 2^-e rounded to nearest, ties to even.  The scale is a
// power of two because a floating-point code loses nothing by it but what lies between the run's largest magnitude and 448, scaling is then
// exact, and block-scaled tcgen05.mma multiplies by such scales itself (a byte e + 127 for each 32 columns; here four
// runs of 32 share one).  A number that is not finite becomes the code for NaN, and so does every sum that it enters.
//
// Layout.  Codes: rows of `ld` bytes, ld a multiple of 16, zeros behind column K.  Scales: tiles of 512 bytes for 128 rows of a group
// and 512 columns, [groups][ceil(rows / 128)][ceil(K / 512)][512]; the byte of row r and run b is at (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4.
// That is the order in which tcgen05.cp (32x128b.warpx4) puts them in tensor memory where the products want them: row r in lane r % 32,
// column r / 32, byte b % 4.  Groups: the matrices of a stack (experts), or the tiles of a plan.
#pragma once

#include "activations.cuh"
#include "gated_unit.cuh"
#include "tcgen05.cuh"

constexpr int FP8_RUN = 128;                 // columns with one scale
constexpr int FP8_TILE = 512;                // bytes of a tile of scales: 128 rows, 4 runs

// The exponent e of a run's scale, from the bits of its largest finite magnitude: 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_exponent(uint32_t top_bits) {
  if (top_bits == 0) return 0;
  const int e = (int)(top_bits >> 23) - 127 - 8 + ((top_bits & 0x7fffffu) > 0x600000u);
  return max(-127, min(127, e));
}
// 2^e for -127 <= e <= 127 (2^-127 is subnormal)
__device__ __forceinline__ float fp8_power(int e) { return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 1u << 22); }
// the magnitude's bits, 0 for what is not finite
__device__ __forceinline__ uint32_t fp8_magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// what the conversion is to make NaN of: it saturates by itself, infinities too
__device__ __forceinline__ float fp8_or_nan(float v) { return fabsf(v) < INFINITY ? v : __uint_as_float(0x7fffffffu); }
// Codes of numbers that were scaled, the first in the low byte.
__device__ __forceinline__ uint32_t fp8_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fp8_quad(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Bytes from a row's place to its scales in a tile, without the run.
__device__ __forceinline__ int fp8_scale_row(int r) { return (r & 31) * 16 + ((r >> 5) & 3) * 4; }

// ---- products

// Instruction descriptor for kind::mxf8f6f4: A and B e4m3 (bits 7-9 and 10-12 = 0), both K-major, N/8 in bits 17-22, scales of type e8m0
// (bit 23), M/16 in bits 24-28; which byte of a scale's column: bits 4-5 for B, 29-30 for A.
__host__ __device__ constexpr uint32_t fp8_idesc(int m, int n) {
  return ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t fp8_idesc_byte(uint32_t b) { return b << 4 | b << 29; }

// 32 columns of K: D (+)= (A * its scales) (B * its scales)^T
template <int CG>
__device__ __forceinline__ void fp8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate) : "memory");
}

// Descriptor of a tile of scales in shared memory: 32 rows of 16 bytes without swizzle, groups of 8 rows 128 bytes apart.
__device__ __forceinline__ uint64_t fp8_scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
// A tile of scales into four columns of tensor memory, the same for the four quarters of its lanes.  Products that are issued behind it by
// the same thread find them there.
template <int CG>
__device__ __forceinline__ void fp8_copy_scales(uint32_t tmem, uint64_t desc) {
  if (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

__device__ __forceinline__ void fp8_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void fp8_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fp8_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fp8_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Numbers that tcgen05.ld was to bring, as they are after the wait: what is formed of them cannot be moved before it.
__device__ __forceinline__ void fp8_arrived(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}

// A bounded wait that looks at no flag: for the way out, where copies and products already issued must come to their end.
__device__ __forceinline__ void fp8_drain(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t p = 0; p < (1u << 20); ++p) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return;
  }
}

// An activation of the list on all of a thread's numbers.  NaN stays NaN: a row that was not finite must show.  (The others than relu see to it themselves; a
// comparison more for each number costs 2048 x 1600 x 6400 with gelu_new 4 us of 32.)
template <bool FAST, int N>
__device__ __forceinline__ void fp8_activate(int act, float (&v)[N]) {
  switch (act) {
#define MLXB_FP8_ACT(ID, CODE, NAME)                                                                                              \
  case CODE:                                                                                                                      \
    _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] = CODE == EPI_RELU && !(v[i] == v[i]) ? v[i] : activate<CODE, FAST>(v[i]); \
    break;
    MLXB_ACTIVATION_LIST(MLXB_FP8_ACT)
#undef MLXB_FP8_ACT
  }
}

// The gated unit of gated_unit.cuh with the library's exponential and the hardware's quotient, in which NaN stays NaN.  For given a and w u the silu unit is off
// by 10 * 2^-24 of its value at most (exponential 2 units in the last place, quotient 2, a sum and a product), whatever a is; where the quotient's divisor passes 2^126,
// below a = -87, it is 0.  (The hardware's exponential is off by more the larger |a| is, and each of these steps that crosses a border of 8 bits moves a number by up to 1/8.  4096
// tokens of 64 experts take 267.9 us in all with this one, 267.0 with the hardware's, 284 with an exact quotient too, whose code is long: 300 tokens 30.7, 30.1 and 37.8.)
__device__ __forceinline__ float fp8_gated_unit(int kind, float g, float u, float w, float limit) {
  if (kind == MLXB_GU_BOUNDED) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
    return w * __fdividef(g, 1.f + expf(-1.702f * g)) * (u + 1.f);
  }
  const float a = w * g;
  return __fdividef(a, 1.f + expf(-a)) * (w * u);
}

// Arguments as records of 8-byte fields (a caller fills one in a tenth of the time of as many arguments), the same for few and for many rows.
struct Fp8LinearRecord {
  const void *x, *xs, *w, *ws;
  const float* bias;
  const void* residual;
  void* out;
  int* status;
  long long out_f32, M, N, K, ldo, epi;
};
struct Fp8ExpertsRecord {
  const void *x, *xs, *w, *ws;
  const int *sorted, *tile_info, *n_tiles;
  const float* sel_weight;
  void *out, *out_scales;
  int* status;
  long long gated, out_f32, E, N, K, S, max_tiles, at_most, tile_rows, ldo, act;
  double limit;
};

// What both kernels ask of their operands: codes in rows of whole 16 bytes, at 16-byte aligned addresses; sizes that the launchers' arithmetic holds.
static inline int fp8_check(const char* what, const void* x, const void* xs, const void* w, const void* ws, const void* out, long long M, long long N,
                            long long K, long long ldo) {
  if (!x || !xs || !w || !ws || !out || M <= 0 || N <= 0 || K <= 0 || (K & 15) || ldo < N || M > 0x7ffffff || N > 0x7ffffff || K > 0x7ffffff ||
      (((uintptr_t)x | (uintptr_t)xs | (uintptr_t)w | (uintptr_t)ws) & 15))
    return mlxb_fail(MLXB_BAD_ARG, "%s: %lld rows of %lld codes by %lld (whole 16 bytes, 16-byte aligned), results at stride %lld", what, M, K, N, ldo);
  return 0;
}
static inline int fp8_check_experts(const Fp8ExpertsRecord& r) {
  if (int e = fp8_check("moe_gemm_fp8", r.x, r.xs, r.w, r.ws, r.out, r.max_tiles * r.tile_rows, r.N, r.K, r.ldo)) return e;
  if (r.E <= 0 || r.S <= 0 || r.S > 0x7fffffffLL || r.E * r.N * 2 > 0x7fffffffLL || !r.sorted || !r.tile_info || !r.n_tiles || !r.status ||
      (r.gated && (!r.out_scales || r.ldo != ((r.N + 15) & ~15LL) || ((uintptr_t)r.out & 15))))
    return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: %lld experts of %lld x %lld, results at stride %lld", r.E, r.N, r.K, r.ldo);
  return 0;
}

// ---- host side: a matrix of codes, `rows` of `cols` bytes at a row stride of `ld` bytes, in boxes of box_rows x 128 columns
static inline int fp8_make_map(CUtensorMap* map, const void* base, long long rows, int cols, int ld, int box_rows, const char* what) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)FP8_RUN, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = cuTensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return 0;
  const char* msg = nullptr;
  cuGetErrorString(r, &msg);
  return mlxb_fail(MLXB_BAD_ARG, "%s: cuTensorMapEncodeTiled(%lld x %d, ld %d): %s", what, rows, cols, ld, msg ? msg : "?");
}
