// Products with weights in 8-bit floating point for many rows (prompt portions), on the 5th-generation tensor cores.
//
//   linear      out[m, n] = act(sum_k x[m, k] w[n, k] + bias[n]) (+ residual[m, n])
//   gated       per tile of a plan (128 slots of one expert): 128 columns of the unit of (gate, up), rounded to 8 bits in the epilogue
//   experts     per tile of a plan: out[slot, n] = sum_k h[row, k] w[expert][n, k]
//
// Operands are rows of codes with scales (fp8.cuh).  Persistent CTAs: warp 0 copies (TMA, 128-byte swizzle, a ring of stages of 128 of K;
// the scales of 512 of K come with every fourth), warp 1 issues tcgen05.mma kind::mxf8f6f4 (scales by tcgen05.cp into one of four places
// in turn), warps 2-17 are the epilogue: four a quadrant of the lanes, a lane a row, a quarter of the columns each.
//
// Tiles of 256 columns fill half of the tensor memory and scales want some of the rest, so there is one accumulator: the epilogue takes all of
// its numbers into registers at once (64 a thread) and hands it back before it does anything with them.  That costs some 500 clocks a
// tile; two accumulators of 128 columns would cost the main loop, whose products read shared memory 128 bytes a clock then.
//
// Pairs (CG = 2): two CTAs on a tile of 256 rows x BN columns; each brings its own rows of x, half of the rows of W and its own scales (of all BN
// columns: each SM multiplies its rows by all of them), the leader issues the products for both.
//
// In us: 8192 x 8192 x 8192 375 (2.9 PFLOP/s; under the power limit's clocks 390 to 450), 4096 x 4096 x 4096 53 (2.6), 1024 x 4096 x 4096 16.1 (2.1),
// 32768 slots over 64 experts 2048 -> 2 x 1024 134 (2.05; tensor pipe 58 % of the time, the rest is the unit's arithmetic where one accumulator is
// waited for) and 1024 -> 2048 84 (1.6; 134 MB of results, tensor pipe 45 %), with float32 results 126 to 140 (268 MB, 30 %).  Experts in pairs of CTAs were slower (145 and 103; 300 tokens: 17 beside 11):
// both CTAs wait for the slower one's epilogue, and an expert's odd tile leaves half a pair idle.
//
// Every wait is bounded (tcgen05.cuh); a wait that runs out raises a status bit and all roles leave through the common exit.
#include "fp8.cuh"

MLXB_DEFINE_LAST_ERROR()

enum { MANY_LINEAR = 0, MANY_GATED = 1, MANY_EXPERTS = 2 };

struct ManyArgs {
  int M, N, runs, kgs, x_tiles, w_tiles;       // x_tiles, w_tiles: of 128 rows (of one matrix of W)
  int tiles_m, tiles_n;                        // of the result; of a plan: tiles_m is what the plan holds
  const int *sorted, *tile_info, *n_tiles;
  const float* sel_weight;
  const float* bias;
  const void* residual;
  void* out;
  long long ldo;
  uint8_t* out_scales;
  int out_kgs, E, S;                           // E, S: experts and slots, a plan's numbers are held to them
  int* status;
  int act;
  float limit;
};
struct ManyMaps { CUtensorMap x, w, xs, ws, out; };      // out: of a linear layer whose rows begin on 16 bytes

constexpr int MANY_EPI = 16, MANY_THREADS = 64 + 32 * MANY_EPI;     // four warps a quadrant of the lanes, a quarter of the columns each

template <int BN, int CG, int KIND>
struct ManyShape {
  static constexpr int W_ROWS = BN / CG, W_TILES = BN / 128;
  static constexpr int STAGE = 16384 + W_ROWS * 128 + (1 + W_TILES) * FP8_TILE;
  // for results on their way out: a box a warp, or none (the gated unit's leave as they are)
  static constexpr int OUT = KIND == MANY_GATED ? 16 : 1024;
  static constexpr int ROOM = 227 * 1024 - 4096 - (KIND == MANY_GATED ? 4096 : 2048) - MANY_EPI * OUT;
  static constexpr int STAGES = ROOM / STAGE < 8 ? ROOM / STAGE : 8;
  static constexpr int SCALES = 4 + 4 * W_TILES;
  static constexpr int ACC = BN == 256 ? 1 : 2;
};

template <int BN, int CG, int KIND>
struct ManySmem {
  using S = ManyShape<BN, CG, KIND>;
  alignas(1024) uint8_t x[S::STAGES][16384];
  alignas(1024) uint8_t w[S::STAGES][S::W_ROWS * 128];
  alignas(128) uint8_t xs[S::STAGES][FP8_TILE];
  alignas(128) uint8_t ws[S::STAGES][S::W_TILES * FP8_TILE];
  // results of a warp's 32 rows on their way out: boxes of 32 bytes a row, whose 16-byte pieces lie as a copy with 32-byte swizzle wants them
  alignas(1024) uint4 stage[MANY_EPI][S::OUT / 16];
  uint32_t top[KIND == MANY_GATED ? 2 : 1][4][4][32];        // gated: the largest magnitudes of a row's 32 columns, by quadrant and slice
  alignas(16) float bias[KIND == MANY_LINEAR ? MANY_EPI : 1][32];
  alignas(8) uint64_t full[S::STAGES];
  uint64_t empty[S::STAGES];
  uint64_t acc_full[2], acc_empty[2], drained;
  uint32_t tmem;
  int abort_flag;
};

__device__ __forceinline__ int many_stage(int row, int piece) { return row * 2 + (piece ^ ((row >> 2) & 1)); }

// 32 rows of 32 bytes from shared memory to columns x .., rows y .. of a matrix; what lies outside it is left out
__device__ __forceinline__ void store_box(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
}

template <typename TO>
__device__ __forceinline__ void store_whole(uint4 u, int n, int N, TO* row) {
  constexpr int PER = 16 / sizeof(TO);
  if (n + PER <= N) {
    *reinterpret_cast<uint4*>(row + n) = u;
  } else {
    const TO* e = reinterpret_cast<const TO*>(&u);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (n + i < N) row[n + i] = e[i];
  }
}

// WHOLE: rows of out (and residual) begin on 16 bytes.
template <int BN, int CG, int KIND, typename TO, bool WHOLE>
__global__ void __launch_bounds__(MANY_THREADS)
fp8_many_kernel(const __grid_constant__ ManyMaps maps, ManyArgs a) {
  using S = ManyShape<BN, CG, KIND>;
  constexpr int STAGES = S::STAGES, SLICE = BN / 4;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<ManySmem<BN, CG, KIND>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cluster_rank() : 0;
  const bool leader = rank == 0;
  const int first_tile = (int)blockIdx.x / CG, step = (int)gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&sm.full[s], 1); mbar_init(&sm.empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&sm.acc_full[b], 1); mbar_init(&sm.acc_empty[b], CG * 32 * MANY_EPI); }
    mbar_init(&sm.drained, 1);
    sm.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.x) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.xs) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.ws) : "memory");
  }
  if (warp == 1) {
    if (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  volatile int* abort_flag = &sm.abort_flag;
  const uint32_t peer_abort = CG == 2 ? peer_addr(&sm.abort_flag, (uint32_t)(rank ^ 1)) : 0u;
  fp8_before_sync();
  __syncthreads();
  if (CG == 2) cluster_sync();
  fp8_after_sync();
  const uint32_t tmem = sm.tmem;
  pdl_trigger();

  // Where a tile lies.  A linear layer's tiles go by groups of 8 row tiles, columns after columns, so that those which run together read few
  // rows of either operand; a plan's by its own tiles, so that an expert's are together and its weights and rows come from memory once (by blocks of
  // columns, 32768 slots of 2048 over 64 experts were read again for every block: 154 us).
  struct Place { int m, n; };
  const int* tile_info = a.tile_info;
  int tiles_m = a.tiles_m;
  auto place_of = [&](int t) {
    if (KIND != MANY_LINEAR) return Place{t / a.tiles_n, t % a.tiles_n};
    const int per = 8 * a.tiles_n, g = t / per, r = t - g * per, rows = min(8, tiles_m - 8 * g);
    return Place{8 * g + r % rows, r / rows};
  };
  auto brings = [&](int k) { return (k & 3) == 0; };
  auto load_x = [&](int s, int k, int m0) {
    const int t = min(m0 >> 7, a.x_tiles - 1) * a.kgs + (k >> 2);
    if (CG == 2) {
      const uint32_t bar = peer_addr(&sm.full[s], 0);
      tma_load_2d_pair(sm.x[s], &maps.x, k * FP8_RUN, m0, bar);
      if (brings(k)) tma_load_2d_pair(sm.xs[s], &maps.xs, 0, t, bar);
    } else {
      tma_load_2d(sm.x[s], &maps.x, k * FP8_RUN, m0, &sm.full[s]);
      if (brings(k)) tma_load_2d(sm.xs[s], &maps.xs, 0, t, &sm.full[s]);
    }
  };
  auto load_w = [&](int s, int k, int expert, int nb) {
    const uint32_t bar = CG == 2 ? peer_addr(&sm.full[s], 0) : 0u;
    if (KIND == MANY_GATED) {             // 128 gate rows, then the up rows of the same columns
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int group = 2 * expert + h;
        tma_load_2d(sm.w[s] + h * 16384, &maps.w, k * FP8_RUN, group * a.N + nb * 128, &sm.full[s]);
        if (brings(k)) tma_load_2d(sm.ws[s] + h * FP8_TILE, &maps.ws, 0, (group * a.w_tiles + nb) * a.kgs + (k >> 2), &sm.full[s]);
      }
    } else {
      const int row = expert * a.N + nb * BN + rank * S::W_ROWS;
      if (CG == 2) tma_load_2d_pair(sm.w[s], &maps.w, k * FP8_RUN, row, bar);
      else tma_load_2d(sm.w[s], &maps.w, k * FP8_RUN, row, &sm.full[s]);
      if (brings(k))
#pragma unroll
        for (int i = 0; i < S::W_TILES; ++i) {
          const int t = (expert * a.w_tiles + min(nb * S::W_TILES + i, a.w_tiles - 1)) * a.kgs + (k >> 2);
          if (CG == 2) tma_load_2d_pair(sm.ws[s] + i * FP8_TILE, &maps.ws, 0, t, bar);
          else tma_load_2d(sm.ws[s] + i * FP8_TILE, &maps.ws, 0, t, &sm.full[s]);
        }
    }
  };
  auto stage_bytes = [&](int k) { return (uint32_t)(CG * (16384 + S::W_ROWS * 128 + (brings(k) ? (1 + S::W_TILES) * FP8_TILE : 0))); };

  pdl_wait();
  tile_info = after_wait(tile_info);
  const int* sorted = after_wait(a.sorted);
  const float* sel_weight = after_wait(a.sel_weight);
  if (KIND != MANY_LINEAR) tiles_m = min(tiles_m, after_wait(a.n_tiles)[0]);
  const int n_tiles = tiles_m * a.tiles_n;

  if (warp == 0) {
    int issued = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = first_tile; t < n_tiles && ok; t += step) {
      const Place p = place_of(t);
      const int m0 = p.m * (CG * 128) + rank * 128, expert = KIND == MANY_LINEAR ? 0 : max(0, min(a.E - 1, tile_info[3 * p.m]));
      for (int k = 0; k < a.runs; ++k) {
        if (issued >= STAGES) {
          ok = mbar_wait_warp(&sm.empty[s], ph ^ 1, abort_flag, peer_abort);
          if (!ok) break;
        }
        if (elect_one()) {
          if (leader) mbar_expect_tx(&sm.full[s], stage_bytes(k));
          load_x(s, k, m0);
          load_w(s, k, expert, p.n);
        }
        ++issued;
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
    if (__any_sync(0xffffffffu, *abort_flag) && leader && lane == 0)      // gave up: copies already issued land before the CTA exits
      for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i) fp8_drain(&sm.full[i % STAGES], (uint32_t)((i / STAGES) & 1));
  } else if (warp == 1) {
    if (leader) {
      constexpr uint32_t idesc = fp8_idesc(CG * 128, BN);
      const uint32_t scales0 = tmem + S::ACC * BN;
      const uint64_t dx0 = umma_desc(smem_u32(sm.x[0])), dw0 = umma_desc(smem_u32(sm.w[0]));
      const uint64_t dxs0 = fp8_scale_desc(smem_u32(sm.xs[0])), dws0 = fp8_scale_desc(smem_u32(sm.ws[0]));
      int s = 0, it = 0, place = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first_tile; t < n_tiles && ok; t += step, ++it) {
        const int b = S::ACC == 2 ? it & 1 : 0;
        ok = mbar_wait_warp(&sm.acc_empty[b], (uint32_t)((S::ACC == 2 ? it >> 1 : it) & 1) ^ 1, abort_flag, peer_abort);
        if (!ok) break;
        fp8_after_sync();
        const uint32_t acc = tmem + (uint32_t)(b * BN);
        for (int k = 0; k < a.runs; ++k) {
          ok = mbar_wait_warp(&sm.full[s], ph, abort_flag, peer_abort);
          if (!ok) break;
          fp8_after_sync();
          const bool fresh = brings(k);
          if (fresh) place = (place + 1) & 3;
          const uint32_t sx = scales0 + (uint32_t)(place * S::SCALES), sw = sx + 4;
          if (elect_one()) {
            if (fresh) {
              fp8_copy_scales<CG>(sx, dxs0 + (uint32_t)(s * (FP8_TILE / 16)));
#pragma unroll
              for (int i = 0; i < S::W_TILES; ++i) fp8_copy_scales<CG>(sw + 4 * i, dws0 + (uint32_t)((s * S::W_TILES + i) * (FP8_TILE / 16)));
            }
            const uint32_t id = idesc | fp8_idesc_byte((uint32_t)(k & 3));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              fp8_mma<CG>(acc, dx0 + (uint32_t)(s * 1024 + 2 * j), dw0 + (uint32_t)(s * S::W_ROWS * 8 + 2 * j), id, sx, sw, k > 0 || j > 0);
            if (CG == 2) umma_commit_both(&sm.empty[s]);
            else umma_commit(&sm.empty[s]);
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
#ifdef MLXB_TEST_WAIT_TIMEOUT
        if (g_test_withhold_arrival && it == 0) continue;
#endif
        if (ok && elect_one()) {
          if (CG == 2) umma_commit_both(&sm.acc_full[b]);
          else umma_commit(&sm.acc_full[b]);
        }
        __syncwarp();
      }
    }
  } else {
    const int q = warp & 3, slice = (warp - 2) >> 2, row = q * 32 + lane;
    uint4* stg = sm.stage[warp - 2];
    const int o_row = lane >> 1, o_piece = lane & 1;
    int it = 0;
    for (int t = first_tile; t < n_tiles; t += step, ++it) {
      const int b = S::ACC == 2 ? it & 1 : 0;
      const Place p = place_of(t);
      // asked for while the products run: a plan's slots and their weights
      constexpr int CHUNKS = SLICE / 32;
      const int m0 = KIND == MANY_LINEAR ? p.m * (CG * 128) + rank * 128 + q * 32 : 0, n0 = KIND == MANY_GATED ? p.n * 128 + slice * 32 : p.n * BN + slice * SLICE;
      const int rows = KIND == MANY_LINEAR ? a.M - m0 : tile_info[3 * p.m + 2] - q * 32;      // of this warp's 32, those that exist
      const TO* res = KIND == MANY_LINEAR ? reinterpret_cast<const TO*>(after_wait(a.residual)) : nullptr;
      int slot = -1;
      float wgt = 1.f;
      if (KIND != MANY_LINEAR && lane < rows) {
        const int place = tile_info[3 * p.m + 1] + row;
        if (place >= 0 && place < a.S) slot = sorted[place];
        if (slot < 0 || slot >= a.S) slot = -1;
        else if (KIND == MANY_GATED && sel_weight) wgt = sel_weight[slot];
      }
      bool ok = mbar_wait(&sm.acc_full[b], (uint32_t)((S::ACC == 2 ? it >> 1 : it) & 1), abort_flag, peer_abort);
      if (KIND == MANY_GATED) {             // the four warps of a quadrant meet below
        uint32_t all;
        asm volatile("{\n\t.reg .pred p, r;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred r, %2, 128, p;\n\tselp.u32 %0, 1, 0, r;\n\t}"
                     : "=r"(all) : "r"((uint32_t)ok), "r"(q + 1) : "memory");
        ok = all != 0;
      }
      if (!ok) break;
      fp8_after_sync();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * BN);
      uint32_t r[CHUNKS][32];
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)      // gated: 32 columns of gate, the same of up
        tmem_ld32(acc + (uint32_t)(KIND == MANY_GATED ? c * 128 + slice * 32 : slice * SLICE + c * 32), r[c]);
      fp8_wait_ld();
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) fp8_arrived(r[c]);
      fp8_before_sync();
      if (CG == 2) mbar_arrive_cluster(peer_addr(&sm.acc_empty[b], 0));
      else mbar_arrive(&sm.acc_empty[b]);

      if constexpr (KIND == MANY_GATED) {
        const bool live = lane < rows;
        uint32_t top = 0;
        auto units = [&](auto kind) {
          constexpr int KIND_OF = decltype(kind)::value;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            r[0][i] = __float_as_uint(fp8_gated_unit(KIND_OF, __uint_as_float(r[0][i]), __uint_as_float(r[1][i]), wgt, a.limit));
            if (n0 + 32 > a.N && n0 + i >= a.N) r[0][i] = 0u;
            top = max(top, r[0][i] & 0x7fffffffu);
          }
        };
        if (a.act == MLXB_GU_BOUNDED) units(std::integral_constant<int, MLXB_GU_BOUNDED>{});
        else units(std::integral_constant<int, MLXB_GU_SILU>{});
        if (top >= 0x7f800000u) {             // rare: something is not finite
          top = 0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            top = max(top, fp8_magnitude(__uint_as_float(r[0][i])));
            r[0][i] = __float_as_uint(fp8_or_nan(__uint_as_float(r[0][i])));
          }
        }
        // the other warps of the quadrant have the rest of the run's columns
        sm.top[it & 1][q][slice][lane] = top;
        asm volatile("bar.sync %0, 128;" ::"r"(q + 1) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, sm.top[it & 1][q][i][lane]);
        const int e = fp8_exponent(top);
        const float f = fp8_power(-e);
        if (live) {
          uint8_t* o = reinterpret_cast<uint8_t*>(a.out) + ((long long)p.m * 128 + row) * a.ldo;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = 16 * g + 4 * i;
              w[i] = fp8_quad(__uint_as_float(r[0][j]) * f, __uint_as_float(r[0][j + 1]) * f, __uint_as_float(r[0][j + 2]) * f, __uint_as_float(r[0][j + 3]) * f);
            }
            const int n = n0 + 16 * g;
            if (n < a.ldo) *reinterpret_cast<uint4*>(o + n) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (slice == 0) a.out_scales[((long long)p.m * a.out_kgs + (p.n >> 2)) * FP8_TILE + fp8_scale_row(row) + (p.n & 3)] = (uint8_t)(e + 127);
        }
      } else {
        constexpr int PER = 16 / sizeof(TO);
        TO* out = reinterpret_cast<TO*>(a.out);
        float bias[CHUNKS];                   // column 32 c + lane of this warp's
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) bias[c] = KIND == MANY_LINEAR && a.bias != nullptr && n0 + 32 * c + lane < a.N ? a.bias[n0 + 32 * c + lane] : 0.f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          float* v = reinterpret_cast<float*>(r[c]);
          const int nc = n0 + 32 * c;
          if (nc >= a.N) break;
          if (KIND == MANY_LINEAR) {
            if (a.bias != nullptr) {
              sm.bias[warp - 2][lane] = bias[c];
              __syncwarp();
              const float4* bp = reinterpret_cast<const float4*>(sm.bias[warp - 2]);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 x = bp[i];
                v[4 * i] += x.x; v[4 * i + 1] += x.y; v[4 * i + 2] += x.z; v[4 * i + 3] += x.w;
              }
              __syncwarp();
            }
            float (&vv)[32] = *reinterpret_cast<float (*)[32]>(r[c]);
            fp8_activate<sizeof(TO) == 2>(a.act, vv);
          }
          if constexpr (!WHOLE) {         // rows that do not begin on 16 bytes: a few columns at a time through shared memory in float32
            constexpr int COLS = S::OUT / 128, STEP = 32 / COLS;         // 8 columns, 4 rows an instruction
            float* f = reinterpret_cast<float*>(stg);
#pragma unroll
            for (int p0 = 0; p0 < 32; p0 += COLS) {
#pragma unroll
              for (int i = 0; i < COLS; ++i) f[lane * COLS + ((i + 2 * lane) & (COLS - 1))] = v[p0 + i];
              __syncwarp();
              const int col = lane & (COLS - 1), n = nc + p0 + col;
#pragma unroll 4
              for (int rr = lane / COLS; rr < 32; rr += STEP) {
                const int to = KIND == MANY_EXPERTS ? __shfl_sync(0xffffffffu, slot, rr) : m0 + rr;
                if (rr < rows && n < a.N && to >= 0) {
                  const long long at = (long long)to * a.ldo + n;
                  float y = f[rr * COLS + ((col + 2 * rr) & (COLS - 1))];
                  if (res != nullptr) y += to_f(res[at]);
                  out[at] = from_f<TO>(y);
                }
              }
              __syncwarp();
            }
            continue;
          } else {
          if (KIND == MANY_LINEAR && res != nullptr && lane < rows) {       // added before the sum is rounded, by rows
            const TO* x = res + (long long)(m0 + lane) * a.ldo + nc;
            if (nc + 32 <= a.N) {
              uint4 u[32 / PER];
#pragma unroll
              for (int i = 0; i < 32 / PER; ++i) u[i] = reinterpret_cast<const uint4*>(x)[i];
#pragma unroll
              for (int i = 0; i < 32 / PER; ++i) {
                if constexpr (sizeof(TO) == 2) {
                  float e[8];
                  unpack8(u[i], e);
#pragma unroll
                  for (int j = 0; j < 8; ++j) v[8 * i + j] += e[j];
                } else {
                  v[4 * i] += __uint_as_float(u[i].x); v[4 * i + 1] += __uint_as_float(u[i].y);
                  v[4 * i + 2] += __uint_as_float(u[i].z); v[4 * i + 3] += __uint_as_float(u[i].w);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (nc + i < a.N) v[i] += to_f(x[i]);
            }
          }
          if (KIND == MANY_LINEAR && (a.N & (PER - 1)) != 0 && nc + 32 > a.N && lane < rows) {      // the last columns, less than 16 bytes of them
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (nc + i >= (a.N & ~(PER - 1)) && nc + i < a.N) out[(long long)(m0 + lane) * a.ldo + nc + i] = from_f<TO>(v[i]);
          }
          auto piece = [&](int i) {                  // 16 bytes of results from this chunk's column i on
            if (sizeof(TO) == 2) {
              float w[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) w[j] = v[(i + j) & 31];
              return pack8(w);
            }
            return make_uint4(r[c][i & 31], r[c][(i + 1) & 31], r[c][(i + 2) & 31], r[c][(i + 3) & 31]);
          };
          if constexpr (KIND == MANY_LINEAR) {
#pragma unroll
            for (int p0 = 0; p0 < 32; p0 += 2 * PER) {        // 32 bytes of each row a box, one copy a box
              uint4* box = stg;
              if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // what was sent from here has been read
              __syncwarp();
#pragma unroll
              for (int x = 0; x < 2; ++x) box[many_stage(lane, x)] = piece(p0 + x * PER);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) {
                if (rows > 0 && nc + p0 < (a.N & ~(PER - 1))) store_box(&maps.out, box, nc + p0, m0);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              }
            }
          } else {
#pragma unroll
            for (int p0 = 0; p0 < 32; p0 += 2 * PER) {        // rows of slots: 32 bytes of each at a time, two lanes a row
#pragma unroll
              for (int x = 0; x < 2; ++x) stg[many_stage(lane, x)] = piece(p0 + x * PER);
              __syncwarp();
              const int n = nc + p0 + o_piece * PER;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int rr = 16 * j + o_row;
                const uint4 u = stg[many_stage(rr, o_piece)];
                const int to = __shfl_sync(0xffffffffu, slot, rr);
                if (rr < rows && n < a.N && to >= 0) store_whole<TO>(u, n, a.N, out + (long long)to * a.ldo);
              }
              __syncwarp();
            }
          }
          }
        }
      }
    }
    if (KIND == MANY_LINEAR && WHOLE && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  __syncwarp();
  fp8_before_sync();
  __syncthreads();
  if (CG == 2) cluster_sync();
  const bool aborted = sm.abort_flag != 0;
  if (threadIdx.x == 0 && aborted) atomicOr(a.status, MLXB_ST_WAIT_TIMEOUT);
  if (warp == 1 && leader) {
    if (aborted && lane == 0) {
      if (CG == 2) umma_commit_pair_local(&sm.drained);
      else umma_commit(&sm.drained);
      fp8_drain(&sm.drained, 0u);
    }
    __syncwarp();
  }
  if (CG == 2 && aborted) cluster_sync();
  if (warp == 1) {
    fp8_after_sync();
    if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------- host side

// scales as rows of 512 bytes, a row a copy
static int scales_map(CUtensorMap* map, const void* base, long long tiles, const char* what) {
  const cuuint64_t dims[2] = {FP8_TILE / 4, (cuuint64_t)tiles};
  const cuuint64_t strides[1] = {FP8_TILE};
  const cuuint32_t box[2] = {FP8_TILE / 4, 1};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = cuTensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, elem,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return 0;
  const char* msg = nullptr;
  cuGetErrorString(r, &msg);
  return mlxb_fail(MLXB_BAD_ARG, "%s: cuTensorMapEncodeTiled(%lld tiles of scales): %s", what, tiles, msg ? msg : "?");
}

template <typename TO>
static int out_map(CUtensorMap* map, const ManyArgs& a) {
  const cuuint64_t dims[2] = {(cuuint64_t)(a.N & ~(16 / (int)sizeof(TO) - 1)), (cuuint64_t)a.M};     // a copy writes whole 16 bytes
  const cuuint64_t strides[1] = {(cuuint64_t)a.ldo * sizeof(TO)};
  const cuuint32_t box[2] = {32 / sizeof(TO), 32};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = cuTensorMapEncodeTiled(map, sizeof(TO) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a.out, dims, strides,
                                            box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return 0;
  const char* msg = nullptr;
  cuGetErrorString(r, &msg);
  return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): cuTensorMapEncodeTiled(%d x %d results at stride %lld): %s", a.M, a.N, a.ldo, msg ? msg : "?");
}

template <int BN, int CG, int KIND, typename TO, bool WHOLE>
static int many_launch_as(const ManyMaps& maps_in, const ManyArgs& a, cudaStream_t stream) {
  ManyMaps maps = maps_in;
  if (KIND == MANY_LINEAR && WHOLE)
    if (int e = out_map<TO>(&maps.out, a)) return e;
  constexpr size_t smem = sizeof(ManySmem<BN, CG, KIND>) + 1024;
  static_assert(smem <= 227 * 1024, "stages and staging buffers fit a CTA's shared memory");
  auto kern = fp8_many_kernel<BN, CG, KIND, TO, WHOLE>;
  static SharedLimit limit;
  if (cudaError_t e = limit.raise(kern, smem)) return mlxb_fail((int)e, "linear (8 bits): %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
  const long long tiles = (long long)a.tiles_m * a.tiles_n;
  const int units = mlxb_sm_count() / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CG * (unsigned)(tiles < units ? tiles : units));
  cfg.blockDim = dim3(MANY_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (CG == 2) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = CG;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (mlxb_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kern, maps, a);
  return mlxb_check_launch("linear (8 bits)");
}

template <int BN, int CG, int KIND, typename TO>
static int many_launch(const ManyMaps& maps, const ManyArgs& a, cudaStream_t stream) {
  if (KIND == MANY_GATED || (a.N >= 8 && !(((uintptr_t)a.out | (uintptr_t)a.residual | (uintptr_t)(a.ldo * (long long)sizeof(TO))) & 15)))
    return many_launch_as<BN, CG, KIND, TO, true>(maps, a, stream);
  if constexpr (KIND != MANY_GATED) return many_launch_as<BN, CG, KIND, TO, false>(maps, a, stream);
  return MLXB_BAD_ARG;
}

// Tile width and pairs or not: the form whose time, as a sum of what was measured, is least: a launch (set-up, the first copies, the last tile's
// results), every run of 128 of K, every further wave of tiles.  A fit to 48 sizes (129 to 4096 rows, K and N of 512 to 14336) where the choice is within 5 % of
// the best form (us at 256 columns in pairs | alone | 128 in pairs | alone): 129 x 4096 x 4096 15.0 | 16.6 | 12.4 | 12.9; 1024 x 1024 x 4096
// 8.9 | 7.7 | 9.5 | 9.0; 1024 x 1024 x 1024 7.5 | 6.8 | 6.3 | 5.7; 4096 x 4096 x 4096 53 | 60 | 71 | 75.
struct ManyForm { int bn, cg; };
struct ManyCost { int bn, cg; double launch, run, wave; };      // microseconds
static constexpr ManyCost MANY_FORMS[] = {{256, 2, 5., .323, 1.9}, {256, 1, 3.8, .395, 1.5}, {128, 2, 4.5, .245, .6}, {128, 1, 3.5, .294, .5}};
static ManyForm many_form(int M, int N, int K) {
  const char *want_pair = getenv("MLXB_FP8_PAIR"), *want_bn = getenv("MLXB_FP8_BN");     // experiments and tests
  const int sms = mlxb_sm_count(), runs = (K + 127) / 128;
  ManyForm best = {128, 1};
  double best_cost = -1.;
  for (const ManyCost& f : MANY_FORMS) {
    if (f.cg == 2 && M <= 128) continue;
    if (want_pair && M > 128 && (want_pair[0] == '1') != (f.cg == 2)) continue;
    if (want_bn && atoi(want_bn) != f.bn) continue;
    const long long tiles = (long long)((M + f.cg * 128 - 1) / (f.cg * 128)) * ((N + f.bn - 1) / f.bn);
    const long long units = sms / f.cg, waves = (tiles + units - 1) / units;
    const double cost = f.launch + waves * runs * f.run + (waves - 1) * f.wave;
    if (best_cost < 0. || cost < best_cost) { best = {f.bn, f.cg}; best_cost = cost; }
  }
  return best;
}

// As mlxb_fp8_linear_few, for any number of rows.
MLXB_EXPORT int mlxb_fp8_linear_many(const Fp8LinearRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(Fp8LinearRecord)) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): a record of %lld bytes", bytes);
  const Fp8LinearRecord& r = *rec;
  if (r.M <= 0 || r.N <= 0) return 0;
  if (int e = fp8_check("linear (8 bits)", r.x, r.xs, r.w, r.ws, r.out, r.M, r.N, r.K, r.ldo)) return e;
  if (!activation_known((int)r.epi) || !r.status) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): epilogue %lld", r.epi);
  const int M = (int)r.M, N = (int)r.N, K = (int)r.K;
  const ManyForm f = many_form(M, N, K);
  ManyArgs a = {};
  a.M = M; a.N = N; a.runs = (K + 127) / 128; a.kgs = (K + 511) / 512; a.x_tiles = (M + 127) / 128; a.w_tiles = (N + 127) / 128;
  a.tiles_m = (M + 128 * f.cg - 1) / (128 * f.cg); a.tiles_n = (N + f.bn - 1) / f.bn;
  a.bias = r.bias; a.residual = r.residual; a.out = r.out; a.ldo = r.ldo; a.status = r.status; a.act = (int)r.epi;
  if ((long long)a.tiles_m * a.tiles_n > 0x3fffffffLL) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): %d x %d outputs", M, N);
  ManyMaps maps;
  if (int e = fp8_make_map(&maps.x, r.x, M, K, K, 128, "linear (8 bits) x")) return e;
  if (int e = fp8_make_map(&maps.w, r.w, N, K, K, f.bn / f.cg, "linear (8 bits) w")) return e;
  if (int e = scales_map(&maps.xs, r.xs, (long long)a.x_tiles * a.kgs, "linear (8 bits)")) return e;
  if (int e = scales_map(&maps.ws, r.ws, (long long)a.w_tiles * a.kgs, "linear (8 bits)")) return e;
#define GO(BN, CG) return r.out_f32 ? many_launch<BN, CG, MANY_LINEAR, float>(maps, a, stream) : many_launch<BN, CG, MANY_LINEAR, __nv_bfloat16>(maps, a, stream);
  if (f.cg == 2) {
    if (f.bn == 256) GO(256, 2)
    GO(128, 2)
  }
  if (f.bn == 256) GO(256, 1)
  GO(128, 1)
#undef GO
}

// As mlxb_fp8_experts_few, for plans with tiles of 128 slots.
MLXB_EXPORT int mlxb_fp8_experts_many(const Fp8ExpertsRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(Fp8ExpertsRecord)) return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: a record of %lld bytes", bytes);
  const Fp8ExpertsRecord& r = *rec;
  if (r.max_tiles <= 0 || r.at_most <= 0) return 0;
  if (int e = fp8_check_experts(r)) return e;
  if (r.tile_rows != 128) return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: tiles of %lld rows", r.tile_rows);
  const int N = (int)r.N, K = (int)r.K;
  ManyArgs a = {};
  a.N = N; a.runs = (K + 127) / 128; a.kgs = (K + 511) / 512; a.x_tiles = (int)r.max_tiles; a.w_tiles = (N + 127) / 128;
  const int bn = 256;
  a.tiles_m = (int)min(r.max_tiles, r.at_most); a.tiles_n = r.gated ? a.w_tiles : (N + bn - 1) / bn;
  a.sorted = r.sorted; a.tile_info = r.tile_info; a.n_tiles = r.n_tiles; a.sel_weight = r.sel_weight;
  a.out = r.out; a.ldo = r.ldo; a.out_scales = (uint8_t*)r.out_scales; a.out_kgs = (N + 511) / 512; a.status = r.status; a.act = (int)r.act;
  a.limit = (float)r.limit; a.E = (int)r.E; a.S = (int)r.S;
  if ((long long)a.tiles_m * a.tiles_n > 0x3fffffffLL) return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: %lld tiles of %d outputs", r.max_tiles, N);
  const long long stack = r.E * (r.gated ? 2 : 1);
  ManyMaps maps;
  if (int e = fp8_make_map(&maps.x, r.x, r.max_tiles * 128, K, K, 128, "moe_gemm_fp8 x")) return e;
  if (int e = fp8_make_map(&maps.w, r.w, stack * N, K, K, r.gated ? 128 : bn, "moe_gemm_fp8 w")) return e;
  if (int e = scales_map(&maps.xs, r.xs, r.max_tiles * a.kgs, "moe_gemm_fp8")) return e;
  if (int e = scales_map(&maps.ws, r.ws, stack * a.w_tiles * a.kgs, "moe_gemm_fp8")) return e;
  if (r.gated) return many_launch<256, 1, MANY_GATED, float>(maps, a, stream);
  return r.out_f32 ? many_launch<256, 1, MANY_EXPERTS, float>(maps, a, stream) : many_launch<256, 1, MANY_EXPERTS, __nv_bfloat16>(maps, a, stream);
}
