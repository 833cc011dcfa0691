// Products with weights in 8-bit floating point for few rows (decode steps): the weights are what is read.
//
//   linear      out[m, n] = act(sum_k x[m, k] w[n, k] + bias[n]) (+ residual[m, n])
//   gated       per tile of a plan (up to 16 slots of one expert): h = unit of (gate, up), rounded to 8 bits in the epilogue, ready to be the
//               next product's operand
//   experts     per tile of a plan: out[slot, n] = sum_k h[row, k] w[expert][n, k]
//
// Both operands are rows of codes with scales (fp8.cuh); tcgen05.mma kind::mxf8f6f4 multiplies codes and scales and adds in float32.  The sides
// are exchanged: 128 rows of W are the product's M side and the NT (16 to 128; of a plan 16) rows of x its N side, so that a step of one token
// wastes 15 columns of a small product instead of 127 rows of a large one, and a CTA's tile is 16 KB of weights a stage whatever the
// number of tokens.  Gated: a stage holds 128 gate rows and the 128 up rows of the same columns, two accumulators, and one thread
// has both numbers of a unit.  The 128 columns of a tile are one run of the result: its scale is found in the epilogue.
//
// One CTA: warp 0 copies (TMA; a ring of stages of 128 of K), warp 1 issues the products, warps 2-5 are the epilogue (a lane a row of W).  A linear
// layer's first stages of W are on their way to the L2 before the wait for the kernel before.  Tensor memory: two accumulators where they fit, and four
// places for scales, one for each 512 of K in turn.
//
// Bound by the bytes of W where there are enough tiles; N / 128 tiles of a square layer are too few for 148 SMs, so K is split over
// a cluster of up to eight CTAs: each sends its sums for a share of the tokens to that share's CTA (distributed shared memory), which
// adds them in the order of the ranks.  How many CTAs share a tile depends on N, K and whether there are more than 64 rows (experts: on
// the largest number of tiles).  What an SM takes in, 64 bytes a clock, bounds a CTA; 148 of them together the memory.  Behind another kernel, in us: 1 x 4096 x 4096
// 6.5 (2.6 TB/s; of this 3 are a kernel's start, its first bytes and its end), 8 x 4096 x 14336 13.0 (4.5 TB/s, 112 tiles for 148 SMs), gated
// products of 32 tokens, 8 of 128 experts each, 2048 to twice 768 columns: 57 (6.1 TB/s).
//
// Every wait is bounded (tcgen05.cuh); a wait that runs out raises a status bit and all roles leave through the common exit.
#include "fp8.cuh"

MLXB_DEFINE_LAST_ERROR()

enum { FEW_LINEAR = 0, FEW_GATED = 1, FEW_EXPERTS = 2 };

struct FewArgs {
  const uint8_t *x_scales, *w_scales;
  int M, N, runs, kgs;                 // runs: of 128 columns of K; kgs: tiles of scales along K
  int w_tiles;                         // of 128 rows of a matrix of W
  const int *sorted, *tile_info, *n_tiles;
  const float* sel_weight;
  const float* bias;
  const void* residual;
  void* out;
  long long ldo;
  uint8_t* out_scales;
  int out_kgs, max_items, E, S;        // E, S: experts and slots, a plan's numbers are held to them
  int* status;
  int act;                             // activation, or kind of gated unit
  float limit;
};

constexpr int FEW_THREADS = 192;

template <int NT, int KIND, bool SPLIT>
struct FewShape {
  static constexpr int NH = KIND == FEW_GATED ? 2 : 1;
  static constexpr int STAGE = NH * (16384 + FP8_TILE) + NT * 128 + FP8_TILE;
  static constexpr int SUMS = SPLIT ? NH * (NT > 32 ? NT : 32) * 512 : 0;   // bytes of partial sums that arrive
  // two CTAs an SM where tiles are split and stages small (the next kernel's first weights are then on their way while this one ends)
  static constexpr bool PAIR = SPLIT && NH == 1 && NT <= 64;
  static constexpr int ROOM = (PAIR ? 112 : 224) * 1024 - SUMS - 2048;
  static constexpr int STAGES = ROOM / STAGE < 12 ? ROOM / STAGE : 12;
  static constexpr int SCALES = 4 * NH + 4;                           // columns of a place for scales
  static constexpr int ACC = 2 * NH * NT + 4 * SCALES <= 512 ? 2 : 1;
  static constexpr int USED = ACC * NH * NT + 4 * SCALES;
  static constexpr int COLS = USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
};

template <int NT, int KIND, bool SPLIT>
struct FewSmem {
  using S = FewShape<NT, KIND, SPLIT>;
  alignas(1024) uint8_t w[S::STAGES][S::NH * 16384];
  alignas(1024) uint8_t x[S::STAGES][NT * 128];
  alignas(128) uint8_t ws[S::STAGES][S::NH * FP8_TILE];
  alignas(128) uint8_t xs[S::STAGES][FP8_TILE];
  alignas(16) float4 sums[SPLIT ? S::SUMS / 16 : 1];    // [rank][a share's tokens / 4][gate, up][row of W]
  uint32_t top[2][4][32];
  alignas(8) uint64_t full[S::STAGES];
  uint64_t empty[S::STAGES];
  uint64_t acc_full[2], acc_empty[2], drained;
  uint32_t tmem;
  int abort_flag;
};

// 1 if `ok` holds for every thread of the four epilogue warps
__device__ __forceinline__ bool epilogue_agrees(bool ok) {
  uint32_t all;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(all) : "r"((uint32_t)ok) : "memory");
  return all != 0;
}

template <int NT, int KIND, bool SPLIT, typename TO>
__global__ void __launch_bounds__(FEW_THREADS)
fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, FewArgs a, int ranks) {
  using S = FewShape<NT, KIND, SPLIT>;
  constexpr int NH = S::NH, STAGES = S::STAGES, CH = NT < 32 ? NT : 32;
  extern __shared__ uint8_t smem_raw[];
  auto& sm = *reinterpret_cast<FewSmem<NT, KIND, SPLIT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLIT ? (int)cluster_rank() : 0;
  const int first_item = SPLIT ? (int)blockIdx.x / ranks : (int)blockIdx.x, step = SPLIT ? 0x40000000 : (int)gridDim.x;
  const int k0 = SPLIT ? (int)((long long)a.runs * rank / ranks) : 0, k1 = SPLIT ? (int)((long long)a.runs * (rank + 1) / ranks) : a.runs;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&sm.full[s], 1); mbar_init(&sm.empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&sm.acc_full[b], 1); mbar_init(&sm.acc_empty[b], 128); }
    mbar_init(&sm.drained, 1);
    sm.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(S::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  volatile int* abort_flag = &sm.abort_flag;
  fp8_before_sync();
  __syncthreads();
  fp8_after_sync();
  if (SPLIT) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // its other half stands before the first store to another CTA
  const uint32_t tmem = sm.tmem;

  // whether the stage of run k brings scales with it, and its bytes
  auto brings = [&](int k) { return (k & 3) == 0 || k == k0; };
  auto stage_bytes = [&](int k) { return (uint32_t)(NH * 16384 + NT * 128 + (brings(k) ? (NH + 1) * FP8_TILE : 0)); };
  auto load_w = [&](int s, int k, int group, int nb) {     // group: of the stack of matrices (gated: of the gate rows, the up rows next)
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      tma_load_2d(sm.w[s] + h * 16384, &map_w, k * FP8_RUN, (group + h) * a.N + nb * 128, &sm.full[s]);
      if (brings(k))
        fp8_bulk_load(sm.ws[s] + h * FP8_TILE, a.w_scales + (((long long)(group + h) * a.w_tiles + nb) * a.kgs + (k >> 2)) * FP8_TILE, FP8_TILE, &sm.full[s]);
    }
  };
  auto load_x = [&](int s, int k, int tile) {
    tma_load_2d(sm.x[s], &map_x, k * FP8_RUN, tile * NT, &sm.full[s]);
    const int at = KIND == FEW_LINEAR ? tile * NT >> 7 : tile;
    if (brings(k)) fp8_bulk_load(sm.xs[s], a.x_scales + ((long long)at * a.kgs + (k >> 2)) * FP8_TILE, FP8_TILE, &sm.full[s]);
  };

  pdl_trigger();
  // A linear layer's first weights are on their way to the L2 before the wait, and read behind it: the kernel before may be the one that writes them.
  if (KIND == FEW_LINEAR && threadIdx.x == 0 && first_item < a.max_items)
    for (int k = k0; k < min(k1, k0 + STAGES); ++k) {
      asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(&map_w), "r"(k * FP8_RUN), "r"(first_item % a.w_tiles * 128) : "memory");
      if (brings(k))
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.w_scales + ((long long)(first_item % a.w_tiles) * a.kgs + (k >> 2)) * FP8_TILE), "r"(FP8_TILE) : "memory");
    }
  pdl_wait();
  const int* tile_info = after_wait(a.tile_info);
  const int* sorted = after_wait(a.sorted);
  const float* sel_weight = after_wait(a.sel_weight);
  const int items = KIND == FEW_LINEAR ? a.max_items : min(a.max_items, after_wait(a.n_tiles)[0] * a.w_tiles);

  if (warp == 0) {
    int issued = 0, s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int w = first_item; w < items && ok; w += step) {
      const int tile = w / a.w_tiles, nb = w - tile * a.w_tiles;
      const int group = KIND == FEW_LINEAR ? 0 : max(0, min(a.E - 1, tile_info[3 * tile])) * NH;
      for (int k = k0; k < k1; ++k) {
        ok = mbar_wait_warp(&sm.empty[s], ph ^ 1, abort_flag);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&sm.full[s], stage_bytes(k));
          load_w(s, k, group, nb);
          load_x(s, k, tile);
        }
        ++issued;
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
    if (__any_sync(0xffffffffu, *abort_flag)) {       // gave up: copies already issued land before the CTA exits
      if (lane == 0)
        for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i) fp8_drain(&sm.full[i % STAGES], (uint32_t)((i / STAGES) & 1));
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = fp8_idesc(128, NT);
    const uint32_t scales0 = tmem + S::ACC * NH * NT;
    const uint64_t dw0 = umma_desc(smem_u32(sm.w[0])), dx0 = umma_desc(smem_u32(sm.x[0]));
    const uint64_t dws0 = fp8_scale_desc(smem_u32(sm.ws[0])), dxs0 = fp8_scale_desc(smem_u32(sm.xs[0]));
    int s = 0, it = 0, place = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int w = first_item; w < items && ok; w += step, ++it) {
      const int b = S::ACC == 2 ? it & 1 : 0;
      ok = mbar_wait_warp(&sm.acc_empty[b], (uint32_t)((S::ACC == 2 ? it >> 1 : it) & 1) ^ 1, abort_flag);
      if (!ok) break;
      fp8_after_sync();
      const uint32_t acc = tmem + (uint32_t)(b * NH * NT);
      for (int k = k0; k < k1; ++k) {
        ok = mbar_wait_warp(&sm.full[s], ph, abort_flag);
        if (!ok) break;
        fp8_after_sync();
        const bool fresh = brings(k);
        if (fresh) place = (place + 1) & 3;
        const uint32_t sw = scales0 + (uint32_t)(place * S::SCALES), sx = sw + 4 * NH;
        if (elect_one()) {
          if (fresh) {
#pragma unroll
            for (int h = 0; h < NH; ++h) fp8_copy_scales<1>(sw + 4 * h, dws0 + (uint32_t)((s * NH + h) * (FP8_TILE / 16)));
            fp8_copy_scales<1>(sx, dxs0 + (uint32_t)(s * (FP8_TILE / 16)));
          }
          const uint32_t id = idesc | fp8_idesc_byte((uint32_t)(k & 3));
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              fp8_mma<1>(acc + h * NT, dw0 + (uint32_t)((s * NH + h) * 1024 + 2 * j), dx0 + (uint32_t)(s * NT * 8 + 2 * j), id, sw + 4 * h, sx, k > k0 || j > 0);
          umma_commit(&sm.empty[s]);
        }
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
#ifdef MLXB_TEST_WAIT_TIMEOUT
      if (g_test_withhold_arrival && it == 0) continue;
#endif
      if (ok && elect_one()) umma_commit(&sm.acc_full[b]);
      __syncwarp();
    }
  }

  // ---- epilogue: a lane holds a row n of W; tokens are columns
  const int q = warp & 3, in_tile = q * 32 + lane;
  // What the epilogue needs from memory for up to CH tokens from tok0 on, asked for while the products run: a plan's slots and their weights, one
  // a lane; a linear layer's bias (of column n) and residuals.
  struct Beside { int slot; float weight, bias, residual[CH]; };
  auto fetch = [&](int w, int tok0, int live) {
    Beside x;
    x.slot = -1;
    x.weight = 1.f;
    x.bias = 0.f;
    const int tile = w / a.w_tiles, n = (w - tile * a.w_tiles) * 128 + in_tile;
    if (KIND != FEW_LINEAR) {
      const int place = tile_info[3 * tile + 1] + tok0 + lane;
      if (tok0 + lane < live && place >= 0 && place < a.S) {
        const int slot = sorted[place];
        if (slot >= 0 && slot < a.S) {
          x.slot = slot;
          if (KIND == FEW_GATED && sel_weight) x.weight = sel_weight[slot];
        }
      }
    } else if (n < a.N) {
      if (a.bias) x.bias = a.bias[n];
      if (a.residual) {
        const TO* res = reinterpret_cast<const TO*>(after_wait(a.residual)) + (long long)(tile * NT + tok0) * a.ldo + n;
#pragma unroll
        for (int j = 0; j < CH; ++j)
          if (tok0 + j < live) x.residual[j] = to_f(res[j * a.ldo]);
      }
    }
    return x;
  };
  // Numbers of tokens tok0 .. (below `live`) of item w: v (gated: gate v, up u) of column n.
  int flip = 0;
  auto finish = [&](int w, int tok0, int live, float (&v)[CH], float (&u)[CH], const Beside& x) {
    const int tile = w / a.w_tiles, n0 = (w - tile * a.w_tiles) * 128, n = n0 + in_tile;
    if (KIND == FEW_GATED) {
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        const float wgt = __shfl_sync(0xffffffffu, x.weight, j);
        v[j] = tok0 + j < live && n < a.N ? fp8_gated_unit(a.act, v[j], u[j], wgt, a.limit) : 0.f;
        const uint32_t top = __reduce_max_sync(0xffffffffu, fp8_magnitude(v[j]));
        if (lane == j) sm.top[flip][q][j] = top;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        if (tok0 + j >= live) break;
        const uint32_t top = max(max(sm.top[flip][0][j], sm.top[flip][1][j]), max(sm.top[flip][2][j], sm.top[flip][3][j]));
        const int e = fp8_exponent(top);
        const long long row = (long long)tile * NT + tok0 + j;
        if (n < a.ldo) reinterpret_cast<uint8_t*>(a.out)[row * a.ldo + n] = (uint8_t)fp8_pair(fp8_or_nan(v[j]) * fp8_power(-e), 0.f);
        if (in_tile == 0) {
          const int run = n0 >> 7;
          a.out_scales[((long long)tile * a.out_kgs + (run >> 2)) * FP8_TILE + fp8_scale_row(tok0 + j) + (run & 3)] = (uint8_t)(e + 127);
        }
      }
      flip ^= 1;
    } else {
      TO* out = reinterpret_cast<TO*>(a.out) + n;
      if (KIND == FEW_LINEAR) {
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] += x.bias;
        fp8_activate<sizeof(TO) == 2>(a.act, v);
        if (a.residual) {
#pragma unroll
          for (int j = 0; j < CH; ++j) v[j] += x.residual[j];
        }
        out += (long long)(tile * NT + tok0) * a.ldo;
      }
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        const long long row = KIND == FEW_LINEAR ? j : __shfl_sync(0xffffffffu, x.slot, j);
        if (tok0 + j < live && n < a.N && row >= 0) out[row * a.ldo] = from_f<TO>(v[j]);
      }
    }
  };
  auto live_of = [&](int w) {
    const int tile = w / a.w_tiles;
    return KIND == FEW_LINEAR ? min(NT, a.M - tile * NT) : min(NT, tile_info[3 * tile + 2]);
  };

  // tokens that a CTA of a cluster adds up and writes out
  const int share = SPLIT ? max(4, NT / ranks) : NT;
  if (warp >= 2) {
    if (SPLIT) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    int it = 0;
    for (int w = first_item; w < items; w += step, ++it) {
      const int b = S::ACC == 2 ? it & 1 : 0;
      const int live = live_of(w);
      Beside x;
      if (!SPLIT) x = fetch(w, 0, live);
      bool ok = mbar_wait(&sm.acc_full[b], (uint32_t)((S::ACC == 2 ? it >> 1 : it) & 1), abort_flag);
      if (KIND == FEW_GATED) ok = epilogue_agrees(ok);        // the four warps meet at barriers below
      if (!ok) break;
      fp8_after_sync();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * NH * NT);
#pragma unroll 1
      for (int c = 0; c < NT; c += CH) {
        uint32_t r[NH][32];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          if (CH == 32) tmem_ld32(acc + (uint32_t)(h * NT + c), r[h]);
          else tmem_ld16(acc + (uint32_t)(h * NT + c), r[h]);
        }
        fp8_wait_ld();
        fp8_arrived(r[0]);
        if (NH == 2) fp8_arrived(r[NH - 1]);
        if (c + CH >= NT) {
          fp8_before_sync();
          mbar_arrive(&sm.acc_empty[b]);
        }
        if (c >= live) continue;
        if (SPLIT) {
          const float4* mine = &sm.sums[rank * (share / 4) * NH * 128 + in_tile];
#pragma unroll
          for (int j = 0; j < CH; j += 4) {
            if (c + j >= live) break;
            const uint32_t at = peer_addr(mine + ((c + j) % share / 4) * NH * 128, (uint32_t)((c + j) / share));
#pragma unroll
            for (int h = 0; h < NH; ++h)
              asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};"
                           ::"r"(at + (uint32_t)(h * 2048)), "r"(r[h][j]), "r"(r[h][j + 1]), "r"(r[h][j + 2]), "r"(r[h][j + 3]) : "memory");
          }
        } else {
          float v[CH], u[CH];
#pragma unroll
          for (int j = 0; j < CH; ++j) { v[j] = __uint_as_float(r[0][j]); u[j] = __uint_as_float(r[NH - 1][j]); }
          if (c > 0) x = fetch(w, c, live);
          finish(w, c, live, v, u, x);
        }
      }
    }
  }
  if (SPLIT) {
    Beside x;
    if (warp >= 2 && first_item < items) x = fetch(first_item, rank * share, min(live_of(first_item), (rank + 1) * share));
    __syncwarp();
    if (warp < 2) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && sm.abort_flag)           // who gave up has sent nothing: nobody adds anything up
      for (int r = 0; r < ranks; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(&sm.abort_flag, (uint32_t)r)), "r"(1) : "memory");
    __syncwarp();
    cluster_sync();                      // all sums have arrived
    if (warp >= 2 && first_item < items && !*abort_flag) {
      const int live = live_of(first_item);
#pragma unroll 1
      for (int c = 0; c < share; c += CH) {
        const int tok0 = rank * share + c, end = min(live, (rank + 1) * share);
        if (tok0 >= end) break;          // the same for all four warps
        float v[CH], u[CH];
#pragma unroll
        for (int j = 0; j < CH; j += 4) {
          v[j] = v[j + 1] = v[j + 2] = v[j + 3] = u[j] = u[j + 1] = u[j + 2] = u[j + 3] = 0.f;
          if (tok0 + j < end) {
            const float4* p = &sm.sums[(c + j) / 4 * NH * 128 + in_tile];
            for (int from = 0; from < ranks; ++from, p += share / 4 * NH * 128) {
              const float4 x = p[0];
              v[j] += x.x; v[j + 1] += x.y; v[j + 2] += x.z; v[j + 3] += x.w;
              if (NH == 2) {
                const float4 y = p[128];
                u[j] += y.x; u[j + 1] += y.y; u[j + 2] += y.z; u[j + 3] += y.w;
              }
            }
          }
        }
        if (c > 0) x = fetch(first_item, tok0, end);
        finish(first_item, tok0, end, v, u, x);
      }
    }
  }

  __syncwarp();
  fp8_before_sync();
  __syncthreads();
  const bool aborted = sm.abort_flag != 0;
  if (threadIdx.x == 0 && aborted) atomicOr(a.status, MLXB_ST_WAIT_TIMEOUT);
  if (warp == 1) {
    if (aborted && lane == 0) {          // products already issued may still run on the memory that is freed below
      umma_commit(&sm.drained);
      fp8_drain(&sm.drained, 0u);
    }
    __syncwarp();
    fp8_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------- host side

// CTAs that share a tile's K (0: the environment asks for a number that cannot be).  A fit to measured times: a stage takes a CTA that has its SM to itself 0.25 us (62 GB/s, what one SM takes in) and two on one SM
// 0.42; a split costs 1.4 us and CTAs that do not find room at once 3.  Within 6 % of the best at 17 sizes.  (Microseconds at 1, 2, 4, 8 CTAs, the rounding of x before
// it included: 1 x 4096 x 4096 13.3, 11.2, 9.4, 9.1; 1 x 1600 x 6400 8.8, 8.6, 8.1, 11.8; 1 x 4096 x 14336 14.8, 15.9, 18.1, 23.9; 64 x 5120 x 1280
// 17.5, 16.3, 12.0, 10.2; 128 x 4096 x 6144 18.5, 19.6, 25.1, 40.5.)
static int few_ranks(long long items, int runs, bool two_an_sm) {
  if (const char* want = getenv("MLXB_FP8_RANKS")) {      // experiments and tests
    const int r = atoi(want);                             // shares of tokens are whole quadruples and every CTA has a run
    return r == 1 || ((r == 2 || r == 4 || r == 8) && runs >= r) ? r : 0;
  }
  const int sms = mlxb_sm_count();
  int best = 1;
  double best_cost = 0.;
  for (int r = 1; r <= 8; r *= 2) {
    if (r > 1 && (runs < 2 * r || items * r > 4LL * sms)) break;
    const long long ctas = items * r, room = two_an_sm && r > 1 && ctas > sms ? 2 * sms : sms;
    const long long waves = (ctas + room - 1) / room;
    const double cost = (double)waves * ((runs + r - 1) / r) * (room > sms ? 0.42 : 0.25) + (r > 1 ? 1.4 : 0.) + 3. * (double)(waves - 1);
    if (r == 1 || cost < best_cost) { best = r; best_cost = cost; }
  }
  return best;
}

template <int NT, int KIND, bool SPLIT, typename TO>
static int few_launch(const CUtensorMap& mw, const CUtensorMap& mx, const FewArgs& a, int ranks, cudaStream_t stream) {
  using S = FewShape<NT, KIND, SPLIT>;
  constexpr size_t smem = sizeof(FewSmem<NT, KIND, SPLIT>) + 1024;
  static_assert(S::STAGES >= 2 && smem <= 227 * 1024, "stages fit a CTA's shared memory");
  static_assert(!S::PAIR || 2 * (smem + 1024) <= 228 * 1024, "two CTAs an SM");
  auto kern = fp8_few_kernel<NT, KIND, SPLIT, TO>;
  static SharedLimit limit;
  if (cudaError_t e = limit.raise(kern, smem)) return mlxb_fail((int)e, "linear (8 bits): %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(SPLIT ? a.max_items * ranks : min(a.max_items, mlxb_sm_count()));
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (SPLIT) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = ranks;
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
  cudaLaunchKernelEx(&cfg, kern, mw, mx, a, ranks);
  return mlxb_check_launch("linear (8 bits)");
}

template <int NT, int KIND, typename TO>
static int few_choose(const CUtensorMap& mw, const CUtensorMap& mx, const FewArgs& a, cudaStream_t stream) {
  const int ranks = few_ranks(a.max_items, a.runs, FewShape<NT, KIND, true>::PAIR);
  if (!ranks) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): MLXB_FP8_RANKS is 1, 2, 4 or 8 and no more than the %d runs of 128 columns", a.runs);
  if (ranks > 1) return few_launch<NT, KIND, true, TO>(mw, mx, a, ranks, stream);
  return few_launch<NT, KIND, false, TO>(mw, mx, a, 1, stream);
}

template <typename TO>
static int few_width(int nt, const CUtensorMap& mw, const CUtensorMap& mx, const FewArgs& a, cudaStream_t stream) {
  switch (nt) {
    case 16: return few_choose<16, FEW_LINEAR, TO>(mw, mx, a, stream);
    case 32: return few_choose<32, FEW_LINEAR, TO>(mw, mx, a, stream);
    case 64: return few_choose<64, FEW_LINEAR, TO>(mw, mx, a, stream);
    default: return few_choose<128, FEW_LINEAR, TO>(mw, mx, a, stream);
  }
}

// x codes [M, K], w codes [N, K] (rows of K bytes, K a multiple of 16), their scales as in fp8.cuh (one group each); bias float32 [N] or null;
// residual of out's type at out's stride or null (may be out); out bfloat16 or float32 [M, N] at row stride ldo.
MLXB_EXPORT int mlxb_fp8_linear_few(const Fp8LinearRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(Fp8LinearRecord)) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): a record of %lld bytes", bytes);
  const Fp8LinearRecord& r = *rec;
  if (r.M <= 0 || r.N <= 0) return 0;
  if (int e = fp8_check("linear (8 bits)", r.x, r.xs, r.w, r.ws, r.out, r.M, r.N, r.K, r.ldo)) return e;
  if (!activation_known((int)r.epi) || !r.status) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): epilogue %lld", r.epi);
  const int M = (int)r.M, N = (int)r.N, K = (int)r.K;
  FewArgs a = {};
  a.x_scales = (const uint8_t*)r.xs; a.w_scales = (const uint8_t*)r.ws;
  a.M = M; a.N = N; a.runs = (K + 127) / 128; a.kgs = (K + 511) / 512; a.w_tiles = (N + 127) / 128;
  a.bias = r.bias; a.residual = r.residual; a.out = r.out; a.ldo = r.ldo; a.status = r.status; a.act = (int)r.epi;
  const int nt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  const long long items = (long long)a.w_tiles * ((M + nt - 1) / nt);
  if (items > 0x7fffff) return mlxb_fail(MLXB_BAD_ARG, "linear (8 bits): %d x %d outputs", M, N);
  a.max_items = (int)items;
  CUtensorMap mw, mx;
  if (int e = fp8_make_map(&mw, r.w, N, K, K, 128, "linear (8 bits) w")) return e;
  if (int e = fp8_make_map(&mx, r.x, M, K, K, nt, "linear (8 bits) x")) return e;
  return r.out_f32 ? few_width<float>(nt, mw, mx, a, stream) : few_width<__nv_bfloat16>(nt, mw, mx, a, stream);
}

// Over a plan with tiles of 16 slots; x codes [max_tiles * 16, K], a tile's rows at 16 t, scales a group a tile.
// gated: w codes [E][2][N][K] (gate rows, up rows), scales of 2 E groups of N rows; out codes [max_tiles * tile_rows, ldo] with their
// scales, ldo = N rounded up to 16.  Else w codes [E][N][K]; out bfloat16 or float32 rows [S, ldo], row sorted[i] for place i of the plan.
// at_most: a bound on the number of tiles.
MLXB_EXPORT int mlxb_fp8_experts_few(const Fp8ExpertsRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(Fp8ExpertsRecord)) return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: a record of %lld bytes", bytes);
  const Fp8ExpertsRecord& r = *rec;
  if (r.max_tiles <= 0 || r.at_most <= 0) return 0;
  if (int e = fp8_check_experts(r)) return e;
  if (r.tile_rows != 16) return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: tiles of %lld rows", r.tile_rows);
  const int N = (int)r.N, K = (int)r.K;
  FewArgs a = {};
  a.x_scales = (const uint8_t*)r.xs; a.w_scales = (const uint8_t*)r.ws;
  a.N = N; a.runs = (K + 127) / 128; a.kgs = (K + 511) / 512; a.w_tiles = (N + 127) / 128;
  a.sorted = r.sorted; a.tile_info = r.tile_info; a.n_tiles = r.n_tiles; a.sel_weight = r.sel_weight;
  a.out = r.out; a.ldo = r.ldo; a.out_scales = (uint8_t*)r.out_scales; a.out_kgs = (N + 511) / 512; a.status = r.status; a.act = (int)r.act;
  a.limit = (float)r.limit; a.E = (int)r.E; a.S = (int)r.S;
  const long long items = min(r.max_tiles, r.at_most) * a.w_tiles;
  if (items > 0x7fffff) return mlxb_fail(MLXB_BAD_ARG, "moe_gemm_fp8: %lld tiles of %d outputs", r.max_tiles, N);
  a.max_items = (int)items;
  CUtensorMap mw, mx;
  if (int e = fp8_make_map(&mw, r.w, r.E * (r.gated ? 2 : 1) * N, K, K, 128, "moe_gemm_fp8 w")) return e;
  if (int e = fp8_make_map(&mx, r.x, r.max_tiles * r.tile_rows, K, K, (int)r.tile_rows, "moe_gemm_fp8 x")) return e;
  if (r.gated) return few_choose<16, FEW_GATED, float>(mw, mx, a, stream);
  return r.out_f32 ? few_choose<16, FEW_EXPERTS, float>(mw, mx, a, stream) : few_choose<16, FEW_EXPERTS, __nv_bfloat16>(mw, mx, a, stream);
}
