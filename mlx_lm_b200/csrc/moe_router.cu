// The router of a feed-forward of experts, with the plan of the experts' products.
//
// route      per token: scores s = sigmoid(z) or softmax(z); choice scores c = s + correction; groups of neighbouring experts judged by their
//            best choice score or by the sum of their two best, the best groups stay; of their experts the `top` with the largest choice
//            scores (ties: the lower index); weights: the scores s, divided by their sum plus eps if wanted, times a factor.
// plan       the (token, choice) slots sorted by expert and, within one, by number; tiles of at most tile_rows slots of one expert.
//
// The choice is exact.  Without a correction the order of the scores is the order of the logits.  With one, or where sums of two decide, a warp
// compares the float32 scores it forms first, and where a choice was by less than they can be off (2^-20 of a score's range, some 16 times their
// error) it forms that token's scores again in 64 bits.  A score that is NaN, or that a correction makes minus infinity, is never chosen; places
// that nobody can take hold expert -1 and weight 0.
//
// A warp takes a token, a lane neighbouring experts, so that the lowest lane with the largest number has the lowest index: a choice is one
// redux.sync and one vote.  Steps of up to 64 tokens are one block and one launch.  More are two launches: blocks of tokens that also count
// their slots by expert, then the same blocks, which add up the counts before theirs and put their slots in place.  No atomics decide
// an order.
#include "common.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int RP_THREADS = 512, RP_WARPS = RP_THREADS / 32, RP_ONE_BLOCK = 64, RP_MOST_BLOCKS = 148;

struct RouterArgs {
  const float* logits;
  long long ldl;
  const int* token_req;
  const float* correction;
  int T, E, top, softmax, two, groups, keep, n_real, renorm;
  float eps, factor;
  int* sel;
  float* weight;
  int* counts;                 // [blocks][E] slots by expert of each block of tokens
  int tokens_a_block, tile_rows, max_tiles;
  int *sorted, *tile_info, *n_tiles;
};

// Whole numbers in the order of floats; 0 (below every number's): not a number, or out of the race.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return v == v ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float number_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The choice in 64 bits, for tokens whose float32 scores are too close: plain and slow.  sC: [E] doubles of this warp.
__device__ __noinline__ void choose_exactly(const RouterArgs& a, const float* z, float zmax, double* sC, int* sPick, int lane) {
  double sum = 0.;
  if (a.softmax) {
    for (int e = lane; e < a.E; e += 32) sum += z[e] == z[e] ? exp((double)z[e] - (double)zmax) : 0.;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  for (int e = lane; e < a.E; e += 32) {
    double s = a.softmax ? exp((double)z[e] - (double)zmax) / sum : 1. / (1. + exp(-(double)z[e]));
    if (a.correction) s += (double)a.correction[e];
    sC[e] = s;
  }
  __syncwarp();
  const int per = a.E / a.groups;
  uint32_t kept[4] = {~0u, ~0u, ~0u, ~0u};                 // of up to 128 groups
  if (a.keep < a.groups) {
    kept[0] = kept[1] = kept[2] = kept[3] = 0;
    for (int c = 0; c < a.keep; ++c) {
      double best = -INFINITY;
      int best_g = 0x7fffffff;
      for (int g = lane; g < a.groups; g += 32) {
        if (kept[g >> 5] >> (g & 31) & 1) continue;
        double b1 = -INFINITY, b2 = -INFINITY;
        int n = 0;
        for (int i = 0; i < per; ++i) {
          const double v = sC[g * per + i];
          if (!(v > -INFINITY)) continue;
          ++n;
          if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) { b2 = v; }
        }
        const double v = a.two && n > 1 ? b1 + b2 : b1;
        if (n && (best_g == 0x7fffffff || v > best)) { best = v; best_g = g; }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int og = __shfl_xor_sync(0xffffffffu, best_g, o);
        if (og != 0x7fffffff && (best_g == 0x7fffffff || ob > best || (ob == best && og < best_g))) { best = ob; best_g = og; }
      }
      if (best_g != 0x7fffffff) kept[best_g >> 5] |= 1u << (best_g & 31);
    }
  }
  for (int c = 0; c < a.top; ++c) {
    double best = -INFINITY;
    int best_e = 0x7fffffff;
    for (int e = lane; e < a.E; e += 32) {
      const int g = e / per;
      const double v = sC[e];
      if (!(v > -INFINITY) || !(kept[g >> 5] >> (g & 31) & 1)) continue;
      if (best_e == 0x7fffffff || v > best) { best = v; best_e = e; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o);
      const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
      if (oe != 0x7fffffff && (best_e == 0x7fffffff || ob > best || (ob == best && oe < best_e))) { best = ob; best_e = oe; }
    }
    if (lane == 0) sPick[c] = best_e == 0x7fffffff ? -1 : best_e;
    __syncwarp();
    if (best_e != 0x7fffffff && (best_e & 31) == lane) sC[best_e] = NAN;
    __syncwarp();
  }
}

// One token by one warp.  VPT experts a lane, neighbours.  sS: [E] scores, sC: room for [E] doubles, sPick: [top].
template <int VPT>
__device__ __forceinline__ void route_token(const RouterArgs& a, const float* logits, int t, float* sS, double* sC, int* sPick, int* sCount, int lane) {
  if (a.token_req && a.token_req[t] < 0) {
    for (int c = lane; c < a.top; c += 32) { a.sel[(size_t)t * a.top + c] = -1; a.weight[(size_t)t * a.top + c] = 0.f; }
    return;
  }
  const float* z = logits + (size_t)t * a.ldl;
  const int e0 = lane * VPT;
  float s[VPT];
  uint32_t key[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) s[i] = e0 + i < a.E ? z[e0 + i] : NAN;
  float zmax = -INFINITY;
  if (a.softmax) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) zmax = fmaxf(zmax, s[i]);
    zmax = warp_max(zmax);
  }
  const bool by_logit = a.correction == nullptr;
  if (by_logit) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) key[i] = order_of(s[i]);
  }
  float range = 1.f;                                        // no score is larger
  if (a.softmax) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      s[i] = expf(s[i] - zmax);
      sum += s[i] == s[i] ? s[i] : 0.f;
    }
    sum = warp_sum(sum);
    range = 1.f / sum;
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] = s[i] / sum;
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] = 1.f / (1.f + expf(-s[i]));
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (e0 + i < a.E) sS[e0 + i] = s[i];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const float c = s[i] + (!by_logit && e0 + i < a.E ? a.correction[e0 + i] : 0.f);
    if (!(c > -INFINITY)) key[i] = 0;
    else if (!by_logit) key[i] = order_of(c);
  }
  bool close = false;
  auto near = [&](float hi, float lo) { return hi - lo <= 9.5e-7f * range + 4.8e-7f * (fabsf(hi) + fabsf(lo)); };

  if (a.keep < a.groups) {
    // a group's members are neighbours, and so are the lanes that hold them; by logits, the sums of two want the scores
    const int per = a.E / a.groups;
    const bool sums = a.two && per > 1;
    uint32_t mine[4];                                       // lane l: groups l, l + 32, ...
#pragma unroll
    for (int x = 0; x < 4; ++x) mine[x] = 0;
    for (int g = 0; g < a.groups; ++g) {
      const int lo = g * per, hi = lo + per;
      uint32_t b1 = 0, b2 = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t k = e0 + i >= lo && e0 + i < hi ? key[i] : 0u;
        if (k > b1) { b2 = b1; b1 = k; } else if (k > b2) { b2 = k; }
      }
      const uint32_t top1 = __reduce_max_sync(0xffffffffu, b1);
      uint32_t v = top1;
      if (sums && top1) {
        const bool owner = __ffs(__ballot_sync(0xffffffffu, b1 == top1)) - 1 == lane;
        const uint32_t top2 = __reduce_max_sync(0xffffffffu, owner ? b2 : b1);
        float f1 = number_of(top1), f2 = top2 ? number_of(top2) : 0.f;
        if (by_logit) {
          f1 = a.softmax ? expf(f1 - zmax) * range : 1.f / (1.f + expf(-f1));
          f2 = !top2 ? 0.f : a.softmax ? expf(f2 - zmax) * range : 1.f / (1.f + expf(-f2));
        }
        v = order_of(f1 + f2);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (g == lane + 32 * x) mine[x] = v;
    }
    uint32_t kept[4] = {0, 0, 0, 0}, last = 0;
    for (int c = 0; c <= a.keep; ++c) {                      // one more than stay: was the last choice close?
      uint32_t b = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) b = max(b, mine[x]);
      const uint32_t best = __reduce_max_sync(0xffffffffu, b);
      if (c > 0 && best && near(number_of(last), number_of(best)) && (sums || !by_logit)) close = true;
      if (!best || c == a.keep) break;
      last = best;
      bool done = false;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t who = __ballot_sync(0xffffffffu, mine[x] == best);
        if (!done && who) {
          const int l = __ffs(who) - 1;
          kept[x] |= 1u << l;
          if (lane == l) mine[x] = 0;
          done = true;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = (e0 + i) / per;
      uint32_t bits = kept[0];
#pragma unroll
      for (int x = 1; x < 4; ++x) bits = g >> 5 == x ? kept[x] : bits;
      if (!(bits >> (g & 31) & 1)) key[i] = 0;
    }
  }

  uint32_t last = 0;
  for (int c = 0; c <= a.top; ++c) {
    uint32_t b = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (key[i] > b) { b = key[i]; at = i; }
    const uint32_t best = __reduce_max_sync(0xffffffffu, b);
    if (c > 0 && best && last && !by_logit && near(number_of(last), number_of(best))) close = true;
    if (c == a.top) break;
    last = best;
    const int l = __ffs(__ballot_sync(0xffffffffu, b == best)) - 1;
    if (lane == l) {
      sPick[c] = best ? e0 + at : -1;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (i == at) key[i] = 0;
    }
  }
  __syncwarp();
  if (close) choose_exactly(a, z, zmax, sC, sPick, lane);    // the same answer in every lane: all it goes by came from votes
  __syncwarp();
  float sum = 0.f;
  for (int c = 0; c < a.top; ++c) sum += sPick[c] >= 0 ? sS[sPick[c]] : 0.f;
  for (int c = lane; c < a.top; c += 32) {
    const int e = sPick[c];
    float w = e >= 0 ? sS[e] : 0.f;
    if (a.renorm && e >= 0) w = w / (sum + a.eps);
    a.weight[(size_t)t * a.top + c] = w * a.factor;
    a.sel[(size_t)t * a.top + c] = e < 0 ? -1 : e < a.n_real ? e : -2;
    if (e >= 0 && e < a.n_real) atomicAdd(&sCount[e], 1);    // only a number of slots: no order comes of it
  }
  __syncwarp();
}

// Puts the slots first .. first + n - 1 of one block in place.  sBase [E]: the place of the block's next slot of each expert; sWarp [RP_WARPS][E].
__device__ __forceinline__ void place_slots(const RouterArgs& a, const int* sel, int first, int n, int* sBase, int* sWarp) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int at = 0; at < n; at += RP_THREADS) {
    for (int i = threadIdx.x; i < RP_WARPS * a.n_real; i += RP_THREADS) sWarp[i] = 0;
    __syncthreads();
    const int i = at + threadIdx.x;
    int e = i < n ? sel[first + i] : -1;
    if (e >= a.n_real) e = -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && before == 0) sWarp[warp * a.n_real + e] = __popc(same);
    __syncthreads();
    for (int x = threadIdx.x; x < a.n_real; x += RP_THREADS) {
      int acc = sBase[x];
      for (int w = 0; w < RP_WARPS; ++w) {
        const int c = sWarp[w * a.n_real + x];
        sWarp[w * a.n_real + x] = acc;
        acc += c;
      }
      sBase[x] = acc;
    }
    __syncthreads();
    if (e >= 0) a.sorted[sWarp[warp * a.n_real + e] + before] = first + i;
    __syncthreads();
  }
}

// From totals sTotal [n_real] by expert: places sFirst; `tiles`: writes the list of tiles too.  By the whole block.
__device__ __forceinline__ void plan_experts(const RouterArgs& a, const int* sTotal, int* sFirst, bool tiles) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, per = (a.n_real + 31) / 32, lo = lane * per, hi = min(a.n_real, lo + per);
    int n = 0, nt = 0;
    for (int e = lo; e < hi; ++e) { n += sTotal[e]; nt += (sTotal[e] + a.tile_rows - 1) / a.tile_rows; }
    int pn = n, pt = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, pn, o), y = __shfl_up_sync(0xffffffffu, pt, o);
      if (lane >= o) { pn += x; pt += y; }
    }
    if (tiles && lane == 31) a.n_tiles[0] = min(pt, a.max_tiles);
    pn -= n;
    pt -= nt;
    for (int e = lo; e < hi; ++e) {
      sFirst[e] = pn;
      if (tiles)
        for (int r = 0; r < sTotal[e]; r += a.tile_rows, ++pt)
          if (pt < a.max_tiles) {
            a.tile_info[3 * pt] = e;
            a.tile_info[3 * pt + 1] = pn + r;
            a.tile_info[3 * pt + 2] = min(a.tile_rows, sTotal[e] - r);
          }
      pn += sTotal[e];
    }
  }
  __syncthreads();
}

// ONE: the whole step in this block, with its plan.  Shared memory: counts [E], places [E], by warp: scores [E], doubles [E], picks [top]; the
// plan's [RP_WARPS][E] lie over the latter.
template <int VPT, bool ONE>
__global__ void __launch_bounds__(RP_THREADS) route_kernel(const __grid_constant__ RouterArgs a) {
  extern __shared__ __align__(16) uint8_t rp_smem[];
  int* sCount = reinterpret_cast<int*>(rp_smem);
  int* sFirst = sCount + a.E;
  double* sC = reinterpret_cast<double*>(rp_smem + ((size_t)8 * a.E + 15) / 16 * 16);
  float* sS = reinterpret_cast<float*>(sC + (size_t)RP_WARPS * a.E);
  int* sPick = reinterpret_cast<int*>(sS + (size_t)RP_WARPS * a.E);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < a.E; e += RP_THREADS) sCount[e] = 0;
  pdl_wait();
  pdl_trigger();
  const float* logits = after_wait(a.logits);
  __syncthreads();
  const int t0 = blockIdx.x * a.tokens_a_block, t1 = min(a.T, t0 + a.tokens_a_block);
  for (int t = t0 + warp; t < t1; t += RP_WARPS)
    route_token<VPT>(a, logits, t, sS + (size_t)warp * a.E, sC + (size_t)warp * a.E, sPick + warp * a.top, sCount, lane);
  __syncthreads();
  if (ONE) {
    plan_experts(a, sCount, sFirst, true);
    place_slots(a, after_wait(a.sel), 0, a.T * a.top, sFirst, reinterpret_cast<int*>(sC));
  } else {
    for (int e = threadIdx.x; e < a.n_real; e += RP_THREADS) a.counts[(size_t)blockIdx.x * a.n_real + e] = sCount[e];
  }
}

__global__ void __launch_bounds__(RP_THREADS) plan_kernel(const __grid_constant__ RouterArgs a, int blocks) {
  extern __shared__ __align__(16) uint8_t rp_smem[];
  int* sTotal = reinterpret_cast<int*>(rp_smem);
  int* sFirst = sTotal + a.E;
  int* sWarp = sFirst + a.E;                     // [RP_WARPS][E]
  pdl_wait();
  pdl_trigger();
  const int* counts = after_wait(a.counts);
  // totals, and what the blocks before this one hold, by warps over the blocks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* sBefore = sWarp;
  for (int e = threadIdx.x; e < a.n_real; e += RP_THREADS) sTotal[e] = sBefore[e] = 0;
  __syncthreads();
  for (int e0 = 0; e0 < a.n_real; e0 += 32) {
    const int e = e0 + lane;
    int all = 0, before = 0;
    if (e < a.n_real)
      for (int b = warp; b < blocks; b += RP_WARPS) {
        const int c = counts[(size_t)b * a.n_real + e];
        all += c;
        if (b < blockIdx.x) before += c;
      }
    if (e < a.n_real && all) { atomicAdd(&sTotal[e], all); atomicAdd(&sBefore[e], before); }
  }
  __syncthreads();
  plan_experts(a, sTotal, sFirst, blockIdx.x == 0);
  for (int e = threadIdx.x; e < a.n_real; e += RP_THREADS) sFirst[e] += sBefore[e];
  __syncthreads();
  const int t0 = blockIdx.x * a.tokens_a_block, t1 = min(a.T, t0 + a.tokens_a_block);
  place_slots(a, after_wait(a.sel), t0 * a.top, (t1 - t0) * a.top, sFirst, sWarp);
}

static int tokens_a_block(int T) { return T <= RP_ONE_BLOCK ? T : max(16, (T + RP_MOST_BLOCKS - 1) / RP_MOST_BLOCKS); }

// How many whole numbers of scratch memory a step of T tokens wants.
MLXB_EXPORT int mlxb_moe_route_scratch(int T, int E) {
  if (T <= RP_ONE_BLOCK || E <= 0) return 1;
  const int tpb = tokens_a_block(T);
  return (T + tpb - 1) / tpb * E;
}

template <int VPT>
static int route_launch(const RouterArgs& a, int blocks, size_t smem, cudaStream_t stream) {
  static SharedLimit one, many;
  constexpr size_t most = 227 * 1024;
  if (blocks == 1) {
    if (cudaError_t e = one.raise(route_kernel<VPT, true>, most)) return mlxb_fail((int)e, "moe_route_plan: shared memory: %s", cudaGetErrorString(e));
    launch_pdl(route_kernel<VPT, true>, dim3(1), dim3(RP_THREADS), smem, stream, a);
  } else {
    if (cudaError_t e = many.raise(route_kernel<VPT, false>, most)) return mlxb_fail((int)e, "moe_route_plan: shared memory: %s", cudaGetErrorString(e));
    launch_pdl(route_kernel<VPT, false>, dim3(blocks), dim3(RP_THREADS), smem, stream, a);
  }
  return mlxb_check_launch("moe_route_plan");
}

// logits float32 [T, E] at row stride ldl.  n_real: experts n_real .. E - 1 have no tensors (identity): chosen, they are marked -2 and the plan passes over them.
// sel, weight [T * top]; sorted [T * top]; tile_info [max_tiles][3]; n_tiles [1]; counts: mlxb_moe_route_scratch(T, E) whole numbers.
MLXB_EXPORT int mlxb_moe_route_plan(const float* logits, long long ldl, const int* token_req, const float* correction, int T, int E, int top, int softmax,
                                    int two, int groups, int keep, int n_real, int renorm, float eps, float factor, int* sel, float* weight, int* counts,
                                    int tile_rows, int max_tiles, int* sorted, int* tile_info, int* n_tiles, cudaStream_t stream) {
  if (T < 0 || E <= 0 || E > 1024 || top <= 0 || top > E || top > 64 || ldl < E || groups < 1 || groups > 128 || E % groups || keep < 1 || keep > groups ||
      n_real < 1 || n_real > E || top > keep * (E / groups) || tile_rows < 1 || (long long)T * top > 0x7ffffff0LL ||
      max_tiles < ((long long)T * top + tile_rows - 1) / tile_rows + n_real)
    return mlxb_fail(MLXB_BAD_ARG, "moe_route_plan: %d tokens, %d of %d experts (%d with tensors; up to 64 of 1024), %d of %d groups (up to 128), tiles of %d rows, room for %d",
                     T, top, E, n_real, keep, groups, tile_rows, max_tiles);
  if (T == 0) {
    const cudaError_t e = cudaMemsetAsync(n_tiles, 0, sizeof(int), stream);
    return e == cudaSuccess ? 0 : mlxb_fail((int)e, "moe_route_plan: %s", cudaGetErrorString(e));
  }
  RouterArgs a = {logits, ldl, token_req, correction, T, E, top, softmax, two, groups, keep, n_real, renorm, eps, factor, sel, weight, counts,
                  tokens_a_block(T), tile_rows, max_tiles, sorted, tile_info, n_tiles};
  const int blocks = (T + a.tokens_a_block - 1) / a.tokens_a_block;
  const size_t head = ((size_t)8 * E + 15) / 16 * 16;
  const size_t smem = head + (size_t)RP_WARPS * (12 * (size_t)E + 4 * (size_t)top);
  int rc;
  if (E <= 32) rc = route_launch<1>(a, blocks, smem, stream);
  else if (E <= 64) rc = route_launch<2>(a, blocks, smem, stream);
  else if (E <= 128) rc = route_launch<4>(a, blocks, smem, stream);
  else if (E <= 256) rc = route_launch<8>(a, blocks, smem, stream);
  else if (E <= 512) rc = route_launch<16>(a, blocks, smem, stream);
  else rc = route_launch<32>(a, blocks, smem, stream);
  if (rc || blocks == 1) return rc;
  static SharedLimit limit;
  if (cudaError_t e = limit.raise(plan_kernel, 128 * 1024)) return mlxb_fail((int)e, "moe_route_plan: shared memory: %s", cudaGetErrorString(e));
  launch_pdl(plan_kernel, dim3(blocks), dim3(RP_THREADS), sizeof(int) * (2 + (size_t)RP_WARPS) * E, stream, a, blocks);
  return mlxb_check_launch("moe_route_plan (plan)");
}
