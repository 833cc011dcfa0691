// The router of a feed-forward of experts, with the plan of the experts' products.
//
// route      per token: scores s = sigmoid(z) or softmax(z); choice scores c = s + correction; groups of neighbouring experts judged by their
//            best choice score or by the sum of their two best, the best groups stay; of their experts the `top` with the largest choice
//            scores (ties: the lower index); weights: the scores s, divided by their sum plus eps if wanted, times a factor.
// plan       the (token, choice) slots sorted by expert and, within one, by number; tiles of at most tile_rows slots of one expert.
//
// The choice is exact: without a correction scores are in the order of the logits, and these are compared; with one, a warp compares float32 scores,
// which it forms with the hardware's exponential and quotient.  Where a choice was by less than these can be off, the two scores it was
// between, if they were two, are formed again in 64 bits, else all of the token's are and it chooses by those.  A score that is NaN, or that a correction
// makes minus infinity, is never chosen; places that nobody can take hold expert -1 and weight 0.
//
// A warp takes a token, a lane neighbouring experts.  Each lane sorts its scores once (a network of minima and maxima); a choice is then a redux.sync
// over the lanes' best, a vote, and a shift in the lane that had it.  Groups: 2^p lanes search one
// group's scores in shared memory and merge their two best; a group's rank is the number of better ones.
//
// Steps of up to 128 tokens are one launch: a cluster of up to eight CTAs, a warp a token, of which the first makes the plan.  More are two launches:
// blocks of tokens that also count their slots by expert, then the same blocks, which add up the counts before theirs and put their slots in place.
// No atomics decide an order.
//
// In us: 64 tokens of 256 experts, 8 groups of which 4 stay, top 8: 10.1, a chain of latencies; 8192 of the same 29.5: 21 of choosing (8 MB of logits;
// bound by instructions), 8 of the plan, which adds up 148 blocks' counts.
#include <float.h>

#include "common.cuh"

MLXB_DEFINE_LAST_ERROR()

constexpr int RP_THREADS = 512, RP_WARPS = RP_THREADS / 32, RP_CLUSTER = 8, RP_ONE_LAUNCH = RP_CLUSTER * RP_WARPS, RP_MOST_BLOCKS = 148;
constexpr int PL_THREADS = 1024, PL_WARPS = PL_THREADS / 32;

struct RouterArgs {
  const float* logits;
  long long ldl;
  const int* token_req;
  const float* correction;
  int T, E, top, softmax, two, groups, keep, n_real, renorm;
  int part;                    // lanes that search a group: a power of two, part * groups <= 32 (0: more than 32 groups)
  float eps, factor;
  int* sel;
  float* weight;
  int* counts;                 // [blocks][n_real rounded up to 4] slots by expert of each block of tokens
  int tokens_a_block, tile_rows, tile_shift, max_tiles;       // tile_shift: -1 where tile_rows is no power of two
  int *sorted, *tile_info, *n_tiles;
};

// Whole numbers in the order of floats, the two zeros one (the sum makes them +0); 0 (below every number's): not a number, or out of the race.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v == v ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float number_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.);
  return v == v ? (b >> 63 ? ~b : b | 1ull << 63) : 0ull;
}

// The choice in 64 bits, for tokens whose float32 scores are too close.  sC: [E] doubles of this warp.  No two scores are taken for different
// that are equal here; of equal ones the lower index is chosen.
template <int VPT>
__device__ __noinline__ void choose_exactly(const RouterArgs& a, const float* z, float zmax, double* sC, int* sPick, int lane) {
  const int e0 = lane * VPT, per = a.E / a.groups;
  double v[VPT], sum = 0.;
#pragma unroll 1
  for (int i = 0; i < VPT; ++i) {
    const double x = e0 + i < a.E ? (double)z[e0 + i] : NAN;
    if (a.softmax && x == x) sum += exp(x - (double)zmax);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  // what the choice goes by (without a correction: the logits), NaN out of the race; in shared memory what groups are judged by
#pragma unroll 1
  for (int i = 0; i < VPT; ++i) {
    const int e = e0 + i;
    const double x = e < a.E ? (double)z[e] : NAN;
    const double s = a.softmax ? exp(x - (double)zmax) / sum : 1. / (1. + exp(-x));
    const double c = s + (a.correction && e < a.E ? (double)a.correction[e] : 0.);
    if (e < a.E) sC[e] = !(c > -INFINITY) ? NAN : a.correction || a.two ? c : x;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    v[i] = e0 + i < a.E ? sC[e0 + i] : NAN;
    if (!a.correction && v[i] == v[i]) v[i] = (double)z[e0 + i];
  }
  if (a.keep < a.groups) {
    unsigned long long judged[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int g = lane + 32 * x;
      double b1 = -INFINITY, b2 = -INFINITY;
      bool any = false, two = false;
      if (g < a.groups)
        for (int i = 0; i < per; ++i) {
          const double c = sC[g * per + i];
          if (!(c == c)) continue;
          two = any;
          any = true;
          if (c > b1) { b2 = b1; b1 = c; } else if (c > b2) { b2 = c; }
        }
      judged[x] = any ? order_of(a.two && two ? b1 + b2 : b1) : 0ull;
    }
    __syncwarp();
    unsigned long long* all = reinterpret_cast<unsigned long long*>(sC);     // [groups], no more than experts
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 32 * x < a.groups) all[lane + 32 * x] = judged[x];
    __syncwarp();
    uint32_t kept[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      int better = 0;
      if (lane + 32 * x < a.groups)
        for (int g = 0; g < a.groups; ++g) better += all[g] > judged[x] || (all[g] == judged[x] && g < lane + 32 * x);
      kept[x] = __ballot_sync(0xffffffffu, judged[x] != 0ull && better < a.keep);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = (e0 + i) / per;
      const uint32_t bits = g < 32 ? kept[0] : g < 64 ? kept[1] : g < 96 ? kept[2] : kept[3];
      if (!(bits >> (g & 31) & 1)) v[i] = NAN;
    }
  }
  for (int c = 0; c < a.top; ++c) {
    unsigned long long best = 0ull;
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const unsigned long long k = order_of(v[i]);
      if (k > best) { best = k; at = i; }
    }
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    const unsigned long long top = (unsigned long long)hi << 32 | lo;
    const int l = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
    if (lane == l) {
      sPick[c] = top ? e0 + at : -1;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (i == at) v[i] = NAN;
    }
  }
  __syncwarp();
}

// What the choice of expert e goes by, in 64 bits.
__device__ __forceinline__ double exact_sigmoid(const RouterArgs& a, const float* z, int e) {
  return 1. / (1. + exp(-(double)z[e])) + (a.correction ? (double)a.correction[e] : 0.);
}
// The two largest of a group's, added up, in 64 bits by the whole warp; numbers out of the race are minus infinity.
__device__ __noinline__ double exact_two(const RouterArgs& a, const float* z, int first, int per, int lane) {
  double b1 = -INFINITY, b2 = -INFINITY;
  for (int i = lane; i < per; i += 32) {
    double v = exact_sigmoid(a, z, first + i);
    v = v == v ? v : -INFINITY;
    if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) { b2 = v; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
    b2 = fmax(fmax(b2, o2), fmin(b1, o1));
    b1 = fmax(b1, o1);
  }
  return a.two && b2 > -INFINITY ? b1 + b2 : b1;
}

// Descending, by a network of comparisons (odd-even merging).
template <int N>
__device__ __forceinline__ void sort_down(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t x = k[i + j], y = k[i + j + q];
            k[i + j] = max(x, y);
            k[i + j + q] = min(x, y);
          }
}

// One token by one warp.  VPT (a power of two) experts a lane, neighbours.  sC: room for [E] doubles, sPick: [top].
template <int VPT>
__device__ __forceinline__ void route_token(const RouterArgs& a, const float* logits, int t, double* sC, int* sPick, int* sCount, int lane) {
  if (a.token_req && a.token_req[t] < 0) {
    for (int c = lane; c < a.top; c += 32) { a.sel[(size_t)t * a.top + c] = -1; a.weight[(size_t)t * a.top + c] = 0.f; }
    return;
  }
  const float* z = logits + (size_t)t * a.ldl;
  const int e0 = lane * VPT;
  float s[VPT];
  if (VPT >= 4 && !(a.ldl & 3) && !(a.E & 3) && !((uintptr_t)logits & 15)) {
#pragma unroll
    for (int i = 0; i < VPT; i += 4) {
      const float4 v = e0 + i < a.E ? *reinterpret_cast<const float4*>(z + e0 + i) : make_float4(NAN, NAN, NAN, NAN);
      s[i] = v.x; s[(i + 1) % VPT] = v.y; s[(i + 2) % VPT] = v.z; s[(i + 3) % VPT] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] = e0 + i < a.E ? z[e0 + i] : NAN;
  }
  float v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) v[i] = s[i];
  float zmax = -INFINITY, sum = 0.f, range = 1.f;           // range: no score is larger
  if (a.softmax) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) zmax = fmaxf(zmax, s[i]);
    zmax = warp_max(zmax);
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] = __expf(s[i] - zmax);
    float part[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) part[i] = s[i] == s[i] ? s[i] : 0.f;
#pragma unroll
    for (int n = VPT / 2; n > 0; n /= 2)
#pragma unroll
      for (int i = 0; i < n; ++i) part[i] += part[i + n];
    sum = warp_sum(part[0]);
    range = __fdividef(1.f, sum);
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] *= range;
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] = __fdividef(1.f, 1.f + __expf(-s[i]));
  }
  if (a.correction) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] += e0 + i < a.E ? a.correction[e0 + i] : 0.f;
  } else {                       // in the race: z is what the choice goes by
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = s[i] == s[i] ? fmaxf(v[i], -FLT_MAX) : NAN;
    if (!a.two) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) s[i] = v[i];
    }
  }
  // How far a choice score is off, in steps of 2^-24.  Sigmoid: by less than 4 (a quarter of the exponential's relative error, a sum, a quotient), so that
  // the difference of two scores is by 8, of two sums of two by 16.  Softmax, steps of the range (the largest score): a term exp(-y) is off by 2 (2 + 1.173 y) + y of
  // itself, with its product by no more than 5 of the range; the sum, added in a tree, by 10 for its additions and by what its terms are off, 19 at most (1024
  // terms, one at y = 0, the others near y = 5); its inverse by 4.  So the range is off by 33 of its own steps, and with it every difference by 33 of itself: 43 for
  // two scores, 86 for two sums of two.  Each sum with a correction or of two adds one step of itself.  Without a correction the logits decide, as they are.
  bool close = false;
  const bool by_score = a.correction || a.two;              // what groups are judged by
  const float steps_one = !a.correction ? 0.f : a.softmax ? 43.f : 16.f, steps_group = !by_score ? 0.f : !a.softmax ? 16.f : a.two ? 86.f : 43.f;
  auto near = [&](float hi, float lo, float steps) {
    return !(hi - lo > (steps == 0.f ? 0.f : steps * 0x1p-24f * range + 1.2e-7f * (fabsf(hi) + fabsf(lo))));
  };

  uint32_t kept = ~0u;                                      // by the first lane of a group
  const int per = a.E / a.groups;
  if (a.keep < a.groups) {
    if (a.part == 0) {
      close = true;
    } else {
      float* sF = reinterpret_cast<float*>(sC);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (e0 + i < a.E) sF[e0 + i] = s[i];
      __syncwarp();
      const int g = lane / a.part, j = lane - g * a.part;
      float b1 = -INFINITY, b2 = -INFINITY;
      if (g < a.groups)
        for (int i = j; i < per; i += a.part) {
          const float x = sF[g * per + i];                  // NaN: neither maximum takes it
          b2 = fmaxf(b2, fminf(b1, x == x ? x : -INFINITY));
          b1 = fmaxf(b1, x);
        }
      for (int o = a.part >> 1; o > 0; o >>= 1) {
        const float o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
        b2 = fmaxf(fmaxf(b2, o2), fminf(b1, o1));
        b1 = fmaxf(b1, o1);
      }
      const bool pair = a.two && b2 > -INFINITY;
      const float score = pair ? fmaxf(b1 + b2, -FLT_MAX) : b1;                       // two of the lowest numbers are still in the race
      // its two may be far larger than their sum: half of what a difference is off, and the roundings of each and of the sum
      const float err = by_score ? 0.5f * steps_group * 0x1p-24f * range + 2.4e-7f * fminf(fabsf(b1) + (pair ? fabsf(b2) : 0.f), FLT_MAX) : 0.f;
      int better = 0;
      for (int x = 0; x < a.groups; ++x) {
        const float other = __shfl_sync(0xffffffffu, score, x * a.part);
        better += other > score || (other == score && x < g);
      }
      const bool mine = g < a.groups && score > -INFINITY, stays = mine && better < a.keep;
      kept = __ballot_sync(0xffffffffu, stays && j == 0);
      // the worst that may stay against the best that may go
      const float least = score - err, most = score + err;
      const uint32_t worst = __reduce_min_sync(0xffffffffu, stays ? order_of(least) : ~0u);
      const uint32_t best = __reduce_max_sync(0xffffffffu, mine && !stays ? order_of(most) : 0u);
      if (best && worst != ~0u && !(number_of(worst) > number_of(best))) {
        // one on either side: formed again in 64 bits; more than that, the whole token
        const uint32_t here = __ballot_sync(0xffffffffu, j == 0 && stays && !(least > number_of(best)));
        const uint32_t there = __ballot_sync(0xffffffffu, j == 0 && mine && !stays && !(number_of(worst) > most));
        if (a.softmax || !by_score || __popc(here) != 1 || __popc(there) != 1) {
          close = true;
        } else {
          const int la = __ffs(here) - 1, lb = __ffs(there) - 1, ga = la / a.part, gb = lb / a.part;
          const double x = exact_two(a, z, ga * per, per, lane), y = exact_two(a, z, gb * per, per, lane);
          if (y > x || (y == x && gb < ga)) kept = (kept & ~(1u << la)) | 1u << lb;
        }
      }
      __syncwarp();
    }
  }

  uint32_t key[VPT], was[VPT];
  const float inv_per = 1.f / (float)per;
  uint32_t open = ~0u;                                      // by this lane's experts: their group stays
  if (kept != ~0u) {
    if (!(per & (VPT - 1))) {                               // all of one group
      open = kept >> (((int)(((float)e0 + 0.5f) * inv_per) * a.part) & 31) & 1 ? ~0u : 0u;
    } else {
      open = 0u;
#pragma unroll 1
      for (int i = 0; i < VPT; ++i) open |= (kept >> (((int)(((float)(e0 + i) + 0.5f) * inv_per) * a.part) & 31) & 1) << i;
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (a.correction) v[i] = s[i];
    was[i] = key[i] = v[i] > -INFINITY && (open >> i & 1) ? order_of(v[i]) : 0u;
  }
  sort_down(key);
  // A choice is the lane and the key; which of the lane's experts it was is looked up for all choices at once, and before that only for two that are close.
  uint32_t* sKey = reinterpret_cast<uint32_t*>(sC);         // [top], no more than experts
  auto expert_of = [&](uint32_t k, int l) {
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) at = was[i] == k ? i : at;         // two equal ones of a lane are close
    return __shfl_sync(0xffffffffu, e0 + at, l);
  };
  uint32_t last = 0;
  int last_l = 0;
  bool again = false;
  // one more than are chosen: was the last choice close?  One more again if it was: a third one may be as close
  for (int c = 0; c <= a.top + 1; ++c) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, key[0]);
    if (!best) {
      for (int x = c + lane; x < a.top; x += 32) sPick[x] = -1;
      break;
    }
    const int l = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
    uint32_t put = best;
    int put_l = l;
    if (c > 0 && near(number_of(last), number_of(best), steps_one)) {
      // two that are close, and none beside them: lane 0 has the one before, the others this one
      const int e = expert_of(best, l), last_e = expert_of(last, last_l);
      if (a.softmax || again || e == last_e || !a.correction) { close = true; break; }
      again = true;
      const double x = exact_sigmoid(a, z, lane == 0 ? last_e : e), before = __shfl_sync(0xffffffffu, x, 0), now = __shfl_sync(0xffffffffu, x, 1);
      if (now > before || (now == before && e < last_e)) {
        if (lane == 0) { sPick[c - 1] = l; sKey[c - 1] = best; }
        put = last;
        put_l = last_l;
      }
    } else {
      again = false;
    }
    if (c >= a.top && !again) break;
    if (lane == 0 && c < a.top) { sPick[c] = put_l; sKey[c] = put; }
    last = best;
    last_l = l;
    if (lane == l) {
#pragma unroll
      for (int i = 0; i + 1 < VPT; ++i) key[i] = key[i + 1];
      key[VPT - 1] = 0;
    }
  }
  __syncwarp();
  if (!close) {
    for (int c0 = 0; c0 < a.top; c0 += 32) {
      const int c = c0 + lane, l = c < a.top ? sPick[c] : -1;
      const uint32_t k = l >= 0 ? sKey[c] : 0u;
      int at = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) at = __shfl_sync(0xffffffffu, was[i], l & 31) == k ? i : at;
      if (l >= 0) sPick[c] = l * VPT + at;
    }
    __syncwarp();
  }
  if (close) choose_exactly<VPT>(a, z, zmax, sC, sPick, lane);    // the same answer in every lane: all it goes by came from votes
  __syncwarp();
  // the weights of those that were chosen, with the library's exponential
  float mass = 0.f;
  for (int c0 = 0; c0 < a.top; c0 += 32) {
    const int e = c0 + lane < a.top ? sPick[c0 + lane] : -1;
    const float w = e < 0 ? 0.f : a.softmax ? expf(z[e] - zmax) / sum : 1.f / (1.f + expf(-z[e]));
    mass += a.renorm ? warp_sum(w) : 0.f;
  }
  for (int c = lane; c < a.top; c += 32) {
    const int e = sPick[c];
    float w = e < 0 ? 0.f : a.softmax ? expf(z[e] - zmax) / sum : 1.f / (1.f + expf(-z[e]));
    if (a.renorm && e >= 0) w = w / (mass + a.eps);
    a.weight[(size_t)t * a.top + c] = w * a.factor;
    a.sel[(size_t)t * a.top + c] = e < 0 ? -1 : e < a.n_real ? e : -2;
    if (sCount && e >= 0 && e < a.n_real) atomicAdd(&sCount[e], 1);    // only a number of slots: no order comes of it
  }
  __syncwarp();
}

// Puts the slots first .. first + n - 1 of one block in place.  sBase [E]: the place of the block's next slot of each expert; sWarp [warps][E].
__device__ __forceinline__ void place_slots(const RouterArgs& a, const int* sel, int first, int n, int* sBase, int* sWarp) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x, warps = threads >> 5;
  for (int at = 0; at < n; at += threads) {
    const int used = min(warps, (n - at + 31) >> 5);         // warps with slots in this round
    for (int i = threadIdx.x; i < used * a.n_real; i += threads) sWarp[i] = 0;
    __syncthreads();
    const int i = at + threadIdx.x;
    int e = i < n ? sel[first + i] : -1;
    if (e >= a.n_real) e = -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && before == 0) sWarp[warp * a.n_real + e] = __popc(same);
    __syncthreads();
    for (int x = threadIdx.x; x < a.n_real; x += threads) {
      int acc = sBase[x];
#pragma unroll 4
      for (int w = 0; w < used; ++w) {
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

__device__ __forceinline__ int tiles_of(const RouterArgs& a, int n) {
  return a.tile_shift >= 0 ? (n + a.tile_rows - 1) >> a.tile_shift : (n + a.tile_rows - 1) / a.tile_rows;
}

// From totals sTotal [n_real] by expert: places sFirst; `tiles`: writes the list of tiles too (sTile [n_real]).  By the whole block.
__device__ __forceinline__ void plan_experts(const RouterArgs& a, const int* sTotal, int* sFirst, int* sTile, bool tiles) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, per = (a.n_real + 31) / 32, lo = lane * per, hi = min(a.n_real, lo + per);
    int n = 0, nt = 0;
    for (int e = lo; e < hi; ++e) { n += sTotal[e]; nt += tiles_of(a, sTotal[e]); }
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
      sTile[e] = pt;
      pn += sTotal[e];
      pt += tiles_of(a, sTotal[e]);
    }
  }
  __syncthreads();
  if (tiles)
    for (int e = threadIdx.x; e < a.n_real; e += blockDim.x)
      for (int r = 0, t = sTile[e]; r < sTotal[e] && t < a.max_tiles; r += a.tile_rows, ++t) {
        a.tile_info[3 * t] = e;
        a.tile_info[3 * t + 1] = sFirst[e] + r;
        a.tile_info[3 * t + 2] = min(a.tile_rows, sTotal[e] - r);
      }
  __syncthreads();                 // the places move on below
}

// ONE: the whole step in this cluster, with its plan.  Shared memory: totals, places and tiles [E], by warp: doubles [E], picks [top]; the
// plan's [RP_WARPS][E] lie over the latter.
// A block has 16 warps; in two launches, where a lane has few experts, 32: the work is a chain of votes, and an SM wants more of them.
template <int VPT, bool ONE>
constexpr int route_threads() { return !ONE && VPT <= 8 ? 2 * RP_THREADS : RP_THREADS; }

template <int VPT, bool ONE>
__global__ void __launch_bounds__(route_threads<VPT, ONE>()) route_kernel(const __grid_constant__ RouterArgs a) {
  constexpr int THREADS = route_threads<VPT, ONE>(), WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint8_t rp_smem[];
  int* sCount = reinterpret_cast<int*>(rp_smem);
  int* sFirst = sCount + a.E;
  int* sTile = sFirst + a.E;
  double* sC = reinterpret_cast<double*>(rp_smem + ((size_t)12 * a.E + 15) / 16 * 16);
  int* sPick = reinterpret_cast<int*>(sC + (size_t)WARPS * a.E);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < a.E; e += THREADS) sCount[e] = 0;
  pdl_wait();
  pdl_trigger();
  const float* logits = after_wait(a.logits);
  __syncthreads();
  const int t0 = blockIdx.x * a.tokens_a_block, t1 = min(a.T, t0 + a.tokens_a_block);
  for (int t = t0 + warp; t < t1; t += WARPS)
    route_token<VPT>(a, logits, t, sC + (size_t)warp * a.E, sPick + warp * a.top, ONE ? nullptr : sCount, lane);
  if (ONE) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // all choices are written
    if (blockIdx.x != 0) return;
    const int* sel = after_wait(a.sel);
    for (int i = threadIdx.x; i < a.T * a.top; i += THREADS) {
      const int e = __ldcg(sel + i);
      if (e >= 0 && e < a.n_real) atomicAdd(&sCount[e], 1);
    }
    __syncthreads();
    plan_experts(a, sCount, sFirst, sTile, true);
    place_slots(a, sel, 0, a.T * a.top, sFirst, reinterpret_cast<int*>(sC));
  } else {
    __syncthreads();
    const int width = (a.n_real + 3) & ~3;
    for (int e = threadIdx.x; e < width; e += THREADS) a.counts[(size_t)blockIdx.x * width + e] = e < a.n_real ? sCount[e] : 0;
  }
}

__global__ void __launch_bounds__(PL_THREADS) plan_kernel(const __grid_constant__ RouterArgs a, int blocks) {
  extern __shared__ __align__(16) uint8_t rp_smem[];
  int* sTotal = reinterpret_cast<int*>(rp_smem);
  int* sBefore = sTotal + a.E;
  int* sFirst = sBefore + a.E;
  int* sTile = sFirst + a.E;
  int* sWarp = sTile + a.E;                      // [PL_WARPS][E]
  for (int e = threadIdx.x; e < a.n_real; e += PL_THREADS) sTotal[e] = sBefore[e] = 0;
  pdl_wait();
  pdl_trigger();
  const int* counts = after_wait(a.counts);
  __syncthreads();
  // totals, and what the blocks before this one hold: four experts a thread, every thread a part of the blocks, eight loads out at a time
  const int quads = (a.n_real + 3) >> 2, parts = max(1, PL_THREADS / quads);
  for (int x = threadIdx.x; x < parts * quads; x += PL_THREADS) {
    const int part = x / quads, e = 4 * (x - part * quads);
    const int4* p = reinterpret_cast<const int4*>(counts) + (e >> 2);
    int all[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
    for (int b0 = part; b0 < blocks; b0 += 8 * parts) {
      int4 c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = b0 + j * parts < blocks ? p[(size_t)(b0 + j * parts) * quads] : make_int4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool old = b0 + j * parts < (int)blockIdx.x;
        all[0] += c[j].x; all[1] += c[j].y; all[2] += c[j].z; all[3] += c[j].w;
        before[0] += old ? c[j].x : 0; before[1] += old ? c[j].y : 0; before[2] += old ? c[j].z : 0; before[3] += old ? c[j].w : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < a.n_real && all[i]) { atomicAdd(&sTotal[e + i], all[i]); atomicAdd(&sBefore[e + i], before[i]); }
  }
  __syncthreads();
  plan_experts(a, sTotal, sFirst, sTile, blockIdx.x == 0);
  for (int e = threadIdx.x; e < a.n_real; e += PL_THREADS) sFirst[e] += sBefore[e];
  __syncthreads();
  const int t0 = blockIdx.x * a.tokens_a_block, t1 = min(a.T, t0 + a.tokens_a_block);
  place_slots(a, after_wait(a.sel), t0 * a.top, (t1 - t0) * a.top, sFirst, sWarp);
}

// Few tokens: a warp a token in as few CTAs of one cluster as that takes.  Many: one block an SM, at least a token a warp.
static int tokens_a_block(int T) { return T <= RP_ONE_LAUNCH ? min(T, RP_WARPS) : max(RP_WARPS, (T + RP_MOST_BLOCKS - 1) / RP_MOST_BLOCKS); }

// How many whole numbers of scratch memory a step of T tokens wants.
MLXB_EXPORT int mlxb_moe_route_scratch(int T, int E) {
  if (T <= RP_ONE_LAUNCH || E <= 0) return 1;
  const int tpb = tokens_a_block(T);
  return (T + tpb - 1) / tpb * ((E + 3) & ~3);
}

template <int VPT>
static int route_launch(const RouterArgs& a, int blocks, cudaStream_t stream) {
  static SharedLimit one, many;
  const int warps = (a.T > RP_ONE_LAUNCH ? route_threads<VPT, false>() : RP_THREADS) / 32;
  const size_t smem = ((size_t)12 * a.E + 15) / 16 * 16 + (size_t)warps * (8 * (size_t)a.E + 4 * (size_t)a.top);
  constexpr size_t most = 227 * 1024;
  if (a.T > RP_ONE_LAUNCH) {
    if (cudaError_t e = many.raise(route_kernel<VPT, false>, most)) return mlxb_fail((int)e, "moe_route_plan: shared memory: %s", cudaGetErrorString(e));
    launch_pdl(route_kernel<VPT, false>, dim3(blocks), dim3(route_threads<VPT, false>()), smem, stream, a);
    return mlxb_check_launch("moe_route_plan");
  }
  if (cudaError_t e = one.raise(route_kernel<VPT, true>, most)) return mlxb_fail((int)e, "moe_route_plan: shared memory: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(RP_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = mlxb_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, route_kernel<VPT, true>, a);
  return mlxb_check_launch("moe_route_plan");
}

// Arguments as a record of 8-byte fields: a caller fills it in a tenth of the time of as many arguments.
struct RouteRecord {
  const float* logits;
  const int* token_req;
  const float* correction;
  int* sel;
  float* weight;
  int *counts, *sorted, *tile_info, *n_tiles;
  long long ldl, T, E, top, softmax, two, groups, keep, n_real, renorm, tile_rows, max_tiles;
  double eps, factor;
};

// logits float32 [T, E] at row stride ldl.  n_real: experts n_real .. E - 1 have no tensors (identity): chosen, they are marked -2 and the plan passes over them.
// sel, weight [T * top]; sorted [T * top]; tile_info [max_tiles][3]; n_tiles [1]; counts: mlxb_moe_route_scratch(T, E) whole numbers.
MLXB_EXPORT int mlxb_moe_route_plan(const RouteRecord* rec, long long bytes, cudaStream_t stream) {
  if (!rec || bytes != sizeof(RouteRecord)) return mlxb_fail(MLXB_BAD_ARG, "moe_route_plan: a record of %lld bytes", bytes);
  const RouteRecord& r = *rec;
  const long long T = r.T, E = r.E, top = r.top, groups = r.groups, keep = r.keep, n_real = r.n_real, tile_rows = r.tile_rows, max_tiles = r.max_tiles;
  const long long ldl = r.ldl;
  if (T == 0 && r.n_tiles) {
    const cudaError_t e = cudaMemsetAsync(r.n_tiles, 0, sizeof(int), stream);
    return e == cudaSuccess ? 0 : mlxb_fail((int)e, "moe_route_plan: %s", cudaGetErrorString(e));
  }
  if (!r.logits || !r.sel || !r.weight || !r.counts || ((uintptr_t)r.counts & 15) || !r.sorted || !r.tile_info || !r.n_tiles || max_tiles > 0x7fffffffLL || tile_rows > 0x7fffffffLL || T < 0 || E <= 0 || E > 1024 || top <= 0 || top > E || top > 64 || ldl < E || groups < 1 || groups > 128 || E % groups || keep < 1 || keep > groups ||
      n_real < 1 || n_real > E || top > keep * (E / groups) || tile_rows < 1 || (long long)T * top > 0x7ffffff0LL ||
      max_tiles < ((long long)T * top + tile_rows - 1) / tile_rows + n_real)
    return mlxb_fail(MLXB_BAD_ARG, "moe_route_plan: %lld tokens, %lld of %lld experts (%lld with tensors; up to 64 of 1024), %lld of %lld groups (up to 128), tiles of %lld rows, room for %lld",
                     T, top, E, n_real, keep, groups, tile_rows, max_tiles);
  int part = 0, shift = -1;
  for (int i = 0; i < 20; ++i)
    if (tile_rows == 1 << i) shift = i;
  if (groups <= 32)
    for (part = 1; 2 * part * groups <= 32; part *= 2) {}
  RouterArgs a = {r.logits, ldl, r.token_req, r.correction, (int)T, (int)E, (int)top, (int)r.softmax, (int)r.two, (int)groups, (int)keep, (int)n_real,
                  (int)r.renorm, part, (float)r.eps, (float)r.factor, r.sel, r.weight, r.counts, tokens_a_block((int)T), (int)tile_rows, shift,
                  (int)max_tiles, r.sorted, r.tile_info, r.n_tiles};
  const int blocks = ((int)T + a.tokens_a_block - 1) / a.tokens_a_block;
  int rc;
  if (E <= 32) rc = route_launch<1>(a, blocks, stream);
  else if (E <= 64) rc = route_launch<2>(a, blocks, stream);
  else if (E <= 128) rc = route_launch<4>(a, blocks, stream);
  else if (E <= 256) rc = route_launch<8>(a, blocks, stream);
  else if (E <= 512) rc = route_launch<16>(a, blocks, stream);
  else rc = route_launch<32>(a, blocks, stream);
  if (rc || T <= RP_ONE_LAUNCH) return rc;
  static SharedLimit limit;
  if (cudaError_t e = limit.raise(plan_kernel, 160 * 1024)) return mlxb_fail((int)e, "moe_route_plan: shared memory: %s", cudaGetErrorString(e));
  launch_pdl(plan_kernel, dim3(blocks), dim3(PL_THREADS), sizeof(int) * (4 + (size_t)PL_WARPS) * E, stream, a, blocks);
  return mlxb_check_launch("moe_route_plan (plan)");
}
