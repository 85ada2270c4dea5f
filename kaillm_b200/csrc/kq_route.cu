// Routing of tokens to experts (kq_moe_route): what fused_moe takes as topk_weights and topk_ids.
//
//   p = softmax(x) or sigmoid(x) over the experts;  c = p + bias, or without a bias the order of x itself
//   groups: a group counts its best expert (no bias) or the sum of its two best c (bias); only the top groups stay
//   ids = the top_k experts by c, descending, ties to the lowest index;  w = p[ids] (/ sum) * scale
//
// A warp per token, NV experts next to each other per lane.  Without a bias the choice compares the logits themselves.  With one, two of
// a few hundred scores lie closer than fp32 tells apart once in some hundred tokens, and a router's choice should not depend on the
// last bit of an exponential: candidates whose scores come within RT_CLOSE of one another are ranked again in fp64, and so are the groups
// of a sigmoid that whole lanes make up; what else is open sends the whole token through fp64 (route_wide), which takes a warp 5 us: left to
// that, one such token among the last ones was felt in the time of the call (16384 x 256 in 8 groups 21.3 us, with groups_wide 17.4; 17.1 now).
//
// Bound by instructions, several hundred per token (886 for 16384 x 256 fp32 logits, 17 MB and 2.7 us of memory; 17.1 us): the best of 32 lanes
// is one redux.sync on order-preserving integers, and where whole lanes make up a group all groups are scored at once.  With up to 102, 64 and
// 51 registers for 16, 8 and fewer experts per lane, as below; left to the compiler 16384 x 256 takes 17.4 us, x 128 11.8 instead of 11.4.
#include "kq_common.cuh"

namespace kq {

namespace {

constexpr int RT_WARPS = 4;
constexpr int RT_MAX_EXPERTS = 1024, RT_MAX_TOP = 32, RT_MAX_GROUPS = 32;

struct RouteParams {
  const void* logits; int64_t stride_t;
  int64_t tokens;
  int experts, top_k, sigmoid, groups, top_groups, group_size, renormalize;
  const float* bias;
  float scale;
  int aligned, bias_aligned;  // rows, the bias start at 16-byte addresses
  float* weights; int32_t* ids;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// NaN counts as -infinity and +infinity as the largest finite value, so that the probabilities of a row stay numbers
__device__ __forceinline__ float sane(float x) { return fminf(fmaxf(x, -INFINITY), 3.4028234663852886e38f); }   // the larger of NaN and y is y

// fp64 scores as integers that compare as they do (both zeros alike); RT_TAKEN below all of them
constexpr unsigned long long RT_TAKEN = 0, RT_OUTSIDE = 1;      // taken; outside the chosen groups (no score maps to either)
__device__ __forceinline__ unsigned long long ordered64(double v) {
  const unsigned long long u = __double_as_longlong(v + 0.);
  return u ^ (u >> 63 ? 0xffffffffffffffffull : 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(unsigned long long k) {
  return __longlong_as_double(k ^ (k >> 63 ? 0x8000000000000000ull : 0xffffffffffffffffull));
}
__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (unsigned long long)hi << 32 | lo;
}

// A token whose choice the kernels below leave open (scores too close for fp32, too many ties): scores, groups and choice in fp64; NV
// experts next to each other per lane.
template <typename T, int NV>
__device__ __noinline__ void route_wide(const RouteParams& p, int64_t t) {
  const int lane = threadIdx.x & 31, e0 = lane * NV;
  const T* row = static_cast<const T*>(p.logits) + t * p.stride_t;
  float x[NV];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    x[i] = e0 + i < p.experts ? sane(to_f32<T>(row[e0 + i])) : -INFINITY;
    top = fmaxf(top, x[i]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  top = fmaxf(top, -3.4028234663852886e38f);
  double sum = 0.;
  double c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    c[i] = exp(p.sigmoid ? -(double)x[i] : (double)x[i] - (double)top);
    sum += c[i];
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  sum = fmax(sum, 1.1754943508222875e-38);
  unsigned long long key[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    key[i] = e0 + i >= p.experts ? RT_TAKEN
             : p.bias ? ordered64((p.sigmoid ? 1. / (1. + c[i]) : c[i] / sum) + (double)sane(p.bias[e0 + i])) : ordered64((double)x[i]);
  if (p.groups > 1) {
    unsigned long long mine = RT_TAKEN;          // score of group `lane`
    for (int g = 0; g < p.groups; ++g) {
      const int lo = g * p.group_size, hi = lo + p.group_size;
      unsigned long long a = RT_TAKEN, b = RT_TAKEN;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned long long k = e0 + i >= lo && e0 + i < hi ? key[i] : RT_TAKEN;
        if (k > a) { b = a; a = k; } else if (k > b) b = k;
      }
      const unsigned long long best = warp_max64(a);
      unsigned long long score = best;
      if (p.bias && p.group_size > 1) {
        const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
        score = ordered64(unordered64(best) + unordered64(warp_max64(lane == owner ? b : a)));
      }
      if (lane == g) mine = score;
    }
    unsigned kept = 0;
    for (int n = 0; n < p.top_groups; ++n) {
      const unsigned long long best = warp_max64(mine);
      const int g = __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1;
      kept |= 1u << g;
      if (lane == g) mine = RT_TAKEN;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e0 + i < p.experts && !(kept >> ((e0 + i) / p.group_size) & 1)) key[i] = RT_OUTSIDE;
  }
  int id = 0;                                    // of rank `lane`
  float chosen = 0.f;
  for (int n = 0; n < p.top_k; ++n) {
    unsigned long long a = key[0];
    int at = 0;
    float xv = x[0];
#pragma unroll
    for (int i = 1; i < NV; ++i)
      if (key[i] > a) { a = key[i]; at = i; xv = x[i]; }
    const unsigned long long best = warp_max64(a);
    const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
    const int e = __shfl_sync(0xffffffffu, e0 + at, owner);
    const float xe = __shfl_sync(0xffffffffu, xv, owner);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (e0 + i == e) key[i] = RT_TAKEN;
    if (lane == n) { id = e; chosen = xe; }
  }
  float w = 0.f;
  if (lane < p.top_k) w = p.sigmoid ? 1.f / (1.f + expf(-chosen)) : expf(chosen - top) / (float)sum;
  if (p.renormalize) w /= fmaxf(warp_sum(w), 1.1754943508222875e-38f);
  if (lane < p.top_k) {
    p.weights[t * p.top_k + lane] = w * p.scale;
    p.ids[t * p.top_k + lane] = id;
  }
}

// Which groups stay, in fp64, where `lanes` whole lanes (a power of two) make up a group: sigmoid with a bias.
template <typename T, int NV>
__device__ __forceinline__ uint32_t groups_wide(const RouteParams& p, int64_t t, int lanes) {
  const int lane = threadIdx.x & 31, e0 = lane * NV;
  const T* row = static_cast<const T*>(p.logits) + t * p.stride_t;
  unsigned long long a = RT_TAKEN, b = RT_TAKEN;                  // the two best of the lane, then of its group
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (e0 + i >= p.experts) break;
    const unsigned long long k = ordered64(1. / (1. + exp(-(double)sane(to_f32<T>(row[e0 + i])))) + (double)sane(p.bias[e0 + i]));
    if (k > a) { b = a; a = k; } else if (k > b) b = k;
  }
  for (int d = 1; d < lanes; d <<= 1) {
    const unsigned long long oa = __shfl_xor_sync(0xffffffffu, a, d), ob = __shfl_xor_sync(0xffffffffu, b, d);
    b = max(min(a, oa), max(b, ob));
    a = max(a, oa);
  }
  unsigned long long mine = p.group_size > 1 ? ordered64(unordered64(a) + unordered64(b)) : a;
  mine = __shfl_sync(0xffffffffu, mine, min(lane * lanes, 31));   // lane g takes group g's score
  int better = 0;
  for (int g = 0; g < p.groups; ++g) {
    const unsigned long long other = __shfl_sync(0xffffffffu, mine, g);
    better += other > mine || (other == mine && g < lane);
  }
  return __ballot_sync(0xffffffffu, lane < p.groups && better < p.top_groups);
}

__device__ __forceinline__ uint32_t ordered(float v) {      // compares as v does (both zeros alike)
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
// fp32 scores nearer than this (times the larger of 1 and their size) may be in the wrong order.  With u = 2^-24:
//   an exponential is off by (4 + 3 |x|) u of itself (x, times a rounded log2(e), 2^-22 of the instruction)
//   a sigmoid by p (1 - p) (4 + 3 |x|) u + 3 p u < 5 u, two of them by 10 u, the four of two groups by 20 u
//   the sum of a softmax by 17.5 u of itself in its terms (the mean of |x| with the weights p stays below 4.5 for 1024 experts) and 14 u
//   in its additions (7 in a lane's four partial sums, 2 to join them, 5 over the lanes): 31.5 u, which two scores have in common
//   the terms of two probabilities, or of the four of two groups, by (6 u + 3 |x| u) p each: 8.5 u for two, 10.5 u for four, as they
//   sum to 1 at most and p |x| stays below 0.37
//   a sum with the bias by u of its size: 2 u for two, 6 u with those of two groups
// so 48 u at most; 64 u are asked for.
constexpr float RT_CLOSE = 1.f / (1 << 18);
__device__ __forceinline__ bool close(float hi, float lo, float size = 1.f) { return !(hi - lo > RT_CLOSE * fmaxf(size, fabsf(hi))); }
// the scores of two groups' best are each rounded at their own size, which their sum may have lost
__device__ __forceinline__ float size_of(float a, float b) {
  const float size = fabsf(a) + fabsf(b);
  return size <= 3.4028234663852886e38f ? fmaxf(size, 1.f) : 1.f;
}
__device__ __forceinline__ float fast_exp(float x) {        // relative error 2^-22 + |x| 2^-24
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {        // relative error 2^-23; 0 from 2^126 on
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// what a candidate must reach so that none is missed whose fp64 score is above that of key `cut`
__device__ __forceinline__ uint32_t below_cut(const RouteParams& p, uint32_t cut) {
  if (cut == 0) return 1;
  const float c = unordered(cut);
  return p.bias ? max(1u, ordered(c - RT_CLOSE * fmaxf(1.f, fabsf(c)))) : cut;
}
// this lane's candidate's score in fp64
template <typename T>
__device__ __forceinline__ unsigned long long score64(const RouteParams& p, const T* row, int e, bool live, float top) {
  const double x = live ? (double)sane(to_f32<T>(row[e])) : 0., c = live ? (double)sane(p.bias[e]) : 0.;
  if (p.sigmoid) return live ? ordered64(1. / (1. + exp(-x)) + c) : RT_TAKEN;
  double sum = 0.;
  for (int i = threadIdx.x & 31; i < p.experts; i += 32) sum += exp((double)sane(to_f32<T>(row[i])) - (double)top);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return live ? ordered64(exp(x - (double)top) / fmax(sum, 1.1754943508222875e-38) + c) : RT_TAKEN;
}

// FULL: 32 x NV experts, in rows (and with a bias) that take vector loads
template <typename T, int NV, bool FULL>
__global__ void __launch_bounds__(RT_WARPS * 32, NV >= 32 ? 2 : NV == 16 ? 5 : NV == 8 ? 8 : 10) route_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * RT_WARPS + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.stride_t;
  const int e0 = lane * NV;
  __shared__ __align__(16) uint32_t s_key[RT_WARPS][36];
  __shared__ int s_id[RT_WARPS][32];
  float x[NV];
  constexpr int VEC = NV * (int)sizeof(T) >= 16 ? 16 / (int)sizeof(T) : NV;      // values of one load
  if (FULL || (p.aligned && (p.experts % NV == 0))) {
#pragma unroll
    for (int i = 0; i < NV; i += VEC) {
      alignas(16) T v[VEC];
      if (FULL || e0 < p.experts) {
        if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(row + e0 + i);
        else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(row + e0 + i);
        else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(row + e0 + i);
        else v[0] = row[e0];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i + j] = FULL || e0 < p.experts ? sane(to_f32<T>(v[j])) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = e0 + i < p.experts ? sane(to_f32<T>(row[e0 + i])) : -INFINITY;
  }
  float top = 0.f, sum = 1.f;
  if (!p.sigmoid) {
    top = x[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) top = fmaxf(top, x[i]);
    top = unordered(__reduce_max_sync(0xffffffffu, ordered(top)));
    top = fmaxf(top, -3.4028234663852886e38f);   // a row of masked experts only: probabilities of zero instead of NaN
    float part[NV < 4 ? NV : 4] = {};            // few additions in a row: RT_CLOSE counts on them
#pragma unroll
    for (int i = 0; i < NV; ++i) part[i % 4] += fast_exp(x[i] - top);
    if constexpr (NV >= 4) part[0] = (part[0] + part[1]) + (part[2] + part[3]);
    else if constexpr (NV == 2) part[0] += part[1];
    sum = fmaxf(warp_sum(part[0]), 1.1754943508222875e-38f);
  }
  // order-preserving keys of the scores; 0: no expert, or taken
  uint32_t key[NV];
  if (p.bias) {
    const float inv = p.sigmoid ? 1.f : 1.f / sum;
    float bias[NV];
    if (NV % 4 == 0 && (FULL || (p.bias_aligned && p.experts % NV == 0))) {
#pragma unroll
      for (int i = 0; i < NV; i += 4)
        if (FULL || e0 < p.experts) *reinterpret_cast<float4*>(bias + i) = *reinterpret_cast<const float4*>(p.bias + e0 + i);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) bias[i] = FULL || e0 + i < p.experts ? p.bias[e0 + i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float pr = p.sigmoid ? fast_rcp(1.f + fast_exp(-x[i])) : fast_exp(x[i] - top) * inv;
      key[i] = FULL || e0 + i < p.experts ? ordered(pr + sane(bias[i])) : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = FULL || e0 + i < p.experts ? ordered(x[i]) : 0u;
  }
  bool wide = false;                             // too close to call
  if (p.groups > 1) {
    uint32_t mine = 0;                           // lane's group's score, or in the general form that of group `lane`
    float size = 1.f;                            // of the two scores in it
    bool whole = p.group_size % NV == 0;         // whole lanes make up a group, a power of two of them
    const int lanes = p.group_size / NV;
    whole = whole && (lanes & (lanes - 1)) == 0;
    if (whole) {
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) { b = max(b, min(a, key[i])); a = max(a, key[i]); }
      for (int d = 1; d < lanes; d <<= 1) {
        const uint32_t oa = __shfl_xor_sync(0xffffffffu, a, d), ob = __shfl_xor_sync(0xffffffffu, b, d);
        b = max(min(a, oa), max(b, ob));
        a = max(a, oa);
      }
      mine = p.bias && p.group_size > 1 ? ordered(unordered(a) + unordered(b)) : a;
      size = size_of(unordered(a), unordered(b));
      if (!FULL && e0 >= p.experts) mine = 0;
    } else {
      for (int g = 0; g < p.groups; ++g) {
        const int lo = g * p.group_size, hi = lo + p.group_size;
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const uint32_t k = e0 + i >= lo && e0 + i < hi ? key[i] : 0u;
          b = max(b, min(a, k)); a = max(a, k);
        }
        const uint32_t best = __reduce_max_sync(0xffffffffu, a);
        uint32_t score = best;
        if (p.bias && p.group_size > 1) {
          const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
          const uint32_t second = __reduce_max_sync(0xffffffffu, lane == owner ? b : a);
          score = ordered(unordered(best) + unordered(second));
          if (lane == g) size = size_of(unordered(best), unordered(second));
        }
        if (lane == g) mine = score;
      }
    }
    // lane g takes group g's score and counts the better ones
    const int group_of_lane = whole ? lane >> (__ffs(lanes) - 1) : lane;
    const uint32_t own = mine;
    if (whole) mine = __shfl_sync(0xffffffffu, mine, min(lane * lanes, 31));
    if (lane >= p.groups) mine = 0;
    int better = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 4)     // lanes behind the groups count as 0
#pragma unroll
      for (int g = g0; g < g0 + 4; ++g) better += __shfl_sync(0xffffffffu, mine, g) >= mine + (g >= lane);
    const bool keep = lane < p.groups && better < p.top_groups;
    uint32_t kept = __ballot_sync(0xffffffffu, keep);
    if (p.bias && p.top_groups < p.groups) {     // the order of the kept ones does not matter
      const uint32_t last = __reduce_min_sync(0xffffffffu, keep ? mine : 0xffffffffu), next = __reduce_max_sync(0xffffffffu, keep ? 0u : mine);
      const uint32_t compared = own == last || own == next ? __float_as_uint(size) : 0u;       // lanes behind the groups have 0
      wide = close(unordered(last), unordered(next), __uint_as_float(__reduce_max_sync(0xffffffffu, compared)));
      if (wide && whole && p.sigmoid) {          // the same for all lanes
        kept = groups_wide<T, NV>(p, t, lanes);
        wide = false;
      }
    }
    if (whole) {
      if (!(kept >> group_of_lane & 1)) {
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (e0 + i < p.experts && !(kept >> ((e0 + i) / p.group_size) & 1)) key[i] = 0;
    }
  }
  // The (top_k + 1)-th of the lanes' best scores, or one shortly below it, bounds what can be chosen, or come next: usually a dozen experts,
  // which go to one lane each and are ranked by counting the better ones.  From 8 experts per lane on the bound is found by halving an
  // interval until top_k + 1 to + 3 lanes reach it (16384 x 256 22.7 -> 21.3 us); below, by taking the best lane top_k + 1 times (x 128 in
  // 11.8, by halving 13.3: all lanes take part, and the list grows).  More than 32 of them (many ties, top_k near 32): one by one.
  int id = 0, rank = 0x7fffffff;
  bool listed = false;
  if (p.top_k < 16) {
    uint32_t best = key[0], cut = 0;
#pragma unroll
    for (int i = 1; i < NV; ++i) best = max(best, key[i]);
    if (NV < 8) {
      for (int n = 0; n <= p.top_k; ++n) {
        cut = __reduce_max_sync(0xffffffffu, best);
        if (lane == __ffs(__ballot_sync(0xffffffffu, best == cut)) - 1) best = 0;
      }
    } else if (__popc(__ballot_sync(0xffffffffu, best != 0)) > p.top_k) {
      uint32_t hi = __reduce_max_sync(0xffffffffu, best);
      cut = __reduce_min_sync(0xffffffffu, best ? best : 0xffffffffu);     // more than top_k lanes reach it
      for (int n = 0; n < 8 && cut < hi; ++n) {
        const uint32_t mid = cut + ((hi - cut + 1) >> 1);
        const int reach = __popc(__ballot_sync(0xffffffffu, best >= mid));
        if (reach > p.top_k) {
          cut = mid;
          if (reach <= p.top_k + 2) break;
        } else {
          hi = mid - 1;
        }
      }
    }
    cut = below_cut(p, cut);
    int at = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const unsigned in = __ballot_sync(0xffffffffu, key[i] >= cut);
      at += __popc(in & ((1u << lane) - 1));
      total += __popc(in);
    }
    if (total <= 32) {
      uint32_t* keys = s_key[threadIdx.x >> 5];
      int* ids = s_id[threadIdx.x >> 5];
      keys[lane] = 0;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (key[i] >= cut) { keys[at] = key[i]; ids[at++] = e0 + i; }     // in the order of the experts
      __syncwarp();
      const uint32_t own = keys[lane];
      const int own_id = ids[lane];
      int better = 0;
      for (int j0 = 0; j0 < total; j0 += 4) {                             // keys behind the last one are 0
        const uint4 other = *reinterpret_cast<const uint4*>(keys + j0);
        better += other.x >= own + (j0 >= lane);
        better += other.y >= own + (j0 + 1 >= lane);
        better += other.z >= own + (j0 + 2 >= lane);
        better += other.w >= own + (j0 + 3 >= lane);
      }
      bool open = false;
      if (p.bias) {                                                       // is the next one too close?
        __syncwarp();
        if (lane < total) keys[better] = own;
        __syncwarp();
        open = better + 1 < total && better < p.top_k && close(unordered(own), unordered(keys[better + 1]));
        open = open && lane < total;
      }
      if (__any_sync(0xffffffffu, open)) {
        const unsigned long long mine = score64<T>(p, row, own_id, lane < total, top);
        better = 0;
#pragma unroll 4
        for (int j = 0; j < total; ++j) {
          const unsigned long long other = __shfl_sync(0xffffffffu, mine, j);
          better += other > mine || (other == mine && j < lane);
        }
      }
      if (lane < total && better < p.top_k) { id = own_id; rank = better; }
    }
    listed = total <= 32;
  }
  if (!listed) {
    uint32_t prev = 0;
    for (int n = 0; n <= p.top_k; ++n) {
      uint32_t a = key[0];
      int at = 0;
#pragma unroll
      for (int i = 1; i < NV; ++i)
        if (key[i] > a) { a = key[i]; at = i; }
      const uint32_t best = __reduce_max_sync(0xffffffffu, a);
      if (n > 0 && p.bias && best) wide |= close(unordered(prev), unordered(best));
      prev = best;
      if (n == p.top_k) break;
      const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
      const int e = __shfl_sync(0xffffffffu, e0 + at, owner);
      if (lane == owner) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (i == at) key[i] = 0;
      }
      if (lane == n) { id = e; rank = n; }
    }
  }
  if (__any_sync(0xffffffffu, wide)) { route_wide<T, NV>(p, t); return; }
  float w = 0.f;
  if (rank < p.top_k) {
    const float xv = sane(to_f32<T>(row[id]));
    w = p.sigmoid ? __fdividef(1.f, 1.f + expf(-xv)) : __fdividef(expf(xv - top), sum);
  }
  if (p.renormalize) w = __fdividef(w, fmaxf(warp_sum(w), 1.1754943508222875e-38f));
  if (rank < p.top_k) {
    p.weights[t * p.top_k + rank] = w * p.scale;
    p.ids[t * p.top_k + rank] = id;
  }
}

template <typename T, int NV>
int run_route(const RouteParams& p, cudaStream_t st) {
  const bool full = p.experts == 32 * NV && p.aligned && (!p.bias || p.bias_aligned);
  KQ_CUDA_TRY(launch_pdl(full ? route_kernel<T, NV, true> : route_kernel<T, NV, false>, dim3((unsigned)((p.tokens + RT_WARPS - 1) / RT_WARPS)), dim3(RT_WARPS * 32),
                         (size_t)0, st, options().pdl != 0, p));
  options().launches += 1;
  return KQ_OK;
}

template <typename T>
int run_route_size(const RouteParams& p, cudaStream_t st) {
  if (p.experts <= 32) return run_route<T, 1>(p, st);
  if (p.experts <= 64) return run_route<T, 2>(p, st);
  if (p.experts <= 128) return run_route<T, 4>(p, st);
  if (p.experts <= 256) return run_route<T, 8>(p, st);
  if (p.experts <= 512) return run_route<T, 16>(p, st);
  return run_route<T, 32>(p, st);
}

}  // namespace

}  // namespace kq

using namespace kq;

extern "C" int kq_moe_route(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t stride_t, int64_t top_k, int sigmoid,
                            const float* bias, int64_t groups, int64_t top_groups, int renormalize, float scale, float* weights,
                            int32_t* ids, void* stream) {
  const char* fn = "kq_moe_route";
  clear_error();
  if (dtype != KQ_F32 && dtype != KQ_F16 && dtype != KQ_BF16) { set_error("%s: unsupported dtype %d", fn, dtype); return KQ_EUNSUPPORTED; }
  if (tokens < 0 || experts <= 0 || top_k <= 0 || top_k > experts) { set_error("%s: top_k=%lld is not between 1 and experts=%lld", fn, (long long)top_k, (long long)experts); return KQ_EINVAL; }
  if (experts > RT_MAX_EXPERTS || top_k > RT_MAX_TOP || groups > RT_MAX_GROUPS || tokens > 0x7fffffff) {
    set_error("%s: at most %d experts, %d of them per token, %d groups", fn, RT_MAX_EXPERTS, RT_MAX_TOP, RT_MAX_GROUPS);
    return KQ_ELIMIT;
  }
  if (groups <= 0 || experts % groups || top_groups <= 0 || top_groups > groups) {
    set_error("%s: experts=%lld in %lld groups, %lld of them kept: not whole groups", fn, (long long)experts, (long long)groups, (long long)top_groups);
    return KQ_EINVAL;
  }
  if (experts / groups * top_groups < top_k) { set_error("%s: the kept groups hold fewer than top_k experts", fn); return KQ_EINVAL; }
  if (tokens == 0) return KQ_OK;
  if (!logits || !weights || !ids) { set_error("%s: null pointer", fn); return KQ_EINVAL; }
  if (tokens > 1 && stride_t < experts) { set_error("%s: rows of the logits overlap", fn); return KQ_EINVAL; }
  if ((uintptr_t)logits % (dtype == KQ_F32 ? 4 : 2) || ((uintptr_t)bias | (uintptr_t)weights | (uintptr_t)ids) % 4) { set_error("%s: misaligned pointer", fn); return KQ_EINVAL; }
  const void *w = weights, *e = ids;
  if (w == logits || e == logits || w == e || w == bias || e == bias) { set_error("%s: outputs must be neither inputs nor each other", fn); return KQ_EINVAL; }
  RouteParams p;
  p.logits = logits; p.stride_t = tokens > 1 ? stride_t : 0; p.tokens = tokens; p.experts = (int)experts; p.top_k = (int)top_k; p.sigmoid = sigmoid != 0;
  p.groups = (int)groups; p.top_groups = (int)top_groups; p.group_size = (int)(experts / groups); p.renormalize = renormalize != 0;
  p.bias = bias; p.scale = scale; p.bias_aligned = (uintptr_t)bias % 16 == 0; p.aligned = (uintptr_t)logits % 16 == 0 && p.stride_t * (dtype == KQ_F32 ? 4 : 2) % 16 == 0; p.weights = weights; p.ids = ids;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case KQ_F32: return run_route_size<float>(p, st);
    case KQ_F16: return run_route_size<__half>(p, st);
    default: return run_route_size<__nv_bfloat16>(p, st);
  }
}
