// Routing of tokens to experts (kq_moe_route): what fused_moe takes as topk_weights and topk_ids.
//
//   p = softmax(x) or sigmoid(x) over the experts;  c = p + bias, or without a bias the order of x itself
//   groups: a group counts its best expert (no bias) or the sum of its two best c (bias); only the top groups stay
//   ids = the top_k experts by c, descending, ties to the lowest index;  w = p[ids] (/ sum) * scale
//
// A warp per token; the experts' values sit in registers, expert i * 32 + lane in slot i of a lane.  Without a bias the choice
// compares the logits themselves and is exact.  With a bias it is made in fp64: two of a few hundred scores lie closer than fp32
// tells apart once in some thousand tokens, and a router's choice should not depend on the last bit of an exponential.
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
  float* weights; int32_t* ids;
};

constexpr double RT_OUT = -1e301;   // below every score: experts outside the chosen groups, or already taken
constexpr double RT_LOW = -1e300;   // a score of -infinity (a masked expert): after every finite one, before RT_OUT

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// NaN counts as -infinity and +infinity as the largest finite value, so that the probabilities of a row stay numbers
__device__ __forceinline__ float sane(float x) { return x != x ? -INFINITY : fminf(x, 3.4028234663852886e38f); }

template <typename T, int NV>
__global__ void __launch_bounds__(RT_WARPS * 32) route_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * RT_WARPS + (threadIdx.x >> 5);
  pdl_trigger();
  pdl_wait();
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.stride_t;
  float x[NV];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = i * 32 + lane;
    x[i] = e < p.experts ? sane(to_f32<T>(row[e])) : -INFINITY;
    top = fmaxf(top, x[i]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  top = fmaxf(top, -3.4028234663852886e38f);     // a row of masked experts only: probabilities of zero instead of NaN
  float sum = 0.f;
  if (!p.sigmoid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += expf(x[i] - top);
    sum = fmaxf(warp_sum(sum), 1.1754943508222875e-38f);
  }
  double c[NV];
  double wide = 0.;
  if (p.bias && !p.sigmoid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) wide += exp((double)x[i] - (double)top);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, d);
    wide = fmax(wide, 1e-300);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = i * 32 + lane;
    if (e >= p.experts) { c[i] = RT_OUT; continue; }
    double v = x[i];
    if (p.bias) v = (p.sigmoid ? 1. / (1. + exp(-(double)x[i])) : exp((double)x[i] - (double)top) / wide) + (double)sane(p.bias[e]);
    c[i] = v < RT_LOW ? RT_LOW : v;
  }
  if (p.groups > 1) {
    // lane g ends with the value of group g
    double value = RT_OUT;
    for (int g = 0; g < p.groups; ++g) {
      const int lo = g * p.group_size, hi = lo + p.group_size;
      double a = RT_OUT, b = RT_OUT;             // the two best of the lane's experts in this group
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = i * 32 + lane;
        if (e >= lo && e < hi) {
          if (c[i] > a) { b = a; a = c[i]; } else if (c[i] > b) b = c[i];
        }
      }
      const double best = warp_max(a);
      double s = best;
      if (p.bias && p.group_size > 1) {
        const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
        s += warp_max(lane == owner ? b : a);
      }
      if (lane == g) value = s < RT_LOW ? RT_LOW : s;
    }
    unsigned keep = 0;
    for (int n = 0; n < p.top_groups; ++n) {
      const double best = warp_max(value);
      const int g = __ffs(__ballot_sync(0xffffffffu, value == best)) - 1;
      keep |= 1u << g;
      if (lane == g) value = 2 * RT_OUT;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = i * 32 + lane;
      if (e < p.experts && !(keep >> (e / p.group_size) & 1)) c[i] = RT_OUT;
    }
  }
  int id = 0;                                    // of rank `lane`
  float w = 0.f;
  for (int n = 0; n < p.top_k; ++n) {
    double a = 2 * RT_OUT;
    int at = 0;
    float xv = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (c[i] > a) { a = c[i]; at = i * 32 + lane; xv = x[i]; }
    const double best = warp_max(a);
    const int e = (int)__reduce_min_sync(0xffffffffu, a == best ? (unsigned)at : 0xffffffffu);
    const float xe = __shfl_sync(0xffffffffu, xv, e & 31);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * 32 + lane == e) c[i] = 2 * RT_OUT;
    if (lane == n) {
      id = e;
      w = p.sigmoid ? 1.f / (1.f + expf(-xe)) : expf(xe - top) / sum;
    }
  }
  if (p.renormalize) w /= fmaxf(warp_sum(w), 1.1754943508222875e-38f);
  if (lane < p.top_k) {
    p.weights[t * p.top_k + lane] = w * p.scale;
    p.ids[t * p.top_k + lane] = id;
  }
}

template <typename T, int NV>
int run_route(const RouteParams& p, cudaStream_t st) {
  KQ_CUDA_TRY(launch_pdl(route_kernel<T, NV>, dim3((unsigned)((p.tokens + RT_WARPS - 1) / RT_WARPS)), dim3(RT_WARPS * 32), (size_t)0, st, options().pdl != 0, p));
  options().launches += 1;
  return KQ_OK;
}

template <typename T>
int run_route_size(const RouteParams& p, cudaStream_t st) {
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
  set_error("%s", "");
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
  if ((uintptr_t)logits % (dtype == KQ_F32 ? 4 : 2) || (uintptr_t)bias % 4) { set_error("%s: misaligned pointer", fn); return KQ_EINVAL; }
  RouteParams p;
  p.logits = logits; p.stride_t = stride_t; p.tokens = tokens; p.experts = (int)experts; p.top_k = (int)top_k; p.sigmoid = sigmoid != 0;
  p.groups = (int)groups; p.top_groups = (int)top_groups; p.group_size = (int)(experts / groups); p.renormalize = renormalize != 0;
  p.bias = bias; p.scale = scale; p.weights = weights; p.ids = ids;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case KQ_F32: return run_route_size<float>(p, st);
    case KQ_F16: return run_route_size<__half>(p, st);
    default: return run_route_size<__nv_bfloat16>(p, st);
  }
}
