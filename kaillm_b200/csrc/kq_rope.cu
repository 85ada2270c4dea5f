// Norms of queries and keys per head and the position rotation in one pass, with the write into a paged cache
// (kq_qk_norm_rope).  For a head x of D values, weight w and rotated width r <= D:
//
//   y = x * rsqrt(mean(x^2) + eps) * w                                  (without a weight: y = x)
//   (y_a, y_b) -> factor * (y_a cos t - y_b sin t, y_b cos t + y_a sin t),  t = position * inv_freq[i],  i < r / 2
//   (a, b) = (i, i + r / 2), or (2i, 2i + 1) interleaved; values from r on are only normalised
//
// All of it in fp32 with one rounding at the end; the angle is the exact product, reduced to one turn in fp64 (position 10^6
// times a frequency near 1 would be off by 0.06 rad in fp32), and its cosine and sine are formed once per token.
#include "kq_common.cuh"

namespace kq {

namespace {

constexpr int RP_THREADS = 256;
constexpr int RP_MAX_DIM = 512;

struct RopeParams {
  const void* qkv; int64_t qkv_t;
  const void* positions; int pos64;
  const float* inv_freq;
  const void* qw; const void* kw; int w_f32;
  float eps, factor;
  int64_t tokens;
  int heads, kv_heads, dim, half, interleaved;
  void* q;                                           // [tokens][heads][dim]
  void* k; int64_t k_page, k_slot, k_head;           // cache, or (store = 0) the dense [tokens][kv_heads][dim]
  void* v; int64_t v_page, v_slot, v_head;
  const void* slots; int slot64;
  int64_t num_slots; int page_size;
  int store;
};

__device__ __forceinline__ int64_t index_at(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

template <typename T>
__device__ __forceinline__ float weight_at(const RopeParams& p, const void* w, int d) {
  return p.w_f32 ? static_cast<const float*>(w)[d] : to_f32<T>(static_cast<const T*>(w)[d]);
}

__device__ __forceinline__ float2 angle_of(const RopeParams& p, int64_t pos, int i) {
  const double t = (double)pos * (double)p.inv_freq[i];
  const double turns = rint(t * 0.15915494309189535);            // 1 / (2 pi)
  float s, c;
  sincosf((float)fma(-turns, 6.283185307179586, t), &s, &c);
  return make_float2(c * p.factor, s * p.factor);
}

// Where row `head` (of all q, k and v heads) of token t goes; null where it is not kept.
template <typename T>
__device__ __forceinline__ T* target_of(const RopeParams& p, int64_t t, int head) {
  if (head < p.heads) return static_cast<T*>(p.q) + (t * p.heads + head) * p.dim;
  const bool key = head < p.heads + p.kv_heads;
  const int h = head - p.heads - (key ? 0 : p.kv_heads);
  if (!p.store) return static_cast<T*>(p.k) + (t * p.kv_heads + h) * p.dim;
  const int64_t slot = index_at(p.slots, p.slot64, t);
  if (slot < 0 || slot >= p.num_slots) return nullptr;
  const int64_t page = slot / p.page_size, place = slot - page * p.page_size;
  return key ? static_cast<T*>(p.k) + page * p.k_page + place * p.k_slot + h * p.k_head
             : static_cast<T*>(p.v) + page * p.v_page + place * p.v_slot + h * p.v_head;
}

// One CTA per token: the angles once into shared memory, then a warp per head; any even width, any alignment.
template <typename T>
__global__ void __launch_bounds__(RP_THREADS) rope_any_kernel(const RopeParams p) {
  __shared__ float2 s_turn[RP_MAX_DIM / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const int64_t pos = index_at(p.positions, p.pos64, t);
  for (int i = threadIdx.x; i < p.half; i += RP_THREADS) s_turn[i] = angle_of(p, pos, i);
  __syncthreads();
  const int all = p.heads + (p.store ? 2 : 1) * p.kv_heads;
  for (int head = blockIdx.y * (RP_THREADS / 32) + warp; head < all; head += gridDim.y * (RP_THREADS / 32)) {
    const T* src = static_cast<const T*>(p.qkv) + t * p.qkv_t + (int64_t)head * p.dim;
    T* dst = target_of<T>(p, t, head);
    if (!dst) continue;
    if (head >= p.heads + p.kv_heads) {
      for (int d = lane; d < p.dim; d += 32) dst[d] = src[d];
      continue;
    }
    const void* w = head < p.heads ? p.qw : p.kw;
    float inv = 1.f;
    if (w) {
      float sum = 0.f;
      for (int d = lane; d < p.dim; d += 32) { const float x = to_f32<T>(src[d]); sum = fmaf(x, x, sum); }
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      inv = rsqrtf(sum / (float)p.dim + p.eps);
    }
    for (int i = lane; i < p.half; i += 32) {
      const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + p.half;
      float x = to_f32<T>(src[a]), y = to_f32<T>(src[b]);
      if (w) { x *= inv * weight_at<T>(p, w, a); y *= inv * weight_at<T>(p, w, b); }
      const float2 cs = s_turn[i];
      dst[a] = from_f32<T>(x * cs.x - y * cs.y);
      dst[b] = from_f32<T>(y * cs.x + x * cs.y);
    }
    for (int d = 2 * p.half + lane; d < p.dim; d += 32) {
      float x = to_f32<T>(src[d]);
      if (w) x *= inv * weight_at<T>(p, w, d);
      dst[d] = from_f32<T>(x);
    }
  }
}

template <typename T>
int run_rope(const RopeParams& p, cudaStream_t st) {
  const int all = p.heads + (p.store ? 2 : 1) * p.kv_heads;
  // few tokens: the heads of one token over several CTAs
  int64_t split = 1;
  while (p.tokens * split < 2 * sm_count() && split * (RP_THREADS / 32) < all) split *= 2;
  KQ_CUDA_TRY(launch_pdl(rope_any_kernel<T>, dim3((unsigned)p.tokens, (unsigned)split), dim3(RP_THREADS), (size_t)0, st, options().pdl != 0, p));
  options().launches += 1;
  return KQ_OK;
}

}  // namespace

}  // namespace kq

using namespace kq;

extern "C" int kq_qk_norm_rope(const void* qkv, int dtype, int64_t tokens, int64_t stride_t, int64_t heads, int64_t kv_heads,
                               int64_t head_dim, const void* positions, int positions64, const float* inv_freq, int64_t rotated,
                               int interleaved, float factor, const void* q_weight, const void* k_weight, int w_dtype, float eps,
                               void* q_out, void* k_out, const int64_t* k_strides, void* v_cache, const int64_t* v_strides,
                               const void* slots, int slots64, int64_t num_pages, int64_t page_size, void* stream) {
  const char* fn = "kq_qk_norm_rope";
  set_error("%s", "");
  if (dtype != KQ_F32 && dtype != KQ_F16 && dtype != KQ_BF16) { set_error("%s: unsupported dtype %d", fn, dtype); return KQ_EUNSUPPORTED; }
  if ((q_weight || k_weight) && w_dtype != KQ_F32 && w_dtype != dtype) { set_error("%s: norm weights must be float32 or of the activations' type", fn); return KQ_EUNSUPPORTED; }
  if (tokens < 0 || heads <= 0 || kv_heads <= 0) { set_error("%s: heads and kv_heads must be positive, tokens not negative", fn); return KQ_EINVAL; }
  if (head_dim < 2 || head_dim > RP_MAX_DIM || head_dim % 2) { set_error("%s: head_dim=%lld is not an even number up to %d", fn, (long long)head_dim, RP_MAX_DIM); return KQ_EUNSUPPORTED; }
  if (rotated < 0 || rotated > head_dim || rotated % 2) { set_error("%s: rotated=%lld is not an even number up to head_dim", fn, (long long)rotated); return KQ_EINVAL; }
  if (tokens > 0x7fffffff || heads > (1 << 16) || kv_heads > (1 << 16) || page_size > 0x7fffffff || num_pages > 0x7fffffff) { set_error("%s: size out of range", fn); return KQ_ELIMIT; }
  if (tokens == 0) return KQ_OK;
  if (tokens > 1 && stride_t < (heads + 2 * kv_heads) * head_dim) { set_error("%s: rows of qkv overlap", fn); return KQ_EINVAL; }
  const bool store = v_cache != nullptr;
  if (!qkv || !positions || (rotated && !inv_freq) || !q_out || !k_out || (store && (!k_strides || !v_strides || !slots))) { set_error("%s: null pointer", fn); return KQ_EINVAL; }
  if (store && (num_pages <= 0 || page_size <= 0)) { set_error("%s: the cache has no pages", fn); return KQ_EINVAL; }
  const uintptr_t size = dtype == KQ_F32 ? 4 : 2;
  if ((uintptr_t)qkv % size || (uintptr_t)q_out % size || (uintptr_t)k_out % size || (uintptr_t)v_cache % size || (uintptr_t)inv_freq % 4) { set_error("%s: misaligned pointer", fn); return KQ_EINVAL; }
  RopeParams p;
  p.qkv = qkv; p.qkv_t = stride_t; p.positions = positions; p.pos64 = positions64; p.inv_freq = inv_freq;
  p.qw = q_weight; p.kw = k_weight; p.w_f32 = w_dtype == KQ_F32; p.eps = eps; p.factor = factor; p.tokens = tokens;
  p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.dim = (int)head_dim; p.half = (int)(rotated / 2); p.interleaved = interleaved != 0;
  p.q = q_out; p.k = k_out; p.v = v_cache; p.slots = slots; p.slot64 = slots64; p.store = store;
  p.num_slots = store ? num_pages * page_size : 0; p.page_size = store ? (int)page_size : 1;
  p.k_page = store ? k_strides[0] : 0; p.k_slot = store ? k_strides[1] : 0; p.k_head = store ? k_strides[2] : 0;
  p.v_page = store ? v_strides[0] : 0; p.v_slot = store ? v_strides[1] : 0; p.v_head = store ? v_strides[2] : 0;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case KQ_F32: return run_rope<float>(p, st);
    case KQ_F16: return run_rope<__half>(p, st);
    default: return run_rope<__nv_bfloat16>(p, st);
  }
}
