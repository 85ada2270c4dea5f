// Norms of queries and keys per head and the position rotation in one pass, with the write into a paged cache
// (kq_qk_norm_rope).  For a head x of D values, weight w and rotated width r <= D:
//
//   y = x * rsqrt(mean(x^2) + eps) * w                                  (without a weight: y = x)
//   (y_a, y_b) -> factor * (y_a cos t - y_b sin t, y_b cos t + y_a sin t),  t = position * inv_freq[i],  i < r / 2
//   (a, b) = (i, i + r / 2), or (2i, 2i + 1) interleaved; values from r on are only normalised
//
// All of it in fp32 with one rounding at the end; the angle is the product in fp64 (exact below position 2^29), reduced there to one turn
// (position 10^6 times a frequency near 1 would be off by 0.06 rad in fp32), and its cosine and sine are formed once per token, in fp32.
#include <type_traits>

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
  float eps, factor, inv_dim;
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

// Rows of pieces of 16 bytes, or 8 where the rotated width or an address asks for it.  A lane owns two pieces A and B of a head, half the rotated width apart (behind the rotated part, half of what is
// left), so that the values of a pair stand at the same place of A and B, or interleaved next to each other in one of them; D / 2V lanes
// share a head (V values per piece), rounded up to a power of two for the sum of squares, and the other lanes take further heads.  So nothing
// but that sum crosses lanes, and out_A = A * c0 + A' * c1, out_B = B * c2 + B' * c3 (A', B': the partners) with factors made of the
// norm's weight and the token's cosine and sine, which a lane forms once for all heads of a kind and token and keeps in registers.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float x, float y) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 unpack2(f32x2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 swap2(f32x2 v) { const float2 u = unpack2(v); return pack2(u.y, u.x); }

template <typename T, typename Piece> __device__ __forceinline__ f32x2 widen(const Piece& v, int i) {   // values 2i, 2i + 1 of a piece
  const T* e = reinterpret_cast<const T*>(&v);
  return pack2(to_f32<T>(e[2 * i]), to_f32<T>(e[2 * i + 1]));
}
template <typename T, typename Piece> __device__ __forceinline__ void narrow(Piece& v, int i, f32x2 x) {
  const float2 u = unpack2(x);
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float2*>(&v)[i] = u;
  } else if constexpr (std::is_same<T, __half>::value) {
    reinterpret_cast<__half2*>(&v)[i] = __floats2half2_rn(u.x, u.y);
  } else {
    reinterpret_cast<__nv_bfloat162*>(&v)[i] = __floats2bfloat162_rn(u.x, u.y);
  }
}

// The values of a norm weight for a piece from d on (without a weight: ones)
template <typename T, typename Piece, int V>
__device__ __forceinline__ void weights_of(const RopeParams& p, const void* w, int d, float (&out)[V]) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = 1.f;
  } else if (p.w_f32) {
    constexpr int N = sizeof(Piece) / 4;
#pragma unroll
    for (int e = 0; e < V; e += N) {
      const Piece f = *reinterpret_cast<const Piece*>(static_cast<const float*>(w) + d + e);
#pragma unroll
      for (int i = 0; i < N; ++i) out[e + i] = reinterpret_cast<const float*>(&f)[i];
    }
  } else {
    const Piece u = *reinterpret_cast<const Piece*>(static_cast<const T*>(w) + d);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = to_f32<T>(reinterpret_cast<const T*>(&u)[e]);
  }
}

enum RopeForm { HALVES, NEIGHBOURS, MIXED };   // all values turn, in pairs half a head apart; all, interleaved; some do not

// A lane's pieces of a head and what they are multiplied by.  Only MIXED has lanes that differ, and choose their partners; it covers the others.
template <typename T, RopeForm FORM, typename Piece> struct RopeLane {
  static constexpr int V = (int)(sizeof(Piece) / sizeof(T)), P = V / 2;                        // values, pairs of them in a piece
  int log2;                                                                       // of the lanes of a head
  bool active, turned, apart;
  int da, db;                                                                     // first values of the pieces
  f32x2 c0[P], c1[P], c2[P], c3[P];

  __device__ __forceinline__ RopeLane(const RopeParams& p, int lanes_log2) : log2(lanes_log2) {
    const int unit = threadIdx.x & ((1 << log2) - 1);
    active = unit * 2 * V < p.dim;
    turned = FORM != MIXED || unit * V < p.half;
    apart = FORM == HALVES || (FORM == MIXED && turned && !p.interleaved);
    da = turned ? unit * V : p.half + unit * V;                                   // 2 half + (unit V - half)
    db = turned ? p.half + unit * V : p.dim / 2 + unit * V;                       // and (dim - 2 half) / 2 behind
  }
  __device__ __forceinline__ int head_of_step() const { return (threadIdx.x & 31) >> log2; }

  __device__ __forceinline__ void factors(const RopeParams& p, const void* w, const float2* s_turn) {
    float wa[V], wb[V];
    weights_of<T, Piece>(p, active ? w : nullptr, da, wa);
    weights_of<T, Piece>(p, active ? w : nullptr, db, wb);
    const bool on = turned && active;
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      if (FORM != NEIGHBOURS && (apart || !turned)) {
        const float2 u = on ? s_turn[da + e] : make_float2(1.f, 0.f), v = on ? s_turn[da + e + 1] : make_float2(1.f, 0.f);
        c0[e / 2] = pack2(wa[e] * u.x, wa[e + 1] * v.x); c1[e / 2] = pack2(-wb[e] * u.y, -wb[e + 1] * v.y);
        c2[e / 2] = pack2(wb[e] * u.x, wb[e + 1] * v.x); c3[e / 2] = pack2(wa[e] * u.y, wa[e + 1] * v.y);
      } else {
        const float2 u = on ? s_turn[(da + e) / 2] : make_float2(1.f, 0.f), v = on ? s_turn[(db + e) / 2] : make_float2(1.f, 0.f);
        c0[e / 2] = pack2(wa[e] * u.x, wa[e + 1] * u.x); c1[e / 2] = pack2(-wa[e + 1] * u.y, wa[e] * u.y);
        c2[e / 2] = pack2(wb[e] * v.x, wb[e + 1] * v.x); c3[e / 2] = pack2(-wb[e + 1] * v.y, wb[e] * v.y);
      }
    }
  }
  // all lanes of the warp together; a lane without a head has zeros
  __device__ __forceinline__ void turn(const RopeParams& p, Piece& ra, Piece& rb, bool normed) const {
    f32x2 x[P], y[P];
#pragma unroll
    for (int e = 0; e < P; ++e) { x[e] = widen<T, Piece>(ra, e); y[e] = widen<T, Piece>(rb, e); }
    f32x2 inv = 0;
    if (normed) {
      f32x2 sq = mul2(x[0], x[0]);
#pragma unroll
      for (int e = 0; e < P; ++e) sq = fma2(y[e], y[e], e ? fma2(x[e], x[e], sq) : sq);
      float sum = unpack2(sq).x + unpack2(sq).y;
      for (int m = 1 << log2 >> 1; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      const float f = rsqrtf(fmaf(sum, p.inv_dim, p.eps));
      inv = pack2(f, f);
    }
#pragma unroll
    for (int e = 0; e < P; ++e) {
      // behind the rotated part the partner counts with 0, also where it is no number
      const f32x2 px = apart ? y[e] : turned ? swap2(x[e]) : 0, py = apart ? x[e] : turned ? swap2(y[e]) : 0;
      f32x2 u = fma2(px, c1[e], mul2(x[e], c0[e])), v = fma2(py, c3[e], mul2(y[e], c2[e]));
      if (normed) { u = mul2(u, inv); v = mul2(v, inv); }
      narrow<T, Piece>(ra, e, u);
      narrow<T, Piece>(rb, e, v);
    }
  }
  __device__ __forceinline__ void put(T* dst, const Piece& ra, const Piece& rb) const {
    *reinterpret_cast<Piece*>(dst + da) = ra;
    *reinterpret_cast<Piece*>(dst + db) = rb;
  }
};

// Where keys and values of token t go; false: nowhere.  Their first head; k_head: from head to head of the keys.
template <typename T>
__device__ __forceinline__ bool rows_of(const RopeParams& p, int64_t t, T** k, T** v, int64_t* k_head) {
  *k = static_cast<T*>(p.k) + t * p.kv_heads * p.dim;
  *v = nullptr;
  *k_head = p.dim;
  if (!p.store) return true;
  const int64_t slot = index_at(p.slots, p.slot64, t);
  if (slot < 0 || slot >= p.num_slots) return false;
  const int64_t page = slot >> 31 ? slot / p.page_size : (int64_t)((uint32_t)slot / (uint32_t)p.page_size), place = slot - page * p.page_size;
  *k = static_cast<T*>(p.k) + page * p.k_page + place * p.k_slot;
  *v = static_cast<T*>(p.v) + page * p.v_page + place * p.v_slot;
  *k_head = p.k_head;
  return true;
}

// A CTA per token, or with SPREAD three (queries, keys and values: blockIdx.z); its warps share the token's steps (a step: as many heads as a
// warp holds).  The first rows of all kinds are on their way while the angles are formed.
template <typename T, int WARPS, int AHEAD, RopeForm FORM, bool SPREAD, typename Piece>
__global__ void __launch_bounds__(WARPS * 32, SPREAD ? 4 : 16 / WARPS) rope_rows_kernel(const RopeParams p, int lanes_log2) {
  __shared__ float2 s_turn[RP_MAX_DIM / 2];
  RopeLane<T, FORM, Piece> L(p, lanes_log2);
  const int warp = threadIdx.x >> 5, sub = L.head_of_step();
  const int64_t t = blockIdx.x;
  const bool q_here = !SPREAD || blockIdx.z == 0, k_here = !SPREAD || blockIdx.z == 1, v_here = p.store && (!SPREAD || blockIdx.z == 2);
  const int per = 32 >> lanes_log2, step = gridDim.y * WARPS * per;               // heads of a step, from step to step of this warp
  const int h0 = (blockIdx.y * WARPS + warp) * per + sub;
  pdl_trigger();
  pdl_wait();
  const T* src = static_cast<const T*>(p.qkv) + t * p.qkv_t + h0 * p.dim;
  auto load = [&](const T* from, bool on, Piece& va, Piece& vb) {
    va = vb = Piece{};
    if (on) { va = *reinterpret_cast<const Piece*>(from + L.da); vb = *reinterpret_cast<const Piece*>(from + L.db); }
  };
  Piece a[AHEAD], b[AHEAD], ka, kb, va, vb;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(src + i * step * p.dim, q_here && L.active && h0 + i * step < p.heads, a[i], b[i]);
  const T* k_src = src + p.heads * p.dim;
  const T* v_src = k_src + p.kv_heads * p.dim;
  load(k_src, k_here && L.active && h0 < p.kv_heads, ka, kb);
  load(v_src, v_here && L.active && h0 < p.kv_heads, va, vb);

  const int64_t pos = index_at(p.positions, p.pos64, t);
  for (int i = threadIdx.x; i < p.half; i += WARPS * 32) s_turn[i] = angle_of(p, pos, i);
  T *k_dst, *v_dst;
  int64_t k_head;
  const bool kept = L.active && rows_of<T>(p, t, &k_dst, &v_dst, &k_head);
  __syncthreads();

  if (v_here) {                                                   // values go as they came
    for (int h = h0; h - sub < p.kv_heads; h += step) {
      if (kept && h < p.kv_heads) L.put(v_dst + h * p.v_head, va, vb);
      v_src += step * p.dim;
      load(v_src, L.active && h + step < p.kv_heads, va, vb);
    }
  }
  L.factors(p, q_here ? p.qw : p.kw, s_turn);
  T* dst = static_cast<T*>(p.q) + (t * p.heads + h0) * p.dim;
  src += AHEAD * step * p.dim;
  for (int h = h0; q_here && h - sub < p.heads; h += AHEAD * step) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int hi = h + i * step;
      if (hi - sub >= p.heads) break;
      Piece ra = a[i], rb = b[i];
      load(src, L.active && hi + AHEAD * step < p.heads, a[i], b[i]);
      src += step * p.dim;
      L.turn(p, ra, rb, p.qw != nullptr);
      if (L.active && hi < p.heads) L.put(dst, ra, rb);
      dst += step * p.dim;
    }
  }
  if (!k_here || h0 - sub >= p.kv_heads) return;
  if (!SPREAD && p.kw != p.qw) L.factors(p, p.kw, s_turn);
  for (int h = h0; h - sub < p.kv_heads; h += step) {
    Piece ra = ka, rb = kb;
    k_src += step * p.dim;
    load(k_src, L.active && h + step < p.kv_heads, ka, kb);
    L.turn(p, ra, rb, p.kw != nullptr);
    if (kept && h < p.kv_heads) L.put(k_dst + h * k_head, ra, rb);
  }
}

// a piece, or with live = false a piece of zeros and no read
__device__ __forceinline__ void copy_piece(uint4* dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_piece(uint2* dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(live ? 8 : 0) : "memory");
}

// Many tokens: a warp per token walks its values, queries and keys through a ring in shared memory, two steps in use and the others under
// way.  A lane copies the pieces that it reads back itself, so nothing but its own copies is waited for.
// Bound by memory: 8192 tokens with 40 + 2 x 8 heads of 128, norms and cache, bf16 (235 MB) 41.5 us, 5.7 TB/s; interleaved 40.9; fp32 78. Two warps
// per token with their next rows in registers (rope_rows_kernel) took 49.6, 52 and 84: as much on the way as registers hold, at 16 warps per
// multiprocessor.  Steps of the ring and least warps of a multiprocessor: 16-bit 6 and 18 (41.5; 8 and 18 43.2, 5 and 20 41.8, 6 and 16
// 44.9), fp32 10 and 16 (4096 tokens 42.4; 6 and 18 46.9), whose heads take twice the steps.
template <typename T> constexpr int RING_WARPS = sizeof(T) == 4 ? 16 : 18;
template <typename T, RopeForm FORM, typename Piece>
__global__ void __launch_bounds__(32, RING_WARPS<T>) rope_ring_kernel(const RopeParams p, int lanes_log2) {
  constexpr int RING_STEPS = sizeof(T) == 4 ? 10 : 6;
  __shared__ float2 s_turn[RP_MAX_DIM / 2];
  __shared__ Piece s_ring[RING_STEPS][2][32];
  RopeLane<T, FORM, Piece> L(p, lanes_log2);
  const int lane = threadIdx.x, h0 = L.head_of_step();
  const int64_t t = blockIdx.x;
  const int per = 32 >> lanes_log2, nq = (p.heads + per - 1) >> (5 - lanes_log2), nk = (p.kv_heads + per - 1) >> (5 - lanes_log2), nv = p.store ? nk : 0;
  pdl_trigger();
  pdl_wait();
  const T* src = static_cast<const T*>(p.qkv) + t * p.qkv_t;
  int into = 0, from = 0, next = RING_STEPS - 2;                                  // places in the ring; the step to be fetched
  auto fetch = [&](int s) {
    if (s < nv + nq + nk) {
      const bool is_v = s < nv, is_q = !is_v && s < nv + nq;
      const int h = h0 + (is_v ? s : is_q ? s - nv : s - nv - nq) * per;
      const bool on = L.active && h < (is_q ? p.heads : p.kv_heads);
      const T* row = src + (on ? (h + (is_q ? 0 : is_v ? p.heads + p.kv_heads : p.heads)) * p.dim : 0);
      copy_piece(&s_ring[into][0][lane], row + (on ? L.da : 0), on);
      copy_piece(&s_ring[into][1][lane], row + (on ? L.db : 0), on);
    }
    into = into + 1 == RING_STEPS ? 0 : into + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < RING_STEPS - 2; ++s) fetch(s);
  auto take = [&](Piece& ra, Piece& rb) {
    asm volatile("cp.async.wait_group %0;" ::"n"(RING_STEPS - 3) : "memory");
    ra = s_ring[from][0][lane];
    rb = s_ring[from][1][lane];
    from = from + 1 == RING_STEPS ? 0 : from + 1;
    fetch(next++);                                                                // into the place of the step before the last one
  };

  const int64_t pos = index_at(p.positions, p.pos64, t);
  for (int i = lane; i < p.half; i += 32) s_turn[i] = angle_of(p, pos, i);
  T *k_dst, *v_dst;
  int64_t k_head;
  const bool kept = L.active && rows_of<T>(p, t, &k_dst, &v_dst, &k_head);
  Piece ra, rb, sa, sb;
  for (int i = 0, h = h0; i < nv; ++i, h += per) {
    take(ra, rb);
    if (kept && h < p.kv_heads) L.put(v_dst + h * p.v_head, ra, rb);
  }
  __syncwarp();
  // two steps at a time, so that one's sum over the lanes overlaps with the other's
  auto turn_all = [&](int steps, int heads, bool normed, T* dst, int64_t to_head, bool on) {
    int i = 0, h = h0;
    for (; i + 2 <= steps; i += 2, h += 2 * per) {
      take(ra, rb);
      take(sa, sb);
      L.turn(p, ra, rb, normed);
      if (on && h < heads) L.put(dst + h * to_head, ra, rb);
      L.turn(p, sa, sb, normed);
      if (on && h + per < heads) L.put(dst + (h + per) * to_head, sa, sb);
    }
    if (i < steps) {
      take(ra, rb);
      L.turn(p, ra, rb, normed);
      if (on && h < heads) L.put(dst + h * to_head, ra, rb);
    }
  };
  L.factors(p, p.qw, s_turn);
  turn_all(nq, p.heads, p.qw != nullptr, static_cast<T*>(p.q) + t * p.heads * p.dim, p.dim, L.active);
  if (p.kw != p.qw) L.factors(p, p.kw, s_turn);
  turn_all(nk, p.kv_heads, p.kw != nullptr, k_dst, k_head, kept);
}

// Any even width, any alignment: one CTA per token (or part of its heads), a warp per head, the angles once into shared memory.
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

// every row, piece pair and target made of pieces at their own alignment
template <typename T, typename Piece>
bool in_pieces(const RopeParams& p) {
  constexpr int V = (int)(sizeof(Piece) / sizeof(T));
  const int64_t strides = p.qkv_t | p.k_page | p.k_slot | p.k_head | p.v_page | p.v_slot | p.v_head;   // zeros where there is no cache
  const uintptr_t at = (uintptr_t)p.qkv | (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.qw | (uintptr_t)p.kw;
  return p.dim % (2 * V) == 0 && p.half % V == 0 && p.dim <= 64 * V && strides % V == 0 && at % sizeof(Piece) == 0;
}

template <typename T, RopeForm FORM, typename Piece>
int run_rows(const RopeParams& p, cudaStream_t st) {
  int log2 = 0;
  while ((1 << log2) * 2 * (int)(sizeof(Piece) / sizeof(T)) < p.dim) ++log2;
  const bool pdl = options().pdl != 0;
  // (pieces of 8 bytes: few, and the ring.)  Few tokens, more than a few, more than a wave of ring_kernel's warps; with 40 + 2 x 8 heads of 128, us: 16 tokens 2.9 spread; 600 7.0 by two warps
  // each, 16 spread, 9.0 by the ring; 2000 16.6, 54.7, 16.0; 5000 33.5, 132, 28.8.  Where the spread form and two warps cross is not measured: at
  // 600 the spread one is behind already, so some hundred tokens below the switch run slower than they could
  if (p.tokens >= (sizeof(Piece) == 16 ? 20 : 4) * sm_count()) {
    KQ_CUDA_TRY(launch_pdl(rope_ring_kernel<T, FORM, Piece>, dim3((unsigned)p.tokens), dim3(32), (size_t)0, st, pdl, p, log2));
  } else if (sizeof(Piece) == 16 && p.tokens >= 4 * sm_count()) {
    // two warps walk a token's heads
    if constexpr (sizeof(Piece) == 16)
      KQ_CUDA_TRY(launch_pdl(rope_rows_kernel<T, 2, 2, FORM, false, Piece>, dim3((unsigned)p.tokens), dim3(64), (size_t)0, st, pdl, p, log2));
  } else {
    // few: a step per warp, queries, keys and values apart, spread over the multiprocessors
    const int steps = ((p.heads > p.kv_heads ? p.heads : p.kv_heads) + (32 >> log2) - 1) >> (5 - log2);
    const dim3 grid((unsigned)p.tokens, (unsigned)((steps + 3) / 4), p.store ? 3 : 2);
    KQ_CUDA_TRY(launch_pdl(rope_rows_kernel<T, 4, 1, FORM, true, Piece>, grid, dim3(128), (size_t)0, st, pdl, p, log2));
  }
  options().launches += 1;
  return KQ_OK;
}

template <typename T>
int run_rope(const RopeParams& p, cudaStream_t st) {
  if (in_pieces<T, uint4>(p))
    return 2 * p.half < p.dim ? run_rows<T, MIXED, uint4>(p, st) : p.interleaved ? run_rows<T, NEIGHBOURS, uint4>(p, st) : run_rows<T, HALVES, uint4>(p, st);
  // heads of 80 of which 40 turn, 16-bit, us, by rope_any_kernel / in pieces of 8 bytes: one token 3.4 / 2.7, 1500 tokens with 56 heads 31.8 / 21.0,
  // 3317 with 73 heads 86.6 / 36.9 (issue: 10 of 16 lanes, half the values per instruction)
  if (in_pieces<T, uint2>(p)) return run_rows<T, MIXED, uint2>(p, st);
  const int all = p.heads + (p.store ? 2 : 1) * p.kv_heads;
  const bool pdl = options().pdl != 0;
  // few tokens: the heads of one token over several CTAs
  int64_t split = 1;
  while (p.tokens * split < 2 * sm_count() && split * (RP_THREADS / 32) < all) split *= 2;
  KQ_CUDA_TRY(launch_pdl(rope_any_kernel<T>, dim3((unsigned)p.tokens, (unsigned)split), dim3(RP_THREADS), (size_t)0, st, pdl, p));
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
  clear_error();
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
  if ((uintptr_t)qkv % size || (uintptr_t)q_out % size || (uintptr_t)k_out % size || (uintptr_t)v_cache % size || (uintptr_t)inv_freq % 4 ||
      (uintptr_t)positions % (positions64 ? 8 : 4) || (store && (uintptr_t)slots % (slots64 ? 8 : 4)) || ((uintptr_t)q_weight | (uintptr_t)k_weight) % (w_dtype == KQ_F32 ? 4 : 2)) {
    set_error("%s: misaligned pointer", fn);
    return KQ_EINVAL;
  }
  if (q_out == qkv || k_out == qkv || v_cache == qkv || k_out == q_out || v_cache == k_out || v_cache == q_out) {
    set_error("%s: outputs must be neither inputs nor each other", fn);
    return KQ_EINVAL;
  }
  RopeParams p;
  p.qkv = qkv; p.qkv_t = tokens > 1 ? stride_t : 0; p.positions = positions; p.pos64 = positions64; p.inv_freq = inv_freq;
  p.qw = q_weight; p.kw = k_weight; p.w_f32 = w_dtype == KQ_F32; p.eps = eps; p.factor = factor; p.inv_dim = 1.f / (float)head_dim; p.tokens = tokens;
  p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.dim = (int)head_dim; p.half = (int)(rotated / 2); p.interleaved = interleaved != 0;
  p.q = q_out; p.k = k_out; p.v = v_cache; p.slots = slots; p.slot64 = slots64; p.store = store;
  p.num_slots = store ? num_pages * page_size : 0; p.page_size = store ? (int)page_size : 1;
  // a stride that no step follows may be anything
  p.k_page = store && num_pages > 1 ? k_strides[0] : 0; p.k_slot = store && page_size > 1 ? k_strides[1] : 0; p.k_head = store && kv_heads > 1 ? k_strides[2] : 0;
  p.v_page = store && num_pages > 1 ? v_strides[0] : 0; p.v_slot = store && page_size > 1 ? v_strides[1] : 0; p.v_head = store && kv_heads > 1 ? v_strides[2] : 0;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case KQ_F32: return run_rope<float>(p, st);
    case KQ_F16: return run_rope<__half>(p, st);
    default: return run_rope<__nv_bfloat16>(p, st);
  }
}
