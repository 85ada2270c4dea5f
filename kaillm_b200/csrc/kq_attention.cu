// Attention of one new token per sequence over a paged key-value cache (kq_paged_attention).
//
//   s_j = f(scale * q . k_j),  f(x) = x or cap * tanh(x / cap),  j in [max(0, len - window), len)
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j;  a sequence without visible keys gives zeros
//
// One pass over the cache: a warp keeps the running maximum, the running sum and the weighted values of the query heads that
// share a key head (their rows are one tile) in registers, in fp32, and rescales them when a new maximum comes.
//
// The work is cut by cached keys, not by sequences: an item is (sequence, key head, row tile) and has one unit of work per
// tile of keys, behind AT_START units for its beginning and end; the units of all items, in order, are divided evenly over the
// CTAs of one wave.  A CTA finds its share from the lengths themselves (a sum and a scan, the lengths stay on the GPU), so a batch of any mix of lengths is balanced and a
// captured call follows the lengths of each replay.  An item inside one CTA is finished there; one that crosses CTAs leaves
// partial results (unnormalised values, maximum, sum) that attend_join_kernel adds in the order of the keys: no atomics, the
// same bits every time.
#include <type_traits>

#include "kq_common.cuh"

namespace kq {

namespace {

constexpr int AT_MAX_CTAS = 2;         // per multiprocessor
constexpr int AT_WARPS = 4;            // warps of a CTA: each walks every fourth tile of keys of the CTA's share on its own
// An item costs as much as so many tiles beside its own (loading q, filling the ring, joining the warps).  Without it the CTAs
// that get the short sequences of a mixed batch end last: 64 sequences of 0..4k tokens, busy cycles of the slowest SM 290k
// against 197k of the fastest.
constexpr int AT_START = 8;
constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr float AT_LN2 = 0.6931471805599453f;

struct AttnParams {
  const void* q; int64_t q_b, q_h;                     // strides in elements; the head dimension is dense everywhere
  const void* k; int64_t k_page, k_slot, k_head;
  const void* v; int64_t v_page, v_slot, v_head;
  const int32_t* table; int64_t table_b; int width;    // page names [batch][width]
  const int32_t* lens;
  int batch, heads, kv_heads, group, dim, page_size;
  int64_t num_pages;
  int row_tiles, rows;                                 // query heads of one key head: row_tiles tiles of up to `rows`
  float scale, cap;                                    // scale: times log2(e) where no cap comes between
  int window;
  void* out;                                           // [batch][heads][dim]
  float* lse;                                          // [batch][heads] or null
  float* part_o; float2* part_ml; int4* meta;          // two partial results per CTA, and which items start here but end elsewhere
  int split;                                           // 0: one CTA per item
};

// tiles of keys of sequence b (at least one, so that an empty row is visited too); *first..*end: its visible keys
template <int TK>
__device__ __forceinline__ int tiles_of(const AttnParams& p, int b, int* first, int* end) {
  const int len = max(p.lens[b], 0);
  const int64_t held = (int64_t)p.width * p.page_size;
  *end = (int)min((int64_t)len, held);
  *first = p.window > 0 && len > p.window ? len - p.window : 0;
  return max(1, (*end + TK - 1) / TK - *first / TK);
}

// The share of this CTA: units [u0, u1), and the sequence and offset of u0.
struct Share { int64_t u0, u1, base; int b; int64_t total; int ctas; };

template <int TK>
__device__ Share find_share(const AttnParams& p, int64_t* s_red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = p.kv_heads * p.row_tiles;
  int64_t sum = 0;
  int f, e;
  for (int b = tid; b < p.batch; b += AT_WARPS * 32) sum += AT_START + tiles_of<TK>(p, b, &f, &e);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) s_red[warp] = sum;
  __syncthreads();
  Share s;
  s.total = 0;
#pragma unroll
  for (int w = 0; w < AT_WARPS; ++w) s.total += s_red[w];
  s.total *= per;
  // a share that is hardly more than a beginning would only add partial results
  s.ctas = (int)min((int64_t)gridDim.x, (s.total + AT_START + AT_WARPS - 1) / (AT_START + AT_WARPS));
  s.u0 = s.total * blockIdx.x / s.ctas;
  s.u1 = s.total * (blockIdx.x + 1) / s.ctas;
  s.b = 0;
  s.base = 0;
  if ((int)blockIdx.x >= s.ctas) { s.u0 = s.u1 = 0; return s; }
  // every warp scans the sequences 32 at a time until it reaches the one that holds u0
  int64_t run = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int64_t v = b0 + lane < p.batch ? (int64_t)(AT_START + tiles_of<TK>(p, b0 + lane, &f, &e)) * per : 0;
    const int64_t own = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, run + v > s.u0);
    if (past) {
      const int at = __ffs(past) - 1;
      s.b = b0 + at;
      s.base = run + __shfl_sync(0xffffffffu, v - own, at);
      break;
    }
    run += __shfl_sync(0xffffffffu, v, 31);
  }
  return s;
}

__device__ __forceinline__ int cta_of(const Share& s, int64_t unit) {   // the CTA whose share holds `unit`
  int c = (int)(unit * s.ctas / s.total);
  while (c + 1 < s.ctas && s.total * (c + 1) / s.ctas <= unit) ++c;
  while (c > 0 && s.total * c / s.ctas > unit) --c;
  return c;
}

// 16 bytes, or with live = false 16 bytes of zeros and no read
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Writes the tile's results: s_o [AT_WARPS][rows][dim] unnormalised values of the warps, s_ml their maxima and sums.
// `slot` < 0: the item is complete; otherwise the index of its partial result.
template <typename T>
__device__ void store_tile(const AttnParams& p, const float* s_o, const float2* s_ml, int b, int head0, int rows, int R, int slot) {
  const int n = rows * p.dim;
  for (int i = threadIdx.x; i < n; i += AT_WARPS * 32) {
    const int r = i / p.dim, d = i - r * p.dim;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) m = fmaxf(m, s_ml[w * R + r].x);
    const float mm = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) {
      const float f = exp2f(s_ml[w * R + r].x - mm);
      l += s_ml[w * R + r].y * f;
      o += s_o[(w * R + r) * p.dim + d] * f;
    }
    if (slot < 0) {
      reinterpret_cast<T*>(p.out)[((int64_t)b * p.heads + head0 + r) * p.dim + d] = from_f32<T>(l == 0.f ? 0.f : o / l);
      if (d == 0 && p.lse) p.lse[(int64_t)b * p.heads + head0 + r] = l == 0.f ? -INFINITY : m * AT_LN2 + logf(l);
    } else {
      p.part_o[((int64_t)slot * p.rows + r) * p.dim + d] = o;
      if (d == 0) p.part_ml[(int64_t)slot * p.rows + r] = make_float2(m, l);
    }
  }
}

// Adds the partial results of the item that starts in share c and ends in share meta.y, in the order of the keys.
template <typename T>
__global__ void __launch_bounds__(128) attend_join_kernel(const AttnParams p) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x;
  const int4 m4 = p.meta[c];
  const int item = m4.x, last = m4.y;
  if (item < 0) return;
  const int per = p.kv_heads * p.row_tiles;
  const int b = item / per, h = item % per / p.row_tiles, x = item % p.row_tiles;
  const int head0 = h * p.group + x * p.rows, rows = min(p.rows, p.group - x * p.rows);
  const int r = blockIdx.y;
  if (r >= rows) return;
  float m = -INFINITY;
  for (int i = c; i <= last; ++i) m = fmaxf(m, p.part_ml[(int64_t)(2 * i + (i == c)) * p.rows + r].x);
  const float mm = m == -INFINITY ? 0.f : m;
  for (int d = threadIdx.x; d < p.dim; d += 128) {
    float l = 0.f, o = 0.f;
#pragma unroll 4
    for (int i = c; i <= last; ++i) {
      const int64_t at = (int64_t)(2 * i + (i == c)) * p.rows + r;
      const float2 ml = p.part_ml[at];
      const float f = exp2f(ml.x - mm);
      l += ml.y * f;
      o += p.part_o[at * p.dim + d] * f;
    }
    reinterpret_cast<T*>(p.out)[((int64_t)b * p.heads + head0 + r) * p.dim + d] = from_f32<T>(l == 0.f ? 0.f : o / l);
    if (d == 0 && p.lse) p.lse[(int64_t)b * p.heads + head0 + r] = l == 0.f ? -INFINITY : m * AT_LN2 + logf(l);
  }
}

// Where key j of sequence b lies: page name and place inside the page; false where there is no such page.
__device__ __forceinline__ bool find_key(const AttnParams& p, int b, int j, int first, int end, int* page, int* place) {
  if (j < first || j >= end) return false;
  const int at = (int)((unsigned)j / (unsigned)p.page_size);
  *place = j - at * p.page_size;
  *page = p.table[(int64_t)b * p.table_b + at];
  return *page >= 0 && *page < p.num_pages;
}

__device__ __forceinline__ float4 lds4(uint32_t a) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(a) : "memory");
  return f;
}

// fp32: products on the fp32 pipes (three tf32 products would be needed for as many bits): a lane owns four neighbouring dimensions in every 128 (NI groups), so a key row is one dense read
// of the warp and q and the values stay in registers; R rows x 32 / R keys of partial dot products are summed over the lanes by
// halving the rows and keys that a lane still holds (31 shuffles for 32 sums), after which lane = (row, key) holds one score.
// Keys and values come through a ring of cp.async copies; a lane copies exactly the bytes that it reads back.
template <int R, int NI, int STAGES>
__global__ void __launch_bounds__(AT_WARPS * 32) attend_fma_kernel(const AttnParams p) {
  constexpr int KB = 32 / R;                      // keys of a tile
  constexpr int CH = 16;                          // bytes of a lane's piece of a row
  constexpr int ROW = NI * 32 * CH;
  constexpr int SLOT = 2 * KB * ROW;              // keys, then values
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_red[AT_WARPS];
  __shared__ float2 s_ml[AT_WARPS * R];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (STAGES * SLOT) + lane * CH;
  float* s_o = reinterpret_cast<float*>(smem);
  pdl_trigger();
  pdl_wait();

  Share s;
  int64_t unit, unit_end;
  int b;
  int64_t base;
  const int per = p.kv_heads * p.row_tiles;
  if (p.split) {
    s = find_share<KB>(p, s_red);
    if (tid == 0) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
    unit = s.u0; unit_end = s.u1; b = s.b; base = s.base;
  } else {
    b = blockIdx.x / per;
    unit = 0; unit_end = 1; base = 0;              // one item, whatever its tiles
  }
  while (unit < unit_end) {
    int first, end;
    const int tiles = tiles_of<KB>(p, b, &first, &end);
    int64_t next_base = base;
    int next_b = b, sub, t0, t1;                   // (key head, row tile), first and last + 1 tile of this segment
    if (p.split) {
      const int cost = AT_START + tiles;
      sub = (int)((unit - base) / cost);
      const int at = (int)((unit - base) % cost);
      const int upto = (int)min((int64_t)cost, at + (unit_end - unit));
      t0 = max(at - AT_START, 0); t1 = upto - AT_START;
      unit += upto - at;
      if (unit == base + (int64_t)cost * per) { next_base = unit; next_b = b + 1; }
      if (t1 <= 0) { base = next_base; b = next_b; continue; }    // the next CTA begins this item
    } else {
      sub = blockIdx.x % per;
      t0 = 0; t1 = tiles;
    }
    const int h = sub / p.row_tiles, x = sub % p.row_tiles;
    const int head0 = h * p.group + x * p.rows, rows = min(p.rows, p.group - x * p.rows);
    const int key0 = first / KB * KB;              // tiles start at multiples of KB

    float q[R][NI * 4], o[R][NI * 4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = i * 128 + lane * 4 + e;
          q[r][i * 4 + e] = r < rows && d < p.dim ? static_cast<const float*>(p.q)[(int64_t)b * p.q_b + (int64_t)(head0 + r) * p.q_h + d] : 0.f;
          o[r][i * 4 + e] = 0.f;
        }
    float m = -INFINITY, l = 0.f;                  // of row lane / KB; l: of the lane's own keys

    uint32_t live_ring[STAGES];
    auto fetch = [&](int t, int slot) -> uint32_t {
      int page = 0, place = 0;
      const int j = key0 + t * KB + (lane % KB);
      const bool ok = t < t1 && find_key(p, b, j, first, end, &page, &place);
      const uint32_t live = __ballot_sync(0xffffffffu, ok);
      if (t < t1) {
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
          const int64_t pg = __shfl_sync(0xffffffffu, page, kk), pl = __shfl_sync(0xffffffffu, place, kk);
          const bool on = live >> kk & 1;
          const float* kr = static_cast<const float*>(p.k) + (on ? pg * p.k_page + pl * p.k_slot + h * p.k_head : 0);
          const float* vr = static_cast<const float*>(p.v) + (on ? pg * p.v_page + pl * p.v_slot + h * p.v_head : 0);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const int d = i * 128 + lane * 4;
            const bool in = on && d < p.dim;       // otherwise zeros are written and nothing is read
            cp_async(ring + slot * SLOT + kk * ROW + i * 32 * CH, kr + (in ? d : 0), in);
            cp_async(ring + slot * SLOT + (KB + kk) * ROW + i * 32 * CH, vr + (in ? d : 0), in);
          }
        }
      }
      cp_commit();
      return live;
    };
    const int mine = t0 + warp;
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) live_ring[st] = fetch(mine + st * AT_WARPS, st);
    int slot = 0;
    for (int t = mine; t < t1; t += AT_WARPS) {
      const uint32_t got = live_ring[0];
#pragma unroll
      for (int st = 0; st + 2 < STAGES; ++st) live_ring[st] = live_ring[st + 1];
      live_ring[STAGES - 2] = fetch(t + (STAGES - 1) * AT_WARPS, (slot + STAGES - 1) % STAGES);
      cp_wait<STAGES - 1>();
      const uint32_t at = ring + slot * SLOT;
      slot = slot + 1 == STAGES ? 0 : slot + 1;
      float v[32];                                 // index r * KB + kk
#pragma unroll
      for (int kk = 0; kk < KB; ++kk) {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r * KB + kk] = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const float4 kx = lds4(at + kk * ROW + i * 32 * CH);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float a = v[r * KB + kk];
            a = fmaf(q[r][i * 4], kx.x, a); a = fmaf(q[r][i * 4 + 1], kx.y, a);
            a = fmaf(q[r][i * 4 + 2], kx.z, a); a = fmaf(q[r][i * 4 + 3], kx.w, a);
            v[r * KB + kk] = a;
          }
        }
      }
#pragma unroll
      for (int half = 16; half > 0; half >>= 1) {
        const bool up = lane & half;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float send = up ? v[i] : v[i + half];
          const float keep = up ? v[i + half] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, half);
        }
      }
      float sc = v[0] * p.scale;
      if (p.cap > 0.f) sc = p.cap * AT_LOG2E * tanhf(sc / p.cap);
      if (!(got >> (lane % KB) & 1)) sc = -INFINITY;
      float top = sc;
#pragma unroll
      for (int d = 1; d < KB; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float mn = fmaxf(m, top);
      const float use = mn == -INFINITY ? 0.f : mn;
      if (__any_sync(0xffffffffu, mn > m)) {       // a new maximum in some row: rescale what is there
        const float f = exp2f(m - use);
        l *= f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float fr = __shfl_sync(0xffffffffu, f, r * KB);
#pragma unroll
          for (int i = 0; i < NI * 4; ++i) o[r][i] *= fr;
        }
      }
      m = mn;
      const float w = exp2f(sc - use);
      l += w;
#pragma unroll
      for (int kk = 0; kk < KB; ++kk) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const float4 vx = lds4(at + (KB + kk) * ROW + i * 32 * CH);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float wr = __shfl_sync(0xffffffffu, w, r * KB + kk);
            o[r][i * 4] = fmaf(wr, vx.x, o[r][i * 4]); o[r][i * 4 + 1] = fmaf(wr, vx.y, o[r][i * 4 + 1]);
            o[r][i * 4 + 2] = fmaf(wr, vx.z, o[r][i * 4 + 2]); o[r][i * 4 + 3] = fmaf(wr, vx.w, o[r][i * 4 + 3]);
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();                               // the ring becomes the place where the warps' results meet
#pragma unroll
    for (int d = 1; d < KB; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (lane % KB == 0) s_ml[warp * R + lane / KB] = make_float2(m, l);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int d = i * 128 + lane * 4;
        if (d < p.dim) *reinterpret_cast<float4*>(s_o + (warp * R + r) * p.dim + d) = make_float4(o[r][i * 4], o[r][i * 4 + 1], o[r][i * 4 + 2], o[r][i * 4 + 3]);
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    store_tile<float>(p, s_o, s_ml, b, head0, rows, R, whole ? -1 : 2 * (int)blockIdx.x + (t0 == 0));
    if (!p.split) break;
    if (!whole && t0 == 0 && tid == 0)
      p.meta[blockIdx.x] = make_int4(b * per + sub, cta_of(s, base + (int64_t)(sub + 1) * (AT_START + tiles) - 1), 0, 0);
    __syncthreads();
    base = next_base;
    b = next_b;
  }
}

// ---- 16-bit types: products on the tensor cores ----
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t bits_of(T lo, T hi) {
  return (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
}
// two weights as two 16-bit parts each: hi = T(w), lo = T(w - hi)
template <typename T> __device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  const T a = from_f32<T>(x), b = from_f32<T>(y);
  hi = bits_of<T>(a, b);
  lo = bits_of<T>(from_f32<T>(x - to_f32<T>(a)), from_f32<T>(y - to_f32<T>(b)));
}

constexpr int MM_KEYS = 16;
template <int DP> struct MmaShape {
  static constexpr int ROW = ((DP / 8) | 1) * 16;                 // an odd number of 16-byte pieces: ldmatrix without bank conflicts
  static constexpr int SLOT = 2 * MM_KEYS * ROW;                  // keys, then values
  static constexpr int STAGES = DP == 64 ? 6 : 3;
  static constexpr int CTAS = DP == 256 ? 1 : 2;                  // per multiprocessor
  static constexpr int SMEM = AT_WARPS * STAGES * SLOT;
};

// m16n8k16 products: the query heads of a tile are the 16 rows, 16 cached keys a step.  Scores: A = q (registers), B = keys;
// values: A = weights (the score accumulators are already in A's layout), B = values (transposed by ldmatrix).  The weights enter as
// two 16-bit parts, so that they count with 16 bits and more; up to eight heads leave the upper eight rows free, and the low
// parts ride there at no cost (TWO = false); above that they are a second product.
template <typename T, int DP, bool TWO>
__global__ void __launch_bounds__(AT_WARPS * 32, MmaShape<DP>::CTAS) attend_mma_kernel(const AttnParams p) {
  using S = MmaShape<DP>;
  constexpr int R = TWO ? 16 : 8;
  constexpr int STAGES = S::STAGES;
  constexpr int LPR = DP / 8;                                     // lanes of a row of the copies
  constexpr int COPIES = MM_KEYS * LPR / 32;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_red[AT_WARPS];
  __shared__ float2 s_ml[AT_WARPS * R];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (STAGES * S::SLOT);
  const uint32_t k_at = ring + ((lane >> 4) * 8 + (lane & 7)) * S::ROW + (lane >> 3 & 1) * 16;
  const uint32_t v_at = ring + (MM_KEYS + (lane >> 3 & 1) * 8 + (lane & 7)) * S::ROW + (lane >> 4) * 16;
  float* s_o = reinterpret_cast<float*>(smem);
  const int nk = p.dim / 16;
  const bool one_page = p.page_size % MM_KEYS == 0;               // tiles start at multiples of 16
  pdl_trigger();
  pdl_wait();

  Share s;
  int64_t unit, unit_end;
  int b;
  int64_t base;
  const int per = p.kv_heads * p.row_tiles;
  if (p.split) {
    s = find_share<MM_KEYS>(p, s_red);
    if (tid == 0) p.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
    unit = s.u0; unit_end = s.u1; b = s.b; base = s.base;
  } else {
    b = blockIdx.x / per;
    unit = 0; unit_end = 1; base = 0;
  }
  while (unit < unit_end) {
    int first, end;
    const int tiles = tiles_of<MM_KEYS>(p, b, &first, &end);
    int64_t next_base = base;
    int next_b = b, sub, t0, t1;
    if (p.split) {
      const int cost = AT_START + tiles;
      sub = (int)((unit - base) / cost);
      const int at = (int)((unit - base) % cost);
      const int upto = (int)min((int64_t)cost, at + (unit_end - unit));
      t0 = max(at - AT_START, 0); t1 = upto - AT_START;
      unit += upto - at;
      if (unit == base + (int64_t)cost * per) { next_base = unit; next_b = b + 1; }
      if (t1 <= 0) { base = next_base; b = next_b; continue; }    // the next CTA begins this item
    } else {
      sub = blockIdx.x % per;
      t0 = 0; t1 = tiles;
    }
    const int h = sub / p.row_tiles, x = sub % p.row_tiles;
    const int head0 = h * p.group + x * p.rows, rows = min(p.rows, p.group - x * p.rows);
    const int key0 = first / MM_KEYS * MM_KEYS;

    uint32_t q[DP / 16][TWO ? 4 : 2];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int i = 0; i < (TWO ? 4 : 2); ++i) {
        const int r = TWO ? g + (i & 1) * 8 : g, d = ks * 16 + t4 * 2 + (TWO ? i >> 1 : i) * 8;
        q[ks][i] = 0;
        if (r < rows && ks < nk) {
          const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_b + (int64_t)(head0 + r) * p.q_h + d;
          q[ks][i] = bits_of<T>(src[0], src[1]);
        }
      }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};       // rows g and g + 8; l: of the lane's own keys

    // the page of the lane's key is looked up a tile before the copies that need it; k_lane, v_lane: the lane's piece of its first
    // row, in the first page
    int page32 = 0, place = 0;
    int64_t page = 0, place0 = 0;                                 // place0: of the tile's first key, seen from the lane's
    bool ok = false;
    auto look = [&](int t) {
      ok = t < t1 && find_key(p, b, key0 + t * MM_KEYS + (lane & 15), first, end, &page32, &place);
      page = page32;
      place0 = place - (lane & 15);
    };
    const int piece = lane % LPR;
    const T* k_lane = static_cast<const T*>(p.k) + ((int64_t)h * p.k_head + (lane / LPR) * p.k_slot + piece * 8);
    const T* v_lane = static_cast<const T*>(p.v) + ((int64_t)h * p.v_head + (lane / LPR) * p.v_slot + piece * 8);
    auto fetch = [&](int slot) -> uint32_t {
      const uint32_t live = __ballot_sync(0xffffffffu, ok) & 0xffffu;
      const uint32_t dst = ring + slot * S::SLOT + (lane / LPR) * S::ROW + piece * 16;
      if (live == 0xffffu && one_page) {                          // 16 tokens of one page: one address and a fixed step
        if (piece * 8 < p.dim) {
          const T* kp = k_lane + (page * p.k_page + place0 * p.k_slot);
          const T* vp = v_lane + (page * p.v_page + place0 * p.v_slot);
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            cp_async(dst + i * (32 / LPR) * S::ROW, kp, true);
            cp_async(dst + (MM_KEYS + i * (32 / LPR)) * S::ROW, vp, true);
            kp += (32 / LPR) * p.k_slot;
            vp += (32 / LPR) * p.v_slot;
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < COPIES; ++i) {
          const int row = i * (32 / LPR) + lane / LPR;
          const int64_t pg = __shfl_sync(0xffffffffu, page, row), pl = __shfl_sync(0xffffffffu, place0 + (lane & 15), row) - lane / LPR;
          const bool on = live >> row & 1;
          if (piece * 8 < p.dim) {                                // rows that are not live are filled with zeros
            cp_async(dst + i * (32 / LPR) * S::ROW, on ? k_lane + (pg * p.k_page + pl * p.k_slot) : k_lane, on);
            cp_async(dst + (MM_KEYS + i * (32 / LPR)) * S::ROW, on ? v_lane + (pg * p.v_page + pl * p.v_slot) : v_lane, on);
          }
        }
      }
      cp_commit();
      return live;
    };
    const int mine = t0 + warp;
    uint32_t live_ring[STAGES - 1];
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) {
      look(mine + st * AT_WARPS);
      live_ring[st] = fetch(st);
    }
    look(mine + (STAGES - 1) * AT_WARPS);
    int slot = 0;
    for (int t = mine; t < t1; t += AT_WARPS) {
      const uint32_t live = live_ring[0];
#pragma unroll
      for (int st = 0; st + 2 < STAGES; ++st) live_ring[st] = live_ring[st + 1];
      __syncwarp();                                               // every lane has read the slot that is filled next
      live_ring[STAGES - 2] = fetch(slot == 0 ? STAGES - 1 : slot - 1);
      look(t + STAGES * AT_WARPS);
      cp_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t off = slot * S::SLOT;
      slot = slot + 1 == STAGES ? 0 : slot + 1;

      float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        if (ks < nk) {
          uint32_t kb[4];
          ldsm4(kb, k_at + off + ks * 32);
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            if constexpr (TWO) mma16816<T>(c[nt], q[ks][0], q[ks][1], q[ks][2], q[ks][3], kb[2 * nt], kb[2 * nt + 1]);
            else mma16816<T>(c[nt], q[ks][0], 0u, q[ks][1], 0u, kb[2 * nt], kb[2 * nt + 1]);
          }
        }
      }
      uint32_t hi[4], lo[4];                                      // weights: [key tile][row half]
#pragma unroll
      for (int half = 0; half < (TWO ? 2 : 1); ++half) {
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = c[i >> 1][half * 2 + (i & 1)] * p.scale;
          if (p.cap > 0.f) v = p.cap * AT_LOG2E * tanhf(v / p.cap);
          sc[i] = live >> ((i >> 1) * 8 + t4 * 2 + (i & 1)) & 1 ? v : -INFINITY;
        }
        float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[half], top);
        const float use = mn == -INFINITY ? 0.f : mn;
        if (__any_sync(0xffffffffu, mn > m[half])) {              // a new maximum in some row: rescale what is there
          const float f = exp2f(m[half] - use);
          l[half] *= f;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            o[i][2 * half] *= f; o[i][2 * half + 1] *= f;
            if constexpr (!TWO) { o[i][2] *= f; o[i][3] *= f; }
          }
        }
        m[half] = mn;
#pragma unroll
        for (int i = 0; i < 4; ++i) { sc[i] = exp2f(sc[i] - use); l[half] += sc[i]; }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) split_pair<T>(sc[2 * nt], sc[2 * nt + 1], hi[2 * nt + half], lo[2 * nt + half]);
      }
#pragma unroll
      for (int cc = 0; cc < DP / 16; ++cc) {
        if (cc < nk) {
          uint32_t vb[4];
          ldsm4_t(vb, v_at + off + cc * 32);
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            if constexpr (TWO) {
              mma16816<T>(o[2 * cc + n2], hi[0], hi[1], hi[2], hi[3], vb[2 * n2], vb[2 * n2 + 1]);
              mma16816<T>(o[2 * cc + n2], lo[0], lo[1], lo[2], lo[3], vb[2 * n2], vb[2 * n2 + 1]);
            } else {
              mma16816<T>(o[2 * cc + n2], hi[0], lo[0], hi[2], lo[2], vb[2 * n2], vb[2 * n2 + 1]);
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();                                              // the ring becomes the place where the warps' results meet
#pragma unroll
    for (int half = 0; half < (TWO ? 2 : 1); ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
      const int r = g + half * 8;
      if (t4 == 0) s_ml[warp * R + r] = make_float2(m[half], l[half]);
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        if (i < 2 * nk) {
          const float a = TWO ? o[i][2 * half] : o[i][0] + o[i][2], e = TWO ? o[i][2 * half + 1] : o[i][1] + o[i][3];
          *reinterpret_cast<float2*>(s_o + (warp * R + r) * p.dim + i * 8 + t4 * 2) = make_float2(a, e);
        }
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    store_tile<T>(p, s_o, s_ml, b, head0, rows, R, whole ? -1 : 2 * (int)blockIdx.x + (t0 == 0));
    if (!p.split) break;
    if (!whole && t0 == 0 && tid == 0)
      p.meta[blockIdx.x] = make_int4(b * per + sub, cta_of(s, base + (int64_t)(sub + 1) * (AT_START + tiles) - 1), 0, 0);
    __syncthreads();
    base = next_base;
    b = next_b;
  }
}

template <typename T>
int launch_both(void (*kern)(const AttnParams), AttnParams& p, int smem, int ctas_per_sm, cudaStream_t st) {
  const bool pdl = options().pdl != 0;
  const unsigned grid = p.split ? (unsigned)(sm_count() * ctas_per_sm) : (unsigned)((int64_t)p.batch * p.kv_heads * p.row_tiles);
  KQ_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(AT_WARPS * 32), (size_t)smem, st, pdl, p));
  options().launches += 1;
  if (p.split) {
    KQ_CUDA_TRY(launch_pdl(attend_join_kernel<T>, dim3(grid, (unsigned)p.rows), dim3(128), (size_t)0, st, pdl, p));
    options().launches += 1;
  }
  return KQ_OK;
}

template <int R, int NI>
int run_fma(AttnParams& p, cudaStream_t st) {
  constexpr int STAGES = R == 8 ? 3 : 2;
  constexpr int ring = AT_WARPS * STAGES * 2 * (32 / R) * NI * 512, join = AT_WARPS * R * NI * 128 * 4;
  constexpr int smem = ring > join ? ring : join;
  auto kern = attend_fma_kernel<R, NI, STAGES>;
  static DeviceOnce attr_set;
  if (attr_set.first_time()) {
    KQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set.done();
  }
  return launch_both<float>(kern, p, smem, AT_MAX_CTAS, st);
}

template <typename T, int DP, bool TWO>
int run_mma(AttnParams& p, cudaStream_t st) {
  using S = MmaShape<DP>;
  constexpr int join = AT_WARPS * (TWO ? 16 : 8) * DP * 4;
  constexpr int smem = S::SMEM > join ? S::SMEM : join;
  auto kern = attend_mma_kernel<T, DP, TWO>;
  static DeviceOnce attr_set;
  if (attr_set.first_time()) {
    KQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set.done();
  }
  return launch_both<T>(kern, p, smem, S::CTAS, st);
}

// the query heads of a key head in tiles of at most `most` rows, of even sizes
void set_rows(AttnParams& p, int most) {
  p.row_tiles = (p.group + most - 1) / most;
  p.rows = (p.group + p.row_tiles - 1) / p.row_tiles;
  p.row_tiles = (p.group + p.rows - 1) / p.rows;
}

int run_f32(AttnParams& p, cudaStream_t st) {
  set_rows(p, 8);
  if (p.rows <= 4) return p.dim > 128 ? run_fma<4, 2>(p, st) : run_fma<4, 1>(p, st);
  return p.dim > 128 ? run_fma<8, 2>(p, st) : run_fma<8, 1>(p, st);
}

template <typename T>
int run_16bit(AttnParams& p, cudaStream_t st) {
  set_rows(p, 16);
  if (p.rows <= 8) return p.dim > 128 ? run_mma<T, 256, false>(p, st) : p.dim > 64 ? run_mma<T, 128, false>(p, st) : run_mma<T, 64, false>(p, st);
  return p.dim > 128 ? run_mma<T, 256, true>(p, st) : p.dim > 64 ? run_mma<T, 128, true>(p, st) : run_mma<T, 64, true>(p, st);
}

constexpr int AT_MAX_ROWS = 16;

struct Scratch { size_t o, ml, meta, total; };
Scratch scratch_of(int64_t ctas, int64_t dim) {
  Scratch s;
  s.o = 0;
  s.ml = s.o + (size_t)(2 * ctas * AT_MAX_ROWS * dim * 4 + 255) / 256 * 256;
  s.meta = s.ml + (size_t)(2 * ctas * AT_MAX_ROWS * 8 + 255) / 256 * 256;
  s.total = s.meta + (size_t)(ctas * 16 + 255) / 256 * 256;
  return s;
}

}  // namespace

}  // namespace kq

using namespace kq;

extern "C" {

size_t kq_paged_attention_workspace_bytes(int64_t head_dim) {
  if (head_dim <= 0 || head_dim > 256) return 0;
  return scratch_of((int64_t)sm_count() * AT_MAX_CTAS, head_dim).total;
}

int kq_paged_attention(const void* q, int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t q_stride_batch,
                       int64_t q_stride_head, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                       const int64_t* v_strides, int64_t num_pages, int64_t page_size, const int32_t* block_table, int64_t table_stride,
                       int64_t table_width, const int32_t* seq_lens, float scale, int64_t window, float softcap, void* out, float* lse,
                       void* scratch, size_t scratch_bytes, void* stream) {
  const char* fn = "kq_paged_attention";
  set_error("%s", "");
  if (dtype != KQ_F32 && dtype != KQ_F16 && dtype != KQ_BF16) { set_error("%s: unsupported dtype %d", fn, dtype); return KQ_EUNSUPPORTED; }
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) {
    set_error("%s: heads=%lld must be a positive multiple of kv_heads=%lld", fn, (long long)heads, (long long)kv_heads);
    return KQ_EINVAL;
  }
  if (head_dim < 16 || head_dim > 256 || head_dim % 16) { set_error("%s: head_dim=%lld is not a multiple of 16 up to 256", fn, (long long)head_dim); return KQ_EUNSUPPORTED; }
  if (batch > (1 << 20) || heads > (1 << 16) || batch * heads > 0x7fffffff || page_size > 0x7fffffff || table_width > 0x7fffffff || num_pages > 0x7fffffff) {
    set_error("%s: size out of range", fn);
    return KQ_ELIMIT;
  }
  if (page_size <= 0 || num_pages < 0 || table_width < 0) { set_error("%s: page_size must be positive, num_pages and table_width not negative", fn); return KQ_EINVAL; }
  if (window < 0 || window > 0x7fffffff) { set_error("%s: window=%lld is outside [0, 2^31)", fn, (long long)window); return KQ_EINVAL; }
  if (!(scale > 0.f) || scale > 3e38f || !(softcap >= 0.f) || softcap > 3e38f) { set_error("%s: scale must be positive and softcap not negative, both finite", fn); return KQ_EINVAL; }
  if (batch == 0) return KQ_OK;
  if (!q || !out || !seq_lens || (table_width > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)) || !k_strides || !v_strides) {
    set_error("%s: null pointer", fn);
    return KQ_EINVAL;
  }
  const int64_t size = dtype == KQ_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] < 0 || v_strides[i] < 0 || k_strides[i] * size % 16 || v_strides[i] * size % 16) {
      set_error("%s: cache strides must be multiples of 16 bytes", fn);
      return KQ_EINVAL;
    }
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)q % size || (uintptr_t)out % 16) { set_error("%s: misaligned pointer", fn); return KQ_EINVAL; }
  const int64_t ctas = (int64_t)sm_count() * AT_MAX_CTAS;
  const Scratch L = scratch_of(ctas, head_dim);
  if (!scratch || (uintptr_t)scratch % 256) { set_error("%s: scratch must be non-null and 256-byte aligned", fn); return KQ_ESCRATCH; }
  if (scratch_bytes < L.total) { set_error("%s: scratch too small (%zu < %zu)", fn, scratch_bytes, L.total); return KQ_ESCRATCH; }

  AttnParams p;
  p.q = q; p.q_b = q_stride_batch; p.q_h = q_stride_head;
  p.k = k_cache; p.k_page = k_strides[0]; p.k_slot = k_strides[1]; p.k_head = k_strides[2];
  p.v = v_cache; p.v_page = v_strides[0]; p.v_slot = v_strides[1]; p.v_head = v_strides[2];
  p.table = block_table; p.table_b = table_stride; p.width = (int)table_width; p.lens = seq_lens;
  p.batch = (int)batch; p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.group = (int)(heads / kv_heads); p.dim = (int)head_dim;
  p.page_size = (int)page_size; p.num_pages = num_pages;
  p.scale = softcap > 0.f ? scale : scale * AT_LOG2E; p.cap = softcap; p.window = (int)window;
  p.out = out; p.lse = lse;
  uint8_t* sb = (uint8_t*)scratch;
  p.part_o = (float*)(sb + L.o); p.part_ml = (float2*)(sb + L.ml); p.meta = (int4*)(sb + L.meta);
  int64_t most = table_width * page_size;          // keys that a sequence can show
  if (window > 0 && window < most) most = window;
  p.split = most > 256;      // short sequences: one launch, one CTA per item
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case KQ_F32: return run_f32(p, st);
    case KQ_F16: return run_16bit<__half>(p, st);
    default: return run_16bit<__nv_bfloat16>(p, st);
  }
}

}  // extern "C"
