// Attention of one new token per sequence over a paged key-value cache (kq_paged_attention).
//
//   s_j = f(scale * q . k_j),  f(x) = x or cap * tanh(x / cap),  j in [max(0, len - window), len)
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j;  a sequence without visible keys gives zeros
//
// One pass over the cache: a warp keeps the running maximum, the running sum and the weighted values of the query heads that
// share a key head (their rows are one tile) in registers, in fp32, and rescales them when a new maximum comes.
//
// The work is cut by cached keys, not by sequences: an item is (sequence, key head, row tile) and has one unit of work per
// tile of keys, behind a few units for its beginning and end; the units of all items, in order, are divided evenly over the workers
// of one wave.  A worker finds its share from the lengths themselves (a sum and a scan, the lengths stay on the GPU), so a batch of any
// mix of lengths is balanced and a captured call follows the lengths of each replay.  An item inside one worker is finished there; one that
// crosses workers leaves partial results (unnormalised values, maximum, sum) that attend_join_kernel adds in the order of the
// keys: no atomics, the same bits every time.
//
// A worker is a CTA whose warps take turns at the tiles and join their results at the end of an item, or, where there are items enough
// for every warp of the wave, a warp on its own, which has nothing to join.  Where no sequence can be long, workers take whole items.
#include <type_traits>

#include "kq_common.cuh"

namespace kq {

namespace {

#include "kq_tile_common.cuh"

constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr float AT_LN2 = 0.6931471805599453f;

__device__ int g_attend_status = 0;

struct AttnParams {
  const void* q; int64_t q_b, q_h; int q_words;        // strides in elements; the head dimension is dense everywhere; q_words: pairs are aligned
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
  float* part_o; float2* part_ml; int2* meta;          // two partial results per worker; which item starts in a worker and ends in which other
  int split;                                           // 0: workers take whole items, in turn
  int solo;                                            // a worker is a warp (of the computing ones), not a CTA
};

// tiles of TK keys of sequence b (at least one, so that an empty row is visited too); *first..*end: its visible keys
template <int TK>
__device__ __forceinline__ int tiles_of(const AttnParams& p, int b, int* first, int* end) {
  const int len = max(p.lens[b], 0);
  const int64_t held = (int64_t)p.width * p.page_size;
  *end = (int)min((int64_t)len, held);
  *first = p.window > 0 && len > p.window ? len - p.window : 0;
  return max(1, (int)(((unsigned)*end + TK - 1) / TK) - *first / TK);     // a length may be 2^31 - 1
}

// A stretch of an item's tiles that one worker covers.
struct Segment {
  int b, sub;            // sequence, (key head, row tile)
  int first, end;        // visible keys
  int t0, t1, tiles;     // tiles [t0, t1) of `tiles`; tile 0 starts at the last multiple of TK not above `first`
  int last;              // the worker that has the item's last tile, where that is another one
};

// The segments of one worker, in order.  START: what an item costs beside its tiles, in tiles (loading q, joining the warps; without
// it the workers that get the short sequences of a mixed batch end last).  As 1 / as chosen / as more, us: 16-bit types, 1 / 3 / 8, one
// sequence of 2000 tokens 12.4 / 11.6 / 10.6, 64 of 0..1000 35.0 / 35.3 / 37.8, 64 of 0..16384 358 / 359 / 365, heads of 256 (1 / 4 / 8)
// 52.3 / 51.3 / 51.4; fp32, 1 / 8 / 16, one of 2000 20.1 / 17.9 / 18.5, 33 with a window of 1024 51.7 / 46.3 / 44.6, 16 of 4000 with heads
// of 64 62.4 / 58.2 / 61.6.
template <int TK, int START>
struct Walk {
  int64_t left, pos;              // units left, unit index
  int b, sub, at, first, end, tiles;
  int first2, end2, tiles2;       // of the next sequence, loaded ahead

  __device__ void load(const AttnParams& p) { tiles2 = b + 1 < p.batch ? tiles_of<TK>(p, b + 1, &first2, &end2) : 0; }

  // without division: whole items from `item` on, each `stride`-th; pos: the next one, left: items behind its end
  __device__ void begin_items(const AttnParams& p, int item) {
    const int per = p.kv_heads * p.row_tiles;
    pos = item; left = (int64_t)p.batch * per;
    if (pos < left) { b = item / per; sub = item - b * per; tiles = tiles_of<TK>(p, b, &first, &end); }
  }
  __device__ bool next_item(const AttnParams& p, int stride, Segment* s) {
    if (pos >= left) return false;
    s->b = b; s->sub = sub; s->first = first; s->end = end; s->tiles = tiles;
    s->t0 = 0; s->t1 = tiles; s->last = -1;
    const int64_t item = pos + stride;
    begin_items(p, (int)min(item, (int64_t)0x7fffffff));
    return true;
  }

  // the worker whose share holds `unit`; s_div: of the workers the first s_div[1] have s_div[0] + 1 units, the others s_div[0]
  static __device__ int worker_of(const int64_t* s_div, int64_t unit) {
    const int64_t share = s_div[0], more = s_div[1];
    return (int)(unit < more * (share + 1) ? div(unit, share + 1) : more + div(unit - more * (share + 1), share));
  }
  static __device__ int64_t div(int64_t x, int64_t y) {
    return (x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
  }

  // called by all `threads` threads of the CTA at once, which meet before next(); worker: the same for a warp; s_red: one int64 per warp
  __device__ void begin_share(const AttnParams& p, int64_t* s_red, int64_t* s_div, int threads, int worker, int workers) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = p.kv_heads * p.row_tiles;
    int f, e;
    int64_t total = 0;
    if (p.batch > 32) {
      for (int i = tid; i < p.batch; i += threads) total += START + tiles_of<TK>(p, i, &f, &e);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
      if (lane == 0) s_red[warp] = total;
      __syncthreads();
      total = 0;
      for (int w = 0; w < threads / 32; ++w) total += s_red[w];
    }
    // every warp scans the sequences 32 at a time until it reaches the one that holds `pos` (up to 32: the scan is the sum as well)
    int64_t run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      int64_t v = b0 + lane < p.batch ? START + tiles_of<TK>(p, b0 + lane, &f, &e) : 0;
      const int64_t own = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
      }
      const int64_t sum = __shfl_sync(0xffffffffu, v, 31);
      if (b0 == 0) {
        if (p.batch <= 32) total = sum;
        total *= per;
        // a share that is hardly more than a beginning would only add partial results
        workers = (int)min((int64_t)workers, div(total + START, START + 2) + 1);
        const int64_t share = div(total, workers), more = total - share * workers;
        if (tid == 0) { s_div[0] = share; s_div[1] = more; }
        pos = share * worker + min((int64_t)worker, more);
        left = share + (worker < more);
        b = sub = at = 0;
        if (worker >= workers) { left = 0; return; }
      }
      const unsigned past = __ballot_sync(0xffffffffu, (run + v) * per > pos);
      if (past) {
        const int i = __ffs(past) - 1;
        b = b0 + i;
        const int64_t in = pos - (run + __shfl_sync(0xffffffffu, v - own, i)) * per;
        tiles = tiles_of<TK>(p, b, &first, &end);
        load(p);
        sub = (int)div(in, START + tiles);
        at = (int)(in - (int64_t)sub * (START + tiles));
        break;
      }
      run += sum;
    }
  }

  __device__ bool next(const AttnParams& p, const int64_t* s_div, int stride, Segment* s) {
    if (!p.split) return next_item(p, stride, s);
    while (left > 0) {
      const int cost = START + tiles, take = (int)min((int64_t)(cost - at), left);
      s->b = b; s->sub = sub; s->first = first; s->end = end; s->tiles = tiles;
      s->t0 = max(at - START, 0); s->t1 = at + take - START;
      s->last = -1;
      if (s->t0 == 0 && s->t1 > 0 && s->t1 < tiles) s->last = worker_of(s_div, pos + cost - at - 1);
      left -= take; pos += take; at += take;
      if (at == cost) {
        at = 0;
        if (++sub == p.kv_heads * p.row_tiles) {
          sub = 0; ++b;
          first = first2; end = end2; tiles = tiles2;
          load(p);
        }
      }
      if (s->t1 > 0) return true;                 // otherwise the next worker begins this item
    }
    return false;
  }
};

// index of a segment's partial result, -1 if it is the whole item
__device__ __forceinline__ int part_of(const Segment& s, int worker) {
  return s.t0 == 0 && s.t1 == s.tiles ? -1 : 2 * worker + (s.t0 == 0);
}

// 16 bytes, or with live = false 16 bytes of zeros and no read
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) {      // 2^x, relative error 2^-22; results below 2^-126 become 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Where row r (of the tile's rows) of a finished item goes, or of a partial one; `scale`: what its values are multiplied by.
template <typename T> struct RowOut {
  T* out; float* part; float scale;
  RowOut() = default;
  __device__ RowOut(const AttnParams& p, int part_index, int b, int head, int r, float m, float l, bool writes_norm) {
    const int64_t row = (int64_t)b * p.heads + head;
    out = static_cast<T*>(p.out) + row * p.dim;
    part = part_index < 0 ? nullptr : p.part_o + ((int64_t)part_index * p.rows + r) * p.dim;
    scale = part_index >= 0 ? 1.f : l == 0.f ? 0.f : 1.f / l;
    if (writes_norm) {
      if (part_index >= 0) p.part_ml[(int64_t)part_index * p.rows + r] = make_float2(m, l);
      else if (p.lse) p.lse[row] = l == 0.f ? -INFINITY : m * AT_LN2 + logf(l);
    }
  }
  __device__ __forceinline__ void put(int d, float o) const {
    if (part) part[d] = o; else out[d] = from_f32<T>(o * scale);
  }
  __device__ __forceinline__ void put2(int d, float a, float b) const {       // d even
    if (part) {
      *reinterpret_cast<float2*>(part + d) = make_float2(a, b);
    } else {
      alignas(2 * sizeof(T)) T v[2] = {from_f32<T>(a * scale), from_f32<T>(b * scale)};
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(out + d) = *reinterpret_cast<const uint32_t*>(v);
      else *reinterpret_cast<float2*>(out + d) = *reinterpret_cast<const float2*>(v);
    }
  }
};

// Adds the partial results of the item that starts in a worker and ends in worker meta.y, for one row, in the order of the keys; a
// thread has two dimensions, 64 threads (128 above 128 dimensions) a worker.
template <typename T>
__global__ void __launch_bounds__(512) attend_join_kernel(const AttnParams p) {
  pdl_trigger();
  pdl_wait();
  const int log2 = p.dim > 128 ? 7 : 6;
  const int c = blockIdx.x * (blockDim.x >> log2) + (threadIdx.x >> log2), r = blockIdx.y, d = (threadIdx.x & ((1 << log2) - 1)) * 2;
  const int2 it = p.meta[c];
  if (it.x < 0) return;
  const int per = p.kv_heads * p.row_tiles;
  const int b = it.x / per, sub = it.x - b * per, h = sub / p.row_tiles, x = sub - h * p.row_tiles;
  const int head0 = h * p.group + x * p.rows;
  if (r >= min(p.rows, p.group - x * p.rows) || d >= p.dim) return;
  const float2* ml0 = p.part_ml + r;
  const float* o0 = p.part_o + (int64_t)r * p.dim + d;
  float m = -INFINITY, l = 0.f;
  float2 o = make_float2(0.f, 0.f);
  // maxima, sums and values are loaded together, eight parts at a time: the chain is two loads long
  for (int i0 = c; i0 <= it.y; i0 += 8) {
    float2 ml[8], v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = min(i0 + k, it.y), at = (2 * i + (i == c)) * p.rows;      // the first part is in slot 2 c + 1, the others in 2 i
      ml[k] = ml0[at];
      v[k] = *reinterpret_cast<const float2*>(o0 + (int64_t)at * p.dim);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i0 + k <= it.y) {
        const float mn = fmaxf(m, ml[k].x), use = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m - use), g = ex2(ml[k].x - use);
        m = mn;
        l = l * f + ml[k].y * g;
        o.x = o.x * f + v[k].x * g;
        o.y = o.y * f + v[k].y * g;
      }
    }
  }
  const RowOut<T> out(p, -1, b, head0 + r, r, m, l, d == 0);
  out.put2(d, o.x, o.y);
}

// Where key j of sequence b lies: page name and place inside the page; false where there is no such page.
__device__ __forceinline__ bool find_key(const AttnParams& p, int b, unsigned j, int first, int end, int* page, int* place) {
  if (j < (unsigned)first || j >= (unsigned)end) return false;
  const int at = (int)(j / (unsigned)p.page_size);
  *place = (int)j - at * p.page_size;
  *page = p.table[(int64_t)b * p.table_b + at];
  return *page >= 0 && *page < p.num_pages;
}

__device__ __forceinline__ float4 lds4(uint32_t a) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(a) : "memory");
  return f;
}

constexpr int FM_WARPS = 4;            // each walks every fourth tile of keys of the CTA's share on its own
constexpr int FM_START = 8;            // in tiles of 4 to 8 keys
constexpr int FM_MOST = 4;             // CTAs per multiprocessor at most

// fp32: products on the fp32 pipes (as many bits from the tensor cores would take three tf32 products).  A lane owns four neighbouring
// dimensions of a key, and NI times as many in steps of 128 from 128 on; up to 64 dimensions a warp covers two keys at once, one on either
// LD = 16 lanes.  A key row is one dense read, q and the values stay in registers.  R rows x KB keys of partial dot products are summed over
// the LD lanes by halving the rows and keys that a lane still holds (31 shuffles for 32 sums), after which a lane holds one
// score.  Keys and values come through a ring of cp.async copies; a lane copies exactly the bytes that it reads back.
template <int R, int LD, int NI, int STAGES, int KB, int LEAST>
__global__ void __launch_bounds__(FM_WARPS * 32, LEAST) attend_fma_kernel(const AttnParams p) {
  constexpr int SIDES = 32 / LD, KT = KB * SIDES;     // keys next to each other, keys of a tile
  constexpr int N = R * KB, SH = LD / N, RL = LD / R;   // scores of a side, lanes that hold the same one, lanes of a row
  static_assert(N <= LD && (LD == 32 || NI == 1), "a score per lane");
  constexpr int CH = 16;                          // bytes of a lane's piece of a row
  constexpr int ROW = NI * 32 * CH;               // of SIDES keys
  constexpr int SLOT = 2 * KB * ROW;              // keys, then values
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_red[FM_WARPS], s_div[2];
  __shared__ float2 s_ml[FM_WARPS * R];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (STAGES * SLOT) + lane * CH;
  float* s_o = reinterpret_cast<float*>(smem);
  pdl_trigger();
  pdl_wait();

  Walk<KT, FM_START> walk;
  if (p.split) {
    walk.begin_share(p, s_red, s_div, FM_WARPS * 32, blockIdx.x, gridDim.x);
    if (tid == 0) p.meta[blockIdx.x] = make_int2(-1, 0);
  } else {
    walk.begin_items(p, blockIdx.x);
  }
  __syncthreads();
  Segment s;
  while (walk.next(p, s_div, gridDim.x, &s)) {
    const int b = s.b, first = s.first, end = s.end, t0 = s.t0, t1 = s.t1;
    const int h = s.sub / p.row_tiles, x = s.sub - h * p.row_tiles;
    const int head0 = h * p.group + x * p.rows, rows = min(p.rows, p.group - x * p.rows);
    const int key0 = first / KT * KT;              // tiles start at multiples of KT

    float q[R][NI * 4], o[R][NI * 4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = i * 128 + lane % LD * 4 + e;
          q[r][i * 4 + e] = r < rows && d < p.dim ? static_cast<const float*>(p.q)[(int64_t)b * p.q_b + (int64_t)(head0 + r) * p.q_h + d] : 0.f;
          o[r][i * 4 + e] = 0.f;
        }
    float m = -INFINITY, l = 0.f;                  // of row lane / KB; l: of the lane's own keys

    uint32_t live_ring[STAGES];
    auto fetch = [&](int t, int slot) -> uint32_t {
      int page = 0, place = 0;
      const unsigned j = (unsigned)key0 + (unsigned)t * KT + (lane % KT);
      const bool ok = t < t1 && find_key(p, b, j, first, end, &page, &place);
      const uint32_t live = __ballot_sync(0xffffffffu, ok);
      if (t < t1) {
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
          const int row = kk * SIDES + lane / LD;
          const int64_t pg = __shfl_sync(0xffffffffu, page, row), pl = __shfl_sync(0xffffffffu, place, row);
          const bool on = live >> row & 1;
          const float* kr = static_cast<const float*>(p.k) + (on ? pg * p.k_page + pl * p.k_slot + h * p.k_head : 0);
          const float* vr = static_cast<const float*>(p.v) + (on ? pg * p.v_page + pl * p.v_slot + h * p.v_head : 0);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const int d = i * 128 + lane % LD * 4;
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
    for (int st = 0; st < STAGES - 1; ++st) live_ring[st] = fetch(mine + st * FM_WARPS, st);
    int slot = 0;
    for (int t = mine; t < t1; t += FM_WARPS) {
      const uint32_t got = live_ring[0];
#pragma unroll
      for (int st = 0; st + 2 < STAGES; ++st) live_ring[st] = live_ring[st + 1];
      live_ring[STAGES - 2] = fetch(t + (STAGES - 1) * FM_WARPS, (slot + STAGES - 1) % STAGES);
      cp_wait<STAGES - 1>();
      const uint32_t at = ring + slot * SLOT;
      slot = slot + 1 == STAGES ? 0 : slot + 1;
      float v[N];                                 // index r * KB + kk
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
      for (int half = N / 2; half > 0; half >>= 1) {
        const bool up = lane & (half * SH);
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float send = up ? v[i] : v[i + half];
          const float keep = up ? v[i + half] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, half * SH);
        }
      }
#pragma unroll
      for (int d = 1; d < SH; d <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
      float sc = v[0] * p.scale;
      if (p.cap > 0.f) sc = p.cap * AT_LOG2E * tanhf(sc / p.cap);
      if (!(got >> (lane / SH % KB * SIDES + lane / LD) & 1)) sc = -INFINITY;
      float top = sc;
#pragma unroll
      for (int d = SH; d < RL; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      if constexpr (SIDES == 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, LD));
      const float mn = fmaxf(m, top);
      const float use = mn == -INFINITY ? 0.f : mn;
      if (__any_sync(0xffffffffu, mn > m)) {       // a new maximum in some row: rescale what is there
        const float f = exp2f(m - use);
        l *= f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float fr = __shfl_sync(0xffffffffu, f, r * RL);
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
            const float wr = __shfl_sync(0xffffffffu, w, (r * KB + kk) * SH + lane / LD * LD);
            o[r][i * 4] = fmaf(wr, vx.x, o[r][i * 4]); o[r][i * 4 + 1] = fmaf(wr, vx.y, o[r][i * 4 + 1]);
            o[r][i * 4 + 2] = fmaf(wr, vx.z, o[r][i * 4 + 2]); o[r][i * 4 + 3] = fmaf(wr, vx.w, o[r][i * 4 + 3]);
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();                               // the ring becomes the place where the warps' results meet
#pragma unroll
    for (int d = SH; d < RL; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if constexpr (SIDES == 2) {
      l += __shfl_xor_sync(0xffffffffu, l, LD);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] += __shfl_xor_sync(0xffffffffu, o[r][e], LD);
    }
    if (lane < LD && lane % RL == 0) s_ml[warp * R + lane / RL] = make_float2(m, l);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int d = i * 128 + lane * 4;          // of both sides, where there are two, the first one
        if (d < p.dim && lane < LD) *reinterpret_cast<float4*>(s_o + (warp * R + r) * p.dim + d) = make_float4(o[r][i * 4], o[r][i * 4 + 1], o[r][i * 4 + 2], o[r][i * 4 + 3]);
      }
    __syncthreads();
    const int part = part_of(s, blockIdx.x);
    for (int i = tid; i < rows * p.dim; i += FM_WARPS * 32) {
      const int r = i / p.dim, d = i - r * p.dim;
      float top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
      for (int w = 0; w < FM_WARPS; ++w) top = fmaxf(top, s_ml[w * R + r].x);
      const float use = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < FM_WARPS; ++w) {
        const float fw = exp2f(s_ml[w * R + r].x - use);
        sum += s_ml[w * R + r].y * fw;
        val += s_o[(w * R + r) * p.dim + d] * fw;
      }
      RowOut<float>(p, part, b, head0 + r, r, top, sum, d == 0).put(d, val);
    }
    if (s.last >= 0 && tid == 0) p.meta[blockIdx.x] = make_int2(b * p.kv_heads * p.row_tiles + s.sub, s.last);
    __syncthreads();
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

constexpr int MM_COPIERS = 4;                                      // warps that fill the ring

template <int DP, bool TWO> struct MmaShape {
  static constexpr int R = TWO ? 16 : 8;                           // rows: query heads of a tile
  static constexpr int NC = 4;                                     // warps that compute
  static constexpr int THREADS = (NC + MM_COPIERS) * 32;
  static constexpr int KEYS = DP > 128 ? 16 : 32;                  // of a tile
  static constexpr int START = DP > 128 ? 4 : 3;
  static constexpr int LPR = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;   // lanes of a row of the copies
  static constexpr int ROW = ((DP / 8) | 1) * 16;                  // an odd number of 16-byte pieces: ldmatrix without bank conflicts
  static constexpr int SLOT = 2 * KEYS * ROW;                      // keys, then values
  static constexpr int JROW = 40;                                  // floats of a row of 32 values in the join buffers: no bank conflicts
  static constexpr int JOIN = 2 * NC * R * JROW * 4;
  static constexpr int FIXED = JOIN + NC * R * 8 + R * 8 + 64 * 24 + 256;
  // a multiple of the warps: each computing warp shares its slots with one copier, so that no barrier is ever a phase ahead of a waiter
  static constexpr int SLOTS = (232448 - FIXED) / SLOT < 24 ? (232448 - FIXED) / SLOT / 4 * 4 : 24;
  static constexpr int SMEM = SLOTS * SLOT + JOIN + NC * R * 8 + R * 8;
};

// Waits for a barrier's phase; when that takes a second the whole CTA stops waiting, runs through its remaining steps (every access
// stays where it would have been) and reports it.
__device__ __forceinline__ void ring_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
  if (bar_try(bar, parity) || *gave_up) return;
  const long long t0 = clock64();
  while (!bar_try(bar, parity)) {
    if (*gave_up) return;
    if (clock64() - t0 > 2000000000ll) { *gave_up = 1; return; }
  }
}

// 16-bit types: m16n8k16 products.  The query heads of a tile are the 16 rows, a step is 16 or 32 cached keys.  Scores: A = q (registers), B =
// keys; values: A = weights (the score accumulators are already in A's layout), B = values (transposed by ldmatrix).
//
// The weights enter as two 16-bit parts: 22 bits of them for fp16, 17 for bf16.  Up to eight heads leave the upper eight rows free, and
// the low parts ride there (TWO = false); above that they are a second product.  Before its rounding to bf16 an output is off by 1.3 to
// 1.9e-6 (of the norm; a step of bf16 is 4e-3); a third part makes that 3 to 7e-7 and costs 64 sequences of 0..16384 tokens 2 %, 16 heads
// per key head 11 %, so it is left out.
// The products cut the sum that they add to off instead of rounding it.  Each tile's sum therefore starts at zero and is added to the
// running one in a rounded fp32 addition: the running sum as the accumulator drifted towards zero by 2.6e-6 over the longest of
// these sequences, 5.2e-6 with 12 heads per key head, and further with the length (now 2 to 3e-7); one addition per value and tile costs up to 1 %.
//
// Bound by memory where sequences are long: 64 of 0..16384 tokens, 40 / 8 heads of 128, bf16 (2.1 GB) 359 us, 6.0 TB/s; one of 131071 (537 MB)
// 99 us, 5.4 TB/s; 16 of 900..3100 (131 MB) 31.4 us, 4.2 TB/s, of which 3 us pass until the first keys are there and 5 us in the join.  The
// tensor pipe is 15 to 19 % busy: with 5 to 16 rows a product of 128 rows would be mostly empty.
//
// Four warps copy, the others compute.  The copiers walk the tiles of all segments of the CTA into one ring without a stop (cp.async,
// whose arrival the slot's barrier counts), so the loads of the next segment are under way while this one's warps join; tile n goes to
// computing warp n % NC, from copier n % NC.  The warps' results of a segment are added through shared memory, 32 columns at a time.
// With SOLO each pair of a copier and a computing warp is a worker with segments of its own, which it finishes from its registers.
template <typename T, int DP, bool TWO, bool SOLO>
__global__ void __launch_bounds__(MmaShape<DP, TWO>::THREADS, 1) attend_mma_kernel(const AttnParams p) {
  using S = MmaShape<DP, TWO>;
  constexpr int R = S::R, NC = S::NC, NS = S::SLOTS, KEYS = S::KEYS, NT = KEYS / 8;
  static_assert(NS % NC == 0 && NC == MM_COPIERS, "private rings");
  constexpr uint32_t ALL = KEYS == 32 ? 0xffffffffu : 0xffffu;
  constexpr int OV = TWO ? 4 : 2;                                // values of a lane per 8 columns
  constexpr float LIFT = std::is_same<T, __half>::value ? 12.f : 0.f;   // weights up to 2^12: fp16's small numbers begin at 2^-24
  extern __shared__ __align__(128) uint8_t tl_smem[];
  float* s_join = reinterpret_cast<float*>(tl_smem + NS * S::SLOT);
  float2* s_ml = reinterpret_cast<float2*>(tl_smem + NS * S::SLOT + S::JOIN);          // [NC][R] maximum and sum of a warp
  float2* s_row = s_ml + NC * R;                                                        // [R] of the segment
  __shared__ __align__(8) uint64_t s_full[NS], s_empty[NS];
  __shared__ uint32_t s_live[NS];
  __shared__ int64_t s_red[S::THREADS / 32], s_div[2];
  __shared__ int s_gave_up;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = s_u32(tl_smem), full = s_u32(s_full), empty = s_u32(s_empty);
  pdl_trigger();
  if (tid < NS) {
    bar_init(full + tid * 8, 33);        // the copies of 32 lanes, and the word of live keys
    bar_init(empty + tid * 8, 1);
  }
  if (tid == 0) s_gave_up = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_wait();
  auto worker_of_warp = [&] { return (int)(SOLO ? blockIdx.x * NC + (threadIdx.x >> 5) % NC : blockIdx.x); };
  const int stride = SOLO ? 1 : NC;                             // from a tile of this warp's to the next one
  Walk<KEYS, S::START> walk;
  if (p.split) {
    walk.begin_share(p, s_red, s_div, S::THREADS, worker_of_warp(), SOLO ? gridDim.x * NC : gridDim.x);
    if (warp < NC && lane == 0 && (SOLO || warp == 0)) p.meta[worker_of_warp()] = make_int2(-1, 0);
  } else {
    walk.begin_items(p, SOLO ? warp % NC * gridDim.x + blockIdx.x : blockIdx.x);      // over the multiprocessors first
  }
  const int item_step = (SOLO ? NC : 1) * gridDim.x;
  __syncthreads();
  Segment s;

  if (warp >= NC) {
    // ------------------------------------------------------------ copiers
    constexpr int LPR = S::LPR;
    constexpr int STEP = 32 / LPR;                                // rows of an instruction
    const int piece = lane % LPR;
    const bool in_row = piece * 8 < DP, in_dim = piece * 8 < p.dim;   // pieces from dim on are filled with zeros
    const bool one_page = p.page_size % 16 == 0;                  // 16 keys from a multiple of 16 on lie in one page
    int n = SOLO ? 0 : warp - NC, n0 = 0;                       // this warp's next tile; tiles before the segment
    int slot = warp - NC, use = 0;                                // every fourth slot, round by round
    while (walk.next(p, s_div, item_step, &s)) {
      const int h = s.sub / p.row_tiles;
      const T* k_lane = static_cast<const T*>(p.k) + ((int64_t)h * p.k_head + (lane / LPR) * p.k_slot + piece * 8);
      const T* v_lane = static_cast<const T*>(p.v) + ((int64_t)h * p.v_head + (lane / LPR) * p.v_slot + piece * 8);
      const unsigned key0 = s.first / KEYS * KEYS + lane;
      const int count = s.t1 - s.t0;
      int page = 0, place = 0;
      bool ok = n - n0 < count && lane < KEYS && find_key(p, s.b, key0 + (s.t0 + n - n0) * KEYS, s.first, s.end, &page, &place);
      for (; n - n0 < count; n += stride) {
        const uint32_t live = __ballot_sync(0xffffffffu, ok);
        if (use > 0) ring_wait(empty + slot * 8, (use - 1) & 1, &s_gave_up);
        const int page_now = page, place_now = place;
        ok = n + stride - n0 < count && lane < KEYS && find_key(p, s.b, key0 + (s.t0 + n + stride - n0) * KEYS, s.first, s.end, &page, &place);
#pragma unroll
        for (int half = 0; half < KEYS / 16; ++half) {
          const uint32_t dst = ring + slot * S::SLOT + (half * 16 + lane / LPR) * S::ROW + piece * 16;
          if (one_page && (live >> (half * 16) & 0xffffu) == 0xffffu) {   // one address and a fixed step
            const int64_t pg = __shfl_sync(0xffffffffu, page_now, half * 16), pl = __shfl_sync(0xffffffffu, place_now, half * 16);
            const T* kp = k_lane + (pg * p.k_page + pl * p.k_slot);
            const T* vp = v_lane + (pg * p.v_page + pl * p.v_slot);
            if (!in_dim) { kp = k_lane; vp = v_lane; }
            if (in_row) {
#pragma unroll
              for (int i = 0; i < 16 / STEP; ++i) {
                cp_async(dst + i * STEP * S::ROW, kp, in_dim);
                kp += STEP * p.k_slot;
              }
#pragma unroll
              for (int i = 0; i < 16 / STEP; ++i) {
                cp_async(dst + (KEYS + i * STEP) * S::ROW, vp, in_dim);
                vp += STEP * p.v_slot;
              }
            }
          } else {
#pragma unroll 4
            for (int i = 0; i < 16 / STEP; ++i) {
              const int row = half * 16 + i * STEP + lane / LPR;
              const int64_t pg = __shfl_sync(0xffffffffu, page_now, row), pl = __shfl_sync(0xffffffffu, place_now, row) - lane / LPR;
              const bool on = in_dim && (live >> row & 1);
              if (in_row) {                                       // rows that are not live are filled with zeros
                cp_async(dst + i * STEP * S::ROW, on ? k_lane + (pg * p.k_page + pl * p.k_slot) : k_lane, on);
                cp_async(dst + (KEYS + i * STEP) * S::ROW, on ? v_lane + (pg * p.v_page + pl * p.v_slot) : v_lane, on);
              }
            }
          }
        }
        if (lane == 0) {
          s_live[slot] = live;
          bar_arrive(full + slot * 8);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full + slot * 8) : "memory");
        slot += MM_COPIERS;
        if (slot >= NS) { slot -= NS; ++use; }
      }
      n0 += count;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (lane == 0 && *(volatile int*)&s_gave_up) atomicExch(&g_attend_status, 1);
    return;
  }

  // -------------------------------------------------------------- computing warps
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t k_at = ring + ((lane >> 4) * 8 + (lane & 7)) * S::ROW + (lane >> 3 & 1) * 16;
  const uint32_t v_at = ring + (KEYS + (lane >> 3 & 1) * 8 + (lane & 7)) * S::ROW + (lane >> 4) * 16;
  uint32_t q[DP / 16][TWO ? 4 : 2];
  int n0 = 0, n = SOLO ? 0 : warp, slot = warp, use = 0;
  bool more = walk.next(p, s_div, item_step, &s);
  auto load_q = [&]() {
    const int h = s.sub / p.row_tiles, x = s.sub - h * p.row_tiles;
    const int head0 = h * p.group + x * p.rows, rows = min(p.rows, p.group - x * p.rows);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int i = 0; i < (TWO ? 4 : 2); ++i) {
        const int r = TWO ? g + (i & 1) * 8 : g, d = ks * 16 + t4 * 2 + (TWO ? i >> 1 : i) * 8;
        q[ks][i] = 0;
        if (r < rows && d < p.dim) {
          const T* src = static_cast<const T*>(p.q) + ((int64_t)s.b * p.q_b + (int64_t)(head0 + r) * p.q_h + d);
          q[ks][i] = p.q_words ? *reinterpret_cast<const uint32_t*>(src) : bits_of<T>(src[0], src[1]);
        }
      }
  };
  if (more) load_q();
  while (more) {
    const Segment now = s;
    const int count = now.t1 - now.t0;
    float o[DP / 8][OV];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < OV; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};       // rows g and g + 8, m less LIFT; l: of the lane's own keys

    for (; n - n0 < count; n += stride) {
      ring_wait(full + slot * 8, use & 1, &s_gave_up);
      const uint32_t live = s_live[slot];
      const uint32_t off = slot * S::SLOT;
      float c[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[nt][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        {
          uint32_t kb[KEYS / 16][4];
#pragma unroll
          for (int j = 0; j < KEYS / 16; ++j) ldsm4(kb[j], k_at + off + ks * 32 + j * 16 * S::ROW);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint32_t b0 = kb[nt >> 1][2 * (nt & 1)], b1 = kb[nt >> 1][2 * (nt & 1) + 1];
            if constexpr (TWO) mma16816<T>(c[nt], q[ks][0], q[ks][1], q[ks][2], q[ks][3], b0, b1);
            else mma16816<T>(c[nt], q[ks][0], 0u, q[ks][1], 0u, b0, b1);
          }
        }
      }
      uint32_t hi[KEYS / 16][4], lo[KEYS / 16][4];                              // weights as A: [16 keys][register]
#pragma unroll
      for (int half = 0; half < (TWO ? 2 : 1); ++half) {
        float sc[2 * NT];
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
          sc[i] = c[i >> 1][half * 2 + (i & 1)] * p.scale;
          if (p.cap > 0.f) sc[i] = p.cap * AT_LOG2E * tanhf(sc[i] / p.cap);
        }
        if (live != ALL) {
#pragma unroll
          for (int i = 0; i < 2 * NT; ++i)
            if (!(live >> ((i >> 1) * 8 + t4 * 2 + (i & 1)) & 1)) sc[i] = -INFINITY;
        }
        float tops[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) tops[nt] = fmaxf(sc[2 * nt], sc[2 * nt + 1]);
        float top = fmaxf(tops[0], tops[1]);
        if constexpr (NT == 4) top = fmaxf(top, fmaxf(tops[2], tops[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[half], top - LIFT);
        const float base = mn == -INFINITY ? 0.f : mn;
        if (__any_sync(0xffffffffu, mn > m[half])) {              // a new maximum in some row: rescale what is there
          const float f = ex2(m[half] - base);
          l[half] *= f;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) { o[i][2 * half] *= f; o[i][2 * half + 1] *= f; }
        }
        m[half] = mn;
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) sc[i] = ex2(sc[i] - base);
        l[half] += (sc[0] + sc[1]) + (sc[2] + sc[3]);
        if constexpr (NT == 4) l[half] += (sc[4] + sc[5]) + (sc[6] + sc[7]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) split_pair<T>(sc[2 * nt], sc[2 * nt + 1], hi[nt >> 1][2 * (nt & 1) + half], lo[nt >> 1][2 * (nt & 1) + half]);
      }
#pragma unroll
      for (int cc = 0; cc < DP / 16; ++cc) {
        float sum[2][4] = {};                                     // of this tile
#pragma unroll
        for (int j = 0; j < KEYS / 16; ++j) {
          uint32_t vb[4];
          ldsm4_t(vb, v_at + off + cc * 32 + j * 16 * S::ROW);
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            if constexpr (TWO) {
              mma16816<T>(sum[n2], hi[j][0], hi[j][1], hi[j][2], hi[j][3], vb[2 * n2], vb[2 * n2 + 1]);
              mma16816<T>(sum[n2], lo[j][0], lo[j][1], lo[j][2], lo[j][3], vb[2 * n2], vb[2 * n2 + 1]);
            } else {
              mma16816<T>(sum[n2], hi[j][0], lo[j][0], hi[j][2], lo[j][2], vb[2 * n2], vb[2 * n2 + 1]);
            }
          }
        }
#pragma unroll
        for (int n2 = 0; n2 < 2; ++n2) {
          if constexpr (!TWO) { sum[n2][0] += sum[n2][2]; sum[n2][1] += sum[n2][3]; }      // high and low parts
#pragma unroll
          for (int e = 0; e < OV; ++e) o[2 * cc + n2][e] += sum[n2][e];
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(empty + slot * 8);
      slot += NC;
      if (slot >= NS) { slot -= NS; ++use; }
    }
    n0 += count;
    more = walk.next(p, s_div, item_step, &s);
    if (more) load_q();                                           // arrives while the warps join

#pragma unroll
    for (int half = 0; half < (TWO ? 2 : 1); ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
      if (t4 == 0) s_ml[warp * R + g + half * 8] = make_float2(m[half], l[half]);
    }
    const int h = now.sub / p.row_tiles, x = now.sub - h * p.row_tiles;
    const int head0 = h * p.group + x * p.rows, rows = min(p.rows, p.group - x * p.rows);
    const int part = part_of(now, worker_of_warp());
    if (now.last >= 0 && lane == 0 && (SOLO || warp == 0)) p.meta[worker_of_warp()] = make_int2(now.b * p.kv_heads * p.row_tiles + now.sub, now.last);
    if constexpr (SOLO) {
#pragma unroll
      for (int half = 0; half < (TWO ? 2 : 1); ++half) {
        const int r = g + half * 8;
        if (r < rows) {
          const RowOut<T> out(p, part, now.b, head0 + r, r, m[half], l[half], t4 == 0);
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            const int d = i * 8 + t4 * 2;
            if (d < p.dim) out.put2(d, o[i][2 * half], o[i][2 * half + 1]);
          }
        }
      }
      continue;
    }
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(NC * 32) : "memory"); };
    meet();
    float f[2] = {0.f, 0.f};
#pragma unroll
    for (int half = 0; half < (TWO ? 2 : 1); ++half) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < NC; ++w) top = fmaxf(top, s_ml[w * R + g + half * 8].x);
      f[half] = ex2(m[half] - (top == -INFINITY ? 0.f : top));
    }
    if (tid < R) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < NC; ++w) top = fmaxf(top, s_ml[w * R + tid].x);
#pragma unroll
      for (int w = 0; w < NC; ++w) sum += s_ml[w * R + tid].y * ex2(s_ml[w * R + tid].x - (top == -INFINITY ? 0.f : top));
      s_row[tid] = make_float2(top, sum);
    }
    auto lay_down = [&](int sl) {
      float* buf = s_join + (sl & 1) * (NC * R * S::JROW) + (warp * R + g) * S::JROW + t4 * 2;
#pragma unroll
      for (int half = 0; half < (TWO ? 2 : 1); ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int nt = sl * 4 + i;
          *reinterpret_cast<float2*>(buf + half * 8 * S::JROW + i * 8) = make_float2(o[nt][2 * half] * f[half], o[nt][2 * half + 1] * f[half]);
        }
    };
    lay_down(0);
    meet();
    RowOut<T> out[R / NC] = {};
#pragma unroll
    for (int e = 0; e < R / NC; ++e) {
      const int r = e * NC + warp;
      const float2 ml = s_row[r];
      if (r < rows) out[e] = RowOut<T>(p, part, now.b, head0 + r, r, ml.x, ml.y, lane == 0);
    }
#pragma unroll
    for (int sl = 0; sl < DP / 32; ++sl) {
      if (sl > 0) meet();
      const float* buf = s_join + (sl & 1) * (NC * R * S::JROW);
#pragma unroll
      for (int e = 0; e < R / NC; ++e) {
        const int r = e * NC + warp, d = sl * 32 + lane;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NC; ++w) sum += buf[(w * R + r) * S::JROW + lane];
        if (r < rows && d < p.dim) out[e].put(d, sum);
      }
      if (sl + 1 < DP / 32) lay_down(sl + 1);
    }
  }
}

template <typename T>
int launch_both(void (*kern)(const AttnParams), AttnParams& p, int threads, int smem, int ctas_per_sm, cudaStream_t st) {
  const bool pdl = options().pdl != 0;
  const int64_t items = (int64_t)p.batch * p.kv_heads * p.row_tiles;
  const unsigned grid = (unsigned)(p.split || p.solo ? sm_count() * ctas_per_sm : items);
  KQ_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(threads), (size_t)smem, st, pdl, p));
  options().launches += 1;
  if (p.split) {
    KQ_CUDA_TRY(launch_pdl(attend_join_kernel<T>, dim3(grid, (unsigned)p.rows), dim3((p.solo ? 4 : 1) * (p.dim > 128 ? 128 : 64)), (size_t)0, st, pdl, p));
    options().launches += 1;
  }
  return KQ_OK;
}

template <int R, int LD, int NI, int STAGES, int KB, int CTAS, int LEAST>
int run_fma(AttnParams& p, cudaStream_t st) {
  constexpr int ring = FM_WARPS * STAGES * 2 * KB * NI * 512, join = FM_WARPS * R * NI * 128 * 4;
  constexpr int smem = ring > join ? ring : join;
  static_assert(CTAS <= (NI == 2 ? 2 : FM_MOST), "more workers than scratch_of counts");
  auto kern = attend_fma_kernel<R, LD, NI, STAGES, KB, LEAST>;
  static DeviceOnce attr_set;
  if (attr_set.first_time()) {
    KQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_set.done();
  }
  return launch_both<float>(kern, p, FM_WARPS * 32, smem, CTAS, st);
}

template <typename T, int DP, bool TWO>
int run_mma(AttnParams& p, cudaStream_t st) {
  using S = MmaShape<DP, TWO>;
  static DeviceOnce attr_set;
  if (attr_set.first_time()) {
    KQ_CUDA_TRY(cudaFuncSetAttribute(attend_mma_kernel<T, DP, TWO, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    KQ_CUDA_TRY(cudaFuncSetAttribute(attend_mma_kernel<T, DP, TWO, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    attr_set.done();
  }
  return launch_both<T>(p.solo ? attend_mma_kernel<T, DP, TWO, true> : attend_mma_kernel<T, DP, TWO, false>, p, S::THREADS, S::SMEM, 1, st);
}

// the query heads of a key head in tiles of at most `most` rows, of even sizes
void set_rows(AttnParams& p, int most) {
  p.row_tiles = (p.group + most - 1) / most;
  p.rows = (p.group + p.row_tiles - 1) / p.row_tiles;
  p.row_tiles = (p.group + p.rows - 1) / p.rows;
}

// Tiles of up to 4 or 8 rows.  Bound by instruction issue, so the tile, the ring and the registers are those that keep most warps busy;
// us before (tiles of 32 / R keys, a warp per key, two CTAs) / as chosen, 16 sequences of 4000 tokens, 8 key heads: heads of 64 in
// groups of 4 103 / 58, of 8 197 / 86; heads of 128 in groups of 8 197 / 139 (2.7 / 3.8 TB/s); 33 sequences of up to 10000 with heads
// of 256 in groups of 4 120 / 104; listed in turn: stages, keys side by side, CTAs per multiprocessor, and those that the registers must allow
// (at least; with 155 instead of 128 registers <4, 32, 1> takes 72 instead of 60 us for 16 sequences of 900..3100).
int run_f32(AttnParams& p, cudaStream_t st) {
  set_rows(p, 8);
  if (p.rows <= 4)
    return p.dim > 128 ? run_fma<4, 32, 2, 3, 4, 2, 2>(p, st) : p.dim > 64 ? run_fma<4, 32, 1, 2, 8, 2, 4>(p, st) : run_fma<4, 16, 1, 2, 4, 4, 4>(p, st);
  return p.dim > 128 ? run_fma<8, 32, 2, 3, 4, 2, 2>(p, st) : p.dim > 64 ? run_fma<8, 32, 1, 2, 4, 3, 3>(p, st) : run_fma<8, 16, 1, 2, 2, 4, 4>(p, st);
}

// From how many items on a worker is a warp.  As warps / as CTAs, us, 148 multiprocessors: 256 sequences of 1..500 tokens with 8 key heads
// 59.3 / 88.8, 64 of 1..1000 34.4 / 41.8, 64 of 4096 187.9 / 185.7, 16 of 900..3100 (128 items) 31.4 / 32.7, 16 of 4000 with heads of 64 31.8 / 37.9;
// 66 items of 100..7001 with heads of 256 57.0 / 53.8, 64 items of 8000 59.2 / 54.5, 8 items of 131071 102.7 / 98.7: few items are cut into
// many more parts.  Short lengths need no division, and no join: each item is a CTA's, or above one per multiprocessor a warp's: 1024 items of
// 1..200 19.8 / 37.4 (divided all the same: 21.4), 408 of 55 with heads of 256 9.6 / 19.0 (16.9), 160 of 1..60 6.3 / 9.1 (8.9); 96 items
// of 200 10.6 / 6.8.
bool solo_pays(int64_t items, bool split) { return split ? 4 * items >= 3 * (int64_t)sm_count() : items > (int64_t)sm_count(); }

template <typename T>
int run_16bit(AttnParams& p, cudaStream_t st) {
  set_rows(p, 16);
  p.solo = solo_pays((int64_t)p.batch * p.kv_heads * p.row_tiles, p.split);
  if (p.rows <= 8)
    return p.dim <= 64 ? run_mma<T, 64, false>(p, st) : p.dim <= 96 ? run_mma<T, 96, false>(p, st) : p.dim <= 128 ? run_mma<T, 128, false>(p, st)
         : p.dim <= 192 ? run_mma<T, 192, false>(p, st) : run_mma<T, 256, false>(p, st);
  return p.dim <= 64 ? run_mma<T, 64, true>(p, st) : p.dim <= 96 ? run_mma<T, 96, true>(p, st) : p.dim <= 128 ? run_mma<T, 128, true>(p, st)
       : p.dim <= 192 ? run_mma<T, 192, true>(p, st) : run_mma<T, 256, true>(p, st);
}

struct Scratch { size_t o, ml, meta, total; };
Scratch scratch_of(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
  AttnParams p;
  p.group = (int)(heads / kv_heads);
  set_rows(p, 16);
  const int64_t rows = p.rows > 8 ? p.rows : 8;              // of either type's tiles
  const int64_t workers = sm_count() * (solo_pays(batch * kv_heads * p.row_tiles, true) || dim <= 128 ? FM_MOST : 2);   // fp32 heads above 128 have two
  auto up = [](int64_t bytes) { return (size_t)((bytes + 255) / 256 * 256); };
  Scratch s;
  s.o = 0;
  s.ml = s.o + up(2 * workers * rows * dim * 4);
  s.meta = s.ml + up(2 * workers * rows * 8);
  s.total = s.meta + up(workers * 8);
  return s;
}

}  // namespace

}  // namespace kq

using namespace kq;

extern "C" {

static bool attention_sizes_ok(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  return batch >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0 &&
         batch <= (1 << 20) && heads <= (1 << 16) && batch * heads <= 0x7fffffff;
}

size_t kq_paged_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  return attention_sizes_ok(batch, heads, kv_heads, head_dim) ? scratch_of(batch, heads, kv_heads, head_dim).total : 0;
}

int kq_paged_attention(const void* q, int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t q_stride_batch,
                       int64_t q_stride_head, const void* k_cache, const int64_t* k_strides, const void* v_cache,
                       const int64_t* v_strides, int64_t num_pages, int64_t page_size, const int32_t* block_table, int64_t table_stride,
                       int64_t table_width, const int32_t* seq_lens, float scale, int64_t window, float softcap, void* out, float* lse,
                       void* scratch, size_t scratch_bytes, void* stream) {
  const char* fn = "kq_paged_attention";
  clear_error();
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
  // up to 1e30, so that neither overflows when multiplied by log2(e), nor score / softcap leaves fp32's normal numbers
  if (!(scale > 0.f) || scale > 1e30f || !(softcap >= 0.f) || softcap > 1e30f) { set_error("%s: scale must be positive and softcap not negative, both at most 1e30", fn); return KQ_EINVAL; }
  if (batch == 0) return KQ_OK;
  if (!q || !out || !seq_lens || (table_width > 0 && !block_table) || (num_pages > 0 && (!k_cache || !v_cache)) || !k_strides || !v_strides) {
    set_error("%s: null pointer", fn);
    return KQ_EINVAL;
  }
  const int64_t size = dtype == KQ_F32 ? 4 : 2;
  const int64_t extent[3] = {num_pages, page_size, kv_heads};
  int64_t ks[3], vs[3];
  for (int i = 0; i < 3; ++i) {
    ks[i] = extent[i] > 1 ? k_strides[i] : 0;          // a stride that no step follows may be anything
    vs[i] = extent[i] > 1 ? v_strides[i] : 0;
    if (ks[i] < 0 || vs[i] < 0 || ks[i] * size % 16 || vs[i] * size % 16) {
      set_error("%s: cache strides must be multiples of 16 bytes", fn);
      return KQ_EINVAL;
    }
  }
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)q % size || (uintptr_t)out % 16 || ((uintptr_t)block_table | (uintptr_t)seq_lens | (uintptr_t)lse) % 4) {
    set_error("%s: misaligned pointer", fn);
    return KQ_EINVAL;
  }
  // several workers read a row of q, and any of them the caches
  if (out == q || out == k_cache || out == v_cache || lse == out) { set_error("%s: out must be neither an input nor lse", fn); return KQ_EINVAL; }
  const Scratch L = scratch_of(batch, heads, kv_heads, head_dim);
  if (!scratch || (uintptr_t)scratch % 256) { set_error("%s: scratch must be non-null and 256-byte aligned", fn); return KQ_ESCRATCH; }
  if (scratch_bytes < L.total) { set_error("%s: scratch too small (%zu < %zu)", fn, scratch_bytes, L.total); return KQ_ESCRATCH; }

  AttnParams p;
  p.q = q; p.q_b = q_stride_batch; p.q_h = q_stride_head; p.q_words = !((uintptr_t)q % 4 || q_stride_batch % 2 || q_stride_head % 2);
  p.k = k_cache; p.k_page = ks[0]; p.k_slot = ks[1]; p.k_head = ks[2];
  p.v = v_cache; p.v_page = vs[0]; p.v_slot = vs[1]; p.v_head = vs[2];
  p.table = block_table; p.table_b = table_stride; p.width = (int)table_width; p.lens = seq_lens;
  p.batch = (int)batch; p.heads = (int)heads; p.kv_heads = (int)kv_heads; p.group = (int)(heads / kv_heads); p.dim = (int)head_dim;
  p.page_size = (int)page_size; p.num_pages = num_pages;
  p.scale = softcap > 0.f ? scale : scale * AT_LOG2E; p.cap = softcap; p.window = (int)window;
  p.out = out; p.lse = lse;
  uint8_t* sb = (uint8_t*)scratch;
  p.part_o = (float*)(sb + L.o); p.part_ml = (float2*)(sb + L.ml); p.meta = (int2*)(sb + L.meta);
  p.solo = 0;
  int64_t most = table_width * page_size;          // keys that a sequence can show
  if (window > 0 && window < most) most = window;
  // Short sequences: one launch.  Up to 1024 instead of 256 keys, divided / whole, us: 64 sequences of 1..500 with 8 key heads 23.7 / 20.6, 24 of
  // them 13.7 / 17.7, 128 of 1..1000 58.3 / 66.0
  p.split = most > 256;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case KQ_F32: return run_f32(p, st);
    case KQ_F16: return run_16bit<__half>(p, st);
    default: return run_16bit<__nv_bfloat16>(p, st);
  }
}

int kq_paged_attention_status(int* status, int clear) {
  clear_error();
  KQ_CUDA_TRY(cudaDeviceSynchronize());   // the copy does not wait for non-blocking streams
  int v = 0;
  KQ_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_attend_status, sizeof(int)));
  if (status) *status = v;
  if (clear && v) { const int z = 0; KQ_CUDA_TRY(cudaMemcpyToSymbol(g_attend_status, &z, sizeof(int))); }
  return KQ_OK;
}

}  // extern "C"
