// Rotary positions, and the append to the 8-bit key/value cache.
//
// Rotation: the first rotary_dim values of a head are pairs (i, i + rotary_dim / 2) ("half") or (2i, 2i + 1)
// ("interleaved"); a pair (a, b) at position p becomes (a c - b s, b c + a s) with c, s = magnitude * cos, sin(p * freq[i]);
// the rest of the head is passed on. cos and sin come from an angle in turns (block_common.h), once per token and pair, and
// are shared by all heads of the token through shared memory. fp32 arithmetic, one rounding at the store.
//
// Append: token i of the n new tokens of a sequence has position kv_len - n + i and lies in page
// table[sequence][position / 64]. One CTA owns one page of one head, keys and values: it turns the keys, takes the largest
// finite |value| of the page's new tokens, chooses the page's scale (the smallest power of two that brings it into e4m3's
// range; never below the scale that earlier tokens of the page were stored with), stores the tokens, and re-scales the
// earlier ones if the scale grew. A page without earlier tokens is filled up with zeros, so that no page holds bytes that were
// never written. Infinities are stored as the largest value of the page's scale. A key that is NaN stays NaN; a value that is
// NaN is stored as 0 and makes the token's key NaN, so that exactly the queries that see the token get NaN and a masked
// token never reaches the product of weights and values.
#include "block_common.h"
#include "kernels.h"

#include <type_traits>

namespace {

using namespace ob_block;

__device__ int g_append_batch;   // see note_bad_batch

struct Rotation {
  const double* freq;          // rotary_dim / 2 angular frequencies
  int half;                    // rotary_dim / 2
  int interleaved;
  float magnitude;
};

struct RotaryArgs {
  const void* x;
  void* y;
  int64_t x_ts, x_hs, y_ts, y_hs;      // elements from one token / head to the next
  const void* positions;               // per token; null: from the batch
  int positions_i64;
  int tokens, heads, head_dim;
  Rotation rot;
};

struct BatchArgs {
  const int* q_start;
  const int* kv_len;
  const int* table;
  int64_t table_stride;
  int table_width, seqs;
};

struct AppendArgs {
  const void *k, *v;
  int64_t k_ts, k_hs, v_ts, v_hs;
  uint8_t *k_pages, *v_pages;
  float *k_scale, *v_scale;
  int64_t pages;
  int kv_heads;
  BatchArgs b;
  Rotation rot;                        // half = 0: keys are stored as they come
  int tokens;
  int page_slots;                      // CTAs of the append half of the grid: page slots x kv_heads
  int least_new, most_new;             // this launch has the sequences with so many new tokens, least_new >= 1
};

constexpr int kAppendTokens = 4, kFewTokens = 4;   // query tokens per CTA of an append: with prompts, with steps
constexpr int kRotThreads = 256;
constexpr int kMaxHalf = 256;
constexpr int kBatch = 4;              // pieces that a thread has under way

// pair i of the head at p: values a, b at offsets (oa, ob)
__device__ __forceinline__ void pair_at(const Rotation& r, int i, int& oa, int& ob) {
  oa = r.interleaved ? 2 * i : i;
  ob = r.interleaved ? 2 * i + 1 : i + r.half;
}

// The heads of up to TOKENS tokens, from the table of their cos and sin in shared memory. A head is cut into pieces, a thread
// keeps its piece and goes from head to head. W = 8: pieces of 8 values (the rotated ones of "half" with their partners), kBatch
// of them loaded before the first is stored; in place, a piece is read and written by its own thread only. make_table() (all
// threads; ends with a barrier) fills cs and skip while the first pieces are on their way.
template <typename T, int W, int THREADS, int TOKENS, typename F>
__device__ __forceinline__ void rotate_tokens(const RotaryArgs& a, int t0, int n, const float2 (&cs)[TOKENS][kMaxHalf], const bool (&skip)[TOKENS], F make_table) {
  const Rotation& r = a.rot;
  const int pairs_per = W == 1 ? 1 : (r.interleaved ? W / 2 : W);
  const int turning = r.half / pairs_per;
  const int passing = a.x == a.y ? 0 : (a.head_dim - 2 * r.half) / W;
  const int per_head = turning + passing;
  if (per_head == 0) return;                                   // nothing is turned and the rest is there already
  if constexpr (W == 1) {
    make_table();
    for (int u = threadIdx.x; u < n * a.heads * per_head; u += THREADS) {
      const int piece = u % per_head, th = u / per_head, head = th % a.heads, tt = th / a.heads;
      if (skip[tt]) continue;
      const T* x = static_cast<const T*>(a.x) + (int64_t)(t0 + tt) * a.x_ts + (int64_t)head * a.x_hs;
      T* y = static_cast<T*>(a.y) + (int64_t)(t0 + tt) * a.y_ts + (int64_t)head * a.y_hs;
      if (piece >= turning) {
        y[2 * r.half + piece - turning] = x[2 * r.half + piece - turning];
        continue;
      }
      int oa, ob;
      pair_at(r, piece, oa, ob);
      const float2 c = cs[tt][piece];
      const float va = to_f32(x[oa]), vb = to_f32(x[ob]);
      y[oa] = from_f32<T>(va * c.x - vb * c.y);
      y[ob] = from_f32<T>(vb * c.x + va * c.y);
    }
  } else {
    const int rows = THREADS / per_head;                       // heads that the CTA takes at once; a head has at most 64 pieces
    const int piece = threadIdx.x % per_head;
    int head = threadIdx.x / per_head, tt = head < rows ? 0 : n;   // threads left over take none
    while (head >= a.heads) { head -= a.heads; ++tt; }
    const bool turn = piece < turning, pairs = turn && !r.interleaved;
    const int o0 = turn ? piece * 8 : 2 * r.half + (piece - turning) * 8;
    for (bool first = true; first || tt < n; first = false) {
      uint4 va[kBatch], vb[kBatch];
      int64_t at[kBatch];
      int tok[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        tok[i] = tt < n ? tt : -1;
        at[i] = (int64_t)(t0 + tt) * a.y_ts + (int64_t)head * a.y_hs + o0;
        if (tt < n) {
          const T* x = static_cast<const T*>(a.x) + (int64_t)(t0 + tt) * a.x_ts + (int64_t)head * a.x_hs + o0;
          va[i] = *reinterpret_cast<const uint4*>(x);
          if (pairs) vb[i] = *reinterpret_cast<const uint4*>(x + r.half);
        }
        head += rows;
        while (head >= a.heads) { head -= a.heads; ++tt; }
      }
      if (first) make_table();
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (tok[i] < 0 || skip[tok[i]]) continue;
        T* y = static_cast<T*>(a.y) + at[i];
        if (!turn) {
          *reinterpret_cast<uint4*>(y) = va[i];
        } else if (r.interleaved) {
          const float4* c4 = reinterpret_cast<const float4*>(&cs[tok[i]][piece * 4]);       // cos, sin of two pairs
          const uint32_t w[4] = {va[i].x, va[i].y, va[i].z, va[i].w};
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 c = c4[e / 2];
            const float2 v = unpack2(w[e], T{});
            const float cc = e & 1 ? c.z : c.x, ss = e & 1 ? c.w : c.y;
            o[e] = pack2(v.x * cc - v.y * ss, v.y * cc + v.x * ss, T{});
          }
          *reinterpret_cast<uint4*>(y) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
          const float4* c4 = reinterpret_cast<const float4*>(&cs[tok[i]][piece * 8]);
          const uint32_t w[4] = {va[i].x, va[i].y, va[i].z, va[i].w}, z[4] = {vb[i].x, vb[i].y, vb[i].z, vb[i].w};
          uint32_t o[4], q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 c = c4[e];
            const float2 v = unpack2(w[e], T{}), u = unpack2(z[e], T{});
            o[e] = pack2(v.x * c.x - u.x * c.y, v.y * c.z - u.y * c.w, T{});
            q[e] = pack2(u.x * c.x + v.x * c.y, u.y * c.z + v.y * c.w, T{});
          }
          *reinterpret_cast<uint4*>(y) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(y + r.half) = make_uint4(q[0], q[1], q[2], q[3]);
        }
      }
    }
  }
}

template <int THREADS, int TOKENS>
__device__ __forceinline__ void fill_cos_sin(const Rotation& r, const int64_t (&pos)[TOKENS], int n, float2 (&cs)[TOKENS][kMaxHalf]) {
  for (int i = threadIdx.x % 64; i < r.half; i += 64)          // 64 pairs of each of THREADS / 64 tokens at a time
    for (int tt = threadIdx.x / 64; tt < n; tt += THREADS / 64) cs[tt][i] = cos_sin(turns_per_position(r.freq[i]), pos[tt], r.magnitude);
}

template <typename T, int W, int TOKENS> __global__ void __launch_bounds__(kRotThreads, 4) ob_rotary_kernel(const RotaryArgs a) {
  follow_previous_kernel();
  __shared__ __align__(16) float2 cs[TOKENS][kMaxHalf];
  __shared__ int64_t pos[TOKENS];
  __shared__ bool skip[TOKENS];
  const int t0 = blockIdx.x * TOKENS, n = min(TOKENS, a.tokens - t0);
  rotate_tokens<T, W, kRotThreads>(a, t0, n, cs, skip, [&] {
    if (threadIdx.x < n) {
      pos[threadIdx.x] = a.positions_i64 ? static_cast<const int64_t*>(a.positions)[t0 + threadIdx.x]
                                         : (int64_t) static_cast<const int*>(a.positions)[t0 + threadIdx.x];
      skip[threadIdx.x] = false;
    }
    __syncthreads();
    fill_cos_sin<kRotThreads>(a.rot, pos, n, cs);
    __syncthreads();
  });
}

__device__ __forceinline__ float finite_max(float m, float v) {
  v = fabsf(v);
  return v <= 3.402823466e38f ? fmaxf(m, v) : m;
}

// the largest value of the CTA's threads
template <int THREADS> __device__ __forceinline__ float cta_max(float v, float (&red)[THREADS / 32]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v = fmaxf(v, red[w]);
  return v;
}

// the larger magnitudes of two pairs of values; a NaN stays
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b, __half) {
  const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), __habs2(*reinterpret_cast<const __half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// 2 D threads: 16 groups of 4 tokens (a word of the transposed values) x D / 8 groups of 8 values. The grid is in two halves:
// 8 prompts of up to 2048 tokens (8 heads of 128, 32 query heads) take 44.1 us, of which the queries alone are 30 (the rate of the
// rotation by itself) and the pages' instructions the rest; the pages among the queries instead of before them: 44.9 us. At 80
// registers three CTAs of 256 threads share an SM and a thread has all kBatch pieces of 4 tokens' queries under way; four CTAs at
// 64 registers spill (49.2 us, with two tokens 46.7), two at 128 are too few (50.3 us).
template <typename T, int D, int W>
__global__ void __launch_bounds__(2 * D, 768 / (2 * D)) ob_cache_append_kernel(const AppendArgs a, const RotaryArgs q) {
  follow_previous_kernel();
  constexpr int kThreads = 2 * D;
  __shared__ __align__(16) float2 cs[kPageTokens][D / 2];
  __shared__ float red[2][kThreads / 32];
  __shared__ int nan_token[kPageTokens];
  __shared__ int found[kThreads / 32][kAppendTokens];
  const int tid = threadIdx.x;
  const BatchArgs& b = a.b;
  const Starts starts{b.q_start, b.seqs, a.tokens};

  // the CTAs of pages come first: they are the longer ones
  const int items = a.page_slots * a.kv_heads;
  if ((int)blockIdx.x >= items) {
    // ---- queries: up to kAppendTokens tokens ----
    auto& qcs = reinterpret_cast<float2(&)[kAppendTokens][kMaxHalf]>(cs);
    static_assert(sizeof(cs) >= sizeof(float2) * kAppendTokens * kMaxHalf, "the queries' table lies in the keys'");
    __shared__ int64_t pos[kAppendTokens];
    __shared__ bool skip[kAppendTokens];
    const int t0 = ((int)blockIdx.x - items) * kAppendTokens, n = min(kAppendTokens, q.tokens - t0);
    rotate_tokens<T, W, kThreads>(q, t0, n, qcs, skip, [&] {
      int c[kAppendTokens];                                      // sequence c - 1 holds the token
      bool bad = false;
#pragma unroll
      for (int tt = 0; tt < kAppendTokens; ++tt) c[tt] = b.seqs + 1;
      for (int s = tid; s <= b.seqs; s += kThreads) {
        const int start = starts.at(s, bad);
#pragma unroll
        for (int tt = 0; tt < kAppendTokens; ++tt) c[tt] = min(c[tt], starts.behind_row(s, start, t0 + tt));
      }
#pragma unroll
      for (int tt = 0; tt < kAppendTokens; ++tt) {
        c[tt] = __reduce_min_sync(~0u, c[tt]);
        if ((tid & 31) == 0) found[tid >> 5][tt] = c[tt];
      }
      bad = __syncthreads_or(bad);
      if (tid < n) {
        int c = found[0][tid];
        for (int w = 1; w < kThreads / 32; ++w) c = min(c, found[w][tid]);
        skip[tid] = c < 1 || c > b.seqs || (bad && starts.left_out(c - 1));     // before the first or behind the last sequence
        pos[tid] = skip[tid] ? 0 : (int64_t)b.kv_len[c - 1] - b.q_start[c] + t0 + tid;
      }
      __syncthreads();
      fill_cos_sin<kThreads>(q.rot, pos, n, qcs);
      __syncthreads();
    });
    return;
  }

  // ---- pages of one head ----
  // Sequence s owns the slots [floor(q_start[s] / 64) + s, floor(q_start[s+1] / 64) + s + 1): at least floor(n / 64) + 1. n tokens
  // touch at most one page more than that, which the first slot then takes too.
  const int head = (int)blockIdx.x % a.kv_heads, slot = (int)blockIdx.x / a.kv_heads;
  int c = min(b.seqs, slot + 1);                              // sequence c - 1 has the slot
  bool bad = false;
  for (int s = tid; s < b.seqs; s += kThreads) {
    const int start = starts.at(s, bad);
    c = min(c, starts.behind_slot(s, start, slot, start / kPageTokens));
  }
  c = __reduce_min_sync(~0u, c);
  if ((tid & 31) == 0) found[tid >> 5][0] = c;
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) c = min(c, found[w][0]);
  if (bad && blockIdx.x == 0 && tid == 0) note_bad_batch(&g_append_batch);
  const int seq = c - 1;
  if (seq < 0) return;
  if (bad && starts.left_out(seq)) return;
  const int q0 = b.q_start[seq], q1 = b.q_start[seq + 1], kv = b.kv_len[seq], n = q1 - q0;
  if (n < a.least_new || n > a.most_new || kv <= 0) return;
  const int before = kv - n;                                  // may be negative: the first -before tokens have no place
  const int mine = slot - (q0 / kPageTokens + seq), slots = q1 / kPageTokens + seq + 1 - (q0 / kPageTokens + seq);
  const Rotation& r = a.rot;
  constexpr int kVecs = D / 8;
  const int quad = (tid & 7) + 8 * ((tid >> 5) / (kVecs / 4)); // a warp: 8 x 4 of the groups
  const int vec = ((tid >> 3) & 3) + 4 * ((tid >> 5) % (kVecs / 4));
  const int d0 = vec * 8;
  // where pair i of a token lies in its row of the table: the eight tokens that a warp reads at a time are in different banks
  auto at = [](int place, int i) { return i ^ ((place >> 2 & 7) << 1); };

  for (int64_t block = max(before, 0) / kPageTokens + mine; block * kPageTokens < kv; block += slots) {
    const int base = (int)block * kPageTokens;
    const int page = block < b.table_width ? b.table[(int64_t)seq * b.table_stride + block] : -1;
    if (page < 0 || page >= a.pages) {
      if (tid == 0) note_bad_batch(&g_append_batch);
      continue;
    }
    const int lo = max(before - base, 0), hi = min(kv - base, kPageTokens);      // places of the new tokens in the page
    const bool fresh = before <= base;
    const int64_t row0 = (int64_t)q0 + base - before;         // row of the token at place 0 (negative if that one is older)
    const int64_t ph = (int64_t)page * a.kv_heads + head;
    const float k_old = fresh ? 0.f : a.k_scale[ph], v_old = fresh ? 0.f : a.v_scale[ph];

    // values first: raw words of four tokens; keys are on their way meanwhile
    uint4 vr[4], kr[4];
    if constexpr (W == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int place = quad * 4 + i;
        const bool in = place >= lo && place < hi;
        vr[i] = in ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + (row0 + place) * a.v_ts + (int64_t)head * a.v_hs + d0) : make_uint4(0, 0, 0, 0);
        kr[i] = in ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.k) + (row0 + place) * a.k_ts + (int64_t)head * a.k_hs + d0) : make_uint4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int place = quad * 4 + i;
        const bool in = place >= lo && place < hi;
        const T* v = static_cast<const T*>(a.v) + (row0 + place) * a.v_ts + (int64_t)head * a.v_hs + d0;
        const T* k = static_cast<const T*>(a.k) + (row0 + place) * a.k_ts + (int64_t)head * a.k_hs + d0;
        uint32_t wv[4] = {}, wk[4] = {};
        if (in)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            wv[e] = pack2(to_f32(v[2 * e]), to_f32(v[2 * e + 1]), T{});
            wk[e] = pack2(to_f32(k[2 * e]), to_f32(k[2 * e + 1]), T{});
          }
        vr[i] = make_uint4(wv[0], wv[1], wv[2], wv[3]);
        kr[i] = make_uint4(wk[0], wk[1], wk[2], wk[3]);
      }
    }
    if (tid < kPageTokens) nan_token[tid] = 0;
    for (int i = tid % (D / 2); i < r.half; i += D / 2)       // D / 2 pairs of 4 tokens at a time
      for (int tt = lo + tid / (D / 2); tt < hi; tt += 4) cs[tt][at(tt, i)] = cos_sin(turns_per_position(r.freq[i]), (int64_t)base + tt, r.magnitude);
    __syncthreads();

    uint32_t v_top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) v_top = abs_max2(v_top, w[e], T{});
    }
    float2 top = unpack2(v_top, T{});
    float v_max = fmaxf(top.x, top.y);
    if (!(top.x <= 3.402823466e38f && top.y <= 3.402823466e38f)) {               // an infinity or a NaN among the 32
      v_max = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&vr[i]);
        bool nan = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2(w[e], T{});
          v_max = finite_max(finite_max(v_max, f.x), f.y);
          if (isnan(f.x)) { w[e] &= 0xFFFF0000u; nan = true; }  // stored as 0
          if (isnan(f.y)) { w[e] &= 0x0000FFFFu; nan = true; }
        }
        if (nan) nan_token[quad * 4 + i] = 1;
      }
    }
    // keys, turned
    float kf[4][8], k_max = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = quad * 4 + i;
      const uint32_t w[4] = {kr[i].x, kr[i].y, kr[i].z, kr[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2(w[e], T{});
        kf[i][2 * e] = f.x, kf[i][2 * e + 1] = f.y;
      }
      if (place >= lo && place < hi && d0 < 2 * r.half) {
        const T* k = static_cast<const T*>(a.k) + (row0 + place) * a.k_ts + (int64_t)head * a.k_hs;
        if constexpr (W == 8) {
          if (r.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 c = *reinterpret_cast<const float4*>(&cs[place][at(place, d0 / 2 + (e & 2))]);
              const float cc = e & 1 ? c.z : c.x, ss = e & 1 ? c.w : c.y, x = kf[i][2 * e], y = kf[i][2 * e + 1];
              kf[i][2 * e] = x * cc - y * ss;
              kf[i][2 * e + 1] = y * cc + x * ss;
            }
          } else {
            const bool front = d0 < r.half;
            const int p0 = front ? d0 : d0 - r.half;
            float other[8];
            load8(k + (front ? d0 + r.half : p0), other);     // a neighbour's piece: from the first-level cache
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float4 c = *reinterpret_cast<const float4*>(&cs[place][at(place, p0 + e)]);
              kf[i][e] = front ? kf[i][e] * c.x - other[e] * c.y : kf[i][e] * c.x + other[e] * c.y;
              kf[i][e + 1] = front ? kf[i][e + 1] * c.z - other[e + 1] * c.w : kf[i][e + 1] * c.z + other[e + 1] * c.w;
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = d0 + e;
            if (d < 2 * r.half) {
              const int p = r.interleaved ? d / 2 : (d < r.half ? d : d - r.half);
              const bool front = r.interleaved ? (d & 1) == 0 : d < r.half;
              const float2 c = cs[place][at(place, p)];
              const float other = to_f32(k[r.interleaved ? d ^ 1 : (front ? d + r.half : d - r.half)]);
              kf[i][e] = front ? kf[i][e] * c.x - other * c.y : kf[i][e] * c.x + other * c.y;
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) k_max = fmaxf(k_max, fabsf(kf[i][e]));        // passes a NaN over
    }
    if (k_max > 3.402823466e38f) {                            // an infinity: the largest value next to it
      k_max = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) k_max = finite_max(k_max, kf[i][e]);
    }
    v_max = cta_max<kThreads>(v_max, red[0]);
    k_max = cta_max<kThreads>(k_max, red[1]);                 // both CTA barriers: every thread has read the old scales
    float k_s = scale_for(k_max), v_s = scale_for(v_max), k_ratio = 1.f, v_ratio = 1.f;
    if (!fresh) {
      k_s = fmaxf(k_s, k_old);
      v_s = fmaxf(v_s, v_old);
      k_ratio = k_old / k_s;
      v_ratio = v_old / v_s;
    }
    if (tid == 0) { a.k_scale[ph] = k_s; a.v_scale[ph] = v_s; }
    const float k_inv = 1.f / k_s, v_inv = 1.f / v_s;         // exact: powers of two

    // keys: 8 bytes of each token
    uint8_t* kp = a.k_pages + ph * (kPageTokens * D) + d0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = quad * 4 + i;
      const bool is_new = place >= lo && place < hi;
      if (!is_new && !(fresh || (place < lo && k_ratio != 1.f))) continue;
      uint2* at = reinterpret_cast<uint2*>(kp + place * D);
      uint32_t c[2] = {0, 0};
      if (is_new) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) c[e / 4] |= to_e4m3x2(kf[i][e] * k_inv, kf[i][e + 1] * k_inv) << (8 * (e & 3));
        if (d0 == 0 && nan_token[place]) c[0] = (c[0] & ~0xFFu) | 0x7Fu;
      } else if (place < lo) {
        const uint2 old = *at;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          c[e / 4] |= (uint32_t)to_e4m3(from_e4m3((uint8_t)((e < 4 ? old.x : old.y) >> (8 * (e & 3)))) * k_ratio) << (8 * (e & 3));
      }
      *at = make_uint2(c[0], c[1]);
    }
    // values: 4 tokens of each of 8 rows
    const bool any_new = quad * 4 < hi && quad * 4 + 4 > lo;
    if (any_new || fresh || (quad * 4 < lo && v_ratio != 1.f)) {
      const bool all_new = quad * 4 >= lo && quad * 4 + 4 <= hi, whole = fresh || all_new;
      uint8_t* vp = a.v_pages + ph * (kPageTokens * D) + quad * 4;
      if (all_new) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float2 f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = unpack2(reinterpret_cast<const uint32_t*>(&vr[i])[e / 2], T{});
          uint32_t* at = reinterpret_cast<uint32_t*>(vp + (d0 + e) * kPageTokens);
          at[0] = to_e4m3x2(f[0].x * v_inv, f[1].x * v_inv) | to_e4m3x2(f[2].x * v_inv, f[3].x * v_inv) << 16;
          at[kPageTokens / 4] = to_e4m3x2(f[0].y * v_inv, f[1].y * v_inv) | to_e4m3x2(f[2].y * v_inv, f[3].y * v_inv) << 16;
        }
      } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t* at = reinterpret_cast<uint32_t*>(vp + (d0 + e) * kPageTokens);
        const uint32_t old = whole ? 0u : *at;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int place = quad * 4 + i;
          uint8_t code = (uint8_t)(old >> (8 * i));
          if (place >= lo && place < hi) {
            const uint32_t half = reinterpret_cast<const uint32_t*>(&vr[i])[e / 2];
            const float2 f = unpack2(half, T{});
            code = to_e4m3((e & 1 ? f.y : f.x) * v_inv);
          } else if (place < lo && v_ratio != 1.f) {
            code = to_e4m3(from_e4m3(code) * v_ratio);
          }
          w |= (uint32_t)code << (8 * i);
        }
        *at = w;
      }
      }
    }
    __syncthreads();                                          // the next page's tables go over this one's
  }
}

// The same for steps of few tokens (rotation of the queries included): a warp owns a page of a head, and everything is a rolled
// loop over the page's new tokens and over 32 values at a time, twice -- for the largest value, then for the codes. The kernel
// above takes 13.4 us for one token in each of 64 sequences, nearly all of it instruction fetches: a CTA runs its unrolled program
// once. This one takes 5.8 us; with more tokens in a page the other is faster (the rule and its figures are in the launcher).
template <typename T, int D, int W> __global__ void __launch_bounds__(128) ob_cache_append_few_kernel(const AppendArgs a, const RotaryArgs q) {
  follow_previous_kernel();
  constexpr int kThreads = 128;
  __shared__ __align__(16) float2 qcs[kFewTokens][kMaxHalf];
  __shared__ int64_t pos[kFewTokens];
  __shared__ bool skip[kFewTokens];
  const int lane = threadIdx.x & 31;
  const BatchArgs& b = a.b;
  const int page_ctas = (a.page_slots * a.kv_heads + 3) / 4;
  const Starts starts{b.q_start, b.seqs, a.tokens};
  if ((int)blockIdx.x >= page_ctas) {
    const int t0 = ((int)blockIdx.x - page_ctas) * kFewTokens, n = min(kFewTokens, q.tokens - t0);
    static_assert(kFewTokens == kThreads / 32, "a token per warp");
    rotate_tokens<T, W, kThreads>(q, t0, n, qcs, skip, [&] {
      const int tt = threadIdx.x >> 5;                        // a warp finds a token's sequence
      int c = b.seqs + 1;
      bool bad = false;
      for (int s = lane; s <= b.seqs; s += 32) {
        const int start = starts.at(s, bad);
        c = min(c, starts.behind_row(s, start, t0 + tt));
      }
      c = __reduce_min_sync(~0u, c);
      bad = __any_sync(~0u, bad);
      if (lane == 0) {
        skip[tt] = c < 1 || c > b.seqs || (bad && starts.left_out(c - 1));
        pos[tt] = skip[tt] ? 0 : (int64_t)b.kv_len[c - 1] - b.q_start[c] + t0 + tt;
      }
      __syncthreads();
      fill_cos_sin<kThreads>(q.rot, pos, n, qcs);
      __syncthreads();
    });
    return;
  }

  const int item = (int)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= a.page_slots * a.kv_heads) return;
  const int head = item % a.kv_heads, slot = item / a.kv_heads;
  int c = min(b.seqs, slot + 1);                              // sequence c - 1 has the slot
  bool bad = false;
  for (int s = lane; s < b.seqs; s += 32) {
    const int start = starts.at(s, bad);
    c = min(c, starts.behind_slot(s, start, slot, start / kPageTokens));
  }
  c = __reduce_min_sync(~0u, c);
  bad = __any_sync(~0u, bad);
  if (bad && item == 0 && lane == 0) note_bad_batch(&g_append_batch);
  const int seq = c - 1;
  if (seq < 0 || (bad && starts.left_out(seq))) return;
  const int q0 = b.q_start[seq], q1 = b.q_start[seq + 1], kv = b.kv_len[seq], n = q1 - q0;
  if (n < a.least_new || n > a.most_new || kv <= 0) return;
  const int before = kv - n, mine = slot - (q0 / kPageTokens + seq), slots = q1 / kPageTokens + 1 - q0 / kPageTokens;
  const Rotation& r = a.rot;
  for (int64_t block = max(before, 0) / kPageTokens + mine; block * kPageTokens < kv; block += slots) {
    const int base = (int)block * kPageTokens;
    const int page = block < b.table_width ? b.table[(int64_t)seq * b.table_stride + block] : -1;
    if (page < 0 || page >= a.pages) {
      if (lane == 0) note_bad_batch(&g_append_batch);
      continue;
    }
    const int lo = max(before - base, 0), hi = min(kv - base, kPageTokens);
    const bool fresh = before <= base;
    const int64_t row0 = (int64_t)q0 + base - before, ph = (int64_t)page * a.kv_heads + head;
    const float k_old = fresh ? 0.f : a.k_scale[ph], v_old = fresh ? 0.f : a.v_scale[ph];
    uint8_t *kp = a.k_pages + ph * (kPageTokens * D), *vp = a.v_pages + ph * (kPageTokens * D);
    float k_max = 0.f, v_max = 0.f, k_inv = 0.f, v_inv = 0.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
      for (int place = lo; place < hi; ++place) {
        const T* k = static_cast<const T*>(a.k) + (row0 + place) * a.k_ts + (int64_t)head * a.k_hs;
        const T* v = static_cast<const T*>(a.v) + (row0 + place) * a.v_ts + (int64_t)head * a.v_hs;
        bool nan = false;
#pragma unroll 1
        for (int d = lane; d < D; d += 32) {
          float kx = to_f32(k[d]);
          const float vx = to_f32(v[d]);
          if (d < 2 * r.half) {
            const bool front = r.interleaved ? (d & 1) == 0 : d < r.half;
            const int pr = r.interleaved ? d >> 1 : (front ? d : d - r.half);
            const float other = to_f32(k[r.interleaved ? d ^ 1 : (front ? d + r.half : d - r.half)]);
            const float2 c = cos_sin(turns_per_position(r.freq[pr]), (int64_t)base + place, r.magnitude);
            kx = front ? kx * c.x - other * c.y : kx * c.x + other * c.y;
          }
          if (pass == 0) {
            k_max = finite_max(k_max, kx);
            v_max = finite_max(v_max, vx);
          } else {
            kp[place * D + d] = to_e4m3(kx * k_inv);
            vp[d * kPageTokens + place] = isnan(vx) ? 0 : to_e4m3(vx * v_inv);
            nan |= isnan(vx);
          }
        }
        if (pass == 1 && __any_sync(~0u, nan) && lane == 0) kp[place * D] = 0x7F;      // lane 0 wrote this byte before
      }
      if (pass == 1) break;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        k_max = fmaxf(k_max, __shfl_xor_sync(~0u, k_max, o));
        v_max = fmaxf(v_max, __shfl_xor_sync(~0u, v_max, o));
      }
      const float k_s = fmaxf(scale_for(k_max), k_old), v_s = fmaxf(scale_for(v_max), v_old);
      k_inv = 1.f / k_s, v_inv = 1.f / v_s;
      if (lane == 0) { a.k_scale[ph] = k_s; a.v_scale[ph] = v_s; }
      if (fresh) {                                            // zeros behind the new tokens
#pragma unroll 1
        for (int i = lane; i < kPageTokens * D / 16; i += 32) {
          if (i * 16 >= hi * D) reinterpret_cast<uint4*>(kp)[i] = make_uint4(0, 0, 0, 0);
          reinterpret_cast<uint4*>(vp)[i] = make_uint4(0, 0, 0, 0);
        }
      } else if (k_s != k_old || v_s != v_old) {              // earlier tokens in the new scale
        const float k_ratio = k_old / k_s, v_ratio = v_old / v_s;
#pragma unroll 1
        for (int i = lane; i < kPageTokens * D; i += 32) {
          const int kd = i % D, kt = i / D, vt = i % kPageTokens;
          if (kt < lo && k_ratio != 1.f) kp[kt * D + kd] = to_e4m3(from_e4m3(kp[kt * D + kd]) * k_ratio);
          if (vt < lo && v_ratio != 1.f) vp[i] = to_e4m3(from_e4m3(vp[i]) * v_ratio);
        }
      }
      __syncwarp();                                           // the codes go over what other lanes wrote here
    }
  }
}

}  // namespace

namespace ob {

static bool wide_rows(const void* p, int64_t ts, int64_t hs) {
  return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ts % 8 == 0 && hs % 8 == 0);
}
static bool wide_rotation(int rotary_dim, bool interleaved) { return rotary_dim % (interleaved ? 8 : 16) == 0; }

cudaError_t launch_rotary(const void* x, int64_t x_ts, int64_t x_hs, void* y, int64_t y_ts, int64_t y_hs, const void* positions,
                          bool positions_i64, const double* inv_freq, int rotary_dim, bool interleaved, float magnitude, int64_t tokens,
                          int64_t heads, int64_t head_dim, bool bf16, cudaStream_t stream) {
  const RotaryArgs a{x, y, x_ts, x_hs, y_ts, y_hs, positions, positions_i64, (int)tokens, (int)heads, (int)head_dim,
                     {inv_freq, rotary_dim / 2, interleaved, magnitude}};
  const bool wide = head_dim % 8 == 0 && wide_rotation(rotary_dim, interleaved) && wide_rows(x, x_ts, x_hs) && wide_rows(y, y_ts, y_hs);
  // tokens per CTA: two where latency counts, eight (one table for all, more under way) on many. 32 heads of 128, 4096 tokens:
  // 18.1 us with two, 15.9 with eight; 20 heads, 37 tokens: 2.7 and 5.0
  auto go = [&](auto t, auto per) {
    constexpr int kTokens = decltype(per)::value;
    using T = decltype(t);
    return launch_following(wide ? ob_rotary_kernel<T, 8, kTokens> : ob_rotary_kernel<T, 1, kTokens>, dim3((unsigned)((tokens + kTokens - 1) / kTokens)), kRotThreads, 0, stream, a);
  };
  auto by_count = [&](auto t) { return tokens <= 1024 ? go(t, std::integral_constant<int, 2>{}) : go(t, std::integral_constant<int, 8>{}); };
  return bf16 ? by_count(__nv_bfloat16{}) : by_count(__half{});
}

cudaError_t launch_cache_append(const CacheAppendCall& c, cudaStream_t stream) {
  AppendArgs a{};
  a.k = c.k, a.v = c.v, a.k_ts = c.k_ts, a.k_hs = c.k_hs, a.v_ts = c.v_ts, a.v_hs = c.v_hs;
  a.k_pages = static_cast<uint8_t*>(c.k_pages), a.v_pages = static_cast<uint8_t*>(c.v_pages);
  a.k_scale = c.k_scale, a.v_scale = c.v_scale, a.pages = c.pages, a.kv_heads = (int)c.kv_heads;
  a.b = {c.q_start, c.kv_len, c.table, c.table_stride, (int)c.table_width, (int)c.seqs};
  a.rot = {c.inv_freq, c.rotary_dim / 2, c.interleaved, c.magnitude};
  a.tokens = (int)c.tokens;
  a.page_slots = (int)(c.tokens / kPageTokens + c.seqs);
  RotaryArgs q{c.q, c.q_out, c.q_ts, c.q_hs, c.qo_ts, c.qo_hs, nullptr, 0, c.q ? (int)c.tokens : 0, (int)c.heads, (int)c.head_dim, a.rot};
  const bool wide = wide_rotation(c.rotary_dim, c.interleaved) && wide_rows(c.k, c.k_ts, c.k_hs) && wide_rows(c.v, c.v_ts, c.v_hs) &&
                    wide_rows(c.q, c.q_ts, c.q_hs) && wide_rows(c.q_out, c.qo_ts, c.qo_hs);
  const int64_t items = (int64_t)a.page_slots * a.kv_heads;
  // Sequences of up to three tokens: a warp's rolled loops. Measured for 64 sequences of 1 / 2 / 3 / 4 / 8 tokens, 8 heads of 128
  // with 32 query heads: 5.8 / 9.5 / 12.7 / 16.8 / 27.8 us, against 13.4 / 14.1 / 18.3 / 12.0 / 15.3 us; a page of 64 takes its warp 200.
  // So the caller's bound decides, not the mean: where some sequences are longer and most are short, both kernels run, each for
  // its sequences (255 single tokens and 200 for one more: 21.5 us, 217 in the warps alone; 1024 and 1000: 64 us, 283).
  constexpr int kMostFew = 3, kAny = 0x7fffffff;
  const bool short_ones = c.max_new <= kMostFew, both = !short_ones && c.tokens <= 2 * c.seqs;
  a.least_new = 1, a.most_new = both ? kMostFew : kAny;
  auto go = [&](auto t, auto d, auto w) {
    constexpr int kDim = decltype(d)::value, kWidth = decltype(w)::value;
    using T = decltype(t);
    if (short_ones || both) {
      const int64_t blocks = (items + 3) / 4 + (q.tokens + kFewTokens - 1) / kFewTokens;
      const cudaError_t e = launch_following(ob_cache_append_few_kernel<T, kDim, kWidth>, dim3((unsigned)blocks), 128, 0, stream, a, q);
      if (e != cudaSuccess || !both) return e;
      a.least_new = kMostFew + 1, a.most_new = kAny;
      q.tokens = 0;                                             // the queries are turned
    }
    const int64_t blocks = items + (q.tokens + kAppendTokens - 1) / kAppendTokens;
    return launch_following(ob_cache_append_kernel<T, kDim, kWidth>, dim3((unsigned)blocks), 2 * kDim, 0, stream, a, q);
  };
  auto by_width = [&](auto t, auto d) {
    return wide ? go(t, d, std::integral_constant<int, 8>{}) : go(t, d, std::integral_constant<int, 1>{});
  };
  auto by_dim = [&](auto t) {
    return c.head_dim == 64 ? by_width(t, std::integral_constant<int, 64>{}) : by_width(t, std::integral_constant<int, 128>{});
  };
  return c.bf16 ? by_dim(__nv_bfloat16{}) : by_dim(__half{});
}

cudaError_t read_append_status(int* batch) { return take_status(g_append_batch, batch); }

}  // namespace ob
