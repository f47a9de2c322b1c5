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

__device__ int g_append_status;

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
};

constexpr int kRotTokens = 4;          // tokens per CTA
constexpr int kRotThreads = 256;
constexpr int kMaxHalf = 256;

// pair i of the head at p: values a, b at offsets (oa, ob)
__device__ __forceinline__ void pair_at(const Rotation& r, int i, int& oa, int& ob) {
  oa = r.interleaved ? 2 * i : i;
  ob = r.interleaved ? 2 * i + 1 : i + r.half;
}

// The heads of up to kRotTokens tokens, from the table of their cos and sin in shared memory. W = 8: rotation and pass-through
// in pieces of 8 values.
template <typename T, int W>
__device__ __forceinline__ void rotate_tokens(const RotaryArgs& a, int t0, int n, const float2 (&cs)[kRotTokens][kMaxHalf], const bool (&skip)[kRotTokens]) {
  const Rotation& r = a.rot;
  const bool in_place = a.x == a.y;
  // units of a head: W pairs each (half) or W / 2 pairs (interleaved), then the pass-through in pieces of W
  const int pairs_per = W == 1 ? 1 : (r.interleaved ? W / 2 : W);
  const int turning = r.half / pairs_per;
  const int passing = in_place ? 0 : (a.head_dim - 2 * r.half) / W;
  const int per_head = turning + passing;
  const int total = n * a.heads * per_head;
  for (int u = threadIdx.x; u < total; u += kRotThreads) {
    const int piece = u % per_head, th = u / per_head;
    const int head = th % a.heads, tt = th / a.heads;
    if (skip[tt]) continue;
    const T* x = static_cast<const T*>(a.x) + (int64_t)(t0 + tt) * a.x_ts + (int64_t)head * a.x_hs;
    T* y = static_cast<T*>(a.y) + (int64_t)(t0 + tt) * a.y_ts + (int64_t)head * a.y_hs;
    if (piece >= turning) {
      const int o = 2 * r.half + (piece - turning) * W;
      if constexpr (W == 8) *reinterpret_cast<uint4*>(y + o) = *reinterpret_cast<const uint4*>(x + o);
      else y[o] = x[o];
      continue;
    }
    if constexpr (W == 1) {
      int oa, ob;
      pair_at(r, piece, oa, ob);
      const float2 c = cs[tt][piece];
      const float va = to_f32(x[oa]), vb = to_f32(x[ob]);
      y[oa] = from_f32<T>(va * c.x - vb * c.y);
      y[ob] = from_f32<T>(vb * c.x + va * c.y);
    } else if (r.interleaved) {
      float v[8];
      load8(x + piece * 8, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 c = cs[tt][piece * 4 + i];
        const float va = v[2 * i], vb = v[2 * i + 1];
        v[2 * i] = va * c.x - vb * c.y;
        v[2 * i + 1] = vb * c.x + va * c.y;
      }
      store8(y + piece * 8, v);
    } else {
      float va[8], vb[8];
      load8(x + piece * 8, va);
      load8(x + r.half + piece * 8, vb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 c = cs[tt][piece * 8 + i];
        const float p = va[i], q = vb[i];
        va[i] = p * c.x - q * c.y;
        vb[i] = q * c.x + p * c.y;
      }
      store8(y + piece * 8, va);
      store8(y + r.half + piece * 8, vb);
    }
  }
}

__device__ __forceinline__ void fill_cos_sin(const Rotation& r, const int64_t (&pos)[kRotTokens], int n, float2 (&cs)[kRotTokens][kMaxHalf]) {
  for (int u = threadIdx.x; u < n * r.half; u += kRotThreads) {
    const int i = u % r.half, tt = u / r.half;
    cs[tt][i] = cos_sin(turns_per_position(r.freq[i]), pos[tt], r.magnitude);
  }
}

template <typename T, int W> __global__ void __launch_bounds__(kRotThreads) ob_rotary_kernel(const RotaryArgs a) {
  __shared__ float2 cs[kRotTokens][kMaxHalf];
  __shared__ int64_t pos[kRotTokens];
  __shared__ bool skip[kRotTokens];
  const int t0 = blockIdx.x * kRotTokens, n = min(kRotTokens, a.tokens - t0);
  if (threadIdx.x < n) {
    pos[threadIdx.x] = a.positions_i64 ? static_cast<const int64_t*>(a.positions)[t0 + threadIdx.x]
                                       : (int64_t) static_cast<const int*>(a.positions)[t0 + threadIdx.x];
    skip[threadIdx.x] = false;
  }
  __syncthreads();
  fill_cos_sin(a.rot, pos, n, cs);
  __syncthreads();
  rotate_tokens<T, W>(a, t0, n, cs, skip);
}

// Number of sequences s with key(s) <= x, counted by the whole CTA (keys do not decrease with s).
template <typename F> __device__ __forceinline__ int count_not_above(int seqs, int x, F key) {
  int c = 0;
  for (int s0 = 0; s0 < seqs; s0 += kRotThreads) {
    const int s = s0 + threadIdx.x;
    c += __syncthreads_count(s < seqs && key(s) <= x);
  }
  return c;
}


template <typename T, int D, int W>
__global__ void __launch_bounds__(kRotThreads) ob_cache_append_kernel(const AppendArgs a, const RotaryArgs q) {
  __shared__ float2 cs[kPageTokens][D / 2];
  __shared__ float red[2][kRotThreads / 32];
  __shared__ int nan_token[kPageTokens];
  const int tid = threadIdx.x;
  const BatchArgs& b = a.b;

  if ((int)blockIdx.x >= a.page_slots * a.kv_heads) {
    // ---- queries: up to kRotTokens tokens ----
    auto& qcs = reinterpret_cast<float2(&)[kRotTokens][kMaxHalf]>(cs);
    static_assert(sizeof(cs) >= sizeof(float2) * kRotTokens * kMaxHalf, "the queries' table lies in the keys'");
    __shared__ int64_t pos[kRotTokens];
    __shared__ bool skip[kRotTokens];
    const int t0 = ((int)blockIdx.x - a.page_slots * a.kv_heads) * kRotTokens, n = min(kRotTokens, q.tokens - t0);
    for (int tt = 0; tt < n; ++tt) {
      const int t = t0 + tt;
      const int c = count_not_above(b.seqs + 1, t, [&](int s) { return b.q_start[s]; });   // sequence c - 1 holds token t
      if (tid == 0) {
        skip[tt] = c < 1 || c > b.seqs;                       // before the first or behind the last sequence
        pos[tt] = 0;
        if (!skip[tt]) pos[tt] = (int64_t)b.kv_len[c - 1] - b.q_start[c] + t;
      }
    }
    __syncthreads();
    fill_cos_sin(q.rot, pos, n, qcs);
    __syncthreads();
    rotate_tokens<T, W>(q, t0, n, qcs, skip);
    return;
  }

  // ---- a page of one head ----
  // Page slots: sequence s owns slots [floor(q_start[s] / 64) + 2 s, floor(q_start[s+1] / 64) + 2 (s + 1)), at least as many as
  // n tokens can touch pages.
  const int head = (int)blockIdx.x % a.kv_heads, slot = (int)blockIdx.x / a.kv_heads;
  auto first_slot = [&](int s) { return b.q_start[s] / kPageTokens + 2 * s; };
  const int seq = count_not_above(b.seqs, slot, first_slot) - 1;
  if (seq < 0) return;
  const int q0 = b.q_start[seq], q1 = b.q_start[seq + 1], kv = b.kv_len[seq], n = q1 - q0;
  if (n <= 0 || kv <= 0) return;
  const int before = kv - n;                                  // may be negative: the first -before tokens have no place
  const int block = max(before, 0) / kPageTokens + slot - first_slot(seq);
  const int base = block * kPageTokens;
  if (block < 0 || base >= kv) return;                        // block < 0: q_start runs backwards
  const int page = block < b.table_width ? b.table[(int64_t)seq * b.table_stride + block] : -1;
  if (q0 < 0 || q1 > a.tokens || page < 0 || page >= a.pages) {
    if (tid == 0) atomicCAS(&g_append_status, 0, kStatusBadBatch);
    return;
  }
  const int lo = max(before - base, 0), hi = min(kv - base, kPageTokens);      // places of the new tokens in the page
  const bool fresh = before <= base;
  const int64_t row0 = (int64_t)q0 + base - before;           // row of the token at place 0 (negative if that one is older)
  const Rotation& r = a.rot;

  if (tid < kPageTokens) nan_token[tid] = 0;
  for (int u = tid; u < (hi - lo) * r.half; u += kRotThreads) {
    const int i = u % r.half, tt = lo + u / r.half;
    cs[tt][i] = cos_sin(turns_per_position(r.freq[i]), (int64_t)base + tt, r.magnitude);
  }
  __syncthreads();

  // thread = 4 tokens (one word of the transposed values) x 8 values; a warp = 8 x 4 of those
  constexpr int kVecs = D / 8;
  constexpr int kUsed = 16 * kVecs;                           // 256 threads at D = 128, 128 at D = 64
  const int quad = (tid & 7) + 8 * ((tid >> 5) / (kVecs / 4));
  const int vec = ((tid >> 3) & 3) + 4 * ((tid >> 5) % (kVecs / 4));
  const bool mine = tid < kUsed;
  const int d0 = vec * 8;
  float kf[4][8], vf[4][8];
  float k_max = 0.f, v_max = 0.f;
  auto finite_max = [](float m, float v) { v = fabsf(v); return v <= 3.402823466e38f ? fmaxf(m, v) : m; };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int place = quad * 4 + i;
    if (!mine || place < lo || place >= hi) {
#pragma unroll
      for (int e = 0; e < 8; ++e) kf[i][e] = vf[i][e] = 0.f;
      continue;
    }
    const T* kr = static_cast<const T*>(a.k) + (row0 + place) * a.k_ts + (int64_t)head * a.k_hs;
    const T* vr = static_cast<const T*>(a.v) + (row0 + place) * a.v_ts + (int64_t)head * a.v_hs;
    if constexpr (W == 8) {
      load8(kr + d0, kf[i]);
      load8(vr + d0, vf[i]);
      if (d0 < 2 * r.half) {
        if (r.interleaved) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 c = cs[place][d0 / 2 + e];
            const float x = kf[i][2 * e], y = kf[i][2 * e + 1];
            kf[i][2 * e] = x * c.x - y * c.y;
            kf[i][2 * e + 1] = y * c.x + x * c.y;
          }
        } else {
          float other[8];
          const bool first = d0 < r.half;
          const int p0 = first ? d0 : d0 - r.half;
          load8(kr + (first ? d0 + r.half : p0), other);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 c = cs[place][p0 + e];
            kf[i][e] = first ? kf[i][e] * c.x - other[e] * c.y : kf[i][e] * c.x + other[e] * c.y;
          }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        kf[i][e] = to_f32(kr[d]);
        vf[i][e] = to_f32(vr[d]);
        if (d < 2 * r.half) {
          const int p = r.interleaved ? d / 2 : (d < r.half ? d : d - r.half);
          const bool first = r.interleaved ? (d & 1) == 0 : d < r.half;
          const float2 c = cs[place][p];
          const float other = to_f32(kr[r.interleaved ? d ^ 1 : (first ? d + r.half : d - r.half)]);
          kf[i][e] = first ? kf[i][e] * c.x - other * c.y : kf[i][e] * c.x + other * c.y;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      k_max = finite_max(k_max, kf[i][e]);
      v_max = finite_max(v_max, vf[i][e]);
      if (isnan(vf[i][e])) { vf[i][e] = 0.f; nan_token[place] = 1; }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    k_max = fmaxf(k_max, __shfl_xor_sync(~0u, k_max, o));
    v_max = fmaxf(v_max, __shfl_xor_sync(~0u, v_max, o));
  }
  if ((tid & 31) == 0) { red[0][tid >> 5] = k_max; red[1][tid >> 5] = v_max; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRotThreads / 32; ++w) { k_max = fmaxf(k_max, red[0][w]); v_max = fmaxf(v_max, red[1][w]); }

  const int64_t ph = (int64_t)page * a.kv_heads + head;
  float k_s = scale_for(k_max), v_s = scale_for(v_max), k_ratio = 1.f, v_ratio = 1.f;
  if (!fresh) {
    const float k_old = a.k_scale[ph], v_old = a.v_scale[ph];
    k_s = fmaxf(k_s, k_old);
    v_s = fmaxf(v_s, v_old);
    k_ratio = k_old / k_s;
    v_ratio = v_old / v_s;
  }
  __syncthreads();                                            // every thread has read the old scales
  if (tid == 0) { a.k_scale[ph] = k_s; a.v_scale[ph] = v_s; }
  if (!mine) return;
  const float k_inv = 1.f / k_s, v_inv = 1.f / v_s;           // exact: powers of two

  // keys: 8 bytes of each token
  uint8_t* kp = a.k_pages + ph * (kPageTokens * D) + d0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int place = quad * 4 + i;
    const bool is_new = place >= lo && place < hi;
    if (!is_new && !(fresh || (place < lo && k_ratio != 1.f))) continue;
    uint2* at = reinterpret_cast<uint2*>(kp + place * D);
    uint8_t c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (is_new) {
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = to_e4m3(kf[i][e] * k_inv);
      if (d0 == 0 && nan_token[place]) c[0] = 0x7F;
    } else if (place < lo) {
      const uint2 old = *at;
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = to_e4m3(from_e4m3((uint8_t)((e < 4 ? old.x : old.y) >> (8 * (e & 3)))) * k_ratio);
    }
    *at = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | (uint32_t)c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | (uint32_t)c[7] << 24);
  }
  // values: 4 tokens of each of 8 rows
  const bool any_new = quad * 4 < hi && quad * 4 + 4 > lo;
  const bool any_old = quad * 4 < lo;
  if (!any_new && !fresh && !(any_old && v_ratio != 1.f)) return;
  const bool whole = fresh || (quad * 4 >= lo && quad * 4 + 4 <= hi);
  uint8_t* vp = a.v_pages + ph * (kPageTokens * D) + quad * 4;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint32_t* at = reinterpret_cast<uint32_t*>(vp + (d0 + e) * kPageTokens);
    const uint32_t old = whole ? 0u : *at;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = quad * 4 + i;
      uint8_t c = (uint8_t)(old >> (8 * i));
      if (place >= lo && place < hi) c = to_e4m3(vf[i][e] * v_inv);
      else if (place < lo && v_ratio != 1.f) c = to_e4m3(from_e4m3(c) * v_ratio);
      w |= (uint32_t)c << (8 * i);
    }
    *at = w;
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
  const unsigned grid = (unsigned)((tokens + kRotTokens - 1) / kRotTokens);
  if (bf16) {
    if (wide) ob_rotary_kernel<__nv_bfloat16, 8><<<grid, kRotThreads, 0, stream>>>(a);
    else ob_rotary_kernel<__nv_bfloat16, 1><<<grid, kRotThreads, 0, stream>>>(a);
  } else {
    if (wide) ob_rotary_kernel<__half, 8><<<grid, kRotThreads, 0, stream>>>(a);
    else ob_rotary_kernel<__half, 1><<<grid, kRotThreads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t launch_cache_append(const CacheAppendCall& c, cudaStream_t stream) {
  AppendArgs a{};
  a.k = c.k, a.v = c.v, a.k_ts = c.k_ts, a.k_hs = c.k_hs, a.v_ts = c.v_ts, a.v_hs = c.v_hs;
  a.k_pages = static_cast<uint8_t*>(c.k_pages), a.v_pages = static_cast<uint8_t*>(c.v_pages);
  a.k_scale = c.k_scale, a.v_scale = c.v_scale, a.pages = c.pages, a.kv_heads = (int)c.kv_heads;
  a.b = {c.q_start, c.kv_len, c.table, c.table_stride, (int)c.table_width, (int)c.seqs};
  a.rot = {c.inv_freq, c.rotary_dim / 2, c.interleaved, c.magnitude};
  a.tokens = (int)c.tokens;
  a.page_slots = (int)(c.tokens / kPageTokens + 2 * c.seqs);
  RotaryArgs q{c.q, c.q_out, c.q_ts, c.q_hs, c.qo_ts, c.qo_hs, nullptr, 0, c.q ? (int)c.tokens : 0, (int)c.heads, (int)c.head_dim, a.rot};
  const bool wide = wide_rotation(c.rotary_dim, c.interleaved) && wide_rows(c.k, c.k_ts, c.k_hs) && wide_rows(c.v, c.v_ts, c.v_hs) &&
                    wide_rows(c.q, c.q_ts, c.q_hs) && wide_rows(c.q_out, c.qo_ts, c.qo_hs);
  const int64_t blocks = (int64_t)a.page_slots * a.kv_heads + (q.tokens + kRotTokens - 1) / kRotTokens;
  auto go = [&](auto t, auto d, auto w) {
    ob_cache_append_kernel<decltype(t), decltype(d)::value, decltype(w)::value><<<(unsigned)blocks, kRotThreads, 0, stream>>>(a, q);
    return cudaGetLastError();
  };
  auto by_width = [&](auto t, auto d) {
    return wide ? go(t, d, std::integral_constant<int, 8>{}) : go(t, d, std::integral_constant<int, 1>{});
  };
  auto by_dim = [&](auto t) {
    return c.head_dim == 64 ? by_width(t, std::integral_constant<int, 64>{}) : by_width(t, std::integral_constant<int, 128>{});
  };
  return c.bf16 ? by_dim(__nv_bfloat16{}) : by_dim(__half{});
}

cudaError_t read_append_status(int* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_append_status, sizeof(int));
  if (e != cudaSuccess || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_append_status, &zero, sizeof(int));
}

}  // namespace ob
