// Attention over the 8-bit cache for few query rows per cache head (decode steps, drafted tokens).
//
// out = softmax(scale q K^T) V; the work is to stream every cached byte once. For at most 16 query rows the products are
// padding on the tensor cores whatever is done, so the kernel is built around the stream:
//   * a segment is a (sequence, cache head, row tile). Where the block table says that none is long, a cluster of 1 to 16 CTAs
//     has one segment and joins its parts through shared memory. Else the pages of all segments form one line that is cut into
//     equal pieces, one per CTA, two CTAs per SM: a ragged batch is balanced without the host knowing a length, and a segment
//     that a cut falls into leaves partial results, which a second small kernel joins (ob_attend_combine_kernel);
//   * every warp takes every fourth page of its CTA's piece and fetches it by itself: bulk asynchronous copies (keys, then
//     values: 64 * D bytes each, contiguous) into a ring of its own, so no warp ever waits for another inside a segment;
//   * keys are the A operand of S^T = K Q^T (16 tokens x 16 values, mma m16n8k16, N = 8 query rows), values of O^T = V^T P^T:
//     the query rows are the narrow dimension, so 8 rows cost half of what they would as 16 padded ones. The order of the
//     contraction is free, so a thread's operands are 16 consecutive bytes: four k-steps of a key row, or of a value row's
//     tokens; the token that stands in row i of a score tile is chosen so that both fit. P goes from the accumulator layout to
//     the B operand by movmatrix (8 x 8 transposes);
//   * e4m3 -> fp16 is exact; the page's key scale multiplies the fp32 scores. The value scale goes
//     into the exponent: t = score + log2(value scale), running maximum M of t, weight w = 2^(t - M + 15), and the sum of the
//     weights without it is sum(w / value scale), in fp32 and of the weights before their rounding. For the product with the values
//     w is rounded to fp16: 2^-11 of it, the one rounding before the output's. The 15 puts the largest weight at the top of fp16's
//     range, so that all weights down to 2^-29 of it keep that precision and what falls below 2^-39 is lost; with the largest at 1,
//     thousands of small weights beside a token that has nearly all of it, or beside a page of 64 times the value scale, came out
//     up to 26 % off (4096 tokens).
// Measured: 64 sequences of up to 8192 tokens, 32 / 8 heads of 128, 530 MB in 100 us (5.3 TB/s, 81 % of the copy rate; the line);
// 1 token of 32 heads over 4096 tokens, 33.6 MB in 9.8 us (clusters of 8: a launch, three dependent loads and two pages a warp).
// What bounds the short ones is latency: a page takes a warp 1.65 us from its bytes to the sums, alone on the SM or not.
// bf16 queries become fp16 with a power of two per row (the row's largest value lands in [1, 2)): their 8 bits fit; a value
// 2^-14 below the row's largest starts losing bits of no consequence.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block_common.h"
#include "cache_attend.h"
#include "kernels.h"
#include "sm100_ptx.h"

namespace {

using namespace ob_block;
using namespace ob_ptx;

__device__ int g_attend_status, g_attend_batch;   // code of a wait that gave up; see note_bad_batch

constexpr int kWarps = 4;
constexpr int kRingBytes = 24 * 1024;             // per warp
constexpr int kMaxCluster = 16;
constexpr int kMinPages = 4;                      // pages of a CTA's piece: one per warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kWeightTop = 15.f;                // log2 of the largest weight: fp16 ends below 2^16

// ---- the line of pages ------------------------------------------------------------------------------------------------

struct Seq {
  bool bad;                                       // its range is not inside the call's rows, or its tokens not inside the table
  int q0, n, kv, pages, tiles;                    // kv: cached tokens; pages: 0 if the sequence has no new token, else at least 1
  int64_t w;                                      // pages of all its segments
};

// quotients of numbers that nearly always fit 32 bits; the 64-bit division is a subroutine of a hundred instructions
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ Seq seq_info(const ob::CacheAttendCall& c, int group, int s, int rows_per_tile) {
  Seq q;
  const int q1 = c.q_start[s + 1];
  q.q0 = c.q_start[s];
  q.kv = c.kv_len[s];
  q.bad = q.q0 < 0 || q1 > c.tokens || q1 < q.q0;
  q.n = q.bad || (int64_t)(q1 - q.q0) * group > c.few_rows ? 0 : q1 - q.q0;
  const int64_t room = c.table_width * kPageTokens;
  q.bad |= q.n > 0 && q.kv > room;
  const int seen = (int)min((int64_t)max(q.kv, 0), room);
  q.pages = q.n > 0 ? max(1, (seen + kPageTokens - 1) / kPageTokens) : 0;
  q.tiles = (q.n * group + rows_per_tile - 1) / rows_per_tile;
  q.w = (int64_t)q.pages * q.tiles * (int)c.kv_heads;
  return q;
}

// What a combine block needs of the segment that starts in CTA c and ends in CTA last (-1: there is none).
struct alignas(16) Header {
  int last, q0, n, head, tile, pad[3];
};

struct FewLayout {                                // the workspace, and what the host works out once
  int group;                                      // query heads of a cache head
  uint64_t per_group;                             // ceil(2^40 / group): row / group = row * per_group >> 40 while row * group < 2^40
  Header* headers;
  int cluster, tiles;                             // CTAs of a segment's cluster; row tiles that the grid has of a (sequence, cache head)
  float* partial;                                 // slots 2 c (segment that started before CTA c), 2 c + 1: rows x (D + 4): M, l at [D], [D + 1]
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load4(const uint8_t* p, uint32_t (&w)[4]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// shared memory of a CTA of the cluster
__device__ __forceinline__ float2 load2_cluster(uint32_t at) {
  float2 r;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ float4 load4_cluster(uint32_t at) {
  float4 r;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "r"(at) : "memory");
  return r;
}

// NT tiles of 8 query rows. LINE: a CTA has a piece of the line of pages. Else a cluster has a segment, CTA i of it the pages
// i, i + cluster, ...
template <typename T, int D, int NT, bool LINE> __global__ void __launch_bounds__(kWarps * 32, 2)
ob_attend_few_kernel(const ob::CacheAttendCall c, const FewLayout ws) {
  constexpr int kRows = 8 * NT;
  constexpr int kGranule = kPageTokens * D;                     // bytes of one page's keys (or values) of a head
  constexpr int kRing = kRingBytes / kGranule;
  constexpr int kMeta = 4;                                      // pages between a request and its use, at most kRing / 2 + 1
  constexpr int kMT = D / 16;                                   // value tiles
  constexpr int kPitch = D + 4;
  static_assert(kRing / 2 + 1 <= kMeta, "page data ring");
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + kWarps * kRingBytes);           // [warp][8][kPitch]
  struct Meta { float ks, log2_vs, inv_vs; int ok; };
  __shared__ Meta meta[kWarps][kMeta];
  __shared__ __align__(8) uint64_t bars[kWarps][kRing];
  __shared__ int64_t scan[kWarps + 1];
  __shared__ int64_t start_off;
  __shared__ int start_seq;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = ws.group;
  const int H = (int)c.kv_heads;
  auto token_of = [&](int r) { return (int)((uint64_t)(uint32_t)r * ws.per_group >> 40); };
  long long budget = 2000000000ll;

  if (lane == 0)
    for (int i = 0; i < kRing; ++i) mbar_init(smem_u32(&bars[warp][i]), 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  follow_previous_kernel();
  int seq = 0, my_pages = 0;
  int64_t off = 0, a = 0, b = 0, chunk = 1;                     // what is this CTA's: pages a .. b of the line, or b rounds of the grid's tiles
  Seq q;
  int page0, head, tile, take, rows_all;
  const int stride = LINE ? 1 : ws.cluster;                     // from one page of this CTA's to its next
  int first_id = -1;

  if constexpr (!LINE) {
    const int unit = blockIdx.x / ws.cluster, pair = unit / ws.tiles;
    page0 = blockIdx.x % ws.cluster, tile = unit % ws.tiles, head = pair % H, seq = pair / H;
    const int p = page0 + stride * (warp + kWarps * lane);      // the first page numbers do not wait for the lengths
    if (p < c.table_width) first_id = c.table[(int64_t)seq * c.table_stride + p];
    q = seq_info(c, group, seq, kRows);
    if (q.bad && page0 == 0 && tile == 0 && head == 0 && threadIdx.x == 0) note_bad_batch(&g_attend_batch);
    if (tile >= q.tiles) return;                                // the whole cluster
    b = (q.tiles - tile + ws.tiles - 1) / ws.tiles;             // more than one round where the caller's bound was wrong
    take = q.pages > page0 ? (q.pages - page0 + stride - 1) / stride : 0;
    my_pages = max(0, (take - warp + kWarps - 1) / kWarps);
    rows_all = q.n * group;
    __syncwarp();
  }

  if constexpr (LINE) {
  // ---- this CTA's piece: every thread sums a run of sequences, the CTA scans the sums ----
  const int run = (int)((c.seqs + kWarps * 32 - 1) / (kWarps * 32));
  const int s_lo = min((int)c.seqs, (int)threadIdx.x * run), s_hi = min((int)c.seqs, s_lo + run);
  int64_t mine = 0;
  bool bad = false;
  for (int s = s_lo; s < s_hi; ++s) {
    const Seq q = seq_info(c, group, s, kRows);
    mine += q.w;
    bad |= q.bad;
  }
  if (bad && blockIdx.x == 0) note_bad_batch(&g_attend_batch);
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(~0u, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  int64_t W = 0, before_warp = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before_warp = W;
    W += scan[w];
  }
  upto += before_warp;                                          // pages of the sequences up to this thread's last
  chunk = max((int64_t)kMinPages, quotient(W + gridDim.x - 1, gridDim.x));
  a = blockIdx.x * chunk, b = min(a + chunk, W);
  if (a >= W) {
    if (threadIdx.x == 0) ws.headers[blockIdx.x].last = -1;
    return;
  }
  if (a >= upto - mine && a < upto) {
    int64_t off = a - (upto - mine);
    int s = s_lo;
    for (Seq q = seq_info(c, group, s, kRows); off >= q.w; q = seq_info(c, group, s, kRows)) { off -= q.w; ++s; }
    start_seq = s;
    start_off = off;
  }
  __syncthreads();
  seq = start_seq;
  off = start_off;
  my_pages = (int)max((int64_t)0, (b - a - warp + kWarps - 1) / kWarps);
  }

  // ---- requests: this warp's pages are those at a + warp, a + warp + 4, ...; 32 of them are looked up at a time, one per lane ----
  int load_seq = seq;
  int64_t load_off = off + warp;
  int64_t ph = -1;                                              // (page, head) of this lane's page; -1: nothing to fetch
  float ph_ks = 0.f, ph_vs = 1.f;
  const uint32_t ring = smem_u32(smem) + warp * kRingBytes;
  auto look_up = [&](int first) {                               // pages first .. first + 31
    int s = load_seq;
    int64_t o = load_off + (int64_t)lane * kWarps;
    ph = -1;
    if constexpr (!LINE) {
      const int pg = page0 + stride * (warp + kWarps * (first + lane));
      if (first + lane < my_pages && (int64_t)pg * kPageTokens < q.kv) {
        const int id = first == 0 ? first_id : c.table[(int64_t)seq * c.table_stride + pg];
        if (id < 0 || id >= c.pages) {
          note_bad_batch(&g_attend_batch);
        } else {
          ph = (int64_t)id * H + head;
          ph_ks = c.k_scale[ph];
          ph_vs = c.v_scale[ph];
        }
      }
      return;
    }
    if (first + lane < my_pages) {
      Seq q = seq_info(c, group, s, kRows);
      while (o >= q.w) { o -= q.w; q = seq_info(c, group, ++s, kRows); }
      const int64_t seg = quotient(o, q.pages);
      const int pg = (int)(o - seg * q.pages), head = (int)quotient(seg, q.tiles);
      if ((int64_t)pg * kPageTokens < q.kv) {
        const int id = c.table[(int64_t)s * c.table_stride + pg];
        if (id < 0 || id >= c.pages) {
          note_bad_batch(&g_attend_batch);
        } else {
          ph = (int64_t)id * H + head;
          ph_ks = c.k_scale[ph];
          ph_vs = c.v_scale[ph];
        }
      }
    }
    load_seq = __shfl_sync(~0u, s, 31);                         // where the next 32 begin, if there are any
    load_off = __shfl_sync(~0u, o, 31) + kWarps;
  };
  // granule gr: keys (even) or values (odd) of page gr / 2, into slot gr % kRing
  int gr0 = 0;                                                  // granules of the rounds before this one
  auto request = [&](int gr) {
    const int i = (gr - gr0) >> 1;
    if (i >= my_pages) return;
    if (i > 0 && (i & 31) == 0 && (gr & 1) == 0) look_up(i);
    const int64_t at = __shfl_sync(~0u, ph, i & 31);
    const uint32_t bar = smem_u32(&bars[warp][gr % kRing]);
    if (lane == 0) {
      if (at >= 0) {
        mbar_expect_tx(bar, kGranule);
        bulk_load(ring + (gr % kRing) * kGranule, static_cast<const uint8_t*>(gr & 1 ? c.v_pages : c.k_pages) + at * kGranule, kGranule, bar);
      } else {
        mbar_arrive(bar);
      }
    }
  };
  // the scales of page i, for its use; by the lane that looked them up
  auto note_scales = [&](int i) {
    if (i < my_pages && lane == (i & 31)) {
      const float vs = fmaxf(ph_vs, 5.421010862e-20f);          // 2^-64: a page that nothing was stored in has scale 0
      meta[warp][(gr0 / 2 + i) % kMeta] = {ph_ks, __log2f(vs), __frcp_rn(vs), ph >= 0};
    }
  };
  // ---- a segment: what its part in this piece is, and its queries (raw: row g of each tile of 8) ----
  uint2 raw[NT][D / 16];
  auto enter = [&](int64_t l) {
    if constexpr (LINE) {
      q = seq_info(c, group, seq, kRows);
      while (off >= q.w) { off -= q.w; q = seq_info(c, group, ++seq, kRows); }
      const int64_t seg = quotient(off, q.pages);
      page0 = (int)(off - seg * q.pages);
      head = (int)quotient(seg, q.tiles);
      tile = (int)(seg - (int64_t)head * q.tiles);
      take = (int)min(b - l, (int64_t)(q.pages - page0));
      rows_all = q.n * group;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = tile * kRows + nt * 8 + g, tok = token_of(r);
      const T* row = static_cast<const T*>(c.q) + (int64_t)(q.q0 + tok) * c.q_ts + (int64_t)(head * group + r - tok * group) * c.q_hs;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) raw[nt][k] = r < rows_all ? *reinterpret_cast<const uint2*>(row + (k / 4) * 64 + t * 16 + (k % 4) * 4) : make_uint2(0, 0);
    }
  };
  auto begin = [&]() {
    look_up(0);                                                 // page numbers and queries are under way together
    enter(a);
    for (int i = 0; i < kRing; ++i) request(gr0 + i);
    for (int i = 0; 2 * i < kRing; ++i) note_scales(i);        // behind all requests: nothing is requested later for their sake
    __syncwarp();
  };
  begin();

  int gr = 0;                                                   // granules used so far by this warp
  for (int64_t l = a; l < b;) {
    // ---- one segment's part in this piece ----
    if (!LINE && l > a) {
      gr0 = gr;
      tile += ws.tiles;
      begin();
    }
    const int kv = (int)min((int64_t)max(q.kv, 0), c.table_width * kPageTokens);

    // queries: B operand of row g, and what the accumulators' columns 2 t, 2 t + 1 need
    uint32_t qf[NT][D / 16][2];
    float coef[NT][2];
    int limit[NT][2], least = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float unit = 1.f;                                         // what the fp16 form is to be multiplied by
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const float2 x = unpack2(raw[nt][k].x, T{}), y = unpack2(raw[nt][k].y, T{});
          m = fmaxf(m, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
        }
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
        // the row's exponent, kept where both 2^e and 2^-e are normal numbers; an infinite row stays infinite
        const int e = min(max((int)(__float_as_uint(m) >> 23), 2), 252);
        unit = __uint_as_float((uint32_t)e << 23);
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const float2 x = unpack2(raw[nt][k].x, T{}), y = unpack2(raw[nt][k].y, T{});
          raw[nt][k] = make_uint2(pack2(x.x * inv, x.y * inv, __half{}), pack2(y.x * inv, y.y * inv, __half{}));
        }
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k) { qf[nt][k][0] = raw[nt][k].x; qf[nt][k][1] = raw[nt][k].y; }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        coef[nt][j] = __shfl_sync(~0u, unit, (2 * t + j) * 4) * (c.scale * kLog2e);
        const int rr = tile * kRows + nt * 8 + 2 * t + j;       // rows behind the last one see everything: nothing of theirs is kept
        limit[nt][j] = rr >= rows_all ? 0x7fffffff : (c.causal ? min(kv, q.kv - q.n + token_of(rr) + 1) : kv);
        least = min(least, limit[nt][j]);
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) least = min(least, __shfl_xor_sync(~0u, least, o));

    float acc[NT][kMT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nt][i][j] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) { m_run[nt][j] = -INFINITY; l_run[nt][j] = 0.f; }
    }

    for (int j = LINE ? (int)((warp - (l - a)) & (kWarps - 1)) : warp; j < take; j += kWarps) {
      const int base = (page0 + j * stride) * kPageTokens;
      const Meta md = meta[warp][(gr >> 1) % kMeta];
      const int k_slot = gr % kRing, v_slot = (gr + 1) % kRing;
      const uint32_t k_par = (gr / kRing) & 1, v_par = ((gr + 1) / kRing) & 1;
      const uint8_t* kp = smem + warp * kRingBytes + k_slot * kGranule;
      const uint8_t* vp = smem + warp * kRingBytes + v_slot * kGranule;
      mbar_wait(smem_u32(&bars[warp][k_slot]), k_par, budget, &g_attend_status, 1);
      __syncwarp();
      float sc[NT][4][4];
      if (md.ok) {
        // score tile s: tokens (g / 2) 16 + 4 s + (g odd), and 2 further. The four tiles go side by side, so that no product waits
        // for the one before it.
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[nt][s][i] = 0.f;
        const uint8_t* k0 = kp + ((g >> 1) * 16 + (g & 1)) * D + t * 16;
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
          uint32_t x[4][4], y[4][4];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            load4(k0 + 4 * s * D + hf * 64, x[s]);
            load4(k0 + (4 * s + 2) * D + hf * 64, y[s]);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const uint32_t a0 = e4m3_lo(x[s][w]), a2 = e4m3_hi(x[s][w]), a1 = e4m3_lo(y[s][w]), a3 = e4m3_hi(y[s][w]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_16816(sc[nt][s], a0, a1, a2, a3, qf[nt][hf * 4 + w][0], qf[nt][hf * 4 + w][1]);
            }
        }
      }
      __syncwarp();
      request(gr + kRing);                                      // the keys' slot is free
      if (((gr + kRing) & 1) == 0) note_scales((gr + kRing - gr0) >> 1);
      uint32_t pf[NT][4][2];                                    // weights: B operand of k-step s
      if (md.ok) {
        bool moved = false;
        float alpha[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float k0 = coef[nt][0] * md.ks, k1 = coef[nt][1] * md.ks;
          float m0 = m_run[nt][0], m1 = m_run[nt][1];
          const bool masked = base + kPageTokens > least;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x = fmaf(sc[nt][s][2 * h], k0, md.log2_vs), y = fmaf(sc[nt][s][2 * h + 1], k1, md.log2_vs);
              if (masked) {
                const int tok = base + (g >> 1) * 16 + 4 * s + 2 * h + (g & 1);
                if (tok >= limit[nt][0]) x = -INFINITY;
                if (tok >= limit[nt][1]) y = -INFINITY;
              }
              sc[nt][s][2 * h] = x;
              sc[nt][s][2 * h + 1] = y;
              m0 = fmaxf(m0, x);
              m1 = fmaxf(m1, y);
            }
          }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(~0u, m0, o));
            m1 = fmaxf(m1, __shfl_xor_sync(~0u, m1, o));
          }
          const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
          moved |= m0 != m_run[nt][0] || m1 != m_run[nt][1];
          alpha[nt][0] = fast_exp2(m_run[nt][0] - r0);
          alpha[nt][1] = fast_exp2(m_run[nt][1] - r1);
          m_run[nt][0] = m0;
          m_run[nt][1] = m1;
          const float w0 = r0 - kWeightTop, w1 = r1 - kWeightTop;
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = fast_exp2(sc[nt][s][2 * h] - w0), y = fast_exp2(sc[nt][s][2 * h + 1] - w1);
              s0 += x;
              s1 += y;
              pf[nt][s][h] = transpose_8x8(pack2(x, y, __half{}));
            }
          }
          l_run[nt][0] = l_run[nt][0] * alpha[nt][0] + s0 * md.inv_vs;
          l_run[nt][1] = l_run[nt][1] * alpha[nt][1] + s1 * md.inv_vs;
        }
        if (__any_sync(~0u, moved)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < kMT; ++i) {
              acc[nt][i][0] *= alpha[nt][0], acc[nt][i][1] *= alpha[nt][1];
              acc[nt][i][2] *= alpha[nt][0], acc[nt][i][3] *= alpha[nt][1];
            }
        }
      }
      mbar_wait(smem_u32(&bars[warp][v_slot]), v_par, budget, &g_attend_status, 2);
      __syncwarp();
      if (md.ok) {
        // bytes behind the sequence's end may be anything, a NaN among them: they are read as zeros
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        const bool tail = base + kPageTokens > kv;
        if (tail) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int live = kv - base - (t * 16 + 4 * s);
            keep[s] = live >= 4 ? ~0u : live <= 0 ? 0u : ~0u >> (8 * (4 - live));
          }
        }
#pragma unroll
        for (int i0 = 0; i0 < kMT; i0 += 4) {                   // four value tiles side by side
          uint32_t x[4][4], y[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            load4(vp + (16 * (i0 + i) + g) * kPageTokens + t * 16, x[i]);
            load4(vp + (16 * (i0 + i) + 8 + g) * kPageTokens + t * 16, y[i]);
          }
          if (tail) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int s = 0; s < 4; ++s) { x[i][s] &= keep[s]; y[i][s] &= keep[s]; }
          }
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = e4m3_lo(x[i][s]), a2 = e4m3_hi(x[i][s]), a1 = e4m3_lo(y[i][s]), a3 = e4m3_hi(y[i][s]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt][i0 + i], a0, a1, a2, a3, pf[nt][s][0], pf[nt][s][1]);
            }
        }
      }
      __syncwarp();
      request(gr + 1 + kRing);
      if (((gr + 1 + kRing) & 1) == 0) note_scales((gr + 1 + kRing - gr0) >> 1);
      gr += 2;
      __syncwarp();
    }

    // ---- the next segment's part: its queries are under way while this one's results are joined ----
    const struct { Seq q; int page0, head, tile, take, rows_all; } now{q, page0, head, tile, take, rows_all};
    if constexpr (LINE) {
      off += take;
      if (l + take < b) enter(l + take);
    }

    // ---- the four warps' results of the segment, 8 rows at a time ----
    const bool from_before = now.page0 > 0 && l == a, goes_on = now.page0 + now.take < now.q.pages;
    // what this CTA has of a segment that others have a part of: to the workspace, or to where the ring was, for the cluster
    float* slot = LINE ? ws.partial + (int64_t)(2 * blockIdx.x + (from_before ? 0 : 1)) * kRows * kPitch : reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* mw = merge + warp * 8 * kPitch;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float s = l_run[nt][j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(~0u, s, o);
        if (g == 0) { mw[(2 * t + j) * kPitch + D] = m_run[nt][j]; mw[(2 * t + j) * kPitch + D + 1] = s; }
      }
#pragma unroll
      for (int i = 0; i < kMT; ++i) {
        mw[(2 * t) * kPitch + 16 * i + g] = acc[nt][i][0];
        mw[(2 * t + 1) * kPitch + 16 * i + g] = acc[nt][i][1];
        mw[(2 * t) * kPitch + 16 * i + 8 + g] = acc[nt][i][2];
        mw[(2 * t + 1) * kPitch + 16 * i + 8 + g] = acc[nt][i][3];
      }
      __syncthreads();
      {
        const int row = threadIdx.x >> 4, x = threadIdx.x & 15;
        float f[kWarps], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) { f[w] = merge[(w * 8 + row) * kPitch + D]; M = fmaxf(M, f[w]); }
        const float R = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) { f[w] = fast_exp2(f[w] - R); L += f[w] * merge[(w * 8 + row) * kPitch + D + 1]; }
        const int r = now.tile * kRows + nt * 8 + row;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 64) {
          const int d = d0 + x * 4;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(&merge[(w * 8 + row) * kPitch + d]);
            o.x += f[w] * v.x, o.y += f[w] * v.y, o.z += f[w] * v.z, o.w += f[w] * v.w;
          }
          if (LINE ? from_before || goes_on : stride > 1) {
            *reinterpret_cast<float4*>(slot + (nt * 8 + row) * kPitch + d) = o;
            if (x == 0 && d0 == 0) { slot[(nt * 8 + row) * kPitch + D] = M; slot[(nt * 8 + row) * kPitch + D + 1] = L; }
          } else if (r < now.rows_all) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            T* out = static_cast<T*>(c.out) + (int64_t)(now.q.q0 + token_of(r)) * c.o_ts + (int64_t)(now.head * group + r - token_of(r) * group) * c.o_hs + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2(o.x * inv, o.y * inv, T{}), pack2(o.z * inv, o.w * inv, T{}));
          }
        }
      }
      __syncthreads();
    }
    if constexpr (!LINE) {
      ++l;
      if (stride == 1) continue;
      cluster_sync_all();
      // in the order of the cluster's CTAs; each of them has every cluster-th row, a thread four values of it
      constexpr int kAtOnce = kWarps * 32 * 4 / D;
      for (int row = now.page0 + stride * ((int)threadIdx.x / (D / 4)); row < kRows; row += stride * kAtOnce) {
        const int d = threadIdx.x % (D / 4) * 4, r = now.tile * kRows + row;
        if (r >= now.rows_all) break;
        const uint32_t at = smem_u32(smem) + row * kPitch * 4;
        float2 ml[kMaxCluster];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxCluster; ++i) {
          ml[i] = i < stride ? load2_cluster(map_to_cta(at + D * 4, i)) : make_float2(-INFINITY, 0.f);
          M = fmaxf(M, ml[i].x);
        }
        const float R = M == -INFINITY ? 0.f : M;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kMaxCluster; ++i)
          if (i < stride) {
            const float f = fast_exp2(ml[i].x - R);
            const float4 v = load4_cluster(map_to_cta(at + d * 4, i));
            L += f * ml[i].y;
            o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
          }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int tok = token_of(r);
        T* out = static_cast<T*>(c.out) + (int64_t)(now.q.q0 + tok) * c.o_ts + (int64_t)(now.head * group + r - tok * group) * c.o_hs + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack2(o.x * inv, o.y * inv, T{}), pack2(o.z * inv, o.w * inv, T{}));
      }
      __syncwarp();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                // the next round's copies land where the results were
      cluster_sync_all();
      continue;
    }
    if (threadIdx.x == 0 && l + now.take == b) {                    // the piece's last segment: does it start here and go on?
      Header h{};
      h.last = !from_before && goes_on ? (int)quotient(l - now.page0 + now.q.pages - 1, chunk) : -1;
      h.q0 = now.q.q0, h.n = now.q.n, h.head = now.head, h.tile = now.tile;
      ws.headers[blockIdx.x] = h;
    }
    l += now.take;
  }
}

// Joins the partial results of the segment that starts in piece blockIdx.x, in a fixed order. WIDE: a CTA per query row, every
// warp a share of the pieces; else a warp per row, eight rows a CTA.
template <typename T, int D, bool WIDE> __global__ void __launch_bounds__(256) ob_attend_combine_kernel(const ob::CacheAttendCall c, const FewLayout ws, int rows) {
  constexpr int kPitch = D + 4, kPer = D / 32;
  __shared__ float red[8], total[8], part[8][D];
  follow_previous_kernel();
  const Header h = ws.headers[blockIdx.x];
  if (h.last < 0) return;
  const int group = ws.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = h.last - (int)blockIdx.x + 1;
  const int row = WIDE ? blockIdx.y : blockIdx.y * 8 + warp, r = h.tile * rows + row;
  if (r >= h.n * group) return;
  auto slot = [&](int i) {                                      // i-th partial of the segment
    return ws.partial + ((int64_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * rows + row) * kPitch;
  };
  float m = -INFINITY;
  for (int i = WIDE ? threadIdx.x : lane; i < count; i += WIDE ? 256 : 32) m = fmaxf(m, slot(i)[D]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  if constexpr (WIDE) {
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  }
  const float R = m == -INFINITY ? 0.f : m;
  float o[kPer] = {}, l = 0.f;
#pragma unroll 4
  for (int i = WIDE ? warp : 0; i < count; i += WIDE ? 8 : 1) {
    const float* p = slot(i);
    const float f = fast_exp2(p[D] - R);
    l += f * p[D + 1];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] += f * p[lane + 32 * e];
  }
  T* out = static_cast<T*>(c.out) + (int64_t)(h.q0 + r / group) * c.o_ts + (int64_t)(h.head * group + r % group) * c.o_hs;
  if constexpr (WIDE) {
    if (lane == 0) total[warp] = l;
#pragma unroll
    for (int e = 0; e < kPer; ++e) part[warp][lane + 32 * e] = o[e];
    __syncthreads();
    if (threadIdx.x < D) {
      float sum = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) { sum += part[w][threadIdx.x]; L += total[w]; }
      out[threadIdx.x] = from_f32<T>(L == 0.f ? 0.f : sum / L);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) out[lane + 32 * e] = from_f32<T>(l == 0.f ? 0.f : o[e] / l);
  }
}

// Which kernel has which sequences (the times: contexts of 4096, 32 / 8 heads of 128, this file's kernel / the tensor-memory
// kernel). A row tile of 16 here costs about a quarter of one of 256 there, so up to 64 rows per cache head are this file's:
// 16 sequences of 8 / 16 / 24 tokens take 48 / 88, 92 / 80 and 136 / 81 us, 64 of 8 / 16 171 / 302 and 315 / 305 us; over contexts of
// 512, and with 4 or 8 sequences, 16 tokens are better off here (17 / 18, 29 / 41 and 47 / 64 us). So are sequences of up to 256 rows
// that have as few on the mean (64 single tokens and one sequence of 64: 136 / 299 us), or that leave half the GPU free (one of 32
// tokens: 17 / 25 us). A longer bound far above the mean is that of a prompt among single tokens. Where the sequences are enough to
// fill the GPU on their own, both kernels run, each for its sequences: n single tokens and a prompt of 512 take, so / in the
// prompt's kernel alone, 113 / 150 us for n = 14 and 174 / 310 us for n = 64. Fewer hide behind the prompt's tiles.
constexpr int kFewRows = 64, kFewRowsMost = 256;
struct Plan { bool few, many; int few_rows; };
Plan plan_of(const ob::CacheAttendCall& c) {
  const int64_t group = c.heads / c.kv_heads, rows = c.max_new * group, sms = ob::sm_count();
  if (rows <= kFewRows || (rows <= kFewRowsMost && (c.tokens * group <= kFewRows * c.seqs || c.seqs * c.kv_heads * ((rows + 15) / 16) <= sms)))
    return {true, false, 0x7fffffff};
  const bool both = 4 * c.tokens < c.seqs * c.max_new && 3 * c.seqs * c.kv_heads >= 2 * sms;
  return {both, true, both ? kFewRows : 0};
}
int few_tiles(const ob::CacheAttendCall& c) { return c.max_new * (c.heads / c.kv_heads) <= 8 ? 1 : 2; }
int64_t row_tiles(const ob::CacheAttendCall& c) {                // of a sequence with as many new tokens as the caller's bound
  const int64_t rows = 8 * few_tiles(c);
  return (c.max_new * (c.heads / c.kv_heads) + rows - 1) / rows;
}
// two CTAs per SM, but no more pieces than the block table could fill
int few_grid(const ob::CacheAttendCall& c) {
  const int64_t rows = 8 * few_tiles(c), group = c.heads / c.kv_heads;
  const int64_t tiles = (c.tokens * group + rows - 1) / rows + c.seqs;          // at least the row tiles of all sequences
  const int64_t most = (tiles * c.kv_heads * c.table_width + kMinPages - 1) / kMinPages;
  return (int)std::max<int64_t>(1, std::min<int64_t>(2 * ob::sm_count(), most));
}

constexpr int few_smem(int head_dim) { return kWarps * kRingBytes + kWarps * 8 * (head_dim + 4) * 4; }

// The largest cluster, up to 16 CTAs, that the kernel of one type can be launched with on the current device.
template <typename T, int D, int NT> int placeable() {
  static std::atomic<uint64_t> ready{0};
  if (allow_shared_memory(ob_attend_few_kernel<T, D, NT, false>, few_smem(D), ready, true) != cudaSuccess) {
    cudaGetLastError();                                         // not a later launch's error
    return 0;
  }
  for (int n = kMaxCluster; n >= 1; n /= 2) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)n, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)n), cfg.blockDim = dim3(kWarps * 32), cfg.dynamicSmemBytes = few_smem(D), cfg.attrs = &attr, cfg.numAttrs = 1;
    int clusters = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, ob_attend_few_kernel<T, D, NT, false>, &cfg);
    if (e != cudaSuccess) cudaGetLastError();
    else if (clusters > 0) return n;
  }
  return 0;
}
// The same for both types of queries (the workspace is asked for without a type), looked up once per device. 0 without a device.
int largest_cluster(int head_dim, int row_tiles) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  static std::atomic<int8_t> known[64][2][2];                   // largest + 1
  std::atomic<int8_t>& k = known[dev & 63][head_dim == 128][row_tiles - 1];
  if (const int v = k.load(std::memory_order_acquire)) return v - 1;
  int n = 0;
  auto of = [&](auto d, auto nt) { n = std::min(placeable<__half, decltype(d)::value, decltype(nt)::value>(), placeable<__nv_bfloat16, decltype(d)::value, decltype(nt)::value>()); };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Narrow = std::integral_constant<int, 64>;
  using Wide = std::integral_constant<int, 128>;
  if (head_dim == 128) row_tiles == 1 ? of(Wide{}, One{}) : of(Wide{}, Two{});
  else row_tiles == 1 ? of(Narrow{}, One{}) : of(Narrow{}, Two{});
  k.store((int8_t)(n + 1), std::memory_order_release);
  return n;
}

// CTAs of a cluster per segment, 0: the line of pages. A cluster knows its segment from its number, asks for page numbers at
// once and joins through shared memory: 1 token of 32 heads over 4096 tokens 9.7 us against 18.3 on the line (2.3 us from the
// lengths to the first request saved, and the join kernel), 64 sequences of up to 1024 tokens 18.9 against 38 us (a CTA each;
// the line cuts a third of the segments). But its time is the longest segment's, 1.65 us a round of a page per warp, whatever
// the rest of the batch is: 4 sequences of up to 32768 tokens 40-49 us, on the line 32-56. So it is taken where the block table's
// width bounds the rounds: by 3 more than the line's if all sequences were as long, and for more than one sequence by 16, or 8
// with several CTAs a segment. Clusters of 16 are slower than of 8 as soon as not all are resident (16 segments: 14.6 / 9.1 us).
// What the device cannot place (largest_cluster) is not asked of it: the line needs no cluster.
int few_cluster(const ob::CacheAttendCall& c) {
  const int largest = largest_cluster((int)c.head_dim, few_tiles(c));
  if (largest == 0) return 0;
  const int64_t segments = c.seqs * c.kv_heads * row_tiles(c), sms = ob::sm_count(), slots = 2 * sms, width = c.table_width;
  if (segments > 1 << 24) return 0;
  int n = 1;
  while (n < 8 && n < largest && segments * n * 2 <= slots && width > kMinPages * n) n *= 2;
  if (n == 8 && largest == 16 && segments * 16 <= sms && width > kMinPages * 8) n = 16;
  const int64_t rounds = (width + kWarps * n - 1) / (kWarps * n), line = segments * width / (kWarps * slots);
  return rounds <= line + 3 && (c.seqs == 1 || rounds <= (n == 1 ? 16 : 8)) ? n : 0;
}

template <typename T, int D, int NT> cudaError_t launch_few(const ob::CacheAttendCall& c, void* workspace, cudaStream_t stream) {
  const int grid = few_grid(c);
  constexpr int smem = few_smem(D);
  const int64_t group = c.heads / c.kv_heads;
  FewLayout ws{(int)group, (uint64_t)(((1ll << 40) + group - 1) / group), static_cast<Header*>(workspace), 0, 0,
               reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ((grid * sizeof(Header) + 255) & ~size_t(255)))};
  ws.cluster = few_cluster(c);
  if (ws.cluster > 0) {
    ws.tiles = (int)row_tiles(c);
    static std::atomic<uint64_t> clusters_ready{0};
    cudaError_t e = allow_shared_memory(ob_attend_few_kernel<T, D, NT, false>, smem, clusters_ready, true);
    if (e != cudaSuccess) return e;
    return launch_following(ob_attend_few_kernel<T, D, NT, false>, dim3((unsigned)(c.seqs * c.kv_heads * ws.tiles * ws.cluster)), kWarps * 32, smem, stream,
                            ClusterOf{ws.cluster}, c, ws);
  }
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_shared_memory(ob_attend_few_kernel<T, D, NT, true>, smem, ready);
  if (e != cudaSuccess) return e;
  e = launch_following(ob_attend_few_kernel<T, D, NT, true>, dim3(grid), kWarps * 32, smem, stream, c, ws);
  if (e != cudaSuccess) return e;
  // With fewer segments than a sixteenth of the pieces a segment may have many partial results: then a row gets a whole CTA. Most
  // CTAs of either grid find nothing to join, and their number is what the small grid saves (5.3 us against 2 us for 16 rows).
  const int64_t segments = c.kv_heads * (c.tokens * group / (8 * NT) + 1);
  if (segments * 16 < grid) return launch_following(ob_attend_combine_kernel<T, D, true>, dim3(grid, 8 * NT), 256, 0, stream, c, ws, 8 * NT);
  return launch_following(ob_attend_combine_kernel<T, D, false>, dim3(grid, NT), 256, 0, stream, c, ws, 8 * NT);
}

}  // namespace

namespace ob {

static CacheAttendCall few_part(CacheAttendCall c, const Plan& p) {
  c.few_rows = p.few_rows;
  if (p.many) c.max_new = 1;                                    // what is short next to a prompt is a single token as a rule
  return c;
}

static int64_t few_workspace(const CacheAttendCall& c) {
  if (few_cluster(c) > 0) return 0;
  const int64_t grid = few_grid(c);
  return ((grid * (int64_t)sizeof(Header) + 255) & ~255ll) + 2 * grid * 8 * few_tiles(c) * (c.head_dim + 4) * 4;
}

int64_t cache_attend_workspace(const CacheAttendCall& c) {
  const Plan p = plan_of(c);
  return (p.few ? (few_workspace(few_part(c, p)) + 255) & ~255ll : 0) + (p.many ? cache_attend_many_workspace(c) : 0);
}

cudaError_t launch_cache_attend(const CacheAttendCall& call, void* workspace, cudaStream_t stream) {
  const Plan p = plan_of(call);
  if (p.few) {
    const CacheAttendCall c = few_part(call, p);
    auto by_tiles = [&](auto t, auto d) {
      return few_tiles(c) == 1 ? launch_few<decltype(t), decltype(d)::value, 1>(c, workspace, stream)
                               : launch_few<decltype(t), decltype(d)::value, 2>(c, workspace, stream);
    };
    auto by_dim = [&](auto t) {
      return c.head_dim == 64 ? by_tiles(t, std::integral_constant<int, 64>{}) : by_tiles(t, std::integral_constant<int, 128>{});
    };
    const cudaError_t e = c.bf16 ? by_dim(__nv_bfloat16{}) : by_dim(__half{});
    if (e != cudaSuccess || !p.many) return e;
    workspace = static_cast<uint8_t*>(workspace) + ((few_workspace(c) + 255) & ~255ll);
  }
  CacheAttendCall c = call;
  c.few_rows = p.few_rows;
  return launch_cache_attend_many(c, workspace, stream);
}

cudaError_t read_attend_status(int* wait, int* batch) {
  const cudaError_t e = take_status(g_attend_status, wait);
  return e == cudaSuccess ? take_status(g_attend_batch, batch) : e;
}

}  // namespace ob
