// Attention over the 8-bit cache for many query rows (prompts, chunks of prompts), on tcgen05.
//
// One CTA owns 256 query rows of a cache head -- the rows of all heads of its group, token by token, so that a group shares
// the keys -- as two tiles of 128, and walks over the cached tokens 128 at a time:
//   * producers (7 warps) fetch two pages' keys and values with 16-byte loads one step ahead, widen e4m3 to fp16 (exact) and
//     store them as K-major operands with the 128-byte swizzle. The pages' layout makes both K-major: keys (token, dim) for
//     S = Q K^T, values (dim, token) for O += P V. Widening once per CTA costs what a TMA load of fp16 would cost in shared
//     memory, and the cache is read at 8 bits;
//   * one warp issues tcgen05.mma (M = 128, fp32 accumulators in tensor memory): the products of one tile run while the other
//     tile's softmax does;
//   * softmax (4 warps per tile, thread = row): the row's scores are read from tensor memory, the weights go back as fp16 over
//     the scores' own columns and are the A operand of the second product. The running maximum is only raised, and O
//     multiplied, when a weight would otherwise pass 2^kRaise (the lazy rescaling that is published for attention kernels of this
//     kind). Weights are 2^(t - M + kWeightShift): fp16's range above the reference holds what the maximum lags behind, all
//     below it keeps small weights. Rounded to fp16 (2^-11) for the product, fp32 in the sum: full precision down to 2^-25 of the
//     reference, lost below 2^-36. Raised at 2^8 / 2^4 / 2^2 a prompt of 8192 takes 593 / 599 / 639 us; at 2^8 the four bits less
//     would be missing where one token has nearly all the weight and its page is louder than the others.
// Scales as in cache_attend.cu: the key scale multiplies the score, the value scale goes into the exponent.
// Long caches with too few row tiles to fill the chip are split along the cached tokens; the parts are joined by a second kernel.
// Measured: a prompt of 8192, 32 / 8 heads of 128, 600 us (916 TFLOP/s of the causal half, 55 % of the cuBLAS rate). No unit is
// saturated: the softmax's instructions and the widening share the issue slots and wait for each other (leaving out either, or
// the products, changes the time by 2 to 8 %).
// Every mbarrier wait is bounded. No TMA.
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

__device__ int g_attend_many_status, g_attend_many_batch;       // code of a wait that gave up; see note_bad_batch

constexpr int kTileRows = 128, kCtaRows = 256, kTileTokens = 128;
constexpr int kProducers = 7;                                   // warps
constexpr int kThreads = 32 * (8 + 1 + kProducers);
// registers: the softmax warps hold a row's 128 scores; 256 threads of either kind share what 512 x 128 were launched with
constexpr int kSoftmaxRegs = 168, kServiceRegs = 88;
static_assert(kThreads == 512 && kSoftmaxRegs + kServiceRegs <= 256, "register split");
constexpr float kRaise = 4.f, kWeightShift = 11.f;              // see above
static_assert(kRaise + kWeightShift <= 15.f, "a weight has to fit fp16");

template <int D> struct Cfg {
  static constexpr int kQBytes = kTileRows * D * 2;             // per tile
  static constexpr int kSlotBytes = kTileTokens * D * 2;        // keys or values of a step as fp16
  static constexpr int kSlots = D == 64 ? 8 : 4;                // keys in even slots, values in odd ones
  static constexpr int kSmem = 2 * kQBytes + kSlots * kSlotBytes + 1024;
  static_assert(kSmem <= 226 * 1024, "shared memory");
  static constexpr int kTmemS = 0, kTmemO = 256;                // S / P of tile g at 128 g, O of tile g at 256 + D g
};

// true in exactly one lane of a converged warp (the same lane every time)
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 columns of this warp's lanes, without the wait
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
// the wait, with the loaded registers as operands: nothing that uses them can be moved before it
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[128]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 128; ++i) asm volatile("" : "+r"(r[i]));
}
// scores from column `seen` on become -inf
__device__ __forceinline__ void hide(uint32_t (&v)[128], int seen) {
#pragma unroll
  for (int i = 0; i < 128; ++i)
    if (i >= seen) v[i] = 0xFF800000u;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T, int D> __global__ void __launch_bounds__(kThreads, 1)
ob_attend_many_kernel(const ob::CacheAttendCall c, float* partial, int splits) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  struct Meta { float ks, vs; };                                // of a page; vs < 0: there is none
  // the pages of step j in [j % kMeta]: a slot is filled again when its scores are done, which is before the softmax has
  // read the page data; by the second refill that softmax is over (its weights were needed for the scores in between)
  constexpr int kMeta = C::kSlots;
  __shared__ Meta meta[kMeta][2];
  __shared__ __align__(8) uint64_t bar_full[C::kSlots], bar_empty[C::kSlots];
  __shared__ __align__(8) uint64_t bar_q[2], bar_s[2], bar_p[2][2], bar_o[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int found;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = (int)(c.heads / c.kv_heads), H = (int)c.kv_heads;
  long long budget = 2000000000ll;

  // ---- which rows: sequence s owns the row tiles [floor(q_start[s] group / 256) + s, the same of s + 1) of the grid ----
  const int slots = gridDim.x / H;
  const int head = blockIdx.x % H, slot = slots - 1 - (int)(blockIdx.x / H);     // the long causal tiles first
  const Starts starts{c.q_start, (int)c.seqs, (int)c.tokens};
  auto place = [&](int start) { return (int)((int64_t)start * group / kCtaRows); };
  if (threadIdx.x == 0) found = min(starts.seqs, slot + 1);
  __syncthreads();
  bool bad = false;
  {
    int n = starts.seqs;
    for (int s = threadIdx.x; s < starts.seqs; s += kThreads) {
      const int start = starts.at(s, bad);
      n = min(n, starts.behind_slot(s, start, slot, place(start)));
    }
    n = __reduce_min_sync(~0u, n);
    if (lane == 0) atomicMin(&found, n);
  }
  bad = __syncthreads_or(bad);
  if (bad && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) note_bad_batch(&g_attend_many_batch);
  const int seq = found - 1;
  if (seq < 0) return;
  if (bad && starts.left_out(seq)) return;
  const int q0 = __ldg(c.q_start + seq), q1 = __ldg(c.q_start + seq + 1), kv_raw = __ldg(c.kv_len + seq);
  const int tile = slot - place(q0) - seq;
  const int n = q1 - q0, rows_all = n * group, row0 = tile * kCtaRows;
  if (rows_all <= c.few_rows) return;                           // cache_attend.cu's
  if (row0 >= rows_all) return;
  const int kv = (int)min((int64_t)max(kv_raw, 0), c.table_width * kPageTokens);
  if (kv < kv_raw && threadIdx.x == 0) note_bad_batch(&g_attend_many_batch);
  auto limit_of = [&](int r) { return c.causal ? min(kv, kv_raw - n + r / group + 1) : kv; };
  const int hi = max(0, limit_of(min(rows_all, row0 + kCtaRows) - 1));
  const int steps_all = (hi + kTileTokens - 1) / kTileTokens;
  const int per = (steps_all + splits - 1) / splits, j0 = (int)blockIdx.y * per;
  const int steps = max(0, min(per, steps_all - j0));
  const bool two = rows_all - row0 > kTileRows;                 // the second tile has rows

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(smem_u32(&bar_full[i]), kProducers);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&bar_q[g]), 4);
      mbar_init(smem_u32(&bar_s[g]), 2);                        // the MMAs' commit, and the issuing thread itself (page data)
      mbar_init(smem_u32(&bar_p[g][0]), 4);
      mbar_init(smem_u32(&bar_p[g][1]), 4);
      mbar_init(smem_u32(&bar_o[g]), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) tcgen05_alloc(smem_u32(&tmem_slot), 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t q_at = base, ring_at = base + 2 * C::kQBytes;

  if (warp < 8) {
    // ---------------- softmax: thread = row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int g = warp >> 2, quad = warp & 3, in_tile = quad * 32 + lane;
    const int r = row0 + g * kTileRows + in_tile;
    const bool live = r < rows_all;
    if (g == 1 && !two) {
    } else {
      const int64_t tok = q0 + r / group;
      const int hd = head * group + r % group;
      float unit = 1.f;
      {
        const T* row = static_cast<const T*>(c.q) + tok * c.q_ts + (int64_t)hd * c.q_hs;
        uint4 raw[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) raw[i] = live ? *reinterpret_cast<const uint4*>(row + 8 * i) : make_uint4(0, 0, 0, 0);
        float inv = 1.f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) { const float2 f = unpack2(w[e], T{}); m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y))); }
          }
          const int e = min(max((int)(__float_as_uint(m) >> 23), 2), 252);       // see cache_attend.cu
          unit = __uint_as_float((uint32_t)e << 23);
          inv = __uint_as_float((uint32_t)(254 - e) << 23);
        }
        const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;                   // the maximum is taken before the scale
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
              const float2 f = unpack2(w[e], T{});
              w[e] = pack2(f.x * inv, f.y * inv, __half{});
            }
            w[e] ^= flip;
          }
          uint8_t* dst = gen + (q_at - base) + g * C::kQBytes + (i / 8) * (kTileRows * 128) + in_tile * 128 + (((i & 7) ^ (in_tile & 7)) << 4);
          *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_q[g]));
      }
      const float coef = unit * fabsf(c.scale) * 1.4426950408889634f;
      const int limit = live ? limit_of(r) : 0x7fffffff;
      int least = limit;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(~0u, least, o));
      const uint32_t s_col = tmem + ((uint32_t)(quad * 32) << 16) + C::kTmemS + 128 * g;
      const uint32_t o_col = tmem + ((uint32_t)(quad * 32) << 16) + C::kTmemO + D * g;
      float M = -INFINITY, L = 0.f;

      for (int j = 0; j < steps; ++j) {
        const int tok0 = (j0 + j) * kTileTokens;
        mbar_wait(smem_u32(&bar_s[g]), j & 1, budget, &g_attend_many_status, 4);
        __syncwarp();
        tcgen05_fence_after();
        const bool masked = tok0 + kTileTokens > least;
        uint32_t v[kTileTokens];
#pragma unroll
        for (int h = 0; h < 4; ++h) tmem_ld32(s_col + h * 32, v + h * 32);
        // never 0: a masked score is -inf, and -inf * 0 would be NaN
        const Meta md[2] = {meta[j % kMeta][0], meta[j % kMeta][1]};
        const float k[2] = {fmaxf(coef * md[0].ks, 1e-37f), fmaxf(coef * md[1].ks, 1e-37f)};
        // no page: no weight
        const float log2_vs[2] = {md[0].vs < 0.f ? -INFINITY : __log2f(md[0].vs), md[1].vs < 0.f ? -INFINITY : __log2f(md[1].vs)};
        tmem_landed(v);
        if (masked) hide(v, limit - tok0);
        float top = -INFINITY;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float m[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(v[p * 64 + i]);
#pragma unroll
          for (int i = 4; i < 60; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], fmaxf(__uint_as_float(v[p * 64 + i + e]), __uint_as_float(v[p * 64 + i + 4 + e])));
#pragma unroll
          for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], __uint_as_float(v[p * 64 + 60 + e]));
          top = fmaxf(top, fmaf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), k[p], log2_vs[p]));
        }
        const bool raise = top > M + kRaise || (M == -INFINITY && top > M);
        if (__any_sync(~0u, raise)) {
          const float to = fmaxf(M, top);
          const float f = to == -INFINITY ? 1.f : exp2f(M - to);
          M = to;
          L *= f;
          if (j > 0) {
            mbar_wait(smem_u32(&bar_o[g]), (j - 1) & 1, budget, &g_attend_many_status, 5);
            __syncwarp();
            tcgen05_fence_after();
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              uint32_t o[16];
              tmem_ld16(o_col + d, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(o_col + d, o);
            }
            tcgen05_wait_st();
          }
        }
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const float off = log2_vs[p] - ref + kWeightShift;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float x = ex2(fmaf(__uint_as_float(v[p * 64 + 2 * i]), k[p], off)), y = ex2(fmaf(__uint_as_float(v[p * 64 + 2 * i + 1]), k[p], off));
            sum[(2 * i) & 3] += x;
            sum[(2 * i + 1) & 3] += y;
            v[p * 32 + i] = pack2(x, y, __half{});              // over scores that have been used
          }
          tcgen05_st_32x32b_x32_nowait(s_col + p * 32, reinterpret_cast<uint32_t(&)[32]>(v[p * 32]));
          L += md[p].vs < 0.f ? 0.f : __fdividef((sum[0] + sum[1]) + (sum[2] + sum[3]), md[p].vs);
          tcgen05_wait_st();                                    // the page's weights can be multiplied while the other's are computed
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_p[g][p]));
        }
      }

      // ---- result ----
      if (steps > 0) {
        mbar_wait(smem_u32(&bar_o[g]), (steps - 1) & 1, budget, &g_attend_many_status, 6);
        __syncwarp();
        tcgen05_fence_after();
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      float* part = partial + ((int64_t)blockIdx.y * c.tokens * c.heads + tok * c.heads + hd) * (D + 4);
      T* out = static_cast<T*>(c.out) + tok * c.o_ts + (int64_t)hd * c.o_hs;
      if (splits > 1 && live) { part[D] = M; part[D + 1] = L; }
#pragma unroll
      for (int d = 0; d < D; d += 32) {
        uint32_t v[32];
        if (steps > 0) {
          tcgen05_ld_32x32b_x32(o_col + d, v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (!live) continue;
        if (splits > 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(part + d + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = L == 0.f ? 0.f : __uint_as_float(v[8 * i + e]) * inv;
            store8(out + d + 8 * i, f);
          }
        }
      }
      tcgen05_fence_before();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kServiceRegs));
    if (warp == 8) {
    // ---------------- MMA issue ----------------
    // The warp stays converged and only the tcgen05 instructions are predicated on one lane, so that descriptors stay in
    // uniform registers: 64 cycles per M = N = 128 instruction, the tensor core's own pace, against 100 from a branch on the lane.
    const uint32_t idesc_s = (1u << 4) | ((uint32_t)(kTileTokens >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
    const uint32_t idesc_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
    const int tiles = two ? 2 : 1;
    const bool first = elect_one();
    const uint64_t q_desc = make_desc(q_at, 16, 1024, kLayoutSw128), ring_desc = make_desc(ring_at, 16, 1024, kLayoutSw128);
    auto wait_full = [&](int item) {
      mbar_wait(smem_u32(&bar_full[item % C::kSlots]), (item / C::kSlots) & 1, budget, &g_attend_many_status, 2);
      tcgen05_fence_after();
    };
    auto scores = [&](int g, int j) {
      const int slot = 2 * j % C::kSlots;
      const uint64_t qd = q_desc + (uint64_t)(g * (C::kQBytes >> 4)), kd = ring_desc + (uint64_t)(slot * (C::kSlotBytes >> 4));
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        if (first)
          mma_f16_ss(tmem + C::kTmemS + 128 * g, qd + (uint64_t)(((k / 4) * (kTileRows * 128) + (k % 4) * 32) >> 4),
                     kd + (uint64_t)(((k / 4) * (kTileTokens * 128) + (k % 4) * 32) >> 4), idesc_s, k > 0);
      if (first) tcgen05_commit(smem_u32(&bar_s[g]));
      if (first) mbar_arrive(smem_u32(&bar_s[g]));
      if (first && g == tiles - 1) tcgen05_commit(smem_u32(&bar_empty[slot]));
    };
    for (int g = 0; g < tiles; ++g) mbar_wait(smem_u32(&bar_q[g]), 0, budget, &g_attend_many_status, 1);
    if (steps > 0) {
      wait_full(0);
      for (int g = 0; g < tiles; ++g) scores(g, 0);
    }
    for (int j = 0; j < steps; ++j) {
      const int slot = (2 * j + 1) % C::kSlots;
      wait_full(2 * j + 1);
      if (j + 1 < steps) wait_full(2 * j + 2);
      for (int g = 0; g < tiles; ++g) {
        const uint64_t vd = ring_desc + (uint64_t)(slot * (C::kSlotBytes >> 4));
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          mbar_wait(smem_u32(&bar_p[g][p]), j & 1, budget, &g_attend_many_status, 3);
          tcgen05_fence_after();
#pragma unroll
          for (int k = 4 * p; k < 4 * p + 4; ++k)
            if (first)
              mma_f16_ts(tmem + C::kTmemO + D * g, tmem + C::kTmemS + 128 * g + 8 * k, vd + (uint64_t)((p * (D * 128) + (k % 4) * 32) >> 4), idesc_o,
                         j > 0 || k > 0);
        }
        if (first) tcgen05_commit(smem_u32(&bar_o[g]));
        if (first && g == tiles - 1) tcgen05_commit(smem_u32(&bar_empty[slot]));
        if (j + 1 < steps) {
          // the next scores go over the weights' columns, and instructions on different accumulators are not ordered among
          // themselves: they wait until the product with those weights is complete (2 % of the kernel's time)
          mbar_wait(smem_u32(&bar_o[g]), j & 1, budget, &g_attend_many_status, 9);
          tcgen05_fence_after();
          scores(g, j + 1);
        }
      }
    }
    } else {
    // ---------------- producers: items 2 j (keys of step j) and 2 j + 1 (values), both by the same code ----------------
    const int pw = warp - 9;
    // Work in units of 8 rows x 64 bytes, one per warp and turn: a lane takes 16 bytes, a quarter warp 8 rows, whose
    // widened halves the swizzle spreads over all banks. An item is two pages; a page's rows are D values of a key or 64 tokens of
    // a value, 128 bytes of fp16 in a row of a column block.
    constexpr int kUnits = kTileTokens * D / 512;               // of an item
    constexpr int kTurns = (kUnits + kProducers - 1) / kProducers;
    constexpr int kPageHead = kPageTokens * D;
    const int row = lane & 7, piece = lane >> 3;
    const int put0 = row * 128 + (((2 * piece) ^ row) << 4), put1 = row * 128 + (((2 * piece + 1) ^ row) << 4);
    const int* table = c.table + (int64_t)seq * c.table_stride;
    // Page numbers are fetched two steps ahead, pages one; nothing is looked at where it is fetched, so that no fetch is
    // waited for. ids < 0: no page.
    auto look_up = [&](int j, int (&ids)[2]) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int64_t pg = (int64_t)(j0 + j) * 2 + p;
        ids[p] = j < steps && pg * kPageTokens < kv ? __ldg(table + pg) : -2;       // -2: behind the end, not an error
      }
    };
    auto held = [&](int id) { return id >= 0 && id < c.pages; };
    auto at_page = [&](int id) { return (int64_t)(held(id) ? id : 0) * H + head; };
    auto load = [&](bool values, const int (&ids)[2], uint4 (&x)[kTurns]) {
      const uint8_t* pool = static_cast<const uint8_t*>(values ? c.v_pages : c.k_pages);
      const bool narrow = values || D == 64;                    // rows of 64 bytes: a unit is 512 bytes in a row
      const int mine = row * (narrow ? 64 : 128) + piece * 16;
      const uint8_t* page[2] = {pool + at_page(ids[0]) * kPageHead + mine, pool + at_page(ids[1]) * kPageHead + mine};
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int u = i * kProducers + pw, w = u & (kUnits / 2 - 1);
        if (u < kUnits) x[i] = __ldg(reinterpret_cast<const uint4*>((u < kUnits / 2 ? page[0] : page[1]) + (narrow ? w * 512 : (w >> 1) * 1024 + (w & 1) * 64)));
      }
    };
    const bool scaler = pw == kProducers - 1 && lane < 2;       // two lanes that also fetch the scales, of a page each
    float2 scales{};
    auto load_scales = [&](const int (&ids)[2]) {
      const int64_t at = at_page(lane == 0 ? ids[0] : ids[1]);
      scales = make_float2(__ldg(c.k_scale + at), __ldg(c.v_scale + at));
    };
    int now[2], next[2], later[2];                              // pages of the step in hand, of the next and of the one behind
    look_up(0, now);
    look_up(1, next);
    look_up(2, later);
    uint4 x[2][kTurns];
    if (steps > 0) {
      load(false, now, x[0]);
      load(true, now, x[1]);
      if (scaler) load_scales(now);
    }
    for (int j = 0; j < steps; ++j) {
#pragma unroll
      for (int values = 0; values < 2; ++values) {
        const int item = 2 * j + values, slot = item % C::kSlots;
        if (!held(now[0]) || !held(now[1])) {
          if ((!held(now[0]) && now[0] != -2) || (!held(now[1]) && now[1] != -2)) note_bad_batch(&g_attend_many_batch);
#pragma unroll
          for (int i = 0; i < kTurns; ++i)
            if (!held(i * kProducers + pw < kUnits / 2 ? now[0] : now[1])) x[values][i] = make_uint4(0, 0, 0, 0);
        }
        const int tok0 = (j0 + j) * kTileTokens;
        if (values && tok0 + kTileTokens > kv) {                // bytes behind the end may be anything: zeros instead
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            const int live = kv - (tok0 + (i * kProducers + pw < kUnits / 2 ? 0 : kPageTokens) + piece * 16);
            uint32_t* w = reinterpret_cast<uint32_t*>(&x[values][i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int l = live - 4 * e;
              w[e] &= l >= 4 ? ~0u : l <= 0 ? 0u : ~0u >> (8 * (4 - l));
            }
          }
        }
        if (!values && scaler) meta[j % kMeta][lane] = {scales.x, held(lane == 0 ? now[0] : now[1]) ? fmaxf(scales.y, 5.421010862e-20f) : -1.f};   // see cache_attend.cu
        mbar_wait(smem_u32(&bar_empty[slot]), ((item / C::kSlots) & 1) ^ 1, budget, &g_attend_many_status, 7);
        __syncwarp();
        uint8_t* dst = gen + (ring_at - base) + slot * C::kSlotBytes;
        const bool narrow = values || D == 64;
        // keys: rows of both pages below each other, a column block for each 64 dims; values: a column block for each page
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
          const int u = i * kProducers + pw;
          if (u >= kUnits) break;
          uint8_t* at = dst + (narrow ? u * 1024 : (u >> 1) * 1024 + (u & 1) * (kTileTokens * 128));
          uint4 a, b;
          a.x = e4m3_lo(x[values][i].x), a.y = e4m3_hi(x[values][i].x), a.z = e4m3_lo(x[values][i].y), a.w = e4m3_hi(x[values][i].y);
          b.x = e4m3_lo(x[values][i].z), b.y = e4m3_hi(x[values][i].z), b.z = e4m3_lo(x[values][i].w), b.w = e4m3_hi(x[values][i].w);
          *reinterpret_cast<uint4*>(at + put0) = a;
          *reinterpret_cast<uint4*>(at + put1) = b;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_full[slot]));
        if (j + 1 < steps) {
          load(values, next, x[values]);
          if (!values && scaler) load_scales(next);
        }
      }
      now[0] = next[0], now[1] = next[1], next[0] = later[0], next[1] = later[1];
      look_up(j + 3, later);
    }
    }
  }
  __syncthreads();
  if (warp == 8) {
    tcgen05_fence_after();
    tcgen05_dealloc(tmem, 512);
  }
}

// Joins the splits of a row: one warp per (token, head).
template <typename T, int D> __global__ void __launch_bounds__(256) ob_attend_join_kernel(const ob::CacheAttendCall c, const float* partial, int splits) {
  follow_previous_kernel();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = c.tokens * c.heads;
  if (row >= rows) return;
  const int t = (int)(row / c.heads);
  const Starts starts{c.q_start, (int)c.seqs, (int)c.tokens};
  int first = starts.seqs + 1;                                  // sequence first - 1 holds the token
  bool bad = false;
  for (int s = lane; s <= starts.seqs; s += 32) {
    const int start = starts.at(s, bad);
    first = min(first, starts.behind_row(s, start, t));
  }
  first = __reduce_min_sync(~0u, first);
  if (first < 1 || first > c.seqs) return;                      // padding: not written
  if (__any_sync(~0u, bad) && starts.left_out(first - 1)) return;
  const int q0 = c.q_start[first - 1], q1 = c.q_start[first];
  if ((q1 - q0) * (c.heads / c.kv_heads) <= c.few_rows) return;
  const float* p = partial + row * (D + 4);
  const int64_t step = rows * (D + 4);
  float M = -INFINITY;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, p[s * step + D]);
  const float R = M == -INFINITY ? 0.f : M;
  float L = 0.f, o[D / 32] = {};
  for (int s = 0; s < splits; ++s) {
    const float f = exp2f(p[s * step + D] - R);
    L += f * p[s * step + D + 1];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] += f * p[s * step + lane + 32 * e];
  }
  T* out = static_cast<T*>(c.out) + t * c.o_ts + (row % c.heads) * c.o_hs;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) out[lane + 32 * e] = from_f32<T>(L == 0.f ? 0.f : o[e] / L);
}

int64_t many_slots(const ob::CacheAttendCall& c) { return c.tokens * (c.heads / c.kv_heads) / kCtaRows + c.seqs; }

// Parts that the cache is cut into, for row tiles too few to fill the GPU: the number with the least estimated time, from what
// was measured for heads of 128 values: 2.3 us a step of 128 tokens (64 values: 1.95), 11 us a CTA besides, and for the join 4 us
// and the partial results at 1.7 TB/s. 32 / 8 heads, in 1 / 2 / 4 / 8 parts: 512 tokens over 4096 86 / 63 / 79 / 111 us (2 taken),
// 128 over 4096 86 / 56 / 39 / 33 (8), 2048 over 2048 58 / 123 / 187 / 307 (1), 3 x 512 over 16384 604 / 510 / 557 / 622 (2; the
// estimate misses 3 parts there, 482 us, by 6 %). It counts the table's width for every sequence: a table much wider than the
// batch's longest sequence is cut too often (2048 tokens in a table of 32768: 159 us), so callers pass a table as wide as they need.
int many_splits(const ob::CacheAttendCall& c) {
  const int64_t group = c.heads / c.kv_heads, sms = ob::sm_count(), steps = (c.table_width + 1) / 2;
  const int64_t ctas = ((c.tokens * group + kCtaRows - 1) / kCtaRows + (c.seqs - 1) / 2) * c.kv_heads;
  const double step = c.head_dim == 128 ? 2.3 : 1.95, bytes = (double)c.tokens * c.heads * (c.head_dim + 4) * 4;
  int best = 1;
  double least = 0;
  for (int n = 1; n <= 64 && n <= steps; ++n) {
    const double waves = ctas * n <= sms ? 1. : (double)(ctas * n) / sms + .5;
    const double us = waves * ((steps + n - 1) / n * step + 11) + (n > 1 ? 4 + n * bytes / 1.7e6 : 0.);
    if (n == 1 || us < least) best = n, least = us;
  }
  return best;
}

template <typename T, int D> cudaError_t launch_many(const ob::CacheAttendCall& c, void* workspace, cudaStream_t stream) {
  const int splits = many_splits(c);
  float* partial = static_cast<float*>(workspace);
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_shared_memory(ob_attend_many_kernel<T, D>, Cfg<D>::kSmem, ready);
  if (e != cudaSuccess) return e;
  ob_attend_many_kernel<T, D><<<dim3((unsigned)(many_slots(c) * c.kv_heads), splits), kThreads, Cfg<D>::kSmem, stream>>>(c, partial, splits);
  e = cudaGetLastError();
  if (e != cudaSuccess || splits == 1) return e;
  return launch_following(ob_attend_join_kernel<T, D>, dim3((unsigned)((c.tokens * c.heads + 7) / 8)), 256, 0, stream, c, partial, splits);
}

}  // namespace

namespace ob {

int64_t cache_attend_many_workspace(const CacheAttendCall& c) {
  const int splits = many_splits(c);
  return splits == 1 ? 0 : splits * c.tokens * c.heads * (c.head_dim + 4) * 4;
}

cudaError_t launch_cache_attend_many(const CacheAttendCall& c, void* workspace, cudaStream_t stream) {
  if (c.bf16) return c.head_dim == 64 ? launch_many<__nv_bfloat16, 64>(c, workspace, stream) : launch_many<__nv_bfloat16, 128>(c, workspace, stream);
  return c.head_dim == 64 ? launch_many<__half, 64>(c, workspace, stream) : launch_many<__half, 128>(c, workspace, stream);
}

cudaError_t read_attend_many_status(int* wait, int* batch) {
  const cudaError_t e = take_status(g_attend_many_status, wait);
  return e == cudaSuccess ? take_status(g_attend_many_batch, batch) : e;
}

}  // namespace ob
