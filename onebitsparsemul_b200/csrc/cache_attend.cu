// Attention over the 8-bit cache, plain form: one warp per query row.
#include "block_common.h"
#include "kernels.h"

namespace {

using namespace ob_block;

__device__ int g_attend_status;

template <typename T, int D> __global__ void __launch_bounds__(128) ob_cache_attend_simple_kernel(const ob::CacheAttendCall c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + warp;
  if (row >= c.tokens * c.heads) return;
  const int t = (int)(row / c.heads), head = (int)(row % c.heads);
  int count = 0;
  for (int s0 = 0; s0 <= c.seqs; s0 += 32) count += __popc(__ballot_sync(~0u, s0 + lane <= c.seqs && c.q_start[s0 + lane] <= t));
  if (count < 1 || count > c.seqs) return;
  const int seq = count - 1;
  const int kv = min(c.kv_len[seq], (int)c.table_width * kPageTokens);
  const int limit = c.causal ? min(kv, c.kv_len[seq] - c.q_start[seq + 1] + t + 1) : kv;   // tokens that this row sees
  const int kvh = head / (int)(c.heads / c.kv_heads);
  __shared__ float qs[4][D];
  const T* q = static_cast<const T*>(c.q) + t * c.q_ts + head * c.q_hs;
  for (int d = lane; d < D; d += 32) qs[warp][d] = to_f32(q[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
  for (int p0 = 0; p0 < limit; p0 += kPageTokens) {
    const int page = c.table[seq * c.table_stride + p0 / kPageTokens];
    if (page < 0 || page >= c.pages) {
      if (lane == 0) atomicCAS(&g_attend_status, 0, kStatusBadBatch);
      continue;
    }
    const int64_t ph = (int64_t)page * c.kv_heads + kvh;
    const uint8_t* kp = static_cast<const uint8_t*>(c.k_pages) + ph * kPageTokens * D;
    const uint8_t* vp = static_cast<const uint8_t*>(c.v_pages) + ph * kPageTokens * D;
    const float ks = c.k_scale[ph] * c.scale, vs = c.v_scale[ph];
    float s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = lane + 32 * h;
      float acc = 0.f;
      for (int d = 0; d < D; ++d) acc += qs[warp][d] * from_e4m3(kp[tok * D + d]);
      s[h] = p0 + tok < limit ? acc * ks : -INFINITY;
    }
    float mx = fmaxf(s[0], s[1]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, k));
    const float mn = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.f : __expf(m - mn);
    l *= f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] *= f;
    m = mn;
    float pr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      pr[h] = p0 + lane + 32 * h < limit ? expf(s[h] - mn) : 0.f;
      l += pr[h];
    }
    const int seen = min(kPageTokens, limit - p0);
    for (int tok = 0; tok < seen; ++tok) {
      const float w = __shfl_sync(~0u, tok < 32 ? pr[0] : pr[1], tok & 31) * vs;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] += w * from_e4m3(vp[(lane + 32 * i) * kPageTokens + tok]);
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(~0u, l, k);
  T* out = static_cast<T*>(c.out) + t * c.o_ts + head * c.o_hs;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) out[lane + 32 * i] = from_f32<T>(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace

namespace ob {

int64_t cache_attend_workspace(const CacheAttendCall&) { return 0; }

cudaError_t launch_cache_attend(const CacheAttendCall& c, void*, cudaStream_t stream) {
  const unsigned grid = (unsigned)((c.tokens * c.heads + 3) / 4);
  if (c.bf16) {
    if (c.head_dim == 64) ob_cache_attend_simple_kernel<__nv_bfloat16, 64><<<grid, 128, 0, stream>>>(c);
    else ob_cache_attend_simple_kernel<__nv_bfloat16, 128><<<grid, 128, 0, stream>>>(c);
  } else {
    if (c.head_dim == 64) ob_cache_attend_simple_kernel<__half, 64><<<grid, 128, 0, stream>>>(c);
    else ob_cache_attend_simple_kernel<__half, 128><<<grid, 128, 0, stream>>>(c);
  }
  return cudaGetLastError();
}

cudaError_t read_attend_status(int* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_attend_status, sizeof(int));
  if (e != cudaSuccess || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_attend_status, &zero, sizeof(int));
}

}  // namespace ob
