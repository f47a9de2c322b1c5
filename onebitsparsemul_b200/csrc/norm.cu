// Residual add with the norms around it, one pass over the row:
//   u = x                                                        (no post_weight)
//   u = x / sqrt(mean(x^2) + eps) * post_weight                  (a norm after the block)
//   h = residual + residual_scale * gate * u                     (gate: one value per channel, per value, or absent)
//   y = h / sqrt(mean(h^2) + eps) * weight                       (the norm before the next block; of h before its rounding)
// Without a residual h = x and only y is written. The row lives in registers between its one read and its one write, both
// sums are fp32: per-thread partial sums, then shuffles (and, above one warp per row, shared memory) in a fixed order.
#include "block_common.h"
#include "kernels.h"

namespace {

using namespace ob_block;

struct NormArgs {
  const void *x, *residual, *gate, *post_weight, *weight;
  void *y, *h;
  int64_t x_stride, r_stride, g_stride, y_stride, h_stride;   // elements from one row to the next; g_stride 0: one gate row for all
  int64_t rows;
  int hidden;
  float residual_scale, eps;
};

// sum over the threads of one row
template <bool WARP_ROW> __device__ __forceinline__ float row_sum(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (WARP_ROW) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < warps ? scratch[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// W values as they lie in memory
template <typename T, int W> struct Raw {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = from_f32<T>(0.f); }
  __device__ __forceinline__ void values(float (&f)[W]) const { f[0] = to_f32(v); }
};
template <typename T> struct Raw<T, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = unpack2(w[i], T{}); f[2 * i] = x.x; f[2 * i + 1] = x.y; }
  }
};
template <> struct Raw<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void values(float (&f)[8]) const { f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w; }
};

// V chunks of W values per thread; chunk j of thread t starts at value (j * threads_of_row + t) * W. W = 8: 16-byte accesses
// (hidden % 8 == 0 and every row aligned); W = 1: any width and alignment, bound by its 2-byte accesses (1111 x 2047: 2.9 TB/s).
// Bound by memory on many rows: what a row is read into stays packed until its sum is there, so that few registers a thread let
// enough rows be under way on an SM (8192 x 4096 with post norm and gate: 268 MB in 47.7 us, 5.6 TB/s, 86 % of the copy rate). One
// row of 4096 takes 1.8 us: the launch and two dependent loads.
template <typename T, typename R, int V, int W, bool WARP_ROW>
__global__ void __launch_bounds__(1024) ob_residual_norm_kernel(const NormArgs a) {
  __shared__ float scratch[2][32];
  follow_previous_kernel();
  const int tpr = WARP_ROW ? 32 : blockDim.x;
  const int t = WARP_ROW ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = WARP_ROW ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;                                  // whole warps (WARP_ROW); never otherwise
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* res = a.residual ? static_cast<const R*>(a.residual) + row * a.r_stride : nullptr;
  const T* gate = a.gate ? static_cast<const T*>(a.gate) + row * a.g_stride : nullptr;
  const T* post = static_cast<const T*>(a.post_weight);
  const T* weight = static_cast<const T*>(a.weight);
  T* y = static_cast<T*>(a.y) + row * a.y_stride;
  R* hout = res ? static_cast<R*>(a.h) + row * a.h_stride : nullptr;
  const float inv_n = 1.f / (float)a.hidden;

  Raw<T, W> xr[V];
  Raw<R, W> rr[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * tpr + t) * W;
    xr[j].zero();
    rr[j].zero();
    if (c < a.hidden) {
      xr[j].load(x + c);
      if (res) rr[j].load(res + c);
    }
  }
  float f = 1.f;
  if (post) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float u[W];
      xr[j].values(u);
#pragma unroll
      for (int i = 0; i < W; ++i) s += u[i] * u[i];
    }
    f = rsqrtf(row_sum<WARP_ROW>(s, scratch[0]) * inv_n + a.eps);
  }
  float h[V][W], s = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * tpr + t) * W;
    xr[j].values(h[j]);
    if (res && c < a.hidden) {
      float r[W];
      rr[j].values(r);
      if (post) {
        Raw<T, W> p;
        p.load(post + c);
        float v[W];
        p.values(v);
#pragma unroll
        for (int i = 0; i < W; ++i) h[j][i] *= f * v[i];
      }
      if (gate) {
        Raw<T, W> g;
        g.load(gate + c);
        float v[W];
        g.values(v);
#pragma unroll
        for (int i = 0; i < W; ++i) h[j][i] *= v[i];
      }
#pragma unroll
      for (int i = 0; i < W; ++i) h[j][i] = r[i] + a.residual_scale * h[j][i];
      if constexpr (W == 8) store8(hout + c, h[j]);
      else hout[c] = from_f32<R>(h[j][0]);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) s += h[j][i] * h[j][i];
  }
  f = rsqrtf(row_sum<WARP_ROW>(s, scratch[1]) * inv_n + a.eps);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * tpr + t) * W;
    if (c >= a.hidden) continue;
    Raw<T, W> w;
    w.load(weight + c);
    float v[W];
    w.values(v);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] *= h[j][i] * f;
    if constexpr (W == 8) store8(y + c, v);
    else y[c] = from_f32<T>(v[0]);
  }
}

// Rows above 4096 values that are not aligned: h waits in shared memory (fp32, up to 128 KB), since in registers it would be up to
// 32 values a thread next to as many of x and the residual. 1111 rows of 8191 fp16 values with a residual: 22.7 us, in registers
// (spilled) 113 us.
constexpr int kLongThreads = 512;
template <typename T, typename R> __global__ void __launch_bounds__(kLongThreads) ob_residual_norm_long_kernel(const NormArgs a) {
  extern __shared__ float hs[];
  __shared__ float scratch[2][32];
  follow_previous_kernel();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const R* res = a.residual ? static_cast<const R*>(a.residual) + row * a.r_stride : nullptr;
  const T* gate = a.gate ? static_cast<const T*>(a.gate) + row * a.g_stride : nullptr;
  const T* post = static_cast<const T*>(a.post_weight);
  const T* weight = static_cast<const T*>(a.weight);
  T* y = static_cast<T*>(a.y) + row * a.y_stride;
  R* hout = res ? static_cast<R*>(a.h) + row * a.h_stride : nullptr;
  const float inv_n = 1.f / (float)a.hidden;
  constexpr int kTogether = 8;                                 // loads under way
  auto each = [&](auto load, auto use) {
    for (int c0 = threadIdx.x; c0 < a.hidden; c0 += kTogether * kLongThreads) {
      decltype(load(0)) v[kTogether];
#pragma unroll
      for (int j = 0; j < kTogether; ++j)
        if (c0 + j * kLongThreads < a.hidden) v[j] = load(c0 + j * kLongThreads);
#pragma unroll
      for (int j = 0; j < kTogether; ++j)
        if (c0 + j * kLongThreads < a.hidden) use(c0 + j * kLongThreads, v[j]);
    }
  };
  float f = 1.f;
  if (post) {
    float s = 0.f;
    each([&](int c) { return x[c]; }, [&](int, T v) { s += to_f32(v) * to_f32(v); });
    f = rsqrtf(row_sum<false>(s, scratch[0]) * inv_n + a.eps);
  }
  struct In { T x, p, g; R r; };
  float s = 0.f;
  each([&](int c) {
         In v{};
         v.x = x[c];
         if (res) v.r = res[c];
         if (post) v.p = post[c];
         if (gate) v.g = gate[c];
         return v;
       },
       [&](int c, const In& v) {
         float h = to_f32(v.x);
         if (res) {
           if (post) h *= f * to_f32(v.p);
           if (gate) h *= to_f32(v.g);
           h = to_f32(v.r) + a.residual_scale * h;
           hout[c] = from_f32<R>(h);
         }
         hs[c] = h;
         s += h * h;
       });
  f = rsqrtf(row_sum<false>(s, scratch[1]) * inv_n + a.eps);
  each([&](int c) { return weight[c]; }, [&](int c, T w) { y[c] = from_f32<T>(to_f32(w) * (hs[c] * f)); });
}

template <typename T, typename R, int V, int W>
cudaError_t launch_rows(const NormArgs& a, int threads, cudaStream_t stream) {
  constexpr int kRows = 4;                                    // rows (warps) per CTA where a warp has a row
  if constexpr (V * W <= 16)                                  // the only chunkings that a warp alone can be given
    if (threads == 32)
      return launch_following(ob_residual_norm_kernel<T, R, V, W, true>, dim3((unsigned)((a.rows + kRows - 1) / kRows)), 32 * kRows, 0, stream, a);
  return launch_following(ob_residual_norm_kernel<T, R, V, W, false>, dim3((unsigned)a.rows), threads, 0, stream, a);
}

template <typename T, typename R> cudaError_t launch_types(const NormArgs& a, bool wide, cudaStream_t stream) {
  const int chunks = wide ? a.hidden / 8 : a.hidden;
  auto threads_for = [&](int per) { return max(32, min(1024, ((chunks + per - 1) / per + 31) / 32 * 32)); };
  if (wide) {
    // Values per thread: the fewest where a row's latency is all there is (64 x 4096 with a residual: 2.0 us with 8, 2.4 with 16,
    // 2.8 with 32), more where the rows fill the GPU, for the sums' barriers (8192 x 4096, post norm and gate: 51.9 / 47.7 / 48.1 us;
    // 1111 x 8192: 10.2 / 9.4 / 8.2 us).
    if (a.rows <= 256 && chunks <= 1024) return launch_rows<T, R, 1, 8>(a, threads_for(1), stream);
    if (chunks <= 512) return launch_rows<T, R, 2, 8>(a, threads_for(2), stream);
    return launch_rows<T, R, 4, 8>(a, threads_for(4), stream);
  }
  // 1111 x 2047 bf16, fp32 residual, gate: 11.2 us with 4 values a thread, 12.6 with 8; 1111 x 4095 with a residual: 14.6 and 14.2
  if (chunks <= 2048) return launch_rows<T, R, 4, 1>(a, threads_for(4), stream);
  if (chunks <= 4096) return launch_rows<T, R, 8, 1>(a, threads_for(8), stream);
  static std::atomic<uint64_t> ready{0};
  const cudaError_t e = allow_shared_memory(ob_residual_norm_long_kernel<T, R>, 32768 * 4, ready);
  if (e != cudaSuccess) return e;
  return launch_following(ob_residual_norm_long_kernel<T, R>, dim3((unsigned)a.rows), kLongThreads, a.hidden * sizeof(float), stream, a);
}

}  // namespace

namespace ob {

cudaError_t launch_residual_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, bool residual_f32,
                                 const void* gate, int64_t gate_stride, const void* post_weight, const void* weight, void* y,
                                 int64_t y_stride, void* h, int64_t h_stride, int64_t rows, int64_t hidden, float residual_scale,
                                 float eps, bool bf16, cudaStream_t stream) {
  const NormArgs a{x, residual, gate, post_weight, weight, y, h, x_stride, residual_stride, gate_stride, y_stride, h_stride,
                   rows, (int)hidden, residual_scale, eps};
  auto rows_ok = [](const void* p, int64_t stride) {   // every row starts on a 16-byte boundary
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0);
  };
  const bool wide = hidden % 8 == 0 && rows_ok(x, x_stride) && rows_ok(residual, residual_stride) &&
                    rows_ok(gate, gate_stride) && rows_ok(post_weight, 0) && rows_ok(weight, 0) && rows_ok(y, y_stride) &&
                    rows_ok(h, h_stride);
  if (bf16) return residual_f32 ? launch_types<__nv_bfloat16, float>(a, wide, stream) : launch_types<__nv_bfloat16, __nv_bfloat16>(a, wide, stream);
  return residual_f32 ? launch_types<__half, float>(a, wide, stream) : launch_types<__half, __half>(a, wide, stream);
}

}  // namespace ob
