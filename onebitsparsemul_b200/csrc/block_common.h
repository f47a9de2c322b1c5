// Shared pieces of the decoder-block kernels (norm.cu, rotary_append.cu, cache_attend*.cu). Internal header.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace ob_block {

// A cache page holds 64 tokens: keys (page, head, 64, dim), values (page, head, dim, 64), both e4m3, one fp32 scale for
// each page and head of either.
constexpr int kPageTokens = 64;
constexpr float kE4m3Max = 448.f;
constexpr int kMinScaleExp = -32, kMaxScaleExp = 32;

// Notes that a batch named a page or a range outside its tensors; what it named was left out. The word is apart from the one that
// bounded waits leave their code in.
__device__ __forceinline__ void note_bad_batch(int* word) { atomicExch(word, 1); }
// A status word's value, and 0 in its place.
template <typename Word> cudaError_t take_status(Word& symbol, int* out) {
  *out = 0;
  cudaError_t e = cudaMemcpyFromSymbol(out, symbol, sizeof(int));
  if (e != cudaSuccess || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(symbol, &zero, sizeof(int));
}

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 8 consecutive values, 16-byte aligned for the 16-bit types and 32-byte for fp32
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(ws[i], T{});
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{}), pack2(v[4], v[5], T{}), pack2(v[6], v[7], T{}));
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// ---- whose rows these are --------------------------------------------------------------------------------------------------
// A batch's q_start has to ascend from 0 or more to the call's rows or less. Where it does not, the batch is reported, and a sequence
// is left out if its range is not inside the rows, runs backwards, or starts before an earlier start. For that the work is dealt
// out by the running maximum Q[s] of the starts that lie in range: it ascends whatever q_start holds, and equals q_start for every
// sequence that is not left out. Row t belongs to sequence s with Q[s] <= t < Q[s + 1]; slot x of a grid that gives sequence s the
// slots Q[s] / per + s .. Q[s + 1] / per + s belongs to the last s with Q[s] / per + s <= x. Either is found by one minimum
// over all starts, without the running maximum itself: the first s that is too far for a start q[i], i <= s.
struct Starts {
  const int* q;
  int seqs, rows;
  __device__ __forceinline__ bool in_range(int start) const { return start >= 0 && start <= rows; }
  // start i, and whether it is out of order with the next one
  __device__ __forceinline__ int at(int i, bool& bad) const {
    const int a = q[i], b = i < seqs ? q[i + 1] : rows;
    bad |= a < 0 || b < a || b > rows;
    return a;
  }
  __device__ __forceinline__ int behind_row(int i, int start, int row) const { return in_range(start) && start > row ? i : seqs + 1; }
  // place: start -> its share of the slot number
  __device__ __forceinline__ int behind_slot(int i, int start, int slot, int place) const { return in_range(start) ? max(i, slot - place + 1) : seqs; }
  // sequence s of a batch that is out of order; a walk over the starts before it, which a batch in order never takes
  __device__ __forceinline__ bool left_out(int s) const {
    const int a = q[s], b = q[s + 1];
    if (a < 0 || b < a || b > rows) return true;
    for (int i = 0; i < s; ++i)
      if (in_range(q[i]) && q[i] > a) return true;
    return false;
  }
};

// ---- rotary angles -----------------------------------------------------------------------------------------------------
// An angle is kept in turns, as a 64-bit binary fraction: the frequency's share of a turn per position, rounded to 2^-64
// (from a double: 53 bits of it are meaningful), times the position, modulo 2^64 -- the integer product wraps exactly where
// the angle does. A position p adds an error of at most p * 2^-54 of a turn, so far positions cost nothing, where an fp32
// product p * freq is off by p * 2^-24 radians.
__device__ __forceinline__ uint64_t turns_per_position(double angular_frequency) {
  double t = angular_frequency * 0.15915494309189533577;   // 1 / (2 pi)
  t -= floor(t);
  return __double2ull_rz(t * 18446744073709551616.0);
}
// cos and sin (times magnitude) by the special function unit: the angle lies in [-pi, pi), where its results are within 2^-21.2
// of the exact ones, a thousandth of the 16-bit types' rounding; sincospif would be several times the instructions of the rest.
__device__ __forceinline__ float2 cos_sin(uint64_t per_position, int64_t position, float magnitude) {
  const uint64_t phase = per_position * (uint64_t)position;
  const float angle = (float)(int32_t)(uint32_t)(phase >> 32) * 1.4629180792671596e-9f;      // pi * 2^-31
  return make_float2(__cosf(angle) * magnitude, __sinf(angle) * magnitude);
}

// ---- e4m3 -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint8_t to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) { return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float from_e4m3(uint8_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}
// The smallest power of two 2^e, e in [-32, 32], with amax <= 448 * 2^e. A power of two keeps every division by the scale
// exact, and a page that is re-scaled later only loses bits that leave e4m3's range.
__device__ __forceinline__ float scale_for(float amax) {
  if (!(amax > 0.f)) return exp2f((float)kMinScaleExp);
  int e;
  const float m = frexpf(amax, &e);                         // amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
  e = m <= 0.875f ? e - 9 : e - 8;
  return ldexpf(1.f, min(max(e, kMinScaleExp), kMaxScaleExp));
}

// ---- programmatic dependent launch -----------------------------------------------------------------------------------------
// A decode step is a chain of kernels of a few microseconds. They are launched so that a grid may start while its
// predecessor drains, and each waits here, before its first access to memory, until the predecessor is complete. What a
// predecessor may have written (lengths, tables, scales, tokens) is read by plain loads only: a read-only load (ld.global.nc)
// promises that nothing writes the data while the kernel lives, and could be moved above the wait.
__device__ __forceinline__ void follow_previous_kernel() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
struct ClusterOf { int ctas; };
template <typename... Params, typename... Args>
cudaError_t launch_following(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, ClusterOf cluster, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = (unsigned)cluster.ctas, attrs[1].val.clusterDim.y = 1, attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs, cfg.numAttrs = cluster.ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... Params, typename... Args>
cudaError_t launch_following(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  return launch_following(kernel, grid, threads, smem, stream, ClusterOf{1}, args...);
}

// Raises a kernel's dynamic shared memory limit, once per device (a bit of `ready` for each); and allows clusters of 16.
template <typename K> cudaError_t allow_shared_memory(K kernel, int bytes, std::atomic<uint64_t>& ready, bool wide_clusters = false) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && wide_clusters) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace ob_block
