// Choosing the largest of many float32 values exactly, equal ones by place: the integer order of floats and the
// workgroup sums the selection kernels share (attn_select.hip, kv_evict.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace q27h {

// Whole numbers in the order of the floats (the two zeros equal, NaN below all).
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = x == 0.0f ? 0u : __builtin_bit_cast(uint32_t, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the threads of WAVES waves before this one, and over all of them. `s` is WAVES words of LDS.
template <int WAVES>
__device__ __forceinline__ int scan_waves(int v, int* s, int& total) {
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (l >= d) x += y;
  }
  __syncthreads();
  if (l == 63) s[w] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < WAVES; i++) {
    if (i < w) before += s[i];
    total += s[i];
  }
  return before + x - v;
}
__device__ __forceinline__ int scan256(int v, int* s, int& total) { return scan_waves<4>(v, s, total); }

}  // namespace q27h
