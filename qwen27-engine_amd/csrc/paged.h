// A K/V cache in pages that many sequences share, and a ragged batch over it, as the kernels see them.
//
// A page of K or V is a cache of `rows` rows as attn_prep lays one out: f16 [nkvh][rows][256], or codes [nkvh][rows][256]
// (4 bits: [nkvh][rows][128]) followed by f16 scales [nkvh][rows][8]. 4 bits: byte j of a block's 16 holds value j in its low
// half and value j + 16 in its high one, each the code 0 .. 15 of (code - 8) * scale. rows is a power of two of at least 32,
// so that a tile of 32 rows lies in one page.
#pragma once
#include "q27h_device.h"
#include "q27h_internal.h"

namespace q27h {

constexpr int kHeadDim = 256;
constexpr int kRowF16 = 512, kRowQ8 = 272, kRowQ4 = 144;  // bytes of a row of one head, scales included

struct Pages {
  uint8_t *k, *v;
  const int* table;  // [n_seqs][max_pages]
  size_t kb, vb;     // bytes of a page of K, of V
  int n_seqs, max_pages, n_pages, nkvh, shift;  // 1 << shift rows a page
  int type;
};

inline int kv_row_bytes(int type, bool v) {
  return type == Q27H_KV_F16 ? kRowF16 : v && type == Q27H_KV_Q8_Q4 ? kRowQ4 : kRowQ8;
}
// Q27H_OK, or the refusal of a bad handle (its sizes, pointers and alignment).
int check_pages(const q27h_kv_pages* kv, const char* what);
Pages pages_of(const q27h_kv_pages* kv);  // of a handle that passed

// A load from memory that no kernel writes while this one runs, of an address that is the same in the whole wave: through
// the scalar cache, so that the vector loads on their way need not be waited for.
__device__ __forceinline__ int uniform_load(const int* p) { return *(const __attribute__((address_space(4))) int*)p; }

// The tokens of sequence b of the batch, t0 .. t0 + nt - 1, whatever cu holds. cu null: token b.
struct Tokens {
  int t0, nt;
};
__device__ __forceinline__ Tokens tokens_of(int c0, int c1, int T, int most) {
  c0 = c0 < 0 ? 0 : c0 > T ? T : c0;
  c1 = c1 < c0 ? c0 : c1 > T ? T : c1;
  return {c0, c1 - c0 < most ? c1 - c0 : most};
}
__device__ __forceinline__ Tokens tokens_of(const int* cu, int b, int T, int most) {
  return cu ? tokens_of(uniform_load(cu + b), uniform_load(cu + b + 1), T, most) : tokens_of(b, b + 1, T, most);
}

// Work of unequal sequences in equal shares: cost(b) >= 0 of each sequence, laid end to end, is cut in `gridDim.x` parts of
// a multiple of `unit`. Gives every thread of the workgroup its part [x, end), the sequence that x lies in and where that
// one begins; where `starts` is given, the first workgroup also leaves the beginnings there, and the total behind them.
struct Share {
  int x, end, per, seq, start;
};
template <int THREADS, typename F>
__device__ __forceinline__ Share share_of(int n_seqs, int unit, int* starts, F cost) {
  __shared__ int s_sum[THREADS / 64], s_at[2];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const int each = (n_seqs + THREADS - 1) / THREADS, b0 = tid * each, b1 = b0 + each < n_seqs ? b0 + each : n_seqs;
  int mine = 0;
  for (int b = b0; b < b1; b++) mine += cost(b);
  int before = mine;  // inclusive sums of the wave
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(before, d);
    before += l >= d ? y : 0;
  }
  if (l == 63) s_sum[w] = before;
  __syncthreads();
  int total = 0;
  before -= mine;
#pragma unroll
  for (int k = 0; k < THREADS / 64; k++) {
    before += k < w ? s_sum[k] : 0;
    total += s_sum[k];
  }
  Share s;
  const int parts = (int)gridDim.x;
  s.per = ((total + parts - 1) / parts + unit - 1) / unit * unit;
  // a workgroup behind the last part: its product may pass 31 bits
  s.x = (long long)blockIdx.x * s.per < total ? (int)blockIdx.x * s.per : total;
  s.end = total - s.x < s.per ? total : s.x + s.per;
  if (starts && blockIdx.x == 0 && tid == 0) starts[n_seqs] = total;
  if ((starts && blockIdx.x == 0) || (before <= s.x && s.x < before + mine)) {
    int at = before;
    for (int b = b0; b < b1; b++) {
      const int c = cost(b);
      if (starts && blockIdx.x == 0) starts[b] = at;
      if (at <= s.x && s.x < at + c) s_at[0] = b, s_at[1] = at;
      at += c;
    }
  }
  __syncthreads();
  s.x = __builtin_amdgcn_readfirstlane(s.x);
  s.end = __builtin_amdgcn_readfirstlane(s.end);
  s.per = __builtin_amdgcn_readfirstlane(s.per);
  s.seq = __builtin_amdgcn_readfirstlane(s_at[0]);
  s.start = __builtin_amdgcn_readfirstlane(s_at[1]);
  return s;
}

}  // namespace q27h
