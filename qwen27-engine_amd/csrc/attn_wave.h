// What a workgroup of waves that walk cache rows of their own shares, whatever the cache's form: the LDS of its queries and
// tiles, a wave's rows at their start, a tile with hidden rows, and the join of its waves (attn_tree.hip, attn_paged.hip).
#pragma once
#include "attn_core.h"

namespace q27h {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

// Rows that every drafted token sees, and the rows that exist.
__device__ __forceinline__ Vis vis_of(long long pos0, int T, int n_ctx) {
  Vis v;
  v.n0 = pos0 > n_ctx ? n_ctx : (int)pos0;
  v.n = pos0 < 0 ? 0 : pos0 > n_ctx ? n_ctx : (int)pos0;
  const long long e = pos0 + T;
  v.end = e < 0 ? 0 : e > n_ctx ? n_ctx : (int)e;
  return v;
}

// LDS of WR * WK waves: WR row tiles of 16 query rows, and for each of them WK waves that share the workgroup's cache rows.
// f16: the queries' image is taken apart before the first K tile takes its place: first terms to registers, second to `lo`.
template <bool Q8, int WR, int WK>
struct AttnShared;
template <int WR, int WK>
struct AttnShared<true, WR, WK> {
  QTile q[WR];
  WaveLds w[WR * WK];
  float ml[WR * WK][16][2];
};
template <int WR, int WK>
struct AttnShared<false, WR, WK> {
  union {
    QTile q[WR];
    HKeysLds w[WR * WK];
  };
  alignas(16) uint32_t lo[WR][8][64][4];
  float ml[WR * WK][16][2];
};

// What a wave has of its queries, by the cache's type.
template <bool Q8>
struct Queries;
template <>
struct Queries<true> {
  const QTile* im;
};
template <>
struct Queries<false> {
  QHalf r[1];
};

// A wave's rows at their start; all waves of the workgroup, behind the barrier that ends load_queries.
template <int WR, int WK>
__device__ __forceinline__ void begin_rows(Rows& st, Queries<true>& q, AttnShared<true, WR, WK>& sh, int wr, int wk) {
  rows_init<true>(st, sh.q[wr]);
  q.im = &sh.q[wr];
}
template <int WR, int WK>
__device__ __forceinline__ void begin_rows(Rows& st, Queries<false>& q, AttnShared<false, WR, WK>& sh, int wr, int wk) {
  const int l = threadIdx.x & 63;
  rows_init<false>(st, sh.q[wr]);
#pragma unroll
  for (int b = 0; b < 8; b++) q.r[0].hi[b] = *(const h8*)sh.q[wr].v[0][b][l];
  q.r[0].lo = sh.lo[wr];
#pragma unroll
  for (int b = 0; b < 8; b += WK)  // each of the row tile's waves moves its share
    *(h8*)sh.lo[wr][b + wk][l] = *(const h8*)sh.q[wr].v[1][b + wk][l];
  __syncthreads();
}

// A wave's tile of which some rows are hidden or do not exist.
// VRows: V's form on its way to LDS, bias_of<VRows> that of its codes there.
template <typename VRows>
constexpr int bias_of = 128;
template <typename VRows = QRows>
__device__ __forceinline__ void tail_tile(Rows& st, const KvHead& kc, const KvHead& vc, const Queries<true>& q, WaveLds& w,
                                          const Vis& vis, uint64_t tree, int j0) {
  QRows k;
  VRows v;
  f4 s[1][2];
  const int left = vis.end - j0;
  const uint64_t trees[1] = {tree};
  load_rows<true>(k, kc, j0, left);
  load_rows<true>(v, vc, j0, left);
  stage_keys(k, w);
  scores<1>(w, q.im, s);
  hide<1, kHidden>(s, vis, trees, j0);
  weights<true, true>(st, s[0]);
  __builtin_amdgcn_wave_barrier();
  stage_values(v, w);
  accumulate<true, bias_of<VRows>>(st, s[0], w);
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ void tail_tile(Rows& st, const KvHead& kc, const KvHead& vc, const Queries<false>& q, HKeysLds& w,
                                          const Vis& vis, uint64_t tree, int j0) {
  HValues v;
  f4 s[1][2];
  const int left = vis.end - j0;
  const uint64_t trees[1] = {tree};
  request_keys<true>(w, kc, j0, left);
  keys_there<0>();
  scores(w, q.r, s);
  load_rows<true>(v, vc, j0, left);
  hide<1, kHidden>(s, vis, trees, j0);
  weights<false, true>(st, s[0]);
  accumulate_tail(st, s[0], v, vc, j0, left, (float*)w.k);
}

// A lane's 64 outputs to its query row's place. BY16: outputs o[i][j] are dims 16 i + 4 g + j; else attn_core.h's f16 order.
template <bool BY16>
__device__ __forceinline__ void store_rows(const Rows& st, float* dst) {
  const int g = (threadIdx.x & 63) >> 4;
  if constexpr (BY16) {
#pragma unroll
    for (int i = 0; i < 16; i++) *(f4*)(dst + 16 * i + 4 * g) = st.o[i];
  } else {
#pragma unroll
    for (int hr = 0; hr < 2; hr++)
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int q = 0; q < 2; q++)
          *(f4*)(dst + 128 * hr + 8 * (4 * g + c) + 4 * q) =
              (f4){st.o[8 * hr + 4 * q][c], st.o[8 * hr + 4 * q + 1][c], st.o[8 * hr + 4 * q + 2][c], st.o[8 * hr + 4 * q + 3][c]};
  }
}

// Joins the WK waves of each row tile; the first of them gives its rows to write(st, m, sum): sum = the row's weights relative
// to 2^m, the outputs not yet divided by it.
template <bool Q8, int WR, int WK, typename F>
__device__ __forceinline__ void finish(Rows& st, AttnShared<Q8, WR, WK>& sh, F write) {
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, n = l & 15, g = l >> 4, wr = w % WR, wk = w / WR;
  auto& ml = sh.ml;                       // [wave][row]
  f4(*ex)[16][64] = (f4(*)[16][64])sh.w;  // outputs of half the waves
  static_assert(sizeof(sh.w) >= WR * WK / 2 * sizeof(f4) * 16 * 64);
  st.l += lane_xor<16>(st.l);
  st.l += lane_xor32(st.l);
  __syncthreads();  // every wave is done with the queries and its tile
  if (g == 0) ml[w][n][0] = st.m, ml[w][n][1] = st.l;
  __syncthreads();
  float m = -3.0e38f, sum = 0.0f;
#pragma unroll
  for (int k = 0; k < WK; k++) m = __builtin_fmaxf(m, ml[k * WR + wr][n][0]);
#pragma unroll
  for (int k = 0; k < WK; k++) sum += ml[k * WR + wr][n][1] * __builtin_amdgcn_exp2f(ml[k * WR + wr][n][0] - m);
  const float f = __builtin_amdgcn_exp2f(st.m - m) * unit_of<Q8>(st);
#pragma unroll
  for (int i = 0; i < 16; i++) st.o[i] *= f;
#pragma unroll
  for (int h = WK / 2; h > 0; h /= 2) {  // the upper half of the waves hands over, the lower adds: always in the same order
    if (wk >= h && wk < 2 * h) {
#pragma unroll
      for (int i = 0; i < 16; i++) ex[w - h * WR][i][l] = st.o[i];
    }
    __syncthreads();
    if (wk < h) {
#pragma unroll
      for (int i = 0; i < 16; i++) st.o[i] += ex[w][i][l];
    }
    __syncthreads();
  }
  if (wk == 0) write(st, m, sum);
}

}  // namespace q27h
