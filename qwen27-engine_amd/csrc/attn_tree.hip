// Attention over the K/V cache that attn_prep writes: a tree of drafted tokens (attn_tree; one token is plain decoding),
// blocks of 64 rows chosen per token (attn_blocks), and the sums of attention weights per cache row (attn_weights).
//
// The rows of the cache are split over workgroups. The query rows of a kv head (tokens x query heads of the group) are taken
// as row tiles of 16. Up to two: each wave of a workgroup walks tiles of 32 cache rows of its own with the online softmax
// of attn_core.h, the next tile's loads in flight behind the current one's arithmetic, so that one or two row tiles are
// bound by HBM (150000 q8_0 rows, one token: 64 us, 5.1 TB/s). More: each wave holds a row tile and the workgroup shares the
// cache rows (attn_shared.h), bound by the matrix instructions of two f16 terms and, over q8_0, the vector work beside
// them; more than 8 row tiles are spread over workgroups that read the same cache rows on the same XCD, so that its L2
// serves all but the first. A second launch joins the splits.
#include <type_traits>

#include "attn_core.h"
#include "attn_shared.h"
#include "q27h_internal.h"

namespace q27h {
namespace {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr int kMaxTree = 64;   // tokens of a tree: a 64-bit mask per token
constexpr int kBlockRows = 64;  // rows of a block of attn_blocks
constexpr int kWaves = 4;      // waves of a workgroup of attn_blocks and attn_weights

// How the cache rows are split. Host: `max` splits are launched. Device: rows become tiles; a split takes `per` tiles,
// at least one for each of its `waves` while there are few, and the splits behind the last one have nothing to do.
struct Split {
  int per, used;
};
__device__ __forceinline__ Split split_of(int tiles, int max, int waves) {
  int per = (tiles + max - 1) / max;
  per = per < waves ? waves : per;
  return {per, tiles ? (tiles + per - 1) / per : 1};  // no rows at all: one split writes zeros
}

// Rows that every drafted token sees, and the rows that exist.
__device__ __forceinline__ Vis vis_of(long long pos0, int T, int n_ctx) {
  Vis v;
  v.n0 = pos0 > n_ctx ? n_ctx : (int)pos0;
  v.n = pos0 < 0 ? 0 : pos0 > n_ctx ? n_ctx : (int)pos0;
  const long long e = pos0 + T;
  v.end = e < 0 ? 0 : e > n_ctx ? n_ctx : (int)e;
  return v;
}
__device__ __forceinline__ uint64_t tree_of(const uint64_t* tree, int t, int T) {
  const uint64_t all = T >= 64 ? ~0ull : (1ull << T) - 1;
  return (tree ? tree[t] : ~0ull >> (63 - t)) & all;
}

struct AttnArgs {
  const float* qn;
  const void *kcache, *vcache;
  const int* pos0;
  const uint64_t* tree;  // attn_tree
  const int* idx;        // attn_blocks
  float *o, *lse;        // lse may be null
  float *part, *ml;      // [row][split][256], [row][split][2]; row = token * nqh + query head
  int T, nqh, nkvh, n_ctx, nsel;
  int splits, groups, waves;  // attn_tree: workgroups over the query rows of a kv head; waves over the cache rows of one
  int tiles;                  // attn_wide_kernel: row tiles of a workgroup
  float scale;
};

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
__device__ __forceinline__ void tail_tile(Rows& st, const KvHead& kc, const KvHead& vc, const Queries<true>& q, WaveLds& w,
                                          const Vis& vis, uint64_t tree, int j0) {
  QRows k, v;
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
  accumulate<true>(st, s[0], w);
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

// The wave's tiles that are wholly visible: next() gives the first cache row of one after the other, then -1. begin()
// requests the first one (q8), ahead of the queries' own round trip to memory; run() takes them all.
// q8: the next tile's K is requested once this one's is in LDS, its V once this one's is, so that one set of registers each
// is enough and the loads fly behind the arithmetic. f16: K's place in LDS is free once the scores are formed (and only
// after the queries' image is taken apart), V's registers once it is consumed.
template <bool Q8>
struct FullTiles;
template <>
struct FullTiles<true> {
  QRows k, v;
  int j0;
  template <typename F>
  __device__ __forceinline__ void begin(const KvHead& kc, const KvHead& vc, F next) {
    j0 = next();
    if (j0 < 0) return;
    load_rows<false>(k, kc, j0, 0);
    load_rows<false>(v, vc, j0, 0);
  }
  template <typename F>
  __device__ __forceinline__ void run(Rows& st, const KvHead& kc, const KvHead& vc, const Queries<true>& q, WaveLds& w, F next) {
    if (j0 < 0) return;
    do {
      f4 s[1][2];
      j0 = next();
      asm volatile("" ::: "memory");  // the queries are read from LDS for each tile: held in registers they would spill
      stage_keys(k, w);
      if (j0 >= 0) load_rows<false>(k, kc, j0, 0);
      loads_issued();
      scores<1>(w, q.im, s);
      weights<true, false>(st, s[0]);
      __builtin_amdgcn_wave_barrier();
      stage_values(v, w);
      if (j0 >= 0) load_rows<false>(v, vc, j0, 0);
      loads_issued();
      accumulate<false>(st, s[0], w);
      __builtin_amdgcn_wave_barrier();
    } while (j0 >= 0);
  }
};
template <>
struct FullTiles<false> {
  HValues v;
  int j0;
  template <typename F>
  __device__ __forceinline__ void begin(const KvHead& kc, const KvHead& vc, F next) {
    j0 = next();
  }
  template <typename F>
  __device__ __forceinline__ void run(Rows& st, const KvHead& kc, const KvHead& vc, const Queries<false>& q, HKeysLds& w, F next) {
    if (j0 < 0) return;
    request_keys<false>(w, kc, j0, 0);
    loads_issued();
    load_rows<false>(v, vc, j0, 0);
    do {
      f4 s[1][2];
      j0 = next();
      keys_there<kValueLoads>();
      scores(w, q.r, s);
      // V, asked for behind this tile's K, is waited for before the next K is: waited for at its use, it would be with a
      // count of zero, the next K included (the compiler does not count loads to LDS)
      keys_there<0>();
      if (j0 >= 0) request_keys<false>(w, kc, j0, 0);
      loads_issued();
      weights<false, false>(st, s[0]);
      accumulate(st, s[0], v);
      if (j0 >= 0) load_rows<false>(v, vc, j0, 0);
      loads_issued();
    } while (j0 >= 0);
  }
};

// Writes a wave's rows: as a split's part, or as the result where there is one split only. gr: the global row (token * nqh
// + head) of this lane's query row, or -1. BY16: outputs o[i][j] are dims 16 i + 4 g + j; else attn_core.h's f16 order.
template <bool BY16>
__device__ __forceinline__ void write_rows(Rows& st, const AttnArgs& a, int split, bool single, int gr, float m, float sum) {
  const int g = (threadIdx.x & 63) >> 4;
  if (gr < 0) return;
  float* dst;
  if (single) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 16; i++) st.o[i] *= inv;
    dst = a.o + (size_t)gr * kHD;
    if (a.lse && g == 0) a.lse[gr] = sum == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
  } else {
    const size_t at = (size_t)gr * a.splits + split;
    dst = a.part + at * kHD;
    if (g == 0) *(float2*)(a.ml + at * 2) = make_float2(m, sum);
  }
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

// Joins the WK waves of each row tile and writes its rows.
template <bool Q8, int WR, int WK>
__device__ __forceinline__ void finish(Rows& st, AttnShared<Q8, WR, WK>& sh, const AttnArgs& a, int split, bool single, int gr) {
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
  if (wk == 0) write_rows<Q8>(st, a, split, single, gr, m, sum);
}

template <bool Q8, int WR, int WK>
__global__ void __launch_bounds__(WR * WK * 64, 2) attn_tree_kernel(AttnArgs a) {
  __shared__ AttnShared<Q8, WR, WK> sh;
  // workgroups 8 apart run on one XCD: those of one (kv head, split) follow each other there
  const int unit = (int)(blockIdx.x / (8 * a.groups)) * 8 + (int)(blockIdx.x & 7), rg = (int)(blockIdx.x >> 3) % a.groups;
  if (unit >= a.nkvh * a.splits) return;
  const int kh = unit % a.nkvh, split = unit / a.nkvh;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = w % WR, wk = w / WR;
  const Vis vis = vis_of(*a.pos0, a.T, a.n_ctx);
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const Split sp = split_of(tiles, a.splits, WK);
  if (split >= sp.used) return;
  const int group = a.nqh / a.nkvh, rows = a.T * group;
  auto row = [&](int r) {
    r += rg * WR * 16;
    return r < rows ? (r / group) * a.nqh + kh * group + r % group : -1;
  };
  const KvHead kc = kv_head<Q8>(a.kcache, kh, a.nkvh, a.n_ctx), vc = kv_head<Q8>(a.vcache, kh, a.nkvh, a.n_ctx);
  const int t1 = split * sp.per + sp.per < tiles ? split * sp.per + sp.per : tiles;
  const int full = vis.n / kTileKeys < t1 ? vis.n / kTileKeys : t1;
  int t = split * sp.per + wk;
  auto next = [&] {
    if (t >= full) return -1;
    t += WK;
    return (t - WK) * kTileKeys;
  };
  FullTiles<Q8> ft;
  ft.begin(kc, vc, next);
  load_queries<Q8, WR * WK, WR>(sh.q, a.scale * kLog2e, [&](int r) {
    const int gr = row(r);
    return gr < 0 ? nullptr : a.qn + (size_t)gr * kHD;
  });
  const int mine = wr * 16 + (threadIdx.x & 15);
  const uint64_t tree = row(mine) >= 0 ? tree_of(a.tree, (rg * WR * 16 + mine) / group, a.T) : 0ull;
  __syncthreads();
  Rows st;
  Queries<Q8> q;
  begin_rows(st, q, sh, wr, wk);
  ft.run(st, kc, vc, q, sh.w[w], next);
  for (; t < t1; t += WK) tail_tile(st, kc, vc, q, sh.w[w], vis, tree, t * kTileKeys);
  finish<Q8, WR, WK>(st, sh, a, split, sp.used == 1, row(mine));
}

// More than 32 query rows: a row tile per wave, the cache rows shared (attn_shared.h). While the waves work on kLag tiles,
// the next ones are on their way through registers to the other LDS buffers, and one barrier keeps the two apart.
template <bool Q8, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) attn_wide_kernel(AttnArgs a) {
  // tiles per barrier. 4 waves: one, for two workgroups' LDS on a compute unit; f16: one, since the second tile's way at the
  // start costs as much as the barriers do (12 tokens, 32771 rows: 49.1, 50.5 us; 64, 65536: 221 us either way)
  constexpr int kLag = WAVES == 8 && Q8 ? 2 : 1;
  constexpr size_t kTiles = sizeof(SharedTile) * 2 * kLag, kImages = sizeof(QTile) * WAVES;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[kTiles > kImages ? kTiles : kImages];  // the queries' image, then the tiles
  __shared__ int s_odd[2 * kLag];
  QTile* im = (QTile*)s_mem;
  SharedTile* buf = (SharedTile*)s_mem;
  const int unit = (int)(blockIdx.x / (8 * a.groups)) * 8 + (int)(blockIdx.x & 7), rg = (int)(blockIdx.x >> 3) % a.groups;
  if (unit >= a.nkvh * a.splits) return;
  const int kh = unit % a.nkvh, split = unit / a.nkvh;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Vis vis = vis_of(*a.pos0, a.T, a.n_ctx);
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const Split sp = split_of(tiles, a.splits, a.waves);
  if (split >= sp.used) return;
  const int t0 = split * sp.per, t1 = t0 + sp.per < tiles ? t0 + sp.per : tiles;
  const int group = a.nqh / a.nkvh, rows = a.T * group, first = rg * a.tiles * 16;
  auto row = [&](int r) {  // global row of the workgroup's query row r
    const int q = first + r;
    return r < a.tiles * 16 && q < rows ? (q / group) * a.nqh + kh * group + q % group : -1;
  };
  const KvHead kc = kv_head<Q8>(a.kcache, kh, a.nkvh, a.n_ctx), vc = kv_head<Q8>(a.vcache, kh, a.nkvh, a.n_ctx);
  auto left_of = [&](int t) { return vis.end - t * kTileKeys < kTileKeys ? vis.end - t * kTileKeys : kTileKeys; };
  auto part_of = [&](int t) { return (t + 1) * kTileKeys > vis.n; };
  auto ask = [&](Staged<Q8, WAVES>& n, int t) {
    if (t < t1) request<Q8, WAVES, true, true>(n, kc, vc, t * kTileKeys, left_of(t));
  };
  // tiles on their way beside those in LDS: 8 waves of f16 two (64 tokens, 65536 rows: 227 -> 219 us); q8's arithmetic
  // takes longer than a load, and 4 waves carry twice as much each, whose registers spill: one
  constexpr int kAhead = WAVES == 8 && !Q8 ? 2 : 1;
  Staged<Q8, WAVES> even, odd;
  ask(even, t0);
  if (kLag == 2) ask(odd, t0 + 1);
  if (threadIdx.x < 2 * kLag) s_odd[threadIdx.x] = 0;
  load_queries<Q8, WAVES, WAVES>(im, a.scale * kLog2e, [&](int r) {
    const int gr = row(r);
    return gr < 0 ? nullptr : a.qn + (size_t)gr * kHD;
  });
  __syncthreads();
  QRegs q;
  take_queries(q, im[w]);
  Rows st;
  rows_init<Q8>(st, im[w]);
  const int mine = w * 16 + (threadIdx.x & 15), gr = row(mine);
  const uint64_t tree[1] = {gr >= 0 ? tree_of(a.tree, (first + mine) / group, a.T) : 0ull};
  const bool active = w < a.tiles && first + w * 16 < rows;
  __syncthreads();
  auto put = [&](Staged<Q8, WAVES>& n, int t) __attribute__((always_inline)) {
    const int at = (t - t0) & (2 * kLag - 1);
    if (t < t1) stage<Q8, WAVES, true, true>(n, buf[at], part_of(t), left_of(t), &s_odd[at]);
  };
  put(even, t0);
  if (kLag == 2) put(odd, t0 + 1);
  ask(even, t0 + kLag);
  if (kAhead == 2) ask(odd, t0 + kLag + 1);
  __syncthreads();
  // `next` holds tile t + kLag and is given the one kAhead behind it. Two loops: a tile with hidden rows takes another form of the product,
  // and with both in one loop the outputs' registers are copied between them (and spill); the first takes an even number
  // of tiles, so that either begins with `even`.
  int t = t0;
  auto step = [&](auto hidden, Staged<Q8, WAVES>& next) __attribute__((always_inline)) {
    constexpr bool kPart = decltype(hidden)::value;
    const int at = (t - t0) & (2 * kLag - 1);
    if (active) {
      f4 s[1][2];
      __builtin_amdgcn_s_setprio(1);  // products before the other wave's staging (32 tokens, 65536 q8_0 rows: 171 -> 162 us)
      scores<Q8>(buf[at], &q, s);
      if (kPart) hide<1, kHidden>(s, vis, tree, t * kTileKeys);
      weights<Q8, kPart>(st, s[0]);
      accumulate<Q8, kPart>(st, s[0], buf[at]);
      if (!Q8 && kPart && s_odd[at]) add_odd(st, s[0], vc, t * kTileKeys, left_of(t));
    }
    __builtin_amdgcn_s_setprio(0);
    put(next, t + kLag);
    ask(next, t + kLag + kAhead);
    if (kLag == 1 || (at & 1)) __syncthreads();
    t++;
  };
  auto walk = [&](auto hidden, int end) __attribute__((always_inline)) {
    if constexpr (kAhead == 1) {
      while (t < end) step(hidden, even);
    } else {
      while (t + 1 < end) {
        step(hidden, even);
        step(hidden, odd);
      }
      if (t < end) step(hidden, even);
    }
  };
  const int full = vis.n / kTileKeys < t1 ? vis.n / kTileKeys : t1;
  if (full > t0) walk(std::false_type(), t0 + (full - t0) / 2 * 2);
  walk(std::true_type(), t1);
  if (!active) return;
  st.l += lane_xor<16>(st.l);
  st.l += lane_xor32(st.l);
  if constexpr (Q8) {
    const float f = unit_of<Q8>(st);
#pragma unroll
    for (int i = 0; i < 16; i++) st.o[i] *= f;
  }
  write_rows<true>(st, a, split, sp.used == 1, gr, st.m, st.l);
}

// attn_blocks: one workgroup per (token, kv head, split of its list); the group's query heads are one row tile.
template <bool Q8>
__global__ void __launch_bounds__(kWaves * 64, 2) attn_blocks_kernel(AttnArgs a) {
  __shared__ AttnShared<Q8, 1, kWaves> sh;
  const int unit = (int)(blockIdx.x / a.splits), split = (int)(blockIdx.x % a.splits);
  const int kh = unit % a.nkvh, t = unit / a.nkvh;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Vis vis = vis_of((long long)*a.pos0 + t + 1, 0, a.n_ctx);
  const int group = a.nqh / a.nkvh;
  auto row = [&](int r) { return r < group ? t * a.nqh + kh * group + r : -1; };
  const KvHead kc = kv_head<Q8>(a.kcache, kh, a.nkvh, a.n_ctx), vc = kv_head<Q8>(a.vcache, kh, a.nkvh, a.n_ctx);
  const int per = (2 * a.nsel + a.splits - 1) / a.splits;
  const int t1 = split * per + per < 2 * a.nsel ? split * per + per : 2 * a.nsel;
  const int* list = a.idx + ((size_t)t * a.nkvh + kh) * a.nsel;
  // the first cache row of the list's i-th tile, or -1: an entry that is no block of the context, or one seen in part
  // where a whole one is asked for (and the other way round)
  const int nb = (vis.n + kBlockRows - 1) / kBlockRows;
  auto tile = [&](int i, bool part) {
    // a scalar load: a vector load's wait would be for the tiles on their way as well
    const int b = *(const __attribute__((address_space(4))) int*)(list + (i >> 1));
    // the entry is any number: the product is formed of one that is a block
    const bool is = (unsigned)b < (unsigned)nb;
    const int j0 = (is ? b : 0) * kBlockRows + (i & 1) * kTileKeys;
    return is && j0 < vis.n && (j0 + kTileKeys > vis.n) == part ? j0 : -1;
  };
  int i = split * per + w;
  auto next = [&] {
    for (; i < t1; i += kWaves) {
      const int j0 = tile(i, false);
      if (j0 >= 0) {
        i += kWaves;
        return j0;
      }
    }
    return -1;
  };
  FullTiles<Q8> ft;
  ft.begin(kc, vc, next);
  load_queries<Q8, kWaves, 1>(sh.q, a.scale * kLog2e, [&](int r) {
    const int gr = row(r);
    return gr < 0 ? nullptr : a.qn + (size_t)gr * kHD;
  });
  __syncthreads();
  Rows st;
  Queries<Q8> q;
  begin_rows(st, q, sh, 0, w);
  ft.run(st, kc, vc, q, sh.w[w], next);
  for (i = split * per + w; i < t1; i += kWaves) {
    const int j0 = tile(i, true);
    if (j0 >= 0) tail_tile(st, kc, vc, q, sh.w[w], vis, 0ull, j0);
  }
  finish<Q8, 1, kWaves>(st, sh, a, split, a.splits == 1, row(threadIdx.x & 15));
}

// Joins the splits of one query row: GROUPS groups of lanes take every GROUPS-th split each, all requested at once, a lane 4
// of the workgroup's 1024 / GROUPS dims; then the groups' sums are added in order. 16 groups where a row has many splits
// (128 splits of 24 rows: 38 us with a thread per dim that walks the splits, 4.7 us so), 4 where it has up to 32 (12 splits
// of 1536 rows: a quarter of the workgroups, 38.6 -> 34.9 us with the splits' own kernel).
// FIXED: every split was written; else those that split_of used, and nothing is left to do where that is one.
constexpr int kMaxSplits = 2 * kCUs, kFewSplits = 32;
template <bool FIXED, int GROUPS>
__global__ void __launch_bounds__(256, 8) attn_join_kernel(AttnArgs a) {
  constexpr int kLanes = 256 / GROUPS;
  __shared__ float s_f[kMaxSplits], s_red[8];
  __shared__ f4 s_o[GROUPS][kLanes];
  const int gr = blockIdx.x, tid = threadIdx.x, c = tid % kLanes, sg = tid / kLanes, w = tid >> 6;
  int used = a.splits;
  if (!FIXED) {
    const Vis vis = vis_of(*a.pos0, a.T, a.n_ctx);
    used = split_of((vis.end + kTileKeys - 1) / kTileKeys, a.splits, a.waves).used;
    if (used == 1) return;
  }
  const float2* ml = (const float2*)a.ml + (size_t)gr * a.splits;
  const f4* part = (const f4*)(a.part + (size_t)gr * a.splits * kHD) + blockIdx.y * kLanes + c;
  constexpr int kBatch = 8;
  f4 x[kBatch];
#pragma unroll
  for (int k = 0; k < kBatch; k++) {
    const int s = sg + GROUPS * k;
    if (s < used) x[k] = part[(size_t)s * (kHD / 4)];
  }
  float2 v[kMaxSplits / 256];
  float m = -3.0e38f;
#pragma unroll
  for (int k = 0; k < kMaxSplits / 256; k++) {
    const int s = tid + 256 * k;
    v[k] = s < used ? ml[s] : make_float2(-3.0e38f, 0.0f);
    m = __builtin_fmaxf(m, v[k].x);
  }
  auto all_lanes = [&](float y, auto op) {
    y = op(y, lane_xor<1>(y));
    y = op(y, lane_xor<2>(y));
    y = op(y, lane_xor<7>(y));
    y = op(y, lane_xor<8>(y));
    y = op(y, lane_xor<16>(y));
    return op(y, lane_xor32(y));
  };
  m = all_lanes(m, [](float p, float q) { return __builtin_fmaxf(p, q); });
  if ((tid & 63) == 0) s_red[w] = m;
  __syncthreads();
  m = __builtin_fmaxf(__builtin_fmaxf(s_red[0], s_red[1]), __builtin_fmaxf(s_red[2], s_red[3]));
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < kMaxSplits / 256; k++) {
    const float f = __builtin_amdgcn_exp2f(v[k].x - m);
    if (tid + 256 * k < used) s_f[tid + 256 * k] = f;
    sum += v[k].y * f;
  }
  sum = all_lanes(sum, [](float p, float q) { return p + q; });
  if ((tid & 63) == 0) s_red[4 + w] = sum;
  __syncthreads();
  sum = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kBatch; k++) {
    const int s = sg + GROUPS * k;
    if (s < used) o += x[k] * s_f[s];
  }
  for (int s = sg + GROUPS * kBatch; s < used; s += GROUPS) o += part[(size_t)s * (kHD / 4)] * s_f[s];
  s_o[sg][c] = o;
  __syncthreads();
  if (tid < kLanes) {
    f4 r = s_o[0][tid];
#pragma unroll
    for (int k = 1; k < GROUPS; k++) r += s_o[k][tid];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *((f4*)(a.o + (size_t)gr * kHD) + blockIdx.y * kLanes + tid) = r * inv;
  }
  if (a.lse && tid == 0 && blockIdx.y == 0)
    a.lse[gr] = sum == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
}
template <bool FIXED>
void launch_join(const AttnArgs& a, hipStream_t s) {
  const bool few = a.splits <= kFewSplits;
  hipLaunchKernelGGL((few ? attn_join_kernel<FIXED, 4> : attn_join_kernel<FIXED, 16>), dim3((unsigned)(a.T * a.nqh), few ? 1 : 4),
                     dim3(256), 0, s, a);
}

// Sums of eight values over the 16 query rows (lanes n) of a lane group: lanes n and n ^ 8 leave with value n & 7 in x[0].
// At each exchange a lane hands over the half of its values that the other keeps, so 4 + 2 + 1 + 1 exchanges, not 32.
__device__ __forceinline__ void sum_rows(float (&x)[8]) {
  const int n = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float keep = n & 4 ? x[i + 4] : x[i], give = n & 4 ? x[i] : x[i + 4];
    x[i] = keep + __shfl_xor(give, 4);
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float keep = n & 2 ? x[i + 2] : x[i], give = n & 2 ? x[i] : x[i + 2];
    x[i] = keep + lane_xor<2>(give);
  }
  const float keep = n & 1 ? x[1] : x[0], give = n & 1 ? x[0] : x[1];
  x[0] = keep + lane_xor<1>(give);
  x[0] += lane_xor<8>(x[0]);
}

struct WeightArgs {
  const float *qn, *lse;
  const void* kcache;
  const int* pos0;
  const uint64_t *tree, *rows;
  float* acc;
  int T, nqh, nkvh, n_ctx, splits, groups, tiles;
  float scale;
};

// attn_weights of up to 16 RT query rows: a workgroup takes a split of the cache rows of one kv head; the sum over the 16
// query rows of a tile is a lane reduction, that over row tiles is taken in order, and a row of the cache belongs to one
// wave: the same bits always.
template <bool Q8, int RT>
__global__ void __launch_bounds__(kWaves * 64, 2) attn_weights_kernel(WeightArgs a) {
  __shared__ union {
    QTile im[RT];
    HKeysLds w[Q8 ? 1 : kWaves];  // f16: the queries move to registers before the first K tile takes their place
  } sh;
  __shared__ float s_lse[RT * 16];
  __shared__ WaveLds s_w[Q8 ? kWaves : 1];
  QTile(&im)[RT] = sh.im;
  const int kh = blockIdx.x % a.nkvh, split = blockIdx.x / a.nkvh;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const Vis vis = vis_of(*a.pos0, a.T, a.n_ctx);
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const Split sp = split_of(tiles, a.splits, kWaves);
  if (split >= sp.used) return;
  const int t1 = split * sp.per + sp.per < tiles ? split * sp.per + sp.per : tiles;
  const int group = a.nqh / a.nkvh, rows = a.T * group;
  const uint64_t used = a.rows ? *a.rows : ~0ull;
  const KvHead kc = kv_head<Q8>(a.kcache, kh, a.nkvh, a.n_ctx);
  float* acc = a.acc + (size_t)kh * a.n_ctx;
  load_queries<Q8, kWaves, RT>(im, a.scale * kLog2e, [&](int r) {
    return r < rows ? a.qn + ((size_t)(r / group) * a.nqh + kh * group + r % group) * kHD : nullptr;
  });
  if (threadIdx.x < RT * 16) {
    const int r = threadIdx.x;
    const bool on = r < rows && ((used >> (r / group)) & 1);
    s_lse[threadIdx.x] = on ? a.lse[(size_t)(r / group) * a.nqh + kh * group + r % group] * kLog2e : __builtin_huge_valf();
  }
  __syncthreads();
  uint64_t tree[RT];
  float c[RT], lse[RT];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) {
    const int r = rt * 16 + n;
    tree[rt] = r < rows ? tree_of(a.tree, r / group, a.T) : 0ull;
    c[rt] = im[rt].c[n];
    lse[rt] = s_lse[rt * 16 + n];
  }
  QRegs q[RT];
  if constexpr (!Q8) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++) take_queries(q[rt], im[rt]);
    __syncthreads();
  }
  for (int t = split * sp.per + w; t < t1; t += kWaves) {
    const int j0 = t * kTileKeys;
    const bool full = j0 + kTileKeys <= vis.n;
    QRows k;
    f4 s[RT][2];
    if constexpr (Q8) {
      if (full) load_rows<false>(k, kc, j0, 0);
      else load_rows<true>(k, kc, j0, vis.end - j0);
    } else {
      if (full) request_keys<false>(sh.w[w], kc, j0, 0);
      else request_keys<true>(sh.w[w], kc, j0, vis.end - j0);
    }
    const int j = j0 + 16 * ((n >> 2) & 1) + 4 * g + (n & 3);  // the row this lane stores (n < 8)
    const bool mine = n < 8 && j < vis.end;
    const float old = mine && j < vis.n ? acc[j] : 0.0f;  // the weights of a drafted row begin here
    asm volatile("" ::: "memory");
    if constexpr (Q8) {
      __builtin_amdgcn_wave_barrier();
      stage_keys(k, s_w[w]);
      scores<RT>(s_w[w], im, s);
    } else {
      keys_there<0>();
      scores(sh.w[w], q, s);
    }
    if (!full) hide<RT, kMinusInf>(s, vis, tree, j0);
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      sum[e] = 0.0f;
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        const float x = s[rt][e >> 2][e & 3];
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c[rt], -lse[rt]));
        // rows not asked for, and hidden cache rows (of a query row that sees none lse is -inf too)
        sum[e] += lse[rt] == __builtin_huge_valf() || x == -__builtin_huge_valf() ? 0.0f : p;
      }
    }
    sum_rows(sum);
    if (mine) acc[j] = old + sum[0];
  }
}

// attn_weights of more than 32 query rows: K shared, row tiles w and WAVES + w in wave w (so that with 12 row tiles every
// SIMD, which runs waves w and w + 4, has three); a wave leaves its sums per cache row in LDS, and the first wave adds them
// up, in the waves' order, behind the barrier that ends the tile.
template <bool Q8, int WAVES, int RT>
__global__ void __launch_bounds__(WAVES * 64, 2) attn_weights_wide_kernel(WeightArgs a) {
  constexpr size_t kLds = sizeof(SharedTile) * 2 > sizeof(QTile) * WAVES ? sizeof(SharedTile) * 2 : sizeof(QTile) * WAVES;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[kLds];
  __shared__ float s_sum[2][WAVES][kTileKeys];
  QTile* im = (QTile*)s_mem;
  SharedTile* buf = (SharedTile*)s_mem;
  const int kh = blockIdx.x % a.nkvh, split = blockIdx.x / a.nkvh;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const Vis vis = vis_of(*a.pos0, a.T, a.n_ctx);
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const Split sp = split_of(tiles, a.splits, 1);
  if (split >= sp.used) return;
  const int t0 = split * sp.per, t1 = t0 + sp.per < tiles ? t0 + sp.per : tiles;
  if (t0 >= t1) return;
  const int group = a.nqh / a.nkvh, rows = a.T * group;
  const uint64_t used = a.rows ? *a.rows : ~0ull;
  const KvHead kc = kv_head<Q8>(a.kcache, kh, a.nkvh, a.n_ctx);
  float* acc = a.acc + (size_t)kh * a.n_ctx;
  auto left_of = [&](int t) { return vis.end - t * kTileKeys < kTileKeys ? vis.end - t * kTileKeys : kTileKeys; };
  for (int rg = 0; rg < a.groups; rg++) {
    const int first = rg * a.tiles * 16;
    auto ask = [&](Staged<Q8, WAVES>& n, int t) {
      if (t < t1) request<Q8, WAVES, true, false>(n, kc, kc, t * kTileKeys, left_of(t));
    };
    constexpr int kAhead = RT == 2 ? 1 : 2;  // tiles on their way; two row tiles' queries leave registers for one
    Staged<Q8, WAVES> even, two;
    Staged<Q8, WAVES>& odd = kAhead == 2 ? two : even;
    ask(even, t0);
    QRegs q[RT];
    float c[RT], lse[RT];
    bool on[RT], active[RT];
    auto row = [&](int rt) { return first + (rt * WAVES + w) * 16 + n; };  // this lane's query row, where it is one
    auto is_row = [&](int rt) { return rt * WAVES + w < a.tiles && row(rt) < rows; };
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      on[rt] = active[rt] = false;
      if (rt * WAVES >= a.tiles) continue;
      load_queries<Q8, WAVES, WAVES>(im, a.scale * kLog2e, [&](int r) {
        r += rt * WAVES * 16;
        const int q = first + r;
        return r < a.tiles * 16 && q < rows ? a.qn + ((size_t)(q / group) * a.nqh + kh * group + q % group) * kHD : nullptr;
      });
      __syncthreads();
      take_queries(q[rt], im[w]);
      c[rt] = im[w].c[n];
      const int r = row(rt);
      on[rt] = is_row(rt) && ((used >> (r / group)) & 1);
      lse[rt] = on[rt] ? a.lse[(size_t)(r / group) * a.nqh + kh * group + r % group] * kLog2e : 0.0f;
      active[rt] = __any(on[rt]);  // a row tile of which no row is asked for adds nothing
      __syncthreads();
    }
    stage<Q8, WAVES, true, false>(even, buf[0], false, 0, nullptr);
    ask(even, t0 + 1);
    if (kAhead == 2) ask(odd, t0 + 2);
    __syncthreads();
    float old = 0.0f;
    // threads 0 .. 31, behind the barrier of the tile before: its sums are added to its rows' weights
    auto add_up = [&](int t, int at) {
      const int j = t * kTileKeys + threadIdx.x;
      if (t < t0 || threadIdx.x >= kTileKeys || j >= vis.end) return;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < WAVES; k++) v += s_sum[at][k][threadIdx.x];
      acc[j] = old + v;
    };
    auto step = [&](int t, int at, Staged<Q8, WAVES>& next) __attribute__((always_inline)) {
      add_up(t - 1, at ^ 1);
      const int j = t * kTileKeys + threadIdx.x;
      if (threadIdx.x < kTileKeys && j < vis.end) old = j < vis.n || rg ? acc[j] : 0.0f;  // the weights of new rows begin here
      float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      auto add = [&](auto count) __attribute__((always_inline)) {  // the first `count` row tiles
        constexpr int kN = decltype(count)::value;
        f4 s[kN][2];
        scores<Q8>(buf[at], q, s);
        if ((t + 1) * kTileKeys > vis.n) {
          uint64_t bits[kN];
#pragma unroll
          for (int rt = 0; rt < kN; rt++) bits[rt] = is_row(rt) ? tree_of(a.tree, row(rt) / group, a.T) : 0ull;
          hide<kN, kMinusInf>(s, vis, bits, t * kTileKeys);
        }
#pragma unroll
        for (int rt = 0; rt < kN; rt++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float x = s[rt][e >> 2][e & 3];
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c[rt], -lse[rt]));
            sum[e] += !on[rt] || x == -__builtin_huge_valf() ? 0.0f : p;
          }
        sum_rows(sum);
      };
      if (RT == 2 && active[RT - 1]) add(std::integral_constant<int, RT>());
      else if (active[0]) add(std::integral_constant<int, 1>());
      if (n < 8) s_sum[at][w][16 * (n >> 2) + 4 * g + (n & 3)] = sum[0];
      if (t + 1 < t1) stage<Q8, WAVES, true, false>(next, buf[at ^ 1], false, 0, nullptr);
      ask(next, t + 1 + kAhead);
      __syncthreads();
    };
    int t = t0;
    if constexpr (kAhead == 1) {
#pragma unroll 1
      for (; t < t1; t++) step(t, (t - t0) & 1, even);
    } else {
      for (; t + 1 < t1; t += 2) {
        step(t, 0, even);
        step(t + 1, 1, odd);
      }
      if (t < t1) step(t++, 0, even);
    }
    add_up(t1 - 1, (t1 - 1 - t0) & 1);
    __syncthreads();  // the sums are read, the buffers free for the next group's queries
  }
}

// How attn_tree's and attn_weights' workgroups are laid out by the row tiles of 16 query rows. Up to two: each wave walks
// cache rows of its own. More: up to 8 waves of a row tile each share them, in as few groups as that takes, of equal size;
// attn_tree over q8_0 takes groups of 4 waves, two to a compute unit, where the fullest SIMD has less to do then (32 tokens,
// 65536 rows: 184 -> 170 us, 48: 275 -> 256 us; f16, bound by the matrix instructions and L2: 137 -> 140, 194 -> 206 us).
struct TreeLayout {
  int row_tiles, wide, groups, tiles, splits, waves;
};
TreeLayout tree_layout(int T, int nqh, int nkvh, int n_ctx, bool quarter) {
  TreeLayout t;
  t.row_tiles = (T * (nqh / nkvh) + 15) / 16;
  t.wide = t.row_tiles > 2;
  t.groups = t.wide ? (t.row_tiles + 7) / 8 : 1;
  const int quarters = (t.row_tiles + 3) / 4;
  if (quarter && t.wide && quarters < t.groups * (((t.row_tiles + t.groups - 1) / t.groups + 3) / 4)) t.groups = quarters;
  t.tiles = (t.row_tiles + t.groups - 1) / t.groups;
  // over the cache rows: a split is at least a tile for each (12 tokens of 500 rows: 27.8 us with four tiles to a split of
  // shared ones, 20 with one)
  t.waves = t.wide ? 1 : 4;
  // enough workgroups for every compute unit: two of 4 waves on each, or one of 8
  const int most = ((n_ctx + kTileKeys - 1) / kTileKeys + t.waves - 1) / t.waves;
  const bool half = t.wide ? t.tiles <= 4 : t.row_tiles == 1;
  int s = (half ? 2 * kCUs : kCUs) / t.groups / 8 * 8 / nkvh;  // the grid has 8 units (kv head, split) a round, see the kernels
  s = s > most ? most : s;
  t.splits = s < 1 ? 1 : s;
  return t;
}
int blocks_splits(int T, int nkvh, int nsel) {
  const long units = (long)T * nkvh;
  long s = 2 * kCUs / units;
  const long most = (2L * nsel + kWaves - 1) / kWaves;
  s = s > most ? most : s;
  return s < 1 ? 1 : (int)s;
}
size_t part_bytes(size_t rows, int splits) { return splits <= 1 ? 0 : rows * splits * (kHD + 2) * sizeof(float); }

bool heads_ok(int nqh, int nkvh) { return nkvh > 0 && nqh > 0 && nqh % nkvh == 0; }
// A grid holds less than 2^32 threads, and the grids below no more than a workgroup of 256 for each query row (the kernels
// with larger ones have 16 and more rows for each) and 7 beside.
bool rows_ok(int T, int nqh) { return (long long)T * nqh <= 0x7fffffffLL / 256; }

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_attn_tree_ws_bytes(int T, int nqh, int nkvh, int n_ctx) {
  if (T <= 0 || T > kMaxTree || !heads_ok(nqh, nkvh) || n_ctx <= 0 || !rows_ok(T, nqh)) return 0;
  const int s0 = tree_layout(T, nqh, nkvh, n_ctx, false).splits, s1 = tree_layout(T, nqh, nkvh, n_ctx, true).splits;
  return part_bytes((size_t)T * nqh, s0 > s1 ? s0 : s1);
}

extern "C" int q27h_attn_tree(const float* qn, const void* kcache, const void* vcache, const int* pos0, const uint64_t* tree,
                              int T, float scale, int nqh, int nkvh, int n_ctx, int q8, float* o, float* lse, void* ws,
                              size_t ws_bytes, q27h_stream_t s) {
  if (T < 0 || T > kMaxTree) return fail(Q27H_ERR_SHAPE, "attn_tree: T must be 0..64");
  if (!heads_ok(nqh, nkvh) || n_ctx <= 0) return fail(Q27H_ERR_SHAPE, "attn_tree: bad shape");
  if (!rows_ok(T, nqh)) return fail(Q27H_ERR_SHAPE, "attn_tree: too many query rows (T * nqh)");
  if (T == 0) return Q27H_OK;
  if (!qn || !kcache || !vcache || !pos0 || !o) return fail(Q27H_ERR_ARG, "attn_tree: null pointer");
  if (!aligned16(qn) || !aligned16(kcache) || !aligned16(vcache) || !aligned16(o) || !aligned16(ws))
    return fail(Q27H_ERR_ARG, "attn_tree: tensors need 16-byte alignment");
  if (!aligned8(tree) || !aligned4(lse) || !aligned4(pos0))
    return fail(Q27H_ERR_ARG, "attn_tree: tree needs 8-byte alignment, lse and pos0 4-byte");
  if (overlaps(qn, (size_t)T * nqh * kHD * 4, o, (size_t)T * nqh * kHD * 4)) return fail(Q27H_ERR_ARG, "attn_tree: o overlaps qn");
  const size_t need = q27h_attn_tree_ws_bytes(T, nqh, nkvh, n_ctx);
  if (ws_bytes < need || (need && !ws)) return fail(Q27H_ERR_ARG, "attn_tree: workspace too small");
  const size_t qb = (size_t)T * nqh * kHD * 4, cb = q27h_kv_cache_bytes(nkvh, n_ctx, q8);
  if (outputs_overlap({{o, qb}, {lse, (size_t)T * nqh * 4}, {ws, need}},
                      {{qn, qb}, {kcache, cb}, {vcache, cb}, {pos0, 4}, {tree, (size_t)T * 8}}))
    return fail(Q27H_ERR_ARG, "attn_tree: o, lse or ws overlaps another argument");
  AttnArgs a = {};
  a.qn = qn, a.kcache = kcache, a.vcache = vcache, a.pos0 = pos0, a.tree = tree, a.o = o, a.lse = lse;
  a.T = T, a.nqh = nqh, a.nkvh = nkvh, a.n_ctx = n_ctx, a.scale = scale;
  const TreeLayout lay = tree_layout(T, nqh, nkvh, n_ctx, q8 != 0);
  a.splits = lay.splits, a.groups = lay.groups, a.waves = lay.waves, a.tiles = lay.tiles;
  a.part = (float*)ws, a.ml = a.part + (size_t)T * nqh * a.splits * kHD;
  const dim3 grid((unsigned)((nkvh * a.splits + 7) / 8 * 8 * a.groups));
  if (lay.row_tiles == 1)
    hipLaunchKernelGGL((q8 ? attn_tree_kernel<true, 1, 4> : attn_tree_kernel<false, 1, 4>), grid, dim3(256), 0, stream_of(s), a);
  else if (lay.row_tiles == 2)
    hipLaunchKernelGGL((q8 ? attn_tree_kernel<true, 2, 4> : attn_tree_kernel<false, 2, 4>), grid, dim3(512), 0, stream_of(s), a);
  else if (lay.tiles <= 4)
    hipLaunchKernelGGL((q8 ? attn_wide_kernel<true, 4> : attn_wide_kernel<false, 4>), grid, dim3(256), 0, stream_of(s), a);
  else
    hipLaunchKernelGGL((q8 ? attn_wide_kernel<true, 8> : attn_wide_kernel<false, 8>), grid, dim3(512), 0, stream_of(s), a);
  if (lay.splits > 1) launch_join<false>(a, stream_of(s));
  return check_launch("attn_tree");
}

extern "C" int q27h_attn_weights(const float* qn, const float* lse, const void* kcache, const int* pos0, const uint64_t* tree,
                                 const uint64_t* rows, int T, float scale, int nqh, int nkvh, int n_ctx, int q8, float* acc,
                                 q27h_stream_t s) {
  if (T < 0 || T > kMaxTree) return fail(Q27H_ERR_SHAPE, "attn_weights: T must be 0..64");
  if (!heads_ok(nqh, nkvh) || n_ctx <= 0) return fail(Q27H_ERR_SHAPE, "attn_weights: bad shape");
  if (!rows_ok(T, nqh)) return fail(Q27H_ERR_SHAPE, "attn_weights: too many query rows (T * nqh)");
  if (T == 0) return Q27H_OK;
  if (!qn || !lse || !kcache || !pos0 || !acc) return fail(Q27H_ERR_ARG, "attn_weights: null pointer");
  if (!aligned16(qn) || !aligned16(kcache)) return fail(Q27H_ERR_ARG, "attn_weights: tensors need 16-byte alignment");
  if (!aligned8(tree) || !aligned8(rows) || !aligned4(lse) || !aligned4(acc) || !aligned4(pos0))
    return fail(Q27H_ERR_ARG, "attn_weights: tree and rows need 8-byte alignment, lse, acc and pos0 4-byte");
  const size_t qb = (size_t)T * nqh * kHD * 4, cb = q27h_kv_cache_bytes(nkvh, n_ctx, q8);
  if (outputs_overlap({{acc, (size_t)nkvh * n_ctx * 4}},
                      {{qn, qb}, {lse, (size_t)T * nqh * 4}, {kcache, cb}, {pos0, 4}, {tree, (size_t)T * 8}, {rows, 8}}))
    return fail(Q27H_ERR_ARG, "attn_weights: acc overlaps another argument");
  WeightArgs a = {};
  a.qn = qn, a.lse = lse, a.kcache = kcache, a.pos0 = pos0, a.tree = tree, a.rows = rows, a.acc = acc;
  a.T = T, a.nqh = nqh, a.nkvh = nkvh, a.n_ctx = n_ctx, a.scale = scale;
  TreeLayout lay = tree_layout(T, nqh, nkvh, n_ctx, false);
  // f16: without outputs a wave has registers for the queries of two row tiles. Taken where the fullest SIMD has less to do
  // (32 tokens, 65536 rows: 100 -> 80 us), not at equal work (64 tokens: 149 us either way). q8's products in flight leave none.
  const int two_groups = (lay.row_tiles + 15) / 16, two_tiles = (lay.row_tiles + two_groups - 1) / two_groups;
  const bool two = !q8 && lay.tiles > 4 && two_groups * ((two_tiles + 3) / 4) < lay.groups * ((lay.tiles + 3) / 4);
  if (two) lay.groups = two_groups, lay.tiles = two_tiles;
  a.groups = lay.groups, a.tiles = lay.tiles;
  const int waves = lay.wide ? 1 : kWaves, most = ((n_ctx + kTileKeys - 1) / kTileKeys + waves - 1) / waves;
  // narrow: two rounds of workgroups (two are resident on a compute unit, by their LDS); wide: as many as are resident
  a.splits = (!lay.wide ? 4 * kCUs : lay.tiles <= 4 ? 2 * kCUs : kCUs) / nkvh;
  a.splits = a.splits > most ? most : a.splits < 1 ? 1 : a.splits;
  const dim3 grid((unsigned)(nkvh * a.splits));
  if (lay.row_tiles == 1)
    hipLaunchKernelGGL((q8 ? attn_weights_kernel<true, 1> : attn_weights_kernel<false, 1>), grid, dim3(256), 0, stream_of(s), a);
  else if (lay.row_tiles == 2)
    hipLaunchKernelGGL((q8 ? attn_weights_kernel<true, 2> : attn_weights_kernel<false, 2>), grid, dim3(256), 0, stream_of(s), a);
  else if (lay.tiles <= 4)
    hipLaunchKernelGGL((q8 ? attn_weights_wide_kernel<true, 4, 1> : attn_weights_wide_kernel<false, 4, 1>), grid, dim3(256), 0,
                       stream_of(s), a);
  else
    hipLaunchKernelGGL((q8    ? attn_weights_wide_kernel<true, 8, 1>
                        : two ? attn_weights_wide_kernel<false, 8, 2>
                              : attn_weights_wide_kernel<false, 8, 1>),
                       grid, dim3(512), 0, stream_of(s), a);
  return check_launch("attn_weights");
}

extern "C" size_t q27h_attn_blocks_ws_bytes(int T, int nqh, int nkvh, int nsel) {
  if (T <= 0 || !heads_ok(nqh, nkvh) || nqh / nkvh > 16 || nsel <= 0) return 0;
  return part_bytes((size_t)T * nqh, blocks_splits(T, nkvh, nsel));
}

extern "C" int q27h_attn_blocks(const float* qn, const void* kcache, const void* vcache, const int* pos0, const int* idx, int T,
                                int nsel, float scale, int nqh, int nkvh, int n_ctx, int q8, float* o, float* lse, void* ws,
                                size_t ws_bytes, q27h_stream_t s) {
  if (T < 0 || nsel <= 0 || !heads_ok(nqh, nkvh) || nqh / nkvh > 16 || n_ctx <= 0)
    return fail(Q27H_ERR_SHAPE, "attn_blocks: bad shape (at most 16 query heads per kv head)");
  if (nsel > (1 << 20) || (long long)T * nqh > 0x7fffffffLL / 128) return fail(Q27H_ERR_SHAPE, "attn_blocks: T or nsel too large");
  if (T == 0) return Q27H_OK;
  if (!qn || !kcache || !vcache || !pos0 || !idx || !o) return fail(Q27H_ERR_ARG, "attn_blocks: null pointer");
  if (!aligned16(qn) || !aligned16(kcache) || !aligned16(vcache) || !aligned16(o) || !aligned16(ws))
    return fail(Q27H_ERR_ARG, "attn_blocks: tensors need 16-byte alignment");
  if (!aligned4(idx) || !aligned4(lse) || !aligned4(pos0))
    return fail(Q27H_ERR_ARG, "attn_blocks: idx, lse and pos0 need 4-byte alignment");
  if (overlaps(qn, (size_t)T * nqh * kHD * 4, o, (size_t)T * nqh * kHD * 4)) return fail(Q27H_ERR_ARG, "attn_blocks: o overlaps qn");
  const size_t need = q27h_attn_blocks_ws_bytes(T, nqh, nkvh, nsel);
  if (ws_bytes < need || (need && !ws)) return fail(Q27H_ERR_ARG, "attn_blocks: workspace too small");
  const size_t qb = (size_t)T * nqh * kHD * 4, cb = q27h_kv_cache_bytes(nkvh, n_ctx, q8);
  if (outputs_overlap({{o, qb}, {lse, (size_t)T * nqh * 4}, {ws, need}},
                      {{qn, qb}, {kcache, cb}, {vcache, cb}, {pos0, 4}, {idx, (size_t)T * nkvh * nsel * 4}}))
    return fail(Q27H_ERR_ARG, "attn_blocks: o, lse or ws overlaps another argument");
  AttnArgs a = {};
  a.qn = qn, a.kcache = kcache, a.vcache = vcache, a.pos0 = pos0, a.idx = idx, a.o = o, a.lse = lse;
  a.T = T, a.nqh = nqh, a.nkvh = nkvh, a.n_ctx = n_ctx, a.nsel = nsel, a.scale = scale;
  a.splits = blocks_splits(T, nkvh, nsel);
  a.part = (float*)ws, a.ml = a.part + (size_t)T * nqh * a.splits * kHD;
  const auto kern = q8 ? attn_blocks_kernel<true> : attn_blocks_kernel<false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((long)T * nkvh * a.splits)), dim3(256), 0, stream_of(s), a);
  if (a.splits > 1) launch_join<true>(a, stream_of(s));
  return check_launch("attn_blocks");
}
