// Attention of a batch of sequences over a K/V cache in pages (attn_paged): the new tokens of each sequence, one for plain
// decoding or a few with drafts, over all of its rows.
//
// A unit of work is (sequence, kv head, 16 or 32 query rows): query rows are tokens x query heads of the kv head, as in
// attn_tree. Sequences are of any length, so a unit's tiles of 32 cache rows are cut in parts none of which is longer than a
// fixed share of the tiles of all units. Every workgroup has a part, which it finds from the lengths of all sequences itself;
// its four waves each walk tiles of their own with the online softmax of attn_core.h. The parts of a unit that was cut go to
// the workspace, and a second launch joins those of each query row in order.
#include <type_traits>

#include "attn_wave.h"
#include "paged.h"

namespace q27h {
namespace {

constexpr int kWaves = 4;          // waves that share a segment's tiles
constexpr int kParts = 2 * kCUs;   // shares of the whole work, see cut_of
constexpr int kMostTokens = 64;    // tokens of one sequence: hide()'s 64-bit masks

struct PagedArgs {
  Pages pg;
  const float* qn;
  const int *pos, *cu;
  float *o, *lse;        // lse may be null
  float *part, *ml;      // [place][row of its unit][256], [..][2]
  int* starts;           // [n_seqs + 1]: each sequence's first place; the total of tiles
  int T, most, nqh;
  float scale;
};

// V in 4 bits: rows of 128 bytes as they lie, 16 a lane (row 8 r + (l >> 3), block l & 7).
struct QRows4 {
  u4 x[4];
  u2 s;
};
template <bool TAIL>
__device__ __forceinline__ void load_rows(QRows4& t, const KvHead& h, int j0, int left) {
  const int l = threadIdx.x & 63;
  const uint8_t* rows = h.rows + (ptrdiff_t)j0 * (kHD / 2);
#pragma unroll
  for (int r = 0; r < 4; r++) t.x[r] = *(const u4*)(rows + (unsigned)(tile_row<TAIL>(8 * r + (l >> 3), left) * (kHD / 2) + 16 * (l & 7)));
  t.s = *(const u2*)(h.scale + (ptrdiff_t)j0 * 16 + (unsigned)(tile_row<TAIL>(l >> 1, left) * 16 + 8 * (l & 1)));
  if (TAIL && (l >> 1) >= left) t.s = (u2){0u, 0u};
}
// To bytes in LDS, where the 8-bit form has its codes: the signs are turned and 8 is taken off with the turn to halves.
__device__ __forceinline__ void stage_values(const QRows4& t, WaveLds& w) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    u4 lo, hi;
#pragma unroll
    for (int i = 0; i < 4; i++) lo[i] = t.x[r][i] & 0x0f0f0f0fu, hi[i] = t.x[r][i] >> 4 & 0x0f0f0f0fu;
    uint8_t* p = w.codes + (r >= 2 ? kUpper + (8 * (r - 2) + (l >> 3)) * kRow : (8 * r + (l >> 3)) * kRow) + 32 * (l & 7);
    *(u4*)p = lo;
    *(u4*)(p + 16) = hi;
  }
  put_value_scales(t.s, w.vs, w.vf);
  __builtin_amdgcn_wave_barrier();
}

}  // namespace
template <>
constexpr int bias_of<QRows4> = 8;
namespace {

// A tile's place: K and V of its page and head, such that the sequence's row j lies at rows + j * (bytes of a row).
struct TileAt {
  KvHead k, v;
  int j0;  // -1: none
};

// The tiles of one wave, t, t + kWaves, ... up to `end`. The page of the next one is asked for a tile ahead. A tile whose
// page is none of the cache's is passed over: its rows do not exist.
template <int TYPE>
struct PageWalk {
  const Pages& pg;
  const int* table;
  int kh, t, end, page;
  __device__ __forceinline__ PageWalk(const Pages& p, int b, int kh_, int first, int end_)
      : pg(p), table(p.table + (size_t)b * p.max_pages), kh(kh_), t(first), end(end_), page(-1) {
    ask();
  }
  __device__ __forceinline__ void ask() {
    if (t < end) page = uniform_load(table + (t >> (pg.shift - 5)));
  }
  __device__ __forceinline__ TileAt next(int limit) {
    TileAt a;
    a.j0 = -1;
    while (t < limit) {
      const int cur = t, p = page;
      t += kWaves;
      ask();
      if ((unsigned)p >= (unsigned)pg.n_pages) continue;
      a.j0 = cur * kTileKeys;
      const int n = 1 << pg.shift, first = a.j0 & -n;  // the sequence's first row in the page
      constexpr int kR = TYPE == Q27H_KV_F16 ? 2 * kHD : kHD, vR = TYPE == Q27H_KV_Q8_Q4 ? kHD / 2 : kR;
      const uint8_t *k = pg.k + (size_t)p * pg.kb, *v = pg.v + (size_t)p * pg.vb;
      const ptrdiff_t row = (ptrdiff_t)kh * n - first;
      a.k.rows = k + row * kR, a.v.rows = v + row * vR;
      a.k.scale = k + (size_t)pg.nkvh * n * kHD + row * 16, a.v.scale = v + (size_t)pg.nkvh * n * vR + row * 16;
      break;
    }
    return a;
  }
};

// A wave's tiles that are wholly visible, as attn_tree's: the loads of the next one behind the arithmetic of this one.
template <int TYPE>
struct PagedTiles {
  QRows k;
  std::conditional_t<TYPE == Q27H_KV_Q8_Q4, QRows4, QRows> v;
  TileAt at;
  template <typename F>
  __device__ __forceinline__ void begin(F next) {
    at = next();
    if (at.j0 < 0) return;
    load_rows<false>(k, at.k, at.j0, 0);
    load_rows<false>(v, at.v, at.j0, 0);
  }
  template <typename F>
  __device__ __forceinline__ void run(Rows& st, const Queries<true>& q, WaveLds& w, F next) {
    if (at.j0 < 0) return;
    do {
      f4 s[1][2];
      at = next();
      asm volatile("" ::: "memory");  // the queries are read from LDS for each tile: held in registers they would spill
      stage_keys(k, w);
      if (at.j0 >= 0) load_rows<false>(k, at.k, at.j0, 0);
      loads_issued();
      scores<1>(w, q.im, s);
      weights<true, false>(st, s[0]);
      __builtin_amdgcn_wave_barrier();
      stage_values(v, w);
      if (at.j0 >= 0) load_rows<false>(v, at.v, at.j0, 0);
      loads_issued();
      accumulate<false, bias_of<decltype(v)>>(st, s[0], w);
      __builtin_amdgcn_wave_barrier();
    } while (at.j0 >= 0);
  }
};
template <>
struct PagedTiles<Q27H_KV_F16> {
  HValues v;
  TileAt at;
  template <typename F>
  __device__ __forceinline__ void begin(F next) {
    at = next();
  }
  template <typename F>
  __device__ __forceinline__ void run(Rows& st, const Queries<false>& q, HKeysLds& w, F next) {
    if (at.j0 < 0) return;
    request_keys<false>(w, at.k, at.j0, 0);
    loads_issued();
    load_rows<false>(v, at.v, at.j0, 0);
    do {
      f4 s[1][2];
      at = next();
      keys_there<kValueLoads>();
      scores(w, q.r, s);
      keys_there<0>();  // V is waited for before the next K is, as in attn_tree
      if (at.j0 >= 0) request_keys<false>(w, at.k, at.j0, 0);
      loads_issued();
      weights<false, false>(st, s[0]);
      accumulate(st, s[0], v);
      if (at.j0 >= 0) load_rows<false>(v, at.v, at.j0, 0);
      loads_issued();
    } while (at.j0 >= 0);
  }
};

// What a sequence asks for: its units (kv heads x groups of `rows` query rows), and the tiles of each, of which a unit of
// the plan has a multiple of kWaves: that is what a step of the workgroup costs. A sequence without rows has a tile too,
// which finds none of them and writes zeros.
struct Demand {
  int units, span;
};
__device__ __forceinline__ Demand demand_of(const PagedArgs& a, int nt, const Vis& vis, int rows) {
  const int tiles = vis.end > 0 ? (vis.end + kTileKeys - 1) / kTileKeys : 1;
  return {a.pg.nkvh * ((nt * (a.nqh / a.pg.nkvh) + rows - 1) / rows), (tiles + kWaves - 1) / kWaves * kWaves};
}
// A unit of `span` tiles, `total` of them in all, is cut in `parts` of `size`: none is longer than a kParts-th of the total.
struct Cut {
  int parts, size;
};
__device__ __forceinline__ Cut cut_of(int span, int total) {
  const int most = ((total + kParts - 1) / kParts + kWaves - 1) / kWaves * kWaves;
  Cut c;
  c.parts = (span + most - 1) / most;
  c.size = ((span + c.parts - 1) / c.parts + kWaves - 1) / kWaves * kWaves;
  c.parts = (span + c.size - 1) / c.size;  // rounding up to a step may leave the last one nothing
  return c;
}

// The part that a workgroup has: sequence, unit of it, the part's number in the unit and the unit's cut, its total of tiles,
// and the part's place in the workspace. seq < 0: none. The first workgroup leaves for the join where the places of each
// sequence begin, and the total behind them.
struct Part {
  int seq, unit, k, place;
  Cut cut;
};
template <int THREADS>
__device__ __forceinline__ Part part_of(const PagedArgs& a, int rows) {
  constexpr int kW = THREADS / 64;
  __shared__ int s_total[kW], s_part[3];
  __shared__ uint64_t s_count[kW];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, cap = a.pg.max_pages << a.pg.shift;
  const int each = (a.pg.n_seqs + THREADS - 1) / THREADS, b0 = tid * each;
  const int b1 = b0 + each < a.pg.n_seqs ? b0 + each : a.pg.n_seqs;
  auto demand = [&](int b) {
    const Tokens tk = a.cu ? tokens_of(a.cu[b], a.cu[b + 1], a.T, a.most) : tokens_of(b, b + 1, a.T, a.most);
    return demand_of(a, tk.nt, vis_of(a.pos[b], tk.nt, cap), rows);
  };
  const Demand first = b0 < b1 ? demand(b0) : Demand{0, 0};
  int sum = first.units * first.span;
  for (int b = b0 + 1; b < b1; b++) {
    const Demand d = demand(b);
    sum += d.units * d.span;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (l == 0) s_total[w] = sum;
  if (tid == 0) s_part[0] = -1;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int k = 0; k < kW; k++) total += s_total[k];
  // workgroups below, and above them the places of the parts that are joined
  auto count = [&](const Demand& d) {
    const int parts = cut_of(d.span, total).parts;
    const uint64_t n = (uint64_t)d.units * parts;
    return d.units == 0 ? 0ull : parts > 1 ? n << 32 | n : n;
  };
  uint64_t mine = count(first);
  for (int b = b0 + 1; b < b1; b++) mine += count(demand(b));
  uint64_t before = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t y = __shfl_up(before, d);
    before += l >= d ? y : 0;
  }
  if (l == 63) s_count[w] = before;
  __syncthreads();
  before -= mine;
#pragma unroll
  for (int k = 0; k < kW; k++) before += k < w ? s_count[k] : 0;
  const int me = (int)blockIdx.x;
  const bool here = (int)before <= me && me < (int)(before + mine);
  if (me == 0 && tid == 0) a.starts[a.pg.n_seqs] = total;
  if (me == 0 || here) {
    uint64_t at = before;
    for (int b = b0; b < b1; b++) {
      const uint64_t n = count(b == b0 ? first : demand(b));
      if (me == 0) a.starts[b] = (int)(at >> 32);
      if ((int)at <= me && me < (int)(at + n)) s_part[0] = b, s_part[1] = me - (int)at, s_part[2] = (int)(at >> 32);
      at += n;
    }
  }
  __syncthreads();
  Part p;
  p.seq = __builtin_amdgcn_readfirstlane(s_part[0]);
  if (p.seq < 0) return p;
  const int i = __builtin_amdgcn_readfirstlane(s_part[1]);
  const Tokens tk = tokens_of(a.cu, p.seq, a.T, a.most);
  p.cut = cut_of(demand_of(a, tk.nt, vis_of(uniform_load(a.pos + p.seq), tk.nt, cap), rows).span, __builtin_amdgcn_readfirstlane(total));
  p.unit = i / p.cut.parts, p.k = i - p.unit * p.cut.parts;
  p.place = __builtin_amdgcn_readfirstlane(s_part[2]) + i;
  return p;
}

template <int TYPE, int WR>
__global__ void __launch_bounds__(WR * kWaves * 64, 2) attn_paged_kernel(PagedArgs a) {
  constexpr bool Q8 = TYPE != Q27H_KV_F16;
  constexpr int kRows = 16 * WR;
  __shared__ AttnShared<Q8, WR, kWaves> sh;
  const Part pt = part_of<WR * kWaves * 64>(a, kRows);
  if (pt.seq < 0) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = w % WR, wk = w / WR;
  const int group = a.nqh / a.pg.nkvh;
  const Tokens tk = tokens_of(a.cu, pt.seq, a.T, a.most);
  const Vis vis = vis_of(uniform_load(a.pos + pt.seq), tk.nt, a.pg.max_pages << a.pg.shift);
  const int rows = tk.nt * group, groups = (rows + kRows - 1) / kRows, kh = pt.unit / groups, first = (pt.unit - kh * groups) * kRows;
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const int t0 = pt.k * pt.cut.size, t1 = t0 + pt.cut.size < tiles ? t0 + pt.cut.size : tiles;
  const int full = vis.n / kTileKeys < t1 ? vis.n / kTileKeys : t1;
  auto row = [&](int r) {  // the global row (token * nqh + head) of the unit's query row r, or -1
    r += first;
    return r < rows ? (tk.t0 + r / group) * a.nqh + kh * group + r % group : -1;
  };
  PageWalk<TYPE> walk(a.pg, pt.seq, kh, t0 + wk, t1);
  PagedTiles<TYPE> ft;
  ft.begin([&] { return walk.next(full); });
  load_queries<Q8, WR * kWaves, WR>(sh.q, a.scale * kLog2e, [&](int r) {
    const int gr = row(r);
    return gr < 0 ? nullptr : a.qn + (size_t)gr * kHD;
  });
  __syncthreads();
  Rows st;
  Queries<Q8> q;
  begin_rows(st, q, sh, wr, wk);
  ft.run(st, q, sh.w[w], [&] { return walk.next(full); });
  int mine = wr * 16 + (threadIdx.x & 15);
  asm volatile("" : "+v"(mine));  // the lane's row is formed here: kept over the tiles it would take registers that they need
  const int gr = row(mine);
  const uint64_t chain = gr >= 0 ? ~0ull >> (63 - (first + mine) / group) : 0ull;
  for (TileAt at = walk.next(t1); at.j0 >= 0; at = walk.next(t1)) {
    if constexpr (TYPE == Q27H_KV_Q8_Q4) tail_tile<QRows4>(st, at.k, at.v, q, sh.w[w], vis, chain, at.j0);
    else tail_tile(st, at.k, at.v, q, sh.w[w], vis, chain, at.j0);
  }
  const bool whole = pt.cut.parts == 1;
  const size_t place = (size_t)pt.place * kRows + mine;
  finish<Q8, WR, kWaves>(st, sh, [&a, gr, whole, place](Rows& st, float m, float sum) {
    if (gr < 0) return;
    const bool lead = (threadIdx.x & 63) < 16;
    float* dst;
    if (whole) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int i = 0; i < 16; i++) st.o[i] *= inv;
      dst = a.o + (size_t)gr * kHD;
      if (a.lse && lead) a.lse[gr] = sum == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
    } else {
      dst = a.part + place * kHD;
      if (lead) *(float2*)(a.ml + place * 2) = make_float2(m, sum);
    }
    store_rows<Q8>(st, dst);
  });
}

// Joins the parts of one query row (token t of sequence b, query head h), in order: wave w of WAVES takes every WAVES-th
// part, a lane four dims; then the waves' sums are added in order. 16 waves where there are few rows, which may have many
// parts; 4 where there are many.
template <int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 8) attn_paged_join_kernel(PagedArgs a, int rows) {
  __shared__ f4 s_o[WAVES][64];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const int h = blockIdx.x % a.nqh, t = (int)(blockIdx.x / a.nqh) % a.most, b = (int)(blockIdx.x / a.nqh) / a.most;
  const int start = uniform_load(a.starts + b), total = uniform_load(a.starts + a.pg.n_seqs), pos = uniform_load(a.pos + b);
  const Tokens tk = tokens_of(a.cu, b, a.T, a.most);
  if (t >= tk.nt) return;
  const Vis vis = vis_of(pos, tk.nt, a.pg.max_pages << a.pg.shift);
  const int n = cut_of(demand_of(a, tk.nt, vis, rows).span, total).parts;
  if (n == 1) return;
  const int group = a.nqh / a.pg.nkvh, r = t * group + h % group, groups = (tk.nt * group + rows - 1) / rows;
  const size_t place = ((size_t)start + (size_t)(h / group * groups + r / rows) * n) * rows + r % rows;
  const f4* part = (const f4*)(a.part + place * kHD) + l;  // part k: k * rows rows on
  const float2* ml = (const float2*)a.ml + place;
  constexpr int kBatch = 4;
  f4 x[kBatch];
#pragma unroll
  for (int k = 0; k < kBatch; k++)
    if (w + WAVES * k < n) x[k] = part[(size_t)(w + WAVES * k) * rows * 64];
  auto all = [&](float y, auto op) {
    y = op(y, lane_xor<1>(y));
    y = op(y, lane_xor<2>(y));
    y = op(y, lane_xor<7>(y));
    y = op(y, lane_xor<8>(y));
    y = op(y, lane_xor<16>(y));
    return op(y, lane_xor32(y));
  };
  // every wave for itself, lane l parts l, l + 64, ..
  float2 v = l < n ? ml[l * rows] : make_float2(-3.0e38f, 0.0f);
  float m = v.x;
  for (int k = l + 64; k < n; k += 64) m = __builtin_fmaxf(m, ml[k * rows].x);
  m = all(m, [](float p, float q) { return __builtin_fmaxf(p, q); });
  const float f = __builtin_amdgcn_exp2f(v.x - m);
  float sum = v.y * f;
  for (int k = l + 64; k < n; k += 64) sum += ml[k * rows].y * __builtin_amdgcn_exp2f(ml[k * rows].x - m);
  sum = all(sum, [](float p, float q) { return p + q; });
  auto factor = [&](int k) {  // of part k, the same in the whole wave
    return k < 64 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), k))
                  : __builtin_amdgcn_exp2f(ml[k * rows].x - m);
  };
  f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  const int w0 = __builtin_amdgcn_readfirstlane(w);
#pragma unroll
  for (int k = 0; k < kBatch; k++)
    if (w0 + WAVES * k < n) o += x[k] * factor(w0 + WAVES * k);
  for (int k0 = w0 + WAVES * kBatch; k0 < n; k0 += WAVES * kBatch) {
#pragma unroll
    for (int k = 0; k < kBatch; k++)
      if (k0 + WAVES * k < n) x[k] = part[(size_t)(k0 + WAVES * k) * rows * 64];
#pragma unroll
    for (int k = 0; k < kBatch; k++)
      if (k0 + WAVES * k < n) o += x[k] * factor(k0 + WAVES * k);
  }
  s_o[w][l] = o;
  __syncthreads();
  if (w) return;
#pragma unroll
  for (int k = 1; k < WAVES; k++) o += s_o[k][l];
  const size_t gr = (size_t)(tk.t0 + t) * a.nqh + h;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  *((f4*)(a.o + gr * kHD) + l) = o * inv;
  if (a.lse && l == 0) a.lse[gr] = sum == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

struct Layout {
  int wr, grid;
  size_t places, bytes;
};
// Up to 16 query rows a kv head: one row tile, two workgroups of four waves a compute unit; more: two row tiles, whose waves
// read the same cache rows, one workgroup of eight.
Layout layout_of(int n_seqs, int max_tokens, int nqh, int nkvh) {
  Layout y;
  const int rows = max_tokens * (nqh / nkvh);
  y.wr = rows <= 16 ? 1 : 2;
  // cut_of gives a unit at most one part more than its share of kParts, and two at least where it is cut at all
  const int units = n_seqs * nkvh * ((rows + 16 * y.wr - 1) / (16 * y.wr));
  y.grid = units + kParts;
  y.places = (size_t)(y.grid < 2 * kParts ? y.grid : 2 * kParts) * 16 * y.wr;
  y.bytes = y.places * (kHD + 2) * sizeof(float) + ((size_t)n_seqs + 1) * sizeof(int);
  return y;
}
bool shape_ok(const q27h_kv_pages* kv, int max_tokens, int nqh) {
  return max_tokens >= 1 && max_tokens <= kMostTokens && nqh > 0 && nqh <= 4096 && nqh % kv->nkvh == 0;
}

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_attn_paged_ws_bytes(const q27h_kv_pages* kv, int T, int max_tokens, int nqh) {
  if (check_pages(kv, "attn_paged") != Q27H_OK || T <= 0 || !shape_ok(kv, max_tokens, nqh)) return 0;
  return layout_of(kv->n_seqs, max_tokens, nqh, kv->nkvh).bytes;
}

extern "C" int q27h_attn_paged(const float* qn, const q27h_kv_pages* kv, const int* pos, const int* cu, int T, int max_tokens,
                               float scale, int nqh, float* o, float* lse, void* ws, size_t ws_bytes, q27h_stream_t s) {
  if (const int bad = check_pages(kv, "attn_paged")) return bad;
  if (T < 0 || !shape_ok(kv, max_tokens, nqh))
    return fail(Q27H_ERR_SHAPE, "attn_paged: bad shape (1 to 64 tokens a sequence, at most 4096 query heads)");
  if (!cu && T != kv->n_seqs) return fail(Q27H_ERR_SHAPE, "attn_paged: without cu there is one token for each sequence");
  const int group = nqh / kv->nkvh;
  const long long tiles = ((long long)kv->max_pages * kv->page_rows / kTileKeys + kWaves - 1) / kWaves * kWaves;
  if ((double)kv->n_seqs * kv->nkvh * ((max_tokens * group + 15) / 16) * (double)tiles > 2.0e9)
    return fail(Q27H_ERR_SHAPE, "attn_paged: too many rows in all");
  if ((long long)kv->n_seqs * max_tokens * nqh > 0x7fffffffLL / 256 || (long long)T * nqh > 0x7fffffffLL / 256)
    return fail(Q27H_ERR_SHAPE, "attn_paged: too many query rows");
  if (T == 0 || kv->n_seqs == 0) return Q27H_OK;
  if (!qn || !pos || !o) return fail(Q27H_ERR_ARG, "attn_paged: null pointer");
  if (!aligned16(qn) || !aligned16(o) || !aligned16(ws)) return fail(Q27H_ERR_ARG, "attn_paged: tensors need 16-byte alignment");
  if (!aligned4(pos) || !aligned4(cu) || !aligned4(lse)) return fail(Q27H_ERR_ARG, "attn_paged: pos, cu and lse need 4-byte alignment");
  const Layout y = layout_of(kv->n_seqs, max_tokens, nqh, kv->nkvh);
  if (ws_bytes < y.bytes || !ws) return fail(Q27H_ERR_ARG, "attn_paged: workspace too small");
  const Pages pg = pages_of(kv);
  const size_t qb = (size_t)T * nqh * kHD * 4, B = (size_t)kv->n_seqs;
  if (outputs_overlap({{o, qb}, {lse, (size_t)T * nqh * 4}, {ws, y.bytes}},
                      {{qn, qb}, {pg.k, pg.kb * pg.n_pages}, {pg.v, pg.vb * pg.n_pages}, {pg.table, B * pg.max_pages * 4},
                       {pos, B * 4}, {cu, (B + 1) * 4}}))
    return fail(Q27H_ERR_ARG, "attn_paged: o, lse or ws overlaps another argument");
  PagedArgs a = {};
  a.pg = pg, a.qn = qn, a.pos = pos, a.cu = cu, a.o = o, a.lse = lse, a.T = T, a.most = max_tokens, a.nqh = nqh, a.scale = scale;
  a.part = (float*)ws, a.ml = a.part + y.places * kHD, a.starts = (int*)(a.ml + y.places * 2);
  const dim3 grid((unsigned)y.grid), block(256 * y.wr);
  auto launch = [&](auto one, auto two) { hipLaunchKernelGGL((y.wr == 1 ? one : two), grid, block, 0, stream_of(s), a); };
  if (kv->type == Q27H_KV_F16) launch(attn_paged_kernel<Q27H_KV_F16, 1>, attn_paged_kernel<Q27H_KV_F16, 2>);
  else if (kv->type == Q27H_KV_Q8) launch(attn_paged_kernel<Q27H_KV_Q8, 1>, attn_paged_kernel<Q27H_KV_Q8, 2>);
  else launch(attn_paged_kernel<Q27H_KV_Q8_Q4, 1>, attn_paged_kernel<Q27H_KV_Q8_Q4, 2>);
  const int qrows = kv->n_seqs * max_tokens * nqh;
  if (qrows <= 2 * kCUs)
    hipLaunchKernelGGL(attn_paged_join_kernel<16>, dim3((unsigned)qrows), dim3(1024), 0, stream_of(s), a, 16 * y.wr);
  else
    hipLaunchKernelGGL(attn_paged_join_kernel<4>, dim3((unsigned)qrows), dim3(256), 0, stream_of(s), a, 16 * y.wr);
  return check_launch("attn_paged");
}
