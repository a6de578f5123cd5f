// Attention of a batch of sequences over a K/V cache in pages (attn_paged): the new tokens of each sequence, one for plain
// decoding or a few with drafts (a chain or a tree), over all of its rows.
//
// A unit of work is (sequence, kv head, 16 or 32 query rows): query rows are tokens x query heads of the kv head, as in
// attn_tree. Sequences are of any length, so a unit's tiles of 32 cache rows are cut in parts none of which is longer than a
// fixed share of the tiles of all units. Every workgroup has a part, which it finds from the lengths of all sequences
// itself. Up to 16 query rows (over f16 32), its waves each walk tiles of their own with the online softmax of attn_core.h,
// bound by HBM (128 sequences of 4096 q8_0 rows, one token: 5.3 TB/s; f16, 2048 rows, four tokens: 5.0); with more they share
// them, see below. The parts of a unit that was cut go to the workspace, and a second launch joins those of each query
// row in order.
#include <type_traits>

#include "attn_shared.h"
#include "attn_wave.h"
#include "paged.h"

namespace q27h {
namespace {

constexpr int kWaves = 4;        // waves that share a part's tiles
constexpr int kMostTokens = 64;  // tokens of one sequence: hide()'s 64-bit masks

struct PagedArgs {
  Pages pg;
  const float* qn;
  const int *pos, *cu;
  const uint64_t* tree;  // may be null
  float *o, *lse;        // lse may be null
  float *part, *ml;      // [place][row of its unit][256], [..][2]
  int* starts;           // [n_seqs][2]: each sequence's first place, and the parts of each of its units
  int T, most, nqh, slots;  // slots: shares of the whole work, about the workgroups that run at a time
  int least;                // tiles; 0: parts are total / slots, else down to half of that where they are no shorter than this
  int rows;                 // query rows of a unit
  int group;                // query heads of a kv head
  float scale;
};

// Which of its sequence's new tokens token t of them sees: a bit for each.
__device__ __forceinline__ uint64_t tree_of(const PagedArgs& a, const Tokens& tk, int t) {
  return a.tree ? a.tree[tk.t0 + t] : ~0ull >> (63 - t);
}

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

// The tiles of one wave, or of a workgroup whose waves share them: t, t + STEP, ... up to `end`. The page of the next one is asked for a tile ahead. A tile whose
// page is none of the cache's is passed over: its rows do not exist.
template <int TYPE, int STEP = kWaves>
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
      t += STEP;
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
  return {a.pg.nkvh * ((nt * a.group + rows - 1) / rows), (tiles + kWaves - 1) / kWaves * kWaves};
}
// Every unit is cut in parts of one size, its last one what is left: the total by the shares. FINE: see a.least.
template <bool FINE>
__device__ __forceinline__ int size_of(const PagedArgs& a, int total) {
  int each = (total + a.slots - 1) / a.slots;
  if (FINE && a.least) {
    const int half = (each + 1) / 2;
    each = half >= a.least ? half : each < a.least ? each : a.least;
  }
  return each ? (each + kWaves - 1) / kWaves * kWaves : kWaves;
}

// The part that a workgroup has: sequence, unit of it, the part's number in the unit and how many it has, their size, and
// the part's place in the workspace. seq < 0: none. Whole parts come before those that are left over, and of these the ones
// over half the size before the others: workgroups start in this order as others end, so that the last to end are short (48
// sequences of 500 to 32768 rows, 4 tokens each, with the kernel of that time: 293 us with parts in any order, 250 so). The
// first workgroup leaves for the join where the places of each sequence begin and how many parts its units have.
struct Part {
  int seq, unit, k, parts, size, place;
  Tokens tk;
  int pos;
};
// The i-th of a sequence's parts of one kind, of which each unit has n. The units of a kv head read the same rows: theirs
// follow each other 8 workgroups apart, which is on one XCD (16 sequences of 32768 q8_0 rows, 12 tokens: 650 -> 632 us).
__device__ __forceinline__ void place_of(const PagedArgs& a, int i, int n, int groups, int& unit, int& k) {
  int at = i, g = 0;
  if (groups > 1) {
    const int all = a.pg.nkvh * n, round = i / (8 * groups), j = i - round * 8 * groups;
    const int wide = all - 8 * round < 8 ? all - 8 * round : 8;
    g = j / wide;
    at = 8 * round + j - g * wide;
  }
  unit = at / n;
  k = at - unit * n;
  unit = unit * groups + g;
}
struct Counts {
  uint64_t a, b;  // whole parts, and above them places of parts that are joined; large rests, and above them small ones
};
// Sums over the lanes up to each one.
__device__ __forceinline__ int lanes_before(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within rows of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31: the rows before
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
// Up to 64 sequences: every wave finds the part by itself, a sequence in each lane, without a barrier.
template <bool FINE>
__device__ __forceinline__ Part part_of_64(const PagedArgs& a, int rows) {
  const int l = threadIdx.x & 63, cap = a.pg.max_pages << a.pg.shift;
  const bool is = l < a.pg.n_seqs;
  int c0 = l, c1 = l + 1, pos = 0;
  if (is) {
    pos = a.pos[l];
    if (a.cu) c0 = a.cu[l], c1 = a.cu[l + 1];
  }
  const Tokens tk = tokens_of(c0, c1, a.T, a.most);
  const Demand d = is ? demand_of(a, tk.nt, vis_of(pos, tk.nt, cap), rows) : Demand{0, kWaves};
  Part p;
  p.size = size_of<FINE>(a, __builtin_amdgcn_readlane(lanes_before(d.units * d.span), 63));
  const int whole = d.span / p.size, rest = d.span - whole * p.size, parts = whole + (rest > 0);
  const int n0 = d.units * whole, n1 = 2 * rest > p.size ? d.units : 0, n2 = rest && !n1 ? d.units : 0, np = parts > 1 ? d.units * parts : 0;
  const int s0 = lanes_before(n0), s1 = lanes_before(n1), s2 = lanes_before(n2), sp = lanes_before(np);
  const int all0 = __builtin_amdgcn_readlane(s0, 63), all1 = __builtin_amdgcn_readlane(s1, 63);
  if (blockIdx.x == 0 && threadIdx.x < 64) {
    if (is) *(int2*)(a.starts + 2 * l) = make_int2(sp - np, parts);
  }
  int me = (int)blockIdx.x, kind = 0;
  if (me >= all0) me -= all0, kind = 1;
  if (kind == 1 && me >= all1) me -= all1, kind = 2;
  const int n = kind == 0 ? n0 : kind == 1 ? n1 : n2, x = (kind == 0 ? s0 : kind == 1 ? s1 : s2) - n;
  const uint64_t here = __ballot(x <= me && me < x + n);
  p.seq = -1;
  if (!here) return p;
  p.seq = __builtin_ctzll(here);
  auto of = [&](int y) { return __builtin_amdgcn_readlane(y, p.seq); };
  const int w = of(whole);
  p.parts = of(parts);
  p.tk = {of(tk.t0), of(tk.nt)};
  place_of(a, me - of(x), kind == 0 ? w : 1, (p.tk.nt * a.group + rows - 1) / rows, p.unit, p.k);
  if (kind) p.k = w;
  p.place = of(sp - np) + p.unit * p.parts + p.k;
  p.pos = of(pos);
  return p;
}
template <int THREADS, bool FINE = false>
__device__ __forceinline__ Part part_of(const PagedArgs& a, int rows) {
  if (a.pg.n_seqs <= 64) return part_of_64<FINE>(a, rows);
  constexpr int kW = THREADS / 64;
  __shared__ int s_total[kW], s_part[3];
  __shared__ Counts s_count[kW];
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
  Part p;
  p.size = size_of<FINE>(a, total);
  auto count = [&](const Demand& d) {
    const int whole = d.span / p.size, rest = d.span - whole * p.size;
    const uint32_t u = (uint32_t)d.units, parts = whole + (rest > 0);
    return Counts{(uint64_t)(parts > 1 ? u * parts : 0) << 32 | u * whole,
                  rest == 0 ? 0ull : 2 * rest > p.size ? (uint64_t)u : (uint64_t)u << 32};
  };
  Counts mine = count(first);
  for (int b = b0 + 1; b < b1; b++) {
    const Counts c = count(demand(b));
    mine.a += c.a, mine.b += c.b;
  }
  Counts at = mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t x = __shfl_up(at.a, d), y = __shfl_up(at.b, d);
    at.a += l >= d ? x : 0, at.b += l >= d ? y : 0;
  }
  if (l == 63) s_count[w] = at;
  __syncthreads();
  at.a -= mine.a, at.b -= mine.b;
  Counts all = {0, 0};
#pragma unroll
  for (int k = 0; k < kW; k++) {
    if (k < w) at.a += s_count[k].a, at.b += s_count[k].b;
    all.a += s_count[k].a, all.b += s_count[k].b;
  }
  // the workgroup's number among the whole parts, the large rests or the small ones
  int me = (int)blockIdx.x, kind = 0;
  if (me >= (int)all.a) me -= (int)all.a, kind = 1;
  if (kind == 1 && me >= (int)all.b) me -= (int)all.b, kind = 2;
  auto of_kind = [&](const Counts& c) { return kind == 0 ? (int)c.a : kind == 1 ? (int)c.b : (int)(c.b >> 32); };
  const int lo = of_kind(at);
  const bool lead = blockIdx.x == 0, here = lo <= me && me < lo + of_kind(mine);
  if (lead || here) {
    for (int b = b0; b < b1; b++) {
      const Demand d = b == b0 ? first : demand(b);
      const Counts c = count(d);
      const int x = of_kind(at);
      if (lead) *(int2*)(a.starts + 2 * b) = make_int2((int)(at.a >> 32), (d.span + p.size - 1) / p.size);
      if (x <= me && me < x + of_kind(c)) s_part[0] = b, s_part[1] = me - x, s_part[2] = (int)(at.a >> 32);
      at.a += c.a, at.b += c.b;
    }
  }
  __syncthreads();
  p.size = __builtin_amdgcn_readfirstlane(p.size);
  p.seq = __builtin_amdgcn_readfirstlane(s_part[0]);
  if (p.seq < 0) return p;
  const int i = __builtin_amdgcn_readfirstlane(s_part[1]);
  kind = __builtin_amdgcn_readfirstlane(kind);
  p.tk = tokens_of(a.cu, p.seq, a.T, a.most);
  p.pos = uniform_load(a.pos + p.seq);
  const Demand d = demand_of(a, p.tk.nt, vis_of(p.pos, p.tk.nt, cap), rows);
  const int whole = d.span / p.size;
  p.parts = (d.span + p.size - 1) / p.size;
  place_of(a, i, kind == 0 ? whole : 1, (p.tk.nt * a.group + rows - 1) / rows, p.unit, p.k);
  if (kind) p.k = whole;
  p.place = __builtin_amdgcn_readfirstlane(s_part[2]) + p.unit * p.parts + p.k;
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
  const int group = a.group;
  const Tokens tk = pt.tk;
  const Vis vis = vis_of(pt.pos, tk.nt, a.pg.max_pages << a.pg.shift);
  const int rows = tk.nt * group, groups = (rows + kRows - 1) / kRows, kh = pt.unit / groups, first = (pt.unit - kh * groups) * kRows;
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const int t0 = pt.k * pt.size, t1 = t0 + pt.size < tiles ? t0 + pt.size : tiles;
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
  const uint64_t tree = gr >= 0 ? tree_of(a, tk, (first + mine) / group) : 0ull;
  for (TileAt at = walk.next(t1); at.j0 >= 0; at = walk.next(t1)) {
    if constexpr (TYPE == Q27H_KV_Q8_Q4) tail_tile<QRows4>(st, at.k, at.v, q, sh.w[w], vis, tree, at.j0);
    else tail_tile(st, at.k, at.v, q, sh.w[w], vis, tree, at.j0);
  }
  const bool whole = pt.parts == 1;
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

// ---------------------------------------------------------------- more than 32 query rows over f16
// A row tile for each wave, the cache rows shared through LDS as in attn_tree (attn_shared.h): a tile is worked on while the
// next one or two are on their way through registers. 16 sequences of 32768 rows, 6 and 12 tokens: 390 and 493 us, where
// units of 32 query rows that each read the rows take 923 and 1409 (the bytes alone take 311 at a large read's rate);
// 8 sequences, 64 tokens: 898 for 2462, of which the products with two terms need 701. One sequence of
// 2000 rows, whose workgroups have four tiles one after the other here: 19.5 and 25.4 for 15.9 and 18.5.
template <int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) attn_paged_shared_kernel(PagedArgs a) {
  constexpr size_t kTiles = sizeof(SharedTile) * 2, kImages = sizeof(QTile) * WAVES;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[kTiles > kImages ? kTiles : kImages];  // the queries' image, then the tiles
  __shared__ int s_odd[2];
  QTile* im = (QTile*)s_mem;
  SharedTile* buf = (SharedTile*)s_mem;
  const Part pt = part_of<WAVES * 64>(a, a.rows);
  if (pt.seq < 0) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.group;
  const Tokens tk = pt.tk;
  const Vis vis = vis_of(pt.pos, tk.nt, a.pg.max_pages << a.pg.shift);
  const int rows = tk.nt * group, groups = (rows + a.rows - 1) / a.rows, kh = pt.unit / groups, first = (pt.unit - kh * groups) * a.rows;
  const int tiles = (vis.end + kTileKeys - 1) / kTileKeys;
  const int t0 = pt.k * pt.size, t1 = t0 + pt.size < tiles ? t0 + pt.size : tiles;
  auto row = [&](int r) {  // the global row of the unit's query row r, or -1
    const int at = first + r;
    return r < a.rows && at < rows ? (tk.t0 + at / group) * a.nqh + kh * group + at % group : -1;
  };
  PageWalk<Q27H_KV_F16, 1> walk(a.pg, pt.seq, kh, t0, t1);
  auto left_of = [&](const TileAt& at) { return vis.end - at.j0 < kTileKeys ? vis.end - at.j0 : kTileKeys; };
  auto part_of_it = [&](const TileAt& at) { return at.j0 + kTileKeys > vis.n; };
  auto ask = [&](Staged<false, WAVES>& n, TileAt& at) __attribute__((always_inline)) {
    at = walk.next(t1);
    if (at.j0 >= 0) request<false, WAVES, true, true>(n, at.k, at.v, at.j0, left_of(at));
  };
  // 8 waves have two tiles on their way; 4 carry twice as much each: one
  constexpr bool kTwo = WAVES == 8;
  Staged<false, WAVES> even, odd;
  TileAt at, te, to;
  ask(even, at);
  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  load_queries<false, WAVES, WAVES>(im, a.scale * kLog2e, [&](int r) {
    const int gr = row(r);
    return gr < 0 ? nullptr : a.qn + (size_t)gr * kHD;
  });
  __syncthreads();
  QRegs q;
  take_queries(q, im[w]);
  Rows st;
  rows_init<false>(st, im[w]);
  const int mine = w * 16 + (threadIdx.x & 15), gr = row(mine);
  const uint64_t tree[1] = {gr >= 0 ? tree_of(a, tk, (first + mine) / group) : 0ull};
  const bool active = w * 16 < a.rows && first + w * 16 < rows;
  __syncthreads();
  int b = 0;
  auto put = [&](Staged<false, WAVES>& n, const TileAt& x, int b) __attribute__((always_inline)) {
    if (x.j0 >= 0) stage<false, WAVES, true, true>(n, buf[b], part_of_it(x), left_of(x), &s_odd[b]);
  };
  put(even, at, 0);
  ask(even, te);
  if (kTwo) ask(odd, to);
  __syncthreads();
  // `at` is in LDS, `x` the next one in `next`, which is then given the one behind those on their way. Two loops, as in
  // attn_tree; the first takes an even number of tiles.
  auto step = [&](auto hidden, Staged<false, WAVES>& next, TileAt& x) __attribute__((always_inline)) {
    constexpr bool kPart = decltype(hidden)::value;
    if (active) {
      f4 s[1][2];
      __builtin_amdgcn_s_setprio(1);
      scores<false>(buf[b], &q, s);
      if (kPart) hide<1, kHidden>(s, vis, tree, at.j0);
      weights<false, kPart>(st, s[0]);
      accumulate<false, kPart>(st, s[0], buf[b]);
      if (kPart && s_odd[b]) add_odd(st, s[0], at.v, at.j0, left_of(at));
    }
    __builtin_amdgcn_s_setprio(0);
    b ^= 1;
    put(next, x, b);
    at = x;
    ask(next, x);
    __syncthreads();
  };
  auto full = [&](const TileAt& x) { return x.j0 >= 0 && !part_of_it(x); };
  if constexpr (kTwo) {
    while (full(at) && full(te)) {
      step(std::false_type(), even, te);
      step(std::false_type(), odd, to);
    }
    while (at.j0 >= 0) {
      step(std::true_type(), even, te);
      if (at.j0 < 0) break;
      step(std::true_type(), odd, to);
    }
  } else {
    while (full(at)) step(std::false_type(), even, te);
    while (at.j0 >= 0) step(std::true_type(), even, te);
  }
  if (!active) return;
  st.l += lane_xor<16>(st.l);
  st.l += lane_xor32(st.l);
  if (gr < 0) return;
  const bool lead = (threadIdx.x & 63) < 16;
  float* dst;
  if (pt.parts == 1) {
    const float inv = st.l == 0.0f ? 0.0f : 1.0f / st.l;
#pragma unroll
    for (int i = 0; i < 16; i++) st.o[i] *= inv;
    dst = a.o + (size_t)gr * kHD;
    if (a.lse && lead) a.lse[gr] = st.l == 0.0f ? -__builtin_huge_valf() : (st.m + __builtin_amdgcn_logf(st.l)) * kLn2;
  } else {
    const size_t place = (size_t)pt.place * a.rows + mine;
    dst = a.part + place * kHD;
    if (lead) *(float2*)(a.ml + place * 2) = make_float2(st.m, st.l);
  }
  store_rows<true>(st, dst);
}

// ---------------------------------------------------------------- more than 16 query rows over codes
// A workgroup's four waves share each tile of 128 cache rows. For the scores a wave takes 32 of the rows, for the outputs 64
// of the 256 dims, both for all of the unit's query rows: no code is turned to a half twice, whatever the number of
// query rows, and a wave holds a quarter of the outputs. The weights and the V rows go from the one to the other through LDS.
// 48 sequences of 500 to 32768 rows with 4 tokens each, V in 4 bits: 178 us of its own, where waves with tiles of their own
// take 270. What bounds it is no one thing: it runs at 3.5 TB/s, its vector instructions fill half the cycles; without the
// weights' scaling it would be 9% faster, without the second f16 terms 16%, without its loads 12%.
//
// One reference E for each query row, the same in all waves: a row's product of weight and V scale is 2^(s - E) f d, f the
// power of two above the V row's scales and d what is left of each (at most 1). E moves when a row's s + log2 f passes
// E + 15, to 12 below it, so that what enters the product as two f16 terms is in their range, as in attn_core.h; the sum of
// the weights is kept in units of 2^E as well. Rows whose V scales are all 0 count as f = 2^-25.
constexpr int QT = 2;  // row tiles of a unit
struct WideLds {
  union {
    QTile q[QT];
    alignas(16) uint8_t codes[kWaves][kCodes];  // a wave's rows of K, then of V, as WaveLds has them
  };
  alignas(16) uint32_t lo[QT][8][64][4];          // the queries' second terms
  alignas(16) uint32_t p[QT][kWaves][2][64][4];  // weights as operands: two terms of 32 rows
  alignas(16) uint8_t ks[kWaves][kScales], vs[kWaves][kScales];
  alignas(16) int lf[kWaves][kTileKeys];  // the logarithms of f
  float mx[kWaves][QT][16];               // of the scores; in the end the sums of the weights
  uint64_t tree[QT][16];                  // which of the new tokens a query row sees
};

// A wave's rows on their way. Rows behind the last one that exists are read from it, those of a group without any from row 0
// of a page; their scales are taken as 0.
template <int TYPE>
struct WideRegs {
  u4 k[8], v[TYPE == Q27H_KV_Q8_Q4 ? 4 : 8];
  u2 ks, vs;
};
struct WideTile {
  const uint8_t *k, *v, *ks, *vs;
  int left;  // of the wave's 32 rows, those that exist
};
template <int TYPE>
__device__ __forceinline__ void wide_load_k(WideRegs<TYPE>& r, const WideTile& t, int l) {
  const int last = t.left > 0 ? t.left - 1 : 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int row = 4 * i + (l >> 4);
    r.k[i] = *(const u4*)(t.k + (unsigned)((row < last ? row : last) * kHD + 16 * (l & 15)));
  }
  const unsigned at = ((l >> 1) < last ? (l >> 1) : last) * 16 + 8 * (l & 1);
  r.ks = *(const u2*)(t.ks + at);
  r.vs = *(const u2*)(t.vs + at);
}
template <int TYPE>
__device__ __forceinline__ void wide_load_v(WideRegs<TYPE>& r, const WideTile& t, int l) {
  const int last = t.left > 0 ? t.left - 1 : 0;
  constexpr bool k4 = TYPE == Q27H_KV_Q8_Q4;
#pragma unroll
  for (int i = 0; i < (k4 ? 4 : 8); i++) {
    const int row = k4 ? 8 * i + (l >> 3) : 4 * i + (l >> 4);
    r.v[i] = *(const u4*)(t.v + (unsigned)((row < last ? row : last) * (k4 ? kHD / 2 : kHD) + 16 * (l & (k4 ? 7 : 15))));
  }
}
template <int TYPE>
__device__ __forceinline__ void wide_stage_k(const WideRegs<TYPE>& r, uint8_t* codes, int l) {
#pragma unroll
  for (int i = 0; i < 8; i++) *(u4*)(codes + (i >= 4 ? kUpper - 16 * kRow : 0) + 4 * i * kRow + (l >> 4) * kRow + 16 * (l & 15)) = r.k[i];
}
template <int TYPE>
__device__ __forceinline__ void wide_stage_v(const WideRegs<TYPE>& r, uint8_t* codes, int l) {
  if constexpr (TYPE == Q27H_KV_Q8_Q4) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      u4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; e++) lo[e] = r.v[i][e] & 0x0f0f0f0fu, hi[e] = r.v[i][e] >> 4 & 0x0f0f0f0fu;
      uint8_t* p = codes + (i >= 2 ? kUpper - 16 * kRow : 0) + 8 * i * kRow + (l >> 3) * kRow + 32 * (l & 7);
      *(u4*)p = lo;
      *(u4*)(p + 16) = hi;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) *(u4*)(codes + (i >= 4 ? kUpper - 16 * kRow : 0) + 4 * i * kRow + (l >> 4) * kRow + 16 * (l & 15)) = r.v[i];
  }
}

// Scores of the wave's 32 rows for the two row tiles, as attn_core.h's. A step is (block, row tile): its four matrix
// instructions with the scaling of the step before and a share of the next block's codes beside them.
__device__ __forceinline__ void wide_scores(const uint8_t* codes, const uint8_t* ks, const h8 (&hi)[QT][8],
                                            const uint32_t (*lo)[8][64][4], f4 (&s)[QT][2]) {
  const int l = threadIdx.x & 63;
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < QT; q++) s[q][0] = s[q][1] = zero;
  h8 ql[2], x[2][2];
  u2 sc[2][2], k[2];
  f4 c[2][2];  // of this step and the one before
  const uint8_t* row = codes + (l & 15) * kRow + 8 * (l >> 4);
  auto ask_q = [&](int i) { ql[i & 1] = *(const h8*)lo[i % QT][i / QT][l]; };
  auto ask_s = [&](int b) {
#pragma unroll
    for (int u = 0; u < 2; u++) sc[b & 1][u] = scales_of(ks, b, u);
  };
  auto ask_k = [&](int b, int u) { k[u] = *(const u2*)(row + kUpper * u + 32 * b); };
  auto turn = [&](int b, int u) { x[b & 1][u] = codes8(k[u].x, k[u].y); };
  auto scale = [&](int i) {
    const int b = i / QT, q = i % QT;
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int e = 0; e < 4; e++) s[q][u][e] = __builtin_fmaf(half_of(sc[b & 1][u][e & 1], e >> 1), c[i & 1][u][e], s[q][u][e]);
      asm("" : "+v"(s[q][u]));
    }
  };
  ask_k(0, 0);
  ask_k(0, 1);
  ask_q(0);
  ask_s(0);
  turn(0, 0);
  turn(0, 1);
  ask_k(1, 0);
  ask_k(1, 1);
#pragma unroll
  for (int i = 0; i < 8 * QT; i++) {
    const int b = i / QT, q = i % QT;
    __builtin_amdgcn_sched_barrier(0);
    if (i + 1 < 8 * QT) ask_q(i + 1);
#pragma unroll
    for (int u = 0; u < 2; u++) c[i & 1][u] = mfma16(x[b & 1][u], ql[i & 1], zero);
#pragma unroll
    for (int u = 0; u < 2; u++) c[i & 1][u] = mfma16(x[b & 1][u], hi[q][b], c[i & 1][u]);
    if (i) scale(i - 1);
    if (q == QT - 1 && b < 7) ask_s(b + 1);
    if (b < 7) {  // a row tile's step: one half of the next block's rows
      turn(b + 1, q);
      if (b < 6) ask_k(b + 2, q);
    }
  }
  scale(8 * QT - 1);
}

template <int TYPE>
__global__ void __launch_bounds__(kWaves * 64, 2) attn_paged_wide_kernel(PagedArgs a) {
  constexpr int kRows = 16 * QT, kV = TYPE == Q27H_KV_Q8_Q4 ? kHD / 2 : kHD, kBias = TYPE == Q27H_KV_Q8_Q4 ? 8 : 128;
  __shared__ WideLds sh;
  const Part pt = part_of<kWaves * 64, true>(a, kRows);
  if (pt.seq < 0) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 15;
  const int group = a.group;
  const Tokens tk = pt.tk;
  const Vis vis = vis_of(pt.pos, tk.nt, a.pg.max_pages << a.pg.shift);
  const int rows = tk.nt * group, groups = (rows + kRows - 1) / kRows, kh = pt.unit / groups, first = (pt.unit - kh * groups) * kRows;
  const int tiles = a.pg.n_pages ? (vis.end + kTileKeys - 1) / kTileKeys : 0;  // without a page there is nothing to read
  const int t0 = pt.k * pt.size, t1 = t0 + pt.size < tiles ? t0 + pt.size : tiles;
  auto row = [&](int r) {  // the global row (token * nqh + head) of the unit's query row r, or -1
    int by = group;
    asm volatile("" : "+s"(by));  // what the division takes is formed where it is used, see `lane`
    r += first;
    return r < rows ? (tk.t0 + r / by) * a.nqh + kh * group + r % by : -1;
  };
  const int* table = a.pg.table + (size_t)pt.seq * a.pg.max_pages;
  const int prow = 1 << a.pg.shift;
  int page[kWaves];  // of the tile's four groups of 32 rows
  auto ask_pages = [&](int t) {
#pragma unroll
    for (int k = 0; k < kWaves; k++) page[k] = t + k < t1 ? uniform_load(table + ((t + k) >> (a.pg.shift - 5))) : -1;
  };
  WideTile wt;
  bool whole;  // every row of the tile is seen by every query
  auto place = [&](int t) {
    whole = (t + kWaves) * kTileKeys <= vis.n && t + kWaves <= t1;
    int mine = page[0];
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      whole = whole && (unsigned)page[k] < (unsigned)a.pg.n_pages;
      mine = k == w ? page[k] : mine;
    }
    const int j0 = (t + w) * kTileKeys;
    const bool is = (unsigned)mine < (unsigned)a.pg.n_pages;
    wt.left = is ? (vis.end - j0 < kTileKeys ? vis.end - j0 : kTileKeys) : 0;
    const size_t at = (size_t)kh * prow + (j0 & (prow - 1)), p = is ? mine : 0;
    wt.k = a.pg.k + p * a.pg.kb + at * kHD;
    wt.v = a.pg.v + p * a.pg.vb + at * kV;
    wt.ks = a.pg.k + p * a.pg.kb + (size_t)a.pg.nkvh * prow * kHD + at * 16;
    wt.vs = a.pg.v + p * a.pg.vb + (size_t)a.pg.nkvh * prow * kV + at * 16;
  };
  WideRegs<TYPE> r;
  if (t0 < t1) {
    ask_pages(t0);
    place(t0);
    wide_load_k(r, wt, l);
    wide_load_v(r, wt, l);
    ask_pages(t0 + kWaves);
  }
  load_queries<true, kWaves, QT>(sh.q, a.scale * kLog2e, [&](int r) {
    const int gr = row(r);
    return gr < 0 ? nullptr : a.qn + (size_t)gr * kHD;
  });
  if (threadIdx.x < kRows) {
    const int at = first + (int)threadIdx.x;
    sh.tree[threadIdx.x >> 4][threadIdx.x & 15] = at < rows ? tree_of(a, tk, at / group) : 0ull;
  }
  __syncthreads();
  h8 hi[QT][8];
  float c[QT], e[QT], sum[QT];
  f4 o[QT][4];
#pragma unroll
  for (int q = 0; q < QT; q++) {
    c[q] = sh.q[q].c[n];
    e[q] = -3.0e38f, sum[q] = 0.0f;
#pragma unroll
    for (int b = 0; b < 8; b++) hi[q][b] = *(const h8*)sh.q[q].v[0][b][l];
#pragma unroll
    for (int b = 0; b < 8; b += kWaves) *(h8*)sh.lo[q][b + w][l] = *(const h8*)sh.q[q].v[1][b + w][l];
#pragma unroll
    for (int i = 0; i < 4; i++) o[q][i] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
  }
  __syncthreads();

  int t = t0, left = 0;  // of the tile in work, where wt is the next one's
  auto step = [&](auto hidden) __attribute__((always_inline)) {
    constexpr bool kPart = decltype(hidden)::value;
    f4 s[QT][2];
    int lane = l;
    asm volatile("" : "+v"(lane));  // addresses are formed for each tile: kept over the loop they would spill
    const int n = lane & 15, g = lane >> 4;
    left = wt.left;
    wide_stage_k(r, sh.codes[w], lane);
    if (kPart && (lane >> 1) >= left) r.ks = r.vs = (u2){0u, 0u};
    put_scales(r.ks, sh.ks[w]);
    // V's scales: f, and what is left of them
    u2 vs;
    {
      float x[4], m = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[i] = half_of(i < 2 ? r.vs.x : r.vs.y, i & 1);
        m = __builtin_fabsf(x[i]) < 65536.0f ? __builtin_fmaxf(m, __builtin_fabsf(x[i])) : m;
      }
      m = __builtin_fmaxf(m, lane_xor<1>(m));
      const int ex = (int)(__builtin_bit_cast(uint32_t, m) >> 23) - 126;  // 2^(ex - 1) <= m < 2^ex
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = m > 0.0f ? __builtin_amdgcn_ldexpf(x[i], -ex) : x[i];
      vs = (u2){pk_rtz(x[0], x[1]), pk_rtz(x[2], x[3])};
      if (!(lane & 1)) sh.lf[w][lane >> 1] = m > 0.0f ? ex : -25;
    }
    const int j0 = (t + w) * kTileKeys;
    t += kWaves;
    if (t < t1) {
      place(t);
      wide_load_k(r, wt, lane);
      ask_pages(t + kWaves);
    }
    loads_issued();
    __builtin_amdgcn_s_setprio(1);  // products before the other workgroup's staging (128 sequences of 4096 rows: 269 -> 263 us)
    wide_scores(sh.codes[w], sh.ks[w], hi, sh.lo, s);
    __builtin_amdgcn_s_setprio(0);
    if (kPart) {
      Vis mine = vis;
      uint64_t tree[QT];
#pragma unroll
      for (int q = 0; q < QT; q++) tree[q] = sh.tree[q][n];
      if (left <= 0) mine.n = mine.end = 0;
      hide<QT, kHidden>(s, mine, tree, j0);
    }
    typedef int i4 __attribute__((ext_vector_type(4)));
    const i4 lf[2] = {*(const i4*)&sh.lf[w][4 * g], *(const i4*)&sh.lf[w][16 + 4 * g]};
#pragma unroll
    for (int q = 0; q < QT; q++) {
      float mx = -3.0e38f;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = __builtin_fmaxf(mx, __builtin_fmaf(s[q][u][i], c[q], (float)lf[u][i]));
      mx = __builtin_fmaxf(mx, lane_xor<16>(mx));
      mx = __builtin_fmaxf(mx, lane_xor32(mx));
      if (g == 0) sh.mx[w][q][n] = mx;
    }
    wide_stage_v(r, sh.codes[w], lane);  // K's rows are read
    if (t < t1) wide_load_v(r, wt, lane);
    loads_issued();
    put_scales(vs, sh.vs[w]);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < QT; q++) {
      const float mx = __builtin_fmaxf(__builtin_fmaxf(sh.mx[0][q][n], sh.mx[1][q][n]), __builtin_fmaxf(sh.mx[2][q][n], sh.mx[3][q][n]));
      if (__any(mx - e[q] > 15.0f)) {
        const float to = mx - e[q] > 15.0f ? mx - 12.0f : e[q];  // by its own row alone
        const float x = __builtin_amdgcn_exp2f(e[q] - to);
        e[q] = to;
        sum[q] *= x;
#pragma unroll
        for (int i = 0; i < 4; i++) o[q][i] *= x;
      }
      f4 p[2];
      float add = 0.0f;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float x = s[q][u][i], y = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c[q], -e[q]));
          const float z = kPart && __builtin_bit_cast(uint32_t, x) == kHidden ? -0.0f : y;
          add += z;
          p[u][i] = __builtin_amdgcn_ldexpf(z, lf[u][i]);
        }
      sum[q] += add;
      u4 ph, pl;
#pragma unroll
      for (int k = 0; k < 4; k++) {  // pairs of rows (0, 2), (1, 3), as codes8 orders them
        const float w0 = p[k >> 1][k & 1], w1 = p[k >> 1][(k & 1) + 2];
        ph[k] = pk_rtz(w0, w1);
        pl[k] = pk_rtz(minus_half(w0, ph[k], 0), minus_half(w1, ph[k], 1));
      }
      *(u4*)sh.p[q][w][0][lane] = ph;
      *(u4*)sh.p[q][w][1][lane] = pl;
    }
    __syncthreads();
    // O += P V: the wave's two blocks of 32 dims; the transposing read as in attn_core.h. A step per (group, block): its
    // products, and the next step's weights and codes beside them
    const uint8_t* vbase = sh.codes[0] + ((n >> 1) >= 4 ? kUpper + (4 * g + (n >> 1) - 4) * kRow : (4 * g + (n >> 1)) * kRow) + 8 * (n & 1) + 64 * w;
    u4 ph[QT], pl[QT], wh[2][QT], wl[2][QT];
    typedef int v2i __attribute__((ext_vector_type(2)));
    v2i x[2];
    u2 d[2];
    h8 v[2][2];
    auto ask_p = [&](int k) {
#pragma unroll
      for (int q = 0; q < QT; q++) ph[q] = *(const u4*)sh.p[q][k][0][lane], pl[q] = *(const u4*)sh.p[q][k][1][lane];
    };
    auto ask = [&](int i) {
      const int k = i >> 1, b = i & 1;
#pragma unroll
      for (int u = 0; u < 2; u++) d[u] = scales_of(sh.vs[k], 2 * w + b, u);
#pragma unroll
      for (int h = 0; h < 2; h++)
        x[h] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(vbase + kCodes * k + 32 * b + 16 * h));
    };
    auto turn = [&](int i) {
#pragma unroll
      for (int q = 0; q < QT; q++) weigh<kPart>(ph[q], pl[q], d, wh[i & 1][q], wl[i & 1][q]);
#pragma unroll
      for (int h = 0; h < 2; h++) v[i & 1][h] = codes8<kBias>((uint32_t)x[h].x, (uint32_t)x[h].y);
    };
    __builtin_amdgcn_s_setprio(1);
    ask_p(0);
    ask(0);
    turn(0);
    ask(1);
#pragma unroll
    for (int i = 0; i < 2 * kWaves; i++) {
      const int b = i & 1;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < QT; q++)
#pragma unroll
        for (int h = 0; h < 2; h++) o[q][2 * b + h] = mfma16(v[b][h], __builtin_bit_cast(h8, wl[b][q]), o[q][2 * b + h]);
#pragma unroll
      for (int q = 0; q < QT; q++)
#pragma unroll
        for (int h = 0; h < 2; h++) o[q][2 * b + h] = mfma16(v[b][h], __builtin_bit_cast(h8, wh[b][q]), o[q][2 * b + h]);
      if (i + 1 < 2 * kWaves) {
        turn(i + 1);
        if (i + 2 < 2 * kWaves) {
          if (!b) ask_p((i + 2) >> 1);
          ask(i + 2);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();  // V's rows are read: K's take their place
  };
  while (t < t1) {
    while (t < t1 && whole) step(std::false_type());
    if (t < t1) step(std::true_type());
  }
  int end = l;
  asm volatile("" : "+v"(end));
  const int n1 = end & 15, g1 = end >> 4;
#pragma unroll
  for (int q = 0; q < QT; q++) {
    sum[q] += lane_xor<16>(sum[q]);
    sum[q] += lane_xor32(sum[q]);
    if (g1 == 0) sh.mx[w][q][n1] = sum[q];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < QT; q++) {
    const int gr = row(16 * q + n1);
    if (gr < 0) continue;
    const float total = (sh.mx[0][q][n1] + sh.mx[1][q][n1]) + (sh.mx[2][q][n1] + sh.mx[3][q][n1]);
    const bool lead = w == 0 && g1 == 0;
    float x = 512.0f;  // codes8's 2^-9
    float* dst;
    if (pt.parts == 1) {
      x = total == 0.0f ? 0.0f : x / total;
      dst = a.o + (size_t)gr * kHD;
      if (a.lse && lead) a.lse[gr] = total == 0.0f ? -__builtin_huge_valf() : (e[q] + __builtin_amdgcn_logf(total)) * kLn2;
    } else {
      const size_t at = (size_t)pt.place * kRows + 16 * q + n1;
      dst = a.part + at * kHD;
      if (lead) *(float2*)(a.ml + at * 2) = make_float2(e[q], total);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) *(f4*)(dst + 64 * w + 16 * i + 4 * g1) = o[q][i] * x;
  }
}

// ---------------------------------------------------------------- the join
// A query row whose unit was cut: its first part in the workspace, and how many.
struct Cut {
  int n;         // 0 or 1: there is nothing to join
  size_t place;  // part k: k * rows rows on
  size_t row;    // its place in the results
};
// Wave w's share of a row, every WAVES-th part in order: a lane four dims; m and sum are the whole row's.
template <int WAVES>
__device__ __forceinline__ f4 join_of(const PagedArgs& a, const Cut& c, int rows, int w, float& m, float& sum) {
  const int l = threadIdx.x & 63, n = c.n;
  const f4* part = (const f4*)(a.part + c.place * kHD) + l;
  const float2* ml = (const float2*)a.ml + c.place;
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
  const float2 v = l < n ? ml[l * rows] : make_float2(-3.0e38f, 0.0f);
  m = v.x;
  for (int k = l + 64; k < n; k += 64) m = __builtin_fmaxf(m, ml[k * rows].x);
  m = all(m, [](float p, float q) { return __builtin_fmaxf(p, q); });
  const float f = __builtin_amdgcn_exp2f(v.x - m);
  sum = v.y * f;
  for (int k = l + 64; k < n; k += 64) sum += ml[k * rows].y * __builtin_amdgcn_exp2f(ml[k * rows].x - m);
  sum = all(sum, [](float p, float q) { return p + q; });
  auto factor = [&](int k) {  // of part k, the same in the whole wave
    return k < 64 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), k))
                  : __builtin_amdgcn_exp2f(ml[k * rows].x - m);
  };
  f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kBatch; k++)
    if (w + WAVES * k < n) o += x[k] * factor(w + WAVES * k);
  for (int k0 = w + WAVES * kBatch; k0 < n; k0 += WAVES * kBatch) {
#pragma unroll
    for (int k = 0; k < kBatch; k++)
      if (k0 + WAVES * k < n) x[k] = part[(size_t)(k0 + WAVES * k) * rows * 64];
#pragma unroll
    for (int k = 0; k < kBatch; k++)
      if (k0 + WAVES * k < n) o += x[k] * factor(k0 + WAVES * k);
  }
  return o;
}
// A workgroup joins a row: sequence blockIdx.x, token y, query head z. 16 waves where there are few rows, which may have many
// parts; 4 where there are many, of which the first joins a few parts alone, so that the others' places are free for other
// rows (200 sequences of 300 to 4096 rows, 4 tokens: 17.5 -> 11.8 us; 48 of 500 to 32768: 12.7 -> 11.6).
template <int WAVES, int ROWS>  // query rows of a unit; 0: a.rows
__global__ void __launch_bounds__(WAVES * 64, 8) attn_paged_join_kernel(PagedArgs a) {
  __shared__ f4 s_o[WAVES][64];
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x, t = blockIdx.y, h = blockIdx.z;
  const int start = uniform_load(a.starts + 2 * b), n = uniform_load(a.starts + 2 * b + 1);
  const Tokens tk = tokens_of(a.cu, b, a.T, a.most);
  if (t >= tk.nt || n <= 1) return;
  const int rows = ROWS ? ROWS : a.rows;
  const int group = a.group, kh = h / group, r = t * group + h - kh * group, groups = (tk.nt * group + rows - 1) / rows;
  const Cut c = {n, ((size_t)start + (size_t)(kh * groups + r / rows) * n) * rows + r % rows, (size_t)(tk.t0 + t) * a.nqh + h};
  const bool alone = WAVES == 4 && n <= 12;
  if (alone && w) return;
  float m, sum;
  f4 o;
  if (alone) {
    o = join_of<1>(a, c, rows, 0, m, sum);
  } else {
    o = join_of<WAVES>(a, c, rows, w, m, sum);
    s_o[w][l] = o;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < WAVES; k++) o += s_o[k][l];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  *((f4*)(a.o + c.row * kHD) + l) = o * inv;
  if (a.lse && l == 0) a.lse[c.row] = sum == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

struct Layout {
  int rows, threads, slots, least, grid;
  size_t places, bytes;
};
// Units of 16 query rows where a kv head has no more, of 32 otherwise; over f16, where a unit's cache rows would be read again
// for each 32 query rows, of up to 128, in equal groups. Two workgroups of four waves run on a compute unit, or one of eight.
Layout layout_of(int n_seqs, int max_tokens, int nqh, int nkvh, int type) {
  Layout y;
  const int tiles = (max_tokens * (nqh / nkvh) + 15) / 16;
  y.rows = tiles == 1 ? 16 : 32;
  y.threads = y.rows == 32 && type == Q27H_KV_F16 ? 512 : 256;
  if (type == Q27H_KV_F16 && tiles > 2) {
    const int groups = (tiles + 7) / 8;
    y.rows = 16 * ((tiles + groups - 1) / groups);
    y.threads = y.rows <= 64 ? 256 : 512;
  }
  const int units = n_seqs * nkvh * ((16 * tiles + y.rows - 1) / y.rows);
  y.slots = 2 * kCUs * 256 / y.threads;
  // over codes, more than 16 query rows are bound by arithmetic: with units of many lengths, parts of half the size leave the
  // last workgroups less of it (33 sequences of 64 to 131072 rows, 4 tokens: 243 -> 236 us; 64 of 300 to 8000, 8 tokens:
  // 150 -> 139; equal ones, 100 of 4096: 210 -> 212), but none under 32 tiles, where its start costs more (48 of 200 to 8000:
  // 65, and 71 with all parts halved). One sequence is cut evenly, and a second round of workgroups costs it (150000 rows:
  // 82 -> 91 us)
  y.least = y.rows == 32 && type != Q27H_KV_F16 && units >= kCUs / 2 ? 32 : 0;
  // beside the whole parts, of which there are `most` at the most, each unit leaves one; a unit that is cut has less than
  // twice its share of parts
  const int most = y.least ? 2 * y.slots : y.slots;
  y.grid = units + most;
  y.places = (size_t)(y.grid < 2 * most ? y.grid : 2 * most) * y.rows;
  y.bytes = y.places * (kHD + 2) * sizeof(float) + (size_t)n_seqs * 2 * sizeof(int);
  return y;
}
// Why a call of these sizes is refused, or null.
const char* refusal(const q27h_kv_pages* kv, int T, int max_tokens, int nqh) {
  if (T < 0 || max_tokens < 1 || max_tokens > kMostTokens || nqh <= 0 || nqh > 4096 || nqh % kv->nkvh)
    return "attn_paged: bad shape (1 to 64 tokens a sequence, at most 4096 query heads)";
  // the tiles of all units are counted in 31 bits
  const int group = nqh / kv->nkvh;
  const long long tiles = ((long long)kv->max_pages * kv->page_rows / kTileKeys + kWaves) / kWaves * kWaves;
  if ((double)kv->n_seqs * kv->nkvh * ((max_tokens * group + 15) / 16) * (double)tiles > 2.0e9) return "attn_paged: too many rows in all";
  if ((long long)kv->n_seqs * max_tokens * nqh > 0x7fffffffLL / 256 || (long long)T * nqh > 0x7fffffffLL / 256)
    return "attn_paged: too many query rows";
  return nullptr;
}

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_attn_paged_ws_bytes(const q27h_kv_pages* kv, int T, int max_tokens, int nqh) {
  if (check_pages(kv, "attn_paged") != Q27H_OK || T <= 0 || refusal(kv, T, max_tokens, nqh)) return 0;
  return layout_of(kv->n_seqs, max_tokens, nqh, kv->nkvh, kv->type).bytes;
}

extern "C" int q27h_attn_paged(const float* qn, const q27h_kv_pages* kv, const int* pos, const int* cu, int T, int max_tokens,
                               float scale, int nqh, float* o, float* lse, void* ws, size_t ws_bytes, q27h_stream_t s,
                               const uint64_t* tree) {
  if (const int bad = check_pages(kv, "attn_paged")) return bad;
  if (const char* why = refusal(kv, T, max_tokens, nqh)) return fail(Q27H_ERR_SHAPE, why);
  if (!cu && T != kv->n_seqs) return fail(Q27H_ERR_SHAPE, "attn_paged: without cu there is one token for each sequence");
  if (T == 0 || kv->n_seqs == 0) return Q27H_OK;
  if (!qn || !pos || !o) return fail(Q27H_ERR_ARG, "attn_paged: null pointer");
  if (!aligned16(qn) || !aligned16(o) || !aligned16(ws)) return fail(Q27H_ERR_ARG, "attn_paged: tensors need 16-byte alignment");
  if (!aligned8(tree) || !aligned4(pos) || !aligned4(cu) || !aligned4(lse))
    return fail(Q27H_ERR_ARG, "attn_paged: tree needs 8-byte alignment, pos, cu and lse 4-byte");
  const Layout y = layout_of(kv->n_seqs, max_tokens, nqh, kv->nkvh, kv->type);
  if (ws_bytes < y.bytes || !ws) return fail(Q27H_ERR_ARG, "attn_paged: workspace too small");
  const Pages pg = pages_of(kv);
  const size_t qb = (size_t)T * nqh * kHD * 4, B = (size_t)kv->n_seqs;
  if (outputs_overlap({{o, qb}, {lse, (size_t)T * nqh * 4}, {ws, y.bytes}},
                      {{qn, qb}, {pg.k, pg.kb * pg.n_pages}, {pg.v, pg.vb * pg.n_pages}, {pg.table, B * pg.max_pages * 4},
                       {pos, B * 4}, {cu, (B + 1) * 4}, {tree, (size_t)T * 8}}))
    return fail(Q27H_ERR_ARG, "attn_paged: o, lse or ws overlaps another argument");
  PagedArgs a = {};
  a.pg = pg, a.qn = qn, a.pos = pos, a.cu = cu, a.tree = tree, a.o = o, a.lse = lse, a.T = T, a.most = max_tokens, a.nqh = nqh, a.scale = scale;
  a.slots = y.slots, a.least = y.least, a.rows = y.rows, a.group = nqh / kv->nkvh;
  a.part = (float*)ws, a.ml = a.part + y.places * kHD, a.starts = (int*)(a.ml + y.places * 2);
  const dim3 grid((unsigned)y.grid), block((unsigned)y.threads);
  auto launch = [&](auto one, auto two) { hipLaunchKernelGGL((y.rows == 16 ? one : two), grid, block, 0, stream_of(s), a); };
  auto shared = y.threads == 256 ? attn_paged_shared_kernel<4> : attn_paged_shared_kernel<8>;
  if (y.rows > 32) hipLaunchKernelGGL(shared, grid, block, 0, stream_of(s), a);
  else if (kv->type == Q27H_KV_F16) launch(attn_paged_kernel<Q27H_KV_F16, 1>, attn_paged_kernel<Q27H_KV_F16, 2>);
  else if (kv->type == Q27H_KV_Q8) launch(attn_paged_kernel<Q27H_KV_Q8, 1>, attn_paged_wide_kernel<Q27H_KV_Q8>);
  else launch(attn_paged_kernel<Q27H_KV_Q8_Q4, 1>, attn_paged_wide_kernel<Q27H_KV_Q8_Q4>);
  const int qrows = kv->n_seqs * max_tokens * nqh;
  const dim3 all((unsigned)kv->n_seqs, (unsigned)max_tokens, (unsigned)nqh);
  auto join = [&](auto kern, int waves) { hipLaunchKernelGGL(kern, all, dim3(64 * waves), 0, stream_of(s), a); };
  auto pick = [&](auto r16, auto r32, auto any) { return y.rows == 16 ? r16 : y.rows == 32 ? r32 : any; };
  if (qrows <= 2 * kCUs) join(pick(attn_paged_join_kernel<16, 16>, attn_paged_join_kernel<16, 32>, attn_paged_join_kernel<16, 0>), 16);
  else join(pick(attn_paged_join_kernel<4, 16>, attn_paged_join_kernel<4, 32>, attn_paged_join_kernel<4, 0>), 4);
  return check_launch("attn_paged");
}
