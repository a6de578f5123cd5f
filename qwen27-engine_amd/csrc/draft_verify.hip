// Verification of drafted tokens against the target's probabilities (draft_verify), for a ragged batch of sequences.
//
// Which drafts stand is a walk over at most 64 tokens, whose probabilities one round of gathers brings: every workgroup of a
// sequence does it for itself (lane t holds token t), and one leaves it for the second launch. What remains is a draw from
// the row where the walk ended, over the whole vocabulary: the sum S of the row's weights, and the first token whose sum up
// to it passes u S. The row is cut in chunks; the first launch leaves each chunk's sum, the second finds the chunk and then
// the token in it. Bound by HBM: a row of p and, behind a refusal in a chain with probabilities, one of q (64 sequences,
// 95 MB: 15.0 us, 6.4 TB/s, and 4.4 for the second launch); one sequence by its round trips (3.9 and 3.4).
//
// Which token that is must not hang on the order of additions, so weights are whole numbers of 2^-40 in [0, 1] and their sums
// 64-bit whole numbers, whatever the row sums to: at most 2^24 weights of at most 2^40. u S is formed exactly as well, and the
// draw is the same in every program that follows the definition.
#include "q27h_device.h"
#include "q27h_internal.h"

namespace q27h {
namespace {

constexpr int kMostTokens = 64;
constexpr int kPerThread = 16, kThreads = 256, kChunk = kThreads * kPerThread;  // values of a chunk

struct Walk;
struct VerifyArgs {
  const float *p, *q;  // q null: drafts without probabilities
  const int *ids, *parent;
  const float *u, *u_last;
  const int* cu;
  int *out, *path, *n_path, *pos;  // pos may be null
  ulonglong2* sums;                // [n_seqs][chunks]: of max(p - q, 0), and of p
  Walk* walks;                     // [n_seqs], for the second launch
  long long ldp, ldq;
  int T, V, chunks;
};

// Where a sequence's walk ended.
struct Walk {
  uint64_t path;   // its accepted tokens, token 0 among them
  uint64_t tried;  // the children of the last one that were refused (drafts without probabilities)
  int t0, nt;
  int node;        // the last one
  int refused;     // a chain with probabilities: token node + 1 was refused, q's row of it is to be taken off
};

__device__ __forceinline__ float read_lane(float x, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
}

// By a whole wave.
__device__ __forceinline__ Walk walk_of(const VerifyArgs& a, int b) {
  const int l = threadIdx.x & 63;
  Walk w;
  int c0 = a.cu[b], c1 = a.cu[b + 1];
  c0 = c0 < 0 ? 0 : c0 > a.T ? a.T : c0;
  c1 = c1 < c0 ? c0 : c1 > a.T ? a.T : c1;
  w.t0 = __builtin_amdgcn_readfirstlane(c0);
  w.nt = __builtin_amdgcn_readfirstlane(c1 - c0 < kMostTokens ? c1 - c0 : kMostTokens);
  w.path = w.nt ? 1ull : 0ull;
  w.tried = 0;
  w.node = 0;
  w.refused = 0;
  const bool draft = l >= 1 && l < w.nt;
  const int mine = l < w.nt ? a.ids[w.t0 + l] : -1;
  int parent = l - 1;
  if (a.parent && draft) parent = a.parent[w.t0 + l];
  const bool sound = draft && parent >= 0 && parent < l && (unsigned)mine < (unsigned)a.V;
  const float u = draft ? a.u[w.t0 + l] : 0.0f;
  const float p = sound ? a.p[(size_t)(w.t0 + parent) * a.ldp + mine] : 0.0f;
  if (a.q) {  // a chain: the first draft that is refused ends it. The products of two floats are exact in 64 bits.
    const float q = sound ? a.q[(size_t)(w.t0 + l) * a.ldq + mine] : 0.0f;
    const uint64_t yes = __ballot(draft && (double)u * q < (double)p) | 1ull;
    const int n = yes == ~0ull ? 64 : __builtin_ctzll(~yes);  // tokens accepted, the first among them
    if (w.nt) w.path = n == 64 ? ~0ull : (1ull << n) - 1;
    w.node = n - 1;
    w.refused = n < w.nt;
    return w;
  }
  double rest = 1.0;  // 1 - the probabilities of the refused children
  const uint64_t drafts = w.nt > 1 ? (w.nt < 64 ? 1ull << w.nt : 0ull) - 2 : 0ull;  // tokens 1 .. nt - 1
  for (uint64_t todo = drafts & __ballot(parent == 0); todo;) {
    const int t = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int id = __builtin_amdgcn_readlane(mine, t);
    const bool again = (__ballot(mine == id) & w.tried) != 0;  // a token that was refused already
    const double x = again ? 0.0 : (double)read_lane(p, t);
    if ((double)read_lane(u, t) * rest < x) {
      w.node = t, w.path |= 1ull << t, w.tried = 0, rest = 1.0;
      todo = drafts & __ballot(parent == t) & ~((2ull << t) - 1);  // a child lies behind its parent
    } else {
      rest -= x, w.tried |= 1ull << t;
    }
  }
  return w;
}

// To the nearest whole number of 2^-40: that is the last bit of a number in 64 bits from 4096 to 8192.
__device__ __forceinline__ uint64_t weight_of(double x) {
  x = x > 0.0 ? x : 0.0;  // NaN: 0
  x = x < 1.0 ? x : 1.0;
  return __builtin_bit_cast(uint64_t, x + 6144.0) - __builtin_bit_cast(uint64_t, 6144.0);
}
// floor(u s) for u in [0, 1), s = 2^64 where `over`: a sum of whole numbers exceeds u s where it exceeds this.
__device__ __forceinline__ uint64_t share_of(float u, uint64_t s, bool over) {
  const uint32_t b = __builtin_bit_cast(uint32_t, u);
  const uint32_t m = b >> 23 ? (b & 0x7fffff) | 0x800000 : b, e = b >> 23 ? 150 - (b >> 23) : 149;  // u = m 2^-e, e >= 24
  const uint64_t lo = (s & 0xffffffff) * m, hi = (s >> 32) * m + (lo >> 32) + (over ? (uint64_t)m << 32 : 0);  // m s = hi 2^32 + lo's low half
  return e < 32 ? hi << (32 - e) | (lo & 0xffffffff) >> e : e < 96 ? hi >> (e - 32) : 0;
}

// Four neighbouring values from any address of a float: rows of an odd vocabulary begin anywhere.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// A thread's 16 values of a chunk: four groups of four, 1024 apart. `n`: values of the row; behind them zeros.
__device__ __forceinline__ void load_chunk(const float* row, int chunk, int n, float (&x)[kPerThread]) {
#pragma unroll
  for (int k = 0; k < kPerThread / 4; k++) {
    const int i = chunk * kChunk + k * 4 * kThreads + 4 * threadIdx.x;
    if (i + 4 <= n) {
      const f4u v = *(const f4u*)(row + i);
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * k + e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * k + e] = i + e < n ? row[i + e] : 0.0f;
    }
  }
}

// Sums over the lanes up to each one; 0 comes from lanes that do not exist.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t from_lanes(uint64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t lanes_before(uint64_t x) {
  x += from_lanes<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: within rows of 16
  x += from_lanes<0x112, 0xf>(x);
  x += from_lanes<0x114, 0xf>(x);
  x += from_lanes<0x118, 0xf>(x);
  x += from_lanes<0x142, 0xa>(x);  // row_bcast 15, 31: the rows before
  x += from_lanes<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ uint64_t read_lane(uint64_t x, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)x, l), hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
  return (uint64_t)hi << 32 | lo;
}

__global__ void __launch_bounds__(kThreads) draft_sums_kernel(VerifyArgs a) {
  __shared__ uint64_t s_red[2][kThreads / 64];
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, w = threadIdx.x >> 6;
  const Walk k = walk_of(a, b);
  if (chunk == 0 && threadIdx.x == 0) a.walks[b] = k;
  if (!k.nt) return;
  float p[kPerThread], q[kPerThread];
  load_chunk(a.p + (size_t)(k.t0 + k.node) * a.ldp, chunk, a.V, p);
  if (k.refused) load_chunk(a.q + (size_t)(k.t0 + k.node + 1) * a.ldq, chunk, a.V, q);
  uint64_t left = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; i++) all += weight_of(p[i]);
  if (k.refused) {
#pragma unroll
    for (int i = 0; i < kPerThread; i++) left += weight_of((double)p[i] - q[i]);
  }
  all = lanes_before(all);
  if (k.refused) left = lanes_before(left);
  if ((threadIdx.x & 63) == 63) s_red[0][w] = left, s_red[1][w] = all;
  __syncthreads();
  if (threadIdx.x) return;
  left = (s_red[0][0] + s_red[0][1]) + (s_red[0][2] + s_red[0][3]);
  all = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  a.sums[(size_t)b * a.chunks + chunk] = make_ulonglong2(left, all);
}

// Every wave finds the chunk by itself, 64 chunks at a time; then a thread has 16 neighbouring values of it.
__global__ void __launch_bounds__(kThreads) draft_pick_kernel(VerifyArgs a) {
  __shared__ uint64_t s_sum[kThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const ulonglong2* sums = a.sums + (size_t)b * a.chunks;
  uint64_t left0 = 0, all0 = 0;  // of the first 64 chunks, on their way with the walk
  if (l < a.chunks) left0 = sums[l].x, all0 = sums[l].y;
  const Walk k = a.walks[b];
  const int n = __builtin_popcountll(k.path);
  if (!k.nt) {
    if (tid == 0) a.n_path[b] = 0;
    return;
  }
  const int id = l < k.nt ? a.ids[k.t0 + l] : -1;  // lane t: token t
  const float* prow = a.p + (size_t)(k.t0 + k.node) * a.ldp;
  const float* qrow = k.refused ? a.q + (size_t)(k.t0 + k.node + 1) * a.ldq : prow;
  // the refused children weigh nothing: each id once (lanes of `bad`), and what it takes from its chunk's sum
  bool lead = (k.tried >> l & 1) && (unsigned)id < (unsigned)a.V;
  for (uint64_t m = k.tried; m; m &= m - 1) {
    const int t = __builtin_amdgcn_readfirstlane(__builtin_ctzll(m));
    if (__builtin_amdgcn_readlane(id, t) == id && t < l) lead = false;
  }
  const uint64_t bad = __ballot(lead);
  const uint64_t takes = lead ? weight_of(prow[id]) : 0;
  bool use_q = k.refused;
  auto sum_of = [&](int c) {  // of chunk c
    uint64_t x = use_q ? left0 : all0;
    if (c != l) x = c >= a.chunks ? 0 : use_q ? sums[c].x : sums[c].y;
    for (uint64_t m = bad; m; m &= m - 1) {
      const int t = __builtin_amdgcn_readfirstlane(__builtin_ctzll(m));
      x -= __builtin_amdgcn_readlane(id, t) / kChunk == c ? read_lane(takes, t) : 0;
    }
    return x;
  };
  uint64_t total = 0;
  bool over = false;  // it is 2^64: every weight of 2^24 is 1
  for (int pass = 0; pass < 2; pass++) {
    total = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) total += read_lane(lanes_before(sum_of(c0 + l)), 63);
    if (!total) over = read_lane(sum_of(l), 0) != 0;
    if (total || over || !use_q) break;
    use_q = false;  // p nowhere above q: the target's own distribution
  }
  float u = a.u_last[b];
  u = u > 0.0f ? u : 0.0f;
  u = u < 0x1.fffffep-1f ? u : 0x1.fffffep-1f;
  const uint64_t want = share_of(u, total, over);
  // The token, as its chunk, is the one with a weight x behind a sum y such that y <= want < y + x: one alone.
  auto holds = [want](uint64_t y, uint64_t x) { return y <= want && want - y < x; };
  uint64_t base = 0;
  int chunk = -1;
  for (int c0 = 0; c0 < a.chunks && chunk < 0; c0 += 64) {
    const uint64_t x = sum_of(c0 + l), to = base + lanes_before(x);
    const uint64_t hit = __ballot(holds(to - x, x));
    if (hit) {
      const int t = __builtin_ctzll(hit);
      chunk = c0 + t;
      base = read_lane(to - x, t);
    } else {
      base = read_lane(to, 63);
    }
  }
  if (tid == 0) a.out[k.t0 + n - 1] = -1;  // unless there is a token, below and behind the barrier
  if (chunk >= 0) {
    const int i0 = chunk * kChunk + tid * kPerThread;
    uint64_t wt[kPerThread], mine = 0;
    if (i0 + kPerThread <= a.V) {
      f4u pv[kPerThread / 4], qv[kPerThread / 4];
#pragma unroll
      for (int g = 0; g < kPerThread / 4; g++) {
        pv[g] = *(const f4u*)(prow + i0 + 4 * g);
        if (use_q) qv[g] = *(const f4u*)(qrow + i0 + 4 * g);
      }
#pragma unroll
      for (int i = 0; i < kPerThread; i++) wt[i] = weight_of(use_q ? (double)pv[i >> 2][i & 3] - qv[i >> 2][i & 3] : (double)pv[i >> 2][i & 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; i++)
        wt[i] = i0 + i < a.V ? weight_of(use_q ? (double)prow[i0 + i] - qrow[i0 + i] : (double)prow[i0 + i]) : 0;
    }
    for (uint64_t m = bad; m; m &= m - 1) {
      const int at = __builtin_amdgcn_readlane(id, __builtin_amdgcn_readfirstlane(__builtin_ctzll(m))) - i0;
#pragma unroll
      for (int i = 0; i < kPerThread; i++) wt[i] = at == i ? 0 : wt[i];
    }
#pragma unroll
    for (int i = 0; i < kPerThread; i++) mine += wt[i];
    uint64_t at = lanes_before(mine);
    if (l == 63) s_sum[w] = at;
    __syncthreads();
    at += base - mine;
#pragma unroll
    for (int j = 0; j < kThreads / 64; j++) at += j < w ? s_sum[j] : 0;
    if (holds(at, mine)) {  // one thread: behind its values whose sums are no more than what is left of `want`
      const uint64_t left = want - at;
      uint64_t to = 0;
      int i = i0;
#pragma unroll
      for (int e = 0; e < kPerThread; e++) {
        to += wt[e];
        i += to <= left;
      }
      a.out[k.t0 + n - 1] = i;
    }
  }
  if (tid >= 64) return;
  // token l of the walk's path goes to its place among them
  const int rank = __builtin_popcountll(k.path & ((1ull << l) - 1));
  if (k.path >> l & 1) {
    a.path[k.t0 + rank] = l;
    if (rank) a.out[k.t0 + rank - 1] = id;
  }
  if (l >= n && l < k.nt) a.path[k.t0 + l] = a.out[k.t0 + l] = -1;
  if (l == 0) {
    a.n_path[b] = n;
    if (a.pos) a.pos[b] += n;
  }
}

int chunks_of(int V) { return (V + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_draft_verify_ws_bytes(int n_seqs, int V) {
  return n_seqs <= 0 || V <= 0 || V > 1 << 24 ? 0 : (size_t)n_seqs * (chunks_of(V) * sizeof(ulonglong2) + sizeof(Walk));
}

extern "C" int q27h_draft_verify(const float* p, int64_t ldp, const float* q, int64_t ldq, const int* ids, const int* parent,
                                 const float* u, const float* u_last, const int* cu, int n_seqs, int T, int V, int* out, int* path,
                                 int* n_path, int* pos, void* ws, size_t ws_bytes, q27h_stream_t s) {
  if (n_seqs < 0 || T < 0 || V <= 0 || V > 1 << 24) return fail(Q27H_ERR_SHAPE, "draft_verify: bad shape (vocabulary 1 .. 2^24)");
  if (ldp < V || (q && ldq < V) || ldp > 1 << 28 || ldq > 1 << 28) return fail(Q27H_ERR_SHAPE, "draft_verify: bad row stride");
  if ((double)n_seqs * chunks_of(V) > 1.6e7) return fail(Q27H_ERR_SHAPE, "draft_verify: too many sequences");
  if (q && parent) return fail(Q27H_ERR_ARG, "draft_verify: drafts with probabilities are a chain: q and parent exclude each other");
  if (n_seqs == 0) return Q27H_OK;
  if (!cu || !u_last || !n_path || (T && (!p || !ids || !u || !out || !path))) return fail(Q27H_ERR_ARG, "draft_verify: null pointer");
  for (const void* x : {(const void*)p, (const void*)q, (const void*)ids, (const void*)parent, (const void*)u, (const void*)u_last,
                        (const void*)cu, (const void*)out, (const void*)path, (const void*)n_path, (const void*)pos})
    if (!aligned4(x)) return fail(Q27H_ERR_ARG, "draft_verify: arrays need 4-byte alignment");
  const size_t need = q27h_draft_verify_ws_bytes(n_seqs, V), B = (size_t)n_seqs * 4, tb = (size_t)T * 4;
  if (ws_bytes < need || !ws || !aligned16(ws)) return fail(Q27H_ERR_ARG, "draft_verify: workspace too small or out of alignment");
  const size_t pb = T ? ((size_t)(T - 1) * ldp + V) * 4 : 0, qb = T ? ((size_t)(T - 1) * ldq + V) * 4 : 0;
  if (outputs_overlap({{out, tb}, {path, tb}, {n_path, B}, {pos, B}, {ws, need}},
                      {{p, pb}, {q, qb}, {ids, tb}, {parent, tb}, {u, tb}, {u_last, B}, {cu, B + 4}}))
    return fail(Q27H_ERR_ARG, "draft_verify: a result, pos or ws overlaps another argument");
  ulonglong2* sums = (ulonglong2*)ws;
  VerifyArgs a = {p, q, ids, parent, u, u_last, cu, out, path, n_path, pos, sums, (Walk*)(sums + (size_t)n_seqs * chunks_of(V)),
                  (long long)ldp, (long long)ldq, T, V, chunks_of(V)};
  hipLaunchKernelGGL(draft_sums_kernel, dim3((unsigned)(n_seqs * a.chunks)), dim3(kThreads), 0, stream_of(s), a);
  hipLaunchKernelGGL(draft_pick_kernel, dim3((unsigned)n_seqs), dim3(kThreads), 0, stream_of(s), a);
  return check_launch("draft_verify");
}
