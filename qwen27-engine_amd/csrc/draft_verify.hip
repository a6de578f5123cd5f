// Verification of drafted tokens against the target's probabilities (draft_verify), for a ragged batch of sequences.
//
// Which drafts stand is a walk over at most 64 tokens, whose probabilities one round of gathers brings: every workgroup of a
// sequence does it for itself (lane t holds token t), and one leaves it for the second launch. What remains is a draw from the row where the walk ended, over the
// whole vocabulary: the sum S of the row's weights, and the first token whose sum up to it passes u S. The row is cut in
// chunks; the first launch leaves each chunk's sum, the second finds the chunk and then the token in it. Bound by HBM: a row
// of p and, behind a refusal in a chain with probabilities, one of q.
//
// Which token that is must not hang on the order of additions, so weights are brought to multiples of 2^-40 in [0, 1]
// (adding and taking away 1.5 * 2^12 in 64 bits does that, to the nearest): sums below 4096 are exact in 64 bits, in any
// order, and the draw is the same in every program that follows the definition.
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
  double2* sums;                   // [n_seqs][chunks]: of max(p - q, 0), and of p
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

__device__ __forceinline__ double weight_of(double x) {
  x = x > 0.0 ? x : 0.0;  // NaN: 0
  x = x < 1.0 ? x : 1.0;
  return (x + 6144.0) - 6144.0;
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

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
  return x;
}

__global__ void __launch_bounds__(kThreads) draft_sums_kernel(VerifyArgs a) {
  __shared__ double s_red[2][kThreads / 64];
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, w = threadIdx.x >> 6;
  const Walk k = walk_of(a, b);
  if (chunk == 0 && threadIdx.x == 0) a.walks[b] = k;
  if (!k.nt) return;
  float p[kPerThread], q[kPerThread];
  load_chunk(a.p + (size_t)(k.t0 + k.node) * a.ldp, chunk, a.V, p);
  if (k.refused) load_chunk(a.q + (size_t)(k.t0 + k.node + 1) * a.ldq, chunk, a.V, q);
  double left = 0.0, all = 0.0;
#pragma unroll
  for (int i = 0; i < kPerThread; i++) all += weight_of(p[i]);
  if (k.refused) {
#pragma unroll
    for (int i = 0; i < kPerThread; i++) left += weight_of((double)p[i] - q[i]);
  }
  left = wave_sum(left);
  all = wave_sum(all);
  if ((threadIdx.x & 63) == 0) s_red[0][w] = left, s_red[1][w] = all;
  __syncthreads();
  if (threadIdx.x) return;
  left = (s_red[0][0] + s_red[0][1]) + (s_red[0][2] + s_red[0][3]);
  all = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  a.sums[(size_t)b * a.chunks + chunk] = make_double2(left, all);
}

// Exclusive sum over the workgroup's threads, and the whole sum.
__device__ __forceinline__ double before_of(double x, double* red, double& total) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  double s = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double y = __shfl_up(s, d);
    s += l >= d ? y : 0.0;
  }
  __syncthreads();
  if (l == 63) red[w] = s;
  __syncthreads();
  total = 0.0;
  double before = s - x;
#pragma unroll
  for (int k = 0; k < kThreads / 64; k++) {
    before += k < w ? red[k] : 0.0;
    total += red[k];
  }
  return before;
}

__global__ void __launch_bounds__(kThreads) draft_pick_kernel(VerifyArgs a) {
  __shared__ double s_red[kThreads / 64], s_before;
  __shared__ int s_chunk, s_token, s_n;
  __shared__ int s_bad[kMostTokens];
  __shared__ double s_takes[kMostTokens];
  const int b = blockIdx.x, tid = threadIdx.x, l = tid & 63;
  const Walk k = a.walks[b];
  if (!k.nt) {
    if (tid == 0) a.n_path[b] = 0;
    return;
  }
  const int id = l < k.nt ? a.ids[k.t0 + l] : -1;  // lane t: token t
  const float* prow = a.p + (size_t)(k.t0 + k.node) * a.ldp;
  const float* qrow = a.q ? a.q + (size_t)(k.t0 + k.node + 1) * a.ldq : nullptr;
  // the refused children weigh nothing: their ids, each once, and what they take from their chunks' sums, exactly
  if (tid < 64) {
    const bool bad = k.tried >> l & 1;
    bool first = bad && (unsigned)id < (unsigned)a.V;
    for (uint64_t m = k.tried; m; m &= m - 1) {
      const int t = __builtin_amdgcn_readfirstlane(__builtin_ctzll(m));
      if (__builtin_amdgcn_readlane(id, t) == id && t < l) first = false;
    }
    const uint64_t each = __ballot(first);
    if (first) {
      const int at = __builtin_popcountll(each & ((1ull << l) - 1));
      s_bad[at] = id;
      s_takes[at] = weight_of(prow[id]);
    }
    if (l == 0) s_n = __builtin_popcountll(each), s_chunk = s_token = -1;
  }
  __syncthreads();
  const int n_bad = s_n;
  auto is_bad = [&](int i) {
    bool bad = false;
    for (int j = 0; j < n_bad; j++) bad |= s_bad[j] == i;
    return bad;
  };
  const double2* sums = a.sums + (size_t)b * a.chunks;
  auto taken = [&](int chunk) {
    double t = 0.0;
    for (int j = 0; j < n_bad; j++) t += s_bad[j] / kChunk == chunk ? s_takes[j] : 0.0;
    return t;
  };
  // the chunk: 256 of them at a time, first their whole sum
  bool use_q = k.refused;
  double total = 0.0;
  for (int pass = 0; pass < 2; pass++) {
    double mine = 0.0;
    for (int c = tid; c < a.chunks; c += kThreads) mine += use_q ? sums[c].x : sums[c].y - taken(c);
    before_of(mine, s_red, total);
    if (total > 0.0 || !use_q) break;
    use_q = false;  // p nowhere above q: the target's own distribution
  }
  double u = a.u_last[b];
  u = u > 0.0 ? u : 0.0;
  u = u < 0x1.fffffep-1 ? u : 0x1.fffffep-1;
  const double want = u * total;
  double base = 0.0;
  for (int c0 = 0; c0 < a.chunks; c0 += kThreads) {
    const int c = c0 + tid;
    const double x = c < a.chunks ? (use_q ? sums[c].x : sums[c].y - taken(c)) : 0.0;
    double part;
    const double before = base + before_of(x, s_red, part);
    if (before <= want && want < before + x) s_chunk = c, s_before = before;
    base += part;
  }
  __syncthreads();
  const int chunk = s_chunk;
  if (chunk >= 0) {
    // its values in order, 16 neighbours a thread
    const int i0 = chunk * kChunk + tid * kPerThread;
    double wt[kPerThread], mine = 0.0;
    if (i0 + kPerThread <= a.V) {
      f4u pv[kPerThread / 4], qv[kPerThread / 4];
#pragma unroll
      for (int g = 0; g < kPerThread / 4; g++) pv[g] = *(const f4u*)(prow + i0 + 4 * g);
      if (use_q) {
#pragma unroll
        for (int g = 0; g < kPerThread / 4; g++) qv[g] = *(const f4u*)(qrow + i0 + 4 * g);
      }
#pragma unroll
      for (int i = 0; i < kPerThread; i++) wt[i] = weight_of(use_q ? (double)pv[i >> 2][i & 3] - qv[i >> 2][i & 3] : (double)pv[i >> 2][i & 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; i++)
        wt[i] = i0 + i < a.V ? weight_of(use_q ? (double)prow[i0 + i] - qrow[i0 + i] : (double)prow[i0 + i]) : 0.0;
    }
    if (n_bad) {
#pragma unroll
      for (int i = 0; i < kPerThread; i++) wt[i] = is_bad(i0 + i) ? 0.0 : wt[i];
    }
#pragma unroll
    for (int i = 0; i < kPerThread; i++) mine += wt[i];
    double part;
    double at = s_before + before_of(mine, s_red, part);
#pragma unroll
    for (int i = 0; i < kPerThread; i++) {
      const double to = at + wt[i];
      if (at <= want && want < to) s_token = i0 + i;
      at = to;
    }
    __syncthreads();
  }
  if (tid >= 64) return;
  // token l of the walk's path goes to its place among them
  const int n = __builtin_popcountll(k.path);
  const int rank = __builtin_popcountll(k.path & ((1ull << l) - 1));
  const bool on = k.path >> l & 1;
  if (on) {
    a.path[k.t0 + rank] = l;
    if (rank) a.out[k.t0 + rank - 1] = id;
  }
  if (l >= n && l < k.nt) a.path[k.t0 + l] = a.out[k.t0 + l] = -1;
  if (l == 0) {
    a.out[k.t0 + n - 1] = s_token;
    a.n_path[b] = n;
    if (a.pos) a.pos[b] += n;
  }
}

int chunks_of(int V) { return (V + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_draft_verify_ws_bytes(int n_seqs, int V) {
  return n_seqs <= 0 || V <= 0 || V > 1 << 24 ? 0 : (size_t)n_seqs * (chunks_of(V) * sizeof(double2) + sizeof(Walk));
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
  double2* sums = (double2*)ws;
  VerifyArgs a = {p, q, ids, parent, u, u_last, cu, out, path, n_path, pos, sums, (Walk*)(sums + (size_t)n_seqs * chunks_of(V)),
                  (long long)ldp, (long long)ldq, T, V, chunks_of(V)};
  hipLaunchKernelGGL(draft_sums_kernel, dim3((unsigned)(n_seqs * a.chunks)), dim3(kThreads), 0, stream_of(s), a);
  hipLaunchKernelGGL(draft_pick_kernel, dim3((unsigned)n_seqs), dim3(kThreads), 0, stream_of(s), a);
  return check_launch("draft_verify");
}
