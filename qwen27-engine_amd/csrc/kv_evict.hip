// Which rows of the K/V cache stay, and moving them: eviction by accumulated attention weight (kv_evict) and the move of
// an accepted path of drafted tokens to its place (kv_accept).
//
// kv_evict keeps, per kv head, the first `first` rows, the last `last` rows and the heaviest of those between, in their
// order. The weights' exact order is found by three histograms (11, 11 and 10 bits of the integer key, counted with
// integer atomics, so in any order to the same result) over workgroups that each hold a segment of the rows; then each
// segment counts its rows above and at the threshold and writes its own part of the list behind the segments before it.
// Up to 32768 rows of context one workgroup a kv head does all of that over keys in LDS (20001 rows: 7 launches, 29 us;
// two, 23 us, 15 of them the choice). Rows are moved by 16 bytes a lane. In place, the kept rows that lie before row
// `keep` go through the workspace, since a row's place may be another one's source there; the others are read where no
// row is written.
#include "pick.h"
#include "q27h_device.h"
#include "q27h_internal.h"

namespace q27h {
namespace {

constexpr int kHD = 256;
constexpr int kBins = 2048;
constexpr int kSegRows = 2048;  // rows of a segment, while there are fewer than kMaxSegs of them
constexpr int kMaxSegs = 128;
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int segs_of(int n_ctx) {
  const int s = (n_ctx + kSegRows - 1) / kSegRows;
  return s > kMaxSegs ? kMaxSegs : s;
}

struct EvictArgs {
  const void *kc, *vc;
  const float* acc;
  const int* pos0;
  void *ko, *vo;
  float* acc_o;
  int* kept;
  uint8_t *k_aside, *v_aside;  // in place: workspace of `keep` rows
  float* acc_aside;
  int* hist;    // [nkvh][3][kBins]
  int2* count;  // [nkvh][segs]: rows above, rows at the threshold
  int keep, first, last, n_out, nkvh, n_ctx, q8, segs;
};

__device__ __forceinline__ int rows_of(const EvictArgs& a) {
  const int n = *a.pos0;
  return n < 0 ? 0 : n > a.n_ctx ? a.n_ctx : n;
}

// The bin (from the top) in which the need-th value of a histogram lies, and how many of that bin are needed.
__device__ __forceinline__ void find_bin(const int* hist, int bins, int& need, int& bin, int* s_scan, int* s_pick) {
  const int per = bins / 256;
  int h[kBins / 256], mine = 0;
#pragma unroll
  for (int i = 0; i < kBins / 256; i++)
    if (i < per) h[i] = hist[bins - 1 - (int)threadIdx.x * per - i], mine += h[i];
  int total;
  int above = scan256(mine, s_scan, total);
#pragma unroll
  for (int i = 0; i < kBins / 256; i++) {
    if (i < per) {
      if (above < need && need <= above + h[i]) s_pick[0] = bins - 1 - (int)threadIdx.x * per - i, s_pick[1] = need - above;
      above += h[i];
    }
  }
  __syncthreads();
  bin = s_pick[0];
  need = s_pick[1];
  __syncthreads();
}
__device__ __forceinline__ int digit_of(uint32_t key, int pass) {
  return pass == 0 ? key >> 21 : pass == 1 ? (key >> 10) & 2047 : key & 1023;
}
__device__ __forceinline__ uint32_t above_digit(uint32_t key, int pass) { return pass == 0 ? 0u : pass == 1 ? key >> 21 : key >> 10; }

// The key's digits found by the first `passes` histograms, and how many of the rows that share them are kept.
__device__ __forceinline__ uint32_t prefix_of(const EvictArgs& a, int kh, int passes, int& need, int* s_scan, int* s_pick) {
  uint32_t key = 0;
  const int* h = a.hist + (size_t)kh * 3 * kBins;
  for (int p = 0; p < passes; p++) {
    int bin;
    find_bin(h + p * kBins, p == 2 ? 1024 : kBins, need, bin, s_scan, s_pick);
    key |= (uint32_t)bin << (p == 0 ? 21 : p == 1 ? 10 : 0);
  }
  return key;
}

__global__ void __launch_bounds__(256) evict_clear_kernel(int* hist) {
  *(int4*)(hist + 4 * ((size_t)blockIdx.x * 256 + threadIdx.x)) = make_int4(0, 0, 0, 0);
}

// One digit's histogram of the rows between the fixed ends; a workgroup per (segment, kv head).
__global__ void __launch_bounds__(256) evict_hist_kernel(EvictArgs a, int pass) {
  __shared__ int s_hist[kBins], s_scan[4], s_pick[2];
  const int kh = blockIdx.y, n = rows_of(a);
  int need = a.keep - a.first - a.last;
  if (n <= a.keep || need == 0) return;
  const int r0 = a.first, r1 = n - a.last, per = (r1 - r0 + a.segs - 1) / a.segs;
  const int b = r0 + blockIdx.x * per, e = b + per < r1 ? b + per : r1;
  if (b >= e) return;
  for (int i = threadIdx.x; i < kBins; i += 256) s_hist[i] = 0;
  const uint32_t key = prefix_of(a, kh, pass, need, s_scan, s_pick);
  __syncthreads();
  const float* acc = a.acc + (size_t)kh * a.n_ctx;
  for (int r = b + threadIdx.x; r < e; r += 256) {
    const uint32_t k = order_key(acc[r]);
    if (above_digit(k, pass) == above_digit(key, pass)) atomicAdd(&s_hist[digit_of(k, pass)], 1);
  }
  __syncthreads();
  int* h = a.hist + ((size_t)kh * 3 + pass) * kBins;
  for (int i = threadIdx.x; i < kBins; i += 256)
    if (s_hist[i]) atomicAdd(h + i, s_hist[i]);
}

__global__ void __launch_bounds__(256) evict_count_kernel(EvictArgs a) {
  __shared__ int s_scan[4], s_pick[2];
  const int kh = blockIdx.y, n = rows_of(a);
  int need = a.keep - a.first - a.last;
  if (n <= a.keep) return;
  const int r0 = a.first, r1 = n - a.last, per = (r1 - r0 + a.segs - 1) / a.segs;
  const int b = r0 + blockIdx.x * per, e = b + per < r1 ? b + per : r1;
  int above = 0, equal = 0;
  if (need) {
    const uint32_t key = prefix_of(a, kh, 3, need, s_scan, s_pick);
    const float* acc = a.acc + (size_t)kh * a.n_ctx;
    for (int r = b + threadIdx.x; r < e; r += 256) {
      const uint32_t k = order_key(acc[r]);
      above += k > key;
      equal += k == key;
    }
    int t0, t1;
    scan256(above, s_scan, t0);
    scan256(equal, s_scan, t1);
    above = t0, equal = t1;
  }
  if (threadIdx.x == 0) a.count[kh * a.segs + blockIdx.x] = make_int2(above, equal);
}

// The whole choice of a kv head by one workgroup, for contexts of up to kLdsRows: keys in LDS, digits of key - (least key)
// from the top (see select_pick_kernel in attn_select.hip), until a bin is kept whole; then each thread lists a stretch
// of consecutive rows, an odd number of them, so that the lanes' reads fall in different banks.
constexpr int kLdsRows = 32768, kListThreads = 1024;
__global__ void __launch_bounds__(kListThreads) evict_choose_kernel(EvictArgs a) {
  __shared__ uint32_t s_key[kLdsRows];
  __shared__ int s_hist[kBins], s_scan[kListThreads / 64], s_pick[3];
  __shared__ uint32_t s_end[2 * kListThreads / 64];
  const int kh = blockIdx.x, tid = threadIdx.x, w = tid >> 6, n = rows_of(a);
  int* out = a.kept + (size_t)kh * a.keep;
  if (n <= a.keep) {
    for (int i = tid; i < a.keep; i += kListThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int r0 = a.first, rows = n - a.last - r0;
  const float* acc = a.acc + (size_t)kh * a.n_ctx + r0;
  uint32_t least = ~0u, most = 0u;
  constexpr int kEach = kLdsRows / kListThreads;
  float x[kEach];  // requested together
#pragma unroll
  for (int i = 0; i < kEach; i++)
    if (tid + i * kListThreads < rows) x[i] = acc[tid + i * kListThreads];
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    if (tid + i * kListThreads >= rows) break;
    const uint32_t k = order_key(x[i]);
    s_key[tid + i * kListThreads] = k;
    least = least < k ? least : k;
    most = most > k ? most : k;
  }
  for (int i = tid; i < a.first; i += kListThreads) out[i] = i;
  for (int i = tid; i < a.last; i += kListThreads) out[a.keep - a.last + i] = n - a.last + i;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t x = __shfl_xor(least, d), y = __shfl_xor(most, d);
    least = least < x ? least : x;
    most = most > y ? most : y;
  }
  if ((tid & 63) == 0) s_end[2 * w] = least, s_end[2 * w + 1] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kListThreads / 64; i++) {
    const uint32_t x = s_end[2 * i], y = s_end[2 * i + 1];
    least = least < x ? least : x;
    most = most > y ? most : y;
  }
  int need = a.keep - a.first - a.last, shift = need && least < most ? 32 - __builtin_clz(most - least) : 0;
  uint32_t prefix = need ? 0u : ~0u;
  auto upper = [](uint32_t k, int by) { return (uint32_t)((uint64_t)k >> by); };
  while (shift > 0) {
    const int next = shift > 11 ? shift - 11 : 0;
    s_hist[tid] = s_hist[tid + 1024] = 0;
    __syncthreads();
#pragma unroll 4
    for (int r = tid; r < rows; r += kListThreads) {
      const uint32_t k = s_key[r] - least;
      if (upper(k, shift) == upper(prefix, shift)) atomicAdd(&s_hist[(k >> next) & ((1u << (shift - next)) - 1u)], 1);
    }
    __syncthreads();
    const int hi = s_hist[kBins - 1 - 2 * tid], lo = s_hist[kBins - 2 - 2 * tid];
    int total;
    int above = scan_waves<kListThreads / 64>(hi + lo, s_scan, total);
    if (above < need && need <= above + hi) s_pick[0] = kBins - 1 - 2 * tid, s_pick[1] = need - above, s_pick[2] = hi;
    above += hi;
    if (above < need && need <= above + lo) s_pick[0] = kBins - 2 - 2 * tid, s_pick[1] = need - above, s_pick[2] = lo;
    __syncthreads();
    prefix |= (uint32_t)s_pick[0] << next;
    need = s_pick[1];
    shift = next;
    if (need == s_pick[2]) break;
    __syncthreads();
  }
  __syncthreads();
  const int per = (rows + kListThreads - 1) / kListThreads | 1, c0 = tid * per < rows ? tid * per : rows;
  const int c1 = c0 + per < rows ? c0 + per : rows;
  const uint32_t p = upper(prefix, shift);
  uint32_t mine = 0;  // above << 16 | equal, together at most kLdsRows
#pragma unroll 8
  for (int r = c0; r < c1; r++) {
    const uint32_t k = upper(s_key[r] - least, shift);
    mine += (k > p ? 1u << 16 : 0u) + (k == p);
  }
  int total;
  const uint32_t before = (uint32_t)scan_waves<kListThreads / 64>((int)mine, s_scan, total);
  int at = (int)(before >> 16), rank = (int)(before & 0xffffu);
  at += a.first + (rank < need ? rank : need);
#pragma unroll 4
  for (int r = c0; r < c1; r++) {
    const uint32_t k = upper(s_key[r] - least, shift);
    const bool take = k > p || (k == p && rank < need);
    rank += k == p;
    if (take) out[at++] = r0 + r;
  }
}

// The list of kept rows: a segment's part starts behind the rows kept by the segments before it.
__global__ void __launch_bounds__(256) evict_list_kernel(EvictArgs a) {
  __shared__ int s_scan[4], s_pick[2];
  __shared__ uint32_t s_key[8 * 256];
  const int kh = blockIdx.y, n = rows_of(a), seg = blockIdx.x;
  int* out = a.kept + (size_t)kh * a.keep;
  if (n <= a.keep) {
    for (int i = seg * 256 + threadIdx.x; i < a.keep; i += a.segs * 256) out[i] = i < n ? i : -1;
    return;
  }
  for (int i = seg * 256 + threadIdx.x; i < a.first; i += a.segs * 256) out[i] = i;
  for (int i = seg * 256 + threadIdx.x; i < a.last; i += a.segs * 256) out[a.keep - a.last + i] = n - a.last + i;
  int need = a.keep - a.first - a.last;
  if (need == 0) return;
  const int r0 = a.first, r1 = n - a.last, per = (r1 - r0 + a.segs - 1) / a.segs;
  const int b = r0 + seg * per, e = b + per < r1 ? b + per : r1;
  if (b >= e) return;
  const uint32_t key = prefix_of(a, kh, 3, need, s_scan, s_pick);
  int above = 0, equal = 0;  // of the segments before this one
  for (int i = threadIdx.x; i < seg; i += 256) above += a.count[kh * a.segs + i].x, equal += a.count[kh * a.segs + i].y;
  int t0, t1;
  scan256(above, s_scan, t0);
  scan256(equal, s_scan, t1);
  equal = t1;
  int done = a.first + t0 + (equal < need ? equal : need);
  const float* acc = a.acc + (size_t)kh * a.n_ctx;
  // 2048 rows at a time: each thread counts and lists 8 consecutive ones
  for (int base = b; base < e; base += 8 * 256) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int r = base + 256 * i + threadIdx.x;
      s_key[256 * i + threadIdx.x] = r < e ? order_key(acc[r]) : 0u;
    }
    __syncthreads();
    uint32_t k[8];
    int n_above = 0, n_equal = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const bool is = base + 8 * (int)threadIdx.x + i < e;
      k[i] = s_key[8 * threadIdx.x + i];
      n_above += is && k[i] > key;
      n_equal += is && k[i] == key;
    }
    int total_above, total_equal;
    int at = scan256(n_above, s_scan, total_above), rank = scan256(n_equal, s_scan, total_equal);
    const int start = equal < need ? equal : need;  // equal rows taken before this stretch of 2048
    rank += equal;
    at += done + (rank < need ? rank : need) - start;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int r = base + 8 * (int)threadIdx.x + i;
      const bool take = r < e && (k[i] > key || (k[i] == key && rank < need));
      rank += r < e && k[i] == key;
      if (take) out[at++] = r;
    }
    equal += total_equal;
    done += total_above + (equal < need ? equal : need) - start;
  }
}

// Rows of K and V (blockIdx.z), 16 or 32 lanes of 16 bytes a row, then for q8 the row's 16 bytes of scales; the weights
// with K. OUT: kept rows to their places in other buffers. In place: ASIDE: those of rows before `keep` that have to move,
// to the workspace; BACK: those to their places, and the others from where they lie.
enum { OUT, ASIDE, BACK };
constexpr int kMoves = 2;  // rows of a thread in flight at once
template <int MODE>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a) {
  const int kh = blockIdx.y, n = rows_of(a), m = n < a.keep ? n : a.keep;
  if (MODE != OUT && n <= a.keep) return;  // nothing evicted: every row is where it belongs
  const bool v = blockIdx.z;
  const uint8_t* cache = (const uint8_t*)(v ? a.vc : a.kc);
  uint8_t* aside = (uint8_t*)(v ? a.v_aside : a.k_aside);
  uint8_t* out = (uint8_t*)(v ? a.vo : a.ko);
  const int lanes = a.q8 ? 16 : 32, sub = threadIdx.x % lanes, rows = 256 / lanes;
  const size_t stride = (size_t)lanes * 16;
  // where row r of kv head kh lies in a buffer of so many rows, and its scales
  auto row = [&](auto* base, int n_rows, int r) { return base + ((size_t)kh * n_rows + r) * stride + sub * 16; };
  auto scale = [&](auto* base, int n_rows, int r) {
    return base + (size_t)a.nkvh * n_rows * kHD + ((size_t)kh * n_rows + r) * 16;
  };
  const int out_rows = MODE == ASIDE ? a.keep : a.n_out;
  uint8_t* to = MODE == ASIDE ? aside : out;
  float* acc_to = MODE == ASIDE ? a.acc_aside : a.acc_o;
  const int* kept = a.kept + (size_t)kh * a.keep;
  for (int i0 = blockIdx.x * rows * kMoves + threadIdx.x / lanes; i0 < m; i0 += gridDim.x * rows * kMoves) {
    int r[kMoves];
    bool go[kMoves], ws[kMoves];  // to be moved here; from the workspace
    u4 x[kMoves], d[kMoves];
    float w[kMoves];
#pragma unroll
    for (int k = 0; k < kMoves; k++) r[k] = i0 + k * rows < m ? kept[i0 + k * rows] : -1;
#pragma unroll
    for (int k = 0; k < kMoves; k++) {
      const int i = i0 + k * rows;
      const bool near = MODE != OUT && r[k] < a.keep;
      go[k] = r[k] >= 0 && (MODE == OUT || (r[k] != i && (MODE != ASIDE || near)));
      ws[k] = MODE == BACK && near;
      const uint8_t* from = ws[k] ? aside : cache;
      const int from_rows = ws[k] ? a.keep : a.n_ctx, fr = ws[k] ? i : r[k];
      if (!go[k]) continue;
      x[k] = *(const u4*)row(from, from_rows, fr);
      if (a.q8 && sub == 0) d[k] = *(const u4*)scale(from, from_rows, fr);
      if (!v && sub == 1) w[k] = ws[k] ? a.acc_aside[(size_t)kh * a.keep + i] : a.acc[(size_t)kh * a.n_ctx + r[k]];
    }
#pragma unroll
    for (int k = 0; k < kMoves; k++) {
      const int i = i0 + k * rows;
      if (!go[k]) continue;
      *(u4*)row(to, out_rows, i) = x[k];
      if (a.q8 && sub == 0) *(u4*)scale(to, out_rows, i) = d[k];
      if (!v && sub == 1) acc_to[(size_t)kh * out_rows + i] = w[k];
    }
  }
}

__global__ void evict_pos_kernel(int* pos0, int* rdelta, int keep) {
  const int n = *pos0, m = n < keep ? n : keep;
  *pos0 = m;
  if (rdelta) *rdelta -= n - m;
}

// kv_accept: one workgroup per (cache or weight array, kv head) holds all the path's rows in registers before it writes
// the first of them, so a path in any order is right.
constexpr int kMaxPath = 64, kMaxPtrs = 64;
struct AcceptArgs {
  void* cache[kMaxPtrs];
  float* acc[kMaxPtrs];
  const int *pos0, *path, *n_path;
  int n_cache, T, nkvh, n_ctx, q8;
};
__global__ void __launch_bounds__(256) accept_kernel(AcceptArgs a) {
  __shared__ int s_src[kMaxPath], s_n;
  const int kh = blockIdx.y, tid = threadIdx.x, pos0 = *a.pos0;
  if (tid < 64) {
    const int want = *a.n_path < a.T ? *a.n_path : a.T;
    const int p = tid < want ? a.path[tid] : -1;
    const bool ok = p >= 0 && p < a.T;
    const uint64_t good = __ballot(ok);
    if (tid == 0) s_n = good == ~0ull ? 64 : __builtin_ctzll(~good);  // the path ends at its first entry outside the tree
    s_src[tid] = p;
  }
  __syncthreads();
  const int n = s_n;
  // row i of the path: from cache row pos0 + path[i] to pos0 + i, where both exist
  auto rows = [&](int i, size_t& from, size_t& to) {
    const long long f = (long long)pos0 + s_src[i], t = (long long)pos0 + i;
    from = (size_t)kh * a.n_ctx + (size_t)(f < 0 ? 0 : f);
    to = (size_t)kh * a.n_ctx + (size_t)(t < 0 ? 0 : t);
    return f >= 0 && f < a.n_ctx && t >= 0 && t < a.n_ctx;
  };
  if ((int)blockIdx.x >= a.n_cache) {
    float* acc = a.acc[blockIdx.x - a.n_cache];
    size_t from = 0, to = 0;
    const bool ok = tid < n && rows(tid, from, to);
    const float x = ok ? acc[from] : 0.0f;
    __syncthreads();
    if (ok) acc[to] = x;
    return;
  }
  uint8_t* c = (uint8_t*)a.cache[blockIdx.x];
  const int lanes = a.q8 ? 16 : 32, sub = tid % lanes, step = 256 / lanes;
  const size_t stride = (size_t)lanes * 16;
  uint8_t* sc = c + (size_t)a.nkvh * a.n_ctx * kHD;
  u4 x[8], d = {0u, 0u, 0u, 0u};
  size_t from = 0, to = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int i = k * step + tid / lanes;
    if (i < n && rows(i, from, to)) x[k] = *(const u4*)(c + from * stride + sub * 16);
  }
  if (a.q8 && tid < n && rows(tid, from, to)) d = *(const u4*)(sc + from * 16);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int i = k * step + tid / lanes;
    if (i < n && rows(i, from, to)) *(u4*)(c + to * stride + sub * 16) = x[k];
  }
  if (a.q8 && tid < n && rows(tid, from, to)) *(u4*)(sc + to * 16) = d;
}

size_t cache_bytes(int nkvh, int n_ctx, int q8) { return q27h_kv_cache_bytes(nkvh, n_ctx, q8); }
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_kv_evict_ws_bytes(int nkvh, int n_ctx, int keep, int q8, int in_place) {
  if (nkvh <= 0 || n_ctx <= 0 || keep <= 0) return 0;
  size_t b = up256((size_t)nkvh * 3 * kBins * 4) + up256((size_t)nkvh * segs_of(n_ctx) * 8) + up256((size_t)nkvh * keep * 4);
  if (in_place) b += 2 * up256(cache_bytes(nkvh, keep, q8)) + up256((size_t)nkvh * keep * 4);
  return b;
}

extern "C" int q27h_kv_evict(const void* kcache, const void* vcache, const float* acc, const int* pos0, int keep, int first,
                             int last, void* kout, void* vout, float* acc_out, int n_ctx_out, int* kept, int nkvh, int n_ctx,
                             int q8, void* ws, size_t ws_bytes, q27h_stream_t s) {
  if (nkvh <= 0 || nkvh > 65535 || n_ctx <= 0 || n_ctx_out <= 0) return fail(Q27H_ERR_SHAPE, "kv_evict: bad shape");
  if (keep <= 0 || first < 0 || last < 0 || (long long)first + last > keep)
    return fail(Q27H_ERR_SHAPE, "kv_evict: keep >= 1 and 0 <= first + last <= keep");
  if (keep > n_ctx_out || keep > n_ctx) return fail(Q27H_ERR_SHAPE, "kv_evict: keep must be <= n_ctx and n_ctx_out");
  if (!kcache || !vcache || !acc || !pos0 || !kout || !vout || !acc_out || !ws)
    return fail(Q27H_ERR_ARG, "kv_evict: null pointer");
  if (!aligned16(kcache) || !aligned16(vcache) || !aligned16(kout) || !aligned16(vout) || !aligned16(ws))
    return fail(Q27H_ERR_ARG, "kv_evict: tensors need 16-byte alignment");
  if (!aligned4(acc) || !aligned4(acc_out) || !aligned4(kept) || !aligned4(pos0))
    return fail(Q27H_ERR_ARG, "kv_evict: acc, acc_out, kept and pos0 need 4-byte alignment");
  const size_t in = cache_bytes(nkvh, n_ctx, q8), out = cache_bytes(nkvh, n_ctx_out, q8);
  const size_t ain = (size_t)nkvh * n_ctx * 4, aout = (size_t)nkvh * n_ctx_out * 4;
  const bool in_place = kout == kcache && vout == vcache && acc_out == acc && n_ctx_out == n_ctx;
  const size_t need = q27h_kv_evict_ws_bytes(nkvh, n_ctx, keep, q8, in_place);
  const Bytes k = {kout, out}, v = {vout, out}, w = {acc_out, aout}, l = {kept, (size_t)nkvh * keep * 4}, work = {ws, need};
  if (overlaps(kcache, in, vcache, in) || outputs_overlap({k, v, w, l, work}, {{pos0, 4}}) ||
      (!in_place && outputs_overlap({k, v, w, l, work}, {{kcache, in}, {vcache, in}, {acc, ain}})))
    return fail(Q27H_ERR_ARG, "kv_evict: the outputs overlap each other or the inputs (all of them in place, or none)");
  if (ws_bytes < need) return fail(Q27H_ERR_ARG, "kv_evict: workspace too small");
  EvictArgs a = {};
  uint8_t* p = (uint8_t*)ws;
  auto take = [&](size_t n) {
    uint8_t* r = p;
    p += up256(n);
    return r;
  };
  a.kc = kcache, a.vc = vcache, a.acc = acc, a.pos0 = pos0;
  a.keep = keep, a.first = first, a.last = last, a.nkvh = nkvh, a.n_ctx = n_ctx, a.q8 = q8, a.segs = segs_of(n_ctx);
  a.hist = (int*)take((size_t)nkvh * 3 * kBins * 4);
  a.count = (int2*)take((size_t)nkvh * a.segs * 8);
  int* list = (int*)take((size_t)nkvh * keep * 4);
  a.kept = kept ? kept : list;
  const dim3 grid((unsigned)a.segs, (unsigned)nkvh), block(256);
  hipStream_t st = stream_of(s);
  if (n_ctx <= kLdsRows) {
    hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)nkvh), dim3(kListThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL(evict_clear_kernel, dim3((unsigned)(nkvh * 3 * kBins / 1024)), block, 0, st, a.hist);
    for (int pass = 0; pass < 3; pass++) hipLaunchKernelGGL(evict_hist_kernel, grid, block, 0, st, a, pass);
    hipLaunchKernelGGL(evict_count_kernel, grid, block, 0, st, a);
    hipLaunchKernelGGL(evict_list_kernel, grid, block, 0, st, a);
  }
  const int rows = (q8 ? 16 : 8) * kMoves;
  int chunks = (keep + rows - 1) / rows;
  const int most = 16 * kCUs / (2 * nkvh) < 1 ? 1 : 16 * kCUs / (2 * nkvh);
  chunks = chunks > most ? most : chunks;
  const dim3 mgrid((unsigned)chunks, (unsigned)nkvh, 2);
  a.ko = kout, a.vo = vout, a.acc_o = acc_out, a.n_out = n_ctx_out;
  if (!in_place) {
    hipLaunchKernelGGL(evict_move_kernel<OUT>, mgrid, block, 0, st, a);
  } else {
    a.k_aside = take(cache_bytes(nkvh, keep, q8)), a.v_aside = take(cache_bytes(nkvh, keep, q8));
    a.acc_aside = (float*)take((size_t)nkvh * keep * 4);
    hipLaunchKernelGGL(evict_move_kernel<ASIDE>, mgrid, block, 0, st, a);
    hipLaunchKernelGGL(evict_move_kernel<BACK>, mgrid, block, 0, st, a);
  }
  return check_launch("kv_evict");
}

extern "C" int q27h_kv_evict_pos(int* pos0, int* rdelta, int keep, q27h_stream_t s) {
  if (keep <= 0) return fail(Q27H_ERR_SHAPE, "kv_evict_pos: keep >= 1");
  if (!pos0) return fail(Q27H_ERR_ARG, "kv_evict_pos: null pointer");
  if (!aligned4(pos0) || !aligned4(rdelta)) return fail(Q27H_ERR_ARG, "kv_evict_pos: pos0 and rdelta need 4-byte alignment");
  if (outputs_overlap({{pos0, 4}, {rdelta, 4}}, {})) return fail(Q27H_ERR_ARG, "kv_evict_pos: pos0 and rdelta overlap");
  hipLaunchKernelGGL(evict_pos_kernel, dim3(1), dim3(1), 0, stream_of(s), pos0, rdelta, keep);
  return check_launch("kv_evict_pos");
}

extern "C" int q27h_kv_accept(void* const* caches, int n_caches, float* const* accs, int n_accs, const int* pos0, const int* path,
                              const int* n_path, int T, int nkvh, int n_ctx, int q8, q27h_stream_t s) {
  if (T < 0 || T > kMaxPath) return fail(Q27H_ERR_SHAPE, "kv_accept: T must be 0..64");
  if (n_caches < 0 || n_accs < 0 || nkvh <= 0 || nkvh > 65535 || n_ctx <= 0) return fail(Q27H_ERR_SHAPE, "kv_accept: bad shape");
  if (T == 0 || n_caches + n_accs == 0) return Q27H_OK;
  if (!pos0 || !path || !n_path || (n_caches && !caches) || (n_accs && !accs)) return fail(Q27H_ERR_ARG, "kv_accept: null pointer");
  for (int i = 0; i < n_caches; i++) {
    if (!caches[i]) return fail(Q27H_ERR_ARG, "kv_accept: null pointer");
    if (!aligned16(caches[i])) return fail(Q27H_ERR_ARG, "kv_accept: caches need 16-byte alignment");
  }
  for (int i = 0; i < n_accs; i++)
    if (!accs[i]) return fail(Q27H_ERR_ARG, "kv_accept: null pointer");
  bool odd = !aligned4(pos0) || !aligned4(path) || !aligned4(n_path);
  for (int i = 0; i < n_accs; i++) odd |= !aligned4(accs[i]);
  if (odd) return fail(Q27H_ERR_ARG, "kv_accept: weight arrays, pos0, path and n_path need 4-byte alignment");
  const size_t cb = cache_bytes(nkvh, n_ctx, q8), ab = (size_t)nkvh * n_ctx * 4;
  bool twice = false;  // a row moved twice, by workgroups that run at once
  for (int i = 0; i < n_caches; i++)
    for (int j = 0; j < i; j++) twice |= overlaps(caches[i], cb, caches[j], cb);
  for (int i = 0; i < n_accs; i++) {
    for (int j = 0; j < i; j++) twice |= overlaps(accs[i], ab, accs[j], ab);
    for (int j = 0; j < n_caches; j++) twice |= overlaps(accs[i], ab, caches[j], cb);
  }
  for (int i = 0; i < n_caches + n_accs; i++)
    twice |= outputs_overlap({i < n_caches ? Bytes{caches[i], cb} : Bytes{accs[i - n_caches], ab}},
                             {{pos0, 4}, {path, 4}, {n_path, 4}});  // path: *n_path entries, which may be one
  if (twice) return fail(Q27H_ERR_ARG, "kv_accept: caches or weight arrays overlap each other or another argument");
  for (int c = 0, w = 0; c < n_caches || w < n_accs;) {
    AcceptArgs a = {};
    a.pos0 = pos0, a.path = path, a.n_path = n_path, a.T = T, a.nkvh = nkvh, a.n_ctx = n_ctx, a.q8 = q8;
    int n_w = 0;
    while (c < n_caches && a.n_cache < kMaxPtrs) a.cache[a.n_cache++] = caches[c++];
    while (w < n_accs && n_w < kMaxPtrs) a.acc[n_w++] = accs[w++];
    hipLaunchKernelGGL(accept_kernel, dim3((unsigned)(a.n_cache + n_w), (unsigned)nkvh), dim3(256), 0, stream_of(s), a);
  }
  return check_launch("kv_accept");
}
