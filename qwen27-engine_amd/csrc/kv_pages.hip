// A K/V cache in pages: its handle's checks, its rows read back as values (kv_pages_read), and the rows of accepted paths moved
// to their places (kv_accept_paged).
//
// Reading back is a copy that widens: rows x nkvh x (144 to 512 bytes in, 512 or 1024 out) for each of K and V, no arithmetic
// but one product a value, so it is bound by HBM. A piece of work is kChunk rows of one head; the sequences' pieces are laid
// end to end and cut in equal parts (share_of), since sequences are of any length.
#include <hip/hip_bfloat16.h>

#include <type_traits>

#include "paged.h"

namespace q27h {

int check_pages(const q27h_kv_pages* kv, const char* what) {
  auto bad = [&](int code, const char* why) { return fail(code, std::string(what) + why); };
  if (!kv) return bad(Q27H_ERR_ARG, ": null handle of pages");
  if (kv->type != Q27H_KV_F16 && kv->type != Q27H_KV_Q8 && kv->type != Q27H_KV_Q8_Q4)
    return bad(Q27H_ERR_SHAPE, ": unknown type of cache");
  if (kv->page_rows < 32 || kv->page_rows > 65536 || (kv->page_rows & (kv->page_rows - 1)))
    return bad(Q27H_ERR_SHAPE, ": the rows of a page must be a power of two, 32 to 65536");
  if (kv->nkvh <= 0 || kv->nkvh > 4096 || kv->n_seqs < 0 || kv->n_pages < 0 || kv->max_pages < 0 ||
      (long long)kv->max_pages * kv->page_rows > 1 << 30)
    return bad(Q27H_ERR_SHAPE, ": bad sizes of the paged cache (at most 2^30 rows a sequence)");
  if ((kv->n_pages && (!kv->k || !kv->v)) || (kv->n_seqs && kv->max_pages && !kv->table))
    return bad(Q27H_ERR_ARG, ": null pointer in the handle of pages");
  if (!aligned16(kv->k) || !aligned16(kv->v) || !aligned4(kv->table))
    return bad(Q27H_ERR_ARG, ": pages need 16-byte alignment, their table 4-byte");
  return Q27H_OK;
}

Pages pages_of(const q27h_kv_pages* kv) {
  Pages p;
  p.k = (uint8_t*)kv->k, p.v = (uint8_t*)kv->v, p.table = kv->table;
  p.kb = q27h_kv_page_bytes(kv->nkvh, kv->page_rows, kv->type, 0), p.vb = q27h_kv_page_bytes(kv->nkvh, kv->page_rows, kv->type, 1);
  p.n_seqs = kv->n_seqs, p.max_pages = kv->max_pages, p.n_pages = kv->n_pages, p.nkvh = kv->nkvh, p.type = kv->type;
  p.shift = __builtin_ctz((unsigned)kv->page_rows);
  return p;
}

namespace {

constexpr int kChunk = 16;    // rows of a piece
constexpr int kBlocks = 16 * kCUs;

struct ReadArgs {
  Pages pg;
  const int *from, *count;
  void *kout, *vout;
  int n_out;
};

typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef uint32_t w2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

// Values as they are stored: 16 bytes a lane and store, so that the 16 lanes of a row write 256 bytes that lie together (a
// lane's values one behind the other in several stores would leave every cache line to be written in pieces: 8 sequences
// with 81250 rows in all, K in 8 bits and V in 4, to f16: 167 us, 112 so).
struct AsF32 {
  typedef float type;
  static constexpr int kN = 4;
  static __device__ __forceinline__ void put(float* p, const float (&x)[kN]) {
    __builtin_nontemporal_store((f4){x[0], x[1], x[2], x[3]}, (f4*)p);
  }
};
struct AsF16 {
  typedef uint16_t type;
  static constexpr int kN = 8;
  static __device__ __forceinline__ uint32_t bits(float x) { return f2h_bits(x); }
};
struct AsBf16 {
  typedef uint16_t type;
  static constexpr int kN = 8;
  static __device__ __forceinline__ uint32_t bits(float x) {  // to the nearest, ties to even; NaN stays one
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return x != x ? (b >> 16) | 0x40 : (b + 0x7fff + (b >> 16 & 1)) >> 16;
  }
};
template <typename OUT>
__device__ __forceinline__ void put(typename OUT::type* p, const float (&x)[OUT::kN]) {
  if constexpr (OUT::kN == 4) {
    OUT::put(p, x);
  } else {
    w4 y;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = OUT::bits(x[2 * i]) | OUT::bits(x[2 * i + 1]) << 16;
    __builtin_nontemporal_store(y, (w4*)p);
  }
}

// What a lane has of a row: N values from dim N l + 16 N i on, i < 16 / N. 16 lanes to a row.
template <int BITS, int N>
struct Piece {
  static constexpr int kStores = 16 / N, kWords = BITS == 4 ? N / 4 : N * BITS / 32;
  uint32_t x[kStores][kWords];
  uint16_t d[kStores];
  __device__ __forceinline__ void load(const uint8_t* page, size_t rows, size_t row, int l) {
#pragma unroll
    for (int i = 0; i < kStores; i++) {
      const int dim = N * l + 16 * N * i;
      // 4 bits: the low halves of bytes e .. of the block, or the high ones
      const uint8_t* p = page + row * (32 * BITS) + (BITS == 4 ? dim / 32 * 16 + (dim & 15) : dim * (BITS / 8));
      if constexpr (kWords == 1) x[i][0] = *(const uint32_t*)p;
      else if constexpr (kWords == 2) *(w2*)x[i] = *(const w2*)p;
      else *(w4*)x[i] = *(const w4*)p;
      if constexpr (BITS != 16) d[i] = *((const uint16_t*)(page + rows * (32 * BITS)) + row * 8 + dim / 32);
    }
  }
  __device__ __forceinline__ void values(int i, int l, float (&y)[N]) const {
    const int high = BITS == 4 ? (N * l + 16 * N * i) & 16 ? 4 : 0 : 0;
    float s = 0.0f;
    if constexpr (BITS != 16) s = h2f_bits(d[i]);
#pragma unroll
    for (int e = 0; e < N; e++) {
      if constexpr (BITS == 16) y[e] = h2f_bits((uint16_t)(x[i][e >> 1] >> 16 * (e & 1)));
      else if constexpr (BITS == 8) y[e] = (float)(int8_t)(x[i][e >> 2] >> 8 * (e & 3)) * s;
      else y[e] = (float)((int)((x[i][e >> 2] >> high) >> 8 * (e & 3) & 15u) - 8) * s;
    }
  }
};

// Work of unequal sequences in equal shares: cost(b) >= 0 of each sequence, laid end to end, is cut in `gridDim.x` parts.
// Gives every thread of the workgroup its part [x, end), the sequence that x lies in and where that one begins.
struct Share {
  int x, end, seq, start;
};
template <int THREADS, typename F>
__device__ __forceinline__ Share share_of(int n_seqs, F cost) {
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
  const int parts = (int)gridDim.x, per = (total + parts - 1) / parts;
  // a workgroup behind the last part: its product may pass 31 bits
  s.x = (long long)blockIdx.x * per < total ? (int)blockIdx.x * per : total;
  s.end = total - s.x < per ? total : s.x + per;
  if (before <= s.x && s.x < before + mine) {
    int at = before;
    for (int b = b0; b < b1; b++) {
      const int c = cost(b);
      if (at <= s.x && s.x < at + c) s_at[0] = b, s_at[1] = at;
      at += c;
    }
  }
  __syncthreads();
  s.x = __builtin_amdgcn_readfirstlane(s.x);
  s.end = __builtin_amdgcn_readfirstlane(s.end);
  s.seq = __builtin_amdgcn_readfirstlane(s_at[0]);
  s.start = __builtin_amdgcn_readfirstlane(s_at[1]);
  return s;
}

// A workgroup takes a chunk of 16 rows, K and V requested together, and then the next. Twice the rows in twice the loads,
// and half the workgroups, were slower (to f16: 112 us against 104). Rows of a page that is none of the cache's are zeros.
template <int KB, int VB, typename OUT>
__global__ void __launch_bounds__(256) kv_pages_read_kernel(ReadArgs a) {
  typedef typename OUT::type O;
  const int l = threadIdx.x & 15, r = threadIdx.x >> 4;
  auto rows_of = [&](int b) {
    const int n = a.count[b];
    return n < 0 ? 0 : n < a.n_out ? n : a.n_out;
  };
  Share sp = share_of<256>(a.pg.n_seqs, [&](int b) { return a.pg.nkvh * ((rows_of(b) + kChunk - 1) / kChunk); });
  const int n = 1 << a.pg.shift;
  while (sp.x < sp.end) {
    const int b = sp.seq, count = rows_of(b), chunks = (count + kChunk - 1) / kChunk;
    if (sp.x >= sp.start + a.pg.nkvh * chunks) {
      sp.start += a.pg.nkvh * chunks;
      sp.seq++;
      continue;
    }
    const int at = sp.x - sp.start, kh = at / chunks, i0 = (at - kh * chunks) * kChunk;
    sp.x++;
    const long long from = a.from ? a.from[b] : 0;
    constexpr int N = OUT::kN;
    Piece<KB, N> k;
    Piece<VB, N> v;
    const int i = i0 + r;
    if (i >= count) continue;
    const long long j = from + i, pi = j >> a.pg.shift;
    const int page = pi >= 0 && pi < a.pg.max_pages ? a.pg.table[(size_t)b * a.pg.max_pages + pi] : -1;
    const bool is = (unsigned)page < (unsigned)a.pg.n_pages;
    if (is) {
      const size_t rows = (size_t)a.pg.nkvh * n, row = (size_t)kh * n + (size_t)(j & (n - 1));
      if (a.kout) k.load(a.pg.k + (size_t)page * a.pg.kb, rows, row, l);
      if (a.vout) v.load(a.pg.v + (size_t)page * a.pg.vb, rows, row, l);
    }
    const size_t o = (((size_t)b * a.pg.nkvh + kh) * a.n_out + i) * kHeadDim + N * l;
    auto give = [&](const auto& x, void* out) {
      if (!out) return;
#pragma unroll
      for (int h = 0; h < 16 / N; h++) {
        float y[N];
        x.values(h, l, y);
#pragma unroll
        for (int e = 0; e < N; e++) y[e] = is ? y[e] : 0.0f;
        put<OUT>((O*)out + o + 16 * N * h, y);
      }
    };
    give(k, a.kout);
    give(v, a.vout);
  }
}

// kv_accept_paged: a workgroup for (sequence, kv head, K or V of a layer). Of a path that is a prefix of the drafts nothing moves,
// which is all that a chain's workgroups find out; otherwise all the rows that move are held in registers before the first
// is written, so a path in any order is right. At most 64 rows of 512 bytes each: bound by its round trips.
constexpr int kMostPath = 64, kMostPools = 64;
struct AcceptArgs {
  Pages pg;                   // of every layer, but for k and v
  uint8_t* pool[kMostPools];  // a layer's K, its V, the next one's K, ..
  const int *pos, *cu, *path, *n_path;
  int T;
};
__global__ void __launch_bounds__(256) kv_accept_paged_kernel(AcceptArgs a) {
  __shared__ long long s_from[kMostPath], s_to[kMostPath];  // row i of the path: rows of the pool, counted over its pages; -1: stays
  __shared__ int s_any;
  const int b = blockIdx.x, kh = blockIdx.y, tid = threadIdx.x, n = 1 << a.pg.shift;
  const bool v = blockIdx.z & 1;
  if (tid < 64) {
    const Tokens tk = tokens_of(a.cu, b, a.T, kMostPath);
    const int got = uniform_load(a.n_path + b), want = got < tk.nt ? got : tk.nt;
    const long long base = (long long)uniform_load(a.pos + b) - got;  // the sequence's rows before the batch
    const int p = tid < want ? a.path[tk.t0 + tid] : -1;
    const uint64_t good = __ballot(p >= 0 && p < tk.nt);
    const int len = good == ~0ull ? 64 : __builtin_ctzll(~good);  // the path ends at its first entry that is no token
    auto place = [&](long long j) {
      const long long i = j >> a.pg.shift;
      const int page = i >= 0 && i < a.pg.max_pages ? a.pg.table[(size_t)b * a.pg.max_pages + i] : -1;
      return (unsigned)page < (unsigned)a.pg.n_pages ? (long long)page << a.pg.shift | (j & (n - 1)) : -1ll;
    };
    long long from = -1, to = -1;
    if (tid < len && p != tid) from = place(base + p), to = place(base + tid);
    const bool moves = from >= 0 && to >= 0;
    s_from[tid] = moves ? from : -1;
    s_to[tid] = to;
    const uint64_t any = __ballot(moves);
    if (tid == 0) s_any = any != 0;
  }
  __syncthreads();
  if (!s_any) return;
  uint8_t* c = a.pool[blockIdx.z];
  const bool f16 = a.pg.type == Q27H_KV_F16;
  const int log = f16 ? 5 : v && a.pg.type == Q27H_KV_Q8_Q4 ? 3 : 4;  // 16 bytes a lane: the lanes of a row
  const int sub = tid & ((1 << log) - 1), step = 256 >> log;
  const size_t bytes = v ? a.pg.vb : a.pg.kb, row = (size_t)16 << log;
  auto codes = [&](long long j) {
    return (w4*)(c + (size_t)(j >> a.pg.shift) * bytes + ((size_t)kh * n + (size_t)(j & (n - 1))) * row + 16 * sub);
  };
  auto scales = [&](long long j) {
    return (w4*)(c + (size_t)(j >> a.pg.shift) * bytes + (size_t)a.pg.nkvh * n * row + ((size_t)kh * n + (size_t)(j & (n - 1))) * 16);
  };
  const bool has_d = !f16 && tid < kMostPath && s_from[tid & 63] >= 0;
  w4 x[8], d = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int i = k * step + (tid >> log);
    if (i < kMostPath && s_from[i & 63] >= 0) x[k] = *codes(s_from[i & 63]);
  }
  if (has_d) d = *scales(s_from[tid & 63]);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int i = k * step + (tid >> log);
    if (i < kMostPath && s_from[i & 63] >= 0) *codes(s_to[i & 63]) = x[k];
  }
  if (has_d) *scales(s_to[tid & 63]) = d;
}

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_kv_page_bytes(int nkvh, int page_rows, int type, int v) {
  if (nkvh <= 0 || page_rows <= 0 || type < Q27H_KV_F16 || type > Q27H_KV_Q8_Q4) return 0;
  return (size_t)nkvh * page_rows * kv_row_bytes(type, v != 0);
}

extern "C" int q27h_kv_pages_read(const q27h_kv_pages* kv, const int* from, const int* count, int n_out, int out_type, void* kout,
                                  void* vout, q27h_stream_t s) {
  if (const int bad = check_pages(kv, "kv_pages_read")) return bad;
  if (n_out < 0 || n_out > 1 << 30 || out_type < Q27H_F32 || out_type > Q27H_BF16)
    return fail(Q27H_ERR_SHAPE, "kv_pages_read: bad n_out or type of the values");
  if ((double)kv->n_seqs * kv->nkvh * ((n_out + kChunk - 1) / kChunk) > 2.0e9)
    return fail(Q27H_ERR_SHAPE, "kv_pages_read: too many rows in all");
  if (kv->n_seqs == 0 || n_out == 0 || (!kout && !vout)) return Q27H_OK;
  if (!count) return fail(Q27H_ERR_ARG, "kv_pages_read: null pointer");
  if (!aligned16(kout) || !aligned16(vout)) return fail(Q27H_ERR_ARG, "kv_pages_read: results need 16-byte alignment");
  if (!aligned4(from) || !aligned4(count)) return fail(Q27H_ERR_ARG, "kv_pages_read: from and count need 4-byte alignment");
  ReadArgs a = {pages_of(kv), from, count, kout, vout, n_out};
  const size_t B = (size_t)kv->n_seqs, ob = B * kv->nkvh * n_out * kHeadDim * (out_type == Q27H_F32 ? 4 : 2);
  if (outputs_overlap({{kout, ob}, {vout, ob}}, {{a.pg.k, a.pg.kb * kv->n_pages}, {a.pg.v, a.pg.vb * kv->n_pages},
                                                 {a.pg.table, B * kv->max_pages * 4}, {from, B * 4}, {count, B * 4}}))
    return fail(Q27H_ERR_ARG, "kv_pages_read: a result overlaps another argument");
  // never more workgroups than there can be pieces
  const double pieces = (double)B * kv->nkvh * ((n_out + kChunk - 1) / kChunk);
  const dim3 grid((unsigned)(pieces < kBlocks ? pieces : kBlocks)), block(256);
  auto launch = [&](auto f32, auto f16, auto bf16) {
    hipLaunchKernelGGL((out_type == Q27H_F32 ? f32 : out_type == Q27H_F16 ? f16 : bf16), grid, block, 0, stream_of(s), a);
  };
  if (kv->type == Q27H_KV_F16)
    launch(kv_pages_read_kernel<16, 16, AsF32>, kv_pages_read_kernel<16, 16, AsF16>, kv_pages_read_kernel<16, 16, AsBf16>);
  else if (kv->type == Q27H_KV_Q8)
    launch(kv_pages_read_kernel<8, 8, AsF32>, kv_pages_read_kernel<8, 8, AsF16>, kv_pages_read_kernel<8, 8, AsBf16>);
  else
    launch(kv_pages_read_kernel<8, 4, AsF32>, kv_pages_read_kernel<8, 4, AsF16>, kv_pages_read_kernel<8, 4, AsBf16>);
  return check_launch("kv_pages_read");
}

extern "C" int q27h_kv_accept_paged(const q27h_kv_pages* layers, int n_layers, const int* pos, const int* cu, const int* path,
                                    const int* n_path, int T, q27h_stream_t s) {
  if (T < 0 || n_layers < 0) return fail(Q27H_ERR_SHAPE, "kv_accept_paged: bad shape");
  if (n_layers == 0) return Q27H_OK;
  if (!layers) return fail(Q27H_ERR_ARG, "kv_accept_paged: null pointer");
  const q27h_kv_pages& one = layers[0];
  for (int i = 0; i < n_layers; i++) {
    const q27h_kv_pages& kv = layers[i];
    if (const int bad = check_pages(&kv, "kv_accept_paged")) return bad;
    if (kv.table != one.table || kv.n_seqs != one.n_seqs || kv.max_pages != one.max_pages || kv.n_pages != one.n_pages ||
        kv.nkvh != one.nkvh || kv.page_rows != one.page_rows || kv.type != one.type)
      return fail(Q27H_ERR_ARG, "kv_accept_paged: layers of different sizes, types or tables");
  }
  if ((long long)one.n_seqs * one.nkvh > 1 << 17) return fail(Q27H_ERR_SHAPE, "kv_accept_paged: too many sequences");
  if (T == 0 || one.n_seqs == 0) return Q27H_OK;
  if (!pos || !cu || !path || !n_path) return fail(Q27H_ERR_ARG, "kv_accept_paged: null pointer");
  if (!aligned4(pos) || !aligned4(cu) || !aligned4(path) || !aligned4(n_path))
    return fail(Q27H_ERR_ARG, "kv_accept_paged: pos, cu, path and n_path need 4-byte alignment");
  AcceptArgs a = {};
  a.pg = pages_of(&one), a.pos = pos, a.cu = cu, a.path = path, a.n_path = n_path, a.T = T;
  const size_t B = (size_t)one.n_seqs * 4, kb = a.pg.kb * one.n_pages, vb = a.pg.vb * one.n_pages;
  auto pool = [&](int i) { return i & 1 ? Bytes{layers[i >> 1].v, vb} : Bytes{layers[i >> 1].k, kb}; };
  bool twice = false;  // a row moved twice, by workgroups that run at once
  for (int i = 0; i < 2 * n_layers; i++) {
    const Bytes x = pool(i);
    for (int j = 0; j < i; j++) twice |= overlaps(x.p, x.n, pool(j).p, pool(j).n);
    twice |= outputs_overlap({x}, {{pos, B}, {cu, B + 4}, {path, (size_t)T * 4}, {n_path, B}, {one.table, B * one.max_pages}});
  }
  if (twice) return fail(Q27H_ERR_ARG, "kv_accept_paged: pages overlap each other or another argument");
  for (int i = 0; i < n_layers; i += kMostPools / 2) {
    const int n = n_layers - i < kMostPools / 2 ? n_layers - i : kMostPools / 2;
    for (int j = 0; j < n; j++) a.pool[2 * j] = (uint8_t*)layers[i + j].k, a.pool[2 * j + 1] = (uint8_t*)layers[i + j].v;
    hipLaunchKernelGGL(kv_accept_paged_kernel, dim3((unsigned)one.n_seqs, (unsigned)one.nkvh, (unsigned)(2 * n)), dim3(256), 0,
                       stream_of(s), a);
  }
  return check_launch("kv_accept_paged");
}
