// Which blocks of 64 cache rows a token's sparse attention (attn_blocks) reads: bounds of every block, kept beside the
// cache (kv_block_bounds), and the choice by a score of the query against them (attn_select).
//
// A block's bounds are, per channel, the least and the greatest K value of its rows, in int8 with one scale for the block:
// d = amax / 127, code = roundf(x * (1 / d)). The query head is quantized the same way. The score of a head is
// sum_c max(q_c lo_c, q_c hi_c) = sum_c max(q_c, 0) hi_c + min(q_c, 0) lo_c, an upper bound of its products with the
// block's rows up to the rounding to int8; a whole number below 2^24, computed exactly. The block's score for the kv head is
// max over the heads of float(sum) * dq, times d of the block: every rounding is fixed, so the choice is the same
// whatever the order of the work, and equal scores go to the lower block.
#include "pick.h"
#include "q27h_device.h"
#include "q27h_internal.h"

namespace q27h {
namespace {

constexpr int kHD = 256;
constexpr int kBlockRows = 64;
constexpr int kMaxBlocks = 16000;  // blocks of a context that attn_select takes (its keys lie in 64 KB of LDS)

typedef int v4i __attribute__((ext_vector_type(4)));

// Blocks kept for n_ctx rows: lo int8 [nkvh][nblk][256], hi the same, d f32 [nkvh][nblk].
__host__ __device__ inline int blocks_of(int n_ctx) { return (n_ctx + kBlockRows - 1) / kBlockRows; }

__device__ __forceinline__ float wave_max(float a) {
  a = __builtin_fmaxf(a, lane_xor<1>(a));
  a = __builtin_fmaxf(a, lane_xor<2>(a));
  a = __builtin_fmaxf(a, lane_xor<7>(a));
  a = __builtin_fmaxf(a, lane_xor<8>(a));
  a = __builtin_fmaxf(a, lane_xor<16>(a));
  return __builtin_fmaxf(a, lane_xor32(a));
}
__device__ __forceinline__ bool not_finite(float x) {
  return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) == 0x7f800000u;
}
// The scale of values up to amax, and its reciprocal; both 0 below 2^-100 (every code is then 0).
__device__ __forceinline__ float scale_of(float amax, float& inv) {
  const float d = amax >= 0x1p-100f ? div127(amax) : 0.0f;
  inv = d != 0.0f ? 1.0f / d : 0.0f;
  return d;
}
__device__ __forceinline__ int code_of(float x, float inv) { return (int)__builtin_roundf(x * inv); }

// One workgroup per block. A thread takes 16 bytes of every 16th (f16: 8th) row, all requested before the first is used: one
// round trip to memory for the block; then thread c joins channel c's parts. (One token: 7.1 us with 4 bytes a lane and two
// round trips, 4.0 us so.)
template <bool Q8>
__global__ void __launch_bounds__(kHD) block_bounds_kernel(const uint8_t* __restrict__ kcache, const int* __restrict__ dpos0,
                                                           int T, int nkvh, int n_ctx, int8_t* __restrict__ lo,
                                                           int8_t* __restrict__ hi, float* __restrict__ kd) {
  constexpr int kLanes = Q8 ? 16 : 32, kChans = kHD / kLanes, kGroups = kHD / kLanes, kRows = kBlockRows / kGroups;
  __shared__ float s_lo[kGroups][kHD], s_hi[kGroups][kHD], s_max[kHD / 64];
  __shared__ int s_odd[kHD / 64];
  const int kh = blockIdx.y, tid = threadIdx.x, c = tid % kLanes, rg = tid / kLanes;
  const long long p0 = *dpos0, e = p0 + T;
  const int begin = p0 < 0 ? 0 : p0 > n_ctx ? n_ctx : (int)p0, end = e < 0 ? 0 : e > n_ctx ? n_ctx : (int)e;
  if (end <= begin) return;
  const int b = begin / kBlockRows + blockIdx.x, nblk = blocks_of(n_ctx);
  const int r0 = b * kBlockRows, r1 = r0 + kBlockRows < end ? r0 + kBlockRows : end;
  if (r0 >= end) return;
  uint4 x[kRows];
  uint16_t d[kRows];
#pragma unroll
  for (int k = 0; k < kRows; k++) {  // a row behind the last one that exists: the block's first again
    const int r = r0 + rg + k * kGroups;
    const size_t row = (size_t)kh * n_ctx + (r < r1 ? r : r0);
    x[k] = *(const uint4*)(kcache + (row * kLanes + c) * 16);
    if (Q8) d[k] = *(const uint16_t*)(kcache + (size_t)nkvh * n_ctx * kHD + row * 16 + 2 * (c >> 1));
  }
  loads_issued();
  float a[kChans], z[kChans];
  bool odd = false;
#pragma unroll
  for (int i = 0; i < kChans; i++) a[i] = __builtin_huge_valf(), z[i] = -__builtin_huge_valf();
#pragma unroll
  for (int k = 0; k < kRows; k++) {
    const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
    for (int i = 0; i < kChans; i++) {
      const float v = Q8 ? (float)(int8_t)(w[i >> 2] >> (8 * (i & 3))) * h2f_bits(d[k]) : h2f_bits((uint16_t)(w[(i >> 1) & 3] >> (16 * (i & 1))));
      odd |= not_finite(v);
      a[i] = __builtin_fminf(a[i], v);
      z[i] = __builtin_fmaxf(z[i], v);
    }
  }
#pragma unroll
  for (int i = 0; i < kChans; i += 4) {
    *(float4*)&s_lo[rg][c * kChans + i] = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
    *(float4*)&s_hi[rg][c * kChans + i] = make_float4(z[i], z[i + 1], z[i + 2], z[i + 3]);
  }
  const int any = __any(odd);
  if ((tid & 63) == 0) s_odd[tid >> 6] = any;
  __syncthreads();
  float least = s_lo[0][tid], most = s_hi[0][tid];
#pragma unroll
  for (int k = 1; k < kGroups; k++) {
    least = __builtin_fminf(least, s_lo[k][tid]);
    most = __builtin_fmaxf(most, s_hi[k][tid]);
  }
  const float m = wave_max(__builtin_fmaxf(__builtin_fabsf(least), __builtin_fabsf(most)));
  if ((tid & 63) == 0) s_max[tid >> 6] = m;
  __syncthreads();
  const float amax = __builtin_fmaxf(__builtin_fmaxf(s_max[0], s_max[1]), __builtin_fmaxf(s_max[2], s_max[3]));
  const bool bad = s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3];  // an infinity or NaN: the block scores +inf and is read
  float inv;
  const float dk = scale_of(bad ? 0.0f : amax, inv);
  const size_t at = (size_t)kh * nblk + b;
  lo[at * kHD + tid] = (int8_t)(bad ? 0 : code_of(least, inv));
  hi[at * kHD + tid] = (int8_t)(bad ? 0 : code_of(most, inv));
  if (tid == 0) kd[at] = bad ? __builtin_huge_valf() : dk;
}

// Scores: one int8 matrix instruction (16 query rows x 16 blocks x 64 channels) per 64 channels of hi and of lo. A token's
// heads are padded to gp = 4, 8 or 16 rows, so that 16 / gp tokens fill a row tile and the maximum over a token's heads
// stays inside a lane and its neighbours 16 and 32 lanes on. A workgroup quantizes the queries of kRowTiles row tiles
// into LDS and walks its blocks, 16 to a wave.
constexpr int kRowTiles = 4;
__global__ void __launch_bounds__(256) select_score_kernel(const float* __restrict__ qn, const int8_t* __restrict__ lo,
                                                           const int8_t* __restrict__ hi, const float* __restrict__ kd,
                                                           const int* __restrict__ dpos0, int T, int nqh, int nkvh, int n_ctx,
                                                           int gp, int splits, float* __restrict__ score) {
  // [row tile][positive, negative part][64-channel step][lane] of 16 codes
  __shared__ __attribute__((aligned(16))) uint8_t s_q[kRowTiles][2][4][64][16];
  __shared__ float s_d[kRowTiles * 16];
  const int group = nqh / nkvh, per_tile = 16 / gp, per_wg = kRowTiles * per_tile;
  const int kh = blockIdx.x % nkvh, split = (blockIdx.x / nkvh) % splits, t0 = (int)(blockIdx.x / nkvh / splits) * per_wg;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, n = l & 15, g = l >> 4, nblk = blocks_of(n_ctx);
  // blocks up to the one of the group's last token
  const long long last = (long long)*dpos0 + (t0 + per_wg < T ? t0 + per_wg : T) - 1;
  const int nb = last < 0 ? 0 : last >= n_ctx ? nblk : (int)(last / kBlockRows) + 1;
  const int tiles = (nb + 15) / 16, per = (tiles + splits - 1) / splits;
  const int b1 = split * per + per < tiles ? split * per + per : tiles;
  if (split * per >= b1) return;
  // this lane's block (column) of 16, requested ahead of the queries and then of the products before
  v4i vh[4], vl[4];
  float d;
  auto ask = [&](int bt) {
    const int b = bt * 16 + n, bb = b < nb ? b : nb - 1;
    const int8_t* ph = hi + ((size_t)kh * nblk + bb) * kHD + 16 * g;
    const int8_t* pl = lo + ((size_t)kh * nblk + bb) * kHD + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; i++) vh[i] = *(const v4i*)(ph + 64 * i), vl[i] = *(const v4i*)(pl + 64 * i);
    d = kd[(size_t)kh * nblk + bb];
  };
  ask(split * per + w);
  loads_issued();
  const int used = (T - t0 + per_tile - 1) / per_tile < kRowTiles ? (T - t0 + per_tile - 1) / per_tile : kRowTiles;
  for (int rt = 0; rt < used; rt++) {
    float4 in[4];  // the wave's four rows of the tile, requested together
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = rt * 16 + w + 4 * k, t = t0 + r / gp, h = r % gp;
      in[k] = t < T && h < group ? ld4(qn + ((size_t)t * nqh + kh * group + h) * kHD + 4 * l) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = w + 4 * k;
      const float x[4] = {in[k].x, in[k].y, in[k].z, in[k].w};
      const float amax = wave_max(__builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])),
                                                  __builtin_fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3]))));
      const bool bad = __any(not_finite(x[0]) || not_finite(x[1]) || not_finite(x[2]) || not_finite(x[3]));
      float inv;
      const float d = scale_of(bad ? 0.0f : amax, inv);
      int p[4], m[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int q = bad ? 0 : code_of(x[c], inv);
        p[c] = q > 0 ? q : 0;
        m[c] = q < 0 ? q : 0;
      }
      const int slot = ((l >> 2) & 3) * 16 + r, at = (l & 3) * 4;
      *(uint32_t*)&s_q[rt][0][l >> 4][slot][at] = pack4_i8(p[0], p[1], p[2], p[3]);
      *(uint32_t*)&s_q[rt][1][l >> 4][slot][at] = pack4_i8(m[0], m[1], m[2], m[3]);
      if (l == 0) s_d[rt * 16 + r] = d;
    }
  }
  __syncthreads();
  for (int bt = split * per + w; bt < b1; bt += 4) {
    const int b = bt * 16 + n;
    v4i wh[4], wl[4];
#pragma unroll
    for (int i = 0; i < 4; i++) wh[i] = vh[i], wl[i] = vl[i];
    const float db = d;
    if (bt + 4 < b1) ask(bt + 4);
    for (int rt = 0; rt < used; rt++) {
      v4i c = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const v4i*)s_q[rt][0][i][l], wh[i], c, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const v4i*)s_q[rt][1][i][l], wl[i], c, 0, 0, 0);
      float m = -__builtin_huge_valf();
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 4 * g + i;
        if ((r & (gp - 1)) < group) m = __builtin_fmaxf(m, (float)c[i] * s_d[rt * 16 + r]);
      }
      if (gp >= 8) m = __builtin_fmaxf(m, lane_xor<16>(m));
      if (gp >= 16) m = __builtin_fmaxf(m, lane_xor32(m));
      const int t = t0 + rt * per_tile + 4 * g / gp;
      if (b < nb && t < T && (4 * g & (gp - 1)) == 0)
        score[((size_t)t * nkvh + kh) * nblk + b] = db == __builtin_huge_valf() ? db : m * db;
    }
  }
}

// One workgroup per (token, kv head). Always taken are the first `first` blocks and the last `last` ones up to the token's
// own; of the others, keys in LDS, the need-th largest is found by digits of key - (least key), so that the first
// digit already tells them apart (digits of the key itself would put most scores, which share their exponents, in one
// histogram bin, and its counter's updates one behind another). It ends as soon as a bin is taken whole. Then a thread
// counts and lists a stretch of consecutive blocks of its own. A digit has as many values as there are threads: 256, or 1024
// while the workgroups leave compute units free. (2345 blocks: 18 us with the key's own digits and a workgroup sum for every
// 256 blocks, 8 us so with 256 threads, 6.8 us with 1024.)
template <int THREADS>
__global__ void __launch_bounds__(THREADS) select_pick_kernel(const float* __restrict__ score, const int* __restrict__ dpos0, int nkvh,
                                                          int n_ctx, int nsel, int first, int last, int* __restrict__ idx) {
  extern __shared__ uint32_t s_key[];
  constexpr int kWaves = THREADS / 64, kBits = THREADS == 256 ? 8 : 10;
  static_assert(THREADS == 1 << kBits && kMaxBlocks < 1 << 15);
  __shared__ int s_hist[THREADS], s_scan[kWaves], s_pick[3];
  __shared__ uint32_t s_end[2 * kWaves];
  const int t = blockIdx.x / nkvh, tid = threadIdx.x, w = tid >> 6, nblk = blocks_of(n_ctx);
  const long long pos = (long long)*dpos0 + t;
  const int nb = pos < 0 ? 0 : pos >= n_ctx ? nblk : (int)(pos / kBlockRows) + 1;
  int* out = idx + (size_t)blockIdx.x * nsel;
  if (nb <= nsel) {
    for (int i = tid; i < nsel; i += THREADS) out[i] = i < nb ? i : -1;
    return;
  }
  const float* row = score + (size_t)blockIdx.x * nblk;
  const int b0 = first, b1 = nb - last;  // the blocks chosen from
  uint32_t least = ~0u, most = 0u;
#pragma unroll 4
  for (int b = b0 + tid; b < b1; b += THREADS) {
    const uint32_t k = order_key(row[b]);
    s_key[b] = k;
    least = least < k ? least : k;
    most = most > k ? most : k;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t x = __shfl_xor(least, d), y = __shfl_xor(most, d);
    least = least < x ? least : x;
    most = most > y ? most : y;
  }
  if ((tid & 63) == 0) s_end[w] = least, s_end[kWaves + w] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    least = least < s_end[i] ? least : s_end[i];
    most = most > s_end[kWaves + i] ? most : s_end[kWaves + i];
  }
  // `need` blocks are still to be taken among the keys whose digits above `shift` are those of `prefix`
  int need = nsel - first - last, shift = need && least < most ? 32 - __builtin_clz(most - least) : 0;
  uint32_t prefix = need ? 0u : ~0u;
  auto upper = [](uint32_t k, int by) { return (uint32_t)((uint64_t)k >> by); };
  while (shift > 0) {
    const int next = shift > kBits ? shift - kBits : 0;
    s_hist[tid] = 0;
    __syncthreads();
    for (int b = b0 + tid; b < b1; b += THREADS) {
      const uint32_t k = s_key[b] - least;
      if (upper(k, shift) == upper(prefix, shift)) atomicAdd(&s_hist[(k >> next) & ((1u << (shift - next)) - 1u)], 1);
    }
    __syncthreads();
    const int bin = THREADS - 1 - tid, h = s_hist[bin];
    int total;
    const int above = scan_waves<kWaves>(h, s_scan, total);
    if (above < need && need <= above + h) s_pick[0] = bin, s_pick[1] = need - above, s_pick[2] = h;
    __syncthreads();
    prefix |= (uint32_t)s_pick[0] << next;
    need = s_pick[1];
    shift = next;
    if (need == s_pick[2]) break;  // every key with these digits is taken
    __syncthreads();
  }
  __syncthreads();
  // taken: keys above the digits found; of those with them the first `need`
  const int per = (b1 - b0 + THREADS - 1) / THREADS, c0 = b0 + tid * per, c1 = c0 + per < b1 ? c0 + per : b1;
  const uint32_t p = upper(prefix, shift);
  int mine = 0;  // above << 16 | equal: each below 2^15
  for (int b = c0; b < c1; b++) {
    const uint32_t k = upper(s_key[b] - least, shift);
    mine += (k > p ? 1 << 16 : 0) + (k == p);
  }
  int total;
  const int before = scan_waves<kWaves>(mine, s_scan, total);
  int at = before >> 16, rank = before & 0xffff;
  at += first + (rank < need ? rank : need);
  for (int b = c0; b < c1; b++) {
    const uint32_t k = upper(s_key[b] - least, shift);
    const bool take = k > p || (k == p && rank < need);
    rank += k == p;
    if (take) out[at++] = b;
  }
  for (int i = tid; i < first; i += THREADS) out[i] = i;
  for (int i = tid; i < last; i += THREADS) out[nsel - last + i] = b1 + i;
}

int padded_group(int group) { return group <= 4 ? 4 : group <= 8 ? 8 : 16; }

}  // namespace
}  // namespace q27h

using namespace q27h;

extern "C" size_t q27h_kv_block_bytes(int nkvh, int n_ctx) {
  if (nkvh <= 0 || n_ctx <= 0) return 0;
  return (size_t)nkvh * blocks_of(n_ctx) * (2 * kHD + 4);
}

extern "C" int q27h_kv_block_bounds(const void* kcache, const int* pos0, int T, int nkvh, int n_ctx, int q8, void* kb,
                                    q27h_stream_t s) {
  if (T < 0 || nkvh <= 0 || nkvh > 65535 || n_ctx <= 0) return fail(Q27H_ERR_SHAPE, "kv_block_bounds: bad shape");
  if (T == 0) return Q27H_OK;
  if (!kcache || !pos0 || !kb) return fail(Q27H_ERR_ARG, "kv_block_bounds: null pointer");
  if (!aligned16(kcache) || !aligned16(kb)) return fail(Q27H_ERR_ARG, "kv_block_bounds: tensors need 16-byte alignment");
  if (!aligned4(pos0)) return fail(Q27H_ERR_ARG, "kv_block_bounds: pos0 needs 4-byte alignment");
  if (outputs_overlap({{kb, q27h_kv_block_bytes(nkvh, n_ctx)}}, {{kcache, q27h_kv_cache_bytes(nkvh, n_ctx, q8)}, {pos0, 4}}))
    return fail(Q27H_ERR_ARG, "kv_block_bounds: kb overlaps another argument");
  const int nblk = blocks_of(n_ctx);
  const long touched = ((long)T + kBlockRows - 1) / kBlockRows + 1;
  int8_t* lo = (int8_t*)kb;
  int8_t* hi = lo + (size_t)nkvh * nblk * kHD;
  hipLaunchKernelGGL((q8 ? block_bounds_kernel<true> : block_bounds_kernel<false>),
                     dim3((unsigned)(touched < nblk ? touched : nblk), (unsigned)nkvh), dim3(kHD), 0, stream_of(s),
                     (const uint8_t*)kcache, pos0, T, nkvh, n_ctx, lo, hi, (float*)(hi + (size_t)nkvh * nblk * kHD));
  return check_launch("kv_block_bounds");
}

extern "C" size_t q27h_attn_select_ws_bytes(int T, int nkvh, int n_ctx) {
  if (T <= 0 || nkvh <= 0 || n_ctx <= 0) return 0;
  return (size_t)T * nkvh * blocks_of(n_ctx) * sizeof(float);
}

extern "C" int q27h_attn_select(const float* qn, const void* kb, const int* pos0, int T, int nqh, int nkvh, int n_ctx, int nsel,
                                int first, int last, int* idx, void* ws, size_t ws_bytes, q27h_stream_t s) {
  if (T < 0 || nkvh <= 0 || nqh <= 0 || nqh % nkvh || nqh / nkvh > 16 || n_ctx <= 0 || nsel <= 0)
    return fail(Q27H_ERR_SHAPE, "attn_select: bad shape (at most 16 query heads per kv head)");
  if (first < 0 || last < 1 || (long long)first + last > nsel)
    return fail(Q27H_ERR_SHAPE, "attn_select: first >= 0, last >= 1 and first + last <= nsel");
  const int nblk = blocks_of(n_ctx);
  if (nblk > kMaxBlocks) return fail(Q27H_ERR_SHAPE, "attn_select: n_ctx must be <= 1024000");
  if ((long long)T * nkvh > 0x7fffffffLL / 128) return fail(Q27H_ERR_SHAPE, "attn_select: T too large");
  if (T == 0) return Q27H_OK;
  if (!qn || !kb || !pos0 || !idx || !ws) return fail(Q27H_ERR_ARG, "attn_select: null pointer");
  if (!aligned16(qn) || !aligned16(kb) || !aligned4(ws)) return fail(Q27H_ERR_ARG, "attn_select: tensors need 16-byte alignment");
  if (!aligned4(idx) || !aligned4(pos0)) return fail(Q27H_ERR_ARG, "attn_select: idx and pos0 need 4-byte alignment");
  const size_t need = q27h_attn_select_ws_bytes(T, nkvh, n_ctx);
  if (ws_bytes < need) return fail(Q27H_ERR_ARG, "attn_select: workspace too small");
  if (outputs_overlap({{idx, (size_t)T * nkvh * nsel * 4}, {ws, need}},
                      {{qn, (size_t)T * nqh * kHD * 4}, {kb, q27h_kv_block_bytes(nkvh, n_ctx)}, {pos0, 4}}))
    return fail(Q27H_ERR_ARG, "attn_select: idx or ws overlaps another argument");
  const int8_t* lo = (const int8_t*)kb;
  const int8_t* hi = lo + (size_t)nkvh * nblk * kHD;
  const float* kd = (const float*)(hi + (size_t)nkvh * nblk * kHD);
  const int gp = padded_group(nqh / nkvh), per_wg = kRowTiles * 16 / gp;
  const int tg = (T + per_wg - 1) / per_wg, most = (nblk + 63) / 64;  // 4 waves of 16 blocks
  int splits = (int)(2L * kCUs / ((long)tg * nkvh));
  splits = splits > most ? most : splits < 1 ? 1 : splits;
  hipLaunchKernelGGL(select_score_kernel, dim3((unsigned)((long)tg * nkvh * splits)), dim3(256), 0, stream_of(s), qn, lo, hi, kd,
                     pos0, T, nqh, nkvh, n_ctx, gp, splits, (float*)ws);
  const bool few = T * nkvh <= kCUs && nblk <= kMaxBlocks - 1024;  // the larger digits' counts take 3 KB of the 64
  hipLaunchKernelGGL((few ? select_pick_kernel<1024> : select_pick_kernel<256>), dim3((unsigned)(T * nkvh)), dim3(few ? 1024 : 256),
                     (size_t)nblk * 4, stream_of(s), (const float*)ws, pos0, nkvh, n_ctx, nsel, first, last, idx);
  return check_launch("attn_select");
}
