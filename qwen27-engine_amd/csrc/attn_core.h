// One wave's work on a tile of 32 rows of the K/V cache, shared by the kernels that read it (attn_tree.hip).
//
// Scores and outputs are float32 results of 16-bit matrix instructions. The cache's values enter them exactly: an f16
// cache as it is, a q8_0 cache as its codes (|code| <= 127 is exact in f16), with the f16 scales applied outside. The
// other operand (q, or the weight p times V's scale) is split in two f16 terms, x = hi + lo, cut off, each product exact
// in the instruction's float32 sum. So a term loses less than 2^-21 of itself (one f16 term would lose 2^-10 of it) or,
// where its second part is subnormal, 2^-24 at the scale it is brought to: 2^-38 of the largest value of its query row,
// 2^-36 of the row's largest weight (see Rows).
//
// mfma_f32_16x16x32_f16: lane l holds row (A) or column (B) l & 15 and the eight k = 8 (l >> 4) + e; of the result it
// holds column l & 15, rows 4 (l >> 4) + i. Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that a
// lane holds scores, weights and outputs of ONE query row n = l & 15: the softmax needs no exchange between lanes but
// the sum and the (rare) new maximum over its 4 lanes g = l >> 4, and the scores of a lane are already the second
// product's operand. Row numbers of the tile in a lane: 16 u + 4 g + i (u = 0, 1; i = 0..3), in the order e = 4 u + i.
#pragma once
#include "q27h_device.h"

namespace q27h {

constexpr int kHD = 256;       // head width
constexpr int kTileKeys = 32;  // cache rows of one wave's step

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// By value: __builtin_bit_cast of a vector's element, as an lvalue, would take the vector's first.
__device__ __forceinline__ h2 as_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ uint32_t pk_rtz(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// x - (float)h, exact for h = x rounded towards zero. The opaque -1 keeps the fma, which v_fma_mix_f32 does on the half
// itself; a plain difference is two instructions (measured: 64 fewer of 690 in a tile).
__device__ __forceinline__ float minus_half(float x, uint32_t pair, int hi) {
  const h2 v = as_h2(pair);
  float m1 = -1.0f;
  asm("" : "+s"(m1));
  return __builtin_fmaf((float)(hi ? v[1] : v[0]), m1, x);
}
__device__ __forceinline__ float half_of(uint32_t pair, int hi) {
  const h2 v = as_h2(pair);
  return (float)(hi ? v[1] : v[0]);
}
// Four int8 codes -> four halves of value code * 2^-9: byte ^ 0x80 = code + 128 = u, which as the low byte of a half is
// the subnormal u 2^-24; fma(u 2^-24, 2^15, -2^-2) = (u - 128) 2^-9, exact. ev = codes 0, 2; od = codes 1, 3.
// BIAS 8: bytes of codes 0 .. 15 of (code - 8), the same without the sign's turn.
template <int BIAS = 128>
__device__ __forceinline__ void codes_to_half(uint32_t x, uint32_t& ev, uint32_t& od) {
  constexpr _Float16 kM = (_Float16)(-0x1p-9f * BIAS);
  const h2 k = {(_Float16)32768.0f, (_Float16)32768.0f}, m = {kM, kM};
  if (BIAS == 128) x ^= 0x80808080u;
  const h2 a = __builtin_bit_cast(h2, x & 0x00ff00ffu);
  const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0u, x, 0x0c030c01u));
  ev = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(a, k, m));
  od = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, k, m));
}
// Eight codes in two dwords -> the operand of eight halves; the order of the eight is 0, 2, 1, 3, 4, 6, 5, 7.
template <int BIAS = 128>
__device__ __forceinline__ h8 codes8(uint32_t x, uint32_t y) {
  uint32_t r[4];
  codes_to_half<BIAS>(x, r[0], r[1]);
  codes_to_half<BIAS>(y, r[2], r[3]);
  return __builtin_bit_cast(h8, (u4){r[0], r[1], r[2], r[3]});
}

// The scheduler's order for a step of a pipeline over the 8 blocks: four matrix instructions, N vector ones behind each.
template <int N>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, N, 0);
  }
}

// Where a K or V cache of one kv head lies.
struct KvHead {
  const uint8_t* rows;   // q8: int8 [n_ctx][256]; else f16 [n_ctx][256]
  const uint8_t* scale;  // q8: f16 [n_ctx][8]
};
template <bool Q8>
__device__ __forceinline__ KvHead kv_head(const void* cache, int kh, int nkvh, int n_ctx) {
  KvHead h;
  h.rows = (const uint8_t*)cache + (size_t)kh * n_ctx * (Q8 ? kHD : 2 * kHD);
  h.scale = (const uint8_t*)cache + (size_t)nkvh * n_ctx * kHD + (size_t)kh * n_ctx * 16;
  return h;
}

// ---------------------------------------------------------------- queries
// LDS image of 16 query rows: [hi, lo][b = 32-dim block][lane] of 16 bytes, and per row the factor that takes a score from
// the operands' units to log2 units. A row is scaled by the power of two that brings its largest value into [2^14, 2^15)
// before the split: neither very large nor very small queries leave f16's range, and its small values, which large ones
// of K may meet, have all of it below them.
struct QTile {
  alignas(16) uint32_t v[2][8][64][4];
  float c[16];
};

// All WAVES waves of the workgroup. Row r (0 .. 16 TILES - 1) is `row_ptr(r)` (nullptr: zeros). q8 caches: the eight
// values of a lane are stored in the order of codes8, and the factor carries codes8's 2^-9. A wave requests up to 8 rows
// before it works on the first: one round trip to memory instead of one a row (attn_weights of 32 tokens, 20001 rows:
// 84 -> 67 us).
template <bool Q8, int WAVES, int TILES, typename F>
__device__ __forceinline__ void load_queries(QTile* im, float mult, F row_ptr) {
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
  constexpr int kRows = (TILES * 16 + WAVES - 1) / WAVES, kBatch = kRows < 8 ? kRows : 8;
#pragma unroll 1
  for (int r0 = 0; r0 < kRows; r0 += kBatch) {
    float4 in[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      const int r = w + (r0 + k) * WAVES;
      const float* src = r < TILES * 16 ? row_ptr(r) : nullptr;
      in[k] = src ? ld4(src + 4 * l) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      const int r = w + (r0 + k) * WAVES;
      if (r >= TILES * 16) break;
      float x[4] = {in[k].x * mult, in[k].y * mult, in[k].z * mult, in[k].w * mult};
      float a = __builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])),
                                __builtin_fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3])));
      a = __builtin_fmaxf(a, lane_xor<1>(a));
      a = __builtin_fmaxf(a, lane_xor<2>(a));
      a = __builtin_fmaxf(a, lane_xor<7>(a));
      a = __builtin_fmaxf(a, lane_xor<8>(a));
      a = __builtin_fmaxf(a, lane_xor<16>(a));
      a = __builtin_fmaxf(a, lane_xor32(a));
      int e = (int)((__builtin_bit_cast(uint32_t, a) >> 23) & 255) - 127 - 14;
      e = e < -124 ? -124 : e;  // a zero row keeps that (its scores are 0); inf and NaN stay what they are
      const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] *= down;
      const int o[4] = {0, Q8 ? 2 : 1, Q8 ? 1 : 2, 3};
      const int b = l >> 3, slot = ((l >> 1) & 3) * 16 + (r & 15), at = (l & 1) * 2;
      const uint32_t h0 = pk_rtz(x[o[0]], x[o[1]]), h1 = pk_rtz(x[o[2]], x[o[3]]);
      const uint32_t l0 = pk_rtz(minus_half(x[o[0]], h0, 0), minus_half(x[o[1]], h0, 1));
      const uint32_t l1 = pk_rtz(minus_half(x[o[2]], h1, 0), minus_half(x[o[3]], h1, 1));
      *(u2*)&im[r >> 4].v[0][b][slot][at] = (u2){h0, h1};
      *(u2*)&im[r >> 4].v[1][b][slot][at] = (u2){l0, l1};
      if (l == 0) im[r >> 4].c[r & 15] = __builtin_bit_cast(float, (uint32_t)(127 + e + (Q8 ? 9 : 0)) << 23);
    }
  }
}

// ---------------------------------------------------------------- 32 rows of K or V
// Rows of a tile are addressed from its first row j0 (the same in the whole wave). TAIL: only `left` rows of the tile
// exist; a row behind them reads the last one (it is hidden, and must not be read outside the cache).
template <bool TAIL>
__device__ __forceinline__ int tile_row(int j, int left) {
  return TAIL ? (j < left ? j : left - 1) : j;
}

// q8: rows of codes as they lie, 16 bytes a lane (row 4 r + g, bytes 16 n ..), and four of the 256 scales (row l >> 1,
// blocks 4 (l & 1) .. + 3). Both go through LDS: the codes to be regrouped (K: 8 bytes of a row per lane, V: 8 rows of a
// column), the scales so that a lane's registers hold 4 and not the 64 it uses.
struct QRows {
  u4 x[8];
  u2 s;
};
// One wave's LDS: 272 bytes a row of codes (4 banks on), the upper 16 rows 128 bytes (32 banks) on: the 32 lanes that read
// together touch every bank once, for K (16 rows, two 8-byte pieces) as for V (two lane groups, 8 rows of 16 bytes).
// K's codes are consumed before V's are staged in their place. Then the scales of K and of V: halves [block b][32 rows],
// four rows in the order 0, 2, 1, 3 of codes8.
constexpr int kRow = 272, kUpper = 16 * kRow + 128, kCodes = kUpper + 16 * kRow;
constexpr int kScales = 8 * 64;
struct WaveLds {
  alignas(16) uint8_t codes[kCodes];
  alignas(16) uint8_t ks[kScales], vs[kScales];
  alignas(16) float vf[kTileKeys];  // V's scales are stored as d / f, f the row's own power of two above them
};

// TAIL: scales of rows that do not exist are 0: whatever the memory behind the last row holds, NaN included, must not meet
// a weight of 0 in the product.
template <bool TAIL>
__device__ __forceinline__ void load_rows(QRows& t, const KvHead& h, int j0, int left) {
  const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const uint8_t* rows = h.rows + (size_t)j0 * kHD;
#pragma unroll
  for (int r = 0; r < 8; r++) {
    if (TAIL) t.x[r] = *(const u4*)(rows + (unsigned)(tile_row<TAIL>(4 * r + g, left) * kHD + 16 * n));
    else t.x[r] = *(const u4*)(rows + (r >> 2) * 16 * kHD + (unsigned)(g * kHD + 16 * n) + (r & 3) * 4 * kHD);
  }
  t.s = *(const u2*)(h.scale + (size_t)j0 * 16 + (unsigned)(tile_row<TAIL>(l >> 1, left) * 16 + 8 * (l & 1)));
  if (TAIL && (l >> 1) >= left) t.s = (u2){0u, 0u};
}
__device__ __forceinline__ void put_scales(u2 s, uint8_t* scales) {
  const int l = threadIdx.x & 63, r = l >> 1;
  uint16_t* p = (uint16_t*)scales + 4 * (l & 1) * 32 + ((r & ~3) | (r & 1) << 1 | (r >> 1 & 1));
  p[0] = (uint16_t)s.x;
  p[32] = (uint16_t)(s.x >> 16);
  p[64] = (uint16_t)s.y;
  p[96] = (uint16_t)(s.y >> 16);
}
// V's: brought to |d / f| <= 1 by the power of two f above the finite scales of the row's 8 blocks, f beside them (0
// where none is above 0: such a row adds zeros, or NaN, and leaves the unit alone). f meets the weight in float32, and
// d / f is a half without loss unless the block's scale is below 2^-14 of f; then it is off by less than 2^-24 of f.
__device__ __forceinline__ float exp2i(uint32_t e) { return __builtin_bit_cast(float, e << 23); }
__device__ __forceinline__ void put_value_scales(u2 s, uint8_t* scales, float* factors) {
  const int l = threadIdx.x & 63;
  float x[4], m = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[i] = half_of(i < 2 ? s.x : s.y, i & 1);
    const bool finite = __builtin_fabsf(x[i]) < 65536.0f;
    m = finite ? __builtin_fmaxf(m, __builtin_fabsf(x[i])) : m;
  }
  m = __builtin_fmaxf(m, lane_xor<1>(m));
  const uint32_t e = __builtin_bit_cast(uint32_t, m) >> 23;  // 2^(e - 127) <= m < 2^(e - 126); 0 for m = 0
  const float down = exp2i(253u - e);
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = e ? x[i] * down : x[i];  // m = 0: zeros, or values that are not finite
  put_scales((u2){pk_rtz(x[0], x[1]), pk_rtz(x[2], x[3])}, scales);
  if (!(l & 1)) factors[l >> 1] = e ? exp2i(e + 1) : 0.0f;
}
__device__ __forceinline__ void stage_codes(const QRows& t, WaveLds& w) {
  const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
#pragma unroll
  for (int r = 0; r < 8; r++)
    *(u4*)(w.codes + (r >= 4 ? kUpper + (4 * (r - 4) + g) * kRow : (4 * r + g) * kRow) + 16 * n) = t.x[r];
}
__device__ __forceinline__ void stage_keys(const QRows& t, WaveLds& w) {
  stage_codes(t, w);
  put_scales(t.s, w.ks);
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ void stage_values(const QRows& t, WaveLds& w) {
  stage_codes(t, w);
  put_value_scales(t.s, w.vs, w.vf);
  __builtin_amdgcn_wave_barrier();
}
// Scales of block b of the lane's rows 16 u + 4 g + i: rows i = 0, 2 in x, 1, 3 in y.
__device__ __forceinline__ u2 scales_of(const uint8_t* scales, int b, int u) {
  const int g = (threadIdx.x & 63) >> 4;
  return *(const u2*)(scales + b * 64 + 32 * u + 8 * g);
}

// f16: V as halves 8 n .. + 7 and 128 + 8 n .. + 7 of the lane's rows 16 u + 4 g + i, in registers. K goes from memory to LDS
// without passing registers (16 KB a tile and wave): as operand loads a lane would read its own row, 16 rows for every 16
// lanes, and the vector cache takes a cycle for each (1280 a tile, which bound attn_blocks: 650 us for 1027 tokens of 32
// blocks; 400 us so). A row of 512 bytes lies in LDS as 32 pieces of 16, piece c at c ^ (row & 15), so that the
// operand reads, the same piece of 16 rows, touch every bank once.
struct HValues {
  u4 x[8][2];
};
struct HKeysLds {
  alignas(16) uint8_t k[kTileKeys * 2 * kHD];
};
template <bool TAIL>
__device__ __forceinline__ void request_keys(HKeysLds& w, const KvHead& h, int j0, int left) {
  const int l = threadIdx.x & 63, up = l >> 5;
  int c = (l & 31) ^ up;
  asm volatile("" : "+v"(c));  // the 16 offsets are formed for each tile: kept over the loop they would take 16 registers
  const uint8_t* rows = h.rows + (size_t)j0 * (2 * kHD);
#pragma unroll TAIL ? 2 : kTileKeys / 2
  for (int r = 0; r < kTileKeys / 2; r++) {  // rows 2 r and 2 r + 1
    const uint8_t* p = rows + (unsigned)(tile_row<TAIL>(2 * r + up, left) * (2 * kHD) + (c ^ (2 * r & 14)) * 16);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)p,
                                     (__attribute__((address_space(3))) uint32_t*)(w.k + r * 4 * kHD), 16, 0, 0);
  }
}
// Waits until the wave's K tile has arrived while at most NEWER loads that were issued behind it have not (they return in
// order), and keeps the reads of it behind that.
template <int NEWER>
__device__ __forceinline__ void keys_there() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((NEWER & 15) | (NEWER >> 4) << 14 | 0x0f70);  // vmcnt(NEWER)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
constexpr int kValueLoads = 16;  // loads of load_rows(HValues)
template <bool TAIL>  // rows that do not exist are zeros, as the scales above
__device__ __forceinline__ void load_rows(HValues& t, const KvHead& h, int j0, int left) {
  const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const uint8_t* rows = h.rows + (size_t)j0 * (2 * kHD);
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int j = 16 * (e >> 2) + 4 * g + (e & 3);
    const uint8_t* p = TAIL ? rows + (unsigned)(tile_row<TAIL>(j, left) * (2 * kHD) + 16 * n)
                            : rows + (e >> 2) * 32 * kHD + (unsigned)(8 * g * kHD + 16 * n) + (e & 3) * 2 * kHD;
    t.x[e][0] = *(const u4*)p;
    t.x[e][1] = *(const u4*)(p + kHD);
    if (TAIL && j >= left) t.x[e][0] = t.x[e][1] = (u4){0u, 0u, 0u, 0u};
  }
}
// A wave's query rows as operands in registers, from their LDS image.
struct QRegs {
  h8 hi[8], lo[8];
  __device__ __forceinline__ h8 low(int b) const { return lo[b]; }
};
// The same with the second terms left in LDS, where 32 registers more would spill.
struct QHalf {
  h8 hi[8];
  const uint32_t (*lo)[64][4];
  __device__ __forceinline__ h8 low(int b) const { return *(const h8*)lo[b][threadIdx.x & 63]; }
};
__device__ __forceinline__ void take_queries(QRegs& q, const QTile& im) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int b = 0; b < 8; b++) q.hi[b] = *(const h8*)im.v[0][b][l], q.lo[b] = *(const h8*)im.v[1][b][l];
}

// Scores in the operands' units: s[rt][u][i] of tile row 16 u + 4 g + i and query row n of im[rt]. q8: `w` holds the
// staged codes and scales. The blocks are a pipeline (see interleave): a wave has only one other to hide latencies behind.
template <int RT>
__device__ __forceinline__ void scores(const WaveLds& w, const QTile* im, f4 (&s)[RT][2]) {
  const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int rt = 0; rt < RT; rt++) s[rt][0] = s[rt][1] = zero;
  const uint8_t* row = w.codes + n * kRow + 8 * g;
  u2 x[2][2], ks[3][2];
  h8 k[2][2];
  f4 c[2][RT][2];
  auto ask = [&](int b) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      x[b & 1][u] = *(const u2*)(row + kUpper * u + 32 * b);
      ks[b % 3][u] = scales_of(w.ks, b, u);
    }
  };
  auto turn = [&](int b) {
#pragma unroll
    for (int u = 0; u < 2; u++) k[b & 1][u] = codes8(x[b & 1][u].x, x[b & 1][u].y);
  };
  auto scale = [&](int b) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int i = 0; i < 4; i++)
          s[rt][u][i] = __builtin_fmaf(half_of(ks[b % 3][u][i & 1], i >> 1), c[b & 1][rt][u][i], s[rt][u][i]);
        asm("" : "+v"(s[rt][u]));  // formed here: sunk to their first use, the eight blocks' products would pile up
      }
  };
  // a step per block: its products, the scaling of the block before, the next block's codes turned, the one after's read
  h8 q[2][RT][2];
  auto ask_q = [&](int b) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++) q[b & 1][rt][0] = *(const h8*)im[rt].v[0][b][l], q[b & 1][rt][1] = *(const h8*)im[rt].v[1][b][l];
  };
  ask(0);
  ask_q(0);
  turn(0);
  ask(1);
#pragma unroll
  for (int b = 0; b < 8; b++) {
    __builtin_amdgcn_sched_barrier(0);  // block by block: all eight at once would not fit the registers
    if (b < 7) ask_q(b + 1);
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
#pragma unroll
      for (int u = 0; u < 2; u++) c[b & 1][rt][u] = mfma16(k[b & 1][u], q[b & 1][rt][1], zero);
#pragma unroll
      for (int u = 0; u < 2; u++) c[b & 1][rt][u] = mfma16(k[b & 1][u], q[b & 1][rt][0], c[b & 1][rt][u]);
    }
    if (b) scale(b - 1);
    if (b < 7) turn(b + 1);
    if (b < 6) ask(b + 2);
    if (RT == 1) interleave<7>();
  }
  scale(7);
}
template <int RT, typename Q>
__device__ __forceinline__ void scores(const HKeysLds& w, const Q (&q)[RT], f4 (&s)[RT][2]) {
  const int l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f4 lo[RT][2];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) s[rt][0] = s[rt][1] = lo[rt][0] = lo[rt][1] = zero;
  h8 k[2][2];
  auto ask = [&](int b) {
#pragma unroll
    for (int u = 0; u < 2; u++) k[b & 1][u] = *(const h8*)(w.k + (16 * u + n) * 2 * kHD + ((4 * b + g) ^ n) * 16);
  };
  ask(0);
#pragma unroll
  for (int b = 0; b < 8; b++) {
    if (b < 7) ask(b + 1);
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
      const h8 ql = q[rt].low(b);  // there by the time the products with the first terms are issued
#pragma unroll
      for (int u = 0; u < 2; u++) s[rt][u] = mfma16(k[b & 1][u], q[rt].hi[b], s[rt][u]);
#pragma unroll
      for (int u = 0; u < 2; u++) lo[rt][u] = mfma16(k[b & 1][u], ql, lo[rt][u]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int rt = 0; rt < RT; rt++) s[rt][0] += lo[rt][0], s[rt][1] += lo[rt][1];
}

// Which rows of a tile a query row sees: every one before n, and row n0 + t where bit t of `tree` is set (rows at or
// behind `end` are none).
struct Vis {
  int n;    // rows [0, n) are seen by all
  int n0;   // first drafted row (may lie outside the cache)
  int end;  // one past the last row that exists
};
// A hidden row's score becomes AS.
constexpr uint32_t kMinusInf = 0xff800000u;
constexpr uint32_t kHidden = 0xffffffffu;  // a NaN that no product gives: told from every score, -inf and NaN among them
template <int RT, uint32_t AS>
__device__ __forceinline__ void hide(f4 (&s)[RT][2], const Vis& vis, const uint64_t (&tree)[RT], int j0) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int j = j0 + 16 * u + 4 * g + i;
      const unsigned d = (unsigned)(j - vis.n0);
#pragma unroll
      for (int rt = 0; rt < RT; rt++) {
        // | and not ||: eight branches a lane cost more than the shift. And hipcc (clang 22) lost the score of the first of
        // them in attn_weights' kernels: it keeps the score's register for the result, sets it to -inf where the first
        // condition is false, and emits nothing under the mask of the lanes where the second is true.
        const bool seen = (j < vis.n) | ((j < vis.end) & (d < 64u) & (bool)((tree[rt] >> (d & 63u)) & 1));
        s[rt][u][i] = seen ? s[rt][u][i] : __builtin_bit_cast(float, AS);
      }
    }
}

// ---------------------------------------------------------------- online softmax
// State of 16 query rows in a wave: lane (n, g) holds of row n the reference M (the same in its four lanes), its own part
// of the sum l and 64 outputs. Weights are p = 2^(s - M). M is not the maximum itself: it is only moved when p would leave
// f16's range, that is when s - M > 15, and then to s - 12, so that the largest weights lie near 2^12, where two f16 terms
// hold 22 bits, and small ones down to 2^-36 of them are still in range. q8: a row's weight enters the product times its
// V row's factor f, as p f / unit, and the outputs are in units of `unit`, a power of two that is moved as M is: up, when
// the quotient would pass 2^15, and then to where the largest lies between 2^12 and 2^13. When M moves, the unit goes
// down with the weights. So neither a row of large values and little weight, nor one whose weight has shrunk since,
// coarsens the others. O, l and M of different waves and workgroups are joined by M alone.
struct Rows {
  f4 o[16];
  float m, l, c, unit, want;  // want: what the outputs are in units of, once M has moved and until split8() scales them
};
constexpr float kLeastUnit = 0x1p-80f;  // f and the quotient by it are in range

template <bool Q8>
__device__ __forceinline__ void rows_init(Rows& st, const QTile& im) {
#pragma unroll
  for (int i = 0; i < 16; i++) st.o[i] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
  st.m = -3.0e38f;
  st.l = 0.0f;
  st.c = im.c[threadIdx.x & 15];
  st.unit = st.want = kLeastUnit;
}

__device__ __forceinline__ float power_below(float x) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0x7f800000u);
}
// What the outputs have to be multiplied by in the end: the unit, and 2^9 for codes8's 2^-9.
template <bool Q8>
__device__ __forceinline__ float unit_of(const Rows& st) {
  return Q8 ? st.unit * 512.0f : 1.0f;
}
// p[u][i] from the scores, with the reference moved where it has to be (maxima pass over NaN). HIDDEN: the weight of a
// hidden row (kHidden) is -0: the sign tells it from a row that is seen with a weight of 0, whose infinities make NaN.
template <bool Q8, bool HIDDEN>
__device__ __forceinline__ void weights(Rows& st, f4 (&s)[2]) {
  float mx = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(s[0][0], s[0][1]), __builtin_fmaxf(s[0][2], s[0][3])),
                             __builtin_fmaxf(__builtin_fmaxf(s[1][0], s[1][1]), __builtin_fmaxf(s[1][2], s[1][3])));
  mx *= st.c;
  if (__any(mx - st.m > 15.0f)) {
    mx = __builtin_fmaxf(mx, lane_xor<16>(mx));
    mx = __builtin_fmaxf(mx, lane_xor32(mx));
    const float m1 = mx - st.m > 15.0f ? mx - 12.0f : st.m;  // by its own row alone: its bits are the same beside any others
    const float a = __builtin_amdgcn_exp2f(st.m - m1);
    st.m = m1;
    st.l *= a;
    if (Q8) {
      st.want *= a;
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) st.o[i] *= a;
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float x = s[u][i], p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, st.c, -st.m));
      s[u][i] = HIDDEN && __builtin_bit_cast(uint32_t, x) == kHidden ? -0.0f : p;
      sum += s[u][i];
    }
  st.l += sum;
}

// Weights as operands: two f16 terms, p = hi + lo, each the rest cut off to f16. f16 caches: rows in order.
__device__ __forceinline__ void split(const f4 (&p)[2], u4& hi, u4& lo) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float w0 = p[e >> 1][2 * (e & 1)], w1 = p[e >> 1][2 * (e & 1) + 1];
    hi[e] = pk_rtz(w0, w1);
    lo[e] = pk_rtz(minus_half(w0, hi[e], 0), minus_half(w1, hi[e], 1));
  }
}

// q8: the same of p f / unit, pairs of rows (0, 2), (1, 3) of u = 0, then of u = 1, as codes8 orders them; factors: the tile's
// f, in LDS. The unit is moved where p f would pass 2^15 of it, or where M has moved, and the outputs are scaled for both at
// once (64 tokens, 65536 rows: 284 -> 279 us).
__device__ __forceinline__ void split8(Rows& st, const f4 (&p)[2], const float* factors, u4& hi, u4& lo) {
  f4 w[2];
  float mx = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    w[u] = p[u] * *(const f4*)(factors + 16 * u + 4 * ((threadIdx.x & 63) >> 4));
#pragma unroll
    for (int i = 0; i < 4; i++) mx = __builtin_fmaxf(mx, w[u][i]);
  }
  if (__any((mx > st.unit * 0x1p15f) | (st.want < st.unit))) {
    mx = __builtin_fmaxf(mx, lane_xor<16>(mx));
    mx = __builtin_fmaxf(mx, lane_xor32(mx));
    const bool move = (mx > st.unit * 0x1p15f) | (st.want < st.unit);
    const float to = move ? power_below(__builtin_fmaxf(__builtin_fmaxf(st.want, kLeastUnit), mx * 0x1p-12f)) : st.unit;
    const float a = __builtin_amdgcn_ldexpf(st.want, 127 - (int)(__builtin_bit_cast(uint32_t, to) >> 23));  // want / to
    st.unit = st.want = to;
#pragma unroll
    for (int i = 0; i < 16; i++) st.o[i] *= a;
  }
  const float inv = __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, st.unit));  // 1 / unit
#pragma unroll
  for (int u = 0; u < 2; u++) w[u] *= inv;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float w0 = w[e >> 1][e & 1], w1 = w[e >> 1][(e & 1) + 2];
    hi[e] = pk_rtz(w0, w1);
    lo[e] = pk_rtz(minus_half(w0, hi[e], 0), minus_half(w1, hi[e], 1));
  }
}
// Times the stored scales d <= 1 of a block of V: hi' = hi d, rounded; the fma gives what that lost, exactly (11 by 11 bits
// leave at most 11 below the first 11), and lo' = lo d + that. HIDDEN: a hidden row (weight -0) is left out whatever its
// scale is (0 times infinity is no part of the sum).
template <bool HIDDEN>
__device__ __forceinline__ void weigh(const u4& ph, const u4& pl, const u2 (&vs)[2], u4& hi, u4& lo) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    uint32_t x = vs[e >> 1][e & 1];
    if (HIDDEN) x &= ~(((ph[e] >> 15) & 0x10001u) * 0xffffu);
    const h2 d = as_h2(x), p = as_h2(ph[e]);
    const h2 h = p * d;
    const h2 lost = __builtin_elementwise_fma(p, d, -h);
    hi[e] = __builtin_bit_cast(uint32_t, h);
    lo[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(as_h2(pl[e]), d, lost));
  }
}

// O += P V. Output o[i][j]: q8: dim 16 i + 4 g + j; f16: dim 128 (i >> 3) + 8 (4 g + j) + (i & 7).
// q8: `w` holds the staged codes and scales. TAIL: some rows are hidden, see weigh(). BIAS: the codes', see codes_to_half.
template <bool TAIL, int BIAS = 128>
__device__ __forceinline__ void accumulate(Rows& st, const f4 (&p)[2], const WaveLds& w) {
  const int l = threadIdx.x & 63, j = l & 15, g = l >> 4;
  // the transposing read: in a group of 16 lanes, lane j gives the address of 8 bytes of row j >> 1 and gets column j of
  // the 8 rows by 16 columns
  const uint8_t* base = w.codes + ((j >> 1) >= 4 ? kUpper + (4 * g + (j >> 1) - 4) * kRow : (4 * g + (j >> 1)) * kRow) + 8 * (j & 1);
  typedef int v2i __attribute__((ext_vector_type(2)));
  v2i c[2][2];
  u2 vs[2][2];
  h8 v[2][2];
  u4 ph, pl, hi[2], lo[2];
  split8(st, p, w.vf, ph, pl);
  auto ask = [&](int b) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      c[b & 1][h] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(base + 32 * b + 16 * h));
      vs[b & 1][h] = scales_of(w.vs, b, h);
    }
  };
  auto turn = [&](int b) {
#pragma unroll
    for (int h = 0; h < 2; h++) v[b & 1][h] = codes8<BIAS>((uint32_t)c[b & 1][h].x, (uint32_t)c[b & 1][h].y);
    weigh<TAIL>(ph, pl, vs[b & 1], hi[b & 1], lo[b & 1]);
  };
  ask(0);
  turn(0);
  ask(1);
#pragma unroll
  for (int b = 0; b < 8; b++) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < 2; h++) st.o[2 * b + h] = mfma16(v[b & 1][h], __builtin_bit_cast(h8, lo[b & 1]), st.o[2 * b + h]);
#pragma unroll
    for (int h = 0; h < 2; h++) st.o[2 * b + h] = mfma16(v[b & 1][h], __builtin_bit_cast(h8, hi[b & 1]), st.o[2 * b + h]);
    if (b < 7) {
      turn(b + 1);
      if (b < 6) ask(b + 2);
      interleave<8>();
    }
  }
}
__device__ __forceinline__ void accumulate(Rows& st, const f4 (&p)[2], const HValues& v) {
  u4 hi, lo;
  split(p, hi, lo);
#pragma unroll
  for (int i = 0; i < 16; i++) {
    u4 x;
#pragma unroll
    for (int e = 0; e < 4; e++)
      x[e] = __builtin_amdgcn_perm(v.x[2 * e + 1][i >> 3][(i & 7) >> 1], v.x[2 * e][i >> 3][(i & 7) >> 1],
                                   i & 1 ? 0x07060302u : 0x05040100u);
    st.o[i] = mfma16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, lo), st.o[i]);
    st.o[i] = mfma16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, hi), st.o[i]);
  }
}

// f16, tiles with hidden rows: infinities and NaN of a drafted row's values must reach the rows that see it and no
// other, but 0 times infinity in the product would reach all. They are taken out of the tile here and added one by one.
// (A tile without them, practically every one, pays the test.) `w`: 2 KB of this wave's LDS.
__device__ __forceinline__ uint32_t finite_halves(uint32_t x, uint32_t& odd) {
  // a half is infinite or NaN where its exponent field is all ones: adding one to the field then carries into the sign
  const uint32_t c = ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
  odd |= c;
  return x & ~((c >> 15) * 0xffffu);
}
__device__ __forceinline__ void accumulate_tail(Rows& st, const f4 (&p)[2], HValues& v, const KvHead& h, int j0, int left,
                                                float* w) {
  uint32_t odd = 0;
#pragma unroll
  for (int e = 0; e < 8; e++)
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
      for (int c = 0; c < 4; c++) v.x[e][q][c] = finite_halves(v.x[e][q][c], odd);
  accumulate(st, p, v);
  if (!__any(odd != 0)) return;
  const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int e = 0; e < 8; e++) w[(16 * (e >> 2) + 4 * g + (e & 3)) * 16 + n] = p[e >> 2][e & 3];  // [row][n]
  __builtin_amdgcn_wave_barrier();
#pragma unroll 1
  for (int j = 0; j < left && j < kTileKeys; j++) {
    const float wt = w[j * 16 + n];
    const u4* row = (const u4*)(h.rows + (size_t)(j0 + j) * (2 * kHD));
#pragma unroll
    for (int q = 0; q < 8; q++) {  // dims 128 (q >> 2) + 8 (4 g + (q & 3)) + 0 .. 7
      const u4 x = row[16 * (q >> 2) + 4 * g + (q & 3)];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float f = half_of(x[e >> 1], e & 1);
        const bool add = (__builtin_bit_cast(uint32_t, f) & 0x7f800000u) == 0x7f800000u && !__builtin_signbit(wt);
        st.o[8 * (q >> 2) + e][q & 3] += add ? wt * f : 0.0f;
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
}

}  // namespace q27h
