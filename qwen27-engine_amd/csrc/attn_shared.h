// A tile of 32 cache rows shared by the waves of a workgroup, for more than 32 query rows: each wave holds one row tile (16
// query rows, in registers) and works on the same cache rows, which the workgroup reads once, turns into operands of the
// matrix instruction once, and keeps in LDS, two tiles in turn. Alone, a wave spends 320 instructions of about 690 on
// turning a q8_0 tile's codes into halves, and reads the 16 KB (q8) or 32 KB (f16) of every tile itself; together 8 waves
// do that once. What remains per wave and tile: 64 matrix instructions, 32 KB of LDS reads.
//
// The arithmetic is that of attn_core.h, with the same bounds. Output o[i][j] of lane (n, g) is dim 16 i + 4 g + j.
#pragma once
#include "attn_core.h"

namespace q27h {

struct SharedTile {
  // operand of rows 16 u + n, dims 32 b + 8 g ..: [8 u + b][16 g + (n ^ ((4 b + g) & 15))]
  alignas(16) uint32_t k[16][64][4];
  // operand of dims 16 i + m, rows 16 u + 4 g + 0 .. 3 at 8 u: [i][16 g + (m ^ i)]. The exchanges (here and in k)
  // spread a wave's writes over the banks: it writes one row's piece of many b, g, or one m of many i
  alignas(16) uint32_t v[16][64][4];
  alignas(16) uint8_t ks[kScales], vs[kScales];
  alignas(16) float vf[kTileKeys];
};

// What a thread holds of the next tile on its way to LDS. 256 threads carry K (and 64 of them its scales), 256 carry V;
// with 4 waves each thread has both parts, with 8 one. Rows behind the last one that exists are read from the last one.
template <bool Q8, int WAVES>
struct Staged {
  static constexpr int kV = WAVES == 4 ? 4 : 0;
  u4 x[kV + 4];  // K from 0, V from kV on
  u2 s;          // q8: scales (K in one wave, V in another)
};
template <int WAVES>
__device__ __forceinline__ bool carries_k() {
  return WAVES == 4 || threadIdx.x < 256;
}
template <int WAVES>
__device__ __forceinline__ bool carries_v() {
  return WAVES == 4 || threadIdx.x >= 256;
}

template <bool Q8, int WAVES, bool K, bool V>
__device__ __forceinline__ void request(Staged<Q8, WAVES>& t, const KvHead& kc, const KvHead& vc, int j0, int left) {
  const int q = threadIdx.x & 255, l = q & 63, n = l & 15, g = l >> 4;
  const int f = __builtin_amdgcn_readfirstlane(q >> 6);
  constexpr int kBytes = Q8 ? kHD : 2 * kHD;
  auto at = [&](const uint8_t* base, int row, int byte) {
    return base + (size_t)j0 * kBytes + (unsigned)((row < left ? row : left - 1) * kBytes + byte);
  };
  if (K && carries_k<WAVES>()) {
#pragma unroll
    for (int j = 0; j < (Q8 ? 2 : 4); j++) {
      if constexpr (Q8) t.x[j] = *(const u4*)at(kc.rows, 16 * j + (q >> 4), 16 * n);
      else t.x[j] = *(const u4*)at(kc.rows, 8 * j + (q >> 5), 16 * (q & 31));
    }
  }
  if (V && carries_v<WAVES>()) {
    if (!Q8 || f < 2) {
      const int u = Q8 ? f : f >> 1, g4 = Q8 ? g : (q >> 5) & 3, c = Q8 ? n : q & 31;
#pragma unroll
      for (int e = 0; e < 4; e++) t.x[t.kV + e] = *(const u4*)at(vc.rows, 16 * u + 4 * g4 + e, 16 * c);
    }
  }
  if constexpr (Q8) {
    if ((f == 2 && K && carries_v<WAVES>()) || (K && !V && f == 2) || (f == 3 && V && carries_v<WAVES>())) {
      const uint8_t* sc = (f == 2 ? kc.scale : vc.scale) + (size_t)j0 * 16;
      const int r = l >> 1;
      t.s = *(const u2*)(sc + (unsigned)((r < left ? r : left - 1) * 16 + 8 * (l & 1)));
      if (r >= left) t.s = (u2){0u, 0u};
    }
  }
}

// Staged rows into LDS as operands. part: some rows of the tile are hidden from some query rows, or do not exist; then f16
// values that are not finite are taken out of V, and *s_odd is set.
template <bool Q8, int WAVES, bool K, bool V>
__device__ __forceinline__ void stage(Staged<Q8, WAVES>& t, SharedTile& sh, bool part, int left, int* s_odd) {
  const int q = threadIdx.x & 255, l = q & 63, n = l & 15, g = l >> 4;
  const int f = __builtin_amdgcn_readfirstlane(q >> 6);
  if (K && carries_k<WAVES>()) {
#pragma unroll
    for (int j = 0; j < (Q8 ? 2 : 4); j++) {
      if constexpr (Q8) {
        // 16 codes: dims 16 n .. of row 16 j + (q >> 4): the 8-dim operands 2 (n & 1) and the next of block n >> 1
        const int b = n >> 1, g0 = 2 * (n & 1), r = q >> 4;
        *(h8*)sh.k[8 * j + b][16 * g0 + (r ^ ((4 * b + g0) & 15))] = codes8(t.x[j].x, t.x[j].y);
        *(h8*)sh.k[8 * j + b][16 * g0 + 16 + (r ^ ((4 * b + g0 + 1) & 15))] = codes8(t.x[j].z, t.x[j].w);
      } else {
        const int c = q & 31, r = 8 * j + (q >> 5);  // dims 8 c .. of row r
        *(u4*)sh.k[8 * (r >> 4) + (c >> 2)][16 * (c & 3) + ((r & 15) ^ (c & 15))] = t.x[j];
      }
    }
  }
  if (V && carries_v<WAVES>()) {
    if constexpr (Q8) {
      if (f < 2) {  // 4 rows x 16 dims: 4 x 4 codes turned at a time
#pragma unroll
        for (int d = 0; d < 4; d++) {
          const uint32_t a = t.x[t.kV + 0][d], b = t.x[t.kV + 1][d], c = t.x[t.kV + 2][d], e = t.x[t.kV + 3][d];
          const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
          const uint32_t ce0 = __builtin_amdgcn_perm(e, c, 0x05010400u), ce1 = __builtin_amdgcn_perm(e, c, 0x07030602u);
          const uint32_t x[4] = {__builtin_amdgcn_perm(ce0, ab0, 0x05040100u), __builtin_amdgcn_perm(ce0, ab0, 0x07060302u),
                                 __builtin_amdgcn_perm(ce1, ab1, 0x05040100u), __builtin_amdgcn_perm(ce1, ab1, 0x07060302u)};
#pragma unroll
          for (int m = 0; m < 4; m++) {
            uint32_t ev, od;
            codes_to_half(x[m], ev, od);
            *(u2*)&sh.v[n][16 * g + ((4 * d + m) ^ n)][2 * f] = (u2){ev, od};
          }
        }
      }
    } else {
      const int u = f >> 1, g4 = (q >> 5) & 3, i = (q & 31) >> 1, half = q & 1;
      if (part) {
        uint32_t odd = 0;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int d = 0; d < 4; d++) {
            uint32_t x = finite_halves(t.x[t.kV + e][d], odd);
            t.x[t.kV + e][d] = 16 * u + 4 * g4 + e < left ? x : 0u;
          }
        if (odd) *s_odd = 1;  // a row that does not exist repeats the last one: nothing is lost by marking it
      }
#pragma unroll
      for (int d = 0; d < 8; d++) {
        const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
        *(u2*)&sh.v[i][16 * g4 + ((8 * half + d) ^ i)][2 * u] =
            (u2){__builtin_amdgcn_perm(t.x[t.kV + 1][d >> 1], t.x[t.kV + 0][d >> 1], sel), __builtin_amdgcn_perm(t.x[t.kV + 3][d >> 1], t.x[t.kV + 2][d >> 1], sel)};
      }
    }
  }
  if constexpr (Q8) {
    if ((f == 2 && K && carries_v<WAVES>()) || (K && !V && f == 2)) put_scales(t.s, sh.ks);
    if (f == 3 && V && carries_v<WAVES>()) put_value_scales(t.s, sh.vs, sh.vf);
  }
}

// Both products walk the 8 blocks of 32 dims as a pipeline, a step per block: its four matrix instructions (no two
// neighbours depend on each other), the vector work that feeds the next block's or finishes the one's before, between
// them, and the LDS reads for the block after the next. A wave has one other beside it on its SIMD at the most, so it
// has to hide these latencies itself (64 tokens, 65536 q8_0 rows: 329 us with each block done in turn, 305 so, 300
// with the weights' products in pairs of halves, see weigh(), and 284 with one barrier for two tiles).
// RT: row tiles of 16 query rows that the wave holds.
template <bool Q8, int RT>
__device__ __forceinline__ void scores(const SharedTile& t, const QRegs* q, f4 (&s)[RT][2]) {
  const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f4 c[2][RT][2];
#pragma unroll
  for (int rt = 0; rt < RT; rt++) s[rt][0] = s[rt][1] = zero;
  h8 k[2][2];
  u2 ks[3][2];
  auto ask = [&](int b) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      k[b & 1][u] = *(const h8*)t.k[8 * u + b][16 * g + (n ^ g ^ (4 * b & 12))];
      if constexpr (Q8) ks[b % 3][u] = scales_of(t.ks, b, u);
    }
  };
  auto scale = [&](int b) {
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int i = 0; i < 4; i++)
          s[rt][u][i] = __builtin_fmaf(half_of(ks[b % 3][u][i & 1], i >> 1), c[b & 1][rt][u][i], s[rt][u][i]);
        asm("" : "+v"(s[rt][u]));  // formed here, as in attn_core.h
      }
  };
  ask(0);
#pragma unroll
  for (int b = 0; b < 8; b++) {
    if (b < 7) ask(b + 1);
    if constexpr (Q8) {
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int u = 0; u < 2; u++) c[b & 1][rt][u] = mfma16(k[b & 1][u], q[rt].lo[b], zero);
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int u = 0; u < 2; u++) c[b & 1][rt][u] = mfma16(k[b & 1][u], q[rt].hi[b], c[b & 1][rt][u]);
      if (b) scale(b - 1);
      interleave<2>();
    } else {
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int u = 0; u < 2; u++) s[rt][u] = mfma16(k[b & 1][u], q[rt].lo[b], s[rt][u]);
#pragma unroll
      for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int u = 0; u < 2; u++) s[rt][u] = mfma16(k[b & 1][u], q[rt].hi[b], s[rt][u]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (Q8) scale(7);
}

// PART: some rows of the tile are hidden.
template <bool Q8, bool PART>
__device__ __forceinline__ void accumulate(Rows& st, const f4 (&p)[2], const SharedTile& t) {
  const int l = threadIdx.x & 63, m = l & 15, g = l >> 4;
  u4 ph, pl, hi[2], lo[2];
  h8 v[2][2];
  u2 vs[2][2];
  if constexpr (Q8) split8(st, p, t.vf, ph, pl);
  auto ask_v = [&](int b) {
#pragma unroll
    for (int h = 0; h < 2; h++) v[b & 1][h] = *(const h8*)t.v[2 * b + h][16 * g + (m ^ (2 * b + h))];
  };
  auto ask_s = [&](int b) {
#pragma unroll
    for (int h = 0; h < 2; h++) vs[b & 1][h] = scales_of(t.vs, b, h);
  };
  if constexpr (Q8) {
    ask_s(0);
    ask_v(0);
    ask_s(1);
    weigh<PART>(ph, pl, vs[0], hi[0], lo[0]);
  } else {
    ask_v(0);
    split(p, hi[0], lo[0]);
  }
#pragma unroll
  for (int b = 0; b < 8; b++) {
    __builtin_amdgcn_sched_barrier(0);
    const int w = Q8 ? b & 1 : 0;
    if (b < 7) ask_v(b + 1);
#pragma unroll
    for (int h = 0; h < 2; h++) st.o[2 * b + h] = mfma16(v[b & 1][h], __builtin_bit_cast(h8, lo[w]), st.o[2 * b + h]);
#pragma unroll
    for (int h = 0; h < 2; h++) st.o[2 * b + h] = mfma16(v[b & 1][h], __builtin_bit_cast(h8, hi[w]), st.o[2 * b + h]);
    if constexpr (Q8) {
      if (b < 7) {
        weigh<PART>(ph, pl, vs[(b + 1) & 1], hi[w ^ 1], lo[w ^ 1]);
        if (b < 6) ask_s(b + 2);
        interleave<3>();
      }
    }
  }
}

// f16: adds what stage() took out of a tile (see accumulate_tail): the values that are not finite, to the rows that see them.
__device__ __forceinline__ void add_odd(Rows& st, const f4 (&p)[2], const KvHead& vc, int j0, int left) {
  const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll 1
  for (int gk = 0; gk < 4; gk++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int j = 16 * (e >> 2) + 4 * gk + (e & 3);
      const float wt = __shfl(p[e >> 2][e & 3], 16 * gk + n);
      const uint8_t* row = vc.rows + (size_t)(j0 + (j < left ? j : left - 1)) * (2 * kHD) + 8 * g;
#pragma unroll 1
      for (int i = 0; i < 16; i += 4)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const u2 x = *(const u2*)(row + 32 * (i + q));
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const float f = half_of(x[c >> 1], c & 1);
            const bool add = (__builtin_bit_cast(uint32_t, f) & 0x7f800000u) == 0x7f800000u && !__builtin_signbit(wt) && j < left;
            const float y = add ? wt * f : 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k += 4) st.o[k + q][c] += k == i ? y : 0.0f;
          }
        }
    }
}

}  // namespace q27h
