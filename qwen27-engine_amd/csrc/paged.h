// A K/V cache in pages that many sequences share, and a ragged batch over it, as the kernels see them.
//
// A page of K or V is a cache of `rows` rows as attn_prep lays one out: f16 [nkvh][rows][256], or codes [nkvh][rows][256]
// (4 bits: [nkvh][rows][128]) followed by f16 scales [nkvh][rows][8]. 4 bits: byte j of a block's 16 holds value j in its low
// half and value j + 16 in its high one, each the code 0 .. 15 of (code - 8) * scale. rows is a power of two of at least 32,
// so that a tile of 32 rows lies in one page.
#pragma once
#include "q27h_device.h"
#include "q27h_internal.h"

namespace q27h {

constexpr int kHeadDim = 256;
constexpr int kRowF16 = 512, kRowQ8 = 272, kRowQ4 = 144;  // bytes of a row of one head, scales included

struct Pages {
  uint8_t *k, *v;
  const int* table;  // [n_seqs][max_pages]
  size_t kb, vb;     // bytes of a page of K, of V
  int n_seqs, max_pages, n_pages, nkvh, shift;  // 1 << shift rows a page
  int type;
};

inline int kv_row_bytes(int type, bool v) {
  return type == Q27H_KV_F16 ? kRowF16 : v && type == Q27H_KV_Q8_Q4 ? kRowQ4 : kRowQ8;
}
// Q27H_OK, or the refusal of a bad handle (its sizes, pointers and alignment).
int check_pages(const q27h_kv_pages* kv, const char* what);
Pages pages_of(const q27h_kv_pages* kv);  // of a handle that passed

// A load from memory that no kernel writes while this one runs, of an address that is the same in the whole wave: through
// the scalar cache, so that the vector loads on their way need not be waited for.
__device__ __forceinline__ int uniform_load(const int* p) { return *(const __attribute__((address_space(4))) int*)p; }

// The tokens of sequence b of the batch, t0 .. t0 + nt - 1, whatever cu holds. cu null: token b.
struct Tokens {
  int t0, nt;
};
__device__ __forceinline__ Tokens tokens_of(int c0, int c1, int T, int most) {
  c0 = c0 < 0 ? 0 : c0 > T ? T : c0;
  c1 = c1 < c0 ? c0 : c1 > T ? T : c1;
  return {c0, c1 - c0 < most ? c1 - c0 : most};
}
__device__ __forceinline__ Tokens tokens_of(const int* cu, int b, int T, int most) {
  return cu ? tokens_of(uniform_load(cu + b), uniform_load(cu + b + 1), T, most) : tokens_of(b, b + 1, T, most);
}

}  // namespace q27h
