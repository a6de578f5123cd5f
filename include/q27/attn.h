// Attention over the K/V cache that attn_prep writes, and the cache's keeping, in namespace q27 over include/q27h.h: a tree
// of drafted tokens, attention weights per row and eviction, blocks chosen per token. No counterparts in the reference's
// headers. The contracts stand in q27h.h; a bad shape or argument throws std::runtime_error.
#pragma once
#include "ops.h"

namespace q27 {

inline size_t attn_tree_ws_bytes(int T, int nqh, int nkvh, int n_ctx) { return q27h_attn_tree_ws_bytes(T, nqh, nkvh, n_ctx); }
inline void attn_tree(const float* qn, const void* kcache, const void* vcache, const int* pos0, const uint64_t* tree, int T,
                      float scale, int nqh, int nkvh, int n_ctx, bool q8, float* o, void* ws, size_t ws_bytes, hipStream_t s,
                      float* lse = nullptr) {
  q27h_check(q27h_attn_tree(qn, kcache, vcache, pos0, tree, T, scale, nqh, nkvh, n_ctx, q8 ? 1 : 0, o, lse, ws, ws_bytes, s));
}
inline void attn_weights(const float* qn, const float* lse, const void* kcache, const int* pos0, const uint64_t* tree, int T,
                         float scale, int nqh, int nkvh, int n_ctx, bool q8, float* acc, hipStream_t s,
                         const uint64_t* rows = nullptr) {
  q27h_check(q27h_attn_weights(qn, lse, kcache, pos0, tree, rows, T, scale, nqh, nkvh, n_ctx, q8 ? 1 : 0, acc, s));
}
inline size_t kv_evict_ws_bytes(int nkvh, int n_ctx, int keep, bool q8, bool in_place) {
  return q27h_kv_evict_ws_bytes(nkvh, n_ctx, keep, q8 ? 1 : 0, in_place ? 1 : 0);
}
inline void kv_evict(const void* kcache, const void* vcache, const float* acc, const int* pos0, int keep, int first, int last,
                     void* kout, void* vout, float* acc_out, int n_ctx_out, int* kept, int nkvh, int n_ctx, bool q8, void* ws,
                     size_t ws_bytes, hipStream_t s) {
  q27h_check(q27h_kv_evict(kcache, vcache, acc, pos0, keep, first, last, kout, vout, acc_out, n_ctx_out, kept, nkvh, n_ctx,
                           q8 ? 1 : 0, ws, ws_bytes, s));
}
inline void kv_evict_pos(int* pos0, int* rdelta, int keep, hipStream_t s) { q27h_check(q27h_kv_evict_pos(pos0, rdelta, keep, s)); }
inline void kv_accept(void* const* caches, int n_caches, float* const* accs, int n_accs, const int* pos0, const int* path,
                      const int* n_path, int T, int nkvh, int n_ctx, bool q8, hipStream_t s) {
  q27h_check(q27h_kv_accept(caches, n_caches, accs, n_accs, pos0, path, n_path, T, nkvh, n_ctx, q8 ? 1 : 0, s));
}
inline size_t kv_block_bytes(int nkvh, int n_ctx) { return q27h_kv_block_bytes(nkvh, n_ctx); }
inline void kv_block_bounds(const void* kcache, const int* pos0, int T, int nkvh, int n_ctx, bool q8, void* kb, hipStream_t s) {
  q27h_check(q27h_kv_block_bounds(kcache, pos0, T, nkvh, n_ctx, q8 ? 1 : 0, kb, s));
}
inline size_t attn_select_ws_bytes(int T, int nkvh, int n_ctx) { return q27h_attn_select_ws_bytes(T, nkvh, n_ctx); }
inline void attn_select(const float* qn, const void* kb, const int* pos0, int T, int nqh, int nkvh, int n_ctx, int nsel, int first,
                        int last, int* idx, void* ws, size_t ws_bytes, hipStream_t s) {
  q27h_check(q27h_attn_select(qn, kb, pos0, T, nqh, nkvh, n_ctx, nsel, first, last, idx, ws, ws_bytes, s));
}
inline size_t attn_blocks_ws_bytes(int T, int nqh, int nkvh, int nsel) { return q27h_attn_blocks_ws_bytes(T, nqh, nkvh, nsel); }
inline void attn_blocks(const float* qn, const void* kcache, const void* vcache, const int* pos0, const int* idx, int T, int nsel,
                        float scale, int nqh, int nkvh, int n_ctx, bool q8, float* o, void* ws, size_t ws_bytes, hipStream_t s,
                        float* lse = nullptr) {
  q27h_check(q27h_attn_blocks(qn, kcache, vcache, pos0, idx, T, nsel, scale, nqh, nkvh, n_ctx, q8 ? 1 : 0, o, lse, ws, ws_bytes, s));
}

}  // namespace q27
