// The paged cache as the kernels see it: which sequence a row belongs to, where a token lies; and the host's checks of the two
// handles (include/dsgx.h). Shared by kv_append.hip and attn.hip.
#pragma once
#include "abi_internal.h"
#include "common.cuh"

namespace dsgx {

constexpr int kMinPage = 16, kMaxPage = 1024;  // a tile of 16 tokens never straddles two pages

// A row's place in its sequence. One wave looks cu_rows through 64 entries at a time (bounds and lengths of all of them are one round
// trip to memory; a binary search would be one a step); the result is wave-uniform. Entries that are not in order are not trusted:
// the row has to lie between the two bounds that are returned.
struct RowPlace {
  int seq;         // -1: in no sequence
  int first, end;  // the sequence's rows
  int len;         // its own tokens, as given
};
__device__ __forceinline__ RowPlace find_row(const dsgx_kv_batch& b, int r, int lane) {
  RowPlace p{-1, 0, 0, 0};
  if (!b.cu_rows) {
    p.seq = r / b.max_rows;
    if (p.seq >= b.B) p.seq = -1;
    else p.first = p.seq * b.max_rows, p.end = p.first + b.max_rows, p.len = b.lens[p.seq];
    return p;
  }
  for (int j0 = 0; j0 < b.B; j0 += kWave) {
    const int j = j0 + lane;
    const bool in = j < b.B;
    const int lo = in ? b.cu_rows[j] : 0, hi = in ? b.cu_rows[j + 1] : 0, len = in ? b.lens[j] : 0;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(in && lo <= r && r < hi);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      p.seq = j0 + l, p.first = __builtin_amdgcn_readlane(lo, l), p.end = __builtin_amdgcn_readlane(hi, l), p.len = __builtin_amdgcn_readlane(len, l);
      break;
    }
  }
  return p;
}

// ---- host checks --------------------------------------------------------------------------------------------------------
inline int check_cache(const char* who, const dsgx_kv_cache* c) {
  if (!c || !c->k || !c->v) return fail(DSGX_EINVAL, "%s: null cache or pool", who);
  if (c->fmt != DSGX_FMT_BF16 && c->fmt != DSGX_KV_E4M3) return fail(DSGX_EFORMAT, "%s: cache format %u (BF16 or e4m3)", who, c->fmt);
  const bool f8 = c->fmt == DSGX_KV_E4M3;
  if (f8 && (!c->ks || !c->vs)) return fail(DSGX_EINVAL, "%s: an e4m3 cache needs its scales", who);
  if (c->D != 64 && c->D != 128 && c->D != 256) return fail(DSGX_EINVAL, "%s: heads of %d (64, 128 or 256)", who, c->D);
  if (c->Hkv < 1 || c->Hkv > 1024 || c->npages < 1) return fail(DSGX_EINVAL, "%s: %d heads, %d pages", who, c->Hkv, c->npages);
  if (c->page < kMinPage || c->page > kMaxPage || (c->page & (c->page - 1)))
    return fail(DSGX_EINVAL, "%s: pages of %d tokens (a power of two, %d .. %d)", who, c->page, kMinPage, kMaxPage);
  const int64_t unit = f8 ? 16 : 8;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15 || c->page_stride % unit || c->tok_stride % unit || c->head_stride % unit)
    return fail(DSGX_EINVAL, "%s: pools and strides have to be multiples of 16 bytes", who);
  if (c->tok_stride < c->D || c->page_stride < 0 || (c->Hkv > 1 && c->head_stride < c->D))
    return fail(DSGX_EINVAL, "%s: strides %lld (token), %lld (head), %lld (page) for heads of %d", who, (long long)c->tok_stride, (long long)c->head_stride,
                (long long)c->page_stride, c->D);
  return DSGX_OK;
}
inline int check_batch(const char* who, const dsgx_kv_cache* c, const dsgx_kv_batch* b) {
  if (!b || !b->lens || !b->table) return fail(DSGX_EINVAL, "%s: null batch, lengths or table", who);
  if (b->B < 1 || b->B > 65535 || b->rows < 0 || b->max_rows < 1 || b->max_len < 0 || b->table_ld < 1)
    return fail(DSGX_EINVAL, "%s: %d sequences, %d rows (%d each at most), %d tokens at most, %d pages each", who, b->B, b->rows, b->max_rows, b->max_len, b->table_ld);
  if (!b->cu_rows && (int64_t)b->B * b->max_rows != b->rows) return fail(DSGX_EINVAL, "%s: %d sequences of %d rows are not %d rows", who, b->B, b->max_rows, b->rows);
  if (b->prefix_len < 0 || (b->prefix_len > 0 && !b->prefix)) return fail(DSGX_EINVAL, "%s: a prefix of %d tokens without pages", who, b->prefix_len);
  if ((int64_t)b->table_ld * c->page > (1 << 30) || (int64_t)b->prefix_len > (1 << 30)) return fail(DSGX_EINVAL, "%s: over 2^30 tokens", who);
  return DSGX_OK;
}

}  // namespace dsgx
