// The paged 8-bit K/V cache as its kernels see it (kv_append.hip,
// paged_attn.hip): which rows of a call belong to which sequence, and how a
// launch's units are found from lengths that only the device knows.
#pragma once
#include "common.h"

constexpr int kPage = FVSR_PAGE;  // tokens of a page
constexpr int64_t kMaxBlocks = 0xffffff;  // workgroups of a launch: 2^32 threads, 256 each
constexpr int64_t kMaxRows = 0x3fffffff;

// Rows of a call that belong to sequence b: T rows packed at cu[0..B], or
// the same number each.  Clamped, so that no offsets reach outside the T rows.
struct SeqRows {
  int lo, n;
};
FVSR_DEV SeqRows seq_rows(const int32_t* cu, int b, int B, int T) {
  if (!cu) return {b * (T / B), T / B};
  const int lo = min(max(cu[b], 0), T);
  return {lo, min(max(cu[b + 1], lo), T) - lo};
}

// One unit of a launch: part `part` of sequence b.
struct SeqPart {
  SeqRows rows;
  int b, part, len;
};

FVSR_DEV int wave_scan(int v) {  // inclusive sum over the lanes
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  return v;
}

// The unit-th part over all sequences, sequence b having parts(n, len) of
// them: every wave sums 64 sequences' counts at a time.  With `tail` the rows
// behind the last sequence count as one more, of length 0.  False past the last
// part: grids are sized by what the host knows, an upper bound.
template <class Parts>
FVSR_DEV bool find_part(const int32_t* cu, const int32_t* lengths, int B, int T, int unit,
                        bool tail, Parts parts, SeqPart& s) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < B + tail; b0 += 64) {
    const int b = b0 + lane;
    SeqRows r{0, 0};
    int len = 0, cnt = 0;
    if (b < B) {
      r = seq_rows(cu, b, B, T);
      len = max(lengths[b], 0);
      cnt = parts(r.n, len);
    } else if (tail && b == B) {
      r.lo = min(max(cu[B], 0), T);
      r.n = T - r.lo;
      cnt = parts(r.n, 0);
    }
    const int upto = wave_scan(cnt) + before;
    const uint64_t hit = __ballot(upto > unit);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      s.b = b0 + l;
      s.rows.lo = __builtin_amdgcn_readlane(r.lo, l);
      s.rows.n = __builtin_amdgcn_readlane(r.n, l);
      s.len = __builtin_amdgcn_readlane(len, l);
      s.part = unit - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(cnt, l));
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// What both entry points check of the cache and the call's rows (rows and units
// are counted in 32 bits).
static inline int kv_cache_ok(const fvsr_kv_cache* c, int64_t T) {
  if (!c) return FVSR_EINVAL;
  if (c->pages < 0 || c->heads <= 0 || c->sequences < 0 || c->table_pages < 0 || T < 0 ||
      c->table_stride < c->table_pages)
    return FVSR_EINVAL;
  if (c->head_dim != 64 && c->head_dim != 128) return FVSR_EUNSUPPORTED;
  if (T > kMaxRows || c->heads > kMaxBlocks || T * c->heads > kMaxBlocks * 64 ||
      c->sequences > 0x3fffff || c->pages > 0x7fffffff || c->table_pages > 0xffffff)
    return FVSR_EUNSUPPORTED;
  if (T == 0 || c->sequences == 0) return FVSR_OK;
  if ((c->pages > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale)) || !c->lengths ||
      (!c->table && c->sequences * c->table_pages > 0))
    return FVSR_EINVAL;
  if (!c->cu && T % c->sequences) return FVSR_EINVAL;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return FVSR_EUNSUPPORTED;
  return FVSR_OK;
}
