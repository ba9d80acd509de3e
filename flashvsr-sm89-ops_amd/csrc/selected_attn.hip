// Attention of each row over pages of its own choice, in an 8-bit paged cache:
//
//   o[q] = sum_k w[k] v[k] / sum_k w[k],  w[k] = exp(sm_scale * q.k) over the tokens up to
//          q's own position in the pages of its list
//
// A list belongs to a row and a key/value head, so a unit of work is the queries of one head's
// group (up to 16, one operand) over up to `top` pages.  Operands, weights and their precision
// are those of paged_attn.hip: K and V are operand A as stored, q and the weights sums of
// e4m3 terms.
#include <algorithm>

#include "attn_terms.h"

namespace {

struct Args {
  fvsr_kv_cache c;
  const uint16_t* q;
  uint16_t* out;
  int64_t q_ts, q_hs, o_ts, o_hs;
  const int32_t* columns;  // [T, heads, top]
  float* part;             // splits > 1: O of each row of each piece, then (M, l)
  float scale_log2;        // sm_scale * log2(e)
  int T, q_heads, group, top, splits, parts, tail;
};

// A row, a head, up to 16 of its queries and a share of its list.
struct Unit {
  int b, row, h, q0, split, limit;  // limit: tokens that the row sees
};

FVSR_DEV bool unit_of(const Args& a, int at, Unit& u) {
  u.split = at % a.splits;
  at /= a.splits;
  u.q0 = at % a.parts * 16;
  at /= a.parts;
  u.h = at / a.T;
  SeqPart s;
  if (a.c.cu) {
    const auto rows = [](int n, int) { return n; };
    if (!find_part(a.c.cu, a.c.lengths, (int)a.c.sequences, a.T, at % a.T, a.tail != 0, rows, s))
      return false;
  } else {
    const int each = a.T / (int)a.c.sequences;
    s.b = at % a.T / each, s.part = at % a.T % each;
    s.rows = SeqRows{s.b * each, each};
    s.len = max(a.c.lengths[s.b], 0);
  }
  u.b = s.b, u.row = s.rows.lo + s.part;
  const int64_t cap = a.c.table_pages * kPage;
  u.limit = (int)min((int64_t)max(s.len - s.rows.n + s.part + 1, 0), cap);
  return true;
}

// One wave's share of a unit: lane (r, g) = (l % 16, l / 16) has positions 16 g .. and 64 + 16 g
// .. of row r of an operand, and accumulators of column r (a query), rows 4 g ...
template <int DT, int D>
struct Rows {
  static constexpr int N = terms(DT);
  static constexpr int W = D / 64;                      // 16-byte pieces of a K row per lane
  static constexpr int F = D == 128 ? N : (N + 1) / 2;  // Q operands (64 dims: two terms each)
  static constexpr int DT16 = D / 16;

  v8i qf[F];
  int qs[F];
  v4f acc[DT16];
  float m, l;

  // Q^T's terms.
  FVSR_DEV void load(Rows& w, const Args& a, const Unit& u, int col, int g) {
    const int hq = u.h * a.group + min(u.q0 + col, a.group - 1);
    const uint16_t* qp = a.q + (int64_t)u.row * a.q_ts + (int64_t)hq * a.q_hs + 16 * g;
    u32x4_t raw[W][2];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      raw[i][0] = *(const u32x4_t*)(qp + 64 * i);
      raw[i][1] = *(const u32x4_t*)(qp + 64 * i + 8);
    }
    const auto el = [&](int i, int j) {
      const uint32_t x = raw[i][j >> 3][(j >> 1) & 3];
      return to_f<DT>((uint16_t)(j & 1 ? x >> 16 : x & 0xffff));
    };
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) top = max_mag(top, el(i, j));
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const int e = row_exp(top);
    const float f = __builtin_ldexpf(1.0f, -e);
    uint32_t t[W][4][N];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        split4<N>(el(i, 4 * j) * f, el(i, 4 * j + 1) * f, el(i, 4 * j + 2) * f,
                  el(i, 4 * j + 3) * f, t[i][j]);
#pragma unroll
    for (int k = 0; k < F; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (D == 128)
          w.qf[k][i] = (int)t[i >> 2][i & 3][k];
        else  // positions 0-63: term 2k, 64-127: term 2k + 1, of the same dims
          w.qf[k][i] = 2 * k + (i >> 2) < N ? (int)t[0][i & 3][min(2 * k + (i >> 2), N - 1)] : 0;
      }
      w.qs[k] = e8m0(e - 5 * (D == 128 ? k : 2 * k + (g >> 1)));
    }
#pragma unroll
    for (int d = 0; d < DT16; ++d) w.acc[d] = v4f{};
    w.m = kNothing, w.l = 0.0f;
  }

  // A page of which the row sees the first `seen` tokens.
  FVSR_DEV void page(Rows& w, const uint8_t* kp, const uint8_t* vp, int ks, int vs, int seen, int g,
                     float scale_log2) {
    v8i kf[8], vf[DT16];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint8_t* x = kp + ((t >> 2) * 64 + (t & 3) * 4) * D;
      const u32x4_t y = *(const u32x4_t*)x;
      kf[t] = join(y, D == 128 ? *(const u32x4_t*)(x + 64) : y);
    }
#pragma unroll
    for (int d = 0; d < DT16; ++d) {
      const uint8_t* x = vp + d * 16 * kPage;
      vf[d] = join(*(const u32x4_t*)x, *(const u32x4_t*)(x + 64));
    }
    v4f sc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const v4f z = {};
      sc[t] = mfma(kf[t], w.qf[0], z, ks, w.qs[0]);
#pragma unroll
      for (int k = 1; k < F; ++k) sc[t] = mfma(kf[t], w.qf[k], sc[t], ks, w.qs[k]);
    }
    // Accumulator (t, j) of lane g is position 64 (t / 4) + 16 g + 4 (t % 4) + j.
    const auto at = [g](int t, int j) { return 16 * g + (t >> 2) * 64 + (t & 3) * 4 + j; };
    const bool masked = seen < kPage;
    if (masked) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at(t, j) >= seen) sc[t][j] = -__builtin_huge_valf();
    }
    float top = -__builtin_huge_valf();
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[t][j]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int shift;
    weigh(sc, top, scale_log2, w.m, w.l, shift, [&](float f) {
#pragma unroll
      for (int d = 0; d < DT16; ++d) w.acc[d] *= f;
    });
    v8i pf[N];
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      uint32_t x[N];
      weights4<N>(sc[t][0], sc[t][1], sc[t][2], sc[t][3], x, sum);
#pragma unroll
      for (int k = 0; k < N; ++k) pf[k][t] = (int)x[k];
    }
    w.l += __builtin_ldexpf(sum, shift);
    if (masked) {
      // Hidden tokens weigh 0, which a NaN code would not survive: NaN codes leave the
      // product and are counted where they are seen.  A NaN scale stands for a page of them.
      if (vs == 255) {
        asm volatile("" :::);  // a branch
        vs = 127;
#pragma unroll
        for (int d = 0; d < DT16; ++d)
#pragma unroll
          for (int i = 0; i < 8; ++i) vf[d][i] = 0x7f7f7f7f;
      }
      bool any = false;
#pragma unroll
      for (int d = 0; d < DT16; ++d) any |= has_nan(vf[d]);
      if (__ballot(any) != 0) {
        v8i ones;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          ones[t] = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at(t, j) < seen) ones[t] |= 0x38 << (8 * j);
        }
#pragma unroll
        for (int d = 0; d < DT16; ++d) {
          const v8i nans = take_nan(vf[d]);
          const v4f z = {};
          const v4f n = mfma(nans, ones, z, 127, 127);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n[j] > 0.0f) w.acc[d][j] = __builtin_nanf("");
        }
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int ps = e8m0(shift - 5 * k);
#pragma unroll
      for (int d = 0; d < DT16; ++d) w.acc[d] = mfma(vf[d], pf[k], w.acc[d], vs, ps);
    }
  }

  // Entries first, first + step, .. below `end` of the unit's list.  64 at a time are looked
  // up together, one a lane, so that no page waits for its id.
  FVSR_DEV void run(Rows& w, const Args& a, const Unit& u, int first, int end, int step, int lane) {
    const int col = lane & 15, g = lane >> 4, H = (int)a.c.heads;
    load(w, a, u, col, g);
    const int32_t* const list = a.columns + ((int64_t)u.row * H + u.h) * a.top;
    const int32_t* const table = a.c.table + (int64_t)u.b * a.c.table_stride;
    const int pages = (u.limit + kPage - 1) / kPage;
    // Row r of K subtile t is key 64 (t / 4) + 16 (r / 4) + 4 (t % 4) + r % 4.
    const int k_off = (16 * (col >> 2) + (col & 3)) * D + 16 * g;
    const int v_off = col * kPage + 16 * g;
    for (int e0 = first; e0 < end; e0 += 64 * step) {
      const int e = e0 + lane * step;
      const int c = e < end ? list[e] : -1;
      const bool sees = c >= 0 && c < pages;
      const int id = sees ? table[c] : -1;
      const bool there = sees && id >= 0 && id < a.c.pages;
      const int64_t mine = there ? (int64_t)id * H + u.h : 0;
      const int scales = there ? ((const uint8_t*)a.c.k_scale)[mine] |
                                     ((const uint8_t*)a.c.v_scale)[mine] << 8
                               : 0;
      if (__ballot(sees && !there)) w.l = __builtin_nanf("");  // no such page
      uint64_t todo = __ballot(there);
      while (todo) {
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int64_t ph = (int64_t)__builtin_amdgcn_readlane(id, i) * H + u.h;
        const int s = __builtin_amdgcn_readlane(scales, i);
        const int seen = u.limit - __builtin_amdgcn_readlane(c, i) * kPage;
        page(w, (const uint8_t*)a.c.k + ph * kPage * D + k_off,
             (const uint8_t*)a.c.v + ph * kPage * D + v_off, s & 255, s >> 8, seen, g,
             a.scale_log2);
      }
    }
    w.l += __shfl_xor(w.l, 16);
    w.l += __shfl_xor(w.l, 32);
  }
};

// Few units: a workgroup's waves take entries of one list in turn, and add what they have.
template <int DT, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_shared(Args a) {
  constexpr int P = D + 4, C = D / 8;
  __shared__ __attribute__((aligned(16))) float lds_o[4 * 16 * P];
  __shared__ float lds_ml[4][16][2];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Unit u;
  if (!unit_of(a, xcd_order(blockIdx.x, gridDim.x), u)) return;
  const int e0 = range_at(a.top, u.split, a.splits), e1 = range_at(a.top, u.split + 1, a.splits);
  Rows<DT, D> w;
  w.run(w, a, u, e0 + wave, e1, 4, lane);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) *(v4f*)&lds_o[(wave * 16 + col) * P + d * 16 + 4 * g] = w.acc[d];
  if (g == 0) lds_ml[wave][col][0] = w.m, lds_ml[wave][col][1] = w.l;
  __syncthreads();
  const int d0 = threadIdx.x % C * 8;
  for (int i = threadIdx.x / C; i < 16 && u.q0 + i < a.group; i += kThreads / C) {
    float top = lds_ml[0][i][0];
#pragma unroll
    for (int v = 1; v < 4; ++v) top = fmaxf(top, lds_ml[v][i][0]);
    float o[8] = {}, sum = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = __builtin_amdgcn_exp2f(lds_ml[v][i][0] - top);
      sum += f * lds_ml[v][i][1];
      const v4f x = *(const v4f*)&lds_o[(v * 16 + i) * P + d0];
      const v4f y = *(const v4f*)&lds_o[(v * 16 + i) * P + d0 + 4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += f * x[j], o[4 + j] += f * y[j];
    }
    const int oh = u.h * a.group + u.q0 + i;
    if (a.splits == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      u32x2_t* op = (u32x2_t*)(a.out + (int64_t)u.row * a.o_ts + oh * a.o_hs + d0);
      op[0] = u32x2_t{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv)};
      op[1] = u32x2_t{pack2<DT>(o[4] * inv, o[5] * inv), pack2<DT>(o[6] * inv, o[7] * inv)};
    } else {
      const int64_t pr = ((int64_t)u.row * a.q_heads + oh) * a.splits + u.split;
      v4f* po = (v4f*)(a.part + pr * D + d0);
      po[0] = v4f{o[0], o[1], o[2], o[3]};
      po[1] = v4f{o[4], o[5], o[6], o[7]};
      if (d0 == 0) {
        float* ml = a.part + (int64_t)a.T * a.q_heads * a.splits * D + pr * 2;
        ml[0] = top, ml[1] = sum;
      }
    }
  }
}

template <int DT, int D>
__global__ __launch_bounds__(kThreads) void join_shared(Args a) {
  const int64_t row = blockIdx.x, rows = (int64_t)a.T * a.q_heads;
  if (a.c.cu && !a.tail && row / a.q_heads >= a.c.cu[a.c.sequences]) return;
  join_row<DT, D>(a.part + row * a.splits * D, D,
                  a.part + rows * a.splits * D + row * a.splits * 2, 2, a.splits,
                  a.out + row / a.q_heads * a.o_ts + row % a.q_heads * a.o_hs);
}

// Many units: one a wave.
template <int DT, int D>
__global__ __launch_bounds__(kThreads, 2) void attend_alone(Args a) {
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int at = xcd_order(blockIdx.x, gridDim.x) * 4 + wave;
  Unit u;
  if (at >= a.T * (int)a.c.heads * a.parts || !unit_of(a, at, u)) return;
  Rows<DT, D> w;
  w.run(w, a, u, 0, a.top, 1, lane);
  if (u.q0 + col >= a.group) return;
  const float inv = w.l == 0.0f ? 0.0f : 1.0f / w.l;
  uint16_t* op = a.out + (int64_t)u.row * a.o_ts + (u.h * a.group + u.q0 + col) * a.o_hs + 4 * g;
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
    *(u32x2_t*)(op + d * 16) = u32x2_t{pack2<DT>(w.acc[d][0] * inv, w.acc[d][1] * inv),
                                       pack2<DT>(w.acc[d][2] * inv, w.acc[d][3] * inv)};
}

// How a call is cut up: a function of its sizes only.
struct Plan {
  int64_t units;  // rows x heads x operands of 16 queries
  int parts, splits;
  bool alone;
  int64_t floats(int64_t T, int64_t q_heads, int64_t D) const {
    return splits > 1 ? T * q_heads * splits * (D + 2) : 0;
  }
};

Plan plan_selected(const fvsr_kv_cache* c, int64_t T, int64_t q_heads, int64_t top) {
  Plan p{};
  const int64_t cus = 256;
  p.parts = (int)((q_heads / c->heads + 15) / 16);
  p.units = T * c->heads * p.parts;
  p.splits = 1;
  p.alone = p.units >= 16 * cus;
  if (!p.alone)
    p.splits = (int)std::min<int64_t>({std::max<int64_t>(1, 2 * cus / std::max<int64_t>(1, p.units)),
                                       std::max<int64_t>(1, top / 4), kMaxSplits});
  return p;
}

template <int DT, int D>
void launch(const Args& a, const Plan& p, hipStream_t st) {
  const dim3 block(kThreads);
  if (p.alone) {
    hipLaunchKernelGGL((attend_alone<DT, D>), dim3((unsigned)((p.units + 3) / 4)), block, 0, st, a);
    return;
  }
  hipLaunchKernelGGL((attend_shared<DT, D>), dim3((unsigned)(p.units * p.splits)), block, 0, st, a);
  if (p.splits > 1)
    hipLaunchKernelGGL((join_shared<DT, D>), dim3((unsigned)((int64_t)a.T * a.q_heads)), block, 0,
                       st, a);
}

bool sizes_ok(const fvsr_kv_cache* c, int64_t T, int64_t q_heads, int64_t top) {
  return q_heads <= kMaxBlocks && top <= 0xffffff && T * q_heads <= kMaxBlocks * 4;
}

}  // namespace

extern "C" int64_t fvsr_selected_attn_workspace_floats(const fvsr_kv_cache* cache, int64_t T,
                                                       int64_t q_heads, int64_t top) {
  if (kv_cache_ok(cache, T) != FVSR_OK || T == 0 || cache->sequences == 0 || q_heads <= 0 ||
      q_heads % cache->heads || top < 0 || !sizes_ok(cache, T, q_heads, top))
    return 0;
  return plan_selected(cache, T, q_heads, top).floats(T, q_heads, cache->head_dim);
}

extern "C" int fvsr_selected_attn(const fvsr_kv_cache* cache, const void* q, int64_t q_tok_stride,
                                  int64_t q_head_stride, int64_t q_heads, void* out,
                                  int64_t o_tok_stride, int64_t o_head_stride, int dtype,
                                  int64_t T, const int32_t* columns, int64_t top, float sm_scale,
                                  int fill_tail, float* workspace, int64_t workspace_floats,
                                  void* stream) {
  const int rc = kv_cache_ok(cache, T);
  if (rc != FVSR_OK) return rc;
  if (dtype != FVSR_DT_BF16 && dtype != FVSR_DT_F16) return FVSR_EINVAL;
  if (q_heads <= 0 || q_heads % cache->heads || top < 0 || !(sm_scale > 0.0f) || sm_scale > 3e38f)
    return FVSR_EINVAL;
  if (!sizes_ok(cache, T, q_heads, top)) return FVSR_EUNSUPPORTED;
  if (T == 0 || cache->sequences == 0) return FVSR_OK;
  if (!q || !out || (top > 0 && !columns)) return FVSR_EINVAL;
  if ((((uintptr_t)q) | (uint64_t)(q_tok_stride * 2) | (uint64_t)(q_head_stride * 2)) & 15)
    return FVSR_EUNSUPPORTED;
  if ((((uintptr_t)out) | (uint64_t)(o_tok_stride * 2) | (uint64_t)(o_head_stride * 2)) & 7)
    return FVSR_EUNSUPPORTED;
  const Plan p = plan_selected(cache, T, q_heads, top);
  const int64_t need = p.floats(T, q_heads, cache->head_dim);
  if (need && (!workspace || workspace_floats < need)) return FVSR_EWORKSPACE;
  if (need && ((uintptr_t)workspace & 15)) return FVSR_EUNSUPPORTED;
  Args a{};
  a.c = *cache;
  a.q = (const uint16_t*)q, a.out = (uint16_t*)out;
  a.q_ts = q_tok_stride, a.q_hs = q_head_stride, a.o_ts = o_tok_stride, a.o_hs = o_head_stride;
  a.columns = columns, a.part = workspace;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.T = (int)T, a.q_heads = (int)q_heads, a.group = (int)(q_heads / cache->heads);
  a.top = (int)top, a.splits = p.splits, a.parts = p.parts, a.tail = fill_tail != 0;
  const hipStream_t st = (hipStream_t)stream;
  const bool half = dtype == FVSR_DT_F16;
  if (cache->head_dim == 128)
    half ? launch<FVSR_DT_F16, 128>(a, p, st) : launch<FVSR_DT_BF16, 128>(a, p, st);
  else
    half ? launch<FVSR_DT_F16, 64>(a, p, st) : launch<FVSR_DT_BF16, 64>(a, p, st);
  return fvsr_launch_status();
}
