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
#include <type_traits>

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
  int rows, tiles;  // rows of a unit at most; tiles of them over all sequences
};

// Up to a.rows rows of a sequence, a head, up to 16 of its queries and a share of the lists.
struct Unit {
  SeqPart s;
  int row, n, h, q0, split;
};

FVSR_DEV bool unit_of(const Args& a, int at, Unit& u) {
  u.split = at % a.splits;
  at /= a.splits;
  u.q0 = at % a.parts * 16;
  at /= a.parts;
  u.h = at / a.tiles;
  SeqPart& s = u.s;
  const int each = a.rows;
  if (a.c.cu) {
    const auto tiles = [each](int n, int) { return (n + each - 1) / each; };
    if (!find_part(a.c.cu, a.c.lengths, (int)a.c.sequences, a.T, at % a.tiles, a.tail != 0, tiles,
                   s))
      return false;
  } else {
    const int per = a.tiles / (int)a.c.sequences;
    s.b = at % a.tiles / per, s.part = at % a.tiles % per;
    s.rows = seq_rows(nullptr, s.b, (int)a.c.sequences, a.T);
    s.len = max(a.c.lengths[s.b], 0);
  }
  u.row = s.rows.lo + s.part * each;
  u.n = min(each, s.rows.n - s.part * each);
  return true;
}

// Tokens that row i of a unit sees.
FVSR_DEV int limit_of(const Args& a, const Unit& u, int i) {
  const int lim = u.s.len - u.s.rows.n + u.s.part * a.rows + i + 1;
  return (int)min((int64_t)max(lim, 0), a.c.table_pages * kPage);
}
FVSR_DEV int pages_of(int limit) { return (limit + kPage - 1) / kPage; }

// The lists of a unit's rows, joined: columns, and which rows list them.
constexpr int kEntries = 1024;
struct Lists {
  int column[kEntries];    // as listed, row by row; kNone where a row does not see it
  uint32_t rows[kEntries];  // 0: a row before it lists the same
  int falls;
};
constexpr int kNone = INT32_MAX;

// Rows of one sequence that stand together want much the same pages.  A page that several
// rows list is read and multiplied once for all of them.  Rising lists (as select_pages gives
// them) are searched for each other's columns; if one of them is not, each entry stands for itself.
FVSR_DEV void join_lists(Lists& l, const Args& a, const Unit& u) {
  const int total = u.n * a.top, H = (int)a.c.heads;
  if (threadIdx.x == 0) l.falls = 0;
  for (int e = threadIdx.x; e < total; e += kThreads) {
    const int i = e / a.top;
    const int c = a.columns[((int64_t)(u.row + i) * H + u.h) * a.top + e % a.top];
    l.column[e] = c >= 0 && c < pages_of(limit_of(a, u, i)) ? c : kNone;
  }
  __syncthreads();
  bool falls = false;
  for (int e = threadIdx.x; e < total; e += kThreads)
    falls |= e % a.top > 0 && l.column[e] != kNone && l.column[e - 1] >= l.column[e];
  if (falls) l.falls = 1;
  __syncthreads();
  const bool search = l.falls == 0;
  for (int e = threadIdx.x; e < total; e += kThreads) {
    const int i = e / a.top, c = l.column[e];
    uint32_t rows = c == kNone ? 0 : 1u << i;
    if (search && rows)
      for (int j = 0; j < u.n; ++j) {
        if (j == i) continue;
        int lo = j * a.top, n = a.top;  // the first entry of row j not below c is in lo .. lo + n
        while (n > 0) {
          const int half = n / 2;
          if (l.column[lo + half] < c)
            lo += half + 1, n -= half + 1;
          else
            n = half;
        }
        if (lo < (j + 1) * a.top && l.column[lo] == c) {
          if (j < i) rows = 0;
          if (rows == 0) break;
          rows |= 1u << j;
        }
      }
    l.rows[e] = rows;
  }
  __syncthreads();
}

// One wave's share of a unit: lane (r, g) = (l % 16, l / 16) has positions 16 g .. and 64 + 16 g
// .. of row r of an operand, and accumulators of column r (a query), rows 4 g ...
template <int DT, int D>
struct Queries {
  static constexpr int N = terms(DT);
  static constexpr int W = D / 64;                      // 16-byte pieces of a K row per lane
  static constexpr int F = D == 128 ? N : (N + 1) / 2;  // Q operands (64 dims: two terms each)
  static constexpr int DT16 = D / 16;

  v8i qf[F];
  int qs[F];
  v4f acc[DT16];
  float m, l;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < DT16; ++d) acc[d] = v4f{};
    m = kNothing, l = 0.0f;
  }

  // Q^T's terms.
  __device__ __forceinline__ void load(const uint16_t* qp, int g) {
    u32x4_t raw[W][2];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      raw[i][0] = *(const u32x4_t*)(qp + 16 * g + 64 * i);
      raw[i][1] = *(const u32x4_t*)(qp + 16 * g + 64 * i + 8);
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
          qf[k][i] = (int)t[i >> 2][i & 3][k];
        else  // positions 0-63: term 2k, 64-127: term 2k + 1, of the same dims
          qf[k][i] = 2 * k + (i >> 2) < N ? (int)t[0][i & 3][min(2 * k + (i >> 2), N - 1)] : 0;
      }
      qs[k] = e8m0(e - 5 * (D == 128 ? k : 2 * k + (g >> 1)));
    }
    clear();
  }

  // A page, of which this lane's query sees the first `seen` tokens; `part`: some query of the
  // wave does not see all of it.  Hidden tokens weigh 0, which a NaN among V's codes would not
  // survive: CAREFUL takes NaN codes out of the product and counts them where they are seen.
  template <bool CAREFUL>
  __device__ __forceinline__ void page(const uint8_t* kp, int k_off, const uint8_t* vp, int v_off,
                                       int ks, int vs, bool part, int seen, int g,
                                       float scale_log2) {
    // (Opaque, so that no sums with them are kept in registers from page to page.)
    asm volatile("" : "+v"(k_off), "+v"(v_off));
    kp += k_off, vp += v_off;
    const auto k_tile = [&](int t) {
      const uint8_t* x = kp + ((t >> 2) * 64 + (t & 3) * 4) * D;
      const u32x4_t y = *(const u32x4_t*)x;
      return ::join(y, D == 128 ? *(const u32x4_t*)(x + 64) : y);
    };
    const auto v_tile = [&](int d) {
      const uint8_t* x = vp + d * 16 * kPage;
      return ::join(*(const u32x4_t*)x, *(const u32x4_t*)(x + 64));
    };
    // (CAREFUL is rare, and keeps no more registers than it needs: operands one by one.)
    v8i kf[8], vf[DT16];
    if constexpr (!CAREFUL) {
#pragma unroll
      for (int t = 0; t < 8; ++t) kf[t] = k_tile(t);
#pragma unroll
      for (int d = 0; d < DT16; ++d) vf[d] = v_tile(d);
    }
    v4f sc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if constexpr (CAREFUL) {
        asm volatile("" ::: "memory");
        kf[t] = k_tile(t);
      }
      const v4f z = {};
      sc[t] = mfma(kf[t], qf[0], z, ks, qs[0]);
#pragma unroll
      for (int k = 1; k < F; ++k) sc[t] = mfma(kf[t], qf[k], sc[t], ks, qs[k]);
    }
    // Accumulator (t, j) of lane g is position 64 (t / 4) + 16 g + 4 (t % 4) + j.
    const auto at = [](int t, int j) { return (t >> 2) * 64 + (t & 3) * 4 + j; };
    const int left = seen - 16 * g;
    if (part) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at(t, j) >= left) sc[t][j] = -__builtin_huge_valf();
    }
    float top = -__builtin_huge_valf();
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[t][j]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int shift;
    weigh(sc, top, scale_log2, m, l, shift, [&](float f) {
#pragma unroll
      for (int d = 0; d < DT16; ++d) acc[d] *= f;
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
    l += __builtin_ldexpf(sum, shift);
    v8i ones;
    if constexpr (CAREFUL) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        ones[t] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at(t, j) < left) ones[t] |= 0x38 << (8 * j);
      }
    }
#pragma unroll
    for (int d = 0; d < DT16; ++d) {
      if constexpr (CAREFUL) {
        asm volatile("" ::: "memory");
        vf[d] = v_tile(d);
        if (vs == 255)  // a page of NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) vf[d][i] = 0x7f7f7f7f;
        const v8i nans = take_nan(vf[d]);
        const v4f z = {};
        const v4f n = mfma(nans, ones, z, 127, 127);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n[j] > 0.0f) acc[d][j] = __builtin_nanf("");
      }
#pragma unroll
      for (int k = 0; k < N; ++k)
        acc[d] = mfma(vf[d], pf[k], acc[d], CAREFUL && vs == 255 ? 127 : vs, e8m0(shift - 5 * k));
    }
  }
};

// A workgroup's waves take the pages of a unit in turn (of all that its splits have, every
// splits * 4th) and add what they have.  GROUP: several rows to a unit, row i's queries in
// columns i * group and on.
template <int DT, int D, bool GROUP>
__global__ __launch_bounds__(kThreads, 2) void attend_chosen(Args a) {
  constexpr int P = D + 4, C = D / 8;
  __shared__ __attribute__((aligned(16))) float lds_o[4 * 16 * P];
  __shared__ float lds_ml[4][16][2];
  __shared__ std::conditional_t<GROUP, Lists, int> lists;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, H = (int)a.c.heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Unit u;
  if (!unit_of(a, xcd_order(blockIdx.x, gridDim.x), u)) return;
  if constexpr (GROUP) join_lists(lists, a, u);
  const int mine = GROUP ? min(col / a.group, u.n - 1) : 0;  // this lane's row of the unit
  const int head = GROUP ? col % a.group : min(u.q0 + col, a.group - 1);
  const int limit = limit_of(a, u, mine), least = limit_of(a, u, 0);
  const int32_t* const list = a.columns + ((int64_t)u.row * H + u.h) * a.top;
  const int32_t* const table = a.c.table + (int64_t)u.s.b * a.c.table_stride;
  const uint32_t all = (1u << u.n) - 1;
  const int total = u.n * a.top, turn = u.split * 4 + wave, turns = a.splits * 4;
  // Row r of K subtile t is key 64 (t / 4) + 16 (r / 4) + 4 (t % 4) + r % 4.
  const int k_off = (16 * (col >> 2) + (col & 3)) * D + 16 * g;
  const int v_off = col * kPage + 16 * g;
  Queries<DT, D> w;
  w.load(a.q + (int64_t)(u.row + mine) * a.q_ts + (int64_t)(u.h * a.group + head) * a.q_hs, g);
  // 64 entries at a time are looked up together, one a lane, so that no page waits for its id.
  const auto pages = [&](auto careful) {
    int before = 0;
    for (int e0 = 0; e0 < total; e0 += 64) {
      const int e = e0 + lane;
      int c = -1;
      uint32_t rows = 0;
      if (e < total) {
        if constexpr (GROUP) {
          c = lists.column[e], rows = lists.rows[e];
        } else {
          c = list[e];
          rows = c >= 0 && c < pages_of(limit) ? 1 : 0;
        }
      }
      const uint64_t there = __ballot(rows != 0);
      const int at = before + __popcll(there & ((1ull << lane) - 1));
      before += __popcll(there);
      const bool take = rows != 0 && at % turns == turn;
      const int id = take ? table[c] : -1;
      const bool good = take && id >= 0 && id < a.c.pages;
      const int64_t ph = good ? (int64_t)id * H + u.h : 0;
      const int scales = good ? ((const uint8_t*)a.c.k_scale)[ph] |
                                    ((const uint8_t*)a.c.v_scale)[ph] << 8
                              : 0;
      // No such page: the rows that list it are NaN.
      for (uint64_t bad = __ballot(take && !good); bad; bad &= bad - 1) {
        const uint32_t who = __builtin_amdgcn_readlane(rows, __builtin_ctzll(bad));
        if (!GROUP || (who >> mine & 1) != 0) w.l = __builtin_nanf("");
      }
      uint64_t todo = __ballot(good);
      while (todo) {
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int page = __builtin_amdgcn_readlane(id, i);
        const int from = __builtin_amdgcn_readlane(c, i) * kPage;
        const uint32_t who = __builtin_amdgcn_readlane(rows, i);
        const bool sees = !GROUP || (who >> mine & 1) != 0;
        const int64_t at = ((int64_t)page * H + u.h) * kPage * D;
        const int s = __builtin_amdgcn_readlane(scales, i);
        w.template page<careful>((const uint8_t*)a.c.k + at, k_off, (const uint8_t*)a.c.v + at,
                                 v_off, s & 255, s >> 8,
                                 (GROUP && who != all) || from + kPage > least,
                                 sees ? limit - from : 0, g, a.scale_log2);
      }
    }
  };
  pages(std::false_type{});
  // A NaN may come from a token that its query does not see.
  float any = 0.0f;
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) any += w.acc[d][j] * 0.0f;
  if (__ballot(any != any) != 0) {
    w.clear();
    pages(std::true_type{});
  }
  float l = w.l + __shfl_xor(w.l, 16);
  l += __shfl_xor(l, 32);

#pragma unroll
  for (int d = 0; d < D / 16; ++d) *(v4f*)&lds_o[(wave * 16 + col) * P + d * 16 + 4 * g] = w.acc[d];
  if (g == 0) lds_ml[wave][col][0] = w.m, lds_ml[wave][col][1] = l;
  __syncthreads();
  const int d0 = threadIdx.x % C * 8;
  const int used = GROUP ? u.n * a.group : min(16, a.group - u.q0);
  for (int i = threadIdx.x / C; i < used; i += kThreads / C) {
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
    const int64_t row = u.row + (GROUP ? i / a.group : 0);
    const int oh = u.h * a.group + (GROUP ? i % a.group : u.q0 + i);
    if (a.splits == 1) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      u32x2_t* op = (u32x2_t*)(a.out + row * a.o_ts + oh * a.o_hs + d0);
      op[0] = u32x2_t{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv)};
      op[1] = u32x2_t{pack2<DT>(o[4] * inv, o[5] * inv), pack2<DT>(o[6] * inv, o[7] * inv)};
    } else {
      const int64_t pr = (row * a.q_heads + oh) * a.splits + u.split;
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
__global__ __launch_bounds__(kThreads) void join_chosen(Args a) {
  const int64_t row = blockIdx.x, rows = (int64_t)a.T * a.q_heads;
  if (a.c.cu && !a.tail && row / a.q_heads >= a.c.cu[a.c.sequences]) return;
  join_row<DT, D>(a.part + row * a.splits * D, D,
                  a.part + rows * a.splits * D + row * a.splits * 2, 2, a.splits,
                  a.out + row / a.q_heads * a.o_ts + row % a.q_heads * a.o_hs);
}

// How a call is cut up: a function of its sizes only.
struct Plan {
  int rows;             // of a unit
  int64_t tiles, units;  // of rows, over all sequences; with heads and operands of 16 queries
  int parts, splits;
  int64_t floats(int64_t T, int64_t q_heads, int64_t D) const {
    return splits > 1 ? T * q_heads * splits * (D + 2) : 0;
  }
};

Plan plan_selected(const fvsr_kv_cache* c, int64_t T, int64_t q_heads, int64_t top) {
  Plan p{};
  const int64_t cus = 256, B = c->sequences, group = q_heads / c->heads;
  const int64_t each = c->cu ? (T > B ? T : 1) : T / B;  // rows of a sequence at most
  p.rows = (int)std::max<int64_t>(
      1, std::min<int64_t>({16 / std::min<int64_t>(group, 16), each,
                            kEntries / std::max<int64_t>(top, 1)}));
  p.parts = (int)((group + 15) / 16);
  p.tiles = c->cu ? T / p.rows + B + 1 : B * ((T / B + p.rows - 1) / p.rows);
  p.units = p.tiles * c->heads * p.parts;
  p.splits = (int)std::min<int64_t>({std::max<int64_t>(1, 2 * cus / p.units),
                                     std::max<int64_t>(1, top / 4), kMaxSplits});
  return p;
}

template <int DT, int D>
void launch(const Args& a, const Plan& p, hipStream_t st) {
  const dim3 block(kThreads), grid((unsigned)(p.units * p.splits));
  if (p.rows > 1)
    hipLaunchKernelGGL((attend_chosen<DT, D, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((attend_chosen<DT, D, false>), grid, block, 0, st, a);
  if (p.splits > 1)
    hipLaunchKernelGGL((join_chosen<DT, D>), dim3((unsigned)((int64_t)a.T * a.q_heads)), block, 0,
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
  if (p.units * p.splits > kMaxBlocks) return FVSR_EUNSUPPORTED;
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
  a.rows = p.rows, a.tiles = (int)p.tiles;
  const hipStream_t st = (hipStream_t)stream;
  const bool half = dtype == FVSR_DT_F16;
  if (cache->head_dim == 128)
    half ? launch<FVSR_DT_F16, 128>(a, p, st) : launch<FVSR_DT_BF16, 128>(a, p, st);
  else
    half ? launch<FVSR_DT_F16, 64>(a, p, st) : launch<FVSR_DT_BF16, 64>(a, p, st);
  return fvsr_launch_status();
}
