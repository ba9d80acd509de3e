// Attention of each row over pages of its own choice, in an 8-bit paged cache:
//
//   o[q] = sum_k w[k] v[k] / sum_k w[k],  w[k] = exp(sm_scale * q.k) over the tokens up to
//          q's own position in the pages of its list
//
// A list belongs to a row and a key/value head.  Operands, weights and their precision are those of
// paged_attn.hip: K and V are operand A as stored, q and the weights sums of e4m3 terms.  (fp16 weights
// as halves alone, 2^-11 of themselves, would take 61 of the 74 us below, and of 128 dims 110 of 116;
// halves and an e4m3 term for what they leave 3 % less than three terms for 64 dims, 4 % more
// for 128.)  An operand has 16 query columns; a head's group seldom fills them, so a unit of work is as
// many rows that follow one another as do, over the pages that any of them lists, each page read and
// multiplied once.
//
// Two kernels.  attend_chosen: single tokens, whose pages come from memory, or few units: four
// waves to a unit, and workgroups where units are too few.  attend_alone: units of rows that stand
// together: one to four waves to a unit, each on pages of its own by way of LDS.
//
// Measured, 32 query and 8 key/value heads of 128 in bf16: one token over 64 of 2047 pages 11.7 us (17
// MB), 128 tokens over 32 pages each 171 us (5.45 TB/s; a copy reaches 5.2); 2048 rows of a prompt
// over 16 of 250 pages, 16 / 4 heads of 64 in fp16, 74 us (233 TFLOP/s of what the rows ask for; 46
// us of vector instructions a SIMD, 20 of matrix ones, and some 12 TB/s from the L2).
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
constexpr int kShared = 1024, kAlone = 256;  // entries at most
template <int N>
struct Lists {
  int column[N];     // as listed, row by row; kNone where a row does not see it
  uint32_t rows[N];  // 0: a row before it lists the same
  int falls;
};
constexpr int kNone = INT32_MAX;

// Rows of one sequence that stand together want much the same pages.  A page that several
// rows list is read and multiplied once for all of them.  Rising lists (as select_pages gives
// them) are searched for each other's columns; if one of them is not, each entry stands for itself.
template <int THREADS, int N>
FVSR_DEV void join_lists(Lists<N>& l, const Args& a, const Unit& u) {
  const int total = u.n * a.top, H = (int)a.c.heads;
  if (threadIdx.x == 0) l.falls = 0;
  for (int e = threadIdx.x; e < total; e += THREADS) {
    const int i = e / a.top;
    const int c = a.columns[((int64_t)(u.row + i) * H + u.h) * a.top + e % a.top];
    l.column[e] = c >= 0 && c < pages_of(limit_of(a, u, i)) ? c : kNone;
  }
  __syncthreads();
  bool falls = false;
  for (int e = threadIdx.x; e < total; e += THREADS)
    falls |= e % a.top > 0 && l.column[e] != kNone && l.column[e - 1] >= l.column[e];
  if (falls) l.falls = 1;
  __syncthreads();
  const bool search = l.falls == 0;
  for (int e = threadIdx.x; e < total; e += THREADS) {
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

  // A page, of which this lane's query sees the first `seen` tokens; `cut`: some query of the
  // wave sees a part of it only, otherwise each sees all or (seen <= 0) nothing.  k_tile(t) and
  // v_tile(d) are its operands, k_done() and v_first() are called behind the last of K's and before
  // the first of V's.  Hidden tokens weigh
  // 0, which a NaN among their codes would not survive: CAREFUL hides each logit, takes V's
  // NaN codes out of the product and counts them where they are seen.
  template <bool CAREFUL, class K, class V, class Done, class First>
  __device__ __forceinline__ void page(K k_tile, V v_tile, Done k_done, First v_first, int ks,
                                       int vs, bool cut, int seen, int g, float scale_log2) {
    v4f sc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const v8i kf = k_tile(t);
      const v4f z = {};
      sc[t] = mfma(kf, qf[0], z, ks, qs[0]);
#pragma unroll
      for (int k = 1; k < F; ++k) sc[t] = mfma(kf, qf[k], sc[t], ks, qs[k]);
    }
    k_done();
    // Accumulator (t, j) of lane g is position 64 (t / 4) + 16 g + 4 (t % 4) + j.
    const auto at = [](int t, int j) { return (t >> 2) * 64 + (t & 3) * 4 + j; };
    const int left = seen - 16 * g;
    if (CAREFUL || cut) {
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
    top = seen > 0 ? top : -__builtin_huge_valf();
    int shift;
    weigh(sc, top, scale_log2, m, l, shift, [&](float f) {
#pragma unroll
      for (int d = 0; d < DT16; ++d) acc[d] *= f;
    }, seen > 0 ? 0.0f : -__builtin_huge_valf());
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
    v_first();
#pragma unroll
    for (int d = 0; d < DT16; ++d) {
      v8i vf = v_tile(d);
      if constexpr (CAREFUL) {
        if (vs == 255)  // a page of NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) vf[i] = 0x7f7f7f7f;
        const v8i nans = take_nan(vf);
        const v4f z = {};
        const v4f n = mfma(nans, ones, z, 127, 127);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n[j] > 0.0f) acc[d][j] = __builtin_nanf("");
      }
#pragma unroll
        for (int k = 0; k < N; ++k)
          acc[d] = mfma(vf, pf[k], acc[d], CAREFUL && vs == 255 ? 127 : vs, e8m0(shift - 5 * k));
    }
  }

  // The same with operands straight from memory: all at once, or (CAREFUL, which is rare and keeps
  // no more registers than it needs) one by one.
  template <bool CAREFUL>
  __device__ __forceinline__ void page_from(const uint8_t* kp, int k_off, const uint8_t* vp,
                                            int v_off, int ks, int vs, bool cut, int seen, int g,
                                            float scale_log2) {
    // (Opaque, so that no sums with them are kept in registers from page to page.)
    asm volatile("" : "+v"(k_off), "+v"(v_off));
    kp += k_off, vp += v_off;
    const auto k_load = [&](int t) {
      const uint8_t* x = kp + ((t >> 2) * 64 + (t & 3) * 4) * D;
      const u32x4_t y = *(const u32x4_t*)x;
      return ::join(y, D == 128 ? *(const u32x4_t*)(x + 64) : y);
    };
    const auto v_load = [&](int d) {
      const uint8_t* x = vp + d * 16 * kPage;
      return ::join(*(const u32x4_t*)x, *(const u32x4_t*)(x + 64));
    };
    const auto nothing = [] {};
    if constexpr (CAREFUL) {
      const auto apart = [](auto load) {
        return [load](int i) {
          asm volatile("" ::: "memory");
          return load(i);
        };
      };
      page<true>(apart(k_load), apart(v_load), nothing, nothing, ks, vs, cut, seen, g, scale_log2);
    } else {
      v8i kf[8], vf[DT16];
#pragma unroll
      for (int t = 0; t < 8; ++t) kf[t] = k_load(t);
#pragma unroll
      for (int d = 0; d < DT16; ++d) vf[d] = v_load(d);
      page<false>([&](int t) { return kf[t]; }, [&](int d) { return vf[d]; }, nothing, nothing, ks, vs,
                  cut, seen, g, scale_log2);
    }
  }

  // Whether O has a NaN (or an infinity), which may come from a token that its query does not see.
  __device__ __forceinline__ bool broken() const {
    float any = 0.0f;
#pragma unroll
    for (int d = 0; d < DT16; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) any += acc[d][j] * 0.0f;
    return __ballot(any != any) != 0;
  }
};

// What a workgroup's waves have of a unit's rows, added up and written.
template <int DT, int D, int WAVES>
FVSR_DEV void join_waves(const Queries<DT, D>& w, float l, float* lds_o, float (&lds_ml)[WAVES][16][2],
                         const Args& a, const Unit& u) {
  constexpr int P = D + 4, C = D / 8;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  const int used = a.parts > 1 ? min(16, a.group - u.q0) : u.n * a.group;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) *(v4f*)&lds_o[(wave * 16 + col) * P + d * 16 + 4 * g] = w.acc[d];
  if (g == 0) lds_ml[wave][col][0] = w.m, lds_ml[wave][col][1] = l;
  __syncthreads();
  const int d0 = threadIdx.x % C * 8;
  for (int i = threadIdx.x / C; i < used; i += 64 * WAVES / C) {
    float top = lds_ml[0][i][0];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) top = fmaxf(top, lds_ml[v][i][0]);
    float o[8] = {}, sum = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      const float f = __builtin_amdgcn_exp2f(lds_ml[v][i][0] - top);
      sum += f * lds_ml[v][i][1];
      const v4f x = *(const v4f*)&lds_o[(v * 16 + i) * P + d0];
      const v4f y = *(const v4f*)&lds_o[(v * 16 + i) * P + d0 + 4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += f * x[j], o[4 + j] += f * y[j];
    }
    const int64_t row = u.row + (a.parts > 1 ? 0 : i / a.group);
    const int oh = u.h * a.group + (a.parts > 1 ? u.q0 + i : i % a.group);
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

// A workgroup's waves take the pages of a unit in turn (of all that its splits have, every
// splits * WAVES-th) and add what they have.  GROUP: several rows to a unit, row i's queries in
// columns i * group and on.
template <int DT, int D, bool GROUP>
__global__ __launch_bounds__(kThreads, D == 64 ? 3 : 2) void attend_chosen(Args a) {
  constexpr int WAVES = kThreads / 64;
  __shared__ __attribute__((aligned(16))) float lds_o[WAVES * 16 * (D + 4)];
  __shared__ float lds_ml[WAVES][16][2];
  __shared__ std::conditional_t<GROUP, Lists<kShared>, int> lists;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, H = (int)a.c.heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Unit u;
  if (!unit_of(a, xcd_order(blockIdx.x, gridDim.x), u)) return;
  if constexpr (GROUP) join_lists<kThreads>(lists, a, u);
  const int mine = GROUP ? min(col / a.group, u.n - 1) : 0;  // this lane's row of the unit
  const int head = GROUP ? col % a.group : min(u.q0 + col, a.group - 1);
  const int limit = limit_of(a, u, mine), least = limit_of(a, u, 0);
  const int32_t* const list = a.columns + ((int64_t)u.row * H + u.h) * a.top;
  const int32_t* const table = a.c.table + (int64_t)u.s.b * a.c.table_stride;
  const int total = u.n * a.top, turn = u.split * WAVES + wave, turns = a.splits * WAVES;
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
        w.template page_from<careful>((const uint8_t*)a.c.k + at, k_off, (const uint8_t*)a.c.v + at,
                                      v_off, s & 255, s >> 8,
                                 from + kPage > least, sees ? limit - from : 0, g, a.scale_log2);
      }
    }
  };
  pages(std::false_type{});
  if (w.broken()) {
    w.clear();
    pages(std::true_type{});
  }
  join_waves<DT, D, WAVES>(w, w.l, lds_o, lds_ml, a, u);
}

// Units of rows that stand together.  Straight loads of an operand touch a cache line for each of
// their 16 rows, four times what its bytes need, and that, not the bytes, is what bounds them
// where pages come from the L2.  Here a page's codes go to LDS in whole lines, K and then V into a
// wave's one buffer (64 dims: 8 KB, 128: 16), and other waves of the SIMD work meanwhile; nobody
// waits for another wave before the end, where a unit's waves add up what they have of its pages.
// (2048 rows, 32 / 8 heads of 128 in bf16, a wave to a unit: 200 us; a buffer each for K and V, which
// leaves a SIMD one wave, 244.)
//
// 16-byte pieces of LDS rows are swapped about so that the 16 lanes that read a piece of 16
// rows touch every bank once: rows of a K operand differ in token bits 0, 1, 4 and 5
// (128-byte rows: bit 0 is the bank half, 64-byte rows: bits 0-1 the quarter), those of V in dim
// bits 0-3.
template <int D>
FVSR_DEV int k_swap(int key) {
  return D == 128 ? ((key >> 1) & 1) | ((key >> 3) & 6) : (key >> 4) & 3;
}
FVSR_DEV int v_swap(int d) { return (d >> 1) & 7; }

// 4 KB from `from` to LDS at `to`: the 16 bytes at from + 1024 i + off[i] of each lane go to to +
// 1024 i, lane by lane.  (Written out: the compiler, which cannot tell K's loads from V's, would wait
// for all of them before any read.  It is the callers who wait; the loads have no registers
// that could be read too early.  The offset counts for both addresses.  Nothing else here uses m0.)
FVSR_DEV void fetch(const uint8_t* to, const uint8_t* from, const int (&off)[4]) {
  const uint32_t lds = (uint32_t)(uintptr_t)(const uint8_t LDS_AS*)to;
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %5\n\t"
      "global_load_lds_dwordx4 %2, %5 offset:%6\n\t"
      "global_load_lds_dwordx4 %3, %5 offset:%7\n\t"
      "global_load_lds_dwordx4 %4, %5 offset:%8"
      :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off[0]), "v"(off[1]), "v"(off[2]),
      "v"(off[3]), "s"(from), "n"(1 << 10), "n"(2 << 10), "n"(3 << 10) : "memory");
}
// Until at most N of them are on their way.
template <int N>
FVSR_DEV void wait_for() {
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

struct Visit {
  int id, column;
  uint32_t what;  // scales of K and V, and (16 bits) the rows that list it
};

template <int DT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void attend_alone(Args a) {
  constexpr int KR = D / 16;                 // pieces of a K row
  constexpr int SEG = kPage * D / 1024;      // of 64 pieces
  constexpr int BUF = kPage * D;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[BUF * WAVES];
  const int wave = WAVES > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  uint8_t* const own = lds + wave * BUF;  // K's codes or V's
  __shared__ Visit visits[kAlone];
  // The lists lie where codes will.
  static_assert(sizeof(Lists<kAlone>) <= BUF, "lists outgrow the codes");
  Lists<kAlone>& lists = *(Lists<kAlone>*)lds;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, H = (int)a.c.heads;
  Unit u;
  if (!unit_of(a, xcd_order(blockIdx.x, gridDim.x), u)) return;
  join_lists<64 * WAVES>(lists, a, u);
  const int mine = min(col / (a.parts > 1 ? 16 : a.group), u.n - 1);
  const int head = a.parts > 1 ? min(u.q0 + col, a.group - 1) : col % a.group;
  const int limit = limit_of(a, u, mine), least = limit_of(a, u, 0);
  const int32_t* const table = a.c.table + (int64_t)u.s.b * a.c.table_stride;
  Queries<DT, D> w;
  w.load(a.q + (int64_t)(u.row + mine) * a.q_ts + (int64_t)(u.h * a.group + head) * a.q_hs, g);
  int n = 0, wrong = 0;
  for (int e0 = 0; e0 < u.n * a.top; e0 += 64) {
    const int e = e0 + lane;
    const int c = e < u.n * a.top ? lists.column[e] : kNone;
    const uint32_t rows = c != kNone ? lists.rows[e] : 0;
    const int id = rows ? table[c] : -1;
    const bool good = id >= 0 && id < a.c.pages;
    for (uint64_t bad = __ballot(rows && !good); bad; bad &= bad - 1)
      wrong |= __builtin_amdgcn_readlane(rows, __builtin_ctzll(bad));
    const uint64_t there = __ballot(good);
    if (good) {
      const int64_t ph = (int64_t)id * H + u.h;
      visits[n + __popcll(there & ((1ull << lane) - 1))] =
          Visit{id, c,
                ((const uint8_t*)a.c.k_scale)[ph] |
                    (uint32_t)((const uint8_t*)a.c.v_scale)[ph] << 8 | rows << 16};
    }
    n += __popcll(there);
  }
  __syncthreads();
  const auto visit = [&](int i) {
    const Visit& v = visits[i];
    return Visit{__builtin_amdgcn_readfirstlane(v.id), __builtin_amdgcn_readfirstlane(v.column),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)v.what)};
  };
  const auto seen_of = [&](const Visit& v) {  // tokens of the page that this lane's query sees
    return (v.what >> (16 + mine) & 1) != 0 ? limit - v.column * kPage : 0;
  };
  const auto codes = [&](const void* p, const Visit& v) {
    return (const uint8_t*)p + ((int64_t)v.id * H + u.h) * kPage * D;
  };
  // What a lane fetches of segment s belongs where it lands: row s * 64 / KR + lane / KR, piece
  // lane % KR, holds the piece with that number and the row's swap.
  const auto fetch_k = [&](const Visit& v) {
    const uint8_t* from = codes(a.c.k, v);
#pragma unroll
    for (int s = 0; s < SEG; s += 4) {
      int off[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        off[i] = lane / KR * D +
                 ((lane % KR) ^ k_swap<D>((s + i) * (64 / KR) + lane / KR)) * 16;
      fetch(own + s * 1024, from + s * 1024, off);
    }
  };
  const auto fetch_v = [&](const Visit& v) {
    const uint8_t* from = codes(a.c.v, v);
#pragma unroll
    for (int s = 0; s < SEG; s += 4) {
      int off[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        off[i] = lane / 8 * kPage + ((lane % 8) ^ v_swap((s + i) * 8 + lane / 8)) * 16;
      fetch(own + s * 1024, from + s * 1024, off);
    }
  };
  // Row r of K subtile t is key 64 (t / 4) + 16 (r / 4) + 4 (t % 4) + r % 4.  (64 dims stand in
  // both halves of an operand: they are read twice, which costs less than copies of registers.)
  const int k_first = 16 * (col >> 2) + (col & 3);
  int k_again = k_first * D + (g ^ k_swap<D>(k_first)) * 16;
  asm("" : "+v"(k_again));
  const auto k_tile = [&](int t) {
    const int key = 64 * (t >> 2) + k_first + 4 * (t & 3);
    const uint8_t* row = own + key * D;
    const u32x4_t x = *(const u32x4_t*)(row + (g ^ k_swap<D>(key)) * 16);
    return ::join(x, D == 128 ? *(const u32x4_t*)(row + ((g + 4) ^ k_swap<D>(key)) * 16)
                              : *(const u32x4_t*)(own + k_again + (key - k_first) * D));
  };
  const auto v_tile = [&](int d) {
    const int dim = d * 16 + col;
    const uint8_t* row = own + dim * kPage;
    return ::join(*(const u32x4_t*)(row + (g ^ v_swap(dim)) * 16),
                  *(const u32x4_t*)(row + ((g + 4) ^ v_swap(dim)) * 16));
  };
  if (wave < n) {
    Visit cur = visit(wave);
    fetch_k(cur);
    for (int i = wave; i < n; i += WAVES) {
      const Visit next = visit(i + WAVES < n ? i + WAVES : i);  // (the last one again: no branch)
      const uint32_t what = cur.what;
      wait_for<0>();
      w.template page<false>(k_tile, v_tile, [&] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K's operands are read
        fetch_v(cur);
      }, [&] { wait_for<0>(); }, what & 255, what >> 8 & 255, (cur.column + 1) * kPage > least,
          seen_of(cur), g, a.scale_log2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and V's
      fetch_k(next);
      cur = next;
    }
    wait_for<0>();  // no load may land in an LDS that the next workgroup has
  }
  if (w.broken()) {
    w.clear();
    const int k_off = (16 * (col >> 2) + (col & 3)) * D + 16 * g, v_off = col * kPage + 16 * g;
    for (int i = wave; i < n; i += WAVES) {
      const Visit v = visit(i);
      w.template page_from<true>(codes(a.c.k, v), k_off, codes(a.c.v, v), v_off, v.what & 255,
                                 v.what >> 8 & 255, true, seen_of(v), g, a.scale_log2);
    }
  }
  if (wrong >> mine & 1) w.l = __builtin_nanf("");  // no such page: the rows that list it are NaN
  if constexpr (WAVES > 1) {
    __shared__ float lds_ml[WAVES][16][2];
    static_assert(16 * (D + 4) * 4 <= BUF, "sums outgrow the codes");
    __syncthreads();  // (codes are read, and no load is on its way)
    join_waves<DT, D, WAVES>(w, w.l, (float*)lds, lds_ml, a, u);
    return;
  }
  float l = w.l + __shfl_xor(w.l, 16);
  l += __shfl_xor(l, 32);
  if (col >= (a.parts > 1 ? min(16, a.group - u.q0) : u.n * a.group)) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* op = a.out + (int64_t)(u.row + mine) * a.o_ts + (u.h * a.group + head) * a.o_hs + 4 * g;
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
    *(u32x2_t*)(op + d * 16) = u32x2_t{pack2<DT>(w.acc[d][0] * inv, w.acc[d][1] * inv),
                                       pack2<DT>(w.acc[d][2] * inv, w.acc[d][3] * inv)};
}

template <int DT, int D>
__global__ __launch_bounds__(kThreads) void join_chosen(Args a) {
  const int64_t row = blockIdx.x, rows = (int64_t)a.T * a.q_heads;
  if (a.c.cu && !a.tail && row / a.q_heads >= a.c.cu[a.c.sequences]) return;
  join_row<DT, D>(a.part + row * a.splits * D, D,
                  a.part + rows * a.splits * D + row * a.splits * 2, 2, a.splits,
                  a.out + row / a.q_heads * a.o_ts + row % a.q_heads * a.o_hs);
}

// How a call is cut up: a function of its sizes (and the CUs) only.
struct Plan {
  int rows;              // of a unit
  int64_t tiles, units;  // of rows, over all sequences; with heads and operands of 16 queries
  int parts, splits;
  int alone;             // attend_alone: waves to a unit (or 0)
  int64_t floats(int64_t T, int64_t q_heads, int64_t D) const {
    return splits > 1 ? T * q_heads * splits * (D + 2) : 0;
  }
};

Plan plan_selected(const fvsr_kv_cache* c, int64_t T, int64_t q_heads, int64_t top) {
  Plan p{};
  const int64_t cus = cu_count(), B = c->sequences, group = q_heads / c->heads;
  const int64_t each = c->cu ? (T > B ? T : 1) : T / B;  // rows of a sequence at most
  const auto cut = [&](int64_t entries) {
    p.rows = (int)std::max<int64_t>(
        1, std::min<int64_t>({16 / std::min<int64_t>(group, 16), each,
                              entries / std::max<int64_t>(top, 1)}));
    p.tiles = c->cu ? T / p.rows + B + 1 : B * ((T / B + p.rows - 1) / p.rows);
    p.units = p.tiles * c->heads * p.parts;
  };
  p.parts = (int)((group + 15) / 16);
  p.splits = 1;
  cut(kAlone);
  // Where rows of a sequence follow one another and there are units for half the CUs: as many
  // waves to a unit, up to four, as all units have room for at a time (LDS holds 16 of 64 dims or 8 of
  // 128 on a CU).  us with 1, 2 and 4 waves, and by attend_chosen, in bf16; 64 dims: 128 units 41,
  // 26, 19 and 19, 512 46, 37, 25 and 30, 1024 50, 41, 38 and 53, 2048 67, 63, 67 and 88; 128 dims:
  // 256 units 57, 36, 26 and 42, 512 59, 47, 34 and 62, 1024 69, 57, 62 and 112, 1400 86, 92, 85 and
  // 154, 2048 99, 113, 116 and 213.  (fp16: up to 25 % more, in the same order.)
  if (each > 1 && top <= kAlone && p.units * 2 >= cus) {
    const int64_t room = cus * (c->head_dim == 64 ? 16 : 8) / p.units;
    p.alone = room >= 4 ? 4 : room >= 2 || c->head_dim == 64 ? 2 : 1;
    return p;
  }
  cut(kShared);
  // Two workgroups to a CU, each with a page for every wave.
  p.splits = (int)std::min<int64_t>({std::max<int64_t>(1, 2 * cus / p.units),
                                     std::max<int64_t>(1, top / 4), kMaxSplits});
  return p;
}

template <int DT, int D>
void launch(const Args& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.units * p.splits)), block(kThreads);
  if (p.alone) {
    if (p.alone == 4)
      hipLaunchKernelGGL((attend_alone<DT, D, 4>), grid, dim3(256), 0, st, a);
    else if (D == 64 || p.alone == 2)
      hipLaunchKernelGGL((attend_alone<DT, D, 2>), grid, dim3(128), 0, st, a);
    else
      hipLaunchKernelGGL((attend_alone<DT, D, D == 64 ? 2 : 1>), grid, dim3(64), 0, st, a);
    return;
  }
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
